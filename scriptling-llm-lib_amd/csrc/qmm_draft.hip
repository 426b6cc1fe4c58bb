// Drafted tokens of a batch's step: the rules that logits pass before a token is chosen, the path of a tree that the
// choices accept, and the move of its rows in the cache.
#include <hip/hip_runtime.h>

#include <climits>

#include "qmm_pages.hpp"

namespace sllm {

namespace {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef int v4i __attribute__((ext_vector_type(4)));

// A step as a kernel reads it; what a call knows of it by value (a captured one takes it from the step's header).
struct StepRef {
    const int *step;
    int rows_at, seqs_at, of_at;  // -1: as the step says
    __device__ __forceinline__ const StepRow *rows() const {
        return (const StepRow *)(step + (rows_at >= 0 ? rows_at : step[kStepRowsAt]));
    }
    __device__ __forceinline__ const int *seqs() const { return step + (seqs_at >= 0 ? seqs_at : step[kStepSeqsAt]); }
    __device__ __forceinline__ const int *of() const { return step + (of_at >= 0 ? of_at : step[kStepOfAt]); }
};
StepRef step_ref(const PageBatch &b, bool capture) {
    return {b.dev, capture ? -1 : b.rows_at, capture ? -1 : b.seqs_at, capture ? -1 : b.of_at};
}

// ----------------------------------------------------------------- logits ----

constexpr int kChunk = 4096;  // elements of a workgroup
constexpr int kRuleThreads = 256;

struct LogitsArgs {
    const float *x;
    float *dst;
    int *chosen;
    int rows, vocab, chunks;
    sllm_logits_params p;
    bool batch;
    StepRef step;
    int2 *best;  // of every row and chunk: the largest value's bits and its index
};

// The first of two candidates in value, then in index. (A NaN is never one.)
__device__ __forceinline__ void better(float &v, int &i, float w, int j) {
    if (w > v || (w == v && j < i)) {
        v = w;
        i = j;
    }
}
__device__ __forceinline__ void wave_best(float &v, int &i) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) better(v, i, __shfl_xor(v, o, 64), __shfl_xor(i, o, 64));
}

// One workgroup per (row, chunk of the vocabulary). The row's tokens (its history, its node's path) that lie in the chunk
// are counted in LDS, a table entry for each element; then the chunk passes once through registers.
__global__ void __launch_bounds__(kRuleThreads) logits_rules_kernel(LogitsArgs a) {
    __shared__ __attribute__((aligned(16))) unsigned count[kChunk];
    __shared__ __attribute__((aligned(16))) unsigned bias[kChunk];  // 1 + the number of the element's bias, 0 without one
    __shared__ unsigned bits[kChunk / 32 + 2];
    __shared__ float wv[kRuleThreads / 64];
    __shared__ int wi[kRuleThreads / 64];
    const int r = blockIdx.y, tid = threadIdx.x;
    if (a.batch && r >= a.step.step[kStepRows]) return;
    const size_t row = (size_t)r * a.vocab;
    // elements are numbered from the 16-byte boundary at or before the row's first, so that fours are aligned
    const int lead = (int)(((uintptr_t)(a.x + row) >> 2) & 3), c0 = blockIdx.x * kChunk;
    const float *x = a.x + row - lead;
    float *dst = a.dst ? a.dst + row - lead : nullptr;
    const int end = a.vocab + lead;
    const int seq = a.batch ? a.step.of()[r] : r;
    sllm_logits_rule rule{1.0f, 0.0f, 0.0f, 0, 0, 0, 0, 0};
    if (seq < a.p.n_rules) rule = a.p.rules[seq];
    // (in 64 bits: a range may name any integers)
    auto range = [](int at, int n, int all, int64_t &from, int64_t &to) {
        from = at < 0 ? 0 : at;
        to = (int64_t)at + n < all ? (int64_t)at + n : all;
    };
    int64_t h0, h1, b0, b1;
    range(rule.history_at, rule.history, a.p.n_history, h0, h1);
    range(rule.bias_at, rule.biases, a.p.n_biases, b0, b1);
    const int mask = a.p.masks ? a.p.mask_ids[r] : -1;
    const bool masked = mask >= 0 && mask < a.p.n_masks;
    for (int i = tid; i < kChunk / 4; i += kRuleThreads) {
        ((v4i *)count)[i] = v4i{0, 0, 0, 0};
        ((v4i *)bias)[i] = v4i{0, 0, 0, 0};
    }
    if (masked) {
        const int words = (a.vocab + 31) / 32;
        const unsigned *m = (const unsigned *)a.p.masks + (size_t)mask * words;
        const int w0 = c0 / 32 - (c0 ? 1 : 0);  // (the first element may lie up to three before c0)
        for (int i = tid; i < kChunk / 32 + 2; i += kRuleThreads) bits[i] = w0 + i < words ? m[w0 + i] : 0u;
    }
    __syncthreads();
    auto add = [&](int t) {
        const unsigned i = (unsigned)t + (unsigned)(lead - c0);
        if (t >= 0 && t < a.vocab && i < kChunk) atomicAdd(&count[i], 1u);
    };
    for (int64_t i = h0 + tid; i < h1; i += kRuleThreads) add(a.p.history[i]);
    if (a.batch && a.p.tokens) {
        const StepRow &me = a.step.rows()[r];
        const int first = a.step.seqs()[seq], base = me.end - 1 - (r - first);
        const uint16_t *sees = (const uint16_t *)a.step.step + me.tree;
        for (int j = first + tid; j <= r; j += kRuleThreads) {
            const int at = base + j - first;
            if (me.tree < 0 || sees[(at >> 4) - (base >> 4)] >> (at & 15) & 1) add(a.p.tokens[j]);
        }
    }
    for (int64_t i = b0 + tid; i < b1; i += kRuleThreads) {
        const int t = a.p.bias_tokens[i];
        const unsigned k = (unsigned)t + (unsigned)(lead - c0);
        if (t >= 0 && t < a.vocab && k < kChunk) atomicMax(&bias[k], (unsigned)(i - b0) + 1u);
    }
    __syncthreads();
    float bv = -INFINITY;
    int bi = INT_MAX;
    const int w0 = c0 ? c0 - 32 : 0;  // the element of bits' first bit
    for (int i = 4 * tid; i < kChunk; i += 4 * kRuleThreads) {
        const int e = c0 + i;
        if (e >= end) break;
        const bool whole = e >= lead && e + 4 <= end;
        v4f y;
        if (whole) y = *(const v4f *)(x + e);
        else
#pragma unroll
            for (int u = 0; u < 4; u++) y[u] = e + u >= lead && e + u < end ? x[e + u] : -INFINITY;
        const v4i n = *(const v4i *)(count + i), b = *(const v4i *)(bias + i);
#pragma unroll
        for (int u = 0; u < 4; u++) {
            if (n[u]) {
                float l = y[u];
                l = l > 0.0f ? l / rule.repeat : l * rule.repeat;
                y[u] = l - (rule.frequency * (float)(unsigned)n[u] + rule.presence);
            }
            if (b[u]) y[u] = y[u] + a.p.bias_values[b0 + (unsigned)b[u] - 1];
            const int t = e + u - lead;
            if (masked && t >= 0 && !(bits[(t - w0) >> 5] >> (t & 31) & 1)) y[u] = -INFINITY;
            if (t >= 0 && t < a.vocab) better(bv, bi, y[u], t);
        }
        if (!dst) continue;
        if (whole && ((uintptr_t)(dst + e) & 15) == 0) *(v4f *)(dst + e) = y;
        else
#pragma unroll
            for (int u = 0; u < 4; u++)
                if (e + u >= lead && e + u < end) dst[e + u] = y[u];
    }
    if (!a.chosen) return;
    wave_best(bv, bi);
    if ((tid & 63) == 0) {
        wv[tid >> 6] = bv;
        wi[tid >> 6] = bi;
    }
    __syncthreads();
    if (tid) return;
#pragma unroll
    for (int w = 1; w < kRuleThreads / 64; w++) better(bv, bi, wv[w], wi[w]);
    a.best[(size_t)r * a.chunks + blockIdx.x] = make_int2(__float_as_int(bv), bi);
}

// The chunks' candidates of a row, by one wave. (-inf is never chosen: -1 where nothing else is there.)
__global__ void __launch_bounds__(64) logits_choose_kernel(LogitsArgs a) {
    const int r = blockIdx.x;
    if (a.batch && r >= a.step.step[kStepRows]) return;
    float v = -INFINITY;
    int i = INT_MAX;
    for (int c = threadIdx.x; c < a.chunks; c += 64) {
        const int2 b = a.best[(size_t)r * a.chunks + c];
        better(v, i, __int_as_float(b.x), b.y);
    }
    wave_best(v, i);
    if (threadIdx.x == 0) a.chosen[r] = v == -INFINITY ? -1 : i;
}

// ------------------------------------------------------- accepted paths ----

// One workgroup per sequence. A row follows its parent where it holds the token chosen behind it (of several such rows the
// first); the path is the rows whose ancestors all follow.
constexpr int kAcceptThreads = 256;
__global__ void __launch_bounds__(kAcceptThreads) page_accept_kernel(StepRef st, const int *tokens, const int *chosen, int *kept,
                                                                     int *counts, int *next) {
    __shared__ int child[kTreeRows];
    __shared__ unsigned follows[kTreeRows / 16 + 2];
    __shared__ int n_path, last;
    const int s = blockIdx.x, tid = threadIdx.x;
    if (s >= st.step[kStepSeqs]) return;
    const int first = st.seqs()[s], n = st.seqs()[s + 1] - first;
    const StepRow *rows = st.rows() + first;
    if (!n) {
        if (tid == 0) {
            counts[s] = 0;
            next[s] = -1;
        }
        return;
    }
    const bool tree = rows[0].tree >= 0;
    if (tid == 0) {
        n_path = tree ? 0 : n;
        last = 0;
    }
    if (!tree) {
        // each row's parent is the one before it: the path ends before the first that does not follow
        __syncthreads();
        for (int r = 1 + tid; r < n; r += kAcceptThreads)
            if (tokens[first + r] != chosen[first + r - 1]) atomicMin(&n_path, r);
        __syncthreads();
        for (int r = tid; r < n; r += kAcceptThreads) kept[first + r] = r < n_path ? first + r : -1;
        if (tid == 0) {
            counts[s] = n_path;
            next[s] = chosen[first + n_path - 1];
        }
        return;
    }
    const int base = rows[0].end - 1, halves = ((base + n - 1) >> 4) - (base >> 4) + 1;
    for (int r = tid; r < n; r += kAcceptThreads) {
        child[r] = INT_MAX;
        kept[first + r] = -1;
    }
    // (rows before the tree count as following)
    for (int i = tid; i < halves; i += kAcceptThreads) follows[i] = i ? 0u : (1u << (base & 15)) - 1u | 1u << (base & 15);
    __syncthreads();
    for (int r = 1 + tid; r < n; r += kAcceptThreads) {
        const int up = rows[r].parent;
        if (up >= 0 && tokens[first + r] == chosen[up]) atomicMin(&child[up - first], r);
    }
    __syncthreads();
    for (int r = 1 + tid; r < n; r += kAcceptThreads) {
        const int up = rows[r].parent, at = base + r;
        if (up >= 0 && child[up - first] == r) atomicOr(&follows[(at >> 4) - (base >> 4)], 1u << (at & 15));
    }
    __syncthreads();
    for (int r = tid; r < n; r += kAcceptThreads) {
        const uint16_t *sees = (const uint16_t *)st.step + rows[r].tree;
        bool in = true;
        for (int i = 0; i < halves; i++) in = in && !(sees[i] & ~follows[i]);
        if (!in) continue;
        kept[first + rows[r].pos - base] = first + r;
        atomicAdd(&n_path, 1);
        atomicMax(&last, r);
    }
    __syncthreads();
    if (tid == 0) {
        counts[s] = n_path;
        next[s] = chosen[first + last];
    }
}

// ----------------------------------------------------------- kept rows ----

struct KeepArgs {
    StepRef step;
    const int *kept;
    char *pool_k, *pool_v;
    int n_pages, n_kv, page_rows, pieces;  // pieces: 16-byte pieces of a row of a head
    size_t layer_bytes;
};

// One workgroup per (sequence, K or V of a layer). A thread has one 16-byte column of a head and moves the path's rows
// there in order: a row goes to a place at or before its own, so that nothing is overwritten before it has been read.
constexpr int kKeepThreads = 256;
__global__ void __launch_bounds__(kKeepThreads) page_keep_kernel(KeepArgs a) {
    __shared__ int2 from[kKeepThreads], to[kKeepThreads];  // page and row of it
    __shared__ int n_moves, first_move;
    const int s = blockIdx.x, tid = threadIdx.x;
    if (s >= a.step.step[kStepSeqs]) return;
    const int first = a.step.seqs()[s], n = a.step.seqs()[s + 1] - first;
    const StepRow *rows = a.step.rows();
    char *pool = (blockIdx.y & 1 ? a.pool_v : a.pool_k) + (blockIdx.y >> 1) * a.layer_bytes;
    for (int j0 = 0; j0 < n; j0 += kKeepThreads) {
        if (tid == 0) first_move = n_moves = min(kKeepThreads, n - j0);
        __syncthreads();
        if (j0 + tid < n) {
            const int k = a.kept[first + j0 + tid];
            // the path ends before the first place without a row (one that is not a later row of the sequence is none)
            if (k < first + j0 + tid || k >= first + n) {
                atomicMin(&n_moves, tid);
            } else {
                if (k != first + j0 + tid) atomicMin(&first_move, tid);
                from[tid] = make_int2(rows[k].page, rows[k].slot);
                to[tid] = make_int2(rows[first + j0 + tid].page, rows[first + j0 + tid].slot);
            }
        }
        __syncthreads();
        const int m = n_moves;
        for (int c = tid; c < a.n_kv * a.pieces; c += kKeepThreads) {
            const int head = c / a.pieces, piece = c - head * a.pieces;
            auto at = [&](int2 p) {
                return (v4i *)pool + (((size_t)p.x * a.n_kv + head) * a.page_rows + p.y) * a.pieces + piece;
            };
            for (int j = first_move; j < m; j += 4) {
                v4i v[4];
#pragma unroll
                for (int u = 0; u < 4; u++)
                    if (j + u < m) v[u] = *at(from[j + u]);
#pragma unroll
                for (int u = 0; u < 4; u++)
                    if (j + u < m) *at(to[j + u]) = v[u];
            }
        }
        __syncthreads();
        if (m < kKeepThreads) break;
    }
}

}  // namespace

}  // namespace sllm

using namespace sllm;

extern "C" {

sllm_status sllm_logits_rules_dev(const float *logits, int rows, int vocab, const sllm_logits_params *p, float *dst,
                                  int *chosen, const sllm_page_batch *batch, void *stream) {
    return guarded([&]() -> sllm_status {
        if (!logits || !p || (!dst && !chosen)) return set_error(SLLM_ERR_ARG, "null pointer");
        if (rows < 0 || vocab <= 0) return set_error(SLLM_ERR_ARG, "rows must not be negative, vocab positive");
        if (p->n_rules < 0 || p->n_history < 0 || p->n_biases < 0 || p->n_masks < 0) return set_error(SLLM_ERR_ARG, "negative count");
        if ((p->n_rules && !p->rules) || (p->n_history && !p->history) || (p->n_biases && (!p->bias_tokens || !p->bias_values)) ||
            (p->n_masks && (!p->masks || !p->mask_ids)))
            return set_error(SLLM_ERR_ARG, "null pointer");
        if (((uintptr_t)logits | (uintptr_t)dst | (uintptr_t)p->rules) & 3) return set_error(SLLM_ERR_ARG, "misaligned pointer");
        if (rows > 65535) return set_error(SLLM_ERR_SHAPE, "at most 65535 rows");
        if (vocab > (1 << 28)) return set_error(SLLM_ERR_SHAPE, "vocab must be at most 2^28");
        hipStream_t s = (hipStream_t)stream;
        LogitsArgs a{};
        if (batch) {
            PageBatch &b = const_cast<sllm_page_batch *>(batch)->b;
            std::lock_guard<std::mutex> lb(b.mu);
            {
                std::lock_guard<std::mutex> lk(b.c->mu);
                const sllm_status st = step_stands(b);
                if (st != SLLM_OK) return st;
            }
            sllm_status st = on_device(b.c->device);
            if (st != SLLM_OK) return st;
            const bool capture = stream_capturing(s);
            if (capture ? rows < b.rows : rows != b.rows) return set_error(SLLM_ERR_SHAPE, "rows differ from those of the batch's step");
            a.batch = true;
            a.step = step_ref(b, capture);
            b.captured |= capture;
        }
        if (!rows) return SLLM_OK;
        sllm_status st = library_init();
        if (st != SLLM_OK) return st;
        a.x = logits;
        a.dst = dst;
        a.chosen = chosen;
        a.rows = rows;
        a.vocab = vocab;
        a.chunks = (vocab + 3 + kChunk - 1) / kChunk;
        a.p = *p;
        if (!p->n_masks) a.p.masks = nullptr;
        if (chosen) {
            void *ws = nullptr;
            size_t cap = 0;
            st = stream_workspace(s, (size_t)rows * a.chunks * sizeof(int2), &ws, &cap);
            if (st != SLLM_OK) return st;
            a.best = (int2 *)ws;
        }
        hipLaunchKernelGGL(logits_rules_kernel, dim3((unsigned)a.chunks, (unsigned)rows), dim3(kRuleThreads), 0, s, a);
        SLLM_HIP(hipGetLastError());
        if (!chosen) return SLLM_OK;
        hipLaunchKernelGGL(logits_choose_kernel, dim3((unsigned)rows), dim3(64), 0, s, a);
        SLLM_HIP(hipGetLastError());
        return SLLM_OK;
    });
}

sllm_status sllm_page_accept_dev(sllm_page_batch *batch, const int *tokens, const int *chosen, int *kept, int *counts,
                                 int *next, void *stream) {
    return guarded([&]() -> sllm_status {
        if (!batch || !tokens || !chosen || !kept || !counts || !next) return set_error(SLLM_ERR_ARG, "null pointer");
        PageBatch &b = batch->b;
        std::lock_guard<std::mutex> lb(b.mu);
        {
            std::lock_guard<std::mutex> lk(b.c->mu);
            const sllm_status st = step_stands(b);
            if (st != SLLM_OK) return st;
        }
        const sllm_status st = on_device(b.c->device);
        if (st != SLLM_OK) return st;
        hipStream_t s = (hipStream_t)stream;
        const bool capture = stream_capturing(s);
        if (b.seqs.empty() && !capture) return SLLM_OK;
        hipLaunchKernelGGL(page_accept_kernel, dim3((unsigned)(capture ? b.max_seqs : (int)b.seqs.size())), dim3(kAcceptThreads), 0, s,
                           step_ref(b, capture), tokens, chosen, kept, counts, next);
        SLLM_HIP(hipGetLastError());
        b.captured |= capture;
        return SLLM_OK;
    });
}

sllm_status sllm_page_keep_dev(sllm_page_batch *batch, const int *kept, void *stream) {
    return guarded([&]() -> sllm_status {
        if (!batch || !kept) return set_error(SLLM_ERR_ARG, "null pointer");
        PageBatch &b = batch->b;
        std::lock_guard<std::mutex> lb(b.mu);
        const PageCache &c = *b.c;
        {
            std::lock_guard<std::mutex> lk(b.c->mu);
            const sllm_status st = step_stands(b);
            if (st != SLLM_OK) return st;
            for (size_t i = 0; i < b.seqs.size(); i++) {
                const PageSeq &q = c.seqs[(size_t)b.seqs[i]];
                for (int p = b.bases[i] >> c.shift; b.counts[i] && p <= (b.bases[i] + b.counts[i] - 1) >> c.shift; p++)
                    if (c.refs[(size_t)q.pages[(size_t)p]] > 1)
                        return set_error(SLLM_ERR_ARG, "a page of the step's rows is shared: fork behind the move");
            }
        }
        const sllm_status st = on_device(c.device);
        if (st != SLLM_OK) return st;
        hipStream_t s = (hipStream_t)stream;
        const bool capture = stream_capturing(s);
        if (b.seqs.empty() && !capture) return SLLM_OK;
        KeepArgs a{};
        a.step = step_ref(b, capture);
        a.kept = kept;
        a.pool_k = c.k;
        a.pool_v = c.v;
        a.n_pages = c.n_pages;
        a.n_kv = c.n_kv;
        a.page_rows = c.page_rows;
        a.pieces = c.d_k * c.elem() / 16;
        a.layer_bytes = (size_t)c.n_pages * c.n_kv * c.page_rows * c.d_k * c.elem();
        hipLaunchKernelGGL(page_keep_kernel, dim3((unsigned)(capture ? b.max_seqs : (int)b.seqs.size()), 2u * (unsigned)c.n_layers),
                           dim3(kKeepThreads), 0, s, a);
        SLLM_HIP(hipGetLastError());
        b.captured |= capture;
        return SLLM_OK;
    });
}

}  // extern "C"
