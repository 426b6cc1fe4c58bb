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

// A workgroup's barrier for what it shares in LDS; loads and stores of memory stay under way.
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

struct LogitsArgs {
    const float *x;
    float *dst;
    int *chosen;
    int vocab, chunks;
    sllm_logits_params p;
    bool batch, follow;  // follow: the step's rows are fewer than the launch has, maybe
    StepRef step;
    int2 *best;  // of every row and chunk: the largest value's bits and its index
};

// The largest value and the lowest index of a wave, in all lanes: the lanes of a row of 16 among themselves, then the four rows'.
template <class T, class F>
__device__ __forceinline__ T wave_all(T v, F better) {
    auto with = [&](auto moved) {
        const T o = __builtin_bit_cast(T, moved);
        v = better(o, v) ? o : v;
    };
    with(__builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0xb1, 0xf, 0xf, false));   // lane ^ 1
    with(__builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0x4e, 0xf, 0xf, false));   // lane ^ 2
    with(__builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0x141, 0xf, 0xf, false));  // the other quad of each 8 lanes
    with(__builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0x140, 0xf, 0xf, false));  // the other 8 lanes of each row
    const int mine = __builtin_bit_cast(int, v);
    v = __builtin_bit_cast(T, __builtin_amdgcn_readlane(mine, 0));
    with(__builtin_amdgcn_readlane(mine, 16));
    with(__builtin_amdgcn_readlane(mine, 32));
    with(__builtin_amdgcn_readlane(mine, 48));
    return v;
}
__device__ __forceinline__ float wave_max(float v) {
    return wave_all(v, [](float a, float b) { return a > b; });
}
__device__ __forceinline__ int wave_min(int v) {
    return wave_all(v, [](int a, int b) { return a < b; });
}

// One workgroup per (row, chunk of the vocabulary), 4 V elements to a thread, which it holds in registers from the first
// load to the store. The row's biases that lie in the chunk go into a table in LDS, an entry for each element (of a token
// named twice the later: the largest number), then, cleared, the counts of the row's tokens (its history, its node's path).
// Bound by the bytes of the logits where there are many rows, by the chain of loads (mask or rule, elements, tokens) where there are
// few; and by the tokens where histories are long, since each workgroup reads all of its row's: 64 rows of 128256 with
// no tokens, 4000 and 16000 to a row take 14.1, 17.4 and 23.1 us, without the values kept 9.8, 16.4 and 22.3 (4000 that are
// none of the vocabulary's: 16.5 and 13.1).
// 64 rows of 128256, histories of up to 4000, 2000 in the mean, 20 biases (67 MB, 13 us at a copy's rate): 15.2 us with the choice. The
// counted elements worked off from a list, a thread for each: 20.2; two tables, one value after the other: 30.8.
constexpr int kRuleThreads = 256;
template <int V>
__global__ void __launch_bounds__(kRuleThreads) logits_rules_kernel(LogitsArgs a) {
    constexpr int T = kRuleThreads, CH = 4 * V * T;
    __shared__ __attribute__((aligned(16))) unsigned table[CH];
    __shared__ unsigned bits[CH / 32 + 2];
    __shared__ float wv[T / 64];
    __shared__ int first, some, biased;  // some: a counted token lies in the chunk; biased: a bias
    const int r = blockIdx.y, tid = threadIdx.x;
    if (a.follow && r >= a.step.step[kStepRows]) return;
    const size_t row = (size_t)r * a.vocab;
    // frequent tokens have low numbers: the rows' first chunks go to different XCDs (22.6 -> 20.1 us at the time)
    const int chunk = (int)((blockIdx.x + blockIdx.y) % gridDim.x);
    // elements are numbered from the 16-byte boundary at or before the row's first, so that fours are aligned
    const int lead = (int)(((uintptr_t)(a.x + row) >> 2) & 3), c0 = chunk * CH;
    const float *x = a.x + row - lead;
    float *dst = a.dst ? a.dst + row - lead : nullptr;
    const int end = a.vocab + lead;
    // Only the first and the last chunk have fours that are not whole.
    const bool whole = c0 >= lead && c0 + CH <= end, aligned = whole && ((uintptr_t)dst & 15) == 0;
    const int mask = a.p.masks ? a.p.mask_ids[r] : -1;
    const bool masked = mask >= 0 && mask < a.p.n_masks;
    v4f v[V];
    if (whole && !masked)
#pragma unroll
        for (int k = 0; k < V; k++) v[k] = *(const v4f *)(x + c0 + 4 * (tid + k * T));
    // (the mask's words are asked for before the rule is: both are waited for at once)
    static_assert(CH / 32 + 2 <= T, "a word of the mask to a thread");
    unsigned word = 0;
    if (masked) {
        const int words = (a.vocab + 31) / 32, w = (c0 ? c0 - 32 : 0) / 32 + tid;
        if (tid < CH / 32 + 2 && w < words) word = ((const unsigned *)a.p.masks)[(size_t)mask * words + w];
    }
    const int seq = a.batch ? a.step.of()[r] : r;
    sllm_logits_rule rule{1.0f, 0.0f, 0.0f, 0, 0, 0, 0, 0};
    if (seq < a.p.n_rules) rule = a.p.rules[seq];
    // what lies in its array of a range, which may name any integers
    auto range = [](int at, int n, int all, int &from) {
        from = at < 0 ? 0 : at;
        const int64_t to = (int64_t)at + n < all ? (int64_t)at + n : all;
        return from < to ? (unsigned)(to - from) : 0u;
    };
    int h0, b0;
    const unsigned nh = range(rule.history_at, rule.history, a.p.n_history, h0);
    const unsigned nb = range(rule.bias_at, rule.biases, a.p.n_biases, b0);
    const bool path = a.batch && a.p.tokens;
    const int *hist = a.p.history + h0, *bias_of = a.p.bias_tokens + b0;
    auto clear = [&] {
#pragma unroll
        for (int k = 0; k < V; k++) ((v4i *)table)[tid + k * T] = v4i{0, 0, 0, 0};
    };
    if (nh || nb || path) clear();
    if (tid == 0) {
        first = INT_MAX;
        some = biased = 0;
    }
    if (masked && tid < CH / 32 + 2) bits[tid] = word;
    lds_barrier();
    // which elements there are and are allowed, a bit for each of the thread's: what is not allowed need not be read. (It is
    // written with the rest: the tokens' loads wait for stores before them, and whole lines can go past the caches. -inf at
    // once: trees with masks 14.9 us against 13.4, 64 rows of which 30 % are allowed 18.0 against 15.3)
    unsigned ok = ~0u;
    if (!whole || masked) {
        const int w0 = c0 ? c0 - 32 : 0;  // the element of bits' first bit (the first element may lie up to three before c0)
        ok = 0;
#pragma unroll
        for (int k = 0; k < V; k++) {
            const int e = c0 + 4 * (tid + k * T);
            unsigned four = (e >= end ? 0u : 15u >> max(e + 4 - end, 0)) & 15u << max(lead - e, 0);
            if (masked) {
                const int at = max(e - lead - w0, 0);
                const unsigned two = __builtin_amdgcn_alignbit(bits[(at >> 5) + 1], bits[at >> 5], (unsigned)(e - lead) & 31);
                four &= e >= lead ? two : bits[0] << (lead - e);
            }
            ok |= four << 4 * k;
        }
        const v4f none = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int k = 0; k < V; k++) v[k] = none;
        if (whole) {
#pragma unroll
            for (int k = 0; k < V; k++)
                if (ok >> 4 * k & 15) v[k] = *(const v4f *)(x + c0 + 4 * (tid + k * T));
        } else {
#pragma unroll
            for (int k = 0; k < V; k++)
#pragma unroll
                for (int u = 0; u < 4; u++) v[k][u] = x[min(max(c0 + 4 * (tid + k * T) + u, lead), end - 1)];
        }
    }
    // tokens t0 .. t0 + nt - 1 are the chunk's, the first one's entry is i0
    const int t0 = max(c0 - lead, 0), nt = max(min(c0 - lead + CH, a.vocab) - t0, 0), i0 = t0 + lead - c0;
    auto mine = [&](int t) { return (unsigned)t - (unsigned)t0 < (unsigned)nt; };
    float y[4 * V];
    int by[4 * V];  // 1 + the number of the element's bias, 0 without one
    if (nb) {
        for (unsigned j = tid; j < nb; j += T) {
            const int t = bias_of[j];
            if (mine(t)) {
                atomicMax(&table[t - t0 + i0], j + 1);
                biased = 1;
            }
        }
        lds_barrier();
        if (biased) {
#pragma unroll
            for (int k = 0; k < V; k++) {
                const v4i b = ((const v4i *)table)[tid + k * T];
#pragma unroll
                for (int u = 0; u < 4; u++) by[4 * k + u] = b[u];
            }
            clear();  // (each thread has read the entries that it clears)
            lds_barrier();
        }
    }
    if (nh || path) {
        auto add = [&](int t) {
            if (mine(t)) {
                atomicAdd(&table[t - t0 + i0], 1u);
                some = 1;
            }
        };
        // the history, four loads of a thread under way at a time
        unsigned i = tid;
        for (; i + 3 * T < nh; i += 4 * T) {
            int t[4];
#pragma unroll
            for (int u = 0; u < 4; u++) t[u] = hist[i + u * T];
#pragma unroll
            for (int u = 0; u < 4; u++) add(t[u]);
        }
        for (; i < nh; i += T) add(hist[i]);
        if (path) {
            const StepRow &me = a.step.rows()[r];
            const int r0 = a.step.seqs()[seq], base = me.end - 1 - (r - r0);
            const uint16_t *sees = (const uint16_t *)a.step.step + me.tree;
            for (int j = r0 + tid; j <= r; j += T) {
                const int at = base + j - r0;
                if (me.tree < 0 || sees[(at >> 4) - (base >> 4)] >> (at & 15) & 1) add(a.p.tokens[j]);
            }
        }
        lds_barrier();
    }
#pragma unroll
    for (int i = 0; i < 4 * V; i++) y[i] = v[i / 4][i % 4];
    if ((nh || path) && some)
#pragma unroll
        for (int k = 0; k < V; k++) {
            const v4i n = ((const v4i *)table)[tid + k * T];
            if (!__ballot(n[0] | n[1] | n[2] | n[3])) continue;
            v4f z = {y[4 * k], y[4 * k + 1], y[4 * k + 2], y[4 * k + 3]};
#pragma unroll
            for (int u = 0; u < 4; u++) {
                const float l = z[u] > 0.0f ? z[u] / rule.repeat : z[u] * rule.repeat;
                z[u] = n[u] ? l - (rule.frequency * (float)(unsigned)n[u] + rule.presence) : z[u];
            }
#pragma unroll
            for (int u = 0; u < 4; u++) y[4 * k + u] = z[u];
        }
    if (nb && biased)
#pragma unroll
        for (int i = 0; i < 4 * V; i++)
            if (by[i]) y[i] = y[i] + a.p.bias_values[b0 + by[i] - 1];
    if (!whole || masked)
#pragma unroll
        for (int i = 0; i < 4 * V; i++) y[i] = ok >> i & 1 ? y[i] : -INFINITY;
    if (dst)
#pragma unroll
        for (int k = 0; k < V; k++) {
            const int e = c0 + 4 * (tid + k * T);
            if (aligned) {
                // whole lines go past the caches (17.4 us without, 15.2; masked 14.8, 13.4)
                const v4f z = {y[4 * k], y[4 * k + 1], y[4 * k + 2], y[4 * k + 3]};
                __builtin_nontemporal_store(z, (v4f *)(dst + e));
            } else {
#pragma unroll
                for (int u = 0; u < 4; u++)
                    if (e + u >= lead && e + u < end) dst[e + u] = y[4 * k + u];
            }
        }
    if (!a.chosen) return;
    // the largest value (no NaN is above another value), then the first element that has it
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < 4 * V; i++) top = y[i] > top ? y[i] : top;
    const float own = top;
    top = wave_max(top);
    if ((tid & 63) == 0) wv[tid >> 6] = top;
    lds_barrier();
#pragma unroll
    for (int w = 0; w < T / 64; w++) top = wv[w] > top ? wv[w] : top;
    if (own == top) {
        int i = 4 * V;
#pragma unroll
        for (int k = 4 * V - 1; k >= 0; k--) i = y[k] == top ? k : i;
        atomicMin(&first, c0 + 4 * (tid + i / 4 * T) + i % 4 - lead);
    }
    lds_barrier();
    if (tid) return;
    if (a.chunks == 1) a.chosen[r] = top == -INFINITY ? -1 : first;
    else a.best[(size_t)r * a.chunks + chunk] = make_int2(__float_as_int(top), first);
}

// The chunks' candidates of a row, by one wave. (-inf is never chosen: -1 where nothing else is there.)
__global__ void __launch_bounds__(64) logits_choose_kernel(LogitsArgs a) {
    const int r = blockIdx.x;
    if (a.follow && r >= a.step.step[kStepRows]) return;
    // (a lane's chunks ascend, and their indices)
    float v = -INFINITY;
    int i = INT_MAX;
    for (int c = threadIdx.x; c < a.chunks; c += 64) {
        const int2 b = a.best[(size_t)r * a.chunks + c];
        const float x = __int_as_float(b.x);
        if (x > v) {
            v = x;
            i = b.y;
        }
    }
    const float top = wave_max(v);
    i = wave_min(v == top ? i : INT_MAX);
    if (threadIdx.x == 0) a.chosen[r] = top == -INFINITY ? -1 : i;
}

// ------------------------------------------------------- accepted paths ----

// One workgroup per sequence. A row follows its parent where it holds the token chosen behind it (of several such rows the
// first); the path is the rows whose ancestors all follow: each row looks whether a bit of those it sees is missing among the
// bits of the rows that follow, so nothing walks from row to row (64 rows of a chain: 64 reads of LDS one after the other).
// Bound by latency: two dependent loads behind the step's description; 2.7 us, 200 sequences of up to 64 rows 4.6.
constexpr int kAcceptThreads = 256;
constexpr int kMostSeqs = 1 << 24;  // a launch has fewer than 2^32 threads: this kernel and the next have 256 to a sequence
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
    int n_kv, page_rows, pieces;  // pieces: 16-byte pieces of a row of a head
    size_t layer_bytes;
};

// One workgroup per (sequence, K or V of a layer). A thread has one 16-byte column of a head and moves the path's rows
// there in order, four loads before their stores: a row goes to a place at or before its own, so that nothing is overwritten
// before it has been read. Bound by latency (path, places, rows: 3.6 us for one sequence of 30 layers) and the rows' bytes
// (24 sequences of 32 layers, 31 MB read and written: 7.6 us).
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
        if (((uintptr_t)logits | (uintptr_t)dst | (uintptr_t)chosen | (uintptr_t)p->rules | (uintptr_t)p->history |
             (uintptr_t)p->bias_tokens | (uintptr_t)p->bias_values | (uintptr_t)p->masks | (uintptr_t)p->mask_ids | (uintptr_t)p->tokens) & 3)
            return set_error(SLLM_ERR_ARG, "misaligned pointer");
        if (rows > 65535) return set_error(SLLM_ERR_SHAPE, "at most 65535 rows");
        if (vocab > (1 << 28)) return set_error(SLLM_ERR_SHAPE, "vocab must be at most 2^28");
        hipStream_t s = (hipStream_t)stream;
        LogitsArgs a{};
        std::unique_lock<std::mutex> lb;  // (until the launches: the step that they are told of is then the batch's)
        if (batch) {
            PageBatch &b = const_cast<sllm_page_batch *>(batch)->b;
            lb = std::unique_lock<std::mutex>(b.mu);
            {
                std::lock_guard<std::mutex> lk(b.c->mu);
                const sllm_status st = step_stands(b);
                if (st != SLLM_OK) return st;
            }
            const sllm_status st = on_device(b.c->device);
            if (st != SLLM_OK) return st;
            const bool capture = stream_capturing(s);
            if (rows != (capture ? b.max_rows : b.rows))
                return set_error(SLLM_ERR_SHAPE, capture ? "a captured call's rows are the batch's max_rows" : "rows differ from those of the batch's step");
            a.batch = true;
            a.follow = capture;
            a.step = step_ref(b, capture);
        }
        if (!rows) return SLLM_OK;
        sllm_status st = library_init();
        if (st != SLLM_OK) return st;
        a.x = logits;
        a.dst = dst;
        a.chosen = chosen;
        a.vocab = vocab;
        a.p = *p;
        if (!p->n_masks) a.p.masks = nullptr;
        // Chunks of 1024 while all of them run at once (eight workgroups to a CU), else of 4096, whose launch and tokens cost
        // less. us with chunks of 1024 and of 4096, values kept, histories of 64: 1 x 49152 6.8, 8.5; 7 x 32003 6.0, 8.2; 8 x 128256 6.8, 7.2;
        // 16 x 128256 8.2, 7.7; 24 x 128256 9.7, 8.4; 64 x 128256 16.9, 14.3 (4000: 25.4, 16.5). Chunks that are not whole read and
        // write one element at a time, which costs more of the larger ones: short vocabularies, and those whose rows do
        // not all begin at 16 bytes, stay faster with 1024 beyond that (80 x 32003 9.5, 11.8; 1000 x 4097, no tokens, 12.5, 21.3).
        const int64_t small = 4 * kRuleThreads, n_small = ((int64_t)vocab + 3 + small - 1) / small;
        const bool four = n_small * rows > 2048;
        a.chunks = (int)(four ? (n_small + 3) / 4 : n_small);
        if (chosen && a.chunks > 1) {
            void *ws = nullptr;
            size_t cap = 0;
            st = stream_workspace(s, (size_t)rows * a.chunks * sizeof(int2), &ws, &cap);
            if (st != SLLM_OK) return st;
            a.best = (int2 *)ws;
        }
        const dim3 grid((unsigned)a.chunks, (unsigned)rows);
        if (four) hipLaunchKernelGGL(logits_rules_kernel<4>, grid, dim3(kRuleThreads), 0, s, a);
        else hipLaunchKernelGGL(logits_rules_kernel<1>, grid, dim3(kRuleThreads), 0, s, a);
        SLLM_HIP(hipGetLastError());
        if (batch) const_cast<sllm_page_batch *>(batch)->b.captured |= a.follow;
        if (!chosen || a.chunks == 1) return SLLM_OK;
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
        const int n = capture ? b.max_seqs : (int)b.seqs.size();
        if (!n) return SLLM_OK;
        if (n >= kMostSeqs) return set_error(SLLM_ERR_SHAPE, "accepted paths of 2^24 sequences or more");
        hipLaunchKernelGGL(page_accept_kernel, dim3((unsigned)n), dim3(kAcceptThreads), 0, s,
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
        const int n = capture ? b.max_seqs : (int)b.seqs.size();
        if (!n) return SLLM_OK;
        if (n >= kMostSeqs) return set_error(SLLM_ERR_SHAPE, "kept rows of 2^24 sequences or more");
        KeepArgs a{};
        a.step = step_ref(b, capture);
        a.kept = kept;
        a.pool_k = c.k;
        a.pool_v = c.v;
        a.n_kv = c.n_kv;
        a.page_rows = c.page_rows;
        a.pieces = c.d_k * c.elem() / 16;
        a.layer_bytes = (size_t)c.n_pages * c.n_kv * c.page_rows * c.d_k * c.elem();
        hipLaunchKernelGGL(page_keep_kernel, dim3((unsigned)n, 2u * (unsigned)c.n_layers), dim3(kKeepThreads), 0, s, a);
        SLLM_HIP(hipGetLastError());
        b.captured |= capture;
        return SLLM_OK;
    });
}

}  // extern "C"
