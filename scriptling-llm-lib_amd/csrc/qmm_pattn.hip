// The attention section (bias, QK norm, RoPE, append, causal GQA attention) of a batch of sequences
// over a page cache.
//
// page_prep_kernel: the step's rows: q heads rotated to the batch's memory, k and v into their pages.
// page_attn_kernel: the attention over pieces of segments (qmm_pages.hip: a segment is a run of positions with the
//   rows that see it: one sequence's own rows, or those of all sequences that share its pages), whose K and V
//   are read once for all rows of a block.
// page_combine_kernel: the pieces' softmax states of every row and head, merged.
#include <hip/hip_runtime.h>

#include <type_traits>
#include <utility>

#include "qmm_device.hpp"
#include "qmm_pages.hpp"

namespace sllm {

namespace {

constexpr int kMaxDk = 256;
typedef float v2f __attribute__((ext_vector_type(2)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef _Float16 v4h __attribute__((ext_vector_type(4)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef unsigned v2u __attribute__((ext_vector_type(2)));
typedef unsigned v4u __attribute__((ext_vector_type(4)));
typedef void __attribute__((address_space(3))) *LdsPtr;
typedef const void __attribute__((address_space(1))) *GlobalPtr;

__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

__device__ __forceinline__ void put4(float *dst, v4f x) { *(v4f *)dst = x; }
__device__ __forceinline__ void put4(_Float16 *dst, v4f x) {
    *(v4h *)dst = v4h{(_Float16)x[0], (_Float16)x[1], (_Float16)x[2], (_Float16)x[3]};
}

// The step's rows. (By value where the launch is the step's own: a read of memory less before everything else.)
__device__ __forceinline__ const StepRow *step_rows(const PageAttnArgs &a) {
    return (const StepRow *)(a.step + (a.rows_at >= 0 ? a.rows_at : a.step[kStepRowsAt]));
}

// A rotated q head (row pair of a.qrot: d_k floats) as the attention takes it. f32: as it is. f16 caches: two f16
// values for each element, d_k leading parts, then d_k rests (together within 2^-23 of it or 2^-35 of the head's largest
// element, whichever is more), of the head times a power of two that puts its largest element between 2^10 and 2^11, so
// that no float32 leaves f16's range; a.qscale undoes it.
// LP lanes hold the head, zeros beyond d_k.
template <class T, int LP>
__device__ __forceinline__ void put_q(const PageAttnArgs &a, size_t pair, int d, int dk, v4f x) {
    if constexpr (sizeof(T) == 4) {
        *(v4f *)(a.qrot + pair * dk + d) = x;
    } else {
        float big = fmaxf(fmaxf(__builtin_fabsf(x[0]), __builtin_fabsf(x[1])), fmaxf(__builtin_fabsf(x[2]), __builtin_fabsf(x[3])));
#pragma unroll
        for (int o = LP / 2; o > 0; o >>= 1) big = fmaxf(big, __shfl_xor(big, o, LP));
        int e = (int)((__builtin_bit_cast(unsigned, big) >> 23) & 255u) - 127 - 10;
        e = e < -110 ? -110 : e;
        x = x * __builtin_bit_cast(float, (unsigned)(127 - e) << 23);
        const v4h hi = {(_Float16)x[0], (_Float16)x[1], (_Float16)x[2], (_Float16)x[3]};
        _Float16 *to = (_Float16 *)(a.qrot + pair * dk);
        if (d < dk) {
            *(v4h *)(to + d) = hi;
            put4(to + dk + d, v4f{x[0] - (float)hi[0], x[1] - (float)hi[1], x[2] - (float)hi[2], x[3] - (float)hi[3]});
        }
        if (d == 0) a.qscale[pair] = __builtin_bit_cast(float, (unsigned)(127 + e) << 23);
    }
}

// Bias (model_f32.go:398-420), per-head RMSNorm (:424-435), RoPE (applyRopeInPlaceF32,
// float32_ops.go:174-188) of every q and k head of a row, and the row's k and v into its page
// (the append, model_f32.go:445-448), rounded to the cache's type, once.
// A workgroup takes heads of one row, LP lanes of four dimensions to a head; the rotation (the same for
// every head: float32 angle, sine and cosine in 64 bits, as the reference) is formed once in LDS, the first
// heads' elements loaded before it. Bound by latency: few rows have a workgroup for every 256 / LP heads.
// (16 rows of 32 + 8 heads of 128, us: one workgroup of eight waves per row, a wave per head 8.2; this 4.0.)
constexpr int kPrepThreads = 256;
template <class T, int LP>
__global__ void __launch_bounds__(kPrepThreads) page_prep_kernel(PageAttnArgs a) {
    __shared__ float rc[kMaxDk / 2], rs[kMaxDk / 2];
    constexpr int HG = kPrepThreads / LP;
    const int r = blockIdx.x, sub = threadIdx.x % LP;
    if (a.rows_at < 0 && r >= a.step[kStepRows]) return;
    const StepRow &row = step_rows(a)[r];
    const int dk = a.d_k, d = 4 * sub, page_rows = 1 << a.shift;
    auto at_of = [&](int t) {
        return t < a.n_heads ? ((size_t)r * a.n_heads + t) * dk + d : ((size_t)r * a.n_kv + t - a.n_heads) * dk + d;
    };
    auto load = [&](int t) {
        return t < a.n_heads + a.n_kv && d < dk ? *(const v4f *)((t < a.n_heads ? a.q : a.k) + at_of(t)) : v4f{0.0f, 0.0f, 0.0f, 0.0f};
    };
    int t = blockIdx.y * HG + threadIdx.x / LP;
    v4f x = load(t);
    if ((int)threadIdx.x < a.half_dim) {
        const float ang = a.freqs[threadIdx.x] * (float)row.pos;
        double sd, cd;
        sincos((double)ang, &sd, &cd);
        rc[threadIdx.x] = (float)cd;
        rs[threadIdx.x] = (float)sd;
    }
    __syncthreads();
    for (; t < a.n_heads + a.n_kv; t += gridDim.y * HG, x = load(t)) {
        const bool isq = t < a.n_heads;
        const int h = isq ? t : t - a.n_heads;
        const size_t off = at_of(t);
        const float *bias = isq ? a.q_bias : a.k_bias, *nw = isq ? a.q_norm : a.k_norm;
        const int blen = isq ? a.qb_len : a.kb_len, j0 = h * dk + d;
        if (bias && d < dk)
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (j0 + i < blen) x[i] = x[i] + bias[j0 + i];
        if (nw) {
            float ss = ((x[0] * x[0] + x[1] * x[1]) + x[2] * x[2]) + x[3] * x[3];
#pragma unroll
            for (int o = LP / 2; o > 0; o >>= 1) ss = ss + __shfl_xor(ss, o, LP);
            const float inv = 1.0f / (float)sqrt((double)ss / (double)dk + (double)a.eps);
            if (d < dk)
#pragma unroll
                for (int i = 0; i < 4; i++) x[i] = (x[i] * inv) * nw[d + i];
        }
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const int f = 2 * sub + i;
            if (f < a.half_dim) {
                const float c = rc[f], s = rs[f], x0 = x[2 * i], x1 = x[2 * i + 1];
                x[2 * i] = x0 * c - x1 * s;
                x[2 * i + 1] = x0 * s + x1 * c;
            }
        }
        if (sizeof(T) == 4 && d >= dk) continue;
        if (isq) {
            put_q<T, LP>(a, (size_t)r * a.n_heads + h, d, dk, x);
            continue;
        }
        if (d >= dk) continue;
        const size_t at = (((size_t)row.page * a.n_kv + h) * page_rows + row.slot) * dk + d;
        v4f w = *(const v4f *)(a.v + off);
        if (a.v_bias)
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (j0 + i < a.vb_len) w[i] = w[i] + a.v_bias[j0 + i];
        put4((T *)a.pool_k + at, x);
        put4((T *)a.pool_v + at, w);
    }
}

// ------------------------------------------------------------ attention ----
//
// A workgroup of four waves takes one piece (positions p0 .. p1 of a segment) for one kv head and a
// block of rows; a row here is a (query row, q head of the kv head) pair. Both products are taken
// transposed on the 16-row matrix instructions, so that a lane keeps one row (lane % 16)
// throughout, and both read K and V straight from memory into the operands' registers, since the order
// of an instruction's k is free and so is that of the output's dimensions:
//   S^T = K Q^T: lane l holds K[position l % 16], dimensions of its quarter q = l / 16;
//   the result leaves positions 4 q + i in lane quarter q: as B operand of O^T = V^T P^T it
//     stays where it is, and the quarter reads V rows 4 q + i, every lane a run of dimensions.
// f16: 32 positions a step; K and V are exact operands, q and the weights go in as two f16 each (the row's q scaled by a
//   power of two, so no float32 leaves f16's range: put_q).
// f32: 16 positions a step, fp32 matrix instructions.
// Softmax weights are 2^(s - m); m follows the largest score when one exceeds it by more than kTop: while none does,
// neither the row's lanes have to agree on a maximum nor the sums to be scaled again. Sums are held in fp32.
// A weight's f16 parts are its nearest f16 and the nearest to what is left: together within 2^-23 of the weight, or, as f16
// ends, within 2^-25. So that small weights of f16 caches keep their bits too (many keys behind one of a large score), the
// largest one lies between 2^13 and 2^15, near f16's other end: m is 13 below the largest score when it follows. Then
// 2^-25 is 2^-38 of the largest weight so far: of a key 14 nats below another 2^-18 at worst (with the largest at 1 and
// the parts cut off, 7 % were lost). Two binades before m follows again cost no time against eight (64 sequences on a
// prefix of 4000 37.6 us either way, 5 prompts of 211 rows 58.4 and 58.0).
// A result that is not finite (a non-finite K or V element, also one that only other rows of the block
// see, where the matrix instruction forms 0 * inf) is computed again, row by row, as the formula says.
constexpr int kWaves = 4;
constexpr int kMergeThreads = 320000;  // of a launch that merges states, above which a pair has one group of lanes
// log2 of the largest weight when m follows it, and from which on it follows
template <class T>
constexpr float kLead = sizeof(T) == 2 ? 13.0f : 0.0f;
template <class T>
constexpr float kTop = sizeof(T) == 2 ? 15.0f : 8.0f;

template <int... G, class F>
__device__ __forceinline__ void each(std::integer_sequence<int, G...>, F f) {
    (f(std::integral_constant<int, G>{}), ...);
}
template <class T>
struct Kind;
template <>
struct Kind<float> {
    static constexpr int kTile = 16;
};
template <>
struct Kind<_Float16> {
    static constexpr int kTile = 32;
};

// What is the same for a wave is read through the scalar cache (the step was written before the kernel began):
// a vector load of a page number would have to wait for the K and V loads before it.
typedef const int __attribute__((address_space(4))) *ScalarInts;

struct Piece {
    StepItem it;
    int g, rep, dk;
    int tid;  // threadIdx.x, as a value that is formed for every piece: what follows from it is not kept beside them all
    ScalarInts table, first;  // the sequence's page ids; the first ones of the piece
    const int *step;
    const StepRow *rows;
    float per_rep;  // 1 / rep
    // row v of the block: its number among the query rows (v < 128: exact), and its query row
    __device__ __forceinline__ int nth(int v) const { return (int)(((float)v + 0.5f) * per_rep); }
    __device__ __forceinline__ int row_of(int v) const {
        const int t = nth(v);
        return it.flags & kItemRun ? it.tok + t : step[it.tok + t];
    }
};

// Where the rows' results go: the output (direct), or the piece's states. Offsets of a row fit 32 bits
// (sllm_page_batch_create bounds them).
struct Results {
    float *to, *ml;
    bool direct;
    __device__ __forceinline__ Results(const PageAttnArgs &a, const Piece &p) {
        const size_t first = (size_t)p.g * a.slots + p.it.slot;
        direct = p.it.flags & kItemDirect;
        to = direct ? a.out + p.g * p.rep * p.dk : a.part + first * p.dk;
        ml = a.ml + first * 2;
    }
    __device__ __forceinline__ int at(const PageAttnArgs &a, const Piece &p, int v) const {
        if (!direct) return v * p.dk;
        const int t = p.nth(v);
        return ((p.it.flags & kItemRun ? p.it.tok + t : p.step[p.it.tok + t]) * a.n_heads + v - t * p.rep) * p.dk;
    }
    __device__ __forceinline__ void state(int v, float m, float l) const {
        ml[2 * v] = m;
        ml[2 * v + 1] = l;
    }
};

// One row after the other, one position after the other, by one wave: rows v0, v0 + dv, ... of the piece.
template <class T>
__device__ __forceinline__ void plain_rows(const PageAttnArgs &a, const Piece &p, int v0, int v1, int dv) {
    int lane = p.tid & 63;
    asm volatile("" : "+v"(lane));
    const int dk = p.dk, d = 4 * lane, page_rows = 1 << a.shift;
    for (int v = v0; v < v1; v += dv) {
        const int row = p.row_of(v);
        const int end = p.it.flags & (kItemCausal | kItemTree) ? min(p.it.p1, p.rows[row].end) : p.it.p1;
        const size_t pair = (size_t)row * a.n_heads + p.g * p.rep + v - p.nth(v) * p.rep;
        v4f q = {0.0f, 0.0f, 0.0f, 0.0f}, o = q;
        if (d < dk) {
            if constexpr (sizeof(T) == 4) {
                q = *(const v4f *)(a.qrot + pair * dk + d);
            } else {
                const _Float16 *qr = (const _Float16 *)(a.qrot + pair * dk) + d;
#pragma unroll
                for (int i = 0; i < 4; i++) q[i] = ((float)qr[i] + (float)qr[dk + i]) * a.qscale[pair];
            }
        }
        float m = -INFINITY, l = 0.0f;
        const uint16_t *sees = (const uint16_t *)p.step + p.rows[row].tree;
        for (int x = p.it.p0; x < end; x++) {
            if (p.it.flags & kItemTree && x >= p.it.lim0 && !(sees[(x >> 4) - (p.it.lim0 >> 4)] >> (x & 15) & 1)) continue;
            const size_t at = (((size_t)p.table[x >> a.shift] * a.n_kv + p.g) * page_rows + (x & (page_rows - 1))) * dk + d;
            v4f k = {0.0f, 0.0f, 0.0f, 0.0f}, w = k;
            if (d < dk)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    k[i] = (float)((const T *)a.pool_k)[at + i];
                    w[i] = (float)((const T *)a.pool_v)[at + i];
                }
            const float s = wave_sum(((q[0] * k[0] + q[1] * k[1]) + q[2] * k[2]) + q[3] * k[3]) * a.scale_log2;
            const float mn = fmaxf(m, s), ref = mn == -INFINITY ? 0.0f : mn;
            const float alpha = exp2_(m - ref), e = exp2_(s - ref);
            l = l * alpha + e;
            // the product of a weight of 0 that another position has made so is that of the formula's small weight
            o = o * alpha + w * e;
            m = mn;
        }
        const Results res(a, p);
        if (d < dk) *(v4f *)(res.to + res.at(a, p, v) + d) = res.direct ? o * (1.0f / l) : o;
        if (!res.direct && lane == 0) res.state(v, m, l);
    }
}

// A lane of V reads VW dimensions at once: lane l % 16 = col the col-th run of 16 (from memory: neighbours read
// neighbours), or, from LDS, run run_of(col). The output's element (tile t, accumulator i) of a lane in quarter q is
// row 4 q + i of its tile, so its dimension is dim_of; with run_of the quarters' runs are neighbours, and a store
// instruction fills a quarter of a row's line, not a run here and there.
__device__ __forceinline__ constexpr int run_of(int col) { return 4 * (col & 3) + (col >> 2); }
template <int VW>
__device__ __forceinline__ constexpr int dim_of(int t, int run) {
    return 16 * VW * (t / VW) + VW * run + t % VW;
}

// The matrix operands' shapes. Tile: TP positions, H halves of 16; K: KS pieces of 16 bytes per lane, each KD
// dimensions over the quarters; V: VE rows per lane, VB runs of VW dimensions of each.
template <class T, int NB, bool FULL, int VM = 8>
struct Shape {
    static constexpr bool F16 = sizeof(T) == 2;
    static constexpr int TP = Kind<T>::kTile, H = TP / 16, NT = 4 * NB, DKP = 64 * NB;
    static constexpr int VW = F16 && FULL && NB % 2 == 0 ? VM : 4;
    static constexpr int KS = F16 ? 2 * NB : 4 * NB, KE = F16 ? 8 : 4, KD = 4 * KE;
    static constexpr int VB = DKP / (16 * VW), VE = 4 * H;
    typedef T VT __attribute__((ext_vector_type(VW)));
};

// 16 MT rows of a wave: their q, running maximum, sum and values.
template <class T, int NB, bool FULL, int MT, int VM = 8>
struct Rows : Shape<T, NB, FULL, VM> {
    typedef Shape<T, NB, FULL, VM> S;
    using S::F16, S::TP, S::H, S::NT, S::VW, S::KS, S::KE, S::KD;
    v4f qf[F16 ? 1 : MT][F16 ? 1 : KS];
    v8h qh[F16 ? MT : 1][F16 ? KS : 1], ql[F16 ? MT : 1][F16 ? KS : 1];
    float sc[MT], m[MT], l[MT];
    int lim[MT];  // positions from here on are not seen; of a tree: what the row sees of it (StepRow)
    v4f o[MT][NT], s[MT][H];

    // rows v0 .. of the block (those past its end repeat the last)
    __device__ __forceinline__ void init(const PageAttnArgs &a, const Piece &p, int v0) {
        const int lane = p.tid & 63, col = lane & 15, qd = lane >> 4;
        const int dk = FULL ? S::DKP : p.dk, nv = p.it.ntok * p.rep;
#pragma unroll
        for (int mt = 0; mt < MT; mt++) {
            const int v = min(v0 + mt * 16 + col, nv - 1);
            const int row = p.row_of(v);
            lim[mt] = p.it.flags & kItemTree ? p.rows[row].tree : p.it.flags & kItemCausal ? min(p.it.p1, p.rows[row].end) : p.it.p1;
            const size_t pair = (size_t)row * a.n_heads + p.g * p.rep + v - p.nth(v) * p.rep;
            sc[mt] = a.scale_log2;
            if constexpr (F16) {
                const _Float16 *qr = (const _Float16 *)(a.qrot + pair * dk);
                sc[mt] = a.scale_log2 * a.qscale[pair];
#pragma unroll
                for (int j = 0; j < KS; j++) {
                    const int d = KD * j + KE * qd;
                    const bool in = FULL || d < dk;
                    const v8h zero = {};
                    qh[mt][j] = in ? *(const v8h *)(qr + d) : zero;
                    ql[mt][j] = in ? *(const v8h *)(qr + dk + d) : zero;
                }
            } else {
                const float *qr = a.qrot + pair * dk;
#pragma unroll
                for (int j = 0; j < KS; j++) {
                    const int d = KD * j + KE * qd;
                    qf[mt][j] = FULL || d < dk ? *(const v4f *)(qr + d) : v4f{0.0f, 0.0f, 0.0f, 0.0f};
                }
            }
            m[mt] = -INFINITY;
            l[mt] = 0.0f;
#pragma unroll
            for (int t = 0; t < NT; t++) o[mt][t] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
        }
    }

    __device__ __forceinline__ void no_scores() {
#pragma unroll
        for (int mt = 0; mt < MT; mt++)
#pragma unroll
            for (int h = 0; h < H; h++) s[mt][h] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    }
    // k(h, j): piece j of the lane's K row in half h; pieces J0 .. J1
    template <int J0, int J1, class K>
    __device__ __forceinline__ void scores(K k) {
#pragma unroll
        for (int j = J0; j < J1; j++) {
            v4u kw[H];
#pragma unroll
            for (int h = 0; h < H; h++) kw[h] = k(h, j);
            // (an instruction's result is the next one's addend only after those of the other halves and rows)
            if constexpr (F16) {
#pragma unroll
                for (int p = 0; p < 2; p++)
#pragma unroll
                    for (int h = 0; h < H; h++)
#pragma unroll
                        for (int mt = 0; mt < MT; mt++)
                            s[mt][h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, kw[h]), p ? ql[mt][j] : qh[mt][j],
                                                                              s[mt][h], 0, 0, 0);
            } else {
#pragma unroll
                for (int c = 0; c < 4; c++)
#pragma unroll
                    for (int h = 0; h < H; h++)
#pragma unroll
                        for (int mt = 0; mt < MT; mt++)
                            s[mt][h] = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(v4f, kw[h])[c], qf[mt][j][c], s[mt][h], 0, 0, 0);
            }
        }
    }

    // scores to weights, for the tile at position tp (masked: some row does not see all of it)
    __device__ __forceinline__ void weights(const Piece &p, int tp, bool masked) {
        if (masked) {
            int lane = __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u));
            asm volatile("" : "+v"(lane));
            const int qd = lane >> 4;
            if (p.it.flags & kItemTree) {
                // (tiles begin at multiples of 16 positions, as the rows' elements; the one behind the tree's last is 0. Asked
                // for before the scores, the bits came no sooner: 54.2 us against 53.9 behind 16000 rows)
                const int half = (tp >> 4) - (p.it.lim0 >> 4);
#pragma unroll
                for (int mt = 0; mt < MT; mt++)
#pragma unroll
                    for (int h = 0; h < H; h++) {
                        if (half + h < 0) continue;
                        const unsigned bits = (unsigned)((const uint16_t *)p.step)[lim[mt] + half + h] >> 4 * qd;
#pragma unroll
                        for (int i = 0; i < 4; i++)
                            if (!(bits >> i & 1)) s[mt][h][i] = -INFINITY;
                    }
            } else
#pragma unroll
            for (int mt = 0; mt < MT; mt++) {
                const int left = lim[mt] - tp - 4 * qd;
#pragma unroll
                for (int h = 0; h < H; h++)
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        if (16 * h + i >= left) s[mt][h][i] = -INFINITY;
            }
        }
#pragma unroll
        for (int mt = 0; mt < MT; mt++) {
            float mx = -INFINITY;
#pragma unroll
            for (int h = 0; h < H; h++)
#pragma unroll
                for (int i = 0; i < 4; i++) mx = fmaxf(mx, s[mt][h][i]);
            mx = mx * sc[mt];
            if (__ballot(mx > m[mt] + kTop<T>)) {  // from -inf on: any score
                float mn = fmaxf(mx, __shfl_xor(mx, 16, 64));
                mn = fmaxf(m[mt], fmaxf(mn, __shfl_xor(mn, 32, 64)) - kLead<T>);
                const float alpha = mn == m[mt] ? 1.0f : exp2_(m[mt] - mn);
                m[mt] = mn;
                l[mt] = l[mt] * alpha;
#pragma unroll
                for (int u = 0; u < NT; u++) o[mt][u] = o[mt][u] * alpha;
            }
            const float ref = m[mt] == -INFINITY ? 0.0f : m[mt];
            float sum = 0.0f;
#pragma unroll
            for (int h = 0; h < H; h++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    s[mt][h][i] = exp2_(__builtin_fmaf(s[mt][h][i], sc[mt], -ref));
                    sum = sum + s[mt][h][i];
                }
            l[mt] = l[mt] + sum;
        }
    }

    // v(u, x): run u of the lane's V rows
    typedef unsigned VU __attribute__((ext_vector_type(S::VW * sizeof(T) / 4)));
    template <class V>
    __device__ __forceinline__ void values(V v) {
        if constexpr (F16) {
            v8h ph[MT], pl[MT];
#pragma unroll
            for (int mt = 0; mt < MT; mt++) {
                v4u hi, lo;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float x = s[mt][i / 2][2 * (i & 1)], y = s[mt][i / 2][2 * (i & 1) + 1];
                    const v2h hp = __builtin_convertvector((v2f{x, y}), v2h);
                    const v2f left = {__builtin_fmaf((float)hp[0], -1.0f, x), __builtin_fmaf((float)hp[1], -1.0f, y)};
                    hi[i] = __builtin_bit_cast(unsigned, hp);
                    lo[i] = __builtin_bit_cast(unsigned, __builtin_convertvector(left, v2h));
                }
                ph[mt] = __builtin_bit_cast(v8h, hi);
                pl[mt] = __builtin_bit_cast(v8h, lo);
            }
#pragma unroll
            for (int u = 0; u < S::VB; u++) {
                VU x[8];
                v(u, x);
#pragma unroll
                for (int g = 0; g < VW; g += 4) {
                    // the eight rows' elements g .. g + 3 of the lane's run
                    v8h va[4];
#pragma unroll
                    for (int c = 0; c < 4; c++) {
                        v4u w;
#pragma unroll
                        for (int i = 0; i < 4; i++)
                            w[i] = __builtin_amdgcn_perm(x[2 * i + 1][(g + c) / 2], x[2 * i][(g + c) / 2], c & 1 ? 0x07060302u : 0x05040100u);
                        va[c] = __builtin_bit_cast(v8h, w);
                    }
#pragma unroll
                    for (int p = 0; p < 2; p++)
#pragma unroll
                        for (int c = 0; c < 4; c++)
#pragma unroll
                            for (int mt = 0; mt < MT; mt++) {
                                v4f &d = o[mt][VW * u + g + c];
                                d = __builtin_amdgcn_mfma_f32_16x16x32_f16(va[c], p ? pl[mt] : ph[mt], d, 0, 0, 0);
                            }
                }
            }
        } else {
#pragma unroll
            for (int u = 0; u < S::VB; u++) {
                VU x[4];
                v(u, x);
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int c = 0; c < VW; c++)
#pragma unroll
                        for (int mt = 0; mt < MT; mt++) {
                            v4f &d = o[mt][VW * u + c];
                            d = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(v4f, x[i])[c], s[mt][0][i], d, 0, 0, 0);
                        }
            }
        }
    }

    // four dimensions from dim_of(t, the run) on of row mt's values, t a multiple of four
    __device__ __forceinline__ v4f four(int mt, int t, int i) const {
        return v4f{o[mt][t][i], o[mt][t + 1][i], o[mt][t + 2][i], o[mt][t + 3][i]};
    }
    __device__ __forceinline__ void sum_up() {
#pragma unroll
        for (int mt = 0; mt < MT; mt++) {
            l[mt] = l[mt] + __shfl_xor(l[mt], 16, 64);
            l[mt] = l[mt] + __shfl_xor(l[mt], 32, 64);
        }
    }
};

__device__ __forceinline__ bool finite4(v4f x) {
    return __builtin_isfinite(x[0]) && __builtin_isfinite(x[1]) && __builtin_isfinite(x[2]) && __builtin_isfinite(x[3]);
}

// Bytes of a tile's K and V in LDS, and how many tiles its ring holds.
template <class T, int NB>
constexpr int tile_bytes() {
    return 2 * Kind<T>::kTile * 64 * NB * (int)sizeof(T);
}
template <int NB>
constexpr int kMergeBytes = kWaves * 16 * (64 * NB + 4) * 4;  // the waves' values of 16 rows
template <int NB>
constexpr int ring_stages() {
    return NB <= 2 ? 4 : 2;
}

// A workgroup's barrier for what it shares in LDS (__syncthreads waits for its stores to memory too).
__device__ __forceinline__ void lds_barrier() {
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// The states of 16 MT rows, each held by all waves, which had different tiles: merged in wave order through LDS.
template <class T, int NB, bool FULL, int MT>
__device__ __forceinline__ void merge_waves(const PageAttnArgs &a, const Piece &p, const Rows<T, NB, FULL, MT> &r, int wave,
                                            char *lds, float *lm) {
    typedef Shape<T, NB, FULL> S;
    constexpr int NT = S::NT, DKP = S::DKP, VW = S::VW, RS = DKP + 4;
    constexpr int D4 = DKP / 4, R = 64 * kWaves / D4;  // threads per row, rows at a time
    const int lane = p.tid & 63, col = lane & 15, qd = lane >> 4;
    const int dk = FULL ? DKP : p.dk, nv = p.it.ntok * p.rep;
    float *wo = (float *)lds;
    int *flag = (int *)(lm + kWaves * 16 * 2);
    const Results res(a, p);
    const int d = (int)p.tid % D4 * 4, u0 = p.tid / D4;
    if (p.tid == 0) *flag = 0;
#pragma unroll
    for (int mt = 0; mt < MT; mt++) {
        lds_barrier();
#pragma unroll
        for (int t = 0; t < NT; t += 4)
#pragma unroll
            for (int i = 0; i < 4; i++) *(v4f *)(wo + (wave * 16 + col) * RS + dim_of<VW>(t, 4 * qd + i)) = r.four(mt, t, i);
        if (qd == 0) {
            // (as a pair, the state would become an array in LDS, whose place per thread the kernel's start would read from
            // the dispatch packet in host memory: 13 us)
            lm[(wave * 16 + col) * 2] = r.m[mt];
            lm[(wave * 16 + col) * 2 + 1] = r.l[mt];
        }
        lds_barrier();
        for (int u = u0; u < 16; u += R) {
            const int v = mt * 16 + u;
            if (v >= nv || (!FULL && d >= dk)) break;
            v2f ml[kWaves];
            v4f x[kWaves];
#pragma unroll
            for (int w = 0; w < kWaves; w++) {
                ml[w] = *(const v2f *)(lm + 2 * (w * 16 + u));
                x[w] = *(const v4f *)(wo + (w * 16 + u) * RS + d);
            }
            float M = ml[0][0];
#pragma unroll
            for (int w = 1; w < kWaves; w++) M = fmaxf(M, ml[w][0]);
            const float ref = M == -INFINITY ? 0.0f : M;  // (then every weight is 2^-inf = 0)
            float L = 0.0f;
            v4f O = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int w = 0; w < kWaves; w++) {
                const float f = exp2_(ml[w][0] - ref);
                L = L + ml[w][1] * f;
                O = O + x[w] * f;
            }
            if (res.direct) O = O * (1.0f / L);
            else if (d == 0) res.state(v, M, L);
            *(v4f *)(res.to + res.at(a, p, v) + d) = O;
            if (!(__builtin_isfinite(L) && finite4(O))) *flag = 1;
        }
    }
    lds_barrier();
    if (*flag) plain_rows<T>(a, p, wave, nv, kWaves);
    lds_barrier();  // the memory is free for the next piece
}

// Up to 16 MT rows: the waves take every fourth tile each, straight into registers, and merge their states.
template <class T, int NB, bool FULL, int MT>
__device__ __forceinline__ void run_split(const PageAttnArgs &a, const Piece &p, char *lds, float *lm) {
    typedef Shape<T, NB, FULL> S;
    constexpr int TP = S::TP, H = S::H, DKP = S::DKP, VW = S::VW, KS = S::KS, KE = S::KE, KD = S::KD;
    typedef typename S::VT VT;
    const int lane = p.tid & 63, col = lane & 15, qd = lane >> 4;
    const int t0 = __builtin_amdgcn_readfirstlane(p.tid >> 6);  // wave
    const int dk = FULL ? DKP : p.dk;
    const int p0 = p.it.p0, p1 = p.it.p1, page_rows = 1 << a.shift;
    const int endh = (p1 - 1) & ~15;  // the last half tile with positions
    const int n = ((p1 - p0 + TP - 1) / TP - t0 + kWaves - 1) / kWaves;  // tiles of this wave (0 or less: none)
    v4u kr[H][KS];
    VT vr[S::VE][S::VB];
    // positions behind the piece's end read its last one; their weights are 0. Page numbers are read a step
    // before the rows that they place.
    auto half = [&](int t, int h) { return min(p0 + t * TP + 16 * h, endh); };
    int pg[H];
    auto pages = [&](int t) {
#pragma unroll
        for (int h = 0; h < H; h++) pg[h] = p.table[half(t, h) >> a.shift];
    };
    auto head = [&](const char *pool, int page, int hb) {
        return (const T *)pool + (((size_t)page * a.n_kv + p.g) * page_rows + (hb & (page_rows - 1))) * dk;
    };
    // the rows go past the caches: this workgroup alone reads them (16 sequences of 1000 rows, f32: 27.5 us with,
    // 24.3 without keeping them)
    auto load_k = [&](int t) {
#pragma unroll
        for (int h = 0; h < H; h++) {
            const int hb = half(t, h);
            const T *b = head(a.pool_k, pg[h], hb) + min(col, p1 - 1 - hb) * dk + KE * qd;
#pragma unroll
            for (int j = 0; j < KS; j++)
                kr[h][j] = FULL || KD * j + KE * qd < dk ? __builtin_nontemporal_load((const v4u *)(b + KD * j)) : v4u{0, 0, 0, 0};
        }
    };
    auto load_v = [&](int t) {
#pragma unroll
        for (int h = 0; h < H; h++) {
            const int hb = half(t, h);
            const T *b = head(a.pool_v, pg[h], hb) + VW * col;
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int u = 0; u < S::VB; u++) {
                    VT z;
#pragma unroll
                    for (int c = 0; c < VW; c++) z[c] = (T)0.0f;
                    if (FULL || 16 * VW * u + VW * col < dk)
                        z = __builtin_nontemporal_load((const VT *)(b + min(4 * qd + i, p1 - 1 - hb) * dk + 16 * VW * u));
                    vr[4 * h + i][u] = z;
                }
        }
    };
    // the first half tiles' pages came with the item (the scalar cache's line of it)
#pragma unroll
    for (int h = 0; h < H; h++) {
        const int u = (half(t0, h) >> a.shift) - (p0 >> a.shift);
        pg[h] = u < 8 ? p.first[u] : p.table[half(t0, h) >> a.shift];
    }
    if (n > 0) load_k(t0);
    Rows<T, NB, FULL, MT> r;
    r.init(a, p, 0);
    if (n > 0) load_v(t0);
    pages(t0 + kWaves);
    // K's and V's registers are loaded with the next tile (more) as soon as they are used up. A branch around the
    // loads would make the waits for the older ones wait for them too, so the last step is one of its own.
    auto step = [&](int i, auto more) __attribute__((always_inline)) {
        constexpr bool MORE = decltype(more)::value;
        const int t = t0 + i * kWaves;
        r.no_scores();
        r.template scores<0, KS>([&](int h, int j) { return kr[h][j]; });
        if constexpr (MORE) load_k(t + kWaves);
        r.weights(p, p0 + t * TP, p0 + t * TP + TP > p.it.lim0);
        r.values([&](int u, auto &x) {
#pragma unroll
            for (int e = 0; e < S::VE; e++) x[e] = __builtin_bit_cast(typename Rows<T, NB, FULL, MT>::VU, vr[e][u]);
        });
        if constexpr (MORE) {
            load_v(t + kWaves);
            pages(t + 2 * kWaves);
        }
    };
    if (n > 0) {
        for (int i = 0; i + 1 < n; i++) step(i, std::true_type{});
        step(n - 1, std::false_type{});
    }
    r.sum_up();
    merge_waves<T, NB, FULL, MT>(a, p, r, t0, lds, lm);
}

// Reads of LDS and the wait for them in one block: the compiler, which cannot tell the stages of the ring below
// apart, would wait for all loads into LDS before any read of it.
__device__ __forceinline__ void lds_read(v4u (&d)[4], const unsigned (&at)[4]) {
    asm volatile("ds_read_b128 %0, %4\n\tds_read_b128 %1, %5\n\tds_read_b128 %2, %6\n\tds_read_b128 %3, %7\n\t"
                 "s_waitcnt lgkmcnt(0)"
                 : "=&v"(d[0]), "=&v"(d[1]), "=&v"(d[2]), "=&v"(d[3])
                 : "v"(at[0]), "v"(at[1]), "v"(at[2]), "v"(at[3])
                 : "memory");
}
__device__ __forceinline__ void lds_read(v2u (&d)[8], const unsigned (&at)[8]) {
    asm volatile("ds_read_b64 %0, %8\n\tds_read_b64 %1, %9\n\tds_read_b64 %2, %10\n\tds_read_b64 %3, %11\n\t"
                 "ds_read_b64 %4, %12\n\tds_read_b64 %5, %13\n\tds_read_b64 %6, %14\n\tds_read_b64 %7, %15\n\t"
                 "s_waitcnt lgkmcnt(0)"
                 : "=&v"(d[0]), "=&v"(d[1]), "=&v"(d[2]), "=&v"(d[3]), "=&v"(d[4]), "=&v"(d[5]), "=&v"(d[6]), "=&v"(d[7])
                 : "v"(at[0]), "v"(at[1]), "v"(at[2]), "v"(at[3]), "v"(at[4]), "v"(at[5]), "v"(at[6]), "v"(at[7])
                 : "memory");
}

// More rows: every wave has 16 MT rows of its own. Tiles pass through LDS, each read from memory once for all waves: a
// ring of them is filled without registers (memory to LDS), all but one on their way while that one is used; a
// row's 16-byte pieces are kept in an order (exclusive or with the row) that lets both the rows of K and the
// runs of V be read with few bank conflicts.
template <class T, int NB, bool FULL, int MT>
__device__ __forceinline__ void run_shared(const PageAttnArgs &a, const Piece &p, char *lds) {
    typedef Shape<T, NB, FULL, 4> S;  // (shorter runs of V: fewer registers)
    constexpr int TP = S::TP, H = S::H, NT = S::NT, DKP = S::DKP, VW = S::VW, KS = S::KS;
    constexpr int ST = ring_stages<NB>(), TB = tile_bytes<T, NB>();
    constexpr int RB = DKP * (int)sizeof(T), CR = RB / 16;  // bytes and pieces of a row in LDS
    constexpr int VP = 16 / (VW * (int)sizeof(T));          // runs of V per piece
    constexpr int X = CR % 16 == 0 && VP == 1 ? 16 : 8;     // pieces are permuted among so many
    constexpr int IN = TP * CR / (64 * kWaves);             // loads per wave for a tile's K, and for its V
    const int lane = p.tid & 63, col = lane & 15, qd = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(p.tid >> 6);
    const int dk = FULL ? DKP : p.dk, nv = p.it.ntok * p.rep;
    const int p0 = p.it.p0, p1 = p.it.p1, page_rows = 1 << a.shift;
    const int n = (p1 - p0 + TP - 1) / TP;
    // tile t's rows into its stage; positions behind the end read the last one. Page numbers are read a tile before.
    int pg[ST][IN], fl = lane;
    auto half_of = [&](int t, int i) { return min(p0 + t * TP + ((wave * IN + i) * 64 / CR & ~15), (p1 - 1) & ~15); };
    auto pages = [&](int t, int to) {
#pragma unroll
        for (int i = 0; i < IN; i++) pg[to][i] = p.table[half_of(t, i) >> a.shift];
    };
    auto fill = [&](int t, int from) {
        char *st = lds + (t % ST) * TB;
#pragma unroll
        for (int i = 0; i < IN; i++) {
            const int slot = (wave * IN + i) * 64 + fl;  // row, then the piece's place in it
            const int row = slot / CR, piece = (slot % CR) ^ (row & (X - 1));
            const int hb = half_of(t, i);  // (a load's rows are all of one half tile)
            const size_t at = ((((size_t)pg[from][i] * a.n_kv + p.g) * page_rows + (hb & (page_rows - 1))) + min(row & 15, p1 - 1 - hb)) *
                                  dk * sizeof(T) +
                              (FULL ? piece : min(piece, dk * (int)sizeof(T) / 16 - 1)) * 16;
            char *to = st + (wave * IN + i) * 1024;
            __builtin_amdgcn_global_load_lds((GlobalPtr)(a.pool_k + at), (LdsPtr)to, 16, 0, 0);
            __builtin_amdgcn_global_load_lds((GlobalPtr)(a.pool_v + at), (LdsPtr)(to + TP * RB), 16, 0, 0);
        }
    };
#pragma unroll
    for (int t = 0; t < ST; t++) pages(t, t);
    fill(0, 0);
    Rows<T, NB, FULL, MT, 4> r;
    const int v0 = wave * 16 * MT;
    r.init(a, p, v0);
    asm volatile("" : : "v"(r.sc[0]) : "memory");
#pragma unroll
    for (int t = 1; t + 1 < ST; t++) fill(t, t);
    // where the lane's first piece of a K row and its first V row's run lie in a tile; the others are at these
    // with bits flipped. (Opaque in the loop: what follows from them is formed again, not kept in registers.)
    static_assert(RB % (X * 16) == 0, "the flipped bits are the address's");
    const unsigned base = (unsigned)(uintptr_t)(LdsPtr)lds;
    const int run = run_of(col);
    unsigned ka = base + col * RB + (qd ^ (col & (X - 1))) * 16;
    unsigned va = base + TP * RB + 4 * qd * RB + (run / VP ^ (4 * qd & (X - 1))) * 16 + run % VP * (16 / VP);
    // before tile t: its loads have landed when those of the ones behind it may be under way, everybody's behind the
    // barrier; nobody reads the stage before it any more either
    auto turn = [&](int t) __attribute__((always_inline)) {
        constexpr int behind = (ST - 2) * 2 * IN;
        __builtin_amdgcn_s_waitcnt((behind & 15) | (behind >> 4 << 14) | 0x0f70);
        __builtin_amdgcn_s_barrier();
        asm volatile("" : "+v"(ka), "+v"(va), "+v"(fl) : : "memory");
        fill(t + ST - 1, ST - 1);
        pages(t + ST, ST - 1);
    };
    if (v0 >= nv) {
        // (a loop of its own: with a way around the products in it the sums were copied for every tile)
        for (int t = 0; t < n; t++) turn(t);
        __syncthreads();
        return;
    }
    for (int t = 0; t < n; t++) {
        const int tp = p0 + t * TP;
        turn(t);
        const unsigned st = (unsigned)(t % ST) * TB;
        r.no_scores();
        // (products before the other waves' weights: 32 trees of up to 32 rows 72.7 us without, 71.5; f32 no better)
        if constexpr (S::F16) __builtin_amdgcn_s_setprio(1);
        // four pieces of K at a time
        each(std::make_integer_sequence<int, H * KS / 4>{}, [&](auto part) __attribute__((always_inline)) {
            constexpr int G = decltype(part)::value;
            v4u kr[4];
            unsigned at[4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int j = (4 * G + e) / H, h = (4 * G + e) % H;
                at[e] = (ka ^ 64 * (j % (X / 4))) + (st + h * 16 * RB + j / (X / 4) * X * 16);
            }
            lds_read(kr, at);
            r.template scores<4 * G / H, 4 * (G + 1) / H>([&](int h, int j) { return kr[j * H + h - 4 * G]; });
        });
        if constexpr (S::F16) __builtin_amdgcn_s_setprio(0);
        r.weights(p, tp, tp + TP > p.it.lim0);
        if constexpr (S::F16) __builtin_amdgcn_s_setprio(1);
        r.values([&](int u, auto &x) __attribute__((always_inline)) {
            constexpr int VE = S::VE;
            unsigned at[VE];
#pragma unroll
            for (int e = 0; e < VE; e++)
                at[e] = (va ^ 16 * (e % 4)) + (st + (e / 4 * 16 + e % 4) * RB + u * (16 / VP) * 16);
            lds_read(x, at);
        });
    }
    __builtin_amdgcn_s_setprio(0);
    __syncthreads();  // nothing is on its way and no stage is read: they are free for the next piece
    r.sum_up();
    const Results res(a, p);
    bool bad = false;
#pragma unroll
    for (int mt = 0; mt < MT; mt++) {
        const int v = v0 + mt * 16 + col;
        const bool live = v < nv;
        const int at = res.at(a, p, min(v, nv - 1)) + dim_of<VW>(0, qd);
        const float f = res.direct ? 1.0f / r.l[mt] : 1.0f;
        bad |= live && !__builtin_isfinite(r.l[mt]);
        float worst = 0.0f;
#pragma unroll
        for (int t = 0; t < NT; t += 4)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int d = dim_of<VW>(t, 4 * i);  // run_of's inverse: run 4 i + quarter
                const v4f x = r.four(mt, t, i) * f;
                // 0 * x: NaN for an x that is not finite
                worst = __builtin_fmaf(0.0f, (x[0] + x[1]) + (x[2] + x[3]), worst);
                if (live && (FULL || dim_of<VW>(t, 4 * i + qd) < dk)) *(v4f *)(res.to + at + d) = x;
            }
        bad |= live && !(worst == 0.0f);
        if (live && !res.direct && qd == 0) res.state(v, r.m[mt], r.l[mt]);
    }
    if (__ballot(bad)) plain_rows<T>(a, p, v0, min(nv, v0 + 16 * MT), 1);
}

// MT: of the blocks that all waves take (a step without blocks of more than 16 rows runs the smaller kernel).
template <class T, int NB, bool FULL, int MT>
__global__ void __launch_bounds__(64 * kWaves) __attribute__((amdgpu_waves_per_eu(2)))
page_attn_kernel(PageAttnArgs a) {
    constexpr const int(&shapes)[3] = kShapeRows[shape_class(FULL ? 64 * NB : 64 * NB - 8, sizeof(T) == 2)];
    constexpr int ring = ring_stages<NB>() * tile_bytes<T, NB>();
    __shared__ __attribute__((aligned(1024))) char lds[ring > kMergeBytes<NB> ? ring : kMergeBytes<NB>];
    __shared__ float lm[kWaves * 16 * 2 + 4];
    // one read of memory (a piece's item) before the first K rows are on their way
    const ScalarInts step = (ScalarInts)(uintptr_t)a.step;
    const int n = a.items >= 0 ? a.items : step[kStepItems] * a.n_kv;
    Piece p;
    p.rep = a.rep;
    p.per_rep = 1.0f / (float)a.rep;
    p.dk = a.d_k;
    p.step = a.step;
    p.rows = step_rows(a);
    for (int w = blockIdx.x; w < n; w += gridDim.x) {
        p.tid = threadIdx.x;
        asm volatile("" : "+v"(p.tid));
        const int i = w / a.n_kv;
        p.g = w - i * a.n_kv;
        const ScalarInts it = step + kStepHeader + 16 * i;
        p.it = {it[0], it[1], it[2], it[3], it[4], it[5], it[6], it[7], {}};
        p.first = it + 8;
        p.table = (ScalarInts)(uintptr_t)(a.step + p.it.table);
        switch (p.it.flags & kItemShape) {
        case 0:
            if constexpr (shapes[0] != 0) run_split<T, NB, FULL, MT>(a, p, lds, lm);
            break;
        case 1: run_shared<T, NB, FULL, 1>(a, p, lds); break;
        default:
            if constexpr (shapes[2] != 0) run_shared<T, NB, FULL, 2>(a, p, lds);
            break;
        }
    }
}

// The states of one (row, q head), merged by G groups of LP lanes of four dimensions, a group every G-th piece,
// the groups' in LDS. Rows with one piece are written already. Bound by latency where there are few rows (long lists
// are shared by groups, four pieces' states in flight), else by the states' bytes.
template <int LP, int G>
__global__ void __launch_bounds__(256) page_combine_kernel(PageAttnArgs a) {
    constexpr int P = 256 / (LP * G);  // pairs per workgroup
    constexpr int U = 4;
    __shared__ v4f os[G > 1 ? 256 : 1];
    __shared__ v2f ss[G > 1 ? G * P : 1];
    const int sub = threadIdx.x % LP, grp = threadIdx.x / LP % G, d = sub * 4;
    const int pair = threadIdx.x / (LP * G), x = blockIdx.x * P + pair;
    const int r = x / a.n_heads, h = x - r * a.n_heads;
    bool live = r < (a.rows_at < 0 ? a.step[kStepRows] : a.grid_rows);
    const StepRow row = step_rows(a)[live ? r : 0];
    live = live && !row.direct;
    if (G == 1 && !live) return;
    const int g = h / a.rep, j = h - g * a.rep;
    const size_t base = (size_t)g * a.slots + j;
    const int n0 = row.parts[0].pieces, n1 = n0 + row.parts[1].pieces, all = live ? n1 + row.parts[2].pieces : 0;
    const int dc = d < a.d_k ? d : 0;
    float M = -INFINITY, L = 0.0f;
    v4f O = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int c0 = grp; c0 < all; c0 += U * G) {
        v2f s[U];
        v4f o[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int c = min(c0 + u * G, all - 1);
            const int at = c < n0   ? row.parts[0].first + c * row.parts[0].step
                           : c < n1 ? row.parts[1].first + (c - n0) * row.parts[1].step
                                    : row.parts[2].first + (c - n1) * row.parts[2].step;
            s[u] = *(const v2f *)(a.ml + (base + at) * 2);
            // (each state is read once: 244 rows of 32 pieces 53.6 -> 52.2 us)
            o[u] = __builtin_nontemporal_load((const v4f *)(a.part + (base + at) * a.d_k + dc));
        }
        float mn = M;
#pragma unroll
        for (int u = 0; u < U; u++)
            if (c0 + u * G < all) mn = fmaxf(mn, s[u][0]);
        const float f = M == -INFINITY ? 0.0f : exp2_(M - mn);
        L = L * f;
        O = O * f;
#pragma unroll
        for (int u = 0; u < U; u++)
            if (c0 + u * G < all) {
                const float w = s[u][0] == -INFINITY ? 0.0f : exp2_(s[u][0] - mn);
                L = L + s[u][1] * w;
                O = O + o[u] * w;
            }
        M = mn;
    }
    if constexpr (G > 1) {
        os[threadIdx.x] = O;
        if (sub == 0) ss[pair * G + grp] = v2f{M, L};
        __syncthreads();
        if (grp || !live) return;
        float mn = M;
#pragma unroll
        for (int u = 1; u < G; u++) mn = fmaxf(mn, ss[pair * G + u][0]);
        const float f = M == -INFINITY ? 0.0f : exp2_(M - mn);
        L = L * f;
        O = O * f;
#pragma unroll
        for (int u = 1; u < G; u++) {
            const v2f s = ss[pair * G + u];
            const float w = s[0] == -INFINITY ? 0.0f : exp2_(s[0] - mn);
            L = L + s[1] * w;
            O = O + os[threadIdx.x + u * LP] * w;
        }
    }
    if (d < a.d_k) *(v4f *)(a.out + ((size_t)r * a.n_heads + h) * a.d_k + d) = O * (1.0f / L);
}

template <class T, int NB, bool FULL>
void launch_attn_full(const PageAttnArgs &a, hipStream_t s) {
    constexpr bool two = kShapeRows[shape_class(FULL ? 64 * NB : 64 * NB - 8, sizeof(T) == 2)][0] > 16;
    if (two && a.wide)
        hipLaunchKernelGGL((page_attn_kernel<T, NB, FULL, two ? 2 : 1>), dim3(a.grid_items), dim3(64 * kWaves), 0, s, a);
    else
        hipLaunchKernelGGL((page_attn_kernel<T, NB, FULL, 1>), dim3(a.grid_items), dim3(64 * kWaves), 0, s, a);
}
template <class T, int NB>
void launch_attn(const PageAttnArgs &a, hipStream_t s) {
    if (a.d_k == 64 * NB) launch_attn_full<T, NB, true>(a, s);
    else launch_attn_full<T, NB, false>(a, s);
}

template <class T, int LP>
sllm_status launch(const PageAttnArgs &a, hipStream_t s) {
    constexpr int hg = kPrepThreads / LP, groups = 256 / LP;
    const int most = (a.n_heads + a.n_kv + hg - 1) / hg, want = 2048 / a.grid_rows;
    const int y = want < 1 ? 1 : want < most ? want : most;
    hipLaunchKernelGGL((page_prep_kernel<T, LP>), dim3(a.grid_rows, y), dim3(kPrepThreads), 0, s, a);
    SLLM_HIP(hipGetLastError());
    switch ((a.d_k + 63) / 64) {
    case 1: launch_attn<T, 1>(a, s); break;
    case 2: launch_attn<T, 2>(a, s); break;
    case 3: launch_attn<T, 3>(a, s); break;
    default: launch_attn<T, 4>(a, s); break;
    }
    SLLM_HIP(hipGetLastError());
    if (!a.combine) return SLLM_OK;
    const int pairs = a.grid_rows * a.n_heads;
    // Groups of lanes to a pair: as many as have two pieces each, while the launch stays small (a captured one may meet any list).
    // us (attention in all) with one, two, four and eight: one row of 32 heads, 32 pieces 23.0, 19.9, 19.2, 18.8; 4 of 16, 9: 15.4,
    // 14.7, 13.7, 13.7; 16 of 16, 8: 14.0, 13.2, 12.8, 12.8; 61 of 32, 32: 53.5, 52.1, 52.1, 52.8; 200 of 32, 4: 37.1, 36.1, 39.2,
    // 41.4; 1055 of 32, 2: 86.5, 91.7, 96.3, 107.9. (Over 782 steps 0.4 % above the best in the mean; with four pieces each 1.2 %.)
    int g = groups;
    while (a.combine != INT32_MAX && g > 1 && (2 * g > a.combine || (int64_t)pairs * g * LP > kMergeThreads)) g /= 2;
    const dim3 grid((unsigned)((pairs + groups / g - 1) / (groups / g)));
    switch (g) {
    case 1: hipLaunchKernelGGL((page_combine_kernel<LP, 1>), grid, dim3(256), 0, s, a); break;
    case 2: hipLaunchKernelGGL((page_combine_kernel<LP, 2>), grid, dim3(256), 0, s, a); break;
    case 4: hipLaunchKernelGGL((page_combine_kernel<LP, 4>), grid, dim3(256), 0, s, a); break;
    default: hipLaunchKernelGGL((page_combine_kernel<LP, groups>), grid, dim3(256), 0, s, a);
    }
    SLLM_HIP(hipGetLastError());
    return SLLM_OK;
}

}  // namespace

sllm_status launch_page_attention(const PageAttnArgs &a, hipStream_t s) {
    if (a.type == SLLM_CACHE_F16) return a.d_k <= 128 ? launch<_Float16, 32>(a, s) : launch<_Float16, 64>(a, s);
    return a.d_k <= 128 ? launch<float, 32>(a, s) : launch<float, 64>(a, s);
}

}  // namespace sllm
