// The attention section (bias, QK norm, RoPE, append, causal GQA attention) of a batch of sequences
// over a page cache.
//
// page_prep_kernel: the step's rows: q heads rotated to the batch's memory, k and v into their pages.
// page_attn_kernel: the attention over pieces of segments (qmm_pages.hip: a segment is a run of positions with the
//   rows that see it: one sequence's own rows, or those of all sequences that share its pages), whose K and V
//   are read once for all rows of a block.
// page_combine_kernel: the pieces' softmax states of every row and head, merged.
#include <hip/hip_runtime.h>

#include "qmm_device.hpp"
#include "qmm_pages.hpp"

namespace sllm {

namespace {

constexpr int kMaxDk = 256;
typedef float v2f __attribute__((ext_vector_type(2)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef _Float16 v4h __attribute__((ext_vector_type(4)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef unsigned v2u __attribute__((ext_vector_type(2)));
typedef unsigned v4u __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

__device__ __forceinline__ void put4(float *dst, v4f x) { *(v4f *)dst = x; }
__device__ __forceinline__ void put4(_Float16 *dst, v4f x) {
    *(v4h *)dst = v4h{(_Float16)x[0], (_Float16)x[1], (_Float16)x[2], (_Float16)x[3]};
}

// Bias (model_f32.go:398-420), per-head RMSNorm (:424-435), RoPE (applyRopeInPlaceF32,
// float32_ops.go:174-188) of every q and k head of a row, and the row's k and v into its page
// (the append, model_f32.go:445-448), rounded to the cache's type, once.
// A workgroup takes heads of one row, LP lanes of four dimensions to a head; the rotation (the same for
// every head: float32 angle, sine and cosine in 64 bits, as the reference) is formed once in LDS, the first
// heads' elements loaded before it. Bound by latency: few rows have a workgroup for every 256 / LP heads.
// (16 rows of 32 + 8 heads of 128, us: one workgroup of eight waves per row, a wave per head 8.2; this 2.7.)
constexpr int kPrepThreads = 256;
template <class T, int LP>
__global__ void __launch_bounds__(kPrepThreads) page_prep_kernel(PageAttnArgs a) {
    __shared__ float rc[kMaxDk / 2], rs[kMaxDk / 2];
    constexpr int HG = kPrepThreads / LP;
    const int r = blockIdx.x, sub = threadIdx.x % LP;
    if (r >= a.step[kStepRows]) return;
    const StepRow &row = ((const StepRow *)(a.step + a.step[kStepRowsAt]))[r];
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
        if (d >= dk) continue;
        if (isq) {
            *(v4f *)(a.qrot + off) = x;
            continue;
        }
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
// f16: 32 positions a step; K and V are exact operands, q and the weights go in as two f16 each (22 bits of
//   them: 2^-22 of the value; the row's q scaled by a power of two, so no float32 leaves f16's range).
// f32: 16 positions a step, fp32 matrix instructions.
// Softmax weights are 2^(s - m) with m the largest score at the last time that one exceeded it by
// more than 2^8: while none does, neither the row's lanes have to agree on a maximum nor the
// sums to be scaled again. Weights stay below 2^8, sums in fp32.
// A result that is not finite (a non-finite K or V element, also one that only other rows of the block
// see, where the matrix instruction forms 0 * inf) is computed again, row by row, as the formula says.
constexpr int kWaves = 4;
constexpr int kFewPieces = 8;    // of a row, up to which one group of lanes merges them
constexpr float kGrow = 8.0f;  // log2 of how far weights may exceed 1

template <bool B>
struct Bool {
    static constexpr bool value = B;
};
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
    ScalarInts table, first;  // the sequence's page ids; the first ones of the piece
    const int *step;
    const StepRow *rows;
    // the query row of row v of the block
    __device__ __forceinline__ int row_of(int v) const {
        const int t = v / rep;
        return it.flags & kItemRun ? it.tok + t : step[it.tok + t];
    }
};

// Row v's result: the output (direct) or the piece's state.
__device__ __forceinline__ size_t out_at(const PageAttnArgs &a, const Piece &p, int v) {
    const int j = v % p.rep;
    return p.it.flags & kItemDirect ? ((size_t)p.row_of(v) * a.n_heads + p.g * p.rep + j) * p.dk
                                    : ((size_t)p.g * a.slots + p.it.slot + v) * p.dk;
}
__device__ __forceinline__ void put_state(const PageAttnArgs &a, const Piece &p, int v, float m, float l) {
    float *ml = a.ml + ((size_t)p.g * a.slots + p.it.slot + v) * 2;
    ml[0] = m;
    ml[1] = l;
}

// One row after the other, one position after the other, by one wave: rows v0, v0 + dv, ... of the piece.
template <class T>
__device__ __forceinline__ void plain_rows(const PageAttnArgs &a, const Piece &p, int v0, int v1, int dv) {
    const int lane = threadIdx.x & 63, dk = p.dk, d = 4 * lane, page_rows = 1 << a.shift;
    for (int v = v0; v < v1; v += dv) {
        const int row = p.row_of(v);
        const int end = p.it.flags & kItemCausal ? min(p.it.p1, p.rows[row].pos + 1) : p.it.p1;
        const float *qr = a.qrot + ((size_t)row * a.n_heads + p.g * p.rep + v % p.rep) * dk;
        v4f q = {0.0f, 0.0f, 0.0f, 0.0f}, o = q;
        if (d < dk) q = *(const v4f *)(qr + d);
        float m = -INFINITY, l = 0.0f;
        for (int x = p.it.p0; x < end; x++) {
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
        const bool direct = p.it.flags & kItemDirect;
        const size_t at = out_at(a, p, v) + d;
        if (d < dk) *(v4f *)((direct ? a.out : a.part) + at) = direct ? o * (1.0f / l) : o;
        if (!direct && lane == 0) put_state(a, p, v, m, l);
    }
}

// Dimension of element (tile t, accumulator i) of a lane in quarter q. A lane of V reads VW dimensions at once.
template <int VW>
__device__ __forceinline__ constexpr int dim_of(int t, int q, int i) {
    return 16 * VW * (t / VW) + VW * (4 * q + i) + t % VW;
}

template <class T, int NB, bool FULL, int MT, int RW>
__device__ __forceinline__ void run_piece(const PageAttnArgs &a, const Piece &p, float *lds) {
    constexpr bool F16 = sizeof(T) == 2;
    constexpr int TP = Kind<T>::kTile, H = TP / 16, NT = 4 * NB, DKP = 64 * NB;
    constexpr int VW = F16 && FULL && NB % 2 == 0 ? 8 : 4;
    constexpr int KS = F16 ? 2 * NB : 4 * NB;  // 16-byte pieces of a K row per lane
    constexpr int KD = F16 ? 32 : 16;          // dimensions of a piece over the quarters
    constexpr int VB = DKP / (16 * VW);        // runs of dimensions per V row and lane
    constexpr int VE = 4 * H;                  // V rows per lane and step
    typedef T VT __attribute__((ext_vector_type(VW)));
    const int lane = threadIdx.x & 63, col = lane & 15, qd = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int dk = FULL ? DKP : p.dk, rep = p.rep, nv = p.it.ntok * rep;
    const int v0 = RW == kWaves ? wave * 16 * MT : 0;
    const int p0 = p.it.p0, p1 = p.it.p1;
    const int page_rows = 1 << a.shift;
    if (v0 >= nv) return;  // (the first wave's rows exist)

    const int tiles = (p1 - p0 + TP - 1) / TP;
    constexpr int dt = RW == kWaves ? 1 : kWaves;
    const int t0 = RW == kWaves ? 0 : wave;
    const int endh = (p1 - 1) & ~15;  // the last half tile with positions
    v4u kr[H][KS];
    VT vr[VE][VB];
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
    // rows that one workgroup alone reads go past the caches (16 sequences of 1000 rows, f32: 27.5 us with, 24.3
    // without keeping them)
    auto load_k = [&](int t) {
#pragma unroll
        for (int h = 0; h < H; h++) {
            const int hb = half(t, h);
            const T *b = head(a.pool_k, pg[h], hb) + min(col, p1 - 1 - hb) * dk + (F16 ? 8 : 4) * qd;
#pragma unroll
            for (int j = 0; j < KS; j++) {
                const v4u *x = (const v4u *)(b + KD * j);
                if (FULL || KD * j + (F16 ? 8 : 4) * qd < dk) kr[h][j] = RW == 1 ? __builtin_nontemporal_load(x) : *x;
                else kr[h][j] = v4u{0, 0, 0, 0};
            }
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
                for (int u = 0; u < VB; u++) {
                    const VT *x = (const VT *)(b + min(4 * qd + i, p1 - 1 - hb) * dk + 16 * VW * u);
                    VT z;
#pragma unroll
                    for (int c = 0; c < VW; c++) z[c] = (T)0.0f;
                    if (FULL || 16 * VW * u + VW * col < dk) z = RW == 1 ? __builtin_nontemporal_load(x) : *x;
                    vr[4 * h + i][u] = z;
                }
        }
    };
    // the first half tiles' pages came with the item (the scalar cache's line of it)
#pragma unroll
    for (int h = 0; h < H; h++) pg[h] = p.first[(half(t0, h) >> a.shift) - (p0 >> a.shift)];
    const int n = (tiles - t0 + dt - 1) / dt;  // tiles of this wave (0 or less: none)
    if (n > 0) load_k(t0);
    v4f qf[F16 ? 1 : MT][F16 ? 1 : KS];
    v8h qh[F16 ? MT : 1][F16 ? KS : 1], ql[F16 ? MT : 1][F16 ? KS : 1];
    float sc[MT], m[MT], l[MT];
    int lim[MT];
    v4f o[MT][NT];
#pragma unroll
    for (int mt = 0; mt < MT; mt++) {
        const int v = min(v0 + mt * 16 + col, nv - 1);
        const int row = p.row_of(v);
        lim[mt] = p.it.flags & kItemCausal ? min(p1, p.rows[row].pos + 1) : p1;
        const float *qr = a.qrot + ((size_t)row * a.n_heads + p.g * rep + v % rep) * dk;
        sc[mt] = a.scale_log2;
        if constexpr (F16) {
            v4f x[2 * KS];
            float big = 0.0f;
#pragma unroll
            for (int j = 0; j < KS; j++)
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const int d = KD * j + 8 * qd + 4 * i;
                    x[2 * j + i] = FULL || d < dk ? *(const v4f *)(qr + d) : v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int c = 0; c < 4; c++) big = fmaxf(big, __builtin_fabsf(x[2 * j + i][c]));
                }
            big = fmaxf(big, __shfl_xor(big, 16, 64));
            big = fmaxf(big, __shfl_xor(big, 32, 64));
            // the row's largest element between 2^10 and 2^11
            int e = (int)((__builtin_bit_cast(unsigned, big) >> 23) & 255u) - 127 - 10;
            e = e < -110 ? -110 : e;
            const float up = __builtin_bit_cast(float, (unsigned)(127 - e) << 23);
            sc[mt] = a.scale_log2 * __builtin_bit_cast(float, (unsigned)(127 + e) << 23);
#pragma unroll
            for (int j = 0; j < KS; j++)
#pragma unroll
                for (int c = 0; c < 8; c++) {
                    const float y = x[2 * j + c / 4][c % 4] * up;
                    qh[mt][j][c] = (_Float16)y;
                    ql[mt][j][c] = (_Float16)(y - (float)(_Float16)y);
                }
        } else {
#pragma unroll
            for (int j = 0; j < KS; j++) {
                const int d = KD * j + 4 * qd;
                qf[mt][j] = FULL || d < dk ? *(const v4f *)(qr + d) : v4f{0.0f, 0.0f, 0.0f, 0.0f};
            }
        }
        m[mt] = -INFINITY;
        l[mt] = 0.0f;
#pragma unroll
        for (int t = 0; t < NT; t++) o[mt][t] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    }

    if (n > 0) load_v(t0);
    pages(t0 + dt);
    // A step: the scores of the wave's i-th tile, the weights, the values. K's and V's registers are
    // loaded with the next tile (more) as soon as they are used up. A branch around the loads would make the
    // waits for the older ones wait for them too, so the last step is one of its own.
    auto step = [&](int i, auto more) __attribute__((always_inline)) {
        constexpr bool MORE = decltype(more)::value;
        const int t = t0 + i * dt;
        v4f s[MT][H];
#pragma unroll
        for (int mt = 0; mt < MT; mt++)
#pragma unroll
            for (int h = 0; h < H; h++) s[mt][h] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < KS; j++)
#pragma unroll
            for (int h = 0; h < H; h++)
#pragma unroll
                for (int mt = 0; mt < MT; mt++) {
                    if constexpr (F16) {
                        const v8h k = __builtin_bit_cast(v8h, kr[h][j]);
                        s[mt][h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, qh[mt][j], s[mt][h], 0, 0, 0);
                        s[mt][h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, ql[mt][j], s[mt][h], 0, 0, 0);
                    } else {
                        const v4f k = __builtin_bit_cast(v4f, kr[h][j]);
#pragma unroll
                        for (int c = 0; c < 4; c++)
                            s[mt][h] = __builtin_amdgcn_mfma_f32_16x16x4f32(k[c], qf[mt][j][c], s[mt][h], 0, 0, 0);
                    }
                }
        if constexpr (MORE) load_k(t + dt);
        const int tp = p0 + t * TP;
        const bool masked = tp + TP > p.it.lim0;  // some row does not see all of the tile
#pragma unroll
        for (int mt = 0; mt < MT; mt++) {
            float mx = -INFINITY;
#pragma unroll
            for (int h = 0; h < H; h++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    float x = s[mt][h][i] * sc[mt];
                    if (masked && tp + 16 * h + 4 * qd + i >= lim[mt]) x = -INFINITY;
                    s[mt][h][i] = x;
                    mx = fmaxf(mx, x);
                }
            if (__ballot(mx > m[mt] + kGrow)) {  // from -inf on: any score
                float mn = fmaxf(mx, __shfl_xor(mx, 16, 64));
                mn = fmaxf(m[mt], fmaxf(mn, __shfl_xor(mn, 32, 64)));
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
                    s[mt][h][i] = exp2_(s[mt][h][i] - ref);
                    sum = sum + s[mt][h][i];
                }
            l[mt] = l[mt] + sum;
        }
        if constexpr (F16) {
            v8h ph[MT], pl[MT];
#pragma unroll
            for (int mt = 0; mt < MT; mt++) {
                v4u hi, lo;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float x = s[mt][i / 2][2 * (i & 1)], y = s[mt][i / 2][2 * (i & 1) + 1];
                    const auto hp = __builtin_amdgcn_cvt_pkrtz(x, y);
                    hi[i] = __builtin_bit_cast(unsigned, hp);
                    lo[i] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_pkrtz(x - (float)hp[0], y - (float)hp[1]));
                }
                ph[mt] = __builtin_bit_cast(v8h, hi);
                pl[mt] = __builtin_bit_cast(v8h, lo);
            }
#pragma unroll
            for (int t2 = 0; t2 < NT; t2++) {
                // the eight rows' element t2 of the lane's run
                const int u = t2 / VW, c = t2 % VW;
                v4u x;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    typedef unsigned VU __attribute__((ext_vector_type(VW / 2)));
                    const unsigned e0 = __builtin_bit_cast(VU, vr[2 * i][u])[c / 2];
                    const unsigned e1 = __builtin_bit_cast(VU, vr[2 * i + 1][u])[c / 2];
                    x[i] = __builtin_amdgcn_perm(e1, e0, c & 1 ? 0x07060302u : 0x05040100u);
                }
                const v8h va = __builtin_bit_cast(v8h, x);
#pragma unroll
                for (int mt = 0; mt < MT; mt++) {
                    o[mt][t2] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, ph[mt], o[mt][t2], 0, 0, 0);
                    o[mt][t2] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, pl[mt], o[mt][t2], 0, 0, 0);
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int t2 = 0; t2 < NT; t2++)
#pragma unroll
                    for (int mt = 0; mt < MT; mt++)
                        o[mt][t2] = __builtin_amdgcn_mfma_f32_16x16x4f32(vr[i][t2 / VW][t2 % VW], s[mt][0][i], o[mt][t2], 0, 0, 0);
        }
        if constexpr (MORE) {
            load_v(t + dt);
            pages(t + 2 * dt);
        }
    };
    if (n > 0) {
        for (int i = 0; i + 1 < n; i++) step(i, Bool<true>{});
        step(n - 1, Bool<false>{});
    }
#pragma unroll
    for (int mt = 0; mt < MT; mt++) {
        l[mt] = l[mt] + __shfl_xor(l[mt], 16, 64);
        l[mt] = l[mt] + __shfl_xor(l[mt], 32, 64);
    }
    const bool direct = p.it.flags & kItemDirect;
    float *dst = direct ? a.out : a.part;
    if constexpr (RW == kWaves) {
        // the wave's rows are its own
        bool bad = false;
#pragma unroll
        for (int mt = 0; mt < MT; mt++) {
            const int v = v0 + mt * 16 + col;
            const bool live = v < nv;
            const size_t at = out_at(a, p, live ? v : 0);
            const float f = direct ? 1.0f / l[mt] : 1.0f;
            bad |= live && !__builtin_isfinite(l[mt]);
#pragma unroll
            for (int t = 0; t < NT; t += 4)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int d = dim_of<VW>(t, qd, i);
                    const v4f x = v4f{o[mt][t][i], o[mt][t + 1][i], o[mt][t + 2][i], o[mt][t + 3][i]} * f;
                    if (live && (FULL || d < dk)) {
                        *(v4f *)(dst + at + d) = x;
                        bad |= !(__builtin_isfinite(x[0]) && __builtin_isfinite(x[1]) && __builtin_isfinite(x[2]) &&
                                 __builtin_isfinite(x[3]));
                    }
                }
            if (live && !direct && qd == 0) put_state(a, p, v, m[mt], l[mt]);
        }
        if (__ballot(bad)) plain_rows<T>(a, p, v0, min(nv, v0 + 16 * MT), 1);
    } else {
        // the waves' states of each row, merged in wave order
        constexpr int RS = DKP + 4;
        float *lo_ = lds, *lm = lds + kWaves * 16 * RS;
        int *flag = (int *)(lm + kWaves * 16 * 2);
        if (threadIdx.x == 0) *flag = 0;
#pragma unroll
        for (int mt = 0; mt < MT; mt++) {
            if (mt) __syncthreads();
#pragma unroll
            for (int t = 0; t < NT; t += 4)
#pragma unroll
                for (int i = 0; i < 4; i++)
                    *(v4f *)(lo_ + (wave * 16 + col) * RS + dim_of<VW>(t, qd, i)) =
                        v4f{o[mt][t][i], o[mt][t + 1][i], o[mt][t + 2][i], o[mt][t + 3][i]};
            if (qd == 0) {
                lm[(wave * 16 + col) * 2] = m[mt];
                lm[(wave * 16 + col) * 2 + 1] = l[mt];
            }
            __syncthreads();
            for (int x = threadIdx.x; x < 16 * (DKP / 4); x += 64 * kWaves) {
                const int r = x / (DKP / 4), d = x % (DKP / 4) * 4, v = mt * 16 + r;
                if (v >= nv || (!FULL && d >= dk)) continue;
                float M = -INFINITY;
#pragma unroll
                for (int w = 0; w < kWaves; w++) M = fmaxf(M, lm[(w * 16 + r) * 2]);
                float L = 0.0f;
                v4f O = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int w = 0; w < kWaves; w++) {
                    const float mw = lm[(w * 16 + r) * 2];
                    const float f = mw == -INFINITY ? 0.0f : exp2_(mw - M);
                    L = L + lm[(w * 16 + r) * 2 + 1] * f;
                    O = O + *(const v4f *)(lo_ + (w * 16 + r) * RS + d) * f;
                }
                if (direct) O = O * (1.0f / L);
                else if (d == 0) put_state(a, p, v, M, L);
                *(v4f *)(dst + out_at(a, p, v) + d) = O;
                if (!(__builtin_isfinite(L) && __builtin_isfinite(O[0]) && __builtin_isfinite(O[1]) &&
                      __builtin_isfinite(O[2]) && __builtin_isfinite(O[3])))
                    *flag = 1;
            }
        }
        __syncthreads();
        if (*flag) plain_rows<T>(a, p, wave, nv, kWaves);
        __syncthreads();  // the memory is free for the next piece
    }
}

template <class T, int NB, bool FULL>
__global__ void __launch_bounds__(64 * kWaves) __attribute__((amdgpu_waves_per_eu(NB <= 2 ? 2 : 1)))
page_attn_kernel(PageAttnArgs a) {
    extern __shared__ __attribute__((aligned(16))) float lds[];
    // one read of memory (a piece's item) before the first K rows are on their way
    const ScalarInts step = (ScalarInts)(uintptr_t)a.step;
    const int n = a.items >= 0 ? a.items : step[kStepItems] * a.n_kv;
    Piece p;
    p.rep = a.rep;
    p.dk = a.d_k;
    p.step = a.step;
    p.rows = (const StepRow *)(a.step + step[kStepRowsAt]);
    for (int w = blockIdx.x; w < n; w += gridDim.x) {
        const int i = w / a.n_kv;
        p.g = w - i * a.n_kv;
        const ScalarInts it = step + kStepHeader + 16 * i;
        p.it = {it[0], it[1], it[2], it[3], it[4], it[5], it[6], it[7], {}};
        p.first = it + 8;
        p.table = (ScalarInts)(uintptr_t)(a.step + p.it.table);
        switch (p.it.flags & kItemShape) {
        case 0: run_piece<T, NB, FULL, 1, 1>(a, p, lds); break;
        case 1: run_piece<T, NB, FULL, 2, 1>(a, p, lds); break;
        default: run_piece<T, NB, FULL, 2, kWaves>(a, p, lds); break;
        }
    }
}

// The states of one (row, q head), merged by G groups of LP lanes of four dimensions, a group every G-th piece,
// the groups' in LDS. Rows with one piece are written already. Bound by latency: one group takes
// few pieces, eight long lists, four pieces' states in flight.
template <int LP, int G>
__global__ void __launch_bounds__(256) page_combine_kernel(PageAttnArgs a) {
    constexpr int P = 256 / (LP * G);  // pairs per workgroup
    constexpr int U = 4;
    __shared__ v4f os[G > 1 ? 256 : 1];
    __shared__ v2f ss[G > 1 ? G : 1];
    const int sub = threadIdx.x % LP, grp = threadIdx.x / LP % G, d = sub * 4;
    const int x = blockIdx.x * P + threadIdx.x / (LP * G);
    const int r = x / a.n_heads, h = x - r * a.n_heads;
    // (G > 1: all of a workgroup's threads have the same pair)
    if (r >= a.step[kStepRows]) return;
    const StepRow row = ((const StepRow *)(a.step + a.step[kStepRowsAt]))[r];
    if (row.direct) return;
    const int g = h / a.rep, j = h - g * a.rep;
    const size_t base = (size_t)g * a.slots + j;
    const int n0 = row.parts[0].pieces, n1 = n0 + row.parts[1].pieces, all = n1 + row.parts[2].pieces;
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
            o[u] = *(const v4f *)(a.part + (base + at) * a.d_k + dc);
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
        if (sub == 0) ss[grp] = v2f{M, L};
        __syncthreads();
        if (grp) return;
        float mn = M;
#pragma unroll
        for (int u = 1; u < G; u++) mn = fmaxf(mn, ss[u][0]);
        const float f = M == -INFINITY ? 0.0f : exp2_(M - mn);
        L = L * f;
        O = O * f;
#pragma unroll
        for (int u = 1; u < G; u++) {
            const float w = ss[u][0] == -INFINITY ? 0.0f : exp2_(ss[u][0] - mn);
            L = L + ss[u][1] * w;
            O = O + os[threadIdx.x + u * LP] * w;
        }
    }
    if (d < a.d_k) *(v4f *)(a.out + ((size_t)r * a.n_heads + h) * a.d_k + d) = O * (1.0f / L);
}

template <class T, int NB>
void launch_attn(const PageAttnArgs &a, hipStream_t s) {
    constexpr size_t lds = (size_t)(kWaves * 16 * (64 * NB + 4 + 2) + 4) * sizeof(float);
    if (a.d_k == 64 * NB) hipLaunchKernelGGL((page_attn_kernel<T, NB, true>), dim3(a.grid_items), dim3(64 * kWaves), lds, s, a);
    else hipLaunchKernelGGL((page_attn_kernel<T, NB, false>), dim3(a.grid_items), dim3(64 * kWaves), lds, s, a);
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
    if (a.combine > kFewPieces)
        hipLaunchKernelGGL((page_combine_kernel<LP, groups>), dim3(pairs), dim3(256), 0, s, a);
    else
        hipLaunchKernelGGL((page_combine_kernel<LP, 1>), dim3((pairs + groups - 1) / groups), dim3(256), 0, s, a);
    SLLM_HIP(hipGetLastError());
    return SLLM_OK;
}

}  // namespace

sllm_status launch_page_attention(const PageAttnArgs &a, hipStream_t s) {
    if (a.type == SLLM_CACHE_F16) return a.d_k <= 128 ? launch<_Float16, 32>(a, s) : launch<_Float16, 64>(a, s);
    return a.d_k <= 128 ? launch<float, 32>(a, s) : launch<float, 64>(a, s);
}

}  // namespace sllm
