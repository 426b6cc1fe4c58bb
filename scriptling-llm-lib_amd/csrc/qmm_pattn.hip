// The attention section (bias, QK norm, RoPE, append, causal GQA attention) of a batch of sequences
// over a page cache.
#include <hip/hip_runtime.h>

#include "qmm_device.hpp"
#include "qmm_pages.hpp"

namespace sllm {

namespace {

constexpr int kMaxDk = 256;
typedef float v4f __attribute__((ext_vector_type(4)));

template <class T>
__device__ __forceinline__ void put4(T *dst, v4f x);
template <>
__device__ __forceinline__ void put4<float>(float *dst, v4f x) {
    *(v4f *)dst = x;
}
template <>
__device__ __forceinline__ void put4<_Float16>(_Float16 *dst, v4f x) {
    typedef _Float16 v4h __attribute__((ext_vector_type(4)));
    *(v4h *)dst = v4h{(_Float16)x[0], (_Float16)x[1], (_Float16)x[2], (_Float16)x[3]};
}

// Bias (model_f32.go:398-420), per-head RMSNorm (:424-435), RoPE (applyRopeInPlaceF32,
// float32_ops.go:174-188) of every q and k head of a row, and the row's k and v into its page
// (the append, model_f32.go:445-448), rounded to the cache's type, once.
// One workgroup per row: the rotation (the same for every head: float32 angle, sine and cosine in 64
// bits, as the reference) once in LDS; then a wave per head, four dimensions a lane.
constexpr int kPrepWaves = 8;
template <class T>
__global__ void __launch_bounds__(64 * kPrepWaves) page_prep_kernel(PageAttnArgs a) {
    __shared__ float rc[kMaxDk / 2], rs[kMaxDk / 2];
    const int r = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (r >= a.step[0]) return;
    const StepRow row = a.rows[r];
    const int dk = a.d_k, d = 4 * lane;
    if ((int)threadIdx.x < a.half_dim) {
        const float ang = a.freqs[threadIdx.x] * (float)row.pos;
        double sd, cd;
        sincos((double)ang, &sd, &cd);
        rc[threadIdx.x] = (float)cd;
        rs[threadIdx.x] = (float)sd;
    }
    __syncthreads();
    const int page_rows = 1 << a.shift;
    for (int t = wave; t < a.n_heads + a.n_kv; t += kPrepWaves) {
        const bool isq = t < a.n_heads;
        const int h = isq ? t : t - a.n_heads;
        const int cols = (isq ? a.n_heads : a.n_kv) * dk;
        const size_t off = (size_t)r * cols + (size_t)h * dk + d;
        const float *bias = isq ? a.q_bias : a.k_bias, *nw = isq ? a.q_norm : a.k_norm;
        const int blen = isq ? a.qb_len : a.kb_len, j0 = h * dk + d;
        v4f x = {0.0f, 0.0f, 0.0f, 0.0f};
        if (d < dk) {
            x = *(const v4f *)((isq ? a.q : a.k) + off);
            if (bias)
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (j0 + i < blen) x[i] = x[i] + bias[j0 + i];
        }
        if (nw) {
            const float ss = wave_sum(((x[0] * x[0] + x[1] * x[1]) + x[2] * x[2]) + x[3] * x[3]);
            const float inv = 1.0f / (float)sqrt((double)ss / (double)dk + (double)a.eps);
            if (d < dk)
#pragma unroll
                for (int i = 0; i < 4; i++) x[i] = (x[i] * inv) * nw[d + i];
        }
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const int f = 2 * lane + i;
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

// out[h] = sum_p softmax_p(q_h . k_p / sqrt(d_k)) v_p over the positions 0 .. pos: a wave per (row, q
// head), one position after the other.
template <class T>
__global__ void __launch_bounds__(64) page_attn_kernel(PageAttnArgs a) {
    const int r = blockIdx.x, h = blockIdx.y, lane = threadIdx.x, dk = a.d_k, d = 4 * lane;
    if (r >= a.step[0]) return;
    const StepRow row = a.rows[r];
    const int g = h / a.rep, page_rows = 1 << a.shift;
    const size_t off = ((size_t)r * a.n_heads + h) * dk + d;
    v4f q = {0.0f, 0.0f, 0.0f, 0.0f}, o = q;
    if (d < dk) q = *(const v4f *)(a.qrot + off);
    float m = -INFINITY, l = 0.0f;
    for (int p = 0; p <= row.pos; p++) {
        const int page = a.tables[row.table + (p >> a.shift)];
        const size_t at = (((size_t)page * a.n_kv + g) * page_rows + (p & (page_rows - 1))) * dk + d;
        v4f k = {0.0f, 0.0f, 0.0f, 0.0f}, v = k;
        if (d < dk)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                k[i] = (float)((const T *)a.pool_k)[at + i];
                v[i] = (float)((const T *)a.pool_v)[at + i];
            }
        const float s = wave_sum(((q[0] * k[0] + q[1] * k[1]) + q[2] * k[2]) + q[3] * k[3]) * a.scale;
        const float mn = fmaxf(m, s), ref = mn == -INFINITY ? 0.0f : mn;
        const float alpha = expf(m - ref), e = expf(s - ref);
        l = l * alpha + e;
        o = o * alpha + v * e;
        m = mn;
    }
    if (d < dk) *(v4f *)(a.out + off) = o * (1.0f / l);
}

template <class T>
sllm_status launch(const PageAttnArgs &a, hipStream_t s) {
    hipLaunchKernelGGL(page_prep_kernel<T>, dim3(a.grid_rows), dim3(64 * kPrepWaves), 0, s, a);
    SLLM_HIP(hipGetLastError());
    hipLaunchKernelGGL(page_attn_kernel<T>, dim3(a.grid_rows, a.n_heads), dim3(64), 0, s, a);
    SLLM_HIP(hipGetLastError());
    return SLLM_OK;
}

}  // namespace

sllm_status launch_page_attention(const PageAttnArgs &a, hipStream_t s) {
    return a.type == SLLM_CACHE_F16 ? launch<_Float16>(a, s) : launch<float>(a, s);
}

}  // namespace sllm
