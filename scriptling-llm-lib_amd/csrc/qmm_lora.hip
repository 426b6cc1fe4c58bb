// Low-rank adapters of many requests beside a shared projection:
//   dst[r] = y[r] + scale_a B_a (A_a x[r]),  a = ids[r]
// for the rows of a batch, each with its own adapter or none.
#include <hip/hip_runtime.h>

#include <cstring>
#include <memory>
#include <new>
#include <string>
#include <vector>

#include "qmm_device.hpp"
#include "qmm_pages.hpp"

namespace sllm {

namespace {

// What the kernels read of one adapter; rank 0: none loaded.
struct Adapter {
    int rank = 0;
    float scale = 0.0f;
};

struct LoraArgs {
    const void *a, *b;  // [slot][max_rank][cols], [slot][rows][max_rank]
    const Adapter *adapters;
    const int *ids;
    const float *x, *y;
    float *t, *dst;  // t: the rows' scale A x (x_rows x max_rank)
    int rows, cols, slots, max_rank;
};

template <class T>
__device__ __forceinline__ float to_f32(T v) {
    return (float)v;
}
template <>
__device__ __forceinline__ float to_f32<uint16_t>(uint16_t v) {  // bf16
    return __builtin_bit_cast(float, (uint32_t)v << 16);
}

__device__ __forceinline__ Adapter adapter_of(const LoraArgs &g, int r, int *slot) {
    const int id = g.ids[r];
    *slot = id;
    return id >= 0 && id < g.slots ? g.adapters[id] : Adapter{};
}

// t[r][k] = scale A[k] . x[r]: a wave per (row, k).
template <class T>
__global__ void __launch_bounds__(64) lora_down_kernel(LoraArgs g) {
    const int r = blockIdx.x, k = blockIdx.y, lane = threadIdx.x;
    int slot;
    const Adapter ad = adapter_of(g, r, &slot);
    if (k >= ad.rank) return;
    const T *a = (const T *)g.a + ((size_t)slot * g.max_rank + k) * g.cols;
    const float *x = g.x + (size_t)r * g.cols;
    float s = 0.0f;
    for (int c = lane; c < g.cols; c += 64) s = __builtin_fmaf(to_f32<T>(a[c]), x[c], s);
    s = wave_sum(s);
    if (lane == 0) g.t[(size_t)r * g.max_rank + k] = s * ad.scale;
}

// dst[r][n] = y[r][n] + B[n] . t[r]: a thread per (row, n).
template <class T>
__global__ void __launch_bounds__(256) lora_up_kernel(LoraArgs g) {
    const int r = blockIdx.x;
    const int n = blockIdx.y * 256 + threadIdx.x;
    if (n >= g.rows) return;
    int slot;
    const Adapter ad = adapter_of(g, r, &slot);
    float s = 0.0f;
    if (ad.rank > 0) {
        const T *b = (const T *)g.b + ((size_t)slot * g.rows + n) * g.max_rank;
        for (int k = 0; k < ad.rank; k++) s = __builtin_fmaf(to_f32<T>(b[k]), g.t[(size_t)r * g.max_rank + k], s);
    }
    const size_t at = (size_t)r * g.rows + n;
    g.dst[at] = ad.rank > 0 ? g.y[at] + s : g.y[at];
}

template <class T>
sllm_status launch(const LoraArgs &g, int x_rows, hipStream_t s) {
    hipLaunchKernelGGL(lora_down_kernel<T>, dim3(x_rows, g.max_rank), dim3(64), 0, s, g);
    SLLM_HIP(hipGetLastError());
    hipLaunchKernelGGL(lora_up_kernel<T>, dim3(x_rows, (g.rows + 255) / 256), dim3(256), 0, s, g);
    SLLM_HIP(hipGetLastError());
    return SLLM_OK;
}

}  // namespace

}  // namespace sllm

struct sllm_lora_set {
    int rows = 0, cols = 0, slots = 0, max_rank = 0, type = 0, device = 0;
    char *a = nullptr, *b = nullptr;
    sllm::Adapter *adapters = nullptr;
    int elem() const { return type == SLLM_LORA_F32 ? 4 : 2; }
    ~sllm_lora_set() {
        (void)hipFree(a);
        (void)hipFree(b);
        (void)hipFree(adapters);
    }
};

using namespace sllm;

extern "C" {

sllm_status sllm_lora_set_create(int rows, int cols, int max_adapters, int max_rank, int type, sllm_lora_set **out) {
    if (!out) return set_error(SLLM_ERR_ARG, "null pointer");
    *out = nullptr;
    if (rows <= 0 || cols <= 0 || max_adapters <= 0 || max_rank <= 0)
        return set_error(SLLM_ERR_ARG, "adapter dimensions must be positive");
    if (cols % 32) return set_error(SLLM_ERR_SHAPE, "cols must be a multiple of 32");
    if (max_rank > 256) return set_error(SLLM_ERR_SHAPE, "max_rank must be at most 256");
    if (type != SLLM_LORA_F32 && type != SLLM_LORA_F16 && type != SLLM_LORA_BF16)
        return set_error(SLLM_ERR_ARG, "unknown adapter type");
    // one adapter's matrices: below 2 GiB each, so that the kernels' offsets in one fit 32 bits
    if ((int64_t)max_rank * (rows > cols ? rows : cols) * 4 >= ((int64_t)1 << 31))
        return set_error(SLLM_ERR_SHAPE, "max_rank x rows (cols) x 4 bytes must stay below 2 GiB");
    sllm_status st = library_init();
    if (st != SLLM_OK) return st;
    std::unique_ptr<sllm_lora_set> w(new (std::nothrow) sllm_lora_set());
    if (!w) return set_error(SLLM_ERR_OOM, "out of memory");
    w->rows = rows;
    w->cols = cols;
    w->slots = max_adapters;
    w->max_rank = max_rank;
    w->type = type;
    SLLM_HIP(hipGetDevice(&w->device));
    const size_t per = (size_t)max_adapters * max_rank * w->elem();
    if ((double)per * (rows > cols ? rows : cols) > 1e15 || hipMalloc(&w->a, per * cols) != hipSuccess ||
        hipMalloc(&w->b, per * rows) != hipSuccess ||
        hipMalloc(&w->adapters, (size_t)max_adapters * sizeof(Adapter)) != hipSuccess) {
        (void)hipGetLastError();
        return set_error(SLLM_ERR_OOM, "adapter allocation failed");
    }
    SLLM_HIP(hipMemsetAsync(w->adapters, 0, (size_t)max_adapters * sizeof(Adapter), nullptr));
    SLLM_HIP(hipStreamSynchronize(nullptr));
    *out = w.release();
    return SLLM_OK;
}

void sllm_lora_set_destroy(sllm_lora_set *set) { delete set; }

sllm_status sllm_lora_set_load(sllm_lora_set *set, int slot, int rank, const void *a, const void *b, float scale) {
    if (!set || (rank > 0 && (!a || !b))) return set_error(SLLM_ERR_ARG, "null pointer");
    if (slot < 0 || slot >= set->slots) return set_error(SLLM_ERR_ARG, "adapter slot out of range");
    if (rank < 0 || rank > set->max_rank) return set_error(SLLM_ERR_ARG, "rank outside 0 .. max_rank");
    int dev = 0;
    SLLM_HIP(hipGetDevice(&dev));
    if (dev != set->device) return set_error(SLLM_ERR_ARG, "the adapter set is another device's");
    const Adapter ad{rank, scale};
    const size_t e = (size_t)set->elem();
    // calls in flight on any stream may still read the slot
    SLLM_HIP(hipDeviceSynchronize());
    if (rank > 0) {
        SLLM_HIP(hipMemcpy(set->a + (size_t)slot * set->max_rank * set->cols * e, a, (size_t)rank * set->cols * e,
                           hipMemcpyHostToDevice));
        SLLM_HIP(hipMemcpy2D(set->b + (size_t)slot * set->rows * set->max_rank * e, set->max_rank * e, b, rank * e, rank * e,
                             (size_t)set->rows, hipMemcpyHostToDevice));
    }
    SLLM_HIP(hipMemcpy(set->adapters + slot, &ad, sizeof ad, hipMemcpyHostToDevice));
    return SLLM_OK;
}

sllm_status sllm_lora_add_dev(const sllm_lora_set *set, const float *x, int x_rows, const int *ids, const float *y,
                              float *dst, void *stream) {
    if (!set || !x || !ids || !y || !dst) return set_error(SLLM_ERR_ARG, "null pointer");
    if (x_rows <= 0) return set_error(SLLM_ERR_ARG, "xRows must be positive");
    if (((uintptr_t)x & 15) != 0) return set_error(SLLM_ERR_ARG, "x must be 16-byte aligned");
    int dev = 0;
    SLLM_HIP(hipGetDevice(&dev));
    if (dev != set->device) return set_error(SLLM_ERR_ARG, "the adapter set is another device's");
    LoraArgs g{};
    g.a = set->a;
    g.b = set->b;
    g.adapters = set->adapters;
    g.ids = ids;
    g.x = x;
    g.y = y;
    g.dst = dst;
    g.rows = set->rows;
    g.cols = set->cols;
    g.slots = set->slots;
    g.max_rank = set->max_rank;
    void *ws = nullptr;
    size_t cap = 0;
    hipStream_t s = (hipStream_t)stream;
    const sllm_status st = stream_workspace(s, (size_t)x_rows * set->max_rank * sizeof(float), &ws, &cap);
    if (st != SLLM_OK) return st;
    g.t = (float *)ws;
    if (set->type == SLLM_LORA_F32) return launch<float>(g, x_rows, s);
    if (set->type == SLLM_LORA_F16) return launch<_Float16>(g, x_rows, s);
    return launch<uint16_t>(g, x_rows, s);
}

}  // extern "C"
