// Low-rank adapters of many requests beside a shared projection:
//   dst[r] = y[r] + scale_a B_a (A_a x[r]),  a = ids[r]
// for the rows of a batch, each with its own adapter or none.
//
// Rows of one adapter are worked on together: 64 rows' ids fit one wave, which splits them into units of up to 16 rows
// with one adapter by ballots (no sort, no launch of its own, and rows in any order read each adapter once per unit).
// Two launches: `down` (t = A x, the columns split over workgroups and their waves) and `up` (adds the parts of t in
// order, dst = y + scale B t). Products are float32 matrix instructions (16 ranks or outputs x 16 rows x 4), exact in
// x for every type of adapter; a unit of a single row wastes 15 of their 16 columns and is bound by the loads all the
// same.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstring>
#include <memory>
#include <new>
#include <string>

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
    const void *a, *b;  // [slot][max_rank][cols], [slot][rows][stride], zeros behind an adapter's rank in b
    const Adapter *adapters;
    const int *ids;
    const float *x, *y;
    float *t, *dst;  // t: parts of A x, [split][x_rows][stride]
    int rows, cols, slots, max_rank, stride, x_rows, splits, chunks;
};

constexpr int kWaves = 4;
constexpr int kStep = 32;  // columns of a load: 128 bytes of x for every row

typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v4fu __attribute__((ext_vector_type(4), aligned(4)));  // rows of any length
typedef _Float16 v4h __attribute__((ext_vector_type(4)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef uint32_t v2u __attribute__((ext_vector_type(2)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float bf16_at(uint32_t w, int j) {
    return __builtin_bit_cast(float, j & 1 ? w & 0xffff0000u : w << 16);
}

// Eight columns of an adapter's A, four ranks of its B.
template <class T>
struct Eight {
    v4f v[2];
    __device__ __forceinline__ void load(const T *p) {
        v[0] = *(const v4f *)p;
        v[1] = *(const v4f *)(p + 4);
    }
    __device__ __forceinline__ float at(int j) const { return v[j >> 2][j & 3]; }
};
template <>
struct Eight<_Float16> {
    v8h v;
    __device__ __forceinline__ void load(const _Float16 *p) { v = *(const v8h *)p; }
    __device__ __forceinline__ float at(int j) const { return (float)v[j]; }
};
template <>
struct Eight<uint16_t> {  // bf16
    v4u v;
    __device__ __forceinline__ void load(const uint16_t *p) { v = *(const v4u *)p; }
    __device__ __forceinline__ float at(int j) const { return bf16_at(v[j >> 1], j); }
};

__device__ __forceinline__ v4f four(const float *p) { return *(const v4f *)p; }
__device__ __forceinline__ v4f four(const _Float16 *p) {
    const v4h h = *(const v4h *)p;
    return v4f{(float)h[0], (float)h[1], (float)h[2], (float)h[3]};
}
__device__ __forceinline__ v4f four(const uint16_t *p) {
    const v2u w = *(const v2u *)p;
    return v4f{bf16_at(w[0], 0), bf16_at(w[0], 1), bf16_at(w[1], 0), bf16_at(w[1], 1)};
}

// Up to 16 rows with one adapter (rank 0: with none).
struct Unit {
    int slot, rank, count, row;  // row: of lane % 16 (behind the count: the first one's)
    float scale;
};

// The ids of 64 rows, a lane each, and their adapters.
struct Rows64 {
    int id, rank;
    float scale;
    uint64_t in;

    __device__ __forceinline__ void load(const LoraArgs &g, int tile, int lane) {
        const int64_t r = (int64_t)tile * 64 + lane;
        in = __ballot(r < g.x_rows);
        id = g.ids[min(r, (int64_t)g.x_rows - 1)];
        const bool valid = id >= 0 && id < g.slots;
        const Adapter ad = g.adapters[valid ? id : 0];
        rank = valid ? ad.rank : 0;
        scale = ad.scale;
        if (rank == 0) id = -1;
    }

    // The u-th unit (in the order of the adapters' first rows); false: there is none.
    __device__ __forceinline__ bool unit(int tile, int lane, int u, Unit *out) const {
        uint64_t left = in;
        while (left) {
            const int first = __builtin_ctzll(left);
            out->slot = __builtin_amdgcn_readlane(id, first);
            const uint64_t same = __ballot(id == out->slot) & in;
            const int n = __builtin_popcountll(same);
            if (u * 16 < n) {
                const uint64_t below = (1ull << lane) - 1;
                const int at = __builtin_popcountll(same & below);
                const uint64_t mine = __ballot((same >> lane & 1) && at >> 4 == u);
                out->count = __builtin_popcountll(mine);
                out->rank = __builtin_amdgcn_readlane(rank, first);
                out->scale = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, scale), first));
                // every lane sends its number: the unit's to the front, in order
                const int to = mine >> lane & 1 ? __builtin_popcountll(mine & below)
                                                : out->count + __builtin_popcountll(~mine & below);
                const int lanes = __builtin_amdgcn_ds_permute(4 * to, lane);
                const int k = lane & 15;
                out->row = tile * 64 + __builtin_amdgcn_ds_bpermute(4 * (k < out->count ? k : 0), lanes);
                return true;
            }
            u -= (n + 15) / 16;
            left &= ~same;
        }
        return false;
    }
};

// Parts of t = A x of the units u, u + gridDim.y, ... of 64 rows: workgroup s takes every unit's s-th share of the
// columns, its waves a quarter of that, and adds them up. RB: tiles of 16 ranks at a time.
template <class T, int RB>
__global__ void __launch_bounds__(64 * kWaves, 2) lora_down_kernel(LoraArgs g) {
    constexpr int kAhead = 2;  // steps whose loads are under way
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), j16 = lane & 15, g4 = lane >> 4;
    const int tile = blockIdx.x / g.splits, s = blockIdx.x % g.splits;
    __shared__ v4f sums[kWaves][RB][64];
    Rows64 rows;
    rows.load(g, tile, lane);
    const int steps = g.cols / kStep, parts = g.splits * kWaves, part = s * kWaves + wave;
    const int from = (int)((int64_t)steps * part / parts), n = (int)((int64_t)steps * (part + 1) / parts) - from;
    Unit u;
    for (int at = blockIdx.y; rows.unit(tile, lane, at, &u); at += gridDim.y) {
        if (u.rank == 0) continue;
        const T *a = (const T *)g.a + (size_t)u.slot * g.max_rank * g.cols + 8 * g4;
        const float *x = g.x + (size_t)u.row * g.cols + 8 * g4;
        for (int k0 = 0; k0 < u.rank; k0 += 16 * RB) {
            int arow[RB];
#pragma unroll
            for (int t = 0; t < RB; t++) arow[t] = min(k0 + 16 * t + j16, u.rank - 1) * g.cols;
            v4f acc[RB] = {};
            Eight<T> av[kAhead][RB];
            Eight<float> xv[kAhead];
            auto load = [&](int b, int i) {
                const int c = (from + min(i, n - 1)) * kStep;
                xv[b].load(x + c);
#pragma unroll
                for (int t = 0; t < RB; t++) av[b][t].load(a + arow[t] + c);
            };
            if (n > 0) {
#pragma unroll
                for (int b = 0; b < kAhead; b++) load(b, b);
                for (int i = 0; i < n; i += kAhead) {
#pragma unroll
                    for (int b = 0; b < kAhead; b++) {
                        if (i + b < n) {
#pragma unroll
                            for (int j = 0; j < 8; j++)
#pragma unroll
                                for (int t = 0; t < RB; t++)
                                    acc[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(av[b][t].at(j), xv[b].at(j), acc[t], 0, 0, 0);
                        }
                        load(b, i + b + kAhead);
                    }
                }
            }
#pragma unroll
            for (int t = 0; t < RB; t++) sums[wave][t][lane] = acc[t];
            __syncthreads();
            // lane: its row's ranks 4 g4 .. + 3 of the tile
            for (int t = wave; t < RB; t += kWaves) {
                const int k = k0 + 16 * t + 4 * g4;
                v4f v = sums[0][t][lane];
#pragma unroll
                for (int w = 1; w < kWaves; w++) v += sums[w][t][lane];
                if (j16 < u.count && k < u.rank) *(v4f *)(g.t + ((size_t)s * g.x_rows + u.row) * g.stride + k) = v;
            }
            __syncthreads();
        }
    }
}

// dst = y + scale B t of the units of 64 rows; a wave: NT tiles of 16 outputs.
template <class T, int NT>
__global__ void __launch_bounds__(64 * kWaves, 2) lora_up_kernel(LoraArgs g) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), j16 = lane & 15, g4 = lane >> 4;
    const int tile = blockIdx.x / g.chunks, n0 = ((blockIdx.x % g.chunks) * kWaves + wave) * 16 * NT;
    extern __shared__ float tl[];  // [16][pitch]: the unit's scale t, zeros behind its rank
    const int pitch = ((g.max_rank + 15) & ~15) + 4;
    __shared__ int list[16];
    Rows64 rows;
    rows.load(g, tile, lane);
    Unit u;
    for (int at = blockIdx.y; rows.unit(tile, lane, at, &u); at += gridDim.y) {
        if (u.rank == 0 && g.dst == g.y) continue;
        const bool mine = j16 < u.count;
        const size_t row = (size_t)u.row * g.rows;
        v4f y[NT], acc[NT] = {};
#pragma unroll
        for (int t = 0; t < NT; t++) {
            const int n = n0 + 16 * t + 4 * g4;
            if (mine && n + 4 <= g.rows) {
                y[t] = *(const v4fu *)(g.y + row + n);
            } else {
                for (int j = 0; j < 4; j++) y[t][j] = mine && n + j < g.rows ? g.y[row + n + j] : 0.0f;
            }
        }
        if (u.rank > 0) {
            if (threadIdx.x < 16) list[lane] = u.row;
            __syncthreads();
            const int k16 = (u.rank + 15) / 16, groups = 4 * k16;
            for (int e = threadIdx.x; e < u.count * groups; e += 64 * kWaves) {
                const int r = e / groups, k = 4 * (e - r * groups);
                v4f v = {};
                if (k < u.rank) {
                    const float *p = g.t + (size_t)list[r] * g.stride + k;
                    const size_t split = (size_t)g.x_rows * g.stride;
#pragma unroll 8
                    for (int s = 0; s < g.splits; s++) v += *(const v4f *)(p + s * split);
                    v *= u.scale;
#pragma unroll
                    for (int j = 0; j < 4; j++) v[j] = k + j < u.rank ? v[j] : 0.0f;
                }
                *(v4f *)(tl + r * pitch + k) = v;
            }
            __syncthreads();
            const T *b = (const T *)g.b + (size_t)u.slot * g.rows * g.stride;
            for (int ks = 0; ks < k16; ks++) {
                const int k = 16 * ks + 4 * g4;
                v4f bv[NT];
#pragma unroll
                for (int t = 0; t < NT; t++)
                    bv[t] = k < g.stride ? four(b + (size_t)min(n0 + 16 * t + j16, g.rows - 1) * g.stride + k) : v4f{};
                const v4f tv = *(const v4f *)(tl + j16 * pitch + k);
#pragma unroll
                for (int j = 0; j < 4; j++)
#pragma unroll
                    for (int t = 0; t < NT; t++)
                        acc[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(bv[t][j], tv[j], acc[t], 0, 0, 0);
            }
            __syncthreads();  // before the next unit's t
        }
        // lane: its row's outputs 4 g4 .. + 3 of the tile
#pragma unroll
        for (int t = 0; t < NT; t++) {
            const int n = n0 + 16 * t + 4 * g4;
            const v4f v = u.rank > 0 ? y[t] + acc[t] : y[t];
            if (mine && n + 4 <= g.rows) {
                *(v4fu *)(g.dst + row + n) = v;
            } else {
                for (int j = 0; j < 4; j++)
                    if (mine && n + j < g.rows) g.dst[row + n + j] = v[j];
            }
        }
    }
}

// Workgroups of 64 rows' units: as many as there can be, or fewer that loop where most would find none.
struct Plan {
    int tiles, units, splits;
};

constexpr int kTarget = 1024;  // workgroups of `down`

Plan plan(const LoraArgs &g) {
    Plan p;
    p.tiles = (g.x_rows + 63) / 64;
    const int64_t rows = std::min(g.x_rows, 64);
    const int most = (int)std::min<int64_t>(rows, (rows + 15) / 16 + (int64_t)g.slots);
    p.units = std::min<int64_t>(most, std::max(8, kTarget / p.tiles));
    p.splits = std::max(1, std::min({kTarget / std::max(1, p.tiles * p.units), g.cols / kStep / kWaves, 16}));
    return p;
}

template <class T>
sllm_status launch(LoraArgs g, const Plan &p, hipStream_t s) {
    const dim3 down(p.tiles * p.splits, p.units), wg(64 * kWaves);
    if (g.max_rank <= 16) hipLaunchKernelGGL((lora_down_kernel<T, 1>), down, wg, 0, s, g);
    else if (g.max_rank <= 32) hipLaunchKernelGGL((lora_down_kernel<T, 2>), down, wg, 0, s, g);
    else hipLaunchKernelGGL((lora_down_kernel<T, 4>), down, wg, 0, s, g);
    SLLM_HIP(hipGetLastError());
    const int wide = kWaves * 16 * 4, lds = 16 * (((g.max_rank + 15) & ~15) + 4) * 4;
    const bool many = (int64_t)p.tiles * p.units * ((g.rows + wide - 1) / wide) >= 256;
    g.chunks = many ? (g.rows + wide - 1) / wide : (g.rows + wide / 4 - 1) / (wide / 4);
    const dim3 up(p.tiles * g.chunks, p.units);
    if (many) hipLaunchKernelGGL((lora_up_kernel<T, 4>), up, wg, lds, s, g);
    else hipLaunchKernelGGL((lora_up_kernel<T, 1>), up, wg, lds, s, g);
    SLLM_HIP(hipGetLastError());
    return SLLM_OK;
}

}  // namespace

}  // namespace sllm

struct sllm_lora_set {
    int rows = 0, cols = 0, slots = 0, max_rank = 0, type = 0, device = 0;
    char *a = nullptr, *b = nullptr;
    sllm::Adapter *adapters = nullptr;
    int stride() const { return (max_rank + 3) & ~3; }  // of B's rows, zeros behind an adapter's rank
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
    if (((int64_t)max_rank + 3) * (rows > cols ? rows : cols) * 4 >= ((int64_t)1 << 31))
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
    const size_t per = (size_t)max_adapters * w->stride() * w->elem();
    if ((double)per * (rows > cols ? rows : cols) > 1e15 ||
        hipMalloc(&w->a, (size_t)max_adapters * max_rank * w->elem() * cols) != hipSuccess ||
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
    // B with its rows at the set's stride (one copy: row by row, 4096 rows of 16 ranks took 40 ms)
    const size_t pitch = set->stride() * e, bytes = rank > 0 ? set->rows * pitch : 0;
    std::unique_ptr<char[]> packed(new (std::nothrow) char[bytes]);
    if (!packed) return set_error(SLLM_ERR_OOM, "out of memory");
    for (size_t r = 0; r * pitch < bytes; r++) {
        std::memcpy(packed.get() + r * pitch, (const char *)b + r * rank * e, rank * e);
        std::memset(packed.get() + r * pitch + rank * e, 0, pitch - rank * e);
    }
    // calls in flight on any stream may still read the slot
    SLLM_HIP(hipDeviceSynchronize());
    if (rank > 0) {
        SLLM_HIP(hipMemcpy(set->a + (size_t)slot * set->max_rank * set->cols * e, a, (size_t)rank * set->cols * e,
                           hipMemcpyHostToDevice));
        SLLM_HIP(hipMemcpy(set->b + (size_t)slot * bytes, packed.get(), bytes, hipMemcpyHostToDevice));
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
    g.stride = set->stride();
    g.x_rows = x_rows;
    const Plan p = plan(g);
    g.splits = p.splits;
    void *ws = nullptr;
    size_t cap = 0;
    hipStream_t s = (hipStream_t)stream;
    const sllm_status st = stream_workspace(s, (size_t)p.splits * x_rows * g.stride * sizeof(float), &ws, &cap);
    if (st != SLLM_OK) return st;
    g.t = (float *)ws;
    if (set->type == SLLM_LORA_F32) return launch<float>(g, p, s);
    if (set->type == SLLM_LORA_F16) return launch<_Float16>(g, p, s);
    return launch<uint16_t>(g, p, s);
}

}  // extern "C"
