// Low-rank adapters of many requests beside a shared projection:
//   dst[r] = y[r] + scale_a B_a (A_a x[r]),  a = ids[r]
// for the rows of a batch, each with its own adapter or none.
//
// Rows of one adapter are worked on together: 64 rows' ids fit one wave, which splits them into units of up to 16
// (prompts: 64) rows with one adapter (no sort, no launch of its own; rows in any order read an adapter once per unit).
// Two launches: `down` (t = A x, the columns split over workgroups and their waves) and `up` (adds the parts of t in
// order, dst = y + scale B t); prompts a third one between them that adds up more parts, small projections one
// launch for all. Products are float32 matrix instructions (16 ranks or outputs x 16 rows x 4), exact in
// x for every type of adapter; a unit of a single row wastes 15 of their 16 columns and is bound by the loads all the
// same.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstring>
#include <memory>
#include <new>
#include <string>
#include <type_traits>

#include "qmm_device.hpp"
#include "qmm_pages.hpp"

namespace sllm {

namespace {

// Where B[n][k] lies in its adapter: 64 outputs by 16 ranks together (fewer at the end of the stride), four operands of a
// matrix instruction (outputs 4 j + t, j < 16) whose lanes' four ranks follow each other, so that a load of `up` reads
// 512 or 1024 bytes in a row (as rows of B, 64 bytes of 16 rows: 17.6 us instead of 14.3 for 700 rows of rank 64, f32).
__host__ __device__ __forceinline__ int b_at(int n, int k, int stride) {
    const int k16 = k & ~15, groups = stride - k16 < 16 ? (stride - k16) / 4 : 4;
    return (n / 64 * stride + k16) * 64 + ((n % 4 * groups + (k - k16) / 4) * 16 + n % 64 / 4) * 4 + k % 4;
}

// What the kernels read of one adapter; rank 0: none loaded.
struct Adapter {
    int rank = 0;
    float scale = 0.0f;
};

struct LoraArgs {
    const void *a, *b;  // [slot][max_rank][cols]; [slot], as b_at has it, zeros behind an adapter's rank
    const Adapter *adapters;
    const int *ids;
    const float *x, *y;
    float *t, *dst;  // t: parts of A x, [split][x_rows][stride]
    int *groups;     // of every 64 rows: how many groups of 16 with one adapter, then their records
    int rows, cols, slots, max_rank, stride, x_rows, tiles, splits, chunks, most;
    int steps, more;  // every wave's steps of columns; the first `more` waves' have one more
};

constexpr int kWaves = 8;  // of a `down` workgroup
constexpr int kGroup = 4 + 16;  // ints of a group's record: slot, rank, count, scale, rows (behind the count: the first)
constexpr int kStep = 32;  // columns of a load: 128 bytes of x for every row

typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v4fu __attribute__((ext_vector_type(4), aligned(4)));  // rows of any length
typedef _Float16 v4h __attribute__((ext_vector_type(4)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef int v4i __attribute__((ext_vector_type(4)));
typedef uint32_t v2u __attribute__((ext_vector_type(2)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float bf16_at(uint32_t w, int j) {
    return __builtin_bit_cast(float, j & 1 ? w & 0xffff0000u : w << 16);
}

// Eight columns of an adapter's A, four ranks of its B.
template <class T>
struct Eight {
    v4f v[2];
    // lane / 16 = g4: its columns of a step (each instruction reads 64 bytes in a row)
    static constexpr int kLane = 4, kSecond = 16;
    __device__ __forceinline__ void load(const T *p, int second = kSecond) {
        v[0] = *(const v4f *)p;
        v[1] = *(const v4f *)(p + second);
    }
    __device__ __forceinline__ float at(int j) const { return v[j >> 2][j & 3]; }
};
template <>
struct Eight<_Float16> {
    v8h v;
    static constexpr int kLane = 8, kSecond = 4;
    __device__ __forceinline__ void load(const _Float16 *p) { v = *(const v8h *)p; }
    __device__ __forceinline__ float at(int j) const { return (float)v[j]; }
};
template <>
struct Eight<uint16_t> {  // bf16
    v4u v;
    static constexpr int kLane = 8, kSecond = 4;
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

// Up to 16 MT rows with one adapter (rank 0: with none).
struct Unit {
    int slot, rank, count;
    float scale;
    int tile, order;  // lane: the number of its row among the 64

    // Its k-th row (behind the count: the first one).
    __device__ __forceinline__ int row(int k) const {
        return tile * 64 + __builtin_amdgcn_ds_bpermute(4 * (k < count ? k : 0), order);
    }
};

// The ids of 64 rows, a lane each, their adapters, and the units of up to 16 MT rows with one adapter: in the order of
// their first rows, whatever the others are.
template <int MT>
struct Rows64 {
    int id, rank, nth;  // nth: of the rows with this id
    float scale;
    uint64_t in, first, first16;  // rows; those that begin a unit, a group of 16 of a unit

    __device__ __forceinline__ int load(const LoraArgs &g, int tile, int lane) {
        const int count = min(64, g.x_rows - tile * 64);
        in = count == 64 ? ~0ull : (1ull << count) - 1;
        id = g.ids[(int64_t)tile * 64 + min(lane, count - 1)];
        const bool valid = id >= 0 && id < g.slots;
        if (g.slots <= 64) {  // all of them, under way beside the ids
            const Adapter ad = g.adapters[min(lane, g.slots - 1)];
            rank = __builtin_amdgcn_ds_bpermute(4 * (valid ? id : 0), ad.rank);
            scale = __builtin_bit_cast(float, __builtin_amdgcn_ds_bpermute(4 * (valid ? id : 0), __builtin_bit_cast(int, ad.scale)));
        } else {
            const Adapter ad = g.adapters[valid ? id : 0];
            rank = ad.rank;
            scale = ad.scale;
        }
        if (!valid) rank = 0;
        if (rank == 0) id = -1;
        nth = 0;
        for (int j0 = 0; j0 < count; j0 += 8) {
#pragma unroll
            for (int j = j0; j < j0 + 8; j++) nth += __builtin_amdgcn_readlane(id, j) == id && j < lane ? 1 : 0;
        }
        first = __ballot(nth % (16 * MT) == 0) & in;
        first16 = __ballot(nth % 16 == 0) & in;
        return __builtin_popcountll(first);
    }

    // the u-th
    __device__ __forceinline__ void unit(int tile, int lane, int u, Unit *out) const {
        const uint64_t below = (1ull << lane) - 1;
        const int lead = __builtin_ctzll(__ballot((first >> lane & 1) && __builtin_popcountll(first & below) == u));
        out->slot = __builtin_amdgcn_readlane(id, lead);
        out->rank = __builtin_amdgcn_readlane(rank, lead);
        out->scale = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, scale), lead));
        const int group = __builtin_amdgcn_readlane(nth, lead) / (16 * MT);
        const uint64_t mine = __ballot(id == out->slot && nth / (16 * MT) == group) & in;
        out->count = __builtin_popcountll(mine);
        // every lane sends its number: the unit's to the front, in order
        const int to = mine >> lane & 1 ? __builtin_popcountll(mine & below)
                                        : out->count + __builtin_popcountll(~mine & below);
        out->order = __builtin_amdgcn_ds_permute(4 * to, lane);
        out->tile = tile;
    }

    // What `up` needs to know of the unit's groups; by one wave.
    __device__ __forceinline__ void record(const LoraArgs &g, int lane, const Unit &u) const {
        for (int k = 0; k < u.count; k += 16) {
            const int row = u.row(k + (lane & 15));
            const int lead = __builtin_amdgcn_readfirstlane(row) - u.tile * 64;
            const int nr = __builtin_popcountll(first16 & ((1ull << lead) - 1));
            int *rec = g.groups + ((g.tiles + 3) & ~3) + ((size_t)u.tile * g.most + nr) * kGroup;
            if (lane < 4) {
                const int count = min(16, u.count - k);
                rec[lane] = lane == 0 ? u.slot : lane == 1 ? u.rank : lane == 2 ? count : __builtin_bit_cast(int, u.scale);
            }
            if (lane < 16) rec[4 + lane] = row;
        }
    }
};

// A workgroup's share of `parts` x `tiles`: every XCD (workgroups b, b + 8, ...) takes parts of its own for all tiles,
// so that one L2 holds what they read of the adapters. False: none (the grid is a multiple of 8).
__device__ __forceinline__ bool share(int parts, int tiles, int *tile, int *part) {
    const int at = (blockIdx.x % 8) * (gridDim.x / 8) + blockIdx.x / 8;
    *part = at / tiles;
    *tile = at % tiles;
    return *part < parts;
}

// acc += A x over n steps of the columns; x, a: the lane's row of either operand (arow: of A's tiles).
template <class T, int RB>
__device__ __forceinline__ void columns(const float *x, const T *a, const int (&arow)[RB], int from, int n, v4f (&acc)[RB]) {
    // some steps, their loads under way together
    auto steps = [&](auto count, int i) {
        constexpr int D = decltype(count)::value;
        Eight<T> av[D][RB];
        Eight<float> xv[D];
#pragma unroll
        for (int d = 0; d < D; d++) {
            const int c = (from + i + d) * kStep;
            xv[d].load(x + c, Eight<T>::kSecond);
#pragma unroll
            for (int t = 0; t < RB; t++) av[d][t].load(a + arow[t] + c);
        }
#pragma unroll
        for (int d = 0; d < D; d++)
#pragma unroll
            for (int j = 0; j < 8; j++)
#pragma unroll
                for (int t = 0; t < RB; t++)
                    acc[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(av[d][t].at(j), xv[d].at(j), acc[t], 0, 0, 0);
    };
    int i = 0;
    for (; i + 4 <= n; i += 4) steps(std::integral_constant<int, 4>(), i);
    if (i + 2 <= n) {
        steps(std::integral_constant<int, 2>(), i);
        i += 2;
    }
    if (i < n) steps(std::integral_constant<int, 1>(), i);
}

// Parts of t = A x of the units u, u + gridDim.y, ... of up to 16 of 64 rows: workgroup s takes every unit's s-th share
// of the columns, its waves parts of that, and adds them up. RB: tiles of 16 ranks at a time.
template <class T, int RB>
__global__ void __launch_bounds__(64 * kWaves, 2) lora_down_kernel(LoraArgs g) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), j16 = lane & 15, g4 = lane >> 4;
    int tile, s;
    if (!share(g.splits, g.tiles, &tile, &s)) return;
    __shared__ v4f sums[kWaves][RB][64];
    Rows64<1> rows;
    const int units = rows.load(g, tile, lane);
    if (s == 0 && blockIdx.y == 0 && threadIdx.x == 0) g.groups[tile] = units;
    const int part = s * kWaves + wave, from = part * g.steps + min(part, g.more), n = g.steps + (part < g.more ? 1 : 0);
    for (int at = blockIdx.y; at < units; at += gridDim.y) {
        Unit u;
        rows.unit(tile, lane, at, &u);
        if (s == 0 && wave == 0) rows.record(g, lane, u);
        if (u.rank == 0) continue;
        constexpr int kLane = Eight<T>::kLane;
        const int row = u.row(j16);
        const T *a = (const T *)g.a + (size_t)u.slot * g.max_rank * g.cols + kLane * g4;
        const float *x = g.x + (size_t)row * g.cols + kLane * g4;
        for (int k0 = 0; k0 < u.rank; k0 += 16 * RB) {
            int arow[RB];
#pragma unroll
            for (int t = 0; t < RB; t++) arow[t] = min(k0 + 16 * t + j16, u.rank - 1) * g.cols;
            v4f acc[RB] = {};
            columns<T, RB>(x, a, arow, from, n, acc);
            // lane: its row's ranks 4 g4 .. + 3 of the tile
#pragma unroll
            for (int t = 0; t < RB; t++) sums[wave][t][lane] = acc[t];
            __syncthreads();
            for (int t = wave; t < RB; t += kWaves) {
                const int k = k0 + 16 * t + 4 * g4;
                v4f v = sums[0][t][lane];
#pragma unroll
                for (int w = 1; w < kWaves; w++) v += sums[w][t][lane];
                if (j16 < u.count && k < u.rank) *(v4f *)(g.t + ((size_t)s * g.x_rows + row) * g.stride + k) = v;
            }
            __syncthreads();
        }
    }
}

// Reads of LDS and the wait for them in one block: the compiler, which cannot tell the two stages of a ring apart, would
// wait for all loads into LDS before any read of it.
__device__ __forceinline__ void lds_read(v4u (&d)[8], unsigned a0, unsigned a1) {  // every 2048 bytes (rows of 128)
    asm volatile("ds_read_b128 %0, %8\n\tds_read_b128 %1, %9\n\tds_read_b128 %2, %8 offset:2048\n\t"
                 "ds_read_b128 %3, %9 offset:2048\n\tds_read_b128 %4, %8 offset:4096\n\tds_read_b128 %5, %9 offset:4096\n\t"
                 "ds_read_b128 %6, %8 offset:6144\n\tds_read_b128 %7, %9 offset:6144\n\ts_waitcnt lgkmcnt(0)"
                 : "=&v"(d[0]), "=&v"(d[1]), "=&v"(d[2]), "=&v"(d[3]), "=&v"(d[4]), "=&v"(d[5]), "=&v"(d[6]), "=&v"(d[7])
                 : "v"(a0), "v"(a1)
                 : "memory");
}
__device__ __forceinline__ void lds_read(v4u (&d)[4], unsigned a0, unsigned a1) {
    asm volatile("ds_read_b128 %0, %4\n\tds_read_b128 %1, %5\n\tds_read_b128 %2, %4 offset:2048\n\t"
                 "ds_read_b128 %3, %5 offset:2048\n\ts_waitcnt lgkmcnt(0)"
                 : "=&v"(d[0]), "=&v"(d[1]), "=&v"(d[2]), "=&v"(d[3])
                 : "v"(a0), "v"(a1)
                 : "memory");
}
__device__ __forceinline__ void lds_read(v4u (&d)[2], unsigned a0, unsigned a1) {
    asm volatile("ds_read_b128 %0, %2\n\tds_read_b128 %1, %3\n\ts_waitcnt lgkmcnt(0)"
                 : "=&v"(d[0]), "=&v"(d[1])
                 : "v"(a0), "v"(a1)
                 : "memory");
}
__device__ __forceinline__ void lds_read(v4u (&d)[4], unsigned a0) {  // every 1024 bytes (rows of 64)
    asm volatile("ds_read_b128 %0, %4\n\tds_read_b128 %1, %4 offset:1024\n\tds_read_b128 %2, %5\n\t"
                 "ds_read_b128 %3, %5 offset:1024\n\ts_waitcnt lgkmcnt(0)"
                 : "=&v"(d[0]), "=&v"(d[1]), "=&v"(d[2]), "=&v"(d[3])
                 : "v"(a0), "v"(a0 + 2048)
                 : "memory");
}
__device__ __forceinline__ void lds_read(v4u (&d)[2], unsigned a0) {
    asm volatile("ds_read_b128 %0, %2\n\tds_read_b128 %1, %2 offset:1024\n\ts_waitcnt lgkmcnt(0)"
                 : "=&v"(d[0]), "=&v"(d[1])
                 : "v"(a0)
                 : "memory");
}
__device__ __forceinline__ void lds_read(v4u (&d)[1], unsigned a0) {
    asm volatile("ds_read_b128 %0, %1\n\ts_waitcnt lgkmcnt(0)" : "=&v"(d[0]) : "v"(a0) : "memory");
}

typedef const __attribute__((address_space(1))) void *GlobalPtr;
typedef __attribute__((address_space(3))) void *LdsPtr;

// LDS of the kernel below for one wave's step: 64 rows of x, 16 RB of A.
template <class T, int RB>
constexpr int stage_bytes() {
    return (64 * 4 + 16 * RB * (int)sizeof(T)) * kStep;
}

// The same of units of up to 64 rows of a prompt: 16 bytes of x or A then bring 4 .. 16 matrix instructions, and read
// straight into their operands (16 rows x 64 bytes an instruction) they were what bounded them (700 rows, 14336 columns,
// rank 64, f32: 41 us). So every wave brings whole lines into two stages of LDS of its own, one on its way while the
// other is used; a row's pieces of 16 bytes are kept in an order (exclusive or with the row) that lets 16 rows' be
// read without conflicts. A workgroup takes the units of its 64 rows one after the other: made for prompts, whose 64 rows
// have one or two (4096 x 4096, rank 16, f16, 256 rows: 16.5 us on 8 adapters in order, 23 in any order; on 32 in any
// order 58, four calls of 64 rows 43).
template <class T, int RB>
__global__ void __launch_bounds__(256, 1) lora_down_rows_kernel(LoraArgs g) {
    constexpr int XB = 64 * 4 * kStep, stage = stage_bytes<T, RB>();
    constexpr int AL = kStep * (int)sizeof(T) / 16;   // pieces of a row of A: 8 or 4
    constexpr int AN = 16 * RB * AL / 64, NL = 8 + AN;  // loads of a step: of A, of both
    extern __shared__ v4f lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), j16 = lane & 15, g4 = lane >> 4;
    int tile, s;
    if (!share(g.splits, g.tiles, &tile, &s)) return;
    char *ring = (char *)lds + wave * 2 * stage;
    const unsigned ring_at = (unsigned)(uintptr_t)(LdsPtr)ring;
    // operands in a stage: lane j16, g4 takes a row's columns as Eight has them
    const unsigned px = j16 * 128 + ((AL == 8 ? g4 : 2 * g4) ^ (j16 >> 1)) * 16;
    const unsigned px2 = j16 * 128 + ((AL == 8 ? 4 + g4 : 2 * g4 + 1) ^ (j16 >> 1)) * 16;
    const unsigned pa = XB + j16 * 64 + (g4 ^ (j16 >> 2)) * 16;  // (AL == 8: as x)
    Rows64<4> rows;
    const int units = rows.load(g, tile, lane);
    if (s == 0 && threadIdx.x == 0) g.groups[tile] = __builtin_popcountll(rows.first16);
    const int part = s * 4 + wave, from = part * g.steps + min(part, g.more), n = g.steps + (part < g.more ? 1 : 0);
    for (int at = 0; at < units; at++) {
        Unit u;
        rows.unit(tile, lane, at, &u);
        if (s == 0 && wave == 0) rows.record(g, lane, u);
        if (u.rank == 0) continue;
        const float *x[8];
#pragma unroll
        for (int q = 0; q < 8; q++)
            x[q] = g.x + (size_t)u.row(8 * q + (lane >> 3)) * g.cols + (size_t)from * kStep + ((lane & 7) ^ ((4 * q + g4) & 7)) * 4;
        const T *a = (const T *)g.a + (size_t)u.slot * g.max_rank * g.cols + (size_t)from * kStep;
        int out[4];
#pragma unroll
        for (int m = 0; m < 4; m++) out[m] = u.row(16 * m + j16);
        for (int k0 = 0; k0 < u.rank; k0 += 16 * RB) {
            int arow[AN];
#pragma unroll
            for (int q = 0; q < AN; q++) {
                const int r = AL == 8 ? 8 * q + (lane >> 3) : 16 * q + (lane >> 2);
                const int piece = AL == 8 ? (lane & 7) ^ ((4 * q + g4) & 7) : (lane & 3) ^ g4;
                arow[q] = min(k0 + r, u.rank - 1) * g.cols + piece * (16 / (int)sizeof(T));
            }
            auto fill = [&](int i) {
                char *to = ring + (i & 1) * stage;
#pragma unroll
                for (int q = 0; q < 8; q++)
                    __builtin_amdgcn_global_load_lds((GlobalPtr)(x[q] + i * kStep), (LdsPtr)(to + q * 1024), 16, 0, 0);
#pragma unroll
                for (int q = 0; q < AN; q++)
                    __builtin_amdgcn_global_load_lds((GlobalPtr)(a + arow[q] + i * kStep), (LdsPtr)(to + XB + q * 1024), 16, 0, 0);
            };
            v4f acc[4][RB] = {};
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // earlier loads and stores don't count below
            if (n > 0) fill(0);
            if (n > 1) fill(1);
            for (int i = 0; i < n; i++) {
                if (i + 1 < n) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(NL) : "memory");
                else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                const unsigned st = ring_at + (i & 1) * stage;
                v4u xr[8], ar[AL == 8 ? 2 * RB : RB];
                lds_read(xr, st + px, st + px2);
                if constexpr (AL == 8) lds_read(ar, st + XB + px, st + XB + px2);
                else lds_read(ar, st + pa);
                if (i + 2 < n) fill(i + 2);
                auto av = [&](int t, int j) {
                    if constexpr (AL == 8) return __builtin_bit_cast(v4f, ar[2 * t + (j >> 2)])[j & 3];
                    else if constexpr (std::is_same_v<T, _Float16>) return (float)__builtin_bit_cast(v8h, ar[t])[j];
                    else return bf16_at(ar[t][j >> 1], j);
                };
                float af[RB][8];
#pragma unroll
                for (int t = 0; t < RB; t++)
#pragma unroll
                    for (int j = 0; j < 8; j++) af[t][j] = av(t, j);
#pragma unroll
                for (int m = 0; m < 4; m++)
                    if (16 * m < u.count) {
#pragma unroll
                        for (int j = 0; j < 8; j++)
#pragma unroll
                            for (int t = 0; t < RB; t++)
                                acc[m][t] = __builtin_amdgcn_mfma_f32_16x16x4f32(
                                    af[t][j], __builtin_bit_cast(v4f, xr[2 * m + (j >> 2)])[j & 3], acc[m][t], 0, 0, 0);
                    }
            }
            // the waves' sums, in stages that none reads or fills any more; lane: its row's ranks 4 g4 .. + 3 of the tile
            v4f *own = (v4f *)ring;
#pragma unroll
            for (int m = 0; m < 4; m++)
#pragma unroll
                for (int t = 0; t < RB; t++) own[(m * RB + t) * 64 + lane] = acc[m][t];
            __syncthreads();
#pragma unroll
            for (int t = 0; t < RB; t++) {
                const int k = k0 + 16 * t + 4 * g4, m = wave;
                v4f v = lds[(m * RB + t) * 64 + lane];
#pragma unroll
                for (int w = 1; w < 4; w++) v += lds[w * 2 * stage / 16 + (m * RB + t) * 64 + lane];
                const int row = m == 0 ? out[0] : m == 1 ? out[1] : m == 2 ? out[2] : out[3];
                if (16 * m + j16 < u.count && k < u.rank) *(v4f *)(g.t + ((size_t)s * g.x_rows + row) * g.stride + k) = v;
            }
            __syncthreads();
        }
    }
}

// Small projections: both products in one launch. A workgroup takes 128 outputs of a unit, 16 a wave, and forms all of
// the unit's t for itself: the waves' shares of the columns meet in LDS as the second product's operands. y and B are on their way
// beside A. Bound by latency (one row, 576 x 576, rank 8, f16: 4.6 us, in two launches 8.1).
template <class T, int RB>
__global__ void __launch_bounds__(64 * kWaves) lora_small_kernel(LoraArgs g) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), j16 = lane & 15, g4 = lane >> 4;
    __shared__ v4f sums[kWaves][RB][64];
    Rows64<1> rows;
    const int units = rows.load(g, 0, lane);
    const int from = wave * g.steps + min(wave, g.more), n = g.steps + (wave < g.more ? 1 : 0);
    // lane: output n of the rows 4 g4 .. + 3 (behind the rows: the last one's, not stored)
    const int out = (blockIdx.x * kWaves + wave) * 16 + j16, nb = min(out, g.rows - 1);
    for (int at = blockIdx.y; at < units; at += gridDim.y) {
        Unit u;
        rows.unit(0, lane, at, &u);
        if (u.rank == 0 && g.dst == g.y) continue;
        size_t to[4];
        float y[4];
#pragma unroll
        for (int r = 0; r < 4; r++) {
            to[r] = (size_t)u.row(4 * g4 + r) * g.rows + nb;
            y[r] = g.y[to[r]];
        }
        if (u.rank > 0) {
            constexpr int kLane = Eight<T>::kLane;
            const int rows64 = (g.rows + 63) & ~63;
            const T *b = (const T *)g.b + (size_t)u.slot * rows64 * g.stride;
            v4f bv[RB], acc[RB] = {};
            int arow[RB];
#pragma unroll
            for (int t = 0; t < RB; t++) {
                bv[t] = four(b + b_at(nb, min(16 * t + 4 * g4, g.stride - 4), g.stride));
                arow[t] = min(16 * t + j16, u.rank - 1) * g.cols;
            }
            columns<T, RB>(g.x + (size_t)u.row(j16) * g.cols + kLane * g4,
                           (const T *)g.a + (size_t)u.slot * g.max_rank * g.cols + kLane * g4, arow, from, n, acc);
#pragma unroll
            for (int t = 0; t < RB; t++) sums[wave][t][lane] = acc[t];
            __syncthreads();
            v4f d = {};
#pragma unroll
            for (int t = 0; t < RB; t++) {
                // lane: its row's ranks k .. + 3, as the product takes them
                v4f tv = sums[0][t][lane];
#pragma unroll
                for (int w = 1; w < kWaves; w++) tv += sums[w][t][lane];
                const int k = 16 * t + 4 * g4;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const bool in = k + j < u.rank;
                    d = __builtin_amdgcn_mfma_f32_16x16x4f32(in ? tv[j] * u.scale : 0.0f, in ? bv[t][j] : 0.0f, d, 0, 0, 0);
                }
            }
#pragma unroll
            for (int r = 0; r < 4; r++) y[r] += d[r];
            __syncthreads();  // before the next unit's sums
        }
#pragma unroll
        for (int r = 0; r < 4; r++)
            if (4 * g4 + r < u.count && out < g.rows) g.dst[to[r]] = y[r];
    }
}

// The parts of t, added up into the first one. Bound by latency: a wave a workgroup, 16 parts' loads under way.
__global__ void __launch_bounds__(64) lora_sum_kernel(float *t, int64_t n4, int splits) {
    const int64_t i = (int64_t)blockIdx.x * 64 + threadIdx.x;
    if (i >= n4) return;
    v4f *p = (v4f *)t + i;
    v4f v = {};
    int s = 0;
    for (; s + 16 <= splits; s += 16) {
        v4f x[16];
#pragma unroll
        for (int j = 0; j < 16; j++) x[j] = p[(s + j) * n4];
#pragma unroll
        for (int j = 0; j < 16; j++) v += x[j];
    }
    if (s < splits) {
        v4f x[16];
#pragma unroll
        for (int j = 0; j < 16; j++) x[j] = p[min(s + j, splits - 1) * n4];
#pragma unroll
        for (int j = 0; j < 16; j++)
            if (s + j < splits) v += x[j];
    }
    *p = v;
}

// dst = y + scale B t of the groups that `down` recorded; a wave: NT tiles of 16 outputs. PARTS: of t.
template <class T, int NT, int PARTS>
__global__ void __launch_bounds__(256, 2) lora_up_kernel(LoraArgs g) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), j16 = lane & 15, g4 = lane >> 4;
    int tile, chunk;
    if (!share(g.chunks, g.tiles, &tile, &chunk)) return;
    const int n0 = (chunk * 4 + wave) * 16 * NT, groups = g.groups[tile];
    const bool whole = n0 + 16 * NT <= g.rows;
    for (int at = blockIdx.y; at < groups; at += gridDim.y) {
        const int *rec = g.groups + ((g.tiles + 3) & ~3) + ((size_t)tile * g.most + at) * kGroup;
        const int slot = rec[0], rank = rec[1], count = rec[2];
        const float scale = __builtin_bit_cast(float, rec[3]);
        if (rank == 0 && g.dst == g.y) continue;
        // lane: NT outputs in a row, n0 + NT j16 .., of the rows 4 g4 .. + 3 (NT 4: whole lines of four rows at a time)
        const v4i r4 = *(const v4i *)(rec + 4 + 4 * g4);
        const int n = n0 + NT * j16;
        float y[4][NT];
        v4f acc[NT] = {};
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const float *p = g.y + (size_t)r4[r] * g.rows;
            if (whole) {
                if constexpr (NT == 4) *(v4f *)y[r] = *(const v4fu *)(p + n);
                else y[r][0] = p[n];
            } else {
#pragma unroll
                for (int t = 0; t < NT; t++) y[r][t] = p[min(n + t, g.rows - 1)];
            }
        }
        if (rank > 0) {
            const int rows64 = (g.rows + 63) & ~63, nb = min(n, rows64 - 64 + n % 64);  // (behind the rows: not stored)
            const T *b = (const T *)g.b + (size_t)slot * rows64 * g.stride;
            const size_t split = (size_t)g.x_rows * g.stride;
            const float *tp = g.t + (size_t)rec[4 + j16] * g.stride;
            // (every load is in range and without a branch; what lies behind the rank is taken as zero)
            v4f bv[2][NT], tv[2];
            auto load = [&](int i, int k16) {
                const int k = min(k16 + 4 * g4, g.stride - 4);
#pragma unroll
                for (int t = 0; t < NT; t++) bv[i][t] = four(b + b_at(nb + t, k, g.stride));
                v4f part[PARTS];
#pragma unroll
                for (int s = 0; s < PARTS; s++) part[s] = *(const v4f *)(tp + s * split + k);
                tv[i] = part[0];
#pragma unroll
                for (int s = 1; s < PARTS; s++) tv[i] += part[s];
            };
            auto product = [&](int i, int k16) {
                const int k = k16 + 4 * g4;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const float tj = k + j < rank ? tv[i][j] * scale : 0.0f;
#pragma unroll
                    for (int t = 0; t < NT; t++) {
                        const float bj = k + j < rank ? bv[i][t][j] : 0.0f;
                        acc[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(tj, bj, acc[t], 0, 0, 0);
                    }
                }
            };
            load(0, 0);
            for (int k = 0; k < rank; k += 32) {
                load(1, k + 16);
                product(0, k);
                if (k + 16 < rank) {
                    load(0, k + 32);
                    product(1, k + 16);
                }
            }
#pragma unroll
            for (int r = 0; r < 4; r++)
#pragma unroll
                for (int t = 0; t < NT; t++) y[r][t] += acc[t][r];
        }
#pragma unroll
        for (int r = 0; r < 4; r++) {
            float *p = g.dst + (size_t)r4[r] * g.rows;
            if (4 * g4 + r < count) {
                if (whole) {
                    if constexpr (NT == 4) *(v4fu *)(p + n) = *(v4f *)y[r];
                    else p[n] = y[r][0];
                } else {
#pragma unroll
                    for (int t = 0; t < NT; t++)
                        if (n + t < g.rows) p[n + t] = y[r][t];
                }
            }
        }
    }
}

// Groups of 16 rows with one adapter that 64 rows can have, splits of the columns, and the tiles of 16 rows in a unit.
struct Plan {
    int tiles, most, splits, mt, waves;
};

constexpr int kCUs = 256;
constexpr int kParts = 8, kManyParts = 32;  // of t; `up` adds 8 up

int eights(int n) { return (n + 7) / 8 * 8; }

Plan plan(const LoraArgs &g) {
    Plan p;
    p.mt = g.x_rows > 64 ? 4 : 1;
    p.tiles = (g.x_rows - 1) / 64 + 1;
    const int64_t rows = std::min(g.x_rows, 64);
    p.most = (int)std::min<int64_t>(rows, (rows + 15) / 16 + (int64_t)g.slots);
    p.waves = p.mt == 1 ? kWaves : 4;  // of a `down` workgroup
    const int fit = std::max(1, g.cols / kStep / p.waves);
    // Few units of many rows: more parts, added up by a launch of their own (64 rows, one adapter, 14336 columns, rank 64,
    // f32: 20.6 us in 8 parts, 9.4 in 32; as many added up by `up` cost it 14 us, the launch 3).
    if (p.mt == 1) p.splits = g.x_rows > 16 && p.most <= 8 && g.cols / kStep >= kManyParts * kWaves ? kManyParts : kParts;
    else p.splits = std::max(1, std::min({kCUs / p.tiles, fit, 32}));  // a workgroup for every CU
    return p;
}

// Both products in one launch: as long as few columns make every workgroup's own t cheap (its columns are a few steps of
// eight waves) and all of them together read little of the adapters from the caches (2048 x 2048, rank 16, f16, us: one
// row 6.6, in two launches 4.0 + 3.6; 32 rows on 8 adapters 8.3, 4.5 + 4.3).
bool small(const LoraArgs &g, const Plan &p, int elem) {
    return p.mt == 1 && g.max_rank <= 64 && g.cols <= 2048 &&
           (int64_t)p.most * ((g.rows + 127) / 128) * g.max_rank * g.cols * elem <= (32 << 20);
}

template <class T>
sllm_status launch_small(LoraArgs g, const Plan &p, hipStream_t s) {
    g.steps = g.cols / kStep / kWaves;
    g.more = g.cols / kStep % kWaves;
    const dim3 grid((g.rows + 16 * kWaves - 1) / (16 * kWaves), p.most), wg(64 * kWaves);
    if (g.max_rank <= 16) hipLaunchKernelGGL((lora_small_kernel<T, 1>), grid, wg, 0, s, g);
    else if (g.max_rank <= 32) hipLaunchKernelGGL((lora_small_kernel<T, 2>), grid, wg, 0, s, g);
    else hipLaunchKernelGGL((lora_small_kernel<T, 4>), grid, wg, 0, s, g);
    SLLM_HIP(hipGetLastError());
    return SLLM_OK;
}

template <class T, int MT>
sllm_status launch_rows(LoraArgs g, const Plan &p, hipStream_t s) {
    // A workgroup for every unit there can be, or (prompts) one for all of 64 rows: they come together, so that 64 have
    // little more than one unit, and two of 32 rows take no more products than one of 64. (Workgroups that may find
    // nothing cost more than that: 700 rows of 3 adapters, f32, rank 64, in an earlier form of the kernel, us: 49 with
    // four for 64 rows, 41 with one.)
    const int grid = eights(p.tiles * p.splits);
    if constexpr (MT == 1) {
        const dim3 down(grid, p.most), wg(64 * kWaves);
        if (g.max_rank <= 16) hipLaunchKernelGGL((lora_down_kernel<T, 1>), down, wg, 0, s, g);
        else if (g.max_rank <= 32) hipLaunchKernelGGL((lora_down_kernel<T, 2>), down, wg, 0, s, g);
        else hipLaunchKernelGGL((lora_down_kernel<T, 4>), down, wg, 0, s, g);
    } else {
        const dim3 down(grid), wg(256);
        if (g.max_rank <= 16) hipLaunchKernelGGL((lora_down_rows_kernel<T, 1>), down, wg, (8 * stage_bytes<T, 1>()), s, g);
        else if (g.max_rank <= 32) hipLaunchKernelGGL((lora_down_rows_kernel<T, 2>), down, wg, (8 * stage_bytes<T, 2>()), s, g);
        else hipLaunchKernelGGL((lora_down_rows_kernel<T, 4>), down, wg, (8 * stage_bytes<T, 4>()), s, g);
    }
    SLLM_HIP(hipGetLastError());
    if (g.splits > 1 && g.splits != (MT == 1 ? kParts : 1)) {
        const int64_t n4 = (int64_t)g.x_rows * g.stride / 4;
        hipLaunchKernelGGL(lora_sum_kernel, dim3((unsigned)((n4 + 63) / 64)), dim3(64), 0, s, g.t, n4, g.splits);
        SLLM_HIP(hipGetLastError());
    }
    constexpr int wide = 4 * 16 * 4, narrow = wide / 4;
    const int groups = MT == 1 ? p.most : std::min(p.most, 8);  // (that case in all, us: 46.9 with 2, 43.9 with 4, 43.0)
    const bool many = (int64_t)p.tiles * groups * ((g.rows + wide - 1) / wide) >= kCUs;
    g.chunks = many ? (g.rows + wide - 1) / wide : (g.rows + narrow - 1) / narrow;
    const dim3 up(eights(p.tiles * g.chunks), groups);
    auto run = [&](auto parts) {
        constexpr int P = decltype(parts)::value;
        if (many) hipLaunchKernelGGL((lora_up_kernel<T, 4, P>), up, dim3(256), 0, s, g);
        else hipLaunchKernelGGL((lora_up_kernel<T, 1, P>), up, dim3(256), 0, s, g);
    };
    if (MT == 1 && p.splits == kParts) run(std::integral_constant<int, kParts>());
    else run(std::integral_constant<int, 1>());
    SLLM_HIP(hipGetLastError());
    return SLLM_OK;
}

template <class T>
sllm_status launch(const LoraArgs &g, const Plan &p, hipStream_t s) {
    if (small(g, p, sizeof(T))) return launch_small<T>(g, p, s);
    return p.mt > 1 ? launch_rows<T, 4>(g, p, s) : launch_rows<T, 1>(g, p, s);
}

}  // namespace

}  // namespace sllm

struct sllm_lora_set {
    int rows = 0, cols = 0, slots = 0, max_rank = 0, type = 0, device = 0;
    char *a = nullptr, *b = nullptr;
    sllm::Adapter *adapters = nullptr;
    int stride() const { return (max_rank + 3) & ~3; }  // of t's and B's rows
    int rows64() const { return (rows + 63) & ~63; }
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
    if (((int64_t)max_rank + 3) * ((int64_t)(rows > cols ? rows : cols) + 63) * 4 >= ((int64_t)1 << 31))
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
        hipMalloc(&w->b, per * w->rows64()) != hipSuccess ||
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
    const int stride = set->stride();
    const size_t bytes = rank > 0 ? (size_t)set->rows64() * stride * e : 0;
    std::unique_ptr<char[]> packed(new (std::nothrow) char[bytes]());
    if (!packed) return set_error(SLLM_ERR_OOM, "out of memory");
    for (int r = 0; rank > 0 && r < set->rows; r++)
        for (int k = 0; k < rank; k++)
            std::memcpy(packed.get() + (size_t)b_at(r, k, stride) * e, (const char *)b + ((size_t)r * rank + k) * e, e);
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
    g.tiles = p.tiles;
    g.splits = p.splits;
    g.most = p.most;
    g.steps = g.cols / kStep / (p.splits * p.waves);
    g.more = g.cols / kStep % (p.splits * p.waves);
    void *ws = nullptr;
    size_t cap = 0;
    hipStream_t s = (hipStream_t)stream;
    const size_t parts = (size_t)p.splits * x_rows * g.stride * sizeof(float);
    const size_t groups = (((size_t)p.tiles + 3) / 4 * 4 + (size_t)p.tiles * p.most * kGroup) * sizeof(int);
    if (!small(g, p, set->elem())) {
        const sllm_status st = stream_workspace(s, parts + groups, &ws, &cap);
        if (st != SLLM_OK) return st;
    }
    g.t = (float *)ws;
    g.groups = (int *)((char *)ws + parts);
    if (set->type == SLLM_LORA_F32) return launch<float>(g, p, s);
    if (set->type == SLLM_LORA_F16) return launch<_Float16>(g, p, s);
    return launch<uint16_t>(g, p, s);
}

}  // extern "C"
