// Rows in 8-bit floating point with a power of two for each 128 values, and their product on the tensor cores.
//
//   value ~ q 2^e,  q = e4m3(value 2^-e),  e = the smallest that brings the block's largest value down to 448
//   out[i, j] = sum over blocks of 2^(ea + eb) sum over the block of qa qb
//
// tcgen05.mma.kind::mxf8f6f4.block_scale multiplies by a power of two per row and 32 values of k as it accumulates in fp32, so
// a block's byte serves four instructions and nothing is left to do between them: the accumulator stays in TMEM over 2048 of k.
//
// What bounds it: the results' bytes where rows are short (512 x 500 000 x 256 to bf16, 512 MB: 117 us, 5.5 TB/s with the table), the
// tensor cores where they are long (8192 x 8192 x 4096: the product alone 2.6 PFLOP/s).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "common.hpp"
#include "log_probs.cuh"
#include "tc_gemm.cuh"
#include "tc_planes.cuh"

namespace kge {
namespace rows8 {

constexpr int kBlock = 128;         // values that share a scale
constexpr int kGroupBytes = 512;    // exponents of 128 rows x 4 blocks
constexpr int kOne = 127;           // the byte of 2^0
constexpr int kNan = 0x7f;          // e4m3 has no infinity

// Bytes from row to row: rows of more than a block begin on a line, so that no two of them share one (100 001 x 256 bf16 values by
// columns: 31 us where they did, 27 us).
__host__ __device__ inline size_t value_stride(size_t cols) { return cols <= kBlock ? (cols + 15) / 16 * 16 : (cols + 127) / 128 * 128; }
inline size_t blocks_of(size_t cols) { return (cols + kBlock - 1) / kBlock; }
inline size_t groups_of(size_t cols) { return (blocks_of(cols) + 3) / 4; }

// The exponent byte of a block whose largest finite value has the bits `largest`: 448 = 1.75 * 2^8.
__device__ __forceinline__ int exponent_byte(uint32_t largest) {
    if (largest == 0) return kOne;
    int e = (int)(largest >> 23);  // biased; a subnormal is far below 2^-127 * 2^8 either way
    if ((largest & 0x7fffffu) > 0x600000u) ++e;
    return max(0, e - 8);
}
// 2^-e, exact for every byte: 0 is 2^127, 247 (the largest there is) 2^-120.
__device__ __forceinline__ float inverse_scale(int byte) { return __uint_as_float((uint32_t)(254 - byte) << 23); }

__device__ __forceinline__ uint32_t finite_magnitude(float x) {
    const uint32_t b = __float_as_uint(x) & 0x7fffffffu;
    return b < 0x7f800000u ? b : 0u;
}
__device__ __forceinline__ uint32_t to_e4m3x2(float lo, float hi) {
    uint16_t w;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(w) : "f"(hi), "f"(lo));
    return w;
}
// Values times `inverse` as e4m3, four to a word.  The conversion saturates an infinity, so where some value is not finite (`special`)
// those become NaN one by one.
template <int N>
__device__ __forceinline__ void to_e4m3(const float (&v)[N], float inverse, bool special, uint32_t (&w)[N / 4]) {
#pragma unroll
    for (int q = 0; q < N / 4; ++q)
        w[q] = to_e4m3x2(v[4 * q] * inverse, v[4 * q + 1] * inverse) | to_e4m3x2(v[4 * q + 2] * inverse, v[4 * q + 3] * inverse) << 16;
    if (special) {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if ((__float_as_uint(v[i]) & 0x7f800000u) == 0x7f800000u) w[i / 4] = (w[i / 4] & ~(0xffu << (8 * (i % 4)))) | (uint32_t)kNan << (8 * (i % 4));
    }
}

// Sixteen values as they lie in memory: 8 words of two or 16 of one.
template <class T>
struct Sixteen {
    static constexpr int kPer = lp::Words<T>::kPer, kWords = 16 / kPer;
    uint32_t w[kWords];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < kWords; ++i) w[i] = 0;
    }
    // The values from p on, `live` of them and zeros after; `first` and `end` are where the whole matrix lies.  Off a 16-byte boundary the
    // vectors around the values are read and shifted into place (512 x 100 001 bf16 values: 61 us read value by value).
    __device__ __forceinline__ void load(const T* p, int live, const T* first, const T* end) {
        const uint32_t off = (uint32_t)(reinterpret_cast<uintptr_t>(p) & 15u);
        const uint4* const q = reinterpret_cast<const uint4*>(reinterpret_cast<uintptr_t>(p) - off);
        if (live >= 16 && off == 0) {
#pragma unroll
            for (int i = 0; i < kWords / 4; ++i) {
                const uint4 t = q[i];
                w[4 * i] = t.x, w[4 * i + 1] = t.y, w[4 * i + 2] = t.z, w[4 * i + 3] = t.w;
            }
        } else if (live >= 16 && reinterpret_cast<const T*>(q) >= first && reinterpret_cast<const T*>(q + kWords / 4 + 1) <= end) {
            uint32_t a[kWords + 4];
#pragma unroll
            for (int i = 0; i <= kWords / 4; ++i) {
                const uint4 t = q[i];
                a[4 * i] = t.x, a[4 * i + 1] = t.y, a[4 * i + 2] = t.z, a[4 * i + 3] = t.w;
            }
            if (off & 8u) {
#pragma unroll
                for (int i = 0; i < kWords + 2; ++i) a[i] = a[i + 2];
            }
            if (off & 4u) {
#pragma unroll
                for (int i = 0; i < kWords + 1; ++i) a[i] = a[i + 1];
            }
#pragma unroll
            for (int i = 0; i < kWords; ++i) w[i] = __funnelshift_r(a[i], a[i + 1], (off & 3u) * 8u);
        } else {
            clear();
#pragma unroll
            for (int j = 0; j < 16; ++j)
                if (j < live) w[j / kPer] |= lp::Row<T>::bits(p + j) << (kPer == 2 ? 16 * (j & 1) : 0);
        }
    }
    // The largest magnitude, as the bits of an fp32; infinities and NaN are above all others.
    __device__ __forceinline__ uint32_t largest() const {
        if constexpr (kPer == 1) {
            uint32_t m = 0;
#pragma unroll
            for (int i = 0; i < kWords; ++i) m = max(m, w[i] & 0x7fffffffu);
            return m;
        } else {
            uint32_t m = 0;
#pragma unroll
            for (int i = 0; i < kWords; ++i) m = larger_halves(m, w[i] & 0x7fff7fffu);
            return magnitude(max(m & 0xffffu, m >> 16));
        }
    }
    static __device__ __forceinline__ uint32_t larger_halves(uint32_t a, uint32_t b) {
        uint32_t r;
        asm("max.u16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
        return r;
    }
    static __device__ __forceinline__ uint32_t magnitude(uint32_t half) { return __float_as_uint(lp::Words<T>::floats(half).x); }
    __device__ __forceinline__ void floats(float (&v)[16]) const {
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
            const float2 t = lp::Words<T>::floats(w[i]);
            v[kPer * i] = t.x;
            if (kPer == 2) v[kPer * i + 1] = t.y;
        }
    }
};

// Eight lanes take a block, 16 consecutive values each.  Bound by memory: what is in flight is as many warps as fit (512 x 100 001 bf16
// values 30.8 us, 5.0 TB/s, fp32 41.1 us, 6.2 TB/s; with four blocks' worth to each lane, all fetched first, but a third of the warps
// 39.0 and 65.2).
template <class T>
static __global__ void __launch_bounds__(256) k_quantise_rows(const T* __restrict__ x, uint32_t rows, size_t cols, long long stride, uint32_t blocks, uint32_t groups,
                                                              uint32_t units, uint8_t* __restrict__ values, uint8_t* __restrict__ exponents) {
    grid_dependency_sync();
    const int lane = threadIdx.x & 31;
    const size_t ld = value_stride(cols);
    const uint32_t unit = (blockIdx.x * 8 + threadIdx.x / 32) * 4 + lane / 8, r = unit / blocks, block = unit - r * blocks;  // rows rounded up to 128
    const size_t c0 = (size_t)block * kBlock + (lane & 7) * 16;
    Sixteen<T> raw;
    if (unit < units && r < rows && c0 < cols)
        raw.load(x + (long long)r * stride + c0, (int)min((size_t)16, cols - c0), x, x + (long long)(rows - 1) * stride + (long long)cols);
    else raw.clear();
    float v[16];
    raw.floats(v);
    uint32_t largest = raw.largest();
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) largest = max(largest, __shfl_xor_sync(~0u, largest, o));
    const bool special = largest >= 0x7f800000u;
    if (__any_sync(~0u, special)) {
        uint32_t finite = 0;
#pragma unroll
        for (int j = 0; j < 16; ++j) finite = max(finite, finite_magnitude(v[j]));
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) finite = max(finite, __shfl_xor_sync(~0u, finite, o));
        largest = finite;
    }
    if (unit >= units) return;
    const int byte = exponent_byte(largest);
    if ((lane & 7) == 0) {
        uint8_t* const bytes = exponents + (size_t)(r / 128) * groups * kGroupBytes + (r % 32) * 16 + (r % 128) / 32 * 4;
        bytes[block / 4 * kGroupBytes + block % 4] = (uint8_t)byte;
        for (uint32_t none = block + 1; block + 1 == blocks && none % 4 != 0; ++none) bytes[none / 4 * kGroupBytes + none % 4] = kOne;
    }
    if (r < rows && c0 < ld) {
        uint32_t w[4];
        to_e4m3(v, inverse_scale(byte), special, w);
        *reinterpret_cast<uint4*>(values + (size_t)r * ld + c0) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// The columns of x as rows: a block is 128 rows of x in one column.  64 columns and 128 rows to a thread block; a warp takes 16 rows,
// a thread two columns of them: neighbours where two fit a word, so that a warp reads 128 bytes of a row at once (value by value
// 512 x 100 001 bf16 values took 96 us, this 39.1; by warps of eight rows, twice as many, 52.7; 256 bytes of a row
// to a block 42.7).  The bytes are turned in shared memory and written 128 side by side.
constexpr int kTurnCols = 64;
template <class T>
static __global__ void __launch_bounds__(256) k_quantise_columns(const T* __restrict__ x, size_t rows, size_t cols, long long stride, size_t groups,
                                                                 uint8_t* __restrict__ values, uint8_t* __restrict__ exponents) {
    using S = Sixteen<T>;
    constexpr int kPer = S::kPer, kPitch = kBlock + 16;
    __shared__ uint32_t s_largest[8][kTurnCols];
    __shared__ alignas(16) uint8_t s_out[kTurnCols * kPitch];
    grid_dependency_sync();
    const size_t blocks = (rows + kBlock - 1) / kBlock;
    const uint32_t tiles = (uint32_t)((cols + 127) / 128 * (128 / kTurnCols));  // columns are rounded up to 128
    const size_t block = blockIdx.x / tiles, tile = blockIdx.x % tiles;  // neighbours read neighbouring parts of the same rows
    const int lane = threadIdx.x & 31, warp = threadIdx.x / 32;
    const size_t c0 = tile * kTurnCols, r0 = block * kBlock + (size_t)warp * 16, ld = value_stride(rows);
    const int own[2] = {kPer == 2 ? 2 * lane : lane, kPer == 2 ? 2 * lane + 1 : lane + 32};  // this thread's columns of the tile
    const int live = r0 < rows ? (int)min((size_t)16, rows - r0) : 0;
    const T* const p = x + (long long)r0 * stride + (long long)c0 + own[0];
    uint32_t w[kPer == 2 ? 16 : 32];  // two columns of 16 rows: side by side in a word, or one after the other
    if (kPer == 2 && live == 16 && c0 >= 1 && c0 + kTurnCols + 1 <= cols) {  // a word to either side is the row's too
        // Every other row begins at the same place in a word, `stride` words further.  A row that begins inside one takes its pairs from
        // two words each.
#pragma unroll
        for (int odd = 0; odd < 2; ++odd) {
            const uintptr_t at = reinterpret_cast<uintptr_t>(p + odd * stride);
            const uint32_t* const word = reinterpret_cast<const uint32_t*>(at & ~(uintptr_t)3);
#pragma unroll
            for (int j = 0; j < 8; ++j) w[2 * j + odd] = word[j * stride];
            if (at & 2u) {
                uint32_t next[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) next[j] = word[j * stride + 1];
#pragma unroll
                for (int j = 0; j < 8; ++j) w[2 * j + odd] = __funnelshift_r(w[2 * j + odd], next[j], 16);
            }
        }
    } else {
        const bool here[2] = {c0 + own[0] < cols, c0 + own[1] < cols};
        const int apart = own[1] - own[0];
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            const uint32_t a = here[0] && j < live ? lp::Row<T>::bits(p + (long long)j * stride) : 0u;
            const uint32_t b = here[1] && j < live ? lp::Row<T>::bits(p + (long long)j * stride + apart) : 0u;
            if (kPer == 2) w[j] = a | b << 16;
            else w[j] = a, w[(j + 16) % (kPer == 2 ? 16 : 32)] = b;
        }
    }
    if constexpr (kPer == 2) {
        uint32_t m = 0;
#pragma unroll
        for (int j = 0; j < 16; ++j) m = S::larger_halves(m, w[j] & 0x7fff7fffu);
        s_largest[warp][own[0]] = S::magnitude(m & 0xffffu);
        s_largest[warp][own[1]] = S::magnitude(m >> 16);
    } else {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            uint32_t m = 0;
#pragma unroll
            for (int j = 0; j < 16; ++j) m = max(m, w[16 * h + j] & 0x7fffffffu);
            s_largest[warp][own[h]] = m;
        }
    }
    const auto column = [&](int h, float (&v)[16]) {
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            const float2 t = lp::Words<T>::floats(w[kPer == 2 ? j : 16 * h + j]);
            v[j] = kPer == 2 && h ? t.y : t.x;
        }
    };
    const auto block_largest = [&](int h) {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) m = max(m, s_largest[i][own[h]]);
        return m;
    };
    __syncthreads();
    uint32_t largest[2] = {block_largest(0), block_largest(1)};
    const bool special[2] = {largest[0] >= 0x7f800000u, largest[1] >= 0x7f800000u};
    if (__syncthreads_or(special[0] || special[1])) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float v[16];
            column(h, v);
            uint32_t m = 0;
#pragma unroll
            for (int j = 0; j < 16; ++j) m = max(m, finite_magnitude(v[j]));
            s_largest[warp][own[h]] = m;
        }
        __syncthreads();
        largest[0] = block_largest(0), largest[1] = block_largest(1);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int byte = block < blocks ? exponent_byte(largest[h]) : kOne;
        const size_t c = c0 + own[h];
        if (warp == 0) exponents[((c / 128) * groups + block / 4) * kGroupBytes + (c % 32) * 16 + (c % 128) / 32 * 4 + block % 4] = (uint8_t)byte;
        float v[16];
        column(h, v);
        uint32_t e[4];
        to_e4m3(v, inverse_scale(byte), special[h], e);
        *reinterpret_cast<uint4*>(s_out + own[h] * kPitch + warp * 16) = make_uint4(e[0], e[1], e[2], e[3]);
    }
    __syncthreads();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int row = (int)threadIdx.x / 8 + 32 * h, piece = (int)threadIdx.x % 8;
        const size_t c = c0 + row, r = block * kBlock + (size_t)piece * 16;
        if (c < cols && r < ld) *reinterpret_cast<uint4*>(values + c * ld + r) = *reinterpret_cast<const uint4*>(s_out + row * kPitch + piece * 16);
    }
}

// ---------------------------------------------------------------------------
// The product.

// Set when a bounded wait of k_product8 has given up.
static __device__ unsigned g_product8_status;

struct ProductArgs {
    const uint8_t* a_exponents;
    const uint8_t* b_exponents;
    void* out;             // [m, n] of the output type, or with splits the partial sums fp32 [split, m, n]
    long long out_stride;  // elements from row to row
    long long split_stride;
    int m, n, blocks, groups;
    int n_tiles, m_tiles, splits;
    int chunk;  // tiles of n that are gone through for all of m before the next ones
    int stages; // of the ring
    int boxes;  // tiles of n whose results go out as boxes of a tile's rows
};

// The tiles of a block, one after another.  Tiles that are worked on at the same time lie side by side along the rows of `out`, so
// that its memory is written in long pieces, in chunks whose part of the table stays in L2 until all of m has met it.  A block that keeps
// its rows of `a` goes along them.  Where few blocks work on a row of `out` each does four tiles side by side (4736 queries, four blocks a row,
// x 62 504 x 128 to bf16: 154 us, one tile at a time 232; eight blocks a row 77 and 79, nine 68 and 66, fourteen 53 and 50), if there
// are tiles enough that none goes without (512 x 1387 x 256 to fp32, eleven tiles: 9.4 us by fours, one at a time 4.7).
template <bool RESIDENT>
struct Tiles {
    int w, step, n_work, stride, run;
    int mt, nt, split;
    __device__ __forceinline__ Tiles(const ProductArgs& g) {
        if (RESIDENT) {
            mt = (int)blockIdx.x % g.m_tiles;
            w = 0;
            step = 1;
            stride = (int)gridDim.x / g.m_tiles;
            run = stride <= 8 && g.n_tiles >= 16 * stride ? 4 : 1;
            n_work = (int)blockIdx.x < stride * g.m_tiles ? g.n_tiles : 0;
            split = 0;
        } else {
            w = (int)blockIdx.x;
            step = (int)gridDim.x;
            n_work = g.n_tiles * g.m_tiles * g.splits;
        }
    }
    __device__ __forceinline__ bool here(const ProductArgs& g) {
        if (RESIDENT) {
            nt = (w / run * stride + (int)blockIdx.x / g.m_tiles) * run + w % run;
            if (nt >= n_work) return false;
        } else {
            if (w >= n_work) return false;
            const int tiles = g.m_tiles * g.n_tiles, i = w % tiles, whole = g.chunk * g.m_tiles;
            split = w / tiles;
            const int at = i / whole, r = i - at * whole, width = min(g.chunk, g.n_tiles - at * g.chunk);
            mt = r / width;
            nt = at * g.chunk + r - mt * width;
        }
        return true;
    }
    __device__ __forceinline__ int first(const ProductArgs& g) const { return (int)((long long)g.blocks * split / g.splits); }
    __device__ __forceinline__ int last(const ProductArgs& g) const { return (int)((long long)g.blocks * (split + 1) / g.splits); }
};

// The tensor core's two operands are the table (128 rows of b to the 128 lanes) and the queries (TM rows of a to as many
// columns), not the other way round: consecutive lanes then hold consecutive columns of `out`, and a warp stores one row's 32
// of them at once.
constexpr int kTileN = 128;
constexpr int kTmemColumns = 512;
// Blocks of k that are summed in tensor memory before the sum joins the others in registers: there every addition rounds toward
// zero, which takes 1e-5 off a sum of 16 384 positive products and 5e-7 off one of 2048.
constexpr int kSegment = 16;
template <int TM, bool RESIDENT>
struct Tile {
    // Four warps reach a tile's 128 lanes, and take 64 of its columns; 128 of 256, for which eight warps have 168 registers each and
    // sixteen would have 96.
    static constexpr int kColumnWarps = TM <= 64 ? 1 : 2;
    static constexpr int kEpilogueWarps = 4 * kColumnWarps;
    static constexpr int kThreads = 32 * (2 + kEpilogueWarps);
    static constexpr int kWarpColumns = TM / kColumnWarps;
    static constexpr int kAGroups = (TM + 127) / 128;
    static constexpr int kBBytes = kTileN * kBlock, kABytes = TM * kBlock;
    // A stage of the ring: a block of the table's rows, with its exponents, and one of the queries' unless the block keeps those.
    static constexpr int kLoneBytes = kBBytes + 1024, kPairBytes = (kBBytes + kABytes + kGroupBytes * (1 + kAGroups) + 1023) / 1024 * 1024;
    static constexpr int kSpace = 220 * 1024, kMostStages = 10;
    // Results on their way out, a box for each two warps: where a block keeps its queries, whose sums are short.
    static constexpr int kBoxBytes = 4096, kBoxes = kColumnWarps * 2 * kBoxBytes;
    static constexpr int kPairStages = kSpace / kPairBytes < kMostStages ? kSpace / kPairBytes : kMostStages;
    static constexpr int kMostResident = 100 * 1024 / kABytes;  // blocks of the queries' rows that a block keeps
    static constexpr bool kOneSegment = RESIDENT && kMostResident <= kSegment;
    // Two accumulators, so that a tile is written out while the next one is summed.  Two of 256 columns leave no room for scales:
    // they share 64, and the next tile begins once those are read, which are read first.
    static constexpr bool kShare = TM > 128;
    static constexpr int kNextColumns = kShare ? TM - 64 : TM < 32 ? 32 : TM;
    static constexpr int kScale0 = kNextColumns + (TM < 32 ? 32 : TM);
    static_assert(!RESIDENT || TM <= 128, "blocks that keep their queries have accumulators of their own, and one group of exponents");
    static_assert(kScale0 + kPairStages * 4 * (1 + kAGroups) <= kTmemColumns, "accumulators and scales share the tensor memory");
    static_assert(kScale0 + (kMostResident + 3) / 4 * 4 * kAGroups + 4 * kMostStages <= kTmemColumns, "accumulators and scales share the tensor memory");
    static int resident_bytes(int blocks) { return blocks * kABytes + (blocks + 3) / 4 * kAGroups * kGroupBytes; }
    static int lone_stages(int blocks) { return std::min(kMostStages, (kSpace - kBoxes - (resident_bytes(blocks) + 1023) / 1024 * 1024) / kLoneBytes); }
    static constexpr size_t smem() { return 1024 + (size_t)kSpace; }
};
// Where `out` takes boxes of whole lines: 64 columns of 16-bit results by 32 rows from two warps, 32 columns of fp32 by 16 rows from
// one.  (4096 x 62 504 bf16 results of 128-wide rows: 138 us, by words from shared memory 197; 512 x 500 000 of 256-wide ones 117 and
// 174; 4096 x 62 504 fp32 ones 199, stored directly 208.)
template <class TOut>
constexpr int kBoxColumns = 128 / (int)sizeof(TOut);
template <class TOut>
constexpr int kBoxRows = sizeof(TOut) == 4 ? 16 : 32;

__device__ __forceinline__ void bulk_load(uint8_t* dst_smem, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(tc::smem_u32(dst_smem)), "l"(src), "r"(bytes), "r"(tc::smem_u32(bar))
                 : "memory");
}
__device__ __forceinline__ void box_store(const CUtensorMap* map, const uint8_t* src_smem, int x, int y) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];"
                 ::"l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(tc::smem_u32(src_smem))
                 : "memory");
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
__device__ __forceinline__ void box_stores_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }  // they have left shared memory
__device__ __forceinline__ void box_stores_done() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }
// Barriers of two warps (1 to 4) and of the four of a part of the columns (5, 6).
__device__ __forceinline__ void two_warps_sync(int which) { asm volatile("bar.sync %0, 64;" ::"r"(1 + which) : "memory"); }
__device__ __forceinline__ void four_warps_sync(int which) { asm volatile("bar.sync %0, 128;" ::"r"(5 + which) : "memory"); }
// Whether any of four warps' threads says so: they meet at barriers of their own from here on, so they go on or end together.
__device__ __forceinline__ bool four_warps_any(int which, bool mine) {
    uint32_t any;
    asm volatile("{\n.reg .pred p, q;\nsetp.ne.u32 p, %2, 0;\nbar.red.or.pred q, %1, 128, p;\nselp.u32 %0, 1, 0, q;\n}" : "=r"(any) : "r"(5 + which), "r"((uint32_t)mine) : "memory");
    return any != 0;
}
// 16 lanes by 32 columns of TMEM, a fragment of 8 x 8 for each two registers: thread t has lane t / 4 (registers 0, 1 of four) or
// t / 4 + 8 (2, 3) and columns 2 (t % 4) and the next, of eight columns for each four registers.  Does not wait.
__device__ __forceinline__ void tmem_ld_fragments(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]),
          "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_ld8(uint32_t taddr, uint32_t (&r)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(taddr)
                 : "memory");
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
// Four fragments of 16-bit values, each turned: lane i gives the address of row i % 8 of fragment i / 8.
__device__ __forceinline__ void store_turned(uint32_t smem, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(smem), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
template <class T>
__device__ __forceinline__ uint32_t rounded_pair(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t rounded_pair<__half>(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
template <>
__device__ __forceinline__ uint32_t rounded_pair<__nv_bfloat16>(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}

// 32 rows of 16 bytes in shared memory (rows 16 bytes apart, groups of 8 rows 128) to 4 columns of TMEM, once for each of the
// four groups of 32 lanes: where block_scale reads the scales of 128 rows and 4 blocks.
__device__ __forceinline__ void copy_scales(uint32_t tmem, uint32_t smem) {
    uint64_t d = 0;
    d |= (uint64_t)((smem >> 4) & 0x3FFF);
    d |= (uint64_t)(128 >> 4) << 16;
    d |= (uint64_t)(128 >> 4) << 32;
    d |= (uint64_t)1 << 46;
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(d) : "memory");
}
__device__ __forceinline__ void mma_scaled(uint32_t tmem_d, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t scale_a, uint32_t scale_b, uint32_t accumulate) {
    asm volatile(
        "{\n.reg .pred p;\n"
        "setp.ne.b32 p, %6, 0;\n"
        "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n}"
        ::"r"(tmem_d), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(scale_a), "r"(scale_b), "r"(accumulate)
        : "memory");
}
// Instruction descriptor: e4m3 on both sides (0 at bits 7-9 and 10-12), N / 8 at bits 17-22, scales in powers of two (bit 23),
// M / 128 at bits 27-28, which byte of a scale column at bits 4-5 (second operand) and 29-30 (first).
__device__ __forceinline__ uint32_t scaled_idesc(int m, int n, int byte) {
    return (uint32_t)byte << 4 | (uint32_t)(n >> 3) << 17 | 1u << 23 | (uint32_t)(m >> 7) << 27 | (uint32_t)byte << 29;
}

// A wait that gives up after about a second, and at once when another of the block's has.
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, volatile int* gave_up) {
    for (uint32_t spins = 0; spins < (1u << 22); ++spins) {
        if (tc::mbar_try_wait(bar, parity)) return true;
        if (*gave_up) return false;
    }
    *gave_up = 1;
    atomicExch(&g_product8_status, 1u);
    return false;
}

// One column of the tile per row of `out`.  With a row's address and a test for each store a tile took 5.8 us, a dependent chain
// of some ten instructions a store with one warp to a scheduler; four addresses apart and no tests leave two.
template <int ROWS, class TOut, int N>
__device__ __forceinline__ void store_columns(TOut* out, long long stride, const float (&acc)[N], int rows) {
    if (rows == ROWS) {
        TOut *p0 = out, *p1 = out + stride, *p2 = p1 + stride, *p3 = p2 + stride;
        const long long four = 4 * stride;
#pragma unroll
        for (int j = 0; j < ROWS; j += 4) {
            lp::store_rounded(p0, acc[j]);
            lp::store_rounded(p1, acc[j + 1]);
            lp::store_rounded(p2, acc[j + 2]);
            lp::store_rounded(p3, acc[j + 3]);
            p0 += four, p1 += four, p2 += four, p3 += four;
        }
    } else {
#pragma unroll
        for (int j = 0; j < ROWS; ++j)
            if (j < rows) lp::store_rounded(out + j * stride, acc[j]);
    }
}

// Rows [first, end) of two boxes side by side, `live` columns of them, to rows of `out` that begin inside a 16-byte vector or a word: words
// where they are whole, the columns at the ends alone.  (512 x 500 001 bf16 results of 256-wide rows: 211 us, and 288 stored 64 bytes of a
// row at a time, where two of three sectors are written in part.  The eight rows are unrolled: with a test for each, 510.)
template <class TOut>
__device__ __forceinline__ void store_rows(const uint8_t* box, TOut* out, long long stride, int first, int end, int live) {
    const int lane = threadIdx.x & 31;
    const uint32_t mine = (uint32_t)(lane * 4);  // two columns of each box; its 16 bytes are where the row's number moves them
    if (live == kTileN && end - first == 8) {
        uint16_t* to = reinterpret_cast<uint16_t*>(out + first * stride);
#pragma unroll
        for (int r = 0; r < 8; ++r, to += stride) {
            const uint8_t* const at = box + first * 128 + r * 128 + (mine ^ (uint32_t)(r << 4));
            const uint32_t a = *reinterpret_cast<const uint32_t*>(at), b = *reinterpret_cast<const uint32_t*>(at + 4096);
            if ((reinterpret_cast<uintptr_t>(to) & 2u) == 0) {
                uint32_t* const words = reinterpret_cast<uint32_t*>(to) + lane;
                words[0] = a, words[32] = b;
            } else {  // a word takes its lower half from the columns before
                const uint32_t before_a = __shfl_up_sync(~0u, a, 1), last_a = __shfl_sync(~0u, a, 31);
                uint32_t before_b = __shfl_up_sync(~0u, b, 1);
                if (lane == 0) before_b = last_a;
                uint32_t* const words = reinterpret_cast<uint32_t*>(to - 1) + lane;
                if (lane > 0) words[0] = __funnelshift_r(before_a, a, 16);
                else to[0] = (uint16_t)a;
                words[32] = __funnelshift_r(before_b, b, 16);
                if (lane == 31) to[kTileN - 1] = (uint16_t)(b >> 16);
            }
        }
    } else {
        for (int row = first; row < end; ++row)
            for (int c = lane; c < live; c += 32)
                reinterpret_cast<uint16_t*>(out + row * stride)[c] =
                    *reinterpret_cast<const uint16_t*>(box + c / 64 * 4096 + row * 128 + ((c % 64 / 8 ^ (row & 7)) << 4) + c % 8 * 2);
    }
}

// Warp 0 fetches, warp 1 multiplies, the others write out; a block takes one tile after another, and its next tile is fetched
// and multiplied while the last one is written.  RESIDENT: the block's rows of `a` fit its shared memory beside the ring and are
// fetched once (512 x 500 000 x 256: per tile 32 KB of the table from L2 instead of 96).
template <int TM, class TOut, bool RESIDENT>
static __global__ void __launch_bounds__(Tile<TM, RESIDENT>::kThreads, 1)
k_product8(const __grid_constant__ CUtensorMap a_map, const __grid_constant__ CUtensorMap b_map, const __grid_constant__ CUtensorMap out_map, ProductArgs g) {
    using L = Tile<TM, RESIDENT>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* const smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    __shared__ uint64_t s_full[L::kMostStages], s_empty[L::kMostStages], s_done[2], s_free[2];  // s_free[0] alone where accumulators share columns
    __shared__ uint64_t s_resident;
    __shared__ uint32_t s_tmem;
    __shared__ int s_gave_up;
    volatile int* const gave_up = &s_gave_up;
    const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < g.stages; ++i) tc::mbar_init(&s_full[i], 1), tc::mbar_init(&s_empty[i], 1);
        for (int i = 0; i < 2; ++i) tc::mbar_init(&s_done[i], 1), tc::mbar_init(&s_free[i], L::kEpilogueWarps);
        tc::mbar_init(&s_resident, 1);
        tc::mbar_fence_init();
        s_gave_up = 0;
    }
    if (warp == 1) tc::tmem_alloc(&s_tmem, kTmemColumns);
    tc::tc_fence_before();
    __syncthreads();
    tc::tc_fence_after();
    grid_dependency_sync();
    const uint32_t tmem = s_tmem;
    // resident: [blocks][TM][128] values, exponents, then the ring
    constexpr int kTileBytes = RESIDENT ? L::kLoneBytes : L::kPairBytes;
    const int a_exponents = g.blocks * L::kABytes;
    uint8_t* const ring = RESIDENT ? smem + (a_exponents + g.groups * L::kAGroups * kGroupBytes + 1023) / 1024 * 1024 : smem;
    uint8_t* const boxes = smem + L::kSpace - L::kBoxes;
    // of the rows past the last group of 128 any group's scales will do: their values are zeros that no one stores
    const auto a_group = [&](int mt, int i, int group) {
        return g.a_exponents + ((size_t)min(mt * L::kAGroups + i, (g.m - 1) / 128) * g.groups + group) * kGroupBytes;
    };

    if (warp == 0) {
        if (tc::elect_one()) {
            int stage = 0;
            uint32_t parity = 1;  // the ring starts empty
            Tiles<RESIDENT> tile(g);
            if (RESIDENT && tile.n_work > 0) {
                tc::mbar_arrive_expect(&s_resident, (uint32_t)(a_exponents + g.groups * L::kAGroups * kGroupBytes));
                for (int kb = 0; kb < g.blocks; ++kb) tc::tma_load_2d(smem + kb * L::kABytes, &a_map, kb * kBlock, tile.mt * TM, &s_resident);
                for (int group = 0; group < g.groups; ++group)
                    for (int i = 0; i < L::kAGroups; ++i)
                        bulk_load(smem + a_exponents + (group * L::kAGroups + i) * kGroupBytes, a_group(tile.mt, i, group), kGroupBytes, &s_resident);
            }
            for (; tile.here(g); tile.w += tile.step) {
                const int first = tile.first(g), last = tile.last(g);
                for (int kb = first; kb < last; ++kb) {
                    if (!wait(&s_empty[stage], parity, gave_up)) goto fetched;
                    uint8_t* const at = ring + stage * kTileBytes;
                    tc::mbar_arrive_expect(&s_full[stage], L::kBBytes + kGroupBytes + (RESIDENT ? 0 : L::kABytes + L::kAGroups * kGroupBytes));
                    tc::tma_load_2d(at, &b_map, kb * kBlock, tile.nt * kTileN, &s_full[stage]);
                    bulk_load(at + L::kBBytes, g.b_exponents + ((size_t)tile.nt * g.groups + kb / 4) * kGroupBytes, kGroupBytes, &s_full[stage]);
                    if (!RESIDENT) {
                        uint8_t* const a = at + L::kBBytes + 1024;
                        tc::tma_load_2d(a, &a_map, kb * kBlock, tile.mt * TM, &s_full[stage]);
#pragma unroll
                        for (int i = 0; i < L::kAGroups; ++i)
                            bulk_load(i == 0 ? at + L::kBBytes + kGroupBytes : a + L::kABytes, a_group(tile.mt, i, kb / 4), kGroupBytes, &s_full[stage]);
                    }
                    if (++stage == g.stages) stage = 0, parity ^= 1;
                }
            }
        fetched:;
        }
    } else if (warp == 1) {
        if (tc::elect_one()) {
            int stage = 0, slot = 0;
            uint32_t parity = 0, slot_parity = 1;
            const uint32_t a_scales = tmem + L::kScale0, ring_scales = a_scales + (RESIDENT ? g.groups * 4 * L::kAGroups : 0);
            Tiles<RESIDENT> tile(g);
            if (RESIDENT && tile.n_work > 0) {
                if (!wait(&s_resident, 0, gave_up)) goto multiplied;
                tc::tc_fence_after();
                for (int i = 0; i < g.groups * L::kAGroups; ++i) copy_scales(a_scales + 4 * i, tc::smem_u32(smem + a_exponents + i * kGroupBytes));
            }
            for (; tile.here(g); tile.w += tile.step) {
                const int last = tile.last(g);
                for (int kb = tile.first(g); kb < last;) {
                    if (!wait(&s_free[L::kShare ? 0 : slot], slot_parity, gave_up)) goto multiplied;
                    tc::tc_fence_after();
                    const int segment = kb, end = min(last, kb + kSegment);
                    for (; kb < end; ++kb) {
                        if (!wait(&s_full[stage], parity, gave_up)) goto multiplied;
                        tc::tc_fence_after();
                        const uint32_t at = tc::smem_u32(ring + stage * kTileBytes);
                        const uint32_t b_scale = ring_scales + stage * 4 * (RESIDENT ? 1 : 1 + L::kAGroups);
                        const uint32_t a_scale = RESIDENT ? a_scales + (kb / 4) * 4 * L::kAGroups : b_scale + 4;
                        copy_scales(b_scale, at + L::kBBytes);
                        if (!RESIDENT) {
#pragma unroll
                            for (int i = 0; i < L::kAGroups; ++i)
                                copy_scales(a_scale + 4 * i, i == 0 ? at + L::kBBytes + kGroupBytes : at + L::kBBytes + 1024 + L::kABytes);
                        }
                        const uint64_t b_desc = tc::make_kmajor_sw128_desc(at);
                        const uint64_t a_desc = tc::make_kmajor_sw128_desc(RESIDENT ? tc::smem_u32(smem + kb * L::kABytes) : at + L::kBBytes + 1024);
                        const uint32_t idesc = scaled_idesc(kTileN, TM, kb & 3);
#pragma unroll
                        for (int q = 0; q < 4; ++q)  // 32 values of k each, 32 bytes further
                            mma_scaled(tmem + slot * L::kNextColumns, b_desc + 2 * q, a_desc + 2 * q, idesc, b_scale, a_scale, kb > segment || q > 0);
                        tc::umma_commit(&s_empty[stage]);
                        if (++stage == g.stages) stage = 0, parity ^= 1;
                    }
                    tc::umma_commit(&s_done[slot]);
                    slot ^= 1;
                    if (L::kShare || slot == 0) slot_parity ^= 1;
                }
            }
        multiplied:;
        }
    } else {
        const int quad = warp & 3;  // the lanes that this warp may read
        const int part = (warp - 2) / 4, column0 = part * L::kWarpColumns, pair = 2 * part + quad / 2;
        int slot = 0;
        uint32_t parity = 0;
        if constexpr (RESIDENT) {
            constexpr int kRows = L::kWarpColumns < 32 ? L::kWarpColumns : 32, kChunks = L::kWarpColumns / kRows;
            // 16-bit results are turned, two warps' into a box; fp32 boxes are one warp's
            constexpr bool kWide = sizeof(TOut) == 4, kTurn = TM >= 64 && !kWide;
            uint8_t* const box = boxes + pair * L::kBoxBytes + (kWide ? quad % 2 * (L::kBoxBytes / 2) : 0);
            const bool issues = lane == 0 && (kWide || quad % 2 == 0);
            for (Tiles<RESIDENT> tile(g); tile.here(g); tile.w += tile.step) {
                const int n0 = tile.nt * kTileN + quad * 32, m0 = tile.mt * TM + column0;
                float acc[kChunks][32];  // 32 columns each, a lane's or (to be turned) two fragments of 16 lanes
                bool ended = false;
                for (int kb = 0; kb < g.blocks; kb += kSegment) {
                    if (four_warps_any(part, !wait(&s_done[slot], parity, gave_up))) {
                        ended = true;
                        break;
                    }
                    tc::tc_fence_after();
                    const uint32_t taddr = tmem + slot * L::kNextColumns + column0 + ((uint32_t)(quad * 32) << 16);
                    uint32_t sum[kChunks][32];
                    if constexpr (kTurn) {
                        uint32_t lo[kChunks][16], hi[kChunks][16];
#pragma unroll
                        for (int i = 0; i < kChunks; ++i) tmem_ld_fragments(taddr + 32 * i, lo[i]), tmem_ld_fragments(taddr + 32 * i + (16u << 16), hi[i]);
                        tmem_ld_wait();
#pragma unroll
                        for (int i = 0; i < kChunks; ++i)
#pragma unroll
                            for (int j = 0; j < 16; ++j) sum[i][j] = lo[i][j], sum[i][16 + j] = hi[i][j];
                    } else {
#pragma unroll
                        for (int i = 0; i < kChunks; ++i) tc::tmem_ld32(taddr + 32 * i, sum[i]);
                    }
                    tc::tc_fence_before();
                    __syncwarp();
                    if (lane == 0) tc::mbar_arrive(&s_free[slot]);
#pragma unroll
                    for (int i = 0; i < kChunks; ++i)
#pragma unroll
                        for (int j = 0; j < 32; ++j) acc[i][j] = L::kOneSegment || kb == 0 ? __uint_as_float(sum[i][j]) : acc[i][j] + __uint_as_float(sum[i][j]);
                    slot ^= 1;
                    if (slot == 0) parity ^= 1;
                }
                if (ended) break;
                TOut* const out = static_cast<TOut*>(g.out) + (long long)m0 * g.out_stride + n0 + lane;
                const bool boxed = tile.nt < g.boxes;  // the others come last: a block's tiles go up
#pragma unroll
                for (int i = 0; i < kChunks; ++i) {
                    const int rows = min(kRows, g.m - m0 - 32 * i);
                    if (rows <= 0) break;  // the same for the four warps
                    if constexpr (kTurn) {
                        if (issues && g.boxes) box_stores_read();
                        if (boxed) two_warps_sync(pair);
                        else four_warps_sync(part);  // the rows before have been read
#pragma unroll
                        for (int q = 0; q < 4; ++q) {  // eight rows of `out` each, of 16 bytes for each eight lanes
                            const uint32_t at = tc::smem_u32(box) + (q * 8 + (lane & 7)) * 128 + (((quad % 2 * 4 + lane / 8) ^ (lane & 7)) << 4);
                            const float* const lo = acc[i] + 4 * q;
                            const float* const hi = acc[i] + 16 + 4 * q;
                            store_turned(at, rounded_pair<TOut>(lo[0], lo[1]), rounded_pair<TOut>(lo[2], lo[3]), rounded_pair<TOut>(hi[0], hi[1]), rounded_pair<TOut>(hi[2], hi[3]));
                        }
                        if (boxed) {
                            tc::fence_async_shared();
                            two_warps_sync(pair);
                            if (issues && n0 < g.n) box_store(&out_map, box, n0, m0 + 32 * i);
                        } else {
                            four_warps_sync(part);
                            store_rows(boxes + part * 2 * L::kBoxBytes, static_cast<TOut*>(g.out) + (long long)(m0 + 32 * i) * g.out_stride + tile.nt * kTileN, g.out_stride,
                                       quad * 8, min(rows, quad * 8 + 8), min(kTileN, g.n - tile.nt * kTileN));
                        }
                    } else if (TM >= 64 && boxed) {
#pragma unroll
                        for (int h = 0; h < 32; h += kBoxRows<TOut>) {
                            if (h >= rows) break;
                            if (issues) box_stores_read();
                            __syncwarp();
                            TOut* const to = reinterpret_cast<TOut*>(box) + lane;
#pragma unroll
                            for (int q = 0; q < kBoxRows<TOut>; ++q) lp::store_rounded(to + q * 32, acc[i][(h + q) % 32]);
                            tc::fence_async_shared();
                            __syncwarp();
                            if (issues && n0 < g.n) box_store(&out_map, box, n0, m0 + 32 * i + h);
                        }
                    } else {
                        store_columns<kRows>(out + (long long)(32 * i) * g.out_stride, g.out_stride, acc[i], n0 + lane < g.n ? rows : 0);
                    }
                }
            }
            if (TM >= 64 && g.boxes && issues) box_stores_done();
        } else {
            // the columns in halves; the upper warps begin with their second one, which is where columns are shared
            constexpr int kHalf = L::kWarpColumns / 2;
            const int turned = L::kShare && part == 1 ? 1 : 0;
            for (Tiles<RESIDENT> tile(g); tile.here(g); tile.w += tile.step) {
                float acc[2][kHalf];
#pragma unroll
                for (int i = 0; i < kHalf; ++i) acc[0][i] = acc[1][i] = 0.f;
                const int last = tile.last(g);
                bool ended = false;
                for (int kb = tile.first(g); kb < last; kb += kSegment) {
                    if (__any_sync(~0u, !wait(&s_done[slot], parity, gave_up))) {
                        ended = true;
                        break;
                    }
                    tc::tc_fence_after();
                    const bool holds = !L::kShare || part != slot;
                    const auto release = [&] {
                        tc::tc_fence_before();
                        __syncwarp();
                        if (lane == 0) tc::mbar_arrive(&s_free[L::kShare ? 0 : slot]);
                    };
                    if (!holds) release();
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint32_t taddr = tmem + slot * L::kNextColumns + column0 + (h ^ turned) * kHalf + ((uint32_t)(quad * 32) << 16);
#pragma unroll
                        for (int i = 0; i < kHalf; i += 8) {
                            uint32_t sum[8];
                            tmem_ld8(taddr + i, sum);
#pragma unroll
                            for (int j = 0; j < 8; ++j) acc[h][i + j] += __uint_as_float(sum[j]);
                        }
                        if (holds && h == (L::kShare ? 0 : 1)) release();
                    }
                    slot ^= 1;
                    if (slot == 0) parity ^= 1;
                }
                if (ended) break;
                const int n = tile.nt * kTileN + quad * 32 + lane;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int m0 = tile.mt * TM + column0 + (h ^ turned) * kHalf;
                    TOut* const out = static_cast<TOut*>(g.out) + (size_t)tile.split * g.split_stride + (long long)m0 * g.out_stride + n;
                    store_columns<kHalf>(out, g.out_stride, acc[h], n < g.n ? min(kHalf, g.m - m0) : 0);
                }
            }
        }
    }
    tc::tc_fence_before();
    __syncthreads();
    if (*gave_up) {  // copies and products in flight end long before this does
        if (threadIdx.x == 0)
            for (int i = 0; i < 1000; ++i) __nanosleep(1000);
        __syncthreads();
    }
    if (warp == 1) {
        tc::tc_fence_after();
        tc::tmem_dealloc(tmem, kTmemColumns);
    }
}

template <class TOut>
static __global__ void __launch_bounds__(256) k_add_splits(const float* __restrict__ partial, long long split_stride, int splits, int m, int n,
                                                           TOut* __restrict__ out, long long out_stride) {
    grid_dependency_sync();
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= (long long)m * n) return;
    float sum = partial[i];
    for (int s = 1; s < splits; ++s) sum += partial[i + s * split_stride];
    lp::store_rounded(out + i / n * out_stride + i % n, sum);
}

}  // namespace rows8
}  // namespace kge
