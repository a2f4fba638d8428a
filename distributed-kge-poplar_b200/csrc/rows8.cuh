// Rows in 8-bit floating point with a power of two for each 128 values, and their product on the tensor cores.
//
//   value ~ q 2^e,  q = e4m3(value 2^-e),  e = the smallest that brings the block's largest value down to 448
//   out[i, j] = sum over blocks of 2^(ea + eb) sum over the block of qa qb
//
// tcgen05.mma.kind::mxf8f6f4.block_scale multiplies by a power of two per row and 32 values of k as it accumulates in fp32, so
// a block's byte serves four instructions and nothing is left to do between them: the accumulator stays in TMEM over all of k.
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

inline size_t value_stride(size_t cols) { return round_up(cols, 16); }
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
// Four values as e4m3, NaN for what is not finite (the conversion would saturate an infinity).
__device__ __forceinline__ uint32_t to_e4m3x4(const float (&x)[4], float inverse) {
    uint16_t lo, hi;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(x[1] * inverse), "f"(x[0] * inverse));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(x[3] * inverse), "f"(x[2] * inverse));
    uint32_t w = (uint32_t)lo | (uint32_t)hi << 16;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if ((__float_as_uint(x[i]) & 0x7f800000u) == 0x7f800000u) w = (w & ~(0xffu << (8 * i))) | (uint32_t)kNan << (8 * i);
    return w;
}

// A thread takes 16 consecutive values: 8 lanes a block, a warp the 4 blocks whose bytes lie side by side.
template <class T>
static __global__ void __launch_bounds__(256) k_quantise_rows(const T* __restrict__ x, size_t rows, size_t cols, long long stride, size_t groups,
                                                              uint8_t* __restrict__ values, uint8_t* __restrict__ exponents) {
    const size_t unit = (size_t)blockIdx.x * 8 + threadIdx.x / 32;  // (row, group), rows rounded up to 128
    const size_t r = unit / groups, group = unit % groups;
    const int lane = threadIdx.x & 31;
    const size_t row_tiles = (rows + 127) / 128;
    if (r >= row_tiles * 128) return;
    uint32_t* const bytes = reinterpret_cast<uint32_t*>(exponents + ((r / 128) * groups + group) * kGroupBytes + (r % 32) * 16 + (r % 128) / 32 * 4);
    if (r >= rows) {
        if (lane == 0) *bytes = 0x01010101u * kOne;
        return;
    }
    const size_t c0 = group * (4 * kBlock) + lane * 16, ld = (cols + 15) / 16 * 16;
    const T* const src = x + (long long)r * stride + c0;
    float v[16];
    if (c0 + 16 <= cols && (reinterpret_cast<uintptr_t>(src) & 15u) == 0) {
        constexpr int V = 16 / (int)sizeof(T);
#pragma unroll
        for (int q = 0; q < 16 / V; ++q) {
            float part[V];
            const uint4 t = reinterpret_cast<const uint4*>(src)[q];
            lp::unpack<T>(lp::Vector{{t.x, t.y, t.z, t.w}}, part);
#pragma unroll
            for (int j = 0; j < V; ++j) v[q * V + j] = part[j];
        }
    } else {
#pragma unroll
        for (int j = 0; j < 16; ++j) v[j] = c0 + j < cols ? lp::as_float(src[j]) : 0.f;
    }
    uint32_t largest = 0;
#pragma unroll
    for (int j = 0; j < 16; ++j) largest = max(largest, finite_magnitude(v[j]));
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) largest = max(largest, __shfl_xor_sync(~0u, largest, o));
    const int byte = exponent_byte(largest);
    const float inverse = inverse_scale(byte);
    uint32_t four = (uint32_t)byte << (8 * (lane / 8));
    four |= __shfl_xor_sync(~0u, four, 8);
    four |= __shfl_xor_sync(~0u, four, 16);
    if (lane == 0) *bytes = four;
    if (c0 < ld) {
        uint4 q;
        q.x = to_e4m3x4({v[0], v[1], v[2], v[3]}, inverse);
        q.y = to_e4m3x4({v[4], v[5], v[6], v[7]}, inverse);
        q.z = to_e4m3x4({v[8], v[9], v[10], v[11]}, inverse);
        q.w = to_e4m3x4({v[12], v[13], v[14], v[15]}, inverse);
        *reinterpret_cast<uint4*>(values + r * ld + c0) = q;
    }
}

// The columns of x as rows: a block is 128 rows of x in one column.  64 columns and 128 rows to a thread block; a thread keeps 32
// rows of its column, so x is read along its rows and each thread writes 32 bytes side by side.
constexpr int kTurnCols = 64;
template <class T>
static __global__ void __launch_bounds__(256) k_quantise_columns(const T* __restrict__ x, size_t rows, size_t cols, long long stride, size_t groups,
                                                                 uint8_t* __restrict__ values, uint8_t* __restrict__ exponents) {
    __shared__ uint32_t s_largest[4][kTurnCols];
    const size_t blocks = (rows + kBlock - 1) / kBlock, all_blocks = groups * 4;
    const size_t tile = blockIdx.x / all_blocks, block = blockIdx.x % all_blocks;  // columns are rounded up to 128
    const int tc = threadIdx.x % kTurnCols, quarter = threadIdx.x / kTurnCols;
    const size_t c = tile * kTurnCols + tc, r0 = block * kBlock + (size_t)quarter * 32, ld = (rows + 15) / 16 * 16;
    float v[32];
    uint32_t largest = 0;
#pragma unroll
    for (int j = 0; j < 32; ++j) {
        v[j] = c < cols && r0 + j < rows ? lp::as_float(x[(long long)(r0 + j) * stride + (long long)c]) : 0.f;
        largest = max(largest, finite_magnitude(v[j]));
    }
    s_largest[quarter][tc] = largest;
    __syncthreads();
    largest = max(max(s_largest[0][tc], s_largest[1][tc]), max(s_largest[2][tc], s_largest[3][tc]));
    const int byte = block < blocks ? exponent_byte(largest) : kOne;
    if (quarter == 0) exponents[((c / 128) * groups + block / 4) * kGroupBytes + (c % 32) * 16 + (c % 128) / 32 * 4 + block % 4] = (uint8_t)byte;
    if (c >= cols) return;
    const float inverse = inverse_scale(byte);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        if (r0 + 16 * h >= ld) continue;
        uint4 q;
        q.x = to_e4m3x4({v[16 * h], v[16 * h + 1], v[16 * h + 2], v[16 * h + 3]}, inverse);
        q.y = to_e4m3x4({v[16 * h + 4], v[16 * h + 5], v[16 * h + 6], v[16 * h + 7]}, inverse);
        q.z = to_e4m3x4({v[16 * h + 8], v[16 * h + 9], v[16 * h + 10], v[16 * h + 11]}, inverse);
        q.w = to_e4m3x4({v[16 * h + 12], v[16 * h + 13], v[16 * h + 14], v[16 * h + 15]}, inverse);
        *reinterpret_cast<uint4*>(values + c * ld + r0 + 16 * h) = q;
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
};

// The tensor core's two operands are the table (128 rows of b to the 128 lanes) and the queries (TM rows of a to as many
// columns), not the other way round: consecutive lanes then hold consecutive columns of `out`, and a warp stores one row's 32
// of them at once.
constexpr int kTileN = 128;
constexpr int kTmemColumns = 512;
template <int TM>
struct Tile {
    // Four warps reach a tile's 128 lanes; from 64 columns on eight share them, two to a scheduler.
    static constexpr int kColumnWarps = TM >= 64 ? 2 : 1;
    static constexpr int kEpilogueWarps = 4 * kColumnWarps;
    static constexpr int kThreads = 32 * (2 + kEpilogueWarps);
    static constexpr int kWarpColumns = TM / kColumnWarps;
    static constexpr int kAGroups = (TM + 127) / 128;
    static constexpr int kBBytes = kTileN * kBlock, kABytes = TM * kBlock;
    static constexpr int kStageBytes = kBBytes + kABytes + kGroupBytes * (1 + kAGroups);
    static constexpr int kTileBytes = (kStageBytes + 1023) / 1024 * 1024;  // the swizzle wants 1024-byte boundaries
    static constexpr int kStages = 200 * 1024 / kTileBytes < 10 ? 200 * 1024 / kTileBytes : 10;
    static constexpr int kAccumulators = TM <= 128 ? 2 : 1;
    static constexpr int kColumns = TM < 32 ? 32 : TM;
    static constexpr int kScaleColumns = 4 * (1 + kAGroups);
    static constexpr int kScale0 = kAccumulators * kColumns;
    static_assert(kScale0 + kStages * kScaleColumns <= kTmemColumns, "accumulators and scales share the tensor memory");
    static constexpr size_t smem() { return 1024 + (size_t)kStages * kTileBytes; }
};

__device__ __forceinline__ void bulk_load(uint8_t* dst_smem, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(tc::smem_u32(dst_smem)), "l"(src), "r"(bytes), "r"(tc::smem_u32(bar))
                 : "memory");
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
template <int ROWS, class TOut>
__device__ __forceinline__ void store_columns(TOut* out, long long stride, const uint32_t (&acc)[32], int rows) {
    if (rows == ROWS) {
        TOut *p0 = out, *p1 = out + stride, *p2 = p1 + stride, *p3 = p2 + stride;
        const long long four = 4 * stride;
#pragma unroll
        for (int j = 0; j < ROWS; j += 4) {
            lp::store_rounded(p0, __uint_as_float(acc[j]));
            lp::store_rounded(p1, __uint_as_float(acc[j + 1]));
            lp::store_rounded(p2, __uint_as_float(acc[j + 2]));
            lp::store_rounded(p3, __uint_as_float(acc[j + 3]));
            p0 += four, p1 += four, p2 += four, p3 += four;
        }
    } else {
#pragma unroll
        for (int j = 0; j < ROWS; ++j)
            if (j < rows) lp::store_rounded(out + j * stride, __uint_as_float(acc[j]));
    }
}

// Warp 0 fetches, warp 1 multiplies, the others write out; a block takes one tile after another, and its next tile is fetched
// and multiplied while the last one is written.
template <int TM, class TOut>
static __global__ void __launch_bounds__(Tile<TM>::kThreads, 1)
k_product8(const __grid_constant__ CUtensorMap a_map, const __grid_constant__ CUtensorMap b_map, ProductArgs g) {
    using L = Tile<TM>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* const smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    __shared__ uint64_t s_full[L::kStages], s_empty[L::kStages], s_done[L::kAccumulators], s_free[L::kAccumulators];
    __shared__ uint32_t s_tmem;
    __shared__ int s_gave_up;
    volatile int* const gave_up = &s_gave_up;
    const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < L::kStages; ++i) tc::mbar_init(&s_full[i], 1), tc::mbar_init(&s_empty[i], 1);
        for (int i = 0; i < L::kAccumulators; ++i) tc::mbar_init(&s_done[i], 1), tc::mbar_init(&s_free[i], L::kEpilogueWarps);
        tc::mbar_fence_init();
        s_gave_up = 0;
    }
    if (warp == 1) tc::tmem_alloc(&s_tmem, kTmemColumns);
    tc::tc_fence_before();
    __syncthreads();
    tc::tc_fence_after();
    const uint32_t tmem = s_tmem;
    const int n_work = g.n_tiles * g.m_tiles * g.splits;

    if (warp == 0) {
        if (tc::elect_one()) {
            int stage = 0;
            uint32_t parity = 1;  // the ring starts empty
            for (int w = blockIdx.x; w < n_work; w += gridDim.x) {
                const int mt = w % g.m_tiles, nt = w / g.m_tiles % g.n_tiles, split = w / (g.m_tiles * g.n_tiles);
                const int first = (int)((long long)g.blocks * split / g.splits), last = (int)((long long)g.blocks * (split + 1) / g.splits);
                for (int kb = first; kb < last; ++kb) {
                    if (!wait(&s_empty[stage], parity, gave_up)) goto fetched;
                    uint8_t* const at = smem + stage * L::kTileBytes;
                    tc::mbar_arrive_expect(&s_full[stage], L::kStageBytes);
                    tc::tma_load_2d(at, &b_map, kb * kBlock, nt * kTileN, &s_full[stage]);
                    tc::tma_load_2d(at + L::kBBytes, &a_map, kb * kBlock, mt * TM, &s_full[stage]);
                    uint8_t* const scales = at + L::kBBytes + L::kABytes;
                    bulk_load(scales, g.b_exponents + ((size_t)nt * g.groups + kb / 4) * kGroupBytes, kGroupBytes, &s_full[stage]);
#pragma unroll
                    for (int i = 0; i < L::kAGroups; ++i) {
                        // rows past the last group of 128: any group's scales will do, their values are zeros that no one stores
                        const int row_group = min(mt * L::kAGroups + i, (g.m - 1) / 128);
                        bulk_load(scales + kGroupBytes * (1 + i), g.a_exponents + ((size_t)row_group * g.groups + kb / 4) * kGroupBytes, kGroupBytes, &s_full[stage]);
                    }
                    if (++stage == L::kStages) stage = 0, parity ^= 1;
                }
            }
        fetched:;
        }
    } else if (warp == 1) {
        if (tc::elect_one()) {
            int stage = 0, slot = 0;
            uint32_t parity = 0, slot_parity = 1;
            for (int w = blockIdx.x; w < n_work; w += gridDim.x) {
                const int split = w / (g.m_tiles * g.n_tiles);
                const int first = (int)((long long)g.blocks * split / g.splits), last = (int)((long long)g.blocks * (split + 1) / g.splits);
                if (!wait(&s_free[slot], slot_parity, gave_up)) goto multiplied;
                tc::tc_fence_after();
                for (int kb = first; kb < last; ++kb) {
                    if (!wait(&s_full[stage], parity, gave_up)) goto multiplied;
                    tc::tc_fence_after();
                    const uint32_t at = tc::smem_u32(smem + stage * L::kTileBytes);
                    const uint32_t scales = tmem + L::kScale0 + stage * L::kScaleColumns;
#pragma unroll
                    for (int i = 0; i < 1 + L::kAGroups; ++i) copy_scales(scales + 4 * i, at + L::kBBytes + L::kABytes + kGroupBytes * i);
                    const uint64_t b_desc = tc::make_kmajor_sw128_desc(at), a_desc = tc::make_kmajor_sw128_desc(at + L::kBBytes);
                    const uint32_t idesc = scaled_idesc(kTileN, TM, kb & 3);
#pragma unroll
                    for (int q = 0; q < 4; ++q)  // 32 values of k each, 32 bytes further
                        mma_scaled(tmem + slot * L::kColumns, b_desc + 2 * q, a_desc + 2 * q, idesc, scales, scales + 4, kb > first || q > 0);
                    tc::umma_commit(&s_empty[stage]);
                    if (++stage == L::kStages) stage = 0, parity ^= 1;
                }
                tc::umma_commit(&s_done[slot]);
                if (++slot == L::kAccumulators) slot = 0, slot_parity ^= 1;
            }
        multiplied:;
        }
    } else {
        const int quad = warp & 3;  // the lanes that this warp may read
        const int column0 = (warp - 2) / 4 * L::kWarpColumns;
        int slot = 0;
        uint32_t parity = 0;
        for (int w = blockIdx.x; w < n_work; w += gridDim.x) {
            const int mt = w % g.m_tiles, nt = w / g.m_tiles % g.n_tiles, split = w / (g.m_tiles * g.n_tiles);
            if (!wait(&s_done[slot], parity, gave_up)) break;
            tc::tc_fence_after();
            const int n = nt * kTileN + quad * 32 + lane, m0 = mt * TM + column0;
            TOut* const out = static_cast<TOut*>(g.out) + (size_t)split * g.split_stride + (long long)m0 * g.out_stride + n;
#pragma unroll
            for (int c = 0; c < L::kWarpColumns; c += 32) {
                uint32_t acc[32];
                tc::tmem_ld32(tmem + slot * L::kColumns + column0 + c + ((uint32_t)(quad * 32) << 16), acc);
                constexpr int kRows = L::kWarpColumns < 32 ? L::kWarpColumns : 32;
                const int rows = min(kRows, g.m - m0 - c);
                store_columns<kRows>(out + (long long)c * g.out_stride, g.out_stride, acc, n < g.n ? rows : 0);
            }
            tc::tc_fence_before();
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(&s_free[slot]);
            if (++slot == L::kAccumulators) slot = 0, parity ^= 1;
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
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= (long long)m * n) return;
    float sum = partial[i];
    for (int s = 1; s < splits; ++s) sum += partial[i + s * split_stride];
    lp::store_rounded(out + i / n * out_stride + i % n, sum);
}

}  // namespace rows8
}  // namespace kge
