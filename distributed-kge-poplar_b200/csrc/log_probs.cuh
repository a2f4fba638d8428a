// Log probabilities of given candidates with the entropy of their distribution and its n_best most probable columns, and the
// gradient of all three with respect to the scores.
//
//   z = scale x over a row's live columns;  m >= max z any reference;  S = sum e^(z-m);  T = sum e^(z-m) (z-m)
//   log_prob = (z_t - m) - log S;   entropy = log S - T / S;   p = e^((z-m) - log S)
//   dx = scale ( sum_l g_l [c = c_l] - G p - g_H p (log p + entropy) ),  G = sum_l g_l over the target and the alternatives
//
// The sums are kept in powers of two, and the reference is a score, not a logit: (x - reference) s2, s2 = scale log2(e), is
// right for scores next to each other however large both are, a row of the type's lowest value included (all equal).  The
// reference and log S stay apart in what is kept for the gradient: their sum loses the bits below the reference's last one,
// which at logits of a thousand is 1e-4 of every probability.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <float.h>
#include <stdint.h>

#include "pdl.cuh"

namespace kge {
namespace lp {

struct Scores {
    const void* x;
    const uint8_t* mask;
    const int32_t* count;
    const int32_t* target;
    long long row_stride, mask_stride;
    int cols;
    float s2;     // scale * log2(e)
    float scale;
};

struct Out {
    float* log_prob;
    float* entropy;
    float* log_sum;
    float4* row_state;  // {reference, log2 S, entropy, 1 if the target has a gradient}
    float* best_log_prob;
    int32_t* best_index;
    int n_best;
};

constexpr int kMaxBest = 128;
constexpr int kCandidates = 1024;   // columns, or groups of columns, that pass the first threshold
constexpr int kGroup = 4;           // 16-byte vectors that a thread fetches at once
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kNoReference = -FLT_MAX;  // no live score is below
constexpr float kFarBelow = -200.f;  // 2^-200 is 0 in fp32: exponents below give the same terms, and 0 * -inf stays out

template <class T>
constexpr int vector_width() { return 16 / (int)sizeof(T); }

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float max_or_nan(float a, float b) {
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}
// Two fp32 in one register pair: one instruction for both.
using Pair = unsigned long long;
__device__ __forceinline__ Pair pair(float lo, float hi) {
    Pair r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ float2 halves(Pair v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ Pair fma_pair(Pair a, Pair b, Pair c) {
    Pair r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ Pair add_pair(Pair a, Pair b) {
    Pair r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ Pair mul_pair(Pair a, Pair b) {
    Pair r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

__device__ __forceinline__ float as_float(float v) { return v; }
__device__ __forceinline__ float as_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float as_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void store_rounded(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_rounded(__half* p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void store_rounded(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// What the kernels need of an element type, by 32-bit words of memory: W words make a vector, a word holds PER scores.
template <class T>
struct Words;
template <>
struct Words<float> {
    static constexpr int kPer = 1;
    static constexpr uint32_t kNone = 0xff800000u;  // -inf in every score of a word
    static constexpr float kLow = -1e30f;
    static __device__ __forceinline__ float2 floats(uint32_t w) { return make_float2(__uint_as_float(w), 0.f); }
    static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) { return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b))); }
    static __device__ __forceinline__ uint32_t raised(uint32_t a) { return __float_as_uint(max_or_nan(__uint_as_float(a), kLow)); }
    static __device__ __forceinline__ float largest(uint32_t w) { return __uint_as_float(w); }
};
template <>
struct Words<__nv_bfloat16> {
    static constexpr int kPer = 2;
    static constexpr uint32_t kNone = 0xff80ff80u;
    static constexpr float kLow = -1.0002555517425873e30f;  // 0xf14a
    static constexpr uint32_t kLowBits = 0xf14af14au;
    static __device__ __forceinline__ float2 floats(uint32_t w) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }
    static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) {
        uint32_t r;
        asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
        return r;
    }
    static __device__ __forceinline__ uint32_t raised(uint32_t a) {
        uint32_t r;
        asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(kLowBits));
        return r;
    }
    static __device__ __forceinline__ float largest(uint32_t w) {
        const float2 v = floats(w);
        return fmaxf(v.x, v.y);
    }
};
template <>
struct Words<__half> {
    static constexpr int kPer = 2;
    static constexpr uint32_t kNone = 0xfc00fc00u;
    static constexpr float kLow = -65504.f;
    static constexpr uint32_t kLowBits = 0xfbfffbffu;
    static __device__ __forceinline__ float2 floats(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
    static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) {
        uint32_t r;
        asm("max.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
        return r;
    }
    static __device__ __forceinline__ uint32_t raised(uint32_t a) {
        uint32_t r;
        asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(kLowBits));
        return r;
    }
    static __device__ __forceinline__ float largest(uint32_t w) {
        const float2 v = floats(w);
        return fmaxf(v.x, v.y);
    }
};

struct Vector {
    uint32_t w[4];
};
template <class T>
__device__ __forceinline__ void unpack(const Vector& raw, float (&x)[vector_width<T>()]) {
    constexpr int kPer = Words<T>::kPer;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 v = Words<T>::floats(raw.w[i]);
        x[kPer * i] = v.x;
        if (kPer == 2) x[kPer * i + 1] = v.y;
    }
}
__device__ __forceinline__ uint4 pack(const float (&v)[4], float) {
    return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
}
__device__ __forceinline__ uint4 pack(const float (&v)[8], __nv_bfloat16) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 t = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&t);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ uint4 pack(const float (&v)[8], __half) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __half2 t = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&t);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// One row, seen as 16-byte vectors of memory: vector v holds the columns from v * V - shift on, so that all but the two at the
// ends of a row (whose stride need not be a multiple of 16 bytes) are read whole.  Columns that are not live come as -inf.
template <class T>
struct Row {
    static constexpr int V = vector_width<T>();
    const T* x;
    const uint8_t* mask;
    int cols;     // of these the row's count
    int shift;
    int n_vectors;
    __device__ __forceinline__ Row(const Scores& s, size_t r) {
        x = static_cast<const T*>(s.x) + (long long)r * s.row_stride;
        mask = s.mask ? s.mask + (long long)r * s.mask_stride : nullptr;
        cols = s.count ? max(0, min(s.cols, s.count[r])) : s.cols;
        shift = (int)((reinterpret_cast<uintptr_t>(x) & 15u) / sizeof(T));
        n_vectors = (cols + shift + V - 1) / V;
    }
    __device__ __forceinline__ int first_column(int v) const { return v * V - shift; }
    __device__ __forceinline__ bool whole(int v) const { return v * V >= shift && v * V - shift + V <= cols; }
    __device__ __forceinline__ static uint32_t bits(const float* p) { return __float_as_uint(*p); }
    __device__ __forceinline__ static uint32_t bits(const __half* p) { return *reinterpret_cast<const uint16_t*>(p); }
    __device__ __forceinline__ static uint32_t bits(const __nv_bfloat16* p) { return *reinterpret_cast<const uint16_t*>(p); }
    // Score j of the vector becomes -inf unless `live`.
    __device__ __forceinline__ static void keep(Vector& raw, int j, bool live) {
        constexpr int kPer = Words<T>::kPer;
        const uint32_t part = kPer == 1 ? 0xffffffffu : j & 1 ? 0xffff0000u : 0x0000ffffu;
        if (!live) raw.w[j / kPer] = (raw.w[j / kPer] & ~part) | (Words<T>::kNone & part);
    }
    __device__ __forceinline__ Vector load(int v) const {
        Vector raw;
        const int c0 = first_column(v);
        const bool all = whole(v);
        if (all) {
            const uint4 t = *reinterpret_cast<const uint4*>(x + c0);
            raw.w[0] = t.x, raw.w[1] = t.y, raw.w[2] = t.z, raw.w[3] = t.w;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) raw.w[i] = Words<T>::kNone;
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (c0 + j >= 0 && c0 + j < cols) {
                    constexpr int kPer = Words<T>::kPer;
                    const uint32_t b = bits(x + c0 + j);
                    raw.w[j / kPer] = kPer == 1 ? b : j & 1 ? (raw.w[j / 2] & 0xffffu) | b << 16 : (raw.w[j / 2] & 0xffff0000u) | b;
                }
        }
        if (mask) {
            if (all && (reinterpret_cast<uintptr_t>(mask + c0) & 3u) == 0) {
#pragma unroll
                for (int q = 0; q < V / 4; ++q) {
                    const uint32_t m = *reinterpret_cast<const uint32_t*>(mask + c0 + 4 * q);
#pragma unroll
                    for (int j = 0; j < 4; ++j) keep(raw, 4 * q + j, (m >> (8 * j)) & 0xffu);
                }
            } else {
#pragma unroll
                for (int j = 0; j < V; ++j) keep(raw, j, c0 + j >= 0 && c0 + j < cols && mask[c0 + j]);
            }
        }
        return raw;
    }
    // The vectors v, v + STEP, ... of a group, those from `end` on empty.
    template <int STEP>
    __device__ __forceinline__ void load_group(int v, int end, Vector (&raw)[kGroup]) const {
        if (!mask && v * V >= shift && (v + (kGroup - 1) * STEP + 1) * V - shift <= cols && v + (kGroup - 1) * STEP < end) {
            const uint4* const p = reinterpret_cast<const uint4*>(x - shift) + v;
#pragma unroll
            for (int u = 0; u < kGroup; ++u) {
                const uint4 t = p[u * STEP];
                raw[u].w[0] = t.x, raw[u].w[1] = t.y, raw[u].w[2] = t.z, raw[u].w[3] = t.w;
            }
        } else {
#pragma unroll
            for (int u = 0; u < kGroup; ++u) raw[u] = v + u * STEP < end ? load(v + u * STEP) : none();
        }
    }
    __device__ __forceinline__ static Vector none() {
        Vector raw;
#pragma unroll
        for (int i = 0; i < 4; ++i) raw.w[i] = Words<T>::kNone;
        return raw;
    }
    __device__ __forceinline__ float at(int c) const { return c < cols && (!mask || mask[c]) ? as_float(x[c]) : -INFINITY; }
};

// An unsigned number in the order of the scores: 0 for what is no candidate (-inf, NaN), -0 beside +0.
__device__ __forceinline__ uint32_t order_key(float x) {
    if (!(x > -INFINITY)) return 0u;
    const uint32_t b = __float_as_uint(x + 0.f);
    return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t key) { return __uint_as_float(key ^ ((key >> 31) ? 0x80000000u : 0xffffffffu)); }
// Key and column in one word, the lower column the larger.
__device__ __forceinline__ unsigned long long candidate(uint32_t key, int column) { return (unsigned long long)key << 32 | (0xffffffffu - (uint32_t)column); }

struct Sums {
    float reference, sum, weighted;  // sum of 2^d and of 2^d d, d = (x - reference) s2
    __device__ __forceinline__ void raise(float to, float s2) {
        const float d = fmaxf((reference - to) * s2, kFarBelow), c = ex2(d);
        weighted = c * fmaf(sum, d, weighted);
        sum *= c;
        reference = to;
    }
    __device__ __forceinline__ void join(Sums o, float s2) {
        if (o.reference > reference) raise(o.reference, s2);
        else if (reference > o.reference) o.raise(reference, s2);
        sum += o.sum;
        weighted += o.weighted;
    }
    __device__ __forceinline__ void add(float x, float s2) {
        if (x > reference) raise(x, s2);
        const float d = max_or_nan((x - reference) * s2, kFarBelow), e = ex2(d);
        sum += e;
        weighted = fmaf(e, d, weighted);
    }
};
__device__ __forceinline__ Sums none_yet() { return Sums{kNoReference, 0.f, 0.f}; }
// Of each warp in shared memory: the largest scores of its groups of vectors, and, in the same place afterwards, the groups that
// reach the threshold and the columns that do.  A part of a row has at most THREADS * kGroups groups.
template <int THREADS>
struct Lists {
    static constexpr int kGroups = THREADS == 128 ? 4 : THREADS == 256 ? 16 : THREADS == 512 ? 8 : 5;
    static constexpr int kHits = THREADS <= 256 ? 96 : THREADS == 512 ? 64 : 32;
    static constexpr int kKeys = THREADS <= 256 ? 184 : THREADS == 512 ? 96 : 64;
    static constexpr int kSlots = kHits + 2 * kKeys > 32 * kGroups ? kHits + 2 * kKeys : 32 * kGroups;
};

template <int THREADS>
struct Shared {
    static constexpr int kWarps = THREADS / 32;
    alignas(16) float groups[kWarps][Lists<THREADS>::kSlots];
    alignas(16) unsigned long long key[kCandidates + 1];
    uint32_t bound[kWarps];
    int reach[8][kWarps];
    int rank[THREADS];
    uint32_t histogram[256];
    float warp_top[kWarps];
    float2 warp_sums[kWarps];
    int count, overflow;
    unsigned long long prefix;
    int wanted;
};

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
    return v;
}
// The threads' sums as one, in every thread: the largest reference first, so that each thread rescales its own once.
template <int THREADS>
__device__ __forceinline__ Sums join_block(Sums sums, float s2, Shared<THREADS>& sh) {
    constexpr int kWarps = THREADS / 32;
    float top = sums.reference;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
    if ((threadIdx.x & 31) == 0) sh.warp_top[threadIdx.x / 32] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kWarps; ++i) top = fmaxf(top, sh.warp_top[i]);
    if (sums.reference != top) sums.raise(top, s2);
    const float sum = warp_sum(sums.sum), weighted = warp_sum(sums.weighted);
    if ((threadIdx.x & 31) == 0) sh.warp_sums[threadIdx.x / 32] = make_float2(sum, weighted);
    __syncthreads();
    Sums all{top, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < kWarps; ++i) all.sum += sh.warp_sums[i].x, all.weighted += sh.warp_sums[i].y;
    return all;
}

// The n_best largest candidates of the part [v0, v1) of a row, exactly, by a radix selection over the 64 bits of key and column:
// for parts where more than kCandidates columns pass the threshold (thousands of equal scores, or all live ones within a few
// threads' reach).  Eight passes over the part, a byte each; at most n_best keys remain.
template <int THREADS, class T>
__device__ __noinline__ void select_exactly(const Row<T>& row, int v0, int v1, int n_best, Shared<THREADS>& sh) {
    constexpr int V = Row<T>::V;
    __syncthreads();
    if (threadIdx.x == 0) sh.prefix = 0, sh.wanted = n_best;
    for (int shift = 56; shift >= 0; shift -= 8) {
        for (int i = threadIdx.x; i < 256; i += THREADS) sh.histogram[i] = 0;
        __syncthreads();
        const unsigned long long prefix = sh.prefix;
        for (int base = v0; base < v1; base += THREADS) {  // the same number of rounds for all lanes of a warp
            const int v = base + (int)threadIdx.x;
            float val[V];
            unpack<T>(v < v1 ? row.load(v) : Row<T>::none(), val);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const uint32_t key = order_key(val[j]);
                const unsigned long long full = candidate(key, row.first_column(v) + j);
                const bool in = key != 0u && (shift == 56 || full >> (shift + 8) == prefix);
                const int digit = in ? (int)(full >> shift & 255u) : 256;
                const uint32_t same = __match_any_sync(~0u, digit);  // one addition for equal digits: equal scores share them
                if (in && __ffs(same) - 1 == (int)(threadIdx.x & 31)) atomicAdd(&sh.histogram[digit], __popc(same));
            }
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            int wanted = sh.wanted, digit = 255;
            while (digit > 0 && (int)sh.histogram[digit] < wanted) wanted -= (int)sh.histogram[digit--];
            sh.wanted = wanted;
            sh.prefix = prefix << 8 | (unsigned long long)digit;
        }
        __syncthreads();
    }
    if (threadIdx.x == 0) sh.count = 0;
    __syncthreads();
    const unsigned long long least = sh.prefix;  // the last one wanted (or 0: there are fewer)
    for (int v = v0 + (int)threadIdx.x; v < v1; v += THREADS) {
        float val[V];
        unpack<T>(row.load(v), val);
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const uint32_t key = order_key(val[j]);
            const unsigned long long full = candidate(key, row.first_column(v) + j);
            if (key != 0u && full >= least) {
                const int at = atomicAdd(&sh.count, 1);
                if (at < kCandidates) sh.key[at] = full;
            }
        }
    }
    __syncthreads();
}

// A threshold that at least `wanted` of the block's threads' keys reach, if so many are not 0 (else 1).  Each warp sorts its lanes'
// keys; the least of the W warps' ceil(wanted / W)-th ones is reached by enough, and of eight of them the largest that is is taken:
// within a tenth of `wanted` for scores in no order.  950 cycles for 256 keys; the exact one, found by bits, took one warp 2300.
template <int THREADS>
__device__ __forceinline__ uint32_t first_threshold(uint32_t mine, int wanted, Shared<THREADS>& sh) {
    constexpr int kWarps = THREADS / 32;
    const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;
    uint32_t sorted = mine;  // largest in lane 0
#pragma unroll
    for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
        for (int stride = size >> 1; stride > 0; stride >>= 1) {
            const uint32_t other = __shfl_xor_sync(~0u, sorted, stride);
            sorted = ((lane & size) == 0) == ((lane & stride) == 0) ? max(sorted, other) : min(sorted, other);
        }
    if (lane == (wanted + kWarps - 1) / kWarps - 1) sh.bound[warp] = sorted;
    if (threadIdx.x == 0) sh.count = sh.overflow = 0;
    __syncthreads();
    constexpr int kBounds = kWarps < 8 ? kWarps : 8;
    uint32_t bound[kBounds];
#pragma unroll
    for (int i = 0; i < kBounds; ++i) {
        bound[i] = sh.bound[i];
        const int reach = __popc(__ballot_sync(~0u, mine >= bound[i]));
        if (lane == i) sh.reach[i][warp] = reach;
    }
    __syncthreads();
    uint32_t threshold = max(1u, __reduce_min_sync(~0u, lane < kWarps ? sh.bound[lane] : ~0u));
#pragma unroll
    for (int i = 0; i < kBounds; ++i) {
        int reach = 0;
        if (kWarps <= 8) {
#pragma unroll
            for (int j = 0; j < kWarps; ++j) reach += sh.reach[i][j];
        } else {
            reach = __reduce_add_sync(~0u, lane < kWarps ? sh.reach[i][lane] : 0);
        }
        if (reach >= wanted) threshold = max(threshold, bound[i]);
    }
    return threshold;
}

// Adds what the lanes have to a list of the warp's, in order; returns the list's new length, past `most` without the rest.
template <class V>
__device__ __forceinline__ int append(V* list, int length, int most, bool mine, V v) {
    const uint32_t who = __ballot_sync(~0u, mine);
    const int at = length + __popc(who & ((1u << (threadIdx.x & 31)) - 1u));
    if (mine && at < most) list[at] = v;
    return length + __popc(who);
}
// Room for `length` more in the block's list of candidates, for all lanes of a warp.
template <int THREADS>
__device__ __forceinline__ int reserve(Shared<THREADS>& sh, int length) {
    int at = 0;
    if ((threadIdx.x & 31) == 0 && length) at = atomicAdd(&sh.count, length);
    return __shfl_sync(~0u, at, 0);
}

// The columns of the part [v0, v1) that reach the threshold, as the block's candidates.  Each warp looks through its own groups, of
// those that reach it through the vectors and their columns, its lanes sharing the groups' vectors out anew.  (Lists of the block's
// with one counter for all took 2000 cycles of additions to it for 130 groups.)
template <int THREADS, class T>
__device__ __forceinline__ void collect(const Row<T>& row, int v0, int v1, uint32_t threshold, Shared<THREADS>& sh) {
    using W = Words<T>;
    constexpr int V = Row<T>::V;
    const int lane = threadIdx.x & 31;
    float* const groups = sh.groups[threadIdx.x / 32];
    int* const hit = reinterpret_cast<int*>(groups);  // never longer than the groups that have been looked at
    constexpr int kWarpHits = Lists<THREADS>::kHits, kWarpKeys = Lists<THREADS>::kKeys;
    unsigned long long* const list = reinterpret_cast<unsigned long long*>(groups + kWarpHits);
    int hits = 0, at = 0, length = 0;
    for (int base = v0 + ((int)threadIdx.x & ~31); base < v1; base += THREADS * kGroup, at += 32) {  // the warp's first vector
        const float top = groups[at + lane];
        __syncwarp();
        hits = append(hit, hits, kWarpHits, base + lane < v1 && order_key(top) >= threshold, base + lane);
    }
    __syncwarp();
    for (int i = lane; i - lane < min(hits, kWarpHits) * kGroup; i += 64) {
        Vector raw[2];
        int v[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {  // two in flight
            v[u] = i + 32 * u < min(hits, kWarpHits) * kGroup ? hit[(i + 32 * u) / kGroup] + i % kGroup * THREADS : v1;
            raw[u] = v[u] < v1 ? row.load(v[u]) : Row<T>::none();
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const uint32_t top = W::larger(W::larger(raw[u].w[0], raw[u].w[1]), W::larger(raw[u].w[2], raw[u].w[3]));
            if (!__any_sync(~0u, order_key(W::largest(top)) >= threshold)) continue;
            float val[V];
            unpack<T>(raw[u], val);
            const int c0 = row.first_column(v[u]);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const uint32_t key = order_key(val[j]);
                length = append(list, length, kWarpKeys, key >= threshold, candidate(key, c0 + j));
            }
        }
    }
    __syncwarp();
    if (hits > kWarpHits || length > kWarpKeys) {
        if (lane == 0) sh.overflow = 1;
        return;
    }
    const int room = reserve(sh, length);
    for (int i = lane; i < length; i += 32)
        if (room + i < kCandidates) sh.key[room + i] = list[i];
}

// put(position, key) for the first n_best of the block's candidates in the order of their scores.  Each is compared with all, which
// all lanes read two at a time, by as many warps' threads as there are, a share each.  (131 of 256 threads' keys: 1960 cycles; a
// sort of 256 took 2330, lanes sharing a key 3800.)
template <int THREADS, class Put>
__device__ __forceinline__ void rank_candidates(int n_best, Shared<THREADS>& sh, Put&& put) {
    const int n = min(sh.count, kCandidates), pairs = (n + 1) / 2;
    sh.rank[threadIdx.x] = 0;
    if ((n & 1) && threadIdx.x == 0) sh.key[n] = 0;
    __syncthreads();
    const ulonglong2* const keys = reinterpret_cast<const ulonglong2*>(sh.key);
    const auto above = [&](unsigned long long key, int from, int to) {
        int rank = 0;
#pragma unroll 8
        for (int j = from; j < to; ++j) {
            const ulonglong2 two = keys[j];
            rank += (two.x > key) + (two.y > key);
        }
        return rank;
    };
    const int wide = (n + 31) & ~31;
    if (2 * wide <= THREADS && n > 0) {
        const int shares = THREADS / wide, share = (int)threadIdx.x / wide, i = (int)threadIdx.x % wide;
        const unsigned long long key = i < n ? sh.key[i] : 0ull;
        if (share < shares && i < n) atomicAdd(&sh.rank[i], above(key, pairs * share / shares, pairs * (share + 1) / shares));
        __syncthreads();
        if (share == 0 && i < n && sh.rank[i] < n_best) put(sh.rank[i], key);
    } else {
        for (int i = threadIdx.x; i < n; i += THREADS) {
            const unsigned long long key = sh.key[i];
            const int rank = above(key, 0, pairs);
            if (rank < n_best) put(rank, key);
        }
    }
    for (int i = n + (int)threadIdx.x; i < n_best; i += THREADS) put(i, 0ull);
}

// Where many candidates are left, those that reach a second threshold, found among them, stay.
template <int THREADS>
__device__ __forceinline__ void thin_candidates(int n_best, Shared<THREADS>& sh) {
    const int n = sh.count;
    if (n <= 2 * kMaxBest || n > kCandidates) return;
    __syncthreads();  // every thread has read the count, and the caller's tests of it are done: first_threshold sets it to 0
    constexpr int kPer = kCandidates / THREADS;
    unsigned long long key[kPer];
    uint32_t largest = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int at = i * THREADS + (int)threadIdx.x;
        key[i] = at < n ? sh.key[at] : 0ull;
        largest = max(largest, (uint32_t)(key[i] >> 32));
    }
    const uint32_t threshold = first_threshold<THREADS>(largest, n_best, sh);  // all have read their keys; the count starts anew
#pragma unroll
    for (int i = 0; i < kPer; ++i)
        if ((uint32_t)(key[i] >> 32) >= threshold) sh.key[atomicAdd(&sh.count, 1)] = key[i];
    __syncthreads();
}

struct RowResult {  // what is written once a row's sums are known
    float reference, log_total;
    bool empty;
};
__device__ __forceinline__ RowResult row_result(const Sums& total) { return RowResult{total.reference, log2f(total.sum), total.sum == 0.f}; }

struct Target {
    bool asked;
    float x;  // -inf: not live
    __device__ __forceinline__ Target() : asked(false), x(-INFINITY) {}
    template <class T>
    __device__ __forceinline__ Target(const Scores& s, size_t r, const Row<T>& row) {
        const int t = s.target ? s.target[r] : -1;
        asked = t >= 0 && t < s.cols;
        x = asked ? row.at(t) : -INFINITY;
    }
};
__device__ __forceinline__ void write_row(const Scores& s, const Out& out, size_t r, const Target& target, const Sums& total, const RowResult& res) {
    const float entropy = res.empty ? 0.f : (res.log_total - total.weighted / total.sum) * kLn2;
    const bool none = target.x == -INFINITY;
    out.log_prob[r] = !target.asked ? 0.f : none ? -INFINITY : fmaf(target.x - total.reference, s.scale, -res.log_total * kLn2);
    out.entropy[r] = entropy;
    out.log_sum[r] = res.empty ? -INFINITY : fmaf(total.reference, s.scale, res.log_total * kLn2);
    out.row_state[r] = make_float4(res.empty ? 0.f : total.reference, res.empty ? 0.f : res.log_total, entropy, none ? 0.f : 1.f);
}
__device__ __forceinline__ void write_best(const Scores& s, const Out& out, size_t r, const RowResult& res, int rank, unsigned long long key) {
    const size_t at = r * (size_t)out.n_best + rank;
    out.best_log_prob[at] = key ? fmaf(key_value((uint32_t)(key >> 32)) - res.reference, s.scale, -res.log_total * kLn2) : -INFINITY;
    out.best_index[at] = key ? (int32_t)(0xffffffffu - (uint32_t)key) : -1;
}

// A row is cut into parts of `vectors` 16-byte vectors, one block each; with more than one part their sums and lists meet in
// k_join_parts.
struct Parts {
    int count, vectors;
    float4* sums;               // [row, part]
    unsigned long long* keys;   // [row, part, n_best], best first, 0: none
};

// The sums of a part's vectors, four vectors a thread in flight at once and the next four while these are summed, in two halves:
//   d = (x - reference) s2, e = 2^d, sum += e, weighted += e d
// The difference is taken first: it is right, and never above 0, however far out the scores are.  (x s2 less the rounded product of the
// reference is one instruction, and off by half a unit of that product: from 2^31 on more than fp32 has exponents for.)  Scores are
// raised to kLow first, so that -inf makes no NaN of e d; where the largest score is no further than 2^64 above kLow that would count
// them, and add_exactly does the part again.
// Reading bounds fp32 rows (1024 x 200 001: 135 us, 6.1 TB/s; 132 without the next four vectors under way); of bf16 ones, twice the scores
// for the same bytes, the exponentials, 16 an SM and cycle, take 45 of 80 us beside the reading's 62 (2048 x 100 001: 5.1 TB/s; 81.4
// without the next four).
template <int THREADS, class T>
__device__ __forceinline__ Sums add_part(const Row<T>& row, int v0, int v1, float s2, float* groups, float& largest) {
    using W = Words<T>;
    float reference = W::kLow;  // until a score is above kLow nothing counts
    Pair sum = pair(0.f, 0.f), weighted = sum;
    const Pair scale = pair(s2, s2);
    int at = threadIdx.x & 31;
    Vector raw[kGroup];
    int base = v0 + (int)threadIdx.x;
    if (base < v1) row.template load_group<THREADS>(base, v1, raw);
    for (; base < v1; at += 32) {
        Vector next[kGroup];
        base += THREADS * kGroup;
        if (base < v1) row.template load_group<THREADS>(base, v1, next);
        uint32_t top = W::kNone;
#pragma unroll
        for (int u = 0; u < kGroup; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i) top = W::larger(top, raw[u].w[i]);
        const float above = W::largest(top);
        largest = fmaxf(largest, above);
        if (groups) groups[at] = above;
        if (above > reference) {
            const float d = fmaxf((reference - above) * s2, kFarBelow), c = ex2(d);
            weighted = mul_pair(pair(c, c), fma_pair(sum, pair(d, d), weighted));
            sum = mul_pair(pair(c, c), sum);
            reference = above;
        }
        const Pair back = pair(-reference, -reference);
#pragma unroll
        for (int u = 0; u < kGroup; ++u)
#pragma unroll
            for (int i = 0; i < 4; i += 3 - W::kPer) {
                const float2 x = W::kPer == 2 ? W::floats(W::raised(raw[u].w[i])) : make_float2(W::floats(W::raised(raw[u].w[i])).x, W::floats(W::raised(raw[u].w[(i + 1) % 4])).x);
                const Pair d = mul_pair(add_pair(pair(x.x, x.y), back), scale);
                const float2 power = halves(d);
                const Pair e = pair(ex2(power.x), ex2(power.y));
                sum = add_pair(sum, e);
                weighted = fma_pair(e, d, weighted);
            }
#pragma unroll
        for (int u = 0; u < kGroup; ++u) raw[u] = next[u];
    }
    const float total = halves(sum).x + halves(sum).y;
    if (reference == W::kLow) {  // nothing counts but a NaN, which has not moved the reference
        const float nan = total == total ? 0.f : total;
        return Sums{reference, nan, nan};
    }
    return Sums{reference, total, halves(weighted).x + halves(weighted).y};
}
template <int THREADS, class T>
__device__ __noinline__ Sums add_exactly(const Row<T>& row, int v0, int v1, float s2) {
    constexpr int V = Row<T>::V;
    Sums sums = none_yet();
    for (int v = v0 + (int)threadIdx.x; v < v1; v += THREADS) {
        float val[V];
        unpack<T>(row.load(v), val);
#pragma unroll
        for (int j = 0; j < V; ++j) sums.add(val[j], s2);
    }
    return sums;
}

// Blocks of 128 threads: eight to an SM, of fp32 scores seven, whose 72 registers hold both groups of vectors (600 x 5001: 6.2 us, with
// eight 7.7; 1000 x 12 001: 11.6 and 14.6).
template <class T, int THREADS>
static __global__ void __launch_bounds__(THREADS, THREADS == 128 ? (sizeof(T) == 4 ? 7 : 8) : 1024 / THREADS) k_log_probs(Scores s, Out out, Parts parts) {
    using W = Words<T>;
    __shared__ Shared<THREADS> sh;
    grid_dependency_sync();
    const uint32_t r = blockIdx.x / (uint32_t)parts.count, part = blockIdx.x % (uint32_t)parts.count;
    const Row<T> row(s, r);
    const int k = out.n_best;
    const int v0 = min(row.n_vectors, (int)part * parts.vectors), v1 = min(row.n_vectors, v0 + parts.vectors);
    const bool writes = threadIdx.x == THREADS - 32;  // not in the warp that looks for the threshold
    const Target target = writes && parts.count == 1 ? Target(s, r, row) : Target();
    float largest = -INFINITY;
    // a scale so large that kLow has no finite exponent is taken the long way
    const bool usual = fabsf(W::kLow * s.s2) < 1e37f;
    Sums total = join_block<THREADS>(add_part<THREADS, T>(row, v0, v1, s.s2, k > 0 ? sh.groups[threadIdx.x / 32] : nullptr, largest), s.s2, sh);
    if (!usual || !((total.reference - W::kLow) * s.s2 > 64.f) || total.reference >= 1e37f / s.s2) {
        __syncthreads();
        total = join_block<THREADS>(add_exactly<THREADS, T>(row, v0, v1, s.s2), s.s2, sh);
    }
    const RowResult res = row_result(total);
    if (writes) {
        if (parts.count == 1) write_row(s, out, r, target, total, res);
        else parts.sums[blockIdx.x] = make_float4(total.reference, total.sum, total.weighted, 0.f);
    }
    if (k == 0) return;
    const uint32_t threshold = first_threshold<THREADS>(order_key(largest), k, sh);
    collect<THREADS, T>(row, v0, v1, threshold, sh);
    __syncthreads();
    if (sh.overflow || sh.count > kCandidates) select_exactly<THREADS, T>(row, v0, v1, k, sh);
    else thin_candidates<THREADS>(k, sh);
    if (parts.count == 1) {
        rank_candidates<THREADS>(k, sh, [&](int rank, unsigned long long key) { write_best(s, out, r, res, rank, key); });
    } else {
        unsigned long long* const keys = parts.keys + (size_t)blockIdx.x * k;
        rank_candidates<THREADS>(k, sh, [&](int rank, unsigned long long key) { keys[rank] = key; });
    }
}

// One block a row: the parts' sums joined in order, and the best of their lists.
template <class T, int THREADS>
static __global__ void __launch_bounds__(THREADS) k_join_parts(Scores s, Out out, Parts parts) {
    __shared__ Shared<THREADS> sh;
    grid_dependency_sync();
    const size_t r = blockIdx.x;
    const Row<T> row(s, r);
    const bool writes = threadIdx.x == THREADS - 32;
    const Target target = writes ? Target(s, r, row) : Target();
    Sums sums = none_yet();
    for (int i = threadIdx.x; i < parts.count; i += THREADS) {
        const float4 p = parts.sums[r * parts.count + i];
        sums.join(Sums{p.x, p.y, p.z}, s.s2);
    }
    const Sums total = join_block<THREADS>(sums, s.s2, sh);
    const RowResult res = row_result(total);
    if (writes) write_row(s, out, r, target, total, res);
    const int k = out.n_best;
    if (k == 0) return;
    const unsigned long long* const keys = parts.keys + r * (size_t)parts.count * k;
    const int n = parts.count * k;
    // The lists are in order: `reach` parts whose `depth`-th best reaches a threshold have k keys that do.  The depth is such that
    // half of the parts are asked for; neighbouring parts go to different warps, which first_threshold takes as they come.
    const int depth = min(k, max(1, (2 * k + parts.count - 1) / parts.count)), reach = (k + depth - 1) / depth;
    uint32_t largest = 0;
    constexpr int kJoinWarps = THREADS / 32;
    for (int i = (threadIdx.x & 31) * kJoinWarps + threadIdx.x / 32; i < parts.count; i += THREADS)
        largest = max(largest, (uint32_t)(keys[(size_t)i * k + depth - 1] >> 32));
    const uint32_t threshold = first_threshold<THREADS>(largest, reach, sh);
    for (int i = threadIdx.x / 32; i < parts.count; i += kJoinWarps) {
        unsigned long long key[kMaxBest / 32];
        int length = 0;
#pragma unroll
        for (int j = 0; j < kMaxBest / 32; ++j) {
            const int at = 32 * j + ((int)threadIdx.x & 31);
            key[j] = at < k ? keys[(size_t)i * k + at] : 0ull;
        }
#pragma unroll
        for (int j = 0; j < kMaxBest / 32; ++j) length += __popc(__ballot_sync(~0u, (uint32_t)(key[j] >> 32) >= threshold));
        const int room = reserve(sh, length);  // the list is in order: those that reach it come first
#pragma unroll
        for (int j = 0; j < kMaxBest / 32; ++j) {
            const int at = 32 * j + ((int)threadIdx.x & 31);
            if (at < length && room + at < kCandidates) sh.key[room + at] = key[j];
        }
    }
    __syncthreads();
    thin_candidates<THREADS>(k, sh);
    if (sh.count > kCandidates) {
        // Equal scores in every part: the lists are in order, so a binary search over key and column finds how far each counts.
        unsigned long long low = (unsigned long long)threshold << 32, high = ~0ull;  // at least k keys are >= low
        while (low < high) {
            const unsigned long long mid = low + (high - low) / 2 + 1;
            __syncthreads();
            if (threadIdx.x == 0) sh.count = 0;
            __syncthreads();
            int mine = 0;
            for (int i = threadIdx.x; i < n; i += THREADS) mine += keys[i] >= mid;
            if (mine) atomicAdd(&sh.count, mine);
            __syncthreads();
            if (sh.count >= k) low = mid;
            else high = mid - 1;
        }
        __syncthreads();
        if (threadIdx.x == 0) sh.count = 0;
        __syncthreads();
        for (int i = threadIdx.x; i < n; i += THREADS)
            if (keys[i] >= low) sh.key[atomicAdd(&sh.count, 1)] = keys[i];  // keys differ: k of them
        __syncthreads();
    }
    rank_candidates<THREADS>(k, sh, [&](int rank, unsigned long long key) { write_best(s, out, r, res, rank, key); });
}

// The gradient: every score is read once and every gradient written once.
struct GradArgs {
    const float4* row_state;
    const float* grad_log_prob;
    const float* grad_entropy;
    const int32_t* best_index;
    const float* grad_best;
    void* grad;
    long long grad_stride;
    int n_best;
    int blocks_per_row;
    uint32_t rows;
};
constexpr int kGradThreads = 256;

// One block for kGradThreads * kGroup vectors of a row, the rows from the last to the first: what the forward pass read last may
// still be in L2.  The vectors are those of the scores' memory: a gradient that is as far from a 16-byte boundary as the scores
// are is written as it is read.  Bound by memory: 2048 x 100 001 bf16 scores 137 us, half as many fp32 ones 148 (127 at the copy rate).
// Five blocks an SM serve both types: with registers for four 148 and 135, for six and a few spills 134 and 153.
template <class T>
static __global__ void __launch_bounds__(kGradThreads, 5) k_log_probs_grad(Scores s, GradArgs g) {
    constexpr int V = Row<T>::V;
    __shared__ float s_sum;
    __shared__ float s_best[kMaxBest];
    __shared__ int s_column[kMaxBest];
    grid_dependency_sync();
    const uint32_t r = g.rows - 1u - blockIdx.x / (uint32_t)g.blocks_per_row;
    const Row<T> row(s, r);
    T* out = static_cast<T*>(g.grad) + (long long)r * g.grad_stride;
    const bool together = (int)((reinterpret_cast<uintptr_t>(out) & 15u) / sizeof(T)) == row.shift;
    const int n_vectors = (s.cols + row.shift + V - 1) / V;
    const int v0 = (int)(blockIdx.x % (uint32_t)g.blocks_per_row) * kGradThreads * kGroup, v1 = min(n_vectors, v0 + kGradThreads * kGroup);
    // this block's alternatives: their scores are taken before any gradient is written (it may take the scores' place)
    const int i = threadIdx.x;
    int column = -1;
    float x_best = 0.f, g_best = 0.f;
    if (g.grad_best && i < g.n_best) {
        column = g.best_index[(size_t)r * g.n_best + i];
        if (column >= 0 && column < row.cols) {
            g_best = g.grad_best[(size_t)r * g.n_best + i];
            if (column >= max(0, row.first_column(v0)) && column < row.first_column(v1)) x_best = as_float(row.x[column]);
        } else column = -1;
    }
    Vector raw[kGroup];
#pragma unroll
    for (int u = 0; u < kGroup; ++u) {
        const int v = v0 + u * kGradThreads + (int)threadIdx.x;
        raw[u] = v < v1 ? row.load(v) : Row<T>::none();
    }
    const float4 state = g.row_state[r];
    const int target = s.target ? s.target[r] : -1;
    const float g_target = state.w != 0.f && g.grad_log_prob ? g.grad_log_prob[r] : 0.f;
    const float g_entropy = g.grad_entropy ? g.grad_entropy[r] : 0.f;
    float total = g_target;
    if (g.grad_best) {
        if (i < kMaxBest) s_best[i] = g_best, s_column[i] = column;
        __syncthreads();
        if (i < 32) {
            float t = 0.f;
            for (int j = i; j < kMaxBest; j += 32) t += s_best[j];
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(~0u, t, o);
            if (i == 0) s_sum = t;
        }
        __syncthreads();
        total += s_sum;
    }
    // -scale p (G + g_H (log p + entropy)) with log2 p = (x - reference) s2 - log2 S, the difference first as in the forward pass
    const float slope = -s.scale * g_entropy * kLn2, level = -s.scale * fmaf(g_entropy, state.z, total);
    auto gradient = [&](float x) {
        const float d = max_or_nan(fmaf(x - state.x, s.s2, -state.y), kFarBelow);
        return x == -INFINITY ? 0.f : ex2(d) * fmaf(slope, d, level);
    };
#pragma unroll
    for (int u = 0; u < kGroup; ++u) {
        const int v = v0 + u * kGradThreads + (int)threadIdx.x;
        if (v >= v1) break;
        float val[V];
        unpack<T>(raw[u], val);
        const int c0 = row.first_column(v);
        const Pair scale = pair(s.s2, s.s2), a = pair(-state.x, -state.x), b = pair(-state.y, -state.y), k1 = pair(slope, slope), k0 = pair(level, level);
#pragma unroll
        for (int j = 0; j < V; j += 2) {
            float2 d = halves(fma_pair(add_pair(pair(val[j], val[j + 1]), a), scale, b));
            d.x = max_or_nan(d.x, kFarBelow), d.y = max_or_nan(d.y, kFarBelow);
            const float2 got = halves(mul_pair(pair(ex2(d.x), ex2(d.y)), fma_pair(k1, pair(d.x, d.y), k0)));
            val[j] = val[j] == -INFINITY ? 0.f : got.x;
            val[j + 1] = val[j + 1] == -INFINITY ? 0.f : got.y;
        }
        const unsigned at = (unsigned)(target - c0);
        if (at < (unsigned)V && target >= 0 && g_target != 0.f) {
#pragma unroll
            for (int j = 0; j < V; ++j) val[j] += at == (unsigned)j ? s.scale * g_target : 0.f;
        }
        if (together && c0 >= 0 && c0 + V <= s.cols) {
            *reinterpret_cast<uint4*>(out + c0) = pack(val, T());
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (c0 + j >= 0 && c0 + j < s.cols) store_rounded(out + c0 + j, val[j]);
        }
    }
    if (!g.grad_best) return;
    __syncthreads();
    if (column >= max(0, row.first_column(v0)) && column < row.first_column(v1)) {  // the whole of what this column gets, once more
        float given = column == target ? g_target : 0.f;
        for (int j = 0; j < g.n_best; ++j) given += s_column[j] == column ? s_best[j] : 0.f;
        store_rounded(out + column, gradient(x_best) + s.scale * given);
    }
}

}  // namespace lp
}  // namespace kge
