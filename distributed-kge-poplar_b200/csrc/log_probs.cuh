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
// Groups of a thread in one part of a row: their largest scores are kept in shared memory.
template <int THREADS>
constexpr int kGroupsPerThread = THREADS == 128 ? 1 : 16;
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
template <int THREADS>
struct Shared {
    float group_max[THREADS == 128 ? 128 * kGroup : THREADS * kGroupsPerThread<THREADS>];  // later a list of vectors
    alignas(16) unsigned long long key[kCandidates + 1];
    int hit[kCandidates];
    uint16_t bin[THREADS];
    uint32_t histogram[256];
    float warp_top[THREADS / 32];
    float2 warp_sums[THREADS / 32];
    uint32_t threshold;
    int hits, vectors, count;
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

// A threshold that `wanted` of the block's threads' keys reach, if so many are not 0: their wanted-th largest, cut to its upper 16
// bits (a few more reach that).  One warp finds it bit by bit: 16 counts of the keys that reach a candidate, 12 instructions each,
// where ranking 256 keys against one another took as many as all sums of a row of 32 000 scores.
template <int THREADS>
__device__ __forceinline__ uint32_t first_threshold(uint32_t mine, int wanted, Shared<THREADS>& sh) {
    sh.bin[threadIdx.x] = (uint16_t)(mine >> 16);
    if (threadIdx.x == 0) sh.hits = sh.vectors = sh.count = 0;
    __syncthreads();
    if (threadIdx.x < 32) {
        constexpr int kPer = THREADS / 32;
        uint32_t bin[kPer], found = 0;
#pragma unroll
        for (int i = 0; i < kPer; ++i) bin[i] = sh.bin[i * 32 + threadIdx.x];
#pragma unroll 1
        for (uint32_t bit = 0x8000u; bit; bit >>= 1) {
            uint32_t reach = 0;
#pragma unroll
            for (int i = 0; i < kPer; ++i) reach += bin[i] >= (found | bit);
            if ((int)__reduce_add_sync(~0u, reach) >= wanted) found |= bit;
        }
        if (threadIdx.x == 0) sh.threshold = max(found << 16, 1u);
    }
    __syncthreads();
    return sh.threshold;
}

// put(position, key) for the first n_best of the block's candidates in the order of their scores.  Each is compared with all, by
// several threads where there are more threads than candidates.
template <int THREADS, class Put>
__device__ __forceinline__ void rank_candidates(int n_best, Shared<THREADS>& sh, Put&& put) {
    const int n = min(sh.count, kCandidates);
    if ((n & 1) && threadIdx.x == 0) sh.key[n] = 0;
    __syncthreads();
    const ulonglong2* const keys = reinterpret_cast<const ulonglong2*>(sh.key);
    const int pairs = (n + 1) / 2;
    const int share = n <= THREADS / 4 ? 4 : n <= THREADS / 2 ? 2 : 1;  // threads to a candidate, lanes side by side
    const int from = (int)threadIdx.x % share, step = share;
    for (int base = 0; base < n; base += THREADS / share) {
        const int i = base + (int)threadIdx.x / share;
        const unsigned long long key = i < n ? sh.key[i] : ~0ull;
        int rank = 0;
#pragma unroll 4
        for (int j = from; j < pairs; j += step) {
            const ulonglong2 two = keys[j];
            rank += (two.x > key) + (two.y > key);
        }
        for (int o = 1; o < share; o <<= 1) rank += __shfl_xor_sync(~0u, rank, o);
        if (i < n && from == 0 && rank < n_best) put(rank, key);
    }
    for (int i = n + (int)threadIdx.x; i < n_best; i += THREADS) put(i, 0ull);
}

// Where many candidates are left, those that reach a second threshold, found among them, stay.
template <int THREADS>
__device__ __forceinline__ void thin_candidates(int n_best, Shared<THREADS>& sh) {
    const int n = sh.count;
    if (n <= 2 * kMaxBest || n > kCandidates) return;
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

template <class T>
__device__ __forceinline__ void write_row(const Scores& s, const Out& out, size_t r, const Row<T>& row, const Sums& total, const RowResult& res) {
    const float entropy = res.empty ? 0.f : (res.log_total - total.weighted / total.sum) * kLn2;
    const int t = s.target ? s.target[r] : -1;
    float log_prob = 0.f, counted = 0.f;
    if (t >= 0 && t < s.cols) {
        const float x = row.at(t);
        log_prob = x == -INFINITY ? -INFINITY : fmaf(x - total.reference, s.scale, -res.log_total * kLn2);
        counted = x == -INFINITY ? 0.f : 1.f;
    }
    out.log_prob[r] = log_prob;
    out.entropy[r] = entropy;
    out.log_sum[r] = res.empty ? -INFINITY : fmaf(total.reference, s.scale, res.log_total * kLn2);
    out.row_state[r] = make_float4(res.empty ? 0.f : total.reference, res.empty ? 0.f : res.log_total, entropy, counted);
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

// The sums of a part's vectors, four vectors a thread in flight at once:
//   d = x s2 - r2 (one fused multiply-add), e = 2^d, sum += e, weighted += e d
// with r2 the reference times s2, rounded: whatever it is off by, all terms are, and it is taken out exactly at the end.  Scores
// are raised to kLow first, so that -inf makes no NaN of e d; where the largest score is no further than 2^64 above kLow that
// would count them, and add_exactly does the part again.
template <int THREADS, class T>
__device__ __forceinline__ Sums add_part(const Row<T>& row, int v0, int v1, float s2, bool keep_groups, float* group_max, float& largest) {
    using W = Words<T>;
    float reference = W::kLow, r2 = 0.f;  // until a score is above kLow nothing counts
    float sum[2] = {}, weighted[2] = {};
    int group = threadIdx.x;
    for (int base = v0 + (int)threadIdx.x; base < v1; base += THREADS * kGroup, group += THREADS) {
        Vector raw[kGroup];
        row.template load_group<THREADS>(base, v1, raw);
        uint32_t top = W::kNone;
#pragma unroll
        for (int u = 0; u < kGroup; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i) top = W::larger(top, raw[u].w[i]);
        const float above = W::largest(top);
        largest = fmaxf(largest, above);
        if (keep_groups) group_max[group] = above;
        if (above > reference) {
            reference = above;
            const float to = above * s2, d = fminf(fmaxf(r2 - to, kFarBelow), 0.f), c = ex2(d);
            weighted[0] = c * fmaf(sum[0], d, weighted[0]), weighted[1] = c * fmaf(sum[1], d, weighted[1]);
            sum[0] *= c, sum[1] *= c;
            r2 = to;
        }
#pragma unroll
        for (int u = 0; u < kGroup; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 x = W::floats(W::raised(raw[u].w[i]));
#pragma unroll
                for (int j = 0; j < W::kPer; ++j) {
                    const int h = W::kPer == 2 ? j : i & 1;
                    const float d = fmaf(j ? x.y : x.x, s2, -r2), e = ex2(d);
                    sum[h] += e;
                    weighted[h] = fmaf(e, d, weighted[h]);
                }
            }
    }
    if (reference == W::kLow) return Sums{reference, 0.f, 0.f};
    const float off = fmaf(reference, s2, -r2), c = ex2(-off), total = sum[0] + sum[1];
    return Sums{reference, c * total, c * fmaf(-off, total, weighted[0] + weighted[1])};
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

template <class T, int THREADS>
static __global__ void __launch_bounds__(THREADS, 1024 / THREADS) k_log_probs(Scores s, Out out, Parts parts) {
    using W = Words<T>;
    constexpr int V = Row<T>::V;
    __shared__ Shared<THREADS> sh;
    grid_dependency_sync();
    const uint32_t r = blockIdx.x / (uint32_t)parts.count, part = blockIdx.x % (uint32_t)parts.count;
    const Row<T> row(s, r);
    const int k = out.n_best;
    const int v0 = min(row.n_vectors, (int)part * parts.vectors), v1 = min(row.n_vectors, v0 + parts.vectors);
    float largest = -INFINITY;
    // a scale so large that kLow has no finite exponent is taken the long way
    const bool usual = fabsf(W::kLow * s.s2) < 1e37f;
    Sums total = join_block<THREADS>(add_part<THREADS, T>(row, v0, v1, s.s2, k > 0, sh.group_max, largest), s.s2, sh);
    if (!usual || !((total.reference - W::kLow) * s.s2 > 64.f) || total.reference >= 1e37f / s.s2) {
        __syncthreads();
        total = join_block<THREADS>(add_exactly<THREADS, T>(row, v0, v1, s.s2), s.s2, sh);
    }
    const RowResult res = row_result(total);
    if (threadIdx.x == 0) {
        if (parts.count == 1) write_row(s, out, r, row, total, res);
        else parts.sums[blockIdx.x] = make_float4(total.reference, total.sum, total.weighted, 0.f);
    }
    if (k == 0) return;
    const uint32_t threshold = first_threshold<THREADS>(order_key(largest), k, sh);
    // the groups that reach it, of these the vectors, of these the columns: each time a list that the block shares out anew
    int group = threadIdx.x;
    for (int base = v0 + (int)threadIdx.x; base < v1; base += THREADS * kGroup, group += THREADS)
        if (order_key(sh.group_max[group]) >= threshold) {
            const int at = atomicAdd(&sh.hits, 1);
            if (at < kCandidates) sh.hit[at] = base;
        }
    __syncthreads();
    const int hits = sh.hits;
    if (hits <= kCandidates) {
        int* const reached = reinterpret_cast<int*>(sh.group_max);
        constexpr int kMost = kGroup * (kCandidates < THREADS * kGroupsPerThread<THREADS> ? kCandidates : THREADS * kGroupsPerThread<THREADS>);
        static_assert(sizeof(sh.group_max) >= sizeof(int) * kMost, "a list of vectors takes the groups' place");
        for (int i = threadIdx.x; i < hits * kGroup; i += THREADS) {
            const int v = sh.hit[i / kGroup] + i % kGroup * THREADS;
            if (v >= v1) continue;
            const Vector raw = row.load(v);
            const float top = W::largest(W::larger(W::larger(raw.w[0], raw.w[1]), W::larger(raw.w[2], raw.w[3])));
            if (order_key(top) >= threshold) reached[atomicAdd(&sh.vectors, 1)] = v;
        }
        __syncthreads();
        const int columns = sh.vectors * V;
        for (int i = threadIdx.x; i < columns; i += THREADS) {
            const int c = row.first_column(reached[i / V]) + i % V;
            const uint32_t key = c >= 0 ? order_key(row.at(c)) : 0u;
            if (key >= threshold) {
                const int at = atomicAdd(&sh.count, 1);
                if (at < kCandidates) sh.key[at] = candidate(key, c);
            }
        }
        __syncthreads();
    }
    if (hits > kCandidates || sh.count > kCandidates) select_exactly<THREADS, T>(row, v0, v1, k, sh);
    else thin_candidates<THREADS>(k, sh);
    if (parts.count == 1) {
        rank_candidates<THREADS>(k, sh, [&](int rank, unsigned long long key) { write_best(s, out, r, res, rank, key); });
    } else {
        unsigned long long* const keys = parts.keys + (size_t)blockIdx.x * k;
        rank_candidates<THREADS>(k, sh, [&](int rank, unsigned long long key) { keys[rank] = key; });
    }
}

// One block a row: the parts' sums joined in order, and the best of their lists.
constexpr int kJoinThreads = 256;
template <class T>
static __global__ void __launch_bounds__(kJoinThreads) k_join_parts(Scores s, Out out, Parts parts) {
    __shared__ Shared<kJoinThreads> sh;
    grid_dependency_sync();
    const size_t r = blockIdx.x;
    const Row<T> row(s, r);
    Sums sums = none_yet();
    for (int i = threadIdx.x; i < parts.count; i += kJoinThreads) {
        const float4 p = parts.sums[r * parts.count + i];
        sums.join(Sums{p.x, p.y, p.z}, s.s2);
    }
    const Sums total = join_block<kJoinThreads>(sums, s.s2, sh);
    const RowResult res = row_result(total);
    if (threadIdx.x == 0) write_row(s, out, r, row, total, res);
    const int k = out.n_best;
    if (k == 0) return;
    const unsigned long long* const keys = parts.keys + r * (size_t)parts.count * k;
    const int n = parts.count * k;
    // The lists are in order: `reach` parts whose `depth`-th best reaches a threshold have k keys that do.  The depth is such that
    // half of the parts are asked for, and a warp follows a list as far as it reaches.
    const int depth = min(k, max(1, (2 * k + parts.count - 1) / parts.count)), reach = (k + depth - 1) / depth;
    uint32_t largest = 0;
    for (int i = threadIdx.x; i < parts.count; i += kJoinThreads) largest = max(largest, (uint32_t)(keys[(size_t)i * k + depth - 1] >> 32));
    const uint32_t threshold = first_threshold<kJoinThreads>(largest, reach, sh);
    for (int i = threadIdx.x / 32; i < parts.count; i += kJoinThreads / 32)
        for (int j = threadIdx.x & 31; j < k; j += 32) {
            const unsigned long long key = keys[(size_t)i * k + j];
            if ((uint32_t)(key >> 32) < threshold) break;
            const int at = atomicAdd(&sh.count, 1);
            if (at < kCandidates) sh.key[at] = key;
        }
    __syncthreads();
    thin_candidates<kJoinThreads>(k, sh);
    if (sh.count > kCandidates) {
        // Equal scores in every part: the lists are in order, so a binary search over key and column finds how far each counts.
        unsigned long long low = (unsigned long long)threshold << 32, high = ~0ull;  // at least k keys are >= low
        while (low < high) {
            const unsigned long long mid = low + (high - low) / 2 + 1;
            __syncthreads();
            if (threadIdx.x == 0) sh.count = 0;
            __syncthreads();
            int mine = 0;
            for (int i = threadIdx.x; i < n; i += kJoinThreads) mine += keys[i] >= mid;
            if (mine) atomicAdd(&sh.count, mine);
            __syncthreads();
            if (sh.count >= k) low = mid;
            else high = mid - 1;
        }
        __syncthreads();
        if (threadIdx.x == 0) sh.count = 0;
        __syncthreads();
        for (int i = threadIdx.x; i < n; i += kJoinThreads)
            if (keys[i] >= low) sh.key[atomicAdd(&sh.count, 1)] = keys[i];  // keys differ: k of them
        __syncthreads();
    }
    rank_candidates<kJoinThreads>(k, sh, [&](int rank, unsigned long long key) { write_best(s, out, r, res, rank, key); });
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
// are is written as it is read.
template <class T>
static __global__ void __launch_bounds__(kGradThreads, 4) k_log_probs_grad(Scores s, GradArgs g) {
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
    // -scale p (G + g_H (log p + entropy)) with log2 p = (x s2 - r2) - (log2 S + what r2 = reference s2 was rounded by); where the
    // reference has no finite r2 (scores of the type's lowest value) from the difference of the scores
    const float r2 = state.x * s.s2;
    const bool usual = fabsf(r2) < 1e37f;
    const float l2 = usual ? state.y + fmaf(state.x, s.s2, -r2) : state.y;
    const float slope = -s.scale * g_entropy * kLn2, level = -s.scale * fmaf(g_entropy, state.z, total);
    auto gradient = [&](float x) {
        const float d = max_or_nan((usual ? fmaf(x, s.s2, -r2) : (x - state.x) * s.s2) - l2, kFarBelow);
        return x == -INFINITY ? 0.f : ex2(d) * fmaf(slope, d, level);
    };
#pragma unroll
    for (int u = 0; u < kGroup; ++u) {
        const int v = v0 + u * kGradThreads + (int)threadIdx.x;
        if (v >= v1) break;
        float val[V];
        unpack<T>(raw[u], val);
        const int c0 = row.first_column(v);
        if (usual) {
            const Pair scale = pair(s.s2, s.s2), a = pair(-r2, -r2), b = pair(-l2, -l2), k1 = pair(slope, slope), k0 = pair(level, level);
#pragma unroll
            for (int j = 0; j < V; j += 2) {
                float2 d = halves(add_pair(fma_pair(pair(val[j], val[j + 1]), scale, a), b));
                d.x = max_or_nan(d.x, kFarBelow), d.y = max_or_nan(d.y, kFarBelow);
                const float2 got = halves(mul_pair(pair(ex2(d.x), ex2(d.y)), fma_pair(k1, pair(d.x, d.y), k0)));
                val[j] = val[j] == -INFINITY ? 0.f : got.x;
                val[j + 1] = val[j + 1] == -INFINITY ? 0.f : got.y;
            }
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) val[j] = gradient(val[j]);
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
