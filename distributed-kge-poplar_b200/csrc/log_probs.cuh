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

constexpr int kThreads = 512;
constexpr int kMaxBest = 128;
constexpr int kBins = 256;          // thread pairs whose largest scores give the first threshold
constexpr int kCandidates = 1024;
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

__device__ __forceinline__ float as_float(float v) { return v; }
__device__ __forceinline__ float as_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float as_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void unpack(const uint4& raw, float (&x)[4], float) {
    x[0] = __uint_as_float(raw.x), x[1] = __uint_as_float(raw.y), x[2] = __uint_as_float(raw.z), x[3] = __uint_as_float(raw.w);
}
__device__ __forceinline__ void unpack(const uint4& raw, float (&x)[8], __nv_bfloat16) {
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) x[2 * i] = __uint_as_float(w[i] << 16), x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
}
__device__ __forceinline__ void unpack(const uint4& raw, float (&x)[8], __half) {
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        x[2 * i] = v.x, x[2 * i + 1] = v.y;
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
__device__ __forceinline__ void store_rounded(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_rounded(__half* p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void store_rounded(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

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
    __device__ __forceinline__ void load(int v, float (&val)[V]) const {
        const int c0 = first_column(v);
        if (whole(v)) {
            unpack(*reinterpret_cast<const uint4*>(x + c0), val, T());
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) val[j] = c0 + j >= 0 && c0 + j < cols ? as_float(x[c0 + j]) : -INFINITY;
        }
        if (mask) {
            if (whole(v) && (reinterpret_cast<uintptr_t>(mask + c0) & 3u) == 0) {
#pragma unroll
                for (int q = 0; q < V / 4; ++q) {
                    const uint32_t m = *reinterpret_cast<const uint32_t*>(mask + c0 + 4 * q);
#pragma unroll
                    for (int j = 0; j < 4; ++j) val[4 * q + j] = (m >> (8 * j)) & 0xffu ? val[4 * q + j] : -INFINITY;
                }
            } else {
#pragma unroll
                for (int j = 0; j < V; ++j) val[j] = c0 + j >= 0 && c0 + j < cols && mask[c0 + j] ? val[j] : -INFINITY;
            }
        }
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
};
__device__ __forceinline__ Sums shuffled(const Sums& s, int lane_mask) {
    return Sums{__shfl_xor_sync(~0u, s.reference, lane_mask), __shfl_xor_sync(~0u, s.sum, lane_mask), __shfl_xor_sync(~0u, s.weighted, lane_mask)};
}

// The sums of a vector's columns join the thread's; the reference follows their largest.  Returns that largest score.
template <int V>
__device__ __forceinline__ float add_vector(Sums& s, const float (&val)[V], float s2) {
    float largest = val[0];
#pragma unroll
    for (int j = 1; j < V; ++j) largest = fmaxf(largest, val[j]);
    if (largest > s.reference) s.raise(largest, s2);
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const float d = max_or_nan((val[j] - s.reference) * s2, kFarBelow), e = ex2(d);
        s.sum += e;
        s.weighted = fmaf(e, d, s.weighted);
    }
    return largest;
}

struct Shared {
    unsigned long long key[kCandidates];
    uint32_t bin[kBins];
    uint32_t histogram[256];
    Sums warp_sums[kThreads / 32];
    Sums sums;
    uint32_t threshold;
    int count;
    unsigned long long prefix;
    int wanted;
};

// The n_best largest candidates of the row, exactly, by a radix selection over the 64 bits of key and column: for rows where
// more than kCandidates columns pass the threshold (thousands of equal scores, or all live ones within a few threads' reach).
// Eight passes over the row, a byte each; at most n_best keys remain.
template <class T>
__device__ void select_exactly(const Row<T>& row, int v0, int v1, int n_best, Shared& sh) {
    constexpr int V = Row<T>::V;
    if (threadIdx.x == 0) sh.prefix = 0, sh.wanted = n_best;
    for (int shift = 56; shift >= 0; shift -= 8) {
        for (int i = threadIdx.x; i < 256; i += kThreads) sh.histogram[i] = 0;
        __syncthreads();
        const unsigned long long prefix = sh.prefix;
        for (int base = v0; base < v1; base += kThreads) {  // the same number of rounds for all lanes of a warp
            const int v = base + (int)threadIdx.x;
            float val[V];
            if (v < v1) row.load(v, val);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const uint32_t key = v < v1 ? order_key(val[j]) : 0u;
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
    for (int v = v0 + (int)threadIdx.x; v < v1; v += kThreads) {
        float val[V];
        row.load(v, val);
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

// One block a row.
template <class T>
static __global__ void __launch_bounds__(kThreads) k_log_probs(Scores s, Out out) {
    constexpr int V = Row<T>::V;
    __shared__ Shared sh;
    const size_t r = blockIdx.x;
    const Row<T> row(s, r);
    Sums sums{kNoReference, 0.f, 0.f};
    float largest = -INFINITY;
    for (int v = threadIdx.x; v < row.n_vectors; v += kThreads) {
        float val[V];
        row.load(v, val);
        largest = fmaxf(largest, add_vector(sums, val, s.s2));
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sums.join(shuffled(sums, o), s.s2);
    if ((threadIdx.x & 31) == 0) sh.warp_sums[threadIdx.x / 32] = sums;
    const uint32_t mine = order_key(largest), other = __shfl_xor_sync(~0u, mine, 1);
    if ((threadIdx.x & 1) == 0) sh.bin[threadIdx.x / 2] = max(mine, other);
    if (threadIdx.x == 0) sh.count = 0, sh.threshold = 0;
    __syncthreads();
    if (threadIdx.x < 32) {
        Sums t = threadIdx.x < kThreads / 32 ? sh.warp_sums[threadIdx.x] : Sums{kNoReference, 0.f, 0.f};
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) t.join(shuffled(t, o), s.s2);
        if (threadIdx.x == 0) sh.sums = t;
    }
    __syncthreads();
    const Sums total = sh.sums;
    const bool empty = total.sum == 0.f;
    const float log_total = log2f(total.sum);
    if (threadIdx.x == 0) {
        const float entropy = empty ? 0.f : (log_total - total.weighted / total.sum) * kLn2;
        const int t = s.target ? s.target[r] : -1;
        float log_prob = 0.f, counted = 0.f;
        if (t >= 0 && t < s.cols) {
            const float x = row.at(t);
            log_prob = x == -INFINITY ? -INFINITY : fmaf(x - total.reference, s.scale, -log_total * kLn2);
            counted = x == -INFINITY ? 0.f : 1.f;
        }
        out.log_prob[r] = log_prob;
        out.entropy[r] = entropy;
        out.log_sum[r] = empty ? -INFINITY : fmaf(total.reference, s.scale, log_total * kLn2);
        out.row_state[r] = make_float4(empty ? 0.f : total.reference, empty ? 0.f : log_total, entropy, counted);
    }
    const int k = out.n_best;
    if (k == 0) return;
    // The k-th largest of the bins' largest scores is no larger than the row's k-th: few columns reach it (half as many again
    // as the list is long at 128 of 256 bins).
    if (threadIdx.x < kBins) {
        const uint32_t key = sh.bin[threadIdx.x];
        int above = 0;
        for (int j = 0; j < kBins; ++j) above += sh.bin[j] > key || (sh.bin[j] == key && j < (int)threadIdx.x);
        if (above == k - 1) sh.threshold = key;
    }
    __syncthreads();
    const uint32_t threshold = max(sh.threshold, 1u);
    for (int v = threadIdx.x; v < row.n_vectors; v += kThreads) {
        float val[V];
        row.load(v, val);
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const uint32_t key = order_key(val[j]);
            if (key >= threshold) {
                const int at = atomicAdd(&sh.count, 1);
                if (at < kCandidates) sh.key[at] = candidate(key, row.first_column(v) + j);
            }
        }
    }
    __syncthreads();
    if (sh.count > kCandidates) select_exactly<T>(row, 0, row.n_vectors, k, sh);
    const int n = min(sh.count, kCandidates);
    float* best = out.best_log_prob + r * (size_t)k;
    int32_t* index = out.best_index + r * (size_t)k;
    for (int i = threadIdx.x; i < n; i += kThreads) {
        const unsigned long long key = sh.key[i];
        int rank = 0;
        for (int j = 0; j < n; ++j) rank += sh.key[j] > key;
        if (rank < k) {
            best[rank] = fmaf(key_value((uint32_t)(key >> 32)) - total.reference, s.scale, -log_total * kLn2);
            index[rank] = (int32_t)(0xffffffffu - (uint32_t)key);
        }
    }
    for (int i = n + (int)threadIdx.x; i < k; i += kThreads) best[i] = -INFINITY, index[i] = -1;
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
};
constexpr int kGradThreads = 256;
constexpr int kGradVectors = 4;  // a thread's

// One block for kGradThreads * kGradVectors vectors of a row.  The vectors are those of the gradient's memory: a gradient that
// is as far from a 16-byte boundary as the scores are is written as it is read.
template <class T>
static __global__ void __launch_bounds__(kGradThreads) k_log_probs_grad(Scores s, GradArgs g) {
    constexpr int V = Row<T>::V;
    const uint32_t r = blockIdx.x / (uint32_t)g.blocks_per_row;
    __shared__ float s_sum;
    const Row<T> row(s, r);
    const int live_cols = row.cols;
    T* out = static_cast<T*>(g.grad) + (long long)r * g.grad_stride;
    const bool together = (int)((reinterpret_cast<uintptr_t>(out) & 15u) / sizeof(T)) == row.shift;
    const int n_vectors = (s.cols + row.shift + V - 1) / V;
    const int v0 = (int)(blockIdx.x % (uint32_t)g.blocks_per_row) * kGradThreads * kGradVectors, v1 = min(n_vectors, v0 + kGradThreads * kGradVectors);
    const float4 state = g.row_state[r];
    const int target = s.target ? s.target[r] : -1;
    const float g_target = state.w != 0.f && g.grad_log_prob ? g.grad_log_prob[r] : 0.f;
    const float g_entropy = g.grad_entropy ? g.grad_entropy[r] : 0.f;
    // this block's alternatives: their scores are taken before any gradient is written (it may take the scores' place)
    const int i = threadIdx.x;
    int column = -1;
    float x_best = 0.f, g_best = 0.f;
    if (g.grad_best && i < g.n_best) {
        column = g.best_index[(size_t)r * g.n_best + i];
        if (column >= 0 && column < live_cols) {
            g_best = g.grad_best[(size_t)r * g.n_best + i];
            x_best = row.at(column);
            if (x_best == -INFINITY) g_best = 0.f, column = -1;
        } else column = -1;
    }
    __shared__ float s_best[kMaxBest];
    __shared__ int s_column[kMaxBest];
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
    auto gradient = [&](float x) {
        const float d = max_or_nan(fmaf(x - state.x, s.s2, -state.y), kFarBelow), p = ex2(d);
        return -s.scale * p * (total + g_entropy * fmaf(d, kLn2, state.z));
    };
    for (int u = 0; u < kGradVectors; ++u) {
        const int v = v0 + u * kGradThreads + (int)threadIdx.x;
        if (v >= v1) break;
        float val[V];
        row.load(v, val);
        const int c0 = row.first_column(v);
#pragma unroll
        for (int j = 0; j < V; ++j) val[j] = val[j] == -INFINITY ? 0.f : gradient(val[j]);
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
        float got = gradient(x_best);
        float given = column == target ? g_target : 0.f;
        for (int j = 0; j < g.n_best; ++j) given += s_column[j] == column ? s_best[j] : 0.f;
        got += s.scale * given;
        store_rounded(out + column, got);
    }
}

}  // namespace lp
}  // namespace kge
