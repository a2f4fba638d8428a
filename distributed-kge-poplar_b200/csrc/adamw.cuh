// One AdamW step over many tensors: moments in 32 bits or, by blocks of 128 values, in 8.
//
//   m = beta_m m + (1 - beta_m) g,  v = beta_v v + (1 - beta_v) g^2,  p = p decay - step_size m / (sqrt(v) correction + epsilon)
//
// One pass: a block's largest new moments are known after one reduction across its lanes, before they are written.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "pdl.cuh"

namespace kge {
namespace adamw {

constexpr int kBlock = 128;
constexpr int kMaxTensors = 256;  // of one launch: their table travels with the kernel's arguments

// A 32-bit mix: two rounds of folding the upper half down and multiplying by an odd number (fraction bits of pi and of the
// square root of 2).  Host and device agree.
__host__ __device__ __forceinline__ uint32_t mix(uint32_t x) {
    x = (x ^ (x >> 16)) * 0x85A308D3u;
    x = (x ^ (x >> 15)) * 0x6A09E667u;
    return x ^ (x >> 16);
}

struct Params {
    float beta_m, one_minus_beta_m, beta_v, one_minus_beta_v, epsilon;  // one_minus_beta times the gradients' scale, or its square
    float decay, step_size, correction;
    uint32_t key;
    const float* schedule;
};

struct Tensor {
    void* param;
    const void* grad;
    unsigned long long size;
    unsigned long long first;  // of its moments
    uint32_t units_end;        // units of this launch (128 values, of 8-bit moments 512) before the next tensor's
    uint32_t aligned;                // 1: the vectors of both arrays are aligned
};

template <int MAX>
struct Table {
    Tensor t[MAX];
    int n;
};

__device__ __forceinline__ float max_or_nan(float a, float b) {
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}
// The codes of a block: TOP = 255 without a sign, 127 with one.  They are kept short: at 60 integer instructions a value a step in 8
// bits was bound by them at three times the time that its bytes take.
template <int TOP>
__device__ __forceinline__ int block_exponent(uint32_t largest) {
    if (largest >= 0x7f800000u) return 255;
    return max((int)((largest + 0xfffffu) >> 23), TOP == 255 ? 33 : 16);
}
// What a code in units of 2^20 is added to, to be its value's bits.
template <int TOP>
__device__ __forceinline__ uint32_t code_base(int exponent) { return (uint32_t)(8 * exponent + 7 - TOP) << 20; }
template <int TOP>
__device__ __forceinline__ float decode(uint32_t byte, uint32_t base) {
    const uint32_t code = TOP == 127 ? byte & 127u : byte;
    const uint32_t bits = code * 0x100000u + min(code, 1u) * base;  // multiplications have a pipe of their own
    return __uint_as_float(TOP == 127 ? (byte * 0x1000000u & 0x80000000u) | bits : bits);
}
// The code of a value of a finite block in the upper byte; none is above TOP, since the block's exponent is that of its largest value
// rounded up.  A sign is not added yet.
template <int TOP>
__device__ __forceinline__ uint32_t encode(float x, uint32_t base, uint32_t r16) {
    const uint32_t magnitude = TOP == 127 ? __float_as_uint(x) & 0x7fffffffu : __float_as_uint(x);
    const int least = TOP == 255 ? (int)(min(magnitude, 1u) * 0x100000u) : 0;
    return (uint32_t)max((int)(r16 * 16u + (magnitude - base)), least) * 16u;
}
__device__ __forceinline__ uint32_t upper_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __byte_perm(__byte_perm(a, b, 0x0073), __byte_perm(c, d, 0x0073), 0x5410);
}
template <int TOP>
__device__ __forceinline__ uint32_t encode_four(const float* x, uint32_t base, const uint32_t* r16) {
    const uint32_t codes = upper_bytes(encode<TOP>(x[0], base, r16[0]), encode<TOP>(x[1], base, r16[1]), encode<TOP>(x[2], base, r16[2]), encode<TOP>(x[3], base, r16[3]));
    if (TOP == 255) return codes;
    return codes | (upper_bytes(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3])) & 0x80808080u);
}

__device__ __forceinline__ float value(const float* p) { return *p; }
__device__ __forceinline__ float value(const __half* p) { return __half2float(*p); }
__device__ __forceinline__ float value(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

constexpr int kThreads = 256;
constexpr int kBlocksPerWarp = 2;  // fetched together

__device__ __forceinline__ float quick_sqrt(float x) {
    float y;
    asm("sqrt.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float quick_reciprocal(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Four values of a lane as they lie in memory.
template <class T>
struct Quad;
template <>
struct Quad<float> {
    float4 raw;
    __device__ __forceinline__ void load(const float* p) { raw = *reinterpret_cast<const float4*>(p); }
    __device__ __forceinline__ void floats(float (&v)[4]) const { v[0] = raw.x, v[1] = raw.y, v[2] = raw.z, v[3] = raw.w; }
    __device__ __forceinline__ void set(const float (&v)[4]) { raw = make_float4(v[0], v[1], v[2], v[3]); }
};
template <class T>
struct HalfQuad {
    uint2 raw;
    __device__ __forceinline__ void load(const T* p) { raw = *reinterpret_cast<const uint2*>(p); }
};
template <>
struct Quad<__nv_bfloat16> : HalfQuad<__nv_bfloat16> {
    __device__ __forceinline__ void floats(float (&v)[4]) const {
        v[0] = __uint_as_float(raw.x << 16), v[1] = __uint_as_float(raw.x & 0xffff0000u), v[2] = __uint_as_float(raw.y << 16), v[3] = __uint_as_float(raw.y & 0xffff0000u);
    }
    __device__ __forceinline__ void set(const float (&v)[4]) {  // of values that are bf16
        raw.x = __byte_perm(__float_as_uint(v[0]), __float_as_uint(v[1]), 0x7632);
        raw.y = __byte_perm(__float_as_uint(v[2]), __float_as_uint(v[3]), 0x7632);
    }
};
template <>
struct Quad<__half> : HalfQuad<__half> {
    __device__ __forceinline__ void floats(float (&v)[4]) const {
        const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&raw.x)), b = __half22float2(*reinterpret_cast<const __half2*>(&raw.y));
        v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y;
    }
    __device__ __forceinline__ void set(const float (&v)[4]) {
        const __half2 a = __floats2half2_rn(v[0], v[1]), b = __floats2half2_rn(v[2], v[3]);
        raw.x = *reinterpret_cast<const uint32_t*>(&a), raw.y = *reinterpret_cast<const uint32_t*>(&b);
    }
};
// The lane's values of a tensor that begin `live` before its end, zeros past it.
template <class T>
__device__ __forceinline__ void load_quad(Quad<T>& q, const T* p, int live, bool whole) {
    if (whole) {
        q.load(p);
        return;
    }
    float v[4] = {};
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (j < live) v[j] = value(p + j);
    q.set(v);
}

// The tensor of a launch's block: the first whose end is past it.  All lanes of a warp look at once.
template <int MAX>
__device__ __forceinline__ int tensor_of(const Table<MAX>& table, uint32_t unit) {
    const int lane = threadIdx.x & 31;
    int at = 0;
    for (int base = 0; base < table.n; base += 32) {
        const bool before = base + lane < table.n && table.t[base + lane].units_end <= unit;
        const int n = __popc(__ballot_sync(~0u, before));
        at += n;
        if (n < 32) break;
    }
    return at;
}

struct Step {
    float beta_m, one_minus_beta_m, beta_v, one_minus_beta_v, epsilon, decay, step_size, correction;
    uint32_t key;
    __device__ __forceinline__ Step(const Params& a)
        : beta_m(a.beta_m), one_minus_beta_m(a.one_minus_beta_m), beta_v(a.beta_v), one_minus_beta_v(a.one_minus_beta_v), epsilon(a.epsilon), decay(a.decay),
          step_size(a.step_size), correction(a.correction), key(a.key) {
        if (a.schedule) decay = a.schedule[0], step_size = a.schedule[1], correction = a.schedule[2], key = __float_as_uint(a.schedule[3]);
    }
    // With 32-bit moments root and division are rounded to nearest, in the shade of the bytes (60 M values 228 us, with the approximations
    // below 231).  With 8-bit ones, whose step is bound by instructions, they are right to 2^-22 (120 M values 444 us, to nearest 500): the
    // step that they scale is a thousandth of the parameter, whose own rounding is 2^-24 or more.  The root's bound holds for every v, subnormal
    // ones included (gradients below 3e-18 make such; taken for 0 they left epsilon alone to divide by), the reciprocal's from 2^-126 to
    // 2^126: epsilon is a normal number, and a root is below 2^64.
    template <bool NEAREST>
    __device__ __forceinline__ void take(float& p, float g, float& m, float& v) const {
        m = fmaf(beta_m, m, one_minus_beta_m * g);
        v = fmaf(beta_v, v, one_minus_beta_v * g * g);
        if (NEAREST) p = fmaf(p, decay, __fdiv_rn(-step_size * m, fmaf(__fsqrt_rn(v), correction, epsilon)));
        else p = fmaf(p, decay, -step_size * m * quick_reciprocal(fmaf(quick_sqrt(v), correction, epsilon)));
    }
    // What is mixed for the values from a position (a multiple of 4) on.
    __device__ __forceinline__ uint32_t mixed(unsigned long long at) const { return (uint32_t)at * 0x9E3779B9u + (uint32_t)(at >> 32) * 0x6A09E667u + key; }
};
// Bits 8 to 23 of a draw.
__device__ __forceinline__ uint32_t middle(uint32_t draw) { return __byte_perm(draw, 0, 0x4421); }
// Four values rounded as their draws say, as they are stored.  fp32 ones are not rounded.
template <class TP>
__device__ __forceinline__ Quad<TP> rounded_quad(const float (&p)[4], const uint32_t (&draw)[4]) {
    Quad<TP> out;
    if constexpr (sizeof(TP) == 4) {
        out.set(p);
    } else {
        uint32_t b[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) b[j] = __float_as_uint(p[j]) + middle(draw[j]);
        if (!(fabsf(p[0]) + fabsf(p[1]) + (fabsf(p[2]) + fabsf(p[3])) < INFINITY)) {  // an infinity stays one; a NaN's bits would run over
#pragma unroll
            for (int j = 0; j < 4; ++j) b[j] = p[j] == p[j] ? b[j] : 0x7fc00000u;
        }
        out.raw.x = __byte_perm(b[0], b[1], 0x7632);
        out.raw.y = __byte_perm(b[2], b[3], 0x7632);
    }
    return out;
}
// The lane's values go back, `live` of them.
template <class T>
__device__ __forceinline__ void store_quad(T* p, const Quad<T>& q, int live, bool whole) {
    if (whole) {
        *reinterpret_cast<decltype(q.raw)*>(p) = q.raw;
        return;
    }
    float v[4];
    q.floats(v);
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (j < live) put(p + j, v[j]);
}

// Moments in fp32: a warp takes 128 values at a time, four to a lane, and two such units, fetched together.
template <class TP, class TG, int MAX>
static __global__ void __launch_bounds__(kThreads, 3) k_adamw32(const __grid_constant__ Table<MAX> table, Params a, float* __restrict__ adam_m, float* __restrict__ adam_v) {
    constexpr int kUnits = kBlocksPerWarp;
    grid_dependency_sync();
    const uint32_t n_units = table.t[table.n - 1].units_end;
    const uint32_t first = (blockIdx.x * (kThreads / 32) + threadIdx.x / 32) * kUnits;
    if (first >= n_units) return;
    const int lane = threadIdx.x & 31;
    const Step step(a);
    Quad<TP> p_raw[kUnits];
    Quad<TG> g_raw[kUnits];
    float4 m_raw[kUnits], v_raw[kUnits];
    TP* param[kUnits];
    unsigned long long at[kUnits];
    int live[kUnits];
    bool whole[kUnits];
    int index = tensor_of(table, first);
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
        const uint32_t unit = min(first + u, n_units - 1);  // the last is read, but not written, again
        while (table.t[index].units_end <= unit) ++index;
        const Tensor& t = table.t[index];
        const unsigned long long i0 = (unsigned long long)(unit - (index > 0 ? table.t[index - 1].units_end : 0u)) * kBlock + lane * 4;  // in the tensor
        at[u] = t.first + i0;  // in the moments
        live[u] = i0 >= t.size ? 0 : t.size - i0 >= 4 ? 4 : (int)(t.size - i0);
        whole[u] = live[u] == 4 && t.aligned;
        param[u] = static_cast<TP*>(t.param) + i0;
        load_quad(p_raw[u], static_cast<const TP*>(param[u]), live[u], whole[u]);
        load_quad(g_raw[u], static_cast<const TG*>(t.grad) + i0, live[u], whole[u]);
        m_raw[u] = *reinterpret_cast<const float4*>(adam_m + at[u]);
        v_raw[u] = *reinterpret_cast<const float4*>(adam_v + at[u]);
    }
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
        if (first + u >= n_units) return;
        float p[4], g[4], m[4] = {m_raw[u].x, m_raw[u].y, m_raw[u].z, m_raw[u].w}, v[4] = {v_raw[u].x, v_raw[u].y, v_raw[u].z, v_raw[u].w};
        p_raw[u].floats(p);
        g_raw[u].floats(g);
        // past the tensor's end gradient and moments are 0, and stay so
#pragma unroll
        for (int j = 0; j < 4; ++j) step.take<true>(p[j], g[j], m[j], v[j]);
        uint32_t draw[4] = {};
        if constexpr (sizeof(TP) == 2) {
#pragma unroll
            for (int j = 0; j < 4; ++j) draw[j] = mix(step.mixed(at[u]) + (uint32_t)j * 0x9E3779B9u);
        }
        store_quad(param[u], rounded_quad<TP>(p, draw), live[u], whole[u]);
        *reinterpret_cast<float4*>(adam_m + at[u]) = make_float4(m[0], m[1], m[2], m[3]);
        *reinterpret_cast<float4*>(adam_v + at[u]) = make_float4(v[0], v[1], v[2], v[3]);
    }
}

// A lane's 16 values, fetched and stored 16 bytes at a time.
template <class T>
struct LaneValues {
    static constexpr int kVectors = 16 * (int)sizeof(T) / 16;
    uint4 raw[kVectors];
    __device__ __forceinline__ void load(const T* p, int live, bool whole) {
        if (whole) {
#pragma unroll
            for (int i = 0; i < kVectors; ++i) raw[i] = reinterpret_cast<const uint4*>(p)[i];
        } else {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                Quad<T> part;
                load_quad(part, p + 4 * q, live - 4 * q, false);
                set(q, part);
            }
        }
    }
    __device__ __forceinline__ void store(T* p, int live, bool whole) const {
        if (whole) {
#pragma unroll
            for (int i = 0; i < kVectors; ++i) reinterpret_cast<uint4*>(p)[i] = raw[i];
        } else {
#pragma unroll
            for (int q = 0; q < 4; ++q) store_quad(p + 4 * q, quad(q), live - 4 * q, false);
        }
    }
    __device__ __forceinline__ Quad<T> quad(int q) const {
        Quad<T> part;
        if constexpr (sizeof(T) == 4) {
            part.raw = make_float4(__uint_as_float(raw[q].x), __uint_as_float(raw[q].y), __uint_as_float(raw[q].z), __uint_as_float(raw[q].w));
        } else {
            part.raw = q & 1 ? make_uint2(raw[q / 2].z, raw[q / 2].w) : make_uint2(raw[q / 2].x, raw[q / 2].y);
        }
        return part;
    }
    __device__ __forceinline__ void set(int q, const Quad<T>& part) {
        if constexpr (sizeof(T) == 4) {
            raw[q] = make_uint4(__float_as_uint(part.raw.x), __float_as_uint(part.raw.y), __float_as_uint(part.raw.z), __float_as_uint(part.raw.w));
        } else if (q & 1) {
            raw[q / 2].z = part.raw.x, raw[q / 2].w = part.raw.y;
        } else {
            raw[q / 2].x = part.raw.x, raw[q / 2].y = part.raw.y;
        }
    }
};

// Moments in 8 bits: a warp takes four blocks of 128 values, eight lanes and 16 values a lane each, so that what a lane does but once
// (finding its place, the exponents) is spread over 16 values: with four a lane a step took 92 instructions a value.
constexpr int kLaneValues = 16;
template <class TP, class TG, int MAX>
static __global__ void __launch_bounds__(kThreads, 3) k_adamw8(const __grid_constant__ Table<MAX> table, Params a, uint8_t* __restrict__ adam_m, uint8_t* __restrict__ adam_v,
                                                               uint8_t* __restrict__ m_exponent, uint8_t* __restrict__ v_exponent) {
    constexpr int N = kLaneValues;
    grid_dependency_sync();
    const uint32_t unit = blockIdx.x * (kThreads / 32) + threadIdx.x / 32;
    if (unit >= table.t[table.n - 1].units_end) return;
    const int lane = threadIdx.x & 31, index = tensor_of(table, unit);
    const Tensor& t = table.t[index];
    const unsigned long long i0 = (unsigned long long)(unit - (index > 0 ? table.t[index - 1].units_end : 0u)) * (4 * kBlock) + lane * N;  // in the tensor
    const bool here = (i0 & ~(unsigned long long)(kBlock - 1)) < t.size;  // the block is this tensor's, for all of its lanes
    const unsigned long long at = t.first + i0, block = at / kBlock;      // in the moments
    const int live = i0 >= t.size ? 0 : t.size - i0 >= N ? N : (int)(t.size - i0);
    const bool whole = live == N && t.aligned;
    TP* const param = static_cast<TP*>(t.param) + i0;
    const TG* const grad = static_cast<const TG*>(t.grad) + i0;
    LaneValues<TP> params;
    LaneValues<TG> grads;
    uint4 m_raw = make_uint4(0, 0, 0, 0), v_raw = m_raw;
    int em = 16, ev = 33;
    if (here) {
        m_raw = *reinterpret_cast<const uint4*>(adam_m + at);
        v_raw = *reinterpret_cast<const uint4*>(adam_v + at);
        em = m_exponent[block], ev = v_exponent[block];
    }
    params.load(param, live, whole);
    grads.load(grad, live, whole);
    const Step step(a);
    float m[N], v[N], largest_m = 0.f, largest_v = 0.f;
    uint32_t draw[N];
    {
        const uint32_t base_m = code_base<127>(em), base_v = code_base<255>(ev);
        const uint32_t mw[4] = {m_raw.x, m_raw.y, m_raw.z, m_raw.w}, vw[4] = {v_raw.x, v_raw.y, v_raw.z, v_raw.w};
#pragma unroll
        for (int j = 0; j < N; ++j) {
            m[j] = decode<127>(__byte_perm(mw[j / 4], 0, 0x4440 + j % 4), base_m);
            v[j] = decode<255>(__byte_perm(vw[j / 4], 0, 0x4440 + j % 4), base_v);
        }
        if (em == 255 || ev == 255) {
            const float nan = __uint_as_float(0x7fc00000u);
#pragma unroll
            for (int j = 0; j < N; ++j) m[j] = em == 255 ? nan : m[j], v[j] = ev == 255 ? nan : v[j];
        }
    }
    const uint32_t base = step.mixed(at);
#pragma unroll
    for (int q = 0; q < N / 4; ++q) {
        float p[4], g[4];
        uint32_t d[4];
        params.quad(q).floats(p);
        grads.quad(q).floats(g);
        // past the tensor's end gradient and moments are 0, and stay so
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            step.take<false>(p[j], g[j], m[4 * q + j], v[4 * q + j]);
            d[j] = draw[4 * q + j] = mix(base + (uint32_t)(4 * q + j) * 0x9E3779B9u);
            largest_m = max_or_nan(largest_m, fabsf(m[4 * q + j]));
            largest_v = max_or_nan(largest_v, v[4 * q + j]);
        }
        params.set(q, rounded_quad<TP>(p, d));
    }
    params.store(param, live, whole);
    uint32_t top_m = __float_as_uint(largest_m), top_v = __float_as_uint(largest_v);
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) top_m = max(top_m, __shfl_xor_sync(~0u, top_m, o)), top_v = max(top_v, __shfl_xor_sync(~0u, top_v, o));
    if (!here) return;
    const int new_em = block_exponent<127>(top_m), new_ev = block_exponent<255>(top_v);
    const uint32_t base_m = code_base<127>(new_em), base_v = code_base<255>(new_ev);
    uint32_t mw[4], vw[4];
#pragma unroll
    for (int q = 0; q < N / 4; ++q) {
        uint32_t low[4], high[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) low[j] = draw[4 * q + j] & 0xffffu, high[j] = draw[4 * q + j] >> 16;
        mw[q] = encode_four<127>(m + 4 * q, base_m, low), vw[q] = encode_four<255>(v + 4 * q, base_v, high);
    }
    *reinterpret_cast<uint4*>(adam_m + at) = make_uint4(mw[0], mw[1], mw[2], mw[3]);
    *reinterpret_cast<uint4*>(adam_v + at) = make_uint4(vw[0], vw[1], vw[2], vw[3]);
    if ((lane & 7) == 0) m_exponent[block] = (uint8_t)new_em, v_exponent[block] = (uint8_t)new_ev;
}

static __global__ void __launch_bounds__(kThreads) k_moments(const uint8_t* __restrict__ adam_m, const uint8_t* __restrict__ m_exponent,
                                                             const uint8_t* __restrict__ adam_v, const uint8_t* __restrict__ v_exponent,
                                                             size_t size, __nv_bfloat16* __restrict__ m_out, __nv_bfloat16* __restrict__ v_out) {
    grid_dependency_sync();
    const size_t at = ((size_t)blockIdx.x * kThreads + threadIdx.x) * 8;  // eight values a thread: 16 bytes of results
    if (at >= size) return;
    const uint2 mw = *reinterpret_cast<const uint2*>(adam_m + at), vw = *reinterpret_cast<const uint2*>(adam_v + at);
    const int em = m_exponent[at / kBlock], ev = v_exponent[at / kBlock];
    const uint32_t base_m = code_base<127>(em), base_v = code_base<255>(ev), words[4] = {mw.x, mw.y, vw.x, vw.y};
    uint32_t bits[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t byte = __byte_perm(words[i], 0, 0x4440 + j);
            bits[i][j] = (i < 2 ? em : ev) == 255 ? 0x7fc00000u : __float_as_uint(i < 2 ? decode<127>(byte, base_m) : decode<255>(byte, base_v));
        }
    const auto packed = [&](int i) {
        return make_uint4(__byte_perm(bits[i][0], bits[i][1], 0x7632), __byte_perm(bits[i][2], bits[i][3], 0x7632), __byte_perm(bits[i + 1][0], bits[i + 1][1], 0x7632),
                          __byte_perm(bits[i + 1][2], bits[i + 1][3], 0x7632));
    };
    *reinterpret_cast<uint4*>(m_out + at) = packed(0);
    *reinterpret_cast<uint4*>(v_out + at) = packed(2);
}

}  // namespace adamw
}  // namespace kge
