// One AdamW step over many tensors: moments in 32 bits or, by blocks of 128 values, in 8.
//
//   m = beta_m m + (1 - beta_m) g,  v = beta_v v + (1 - beta_v) g^2,  p = p decay - step_size m / (sqrt(v) correction + epsilon)
//
// A warp takes a block of 128 values, 4 to a lane, in one pass: the block's largest new moments are known after one reduction
// across the warp, before anything is written.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

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
    float beta_m, one_minus_beta_m, beta_v, one_minus_beta_v, epsilon, grad_scale;
    float decay, step_size, correction;
    uint32_t key;
    const float* schedule;
};

struct Tensor {
    void* param;
    const void* grad;
    unsigned long long size;
    unsigned long long first_block;  // of its moments
    uint32_t blocks_end;             // blocks of this launch before the next tensor's (all tensors so far)
    uint32_t aligned;                // 1: the vectors of both arrays are aligned
};

template <int MAX>
struct Table {
    Tensor t[MAX];
    int n;
};

__device__ __forceinline__ float rounded_stochastically(float x, uint32_t r16) {  // to bf16, toward zero or away from it
    const uint32_t b = __float_as_uint(x);
    if ((b & 0x7f800000u) == 0x7f800000u) return __bfloat162float(__float2bfloat16_rn(x));  // stays infinite, or NaN
    return __uint_as_float((b + r16) & 0xffff0000u);
}

// The codes of a block: TOP = 255 without a sign, 127 with one.
template <int TOP>
__device__ __forceinline__ int block_exponent(uint32_t largest) {
    if (largest >= 0x7f800000u) return 255;
    return max((int)((largest + 0xfffffu) >> 23), TOP == 255 ? 33 : 16);
}
template <int TOP>
__device__ __forceinline__ uint32_t encode(float x, int exponent, uint32_t r16) {
    const uint32_t b = __float_as_uint(x), magnitude = b & 0x7fffffffu;
    const int step = (int)((magnitude + (r16 << 4)) >> 20) - (8 * exponent + 7 - TOP);
    int code = min(max(step, TOP == 255 && magnitude > 0 ? 1 : 0), TOP);
    if (TOP == 127 && (b >> 31) && code > 0) code |= 128;
    return (uint32_t)code;
}
template <int TOP>
__device__ __forceinline__ float decode(uint32_t code, int exponent) {
    if (exponent == 255) return __uint_as_float(0x7fc00000u);
    const uint32_t c = code & (uint32_t)TOP;
    const uint32_t magnitude = c ? (uint32_t)((int)c + (8 * exponent + 7 - TOP)) << 20 : 0u;
    return __uint_as_float(magnitude | (TOP == 127 ? (code & 128u) << 24 : 0u));
}

__device__ __forceinline__ void load_values(const float* p, float (&v)[4]) {
    const float4 t = *reinterpret_cast<const float4*>(p);
    v[0] = t.x, v[1] = t.y, v[2] = t.z, v[3] = t.w;
}
__device__ __forceinline__ void load_values(const __nv_bfloat16* p, float (&v)[4]) {
    const uint2 t = *reinterpret_cast<const uint2*>(p);
    v[0] = __uint_as_float(t.x << 16), v[1] = __uint_as_float(t.x & 0xffff0000u);
    v[2] = __uint_as_float(t.y << 16), v[3] = __uint_as_float(t.y & 0xffff0000u);
}
__device__ __forceinline__ void load_values(const __half* p, float (&v)[4]) {
    const uint2 t = *reinterpret_cast<const uint2*>(p);
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&t.x)), b = __half22float2(*reinterpret_cast<const __half2*>(&t.y));
    v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y;
}
__device__ __forceinline__ void store_values(float* p, const float (&v)[4]) { *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]); }
__device__ __forceinline__ void store_values(__nv_bfloat16* p, const float (&v)[4]) {  // exact: the values are bf16 already
    uint2 t;
    t.x = __float_as_uint(v[0]) >> 16 | (__float_as_uint(v[1]) & 0xffff0000u);
    t.y = __float_as_uint(v[2]) >> 16 | (__float_as_uint(v[3]) & 0xffff0000u);
    *reinterpret_cast<uint2*>(p) = t;
}
__device__ __forceinline__ float value(const float* p) { return *p; }
__device__ __forceinline__ float value(const __half* p) { return __half2float(*p); }
__device__ __forceinline__ float value(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

constexpr int kThreads = 256;

template <class TP, class TG, int BITS, int MAX>
static __global__ void __launch_bounds__(kThreads) k_adamw(const __grid_constant__ Table<MAX> table, Params a, void* adam_m, void* adam_v,
                                                           uint8_t* __restrict__ m_exponent, uint8_t* __restrict__ v_exponent) {
    constexpr bool kBf16 = sizeof(TP) == 2;
    const uint32_t unit = blockIdx.x * (kThreads / 32) + threadIdx.x / 32;
    if (unit >= table.t[table.n - 1].blocks_end) return;
    int lo = 0, hi = table.n - 1;  // the first tensor whose end is past this block
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (table.t[mid].blocks_end > unit) hi = mid;
        else lo = mid + 1;
    }
    const Tensor& t = table.t[lo];
    const uint32_t local = unit - (lo > 0 ? table.t[lo - 1].blocks_end : 0u);
    const int lane = threadIdx.x & 31;
    const unsigned long long i0 = (unsigned long long)local * kBlock + lane * 4;           // in the tensor
    const unsigned long long block = t.first_block + local, at = block * kBlock + lane * 4;  // in the moments
    float decay = a.decay, step_size = a.step_size, correction = a.correction;
    uint32_t key = a.key;
    if (a.schedule) decay = a.schedule[0], step_size = a.schedule[1], correction = a.schedule[2], key = __float_as_uint(a.schedule[3]);

    TP* const param = static_cast<TP*>(t.param) + i0;
    const TG* const grad = static_cast<const TG*>(t.grad) + i0;
    const int live = i0 >= t.size ? 0 : t.size - i0 >= 4 ? 4 : (int)(t.size - i0);
    const bool whole = live == 4 && t.aligned;
    float p[4] = {}, g[4] = {}, m[4], v[4];
    if (whole) {
        load_values(param, p);
        load_values(grad, g);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (j < live) p[j] = value(param + j), g[j] = value(grad + j);
    }
    if (BITS == 32) {
        load_values(static_cast<const float*>(adam_m) + at, m);
        load_values(static_cast<const float*>(adam_v) + at, v);
    } else {
        const uint32_t cm = *reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(adam_m) + at);
        const uint32_t cv = *reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(adam_v) + at);
        const int em = m_exponent[block], ev = v_exponent[block];
#pragma unroll
        for (int j = 0; j < 4; ++j) m[j] = decode<127>(cm >> (8 * j) & 255u, em), v[j] = decode<255>(cv >> (8 * j) & 255u, ev);
    }
    uint32_t draw[4];
    const uint32_t base = (uint32_t)at * 0x9E3779B9u + (uint32_t)(at >> 32) * 0x6A09E667u + key;
    uint32_t largest_m = 0, largest_v = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float gj = g[j] * a.grad_scale;
        m[j] = fmaf(a.beta_m, m[j], a.one_minus_beta_m * gj);
        v[j] = fmaf(a.beta_v, v[j], a.one_minus_beta_v * gj * gj);
        p[j] = p[j] * decay - step_size * m[j] / (sqrtf(v[j]) * correction + a.epsilon);
        if (BITS == 8 || kBf16) draw[j] = mix(base + (uint32_t)j * 0x9E3779B9u);
        if (kBf16) p[j] = rounded_stochastically(p[j], draw[j] >> 8 & 0xffffu);
        if (j >= live) m[j] = v[j] = 0.f;  // the block's rest stays zero
        largest_m = max(largest_m, __float_as_uint(m[j]) & 0x7fffffffu);
        largest_v = max(largest_v, __float_as_uint(v[j]) & 0x7fffffffu);
    }
    if (whole) {
        store_values(param, p);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (j < live) put(param + j, p[j]);
    }
    if (BITS == 32) {
        store_values(static_cast<float*>(adam_m) + at, m);
        store_values(static_cast<float*>(adam_v) + at, v);
    } else {
        const int em = block_exponent<127>(__reduce_max_sync(~0u, largest_m)), ev = block_exponent<255>(__reduce_max_sync(~0u, largest_v));
        uint32_t cm = 0, cv = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            cm |= encode<127>(m[j], em, draw[j] & 0xffffu) << (8 * j);
            cv |= encode<255>(v[j], ev, draw[j] >> 16) << (8 * j);
        }
        *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(adam_m) + at) = cm;
        *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(adam_v) + at) = cv;
        if (lane == 0) m_exponent[block] = (uint8_t)em, v_exponent[block] = (uint8_t)ev;
    }
}

static __global__ void __launch_bounds__(kThreads) k_moments(const uint8_t* __restrict__ adam_m, const uint8_t* __restrict__ m_exponent,
                                                             const uint8_t* __restrict__ adam_v, const uint8_t* __restrict__ v_exponent,
                                                             size_t blocks, __nv_bfloat16* __restrict__ m_out, __nv_bfloat16* __restrict__ v_out) {
    const size_t block = (size_t)blockIdx.x * (kThreads / 32) + threadIdx.x / 32;
    if (block >= blocks) return;
    const size_t at = block * kBlock + (threadIdx.x & 31) * 4;
    const uint32_t cm = *reinterpret_cast<const uint32_t*>(adam_m + at), cv = *reinterpret_cast<const uint32_t*>(adam_v + at);
    const int em = m_exponent[block], ev = v_exponent[block];
    float m[4], v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) m[j] = decode<127>(cm >> (8 * j) & 255u, em), v[j] = decode<255>(cv >> (8 * j) & 255u, ev);
    store_values(m_out + at, m);
    store_values(v_out + at, v);
}

}  // namespace adamw
}  // namespace kge
