// Chunks of VE neighbouring elements (one memory access each), warp and block sums, and the
// column reduction that ends the backward passes of the joiner's operators.
#pragma once

#include <string.h>

#include "common.cuh"

namespace ctct {

template <int BYTES>
struct RawBytes;
template <>
struct RawBytes<16> {
    using type = uint4;
};
template <>
struct RawBytes<8> {
    using type = uint2;
};
template <>
struct RawBytes<4> {
    using type = unsigned;
};
template <>
struct RawBytes<2> {
    using type = unsigned short;
};
// VE elements of T as they lie in memory
template <typename T, int VE>
using Raw = typename RawBytes<VE * static_cast<int>(sizeof(T))>::type;

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }

// one rounding to nearest even: the only one between the float32 arithmetic and a 16-bit output
template <typename T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ float from_float<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// data that a launch reads once: no L1 line is kept for it
__device__ __forceinline__ uint4 ld_once(const uint4 *p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "l"(p));
    return v;
}
__device__ __forceinline__ uint2 ld_once(const uint2 *p) {
    uint2 v;
    asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
    return v;
}
// narrow accesses of neighbouring lanes share a line: they keep it
__device__ __forceinline__ unsigned ld_once(const unsigned *p) { return __ldg(p); }
__device__ __forceinline__ unsigned short ld_once(const unsigned short *p) { return __ldg(p); }

template <typename T, int VE>
__device__ __forceinline__ Raw<T, VE> load_once(const T *p) {
    return ld_once(reinterpret_cast<const Raw<T, VE> *>(p));
}
template <typename T, int VE>
__device__ __forceinline__ Raw<T, VE> load_kept(const T *p) {
    return __ldg(reinterpret_cast<const Raw<T, VE> *>(p));
}
template <typename T, int VE>
__device__ __forceinline__ void store_raw(T *p, const Raw<T, VE> &v) {
    *reinterpret_cast<Raw<T, VE> *>(p) = v;
}

template <typename T, int VE>
__device__ __forceinline__ void unpack(const Raw<T, VE> &raw, float *x) {
    T t[VE];
    memcpy(t, &raw, sizeof(raw));
#pragma unroll
    for (int i = 0; i < VE; ++i) x[i] = to_float(t[i]);
}
template <typename T, int VE>
__device__ __forceinline__ Raw<T, VE> pack(const float *x) {
    T t[VE];
#pragma unroll
    for (int i = 0; i < VE; ++i) t[i] = from_float<T>(x[i]);
    Raw<T, VE> raw;
    memcpy(&raw, t, sizeof(raw));
    return raw;
}

// 16 bytes into shared memory, or zeros without a look at `src`
__device__ __forceinline__ void cp_async16_or_zero(void *dst, const void *src, bool there) {
    const unsigned to = static_cast<unsigned>(__cvta_generic_to_shared(dst));
    const int bytes = there ? 16 : 0;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(src), "r"(bytes) : "memory");
}

// VE values of a parameter vector stored in float32 or in the activations' type T
template <typename T, int VE>
__device__ __forceinline__ void load_param(const void *p, int is_f32, int64_t at, float *v) {
    if (is_f32) {
        constexpr int W = VE < 4 ? VE : 4;
#pragma unroll
        for (int i = 0; i < VE; i += W) unpack<float, W>(load_kept<float, W>(static_cast<const float *>(p) + at + i), v + i);
    } else {
        unpack<T, VE>(load_kept<T, VE>(static_cast<const T *>(p) + at), v);
    }
}

// Two float32 in one 64-bit register, added and multiplied by one instruction (sm_100): the kernels that are held
// back by instruction issue do their arithmetic in pairs.
struct F2 {
    unsigned long long v;
};
__device__ __forceinline__ F2 f2(float x, float y) {
    F2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ void split(const F2 &a, float &x, float &y) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(a.v));
}
__device__ __forceinline__ F2 add2(const F2 &a, const F2 &b) {
    F2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ F2 mul2(const F2 &a, const F2 &b) {
    F2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ F2 fma2(const F2 &a, const F2 &b, const F2 &c) {
    F2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return r;
}
__device__ __forceinline__ float sum2(const F2 &a) {
    float x, y;
    split(a, x, y);
    return x + y;
}
// P values as P / 2 pairs and back
template <int P>
__device__ __forceinline__ void pair_up(const float (&x)[P], F2 (&y)[P / 2]) {
#pragma unroll
    for (int i = 0; i < P / 2; ++i) y[i] = f2(x[2 * i], x[2 * i + 1]);
}
template <int P>
__device__ __forceinline__ void unpair(const F2 (&y)[P / 2], float (&x)[P]) {
#pragma unroll
    for (int i = 0; i < P / 2; ++i) split(y[i], x[2 * i], x[2 * i + 1]);
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Sums of K values over the thread block (blockDim.x a multiple of 32, at most 1024), the same in every thread and
// in a fixed order.  One barrier: `slot` alternates between calls, so that a warp that is a call ahead
// writes the other half of `sm` (2 * K * 32 floats).
template <int K>
__device__ __forceinline__ void block_sum(float (&v)[K], float *sm, int slot) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    float *s = sm + slot * (K * 32);
#pragma unroll
    for (int k = 0; k < K; ++k) {
        v[k] = warp_sum(v[k]);
        if (lane == 0) s[k * 32 + warp] = v[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] = warp_sum(lane < warps ? s[k * 32 + lane] : 0.0f);
}

// out[o][c] = sum over p of part[o][p][c]: the partial sums that the blocks of a launch leave, added
// in a fixed order, so that gradients do not depend on which block came first.  Blocks of COLS columns x LANES
// threads; a thread adds every LANES-th partial, shared memory joins them.
struct ReduceArgs {
    const float *part;
    void *out;
    int out_f32;     // out in float32, else in T
    int64_t P, C;    // partials, columns
};
template <typename T, int COLS, int LANES>
__device__ __forceinline__ void reduce_columns(const ReduceArgs &a, int64_t col_block, int64_t o, float (*sm)[COLS + 1]) {
    const int tx = threadIdx.x % COLS, ty = threadIdx.x / COLS;
    const int64_t c = col_block * COLS + tx;
    float s = 0.0f;
    if (c < a.C) {
        const float *p = a.part + o * a.P * a.C + c;
        float s8[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) s8[k] = 0.0f;
        int64_t i = ty;
        for (; i + 7 * LANES < a.P; i += 8 * LANES)
#pragma unroll
            for (int k = 0; k < 8; ++k) s8[k] += p[(i + LANES * k) * a.C];
        for (; i < a.P; i += LANES) s8[0] += p[i * a.C];
        s = ((s8[0] + s8[1]) + (s8[2] + s8[3])) + ((s8[4] + s8[5]) + (s8[6] + s8[7]));
    }
    sm[ty][tx] = s;
    __syncthreads();
    if (ty == 0 && c < a.C) {
        float t = 0.0f;
#pragma unroll
        for (int k = 0; k < LANES; ++k) t += sm[k][tx];
        if (a.out_f32)
            static_cast<float *>(a.out)[o * a.C + c] = t;
        else
            static_cast<T *>(a.out)[o * a.C + c] = from_float<T>(t);
    }
}

}  // namespace ctct
