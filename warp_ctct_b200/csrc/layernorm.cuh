// Layer norm over the last dimension, forward and backward.
//
//   mu = mean(x), r = 1 / sqrt(mean((x - mu)^2) + eps), xh = (x - mu) r, y = w xh + b
//   q = w dy,  dx = r (q - mean(q) - xh mean(q xh)),  dw = sum over rows of dy xh,  db = sum over rows of dy
//
// A row stays in registers between the two sums and the output, so every element is read once and
// written once: the bound is HBM traffic.  The variance is the mean of squared deviations (a second
// pass over the registers), not a difference of moments, so a large common offset costs no digits.
// The weight's and the bias's gradient are accumulated in registers over all rows that a block takes
// (a thread owns its columns), leave as one float32 partial row per block, and are added up in a fixed order.
#pragma once

#include "elem.cuh"

namespace ctct {

struct LnArgs {
    const void *x;        // rows x H, `x_stride` elements from row to row
    int64_t x_stride;
    const void *w, *b;    // H each, or nullptr
    int p_f32;            // w and b (and their gradients) in float32, else in the type of x
    float eps;
    void *y;              // rows x H
    float2 *stats;        // {mean, 1 / standard deviation} per row, kept for the backward pass; or nullptr
    int64_t rows;
    int H;
};
struct LnGradArgs {
    const void *dy;       // rows x H, `dy_stride` elements from row to row
    int64_t dy_stride;
    const void *x;
    int64_t x_stride;
    const void *w;
    int p_f32;
    const float2 *stats;
    void *dx;             // rows x H, or nullptr
    float *part;          // [2][gridDim.x][H]: partial dw, db; or nullptr
    int64_t rows;
    int H;
};

constexpr int LN_WARPS = 4;          // rows (warps) per block of the narrow kernels
constexpr int LN_WIDE_THREADS = 512; // largest block that shares one row

// WIDE: all threads of the block share a row (thread i holds chunks i, i + blockDim.x, ...), else every
// warp has its own.  P elements per thread in chunks of VE.
template <typename T, int VE, int P, bool WIDE>
__global__ void __launch_bounds__(WIDE ? LN_WIDE_THREADS : 32 * LN_WARPS) k_ln_forward(const LnArgs a) {
    constexpr int NV = P / VE;
    __shared__ float sm[2 * 32];
    pdl_wait();
    const int team = WIDE ? blockDim.x : 32, tid = WIDE ? threadIdx.x : (threadIdx.x & 31);
    const int64_t step = WIDE ? gridDim.x : static_cast<int64_t>(gridDim.x) * LN_WARPS;
    int64_t row = WIDE ? blockIdx.x : static_cast<int64_t>(blockIdx.x) * LN_WARPS + (threadIdx.x >> 5);
    const float inv_h = 1.0f / static_cast<float>(a.H);
    Raw<T, VE> raw[NV];
    auto fetch = [&](int64_t r) {
        const T *x = static_cast<const T *>(a.x) + r * a.x_stride;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int col = (i * team + tid) * VE;
            if (col < a.H) raw[i] = load_once<T, VE>(x + col);
        }
    };
    if (row < a.rows) fetch(row);
    float w[P], b[P];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int col = (i * team + tid) * VE;
#pragma unroll
        for (int e = 0; e < VE; ++e) {
            w[i * VE + e] = 1.0f;
            b[i * VE + e] = 0.0f;
        }
        if (col < a.H && a.w) load_param<T, VE>(a.w, a.p_f32, col, w + i * VE);
        if (col < a.H && a.b) load_param<T, VE>(a.b, a.p_f32, col, b + i * VE);
    }
    int slot = 0;
    auto total = [&](float v) {
        if (!WIDE) return warp_sum(v);
        float one[1] = {v};
        block_sum<1>(one, sm, slot);
        slot ^= 1;
        return one[0];
    };
    for (; row < a.rows; row += step) {
        float x[P];
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if ((i * team + tid) * VE < a.H) {
                unpack<T, VE>(raw[i], x + i * VE);
#pragma unroll
                for (int e = 0; e < VE; ++e) s += x[i * VE + e];
            }
        }
        if (row + step < a.rows) fetch(row + step);  // the next row is on its way during this one's sums
        const float mean = total(s) * inv_h;
        s = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if ((i * team + tid) * VE < a.H) {
#pragma unroll
                for (int e = 0; e < VE; ++e) {
                    const float d = x[i * VE + e] - mean;
                    x[i * VE + e] = d;
                    s = fmaf(d, d, s);
                }
            }
        }
        const float rstd = rsqrtf(fmaf(total(s), inv_h, a.eps));
        T *y = static_cast<T *>(a.y) + row * a.H;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int col = (i * team + tid) * VE;
            if (col < a.H) {
                float o[VE];
#pragma unroll
                for (int e = 0; e < VE; ++e) o[e] = fmaf(x[i * VE + e] * rstd, w[i * VE + e], b[i * VE + e]);
                store_raw<T, VE>(y + col, pack<T, VE>(o));
            }
        }
        if (a.stats && tid == 0) a.stats[row] = make_float2(mean, rstd);
    }
}

template <typename T, int VE, int P, bool WIDE>
__global__ void __launch_bounds__(WIDE ? LN_WIDE_THREADS : 32 * LN_WARPS) k_ln_backward(const LnGradArgs a) {
    constexpr int NV = P / VE;
    __shared__ float sm[2 * 2 * 32];
    pdl_wait();
    pdl_trigger();
    const int team = WIDE ? blockDim.x : 32, tid = WIDE ? threadIdx.x : (threadIdx.x & 31);
    const int64_t step = WIDE ? gridDim.x : static_cast<int64_t>(gridDim.x) * LN_WARPS;
    int64_t row = WIDE ? blockIdx.x : static_cast<int64_t>(blockIdx.x) * LN_WARPS + (threadIdx.x >> 5);
    const float inv_h = 1.0f / static_cast<float>(a.H);
    Raw<T, VE> rx[NV], rd[NV];
    float2 st = make_float2(0.0f, 0.0f);
    auto fetch = [&](int64_t r) {
        const T *x = static_cast<const T *>(a.x) + r * a.x_stride;
        const T *d = static_cast<const T *>(a.dy) + r * a.dy_stride;
        st = a.stats[r];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int col = (i * team + tid) * VE;
            if (col < a.H) {
                rx[i] = load_once<T, VE>(x + col);
                rd[i] = load_once<T, VE>(d + col);
            }
        }
    };
    if (row < a.rows) fetch(row);
    float w[P], dw[P], db[P];
#pragma unroll
    for (int i = 0; i < P; ++i) {
        w[i] = 1.0f;
        dw[i] = db[i] = 0.0f;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int col = (i * team + tid) * VE;
        if (col < a.H && a.w) load_param<T, VE>(a.w, a.p_f32, col, w + i * VE);
    }
    int slot = 0;
    for (; row < a.rows; row += step) {
        float xh[P], d[P];
        const float rstd = st.y, mean = st.x;
        float sums[2] = {0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if ((i * team + tid) * VE < a.H) {
                unpack<T, VE>(rx[i], xh + i * VE);
                unpack<T, VE>(rd[i], d + i * VE);
#pragma unroll
                for (int e = i * VE; e < (i + 1) * VE; ++e) {
                    xh[e] = (xh[e] - mean) * rstd;
                    const float q = w[e] * d[e];
                    sums[0] += q;
                    sums[1] = fmaf(q, xh[e], sums[1]);
                    dw[e] = fmaf(d[e], xh[e], dw[e]);
                    db[e] += d[e];
                }
            }
        }
        if (row + step < a.rows) fetch(row + step);
        if (!a.dx) continue;
        if (WIDE) {
            block_sum<2>(sums, sm, slot);
            slot ^= 1;
        } else {
            sums[0] = warp_sum(sums[0]);
            sums[1] = warp_sum(sums[1]);
        }
        const float c1 = sums[0] * inv_h, c2 = sums[1] * inv_h;
        T *dx = static_cast<T *>(a.dx) + row * a.H;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int col = (i * team + tid) * VE;
            if (col < a.H) {
                float o[VE];
#pragma unroll
                for (int e = 0; e < VE; ++e) {
                    const int k = i * VE + e;
                    o[e] = (fmaf(w[k], d[k], -c1) - xh[k] * c2) * rstd;
                }
                store_raw<T, VE>(dx + col, pack<T, VE>(o));
            }
        }
    }
    if (!a.part) return;
    float *pw = a.part + static_cast<int64_t>(blockIdx.x) * a.H;
    float *pb = pw + static_cast<int64_t>(gridDim.x) * a.H;
    if (WIDE) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int col = (i * team + tid) * VE;
            if (col < a.H) {
#pragma unroll
                for (int e = 0; e < VE; ++e) {
                    pw[col + e] = dw[i * VE + e];
                    pb[col + e] = db[i * VE + e];
                }
            }
        }
    } else {  // join the rows of the block's warps, one warp after the other
        __shared__ float acc[2][32 * P];
        for (int k = 0; k < LN_WARPS; ++k) {
            if ((threadIdx.x >> 5) == k) {
#pragma unroll
                for (int i = 0; i < P; ++i) {
                    acc[0][i * 32 + tid] = k == 0 ? dw[i] : acc[0][i * 32 + tid] + dw[i];
                    acc[1][i * 32 + tid] = k == 0 ? db[i] : acc[1][i * 32 + tid] + db[i];
                }
            }
            __syncthreads();
        }
        for (int i = threadIdx.x; i < 32 * P; i += 32 * LN_WARPS) {
            // value i belongs to lane i % 32, its element i / 32
            const int e = i / 32, col = ((e / VE) * 32 + (i & 31)) * VE + e % VE;
            if (col < a.H) {
                pw[col] = acc[0][i];
                pb[col] = acc[1][i];
            }
        }
    }
}

// Rows too long for the registers of a block (H > LN_WIDE_THREADS * 16): one block per row, three passes
// over the row forward and two backward, the later ones out of L2.  The partial gradients of the weights
// are accumulated in the block's own partial row.
template <typename T, int VE>
__global__ void __launch_bounds__(LN_WIDE_THREADS) k_ln_forward_long(const LnArgs a) {
    __shared__ float sm[2 * 32];
    pdl_wait();
    const float inv_h = 1.0f / static_cast<float>(a.H);
    const int first = threadIdx.x * VE, stride = blockDim.x * VE;
    int slot = 0;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T *x = static_cast<const T *>(a.x) + row * a.x_stride;
        T *y = static_cast<T *>(a.y) + row * a.H;
        float s[1] = {0.0f};
        for (int col = first; col < a.H; col += stride) {
            float v[VE];
            unpack<T, VE>(load_kept<T, VE>(x + col), v);
#pragma unroll
            for (int e = 0; e < VE; ++e) s[0] += v[e];
        }
        block_sum<1>(s, sm, slot);
        slot ^= 1;
        const float mean = s[0] * inv_h;
        s[0] = 0.0f;
        for (int col = first; col < a.H; col += stride) {
            float v[VE];
            unpack<T, VE>(load_kept<T, VE>(x + col), v);
#pragma unroll
            for (int e = 0; e < VE; ++e) s[0] = fmaf(v[e] - mean, v[e] - mean, s[0]);
        }
        block_sum<1>(s, sm, slot);
        slot ^= 1;
        const float rstd = rsqrtf(fmaf(s[0], inv_h, a.eps));
        for (int col = first; col < a.H; col += stride) {
            float v[VE], w[VE], b[VE];
            unpack<T, VE>(load_kept<T, VE>(x + col), v);
#pragma unroll
            for (int e = 0; e < VE; ++e) {
                w[e] = 1.0f;
                b[e] = 0.0f;
            }
            if (a.w) load_param<T, VE>(a.w, a.p_f32, col, w);
            if (a.b) load_param<T, VE>(a.b, a.p_f32, col, b);
#pragma unroll
            for (int e = 0; e < VE; ++e) v[e] = fmaf((v[e] - mean) * rstd, w[e], b[e]);
            store_raw<T, VE>(y + col, pack<T, VE>(v));
        }
        if (a.stats && threadIdx.x == 0) a.stats[row] = make_float2(mean, rstd);
    }
}

template <typename T, int VE>
__global__ void __launch_bounds__(LN_WIDE_THREADS) k_ln_backward_long(const LnGradArgs a) {
    __shared__ float sm[2 * 2 * 32];
    pdl_wait();
    pdl_trigger();
    const float inv_h = 1.0f / static_cast<float>(a.H);
    const int first = threadIdx.x * VE, stride = blockDim.x * VE;
    float *pw = a.part ? a.part + static_cast<int64_t>(blockIdx.x) * a.H : nullptr;
    float *pb = a.part ? pw + static_cast<int64_t>(gridDim.x) * a.H : nullptr;
    if (a.part) {
        for (int col = first; col < a.H; col += stride) {
#pragma unroll
            for (int e = 0; e < VE; ++e) pw[col + e] = pb[col + e] = 0.0f;
        }
    }
    int slot = 0;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T *x = static_cast<const T *>(a.x) + row * a.x_stride;
        const T *dy = static_cast<const T *>(a.dy) + row * a.dy_stride;
        const float2 st = a.stats[row];
        float sums[2] = {0.0f, 0.0f};
        auto chunk = [&](int col, float *xh, float *d, float *w) {
            unpack<T, VE>(load_kept<T, VE>(x + col), xh);
            unpack<T, VE>(load_kept<T, VE>(dy + col), d);
#pragma unroll
            for (int e = 0; e < VE; ++e) {
                w[e] = 1.0f;
                xh[e] = (xh[e] - st.x) * st.y;
            }
            if (a.w) load_param<T, VE>(a.w, a.p_f32, col, w);
        };
        for (int col = first; col < a.H; col += stride) {
            float xh[VE], d[VE], w[VE];
            chunk(col, xh, d, w);
#pragma unroll
            for (int e = 0; e < VE; ++e) {
                sums[0] = fmaf(w[e], d[e], sums[0]);
                sums[1] = fmaf(w[e] * d[e], xh[e], sums[1]);
                if (a.part) {
                    pw[col + e] = fmaf(d[e], xh[e], pw[col + e]);
                    pb[col + e] += d[e];
                }
            }
        }
        if (!a.dx) continue;
        block_sum<2>(sums, sm, slot);
        slot ^= 1;
        const float c1 = sums[0] * inv_h, c2 = sums[1] * inv_h;
        T *dx = static_cast<T *>(a.dx) + row * a.H;
        for (int col = first; col < a.H; col += stride) {
            float xh[VE], d[VE], w[VE];
            chunk(col, xh, d, w);
#pragma unroll
            for (int e = 0; e < VE; ++e) d[e] = (fmaf(w[e], d[e], -c1) - xh[e] * c2) * st.y;
            store_raw<T, VE>(dx + col, pack<T, VE>(d));
        }
    }
}

// dw (blockIdx.y = 0) and db (1) out of the partial rows
template <typename T>
__global__ void __launch_bounds__(1024) k_ln_reduce(const float *part, int64_t P, int H, void *dw, void *db, int p_f32) {
    __shared__ float sm[32][33];
    pdl_wait();
    void *out = blockIdx.y == 0 ? dw : db;
    if (!out) return;
    reduce_columns<T, 32, 32>(ReduceArgs{part + blockIdx.y * P * H, out, p_f32, P, H}, blockIdx.x, 0, sm);
}

}  // namespace ctct
