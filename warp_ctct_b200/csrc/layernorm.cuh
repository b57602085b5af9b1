// Layer norm over the last dimension, forward and backward.
//
//   mu = mean(x), r = 1 / sqrt(mean((x - mu)^2) + eps), xh = (x - mu) r, y = w xh + b
//   q = w dy,  dx = r (q - mean(q) - xh mean(q xh)),  dw = sum over rows of dy xh,  db = sum over rows of dy
//
// A row stays in registers between the two sums and the output, so every element is read once and
// written once: the bound is HBM traffic (16000 x 4096 f32: 6.2 TB/s forward, 85 us; 5.6 backward, 140 us).  The variance is the mean of squared deviations (a second
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

// A thread's P columns of a row: chunks of VE neighbours, chunk i at (i * team + tid) * VE.  ODD: rows that are no whole number
// of 16-byte vectors, one behind the other: chunks are the aligned vectors that a row lies in, so its first column stands
// `shift` elements inside a vector.  A block's rows are a multiple of a vector's elements apart, so the shift
// is the block's and a thread keeps its columns; only the row's two ends are accessed element by element.  (With
// 2-byte accesses 16000 rows of 1023 bf16 took 37 us forward and 148 backward, so 33 and 48; rows of 1024 take 14 and 29.)
template <typename T, int VE, int NV, bool ODD>
struct LnCols {
    int col[NV];
    bool whole[NV], some[NV];
    __device__ __forceinline__ LnCols(int team, int tid, int H, int64_t first_row) {
        const int shift = ODD ? static_cast<int>((first_row * H) & (VE - 1)) : 0;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            col[i] = (i * team + tid) * VE - shift;
            whole[i] = ODD ? col[i] >= 0 && col[i] + VE <= H : col[i] < H;
            some[i] = ODD ? col[i] + VE > 0 && col[i] < H : whole[i];
        }
    }
    __device__ __forceinline__ bool has(int i, int e, int H) const {
        return ODD ? whole[i] || (col[i] + e >= 0 && col[i] + e < H) : whole[i];
    }
    // a chunk as it lies in memory: with the neighbouring rows' elements where the row has none, but for the tensor's last vector,
    // which may end behind the tensor and is read element by element
    __device__ __forceinline__ Raw<T, VE> load(int i, const T *row, int H, const T *end) const {
        if (whole[i] || (ODD && some[i] && row + col[i] + VE <= end)) return load_once<T, VE>(row + col[i]);
        Raw<T, VE> raw{};
        if (ODD && some[i]) {
            T t[VE];
            memcpy(t, &raw, sizeof(raw));
#pragma unroll
            for (int e = 0; e < VE; ++e)
                if (has(i, e, H)) t[e] = row[col[i] + e];
            memcpy(&raw, t, sizeof(raw));
        }
        return raw;
    }
    // its values, zeros where there is no column
    __device__ __forceinline__ void values(int i, const Raw<T, VE> &raw, int H, float *x) const {
        unpack<T, VE>(raw, x);
        if (ODD && !whole[i]) {
#pragma unroll
            for (int e = 0; e < VE; ++e)
                if (!has(i, e, H)) x[e] = 0.0f;
        }
    }
    __device__ __forceinline__ void store(int i, T *row, int H, const float (&v)[VE]) const {
        if (whole[i]) {
            store_raw<T, VE>(row + col[i], pack<T, VE>(v));
        } else if (ODD && some[i]) {
#pragma unroll
            for (int e = 0; e < VE; ++e)
                if (has(i, e, H)) row[col[i] + e] = from_float<T>(v[e]);
        }
    }
    // a parameter vector's values at the columns; `none` where there is no column or no vector
    __device__ __forceinline__ void param(const void *p, int is_f32, int H, float none, float (&v)[NV * VE]) const {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
#pragma unroll
            for (int e = 0; e < VE; ++e) v[i * VE + e] = none;
            if (!p) continue;
            if (ODD) {
#pragma unroll
                for (int e = 0; e < VE; ++e)
                    if (has(i, e, H)) load_param<T, 1>(p, is_f32, col[i] + e, v + i * VE + e);
            } else if (whole[i]) {
                load_param<T, VE>(p, is_f32, col[i], v + i * VE);
            }
        }
    }
};

// WIDE: all threads of the block share a row, else every warp has its own: rows blockIdx.x + gridDim.x * k, k dealt to the
// warps in turn.
template <typename T, int VE, int P, bool WIDE, bool ODD>
__global__ void __launch_bounds__(WIDE ? LN_WIDE_THREADS : 32 * LN_WARPS) k_ln_forward(const LnArgs a) {
    constexpr int NV = P / VE;
    __shared__ float sm[2 * 32];
    pdl_wait();
    const int team = WIDE ? blockDim.x : 32, tid = WIDE ? threadIdx.x : (threadIdx.x & 31);
    const int64_t step = WIDE ? gridDim.x : static_cast<int64_t>(gridDim.x) * LN_WARPS;
    int64_t row = blockIdx.x + (WIDE ? 0 : static_cast<int64_t>(threadIdx.x >> 5) * gridDim.x);
    const float inv_h = 1.0f / static_cast<float>(a.H);
    const LnCols<T, VE, NV, ODD> c(team, tid, a.H, row);
    const T *const x_end = static_cast<const T *>(a.x) + a.rows * a.H;   // of contiguous rows
    Raw<T, VE> raw[NV];
    auto fetch = [&](int64_t r) {
        const T *x = static_cast<const T *>(a.x) + r * a.x_stride;
#pragma unroll
        for (int i = 0; i < NV; ++i) raw[i] = c.load(i, x, a.H, x_end);
    };
    if (row < a.rows) fetch(row);
    float w[P], b[P];
    c.param(a.w, a.p_f32, a.H, 1.0f, w);
    c.param(a.b, a.p_f32, a.H, 0.0f, b);
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
            c.values(i, raw[i], a.H, x + i * VE);
#pragma unroll
            for (int e = 0; e < VE; ++e) s += x[i * VE + e];
        }
        if (row + step < a.rows) fetch(row + step);  // the next row is on its way during this one's sums
        const float mean = total(s) * inv_h;
        s = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if (c.some[i]) {
#pragma unroll
                for (int e = 0; e < VE; ++e) x[i * VE + e] -= mean;
                if (ODD && !c.whole[i]) {
#pragma unroll
                    for (int e = 0; e < VE; ++e)
                        if (!c.has(i, e, a.H)) x[i * VE + e] = 0.0f;
                }
#pragma unroll
                for (int e = 0; e < VE; ++e) s = fmaf(x[i * VE + e], x[i * VE + e], s);
            }
        }
        const float rstd = rsqrtf(fmaf(total(s), inv_h, a.eps));
        T *y = static_cast<T *>(a.y) + row * a.H;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if (c.some[i]) {
                float o[VE];
#pragma unroll
                for (int e = 0; e < VE; ++e) o[e] = fmaf(x[i * VE + e] * rstd, w[i * VE + e], b[i * VE + e]);
                c.store(i, y, a.H, o);
            }
        }
        if (a.stats && tid == 0) a.stats[row] = make_float2(mean, rstd);
    }
}

template <typename T, int VE, int P, bool WIDE, bool ODD>
__global__ void __launch_bounds__(WIDE ? LN_WIDE_THREADS : 32 * LN_WARPS) k_ln_backward(const LnGradArgs a) {
    constexpr int NV = P / VE;
    __shared__ float sm[2 * 2 * 32];
    pdl_wait();
    pdl_trigger();
    const int team = WIDE ? blockDim.x : 32, tid = WIDE ? threadIdx.x : (threadIdx.x & 31);
    const int64_t step = WIDE ? gridDim.x : static_cast<int64_t>(gridDim.x) * LN_WARPS;
    int64_t row = blockIdx.x + (WIDE ? 0 : static_cast<int64_t>(threadIdx.x >> 5) * gridDim.x);
    const float inv_h = 1.0f / static_cast<float>(a.H);
    const LnCols<T, VE, NV, ODD> c(team, tid, a.H, row);
    const T *const x_end = static_cast<const T *>(a.x) + a.rows * a.H, *const d_end = static_cast<const T *>(a.dy) + a.rows * a.H;
    Raw<T, VE> rx[NV], rd[NV];
    float2 st = make_float2(0.0f, 0.0f);
    auto fetch = [&](int64_t r) {
        const T *x = static_cast<const T *>(a.x) + r * a.x_stride;
        const T *d = static_cast<const T *>(a.dy) + r * a.dy_stride;
        st = a.stats[r];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            rx[i] = c.load(i, x, a.H, x_end);
            rd[i] = c.load(i, d, a.H, d_end);
        }
    };
    if (row < a.rows) fetch(row);
    float w[P], dw[P], db[P];
    c.param(a.w, a.p_f32, a.H, 1.0f, w);
#pragma unroll
    for (int i = 0; i < P; ++i) dw[i] = db[i] = 0.0f;
    int slot = 0;
    for (; row < a.rows; row += step) {
        float xh[P], d[P];
        const float rstd = st.y, mean = st.x;
        float sums[2] = {0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < NV; ++i) {   // where there is no column dy is zero, and so is all that it enters
            c.values(i, rx[i], a.H, xh + i * VE);
            c.values(i, rd[i], a.H, d + i * VE);
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
            if (c.some[i]) {
                float o[VE];
#pragma unroll
                for (int e = 0; e < VE; ++e) {
                    const int k = i * VE + e;
                    o[e] = (fmaf(w[k], d[k], -c1) - xh[k] * c2) * rstd;
                }
                c.store(i, dx, a.H, o);
            }
        }
    }
    if (!a.part) return;
    float *pw = a.part + static_cast<int64_t>(blockIdx.x) * a.H;
    float *pb = pw + static_cast<int64_t>(gridDim.x) * a.H;
    if (WIDE) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
#pragma unroll
            for (int e = 0; e < VE; ++e)
                if (c.has(i, e, a.H)) {
                    pw[c.col[i] + e] = dw[i * VE + e];
                    pb[c.col[i] + e] = db[i * VE + e];
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
        if (threadIdx.x < 32) {   // the first warp has the columns that all of them have
#pragma unroll
            for (int i = 0; i < NV; ++i) {
#pragma unroll
                for (int e = 0; e < VE; ++e)
                    if (c.has(i, e, a.H)) {
                        pw[c.col[i] + e] = acc[0][(i * VE + e) * 32 + tid];
                        pb[c.col[i] + e] = acc[1][(i * VE + e) * 32 + tid];
                    }
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
