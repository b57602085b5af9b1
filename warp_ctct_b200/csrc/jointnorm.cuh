// Layer norm of an additive joiner:  y[n,t,u] = LN(f[n,t] + g[n,u]) * w + b  and its backward pass, in the padded
// (N,T,U1,H) and the packed (valid rows, H) layout of the loss.
//
//   s = f + g, mu = mean(s) = mean(f) + mean(g), r = 1 / sqrt(mean((s - mu)^2) + eps), y = w (s - mu) r + b
//   q = w dy,  ds = r q - r mean(q) - (s - mu) r^3 mean(q (s - mu))
//   df[n,t] = sum over u of ds,  dg[n,u] = sum over t of ds,  dw = sum of dy (s - mu) r,  db = sum of dy
//
// The sum f + g exists in registers only: forward writes rows x H, backward reads rows x H once, everything else
// is (T + U1) / (T U1) of that.  f and g are centred row by row before they meet, so s - mu is one
// addition without cancellation against the means and needs no reduction of its own.
//
// Forward: a block takes TF frames of one utterance in registers (a thread owns P columns of each) and walks over a
// range of contexts: g is loaded once for TF rows, and one round of reductions (a butterfly that halves the
// number of values with every exchange) serves TF rows.
//
// Backward: with r known, everything that reads dy is one pass without a dependency on a row's own sums,
//   A[t] = sum_u r dy, B[u] = sum_t r dy, db = sum dy, c1 = sum_h w dy, c2 = sum_h w dy (f + g) (f, g centred)
// and the rest follows from sums over k1 = r c1 / H and k2 = r^3 c2 / H, which is 1 / H of the data:
//   df[t] = w A[t] - sum_u k1 - f[t] sum_u k2 - sum_u k2 g[u]   (dg[u] with t and u exchanged)
//   dw    = sum_t f[t] A[t] + sum_u g[u] B[u]
// The first kernel streams dy: a thread has P columns of TF frames, A in registers, B in shared memory at places
// that only it touches, no barrier anywhere (a warp's share of c1 and c2 goes out by itself).  That is 7 float32
// operations an element where the direct form takes 12 and waits for two reductions per row in
// between.  The second kernel multiplies k2 with f and g (two small products per utterance) and adds the partial
// sums in a fixed order: no atomics, the same bits every time.
#pragma once

#include <type_traits>

#include "elem.cuh"

namespace ctct {


struct JnShape {
    const int *lx, *ly;      // frames and labels per utterance, or nullptr: all of them
    const int64_t *cu;       // packed: row offsets per utterance (N + 1); nullptr = padded
    int64_t packed_rows;     // rows of the packed tensor: rows that the lengths place beyond it are not touched
    int N, T, U1, H;
    int tspan, uspan;        // frames and contexts of a block
    int tblocks, ublocks;    // blocks along T and U1
    // frames of utterance n, contexts of utterance n, tensor row of (n, t, u)
    __device__ __forceinline__ int frames(int n) const { return lx ? max(0, min(lx[n], T)) : T; }
    __device__ __forceinline__ int contexts(int n) const { return ly ? max(0, min(ly[n], U1 - 1)) + 1 : U1; }
    __device__ __forceinline__ int64_t first_row(int n) const { return cu ? cu[n] : static_cast<int64_t>(n) * T * U1; }
    __device__ __forceinline__ int row_pitch(int contexts) const { return cu ? contexts : U1; }  // rows per frame
};

struct JnArgs {
    JnShape s;
    const void *f, *g;
    int64_t f_sn, f_st, g_sn, g_su;   // strides in elements
    const void *w, *b;                // or nullptr
    int p_f32;
    float eps;
    void *y;
    float *fm, *gm, *rstd;            // means of f (N,T), of g (N,U1), 1 / deviation per tensor row; or nullptr
    unsigned main_blocks;             // blocks beyond it clear packed rows behind the last utterance
};

struct JnGradArgs {
    JnShape s;
    const void *f, *g;
    int64_t f_sn, f_st, g_sn, g_su;
    const void *w;
    int p_f32;
    const void *dy;
    const float *fm, *gm, *rstd;
    float *part_a;       // [N][ublocks][T][H]
    float *part_b;       // [N][tblocks][U1][H]
    float *part_w;       // [2][tiles][H]: dw, db
    float2 *part_c;      // [warps of a row][tensor rows]: {c1, c2}
    int64_t rows;        // rows of the tensor
    int slices;          // blocks along the columns
};

// K sums over the warp (K = 4, 8, 16) with K - 1 + log2(32 / K) exchanges: every step sends half of the values
// away and adds the other half.  Lane l ends up with the total of value l * K / 32.
template <int K>
__device__ __forceinline__ float warp_sums(float (&v)[K]) {
    const int lane = threadIdx.x & 31;
    int o = 16;
#pragma unroll
    for (int n = K; n > 1; n >>= 1, o >>= 1) {
        const bool up = lane & o;
#pragma unroll
        for (int i = 0; i < n / 2; ++i) {
            const float send = up ? v[i] : v[i + n / 2];
            const float keep = up ? v[i + n / 2] : v[i];
            v[i] = keep + __shfl_xor_sync(0xffffffffu, send, o);
        }
    }
#pragma unroll
    for (; o > 0; o >>= 1) v[0] += __shfl_xor_sync(0xffffffffu, v[0], o);
    return v[0];
}
// The same over the block: lane l of every warp gets the block's total of value l * K / 32.  Up to 32 / K
// warps, so that one lane per warp and value joins them.  `sm`: 2 * 32 floats; `slot` alternates between calls (one
// barrier a call, none for a block of one warp).
template <int K>
__device__ __forceinline__ float block_sums(float (&v)[K], float *sm, int slot) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    constexpr int SAME = 32 / K;  // lanes that hold the same value
    float t = warp_sums<K>(v);
    if (warps == 1) return t;
    float *s = sm + slot * 32;    // [value][warp]
    if (lane % SAME == 0) s[lane + warp] = t;
    __syncthreads();
    t = lane % SAME < warps ? s[lane] : 0.0f;
#pragma unroll
    for (int o = SAME / 2; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
    return t;
}

// A thread's P columns: chunks of VE neighbours, chunk i at (i * team + tid) * VE.
template <int VE, int P>
struct JnCols {
    static constexpr int NV = P / VE;
    int col[NV];
    bool ok[NV];
    __device__ __forceinline__ JnCols(int H) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            col[i] = (i * static_cast<int>(blockDim.x) + static_cast<int>(threadIdx.x)) * VE;
            ok[i] = col[i] < H;
        }
    }
};

template <typename T, int VE, int P, int TF>
__global__ void __maxnreg__(128) k_joint_norm(const JnArgs a) {
    constexpr int NV = P / VE, Q = P / 2;
    constexpr int SAME = 32 / TF;                   // also the most warps of a block
    constexpr int GW = TF == 1 ? 16 : 8;            // warps that leave a share of g's sum (blocks have at most GW)
    __shared__ float sm[2 * 32];
    __shared__ __align__(16) float sg[2][GW];
    __shared__ __align__(16) float bc[GW][2 * TF];  // a warp's copy of the TF values that all its lanes read, doubled
    pdl_wait();
    const JnShape &s = a.s;
    const int tid = threadIdx.x, team = blockDim.x, lane = tid & 31, warp = tid >> 5, warps = team >> 5;
    const JnCols<VE, P> c(s.H);
    const Raw<T, VE> zero = Raw<T, VE>{};
    T *y = static_cast<T *>(a.y);
    if (blockIdx.x >= a.main_blocks) {
        for (int64_t r = s.cu[s.N] + (blockIdx.x - a.main_blocks); r < s.packed_rows; r += gridDim.x - a.main_blocks)
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if (c.ok[i]) store_raw<T, VE>(y + r * s.H + c.col[i], zero);
        return;
    }
    const int ub = blockIdx.x % s.ublocks, q = blockIdx.x / s.ublocks;
    const int tb = q % s.tblocks, n = q / s.tblocks;
    const int Tn = s.frames(n), Un = s.contexts(n);
    const int u0 = ub * s.uspan, u1 = min(u0 + s.uspan, s.U1), ue = min(u1, Un);
    const int t0 = tb * TF, tn = min(TF, Tn - t0);  // valid frames of the block's TF
    const int64_t base = s.first_row(n);
    const int pitch = s.row_pitch(Un);
    if (tn > 0 && u0 < ue) {
        const float inv_h = 1.0f / static_cast<float>(s.H);
        const int64_t pitch_h = static_cast<int64_t>(pitch) * s.H;
        if (tid < 2 * GW) sg[tid / GW][tid % GW] = 0.0f;
        F2 w[Q], b[Q], f[TF][Q], inside[NV];
        Raw<T, VE> rg[NV];
        const T *gr = static_cast<const T *>(a.g) + n * a.g_sn + u0 * a.g_su;
        auto fetch_g = [&]() {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                rg[i] = Raw<T, VE>{};
                if (c.ok[i]) rg[i] = load_kept<T, VE>(gr + c.col[i]);
            }
            gr += a.g_su;
        };
        fetch_g();
        float fv[TF][P];
#pragma unroll
        for (int k = 0; k < TF; ++k) {
            const T *fr = static_cast<const T *>(a.f) + n * a.f_sn + (t0 + k) * a.f_st;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
#pragma unroll
                for (int e = 0; e < VE; ++e) fv[k][i * VE + e] = 0.0f;
                if (c.ok[i] && k < tn) unpack<T, VE>(load_kept<T, VE>(fr + c.col[i]), fv[k] + i * VE);
            }
        }
        {
            float wv[P], bv[P];
#pragma unroll
            for (int i = 0; i < P; ++i) {
                wv[i] = 1.0f;
                bv[i] = 0.0f;
            }
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                if (c.ok[i] && a.w) load_param<T, VE>(a.w, a.p_f32, c.col[i], wv + i * VE);
                if (c.ok[i] && a.b) load_param<T, VE>(a.b, a.p_f32, c.col[i], bv + i * VE);
                // columns beyond H hold 0 - mean: they are left out of the squares
                inside[i] = c.ok[i] ? f2(1.0f, 1.0f) : f2(0.0f, 0.0f);
            }
            pair_up<P>(wv, w);
            pair_up<P>(bv, b);
        }
        __syncthreads();   // sg
        float gv[P];
        int slot = 0;
        auto sum_g = [&]() {   // unpacks rg into gv; this warp's part of its sum
            float x = 0.0f;
#pragma unroll
            for (int i = 0; i < NV; ++i) unpack<T, VE>(rg[i], gv + i * VE);
#pragma unroll
            for (int i = 0; i < P; ++i) x += gv[i];
            return warp_sum(x);
        };
        // One round gives TF sums (lane l: value l * TF / 32) and the sum of the next context's g.
        float g_sum = 0.0f;
        auto round = [&](float (&v)[TF], float g_part) {
            if (lane == 0) sg[slot][warp] = g_part;
            const float t = block_sums<TF>(v, sm, slot);
            if (warps == 1) __syncwarp();
            g_sum = 0.0f;
#pragma unroll
            for (int i = 0; i < GW; i += 4) {
                const float4 x = *reinterpret_cast<const float4 *>(&sg[slot][i]);
                g_sum += (x.x + x.y) + (x.z + x.w);
            }
            slot ^= 1;
            return t;
        };
        // spread the lanes' values over the warp
        auto spread = [&](float mine, F2 (&v)[TF]) {
            __syncwarp();
            if ((lane & (SAME - 1)) == 0) *reinterpret_cast<float2 *>(&bc[warp][2 * (lane / SAME)]) = make_float2(mine, mine);
            __syncwarp();
#pragma unroll
            for (int k = 0; k < TF; ++k) v[k] = *reinterpret_cast<const F2 *>(&bc[warp][2 * k]);
        };
        F2 all[TF];
        {
            float v[TF];
#pragma unroll
            for (int k = 0; k < TF; ++k) {
                v[k] = 0.0f;
#pragma unroll
                for (int i = 0; i < P; ++i) v[k] += fv[k][i];
            }
            const float mine = round(v, sum_g()) * inv_h;
            if (a.fm && ub == 0 && warp == 0 && (lane & (SAME - 1)) == 0 && lane / SAME < tn)
                a.fm[static_cast<int64_t>(n) * s.T + t0 + lane / SAME] = mine;
            spread(-mine, all);
        }
#pragma unroll
        for (int k = 0; k < TF; ++k) {
            pair_up<P>(fv[k], f[k]);
#pragma unroll
            for (int i = 0; i < Q; ++i) f[k][i] = add2(f[k][i], all[k]);
        }
        int64_t row = base + static_cast<int64_t>(t0) * pitch + u0;   // of the first of the TF frames
        T *out[TF];
#pragma unroll
        for (int k = 0; k < TF; ++k) out[k] = y + row * s.H + k * pitch_h;
        float *rstd = a.rstd && warp == 0 && (lane & (SAME - 1)) == 0 && lane / SAME < tn
                          ? a.rstd + row + static_cast<int64_t>(lane / SAME) * pitch : nullptr;
        float *gm = a.gm && t0 == 0 && tid == 0 ? a.gm + static_cast<int64_t>(n) * s.U1 + u0 : nullptr;
        // FULL: all frames, all columns and all rows are there, the case that is free of predicates
        auto walk = [&](auto full_tag) {
            constexpr bool FULL = decltype(full_tag)::value;
            for (int u = u0; u < ue; ++u, ++row) {
                const float gmean = g_sum * inv_h;
                if (gm) *gm++ = gmean;
                F2 gc[Q];
                pair_up<P>(gv, gc);
                const F2 minus = f2(-gmean, -gmean);
#pragma unroll
                for (int i = 0; i < Q; ++i) gc[i] = add2(gc[i], minus);
                if (u + 1 < ue) fetch_g();
                float v[TF];
#pragma unroll
                for (int k = 0; k < TF; ++k) {
                    F2 acc = f2(0.0f, 0.0f);
                    if (VE == 1 && !FULL) {   // a pair is two chunks, either may lie beyond H
#pragma unroll
                        for (int i = 0; i < Q; ++i) {
                            float x0, x1;
                            split(add2(f[k][i], gc[i]), x0, x1);
                            const F2 d = f2(c.ok[(2 * i) % NV] ? x0 : 0.0f, c.ok[(2 * i + 1) % NV] ? x1 : 0.0f);
                            acc = fma2(d, d, acc);
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < Q; ++i) {
                            const F2 d = add2(f[k][i], gc[i]);
                            acc = fma2(FULL ? d : mul2(d, inside[2 * i / VE]), d, acc);
                        }
                    }
                    v[k] = sum2(acc);
                }
                const float mine = rsqrtf(fmaf(round(v, sum_g()), inv_h, a.eps));
                int kn = tn;   // frames whose row of this context is inside the tensor
                if (!FULL && s.cu) kn = static_cast<int>(min(static_cast<int64_t>(tn), max(static_cast<int64_t>(0), (s.packed_rows - row + pitch - 1) / pitch)));
                if (rstd) {
                    if (FULL || lane / SAME < kn) *rstd = mine;
                    ++rstd;
                }
                spread(mine, all);
#pragma unroll
                for (int k = 0; k < TF; ++k) {
                    if (FULL || k < kn) {
#pragma unroll
                        for (int i = 0; i < NV; ++i) {
                            if (FULL || c.ok[i]) {
                                float o[VE];
                                if (VE == 1) {
                                    float lo, hi;
                                    split(fma2(mul2(add2(f[k][i / 2], gc[i / 2]), all[k]), w[i / 2], b[i / 2]), lo, hi);
                                    o[0] = i % 2 ? hi : lo;
                                } else {
#pragma unroll
                                    for (int e = 0; e < VE / 2; ++e) {
                                        const int j = i * VE / 2 + e;
                                        split(fma2(mul2(add2(f[k][j], gc[j]), all[k]), w[j], b[j]), o[(2 * e) % VE], o[(2 * e + 1) % VE]);
                                    }
                                }
                                store_raw<T, VE>(out[k] + c.col[i], pack<T, VE>(o));
                            }
                        }
                    }
                    out[k] += s.H;
                }
            }
        };
        const int64_t last = base + static_cast<int64_t>(t0 + tn - 1) * pitch + ue - 1;
        if (tn == TF && s.H == team * P && (!s.cu || last < s.packed_rows))   // the same for the whole block
            walk(std::true_type{});
        else
            walk(std::false_type{});
    }
    if (s.cu) return;
    // padding rows of the padded layout are zeros
    for (int k = 0; k < min(TF, s.T - t0); ++k) {
        for (int u = (k < tn) ? max(u0, ue) : u0; u < u1; ++u) {
            T *out = y + (base + static_cast<int64_t>(t0 + k) * s.U1 + u) * s.H;
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if (c.ok[i]) store_raw<T, VE>(out + c.col[i], zero);
        }
    }
}

constexpr int JG_P = 8, JG_TF = 4;      // columns per thread, frames per block of registers
constexpr int JG_MAX_THREADS = 256;
#ifndef JG_REGS
#define JG_REGS 168
#endif

template <typename T, int VE>
__global__ void __maxnreg__(JG_REGS) k_joint_norm_grad(const JnGradArgs a) {
    constexpr int P = JG_P, TF = JG_TF, NV = P / VE, Q = P / 2;
    extern __shared__ __align__(16) float acc_b[];  // [uspan][P / 4][team][4]: B of this block, private to the threads
    pdl_wait();
    pdl_trigger();
    const JnShape &s = a.s;
    const int tid = threadIdx.x, team = blockDim.x, lane = tid & 31;
    const int slice = blockIdx.x % a.slices;
    const unsigned tile = blockIdx.x / a.slices;
    int col[NV], at[NV];
    bool in[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        col[i] = slice * (JG_MAX_THREADS * P) + (i * team + tid) * VE;
        in[i] = col[i] < s.H;
        at[i] = in[i] ? col[i] : 0;
    }
    const int ub = tile % s.ublocks, q_ = tile / s.ublocks;
    const int tb = q_ % s.tblocks, n = q_ / s.tblocks;
    const int Tn = s.frames(n), Un = s.contexts(n);
    const int u0 = ub * s.uspan, ue = min(min(u0 + s.uspan, s.U1), Un);
    const int ta = tb * s.tspan, te = min(min(ta + s.tspan, s.T), Tn);
    const int64_t base = s.first_row(n);
    const int pitch = s.row_pitch(Un);
    const int64_t pitch_h = static_cast<int64_t>(pitch) * s.H;
    const F2 z2 = f2(0.0f, 0.0f);
    F2 dw[Q], db[Q];
#pragma unroll
    for (int i = 0; i < Q; ++i) dw[i] = db[i] = z2;
    if (ta < te && u0 < ue) {
        F2 w[Q];
        {
            float wv[P];
#pragma unroll
            for (int i = 0; i < P; ++i) wv[i] = in[i / VE] ? 1.0f : 0.0f;
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if (in[i] && a.w) load_param<T, VE>(a.w, a.p_f32, col[i], wv + i * VE);
            pair_up<P>(wv, w);
        }
        for (int i = 0; i < (ue - u0) * (P / 4); ++i)
            *reinterpret_cast<float4 *>(acc_b + (static_cast<size_t>(i) * team + tid) * 4) = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        const T *g = static_cast<const T *>(a.g) + n * a.g_sn;
        const float *gms = a.gm + static_cast<int64_t>(n) * s.U1;
        auto centred_g = [&](const Raw<T, VE> (&rg)[NV], float mean, F2 (&gc)[Q]) {
            float gv[P];
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                unpack<T, VE>(rg[i], gv + i * VE);
#pragma unroll
                for (int e = 0; e < VE; ++e) gv[i * VE + e] -= mean;
            }
            pair_up<P>(gv, gc);
        };
        // warps of a row, counted over all slices
        float2 *part_c = a.part_c + static_cast<int64_t>(slice * (JG_MAX_THREADS / 32) + (tid >> 5)) * a.rows;
        const int kl = (lane >> 2) & (TF - 1);   // the frame whose sums this lane ends up with
        for (int t0 = ta; t0 < te; t0 += TF) {
            const int tn = min(TF, te - t0);
            F2 f[TF][Q], A[TF][Q];
#pragma unroll
            for (int k = 0; k < TF; ++k) {
                const T *fr = static_cast<const T *>(a.f) + n * a.f_sn + (t0 + k) * a.f_st;
                const float mean = k < tn ? a.fm[static_cast<int64_t>(n) * s.T + t0 + k] : 0.0f;
                float fv[P];
#pragma unroll
                for (int i = 0; i < NV; ++i) {
#pragma unroll
                    for (int e = 0; e < VE; ++e) fv[i * VE + e] = 0.0f;
                    if (in[i] && k < tn) {
                        unpack<T, VE>(load_kept<T, VE>(fr + col[i]), fv + i * VE);
#pragma unroll
                        for (int e = 0; e < VE; ++e) fv[i * VE + e] -= mean;
                    }
                }
                pair_up<P>(fv, f[k]);
#pragma unroll
                for (int i = 0; i < Q; ++i) A[k][i] = z2;
            }
            int64_t row = base + static_cast<int64_t>(t0) * pitch + u0;   // of the first of the TF frames
            const T *dy[TF];
#pragma unroll
            for (int k = 0; k < TF; ++k) dy[k] = static_cast<const T *>(a.dy) + row * s.H + k * pitch_h;
            const T *gr = g + u0 * a.g_su;
            const float *my_r = a.rstd + row + static_cast<int64_t>(kl) * pitch;
            float *my_c = reinterpret_cast<float *>(part_c + row + static_cast<int64_t>(kl) * pitch) + (lane >> 4);
            // FULL: all frames and rows are there; threads without columns read column 0 with a weight of zero
            auto walk = [&](auto full_tag) {
                constexpr bool FULL = decltype(full_tag)::value;
                Raw<T, VE> rd[TF][NV], rg[NV];
                // frames whose row of the context is inside the tensor (a packed one may end early: zeros from there)
                auto inside = [&](int64_t first) {
                    if (FULL) return TF;
                    if (!s.cu) return tn;
                    return static_cast<int>(min(static_cast<int64_t>(tn), max(static_cast<int64_t>(0), (s.packed_rows - first + pitch - 1) / pitch)));
                };
                auto fetch_row = [&](int k, int kn) {
#pragma unroll
                    for (int i = 0; i < NV; ++i) {
                        if (FULL) {
                            rd[k][i] = load_once<T, VE>(dy[k] + at[i]);
                        } else {
                            rd[k][i] = Raw<T, VE>{};
                            if (in[i] && k < kn) rd[k][i] = load_once<T, VE>(dy[k] + at[i]);
                        }
                    }
                    dy[k] += s.H;
                };
                auto fetch_g = [&]() {
#pragma unroll
                    for (int i = 0; i < NV; ++i) rg[i] = load_kept<T, VE>(gr + at[i]);
                    gr += a.g_su;
                };
                int kn = inside(row);
#pragma unroll
                for (int k = 0; k < TF; ++k) fetch_row(k, kn);
                fetch_g();
                float r_next = (FULL || kl < kn) ? *my_r : 0.0f, gmean = gms[u0];
                float *acc = acc_b + tid * 4;
                for (int u = u0; u < ue; ++u) {
                    const float r_mine = r_next;
                    F2 gc[Q], B[Q];
                    centred_g(rg, gmean, gc);
                    const bool more = u + 1 < ue;
                    const int kn_now = kn;
                    ++row;
                    ++my_r;
                    if (more) {
                        kn = inside(row);
                        fetch_g();
                        r_next = (FULL || kl < kn) ? *my_r : 0.0f;
                        gmean = gms[u + 1];
                    }
                    float v[2 * TF];
#pragma unroll
                    for (int i = 0; i < Q; ++i) B[i] = z2;
#pragma unroll
                    for (int k = 0; k < TF; ++k) {
                        float dv[P];
#pragma unroll
                        for (int i = 0; i < NV; ++i) unpack<T, VE>(rd[k][i], dv + i * VE);
                        F2 d[Q];
                        pair_up<P>(dv, d);
                        if (more) fetch_row(k, kn);   // on its way for a whole step
                        const float r = __shfl_sync(0xffffffffu, r_mine, 4 * k);
                        const F2 r2 = f2(r, r);
                        F2 s1 = z2, s2 = z2;
#pragma unroll
                        for (int i = 0; i < Q; ++i) {
                            const F2 q = mul2(w[i], d[i]);
                            s1 = add2(s1, q);
                            s2 = fma2(q, add2(f[k][i], gc[i]), s2);
                            A[k][i] = fma2(d[i], r2, A[k][i]);
                            B[i] = fma2(d[i], r2, B[i]);
                            db[i] = add2(db[i], d[i]);
                        }
                        v[k] = sum2(s1);
                        v[TF + k] = sum2(s2);
                    }
                    const float sum = warp_sums<2 * TF>(v);
                    if ((lane & 3) == 0 && (FULL || kl < kn_now)) *my_c = sum;
                    my_c += 2;
#pragma unroll
                    for (int i = 0; i < P / 4; ++i, acc += 4 * team) {
                        ulonglong2 old = *reinterpret_cast<const ulonglong2 *>(acc);
                        old.x = add2(F2{old.x}, B[2 * i]).v;
                        old.y = add2(F2{old.y}, B[2 * i + 1]).v;
                        *reinterpret_cast<ulonglong2 *>(acc) = old;
                    }
                }
            };
            const int64_t last = base + static_cast<int64_t>(t0 + tn - 1) * pitch + ue - 1;
            if (tn == TF && (!s.cu || last < s.packed_rows))   // the same for the whole block
                walk(std::true_type{});
            else
                walk(std::false_type{});
#pragma unroll
            for (int k = 0; k < TF; ++k) {
                float *out = a.part_a + ((static_cast<int64_t>(n) * s.ublocks + ub) * s.T + t0 + k) * s.H;
                float o[P];
                unpair<P>(A[k], o);
#pragma unroll
                for (int i = 0; i < Q; ++i) dw[i] = fma2(f[k][i], A[k][i], dw[i]);
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    if (k < tn && in[i]) {
                        constexpr int W = VE < 4 ? VE : 4;
#pragma unroll
                        for (int e = 0; e < VE; e += W) store_raw<float, W>(out + col[i] + e, pack<float, W>(o + i * VE + e));
                    }
                }
            }
        }
        for (int u = u0; u < ue; ++u) {
            float *out = a.part_b + ((static_cast<int64_t>(n) * s.tblocks + tb) * s.U1 + u) * s.H;
            Raw<T, VE> rg[NV];
            F2 gc[Q], B[Q];
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                rg[i] = Raw<T, VE>{};
                if (in[i]) rg[i] = load_kept<T, VE>(g + u * a.g_su + col[i]);
            }
            centred_g(rg, gms[u], gc);
            float o[P];
#pragma unroll
            for (int i = 0; i < P / 4; ++i)
                unpack<float, 4>(*reinterpret_cast<const uint4 *>(acc_b + (static_cast<size_t>((u - u0) * (P / 4) + i) * team + tid) * 4), o + 4 * i);
            pair_up<P>(o, B);
#pragma unroll
            for (int i = 0; i < Q; ++i) dw[i] = fma2(gc[i], B[i], dw[i]);
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                if (in[i]) {
                    constexpr int W = VE < 4 ? VE : 4;
#pragma unroll
                    for (int e = 0; e < VE; e += W) store_raw<float, W>(out + col[i] + e, pack<float, W>(o + i * VE + e));
                }
            }
        }
    }
    float *pw = a.part_w + static_cast<int64_t>(tile) * s.H;
    float *pb = pw + static_cast<int64_t>(gridDim.x / a.slices) * s.H;
    float ow[P], ob[P];
    unpair<P>(dw, ow);
    unpair<P>(db, ob);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        if (in[i]) {
            constexpr int W = VE < 4 ? VE : 4;
#pragma unroll
            for (int e = 0; e < VE; e += W) {
                store_raw<float, W>(pw + col[i] + e, pack<float, W>(ow + i * VE + e));
                store_raw<float, W>(pb + col[i] + e, pack<float, W>(ob + i * VE + e));
            }
        }
    }
}

// Second half of the backward pass, three kinds of blocks: [0, w_blocks) add up dw and db, then JF_ROWS contexts
// of dg each, then JF_ROWS frames of df each.  A frame t >= lx and a context u > ly get zeros.
constexpr int JF_ROWS = 8, JF_CHUNK = 64, JF_THREADS = 128, JF_COLS = 4, JF_BATCH = 8;  // 512 columns a block
constexpr int JF_W_COLS = 8;  // columns of a block that adds up dw or db: whole 32-byte sectors, 16 partials at a time
struct JnFinishArgs {
    JnShape s;
    const void *f, *g;
    int64_t f_sn, f_st, g_sn, g_su;
    const void *w;
    int p_f32;
    const float *fm, *gm, *rstd;
    const float *part_a, *part_b, *part_w;
    const float2 *part_c;
    int64_t rows;
    int warps;                 // shares of c1 and c2 per row
    void *df, *dg, *dw, *db;   // any of them nullptr
    int64_t tiles;             // partial rows of dw and db
    int no_rows;               // there was none: every gradient is zero
    unsigned w_blocks, g_blocks;
    int w_cols, g_slices;      // blocks along the columns of dw and db; of df and dg
};

// df of JF_ROWS frames ("own" rows; "other" are the contexts) or dg of JF_ROWS contexts (the other way round)
template <typename T>
__device__ __forceinline__ void joint_norm_finish_rows(const JnFinishArgs &a, bool is_f, unsigned block) {
    __shared__ __align__(16) float k1s[JF_CHUNK][JF_ROWS], k2s[JF_CHUNK][JF_ROWS];
    __shared__ float means[JF_CHUNK], totals[2][JF_ROWS];
    const JnShape &s = a.s;
    const int tid = threadIdx.x, team = blockDim.x;
    const int rows = is_f ? s.T : s.U1;
    const int groups = (rows + JF_ROWS - 1) / JF_ROWS;
    const int slice = block % a.g_slices;
    const unsigned q = block / a.g_slices;
    const int n = static_cast<int>(q / groups), i0 = static_cast<int>(q - static_cast<unsigned>(n) * groups) * JF_ROWS;
    const int Tn = a.no_rows ? 0 : s.frames(n), Un = a.no_rows ? 0 : s.contexts(n);
    const int others = is_f ? Un : Tn;
    const int own = others > 0 ? (is_f ? Tn : Un) - i0 : 0;   // own rows that take part: nothing is known of the rest
    const int col = (slice * team + tid) * JF_COLS;     // JF_COLS neighbours; the last thread of a row may have fewer
    const int cols = min(max(s.H - col, 0), JF_COLS);
    const bool vec = (s.H | (is_f ? a.g_su | a.g_sn : a.f_st | a.f_sn)) % JF_COLS == 0 &&
                     reinterpret_cast<uintptr_t>(is_f ? a.g : a.f) % (JF_COLS * sizeof(T)) == 0;
    const int64_t base = s.first_row(n);
    const int pitch = s.row_pitch(Un);
    const int64_t si = is_f ? pitch : 1, sj = is_f ? 1 : pitch;
    const float inv_h = 1.0f / static_cast<float>(s.H);
    const float *other_mean = is_f ? a.gm + static_cast<int64_t>(n) * s.U1 : a.fm + static_cast<int64_t>(n) * s.T;
    const T *other = is_f ? static_cast<const T *>(a.g) + n * a.g_sn : static_cast<const T *>(a.f) + n * a.f_sn;
    const int64_t other_st = is_f ? a.g_su : a.f_st;
    F2 acc[JF_ROWS][2];
#pragma unroll
    for (int k = 0; k < JF_ROWS; ++k) acc[k][0] = acc[k][1] = f2(0.0f, 0.0f);
    if (tid < 2 * JF_ROWS) totals[tid / JF_ROWS][tid % JF_ROWS] = 0.0f;
    for (int j0 = 0; own > 0 && j0 < others; j0 += JF_CHUNK) {
        const int jn = min(JF_CHUNK, others - j0);
        __syncthreads();
        // lanes along the axis whose rows are neighbours in memory: contexts
#pragma unroll 2
        for (int i = tid; i < JF_ROWS * JF_CHUNK; i += team) {
            const int k = is_f ? i / JF_CHUNK : i % JF_ROWS, j = is_f ? i % JF_CHUNK : i / JF_ROWS;
            const int64_t row = base + (i0 + k) * si + (j0 + j) * sj;
            float k1 = 0.0f, k2 = 0.0f;
            if (k < own && j < jn && (!s.cu || row < s.packed_rows)) {
                float c1 = 0.0f, c2 = 0.0f;
                const float r = a.rstd[row];
#pragma unroll 2
                for (int p = 0; p < a.warps; ++p) {
                    const float2 c = a.part_c[p * a.rows + row];
                    c1 += c.x;
                    c2 += c.y;
                }
                k1 = r * (c1 * inv_h);
                k2 = r * r * (r * (c2 * inv_h));
            }
            k1s[j][k] = k1;
            k2s[j][k] = k2;
        }
        for (int j = tid; j < JF_CHUNK; j += team) means[j] = j < jn ? other_mean[j0 + j] : 0.0f;
        __syncthreads();
        if (tid < 2 * JF_ROWS * 4) {   // four lanes per own row and sum
            const float(*from)[JF_ROWS] = tid < JF_ROWS * 4 ? k1s : k2s;
            const int k = (tid >> 2) % JF_ROWS;
            float t = 0.0f;
            for (int j = tid & 3; j < JF_CHUNK; j += 4) t += from[j][k];
            t += __shfl_xor_sync(0xffffffffu, t, 1);
            t += __shfl_xor_sync(0xffffffffu, t, 2);
            if ((tid & 3) == 0) totals[tid >= JF_ROWS * 4][k] += t;
        }
        if (cols > 0) {
            for (int j1 = 0; j1 < jn; j1 += JF_BATCH) {   // a batch of rows is on its way together
                float x[JF_BATCH][JF_COLS];
                Raw<T, JF_COLS> raw[JF_BATCH];
#pragma unroll
                for (int b = 0; b < JF_BATCH; ++b) {
                    // behind the last row: that row again, with a factor of zero
                    const T *p = other + static_cast<int64_t>(min(j0 + j1 + b, others - 1)) * other_st + col;
                    if (vec) {
                        raw[b] = load_kept<T, JF_COLS>(p);
                    } else {
#pragma unroll
                        for (int e = 0; e < JF_COLS; ++e) x[b][e] = e < cols ? to_float(p[e]) : 0.0f;
                    }
                }
#pragma unroll
                for (int b = 0; b < JF_BATCH; ++b) {
                    if (vec) unpack<T, JF_COLS>(raw[b], x[b]);
                    const float mean = j1 + b < jn ? means[j1 + b] : 0.0f;
                    const F2 m = f2(-mean, -mean);
                    const F2 x0 = add2(f2(x[b][0], x[b][1]), m), x1 = add2(f2(x[b][2], x[b][3]), m);
                    float k2[JF_ROWS];
                    unpack<float, 4>(*reinterpret_cast<const uint4 *>(&k2s[j1 + b][0]), k2);
                    unpack<float, 4>(*reinterpret_cast<const uint4 *>(&k2s[j1 + b][4]), k2 + 4);
#pragma unroll
                    for (int k = 0; k < JF_ROWS; ++k) {
                        const F2 kk = f2(k2[k], k2[k]);
                        acc[k][0] = fma2(kk, x0, acc[k][0]);
                        acc[k][1] = fma2(kk, x1, acc[k][1]);
                    }
                }
            }
        }
    }
    __syncthreads();
    if (cols <= 0) return;
    const int parts = own > 0 ? (others + (is_f ? s.uspan : s.tspan) - 1) / (is_f ? s.uspan : s.tspan) : 0;
    const int parts_all = is_f ? s.ublocks : s.tblocks;
    const int64_t plane = static_cast<int64_t>(rows) * s.H;
    const float *part = (is_f ? a.part_a : a.part_b) + static_cast<int64_t>(n) * parts_all * plane + static_cast<int64_t>(i0) * s.H + col;
    T *out = static_cast<T *>(is_f ? a.df : a.dg) + (static_cast<int64_t>(n) * rows + i0) * s.H + col;
    const T *mine = (is_f ? static_cast<const T *>(a.f) + n * a.f_sn + i0 * a.f_st : static_cast<const T *>(a.g) + n * a.g_sn + i0 * a.g_su) + col;
    const int64_t mine_st = is_f ? a.f_st : a.g_su;
    const float *own_mean = (is_f ? a.fm + static_cast<int64_t>(n) * s.T : a.gm + static_cast<int64_t>(n) * s.U1) + i0;
    float w[JF_COLS];
#pragma unroll
    for (int e = 0; e < JF_COLS; ++e) {
        w[e] = 1.0f;
        if (a.w && e < cols) load_param<T, 1>(a.w, a.p_f32, col + e, w + e);
    }
#pragma unroll
    for (int k = 0; k < JF_ROWS; ++k) {
        if (i0 + k >= rows) break;
        float x[JF_COLS];
        split(acc[k][0], x[0], x[1]);
        split(acc[k][1], x[2], x[3]);
        float sum[JF_COLS] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (k < own) {
#pragma unroll 4
            for (int p = 0; p < parts; ++p) {
                const float *from = part + p * plane + static_cast<int64_t>(k) * s.H;
                if (s.H % JF_COLS == 0) {
                    float v[JF_COLS];
                    unpack<float, 4>(*reinterpret_cast<const uint4 *>(from), v);
#pragma unroll
                    for (int e = 0; e < JF_COLS; ++e) sum[e] += v[e];
                } else {
#pragma unroll
                    for (int e = 0; e < JF_COLS; ++e)
                        if (e < cols) sum[e] += from[e];
                }
            }
            const float t1 = totals[0][k], t2 = totals[1][k], mean = own_mean[k];
#pragma unroll
            for (int e = 0; e < JF_COLS; ++e) {
                const float c = e < cols ? to_float(mine[k * mine_st + e]) - mean : 0.0f;
                sum[e] = fmaf(w[e], sum[e], -t1) - fmaf(c, t2, x[e]);
            }
        }
        if (s.H % JF_COLS == 0) {
            store_raw<T, JF_COLS>(out + static_cast<int64_t>(k) * s.H, pack<T, JF_COLS>(sum));
        } else {
#pragma unroll
            for (int e = 0; e < JF_COLS; ++e)
                if (e < cols) out[static_cast<int64_t>(k) * s.H + e] = from_float<T>(sum[e]);
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(JF_THREADS) k_joint_norm_finish(const JnFinishArgs a) {
    pdl_wait();
    if (blockIdx.x < a.w_blocks) {
        __shared__ float sm[JF_THREADS / JF_W_COLS][JF_W_COLS + 1];
        const int which = blockIdx.x / a.w_cols;
        void *out = which ? a.db : a.dw;
        if (out)
            reduce_columns<T, JF_W_COLS, JF_THREADS / JF_W_COLS>(ReduceArgs{a.part_w + which * a.tiles * a.s.H, out, a.p_f32, a.tiles, a.s.H},
                                               blockIdx.x - which * a.w_cols, 0, sm);
        return;
    }
    const unsigned block = blockIdx.x - a.w_blocks;
    const bool is_f = block >= a.g_blocks;
    if (!(is_f ? a.df : a.dg)) return;
    joint_norm_finish_rows<T>(a, is_f, is_f ? block - a.g_blocks : block);
}

}  // namespace ctct
