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
// A block takes TF frames of one utterance in registers (a thread owns P columns of each) and walks over a range of
// contexts: g is loaded once for TF rows, and one round of reductions (a butterfly that halves the number of
// values with every exchange) serves TF rows.  In the backward pass df accumulates in the same
// registers, dg in the block's shared memory at places that only their own thread touches, dw and db in
// registers over the block's life.  All sums are float32 and leave as partial rows that a second launch
// adds in a fixed order: no atomics, the same bits every time.
#pragma once

#include "elem.cuh"

namespace ctct {

constexpr int JN_MAX_THREADS = 512;

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
    float *part_f;       // [N][ublocks][T][H]
    float *part_g;       // [N][tblocks][U1][H]
    float *part_w;       // [2][gridDim.x][H]
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
// The same over the block: lane l of every warp gets the block's total of value l * K / 32.  `sm`: 2 * K * 16
// floats (up to 16 warps); `slot` alternates between calls (one barrier a call, none for a block of one warp).
template <int K>
__device__ __forceinline__ float block_sums(float (&v)[K], float *sm, int slot) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    constexpr int SAME = 32 / K;  // lanes that hold the same value
    float t = warp_sums<K>(v);
    if (warps == 1) return t;
    float *s = sm + slot * (K * 16);
    if ((lane & (SAME - 1)) == 0) s[warp * K + lane / SAME] = t;
    __syncthreads();
    t = 0.0f;
    for (int w = 0; w < warps; ++w) t += s[w * K + lane / SAME];
    return t;
}

template <typename T, int VE, int P, int TF>
__global__ void __launch_bounds__(JN_MAX_THREADS) k_joint_norm(const JnArgs a) {
    constexpr int NV = P / VE;
    constexpr int SAME = 32 / TF;
    __shared__ float sm[2 * TF * 16];
    __shared__ float sg[2 * 32];
    __shared__ __align__(16) float bc[16][TF];  // a warp's copy of the TF values that all its lanes read
    pdl_wait();
    const JnShape &s = a.s;
    const int tid = threadIdx.x, team = blockDim.x, lane = tid & 31, warp = tid >> 5;
    const Raw<T, VE> zero = Raw<T, VE>{};
    T *y = static_cast<T *>(a.y);
    if (blockIdx.x >= a.main_blocks) {
        for (int64_t r = s.cu[s.N] + (blockIdx.x - a.main_blocks); r < s.packed_rows; r += gridDim.x - a.main_blocks)
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int col = (i * team + tid) * VE;
                if (col < s.H) store_raw<T, VE>(y + r * s.H + col, zero);
            }
        return;
    }
    const int ub = blockIdx.x % s.ublocks, q = blockIdx.x / s.ublocks;
    const int tb = q % s.tblocks, n = q / s.tblocks;
    const int Tn = s.frames(n), Un = s.contexts(n);
    const int u0 = ub * s.uspan, u1 = min(u0 + s.uspan, s.U1), ue = min(u1, Un);
    const int t_end = min((tb + 1) * s.tspan, s.T);
    const int64_t base = s.first_row(n);
    const int pitch = s.row_pitch(Un);
    const float inv_h = 1.0f / static_cast<float>(s.H);
    float w[P], b[P];
#pragma unroll
    for (int i = 0; i < P; ++i) {
        w[i] = 1.0f;
        b[i] = 0.0f;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int col = (i * team + tid) * VE;
        if (col < s.H && a.w) load_param<T, VE>(a.w, a.p_f32, col, w + i * VE);
        if (col < s.H && a.b) load_param<T, VE>(a.b, a.p_f32, col, b + i * VE);
    }
    const T *g = static_cast<const T *>(a.g) + n * a.g_sn;
    int slot = 0;
    for (int t0 = tb * s.tspan; t0 < t_end; t0 += TF) {
        const int tn = min(min(TF, t_end - t0), Tn - t0);  // valid frames of the block's TF
        if (tn > 0 && u0 < ue) {
            float f[TF][P];
            Raw<T, VE> rg[NV];
            auto fetch_g = [&](int u) {
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    const int col = (i * team + tid) * VE;
                    if (col < s.H) rg[i] = load_kept<T, VE>(g + u * a.g_su + col);
                }
            };
            auto sum_g = [&]() {
                float x = 0.0f;
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    if ((i * team + tid) * VE < s.H) {
                        float v[VE];
                        unpack<T, VE>(rg[i], v);
#pragma unroll
                        for (int e = 0; e < VE; ++e) x += v[e];
                    }
                }
                return warp_sum(x);
            };
            fetch_g(u0);
#pragma unroll
            for (int k = 0; k < TF; ++k) {
                const T *fr = static_cast<const T *>(a.f) + n * a.f_sn + (t0 + k) * a.f_st;
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    const int col = (i * team + tid) * VE;
#pragma unroll
                    for (int e = 0; e < VE; ++e) f[k][i * VE + e] = 0.0f;
                    if (col < s.H && k < tn) unpack<T, VE>(load_kept<T, VE>(fr + col), f[k] + i * VE);
                }
            }
            // One round gives TF sums and the sum of the next context's g: sg holds a warp's share of it.
            auto round = [&](float (&v)[TF], float g_part, float &g_sum) {
                if (lane == 0) sg[slot * 32 + warp] = g_part;
                const float t = block_sums<TF>(v, sm, slot);
                if (team == 32) __syncwarp();
                g_sum = 0.0f;
                for (int k = 0; k < (team >> 5); ++k) g_sum += sg[slot * 32 + k];
                slot ^= 1;
                return t;
            };
            // spread the lanes' values (lane l: value l * TF / 32) over the warp
            auto spread = [&](float mine, float (&v)[TF]) {
                __syncwarp();
                if ((lane & (SAME - 1)) == 0) bc[warp][lane / SAME] = mine;
                __syncwarp();
#pragma unroll
                for (int k = 0; k < TF; ++k) v[k] = bc[warp][k];
            };
            float v[TF], g_sum;
#pragma unroll
            for (int k = 0; k < TF; ++k) {
                v[k] = 0.0f;
#pragma unroll
                for (int i = 0; i < P; ++i) v[k] += f[k][i];
            }
            float mine = round(v, sum_g(), g_sum) * inv_h;
            if (a.fm && ub == 0 && warp == 0 && (lane & (SAME - 1)) == 0 && lane / SAME < tn)
                a.fm[static_cast<int64_t>(n) * s.T + t0 + lane / SAME] = mine;
            spread(mine, v);
#pragma unroll
            for (int k = 0; k < TF; ++k)
#pragma unroll
                for (int i = 0; i < P; ++i) f[k][i] -= v[k];
            for (int u = u0; u < ue; ++u) {
                const float gmean = g_sum * inv_h;
                if (a.gm && t0 == 0 && tid == 0) a.gm[static_cast<int64_t>(n) * s.U1 + u] = gmean;
                float gc[P];
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    const int col = (i * team + tid) * VE;
                    if (col < s.H) {
                        unpack<T, VE>(rg[i], gc + i * VE);
#pragma unroll
                        for (int e = 0; e < VE; ++e) gc[i * VE + e] -= gmean;
                    }
                }
                if (u + 1 < ue) fetch_g(u + 1);
#pragma unroll
                for (int k = 0; k < TF; ++k) {
                    v[k] = 0.0f;
#pragma unroll
                    for (int i = 0; i < NV; ++i) {
                        if ((i * team + tid) * VE < s.H) {
#pragma unroll
                            for (int e = i * VE; e < (i + 1) * VE; ++e) {
                                const float d = f[k][e] + gc[e];
                                v[k] = fmaf(d, d, v[k]);
                            }
                        }
                    }
                }
                mine = rsqrtf(fmaf(round(v, sum_g(), g_sum), inv_h, a.eps));
                const int64_t row0 = base + static_cast<int64_t>(t0) * pitch + u;
                if (a.rstd && warp == 0 && (lane & (SAME - 1)) == 0 && lane / SAME < tn) {
                    const int64_t row = row0 + static_cast<int64_t>(lane / SAME) * pitch;
                    if (!s.cu || row < s.packed_rows) a.rstd[row] = mine;
                }
                spread(mine, v);
#pragma unroll
                for (int k = 0; k < TF; ++k) {
                    const int64_t row = row0 + static_cast<int64_t>(k) * pitch;
                    if (k < tn && (!s.cu || row < s.packed_rows)) {
                        T *out = y + row * s.H;
#pragma unroll
                        for (int i = 0; i < NV; ++i) {
                            const int col = (i * team + tid) * VE;
                            if (col < s.H) {
                                float o[VE];
#pragma unroll
                                for (int e = 0; e < VE; ++e) {
                                    const int c = i * VE + e;
                                    o[e] = fmaf((f[k][c] + gc[c]) * v[k], w[c], b[c]);
                                }
                                store_raw<T, VE>(out + col, pack<T, VE>(o));
                            }
                        }
                    }
                }
            }
        }
        if (s.cu) continue;
        // padding rows of the padded layout are zeros
        for (int k = 0; k < min(TF, t_end - t0); ++k) {
            for (int u = (k < tn) ? max(u0, ue) : u0; u < u1; ++u) {
                T *out = y + (base + static_cast<int64_t>(t0 + k) * s.U1 + u) * s.H;
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    const int col = (i * team + tid) * VE;
                    if (col < s.H) store_raw<T, VE>(out + col, zero);
                }
            }
        }
    }
}

template <typename T, int VE, int P, int TF>
__global__ void __launch_bounds__(JN_MAX_THREADS) k_joint_norm_grad(const JnGradArgs a) {
    constexpr int NV = P / VE;
    constexpr int SAME = 16 / TF;  // lanes that hold the same of 2 * TF values
    extern __shared__ __align__(16) float acc_g[];  // [uspan][NV][team][VE]: dg of this block, private to the threads
    __shared__ float sm[2 * 2 * TF * 16];
    __shared__ __align__(16) float4 bc[16][TF];     // {r, r mean(q), r^3 mean(q s), -} per frame, a copy per warp
    pdl_wait();
    pdl_trigger();
    const JnShape &s = a.s;
    const int tid = threadIdx.x, team = blockDim.x, lane = tid & 31, warp = tid >> 5;
    const int ub = blockIdx.x % s.ublocks, q_ = blockIdx.x / s.ublocks;
    const int tb = q_ % s.tblocks, n = q_ / s.tblocks;
    const int Tn = s.frames(n), Un = s.contexts(n);
    const int u0 = ub * s.uspan, ue = min(min(u0 + s.uspan, s.U1), Un);
    const int ta = tb * s.tspan, te = min(min(ta + s.tspan, s.T), Tn);
    const int64_t base = s.first_row(n);
    const int pitch = s.row_pitch(Un);
    const float inv_h = 1.0f / static_cast<float>(s.H);
    float dw[P], db[P], w[P];
#pragma unroll
    for (int i = 0; i < P; ++i) {
        dw[i] = db[i] = 0.0f;
        w[i] = 1.0f;
    }
    if (ta < te && u0 < ue) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int col = (i * team + tid) * VE;
            if (col < s.H && a.w) load_param<T, VE>(a.w, a.p_f32, col, w + i * VE);
            for (int u = 0; u < ue - u0; ++u)
#pragma unroll
                for (int e = 0; e < VE; ++e) acc_g[(static_cast<size_t>(u * NV + i) * team + tid) * VE + e] = 0.0f;
        }
        const T *g = static_cast<const T *>(a.g) + n * a.g_sn;
        const T *dy = static_cast<const T *>(a.dy);
        int slot = 0;
        for (int t0 = ta; t0 < te; t0 += TF) {
            const int tn = min(TF, te - t0);
            float f[TF][P], df[TF][P];
#pragma unroll
            for (int k = 0; k < TF; ++k) {
                const T *fr = static_cast<const T *>(a.f) + n * a.f_sn + (t0 + k) * a.f_st;
                const float mean = k < tn ? a.fm[static_cast<int64_t>(n) * s.T + t0 + k] : 0.0f;
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    const int col = (i * team + tid) * VE;
#pragma unroll
                    for (int e = 0; e < VE; ++e) f[k][i * VE + e] = df[k][i * VE + e] = 0.0f;
                    if (col < s.H && k < tn) {
                        unpack<T, VE>(load_kept<T, VE>(fr + col), f[k] + i * VE);
#pragma unroll
                        for (int e = 0; e < VE; ++e) f[k][i * VE + e] -= mean;
                    }
                }
            }
            Raw<T, VE> rd[TF][NV], rg[NV];
            float r_next = 0.0f, gmean = 0.0f;
            const int kl = (lane / SAME) % TF;  // the frame whose reductions this lane finishes
            auto fetch = [&](int u) {
                const int64_t row0 = base + static_cast<int64_t>(t0) * pitch + u;
                const int64_t mine = row0 + static_cast<int64_t>(kl) * pitch;
                r_next = (kl < tn && (!s.cu || mine < s.packed_rows)) ? a.rstd[mine] : 0.0f;
                gmean = a.gm[static_cast<int64_t>(n) * s.U1 + u];
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    const int col = (i * team + tid) * VE;
                    if (col < s.H) rg[i] = load_kept<T, VE>(g + u * a.g_su + col);
                }
#pragma unroll
                for (int k = 0; k < TF; ++k) {
                    const int64_t row = row0 + static_cast<int64_t>(k) * pitch;
                    const bool ok = k < tn && (!s.cu || row < s.packed_rows);
#pragma unroll
                    for (int i = 0; i < NV; ++i) {
                        const int col = (i * team + tid) * VE;
                        rd[k][i] = Raw<T, VE>{};
                        if (col < s.H && ok) rd[k][i] = load_once<T, VE>(dy + row * s.H + col);
                    }
                }
            };
            fetch(u0);
            for (int u = u0; u < ue; ++u) {
                float d[TF][P], gc[P];
                float v[2 * TF];
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    unpack<T, VE>(rg[i], gc + i * VE);
#pragma unroll
                    for (int e = 0; e < VE; ++e) gc[i * VE + e] = (i * team + tid) * VE < s.H ? gc[i * VE + e] - gmean : 0.0f;
                }
#pragma unroll
                for (int k = 0; k < TF; ++k) {
                    v[k] = v[TF + k] = 0.0f;
#pragma unroll
                    for (int i = 0; i < NV; ++i) unpack<T, VE>(rd[k][i], d[k] + i * VE);
#pragma unroll
                    for (int e = 0; e < P; ++e) {
                        const float q = w[e] * d[k][e];
                        v[k] += q;
                        v[TF + k] = fmaf(q, f[k][e] + gc[e], v[TF + k]);
                    }
                }
                const float r = r_next;
                if (u + 1 < ue) fetch(u + 1);
                const float sum = block_sums<2 * TF>(v, sm, slot) * inv_h;
                slot ^= 1;
                __syncwarp();
                if (lane % SAME == 0) {
                    float *to = reinterpret_cast<float *>(&bc[warp][kl]);
                    if (lane < 16) {
                        to[0] = r;
                        to[1] = r * sum;
                    } else {
                        to[2] = r * r * r * sum;
                    }
                }
                __syncwarp();
                float dg[P];
#pragma unroll
                for (int e = 0; e < P; ++e) dg[e] = 0.0f;
#pragma unroll
                for (int k = 0; k < TF; ++k) {
                    const float4 c = bc[warp][k];
#pragma unroll
                    for (int e = 0; e < P; ++e) {
                        const float x = f[k][e] + gc[e];
                        const float dr = d[k][e] * c.x;
                        const float ds = fmaf(w[e], dr, fmaf(-c.z, x, -c.y));
                        df[k][e] += ds;
                        dg[e] += ds;
                        dw[e] = fmaf(dr, x, dw[e]);
                        db[e] += d[k][e];
                    }
                }
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    float *to = acc_g + (static_cast<size_t>((u - u0) * NV + i) * team + tid) * VE;
                    float old[VE];
                    unpack<float, VE>(*reinterpret_cast<const Raw<float, VE> *>(to), old);
#pragma unroll
                    for (int e = 0; e < VE; ++e) old[e] += dg[i * VE + e];
                    *reinterpret_cast<Raw<float, VE> *>(to) = pack<float, VE>(old);
                }
            }
#pragma unroll
            for (int k = 0; k < TF; ++k) {
                float *out = a.part_f + ((static_cast<int64_t>(n) * s.ublocks + ub) * s.T + t0 + k) * s.H;
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    const int col = (i * team + tid) * VE;
                    if (k < tn && col < s.H) store_raw<float, VE>(out + col, pack<float, VE>(df[k] + i * VE));
                }
            }
        }
        for (int u = u0; u < ue; ++u) {
            float *out = a.part_g + ((static_cast<int64_t>(n) * s.tblocks + tb) * s.U1 + u) * s.H;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int col = (i * team + tid) * VE;
                const float *from = acc_g + (static_cast<size_t>((u - u0) * NV + i) * team + tid) * VE;
                if (col < s.H) store_raw<float, VE>(out + col, *reinterpret_cast<const Raw<float, VE> *>(from));
            }
        }
    }
    float *pw = a.part_w + static_cast<int64_t>(blockIdx.x) * s.H;
    float *pb = pw + static_cast<int64_t>(gridDim.x) * s.H;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int col = (i * team + tid) * VE;
        if (col < s.H) {
            store_raw<float, VE>(pw + col, pack<float, VE>(dw + i * VE));
            store_raw<float, VE>(pb + col, pack<float, VE>(db + i * VE));
        }
    }
}

// The partial sums of k_joint_norm_grad, three kinds of blocks: [0, w_blocks) dw and db, then df, then dg.  A frame that
// no context range has touched (t >= lx) and a context beyond ly get zeros.
struct JnReduceArgs {
    JnShape s;
    const float *part_f, *part_g, *part_w;
    void *df, *dg, *dw, *db;   // any of them nullptr
    int p_f32;
    int64_t parts_w;           // blocks of the gradient launch
    int no_rows;               // there was none: every gradient is zero
    unsigned w_blocks, f_blocks;
};
template <typename T>
__global__ void __launch_bounds__(1024) k_joint_norm_reduce(const JnReduceArgs a) {
    __shared__ float sm[32][33];
    pdl_wait();
    const JnShape &s = a.s;
    if (blockIdx.x < a.w_blocks) {
        const int which = blockIdx.x & 1;
        void *out = which ? a.db : a.dw;
        if (out) reduce_columns<T>(ReduceArgs{a.part_w + which * a.parts_w * s.H, out, a.p_f32, a.parts_w, s.H}, blockIdx.x >> 1, 0, sm);
        return;
    }
    const bool is_f = blockIdx.x < a.w_blocks + a.f_blocks;
    const int64_t i = static_cast<int64_t>(blockIdx.x - a.w_blocks - (is_f ? 0 : a.f_blocks)) * 1024 + threadIdx.x;
    const int rows = is_f ? s.T : s.U1, parts_all = is_f ? s.ublocks : s.tblocks;
    void *out = is_f ? a.df : a.dg;
    const int64_t plane = static_cast<int64_t>(rows) * s.H;
    if (!out || i >= plane * s.N) return;
    const int n = static_cast<int>(i / plane);
    const int64_t at = i - n * plane;
    const int r = static_cast<int>(at / s.H);
    const int Tn = a.no_rows ? 0 : s.frames(n), Un = a.no_rows ? 0 : s.contexts(n);
    const int along = is_f ? Un : Tn, span = is_f ? s.uspan : s.tspan;
    const int parts = r < (is_f ? Tn : Un) ? (along + span - 1) / span : 0;
    const float *p = (is_f ? a.part_f : a.part_g) + static_cast<int64_t>(n) * parts_all * plane + at;
    float sum = 0.0f;
    for (int k = 0; k < parts; ++k) sum += p[k * plane];
    static_cast<T *>(out)[i] = from_float<T>(sum);
}

}  // namespace ctct
