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
// number of values with every exchange) serves TF rows.  32x256x65x512 bf16 with 46 % of the rows valid: 112 us, 4.9 TB/s;
// bound by the latency of a round (DRAM half used).
//
// Backward: with r known, everything that reads dy is one pass that waits for nothing,
//   A[t] = sum_u r dy, B[u] = sum_t r dy, db = sum dy, c1 = sum_h w dy, c2 = sum_h w dy (f + g) (f, g centred)
// and the rest follows from k1 = r c1 / H and k2 = r^3 c2 / H, which are 1 / H of the data:
//   df[t] = w A[t] - sum_u k1 - f[t] sum_u k2 - sum_u k2 g[u]   (dg[u] with t and u exchanged)
//   dw    = sum_t f[t] A[t] + sum_u g[u] B[u]
// A block streams the rows of TF frames and a range of contexts with a thread's P columns of A in registers and of
// B in shared memory at places that only it touches; a warp leaves its share of c1 and c2 in shared
// memory and goes on.  Only behind the last context the block meets, forms k1 and k2 and adds their terms.  That is
// 7 float32 operations an element in the stream and 2 after it, where the direct form takes 12 with two
// reductions per row to wait for in the middle.  All sums are float32 and leave as partial rows that a second
// launch adds in a fixed order: no atomics, the same bits every time.  The same case: 156 us, DRAM a quarter used, 290 warp
// instructions a row; of it the terms behind the stream take about 35, c1 and c2 about 24 (timed with them left out).
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
    float *part_f;       // [N][ublocks][T][H]: df
    float *part_g;       // [segment][uspan][H]: dg
    float *part_w;       // [2][gridDim.x][H]: dw, db
    int64_t *cells;      // out: cells before utterance n (N + 1)
    int ring_offset;     // bytes of shared memory before the ring
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
constexpr int JG_REGS = 168, JG_WIDE_REGS = 64;   // registers per thread up to JG_MAX_THREADS, and of the wide kernels
constexpr int JG_BATCH = 8;             // contexts whose g is on its way together behind the stream
// Most blocks of TF frames that a thread block takes.  Few mean many partial sums, many mean fewer contexts a block, whose
// shared memory they share: forward and backward with 8, 16, 32 took 329, 298, 294 us at 32x256x65x512 bf16 (padded), 535, 488,
// 451 at 16x512x129x512 fp16 (packed).
constexpr int JG_BLOCKS = 32;
constexpr int JG_STAGES = 2;            // of a thread's ring of rows of dy
// Shared memory of a block (floats): B [uspan][P / 4][team][4] and dw [P / 2][team][2], private to the threads; c1 and c2
// [uspan][warps][2 * TF];
// k1 and k2 of the present frames [uspan][2 * TF]; r of the present frames [uspan][TF]; -k2 of all frames
// [JG_BLOCKS][uspan][TF]; sums of k1 and of -k2 over the frames [uspan][2].
inline size_t jg_ring_bytes(int threads, int esize) { return static_cast<size_t>(JG_STAGES) * JG_TF * JG_P * esize * threads; }
inline size_t jg_smem_bytes(int threads, int uspan) {
    return 4 * (static_cast<size_t>(uspan) * (threads * JG_P + threads / 32 * 2 * JG_TF + 3 * JG_TF + JG_BLOCKS * JG_TF + 2) + threads * JG_P);
}

// The work of the gradient launch: cells of TF frames x uspan contexts, utterance after utterance, range of contexts after
// range of contexts, along the frames last.  Block i of G (at most W) takes cells [i W / G, (i + 1) W / G) of the W that hold
// valid rows, so that blocks of ragged batches end together (forward and backward at 16x512x129x512 fp16: 490 us with fixed tiles of 16
// frames, 450 with this and runs of up to 128).  A block's run inside one (utterance, range) is a segment; segments are numbered block + N-th (utterance, range),
// which grows with every step along the runs, and each leaves one partial sum of dg.
__device__ __forceinline__ int64_t jg_cells(const JnShape &s, int n) {
    const int Tn = s.frames(n);
    return static_cast<int64_t>((Tn + JG_TF - 1) / JG_TF) * ((s.contexts(n) + s.uspan - 1) / s.uspan);
}

// REGS: registers per thread; six blocks of 64 threads on an SM with 168
template <typename T, int VE, int REGS>
__global__ void __maxnreg__(REGS) k_joint_norm_grad(const JnGradArgs a) {
    constexpr int P = JG_P, TF = JG_TF, NV = P / VE, Q = P / 2;
    extern __shared__ __align__(16) float acc_b[];
    pdl_wait();
    pdl_trigger();
    const JnShape &s = a.s;
    const int tid = threadIdx.x, team = blockDim.x, lane = tid & 31, warps = team >> 5;
    float *const dws = acc_b + static_cast<size_t>(s.uspan) * P * team;
    float *const cs = dws + P * team;
    float *const ks = cs + s.uspan * warps * 2 * TF;
    float *const rs = ks + s.uspan * 2 * TF;
    float *const k2s = rs + s.uspan * TF;
    float *const sums = k2s + JG_BLOCKS * s.uspan * TF;
    uint4 *const ring = reinterpret_cast<uint4 *>(reinterpret_cast<char *>(acc_b) + a.ring_offset) + tid;
    int col[NV], at[NV];
    bool in[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        col[i] = (i * team + tid) * VE;
        in[i] = col[i] < s.H;
        at[i] = in[i] ? col[i] : 0;
    }
    // this block's cells: a scan of the utterances' (a thread has a run of them)
    __shared__ int64_t scan[32];
    // where the block stands: utterance, cells of it that lie behind, cells still to do.  Here, not in registers,
    // since the loops below need all of those.
    __shared__ int64_t at_cell;
    __shared__ int at_n, left;
    const int per = (s.N + team - 1) / team, n_lo = min(tid * per, s.N), n_hi = min(n_lo + per, s.N);
    int64_t mine = 0;
    for (int i = n_lo; i < n_hi; ++i) mine += jg_cells(s, i);
    int64_t upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t v = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += v;
    }
    if (lane == 31) scan[tid >> 5] = upto;
    __syncthreads();
    int64_t before = upto - mine, W = 0;
    for (int i = 0; i < warps; ++i) {
        if (i < (tid >> 5)) before += scan[i];
        W += scan[i];
    }
    if (blockIdx.x == 0) {
        int64_t c = before;
        for (int i = n_lo; i < n_hi; ++i) {
            a.cells[i] = c;
            c += jg_cells(s, i);
        }
        if (tid == 0) a.cells[s.N] = W;
    }
    const int64_t G = min(static_cast<int64_t>(gridDim.x), W);   // every block below G has a cell, so has every segment
    const int64_t cell = blockIdx.x < G ? W * blockIdx.x / G : W;
    if (tid == 0) left = blockIdx.x < G ? static_cast<int>(W * (blockIdx.x + 1) / G - cell) : 0;
    if (before <= cell && cell < before + mine) {
        int64_t c = before;
        int i = n_lo;
        for (;; ++i) {
            const int64_t v = jg_cells(s, i);
            if (cell < c + v) break;
            c += v;
        }
        at_n = i;
        at_cell = cell - c;
    }
    __syncthreads();
    const float inv_h = 1.0f / static_cast<float>(s.H);
    const F2 z2 = f2(0.0f, 0.0f);
    F2 db[Q], w[Q];
    // dw is added to once per TF frames: it lives in shared memory, two columns at a time in the thread's own places
    auto add_dw = [&](int i, const F2 &x, const F2 &y) {
        F2 *to = reinterpret_cast<F2 *>(dws) + i * team + tid;
        *to = fma2(x, y, *to);
    };
#pragma unroll
    for (int i = 0; i < Q; ++i) {
        db[i] = z2;
        reinterpret_cast<F2 *>(dws)[i * team + tid] = z2;
    }
    {
        float wv[P];
#pragma unroll
        for (int i = 0; i < P; ++i) wv[i] = in[i / VE] ? 1.0f : 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (in[i] && a.w) load_param<T, VE>(a.w, a.p_f32, col[i], wv + i * VE);
        pair_up<P>(wv, w);
    }
    while (left > 0) {
        const int n = at_n;
        const int Tn = s.frames(n), Un = s.contexts(n);
        const int cells_t = (Tn + TF - 1) / TF;
        const int ub = static_cast<int>(at_cell / cells_t), tb = static_cast<int>(at_cell - static_cast<int64_t>(ub) * cells_t);
        const int run = min(cells_t - tb, left);
        const int u0 = ub * s.uspan, ue = min(min(u0 + s.uspan, s.U1), Un);
        const int ta = tb * TF, te = min(ta + run * TF, Tn);
        const int64_t base = s.first_row(n);
        const int pitch = s.row_pitch(Un);
        const int64_t pitch_h = static_cast<int64_t>(pitch) * s.H;
        for (int i = 0; i < (ue - u0) * (P / 4); ++i)
            *reinterpret_cast<float4 *>(acc_b + (static_cast<size_t>(i) * team + tid) * 4) = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int u = tid; u < ue - u0; u += team) sums[2 * u] = 0.0f;
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
        auto load_f = [&](int t0, int tn, F2 (&f)[TF][Q]) {
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
            }
        };
        // visit(u - u0, centred g) for the block's contexts, JG_BATCH of them on their way together
        auto for_g = [&](auto &&visit) {
            for (int b = u0; b < ue; b += JG_BATCH) {
                Raw<T, VE> rg[JG_BATCH][NV];
                float mean[JG_BATCH];
#pragma unroll
                for (int j = 0; j < JG_BATCH; ++j) {
                    const int u = min(b + j, ue - 1);
                    mean[j] = gms[u];
#pragma unroll
                    for (int i = 0; i < NV; ++i) rg[j][i] = load_kept<T, VE>(g + u * a.g_su + at[i]);
                }
#pragma unroll
                for (int j = 0; j < JG_BATCH; ++j) {
                    if (b + j < ue) {
                        F2 gc[Q];
                        centred_g(rg[j], mean[j], gc);
                        visit(b + j - u0, gc);
                    }
                }
            }
        };
        const int kl = (lane >> 2) & (TF - 1);   // the frame whose sums this lane ends up with
        for (int t0 = ta; t0 < te; t0 += TF) {
            const int tn = min(TF, te - t0);
            F2 f[TF][Q], A[TF][Q];
            load_f(t0, tn, f);
#pragma unroll
            for (int k = 0; k < TF; ++k)
#pragma unroll
                for (int i = 0; i < Q; ++i) A[k][i] = z2;
            int64_t row = base + static_cast<int64_t>(t0) * pitch + u0;   // of the first of the TF frames
            const T *dy = static_cast<const T *>(a.dy) + row * s.H;
            const T *gr = g + u0 * a.g_su;
            const float *my_r = a.rstd + row + static_cast<int64_t>(kl) * pitch;
            float *my_c = cs + (tid >> 5) * 2 * TF + (lane >> 2);   // this lane's of {c1 of TF frames, c2 of TF frames}
            // FULL: all frames and rows are there; threads without columns read column 0 with a weight of zero
            auto walk = [&](auto full_tag) {
                constexpr bool FULL = decltype(full_tag)::value;
                constexpr bool RING = VE * sizeof(T) == 16 && REGS > JG_WIDE_REGS;   // 1024 threads leave no room for it
                Raw<T, VE> rd[RING ? 1 : TF][NV], rg[NV];
                int p_slot = 0, c_slot = 0;
                auto issue = [&](bool some, int kn) {
                    if (some) {
                        uint4 *to = ring + p_slot * (TF * NV) * team;
#pragma unroll
                        for (int k = 0; k < TF; ++k) {
#pragma unroll
                            for (int i = 0; i < NV; ++i) {
                                if (FULL)
                                    cp_async16(to + (k * NV + i) * team, dy + k * pitch_h + at[i]);
                                else   // rows that are not there are filled with zeros, and not read
                                    cp_async16_or_zero(to + (k * NV + i) * team,
                                                       k < kn ? dy + k * pitch_h + at[i] : static_cast<const T *>(a.dy), k < kn);
                            }
                        }
                        dy += s.H;
                    }
                    cp_async_commit();
                    p_slot = p_slot + 1 == JG_STAGES ? 0 : p_slot + 1;
                };
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
                            rd[k][i] = load_once<T, VE>(dy + k * pitch_h + at[i]);
                        } else {
                            rd[k][i] = Raw<T, VE>{};
                            if (in[i] && k < kn) rd[k][i] = load_once<T, VE>(dy + k * pitch_h + at[i]);
                        }
                    }
                    if (k == TF - 1) dy += s.H;
                };
                auto fetch_g = [&]() {
#pragma unroll
                    for (int i = 0; i < NV; ++i) rg[i] = load_kept<T, VE>(gr + at[i]);
                    gr += a.g_su;
                };
                int kn = inside(row);
                if constexpr (RING) {
#pragma unroll
                    for (int i = 0; i < JG_STAGES - 1; ++i) issue(u0 + i < ue, inside(row + i));
                } else {
#pragma unroll
                    for (int k = 0; k < TF; ++k) fetch_row(k, kn);
                }
                fetch_g();
                float r_next = (FULL || kl < kn) ? *my_r : 0.0f, gmean = gms[u0];
                float *acc = acc_b + tid * 4;
                for (int u = u0; u < ue; ++u) {
                    const float r_mine = r_next;
                    F2 gc[Q], B[Q];
                    centred_g(rg, gmean, gc);
                    const bool more = u + 1 < ue;
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
                    [[maybe_unused]] const uint4 *slot = ring + c_slot * (TF * NV) * team;
                    if constexpr (RING) {
                        issue(u + JG_STAGES - 1 < ue, FULL ? TF : inside(row - 1 + JG_STAGES - 1));
                        cp_async_wait<JG_STAGES - 1>();
                        c_slot = c_slot + 1 == JG_STAGES ? 0 : c_slot + 1;
                    }
#pragma unroll
                    for (int k = 0; k < TF; ++k) {
                        float dv[P];
#pragma unroll
                        for (int i = 0; i < NV; ++i) {
                            if constexpr (RING) {
                                const uint4 raw = slot[(k * NV + i) * team];
                                memcpy(&rd[0][i], &raw, sizeof(rd[0][i]));
                            }
                            unpack<T, VE>(rd[RING ? 0 : k][i], dv + i * VE);
                        }
                        F2 d[Q];
                        pair_up<P>(dv, d);
                        if (!RING && more) fetch_row(k, kn);   // on its way for a whole step
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
                    if ((lane & 3) == 0) {
                        *my_c = sum;
                        if (tid < 4 * TF) rs[(u - u0) * TF + kl] = r_mine;
                    }
                    my_c += warps * 2 * TF;
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
            __syncthreads();
            for (int i = tid; i < (ue - u0) * TF; i += team) {
                const int u = i / TF, k = i % TF;
                const float r = rs[i];   // left there by the stream
                float c1 = 0.0f, c2 = 0.0f;
                for (int p = 0; p < warps; ++p) {
                    const float *c = cs + (u * warps + p) * 2 * TF + k;
                    c1 += c[0];
                    c2 += c[TF];
                }
                const float k1 = r * (c1 * inv_h), k2 = r * r * (r * (c2 * inv_h));
                ks[u * 2 * TF + k] = k1;
                ks[u * 2 * TF + TF + k] = k2;
                k2s[((t0 - ta) / TF * s.uspan + u) * TF + k] = -k2;
            }
            __syncthreads();
            for (int u = tid; u < ue - u0; u += team) {
                const float *k1 = ks + u * 2 * TF;
                sums[2 * u] += (k1[0] + k1[1]) + (k1[2] + k1[3]);
            }
            // dw takes A as it is; df = w A - sum k1 - f sum k2 - sum k2 g
            F2 k1_sum[TF / 2], k2_sum[TF / 2];
#pragma unroll
            for (int k = 0; k < TF / 2; ++k) k1_sum[k] = k2_sum[k] = z2;
#pragma unroll
            for (int i = 0; i < Q; ++i) {
                F2 sum = z2;
#pragma unroll
                for (int k = 0; k < TF; ++k) {
                    sum = fma2(f[k][i], A[k][i], sum);
                    A[k][i] = mul2(w[i], A[k][i]);
                }
                add_dw(i, sum, f2(1.0f, 1.0f));
            }
            {
                for_g([&](int u, const F2 (&gc)[Q]) {
                    const ulonglong2 p1 = *reinterpret_cast<const ulonglong2 *>(ks + u * 2 * TF);
                    const ulonglong2 p2 = *reinterpret_cast<const ulonglong2 *>(ks + u * 2 * TF + TF);
                    k1_sum[0] = add2(k1_sum[0], F2{p1.x});
                    k1_sum[1] = add2(k1_sum[1], F2{p1.y});
                    k2_sum[0] = add2(k2_sum[0], F2{p2.x});
                    k2_sum[1] = add2(k2_sum[1], F2{p2.y});
                    float k2[TF];
                    split(F2{p2.x}, k2[0], k2[1]);
                    split(F2{p2.y}, k2[2], k2[3]);
#pragma unroll
                    for (int k = 0; k < TF; ++k) {
                        const F2 m = f2(-k2[k], -k2[k]);
#pragma unroll
                        for (int i = 0; i < Q; ++i) A[k][i] = fma2(m, gc[i], A[k][i]);
                    }
                });
            }
            float s1[TF], s2[TF];
            unpair<TF>(k1_sum, s1);
            unpair<TF>(k2_sum, s2);
#pragma unroll
            for (int k = 0; k < TF; ++k) {
                float *out = a.part_f + ((static_cast<int64_t>(n) * s.ublocks + ub) * s.T + t0 + k) * s.H;
                const F2 m1 = f2(-s1[k], -s1[k]), m2 = f2(-s2[k], -s2[k]);
#pragma unroll
                for (int i = 0; i < Q; ++i) A[k][i] = add2(fma2(m2, f[k][i], A[k][i]), m1);
                float o[P];
                unpair<P>(A[k], o);
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
        // dw takes B as it is; dg = w B - sum k1 - g sum k2 - sum k2 f, TF frames at a time
        const int blocks = (te - ta + TF - 1) / TF;
        for (int u = tid; u < ue - u0; u += team) {
            float t = 0.0f;
            for (int i = 0; i < blocks; ++i)
#pragma unroll
                for (int k = 0; k < TF; ++k) t += k2s[(i * s.uspan + u) * TF + k];
            sums[2 * u + 1] = t;
        }
        __syncthreads();
        auto load_b = [&](int u, F2 (&B)[Q]) {
            const float *acc = acc_b + (static_cast<size_t>(u) * (P / 4) * team + tid) * 4;
#pragma unroll
            for (int e = 0; e < P / 4; ++e) {
                const ulonglong2 v = *reinterpret_cast<const ulonglong2 *>(acc + e * 4 * team);
                B[2 * e] = F2{v.x};
                B[2 * e + 1] = F2{v.y};
            }
        };
        auto store_b = [&](int u, const F2 (&B)[Q]) {
            float *acc = acc_b + (static_cast<size_t>(u) * (P / 4) * team + tid) * 4;
#pragma unroll
            for (int e = 0; e < P / 4; ++e) *reinterpret_cast<ulonglong2 *>(acc + e * 4 * team) = make_ulonglong2(B[2 * e].v, B[2 * e + 1].v);
        };
        for_g([&](int u, const F2 (&gc)[Q]) {
            F2 B[Q];
            load_b(u, B);
            const float k1 = sums[2 * u], k2 = sums[2 * u + 1];
            const F2 m1 = f2(-k1, -k1), m2 = f2(k2, k2);
#pragma unroll
            for (int e = 0; e < Q; ++e) {
                add_dw(e, gc[e], B[e]);
                B[e] = fma2(w[e], B[e], fma2(m2, gc[e], m1));
            }
            store_b(u, B);
        });
        for (int i = 0; i < blocks; ++i) {
            F2 f[TF][Q];
            load_f(ta + i * TF, min(TF, te - ta - i * TF), f);
#pragma unroll 4
            for (int u = 0; u < ue - u0; ++u) {
                F2 B[Q];
                load_b(u, B);
                float k2[TF];
                unpack<float, 4>(*reinterpret_cast<const uint4 *>(k2s + (i * s.uspan + u) * TF), k2);
#pragma unroll
                for (int k = 0; k < TF; ++k) {
                    const F2 m = f2(k2[k], k2[k]);
#pragma unroll
                    for (int e = 0; e < Q; ++e) B[e] = fma2(m, f[k][e], B[e]);
                }
                if (i + 1 < blocks) {
                    store_b(u, B);
                } else {
                    const int64_t segment = static_cast<int64_t>(blockIdx.x) + static_cast<int64_t>(n) * s.ublocks + ub;
                    float *out = a.part_g + (segment * s.uspan + u) * s.H;
                    float o[P];
                    unpair<P>(B, o);
#pragma unroll
                    for (int c = 0; c < NV; ++c) {
                        if (in[c]) {
                            constexpr int W = VE < 4 ? VE : 4;
#pragma unroll
                            for (int e = 0; e < VE; e += W) store_raw<float, W>(out + col[c] + e, pack<float, W>(o + c * VE + e));
                        }
                    }
                }
            }
        }
        __syncthreads();   // all have read where the block stands, and the sums of this segment
        if (tid == 0) {
            left -= run;
            int64_t c = at_cell + run;
            int m = n;
            if (left > 0)   // on to the next utterance with frames, if this one is done
                while (c == jg_cells(s, m)) {
                    ++m;
                    c = 0;
                }
            at_n = m;
            at_cell = c;
        }
        __syncthreads();
    }
    float *pw = a.part_w + static_cast<int64_t>(blockIdx.x) * s.H;
    float *pb = pw + static_cast<int64_t>(gridDim.x) * s.H;
    float ow[P], ob[P];
    unpair<P>(db, ob);
#pragma unroll
    for (int i = 0; i < Q; ++i) split(reinterpret_cast<const F2 *>(dws)[i * team + tid], ow[2 * i], ow[2 * i + 1]);
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

// The partial sums of k_joint_norm_grad, three kinds of blocks: [0, w_blocks) dw and db, then df, then dg, a warp per
// row.  A frame that no range of contexts has touched (t >= lx) and a context beyond ly get zeros.
constexpr int JR_THREADS = 256, JR_COLS = 8;   // JR_COLS columns of dw or db a block: whole 32-byte sectors, 32 partials at a time
struct JnReduceArgs {
    JnShape s;
    const float *part_f, *part_g, *part_w;
    const int64_t *cells;
    void *df, *dg, *dw, *db;   // any of them nullptr
    int p_f32;
    int64_t parts_w;           // blocks of the gradient launch
    int no_rows;               // there was none: every gradient is zero
    unsigned w_blocks, f_blocks;
    int w_cols;                // blocks along the columns of dw, and of db
};
template <typename T>
__global__ void __launch_bounds__(JR_THREADS) k_joint_norm_reduce(const JnReduceArgs a) {
    pdl_wait();
    const JnShape &s = a.s;
    if (blockIdx.x < a.w_blocks) {
        __shared__ float sm[JR_THREADS / JR_COLS][JR_COLS + 1];
        const int which = blockIdx.x / a.w_cols;
        void *out = which ? a.db : a.dw;
        if (out)
            reduce_columns<T, JR_COLS, JR_THREADS / JR_COLS>(ReduceArgs{a.part_w + which * a.parts_w * s.H, out, a.p_f32, a.parts_w, s.H},
                                                             blockIdx.x - which * a.w_cols, 0, sm);
        return;
    }
    const bool is_f = blockIdx.x < a.w_blocks + a.f_blocks;
    const int rows = is_f ? s.T : s.U1;
    void *out = is_f ? a.df : a.dg;
    const unsigned i = (blockIdx.x - a.w_blocks - (is_f ? 0 : a.f_blocks)) * (JR_THREADS / 32) + (threadIdx.x >> 5);
    if (!out || i >= static_cast<unsigned>(rows) * s.N) return;
    const int n = static_cast<int>(i / rows), r = static_cast<int>(i - static_cast<unsigned>(n) * rows);
    const int Tn = a.no_rows ? 0 : s.frames(n), Un = a.no_rows ? 0 : s.contexts(n);
    int parts = 0;
    int64_t plane = 0;     // from partial to partial
    const float *p = nullptr;
    if (is_f) {
        plane = static_cast<int64_t>(s.T) * s.H;
        p = a.part_f + (static_cast<int64_t>(n) * s.ublocks * s.T + r) * s.H;
        if (r < Tn) parts = (Un + s.uspan - 1) / s.uspan;
    } else if (r < Un && Tn > 0) {   // the segments of (n, r / uspan): one for every block that has cells of it
        const int ub = r / s.uspan;
        const int64_t W = a.cells[s.N], G = min(a.parts_w, W), cells_t = (Tn + JG_TF - 1) / JG_TF;
        const int64_t c0 = a.cells[n] + ub * cells_t, c1 = c0 + cells_t - 1;
        const int64_t b0 = ((c0 + 1) * G - 1) / W, b1 = ((c1 + 1) * G - 1) / W;   // the last block that begins at or before the cell
        plane = static_cast<int64_t>(s.uspan) * s.H;
        p = a.part_g + ((b0 + static_cast<int64_t>(n) * s.ublocks + ub) * s.uspan + (r - ub * s.uspan)) * s.H;
        parts = static_cast<int>(b1 - b0 + 1);
    }
    T *o = static_cast<T *>(out) + static_cast<int64_t>(i) * s.H;
    if (s.H % 4 == 0) {   // both buffers are whole vectors apart
        for (int col = (threadIdx.x & 31) * 4; col < s.H; col += 128) {
            float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 8
            for (int k = 0; k < parts; ++k) {
                const float4 v = *reinterpret_cast<const float4 *>(p + k * plane + col);
                x[0] += v.x;
                x[1] += v.y;
                x[2] += v.z;
                x[3] += v.w;
            }
            store_raw<T, 4>(o + col, pack<T, 4>(x));
        }
    } else {
        for (int col = threadIdx.x & 31; col < s.H; col += 32) {
            float sum = 0.0f;
#pragma unroll 8
            for (int k = 0; k < parts; ++k) sum += p[k * plane + col];
            o[col] = from_float<T>(sum);
        }
    }
}

}  // namespace ctct
