// Adjustment of raw logits before the loss or before a decoder's choice: penalties for tokens that the history
// holds already, an additive bias, a mask of allowed tokens.
//
//   c(v) = times token v occurs in the row's history;  z = x
//   c > 0:  z = x > 0 ? x / rho : x * rho
//   z -= presence * [c > 0] + frequency * c;   z += bias[v];   y = allowed(v) ? z : -inf
//   dx = allowed ? dy * (c > 0 ? (x > 0 ? 1 / rho : rho) : 1) : 0;   dbias = sum over rows of allowed ? dy : 0
//
// Rows: (N,T,U1,V), where the history of context u is the utterance's first u labels, the packed (valid rows, V)
// of the same, or (N,V) of a decoder's step (T = U1 = 1) with a history of its own per row.
//
// What is done to an element depends on (n,u,v), not on the frame: a thread owns VE neighbouring elements of
// the U1 x V plane of an utterance, keeps what is added to them and two bits each in registers, and walks over
// frames, so that the passes are one streaming read and one streaming write of the rows (HBM-bound) and histories,
// bias and mask are read once per block: 6.2 TB/s forward at 32x256x65x512 f32 (258 us).  Histories are counted by the whole block into shared memory, integers, so
// the order of the atomic additions does not matter.  Outputs that are masked are selected, not
// multiplied: NaN and infinities in masked places do not come through.
#pragma once

#include "elem.cuh"

namespace ctct {

constexpr int ADJ_THREADS = 256;
constexpr int ADJ_UNROLL = 4;   // frames whose loads are in flight together
constexpr int ADJ_PRE = 4;      // tokens of a step's history that a thread asks for before anything else

struct AdjArgs {
    const void *x;             // logits; in the backward pass needed only where rho != 1
    int64_t x_sn;              // elements from row to row of a step's (N,V) logits (T = U1 = 1); unused otherwise
    const int *tokens;         // step: histories (N, L); joint: labels (N, U1 - 1); nullptr: none, or nothing to do with them
    const int *tokens_len;     // step: tokens per history; joint: nullptr (context u has u)
    int64_t L;                 // row pitch of `tokens`
    const int *lx, *ly;        // frames, labels per utterance, or nullptr: all
    const int64_t *cu;         // packed row offsets, or nullptr
    int64_t packed_rows;
    const void *bias;          // (V), (N,V) or (N,U1,V) by its strides, or nullptr
    int64_t bias_sn, bias_su;
    int bias_f32;
    const unsigned *allowed;   // words of (V), (N,V) or (N,U1,V) bits by its strides, or nullptr
    int64_t mask_sn, mask_su;
    float rho, presence, frequency;                    // for every row,
    const float *rho_n, *presence_n, *frequency_n;     // or per utterance (row of a step)
    void *y;                   // forward: adjusted logits; backward: dx, or nullptr
    const void *dy;            // backward only
    float *part;               // backward: bias gradient of every block, [N][chunks][U1 * V], or nullptr
    int N, T, U1, V;
    int tspan, chunks;         // frames of a block, blocks along T
    int classes;               // a block's frames are `classes` apart; `chunks` counts all classes of all runs
    int tiles;                 // blocks along the plane of U1 * V elements
    unsigned main_blocks;      // blocks beyond it clear packed rows behind the last utterance
};

// A thread's elements: NV chunks of VE neighbours, threads * VE apart.  STEP: one row per n (T = U1 = 1), without the
// walk over frames and with more elements per thread, since there the set-up of a block is most of its work.
// Four blocks of 256 threads on an SM (64 registers).  Three or four make little difference: forward and backward 555 and 558
// us at 32x256x65x512 f32, 729 and 717 at 16x512x129x1024 fp16.
template <typename T, int VE, int NV, bool GRAD, bool STEP>
__global__ void __launch_bounds__(ADJ_THREADS, 4) k_adjust(const AdjArgs a) {
    constexpr int NE = VE * NV, UNROLL = STEP ? 1 : ADJ_UNROLL;
    constexpr bool STAGE = GRAD && !STEP && VE * sizeof(T) == 16;   // logits beside repeated tokens go through shared memory
    __shared__ __align__(16) int count[ADJ_THREADS * NE];
    __shared__ uint4 xs[STAGE ? UNROLL * ADJ_THREADS : 1];
    pdl_wait();
    pdl_trigger();
    const int tid = threadIdx.x, threads = blockDim.x;
    const Raw<T, VE> zero = Raw<T, VE>{};
    T *out = static_cast<T *>(a.y);
    if (blockIdx.x >= a.main_blocks) {
        const int64_t end = a.packed_rows * a.V, step = static_cast<int64_t>(gridDim.x - a.main_blocks) * threads * VE;
        for (int64_t i = a.cu[a.N] * a.V + (static_cast<int64_t>(blockIdx.x - a.main_blocks) * threads + tid) * VE; i < end; i += step)
            store_raw<T, VE>(out + i, zero);
        return;
    }
    const unsigned q = blockIdx.x / static_cast<unsigned>(a.tiles), tile = blockIdx.x - q * a.tiles;
    const int chunk = STEP ? 0 : q % static_cast<unsigned>(a.chunks);
    const int64_t n = STEP ? q : q / static_cast<unsigned>(a.chunks);
    // Everything that needs no other load is asked for first, so that a block of a decoder's step pays one memory
    // latency, not a chain of them.
    const int *tok = a.tokens ? a.tokens + n * a.L : nullptr;
    int pre[ADJ_PRE], step_len = 0;
    if (tok && a.tokens_len) {
        step_len = a.tokens_len[n];
#pragma unroll
        for (int i = 0; i < ADJ_PRE; ++i) pre[i] = tid + i * threads < a.L ? __ldg(tok + tid + i * threads) : -1;
    }
    const float rho = a.rho_n ? a.rho_n[n] : a.rho;
    const float presence = a.presence_n ? a.presence_n[n] : a.presence;
    const float frequency = a.frequency_n ? a.frequency_n[n] : a.frequency;
    const int Tn = STEP ? 1 : a.lx ? max(0, min(a.lx[n], a.T)) : a.T;
    const int Un = STEP ? 1 : a.ly ? max(0, min(a.ly[n], a.U1 - 1)) + 1 : a.U1;
    const unsigned V = a.V, plane = STEP ? V : static_cast<unsigned>(a.U1) * V;  // below 2^31
    const unsigned tile0 = tile * threads * NE, tile1 = min(tile0 + threads * NE, plane);
    const int u_first = STEP ? 0 : static_cast<int>(tile0 / V);
    const int u_last = STEP ? 0 : min(static_cast<int>((tile1 - 1) / V), Un - 1);
    // the block's frames: ta, ta + ts, ... below tb
    const int ts = STEP ? 1 : a.classes, run = STEP ? 0 : chunk / ts;
    const int ta = STEP ? 0 : run * (a.tspan * ts) + (chunk - run * ts), tb = STEP ? 1 : min((run + 1) * (a.tspan * ts), a.T);
    const int te = max(ta, min(tb, Tn));
    const bool work = u_first < Un && ta < te;
    // rows of this thread's elements: one every `pitch` elements
    const bool packed = !STEP && a.cu;
    const int64_t base = packed ? a.cu[n] * a.V : STEP ? n * V : n * a.T * static_cast<int64_t>(plane);
    const int64_t pitch = packed ? static_cast<int64_t>(Un) * a.V : static_cast<int64_t>(plane);
    const T *x = static_cast<const T *>(a.x) + (a.x_sn ? n * a.x_sn : base);
    const T *dy = static_cast<const T *>(a.dy) + base;
    unsigned at[NV];       // place in the plane
    int u[NV], v0[NV], t_stop[NV];
    float add[NE];
    unsigned ok = 0;
#pragma unroll
    for (int c = 0; c < NV; ++c) {
        at[c] = tile0 + (c * threads + tid) * VE;
        u[c] = STEP ? 0 : static_cast<int>(at[c] / V);
        v0[c] = static_cast<int>(at[c] - u[c] * V);
        t_stop[c] = work && at[c] < plane && u[c] < Un ? te : ta;
        if (packed && t_stop[c] > ta) {   // rows beyond the packed tensor are not touched: t * Un < rows_left
            const int64_t rows_left = a.packed_rows - a.cu[n] - u[c];
            const int64_t fit = rows_left > 0 ? (rows_left + Un - 1) / Un : 0;
            if (fit < t_stop[c]) t_stop[c] = static_cast<int>(max(fit, static_cast<int64_t>(ta)));
        }
#pragma unroll
        for (int e = 0; e < VE; ++e) add[c * VE + e] = 0.0f;
        if (t_stop[c] > ta) {
            if (!GRAD && a.bias) load_param<T, VE>(a.bias, a.bias_f32, n * a.bias_sn + u[c] * a.bias_su + v0[c], add + c * VE);
            unsigned bits = (1u << VE) - 1;
            if (a.allowed) bits &= a.allowed[n * a.mask_sn + u[c] * a.mask_su + (v0[c] >> 5)] >> (v0[c] & 31);
            ok |= bits << (c * VE);
        }
    }
    // the stream: logits forward, their adjusted values' gradient backward, ADJ_UNROLL frames on their way
    const T *from = GRAD ? dy : x;
    Raw<T, VE> in[UNROLL][NV];
    auto fetch = [&](int t) {
#pragma unroll
        for (int k = 0; k < UNROLL; ++k)
#pragma unroll
            for (int c = 0; c < NV; ++c)
                if (t + k * ts < t_stop[c]) in[k][c] = load_once<T, VE>(from + (t + k * ts) * pitch + at[c]);
    };
    fetch(ta);
    const bool history = work && tok;
    if (history) {  // the same for the whole block
        if (NE % 4 == 0) {
            for (int i = tid; i < threads * NE / 4; i += threads) reinterpret_cast<int4 *>(count)[i] = make_int4(0, 0, 0, 0);
        } else {
            for (int i = tid; i < threads * NE; i += threads) count[i] = 0;
        }
        __syncthreads();
        auto note = [&](int row, int v) {   // `row`: place of the row's first element in the tile, may be negative
            if (v < 0 || v >= a.V) return;  // no token: ignored
            const int to = row + v;
            if (to >= 0 && to < threads * NE) atomicAdd(count + to, 1);
        };
        if (STEP || a.tokens_len) {
            const int len = max(0, min(step_len, static_cast<int>(a.L)));
#pragma unroll
            for (int i = 0; i < ADJ_PRE; ++i)
                if (tid + i * threads < len) note(-static_cast<int>(tile0), pre[i]);
            for (int j = tid + ADJ_PRE * threads; j < len; j += threads) note(-static_cast<int>(tile0), tok[j]);
        } else {
            for (int r = u_first; r <= u_last; ++r)
                for (int j = tid; j < r; j += threads) note(static_cast<int>(r * V - tile0), tok[j]);
        }
        __syncthreads();
    }
    unsigned hit = 0;
    if (history) {
#pragma unroll
        for (int c = 0; c < NV; ++c) {
            constexpr int W = VE < 4 ? VE : 4;
#pragma unroll
            for (int e = 0; e < VE; e += W) {
                int times[W];
                memcpy(times, __builtin_assume_aligned(&count[(c * threads + tid) * VE + e], 4 * W), sizeof(times));
#pragma unroll
                for (int i = 0; i < W; ++i)
                    if (times[i] > 0) {
                        hit |= 1u << (c * VE + e + i);
                        add[c * VE + e + i] -= presence + frequency * static_cast<float>(times[i]);
                    }
            }
        }
    }
    const bool scaled = hit && rho != 1.0f;
    const float inv_rho = scaled ? 1.0f / rho : 1.0f;
    float db[GRAD ? NE : 1];
#pragma unroll
    for (int e = 0; e < (GRAD ? NE : 1); ++e) db[e] = 0.0f;
    const float ninf = -__int_as_float(0x7f800000);
    int t_end = ta;
#pragma unroll
    for (int c = 0; c < NV; ++c) t_end = max(t_end, t_stop[c]);
    for (int t = ta; t < t_end; t += UNROLL * ts) {
        if (t > ta) fetch(t);
        if (STAGE && scaled && out) {   // a thread reads back what it copied itself: no barrier, and no registers
#pragma unroll
            for (int k = 0; k < UNROLL; ++k)
                if (t + k * ts < t_stop[0]) cp_async16(xs + k * ADJ_THREADS + tid, x + (t + k * ts) * pitch + at[0]);
            cp_async_commit();
            cp_async_wait<0>();
        }
#pragma unroll
        for (int k = 0; k < UNROLL; ++k)
#pragma unroll
            for (int c = 0; c < NV; ++c)
                if (t + k * ts < t_stop[c]) {
                    const int64_t o = (t + k * ts) * pitch + at[c];
                    float z[VE], g[VE];
                    unpack<T, VE>(in[k][c], z);
                    if (GRAD) {
#pragma unroll
                        for (int e = 0; e < VE; ++e) {
                            g[e] = (ok >> (c * VE + e) & 1u) ? z[e] : 0.0f;
                            db[(GRAD ? c * VE + e : 0)] += g[e];
                        }
                        if (!out) continue;
                        if (scaled) {   // only the few chunks that hold a repeated token
                            Raw<T, VE> rx;
                            if constexpr (STAGE)
                                memcpy(&rx, &xs[k * ADJ_THREADS + tid], sizeof(rx));
                            else
                                rx = load_once<T, VE>(x + o);
                            unpack<T, VE>(rx, z);
#pragma unroll
                            for (int e = 0; e < VE; ++e)
                                if ((hit & ok) >> (c * VE + e) & 1u) g[e] *= z[e] > 0.0f ? inv_rho : rho;
                        }
                    } else {
                        if (scaled) {
#pragma unroll
                            for (int e = 0; e < VE; ++e)
                                if (hit >> (c * VE + e) & 1u) z[e] *= z[e] > 0.0f ? inv_rho : rho;
                        }
#pragma unroll
                        for (int e = 0; e < VE; ++e) g[e] = (ok >> (c * VE + e) & 1u) ? z[e] + add[c * VE + e] : ninf;
                    }
                    store_raw<T, VE>(out + base + o, pack<T, VE>(g));
                }
    }
#pragma unroll
    for (int c = 0; c < NV; ++c) {
        if (at[c] >= plane) continue;
        if (!STEP && !packed && out)   // padding rows of the padded layout are zeros
            for (int t = ta; t < tb; t += ts)
                if (t >= t_stop[c]) store_raw<T, VE>(out + base + t * pitch + at[c], zero);
        if (GRAD && a.part) {
            constexpr int W = VE < 4 ? VE : 4;
            float *p = a.part + (n * a.chunks + chunk) * plane + at[c];
#pragma unroll
            for (int e = 0; e < VE; e += W) store_raw<float, W>(p + e, pack<float, W>(db + (GRAD ? c * VE + e : 0)));
        }
    }
}

// Rows that are no whole number of 16-byte vectors.  The plane of an utterance's frame is taken as one run of elements that
// begins somewhere inside a vector: a thread owns one aligned vector of it, wherever that stands against rows.  The run
// begins at the same place for frames that are a vector's number of elements apart, so a block's frames are that far
// apart, and what is added to an element stays in its thread.  Only the two ends of a plane are accessed
// element by element.  32x256x65x511 bf16, all rows valid: 414 us backward and 305 forward, with 2-byte accesses 1146 and
// 416; rows of 512, which are whole vectors, take 277 and 206.
template <typename T, bool GRAD>
__global__ void __launch_bounds__(ADJ_THREADS, 4) k_adjust_flat(const AdjArgs a) {
    constexpr int VE = 16 / static_cast<int>(sizeof(T));
    __shared__ __align__(16) int count[ADJ_THREADS * VE];
    __shared__ uint4 xs[GRAD ? ADJ_UNROLL * ADJ_THREADS : 1];
    pdl_wait();
    pdl_trigger();
    const int tid = threadIdx.x, threads = blockDim.x;
    const Raw<T, VE> zero = Raw<T, VE>{};
    T *out = static_cast<T *>(a.y);
    if (blockIdx.x >= a.main_blocks) {
        const int64_t end = a.packed_rows * a.V, step = static_cast<int64_t>(gridDim.x - a.main_blocks) * threads;
        for (int64_t i = a.cu[a.N] * a.V + static_cast<int64_t>(blockIdx.x - a.main_blocks) * threads + tid; i < end; i += step)
            out[i] = from_float<T>(0.0f);
        return;
    }
    const unsigned q = blockIdx.x / static_cast<unsigned>(a.tiles), tile = blockIdx.x - q * a.tiles;
    const int chunk = q % static_cast<unsigned>(a.chunks);
    const int64_t n = q / static_cast<unsigned>(a.chunks);
    const int *tok = a.tokens ? a.tokens + n * a.L : nullptr;
    int pre[ADJ_PRE], step_len = 0;
    if (tok && a.tokens_len) {
        step_len = a.tokens_len[n];
#pragma unroll
        for (int i = 0; i < ADJ_PRE; ++i) pre[i] = tid + i * threads < a.L ? __ldg(tok + tid + i * threads) : -1;
    }
    const float rho = a.rho_n ? a.rho_n[n] : a.rho;
    const float presence = a.presence_n ? a.presence_n[n] : a.presence;
    const float frequency = a.frequency_n ? a.frequency_n[n] : a.frequency;
    const int Tn = a.lx ? max(0, min(a.lx[n], a.T)) : a.T;
    const int Un = a.ly ? max(0, min(a.ly[n], a.U1 - 1)) + 1 : a.U1;
    const int V = a.V, plane = a.U1 * V, valid = Un * V;      // rows u < Un are the plane's first elements
    const int limit = a.cu ? valid : plane;                   // elements of a frame in memory
    const int ts = a.classes, run = chunk / ts;
    const int ta = run * (a.tspan * ts) + (chunk - run * ts), tb = min((run + 1) * (a.tspan * ts), a.T), te = max(ta, min(tb, Tn));
    const int64_t base = a.cu ? a.cu[n] * V : n * a.T * static_cast<int64_t>(plane), pitch = limit;
    const int shift = static_cast<int>((base + ta * pitch) & (VE - 1));
    const int p_tile = static_cast<int>(tile) * threads * VE - shift, p0 = p_tile + tid * VE;
    const int lo = max(p0, 0), hi = min(p0 + VE, limit);
    const bool whole = hi - lo == VE;
    const bool work = ta < te && p_tile < valid;
    const T *x = static_cast<const T *>(a.x) + base, *from = GRAD ? static_cast<const T *>(a.dy) + base : x;
    const int64_t total = a.cu ? a.packed_rows * V - base : 0;   // a packed tensor may end inside a frame
    // frames from which on the vector is not all inside the tensor
    const int t_vec = !whole ? ta : a.cu ? static_cast<int>(max(static_cast<int64_t>(0), min(static_cast<int64_t>(te), (total - hi) >= 0 ? (total - hi) / max(pitch, static_cast<int64_t>(1)) + 1 : 0))) : te;
    Raw<T, VE> in[ADJ_UNROLL];
    auto fetch = [&](int t) {
#pragma unroll
        for (int k = 0; k < ADJ_UNROLL; ++k)
            if (t + k * ts < t_vec) in[k] = load_once<T, VE>(from + (t + k * ts) * pitch + p0);
    };
    fetch(ta);
    float add[VE];
    unsigned ok = 0, hit = 0;   // allowed; row exists and token stands in the history
#pragma unroll
    for (int e = 0; e < VE; ++e) add[e] = 0.0f;
    if (work && lo < min(hi, valid)) {
        int u = lo / V, v = lo - u * V;
#pragma unroll
        for (int e = 0; e < VE; ++e) {
            if (p0 + e < lo || p0 + e >= valid) continue;
            bool allow = true;
            if (a.allowed) allow = a.allowed[n * a.mask_sn + u * a.mask_su + (v >> 5)] >> (v & 31) & 1u;
            if (!GRAD && a.bias) {
                const int64_t at = n * a.bias_sn + u * a.bias_su + v;
                add[e] = a.bias_f32 ? static_cast<const float *>(a.bias)[at] : to_float(static_cast<const T *>(a.bias)[at]);
            }
            if (allow) ok |= 1u << e;
            if (++v == V) {
                v = 0;
                ++u;
            }
        }
    }
    const bool history = work && tok;
    if (history) {  // the same for the whole block
        for (int i = tid; i < threads * VE / 4; i += threads) reinterpret_cast<int4 *>(count)[i] = make_int4(0, 0, 0, 0);
        __syncthreads();
        auto note = [&](int row, int v) {   // `row`: place of the row's first element in the tile, may be negative
            if (v < 0 || v >= V) return;    // no token: ignored
            const int to = row + v;
            if (to >= 0 && to < threads * VE) atomicAdd(count + to, 1);
        };
        if (a.tokens_len) {
            const int len = max(0, min(step_len, static_cast<int>(a.L)));
#pragma unroll
            for (int i = 0; i < ADJ_PRE; ++i)
                if (tid + i * threads < len) note(-p_tile, pre[i]);
            for (int j = tid + ADJ_PRE * threads; j < len; j += threads) note(-p_tile, tok[j]);
        } else {
            const int last = min((p_tile + threads * VE - 1) / V, Un - 1);
            for (int r = max(p_tile, 0) / V; r <= last; ++r)
                for (int j = tid; j < r; j += threads) note(r * V - p_tile, tok[j]);
        }
        __syncthreads();
#pragma unroll
        for (int e = 0; e < VE; e += 4) {
            const int4 c4 = *reinterpret_cast<const int4 *>(&count[tid * VE + e]);
            const int times[4] = {c4.x, c4.y, c4.z, c4.w};
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (times[i] > 0) {
                    hit |= 1u << (e + i);
                    add[e + i] -= presence + frequency * static_cast<float>(times[i]);
                }
        }
    }
    const int pad_from = valid - p0;   // elements from here on are padding rows: zeros
    const bool scaled = hit && rho != 1.0f;
    const float inv_rho = scaled ? 1.0f / rho : 1.0f;
    float db[GRAD ? VE : 1];
#pragma unroll
    for (int e = 0; e < (GRAD ? VE : 1); ++e) db[e] = 0.0f;
    const float ninf = -__int_as_float(0x7f800000);
    auto one = [&](int e, float z, float xv) {   // element e: the logit, or its gradient and the logit
        if (e >= pad_from) return 0.0f;
        const bool allow = ok >> e & 1u;
        if (GRAD) {
            if (!allow) z = 0.0f;
            db[GRAD ? e : 0] += z;
            return (hit & ok) >> e & 1u ? z * (xv > 0.0f ? inv_rho : rho) : z;
        }
        if (scaled && (hit >> e & 1u)) z *= z > 0.0f ? inv_rho : rho;
        return allow ? z + add[e] : ninf;
    };
    for (int t = ta; t < te; t += ADJ_UNROLL * ts) {
        if (t > ta) fetch(t);
        if (GRAD && scaled && out) {   // a thread reads back what it copied itself: no barrier, and no registers
#pragma unroll
            for (int k = 0; k < ADJ_UNROLL; ++k)
                if (t + k * ts < t_vec) cp_async16(xs + k * ADJ_THREADS + tid, x + (t + k * ts) * pitch + p0);
            cp_async_commit();
            cp_async_wait<0>();
        }
#pragma unroll
        for (int k = 0; k < ADJ_UNROLL; ++k) {
            const int tk = t + k * ts;
            if (tk >= te || lo >= hi) continue;
            const int64_t o = tk * pitch + p0;
            if (tk < t_vec) {
                float z[VE], xv[VE];
                unpack<T, VE>(in[k], z);
#pragma unroll
                for (int e = 0; e < VE; ++e) xv[e] = 0.0f;
                if (GRAD && scaled && out) {
                    Raw<T, VE> rx;
                    memcpy(&rx, &xs[GRAD ? k * ADJ_THREADS + tid : 0], sizeof(rx));
                    unpack<T, VE>(rx, xv);
                }
#pragma unroll
                for (int e = 0; e < VE; ++e) z[e] = one(e, z[e], xv[e]);
                if (!GRAD || out) store_raw<T, VE>(out + base + o, pack<T, VE>(z));
            } else {
#pragma unroll
                for (int e = 0; e < VE; ++e) {
                    if (p0 + e < lo || p0 + e >= hi || (a.cu && o + e >= total)) continue;
                    const float r = one(e, to_float(from[o + e]), GRAD && scaled && out ? to_float(x[o + e]) : 0.0f);
                    if (!GRAD || out) out[base + o + e] = from_float<T>(r);
                }
            }
        }
    }
    if (!a.cu && out && lo < hi)   // frames behind the last one are zeros
        for (int t = ta; t < tb; t += ts) {
            if (t < te) continue;
            if (whole) {
                store_raw<T, VE>(out + base + t * pitch + p0, zero);
            } else {
                for (int p = lo; p < hi; ++p) out[base + t * pitch + p] = from_float<T>(0.0f);
            }
        }
    if (GRAD && a.part) {
        float *p = a.part + (n * a.chunks + chunk) * plane + p0;
#pragma unroll
        for (int e = 0; e < VE; ++e)
            if (p0 + e >= 0 && p0 + e < plane) p[e] = db[GRAD ? e : 0];
    }
}

// Bias gradient out of the blocks' partial sums, out[o][c] = sum over p of part[o][p][c].  With few partials a thread
// adds up four columns by itself; with many a block has 32 columns and one of `segments` runs of partials, and
// where there is more than one run a second launch adds up the runs.
template <typename T>
__global__ void __launch_bounds__(256) k_adjust_reduce_few(const ReduceArgs a, int64_t outer) {
    pdl_wait();
    pdl_trigger();
    if (a.C % 4 == 0) {
        const int64_t i = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) * 4;
        if (i >= outer * a.C) return;
        const int64_t o = i / a.C;
        const float *p = a.part + o * (a.P - 1) * a.C + i;
        float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 8
        for (int k = 0; k < static_cast<int>(a.P); ++k) {
            const float4 v = *reinterpret_cast<const float4 *>(p + k * a.C);
            x[0] += v.x;
            x[1] += v.y;
            x[2] += v.z;
            x[3] += v.w;
        }
        if (a.out_f32)
            store_raw<float, 4>(static_cast<float *>(a.out) + i, pack<float, 4>(x));
        else
            store_raw<T, 4>(static_cast<T *>(a.out) + i, pack<T, 4>(x));
    } else {
        const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
        if (i >= outer * a.C) return;
        const float *p = a.part + i / a.C * (a.P - 1) * a.C + i;
        float x = 0.0f;
#pragma unroll 8
        for (int k = 0; k < static_cast<int>(a.P); ++k) x += p[k * a.C];
        if (a.out_f32)
            static_cast<float *>(a.out)[i] = x;
        else
            static_cast<T *>(a.out)[i] = from_float<T>(x);
    }
}

template <typename T>
__global__ void __launch_bounds__(1024) k_adjust_reduce(const ReduceArgs a, int segments, float *runs) {
    __shared__ float sm[32][33];
    pdl_wait();
    pdl_trigger();
    const unsigned col_blocks = static_cast<unsigned>((a.C + 31) / 32);
    const unsigned col = blockIdx.x % col_blocks, q = blockIdx.x / col_blocks;
    const int seg = q % segments;
    const int64_t o = q / segments, len = (a.P + segments - 1) / segments, first = min(seg * len, a.P);
    ReduceArgs r = a;
    r.part = a.part + (o * a.P + first) * a.C;
    r.P = min(len, a.P - first);
    if (segments > 1) {
        r.out = runs + (o * segments + seg) * a.C;
        r.out_f32 = 1;
    } else {
        r.out = a.out_f32 ? static_cast<void *>(static_cast<float *>(a.out) + o * a.C) : static_cast<void *>(static_cast<T *>(a.out) + o * a.C);
    }
    reduce_columns<T, 32, 32>(r, col, 0, sm);
}

}  // namespace ctct
