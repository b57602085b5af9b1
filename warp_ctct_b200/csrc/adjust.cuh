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
// bias and mask are read once per block.  Histories are counted by the whole block into shared memory, integers, so
// the order of the atomic additions does not matter.  Outputs that are masked are selected, not
// multiplied: NaN and infinities in masked places do not come through.
#pragma once

#include "elem.cuh"

namespace ctct {

constexpr int ADJ_THREADS = 256;
constexpr int ADJ_UNROLL = 4;   // frames whose loads are in flight together

struct AdjArgs {
    const void *x;             // logits; in the backward pass needed only where rho != 1
    int64_t x_sn;              // elements from row to row of a step's (N,V) logits (T = U1 = 1); unused otherwise
    const int *tokens;         // step: histories (N, L); joint: labels (N, U1 - 1); or nullptr
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
    int tiles;                 // blocks along the plane of U1 * V elements
    unsigned main_blocks;      // blocks beyond it clear packed rows behind the last utterance
};

template <typename T, int VE, bool GRAD>
__global__ void __launch_bounds__(ADJ_THREADS) k_adjust(const AdjArgs a) {
    __shared__ int count[ADJ_THREADS * VE];
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
    const int tile = blockIdx.x % a.tiles, q = blockIdx.x / a.tiles;
    const int chunk = q % a.chunks;
    const int64_t n = q / a.chunks;
    const int Tn = a.lx ? max(0, min(a.lx[n], a.T)) : a.T;
    const int Un = a.ly ? max(0, min(a.ly[n], a.U1 - 1)) + 1 : a.U1;
    const unsigned V = a.V, plane = static_cast<unsigned>(a.U1) * V;  // below 2^31
    const unsigned tile0 = static_cast<unsigned>(tile) * threads * VE;
    const unsigned at = tile0 + tid * VE;          // this thread's first element of the plane
    const int u_first = static_cast<int>(tile0 / V);
    const int u_last = min(static_cast<int>((min(tile0 + threads * VE, plane) - 1) / V), Un - 1);
    const int ta = chunk * a.tspan, tb = min(ta + a.tspan, a.T), te = max(ta, min(tb, Tn));
    const bool work = u_first < Un && ta < te;
    float rho = a.rho, presence = a.presence, frequency = a.frequency;
    if (a.rho_n) rho = a.rho_n[n];
    if (a.presence_n) presence = a.presence_n[n];
    if (a.frequency_n) frequency = a.frequency_n[n];
    const bool history = work && a.tokens && (rho != 1.0f || (!GRAD && (presence != 0.0f || frequency != 0.0f)));
    if (history) {  // the same for the whole block
        for (int i = tid; i < threads * VE; i += threads) count[i] = 0;
        __syncthreads();
        const int *tok = a.tokens + n * a.L;
        for (int u = u_first; u <= u_last; ++u) {
            const int len = a.tokens_len ? max(0, min(a.tokens_len[n], static_cast<int>(a.L))) : u;
            const int row = static_cast<int>(u * V - tile0);  // may be negative: the tile may begin inside the row
            for (int j = tid; j < len; j += threads) {
                const int v = tok[j];
                if (v < 0 || v >= a.V) continue;  // no token: ignored
                const int to = row + v;
                if (to >= 0 && to < threads * VE) atomicAdd(count + to, 1);
            }
        }
        __syncthreads();
    }
    if (at >= plane) return;
    const int u = static_cast<int>(at / V), v0 = static_cast<int>(at - u * V);
    const bool row_ok = u < Un;
    float add[VE];
    unsigned hit = 0, ok = 0;
#pragma unroll
    for (int e = 0; e < VE; ++e) add[e] = 0.0f;
    if (work && row_ok) {
        if (!GRAD && a.bias) load_param<T, VE>(a.bias, a.bias_f32, n * a.bias_sn + u * a.bias_su + v0, add);
        ok = (1u << VE) - 1;
        if (a.allowed) ok &= a.allowed[n * a.mask_sn + u * a.mask_su + (v0 >> 5)] >> (v0 & 31);
        if (history) {
#pragma unroll
            for (int e = 0; e < VE; ++e) {
                const int c = count[tid * VE + e];
                if (c > 0) {
                    hit |= 1u << e;
                    add[e] -= presence + frequency * static_cast<float>(c);
                }
            }
        }
    }
    const float inv_rho = 1.0f / rho;
    const bool scaled = hit && rho != 1.0f;
    // rows of this thread's elements: one every `pitch` elements
    const int64_t base = a.cu ? a.cu[n] * a.V : static_cast<int64_t>(n) * a.T * plane;
    const int64_t pitch = a.cu ? static_cast<int64_t>(Un) * a.V : static_cast<int64_t>(plane);
    const T *x = static_cast<const T *>(a.x), *dy = static_cast<const T *>(a.dy);
    const int64_t x_base = a.x_sn ? n * a.x_sn : base;
    int t_stop = row_ok ? te : ta;
    if (a.cu && row_ok) {   // rows beyond the packed tensor are not touched
        const int64_t rows_left = a.packed_rows - a.cu[n] - u;   // t * Un < rows_left
        const int64_t fit = rows_left > 0 ? (rows_left + Un - 1) / Un : 0;
        if (fit < t_stop) t_stop = static_cast<int>(fit);
    }
    float db[VE];
#pragma unroll
    for (int e = 0; e < VE; ++e) db[e] = 0.0f;
    const float ninf = -__int_as_float(0x7f800000);
    for (int t = ta; t < t_stop; t += ADJ_UNROLL) {
        Raw<T, VE> in[ADJ_UNROLL], grad[ADJ_UNROLL];
#pragma unroll
        for (int k = 0; k < ADJ_UNROLL; ++k) {
            if (t + k < t_stop) {
                const int64_t o = (t + k) * pitch + at;
                if (GRAD) grad[k] = load_once<T, VE>(dy + base + o);
                if (!GRAD || (scaled && out)) in[k] = load_once<T, VE>(x + x_base + o);
            }
        }
#pragma unroll
        for (int k = 0; k < ADJ_UNROLL; ++k) {
            if (t + k < t_stop) {
                float z[VE], g[VE];
                if (GRAD) {
                    unpack<T, VE>(grad[k], g);
#pragma unroll
                    for (int e = 0; e < VE; ++e) {
                        g[e] = (ok >> e & 1u) ? g[e] : 0.0f;
                        db[e] += g[e];
                    }
                    if (!out) continue;
                    if (scaled) {
                        unpack<T, VE>(in[k], z);
#pragma unroll
                        for (int e = 0; e < VE; ++e)
                            if ((hit & ok) >> e & 1u) g[e] *= z[e] > 0.0f ? inv_rho : rho;
                    }
                } else {
                    unpack<T, VE>(in[k], z);
                    if (scaled) {
#pragma unroll
                        for (int e = 0; e < VE; ++e)
                            if (hit >> e & 1u) z[e] *= z[e] > 0.0f ? inv_rho : rho;
                    }
#pragma unroll
                    for (int e = 0; e < VE; ++e) g[e] = (ok >> e & 1u) ? z[e] + add[e] : ninf;
                }
                store_raw<T, VE>(out + base + (t + k) * pitch + at, pack<T, VE>(g));
            }
        }
    }
    if (!a.cu && out)   // padding rows of the padded layout are zeros
        for (int t = t_stop; t < tb; ++t) store_raw<T, VE>(out + base + t * pitch + at, zero);
    if (GRAD && a.part) {
        float *p = a.part + (static_cast<int64_t>(n) * a.chunks + chunk) * plane + at;
#pragma unroll
        for (int e = 0; e < VE; ++e) p[e] = db[e];
    }
}

// bias gradient: out[o][c] = sum over p of part[o][p][c], a block for every 32 columns of every o
template <typename T>
__global__ void __launch_bounds__(1024) k_adjust_reduce(const ReduceArgs a) {
    __shared__ float sm[32][33];
    pdl_wait();
    const unsigned col_blocks = static_cast<unsigned>((a.C + 31) / 32);
    reduce_columns<T, 32, 32>(a, blockIdx.x % col_blocks, blockIdx.x / col_blocks, sm);
}

}  // namespace ctct
