// extern "C" entry points of the joiner's operators: layer norm, the additive joiner's layer norm, the
// adjustment of logits (declared in include/ctct_b200.h).  Argument checks, choice of a kernel variant,
// workspace carving and launches; nothing here allocates or synchronises.
#include "../../include/ctct_b200.h"

#include <type_traits>

#include "adjust.cuh"
#include "elem.cuh"
#include "jointnorm.cuh"
#include "launch.cuh"
#include "layernorm.cuh"

using namespace ctct;

namespace {

size_t esize(int dtype) { return dtype == CTCT_F32 ? 4 : 2; }
bool dtype_ok(int dtype) { return dtype == CTCT_F32 || dtype == CTCT_F16 || dtype == CTCT_BF16; }
bool aligned(const void *p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

// call fn(T{}) with the element type of a dtype code
template <typename F>
int with_type(int dtype, F &&fn) {
    switch (dtype) {
    case CTCT_F32: return fn(float{});
    case CTCT_F16: return fn(__half{});
    default: return fn(__nv_bfloat16{});
    }
}

constexpr int64_t kMaxGrid = 0x7fffffff;
constexpr int64_t kMaxRun = (int64_t(1) << 31) - 4096;  // frames, contexts: loops step past the end by a block's share
constexpr int kSms = 148;  // SMs of a B200: grids and workspaces are sized by it

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// ---- layer norm ----
// Elements of a row per thread: 8 up to 256 per row (a warp each), else 16; float32 rows stay at 8 as long as
// 512 threads cover the row, since 16 float32 of x and dy and their successors do not fit 128 registers.
int ln_elems(int64_t H, int dtype) { return H <= 256 || (dtype == CTCT_F32 && H <= 8 * LN_WIDE_THREADS) ? 8 : 16; }
// Threads per SM: forward 1024 (85 us at 16000 x 4096 f32, 110 with 512).  Backward as many as its registers leave (up to 148
// a thread with 16 elements), so that all blocks run at a time; every block leaves a partial row of the weights'
// gradients (16000 x 1024 bf16: 29 us, 40 with twice the blocks).
constexpr int LN_FORWARD_THREADS = 1024;
int ln_backward_threads(int P, bool wide, int dtype) { return wide ? 512 : P == 16 ? 384 : dtype == CTCT_F32 ? 512 : 640; }
struct LnGeom {
    int P;
    bool wide, is_long;
    int threads;
    int64_t grid;
};
LnGeom ln_geom(int64_t rows, int64_t H, int dtype, bool backward) {
    const int64_t E = 16 / static_cast<int64_t>(esize(dtype));
    const int64_t span = H % E == 0 ? H : H + E - 1;   // a row may begin inside a vector
    LnGeom g;
    g.P = ln_elems(span, dtype);
    g.is_long = span > static_cast<int64_t>(g.P) * LN_WIDE_THREADS;
    g.wide = span > 32 * g.P;
    g.threads = g.is_long ? LN_WIDE_THREADS : g.wide ? static_cast<int>(ceil_div(span, 32 * g.P)) * 32 : 32 * LN_WARPS;
    const int64_t blocks = g.wide ? rows : ceil_div(rows, LN_WARPS);
    const int per_sm = backward ? ln_backward_threads(g.P, g.wide, dtype) : LN_FORWARD_THREADS;
    const int64_t most = static_cast<int64_t>(kSms) * (per_sm / g.threads > 0 ? per_sm / g.threads : 1);
    g.grid = blocks < most ? blocks : most;
    // a block's rows are the grid apart: a multiple of a vector's elements where they begin inside vectors
    if (H % E != 0 && !g.is_long) g.grid = g.grid < most ? ceil_div(g.grid, E) * E : g.grid / E * E;
    return g;
}

// `vec`: rows are whole vectors; `odd`: they are not, but follow one another from an aligned first one
template <typename T, int P, typename Args>
void ln_launch(const LnGeom &g, bool vec, bool odd, const Args &a, cudaStream_t st) {
    constexpr int E = 16 / static_cast<int>(sizeof(T));
    void (*kernel)(Args);
    if constexpr (std::is_same<Args, LnArgs>::value) {
        if (g.wide)
            kernel = vec ? k_ln_forward<T, E, P, true, false> : odd ? k_ln_forward<T, E, P, true, true> : k_ln_forward<T, 1, P, true, false>;
        else
            kernel = vec ? k_ln_forward<T, E, P, false, false> : odd ? k_ln_forward<T, E, P, false, true> : k_ln_forward<T, 1, P, false, false>;
    } else {
        if (g.wide)
            kernel = vec ? k_ln_backward<T, E, P, true, false> : odd ? k_ln_backward<T, E, P, true, true> : k_ln_backward<T, 1, P, true, false>;
        else
            kernel = vec ? k_ln_backward<T, E, P, false, false> : odd ? k_ln_backward<T, E, P, false, true> : k_ln_backward<T, 1, P, false, false>;
    }
    launch_pdl(kernel, dim3(static_cast<unsigned>(g.grid)), dim3(g.threads), 0, st, a);
}
template <typename T, int VE>
void ln_launch_long(const LnGeom &g, const LnArgs &a, cudaStream_t st) {
    launch_pdl(k_ln_forward_long<T, VE>, dim3(static_cast<unsigned>(g.grid)), dim3(g.threads), 0, st, a);
}
template <typename T, int VE>
void ln_launch_long(const LnGeom &g, const LnGradArgs &a, cudaStream_t st) {
    launch_pdl(k_ln_backward_long<T, VE>, dim3(static_cast<unsigned>(g.grid)), dim3(g.threads), 0, st, a);
}
template <typename T, typename Args>
void ln_dispatch(const LnGeom &g, bool vec, bool odd, const Args &a, cudaStream_t st) {
    constexpr int E = 16 / static_cast<int>(sizeof(T));
    if (g.is_long)
        vec ? ln_launch_long<T, E>(g, a, st) : ln_launch_long<T, 1>(g, a, st);
    else if (g.P == 8)
        ln_launch<T, 8>(g, vec, odd, a, st);
    else
        ln_launch<T, 16>(g, vec, odd, a, st);
}

// ---- the additive joiner's layer norm ----
struct JnGeom {
    int P, threads;
    int tspan, uspan, tblocks, ublocks;
    int64_t blocks;
    size_t smem;
};
// Forward: columns per thread and frames per block: 8 x 4 up to 2048 columns (16-byte accesses of 16-bit types, at
// most 256 threads), 32 x 1 beyond, where a row's sums need all threads of a block (a path for completeness).
constexpr int JN_THREADS = 256;
void jn_split(int64_t N, int64_t T, int64_t U1, int64_t tspan, int64_t uspan, JnGeom *g) {
    g->ublocks = static_cast<int>(ceil_div(U1, uspan));
    g->uspan = static_cast<int>(ceil_div(U1, g->ublocks));
    g->ublocks = static_cast<int>(ceil_div(U1, g->uspan));
    g->tspan = static_cast<int>(tspan);
    g->tblocks = static_cast<int>(ceil_div(T, tspan));
    g->blocks = N * g->tblocks * g->ublocks;
}
bool jn_forward_geom(int64_t N, int64_t T, int64_t U1, int64_t H, JnGeom *g) {
    if (H < 1 || H > CTCT_MAX_JOINT_H) return false;
    g->P = H <= 8 * JN_THREADS ? 8 : 32;
    g->threads = static_cast<int>(ceil_div(H, 32 * g->P)) * 32;
    const int TF = 32 / g->P;
    int64_t uspan = U1 < 32 ? U1 : 32;
    while (uspan > 1 && N * ceil_div(T, TF) * ceil_div(U1, uspan) < 2 * kSms) uspan = (uspan + 1) / 2;
    jn_split(N, T, U1, TF, uspan, g);
    return g->blocks <= kMaxGrid - 64;
}
// Backward: a thread has 8 columns, a block all of a row.  Registers say how many blocks an SM holds, their share of
// shared memory then how many contexts a block takes beside its ring.  As many blocks as the GPU holds at a
// time, or a multiple of it, each with an equal share of the cells, at most JG_BLOCKS of them.
bool jn_grad_geom(int64_t N, int64_t T, int64_t U1, int64_t H, int dtype, JnGeom *g) {
    if (H < 1 || H > CTCT_MAX_JOINT_H) return false;
    g->P = JG_P;
    g->threads = static_cast<int>(ceil_div(H, 32 * JG_P) * 32);
    const bool wide = g->threads > JG_MAX_THREADS;
    const int64_t regs = wide ? JG_WIDE_REGS : JG_REGS;
    int64_t resident = 65536 / (regs * g->threads);
    resident = resident < 1 ? 1 : resident > 12 ? 12 : resident;
    const int64_t ring = wide ? 0 : static_cast<int64_t>(jg_ring_bytes(g->threads, static_cast<int>(esize(dtype))));
    // of an SM's 228 KB a block pays 1 KB to the system, and 512 bytes of static memory and padding
    const int64_t share = 228 * 1024 / resident - 1024 - 512 - ring;
    const int64_t fixed = static_cast<int64_t>(jg_smem_bytes(g->threads, 0)), per = static_cast<int64_t>(jg_smem_bytes(g->threads, 1)) - fixed;
    int64_t uspan = (share - fixed) / per;
    uspan = uspan < 1 ? 1 : uspan > 32 ? 32 : uspan;
    if (uspan > U1) uspan = U1;
    const int64_t cells_t = ceil_div(T, JG_TF), slots = kSms * resident;
    while (uspan > 1 && N * cells_t * ceil_div(U1, uspan) < kSms) uspan = (uspan + 1) / 2;   // small: use all SMs
    jn_split(N, T, U1, JG_TF, uspan, g);
    const int64_t cells = g->blocks;
    g->blocks = slots * ceil_div(cells, slots * JG_BLOCKS);
    if (g->blocks > cells) g->blocks = cells;
    g->smem = jg_smem_bytes(g->threads, g->uspan);
    return g->blocks <= kMaxGrid;
}
bool jn_dims_ok(int64_t N, int64_t T, int64_t U1, int64_t H) {
    return N >= 0 && N <= 65535 && T >= 0 && U1 >= 1 && H >= 1 && H < (int64_t(1) << 31) && T < kMaxRun && U1 < kMaxRun &&
           T * U1 < (int64_t(1) << 31) && N * T < (int64_t(1) << 31) && N * U1 < (int64_t(1) << 31) && N * T * U1 < (int64_t(1) << 38);
}
struct JnSaved {
    size_t cu, fm, gm, rstd, total;
};
JnSaved jn_saved(int64_t N, int64_t T, int64_t U1, int64_t packed_rows, int want_grad) {
    JnSaved s;
    size_t o = 0;
    s.cu = o;
    if (packed_rows >= 0) o = align256(o + static_cast<size_t>(N + 1) * 8);
    s.fm = s.gm = s.rstd = o;
    if (want_grad) {
        s.gm = align256(s.fm + static_cast<size_t>(N * T) * 4);
        s.rstd = align256(s.gm + static_cast<size_t>(N * U1) * 4);
        o = align256(s.rstd + static_cast<size_t>(packed_rows >= 0 ? packed_rows : N * T * U1) * 4);
    }
    s.total = o;
    return s;
}
struct JnWs {
    size_t f, g, w, cells, total;
};
JnWs jn_ws(int64_t N, int64_t T, int64_t U1, int64_t H, const JnGeom &g) {
    JnWs w;
    w.f = 0;
    w.g = align256(static_cast<size_t>(N) * g.ublocks * T * H * 4);
    w.w = align256(w.g + static_cast<size_t>(g.blocks + N * g.ublocks) * g.uspan * H * 4);
    w.cells = align256(w.w + 2 * static_cast<size_t>(g.blocks) * H * 4);
    w.total = align256(w.cells + static_cast<size_t>(N + 1) * 8);
    return w;
}
JnShape jn_shape(const int32_t *lx, const int32_t *ly, const int64_t *cu, int64_t packed_rows, int64_t N, int64_t T, int64_t U1,
                 int64_t H, const JnGeom &g) {
    JnShape s;
    s.lx = lx;
    s.ly = ly;
    s.cu = cu;
    s.packed_rows = packed_rows;
    s.N = static_cast<int>(N);
    s.T = static_cast<int>(T);
    s.U1 = static_cast<int>(U1);
    s.H = static_cast<int>(H);
    s.tspan = g.tspan;
    s.uspan = g.uspan;
    s.tblocks = g.tblocks;
    s.ublocks = g.ublocks;
    return s;
}
template <typename T>
void jn_launch(const JnGeom &g, bool vec, const JnArgs &a, unsigned grid, cudaStream_t st) {
    constexpr int VE = 16 / static_cast<int>(sizeof(T));
    if (g.P == 8)
        launch_pdl(vec ? k_joint_norm<T, VE, 8, 4> : k_joint_norm<T, 1, 8, 4>, dim3(grid), dim3(g.threads), 0, st, a);
    else
        launch_pdl(vec ? k_joint_norm<T, VE, 32, 1> : k_joint_norm<T, 1, 32, 1>, dim3(grid),
                   dim3(g.threads), 0, st, a);
}
// ---- adjustment of logits ----
// Frames of a block: enough blocks for a few waves, and as many frames as that leaves, since the set-up of a
// block (histories, bias, mask) is paid once for all its frames.  Where planes of U1 V elements (packed: rows of V) are no
// whole number of vectors, frames come in classes that begin at the same place inside a vector.
struct AdjGeom {
    int64_t tspan, chunks, classes;
};
AdjGeom adj_geom(int64_t N, int64_t T, int64_t U1, int64_t V, int dtype, bool packed) {
    AdjGeom g;
    const int64_t E = 16 / static_cast<int64_t>(esize(dtype));
    g.classes = (packed ? V : U1 * V) % E == 0 ? 1 : T < E ? (T < 1 ? 1 : T) : E;
    const int64_t tiles = ceil_div(U1 * V, 1024);
    g.tspan = 64;
    while (g.tspan > ADJ_UNROLL && N * tiles * g.classes * ceil_div(T, g.tspan * g.classes) < 16 * kSms) g.tspan /= 2;
    g.chunks = T > 0 ? ceil_div(T, g.tspan * g.classes) * g.classes : 1;
    return g;
}
// Partial sums of the bias gradient: `outer` results of `P` partials of `C` columns.  Up to ADJ_FEW partials a thread
// adds them up (at N = 16, T = 512, U1 V = 132096 the blocks of 32 x 32 threads took 320 us for 8 partials
// a column, most of their threads idle); beyond, runs of about 512 so that one shared row of V columns still
// fills the GPU (8320 partials of 512 columns in one run: 52 us on 16 blocks).
constexpr int64_t ADJ_FEW = 16;
struct AdjReduce {
    int64_t outer, P, C, segments;
    size_t parts, total;   // bytes: partial sums, and with the runs behind them
};
AdjReduce adj_reduce(int64_t N, int64_t T, int64_t U1, int64_t V, int dtype, bool packed, int bias_kind) {
    const int64_t chunks = adj_geom(N, T, U1, V, dtype, packed).chunks;
    AdjReduce r;
    r.outer = bias_kind == 1 ? 1 : N;
    r.P = bias_kind == 1 ? N * chunks * U1 : bias_kind == 2 ? chunks * U1 : chunks;
    r.C = bias_kind == 3 ? U1 * V : V;
    r.segments = ceil_div(r.P, 512);
    if (r.segments > 32) r.segments = 32;
    if (r.segments < 1) r.segments = 1;
    r.parts = align256(static_cast<size_t>(N) * chunks * U1 * V * 4);
    r.total = r.parts + (r.segments > 1 ? align256(static_cast<size_t>(r.outer) * r.segments * r.C * 4) : 0);
    return r;
}
bool adj_dims_ok(int64_t N, int64_t T, int64_t U1, int64_t V) {
    return N >= 0 && N <= kMaxGrid && T >= 0 && U1 >= 1 && V >= 1 && U1 < (int64_t(1) << 31) && V < (int64_t(1) << 31) &&
           T < kMaxRun && U1 * V < kMaxRun;
}
// `vec`: rows are whole vectors; `flat`: they are not, but the tensors begin with one and their rows follow one another
template <typename T, bool GRAD>
int adj_launch(AdjArgs &a, bool vec, bool flat, int64_t N, bool tail, cudaStream_t st) {
    constexpr int VE = 16 / static_cast<int>(sizeof(T));
    const int64_t plane = static_cast<int64_t>(a.U1) * a.V;
    // one row per n: a decoder's step
    const bool step = a.T == 1 && a.U1 == 1 && !a.cu && !a.lx && !a.ly && (!a.tokens || a.tokens_len);
    // which has one frame to pay the set-up of an element with: odd rows go element by element (256 x 32001 bf16: 27 us, not 44)
    if (step) flat = false;
    const int64_t per = vec ? (step ? 2 * VE : VE) : flat ? VE : step ? 8 : 4;   // elements of a thread
    const int64_t span = vec || !flat ? plane : plane + VE - 1;                  // a run may begin inside a vector
    const int64_t need = ceil_div(span, per);
    const int threads = need < ADJ_THREADS ? static_cast<int>(ceil_div(need, 32) * 32) : ADJ_THREADS;
    a.tiles = static_cast<int>(ceil_div(span, threads * per));
    const int64_t blocks = N * a.tiles * a.chunks;
    if (blocks > kMaxGrid - 64) return CTCT_ERR_UNSUPPORTED;
    a.main_blocks = static_cast<unsigned>(blocks);
    auto kernel = vec    ? (step ? k_adjust<T, VE, 2, GRAD, true> : k_adjust<T, VE, 1, GRAD, false>)
                  : flat ? k_adjust_flat<T, GRAD>
                         : (step ? k_adjust<T, 1, 8, GRAD, true> : k_adjust<T, 1, 4, GRAD, false>);
    launch_pdl(kernel, dim3(static_cast<unsigned>(blocks + (tail ? 16 : 0))), dim3(threads), 0, st, a);
    return check_launch("adjust");
}

}  // namespace

extern "C" {

size_t ctct_b200_layer_norm_workspace_bytes(int64_t rows, int64_t H, int dtype) {
    if (rows < 0 || H < 1 || H >= (int64_t(1) << 31) || !dtype_ok(dtype)) return 0;
    return align256(2 * static_cast<size_t>(ln_geom(rows, H, dtype, true).grid) * H * 4);
}

int ctct_b200_layer_norm_forward(const void *x, int64_t x_stride, int dtype, int64_t rows, int64_t H, const void *weight,
                                 const void *bias, int param_f32, float eps, void *y, float *stats, void *stream) {
    if (rows < 0 || H < 1 || H >= (int64_t(1) << 31) || !dtype_ok(dtype) || (rows > 0 && (!x || !y))) return CTCT_ERR_ARG;
    if (rows == 0) return CTCT_OK;
    const size_t es = esize(dtype);
    const int64_t E = 16 / static_cast<int64_t>(es);
    const bool base_ok = aligned(x, 16) && aligned(y, 16);
    const bool vec = H % E == 0 && x_stride % E == 0 && base_ok && aligned(weight, 16) && aligned(bias, 16);
    const bool odd = H % E != 0 && x_stride == H && base_ok;
    LnArgs a{x, x_stride, weight, bias, param_f32 || dtype == CTCT_F32, eps, y, reinterpret_cast<float2 *>(stats), rows,
             static_cast<int>(H)};
    const LnGeom g = ln_geom(rows, H, dtype, false);
    return with_type(dtype, [&](auto t) {
        ln_dispatch<decltype(t)>(g, vec, odd, a, static_cast<cudaStream_t>(stream));
        return check_launch("layer_norm");
    });
}

int ctct_b200_layer_norm_backward(const void *dy, int64_t dy_stride, const void *x, int64_t x_stride, int dtype, int64_t rows,
                                  int64_t H, const void *weight, int param_f32, const float *stats, void *dx, void *dweight,
                                  void *dbias, void *workspace, size_t workspace_bytes, void *stream) {
    if (rows < 0 || H < 1 || H >= (int64_t(1) << 31) || !dtype_ok(dtype) || (rows > 0 && (!dy || !x || !stats))) return CTCT_ERR_ARG;
    const bool params = dweight || dbias;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const LnGeom g = ln_geom(rows, H, dtype, true);
    if (params && rows > 0 && (!workspace || !aligned(workspace, 256) || workspace_bytes < 2 * static_cast<size_t>(g.grid) * H * 4))
        return CTCT_ERR_WORKSPACE;
    const size_t es = esize(dtype);
    const int64_t E = 16 / static_cast<int64_t>(es);
    const bool base_ok = aligned(x, 16) && aligned(dy, 16) && aligned(dx, 16);
    const bool vec = H % E == 0 && x_stride % E == 0 && dy_stride % E == 0 && base_ok && aligned(weight, 16);
    const bool odd = H % E != 0 && x_stride == H && dy_stride == H && base_ok;
    const int p_f32 = param_f32 || dtype == CTCT_F32;
    LnGradArgs a{dy, dy_stride, x, x_stride, weight, p_f32, reinterpret_cast<const float2 *>(stats), dx,
                 params ? static_cast<float *>(workspace) : nullptr, rows, static_cast<int>(H)};
    return with_type(dtype, [&](auto t) -> int {
        using T = decltype(t);
        if (rows > 0) {
            ln_dispatch<T>(g, vec, odd, a, st);
            if (int rc = check_launch("layer_norm_grad")) return rc;
        }
        if (!params) return CTCT_OK;
        launch_pdl(k_ln_reduce<T>, dim3(static_cast<unsigned>(ceil_div(H, 32)), 2), dim3(1024), 0, st,
                   static_cast<const float *>(workspace), rows > 0 ? g.grid : int64_t(0), static_cast<int>(H), dweight, dbias, p_f32);
        return check_launch("layer_norm_reduce");
    });
}

size_t ctct_b200_joint_norm_saved_bytes(int64_t N, int64_t T, int64_t U1, int64_t packed_rows, int want_grad) {
    if (!jn_dims_ok(N, T, U1, 1)) return 0;
    return jn_saved(N, T, U1, packed_rows, want_grad).total;
}

size_t ctct_b200_joint_norm_workspace_bytes(int64_t N, int64_t T, int64_t U1, int64_t H, int dtype) {
    JnGeom g;
    if (!jn_dims_ok(N, T, U1, H) || !dtype_ok(dtype) || !jn_grad_geom(N, T, U1, H, dtype, &g)) return 0;
    return jn_ws(N, T, U1, H, g).total;
}

int ctct_b200_joint_norm_forward(const void *f, int64_t f_sn, int64_t f_st, const void *g, int64_t g_sn, int64_t g_su, int dtype,
                                 const int32_t *lx, const int32_t *ly, int64_t N, int64_t T, int64_t U1, int64_t H,
                                 int64_t packed_rows, const void *weight, const void *bias, int param_f32, float eps, void *y,
                                 int want_grad, void *saved, size_t saved_bytes, void *stream) {
    const bool packed = packed_rows >= 0;
    const int64_t rows = packed ? packed_rows : N * T * U1;
    if (!jn_dims_ok(N, T, U1, H) || !dtype_ok(dtype)) return CTCT_ERR_ARG;
    if (packed && (!lx || !ly) && N > 0) return CTCT_ERR_ARG;
    if (rows == 0) return CTCT_OK;
    if (!y || (N > 0 && T > 0 && (!f || !g))) return CTCT_ERR_ARG;
    const JnSaved sv = jn_saved(N, T, U1, packed_rows, want_grad);
    if (sv.total > 0 && (!saved || !aligned(saved, 256) || saved_bytes < sv.total)) return CTCT_ERR_WORKSPACE;
    JnGeom geo;
    if (!jn_forward_geom(N, T, U1, H, &geo)) return CTCT_ERR_UNSUPPORTED;
    char *sb = static_cast<char *>(saved);
    int64_t *cu = packed ? reinterpret_cast<int64_t *>(sb + sv.cu) : nullptr;
    if (packed)
        if (int rc = ctct_b200_packed_offsets(lx, ly, N, T, U1, cu, stream)) return rc;
    const int64_t E = 16 / static_cast<int64_t>(esize(dtype));
    const bool vec = H % E == 0 && f_sn % E == 0 && f_st % E == 0 && g_sn % E == 0 && g_su % E == 0 && aligned(f, 16) && aligned(g, 16) &&
                     aligned(y, 16) && aligned(weight, 16) && aligned(bias, 16);
    JnArgs a;
    a.s = jn_shape(lx, ly, cu, packed_rows, N, T, U1, H, geo);
    a.f = f;
    a.g = g;
    a.f_sn = f_sn;
    a.f_st = f_st;
    a.g_sn = g_sn;
    a.g_su = g_su;
    a.w = weight;
    a.b = bias;
    a.p_f32 = param_f32 || dtype == CTCT_F32;
    a.eps = eps;
    a.y = y;
    a.fm = want_grad ? reinterpret_cast<float *>(sb + sv.fm) : nullptr;
    a.gm = want_grad ? reinterpret_cast<float *>(sb + sv.gm) : nullptr;
    a.rstd = want_grad ? reinterpret_cast<float *>(sb + sv.rstd) : nullptr;
    a.main_blocks = static_cast<unsigned>(geo.blocks);
    const unsigned grid = static_cast<unsigned>(geo.blocks + (packed ? 16 : 0));
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    return with_type(dtype, [&](auto t) {
        jn_launch<decltype(t)>(geo, vec, a, grid, st);
        return check_launch("joint_norm");
    });
}

int ctct_b200_joint_norm_backward(const void *dy, const void *f, int64_t f_sn, int64_t f_st, const void *g, int64_t g_sn,
                                  int64_t g_su, int dtype, const int32_t *lx, const int32_t *ly, int64_t N, int64_t T, int64_t U1,
                                  int64_t H, int64_t packed_rows, const void *weight, int param_f32, const void *saved,
                                  size_t saved_bytes, void *df, void *dg, void *dweight, void *dbias, void *workspace,
                                  size_t workspace_bytes, void *stream) {
    const bool packed = packed_rows >= 0;
    const int64_t rows = packed ? packed_rows : N * T * U1;
    if (!jn_dims_ok(N, T, U1, H) || !dtype_ok(dtype)) return CTCT_ERR_ARG;
    if (packed && (!lx || !ly) && N > 0) return CTCT_ERR_ARG;
    JnGeom geo;
    if (!jn_grad_geom(N, T, U1, H, dtype, &geo)) return CTCT_ERR_UNSUPPORTED;
    if (!aligned(df, 16) || !aligned(dg, 16)) return CTCT_ERR_ARG;   // their sums are stored as vectors
    const JnSaved sv = jn_saved(N, T, U1, packed_rows, 1);
    const JnWs ws = jn_ws(N, T, U1, H, geo);
    if (rows > 0 && (!dy || (N > 0 && T > 0 && (!f || !g)))) return CTCT_ERR_ARG;
    if (rows > 0 && geo.blocks > 0 && (!saved || !aligned(saved, 256) || saved_bytes < sv.total)) return CTCT_ERR_WORKSPACE;
    if (geo.blocks > 0 && (!workspace || !aligned(workspace, 256) || workspace_bytes < ws.total)) return CTCT_ERR_WORKSPACE;
    const char *sb = static_cast<const char *>(saved);
    char *wb = static_cast<char *>(workspace);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int64_t E = 16 / static_cast<int64_t>(esize(dtype));
    const bool vec = H % E == 0 && f_sn % E == 0 && f_st % E == 0 && g_sn % E == 0 && g_su % E == 0 && aligned(f, 16) && aligned(g, 16) &&
                     aligned(dy, 16) && aligned(weight, 16);
    JnGradArgs a;
    a.s = jn_shape(lx, ly, packed && rows > 0 ? reinterpret_cast<const int64_t *>(sb + sv.cu) : nullptr, packed_rows, N, T, U1, H, geo);
    a.f = f;
    a.g = g;
    a.f_sn = f_sn;
    a.f_st = f_st;
    a.g_sn = g_sn;
    a.g_su = g_su;
    a.w = weight;
    a.p_f32 = param_f32 || dtype == CTCT_F32;
    a.dy = dy;
    a.fm = reinterpret_cast<const float *>(sb + sv.fm);
    a.gm = reinterpret_cast<const float *>(sb + sv.gm);
    a.rstd = reinterpret_cast<const float *>(sb + sv.rstd);
    a.part_f = reinterpret_cast<float *>(wb + ws.f);
    a.part_g = reinterpret_cast<float *>(wb + ws.g);
    a.part_w = reinterpret_cast<float *>(wb + ws.w);
    a.cells = reinterpret_cast<int64_t *>(wb + ws.cells);
    const bool some = rows > 0 && geo.blocks > 0;
    JnReduceArgs r;
    r.cells = a.cells;
    r.s = a.s;
    r.part_f = a.part_f;
    r.part_g = a.part_g;
    r.part_w = a.part_w;
    r.df = df;
    r.dg = dg;
    r.dw = dweight;
    r.db = dbias;
    r.p_f32 = a.p_f32;
    r.parts_w = some ? geo.blocks : 0;
    r.no_rows = !some;
    r.w_cols = static_cast<int>(ceil_div(H, JR_COLS));
    const int64_t w_blocks = dweight || dbias ? 2 * static_cast<int64_t>(r.w_cols) : 0;
    const int64_t f_blocks = ceil_div(N * T, JR_THREADS / 32), g_blocks = ceil_div(N * U1, JR_THREADS / 32);
    if (w_blocks + f_blocks + g_blocks > kMaxGrid) return CTCT_ERR_UNSUPPORTED;
    r.w_blocks = static_cast<unsigned>(w_blocks);
    r.f_blocks = static_cast<unsigned>(f_blocks);
    return with_type(dtype, [&](auto t) -> int {
        using E_ = decltype(t);
        constexpr int VE = sizeof(E_) == 4 ? 4 : 8;
        if (some) {
            auto kernel = geo.threads <= JG_MAX_THREADS ? (vec ? k_joint_norm_grad<E_, VE, JG_REGS> : k_joint_norm_grad<E_, 1, JG_REGS>)
                                                        : (vec ? k_joint_norm_grad<E_, VE, JG_WIDE_REGS> : k_joint_norm_grad<E_, 1, JG_WIDE_REGS>);
            // beyond 48 KB an attribute is needed; it belongs to the current device: set with the launch
            const size_t smem = align256(geo.smem) + (vec && geo.threads <= JG_MAX_THREADS ? jg_ring_bytes(geo.threads, sizeof(E_)) : 0);
            if (smem > 48 * 1024 &&
                cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)) != cudaSuccess)
                return check_launch("joint_norm_grad smem attribute");
            a.ring_offset = static_cast<int>(align256(geo.smem));
            launch_pdl(kernel, dim3(static_cast<unsigned>(geo.blocks)), dim3(geo.threads), smem, st, a);
            if (int rc = check_launch("joint_norm_grad")) return rc;
        }
        if (w_blocks + f_blocks + g_blocks == 0) return CTCT_OK;
        launch_pdl(k_joint_norm_reduce<E_>, dim3(static_cast<unsigned>(w_blocks + f_blocks + g_blocks)), dim3(JR_THREADS), 0, st, r);
        return check_launch("joint_norm_reduce");
    });
}

size_t ctct_b200_adjust_workspace_bytes(int64_t N, int64_t T, int64_t U1, int64_t V, int dtype, int packed, int bias_kind) {
    if (!adj_dims_ok(N, T, U1, V) || !dtype_ok(dtype) || bias_kind < 1 || bias_kind > 3) return 0;
    return adj_reduce(N, T, U1, V, dtype, packed != 0, bias_kind).total;
}

namespace {

struct AdjCall {
    const int32_t *tokens, *tokens_len;
    int64_t tokens_pitch;
    const int32_t *lx, *ly;
    int64_t N, T, U1, V, packed_rows;
    const int64_t *cu;
    const void *bias;
    int bias_kind, bias_f32;
    const int32_t *allowed;
    int mask_kind;
    float rho, presence, frequency;
    const float *rho_n, *presence_n, *frequency_n;
};
// the common part of both directions; CTCT_OK, or why the call is refused
int adj_fill(const AdjCall &c, int dtype, bool forward, AdjArgs *a) {
    if (!adj_dims_ok(c.N, c.T, c.U1, c.V) || !dtype_ok(dtype)) return CTCT_ERR_ARG;
    if (c.packed_rows >= 0 && (((!c.lx || !c.ly) && c.N > 0) || !c.cu)) return CTCT_ERR_ARG;
    if (c.bias_kind < 0 || c.bias_kind > 3 || c.mask_kind < 0 || c.mask_kind > 3) return CTCT_ERR_ARG;
    const bool rows = c.N > 0 && (c.packed_rows >= 0 ? c.packed_rows > 0 : c.T > 0);   // a tensor without elements may have no address
    if (c.mask_kind == 0 ? c.allowed != nullptr : rows && !c.allowed) return CTCT_ERR_ARG;
    if (forward && (c.bias_kind == 0 ? c.bias != nullptr : rows && !c.bias)) return CTCT_ERR_ARG;
    if (c.tokens_pitch < 0 || (c.tokens && !c.tokens_len && c.tokens_pitch < c.U1 - 1)) return CTCT_ERR_ARG;
    if (!c.rho_n && !(c.rho > 0.0f)) return CTCT_ERR_ARG;
    const int64_t words = ceil_div(c.V, 32);
    // histories that change nothing are not counted
    const bool counts = c.rho_n || c.rho != 1.0f || c.presence_n || c.presence != 0.0f || c.frequency_n || c.frequency != 0.0f;
    a->tokens = c.tokens_pitch > 0 && counts ? c.tokens : nullptr;
    a->tokens_len = c.tokens_len;
    a->L = c.tokens_pitch;
    a->lx = c.lx;
    a->ly = c.ly;
    a->cu = c.packed_rows >= 0 ? c.cu : nullptr;
    a->packed_rows = c.packed_rows;
    a->bias = c.bias;
    a->bias_f32 = c.bias_f32 || dtype == CTCT_F32;
    a->bias_sn = c.bias_kind == 2 ? c.V : c.bias_kind == 3 ? c.U1 * c.V : 0;
    a->bias_su = c.bias_kind == 3 ? c.V : 0;
    a->allowed = reinterpret_cast<const unsigned *>(c.allowed);
    a->mask_sn = c.mask_kind == 2 ? words : c.mask_kind == 3 ? c.U1 * words : 0;
    a->mask_su = c.mask_kind == 3 ? words : 0;
    a->rho = c.rho;
    a->presence = c.presence;
    a->frequency = c.frequency;
    a->rho_n = c.rho_n;
    a->presence_n = c.presence_n;
    a->frequency_n = c.frequency_n;
    a->N = static_cast<int>(c.N);
    a->T = static_cast<int>(c.T);
    a->U1 = static_cast<int>(c.U1);
    a->V = static_cast<int>(c.V);
    const AdjGeom g = adj_geom(c.N, c.T, c.U1, c.V, dtype, c.packed_rows >= 0);
    a->tspan = static_cast<int>(g.tspan);
    a->chunks = static_cast<int>(g.chunks);
    a->classes = static_cast<int>(g.classes);
    return CTCT_OK;
}

}  // namespace

int ctct_b200_adjust_forward(const void *logits, int64_t row_stride, int dtype, const int32_t *tokens, int64_t tokens_pitch,
                             const int32_t *tokens_lengths, const int32_t *lx, const int32_t *ly, int64_t N, int64_t T, int64_t U1,
                             int64_t V, int64_t packed_rows, int64_t *cu_rows, const void *bias, int bias_kind, int bias_f32,
                             const int32_t *allowed, int mask_kind, float repetition, float presence, float frequency,
                             const float *repetition_n, const float *presence_n, const float *frequency_n, void *out, void *stream) {
    AdjArgs a = {};
    const AdjCall c{tokens, tokens_lengths, tokens_pitch, lx, ly, N, T, U1, V, packed_rows, cu_rows, bias, bias_kind, bias_f32,
                    allowed, mask_kind, repetition, presence, frequency, repetition_n, presence_n, frequency_n};
    if (int rc = adj_fill(c, dtype, true, &a)) return rc;
    if (row_stride < 0 || (row_stride > 0 && (T != 1 || U1 != 1 || packed_rows >= 0)))
        return CTCT_ERR_ARG;
    const int64_t rows = packed_rows >= 0 ? packed_rows : N * T * U1;
    if (rows == 0) return CTCT_OK;
    if (!logits || !out) return CTCT_ERR_ARG;
    if (packed_rows >= 0)
        if (int rc = ctct_b200_packed_offsets(lx, ly, N, T, U1, cu_rows, stream)) return rc;
    a.x = logits;
    a.x_sn = row_stride;
    a.y = out;
    const size_t es = esize(dtype);
    const int64_t E = 16 / static_cast<int64_t>(es);
    const bool base_ok = aligned(logits, 16) && aligned(out, 16);
    const bool vec = V % E == 0 && row_stride % E == 0 && base_ok && aligned(bias, 16);
    const bool flat = base_ok && (row_stride == 0 || row_stride == V);
    return with_type(dtype, [&](auto t) {
        return adj_launch<decltype(t), false>(a, vec, flat, N, packed_rows >= 0, static_cast<cudaStream_t>(stream));
    });
}

int ctct_b200_adjust_backward(const void *dy, const void *logits, int64_t row_stride, int dtype, const int32_t *tokens,
                              int64_t tokens_pitch, const int32_t *tokens_lengths, const int32_t *lx, const int32_t *ly, int64_t N,
                              int64_t T, int64_t U1, int64_t V, int64_t packed_rows, const int64_t *cu_rows, int bias_kind,
                              int bias_f32, const int32_t *allowed, int mask_kind, float repetition, const float *repetition_n,
                              void *dx, void *dbias, void *workspace, size_t workspace_bytes, void *stream) {
    AdjArgs a = {};
    const AdjCall c{tokens, tokens_lengths, tokens_pitch, lx, ly, N, T, U1, V, packed_rows, cu_rows, nullptr, bias_kind, bias_f32,
                    allowed, mask_kind, repetition, 0.0f, 0.0f, repetition_n, nullptr, nullptr};
    if (int rc = adj_fill(c, dtype, false, &a)) return rc;
    if (!aligned(dbias, 16)) return CTCT_ERR_ARG;   // its sums are stored as vectors
    if ((dbias && bias_kind == 0) || row_stride < 0 || (row_stride > 0 && (T != 1 || U1 != 1 || packed_rows >= 0))) return CTCT_ERR_ARG;
    const int64_t rows = packed_rows >= 0 ? packed_rows : N * T * U1;
    const AdjReduce red = adj_reduce(N, T, U1, V, dtype, packed_rows >= 0, bias_kind);
    // one partial sum, laid out like the result: the blocks write the result themselves
    const bool direct = dbias && red.P == 1 && a.bias_f32;
    if (rows > 0 && (!dy || (dx && a.tokens && (repetition_n || repetition != 1.0f) && !logits))) return CTCT_ERR_ARG;
    // a packed tensor without frames has surplus rows only: no sums without utterances, but zeros in dx
    const bool sums = rows > 0 && N > 0, some = sums || (rows > 0 && dx);
    if (sums && dbias && !direct && (!workspace || !aligned(workspace, 256) || workspace_bytes < red.total)) return CTCT_ERR_WORKSPACE;
    a.x = logits;
    a.x_sn = row_stride;
    a.dy = dy;
    a.y = dx;
    a.part = dbias ? static_cast<float *>(direct ? dbias : workspace) : nullptr;
    const size_t es = esize(dtype);
    const int64_t E = 16 / static_cast<int64_t>(es);
    const bool base_ok = aligned(logits, 16) && aligned(dx, 16) && aligned(dy, 16);
    const bool vec = V % E == 0 && row_stride % E == 0 && base_ok && aligned(a.part, 16);
    const bool flat = base_ok && (row_stride == 0 || row_stride == V);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    return with_type(dtype, [&](auto t) -> int {
        using T_ = decltype(t);
        if (some)
            if (int rc = adj_launch<T_, true>(a, vec, flat, N, packed_rows >= 0 && dx, st)) return rc;
        if (!dbias || (direct && sums) || red.outer == 0) return CTCT_OK;
        float *parts = static_cast<float *>(workspace), *runs = sums ? parts + red.parts / 4 : nullptr;
        ReduceArgs r{parts, dbias, a.bias_f32, sums ? red.P : 0, red.C};   // no row: zeros
        auto few = [&](const ReduceArgs &r) {
            const int64_t blocks = ceil_div(red.outer * r.C, r.C % 4 == 0 ? 1024 : 256);
            if (blocks > kMaxGrid) return static_cast<int>(CTCT_ERR_UNSUPPORTED);
            launch_pdl(k_adjust_reduce_few<T_>, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, st, r, red.outer);
            return check_launch("adjust_reduce");
        };
        if (r.P <= ADJ_FEW) return few(r);
        const int64_t blocks = red.outer * red.segments * ceil_div(r.C, 32);
        if (blocks > kMaxGrid) return CTCT_ERR_UNSUPPORTED;
        launch_pdl(k_adjust_reduce<T_>, dim3(static_cast<unsigned>(blocks)), dim3(1024), 0, st, r, static_cast<int>(red.segments), runs);
        int rc = check_launch("adjust_reduce");
        if (rc || red.segments == 1) return rc;
        r.part = runs;
        r.P = red.segments;
        return few(r);
    });
}

}  // extern "C"
