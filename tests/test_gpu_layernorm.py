"""GPU parity of layer_norm, joint_layer_norm and joint_layer_norm_packed against their formulas in 64 bits.

Bounds come from the arithmetic (tests/joiner_ref.py); k = 64 + H / 512 covers the longest chain of additions of
a row (16 in a thread and 10 exchanges, or H / 512 chunks of 8 in the kernel for very long rows)."""
import pytest
import torch

from joiner_ref import U, check, half_step, norm_reference, valid_rows

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.fixture(scope="module")
def W():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import warp_ctct_b200
    from warp_ctct_b200 import _lib
    _lib.lib()
    return warp_ctct_b200


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _rand(g, shape, dtype=torch.float32, scale=1.0, shift=0.0):
    return (torch.randn(shape, generator=g, device=DEV) * scale + shift).to(dtype)


def _chain(H):
    return 64 + H / 64


def _check_ln(W, x, w, b, eps, dy):
    """Forward and all gradients of x (R, H); x may be strided."""
    leaves = [t.detach().requires_grad_(True) if t is not None else None for t in (x, w, b)]
    y = W.layer_norm(leaves[0], leaves[1], leaves[2], eps)
    assert y.dtype == x.dtype and y.shape == x.shape and y.is_contiguous()
    with torch.no_grad():
        assert torch.equal(W.layer_norm(x, w, b, eps), y)
    want = [t for t in leaves if t is not None]
    got = torch.autograd.grad(y, want, dy, retain_graph=True)
    again = torch.autograd.grad(y, want, dy)
    for p, q in zip(got, again):
        assert torch.equal(p, q)   # the same bits every time
    x64 = x.detach().double().reshape(-1, x.size(-1))
    pd = w.dtype if w is not None else b.dtype if b is not None else torch.float32
    val, tol = norm_reference(x64, w, b, eps, dy.reshape(x64.shape), x64.abs().amax(-1, keepdim=True), _chain(x.size(-1)),
                              64 + x64.size(0), x.dtype, pd)
    check("y", y.reshape(x64.shape), val["y"], tol["y"])
    got = list(got)
    check("dx", got.pop(0).reshape(x64.shape), val["ds"], tol["ds"] + half_step(val["ds"], x.dtype))
    if w is not None:
        check("dw", got.pop(0), val["dw"], tol["dw"])
    if b is not None:
        check("db", got.pop(0), val["db"], tol["db"])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,H", [(1, 1), (5, 2), (3, 7), (1, 8), (70, 64), (33, 255), (9, 256), (601, 257), (40, 512), (2000, 513),
                                    (7, 640), (50, 1024), (11, 1027), (5, 4096), (6, 4104), (3, 8200), (2, 9001), (4, 20000)])
def test_layer_norm(W, dtype, rows, H):
    g = _gen(rows * 31 + H)
    x = _rand(g, (rows, H), dtype, 1.5, 0.5)
    dy = _rand(g, (rows, H), dtype)
    for wdt in {torch.float32, dtype}:
        _check_ln(W, x, _rand(g, (H,), wdt, 0.3, 1.0), _rand(g, (H,), wdt, 0.3), 1e-5, dy)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,H", [(30000, 96), (20000, 520), (9001, 1031), (5003, 2047), (3000, 4100)])
def test_layer_norm_many_rows(W, dtype, rows, H):
    """More rows than the GPU has blocks: each takes several, and its share of the weights' gradients with it."""
    g = _gen(rows)
    _check_ln(W, _rand(g, (rows, H), dtype, 1.5, 0.5), _rand(g, (H,), torch.float32, 0.3, 1.0), _rand(g, (H,), torch.float32, 0.3), 1e-5,
              _rand(g, (rows, H), dtype))


@pytest.mark.parametrize("dtype", DTYPES)
def test_layer_norm_without_parameters_and_with_one(W, dtype):
    g = _gen(3)
    x, dy = _rand(g, (37, 96), dtype), _rand(g, (37, 96), dtype)
    w, b = _rand(g, (96,), dtype), _rand(g, (96,), dtype)
    _check_ln(W, x, None, None, 1e-3, dy)
    _check_ln(W, x, w, None, 1e-3, dy)
    _check_ln(W, x, None, b, 1e-3, dy)


@pytest.mark.parametrize("dtype", DTYPES)
def test_layer_norm_large_offset_and_constant_rows(W, dtype):
    """An offset of 200 deviations costs no more than the mean's own rounding; a constant row gives the bias."""
    g = _gen(4)
    x = _rand(g, (20, 300), torch.float32, 0.5, 100.0).to(dtype)
    x[3] = 7.0
    w, b, dy = _rand(g, (300,)), _rand(g, (300,)), _rand(g, (20, 300), dtype)
    _check_ln(W, x, w, b, 1e-5, dy)
    assert torch.equal(W.layer_norm(x, w, b)[3], b.to(dtype))


@pytest.mark.parametrize("dtype", DTYPES)
def test_layer_norm_strides_and_shapes(W, dtype):
    g = _gen(5)
    w, b = _rand(g, (48,)), _rand(g, (48,))
    wide = _rand(g, (10, 6, 100), dtype)
    for x in (wide[:, 2, 3:51], wide[:, 2, 8:56], wide[:, :, 4:52], wide[:, :, 52:].transpose(0, 1), wide[0, 0, :48],
              _rand(g, (48, 7), dtype).t(), wide[:1, 0, :48].expand(7, 48), wide[:, ::2, 16:64]):
        _check_ln(W, x, w, b, 1e-5, _rand(g, x.shape, dtype))
    x = wide[:, 0, :48]
    for dy in (torch.ones((), device=DEV, dtype=dtype).expand(10, 48), _rand(g, (48, 10), dtype).t(), _rand(g, (10, 99), dtype)[:, 7:55]):
        _check_ln(W, x, w, b, 1e-5, dy)
    _check_ln(W, x, _rand(g, (96,))[::2], _rand(g, (49,))[1:], 1e-5, _rand(g, (10, 48), dtype))   # strided, misaligned
    for shape in ((0, 48), (3, 0, 48)):
        e = torch.empty(shape, device=DEV, dtype=dtype, requires_grad=True)
        wl = w.clone().requires_grad_(True)
        y = W.layer_norm(e, wl, b)
        assert y.shape == e.shape
        dw, = torch.autograd.grad(y, [wl], torch.empty_like(y))
        assert torch.equal(dw, torch.zeros_like(dw))


def test_layer_norm_some_gradients_only(W):
    g = _gen(6)
    x, w, b, dy = _rand(g, (30, 80)), _rand(g, (80,)), _rand(g, (80,)), _rand(g, (30, 80))
    full = [t.clone().requires_grad_(True) for t in (x, w, b)]
    want = torch.autograd.grad(W.layer_norm(*full), full, dy)
    for keep in ((0,), (1,), (2,), (0, 2), (1, 2)):
        some = [t.clone().requires_grad_(i in keep) for i, t in enumerate((x, w, b))]
        got = torch.autograd.grad(W.layer_norm(*some), [some[i] for i in keep], dy)
        for i, t in zip(keep, got):
            assert torch.equal(t, want[i])
    y = W.layer_norm(*full)
    gx, = torch.autograd.grad(y, [full[0]], dy, create_graph=True)
    with pytest.raises(RuntimeError):   # differentiated once
        gx.sum().backward()


def _joint_args(seed, N, T, U1, H, dtype, wdt, lens):
    g = _gen(seed)
    f, gg = _rand(g, (N, T, H), dtype, 1.0, 0.3), _rand(g, (N, U1, H), dtype, 1.0, -0.2)
    w, b = _rand(g, (H,), wdt, 0.3, 1.0), _rand(g, (H,), wdt, 0.3)
    lx = ly = None
    if lens:
        lx = torch.randint(0, T + 1, (N,), generator=g, device=DEV, dtype=torch.int32)
        ly = torch.randint(0, U1, (N,), generator=g, device=DEV, dtype=torch.int32)
        lx[0], ly[0] = T, U1 - 1
    return g, f, gg, w, b, lx, ly


def _check_joint(W, f, g, lx, ly, w, b, eps, dy, packed):
    """dy: padded (N,T,U1,H); its padding is NaN here and must not be read."""
    N, T, H = f.shape
    U1 = g.size(1)
    valid = valid_rows(lx, ly, N, T, U1, DEV)
    leaves = [t.detach().requires_grad_(True) for t in (f, g, w, b)]
    dy = torch.where(valid.unsqueeze(-1), dy, torch.full_like(dy, float("nan")))
    if packed:
        call = lambda *a: W.joint_layer_norm_packed(a[0], a[1], lx, ly, a[2], a[3], eps, rows=int(valid.sum()))  # noqa: E731
    else:
        call = lambda *a: W.joint_layer_norm(a[0], a[1], lx, ly, a[2], a[3], eps)  # noqa: E731
    y = call(*leaves)
    up = dy[valid] if packed else dy
    got = torch.autograd.grad(y, leaves, up, retain_graph=True)
    for p, q in zip(got, torch.autograd.grad(y, leaves, up)):
        assert torch.equal(p, q)
    with torch.no_grad():
        assert torch.equal(call(f, g, w, b), y)
    if packed:
        assert y.shape == (int(valid.sum()), H)
    else:
        assert y.shape == (N, T, U1, H) and not y[~valid].any()   # padding rows are zeros
    rows = y if packed else y[valid]
    s = (f.double().unsqueeze(2) + g.double().unsqueeze(1))[valid]
    amax = (f.double().abs().amax(-1).unsqueeze(2) + g.double().abs().amax(-1).unsqueeze(1))[valid].unsqueeze(-1)
    # dw and db: chains of at most 64 frames x 128 contexts in a block, then the blocks
    mag = lambda t: (t.double() - t.double().mean(-1, keepdim=True)).abs()  # noqa: E731
    parts = (mag(f).unsqueeze(2) + mag(g).unsqueeze(1))[valid]
    val, tol = norm_reference(s, w, b, eps, dy[valid], amax, _chain(H), min(s.size(0), 64 * 128) + 64, f.dtype, w.dtype, parts)
    check("y", rows, val["y"], tol["y"])
    full = torch.zeros((N, T, U1, H), dtype=torch.float64, device=DEV)
    ds, e, terms = full.clone(), full.clone(), full.clone()
    ds[valid], e[valid], terms[valid] = val["ds"], tol["ds"], val["terms"]
    for name, t, dim, n in (("df", got[0], 2, U1), ("dg", got[1], 1, T)):
        want = ds.sum(dim)
        check(name, t, want, e.sum(dim) + (n + 8) * U * terms.sum(dim) + half_step(want, f.dtype))
    check("dw", got[2], val["dw"], tol["dw"])
    check("db", got[3], val["db"], tol["db"])
    return got


JOINT = [(1, 1, 1, 1), (2, 3, 4, 8), (3, 9, 1, 16), (2, 1, 5, 33), (1, 40, 70, 64), (3, 17, 23, 127), (2, 65, 35, 128), (2, 30, 12, 321),
         (5, 12, 9, 512), (2, 8, 7, 640), (2, 9, 6, 1028), (1, 5, 3, 2050), (1, 6, 4, 2052), (1, 3, 5, 4097), (1, 4, 3, 8192)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("shape", JOINT)
def test_joint_layer_norm(W, dtype, packed, shape):
    N, T, U1, H = shape
    g, f, gg, w, b, lx, ly = _joint_args(sum(shape), N, T, U1, H, dtype, dtype if H % 2 else torch.float32, True)
    _check_joint(W, f, gg, lx, ly, w, b, 1e-5, _rand(g, (N, T, U1, H), dtype), packed)


@pytest.mark.parametrize("dtype,packed,shape", [(torch.float32, True, (64, 128, 40, 64)), (torch.bfloat16, False, (64, 128, 40, 72)),
                                                (torch.float16, True, (4, 200, 25, 1030)), (torch.bfloat16, False, (3, 260, 50, 2048)),
                                                (torch.float32, False, (300, 30, 3, 40)), (torch.float16, True, (20, 150, 70, 96))])
def test_joint_layer_norm_large_ragged_batches(W, dtype, packed, shape):
    """More cells than blocks: runs of several, over ranges of contexts and over utterances, some of which have no frames."""
    N, T, U1, H = shape
    g, f, gg, w, b, lx, ly = _joint_args(sum(shape), N, T, U1, H, dtype, torch.float32, True)
    lx[1:N - 1:3] = 0
    lx[-1] = min(1, T)
    _check_joint(W, f, gg, lx, ly, w, b, 1e-5, _rand(g, (N, T, U1, H), dtype), packed)


def test_workspaces_may_hold_anything(W):
    """Memory that the allocator hands out again full of NaN does not show, not even for utterances without frames."""
    N, T, U1, H = 3, 9, 6, 64
    g, f, gg, w, b, _, ly = _joint_args(8, N, T, U1, H, torch.float32, torch.float32, True)
    lx = torch.tensor([9, 0, 4], dtype=torch.int32, device=DEV)
    leaves = [t.requires_grad_(True) for t in (f, gg, w, b)]
    first = None
    for _ in range(3):
        junk = [torch.full((k,), float("nan"), device=DEV) for k in (1 << 10, 1 << 12, 1 << 14, 1 << 16, 1 << 18, 1 << 20)]
        del junk
        y = W.joint_layer_norm(leaves[0], leaves[1], lx, ly, leaves[2], leaves[3])
        got = [y.detach(), *torch.autograd.grad(y, leaves, torch.ones_like(y))]
        assert all(bool(t.isfinite().all()) for t in got)
        first = first or got
        for p, q in zip(first, got):
            assert torch.equal(p, q)


@pytest.mark.parametrize("dtype", DTYPES)
def test_joint_layer_norm_full_lengths_strides_and_offsets(W, dtype):
    N, T, U1, H = 3, 21, 10, 96
    g, f, gg, w, b, _, _ = _joint_args(1, N, T, U1, H, dtype, torch.float32, False)
    dy = _rand(g, (N, T, U1, H), dtype)
    _check_joint(W, f, gg, None, None, w, b, 1e-5, dy, False)
    wide = _rand(g, (T, N, 2 * H + 3), dtype)
    for fs in (wide[..., :H].transpose(0, 1), wide[..., 5:5 + H].transpose(0, 1), f[:1].expand(N, T, H), f[:, :1].expand(N, T, H)):
        _check_joint(W, fs, gg, None, None, w, b, 1e-5, dy, False)
    _check_joint(W, f, gg[:, :1].expand(N, U1, H), None, None, w, b, 1e-5, dy, False)
    _check_joint(W, f.transpose(1, 2).contiguous().transpose(1, 2), gg, None, None, w, b, 1e-5, dy, False)
    # a common offset of f and the opposite one of g: each is centred by itself
    _check_joint(W, (f.float() + 50).to(dtype), (gg.float() - 40).to(dtype), None, None, w, b, 1e-5, dy, False)


def test_joint_layer_norm_values_behind_the_lengths_are_not_read(W):
    N, T, U1, H = 3, 20, 9, 64
    g, f, gg, w, b, _, _ = _joint_args(2, N, T, U1, H, torch.float32, torch.float32, False)
    lx = torch.tensor([20, 7, 0], dtype=torch.int64, device=DEV)     # 64-bit lengths, one utterance without frames
    ly = torch.tensor([3, 8, 5], dtype=torch.int64, device=DEV)
    for n in range(N):
        f[n, int(lx[n]):] = float("nan")
        gg[n, int(ly[n]) + 1:] = float("nan")
    dy = _rand(g, (N, T, U1, H))
    leaves = [t.requires_grad_(True) for t in (f, gg, w, b)]
    y = W.joint_layer_norm(leaves[0], leaves[1], lx, ly, leaves[2], leaves[3])
    grads = torch.autograd.grad(y, leaves, dy)
    assert all(bool(t.isfinite().all()) for t in (y, *grads))
    assert not grads[0][1, 7:].any() and not grads[0][2].any() and not grads[1][2].any() and not grads[1][0, 4:].any()
    # lengths outside the tensor are clamped into it
    big = torch.tensor([99, 7, -3], dtype=torch.int64, device=DEV)
    y2 = W.joint_layer_norm(f, gg, big, torch.where(ly == 8, 99, ly), w, b)
    assert torch.equal(y2, y)


def test_joint_layer_norm_packed_rows_that_do_not_match(W):
    N, T, U1, H = 4, 15, 6, 40
    g, f, gg, w, b, lx, ly = _joint_args(3, N, T, U1, H, torch.float32, torch.float32, True)
    full = W.joint_layer_norm_packed(f, gg, lx, ly, w, b)            # the number of rows read back
    assert torch.equal(full, W.pack_joint(W.joint_layer_norm(f, gg, lx, ly, w, b), lx, ly))
    n = full.size(0)
    for rows in (n + 37, n - 11, 1, 0):
        fl, wl = f.clone().requires_grad_(True), w.clone().requires_grad_(True)
        y = W.joint_layer_norm_packed(fl, gg, lx, ly, wl, b, rows=rows)
        k = min(n, rows)
        assert y.shape == (rows, H) and torch.equal(y[:k], full[:k]) and not y[k:].any()
        dy = _rand(g, (rows, H))
        df, dw = torch.autograd.grad(y, [fl, wl], dy)
        # the same as the whole tensor with a gradient that is zero where rows are missing
        f2, w2 = f.clone().requires_grad_(True), w.clone().requires_grad_(True)
        up = torch.zeros((n, H), device=DEV)
        up[:k] = dy[:k]
        df2, dw2 = torch.autograd.grad(W.joint_layer_norm_packed(f2, gg, lx, ly, w2, b, rows=n), [f2, w2], up)
        assert torch.equal(df, df2)
        check("dw", dw, dw2, 200 * U * dw2.abs().max().double() * torch.ones_like(dw2, dtype=torch.float64))


def test_joint_layer_norm_empty_and_partial_gradients(W):
    w = torch.ones(8, device=DEV, requires_grad=True)
    for N, T in ((0, 4), (2, 0)):
        f, g = torch.zeros((N, T, 8), device=DEV, requires_grad=True), torch.zeros((N, 3, 8), device=DEV, requires_grad=True)
        y = W.joint_layer_norm(f, g, weight=w)
        assert y.shape == (N, T, 3, 8)
        for t in torch.autograd.grad(y, [f, g, w], torch.ones_like(y)):
            assert not t.any()
    gen, f, g, w, b, lx, ly = _joint_args(4, 2, 13, 7, 64, torch.float32, torch.float32, True)
    dy = _rand(gen, (2, 13, 7, 64))
    full = [t.clone().requires_grad_(True) for t in (f, g, w, b)]
    want = torch.autograd.grad(W.joint_layer_norm(full[0], full[1], lx, ly, full[2], full[3]), full, dy)
    for keep in ((0,), (1,), (2,), (3,), (0, 1), (1, 3)):
        some = [t.clone().requires_grad_(i in keep) for i, t in enumerate((f, g, w, b))]
        got = torch.autograd.grad(W.joint_layer_norm(some[0], some[1], lx, ly, some[2], some[3]), [some[i] for i in keep], dy)
        for i, t in zip(keep, got):
            assert torch.equal(t, want[i]), (keep, i)


def test_gradients_against_differences(W):
    """Central differences of the 64-bit definition along random directions (truncation h^2, rounding 1e-16 / h)."""
    gen, f, g, w, b, lx, ly = _joint_args(5, 2, 9, 6, 48, torch.float32, torch.float32, True)
    valid = valid_rows(lx, ly, 2, 9, 6, DEV)
    dy = _rand(gen, (2, 9, 6, 48))
    leaves = [t.requires_grad_(True) for t in (f, g, w, b)]
    grads = torch.autograd.grad(W.joint_layer_norm(leaves[0], leaves[1], lx, ly, leaves[2], leaves[3]), leaves, dy)

    def value(args):
        s = args[0].unsqueeze(2) + args[1].unsqueeze(1)
        d = s - s.mean(-1, keepdim=True)
        y = d / (d.square().mean(-1, keepdim=True) + 1e-5).sqrt() * args[2] + args[3]
        return (y * dy.double())[valid].sum()

    base = [t.detach().double() for t in leaves]
    for i in range(4):
        v = _rand(gen, base[i].shape).double()
        h = 1e-4
        up, down = list(base), list(base)
        up[i], down[i] = base[i] + h * v, base[i] - h * v
        slope = (value(up) - value(down)) / (2 * h)
        got = (grads[i].double() * v).sum()
        # every product of the sum carries at most 200 steps of float32; truncation is below 1e-6 of the same sum here
        assert abs(got - slope) <= (200 * U + 1e-6) * (grads[i].double() * v).abs().sum() + 1e-6, (i, got.item(), slope.item())


def test_refusals(W):
    x = torch.randn(4, 8, device=DEV)
    w = torch.ones(8, device=DEV)
    f, g = torch.randn(2, 3, 8, device=DEV), torch.randn(2, 4, 8, device=DEV)
    for bad in (lambda: W.layer_norm(x.double()), lambda: W.layer_norm(x, w[:7]), lambda: W.layer_norm(x, w.half()),
                lambda: W.layer_norm(x.half(), w, w.half()), lambda: W.layer_norm(x, w.cpu()), lambda: W.layer_norm(x, eps=-1e-5),
                lambda: W.layer_norm(x, eps=float("nan")), lambda: W.layer_norm(torch.zeros((), device=DEV)),
                lambda: W.layer_norm(torch.zeros((3, 0), device=DEV)), lambda: W.joint_layer_norm(f, g.half()),
                lambda: W.joint_layer_norm(f, g[..., :7]), lambda: W.joint_layer_norm(f, g[:1]), lambda: W.joint_layer_norm(f[0], g[0]),
                lambda: W.joint_layer_norm(f, g, torch.ones(3, dtype=torch.int32, device=DEV)),
                lambda: W.joint_layer_norm(f, g, torch.ones(2, dtype=torch.int32)), lambda: W.joint_layer_norm(f, g[:, :0]),
                lambda: W.joint_layer_norm(f, g, weight=w.half()),
                lambda: W.joint_layer_norm_packed(f, g, torch.ones(2, dtype=torch.int32, device=DEV), torch.ones(2, dtype=torch.int32, device=DEV), rows=-1)):
        with pytest.raises(RuntimeError):
            bad()
    wide = torch.zeros((1, 1, 8193), device=DEV)
    with pytest.raises(RuntimeError, match="not supported"):
        W.joint_layer_norm(wide, wide)


def test_side_stream_and_captured_graph(W):
    """On a stream other than the default, and replayed from a graph with new inputs in the captured buffers."""
    gen, f, g, w, b, lx, ly = _joint_args(6, 3, 25, 11, 128, torch.bfloat16, torch.float32, True)
    rows = int(valid_rows(lx, ly, 3, 25, 11, DEV).sum())
    dy = _rand(gen, (rows, 128), torch.bfloat16)

    def step(f, g, w, b):
        f, g, w, b = (t.detach().requires_grad_(True) for t in (f, g, w, b))
        fn, gn = W.layer_norm(f, w, b), W.layer_norm(g, w, b)
        y = W.joint_layer_norm_packed(fn, gn, lx, ly, w, b, rows=rows)
        return [y.detach(), *torch.autograd.grad(y, [f, g, w, b], dy)]

    want = step(f, g, w, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(f, g, w, b)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for p, q in zip(got, want):
        assert torch.equal(p, q)
    graph = torch.cuda.CUDAGraph()
    cf, cg = torch.zeros_like(f), torch.zeros_like(g)
    with torch.cuda.graph(graph):
        out = step(cf, cg, w, b)
    for seed in (1, 2):
        gg = _gen(seed)
        nf, ng = _rand(gg, f.shape, f.dtype), _rand(gg, g.shape, g.dtype)
        cf.copy_(nf)
        cg.copy_(ng)
        graph.replay()
        for p, q in zip(out, step(nf, ng, w, b)):
            assert torch.equal(p, q)


def test_joint_layer_norm_beyond_32_bit_offsets(W):
    """A joint tensor of more than 2^32 elements: the last utterance is what it is by itself, forward and backward."""
    N, T, U1, H = 3, 4000, 700, 520
    assert N * T * U1 * H > 2 ** 32
    g = _gen(7)
    f, gg = _rand(g, (N, T, H), torch.bfloat16), _rand(g, (N, U1, H), torch.bfloat16)
    w, b = _rand(g, (H,), torch.float32), _rand(g, (H,), torch.float32)
    lx, ly = torch.tensor([3, 1, T], dtype=torch.int32, device=DEV), torch.tensor([2, 0, 4], dtype=torch.int32, device=DEV)
    leaves = [f.requires_grad_(True), gg.requires_grad_(True)]
    y = W.joint_layer_norm(f, gg, lx, ly, w, b)
    small = [f.detach()[2:].requires_grad_(True), gg.detach()[2:, :5].requires_grad_(True)]
    one = W.joint_layer_norm(small[0], small[1], None, None, w, b)
    assert torch.equal(y[2, :, :5], one[0])
    assert not y[1, 1:].any() and not y[0, :, 3:].any() and not y[2, :, 5:].any()
    dy = _rand(g, one.shape, torch.bfloat16)
    up = torch.zeros_like(y)
    up[2, :, :5] = dy[0]
    df, dg = torch.autograd.grad(y, leaves, up)
    sf, sg = torch.autograd.grad(one, small, dy)
    # the same terms in another grouping: each side's float32 sum is within T u of the sum of magnitudes
    for p, q in ((df[2:], sf), (dg[2:, :5], sg)):
        p, q = p.double(), q.double()
        assert (p - q).norm() <= torch.finfo(torch.bfloat16).eps * q.norm()
    assert not df[0].any() and not df[1].any() and not dg[0].any() and not dg[1].any()
