"""GPU parity of adjust_logits, adjust_joint_logits and adjust_joint_logits_packed against their formulas in 64 bits.

Bounds: five float32 roundings of values no larger than the terms, then half a step of the output's type
(tests/joiner_ref.py); the bias gradient is a float32 sum of at most as many terms as there are rows."""
import pytest
import torch

from joiner_ref import U, adjust_reference, check, half_step, unpack_words, valid_rows

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
NINF = float("-inf")


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


def _mask(W, g, shape, V):
    m = torch.rand((*shape, V), generator=g, device=DEV) < 0.7
    if shape:
        m.view(-1, V)[-1] = False   # a row that is left with nothing
    return W.pack_token_mask(m)


def _counts(tokens, lens, V):
    R, L = tokens.shape
    one = (tokens.long().unsqueeze(-1) == torch.arange(V, device=DEV)) & (torch.arange(L, device=DEV) < lens.view(-1, 1)).unsqueeze(-1)
    return one.sum(1).double()


def _check_bias(name, db, dy, like, dims, rows):
    total = lambda t: (t.sum(dims) if dims else t).reshape(like.shape)  # noqa: E731  (an empty tuple means all to sum)
    want = total(dy)
    check(name, db, want, (rows + 8) * U * total(dy.abs()) + half_step(want, like.dtype))


STEP = [(1, 1, 0), (3, 2, 5), (4, 7, 1), (5, 33, 12), (2, 512, 16), (7, 1000, 300), (2, 4097, 70), (64, 264, 9), (1, 70001, 1500), (3, 16384, 33)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("R,V,L", STEP)
@pytest.mark.parametrize("bias_kind,mask_kind", [(0, 0), (1, 2), (2, 1)])
def test_step(W, dtype, R, V, L, bias_kind, mask_kind):
    g = _gen(R * 7 + V + L)
    x = _rand(g, (R, V), dtype, 2.0)
    tokens = torch.randint(0, max(1, min(V, L // 2 + 1)), (R, L), generator=g, device=DEV, dtype=torch.int32)
    lens = torch.randint(0, L + 1, (R,), generator=g, device=DEV, dtype=torch.int32)
    if L > 3:
        tokens[0, 1], tokens[0, 2] = -1, V     # no tokens: ignored
        lens[0] = L
    rho, pres, freq = (0.8 + 0.5 * torch.rand(R, generator=g, device=DEV) for _ in range(3))
    bias = None if bias_kind == 0 else _rand(g, (V,) if bias_kind == 1 else (R, V), torch.float32 if V % 2 else dtype)
    allowed = None if mask_kind == 0 else _mask(W, g, () if mask_kind == 1 else (R,), V)
    dy = _rand(g, (R, V), dtype)
    leaves = [t.requires_grad_(True) for t in (x, bias) if t is not None]
    y = W.adjust_logits(x, tokens, lens, bias, allowed, rho, pres, freq)
    assert y.dtype == dtype and y.is_contiguous()
    got = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    for p, q in zip(got, torch.autograd.grad(y, leaves, dy)):
        assert torch.equal(p, q)
    with torch.no_grad():
        assert torch.equal(W.adjust_logits(x, tokens, lens, bias, allowed, rho, pres, freq), y)
    ok = None if allowed is None else unpack_words(allowed, V)
    col = lambda t: t.double().view(-1, 1)  # noqa: E731
    val, tol, dz = adjust_reference(x.detach(), _counts(tokens, lens, V), None if bias is None else bias.detach(), ok, col(rho), col(pres),
                                    col(freq), dy, dtype)
    check("y", y, val["y"], tol["y"])
    check("dx", got[0], val["dx"], tol["dx"])
    if bias is not None:
        _check_bias("dbias", got[1], dz, bias, (0,) if bias_kind == 1 else (), R)


def test_step_forms(W):
    """Numbers for penalties, no history, all of a history, 64-bit tokens, rows that are apart."""
    g = _gen(1)
    scores = _rand(g, (6, 3, 200), torch.bfloat16, 2.0)
    x = scores[:, -1]
    tokens = torch.randint(0, 9, (6, 11), generator=g, device=DEV)
    assert torch.equal(W.adjust_logits(x), x)
    dense = W.adjust_logits(x.contiguous(), tokens, None, None, None, 1.3, 0.5, 0.25)
    assert torch.equal(W.adjust_logits(x, tokens, None, None, None, 1.3, 0.5, 0.25), dense)
    full = torch.full((6,), 11, device=DEV)
    assert torch.equal(W.adjust_logits(x, tokens, full, repetition_penalty=torch.full((6,), 1.3, device=DEV), presence_penalty=0.5,
                                       frequency_penalty=torch.full((6,), 0.25, device=DEV)), dense)
    val, tol, _ = adjust_reference(x, _counts(tokens, full, 200), None, None, 1.3, 0.5, 0.25, None, torch.bfloat16)
    check("y", dense, val["y"], tol["y"])
    odd = scores.view(6, 600)[:, 1:200]    # misaligned rows of 199
    assert torch.equal(W.adjust_logits(odd, tokens, None, None, None, 1.3, 0.5, 0.25),
                       W.adjust_logits(odd.contiguous(), tokens, None, None, None, 1.3, 0.5, 0.25))
    leaf = scores.clone().requires_grad_(True)
    dy = _rand(g, (6, 200), torch.bfloat16)
    got, = torch.autograd.grad(W.adjust_logits(leaf[:, 1], tokens, None, None, None, 1.3), [leaf], dy)
    flat = x = scores[:, 1].contiguous().requires_grad_(True)
    want, = torch.autograd.grad(W.adjust_logits(flat, tokens, None, None, None, 1.3), [flat], dy)
    assert torch.equal(got[:, 1], want) and not got[:, 0].any() and not got[:, 2].any()
    for shape in ((0, 10), ):
        assert W.adjust_logits(torch.zeros(shape, device=DEV), torch.zeros((0, 4), dtype=torch.int32, device=DEV)).shape == shape
    one = x.detach()[:1].expand(6, 200)      # the same row seen six times
    assert torch.equal(W.adjust_logits(one, tokens, full, repetition_penalty=1.3), W.adjust_logits(one.contiguous(), tokens, full, repetition_penalty=1.3))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [40, 37])
def test_what_stands_in_masked_places_does_not_come_through(W, dtype, V):
    g = _gen(2)
    x = _rand(g, (5, V), dtype)
    keep = torch.rand((5, V), generator=g, device=DEV) < 0.5
    keep[3] = False
    bad = torch.tensor([float("nan"), float("inf"), NINF, torch.finfo(dtype).min], device=DEV, dtype=dtype)
    dirty = torch.where(keep, x, bad[torch.randint(0, 4, (5, V), generator=g, device=DEV)])
    dy = _rand(g, (5, V), dtype)
    dirty_dy = torch.where(keep, dy, bad[torch.randint(0, 4, (5, V), generator=g, device=DEV)])
    words = W.pack_token_mask(keep)
    tokens = torch.arange(V, device=DEV).expand(5, V).contiguous()
    out = []
    for a, d in ((x, dy), (dirty, dirty_dy)):
        a = a.clone().requires_grad_(True)
        b = torch.zeros(V, device=DEV, requires_grad=True)
        y = W.adjust_logits(a, tokens, None, b, words, 1.5)
        out.append([y.detach(), *torch.autograd.grad(y, [a, b], d)])
    for p, q in zip(*out):
        assert torch.equal(p, q)
    assert bool((out[0][0][~keep] == NINF).all()) and not out[0][1][~keep].any()
    # unmasked -inf and the type's lowest value stay what they are under an additive bias of zero
    z = torch.full((1, V), NINF, device=DEV, dtype=dtype)
    assert bool((W.adjust_logits(z) == NINF).all())


JOINT = [(1, 1, 1, 2), (2, 3, 4, 8), (3, 9, 1, 16), (2, 70, 5, 33), (1, 40, 70, 64), (3, 17, 23, 127), (2, 65, 35, 512), (2, 30, 12, 1024),
         (1, 3, 6, 4100), (4, 100, 130, 3)]


def _joint_case(W, seed, N, T, U1, V, dtype, bias_kind, mask_kind):
    g = _gen(seed)
    x = _rand(g, (N, T, U1, V), dtype, 2.0)
    labels = torch.randint(0, max(1, min(V, U1 // 2 + 1)), (N, U1 - 1), generator=g, device=DEV, dtype=torch.int32)
    lx = torch.randint(0, T + 1, (N,), generator=g, device=DEV, dtype=torch.int32)
    ly = torch.randint(0, U1, (N,), generator=g, device=DEV, dtype=torch.int32)
    lx[0], ly[0] = T, U1 - 1
    shapes = {1: (), 2: (N,), 3: (N, U1)}
    bias = None if bias_kind == 0 else _rand(g, (*shapes[bias_kind], V), dtype if V % 2 else torch.float32)
    allowed = None if mask_kind == 0 else _mask(W, g, shapes[mask_kind], V)
    dy = _rand(g, (N, T, U1, V), dtype)
    return x, labels, lx, ly, bias, allowed, dy


def _wide(t, N, U1):
    return None if t is None else t if t.dim() == 1 else t[:, None, None] if t.dim() == 2 else t[:, None]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("shape", JOINT)
@pytest.mark.parametrize("bias_kind,mask_kind", [(1, 3), (2, 1), (3, 2), (0, 0)])
def test_joint(W, dtype, packed, shape, bias_kind, mask_kind):
    N, T, U1, V = shape
    x, labels, lx, ly, bias, allowed, dy = _joint_case(W, sum(shape), N, T, U1, V, dtype, bias_kind, mask_kind)
    valid = valid_rows(lx, ly, N, T, U1, DEV)
    nan = torch.full_like(dy, float("nan"))
    # padding is not read in either direction
    xin, din = torch.where(valid.unsqueeze(-1), x, nan), torch.where(valid.unsqueeze(-1), dy, nan)
    how = dict(bias=bias, allowed=allowed, repetition_penalty=1.25, presence_penalty=0.5, frequency_penalty=0.125)
    if packed:
        xin, din = x[valid], dy[valid]
    leaves = [t.requires_grad_(True) for t in (xin, bias) if t is not None]
    if packed:
        y = W.adjust_joint_logits_packed(xin, labels, lx, ly, max_frames=T, **how)
    else:
        y = W.adjust_joint_logits(xin, labels, lx, ly, **how)
        assert not y[~valid].any()
    got = torch.autograd.grad(y, leaves, din, retain_graph=True)
    for p, q in zip(got, torch.autograd.grad(y, leaves, din)):
        assert torch.equal(p, q)
    counts = torch.cat([torch.zeros((N, 1, V), device=DEV, dtype=torch.float64),
                        (labels.long().unsqueeze(-1) == torch.arange(V, device=DEV)).double().cumsum(1)], 1).unsqueeze(1)
    ok = None if allowed is None else _wide(unpack_words(allowed, V), N, U1)
    b4 = None if bias is None else _wide(bias.detach(), N, U1)
    val, tol, dz = adjust_reference(x.detach(), counts, b4, ok, 1.25, 0.5, 0.125, dy, dtype)
    pick = lambda t: t.expand(x.shape)[valid]  # noqa: E731
    rows = lambda t: t if packed else t[valid]  # noqa: E731
    check("y", rows(y), pick(val["y"]), pick(tol["y"]))
    check("dx", rows(got[0]), pick(val["dx"]), pick(tol["dx"]))
    if not packed:
        assert not got[0][~valid].any()
    if bias is not None:
        dz = torch.where(valid.unsqueeze(-1), dz.expand(x.shape), 0.0)
        _check_bias("dbias", got[1], dz, bias, {1: (0, 1, 2), 2: (1, 2), 3: (1,)}[bias_kind], int(valid.sum()))


@pytest.mark.parametrize("dtype,packed,V,bias_kind", [(torch.float32, False, 512, 1), (torch.float16, True, 509, 3), (torch.bfloat16, False, 510, 2),
                                                      (torch.bfloat16, True, 264, 1), (torch.float32, True, 203, 1)])
def test_joint_large(W, dtype, packed, V, bias_kind):
    """Blocks that walk over many frames, and many partial sums of the bias gradient."""
    test_joint(W, dtype, packed, (12, 300, 33, V), bias_kind, 3)


def test_nothing_to_adjust(W):
    """No rows, no frames: gradients of the bias are zeros; 64-bit tokens beyond 32 bits are no tokens."""
    for shape in ((0, 5, 3, 8), (2, 0, 3, 8)):
        x = torch.zeros(shape, device=DEV, requires_grad=True)
        for bias_shape in ((8,), (shape[0], 8), (shape[0], 3, 8)):
            b = torch.ones(bias_shape, device=DEV, requires_grad=True)
            y = W.adjust_joint_logits(x, torch.ones((shape[0], 2), dtype=torch.int32, device=DEV), bias=b, repetition_penalty=1.5)
            assert y.shape == shape
            dx, db = torch.autograd.grad(y, [x, b], torch.ones_like(y))
            assert dx.shape == shape and db.shape == b.shape and not db.any()
    x = torch.randn((2, 9), device=DEV)
    far = torch.tensor([[2 ** 32 + 3, -2 ** 40, 3], [2 ** 31 + 1, 2 ** 33, 4]], device=DEV)
    near = torch.tensor([[3], [4]], device=DEV)
    assert torch.equal(W.adjust_logits(x, far, None, None, None, 1.5, 0.5, 0.25), W.adjust_logits(x, near, None, None, None, 1.5, 0.5, 0.25))


@pytest.mark.parametrize("V", [24, 23])
@pytest.mark.parametrize("bias_kind", [0, 1, 2, 3])
def test_surplus_rows_without_any_frame(W, V, bias_kind):
    """A packed tensor of surplus rows only: zeros, and so are their gradients, whatever the memory held."""
    rows, N, U1 = 70, 2, 3
    lengths = torch.zeros((N,), dtype=torch.int32, device=DEV)
    labels = torch.ones((N, U1 - 1), dtype=torch.int32, device=DEV)
    bias = torch.ones([(), (V,), (N, V), (N, U1, V)][bias_kind], device=DEV, requires_grad=True) if bias_kind else None
    for max_frames in (0, 4):
        x = torch.randn((rows, V), device=DEV, requires_grad=True)
        y = W.adjust_joint_logits_packed(x, labels, lengths, lengths, max_frames=max_frames, bias=bias, repetition_penalty=1.5)
        assert y.shape == x.shape and not y.any()
        dy = torch.ones_like(y)
        dirty = [torch.full((rows, V), float("nan"), device=DEV) for _ in range(4)]
        del dirty
        got = torch.autograd.grad(y, [x] + [bias] * (bias_kind > 0), dy)
        assert not any(t.any() for t in got)


@pytest.mark.parametrize("rows", [0, 5])
def test_packed_without_utterances(W, rows):
    none = torch.zeros((0,), dtype=torch.int32, device=DEV)
    labels = torch.zeros((0, 2), dtype=torch.int32, device=DEV)
    for dtype in (torch.float32, torch.bfloat16):
        x = torch.randn((rows, 11), device=DEV).to(dtype).requires_grad_(True)
        b = torch.ones((11,), device=DEV, requires_grad=True)
        for max_frames in (None, 0, 6):
            y = W.adjust_joint_logits_packed(x, labels, none, none, max_frames=max_frames, bias=b, repetition_penalty=1.5)
            assert y.shape == x.shape and not y.any()
            dx, db = torch.autograd.grad(y, [x, b], torch.ones_like(y))
            assert dx.shape == x.shape and not dx.any() and not db.any()
            only_b, = torch.autograd.grad(W.adjust_joint_logits_packed(x.detach(), labels, none, none, max_frames=max_frames, bias=b),
                                          [b], torch.ones_like(y))
            assert not only_b.any()


def test_joint_without_lengths_and_per_utterance_penalties(W):
    N, T, U1, V = 3, 14, 8, 50
    x, labels, _, _, bias, allowed, dy = _joint_case(W, 11, N, T, U1, V, torch.float32, 1, 2)
    rho, pres, freq = (torch.tensor(v, device=DEV) for v in ([1.0, 1.4, 0.7], [0.0, 0.5, -0.25], [0.1, 0.0, 0.3]))
    x.requires_grad_(True)
    y = W.adjust_joint_logits(x, labels, None, None, bias, allowed, rho, pres, freq)
    dx, = torch.autograd.grad(y, [x], dy)
    for n in range(N):
        one = x.detach()[n:n + 1].clone().requires_grad_(True)
        y1 = W.adjust_joint_logits(one, labels[n:n + 1], None, None, bias, allowed[n:n + 1], rho[n].item(), pres[n].item(), freq[n].item())
        assert torch.equal(y1[0], y[n])
        d1, = torch.autograd.grad(y1, [one], dy[n:n + 1])
        assert torch.equal(d1[0], dx[n])


def test_packed_rows_that_do_not_match(W):
    N, T, U1, V = 4, 13, 6, 24
    x, labels, lx, ly, bias, allowed, dy = _joint_case(W, 12, N, T, U1, V, torch.float32, 1, 3)
    valid = valid_rows(lx, ly, N, T, U1, DEV)
    p = x[valid]
    n = p.size(0)
    full = W.adjust_joint_logits_packed(p, labels, lx, ly, bias=bias, allowed=allowed, repetition_penalty=1.3)
    for rows in (n + 29, n - 7, 1, 0):
        a = torch.ones((rows, V), device=DEV)
        k = min(n, rows)
        a[:k] = p[:k]
        a.requires_grad_(True)
        y = W.adjust_joint_logits_packed(a, labels, lx, ly, max_frames=T, bias=bias, allowed=allowed, repetition_penalty=1.3)
        assert torch.equal(y[:k], full[:k]) and not y[k:].any()
        dx, = torch.autograd.grad(y, [a], torch.ones_like(y))
        assert not dx[k:].any()


def test_gradients_against_differences(W):
    """The operator is linear in logits and bias away from zero logits: a difference has no truncation error."""
    N, T, U1, V = 2, 6, 5, 20
    x, labels, lx, ly, bias, _, dy = _joint_case(W, 13, N, T, U1, V, torch.float32, 3, 0)
    x = torch.where(x.abs() < 0.1, torch.ones_like(x), x)
    valid = valid_rows(lx, ly, N, T, U1, DEV)
    leaves = [x.requires_grad_(True), bias.requires_grad_(True)]
    grads = torch.autograd.grad(W.adjust_joint_logits(x, labels, lx, ly, bias, None, 1.25, 0.5, 0.25), leaves, dy)
    counts = torch.cat([torch.zeros((N, 1, V), device=DEV, dtype=torch.float64),
                        (labels.long().unsqueeze(-1) == torch.arange(V, device=DEV)).double().cumsum(1)], 1).unsqueeze(1)

    def value(a, b):
        y = torch.where(counts > 0, torch.where(a > 0, a / 1.25, a * 1.25), a) - 0.5 * (counts > 0) - 0.25 * counts + b[:, None]
        return (y * dy.double())[valid].sum()

    g, h = _gen(14), 1e-3
    for i in range(2):
        base = [t.detach().double() for t in leaves]
        v = _rand(g, base[i].shape).clamp(-3, 3).double()
        up, down = list(base), list(base)
        up[i], down[i] = base[i] + h * v, base[i] - h * v
        slope = (value(*up) - value(*down)) / (2 * h)
        got = (grads[i].double() * v).sum()
        assert abs(got - slope) <= 40 * U * (grads[i].double() * v).abs().sum() + 1e-8, (i, got.item(), slope.item())


def test_refusals(W):
    x = torch.randn(4, 40, device=DEV)
    tok = torch.zeros((4, 3), dtype=torch.int32, device=DEV)
    words = torch.zeros((4, 2), dtype=torch.int32, device=DEV)
    j, lab = torch.randn(2, 3, 4, 40, device=DEV), torch.ones((2, 3), dtype=torch.int32, device=DEV)
    ln = torch.ones(2, dtype=torch.int32, device=DEV)
    pen = torch.ones(4, device=DEV)
    for bad in (lambda: W.adjust_logits(x.double()), lambda: W.adjust_logits(x[0]), lambda: W.adjust_logits(x, tok[:3]),
                lambda: W.adjust_logits(x, tok.cpu()), lambda: W.adjust_logits(x, tok.float()), lambda: W.adjust_logits(x, tok, ln),
                lambda: W.adjust_logits(x, None, ln), lambda: W.adjust_logits(x, bias=x[:, :39]), lambda: W.adjust_logits(x, bias=x[:3]),
                lambda: W.adjust_logits(x, bias=x.half()), lambda: W.adjust_logits(x, allowed=words[:, :1]),
                lambda: W.adjust_logits(x, allowed=words.long()), lambda: W.adjust_logits(x, allowed=words.cpu()),
                lambda: W.adjust_logits(x, tok, repetition_penalty=0.0), lambda: W.adjust_logits(x, tok, repetition_penalty=float("nan")),
                lambda: W.adjust_logits(x, tok, presence_penalty=float("inf")), lambda: W.adjust_logits(x, tok, repetition_penalty=pen[:3]),
                lambda: W.adjust_logits(x, tok, repetition_penalty=pen.double()),
                lambda: W.adjust_logits(x, tok, frequency_penalty=pen.clone().requires_grad_(True)),
                lambda: W.adjust_joint_logits(j, lab[:, :2]), lambda: W.adjust_joint_logits(j, lab[:1]),
                lambda: W.adjust_joint_logits(j[0], lab), lambda: W.adjust_joint_logits(j, lab, ln[:1], ln),
                lambda: W.adjust_joint_logits(j, lab, ln.float(), ln), lambda: W.adjust_joint_logits(j, lab, bias=j[:, 0, :2]),
                lambda: W.adjust_joint_logits_packed(j, lab, ln, ln), lambda: W.adjust_joint_logits_packed(j[0, 0], lab, ln, ln, max_frames=-1)):
        with pytest.raises(RuntimeError):
            bad()
    y = W.adjust_logits(x.requires_grad_(True), tok, repetition_penalty=1.5)
    gx, = torch.autograd.grad(y, [x], torch.ones_like(y), create_graph=True)
    with pytest.raises(RuntimeError):
        gx.sum().backward()
    with pytest.raises(RuntimeError):   # a history that was changed between forward and backward is noticed
        y = W.adjust_logits(x, tok, repetition_penalty=1.5)
        tok += 1
        y.sum().backward()


def test_side_stream_and_captured_graph(W):
    N, T, U1, V = 3, 18, 7, 64
    x, labels, lx, ly, bias, allowed, dy = _joint_case(W, 15, N, T, U1, V, torch.float16, 1, 3)

    def step(x, labels):
        x, b = x.detach().requires_grad_(True), bias.detach().requires_grad_(True)
        y = W.adjust_joint_logits(x, labels, lx, ly, b, allowed, 1.2, 0.5, 0.1)
        return [y.detach(), *torch.autograd.grad(y, [x, b], dy)]

    want = step(x, labels)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(x, labels)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for p, q in zip(got, want):
        assert torch.equal(p, q)
    cx, cl = torch.zeros_like(x), torch.zeros_like(labels)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(cx, cl)
    for a, b in ((x, labels), (x * 0.5, labels.flip(0))):
        cx.copy_(a)
        cl.copy_(b)
        graph.replay()
        for p, q in zip(out, step(a, b)):
            assert torch.equal(p, q)


def test_joint_beyond_32_bit_offsets(W):
    """More than 2^31 elements: the last utterance is what it is by itself."""
    N, T, U1, V = 2, 1100, 1000, 1024
    g = _gen(16)
    x = torch.empty((N, T, U1, V), dtype=torch.float16, device=DEV)
    x[1] = _rand(g, (1, U1, V), torch.float16)
    labels = torch.randint(1, 30, (N, U1 - 1), generator=g, device=DEV, dtype=torch.int32)
    bias = _rand(g, (V,))
    lx, ly = torch.tensor([1, T], dtype=torch.int32, device=DEV), torch.tensor([0, U1 - 1], dtype=torch.int32, device=DEV)
    y = W.adjust_joint_logits(x, labels, lx, ly, bias, None, 1.2, 0.5, 0.01)
    one = W.adjust_joint_logits(x[1:, :1], labels[1:], None, None, bias, None, 1.2, 0.5, 0.01)
    assert torch.equal(y[1, -1], one[0, 0]) and torch.equal(y[1, 0], one[0, 0])
    assert not y[0, 1:].any()
