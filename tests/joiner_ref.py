"""Plain 64-bit forms of the joiner's operators and bounds for the kernels' float32 arithmetic, for the tests.

Bounds.  u = 2^-24 is half a step of float32.  A float32 sum of n terms whose longest chain of additions has k
additions is off by at most k u sum|terms| (first order).  With A the largest |x| of a row, r = 1/sqrt(var + eps) and
xh = (x - mean) r the mean is off by at most k u A, hence x - mean by k u A + u |x - mean|; the variance by
2 k u A / (r) relative to 1 / r^2 plus (k + 2) u, the reciprocal root by half of that and its own two steps (4 u):

    E(xh) = k u A r (1 + |xh|) + (k / 2 + 6) u |xh|

Every further product or sum adds u of its value.  An output of type t is rounded once: half a step of t,
finfo(t).eps / 2 of the value, or half of the smallest subnormal."""
import torch

U = 2.0 ** -24


def half_step(v, dtype):
    tiny = {torch.float32: 2.0 ** -150, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}[dtype]
    return v.abs() * (torch.finfo(dtype).eps / 2) + tiny


def norm_reference(s, w, b, eps, dy, amax, k, rows_k, dtype, pdtype, parts=None):
    """Layer norm of the rows `s` (R, H) float64 with gradients for `dy` (or None), and bounds of everything.

    amax: (R, 1) largest magnitude that entered a row's float32 sums; k: longest chain of additions along a row,
    rows_k: over rows.  Returns ({name: value}, {name: bound}); the bound of ds is the one before its rounding."""
    H = s.size(-1)
    w = torch.ones(H, dtype=torch.float64, device=s.device) if w is None else w.double()
    b = torch.zeros(H, dtype=torch.float64, device=s.device) if b is None else b.double()
    d = s - s.mean(-1, keepdim=True)
    r = (d.square().mean(-1, keepdim=True) + eps).rsqrt()
    xh = d * r
    y = xh * w + b
    E = k * U * amax * r * (1 + xh.abs()) + (k / 2 + 6) * U * xh.abs()
    val = {"y": y}
    tol = {"y": E * w.abs() + 3 * U * ((xh * w).abs() + b.abs()) + half_step(y, dtype)}
    if dy is None:
        return val, tol
    dy = dy.double()
    q = dy * w
    c1, c2 = q.mean(-1, keepdim=True), (q * xh).mean(-1, keepdim=True)
    ds = r * (q - c1 - xh * c2)
    mq, mqx = q.abs().mean(-1, keepdim=True), (q * xh).abs().mean(-1, keepdim=True)
    Er = k * U * amax * r + (k / 2 + 6) * U   # relative error of r
    e_c2 = (k + 4) * U * mqx + (q.abs() * E).mean(-1, keepdim=True)
    e_ds = r * (4 * U * q.abs() + (k + 4) * U * mq + xh.abs() * e_c2 + E * c2.abs() + 4 * U * (xh * c2).abs())
    # r enters up to its third power in some kernels
    e_ds = e_ds + 3 * Er * r * (q.abs() + c1.abs() + (xh * c2).abs())
    dw, db = (dy * xh).sum(0), dy.sum(0)
    val.update(ds=ds, dw=dw, db=db)
    # a sum of ds over rows may be taken as three sums, of r q, r c1 and r xh c2: its rounding goes by their magnitudes
    val["terms"] = r * (q.abs() + c1.abs() + (xh * c2).abs())
    tol["ds"] = e_ds
    # dy xh may be summed as dy f r and dy g r apart (f, g centred, at most amax): "parts" is the bound of |f| + |g|
    tol["dw"] = (dy.abs() * E).sum(0) + (rows_k + 4) * U * (dy.abs() * (xh.abs() if parts is None else parts * r)).sum(0) + half_step(dw, pdtype)
    tol["db"] = (rows_k + 4) * U * dy.abs().sum(0) + half_step(db, pdtype)
    return val, tol


def check(name, got, want, bound):
    assert got.shape == want.shape, (name, got.shape, want.shape)
    got, want = got.detach().double(), want.double()
    same = (got == want) | (got.isnan() & want.isnan())
    bad = ~(same | ((got - want).abs() <= bound))
    if bool(bad.any()):
        at = bad.nonzero()[0].tolist()
        i = tuple(at)
        raise AssertionError(f"{name}{at}: {got[i].item()!r} instead of {want[i].item()!r}, bound "
                             f"{bound.expand_as(want)[i].item():.3g}; {int(bad.sum())} of {bad.numel()} off")


def valid_rows(lx, ly, N, T, U1, device):
    t = torch.arange(T, device=device).view(1, -1, 1)
    u = torch.arange(U1, device=device).view(1, 1, -1)
    lx = torch.full((N,), T, device=device) if lx is None else lx.to(device).long().clamp(0, T)
    ly = torch.full((N,), U1 - 1, device=device) if ly is None else ly.to(device).long().clamp(0, U1 - 1)
    return (t < lx.view(-1, 1, 1)) & (u <= ly.view(-1, 1, 1))


def adjust_reference(x, counts, bias, ok, rho, presence, frequency, dy, dtype):
    """All arguments broadcast against x; returns ({y, dx}, bounds, the masked dy).  counts float64; ok bool or None."""
    x = x.double()
    hit = counts > 0
    scale = torch.where(hit, torch.where(x > 0, 1 / rho, rho), torch.ones_like(x))
    pen = presence * hit + frequency * counts
    z = x * scale - pen + (0.0 if bias is None else bias.double())
    size = (x * scale).abs() + presence * hit + (frequency * counts).abs() + (0.0 if bias is None else bias.double().abs())
    y = z if ok is None else torch.where(ok, z, float("-inf"))
    val, tol = {"y": y}, {"y": 5 * U * size + half_step(torch.where(y.isfinite(), y, 0.0), dtype)}
    if dy is None:
        return val, tol, None
    dy = dy.double()
    if ok is not None:
        dy = torch.where(ok, dy, 0.0)
    dx = dy * scale
    val["dx"], tol["dx"] = dx, 3 * U * dx.abs() + half_step(dx, dtype)
    return val, tol, dy


def unpack_words(words, V):
    v = torch.arange(V, device=words.device)
    return ((words[..., v // 32].long() >> (v % 32)) & 1).bool()
