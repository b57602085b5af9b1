"""Timed cases of the joiner's operators: layer norm, the additive joiner's layer norm, and the adjustment of logits.

``run`` makes one pass through an operator on what ``prepare`` gives: with ``own`` the calls that a user makes of
``warp_ctct_b200``, without it the same operator as elementary torch operations in 32 bits.  ``exact`` is the
operator's definition in 64 bits, differentiated by autograd where the case is a training step.
"""
import math
import random

import torch

own = False

DEV = "cuda:0"
EPS = 1e-5
_DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2}


# ---------------------------------------------------------------------------------------------- cases

def listed():
    return [
        # one step of a streaming predictor: its output of a few sequences
        {"name": "ln_step", "op": "ln", "rows": 8, "H": 512, "dtype": "bf16", "wdtype": "bf16", "train": False},
        # encoder output of a training batch (32 utterances of 500 frames), 16-bit activations, 32-bit weights
        {"name": "ln_train_encoder", "op": "ln", "rows": 16000, "H": 1024, "dtype": "bf16", "wdtype": "f32", "train": True},
        # normalised inputs of the log-add joiner: f of 32 utterances of 500 frames over 4096 units
        {"name": "ln_train_wide", "op": "ln", "rows": 16000, "H": 4096, "dtype": "f32", "wdtype": "f32", "train": True},
        # decoding: one frame of 16 utterances against 8 hypotheses each
        {"name": "joint_ln_step", "op": "joint_ln", "N": 16, "T": 1, "U1": 8, "H": 640, "dtype": "f16", "wdtype": "f16",
         "packed": False, "train": False},
        # joiner of the first loss benchmark (32 x 256 frames x 65 contexts), padded layout
        {"name": "joint_ln_train", "op": "joint_ln", "N": 32, "T": 256, "U1": 65, "H": 512, "dtype": "bf16", "wdtype": "f32",
         "packed": False, "train": True},
        # longer utterances, valid rows only
        {"name": "joint_ln_train_packed", "op": "joint_ln", "N": 16, "T": 512, "U1": 129, "H": 512, "dtype": "f16",
         "wdtype": "f32", "packed": True, "train": True},
        # an odd small batch in 32 bits, as a debugging run or a fine-tuning step has it
        {"name": "joint_ln_train_odd", "op": "joint_ln", "N": 3, "T": 77, "U1": 19, "H": 321, "dtype": "f32", "wdtype": "f32",
         "packed": True, "train": True},
        # a decoder's step on a few streams, short histories
        {"name": "logits_step_small", "op": "logits", "R": 4, "V": 512, "L": 16, "dtype": "f32", "mask": "row", "bias": "V",
         "train": False},
        # a beam search's step over a batch, a vocabulary that is no whole number of vectors
        {"name": "logits_step_odd", "op": "logits", "R": 129, "V": 4097, "L": 100, "dtype": "f16", "mask": "row", "bias": "none",
         "train": False},
        # a large vocabulary, long histories, a grammar and a biasing list for each request
        {"name": "logits_step_large", "op": "logits", "R": 256, "V": 32000, "L": 1000, "dtype": "bf16", "mask": "row",
         "bias": "row", "train": False},
        # joint logits of the first loss benchmark: a trained bias, a grammar state for each context
        {"name": "joint_logits_train", "op": "joint_logits", "N": 32, "T": 256, "U1": 65, "V": 512, "dtype": "f32",
         "mask": "context", "bias": "V", "packed": False, "penalty": True, "train": True},
        # joint logits of the fp16 loss benchmark, valid rows only, a biasing list for each context
        {"name": "joint_logits_train_packed", "op": "joint_logits", "N": 16, "T": 512, "U1": 129, "V": 1024, "dtype": "f16",
         "mask": "shared", "bias": "context", "packed": True, "penalty": True, "train": True},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["ln", "joint_ln", "logits", "joint_logits"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    case = {"op": op, "dtype": dtype, "train": rng.random() < (0.3 if op == "logits" else 0.7)}
    if op == "ln":
        H = _log_int(rng, 8, 8192)  # a norm over one or two values has no gradient to speak of
        case.update(rows=_log_int(rng, 1, min(65536, 65_000_000 // H)), H=H, wdtype=rng.choice(["f32", dtype]))
    elif op == "logits":
        V = _log_int(rng, 2, 131072)
        case.update(R=_log_int(rng, 1, min(512, max(1, 8_000_000 // V))), V=V, L=rng.choice([0, _log_int(rng, 1, 2048)]),
                    mask=rng.choice(["none", "shared", "row"]), bias=rng.choice(["none", "V", "row"]))
    else:
        N, T, U1 = _log_int(rng, 1, 32), _log_int(rng, 1, 512), _log_int(rng, 1, 129)
        width = _log_int(rng, 8, max(8, min(2048 if op == "joint_ln" else 4096, 400_000_000 // (N * T * U1))))
        case.update(N=N, T=T, U1=U1, packed=rng.random() < 0.5)
        if op == "joint_ln":
            case.update(H=width, wdtype=rng.choice(["f32", dtype]))
        else:
            case.update(V=width, mask=rng.choice(["none", "shared", "row", "context"]), penalty=rng.random() < 0.7,
                        bias=rng.choice(["none", "V", "row", "context"]))
    return case


def _lengths(case):
    """Frame and label counts of a ragged batch: a function of the case, so that its traffic is known without a seed."""
    rng = random.Random(case["N"] * 1000003 + case["T"] * 1009 + case["U1"])
    T, U = case["T"], case["U1"] - 1
    lx = [rng.randint((T + 1) // 2, T) for _ in range(case["N"])]
    ly = [rng.randint(U // 4, U) for _ in range(case["N"])]
    lx[0], ly[0] = T, U
    return lx, ly


# --------------------------------------------------------------------------------------------- inputs

def _randn(gen, shape, dtype, scale=1.0, shift=0.0):
    return (torch.randn(shape, generator=gen, device=DEV) * scale + shift).to(dtype)


def _random_words(gen, shape, V, keep):
    """Words of a token mask, bit v % 32 of word v // 32 set where token v is allowed (with probability `keep`)."""
    W = (V + 31) // 32
    bits = (torch.rand((*shape, W * 32), generator=gen, device=DEV) < keep).view(*shape, W, 32).to(torch.int64)
    words = (bits << torch.arange(32, device=DEV)).sum(-1)
    return torch.where(words >= 2 ** 31, words - 2 ** 32, words).to(torch.int32)


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    dt = _DT[case["dtype"]]
    s = {"op": case["op"], "train": case["train"], "packed": case.get("packed", False)}
    if case["op"] in ("joint_ln", "joint_logits"):
        lx, ly = _lengths(case)
        order = torch.randperm(case["N"], generator=gen, device=DEV).tolist()
        lx, ly = [lx[i] for i in order], [ly[i] for i in order]
        s["lx"] = torch.tensor(lx, dtype=torch.int32, device=DEV)
        s["ly"] = torch.tensor(ly, dtype=torch.int32, device=DEV)
        s["rows"] = sum(a * (b + 1) for a, b in zip(lx, ly))
        s["T"], s["U1"] = case["T"], case["U1"]
        t = torch.arange(case["T"], device=DEV).view(1, -1, 1)
        u = torch.arange(case["U1"], device=DEV).view(1, 1, -1)
        s["valid"] = (t < s["lx"].view(-1, 1, 1)) & (u <= s["ly"].view(-1, 1, 1))
        lead = (s["rows"],) if s["packed"] else (case["N"], case["T"], case["U1"])
    if case["op"] in ("ln", "joint_ln"):
        H, wdt = case["H"], _DT[case["wdtype"]]
        s["w"] = _randn(gen, (H,), wdt, 0.3, 1.0)
        s["b"] = _randn(gen, (H,), wdt, 0.3)
        if case["op"] == "ln":
            lead = (case["rows"],)
            s["x"] = _randn(gen, (case["rows"], H), dt, 1.5, 0.5)
            s["leaves"] = ["x", "w", "b"]
        else:
            s["f"] = _randn(gen, (case["N"], case["T"], H), dt, 1.0, 0.3)
            s["g"] = _randn(gen, (case["N"], case["U1"], H), dt, 1.0, -0.2)
            s["leaves"] = ["f", "g", "w", "b"]
        s["dy"] = _randn(gen, (*lead, H), dt, 0.5) if case["train"] else None
    else:
        V = case["V"]
        if case["op"] == "logits":
            R, L = case["R"], case["L"]
            lead = (R,)
            pool = max(1, min(V, (L + 1) // 2))  # histories repeat tokens
            s["tokens"] = torch.randint(0, pool, (R, L), generator=gen, device=DEV, dtype=torch.int32) * (V // pool)
            s["lens"] = torch.randint(0, L + 1, (R,), generator=gen, device=DEV, dtype=torch.int32)
            # each request brings its own settings
            s["rho"] = 1.0 + 0.3 * torch.rand(R, generator=gen, device=DEV)
            s["presence"] = 0.5 * torch.rand(R, generator=gen, device=DEV)
            s["frequency"] = 0.2 * torch.rand(R, generator=gen, device=DEV)
            shapes = {"V": (), "shared": (), "row": (R,)}
        else:
            N, U1 = case["N"], case["U1"]
            pool = max(1, min(V - 1, U1))
            s["labels"] = 1 + torch.randint(0, pool, (N, U1 - 1), generator=gen, device=DEV, dtype=torch.int32)
            on = 1.0 if case["penalty"] else 0.0
            s["rho"], s["presence"], s["frequency"] = 1.0 + 0.2 * on, 0.3 * on, 0.1 * on
            shapes = {"V": (), "shared": (), "row": (N,), "context": (N, U1)}
        s["x"] = _randn(gen, (*lead, V), dt, 2.0)
        s["bias"] = None if case["bias"] == "none" else _randn(gen, (*shapes[case["bias"]], V), torch.float32, 0.5)
        s["allowed"] = None if case["mask"] == "none" else _random_words(gen, shapes[case["mask"]], V, 0.8)
        if case["mask"] in ("row", "context"):
            s["allowed"].view(-1, s["allowed"].size(-1))[-1] = 0  # a grammar's dead end: nothing is allowed
        s["leaves"] = ["x"] + (["bias"] if s["bias"] is not None else [])
        s["dy"] = _randn(gen, (*lead, V), dt, 0.5) if case["train"] else None
    if case["train"]:
        for k in s["leaves"]:
            s[k].requires_grad_(True)
    return s


# ------------------------------------------------------------------------------------ the calls of a user

def _run_own(s):
    import warp_ctct_b200 as W
    if s["op"] == "ln":
        y = W.layer_norm(s["x"], s["w"], s["b"], EPS)
    elif s["op"] == "joint_ln":
        if s["packed"]:
            y = W.joint_layer_norm_packed(s["f"], s["g"], s["lx"], s["ly"], s["w"], s["b"], EPS, rows=s["rows"])
        else:
            y = W.joint_layer_norm(s["f"], s["g"], s["lx"], s["ly"], s["w"], s["b"], EPS)
    else:
        how = dict(bias=s["bias"], allowed=s["allowed"], repetition_penalty=s["rho"], presence_penalty=s["presence"],
                   frequency_penalty=s["frequency"])
        if s["op"] == "logits":
            y = W.adjust_logits(s["x"], s["tokens"], s["lens"], **how)
        elif s["packed"]:
            y = W.adjust_joint_logits_packed(s["x"], s["labels"], s["lx"], s["ly"], max_frames=s["T"], **how)
        else:
            y = W.adjust_joint_logits(s["x"], s["labels"], s["lx"], s["ly"], **how)
    if not s["train"]:
        return [y]
    return [y.detach(), *torch.autograd.grad(y, [s[k] for k in s["leaves"]], s["dy"])]


# ------------------------------------------------------------------------------- plain forms, in 32 bits

def _spread(packed, valid):
    """(rows, C) of the valid rows -> (N, T, U1, C), zeros elsewhere."""
    out = packed.new_zeros((*valid.shape, packed.size(-1)))
    out[valid] = packed
    return out


def _norm(x):
    d = x - x.mean(-1, keepdim=True)
    r = (d.square().mean(-1, keepdim=True) + EPS).rsqrt()
    return d.mul_(r), r


def _norm_grads(dy, xh, r, w, rows):
    """Gradients of x, weight and bias; `rows`: the dimensions that the weight's gradient sums over."""
    q = dy * w
    dx = (q - q.mean(-1, keepdim=True) - xh * (q * xh).mean(-1, keepdim=True)).mul_(r)
    return dx, (dy * xh).sum(rows), dy.sum(rows)


def _plain_ln(s):
    x, w, b = s["x"].detach(), s["w"].detach(), s["b"].detach()
    xh, r = _norm(x.float())
    y = (xh * w.float() + b.float()).to(x.dtype)
    if not s["train"]:
        return [y]
    dx, dw, db = _norm_grads(s["dy"].float(), xh, r, w.float(), (0,))
    return [y, dx.to(x.dtype), dw.to(w.dtype), db.to(b.dtype)]


def _plain_joint_ln(s):
    f, g, w, b = (s[k].detach() for k in ("f", "g", "w", "b"))
    keep = s["valid"].unsqueeze(-1)
    xh, r = _norm(f.float().unsqueeze(2) + g.float().unsqueeze(1))
    y = torch.where(keep, xh * w.float() + b.float(), 0.0).to(f.dtype)
    y = y[s["valid"]] if s["packed"] else y
    if not s["train"]:
        return [y]
    dy = _spread(s["dy"], s["valid"]).float() if s["packed"] else torch.where(keep, s["dy"].float(), 0.0)
    ds, dw, db = _norm_grads(dy, xh, r, w.float(), (0, 1, 2))
    return [y, ds.sum(2).to(f.dtype), ds.sum(1).to(g.dtype), dw.to(w.dtype), db.to(b.dtype)]


def _allowed(words, V):
    v = torch.arange(V, device=words.device)
    return ((words[..., v // 32] >> (v % 32)) & 1).bool()


def _plain_adjust(s):
    x = s["x"].detach()
    V = x.size(-1)
    if s["op"] == "logits":
        tok, R = s["tokens"].long(), x.size(0)
        seen = torch.arange(tok.size(1), device=x.device) < s["lens"].view(-1, 1)
        count = torch.zeros((R, V + 1), device=x.device)
        count.scatter_add_(1, torch.where(seen, tok, V), torch.ones_like(tok, dtype=torch.float32))
        count = count[:, :V]
        rho, presence, frequency = (s[k].view(-1, 1) for k in ("rho", "presence", "frequency"))
        keep = None
        x4, wide = x.float(), lambda v: v
    else:
        one = (s["labels"].long().unsqueeze(-1) == torch.arange(V, device=x.device)).float()
        count = torch.nn.functional.pad(one.cumsum(1), (0, 0, 1, 0)).unsqueeze(1)  # (N, 1, U1, V)
        rho, presence, frequency = s["rho"], s["presence"], s["frequency"]
        keep = s["valid"].unsqueeze(-1)
        x4 = (_spread(x, s["valid"]) if s["packed"] else x).float()

        def wide(v):  # (V), (N, V) or (N, U1, V) against (N, T, U1, V)
            return v if v.dim() == 1 else v[:, None, None] if v.dim() == 2 else v[:, None]
    hit = count > 0
    y = torch.where(hit, torch.where(x4 > 0, x4 / rho, x4 * rho), x4)
    y = y - (presence * hit + frequency * count)
    if s["bias"] is not None:
        y = y + wide(s["bias"].detach())
    ok = None if s["allowed"] is None else wide(_allowed(s["allowed"], V))
    if ok is not None:
        y = torch.where(ok, y, -math.inf)
    if keep is not None:
        y = y[s["valid"]] if s["packed"] else torch.where(keep, y, 0.0)
    y = y.to(x.dtype)
    if not s["train"]:
        return [y]
    dy = (_spread(s["dy"], s["valid"]) if s["packed"] else s["dy"]).float()
    if ok is not None:
        dy = torch.where(ok, dy, 0.0)
    if keep is not None:
        dy = torch.where(keep, dy, 0.0)
    dx = torch.where(hit, torch.where(x4 > 0, dy / rho, dy * rho), dy)
    out = [y, (dx[s["valid"]] if s["packed"] else dx).to(x.dtype)]
    if s["bias"] is not None:
        if s["op"] == "logits":
            out.append(dy.sum(0, dtype=torch.float64).float() if s["bias"].dim() == 1 else dy)
        else:
            over = {1: (0, 1, 2), 2: (1, 2), 3: (1,)}[s["bias"].dim()]
            out.append(dy.sum(over, dtype=torch.float64).float())
    return out


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return {"ln": _plain_ln, "joint_ln": _plain_joint_ln}.get(state["op"], _plain_adjust)(state)


# ----------------------------------------------------------------------------- the definitions, in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    d = {k: (s[k].detach().double().requires_grad_(case["train"]) if s.get(k) is not None else None)
         for k in ("x", "f", "g", "w", "b", "bias") if k in s}
    if case["op"] in ("ln", "joint_ln"):
        z = d["x"] if case["op"] == "ln" else d["f"][:, :, None, :] + d["g"][:, None, :, :]
        if case["op"] == "joint_ln" and s["packed"]:
            z = z[s["valid"]]
        var, mean = torch.var_mean(z, -1, unbiased=False, keepdim=True)
        y = (z - mean) / torch.sqrt(var + EPS) * d["w"] + d["b"]
    else:
        V = case["V"]
        bits = torch.arange(32, device=DEV)
        if case["op"] == "logits":
            table = torch.zeros((case["R"], V), dtype=torch.float64, device=DEV)
            inside = torch.arange(case["L"], device=DEV)[None, :] < s["lens"][:, None]
            r, j = inside.nonzero(as_tuple=True)
            table.index_put_((r, s["tokens"][r, j].long()), torch.ones(r.numel(), dtype=torch.float64, device=DEV), accumulate=True)
            par = [s[k].double()[:, None] for k in ("rho", "presence", "frequency")]
        else:
            # times label position j < u holds token v
            before = torch.ones((s["U1"], s["U1"] - 1), dtype=torch.float64, device=DEV).tril(-1)
            table = before @ torch.nn.functional.one_hot(s["labels"].long(), V).double()
            par = [s[k] for k in ("rho", "presence", "frequency")]
        mask = None
        if s["allowed"] is not None:
            mask = ((s["allowed"].unsqueeze(-1) >> bits) & 1).flatten(-2)[..., :V] != 0
        bias = d["bias"]
        if case["op"] == "joint_logits":
            full = (case["N"], case["T"], case["U1"], V)

            def rows(v, dims):  # a table over (N,) or (N, U1) or nothing, seen at the rows of the joint tensor
                v = {1: lambda a: a, 2: lambda a: a[:, None, None, :], 3: lambda a: a[:, None, :, :]}[dims](v).expand(full)
                return v[s["valid"]] if s["packed"] else v

            table = rows(table, 3)
            mask = None if mask is None else rows(mask, mask.dim())
            bias = None if bias is None else rows(bias, bias.dim())
        z = d["x"]
        scale = torch.where(z.detach() > 0, 1.0 / par[0], torch.ones_like(z) * par[0])
        z = torch.where(table > 0, z * scale, z)
        z = z - par[1] * (table > 0) - par[2] * table
        if bias is not None:
            z = z + bias
        y = z if mask is None else z.masked_fill(~mask, -math.inf)
    if "valid" in s and not s["packed"]:
        y = y.masked_fill(~s["valid"].unsqueeze(-1), 0.0)
    if not case["train"]:
        return [y.detach()]
    return [y.detach(), *torch.autograd.grad(y, [d[k] for k in s["leaves"]], s["dy"].double())]


# ------------------------------------------------------------------------------------------------- work

def work(case):
    e = _BYTES[case["dtype"]]
    if case["op"] == "ln":
        n = case["rows"] * case["H"]
        par = 2 * case["H"] * _BYTES[case["wdtype"]]
        if case["train"]:  # x, dy in; y, dx out; the weights and their gradients
            return {"bytes": 4 * n * e + 2 * par, "flops": 20 * n}
        return {"bytes": 2 * n * e + par, "flops": 8 * n}
    if case["op"] == "logits":
        n, V = case["R"] * case["V"], case["V"]
        side = {"none": 0, "shared": V / 8, "row": n / 8}[case["mask"]] + {"none": 0, "V": 4 * V, "row": 4 * n}[case["bias"]]
        side += case["R"] * case["L"] * 2  # half of the histories' places are taken, 4 bytes each
        if case["train"]:
            return {"bytes": 4 * n * e + side + {"none": 0, "V": 4 * V, "row": 4 * n}[case["bias"]], "flops": 6 * n}
        return {"bytes": 2 * n * e + side, "flops": 4 * n}
    lx, ly = _lengths(case)
    valid = sum(a * (b + 1) for a, b in zip(lx, ly))
    rows = valid if case["packed"] else case["N"] * case["T"] * case["U1"]  # the padded layout's padding is written too
    if case["op"] == "joint_ln":
        H = case["H"]
        small = (sum(lx) + sum(b + 1 for b in ly)) * H * e + 2 * H * _BYTES[case["wdtype"]]
        if not case["train"]:
            return {"bytes": rows * H * e + small, "flops": 8 * valid * H}
        grads = case["N"] * (case["T"] + case["U1"]) * H * e + 2 * H * _BYTES[case["wdtype"]]
        return {"bytes": (rows + valid) * H * e + small + grads, "flops": 20 * valid * H}
    N, U1, V = case["N"], case["U1"], case["V"]
    mask = {"none": 0, "shared": V, "row": N * V, "context": N * U1 * V}[case["mask"]] / 8
    bias = {"none": 0, "V": V, "row": N * V, "context": N * U1 * V}[case["bias"]] * 4
    step = {"bytes": (valid + rows) * V * e + mask + bias, "flops": 4 * valid * V}
    if case["train"]:
        step = {"bytes": 2 * step["bytes"], "flops": 6 * valid * V}
    return step
