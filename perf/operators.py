"""Cases of the recurrent decoder block's operators, in plain torch and as the
framework computes them.

Three operators of `marian_amd.ops` are covered:

- ``gated_scan`` (and ``gated_scan_xg`` on a fused projection): the gated linear
  recurrence  c_t = f_t c_{t-1} + (1 - f_t) x_t,  f_t = sigmoid(gate_t),  over whole
  sequences, with its gradients in a training pass;
- ``gated_step``: the same recurrence for one new token of each running request;
- ``block_norm``: a block's output norm, its gate, the scaled residual sum and the
  norm before the next block, with their gradients in a training pass.

``own`` selects which side ``run`` computes.
"""
import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------

def _scan(name, B, T, D, dtype, train, lens=False, reverse=False, act="none",
          fused=False, state=False):
    return {"op": "scan", "name": name, "B": B, "T": T, "D": D, "dtype": dtype,
            "train": train, "lens": lens, "reverse": reverse, "act": act,
            "fused": fused, "state": state}


def _step(name, N, D, dtype, act="relu"):
    return {"op": "step", "name": name, "N": N, "D": D, "dtype": dtype,
            "act": act}


def _norm(name, rows, D, dtype, train, norm="layer", post=True, pre=True,
          gate="none", per_token=False, res_scale=1.0):
    return {"op": "norm", "name": name, "rows": rows, "D": D, "dtype": dtype,
            "train": train, "norm": norm, "post": post, "pre": pre,
            "gate": gate, "per_token": per_token, "res_scale": res_scale}


def listed():
    return [
        # the training benchmark's batch (1024 sentences of 64 words, width
        # 1024) through a recurrent decoder layer, on the fused projection
        _scan("scan_train_big", 1024, 64, 1024, "bf16", True, fused=True),
        # one long document: little batch, so the time axis has to be split
        _scan("scan_train_long", 1, 16384, 1024, "bf16", True, state=True),
        # a ragged mini-batch read right to left (bidirectional encoder) at an
        # odd width, in full precision
        _scan("scan_train_ragged", 37, 331, 509, "fp32", True, lens=True,
              reverse=True),
        # scoring: forward only, a few sequences of middle length
        _scan("scan_score", 4, 2048, 512, "fp16", False, lens=True,
              act="relu"),
        # the start of one request: a short prefix at the tiny model's width,
        # where the launch is all the time there is
        _scan("scan_prefix", 1, 17, 128, "bf16", False, act="relu",
              state=True),
        # interactive decoding: one sentence, beam 4
        _step("step_beam4", 4, 1024, "bf16"),
        # the decoding benchmark's batch with a larger beam
        _step("step_batch", 4096, 1024, "bf16"),
        # a pre-norm layer of the training benchmark's batch: norm on the
        # block's output, a learned gate per channel, residual, next norm
        _norm("norm_train_big", 65536, 1024, "bf16", True, gate="scale"),
        # highway gate computed for every token, RMS norms
        _norm("norm_train_highway", 4096, 512, "fp16", True, norm="rms",
              gate="highway", per_token=True, post=False),
        # wide rows: a block of threads works on each
        _norm("norm_train_wide", 2048, 8192, "bf16", True, norm="rms",
              res_scale=0.5),
        # an odd width in full precision
        _norm("norm_train_odd", 999, 1021, "fp32", True, gate="highway",
              res_scale=0.7071),
        # interactive decoding: one row per beam
        _norm("norm_beam4", 4, 1024, "bf16", False, gate="scale"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    limit = max(work(c)["bytes"] for c in listed())
    op = rng.choice(["scan", "scan", "scan", "step", "norm", "norm", "norm"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op == "scan":
        c = _scan("", _log_int(rng, 1, 1024), _log_int(rng, 1, 16384),
                  _log_int(rng, 16, 4096), dtype, rng.random() < 0.7,
                  lens=rng.random() < 0.4, reverse=rng.random() < 0.4,
                  fused=rng.random() < 0.4, state=rng.random() < 0.5)
        if not c["train"]:
            # forward only: relu's derivative jumps at a state of 0, on whose
            # side 32 and 64 bits need not agree
            c["act"] = rng.choice(["none", "relu"])
        if rng.random() < 0.5:          # model widths are mostly multiples
            c["D"] = -(-c["D"] // 32) * 32
        while work(c)["bytes"] > limit // 2:
            big = max(("B", "T"), key=lambda k: c[k])
            c[big] = max(1, c[big] * 2 // 3)
    elif op == "step":
        c = _step("", _log_int(rng, 1, 4096), _log_int(rng, 16, 4096), dtype,
                  act=rng.choice(["none", "relu"]))
    else:
        gate = rng.choice(["none", "scale", "highway"])
        c = _norm("", _log_int(rng, 1, 65536), _log_int(rng, 32, 16384), dtype,
                  rng.random() < 0.7, norm=rng.choice(["layer", "rms"]),
                  post=rng.random() < 0.6, pre=rng.random() < 0.8,
                  gate=gate, per_token=gate != "none" and rng.random() < 0.5,
                  res_scale=rng.choice([1.0, 1.0, 0.5, 0.7071]))
        if rng.random() < 0.5:
            c["D"] = -(-c["D"] // 32) * 32
        while work(c)["bytes"] > limit // 2:
            c["rows"] = max(1, c["rows"] * 2 // 3)
    del c["name"]
    return c


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 7919 + 17)
    return g


def _randn(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


def prepare(case, seed):
    g = _gen(seed)
    dt = _DT[case["dtype"]]
    st = {"case": case}
    if case["op"] == "scan":
        B, T, D = case["B"], case["T"], case["D"]
        # gate logits lean to "keep" as a trained forget gate's do
        xg = torch.cat([_randn(g, B, T, D), _randn(g, B, T, D) * 1.5 + 1.0],
                       dim=-1).to(dt)
        if case["fused"]:
            st["xg"] = xg
        else:
            st["x"] = xg[..., :D].contiguous()
            st["gate"] = xg[..., D:].contiguous()
        del xg
        st["state"] = _randn(g, B, D) if case["state"] else None
        st["lens"] = None
        if case["lens"]:
            st["lens"] = torch.randint(0, T + 1, (B,), device="cuda",
                                       generator=g).to(torch.int32)
        if case["train"]:
            st["dy"] = _randn(g, B, T, D).to(dt)
            st["dlast"] = _randn(g, B, D)
            for k in ("xg", "x", "gate", "state"):
                if st.get(k) is not None:
                    st[k].requires_grad_()
    elif case["op"] == "step":
        N, D = case["N"], case["D"]
        # the projection of the new tokens: values and gates side by side
        st["xg"] = torch.cat([_randn(g, N, D), _randn(g, N, D) * 1.5 + 1.0],
                             dim=-1).to(dt)
        st["state"] = _randn(g, N, D)
    else:
        R, D = case["rows"], case["D"]
        st["x"] = (_randn(g, R, D) * 2.0 + 0.3).to(dt)
        st["res"] = (_randn(g, R, D) * 3.0 - 0.5).to(dt)
        st["gate"] = None
        if case["gate"] != "none":
            shape = (R, D) if case["per_token"] else (D,)
            st["gate"] = (_randn(g, *shape) * 0.5 + 0.5).to(dt)
        for side in ("post", "pre"):
            on = case[side]
            st[side + "_scale"] = (1.0 + 0.2 * _randn(g, D)).to(dt) if on \
                else None
            st[side + "_bias"] = (0.2 * _randn(g, D)).to(dt) \
                if on and case["norm"] == "layer" else None
        if case["train"]:
            st["dsum"] = _randn(g, R, D).to(dt)
            st["dh"] = _randn(g, R, D).to(dt) if case["pre"] else None
            for k in _NORM_LEAVES:
                if st[k] is not None:
                    st[k].requires_grad_()
    return st


_NORM_LEAVES = ("x", "res", "gate", "post_scale", "post_bias", "pre_scale",
                "pre_bias")


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(st):
    case = st["case"]
    if case["op"] == "scan":
        return _own_scan(st) if own else _plain_scan(st)
    if case["op"] == "step":
        return _own_step(st) if own else _plain_step(st)
    return _own_norm(st) if own else _plain_norm(st)


def _scan_leaves(st):
    keys = ("xg",) if st["case"]["fused"] else ("x", "gate")
    return keys + (("state",) if st["state"] is not None else ())


def _own_scan(st):
    from marian_amd import ops
    c = st["case"]
    kw = {"state": st["state"], "lens": st["lens"], "reverse": c["reverse"],
          "act": c["act"]}
    if c["fused"]:
        y, last = ops.gated_scan_xg(st["xg"], **kw)
    else:
        y, last = ops.gated_scan(st["x"], st["gate"], **kw)
    if not c["train"]:
        return y, last
    keys = _scan_leaves(st)
    grads = torch.autograd.grad((y, last), [st[k] for k in keys],
                                (st["dy"], st["dlast"]))
    return (y.detach(), last.detach()) + tuple(grads)


def _own_step(st):
    from marian_amd import ops
    D = st["case"]["D"]
    return ops.gated_step(st["xg"][:, :D], st["xg"][:, D:], st["state"],
                          act=st["case"]["act"])


def _own_norm(st):
    from marian_amd import ops
    c = st["case"]
    s, h = ops.block_norm(
        st["x"], st["res"], gate=st["gate"],
        gate_kind=c["gate"] if c["gate"] != "none" else "scale",
        res_scale=c["res_scale"], post_scale=st["post_scale"],
        post_bias=st["post_bias"], pre_scale=st["pre_scale"],
        pre_bias=st["pre_bias"], norm=c["norm"])
    outs, douts = [s], [st.get("dsum")]
    if h is not None:
        outs.append(h)
        douts.append(st.get("dh"))
    if not c["train"]:
        return tuple(outs)
    leaves = [st[k] for k in _NORM_LEAVES if st[k] is not None]
    grads = torch.autograd.grad(outs, leaves, douts)
    return tuple(o.detach() for o in outs) + tuple(grads)


# ---------------------------------------------------------------------------
# plain forms: elementary torch operations in 32 bits
# ---------------------------------------------------------------------------

def _prefix(a, h):
    """All states of  c_t = a_t c_{t-1} + h_t  (c_{-1} = 0) over dim 1, by
    combining neighbours at doubling distances."""
    a, h = a.clone(), h.clone()
    k, T = 1, a.shape[1]
    while k < T:
        h[:, k:] = h[:, k:] + a[:, k:] * h[:, :-k]
        a[:, k:] = a[:, k:] * a[:, :-k]
        k *= 2
    return h


@torch.no_grad()
def _plain_scan(st):
    c = st["case"]
    B, T, D = c["B"], c["T"], c["D"]
    dt = _DT[c["dtype"]]
    if c["fused"]:
        x, g = st["xg"][..., :D].float(), st["xg"][..., D:].float()
    else:
        x, g = st["x"].float(), st["gate"].float()
    f = 1.0 / (1.0 + torch.exp(-g))
    b = (1.0 - f) * x
    valid = None
    if st["lens"] is not None:
        valid = (torch.arange(T, device=x.device)[None, :]
                 < st["lens"][:, None])[..., None]
        # a padded step holds the state
        f = torch.where(valid, f, torch.ones_like(f))
        b = torch.where(valid, b, torch.zeros_like(b))
    flip = (lambda t: t.flip(1)) if c["reverse"] else (lambda t: t)
    f, b = flip(f), flip(b)
    c0 = st["state"] if st["state"] is not None \
        else torch.zeros(B, D, device=x.device)
    b0 = b.clone()
    b0[:, 0] += f[:, 0] * c0
    cs = _prefix(f, b0)
    last = cs[:, -1].clone()
    y = torch.where(cs > 0, cs, torch.zeros_like(cs)) \
        if c["act"] == "relu" else cs
    if valid is not None:
        y = flip(y) * valid
        y = flip(y)
    y = flip(y).to(dt).contiguous()
    if not c["train"]:
        return y, last
    dy = st["dy"].float()
    if valid is not None:
        dy = torch.where(valid, dy, torch.zeros_like(dy))
    dy = flip(dy)
    if c["act"] == "relu":
        dy = dy * (cs > 0)
    dy = dy.clone()
    dy[:, -1] += st["dlast"]
    # lam_t = dy_t + f_{t+1} lam_{t+1}: the same recurrence, backwards
    fn = torch.cat([f[:, 1:], torch.zeros_like(f[:, :1])], dim=1)
    lam = _prefix(fn.flip(1), dy.flip(1)).flip(1)
    dstate = f[:, 0] * lam[:, 0]
    prev = torch.cat([c0[:, None], cs[:, :-1]], dim=1)
    dx = flip((1.0 - f) * lam)
    dg = flip(f * (1.0 - f) * lam * (prev - flip(x)))
    if valid is not None:
        dx, dg = dx * valid, dg * valid
    if c["fused"]:
        grads = (torch.cat([dx, dg], dim=-1).to(dt),)
    else:
        grads = (dx.to(dt).contiguous(), dg.to(dt).contiguous())
    if st["state"] is not None:
        grads += (dstate,)
    return (y, last) + grads


@torch.no_grad()
def _plain_step(st):
    c = st["case"]
    D = c["D"]
    x, g = st["xg"][:, :D].float(), st["xg"][:, D:].float()
    f = 1.0 / (1.0 + torch.exp(-g))
    new = f * st["state"] + (1.0 - f) * x
    y = torch.where(new > 0, new, torch.zeros_like(new)) \
        if c["act"] == "relu" else new
    return y.to(_DT[c["dtype"]]), new


_EPS = 1e-9


def _plain_stats(v, norm):
    """(v - mean) / deviation, and 1 / deviation."""
    if norm == "layer":
        v = v - v.mean(dim=-1, keepdim=True)
    r = 1.0 / torch.sqrt((v * v).mean(dim=-1, keepdim=True) + _EPS)
    return v * r, r


def _plain_norm_grad(d, xhat, r, norm):
    d2 = d - xhat * (d * xhat).mean(dim=-1, keepdim=True)
    if norm == "layer":
        d2 = d2 - d.mean(dim=-1, keepdim=True)
    return d2 * r


@torch.no_grad()
def _plain_norm(st):
    c = st["case"]
    dt = _DT[c["dtype"]]
    norm, alpha = c["norm"], c["res_scale"]
    x, res = st["x"].float(), st["res"].float()
    w = {k: st[k].float() if st[k] is not None else None
         for k in ("gate", "post_scale", "post_bias", "pre_scale", "pre_bias")}
    u = x
    if c["post"]:
        xh, xr = _plain_stats(x, norm)
        u = xh * w["post_scale"]
        if w["post_bias"] is not None:
            u = u + w["post_bias"]
    a, b, sg = alpha, 1.0, None
    if c["gate"] == "scale":
        b = w["gate"]
    elif c["gate"] == "highway":
        sg = 1.0 / (1.0 + torch.exp(-w["gate"]))
        a, b = alpha * (1.0 - sg), sg
    s = a * res + b * u
    outs = (s.to(dt),)
    if c["pre"]:
        sh, sr = _plain_stats(s, norm)
        h = sh * w["pre_scale"]
        if w["pre_bias"] is not None:
            h = h + w["pre_bias"]
        outs += (h.to(dt),)
    if not c["train"]:
        return outs
    ds = st["dsum"].float()
    gr = dict.fromkeys(_NORM_LEAVES)
    if c["pre"]:
        dh = st["dh"].float()
        gr["pre_scale"] = (dh * sh).sum(0)
        gr["pre_bias"] = dh.sum(0)
        ds = ds + _plain_norm_grad(dh * w["pre_scale"], sh, sr, norm)
    gr["res"] = a * ds
    du = b * ds
    if c["gate"] == "scale":
        gr["gate"] = u * ds
    elif c["gate"] == "highway":
        gr["gate"] = sg * (1.0 - sg) * (u - alpha * res) * ds
    if gr["gate"] is not None and not c["per_token"]:
        gr["gate"] = gr["gate"].sum(0)
    gr["x"] = du
    if c["post"]:
        gr["post_scale"] = (du * xh).sum(0)
        gr["post_bias"] = du.sum(0)
        gr["x"] = _plain_norm_grad(du * w["post_scale"], xh, xr, norm)
    return outs + tuple(gr[k].to(dt) for k in _NORM_LEAVES
                        if st[k] is not None)


# ---------------------------------------------------------------------------
# what one pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    e = _SIZE[case["dtype"]]
    D = case["D"]
    if case["op"] == "scan":
        n = case["B"] * case["T"] * D
        # lengths are uniform over 0..T: half of the inputs are read, all of
        # the outputs are written
        rd = 0.5 if case["lens"] else 1.0
        vec = case["B"] * D * 4
        nbytes = n * e * (2 * rd + 1) + vec * (1 + int(case["state"]))
        flops = 10 * n * rd
        if case["train"]:
            nbytes += n * e * (rd + 2) + vec * (1 + int(case["state"]))
            flops += 14 * n * rd
    elif case["op"] == "step":
        n = case["N"] * D
        nbytes, flops = n * (3 * e + 8), 10 * n
    else:
        n = case["rows"] * D
        gate_t = int(case["per_token"])
        gate_c = int(case["gate"] != "none" and not case["per_token"])
        vecs = gate_c + (int(case["post"]) + int(case["pre"])) \
            * (2 if case["norm"] == "layer" else 1)
        pre = int(case["pre"])
        nbytes = e * (n * (3 + gate_t + pre) + vecs * D)
        flops = n * (4 + 8 * (int(case["post"]) + pre))
        if case["train"]:
            nbytes += e * (n * (3 + gate_t + pre) + vecs * D)
            flops += n * (6 + 14 * (int(case["post"]) + pre))
    return {"bytes": int(nbytes), "flops": int(flops)}


# ---------------------------------------------------------------------------
# the definitions in 64 bits, step by step; gradients by differentiating them
# ---------------------------------------------------------------------------

def _leaf(t):
    return None if t is None else t.detach().double().requires_grad_()


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "scan":
        return _exact_scan(st)
    if case["op"] == "step":
        D = case["D"]
        xg = st["xg"].double()
        f = torch.sigmoid(xg[:, D:])
        new = f * st["state"].double() + torch.sigmoid(-xg[:, D:]) * xg[:, :D]
        return (new.clamp_min(0) if case["act"] == "relu" else new), new
    return _exact_norm(st)


def _exact_scan(st):
    c = st["case"]
    T, D = c["T"], c["D"]
    keys = _scan_leaves(st)
    lv = {k: _leaf(st[k]) for k in keys}
    if c["fused"]:
        parts = lv["xg"].unbind(1)
        xs = [p[:, :D] for p in parts]
        gs = [p[:, D:] for p in parts]
    else:
        xs, gs = lv["x"].unbind(1), lv["gate"].unbind(1)
    cur = lv.get("state")
    if cur is None:
        cur = torch.zeros(c["B"], D, dtype=torch.float64, device="cuda")
    ys = [None] * T
    with torch.set_grad_enabled(c["train"]):
        for t in range(T - 1, -1, -1) if c["reverse"] else range(T):
            f = torch.sigmoid(gs[t])
            new = f * cur + (1 - f) * xs[t]
            out = torch.relu(new) if c["act"] == "relu" else new
            if st["lens"] is not None:
                on = (st["lens"] > t)[:, None]
                new = torch.where(on, new, cur)
                out = torch.where(on, out, torch.zeros_like(out))
            cur, ys[t] = new, out
        y = torch.stack(ys, dim=1)
    if not c["train"]:
        return y.detach(), cur.detach()
    grads = torch.autograd.grad((y, cur), [lv[k] for k in keys],
                                (st["dy"].double(), st["dlast"].double()))
    return (y.detach(), cur.detach()) + tuple(grads)


def _exact_norm(st):
    c = st["case"]
    lv = {k: _leaf(st[k]) for k in _NORM_LEAVES}

    def normed(v, side):
        if c["norm"] == "layer":
            z = (v - v.mean(-1, keepdim=True)) \
                * (v.var(-1, unbiased=False, keepdim=True) + _EPS).rsqrt()
            return z * lv[side + "_scale"] + lv[side + "_bias"]
        return v * (v.square().mean(-1, keepdim=True) + _EPS).rsqrt() \
            * lv[side + "_scale"]

    u = normed(lv["x"], "post") if c["post"] else lv["x"]
    r = c["res_scale"] * lv["res"]
    if c["gate"] == "highway":
        k = torch.sigmoid(lv["gate"])
        s = (1 - k) * r + k * u
    elif c["gate"] == "scale":
        s = r + lv["gate"] * u
    else:
        s = r + u
    outs = [s] + ([normed(s, "pre")] if c["pre"] else [])
    if not c["train"]:
        return tuple(o.detach() for o in outs)
    douts = [st["dsum"].double()] + ([st["dh"].double()] if c["pre"] else [])
    grads = torch.autograd.grad(outs, [v for v in lv.values()
                                       if v is not None], douts)
    return tuple(o.detach() for o in outs) + tuple(grads)
