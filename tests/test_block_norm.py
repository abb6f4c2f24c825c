"""The fused block join (ops.block_norm) against its formulas and gradients in
64 bits.

Tolerances come from a running error bound: the oracle carries, beside every
64-bit value, how far 32-bit arithmetic with unit u = 2^-24 may be from it
(sums and products add u of their result to what their operands bring, a mean
over a row 32 u of the mean of absolute values - a lane adds at most 16
elements, a wave joins in 6 steps and a row's waves in at most 16 - and a sum
over rows 128 u of the sum of absolute values). Twice that bound covers the
order of the operations, and the last rounding adds eps / 2 of the value.
"""
import pytest
import torch

from marian_amd import ops

U = 2.0 ** -24


class Num:
    """A 64-bit value and the bound on a 32-bit computation's error."""

    def __init__(self, v, e=None):
        self.v, self.e = v, torch.zeros_like(v) if e is None else e

    def _out(self, v, e):
        return Num(v, e + U * (v.abs() + e))

    def __add__(self, o):
        return self._out(self.v + o.v, self.e + o.e)

    def __sub__(self, o):
        return self._out(self.v - o.v, self.e + o.e)

    def __mul__(self, o):
        return self._out(self.v * o.v, self.v.abs() * o.e
                         + o.v.abs() * self.e + self.e * o.e)

    def times(self, c):
        return self._out(self.v * c, self.e * abs(c))

    def mean(self):
        return Num(self.v.mean(-1, keepdim=True),
                   self.e.mean(-1, keepdim=True)
                   + 32 * U * self.v.abs().mean(-1, keepdim=True))

    def rows(self):
        return Num(self.v.sum(0),
                   self.e.sum(0) + 128 * U * self.v.abs().sum(0))

    def rsqrt(self, eps):
        x = self.v + eps
        r = x.rsqrt()
        # the error of x, when it is small beside x, halves; floor at 0
        lo = (x - self.e - U * x).clamp_min(eps / 2)
        return Num(r, (lo.rsqrt() - r) + 3 * U * r)

    def sigmoid(self):
        v = torch.sigmoid(self.v)
        return Num(v, v * (2 * self.v.abs() + 6) * U)


def oracle(t, norm, gate_kind, alpha, eps=1e-9):
    d = {k: None if v is None else Num(v.detach().double().cpu())
         for k, v in t.items()}

    def normed(v, side):
        if norm == "layer":
            v = v - v.mean()
        r = (v * v).mean().rsqrt(eps)
        xh = v * r
        y = xh * d[side + "_scale"]
        return (y if d[side + "_bias"] is None else y + d[side + "_bias"]), \
            xh, r

    def norm_grad(g, xh, r):
        o = g - xh * (g * xh).mean()
        return (o - g.mean() if norm == "layer" else o) * r

    x = d["x"]
    res = d["res"] or Num(torch.zeros_like(x.v))
    u, xh, xr = normed(x, "post") if d["post_scale"] is not None \
        else (x, None, None)
    one = Num(torch.ones(1, dtype=torch.float64))
    ca, cb, k, k1 = one.times(alpha), one, None, None
    if d["gate"] is not None:
        if gate_kind == "highway":
            k, k1 = d["gate"].sigmoid(), Num(-d["gate"].v).sigmoid()
            ca, cb = k1.times(alpha), k
        else:
            cb = d["gate"]
    s = ca * res + cb * u
    out = {"s": s}
    ds = d["dsum"]
    if d["pre_scale"] is not None:
        out["h"], sh, sr = normed(s, "pre")
        dh = d["dh"]
        out["pre_scale"], out["pre_bias"] = (dh * sh).rows(), dh.rows()
        ds = ds + norm_grad(dh * d["pre_scale"], sh, sr)
    out["res"] = ca * ds
    du = cb * ds
    if d["gate"] is not None:
        g = u * ds if gate_kind == "scale" else \
            k * k1 * (u - res.times(alpha)) * ds
        out["gate"] = g.rows() if d["gate"].v.dim() == 1 else g
    out["x"] = du
    if d["post_scale"] is not None:
        out["post_scale"], out["post_bias"] = (du * xh).rows(), du.rows()
        out["x"] = norm_grad(du * d["post_scale"], xh, xr)
    return out


# make(no_res=True): the residual's term is left out
LEAVES = ("x", "res", "gate", "post_scale", "post_bias", "pre_scale",
          "pre_bias")


def make(R, D, dtype, dev, norm="layer", gate=None, per_token=False, post=True,
         pre=True, bias=True, pdt=None, seed=0, shift=0.5, no_res=False):
    gen = torch.Generator().manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=gen)
    pdt = pdt or dtype
    t = {"x": (rnd(R, D) * 2 + shift).to(dtype),
         "res": (rnd(R, D) * 3 - 0.5).to(dtype), "gate": None,
         "dsum": rnd(R, D).to(dtype),
         "dh": rnd(R, D).to(dtype) if pre else None}
    if no_res:
        t["res"] = None
    if gate:
        t["gate"] = (rnd(R, D) if per_token else rnd(D)).add(0.3).to(
            dtype if per_token else pdt)
    for side, on in (("post", post), ("pre", pre)):
        t[side + "_scale"] = (1 + 0.2 * rnd(D)).to(pdt) if on else None
        t[side + "_bias"] = (0.3 * rnd(D)).to(pdt) \
            if on and bias and norm == "layer" else None
    return {k: None if v is None else v.to(dev) for k, v in t.items()}


def close(name, got, want, dtype):
    assert got.dtype == dtype and got.shape == want.v.shape, name
    half = torch.finfo(dtype).eps / 2 * (1 + 2.0 ** -7)
    err = (got.detach().double().cpu() - want.v).abs()
    # below the normal range a half step is absolute
    lim = 2 * want.e + half * (want.v.abs() + 2 * want.e) \
        + torch.finfo(dtype).smallest_normal * half
    assert bool((err <= lim).all()), \
        f"{name}: off by {float((err - lim).max())} over the limit"


def call(t, norm, gate_kind, alpha):
    return ops.block_norm(t["x"], t["res"], t["gate"], gate_kind, alpha,
                          t["post_scale"], t["post_bias"], t["pre_scale"],
                          t["pre_bias"], norm)


def run(t, norm, gate_kind, alpha):
    leaves = [k for k in LEAVES if t[k] is not None]
    for k in leaves:
        t[k].requires_grad_()
    s, h = call(t, norm, gate_kind, alpha)
    outs = [s] + ([h] if h is not None else [])
    grads = torch.autograd.grad(outs, [t[k] for k in leaves],
                                [t["dsum"], t["dh"]][:len(outs)])
    return s, h, dict(zip(leaves, grads))


def check_case(dev, R, D, dtype, norm="layer", gate=None, alpha=1.0, **kw):
    t = make(R, D, dtype, dev, norm=norm, gate=gate, **kw)
    s, h, grads = run(t, norm, gate or "scale", alpha)
    want = oracle(t, norm, gate, alpha)
    close("s", s, want["s"], dtype)
    assert (h is None) == (t["pre_scale"] is None)
    if h is not None:
        close("h", h, want["h"], dtype)
    for k, g in grads.items():
        close(k, g, want[k], t[k].dtype)


CPU_CASES = [
    dict(R=3, D=8, dtype=torch.float32),
    dict(R=3, D=5, dtype=torch.float32, norm="rms", gate="scale", alpha=0.5),
    dict(R=4, D=16, dtype=torch.bfloat16, gate="highway", per_token=True),
    dict(R=4, D=16, dtype=torch.float32, gate="highway", post=False),
    dict(R=4, D=16, dtype=torch.float32, gate="scale", pre=False, alpha=0.7),
    dict(R=4, D=9, dtype=torch.float32, norm="rms", pre=False, no_res=True),
]


@pytest.mark.parametrize("case", CPU_CASES)
def test_plain_matches_oracle(case):
    check_case("cpu", **case)


@pytest.mark.parametrize("norm", ["layer", "rms"])
@pytest.mark.parametrize("gate", [None, "scale", "highway"])
def test_plain_gradients_by_differences(norm, gate):
    t = make(3, 6, torch.float64, "cpu", norm=norm, gate=gate, seed=2)
    keys = [k for k in LEAVES if t[k] is not None]

    def fn(*a):
        return call({**t, **dict(zip(keys, a))}, norm, gate or "scale", 0.7)
    assert torch.autograd.gradcheck(
        fn, [t[k].clone().requires_grad_() for k in keys])


@pytest.mark.parametrize("dev", ["cpu", pytest.param(
    "cuda", marks=pytest.mark.gpu)])
def test_refusals(dev):
    x, w = torch.zeros(2, 3, 4, device=dev), torch.ones(4, device=dev)
    zeros = lambda *s: torch.zeros(*s, device=dev)

    def refused(*a, **k):
        with pytest.raises(ValueError):
            ops.block_norm(*a, **k)
    refused(x, x[:1])
    refused(x, x.bfloat16())
    refused(x.long(), x.long())
    refused(x[..., :0], x[..., :0])
    refused(zeros(()), zeros(()))
    refused(zeros(1, 16385), zeros(1, 16385))
    refused(x, x, norm="batch")
    refused(x, x, gate_kind="tanh")
    refused(x, x, gate=w[:3])
    refused(x, x, gate=zeros(3, 4))
    refused(x, x, gate=zeros(2, 1, 4))
    refused(x, x, gate=zeros(2, 3, 4).bfloat16())
    refused(x, None, gate=x, gate_kind="highway")
    refused(x, x, post_bias=w)
    refused(x, x, pre_scale=w[:3])
    refused(x, x, pre_scale=w.double())
    refused(x, x, pre_scale=w, pre_bias=w.bfloat16())
    refused(x, x, pre_scale=w[None])
    if dev == "cuda":
        refused(x, x.cpu())
        refused(x, x, pre_scale=w.cpu())
        refused(x.double(), x.double())


@pytest.mark.parametrize("dev", ["cpu", pytest.param(
    "cuda", marks=pytest.mark.gpu)])
def test_gpu_call_refuses_modes(dev):
    """No tangent is dropped and no trace holds a constant. Off the GPU the
    extension is called, which looks at the mode before it asks for a GPU."""
    import torch.autograd.forward_ad as fwd
    ext = ops.hip_ext()
    if ext is None:
        pytest.skip("the extension is not built")

    def fn(x, res, gate, w1, b1, w2, b2):
        if dev == "cuda":
            return ops.block_norm(x, res, gate, "highway", 0.5, w1, b1, w2, b2)
        return ext.block_norm(x, res, gate, "highway", 0.5, w1, b1, w2, b2,
                              "layer", 1e-9)
    tensors = tuple(torch.randn(2, 3, 4, device=dev) for _ in range(3)) \
        + tuple(torch.randn(4, device=dev) for _ in range(4))
    for i, t in enumerate(tensors):
        for grad in (True, False):
            with fwd.dual_level(), torch.set_grad_enabled(grad):
                a = list(tensors)
                a[i] = fwd.make_dual(t, torch.ones_like(t))
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    fn(*a)
    with torch.no_grad(), pytest.raises(NotImplementedError, match="traced"):
        torch.jit.trace(fn, tensors, check_trace=False)


@pytest.mark.parametrize("gate", ["scale", "highway"])
@pytest.mark.parametrize("per_token", [True, False])
def test_plain_other_derivatives(gate, per_token):
    """Off the GPU: forward mode, second derivatives, batches, traces."""
    t = make(3, 6, torch.float64, "cpu", gate=gate, per_token=per_token,
             seed=2)
    keys = [k for k in LEAVES if t[k] is not None]

    def fn(*a):
        return call({**t, **dict(zip(keys, a))}, "layer", gate, 0.7)
    leaves = [t[k].clone().requires_grad_() for k in keys]
    assert torch.autograd.gradcheck(fn, leaves, check_forward_ad=True)
    assert torch.autograd.gradgradcheck(fn, leaves)
    plain = [t[k] for k in keys]
    at = [keys.index("x"), keys.index("res")]
    rows = lambda x, r: fn(*[x if i == at[0] else r if i == at[1] else v
                             for i, v in enumerate(plain)])[1]
    x, r = (torch.stack([plain[i], 3 * plain[i]]) for i in at)
    many = torch.func.vmap(rows)(x, r)
    jac = torch.func.vmap(torch.func.jacrev(rows))(x, r)
    for i in range(2):
        assert torch.allclose(many[i], rows(x[i], r[i]), rtol=1e-12)
        assert torch.allclose(jac[i], torch.func.jacfwd(rows)(x[i], r[i]),
                              rtol=1e-9, atol=1e-12)
    traced = torch.jit.trace(fn, plain, check_trace=False)
    other = [2 * v for v in plain]
    for a, b in zip(traced(*other), fn(*other)):
        assert torch.allclose(a, b, rtol=1e-12, atol=1e-12)


@pytest.mark.parametrize("dev", ["cpu", pytest.param(
    "cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("pre", [True, False])
@pytest.mark.parametrize("lead", [(6,), (2, 3), (2, 1, 3)])
def test_outputs_may_be_changed_in_place(dev, lead, pre):
    """As a following in-place op does, whatever the number of dimensions:
    with a gradient of its own, and where only what changes them has one."""
    t = make(6, 40, torch.float32, dev, gate="scale", pre=pre)
    v = {k: a.view(*lead, 40) if a is not None and a.dim() == 2 else a
         for k, a in t.items()}
    leaves = [v[k] for k in LEAVES if v[k] is not None]
    c = torch.full_like(v["x"], 1.5)
    changed = lambda o, c: o.mul_(c).relu_()

    outs = [o for o in call(v, "layer", "scale", 0.5) if o is not None]
    for o in outs:              # no gradient but c's
        got = changed(o.clone(), c)
        cg = c.clone().requires_grad_()
        now = changed(o, cg)
        assert torch.equal(now, got)
        g, = torch.autograd.grad(now.sum(), cg)
        assert torch.equal(g != 0, now > 0)
    for a in leaves:
        a.requires_grad_()

    def grads(fn):
        outs = [o for o in call(v, "layer", "scale", 0.5) if o is not None]
        outs = [fn(o) for o in outs]
        return outs + list(torch.autograd.grad(
            outs, leaves, [torch.ones_like(o) for o in outs]))
    for p, q in zip(grads(lambda o: changed(o, c)),
                    grads(lambda o: changed(o.clone(), c))):
        assert torch.equal(p, q)


@pytest.mark.parametrize("dev", ["cpu", pytest.param(
    "cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("name", ["x", "res", "gate", "pre_scale"])
def test_broadcast_inputs(dev, name):
    """An expanded input, and the sum that its gradient is."""
    t = make(5, 24, torch.float32, dev, gate="scale", per_token=True)
    one = t[name][:1].clone().requires_grad_()
    shape = t[name].shape
    res = []
    for full in (one.expand(shape), one.expand(shape).contiguous()):
        o = call({**t, name: full}, "layer", "scale", 0.5)
        d = [(a, b) for a, b in zip(o, (t["dsum"], t["dh"]))
             if a.requires_grad]
        res.append(o + torch.autograd.grad([a for a, _ in d], one,
                                           [b for _, b in d]))
    assert res[0][2].shape == one.shape
    assert all(torch.equal(p, q) for p, q in zip(*res))


@pytest.mark.parametrize("dev", ["cpu", pytest.param(
    "cuda", marks=pytest.mark.gpu)])
def test_inference_mode(dev):
    t = make(6, 24, torch.bfloat16, dev, gate="highway")
    want = call(t, "layer", "highway", 0.5)
    with torch.inference_mode():
        got = call(t, "layer", "highway", 0.5)
    assert all(o.is_inference() for o in got)
    assert all(torch.equal(p, q) for p, q in zip(got, want))


# ------------------------------------------------------------------ on the GPU

GPU_CASES = [
    dict(R=1, D=1, dtype=torch.float32),
    dict(R=5, D=1, dtype=torch.bfloat16, norm="rms", gate="scale"),
    dict(R=300, D=3, dtype=torch.float32, norm="rms", gate="highway",
         alpha=0.7),
    dict(R=7, D=8, dtype=torch.float16),
    dict(R=257, D=20, dtype=torch.float32, gate="scale", bias=False),
    dict(R=33, D=64, dtype=torch.bfloat16, gate="highway", per_token=True),
    dict(R=9, D=130, dtype=torch.float16, norm="rms", gate="scale",
         per_token=True, alpha=0.5),
    dict(R=1030, D=257, dtype=torch.bfloat16, gate="scale"),
    dict(R=17, D=511, dtype=torch.float32, gate="highway"),
    dict(R=6, D=512, dtype=torch.bfloat16, pdt=torch.float32, gate="scale"),
    dict(R=6, D=513, dtype=torch.float16, pdt=torch.float32, gate="highway"),
    dict(R=2500, D=1024, dtype=torch.bfloat16, gate="scale", alpha=0.5),
    dict(R=3, D=1021, dtype=torch.float32, norm="rms"),
    dict(R=4, D=2050, dtype=torch.bfloat16, gate="highway"),
    dict(R=5, D=4096, dtype=torch.float32, gate="scale", per_token=True),
    dict(R=5, D=4097, dtype=torch.bfloat16, gate="scale"),
    dict(R=3, D=8191, dtype=torch.float32, gate="highway"),
    dict(R=3, D=8200, dtype=torch.float16, norm="rms", gate="scale"),
    dict(R=2, D=16384, dtype=torch.float32, gate="highway", per_token=True),
    dict(R=9, D=96, dtype=torch.float32, post=False),
    dict(R=9, D=96, dtype=torch.bfloat16, pre=False, gate="scale"),
    dict(R=9, D=96, dtype=torch.bfloat16, pre=False, post=False),
    dict(R=9, D=96, dtype=torch.float16, pre=False, post=False,
         gate="highway", alpha=0.5),
    dict(R=9, D=1000, dtype=torch.float32, pre=False, post=False,
         gate="scale", per_token=True),
    dict(R=9, D=96, dtype=torch.float32, norm="rms", pre=False, no_res=True),
    dict(R=9, D=700, dtype=torch.bfloat16, gate="scale", no_res=True),
    dict(R=9, D=50, dtype=torch.float16, gate="scale", per_token=True,
         post=False, pre=False, no_res=True),
    # a mean far from 0 beside the deviation
    dict(R=12, D=700, dtype=torch.float32, shift=300.0),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", GPU_CASES)
def test_gpu_matches_oracle(case):
    check_case("cuda", **case)


@pytest.mark.gpu
def test_gpu_no_rows():
    w = torch.ones(8, device="cuda", requires_grad=True)
    x = torch.zeros(0, 3, 8, device="cuda", requires_grad=True)
    s, h = ops.block_norm(x, x, gate=w, post_scale=w, pre_scale=w, pre_bias=w)
    assert s.shape == h.shape == x.shape
    gx, gw = torch.autograd.grad((s.sum() + h.sum()), (x, w))
    assert gx.shape == x.shape and bool((gw == 0).all())


@pytest.mark.gpu
def test_gpu_shapes_and_strides():
    """Leading dimensions, views that are not dense, one row as a vector."""
    t = make(12, 40, torch.float32, "cuda", gate="scale", per_token=True)
    base = call(t, "layer", "scale", 1.0)
    r = {k: v.view(3, 4, 40) if v is not None and v.dim() == 2 else v
         for k, v in t.items()}
    got = call(r, "layer", "scale", 1.0)
    assert all(torch.equal(a, b.view(12, 40)) for a, b in zip(base, got))
    wide = torch.cat([t["x"], t["res"]], 1)
    v = {**t, "x": wide[:, :40], "res": wide[:, 40:],
         "gate": t["gate"].t().contiguous().t(),
         "pre_scale": t["pre_scale"].repeat_interleave(2)[::2]}
    got = call(v, "layer", "scale", 1.0)
    assert all(torch.equal(a, b) for a, b in zip(base, got))
    one = {k: w[0] if w is not None and w.dim() == 2 else w
           for k, w in t.items()}
    got = call(one, "layer", "scale", 1.0)
    assert all(torch.equal(a[0], b) for a, b in zip(base, got))


@pytest.mark.gpu
def test_gpu_partial_gradients():
    t = make(70, 300, torch.float32, "cuda", gate="highway")
    s, h, full = run(t, "layer", "highway", 1.0)
    zero = torch.zeros_like(t["dsum"])
    keys = list(full)
    ins = [t[k] for k in keys]
    both = call(t, "layer", "highway", 1.0)
    for i, d in ((0, t["dsum"]), (1, t["dh"])):
        a = torch.autograd.grad(both[i], ins, d, retain_graph=True,
                                allow_unused=True)
        b = torch.autograd.grad(both, ins, (d, zero) if i == 0 else (zero, d),
                                retain_graph=True)
        assert all(torch.equal(p, q) for p, q in zip(a, b))
    for k in keys:      # one input at a time
        r = {n: None if v is None else v.detach() for n, v in t.items()}
        r[k] = r[k].clone().requires_grad_()
        g, = torch.autograd.grad(call(r, "layer", "highway", 1.0), r[k],
                                 (t["dsum"], t["dh"]))
        assert torch.equal(g, full[k]), k


@pytest.mark.gpu
@pytest.mark.parametrize("gate", ["scale", "highway"])
@pytest.mark.parametrize("norm,post", [("layer", True), ("rms", True),
                                       ("layer", False)])
@pytest.mark.parametrize("D", [3, 100, 300, 1000, 2000, 4200, 8300])
def test_gpu_each_gradient_alone(D, norm, post, gate):
    """A parameter's sums do not depend on which others are asked for."""
    t = make(20, D, torch.float32, "cuda", norm=norm, gate=gate, post=post)
    full = run(t, norm, gate, 0.5)[2]
    for k in full:
        r = {n: None if v is None else v.detach() for n, v in t.items()}
        r[k] = r[k].clone().requires_grad_()
        g, = torch.autograd.grad(call(r, norm, gate, 0.5), r[k],
                                 (t["dsum"], t["dh"]))
        assert torch.equal(g, full[k]), k


@pytest.mark.gpu
def test_gpu_is_differentiable_once():
    t = make(4, 32, torch.float32, "cuda", gate="scale")
    t["x"].requires_grad_()
    g, = torch.autograd.grad(call(t, "layer", "scale", 1.0)[1], t["x"],
                             t["dh"], create_graph=True)
    with pytest.raises(RuntimeError, match="once"):
        g.sum().backward()


@pytest.mark.gpu
def test_gpu_bad_rows_stay_alone():
    """NaN and infinity in one row, at the end of the last block too."""
    for bad in (3, 44):
        t = make(45, 100, torch.float32, "cuda", gate="scale")
        ok = call(t, "layer", "scale", 1.0)
        t["x"][bad, 5] = float("nan")
        t["res"][bad, 7] = float("inf")
        got = call(t, "layer", "scale", 1.0)
        keep = torch.arange(45, device="cuda") != bad
        for a, b in zip(ok, got):
            assert torch.equal(a[keep], b[keep])
        assert bool(torch.isnan(got[1][bad]).all())


@pytest.mark.gpu
def test_gpu_repeats_bit_for_bit():
    t = make(3001, 520, torch.bfloat16, "cuda", gate="highway")
    first = run(t, "layer", "highway", 1.0)
    for _ in range(3):
        again = run(t, "layer", "highway", 1.0)
        assert torch.equal(first[0], again[0])
        assert torch.equal(first[1], again[1])
        assert all(torch.equal(first[2][k], again[2][k]) for k in first[2])


@pytest.mark.gpu
@pytest.mark.parametrize("R,D", [(1000, 700), (1000, 200), (1500, 1024),
                                 (2000, 4200)])
def test_gpu_sums_over_rows_in_pairs(R, D):
    """dpre_bias is the sum of dh. A rounding of a partial sum v is at most
    u v and spreads evenly, u v / sqrt(3) in the root mean square. For terms of
    one sign partial sums grow in proportion: 64 lane groups' sums in 16 runs
    of 4 and then in pairs have squares of 0.12 + 1.88 of the whole sum's, what
    comes before (a block's rows, 4 to 16 blocks a group) below 0.25, the last
    rounding 1: u S sqrt(3.25 / 3). One run of 64 has 21 in place of 2."""
    gen = torch.Generator().manual_seed(8)
    x = torch.randn(R, D, generator=gen).cuda()
    dh = (torch.rand(R, D, generator=gen) + 0.5).cuda()
    w, b = torch.ones(D).cuda(), torch.zeros(D).cuda().requires_grad_()
    _, h = ops.block_norm(x, None, pre_scale=w, pre_bias=b)
    got, = torch.autograd.grad(h, b, dh)
    want = dh.double().sum(0)
    rms = ((got.double() - want) / want).square().mean().sqrt()
    assert float(rms) <= U * (3.25 / 3) ** 0.5


@pytest.mark.gpu
def test_gpu_two_streams_at_once():
    """Calls that overlap on two streams share nothing."""
    jobs = []
    for seed, D in ((1, 300), (2, 1024)):
        t = make(3000, D, torch.bfloat16, "cuda", gate="scale", seed=seed)

        def once(t=t):
            s, h, g = run(t, "layer", "scale", 1.0)
            return [s, h] + list(g.values())
        jobs.append((once, torch.cuda.Stream(), once()))
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for (once, side, _), outs in zip(jobs, got):
            with torch.cuda.stream(side):
                outs.append(once())
    torch.cuda.synchronize()
    for (_, _, want), outs in zip(jobs, got):
        for o in outs:
            assert all(torch.equal(p, q) for p, q in zip(o, want))


@pytest.mark.gpu
def test_gpu_captured():
    """Forward and backward replayed from two graphs that interleave."""
    graphs = []
    for seed, D in ((1, 256), (2, 700)):
        t = make(500, D, torch.bfloat16, "cuda", gate="scale", seed=seed)

        def once(t=t):
            s, h, g = run(t, "layer", "scale", 1.0)
            return [s.detach(), h.detach()] + list(g.values())
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            once()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = once()
        graphs.append((graph, outs, once))
    for _ in range(3):
        for _, outs, _ in graphs:
            for o in outs:
                o.zero_()
        for graph, _, _ in graphs:
            graph.replay()
        for _, outs, once in graphs:
            assert all(torch.equal(p, q) for p, q in zip(outs, once()))


@pytest.mark.gpu
def test_gpu_offsets_beyond_32_bits():
    """More than 2^31 elements: the last rows come out as they do on their
    own, gradients too."""
    R, n, D = 4_400_000, 1000, 512
    t = make(n, D, torch.bfloat16, "cuda", gate="scale", per_token=True)
    big = {k: v.repeat(R // n, 1) if v is not None and v.dim() == 2 else v
           for k, v in t.items()}
    s, h, g = run(big, "layer", "scale", 0.5)
    s2, h2, g2 = run(t, "layer", "scale", 0.5)
    assert torch.equal(s[-n:], s2) and torch.equal(h[-n:], h2)
    for k in ("x", "res", "gate"):
        assert torch.equal(g[k][-n:], g2[k]), k


@pytest.mark.parametrize("dev", ["cpu", pytest.param(
    "cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("R,D", [(3000, 3), (3000, 40), (2000, 700),
                                 (600, 1500), (300, 4100), (40, 8200)])
@pytest.mark.parametrize("mean", [0.0, 300.0])
def test_highway_gate_beside_a_common_mean(dev, mean, R, D):
    """The gate of a channel's highway gets the sum of (x - res) ds, however
    far from 0 both of them are. Without norms and with a factor of 1, x - res
    is rounded once, its product with ds once, and the sum over rows stays
    within 128 u of the sum of absolute values; the sigmoid's parts are good to
    3 u each and three products follow."""
    gen = torch.Generator().manual_seed(5)
    res = torch.randn(R, D, generator=gen) + mean
    x = res + 0.01 * torch.randn(R, D, generator=gen)
    ds = torch.randn(R, D, generator=gen) + 0.5
    gate = torch.randn(D, generator=gen)
    g = gate.to(dev).requires_grad_()
    s, _ = ops.block_norm(x.to(dev), res.to(dev), g, "highway")
    got, = torch.autograd.grad(s, g, ds.to(dev))
    k = torch.sigmoid(gate.double())
    terms = (x.double() - res.double()) * ds.double()
    want = k * (1 - k) * terms.sum(0)
    lim = (128 + 2 + 6 + 3) * U * k * (1 - k) * terms.abs().sum(0)
    err = (got.double().cpu() - want).abs()
    assert bool((err <= lim + U * want.abs()).all()), float((err / lim).max())


@pytest.mark.parametrize("dev", ["cpu", pytest.param(
    "cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("R,D", [(4096, 2), (4096, 64), (3000, 256),
                                 (3000, 512), (3000, 1024), (1500, 2048),
                                 (600, 8192), (600, 16384)])
def test_factor_behind_a_cancelled_channel(dev, R, D):
    """The factor of a channel whose bias takes back what the norm makes of it
    gets the sum of u ds. Rows of 1 and -1 have a root mean square of 1 exactly
    (D is a power of two, eps vanishes beside 1), so a channel of ones with
    the bias -1 + 2^-16 has u = 2^-16 exactly; the product with ds is rounded
    once and the sum over rows stays within 128 u of the sum of absolute
    values. The sums of xh ds and of ds themselves are 2^16 times as large."""
    gen = torch.Generator().manual_seed(6)
    x = torch.randint(0, 2, (R, D), generator=gen).float() * 2 - 1
    x[:, 1] = 1
    ds = torch.randn(R, D, generator=gen) + 0.5
    w, b = torch.ones(D), torch.zeros(D)
    b[1] = -1 + 2.0 ** -16
    g = torch.ones(D).to(dev).requires_grad_()
    s, _ = ops.block_norm(x.to(dev), None, g, post_scale=w.to(dev),
                          post_bias=b.to(dev), norm="rms", eps=1e-30)
    got, = torch.autograd.grad(s, g, ds.to(dev))
    terms = (x.double() + b.double()) * ds.double()
    err = (got.double().cpu() - terms.sum(0)).abs()
    lim = 130 * U * terms.abs().sum(0)
    assert bool((err <= lim).all()), float((err / lim).max())


@pytest.mark.gpu
@pytest.mark.parametrize("case", [
    dict(R=600, D=4097, dtype=torch.bfloat16, gate="scale", alpha=0.5),
    dict(R=520, D=9001, dtype=torch.float32),
    dict(R=3, D=4104, dtype=torch.float16, pdt=torch.float32),
    dict(R=4, D=6001, dtype=torch.bfloat16, gate="highway"),
    dict(R=4, D=8192, dtype=torch.bfloat16, gate="scale", per_token=True),
    dict(R=4, D=8191, dtype=torch.float32, gate="highway", per_token=True),
    dict(R=4, D=8192, dtype=torch.float32, post=False, gate="scale"),
    dict(R=4, D=5000, dtype=torch.float16, pre=False),
    dict(R=3, D=8193, dtype=torch.bfloat16, gate="highway", alpha=0.7),
    dict(R=3, D=16384, dtype=torch.bfloat16, no_res=True),
    dict(R=3, D=16384, dtype=torch.float16, pre=False, gate="scale"),
])
def test_gpu_wide_rms(case):
    """rms norms without biases have a backward kernel of their own for wide
    rows; 520 and 600 rows give a block several."""
    check_case("cuda", norm="rms", **case)


@pytest.mark.gpu
@pytest.mark.parametrize("bias", ["post_bias", "pre_bias"])
def test_gpu_wide_rms_with_a_bias(bias):
    t = make(300, 4500, torch.float32, "cuda", norm="rms", gate="scale")
    t[bias] = torch.linspace(-1, 1, 4500, device="cuda")
    _, _, grads = run(t, "rms", "scale", 1.0)
    want = oracle_with_bias(t, bias)
    for k, g in grads.items():
        close(k, g, want[k], t[k].dtype)


def oracle_with_bias(t, bias):
    """The oracle takes both biases or none: the other one is zero."""
    zero = torch.zeros(t["x"].shape[-1], device=t["x"].device)
    return oracle({k: zero if v is None and k.endswith("bias") else v
                   for k, v in t.items()}, "rms", "scale", 1.0)


def test_every_kernel_has_a_width():
    """The extension holds the kernels that some width picks, and no others:
    (vector, elements a lane, place of a row's lanes, threads at most)."""
    import re
    from marian_amd.ops import _load
    path = _load.extension_path()
    if path is None:
        pytest.skip("the extension is not built")
    part_wave, wave, pair, block = range(4)

    def plan(D, vec, bwd):
        if D < vec:
            return 1, 1, part_wave, 256
        if D <= 256:
            return vec, 8, part_wave, 256
        if D <= 512:
            return vec, 8, wave, 256
        if D <= 1024:
            return (vec, 8, pair, 256) if bwd else \
                (vec, 16, wave, 256) if vec == 8 else (vec, 8, block, 512)
        if D <= 4096:
            return vec, 8, block, 512
        return vec, 16, block, 512 if D <= 8192 else 1024
    with open(path, "rb") as f:
        names = set(re.findall(
            rb"join_(fwd|bwd)_kernelI(f|DF16b|DF16_)Li(\d+)ELi(\d+)ELi(\d+)E"
            rb"Lb[01]ELb[01]ELi\d+ELi(\d+)E", f.read()))
    for way in ("fwd", "bwd"):
        for name, vec in (("f", 4), ("DF16b", 8), ("DF16_", 8)):
            held = {tuple(map(int, n[2:])) for n in names
                    if n[0].decode() == way and n[1].decode() == name}
            assert held == {plan(D, vec, way == "bwd")
                            for D in range(1, 16385)}, (way, name)
