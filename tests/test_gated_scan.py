"""Gated linear recurrence (ops.gated_scan, gated_scan_xg, gated_step) against
the recurrence and its gradient written out step by step in 64 bits.

Tolerances. With u = 2^-24 one step  c = f c' + om x  has an error of at most
(e_f + e_om + 3) u amax, where the sigmoid's parts are good to e = |g| + 3
units (its exponential's argument is rounded once, exp, sum and reciprocal
add one unit each); earlier errors are multiplied by f <= 1, and joining runs
of steps costs a product and a sum per join, at most one join per step. So T
steps stay within K u amax with K = T (4 gmax + 32), amax the largest |x| or
|state|. The gradient's recurrence is the same one, over lam; dg multiplies
lam, c - x and f om <= 1/4. The last rounding to the output's type adds
eps / 2 of the value.
"""
import numpy as np
import pytest
import torch

from marian_amd import ops

U = 2.0 ** -24


def oracle(x, g, state, lens, reverse, act, dy, dlast):
    """All results in float64, and the largest |lam|."""
    x, g, dy = x.double().cpu(), g.double().cpu(), dy.double().cpu()
    B, T, D = x.shape
    c = torch.zeros(B, D, dtype=torch.float64) if state is None \
        else state.double().cpu()
    lam_in = dlast.double().cpu().clone()
    y, dx, dg = (torch.zeros_like(x) for _ in range(3))
    dstate = torch.zeros(B, D, dtype=torch.float64)
    last = c.clone()
    lmax, cmin = float(lam_in.abs().max()) if lam_in.numel() else 0.0, 1e9
    for b in range(B):
        n = T if lens is None else min(max(int(lens[b]), 0), T)
        order = list(range(n))[::-1] if reverse else list(range(n))
        cur, prevs = c[b].clone(), []
        for t in order:
            f = 1 / (1 + torch.exp(-g[b, t]))
            prevs.append(cur)
            cur = f * cur + (1 - f) * x[b, t]
            y[b, t] = torch.where(cur < 0, 0 * cur, cur) if act == "relu" \
                else cur
            if act == "relu":
                cmin = min(cmin, float(cur.abs().min()))
        last[b] = cur
        mu = lam_in[b].clone()
        for t, prev in zip(order[::-1], prevs[::-1]):
            f = 1 / (1 + torch.exp(-g[b, t]))
            now = f * prev + (1 - f) * x[b, t]
            d = torch.where(now > 0, dy[b, t], 0 * now) if act == "relu" \
                else dy[b, t]
            lam = d + mu
            lmax = max(lmax, float(lam.abs().max()))
            dx[b, t] = (1 - f) * lam
            dg[b, t] = f * (1 - f) * (prev - x[b, t]) * lam
            mu = f * lam
        dstate[b] = mu
    return y, last, dx, dg, dstate, lmax, cmin


def close(got, want, atol, dtype):
    half = torch.finfo(dtype).eps / 2 * (1 + 2.0 ** -7)
    got = got.detach().double().cpu()
    assert got.shape == want.shape
    err = (got - want).abs()
    lim = atol + half * (want.abs() + atol)
    assert bool((err <= lim).all()), \
        f"off by {float((err - lim).max())} over the limit"


def make(B, T, D, dtype, dev, seed, state=True, lens=None):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen)
    xg = torch.cat([r(B, T, D), r(B, T, D) * 2 + 0.5], -1).to(dtype).to(dev)
    sdt = torch.float64 if dtype == torch.float64 else torch.float32
    st = r(B, D).to(sdt).to(dev) if state else None
    ln = None
    if lens == "ragged":
        ln = torch.randint(0, T + 1, (B,), generator=gen).to(torch.int32)
        ln[0] = 0
        if B > 1:
            ln[1] = T
        ln = ln.to(dev)
    dy = r(B, T, D).to(dtype).to(dev)
    dlast = r(B, D).to(sdt).to(dev)
    return xg, st, ln, dy, dlast


def check_case(dev, B, T, D, dtype, lens=None, reverse=False, act="none",
               state=True, layout="split", seed=0):
    # relu's side must not be a matter of rounding: the first inputs whose
    # states, by the oracle, all stay further from 0 than the tolerance
    for seed in range(seed, seed + 200):
        xg, st, ln, dy, dlast = make(B, T, D, dtype, dev, seed, state, lens)
        want = oracle(xg[..., :D], xg[..., D:], st, ln, reverse, act, dy,
                      dlast)
        gmax = float(xg[..., D:].abs().max()) if xg.numel() else 0.0
        K = max(T, 1) * (4 * gmax + 32) * U
        amax = float(xg[..., :D].abs().max()) if xg.numel() else 0.0
        if st is not None:
            amax = max(amax, float(st.abs().max()))
        if want[6] > K * amax:
            break
    assert want[6] > K * amax
    if st is not None:
        st.requires_grad_()
    kw = dict(state=st, lens=ln, reverse=reverse, act=act)
    if layout == "fused":
        xg.requires_grad_()
        leaves = [xg]
        y, last = ops.gated_scan_xg(xg, **kw)
    else:
        if layout == "views":       # halves of one buffer, transposed batch
            buf = xg.transpose(0, 1).contiguous().transpose(0, 1)
            x, g = buf[..., :D], buf[..., D:]
        else:
            x, g = xg[..., :D].contiguous(), xg[..., D:].contiguous()
        if layout == "columns":     # the last dimension is not dense
            x = x.transpose(1, 2).contiguous().transpose(1, 2)
        x, g = x.detach().requires_grad_(), g.detach().requires_grad_()
        leaves = [x, g]
        y, last = ops.gated_scan(x, g, **kw)
    assert y.dtype == dtype and y.is_contiguous()
    if st is not None:
        leaves.append(st)
    grads = torch.autograd.grad((y, last), leaves, (dy, dlast))
    if layout == "fused":
        grads = (grads[0][..., :D], grads[0][..., D:]) + grads[1:]
    sdt = last.dtype
    lmax = want[5]
    close(y, want[0], K * amax, dtype)
    close(last, want[1], K * amax, sdt)
    close(grads[0], want[2], K * lmax, dtype)
    close(grads[1], want[3], K * lmax * 2 * amax, dtype)
    if st is not None:
        close(grads[2], want[4], K * lmax, sdt)


CPU_CASES = [
    dict(B=2, T=5, D=3, dtype=torch.float32),
    dict(B=3, T=9, D=4, dtype=torch.float32, lens="ragged", reverse=True),
    dict(B=2, T=7, D=5, dtype=torch.bfloat16, act="relu", layout="fused"),
    dict(B=2, T=1, D=2, dtype=torch.float64, state=False),
    dict(B=1, T=0, D=2, dtype=torch.float32),
]


@pytest.mark.parametrize("case", CPU_CASES)
def test_scan_plain_matches_oracle(case):
    check_case("cpu", **case)


def test_scan_plain_gradients_by_differences():
    xg, st, ln, _, _ = make(2, 6, 3, torch.float64, "cpu", 3, True, "ragged")
    xg.requires_grad_()
    st.requires_grad_()
    for rev in (False, True):
        assert torch.autograd.gradcheck(
            lambda a, s: ops.gated_scan_xg(a, s, ln, rev), (xg, st))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_step_walks_like_the_scan(dtype):
    xg, st, _, dy, dl = make(3, 5, 7, dtype, "cpu", 4)
    y, last = ops.gated_scan_xg(xg, st, act="relu")
    want = oracle(xg[..., :7], xg[..., 7:], st, None, False, "relu", dy, dl)
    lim = 5 * (4 * float(xg[..., 7:].abs().max()) + 32) * U \
        * max(float(xg[..., :7].abs().max()), float(st.abs().max()))
    close(y, want[0], lim, dtype)
    cur = st.clone()
    for t in range(5):
        o, new = ops.gated_step(xg[:, t, :7], xg[:, t, 7:], cur, act="relu",
                                inplace=True)
        assert new is cur
        close(o, want[0][:, t], lim, dtype)
    close(last, want[1], lim, torch.float32)
    close(cur, want[1], lim, torch.float32)


def test_step_gradient_is_the_scans():
    xg, st, _, _, _ = make(3, 1, 4, torch.float64, "cpu", 5)
    xg.requires_grad_()
    st.requires_grad_()
    assert torch.autograd.gradcheck(
        lambda a, s: ops.gated_step(a[:, 0, :4], a[:, 0, 4:], s), (xg, st))


def _refused(fn, *a, **k):
    with pytest.raises(ValueError):
        fn(*a, **k)


DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


@pytest.mark.parametrize("dev", DEVICES)
def test_scan_refusals(dev):
    x = torch.zeros(2, 3, 4, device=dev)
    s = torch.zeros(2, 4, device=dev)
    zeros = lambda n, dtype=torch.float32: torch.zeros(n, dtype=dtype,
                                                       device=dev)
    _refused(ops.gated_scan, x[0], x[0])
    _refused(ops.gated_scan, x, x[:, :2])
    _refused(ops.gated_scan, x, x.bfloat16())
    _refused(ops.gated_scan, x.long(), x.long())
    _refused(ops.gated_scan, x[..., :0], x[..., :0])
    _refused(ops.gated_scan, x, x, act="tanh")
    _refused(ops.gated_scan, x, x, state=s.bfloat16())
    _refused(ops.gated_scan, x, x, state=s[:1])
    _refused(ops.gated_scan, x, x, lens=zeros(2))
    _refused(ops.gated_scan, x, x, lens=zeros(3, torch.int32))
    _refused(ops.gated_scan, x, x, lens=zeros(2, torch.int64))
    if dev == "cuda":
        _refused(ops.gated_scan, x, x.cpu())
        _refused(ops.gated_scan, x, x, state=s.cpu())
        _refused(ops.gated_scan, x, x, lens=zeros(2, torch.int32).cpu())
        _refused(ops.gated_scan, x.double(), x.double())
    _refused(ops.gated_scan_xg, x[..., :3])
    _refused(ops.gated_scan_xg, x[0])


@pytest.mark.parametrize("dev", DEVICES)
def test_step_refusals(dev):
    x, s = torch.zeros(2, 4, device=dev), torch.zeros(2, 4, device=dev)
    _refused(ops.gated_step, x, x, None)
    _refused(ops.gated_step, x[:, None], x[:, None], s)
    _refused(ops.gated_step, x, x, s[:1])
    _refused(ops.gated_step, x, x, s.half())
    _refused(ops.gated_step, x, x, torch.zeros(4, 2, device=dev).t(),
             inplace=True)
    _refused(ops.gated_step, x, s, s, inplace=True)
    _refused(ops.gated_step, x.requires_grad_(), x, s, inplace=True)


@pytest.mark.parametrize("dev", DEVICES)
def test_step_in_place_is_seen_by_autograd(dev):
    """A graph that holds the old state does not use the new one."""
    x = torch.randn(2, 4, device=dev, requires_grad=True)
    s = torch.randn(2, 4, device=dev)
    y, _ = ops.gated_step(x, x, s)
    with torch.no_grad():
        ops.gated_step(x.detach().clone(), x.detach().clone(), s,
                       inplace=True)
    with pytest.raises(RuntimeError, match="inplace"):
        y.sum().backward()


def refused_modes(call, *tensors):
    """No tangent is dropped and no trace holds a constant: each tensor as a
    dual one, and the call traced."""
    import torch.autograd.forward_ad as fwd
    for i, t in enumerate(tensors):
        for grad in (True, False):
            with fwd.dual_level(), torch.set_grad_enabled(grad):
                a = list(tensors)
                a[i] = fwd.make_dual(t, torch.ones_like(t))
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    call(*a)
    with torch.no_grad(), pytest.raises(NotImplementedError, match="traced"):
        torch.jit.trace(call, tensors, check_trace=False)


def gpu_entries(dev):
    """The GPU's entry points; off the GPU the extension's, which look at the
    mode before they ask for a GPU."""
    if dev == "cuda":
        return ops.gated_scan, ops.gated_scan_xg, ops.gated_step
    ext = ops.hip_ext()
    if ext is None:
        pytest.skip("the extension is not built")
    return (lambda x, g, s: ext.gated_scan(x, g, s, None, False, "none"),
            lambda xg, s: ext.gated_scan_xg(xg, s, None, False, "none"),
            lambda x, g, s: ext.gated_step(x, g, s, "none", False))


@pytest.mark.parametrize("dev", DEVICES)
def test_gpu_calls_refuse_modes(dev):
    scan, scan_xg, step = gpu_entries(dev)
    xg, s = torch.randn(2, 3, 8, device=dev), torch.randn(2, 4, device=dev)
    refused_modes(lambda x, g, s: scan(x, g, s), xg[..., :4], xg[..., 4:], s)
    refused_modes(lambda a, s: scan_xg(a, s), xg, s)
    refused_modes(lambda x, g, s: step(x, g, s), xg[:, 0, :4], xg[:, 0, 4:],
                  s)


def test_traces_off_the_gpu():
    """A scan's trace would hold the number of steps; a single step's does
    not."""
    xg, st, _, _, _ = make(2, 3, 4, torch.float32, "cpu", 3)
    for fn in (lambda a, s: ops.gated_scan_xg(a, s),
               lambda a, s: ops.gated_scan(a[..., :4], a[..., 4:], s)):
        with pytest.raises(NotImplementedError, match="traced"):
            torch.jit.trace(fn, (xg, st), check_trace=False)
    step = lambda a, s: ops.gated_step(a[:, :4], a[:, 4:], s, act="relu")
    traced = torch.jit.trace(step, (xg[:, 0], st), check_trace=False)
    more = torch.randn(5, 8), torch.randn(5, 4)
    for a, b in zip(traced(*more), step(*more)):
        assert torch.equal(a, b)


def test_forward_mode_off_the_gpu():
    """There the tangent comes out: against differences."""
    import torch.autograd.forward_ad as fwd
    xg, st, ln, _, _ = make(2, 6, 3, torch.float64, "cpu", 3, True, "ragged")
    v, e = torch.randn_like(xg), 1e-6
    with fwd.dual_level():
        y, last = ops.gated_scan_xg(fwd.make_dual(xg, v), st, ln)
        got = [fwd.unpack_dual(t).tangent for t in (y, last)]
    up, dn = (ops.gated_scan_xg(xg + k * v, st, ln) for k in (e, -e))
    for g, a, b in zip(got, up, dn):
        assert torch.allclose(g, (a - b) / (2 * e), rtol=0, atol=1e-7)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("T,lens", [(0, None), (3, 0)])
def test_last_state_has_memory_of_its_own(dev, T, lens):
    """Without a step the last state is the first one's value, not its
    memory."""
    x, st = torch.ones(2, T, 4, device=dev), torch.ones(2, 4, device=dev)
    ln = None if lens is None else torch.full((2,), lens, dtype=torch.int32,
                                              device=dev)
    _, last = ops.gated_scan(x, x, st, ln)
    assert torch.equal(last, st)
    last.zero_()
    assert bool((st == 1).all())


@pytest.mark.parametrize("dev", DEVICES)
def test_empty_batches(dev):
    for B, T in ((0, 3), (0, 100), (2, 0), (0, 0)):
        xg = torch.zeros(B, T, 8, device=dev, requires_grad=True)
        st = torch.ones(B, 4, device=dev, requires_grad=True)
        y, last = ops.gated_scan_xg(xg, st)
        assert y.shape == (B, T, 4) and torch.equal(last, st)
        a, b = torch.autograd.grad((y, last), (xg, st), (
            torch.ones_like(y), torch.ones_like(last)))
        assert a.shape == xg.shape and torch.equal(b, torch.ones_like(st))
    x, st = torch.zeros(0, 4, device=dev), torch.zeros(0, 4, device=dev)
    for inplace in (False, True):
        y, new = ops.gated_step(x, x.clone(), st, inplace=inplace)
        assert y.shape == new.shape == (0, 4)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("T", [5, 70])
def test_lengths_outside_the_axis(dev, T):
    """Lengths are clamped to 0..T."""
    xg, st, _, dy, dl = make(4, T, 6, torch.float32, dev, 12)
    xg.requires_grad_(), st.requires_grad_()
    res = []
    for lens in ([-3, T + 9, 2 ** 31 - 1, -2 ** 31], [0, T, T, 0]):
        ln = torch.tensor(lens, dtype=torch.int32, device=dev)
        for rev in (False, True):
            o = ops.gated_scan_xg(xg, st, ln, rev)
            res.append(o + torch.autograd.grad(o, (xg, st), (dy, dl)))
    for a, b in ((0, 2), (1, 3)):
        assert all(torch.equal(p, q) for p, q in zip(res[a], res[b]))


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dims", [(0,), (1,), (0, 1), (2,), (0, 1, 2)])
def test_broadcast_inputs(dev, dims):
    """Expanded inputs, and the sums that their gradients are."""
    xg, st, _, dy, dl = make(3, 70, 6, torch.float64 if dev == "cpu" else
                             torch.float32, dev, 13)
    x, g = (a.clone() for a in (xg[..., :6], xg[..., 6:]))
    for d in dims:
        x, g = x.narrow(d, 0, 1), g.narrow(d, 0, 1)
    x, g = x.clone().requires_grad_(), g.clone().requires_grad_()
    res = []
    for full in (lambda a: a.expand(3, 70, 6),
                 lambda a: a.expand(3, 70, 6).contiguous()):
        o = ops.gated_scan(full(x), full(g), st)
        res.append(o + torch.autograd.grad(o, (x, g), (dy, dl)))
    assert res[0][2].shape == x.shape
    # off the GPU torch sums the two layouts in another order: up to 1260 terms
    # in 64 bits are within 1260 x 2^-53 of the sum of their sizes, below 2^14
    lim = 0 if dev == "cuda" else 1260 * 2.0 ** -53 * 2 ** 14
    for p, q in zip(*res):
        assert float((p - q).abs().max()) <= lim


@pytest.mark.parametrize("dev", DEVICES)
def test_inference_mode(dev):
    xg, st, ln, _, _ = make(3, 20, 6, torch.bfloat16, dev, 14, True, "ragged")
    want = ops.gated_scan_xg(xg, st, ln) + ops.gated_step(
        xg[:, 0, :6], xg[:, 0, 6:], st)
    with torch.inference_mode():
        own = st.clone()
        got = ops.gated_scan_xg(xg, st, ln) + ops.gated_step(
            xg[:, 0, :6], xg[:, 0, 6:], own, inplace=True)
    assert got[3] is own and all(t.is_inference() for t in got)
    assert all(torch.equal(p, q) for p, q in zip(got, want))


@pytest.mark.parametrize("dev", DEVICES)
def test_outputs_may_be_changed_in_place(dev):
    xg, st, _, _, _ = make(2, 5, 6, torch.float32, dev, 3)
    xg.requires_grad_(), st.requires_grad_()
    calls = [lambda: ops.gated_scan_xg(xg, st),
             lambda: ops.gated_scan(xg[..., :6], xg[..., 6:], st),
             lambda: ops.gated_step(xg[:, 0, :6], xg[:, 0, 6:], st)]
    for fn in calls:
        res = []
        for copy in (False, True):
            outs = [o.clone() if copy else o for o in fn()]
            for o in outs:
                o.mul_(1.5).relu_()
            res.append(outs + list(torch.autograd.grad(
                outs, (xg, st), [torch.ones_like(o) for o in outs])))
        assert all(torch.equal(p, q) for p, q in zip(*res))


# ------------------------------------------------------------------ on the GPU

GPU_CASES = [
    dict(B=1, T=1, D=1, dtype=torch.float32),
    dict(B=2, T=1, D=3, dtype=torch.bfloat16, state=False),
    dict(B=1, T=0, D=8, dtype=torch.float32),
    dict(B=3, T=2, D=2, dtype=torch.float16),
    dict(B=2, T=63, D=5, dtype=torch.float32, lens="ragged"),
    dict(B=2, T=64, D=64, dtype=torch.bfloat16, layout="fused"),
    dict(B=2, T=65, D=257, dtype=torch.float16, layout="views"),
    dict(B=3, T=66, D=30, dtype=torch.float32, layout="columns"),
    dict(B=4, T=130, D=509, dtype=torch.float32, lens="ragged", reverse=True),
    dict(B=5, T=200, D=33, dtype=torch.bfloat16, lens="ragged", reverse=True,
         layout="fused"),
    dict(B=1, T=1000, D=70, dtype=torch.float32, reverse=True),
    dict(B=1, T=1025, D=256, dtype=torch.bfloat16, layout="fused"),
    dict(B=2, T=40, D=6, dtype=torch.float32, act="relu", lens="ragged"),
    dict(B=2, T=40, D=6, dtype=torch.float32, act="relu", reverse=True),
    # the time axis split over blocks, with relu, raggedness and both ways
    dict(B=1, T=150, D=2, dtype=torch.float32, act="relu"),
    dict(B=2, T=140, D=2, dtype=torch.float32, act="relu", lens="ragged",
         reverse=True),
    dict(B=7, T=700, D=40, dtype=torch.float32, lens="ragged"),
    dict(B=7, T=700, D=41, dtype=torch.bfloat16, lens="ragged", reverse=True,
         layout="views"),
    dict(B=1, T=4200, D=1, dtype=torch.float16),
    dict(B=300, T=3, D=17, dtype=torch.float16, lens="ragged"),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", GPU_CASES)
def test_scan_gpu_matches_oracle(case):
    check_case("cuda", **case)


@pytest.mark.gpu
def test_scan_gpu_padded_values_are_ignored():
    """NaN and infinities behind the sequences, in inputs and gradients."""
    for rev in (False, True):
        xg, st, ln, dy, dlast = make(4, 70, 24, torch.float32, "cuda", 7, True,
                                     "ragged")
        pad = (torch.arange(70, device="cuda")[None] >= ln[:, None])[..., None]
        bad = torch.where(pad, float("nan"), xg).requires_grad_()
        good = xg.clone().requires_grad_()
        st.requires_grad_()
        outs = []
        for a, d in ((good, dy), (bad, torch.where(pad, float("inf"), dy))):
            y, last = ops.gated_scan_xg(a, st, ln, rev)
            outs.append((y, last) + torch.autograd.grad((y, last), (a, st),
                                                        (d, dlast)))
        for p, q in zip(*outs):
            assert torch.equal(p, q)
        assert bool((outs[1][0] * pad == 0).all())
        assert bool((outs[1][2] * pad == 0).all())


@pytest.mark.gpu
def test_scan_gpu_extreme_gates_and_nan():
    """Infinite gate logits keep or replace the state; NaN stays in its
    channel and is not hidden by relu."""
    x = torch.randn(1, 4, 8, device="cuda")
    g = torch.full_like(x, float("inf"))
    st = torch.randn(1, 8, device="cuda")
    y, last = ops.gated_scan(x, g, st)
    assert torch.equal(last, st) and torch.equal(y, st[:, None].expand_as(y))
    y, last = ops.gated_scan(x, -g, st)
    assert torch.equal(y, x) and torch.equal(last, x[:, -1])
    x[0, 1, 3] = float("nan")
    y, last = ops.gated_scan(x, torch.zeros_like(x), st, act="relu")
    want = torch.zeros(1, 4, 8, dtype=torch.bool, device="cuda")
    want[0, 1:, 3] = True
    assert torch.equal(torch.isnan(y), want)


@pytest.mark.gpu
def test_scan_gpu_partial_gradients():
    """Only one of the outputs is used; only one of the inputs wants one."""
    xg, st, _, dy, dlast = make(2, 70, 12, torch.float32, "cuda", 8)
    x, g = xg[..., :12].contiguous(), xg[..., 12:].contiguous()
    x.requires_grad_(), g.requires_grad_(), st.requires_grad_()
    zl, zy = torch.zeros_like(dlast), torch.zeros_like(dy)
    a = torch.autograd.grad(ops.gated_scan(x, g, st)[0], (x, g, st), dy)
    b = torch.autograd.grad(ops.gated_scan(x, g, st), (x, g, st), (dy, zl))
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    a = torch.autograd.grad(ops.gated_scan(x, g, st)[1], (x, g, st), dlast)
    b = torch.autograd.grad(ops.gated_scan(x, g, st), (x, g, st), (zy, dlast))
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    a = torch.autograd.grad(ops.gated_scan(x.detach(), g, st.detach())[0], g,
                            dy.expand_as(dy))
    b = torch.autograd.grad(ops.gated_scan(x, g, st)[0], g, dy)
    assert torch.equal(a[0], b[0])
    # a gradient that is broadcast, as sum() gives
    a = torch.autograd.grad(ops.gated_scan(x, g)[0].sum(), x)
    b = torch.autograd.grad(ops.gated_scan(x, g)[0], x, torch.ones_like(dy))
    assert torch.equal(a[0], b[0])


@pytest.mark.gpu
def test_scan_gpu_is_differentiable_once():
    xg, st, _, dy, _ = make(2, 5, 6, torch.float32, "cuda", 3)
    xg.requires_grad_()
    g, = torch.autograd.grad(ops.gated_scan_xg(xg, st)[0], xg, dy,
                             create_graph=True)
    with pytest.raises(RuntimeError, match="once"):
        g.sum().backward()


@pytest.mark.gpu
def test_scan_gpu_repeats_bit_for_bit():
    xg, st, ln, dy, dlast = make(3, 700, 40, torch.bfloat16, "cuda", 9, True,
                                 "ragged")
    xg.requires_grad_(), st.requires_grad_()

    def once():
        o = ops.gated_scan_xg(xg, st, ln, True)
        return o + torch.autograd.grad(o, (xg, st), (dy, dlast))
    first = once()
    for _ in range(3):
        assert all(torch.equal(p, q) for p, q in zip(first, once()))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16,
                                   torch.float16])
@pytest.mark.parametrize("N,D", [(1, 1), (3, 5), (4, 64), (7, 1023),
                                 (130, 6)])
@pytest.mark.parametrize("inplace", [False, True])
def test_step_gpu(dtype, N, D, inplace):
    xg, st, _, dy, dlast = make(N, 1, D, dtype, "cuda", N + D)
    want = oracle(xg[..., :D], xg[..., D:], st, None, False, "relu", dy, dlast)
    K = (4 * float(xg[..., D:].abs().max()) + 32) * U
    amax = max(float(xg[..., :D].abs().max()), float(st.abs().max()))
    before = st.clone()
    y, new = ops.gated_step(xg[:, 0, :D], xg[:, 0, D:], st, act="relu",
                            inplace=inplace)
    assert (new is st) == inplace
    if not inplace:
        assert torch.equal(st, before)
    close(y, want[0][:, 0], K * amax, dtype)
    close(new, want[1], K * amax, torch.float32)


@pytest.mark.gpu
def test_step_gpu_captured():
    """An in-place step replayed from a graph advances the state each time,
    as eager steps on another stream do."""
    xg, st, _, _, _ = make(5, 6, 48, torch.bfloat16, "cuda", 11)
    y, last = ops.gated_scan_xg(xg, st)
    tok = xg[:, 0].clone()
    state = st.clone()
    ops.gated_step(tok[:, :48], tok[:, 48:], state.clone(), inplace=True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, _ = ops.gated_step(tok[:, :48], tok[:, 48:], state, inplace=True)
    side = torch.cuda.Stream()
    eager = st.clone()
    side.wait_stream(torch.cuda.current_stream())
    for t in range(6):
        tok.copy_(xg[:, t])
        graph.replay()
        with torch.cuda.stream(side):
            ye, eager = ops.gated_step(xg[:, t, :48], xg[:, t, 48:], eager)
        torch.cuda.synchronize()
        assert torch.equal(out, ye) and torch.equal(state, eager)
    close(state, last.double().cpu(), 6 * 80 * U * 4, torch.float32)


@pytest.mark.gpu
def test_gpu_two_streams_at_once():
    """Calls that overlap on two streams share nothing."""
    jobs = []
    for seed in (1, 2):
        xg, st, ln, dy, dl = make(2, 3000, 96, torch.bfloat16, "cuda", seed,
                                  True, "ragged")
        xg.requires_grad_(), st.requires_grad_()

        def once(a=xg, s=st, n=ln, d=(dy, dl)):
            o = ops.gated_scan_xg(a, s, n)
            return o + torch.autograd.grad(o, (a, s), d)
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
def test_scan_gpu_captured():
    """Forward and backward replayed from two graphs that interleave."""
    graphs = []
    for seed in (1, 2):
        xg, st, ln, dy, dlast = make(2, 900, 64, torch.bfloat16, "cuda", seed,
                                     True, "ragged")
        xg.requires_grad_(), st.requires_grad_()

        def once(a=xg, s=st, n=ln, d=(dy, dlast)):
            o = ops.gated_scan_xg(a, s, n)
            return [t.detach() for t in o] + list(
                torch.autograd.grad(o, (a, s), d))
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
        for graph, outs, _ in graphs:
            for o in outs:
                o.zero_()
        for graph, _, _ in graphs:
            graph.replay()
        for _, outs, once in graphs:
            assert all(torch.equal(p, q) for p, q in zip(outs, once()))


@pytest.mark.gpu
def test_scan_gpu_offsets_beyond_32_bits():
    """More than 2^31 elements: the last sequences come out as they do on
    their own."""
    B, T, D = 540_000, 64, 64
    part = torch.randn(1000, T, 2 * D, device="cuda").bfloat16()
    xg = part.repeat(B // 1000, 1, 1).requires_grad_()
    st = torch.randn(B, D, device="cuda")
    dy = torch.randn(1000, T, D, device="cuda").bfloat16()
    y, last = ops.gated_scan_xg(xg, st, reverse=True)
    g, = torch.autograd.grad(y, xg, dy.repeat(B // 1000, 1, 1))
    tail = xg.detach()[-3:].clone().requires_grad_()
    y2, last2 = ops.gated_scan_xg(tail, st[-3:], reverse=True)
    g2, = torch.autograd.grad(y2, tail, dy[-3:])
    assert torch.equal(y[-3:], y2) and torch.equal(last[-3:], last2)
    assert torch.equal(g[-3:], g2)


@pytest.mark.gpu
def test_step_gpu_offsets_beyond_32_bits():
    N, D = 2_200_000, 1000
    part = torch.randn(1000, 2 * D, device="cuda").bfloat16()
    xg = part.repeat(N // 1000, 1)
    st = torch.randn(1000, D, device="cuda").repeat(N // 1000, 1)
    y, new = ops.gated_step(xg[:, :D], xg[:, D:], st, act="relu")
    y2, new2 = ops.gated_step(part[:, :D], part[:, D:], st[:1000], act="relu")
    assert torch.equal(y[-1000:], y2) and torch.equal(new[-1000:], new2)


# ------------------------------------------------- bounds that a gate damps
# The limits above grow by a whole step's error with every step. These carry
# the error through the recurrence, element by element, as the gates damp it.
#
# In units of u = 2^-24 the sigmoid's exponential e has an error of at most
# 2 |g| + 3 (its argument's product and log2(e) are rounded, exp2 is good to
# one unit in the last place), so f, that is 1 / (1 + e) or e / (1 + e), has
# om (2 |g| + 3) + 4 and om has f (2 |g| + 3) + 4. A state is the sum of terms
# om x, each multiplied by the f of the steps behind it, however the steps are
# grouped: a step brings f's error, one rounding of a product and one of a sum
# to what is there; joining groups of steps brings at most 32 more to a term
# (5 in its tile, and folding tiles and chunks rounds less often than their
# steps would). With M the sum of the terms' absolute values:
#     E' = f (E + (ef + 2) M) + om |x| (eom + 2),   M' = f M + om |x|
# and a state is within (E + 32 M) u. The gradient's recurrence is the same
# one. Where relu's side is not certain within the state's bound, dy may be
# there or not, which is carried on as an absolute error. 2 % are added for
# products of errors (1e5 roundings are 0.6 %).

JOINS, MORE = 32, 1.02


def sharp(x, g, state, lens, reverse, act, dy, dlast, drop=0, states=None):
    """{name: (value, bound)} in float64, before the last rounding. Mistakes
    for the checks of the bounds: drop > 0 loses the gradient's carry every
    `drop` steps, states rounds the state at each 64th step to that type."""
    B, T, D = x.shape
    f, om = torch.sigmoid(g.double()), torch.sigmoid(-g.double())
    ee = 2 * g.double().abs() + 3
    ef, eom = om * ee + 4, f * ee + 4
    x, dy, dlast, f, om, ef, eom = (
        a.detach().double().cpu().numpy()
        for a in (x, dy, dlast, f, om, ef, eom))
    c0 = np.zeros((B, D)) if state is None \
        else state.detach().double().cpu().numpy()
    out = {k: (np.zeros(x.shape), np.zeros(x.shape))
           for k in ("y", "dx", "dg", "dg_plain")}
    out.update({k: (np.zeros(c0.shape), np.zeros(c0.shape))
                for k in ("last", "dstate")})

    def put(name, at, v, e):
        out[name][0][at], out[name][1][at] = v, e * MORE
    relu = act == "relu"
    for b in range(B):
        n = T if lens is None else min(max(int(lens[b]), 0), T)
        order = list(range(n))[::-1] if reverse else list(range(n))
        c, M, E = c0[b], abs(c0[b]), np.zeros(D)
        prev, side = [], []
        for i, t in enumerate(order):
            if states is not None and i % 64 == 0:
                c = torch.from_numpy(c).to(states).double().numpy()
            prev.append((c, (E + JOINS * M) * U if i else E))
            F, a = f[b, t], om[b, t] * x[b, t]
            c = F * c + a
            E = F * (E + (ef[b, t] + 2) * M) + abs(a) * (eom[b, t] + 2)
            M = F * M + abs(a)
            bound = (E + JOINS * M) * U
            on = c > 0 if relu else np.ones(D)
            side.append((on, abs(c) <= bound * MORE if relu else 0 * c))
            put("y", (b, t), c * on, bound)
        put("last", b, c, (E + JOINS * M) * U if n else E)
        mu, K = dlast[b], abs(dlast[b])
        Em, Am = np.zeros(D), np.zeros(D)
        for i in range(n - 1, -1, -1):
            t = order[i]
            if drop and i % drop == drop - 1:
                mu = 0 * mu
            (on, maybe), (p, pe) = side[i], prev[i]
            lam, L = on * dy[b, t] + mu, abs(dy[b, t]) + K
            El, Al = Em + L, Am + maybe * abs(dy[b, t])
            bl, al = (El + JOINS * L) * U + Al, abs(lam)
            F, O, rf, ro = f[b, t], om[b, t], ef[b, t], eom[b, t]
            put("dx", (b, t), O * lam, O * (bl + al * (ro + 1) * U))
            w = p - x[b, t]
            we = pe + U * abs(w)
            e = F * O * (bl * (abs(w) + we) + al * we
                         + al * abs(w) * (rf + ro + 4) * U)
            put("dg", (b, t), F * O * w * lam, e)
            # off the GPU the sigmoids are differentiated one by one: 1 - f
            # and 1 - om are off by what f and om are and a rounding, and
            # neither cancels with the other side's
            put("dg_plain", (b, t), F * O * w * lam, e + U * al * (
                abs(p) * F * (rf * F + 1 + 4 * O)
                + abs(x[b, t]) * O * (ro * O + 1 + 4 * F)))
            mu, K = F * lam, F * L
            Em, Am = F * (El + (rf + 1) * L), F * Al
        put("dstate", b, mu, (Em + JOINS * K) * U + Am if n else Em)
    return {k: tuple(torch.from_numpy(a) for a in v) for k, v in out.items()}


def limits(want, dtype):
    """How far a result of this type may be from the value."""
    half = torch.finfo(dtype).eps / 2
    v, e = want
    return e + half * (v.abs() + e) + torch.finfo(dtype).tiny * half


def within(name, got, want, dtype):
    assert got.dtype == dtype and got.shape == want[0].shape, name
    err = (got.detach().double().cpu() - want[0]).abs()
    lim = limits(want, dtype)
    assert bool((err <= lim).all()), \
        f"{name}: {float((err / lim.clamp_min(1e-300)).max())} of the limit"


SHARP_CASES = [
    dict(B=2, T=1, D=3, dtype=torch.float32),
    dict(B=3, T=17, D=30, dtype=torch.float16, lens="ragged"),
    dict(B=2, T=65, D=257, dtype=torch.float32, act="relu"),
    dict(B=4, T=130, D=130, dtype=torch.bfloat16, lens="ragged", reverse=True,
         act="relu", layout="fused"),
    dict(B=1, T=1000, D=70, dtype=torch.float32, reverse=True),
    dict(B=1, T=1025, D=256, dtype=torch.bfloat16, layout="fused"),
    dict(B=1, T=1025, D=256, dtype=torch.bfloat16, layout="fused",
         act="relu"),
    dict(B=7, T=700, D=40, dtype=torch.float32, lens="ragged", act="relu"),
    dict(B=7, T=700, D=41, dtype=torch.bfloat16, lens="ragged", reverse=True),
    dict(B=3, T=1500, D=66, dtype=torch.float16, act="relu", layout="fused",
         state=False),
    dict(B=1, T=4200, D=1, dtype=torch.float16),
    dict(B=1, T=4200, D=33, dtype=torch.float32, act="relu", reverse=True),
    # not split: many blocks
    dict(B=40, T=150, D=330, dtype=torch.float32, act="relu", lens="ragged"),
]


def sharp_case(dev, B, T, D, dtype, lens=None, reverse=False, act="none",
               state=True, layout="split"):
    xg, st, ln, dy, dlast = make(B, T, D, dtype, dev, 21, state, lens)
    want = sharp(xg[..., :D], xg[..., D:], st, ln, reverse, act, dy, dlast)
    kw = dict(state=st, lens=ln, reverse=reverse, act=act)
    leaves = [] if st is None else [st.requires_grad_()]
    if layout == "fused":
        leaves = [xg.requires_grad_()] + leaves
        y, last = ops.gated_scan_xg(xg, **kw)
    else:
        x, g = (a.contiguous().requires_grad_()
                for a in (xg[..., :D], xg[..., D:]))
        leaves = [x, g] + leaves
        y, last = ops.gated_scan(x, g, **kw)
    grads = torch.autograd.grad((y, last), leaves, (dy, dlast))
    if layout == "fused":
        grads = (grads[0][..., :D], grads[0][..., D:]) + grads[1:]
    within("y", y, want["y"], dtype)
    within("last", last, want["last"], torch.float32)
    within("dx", grads[0], want["dx"], dtype)
    within("dg", grads[1], want["dg" if dev == "cuda" else "dg_plain"], dtype)
    if st is not None:
        within("dstate", grads[2], want["dstate"], torch.float32)


@pytest.mark.parametrize("case", SHARP_CASES)
def test_scan_plain_within_damped_bounds(case):
    sharp_case("cpu", **{**case, "B": min(case["B"], 4)})


@pytest.mark.gpu
@pytest.mark.parametrize("case", SHARP_CASES)
def test_scan_gpu_within_damped_bounds(case):
    sharp_case("cuda", **case)


@pytest.mark.parametrize("T,D", [(1000, 70), (1025, 64), (4200, 16)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16,
                                   torch.float16])
def test_damped_bounds_reject_mistakes(T, D, dtype):
    """Planted in the oracle: no gate gradient, a carry lost every 64 steps or
    every 2048, tile states kept in 16 bits."""
    xg, st, _, dy, dlast = make(1, T, D, dtype, "cpu", 22)
    args = (xg[..., :D], xg[..., D:], st, None, False, "none", dy, dlast)
    right = sharp(*args)
    out = lambda name, v, t: ((v - right[name][0]).abs()
                              > limits(right[name], t)).double().mean()
    assert out("dg", torch.zeros_like(right["dg"][0]), dtype) > 0.9
    for drop, share in ((64, 64), (2048, 2048)):
        if T > drop:
            lost = sharp(*args, drop=drop)
            # the step before each loss sees it at once
            for k in ("dx", "dg"):
                assert out(k, lost[k][0], dtype) > 0.5 / share
    few = sharp(*args, states=torch.bfloat16)
    if dtype == torch.float32:
        assert out("y", few["y"][0], dtype) > 0.02
        assert out("dg", few["dg"][0], dtype) > 0.005
    if T % 64 == 1:     # 40 steps behind its mistake a state has lost it
        assert out("last", few["last"][0], torch.float32) > 0.1


def test_every_kernel_is_reached():
    """(channels a lane, waves, chunks' maps): one wave has no chunks."""
    import re
    from marian_amd.ops import _load
    path = _load.extension_path()
    if path is None:
        pytest.skip("the extension is not built")
    with open(path, "rb") as f:
        names = set(re.findall(rb"scan_(fwd|bwd)_kernelI(?:f|DF16b|DF16_)"
                               rb"Li(\d+)ELi(\d+)ELb([01])E", f.read()))
    held = {tuple(map(int, n[1:])) for n in names}
    assert {n[0] for n in names} == {b"fwd", b"bwd"}
    assert held == {(v, 4, m) for v in (1, 2) for m in (0, 1)} \
        | {(v, 1, 0) for v in (1, 2)}
