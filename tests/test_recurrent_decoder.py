"""The recurrent decoder layer (--transformer-decoder-autoreg rnn) and the
fused pre/postprocess ops (r, g, h, --transformer-residual-scale): the three
operators of a block as the models run them together."""
import numpy as np
import pytest
import torch

from marian_amd import ops
from marian_amd.common.config_parser import ConfigParser, MODE_TRAINING
from marian_amd.common.options import Options
from marian_amd.data.batch import CorpusBatch, SubBatch
from marian_amd.data.synthetic import synthetic_batch
from marian_amd.models.layers import PrePostProcessor, SSRU, join_blocks
from marian_amd.models.model_factory import create_model
from marian_amd.translator.beam_search import BeamSearch, ModelScorer

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
# pre and postprocess strings of a layer
STYLES = [("", "dan", 1.0), ("n", "da", 1.0), ("r", "da", 1.0),
          ("n", "dnga", 0.5), ("r", "drga", 1.0), ("r", "dh", 1.0),
          ("", "dhn", 0.7), ("n", "dra", 1.0)]


def options(pre="n", post="dnga", alpha=1.0, **kw):
    base = {
        "type": "transformer", "dim-emb": 32, "enc-depth": 2, "dec-depth": 2,
        "transformer-heads": 4, "transformer-dim-ffn": 64,
        "transformer-preprocess": pre, "transformer-postprocess": post,
        "transformer-postprocess-emb": "d",
        "transformer-postprocess-top": "n" if pre else "",
        "transformer-residual-scale": alpha,
        "transformer-decoder-autoreg": "rnn", "dec-cell": "ssru",
        "transformer-ffn-activation": "relu", "transformer-dropout": 0.0,
        "dim-vocabs": [37, 37], "tied-embeddings-all": True,
        "transformer-train-position-embeddings": False,
        "transformer-decoder-dim-ffn": 0,
    }
    base.update(kw)
    return Options(base)




def shake(m, seed=1):
    """Parameters that start as 0 or 1 take values of their own."""
    gen = torch.Generator().manual_seed(seed)
    with torch.no_grad():
        for n, p in m.named_parameters():
            if p.dim() == 1:
                p.add_(0.2 * torch.randn(p.shape, generator=gen).to(p))
    return m


def by_hand(post, x, residual):
    """A postprocess string written out in plain torch, op by op."""
    for op in post.ops_str:
        if op == "a":
            x = x + post.res_scale * residual
        elif op == "h":
            k = torch.sigmoid(residual @ post.highway.W + post.highway.b)
            x = k * x + (1 - k) * post.res_scale * residual
        elif op == "g":
            x = x * post.gate
        elif op == "r":
            x = x / (x.square().mean(-1, keepdim=True) + 1e-9).sqrt() \
                * post.rms.scale
        elif op == "n":
            mu = x.mean(-1, keepdim=True)
            sd = (x.var(-1, unbiased=False, keepdim=True) + 1e-9).sqrt()
            x = (x - mu) / sd * post.ln.scale + post.ln.bias
    return x


# float32 against float32: both sides are within some 100 roundings of values
# below 2^5 through at most two norms
TOL = 2.0 ** -12


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("post_s", ["dga", "dnga", "drgan", "dh", "dhn", "dra",
                                    "da", "dan", "gd", "nargh", "nan", "rar"])
@pytest.mark.parametrize("pre_s", ["n", "r", ""])
def test_strings_and_their_gradients(dev, post_s, pre_s):
    torch.manual_seed(3)
    post = shake(PrePostProcessor(post_s, 24, 0.0, 0.5)).to(dev)
    pre = shake(PrePostProcessor(pre_s, 24, 0.0)).to(dev)
    x, r, dy, dh = (torch.randn(3, 5, 24).to(dev) for _ in range(4))
    leaves = [x.requires_grad_(), r.requires_grad_()] \
        + list(post.parameters()) + list(pre.parameters())

    def grads(y, h):
        return torch.autograd.grad((y, h), leaves, (dy, dh),
                                   allow_unused=True)
    got = join_blocks(post, pre, x, r)
    y = by_hand(post, x, r)
    want = (y, by_hand(pre, y, None))
    for a, b in zip(got + grads(*got), want + grads(*want)):
        if a is None or b is None:      # unused, or used with factor 0
            assert not any(t is not None and bool((t != 0).any())
                           for t in (a, b))
            continue
        assert torch.allclose(a, b, rtol=TOL, atol=TOL * float(
            b.detach().abs().max().clamp_min(1)))


@pytest.mark.parametrize("pre,post,alpha", STYLES)
def test_teacher_forcing_equals_steps(pre, post, alpha):
    torch.manual_seed(7)
    m = shake(create_model(options(pre, post, alpha))).eval()
    b = synthetic_batch(3, 5, 9, 37)
    with torch.no_grad():
        enc = m.encode(b.source.indices, b.source.mask)
        full = m.decode_train(b.target.indices, b.target.mask, enc,
                              b.source.mask)
        cache, outs = {"max_len": 20}, []
        for t in range(9):
            prev = b.target.indices[:, t - 1] if t else \
                torch.zeros(3, dtype=torch.long)
            outs.append(m.decode_step(prev, enc, b.source.mask, cache, t))
    assert cache["l0_self_cell"].dtype == torch.float32
    assert torch.allclose(full, torch.stack(outs, 1), atol=1e-4)


@pytest.mark.parametrize("pre,post,alpha", STYLES)
def test_parameters_train_and_round_trip(pre, post, alpha):
    torch.manual_seed(8)
    m = shake(create_model(options(pre, post, alpha)))
    b = synthetic_batch(2, 5, 6, 37)
    m(b).float().pow(2).mean().backward()
    for n, p in m.named_parameters():
        assert p.grad is not None and torch.isfinite(p.grad).all(), n
    items = m.marian_items()
    assert sum(v.size for v in items.values()) \
        == sum(p.numel() for p in m.parameters())
    for k in ("decoder_l1_rnn_W", "decoder_l1_rnn_Wf", "decoder_l1_rnn_bf"):
        assert k in items
    other = create_model(options(pre, post, alpha))
    other.load_marian_items(items)
    assert torch.equal(m(b), other(b))
    cfg = m.model_config()
    assert cfg["dec-cell"] == "ssru"
    assert cfg.get("transformer-residual-scale", 1.0) == alpha


def test_language_model():
    torch.manual_seed(9)
    m = create_model(options("r", "dga", type="lm-transformer"))
    b = synthetic_batch(2, 4, 7, 37)
    logits = m(b)
    assert logits.shape == (2, 7, 37)
    logits.float().pow(2).mean().backward()
    assert m.decoder[0].self_attn.W_xg.grad is not None


def test_refusals():
    with pytest.raises(ValueError, match="dec-cell"):
        create_model(options(**{"dec-cell": "gru"}))
    for key, s in (("preprocess", "g"), ("postprocess-top", "h"),
                   ("postprocess-emb", "r")):
        with pytest.raises(ValueError, match=key):
            create_model(options(**{"transformer-" + key: s}))
    with pytest.raises(ValueError, match="Unknown"):
        PrePostProcessor("rx", 8, 0.0)(torch.zeros(2, 8))


def test_options_are_parsed():
    o = ConfigParser(MODE_TRAINING).parse_options([
        "--type", "transformer", "--transformer-decoder-autoreg", "rnn",
        "--dec-cell", "ssru", "--transformer-postprocess", "drga",
        "--transformer-residual-scale", "0.5", "--train-sets", "a", "b",
        "--vocabs", "a.yml", "b.yml", "--model", "m.npz"])
    assert o.get("transformer-decoder-autoreg") == "rnn"
    assert o.get("transformer-residual-scale") == 0.5


def sentences():
    sub = SubBatch.from_sentences([[5, 6, 7, 8, 0], [9, 10, 0], [4, 0]],
                                  pad_id=0)
    return CorpusBatch([sub], sentence_ids=[0, 1, 2])


def test_beam_search():
    torch.manual_seed(10)
    m = shake(create_model(options()))
    res = BeamSearch([ModelScorer(m, torch.device("cpu"))], beam_size=3,
                     normalize=0.6, max_length=10).search(
                         sentences(), torch.device("cpu"))
    assert len(res) == 3 and all(r.best.tokens for r in res)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("params", ["own", "float32"])
def test_projection_is_rounded_once(dev, dtype, params):
    """Scoring and decoding take the projection that training takes: the
    gate's bias is added before the only rounding. An error of the 32-bit sum
    over d products is below d + 2 units of the sum of absolute values."""
    torch.manual_seed(14)
    cell = SSRU(64)
    with torch.no_grad():
        cell.bf.uniform_(-3, 3)
    if params == "own":
        cell = cell.to(dtype)
    cell = cell.to(dev)
    x = torch.randn(5, 7, 64).to(dtype).to(dev)
    with_grad = cell.project(x).detach()
    with torch.no_grad():
        got = cell.project(x)
    assert got.dtype == dtype and torch.equal(got, with_grad)
    W, bf = (p.detach().to(dtype).double().cpu() for p in (cell.W_xg, cell.bf))
    b = torch.cat([torch.zeros(64, dtype=torch.float64), bf])
    xd = x.double().cpu()
    want, size = xd @ W + b, xd.abs() @ W.abs() + b.abs()
    lim = 66 * 2.0 ** -24 * size
    half = torch.finfo(dtype).eps / 2 * (1 + 2.0 ** -7)
    assert bool(((got.double().cpu() - want).abs()
                 <= lim + half * (want.abs() + lim)).all())


def test_projection_with_int8_weights():
    """Weights are packed once, and the bias is there."""
    from marian_amd.ops import cpu_int8
    torch.manual_seed(15)
    cell, x = SSRU(64), torch.randn(9, 64)
    with torch.no_grad():
        cell.bf.uniform_(-3, 3)
        want = cell.project(x)
        cpu_int8.enable_int8(True)
        try:
            for _ in range(3):
                got = cell.project(x)
                assert len(cpu_int8._qcache) == 1
        finally:
            cpu_int8.enable_int8(False)
    assert float((got - want).abs().max()) < 0.1
    assert not torch.equal(got, want)


def test_export(tmp_path):
    """A recurrent decoder is refused before a file is written; the other
    decoders export with the fused pre/postprocess ops."""
    from marian_amd.translator.onnx_export import export_onnx
    with pytest.raises(ValueError, match="recurrent"):
        export_onnx(create_model(options("n", "da")), str(tmp_path / "m"), 37)
    assert not list(tmp_path.iterdir())
    for pre, post in (("r", "drga"), ("n", "dh"), ("", "dhn")):
        m = create_model(options(pre, post, 0.5, **{
            "transformer-decoder-autoreg": "self-attention"}))
        for f in export_onnx(m, str(tmp_path / "m"), 37):
            assert (tmp_path / f).stat().st_size > 0


# ------------------------------------------------------------------ on the GPU

@pytest.mark.gpu
@pytest.mark.parametrize("pre,post,alpha", STYLES)
def test_gpu_model_matches_cpu(pre, post, alpha):
    """One model in float32 on both devices: logits and all gradients."""
    torch.manual_seed(11)
    m = shake(create_model(options(pre, post, alpha)))
    b = synthetic_batch(3, 6, 70, 37)
    out = []
    for dev in ("cpu", "cuda"):
        m = m.to(dev)
        m.zero_grad(set_to_none=True)
        bd = CorpusBatch([s.to(torch.device(dev)) for s in
                          (b.source, b.target)])
        logits = m(bd)
        logits.float().pow(2).mean().backward()
        out.append([logits.detach().cpu()]
                   + [p.grad.detach().cpu().clone() for p in m.parameters()])
    for a, c in zip(*out):
        assert torch.allclose(a, c, rtol=1e-3,
                              atol=1e-3 * float(a.abs().max()))


@pytest.mark.gpu
def test_gpu_bf16_training_step():
    """Scan, step and join under the graph group's bf16 update."""
    from marian_amd.training.graph_group import SyncGraphGroup
    o = options("r", "drga", 0.5, **{
        "dim-emb": 256, "transformer-dim-ffn": 512, "dim-vocabs": [64, 64],
        "precision": ["bfloat16", "float32"], "cost-type": "ce-mean-words",
        "label-smoothing": 0.1, "optimizer": "adam", "learn-rate": 3e-4,
        "clip-norm": 0.0})
    torch.manual_seed(7)
    m = create_model(o)
    gg = SyncGraphGroup(o, m, torch.device("cuda", 0))
    gg.set_lr(3e-4)
    batch = synthetic_batch(8, 16, 80, 64, device=torch.device("cuda", 0))
    before = m.decoder[0].self_attn.W_xg.detach().clone()
    lv = gg.update(batch)
    torch.cuda.synchronize()
    assert 0 < float(lv.ce_sum) / max(1, lv.label_count) < 20
    assert not torch.equal(before, m.decoder[0].self_attn.W_xg)


@pytest.mark.gpu
def test_gpu_graphed_decode_matches_eager():
    """The captured beam search of a recurrent decoder, over batches of one
    shape that follow each other, against the eager one."""
    torch.manual_seed(12)
    dev = torch.device("cuda", 0)
    o = options("r", "drga", **{"dim-emb": 256, "transformer-dim-ffn": 512,
                                "dim-vocabs": [64, 64]})
    m = shake(create_model(o)).to(dev)
    m.set_compute_dtype(torch.bfloat16)
    for p in m.parameters():
        p.data = p.data.bfloat16()
    bs = BeamSearch([ModelScorer(m, dev)], beam_size=3, normalize=0.6,
                    max_length=9)
    for rep in range(3):
        got = bs.search(sentences(), dev)
        assert len(bs._graph_cache) == 1
        eager = BeamSearch([ModelScorer(m, dev)], beam_size=3, normalize=0.6,
                           max_length=9)
        eager._try_graphed = lambda *a, **k: None
        want = eager.search(sentences(), dev)
        for a, b in zip(got, want):
            assert a.best.tokens == b.best.tokens
            assert abs(a.best.score - b.best.score) < 0.05 * abs(b.best.score)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gpu_block_prefix_then_steps(dtype):
    """Serving: a prefix through the scan, then single steps from its state,
    gives what one scan over all of it gives; each followed by the join."""
    torch.manual_seed(13)
    B, T, P, D = 3, 150, 140, 72
    xg = torch.randn(B, T, 2 * D, device="cuda").to(dtype)
    res = torch.randn(B, T, D, device="cuda").to(dtype)
    w = (1 + 0.1 * torch.randn(D, device="cuda")).to(dtype)

    def join(y, r):
        return ops.block_norm(y, r, post_scale=w, pre_scale=w, norm="rms")
    y, last = ops.gated_scan_xg(xg, act="relu")
    whole = join(y, res)
    y1, state = ops.gated_scan_xg(xg[:, :P], act="relu")
    assert torch.equal(y1, y[:, :P])
    # a state is good to some 100 roundings per step (see the scan's tests);
    # a different grouping may round y, and then s and h, the other way
    lim = T * 100 * 2.0 ** -24
    step = 2 * torch.finfo(dtype).eps
    for t in range(P, T):
        o, state = ops.gated_step(xg[:, t, :D], xg[:, t, D:], state,
                                  act="relu", inplace=True)
        assert torch.allclose(o.float(), y[:, t].float(), rtol=step, atol=lim)
        for a, b in zip(join(y[:, t], res[:, t]), whole):
            assert torch.equal(a, b[:, t])
    assert torch.allclose(state, last, rtol=0, atol=lim)
