"""ONNX export for encoder-decoder models
(ref: src/onnx/expression_graph_onnx_exporter.{h,cpp} — the reference's
`marian-conv --export-as onnx` with the same scope: encoder + decoder
pieces for an EXTERNAL beam-search driver; its coverage was partial too).

MI355X-repo realization: the torch TorchScript ONNX exporter over the
CPU composite paths of the model (attention/LN/CE all have pure-torch
composites, so the trace contains only standard ONNX ops). The offline
image has protobuf but not the `onnx` python package; the exporter's one
hard `import onnx` lives in `_add_onnxscript_fn`, which only injects
CUSTOM onnxscript functions — none exist in these graphs — so when the
package is missing we patch that step to the identity and write the
already-complete ModelProto bytes.

Exports two graphs (the reference splits the model the same way):
  <prefix>.encoder.onnx  src_ids[B,Ts], src_mask[B,Ts] -> enc[B,Ts,d]
  <prefix>.decoder.onnx  trg_prefix[B,Tt], enc[B,Ts,d], src_mask[B,Ts]
                         -> logits[B,V] for the NEXT token (prefix
                         re-run per step; no KV-cache I/O, like the
                         reference's exported decoder)
"""
from __future__ import annotations

import warnings

import torch


def _patch_missing_onnx() -> bool:
    try:
        import onnx  # noqa: F401
        return False
    except ImportError:
        from torch.onnx._internal.torchscript_exporter import (
            onnx_proto_utils)
        onnx_proto_utils._add_onnxscript_fn = \
            lambda model_bytes, custom_opsets: model_bytes
        return True


class _Encoder(torch.nn.Module):
    def __init__(self, model):
        super().__init__()
        self.model = model

    def forward(self, src_ids, src_mask):
        return self.model.encode(src_ids, src_mask)


class _DecoderStep(torch.nn.Module):
    def __init__(self, model):
        super().__init__()
        self.model = model

    def forward(self, trg_prefix, enc, src_mask):
        trg_mask = torch.ones_like(trg_prefix, dtype=src_mask.dtype)
        logits = self.model.decode_train(trg_prefix, trg_mask, enc,
                                         src_mask)
        return logits[:, -1]


def export_onnx(model, prefix: str, vocab_size: int) -> list:
    """Write <prefix>.encoder.onnx / <prefix>.decoder.onnx; returns the
    file list. Model must be a TransformerModel on CPU in eval mode."""
    if model.opt.get("transformer-decoder-autoreg", "") == "rnn":
        # a trace holds the number of steps that it has seen
        raise ValueError("ONNX export does not take a recurrent decoder "
                         "(--transformer-decoder-autoreg rnn)")
    model = model.float().cpu().eval()
    _patch_missing_onnx()
    B, Ts, Tt = 2, 5, 3
    src_ids = torch.randint(2, vocab_size, (B, Ts))
    src_mask = torch.ones(B, Ts)
    trg_prefix = torch.randint(2, vocab_size, (B, Tt))
    files = []
    with warnings.catch_warnings(), torch.no_grad():
        warnings.simplefilter("ignore")
        enc_path = prefix + ".encoder.onnx"
        torch.onnx.export(
            _Encoder(model), (src_ids, src_mask), enc_path,
            input_names=["src_ids", "src_mask"], output_names=["enc"],
            dynamic_axes={"src_ids": {0: "B", 1: "Ts"},
                          "src_mask": {0: "B", 1: "Ts"},
                          "enc": {0: "B", 1: "Ts"}},
            dynamo=False)
        files.append(enc_path)
        enc = model.encode(src_ids, src_mask)
        dec_path = prefix + ".decoder.onnx"
        torch.onnx.export(
            _DecoderStep(model), (trg_prefix, enc, src_mask), dec_path,
            input_names=["trg_prefix", "enc", "src_mask"],
            output_names=["logits"],
            dynamic_axes={"trg_prefix": {0: "B", 1: "Tt"},
                          "enc": {0: "B", 1: "Ts"},
                          "src_mask": {0: "B", 1: "Ts"},
                          "logits": {0: "B"}},
            dynamo=False)
        files.append(dec_path)
    return files
