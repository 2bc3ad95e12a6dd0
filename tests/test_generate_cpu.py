"""A packed stack's walk, what needs no GPU: where the buffers of ``generate`` and
the weights of ``attach_packed`` are put.  The operators' kernels are replaced
by torch."""

import contextlib
import types

import pytest
import torch

from jax_gptq_b200 import packing, pipeline

CFG = pipeline.BlockConfig(hidden=32, intermediate=48, heads=2, kv_heads=1)


def _turn(q, k, positions, plan, out=None, transpose=False):
    out[0].copy_(q)
    out[1].copy_(k)
    return out


def _choose(logits, u, *settings):
    return pipeline.sampling.Sampled(logits.argmax(-1), torch.zeros(logits.shape[0]))


def _model():
    """A TinyLM that stays on the CPU."""
    lm = pipeline.TinyLM.__new__(pipeline.TinyLM)
    torch.nn.Module.__init__(lm)
    lm.embed = torch.nn.Embedding(20, CFG.hidden)
    lm.blocks = torch.nn.ModuleList([pipeline.DecoderBlock(CFG) for _ in range(2)])
    lm.norm = pipeline.RMSNorm(CFG.hidden, CFG.eps)
    lm.lm_head = torch.nn.Linear(CFG.hidden, 20, bias=False)
    return lm


def test_generate_keeps_to_the_device_of_its_prompts(monkeypatch):
    entered = []

    @contextlib.contextmanager
    def device_of(t):
        entered.append(t)
        yield

    monkeypatch.setattr(torch.cuda, "device_of", device_of)
    monkeypatch.setattr(pipeline.rotary, "rotary_plan",
                        lambda *a, **k: types.SimpleNamespace(made_inside=len(entered)))
    monkeypatch.setattr(pipeline.rotary, "apply_rotary", _turn)
    monkeypatch.setattr(pipeline.sampling, "sample_tokens", _choose)
    monkeypatch.setattr(pipeline._lib, "check_device", lambda *a: None)
    ids = torch.tensor([[1, 2, 3], [4, 5, 6]])
    got = _model().generate(ids, torch.rand(2, 4))
    assert len(entered) == 1 and entered[0] is ids
    assert got.tokens.shape == (2, 4) and got.tokens.device == ids.device
    assert got.logprobs.device == ids.device


def test_attach_packed_lays_out_on_the_device_of_the_block(monkeypatch, tmp_path):
    where = []

    @contextlib.contextmanager
    def device_of(t):
        where.append(t)
        yield
        where.pop()

    class Laid(torch.nn.Module):
        def __init__(self, p):
            super().__init__()
            assert p.qweight.device.type == "cpu"  # from here to that device, not by another
            self.out_features, self.in_features, self.at = p.m, p.n, where[-1]

    monkeypatch.setattr(torch.cuda, "device_of", device_of)
    monkeypatch.setattr(pipeline.linear, "QuantLinear", Laid)
    blocks = [pipeline.DecoderBlock(CFG) for _ in range(2)]
    for i, blk in enumerate(blocks):
        layer = {}
        for n in pipeline.GROUPS:
            m, k = getattr(blk, n).weight.shape
            order = torch.arange(k, dtype=torch.int32)
            layer[n] = packing.PackedLinear(torch.zeros((m, k // 8), dtype=torch.int32),
                                            torch.ones((m, 1)), torch.zeros((m, 1)), order * 0,
                                            order, 4, k, False, k)
        packing.save_layer(str(tmp_path / f"layer{i}.pt"), layer)
    pipeline.attach_packed(blocks, str(tmp_path))
    assert not where
    for blk in blocks:
        assert all(getattr(blk, n).at is blk.input_layernorm.weight for n in pipeline.GROUPS)


def test_generate_refuses_shapes():
    lm = _model()
    for ids, u in ((torch.zeros(3, dtype=torch.int64), torch.rand(1, 2)),
                   (torch.zeros((2, 0), dtype=torch.int64), torch.rand(2, 2)),
                   (torch.zeros((2, 3), dtype=torch.int64), torch.rand(3, 2))):
        with pytest.raises(ValueError, match="ids must be"):
            lm.generate(ids, u)
