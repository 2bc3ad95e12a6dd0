"""A quantized stack run from its packed layer files: the same model as with
dequantized weights, in one pass and decoded step by step with the cache.

All in float32, so that only the order of additions and the angles differ:
the cached path takes its angles from 64-bit turns, ``forward`` from float32
(positions below 64: off by at most 64 * 2^-23 = 2^-17).  A relative
disturbance of 2^-16 of every intermediate value through two blocks of sums
over at most 640 terms with gain of order 1 stays below 2^-8 of the largest
logit; equality to 2^-8 tells the paths apart from a wrong position, mask or
weight, which move logits by their own size.
"""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

from jax_gptq_b200 import eval as E
from jax_gptq_b200 import linear, pipeline
from jax_gptq_b200.config import QuantConfig

CFG = pipeline.BlockConfig(hidden=256, intermediate=640, heads=4, kv_heads=2)
VOCAB = 500
TOL = 2.0 ** -8


@pytest.fixture(scope="module")
def models(tmp_path_factory):
    """(model with dequantized weights, the same on packed weights), float32."""
    path = str(tmp_path_factory.mktemp("layers"))
    lms = [pipeline.TinyLM(pipeline.synth_stack(2, CFG, seed=1, dtype=torch.float32), VOCAB, CFG,
                           seed=11, dtype=torch.float32) for _ in range(2)]
    rng = np.random.default_rng(0)
    calib = [lms[0].hidden(torch.from_numpy(rng.integers(0, VOCAB, (4, 64))).cuda())
             for _ in range(2)]
    cfg = QuantConfig(w_bits=4, group_size=128, ordering_mode="diag_h", semantics="intended")
    pipeline.quantize_stack(list(lms[0].blocks), calib, cfg, checkpoint_dir=path)
    pipeline.attach_packed(list(lms[1].blocks), path)
    assert all(isinstance(getattr(b, n), linear.QuantLinear) for b in lms[1].blocks
               for n in pipeline.GROUPS)
    return (*lms, path)


def _ids(seed, b, t):
    return torch.from_numpy(np.random.default_rng(seed).integers(0, VOCAB, (b, t))).cuda()


@torch.no_grad()
def test_packed_model_is_the_dequantized_model(models):
    floats, packed, _ = models
    ids = _ids(1, 3, 50)
    a, b = floats(ids), packed(ids)
    assert float((a - b).abs().max()) <= TOL * float(a.abs().max())
    windows, labels = [ids.cpu().numpy()], [ids.cpu().numpy()]
    pa = E.evaluate_perplexity(floats, windows, labels)
    pb = E.evaluate_perplexity(packed, windows, labels)
    assert abs(np.log(pa) - np.log(pb)) <= 2 * TOL * float(a.abs().max())


@torch.no_grad()
def test_decoding_agrees_with_one_pass(models):
    _, packed, _ = models
    for t, new in ((1, 6), (7, 12)):
        ids = _ids(2, 4, t)
        u = torch.rand((4, new), device="cuda", generator=torch.Generator("cuda").manual_seed(3))
        got = packed.generate(ids, u, temperature=0.0)
        full = torch.cat([ids, got.tokens], dim=1)
        logits = packed(full)[:, t - 1:-1]
        top = logits.max(-1).values
        chosen = logits.gather(-1, got.tokens[..., None])[..., 0]
        assert float((top - chosen).max()) <= 2 * TOL * float(logits.abs().max())
        assert torch.equal(got.logprobs, torch.zeros_like(got.logprobs))


@torch.no_grad()
def test_sampled_tokens_are_of_the_filtered_distribution(models):
    _, packed, _ = models
    ids = _ids(4, 5, 9)
    u = torch.rand((5, 10), device="cuda", generator=torch.Generator("cuda").manual_seed(5))
    got = packed.generate(ids, u, temperature=0.9, top_k=8, top_p=0.95)
    again = packed.generate(ids, u, temperature=0.9, top_k=8, top_p=0.95)
    assert torch.equal(got.tokens, again.tokens) and torch.equal(got.logprobs, again.logprobs)
    assert int(got.tokens.min()) >= 0 and int(got.tokens.max()) < VOCAB
    assert bool((got.logprobs <= 0).all())
    logits = packed(torch.cat([ids, got.tokens], dim=1))[:, 8:-1]
    eighth = logits.topk(8, -1).values[..., -1]
    chosen = logits.gather(-1, got.tokens[..., None])[..., 0]
    assert float((eighth - chosen).max()) <= 2 * TOL * float(logits.abs().max())
    empty = packed.generate(ids, u[:, :0])
    assert empty.tokens.shape == (5, 0)


@torch.no_grad()
def test_bf16_model_runs(models):
    path = models[2]
    lm = pipeline.TinyLM(pipeline.synth_stack(2, CFG, seed=1), VOCAB, CFG, seed=11)
    pipeline.attach_packed(list(lm.blocks), path)
    u = torch.rand((2, 5), device="cuda")
    got = lm.generate(_ids(6, 2, 4), u, top_p=0.9)
    assert got.tokens.shape == (2, 5)
    # a model whose logits are all NaN: no token, and no fault on the next step
    with torch.no_grad():
        lm.lm_head.weight.fill_(float("nan"))
    got = lm.generate(_ids(6, 2, 4), u)
    assert bool((got.tokens == -1).all())


def test_refusals(models, tmp_path):
    _, packed, path = models
    with pytest.raises(ValueError, match="ids must be"):
        packed.generate(_ids(1, 2, 3), torch.rand((3, 4), device="cuda"))
    small = pipeline.BlockConfig(hidden=128, intermediate=640, heads=4, kv_heads=2)
    with pytest.raises(ValueError, match="the block's is"):
        pipeline.attach_packed(pipeline.synth_stack(1, small), path)
    blk = pipeline.synth_stack(1, CFG)[0]
    cache = pipeline.KVCache.empty(CFG, 1, 4, torch.bfloat16)
    from jax_gptq_b200 import rotary
    with pytest.raises(ValueError, match="4 positions"):
        blk.decode(torch.zeros((1, 5, 256), dtype=torch.bfloat16, device="cuda"), cache,
                   rotary.rotary_plan(64))


def test_a_bad_file_leaves_every_block_as_it_was(models, tmp_path):
    import shutil

    from jax_gptq_b200 import packing
    path = models[2]
    blocks = pipeline.synth_stack(2, CFG)
    before = [{n: getattr(b, n) for n in pipeline.GROUPS} for b in blocks]
    good = packing.load_layer(f"{path}/layer1.pt")
    last = list(pipeline.GROUPS)[-1]
    scales = good[last].scales.clone()
    scales[0, 0] = float("nan")
    bad = [None, {n: good[n] for n in list(pipeline.GROUPS)[:-1]},
           {**good, last: packing.PackedLinear(**{**good[last].__dict__, "scales": scales})}]
    for layer, error in zip(bad, ((FileNotFoundError, "layer1"), (ValueError, "a block has"),
                                  (ValueError, f"layer1.pt: {last}: scales must be finite"))):
        shutil.copy(f"{path}/layer0.pt", tmp_path / "layer0.pt")
        if layer is not None:
            packing.save_layer(str(tmp_path / "layer1.pt"), layer)
        with pytest.raises(error[0], match=error[1]):
            pipeline.attach_packed(blocks, str(tmp_path))
        assert all(getattr(b, n) is lin for b, kept in zip(blocks, before) for n, lin in kept.items())
    pipeline.attach_packed(blocks, path)
    assert all(isinstance(getattr(b, n), linear.QuantLinear) for b in blocks for n in pipeline.GROUPS)
