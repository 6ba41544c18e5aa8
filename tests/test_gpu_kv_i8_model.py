"""BitNetDecoder over the int8 key/value cache: prompts cut into chunks, decode steps in a graph, a shared prefix.

The same tokens through different cuts give attention outputs that differ by their rounding (fp32: 2^-20 and less), which
the int8 activation quantisers behind them turn into a code's step here and there: a changed code moves a projection's
output by 1/127 of one of its K terms.  Logits of the two-layer fp32 models here are held to 2e-2 of their norm (a few
codes of 256 per layer changed by one step: sqrt(8 / 256) / 127 * sqrt(14 projections) = 0.5 %, with a margin of four);
the same calls again, eager or replayed from a graph, give the same bits.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu


def _model(pkg, dev, dtype=torch.float32, **kw):
    M = pkg.model
    cfg = M.BitNetConfig(vocab_size=512, hidden_size=256, intermediate_size=512, num_layers=2, num_heads=4,
                         num_kv_heads=2, head_dim=64, rope_theta=10000.0)
    return M.BitNetDecoder(cfg, seed=5, device=dev, dtype=dtype, backend=M.HipBackend(
        out_dtype=dtype, fused=True), kv_cache="int8", **kw)


def _rel(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_graph_replays_are_the_eager_steps(pkg, dev, dtype):
    model = _model(pkg, dev, dtype)
    prompt = torch.randint(0, 512, (3, 70), generator=torch.Generator().manual_seed(1))
    eager = model.generate(prompt, 90)
    assert torch.equal(model.generate(prompt, 90, graph=True), eager)
    model.share_prefix(prompt[0, :33])
    eager = model.generate(prompt, 40)
    assert torch.equal(model.generate(prompt, 40, graph=True), eager)


def test_prompt_cuts_steps_and_a_shared_prefix_agree(pkg, dev):
    model = _model(pkg, dev)
    ids = torch.randint(0, 512, (2, 150), generator=torch.Generator().manual_seed(2)).to(dev)
    ids[1, :100] = ids[0, :100]
    model.reset(2, 160)
    whole = model.forward(ids, 0)
    model.reset(2, 160)
    model.forward(ids[:, :77], 0)
    model.forward(ids[:, 77:149], 77)
    assert _rel(model.decode_step(ids[:, 149:], torch.full((2,), 149, device=dev)), whole) <= 2e-2
    model.share_prefix(ids[0, :100])
    model.reset(2, 60)
    assert _rel(model.forward(ids[:, 100:], 0), whole) <= 2e-2
    model.reset(2, 60)
    model.forward(ids[:, 100:149], 0)
    assert _rel(model.decode_step(ids[:, 149:], torch.full((2,), 49, device=dev)), whole) <= 2e-2
    # without it again
    model.share_prefix(None)
    model.reset(2, 160)
    assert torch.equal(model.forward(ids, 0), whole)


def test_close_to_the_cache_in_the_model_dtype(pkg, dev):
    """An int8 row is off by 1/254 of its largest element at most: the logits stay within a tenth of those over the fp32
    cache (the activations are int8 in both)."""
    M = pkg.model
    int8 = _model(pkg, dev)
    full = M.BitNetDecoder(int8.cfg, seed=5, device=dev, backend=M.HipBackend(out_dtype=torch.float32, fused=True))
    ids = torch.randint(0, 512, (2, 96), generator=torch.Generator().manual_seed(3)).to(dev)
    for m in (int8, full):
        m.reset(2, 100)
    assert _rel(int8.forward(ids, 0), full.forward(ids, 0)) <= 0.1


def test_refusals(pkg, dev):
    model = _model(pkg, dev)
    with pytest.raises(ValueError, match="on_host"):
        model.on_host(None)
    M = pkg.model
    with pytest.raises(ValueError, match="share_prefix"):
        M.BitNetDecoder(model.cfg, device=dev).share_prefix(torch.zeros(3, dtype=torch.long))
