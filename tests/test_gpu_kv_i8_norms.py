"""The decode and prompt attentions over the int8 cache in the norm, on the cases of test_gpu_kv_i8: per row and over a whole
case their outputs are off by what their roundings give as independent errors (test_kv_i8_norms.py has the derivation, and
shows that the bound rejects 2% or a block of keys)."""

import pytest
import torch

from test_gpu_kv_i8 import DECODES, PROMPTS
from test_kv_i8_norms import Case, beyond, expected

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("entry", DECODES + PROMPTS, ids=[f"{'step' if i < len(DECODES) else 'prompt'}{i}" for i in
                                                          range(len(DECODES) + len(PROMPTS))])
def test_outputs_are_as_close_as_their_roundings(pkg, dev, entry):
    print(f"[kv norms] {entry}", flush=True)
    c = Case(entry)
    cache = c.host.to(pkg, dev)
    kw = {"prefix": c.pre.to(pkg, dev), "prefix_len": c.npre} if c.npre else {}
    args = [z.to(dev) for z in (c.q, c.k, c.v)]
    tabs = (c.cos.to(dev), c.sin.to(dev))
    start = torch.tensor(c.start, device=dev)
    if c.step:
        got = pkg.gqa_decode_attention_i8(*args, cache, start, *tabs, **kw)
    else:
        got = pkg.gqa_prefill_attention_i8(*args, cache, start, c.t, *tabs, lengths=torch.tensor(c.lens, device=dev), **kw)
    c.write()
    out, e_out, e_in = expected(c, dev)
    row, whole = beyond(got, out, e_out, e_in)
    off = float((got.cpu().double() - out.reshape(got.shape)).norm() / out.norm())
    print(f"[kv norms] off by {off:.3g}, of the bound: a row {row:.3g}, the case {whole:.3g}", flush=True)
    assert row <= 1.0 and whole <= 1.0
