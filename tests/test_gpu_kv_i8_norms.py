"""The decode and prompt attentions over the int8 cache in the norm, on the cases of test_gpu_kv_i8: per row and over a whole
case their outputs are off by what their roundings give as independent errors (test_kv_i8_norms.py has the derivation, and
shows that the bound rejects 2% or a block of keys)."""

import pytest
import torch

from test_gpu_kv_i8 import DECODES, F32, PROMPTS
from test_kv_i8_norms import Case, beyond, expected

pytestmark = pytest.mark.gpu


# steps whose fp32 rows meet a long prefix as a prompt's do (compared in every seventh head)
MORE = [
    (64, 64, 8, 128, 64, [i % 64 for i in range(64)], F32, 6220),
    (33, 64, 4, 64, 64, list(range(33)), F32, 16000),
]
CASES = DECODES + MORE + PROMPTS


@pytest.mark.parametrize("entry", CASES, ids=[f"{'prompt' if isinstance(e[6], list) else 'step'}{i}" for i, e in enumerate(CASES)])
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
    every = 7 if entry in MORE else 1
    row, whole = beyond(got, *expected(c, dev, every), every)
    print(f"[kv norms] of the bound: a row {row:.3g}, the case {whole:.3g}", flush=True)
    assert row <= 1.0 and whole <= 1.0
