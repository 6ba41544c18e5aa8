"""GatedBitLinear's pack on several streams and around captured graphs: every call multiplies by what the weights hold when
it runs."""

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def _module(pkg, dev, k=256, f=192):
    torch.manual_seed(0)
    mod = pkg.GatedBitLinear(k, f, act="silu", device=dev)
    return mod, torch.randn(8, k, device=dev)


def _fresh(pkg, mod, x):
    """The module's value from a pack made for it alone."""
    with torch.no_grad():
        return pkg.gated_bitlinear(x, mod.gate_proj.weight, mod.up_proj.weight, act=mod.act)


@torch.no_grad()
def _change(mod, seed):
    g = torch.Generator(device=mod.gate_proj.weight.device).manual_seed(seed)
    for w in mod.parameters():
        w.copy_(torch.randn(w.shape, generator=g, device=w.device))


def test_one_module_on_two_streams(pkg, dev):
    """The first stream is busy when it queues the pack; the second finds the pack current and has to wait for it.  The next
    change replaces it while both may still read it."""
    mod, x = _module(pkg, dev)
    big = torch.randn(4096, 4096, device=dev, dtype=BF16)
    streams = [torch.cuda.Stream() for _ in range(2)]
    got, want = [], []
    for i in range(6):
        _change(mod, i)
        want.append(_fresh(pkg, mod, x))
        changed = torch.cuda.current_stream().record_event()
        for s, work in zip(streams, (10, 0)):
            s.wait_event(changed)
            with torch.cuda.stream(s), torch.no_grad():
                for _ in range(work):
                    big @ big
                got.append(mod(x))
        for s in streams:
            torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    for i, h in enumerate(got):
        assert torch.equal(h, want[i // 2]), i


def test_an_eager_call_between_a_capture_and_its_replay(pkg, dev):
    for warm in (True, False):
        mod, x = _module(pkg, dev)
        with torch.no_grad():
            pkg.gated_bitlinear(x, mod.gate_proj.weight, mod.up_proj.weight)
            if warm:
                mod(x)
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                mod.pack()
                h = mod(x)
            want = _fresh(pkg, mod, x)
            assert torch.equal(mod(x), want)  # nothing of the graph has run yet
            for seed in range(3):
                graph.replay()
                torch.cuda.synchronize()
                assert torch.equal(h, want)
                _change(mod, seed)
                want = _fresh(pkg, mod, x)
                assert torch.equal(mod(x), want)
                mod.pack()
                assert torch.equal(mod(x), want)
        del graph


def test_a_training_step_without_a_pack_in_it(pkg, dev):
    """The weights are unchanged between the warm-up and the capture, whose replays change them: each packs what it finds."""
    mod, x = _module(pkg, dev)
    twin, _ = _module(pkg, dev)
    target = torch.randn(8, 192, device=dev)
    weights = [list(m.parameters()) for m in (mod, twin)]

    def step(m, ws):
        grads = torch.autograd.grad((m(x) * target).sum(), ws)
        with torch.no_grad():
            for w, g in zip(ws, grads):
                w.sub_(g, alpha=0.05)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad((mod(x) * target).sum(), weights[0])
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(mod, weights[0])
    for _ in range(4):
        graph.replay()
        torch.cuda.synchronize()
        step(twin, weights[1])
        assert all(torch.equal(a, b) for a, b in zip(*weights))
    assert not torch.equal(_fresh(pkg, mod, x), _fresh(pkg, _module(pkg, dev)[0], x))  # (the packs did change)
    assert torch.equal(mod.pack()(x).detach(), _fresh(pkg, mod, x))


def test_weights_replaced_by_apply(pkg, dev):
    """What a module's casts and moves go through may leave other values at the same address and version: so may a cast to
    bf16 and back, whose last memory is the first one's, and here a function that writes through .data."""
    mod, x = _module(pkg, dev)
    with torch.no_grad():
        first = mod(x)
        stamps = [(w.data_ptr(), w._version) for w in mod.parameters()]
        mod.apply(lambda m: None)
        assert torch.equal(mod(x), first)
        mod._apply(lambda t: t.data.mul_(torch.where(torch.arange(t.shape[1], device=dev) % 3 == 0, -1.0, 1.0)))
        assert [(w.data_ptr(), w._version) for w in mod.parameters()] == stamps
        assert torch.equal(mod(x), _fresh(pkg, mod, x)) and not torch.equal(mod(x), first)
        mod.bfloat16().float()
        assert torch.equal(mod(x), _fresh(pkg, mod, x))
