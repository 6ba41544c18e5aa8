"""The optimizer class: steps counted for each tensor as torch counts them, refusals that leave no trace, state dicts that are
checked before they are taken."""

import copy
import pickle

import pytest
import torch

pytestmark = pytest.mark.gpu

SHAPES = ((64, 33), (5,), (1000,), (300,))


def _models(dev, n=2):
    torch.manual_seed(0)
    first = [torch.randn(s, device=dev) for s in SHAPES]
    return [[torch.nn.Parameter(t.clone()) for t in first] for _ in range(n)]


def _fill(models, have, seed):
    g = torch.Generator(device=models[0][0].device).manual_seed(seed)
    for i, ps in enumerate(zip(*models)):
        grad = torch.randn(ps[0].shape, generator=g, device=ps[0].device)
        for p in ps:
            p.grad = grad.clone() if i in have else None


# tensors that come late, that pause, that never come, and all from the start
PATTERNS = [[{0, 1}] * 4 + [{0, 1, 2}] * 3 + [{0, 2}, {0, 1, 2}, {1}], [set(range(4))] * 5 + [{1, 3}] * 3 + [set(range(4))] * 2]


@pytest.mark.parametrize("capturable", [False, True])
@pytest.mark.parametrize("pattern", PATTERNS)
def test_each_tensor_counts_its_own_steps(pkg, dev, pattern, capturable):
    """Against torch.optim.AdamW, whose operations are ordered otherwise: 10 steps of at most 4 lr (a moment that paused keeps
    its size while its count stands) by 10 * 8 * 4 * 2^-24 lr, and 10 roundings of the parameter."""
    a, b = _models(dev)
    ours, theirs = pkg.AdamW(a, lr=1e-2, capturable=capturable), torch.optim.AdamW(b, lr=1e-2)
    for t, have in enumerate(pattern):
        _fill((a, b), have, t)
        ours.step()
        theirs.step()
        if t == 5:  # a copy and a state dict on the way carry the counts
            saved = pickle.loads(pickle.dumps(ours.state_dict()))
            a, ours = copy.deepcopy((a, ours))
            ours.load_state_dict(saved)
    for p, q in zip(a, b):
        bound = 10 * (8 * 4 * 1e-2 + float(q.detach().abs().max())) * 2.0 ** -24
        assert float((p - q).detach().abs().max()) <= bound


def test_a_refused_step_is_not_counted(pkg, dev):
    for capturable in (False, True):
        a, b = _models(dev)
        oa, ob = (pkg.AdamW(m, lr=1e-2, capturable=capturable) for m in (a, b))
        for t in range(3):
            _fill((a, b), set(range(4)), t)
            if t == 1:
                good = a[2].data
                a[2].grad, a[2].data = None, torch.randn(1000, 2, device=dev).t()[:1].reshape(1000).as_strided((1000,), (0,))
                a[2].grad = torch.zeros(1000, device=dev)
                with pytest.raises(RuntimeError, match="contiguous"):
                    oa.step()
                a[2].grad, a[2].data = None, good
                a[2].grad = b[2].grad.clone()
            oa.step()
            ob.step()
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_captures_that_would_not_count(pkg, dev, monkeypatch):
    (a,) = _models(dev, 1)
    _fill((a,), {0, 1}, 0)
    plain, fresh, warm = pkg.AdamW(a), pkg.AdamW(a, capturable=True), pkg.AdamW(a, capturable=True)
    plain.step()
    warm.step()
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="capturable"):
        plain.step()
    with pytest.raises(RuntimeError, match="first step"):
        fresh.step()
    assert fresh.group_state() is None
    _fill((a,), {0}, 1)
    with pytest.raises(RuntimeError, match="together"):
        warm.step()
    _fill((a,), {0, 1}, 1)
    warm.step()
    assert [int(c) for c, _ in warm.state_dict()["flat"][0]["steps"]] == [2, 0]


def test_captured_steps_of_some_tensors(pkg, dev):
    a, b = _models(dev)
    oa, ob = pkg.AdamW(a, lr=1e-2, capturable=True), pkg.AdamW(b, lr=1e-2)
    for have, seed in ((set(range(4)), 0), ({0, 2}, 1)):
        _fill((a, b), have, seed)
        oa.step()
        ob.step()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        oa.step()
    for t in range(4):
        grads = [p.grad for p in a]
        _fill((b,), {0, 2}, 10 + t)
        for g, q in zip(grads, b):
            if g is not None:
                g.copy_(q.grad)
        graph.replay()
        torch.cuda.synchronize()
        ob.step()
        assert all(torch.equal(x, y) for x, y in zip(a, b))
    _fill((a, b), set(range(4)), 20)  # and on, outside the graph
    oa.step()
    ob.step()
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_state_dicts_are_checked_first(pkg, dev):
    (a, b) = _models(dev)
    opt, other = pkg.AdamW(a, lr=1e-2, state_bits=8), pkg.AdamW(b, lr=2e-2, state_bits=8)
    _fill((a, b), {0, 1, 3}, 0)
    opt.step()
    other.step()
    good = opt.state_dict()
    before = [t.clone() for t in other.group_state()]

    def refused(match, d):
        with pytest.raises(ValueError, match=match):
            other.load_state_dict(d)
        assert other.param_groups[0]["lr"] == 2e-2
        assert all(torch.equal(x, y) for x, y in zip(other.group_state(), before))

    flat = good["flat"][0]
    refused("not this optimizer's", torch.optim.AdamW(a).state_dict())
    refused("not this optimizer's", {**good, "flat": []})
    refused("elements", {**good, "flat": [{**flat, "state": pkg.adamw_state(a[:2], 8)}]})
    refused("bits", {**good, "flat": [{**flat, "state": pkg.adamw_state(a)}]})
    refused("counts", {**good, "flat": [{**flat, "steps": flat["steps"][:1]}]})
    other.load_state_dict(good)
    assert other.param_groups[0]["lr"] == 1e-2
    assert all(torch.equal(x, y) for x, y in zip(other.group_state(), opt.group_state()))
    other.load_state_dict({**good, "flat": [{"state": flat["state"], "step": 1}]})  # one count for a whole group
    assert other.state_dict()["flat"][0]["steps"] == [(1, [0, 1, 2, 3])]
