"""The speculative decoding example: the draft-tree attention, the append of accepted tokens, the
attention mass and the eviction together, against decoding one token at a time."""
import importlib.util
import os

import pytest
import torch

import dvattn_b200

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def example():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "speculative_decode.py")
    spec = importlib.util.spec_from_file_location("speculative_decode", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def setup(X, W, n, vocab=64, capacity=400):
    model = X.Toy(Hq=8, Hkv=2, E=64, R=32, vocab=vocab, dtype=torch.float32, device=DEV, seed=3)
    prompt = torch.randint(0, vocab, (W, n), generator=torch.Generator().manual_seed(4)).to(DEV)
    return model, X.Decoder(model, prompt, capacity)


def greedy(d, n):
    """The next n tokens of every sequence, one at a time."""
    m, got = d.model, []
    for _ in range(n):
        t = d.pending[:, None]
        q, k, v = m.qkv(t)
        cos, sin = m.angles(d.seen[:, None])
        dvattn_b200.dvattn_paged_append(d.k, d.v, k, v, cos, sin, d.tables, d.cached)
        loc = d.cached[None, :, None].contiguous()
        out = dvattn_b200.dvattn_paged_sdpa(q, loc, cos[None], sin[None], d.turns, d.k, d.v, d.tables, m.scale)
        d.cached += 1
        d.seen += 1
        d.pending = m.choose(t, out)[:, 0]
        got.append(d.pending)
    return torch.stack(got, 1)


def test_speculative_steps_equal_greedy_decoding():
    X = example()
    model, d = setup(X, 5, 120)
    steps = 25
    gained = [d.step() for _ in range(steps)]
    per = torch.stack([(g >= 0).sum(1) for g in gained], 1)
    assert int(per.min()) == 1 and int(per.max()) == X.LEVELS + 1  # the draft is right at times
    _, ref = setup(X, 5, 120)
    want = greedy(ref, int(per.sum(1).max()))
    for w in range(5):
        mine = torch.cat([g[w][g[w] >= 0] for g in gained])
        assert torch.equal(mine, want[w, :mine.numel()])
    # every accepted token's weight over its cached keys is part of the mass: at most one a query head
    total = d.mass.sum(-1).double()
    queries = per.sum(1, keepdim=True) * (model.Hq // model.Hkv)
    assert bool((total > 0).all()) and bool((total <= queries * (1 + 1e-4)).all())


def test_the_mass_holds_all_weight_of_the_accepted_tokens():
    """Everything that an accepted token attended to is in the cache after its step, itself and the tokens
    accepted before it included: a query head's weights add up to one."""
    X = example()
    model, d = setup(X, 5, 120)
    gained = torch.stack([d.step() for _ in range(25)])
    accepted = (gained >= 0).sum((0, 2)).double()
    assert int((gained >= 0).sum(2).max()) > 1
    want = (accepted * (model.Hq // model.Hkv))[:, None].expand(5, model.Hkv)
    # scores and sums of both calls in 32 bits are within 1e-4 (the lse tolerance)
    assert bool(((d.mass.sum(-1).double() - want).abs() <= 2e-4 * want).all())


def test_speculative_steps_within_a_budget():
    X = example()
    _, d = setup(X, 5, 120)
    for _ in range(25):
        gained = d.step(budget=100, sink=4, recent=16)
        assert int(d.cached.max()) == 100
        assert bool((gained[:, 0] >= 0).all())
    assert int(d.seen.min()) >= 119 + 25
    beyond = torch.arange(d.mass.size(2), device=DEV) >= 100
    assert bool((d.mass[:, :, beyond] == 0).all()) and bool(torch.isfinite(d.mass).all())
    # a budget that holds everything changes nothing
    (_, a), (_, b) = setup(X, 3, 50), setup(X, 3, 50)
    for _ in range(8):
        assert torch.equal(a.step(), b.step(budget=1000))
