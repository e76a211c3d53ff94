"""Masked attention on the GPU: every position that a row sees is counted, and none other.

All queries are zero, so a row's weights are equal, 1 / n for n visible positions.  The value of position p is `MAG` in dimension (p + 5 * kv head) mod d and zero
elsewhere, so element e of a row is MAG / n times the number of visible positions of that residue.  MAG is 255 / 4: exact in every type, and with a scale of 1 / 4
in the u8 cache.  Weights (1), values and their sums are exact in 32 bits, so an element is off by the reciprocal and the products behind it
(8 roundings of 2^-24), the zero-points' share that is taken off (2^-21 of MAG at most, u8) and the output's own rounding.  A position too many or too few
changes a count of c by 1: more than that for c up to 100, which the sizes keep."""
import numpy as np
import pytest
import torch

from tests import masked_harness as H

pytestmark = pytest.mark.gpu
MAG = 63.75
CACHES = [("f16", "f16"), ("bf16", "bf16"), ("bf16", "u8"), ("f16", "u8"), ("f32", "bf16"), ("f32", "u8")]


def _count(step, op=None):
    dev, d = step.dev, step.d
    heads = torch.arange(step.hkv, device=dev)
    old, new, where = torch.zeros(step.pool, step.hkv, step.bs, d, device=dev), torch.zeros(step.T, step.hkv, d, device=dev), torch.ones((step.pool, step.bs), dtype=torch.bool)
    counts, seen = torch.zeros(step.T, step.hkv, d, dtype=torch.float64, device=dev), torch.zeros(step.T, dtype=torch.float64, device=dev)
    for s, (past, n) in enumerate(zip(step.past, step.new)):
        pos = torch.arange(past + n, device=dev)
        blocks = torch.from_numpy(step.table[step.first[s]:step.first[s + 1]].astype(np.int64)).to(dev)
        dim = (pos[:, None] + 5 * heads) % d
        at = pos[:past]
        old[blocks[at // step.bs][:, None], heads, (at % step.bs)[:, None], dim[:past]] = MAG
        t0 = int(step.begins[s])
        new[torch.arange(t0, t0 + n, device=dev)[:, None], heads, dim[past:]] = MAG
        sees = torch.from_numpy(step.sees[s]).to(dev).double()
        code = torch.zeros(past + n, step.hkv, d, dtype=torch.float64, device=dev)
        code[pos[:, None], heads, dim] = 1
        counts[t0:t0 + n] = torch.einsum("rp,phd->rhd", sees, code)
        seen[t0:t0 + n] = sees.sum(1)
        for p in np.flatnonzero(step.sees[s].any(0)) if n else []:
            where[int(step.table[step.first[s] + p // step.bs]), p % step.bs] = False
    step.packed["value"] = step.pack(old, True)
    step.poison(where.to(dev))
    step.value = new.view(step.T, -1).to(step.value.dtype)
    step.query.zero_()
    out, _, _, status = step.run(op)
    assert status == 0
    got = out.double().view(step.T, step.hkv, step.hq // step.hkv, d)
    want = (MAG * counts / seen[:, None, None])[:, :, None].expand_as(got)
    assert counts.max().item() <= 100
    off = (got - want).abs() - want * (torch.finfo(H.DT[step.act]).eps / 2 + 2.0 ** -21) - MAG * 2.0 ** -21
    bad = (~(off <= 0)).nonzero()
    assert len(bad) == 0, f"{len(bad)} elements, first [token, kv head, q head, dim] {bad[0].tolist()}: {got[tuple(bad[0])].item()} for {want[tuple(bad[0])].item()}"


@pytest.mark.parametrize("act,cache", CACHES)
@pytest.mark.parametrize("d,bs", [(64, 16), (128, 32)])
def test_single_tokens(act, cache, d, bs):
    """Streams short and long, with and without a gap behind the sinks."""
    past = [0, 1, 15, 16, 31, 32, 33, 63, 64, 65, 300, 1023, 1024, 1025, 4000]
    for window, sinks in ((1, 0), (2, 1), (31, 0), (32, 5), (33, 64), (64, 1), (65, 33), (1000, 4), (2500, 700)):
        _count(H.Step(past, [1] * len(past), d=d, bs=bs, act=act, cache=cache, window=window, sinks=sinks, seed=window))


@pytest.mark.parametrize("act,cache", CACHES)
@pytest.mark.parametrize("d,bs", [(64, 16), (128, 32)])
def test_prompts(act, cache, d, bs):
    for window, sinks in ((0, 0), (1, 0), (2, 65), (63, 0), (64, 1), (65, 4), (127, 64), (129, 200), (600, 3)):
        _count(H.Step([0, 1, 63, 64, 700], [300, 65, 2, 130, 64], d=d, bs=bs, act=act, cache=cache, window=window, sinks=sinks, seed=window))


@pytest.mark.parametrize("hq,hkv", [(7, 1), (12, 2), (40, 2)])
def test_head_layouts(hq, hkv):
    rng = np.random.default_rng(1)
    new, past = [1, 90, 33, 1, 200], [500, 30, 120, 0, 64]
    for cache in ("f16", "u8"):
        for window, sinks in ((0, 0), (50, 3)):
            _count(H.Step(past, new, hq=hq, hkv=hkv, d=128, bs=32, cache=cache, window=window, sinks=sinks, trees=[None, None, H.tree(rng, 33), None, None], seed=hq))


@pytest.mark.parametrize("act,cache", CACHES)
def test_long_contexts(act, cache):
    """Lists that are cut between CTAs, streams that are cut between warps."""
    rng = np.random.default_rng(2)
    _count(H.Step([6001, 3], [30, 2], hq=8, hkv=2, d=128, bs=32, act=act, cache=cache, trees=[H.tree(rng, 30), None], seed=4))
    _count(H.Step([9000], [40], hq=8, hkv=1, d=128, bs=32, act=act, cache=cache, window=5000, sinks=100, seed=5))
    _count(H.Step([12000], [1], hq=8, hkv=1, d=128, bs=32, act=act, cache=cache, window=9000, sinks=100, seed=6))
    _count(H.Step([12000, 20], [1, 1], hq=8, hkv=1, d=128, bs=32, act=act, cache=cache, window=1500, sinks=100, seed=7))


def bush(n, children, root=2):
    """A chain to token `root`, `children` children of it, and a chain below the last of them: ancestors whose places in the chunk are far from their positions."""
    return [i - 1 if i <= root else root if i <= root + children else i - 1 for i in range(n)]


@pytest.mark.parametrize("act,cache", CACHES + [("f16", "bf16")])
@pytest.mark.parametrize("d,bs", [(64, 16), (128, 32)])
def test_trees(act, cache, d, bs):
    """Chains, bushes and both: an ancestor that is a sink by its position lies anywhere in the chunk."""
    rng = np.random.default_rng(3)
    for past, window, sinks in (([0, 3], 2, 4), ([0, 1], 16, 4), ([2, 0], 64, 70), ([5, 90], 9, 0), ([31, 700], 0, 0), ([64, 10], 20, 66)):
        for trees in ([bush(256, 40), bush(150, 100, 0)], [H.tree(rng, 200, 3), H.tree(rng, 77, 1)], [bush(100, 1), list(range(-1, 63))]):
            _count(H.Step(past, [len(t) for t in trees], d=d, bs=bs, act=act, cache=cache, window=window, sinks=sinks, trees=trees, seed=window))


@pytest.mark.parametrize("act,cache", [("f16", "f16"), ("bf16", "bf16"), ("f16", "u8")])
def test_rows_of_a_bush_that_are_computed_again(act, cache):
    """A value that is not a number at a position that some rows see: the others of its tile go through the row-by-row path."""
    parents = bush(200, 60)
    step = H.Step([0], [200], act=act, cache=cache, window=8, sinks=4, trees=[parents], seed=8)
    leaf = 20                                              # a child of token 2: seen by nobody but itself
    step.value[leaf, 3] = float("nan") if cache != "u8" else float("-inf")      # (the lowest value is what a u8 token's zero-point is made of)
    out, _, _, status = step.run()
    blind = torch.arange(step.T, device=step.dev) != leaf
    assert status == 0
    step.key, step.value = step.key.clone(), step.value.clone()
    step.value[leaf] = 0                                   # (the definition of the rows that do not see it)
    step.check(out, rows=blind)
    assert not bool(torch.isfinite(out[leaf]).all())


@pytest.mark.parametrize("cache", ["f16", "u8"])
def test_a_step_of_many_kinds(cache):
    """Single tokens, chunks and trees together, more of them than the SMs take at once."""
    rng = np.random.default_rng(4)
    new = [int(x) for x in rng.choice([1, 1, 2, 17, 64, 100], 40)]
    past = [int(rng.integers(0, 900)) for _ in new]
    trees = [H.tree(rng, n) if n > 1 and rng.random() < 0.5 else None for n in new]
    for window, sinks in ((0, 0), (40, 3), (500, 70)):
        _count(H.Step(past, new, cache=cache, window=window, sinks=sinks, trees=trees, seed=window))
