"""Masked attention on the GPU (include/masked_b200.h): windows with sinks, trees of drafts, both, against 64 bits, with everything poisoned that no row sees."""
import numpy as np
import pytest
import torch

from tests import masked_harness as H

pytestmark = pytest.mark.gpu
CACHES = [("f16", "f16"), ("bf16", "bf16"), ("bf16", "u8"), ("f16", "u8"), ("f32", "bf16"), ("f16", "bf16"), ("f32", "f16"), ("f32", "u8")]


def _whole(step):
    out, kc, vc, status = step.run()
    assert status == 0
    step.check(out)
    k, v = step.cache_after()
    same = lambda a, b: torch.equal(a, b)
    assert same(kc, k) and same(vc, v), "the caches differ from what the step writes"


@pytest.mark.parametrize("act,cache", CACHES)
@pytest.mark.parametrize("d,bs", [(64, 16), (128, 32), (128, 16), (64, 32)])
def test_rows_under_a_window(act, cache, d, bs):
    past = [0, 1, 4, 31, 32, 33, 63, 64, 99, 100, 101, 500, 1000, 1023]
    for window, sinks in ((1, 0), (5, 2), (33, 4), (64, 64), (100, 0), (257, 33)):
        _whole(H.Step(past, [1] * len(past), d=d, bs=bs, act=act, cache=cache, window=window, sinks=sinks, seed=window))


@pytest.mark.parametrize("act,cache", CACHES)
@pytest.mark.parametrize("d,bs", [(64, 16), (128, 32)])
def test_prompts_under_a_window(act, cache, d, bs):
    for window, sinks in ((1, 0), (7, 3), (64, 0), (130, 70), (5000, 4)):
        _whole(H.Step([0, 0, 3, 77, 600], [2, 300, 64, 129, 70], d=d, bs=bs, act=act, cache=cache, window=window, sinks=sinks, seed=window))


@pytest.mark.parametrize("act,cache", CACHES)
@pytest.mark.parametrize("d,bs", [(64, 16), (128, 32)])
def test_trees(act, cache, d, bs):
    rng = np.random.default_rng(3)
    new = [1, 2, 5, 17, 64, 65, 128]
    past = [9, 0, 63, 64, 100, 1, 700]
    for bushy in (1, 3):
        _whole(H.Step(past, new, d=d, bs=bs, act=act, cache=cache, trees=[H.tree(rng, n, bushy) for n in new], seed=bushy))


@pytest.mark.parametrize("act,cache", [("f16", "f16"), ("bf16", "bf16"), ("f16", "u8"), ("f32", "bf16")])
def test_trees_under_a_window(act, cache):
    rng = np.random.default_rng(4)
    new, past = [1, 7, 30, 100, 33], [40, 0, 90, 300, 31]
    for window, sinks in ((1, 0), (2, 1), (3, 50), (20, 4), (90, 310)):
        _whole(H.Step(past, new, act=act, cache=cache, window=window, sinks=sinks, trees=[H.tree(rng, n, 1) for n in new], seed=window))


@pytest.mark.parametrize("hq,hkv", [(1, 1), (4, 4), (7, 1), (12, 1), (16, 1), (40, 2), (28, 4)])
@pytest.mark.parametrize("cache", ["f16", "u8"])
def test_head_layouts_and_mixed_steps(hq, hkv, cache):
    """Single tokens, prompts, trees and sequences without tokens in one step."""
    rng = np.random.default_rng(5)
    new, past = [1, 40, 12, 0, 1, 150, 3, 0], [200, 30, 120, 50, 0, 5, 64, 0]
    trees = [None, None, H.tree(rng, 12), None, None, None, H.tree(rng, 3), None]
    for window, sinks in ((0, 0), (48, 2)):
        _whole(H.Step(past, new, hq=hq, hkv=hkv, d=128, bs=32, cache=cache, window=window, sinks=sinks, trees=trees, seed=hq))


def test_the_largest_tree_is_a_chain_of_256_and_more_is_skipped():
    chain = list(range(-1, 255))
    _whole(H.Step([10, 300], [256, 256], trees=[chain, [-1] * 256], seed=1))
    big = H.Step([10, 5, 7], [257, 4, 1], trees=[list(range(-1, 256)), [-1, 0, 1, 0], None], seed=2)
    out, kc, vc, status = big.run()
    assert status == H.M.PA_DEV_BAD_TREE
    assert bool((out[:257] == 77).all()), "rows of a tree that is too large are left as they were"
    big.check(out, rows=slice(257, None))
    k, v = big.cache_after()
    assert torch.equal(kc, k) and torch.equal(vc, v)


def test_bad_parents_count_as_followers_of_the_cache():
    for bad in (5, 3, 100, -3, -2147483648, 2147483647):
        step = H.Step([33], [5], trees=[[-1, 0, 1, -1, 2]], seed=3)      # token 3: the tree as it will be taken
        step.parents[3] = bad
        out, _, _, status = step.run()
        assert status == H.M.PA_DEV_BAD_TREE
        step.check(out)


@pytest.mark.parametrize("cache", ["f16", "bf16", "u8"])
def test_a_long_context_is_cut_and_joined(cache):
    rng = np.random.default_rng(6)
    act = "bf16" if cache == "bf16" else "f16"
    _whole(H.Step([7001, 3], [30, 2], hq=8, hkv=2, d=128, bs=32, act=act, cache=cache, trees=[H.tree(rng, 30), H.tree(rng, 2)], seed=4))
    _whole(H.Step([9000], [40], hq=8, hkv=1, d=128, bs=32, act=act, cache=cache, window=6000, sinks=100, seed=5))
    _whole(H.Step([20000], [1], hq=8, hkv=1, d=128, bs=32, act=act, cache=cache, window=15000, sinks=100, seed=6))


@pytest.mark.parametrize("act,cache", [("f16", "f16"), ("bf16", "bf16"), ("f16", "u8"), ("f32", "bf16")])
def test_what_a_row_does_not_see_takes_no_part_in_it(act, cache):
    """Not-a-number and infinities at positions that some rows of a sequence see and others do not."""
    rng = np.random.default_rng(7)
    for value in (float("nan"), float("inf")):
        for trees, window, sinks in (([H.tree(rng, 20)], 4, 0), ([None], 16, 2)):
            step = H.Step([40], [20], act=act, cache=cache, window=window, sinks=sinks, trees=trees, seed=8)
            first = int(np.argmax(step.sees[0].any(0)[sinks:])) + sinks      # the lowest position in any row's window
            where = torch.zeros((step.pool, step.bs), dtype=torch.bool, device=step.dev)
            where[int(step.table[first // step.bs]), first % step.bs] = True
            step.poison(where, value)
            out, _, _, status = step.run()
            blind = torch.from_numpy(~step.sees[0][:, first]).to(step.dev)
            assert status == 0 and 0 < int(blind.sum()) < 20
            step.check(out, rows=blind)
            assert not bool(torch.isfinite(out[~blind]).all(1).any()), "a row that sees it has no finite result"


def test_large_queries_and_a_scale_of_ones_own():
    for cache in ("f16", "u8"):
        _whole(H.Step([100, 50], [1, 40], act="f32", cache=cache, window=60, sinks=2, magnitude=300.0, scale=1e-3, seed=9))
    _whole(H.Step([100, 50], [1, 40], act="bf16", cache="bf16", window=60, scale=0.5, magnitude=0.5, seed=10))


def test_a_window_of_the_whole_context_is_the_causal_step():
    """And the causal step by itself takes no window."""
    for cache in ("f16", "u8"):
        wide = H.Step([300, 40, 0], [1, 50, 20], cache=cache, window=1 << 30, seed=11)
        out, kc, vc, status = wide.run()
        assert status == 0
        wide.check(out)
        op = wide.operator()
        x = wide.inputs(wide.packed["key"].clone(), wide.packed["value"].clone())
        y = torch.zeros_like(out)
        with pytest.raises(H.pkg.GenaiB200Error, match="sink"):
            op.evaluate({k: v for k, v in x.items() if k != "sink_tokens"}, {"output": y})
        op.evaluate({k: v for k, v in x.items() if k not in ("sink_tokens", "sliding_window")}, {"output": y})
        torch.cuda.synchronize()
        wide.check(y)
        assert torch.equal(x["key_cache"], kc) and torch.equal(x["value_cache"], vc)


def test_host_tensors():
    rng = np.random.default_rng(8)
    for trees, window in (([H.tree(rng, 9), None], 0), (None, 20)):
        step = H.Step([50, 30], [9, 1], trees=trees, window=window, seed=12)
        dev = step.inputs(step.packed["key"].clone(), step.packed["value"].clone())
        host = {k: v.cpu() if isinstance(v, torch.Tensor) and "cache" not in k else v for k, v in dev.items()}
        out = torch.zeros((step.T, step.hq * step.d), dtype=torch.float16)
        op = step.operator()
        op.evaluate(host, {"output": out})
        step.check(out.to(step.dev))


def test_captured_steps_replay_beside_larger_ones():
    """Two graphs of one operator, a larger step between them that outgrows their scratch, inputs changed before the replays."""
    rng = np.random.default_rng(9)
    small = [H.Step([90, 40], [6, 1], trees=[H.tree(rng, 6), None], window=w, seed=20 + w) for w in (0, 30)]
    op = small[0].operator()
    with pytest.raises(H.pkg.GenaiB200Error, match="capture"):
        g = torch.cuda.CUDAGraph()
        s = small[0]
        kc, vc, out = s.packed["key"].clone(), s.packed["value"].clone(), torch.zeros((s.T, s.hq * s.d), dtype=torch.float16, device=s.dev)
        torch.cuda.synchronize()
        with torch.cuda.graph(g):
            op.evaluate(s.inputs(kc, vc), {"output": out})
    op.masked_reserve(7, 2, 16)
    graphs = []
    for s in small:
        kc, vc, out = s.packed["key"].clone(), s.packed["value"].clone(), torch.zeros((s.T, s.hq * s.d), dtype=torch.float16, device=s.dev)
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g):
            op.evaluate(s.inputs(kc, vc), {"output": out})
        graphs.append((g, out, s, kc, vc))      # (a graph names its caches)
    big = H.Step([3000] * 40, [60] * 40, window=100, seed=30)
    _, _, _, status = big.run(op)
    for g, out, s, _, _ in graphs * 2:
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        s.check(out)
    assert op.device_status() == 0


def test_two_operators_on_two_streams():
    steps = [H.Step([500, 20], [30, 1], cache=c, window=77, sinks=3, seed=31) for c in ("f16", "u8")]
    ops = [s.operator() for s in steps]
    streams = [torch.cuda.Stream() for _ in steps]
    outs = []
    torch.cuda.synchronize()
    for _ in range(5):
        for s, op, stream in zip(steps, ops, streams):
            with torch.cuda.stream(stream):
                out = torch.zeros((s.T, s.hq * s.d), dtype=torch.float16, device=s.dev)
                op.evaluate(s.inputs(s.packed["key"].clone(), s.packed["value"].clone()), {"output": out})
                outs.append((s, out))
    torch.cuda.synchronize()
    for s, out in outs:
        s.check(out)


def test_bad_metadata_and_pages_set_a_status_bit_and_touch_nothing_else():
    step = H.Step([100, 70, 90], [1, 30, 12], trees=[None, None, H.tree(np.random.default_rng(1), 12)], window=64, seed=13)
    op = step.operator()
    for name, at, value, rows in (("past_lens", 1, -1, slice(1, 31)), ("past_lens", 2, 10 ** 9, slice(31, 43)), ("past_lens", 0, 2147483647, slice(0, 1))):
        keep = step.meta[name].clone()
        step.meta[name][at] = value
        out, _, _, status = step.run(op)
        assert status & 0x6
        assert bool((out[rows] == 77).all())
        others = [r for r in range(step.T) if r not in range(*rows.indices(step.T))]
        step.check(out, rows=torch.tensor(others, device=step.dev))
        step.meta[name] = keep
    # a page that a row sees with a number out of range: reported, the others' rows are right
    keep = step.meta["block_indices"].clone()
    at = int(step.first[1]) + 100 // step.bs - 1
    for bad in (-1, step.pool, 2147483647):
        step.meta["block_indices"][at] = bad
        out, _, _, status = step.run(op)
        assert status & 1
        step.check(out, rows=torch.tensor([0] + list(range(31, 43)), device=step.dev))
    step.meta["block_indices"] = keep
    out, _, _, status = step.run(op)
    assert status == 0
    step.check(out)


def test_refusals_of_tensors():
    step = H.Step([30], [4], trees=[[-1, 0, 0, 1]], window=8, seed=14)
    op = step.operator()
    good = step.inputs(step.packed["key"].clone(), step.packed["value"].clone())
    out = torch.zeros((4, step.hq * step.d), dtype=torch.float16, device=step.dev)
    wide = torch.zeros((4, 2 * step.hq * step.d), dtype=torch.float16, device=step.dev)
    for change in ({"sliding_window": -1}, {"sink_tokens": -1}, {"tree_parents": step.parents.long()}, {"tree_parents": step.parents[:3]}, {"tree_parents": step.parents.cpu()},
                   {"query": step.query.float()}, {"query": wide[:, ::2]}, {"query": step.query[:3]}, {"key": step.key[:, :-1]}, {"past_lens": step.meta["past_lens"].long()},
                   {"block_indices_begins": step.meta["block_indices_begins"][:1]}, {"key_cache": good["key_cache"].flatten()[:-16]},
                   {"score_aggregation_window": step.meta["past_lens"]}, {"alibi_slopes": torch.zeros(8, device=step.dev)}, {"scale": -1.0}, {"scale": float("nan")},
                   {"scale": float("inf")}):
        with pytest.raises(H.pkg.GenaiB200Error):
            op.evaluate({**good, **change}, {"output": out})
    for bad in (wide[:, ::2], wide.flatten()[1:1 + out.numel()].view_as(out), out.cpu()):
        with pytest.raises(H.pkg.GenaiB200Error):
            op.evaluate(good, {"output": bad})
    torch.cuda.synchronize()
    assert bool((out == 0).all())
    op.evaluate(good, {"output": out})
    step.check(out)


@pytest.mark.parametrize("act,cache", [("f16", "f16"), ("bf16", "bf16"), ("f16", "u8"), ("f32", "bf16")])
def test_chunks_beside_sequences_without_tokens(act, cache):
    """As many tokens as sequences, or fewer, and chunks among them all the same."""
    rng = np.random.default_rng(2)
    for new in ([0, 2], [3, 0, 0], [0, 0, 2, 1, 0, 0], [1, 5, 0, 0, 0, 0], [0, 4, 0, 0, 0, 0, 0]):
        past = [int(rng.integers(0, 90)) for _ in new]
        _whole(H.Step(past, new, act=act, cache=cache, window=20, sinks=2, seed=len(new)))
        _whole(H.Step(past, new, act=act, cache=cache, trees=[H.tree(rng, n) if n > 1 else None for n in new], seed=len(new)))


def test_rows_behind_the_last_sequence_stay_as_they_were():
    for new, trees in (([1, 1], None), ([1, 20], None), ([7, 3], [[-1, 0, 0, 1, 1, 2, 5], None])):
        step = H.Step([50, 30, 0], new + [4], trees=trees + [None] if trees else None, window=16, seed=40)
        op = step.operator()
        for name in ("past_lens", "subsequence_begins", "block_indices_begins"):      # the third sequence is not told of
            step.meta[name] = step.meta[name][:-1].contiguous()
        out, kc, vc, status = step.run(op)
        n = sum(new)
        assert status in (0, 2)                 # tokens that no sequence owns may be reported
        assert bool((out[n:] == 77).all())
        step.check(out, rows=slice(0, n))


@pytest.mark.parametrize("cache", ["f16", "u8"])
def test_sequences_that_share_their_first_blocks(cache):
    rng = np.random.default_rng(3)
    for new, trees, window in (([1, 1, 1], None, 0), ([1, 1, 1], None, 50), ([12, 5, 1], [H.tree(rng, 12), H.tree(rng, 5), [-1]], 0), ([30, 40, 1], None, 70)):
        step = H.Step([100, 100, 100], new, cache=cache, trees=trees, window=window, poison=False, seed=41)
        shared = 96 // step.bs
        for s in (1, 2):
            a, b = int(step.first[s]), int(step.first[0])
            step.table[a:a + shared] = step.table[b:b + shared]
        step.meta["block_indices"] = torch.from_numpy(step.table.copy()).to(step.dev)
        out, _, _, status = step.run()
        assert status == 0
        step.check(out)


@pytest.mark.parametrize("act,cache", [("f16", "f16"), ("bf16", "bf16"), ("f16", "u8")])
def test_trees_of_one_token_in_a_step_without_a_window(act, cache):
    past = [0, 5, 31, 32, 200, 1000, 1500]
    _whole(H.Step(past, [1] * 7, act=act, cache=cache, trees=[[-1]] * 7, seed=42))
    _whole(H.Step([4000, 100], [1, 1], act=act, cache=cache, trees=[[-1], None], seed=43))


def test_blocks_of_zeros_and_rows_of_one_value():
    """Keys that are all alike: every visible position has the same weight."""
    for cache in ("f16", "u8"):
        step = H.Step([77, 40], [1, 25], cache=cache, window=33, sinks=3, poison=False, seed=44)
        for c in step.packed.values():
            c.zero_()
        step.key.zero_()
        out, _, _, status = step.run()
        assert status == 0
        step.check(out)


def test_a_step_of_nothing():
    step = H.Step([10], [3], window=4, seed=45)
    op = step.operator()
    empty = {k: v[:0].contiguous() if k in ("query", "key", "value", "past_lens", "block_indices") else v for k, v in
             step.inputs(step.packed["key"].clone(), step.packed["value"].clone()).items()}
    empty["subsequence_begins"], empty["block_indices_begins"] = (torch.zeros(1, dtype=torch.int32, device=step.dev) for _ in range(2))
    op.evaluate(empty, {"output": step.query[:0].clone()})
    torch.cuda.synchronize()
    assert op.device_status() == 0
    idle = H.Step([10, 20], [0, 0], window=4, seed=46)
    out, _, _, status = idle.run(op)
    assert status == 0 and out.numel() == 0


@pytest.mark.parametrize("act,cache", [("f16", "f16"), ("bf16", "bf16"), ("f16", "u8")])
def test_keys_that_are_not_numbers_and_seen_reach_the_result(act, cache):
    """Whichever piece of a cut list they fill: a piece with no other keys has no maximum, and still counts."""
    past, trees = 64 * 30, [[-1, 0, 0, 1]]
    whole = None
    for first in range(0, 30, 2):
        for tiles in (1, 3, 4):
            step = H.Step([past], [4], hq=4, hkv=1, act=act, cache=cache, trees=trees, seed=3)
            where = torch.zeros((step.pool, step.bs), dtype=torch.bool, device=step.dev)
            for pos in range(64 * first, min(64 * (first + tiles), past)):
                where[int(step.table[pos // step.bs]), pos % step.bs] = True
            values = step.packed["value"].clone()
            step.poison(where)
            step.packed["value"] = values          # (of the keys alone)
            whole = whole or step.operator()
            out, *_, status = step.run(whole)
            assert status == 0 and bool(out.isnan().all())


@pytest.mark.parametrize("new", [[1], [3], [1, 1, 2], [0, 1]])
def test_steps_padded_with_tokens_of_no_sequence(new):
    """More rows than the sequences have, and as many rows as sequences though none has just one."""
    step = H.Step([30 + 7 * i for i in range(len(new))], new, window=20, sinks=3, seed=len(new) + sum(new))
    for rows in (step.T + 1, step.T + 4, len(new) + 3):
        pad = rows - step.T
        if pad <= 0:
            continue
        op, (kc, vc) = step.operator(), (step.packed["key"].clone(), step.packed["value"].clone())
        given = step.inputs(kc, vc)
        for name in ("query", "key", "value"):
            given[name] = torch.cat([given[name], given[name].new_full((pad, given[name].shape[1]), float("nan"))])
        out = torch.full((rows, step.hq * step.d), 77.0, dtype=torch.float16, device=step.dev)
        op.evaluate(given, {"output": out})
        torch.cuda.synchronize()
        assert op.device_status() in (0, 2)     # tokens that no sequence owns may be reported
        step.check(out[:step.T])
        assert bool((out[step.T:] == 77).all())


@pytest.mark.parametrize("act,cache", [("f16", "f16"), ("f16", "u8"), ("f32", "bf16")])
def test_begins_that_go_back_are_reported(act, cache):
    """The same tokens given to several sequences: more q tiles than tokens make."""
    past, n = [40] * 9, 300
    step = H.Step(past, [n] + [0] * 8, hq=8, hkv=2, act=act, cache=cache, window=64, seed=50, spare_blocks=400)
    op = step.operator()
    good, blocks = dict(step.meta), (past[0] + n + step.bs - 1) // step.bs
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device=step.dev)
    step.meta["subsequence_begins"] = i32([0, n] * 5)          # 0 .. n, back, 0 .. n, back, ...
    step.meta["block_indices"] = i32([(s * blocks + b) % step.pool for s in range(9) for b in range(blocks)])
    step.meta["block_indices_begins"] = i32([s * blocks for s in range(10)])
    out, *_, status = step.run(op)
    assert status & 2
    step.meta = good
    out, *_, status = step.run(op)
    assert status == 0
    step.check(out)


@pytest.mark.parametrize("cache", ["f16", "u8"])
def test_rotated_blocks_are_rotated_first(cache):
    """Keys that the step rotates are rotated for its rows, as in a causal step."""
    for new in ([1, 1, 1], [1, 30, 5]):
        step = H.Step([200, 90, 140], new, cache=cache, window=1 << 30, sinks=2, seed=61)
        op, dev = step.operator(), step.dev
        angle = torch.rand(9, step.d // 2, device=dev)
        blocks = torch.tensor([int(step.table[step.first[s] + b]) for s, b in ((0, 0), (0, 3), (1, 2), (2, 7))], dtype=torch.int32, device=dev)
        extra = {"rotated_block_indices": blocks, "rotation_deltas": torch.tensor([[1], [7], [2], [5]], dtype=torch.int32, device=dev),
                 "rotation_trig_lut": torch.cat([angle.cos(), angle.sin()], 1).contiguous()}
        got = []
        for masked in (True, False):
            kc, vc = step.packed["key"].clone(), step.packed["value"].clone()
            given = {**step.inputs(kc, vc), **extra}
            if not masked:
                del given["sliding_window"], given["sink_tokens"]
            out = torch.zeros((step.T, step.hq * step.d), dtype=torch.float16, device=dev)
            op.evaluate(given, {"output": out})
            torch.cuda.synchronize()
            assert op.device_status() == 0
            got.append((out.double(), kc, vc))
        assert torch.equal(got[0][1], got[1][1]) and torch.equal(got[0][2], got[1][2])
        assert not torch.equal(got[0][1], step.cache_after()[0])
        # each side is within the tolerance that a row has against the definition
        tol = 2 * 4 * {"f16": 2e-3, "u8": 1e-2}[cache]
        heads = lambda y: y.view(-1, step.hq, step.d)
        assert bool((heads(got[0][0] - got[1][0]).norm(dim=-1) <= tol * heads(got[1][0]).norm(dim=-1)).all())


@pytest.mark.parametrize("hq,d,bs", [(8, 64, 16), (8, 128, 32)])
def test_rows_that_see_each_others_new_tokens(hq, d, bs):
    """Single tokens given as sequences of their own over the same blocks: every new token is written before a row reads it."""
    for last in (30, 31, 32, 63, 64):        # positions last .. last + 3, tiles of 32 end among them
        rows = 4
        one = H.Step([last], [rows], hq=hq, d=d, bs=bs, window=1 << 20, sinks=1, seed=70 + last)
        op = one.operator()
        i32 = lambda a: torch.tensor(a, dtype=torch.int32, device=one.dev)
        blocks = one.meta["block_indices"].numel()
        for window in (1 << 20, 50):
            one.window, one.sinks = window, 1
            one.sees = [one.seen(0)]
            kc, vc = one.packed["key"].clone(), one.packed["value"].clone()
            given = {**one.inputs(kc, vc), "sliding_window": window, "sink_tokens": 1, "past_lens": i32([last + i for i in range(rows)]),
                     "subsequence_begins": i32(list(range(rows + 1))), "block_indices": one.meta["block_indices"].repeat(rows),
                     "block_indices_begins": i32([i * blocks for i in range(rows + 1)])}
            out = torch.zeros((rows, one.hq * one.d), dtype=torch.float16, device=one.dev)
            for _ in range(20):
                kc.copy_(one.packed["key"]); vc.copy_(one.packed["value"])
                op.evaluate(given, {"output": out})
                torch.cuda.synchronize()
                assert op.device_status() == 0
                one.check(out)
