"""Acceptance of drafted trees on the GPU: paths, counts and next tokens against the walk in Python, and the caches byte by byte; and a step of drafts
from the attention to the step behind it."""
import numpy as np
import pytest
import torch

from tests import masked_harness as H

pytestmark = pytest.mark.gpu


def _moved(step, caches, paths):
    """The caches once the accepted tokens' rows lie where the paths say."""
    res = []
    for which, c in zip(("key", "value"), caches):
        c = c.clone()
        bs, d, h = step.bs, step.d, step.hkv
        for s, path in enumerate(paths):
            at = lambda pos: (int(step.table[step.first[s] + pos // bs]), pos % bs)
            rows = [at(step.past[s] + p) for p in path]
            if step.cache != "u8":
                x = c.view(torch.uint8).view(step.pool, h, bs, 2 * d)
                keep = [x[b, :, i].clone() for b, i in rows]
                for k, r in enumerate(keep):
                    b, i = at(step.past[s] + k)
                    x[b, :, i] = r
                continue
            data = c[:, :, :bs * d]
            data = data.unflatten(2, (d, bs)).transpose(2, 3) if which == "value" else data.unflatten(2, (bs, d))
            par = c[:, :, bs * d:].unflatten(2, (2, bs, 4))
            keep = [(data[b, :, i].clone(), par[b, :, :, i].clone()) for b, i in rows]
            for k, (r, q) in enumerate(keep):
                b, i = at(step.past[s] + k)
                data[b, :, i] = r
                par[b, :, :, i] = q
        res.append(c)
    return res


def _tokens(rng, step, vocab, right=0.7):
    """Draft ids, and ids sampled behind them: often a child's."""
    draft, sampled = rng.integers(0, vocab, step.T), rng.integers(0, vocab, step.T)
    for s, t in enumerate(step.trees):
        if t is None:
            continue
        t0 = int(step.begins[s])
        for i in range(len(t)):
            kids = [c for c in range(len(t)) if t[c] == i]
            if kids and rng.random() < right:
                sampled[t0 + i] = draft[t0 + int(rng.choice(kids))]
    return draft, sampled


def _run(step, draft, sampled, max_path, layers=2, op=None, in_place=False):
    op = op or step.operator()
    dev = step.dev
    i64 = lambda a: torch.from_numpy(np.asarray(a, np.int64)).to(dev)
    keys, values = [step.packed["key"].roll(i, 0).contiguous() for i in range(layers)], [step.packed["value"].roll(i, 0).contiguous() for i in range(layers)]
    before = [(k.clone(), v.clone()) for k, v in zip(keys, values)]
    B = len(step.new)
    parents = step.parents if step.parents is not None else torch.full((step.T,), H.NONE, dtype=torch.int32, device=dev)
    out = {"path": torch.full((B, max_path), 99, dtype=torch.int32, device=dev), "num_accepted": torch.full((B,), 99, dtype=torch.int32, device=dev),
           "next_token": torch.full((B,), 99, dtype=torch.int64, device=dev),
           "new_past_lens": step.meta["past_lens"].clone() if in_place else torch.full((B,), 99, dtype=torch.int32, device=dev)}
    meta = {**step.meta, "past_lens": out["new_past_lens"]} if in_place else step.meta
    op.tree_accept({**meta, "tree_parents": parents, "draft_tokens": i64(draft), "sampled_tokens": i64(sampled), "key_caches": keys, "value_caches": values}, out)
    torch.cuda.synchronize()
    return out, keys, values, before, op.device_status()


def _check(step, draft, sampled, max_path, got, layers=2):
    out, keys, values, before, status = got
    assert status == 0
    paths = []
    for s, t in enumerate(step.trees):
        a, b = int(step.begins[s]), int(step.begins[s + 1])
        if b == a:
            path, count, token = [], 0, -1
        elif t is None:
            path, count, token = [], b - a, int(sampled[b - 1])
        else:
            path = H.accept(t, draft[a:b], sampled[a:b], max_path)
            count, token = len(path), int(sampled[a + path[-1]])
        paths.append(path)
        assert out["path"][s].tolist() == path + [-1] * (max_path - len(path)), s
        assert int(out["num_accepted"][s]) == count and int(out["next_token"][s]) == token and int(out["new_past_lens"][s]) == step.past[s] + count, s
    for i in range(layers):
        k, v = _moved(step, before[i], paths)
        assert torch.equal(keys[i], k) and torch.equal(values[i], v), f"layer {i}"
    return paths


@pytest.mark.parametrize("act,cache", [("f16", "f16"), ("bf16", "u8")])
@pytest.mark.parametrize("d,bs", [(64, 16), (128, 32), (128, 16), (64, 32)])
def test_walk_and_move(act, cache, d, bs):
    rng = np.random.default_rng(d + bs)
    new = [1, 2, 30, 64, 3, 0, 100, 256, 1, 17]
    past = [0, 31, 16, 200, 5, 0, 63, 40, 7, 500]
    trees = [[-1], [-1, 0], H.tree(rng, 30), H.tree(rng, 64, 1), None, None, H.tree(rng, 100, 1), list(range(-1, 255)), None, H.tree(rng, 17, 1)]
    step = H.Step(past, new, hq=6, hkv=3, d=d, bs=bs, act=act, cache=cache, trees=trees, poison=False, seed=1)
    longest = 0
    for vocab, right, max_path in ((4, 0.5, 256), (50, 0.9, 256), (50, 1.0, 5), (2, 0.3, 1), (1, 0.0, 256)):
        draft, sampled = _tokens(rng, step, vocab, right)
        paths = _check(step, draft, sampled, max_path, _run(step, draft, sampled, max_path))
        longest = max(longest, max(map(len, paths)))
    assert longest == 256


def test_a_path_along_rows_that_are_overwritten():
    """The accepted tokens 0, 2, 4, 5: row 2 goes to 1, row 4 to where 2 was."""
    for cache in ("f16", "bf16", "u8"):
        step = H.Step([30], [6], d=64, bs=16, cache=cache, trees=[[-1, 0, 0, 1, 2, 4]], poison=False, seed=2)
        draft, sampled = np.arange(10, 16), np.array([12, 0, 14, 0, 15, 7])
        assert _check(step, draft, sampled, 8, _run(step, draft, sampled, 8)) == [[0, 2, 4, 5]]


def test_the_first_of_equal_children_and_ids_of_64_bits():
    step = H.Step([3], [5], trees=[[-1, 0, 0, 0, 2]], poison=False, seed=3)
    big = 1 << 40
    draft, sampled = np.array([1, big + 5, big + 6, big + 6, 9]), np.array([big + 6, 0, 9, 9, -1])
    assert _check(step, draft, sampled, 4, _run(step, draft, sampled, 4)) == [[0, 2, 4]]
    sampled[0] = 6        # the low bits alone are no match
    assert _check(step, draft, sampled, 4, _run(step, draft, sampled, 4)) == [[0]]


def test_many_layers_and_past_lens_in_place():
    rng = np.random.default_rng(4)
    step = H.Step([20, 40], [12, 9], d=64, bs=16, cache="u8", trees=[H.tree(rng, 12, 1), H.tree(rng, 9, 1)], poison=False, seed=4)
    draft, sampled = _tokens(rng, step, 9, 0.9)
    _check(step, draft, sampled, 16, _run(step, draft, sampled, 16, layers=200, in_place=True), layers=200)
    out, _, _, _, status = _run(step, draft, sampled, 16, layers=0)
    assert status == 0 and int(out["num_accepted"][0]) >= 1


def test_bad_trees_pages_and_lengths():
    rng = np.random.default_rng(5)
    step = H.Step([20, 40, 8], [12, 257, 6], d=64, bs=16, trees=[H.tree(rng, 12, 1), list(range(-1, 256)), [-1, 0, 1, 2, 3, 4]], poison=False, seed=5)
    draft, sampled = np.arange(step.T), np.arange(step.T) + 1      # every token is followed by the next one
    out, keys, _, before, status = _run(step, draft, sampled, 9, layers=1)
    assert status == H.M.PA_DEV_BAD_TREE
    assert out["num_accepted"].tolist()[1:] == [0, 6] and out["path"][1].tolist() == [-1] * 9 and int(out["next_token"][1]) == -1
    assert int(out["new_past_lens"][1]) == 40
    for value in (-1, 2147483647):
        keep = step.meta["past_lens"].clone()
        step.meta["past_lens"][2] = value
        out, _, _, _, status = _run(step, draft, sampled, 9, layers=1)
        assert status & 0x4 and int(out["num_accepted"][2]) == 0
        step.meta["past_lens"] = keep
    # a page out of range on the way: its row is not moved, the path is as it was
    step = H.Step([8], [6], d=64, bs=16, trees=[[-1, 0, 0, 2, 3, 4]], poison=False, seed=6)
    draft, sampled = np.arange(6), np.array([2, 9, 3, 4, 5, 9])
    for bad in (-1, step.pool, 1 << 30):
        keep = step.meta["block_indices"].clone()
        step.meta["block_indices"][0] = bad
        out, keys, _, before, status = _run(step, draft, sampled, 6, layers=1)
        assert status == 1 and out["path"][0].tolist() == [0, 2, 3, 4, 5, -1]
        assert torch.equal(keys[0], before[0][0])
        step.meta["block_indices"] = keep


def test_refusals():
    step = H.Step([20], [4], d=64, bs=16, trees=[[-1, 0, 0, 1]], poison=False, seed=7)
    op, dev = step.operator(), step.dev
    ids = torch.zeros(4, dtype=torch.int64, device=dev)
    k, v = step.packed["key"], step.packed["value"]
    good = {**step.meta, "tree_parents": step.parents, "draft_tokens": ids, "sampled_tokens": ids, "key_caches": [k], "value_caches": [v]}
    mk = lambda *s, t=torch.int32: torch.zeros(s, dtype=t, device=dev)
    out = {"path": mk(1, 4), "num_accepted": mk(1), "next_token": mk(1, t=torch.int64)}
    for change in ({"draft_tokens": ids.int()}, {"sampled_tokens": ids[:3]}, {"tree_parents": step.parents.cpu()}, {"key_caches": []}, {"key_caches": [k[:-1]]},
                   {"key_caches": [k.flatten()[:-16]]}, {"key_caches": [k.cpu()]}, {"past_lens": step.meta["past_lens"].long()}):
        with pytest.raises(H.pkg.GenaiB200Error):
            op.tree_accept({**good, **change}, out)
    for twice in ({"key_caches": [k, k], "value_caches": [v, v.clone()]}, {"key_caches": [k], "value_caches": [k]}):
        with pytest.raises(H.pkg.GenaiB200Error, match="twice"):
            op.tree_accept({**good, **twice}, out)
    for change in ({"path": mk(1, 0)}, {"path": mk(1, 257)}, {"path": mk(2, 4)}, {"path": mk(4)}, {"num_accepted": mk(2)}, {"next_token": mk(1)}, {"new_past_lens": mk(2)}):
        with pytest.raises(H.pkg.GenaiB200Error):
            op.tree_accept(good, {**out, **change})
    op.tree_accept(good, out)


@pytest.mark.parametrize("cache,window", [("f16", 0), ("bf16", 40), ("u8", 0)])
def test_a_step_of_drafts_and_the_step_behind_it(cache, window):
    """Attention over a tree, acceptance, and the next token's attention: the same as if the accepted tokens had come one by one."""
    rng = np.random.default_rng(6)
    act = "bf16" if cache == "bf16" else "f16"
    trees = [H.tree(rng, 20, 1), H.tree(rng, 9, 1)]
    step = H.Step([70, 33], [20, 9], act=act, cache=cache, window=window, sinks=2, trees=trees, poison=False, seed=8)
    op = step.operator()
    out, kc, vc, status = step.run(op)
    assert status == 0
    step.check(out)
    draft, sampled = _tokens(rng, step, 30, 1.0)
    dev = step.dev
    i64 = lambda a: torch.from_numpy(np.asarray(a, np.int64)).to(dev)
    got = {"path": torch.zeros((2, 12), dtype=torch.int32, device=dev), "num_accepted": torch.zeros(2, dtype=torch.int32, device=dev),
           "next_token": torch.zeros(2, dtype=torch.int64, device=dev), "new_past_lens": torch.zeros(2, dtype=torch.int32, device=dev)}
    op.tree_accept({**step.meta, "tree_parents": step.parents, "draft_tokens": i64(draft), "sampled_tokens": i64(sampled), "key_caches": [kc], "value_caches": [vc]}, got)
    paths = [[p for p in row if p >= 0] for row in got["path"].tolist()]
    assert [len(p) for p in paths] == got["num_accepted"].tolist() and max(map(len, paths)) > 2
    # the accepted rows' outputs are those of a causal step over the path
    rows = [int(step.begins[s]) + p for s in range(2) for p in paths[s]]
    plain = H.Step(step.past, [len(p) for p in paths], act=act, cache=cache, window=window, sinks=2, poison=False, seed=8)
    plain.packed, plain.table, plain.first, plain.pool = step.packed, step.table, step.first, step.pool
    plain.query, plain.key, plain.value = (x[rows] for x in (step.query, step.key, step.value))
    plain.meta["block_indices"], plain.meta["block_indices_begins"] = step.meta["block_indices"], step.meta["block_indices_begins"]
    plain.check(out[rows])
    ref, kc2, vc2, status = plain.run(op)
    plain.check(ref)
    # and the caches' contexts too
    for c, c2, value in ((kc, kc2, False), (vc, vc2, True)):
        for s in range(2):
            n = step.past[s] + len(paths[s])
            blocks = torch.from_numpy(step.table[step.first[s]:step.first[s + 1]].astype(np.int64)).to(dev)
            a, b = (step.unpack(x[blocks], value).transpose(1, 2).reshape(-1, step.hkv, step.d)[:n] for x in (c, c2))
            assert torch.equal(a, b)
