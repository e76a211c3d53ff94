"""Acceptance of drafted trees on the GPU: corrupt trees, and calls that are refused."""
import numpy as np
import pytest
import torch

from tests import masked_harness as H
from tests.test_tree_accept_gpu import _run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("at,bad", [(0, 0), (0, 7), (2, 2), (3, 4), (4, 5), (5, 100), (1, -2), (5, -3), (3, -2147483648), (2, 2147483647)])
def test_a_tree_with_a_bad_parent_is_not_walked(at, bad):
    """On the path (tokens 0, 2, 3) or beside it: nothing of its sequence is accepted, the others' are."""
    trees = [[-1, 0, 1], [-1, 0, 0, 2, 1, 1], [-1, 0]]
    step = H.Step([20, 33, 40], [3, 6, 2], d=64, bs=16, trees=trees, poison=False, seed=1)
    step.parents[3 + at] = bad
    draft = np.array([1, 2, 3, 10, 11, 12, 13, 14, 15, 1, 2])
    sampled = np.array([2, 3, 4, 12, 0, 13, 99, 0, 0, 2, 77])
    for in_place in (False, True):
        out, keys, values, before, status = _run(step, draft, sampled, 4, in_place=in_place)
        assert status == H.M.PA_DEV_BAD_TREE
        assert out["num_accepted"].tolist() == [3, 0, 2] and out["next_token"].tolist() == [4, -1, 77] and out["new_past_lens"].tolist() == [23, 33, 42]
        assert out["path"].tolist() == [[0, 1, 2, -1], [-1] * 4, [0, 1, -1, -1]]
        for i in range(2):
            assert torch.equal(keys[i], before[i][0]) and torch.equal(values[i], before[i][1])
    step.parents[3 + at] = trees[1][at]
    out, _, _, _, status = _run(step, draft, sampled, 4)
    assert status == 0 and out["num_accepted"].tolist() == [3, 3, 2] and out["next_token"].tolist() == [4, 99, 77]


def test_caches_that_overlap_are_refused():
    """A layer's caches inside another's: each would be moved by blocks of its own, at once."""
    step = H.Step([20], [4], d=64, bs=16, trees=[[-1, 0, 0, 1]], poison=False, seed=7)
    op, dev = step.operator(), step.dev
    ids = torch.zeros(4, dtype=torch.int64, device=dev)
    n, block = step.packed["key"].numel(), step.packed["key"][0].numel()
    mk = lambda *s, t=torch.int32: torch.full(s, 99, dtype=t, device=dev)
    out = {"path": mk(1, 4), "num_accepted": mk(1), "next_token": mk(1, t=torch.int64)}
    memory = torch.zeros(4 * n, dtype=torch.uint8, device=dev)
    at = lambda offset: memory[offset:offset + n]
    good = {**step.meta, "tree_parents": step.parents, "draft_tokens": ids, "sampled_tokens": ids}
    for keys, values in (([at(0)], [at(block)]), ([at(n - block)], [at(0)]), ([at(0), at(2 * n)], [at(n), at(3 * n - block)]), ([at(0), at(16)], [at(2 * n), at(3 * n)])):
        with pytest.raises(H.pkg.GenaiB200Error, match="overlap"):
            op.tree_accept({**good, "key_caches": keys, "value_caches": values}, out)
    torch.cuda.synchronize()
    assert all(bool((x == 99).all()) for x in out.values())
    op.tree_accept({**good, "key_caches": [at(0), at(2 * n)], "value_caches": [at(3 * n), at(n)]}, out)      # side by side
    torch.cuda.synchronize()
    assert int(out["num_accepted"][0]) >= 1


@pytest.mark.parametrize("cache", ["f16", "u8"])
def test_caches_of_all_layers_in_one_tensor(cache):
    """The same as the list of them."""
    step = H.Step([20, 9], [4, 3], d=64, bs=16, cache=cache, trees=[[-1, 0, 0, 2], [-1, 0, 0]], poison=False, seed=8)
    op, dev = step.operator(), step.dev
    draft, sampled = (torch.tensor(x, dtype=torch.int64, device=dev) for x in ([1, 2, 3, 4, 5, 6, 7], [3, 0, 4, 9, 7, 0, 0]))
    res = []
    for stacked in (False, True):
        keys, values = (torch.stack([step.packed[k].roll(i, 0) for i in range(5)]) for k in ("key", "value"))
        mk = lambda *s, t=torch.int32: torch.full(s, 99, dtype=t, device=dev)
        out = {"path": mk(2, 4), "num_accepted": mk(2), "next_token": mk(2, t=torch.int64)}
        op.tree_accept({**step.meta, "tree_parents": step.parents, "draft_tokens": draft, "sampled_tokens": sampled, "key_caches": keys if stacked else list(keys),
                        "value_caches": values if stacked else list(values)}, out)
        torch.cuda.synchronize()
        assert out["path"].tolist() == [[0, 2, 3, -1], [0, 2, -1, -1]]
        res.append((keys, values))
    assert torch.equal(res[0][0], res[1][0]) and torch.equal(res[0][1], res[1][1])
    assert not torch.equal(res[0][0], torch.stack([step.packed["key"].roll(i, 0) for i in range(5)]))
