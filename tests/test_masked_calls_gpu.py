"""Masked steps and acceptance on the GPU, as calls: what a handle tells of its last one, caches beyond 4 GB, repeats, other streams, other devices."""
import numpy as np
import pytest
import torch

from tests import masked_harness as H

pytestmark = pytest.mark.gpu


def test_the_last_prefill_kernel_is_that_of_the_last_step():
    chunk, rows = H.Step([40, 9], [20, 1], window=16, seed=1), H.Step([40, 9], [1, 1], window=16, seed=2)
    op = chunk.operator()
    assert chunk.run(op)[3] == 0 and op.last_prefill_kernel() == "tcgen05"
    assert rows.run(op)[3] == 0 and op.last_prefill_kernel() == "none"
    causal = H.Step([40, 9], [20, 1], seed=3)
    given = {k: v for k, v in causal.inputs(causal.packed["key"].clone(), causal.packed["value"].clone()).items() if k not in ("sliding_window", "sink_tokens")}
    op.evaluate(given, {"output": torch.zeros_like(causal.query)})
    torch.cuda.synchronize()
    assert op.last_prefill_kernel() == "tcgen05"
    assert rows.run(op)[3] == 0 and op.last_prefill_kernel() == "none"
    slow = H.Step([40, 9], [20, 1], act="f16", cache="bf16", window=16, seed=4)
    op = slow.operator()
    assert slow.run(op)[3] == 0 and op.last_prefill_kernel() == "generic"


@pytest.mark.parametrize("act,cache", [("f16", "f16"), ("bf16", "bf16"), ("f16", "u8"), ("f16", "bf16")])
def test_blocks_beyond_four_gigabytes(act, cache):
    """The same step over a small cache and over the last blocks of one whose bytes and elements pass 32 bits: the same bits.  And the acceptance behind it."""
    rng = np.random.default_rng(1)
    new, trees = [1, 70, 30, 1], [None, None, H.tree(rng, 30, 1), None]
    step = H.Step([300, 90, 200, 40], new, hq=16, hkv=8, d=128, bs=32, act=act, cache=cache, window=150, sinks=3, trees=trees, poison=False, seed=5)
    op = step.operator()
    out, kc, vc, status = step.run(op)
    assert status == 0
    step.check(out)
    block = step.packed["key"][0].numel()
    front = ((1 << 33) if cache != "u8" else (1 << 32)) // block + 77
    big = [torch.zeros((front + step.pool, *c.shape[1:]), dtype=torch.uint8, device=step.dev) for c in (kc, vc)]
    for b, name in zip(big, ("key", "value")):
        b[front:] = step.packed[name]
    far = {**step.inputs(*big), "block_indices": step.meta["block_indices"] + front}
    got = torch.zeros_like(out)
    op.evaluate(far, {"output": got})
    torch.cuda.synchronize()
    assert op.device_status() == 0
    assert torch.equal(got, out) and torch.equal(big[0][front:], kc) and torch.equal(big[1][front:], vc)
    draft = torch.arange(step.T, device=step.dev)
    sampled = torch.zeros(step.T, dtype=torch.int64, device=step.dev)
    t0 = int(step.begins[2])
    for i, p in enumerate(trees[2]):
        if p >= 0:
            sampled[t0 + p] = draft[t0 + i]                  # every token's last child
    mk = lambda *s, t=torch.int32: torch.zeros(s, dtype=t, device=step.dev)
    res = {"path": mk(4, 30), "num_accepted": mk(4), "next_token": mk(4, t=torch.int64)}
    for inputs, caches in ((step.meta, (kc, vc)), ({**step.meta, "block_indices": far["block_indices"]}, big)):
        op.tree_accept({**inputs, "tree_parents": step.parents, "draft_tokens": draft, "sampled_tokens": sampled, "key_caches": [caches[0]], "value_caches": [caches[1]]}, res)
    torch.cuda.synchronize()
    assert op.device_status() == 0 and int(res["num_accepted"][2]) > 2
    assert torch.equal(big[0][front:], kc) and torch.equal(big[1][front:], vc)
    assert not any(bool(b[:front].any()) for b in big)


@pytest.mark.parametrize("act,cache", [("f16", "f16"), ("bf16", "bf16"), ("f16", "u8")])
def test_repeats_give_the_same_bits(act, cache):
    """Whatever the order in which CTAs end: cut lists, both halves on one list, rows that are computed again, single tokens with and without a plan."""
    rng = np.random.default_rng(2)
    for step in (H.Step([9000, 100, 7], [30, 1, 200], d=128, bs=32, act=act, cache=cache, trees=[H.tree(rng, 30), None, None], seed=6),
                 H.Step([3000] * 5, [1] * 5, d=128, bs=32, act=act, cache=cache, window=700, sinks=4, seed=7),
                 H.Step([6000] * 3, [1] * 3, d=128, bs=32, act=act, cache=cache, window=5000, sinks=4, seed=8)):
        op = step.operator()
        first, kc, vc, status = step.run(op)
        assert status == 0
        for _ in range(10):
            out, k, v, status = step.run(op)
            assert status == 0 and torch.equal(out, first) and torch.equal(k, kc) and torch.equal(v, vc)


def test_a_layer_behind_a_layer_on_one_handle_and_a_stream_of_its_own():
    """Steps of one handle without a wait between them, on a stream that is not the current one."""
    steps = [H.Step([200 + i, 90], [1 if i % 3 else 40, 1], window=60 + i, sinks=i % 5, seed=10 + i) for i in range(12)]
    op, stream = steps[0].operator(), torch.cuda.Stream()
    caches = [(s.packed["key"].clone(), s.packed["value"].clone()) for s in steps]
    outs = [torch.zeros_like(s.query) for s in steps]
    torch.cuda.synchronize()
    for _ in range(3):
        for s, c, out in zip(steps, caches, outs):
            op.evaluate({**s.inputs(*c), "stream": stream.cuda_stream}, {"output": out})
    torch.cuda.synchronize()
    assert op.device_status() == 0
    for s, out in zip(steps, outs):
        s.check(out)


@pytest.mark.parametrize("act,cache", [("f16", "bf16"), ("f32", "bf16"), ("f16", "f16"), ("f16", "u8")])
def test_trees_that_claim_each_others_tokens_are_left_to_their_own_pages(act, cache):
    """Begins that go back: a token is the seventh of one sequence's tree and the second of another's, whose block table ends with its own tokens."""
    step = H.Step([20], [200], d=64, bs=16, act=act, cache=cache, trees=[list(range(-1, 199))], seed=9, spare_blocks=30)
    op, dev = step.operator(), step.dev
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device=dev)
    pages = (20 + 200 + 15) // 16
    good = dict(step.meta)
    step.meta["past_lens"], step.meta["subsequence_begins"] = i32([20, 0, 26]), i32([0, 200, 5, 11])          # (the second one's tokens are less than none)
    step.meta["block_indices"] = torch.cat([good["block_indices"][:pages], good["block_indices"][:2]])
    step.meta["block_indices_begins"] = i32([0, pages, pages, pages + 2])
    step.parents[5:11] = i32([-1, 0, 1, 2, 3, 4])
    for window in (0, 7):
        step.window = window
        out, _, _, status = step.run(op)
        assert status & 0x2
    step.window, step.meta = 0, good
    step.parents = i32(list(range(-1, 199)))
    out, _, _, status = step.run(op)
    assert status == 0
    step.check(out)
