"""What a handle of masked steps holds on the device."""
import pytest
import torch

from tests import masked_harness as H

pytestmark = pytest.mark.gpu


def test_steps_of_single_tokens_take_no_scratch_for_chunks():
    """Partial results of the tensor-core kernel's CTAs are tens of MB: held by handles that serve chunks with it only."""
    free = lambda: (torch.cuda.synchronize(), torch.cuda.mem_get_info()[0])[1]
    ops = [H.pkg.PagedAttentionExtension(8, 8, 64, 32, torch.bfloat16, "bf16") for _ in range(4)]
    ops += [H.pkg.PagedAttentionExtension(8, 8, 64, 32, torch.float16, "bf16") for _ in range(4)]      # (chunks go row by row)
    before = free()
    for op in ops[:4]:
        op.masked_reserve(1, 1, 64)
    for op in ops[4:]:
        op.masked_reserve(64, 4, 64)
    assert before - free() < len(ops) * (8 << 20)


def test_a_step_of_single_tokens_and_chunks_behind_it():
    """The scratch grows where a handle's first chunks come behind its single tokens, and graphs of the former still run."""
    rows = H.Step([90, 40, 7], [1, 1, 1], window=30, seed=1)
    chunk = H.Step([90, 400], [60, 1], window=30, seed=2)
    op = rows.operator()
    op.masked_reserve(1, 1, 16)
    out, *_, status = H.Step([50], [1], window=30, seed=3).run(op)
    assert status == 0
    op.masked_reserve(3, 3, 64)
    kc, vc, out = rows.packed["key"].clone(), rows.packed["value"].clone(), torch.zeros((rows.T, rows.hq * rows.d), dtype=torch.float16, device=rows.dev)
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        op.evaluate(rows.inputs(kc, vc), {"output": out})
    got, *_, status = chunk.run(op)
    assert status == 0
    chunk.check(got)
    g.replay()
    torch.cuda.synchronize()
    rows.check(out)
