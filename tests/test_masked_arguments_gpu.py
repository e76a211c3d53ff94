"""Arguments of masked steps that do not fit their types, from host and device tensors."""
import pytest
import torch

from tests import masked_harness as H

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("host", [False, True])
def test_windows_and_sinks_that_are_no_32_bit_numbers_are_refused(host):
    step = H.Step([30], [4], window=8, seed=1)
    op = step.operator()
    good = step.inputs(step.packed["key"].clone(), step.packed["value"].clone())
    out = torch.zeros((4, step.hq * step.d), dtype=torch.float16, device=step.dev)
    if host:
        good, out = {k: v.cpu() if isinstance(v, torch.Tensor) and "cache" not in k else v for k, v in good.items()}, out.cpu()
    for name in ("sliding_window", "sink_tokens"):
        for value in (1 << 31, 1 << 32, (1 << 32) + 8, -1, -(1 << 32), 7.5, "8"):
            with pytest.raises(H.pkg.GenaiB200Error, match=name):
                op.evaluate({**good, name: value}, {"output": out})
    torch.cuda.synchronize()
    assert bool((out == 0).all())
    op.evaluate(good, {"output": out})
    torch.cuda.synchronize()
    step.check(out.to(step.dev))


def test_parents_on_the_host_that_are_not_contiguous_are_refused():
    step = H.Step([30], [4], trees=[[-1, 0, 0, 1]], seed=2)
    op = step.operator()
    dev = step.inputs(step.packed["key"].clone(), step.packed["value"].clone())
    host = {k: v.cpu() if isinstance(v, torch.Tensor) and "cache" not in k else v for k, v in dev.items()}
    out = torch.zeros((4, step.hq * step.d), dtype=torch.float16)
    wide = torch.zeros(8, dtype=torch.int32)
    wide[::2] = host["tree_parents"]
    for parents in (wide[::2], wide[::2].numpy()):
        with pytest.raises(H.pkg.GenaiB200Error, match="tree_parents"):
            op.evaluate({**host, "tree_parents": parents}, {"output": out})
    assert bool((out == 0).all())
    for parents in (host["tree_parents"], host["tree_parents"].numpy()):
        op.evaluate({**host, "tree_parents": parents}, {"output": out})
        step.check(out.to(step.dev))


def test_more_tiles_than_32_bits_number_are_refused():
    """Before anything of the step is looked at: the pointers are small."""
    import ctypes as C
    from openvino_genai_b200 import _abi, _masked_abi as M
    step = H.Step([30], [1], hq=64, hkv=64, d=64, bs=16, window=8, seed=3)
    op = step.operator()
    good = step.inputs(step.packed["key"].clone(), step.packed["value"].clone())
    out = torch.zeros((1, step.hq * step.d), dtype=torch.float16, device=step.dev)
    args = op.make_args(good["query"], good["key"], good["value"], out, good["key_cache"], good["value_cache"], good["past_lens"], good["subsequence_begins"],
                        good["block_indices"], good["block_indices_begins"])
    mask = M.pa_mask_args(C.sizeof(M.pa_mask_args), 8, 0, None)
    indices = args.num_block_indices
    for n in (1 << 26, (1 << 31) // 16 - 512):
        args.num_block_indices = n
        assert op.lib.pa_b200_forward_masked(op._h, C.byref(args), C.byref(mask)) == _abi.PA_ERR_TOO_LARGE
    args.num_block_indices = indices
    assert op.lib.pa_b200_forward_masked(op._h, C.byref(args), C.byref(mask)) == 0
    torch.cuda.synchronize()
    assert op.device_status() == 0
    step.check(out)
