"""LatentAttention.reserve: steps within it allocate nothing, whatever their form."""
import pytest
import torch

from tests import latent_harness as LH

pytestmark = pytest.mark.gpu

WIDE_HEADS, BLOCK = 128, 64


class _Call:
    """A step whose block tables are as long as asked for, longer than its context: their entries count for the scratch."""

    def __init__(self, op, tokens, sequences, blocks, form):
        R, P, Dn, Dv = LH.WIDE
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
        rnd = lambda *s: torch.randn(s, device="cuda").to(torch.bfloat16)
        H, pool = op.num_heads, 64
        part = lambda n: [n * k // sequences for k in range(sequences + 1)]
        self.op, self.form = op, form
        self.inputs = {"past_lens": i32([0] * sequences), "subsequence_begins": i32(part(tokens)), "block_indices_begins": i32(part(blocks)),
                       "block_indices": torch.arange(blocks, dtype=torch.int32, device="cuda") % pool, "cache": rnd(pool, BLOCK, R + P),
                       "query_nope": rnd(tokens, H, Dn), "query_rope": rnd(tokens, H, P), "key_up": rnd(H, Dn, R) / 23, "value_up": rnd(H, Dv, R) / 23}
        self.outputs = {"output": torch.empty((tokens, H * Dv), dtype=torch.bfloat16, device="cuda")}

    def __call__(self):
        self.op.attend(self.inputs, self.outputs, form=self.form)


def _held(call):
    """Bytes of device memory that a call takes for good."""
    torch.cuda.synchronize()
    before = torch.cuda.mem_get_info()[0]
    call()
    torch.cuda.synchronize()
    return before - torch.cuda.mem_get_info()[0]


@pytest.mark.parametrize("reserved,calls", [
    ((4096, 2, 64, "auto"), [(4096, 2, 64, "absorbed"), (4096, 2, 64, "expanded"), (4096, 2, 64, "auto"), (1000, 1, 60, "absorbed"), (40, 2, 64, "auto")]),
    ((2048, 64, 16384, "expanded"), [(2048, 64, 12000, "expanded"), (2048, 64, 16000, "expanded"), (2048, 3, 8000, "expanded"), (100, 20, 300, "expanded")]),
    ((2048, 64, 20000, "auto"), [(2048, 64, 16000, "auto"), (2048, 64, 11000, "expanded"), (64, 64, 20000, "auto"), (64, 64, 20000, "absorbed")]),
])
def test_steps_within_a_reserve_do_not_allocate(pkg, reserved, calls):
    op = pkg.LatentAttention(WIDE_HEADS, *LH.WIDE, BLOCK, torch.bfloat16)
    steps = [_Call(op, *c) for c in calls]
    steps[-1].inputs["cache"].add_(0)      # (torch has what it needs)
    assert _held(lambda: op.reserve(*reserved)) > 0
    for c, step in zip(calls, steps):
        assert _held(step) == 0, f"reserve{reserved}: attend{c} took memory"
    assert op.device_status() == 0
