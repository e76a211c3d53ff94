"""LatentAttention.reserve: steps within it allocate nothing, whatever their form, and can be captured; graphs outlive the scratch they were captured with."""
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


def _captured(st, op, form):
    """A graph of one append and one attend, its inputs and its output."""
    x = st.append_inputs()
    turned = torch.empty((st.tokens, st.heads, st.sizes[1]), dtype=LH.DTYPE[st.dtype], device="cuda")
    out = torch.empty((st.tokens, st.heads * st.sizes[3]), dtype=LH.DTYPE[st.dtype], device="cuda")
    op.reserve(st.tokens, len(st.new), len(st.meta["block_indices"]), form)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        op.append(x, {"query_rope": turned})
        op.attend({**x, "query_rope": turned}, {"output": out}, form=form)
    return graph, x, turned, out


@pytest.mark.parametrize("form", ["absorbed", "expanded", "auto"])
def test_a_captured_step_is_replayed_behind_other_steps(pkg, form):
    st = LH.Step([700, 0, 90], [1, 130, 3], heads=10, seed=31)
    op = st.operator(pkg)
    graph, x, turned, out = _captured(st, op, form)
    eager = st.append_inputs()
    other = st.operator(pkg)
    other.append(eager, {"query_rope": turned.clone()})
    want_out = torch.empty_like(out)
    rotated = torch.empty_like(turned)
    other.append(eager, {"query_rope": rotated})
    other.attend({**eager, "query_rope": rotated}, {"output": want_out}, form=form)

    def replay():
        out.fill_(float("nan"))
        turned.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want_out) and torch.equal(turned, rotated)

    replay()
    small = LH.Step([40], [2], heads=10, seed=32)      # within the scratch
    small.check(small.attend(op, form))
    replay()
    large = LH.Step([3000, 200, 5000], [400, 1, 70], heads=10, seed=33)      # outgrows it
    assert _held(lambda: op.reserve(4 * large.tokens, 3, 8 * len(large.meta["block_indices"]), form)) > 0
    junk = [torch.full((64 << 20,), 0xff, dtype=torch.uint8, device="cuda") for _ in range(8)]
    replay()
    assert all(bool((j == 0xff).all()) for j in junk), "a replay wrote into memory that is somebody else's"
    large.check(large.attend(op, form))
    replay()
    graph2, *kept, out2 = _captured(large, op, form)    # and one with the new scratch (a graph's inputs are the caller's to keep)
    graph2.replay()
    replay()
    graph2.replay()
    torch.cuda.synchronize()
    assert bool(torch.isfinite(out2).all()) and op.device_status() == 0


def test_a_capture_that_would_have_to_grow_the_scratch_is_refused(pkg):
    from openvino_genai_b200 import GenaiB200Error
    st = LH.Step([700, 9], [1, 40], heads=10, seed=34)
    op = st.operator(pkg)
    x = st.device_inputs()
    out = torch.empty((st.tokens, 10 * 128), dtype=torch.bfloat16, device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(GenaiB200Error, match="reserve"):
            op.attend(x, {"output": out})
        out.zero_()        # (the capture goes on)
    graph.replay()
    torch.cuda.synchronize()
    assert bool((out == 0).all())
    st.check(st.attend(op, inputs=x))
    assert op.device_status() == 0


def test_refusals(pkg):
    from openvino_genai_b200 import GenaiB200Error
    op = pkg.LatentAttention(8, *LH.WIDE, BLOCK, torch.bfloat16)
    with pytest.raises(GenaiB200Error, match="unknown form"):
        op.reserve(10, 2, 3, "both")
    for sizes in ((-1, 2, 3), (1, -2, 3), (1, 2, -3)):
        with pytest.raises(GenaiB200Error, match="negative"):
            op.reserve(*sizes)
    op.reserve(0, 0, 0)
