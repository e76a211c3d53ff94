"""Latent attention on the GPU against its definition in 64 bits: the cache append, both forms of the attention, odd lengths, strides,
streams, bad metadata."""
import math
import pathlib

import numpy as np
import pytest
import torch

from tests import latent_harness as LH

pytestmark = pytest.mark.gpu


# ---- append ---------------------------------------------------------------------------------------------------------
def _appended(st, interleaved, positions=None, norm=True):
    """cache and rotated queries in 64 bits."""
    R, P, Dn, _ = st.sizes
    cache, w = st.cache.double(), st.norm_weight.double()
    q = st.query[..., Dn:].double()

    def rotate(x, pos):
        c, s = st.rope_table[pos].double().chunk(2, -1)
        if x.dim() == 3:
            c, s = c[:, None], s[:, None]
        if interleaved:
            a, b = x[..., 0::2], x[..., 1::2]
            return torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
        a, b = x[..., :P // 2], x[..., P // 2:]
        return torch.cat([a * c - b * s, b * c + a * s], -1)

    out = torch.empty_like(q)
    t = 0
    table, first = st.meta["block_indices"].numpy(), st.meta["block_indices_begins"].numpy()
    for s in range(len(st.new)):
        n = int(st.new[s])
        at = np.arange(int(st.past[s]), int(st.past[s]) + n)
        pos = torch.from_numpy(at) if positions is None else positions[t:t + n].long()
        x = st.latent[t:t + n].double()
        c = x[:, :R]
        if norm:
            c = c / torch.sqrt(c.square().mean(-1, keepdim=True) + 1e-6) * w
        page = torch.from_numpy(table[first[s] + at // st.bs].astype(np.int64))
        cache[page, torch.from_numpy(at % st.bs)] = torch.cat([c, rotate(x[:, R:], pos)], -1)
        out[t:t + n] = rotate(q[t:t + n], pos)
        t += n
    return cache, out


def _check_append(st, cache, query, want):
    """One rounding of a value that f32 arithmetic gives to some 2^-20 of the sum of its terms' magnitudes: half a unit in the last place, and
    2^-20 of the largest element (inputs are below 8)."""
    u = LH.UNIT[st.dtype]
    for got, exp in ((cache, want[0]), (query, want[1])):
        got = got.cpu().double()
        assert torch.equal(torch.isnan(got), torch.isnan(exp)), "a slot that holds no new token was written"
        ok = ~torch.isnan(exp)
        assert bool(((got - exp)[ok].abs() <= u * exp[ok].abs() + 8 * 2.0 ** -20).all())


@pytest.mark.parametrize("sizes", [LH.WIDE, LH.SMALL, LH.MIXED])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("heads", [1, 20, 128])
def test_append(pkg, sizes, dtype, interleaved, heads):
    st = LH.Step([0, 5, 31, 32, 100, 7], [1, 3, 1, 40, 0, 65], heads=heads, sizes=sizes, bs=32, dtype=dtype, seed=heads)
    x = st.append_inputs(interleaved=interleaved)
    out = torch.empty((st.tokens, heads, sizes[1]), dtype=LH.DTYPE[dtype], device="cuda")
    op = st.operator(pkg)
    op.append(x, {"query_rope": out})
    _check_append(st, x["cache"], out, _appended(st, interleaved))
    assert op.device_status() == 0


@pytest.mark.parametrize("bs", [16, 32, 64])
@pytest.mark.parametrize("rows", [1, 3, 300])
def test_append_decode_rows(pkg, bs, rows):
    st = LH.Step(np.arange(rows) * 7 % 131, np.ones(rows, np.int64), heads=8, bs=bs, seed=rows)
    x = st.append_inputs()
    op = st.operator(pkg)
    out = torch.empty((rows, 8, 64), dtype=torch.bfloat16, device="cuda")
    op.append(x, {"query_rope": out})
    _check_append(st, x["cache"], out, _appended(st, False))


def test_append_in_place_with_positions_and_without_norm(pkg):
    """The queries are turned where they are, positions come from a tensor, the latent is written as it is; strides are a wider tensor's."""
    st = LH.Step([4, 0, 60], [5, 17, 1], heads=5, sizes=LH.SMALL, bs=16, dtype="f16", seed=9)
    positions = torch.arange(st.tokens, dtype=torch.int32).flip(0)
    x = st.append_inputs(positions=positions.cuda(), norm_weight=None)
    wide = torch.full((st.tokens, 256 + 32 + 24), 7.0, dtype=torch.float16, device="cuda")
    wide[:, :288] = st.latent.cuda()
    x["latent"] = wide[:, :288]
    whole = x["query_rope"]
    st.operator(pkg).append(x, {"query_rope": whole})
    _check_append(st, x["cache"], whole, _appended(st, False, positions, norm=False))
    assert torch.equal(x["query_nope"].cpu(), st.query[..., :64]) and bool((wide[:, 288:] == 7.0).all())


def test_append_without_queries(pkg):
    st = LH.Step([4, 0], [5, 17], seed=2)
    x = st.append_inputs()
    x.pop("query_rope")
    st.operator(pkg).append(x)
    _check_append(st, x["cache"], st.query[..., 128:], (_appended(st, False)[0], st.query[..., 128:].double()))


def test_append_then_attend(pkg):
    """A prompt in two chunks, then a token: the cache that append writes is the one that attend reads."""
    from openvino_genai_b200 import LatentAttention
    R, P, Dn, Dv = LH.WIDE
    H, bs, L = 8, 16, 90
    st = LH.Step([0], [L], heads=H, bs=bs, seed=4)
    op = LatentAttention(H, R, P, Dn, Dv, bs, torch.bfloat16)
    cache = op.allocate_cache(len(st.meta["block_indices"]) + 3)
    want_cache, turned = _appended(st, False)
    st.query[..., Dn:] = turned.to(torch.bfloat16)
    table, first = st.meta["block_indices"].long(), 0
    st.context = [want_cache[table].reshape(-1, R + P)[:L].to(torch.bfloat16)]
    want = st.expected()
    raw = LH.Step([0], [L], heads=H, bs=bs, seed=4)
    for lo, hi, form in ((0, 50, "expanded"), (50, 89, "auto"), (89, 90, "auto")):
        meta = {"past_lens": [lo], "subsequence_begins": [0, hi - lo], "block_indices_begins": [0, len(table)]}
        x = {k: torch.tensor(v, dtype=torch.int32, device="cuda") for k, v in meta.items()}
        q, up = raw.query[lo:hi].cuda(), raw.up.cuda()
        x.update(block_indices=st.meta["block_indices"].cuda(), cache=cache, latent=raw.latent[lo:hi].cuda(), norm_weight=raw.norm_weight.cuda(),
                 norm_eps=1e-6, rope_table=raw.rope_table.cuda(), query_nope=q[..., :Dn], query_rope=q[..., Dn:], key_up=up[:, :Dn], value_up=up[:, Dn:])
        op.append(x, {"query_rope": x["query_rope"]})
        out = torch.empty((hi - lo, H * Dv), dtype=torch.bfloat16, device="cuda")
        op.attend(x, {"output": out}, form=form)
        part = LH.Step([lo], [hi - lo], heads=H, bs=bs)
        part.check(out.cpu(), want[lo:hi])
    assert op.device_status() == 0


# ---- attention ------------------------------------------------------------------------------------------------------
EDGES = [0, 1, 14, 15, 16, 31, 32, 62, 63, 64, 65, 127, 128, 191, 200, 255, 256, 511, 1000]


@pytest.mark.parametrize("sizes", [LH.WIDE, LH.SMALL, LH.MIXED])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("bs", [16, 32, 64])
def test_decode_rows(pkg, sizes, dtype, bs):
    st = LH.Step(EDGES, [1] * len(EDGES), heads=16, sizes=sizes, bs=bs, dtype=dtype, seed=bs)
    op = st.operator(pkg)
    st.check(st.attend(op, "absorbed"))
    assert op.device_status() == 0


@pytest.mark.parametrize("heads", [1, 3, 8, 20, 40, 64, 65, 96, 128, 200])
def test_heads(pkg, heads):
    st = LH.Step([70, 0, 300, 63], [1, 4, 2, 1], heads=heads, seed=heads)
    op = st.operator(pkg)
    want = st.expected()
    st.check(st.attend(op, "absorbed"), want)
    st.check(st.attend(op, "expanded"), want)
    assert op.device_status() == 0


@pytest.mark.parametrize("form", ["absorbed", "expanded", "auto"])
@pytest.mark.parametrize("sizes,dtype,bs", [(LH.WIDE, "bf16", 64), (LH.SMALL, "f16", 16), (LH.MIXED, "bf16", 32)])
def test_drafts_prompts_and_empty_sequences(pkg, form, sizes, dtype, bs):
    past = [0, 37, 0, 512, 90, 0, 5, 128, 700, 0]
    new = [1, 5, 0, 1, 130, 300, 0, 128, 17, 257]
    st = LH.Step(past, new, heads=12, sizes=sizes, bs=bs, dtype=dtype, seed=3)
    op = st.operator(pkg)
    st.check(st.attend(op, form))
    assert op.device_status() == 0


@pytest.mark.parametrize("form", ["absorbed", "expanded"])
def test_long_context(pkg, form):
    st = LH.Step([20011, 3], [2, 1], heads=8, bs=64, seed=5)
    st.check(st.attend(st.operator(pkg), form))


@pytest.mark.parametrize("rows", [2, 40, 600])
def test_many_rows(pkg, rows):
    rng = np.random.default_rng(rows)
    st = LH.Step(rng.integers(0, 200, rows), np.ones(rows, np.int64), heads=6, sizes=LH.SMALL, bs=16, dtype="f16", seed=rows)
    st.check(st.attend(st.operator(pkg), "auto"))


@pytest.mark.parametrize("form", ["absorbed", "expanded"])
def test_scale_and_growing_maxima(pkg, form):
    """Logits whose maximum grows along the context (later rows are larger), with a scale of the caller's."""
    st = LH.Step([300, 700], [1, 60], heads=4, sizes=LH.MIXED, bs=32, dtype="f16", seed=8)
    for rows in st.context:
        rows *= torch.linspace(0.01, 1.5, len(rows))[:, None].to(rows.dtype)
    table, first = st.meta["block_indices"].long(), st.meta["block_indices_begins"].tolist()
    for s, rows in enumerate(st.context):
        pos = torch.arange(len(rows))
        st.cache[table[first[s] + pos // st.bs], pos % st.bs] = rows
    x = st.device_inputs()
    x["scale"] = 0.09
    st.check(st.attend(st.operator(pkg), form, x), st.expected(0.09))


@pytest.mark.parametrize("form", ["absorbed", "expanded"])
def test_strides_of_other_tensors(pkg, form):
    """Queries and weights as views of wider tensors, with the nope and the rope part in tensors of their own."""
    st = LH.Step([33, 0, 129], [1, 70, 2], heads=6, sizes=LH.MIXED, bs=16, seed=6)
    R, P, Dn, Dv = st.sizes
    x = st.device_inputs()
    qn = torch.full((st.tokens, 6, Dn + 40), math.nan, dtype=torch.bfloat16, device="cuda")
    qr = torch.full((6, st.tokens, P + 8), math.nan, dtype=torch.bfloat16, device="cuda")
    qn[..., 8:8 + Dn] = x["query_nope"]
    qr[..., :P] = x["query_rope"].transpose(0, 1)
    ku = torch.full((6, Dn + 3, R), math.nan, dtype=torch.bfloat16, device="cuda")
    ku[:, 1:1 + Dn] = x["key_up"]
    x.update(query_nope=qn[..., 8:8 + Dn], query_rope=qr[..., :P].transpose(0, 1), key_up=ku[:, 1:1 + Dn], value_up=x["value_up"].contiguous())
    st.check(st.attend(st.operator(pkg), form, x))


@pytest.mark.parametrize("form", ["absorbed", "expanded", "auto"])
def test_another_stream_and_repeated_calls(pkg, form):
    """Two steps of different shapes in turn on a side stream: nothing of one call is left in the next."""
    a = LH.Step([200, 77], [1, 90], heads=10, seed=1)
    b = LH.Step([5, 900, 64, 2], [3, 1, 1, 33], heads=10, seed=2)
    op = a.operator(pkg)
    side = torch.cuda.Stream()
    xs = [s.device_inputs() for s in (a, b)]
    outs = []
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for k in range(6):
            s = (a, b)[k % 2]
            out = torch.full((s.tokens, 10 * 128), math.nan, dtype=torch.bfloat16, device="cuda")
            op.attend(xs[k % 2], {"output": out}, form=form)
            outs.append(out)
    side.synchronize()
    want = [a.expected(), b.expected()]
    for k, out in enumerate(outs):
        (a, b)[k % 2].check(out.cpu(), want[k % 2])
        assert torch.equal(out, outs[k % 2]), "the same inputs gave other bits"


@pytest.mark.parametrize("form", ["absorbed", "expanded"])
def test_offsets_beyond_32_bits(pkg, form):
    """Blocks behind the first 2^32 bytes and 2^31 elements of the cache."""
    st = LH.Step([100, 30], [1, 9], heads=4, bs=64, seed=7)
    pool = (1 << 32) // (64 * 576 * 2) * 2 + 50
    x = st.device_inputs()
    small = x["cache"]
    x["cache"] = torch.empty((pool, 64, 576), dtype=torch.bfloat16, device="cuda")
    x["cache"][pool - len(small):] = small
    x["block_indices"] = x["block_indices"] + (pool - len(small))
    st.check(st.attend(st.operator(pkg), form, x))
    y = st.append_inputs(cache=x["cache"], block_indices=x["block_indices"])
    out = torch.empty((st.tokens, 4, 64), dtype=torch.bfloat16, device="cuda")
    st.operator(pkg).append(y, {"query_rope": out})
    _check_append(st, x["cache"][pool - len(small):], out, _appended(st, False))


# ---- bad metadata ---------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("sizes,dtype,bs", [(LH.WIDE, "bf16", 64), (LH.SMALL, "f16", 16), (LH.MIXED, "bf16", 32)])
@pytest.mark.parametrize("heads,past,new", [(1, [9000], [1]), (3, [2500, 0, 1300, 5000], [300, 200, 129, 1]), (2, [4096 - 256, 4000], [256, 257])])
def test_contexts_that_are_cut(pkg, heads, past, new, sizes, dtype, bs):
    """Few query tiles over long contexts: their pieces are computed apart and joined."""
    st = LH.Step(past, new, heads=heads, sizes=sizes, bs=bs, dtype=dtype, seed=21)
    op = st.operator(pkg)
    x = st.device_inputs()
    first = st.attend(op, "expanded", x)
    st.check(first)
    assert torch.equal(first, st.attend(op, "expanded", x))      # the pieces join in their order, whichever is last
    assert op.device_status() == 0


@pytest.mark.parametrize("form", ["absorbed", "expanded", "auto"])
def test_operators_of_several_sizes_take_turns(pkg, form):
    steps = [LH.Step([70, 200], [1, 90], heads=4, sizes=sizes, bs=32, seed=7) for sizes in (LH.WIDE, LH.SMALL, LH.MIXED)]
    ops = [st.operator(pkg) for st in steps]
    for _ in range(2):
        for st, op in zip(steps, ops):
            st.check(st.attend(op, form))
            assert op.device_status() == 0


@pytest.mark.parametrize("heads,past,new", [(32, [120000], [200]), (24, [90000, 40000, 3], [300, 5, 40])])
def test_scratch_of_several_passes(pkg, heads, past, new):
    """Keys and values of these contexts do not fit the scratch at once: the heads are served in passes, their contexts cut in each.  Each form is within
    2 u of the definition, so the two are within 4 u of one another."""
    st = LH.Step(past, new, heads=heads, bs=64, seed=3)
    op = st.operator(pkg)
    x = st.device_inputs()
    absorbed = st.attend(op, "absorbed", x).double()
    before = op.launch_count()
    expanded = st.attend(op, "expanded", x)
    assert op.launch_count() - before == 5      # the plan, two passes of two
    assert float((expanded.double() - absorbed).norm() / absorbed.norm()) < 4 * LH.UNIT["bf16"]
    assert torch.equal(expanded, st.attend(op, "expanded", x)) and op.device_status() == 0


def test_example_layer():
    """The layer of integration/latent_layer.py over mixed steps.  Seven roundings to bfloat16 (2^-9 each) lie between its input and its output:
    projections, rotation or norm, q~ or keys and values, weights, output, projection."""
    import importlib.util
    spec = importlib.util.spec_from_file_location("latent_layer", pathlib.Path(__file__).resolve().parents[1] / "integration" / "latent_layer.py")
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    assert example.main() < 7 * 2.0 ** -9


BAD_INDEX, BAD_BEGINS, BAD_PAST, BAD_ROTATION = 1, 2, 4, 8


@pytest.mark.parametrize("form", ["absorbed", "expanded", "auto"])
@pytest.mark.parametrize("what,bit", [("index", BAD_INDEX), ("begins", BAD_BEGINS), ("past", BAD_PAST), ("short table", BAD_PAST)])
def test_bad_metadata_is_reported_and_other_sequences_are_served(pkg, form, what, bit):
    st = LH.Step([40, 90, 10], [1, 70, 2], heads=6, bs=16, seed=3)
    op = st.operator(pkg)
    x = st.device_inputs()
    bad = 1
    if what == "index":
        x["block_indices"][int(x["block_indices_begins"][1]) + 2] = 1 << 20
    elif what == "begins":
        x["block_indices_begins"][2] = 10 ** 6
        bad = None   # both of its neighbours
    elif what == "past":
        x["past_lens"][1] = -1
    else:
        x["past_lens"][1] = 10 ** 6
    out = st.attend(op, form, x)
    assert op.device_status() & bit
    assert op.device_status() == 0
    st.check(torch.where(torch.isnan(out), torch.zeros_like(out), out) if bad is None else out, rows=[0, 2] if bad else [0])


@pytest.mark.parametrize("form", ["absorbed", "expanded"])
@pytest.mark.parametrize("what", ["subsequence_begins", "block_indices_begins"])
def test_falling_prefix_sums_write_nothing(pkg, form, what):
    """Sequences that are given the same tokens, or the same blocks, several times over: more rows in all than the step's workspace has."""
    st = LH.Step([200, 0, 200, 0, 200], [40, 0, 40, 0, 40], heads=6, bs=16, seed=4)
    op = st.operator(pkg)
    x = st.device_inputs()
    last = int(x[what][-1])
    x[what].copy_(torch.tensor([0, last, 0, last, 0, last], dtype=torch.int32))
    x["past_lens"].fill_(0 if what == "subsequence_begins" else last * 16 - 40)
    if what == "block_indices_begins" and form == "absorbed":      # (its workspace goes by the tokens only: the sequences that are left are served)
        st.attend(op, form, x)
    else:
        assert bool(torch.isnan(st.attend(op, form, x)).all())
    assert op.device_status() & BAD_BEGINS


def test_append_reports_positions_outside_the_table_and_bad_blocks(pkg):
    st = LH.Step([4, 6], [3, 2], heads=3, seed=2)
    x = st.append_inputs(rope_table=st.rope_table[:7].contiguous().cuda())
    x["block_indices"][0] = -1
    op = st.operator(pkg)
    out = torch.zeros((5, 3, 64), dtype=torch.bfloat16, device="cuda")
    op.append(x, {"query_rope": out})
    assert op.device_status() == BAD_INDEX | BAD_ROTATION
    want = _appended(st, False)[1]
    assert bool((out[4] == 0).all()) and float((out[:4].cpu().double() - want[:4]).norm() / want[:4].norm()) < LH.UNIT["bf16"]


# ---- refusals -------------------------------------------------------------------------------------------------------
def test_refusals(pkg):
    from openvino_genai_b200 import GenaiB200Error, LatentAttention
    for bad in ({"latent_size": 384}, {"rope_size": 48}, {"nope_size": 96}, {"value_size": 32}, {"block_size": 8}, {"num_heads": 0},
                {"dtype": torch.float32}):
        args = {"num_heads": 4, "latent_size": 512, "rope_size": 64, "nope_size": 128, "value_size": 128, "block_size": 16, **bad}
        with pytest.raises(GenaiB200Error):
            LatentAttention(**args)
    st = LH.Step([3], [2], heads=4, seed=1)
    op = st.operator(pkg)
    good = st.append_inputs()
    out = {"output": torch.empty((2, 512), dtype=torch.bfloat16, device="cuda")}
    turned = {"query_rope": torch.empty((2, 4, 64), dtype=torch.bfloat16, device="cuda")}
    op.append(good, turned)
    op.attend(good, out)

    def refuses(what, call, text):
        with pytest.raises(GenaiB200Error, match=text):
            call({**good, **what})

    attend, append = lambda x: op.attend(x, out), lambda x: op.append(x, turned)
    refuses({"query_nope": good["query_nope"].half()}, attend, "query_nope")
    refuses({"query_nope": good["query_nope"].cpu()}, attend, "query_nope")
    refuses({"query_rope": good["query_rope"][:1]}, attend, "query_rope")
    refuses({"key_up": good["key_up"][:, ::2]}, attend, "key_up")
    refuses({"key_up": torch.empty((4, 256, 512), dtype=torch.bfloat16, device="cuda")[:, ::2]}, attend, "rows have to be contiguous")
    refuses({"cache": good["cache"].transpose(0, 1)}, attend, "cache")
    refuses({"past_lens": good["past_lens"].long()}, attend, "past_lens")
    refuses({"block_indices_begins": good["block_indices"][:1]}, attend, "num_sequences")
    wide = torch.empty((2, 4, 132), dtype=torch.bfloat16, device="cuda")
    refuses({"query_nope": wide[..., :128]}, attend, "multiple of 8")
    flat = torch.empty(2 * 4 * 128 + 8, dtype=torch.bfloat16, device="cuda")
    refuses({"query_nope": flat[4:4 + 1024].view(2, 4, 128)}, attend, "aligned")
    with pytest.raises(GenaiB200Error, match="form"):
        op.attend(good, out, form="both")
    with pytest.raises(GenaiB200Error, match="output"):
        op.attend(good, {"output": torch.empty((3, 512), dtype=torch.bfloat16, device="cuda")})
    refuses({"rope_table": good["rope_table"].half()}, append, "rope_table")
    refuses({"rope_table": good["rope_table"][:0]}, append, "rope_table")
    refuses({"latent": good["latent"][:, :512]}, append, "latent")
    refuses({"positions": torch.zeros(3, dtype=torch.int32, device="cuda")}, append, "positions")
    with pytest.raises(GenaiB200Error, match="output query_rope"):
        op.append(good, {})
    assert op.device_status() == 0


def test_no_tokens_and_no_sequences(pkg):
    st = LH.Step([3, 8], [0, 0], heads=4, seed=1)
    op = st.operator(pkg)
    before = op.launch_count()
    assert st.attend(op).shape == (0, 512)
    assert op.launch_count() == before
