"""Performance cases of latent attention: one cached vector a token, from which every head's key and value come.

A layer of such a model calls the framework twice a step: `LatentAttention.append` normalises the new tokens' latent vectors, rotates
their shared key part and the queries' rotated part and writes the paged cache; `LatentAttention.attend` attends over it, either in the
absorbed form (the up-projections moved to the query and the output: decode steps, drafted tokens), or in the expanded form (keys and values
of the context made per head: prompts), or each sequence in the form that suits it.  Lengths follow from the case alone (`layout` seeds
them); values and block tables follow from the seed.

With `own` false `run` computes the same in elementary torch operations in 32 bits; `exact` restates the definition in 64 bits.
"""
import functools
import math

import numpy as np
import torch

own = False

DEV = "cuda:0"
DTYPE = {"f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-6
THETA = 1e4


# ---- the cases -------------------------------------------------------------------------------------------------------
def _case(name, kind, **kw):
    case = {"kind": kind, "heads": 16, "latent": 512, "rope": 64, "nope": 128, "value": 128, "bs": 32, "dtype": "bf16",
            "decode": 0, "decode_new": 1, "past_lo": 0, "past_hi": 0, "chunks": 0, "chunk_lo": 0, "chunk_hi": 0, "chunk_past_hi": 0,
            "form": "absorbed", "interleaved": False, "layout": 1}
    case.update(kw)
    if name:
        case["name"] = name
    return case


def listed():
    return [
        # one user's chat, one token: the launch is all there is
        _case("append one token", "append", decode=1, past_lo=700, past_hi=700),
        # a full batch of decode rows of a wide layer
        _case("append batch 256x128", "append", heads=128, decode=256, past_lo=200, past_hi=4000, bs=64, interleaved=True),
        # a batch of ragged prompts
        _case("append prompts f16", "append", heads=32, dtype="f16", chunks=8, chunk_lo=900, chunk_hi=3100, bs=16),
        # one user's chat, one token over a short context: latency
        _case("absorbed one row", "attend", decode=1, past_lo=701, past_hi=701),
        # drafted tokens being checked: a few rows a sequence, masked among themselves
        _case("absorbed drafts 24x4", "attend", decode=24, decode_new=4, past_lo=300, past_hi=6000, layout=2),
        # a serving batch of a wide layer
        _case("absorbed batch 64x128", "attend", heads=128, decode=64, past_lo=512, past_hi=8192, bs=64, layout=3),
        # the small geometry, many rows, f16
        _case("absorbed small 96x40 f16", "attend", heads=40, latent=256, rope=32, nope=64, value=64, dtype="f16", decode=96,
              past_lo=64, past_hi=6000, layout=4),
        # one long document: the split of one row's context over the whole GPU
        _case("absorbed long 120k", "attend", heads=128, decode=1, past_lo=120011, past_hi=120011, bs=64, layout=5),
        # one short prompt: latency of the expanded form
        _case("expanded one prompt", "attend", form="expanded", chunks=1, chunk_lo=333, chunk_hi=333, layout=6),
        # ragged prompts, some behind a cached prefix
        _case("expanded prompts 4x32", "attend", form="expanded", heads=32, chunks=4, chunk_lo=1100, chunk_hi=2048, chunk_past_hi=2048, layout=7),
        # chunks of long prompts, the small geometry
        _case("expanded chunks small f16", "attend", form="expanded", heads=40, latent=256, rope=32, nope=64, value=64, dtype="f16",
              chunks=5, chunk_lo=256, chunk_hi=512, chunk_past_hi=7000, bs=16, layout=8),
        # a mixed step: decode rows beside prompt chunks, each sequence in the form that suits it
        _case("mixed step 40+3", "attend", form="auto", decode=40, past_lo=256, past_hi=4000, chunks=3, chunk_lo=200, chunk_hi=512,
              chunk_past_hi=2000, layout=9),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    most = {}
    for c in listed():
        k = (c["kind"], c["form"])
        w = work(c)
        most[k] = tuple(max(a, b) for a, b in zip(most.get(k, (0, 0)), (w["bytes"], w["flops"])))
    while True:
        small = rng.random() < 0.35
        c = _case(None, rng.choice(["append", "attend", "attend", "attend"]), heads=rng.choice([8, 12, 16, 20, 32, 40, 64, 96, 128]),
                  dtype=rng.choice(["bf16", "bf16", "f16"]), bs=rng.choice([16, 32, 64]), layout=rng.randrange(1, 1 << 20))
        if small:
            c.update(latent=256, rope=32, nope=64, value=64)
        if c["kind"] == "append":
            c["interleaved"] = rng.random() < 0.5
            if rng.random() < 0.5:
                c.update(decode=_log(rng, 1, 256), past_hi=_log(rng, 1, 8000))
            else:
                c.update(chunks=rng.randint(1, 8), chunk_lo=1, chunk_hi=_log(rng, 2, 3000), chunk_past_hi=rng.choice([0, 500]))
        else:
            c["form"] = rng.choice(["absorbed", "absorbed", "expanded", "auto"])
            if c["form"] != "expanded":
                c.update(decode=_log(rng, 1, 96), past_hi=_log(rng, 16, 40000))
                c["past_lo"] = c["past_hi"] // rng.randint(1, 12)
                if c["form"] == "absorbed":
                    c["decode_new"] = rng.choice([1, 1, 1, 2, 5])
            if c["form"] != "absorbed":
                c.update(chunks=rng.randint(1, 5), chunk_hi=_log(rng, 16, 2048), chunk_past_hi=rng.choice([0, 100, 3000]))
                c["chunk_lo"] = max(1, c["chunk_hi"] // rng.randint(1, 4))
        past, new = _lengths(c)
        top = most[(c["kind"], c["form"])]
        w = work(c)
        ahead = len(new) * int(new.max()) * int((past + new).max()) * c["heads"]     # what a padded batch of scores holds
        if w["bytes"] <= top[0] and w["flops"] <= top[1] and ahead < 1.2e9:
            return c


def _lengths(case):
    rng = np.random.default_rng(case["layout"])
    d, c = case["decode"], case["chunks"]
    past = np.concatenate([rng.integers(case["past_lo"], case["past_hi"] + 1, size=d), rng.integers(0, case["chunk_past_hi"] + 1, size=c)])
    new = np.concatenate([np.full(d, case["decode_new"]), rng.integers(case["chunk_lo"], max(case["chunk_lo"], case["chunk_hi"]) + 1, size=c)])
    return past.astype(np.int64), new.astype(np.int64)


def _absorbed(case, new):
    """Which sequences a mixed step counts as decode rows."""
    return new <= case["decode_new"] if case["form"] == "auto" else np.full(len(new), case["form"] == "absorbed")


def work(case):
    past, new = _lengths(case)
    H, R, P, Dn, Dv = case["heads"], case["latent"], case["rope"], case["nope"], case["value"]
    tokens, context = int(new.sum()), past + new
    if case["kind"] == "append":
        return {"bytes": tokens * (4 * (R + P) + 4 * H * P + 4 * P) + 2 * R, "flops": tokens * (4 * R + 3 * P * (1 + H))}
    pairs = new * past + new * (new + 1) // 2
    ab = _absorbed(case, new)
    flops = int((pairs * ab).sum()) * H * 2 * (2 * R + P) + int((new * ab).sum()) * H * 2 * R * (Dn + Dv)
    flops += int((pairs * ~ab).sum()) * H * 2 * (Dn + P + Dv) + int((context * ~ab).sum()) * H * 2 * R * (Dn + Dv)
    return {"bytes": int(context.sum()) * 2 * (R + P) + 2 * H * (Dn + Dv) * R + tokens * 2 * H * (Dn + P + Dv), "flops": flops}


# ---- inputs ----------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    past, new = _lengths(case)
    bs, H, R, P, Dn, Dv = case["bs"], case["heads"], case["latent"], case["rope"], case["nope"], case["value"]
    dt = DTYPE[case["dtype"]]
    blocks = (past + new + bs - 1) // bs
    total = int(blocks.sum())
    pool = total + total // 10 + 1
    rng = np.random.default_rng(int(seed) + 7)
    gen = torch.Generator(device=DEV)
    gen.manual_seed(int(seed) * 7919 + 11)
    rnd = lambda *shape: torch.randn(shape, generator=gen, device=DEV)
    i32 = lambda a: torch.from_numpy(np.ascontiguousarray(a).astype(np.int32)).to(DEV)
    begins = lambda n: i32(np.concatenate([[0], np.cumsum(n)]))
    tokens = int(new.sum())
    s = {"case": dict(case), "cache": rnd(pool, bs, R + P).to(dt), "past_lens": i32(past), "subsequence_begins": begins(new),
         "block_indices": i32(rng.permutation(pool)[:total]), "block_indices_begins": begins(blocks),
         "max_context_len": int((past + new).max()), "max_new": int(new.max()),
         "query": rnd(tokens, H, Dn + P).to(dt)}
    if case["kind"] == "append":
        s["latent"] = rnd(tokens, R + P).to(dt)
        s["norm_weight"] = (1 + 0.1 * rnd(R)).to(dt)
        angle = np.arange(s["max_context_len"])[:, None] * np.power(THETA, -np.arange(P // 2) * 2.0 / P)[None, :]
        s["rope_table"] = torch.from_numpy(np.concatenate([np.cos(angle), np.sin(angle)], 1).astype(np.float32)).to(DEV)
        s["query_rope"] = torch.empty((tokens, H, P), dtype=dt, device=DEV)
    else:
        s["up"] = (rnd(H, Dn + Dv, R) / math.sqrt(R)).to(dt)     # the model's weight: [key rows | value rows] of each head
        s["output"] = torch.empty((tokens, H * Dv), dtype=dt, device=DEV)
    return s


# ---- the framework's calls -------------------------------------------------------------------------------------------
@functools.lru_cache(maxsize=None)
def _layer(heads, latent, rope, nope, value, bs, dtype):
    """The operator object of a layer, which a program makes once and keeps over its steps."""
    import __graft_entry__ as entry   # the package folder has a dot in its name: this loads it as `openvino_genai_b200`
    return entry.load_package().LatentAttention(heads, latent, rope, nope, value, bs, DTYPE[dtype])


def _run_own(s):
    case = s["case"]
    op = _layer(*(case[k] for k in ("heads", "latent", "rope", "nope", "value", "bs", "dtype")))
    inputs = {k: s[k] for k in ("cache", "past_lens", "subsequence_begins", "block_indices", "block_indices_begins")}
    Dn = case["nope"]
    if case["kind"] == "append":
        inputs.update(latent=s["latent"], norm_weight=s["norm_weight"], norm_eps=EPS, query_rope=s["query"][..., Dn:],
                      rope_table=s["rope_table"], interleaved=case["interleaved"])
        op.append(inputs, {"query_rope": s["query_rope"]})
        return {"cache": s["cache"], "query_rope": s["query_rope"]}
    inputs.update(query_nope=s["query"][..., :Dn], query_rope=s["query"][..., Dn:], key_up=s["up"][:, :Dn], value_up=s["up"][:, Dn:])
    op.attend(inputs, {"output": s["output"]}, form=case["form"])
    return {"output": s["output"]}


# ---- the plain form --------------------------------------------------------------------------------------------------
def _rotate(x, cos, sin, interleaved):
    if interleaved:
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    a, b = x.chunk(2, -1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _run_append(s):
    case = s["case"]
    R, P, Dn, bs = case["latent"], case["rope"], case["nope"], case["bs"]
    dt = s["cache"].dtype
    begins = s["subsequence_begins"].long()
    t = torch.arange(s["latent"].shape[0], device=DEV)
    seq = torch.searchsorted(begins, t, right=True) - 1
    pos = s["past_lens"].long()[seq] + t - begins[seq]
    page = s["block_indices"].long()[s["block_indices_begins"].long()[seq] + pos // bs]
    cos, sin = s["rope_table"][pos].chunk(2, -1)
    x = s["latent"].float()
    c = x[:, :R]
    c = c * torch.rsqrt((c * c).mean(-1, keepdim=True) + EPS) * s["norm_weight"].float()
    s["cache"][page, pos % bs] = torch.cat([c, _rotate(x[:, R:], cos, sin, case["interleaved"])], -1).to(dt)
    s["query_rope"] = _rotate(s["query"][..., Dn:].float(), cos[:, None], sin[:, None], case["interleaved"]).to(dt)
    return {"cache": s["cache"], "query_rope": s["query_rope"]}


def _run_attend(s):
    case = s["case"]
    R, P, Dn, Dv, H, bs = case["latent"], case["rope"], case["nope"], case["value"], case["heads"], case["bs"]
    past, begins = s["past_lens"].long(), s["subsequence_begins"].long()
    B, N, L = past.numel(), s["max_new"], s["max_context_len"]
    i, j = torch.arange(N, device=DEV), torch.arange(L, device=DEV)
    new = begins[1:] - begins[:-1]
    row = (begins[:-1, None] + i).clamp_(max=s["query"].shape[0] - 1)                                    # [B, N]
    at = (s["block_indices_begins"].long()[:-1, None] + j // bs).clamp_(max=s["block_indices"].numel() - 1)
    kv = s["cache"][s["block_indices"].long()[at], j % bs].float()                                       # [B, L, R + P]
    q = s["query"].float()[row]                                                                          # [B, N, H, Dn + P]
    up = s["up"].float()
    seen = j <= (past[:, None] + i)[:, :, None]                                                          # [B, N, L]
    scale = 1.0 / math.sqrt(Dn + P)
    c, kr = kv[..., :R], kv[..., R:]
    if case["form"] == "expanded":
        k = torch.einsum("blr,hdr->bhld", c, up[:, :Dn])
        a = torch.einsum("bnhd,bhld->bhnl", q[..., :Dn], k) + torch.einsum("bnhd,bld->bhnl", q[..., Dn:], kr)
    else:
        qa = torch.cat([torch.einsum("bnhd,hdr->bnhr", q[..., :Dn], up[:, :Dn]), q[..., Dn:]], -1)
        a = torch.einsum("bnhr,blr->bhnl", qa, kv)
    a = torch.where(seen[:, None], a * scale, -math.inf)
    a = torch.exp(a - a.amax(-1, keepdim=True))
    a = a / a.sum(-1, keepdim=True)
    if case["form"] == "expanded":
        o = torch.einsum("bhnl,bhld->bnhd", a, torch.einsum("blr,hdr->bhld", c, up[:, Dn:]))
    else:
        o = torch.einsum("bnhr,hdr->bnhd", torch.einsum("bhnl,blr->bnhr", a, c), up[:, Dn:])
    s["output"] = o[i < new[:, None]].reshape(-1, H * Dv).to(s["query"].dtype)
    return {"output": s["output"]}


def run(state):
    if own:
        return _run_own(state)
    return _run_append(state) if state["case"]["kind"] == "append" else _run_attend(state)


# ---- the definition in 64 bits ---------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    past, new = _lengths(case)
    bs, H, R, P, Dn, Dv = case["bs"], case["heads"], case["latent"], case["rope"], case["nope"], case["value"]
    table, first = s["block_indices"].long(), s["block_indices_begins"].tolist()
    query = s["query"].double()
    cache = s["cache"].double()
    if case["kind"] == "append":
        w, rope = s["norm_weight"].double(), s["rope_table"].double()
        # a rotation by an angle is a product of complex numbers
        pair = lambda x: torch.complex(x[..., 0::2].contiguous(), x[..., 1::2].contiguous()) if case["interleaved"] else \
            torch.complex(x[..., :P // 2].contiguous(), x[..., P // 2:].contiguous())
        flat = lambda z: torch.view_as_real(z).flatten(-2) if case["interleaved"] else torch.cat([z.real, z.imag], -1)
        turned = torch.empty((int(new.sum()), H, P), dtype=torch.float64, device=DEV)
        t = 0
        for b in range(len(past)):
            n, p = int(new[b]), int(past[b])
            z = rope[p:p + n]
            z = torch.complex(z[:, :P // 2].contiguous(), z[:, P // 2:].contiguous())
            x = s["latent"][t:t + n].double()
            norm = torch.sqrt(x[:, :R].square().sum(-1, keepdim=True) / R + EPS)
            pos = torch.arange(p, p + n, device=DEV)
            cache[table[first[b] + pos // bs], pos % bs] = torch.cat([x[:, :R] / norm * w, flat(pair(x[:, R:]) * z)], -1)
            turned[t:t + n] = flat(pair(query[t:t + n, :, Dn:]) * z[:, None])
            t += n
        return {"cache": cache, "query_rope": turned}
    up = s["up"].double()
    out = torch.empty((int(new.sum()), H, Dv), dtype=torch.float64, device=DEV)
    t = 0
    for b in range(len(past)):
        n, p = int(new[b]), int(past[b])
        kv = cache[table[first[b]:first[b + 1]]].reshape(-1, R + P)[:p + n]
        hidden = torch.arange(p + n, device=DEV)[None, :] > p + torch.arange(n, device=DEV)[:, None]
        few = max(1, int(4e8 // ((p + n) * max(n, Dn + Dv))))
        for h in range(0, H, few):
            g = slice(h, min(H, h + few))
            e = torch.matmul(kv[None, :, :R], up[g].transpose(1, 2))                                     # [h, L, Dn + Dv]
            q = query[t:t + n, g].transpose(0, 1)                                                        # [h, n, Dn + P]
            a = torch.matmul(q[..., :Dn], e[..., :Dn].transpose(1, 2)) + torch.matmul(q[..., Dn:], kv[:, R:].T)
            a = torch.softmax((a / math.sqrt(Dn + P)).masked_fill_(hidden, -math.inf), -1)
            out[t:t + n, g] = torch.matmul(a, e[..., Dn:]).transpose(0, 1)
        t += n
    return {"output": out.reshape(-1, H * Dv)}
