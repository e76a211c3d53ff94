"""Performance cases of attention over the paged cache under masks, and of what a step with a tree of drafted tokens does behind it.

  window  `PagedAttentionExtension.evaluate` with `sliding_window` and `sink_tokens`: a row at position p sees the cached positions above
          p - W and the first few of its sequence; single tokens, prompts, and steps that hold both.
  tree    the same call with `tree_parents`: a sequence's new tokens are a tree of drafts, a row sees the cache, its ancestors and itself.
          A layer with a sliding window takes both.
  accept  `PagedAttentionExtension.tree_accept`: follows the sampled tokens down every tree, and moves the accepted tokens' keys and
          values of all layers to where the next step expects them.

Lengths and trees follow from the case alone (`layout` seeds them); values and block tables follow from the seed.  With `own` false `run`
computes the same in elementary torch operations in 32 bits; `exact` restates the definition in 64 bits.
"""
import functools
import math

import numpy as np
import torch

own = False

DEV = "cuda:0"
DTYPE = {"f16": torch.float16, "bf16": torch.bfloat16}
VOCAB = 128256
NONE = -2          # tree_parents of a sequence without a tree


# ---- the cases -------------------------------------------------------------------------------------------------------
def _case(name, kind, **kw):
    case = {"kind": kind, "hq": 32, "hkv": 8, "d": 128, "bs": 32, "act": "bf16", "cache": "bf16", "window": 0, "sinks": 0, "decode": 0, "past_lo": 0,
            "past_hi": 0, "chunks": 0, "chunk_lo": 0, "chunk_hi": 0, "chunk_past_hi": 0, "trees": 0, "tree_lo": 0, "tree_hi": 0, "layers": 0, "layout": 1}
    case.update(kw)
    if name:
        case["name"] = name
    return case


def listed():
    return [
        # one user's chat far beyond the window: a layer's call is a few microseconds of work
        _case("window one row", "window", decode=1, past_lo=9001, past_hi=9001, window=1024, sinks=4, layout=11),
        # the decode step of a served batch, u8 cache, some contexts still shorter than the window
        _case("window rows 64 u8", "window", cache="u8", decode=64, past_lo=512, past_hi=8192, window=4096, sinks=4, layout=12),
        # many rows through a layer of a short window, small heads and blocks, no sinks
        _case("window rows 256 short", "window", hq=64, d=64, bs=16, act="f16", cache="f16", decode=256, past_lo=40, past_hi=6000, window=128, layout=13),
        # fresh and continued prompts of ragged lengths, unquantised cache
        _case("window prompts ragged", "window", chunks=9, chunk_lo=37, chunk_hi=2048, chunk_past_hi=3000, window=1024, sinks=4, layout=14),
        # long chunks over contexts longer than the window, u8 cache, seven query heads a kv head
        _case("window prompts u8", "window", hq=28, hkv=4, cache="u8", chunks=3, chunk_lo=2000, chunk_hi=4096, chunk_past_hi=9000, window=4096, sinks=64, layout=15),
        # a step of an engine that schedules chunks beside single tokens
        _case("window mixed step", "window", act="f16", cache="u8", decode=40, past_lo=100, past_hi=12000, chunks=3, chunk_lo=200, chunk_hi=512,
              chunk_past_hi=4096, window=2048, sinks=16, layout=16),
        # one user's drafts over a conversation
        _case("tree one", "tree", trees=1, tree_lo=27, tree_hi=27, past_lo=4501, past_hi=4501, layout=21),
        # a batch of trees over served contexts, u8 cache
        _case("tree batch 32 u8", "tree", cache="u8", trees=32, tree_lo=48, tree_hi=64, past_lo=512, past_hi=8192, layout=22),
        # two long documents, more query rows a kv head than one product takes
        _case("tree long", "tree", hq=28, hkv=4, trees=2, tree_lo=61, tree_hi=61, past_lo=90001, past_hi=120001, layout=23),
        # trees through a layer with a sliding window
        _case("tree in a window", "tree", act="f16", cache="f16", trees=16, tree_lo=9, tree_hi=40, past_lo=300, past_hi=9000, window=1024, sinks=4, layout=24),
        # the drafts of one user are judged, two accepted or so, over all layers of a model
        _case("accept one", "accept", trees=1, tree_lo=27, tree_hi=27, past_lo=501, past_hi=501, layers=32, layout=31),
        # a batch of them, u8 cache
        _case("accept batch 64 u8", "accept", cache="u8", trees=64, tree_lo=48, tree_hi=64, past_lo=100, past_hi=400, layers=32, layout=32),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    layout = rng.randrange(1, 1 << 30)
    hq, hkv, d, bs = rng.choice([(32, 4, 64, 32), (32, 8, 128, 32), (28, 4, 128, 32), (64, 8, 128, 16), (64, 8, 64, 16)])
    act, cache = rng.choice([("bf16", "u8"), ("bf16", "bf16"), ("f16", "u8"), ("f16", "f16"), ("bf16", "bf16")])
    base = dict(hq=hq, hkv=hkv, d=d, bs=bs, act=act, cache=cache, layout=layout)
    window, sinks = _log_int(rng, 63, 4096), rng.choice([0, 1, 4, 16, 64])
    kind = rng.choice(["rows", "rows", "prompts", "mixed", "tree", "tree", "tree window", "accept"])
    if kind == "rows":
        n = _log_int(rng, 1, 128)
        hi = _log_int(rng, 100, 8192)
        return _case(None, "window", decode=n, past_lo=max(1, hi // rng.choice([1, 4, 16])), past_hi=hi, window=window, sinks=sinks, **base)
    if kind == "prompts":
        chunk = _log_int(rng, 17, 2048)
        n = max(1, min(6, _log_int(rng, 17, 4096) // chunk))
        return _case(None, "window", chunks=n, chunk_lo=max(2, chunk // rng.choice([1, 3])), chunk_hi=chunk, chunk_past_hi=rng.choice([0, _log_int(rng, 50, 8000)]),
                     window=window, sinks=sinks, **base)
    if kind == "mixed":
        chunk = _log_int(rng, 17, 400)
        return _case(None, "window", decode=_log_int(rng, 2, 40), past_lo=50, past_hi=_log_int(rng, 200, 8000), chunks=rng.randrange(1, 4), chunk_lo=max(2, chunk // 2),
                     chunk_hi=chunk, chunk_past_hi=_log_int(rng, 50, 4096), window=window, sinks=sinks, **base)
    nodes = _log_int(rng, 2, 100)
    if kind == "accept":
        hi = _log_int(rng, 10, 500)
        return _case(None, "accept", trees=_log_int(rng, 1, 48), tree_lo=max(1, nodes // rng.choice([1, 2])), tree_hi=nodes, past_lo=max(0, hi // 3), past_hi=hi,
                     layers=rng.choice([1, 4, 16, 32]), **base)
    n = _log_int(rng, 1, 24)
    hi = _log_int(rng, 64, 160000) // n + 64
    return _case(None, "tree", trees=n, tree_lo=max(1, nodes // rng.choice([1, 2])), tree_hi=nodes, past_lo=max(0, hi // rng.choice([1, 4])), past_hi=hi,
                 window=window if kind == "tree window" else 0, sinks=sinks if kind == "tree window" else 0, **base)


def _tree(rng, n):
    """Parents of a tree of n drafts: token 0 is the last token that is certain, -1 its parent; every later token follows one in front of it."""
    return np.array([-1] + [int(rng.integers((i - 1) // 4, (i - 1) // 2 + 1)) for i in range(1, n)], np.int32)


def _depth(parents):
    depth = np.zeros(len(parents), np.int64)
    for i, p in enumerate(parents):
        depth[i] = depth[p] + 1 if p >= 0 else 0
    return depth


def _layout(case):
    """Cached tokens and new tokens of every sequence, and its tree or None."""
    rng = np.random.default_rng(case["layout"])
    past = np.concatenate([rng.integers(0, case["chunk_past_hi"] + 1, case["chunks"]),
                           rng.integers(case["past_lo"], case["past_hi"] + 1, case["decode"] + case["trees"])]).astype(np.int64)
    new = np.concatenate([np.maximum(rng.integers(case["chunk_lo"], case["chunk_hi"] + 1, case["chunks"]), 1), np.ones(case["decode"], np.int64),
                          np.maximum(rng.integers(case["tree_lo"], case["tree_hi"] + 1, case["trees"]), 1)]).astype(np.int64)
    trees = [None] * (case["chunks"] + case["decode"]) + [_tree(rng, int(n)) for n in new[case["chunks"] + case["decode"]:]]
    return past, new, trees


def _accepted(rng, parents):
    """A path of the tree that ends where no place that it is moved to holds another of its tokens, so that a repeated call finds the same."""
    best = [0]
    for leaf in rng.permutation(len(parents)):
        path = [int(leaf)]
        while parents[path[-1]] >= 0:
            path.append(int(parents[path[-1]]))
        path = path[::-1]
        fits = [L for L in range(1, len(path) + 1) if all(p == k or p >= L for k, p in enumerate(path[:L]))]
        if len(path[:fits[-1]]) > len(best):
            best = path[:fits[-1]]
    return best


def _record(case):
    return case["bs"] * (case["d"] + 8) if case["cache"] == "u8" else case["bs"] * case["d"] * 2


def _row_bytes(case):
    return case["d"] + 8 if case["cache"] == "u8" else 2 * case["d"]


def work(case):
    past, new, trees = _layout(case)
    hq, hkv, d, W, S = case["hq"], case["hkv"], case["d"], case["window"], case["sinks"]
    tokens = int(new.sum())
    if case["kind"] == "accept":
        rng = np.random.default_rng(case["layout"] + 1)
        moved = sum(sum(p != k for k, p in enumerate(_accepted(rng, t))) for t in trees)
        return {"bytes": tokens * 20 + 20 * len(past) + moved * case["layers"] * 2 * 2 * hkv * _row_bytes(case), "flops": 0}
    cached, pairs = 0, 0
    for p, n, tree in zip(past.tolist(), new.tolist(), trees):
        depth = np.arange(n) if tree is None else _depth(tree)
        seen = np.full(n, p) if W == 0 else np.minimum(p, np.minimum(p, S) + np.maximum(0, p - np.maximum(p + depth - W + 1, min(p, S))))
        cached += int(seen.max())
        own_ = depth + 1 if W == 0 else np.minimum(depth + 1, W)
        pairs += int(seen.sum() + own_.sum())
    return {"bytes": (cached + tokens) * 2 * hkv * _row_bytes(case) + tokens * (2 * hq + 2 * hkv) * d * 2, "flops": 4 * hq * d * pairs}


# ---- inputs ----------------------------------------------------------------------------------------------------------
def _gen(seed, salt):
    g = torch.Generator(device=DEV)
    g.manual_seed((int(seed) * 1000003 + salt) & 0x7FFFFFFFFFFF)
    return g


def _cache(case, blocks, g, value):
    """Bytes of `blocks` cache blocks of N(0, 1) rows, in the operator's layout: [blocks, hkv, record]."""
    hkv, bs, d = case["hkv"], case["bs"], case["d"]
    out = torch.empty((blocks, hkv, _record(case)), dtype=torch.uint8, device=DEV)
    step = max(1, (1 << 27) // (hkv * bs * d))
    for b in range(0, blocks, step):
        x = torch.randn((min(step, blocks - b), hkv, bs, d), generator=g, device=DEV)
        if case["cache"] != "u8":
            out[b:b + step] = x.to(DTYPE[case["cache"]]).view(torch.uint8).flatten(2)
            continue
        q, scale, zp = _quantise(x)
        out[b:b + step] = torch.cat([(q.transpose(2, 3) if value else q).reshape(*q.shape[:2], bs * d), scale.view(torch.uint8), zp.view(torch.uint8)], 2)
    return out


def _quantise(x):
    """Bytes, scale and zero-point of the last dimension's rows, in the operator's documented steps of 32 bits."""
    mn, mx = x.amin(-1), x.amax(-1)
    scale = (mx - mn) / torch.full_like(mx, 255.0)      # (by a number torch would multiply with its reciprocal)
    scale = torch.where(scale > 0, scale, torch.ones_like(scale))
    zp, inv = -mn / scale, 1.0 / scale
    q = (x.double() * inv.double()[..., None] + zp.double()[..., None]).float()      # one rounding, as a fused multiply-add has
    return q.clamp(0, 255).round().to(torch.uint8), scale, zp


def prepare(case, seed):
    past, new, trees = _layout(case)
    bs, hkv, d, tokens = case["bs"], case["hkv"], case["d"], int(new.sum())
    rng = np.random.default_rng(int(seed) + 7)
    blocks = (past + new + bs - 1) // bs
    total = int(blocks.sum())
    pool = total + total // 10 + 1
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(DEV)
    i32 = lambda a: dev(np.asarray(a, np.int32))
    begins = lambda n: i32(np.concatenate([[0], np.cumsum(n)]))
    g = _gen(seed, 1)
    s = {"case": case, "max_new": int(new.max()), "past_lens": i32(past), "subsequence_begins": begins(new), "block_indices": i32(rng.permutation(pool)[:total]),
         "block_indices_begins": begins(blocks), "max_context_len": int((past + new).max())}
    if case["trees"]:
        s["tree_parents"] = i32(np.concatenate([np.full(int(n), NONE) if t is None else t for n, t in zip(new, trees)]))
    if case["kind"] != "accept":
        s["key_cache"], s["value_cache"] = _cache(case, pool, g, False), _cache(case, pool, g, True)
        rnd = lambda h: torch.randn((tokens, h * d), generator=g, device=DEV).to(DTYPE[case["act"]])
        s["query"], s["key"], s["value"] = rnd(case["hq"]), rnd(hkv), rnd(hkv)
        s["output"] = torch.empty_like(s["query"])
        # rows of the plain form's gathered keys: the sinks, then all from the first row's window on
        first = np.maximum(np.maximum(past - case["window"] + 1, 0), case["sinks"]) if case["window"] else np.full(len(past), case["sinks"])
        s["gathered"] = case["sinks"] + int(np.maximum(past + new - first, 0).max())
        return s
    s["key_caches"], s["value_caches"] = (_cache(case, case["layers"] * pool, g, v).unflatten(0, (case["layers"], pool)) for v in (False, True))
    draft, sampled = rng.integers(0, VOCAB, tokens), rng.integers(0, VOCAB, tokens)
    choice = np.random.default_rng(case["layout"] + 1)
    t, longest = 0, 1
    for n, tree in zip(new.tolist(), trees):
        path = _accepted(choice, tree)
        longest = max(longest, len(path))
        for a, b in zip(path, path[1:]):
            draft[t + b] = VOCAB + b                   # a sibling's token is another one
            sampled[t + a] = VOCAB + b
        sampled[t + path[-1]] = 2 * VOCAB
        t += n
    s["draft_tokens"], s["sampled_tokens"] = dev(draft), dev(sampled)
    B, s["max_path"] = len(past), longest + 2
    mk = lambda shape, dt: torch.empty(shape, dtype=dt, device=DEV)
    s["out"] = {"path": mk((B, s["max_path"]), torch.int32), "num_accepted": mk(B, torch.int32), "next_token": mk(B, torch.int64), "new_past_lens": mk(B, torch.int32)}
    s["closure"] = max(1, int(max(new)).bit_length())
    return s


# ---- the framework's calls -------------------------------------------------------------------------------------------
@functools.lru_cache(maxsize=None)
def _layer(hq, hkv, d, bs, act, cache):
    """The operator object of a geometry, which a program makes once and keeps over its steps."""
    import __graft_entry__ as entry   # the package folder has a dot in its name: this loads it as `openvino_genai_b200`
    return entry.load_package().PagedAttentionExtension(hq, hkv, d, bs, DTYPE[act], cache)


META = ("past_lens", "subsequence_begins", "block_indices", "block_indices_begins")


def _run_own(s):
    case = s["case"]
    op = _layer(*(case[k] for k in ("hq", "hkv", "d", "bs", "act", "cache")))
    inputs = {k: s[k] for k in META}
    if case["kind"] == "accept":
        inputs.update({k: s[k] for k in ("tree_parents", "draft_tokens", "sampled_tokens")}, key_caches=s["key_caches"].unbind(), value_caches=s["value_caches"].unbind())
        op.tree_accept(inputs, s["out"])
        return {**s["out"], "key_caches": s["key_caches"], "value_caches": s["value_caches"]}
    inputs.update({k: s[k] for k in ("query", "key", "value", "key_cache", "value_cache", "max_context_len")}, sliding_window=case["window"], sink_tokens=case["sinks"])
    if case["trees"]:
        inputs["tree_parents"] = s["tree_parents"]
    op.evaluate(inputs, {"output": s["output"]})
    return _attended(s)


def _attended(s):
    """The attention's outputs: the rows, and the caches that got the new tokens (bytes of records where they hold 8 bits with their scales)."""
    dt = DTYPE.get(s["case"]["cache"])
    kc, vc = (c if dt is None else c.view(dt) for c in (s["key_cache"], s["value_cache"]))
    return {"output": s["output"], "key_cache": kc, "value_cache": vc}


# ---- the plain form --------------------------------------------------------------------------------------------------
def _rows(case, cache, value):
    """View of cache bytes [..., hkv, record] as [..., hkv, slot, d] elements."""
    bs, d = case["bs"], case["d"]
    if case["cache"] != "u8":
        return cache.view(DTYPE[case["cache"]]).unflatten(-1, (bs, d))
    x = cache[..., :bs * d]
    return x.unflatten(-1, (d, bs)).transpose(-1, -2) if value else x.unflatten(-1, (bs, d))


def _params(case, cache):
    """View of a u8 cache's scales and zero-points: [..., hkv, 2, slot]."""
    return cache.view(torch.float32)[..., case["bs"] * case["d"] // 4:].unflatten(-1, (2, case["bs"]))


def _ancestors(parents, new, N, steps):
    """[B, N, N] whether a sequence's token i descends from token a, or is it; a sequence without a tree is a chain."""
    i = torch.arange(N, device=DEV)
    p = torch.where(parents == NONE, i - 1, parents)
    R = ((p[:, :, None] == i) | (i[:, None] == i)).float() * (i < new[:, None])[:, :, None]
    return functools.reduce(lambda R, _: (R @ R > 0).float(), range(steps), R) > 0


def _padded(s, x, fill):
    """[tokens] -> [B, N], and which of them are there."""
    begins = s["subsequence_begins"].long()
    i = torch.arange(s["max_new"], device=DEV)
    there = i < (begins[1:] - begins[:-1])[:, None]
    at = (begins[:-1, None] + i).clamp_(max=x.shape[0] - 1)
    return torch.where(there, x[at], fill), there, at


def _run_attention(s):
    case = s["case"]
    hq, hkv, d, bs, W, S = (case[k] for k in ("hq", "hkv", "d", "bs", "window", "sinks"))
    G = hq // hkv
    past, begins, first_block = s["past_lens"].long(), s["subsequence_begins"].long(), s["block_indices_begins"].long()
    table = s["block_indices"].long()
    B, N, tokens = past.numel(), s["max_new"], s["query"].shape[0]
    new = begins[1:] - begins[:-1]
    # the new tokens' rows go into the cache
    t = torch.arange(tokens, device=DEV)
    seq = torch.searchsorted(begins, t, right=True) - 1
    pos = past[seq] + t - begins[seq]
    blk, slot = table[first_block[seq] + pos // bs], pos % bs
    put = lambda cache, x, value: _rows(case, cache, value).transpose(1, 2).__setitem__((blk, slot), x)
    for cache, x, value in ((s["key_cache"], s["key"], False), (s["value_cache"], s["value"], True)):
        x = x.unflatten(-1, (hkv, d))
        if case["cache"] != "u8":
            put(cache, x.float().to(DTYPE[case["cache"]]), value)
        else:
            q, scale, zp = _quantise(x.float())
            put(cache, q, value)
            _params(case, cache).permute(0, 3, 1, 2)[blk, slot] = torch.stack([scale, zp], -1)
    # the keys and values that any row sees
    v = torch.arange(s["gathered"], device=DEV)
    low = (past - W + 1).clamp_(min=S) if W else torch.full_like(past, S)
    pos = torch.where(v < S, v, low[:, None] + v - S)                                                     # [B, L]
    here = pos < (past + new)[:, None]
    page = table[(first_block[:-1, None] + pos // bs).clamp_(max=table.numel() - 1)]
    slot = pos % bs

    def get(cache, value):
        x = _rows(case, cache, value).transpose(1, 2)[page, slot].float()                                 # [B, L, hkv, d]
        if case["cache"] == "u8":
            scale, zp = _params(case, cache).permute(0, 3, 1, 2)[page, slot].unbind(-1)
            x = (x - zp[..., None]) * scale[..., None]
        return x.permute(0, 2, 1, 3)

    k, val = get(s["key_cache"], False), get(s["value_cache"], True)
    # what a row sees of them
    parents, there, at = _padded(s, s["tree_parents"].long() if case["trees"] else torch.full((tokens,), NONE, device=DEV), NONE)
    anc = _ancestors(parents, new, N, s["max_new"].bit_length()) if case["trees"] else (torch.arange(N, device=DEV)[:, None] >= torch.arange(N, device=DEV)).expand(B, N, N)
    depth = anc.sum(-1) - 1
    p = past[:, None] + depth                                                                             # [B, N]
    a = pos - past[:, None]
    fresh = a >= 0
    a = a.clamp(0, N - 1)
    key_pos = torch.where(fresh, torch.gather(p, 1, a), pos)
    seen = ~fresh[:, None] | torch.gather(anc, 2, a[:, None].expand(B, N, -1))
    if W:
        seen = seen & ((key_pos[:, None] < S) | (key_pos[:, None] > p[:, :, None] - W))
    seen = seen & here[:, None]
    q = s["query"].float()[at].view(B, N, hkv, G, d).permute(0, 2, 3, 1, 4).reshape(B, hkv, G * N, d)
    x = torch.matmul(q, k.transpose(-1, -2)).view(B, hkv, G, N, -1) * (1.0 / math.sqrt(d))
    x = torch.where(seen[:, None, None], x, -math.inf)
    x = torch.exp(x - x.amax(-1, keepdim=True))
    x = x / x.sum(-1, keepdim=True)
    o = torch.matmul(x.view(B, hkv, G * N, -1), val).view(B, hkv, G, N, d).permute(0, 3, 1, 2, 4).reshape(B, N, hq * d)
    s["output"] = o[there].to(s["query"].dtype)
    return _attended(s)


def _run_accept(s):
    case = s["case"]
    bs, P = case["bs"], s["max_path"]
    past, begins, first_block = s["past_lens"].long(), s["subsequence_begins"].long(), s["block_indices_begins"].long()
    new = begins[1:] - begins[:-1]
    N, B = s["max_new"], past.numel()
    parents, there, _ = _padded(s, s["tree_parents"].long(), NONE)
    draft, _, _ = _padded(s, s["draft_tokens"], -1)
    sampled, _, _ = _padded(s, s["sampled_tokens"], -1)
    i = torch.arange(N, device=DEV)
    up = parents.clamp(min=0)
    right = (draft == torch.gather(sampled, 1, up)) & there & (parents >= 0)
    # the first of several children of one token with the sampled token
    same = (parents[:, :, None] == parents[:, None]) & right[:, None] & (i < i[:, None])
    right = (right & ~same.any(-1)) | (i == 0)
    anc = _ancestors(parents, new, N, s["closure"])
    good = (~anc | right[:, None]).all(-1) & there
    depth = anc.sum(-1) - 1
    good = good & (depth < P)
    count = good.sum(-1)
    path = torch.full((B, P + 1), -1, dtype=torch.int64, device=DEV).scatter_(1, torch.where(good, depth, P), i.expand(B, N))[:, :P]
    path = torch.where(torch.arange(P, device=DEV) < count[:, None], path, -1)
    last = torch.gather(path, 1, (count - 1)[:, None])
    out = {"path": path.int(), "num_accepted": count.int(), "next_token": torch.gather(sampled, 1, last)[:, 0], "new_past_lens": (past + count).int()}
    # the accepted tokens' rows move up
    k = torch.arange(P, device=DEV).expand(B, P)
    b, k = torch.nonzero((path >= 0) & (path != k), as_tuple=True)
    table = s["block_indices"].long()
    place = lambda pos: (table[first_block[b] + pos // bs], pos % bs)
    (b0, s0), (b1, s1) = place(past[b] + path[b, k]), place(past[b] + k)
    for caches, value in ((s["key_caches"], False), (s["value_caches"], True)):
        x = _rows(case, caches, value).transpose(2, 3)                                                    # [layers, pool, slot, hkv, d]
        x[:, b1, s1] = x[:, b0, s0]
        if case["cache"] == "u8":
            y = _params(case, caches).permute(0, 1, 4, 2, 3)
            y[:, b1, s1] = y[:, b0, s0]
    return {**out, "key_caches": s["key_caches"], "value_caches": s["value_caches"]}


def run(state):
    if own:
        return _run_own(state)
    return _run_accept(state) if state["case"]["kind"] == "accept" else _run_attention(state)


# ---- the definition in 64 bits ---------------------------------------------------------------------------------------
def exact(case, seed):
    if case["kind"] == "accept":
        return None                                    # whole values and moved bytes: nothing is computed
    s = prepare(case, seed)
    past, new, trees = _layout(case)
    hq, hkv, d, bs, W, S = (case[k] for k in ("hq", "hkv", "d", "bs", "window", "sinks"))
    G = hq // hkv
    table, first = s["block_indices"].long(), s["block_indices_begins"].tolist()
    out = torch.empty((int(new.sum()), hq, d), dtype=torch.float64, device=DEV)

    def stored(x):
        """What the cache holds of new rows."""
        x = x.float()
        if case["cache"] != "u8":
            return x.to(DTYPE[case["cache"]]).double()
        q, scale, zp = _quantise(x)
        return (q.double() - zp.double()[..., None]) * scale.double()[..., None]

    def cached(cache, blocks, value):
        rec = cache[blocks]
        if case["cache"] != "u8":
            return rec.view(DTYPE[case["cache"]]).view(-1, hkv, bs, d).transpose(1, 2).reshape(-1, hkv, d).double()
        x = rec[..., :bs * d].double()
        x = x.view(-1, hkv, d, bs).permute(0, 3, 1, 2) if value else x.view(-1, hkv, bs, d).transpose(1, 2)
        par = rec[..., bs * d:].contiguous().view(torch.float32).view(-1, hkv, 2, bs).double()
        return ((x - par[:, :, 1].transpose(1, 2)[..., None]) * par[:, :, 0].transpose(1, 2)[..., None]).reshape(-1, hkv, d)

    t = 0
    for b in range(len(past)):
        n, p = int(new[b]), int(past[b])
        blocks = table[first[b]:first[b + 1]]
        keys, values = (torch.cat([cached(s[c], blocks, v)[:p], stored(s[x][t:t + n].view(n, hkv, d))]) for c, x, v in
                        (("key_cache", "key", False), ("value_cache", "value", True)))
        parents = np.arange(-1, n - 1) if trees[b] is None else trees[b]
        sees = np.zeros((n, n), bool)                  # of the new tokens
        for i in range(n):
            if parents[i] >= 0:
                sees[i] = sees[parents[i]]
            sees[i, i] = True
        depth = _depth(parents)
        at = torch.from_numpy(np.concatenate([np.arange(p), p + depth])).to(DEV)      # positions of all keys
        seen = torch.cat([torch.ones((n, p), dtype=torch.bool, device=DEV), torch.from_numpy(sees).to(DEV)], 1)
        if W:
            row = torch.from_numpy(p + depth).to(DEV)[:, None]
            seen &= (at < S) | (at > row - W)
        q = s["query"][t:t + n].double().view(n, hkv, G, d)
        few = max(1, int(3e8 // (G * (p + n))))
        for h in range(hkv):
            for r in range(0, n, few):
                e = min(n, r + few)
                x = torch.matmul(q[r:e, h], keys[:, h].T) / math.sqrt(d)                                   # [rows, G, L]
                x = torch.softmax(x.masked_fill_(~seen[r:e, None], -math.inf), -1)
                out[t + r:t + e, h * G:(h + 1) * G] = torch.matmul(x, values[:, h])
        t += n
    return {"output": out.reshape(-1, hq * d), "key_cache": None, "value_cache": None}
