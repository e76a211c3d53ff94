"""Shared plumbing of the tests of masked attention (include/masked_b200.h): small steps over a paged cache, what every row sees of it,
the result in 64 bits, and what the acceptance of drafts leaves behind.  Everything that no row sees is poisoned: blocks have impossible numbers in
the block table, positions hold not-a-number.

Tolerances, fixed before the kernels were run, from the roundings of the operator's arithmetic (half a step: bf16 2^-8, f16 2^-11).  With A the row's
attention over |values|, an error of the probabilities by a factor of at most 1 + d moves an output element by at most 2 d A:
  probabilities      f16 cache 2^-11; bf16 cache 2^-8; u8 cache 2^-9 (packed exponential) + 2^-11 e ln 2 for an exponent e of at most 16 in f16
  u8 keys            scale and product rounded to f16: 2^-10 of the keys' range, times the query's sum of magnitudes, times the softmax scale
  u8 values          scale and product rounded to f16: 2^-10 of the values' range
  accumulation       32-bit sums of D products, each step truncated at 2^-23 of the terms' magnitude
and the output is rounded once.  That is the bound of an element.  A row's error as a whole is that of many independent roundings: four times the
tolerance the operator is specified to for whole tensors (2e-3 for 16-bit caches, 1e-2 for u8, 8e-3 where the output or a bf16 cache's probabilities have 8 significant bits)."""
from __future__ import annotations

import math

import numpy as np
import torch

import __graft_entry__ as entry

pkg = entry.load_package()
from openvino_genai_b200 import _masked_abi as M  # noqa: E402

DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
NONE = M.PA_TREE_NONE


def tree(rng, n, bushy=2):
    return [-1] + [int(rng.integers(max(0, (i - 1) // bushy - 1), i)) for i in range(1, n)]


def quantise(x):
    """The documented by-token quantiser, in steps of 32 bits."""
    mn, mx = x.amin(-1), x.amax(-1)
    scale = (mx - mn) / torch.full_like(mx, 255.0)      # (by a number torch would multiply with its reciprocal)
    scale = torch.where(scale > 0, scale, torch.ones_like(scale))
    zp, inv = -mn / scale, 1.0 / scale
    q = (x.double() * inv.double()[..., None] + zp.double()[..., None]).float()
    return q.clamp(0, 255).round().to(torch.uint8), scale, zp


class Step:
    """One step: `past` and `new` tokens of every sequence; trees[s] is a list of parents or None."""

    def __init__(self, past, new, hq=8, hkv=2, d=64, bs=16, act="f16", cache="f16", window=0, sinks=0, trees=None, seed=0, dev="cuda:0", poison=True,
                 spare_blocks=3, scale=None, magnitude=1.0):
        self.__dict__.update(past=list(past), new=list(new), hq=hq, hkv=hkv, d=d, bs=bs, act=act, cache=cache, window=window, sinks=sinks, dev=dev, scale=scale)
        self.trees = trees if trees is not None else [None] * len(self.new)
        rng = np.random.default_rng(seed)
        g = torch.Generator(device=dev)
        g.manual_seed(seed + 1)
        B, self.T = len(self.past), int(sum(self.new))
        blocks = [(p + n + bs - 1) // bs for p, n in zip(self.past, self.new)]
        self.pool = sum(blocks) + spare_blocks
        self.table = rng.permutation(self.pool)[:sum(blocks)].astype(np.int32)
        self.first = np.concatenate([[0], np.cumsum(blocks)]).astype(np.int64)
        self.begins = np.concatenate([[0], np.cumsum(self.new)]).astype(np.int64)
        rnd = lambda *s: torch.randn(s, generator=g, device=dev)
        self.query, self.key, self.value = ((rnd(self.T, h * d) * m).to(DT[act]) for h, m in ((hq, magnitude), (hkv, 1), (hkv, 1)))
        self.values = {"key": rnd(self.pool, hkv, bs, d), "value": rnd(self.pool, hkv, bs, d)}
        self.packed = {k: self.pack(v, k == "value") for k, v in self.values.items()}
        self.sees = [self.seen(s) for s in range(B)]
        given = self.table.copy()
        if poison:
            used = {k: torch.zeros((self.pool, bs), dtype=torch.bool) for k in ("seen", "new")}
            for s in range(B):
                any_row = self.sees[s].any(0) if self.new[s] else np.zeros(self.past[s], bool)
                for pos in range(len(any_row)):
                    blk = self.table[self.first[s] + pos // bs]
                    used["seen"][blk, pos % bs] |= bool(any_row[pos])
                for j in range(blocks[s]):
                    if not any_row[j * bs:(j + 1) * bs].any():
                        given[self.first[s] + j] = [-7, 1 << 30, self.pool][int(rng.integers(0, 3))]
            self.poison(~used["seen"].to(dev))
        i32 = lambda a: torch.from_numpy(np.asarray(a, np.int32)).to(dev)
        self.meta = {"past_lens": i32(self.past), "subsequence_begins": i32(self.begins), "block_indices": i32(given), "block_indices_begins": i32(self.first)}
        self.parents = None
        if any(t is not None for t in self.trees):
            self.parents = i32(np.concatenate([np.asarray(t if t is not None else [NONE] * n, np.int32) for t, n in zip(self.trees, self.new)] + [np.zeros(0, np.int32)]))

    # ---- the cache, in the operator's layout: [blocks, hkv, record] bytes -------------------------
    def pack(self, x, value):
        n, h, bs, d = x.shape
        if self.cache != "u8":
            return x.to(DT[self.cache]).contiguous().view(torch.uint8).reshape(n, h, -1)
        q, s, z = quantise(x)
        q = q.transpose(2, 3) if value else q
        return torch.cat([q.reshape(n, h, bs * d), s.contiguous().view(torch.uint8), z.contiguous().view(torch.uint8)], 2)

    def unpack(self, rec, value):
        n, h = rec.shape[:2]
        if self.cache != "u8":
            return rec.contiguous().view(DT[self.cache]).reshape(n, h, self.bs, self.d).double()
        q = rec[:, :, :self.bs * self.d]
        q = q.reshape(n, h, self.d, self.bs).transpose(2, 3) if value else q.reshape(n, h, self.bs, self.d)
        par = rec[:, :, self.bs * self.d:].contiguous().view(torch.float32).reshape(n, h, 2, self.bs).double()
        return (q.double() - par[:, :, 1, :, None]) * par[:, :, 0, :, None]

    def poison(self, where, value=float("nan")):
        """where [blocks, bs]: those positions hold `value` (u8: as their scale)."""
        for c in self.packed.values():
            if self.cache == "u8":
                par = c[:, :, self.bs * self.d:].clone(memory_format=torch.contiguous_format).view(torch.float32).reshape(self.pool, self.hkv, 2, self.bs)
                par[where[:, None, None, :].expand_as(par)] = value
                c[:, :, self.bs * self.d:] = par.reshape(self.pool, self.hkv, -1).view(torch.uint8)
            else:
                x = c.view(DT[self.cache]).view(self.pool, self.hkv, self.bs, self.d)
                x[where[:, None, :, None].expand_as(x)] = value

    # ---- the definition -----------------------------------------------------------------------------
    def depth(self, s):
        t = self.trees[s]
        if t is None:
            return np.arange(self.new[s])
        depth = np.zeros(len(t), np.int64)
        for i, p in enumerate(t):
            depth[i] = 0 if p < 0 else depth[p] + 1
        return depth

    def seen(self, s):
        """[new, past + new] what the rows of sequence s see."""
        p, n, t = self.past[s], self.new[s], self.trees[s]
        depth = self.depth(s)
        of_chunk = np.zeros((n, n), bool)
        for i in range(n):
            j = i
            while j >= 0:
                of_chunk[i, j] = True
                j = j - 1 if t is None else t[j]
        seen = np.concatenate([np.ones((n, p), bool), of_chunk], 1)
        if self.window:
            at = np.concatenate([np.arange(p), p + depth])
            seen &= (at[None, :] < self.sinks) | (at[None, :] > (p + depth)[:, None] - self.window)
        return seen

    def stored(self, x):
        """What the cache holds of new rows [tokens, hkv * d], in 64 bits: [tokens, hkv, d]."""
        x = x.float().view(-1, self.hkv, self.d)
        if self.cache != "u8":
            return x.to(DT[self.cache]).double()
        q, s, z = quantise(x)
        return (q.double() - z.double()[..., None]) * s.double()[..., None]

    def context(self, s, which, fresh):
        """Keys or values [past + new, hkv, d] of sequence s in 64 bits."""
        blocks = torch.from_numpy(self.table[self.first[s]:self.first[s + 1]].astype(np.int64)).to(self.dev)
        old = self.unpack(self.packed[which][blocks], which == "value").transpose(1, 2).reshape(-1, self.hkv, self.d)[:self.past[s]]
        return torch.cat([old, self.stored(fresh[self.begins[s]:self.begins[s + 1]])])

    def reference(self):
        """Output [T, hq * d] and what an element of it may be off by, in 64 bits."""
        G, scale = self.hq // self.hkv, self.scale or 1 / math.sqrt(self.d)
        out = torch.zeros((self.T, self.hq, self.d), dtype=torch.float64, device=self.dev)
        off = torch.zeros_like(out)
        for s in range(len(self.new)):
            t0, n = int(self.begins[s]), self.new[s]
            if n == 0:
                continue
            seen = torch.from_numpy(self.sees[s]).to(self.dev)
            k, v = self.context(s, "key", self.key), self.context(s, "value", self.value)
            gone = ~seen.any(0)
            k[gone], v[gone] = 0, 0
            for h in range(self.hq):
                q, kk, vv = self.query[t0:t0 + n].double().view(n, self.hq, self.d)[:, h], k[:, h // G], v[:, h // G]
                # (what a row does not see takes no part: not-a-number in it neither)
                x = (q @ kk.T * scale).masked_fill(~seen, -math.inf)
                p = torch.softmax(x, -1)
                finite = lambda y: torch.nan_to_num(y, nan=0.0, posinf=0.0, neginf=0.0)
                fk, fv = finite(kk), finite(vv)
                out[t0:t0 + n, h] = p @ vv if bool(torch.isfinite(vv).all()) else torch.stack([p[i, seen[i]] @ vv[seen[i]] for i in range(n)])
                d = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8, "u8": 2.0 ** -9 + 2.0 ** -11 * 16 * math.log(2)}[self.cache]
                d = d + (q.abs() @ fk.abs().T * scale).amax(-1) * self.d * 2.0 ** -23
                extra = 0.0
                if self.cache == "u8":
                    d = d + scale * q.abs().sum(-1) * 2.0 ** -10 * fk.abs().max() * 2
                    extra = 2.0 ** -10 * 2 * fv.abs().max()
                off[t0:t0 + n, h] = 2 * d[:, None] * (finite(p) @ fv.abs()) + extra
        off = off + out.abs() * (torch.finfo(DT[self.act]).eps / 2)
        return out.view(self.T, -1), off.view(self.T, -1)

    def cache_after(self):
        """The caches' bytes once the step has written its rows."""
        res = []
        for which, fresh in (("key", self.key), ("value", self.value)):
            c = self.packed[which].clone()
            value = which == "value"
            x = fresh.float().view(-1, self.hkv, self.d)
            for s in range(len(self.new)):
                for i in range(self.new[s]):
                    pos = self.past[s] + i
                    blk, slot, row = int(self.table[self.first[s] + pos // self.bs]), pos % self.bs, x[int(self.begins[s]) + i]
                    if self.cache != "u8":
                        c[blk].view(DT[self.cache]).view(self.hkv, self.bs, self.d)[:, slot] = row.to(DT[self.cache])
                        continue
                    q, sc, z = quantise(row)
                    data = c[blk][:, :self.bs * self.d]
                    if value:
                        data.view(self.hkv, self.d, self.bs)[:, :, slot] = q
                    else:
                        data.view(self.hkv, self.bs, self.d)[:, slot] = q
                    par = c[blk][:, self.bs * self.d:].clone(memory_format=torch.contiguous_format).view(torch.float32).view(self.hkv, 2, self.bs)
                    par[:, 0, slot], par[:, 1, slot] = sc, z
                    c[blk][:, self.bs * self.d:] = par.reshape(self.hkv, -1).view(torch.uint8)
            res.append(c)
        return res

    # ---- the framework --------------------------------------------------------------------------------
    def operator(self):
        return pkg.PagedAttentionExtension(self.hq, self.hkv, self.d, self.bs, DT[self.act], self.cache)

    def inputs(self, kc, vc):
        x = {"query": self.query, "key": self.key, "value": self.value, "key_cache": kc, "value_cache": vc, **self.meta,
             "max_context_len": max([p + n for p, n in zip(self.past, self.new)] + [0]), "sliding_window": self.window, "sink_tokens": self.sinks}
        if self.scale is not None:
            x["scale"] = self.scale
        if self.parents is not None:
            x["tree_parents"] = self.parents
        return x

    def run(self, op=None):
        """output, key cache, value cache and device status of one call."""
        op = op or self.operator()
        kc, vc = self.packed["key"].clone(), self.packed["value"].clone()
        out = torch.full((self.T, self.hq * self.d), 77.0, dtype=DT[self.act], device=self.dev)
        op.evaluate(self.inputs(kc, vc), {"output": out})
        torch.cuda.synchronize()
        return out, kc, vc, op.device_status()

    def check(self, out, rows=None):
        """`out` against the reference, by element and by row."""
        ref, off = self.reference()
        x = out.double()
        if rows is not None:
            x, ref, off = x[rows], ref[rows], off[rows]
        nan = torch.isnan(ref)
        assert torch.equal(torch.isnan(x), nan), f"{int((torch.isnan(x) != nan).sum())} elements are or are not numbers against the definition"
        x, ref, off = (torch.nan_to_num(y, nan=0.0, posinf=0.0, neginf=0.0) for y in (x, ref, off))
        err = (x - ref).abs()
        worst = (err - off).max().item()
        assert worst <= 0, f"an element is {worst:.3e} further off than its bound"
        tol = {"f16": 2e-3, "bf16": 8e-3, "u8": 1e-2}[self.cache]
        tol = 4 * max(tol, 8e-3 if self.act == "bf16" else 0)
        heads = lambda y: y.view(-1, self.hq, self.d)
        rel = heads(err).norm(dim=-1) / heads(ref).norm(dim=-1).clamp_min(1e-30)
        rel = torch.where(heads(ref).norm(dim=-1) > 0, rel, torch.zeros_like(rel))
        assert rel.max().item() <= tol, f"row {int(rel.amax(1).argmax())} is {rel.max().item():.3e} off, {tol} allowed"
        return rel.max().item()


def accept(trees, draft, sampled, max_path):
    """The definition of the walk, for one sequence: path."""
    path = [0]
    while len(path) < max_path:
        at = path[-1]
        nxt = [c for c in range(1, len(trees)) if trees[c] == at and draft[c] == sampled[at]]
        if not nxt:
            break
        path.append(nxt[0])
    return path
