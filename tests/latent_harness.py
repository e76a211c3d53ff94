"""Steps of latent attention for the tests: inputs, the operator's call, and the definition in 64 bits on the CPU."""
import math

import numpy as np
import torch

DTYPE = {"bf16": torch.bfloat16, "f16": torch.float16}
# half a unit in the last place, relative
UNIT = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11}
# latent, rope, nope, value
WIDE, SMALL, MIXED = (512, 64, 128, 128), (256, 32, 64, 64), (256, 64, 128, 64)


class Step:
    """One step's tensors on the CPU; slots of the cache that hold no token are NaN."""

    def __init__(self, past, new, heads=16, sizes=WIDE, bs=32, dtype="bf16", seed=0, spread=1.0, extra_blocks=3):
        self.past, self.new = np.asarray(past, np.int64), np.asarray(new, np.int64)
        self.heads, self.sizes, self.bs, self.dtype = heads, sizes, bs, dtype
        R, P, Dn, Dv = sizes
        dt = DTYPE[dtype]
        rng = np.random.default_rng(seed)
        gen = torch.Generator().manual_seed(seed + 1)
        rnd = lambda *s: torch.randn(s, generator=gen)
        nblk = (self.past + self.new + bs - 1) // bs
        total = int(nblk.sum())
        pool = total + extra_blocks
        table = rng.permutation(pool)[:total].astype(np.int32)
        first = np.concatenate([[0], np.cumsum(nblk)]).astype(np.int32)
        begins = np.concatenate([[0], np.cumsum(self.new)]).astype(np.int32)
        self.tokens = int(self.new.sum())
        self.cache = torch.full((pool, bs, R + P), math.nan).to(dt)
        self.context = []
        for s in range(len(self.past)):
            rows = rnd(int(self.past[s] + self.new[s]), R + P).to(dt)
            self.context.append(rows)
            pos = np.arange(len(rows))
            if len(rows):
                self.cache[torch.from_numpy(table[first[s] + pos // bs].astype(np.int64)), torch.from_numpy(pos % bs)] = rows
        t = lambda a: torch.from_numpy(np.ascontiguousarray(a).astype(np.int32))
        self.meta = {"past_lens": t(self.past), "subsequence_begins": t(begins), "block_indices": t(table), "block_indices_begins": t(first)}
        self.query = (rnd(self.tokens, heads, Dn + P) * spread).to(dt)
        self.up = (rnd(heads, Dn + Dv, R) / math.sqrt(R)).to(dt)
        self.latent = rnd(self.tokens, R + P).to(dt)
        self.norm_weight = (1 + 0.1 * rnd(R)).to(dt)
        rows = int((self.past + self.new).max()) + 8
        angle = np.arange(rows)[:, None] * np.power(1e4, -np.arange(P // 2) * 2.0 / P)[None, :]
        self.rope_table = torch.from_numpy(np.concatenate([np.cos(angle), np.sin(angle)], 1).astype(np.float32))

    def operator(self, pkg):
        return pkg.LatentAttention(self.heads, *self.sizes, self.bs, DTYPE[self.dtype])

    def device_inputs(self):
        Dn = self.sizes[2]
        q, up = self.query.cuda(), self.up.cuda()
        x = {k: v.cuda() for k, v in self.meta.items()}
        x.update(cache=self.cache.cuda(), query_nope=q[..., :Dn], query_rope=q[..., Dn:], key_up=up[:, :Dn], value_up=up[:, Dn:])
        return x

    def append_inputs(self, **kw):
        x = self.device_inputs()
        x.update(latent=self.latent.cuda(), norm_weight=self.norm_weight.cuda(), norm_eps=1e-6, rope_table=self.rope_table.cuda())
        x.update(kw)
        return x

    def attend(self, op, form="auto", inputs=None):
        x = inputs if inputs is not None else self.device_inputs()
        out = torch.full((self.tokens, self.heads * self.sizes[3]), math.nan, dtype=DTYPE[self.dtype], device="cuda")
        op.attend(x, {"output": out}, form=form)
        return out.cpu()

    def expected(self, scale=None):
        """The output in 64 bits [T, H, Dv]."""
        R, P, Dn, Dv = self.sizes
        scale = scale if scale is not None else 1.0 / math.sqrt(Dn + P)
        up, q = self.up.double(), self.query.double()
        out = torch.empty((self.tokens, self.heads, Dv), dtype=torch.float64)
        t = 0
        for s, rows in enumerate(self.context):
            n, p = int(self.new[s]), int(self.past[s])
            if n == 0:
                continue
            c = rows.double()
            k = torch.einsum("lr,hdr->hld", c[:, :R], up[:, :Dn])
            v = torch.einsum("lr,hdr->hld", c[:, :R], up[:, Dn:])
            a = torch.einsum("nhd,hld->hnl", q[t:t + n, :, :Dn], k) + torch.einsum("nhd,ld->hnl", q[t:t + n, :, Dn:], c[:, R:])
            hidden = torch.arange(p + n)[None] > p + torch.arange(n)[:, None]
            a = torch.softmax((a * scale).masked_fill(hidden, -math.inf), -1)
            out[t:t + n] = torch.einsum("hnl,hld->nhd", a, v)
            t += n
        return out

    def check(self, out, expected=None, rows=None):
        """Four roundings to the 16-bit type stand between the inputs and an output: the absorbed query or the expanded keys, the
        probabilities, the sum of latents or the expanded values, the output.  Each has an rms error of at most u / sqrt(3) relative
        to what it rounds; all but the first reach the output as they are, the first multiplied by the logits' standard
        deviation, which is at most 2 in these inputs.  Together u / sqrt(3) * sqrt(3 + 4) = 1.53 u: a sequence's
        outputs may be 2 u off in the 2-norm, an element (eight of its standard deviations) 12.3 u of the larger of its magnitude and the
        root mean square of its sequence's."""
        u = UNIT[self.dtype]
        want = expected if expected is not None else self.expected()
        got = out.double().reshape(want.shape)
        t = 0
        for s in range(len(self.new)):
            n = int(self.new[s])
            if n and (rows is None or s in rows):
                a, b = got[t:t + n], want[t:t + n]
                assert torch.isfinite(a).all(), f"sequence {s}: not finite"
                rel = float((a - b).norm() / b.norm())
                assert rel <= 2 * u, f"sequence {s} (past {self.past[s]}, new {n}): rel {rel / u:.2f} u"
                rms = float(b.square().mean().sqrt())
                big = float(((a - b).abs() / b.abs().clamp(min=rms)).max())
                assert big <= 12.3 * u, f"sequence {s} (past {self.past[s]}, new {n}): element {big / u:.2f} u"
            t += n
