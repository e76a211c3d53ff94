"""One attention layer of a model with latent attention, served from a paged cache: `python integration/latent_layer.py`.

A batch is served as an engine would: steps that mix a chunk of one prompt with single tokens of other sequences, every step an
`append` (norm, rotation, cache write) and an `attend` on the same metadata.  The result is compared with the layer computed whole,
from its formulas, in 64 bits."""
import pathlib
import sys

import torch

ROOT = pathlib.Path(__file__).resolve().parents[1]


class LatentLayer:
    """Weights of one layer and its cache; `step` takes the hidden rows of a step's new tokens."""

    def __init__(self, hidden=512, heads=16, latent=512, rope=64, nope=128, value=128, block_size=32, blocks=64, positions=4096, seed=0):
        from openvino_genai_b200 import LatentAttention
        g = torch.Generator().manual_seed(seed)
        w = lambda *shape: (torch.randn(shape, generator=g) * shape[-1] ** -0.5).to(torch.bfloat16).cuda()
        self.sizes = (heads, latent, rope, nope, value)
        self.query, self.down, self.up, self.out = w(heads * (nope + rope), hidden), w(latent + rope, hidden), w(heads, nope + value, latent), w(hidden, heads * value)
        self.norm_weight = (1 + 0.1 * torch.randn(latent, generator=g)).to(torch.bfloat16).cuda()
        angle = torch.arange(positions)[:, None] * 10000.0 ** -(torch.arange(rope // 2) / (rope // 2))
        self.rope_table = torch.cat([angle.cos(), angle.sin()], 1).float().cuda()
        self.op = LatentAttention(heads, latent, rope, nope, value, block_size, torch.bfloat16)
        self.cache = self.op.allocate_cache(blocks)

    def step(self, x, metadata, form="auto"):
        """x: [tokens, hidden].  metadata: past_lens, subsequence_begins, block_indices, block_indices_begins.  form: what the caller knows of the step."""
        heads, latent, rope, nope, value = self.sizes
        q = (x @ self.query.T).view(-1, heads, nope + rope)
        inputs = {"cache": self.cache, "latent": x @ self.down.T, "norm_weight": self.norm_weight, "norm_eps": 1e-6, "rope_table": self.rope_table,
                  "query_nope": q[..., :nope], "query_rope": q[..., nope:], "key_up": self.up[:, :nope], "value_up": self.up[:, nope:], **metadata}
        self.op.append(inputs, {"query_rope": inputs["query_rope"]})
        o = torch.empty((x.shape[0], heads * value), dtype=x.dtype, device=x.device)
        self.op.attend(inputs, {"output": o}, form=form)
        return o @ self.out.T

    def whole(self, x):
        """A whole sequence at once, in 64 bits."""
        heads, latent, rope, nope, value = self.sizes
        x = x.double()
        q = (x @ self.query.double().T).view(-1, heads, nope + rope)
        down = x @ self.down.double().T
        c = down[:, :latent] * torch.rsqrt(down[:, :latent].square().mean(1, keepdim=True) + 1e-6) * self.norm_weight.double()
        cos, sin = self.rope_table[:x.shape[0]].double().chunk(2, 1)

        def rotate(y, cos, sin):
            a, b = y.chunk(2, -1)
            return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)

        kr, qr = rotate(down[:, latent:], cos, sin), rotate(q[..., nope:], cos[:, None], sin[:, None])
        k, v = (torch.einsum("tr,hdr->thd", c, part) for part in (self.up[:, :nope].double(), self.up[:, nope:].double()))
        s = (torch.einsum("thd,uhd->htu", q[..., :nope], k) + torch.einsum("thd,ud->htu", qr, kr)) * (nope + rope) ** -0.5
        s = s.masked_fill(torch.ones(s.shape[1:], dtype=torch.bool, device=x.device).triu(1), float("-inf"))
        return torch.einsum("htu,uhd->thd", s.softmax(-1), v).reshape(-1, heads * value) @ self.out.double().T


def serve(layer, sequences, chunk=128, block_size=32):
    """Serves the sequences (hidden rows) in steps: each brings the next chunk of every sequence's prompt part, or one token behind it."""
    length = [x.shape[0] for x in sequences]
    prompt = [3 * n // 4 for n in length]
    done, out, blocks, first = [0] * len(length), [torch.empty_like(x) for x in sequences], [], 0
    for n in length:      # (every sequence has its blocks from the beginning)
        need = -(-n // block_size)
        blocks.append(list(range(first, first + need)))
        first += need
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    steps = 0
    while any(d < n for d, n in zip(done, length)):
        live = [s for s, n in enumerate(length) if done[s] < n]
        new = [min(chunk, prompt[s] - done[s]) if done[s] < prompt[s] else 1 for s in live]
        cumulative = lambda v: [sum(v[:i]) for i in range(len(v) + 1)]
        metadata = {"past_lens": i32([done[s] for s in live]), "subsequence_begins": i32(cumulative(new)),
                    "block_indices": i32([b for s in live for b in blocks[s]]), "block_indices_begins": i32(cumulative([len(blocks[s]) for s in live]))}
        # (the lengths are known here: steps of single tokens only need nothing of the expanded form)
        y = layer.step(torch.cat([sequences[s][done[s]:done[s] + n] for s, n in zip(live, new)]), metadata, "absorbed" if max(new) == 1 else "auto")
        for s, n, rows in zip(live, new, y.split(new)):
            out[s][done[s]:done[s] + n] = rows
            done[s] += n
        steps += 1
    return out, steps


def main():
    sys.path.insert(0, str(ROOT))
    import __graft_entry__
    __graft_entry__.load_package()
    layer = LatentLayer()
    g = torch.Generator().manual_seed(1)
    sequences = [torch.randn((n, 512), generator=g).to(torch.bfloat16).cuda() for n in (400, 61, 230, 8)]
    out, steps = serve(layer, sequences)
    worst = max(float((y.double() - (want := layer.whole(x))).norm() / want.norm()) for x, y in zip(sequences, out))
    print(f"{len(sequences)} sequences in {steps} steps, {layer.op.launch_count()} kernel launches, rel error {worst:.1e}, device status {layer.op.device_status()}")
    return worst


if __name__ == "__main__":
    main()
