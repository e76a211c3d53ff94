"""Host-side mirror of latent attention (include/latent_b200.h): attention whose keys and values all come from one cached vector a
token, as a layer of a continuous-batching step calls it.

`LatentAttention.append` writes the step's new rows into the paged cache (norm, rotation) and rotates the queries' part;
`LatentAttention.attend` attends over the cache.  Both take their tensors by name, as `PagedAttentionExtension.evaluate` does;
`past_lens`, `subsequence_begins`, `block_indices` and `block_indices_begins` are the same tensors.  Everything is device memory, the
caller owns every buffer, and the calls run on the current stream of the operator's device.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional

import torch

from . import _abi, _latent_abi as A

_DTYPES = {torch.float16: _abi.PA_DTYPE_F16, torch.bfloat16: _abi.PA_DTYPE_BF16}
_FORMS = {"auto": A.PA_LATENT_AUTO, "absorbed": A.PA_LATENT_ABSORBED, "expanded": A.PA_LATENT_EXPANDED}
_METADATA = ("past_lens", "subsequence_begins", "block_indices", "block_indices_begins")


class LatentAttention:
    """One layer's operator instance (owns a C-ABI handle and its scratch)."""

    def __init__(self, num_heads: int, latent_size: int, rope_size: int, nope_size: int, value_size: int, block_size: int,
                 dtype: torch.dtype = torch.bfloat16, device: int = 0):
        from . import GenaiB200Error, load_library
        self._err = GenaiB200Error
        self._h = C.c_void_p()
        self.lib = load_library()
        if dtype not in _DTYPES:
            raise GenaiB200Error(f"LatentAttention: dtype {dtype} is not supported")
        self.num_heads, self.latent_size, self.rope_size = num_heads, latent_size, rope_size
        self.nope_size, self.value_size, self.block_size = nope_size, value_size, block_size
        self.dtype, self.device = dtype, torch.device("cuda", device)
        desc = A.pa_latent_desc(C.sizeof(A.pa_latent_desc), num_heads, latent_size, rope_size, nope_size, value_size, block_size, _DTYPES[dtype])
        self._check(self.lib.pa_b200_latent_create(C.byref(desc), device, C.byref(self._h)))

    def __del__(self):
        h = getattr(self, "_h", None)
        if h:
            self.lib.pa_b200_latent_destroy(h)
            self._h = None

    def _check(self, rc: int) -> None:
        if rc != _abi.PA_OK:
            raise self._err(f"pa_b200_latent status {rc}: {self.lib.pa_b200_last_error().decode()}")

    def allocate_cache(self, num_blocks: int) -> torch.Tensor:
        """A zeroed cache [num_blocks, block_size, latent_size + rope_size]."""
        return torch.zeros((num_blocks, self.block_size, self.latent_size + self.rope_size), dtype=self.dtype, device=self.device)

    # ---- checks --------------------------------------------------------------------------------
    def _tensor(self, name: str, t, dtype: torch.dtype, shape: tuple, contiguous: bool = False) -> torch.Tensor:
        """`t` if it is a device tensor of this type and shape (None: any size) whose last dimension, or all of it, is contiguous."""
        if not isinstance(t, torch.Tensor) or t.dtype != dtype or t.device != self.device or t.dim() != len(shape) or \
                any(want is not None and want != have for want, have in zip(shape, t.shape)):
            what = f"{t.dtype} {tuple(t.shape)} on {t.device}" if isinstance(t, torch.Tensor) else type(t).__name__
            raise self._err(f"{name}: expected {dtype} {shape} on {self.device}, got {what}")
        if not (t.is_contiguous() if contiguous else t.stride(-1) == 1 or t.shape[-1] == 1):
            raise self._err(f"{name}: strides {t.stride()} are not supported")
        return t

    def _metadata(self, a, inputs: dict) -> None:
        past, begins, blocks, block_begins = (self._tensor(n, inputs[n], torch.int32, (None,), True) for n in _METADATA)
        a.num_sequences, a.num_block_indices = past.shape[0], blocks.shape[0]
        if begins.shape[0] != a.num_sequences + 1 or block_begins.shape[0] != a.num_sequences + 1:
            raise self._err("subsequence_begins and block_indices_begins need num_sequences + 1 entries")
        a.past_lens, a.subsequence_begins, a.block_indices, a.block_indices_begins = (t.data_ptr() for t in (past, begins, blocks, block_begins))
        cache = self._tensor("cache", inputs["cache"], self.dtype, (None, self.block_size, self.latent_size + self.rope_size), True)
        a.cache, a.num_blocks = cache.data_ptr(), cache.shape[0]
        # 1 = cudaStreamLegacy: a null handle would select the operator's own stream
        a.stream = inputs.get("stream") or torch.cuda.current_stream(self.device).cuda_stream or 1

    # ---- the operators -------------------------------------------------------------------------
    def append(self, inputs: dict, outputs: Optional[dict] = None) -> None:
        """inputs: latent [T, latent + rope], norm_weight [latent] (optional) with norm_eps, rope_table f32 [rows, rope] (cos | sin),
        interleaved (default False), positions i32 [T] (optional), query_rope [T, heads, rope] (optional), cache and the paged
        metadata.  outputs: query_rope, which may be the input itself; the cache is written in place."""
        a = A.pa_latent_append_args()
        a.struct_size = C.sizeof(A.pa_latent_append_args)
        latent = self._tensor("latent", inputs["latent"], self.dtype, (None, self.latent_size + self.rope_size))
        tokens = latent.shape[0]
        a.latent, a.latent_stride, a.num_tokens = latent.data_ptr(), latent.stride(0), tokens
        weight = inputs.get("norm_weight")
        if weight is not None:
            a.norm_weight = self._tensor("norm_weight", weight, self.dtype, (self.latent_size,)).data_ptr()
            a.norm_eps = inputs["norm_eps"]
        query = inputs.get("query_rope")
        if query is not None:
            query = self._tensor("query_rope", query, self.dtype, (tokens, self.num_heads, self.rope_size))
            out = self._tensor("output query_rope", (outputs or {}).get("query_rope"), self.dtype, (tokens, self.num_heads, self.rope_size))
            a.query_rope, a.query_rope_out = query.data_ptr(), out.data_ptr()
            a.query_rope_token_stride, a.query_rope_head_stride, _ = query.stride()
            a.query_rope_out_token_stride, a.query_rope_out_head_stride, _ = out.stride()
        table = self._tensor("rope_table", inputs["rope_table"], torch.float32, (None, self.rope_size), True)
        a.rope_table, a.rope_table_rows = table.data_ptr(), table.shape[0]
        a.interleaved = 1 if inputs.get("interleaved") else 0
        if inputs.get("positions") is not None:
            a.positions = self._tensor("positions", inputs["positions"], torch.int32, (tokens,), True).data_ptr()
        self._metadata(a, inputs)
        self._check(self.lib.pa_b200_latent_append(self._h, C.byref(a)))

    def attend(self, inputs: dict, outputs: dict, form: str = "auto") -> None:
        """inputs: query_nope [T, heads, nope], query_rope [T, heads, rope] (rotated), key_up [heads, nope, latent],
        value_up [heads, value, latent], scale (default 1/sqrt(nope + rope)), cache and the paged metadata.
        outputs: output [T, heads * value].  form: "absorbed", "expanded", or "auto" (each sequence in the one that suits it)."""
        if form not in _FORMS:
            raise self._err(f"unknown form {form!r}: one of {', '.join(_FORMS)}")
        a = A.pa_latent_attention_args()
        a.struct_size = C.sizeof(A.pa_latent_attention_args)
        a.form = _FORMS[form]
        nope = self._tensor("query_nope", inputs["query_nope"], self.dtype, (None, self.num_heads, self.nope_size))
        tokens = nope.shape[0]
        rope = self._tensor("query_rope", inputs["query_rope"], self.dtype, (tokens, self.num_heads, self.rope_size))
        key_up = self._tensor("key_up", inputs["key_up"], self.dtype, (self.num_heads, self.nope_size, self.latent_size))
        value_up = self._tensor("value_up", inputs["value_up"], self.dtype, (self.num_heads, self.value_size, self.latent_size))
        for name, t in (("key_up", key_up), ("value_up", value_up)):
            if t.stride(1) != self.latent_size:
                raise self._err(f"{name}: a head's rows have to be contiguous")
        out = self._tensor("output", outputs["output"], self.dtype, (tokens, self.num_heads * self.value_size), True)
        a.num_tokens, a.output = tokens, out.data_ptr()
        a.query_nope, a.query_rope, a.key_up, a.value_up = nope.data_ptr(), rope.data_ptr(), key_up.data_ptr(), value_up.data_ptr()
        a.query_nope_token_stride, a.query_nope_head_stride, _ = nope.stride()
        a.query_rope_token_stride, a.query_rope_head_stride, _ = rope.stride()
        a.key_up_head_stride, a.value_up_head_stride = key_up.stride(0), value_up.stride(0)
        a.scale = inputs.get("scale") or 0.0
        self._metadata(a, inputs)
        self._check(self.lib.pa_b200_latent_attention(self._h, C.byref(a)))

    def reserve(self, num_tokens: int, num_sequences: int, num_block_indices: int, form: str = "auto") -> None:
        """Grows the scratch for steps of up to this size, so that `attend` does not allocate (stream captures need that)."""
        self._check(self.lib.pa_b200_latent_reserve(self._h, num_tokens, num_sequences, num_block_indices, _FORMS[form]))

    def device_status(self) -> int:
        """Reads and clears the device status word (PA_DEV_* bits)."""
        bits = C.c_uint32(0)
        self._check(self.lib.pa_b200_latent_last_device_status(self._h, C.byref(bits)))
        return bits.value

    def launch_count(self) -> int:
        return int(self.lib.pa_b200_latent_launch_count(self._h))
