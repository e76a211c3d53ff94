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


class LatentAttention:
    """The operator for layers of one geometry (owns a C-ABI handle and its scratch).  One instance serves all such layers of a model in turn: every call
    brings its own weights, cache and metadata, and the scratch of a step can be gigabytes."""

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
        row = latent_size + rope_size
        self._ordinal = device
        self._row_shape, self._block_shape, self._output_shape = (row,), (block_size, row), (num_heads * value_size,)
        self._nope_shape, self._rope_shape = (num_heads, nope_size), (num_heads, rope_size)
        self._key_shape, self._value_shape = (nope_size, latent_size), (value_size, latent_size)
        self._args = C.create_string_buffer(max(A.APPEND_ARGS.size, A.ATTENTION_ARGS.size))
        self._append, self._attend = self.lib.pa_b200_latent_append, self.lib.pa_b200_latent_attention
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
    # (they run before every launch: a small step's time is the host's)
    def _refuse(self, name: str, t, expected: str):
        what = f"{t.dtype} {tuple(t.shape)}, strides {t.stride()}, on {t.device}" if isinstance(t, torch.Tensor) else type(t).__name__
        raise self._err(f"{name}: expected {expected} on {self.device}, got {what}")

    def _rows(self, name: str, t, shape: tuple):
        """The strides of a device tensor of the operator's type whose dimensions behind the first are `shape` and whose last is contiguous."""
        if not isinstance(t, torch.Tensor) or t.dtype is not self.dtype or t.device != self.device or t.shape[1:] != shape:
            self._refuse(name, t, f"{self.dtype} [rows, {', '.join(map(str, shape))}]")
        strides = t.stride()
        if strides[-1] != 1:
            self._refuse(name, t, "a contiguous last dimension")
        return strides

    def _whole(self, name: str, t, dtype: torch.dtype, shape: tuple) -> int:
        """The address of a contiguous device tensor of this type whose dimensions behind the first are `shape`."""
        if not isinstance(t, torch.Tensor) or t.dtype is not dtype or t.device != self.device or t.dim() == 0 or t.shape[1:] != shape or not t.is_contiguous():
            self._refuse(name, t, f"contiguous {dtype} [rows{''.join(', ' + str(n) for n in shape)}]")
        return t.data_ptr()

    def _step(self, inputs: dict) -> tuple:
        """cache, num_blocks, the paged metadata and its sizes, in the order of the argument structs."""
        past, begins, blocks, block_begins, cache = inputs["past_lens"], inputs["subsequence_begins"], inputs["block_indices"], \
            inputs["block_indices_begins"], inputs["cache"]
        whole, i32 = self._whole, torch.int32
        addresses = (whole("past_lens", past, i32, ()), whole("subsequence_begins", begins, i32, ()), whole("block_indices", blocks, i32, ()),
                     whole("block_indices_begins", block_begins, i32, ()))
        sequences = past.shape[0]
        if begins.shape[0] != sequences + 1 or block_begins.shape[0] != sequences + 1:
            raise self._err("subsequence_begins and block_indices_begins need num_sequences + 1 entries")
        return (whole("cache", cache, self.dtype, self._block_shape), cache.shape[0], *addresses, sequences, blocks.shape[0])

    def _stream(self, inputs: dict) -> int:
        # 1 = cudaStreamLegacy: a null handle would select the operator's own stream
        return inputs.get("stream") or torch._C._cuda_getCurrentRawStream(self._ordinal) or 1

    def _form(self, form: str) -> int:
        if form not in _FORMS:
            raise self._err(f"unknown form {form!r}: one of {', '.join(_FORMS)}")
        return _FORMS[form]

    # ---- the operators -------------------------------------------------------------------------
    def append(self, inputs: dict, outputs: Optional[dict] = None) -> None:
        """inputs: latent [T, latent + rope], norm_weight [latent] (optional) with norm_eps, rope_table f32 [rows, rope] (cos | sin),
        interleaved (default False), positions i32 [T] (optional), query_rope [T, heads, rope] (optional), cache and the paged
        metadata.  outputs: query_rope, which may be the input itself; the cache is written in place."""
        latent, weight, query, table = inputs["latent"], inputs.get("norm_weight"), inputs.get("query_rope"), inputs["rope_table"]
        latent_stride = self._rows("latent", latent, self._row_shape)[0]
        tokens = latent.shape[0]
        norm = eps = 0
        if weight is not None:
            norm, eps = self._whole("norm_weight", weight, self.dtype, ()), inputs["norm_eps"]
            if weight.shape[0] != self.latent_size:
                self._refuse("norm_weight", weight, f"[{self.latent_size}]")
        query_address = out_address = 0
        q = o = (0, 0)
        if query is not None:
            out = (outputs or {}).get("query_rope")
            q, o = self._rows("query_rope", query, self._rope_shape), self._rows("output query_rope", out, self._rope_shape)
            if query.shape[0] != tokens or out.shape[0] != tokens:
                raise self._err("latent, query_rope and output query_rope need the same number of tokens")
            query_address, out_address = query.data_ptr(), out.data_ptr()
        table_address = self._whole("rope_table", table, torch.float32, (self.rope_size,))
        positions = inputs.get("positions")
        if positions is not None:
            if positions.shape != (tokens,):
                self._refuse("positions", positions, f"[{tokens}]")
            positions = self._whole("positions", positions, torch.int32, ())
        A.APPEND_ARGS.pack_into(self._args, 0, A.APPEND_ARGS.size, latent.data_ptr(), latent_stride, norm, eps, query_address, q[0], q[1],
                                out_address, o[0], o[1], table_address, table.shape[0], 1 if inputs.get("interleaved") else 0, positions or 0, tokens,
                                *self._step(inputs), self._stream(inputs))
        rc = self._append(self._h, self._args)
        if rc:
            self._check(rc)

    def attend(self, inputs: dict, outputs: dict, form: str = "auto") -> None:
        """inputs: query_nope [T, heads, nope], query_rope [T, heads, rope] (rotated), key_up [heads, nope, latent],
        value_up [heads, value, latent], scale (default 1/sqrt(nope + rope)), cache and the paged metadata.
        outputs: output [T, heads * value].  form: "absorbed", "expanded", or "auto": each sequence in the one that suits it, which the device finds out.
        A step known to hold single tokens and drafts only ("absorbed"), or prompts only ("expanded"), is faster by name and takes less scratch."""
        self._form(form)
        nope, rope, key_up, value_up, output = inputs["query_nope"], inputs["query_rope"], inputs["key_up"], inputs["value_up"], outputs["output"]
        n, r = self._rows("query_nope", nope, self._nope_shape), self._rows("query_rope", rope, self._rope_shape)
        k, v = self._rows("key_up", key_up, self._key_shape), self._rows("value_up", value_up, self._value_shape)
        out = self._whole("output", output, self.dtype, self._output_shape)
        tokens = nope.shape[0]
        if rope.shape[0] != tokens or output.shape[0] != tokens:
            raise self._err("query_nope, query_rope and output need the same number of tokens")
        if key_up.shape[0] != self.num_heads or value_up.shape[0] != self.num_heads:
            raise self._err(f"key_up and value_up need {self.num_heads} heads")
        if k[1] != self.latent_size or v[1] != self.latent_size:
            raise self._err("key_up and value_up: a head's rows have to be contiguous")
        A.ATTENTION_ARGS.pack_into(self._args, 0, A.ATTENTION_ARGS.size, nope.data_ptr(), n[0], n[1], rope.data_ptr(), r[0], r[1], key_up.data_ptr(), k[0],
                                   value_up.data_ptr(), v[0], out, tokens, *self._step(inputs), inputs.get("scale") or 0.0, _FORMS[form], self._stream(inputs))
        rc = self._attend(self._h, self._args)
        if rc:
            self._check(rc)

    def reserve(self, num_tokens: int, num_sequences: int, num_block_indices: int, form: str = "auto") -> None:
        """Grows the scratch for steps of up to this size, so that `attend` does not allocate (inside a stream capture it would be refused).  A
        captured graph needs the operator for as long as it is replayed."""
        self._check(self.lib.pa_b200_latent_reserve(self._h, num_tokens, num_sequences, num_block_indices, self._form(form)))

    def device_status(self) -> int:
        """Reads and clears the device status word (PA_DEV_* bits)."""
        bits = C.c_uint32(0)
        self._check(self.lib.pa_b200_latent_last_device_status(self._h, C.byref(bits)))
        return bits.value

    def launch_count(self) -> int:
        return int(self.lib.pa_b200_latent_launch_count(self._h))
