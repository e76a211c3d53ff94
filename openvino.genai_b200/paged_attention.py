"""Host-side mirror of the PagedAttentionExtension operator interface.

The reference reaches this operator through named model tensors that ModelRunner::forward fills
(src/cpp/src/continuous_batching/model_runner.hpp:505-522, 802-853, 1420-1509); an OpenVINO
extension op would receive the same tensors in `evaluate(outputs, inputs)`
(tests/cpp/custom_op/custom_add.cpp:49-80).  `PagedAttentionExtension.evaluate` takes them by
those names and forwards to the C ABI: device tensors go to pa_b200_forward, host tensors to
pa_b200_forward_host.  Errors raise GenaiB200Error where the reference raises ov::Exception.

A step whose inputs name `sink_tokens` (with `sliding_window`) or `tree_parents` goes to pa_b200_forward_masked
(include/masked_b200.h): rows see a window of their context and its first few tokens, or the tree of drafts that they are part
of.  `tree_accept` follows the sampled tokens down the trees behind such a step and moves what was accepted.
"""
from __future__ import annotations

import ctypes as C
import operator
from typing import Optional

import numpy as np
import torch

from . import _abi, _masked_abi as M

_ACT = {torch.float32: _abi.PA_DTYPE_F32, torch.float16: _abi.PA_DTYPE_F16, torch.bfloat16: _abi.PA_DTYPE_BF16}
_CACHE = {"f16": _abi.PA_DTYPE_F16, "bf16": _abi.PA_DTYPE_BF16, "u8": _abi.PA_DTYPE_U8}


def _ptr(t) -> Optional[int]:
    if t is None:
        return None
    if isinstance(t, np.ndarray):
        return t.ctypes.data
    return t.data_ptr()


_nbytes = operator.attrgetter("nbytes")


def _alike(tensors) -> bool:
    """Whether all of them are contiguous tensors of one size in bytes on one device."""
    T = torch.Tensor
    try:
        return all(map(T.is_contiguous, tensors)) and len(set(map(T.get_device, tensors))) <= 1 and len(set(map(_nbytes, tensors))) <= 1
    except TypeError:    # (not all of them are tensors)
        return False


class PagedAttentionExtension:
    """One attention layer's operator instance (owns a C-ABI handle and its scratch)."""

    TREE_NONE = M.PA_TREE_NONE

    def __init__(self, num_q_heads: int, num_kv_heads: int, head_size: int, block_size: int,
                 act_dtype: torch.dtype = torch.float16, cache_dtype: str = "f16", device: int = 0):
        from . import GenaiB200Error, load_library
        self._err = GenaiB200Error
        self.lib = load_library()
        self.desc = _abi.pa_model_desc(C.sizeof(_abi.pa_model_desc), num_q_heads, num_kv_heads, head_size, block_size,
                                       _ACT[act_dtype], _CACHE[cache_dtype])
        self.act_dtype = act_dtype
        self.cache_dtype = cache_dtype
        self.device = device
        self.num_q_heads, self.num_kv_heads, self.head_size, self.block_size = num_q_heads, num_kv_heads, head_size, block_size
        self._h = C.c_void_p()
        self._where = torch.device("cuda", device)
        self._cache_bytes = 0    # of a block: asked for once
        self._forward_buffer, self._mask_buffer, self._accept_buffer = (C.create_string_buffer(p.size) for p in (M.FORWARD_ARGS, M.MASK_ARGS, M.ACCEPT_ARGS))
        self._check(self.lib.pa_b200_create(C.byref(self.desc), device, C.byref(self._h)))

    def __del__(self):
        h = getattr(self, "_h", None)
        if h:
            self.lib.pa_b200_destroy(h)
            self._h = None

    def _check(self, rc: int) -> None:
        if rc != _abi.PA_OK:
            raise self._err(f"pa_b200 status {rc}: {self.lib.pa_b200_last_error().decode()}")

    # ---- cache ---------------------------------------------------------------------------------
    def cache_layout(self) -> _abi.pa_cache_layout:
        out = _abi.pa_cache_layout()
        out.struct_size = C.sizeof(_abi.pa_cache_layout)
        self._check(self.lib.pa_b200_query_cache_layout(C.byref(self.desc), C.byref(out)))
        return out

    def allocate_cache(self, num_blocks: int, fill: Optional[int] = 0):
        """Returns (key_cache, value_cache) as flat uint8 device tensors of the declared byte size."""
        lay = self.cache_layout()
        dev = torch.device("cuda", self.device)
        mk = (lambda n: torch.full((n,), fill, dtype=torch.uint8, device=dev)) if fill is not None else \
             (lambda n: torch.empty((n,), dtype=torch.uint8, device=dev))
        return mk(num_blocks * lay.key_block_bytes), mk(num_blocks * lay.value_block_bytes)

    # ---- the operator --------------------------------------------------------------------------
    def make_args(self, query, key, value, output, key_cache, value_cache, past_lens, subsequence_begins, block_indices,
                  block_indices_begins, scale=None, max_context_len=None, score_aggregation_window=None, scores=None,
                  rotated_block_indices=None, rotation_deltas=None, rotation_trig_lut=None, stream=None,
                  sliding_window=0, alibi_slopes=None) -> _abi.pa_forward_args:
        a = _abi.pa_forward_args()
        a.struct_size = C.sizeof(_abi.pa_forward_args)
        a.query, a.key, a.value, a.output = _ptr(query), _ptr(key), _ptr(value), _ptr(output)
        a.num_tokens = int(query.shape[0])
        a.key_cache, a.value_cache = _ptr(key_cache), _ptr(value_cache)
        lay = self.cache_layout()
        a.num_blocks = int(key_cache.numel() // lay.key_block_bytes)
        a.past_lens, a.subsequence_begins = _ptr(past_lens), _ptr(subsequence_begins)
        a.block_indices, a.block_indices_begins = _ptr(block_indices), _ptr(block_indices_begins)
        a.num_sequences = int(past_lens.shape[0])
        a.num_block_indices = int(block_indices.shape[0])
        a.max_context_len = int(max_context_len) if max_context_len is not None else 0
        a.scale = float(scale) if scale is not None else 0.0
        a.sliding_window = int(sliding_window)
        a.alibi_slopes = _ptr(alibi_slopes)
        a.score_aggregation_window = _ptr(score_aggregation_window)
        a.scores = _ptr(scores)
        a.scores_len = int(scores.shape[0]) if scores is not None else 0
        a.rotated_block_indices = _ptr(rotated_block_indices)
        a.rotation_deltas = _ptr(rotation_deltas)
        a.num_rotated_blocks = int(rotated_block_indices.shape[0]) if rotated_block_indices is not None else 0
        a.rotation_trig_lut = _ptr(rotation_trig_lut)
        a.rotation_lut_rows = int(rotation_trig_lut.shape[0]) if rotation_trig_lut is not None else 0
        if stream is None and isinstance(query, torch.Tensor) and query.is_cuda:
            stream = torch.cuda.current_stream(query.device).cuda_stream  # order after the caller's torch work
        if stream == 0:
            stream = 1  # cudaStreamLegacy: NULL would select the handle's own stream instead of the default stream
        a.stream = stream
        # the struct holds raw addresses: keep every buffer alive for as long as the struct is
        a._buffers = (query, key, value, output, key_cache, value_cache, past_lens, subsequence_begins, block_indices,
                      block_indices_begins, alibi_slopes, score_aggregation_window, scores, rotated_block_indices,
                      rotation_deltas, rotation_trig_lut)
        return a

    def forward_args(self, args: _abi.pa_forward_args, host: bool = False) -> None:
        fn = self.lib.pa_b200_forward_host if host else self.lib.pa_b200_forward
        self._check(fn(self._h, C.byref(args)))

    def evaluate(self, inputs: dict, outputs: dict) -> None:
        """inputs / outputs are keyed by the reference's tensor names; `output` (and `scores`)
        must be preallocated by the caller, who owns every buffer.

        Masks: `sink_tokens` S with `sliding_window` W leaves a row at position p the cached positions above p - W and those below S (a window
        without sinks has S = 0; without S `sliding_window` is refused, as it is of a causal step); `tree_parents` (i32 [T], an index among the sequence's new tokens that is smaller than the token's own, -1: it follows
        the last cached token, TREE_NONE at a sequence's first token: no tree) makes a sequence's new tokens a tree of drafts, whose rows
        see the cache, their ancestors and themselves, at position past_len + depth.  Blocks that no row sees are not looked up.  A step under
        a mask has no `scores`."""
        sinks, parents = inputs.get("sink_tokens"), inputs.get("tree_parents")
        if sinks is not None or parents is not None:
            self._evaluate_masked(inputs, outputs, self._count("sliding_window", inputs.get("sliding_window") or 0), self._count("sink_tokens", sinks or 0), parents)
            return
        q = inputs["query"]
        host = isinstance(q, np.ndarray) or (isinstance(q, torch.Tensor) and not q.is_cuda)
        mcl = inputs.get("max_context_len")
        if mcl is not None and not isinstance(mcl, int):
            mcl = int(mcl.item() if hasattr(mcl, "item") else mcl)
        args = self.make_args(q, inputs["key"], inputs["value"], outputs["output"], inputs["key_cache"], inputs["value_cache"],
                              inputs["past_lens"], inputs["subsequence_begins"], inputs["block_indices"],
                              inputs["block_indices_begins"], inputs.get("scale"), mcl,
                              inputs.get("score_aggregation_window"), outputs.get("scores"),
                              inputs.get("rotated_block_indices"), inputs.get("rotation_deltas"),
                              inputs.get("rotation_trig_lut"), inputs.get("stream"),
                              inputs.get("sliding_window", 0), inputs.get("alibi_slopes"))
        self.forward_args(args, host=host)

    # ---- masked steps --------------------------------------------------------------------------
    # (the checks run before every launch: a small step's time is the host's)
    def _refuse(self, name: str, t, expected: str):
        what = f"{t.dtype} {tuple(t.shape)}, strides {t.stride()}, on {t.device}" if isinstance(t, torch.Tensor) else type(t).__name__
        raise self._err(f"{name}: expected {expected} on {self._where}, got {what}")

    def _count(self, name: str, n) -> int:
        try:
            n = operator.index(n)
        except TypeError:
            n = -1
        if not 0 <= n < 1 << 31:
            raise self._err(f"{name}: expected a whole number from 0 to 2^31 - 1")
        return n

    def _whole(self, name: str, t, dtype: torch.dtype, shape: tuple) -> int:
        """The address of a contiguous device tensor of this type and shape."""
        try:
            if t.dtype is dtype and t.shape == shape and t.get_device() == self.device and t.is_contiguous():
                return t.data_ptr()
        except (AttributeError, TypeError):
            pass
        self._refuse(name, t, f"contiguous {dtype} {list(shape)}")

    def _blocks(self, name: str, t) -> int:
        """Blocks of a cache tensor: contiguous, of any type, in the operator's layout."""
        if not self._cache_bytes:
            self._cache_bytes = self.cache_layout().key_block_bytes
        if isinstance(t, torch.Tensor) and t.get_device() == self.device and t.is_contiguous():
            blocks, rest = divmod(t.numel() * t.element_size(), self._cache_bytes)
            if not rest:
                return blocks
        self._refuse(name, t, f"a contiguous tensor of whole blocks of {self._cache_bytes} bytes")

    def _paged(self, inputs: dict) -> tuple:
        """Addresses of the paged metadata, number of sequences and of block indices."""
        past, blocks = inputs["past_lens"], inputs["block_indices"]
        B, n = past.shape[0] if isinstance(past, torch.Tensor) and past.dim() else 0, blocks.shape[0] if isinstance(blocks, torch.Tensor) and blocks.dim() else 0
        i32, whole = torch.int32, self._whole
        return (whole("past_lens", past, i32, (B,)), whole("subsequence_begins", inputs["subsequence_begins"], i32, (B + 1,)),
                whole("block_indices", blocks, i32, (n,)), whole("block_indices_begins", inputs["block_indices_begins"], i32, (B + 1,))), B, n

    def _stream(self, inputs: dict) -> int:
        # 1 = cudaStreamLegacy: a null handle would select the operator's own stream
        return inputs.get("stream") or torch._C._cuda_getCurrentRawStream(self.device) or 1

    def _evaluate_masked(self, inputs: dict, outputs: dict, window: int, sinks: int, parents) -> None:
        if inputs.get("score_aggregation_window") is not None or outputs.get("scores") is not None:
            raise self._err("a masked step has no score output")
        if inputs.get("alibi_slopes") is not None:
            raise self._err("alibi_slopes is not supported")
        query, key_cache, value_cache = inputs["query"], inputs["key_cache"], inputs["value_cache"]
        limit = inputs.get("max_context_len")
        limit = 0 if limit is None else int(limit)
        scale = inputs.get("scale")
        scale = 0.0 if scale is None else float(scale)
        if isinstance(query, np.ndarray) or (isinstance(query, torch.Tensor) and not query.is_cuda):
            if parents is not None and (parents.shape != (query.shape[0],) or str(parents.dtype).split(".")[-1] != "int32" or getattr(parents, "is_cuda", False) or
                                        not (parents.flags.c_contiguous if isinstance(parents, np.ndarray) else parents.is_contiguous())):
                raise self._err("tree_parents: expected contiguous host int32 of one entry per token")
            args = self.make_args(query, inputs["key"], inputs["value"], outputs["output"], key_cache, value_cache, inputs["past_lens"], inputs["subsequence_begins"],
                                  inputs["block_indices"], inputs["block_indices_begins"], scale, limit, None, None, inputs.get("rotated_block_indices"),
                                  inputs.get("rotation_deltas"), inputs.get("rotation_trig_lut"), inputs.get("stream"))
            mask = M.pa_mask_args(C.sizeof(M.pa_mask_args), window, sinks, _ptr(parents))
            self._check(self.lib.pa_b200_forward_masked_host(self._h, C.byref(args), C.byref(mask)))
            return
        whole, act = self._whole, self.act_dtype
        T = query.shape[0] if isinstance(query, torch.Tensor) and query.dim() else 0
        rows, kv_rows = (T, self.num_q_heads * self.head_size), (T, self.num_kv_heads * self.head_size)
        meta, B, num_indices = self._paged(inputs)
        num_blocks = self._blocks("key_cache", key_cache)
        if self._blocks("value_cache", value_cache) != num_blocks:
            raise self._err("key_cache and value_cache differ in blocks")
        rotated = (0, 0, 0, 0, 0)
        if inputs.get("rotated_block_indices") is not None:
            blocks, table = inputs["rotated_block_indices"], inputs["rotation_trig_lut"]
            n = blocks.shape[0]
            rotated = (whole("rotated_block_indices", blocks, torch.int32, (n,)),
                       whole("rotation_deltas", inputs["rotation_deltas"], torch.int32, tuple(inputs["rotation_deltas"].shape) if inputs["rotation_deltas"].numel() == n else (n,)),
                       n, whole("rotation_trig_lut", table, torch.float32, (table.shape[0], self.head_size)), table.shape[0])
        M.FORWARD_ARGS.pack_into(self._forward_buffer, 0, M.FORWARD_ARGS.size, whole("query", query, act, rows), whole("key", inputs["key"], act, kv_rows),
                                 whole("value", inputs["value"], act, kv_rows), whole("output", outputs["output"], act, rows), T, key_cache.data_ptr(),
                                 value_cache.data_ptr(), num_blocks, *meta, B, num_indices, limit, scale, 0, 0, 0, 0, 0, *rotated, self._stream(inputs))
        M.MASK_ARGS.pack_into(self._mask_buffer, 0, M.MASK_ARGS.size, window, sinks, 0 if parents is None else whole("tree_parents", parents, torch.int32, (T,)))
        rc = self.lib.pa_b200_forward_masked(self._h, self._forward_buffer, self._mask_buffer)
        if rc:
            self._check(rc)

    def masked_reserve(self, num_tokens: int, num_sequences: int, num_block_indices: int) -> None:
        """Grows the scratch for masked steps of up to this size, so that they do not allocate (inside a stream capture they would be
        refused).  A captured graph needs the operator for as long as it is replayed."""
        self._check(self.lib.pa_b200_masked_reserve(self._h, num_tokens, num_sequences, num_block_indices))

    def tree_accept(self, inputs: dict, outputs: dict) -> None:
        """Judges trees of drafts behind a step that had them, and makes the accepted tokens the cache's newest.

        inputs: tree_parents i32 [T] (as `evaluate` takes it), draft_tokens i64 [T] (the step's input ids; a sequence's first one is
        certain), sampled_tokens i64 [T] (what was sampled behind each of them), the paged metadata, and key_caches / value_caches: a
        sequence of the layers' caches, or a tensor of them one behind the other (may be left out: nothing is moved).  From an accepted token the path goes on to its
        first child whose id was sampled behind it.
        outputs: path i32 [B, max_path] (accepted tokens, -1 behind them), num_accepted i32 [B], next_token i64 [B] (sampled behind
        the last accepted token), new_past_lens i32 [B] (optional, may be past_lens).  A sequence without a tree keeps all its tokens."""
        whole, i32, i64 = self._whole, torch.int32, torch.int64
        parents, path = inputs["tree_parents"], outputs["path"]
        T = parents.shape[0] if isinstance(parents, torch.Tensor) and parents.dim() else 0
        meta, B, num_indices = self._paged(inputs)
        keys, values = (() if inputs.get(name) is None else inputs[name] for name in ("key_caches", "value_caches"))
        if len(keys) != len(values):
            raise self._err("key_caches and value_caches differ in layers")
        caches = (*keys, *values)
        if not _alike(caches):    # (a model's worth of tensors: who is not like the others is asked for by name)
            counts = {self._blocks("key_caches and value_caches", t) for t in caches}
            if len(counts) > 1:
                raise self._err("the layers' caches differ in blocks")
        num_blocks = self._blocks("key_caches", caches[0]) if caches else 0
        if not isinstance(path, torch.Tensor) or path.dim() != 2:
            self._refuse("path", path, "contiguous int32 [sequences, max_path]")
        layers = len(keys)
        addresses = tuple((C.c_void_p * layers)(*map(torch.Tensor.data_ptr, group)) for group in (keys, values))
        past_out = outputs.get("new_past_lens")
        M.ACCEPT_ARGS.pack_into(self._accept_buffer, 0, M.ACCEPT_ARGS.size, whole("tree_parents", parents, i32, (T,)),
                                whole("draft_tokens", inputs["draft_tokens"], i64, (T,)), whole("sampled_tokens", inputs["sampled_tokens"], i64, (T,)), *meta, T, B,
                                num_indices, num_blocks, path.shape[1], layers, C.addressof(addresses[0]), C.addressof(addresses[1]),
                                whole("path", path, i32, (B, path.shape[1])), whole("num_accepted", outputs["num_accepted"], i32, (B,)),
                                whole("next_token", outputs["next_token"], i64, (B,)), 0 if past_out is None else whole("new_past_lens", past_out, i32, (B,)),
                                self._stream(inputs))
        rc = self.lib.pa_b200_tree_accept(self._h, self._accept_buffer)
        if rc:
            self._check(rc)

    def device_status(self) -> int:
        bits = C.c_uint32(0)
        self._check(self.lib.pa_b200_last_device_status(self._h, C.byref(bits)))
        return bits.value

    def launch_count(self) -> int:
        return int(self.lib.pa_b200_launch_count(self._h))

    def last_prefill_kernel(self) -> str:
        """Which kernel served the prefill chunks of the last forward call: "none", "generic", "mma_sync" or "tcgen05"."""
        return ("none", "generic", "mma_sync", "tcgen05")[int(self.lib.pa_b200_last_prefill_kernel(self._h))]

    def copy_blocks(self, key_cache, value_cache, pairs, stream=None) -> None:
        lay = self.cache_layout()
        self._check(self.lib.pa_b200_copy_blocks(self._h, _ptr(key_cache), _ptr(value_cache),
                                                 int(key_cache.numel() // lay.key_block_bytes), _ptr(pairs),
                                                 int(pairs.shape[0]), stream))
