"""ctypes mirror of include/latent_b200.h (struct layouts and prototypes)."""
from __future__ import annotations

import ctypes as C
import struct

PA_LATENT_AUTO = 0
PA_LATENT_ABSORBED = 1
PA_LATENT_EXPANDED = 2
PA_DEV_WAIT_TIMEOUT_LATENT = 0x10000000


class pa_latent_desc(C.Structure):
    _fields_ = [("struct_size", C.c_uint32)] + [(n, C.c_int32) for n in (
        "num_heads", "latent_size", "rope_size", "nope_size", "value_size", "block_size", "dtype")]


class pa_latent_append_args(C.Structure):
    _fields_ = [
        ("struct_size", C.c_uint32),
        ("latent", C.c_void_p),
        ("latent_stride", C.c_int64),
        ("norm_weight", C.c_void_p),
        ("norm_eps", C.c_float),
        ("query_rope", C.c_void_p),
        ("query_rope_token_stride", C.c_int64),
        ("query_rope_head_stride", C.c_int64),
        ("query_rope_out", C.c_void_p),
        ("query_rope_out_token_stride", C.c_int64),
        ("query_rope_out_head_stride", C.c_int64),
        ("rope_table", C.c_void_p),
        ("rope_table_rows", C.c_int32),
        ("interleaved", C.c_int32),
        ("positions", C.c_void_p),
        ("num_tokens", C.c_int32),
        ("cache", C.c_void_p),
        ("num_blocks", C.c_int32),
        ("past_lens", C.c_void_p),
        ("subsequence_begins", C.c_void_p),
        ("block_indices", C.c_void_p),
        ("block_indices_begins", C.c_void_p),
        ("num_sequences", C.c_int32),
        ("num_block_indices", C.c_int32),
        ("stream", C.c_void_p),
    ]


class pa_latent_attention_args(C.Structure):
    _fields_ = [
        ("struct_size", C.c_uint32),
        ("query_nope", C.c_void_p),
        ("query_nope_token_stride", C.c_int64),
        ("query_nope_head_stride", C.c_int64),
        ("query_rope", C.c_void_p),
        ("query_rope_token_stride", C.c_int64),
        ("query_rope_head_stride", C.c_int64),
        ("key_up", C.c_void_p),
        ("key_up_head_stride", C.c_int64),
        ("value_up", C.c_void_p),
        ("value_up_head_stride", C.c_int64),
        ("output", C.c_void_p),
        ("num_tokens", C.c_int32),
        ("cache", C.c_void_p),
        ("num_blocks", C.c_int32),
        ("past_lens", C.c_void_p),
        ("subsequence_begins", C.c_void_p),
        ("block_indices", C.c_void_p),
        ("block_indices_begins", C.c_void_p),
        ("num_sequences", C.c_int32),
        ("num_block_indices", C.c_int32),
        ("scale", C.c_float),
        ("form", C.c_int32),
        ("stream", C.c_void_p),
    ]


_FORMAT = {C.c_uint32: "I", C.c_int32: "i", C.c_int64: "q", C.c_float: "f", C.c_void_p: "P"}


def packer(args) -> struct.Struct:
    """Writes all fields of an argument struct at once: filling a ctypes structure costs several times as much, which single rows notice."""
    p = struct.Struct("@" + "".join(_FORMAT[kind] for _, kind in args._fields_))
    assert p.size == C.sizeof(args)
    return p


APPEND_ARGS = packer(pa_latent_append_args)
ATTENTION_ARGS = packer(pa_latent_attention_args)

LATENT_SYMBOLS = {
    "pa_b200_latent_create": (C.c_int, [C.POINTER(pa_latent_desc), C.c_int, C.POINTER(C.c_void_p)]),
    "pa_b200_latent_destroy": (C.c_int, [C.c_void_p]),
    "pa_b200_latent_append": (C.c_int, [C.c_void_p, C.c_void_p]),
    "pa_b200_latent_attention": (C.c_int, [C.c_void_p, C.c_void_p]),
    "pa_b200_latent_reserve": (C.c_int, [C.c_void_p, C.c_int32, C.c_int32, C.c_int32, C.c_int32]),
    "pa_b200_latent_last_device_status": (C.c_int, [C.c_void_p, C.POINTER(C.c_uint32)]),
    "pa_b200_latent_launch_count": (C.c_int64, [C.c_void_p]),
}
