"""ctypes mirror of include/masked_b200.h (struct layouts and prototypes)."""
from __future__ import annotations

import ctypes as C

from ._abi import pa_forward_args
from ._latent_abi import packer

PA_DEV_BAD_TREE = 0x10
PA_TREE_MAX_TOKENS = 256
PA_TREE_NONE = -2


class pa_mask_args(C.Structure):
    _fields_ = [("struct_size", C.c_uint32), ("sliding_window", C.c_int32), ("sink_tokens", C.c_int32), ("tree_parents", C.c_void_p)]


class pa_tree_accept_args(C.Structure):
    _fields_ = [
        ("struct_size", C.c_uint32),
        ("tree_parents", C.c_void_p),
        ("draft_tokens", C.c_void_p),
        ("sampled_tokens", C.c_void_p),
        ("past_lens", C.c_void_p),
        ("subsequence_begins", C.c_void_p),
        ("block_indices", C.c_void_p),
        ("block_indices_begins", C.c_void_p),
        ("num_tokens", C.c_int32),
        ("num_sequences", C.c_int32),
        ("num_block_indices", C.c_int32),
        ("num_blocks", C.c_int32),
        ("max_path", C.c_int32),
        ("num_layers", C.c_int32),
        ("key_caches", C.c_void_p),
        ("value_caches", C.c_void_p),
        ("path", C.c_void_p),
        ("num_accepted", C.c_void_p),
        ("next_token", C.c_void_p),
        ("new_past_lens", C.c_void_p),
        ("stream", C.c_void_p),
    ]


FORWARD_ARGS, MASK_ARGS, ACCEPT_ARGS = packer(pa_forward_args), packer(pa_mask_args), packer(pa_tree_accept_args)

MASKED_SYMBOLS = {
    "pa_b200_forward_masked": (C.c_int, [C.c_void_p, C.c_void_p, C.c_void_p]),
    "pa_b200_forward_masked_host": (C.c_int, [C.c_void_p, C.POINTER(pa_forward_args), C.POINTER(pa_mask_args)]),
    "pa_b200_masked_reserve": (C.c_int, [C.c_void_p, C.c_int32, C.c_int32, C.c_int32]),
    "pa_b200_tree_accept": (C.c_int, [C.c_void_p, C.c_void_p]),
}
