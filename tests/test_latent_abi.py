"""Latent attention's C ABI without a GPU: the struct layouts agree with the header, arguments are refused with a status and a text."""
import ctypes as C
import re
from pathlib import Path

import pytest

HEADER = Path(__file__).resolve().parent.parent / "include" / "latent_b200.h"


@pytest.fixture(scope="module")
def lib(pkg):
    pkg.build_all()
    return pkg.load_library()


@pytest.mark.parametrize("name", ["pa_latent_desc", "pa_latent_append_args", "pa_latent_attention_args"])
def test_the_mirror_has_the_header_s_fields(pkg, name):
    from openvino_genai_b200 import _latent_abi
    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), text, flags=re.S).group(1)
    kinds = {"uint32_t": C.c_uint32, "int32_t": C.c_int32, "int64_t": C.c_int64, "float": C.c_float}
    want = []
    for line in filter(None, (p.strip() for p in body.split(";"))):
        m = re.match(r"(?:const )?(\w+)(\s*\*)?\s*(.*)", line, flags=re.S)
        for field in m.group(3).split(","):
            want.append((field.strip(), C.c_void_p if m.group(2) else kinds[m.group(1)]))
    assert want == list(getattr(_latent_abi, name)._fields_)


def test_descriptors_and_handles_are_refused(lib):
    from openvino_genai_b200 import _abi, _latent_abi as A
    h = C.c_void_p()
    good = [C.sizeof(A.pa_latent_desc), 16, 512, 64, 128, 128, 32, _abi.PA_DTYPE_BF16]
    for at, value, status in ((0, 4, 1), (1, 0, 1), (1, 1025, 1), (2, 384, 2), (3, 16, 2), (4, 96, 2), (5, 192, 2), (6, 128, 2), (7, _abi.PA_DTYPE_F32, 2)):
        bad = list(good)
        bad[at] = value
        assert lib.pa_b200_latent_create(C.byref(A.pa_latent_desc(*bad)), 0, C.byref(h)) == status
        assert lib.pa_b200_last_error() and not h
    assert lib.pa_b200_latent_create(None, 0, C.byref(h)) == 1
    assert lib.pa_b200_latent_append(None, C.byref(A.pa_latent_append_args())) == 1
    assert lib.pa_b200_latent_attention(None, C.byref(A.pa_latent_attention_args())) == 1
    assert lib.pa_b200_latent_last_device_status(None, None) == 1
    assert lib.pa_b200_latent_launch_count(None) == -1
    assert lib.pa_b200_latent_destroy(None) == 0
