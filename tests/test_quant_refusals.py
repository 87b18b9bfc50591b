"""What the C entry points of the quantised cache refuse before anything is launched: no device is needed, and no address here is one."""
import ctypes

import pytest

from kipp_b200.csrc.build import load_library
from kipp_b200.kernels import cache_quant as C

AT = 1 << 20                                               # an address on every boundary


def call(lib, name, layout, fields, change):
    """The entry point's answer to its structure with some fields changed."""
    assert not set(change) - set(fields)
    f = getattr(load_library(lib), name)
    f.argtypes, f.restype = [ctypes.c_char_p], ctypes.c_int
    return f(layout.pack(*{**fields, **change}.values()))


WRITE = dict(qkv=AT, q_out=AT, k_codes=AT, k_scales=AT, v_codes=AT, v_scales=AT, q_norm=0, k_norm=0, cos_sin=AT, positions=AT, entry_of_token=AT,
             block_table=AT, status=AT, stream=0, ld=512, bits=8, n_pages=4, page_size=16, dtype=0, norm_dtype=0, rotary_dim=64, table_width=2,
             tokens=3, n_q=4, n_kv=2, head_dim=64, write_cache=1, eps=1e-6)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("off", [1, 2, 4])
def test_angles_off_their_boundary(off, dtype, bits):
    """A rotation's cosine and sine are read as one eight-byte number."""
    assert call("cache_quant", "kipp_quant_cache_write", C._WRITE, WRITE, dict(cos_sin=AT + off, dtype=dtype, bits=bits)) == -3
