"""The C entries of the paged operators refuse on the host what their kernels do not take (no pointer below is followed)."""

import ctypes
from ctypes import Structure, c_float, c_int32, c_int64, c_void_p

import pytest

from generative_recommenders_b200 import _cabi

I64 = c_int64


class Cache(Structure):
    _fields_ = [("pages", c_void_p), ("page_table", c_void_p), ("num_pages", I64), ("table_stride", I64), ("B", c_int32),
                ("H", c_int32), ("d", c_int32), ("page_size", c_int32), ("table_width", c_int32), ("reserved0", c_int32)]


class NormRotary(Structure):
    _fields_ = [("x", c_void_p * 2), ("y", c_void_p * 2), ("dy", c_void_p * 2), ("dx", c_void_p * 2), ("weight", c_void_p * 2),
                ("dweight", c_void_p * 2), ("positions", c_void_p), ("cos", c_void_p), ("sin", c_void_p), ("workspace", c_void_p),
                ("workspace_bytes", I64), ("x_row_stride", I64 * 2), ("x_head_stride", I64 * 2), ("dy_row_stride", I64 * 2),
                ("dy_head_stride", I64 * 2), ("rows", I64), ("table_rows", I64), ("H", c_int32 * 2), ("weight_dtype", c_int32 * 2),
                ("d", c_int32), ("rotary", c_int32), ("interleaved", c_int32), ("index_flags", c_int32), ("dtype", c_int32),
                ("eps", c_float)]


class Read(Structure):
    _fields_ = [("cache", Cache), ("k", c_void_p), ("v", c_void_p), ("seq_offsets", c_void_p), ("rows", I64),
                ("index_flags", c_int32), ("dtype", c_int32)]


class Attn(Structure):
    _fields_ = [("cache", Cache), ("q", c_void_p), ("out", c_void_p), ("seq_lengths", c_void_p), ("q_offsets", c_void_p),
                ("num_targets", c_void_p), ("workspace", c_void_p), ("workspace_bytes", I64), ("q_row_stride", I64),
                ("q_head_stride", I64), ("rows", I64), ("Hq", c_int32), ("max_attn_len", c_int32),
                ("contextual_seq_len", c_int32), ("softmax", c_int32), ("index_flags", c_int32), ("dtype", c_int32),
                ("alpha", c_float), ("scale", c_float)]


def cache():
    return Cache(pages=256, page_table=256, num_pages=4, table_stride=2, B=2, H=2, d=64, page_size=16, table_width=2)


def call(name, args):
    lib = ctypes.CDLL(_cabi.LIB_PATH)
    lib.b200_hstu_last_error.restype = ctypes.c_char_p
    return getattr(lib, name)(ctypes.byref(args), None), lib.b200_hstu_last_error() or b""


@pytest.mark.parametrize("field", ["k", "v"])
@pytest.mark.parametrize("at", [258, 260, 264])
def test_read_into_an_address_of_no_vector(field, at):
    a = Read(cache=cache(), k=256, v=256, seq_offsets=256, rows=4, dtype=_cabi.F32)
    setattr(a, field, at)
    rc, why = call("b200_hstu_paged_read", a)
    assert rc == -1 and b"aligned" in why


def attn(**other):
    a = Attn(cache=cache(), q=256, out=256, seq_lengths=256, q_offsets=256, workspace=256, workspace_bytes=1 << 40,
             q_row_stride=128, q_head_stride=64, rows=4, Hq=2, dtype=_cabi.BF16, alpha=1.0, scale=1.0)
    for name, value in other.items():
        setattr(a, name, value)
    return a


@pytest.mark.parametrize("field", ["out", "workspace"])
def test_attention_into_an_address_of_no_vector(field):
    rc, why = call("b200_hstu_paged_attn_fwd", attn(**{field: 264}))
    assert rc == -1 and b"aligned" in why


@pytest.mark.parametrize("rows", [-1, 1 << 31, 1 << 62, (1 << 62) + 1])
def test_numbers_of_rows_that_overflow(rows):
    rc, why = call("b200_hstu_paged_attn_fwd", attn(rows=rows, Hq=4))
    assert rc == -1 and b"rows" in why
    lib = ctypes.CDLL(_cabi.LIB_PATH)
    lib.b200_hstu_paged_attn_workspace_bytes.restype = I64
    assert lib.b200_hstu_paged_attn_workspace_bytes(ctypes.byref(attn(rows=rows, Hq=4))) == 0


@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("backward", [False, True])
def test_norm_and_rotation_into_an_address_of_no_vector(backward, which):
    a = NormRotary(rows=4, d=64, dtype=_cabi.F32, eps=1e-6)
    for i in range(2):
        a.x[i] = a.y[i] = a.dy[i] = a.dx[i] = 256
        a.H[i] = 2
    (a.dx if backward else a.y)[which] = 264
    rc, why = call("b200_hstu_norm_rotary_" + ("bwd" if backward else "fwd"), a)
    assert rc == -1 and b"aligned" in why
