"""The argument structs of the vocabulary-table operators: header and ctypes mirror agree, and so does the packed form adamw_multi passes."""
import ctypes
import struct

import pytest

from open_flamingo_amd.hip import abi
from tests.test_abi_layout import _c_layout


@pytest.mark.parametrize("name,mirror", [("OfLinearCeArgs", abi.OfLinearCeArgs), ("OfAdamwTensor", abi.OfAdamwTensor)])
def test_ctypes_mirror_has_the_layout_of_the_header(tmp_path, name, mirror):
    names = [f[0] for f in mirror._fields_]
    c = _c_layout(tmp_path, name, names)
    assert c["sizeof"] == ctypes.sizeof(mirror)
    assert all(c[n] == getattr(mirror, n).offset for n in names)


def test_packed_tensor_descriptions():
    t = abi.OfAdamwTensor.from_buffer_copy(struct.pack("=7q2fi4x", 1, 2, 3, 4, 5, 6, 7, 0.5, 0.25, 1))
    assert ctypes.sizeof(t) == struct.calcsize("=7q2fi4x")
    assert (t.p, t.g, t.m, t.v, t.m_scale, t.v_scale, t.n, t.lr, t.weight_decay, t.g_bf16) == (1, 2, 3, 4, 5, 6, 7, 0.5, 0.25, 1)
