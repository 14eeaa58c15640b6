"""Low-bit formats on the CPU: the oracle against hand-worked values, the C ABI's names, and what calls refuse."""

import re
from pathlib import Path

import numpy as np
import pytest

from oracle import lowbit

REPO = Path(__file__).resolve().parents[1]


def test_mxfp4_values_by_hand():
    x = np.zeros((1, 64))
    # block 0: largest 7 -> scale 1 (2^(2 - 2)); ties go to even codes, 7 saturates
    x[0, :12] = [7.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -5.0, 0.26, -0.24, 6.0]
    x[0, 32:35] = [0.75, 0.1, -0.5]  # largest 0.75: scale 2^-3
    v, byte = lowbit.mxfp4_values(x)
    assert v[0, :12].tolist() == [6.0, 0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0, -4.0, 0.5, -0.0, 6.0]
    assert v[0, 32:35].tolist() == [0.75, 0.125, -0.5]  # 6, 0.8 -> 1, 4 eighths
    assert byte.tolist() == [[127, 124]]


def test_kv8_values_by_hand():
    x = np.zeros((65, 1, 16))
    x[0, 0, :4] = [448.0, 17.0, 19.0, 0.001]  # the last: over half of the least code, 2^-9
    x[64, 0, 0] = 449.0
    v, byte = lowbit.kv8_values(x, "e4m3")
    assert v[0, 0, :4].tolist() == [448.0, 16.0, 20.0, 2.0**-9] and byte[:, 0].tolist() == [127, 128]
    assert v[64, 0, 0] == 448.0  # 224.5 of steps of 16 (times 2)
    v, byte = lowbit.kv8_values(x / 448.0 * 127.0, "int8")
    assert byte[0, 0] == 127 and v[0, 0, 0] == 127.0


def test_every_declared_entry_is_bound():
    from taomate_hd_amd import _native

    text = (REPO / "include" / "tmhd_lowbit.h").read_text()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    declared = set(re.findall(r"\b(tmhd_[a-z0-9_]+)\s*\(", text))
    assert declared == set(_native._LOWBIT_SIGNATURES)


def test_mxfp4_refuses_on_the_host():
    import torch

    import taomate_hd_amd as tm

    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="GPU tensor"):
        tm.mxfp4_quant(x)
    with pytest.raises(ValueError, match="GPU tensor"):
        tm.mxfp4_dequant(torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(1, 4, 4, 4, dtype=torch.uint8))
    with pytest.raises(ValueError, match="uint8"):
        tm.mxfp4_scale_from_rows(torch.zeros(4, 2))
    with pytest.raises(ValueError, match="contiguous uint8"):
        tm.mxfp4_scale_to_rows(torch.zeros(1, 4, 8, 4, dtype=torch.uint8), 4, 64)


def _bad(lib, status):
    return status, lib.tmhd_last_error().decode()


def test_mxfp4_c_entries_refuse():
    """Arguments are checked before anything is launched (no GPU here)."""
    from taomate_hd_amd import _native

    lib = _native.load()
    ok = 4096  # stands for an aligned address that is never read
    q = lib.tmhd_mxfp4_quant
    assert q(ok, ok, ok, 4, 33, 64, None) == _native.TMHD_ERR_UNSUPPORTED
    assert q(ok, ok, ok, -1, 32, 64, None) == _native.TMHD_ERR_INVALID
    assert q(ok, ok, ok, 4, 64, 32, None) == _native.TMHD_ERR_INVALID
    assert q(ok, ok, ok, 4, 64, 68, None) == _native.TMHD_ERR_INVALID
    assert q(ok, ok, ok + 2, 4, 64, 64, None) == _native.TMHD_ERR_INVALID
    assert q(None, ok, ok, 4, 64, 64, None) == _native.TMHD_ERR_INVALID
    assert q(None, None, None, 0, 64, 64, None) == _native.TMHD_OK
    d = lib.tmhd_mxfp4_dequant
    assert d(ok, ok, ok, 4, 48, None) == _native.TMHD_ERR_UNSUPPORTED
    assert d(ok, ok + 4, ok, 4, 64, None) == _native.TMHD_ERR_INVALID
    g = lib.tmhd_gemm_mxfp4
    args = dict(out=ok, a=ok, b=ok, sa=ok, sb=ok, bias=None, m=4, n=8, k=64, lda=32, ldb=32, ldo=8)
    for change in (dict(n=0), dict(m=-1), dict(lda=16), dict(ldb=40), dict(ldo=7), dict(a=ok + 8), dict(sb=ok + 4),
                   dict(out=None), dict(bias=ok + 1)):
        assert g(*{**args, **change}.values(), None) == _native.TMHD_ERR_INVALID, change
    assert g(*{**args, "k": 48}.values(), None) == _native.TMHD_ERR_UNSUPPORTED
    assert g(*{**args, "m": 0}.values(), None) == _native.TMHD_OK
