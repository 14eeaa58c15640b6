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
    # more rows than an index or a launch holds
    most = 2 ** 31 - 1
    assert q(ok, ok, ok, most - 255, 32, 32, None) == _native.TMHD_ERR_INVALID
    assert q(ok, ok, ok, most - 256, 32, 32, None) == _native.TMHD_ERR_UNSUPPORTED
    assert d(ok, ok, ok, most - 256, 32, None) == _native.TMHD_ERR_UNSUPPORTED
    wide = dict(k=32, lda=16, ldb=16, n=most - 256, ldo=most)
    assert g(*{**args, **wide, "n": most - 255}.values(), None) == _native.TMHD_ERR_INVALID
    assert g(*{**args, **wide, "m": 4096}.values(), None) == _native.TMHD_ERR_UNSUPPORTED


def _view(**change):
    from taomate_hd_amd import _native

    base = dict(k=4096, v=4096, ks=4096, vs=4096, cap=128, row0=0, tokens=100, format=0)
    return _native.KV8Segment(**{**base, **change})


def test_kv8_c_entries_refuse():
    from taomate_hd_amd import _native

    lib, ok, inv, uns = _native.load(), 4096, _native.TMHD_ERR_INVALID, _native.TMHD_ERR_UNSUPPORTED
    ranges = (_native.PackRange * 2)(_native.PackRange(None, 0, 70, 0, 0), _native.PackRange(None, 0, 10, 64, 0))

    def pack(n=1, slot=None, k=ok, ts=64, hs=64, heads=2, dim=64):
        return lib.tmhd_kv8_pack_ranges(k, ok, ts, hs, ranges, n, slot or _view(), heads, dim, None)

    assert pack(n=2) == inv and "share a 64-row block" in lib.tmhd_last_error().decode()
    assert pack(heads=0) == inv and pack(dim=96) == uns and pack(n=-1) == inv
    assert pack(ts=60) == inv and pack(k=ok + 2) == inv and pack(slot=_view(cap=100)) == inv
    assert pack(slot=_view(cap=64)) == inv and pack(slot=_view(format=2)) == uns and pack(slot=_view(ks=None)) == inv
    assert pack(n=0) == _native.TMHD_OK

    def expand(view, dst=0, row=128, head=128 * 64, n=1):
        return lib.tmhd_kv8_expand(view, (_native.c_int32 * 1)(dst), n, ok, ok, head, head, row, 2, 64, None)

    assert expand(_view(tokens=0)) == inv and expand(_view(row0=32)) == inv and expand(_view(row0=64, tokens=65)) == inv
    assert expand(_view(), dst=64) == inv and expand(_view(), dst=1) == inv and expand(_view(), head=64 * 64) == inv
    assert expand(_view(), n=0) == _native.TMHD_OK
    assert lib.tmhd_kv8_token_major(_view(tokens=129), ok, ok, 2, 64, None) == inv
    assert lib.tmhd_kv8_token_major(_view(), ok + 8, ok, 2, 64, None) == inv


def test_kv8_attention_c_entry_refuses():
    from taomate_hd_amd import _native

    lib, ok, inv = _native.load(), 4096, _native.TMHD_ERR_INVALID

    def attend(view=None, n_segments=1, heads=2, dim=64, ws=None, ws_bytes=0, second=None, **change):
        base = dict(q=ok, q_token_stride=128, q_head_stride=64, lq=1, o=ok, o_token_stride=128, o_head_stride=64)
        c = _native.KV8Call(**{**base, **change}, n_segments=n_segments)
        for i, s in enumerate([view or _view(), second or _view()]):
            c.seg[i] = s
        calls = (_native.KV8Call * 1)(c)
        return lib.tmhd_attn_fwd_kv8(calls, 1, heads, dim, 1.0, ws, ws_bytes, None)

    assert attend(n_segments=0) == inv and attend(n_segments=17) == inv and attend(lq=-1) == inv
    assert attend(view=_view(tokens=0)) == inv and attend(q=ok + 8) == inv and attend(q_head_stride=60) == inv
    assert attend(o_token_stride=126) == inv and attend(o=ok + 2) == inv and attend(q_row0=-1) == inv
    assert attend(n_segments=2, second=_view(format=1)) == _native.TMHD_ERR_UNSUPPORTED
    assert attend(dim=256) == _native.TMHD_ERR_UNSUPPORTED and attend(ws=ok + 4, ws_bytes=64) == inv
    # a long cache is dealt to key ranges: no workspace, no call
    assert attend(view=_view(cap=1 << 20, tokens=1 << 20), heads=1) == inv and "workspace" in lib.tmhd_last_error().decode()
    # more rows than the merge's launch holds, and more (row tile, block) pairs than an index does
    uns = _native.TMHD_ERR_UNSUPPORTED
    assert attend(lq=1 << 22, heads=64, view=_view(tokens=64)) == uns and "too many" in lib.tmhd_last_error().decode()
    assert attend(lq=1 << 20, heads=32767, view=_view(cap=1 << 22, tokens=1 << 22)) == uns
    assert attend(lq=0) == _native.TMHD_OK


def test_slots_refuse_on_the_host():
    import torch

    import taomate_hd_amd as tm

    with pytest.raises(ValueError, match="K/V storage"):
        tm.HeadMajorRingKVCache(storage="fp8")
    with pytest.raises(ValueError, match="K/V storage"):
        tm.SlotPool(torch, heads=1, head_dim=64, device="cpu", storage="e5m2")
    with pytest.raises(ValueError, match="head_dim"):
        tm.KVSlot8(torch, heads=1, head_dim=96, capacity=64, device="cpu")
    with pytest.raises(ValueError, match="storage differ"):
        tm.StreamingSession(type("P", (), {"phases": ()})(), cache=tm.HeadMajorRingKVCache(storage="int8"), kv_storage="e4m3")
    slot = tm.KVSlot8(torch, heads=1, head_dim=64, capacity=65, device="cpu", fmt="int8")
    assert slot.capacity == 128 and slot.nbytes == 2 * 128 * 64 + 4
    k = torch.zeros(10, 1, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="GPU tensor"):
        slot.pack(k, k)


def test_mxfp4_linear_c_entry_refuses():
    from taomate_hd_amd import _native

    lib, ok, inv = _native.load(), 4096, _native.TMHD_ERR_INVALID
    need = lib.tmhd_linear_mxfp4_workspace_bytes(100, 8, 64)
    assert need == (100 * 32 + 255) // 256 * 256 + 16 * 100 and lib.tmhd_linear_mxfp4_workspace_bytes(1, 8, 64) == 0
    args = dict(out=ok, x=ok, b=ok, sb=ok, bias=None, m=100, n=8, k=64, ldx=64, ldb=32, ldo=8, ws=ok, bytes=need)
    for change in (dict(x=ok + 8), dict(ldx=60), dict(ldx=56), dict(ws=None), dict(bytes=need - 1), dict(ws=ok + 8),
                   dict(n=0), dict(ldb=16)):
        assert lib.tmhd_linear_mxfp4(*{**args, **change}.values(), None) == inv, change
    assert lib.tmhd_linear_mxfp4(*{**args, "k": 48}.values(), None) == _native.TMHD_ERR_UNSUPPORTED
    assert lib.tmhd_linear_mxfp4(*{**args, "m": 0}.values(), None) == _native.TMHD_OK


def _form(m, n, k):
    from taomate_hd_amd import _native

    return _native.load().tmhd_gemm_mxfp4_form(m, n, k, 256)


def test_mxfp4_forms():
    """The rule's choices at sizes whose forms were all timed, and for what no product has."""
    from taomate_hd_amd import _native as n

    assert _form(1, 5376, 5376) == n.MXFP4_ROWS and _form(16, 640, 2048) == n.MXFP4_ROWS
    assert _form(1, 13824, 5120) == n.MXFP4_64X64 and _form(17, 640, 2048) == n.MXFP4_64X64
    assert _form(100, 13824, 5120) == n.MXFP4_128X64 and _form(331, 5376, 5376) == n.MXFP4_128X64
    assert _form(331, 10752, 5376) == n.MXFP4_128X128 and _form(512, 5376, 5376) == n.MXFP4_128X128
    assert _form(331, 13824, 5120) == n.MXFP4_128X128X2 and _form(1500, 13824, 5120) == n.MXFP4_128X128X2
    assert _form(12252, 5376, 5376) == n.MXFP4_256X256 and _form(2048, 13824, 5120) == n.MXFP4_256X256
    assert _form(12252, 13824, 5120) in (n.MXFP4_128X64, n.MXFP4_128X128)  # behind ten rounds of 256 x 256
    for bad in ((0, 16, 32), (1, 0, 32), (1, 16, 0), (1, 16, 48)):
        assert _form(*bad) == -1


def test_kv8_item_rows():
    """The rule's choices at sizes whose forms were all timed (256 CUs), and for calls that are refused."""
    from taomate_hd_amd import _native

    def rows(lq, heads, tokens, dim=128, calls=1, **change):
        cap = -(-tokens // 64) * 64
        c = _native.KV8Call(q=4096, q_token_stride=128, q_head_stride=64, lq=lq, o=4096, o_token_stride=128,
                            o_head_stride=64, n_segments=1)
        c.seg[0] = _view(cap=cap, tokens=tokens, **change)
        return _native.load().tmhd_attn_kv8_item_rows((_native.KV8Call * calls)(*[c] * calls), calls, heads, dim, 256)

    assert rows(1, 14, 40788) == rows(32, 40, 100000) == 32
    assert rows(256, 14, 2800) == rows(400, 40, 1500) == rows(128, 14, 12000) == 32
    assert rows(91, 40, 12000) == rows(128, 14, 41000) == 128
    assert rows(256, 40, 6000) == rows(1024, 14, 41000) == 256
    assert rows(300, 14, 11000, dim=64) == 32 and rows(300, 14, 41000, dim=64) == 256
    assert rows(100, 14, 2800, calls=12) == 128  # (together as large as one long call)
    assert rows(0, 14, 2800) == 32 and rows(-1, 14, 2800) == -1 and rows(1, 14, 2800, dim=96) == -1
    assert rows(1, 0, 2800) == -1 and rows(1, 14, 2800, row0=32) == -1


def test_kv8_workspace():
    """Short items of 32 rows are not cut, longer ones are."""
    from taomate_hd_amd import _native

    def need(lq, tokens, heads=14):
        c = _native.KV8Call(q=4096, q_token_stride=128, q_head_stride=64, lq=lq, o=4096, o_token_stride=128,
                            o_head_stride=64, n_segments=1)
        c.seg[0] = _view(cap=1 << 16, tokens=tokens)
        return _native.load().tmhd_attn_kv8_workspace_bytes((_native.KV8Call * 1)(c), 1, heads, 128)

    assert need(1, 1) == need(32, 48 * 64) == need(0, 60000) == need(-1, 64) == 0
    assert need(1, 48 * 64 + 1) > 0 and need(40, 60000) > 0
