"""The K/V slots held in 8 bits: quantizing pack, exact readers, attention over them."""

import numpy as np
import pytest

from oracle import bf16, lowbit

pytestmark = pytest.mark.gpu

HALF_BF16 = 2.0 ** -8  # half a bf16 step, relative to the value
FORMATS = ("e4m3", "int8")


def _kv(torch, tokens, heads, dim, seed, dev, spread=0):
    g = torch.Generator().manual_seed(seed)
    k = torch.randn(tokens, heads, dim, generator=g) + 0.5 * torch.randn(heads, dim, generator=g)
    v = torch.randn(tokens, heads, dim, generator=g)
    if spread:
        f = torch.exp2(torch.randint(-spread, spread + 1, (tokens, heads, dim), generator=g).float())
        k, v = k * f, v * f.flip(0)
    return k.to(torch.bfloat16).to(dev), v.to(torch.bfloat16).to(dev)


def _f64(t):
    return bf16.from_torch(t.cpu()).astype(np.float64)


def _slot(torch, k, v, fmt, dev, capacity=None, **pack):
    from taomate_hd_amd import KVSlot8

    slot = KVSlot8(torch, heads=int(k.shape[1]), head_dim=int(k.shape[2]), capacity=capacity or int(k.shape[0]), device=dev,
                   fmt=fmt)
    for b in slot.buffers():
        b.fill_(0xA5)  # stale contents
    slot.pack(k, v, **pack)
    return slot


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("tokens,heads,dim", [(1, 1, 64), (63, 3, 128), (64, 2, 64), (65, 5, 128), (331, 14, 128), (1000, 8, 64)])
def test_pack_is_exact(torch_mod, dev, tokens, heads, dim, fmt):
    torch = torch_mod
    k, v = _kv(torch, tokens, heads, dim, tokens + dim, dev, spread=5)
    slot = _slot(torch, k, v, fmt, dev)
    got_k, got_v = slot.token_major()
    for src, got, scale in ((k, got_k, slot.k_scale), (v, got_v, slot.v_scale)):
        want, byte = lowbit.kv8_values(_f64(src), fmt)
        np.testing.assert_array_equal(scale.cpu().numpy().T[: len(byte)], byte)
        np.testing.assert_array_equal(_f64(got), want)
    assert slot.nbytes == slot.capacity * heads * (2 * dim) + 2 * heads * slot.capacity // 64


@pytest.mark.parametrize("fmt", FORMATS)
def test_pack_of_every_bf16_value(torch_mod, dev, fmt):
    """Every finite bf16 as the largest of its 64-token block, among random smaller ones."""
    torch, d = torch_mod, 64
    g = torch.Generator().manual_seed(6)
    bits = torch.arange(65536, dtype=torch.int32)
    bits = bits[(bits & 0x7FF0) != 0x7F80][::16]  # a block for every 16th, all of them as other values below
    bits = bits[(bits & 0x7F80) != 0x7F80]
    n = int(bits.numel())
    mag = (bits & 0x7FFF).unsqueeze(1)
    other = (mag - torch.randint(0, 1600, (n, 64 * d - 1), generator=g)).clamp_min(0)
    other = other | (torch.randint(0, 2, other.shape, generator=g) << 15)
    block = torch.cat([bits.unsqueeze(1), other], 1)
    x = torch.where(block >= 32768, block - 65536, block).to(torch.int16).view(torch.bfloat16)
    x = x.view(n * 64, 1, d).to(dev)
    slot = _slot(torch, x, x, fmt, dev)
    want, byte = lowbit.kv8_values(_f64(x), fmt)
    for got, scale in zip(slot.token_major(), (slot.k_scale, slot.v_scale)):
        np.testing.assert_array_equal(scale.cpu().numpy().T, byte)
        np.testing.assert_array_equal(_f64(got), want)


@pytest.mark.parametrize("fmt", FORMATS)
def test_pack_ranges_rows_and_stale_blocks(torch_mod, dev, fmt):
    """Ranges and a row list of strided K/V land where they are sent; other blocks stay; a block's tail is zero."""
    from taomate_hd_amd.slots import PackRows

    torch = torch_mod
    qkv = torch.cat(_kv(torch, 500, 4, 128, 1, dev) + _kv(torch, 500, 4, 128, 2, dev), 2)
    k, v = qkv[:, :, 128:256], qkv[:, :, 256:384]
    rows = torch.randperm(500, generator=torch.Generator().manual_seed(3))[:100].to(dev)
    slot = _slot(torch, k, v, fmt, dev, capacity=640, row0=7, count=70)
    slot.pack_ranges(k, v, [PackRows(rows=rows, dst=256), PackRows(row0=490, count=10, dst=448)])
    assert slot.tokens == 458
    slot.tokens = 640
    got = slot.token_major()
    for src, out, codes in zip((k, v), got, (slot.k, slot.vt)):
        for at, part in ((0, src[7:77]), (256, src[rows]), (448, src[490:])):
            want, _ = lowbit.kv8_values(_f64(part), fmt)
            np.testing.assert_array_equal(_f64(out[at : at + len(want)]), want)
            tail = out[at + len(want) : (at + len(want) + 63) // 64 * 64]
            assert bool((tail == 0).all())
        blocks = codes.view(4, 10, 64 * 128)
        assert bool((blocks[:, [2, 3, 6, 8, 9]] == 0xA5).all())


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dim", [64, 128])
def test_expand_equals_a_bf16_pack_of_the_values(torch_mod, dev, fmt, dim):
    from taomate_hd_amd.slots import KVSlot, SlotView, expand_views

    torch = torch_mod
    slots, views = [], []
    for i, n in enumerate((1, 64, 130, 333)):
        k, v = _kv(torch, n + 64, 3, dim, i, dev, spread=3)
        slots.append(_slot(torch, k, v, fmt, dev))
        views.append(SlotView(slots[-1], n, 64 if n > 1 else 0))
    views.append(views[2])  # the same rows again
    out = expand_views(torch, views)
    assert out[4].row0 == out[2].row0 and out[4].slot is out[2].slot
    for view, got in zip(views, out):
        k, v = (t[view.row0 : view.row0 + view.tokens] for t in view.slot.token_major())
        want = KVSlot(torch, heads=3, head_dim=dim, capacity=view.tokens, device=dev)
        want.pack(k.contiguous(), v.contiguous())
        at, cap = got.row0, want.capacity
        if view.row0 + cap <= view.slot.tokens:  # rows behind the view are the block's own here
            cap = view.tokens // 64 * 64
        assert torch.equal(got.slot.k[:, at : at + cap], want.k[:, :cap])
        assert torch.equal(got.slot.vt[:, :, at : at + cap], want.vt[:, :, :cap])


def test_expand_of_more_rows_than_a_slot_holds(torch_mod, dev, monkeypatch):
    """The views then lie in several bf16 slots, in the order given, the same view again in the same place."""
    from taomate_hd_amd import slots

    torch = torch_mod
    views = [_slot(torch, *_kv(torch, n, 2, 64, n, dev), "int8", dev).view() for n in (100, 64, 130, 1)]
    views += [views[1]]
    whole = slots.expand_views(torch, views)
    monkeypatch.setattr(slots, "MAX_SLOT_CAPACITY", 256)
    parts = slots.expand_views(torch, views)
    assert len({id(v.slot) for v in whole}) == 1 and len({id(v.slot) for v in parts}) == 2 and parts[4] == parts[1]
    for a, b in zip(whole, parts):
        assert a.tokens == b.tokens
        for x, y in zip(a.slot.token_major(), b.slot.token_major()):
            assert torch.equal(x[a.row0 : a.row0 + a.tokens], y[b.row0 : b.row0 + b.tokens])


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("rows,heads,dim,items", [(1, 4, 64, 32), (40, 4, 64, 32), (100, 1900, 64, 128), (200, 1100, 64, 256), (300, 400, 128, 256)])
def test_blocks_without_finite_values(torch_mod, dev, rows, heads, dim, items, fmt):
    """An infinity or NaN makes its block and head NaN, in every reader, and nothing else."""
    from taomate_hd_amd import segment_attention
    from taomate_hd_amd.slots import expand_views

    torch = torch_mod
    assert _item_rows(heads, dim, (rows, [200])) == items
    k, v = _kv(torch, 200, heads, dim, 1, dev)
    k[70, 1, 3], v[130, 2, 60] = float("inf"), float("nan")
    slot = _slot(torch, k, v, fmt, dev)
    nan = [torch.isnan(t) for t in slot.token_major()]
    assert int(nan[0].sum()) == 64 * dim == int(nan[0][64:128, 1].sum())
    assert int(nan[1].sum()) == 64 * dim == int(nan[1][128:192, 2].sum())
    big = expand_views(torch, [slot.view()])[0].slot
    assert int(torch.isnan(big.k).sum()) == 64 * dim == int(torch.isnan(big.vt).sum())
    q = _kv(torch, rows, heads, dim, 2, dev)[0]
    bad = torch.isnan(segment_attention(torch, q, [slot.view()], scale=0.125))
    assert bool(bad[:, 1:3].all()) and not bool(bad[:, 0].any()) and not bool(bad[:, 3:].any())


def _want(q, segments, scale):
    """fp64 attention over the slots' own values, and the bound of a bf16-weight kernel's error."""
    k = np.concatenate([_f64(s.slot.token_major()[0])[s.row0 : s.row0 + s.tokens] for s in segments])
    v = np.concatenate([_f64(s.slot.token_major()[1])[s.row0 : s.row0 + s.tokens] for s in segments])
    q = _f64(q)
    want = lowbit.attention(q, k, v, scale)
    size = lowbit.attention(q, k, np.abs(v), scale)  # sum of weight * |v|
    # scores: fp32 sums of D products, each add off by at most 2^-23 of the size; then a few roundings of
    # a number of the score's size and the hardware exponential (2^-22)
    reach = max(float((np.abs(q[:, i]) @ np.abs(k[:, i]).T).max()) for i in range(q.shape[1])) * abs(scale)
    weight = HALF_BF16 + 2 * (q.shape[2] + 8) * 2.0 ** -23 * reach + len(k) * 2.0 ** -23 + 2.0 ** -20
    # a weight below 2^-126 of the largest is not a normal fp32 number and may count as zero: at most 2^-126 of
    # each value's size (scores 969.0 and 801.9, the larger's value 0, give an output of 1.6e-74 in fp64, 0 in fp32)
    lost = 2.0 ** -126 * np.abs(v).sum(0)
    return want, HALF_BF16 * np.abs(want) + 1.02 * weight * size + lost


def _item_rows(heads, dim, *calls):
    """Rows of the items that calls of (rows, segment lengths) are cut into: which kernel they run."""
    from taomate_hd_amd import _native

    table = (_native.KV8Call * len(calls))()
    for c, (rows, sizes) in zip(table, calls):
        c.q, c.o, c.q_token_stride, c.q_head_stride, c.o_token_stride, c.o_head_stride = 4096, 4096, 128, 64, 128, 64
        c.lq, c.n_segments = rows, len(sizes)
        for i, n in enumerate(sizes):
            c.seg[i] = _native.KV8Segment(4096, 4096, 4096, 4096, -(-n // 64) * 64, 0, n, 0)
    return _native.load().tmhd_attn_kv8_item_rows(table, len(calls), heads, dim, 0)


# (rows, heads) whose calls over two blocks take each kernel: a head size of 64, and of 128
KERNELS = [(3, 2, 64, 32), (100, 3700, 64, 128), (200, 2200, 64, 256), (90, 2500, 128, 128), (300, 800, 128, 256)]
CASES = [(1, 1, 64, [1]), (1, 3, 128, [33]), (5, 2, 64, [64, 1, 130]), (32, 4, 128, [500]), (33, 2, 128, [65]),
         (64, 3, 64, [1000, 70]), (1, 14, 128, [9000, 777, 64]), (17, 1, 128, [20000]), (40, 1, 128, [30]),
         (100, 5, 128, [64, 700, 33]), (128, 2, 64, [2000]), (129, 3, 128, [1]), (300, 2, 64, [65, 128]),
         (256, 9, 128, [500, 640]), (700, 1, 128, [5000, 64]), (33, 7300, 64, [65]), (128, 2600, 128, [1, 64]),
         (97, 40, 128, [6000, 65, 200]), (129, 1000, 128, [65, 1]), (257, 12, 128, [9000, 130, 64, 63]),
         (513, 3, 64, [17000, 20000]), (33, 200, 64, [65, 100]), (3, 300, 128, [700])]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("rows,heads,dim,sizes", CASES)
def test_attention_over_codes(torch_mod, dev, rows, heads, dim, sizes, fmt):
    from taomate_hd_amd import segment_attention

    torch = torch_mod
    views = []
    for i, n in enumerate(sizes):
        k, v = _kv(torch, n, heads, dim, 10 * i + n, dev)
        views.append(_slot(torch, k, v * (4.0 ** i), fmt, dev).view())
    q = _kv(torch, rows, heads, dim, rows, dev)[0]
    got = segment_attention(torch, q, views, scale=dim ** -0.5)
    want, bound = _want(q, views, dim ** -0.5)
    err = np.abs(_f64(got) - want)
    assert (err <= bound).all(), float((err / bound).max())


@pytest.mark.parametrize("fmt", FORMATS)
def test_calls_on_both_sides_of_the_in_place_rule(torch_mod, dev, fmt):
    """One row more and the slot is expanded: the call is one over a bf16 slot, bit for bit."""
    from taomate_hd_amd import KVSlot, attention, segment_attention

    torch = torch_mod
    heads, dim, tokens, most = 6, 128, 4264, attention.KV8_ROWS
    assert (most + 1) * tokens * heads * dim > attention.KV8_WORK
    k, v = _kv(torch, tokens, heads, dim, 8, dev)
    slot = _slot(torch, k, v, fmt, dev)
    plain = KVSlot(torch, heads=heads, head_dim=dim, capacity=tokens, device=dev)
    plain.pack(*slot.token_major())
    q = _kv(torch, most + 1, heads, dim, 9, dev)[0]
    in_place = segment_attention(torch, q[:most], [slot.view()], scale=dim ** -0.5)
    want, bound = _want(q[:most], [slot.view()], dim ** -0.5)
    assert (np.abs(_f64(in_place) - want) <= bound).all()
    expanded = segment_attention(torch, q, [slot.view()], scale=dim ** -0.5)
    assert torch.equal(expanded, segment_attention(torch, q, [plain.view()], scale=dim ** -0.5))
    assert not torch.equal(expanded[:most], in_place)


@pytest.mark.parametrize("fmt", FORMATS)
def test_expanded_calls_equal_calls_over_bf16_slots(torch_mod, dev, fmt):
    """With bf16 segments beside the 8-bit ones, and with the INT8-QK backend, a call gives the bits of the same call
    over a bf16 slot packed with the 8-bit slot's values."""
    from taomate_hd_amd import segment_attention
    from taomate_hd_amd.slots import KVSlot

    torch = torch_mod
    k, v = _kv(torch, 700, 4, 128, 1, dev)
    slot = _slot(torch, k, v, fmt, dev)
    plain = KVSlot(torch, heads=4, head_dim=128, capacity=700, device=dev)
    plain.pack(*slot.token_major())
    beside = KVSlot(torch, heads=4, head_dim=128, capacity=90, device=dev)
    beside.pack(*_kv(torch, 90, 4, 128, 3, dev))
    q = _kv(torch, 300, 4, 128, 2, dev)[0]
    for backend, rows, more in (("bf16", 300, [beside.view()]), ("bf16", 2, [beside.view()]), ("i8qk", 300, []), ("i8qk", 3, [])):
        a = segment_attention(torch, q[:rows], [slot.view(), *more], scale=0.1, backend=backend)
        b = segment_attention(torch, q[:rows], [plain.view(), *more], scale=0.1, backend=backend)
        assert torch.equal(a, b)


@pytest.mark.parametrize("fmt", FORMATS)
def test_batch_of_unlike_calls(torch_mod, dev, fmt):
    """Calls of few and many rows, over 8-bit, bf16 and mixed segments, views inside a slot, row lists, strided
    queries and outputs: each as alone, and rows that belong to no call stay."""
    from taomate_hd_amd import AttentionCall, KVSlot, segment_attention_batch
    from taomate_hd_amd.slots import SlotView

    torch, heads, dim = torch_mod, 3, 64
    other = "int8" if fmt == "e4m3" else "e4m3"
    a = _slot(torch, *_kv(torch, 400, heads, dim, 1, dev), fmt, dev)
    b = _slot(torch, *_kv(torch, 90, heads, dim, 2, dev), other, dev)
    c = KVSlot(torch, heads=heads, head_dim=dim, capacity=100, device=dev)
    ck, cv = _kv(torch, 100, heads, dim, 3, dev)
    c.pack(ck, cv)
    q = _kv(torch, 400, 3 * heads, dim, 4, dev)[0][:, heads : 2 * heads]
    out = torch.full((400, 2 * heads, dim), 7.0, dtype=torch.bfloat16, device=dev)
    o = out[:, heads:]
    rows = torch.tensor([390, 5, 17, 399], device=dev)
    plan = [
        (AttentionCall(q, [SlotView(a, 130, 64), SlotView(a, 8, 320)], q_row0=20, lq=9, out=o, o_row0=20), range(20, 29)),
        (AttentionCall(q, [b.view()], q_rows=rows, out=o, o_rows=rows), rows.tolist()),
        (AttentionCall(q, [a.view(), c.view()], q_row0=100, lq=2, out=o, o_row0=100), range(100, 102)),
        (AttentionCall(q, [a.view(), b.view()], q_row0=110, lq=70, out=o, o_row0=110), range(110, 180)),
        (AttentionCall(q, [a.view()], q_row0=200, lq=0, out=o, o_row0=200), ()),
        (AttentionCall(q, [c.view()], q_row0=300, lq=5, out=o, o_row0=300), range(300, 305)),
    ]
    segment_attention_batch(torch, [call for call, _ in plan], scale=0.125)
    torch.cuda.synchronize()
    values = {}
    for slot in (a, b):
        values[id(slot)] = slot.token_major()
    values[id(c)] = (ck, cv)

    class _Held:
        def __init__(self, slot):
            self.token_major = lambda: values[id(slot)]

    touched = torch.zeros(400, dtype=torch.bool)
    for call, where in plan:
        where = list(where)
        touched[where] = True
        if where:
            want, bound = _want(q[where], [SlotView(_Held(s.slot), s.tokens, s.row0) for s in call.segments], 0.125)
            assert (np.abs(_f64(o[where]) - want) <= bound).all()
    assert bool((out[:, :heads] == 7.0).all()) and bool((o[~touched.to(dev)] == 7.0).all())


@pytest.mark.parametrize("rows", [2, 300])
def test_more_segments_than_one_launch(torch_mod, dev, rows):
    """Then they are expanded and the oldest copied together: the call over bf16 slots of the same values."""
    from taomate_hd_amd import KVSlot, segment_attention

    torch, heads, dim = torch_mod, 2, 64
    views, plain = [], []
    for i in range(21):
        slot = _slot(torch, *_kv(torch, 20 + 13 * i, heads, dim, i, dev), FORMATS[i % 2], dev)
        views.append(slot.view())
        plain.append(KVSlot(torch, heads=heads, head_dim=dim, capacity=slot.capacity, device=dev))
        plain[-1].pack(*slot.token_major())
    q = _kv(torch, rows, heads, dim, 99, dev)[0]
    got = segment_attention(torch, q, views, scale=0.125)
    assert torch.equal(got, segment_attention(torch, q, [p.view() for p in plain], scale=0.125))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("heads,lengths,items", [(3, (100, 60, 5), 32), (830, (100, 60, 5), 128), (520, (200, 140, 5), 256)])
def test_batch_in_each_kernel(torch_mod, dev, heads, lengths, items, fmt):
    """Rows by range and by list (one of them twice in the queries), views inside a slot, strided queries and outputs,
    a call without rows: rows that belong to no call stay."""
    from taomate_hd_amd import AttentionCall, segment_attention_batch
    from taomate_hd_amd.slots import SlotView

    torch, dim = torch_mod, 64
    sizes = ([130, 60], [150], [300, 150, 300])
    assert _item_rows(heads, dim, *zip(lengths, sizes)) == items
    a = _slot(torch, *_kv(torch, 300, heads, dim, 1, dev), fmt, dev)
    b = _slot(torch, *_kv(torch, 150, heads, dim, 2, dev), fmt, dev)
    q = _kv(torch, 420, 2 * heads, dim, 4, dev)[0][:, heads:]
    out = torch.full((420, heads, dim), 7.0, dtype=torch.bfloat16, device=dev)
    order = torch.randperm(100, generator=torch.Generator().manual_seed(1)) + 10
    take = torch.cat([order, order])[: lengths[1]].to(dev)
    put = (torch.randperm(lengths[1], generator=torch.Generator().manual_seed(2)) + 215).to(dev)
    n = lengths[0]
    plan = [
        (AttentionCall(q, [SlotView(a, 130, 64), SlotView(a, 60, 192)], q_row0=1, lq=n, out=out, o_row0=2), q[1 : n + 1],
         range(2, n + 2)),
        (AttentionCall(q, [b.view()], q_rows=take, out=out, o_rows=put), q[take], put.tolist()),
        (AttentionCall(q, [b.view()], lq=0, out=out), q[:0], ()),
        (AttentionCall(q, [a.view(), b.view(), a.view()], q_row0=415, lq=5, out=out, o_row0=400), q[415:], range(400, 405)),
    ]
    segment_attention_batch(torch, [call for call, *_ in plan], scale=0.125)
    touched = torch.zeros(420, dtype=torch.bool)
    for call, rows, where in plan:
        where = list(where)
        touched[where] = True
        if where:
            want, bound = _want(rows, call.segments, 0.125)
            assert (np.abs(_f64(out[where]) - want) <= bound).all()
    assert bool((out[~touched.to(dev)] == 7.0).all())


def test_more_calls_than_one_launch(torch_mod, dev):
    from taomate_hd_amd import AttentionCall, segment_attention, segment_attention_batch

    torch = torch_mod
    calls = []
    for i in range(19):
        views = [_slot(torch, *_kv(torch, 40 + 70 * i + j, 2, 64, i + j, dev), "e4m3", dev).view() for j in range(1 + i % 3)]
        calls.append(AttentionCall(_kv(torch, 1 + i, 2, 64, 100 + i, dev)[0], views))
    outs, _ = segment_attention_batch(torch, calls, scale=0.125)
    for call, out in zip(calls, outs):
        want, bound = _want(call.query, call.segments, 0.125)
        assert (np.abs(_f64(out) - want) <= bound).all()
        again = segment_attention(torch, call.query, call.segments, scale=0.125)
        assert (np.abs(_f64(again) - want) <= bound).all()


@pytest.mark.parametrize("rows,heads,dim,items", [(20, 2, 128, 32), (90, 210, 128, 128), (300, 64, 128, 256), (150, 256, 64, 256)])
def test_large_scores_move_the_running_maximum(torch_mod, dev, rows, heads, dim, items):
    from taomate_hd_amd import segment_attention

    torch = torch_mod
    assert _item_rows(heads, dim, (rows, [1500])) == items
    k, v = _kv(torch, 1500, heads, dim, 1, dev)
    k = k * torch.linspace(0.1, 6.0, 1500, device=dev).view(-1, 1, 1).to(torch.bfloat16)
    slot = _slot(torch, k, v, "int8", dev)
    q = 8 * _kv(torch, rows, heads, dim, 2, dev)[0]
    got = segment_attention(torch, q, [slot.view()], scale=dim ** -0.5)
    want, bound = _want(q, [slot.view()], dim ** -0.5)
    assert (np.abs(_f64(got) - want) <= bound).all()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("rows,heads,dim,items", KERNELS)
def test_values_behind_a_view_that_overflow(torch_mod, dev, rows, heads, dim, items, fmt):
    """Rows of the view's last block that it does not hold: their scores are infinite, their weights nothing."""
    from taomate_hd_amd import segment_attention
    from taomate_hd_amd.slots import SlotView

    torch = torch_mod
    assert _item_rows(heads, dim, (rows, [70])) == items
    k, v = _kv(torch, 192, heads, dim, 1, dev)
    k[70:], v[70:] = 2.0 ** 100, 2.0 ** 100
    slot = _slot(torch, k, v, fmt, dev)
    q = 2.0 ** 40 * _kv(torch, rows, heads, dim, 2, dev)[0].abs()
    for view in (SlotView(slot, 70, 0), SlotView(slot, 6, 64)):  # (of two blocks, and of one)
        got = segment_attention(torch, q, [view], scale=2.0 ** -43)
        want, bound = _want(q, [view], 2.0 ** -43)
        assert (np.abs(_f64(got) - want) <= bound).all()


@pytest.mark.parametrize("rows,heads,dim,items", KERNELS)
@pytest.mark.parametrize("scale", [0.0, -0.3, 1e-30, 40.0])
def test_any_softmax_scale(torch_mod, dev, scale, rows, heads, dim, items):
    """No scale (the mean of the values), a negative, a vanishing and a large one, with a ragged last tile."""
    from taomate_hd_amd import segment_attention

    torch = torch_mod
    assert _item_rows(heads, dim, (rows, [71])) == items
    slot = _slot(torch, *_kv(torch, 71, heads, dim, 1, dev), "int8", dev)
    q = _kv(torch, rows, heads, dim, 2, dev)[0]
    got = segment_attention(torch, q, [slot.view()], scale=scale)
    want, bound = _want(q, [slot.view()], scale)
    assert (np.abs(_f64(got) - want) <= bound).all()


@pytest.mark.parametrize("rows,heads,dim,items", KERNELS)
def test_first_scores_below_every_number(torch_mod, dev, rows, heads, dim, items):
    """Scores of a call's first block that overflow to -inf weigh nothing, and leave what follows alone."""
    from taomate_hd_amd import segment_attention
    from taomate_hd_amd.slots import SlotView

    torch = torch_mod
    assert _item_rows(heads, dim, (rows, [71])) == items
    k, v = _kv(torch, 71, heads, dim, 1, dev)
    k[:64] = -(2.0 ** 100)
    slot = _slot(torch, k, v, "int8", dev)
    q = 2.0 ** 40 * (1 + _kv(torch, rows, heads, dim, 2, dev)[0].abs())
    got = segment_attention(torch, q, [slot.view()], scale=2.0 ** -43)
    want, bound = _want(q, [SlotView(slot, 7, 64)], 2.0 ** -43)
    assert (np.abs(_f64(got) - want) <= bound).all()


@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("rows,heads,dim,items", KERNELS)
def test_scores_beyond_every_fraction(torch_mod, dev, rows, heads, dim, items, sign):
    """Equal scores of 2^44 and more, all of an fp32's bits above the point: the mean of the values, then one larger
    score that outweighs them all."""
    from taomate_hd_amd import segment_attention
    from taomate_hd_amd.slots import SlotView

    torch = torch_mod
    assert _item_rows(heads, dim, (rows, [71])) == items
    k, v = _kv(torch, 71, heads, dim, 1, dev)
    k[:] = sign * 2.0 ** 20
    k[70] = 2.0 ** 21
    slot = _slot(torch, k, v, "int8", dev)
    q = 2.0 ** 24 * (1 + _kv(torch, rows, heads, dim, 2, dev)[0].abs())
    values = _f64(slot.token_major()[1])
    for view, want in ((SlotView(slot, 70, 0), values[:70].mean(0)), (SlotView(slot, 6, 64), values[64:70].mean(0)),
                       (slot.view(), values[70])):
        got = _f64(segment_attention(torch, q, [view], scale=0.9))
        size = np.abs(values).max(0)
        assert (np.abs(got - want) <= HALF_BF16 * np.abs(want) + 1.02 * (HALF_BF16 + 2.0 ** -20) * size).all()


@pytest.mark.parametrize("rows,heads,dim,items", KERNELS)
def test_scale_that_is_no_number(torch_mod, dev, rows, heads, dim, items):
    from taomate_hd_amd import segment_attention

    torch = torch_mod
    assert _item_rows(heads, dim, (rows, [71])) == items
    slot = _slot(torch, *_kv(torch, 71, heads, dim, 1, dev), "e4m3", dev)
    q = _kv(torch, rows, heads, dim, 2, dev)[0]
    assert bool(torch.isnan(segment_attention(torch, q, [slot.view()], scale=float("nan"))).all())


def test_refusals(torch_mod, dev):
    from taomate_hd_amd import KVSlot8, fused_qkv_qk_norm_rope_stage_, segment_attention

    torch = torch_mod
    slot = _slot(torch, *_kv(torch, 100, 2, 64, 1, dev), "e4m3", dev)
    q = _kv(torch, 3, 2, 64, 2, dev)[0]
    with pytest.raises(ValueError, match="at least one key"):
        segment_attention(torch, q, [], scale=1.0)
    with pytest.raises(ValueError, match="differ from the query"):
        segment_attention(torch, q[:, :1], [slot.view()], scale=1.0)
    with pytest.raises(ValueError, match="outside query"):
        segment_attention(torch, q, [slot.view()], scale=1.0, q_row0=1, lq=3)
    with pytest.raises(ValueError, match="entries must lie"):
        segment_attention(torch, q, [slot.view()], scale=1.0, q_rows=torch.tensor([3], device=dev))
    with pytest.raises(ValueError, match="differ from slot"):
        slot.pack(*_kv(torch, 10, 3, 64, 1, dev))
    with pytest.raises(ValueError, match="fit the slot"):
        slot.pack(*_kv(torch, 10, 2, 64, 1, dev), dst=32)
    with pytest.raises(ValueError, match="bfloat16|bf16"):
        slot.pack(*(t.float() for t in _kv(torch, 10, 2, 64, 1, dev)))
    with pytest.raises(ValueError, match="8-bit K/V format"):
        KVSlot8(torch, heads=1, head_dim=64, capacity=64, device=dev, fmt="e5m2")
    with pytest.raises(ValueError, match="bf16 slots"):
        fused_qkv_qk_norm_rope_stage_(q, None, None, None, None, 1e-6, slot)
    with pytest.raises(ValueError, match="no bf16 segment"):
        slot.view().to_segment()


@pytest.mark.parametrize("rows,heads,items", [(2, 4, 32), (100, 48, 128), (400, 48, 256)])
def test_streams_and_graph(torch_mod, dev, rows, heads, items):
    """A pack and a decode call on another stream, and captured and replayed with new K/V between eager calls."""
    from taomate_hd_amd import KVSlot8, segment_attention

    torch = torch_mod
    assert _item_rows(heads, 128, (rows, [5000])) == items
    slot = KVSlot8(torch, heads=heads, head_dim=128, capacity=5000, device=dev)
    k, v = _kv(torch, 5000, heads, 128, 1, dev)
    q = _kv(torch, rows, heads, 128, 2, dev)[0]

    def step():
        slot.pack(k, v)
        return segment_attention(torch, q, [slot.view()], scale=0.1)

    want = step().clone()
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        other = step()
    stream.synchronize()
    assert torch.equal(other, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (5, 6, 7):
        nk, nv = _kv(torch, 5000, heads, 128, seed, dev)
        k.copy_(nk), v.copy_(nv)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, step())


def test_two_streams_at_once(torch_mod, dev):
    """Calls over one slot, queued on two streams side by side: their parts do not meet."""
    from taomate_hd_amd import segment_attention

    torch = torch_mod
    slot = _slot(torch, *_kv(torch, 9000, 8, 128, 1, dev), "e4m3", dev)
    queries = [_kv(torch, rows, 8, 128, rows, dev)[0] for rows in (1, 700, 100, 5)]
    want = [segment_attention(torch, q, [slot.view()], scale=0.1) for q in queries]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for _ in range(10):
        for i, q in enumerate(queries):
            with torch.cuda.stream(streams[i % 2]):
                got.append((i, segment_attention(torch, q, [slot.view()], scale=0.1)))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i]) for i, y in got)


@pytest.mark.parametrize("fmt", FORMATS)
def test_end_of_the_longest_slot(torch_mod, dev, fmt):
    """The last rows of a slot of all the tokens one can hold: codes, scales and values beyond 32-bit offsets."""
    from taomate_hd_amd import KVSlot8, segment_attention
    from taomate_hd_amd.slots import MAX_SLOT_CAPACITY, SlotView, expand_views

    torch, heads, dim, n = torch_mod, 5, 128, 46010
    assert MAX_SLOT_CAPACITY * heads * dim > 1 << 32
    slot = KVSlot8(torch, heads=heads, head_dim=dim, capacity=MAX_SLOT_CAPACITY, device=dev, fmt=fmt)
    k, v = _kv(torch, n, heads, dim, 3, dev)
    at = MAX_SLOT_CAPACITY - 46016
    slot.pack(k, v, dst=at)
    near = _slot(torch, k, v, fmt, dev)
    view = SlotView(slot, n, at)
    for a, b in zip(expand_views(torch, [view])[0].slot.token_major(n), near.token_major()):
        assert torch.equal(a, b)
    for rows, items in ((2, 32), (128, 128), (300, 256)):
        assert _item_rows(heads, dim, (rows, [n])) == items
        q = _kv(torch, rows, heads, dim, 4, dev)[0]
        got = segment_attention(torch, q, [view], scale=0.1)
        assert torch.equal(got, segment_attention(torch, q, [near.view()], scale=0.1))


@pytest.mark.parametrize("backend", ["sdpa", "sage_attn"])
@pytest.mark.parametrize("storage", FORMATS)
def test_hook_over_an_8bit_cache(torch_mod, dev, storage, backend):
    """Commits and noisy steps through the hook: outputs near those over a bf16 cache, equal to attention over the
    values the cache gives back, history read back as packed, and half the memory."""
    from taomate_hd_amd import HeadMajorRingKVCache, HookMode, KVContract, KVSlot, StreamingAttentionHook, segment_attention

    torch, heads, dim, layer = torch_mod, 4, 64, "blocks.0.attn"
    contract = KVContract(layer_names=(layer,), local_heads=heads, head_dim=dim)

    class Attn:
        softmax_scale = dim ** -0.5

    def call(hook, n, seed, mode, block):
        q, k = _kv(torch, n, heads, dim, seed, dev)
        v = _kv(torch, n, heads, dim, seed + 1, dev)[1]
        tags = torch.zeros(n, dtype=torch.int64, device=dev)
        tags[::7] = 2
        hook.activate(mode=mode, block_index=block)
        out = hook(attention=Attn(), layer_name=layer, query=q, key=k, value=v, token_tags=tags,
                   commit_mask=torch.ones(n, dtype=torch.bool, device=dev), cu_seqlens=None, cu_seqlens_host=(0, n),
                   max_seqlen=n)
        hook.deactivate()
        return out, q, k, v

    caches = {s: HeadMajorRingKVCache(contract, storage=s) for s in ("bf16", storage)}
    last = {}
    for s, cache in caches.items():
        hook = StreamingAttentionHook(cache, attention_backend=backend)
        for block, n in enumerate((210, 130)):
            cache.begin_clean_commit(block)
            call(hook, n, 10 * block, HookMode.CLEAN_COMMIT, block)
            cache.commit()
        last[s] = call(hook, 300, 50, HookMode.NOISY, 2)
    cache = caches[storage]
    assert 0.5 <= cache.slot_bytes / caches["bf16"].slot_bytes < 0.52
    hist = cache.history(layer)
    views = []
    for k, v in ((hist.key, hist.value), last[storage][2:]):
        views.append(KVSlot(torch, heads=heads, head_dim=dim, capacity=len(k), device=dev))
        views[-1].pack(k.contiguous(), v.contiguous())
    want = segment_attention(torch, last[storage][1], [s.view() for s in views], scale=dim ** -0.5)
    got, plain = _f64(last[storage][0]), _f64(last["bf16"][0])
    # against attention over the cache's own values: both backends within their rounding of it
    tol = 2e-2 if backend == "sdpa" else 6e-2
    assert np.abs(got - _f64(want)).max() <= tol
    cos = (got * plain).sum() / np.sqrt((got ** 2).sum() * (plain ** 2).sum())
    assert cos >= 0.99, cos
