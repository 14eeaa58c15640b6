"""Attention over long 8-bit caches: no key lost and none counted twice.

The error is taken in the 2-norm of each row and head, against fp64 over the slots' own values.  A result is rounded to
bf16 (at most 2^-8 of it); each weight is too, independently of the others, so that their errors shrink with the keys as
the result itself does (at most 2^-8 of it in the 2-norm); both together stay below 2^-7, measured 0.0024.  Of n keys of
like weight, m lost or counted twice change the result by about (m / n)^(1/2) of it: one tile of 32 keys of 40,788 by
2.8%, 3.6 times the bound.  The first test shows that on the oracle."""

import numpy as np
import pytest

from oracle import bf16, lowbit

BOUND = 2.0 ** -7
LONG = [13596, 13597, 13595]  # 40,788 tokens: three blocks of the history, two of them ragged


def _kv(torch, tokens, heads, dim, seed):
    g = torch.Generator().manual_seed(seed)
    k = torch.randn(tokens, heads, dim, generator=g) + 0.5 * torch.randn(heads, dim, generator=g)
    return k.to(torch.bfloat16), torch.randn(tokens, heads, dim, generator=g).to(torch.bfloat16)


def _row_errors(got, want):
    """The largest of the rows' errors, relative to the row, in the 2-norm over the channels."""
    return float(((got - want).norm(dim=-1) / want.norm(dim=-1)).max())


@pytest.mark.parametrize("dim", [64, 128])
def test_a_lost_tile_is_seen(torch_mod, dim):
    torch, n = torch_mod, sum(LONG)
    q, (k, v) = _kv(torch, 3, 1, dim, 1)[0], _kv(torch, n, 1, dim, 2)
    q, k, v = (bf16.from_torch(t).astype(np.float64) for t in (q, k, v))
    want = torch.from_numpy(lowbit.attention(q, k, v, dim ** -0.5))
    for first in (0, 64, 13568, 20032, n - n % 32 - 32):
        keep = np.r_[0:first, first + 32 : n]
        twice = np.r_[0:n, first : first + 32]
        for rows in (keep, twice):
            got = torch.from_numpy(lowbit.attention(q, k[rows], v[rows], dim ** -0.5))
            err = (got - want).norm(dim=-1) / want.norm(dim=-1)
            assert float(err.min()) > 1.5 * BOUND, (first, err)


def _want(torch, q, views, scale):
    """fp64 attention on the GPU, a head at a time."""
    parts = [[t[s.row0 : s.row0 + s.tokens] for t in s.slot.token_major()] for s in views]
    k, v = (torch.cat([p[i] for p in parts]) for i in (0, 1))
    out = torch.empty(q.shape, dtype=torch.float64, device=q.device)
    for i in range(q.shape[1]):
        s = q[:, i].double() @ k[:, i].double().t().contiguous() * scale
        out[:, i] = torch.softmax(s, -1) @ v[:, i].double()
    return out


def _item_rows(heads, dim, *calls):
    from taomate_hd_amd import _native

    table = (_native.KV8Call * len(calls))()
    for c, (rows, sizes) in zip(table, calls):
        c.q, c.o, c.q_token_stride, c.q_head_stride, c.o_token_stride, c.o_head_stride = 4096, 4096, 128, 64, 128, 64
        c.lq, c.n_segments = rows, len(sizes)
        for i, n in enumerate(sizes):
            c.seg[i] = _native.KV8Segment(4096, 4096, 4096, 4096, -(-n // 64) * 64, 0, n, 0)
    return _native.load().tmhd_attn_kv8_item_rows(table, len(calls), heads, dim, 0)


def _views(torch, dev, sizes, heads, dim, fmt):
    from taomate_hd_amd import KVSlot8

    views = []
    for i, n in enumerate(sizes):
        slot = KVSlot8(torch, heads=heads, head_dim=dim, capacity=n, device=dev, fmt=fmt)
        slot.pack(*(t.to(dev) for t in _kv(torch, n, heads, dim, 10 + i)))
        views.append(slot.view())
    return views


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("rows,heads,dim,sizes,items", [
    (1, 14, 128, LONG, 32), (19, 5, 128, LONG, 32), (32, 14, 64, LONG, 32), (40, 2, 64, LONG, 32),
    (64, 14, 128, LONG, 128), (91, 40, 128, [3000, 4000, 4232], 128), (128, 14, 64, LONG, 128), (125, 12, 128, LONG, 128),
    (256, 14, 128, LONG, 256), (700, 3, 128, LONG, 256), (513, 14, 64, LONG, 256), (1, 1, 128, [20000], 32),
    (513, 3, 64, [17000, 20000], 256)])
def test_every_key_counts_once(torch_mod, dev, rows, heads, dim, sizes, items, fmt):
    from taomate_hd_amd import segment_attention

    torch = torch_mod
    assert _item_rows(heads, dim, (rows, sizes)) == items
    views = _views(torch, dev, sizes, heads, dim, fmt)
    q = _kv(torch, rows, heads, dim, 5)[0].to(dev)
    got = segment_attention(torch, q, views, scale=dim ** -0.5)
    assert _row_errors(got.double(), _want(torch, q, views, dim ** -0.5)) <= BOUND


@pytest.mark.gpu
@pytest.mark.parametrize("lengths,items", [((1, 3, 32), 32), ((5, 100, 64), 128), ((7, 300, 40), 256)])
def test_every_key_of_a_batch_counts_once(torch_mod, dev, lengths, items):
    """Calls of several lengths over parts of one cache, their items cut anywhere: views that start inside a slot."""
    from taomate_hd_amd import AttentionCall, segment_attention_batch
    from taomate_hd_amd.slots import SlotView

    torch, heads, dim = torch_mod, 14, 128
    a, b, c = (v.slot for v in _views(torch, dev, LONG, heads, dim, "e4m3"))
    plan = [[SlotView(a, 13000, 576), b.view()], [b.view(), c.view(), a.view()], [SlotView(c, 12001, 64)]]
    calls = [AttentionCall(_kv(torch, n, heads, dim, 7 + n)[0].to(dev), views) for n, views in zip(lengths, plan)]
    assert _item_rows(heads, dim, *((n, [v.tokens for v in views]) for n, views in zip(lengths, plan))) == items
    for call, got in zip(calls, segment_attention_batch(torch, calls, scale=dim ** -0.5)[0]):
        assert _row_errors(got.double(), _want(torch, call.query, call.segments, dim ** -0.5)) <= BOUND
