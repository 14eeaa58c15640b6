"""Attention of many query rows over 8-bit slots is as exact as that of few: the scaled Q is not rounded to bf16."""

import numpy as np
import pytest

from oracle import bf16, lowbit

pytestmark = pytest.mark.gpu

HALF_BF16 = 2.0 ** -8
FORMATS = ("e4m3", "int8")


def _f64(t):
    return bf16.from_torch(t.cpu()).astype(np.float64)


def _randn(torch, dev, *shape, seed):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16).to(dev)


def _slot(torch, k, v, fmt, dev):
    from taomate_hd_amd import KVSlot8

    slot = KVSlot8(torch, heads=int(k.shape[1]), head_dim=int(k.shape[2]), capacity=int(k.shape[0]), device=dev, fmt=fmt)
    slot.pack(k, v)
    return slot


def _want(q, slot, scale, tokens=None, row0=0):
    """fp64 attention over the slot's values, and how far a kernel with exact Q, fp32 scores and bf16 weights may be off.

    Scores: fp32 sums of D products, each add off by at most 2^-23 of the size, and a few roundings of a number of the
    score's size with the hardware exponential (2^-22); weights rounded to bf16; fp32 sums over the keys; one rounding
    of the result; a weight below 2^-126 of the largest may count as zero."""
    k, v = (_f64(t)[row0 : row0 + (tokens or len(t))] for t in slot.token_major())
    q = _f64(q)
    want, size = lowbit.attention(q, k, v, scale), lowbit.attention(q, k, np.abs(v), scale)
    reach = max(float((np.abs(q[:, i]) @ np.abs(k[:, i]).T).max()) for i in range(q.shape[1])) * abs(scale)
    weight = HALF_BF16 + 2 * (q.shape[2] + 8) * 2.0 ** -23 * reach + len(k) * 2.0 ** -23 + 2.0 ** -20
    return want, HALF_BF16 * np.abs(want) + 1.02 * weight * size + 2.0 ** -126 * np.abs(v).sum(0)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("rows,heads,dim,tokens", [(4700, 3, 128, 1500), (1025, 14, 128, 1500), (9000, 2, 64, 2500)])
def test_large_scores(torch_mod, dev, rows, heads, dim, tokens, fmt):
    from taomate_hd_amd import segment_attention

    torch = torch_mod
    k = _randn(torch, dev, tokens, heads, dim, seed=1) * torch.linspace(0.1, 6.0, tokens, device=dev).view(-1, 1, 1).to(torch.bfloat16)
    slot = _slot(torch, k, _randn(torch, dev, tokens, heads, dim, seed=2), fmt, dev)
    q = 8 * _randn(torch, dev, rows, heads, dim, seed=3)
    got = segment_attention(torch, q, [slot.view()], scale=dim ** -0.5)
    want, bound = _want(q, slot, dim ** -0.5)
    assert (np.abs(_f64(got) - want) <= bound).all()


@pytest.mark.parametrize("scale", [-0.3, 0.0, 40.0])
def test_other_scales(torch_mod, dev, scale):
    from taomate_hd_amd import segment_attention

    torch, rows, heads, dim, tokens = torch_mod, 4700, 3, 128, 1501
    slot = _slot(torch, *(_randn(torch, dev, tokens, heads, dim, seed=s) for s in (1, 2)), "int8", dev)
    q = _randn(torch, dev, rows, heads, dim, seed=3)
    got = segment_attention(torch, q, [slot.view()], scale=scale)
    want, bound = _want(q, slot, scale)
    assert (np.abs(_f64(got) - want) <= bound).all()


def test_scores_below_every_number(torch_mod, dev):
    """Scores of all but the last 34 keys overflow to -inf: they weigh nothing."""
    from taomate_hd_amd import segment_attention

    torch, rows, heads, dim, tokens = torch_mod, 6000, 3, 128, 1250
    k, v = (_randn(torch, dev, tokens, heads, dim, seed=s) for s in (1, 2))
    k[:1216] = -(2.0 ** 100)
    slot = _slot(torch, k, v, "int8", dev)
    q = 2.0 ** 40 * (1 + _randn(torch, dev, rows, heads, dim, seed=3).abs())
    got = segment_attention(torch, q, [slot.view()], scale=2.0 ** -43)
    want, bound = _want(q, slot, 2.0 ** -43, tokens=34, row0=1216)
    assert (np.abs(_f64(got) - want) <= bound).all()


@pytest.mark.parametrize("fmt", FORMATS)
def test_a_row_keeps_its_accuracy_in_a_larger_call(torch_mod, dev, fmt):
    """The 2-norm of the error of the same 300 rows, alone and among 5,000."""
    from taomate_hd_amd import segment_attention

    torch, heads, dim, tokens = torch_mod, 4, 128, 3000
    slot = _slot(torch, *(_randn(torch, dev, tokens, heads, dim, seed=s) for s in (1, 2)), fmt, dev)
    q = _randn(torch, dev, 5000, heads, dim, seed=3)
    want, _ = _want(q[:300], slot, dim ** -0.5)
    off = []
    for n in (300, 5000):
        got = _f64(segment_attention(torch, q[:n], [slot.view()], scale=dim ** -0.5)[:300])
        off.append(np.linalg.norm(got - want) / np.linalg.norm(want))
    # the same roundings of weights and results in another order of sums: the norms of n = 153,600 nearly independent
    # errors differ by about (2 n)^-1/2 = 0.2%
    assert abs(off[1] - off[0]) <= 0.02 * off[0], off


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("rows,heads,tokens,beside", [(None, 2, 1301, 0), (70, 3, 333, 90)])
def test_expanded_calls(torch_mod, dev, rows, heads, tokens, beside, fmt):
    """Calls beyond the in-place rule, and calls with a bf16 segment: within fp64's bound and what rounding the scaled Q
    to bf16 adds, 2^-8 of a score's products, twice (score and sum of weights)."""
    from taomate_hd_amd import KVSlot, attention, segment_attention

    torch, dim = torch_mod, 64
    rows = rows or attention.KV8_ROWS + 1
    assert beside or rows * heads * dim * tokens > attention.KV8_WORK
    k, v = (_randn(torch, dev, tokens + beside, heads, dim, seed=s) for s in (1, 2))
    slot = _slot(torch, k[:tokens], v[:tokens], fmt, dev)
    views = [slot.view()]
    kv = [_f64(t) for t in slot.token_major()]
    if beside:
        plain = KVSlot(torch, heads=heads, head_dim=dim, capacity=beside, device=dev)
        plain.pack(k[tokens:], v[tokens:])
        views.append(plain.view())
        kv = [np.concatenate([a, _f64(b[tokens:])]) for a, b in zip(kv, (k, v))]
    q = _randn(torch, dev, rows, heads, dim, seed=3)
    got = _f64(segment_attention(torch, q, views, scale=dim ** -0.5))
    qv = _f64(q)
    want = lowbit.attention(qv, *kv, dim ** -0.5)
    for i in range(heads):
        s = np.abs(qv[:, i]) @ np.abs(kv[0][:, i]).T * dim ** -0.5  # the size of a score's products
        p = np.exp(qv[:, i] @ kv[0][:, i].T * dim ** -0.5)
        p /= p.sum(-1, keepdims=True)
        # each score off by at most 2^-8 of its products (and 2^-15 of fp32's roundings): a weight by a factor of up to
        # e^that, the sum of weights by the largest of them; then as in _want
        off = np.exp(HALF_BF16 * s + 2.0 ** -15) - 1
        off = off + off.max(-1, keepdims=True) + HALF_BF16 + 2.0 ** -12
        bound = HALF_BF16 * np.abs(want[:, i]) + 1.05 * (p * off) @ np.abs(kv[1][:, i])
        assert (np.abs(got[:, i] - want[:, i]) <= bound).all()
    err = np.linalg.norm(got - want, axis=-1) / np.linalg.norm(want, axis=-1)
    assert np.median(err) <= 2.0 ** -7
