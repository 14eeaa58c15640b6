"""The low-bit operators together, as a layer of a decoder runs them: MXFP4 projection, norm + RoPE, the K/V rows into
an 8-bit block, attention over history and chunk in 8 bits, MXFP4 output projection."""

import numpy as np
import pytest

from oracle import bf16, lowbit

pytestmark = pytest.mark.gpu

HALF_BF16 = 2.0 ** -8
HEADS, DIM, HIDDEN, HISTORY = 6, 128, 544, 200


def _f64(t):
    return bf16.from_torch(t.cpu()).astype(np.float64)


def _randn(torch, dev, *shape, seed):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16).to(dev)


class _Layer:
    def __init__(self, torch, dev, fmt, tokens):
        from taomate_hd_amd import KVSlot8, mxfp4_quant

        width = HEADS * DIM
        self.torch, self.tokens = torch, tokens
        self.weights = [_randn(torch, dev, 3 * width, HIDDEN, seed=1) / 16, _randn(torch, dev, HIDDEN, width, seed=2) / 16]
        self.qkv_w, self.out_w = (mxfp4_quant(w) for w in self.weights)
        self.bias = _randn(torch, dev, HIDDEN, seed=3)
        self.norm = 1 + _randn(torch, dev, DIM, seed=4) / 8
        angle = torch.arange(4 * HISTORY).float()[:, None] / 10 ** (torch.arange(DIM // 2) / 16)
        self.cos_sin = torch.cat([angle.cos(), angle.sin()], 1).to(torch.bfloat16).to(dev)
        self.positions = torch.arange(HISTORY, HISTORY + tokens, device=dev)
        self.history = KVSlot8(torch, heads=HEADS, head_dim=DIM, capacity=HISTORY, device=dev, fmt=fmt)
        self.history.pack(*(_randn(torch, dev, HISTORY, HEADS, DIM, seed=s) for s in (5, 6)))
        self.chunk = KVSlot8(torch, heads=HEADS, head_dim=DIM, capacity=tokens, device=dev, fmt=fmt)

    def __call__(self, x):
        from taomate_hd_amd import fused_qkv_qk_norm_rope_, mxfp4_linear, segment_attention

        raw = mxfp4_linear(x, *self.qkv_w)
        qkv = fused_qkv_qk_norm_rope_(raw.clone(), self.norm, self.norm, self.cos_sin, self.positions, 1e-6)
        q, k, v = qkv.view(self.tokens, 3, HEADS, DIM).unbind(1)
        self.chunk.pack(k, v)
        views = [self.history.view(), self.chunk.view()]
        attended = segment_attention(self.torch, q, views, scale=DIM ** -0.5)
        return raw, q, k, v, attended, mxfp4_linear(attended.flatten(1), *self.out_w, bias=self.bias)


def _projection(got, x, weight, bias=None):
    """A projection's output against the float64 product of what its operands' codes stand for."""
    a, w = lowbit.mxfp4_values(_f64(x))[0], lowbit.mxfp4_values(_f64(weight))[0]
    want, size = a @ w.T, np.abs(a) @ np.abs(w).T
    if bias is not None:
        want, size = want + _f64(bias), size + np.abs(_f64(bias))
    # fp32 sums of K terms (and the bias), each off by at most 2^-23 of the size, then one rounding
    slack = (a.shape[1] + 1) * 2.0 ** -23 * size
    assert (np.abs(_f64(got) - want) <= HALF_BF16 * (np.abs(want) + slack) + slack).all()


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("tokens", [1, 70, 333])
def test_layer(torch_mod, dev, fmt, tokens):
    torch = torch_mod
    layer = _Layer(torch, dev, fmt, tokens)
    x = _randn(torch, dev, tokens, HIDDEN, seed=7)
    raw, q, k, v, attended, y = layer(x)
    _projection(raw, x, layer.weights[0])
    for got, rows in zip(layer.chunk.token_major(), (k, v)):
        np.testing.assert_array_equal(_f64(got), lowbit.kv8_values(_f64(rows), fmt)[0])
    past = [_f64(t) for t in layer.history.token_major()]
    keys, values = (np.concatenate([p, lowbit.kv8_values(_f64(t), fmt)[0]]) for p, t in zip(past, (k, v)))
    qv = _f64(q)
    want = lowbit.attention(qv, keys, values, DIM ** -0.5)
    size = lowbit.attention(qv, keys, np.abs(values), DIM ** -0.5)
    # scores: fp32 sums of DIM products, then a few roundings of a number of the score's size and the hardware
    # exponential (2^-22); weights rounded to bf16; fp32 sums over the keys; one rounding of the result
    reach = max(float((np.abs(qv[:, i]) @ np.abs(keys[:, i]).T).max()) for i in range(HEADS)) * DIM ** -0.5
    weight = HALF_BF16 + 2 * (DIM + 8) * 2.0 ** -23 * reach + len(keys) * 2.0 ** -23 + 2.0 ** -20
    assert (np.abs(_f64(attended) - want) <= HALF_BF16 * np.abs(want) + 1.02 * weight * size).all()
    _projection(y, attended.flatten(1), layer.weights[1], layer.bias)


@pytest.mark.parametrize("tokens", [1, 333])
def test_layer_captured(torch_mod, dev, tokens):
    """Captured once and replayed with other rows, eager runs of the same layer in between."""
    torch = torch_mod
    layer = _Layer(torch, dev, "e4m3", tokens)
    x = _randn(torch, dev, tokens, HIDDEN, seed=8)
    layer(x)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer(x)[-1]
    for seed in (9, 10, 11):
        x.copy_(_randn(torch, dev, tokens, HIDDEN, seed=seed))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, layer(x)[-1])
