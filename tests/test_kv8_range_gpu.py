"""K/V slots in 8 bits at the ends of what bf16 holds."""

import numpy as np
import pytest

from oracle import bf16, lowbit

pytestmark = pytest.mark.gpu

FORMATS = ("e4m3", "int8")
# (rows, heads, head_dim, rows of an item) of calls over 71 tokens that take each attention kernel
KERNELS = [(3, 2, 64, 32), (100, 3700, 64, 128), (200, 2200, 64, 256), (90, 2500, 128, 128), (300, 800, 128, 256)]


def _slot(torch, k, v, fmt, dev):
    from taomate_hd_amd import KVSlot8

    slot = KVSlot8(torch, heads=int(k.shape[1]), head_dim=int(k.shape[2]), capacity=int(k.shape[0]), device=dev, fmt=fmt)
    slot.pack(k, v)
    return slot


def _from_bits(torch, bits):
    return torch.where(bits >= 32768, bits - 65536, bits).to(torch.int16).view(torch.bfloat16)


def _f64(t):
    return bf16.from_torch(t.cpu()).astype(np.float64)


@pytest.mark.parametrize("fmt", FORMATS)
def test_pack_of_the_largest_numbers(torch_mod, dev, fmt):
    """Each of the largest 256 magnitudes, of both signs, as the largest of its block: what is read back is finite and
    what the oracle says, in each reader."""
    from taomate_hd_amd.slots import expand_views

    torch, d = torch_mod, 64
    g = torch.Generator().manual_seed(11)
    top = torch.cat([torch.arange(0x7E80, 0x7F80), torch.arange(0xFE80, 0xFF80)]).to(torch.int32)
    mag = (top & 0x7FFF).unsqueeze(1)
    # most of a block within 32 steps of its largest, some far below
    near = (mag - torch.randint(0, 32, (512, 64 * d - 1), generator=g)).clamp_min(0)
    far = (mag - torch.randint(0, 1600, near.shape, generator=g)).clamp_min(0)
    other = torch.where(torch.rand(near.shape, generator=g) < 0.7, near, far)
    other = other | (torch.randint(0, 2, other.shape, generator=g, dtype=torch.int32) << 15)
    x = _from_bits(torch, torch.cat([top.unsqueeze(1), other], 1)).view(512 * 64, 1, d).to(dev)
    slot = _slot(torch, x, x, fmt, dev)
    want, byte = lowbit.kv8_values(_f64(x), fmt)
    assert np.abs(want).max() < 2.0 ** 128
    for got, scale in zip(slot.token_major(), (slot.k_scale, slot.v_scale)):
        np.testing.assert_array_equal(scale.cpu().numpy().T, byte)
        np.testing.assert_array_equal(_f64(got), want)
    for got in expand_views(torch, [slot.view()])[0].slot.token_major():
        np.testing.assert_array_equal(_f64(got), want)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("rows,heads,dim,items", KERNELS)
def test_attention_over_the_largest_numbers(torch_mod, dev, rows, heads, dim, items, fmt):
    """Values of the largest magnitude bf16 holds, one of them with all of the weight: it comes out."""
    from taomate_hd_amd import _native, segment_attention

    torch, n = torch_mod, 71
    call = (_native.KV8Call * 1)()
    c = call[0]
    c.q, c.o, c.q_token_stride, c.q_head_stride, c.o_token_stride, c.o_head_stride = 4096, 4096, 128, 64, 128, 64
    c.lq, c.n_segments = rows, 1
    c.seg[0] = _native.KV8Segment(4096, 4096, 4096, 4096, 128, 0, n, 0)
    assert _native.load().tmhd_attn_kv8_item_rows(call, 1, heads, dim, 0) == items
    k = torch.zeros(n, heads, dim, dtype=torch.bfloat16, device=dev)
    k[3] = 8.0  # a score of 8 dim against 0: the other weights are zero
    bits = torch.tensor([0x7F7F, 0xFF7F, 0x7F78], dtype=torch.int32).repeat(n)[: n].view(n, 1, 1).expand(n, heads, dim)
    v = _from_bits(torch, bits).contiguous().to(dev)
    v[64:] = 0.0  # (keys that another wave sums before it sees the large score)
    slot = _slot(torch, k, v, fmt, dev)
    q = torch.ones(rows, heads, dim, dtype=torch.bfloat16, device=dev)
    got = segment_attention(torch, q, [slot.view()], scale=1.0)
    # one weight of 1, a product and a quotient by 1: no rounding
    want = slot.token_major()[1][3]
    assert bool(torch.isfinite(want).all())
    assert torch.equal(got, want.expand(rows, heads, dim))
