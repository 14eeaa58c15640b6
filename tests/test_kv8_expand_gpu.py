"""Expansion of 8-bit views: the bf16 slot is zero behind each view, whatever the 8-bit slot holds there."""

import pytest

pytestmark = pytest.mark.gpu

FORMATS = ("e4m3", "int8")


def _randn(torch, dev, *shape, seed):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16).to(dev)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("bad", [False, True])
def test_rows_behind_a_view_are_zero(torch_mod, dev, bad, dim, fmt):
    """Every length that ends inside a block, alone in one call; with ``bad`` the block has no finite values."""
    from taomate_hd_amd import KVSlot, KVSlot8
    from taomate_hd_amd.slots import SlotView, expand_views

    torch, heads = torch_mod, 2
    k, v = (_randn(torch, dev, 192, heads, dim, seed=s) for s in (1, 2))
    if bad:
        k[130, 1, 5], v[131, 0, 7] = float("inf"), float("nan")  # the block from row 128 on
    slot = KVSlot8(torch, heads=heads, head_dim=dim, capacity=192, device=dev, fmt=fmt)
    slot.pack(k, v)
    keys, values = slot.token_major()
    if bad:
        assert bool(torch.isnan(keys[128:, 1]).all()) and bool(torch.isnan(values[128:, 0]).all())
    views = [SlotView(slot, n, 128) for n in range(1, 65)] + [SlotView(slot, 64 + n, 64) for n in (1, 13, 36, 63)]
    views = expand_views(torch, views)
    for n, view in zip((*range(1, 65), 65, 77, 100, 127), views):
        first = 128 if n <= 64 else 64
        want = KVSlot(torch, heads=heads, head_dim=dim, capacity=n, device=dev)
        want.pack(keys[first : first + n].contiguous(), values[first : first + n].contiguous())
        at, cap = view.row0, want.capacity
        got_k, got_v = view.slot.k[:, at : at + cap], view.slot.vt[:, :, at : at + cap]
        for got, exp in ((got_k, want.k), (got_v, want.vt)):  # (bits, for the NaN)
            assert torch.equal(got.contiguous().view(torch.int16), exp.contiguous().view(torch.int16)), n
