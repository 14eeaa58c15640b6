"""mxfp4_quant into caller storage."""

import pytest

pytestmark = pytest.mark.gpu


def _rows(torch, dev, rows, cols, seed):
    return torch.randn(rows, cols, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16).to(dev)


@pytest.mark.parametrize("rows,cols", [(1, 32), (3, 96), (4, 512), (37, 1056), (331, 5376), (0, 64)])
def test_same_bits_and_nothing_beside(torch_mod, dev, rows, cols):
    """Into the middle of larger buffers with stale contents, from contiguous and from strided rows."""
    from taomate_hd_amd import mxfp4_quant, mxfp4_quant_into
    from taomate_hd_amd.mxfp4 import scale_shape

    torch = torch_mod
    wide = _rows(torch, dev, rows, 2 * cols, rows + cols)
    shape = scale_shape(rows, cols)
    n = shape[0] * shape[1] * shape[2] * shape[3]
    for x in (wide[:, :cols].contiguous(), wide[:, cols:], wide[:, :cols].view(rows, 1, cols)):
        codes = torch.full((rows + 2, cols // 2), 0xA5, dtype=torch.uint8, device=dev)
        store = torch.full((n + 32,), 0xA5, dtype=torch.uint8, device=dev)
        q, scale = codes[1 : rows + 1], store[16 : n + 16].view(shape)
        assert mxfp4_quant_into(q, scale, x) is None
        want_q, want_scale = mxfp4_quant(x)
        assert torch.equal(q, want_q.view(rows, cols // 2)) and torch.equal(scale, want_scale)
        assert bool((codes[0] == 0xA5).all()) and bool((codes[rows + 1] == 0xA5).all())
        assert bool((store[:16] == 0xA5).all()) and bool((store[n + 16 :] == 0xA5).all())


def test_refusals(torch_mod, dev):
    from taomate_hd_amd import mxfp4_quant_into
    from taomate_hd_amd.mxfp4 import scale_shape

    torch = torch_mod
    x = _rows(torch, dev, 6, 64, 1)
    q = torch.empty(6, 32, dtype=torch.uint8, device=dev)
    scale = torch.empty(scale_shape(6, 64), dtype=torch.uint8, device=dev)
    for bad in (q[:5], q.view(12, 16), q.view(torch.int8), torch.empty(6, 64, dtype=torch.uint8, device=dev)[:, :32],
                torch.empty(6, 33, dtype=torch.uint8, device=dev)):
        with pytest.raises(ValueError, match="q must be"):
            mxfp4_quant_into(bad, scale, x)
    for bad in (scale[:, :, :4], scale.view(torch.int8), scale.transpose(1, 2)):
        with pytest.raises(ValueError, match="scale must be"):
            mxfp4_quant_into(q, bad, x)
    with pytest.raises(ValueError, match="multiple of 32"):
        mxfp4_quant_into(q, scale, x[:, :48])
    with pytest.raises(ValueError, match="bf16"):
        mxfp4_quant_into(q, scale, x.float())
    with pytest.raises(ValueError):
        mxfp4_quant_into(q.cpu(), scale, x)
    odd = torch.empty(6 * 32 + 8, dtype=torch.uint8, device=dev)[8:].view(6, 32)  # not 16-byte aligned
    with pytest.raises(ValueError, match="misaligned"):
        mxfp4_quant_into(odd, scale, x)
