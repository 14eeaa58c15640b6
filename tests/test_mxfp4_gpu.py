"""MXFP4 quantization and product against the float64 oracle."""

import numpy as np
import pytest

from oracle import bf16, lowbit

pytestmark = pytest.mark.gpu

# half a bf16 step, relative to the value
HALF_BF16 = 2.0 ** -8


def _rows(torch, rows, cols, seed, dev, spread=0.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=g)
    if spread:  # blocks of very different sizes
        x = x * torch.exp2(torch.randint(-int(spread), int(spread) + 1, (rows, cols), generator=g).float())
    return x.to(torch.bfloat16).to(dev)


def _f64(t):
    return bf16.from_torch(t.cpu()).astype(np.float64)


def _check_quant(torch, x):
    from taomate_hd_amd import mxfp4_dequant, mxfp4_quant, mxfp4_scale_to_rows

    q, scale = mxfp4_quant(x)
    flat = x.reshape(-1, x.shape[-1])
    want, byte = lowbit.mxfp4_values(_f64(flat))
    got = _f64(mxfp4_dequant(q, scale)).reshape(want.shape)
    np.testing.assert_array_equal(mxfp4_scale_to_rows(scale, *flat.shape).cpu().numpy(), byte)
    np.testing.assert_array_equal(got, want)
    # entries of rows and columns that do not exist are zero
    assert int((scale != 0).sum()) == byte.size
    return q, scale


@pytest.mark.parametrize("rows,cols", [(1, 32), (3, 64), (5, 480), (4, 512), (17, 544), (33, 5376), (130, 1056)])
def test_quant_is_exact(torch_mod, dev, rows, cols):
    _check_quant(torch_mod, _rows(torch_mod, rows, cols, rows * 7 + cols, dev, spread=3))


def test_quant_of_every_bf16_value(torch_mod, dev):
    """Every finite bf16 as the largest of its block, among random smaller ones."""
    torch = torch_mod
    g = torch.Generator().manual_seed(5)
    bits = torch.arange(65536, dtype=torch.int32)
    bits = bits[(bits & 0x7F80) != 0x7F80]
    n = int(bits.numel())
    mag = (bits & 0x7FFF).unsqueeze(1)
    other = (torch.rand(n, 31, generator=g) * (mag + 1)).int().clamp(max=mag.expand(n, 31))
    near = (mag - torch.randint(0, 512, (n, 31), generator=g)).clamp_min(0)  # within four binades
    other = torch.where(torch.rand(n, 31, generator=g) < 0.7, near, other)
    other = other | (torch.randint(0, 2, (n, 31), generator=g) << 15)
    block = torch.cat([bits.unsqueeze(1), other], 1)
    x = torch.where(block >= 32768, block - 65536, block).to(torch.int16).view(torch.bfloat16)
    _check_quant(torch, x.reshape(-1, 128).to(dev))


def test_quant_of_strided_views_and_nonfinite_blocks(torch_mod, dev):
    torch = torch_mod
    base = _rows(torch, 37, 1536, 3, dev)
    _check_quant(torch, base[:, 512:1056])  # row stride 1536
    _check_quant(torch, base[:, 4:516])  # rows not 16-byte aligned: copied
    _check_quant(torch, base.view(37, 3, 512).transpose(0, 1))
    _check_quant(torch, base[:1].expand(5, 1536))
    x = _rows(torch, 6, 512, 4, dev)
    x[0, 3], x[1, 40], x[2, 511], x[4] = float("inf"), float("-inf"), float("nan"), 0.0
    _check_quant(torch, x)


def _product(torch, dev, m, n, k, seed, bias):
    from taomate_hd_amd import mxfp4_quant

    x, w = _rows(torch, m, k, seed, dev, spread=1), _rows(torch, n, k, seed + 1, dev, spread=1)
    b = _rows(torch, 1, n, seed + 2, dev)[0] if bias else None
    (a, sa), (wq, sw) = mxfp4_quant(x), mxfp4_quant(w)
    av, wv = lowbit.mxfp4_values(_f64(x))[0], lowbit.mxfp4_values(_f64(w))[0]
    want = av @ wv.T
    size = np.abs(av) @ np.abs(wv).T  # an fp32 sum of k terms is off by at most k steps of 2^-23 of it
    if bias:
        want = want + _f64(b)
        size = size + np.abs(_f64(b))
    return a, sa, wq, sw, b, want, (k + 1) * 2.0 ** -23 * size


def _close(got, want, slack):
    err = np.abs(_f64(got) - want)
    assert (err <= HALF_BF16 * (np.abs(want) + slack) + slack).all(), float((err - HALF_BF16 * np.abs(want)).max())


PRODUCTS = [(1, 16, 32), (1, 1, 32), (2, 17, 96), (16, 40, 512), (17, 33, 544), (64, 70, 1024), (65, 130, 480),
            (130, 257, 2048), (300, 520, 5376), (513, 300, 288)]


@pytest.mark.parametrize("m,n,k", PRODUCTS)
@pytest.mark.parametrize("bias", [False, True])
def test_product(torch_mod, dev, m, n, k, bias):
    from taomate_hd_amd import mxfp4_scaled_mm

    a, sa, w, sw, b, want, slack = _product(torch_mod, dev, m, n, k, m + n + k, bias)
    _close(mxfp4_scaled_mm(a, w.t(), sa, sw, bias=b), want, slack)


@pytest.mark.parametrize("m", [1, 40, 300])
def test_product_of_views(torch_mod, dev, m):
    """Operand rows with a stride, an output inside a larger matrix, and rows past it left alone."""
    from taomate_hd_amd import mxfp4_scaled_mm_out

    torch, n, k = torch_mod, 259, 640
    a, sa, w, sw, b, want, slack = _product(torch, dev, m, n, k, 11, True)
    wide_a = torch.full((m, k), 0xFF, dtype=torch.uint8, device=dev)
    wide_w = torch.full((n, k), 0xFF, dtype=torch.uint8, device=dev)
    wide_a[:, : k // 2], wide_w[:, : k // 2] = a, w
    for at in (8, 3):  # an odd first column: no wide stores
        out = torch.full((m + 2, n + 16), 7.0, dtype=torch.bfloat16, device=dev)
        mxfp4_scaled_mm_out(out[1 : m + 1, at : at + n], wide_a[:, : k // 2], wide_w[:, : k // 2].t(), sa, sw, b)
        _close(out[1 : m + 1, at : at + n], want, slack)
        out[1 : m + 1, at : at + n] = 7.0
        assert bool((out == 7.0).all())


@pytest.mark.parametrize("m", [256, 300])
def test_rows_far_apart(torch_mod, dev, m):
    """Rows 16 MiB apart: offsets just below 2^32 (tiles) and beyond (rows), of codes, of bf16 rows and of outputs."""
    from taomate_hd_amd import mxfp4_linear, mxfp4_quant, mxfp4_scaled_mm, mxfp4_scaled_mm_out

    torch, n, k, far = torch_mod, 40, 544, 1 << 24
    a, sa, w, sw, b, want, slack = _product(torch, dev, m, n, k, 21, True)
    codes = torch.empty(m, far, dtype=torch.uint8, device=dev)[:, : k // 2]
    codes.copy_(a)
    got = mxfp4_scaled_mm(codes, w.t(), sa, sw, bias=b)
    _close(got, want, slack)
    out = torch.empty(m, far // 2, dtype=torch.bfloat16, device=dev)[:, 8 : 8 + n]
    mxfp4_scaled_mm_out(out, codes, w.t(), sa, sw, b)
    assert torch.equal(out, got)
    weight = torch.empty(m, far, dtype=torch.uint8, device=dev)[:, : k // 2]  # as the other operand
    weight.copy_(a)
    _close(mxfp4_scaled_mm(w, weight.t(), sw, sa), (want - _f64(b)).T, slack.T)
    x = torch.empty(m, far // 2, dtype=torch.bfloat16, device=dev)[:, :k]
    x.copy_(_rows(torch, m, k, 22, dev))
    q, scale = mxfp4_quant(x)
    for got, same in zip((q, scale), mxfp4_quant(x.contiguous())):
        assert torch.equal(got, same)
    assert torch.equal(mxfp4_linear(x, w, sw), mxfp4_scaled_mm(q, w.t(), scale, sw))


def test_two_streams_at_once(torch_mod, dev):
    """Projections of other rows on the same weight, queued on two streams side by side."""
    from taomate_hd_amd import mxfp4_linear, mxfp4_quant

    torch = torch_mod
    w, ws = mxfp4_quant(_rows(torch, 5376, 1056, 1, dev))
    rows = [_rows(torch, m, 1056, m, dev) for m in (900, 1, 333, 16)]
    want = [mxfp4_linear(x, w, ws) for x in rows]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for _ in range(10):
        for i, x in enumerate(rows):
            with torch.cuda.stream(streams[i % 2]):
                got.append((i, mxfp4_linear(x, w, ws)))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i]) for i, y in got)


def test_product_with_a_nan_block(torch_mod, dev):
    """A block of NaN makes its row (or column) NaN and nothing else."""
    from taomate_hd_amd import mxfp4_quant, mxfp4_scaled_mm

    torch = torch_mod
    for m in (3, 70, 300):
        x, w = _rows(torch, m, 512, 1, dev), _rows(torch, 40, 512, 2, dev)
        x[2, 100] = float("nan")
        w[5, 3] = float("inf")
        a, sa = mxfp4_quant(x)
        b, sb = mxfp4_quant(w)
        nan = torch.isnan(mxfp4_scaled_mm(a, b.t(), sa, sb)).cpu()
        want = torch.zeros(m, 40, dtype=torch.bool)
        want[2], want[:, 5] = True, True
        assert torch.equal(nan, want)


def test_linear_equals_its_parts(torch_mod, dev):
    from taomate_hd_amd import mxfp4_linear, mxfp4_quant, mxfp4_scaled_mm

    torch = torch_mod
    w, ws = mxfp4_quant(_rows(torch, 200, 544, 1, dev))
    bias = _rows(torch, 1, 200, 2, dev)[0]
    for shape in ((1,), (16,), (3, 7), (65,), (2, 150), (0,)):
        x = _rows(torch, max(1, int(np.prod(shape))), 544, 3, dev)[: int(np.prod(shape))].view(*shape, 544)
        got = mxfp4_linear(x, w, ws, bias)
        assert got.shape == (*shape, 200)
        a, sa = mxfp4_quant(x.reshape(-1, 544))
        assert torch.equal(got.reshape(-1, 200), mxfp4_scaled_mm(a, w.t(), sa, ws, bias=bias))


def test_scale_orders(torch_mod, dev):
    from taomate_hd_amd import mxfp4_scale_from_rows, mxfp4_scale_to_rows

    torch = torch_mod
    for rows, nb in ((1, 1), (3, 17), (4, 16), (9, 33)):
        s = torch.randint(1, 255, (rows, nb), dtype=torch.uint8, device=dev)
        assert torch.equal(mxfp4_scale_to_rows(mxfp4_scale_from_rows(s), rows, nb * 32), s)


def test_on_another_stream_and_in_a_graph(torch_mod, dev):
    from taomate_hd_amd import mxfp4_linear, mxfp4_quant

    torch = torch_mod
    w, ws = mxfp4_quant(_rows(torch, 300, 1024, 1, dev))
    x = _rows(torch, 70, 1024, 2, dev)
    want = mxfp4_linear(x, w, ws)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        other = mxfp4_linear(x, w, ws)
    stream.synchronize()
    assert torch.equal(other, want)
    graph = torch.cuda.CUDAGraph()
    held = x.clone()
    with torch.cuda.graph(graph):
        out = mxfp4_linear(held, w, ws)
    for seed in (3, 4, 5):
        new = _rows(torch, 70, 1024, seed, dev)
        held.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, mxfp4_linear(new, w, ws))


# Products that take each form: one and more blocks of k, odd numbers of them, k ending inside a block and inside a
# scale word, ragged edges, one and several tiles a workgroup, last rounds in parts
TILED = {
    "ROWS": [(16, 640, 2080), (5, 4000, 96)],
    "64X64": [(17, 130, 32), (65, 128, 768), (129, 131, 800), (1, 13824, 1056), (1000, 640, 544)],
    "128X64": [(200, 5376, 512), (331, 5300, 1312), (2048, 640, 2048)],
    "128X128": [(200, 10752, 544), (512, 5376, 1024), (700, 5003, 288)],
    "128X128X2": [(331, 13824, 256), (2048, 5376, 1056), (1030, 8200, 32)],
    "256X256": [(12252, 5376, 512), (12252, 5376, 2336), (12000, 5200, 64)],
}


@pytest.mark.parametrize("form,m,n,k", [(f, *size) for f, sizes in TILED.items() for size in sizes])
def test_forms_of_the_product(torch_mod, dev, form, m, n, k):
    from taomate_hd_amd import _native

    assert _native.load().tmhd_gemm_mxfp4_form(m, n, k, 0) == getattr(_native, f"MXFP4_{form}")
    _check_whole(torch_mod, dev, m, n, k)


# 256 x 256 tiles in whole rounds, the last ones in parts
@pytest.mark.parametrize("m,n,k", [(4836, 10752, 5376), (12252, 13824, 1056), (4352, 4000, 2080)])
def test_last_rounds_in_parts(torch_mod, dev, m, n, k):
    from taomate_hd_amd import _native

    assert -(-m // 256) * -(-n // 256) > 256
    assert _native.load().tmhd_gemm_mxfp4_form(m, n, k, 0) in (
        _native.MXFP4_64X64, _native.MXFP4_128X64, _native.MXFP4_128X128)
    _check_whole(torch_mod, dev, m, n, k)


def _check_whole(torch, dev, m, n, k):
    """A whole product against an fp64 product on the GPU, and the row behind it left alone."""
    from taomate_hd_amd import mxfp4_dequant, mxfp4_quant, mxfp4_scaled_mm_out

    x, w, b = _rows(torch, m, k, 1, dev, spread=1), _rows(torch, n, k, 2, dev, spread=1), _rows(torch, 1, n, 3, dev)[0]
    (a, sa), (wq, sw) = mxfp4_quant(x), mxfp4_quant(w)
    av, wv = mxfp4_dequant(a, sa).double(), mxfp4_dequant(wq, sw).double()
    for bias in (b, None):
        want = av @ wv.t()
        slack = av.abs() @ wv.abs().t()
        if bias is not None:
            want += b.double()
            slack += b.double().abs()
        slack *= (k + 1) * 2.0 ** -23
        out = torch.full((m + 1, n), 7.0, dtype=torch.bfloat16, device=dev)
        mxfp4_scaled_mm_out(out[:m], a, wq.t(), sa, sw, bias)
        err = (out[:m].double() - want).abs()
        assert bool((err <= HALF_BF16 * (want.abs() + slack) + slack).all())
        assert bool((out[m] == 7.0).all())
