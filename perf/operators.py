"""The block-scaled low-bit operators as timed cases: MXFP4 projections and the K/V cache held in 8 bits.

Kinds of case:

* ``quant``   rows of bf16 activations to MXFP4 (e2m1 codes, a power-of-two scale for each 32 values of a row) and
              back to the values they stand for;
* ``mm``      the product of activations and a weight that are both held in MXFP4, with or without a bias;
* ``linear``  a projection of bf16 rows on an MXFP4 weight: the rows quantised, then the product;
* ``pack``    K/V rows of a chunk written into a cache block held in 8 bits (a power-of-two scale for each 64 tokens
              of a head), and read back token-major as the cache's history is;
* ``attend``  attention of one or several calls' queries over such blocks, without a mask.

With ``own`` false ``run`` computes them from elementary torch operations in 32 bits; with ``own`` true it calls the
package.  ``exact`` gives the same outputs in 64 bits.
"""

import sys
from pathlib import Path

import torch

own = False

DEV = "cuda:0"
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
# largest value of an 8-bit code, as m * 2^x with 0.5 <= m < 1
TOP = {"e4m3": (0.875, 9), "int8": (0.9921875, 7)}


def _package():
    root = str(Path("taomate-hd_amd").resolve())
    if root not in sys.path:
        sys.path.insert(1, root)
    import taomate_hd_amd

    return taomate_hd_amd


def listed():
    return [
        # the prompt's rows in front of a projection: ragged row count, a call of a few microseconds
        {"name": "quant_prompt", "kind": "quant", "rows": 331, "cols": 5376},
        # the 768p chunk's hidden rows
        {"name": "quant_768p", "kind": "quant", "rows": 12252, "cols": 5376},
        # one token's projection, operands ready: the weight is what is read, latency counts
        {"name": "mm_token", "kind": "mm", "rows": 1, "cols": 5120, "out": 13824, "bias": True},
        # the prompt's rows on one rank's QKV weight
        {"name": "mm_prompt", "kind": "mm", "rows": 331, "cols": 5376, "out": 10752, "bias": False},
        # QKV projection of the 480p chunk on one rank
        {"name": "linear_480p", "kind": "linear", "rows": 4836, "cols": 5376, "out": 10752, "bias": False},
        # the 768p chunk's projection with a bias: the largest product
        {"name": "linear_768p", "kind": "linear", "rows": 12252, "cols": 5120, "out": 13824, "bias": True},
        # a clean 480p chunk of one rank written into its cache block
        {"name": "pack_480p", "kind": "pack", "fmt": "int8", "heads": 14, "dim": 128, "tokens": 4836, "gaps": False},
        # the same for all heads of the 480p history, its rows picked out of a packed sequence
        {"name": "pack_rows", "kind": "pack", "fmt": "e4m3", "heads": 40, "dim": 128, "tokens": 11232, "gaps": True},
        # one query token over the 768p history and chunk of one rank: three blocks, the cache is what is read
        {"name": "attend_token", "kind": "attend", "fmt": "e4m3", "heads": 14, "dim": 128, "calls": 1, "rows": 1,
         "tokens": 40788, "blocks": 3},
        # a few rows of several sequences in one batch, each over a cache of its own, heads of 64
        {"name": "attend_batch", "kind": "attend", "fmt": "int8", "heads": 8, "dim": 64, "calls": 8, "rows": 5,
         "tokens": 2717, "blocks": 1},
        # a chunk's audio rows over the 480p history, all heads
        {"name": "attend_audio", "kind": "attend", "fmt": "int8", "heads": 40, "dim": 128, "calls": 1, "rows": 91,
         "tokens": 11232, "blocks": 3},
        # the 480p chunk's queries of one rank over the 768p-long cache: bound by the matrix products
        {"name": "attend_480p", "kind": "attend", "fmt": "e4m3", "heads": 14, "dim": 128, "calls": 1, "rows": 4836,
         "tokens": 40788, "blocks": 3},
    ]


def _log_int(rng, low, high):
    return max(low, min(high, round(low * (high / low) ** rng.random())))


def draw(rng):
    kind = rng.choice(("quant", "mm", "mm", "linear", "linear", "pack", "attend", "attend", "attend"))
    if kind == "quant":
        return {"kind": kind, "rows": _log_int(rng, 1, 12252), "cols": 32 * _log_int(rng, 2, 168)}
    if kind in ("mm", "linear"):
        return {"kind": kind, "rows": _log_int(rng, 1, 12252), "cols": 32 * _log_int(rng, 4, 160),
                "out": _log_int(rng, 16, 13824), "bias": rng.random() < 0.5}
    heads, dim = rng.choice((8, 14, 28, 40)), 64 if rng.random() < 0.3 else 128
    if kind == "pack":
        return {"kind": kind, "fmt": rng.choice(("e4m3", "int8")), "heads": heads, "dim": dim,
                "tokens": _log_int(rng, 1, 11232), "gaps": rng.random() < 0.5}
    case = {"kind": kind, "fmt": rng.choice(("e4m3", "int8")), "heads": heads, "dim": dim,
            "calls": rng.choice((1, 1, 2, 5, 12)), "rows": _log_int(rng, 1, 4836), "tokens": _log_int(rng, 1, 40788),
            "blocks": rng.choice((1, 2, 3))}
    while case["calls"] * heads * case["rows"] * case["tokens"] > 14 * 4836 * 40788:
        case["rows"] = max(1, case["rows"] // 2)
        case["tokens"] = max(1, case["tokens"] * 3 // 4)
    return case


def _lengths(case):
    """Query rows and cached tokens of each block, for each call: ragged."""
    out = []
    for i in range(case["calls"]):
        rows = max(1, case["rows"] - i * case["rows"] // (2 * case["calls"]))
        tokens = max(1, case["tokens"] - i * case["tokens"] // (case["calls"] + 1))
        blocks = min(case["blocks"], tokens)
        first = max(1, tokens * 3 // (3 * blocks + 1))
        sizes = [first] * (blocks - 1)
        out.append((rows, [tokens - sum(sizes), *sizes]))
    return out


def work(case):
    if case["kind"] in ("quant", "mm", "linear"):
        m, k = case["rows"], case["cols"]
        if case["kind"] == "quant":
            # the rows once in, codes and scales once out; the values they stand for once out
            return {"bytes": m * k * 2 + m * k * 17 // 32 + m * k * 2, "flops": 2 * m * k}
        n = case["out"]
        a = m * k * 2 if case["kind"] == "linear" else m * k * 17 // 32
        return {"bytes": a + n * k * 17 // 32 + 2 * m * n + (2 * n if case["bias"] else 0), "flops": 2 * m * n * k}
    h, d = case["heads"], case["dim"]
    if case["kind"] == "pack":
        # K and V in bf16 in, codes out, and the values token-major in bf16 out
        n = case["tokens"] * h * d
        return {"bytes": 4 * n + 2 * n + 4 * n, "flops": 4 * n}
    rows = sum(r for r, _ in _lengths(case))
    tokens = sum(sum(s) for _, s in _lengths(case))
    pairs = sum(r * sum(s) for r, s in _lengths(case))
    return {"bytes": 4 * rows * h * d + 2 * tokens * h * d, "flops": 4 * h * d * pairs}


# ---- inputs


def _generator(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _normal(g, *shape, std=1.0):
    return (torch.randn(*shape, generator=g, device=DEV) * std).to(torch.bfloat16)


def _activations(g, rows, cols):
    """N(0, 1) with 1% outlier channels, as the block's hidden rows have them."""
    x = torch.randn(rows, cols, generator=g, device=DEV)
    x *= torch.where(torch.rand(cols, generator=g, device=DEV) < 0.01, 12.0, 1.0)
    return x.to(torch.bfloat16)


def _keys_values(g, tokens, heads, dim):
    """Keys N(0, 1) with a per-channel offset (after Q/K norm and rotation), values N(0, 1)."""
    k = torch.randn(tokens, heads, dim, generator=g, device=DEV) + 0.5 * torch.randn(heads, dim, generator=g, device=DEV)
    return k.to(torch.bfloat16), _normal(g, tokens, heads, dim)


# ---- plain forms


def _pow2(e):
    """2 ** e in 32 bits, exactly, for whole e in [-126, 127]."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _mx_quant(x):
    """MXFP4 of rows: the e2m1 values and the scales' exponents, one for each 32 values."""
    blocks = x.float().unflatten(-1, (-1, 32))
    amax = blocks.abs().amax(-1)
    e = torch.where(amax > 0, torch.frexp(amax).exponent - 3, -125).clamp_min(-125)  # floor(log2 amax) - 2
    y = (blocks * _pow2(-e).unsqueeze(-1)).clamp(-6.0, 6.0)
    size = y.abs()
    step = torch.where(size < 2.0, 0.5, torch.where(size < 4.0, 1.0, 2.0))
    return (torch.round(y / step) * step).flatten(-2), e


def _mx_values(v, e):
    return (v.unflatten(-1, (-1, 32)) * _pow2(e).unsqueeze(-1)).flatten(-2)


def _mx_pack(v, e):
    """Stored form: two codes a byte (the even column in the low half), and the scale bytes in the product's order:
    [512-column blocks][4][rows, to a multiple of 4][4], where byte b of entry g is that of columns 32 (4 b + g) .. of
    the 512; zero where there is no such column or row."""
    index = torch.tensor([0, 1, 2, 3, 4, 0, 5, 0, 6, 0, 0, 0, 7], dtype=torch.uint8, device=v.device)
    code = index[(v.abs() * 2).long()] | (torch.signbit(v).to(torch.uint8) << 3)
    rows, nb = e.shape
    scale = torch.zeros(-(-rows // 4) * 4, -(-nb // 16) * 16, dtype=torch.uint8, device=v.device)
    scale[:rows, :nb] = (e + 127).to(torch.uint8)
    scale = scale.view(scale.shape[0], -1, 4, 4).permute(1, 3, 0, 2).contiguous()
    return (code[:, 0::2] | (code[:, 1::2] << 4)).contiguous(), scale


def _mx_unpack(codes, scale):
    table = torch.tensor([*E2M1, *(-t for t in E2M1)], device=codes.device)
    v = torch.stack((table[(codes & 15).long()], table[(codes >> 4).long()]), -1).flatten(-2)
    e = scale.permute(2, 0, 3, 1).flatten(1)[: v.shape[0], : v.shape[1] // 32].int() - 127
    return _mx_values(v, e)


def _kv_quant(x, fmt):
    """[tokens, heads, dim] in 8 bits: codes token-major and the exponents [blocks of 64 tokens, heads]."""
    n, h, d = x.shape
    blocks = torch.nn.functional.pad(x.float(), (0, 0, 0, 0, 0, -n % 64)).view(-1, 64, h, d)
    m, ex = torch.frexp(blocks.abs().amax((1, 3)))
    top, shift = TOP[fmt]
    e = torch.where(m > 0, ex - shift + (m > top).int(), -117).clamp_min(-117)
    y = (blocks * _pow2(-e)[:, None, :, None]).view(-1, h, d)[:n]
    return (y.to(torch.float8_e4m3fn) if fmt == "e4m3" else torch.round(y).to(torch.int8)), e


def _kv_values(codes, e):
    return codes.float() * _pow2(e).repeat_interleave(64, 0)[: codes.shape[0], :, None]


def _plain_attend(q, blocks, scale):
    """One call: softmax over every block's keys, in 32 bits."""
    k = torch.cat([_kv_values(kc, ke) for kc, ke, _, _ in blocks]).permute(1, 2, 0).contiguous()
    v = torch.cat([_kv_values(vc, ve) for _, _, vc, ve in blocks]).permute(1, 0, 2).contiguous()
    s = torch.matmul(q.float().permute(1, 0, 2) * scale, k)
    s -= s.amax(-1, keepdim=True)
    p = s.exp_()
    total = p.sum(-1, keepdim=True)
    return (torch.matmul(p, v) / total).permute(1, 0, 2).to(torch.bfloat16)


# ---- the tools' entry points


def prepare(case, seed):
    g = _generator(seed)
    kind = case["kind"]
    if kind == "quant":
        return {"kind": kind, "x": _activations(g, case["rows"], case["cols"])}
    if kind in ("mm", "linear"):
        x = _activations(g, case["rows"], case["cols"])
        w = _normal(g, case["out"], case["cols"], std=0.02)
        bias = _normal(g, case["out"], std=0.5) if case["bias"] else None
        weight, weight_scale = _mx_pack(*_mx_quant(w))
        state = {"kind": kind, "weight": weight, "weight_scale": weight_scale, "bias": bias}
        if kind == "mm":
            state["a"], state["a_scale"] = _mx_pack(*_mx_quant(x))
        else:
            state["x"] = x
        return state
    h, d, fmt = case["heads"], case["dim"], case["fmt"]
    if kind == "pack":
        total = case["tokens"] * (2 if case["gaps"] else 1)
        k, v = _keys_values(g, total, h, d)
        rows = torch.randperm(total, generator=g, device=DEV)[: case["tokens"]].sort().values if case["gaps"] else None
        state = {"kind": kind, "fmt": fmt, "k": k, "v": v, "rows": rows}
        if own:  # the cache block that the rows are written to
            state["slot"] = _package().KVSlot8(torch, heads=h, head_dim=d, capacity=case["tokens"], device=DEV, fmt=fmt)
        return state
    calls = []
    for rows, sizes in _lengths(case):
        q = _normal(g, rows, 3 * h * d)[:, : h * d].view(rows, h, d)  # the Q part of a merged projection
        blocks = []
        for n in sizes:
            k, v = _keys_values(g, n, h, d)
            if own:  # the cache holds its blocks in the package's slots
                slot = _package().KVSlot8(torch, heads=h, head_dim=d, capacity=n, device=DEV, fmt=fmt)
                slot.pack(k, v)
                blocks.append(slot.view())
            else:
                blocks.append((*_kv_quant(k, fmt), *_kv_quant(v, fmt)))
        calls.append((q, blocks))
    return {"kind": kind, "calls": calls, "scale": d ** -0.5}


def _run_own(state):
    tm = _package()
    kind = state["kind"]
    if kind == "quant":
        return tm.mxfp4_dequant(*tm.mxfp4_quant(state["x"]))
    if kind == "mm":
        return tm.mxfp4_scaled_mm(state["a"], state["weight"].t(), state["a_scale"], state["weight_scale"],
                                  bias=state["bias"])
    if kind == "linear":
        return tm.mxfp4_linear(state["x"], state["weight"], state["weight_scale"], state["bias"])
    if kind == "pack":
        state["slot"].pack(state["k"], state["v"], rows=state["rows"], rows_checked=True)
        return state["slot"].token_major()
    if len(state["calls"]) == 1:
        q, blocks = state["calls"][0]
        return tm.segment_attention(torch, q, blocks, scale=state["scale"])
    return tm.segment_attention_batch(torch, [tm.AttentionCall(q, blocks) for q, blocks in state["calls"]],
                                      scale=state["scale"])[0]


def run(state):
    if own:
        return _run_own(state)
    kind = state["kind"]
    if kind == "quant":
        return _mx_values(*_mx_quant(state["x"])).to(torch.bfloat16)
    if kind in ("mm", "linear"):
        a = _mx_values(*_mx_quant(state["x"])) if kind == "linear" else _mx_unpack(state["a"], state["a_scale"])
        out = torch.matmul(a, _mx_unpack(state["weight"], state["weight_scale"]).t())
        return (out if state["bias"] is None else out + state["bias"].float()).to(torch.bfloat16)
    if kind == "pack":
        k, v = (t if state["rows"] is None else t[state["rows"]] for t in (state["k"], state["v"]))
        return tuple(_kv_values(*_kv_quant(t, state["fmt"])).to(torch.bfloat16) for t in (k, v))
    outs = [_plain_attend(q, blocks, state["scale"]) for q, blocks in state["calls"]]
    return outs[0] if len(outs) == 1 else outs


# ---- 64 bits, from the definitions


def _floor_log2(x):
    """floor(log2 x) of positive doubles, from the exponent field."""
    return (x.view(torch.int64) >> 52) - 1023


def _power(e):
    return ((e + 1023) << 52).view(torch.float64)


def _exact_mx(x):
    """The values that MXFP4 of ``x`` stands for."""
    b = x.double().reshape(x.shape[0], -1, 32)
    amax = b.abs().max(2, keepdim=True).values
    scale = _power((_floor_log2(amax.clamp_min(2.0 ** -140)) - 2).clamp_min(-125))
    size = b.abs() / scale
    # the number of grid midpoints passed; at a midpoint the neighbour with the even code is taken
    grid = torch.tensor(E2M1, dtype=torch.float64, device=x.device)
    passed = torch.zeros_like(size, dtype=torch.long)
    for i in range(7):
        mid = (E2M1[i] + E2M1[i + 1]) / 2
        passed += (size > mid) if i % 2 == 0 else (size >= mid)
    return (torch.copysign(grid[passed], b) * scale).reshape(x.shape)


def _exact_kv(x, fmt):
    """The values that the 8-bit form of ``x`` ([tokens, heads, dim]) stands for."""
    top = 448.0 if fmt == "e4m3" else 127.0
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    for at in range(0, x.shape[0], 64):
        b = x[at : at + 64].double()
        amax = b.abs().amax((0, 2), keepdim=True)
        e = _floor_log2((amax / top).clamp_min(2.0 ** -117))  # the least e with amax <= top * 2 ** e, or one below it
        e = torch.where(amax > top * _power(e), e + 1, e)
        y = b / _power(e)
        if fmt == "e4m3":
            step = _power(_floor_log2(y.abs().clamp_min(2.0 ** -6)) - 3)
            y = torch.round(y / step) * step
        else:
            y = torch.round(y)
        out[at : at + 64] = y * _power(e)
    return out


def exact(case, seed):
    g = _generator(seed)
    kind = case["kind"]
    if kind == "quant":
        return _exact_mx(_activations(g, case["rows"], case["cols"]))
    if kind in ("mm", "linear"):
        x = _activations(g, case["rows"], case["cols"])
        w = _normal(g, case["out"], case["cols"], std=0.02)
        bias = _normal(g, case["out"], std=0.5) if case["bias"] else None
        out = _exact_mx(x) @ _exact_mx(w).t()
        return out if bias is None else out + bias.double()
    h, d, fmt = case["heads"], case["dim"], case["fmt"]
    if kind == "pack":
        total = case["tokens"] * (2 if case["gaps"] else 1)
        k, v = _keys_values(g, total, h, d)
        if case["gaps"]:
            rows = torch.randperm(total, generator=g, device=DEV)[: case["tokens"]].sort().values
            k, v = k[rows], v[rows]
        return _exact_kv(k, fmt), _exact_kv(v, fmt)
    outs = []
    for rows, sizes in _lengths(case):
        q = _normal(g, rows, 3 * h * d)[:, : h * d].reshape(rows, h, d).double()
        pairs = [tuple(_exact_kv(t, fmt) for t in _keys_values(g, n, h, d)) for n in sizes]
        k, v = torch.cat([p[0] for p in pairs]), torch.cat([p[1] for p in pairs])
        out = torch.empty(rows, h, d, dtype=torch.float64, device=DEV)
        for i in range(h):
            p = torch.softmax(q[:, i] @ k[:, i].t() * d ** -0.5, -1)
            out[:, i] = p @ v[:, i]
        outs.append(out)
    return outs[0] if len(outs) == 1 else outs
