"""The streaming hook over a cache held in 8 bits, against the same hook over a bf16 cache of the same values.

Where a call has bf16 segments (condition rows, a noisy step's own rows) or the INT8-QK backend, history is expanded,
which is exact: the outputs are the same bits.  Where all of its segments are 8-bit ones their codes are read in place:
the outputs are held against fp64."""

import numpy as np
import pytest

from oracle import bf16, lowbit
from oracle import stream as ost
from tests.helpers import key_offset, randn_bf16, to_dev

pytestmark = pytest.mark.gpu

LAYERS = ("blocks.0.attn", "blocks.1.attn")
H, D = 2, 128
FORMATS = ("e4m3", "int8")


class _Attn:
    softmax_scale = D ** -0.5


def _data(dev, tokens, seed):
    q = randn_bf16((tokens, H, D), seed)
    k = randn_bf16((tokens, H, D), seed + 1, offset=key_offset(H, D, seed + 2))
    return [to_dev(x, dev) for x in (q, k, randn_bf16((tokens, H, D), seed + 3))]


class _Run:
    """One hook and its cache, driven step by step."""

    def __init__(self, torch, dev, storage, backend):
        from taomate_hd_amd import HeadMajorRingKVCache, KVContract, StreamingAttentionHook

        self.torch, self.dev = torch, dev
        self.cache = HeadMajorRingKVCache(KVContract(layer_names=LAYERS, local_heads=H, head_dim=D), storage=storage)
        self.hook = StreamingAttentionHook(self.cache, attention_backend=backend)

    def step(self, mode, block, data, layout, hint=None, **policy):
        """Outputs of both layers, and the K/V rows that the step staged, in the order of its commit rows."""
        from taomate_hd_amd.hook import HookMode

        torch, (tags, mask, bounds) = self.torch, layout
        outs, staged = [], []
        self.hook.activate(mode=HookMode(mode), block_index=block, **policy)
        for layer, (q, k, v) in zip(LAYERS, data):
            outs.append(self.hook(
                attention=_Attn(), layer_name=layer, query=q, key=k, value=v,
                token_tags=torch.tensor(tags, device=self.dev), commit_mask=torch.tensor(mask, device=self.dev),
                cu_seqlens=None, cu_seqlens_host=tuple(bounds), max_seqlen=len(tags), live_documents_hint=hint))
            view = self.cache.staged_view(layer)
            if view is not None:
                order = self.cache._staged.order
                index = torch.tensor(sorted(range(len(order)), key=order.__getitem__), device=self.dev)
                staged.append(view.slot.token_major(len(order), order=index))
        self.hook.deactivate()
        return outs, staged


def _replaced(torch, data, rows, staged):
    """The same inputs with the staged rows' K/V as the 8-bit cache holds them."""
    out = []
    for (q, k, v), (sk, sv) in zip(data, staged):
        k, v = k.clone(), v.clone()
        k[rows], v[rows] = sk, sv
        out.append((q, k, v))
    return out


def _same(torch, a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("backend", ["sdpa", "sage_attn"])
@pytest.mark.parametrize("storage", FORMATS)
def test_noisy_steps_commits_retention_and_rollback(torch_mod, dev, storage, backend):
    """With condition rows: bit for bit the steps over a bf16 cache of the same values."""
    torch = torch_mod
    low, plain = _Run(torch, dev, storage, backend), _Run(torch, dev, "bf16", backend)
    layout = ost.packed_layout(37, 20, 14, 90)
    rows, seed = torch.tensor(layout[1], device=dev), 100

    def commit(block):
        nonlocal seed
        seed += 20
        data = [_data(dev, len(layout[0]), seed + 7 * i) for i in range(2)]
        for run in (low, plain):
            run.cache.begin_clean_commit(block)
        outs, staged = low.step("clean_commit", block, data, layout)
        again, _ = plain.step("clean_commit", block, _replaced(torch, data, rows, staged), layout)
        assert _same(torch, outs, again)

    for block in range(4):
        seed += 20
        data = [_data(dev, len(layout[0]), seed + 7 * i) for i in range(2)]
        assert _same(torch, low.step("noisy", block, data, layout)[0], plain.step("noisy", block, data, layout)[0])
        commit(block)
        for run in (low, plain):
            run.cache.rollback()
        commit(block)
        for run in (low, plain):
            run.cache.commit()
            run.cache.retain_sink_and_recent_commits(2)
        for layer in LAYERS:
            a, b = low.cache.history(layer), plain.cache.history(layer)
            assert torch.equal(a.key, b.key) and torch.equal(a.value, b.value)
    assert low.cache.commit_token_tags == plain.cache.commit_token_tags
    assert 0.5 <= low.cache.slot_bytes / plain.cache.slot_bytes < 0.52


@pytest.mark.parametrize("backend", ["sdpa", "sage_attn"])
@pytest.mark.parametrize("storage", FORMATS)
def test_fused_progress_denoise(torch_mod, dev, storage, backend):
    """Fused steps (staged previous media, recent and sink prefixes, the sink cut to its video rows), with condition
    rows in both documents: bit for bit those over a bf16 cache of the same values."""
    torch = torch_mod
    low, plain = _Run(torch, dev, storage, backend), _Run(torch, dev, "bf16", backend)
    (tags1, mask1, b1), (tags2, mask2, b2) = ost.packed_layout(9, 0, 6, 40, align=8), ost.packed_layout(5, 0, 8, 48, align=8)
    tags, mask = np.concatenate([tags1, tags2]), np.concatenate([mask1, mask2])
    layout = (tags, mask, (*b1, *(len(tags1) + b for b in b2[1:])))
    previous = torch.tensor(np.concatenate([mask1, np.zeros_like(mask2)]), device=dev)
    seed = 500
    for block in range(4):
        for recent, sink in ((2, True), (3, True), (1, True), (2, False), (None, None)):
            policy = {"fused_current_use_sink": sink, "fused_current_recent_blocks": recent}
            policy = {} if recent is None else policy
            seed += 20
            data = [_data(dev, len(tags), seed + 7 * i) for i in range(2)]
            for run in (low, plain):
                run.cache.begin_clean_commit(block)
            outs, staged = low.step("fused_progress_denoise", block, data, layout, hint=(0, 2), **policy)
            data = _replaced(torch, data, previous, staged)
            again, _ = plain.step("fused_progress_denoise", block, data, layout, hint=(0, 2), **policy)
            assert _same(torch, outs, again), (block, policy)
            for run in (low, plain):
                run.cache.rollback()
        seed += 20
        data = [_data(dev, len(tags), seed + 7 * i) for i in range(2)]
        policy = {"fused_current_use_sink": True, "fused_current_recent_blocks": 2}
        for run in (low, plain):
            run.cache.begin_clean_commit(block)
        outs, staged = low.step("fused_progress_denoise", block, data, layout, **policy)
        again, _ = plain.step("fused_progress_denoise", block, _replaced(torch, data, previous, staged), layout, **policy)
        assert _same(torch, outs, again)
        for run in (low, plain):
            run.cache.commit()
            run.cache.retain_sink_and_recent_commits(2)


@pytest.mark.parametrize("storage", FORMATS)
def test_commit_without_condition_rows(torch_mod, dev, storage):
    """Every segment is an 8-bit one: the codes are read in place, within the kernels' bound of fp64 (each row's result
    and its weights rounded to bf16: below 2^-7 of the row in the 2-norm)."""
    torch = torch_mod
    low = _Run(torch, dev, storage, "sdpa")
    layout = ost.packed_layout(0, 0, 150, 250, align=8)
    assert bool(layout[1].all())
    for block in range(3):
        data = [_data(dev, 400, 900 + 20 * block + 7 * i) for i in range(2)]
        low.cache.begin_clean_commit(block)
        past = [low.cache.history(layer) for layer in LAYERS]
        outs, staged = low.step("clean_commit", block, data, layout)
        low.cache.commit()
        for (q, k, v), out, hist, (sk, sv) in zip(data, outs, past, staged):
            keys = sk if hist is None else torch.cat([hist.key, sk])
            values = sv if hist is None else torch.cat([hist.value, sv])
            q, keys, values, out = (bf16.from_torch(t).astype(np.float64) for t in (q, keys, values, out))
            want = lowbit.attention(q, keys, values, D ** -0.5)
            err = np.linalg.norm(out - want, axis=-1) / np.linalg.norm(want, axis=-1)
            assert err.max() <= 2.0 ** -7, err.max()
