"""Every key of a long call by its name: queries of zero weigh all keys alike (or by distance alone), and each key's value stands in a feature of its own,
one call for as many keys as there are features. A key that is left out, counted twice or taken for another shows, wherever chunks, ranges, tiles, pages
or windows meet."""

import ctypes

import pytest
import torch

from test_gpu_text_stage import BF16, F16, _i32, _paged_problem, _randn
from text_stage import HALF_STEP
from vllm_omni_amd import _lib, kernels

pytestmark = pytest.mark.gpu


def _names(n, Hkv, D):
    """For each call: its first key and the (key, head, feature) of all that it names."""
    for first in range(0, n, Hkv * D):
        at = torch.arange(min(Hkv * D, n - first), device="cuda:0")
        yield first, first + at, at // D, at % D


def _close(o, want, tol):
    off = (o.double() - want).abs()
    bad = ~(off <= tol)
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:4].tolist())


# ------------------------------------------------------------------------------------------------ one token
@pytest.mark.parametrize("lengths,page", [([5000], 16), ([5000, 1, 130, 0, 2500], 16), ([4097, 3000, 257], 7), ([300] * 70 + [1500], 16), ([256, 257, 128, 129], 1)],
                         ids=["5000", "5000-1-130-0-2500", "4097-3000-257", "71", "256"])
@pytest.mark.parametrize("window", [None, 1000, 37])
@pytest.mark.parametrize("H,Hkv,D,dtype", [(8, 4, 128, BF16), (20, 1, 64, F16)])
def test_paged_keys(gpu, lengths, page, window, H, Hkv, D, dtype):
    """Joined by the last workgroup and, in a graph, by a second launch."""
    (q, kc, vc, table, n), _ = _paged_problem(1, lengths, page, H, Hkv, D, dtype)
    q.zero_()
    most = max(lengths)
    own = torch.cat([torch.arange(m, device="cuda:0") for m in lengths])  # each stored key's number in its sequence
    of = torch.cat([torch.full((m,), b, device="cuda:0") for b, m in enumerate(lengths)])
    page_of, row_of = table[of, own // page].long(), own % page
    counted = torch.minimum(n, torch.full_like(n, window or most)).double()
    vc[page_of, row_of] = 0.0
    call = lambda: kernels.attn_paged(q, kc, vc, table, n, 0.125, window=window)  # noqa: E731
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        joined = call()
    for first, key, head, feature in _names(most, Hkv, D):
        here = (own >= first) & (own < first + len(key))
        at = (own[here] - first)
        vc[page_of[here], row_of[here], at // D, at % D] = 1024.0
        seen = (key[None] < n[:, None]) & (key[None] >= n[:, None] - (window or most))
        want = torch.zeros(len(lengths), Hkv, D, dtype=torch.float64, device="cuda:0")
        want[:, head, feature] = torch.where(seen, 1024.0 / counted.clamp_min(1.0)[:, None], 0.0)
        want = want.repeat_interleave(H // Hkv, dim=1)
        o = call()
        graph.replay()
        _close(o, want, want * HALF_STEP[dtype] * 1.01)
        assert torch.equal(o, joined)
        vc[page_of[here], row_of[here]] = 0.0


# ------------------------------------------------------------------------------------------------ whole prompts
def _chunks_bytes(Sq, Sk, H, D, **rules):
    return _lib.load().odit_attn_ruled_workspace_bytes(1, Sq, Sk, H, D, ctypes.byref(_lib.AttnRules(**rules)))


def _seen(Sq, Sk, causal=False, window=None, prefix=None, starts=None):
    """[Sq,Sk] on the GPU; `starts`: of queries and keys."""
    i, j = torch.arange(Sq, device="cuda:0")[:, None], torch.arange(Sk, device="cuda:0")[None]
    seen = torch.zeros(Sq, Sk, dtype=torch.bool, device="cuda:0")
    qs, ks = starts or ([0, Sq], [0, Sk])
    for n in range(len(qs) - 1):
        rows, keys = (i >= qs[n]) & (i < qs[n + 1]), (j >= ks[n]) & (j < ks[n + 1])
        away = (j - ks[n + 1]) - (i - qs[n + 1])
        see = torch.ones_like(seen)
        if causal:
            see &= away <= 0
        if window:
            see &= away.abs() < window
        if prefix:
            see |= j - ks[n] < prefix[n]
        seen |= rows & keys & see
    return seen


@pytest.mark.parametrize("Sq,Sk,H,Hkv,rules,cut", [
    (1, 8192, 8, 8, {}, True), (100, 8192, 8, 4, dict(causal=True), True), (5, 3001, 4, 4, dict(causal=True), True), (70, 2500, 4, 2, dict(causal=True, window=1900, prefix=[300]), True),
    (60, 2600, 4, 4, dict(starts=([0, 3, 50], [0, 1300, 2590]), causal=True), True), (130, 2100, 2, 2, dict(window=700), True), (1030, 4100, 2, 2, dict(causal=True), True),
    (700, 700, 16, 8, dict(causal=True, window=130), False), (700, 700, 64, 8, dict(causal=True, prefix=[70]), False), (900, 900, 64, 8, {}, False),
    (1000, 1000, 32, 8, dict(starts=([0, 63, 64, 500, 1000],) * 2, window=90), False), (1000, 1000, 64, 8, dict(starts=([0, 63, 64, 500, 1000],) * 2, causal=True), False),
    (1500, 1500, 64, 8, dict(starts=(list(range(0, 1501, 15)),) * 2, prefix=[4] * 100, causal=True), False)], ids=str)
@pytest.mark.parametrize("D,dtype", [(128, BF16), (64, F16)])
def test_prompt_keys(gpu, Sq, Sk, H, Hkv, rules, cut, D, dtype):
    q = torch.zeros(1, Sq, H, D, dtype=dtype, device="cuda:0")
    k, v = _randn(2, 1, Sk, Hkv, D, dtype=dtype), torch.zeros(1, Sk, Hkv, D, dtype=dtype, device="cuda:0")
    starts = rules.get("starts")
    docs = 0 if starts is None else len(starts[0]) - 1
    assert (_chunks_bytes(Sq, Sk, H, D, causal=int(rules.get("causal", False)), window=rules.get("window") or 0, docs=docs) > 0) == cut
    seen = _seen(Sq, Sk, **rules)
    counted = seen.sum(dim=1).clamp_min(1).double()
    kw = dict(causal=rules.get("causal", False), window=rules.get("window"), prefix=_i32(rules.get("prefix")), q_starts=_i32(starts and starts[0]), k_starts=_i32(starts and starts[1]))
    for first, key, head, feature in _names(Sk, Hkv, D):
        v[0, key, head, feature] = 1024.0
        want = torch.zeros(Sq, Hkv, D, dtype=torch.float64, device="cuda:0")
        want[:, head, feature] = seen[:, key] * (1024.0 / counted)[:, None]
        want = want.repeat_interleave(H // Hkv, dim=1)
        _close(kernels.attn_ruled(q, k, v, 0.125, **kw)[0], want, want * HALF_STEP[dtype] * 1.01)
        v[0, key] = 0.0


@pytest.mark.parametrize("Sq,Sk,causal,window,H", [(6200, 6200, True, None, 4), (6144, 6144, False, None, 4), (1030, 9000, True, None, 2), (1030, 6145, False, None, 2),
                                                   (6300, 6300, True, 3000, 4), (300, 2000, True, None, 4)])
@pytest.mark.parametrize("cap", [0.0, 5.0])
@pytest.mark.parametrize("D", [64, 128])
def test_prompt_keys_by_distance(gpu, Sq, Sk, causal, window, H, cap, D):
    """Slopes, of which far tiles are left out: a key counts by 2^-(slope away) down to where 32 bits end (values of 2^60 keep that in bf16's range). The
    probability's and the result's rounding, and an exponent of up to 118 in 32 bits (six roundings of 2^-24 of it)."""
    Hkv, slopes = 4 if H == 4 else 2, torch.tensor([0.5, 0.05, 0.02, 0.011][:H], device="cuda:0")
    q = torch.zeros(1, Sq, H, D, dtype=BF16, device="cuda:0")
    k, v = _randn(3, 1, Sk, Hkv, D), torch.zeros(1, Sk, Hkv, D, dtype=BF16, device="cuda:0")
    away = torch.arange(Sk, device="cuda:0")[None] - (torch.arange(Sq, device="cuda:0")[:, None] + Sk - Sq)
    seen = _seen(Sq, Sk, causal, window)
    weights = [torch.where(seen, torch.exp(-float(s) * away.abs().double()), 0.0) for s in slopes]
    weights = [w / w.sum(dim=1, keepdim=True) for w in weights]
    for first, key, _, _ in _names(Sk, 1, D):
        if D == 64 and first // D % 2:
            continue  # (every other tile of 64 is enough there)
        v[0, key, :, key - first] = 2.0 ** 60
        o = kernels.attn_ruled(q, k, v, 0.125, causal=causal, window=window, slopes=slopes, cap=cap)[0]
        for h in range(H):
            want = torch.zeros(Sq, D, dtype=torch.float64, device="cuda:0")
            want[:, key - first] = weights[h][:, key] * 2.0 ** 60
            _close(o[:, h], want, want * (2.02 * HALF_STEP[BF16] + 6.0 * 118.0 * 2.0 ** -24) + 2.0 ** (60 - 118))
        v[0, key] = 0.0
