"""A text stage's operators at the edges of their numbers."""

import ctypes

import pytest
import torch

from test_gpu_text_stage import BF16, F16, _all_tiles, _bias, _paged_problem, _randn, _ruled
from text_stage import attention, seen_keys, within
from vllm_omni_amd import _lib, kernels

pytestmark = pytest.mark.gpu

LEAST = torch.finfo(torch.float32).min


# ------------------------------------------------------------------------------------------------ biases and scores of any size
@pytest.mark.parametrize("scale", [1.0, 0.125, 128.0 ** -0.5])
@pytest.mark.parametrize("entry", [-1e9, -1e10, -1e30, LEAST, -float("inf")])
@pytest.mark.parametrize("ahead", [True, False])
@pytest.mark.parametrize("cap,D,dtype", [(0.0, 64, F16), (0.0, 128, BF16), (5.0, 64, BF16)])
def test_distances_that_finite_biases_forbid(gpu, scale, entry, ahead, cap, D, dtype):
    """Keys on one side of the query have a bias so low that they weigh nothing beside the others: as if they were not seen."""
    S, r = 300, 5
    q, k, v = _randn(1, 1, S, 2, D, dtype=dtype), _randn(2, 1, S, 1, D, dtype=dtype), _randn(3, 1, S, 1, D, dtype=dtype)
    distance = torch.zeros(2, 2 * r + 1, device="cuda:0")
    distance[:, r + 1:] = entry
    if not ahead:
        distance = distance.flip(1).contiguous()
    away = torch.arange(S)[None] - torch.arange(S)[:, None]
    want, tol = attention(q[0], k[0], v[0], scale, away <= 0 if ahead else away >= 0, away, cap)
    for o in _ruled(q, k, v, scale, {}, dict(distance=distance), cap):
        within(o[0], want, tol)


@pytest.mark.parametrize("scale", [1.0, 0.125])
@pytest.mark.parametrize("cap", [0.0, 5.0])
@pytest.mark.parametrize("D,dtype", [(64, F16), (128, BF16)])
def test_queries_left_with_the_least_bias(gpu, scale, cap, D, dtype):
    """All keys of a query have the least float32 as bias, beside which a score is nothing: the keys' average. Few rows' keys are cut into ranges."""
    for S, Sk in ((150, 150), (3, 3000)):
        q, k, v = _randn(4, 1, S, 2, D, dtype=dtype), _randn(5, 1, Sk, 1, D, dtype=dtype), _randn(6, 1, Sk, 1, D, dtype=dtype)
        for entry in (LEAST, -1e30):
            bias = dict(distance=torch.full((2, 7), entry, device="cuda:0"))
            seen, away = seen_keys(S, Sk, causal=True)
            want, tol = attention(torch.zeros_like(q[0]), k[0], v[0], scale, seen, away)
            for o in _ruled(q, k, v, scale, dict(causal=True), bias, cap):
                within(o[0], want, tol)


@pytest.mark.parametrize("scale", [1.0, 0.1, 1e-9])
@pytest.mark.parametrize("cap", [0.0, 5.0])
@pytest.mark.parametrize("causal", [True, False])
def test_slopes_of_any_size(gpu, scale, cap, causal):
    """So steep that a query is left with its own key."""
    q, k, v = _randn(7, 1, 200, 2, 64), _randn(8, 1, 200, 2, 64), _randn(9, 1, 200, 2, 64)
    for steep in (1e6, 1e20, 1e35, -LEAST):
        for o in _ruled(q, k, v, scale, dict(causal=causal), dict(slopes=torch.tensor([steep, 1e6], device="cuda:0")), cap):
            assert torch.equal(o, v), steep


def _large_scores(seed, rows, n, D, size):
    """Queries and keys whose products are of this size, exact in 32 bits and far apart or equal; the weights are those of the largest of those seen."""
    q = torch.full((rows, 1, D), 1.0, dtype=BF16, device="cuda:0")
    rank = torch.randperm(n, generator=torch.Generator().manual_seed(seed)) - n // 2
    k = (rank.double() * size).view(n, 1, 1).expand(n, 1, D).to(BF16).contiguous().to("cuda:0")
    return q, k


@pytest.mark.parametrize("size", [1.0, 2.0 ** 20, 2.0 ** 40, 2.0 ** 60, 2.0 ** 100])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("rows,n,rules", [(200, 200, dict(causal=True)), (70, 300, dict(window=90)), (2, 3000, {})], ids=str)
def test_scores_of_any_size(gpu, size, D, rows, n, rules):
    q, k = _large_scores(10, rows, n, D, size)
    v = _randn(11, n, 1, D)
    seen, away = seen_keys(rows, n, **rules)
    s = (k[:, 0].double().cpu() @ q[0, 0].double().cpu()) * 0.25
    p = torch.softmax(s[None].masked_fill(~seen, -float("inf")), dim=1)
    want = p @ v[:, 0].double().cpu()
    tol = 2.0 ** -8 * 2.04 * (p @ v[:, 0].double().cpu().abs()) + 1e-30  # (a probability's rounding and the result's; scores are exact)
    for o in _ruled(q[None], k[None], v[None], 0.25, rules, {}, 0.0):
        within(o[0, :, 0], want, tol)


def _single_and_joined(*args, **kw):
    """The result of a call, and of one in a captured graph, whose chunks a second launch joins: the same bits."""
    o = kernels.attn_paged(*args, **kw)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        other = kernels.attn_paged(*args, **kw)
    graph.replay()
    assert torch.equal(o.nan_to_num(7.0), other.nan_to_num(7.0))
    return o


@pytest.mark.parametrize("kind", ["least", "steep"])
@pytest.mark.parametrize("cap", [0.0, 5.0])
@pytest.mark.parametrize("D,dtype", [(64, F16), (128, BF16)])
def test_decode_biases_of_any_size(gpu, kind, cap, D, dtype):
    """The least float32 at all keys leaves their average, the steepest slopes the last key; also where the keys are cut into chunks."""
    lengths = [1, 40, 300, 3000]
    (q, kc, vc, table, n), rows = _paged_problem(20, lengths, 16, 4, 2, D, dtype)
    for size in (-LEAST, 1e30, 1e10) if kind == "steep" else (LEAST, -1e30):
        bias = dict(slopes=torch.full((4,), size, device="cuda:0")) if kind == "steep" else dict(distance=torch.full((4, 7), size, device="cuda:0"))
        o = _single_and_joined(q, kc, vc, table, n, 0.125, cap=cap, **bias)
        for b, (k, v) in enumerate(rows):
            if kind == "steep":
                assert torch.equal(o[b].cpu(), v[-1].repeat_interleave(2, dim=0))
            else:
                seen, away = seen_keys(1, len(k), causal=True)
                want, tol = attention(torch.zeros_like(q[b:b + 1]), k, v, 0.125, seen, away)
                within(o[b:b + 1], want, tol)


@pytest.mark.parametrize("size", [1.0, 2.0 ** 20, 2.0 ** 40, 2.0 ** 60, 2.0 ** 100])
@pytest.mark.parametrize("n", [100, 3000])
@pytest.mark.parametrize("D", [64, 128])
def test_decode_scores_of_any_size(gpu, size, n, D):
    q, k = _large_scores(12, 1, n, D, size)
    v, page = _randn(13, n, 1, D), 16
    pages = -(-n // page)
    kc, vc = (torch.cat([t, torch.zeros(pages * page - n, 1, D, dtype=BF16, device="cuda:0")]).view(pages, page, 1, D) for t in (k, v))
    table = torch.arange(pages, dtype=torch.int32, device="cuda:0")[None]
    o = _single_and_joined(q, kc, vc, table, torch.tensor([n], dtype=torch.int32, device="cuda:0"), 0.25)
    p = torch.softmax((k[:, 0].double().cpu() @ q[0, 0].double().cpu()) * 0.25, dim=0)
    within(o[0], (p @ v[:, 0].double().cpu())[None], 2.0 ** -8 * 2.04 * (p @ v[:, 0].double().cpu().abs())[None] + 1e-30)


# ------------------------------------------------------------------------------------------------ values that are not finite
def _class_of(want, v, seen):
    """The definition's result where some values are not finite: the kinds that a row sees decide. want [Sq,H,D] is of the others."""
    Hkv, H = v.shape[1], want.shape[1]
    v = v.double().cpu().repeat_interleave(H // Hkv, dim=1)
    count = lambda what: torch.einsum("ij,jhd->ihd", seen.double(), what.double()) > 0  # noqa: E731
    plus, minus, none = count(v == float("inf")), count(v == -float("inf")), count(v.isnan())
    want = want.clone()
    want[plus] = float("inf")
    want[minus] = -float("inf")
    want[none | (plus & minus)] = float("nan")
    return want


def _same(o, want, tol):
    o = o.double().cpu()
    for kind in (float("inf"), -float("inf")):
        assert torch.equal(o == kind, want == kind)
    assert torch.equal(o.isnan(), want.isnan())
    finite = want.isfinite()
    within(o[finite], want[finite], tol[finite])


@pytest.mark.parametrize("rules", [
    dict(causal=True), dict(window=40), dict(causal=True, window=70, prefix=[9]), dict(causal=True, q_starts=[0, 31, 32, 150, 200], k_starts=[0, 31, 32, 150, 200]),
    dict(q_starts=[3, 60, 190], k_starts=[0, 57, 260], prefix=[2, 100], window=20)], ids=str)
@pytest.mark.parametrize("cap,kind", [(0.0, ""), (3.0, ""), (0.0, "slopes"), (2.0, "table"), (0.0, "table")])
@pytest.mark.parametrize("D,dtype", [(64, F16), (128, BF16)])
def test_values_that_are_not_finite(gpu, rules, cap, kind, D, dtype):
    """Each row and feature gets what the values it sees make of it: infinities of one sign, NaN of both, and nothing of those that it does not see."""
    Sq, Sk = 200, 260 if "q_starts" in rules and rules["k_starts"][-1] == 260 else 200
    q, k, v = _randn(30, 1, Sq, 2, D, dtype=dtype, std=0.5), _randn(31, 1, Sk, 1, D, dtype=dtype, std=0.5), _randn(32, 1, Sk, 1, D, dtype=dtype)
    seen, away = seen_keys(Sq, Sk, **rules)
    bias = dict(slopes=torch.tensor([0.01, 0.001], device="cuda:0")) if kind == "slopes" else _bias(kind, 2, 33)
    want, tol = attention(q[0], k[0], v[0], 0.1, seen, away, cap, **bias)
    for j, d, what in ((0, 0, "inf"), (5, 1, "nan"), (33, 1, "-inf"), (40, 2, "inf"), (90, 2, "-inf"), (64, D - 1, "nan"), (127, 3, "inf"), (128, 3, "inf"),
                       (Sk - 1, 4, "-inf"), (150, slice(None), "nan"), (170, slice(8, 40), "inf")):
        v[0, j, 0, d] = float(what)
    clean = v.masked_fill(~v.isfinite(), 0.0)
    want, tol = attention(q[0], k[0], clean[0], 0.1, seen, away, cap, **bias)
    want = _class_of(want, v[0], seen)
    for o in _ruled(q, k, v, 0.1, rules, bias, cap):
        _same(o[0], want, tol)


@pytest.mark.parametrize("Sq,Sk", [(3, 3000), (130, 2100)])
@pytest.mark.parametrize("D,dtype", [(64, F16), (128, BF16)])
def test_values_that_are_not_finite_in_cut_keys(gpu, Sq, Sk, D, dtype):
    q, k, v = _randn(34, 1, Sq, 2, D, dtype=dtype, std=0.5), _randn(35, 1, Sk, 1, D, dtype=dtype, std=0.5), _randn(36, 1, Sk, 1, D, dtype=dtype)
    for j, d, what in ((0, 0, "inf"), (700, 1, "nan"), (Sk - 1, 2, "inf"), (Sk - 2, 3, "nan"), (Sk - 3, 0, "-inf"), (1000, 4, "-inf")):
        v[0, j, 0, d] = float(what)
    seen, away = seen_keys(Sq, Sk, causal=True)
    want, tol = attention(q[0], k[0], v[0].masked_fill(~v[0].isfinite(), 0.0), 0.1, seen, away)
    want = _class_of(want, v[0], seen)
    for o in _ruled(q, k, v, 0.1, dict(causal=True), {}, 0.0):
        _same(o[0], want, tol)


@pytest.mark.parametrize("Sq,Sk,causal", [(6200, 6200, True), (6144, 6144, False), (1030, 6145, True), (100, 300, True)])
@pytest.mark.parametrize("D,dtype,H,Hkv", [(128, BF16, 8, 4), (64, F16, 40, 40)])
def test_keys_that_are_no_numbers_reach_rows_behind_slopes_and_a_cap(gpu, Sq, Sk, causal, D, dtype, H, Hkv):
    """However far they are; a key with infinities counts by the cap. The call without scratch visits all tiles."""
    q, k, v = _randn(40, 1, Sq, H, D, dtype=dtype), _randn(41, 1, Sk, Hkv, D, dtype=dtype), _randn(42, 1, Sk, Hkv, D, dtype=dtype)
    slopes = torch.tensor([4.0 * 2.0 ** (-12.0 * h / H) for h in range(H)], device="cuda:0")
    group, clean = H // Hkv, kernels.attn_ruled(q, k, v, D ** -0.5, causal=causal, slopes=slopes, cap=5.0)
    # (keys that are cut into ranges are summed in another order than those of a call without scratch)
    whole = _lib.load().odit_attn_ruled_workspace_bytes(1, Sq, Sk, H, D, ctypes.byref(_lib.AttnRules(causal=int(causal), cap=5.0))) == 0
    for what in (float("nan"), float("inf"), 1e30 if dtype == BF16 else 60000.0):
        bad = k.clone()
        bad[0, 3, 0, :7] = what
        o = kernels.attn_ruled(q, bad, v, D ** -0.5, causal=causal, slopes=slopes, cap=5.0)
        full = _all_tiles(q, bad, v, D ** -0.5, causal, None, 5.0, slopes)
        assert torch.equal(o.isnan(), full.isnan())
        assert torch.equal(o[:, :, group:], clean[:, :, group:])
        sees = torch.arange(Sq, device="cuda:0") + Sk - Sq >= (3 if causal else 0)
        if what != what:
            assert o[0, sees, :group].isnan().all() and not o[0, ~sees].isnan().any()
        if causal and whole:
            assert torch.equal(o.nan_to_num(77.0), full.nan_to_num(77.0))
    q[0, 70, 0, 0] = float("nan")  # (and a query that is none spoils its own row)
    o = kernels.attn_ruled(q, k, v, D ** -0.5, causal=causal, slopes=slopes, cap=5.0)
    assert o[0, 70, 0].isnan().all()
    o[0, 70, 0] = clean[0, 70, 0]
    if causal and whole:
        assert torch.equal(o, clean)
    else:
        assert o.isfinite().all()


def _us(call):
    call()
    torch.cuda.synchronize()
    a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    a.record()
    call()
    b.record()
    torch.cuda.synchronize()
    return a.elapsed_time(b) * 1e3


@pytest.mark.parametrize("S,H,Hkv,D,dtype", [(2048, 4, 2, 128, BF16), (4096, 16, 4, 128, BF16), (4096, 16, 4, 64, F16)])
def test_an_overflow_that_all_rows_see(gpu, S, H, Hkv, D, dtype):
    """One infinite value at the head of a long prompt, and a feature that has overflowed at every key: right, and not far more work than a call is
    anyhow (rows that see them are done again by wavefronts, if at all; the allowance is 20 times and a millisecond)."""
    q, k, v = _randn(37, 1, S, H, D, dtype=dtype), _randn(38, 1, S, Hkv, D, dtype=dtype), _randn(39, 1, S, Hkv, D, dtype=dtype)
    call = lambda: kernels.attn_ruled(q, k, v, 0.1, causal=True)  # noqa: E731
    plain, time = call(), _us(call)
    one, v = v, v.clone()
    v[0, 3, 0, 5] = float("inf")
    o = call()
    group = H // Hkv
    assert (o[0, 3:, :group, 5] == float("inf")).all()
    o[0, 3:, :group, 5] = plain[0, 3:, :group, 5]
    assert torch.equal(o[:, 64:], plain[:, 64:]) and torch.equal(o[:, :, group:], plain[:, :, group:])
    seen, away = seen_keys(64, 64, causal=True)
    want, tol = attention(q[0, :64], k[0, :64], one[0, :64], 0.1, seen, away)
    within(o[0, :64], want, tol)
    assert _us(call) < 20 * time + 1000
    v = one.clone()
    v[..., 5] = float("inf")
    o = call()
    assert (o[..., 5] == float("inf")).all()
    rows = torch.tensor([0, 1, 31, 32, 63, 64, 1000, S - 1])
    away = torch.arange(S)[None] - rows[:, None]
    want, tol = attention(q[0, rows], k[0], one[0], 0.1, away <= 0, away)
    keep = torch.arange(D) != 5
    within(o[0, rows][..., keep.to("cuda:0")], want[..., keep], tol[..., keep])
    assert _us(call) < 20 * time + 1000


# ------------------------------------------------------------------------------------------------ caps
def _pairs(seed, n, D, step):
    """Queries and pairs of keys whose products are exact in 32 bits, the two of a pair's up to 4 `step` apart."""
    g = torch.Generator().manual_seed(seed)
    q = torch.randint(-4, 5, (n, 1, D), generator=g).float()
    k = torch.randint(-2, 3, (n, 1, D), generator=g).float() + q.sign() * torch.randint(0, 2, (n, 1, 1), generator=g)
    other = k.clone()
    other[:, :, 0] += step * torch.randint(-1, 2, (n, 1), generator=g)
    return q.half(), torch.stack([k, other], dim=1).half()


def _capped_pair(q, k, scale, cap, bias):
    """(o, tolerance) of values 1 and -1. The larger probability is 1; the other one's rounding (below 1: 2^-12) and the result's (below 1/2, 2^-13, or
    below 1, 2^-12) are halved by the sum; a score's own error is 2^-21 of it, and six roundings of what is added in 32 bits."""
    s = (q.double()[:, None] * k.double()).sum(dim=-1)[..., 0] * scale
    s = cap * torch.tanh(s / cap) + bias
    p = torch.softmax(s, dim=1)
    o = p[:, 0] - p[:, 1]
    assert (p.min(dim=1).values > 0.05).all()
    return o, 2.0 ** -13 + 2.0 ** -12 * o.abs().clamp_min(0.5) + 2.0 ** -21 * s.abs().amax(dim=1) + 6.0 * 2.0 ** -24 * s.abs().amax(dim=1)


@pytest.mark.parametrize("kind", ["", "slopes", "table"])
@pytest.mark.parametrize("cap", [30.0, 512.0, 513.0, 1000.0, 3000.0, 8192.0])
@pytest.mark.parametrize("scale,step", [(0.125, 1.0), (4.0, 2.0 ** -5)])  # scores of tens, and up to a thousand
@pytest.mark.parametrize("D", [64, 128])
def test_scores_keep_their_digits_under_any_cap(gpu, cap, kind, scale, step, D):
    """In fp16, whose probabilities tell scores apart that differ by 2^-11: whole prompts of two keys, and sequences of two."""
    n = 3000
    q, k = (t.to("cuda:0") for t in _pairs(50, n, D, step))
    v = torch.ones_like(k)
    v[:, 1] = -1.0
    slope = 0.25
    kw = dict(slopes=torch.full((1,), slope, device="cuda:0")) if kind == "slopes" else dict(distance=torch.full((1, 3), -slope, device="cuda:0")) if kind == "table" else {}
    # away: the query stands at the second key
    bias = torch.tensor([-slope, 0.0] if kind == "slopes" else [-slope, -slope] if kind else [0.0, 0.0], dtype=torch.float64)
    want, tol = _capped_pair(q.cpu(), k.cpu(), scale, cap, bias)
    if cap <= 512.0:
        tol = tol + 2.0 * cap * 2.0 ** -21 / 2.0  # (both scores' errors, of the cap, of which half is the result's)
    for o in (kernels.attn_ruled(q[:, None], k, v, scale, cap=cap, **kw)[:, 0],
              kernels.attn_ruled(q[:, None].expand(n, 70, 1, D), k, v, scale, cap=cap, **kw)[:, -1],
              kernels.attn_paged(q, k, v, torch.arange(n, dtype=torch.int32, device="cuda:0")[:, None], torch.full((n,), 2, dtype=torch.int32, device="cuda:0"),
                                 scale, cap=cap, **kw)):
        assert (o == o[..., :1]).all()
        within(o[:, 0, 0], want, tol)


# ------------------------------------------------------------------------------------------------ derivatives
def test_tangents_are_refused(gpu):
    """Forward-mode derivatives, like gradients: not dropped without a word. Inference mode is for calls that want none."""
    q, kv, slopes = _randn(60, 1, 8, 4, 64), _randn(61, 1, 8, 2, 64), torch.ones(4, device="cuda:0")
    table, lengths, at = (torch.zeros(8, 1, dtype=torch.int32, device="cuda:0"), torch.full((8,), 3, dtype=torch.int32, device="cuda:0"), torch.arange(8, device="cuda:0"))
    turns = torch.rand(32, dtype=torch.float64, device="cuda:0")
    calls = {"attn_ruled": (lambda q, kv, s: kernels.attn_ruled(q, kv, kv, 0.1, slopes=s)),
             "attn_paged": (lambda q, kv, s: kernels.attn_paged(q[0], kv, kv, table, lengths, 0.1, slopes=s)),
             "rope_append": (lambda q, kv, s: kernels.rope_append(q[0], kv[0], None, at, turns * s[0]))}
    dual = torch.autograd.forward_ad
    for name, call in calls.items():
        call(q, kv, slopes)
        with dual.dual_level():
            call(q, kv, slopes)
            for i, t in enumerate((q, kv, slopes)):
                args = [q, kv, slopes]
                args[i] = dual.make_dual(t, torch.ones_like(t))
                for grad in (True, False):
                    with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match=name):
                        call(*args)
                with torch.inference_mode():
                    call(*args)
