"""A text stage's operators (``rope_append``, ``attn_ruled``, ``attn_paged``) against their definitions in 64 bits."""

import ctypes
import itertools
import threading

import pytest
import torch

from text_stage import attention, rotated, seen_keys, within
from vllm_omni_amd import _lib, kernels

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


def _randn(seed, *shape, dtype=BF16, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * std).to(dtype).to("cuda:0")


def _i32(values):
    return None if values is None else torch.tensor(values, dtype=torch.int32, device="cuda:0")


def _bias(kind, H, seed, radius=5):
    if kind == "slopes":
        return dict(slopes=torch.tensor([2.0 ** -(1 + h % 8) for h in range(H)], device="cuda:0"))
    if kind == "table":
        return dict(distance=_randn(seed, H, 2 * radius + 1, dtype=torch.float32))
    return {}


def _check_ruled(q, k, v, os, scale, rules, bias, cap):
    seen, away = seen_keys(q.shape[1], k.shape[1], **rules)
    for b in range(q.shape[0]):
        want, tol = attention(q[b], k[b], v[b], scale, seen, away, cap, **bias)
        for o in os:
            within(o[b], want, tol)


def _ruled(q, k, v, scale, rules, bias, cap):
    """The results of the call as it is and of one with 300 times the batch rows, whose workgroups are cut otherwise; all copies' bits are one's."""
    r = dict(rules)
    for name in ("q_starts", "k_starts", "prefix"):
        r[name] = _i32(r.get(name))
    o = kernels.attn_ruled(q, k, v, scale, cap=cap, **r, **bias)
    B, n = q.shape[0], 300
    if r["prefix"] is not None and r["q_starts"] is None:
        r["prefix"] = r["prefix"].repeat(n)
    many = kernels.attn_ruled(*(t[None].expand(n, *t.shape).flatten(0, 1) if B > 1 else t.expand(n, *t.shape[1:]) for t in (q, k, v)), scale, cap=cap, **r, **bias)
    many = many.view(n, *o.shape)
    assert torch.equal(many[1:].nan_to_num(7.0), many[:1].nan_to_num(7.0).expand_as(many[1:]))
    return o, many[0]


# ------------------------------------------------------------------------------------------------ whole prompts
@pytest.mark.parametrize("Sq,Sk", [(1, 1), (1, 200), (63, 64), (65, 65), (130, 193), (129, 1), (200, 70)])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("D,dtype", [(64, F16), (128, BF16)])
def test_prompt_lengths(gpu, Sq, Sk, causal, D, dtype):
    q, k, v = _randn(1, 1, Sq, 2, D, dtype=dtype, std=2), _randn(2, 1, Sk, 1, D, dtype=dtype), _randn(3, 1, Sk, 1, D, dtype=dtype)
    rules = dict(causal=causal)
    _check_ruled(q, k, v, _ruled(q, k, v, D ** -0.5, rules, {}, 0.0), D ** -0.5, rules, {}, 0.0)


@pytest.mark.parametrize("rules", [
    dict(window=1), dict(window=7, causal=True), dict(window=70), dict(causal=True, prefix=[3, 200]), dict(causal=True, window=20, prefix=[66, 0]),
    dict(window=10, prefix=[500, -4]), dict(window=1 << 30, causal=True)], ids=str)
@pytest.mark.parametrize("cap,kind", [(0.0, ""), (5.0, "slopes"), (0.0, "table")])
@pytest.mark.parametrize("D,dtype", [(64, BF16), (128, F16)])
def test_prompt_rules(gpu, rules, cap, kind, D, dtype):
    q, k, v = _randn(4, 2, 150, 4, D, dtype=dtype, std=2), _randn(5, 2, 190, 2, D, dtype=dtype), _randn(6, 2, 190, 2, D, dtype=dtype)
    bias = _bias(kind, 4, 7)
    os = _ruled(q, k, v, 0.1, rules, bias, cap)
    for b in range(2):  # (prefixes differ from batch row to batch row)
        own = dict(rules, prefix=[rules["prefix"][b]]) if "prefix" in rules else rules
        _check_ruled(q[b:b + 1], k[b:b + 1], v[b:b + 1], [o[b:b + 1] for o in os], 0.1, own, bias, cap)


@pytest.mark.parametrize("cap,kind", list(itertools.product([0.0, 3.0], ["", "slopes", "table"])))
@pytest.mark.parametrize("q_starts,k_starts", [
    ([0, 40, 40, 41, 170, 300], [0, 40, 40, 41, 170, 300]),    # an empty document, one of one token
    ([0, 1, 2, 3, 130, 131], [0, 100, 100, 101, 160, 300]),    # other lengths of keys; a document without keys; rows behind the last one
    ([5, 60, 150], [10, 200, 250])], ids=str)                  # rows and keys ahead of the first one
@pytest.mark.parametrize("causal,window,prefix", [(False, None, False), (True, None, True), (True, 30, True), (False, 9, False)])
def test_documents(gpu, cap, kind, q_starts, k_starts, causal, window, prefix):
    q, k, v = _randn(8, 1, 300, 2, 64, std=2), _randn(9, 1, 300, 2, 64), _randn(10, 1, 300, 2, 64)
    rules = dict(q_starts=q_starts, k_starts=k_starts, causal=causal, window=window, prefix=[2, 70, 0, 5, 1][:len(q_starts) - 1] if prefix else None)
    bias = _bias(kind, 2, 11)
    os = _ruled(q, k, v, 0.125, rules, bias, cap)
    _check_ruled(q, k, v, os, 0.125, rules, bias, cap)
    assert not any(o[0, q_starts[-1]:].any() or o[0, :q_starts[0]].any() for o in os)


def test_many_documents_and_a_long_gap(gpu):
    """More documents than a wavefront has lanes; a prefix far ahead of the window, so that a workgroup's tiles are two runs."""
    starts = list(range(0, 261, 2))
    q, k, v = _randn(12, 2, 260, 2, 64), _randn(13, 2, 260, 1, 64), _randn(14, 2, 260, 1, 64)
    rules = dict(q_starts=starts, k_starts=starts, causal=True)
    _check_ruled(q, k, v, _ruled(q, k, v, 0.125, rules, {}, 0.0), 0.125, rules, {}, 0.0)
    q, k, v = _randn(15, 1, 40, 1, 128), _randn(16, 1, 1000, 1, 128), _randn(17, 1, 1000, 1, 128)
    for prefix in (1, 64, 130):
        rules = dict(causal=True, window=33, prefix=[prefix])
        _check_ruled(q, k, v, _ruled(q, k, v, 0.1, rules, {}, 0.0), 0.1, rules, {}, 0.0)


@pytest.mark.parametrize("causal,window,cap,kind", [(True, None, 0.0, ""), (True, 1000, 5.0, ""), (True, None, 0.0, "slopes"), (False, 700, 0.0, "table"),
                                                    (False, None, 5.0, "slopes")])
@pytest.mark.parametrize("D,dtype", [(64, BF16), (128, F16)])
def test_long_prompts_at_some_rows(gpu, causal, window, cap, kind, D, dtype):
    S, H, Hkv = 4100, 16, 4  # 33 blocks of 128 queries, the last one of 4
    q, k, v = _randn(90, 1, S, H, D, dtype=dtype, std=2), _randn(91, 1, S, Hkv, D, dtype=dtype), _randn(92, 1, S, Hkv, D, dtype=dtype)
    bias = _bias(kind, H, 93, radius=100)
    o = kernels.attn_ruled(q, k, v, 0.1, causal=causal, window=window, cap=cap, **bias)
    rows = torch.tensor([0, 1, 127, 128, 1700, 2047, 4090, 4099])
    away = torch.arange(S)[None] - rows[:, None]
    seen = (away <= 0 if causal else torch.ones_like(away, dtype=torch.bool)) & (away.abs() < (window or S))
    want, tol = attention(q[0, rows], k[0], v[0], 0.1, seen, away, cap, **bias)
    within(o[0, rows], want, tol)


def _all_tiles(q, k, v, scale, causal, window, cap, slopes, prefix=None):
    """The call without scratch, which visits all tiles that are seen."""
    lib = _lib.load()
    rules = _lib.AttnRules(causal=int(causal), window=window or 0, cap=cap, slopes=slopes.data_ptr(), prefix=None if prefix is None else prefix.data_ptr())
    o = torch.empty_like(q)
    (B, Sq, H, D), (_, Sk, Hkv, _) = q.shape, k.shape
    _lib.check(lib.odit_attn_ruled(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), B, Sq, Sk, H, Hkv, D, *(_lib.i64_array(t.stride()[:3]) for t in (q, k, v, o)), scale,
        ctypes.byref(rules), 0 if q.dtype == BF16 else 1, None, 0, torch.cuda.current_stream().cuda_stream), "odit_attn_ruled")
    return o


@pytest.mark.parametrize("Sq,Sk,causal,window", [(6200, 6200, True, None), (1030, 6145, True, None), (6144, 6144, False, None), (6300, 6300, True, 700)])
@pytest.mark.parametrize("D,dtype,H,Hkv", [(128, BF16, 24, 8), (64, F16, 40, 40)])
def test_slopes_leave_far_tiles_out(gpu, Sq, Sk, causal, window, D, dtype, H, Hkv):
    """What is left out has no weight in 32 bits: the bits of the call that visits all tiles, under a causal order, where both begin at a query's own
    key. (Otherwise the far keys come first, and the running maximum, which may lag by a factor of 2^8, goes another way: other roundings of the
    probabilities, so some rows against the definition.) Also with one long key far away, one that holds NaN, one that holds infinities, slopes of
    zero and below, and a prefix that all see."""
    q, k, v = _randn(100, 1, Sq, H, D, dtype=dtype), _randn(101, 1, Sk, Hkv, D, dtype=dtype), _randn(102, 1, Sk, Hkv, D, dtype=dtype)
    slopes = torch.tensor([4.0 * 2.0 ** (-12.0 * h / H) for h in range(H)], device="cuda:0")
    slopes[5], slopes[7] = 0.0, -0.01
    rows = torch.tensor([0, 600, Sq - 1])
    away = torch.arange(Sk)[None] - (rows[:, None] + Sk - Sq)
    seen = (away <= 0 if causal else torch.ones_like(away, dtype=torch.bool)) & (away.abs() < (window or Sk))
    for what in (None, 30.0, float("nan"), float("inf")):
        if what is not None:
            k[0, 3, 0] = k[0, 3, 0] * what
        for prefix in (None, _i32([70])):
            o = kernels.attn_ruled(q, k, v, D ** -0.5, causal=causal, window=window, slopes=slopes, prefix=prefix)
            full = _all_tiles(q, k, v, D ** -0.5, causal, window, 0.0, slopes, prefix)
            assert torch.equal(o.isnan(), full.isnan())
            if causal:
                assert torch.equal(o.nan_to_num(77.0), full.nan_to_num(77.0)), (what, prefix)
            if what in (None, 30.0) and prefix is None:
                want, tol = attention(q[0, rows], k[0], v[0], D ** -0.5, seen, away, 0.0, slopes=slopes)
                within(o[0, rows], want, tol)
                within(full[0, rows], want, tol)
    k = _randn(101, 1, Sk, Hkv, D, dtype=dtype)
    o = kernels.attn_ruled(q, k, v, D ** -0.5, causal=causal, window=window, slopes=slopes, cap=5.0)  # (a cap is a bound by itself)
    want, tol = attention(q[0, rows], k[0], v[0], D ** -0.5, seen, away, 5.0, slopes=slopes)
    within(o[0, rows], want, tol)


@pytest.mark.parametrize("causal", [True, False])
def test_slopes_over_cut_keys(gpu, causal):
    """Few heads, whose keys are cut into ranges of the tiles that are left; the scratch is for both."""
    Sq, Sk, H, D = 1030, 9000, 2, 64
    need = lambda **rules: _lib.load().odit_attn_ruled_workspace_bytes(1, Sq, Sk, H, D, ctypes.byref(_lib.AttnRules(causal=int(causal), **rules)))  # noqa: E731
    q, k, v = _randn(110, 1, Sq, H, D), _randn(111, 1, Sk, 1, D), _randn(112, 1, Sk, 1, D)
    slopes = torch.tensor([0.5, 0.02], device="cuda:0")
    assert need() > 0 and need(slopes=slopes.data_ptr()) - need() == H * 64 * 4
    o = kernels.attn_ruled(q, k, v, 0.125, causal=causal, slopes=slopes)
    rows = torch.tensor([0, 63, 64, 500, Sq - 1])
    away = torch.arange(Sk)[None] - (rows[:, None] + Sk - Sq)
    want, tol = attention(q[0, rows], k[0], v[0], 0.125, away <= 0 if causal else torch.ones_like(away, dtype=torch.bool), away, 0.0, slopes=slopes)
    within(o[0, rows], want, tol)


@pytest.mark.parametrize("D", [64, 128])
def test_prompt_strides(gpu, D):
    """q, k and v as parts of one projection; keys and values with the head ahead of the row; odd strides, which are copied."""
    qkv = _randn(18, 2, 100, (4 + 2 * 2) * D)
    q, k, v = (t.unflatten(2, (-1, D)) for t in qkv.split((4 * D, 2 * D, 2 * D), dim=2))
    rules = dict(causal=True)
    _check_ruled(q, k, v, _ruled(q, k, v, 0.1, rules, {}, 0.0), 0.1, rules, {}, 0.0)
    k2, v2 = k.transpose(1, 2).contiguous().transpose(1, 2), v.transpose(1, 2).contiguous().transpose(1, 2)
    assert all(map(torch.equal, _ruled(q, k2, v2, 0.1, rules, {}, 0.0), _ruled(q, k, v, 0.1, rules, {}, 0.0)))
    odd = _randn(19, 2, 100, 2, D + 1)[..., 1:]
    assert all(map(torch.equal, _ruled(q, odd, v, 0.1, rules, {}, 0.0), _ruled(q, odd.contiguous(), v, 0.1, rules, {}, 0.0)))
    wide = torch.cat([k, k.roll(1, 3)], dim=3)[..., 24:24 + D]  # (row stride 2 D Hkv, rows that do not start on a multiple of their length)
    _check_ruled(q, wide, v, _ruled(q, wide, v, 0.1, rules, {}, 0.0), 0.1, rules, {}, 0.0)
    one = k[:, :1].expand(2, 100, 2, D)
    _check_ruled(q, one, v, _ruled(q, one, v, 0.1, rules, {}, 0.0), 0.1, rules, {}, 0.0)


@pytest.mark.parametrize("what", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("cap,kind", [(0.0, ""), (4.0, "table"), (0.0, "slopes")])
@pytest.mark.parametrize("D,dtype", [(64, BF16), (128, F16)])
def test_what_is_not_seen_does_not_count(gpu, what, cap, kind, D, dtype):
    """A document of padding that holds NaN or infinities, and such a key behind the other queries of its own document."""
    q, k, v = _randn(20, 1, 200, 2, D, dtype=dtype, std=2), _randn(21, 1, 200, 1, D, dtype=dtype), _randn(22, 1, 200, 1, D, dtype=dtype)
    starts = [0, 90, 150, 200]
    rules, bias = dict(q_starts=starts, k_starts=starts, causal=True, prefix=[4, 5, 0]), _bias(kind, 2, 23)
    clean = _ruled(q, k, v, 0.1, rules, bias, cap)
    for t in (k, v):
        t[0, 90:150] = what  # the second document
        t[0, 199] = what     # the last key of the third: its last query alone sees it
    dirty = _ruled(q, k, v, 0.1, rules, bias, cap)
    keep = list(range(90)) + list(range(150, 199))
    zero = k.clone(), v.clone()
    for t in zero:
        t[0, 90:150] = 0
        t[0, 199] = 0
    seen, away = seen_keys(200, 200, **rules)
    want, tol = attention(q[0], zero[0][0], zero[1][0], 0.1, seen, away, cap, **bias)
    for o in dirty + clean:
        within(o[0][keep], want[keep], tol[keep])
    for o in dirty:
        assert not o[0, 90:150].isfinite().any() and not o[0, 199].isfinite().any()


def test_scores_far_apart(gpu):
    """Scores of thousands in units of log2, rising and falling: the running maximum moves at every tile or never."""
    for sign in (1.0, -1.0):
        q, v = _randn(24, 1, 70, 1, 64), _randn(25, 1, 300, 1, 64)
        q = torch.full_like(q, 1.0)
        k = (torch.arange(300, device="cuda:0").view(1, 300, 1, 1) * sign).expand(1, 300, 1, 64).to(BF16).contiguous()
        for rules in ({}, dict(causal=True), dict(window=40)):
            _check_ruled(q, k, v, _ruled(q, k, v, 0.25, rules, {}, 0.0), 0.25, rules, {}, 0.0)
            _check_ruled(q, k, v, _ruled(q, k, v, 0.25, rules, {}, 20.0), 0.25, rules, {}, 20.0)


def test_biases_that_forbid(gpu):
    """Distances with a bias of minus infinity are not attended to; a query left with nothing gets zeros."""
    q, k, v = _randn(26, 1, 100, 2, 64), _randn(27, 1, 100, 2, 64), _randn(28, 1, 100, 2, 64)
    distance = torch.zeros(2, 7, device="cuda:0")
    distance[0, :2] = -float("inf")     # head 0: away <= -2 is out
    distance[1, :] = -float("inf")      # head 1: everything is
    os = _ruled(q, k, v, 0.1, dict(causal=True), dict(distance=distance), 0.0)
    assert not any(o[:, :, 1].any() for o in os)
    _check_ruled(q[:, :, :1], k[:, :, :1], v[:, :, :1], [o[:, :, :1] for o in os], 0.1, dict(causal=True, window=2), {}, 0.0)


@pytest.mark.parametrize("Sq,Sk,rules", [
    (1, 4000, {}), (5, 3001, dict(causal=True)), (70, 2500, dict(causal=True, window=1900, prefix=[300])), (3, 2000, dict(window=700)),
    (60, 2600, dict(q_starts=[0, 3, 50], k_starts=[0, 1300, 2590], causal=True)), (130, 2100, dict(causal=True, prefix=[2100]))], ids=str)
@pytest.mark.parametrize("cap,kind,D,dtype", [(0.0, "", 128, BF16), (5.0, "", 64, F16), (0.0, "slopes", 64, BF16), (3.0, "table", 128, F16)])
def test_few_rows_of_many_keys(gpu, Sq, Sk, rules, cap, kind, D, dtype):
    """Calls whose keys are cut into ranges that run side by side."""
    q, k, v = _randn(40, 1, Sq, 2, D, dtype=dtype, std=2), _randn(41, 1, Sk, 1, D, dtype=dtype), _randn(42, 1, Sk, 1, D, dtype=dtype)
    bias = _bias(kind, 2, 43, 200)
    _check_ruled(q, k, v, _ruled(q, k, v, 0.1, rules, bias, cap), 0.1, rules, bias, cap)
    if "q_starts" in rules:  # what no query sees spoils no range's sum
        k[0, 2590:], v[0, 2590:], v[0, 1299] = float("nan"), float("inf"), float("nan")
        seen, away = seen_keys(Sq, Sk, **rules)
        keep = [i for i in range(Sq) if i != 2]  # (the first document's last query sees key 1299)
        zeroed = v.nan_to_num(0.0, 0.0, 0.0), k.nan_to_num(0.0)
        want, tol = attention(q[0], zeroed[1][0], zeroed[0][0], 0.1, seen, away, cap, **bias)
        for o in _ruled(q, k, v, 0.1, rules, bias, cap):
            within(o[0][keep], want[keep], tol[keep])
            assert o[0, 2].isnan().all()


@pytest.mark.parametrize("copies", [1, 60])
@pytest.mark.parametrize("D", [64, 128])
def test_bits_repeat(gpu, D, copies):
    """The same call gives the same bits, whatever is in the caches and registers before it."""
    q, k, v = _randn(50, copies, 300, 4, D, std=2), _randn(51, copies, 300, 2, D), _randn(52, copies, 300, 2, D)
    other = torch.empty(1 << 28, dtype=torch.int8, device="cuda:0")
    starts = _i32([5, 60, 150]), _i32([10, 200, 250])
    for kw in (dict(q_starts=starts[0], k_starts=starts[1]), dict(causal=True, window=40), dict(causal=True, cap=5.0), dict(causal=True, **_bias("slopes", 4, 0)),
               dict(q_starts=starts[0], k_starts=starts[1], cap=2.0, **_bias("table", 4, 1))):
        first = kernels.attn_ruled(q, k, v, 0.1, **kw)
        for i in range(10):
            other.fill_(i)
            kernels.attn_ruled(k, q[:, :, :2], q[:, :, 2:], 3.0)  # (large scores left behind)
            assert torch.equal(kernels.attn_ruled(q, k, v, 0.1, **kw), first), kw


def test_prompt_empty(gpu):
    q, k = _randn(29, 2, 5, 2, 64), _randn(30, 2, 0, 2, 64)
    assert not kernels.attn_ruled(q, k, k, 0.1).any()
    assert kernels.attn_ruled(q[:, :0], q, q, 0.1).shape == (2, 0, 2, 64)
    assert kernels.attn_ruled(q[:0], k[:0], k[:0], 0.1).shape == (0, 5, 2, 64)
    nothing = kernels.attn_ruled(q, q, q, 0.1, q_starts=_i32([0, 0]), k_starts=_i32([0, 5]))
    assert not nothing.any()


def test_starts_that_make_no_sense_stay_inside(gpu):
    """Starts outside the tensors or out of order: rows come from somewhere inside the keys, or are zeros."""
    q = _randn(31, 1, 70, 2, 64)
    for starts in ([-5, 400], [60, 10, 300], [0, 1 << 30], [-(1 << 31), (1 << 31) - 1], [3, 3, 2, 1]):
        o = kernels.attn_ruled(q, q, q, 0.1, causal=True, window=9, q_starts=_i32(starts), k_starts=_i32(starts), prefix=_i32([1 << 30] * (len(starts) - 1)))
        assert o.isfinite().all()


# ------------------------------------------------------------------------------------------------ one token
def _paged_problem(seed, lengths, page, H, Hkv, D, dtype, spare=3):
    """Caches whose rows beyond the sequences' hold NaN, pages in no order, and the same keys and values in rows."""
    used = [-(-n // page) for n in lengths]
    pages, most = sum(used) + spare, max(max(used), 1) + 1
    g = torch.Generator().manual_seed(seed)
    order = torch.randperm(pages, generator=g).tolist()
    kc = torch.full((pages, page, Hkv, D), float("nan"), dtype=dtype)
    vc = kc.clone()
    table, rows = torch.full((len(lengths), most), pages + 7, dtype=torch.int32), []
    for b, n in enumerate(lengths):
        k, v = (torch.randn(n, Hkv, D, generator=g).to(dtype) for _ in range(2))
        rows.append((k, v))
        for i in range(used[b]):
            at = order.pop()
            table[b, i] = at
            part = slice(i * page, min(n, (i + 1) * page))
            kc[at, :part.stop - part.start], vc[at, :part.stop - part.start] = k[part], v[part]
    q = (torch.randn(len(lengths), H, D, generator=g) * 2).to(dtype)
    return [t.to("cuda:0") for t in (q, kc, vc, table, torch.tensor(lengths, dtype=torch.int32))], rows


def _check_paged(q, rows, o, scale, window, cap, bias):
    for b, (k, v) in enumerate(rows):
        n = k.shape[0]
        if n == 0:
            assert not o[b].any()
            continue
        seen, away = seen_keys(1, n, causal=True, window=window)
        want, tol = attention(q[b:b + 1], k, v, scale, seen, away, cap, **bias)
        within(o[b:b + 1], want, tol)


@pytest.mark.parametrize("page", [1, 7, 16, 64])
@pytest.mark.parametrize("H,Hkv,D,dtype", [(8, 2, 128, BF16), (3, 3, 64, F16), (40, 2, 64, BF16), (16, 1, 128, F16)])
@pytest.mark.parametrize("window", [None, 1, 37])
def test_decode_lengths(gpu, page, H, Hkv, D, dtype, window):
    (q, kc, vc, table, lengths), rows = _paged_problem(1, [1, 0, 2, 31, 33, 128, 129, 300], page, H, Hkv, D, dtype)
    o = kernels.attn_paged(q, kc, vc, table, lengths, D ** -0.5, window=window)
    _check_paged(q, rows, o, D ** -0.5, window, 0.0, {})


@pytest.mark.parametrize("cap,kind", list(itertools.product([0.0, 5.0], ["", "slopes", "table"])))
@pytest.mark.parametrize("D,dtype", [(128, BF16), (64, F16)])
@pytest.mark.parametrize("window", [None, 100])
def test_decode_rules(gpu, cap, kind, D, dtype, window):
    (q, kc, vc, table, lengths), rows = _paged_problem(2, [1, 40, 700, 129], 16, 6, 2, D, dtype)
    for radius in (0, 3, 45, 1024):
        bias = _bias(kind, 6, 3, radius)
        _check_paged(q, rows, kernels.attn_paged(q, kc, vc, table, lengths, 0.1, window=window, cap=cap, **bias), 0.1, window, cap, bias)
        if kind != "table":
            break


@pytest.mark.parametrize("lengths", [[5000], [5000, 1, 130, 0, 2500]], ids=str)
@pytest.mark.parametrize("D,dtype", [(128, BF16), (64, F16)])
def test_decode_many_chunks(gpu, lengths, D, dtype):
    """More chunks than the last workgroup joins by itself, beside sequences of a few and of one; repeated, on two streams, the same bits."""
    (q, kc, vc, table, n), rows = _paged_problem(8, lengths, 16, 4, 1, D, dtype)
    o = kernels.attn_paged(q, kc, vc, table, n, 0.1)
    _check_paged(q, rows, o, 0.1, None, 0.0, {})
    few = table[:, :100].contiguous()  # (up to 1600 keys: up to 13 chunks)
    want = kernels.attn_paged(q, kc, vc, few, n, 0.1)
    _check_paged(q, [(k[:1600], v[:1600]) for k, v in rows], want, 0.1, None, 0.0, {})
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(20):
        a, b = kernels.attn_paged(q, kc, vc, few, n, 0.1), kernels.attn_paged(q, kc, vc, table, n, 0.1)
        with torch.cuda.stream(side):
            c = kernels.attn_paged(q, kc, vc, few, n, 0.1)
        torch.cuda.synchronize()
        assert torch.equal(a, want) and torch.equal(b, o) and torch.equal(c, want)


@pytest.mark.parametrize("B,most", [(63, 700), (64, 700), (65, 300), (200, 200)])
def test_decode_many_sequences(gpu, B, most):
    """More sequences than a wavefront has lanes, of any lengths."""
    g = torch.Generator().manual_seed(B)
    (q, kc, vc, table, n), rows = _paged_problem(9, torch.randint(0, most, (B,), generator=g).tolist(), 16, 2, 1, 64, BF16)
    for window in (None, 100):
        _check_paged(q, rows, kernels.attn_paged(q, kc, vc, table, n, 0.1, window=window), 0.1, window, 0.0, {})


@pytest.mark.parametrize("B,few", [(1100, {0: 900, 63: 700, 64: 300, 511: 1000, 512: 257, 1050: 600, 1099: 2000}), (600, {}), (513, {512: 5000})], ids=str)
def test_decode_long_sequences_among_many_short(gpu, B, few):
    g = torch.Generator().manual_seed(B)
    lengths = [few.get(b, n) for b, n in enumerate(torch.randint(0, 40, (B,), generator=g).tolist())]
    (q, kc, vc, table, n), rows = _paged_problem(10, lengths, 16, 2, 1, 64, BF16)
    o = kernels.attn_paged(q, kc, vc, torch.nn.functional.pad(table, (0, 40)), n, 0.1)  # (also the short ones have a table for more keys than one chunk has)
    _check_paged(q, rows, o, 0.1, None, 0.0, {})
    assert torch.equal(o, kernels.attn_paged(q, kc, vc, torch.nn.functional.pad(table, (0, 40)), n, 0.1))


def test_decode_strides_and_long_tables(gpu):
    """Keys and values as halves of one cache with the head ahead of the row; a table and lengths that are parts of larger ones; a table for far
    more pages than there are (many chunks, most of them empty)."""
    (q, kc, vc, table, lengths), rows = _paged_problem(4, [100, 5, 333], 16, 4, 2, 128, BF16)
    pages = kc.shape[0]
    both = torch.empty(pages, 2, 2, 16, 128, dtype=BF16, device="cuda:0")
    both[:, 0], both[:, 1] = kc.transpose(1, 2), vc.transpose(1, 2)
    wide = torch.full((3, 5000), -1, dtype=torch.int32, device="cuda:0")
    wide[:, :table.shape[1]] = table
    qq = torch.cat([q, q], dim=2)[..., :128]
    for tab in (table, wide, wide[:, :4000]):
        o = kernels.attn_paged(qq, both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2), tab, lengths, 0.1)
        _check_paged(q, rows, o, 0.1, None, 0.0, {})


def test_decode_pages_outside_the_cache_are_not_seen(gpu):
    (q, kc, vc, table, lengths), rows = _paged_problem(5, [100, 64, 40], 16, 4, 2, 64, BF16)
    table[0, 2], table[0, 5], table[1, :] = -3, kc.shape[0], 1 << 30
    o = kernels.attn_paged(q, kc, vc, table, lengths, 0.1)
    keep = torch.tensor([j for j in range(100) if j // 16 not in (2, 5)])
    k, v = rows[0]
    want, tol = attention(q[:1], k[keep], v[keep], 0.1, torch.ones(1, len(keep), dtype=torch.bool), torch.zeros(1, len(keep), dtype=torch.int64))
    within(o[:1], want, tol)
    assert not o[1].any()
    _check_paged(q[2:], rows[2:], o[2:], 0.1, None, 0.0, {})


def test_decode_lengths_past_the_table_or_below_zero(gpu):
    (q, kc, vc, table, lengths), rows = _paged_problem(6, [64, 64], 16, 4, 2, 64, BF16)
    o = kernels.attn_paged(q, kc, vc, table[:, :4], torch.tensor([1 << 30, -5], dtype=torch.int32, device="cuda:0"), 0.1)
    _check_paged(q[:1], rows[:1], o[:1], 0.1, None, 0.0, {})
    assert not o[1].any()
    assert not kernels.attn_paged(q, kc[:0], vc[:0], table, lengths, 0.1).any()
    assert not kernels.attn_paged(q, kc, vc, table[:, :0], lengths, 0.1).any()
    assert kernels.attn_paged(q[:0], kc, vc, table[:0], lengths[:0], 0.1).shape == (0, 4, 64)


def test_decode_infinite_last_value(gpu):
    """The last key stands in for the tile's missing ones: what it holds counts once."""
    (q, kc, vc, table, lengths), rows = _paged_problem(7, [37], 16, 2, 2, 64, BF16)
    vc[table[0, 2], 4, :, 3] = float("inf")
    o = kernels.attn_paged(q, kc, vc, table, lengths, 0.1)
    assert (o[0, :, 3] == float("inf")).all() and o[0, :, :3].isfinite().all() and o[0, :, 4:].isfinite().all()


# ------------------------------------------------------------------------------------------------ rotary positions
@pytest.mark.parametrize("neox", [True, False])
@pytest.mark.parametrize("D,rot", [(128, 128), (128, 32), (64, 16), (64, 10), (64, 2), (8, 8), (256, 256), (96, 80)])
@pytest.mark.parametrize("T", [1, 5, 4099])
def test_rotary(gpu, neox, D, rot, T):
    dtype = BF16 if T == 5 else F16
    if T > 1000 and D > 96:
        T = 4097
    qkv = _randn(1, T, (3 + 2) * D, dtype=dtype)
    q, k = qkv[:, :3 * D].unflatten(1, (3, D)), qkv[:, 3 * D:].unflatten(1, (2, D))
    g = torch.Generator().manual_seed(2)
    positions = torch.randint(0, 1 << 20, (T,), generator=g)
    positions[0] = 0
    turns = torch.pow(10000.0, -torch.arange(rot // 2, dtype=torch.float64) / (rot // 2)) / 6.283185307179586
    got = kernels.rope_append(q, k, None, positions.to("cuda:0"), turns.to("cuda:0"), neox=neox, magnitude=1.25)
    some = torch.randperm(T, generator=g)[:40]
    for x, y in zip((q, k), got):
        assert y.is_contiguous()
        want, tol = rotated(x[some.to("cuda:0")], positions[some], turns, neox, 1.25)
        within(y[some.to("cuda:0")], want, tol)


@pytest.mark.parametrize("neox,rot,dtype", [(True, 128, BF16), (False, 64, F16), (True, 24, BF16)])
@pytest.mark.parametrize("page", [1, 5, 16])
def test_rotary_into_a_cache(gpu, neox, rot, dtype, page):
    T, H, Hkv, D, pages = 23, 4, 2, 128, 40
    q, k, v = _randn(3, T, H, D, dtype=dtype), _randn(4, T, Hkv, D, dtype=dtype), _randn(5, T, Hkv, D, dtype=dtype)
    g = torch.Generator().manual_seed(6)
    positions, slots = torch.randint(-50, 5000, (T,), generator=g), torch.randperm(pages * page, generator=g)[:T]
    slots[3], slots[7], slots[11] = -1, pages * page, 1 << 40  # not stored
    turns = torch.rand(rot // 2, generator=g, dtype=torch.float64)
    both = _randn(7, pages, 2, Hkv, page, D, dtype=dtype)
    kc, vc = both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2)
    before = kc.clone(), vc.clone()
    q_out, k_out = kernels.rope_append(q, k, v, positions.to("cuda:0"), turns.to("cuda:0"), neox=neox, slots=slots.to("cuda:0"), key_cache=kc, value_cache=vc)
    assert k_out is None
    want, tol = rotated(q, positions, turns, neox, 1.0)
    within(q_out, want, tol)
    want, tol = rotated(k, positions, turns, neox, 1.0)
    left = torch.ones(pages, page, dtype=torch.bool)
    for t, slot in enumerate(slots.tolist()):
        if not 0 <= slot < pages * page:
            continue
        at = slot // page, slot % page
        left[at] = False
        within(kc[at], want[t], tol[t])
        assert torch.equal(vc[at], v[t])
    for now, then in zip((kc, vc), before):
        assert torch.equal(now.cpu()[left], then.cpu()[left])


# ------------------------------------------------------------------------------------------------ together
@pytest.mark.parametrize("cap,kind,window", [(0.0, "", None), (8.0, "slopes", 50), (0.0, "table", None)])
def test_prompt_then_tokens(gpu, cap, kind, window):
    """Two prompts go into the cache and through their attention, then three tokens each, one by one: every step gives what whole-prompt
    attention over all rows so far gives its last row, and that of the definitions."""
    H, Hkv, D, page, lengths = 8, 2, 64, 16, [37, 90]
    kc, vc = (torch.full((20, page, Hkv, D), float("nan"), dtype=BF16, device="cuda:0") for _ in range(2))
    table = torch.arange(19, -1, -1, dtype=torch.int32, device="cuda:0")[:16].view(2, 8)
    turns = (torch.pow(10000.0, -torch.arange(D // 2, dtype=torch.float64) / (D // 2)) / 6.283185307179586).to("cuda:0")
    bias = _bias(kind, H, 8)
    total = [n + 3 for n in lengths]
    data = [[_randn(10 * b + i, total[b], h, D) for i, h in enumerate((H, Hkv, Hkv))] for b in range(2)]

    def append(parts, positions, seqs):
        slots = torch.tensor([int(table[b, p // page]) * page + p % page for b, p in zip(seqs, positions)], device="cuda:0")
        return kernels.rope_append(*parts, torch.tensor(positions, device="cuda:0"), turns, slots=slots, key_cache=kc, value_cache=vc)[0]

    with torch.inference_mode():
        packed = [torch.cat([data[b][i][:lengths[b]] for b in range(2)]) for i in range(3)]
        positions = [p for n in lengths for p in range(n)]
        q = append(packed, positions, [0] * lengths[0] + [1] * lengths[1])
        k = kernels.rope_append(packed[1], packed[1], None, torch.tensor(positions, device="cuda:0"), turns)[1]
        starts = [0, lengths[0], sum(lengths)]
        rules = dict(causal=True, window=window, q_starts=starts, k_starts=starts)
        os = _ruled(q[None], k[None], packed[2][None], 0.125, rules, bias, cap)
        _check_ruled(q[None], k[None], packed[2][None], os, 0.125, rules, bias, cap)
        for step in range(3):
            now = [n + step for n in lengths]
            parts = [torch.stack([data[b][i][now[b]] for b in range(2)]) for i in range(3)]
            q = append(parts, now, [0, 1])
            o = kernels.attn_paged(q, kc, vc, table, _i32([n + 1 for n in now]), 0.125, window=window, cap=cap, **bias)
            for b in range(2):
                at = torch.tensor([int(table[b, p // page]) * page + p % page for p in range(now[b] + 1)], device="cuda:0")
                kk, vv = kc.flatten(0, 1)[at], vc.flatten(0, 1)[at]
                whole = _ruled(q[None, b:b + 1], kk[None], vv[None], 0.125, dict(causal=True, window=window), bias, cap)
                seen, away = seen_keys(1, now[b] + 1, causal=True, window=window)
                want, tol = attention(q[b:b + 1], kk, vv, 0.125, seen, away, cap, **bias)
                within(o[b:b + 1], want, tol)
                for w in whole:
                    within(w[0], want, tol)


def test_streams_graphs_and_threads_of_work(gpu):
    """Calls on a side stream, and two captured graphs of decoding replayed side by side with eager calls between, give the eager bits."""
    (q, kc, vc, table, lengths), _ = _paged_problem(9, [900, 1500], 16, 8, 2, 64, BF16)
    p = _randn(10, 1, 3000, 8, 64)
    few = p[:, :9]
    eager = kernels.attn_paged(q, kc, vc, table, lengths, 0.1), kernels.attn_ruled(few, p, p, 0.1, causal=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = kernels.attn_paged(q, kc, vc, table, lengths, 0.1), kernels.attn_ruled(few, p, p, 0.1, causal=True)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(eager, other))
    q2 = q.flip(0).contiguous()
    graphs, outs = [], []
    for x in (q, q2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append((kernels.attn_paged(x, kc, vc, table, lengths, 0.1), kernels.attn_ruled(few, p, p, 0.1, causal=True)))
        graphs.append(graph)
    want = [eager[0], kernels.attn_paged(q2, kc, vc, table, lengths, 0.1)]
    for _ in range(3):
        for o in outs:
            o[0].zero_()
            o[1].zero_()
        side.wait_stream(torch.cuda.current_stream())
        graphs[0].replay()
        with torch.cuda.stream(side):
            graphs[1].replay()
        torch.cuda.synchronize()
        for i in range(2):
            assert torch.equal(outs[i][0], want[i]) and torch.equal(outs[i][1], eager[1])
        assert torch.equal(kernels.attn_paged(q, kc, vc, table, lengths, 0.1), eager[0])


def test_a_replayed_graph_follows_its_lengths_and_places(gpu):
    """One captured step of two sequences, replayed as they grow from one chunk to many: each replay gives the eager bits, caches included."""
    H, Hkv, D, page, pages = 8, 2, 128, 16, 260
    caches = [[_randn(60 + i, pages, page, Hkv, D) for i in range(2)] for _ in range(2)]  # the graph's and the eager calls'
    table = torch.randperm(pages, generator=torch.Generator().manual_seed(62)).int().view(2, 130).to("cuda:0")
    turns = torch.rand(D // 2, generator=torch.Generator().manual_seed(63), dtype=torch.float64).to("cuda:0")
    q, k, v = (torch.empty(2, h, D, dtype=BF16, device="cuda:0") for h in (H, Hkv, Hkv))
    lengths, slots = torch.ones(2, dtype=torch.int32, device="cuda:0"), torch.zeros(2, dtype=torch.int64, device="cuda:0")

    def step(kc, vc):
        turned = kernels.rope_append(q, k, v, lengths.long() - 1, turns, slots=slots, key_cache=kc, value_cache=vc)[0]
        return kernels.attn_paged(turned, kc, vc, table, lengths, 0.1, window=1500)

    def fill(i, n):
        for j, t in enumerate((q, k, v)):
            t.copy_(_randn(64 + 3 * i + j, *t.shape))
        lengths.copy_(_i32(n))
        slots.copy_(torch.tensor([int(table[b, (m - 1) // page]) * page + (m - 1) % page for b, m in enumerate(n)], device="cuda:0"))

    fill(0, [1, 1])
    for both in caches:
        step(*both)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = step(*caches[0])
    for i, n in enumerate([[1, 30], [700, 2080], [2, 257], [2000, 2000], [1, 1]]):
        fill(i, n)
        o.zero_()
        graph.replay()
        want = step(*caches[1])
        torch.cuda.synchronize()
        assert torch.equal(o, want), n
        assert all(map(torch.equal, caches[0], caches[1]))


def test_threads_on_one_stream(gpu):
    """Each thread's calls join their own chunks."""
    problems = [_paged_problem(70 + i, n, 16, 8, 2, 64, BF16)[0] for i, n in enumerate([[3000, 40], [500, 4000]])]
    wants = [kernels.attn_paged(*p, 0.1) for p in problems]
    torch.cuda.synchronize()
    failed = []

    def run(i):
        for _ in range(60):
            if not torch.equal(kernels.attn_paged(*problems[i], 0.1), wants[i]):
                failed.append(i)

    threads = [threading.Thread(target=run, args=(i,)) for i in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed


def test_places_past_32_bits(gpu):
    """Caches and prompts of more than 2^31 elements, their last rows used."""
    H, Hkv, D, page = 4, 2, 128, 16
    pages = (1 << 31) // (page * Hkv * D) + 300
    kc, vc = (torch.empty(pages, page, Hkv, D, dtype=BF16, device="cuda:0") for _ in range(2))
    n = 70
    q, k, v = _randn(80, n, H, D), _randn(81, n, Hkv, D), _randn(82, n, Hkv, D)
    order = [pages - 1 - 7 * i for i in range(-(-n // page))]
    slots = torch.tensor([order[t // page] * page + t % page for t in range(n)], device="cuda:0")
    turns, at = torch.zeros(D // 2, dtype=torch.float64, device="cuda:0"), torch.arange(n, device="cuda:0")
    kernels.rope_append(q, k, v, at, turns, slots=slots, key_cache=kc, value_cache=vc)
    for t in (0, 15, 16, n - 1):
        assert torch.equal(kc[order[t // page], t % page], k[t]) and torch.equal(vc[order[t // page], t % page], v[t])
    o = kernels.attn_paged(q[-1:], kc, vc, _i32([order]), _i32([n]), 0.1)
    _check_paged(q[-1:], [(k, v)], o, 0.1, None, 0.0, {})
    far_k, far_v = (t.view(-1, 1).view(-1).as_strided((2, n, Hkv, D), ((1 << 31) + 1024, Hkv * D, D, 1)) for t in (kc, vc))
    for t, x in ((far_k, k), (far_v, v)):
        t[0], t[1] = x, x.flip(0)
    rules = dict(causal=True)
    os = (kernels.attn_ruled(q[None].expand(2, n, H, D), far_k, far_v, 0.1, **rules),)
    _check_ruled(q[None].expand(2, n, H, D), torch.stack([k, k.flip(0)]), torch.stack([v, v.flip(0)]), os, 0.1, rules, {}, 0.0)


# ------------------------------------------------------------------------------------------------ refusals
def test_refusals(gpu):
    q, k, pos = _randn(1, 1, 8, 4, 64), _randn(2, 1, 8, 2, 64), torch.arange(8, device="cuda:0")
    lone, cache = q[0], _randn(3, 4, 16, 2, 64)
    turns = torch.rand(32, dtype=torch.float64, device="cuda:0")
    table, lengths = torch.zeros(8, 4, dtype=torch.int32, device="cuda:0"), torch.ones(8, dtype=torch.int32, device="cuda:0")
    ruled = lambda *a, **kw: kernels.attn_ruled(q, *(a or (k, k)), 0.1, **kw)  # noqa: E731
    paged = lambda **kw: kernels.attn_paged(*[kw.pop(n, x) for n, x in dict(q=lone, k=cache, v=cache, table=table, lengths=lengths).items()], 0.1, **kw)  # noqa: E731
    rope = lambda **kw: kernels.rope_append(*[kw.pop(n, x) for n, x in dict(q=lone, k=k[0], v=None, p=pos, t=turns).items()], **kw)  # noqa: E731
    into = dict(v=k[0], slots=pos, key_cache=cache, value_cache=cache.clone())
    for call, error in [
        (lambda: ruled(k, k[:, :7]), ValueError), (lambda: ruled(k.half(), k), TypeError), (lambda: ruled(window=0), ValueError),
        (lambda: ruled(window=-3), ValueError), (lambda: ruled(cap=-1.0), ValueError), (lambda: ruled(cap=1e5), ValueError),
        (lambda: ruled(cap=float("nan")), ValueError), (lambda: ruled(q_starts=_i32([0, 8])), ValueError),
        (lambda: ruled(q_starts=_i32([0, 8]), k_starts=_i32([0, 4, 8])), ValueError), (lambda: ruled(q_starts=_i32([0]), k_starts=_i32([0])), ValueError),
        (lambda: ruled(q_starts=pos, k_starts=pos), TypeError), (lambda: ruled(prefix=_i32([1, 2])), ValueError), (lambda: ruled(prefix=pos[:1]), TypeError),
        (lambda: ruled(slopes=torch.ones(3, device="cuda:0")), ValueError), (lambda: ruled(slopes=torch.ones(4, device="cuda:0").half()), TypeError),
        (lambda: ruled(distance=torch.ones(4, 6, device="cuda:0")), ValueError), (lambda: ruled(distance=torch.ones(4, 2051, device="cuda:0")), ValueError),
        (lambda: ruled(slopes=torch.ones(4, device="cuda:0"), distance=torch.ones(4, 5, device="cuda:0")), ValueError),
        (lambda: kernels.attn_ruled(q.float(), k.float(), k.float(), 0.1), TypeError), (lambda: kernels.attn_ruled(q, k, k, -0.1), RuntimeError),
        (lambda: kernels.attn_ruled(q[..., :48], k[..., :48], k[..., :48], 0.1), RuntimeError), (lambda: kernels.attn_ruled(q[:, :, :3], k, k, 0.1), RuntimeError),
        (lambda: ruled(k.cpu(), k), RuntimeError), (lambda: kernels.attn_ruled(lone, k, k, 0.1), ValueError),
        (lambda: paged(lengths=lengths.long()), TypeError), (lambda: paged(table=table.long()), TypeError), (lambda: paged(table=table[:7]), ValueError),
        (lambda: paged(v=cache[:3]), ValueError), (lambda: paged(k=cache.transpose(2, 3)), ValueError), (lambda: paged(k=cache.half()), TypeError),
        (lambda: paged(k=_randn(4, 4, 16, 2, 65)[..., :64]), ValueError), (lambda: paged(k=cache[:, :0], v=cache[:, :0]), ValueError),
        (lambda: paged(q=lone[:, :3]), RuntimeError), (lambda: paged(q=q), ValueError), (lambda: paged(window=0), ValueError),
        (lambda: paged(table=table[:, :1].expand(8, 1 << 27)), RuntimeError),
        (lambda: rope(v=k[0]), ValueError), (lambda: rope(slots=pos), ValueError), (lambda: rope(p=pos.int()), TypeError), (lambda: rope(p=pos[:7]), ValueError),
        (lambda: rope(t=turns.float()), TypeError), (lambda: rope(t=torch.rand(33, dtype=torch.float64, device="cuda:0")), RuntimeError),
        (lambda: rope(t=turns[:0]), RuntimeError), (lambda: rope(q=lone[..., :60], k=k[0, ..., :60]), RuntimeError), (lambda: rope(k=k[0, :7]), ValueError),
        (lambda: rope(**dict(into, slots=pos.int())), TypeError), (lambda: rope(**dict(into, key_cache=cache[..., :32])), ValueError),
        (lambda: rope(**dict(into, value_cache=cache[:3])), ValueError), (lambda: rope(**dict(into, key_cache=cache.half())), TypeError),
        (lambda: rope(q=lone.float(), k=k[0].float()), TypeError), (lambda: rope(**dict(into, key_cache=cache[:, :, :1].expand(-1, -1, 2, -1))), RuntimeError),
        (lambda: ruled(cap=1e-12), ValueError), (lambda: kernels.attn_ruled(q, k, k, 1e-12), RuntimeError), (lambda: paged(cap=1e-12), ValueError),
        (lambda: kernels.attn_ruled(q.clone().requires_grad_(), k, k, 0.1), RuntimeError), (lambda: paged(q=lone.clone().requires_grad_()), RuntimeError),
        (lambda: rope(q=lone.clone().requires_grad_()), RuntimeError),
    ]:
        with pytest.raises(error):
            call()
    with torch.no_grad():
        kernels.attn_ruled(q.clone().requires_grad_(), k, k, 0.1)
    assert kernels.rope_append(lone[:0], k[0, :0], None, pos[:0], turns)[1].shape == (0, 2, 64)
