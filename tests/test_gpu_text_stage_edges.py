"""A text stage's operators at the edges of their numbers."""

import pytest
import torch

from test_gpu_text_stage import BF16, F16, _paged_problem, _randn, _ruled
from text_stage import attention, seen_keys, within
from vllm_omni_amd import kernels

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
