"""What the C entries of a text stage's operators refuse, before any launch (so without a GPU)."""

import ctypes as C

import pytest
import torch

from vllm_omni_amd import _lib, kernels

_BUF = C.create_string_buffer(1 << 16)
P = (C.addressof(_BUF) + 63) & ~63
BF16, F32 = 0, 2


def _s(*v):
    return _lib.i64_array(v)


def _error():
    return _lib.load().odit_last_error().decode()


def _ruled(q=P, k=P, v=P, o=P, B=1, Sq=4, Sk=4, H=2, Hkv=1, D=64, qs=(512, 128, 64), ks=(256, 64, 64), vs=(256, 64, 64), os=(512, 128, 64), scale=0.1,
           dtype=BF16, ws=None, ws_bytes=0, **rules):
    r = _lib.AttnRules(**rules)
    return _lib.load().odit_attn_ruled(q, k, v, o, B, Sq, Sk, H, Hkv, D, _s(*qs), _s(*ks), _s(*vs), _s(*os), scale, C.byref(r), dtype, ws, ws_bytes, None)


def _paged(q=P, k=P, v=P, table=P, lengths=P, o=P, B=2, H=4, Hkv=2, D=64, pages=3, page=16, most=5, qs=(256, 64), ks=(2048, 128, 64), vs=(2048, 128, 64), ts=5,
           os=(256, 64), scale=0.1, dtype=BF16, ws=P, ws_bytes=1 << 30, **rules):
    r = _lib.AttnRules(**rules)
    return _lib.load().odit_attn_paged(q, k, v, table, lengths, o, B, H, Hkv, D, pages, page, most, _s(*qs), _s(*ks), _s(*vs), ts, _s(*os), scale, C.byref(r),
                                       dtype, ws, ws_bytes, None, 0, None)


def _rope(q=P, k=P, v=None, pos=P, turns=P, qo=P, ko=P, slots=None, kc=None, vc=None, T=4, H=2, Hkv=1, D=64, rot=64, pages=0, page=1, qs=(128, 64), ks=(64, 64),
          vs=(64, 64), kcs=(64, 64, 64), vcs=(64, 64, 64), dtype=BF16):
    return _lib.load().odit_rope_append(q, k, v, pos, turns, qo, ko, slots, kc, vc, T, H, Hkv, D, rot, pages, page, _s(*qs), _s(*ks), _s(*vs), _s(*kcs), _s(*vcs),
                                        1.0, dtype, 0, None)


@pytest.mark.parametrize("change,status,text", [
    (dict(D=96), -2, "head size"), (dict(dtype=F32), -2, "dtype"), (dict(H=3, Hkv=2), -1, "multiple"), (dict(scale=0.0), -1, "scale"),
    (dict(scale=float("nan")), -1, "scale"), (dict(window=-1), -1, "window"), (dict(window=(1 << 30) + 1), -1, "window"), (dict(docs=2), -1, "q_starts"),
    (dict(docs=-1), -1, "q_starts"), (dict(cap=-1.0), -1, "cap"), (dict(cap=9000.0), -1, "cap"), (dict(cap=float("nan")), -1, "cap"),
    (dict(slopes=P, distance=P), -1, "exclude"), (dict(distance=P, radius=1025), -1, "radius"), (dict(distance=P, radius=-1), -1, "radius"),
    (dict(k=P + 8), -1, "aligned"), (dict(ws=P + 8), -1, "aligned"), (dict(vs=(256, 60, 64)), -1, "multiples"), (dict(ks=(256, 1 << 23, 64)), -1, "apart"), (dict(ks=(256, -64, 64)), -1, "apart"),
    (dict(q=None), -1, "null"), (dict(v=None), -1, "null"), (dict(Sq=-1), -1, "shape"), (dict(Sk=(1 << 30) + 1), -1, "shape"), (dict(B=1 << 30, H=8), -1, "too many"),
    (dict(scale=1e-10), -1, "scale"), (dict(scale=float("inf")), -1, "scale"), (dict(cap=1e-12), -1, "cap"), (dict(B=1 << 10, Sq=1 << 29, H=64), -1, "too large"),
    (dict(B=1 << 12, Sq=1 << 16, H=8), -1, "too large")])
def test_ruled_refuses(change, status, text):
    assert _ruled(**change) == status and text in _error(), _error()


def test_ruled_takes_empty_problems():
    assert _ruled(B=0) == 0 and _ruled(Sq=0) == 0


def test_ruled_workspace():
    """Few query blocks with many keys are cut, into at most 32; what fills the GPU, and what has few keys, is not."""
    def chunks(B, Sq, Sk, H, D, block, **rules):
        need = _lib.load().odit_attn_ruled_workspace_bytes(B, Sq, Sk, H, D, C.byref(_lib.AttnRules(**rules)))
        part = (Sq + block - 1) // block * H * B * block * (D + 2) * 4
        assert need % part == 0
        return need // part or 1

    assert chunks(1, 1, 8192, 8, 128, 64) > 16 and chunks(1, 100, 8192, 32, 64, 64) > 8
    assert chunks(1, 1, 8192, 100, 128, 64) == 5 and chunks(1, 1, 8192, 256, 128, 128) == 2  # 512 workgroups run at once
    assert chunks(1, 1, 8192, 257, 128, 128) == 1 and chunks(1, 77, 77, 24, 128, 64) == 1 and chunks(1, 16384, 16384, 16, 128, 128) == 1
    assert chunks(1, 1, 1 << 20, 8, 128, 64, window=64, causal=1) == 1
    assert chunks(1, 64, 1 << 20, 8, 128, 64, docs=1 << 16, q_starts=P, k_starts=P) == 1
    assert _lib.load().odit_attn_ruled_workspace_bytes(0, 1, 8192, 8, 128, C.byref(_lib.AttnRules())) == 0


@pytest.mark.parametrize("change,status,text", [
    (dict(D=32), -2, "head size"), (dict(dtype=F32), -2, "dtype"), (dict(H=3), -1, "multiple"), (dict(scale=-1.0), -1, "scale"), (dict(page=0), -1, "shape"),
    (dict(pages=-1), -1, "shape"), (dict(most=1 << 27), -1, "keys"), (dict(window=-1), -1, "window"), (dict(docs=1, q_starts=P, k_starts=P), -1, "prompts"),
    (dict(prefix=P), -1, "prompts"), (dict(cap=1e9), -1, "cap"), (dict(slopes=P, distance=P), -1, "exclude"), (dict(distance=P, radius=2000), -1, "radius"),
    (dict(q=P + 2), -1, "aligned"), (dict(qs=(256, 60)), -1, "multiples"), (dict(vs=(2048, 128, 4)), -1, "multiples"), (dict(k=None), -1, "null"),
    (dict(lengths=None), -1, "null"), (dict(most=100, ws_bytes=16), -4, "workspace"), (dict(most=100, ws=None), -4, "workspace"), (dict(most=100, ws=P + 4), -4, "workspace"),
    (dict(scale=1e-10), -1, "scale"), (dict(scale=float("inf")), -1, "scale"), (dict(cap=1e-12), -1, "cap"), (dict(B=1 << 20, H=1 << 12, Hkv=1 << 12), -1, "too many"),
    (dict(B=1 << 22, H=8, Hkv=8), -1, "too large")])
def test_paged_refuses(change, status, text):
    assert _paged(**change) == status and text in _error(), _error()


def test_paged_empty_and_workspace():
    assert _paged(B=0) == 0
    need = _lib.load().odit_attn_paged_workspace_bytes
    assert need(3, 8, 2, 128, 16, 16, 0) == 0                               # 256 keys are one chunk
    assert need(3, 8, 2, 128, 1000, 16, 100) == 0                           # as is a window of 100
    one = need(1, 8, 2, 128, 17, 16, 0)
    assert one > 0 and one % (2 * 4 * 130 * 4) == 0                         # chunks of 2 kv heads, 4 heads each, 128 features and two statistics
    assert need(1, 48, 2, 64, 17, 16, 0) % (4 * 16 * 66 * 4) == 0           # 24 heads of a group are two blocks of up to 16
    assert need(0, 8, 2, 128, 8, 16, 0) == 0 and need(1, 8, 2, 128, 0, 16, 0) == 0


@pytest.mark.parametrize("page", [1, 2, 3, 16, 100])
def test_the_workspace_has_room_for_chunks_of_small_pages(page):
    """A chunk has the page numbers of 1024 pages at most: the longest sequences make as many chunks as that takes."""
    for B in (1, 70):
        most = (1 << 22) // page // B
        chunks = _lib.load().odit_attn_paged_workspace_bytes(B, 1, 1, 64, most, page, 0) // (66 * 4)
        room = max(64, 1023 * page // 64 * 64)
        assert chunks >= B * -(-most * page // room) and (page - 1 + room - 1) // page + 1 <= 1024


@pytest.mark.parametrize("change,status,text", [
    (dict(dtype=F32), -2, "dtype"), (dict(D=60, rot=60), -1, "head size"), (dict(D=1032), -1, "head size"), (dict(rot=0), -1, "rotary width"),
    (dict(rot=7), -1, "rotary width"), (dict(rot=66), -1, "rotary width"), (dict(v=P), -1, "slots"), (dict(kc=P), -1, "slots"), (dict(T=-1), -1, "shape"),
    (dict(slots=P, v=P, kc=P, vc=P, pages=2, page=4), -1, "slots"), (dict(slots=P, v=P, kc=P, vc=P, ko=None, page=0), -1, "slots"),
    (dict(slots=P, v=P, kc=P, ko=None, pages=2), -1, "null"), (dict(slots=P, kc=P, vc=P, ko=None, pages=2), -1, "null"),
    (dict(slots=P, v=P, kc=P, vc=P, ko=None, pages=2, kcs=(64, 60, 64)), -1, "multiples"), (dict(qs=(127, 64)), -1, "multiples"), (dict(k=P + 4), -1, "aligned"),
    (dict(slots=P, v=P, kc=P, vc=P, ko=None, pages=2, page=4, kcs=(64, 0, 64), vcs=(256, 64, 64)), -1, "share"), (dict(turns=None), -1, "null"), (dict(ko=None), -1, "null"), (dict(T=1 << 24), -1, "too many")])
def test_rope_refuses(change, status, text):
    assert _rope(**change) == status and text in _error(), _error()


def test_rope_takes_no_tokens():
    assert _rope(T=0) == 0


def test_wrappers_refuse_cpu_tensors():
    q = torch.zeros(1, 4, 2, 64, dtype=torch.bfloat16)
    i = torch.zeros(4, dtype=torch.int32)
    for call in (lambda: kernels.attn_ruled(q, q, q, 0.1), lambda: kernels.attn_paged(q[0], q, q, i[:, None], i, 0.1),
                 lambda: kernels.rope_append(q[0], q[0], None, i.long(), torch.zeros(32, dtype=torch.float64))):
        with pytest.raises(RuntimeError, match="GPU"):
            call()
