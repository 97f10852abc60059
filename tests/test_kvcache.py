"""KV-cache operators, without a GPU: shapes, sizes and refusals.  Nothing here launches; the pointers are never followed."""
import ctypes as C

import pytest

from kernelcore_b200 import kvcache
from kernelcore_b200 import lib

L = lib.raw
OK, INVALID_VALUE, INVALID_POINTER, UNSUPPORTED = 0, 2, 5, 7
GOOD = 0x7000_0000_1000


def cache(**kw):
    c = kvcache._Cache(bits=16, n_seqs=2, kv_heads=4, head_dim=64, capacity=100, k=GOOD, v=GOOD, k_row=256, k_head=64, k_seq=25600, v_row=256, v_head=64,
                       v_seq=25600, n_keys=GOOD, next_pos=GOOD, positions=GOOD, weights=GOOD)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def attn(**kw):
    a = kvcache._Attn(n_tokens=1, heads=8, scale=0.125, softcap=0.0, max_bias=0.0, causal=1, accumulate=0, q_token=512, q_head=64, q_seq=512, out_token=512,
                      out_head=64, out_seq=512)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def attention(c, a, q=GOOD, out=GOOD, ws=GOOD, ws_bytes=1 << 30):
    return L.kcb_cache_attention(C.byref(c) if c else None, C.byref(a) if a else None, q, out, ws, ws_bytes, None)


def test_sizes_of_the_buffers():
    b = kvcache.cache_bytes
    assert b(16, 2, 4, 64, 100) == 2 * 4 * 100 * 64 * 2
    assert b(4, 1, 8, 128, 1000) == 8 * 1000 * 80
    assert b(4, 3, 1, 32, 1) == 3 * 32          # 20 bytes, and a sequence begins at 16
    assert b(4, 1, 2, 256, 1 << 24) == 2 * (1 << 24) * 160   # 5 GB: no 32-bit product
    for bad in ((8, 1, 1, 32, 1), (4, 1, 1, 48, 1), (4, 1, 0, 32, 1), (4, -1, 1, 32, 1), (16, 1, 1, 32, 0)):
        assert b(*bad) == 0


BAD_CACHES = [(dict(bits=8), INVALID_VALUE), (dict(n_seqs=-1), INVALID_VALUE), (dict(n_seqs=70000), INVALID_VALUE), (dict(kv_heads=0), INVALID_VALUE),
              (dict(head_dim=48), INVALID_VALUE), (dict(head_dim=288), INVALID_VALUE), (dict(capacity=0), INVALID_VALUE), (dict(k=None), INVALID_VALUE),
              (dict(v=None), INVALID_VALUE), (dict(k_row=-8), INVALID_VALUE), (dict(k=GOOD + 8), INVALID_POINTER), (dict(v=GOOD + 2), INVALID_POINTER),
              (dict(k_row=252), INVALID_POINTER), (dict(v_seq=4), INVALID_POINTER), (dict(n_keys=GOOD + 2), INVALID_POINTER), (dict(weights=GOOD + 1), INVALID_POINTER)]


@pytest.mark.parametrize("kw, status", BAD_CACHES)
def test_every_entry_refuses_a_bad_cache(kw, status):
    c = cache(**kw)
    assert attention(c, attn()) == status
    assert L.kcb_cache_attention_workspace_bytes(C.byref(c), C.byref(attn())) == 0
    assert L.kcb_cache_append(C.byref(c), GOOD, GOOD, 1, 256, 256, None) == status
    assert L.kcb_cache_read(C.byref(c), 0, 1, GOOD, GOOD, None) == status
    assert L.kcb_cache_evict(C.byref(c), 10, 2, GOOD, 1 << 30, None) == status


@pytest.mark.parametrize("ckw, akw, status", [
    ({}, dict(n_tokens=-1), INVALID_VALUE), ({}, dict(heads=6), INVALID_VALUE), ({}, dict(heads=0), INVALID_VALUE),
    ({}, dict(scale=float("nan")), INVALID_VALUE), ({}, dict(softcap=-1.0), INVALID_VALUE), ({}, dict(softcap=float("inf")), INVALID_VALUE),
    ({}, dict(max_bias=float("nan")), INVALID_VALUE), ({}, dict(n_tokens=1 << 24), INVALID_VALUE),
    (dict(positions=None), dict(q_doc=GOOD), INVALID_VALUE), (dict(positions=None), dict(k_doc=GOOD), INVALID_VALUE),
    ({}, dict(q_doc=GOOD, k_doc=GOOD), INVALID_VALUE), ({}, dict(mask=GOOD), INVALID_VALUE),   # by slot, but the cache has positions
    ({}, dict(prefix=GOOD, causal=0), INVALID_VALUE), (dict(weights=None), dict(accumulate=1), INVALID_VALUE),
    ({}, dict(q_token=-4), INVALID_VALUE), ({}, dict(q_token=510), INVALID_POINTER), ({}, dict(out_head=2), INVALID_POINTER),
    ({}, dict(q_pos=GOOD + 2), INVALID_POINTER), (dict(positions=None), dict(mask=GOOD + 1), INVALID_POINTER),
    (dict(positions=None), dict(mask=GOOD, mask_token=-1), INVALID_VALUE),
    (dict(bits=4, head_dim=160), {}, UNSUPPORTED), (dict(bits=4, head_dim=192), {}, UNSUPPORTED), (dict(bits=4, head_dim=224), {}, UNSUPPORTED)])
def test_attention_refusals(ckw, akw, status):
    c, a = cache(**ckw), attn(**akw)
    assert attention(c, a) == status
    assert L.kcb_cache_attention_workspace_bytes(C.byref(c), C.byref(a)) == 0


def test_attention_refuses_missing_tensors_and_a_short_workspace():
    c, a = cache(capacity=5000, n_seqs=1), attn(accumulate=1)
    need = L.kcb_cache_attention_workspace_bytes(C.byref(c), C.byref(a))
    assert need > 0
    assert attention(None, a) == INVALID_VALUE and attention(c, None) == INVALID_VALUE
    assert attention(c, a, q=None) == INVALID_VALUE and attention(c, a, out=None) == INVALID_VALUE
    assert attention(c, a, q=GOOD + 4) == INVALID_POINTER and attention(c, a, out=GOOD + 8) == INVALID_POINTER
    assert attention(c, a, ws=None) == INVALID_VALUE and attention(c, a, ws_bytes=need - 1) == INVALID_VALUE
    assert attention(c, a, ws=GOOD + 8) == INVALID_POINTER
    # nothing to do is done
    assert attention(c, attn(n_tokens=0), ws=None, ws_bytes=0) == OK
    assert attention(cache(n_seqs=0), a, ws=None, ws_bytes=0) == OK


def test_append_read_and_evict_refusals():
    c = cache()
    ap = lambda c, k=GOOD, v=GOOD, n=1, tok=256, seq=256: L.kcb_cache_append(C.byref(c), k, v, n, tok, seq, None)  # noqa: E731
    assert ap(cache(n_keys=None)) == INVALID_VALUE and ap(c, k=None) == INVALID_VALUE and ap(c, n=-1) == INVALID_VALUE and ap(c, tok=-4) == INVALID_VALUE
    assert ap(c, k=GOOD + 4) == INVALID_POINTER and ap(c, tok=254) == INVALID_POINTER and ap(c, seq=2) == INVALID_POINTER
    assert ap(c, n=0) == OK and ap(cache(n_seqs=0)) == OK
    rd = lambda c, first=0, count=1, k=GOOD, v=GOOD: L.kcb_cache_read(C.byref(c), first, count, k, v, None)  # noqa: E731
    assert rd(c, first=-1) == INVALID_VALUE and rd(c, count=-1) == INVALID_VALUE and rd(c, first=100, count=1) == INVALID_VALUE
    assert rd(c, first=1, count=2 ** 31 - 1) == INVALID_VALUE and rd(c, k=None) == INVALID_VALUE and rd(c, v=GOOD + 4) == INVALID_POINTER
    assert rd(c, first=100, count=0) == OK
    ev = lambda c, keep=10, recent=2, ws=GOOD, n=1 << 20: L.kcb_cache_evict(C.byref(c), keep, recent, ws, n, None)  # noqa: E731
    for missing in ("n_keys", "next_pos", "positions", "weights"):
        assert ev(cache(**{missing: None})) == INVALID_VALUE
    assert ev(c, keep=0) == INVALID_VALUE and ev(c, recent=-1) == INVALID_VALUE and ev(c, recent=11) == INVALID_VALUE
    need = L.kcb_cache_evict_workspace_bytes(C.byref(c), 10)
    assert need > 0 and ev(c, n=need - 1) == INVALID_VALUE and ev(c, ws=None) == INVALID_VALUE and ev(c, ws=GOOD + 4) == INVALID_POINTER
    assert ev(c, keep=100, ws=None, n=0) == OK and L.kcb_cache_evict_workspace_bytes(C.byref(c), 100) == 0   # no sequence can hold more


def test_python_side_refuses_tensors_that_do_not_fit():
    import torch
    cpu = torch.zeros(1, 4, 2, 64, dtype=torch.float16)
    with pytest.raises(ValueError):
        kvcache.KVCache(cpu, cpu, kv_heads=2, head_dim=64, capacity=4)


@pytest.mark.parametrize("scale, softcap, fine", [(0.125, 1e30, False), (0.125, 1e19, True), (1e10, 1e-15, False), (0.125, 3e38, False), (3e38, 0.0, False), (0.0, 1e30, True),
                                                 (0.125, 50.0, True), (-0.125, 1e10, True), (1e10, 0.0, True)])
def test_caps_and_scales_stay_inside_the_range_of_fp32(scale, softcap, fine):
    c, a = cache(capacity=5000, n_seqs=1), attn(scale=scale, softcap=softcap)
    assert (L.kcb_cache_attention_workspace_bytes(C.byref(c), C.byref(a)) > 0) == fine
    assert attention(c, a, ws=None, ws_bytes=0) == INVALID_VALUE   # refused for the cap, else for the missing workspace


@pytest.mark.parametrize("kw", [dict(k_seq=0), dict(v_seq=0), dict(k_head=0), dict(v_row=0)])
def test_shared_rows_are_read_only(kw):
    c = cache(**kw)
    assert L.kcb_cache_append(C.byref(c), GOOD, GOOD, 1, 256, 256, None) == INVALID_VALUE
    assert L.kcb_cache_evict(C.byref(c), 10, 2, GOOD, 1 << 30, None) == INVALID_VALUE
    assert attention(c, attn(n_tokens=0), ws=None, ws_bytes=0) == OK


def test_outputs_on_top_of_each_other_are_refused():
    c = cache(positions=None, capacity=5000)
    for kw in (dict(n_tokens=2, out_token=0), dict(out_head=0), dict(out_seq=0)):
        assert attention(c, attn(**kw)) == INVALID_VALUE
