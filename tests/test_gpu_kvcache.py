"""KV-cache operators on the GPU against their 64-bit forms (kv_reference.py)."""
import math
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import kv_reference as ref
from kernelcore_b200 import kvcache, lib

pytestmark = pytest.mark.gpu


def rows(gen, *shape, size=1.0):
    x = torch.randn(*shape, generator=gen, device="cuda")
    return size * x * torch.exp(0.5 * torch.randn(*shape[2:], generator=gen, device="cuda"))


def filled(bits, S, cap, Hkv, D, n, seed, evictable=False, size=1.0):
    """A cache with n[s] rows in use, and its values [S][cap][Hkv][D] in 64 bits."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    c = kvcache.KVCache.empty(S, Hkv, D, cap, bits=bits, evictable=evictable)
    c.append(rows(gen, S, cap, Hkv, D, size=size), rows(gen, S, cap, Hkv, D, size=size))
    k, v = (x.double() for x in c.read(0, cap))
    c.n_keys.copy_(torch.tensor(n, dtype=torch.int32))
    c.next_pos.copy_(c.n_keys)
    return c, k, v, gen


def check(c, k, v, q, N, H, tol_factor=1.0, accumulate=False, **kw):
    kw.setdefault("scale", c.head_dim ** -0.5)
    w0 = c.weights.clone() if accumulate else None
    att = kvcache.Attention(c, n_tokens=N, heads=H, accumulate=accumulate, **kw)
    out = att(q)
    want, w, tol = ref.attend(q.double(), k, v, c.n_keys, next_pos=c.next_pos, k_pos=c.positions, **kw)
    err = (out.double() - want).abs().amax(-1)
    assert (err <= tol_factor * tol + 1e-30).all(), (err / tol.clamp(min=1e-30)).max().item()
    assert (out[(tol == 0).unsqueeze(-1).expand_as(out)] == 0).all()      # rows that see nothing
    if accumulate:
        # a weight's relative error is at most half of what moves an output; sums of up to N * group of them, plus the addition's rounding
        rel = (tol / v.abs().amax().clamp(min=1e-30)).amax().item() + 2.0 ** -22
        got = (c.weights - w0).double()
        assert ((got - w).abs() <= rel * w + 2.0 ** -23 * (w0.abs().double() + w)).all()
        for s in range(c.n_seqs):                                         # slots that are not in use keep what they hold
            assert torch.equal(c.weights[s, :, int(c.n_keys[s]):], w0[s, :, int(c.n_keys[s]):])
    return out


# ---- the 4-bit format -------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("S, N, Hkv, D, cap", [(1, 1, 1, 32, 1), (2, 5, 3, 96, 7), (3, 33, 2, 64, 40), (1, 130, 8, 128, 131), (2, 9, 1, 256, 9)])
def test_append_and_read_four_bits(S, N, Hkv, D, cap):
    gen = torch.Generator(device="cuda").manual_seed(S * 1000 + N)
    k, v = rows(gen, S, N, Hkv, D), rows(gen, S, N, Hkv, D, size=1e-3)
    k.view(-1)[:: 7] = 0.25                       # ties between codes, and blocks in which they meet the minimum
    c = kvcache.KVCache.empty(S, Hkv, D, cap, bits=4, evictable=True)
    c.weights.fill_(7.0)
    c.append(k, v)
    assert c.n_keys.tolist() == [N] * S and c.next_pos.tolist() == [N] * S
    assert torch.equal(c.positions[:, :, :N], torch.arange(N, dtype=torch.int32, device="cuda").expand(S, Hkv, N))
    assert (c.weights[:, :, :N] == 0).all() and (c.weights[:, :, N:] == 7).all()
    got = c.read(0, cap)
    for which, x, buf, g in (("k", k, c.k, got[0]), ("v", v, c.v, got[1])):
        val, code, d, m = ref.q4_block_values(x.cpu().numpy())
        for s in range(S):
            pc, pd, pm = ref.q4_unpack(buf[s].cpu().numpy(), Hkv, D, cap, which)
            assert (pc[:N].reshape(N, Hkv, -1, 32) == code[s]).all() and (pd[:N] == d[s]).all() and (pm[:N] == m[s]).all()
        assert (g[:, :N].cpu().numpy() == val.astype(np.float32)).all()   # d * code is exact, one rounding in the addition
        assert (g[:, N:] == 0).all()


def test_append_special_values_four_bits():
    x = torch.zeros(1, 4, 1, 64, device="cuda")
    x[0, 0, 0, :32] = 3.0                          # one value: scale 0
    x[0, 0, 0, 40] = math.nan                      # counts as 0
    x[0, 1, 0, 3], x[0, 1, 0, 4] = math.inf, -math.inf
    x[0, 2, 0, :32] = torch.linspace(-1e-7, 1e-7, 32)   # scale far below fp16's smallest
    x[0, 3, 0, :32] = torch.linspace(0, 15, 32)
    c = kvcache.KVCache.empty(1, 1, 64, 4, bits=4)
    c.append(x, x)
    val, *_ = ref.q4_block_values(x.cpu().numpy())
    for g in c.read(0, 4):
        assert torch.isfinite(g).all() and (g.cpu().numpy() == val.astype(np.float32)).all()


def test_codes_next_to_a_tie_are_rounded_from_the_exact_quotient():
    """d = 1/16 and m = 0 exactly: values a few fp32 steps around (j + 1/2) / 16."""
    base = (torch.arange(15, dtype=torch.float32) + 0.5) / 16
    steps = [base.clone() for _ in range(5)]
    for i in (0, 1):
        steps[i] = torch.nextafter(steps[i], torch.tensor(0.0)) if i == 0 else torch.nextafter(steps[i], torch.tensor(1.0))
    steps[3], steps[4] = base * (1 - 3e-7), base * (1 + 3e-7)
    x = torch.zeros(1, 5, 1, 32)
    for i, b in enumerate(steps):
        x[0, i, 0, :15], x[0, i, 0, 31] = b, 15 / 16
    c = kvcache.KVCache.empty(1, 1, 32, 5, bits=4)
    c.append(x.cuda(), x.cuda())
    val, *_ = ref.q4_block_values(x.numpy())
    assert (c.read(0, 5)[0].cpu().numpy() == val.astype(np.float32)).all()


@pytest.mark.parametrize("bits", [16, 4])
def test_append_step_by_step_strided_and_past_the_capacity(bits):
    """Slices of a q|k|v product, one token at a time, equal one append of all; what does not fit is dropped."""
    S, Hkv, D, cap, N = 2, 2, 64, 6, 9
    gen = torch.Generator(device="cuda").manual_seed(3)
    qkv = torch.randn(S, N, 8, D, generator=gen, device="cuda")
    k, v = qkv[:, :, 4:6], qkv[:, :, 6:8]
    a, b = kvcache.KVCache.empty(S, Hkv, D, cap, bits=bits, evictable=True), kvcache.KVCache.empty(S, Hkv, D, cap, bits=bits, evictable=True)
    a.append(k, v)
    for i in range(N):
        b.append(k[:, i:i + 1], v[:, i:i + 1])
    a.append(k[:, :0], v[:, :0])
    assert torch.equal(a.k, b.k) and torch.equal(a.v, b.v) and torch.equal(a.positions, b.positions)
    assert a.n_keys.tolist() == b.n_keys.tolist() == [cap] * S and a.next_pos.tolist() == b.next_pos.tolist() == [N] * S
    if bits == 16:
        assert torch.equal(a.k, k[:, :cap].half()) and torch.equal(a.v, v[:, :cap].half())
        assert torch.equal(a.read(2, 3)[0], k[:, 2:5].half().float())


# ---- attention ----------------------------------------------------------------------------------------------------------

SHAPES = [  # S, N, heads, kv heads, D, capacity, rows in use
    (1, 1, 1, 1, 32, 1, [1]), (1, 1, 4, 1, 64, 17, [16]), (2, 1, 12, 4, 64, 77, [77, 0]), (3, 1, 6, 2, 128, 300, [300, 1, 129]), (1, 1, 10, 2, 96, 65, [64]),
    (1, 1, 16, 1, 256, 50, [33]), (1, 2, 32, 8, 128, 1000, [999]), (2, 5, 3, 3, 32, 40, [40, 3]), (1, 1, 24, 1, 64, 700, [700]),
    (1, 17, 4, 4, 128, 64, [64]), (2, 33, 8, 2, 64, 130, [129, 40]), (1, 65, 2, 1, 96, 65, [65]), (1, 40, 6, 2, 256, 100, [90]), (1, 130, 5, 1, 32, 300, [290]),
    (1, 100, 8, 8, 128, 1300, [1222]), (1, 16, 8, 4, 64, 5000, [4801]),
    # the tcgen05 kernel: one row tile and several, one key tile, few, many, split
    (1, 96, 1, 1, 64, 96, [96]), (1, 97, 3, 3, 128, 97, [97]), (2, 130, 4, 2, 128, 150, [150, 131]), (1, 300, 6, 2, 64, 700, [650]), (1, 128, 1, 1, 128, 3000, [2999]),
    (3, 64, 4, 2, 64, 64, [64, 0, 1]), (1, 1000, 2, 2, 128, 1000, [1000]), (1, 50, 16, 2, 128, 63, [63])]


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_attention_shapes(bits, shape):
    S, N, H, Hkv, D, cap, n = shape
    c, k, v, gen = filled(bits, S, cap, Hkv, D, n, seed=sum(shape[:6]))
    q = torch.randn(S, N, H, D, generator=gen, device="cuda")
    check(c, k, v, q, N, H)
    check(c, k, v, q, N, H, causal=False)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("weights", [False, True], ids=["", "weights"])
@pytest.mark.parametrize("rows, Hkv, D, cap", [(8, 1, 64, 500), (9, 1, 128, 500), (15, 2, 64, 300), (16, 1, 128, 2100), (17, 2, 128, 300), (32, 2, 64, 333), (32, 1, 128, 2500),
                                               (33, 1, 128, 300), (9, 4, 32, 33000), (16, 4, 64, 33000), (24, 1, 256, 300), (17, 1, 96, 200)])
def test_attention_at_the_rows_where_kernels_change(bits, weights, rows, Hkv, D, cap):
    """Query rows of a kv head, as tokens times grouped heads, around every limit of the choice; 2^17 slots are one of them."""
    group = 4 if rows % 4 == 0 else 3 if rows % 3 == 0 else 1
    N, H = rows // group, group * Hkv
    c, k, v, gen = filled(bits, 1, cap, Hkv, D, [cap - 3], seed=rows + D, evictable=weights)
    q = torch.randn(1, N, H, D, generator=gen, device="cuda")
    check(c, k, v, q, N, H, accumulate=weights)
    check(c, k, v, q, N, H, accumulate=weights, softcap=8.0, max_bias=2.0)


FORMS = ["cap", "bias", "cap bias", "prefix", "docs", "mask", "mask slopes", "positions", "weights", "all"]


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("N, H, Hkv, D, cap", [(1, 8, 2, 64, 150), (3, 6, 3, 128, 70), (37, 6, 2, 64, 150), (20, 12, 2, 128, 333), (9, 4, 2, 256, 90)])
@pytest.mark.parametrize("form", FORMS)
def test_attention_forms(bits, N, H, Hkv, D, cap, form):
    S = 2
    n = [cap, cap // 2 + 1]
    c, k, v, gen = filled(bits, S, cap, Hkv, D, n, seed=N * 7 + H + len(form), evictable=form in ("positions", "weights", "all"))
    q = 2.0 * torch.randn(S, N, H, D, generator=gen, device="cuda")
    kw = {}
    if "cap" in form or form == "all":
        kw["softcap"] = 5.0                       # small enough to bend most scores
    if "bias" in form or form == "all":
        kw["max_bias"] = 8.0
    if form in ("prefix", "all"):
        kw["prefix"] = torch.tensor([cap // 3, 5], dtype=torch.int32, device="cuda")
    if form == "docs":
        kw["k_doc"] = torch.randint(0, 4, (S, cap), generator=gen, device="cuda").int().sort(1).values.contiguous()
        kw["q_doc"] = torch.randint(0, 5, (S, N), generator=gen, device="cuda").int()     # document 4 has no keys
        kw["causal"] = False
    if form.startswith("mask"):
        m = torch.randn(S, N, cap + 3, generator=gen, device="cuda").half()
        m[torch.rand(S, N, cap + 3, generator=gen, device="cuda") < 0.4] = -math.inf
        m[:, N // 2] = -math.inf                                                          # a row that sees nothing
        m[:, 0, ::3] = -65504.0                                                           # the lowest finite value
        kw["mask"], kw["causal"] = m, False
        if form == "mask slopes":
            kw["max_bias"] = 4.0
    if form in ("positions", "all"):
        order = torch.argsort(torch.rand(S, Hkv, cap, generator=gen, device="cuda"), -1).int()
        c.positions.copy_(order)
        c.next_pos.copy_(torch.tensor([cap, cap - 3], dtype=torch.int32))
        kw["q_pos"] = torch.randint(-1, cap, (S, N), generator=gen, device="cuda").int()  # -1: a padding query
    if form == "weights" or form == "all":
        c.weights.uniform_(0, 1, generator=gen)
    check(c, k, v, q, N, H, accumulate=form in ("weights", "all"), **kw)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("size", [1e-4, 1e-2, 30.0, 3000.0])
@pytest.mark.parametrize("N", [1, 24, 150])
def test_attention_of_small_and_large_values(bits, size, N):
    """Values (and, scaled back, keys) of every magnitude that fp16 holds: the probabilities' split must not lose them."""
    c, k, v, gen = filled(bits, 1, 200, 2, 64, [200], seed=11, size=size)
    q = torch.randn(1, N, 4, 64, generator=gen, device="cuda")
    check(c, k, v, q, N, 4, scale=0.125 / size)
    check(c, k, v, 1e-6 * q, N, 4, scale=1e6 * 0.125 / size)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("N", [1, 40, 130])
def test_what_is_hidden_never_reaches_an_output(bits, N):
    """Garbage behind the rows in use and in hidden slots: infinities and NaN, as keys, values or 4-bit scales."""
    S, H, Hkv, D, cap = 1, 4, 2, 128, 200
    c, k, v, gen = filled(bits, S, cap, Hkv, D, [150], seed=5)
    q = torch.randn(S, N, H, D, generator=gen, device="cuda")
    mask = torch.zeros(S, N, cap, dtype=torch.float16, device="cuda")
    hidden = [3, 64, 100, 149]
    mask[:, :, hidden] = -math.inf
    want = kvcache.Attention(c, n_tokens=N, heads=H, mask=mask, causal=False)(q)
    plain = kvcache.Attention(c, n_tokens=N, heads=H)(q)
    for value in (math.nan, math.inf, -math.inf):
        spots = hidden + list(range(150, cap))
        for buf in (c.k, c.v):
            if bits == 16:
                buf[:, spots] = value
            else:
                at = Hkv * cap * D // 2
                buf[0, at:at + Hkv * cap * D // 8].view(torch.float16).reshape(Hkv, cap, D // 32, 2)[:, spots] = value
        got = kvcache.Attention(c, n_tokens=N, heads=H, mask=mask, causal=False)(q)
        assert torch.equal(got, want)
    # rows behind those in use alone, without any mask
    c2, _, _, gen = filled(bits, S, cap, Hkv, D, [150], seed=5)
    q2 = torch.randn(S, N, H, D, generator=gen, device="cuda")
    c2.k.view(-1).view(torch.uint8)
    if bits == 16:
        c2.k[:, 150:], c2.v[:, 150:] = math.nan, math.inf
    else:
        at = Hkv * cap * D // 2
        for buf in (c2.k, c2.v):
            buf[0, at:at + Hkv * cap * D // 8].view(torch.float16).reshape(Hkv, cap, D // 32, 2)[:, 150:] = math.nan
    assert torch.equal(kvcache.Attention(c2, n_tokens=N, heads=H)(q2), plain)


@pytest.mark.parametrize("N", [4, 40, 80])
def test_an_infinite_value_reaches_those_who_see_it(N):
    """Causal: the newest slot holds an infinity and a NaN; the last token sees them, the ones before it do not."""
    c, k, v, gen = filled(16, 1, 100, 1, 64, [100], seed=9)
    q = torch.randn(1, N, 2, 64, generator=gen, device="cuda")
    clean = kvcache.Attention(c, n_tokens=N, heads=2)(q)
    c.v[0, 99, 0, 5], c.v[0, 99, 0, 6] = math.inf, math.nan
    got = kvcache.Attention(c, n_tokens=N, heads=2)(q)
    assert torch.isfinite(got[:, :-1]).all()
    # that tile's products run on the CUDA cores then: both paths are within the kernel's error of the definition
    want, _, tol = ref.attend(q.double(), k, v, c.n_keys, scale=0.125)
    assert ((got[:, :-1] - want[:, :-1]).abs().amax(-1) <= tol[:, :-1]).all() and ((clean - want).abs().amax(-1) <= tol).all()
    assert (got[0, -1, :, 5] == math.inf).all() and torch.isnan(got[0, -1, :, 6]).all() and torch.isfinite(got[0, -1, :, :5]).all()


def test_a_nan_query_spoils_its_own_row_only():
    for N in (3, 30, 55):
        c, k, v, gen = filled(16, 1, 60, 2, 64, [60], seed=2)
        q = torch.randn(1, N, 4, 64, generator=gen, device="cuda")
        clean = kvcache.Attention(c, n_tokens=N, heads=4)(q)
        q[0, 1, 2, 7] = math.nan
        got = kvcache.Attention(c, n_tokens=N, heads=4)(q)
        assert torch.isnan(got[0, 1, 2]).all()
        got[0, 1, 2] = clean[0, 1, 2]
        assert torch.equal(got, clean)


@pytest.mark.parametrize("bits", [16, 4])
def test_strided_queries_outputs_and_caches(bits):
    S, N, H, Hkv, D, cap = 2, 3, 4, 2, 64, 90
    c, k, v, gen = filled(bits, S, cap, Hkv, D, [90, 31], seed=4)
    wide = torch.randn(S, H, N, 2 * D, generator=gen, device="cuda")      # ggml's order: heads outside tokens, rows inside wider ones
    q = wide[..., D:].transpose(1, 2)
    out = torch.full((S, H, N, 2 * D), 9.0, device="cuda")
    want = kvcache.Attention(c, n_tokens=N, heads=H)(q.contiguous())
    kvcache.Attention(c, n_tokens=N, heads=H)(q, out[..., :D].transpose(1, 2))
    assert torch.equal(out[..., :D].transpose(1, 2), want) and (out[..., D:] == 9.0).all()
    if bits == 16:                                                         # head-major cache, and one inside a larger buffer
        for make in (lambda x: x.transpose(1, 2).contiguous().transpose(1, 2), lambda x: torch.cat([x, x], 3)[..., :D]):
            c2 = kvcache.KVCache(make(c.k), make(c.v), kv_heads=Hkv, head_dim=D, capacity=cap, n_keys=c.n_keys)
            assert torch.equal(kvcache.Attention(c2, n_tokens=N, heads=H)(q), want)


@pytest.mark.parametrize("N", [1, 20, 100])
def test_sequences_that_share_one_cache(N):
    """A sequence stride of zero: one cache (a common system prompt) for all sequences."""
    S, H, Hkv, D, cap = 3, 4, 2, 64, 200
    c, k, v, gen = filled(16, 1, cap, Hkv, D, [200], seed=3)
    n = torch.tensor([200, 150, 37], dtype=torch.int32, device="cuda")
    shared = kvcache.KVCache(c.k.expand(S, -1, -1, -1), c.v.expand(S, -1, -1, -1), kv_heads=Hkv, head_dim=D, capacity=cap, n_keys=n, next_pos=n)
    q = torch.randn(S, N, H, D, generator=gen, device="cuda")
    check(shared, k.expand(S, -1, -1, -1), v.expand(S, -1, -1, -1), q, N, H)


def test_offsets_past_32_bits():
    """Slots whose byte offsets pass 2^32 (4 bits) and whose element offsets pass 2^31 (fp16)."""
    Hkv, D = 1, 256
    for bits, cap in ((4, (1 << 25) + 5000), (16, (1 << 23) + 5000)):
        k, v = (torch.zeros(kvcache.cache_bytes(bits, 1, Hkv, D, cap), dtype=torch.uint8, device="cuda") for _ in range(2))
        if bits == 16:
            k, v = (x.view(torch.float16).reshape(1, cap, Hkv, D) for x in (k, v))
        n = torch.tensor([cap - 100], dtype=torch.int32, device="cuda")
        c = kvcache.KVCache(k, v, kv_heads=Hkv, head_dim=D, capacity=cap, bits=bits, n_keys=n)
        gen = torch.Generator(device="cuda").manual_seed(1)
        nk, nv = rows(gen, 1, 100, Hkv, D), rows(gen, 1, 100, Hkv, D)
        c.append(nk, nv)
        assert n.tolist() == [cap]
        rk, rv = c.read(cap - 100, 100)
        if bits == 16:
            assert torch.equal(rk, nk.half().float()) and torch.equal(rv, nv.half().float())
        else:
            assert (rk.cpu().numpy() == ref.q4_block_values(nk.cpu().numpy())[0].astype(np.float32)).all()
        # the last document is the last hundred rows: everything in front of it is hidden
        doc = torch.zeros(1, cap, dtype=torch.int32, device="cuda")
        doc[0, cap - 100:] = 1
        for N in (1, 20):
            q = torch.randn(1, N, 4, D, generator=gen, device="cuda")
            got = kvcache.Attention(c, n_tokens=N, heads=4, q_doc=torch.ones(1, N, dtype=torch.int32, device="cuda"), k_doc=doc)(q)
            small = torch.tensor([100], device="cuda")
            want, _, tol = ref.attend(q.double(), rk.double(), rv.double(), small, scale=D ** -0.5)
            assert ((got - want).abs().amax(-1) <= tol).all()
        del c, k, v, doc
        torch.cuda.empty_cache()


@pytest.mark.parametrize("bits", [16, 4])
def test_long_contexts_keep_their_digits(bits):
    """Over many keys an output is far smaller than the values it is made of.  Relative to the output's norm: a warp's sums are
    truncated at most 34 times by at most 2^-23 (4.1e-6; the splits' errors are independent, as their sums are), operands carry
    22 bits (5e-7), scores move weights by 1.5e-6: below 1e-5."""
    Hkv, D, cap = 1, 64, 300000
    c, k, v, gen = filled(bits, 1, cap, Hkv, D, [cap], seed=21)
    for N in (1, 130):
        q = torch.randn(1, N, 2, D, generator=gen, device="cuda")
        out = kvcache.Attention(c, n_tokens=N, heads=2, causal=False)(q).double()
        want, *_ = ref.attend(q.double(), k, v, c.n_keys, scale=D ** -0.5, causal=False)
        assert ((out - want).norm() / want.norm()).item() < 1e-5


@pytest.mark.parametrize("N", [1, 20, 100])
def test_query_positions_at_the_ends_of_their_range(N):
    """The largest position sees everything, the smallest nothing."""
    c, k, v, gen = filled(16, 1, 90, 1, 64, [90], seed=12)
    q = torch.randn(1, N, 2, 64, generator=gen, device="cuda")
    pos = torch.full((1, N), 2 ** 31 - 1, dtype=torch.int32, device="cuda")
    far = kvcache.Attention(c, n_tokens=N, heads=2, q_pos=pos)(q)
    assert torch.equal(far, kvcache.Attention(c, n_tokens=N, heads=2, causal=False)(q))
    pos.fill_(-2 ** 31)
    assert (kvcache.Attention(c, n_tokens=N, heads=2, q_pos=pos)(q) == 0).all()


def test_first_call_inside_a_capture():
    """A fresh process whose first attention, append and eviction are captured."""
    code = """
import torch
from kernelcore_b200 import kvcache
torch.cuda.set_device(0)
c = kvcache.KVCache.empty(1, 2, 64, 300, bits=4, evictable=True)
k = torch.randn(1, 200, 2, 64, device="cuda")
q = torch.randn(1, 100, 4, 64, device="cuda")
att = kvcache.Attention(c, n_tokens=100, heads=4, accumulate=True)
out = torch.empty_like(q)
c._evict_ws
c.evict(299, 1)
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    c.append(k, k)
    att(q, out)
c.n_keys.zero_(); c.next_pos.zero_()
g.replay()
torch.cuda.synchronize()
first = out.clone()
c.n_keys.zero_(); c.next_pos.zero_()
c.append(k, k)
assert torch.equal(att(q), first) and c.n_keys.tolist() == [200]
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120, cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    assert r.returncode == 0, r.stderr


# ---- eviction -------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("S, Hkv, D, cap, n, keep, recent", [(1, 1, 32, 5, [5], 4, 0), (2, 3, 64, 40, [40, 9], 10, 3), (1, 2, 96, 300, [299], 298, 298), (2, 2, 128, 2500, [2500, 1700], 600, 50),
                                                             (1, 1, 256, 100, [100], 1, 1), (3, 1, 64, 30, [0, 7, 30], 7, 2)])
def test_evict(bits, S, Hkv, D, cap, n, keep, recent):
    c, k, v, gen = filled(bits, S, cap, Hkv, D, n, seed=cap + keep, evictable=True)
    for s in range(S):                                                       # an order that earlier evictions left, gaps in it
        c.positions[s, :, :n[s]] = torch.stack([torch.randperm(n[s] + 5, generator=gen, device="cuda")[:n[s]].int() for _ in range(Hkv)])
        c.next_pos[s] = n[s] + 5
    c.weights.copy_(torch.randint(0, 12, (S, Hkv, cap), generator=gen, device="cuda").float())   # many ties
    c.weights[:, :, ::17] = -0.0
    c.weights[:, :, 1::19] = math.nan
    pos, w, cnt = c.positions.cpu().numpy().copy(), c.weights.cpu().numpy().copy(), list(n)
    kk, vv = k.cpu().numpy().copy(), v.cpu().numpy().copy()
    before = (c.k.clone(), c.v.clone())
    ref.evict([kk, vv], pos, w, cnt, c.next_pos.tolist(), keep, recent)
    c.evict(keep, recent)
    assert c.n_keys.tolist() == cnt
    assert (c.positions.cpu().numpy() == pos).all() and np.array_equal(c.weights.cpu().numpy(), w, equal_nan=True)
    gk, gv = c.read(0, cap)
    for s in range(S):
        assert (gk[s, :cnt[s]].cpu().numpy() == kk[s, :cnt[s]]).all() and (gv[s, :cnt[s]].cpu().numpy() == vv[s, :cnt[s]]).all()
    if bits == 16:                                                           # rows behind those in use stay as they were
        assert torch.equal(c.k[:, keep:], before[0][:, keep:]) and torch.equal(c.v[:, keep:], before[1][:, keep:])
    c.evict(keep, recent)                                                    # nothing left to drop
    assert c.n_keys.tolist() == cnt and (c.positions.cpu().numpy() == pos).all()


def test_evict_a_cache_longer_than_shared_memory_holds_keys():
    cap, keep = 60000, 20000
    c, k, v, gen = filled(16, 1, cap, 1, 32, [cap], seed=8, evictable=True)
    c.weights.copy_(torch.rand(1, 1, cap, generator=gen, device="cuda").mul(4096).round())
    pos, w, cnt = c.positions.cpu().numpy().copy(), c.weights.cpu().numpy().copy(), [cap]
    kk = k.cpu().numpy().copy()
    ref.evict([kk], pos, w, cnt, [cap], keep, 100)
    c.evict(keep, 100)
    assert c.n_keys.tolist() == cnt and (c.positions.cpu().numpy() == pos).all() and np.array_equal(c.weights.cpu().numpy(), w)
    assert (c.read(0, keep)[0].cpu().numpy() == kk[:, :keep]).all()


# ---- together ---------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("graph", [False, True])
def test_a_streaming_decode_loop(bits, graph):
    """Prompt, then tokens one by one: append, attend with accumulated weights and distance bias, evict to a budget; in
    64 bits beside it.  The same step, captured once and replayed, gives the same bits as the eager one."""
    S, H, Hkv, D, cap, keep, recent, prompt, steps = 2, 6, 2, 64, 40, 24, 6, 20, 14
    gen = torch.Generator(device="cuda").manual_seed(6)
    c = kvcache.KVCache.empty(S, Hkv, D, cap, bits=bits, evictable=True)
    side = torch.cuda.Stream()
    kp, vp, qp = rows(gen, S, prompt, Hkv, D), rows(gen, S, prompt, Hkv, D), torch.randn(S, prompt, H, D, generator=gen, device="cuda")
    toks = [(rows(gen, S, 1, Hkv, D), rows(gen, S, 1, Hkv, D), torch.randn(S, 1, H, D, generator=gen, device="cuda")) for _ in range(steps)]
    c.append(kp, vp)
    first = kvcache.Attention(c, n_tokens=prompt, heads=H, max_bias=8.0, accumulate=True)
    first(qp)
    step = kvcache.Attention(c, n_tokens=1, heads=H, max_bias=8.0, softcap=20.0, accumulate=True)
    ink, inv, inq = (torch.empty_like(x) for x in toks[0])
    out = torch.empty(S, 1, H, D, device="cuda")

    def one():
        c.append(ink, inv)
        step(inq, out)
        c.evict(keep, recent)

    state = lambda: [x.clone() for x in (c.k, c.v, c.n_keys, c.next_pos, c.positions, c.weights)]  # noqa: E731
    saved = state()
    g = None
    if graph:
        for x, t in zip((ink, inv, inq), toks[0]):
            x.copy_(t)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            one()                                                             # workspaces are made before the capture
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            one()
        for x, t in zip((c.k, c.v, c.n_keys, c.next_pos, c.positions, c.weights), saved):
            x.copy_(t)
    for i, (k1, v1, q1) in enumerate(toks):
        for x, t in zip((ink, inv, inq), (k1, v1, q1)):
            x.copy_(t)
        k0, v0 = (x.double().cpu().numpy() for x in c.read(0, cap))
        n = c.n_keys.tolist()
        nk = ref.q4_block_values(k1.cpu().numpy())[0] if bits == 4 else k1.half().double().cpu().numpy()
        nv = ref.q4_block_values(v1.cpu().numpy())[0] if bits == 4 else v1.half().double().cpu().numpy()
        pos, w = c.positions.cpu().numpy().copy(), c.weights.double()
        for s in range(S):
            k0[s, n[s]], v0[s, n[s]], pos[s, :, n[s]], w[s, :, n[s]] = nk[s, 0], nv[s, 0], int(c.next_pos[s]), 0.0
        nxt = (c.next_pos + 1).tolist()
        cnt = [x + 1 for x in n]
        want, dw, tol = ref.attend(q1.double(), torch.tensor(k0).cuda(), torch.tensor(v0).cuda(), cnt, scale=D ** -0.5, max_bias=8.0, softcap=20.0,
                                   k_pos=torch.tensor(pos).cuda(), next_pos=nxt)
        if graph:
            g.replay()
        else:
            one()
        assert ((out - want).abs().amax(-1) <= tol).all(), i
        w = (w + dw).cpu().numpy()
        live = [x.copy() for x in (k0, v0)]
        ref.evict(live, pos, w, cnt, nxt, keep, recent)
        assert c.n_keys.tolist() == cnt and c.next_pos.tolist() == nxt
        for s in range(S):
            assert (c.positions[s, :, :cnt[s]].cpu().numpy() == pos[s, :, :cnt[s]]).all()
            assert np.allclose(c.weights[s, :, :cnt[s]].cpu().numpy(), w[s, :, :cnt[s]], rtol=1e-4, atol=1e-7)
            assert (c.read(0, cap)[0][s, :cnt[s]].cpu().numpy() == live[0][s, :cnt[s]].astype(np.float32)).all()


@pytest.mark.parametrize("N, H, Hkv, softcap, max_bias", [(3, 6, 2, 30.0, 0.0), (1, 8, 4, 0.0, 8.0), (60, 6, 2, 20.0, 8.0)])
def test_the_ggml_operator_takes_caps_and_biases(N, H, Hkv, softcap, max_bias):
    """FLASH_ATTN_EXT with a logit softcap and with ALiBi (slope times the mask, which holds the distances)."""
    import ctypes as C

    from test_gpu_ggml_ops import F16, F32, f32_bits, op, tensor
    D, T = 64, 77
    gen = torch.Generator(device="cuda").manual_seed(N)
    kc, vc = (torch.randn(T, Hkv, D, generator=gen, device="cuda").half() for _ in range(2))
    q = torch.randn(H, N, D, generator=gen, device="cuda")                              # ggml's [D, N, H]
    at = T - N + torch.arange(N, device="cuda").unsqueeze(1)
    t = torch.arange(80, device="cuda")
    mask = torch.where((t <= at) & (t < T), -(at - t).abs().float(), -math.inf).half().contiguous()
    out = torch.zeros(N, H, D, device="cuda")
    h = C.c_void_p()
    assert lib.raw.kcb_ggml_ctx_create(None, C.byref(h)) == 0 and lib.raw.kcb_ggml_ctx_begin_graph(h) == 0
    kt, vt = (tensor(x, F16, [D, T, Hkv], nb=[2, 2 * Hkv * D, 2 * D, 2 * Hkv * D * T]) for x in (kc, vc))
    params = [f32_bits(0.125), f32_bits(max_bias), f32_bits(softcap)]
    op("flash_attn", h, tensor(out, F32, [D, H, N], src=(tensor(q, F32, [D, N, H]), kt, vt, tensor(mask, F16, [80, N])), params=params))
    lib.raw.kcb_ggml_ctx_destroy(h)
    want, _, tol = ref.attend(q.transpose(0, 1).unsqueeze(0).double(), kc.unsqueeze(0).double(), vc.unsqueeze(0).double(), [T], scale=0.125, softcap=softcap,
                              max_bias=max_bias, causal=False, mask=mask.unsqueeze(0))
    assert ((out - want[0]).abs().amax(-1) <= tol[0]).all()


def test_two_streams_and_the_same_call_twice():
    c, k, v, gen = filled(4, 2, 3000, 2, 128, [3000, 2000], seed=1)
    q = torch.randn(2, 1, 8, 128, generator=gen, device="cuda")
    a, b = (kvcache.Attention(c, n_tokens=1, heads=8) for _ in range(2))
    want = a(q)
    assert torch.equal(a(q), want)                                              # no atomics: the same bits every time
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    outs = []
    for _ in range(5):
        with torch.cuda.stream(side):
            outs.append(a(q))
        outs.append(b(q))                                                       # another object, another workspace
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_python_side_refusals():
    c = kvcache.KVCache.empty(1, 2, 64, 10)
    with pytest.raises(ValueError):
        c.append(torch.zeros(1, 1, 3, 64, device="cuda"), torch.zeros(1, 1, 3, 64, device="cuda"))
    with pytest.raises(ValueError):
        c.append(torch.zeros(1, 1, 2, 64), torch.zeros(1, 1, 2, 64))
    with pytest.raises(ValueError):
        c.read(5, 6)
    with pytest.raises(lib.KcbError):
        c.evict(5, 1)                                                           # no positions beside the rows
    with pytest.raises(ValueError):
        kvcache.Attention(c, n_tokens=1, heads=2)(torch.zeros(1, 1, 2, 64))
    with pytest.raises(ValueError):
        kvcache.Attention(c, n_tokens=1, heads=2, mask=torch.zeros(1, 1, 9, dtype=torch.float16, device="cuda"))


def test_objects_created_on_one_stream_and_dropped_after_use_on_another():
    """The workspace of a dropped object is not handed to the next tensor while the call on the other stream still uses it."""
    c, k, v, gen = filled(4, 1, 20000, 2, 64, [20000], seed=3)
    q = torch.randn(1, 1, 8, 64, generator=gen, device="cuda")
    want = kvcache.Attention(c, n_tokens=1, heads=8)(q)
    out, side = torch.empty_like(want), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    a = kvcache.Attention(c, n_tokens=1, heads=8)
    n = a.workspace.numel()
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
        a(q, out)
    del a
    for _ in range(4):
        torch.empty(n, dtype=torch.uint8, device="cuda").fill_(0x7F)   # would be the workspace
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, want)


def test_evict_on_another_stream_and_with_no_sequence():
    c, k, v, gen = filled(16, 2, 300, 2, 64, [300, 200], seed=4, evictable=True)
    c.weights.uniform_(0, 1, generator=gen)
    d = kvcache.KVCache(c.k.clone(), c.v.clone(), kv_heads=2, head_dim=64, capacity=300, n_keys=c.n_keys.clone(), next_pos=c.next_pos.clone(),
                        positions=c.positions.clone(), weights=c.weights.clone())
    c.evict(100, 10)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        d.evict(100, 10)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(c.n_keys, d.n_keys) and torch.equal(c.positions[:, :, :100], d.positions[:, :, :100]) and torch.equal(c.k[:, :100], d.k[:, :100])
    kvcache.KVCache.empty(0, 2, 64, 300, evictable=True).evict(100, 10)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("N, H, Hkv, D, cap, n", [(64, 4, 2, 64, 64, 64), (65, 2, 1, 128, 100, 100), (200, 2, 1, 128, 300, 290), (300, 8, 2, 64, 500, 400), (500, 2, 1, 32, 70, 70),
                                                  (700, 1, 1, 256, 700, 700), (40, 4, 4, 96, 1300, 65)])
def test_weights_of_prompts_by_one_cta_and_by_clusters(bits, N, H, Hkv, D, cap, n):
    """Query tiles of 64 rows shared out over 1, 2, 4 or 8 CTAs, tiles that do not divide evenly, ranks that have none left."""
    c, k, v, gen = filled(bits, 1, cap, Hkv, D, [n], seed=N + D, evictable=True)
    q = torch.randn(1, N, H, D, generator=gen, device="cuda")
    check(c, k, v, q, N, H, accumulate=True)
    check(c, k, v, q, N, H, accumulate=True, softcap=10.0, prefix=torch.tensor([n // 2], dtype=torch.int32, device="cuda"))
    w0 = c.weights.clone()
    att = kvcache.Attention(c, n_tokens=N, heads=H, accumulate=True)
    att(q)
    first = c.weights.clone()
    c.weights.copy_(w0)
    att(q)
    assert torch.equal(c.weights, first)   # the order of the sums is fixed
