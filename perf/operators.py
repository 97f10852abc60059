"""What is measured of the KV-cache operators: attention with capped or biased scores and document or prefix masks over an
fp16 or a 4-bit cache, appending to and reading back a cache, and eviction by accumulated attention weight.

A state is what a serving program has in hand: the cache's buffers (fp16 rows, or the packed 4-bit planes), the row
counts, positions and weights that live beside them, the step's queries and masks.  `run` takes one pass through an
operator, either in elementary torch operations or through kernelcore_b200.kvcache."""
from __future__ import annotations

import math

import torch

own = False

BLOCK = 32          # channels that share a scale and a minimum in the 4-bit cache
F16_MAX = 65504.0


# ---- cases --------------------------------------------------------------------------------------------------------

def _attn(name, **kw):
    c = {"op": "attend", "bits": 16, "seqs": 1, "tokens": 1, "heads": 32, "kv_heads": 8, "dim": 128, "capacity": 512, "ragged": False,
         "softcap": 0.0, "max_bias": 0.0, "causal": True, "prefix": 0, "docs": 0, "mask": False, "weights": False}
    c.update(kw)
    if name:
        c["name"] = name
    return c


def _cache(name, op, **kw):
    c = {"op": op, "bits": 16, "seqs": 1, "tokens": 1, "kv_heads": 8, "dim": 128, "capacity": 512, "keep": 0, "recent": 0}
    c.update(kw)
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # one user's chat, early in the conversation: a single token over a short cache, capped scores; latency counts
        _attn("f16 decode short capped", capacity=333, softcap=50.0),
        # a server's step over many users with distance-biased scores, every sequence at its own length
        _attn("f16 decode batch biased", seqs=32, capacity=4096, ragged=True, max_bias=8.0),
        # a packed batch of short documents in one row: each token sees its own document only
        _attn("f16 prompt documents", tokens=4096, capacity=4096, docs=9),
        # a long prompt whose first part is read in both directions, capped scores: the largest product here
        _attn("f16 prompt prefix capped", tokens=4096, capacity=4096, prefix=1000, softcap=30.0),
        # a small model's odd-sized prompt under an additive mask, some of whose rows are padding
        _attn("f16 prompt mask small", seqs=2, tokens=157, heads=12, kv_heads=4, dim=64, capacity=201, ragged=True, causal=False, mask=True),
        # single token over a short 4-bit cache of a small model: the smallest call
        _attn("q4 decode short", bits=4, heads=12, kv_heads=4, dim=64, capacity=77),
        # one user with a book in the context: the cache that 4 bits are for
        _attn("q4 decode long", bits=4, capacity=131072),
        # a server's step that also accumulates the attention weights which eviction goes by
        _attn("q4 decode batch weights", bits=4, seqs=32, capacity=4096, ragged=True, weights=True),
        # a chunk of a long prompt: its queries over everything read so far, the chunk included
        _attn("q4 prompt chunk", bits=4, tokens=256, capacity=8192 + 256),
        # a prompt's keys and values into the 4-bit cache and back (what a program that saves a session reads)
        _cache("q4 append and read prompt", "store", bits=4, tokens=4096, capacity=5000),
        # a streaming server's step at a full budget: one token in, the least attended row out
        _cache("f16 evict step", "step", seqs=16, capacity=1100, keep=1024, recent=64),
        # after long prompts: a quarter of the rows stays
        _cache("f16 evict prompt", "evict", seqs=8, capacity=8192, keep=2048, recent=256),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["decode", "decode", "prompt", "prompt", "store", "step", "evict"])
    bits = rng.choice([16, 4])
    dim = rng.choice([32, 64, 96, 128, 128, 256])
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    if kind == "decode":
        heads = kv_heads * rng.choice([1, 2, 3, 4, 5, 8, 16])
        seqs = _log(rng, 1, 32)
        capacity = max(1, _log(rng, 1, min(65536, (1 << 26) // (seqs * kv_heads * dim))))
        form = rng.choice(["plain", "cap", "bias", "both", "docs", "weights"])
        return _attn(None, bits=bits, seqs=seqs, tokens=rng.choice([1, 1, 1, 2, 5]), heads=heads, kv_heads=kv_heads, dim=dim, capacity=capacity,
                     ragged=rng.random() < 0.6, softcap=rng.choice([20.0, 50.0]) if form in ("cap", "both") else 0.0,
                     max_bias=8.0 if form in ("bias", "both") else 0.0, docs=3 if form == "docs" else 0, weights=form == "weights")
    if kind == "prompt":
        group = rng.choice([1, 2, 3, 4, 8])
        tokens = _log(rng, 6, 2048)
        before = _log(rng, 1, 2048) if rng.random() < 0.5 else 0
        while tokens * (tokens + before) * kv_heads * group * dim > 1 << 34:               # the largest listed case has that many products
            tokens = tokens * 2 // 3
        capacity = tokens + before
        seqs = max(1, min(_log(rng, 1, 8), (1 << 34) // (tokens * capacity * kv_heads * group * dim), 4096 // tokens))
        form = rng.choice(["plain", "cap", "bias", "docs", "prefix", "mask", "full", "weights"])
        return _attn(None, bits=bits, seqs=seqs, tokens=tokens, heads=kv_heads * group, kv_heads=kv_heads, dim=dim, capacity=capacity,
                     ragged=rng.random() < 0.4, softcap=30.0 if form in ("cap", "prefix") else 0.0, max_bias=8.0 if form == "bias" else 0.0,
                     docs=rng.choice([2, 7]) if form == "docs" else 0, prefix=max(1, capacity // 3) if form == "prefix" else 0,
                     mask=form == "mask", causal=form not in ("mask", "full"), weights=form == "weights")
    seqs = _log(rng, 1, 16)
    if kind == "store":
        tokens = _log(rng, 1, max(1, (1 << 22) // (seqs * kv_heads * dim)))
        return _cache(None, "store", bits=bits, seqs=seqs, tokens=tokens, kv_heads=kv_heads, dim=dim, capacity=tokens + rng.randrange(0, 50))
    keep = _log(rng, 5, 2048)
    recent = rng.randrange(0, keep)
    if kind == "step":
        return _cache(None, "step", seqs=seqs, kv_heads=kv_heads, dim=dim, capacity=keep + rng.randrange(1, 100), keep=keep, recent=recent)
    return _cache(None, "evict", seqs=seqs, kv_heads=kv_heads, dim=dim, capacity=keep + _log(rng, 1, 4096), keep=keep, recent=recent)


# ---- inputs -------------------------------------------------------------------------------------------------------

def _rows(gen, shape, dim):
    """Keys or values as a model makes them: some channels several times larger than others."""
    x = torch.randn(*shape, dim, generator=gen, device="cuda")
    return x * torch.exp(0.5 * torch.randn(shape[-1], dim, generator=gen, device="cuda"))


def _quantize(x):
    """Codes, scales and minima of blocks of 32 channels."""
    b = x.clamp(-F16_MAX, F16_MAX).unflatten(-1, (-1, BLOCK))
    lo, hi = b.amin(-1), b.amax(-1)
    m = lo.half()
    d = ((hi - lo) / 15.0).half()
    t = (b.double() - m.double().unsqueeze(-1)) / torch.where(d > 0, d, 1).double().unsqueeze(-1)
    code = torch.where((d > 0).unsqueeze(-1), torch.round(t).clamp(0, 15), 0).to(torch.uint8)
    return code, d, m


def _pack(code, d, m, value_plane):
    """[seqs][rows][kv_heads][blocks][32] codes as the cache holds them: per sequence a plane of nibbles and one of (scale,
    minimum) pairs, both [kv_heads][rows].  A row's nibbles are grouped for the lane that multiplies them: for keys the
    8 channels 8 c .. 8 c + 7 of every block lie together for c = 0..3, for values the 4 channels 4 g .. 4 g + 3 for
    g = 0..7; inside a group two channels to a byte, the lower one in the low nibble."""
    s = code.shape[0]
    by = (code[..., 0::2] | (code[..., 1::2] << 4)).transpose(1, 2)                      # [seqs][heads][rows][blocks][16]
    groups, size = (8, 2) if value_plane else (4, 4)
    by = by.unflatten(-1, (groups, size)).transpose(-2, -3).reshape(s, -1)
    par = torch.stack([d, m], -1).transpose(1, 2).reshape(s, -1).view(torch.uint8)
    whole = torch.cat([by, par], 1)
    return torch.nn.functional.pad(whole, (0, -whole.shape[1] % 16)).contiguous()           # a sequence begins at 16 bytes


def _unpack(buf, rows, kv_heads, dim, value_plane):
    """The codes, scales and minima of a packed cache, [seqs][rows][kv_heads][blocks]..."""
    s, nb = buf.shape[0], dim // BLOCK
    cut = kv_heads * rows * dim // 2
    groups, size = (8, 2) if value_plane else (4, 4)
    by = buf[:, :cut].reshape(s, kv_heads, rows, groups, nb, size).transpose(-2, -3).reshape(s, kv_heads, rows, nb, 16)
    code = torch.stack([by & 15, by >> 4], -1).flatten(-2).transpose(1, 2)
    par = buf[:, cut:cut + kv_heads * rows * dim // 8].contiguous().view(torch.float16).reshape(s, kv_heads, rows, nb, 2).transpose(1, 2)
    return code, par[..., 0], par[..., 1]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    c, S, cap, H, D = case, case["seqs"], case["capacity"], case["kv_heads"], case["dim"]
    st = {"case": c}
    if c["op"] == "store":
        st["new_k"], st["new_v"] = _rows(gen, (S, c["tokens"], H), D), _rows(gen, (S, c["tokens"], H), D)
        if c["bits"] == 4:
            st["k"] = torch.zeros(S, -(-H * cap * (D // 2 + D // 8) // 16) * 16, dtype=torch.uint8, device="cuda")
        else:
            st["k"] = torch.zeros(S, cap, H, D, dtype=torch.float16, device="cuda")
        st["v"] = torch.zeros_like(st["k"])
        st["n_keys"] = torch.zeros(S, dtype=torch.int32, device="cuda")
        return st
    k, v = _rows(gen, (S, cap, H), D), _rows(gen, (S, cap, H), D)
    if c["bits"] == 4:
        st["k"], st["v"] = _pack(*_quantize(k), False), _pack(*_quantize(v), True)
    else:
        st["k"], st["v"] = k.half(), v.half()
    del k, v
    if c["op"] == "attend":
        N = c["tokens"]
        n = torch.full((S,), cap, dtype=torch.int32, device="cuda")
        if c["ragged"]:
            n = (cap * (0.4 + 0.6 * torch.rand(S, generator=gen, device="cuda"))).ceil().int().clamp(1, cap)
        st["n_keys"] = n
        st["q"] = torch.randn(S, N, c["heads"], D, generator=gen, device="cuda")
        if c["prefix"]:
            st["prefix"] = torch.full((S,), c["prefix"], dtype=torch.int32, device="cuda")
        if c["docs"]:
            # documents of unequal length, one behind the other; a query belongs to the document at its position
            ends = torch.sort(torch.randint(0, cap, (S, c["docs"]), generator=gen, device="cuda"), 1).values
            st["k_doc"] = (torch.arange(cap, device="cuda") >= ends.unsqueeze(-1)).sum(1).int().contiguous()
            at = (n.unsqueeze(1) - N + torch.arange(N, device="cuda")).clamp(min=0).long()
            st["q_doc"] = torch.gather(st["k_doc"], 1, at).contiguous()
        if c["mask"]:
            hide = torch.rand(S, N, cap, generator=gen, device="cuda") < 0.3
            hide |= torch.rand(S, N, 1, generator=gen, device="cuda") < 0.1                # padding rows see nothing
            bias = torch.randn(S, N, cap, generator=gen, device="cuda")
            pad = (cap + 7) // 8 * 8                                                        # rows at 16-byte strides
            st["mask"] = torch.full((S, N, pad), -math.inf, dtype=torch.float16, device="cuda")
            st["mask"][:, :, :cap] = torch.where(hide, -math.inf, bias)
        if c["weights"]:
            st["weights"] = torch.rand(S, H, cap, generator=gen, device="cuda")
        return st
    # a cache that eviction has been at before: positions out of order, weights as accumulated over many steps
    full = cap if c["op"] == "evict" else c["keep"]
    order = torch.argsort(torch.rand(S, H, full, generator=gen, device="cuda"), dim=-1).int()
    st["positions"] = torch.zeros(S, H, cap, dtype=torch.int32, device="cuda")
    st["positions"][:, :, :full] = order
    st["weights"] = torch.zeros(S, H, cap, device="cuda")
    st["weights"][:, :, :full] = torch.exp(2.0 * torch.randn(S, H, full, generator=gen, device="cuda"))
    st["n_keys"] = torch.full((S,), full, dtype=torch.int32, device="cuda")
    st["next_pos"] = torch.full((S,), full, dtype=torch.int32, device="cuda")
    if c["op"] == "step":
        st["new_k"], st["new_v"] = _rows(gen, (S, 1, H), D), _rows(gen, (S, 1, H), D)
    else:
        st["as_was"] = (st["n_keys"].clone(), st["positions"].clone(), st["weights"].clone())
    return st


# ---- one pass -----------------------------------------------------------------------------------------------------

def _handle(st):
    """The cache object that a program keeps for these buffers."""
    if "handle" not in st:
        from kernelcore_b200 import kvcache
        c = st["case"]
        st["handle"] = kvcache.KVCache(st["k"], st["v"], kv_heads=c["kv_heads"], head_dim=c["dim"], capacity=c["capacity"], bits=c["bits"],
                                       n_keys=st["n_keys"], next_pos=st.get("next_pos"), positions=st.get("positions"), weights=st.get("weights"))
        if c["op"] == "attend":
            st["attend"] = kvcache.Attention(st["handle"], n_tokens=c["tokens"], heads=c["heads"], scale=c["dim"] ** -0.5, softcap=c["softcap"],
                                             max_bias=c["max_bias"], causal=c["causal"], prefix=st.get("prefix"), q_doc=st.get("q_doc"),
                                             k_doc=st.get("k_doc"), mask=st.get("mask"), accumulate=c["weights"])
            st["out"] = torch.empty_like(st["q"])
    return st["handle"]


def _values(st, which):
    """Keys or values as fp32 [seqs][capacity][kv_heads][dim]."""
    c = st["case"]
    if c["bits"] == 16:
        return st[which].float()
    code, d, m = _unpack(st[which], c["capacity"], c["kv_heads"], c["dim"], which == "v")
    return (d.float().unsqueeze(-1) * code.float() + m.float().unsqueeze(-1)).flatten(-2)


def _slopes(heads, max_bias):
    """Distance-bias slopes: a geometric sequence over the largest power of two of heads, the odd steps of a finer one for the rest."""
    p2 = 1 << (heads.bit_length() - 1)
    h = torch.arange(heads, dtype=torch.float64, device="cuda")
    e = torch.where(h < p2, (h + 1) * (max_bias / p2), (2 * (h - p2) + 1) * (max_bias / 2 / p2))
    return torch.exp2(-e)


def _plain_attend(st):
    c = st["case"]
    S, N, D, H, T = c["seqs"], c["tokens"], c["dim"], c["kv_heads"], c["capacity"]
    G = c["heads"] // H
    k, v = _values(st, "k"), _values(st, "v")
    q = st["q"].reshape(S, N, H, G, D).permute(0, 2, 3, 1, 4).reshape(S, H, G * N, D)
    z = torch.matmul(q, k.permute(0, 2, 3, 1)).reshape(S, H, G, N, T) * (D ** -0.5)
    if c["softcap"]:
        z = c["softcap"] * torch.tanh(z / c["softcap"])
    t = torch.arange(T, device="cuda")
    q_pos = st["n_keys"].unsqueeze(1) - N + torch.arange(N, device="cuda")                 # [S][N]
    if c["max_bias"]:
        far = (q_pos.unsqueeze(-1) - t).abs().float()
        z = z - _slopes(c["heads"], c["max_bias"]).float().reshape(H, G, 1, 1) * far.reshape(S, 1, 1, N, T)
    seen = (t < st["n_keys"].unsqueeze(-1)).unsqueeze(1).expand(S, N, T)
    if c["causal"]:
        early = t <= q_pos.unsqueeze(-1)
        if c["prefix"]:
            early = early | (t < st["prefix"].reshape(S, 1, 1))
        seen = seen & early
    if c["docs"]:
        seen = seen & (st["q_doc"].unsqueeze(-1) == st["k_doc"].unsqueeze(1))
    if c["mask"]:
        z = z + st["mask"][:, :, :T].float().reshape(S, 1, 1, N, T)
    z = torch.where(seen.reshape(S, 1, 1, N, T), z, -math.inf)
    top = z.amax(-1, keepdim=True)
    p = torch.exp(z - torch.where(torch.isfinite(top), top, 0))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, 1)
    out = torch.matmul(p.reshape(S, H, G * N, T), v.permute(0, 2, 1, 3)).reshape(S, H, G, N, D).permute(0, 3, 1, 2, 4).reshape(S, N, c["heads"], D)
    if not c["weights"]:
        return {"out": out}
    st["weights"] += p.sum((2, 3))
    return {"out": out, "weights": st["weights"]}


def _plain_store(st):
    c = st["case"]
    N, cap = c["tokens"], c["capacity"]
    st["n_keys"].fill_(N)
    if c["bits"] == 16:
        st["k"][:, :N], st["v"][:, :N] = st["new_k"].half(), st["new_v"].half()
    else:
        kc, kd, km = _unpack(st["k"], cap, c["kv_heads"], c["dim"], False)
        vc, vd, vm = _unpack(st["v"], cap, c["kv_heads"], c["dim"], True)
        nk, nv = _quantize(st["new_k"]), _quantize(st["new_v"])
        join = lambda new, old: torch.cat([new, old[:, N:]], 1)  # noqa: E731
        st["k"].copy_(_pack(join(nk[0], kc), join(nk[1], kd), join(nk[2], km), False))
        st["v"].copy_(_pack(join(nv[0], vc), join(nv[1], vd), join(nv[2], vm), True))
    return {"k": _values(st, "k")[:, :N], "v": _values(st, "v")[:, :N], "n_keys": st["n_keys"]}


def _plain_evict(st):
    """Every sequence holds more than `keep` rows here."""
    c = st["case"]
    S, H, keep, n = c["seqs"], c["kv_heads"], c["keep"], st["full"]
    pos, w = st["positions"][:, :, :n], st["weights"][:, :, :n]
    rank = torch.where(pos >= (st["next_pos"] - c["recent"]).reshape(S, 1, 1), math.inf, w)
    order = torch.argsort(rank, dim=-1, descending=True, stable=True)                        # ties: the lowest slot first
    kept = torch.zeros(S, H, n, dtype=torch.bool, device="cuda").scatter_(-1, order[..., :keep], True)
    # slot -> where it comes from: itself, or the j-th kept row behind `keep` for the j-th free slot
    tail = torch.sort(torch.where(kept[..., keep:], torch.arange(keep, n, device="cuda"), n), -1).values
    tail = torch.nn.functional.pad(tail, (0, max(0, keep - tail.shape[-1])), value=n)
    nth = (torch.cumsum((~kept[..., :keep]).int(), -1) - 1).clamp(min=0)
    src = torch.where(kept[..., :keep], torch.arange(keep, device="cuda"), torch.gather(tail, -1, nth))
    for_rows = src.transpose(1, 2).unsqueeze(-1).expand(S, keep, H, c["dim"])
    st["k"][:, :keep] = torch.gather(st["k"][:, :n], 1, for_rows)
    st["v"][:, :keep] = torch.gather(st["v"][:, :n], 1, for_rows)
    st["positions"][:, :, :keep], st["weights"][:, :, :keep] = torch.gather(pos, -1, src), torch.gather(w, -1, src)
    st["n_keys"].fill_(keep)


def _cache_state(st):
    """The rows in use (those behind them are nobody's), and the arrays beside them."""
    keep = st["case"]["keep"]
    return {"k": st["k"][:, :keep], "v": st["v"][:, :keep], "positions": st["positions"][:, :, :keep], "weights": st["weights"][:, :, :keep],
            "n_keys": st["n_keys"]}


def run(st):
    c = st["case"]
    if c["op"] == "attend":
        if not own:
            return _plain_attend(st)
        _handle(st)
        out = st["attend"](st["q"], st["out"])
        return {"out": out, "weights": st["weights"]} if c["weights"] else {"out": out}
    if c["op"] == "store":
        if not own:
            return _plain_store(st)
        cache = _handle(st)
        st["n_keys"].zero_()
        cache.append(st["new_k"], st["new_v"])
        k, v = cache.read(0, c["tokens"])
        return {"k": k, "v": v, "n_keys": st["n_keys"]}
    if c["op"] == "step":
        if own:
            cache = _handle(st)
            cache.append(st["new_k"], st["new_v"])
            cache.evict(c["keep"], c["recent"])
        else:
            st["full"] = c["keep"] + 1
            st["k"][:, c["keep"]], st["v"][:, c["keep"]] = st["new_k"][:, 0].half(), st["new_v"][:, 0].half()
            st["positions"][:, :, c["keep"]] = st["next_pos"].unsqueeze(-1)
            st["weights"][:, :, c["keep"]] = 0.0
            st["next_pos"] += 1
            _plain_evict(st)
        return _cache_state(st)
    # the rows stay where the last pass left them; their counts, positions and weights are as before it
    st["n_keys"].copy_(st["as_was"][0])
    st["positions"].copy_(st["as_was"][1])
    st["weights"].copy_(st["as_was"][2])
    if own:
        _handle(st).evict(c["keep"], c["recent"])
    else:
        st["full"] = c["capacity"]
        _plain_evict(st)
    return _cache_state(st)


# ---- what a pass cannot do without --------------------------------------------------------------------------------

def _pairs(c, n):
    """Visible (query, key) pairs of a sequence with n rows; documents are taken as of equal length."""
    N = c["tokens"]
    if c["mask"]:
        return 0.63 * N * n
    if not c["causal"]:
        return float(N * n)
    first = n - N + 1                                                                      # keys that the first query sees
    lo = max(0, -(first - 1))                                                              # queries in front of the sequence see none
    seen = (N - lo) * (max(first, 1) + n) / 2.0
    if c["prefix"]:
        p = min(c["prefix"], n)
        seen += sum(max(0, p - max(0, first + i)) for i in range(N))
    if c["docs"]:
        seen = min(seen, max(N - lo, seen / (c["docs"] + 1))) if N > 1 else seen / (c["docs"] + 1)
    return seen


def work(case):
    c = case
    S, H, D = c["seqs"], c["kv_heads"], c["dim"]
    row = H * (2 * D if c["bits"] == 16 else D // 2 + D // 8)                              # bytes of one token's keys (or values)
    if c["op"] == "attend":
        n = int(0.7 * c["capacity"]) if c["ragged"] else c["capacity"]
        n = max(1, n)
        used = n / (c["docs"] + 1) if c["docs"] and c["tokens"] == 1 else n
        b = S * (used * 2 * row + 2 * 4 * c["tokens"] * c["heads"] * D)
        b += S * (2 * c["tokens"] * n if c["mask"] else 0) + (S * H * n * 8 if c["weights"] else 0)
        return {"bytes": b, "flops": 4.0 * D * c["heads"] * S * _pairs(c, n)}
    if c["op"] == "store":
        values = 2.0 * S * c["tokens"] * H * D
        return {"bytes": values * 4 + 2 * 2 * S * c["tokens"] * row + values * 4, "flops": 8 * values}
    full = c["capacity"] if c["op"] == "evict" else c["keep"] + 1
    moved = c["keep"] * (full - c["keep"]) / full                                          # kept rows that sit behind `keep`
    b = S * H * full * 8 + S * moved * (2 * 2 * row + H * 16) + (S * 2 * (4 * H * D + row) if c["op"] == "step" else 0)
    return {"bytes": b, "flops": S * H * full * 4.0}


# ---- the definition in 64 bits --------------------------------------------------------------------------------------

def _exact_rows(st, which):
    """Stored values in 64 bits, read nibble by nibble from the description of the format."""
    c = st["case"]
    if c["bits"] == 16:
        return st[which].double()
    S, cap, H, D = c["seqs"], c["capacity"], c["kv_heads"], c["dim"]
    nb, ch = D // BLOCK, torch.arange(D, device="cuda")
    b, i = ch // BLOCK, ch % BLOCK
    byte = ((i // 8) * nb + b) * 4 + (i % 8) // 2 if which == "k" else ((i // 4) * nb + b) * 2 + (i % 4) // 2
    rows = st[which][:, :H * cap * D // 2].reshape(S, H, cap, D // 2)[..., byte].int()
    code = (rows >> (4 * (i % 2))) & 15
    par = st[which][:, H * cap * D // 2:H * cap * (D // 2 + D // 8)].contiguous().view(torch.float16).reshape(S, H, cap, nb, 2).double()
    return (par[..., 0][..., b] * code + par[..., 1][..., b]).transpose(1, 2)


def _exact_attend(st):
    c = st["case"]
    S, N, D, H, cap = c["seqs"], c["tokens"], c["dim"], c["kv_heads"], c["capacity"]
    G = c["heads"] // H
    k, v = _exact_rows(st, "k"), _exact_rows(st, "v")
    slope = _slopes(c["heads"], c["max_bias"])
    out = torch.zeros(S, N, c["heads"], D, dtype=torch.float64, device="cuda")
    w = st["weights"].double() if c["weights"] else None
    for s in range(S):
        n = int(st["n_keys"][s])
        t = torch.arange(n, device="cuda")
        at = n - N + torch.arange(N, device="cuda")
        hide = torch.zeros(N, n, dtype=torch.bool, device="cuda")
        if c["causal"]:
            hide |= (t[None] > at[:, None]) & (t[None] >= c["prefix"])
        if c["docs"]:
            hide |= st["q_doc"][s][:, None] != st["k_doc"][s][None, :n]
        add = st["mask"][s][:, :n].double() if c["mask"] else 0.0
        for head in range(c["heads"]):
            z = (st["q"][s, :, head].double() @ k[s, :n, head // G].T) / math.sqrt(D)
            if c["softcap"]:
                z = c["softcap"] * torch.tanh(z / c["softcap"])
            if c["max_bias"]:
                z = z - slope[head] * (at[:, None] - t[None]).abs()
            z = (z + add).masked_fill(hide, -math.inf)
            p = torch.nan_to_num(torch.softmax(z, -1), nan=0.0)
            out[s, :, head] = p @ v[s, :n, head // G]
            if w is not None:
                w[s, head // G, :n] += p.sum(0)
    return {"out": out} if w is None else {"out": out, "weights": w}


def _exact_store(st):
    c = st["case"]
    got = {}
    for which in ("k", "v"):
        x = st["new_" + which]
        if c["bits"] == 16:
            got[which] = x.half().double()
            continue
        x = x.reshape(*x.shape[:-1], -1, BLOCK)
        least, most = torch.aminmax(x, dim=-1, keepdim=True)
        d, m = ((most - least) / 15.0).half().double(), least.half().double()              # the format's scales are defined in 32 bits
        code = torch.where(d > 0, torch.round((x.double() - m) / d), 0.0).clamp(0, 15)
        got[which] = (code * d + m).flatten(-2)
    return {"k": got["k"], "v": got["v"], "n_keys": None}


def exact(case, seed):
    if case["op"] in ("step", "evict"):
        return None                                                                         # rows are moved, nothing is computed
    if case["op"] == "attend" and case["seqs"] * case["heads"] > 4096:
        return None
    st = prepare(case, seed)
    return _exact_attend(st) if case["op"] == "attend" else _exact_store(st)
