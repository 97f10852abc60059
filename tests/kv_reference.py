"""Plain 64-bit forms of the KV-cache operators, for tests: the 4-bit format code by code, attention head by head, eviction
by sorting."""
import math

import numpy as np
import torch

F16_MAX = 65504.0


def q4_block_values(x):
    """The values a 4-bit cache stands for, [..., 32 * blocks] fp32 in, fp64 out.  Scales are defined by fp32 steps."""
    x = np.nan_to_num(np.asarray(x, np.float32), nan=0.0, posinf=F16_MAX, neginf=-F16_MAX)
    x = np.clip(x, -F16_MAX, F16_MAX).astype(np.float32)
    b = x.reshape(*x.shape[:-1], -1, 32)
    lo, hi = b.min(-1, keepdims=True), b.max(-1, keepdims=True)
    m = lo.astype(np.float16).astype(np.float64)
    d = ((hi - lo).astype(np.float32) * np.float32(1 / 15)).astype(np.float16).astype(np.float64)
    code = np.where(d > 0, np.clip(np.rint((b.astype(np.float64) - m) / np.where(d > 0, d, 1)), 0, 15), 0)
    return (d * code + m).reshape(x.shape), code.astype(np.int64), d[..., 0], m[..., 0]


def q4_unpack(buf, kv_heads, dim, capacity, which):
    """(codes [cap][heads][dim], d, m [cap][heads][blocks]) of one sequence's bytes, nibble by nibble."""
    nb = dim // 32
    raw = np.asarray(buf, np.uint8)
    rows = raw[:kv_heads * capacity * dim // 2].reshape(kv_heads, capacity, dim // 2)
    code = np.zeros((capacity, kv_heads, dim), np.int64)
    for ch in range(dim):
        b, i = ch // 32, ch % 32
        byte = ((i // 8) * nb + b) * 4 + (i % 8) // 2 if which == "k" else ((i // 4) * nb + b) * 2 + (i % 4) // 2
        code[:, :, ch] = ((rows[:, :, byte] >> (4 * (i % 2))) & 15).T
    par = raw[kv_heads * capacity * dim // 2:][:kv_heads * capacity * dim // 8].copy().view(np.float16).reshape(kv_heads, capacity, nb, 2).transpose(1, 0, 2, 3)
    return code, par[..., 0].astype(np.float64), par[..., 1].astype(np.float64)


def slopes(heads, max_bias):
    h2 = 1 << int(math.floor(math.log2(heads)))
    return np.array([2.0 ** (-max_bias * (h + 1) / h2) if h < h2 else 2.0 ** (-max_bias / 2 * (2 * (h - h2) + 1) / h2) for h in range(heads)])


def attend(q, k, v, n_keys, *, scale, softcap=0.0, max_bias=0.0, causal=True, prefix=None, q_pos=None, k_pos=None, next_pos=None, q_doc=None, k_doc=None,
           mask=None):
    """q [S][N][H][D], k, v [S][T][Hkv][D] (fp64 tensors); k_pos [S][Hkv][T].  Returns (out, weights [S][Hkv][T], tolerance [S][N][H]).

    The tolerance is the kernel's, from its arithmetic, in units of the largest |v| that a row sees.  With S1 = the largest
    scale * sum |q_c k_c| of a row (with a minimum and a scale per block, sum over the parts, at most 3 S1 for them) and
    u = 2^-24:
      score: operands carry 22 bits (2^-22 S1); D / 16 products of 16, hi and lo, each sum truncated to 24 bits: at most
             (D / 8 + 4) 2u S1; factors, cap and bias round a few times: 8 u (S1 + |bias| of the best slot + cap).
      weight: relative error of the score's error, of the exponential (2^-21) and of its split (2^-21).
      sum:    slots are added in blocks of 16 with truncation, at most 64 of them in a row and 16 joins: (64 + 16) 2u.
    A weighted mean moves by at most twice the largest relative error of its weights."""
    S, N, H, D = q.shape
    Hkv, T = k.shape[2], k.shape[1]
    G = H // Hkv
    u = 2.0 ** -24
    out = torch.zeros(S, N, H, D, dtype=torch.float64, device=q.device)
    w = torch.zeros(S, Hkv, T, dtype=torch.float64, device=q.device)
    tol = torch.zeros(S, N, H, dtype=torch.float64, device=q.device)
    sl = slopes(H, max_bias) if max_bias else np.ones(H)
    for s in range(S):
        n = int(n_keys[s])
        t = torch.arange(n, device=q.device)
        qp = q_pos[s].long() if q_pos is not None else (int(next_pos[s]) if next_pos is not None else n) - N + torch.arange(N, device=q.device)
        for h in range(H):
            kv = h // G
            kp = (k_pos[s, kv, :n] if k_pos is not None else t).long()
            see = torch.ones(N, n, dtype=torch.bool, device=q.device)
            if causal:
                see &= (kp[None] <= qp[:, None]) | (kp[None] < (int(prefix[s]) if prefix is not None else -2 ** 31))
            if q_doc is not None:
                see &= q_doc[s][:, None] == k_doc[s][None, :n]
            kk, vv = k[s, :n, kv], v[s, :n, kv]
            z = (q[s, :, h] @ torch.nan_to_num(kk).T) * scale
            s1 = (q[s, :, h].abs() @ torch.nan_to_num(kk).abs().T) * abs(scale)
            if softcap:
                z = softcap * torch.tanh(z / softcap)
            bias = torch.zeros(N, n, dtype=torch.float64, device=q.device)
            if mask is not None:
                bias = sl[h] * mask[s, :, :n].double()
            elif max_bias:
                bias = -sl[h] * (qp[:, None] - kp[None]).abs().double()
            z = z + bias
            see = see & (z != -math.inf)
            z = torch.where(see, z, -math.inf)
            p = torch.nan_to_num(torch.softmax(z, -1), nan=0.0) if n else torch.zeros(N, 0, dtype=torch.float64, device=q.device)
            vz = torch.where(see.any(0)[:, None], vv, 0.0)
            out[s, :, h] = p @ torch.nan_to_num(vz)
            w[s, kv, :n] += p.sum(0)
            if n:
                big = torch.where(see, s1, 0.0).amax(-1)
                best = bias.gather(1, torch.where(see, z, -math.inf).argmax(-1, keepdim=True))[:, 0].nan_to_num(posinf=0, neginf=0).abs()
                dz = 3 * big * (4 + 2 * (D / 8 + 4)) * u + 8 * u * (big + best + softcap)
                vmax = torch.where(see, torch.nan_to_num(vv).abs().amax(-1)[None], 0.0).amax(-1)
                tol[s, :, h] = vmax * (2 * (dz + 2 * 8 * u) + 80 * 2 * u)
    return out, w, tol


def evict(rows, positions, weights, n_keys, next_pos, keep, recent):
    """rows: list of arrays [S][T][Hkv]...; all modified in place, as are positions and weights [S][Hkv][T] and n_keys."""
    S, Hkv, _ = positions.shape
    for s in range(S):
        n = int(n_keys[s])
        if n <= keep:
            continue
        for h in range(Hkv):
            def rank(t):
                if positions[s, h, t] >= int(next_pos[s]) - recent:
                    return (0, 0.0, t)
                x = float(weights[s, h, t])
                return (2, 0.0, t) if x != x else (1, -x, t)
            kept = sorted(sorted(range(n), key=rank)[:keep])
            holes = sorted(set(range(keep)) - set(kept))
            tails = [t for t in kept if t >= keep]
            assert len(holes) == len(tails)
            for a, b in zip(tails, holes):
                for r in rows:
                    r[s, b, h] = r[s, a, h]
                positions[s, h, b], weights[s, h, b] = positions[s, h, a], weights[s, h, a]
        n_keys[s] = keep
