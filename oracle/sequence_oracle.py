"""Attention over token sequences in 64 bits on the CPU, with bounds for the rounding errors of the kernels.

Plain restatements of functional.qk_norm_rotary and functional.band_attention (test infrastructure only).  Next to each
result stands how far a kernel may be from it: u = finfo(dtype).eps / 2 for every rounding to the tensors' type, and a
multiple of 2^-24 for the arithmetic in fp32.
"""
import math

import torch

F = 2.0 ** -24


def unit(dtype):
    return torch.finfo(dtype).eps / 2


def rotary(x, weight, angles, pairs, eps, interleaved):
    """x [B, L, H, D], angles [B or 1, L, pairs] radians -> the normalised and turned rows, in x's dtype (double)"""
    u = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    if weight is not None:
        u = u * weight
    c, s = torch.cos(angles).unsqueeze(2), torch.sin(angles).unsqueeze(2)
    first = torch.arange(pairs) * 2 if interleaved else torch.arange(pairs)
    second = first + (1 if interleaved else pairs)
    parts = [None] * x.shape[-1]
    for n, (i, j) in enumerate(zip(first.tolist(), second.tolist())):
        parts[i] = u[..., i] * c[..., n] - u[..., j] * s[..., n]
        parts[j] = u[..., i] * s[..., n] + u[..., j] * c[..., n]
    return torch.stack([u[..., i] if t is None else t for i, t in enumerate(parts)], -1)


def visible(Lq, Lk, qn, kn, left, right, sinks):
    p = (kn - qn) + torch.arange(Lq).unsqueeze(1)
    j = torch.arange(Lk).unsqueeze(0)
    vis = (j < kn) & (torch.arange(Lq).unsqueeze(1) < qn)
    if right is not None:
        vis = vis & (j <= p + right)
    if left is not None:
        vis = vis & ((j >= p - left) | (j < sinks))
    return vis, j - p


def attention(q, k, v, left, right, sinks, scale, q_lens=None, k_lens=None, table=None, buckets=None, dout=None, dtype=torch.float32,
              table_grad=True, score_roundings=None, whole_delta=False):
    """double tensors [B, L, H, D]; returns {"out": (value, bound), and with dout "dq", "dk", "dv", "dtable" likewise}.

    Bounds, entry by entry.  Scores: a sum of D products in fp32 and its scaling are off by at most
    (D + 4) F scale sum|q k|, the bias and the exponential add F each time their size (|x| F) and a few F, so a
    probability is off by the relative e = 2 F ((D + 4) smax + |x|max + n + 16) (n: the denominator's terms), and, where
    it enters a product in 16 bits, by u more.  The result then carries (u + e) sum P |v| and its own rounding u |out|.
    delta = dout . out inherits the result's error (where a table's gradient is wanted: that of the fp32 copy that the
    kernels keep then), and
    dS = P (dP - delta) carries u |dS| + P |delta's error| + e P (|dP| + |delta|) + D F P sum|dout v|.

    score_roundings: in the place of D + 4, for q and k whose products and sums are exact in fp32.
    whole_delta: the result's own rounding does not enter delta (what it leaves behind is kept, rounded: u^2), and the rounded
    probabilities are divided by their own sum: to first order delta is then off by sum_j P_j u_j (dP_j - delta), u_j the
    rounding of P_j, at most u sum |dS|; (1 + 4 u) for the second.  An error e of P itself multiplies dP - delta.  The same sum
    makes the backward's P = p / sum p (1 + u_j), off by the relative sum P_j u_j of at most u (1 + 2 u) in a whole row."""
    B, Lq, Hq, D = q.shape
    Lk, Hkv = k.shape[1:3]
    u = unit(dtype) if dtype != torch.float32 else 0.0     # rounding of probabilities and of dS
    uo = unit(dtype)                                        # rounding of results
    M = None if buckets is None else buckets.numel() // 2
    out, b_out = torch.zeros_like(q), torch.zeros_like(q)
    res = {n: [torch.zeros_like(t), torch.zeros_like(t)] for n, t in (("dq", q), ("dk", k), ("dv", v))}
    if table is not None:
        res["dtable"] = [torch.zeros_like(table), torch.zeros_like(table)]
    for b in range(B):
        kn = Lk if k_lens is None else min(max(int(k_lens[b]), 0), Lk)
        qn = Lq if q_lens is None else min(max(int(q_lens[b]), 0), Lq)
        vis, rel = visible(Lq, Lk, qn, kn, left, right, sinks)
        for h in range(Hq):
            g = h // (Hq // Hkv)
            Q, Kb, V = q[b, :, h], k[b, :, g].clone(), v[b, :, g].clone()
            Kb[kn:], V[kn:] = 0, 0
            x = Q @ Kb.T * scale
            xabs = Q.abs() @ Kb.abs().T * scale
            if table is not None:
                bucket = buckets.long().clamp(0, table.shape[0] - 1)[rel.clamp(-M, M) + M]
                x = x + table[bucket, h]
                xabs = xabs + table[bucket, h].abs()
            x = x.masked_fill(~vis, -math.inf)
            m = x.amax(-1, keepdim=True) if Lk else torch.full((Lq, 1), -math.inf, dtype=q.dtype)
            e = torch.exp(x - m.masked_fill(m == -math.inf, 0.0))
            tot = e.sum(-1, keepdim=True)
            P = e / tot.masked_fill(tot == 0, 1.0)
            O = P @ V
            A = P @ V.abs()
            rel_e = (2 * F * ((D + 4 if score_roundings is None else score_roundings) * xabs.masked_fill(~vis, 0).amax(-1, keepdim=True) + vis.sum(-1, keepdim=True) + 16)
                     if Lk else torch.zeros(Lq, 1, dtype=q.dtype))
            out[b, :, h] = O
            b_out[b, :, h] = (u + rel_e) * A + uo * O.abs() + F * A * 8
            if dout is None:
                continue
            G = dout[b, :, h].clone()
            G[qn:] = 0
            dP = G @ V.T
            absGV = G.abs() @ V.abs().T
            delta = (G * O).sum(-1, keepdim=True)
            dS = P * (dP - delta)
            # how far delta may be off: with the rounded result, and with the fp32 copy that a wanted table gradient keeps
            # (probabilities in three parts of 8 bits: u^3)
            def ds_bound(up, ur):
                d_delta = (G.abs() * ((up + rel_e) * A + ur * O.abs() + 8 * F * A)).sum(-1, keepdim=True) + (D + 4) * F * (G * O).abs().sum(-1, keepdim=True)
                return P * d_delta + rel_e * P * (dP.abs() + delta.abs()) + (D + 8) * F * P * absGV
            exact = table is not None and table_grad and dtype != torch.float32
            raw = ds_bound(u ** 3, 0.0) if exact else ds_bound(u, uo)
            if whole_delta and not exact:
                d_delta = (u * (1 + 4 * u) * dS.abs().sum(-1, keepdim=True)
                           + (G.abs() * ((rel_e + 8 * F) * A + u * u * O.abs())).sum(-1, keepdim=True) + (D + 4) * F * (G * O).abs().sum(-1, keepdim=True))
                raw = P * d_delta + (rel_e + u * (1 + 2 * u)) * (1 + u) * dS.abs() + (D + 8) * F * P * absGV
            bS = u * dS.abs() + raw
            nrow = Lq * (Hq // Hkv)
            res["dq"][0][b, :, h] = dS @ Kb * scale
            res["dq"][1][b, :, h] = (bS + (Lk + 8) * F * dS.abs()) @ Kb.abs() * scale
            res["dk"][0][b, :, g] += dS.T @ Q * scale
            res["dk"][1][b, :, g] += (bS + (nrow + 8) * F * dS.abs()).T @ Q.abs() * scale
            res["dv"][0][b, :, g] += P.T @ G
            res["dv"][1][b, :, g] += (P * (u + rel_e + (nrow + 8) * F + (u * (1 + 2 * u) if whole_delta else 0.0))).T @ G.abs()
            if table is not None:
                n = table.shape[0]
                flat = bucket.flatten()
                res["dtable"][0][:, h] += torch.zeros(n, dtype=q.dtype).index_add_(0, flat, dS.flatten())
                # (a bucket's sum runs over at most 16 terms in a register, the tiles of a row block, the blocks)
                res["dtable"][1][:, h] += torch.zeros(n, dtype=q.dtype).index_add_(0, flat, (raw + (Lk + B * Lq / 128 + 600) * F * dS.abs()).flatten())
    for n in ("dq", "dk", "dv"):
        res[n][1] += uo * res[n][0].abs()
    got = {"out": (out, b_out)}
    if dout is not None:
        got.update({n: tuple(t) for n, t in res.items()})
    return got


def bucket_map(buckets, distance, causal):
    """the module's map restated with logarithms (only compared away from the borders, where whole numbers decide)"""
    side = buckets if causal else buckets // 2
    near = side // 2
    out = []
    for rel in range(-distance, distance + 1):
        n = max(-rel, 0) if causal else abs(rel)
        b = n if n < near else min(side - 1, near + int(math.log(n / near) / math.log(distance / near) * (side - near) + 1e-9))
        out.append(b + (side if rel > 0 and not causal else 0))
    return out
