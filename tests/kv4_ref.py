"""Plain 64-bit reference of the paged 4-bit KV cache (numpy / torch on the CPU or GPU): the number
format from its definition, the page layout word by word, the plan as a loop over requests, and
attention over the values that the cache holds, with the error bounds the tests use."""
from __future__ import annotations

import math

import numpy as np
import torch

FLOOR = {torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -21}
ROUND = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}  # largest relative rounding error (half a step)


def quantise(x):
    """codes (..., D), scale and zero point (..., D / 64), float64, of 16-bit values x."""
    dt = x.dtype
    x = x.double().unflatten(-1, (-1, 64))
    hi, lo = x.amax(-1, keepdim=True).clamp(min=0), x.amin(-1, keepdim=True).clamp(max=0)
    m, e = torch.frexp((hi - lo) / 15)
    s = torch.ldexp(torch.ceil(m * 16) / 16, e).clamp(min=FLOOR[dt])
    z = torch.floor(0.5 - lo / s)
    c = torch.minimum(torch.floor(x / s + 0.5) + z, torch.full_like(x, 15))
    far = s * (c - z)
    most = torch.finfo(dt).max
    c = c - (far > most).double() + (far < -most).double()
    bad = ~torch.isfinite(x).all(-1, keepdim=True)
    c, z = c.masked_fill(bad, 0), z.masked_fill(bad, 0)
    return c.flatten(-2), s.masked_fill(bad, math.nan).squeeze(-1), z.squeeze(-1)


def values(c, s, z):
    c = c.unflatten(-1, (-1, 64))
    return ((c - z[..., None]) * s[..., None]).flatten(-2)


def unpack(pages, num_kv_heads, head_dim, page_size):
    """float64 values (num_pages * page_size slots, 2, H_KV, D) of a cache's pages, word by word."""
    raw = pages.cpu().numpy()
    P, groups = raw.shape[0], head_dim // 64
    raw = raw.reshape(P, 2, num_kv_heads, page_size // 16, groups * 544)
    out = np.zeros((P * page_size, 2, num_kv_heads, head_dim))
    with np.errstate(invalid="ignore"):
        for r in range(16):
            t, half = (r % 8) // 2, r // 8
            for g in range(groups):
                for kind in range(2):
                    at = groups * 512 + g * 32
                    at += 2 * ((r % 8) * 2 + half) if kind == 0 else 2 * (t * 4 + half * 2 + r % 2)
                    meta = raw[..., at:at + 2].copy().view("<u2")[:, kind, :, :, 0].astype(np.uint32)
                    s = ((meta & 0xFFF0) << 16).astype(np.uint32).view(np.float32).astype(np.float64)
                    z = (meta & 15).astype(np.float64)
                    for j in range(8):
                        if kind == 0:
                            at = g * 512 + ((r % 8) * 4 + j // 2) * 16 + half * 8 + (j % 2) * 4
                            order = [0, 2, 4, 6, 1, 3, 5, 7]
                        else:
                            at = g * 512 + (t * 8 + (j ^ (2 * t))) * 16 + (half * 2 + r % 2) * 4
                            order = range(8)
                        word = raw[..., at:at + 4].copy().view("<u4")[:, kind, :, :, 0]
                        for nib, dim in enumerate(order):
                            v = s * (((word >> (4 * nib)) & 15) - z)  # (P, H, blocks)
                            for blk in range(page_size // 16):
                                slots = np.arange(P) * page_size + blk * 16 + r
                                out[slots, kind, :, g * 64 + j * 8 + dim] = v[:, :, blk]
    return out


def plan(kv_lens, new_lens, table, free, state, page, max_new):
    """The step's plan by a loop over the requests (numpy int64)."""
    B, cols = table.shape
    head, count = int(state[0]), int(state[1])
    F = free.size
    out = dict(block_table=np.full((B, cols), -1), kv_lens=np.zeros(B, int), new_lens=np.zeros(B, int),
               slot_map=np.full((B, max_new), -1), positions=np.full((B, max_new), -1), accepted=np.zeros(B, int))
    ring, wanted, taken, back = free.copy(), 0, 0, 0
    for b in range(B):
        n, used = int(kv_lens[b]), -(-int(kv_lens[b]) // page)
        add = int(new_lens[b])
        if add < 0:
            for j in range(used):
                ring[(head + count + back) % F] = table[b, j]
                back += 1
            out["accepted"][b] = 1
            continue
        out["block_table"][b, :used] = table[b, :used]
        out["kv_lens"][b] = n
        if add > max_new or n + add > cols * page:
            continue
        need = -(-(n + add) // page) - used
        wanted += need
        if need and wanted > count:
            continue
        for j in range(need):
            out["block_table"][b, used + j] = free[(head + taken) % F]
            taken += 1
        out["accepted"][b], out["new_lens"][b], out["kv_lens"][b] = 1, add, n + add
        for i in range(add):
            out["positions"][b, i] = n + i
            out["slot_map"][b, i] = out["block_table"][b, (n + i) // page] * page + (n + i) % page
    out["free_pages"] = ring
    out["free_state"] = np.array([(head + taken) % F, count - taken + back])
    return out


def attention(q, k, v, kv_lens, q_lens, causal, window, scale):
    """O, LSE and an element-wise error bound in float64. k, v: values (B, H_KV, L, D) float64 that the
    cache holds (padding ignored); q 16-bit (B, H_Q, N, D).

    The bound counts the roundings that the kernel makes to first order (u: half a step of the 16-bit type,
    e = 2^-23 a step of fp32):
      output       u |O|;
      s * P        u per key: u sum_j P_j |v_j| (the rounded products cancel the offset exactly);
      scores       fp32 sums of up to D / 16 + groups + 8 steps of terms |q_d| s (16 + 15): a score is off by at most
                   e * steps * scale * 31 * sum_d |q_d| s, and P by twice that, relative; the query's 16-bit integers
                   are half a step off, 2^-16 of its row's largest value: 2^-16 * scale * max|q| * sum_d |k_d|;
      accumulation fp32 sums over keys of terms s P (F + 15), joined after every tile of up to 32 MMA steps: at
                   most e * 32 * (256 + 15) s P in a tile, and L / 16 + 64 steps of the joined sums (31 s P);
      exp2 and the joins of parts: 16 steps of fp32 relative to P."""
    B, Hq, N, D = q.shape
    G = Hq // k.shape[1]
    u, e = ROUND[q.dtype], 2.0 ** -23
    O = torch.zeros(B, Hq, N, D, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(O)
    lse = torch.full((B, Hq, N), -math.inf, dtype=torch.float64, device=q.device)
    for b in range(B):
        L, n = int(kv_lens[b]), int(q_lens[b])
        if n == 0 or L == 0:
            continue
        pos = L - n + torch.arange(n, device=q.device)[:, None]
        key = torch.arange(L, device=q.device)[None, :]
        ok = torch.ones(n, L, dtype=torch.bool, device=q.device)
        if causal:
            ok = key <= pos
            if window:
                ok &= key > pos - window
        kk = k[b, :, :L].repeat_interleave(G, 0)
        vv = v[b, :, :L].repeat_interleave(G, 0)
        step = vv.unflatten(-1, (-1, 64)).abs().amax(-1, keepdim=True).expand(-1, -1, -1, 64).flatten(-2)  # >= s
        kstep = kk.unflatten(-1, (-1, 64)).abs().amax(-1, keepdim=True).expand(-1, -1, -1, 64).flatten(-2)
        qq = q[b, :, :n].double()
        s = (qq @ kk.transpose(-1, -2) * scale).masked_fill(~ok, -math.inf)
        off = e * (D / 16 + D / 64 + 8) * scale * 31 * (qq.abs() @ kstep.transpose(-1, -2))
        off = off + 2.0 ** -16 * scale * qq.abs().amax(-1, keepdim=True) * kk.abs().sum(-1).unsqueeze(-2)
        off = off.masked_fill(~ok, 0).amax(-1, keepdim=True) + 16 * e
        top = s.amax(-1, keepdim=True)
        seen = ~torch.isinf(top)
        p = torch.where(seen, torch.exp(s - torch.where(seen, top, 0.0)), 0.0)
        l = p.sum(-1, keepdim=True)
        p = torch.where(l > 0, p / l, 0.0)
        o = p @ vv
        size = p @ vv.abs()
        O[b, :, :n] = o
        lse[b, :, :n] = torch.where(l > 0, torch.log(l) + torch.where(seen, top, 0.0), -math.inf).squeeze(-1)
        bound[b, :, :n] = u * o.abs() + 1.01 * u * size + 2 * off * size + e * ((L / 16 + 64) * 31 + 32 * 271) * (p @ step)
        # numbers too small for the type round to its smallest step
        bound[b, :, :n] += torch.finfo(q.dtype).smallest_normal * torch.finfo(q.dtype).eps + (2.0 ** -25 * (p > 0).sum(-1, keepdim=True) * 31 if q.dtype == torch.float16 else 0.0)
    return O, lse, bound
