"""The paged 8-bit cache's operators and rotary positions from their definitions, on the CPU in 64 bits (int8 quotients in the
fp32 that their definition names), in plain loops."""
from __future__ import annotations

import math

import numpy as np
import torch

F8 = torch.float8_e4m3fn


def plan(cached, new, table, free_pages, free_count, page, max_tokens):
    """-> dict of what paged_plan returns and the table, as numpy arrays; `table` is not changed."""
    B, width = table.shape
    table = table.copy()
    cached, new = [max(int(c), 0) for c in cached], [max(int(n), 0) for n in new]
    free = min(max(int(free_count), 0), len(free_pages))
    cu, pos, slots, used, ok, asked, left = [0], [0] * max_tokens, [-1] * max_tokens, [], [], 0, free
    for b in range(B):
        start, end = cu[-1], cu[-1] + new[b]
        cu.append(end)
        have, want = -(-cached[b] // page), -(-(cached[b] + new[b]) // page)
        fits = end <= max_tokens and cached[b] + new[b] <= width * page
        first = asked
        asked += want - have if fits else 0
        good = fits and (want == have or asked <= free)
        if good and want > have:
            left = free - asked
            for i in range(want - have):
                table[b, have + i] = free_pages[free - 1 - first - i]
        ok.append(good)
        used.append(cached[b] + new[b] if good else cached[b])
        for t in range(start, min(end, max_tokens)):
            pos[t] = min(cached[b] + t - start, 2 ** 31 - 1)
            if good and table[b, pos[t] // page] >= 0:
                slots[t] = int(table[b, pos[t] // page]) * page + pos[t] % page
    return dict(table=table, cu_seqlens=np.minimum(np.array(cu), max_tokens), seqused_k=np.array(used, dtype=np.int64), positions=np.array(pos),
                slots=np.array(slots), admitted=np.array(ok, dtype=bool), free_count=np.array([left]))


def e4m3(x):
    """Nearest e4m3 value, ties to even, saturating; NaN stays."""
    a = np.abs(x)
    with np.errstate(divide="ignore", invalid="ignore"):
        e = np.floor(np.log2(np.maximum(a, 2.0 ** -6)))
        e = np.where(np.isfinite(e), e, 0)
        step = np.exp2(e - 3)
        y = np.rint(np.where(np.isfinite(x), x, 0) / step) * step
        y = np.where(np.isinf(x), np.copysign(448.0, x), np.clip(y, -448, 448))
    return np.where(np.isnan(x), np.nan, y)


def write(x, pages, scales, slots, int8):
    """x [T, H, D] float64, pages [P, page, H, D] stored values as float64, scales [P, nb, H] float32 -> new (pages, scales)."""
    pages, scales = pages.copy(), scales.copy()
    P, page, H, D = pages.shape
    block = page // scales.shape[1]
    flat, sc = pages.reshape(-1, block, H, D), scales.reshape(-1, H)
    runs = {}
    for t, s in enumerate(slots):
        if 0 <= s < P * page:
            runs.setdefault(int(s) // block, []).append(t)
    for u, ts in runs.items():
        offs = [int(slots[t]) % block for t in ts]
        for h in range(H):
            rows = x[ts, h]
            fin = np.abs(rows[np.isfinite(rows)])
            top = np.float32(fin.max()) if fin.size else np.float32(0)
            if int8:
                need = max(np.float32(top * np.float32(1 / 127)), np.float32(2.0 ** -100))
            else:
                e = -100
                if top > 0:
                    e = max(-100, math.frexp(float(top))[1] - 9 - 2)
                    while 448 * 2.0 ** e < top:
                        e += 1
                need = np.float32(2.0 ** e)
            old = np.float32(0) if 0 in offs else sc[u, h]
            now = max(old, need)
            if 0 not in offs and now > old:
                f = np.float32(old / now)
                again = (flat[u, :, h].astype(np.float32) * f).astype(np.float64)
                flat[u, :, h] = np.clip(np.rint(again), -127, 127) if int8 else e4m3(again)
            sc[u, h] = now
            inv = np.float32(1) / now
            with np.errstate(invalid="ignore", over="ignore"):
                q = (rows.astype(np.float32) * inv).astype(np.float64)
            q = np.clip(np.rint(np.where(np.isnan(q), 0, q)), -127, 127) if int8 else e4m3(q)
            flat[u, offs, h] = q
    return pages, scales


def gathered(pages, scales, row, n):
    """The first n keys of a table row, dequantised, float64 [n, H, D]; keys of entries outside the pool are left out.
    -> (values, their positions)."""
    P, page, H, D = pages.shape
    block = page // scales.shape[1]
    vals, at = [], []
    for j in range(-(-n // page)):
        p = int(row[j])
        if not 0 <= p < P:
            continue
        m = min(page, n - j * page)
        x = pages[p, :m].double() * scales[p].double().repeat_interleave(block, 0)[:m, :, None]
        vals.append(x)
        at += list(range(j * page, j * page + m))
    return (torch.cat(vals) if vals else torch.zeros(0, H, D, dtype=torch.float64)), torch.tensor(at, dtype=torch.long)


def attention(q, pages, scales, row, n, causal, scale, eps):
    """One sequence: q [Lq, Hq, D] float64, pages = (K, V) stored values, scales = (ks, vs).  -> out [Lq, Hq, D], lse [Lq, Hq] and
    how far a kernel may be off each: it rounds each probability and each output to steps of half `eps` relative, and fp32
    score sums over D terms to 2^-24 of the terms' magnitudes each."""
    Lq, Hq, D = q.shape
    (K, at), (V, _) = gathered(pages[0], scales[0], row, n), gathered(pages[1], scales[1], row, n)
    V8, _ = gathered(pages[1], torch.ones_like(scales[1]), row, n)  # as stored
    VS, _ = gathered(torch.ones(pages[1].shape[:3] + (1,)), scales[1], row, n)
    g = Hq // K.shape[1]
    out, lse = torch.zeros(Lq, Hq, D, dtype=torch.float64), torch.full((Lq, Hq), math.inf, dtype=torch.float64)
    tol, ltol = torch.zeros_like(out), torch.zeros_like(lse)
    u = eps / 2
    for h in range(Hq):
        k, v = K[:, h // g], V[:, h // g]
        s = q[:, h] @ k.T * scale
        size = (q[:, h].abs() @ k.abs().T * abs(scale))
        seen = torch.ones(Lq, len(at), dtype=torch.bool)
        if causal:
            seen = at[None, :] <= n - Lq + torch.arange(Lq)[:, None]
        s = torch.where(seen, s, -math.inf)
        live = seen.any(1)
        if not live.any():
            continue
        z = torch.logsumexp(s[live], 1)
        p = torch.exp(s[live] - z[:, None])
        o = p @ v
        mass = p @ v.abs()
        off = (size * seen)[live].max(1).values * (D + 8) * 2.0 ** -24 + 2.0 ** -20
        sums = (len(at) / 16 + 16) * 2.0 ** -24
        # fp16 is rounded to steps of 2^-24 below 2^-14: outputs to half of one, and probabilities, which enter times 2^15 and in
        # units of the largest scale among the blocks, to 2^-25 x 2^-15 x that scale x the stored values (their sum's share of
        # the row is no larger, as the row's own sum is at least 1)
        small = 0.0
        if eps == torch.finfo(torch.float16).eps:
            small = 2.0 ** -25 + 2.0 ** -40 * float(VS.max()) * V8[:, h // g].abs().sum(0)
        out[live, h], lse[live, h] = o, z
        tol[live, h] = (u * (mass + o.abs()) * (1 + u) + 2 * (off + sums)[:, None] * mass + small) + 1e-30
        ltol[live, h] = off + sums + z.abs() * 2.0 ** -22
    return out, lse, tol, ltol


def rotary(x, positions, inv_freq, axes, interleaved, inverse=False):
    """x [..., H, T, D]-like with tokens described by positions [A, tokens...] broadcast to x[..., 0, 0]'s shape without heads:
    x is [B, H, S, D] with positions [A, B, S], or [T, H, D] with [A, T].  float64 -> (turned, how far a kernel may be off before
    its rounding): angles reduced in 64 bits are good to 2^-25 of a half turn, sine and cosine in 32 bits to 2 units, and the two
    products and the sum are fp32: below (|a| + |b|) 2^-21."""
    y, tol = x.clone(), torch.zeros_like(x)
    n = len(inv_freq)
    for i in range(n):
        t = positions[int(axes[i])].double() * float(inv_freq[i]) * (-1 if inverse else 1)
        t = t[:, None, :] if x.dim() == 4 else t[:, None]
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + n)
        y[..., a] = x[..., a] * torch.cos(t) - x[..., b] * torch.sin(t)
        y[..., b] = x[..., b] * torch.cos(t) + x[..., a] * torch.sin(t)
        tol[..., a] = tol[..., b] = (x[..., a].abs() + x[..., b].abs()) * 2.0 ** -21
    return y, tol
