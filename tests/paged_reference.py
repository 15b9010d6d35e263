"""Plain forms of the paged-cache operators on the CPU: block tables in Python integers, the cache's codes in
numpy fp32 (IEEE divisions, half-even rounding: bit for bit what the kernels compute), attention in float64."""
from __future__ import annotations

import numpy as np
import torch

UNIT = 16


def tables_step(table, lengths, free, count, new, finished, block, max_tokens):
    """In place on lists; returns (slots, positions, query_start, granted, count)."""
    rows, width = len(table), len(table[0]) if table else 0
    held = lambda n: -(-n // block)   # noqa: E731
    for b in range(rows):
        if finished is not None and finished[b]:
            for j in range(held(lengths[b])):
                free[count] = table[b][j]
                table[b][j] = -1
                count += 1
            lengths[b] = 0
    available, pages_asked, tokens_asked = count, 0, 0
    slots, positions, starts, granted = [], [], [], []
    for b in range(rows):
        n = max(new[b], 0)
        starts.append(len(slots))
        fits = lengths[b] + n <= width * block
        need = held(lengths[b] + n) - held(lengths[b])
        if fits:
            pages_asked += need
            tokens_asked += n
        ok = fits and (need == 0 or pages_asked <= available) and tokens_asked <= max_tokens
        granted.append(ok)
        if not ok:
            continue
        for j in range(need):
            count -= 1
            table[b][held(lengths[b]) + j] = free[count]
        for pos in range(lengths[b], lengths[b] + n):
            slots.append(table[b][pos // block] * block + pos % block)
            positions.append(pos)
        lengths[b] += n
    starts.append(len(slots))
    rest = max_tokens - len(slots)
    return slots + [-1] * rest, positions + [0] * rest, starts, granted, count


def append(x, codes, scales, slots, transposed):
    """x float32 numpy [T, H, D] (finite, the 16-bit values); codes int8 [pages, H, units, 16, D] (or [.., D, 16]),
    scales float32, updated in place."""
    per = codes.shape[2]
    t, f32 = 0, np.float32
    while t < len(slots):
        s = int(slots[t])
        if s < 0 or s >= codes.shape[0] * per * UNIT:
            t += 1
            continue
        e, src = t, {}
        while e < len(slots) and int(slots[e]) // UNIT == s // UNIT and int(slots[e]) >= 0:
            src[int(slots[e]) % UNIT] = e
            e += 1
        begun, page, unit = min(src), s // UNIT // per, s // UNIT % per
        for h in range(codes.shape[1]):
            c = codes[page, h, unit].T if transposed else codes[page, h, unit]   # [16, D] view
            top = f32(max(np.abs(x[i, h]).max() for i in src.values()))
            top = f32(0) if top < f32(2.0 ** -100) else top
            old = scales[page, h, unit] if begun else f32(0)
            new = max(old, f32(top / f32(127)))
            inv = f32(1) / new if new > 0 else f32(0)
            if begun and new > old:
                c[:begun] = np.rint(c[:begun].astype(f32) * f32(old / new)).astype(np.int8)
            for o, i in src.items():
                c[o] = np.clip(np.rint(x[i, h].astype(f32) * inv), -127, 127).astype(np.int8)
            scales[page, h, unit] = new
        t = e


def values(codes, scales, slots, transposed):
    """float64 [N, H, D] of the slots (>= 0)."""
    per = codes.shape[2]
    s = np.asarray(slots, dtype=np.int64)
    page, unit, at = s // UNIT // per, s // UNIT % per, s % UNIT
    c = codes[page, :, unit][np.arange(len(s)), :, :, at] if transposed else codes[page, :, unit][np.arange(len(s)), :, at]
    return c.astype(np.float64) * scales[page, :, unit].astype(np.float64)[..., None]


def attend(q, k_codes, v_codes, k_scales, v_scales, table, lengths, starts, scale, dtype):
    """float64 attention [T, Hq, D] and the bound of the kernel's error for outputs in ``dtype``.

    q float64 [T, Hq, D]; caches as numpy; table rows of page ids (ids outside the cache: those keys are left out).
    The bound, with A = sum p |v| / sum p, S = scale sum |q k| log2(e) at most, N keys:
      one rounding to dtype             eps/2 |out|
      P rounded to fp16                 2^-11 A, and half a subnormal step 2^-25 per key under 2^-14 of the largest
                                        p t: times its codes (<= 127) and over the sum (>= 1 / t): 2^-25 N max|v|
      q rounded to 2^-25 of its row's   2^-25 max|q| sum |k| scale (a log2 score's error, as the next line)
      fp32 scores, exp2, log2, sums     each within a few 2^-23 of S or 1, D / 32 + 4 operations deep: 2^-19 (1 + S)
    and a score's error e moves the result by at most 2 e A."""
    pages, _, units = k_codes.shape[:3]
    block = units * UNIT
    T, hq, dim = q.shape
    group = hq // k_codes.shape[1]
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    half = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}[dtype]
    for b in range(len(lengths)):
        n_q = starts[b + 1] - starts[b]
        pos = np.arange(lengths[b])
        page = np.asarray(table[b], dtype=np.int64)[pos // block] if len(pos) else pos
        there = (page >= 0) & (page < pages)
        slots = np.where(there, page * block + pos % block, 0)
        k = values(k_codes, k_scales, slots, False)
        v = values(v_codes, v_scales, slots, True)
        for i in range(n_q):
            seen = there & (pos <= lengths[b] - n_q + i)
            if not seen.any():
                continue
            for h in range(hq):
                kk, vv, qq = k[seen, h // group], v[seen, h // group], q[starts[b] + i, h]
                s = kk @ qq * scale
                p = np.exp(s - s.max())
                p /= p.sum()
                o, A = p @ vv, p @ np.abs(vv)
                S = abs(scale) * 1.4427 * (np.abs(kk) @ np.abs(qq)).max()
                eq = 2.0 ** -25 * np.abs(qq).max() * np.abs(kk).sum(1).max() * abs(scale) * 1.4427
                e = 2.0 ** -19 * (1 + S) + eq
                out[starts[b] + i, h] = o
                tol[starts[b] + i, h] = half * np.abs(o) + (2.0 ** -11 + 2 * e) * A \
                    + 2.0 ** -25 * seen.sum() * np.abs(vv).max()
    return out, tol + 1e-30
