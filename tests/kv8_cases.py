"""Plain 64-bit restatement of the 8-bit page cache operators, for their tests (CPU)."""
from __future__ import annotations

import math

import numpy as np
import torch

PAGE, LOW, HIGH, TOP = 16, -32, 31, 448.0
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
CODES = torch.arange(127, dtype=torch.uint8).view(E4M3).double().numpy()  # the numbers of codes 0 .. 126, rising


def encode(x: np.ndarray) -> np.ndarray:
    """e4m3 codes of 64-bit numbers: the nearest, of two the even code; beyond 448 the largest; infinities and NaN the NaN code."""
    a = np.abs(x)
    fine = np.isfinite(x)
    a = np.where(fine, np.minimum(a, TOP), 0.0)
    hi = np.clip(np.searchsorted(CODES, a), 1, 126)
    lo = hi - 1
    down, up = a - CODES[lo], CODES[hi] - a
    code = np.where(down < up, lo, np.where(up < down, hi, np.where(lo % 2 == 0, lo, hi)))
    return np.where(fine, code + 128 * np.signbit(x), 127).astype(np.uint8)


def decode(codes: np.ndarray) -> np.ndarray:
    return torch.from_numpy(codes.copy()).view(E4M3).double().numpy()


def fit(top: float) -> int:
    e = LOW
    while e < HIGH and top > TOP * 2.0 ** e:
        e += 1
    return e


def append(rows: np.ndarray, slots: list[int], codes: np.ndarray, exps: np.ndarray) -> None:
    """rows [R, H, D] (64 bits) into codes [blocks, H, 16, D] and exps [blocks, H], in place."""
    at = 0
    while at < len(slots):
        if slots[at] < 0:
            at += 1
            continue
        page, to = slots[at] // PAGE, at
        while to < len(slots) and slots[to] >= 0 and slots[to] // PAGE == page:
            to += 1
        low = min(s % PAGE for s in slots[at:to])
        for h in range(rows.shape[1]):
            x = rows[at:to, h]
            e = fit(float(np.max(np.where(np.isfinite(x), np.abs(x), 0.0))))
            if low:
                was = min(max(int(exps[page, h]), LOW), HIGH)
                e = max(e, was)
                if e > was:
                    old = decode(codes[page, h, :low])
                    codes[page, h, :low] = encode(old * 2.0 ** (was - e))
            if not low or e > was:
                exps[page, h] = e
            for r in range(at, to):
                codes[page, h, slots[r] % PAGE] = encode(rows[r, h] * 2.0 ** -e)
        at = to


def pool_of(codes: np.ndarray, device="cuda") -> torch.Tensor:
    return torch.from_numpy(codes).to(device).view(E4M3)


def scale_of(exps: np.ndarray, device="cuda") -> torch.Tensor:
    return torch.from_numpy((exps + 127).astype(np.uint8)).to(device).view(E8M0)


def random_cache(rng, blocks: int, H: int, D: int, spread: int = 3):
    """Codes without NaN and exponents."""
    codes = rng.integers(0, 127, (blocks, H, PAGE, D)).astype(np.uint8) | (rng.integers(0, 2, (blocks, H, PAGE, D)) << 7).astype(np.uint8)
    return codes, rng.integers(-6 - spread, -6 + spread + 1, (blocks, H))


def attention(q: np.ndarray, k: np.ndarray, v: np.ndarray, unit: np.ndarray, scale: float, q_step: float = 0.0):
    """(softmax(q k^T scale) v, a bound on the error of the kernels) for one query row q [Hq, D] over k, v [L, H, D], whose values have
    scales unit [L, H].  `q_step`: how far a kernel's query may be off, as a part of the row's largest."""
    Hq, D = q.shape
    L, H, _ = k.shape
    out, tol = np.zeros((Hq, D)), np.zeros((Hq, D))
    if L == 0:
        return out, tol
    for h in range(Hq):
        g = h * H // Hq
        kh, vh = k[:, g], v[:, g]
        s = kh @ q[h] * scale
        p = np.exp(s - s.max())
        p /= p.sum()
        out[h] = p @ vh
        # ds: a score is a sum of D products in fp32, in any order, off by D 2^-24 of the sum of magnitudes at most.  The exponent that it becomes
        # (times log2 e, plus a value scale's exponent of up to 32, minus a reference) takes four roundings of at most 2^-24 of its
        # size, and exp2 is good to 2^-22.
        # A weight is then rounded to 11 bits, 2^-11.  f16 numbers below 2^-14 have steps of 2^-24, and the largest weight, with its value's
        # scale in it, is 2^6 at least: 2^-31 of that, times a code of at most 448.  The sum of the weights is off by ds, and the
        # result is rounded to 8 bits, 2^-8 with what an approximate quotient adds.
        ds = D * 2.0 ** -24 * (np.abs(kh) @ np.abs(q[h])).max() * scale + (np.abs(s).max() * 1.45 + 32) * 2.0 ** -22 + 2.0 ** -22
        ds += q_step * np.abs(q[h]).max() * np.abs(kh).sum(1).max() * scale
        tol[h] = 2.0 ** -8 * np.abs(out[h]) + (2 * ds + 2.0 ** -11) * (p @ np.abs(vh)) + L * 448 * 2.0 ** -31 * (p * unit[:, g]).max()
    return out, tol


def slot_map(ctx, new, table, supply, used, rows, blocks):
    """Plain bookkeeping: (lens, row_start, row_seq, positions, slots, used), table changed in place."""
    width = table.shape[1]
    lens, start, seq, pos, slot = [], [0], [], [], []
    n_used = used if 0 <= used <= len(supply) else len(supply)
    for b, (c, n) in enumerate(zip(ctx, new)):
        if c < 0 or n < 0 or c + n > width * PAGE:
            c, n = min(max(c, 0), width * PAGE), 0
        page = {}
        have, need = math.ceil(c / PAGE), math.ceil((c + n) / PAGE)
        for p in range(have, need):
            if n_used < len(supply):
                page[p] = supply[n_used]
                if 0 <= supply[n_used] < blocks:
                    table[b, p] = supply[n_used]
                n_used += 1
        for p in range(c, c + n):
            id = int(table[b, p // PAGE]) if p // PAGE < have else page.get(p // PAGE, -1)
            seq.append(b)
            pos.append(p)
            slot.append(id * PAGE + p % PAGE if 0 <= id < blocks else -1)
        lens.append(c + n)
        start.append(start[-1] + n)
    pad = max(0, rows - len(seq))
    return lens, start, (seq + [-1] * pad)[:rows], (pos + [0] * pad)[:rows], (slot + [-1] * pad)[:rows], n_used
