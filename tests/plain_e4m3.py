"""The cache in 8 bits written down plainly, in 64 bits on the host: what a step's rows become in their blocks, and attention over
what the blocks hold.  Codes are 8-bit patterns of e4m3 (torch.float8_e4m3fn as uint8)."""

import math

import numpy as np
import torch

BLOCK, TOP = 16, 448.0


def _table():
    values = np.zeros(256)
    for code in range(256):
        sign, exponent, fraction = (-1.0 if code & 128 else 1.0), (code >> 3) & 15, code & 7
        if code & 127 == 127:
            values[code] = np.nan
        elif exponent == 0:
            values[code] = sign * fraction * 2.0 ** -9
        else:
            values[code] = sign * (1 + fraction / 8) * 2.0 ** (exponent - 7)
    return values


VALUES = _table()


def nearest_code(x):
    """Codes of 64-bit numbers, nearest, ties to an even fraction, beyond 448 to 448, NaN to 0x7f."""
    x = np.asarray(x, np.float64)
    size = np.minimum(np.abs(x), TOP)
    step = 2.0 ** (np.floor(np.log2(np.maximum(size, 2.0 ** -6))) - 3.0)
    value = np.minimum(np.round(np.where(np.isnan(x), 0.0, size) / step) * step, TOP)
    code = np.searchsorted(VALUES[:127], value).astype(np.uint8)
    return np.where(np.isnan(x), np.uint8(127), code | np.where(np.signbit(x), np.uint8(128), np.uint8(0))).astype(np.uint8)


def least_scale(square):
    """The least power of two s >= 2^-64 with square <= (448 s)^2."""
    e = -64
    while square > TOP ** 2 * 4.0 ** e:
        e += 1
    return 2.0 ** e


def squares(row, rot, amplitude=1.0):
    """What bounds the entries of a head: 32-bit squares of its entries and of its pairs' lengths, as the definition has them."""
    row = row.astype(np.float32)
    with np.errstate(over="ignore", invalid="ignore"):
        s = row * row
        a = np.float32(amplitude) * np.float32(amplitude)
        return np.concatenate(((s[0:rot:2] + s[1:rot:2]) * a, s[rot:]))


def turned(row, rot, position, inv_freq, amplitude=1.0):
    out = row.astype(np.float64).copy()
    for i in range(rot // 2):
        angle = float(position) * float(inv_freq[i])
        c, s = math.cos(angle) * amplitude, math.sin(angle) * amplitude
        x, y = float(row[2 * i]), float(row[2 * i + 1])
        out[2 * i], out[2 * i + 1] = x * c - y * s, x * s + y * c
    return out


def append(pages, scales, rows, rot, positions, items, table, inv_freq, amplitude=1.0):
    """Rows [T, heads, size] into pages (uint8 [pages, heads, page, size]) and scales [pages, heads, page / 16], in place.
    Returns the 64-bit numbers that the new codes stand for when nothing were rounded, [T, heads, size] (None where a row is stored nowhere)."""
    page, n = pages.shape[2], len(positions)
    wanted, t = [None] * n, 0
    while t < n:
        end = t + 1
        while (end < n and items[end] == items[t] and positions[end] == positions[end - 1] + 1 and positions[end] % BLOCK != 0
               and positions[t] >= 0):
            end += 1
        position, first = int(positions[t]), t
        t = end
        if position < 0 or position // page >= table.shape[1]:
            continue
        where = int(table[items[first], position // page])
        if not 0 <= where < pages.shape[0]:
            continue
        slot, lead = position % page, position % BLOCK
        for head in range(rows.shape[1]):
            every = [squares(rows[r, head], rot, amplitude) for r in range(first, end)]
            fine = [bool(np.isfinite(s).all()) for s in every]
            scale = max([least_scale(float(s.max())) for s, ok in zip(every, fine) if ok] or [2.0 ** -64])
            held = float(scales[where, head, slot // BLOCK])
            block = pages[where, head, slot - lead:slot - lead + BLOCK]
            if lead and held >= scale:
                scale = held
            elif lead:
                block[:lead] = nearest_code(VALUES[block[:lead]] * (held / scale))
            scales[where, head, slot // BLOCK] = scale
            for r in range(first, end):
                value = turned(rows[r, head], rot, positions[r], inv_freq, amplitude) if fine[r - first] else np.full(rows.shape[2], np.nan)
                block[lead + r - first] = nearest_code(value / scale)
                wanted[r] = wanted[r] or []
                wanted[r].append(value)
    return wanted


def attention(q, k_pages, v_pages, k_scales, v_scales, table, entries, heads, scale, cap=0.0, window=0):
    """q [T, heads * dim]; entries (offset, count, start).  Returns (out [T, heads * vdim] with NaN-free zeros in rows of no entry,
    weights' sums of |v| per entry of out, the largest sum of |q k| scale, and per entry of out the number of keys times the largest
    value a code may have times the largest weight times its value's scale)."""
    n_pages, kv_heads, page, dim = k_pages.shape
    vdim = v_pages.shape[3]
    out = np.zeros((q.shape[0], heads * vdim))
    spread, edge, most = np.zeros_like(out), np.zeros_like(out), 0.0
    for item, (offset, count, start) in enumerate(entries):
        for i in range(count):
            position = start + i
            first = max(0, position - window + 1) if window else 0
            keys = [j for j in range(first, position + 1)
                    if j // page < table.shape[1] and 0 <= int(table[item, j // page]) < n_pages]
            if not keys:
                continue
            at = np.array([int(table[item, j // page]) for j in keys])
            slot = np.array([j % page for j in keys])
            for head in range(heads):
                kv = head // (heads // kv_heads)
                k = VALUES[k_pages[at, kv, slot]] * k_scales[at, kv, slot // BLOCK][:, None].astype(np.float64)
                v = VALUES[v_pages[at, kv, slot]] * v_scales[at, kv, slot // BLOCK][:, None].astype(np.float64)
                row = q[offset + i, head * dim:(head + 1) * dim].astype(np.float64)
                with np.errstate(invalid="ignore", over="ignore"):
                    s = k @ row * scale
                    if cap:
                        s = cap * np.tanh(s / cap)
                    p = np.exp(s - s.max())
                    p = p / p.sum()
                    columns = slice(head * vdim, (head + 1) * vdim)
                    out[offset + i, columns] = p @ v
                    spread[offset + i, columns] = p @ np.abs(v)
                    edge[offset + i, columns] = len(keys) * TOP * np.nanmax(np.append(p * v_scales[at, kv, slot // BLOCK], 0.0))
                    most = max(most, float(np.nan_to_num(np.abs(k) @ np.abs(row) * scale).max()))
    return out, spread, most, edge


def codes_of(pages):
    return pages.view(torch.uint8).cpu().numpy()
