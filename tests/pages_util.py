"""The paged 4-bit cache in plain Python and 64 bits: a page's layout element by
element, the rounding to 4 bits, and the rows of pages one after the other."""

import math

import numpy as np
import torch


def d8(x):
    """x to 8 significant bits, ties to even, at the bottom to multiples of 2^-24."""
    if x == 0 or not math.isfinite(x):
        return x
    unit = 2.0 ** max(math.frexp(x)[1] - 8, -24)
    return round(x / unit) * unit  # (exact quotient; round() takes ties to even)


def quantised(x):
    """(codes, scales, held) of x [..., hd] (float64, CPU), 32 at a time."""
    x = np.asarray(x, np.float64)
    y = x.reshape(-1, 32)
    size = np.abs(y)
    with np.errstate(invalid="ignore"):
        bad = ~(size < 16384.0).all(1)
    at = np.where(np.isnan(size), -1.0, size).argmax(1)  # (the first of equals)
    d = np.array([math.nan if b else d8(float(v)) for v, b in zip(y[np.arange(len(y)), at] / -8, bad)])
    with np.errstate(invalid="ignore", divide="ignore"):
        code = np.where((d == 0)[:, None] | bad[:, None], 0.0, np.clip(np.rint(y / d[:, None]), -8, 7))
        held = np.where((d == 0)[:, None], 0.0, code * d[:, None])
    return (code + 8).astype(np.int64).reshape(x.shape), d.reshape(*x.shape[:-1], -1), held.reshape(x.shape)


class Layout:
    """Byte and half of every element of a kv head's part of a page."""

    def __init__(self, page, hd):
        self.page, self.hd, self.part = page, hd, page * (hd + hd // 8)
        s, d = np.meshgrid(np.arange(page), np.arange(hd), indexing="ij")
        j, r, groups = d // 32, d % 32, hd // 32
        i, e = r // 8, r % 8
        bit = e // 2 * 4 + e % 2 * 16
        self.key = ((s * 4 + i) * groups + j) * 4 + bit // 8, bit % 8
        u, i, t, m = s // 16, s % 16 // 4, s % 4, r // 2
        self.value = page * hd // 2 + (((u * 4 + i) * 16 + m) * groups + j) * 4 + t, (d % 2) * 4
        s, j = np.meshgrid(np.arange(page), np.arange(groups), indexing="ij")
        self.key_scale = page * hd + (s * groups + j) * 2
        self.value_scale = page * hd + page * hd // 16 + ((s // 4 * groups + j) * 4 + s % 4) * 2

    def read(self, part):
        """Keys and values [..., page, hd] (float64) of parts [..., bytes] (uint8)."""
        part = np.asarray(part)
        res = []
        for (at, shift), scale in ((self.key, self.key_scale), (self.value, self.value_scale)):
            code = (part[..., at] >> shift) & 15
            bits = part[..., scale].astype(np.uint16) | part[..., scale + 1].astype(np.uint16) << 8
            d = np.ascontiguousarray(bits).view(np.float16).astype(np.float64)
            with np.errstate(invalid="ignore"):
                res.append((code.astype(np.float64) - 8) * np.repeat(d, 32, -1))
        return res

    def write(self, part, slot, key, value):
        """Codes and scales ((codes, scales) each) of one token into a part [bytes]."""
        for (code, d), (at, shift), scale in ((key, self.key, self.key_scale), (value, self.value, self.value_scale)):
            for x in range(self.hd):
                a, sh = at[slot, x], int(shift[slot, x])
                part[a] = (int(part[a]) & ~(15 << sh) & 255) | int(code[x]) << sh
            part[scale[slot][:, None] + np.arange(2)] = np.asarray(d, np.float16).view(np.uint8).reshape(-1, 2)


def rotated(x, positions, gain, dims, half, freq, mult, eps):
    """Heads x [..., heads, hd] normed (gain not None) and rotated at positions [...], float64."""
    x = x.double()
    if gain is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * gain.double()
    a = positions.double()[..., None, None] * torch.as_tensor(freq, dtype=torch.float64, device=x.device)
    c, s = a.cos() * mult, a.sin() * mult
    out = x.clone()
    i = torch.arange(dims // 2, device=x.device)
    p, q = (i, i + dims // 2) if half else (2 * i, 2 * i + 1)
    out[..., p] = x[..., p] * c - x[..., q] * s
    out[..., q] = x[..., p] * s + x[..., q] * c
    return out


def update(table, lens, refs, source, keep, add, page, width):
    """(table, lens, refs, copies) after s2hip_pages_update, row by row; None where it changes nothing."""
    rows, pages_of = len(lens), lambda n: -(-n // page)
    cap = width * page
    kept = []
    for b in range(rows):
        if not (0 <= lens[b] <= cap and -1 <= source[b] < rows and keep[b] >= 0 and add[b] >= 0):
            return None
    for b in range(rows):
        kept.append(0 if source[b] < 0 else min(keep[b], lens[source[b]]))
        if kept[b] + add[b] > cap:
            return None
    new = [[-1] * width for _ in range(rows)]
    refs = list(refs)
    for b in range(rows):
        for p in table[b][: pages_of(lens[b])]:
            if not 0 <= p < len(refs):
                return None
            refs[p] -= 1
    for b in range(rows):
        for i in range(pages_of(kept[b])):
            new[b][i] = table[source[b]][i]
            refs[new[b][i]] += 1
    if any(r < 0 for r in refs) or any(refs[p] < 1 for b in range(rows) for p in new[b][: pages_of(kept[b])]):
        return None
    free = [p for p in range(len(refs)) if refs[p] == 0]
    copies = {}
    for b in range(rows):
        at = kept[b] // page
        if add[b] and kept[b] % page and refs[new[b][at]] > 1:
            if not free:
                return None
            old = new[b][at]
            refs[old] -= 1
            new[b][at] = free.pop(0)
            refs[new[b][at]] = 1
            copies[new[b][at]] = old
        for i in range(pages_of(kept[b]), pages_of(kept[b] + add[b])):
            if not free:
                return None
            new[b][i] = free.pop(0)
            refs[new[b][i]] = 1
    return new, [k + a for k, a in zip(kept, add)], refs, copies


def compact(table, lens, refs, page):
    """(table, refs, moves, used) after s2hip_pages_compact."""
    used = sum(r > 0 for r in refs)
    holes = [p for p in range(used) if refs[p] == 0]
    movers = [p for p in range(used, len(refs)) if refs[p] > 0]
    to = dict(zip(movers, holes))
    table = [[to.get(p, p) if i < -(-n // page) else p for i, p in enumerate(row)] for row, n in zip(table, lens)]
    out = [0] * len(refs)
    for p, r in enumerate(refs):
        if r > 0:
            out[to.get(p, p)] = r
    return table, out, to, used
