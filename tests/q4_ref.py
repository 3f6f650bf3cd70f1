"""Plain restatements, in 64 bits and Python integers, of the block maps and the 4-bit paged KV pool."""
from __future__ import annotations

import math

import numpy as np

from oracle import oracle as O

F16, BF16 = O.F16, O.BF16
EPS = {F16: 2.0 ** -10, BF16: 2.0 ** -7}  # torch.finfo(t).eps


def widen(dt, bits):
    """16-bit patterns -> float64."""
    bits = np.asarray(bits, np.uint16)
    if dt == F16:
        return bits.view(np.float16).astype(np.float64)
    return (bits.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def quantise(x):
    """x float64 [..., dim] -> codes uint8 [..., G, 32], s and m float16 [..., G]."""
    v = x.reshape(*x.shape[:-1], -1, 32)
    finite = np.isfinite(v).all(-1)
    w = np.clip(np.where(finite[..., None], v, 0.0), -65504.0, 65504.0)
    lo, hi = w.min(-1), w.max(-1)
    s = ((hi - lo) / 15.0).astype(np.float16)
    m = (lo + 8.0 * s.astype(np.float64)).astype(np.float16)
    s64, m64 = s.astype(np.float64)[..., None], m.astype(np.float64)[..., None]
    c = np.where(s64 > 0, np.clip(np.rint((w - m64) / np.where(s64 > 0, s64, 1.0)) + 8, 0, 15), 8).astype(np.uint8)
    s = np.where(finite, s, np.uint16(0x7FFF).view(np.float16))
    m = np.where(finite, m, np.uint16(0x7FFF).view(np.float16))
    return c, s, m


def values(c, s, m):
    """What codes, s, m stand for, float64 [..., dim]."""
    v = (c.astype(np.float64) - 8.0) * s.astype(np.float64)[..., None] + m.astype(np.float64)[..., None]
    return v.reshape(*v.shape[:-2], -1)


def chunk_offsets(dim):
    """(byte of each K dim, of each V dim within a chunk at token 0, their token strides, nibble), K / V param base."""
    g = dim // 32
    d = np.arange(dim)
    grp, e = d // 32, d % 32
    k = (e // 8 * g + grp) * 4 + e % 8 // 2
    per = 16 // g
    r = e // 4
    v = 10 * dim + (r // per) * 16 * 32 + (r % per * g + grp) * 2 + e % 4 // 2
    return k, v, d % 2


class Pool:
    """A 4-bit pool as bytes [block][layer][head][20 dim]."""

    def __init__(self, blocks, layers, heads, dim, fill):
        self.b = np.asarray(fill, np.uint8).reshape(blocks, layers, heads, 20 * dim).copy()
        self.dim = dim

    def put(self, slot, layer, k, v):
        """Rows k, v float64 [heads, dim] into a slot."""
        dim, g = self.dim, self.dim // 32
        t, ch = slot % 16, self.b[slot // 16, layer]
        ko, vo, odd = chunk_offsets(dim)
        for x, off, par in ((k, ko + t * (dim // 2), 8 * dim), (v, vo + t * 32, 18 * dim)):
            c, s, m = quantise(x)
            c = c.reshape(x.shape[0], dim)
            for h in range(x.shape[0]):
                row = np.zeros(20 * dim, np.uint8)
                np.add.at(row, off, (c[h] << (4 * odd)).astype(np.uint8))
                ch[h][off] = row[off]
                word = (s[h].view(np.uint16).astype(np.uint32) << 16 | m[h].view(np.uint16)).astype("<u4")
                ch[h][par + t * g * 4: par + (t + 1) * g * 4] = word.view(np.uint8)

    def rows(self, slots, layer):
        """(K, V, steps K, middles K, steps V, middles V) of the slots: values [n, heads, dim] in float64 and [n, heads, G]."""
        dim, g = self.dim, self.dim // 32
        slots = np.asarray(slots)
        ch = self.b[slots // 16, layer]  # [n, heads, bytes]
        t = slots % 16
        ko, vo, odd = chunk_offsets(dim)
        out = []
        for off, stride, par in ((ko, dim // 2, 8 * dim), (vo, 32, 18 * dim)):
            at = off[None, :] + t[:, None] * stride
            c = np.take_along_axis(ch, at[:, None, :].repeat(ch.shape[1], 1), -1) >> (4 * odd) & 15
            pat = par + t[:, None] * g * 4 + np.arange(4 * g)[None, :]
            w = np.ascontiguousarray(np.take_along_axis(ch, pat[:, None, :].repeat(ch.shape[1], 1), -1)).view("<u4")
            s = (w >> 16).astype(np.uint16).view(np.float16)
            m = (w & 0xFFFF).astype(np.uint16).view(np.float16)
            out.append((values(c.reshape(*c.shape[:2], g, 32), s, m), s.astype(np.float64), m.astype(np.float64)))
        (k, ks, km), (v, vs, vm) = out
        return k, v, ks, km, vs, vm


def attention(pool, q, tables, lens, *, group, layer=0, scale=0.0, softcap=0.0, window=0, starts=None, slopes=None):
    """(out, bound) in float64, [batch, heads, dim].  q float64 [batch, heads, dim].

    bound: how far a kernel may be that rounds each weight times step once to f16 (2^-11 of a term with |c - 8| <= 8),
    each weight times middle once to f16, and scores in fp32 sums of up to 2 * dim terms (2^-18 of the sum of
    magnitudes, which also covers the exponential's 2^-21), before the output's own rounding."""
    batch, heads, dim = q.shape
    scale = scale or 1.0 / math.sqrt(dim)
    out, bound = np.zeros_like(q), np.zeros_like(q)
    for b in range(batch):
        n = int(lens[b])
        first = max(0, int(starts[b]) if starts is not None else 0, n - window if window else 0)
        if first >= n:
            continue
        j = np.arange(first, n)
        k, v, ks, km, vs, vm = pool.rows(tables[b][j // 16].astype(np.int64) * 16 + j % 16, layer)
        for h in range(heads):
            hk = h // group
            x = scale * (k[:, hk] @ q[b, h])
            mag = abs(scale) * ((8 * ks[:, hk] + np.abs(km[:, hk])).repeat(32, -1) @ np.abs(q[b, h]))
            if softcap:
                x = softcap * np.tanh(x / softcap)
            err_x = 2.0 ** -18 * (mag.max() + 1.0) + 2.0 ** -22 * softcap
            if slopes is not None:
                x = x + float(slopes[h]) * (j - (n - 1))
                err_x += 2.0 ** -22 * abs(float(slopes[h])) * (n - first)
            w = np.exp(x - x.max())
            w /= w.sum()
            out[b, h] = w @ v[:, hk]
            each = (8 * vs[:, hk] + np.abs(vm[:, hk])).repeat(32, -1)
            bound[b, h] = (2.0 ** -11 + 2 * err_x) * (w @ each) + 2.0 ** -20 * (w.max() * each.max())
    return out, bound


def block_map(tables, pre, new, free, count, num_blocks, max_rows):
    """tables' , slots, q_start, post, count', error bits -- one sequence after another."""
    tables = tables.copy()
    slots = np.full(max_rows, -1, np.int32)
    starts, post, err, upto, used, row = [], [], 0, 0, 0, 0
    if not 0 <= count <= num_blocks:
        err |= 1
    count = min(max(count, 0), num_blocks)
    for b in range(len(pre)):
        p, a = int(pre[b]), int(new[b])
        start = min(row, max_rows)
        starts.append(start)
        row = min(row + max(a, 0), max_rows)
        if p < 0 or a < 0 or p + a > tables.shape[1] * 16 or start + a > max_rows:
            err |= 2
            post.append(p)
            continue
        have, need = -(-p // 16), -(-(p + a) // 16) - -(-p // 16)
        upto += need
        if need and upto > count:
            err |= 16
            post.append(p)
            continue
        if need:
            used = upto
        for i in range(need):
            tables[b, have + i] = free[count - 1 - (upto - need + i)]
        for i in range(a):
            blk = int(tables[b, (p + i) // 16])
            if 0 <= blk < num_blocks:
                slots[start + i] = blk * 16 + (p + i) % 16
            else:
                err |= 1
        post.append(p + a)
    return tables, slots, np.array(starts, np.int32), np.array(post, np.int32), count - used, err


def block_release(tables, lens, release, free, count, num_blocks):
    free, lens, err = free.copy(), lens.copy(), 0
    if not 0 <= count <= num_blocks:
        err |= 1
    count = min(max(count, 0), num_blocks)
    for b in range(len(lens)):
        if not release[b]:
            continue
        n = min(max(int(lens[b]), 0), tables.shape[1] * 16)
        if n != lens[b]:
            err |= 2
        for i in range(-(-n // 16)):
            blk = int(tables[b, i])
            if not 0 <= blk < num_blocks:
                err |= 1
            elif count < num_blocks:
                free[count] = blk
                count += 1
            else:
                err |= 1
        lens[b] = 0
    return free, lens, count, err
