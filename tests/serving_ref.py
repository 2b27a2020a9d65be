"""Plain 64-bit forms of the serving operators, and what their outputs may be off by."""
import math

import numpy as np
import torch

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def attend(q, k, v, first, scale):
    """q [n][H][hd] against k, v [m][G][hd] in 64 bits: row i sees keys 0..first + i (none
    where that is negative).  Values no row sees stay out of it, NaN or not.
    Returns (out [n][H][hd], sum p |v|, largest scale * sum |q k| seen per row)."""
    n, H, hd = q.shape
    m, G, _ = k.shape
    out, mass, top = torch.zeros(n, H, hd, dtype=torch.float64), torch.zeros(n, H, hd, dtype=torch.float64), torch.zeros(n, H, 1, dtype=torch.float64)
    q, k, v = q.double(), k.double(), v.double()
    for i in range(n):
        seen = min(first + i + 1, m)
        if seen <= 0:
            continue
        for g in range(G):
            h = slice(g * (H // G), (g + 1) * (H // G))
            p = torch.softmax(q[i, h] @ k[:seen, g].T * scale, dim=1)
            out[i, h], mass[i, h] = p @ v[:seen, g], p @ v[:seen, g].abs()
            top[i, h] = (q[i, h].abs() @ k[:seen, g].abs().T * scale).amax(1, keepdim=True)
    return out, mass, top


def bound(dtype, out, mass, top, hd, keys):
    """How far an output may be off.  A rounding is half a step, eps / 2 relative:
    - the output's own: eps_t / 2 |o|, and half the least subnormal in f16;
    - 16-bit types: the weights', eps_t / 2 of sum p |v|; in f16 also half the least
      subnormal (2^-25) per key, against weights whose largest is 1 and a sum of at
      least 1: keys 2^-25 max |v|, max |v| <= the largest of the data (6 here);
    - scores: hd products and sums in f32, the scale and the exponent's argument, off by
      (hd + 8) 2^-24 of scale sum |q k| <= top; a weight is then off by the factor
      1 +- that, top and bottom of the quotient, so twice: 2 (hd + 8) 2^-24 (top + 1);
      the exponentials themselves 2^-22 twice, and once more for each of the partial
      results that are joined: 16 2^-24;
    - the two sums over keys in f32: 2 keys 2^-24."""
    eps = torch.finfo(TYPES[dtype]).eps / 2
    u = 2.0 ** -24
    tol = eps * out.abs() + u * mass * (2 * (hd + 8) * (top + 1) + 16 + 2 * keys)
    if dtype != "f32":
        tol = tol + eps * mass
    if dtype == "f16":
        tol = tol + 2.0 ** -25 * (1 + 6 * keys)
    return tol


class Cache:
    """A paged cache on the host, filled with NaN where no position is: pages in an
    order of their own, lengths as given; to(device) makes the device's arrays."""

    def __init__(self, lengths, page, kv, hd, dtype, layers=1, spare=3, seed=0, max_pages=None):
        g = torch.Generator().manual_seed(seed)
        used = [-(-n // page) for n in lengths]
        self.page, self.dtype, self.lengths = page, dtype, list(lengths)
        self.n_pages = sum(used) + spare
        self.max_pages = max_pages or max(max(used), 1) + 1
        shape = (layers, self.n_pages, page, kv, hd)
        self.k = torch.full(shape, math.nan, dtype=TYPES[dtype])
        self.v = torch.full(shape, math.nan, dtype=TYPES[dtype])
        order = torch.randperm(self.n_pages, generator=g).tolist()
        self.table = torch.full((len(lengths), self.max_pages), -1, dtype=torch.int32)
        self.ref = torch.zeros(self.n_pages, dtype=torch.int32)
        for s, n in enumerate(used):
            for i in range(n):
                self.table[s, i] = order.pop()
                self.ref[self.table[s, i]] = 1
        for s, n in enumerate(lengths):
            for pool in (self.k, self.v):
                for layer in range(layers):
                    self.rows(pool, layer, s, n)[:] = 0
                    self.write(pool, layer, s, torch.randn(n, kv, hd, generator=g).clamp(-6, 6).to(TYPES[dtype]))

    def at(self, s, n):
        pos = torch.arange(n)
        return self.table[s].long()[pos // self.page], pos % self.page

    def rows(self, pool, layer, s, n):
        a, b = self.at(s, n)
        return pool[layer][a, b]

    def write(self, pool, layer, s, x):
        a, b = self.at(s, x.shape[0])
        pool[layer][a, b] = x


def update(table, length, ref, source, add, page):
    """kv_update step by step: (table, len, ref, copies [(from, to)], status)."""
    n, width = table.shape
    pages = len(ref)
    source = list(range(n)) if source is None else [int(v) for v in source]
    add = [0] * n if add is None else [int(v) for v in add]
    status, plan = 0, []
    for d in range(n):
        s = source[d]
        if s < -1 or s >= n:
            status |= 1
            s = -1
        base = 0 if s < 0 else min(max(int(length[s]), 0), width * page)
        size = base + add[d]
        if size < 0 or size > width * page:
            status |= 2
            size = 0
        kept = min(base, size)
        whole, part = kept // page, kept % page > 0
        held = [int(x) for x in table[s, :whole + part]] if s >= 0 else []
        if any(x < 0 or x >= pages for x in held):
            status |= 8
        plan.append((size, whole, part, held))
    if status:
        return table.copy(), length.copy(), ref.copy(), [], status
    count = np.zeros(pages, np.int32)
    for size, whole, part, held in plan:
        for x in held[:whole]:
            count[x] += 1
    owner = {}
    for d, (size, whole, part, held) in enumerate(plan):
        if part:
            owner.setdefault(held[whole], d)
    free = [i for i in range(pages) if ref[i] <= 0]
    new = np.full_like(table, -1)
    copies = []
    for d, (size, whole, part, held) in enumerate(plan):
        keep = part and count[held[whole]] == 0 and owner[held[whole]] == d
        ids = held[:whole] + ([held[whole]] if keep else [])
        while len(ids) < -(-size // page):
            if not free:
                return table.copy(), length.copy(), ref.copy(), [], 4
            ids.append(free.pop(0))
            if part and not keep and len(ids) == whole + 1:
                copies.append((held[whole], ids[-1]))
        new[d, :len(ids)] = ids
    counts = np.zeros(pages, np.int32)
    for x in new[new >= 0]:
        counts[x] += 1
    return new, np.array([p[0] for p in plan], np.int32), counts, copies, 0


def compact(table, ref):
    """kv_compact: (table, ref, live pages, moves [(from, to)])."""
    live = int((ref > 0).sum())
    moves = list(zip([i for i in range(len(ref)) if i >= live and ref[i] > 0], [i for i in range(live) if ref[i] <= 0]))
    to = np.arange(len(ref), dtype=np.int32)
    new_ref = np.where(np.arange(len(ref)) < live, ref, 0).astype(np.int32)
    for a, b in moves:
        to[a] = b
        new_ref[b] = ref[a]
    new_ref[[i for i in range(live) if ref[i] <= 0 and i not in [b for _, b in moves]]] = 0
    ok = (table >= 0) & (table < len(ref))
    return np.where(ok, to[np.where(ok, table, 0)], -1).astype(np.int32), new_ref, live, moves
