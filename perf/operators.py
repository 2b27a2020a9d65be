"""Performance cases of the serving operators: attention over packed prompts and over a
paged KV cache, the cache's pages, and decode of a batch that shares a prefix.

  packed   causal attention of several prompts whose rows stand one after another
           (ops.attention_packed): no cache yet, K and V beside Q
  paged    the same attention, keys and values read from the pages of a cache
           (ops.attention_paged): single tokens, drafted tokens, a prompt's next chunk
  prefix   one token per sequence over a long prefix that all sequences share, then
           over what each has of its own (ops.attention_prefix)
  append   a layer's new K and V rows into the cache's pages (ops.kv_append)
  update   sequences forked, freed, cut and grown: page tables, counts of references,
           and the copies of pages that two sequences would write (ops.kv_update)
  compact  the pages in use moved to the front of the pool (ops.kv_compact)

Head layouts are those of the presets of gaje_hip.synth (9/3 x 64, 14/2 x 64, 12/2 x 128)
and generic ones; a cache has the presets' 24 to 30 layers where its pages are
copied, and one or two where one layer is read or written.
"""
import math
import os
import random
import sys

import numpy as np
import torch

own = False  # True: the framework's operators; False: their plain forms

DEV = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # a few short prompts together at the 0.5B heads: the smallest call, latency
        dict(name="packed-short-f32", kind="packed", dtype="f32", seqs=5, low=1, high=60, mix=1, heads=14, kv=2, hd=64),
        # several prompts of a batch in the framework's own type, 1.5B heads
        dict(name="packed-f32", kind="packed", dtype="f32", seqs=4, low=300, high=1500, mix=2, heads=12, kv=2, hd=128),
        # many ragged prompts in one pass, 1.5B heads
        dict(name="packed-bf16", kind="packed", dtype="bf16", seqs=24, low=1, high=2000, mix=3, heads=12, kv=2, hd=128),
        # one long document
        dict(name="packed-long-f16", kind="packed", dtype="f16", seqs=1, low=8190, high=8190, mix=4, heads=32, kv=8, hd=128),
        # a decode step of a full batch: one token each, contexts of all lengths
        dict(name="paged-decode-bf16", kind="paged", dtype="bf16", seqs=64, rows=1, low=50, high=4000, mix=5, heads=12, kv=2,
             hd=128, page=16),
        # a small batch over a system prompt, 0.5B heads
        dict(name="prefix-f32", kind="prefix", dtype="f32", seqs=16, prefix=1000, high=150, mix=6, heads=14, kv=2, hd=64, page=16),
        # many users of one long document
        dict(name="prefix-bf16", kind="prefix", dtype="bf16", seqs=64, prefix=16000, high=500, mix=7, heads=12, kv=2, hd=128,
             page=16),
        # one token's K and V of every sequence of a batch
        dict(name="append-token", kind="append", source="f32", dtype="f16", seqs=64, rows=1, mix=8, kv=2, hd=128, page=16),
        # the K and V rows of a prefill pass
        dict(name="append-prompts", kind="append", source="f32", dtype="f16", seqs=12, rows=1400, mix=9, kv=8, hd=128, page=16),
        # one prompt becomes sixteen samples
        dict(name="update-fork", kind="update", mode="fork", dtype="f16", seqs=16, context=1003, mix=10, layers=28, kv=2, hd=128,
             page=16),
        # a serving step of a large batch: finished sequences go, forks take places, all grow
        dict(name="update-step", kind="update", mode="step", dtype="f16", seqs=256, context=700, mix=11, layers=24, kv=2, hd=64,
             page=16),
        # a pool half empty after a busy hour
        dict(name="compact", kind="compact", dtype="f16", seqs=48, context=900, mix=12, layers=28, kv=2, hd=128, page=16),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


HEADS = [(14, 2, 64), (12, 2, 128), (9, 3, 64), (16, 16, 64), (32, 8, 128), (6, 1, 80), (4, 2, 256), (8, 8, 32)]


def draw(rng):
    kind = rng.choice(["packed", "packed", "packed", "paged", "paged", "prefix", "prefix", "append", "update", "compact"])
    heads, kv, hd = rng.choice(HEADS)
    dtype = rng.choice(["f32", "f16", "bf16"])
    mix, page = rng.randint(100, 10 ** 6), rng.choice([8, 16, 16, 32, 64])
    base = dict(kind=kind, dtype=dtype, mix=mix)
    if kind == "packed":
        high = _log(rng, 16, 4000 if dtype != "f32" else 2000)
        most = max(1, min(32, 8190 * 8190 * 32 // (8 * high * high * heads)))
        return dict(base, seqs=rng.randint(1, most), low=rng.choice([1, max(1, high // 2)]), high=high, heads=heads, kv=kv, hd=hd)
    if kind == "paged":
        seqs = _log(rng, 1, 96)
        high = _log(rng, 64, min(16000, 10 ** 9 // (seqs * kv * hd * 4)))
        return dict(base, seqs=seqs, rows=rng.choice([1, 1, 1, 4, 7, 40]), low=rng.choice([1, high // 2]), high=high, heads=heads,
                    kv=kv, hd=hd, page=page)
    if kind == "prefix":
        seqs = _log(rng, 2, 128)
        return dict(base, seqs=seqs, prefix=_log(rng, 64, min(16000, 10 ** 9 // (4 * seqs * heads))), high=_log(rng, 4, 500),
                    heads=heads, kv=kv, hd=hd, page=page)
    layers = rng.randint(8, 30)
    if kind == "append":
        seqs = _log(rng, 1, 64)
        return dict(base, source=rng.choice(["f32", dtype]), seqs=seqs, rows=_log(rng, 1, 20000 // seqs), kv=kv, hd=hd, page=page)
    context = _log(rng, 20, 2000)
    seqs = rng.randint(2, max(2, min(256, 2 * 10 ** 9 // (context * layers * kv * hd * 16))))
    if kind == "update":
        return dict(base, mode=rng.choice(["fork", "step"]), seqs=seqs, context=context, layers=layers, kv=kv, hd=hd, page=page)
    return dict(base, seqs=seqs, context=context, layers=layers, kv=kv, hd=hd, page=page)


# ------------------------------------------------------------- what a case has --
def _size(dtype):
    return 4 if dtype == "f32" else 2


def _lengths(case):
    """The lengths of a case's sequences, the same for every seed: packed prompts or
    cached positions, even over their range."""
    rng = random.Random(case["mix"])
    if case["kind"] in ("packed", "paged"):
        n = [rng.randint(case["low"], case["high"]) for _ in range(case["seqs"])]
        return [v + case["rows"] - 1 for v in n] if case["kind"] == "paged" else n
    if case["kind"] == "prefix":
        return [case["prefix"] + rng.randint(1, case["high"]) for _ in range(case["seqs"])]
    if case["kind"] == "append":
        return [case["rows"] + rng.randint(0, 200) for _ in range(case["seqs"])]
    if case["kind"] == "update" and case["mode"] == "fork":
        return [case["context"]] + [0] * (case["seqs"] - 1)
    return [rng.randint(case["context"] // 2, case["context"]) for _ in range(case["seqs"])]


def _rows(case):
    """New rows of each sequence of an append: ragged around the case's number."""
    rng = random.Random(case["mix"] + 1)
    return [rng.randint((case["rows"] + 1) // 2, case["rows"]) for _ in range(case["seqs"])]


def _change(case):
    """(source of each slot, change of its length) of an update."""
    rng, n = random.Random(case["mix"] + 1), case["seqs"]
    if case["mode"] == "fork":
        return [0] * n, [1] * n
    slots = list(range(n))
    rng.shuffle(slots)
    some = max(1, n // 10)
    source, add = list(range(n)), [1] * n
    for s in slots[:some]:            # finished, and their places taken by forks
        source[s] = slots[rng.randrange(min(some, n - 1), n)]
    for s in slots[some:min(2 * some, n - 1)]:  # finished
        source[s], add[s] = -1, 0
    for s in slots[2 * some:3 * some]:          # drafted tokens refused
        add[s] = -min(5, case["context"] // 2)
    return source, add


def _page_bytes(case):
    return case["layers"] * 2 * case["page"] * case["kv"] * case["hd"] * _size(case["dtype"])


def work(case):
    """Bytes and operations that one pass cannot do without."""
    kind, n, es = case["kind"], _lengths(case), _size(case["dtype"])
    if kind == "packed":
        pairs, t = sum(v * (v + 1) // 2 for v in n), sum(n)
        return {"bytes": es * t * case["hd"] * 2 * (case["heads"] + case["kv"]), "flops": 4 * pairs * case["hd"] * case["heads"]}
    if kind == "paged":
        r = case["rows"]
        pairs, t = sum(r * v - r * (r - 1) // 2 for v in n), r * len(n)
        return {"bytes": es * case["hd"] * 2 * (t * case["heads"] + sum(n) * case["kv"]), "flops": 4 * pairs * case["hd"] * case["heads"]}
    if kind == "prefix":
        rows = case["prefix"] + sum(v - case["prefix"] for v in n)
        return {"bytes": es * case["hd"] * 2 * (len(n) * case["heads"] + rows * case["kv"]),
                "flops": 4 * sum(n) * case["hd"] * case["heads"]}
    if kind == "append":
        return {"bytes": sum(_rows(case)) * 2 * case["kv"] * case["hd"] * (es + _size(case["source"])), "flops": 0}
    pages = sum(-(-v // case["page"]) for v in n)
    tables = 8 * pages + 8 * _pool_pages(case)  # entries and counts, read and written
    if kind == "update":
        source, add = _change(case)
        at = [n[s] if s >= 0 else 0 for s in source]
        split = [s for s, v, a in zip(source, at, add) if s >= 0 and min(v, v + a) % case["page"]]
        return {"bytes": tables + 2 * _page_bytes(case) * (len(split) - len(set(split))), "flops": 0}
    live = pages - pages // 2
    return {"bytes": tables + 2 * _page_bytes(case) * (live - live * live // _pool_pages(case)), "flops": 0}


# ------------------------------------------------------------------ inputs --
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _normal(g, dtype, *shape, std=1.0):
    return (torch.randn(*shape, generator=g, device=DEV) * std).to(TYPES[dtype])


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _offsets(rows):
    return _ints([0] + list(np.cumsum(rows)))


def _pool_pages(case):
    n = _lengths(case)
    pages = sum(-(-v // case["page"]) for v in n)
    return pages + (0 if case["kind"] == "compact" else 2 * case["seqs"]) + 3


def _cache(case, g, layers, lengths, extra=0):
    """A paged cache: K and V pools, the sequences' page tables (pages in random
    order, as after a while of serving), their lengths, the pages' counts."""
    page, kv, hd, n = case["page"], case["kv"], case["hd"], len(lengths)
    pages = _pool_pages(case)
    shape = (layers, pages, page, kv, hd)
    k, v = _normal(g, case["dtype"], *shape), _normal(g, case["dtype"], *shape)
    width = -(-(max(lengths) + extra) // page) + 1
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    used = torch.tensor([-(-x // page) for x in lengths], device=DEV)
    at = torch.arange(width, device=DEV)[None, :]
    start = (torch.cumsum(used, 0) - used)[:, None]
    table = torch.where(at < used[:, None], order[(start + at).clamp(max=pages - 1)], -1).to(torch.int32)
    ref = torch.zeros(pages, dtype=torch.int32, device=DEV)
    ref[table[table >= 0].long()] = 1
    return dict(k=k, v=v, table=table.contiguous(), length=_ints(lengths), ref=ref)


def prepare(case, seed):
    g, kind = _gen(seed), case["kind"]
    n = _lengths(case)
    if kind == "packed":
        heads, kv, hd, t = case["heads"], case["kv"], case["hd"], sum(n)
        # the rows of a fused QKV product: [q heads | k heads | v heads]
        x = _normal(g, case["dtype"], t, (heads + 2 * kv) * hd)
        x[:, :heads * hd] *= 1.5
        return dict(case=case, x=x, off=_offsets(n), most=max(n), out=torch.empty(t, heads * hd, dtype=x.dtype, device=DEV))
    if kind == "paged":
        s = _cache(case, g, 1, n)
        t = case["rows"] * len(n)
        q = _normal(g, case["dtype"], t, case["heads"] * case["hd"], std=1.5)
        return dict(s, case=case, q=q, off=_offsets([case["rows"]] * len(n)), most=max(n), out=torch.empty_like(q))
    if kind == "prefix":
        s = _cache(case, g, 1, n)
        whole, part = divmod(case["prefix"], case["page"])
        if part:  # every sequence has its own copy of the page that the prefix ends in
            ends = s["table"][:, whole].long()
            for pool in (s["k"], s["v"]):
                pool[0, ends, :part] = pool[0, ends[0], :part].clone()
        s["ref"][s["table"][1:, :whole].reshape(-1).long()] = 0
        s["table"][1:, :whole] = s["table"][0, :whole]
        s["ref"][s["table"][0, :whole].long()] = len(n)
        q = _normal(g, case["dtype"], len(n), case["heads"] * case["hd"], std=1.5)
        return dict(s, case=case, q=q, most=max(n), out=torch.empty_like(q))
    if kind == "append":
        s = _cache(case, g, 2, n)
        rows = _rows(case)
        x = _normal(g, case["source"], sum(rows), 2 * case["kv"] * case["hd"])
        return dict(s, case=case, x=x, off=_offsets(rows))
    s = _cache(case, g, case["layers"], n, extra=1)
    out = dict(new_table=torch.empty_like(s["table"]), new_ref=torch.empty_like(s["ref"]))
    if kind == "update":
        source, add = _change(case)
        return dict(s, **out, case=case, source=_ints(source), add=_ints(add), new_length=torch.empty_like(s["length"]),
                    status=torch.empty(1, dtype=torch.int32, device=DEV))
    # compact: half of the sequences are gone
    s["table"][1::2] = -1
    s["length"][1::2] = 0
    s["ref"].zero_()
    s["ref"][s["table"][s["table"] >= 0].long()] = 1
    return dict(s, **out, case=case, live=torch.empty(1, dtype=torch.int32, device=DEV))


# ------------------------------------------------------------- plain forms --
def _slots(table, page, pos):
    """Rows of a layer's pool (as [pages * page]) of positions pos [n][m] of n sequences."""
    at = torch.gather(table.long(), 1, (pos // page).clamp(max=table.shape[1] - 1))
    return at.clamp(min=0) * page + pos % page


def _softmax_rows(s):
    """Softmax of the last axis in place; rows without a visible key give zeros."""
    m = s.amax(-1, keepdim=True)
    s.sub_(torch.where(torch.isinf(m), 0.0, m)).exp_()
    return s.div_(s.sum(-1, keepdim=True).clamp(min=1e-37))


def _causal(q, k, v, first, kv):
    """q [S][L][heads][hd] against k, v [S][M][kv][hd]: row i sees the keys up to first + i."""
    n, l, heads, hd = q.shape
    group = heads // kv
    q = q.view(n, l, kv, group, hd).permute(0, 2, 3, 1, 4).reshape(n, kv, group * l, hd)
    k, v = k.permute(0, 2, 3, 1).contiguous(), v.permute(0, 2, 1, 3).contiguous()
    s = torch.matmul(q, k).mul_(1.0 / math.sqrt(hd)).view(n, kv, group, l, -1)
    last = first[:, None] + torch.arange(l, device=DEV)[None, :]
    hidden = torch.arange(k.shape[3], device=DEV)[None, None, :] > last[:, :, None]
    s.masked_fill_(hidden[:, None, None], -math.inf)
    o = torch.matmul(_softmax_rows(s).view(n, kv, group * l, -1), v)
    return o.view(n, kv, group, l, hd).permute(0, 3, 1, 2, 4).reshape(n, l, heads, hd)


def _plain_packed(s):
    case, x, off = s["case"], s["x"], s["off"].long()
    heads, kv, hd = case["heads"], case["kv"], case["hd"]
    n, pos = off[1:] - off[:-1], torch.arange(s["most"], device=DEV)
    at = (off[:-1, None] + pos[None, :]).clamp(max=x.shape[0] - 1)
    rows = x[at].float()
    q, k, v = rows.split([heads * hd, kv * hd, kv * hd], dim=2)
    o = _causal(q.unflatten(2, (heads, hd)), k.unflatten(2, (kv, hd)), v.unflatten(2, (kv, hd)), torch.zeros_like(n), kv)
    return o[pos[None, :] < n[:, None]].view(-1, heads * hd).to(x.dtype)


def _plain_paged(s):
    case, length = s["case"], s["length"].long()
    heads, kv, hd, rows, n = case["heads"], case["kv"], case["hd"], case["rows"], s["length"].shape[0]
    pos = torch.arange(s["most"], device=DEV)[None, :].expand(n, -1)
    at = _slots(s["table"], case["page"], pos)
    k, v = (s[p][0].reshape(-1, kv, hd)[at].float() for p in ("k", "v"))
    o = _causal(s["q"].float().view(n, rows, heads, hd), k, v, length - rows, kv)
    return o.reshape(n * rows, heads * hd).to(s["q"].dtype)


def _plain_prefix(s):
    case, length = s["case"], s["length"].long()
    heads, kv, hd, first, n = case["heads"], case["kv"], case["hd"], case["prefix"], s["length"].shape[0]
    scale = 1.0 / math.sqrt(hd)
    q = s["q"].float().view(n, kv, heads // kv, hd)
    k, v = (s[p][0].reshape(-1, kv, hd) for p in ("k", "v"))
    # the shared rows, once for all queries of a head
    at = _slots(s["table"][:1], case["page"], torch.arange(first, device=DEV)[None, :])[0]
    kp, vp = k[at].float().permute(1, 2, 0).contiguous(), v[at].float().transpose(0, 1).contiguous()
    qp = q.transpose(0, 1).reshape(kv, -1, hd)
    sp = torch.matmul(qp, kp).mul_(scale).view(kv, n, -1, first).transpose(0, 1)
    # and each sequence's own
    pos = (first + torch.arange(s["most"] - first, device=DEV))[None, :].expand(n, -1)
    at = _slots(s["table"], case["page"], pos)
    ks, vs = k[at].float().permute(0, 2, 3, 1).contiguous(), v[at].float().transpose(1, 2).contiguous()
    so = torch.matmul(q, ks).mul_(scale).masked_fill_((pos >= length[:, None])[:, None, None], -math.inf)
    p = _softmax_rows(torch.cat([sp, so], dim=3))
    o = torch.matmul(p[..., :first].transpose(0, 1).reshape(kv, -1, first), vp).view(kv, n, -1, hd).transpose(0, 1)
    o = o + torch.matmul(p[..., first:], vs)
    return o.reshape(n, heads * hd).to(s["q"].dtype)


def _plain_append(s):
    case, off, length = s["case"], s["off"].long(), s["length"].long()
    kv, hd, t = case["kv"], case["hd"], s["x"].shape[0]
    row = torch.arange(t, device=DEV)
    seq = torch.searchsorted(off, row, right=True) - 1
    pos = length[seq] - off[seq + 1] + row
    at = _slots(s["table"][seq], case["page"], pos[:, None])[:, 0]
    k, v = s["x"].view(t, 2, kv, hd).to(s["k"].dtype).unbind(1)
    s["k"][1].view(-1, kv, hd)[at] = k
    s["v"][1].view(-1, kv, hd)[at] = v
    return {"k": s["k"], "v": s["v"]}


def _plain_update(s):
    page, table, pages = s["case"]["page"], s["table"].long(), s["ref"].shape[0]
    n, width = table.shape
    slot, column = torch.arange(n, device=DEV), torch.arange(width, device=DEV)[None, :]
    source = s["source"].long()
    base = torch.where(source < 0, 0, s["length"].long()[source.clamp(min=0)])
    length = base + s["add"]
    kept = torch.minimum(base, length)
    whole, part = kept // page, kept % page > 0
    rows = table[source.clamp(min=0)]
    full = column < whole[:, None]
    counts = torch.zeros(pages + 1, dtype=torch.long, device=DEV)
    counts.index_add_(0, torch.where(full, rows, pages).reshape(-1), torch.ones(n * width, dtype=torch.long, device=DEV))
    split = torch.where(part, rows.gather(1, whole[:, None].clamp(max=width - 1))[:, 0], pages)
    owner = torch.full((pages + 1,), n, dtype=torch.long, device=DEV).scatter_reduce(0, split, slot, "amin")
    keeps = part & (counts[split] == 0) & (owner[split] == slot)
    need = (length + page - 1) // page - whole - keeps.long()
    free = torch.argsort((s["ref"] != 0).int(), stable=True)
    start = (torch.cumsum(need, 0) - need - whole - keeps.long())[:, None]
    fresh = free[(start + column).clamp(0, pages - 1)]
    same = full | (keeps[:, None] & (column == whole[:, None]))
    new = torch.where(same, rows, torch.where(column < ((length + page - 1) // page)[:, None], fresh, -1))
    copied = part & ~keeps
    old_page, new_page = split[copied], new.gather(1, whole[:, None].clamp(max=width - 1))[:, 0][copied]
    s["k"][:, new_page] = s["k"][:, old_page]
    s["v"][:, new_page] = s["v"][:, old_page]
    ref = torch.zeros(pages + 1, dtype=torch.int32, device=DEV)
    ref.index_add_(0, torch.where(new < 0, pages, new).reshape(-1), torch.ones(n * width, dtype=torch.int32, device=DEV))
    return {"table": new.int(), "length": length.int(), "ref": ref[:-1], "status": torch.zeros_like(s["status"]),
            "k": s["k"], "v": s["v"]}


def _plain_compact(s):
    live = s["ref"] > 0
    count, index = live.sum(), torch.arange(live.shape[0], device=DEV)
    moved, holes = index[live & (index >= count)], index[~live & (index < count)]
    to = index.clone()
    to[moved] = holes
    s["k"][:, holes] = s["k"][:, moved]
    s["v"][:, holes] = s["v"][:, moved]
    ref = torch.zeros_like(s["ref"])
    ref[to[live]] = s["ref"][live]
    table = torch.where(s["table"] < 0, -1, to[s["table"].clamp(min=0).long()]).int()
    return {"table": table, "ref": ref, "live": count.int().view(1), "k": s["k"], "v": s["v"]}


# ------------------------------------------------------- the framework's calls --
class _At:
    """A torch tensor's memory, from one of its elements on, as the operators take it."""

    def __init__(self, t, first=0):
        self.ptr = t.data_ptr() + first * t.element_size()
        self.nbytes = (t.numel() - first) * t.element_size()


def _own(s):
    here = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "gaje-semantic-compression_amd")
    if here not in sys.path:
        sys.path.insert(0, here)
    from gaje_hip import ops
    case, kind = s["case"], s["case"]["kind"]
    stream = torch.cuda.current_stream().cuda_stream
    if "cache" not in s and kind != "packed":
        s["cache"] = ops.kv_pages(_At(s["k"]), _At(s["v"]), _At(s["table"]), _At(s["length"]), _At(s["ref"]),
                                  n_layer=s["k"].shape[0], n_pages=s["k"].shape[1], page=case["page"],
                                  n_seq=s["table"].shape[0], max_pages=s["table"].shape[1], n_head_kv=case["kv"],
                                  head_dim=case["hd"], dtype=case["dtype"])
    if "ws" not in s and kind != "append":
        if kind == "packed":
            size = ops.attention_packed_workspace(s["x"].shape[0], case["seqs"], case["heads"], case["kv"], case["hd"])
        elif kind == "paged":
            size = ops.attention_paged_workspace(s["cache"], s["q"].shape[0], case["heads"])
        elif kind == "prefix":
            size = ops.attention_prefix_workspace(s["cache"], case["prefix"], case["heads"])
        else:
            size = ops.kv_workspace(s["cache"])
        s["ws"] = torch.empty(max(size, 256), dtype=torch.uint8, device=DEV)
    if kind == "packed":
        heads, kv, hd, x = case["heads"], case["kv"], case["hd"], s["x"]
        ops.attention_packed(_At(x), x.shape[1], _At(x, heads * hd), x.shape[1], _At(x, (heads + kv) * hd), x.shape[1],
                             _At(s["off"]), case["seqs"], x.shape[0], heads, kv, hd, 1.0 / math.sqrt(hd), _At(s["out"]),
                             heads * hd, _At(s["ws"]), dtype=case["dtype"], stream=stream)
        return s["out"]
    if kind == "paged":
        width = s["q"].shape[1]
        ops.attention_paged(_At(s["q"]), width, s["cache"], 0, _At(s["off"]), s["q"].shape[0], case["heads"],
                            1.0 / math.sqrt(case["hd"]), _At(s["out"]), width, _At(s["ws"]), stream=stream)
        return s["out"]
    if kind == "prefix":
        width = s["q"].shape[1]
        ops.attention_prefix(_At(s["q"]), width, s["cache"], 0, _At(s["table"]), case["prefix"], case["heads"],
                             1.0 / math.sqrt(case["hd"]), _At(s["out"]), width, _At(s["ws"]), stream=stream)
        return s["out"]
    if kind == "append":
        x, width = s["x"], case["kv"] * case["hd"]
        ops.kv_append(s["cache"], 1, _At(x), 2 * width, _At(x, width), 2 * width, _At(s["off"]), x.shape[0],
                      source=case["source"], stream=stream)
        return {"k": s["k"], "v": s["v"]}
    if kind == "update":
        ops.kv_update(s["cache"], _At(s["new_table"]), _At(s["new_length"]), _At(s["new_ref"]), _At(s["status"]), _At(s["ws"]),
                      source=_At(s["source"]), add=_At(s["add"]), stream=stream)
        return {"table": s["new_table"], "length": s["new_length"], "ref": s["new_ref"], "status": s["status"], "k": s["k"],
                "v": s["v"]}
    ops.kv_compact(s["cache"], _At(s["new_table"]), _At(s["new_ref"]), _At(s["live"]), _At(s["ws"]), stream=stream)
    return {"table": s["new_table"], "ref": s["new_ref"], "live": s["live"], "k": s["k"], "v": s["v"]}


PLAIN = {"packed": _plain_packed, "paged": _plain_paged, "prefix": _plain_prefix, "append": _plain_append,
         "update": _plain_update, "compact": _plain_compact}


def run(state):
    if own:
        return _own(state)
    return PLAIN[state["case"]["kind"]](state)


# ------------------------------------------------------------ in 64 bits --
def exact(case, seed):
    """The attention of each row from its definition, one head at a time; the appended
    pools as the values they are given.  Page numbers and copies have no 64-bit value."""
    s, kind = prepare(case, seed), case["kind"]
    if kind in ("update", "compact"):
        return None
    n, hd, kv = _lengths(case), case["hd"], case["kv"]
    if kind == "append":
        k, v = s["k"].double(), s["v"].double()
        x, row, width = s["x"].double(), 0, kv * hd
        for i, count in enumerate(_rows(case)):
            pos = torch.arange(n[i] - count, n[i], device=DEV)
            pages = s["table"][i].long()[pos // case["page"]]
            k[1, pages, pos % case["page"]] = x[row:row + count, :width].view(count, kv, hd)
            v[1, pages, pos % case["page"]] = x[row:row + count, width:].view(count, kv, hd)
            row += count
        return {"k": k, "v": v}
    heads = case["heads"]
    group = heads // kv
    out, row = [], 0
    for i, length in enumerate(n):
        if kind == "packed":
            x = s["x"][row:row + length].double()
            q, k, v = x[:, :heads * hd], x[:, heads * hd:(heads + kv) * hd], x[:, (heads + kv) * hd:]
            k, v, new = k.view(length, kv, hd), v.view(length, kv, hd), length
        else:
            new = case["rows"] if kind == "paged" else 1
            pages = s["table"][i, :-(-length // case["page"])].long()
            k, v = (s[p][0][pages].reshape(-1, kv, hd)[:length].double() for p in ("k", "v"))
            q = s["q"][row:row + new].double()
        o = torch.empty(new, heads, hd, dtype=torch.float64, device=DEV)
        seen = torch.ones(new, length, dtype=torch.bool, device=DEV).tril_(length - new)
        for h in range(heads):
            a = (q[:, h * hd:(h + 1) * hd] @ k[:, h // group].T.contiguous()) / math.sqrt(hd)
            o[:, h] = torch.softmax(a.masked_fill_(~seen, -math.inf), dim=1) @ v[:, h // group].contiguous()
        out.append(o.view(new, heads * hd))
        row += new
    return torch.cat(out)
