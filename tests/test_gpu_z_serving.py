"""The serving operators on the GPU against their 64-bit forms (serving_ref): attention
over packed prompts, over a paged cache and over a shared prefix; the cache's pages."""
import math

import numpy as np
import pytest
import torch

import serving_ref as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from gaje_hip import ops
    if ops.device_count() < 1:
        pytest.fail("no HIP device visible")
    return ops


class Buf:
    """A torch tensor's memory from one of its elements on."""

    def __init__(self, t, first=0):
        self.t, self.ptr = t, t.data_ptr() + first * t.element_size()
        self.nbytes = (t.numel() - first) * t.element_size()


def ints(v):
    return torch.tensor(list(v), dtype=torch.int32, device="cuda")


def offsets(rows):
    return ints([0] + list(np.cumsum(rows)))


def space(n):
    return torch.full((max(int(n), 256) // 4 + 1,), math.nan, device="cuda")


def normal(shape, dtype, seed, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * std).clamp(-6, 6).to(R.TYPES[dtype])


def close(got, ref, tol, what=""):
    off = (got.double().cpu() - ref).abs()
    ok = (off <= tol) | (torch.isnan(ref) & torch.isnan(got.double().cpu()))
    assert bool(ok.all()), (what, (off / tol.clamp(min=1e-300)).max().item(), int((~ok).sum()))


def run_packed(ops, x, rows, H, G, hd, scale, stream=None, off=None, T=None, ldo=None):
    """x [T][>= (H + 2 G) hd]: q, k and v as columns; returns out [T][ldo] over a sentinel."""
    T, ld = T or x.shape[0], x.shape[1]
    ldo = ldo or H * hd
    out = torch.full((T, ldo), 7.0, dtype=x.dtype, device="cuda")
    ws = space(ops.attention_packed_workspace(T, len(rows), H, G, hd))
    dtype = {v: k for k, v in R.TYPES.items()}[x.dtype]
    ops.attention_packed(Buf(x), ld, Buf(x, H * hd), ld, Buf(x, (H + G) * hd), ld, Buf(off if off is not None else offsets(rows)),
                         len(rows), T, H, G, hd, scale, Buf(out), ldo, Buf(ws), dtype=dtype, stream=stream)
    return out


def check_packed(x, out, rows, H, G, hd, scale, dtype):
    at, x, out = 0, x.cpu(), out.cpu()
    for s, n in enumerate(rows):
        r = x[at:at + n]
        q, k, v = (r[:, a * hd:b * hd].reshape(n, b - a, hd) for a, b in ((0, H), (H, H + G), (H + G, H + 2 * G)))
        ref, mass, top = R.attend(q, k, v, 0, scale)
        close(out[at:at + n, :H * hd].reshape(n, H, hd), ref, R.bound(dtype, ref, mass, top, hd, n), (s, n))
        at += n


HEADS = [(14, 2, 64), (12, 2, 128), (9, 3, 64), (4, 4, 8), (5, 1, 24), (6, 1, 80), (4, 2, 256), (3, 3, 136), (40, 2, 32)]
ROWS = [[1], [2, 0, 1], [37, 5, 1, 0, 64, 17], [129, 63, 65, 200]]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("H,G,hd", HEADS)
@pytest.mark.parametrize("rows", ROWS, ids=str)
def test_packed(ops, dtype, H, G, hd, rows):
    x = normal((sum(rows), (H + 2 * G) * hd), dtype, seed=hd + sum(rows)).cuda()
    scale = 1.3 / math.sqrt(hd)
    check_packed(x, run_packed(ops, x, rows, H, G, hd, scale), rows, H, G, hd, scale, dtype)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows", [[1100], [700, 3, 900], [1] * 130, [5] * 70 + [400]], ids=lambda r: f"{len(r)}x{max(r)}")
def test_packed_long(ops, dtype, rows):
    H, G, hd = 6, 2, 64
    x = normal((sum(rows), (H + 2 * G) * hd), dtype, seed=sum(rows)).cuda()
    check_packed(x, run_packed(ops, x, rows, H, G, hd, 0.125), rows, H, G, hd, 0.125, dtype)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_packed_large_scores(ops, dtype):
    """Scores to some hundreds, where one key takes nearly all the weight."""
    rows, H, G, hd = [150, 90], 4, 2, 64
    x = normal((sum(rows), (H + 2 * G) * hd), dtype, seed=5)
    x[:, :H * hd] *= 8
    x = x.cuda()
    check_packed(x, run_packed(ops, x, rows, H, G, hd, 1.0), rows, H, G, hd, 1.0, dtype)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_packed_strides_and_rows_behind(ops, dtype):
    """Wider rows on both sides; rows before the first and behind the last sequence keep what they had."""
    rows, H, G, hd = [33, 70], 6, 2, 64
    T, width = 2 + sum(rows) + 9, (H + 2 * G) * hd + 24
    x = normal((T, width), dtype, seed=9)
    x[:2] = math.nan
    x[-9:] = math.nan
    x = x.cuda()
    out = run_packed(ops, x, rows, H, G, hd, 0.1, off=ints([2, 35, 105]), ldo=H * hd + 16)
    check_packed(x[2:], out[2:], rows, H, G, hd, 0.1, dtype)
    o = out.float().cpu()
    assert bool((o[:2] == 7).all()) and bool((o[-9:] == 7).all()) and bool((o[:, H * hd:] == 7).all())


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("n", [70, 300])
def test_packed_values_that_are_not_seen(ops, dtype, bad, n):
    """A key or value that is no number reaches the rows that see it and no others."""
    H, G, hd = 6, 2, 64
    x = normal((n, (H + 2 * G) * hd), dtype, seed=n)
    x[n - 7, (H + G) * hd + 5] = bad      # a value of K/V head 0
    x[n - 3, H * hd + hd + 9] = bad       # a key of K/V head 1
    out = run_packed(ops, x.cuda(), [n], H, G, hd, 0.1).cpu().reshape(n, H, hd)
    clean = x.clone()
    clean[n - 7, (H + G) * hd + 5] = 0
    clean[n - 3, H * hd + hd + 9] = 0
    q, k, v = (clean[:, a * hd:b * hd].reshape(n, b - a, hd) for a, b in ((0, H), (H, H + G), (H + G, H + 2 * G)))
    ref, mass, top = R.attend(q, k, v, 0, 0.1)
    tol = R.bound(dtype, ref, mass, top, hd, n)
    close(out[:n - 7], ref[:n - 7], tol[:n - 7])
    close(out[n - 7:n - 3, 3:], ref[n - 7:n - 3, 3:], tol[n - 7:n - 3, 3:])
    others = [d for d in range(hd) if d != 5]
    close(out[n - 7:, :3][..., others], ref[n - 7:, :3][..., others], tol[n - 7:, :3][..., others])
    seen = out[n - 7:, :3, 5].float()
    assert bool(torch.isnan(seen).all()) if math.isnan(bad) else bool((seen == bad).all())
    if math.isnan(bad):
        assert bool(torch.isnan(out[n - 3:, 3:].float()).all())


def device_cache(ops, c):
    t = dict(k=c.k.cuda(), v=c.v.cuda(), table=c.table.cuda(), length=ints(c.lengths), ref=c.ref.cuda())
    layers, pages, page, kv, hd = c.k.shape
    h = ops.kv_pages(Buf(t["k"]), Buf(t["v"]), Buf(t["table"]), Buf(t["length"]), Buf(t["ref"]), n_layer=layers, n_pages=pages,
                     page=page, n_seq=len(c.lengths), max_pages=c.max_pages, n_head_kv=kv, head_dim=hd, dtype=c.dtype)
    return t, h


def run_paged(ops, h, q, rows, H, scale, layer=0, stream=None):
    out = torch.full(q.shape, 7.0, dtype=q.dtype, device="cuda")
    ws = space(ops.attention_paged_workspace(h, q.shape[0], H))
    ops.attention_paged(Buf(q), q.shape[1], h, layer, Buf(offsets(rows)), q.shape[0], H, scale, Buf(out), q.shape[1], Buf(ws),
                        stream=stream)
    return out


def check_paged(c, q, out, rows, H, scale, layer=0):
    at, hd = 0, c.k.shape[4]
    q, out = q.cpu(), out.cpu()
    for s, n in enumerate(rows):
        m = c.lengths[s]
        k, v = c.rows(c.k, layer, s, m), c.rows(c.v, layer, s, m)
        ref, mass, top = R.attend(q[at:at + n].reshape(n, H, hd), k, v, m - n, scale)
        close(out[at:at + n].reshape(n, H, hd), ref, R.bound(c.dtype, ref, mass, top, hd, m), (s, n, m))
        at += n


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("H,G,hd", HEADS)
@pytest.mark.parametrize("page", [8, 16, 128])
def test_paged_tokens(ops, dtype, H, G, hd, page):
    """One token each, contexts from one position on; an idle sequence; NaN in all rows no position is in."""
    lengths, rows = [1, 2, 0, 17, 64, 65, 300], [1, 1, 0, 1, 1, 1, 1]
    c = R.Cache(lengths, page, G, hd, dtype, layers=2, seed=hd)
    _, h = device_cache(ops, c)
    q = normal((sum(rows), H * hd), dtype, seed=3).cuda()
    check_paged(c, q, run_paged(ops, h, q, rows, H, 1 / math.sqrt(hd), layer=1), rows, H, 1 / math.sqrt(hd), layer=1)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("H,G,hd,page", [(14, 2, 64, 16), (12, 2, 128, 32), (6, 1, 80, 8), (8, 8, 32, 64), (40, 2, 64, 16)])
@pytest.mark.parametrize("rows,lengths", [([5, 5, 5], [5, 123, 700]), ([1, 40, 0, 130], [2000, 40, 9, 1000]),
                                          ([3, 9, 4], [0, 5, 4])], ids=["drafts", "mixed", "more-rows-than-positions"])
def test_paged_rows(ops, dtype, H, G, hd, page, rows, lengths):
    c = R.Cache(lengths, page, G, hd, dtype, seed=hd)
    _, h = device_cache(ops, c)
    q = normal((sum(rows), H * hd), dtype, seed=4).cuda()
    check_paged(c, q, run_paged(ops, h, q, rows, H, 0.11), rows, H, 0.11)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("seqs", [1, 3, 90])
def test_paged_long(ops, dtype, seqs):
    """Few sequences over long caches (the keys are split), and many."""
    H, G, hd = 6, 2, 64
    lengths = [4000 - 37 * i for i in range(seqs)] if seqs < 10 else [1 + (i * 131) % 600 for i in range(seqs)]
    c = R.Cache(lengths, 16, G, hd, dtype, seed=seqs, max_pages=512)
    _, h = device_cache(ops, c)
    rows = [1] * seqs
    q = normal((seqs, H * hd), dtype, seed=seqs).cuda()
    check_paged(c, q, run_paged(ops, h, q, rows, H, 0.125), rows, H, 0.125)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_paged_bad_pages(ops, dtype):
    """Entries outside the pool read as rows of zeros; lengths past the table are the table's."""
    H, G, hd, page = 6, 2, 64, 16
    c = R.Cache([100, 64], page, G, hd, dtype, max_pages=8)
    t, h = device_cache(ops, c)
    n = c.n_pages
    t["table"][0, 2] = n
    t["table"][0, 4] = -5
    t["table"][1, 1] = 2 ** 31 - 1
    t["length"][1] = 10 ** 9
    t["table"][1, 4:] = -1
    q = normal((2, H * hd), dtype, seed=4).cuda()
    out = run_paged(ops, h, q, [1, 1], H, 0.11).cpu()
    for s, m, holes in ((0, 100, (2, 4)), (1, 128, (1, 4, 5, 6, 7))):
        k, v = torch.zeros(m, G, hd, dtype=q.dtype), torch.zeros(m, G, hd, dtype=q.dtype)
        have = min(m, c.lengths[s])
        k[:have], v[:have] = c.rows(c.k, 0, s, have), c.rows(c.v, 0, s, have)
        for i in holes:
            k[i * page:(i + 1) * page], v[i * page:(i + 1) * page] = 0, 0
        ref, mass, top = R.attend(q[s:s + 1].cpu().reshape(1, H, hd), k, v, m - 1, 0.11)
        close(out[s].reshape(1, H, hd), ref, R.bound(dtype, ref, mass, top, hd, m), s)


def test_paged_offsets_past_32_bits(ops):
    """Rows whose elements lie past 2^31 of their pool."""
    H, G, hd, page, n_pages = 4, 2, 128, 64, 140000
    k = torch.empty(n_pages, page, G, hd, dtype=torch.float16, device="cuda")
    v = torch.empty_like(k)
    assert k.numel() > 2 ** 31
    length, ids = 150, [n_pages - 1, 3, n_pages - 7]
    g = torch.Generator().manual_seed(2)
    rows = [torch.randn(3 * page, G, hd, generator=g).half() for _ in range(2)]
    for pool, r in zip((k, v), rows):
        pool[ids] = r.view(3, page, G, hd).cuda()
    table, ln, ref_ = ints(ids).view(1, 3), ints([length]), torch.ones(n_pages, dtype=torch.int32, device="cuda")
    h = ops.kv_pages(Buf(k), Buf(v), Buf(table), Buf(ln), Buf(ref_), n_layer=1, n_pages=n_pages, page=page, n_seq=1,
                     max_pages=3, n_head_kv=G, head_dim=hd, dtype="f16")
    for n in (1, 150):
        q = normal((n, H * hd), "f16", seed=n).cuda()
        out = run_paged(ops, h, q, [n], H, 0.08).cpu()
        ref, mass, top = R.attend(q.cpu().reshape(n, H, hd), rows[0][:length], rows[1][:length], length - n, 0.08)
        close(out.reshape(n, H, hd), ref, R.bound("f16", ref, mass, top, hd, length))
    x = normal((2, 2 * G * hd), "f16", seed=8).cuda()
    ops.kv_append(h, 0, Buf(x), 2 * G * hd, Buf(x, G * hd), 2 * G * hd, Buf(ints([0, 2])), 2, source="f16")
    torch.cuda.synchronize()
    assert torch.equal(k[ids[2], 20:22].reshape(2, -1), x[:, :G * hd]) and torch.equal(v[ids[2], 20:22].reshape(2, -1), x[:, G * hd:])


def run_prefix(ops, h, q, prefix, H, scale, table, layer=0, stream=None):
    out = torch.full(q.shape, 7.0, dtype=q.dtype, device="cuda")
    ws = space(ops.attention_prefix_workspace(h, prefix, H))
    ops.attention_prefix(Buf(q), q.shape[1], h, layer, Buf(table), prefix, H, scale, Buf(out), q.shape[1], Buf(ws),
                         stream=stream)
    return out


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("H,G,hd,page", [(14, 2, 64, 16), (12, 2, 128, 32), (9, 3, 64, 8), (6, 1, 80, 64), (4, 2, 256, 16), (4, 4, 8, 16),
                                         (40, 2, 32, 16)])
@pytest.mark.parametrize("prefix,own", [(0, [5, 1, 0, 90]), (100, [3, 0, 1, 40, 700]), (1000, [1, 30] * 12), (37, [-30, -37, 0, 5])],
                         ids=["none", "ragged", "many", "shorter-than-the-prefix"])
def test_prefix(ops, dtype, H, G, hd, page, prefix, own):
    lengths = [prefix + n for n in own]
    first = max(range(len(own)), key=lambda s: lengths[s])
    c = R.Cache(lengths, page, G, hd, dtype, layers=2, seed=prefix)
    for s, n in enumerate(lengths):  # all sequences begin with the same rows, in pages of their own
        n = min(n, prefix)
        for pool in (c.k, c.v):
            c.write(pool, 1, s, c.rows(pool, 1, first, n).clone())
    _, h = device_cache(ops, c)
    q = normal((len(own), H * hd), dtype, seed=prefix).cuda()
    out = run_prefix(ops, h, q, prefix, H, 0.12, c.table[first].clone().cuda(), layer=1)
    check_paged(c, q, out, [1] * len(own), H, 0.12, layer=1)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_prefix_values_that_are_not_seen(ops, dtype):
    """A NaN in the prefix reaches the sequences that are long enough, one in a sequence's own rows only that one."""
    H, G, hd, prefix, own = 6, 2, 64, 300, [5, -20, 4, 1]
    c = R.Cache([prefix + n for n in own], 16, G, hd, dtype)
    for s, n in enumerate(c.lengths):
        for pool in (c.k, c.v):
            c.write(pool, 0, s, c.rows(pool, 0, 0, min(n, prefix)).clone())
    a, b = c.at(0, prefix)
    c.v[0, a[290], b[290], 0, 3] = math.nan
    a, b = c.at(2, prefix + 4)
    c.v[0, a[-1], b[-1], 1, 9] = math.nan
    _, h = device_cache(ops, c)
    q = normal((4, H * hd), dtype, seed=1).cuda()
    out = run_prefix(ops, h, q, prefix, H, 0.12, c.table[0].clone().cuda()).float().cpu().reshape(4, H, hd)
    nan = torch.zeros(4, H, hd, dtype=torch.bool)
    nan[[0, 2, 3], :3, 3] = True
    nan[2, 3:, 9] = True
    assert torch.equal(torch.isnan(out), nan)


# ---------------------------------------------------------------- the pages --
def run_update(ops, t, h, source, add):
    new = dict(table=torch.full_like(t["table"], 77), length=torch.full_like(t["length"], 77), ref=torch.full_like(t["ref"], 77))
    status, ws = ints([99]), space(ops.kv_workspace(h))
    ops.kv_update(h, Buf(new["table"]), Buf(new["length"]), Buf(new["ref"]), Buf(status), Buf(ws),
                  source=None if source is None else Buf(ints(source)), add=None if add is None else Buf(ints(add)))
    return new, int(status.cpu()[0])


UPDATES = [
    ([20, 0, 5], None, [1, 1, 1]), ([20, 0, 0, 0], [0, 0, 0, 0], [1, 1, 1, 1]), ([16, 0, 0], [0, 0, 0], None),
    ([20, 33, 7], [-1, 1, 1], [5, 0, 1]), ([20, 33, 7], [1, 2, 0], [1, 1, 1]), ([20, 33, 7], [0, 1, 2], [-20, -2, -7]),
    ([40, 0, 0], [0, 0, 0], [0, -5, -25]), ([40, 0], [0, 0], [-3, -12]), ([8, 9], [1, 1], [0, -9]),
    ([20, 33, 7], [-1, -1, -1], [17, 1, 0]), ([0, 0], None, None), ([47, 3], None, [1, 60]),
]


@pytest.mark.parametrize("lengths,source,add", UPDATES)
@pytest.mark.parametrize("page", [8, 16])
def test_update(ops, lengths, source, add, page):
    """Against the steps one by one: tables, lengths, counts, and the pools with their copies."""
    c = R.Cache(lengths, page, 2, 16, "f16", layers=3, spare=12, max_pages=10)
    t, h = device_cache(ops, c)
    table, length, ref, copies, status = R.update(c.table.numpy(), np.array(lengths, np.int32), c.ref.numpy(), source, add, page)
    new, got = run_update(ops, t, h, source, add)
    assert got == status == 0
    assert np.array_equal(new["table"].cpu().numpy(), table)
    assert np.array_equal(new["length"].cpu().numpy(), length) and np.array_equal(new["ref"].cpu().numpy(), ref)
    for pool, now in ((c.k, t["k"]), (c.v, t["v"])):
        want = pool.clone()
        for a, b in copies:
            want[:, b] = pool[:, a]
        assert torch.equal(now.cpu().view(torch.int16), want.view(torch.int16))


def test_update_many_steps(ops):
    """A hundred random steps, the result of each the next one's cache; more slots than a workgroup has threads."""
    import random
    rng = random.Random(4)
    n, page = 1100, 8
    c = R.Cache([rng.randint(0, 30) for _ in range(n)], page, 1, 8, "f32", layers=1, spare=5000, max_pages=9)
    table, length, ref = c.table.numpy(), np.array(c.lengths, np.int32), c.ref.numpy()
    t, h = device_cache(ops, c)
    pool = c.k.clone()
    for _ in range(100):
        source = [rng.choice([d, d, d, d, rng.randrange(n), -1]) for d in range(n)]
        add = []
        for s in source:
            base = 0 if s < 0 else int(length[s])
            add.append(rng.randint(-min(base, 9), min(72 - base, 9)))
        table, length, ref, copies, status = R.update(table, length, ref, source, add, page)
        new, got = run_update(ops, t, h, source, add)
        assert got == status
        assert np.array_equal(new["table"].cpu().numpy(), table)
        assert np.array_equal(new["length"].cpu().numpy(), length) and np.array_equal(new["ref"].cpu().numpy(), ref)
        for a, b in copies:
            pool[:, b] = pool[:, a]
        for name in ("table", "length", "ref"):
            t[name].copy_(new[name])
    assert torch.equal(t["k"].cpu().view(torch.int32), pool.view(torch.int32))


@pytest.mark.parametrize("source,add,spare,status", [
    ([0, 3, 1], None, 9, 1), ([-2, 0, 1], None, 9, 1), (None, [-21, 0, 0], 9, 2), (None, [100, 0, 0], 9, 2),
    ([0, 0, 3], [0, 0, -1], 9, 3), (None, [40, 40, 0], 3, 4), ([0, 0, 0], [90, 90, 90], 9, 2)])
def test_update_refusals(ops, source, add, spare, status):
    c = R.Cache([20, 33, 7], 8, 2, 16, "f16", spare=spare, max_pages=12)
    t, h = device_cache(ops, c)
    before = {k: v.clone() for k, v in t.items()}
    new, got = run_update(ops, t, h, source, add)
    assert got == status == R.update(c.table.numpy(), np.array([20, 33, 7], np.int32), c.ref.numpy(), source, add, 8)[4]
    assert all(torch.equal(new[k], before[k]) for k in new)
    for p in ("k", "v"):
        assert torch.equal(t[p].view(torch.int16), before[p].view(torch.int16))


def test_update_bad_table(ops):
    c = R.Cache([20, 33, 7], 8, 2, 16, "f16", max_pages=12)
    for entry, bad in ((1, c.n_pages), (4, -1)):
        t, h = device_cache(ops, c)
        t["table"][1, entry] = bad
        new, got = run_update(ops, t, h, None, [1, 1, 1])
        assert got == 8 and torch.equal(new["table"], t["table"])
        new, got = run_update(ops, t, h, [0, -1, 2], [1, 0, 1])  # nobody keeps it
        assert got == 0


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("gone", [[], [0], [1, 3], [0, 1, 2, 3, 4]])
def test_compact(ops, dtype, gone):
    c = R.Cache([90, 20, 0, 55, 33], 8, 2, 24, dtype, layers=2, spare=7)
    for s in gone:
        for i in c.table[s]:
            if i >= 0:
                c.ref[i] = 0
        c.table[s] = -1
        c.lengths[s] = 0
    t, h = device_cache(ops, c)
    table, ref, live, moves = R.compact(c.table.numpy(), c.ref.numpy())
    new_table, new_ref, n_live, ws = torch.full_like(t["table"], 77), torch.full_like(t["ref"], 77), ints([99]), space(ops.kv_workspace(h))
    ops.kv_compact(h, Buf(new_table), Buf(new_ref), Buf(n_live), Buf(ws))
    assert int(n_live.cpu()[0]) == live
    assert np.array_equal(new_table.cpu().numpy(), table) and np.array_equal(new_ref.cpu().numpy(), ref)
    for pool, now in ((c.k, t["k"]), (c.v, t["v"])):
        want = pool.clone()
        for a, b in moves:
            want[:, b] = pool[:, a]
        as_int = torch.int32 if dtype == "f32" else torch.int16
        assert torch.equal(now.cpu().view(as_int), want.view(as_int))


@pytest.mark.parametrize("dtype,source", [("f32", "f32"), ("f16", "f32"), ("bf16", "f32"), ("f16", "f16"), ("bf16", "bf16")])
@pytest.mark.parametrize("G,hd", [(2, 64), (1, 8), (3, 136)])
def test_append(ops, dtype, source, G, hd):
    """Rows to the last positions, the rest of the pools untouched; rounding to nearest even, NaN and
    infinities kept; sequences with more rows than positions, and rows behind the last."""
    lengths, rows = [40, 0, 17, 3, 64], [7, 0, 17, 5, 1]
    c = R.Cache(lengths, 16, G, hd, dtype, layers=2)
    t, h = device_cache(ops, c)
    width, T = G * hd, sum(rows) + 4
    x = normal((T, 2 * width + 8), source, seed=1)
    x[3, 0], x[4, 1], x[5, 2], x[6, 3] = math.nan, math.inf, -math.inf, 1 + 2.0 ** -9
    if dtype == "f16" and source == "f32":
        x[0, :4] = torch.tensor([65519.0, 65520.0, 2.0 ** -25, 3 * 2.0 ** -25])
    d = x.cuda()
    ops.kv_append(h, 1, Buf(d), d.shape[1], Buf(d, width), d.shape[1], Buf(offsets(rows)), T, source=source)
    k, v, at = c.k.clone(), c.v.clone(), 0
    for s, n in enumerate(rows):
        skip = max(n - lengths[s], 0)
        a, b = c.at(s, lengths[s])
        for pool, col in ((k, 0), (v, width)):
            pool[1, a[lengths[s] - n + skip:], b[lengths[s] - n + skip:]] = x[at + skip:at + n, col:col + width].reshape(-1, G, hd).to(R.TYPES[dtype])
        at += n
    for got, want in ((t["k"], k), (t["v"], v)):
        got = got.cpu()
        assert bool(((got == want) | (torch.isnan(got) & torch.isnan(want))).all())


# ------------------------------------------------------------- used together --
def test_serving_steps(ops):
    """As a server uses them: prompts packed and cached, one forked, tokens decoded over the shared
    prefix and through the pages, a finished one freed, the pool compacted, decoding on."""
    H, G, hd, page, layers, dtype = 6, 2, 64, 16, 2, "f16"
    n_seq, n_pages, max_pages, scale = 5, 64, 16, 0.125
    pools = [torch.full((layers, n_pages, page, G, hd), math.nan, dtype=torch.float16, device="cuda") for _ in range(2)]
    t = dict(table=torch.full((n_seq, max_pages), -1, dtype=torch.int32, device="cuda"), length=ints([0] * n_seq), ref=ints([0] * n_pages))
    h = ops.kv_pages(Buf(pools[0]), Buf(pools[1]), Buf(t["table"]), Buf(t["length"]), Buf(t["ref"]), n_layer=layers, n_pages=n_pages,
                     page=page, n_seq=n_seq, max_pages=max_pages, n_head_kv=G, head_dim=hd, dtype=dtype)
    history = [[torch.zeros(0, G, hd, dtype=torch.float16)] * 2 for _ in range(n_seq)]  # K and V of each slot

    def step(source=None, add=None):
        new, status = run_update(ops, t, h, source, add)
        assert status == 0
        for name in t:
            t[name].copy_(new[name])
        if source is not None:
            old = [list(x) for x in history]
            for d, s in enumerate(source):
                history[d] = list(old[s]) if s >= 0 else [torch.zeros(0, G, hd, dtype=torch.float16)] * 2

    def append(rows, seed):
        x = normal((sum(rows), (H + 2 * G) * hd), dtype, seed)
        d, at = x.cuda(), 0
        for layer in range(layers):
            ops.kv_append(h, layer, Buf(d, H * hd), d.shape[1], Buf(d, (H + G) * hd), d.shape[1], Buf(offsets(rows)), sum(rows), source=dtype)
        for s, n in enumerate(rows):
            for i in range(2):
                a = (H + i * G) * hd
                history[s][i] = torch.cat([history[s][i], x[at:at + n, a:a + G * hd].reshape(n, G, hd)])
            at += n
        return d

    def check(out, q, rows):
        at = 0
        for s, n in enumerate(rows):
            k, v = history[s]
            ref, mass, top = R.attend(q[at:at + n].cpu().reshape(n, H, hd), k, v, len(k) - n, scale)
            close(out[at:at + n].cpu().reshape(n, H, hd), ref, R.bound(dtype, ref, mass, top, hd, max(len(k), 1)), s)
            at += n

    rows = [75, 20, 0, 0, 0]
    step(add=rows)
    x = append(rows, 1)
    q = x[:, :H * hd].contiguous()
    packed = run_packed(ops, x, rows, H, G, hd, scale)
    check(packed, q, rows)
    check(run_paged(ops, h, q, rows, H, scale, layer=1), q, rows)
    step(source=[0, 1, 0, 0, -1], add=[1, 1, 1, 1, 0])  # slot 0 forked twice
    rows = [1, 1, 1, 1, 0]
    x = append(rows, 2)
    q = x[:, :H * hd].contiguous()
    check(run_paged(ops, h, q, rows, H, scale), q, rows)
    step(source=[0, -1, 2, 3, -1], add=[4, 0, 4, 4, 0])  # slot 1 done; drafts of four
    rows = [4, 0, 4, 4, 0]
    x = append(rows, 3)
    q = x[:, :H * hd].contiguous()
    check(run_paged(ops, h, q, rows, H, scale), q, rows)
    step(add=[-3, 0, -1, 0, 0])  # some of them refused
    for s, n in ((0, 3), (2, 1)):
        history[s] = [r[:-n] for r in history[s]]
    new_table, new_ref, live, ws = torch.empty_like(t["table"]), torch.empty_like(t["ref"]), ints([0]), space(ops.kv_workspace(h))
    ops.kv_compact(h, Buf(new_table), Buf(new_ref), Buf(live), Buf(ws))
    t["table"].copy_(new_table)
    t["ref"].copy_(new_ref)
    assert int(live.cpu()[0]) == int((new_ref > 0).sum()) and int(new_table.max()) < int(live.cpu()[0])
    step(add=[1, 0, 1, 1, 0])
    rows = [1, 0, 1, 1, 0]
    x = append(rows, 4)
    q = torch.zeros(n_seq, H * hd, dtype=torch.float16, device="cuda")
    q[[0, 2, 3]] = x[:, :H * hd]
    check(run_prefix(ops, h, q, 75, H, scale, t["table"][0].clone()), q, [1] * n_seq)
    check(run_paged(ops, h, x[:, :H * hd].contiguous(), rows, H, scale), x[:, :H * hd], rows)


def test_graph_and_streams(ops):
    """A decode step captured once on another stream and replayed, the eager calls between the replays."""
    H, G, hd, page = 14, 2, 64, 16
    c = R.Cache([500, 30, 1, 77], page, G, hd, "f16", spare=40, max_pages=40)
    t, h = device_cache(ops, c)
    q, x = normal((4, H * hd), "f16", 1).cuda(), normal((4, 2 * G * hd), "f32", 2).cuda()
    off, add = offsets([1] * 4), ints([1] * 4)
    new = {k: torch.empty_like(t[k]) for k in ("table", "length", "ref")}
    status, ws = ints([9]), space(ops.kv_workspace(h))
    wa = space(ops.attention_paged_workspace(h, 4, H))
    wp = space(ops.attention_prefix_workspace(h, 1, H))
    out, shared = torch.empty_like(q), torch.empty_like(q)

    def step():
        s = torch.cuda.current_stream().cuda_stream
        ops.kv_update(h, Buf(new["table"]), Buf(new["length"]), Buf(new["ref"]), Buf(status), Buf(ws), add=Buf(add), stream=s)
        for k in new:
            t[k].copy_(new[k])
        ops.kv_append(h, 0, Buf(x), 2 * G * hd, Buf(x, G * hd), 2 * G * hd, Buf(off), 4, stream=s)
        ops.attention_paged(Buf(q), H * hd, h, 0, Buf(off), 4, H, 0.125, Buf(out), H * hd, Buf(wa), stream=s)
        ops.attention_prefix(Buf(q), H * hd, h, 0, Buf(t["table"]), 1, H, 0.125, Buf(shared), H * hd, Buf(wp), stream=s)

    start = {k: v.clone() for k, v in t.items()}
    want = []
    for i in range(5):
        x.copy_(normal((4, 2 * G * hd), "f32", 10 + i))
        step()
        want.append((out.clone(), shared.clone(), t["table"].clone(), t["length"].clone()))
    for k in start:
        t[k].copy_(start[k])
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=side):
        step()
    for i in range(5):
        x.copy_(normal((4, 2 * G * hd), "f32", 10 + i))
        graph.replay()
        torch.cuda.synchronize()
        assert int(status.cpu()[0]) == 0
        for a, b in zip(want[i], (out, shared, t["table"], t["length"])):
            assert torch.equal(a, b), i
        run_paged(ops, h, q, [1] * 4, H, 0.125)
    check_end = run_paged(ops, h, q, [1] * 4, H, 0.125)
    assert torch.equal(check_end, out)


def test_same_bits_again(ops):
    """The same call gives the same bits, whatever else the workspace held."""
    H, G, hd = 12, 2, 128
    rows = [900, 3, 77]
    x = normal((sum(rows), (H + 2 * G) * hd), "bf16", 3).cuda()
    a, b = (run_packed(ops, x, rows, H, G, hd, 0.1) for _ in range(2))
    assert torch.equal(a, b)
    c = R.Cache([3000, 5, 800], 16, G, hd, "f32", max_pages=400)
    _, h = device_cache(ops, c)
    q = normal((3, H * hd), "f32", 4).cuda()
    assert torch.equal(run_paged(ops, h, q, [1] * 3, H, 0.1), run_paged(ops, h, q, [1] * 3, H, 0.1))


def guarded(nbytes):
    """A workspace of exactly nbytes (a multiple of 4), and the words behind it."""
    t = torch.full((nbytes // 4 + 64,), 7.0, device="cuda")

    class W:
        ptr, buf = t.data_ptr(), t
    W.nbytes = nbytes
    return W, t[nbytes // 4:]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("H,G,hd,rows,seqs,length", [(14, 2, 64, 1, 5, 3000), (6, 2, 128, 9, 2, 2500), (3, 3, 24, 1, 70, 300)])
def test_workspaces_are_kept_to(ops, dtype, H, G, hd, rows, seqs, length):
    """Calls write no further than their _workspace() bytes."""
    c = R.Cache([length - 7 * i for i in range(seqs)] if length > 7 * seqs else [length] * seqs, 16, G, hd, dtype, spare=80, max_pages=256)
    t, h = device_cache(ops, c)
    q = normal((rows * seqs, H * hd), dtype, 3).cuda()
    out, off = torch.empty_like(q), offsets([rows] * seqs)
    ws, tail = guarded(ops.attention_paged_workspace(h, rows * seqs, H) // 4 * 4)
    ops.attention_paged(Buf(q), H * hd, h, 0, Buf(off), rows * seqs, H, 0.1, Buf(out), H * hd, ws)
    assert bool((tail == 7).all())
    check_paged(c, q, out, [rows] * seqs, H, 0.1)
    ws, tail = guarded(ops.attention_prefix_workspace(h, 100, H) // 4 * 4)
    ops.attention_prefix(Buf(q), H * hd, h, 0, Buf(t["table"]), 100, H, 0.1, Buf(out), H * hd, ws)
    assert bool((tail == 7).all())
    x = normal((rows * seqs, (H + 2 * G) * hd), dtype, 4).cuda()
    ws, tail = guarded(ops.attention_packed_workspace(rows * seqs, seqs, H, G, hd) // 4 * 4)
    ops.attention_packed(Buf(x), x.shape[1], Buf(x, H * hd), x.shape[1], Buf(x, (H + G) * hd), x.shape[1], Buf(off), seqs, rows * seqs, H,
                         G, hd, 0.1, Buf(out), H * hd, ws, dtype=dtype)
    assert bool((tail == 7).all())
    check_packed(x, out, [rows] * seqs, H, G, hd, 0.1, dtype)
    ws, tail = guarded(ops.kv_workspace(h) // 4 * 4)
    new, status = {k: torch.empty_like(t[k]) for k in ("table", "length", "ref")}, ints([9])
    ops.kv_update(h, Buf(new["table"]), Buf(new["length"]), Buf(new["ref"]), Buf(status), ws, add=Buf(ints([1] * seqs)))
    assert int(status.cpu()[0]) == 0 and bool((tail == 7).all())
    ops.kv_compact(h, Buf(new["table"]), Buf(new["ref"]), Buf(status), ws)
    torch.cuda.synchronize()
    assert bool((tail == 7).all())


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_many_sequences(ops, dtype):
    """Thousands of short ones, and a few thousand rows over a few of many slots."""
    rows = [(i * 7) % 4 for i in range(3000)]
    H, G, hd = 4, 2, 32
    x = normal((sum(rows), (H + 2 * G) * hd), dtype, 5).cuda()
    check_packed(x, run_packed(ops, x, rows, H, G, hd, 0.2), rows, H, G, hd, 0.2, dtype)
    rows = [0] * 200 + [90] + [0] * 150 + [300] + [0] * 100
    x = normal((sum(rows), (H + 2 * G) * hd), dtype, 6).cuda()
    check_packed(x, run_packed(ops, x, rows, H, G, hd, 0.2), rows, H, G, hd, 0.2, dtype)


def test_two_calls_at_once(ops):
    """Calls on two streams, each with a workspace of its own."""
    H, G, hd = 6, 2, 64
    c = R.Cache([2000, 900, 3], 16, G, hd, "f16", max_pages=256)
    _, h = device_cache(ops, c)
    q = [normal((3, H * hd), "f16", s).cuda() for s in (1, 2)]
    want = [run_paged(ops, h, x, [1] * 3, H, 0.1) for x in q]
    streams, out, off = [torch.cuda.Stream() for _ in q], [torch.empty_like(x) for x in q], offsets([1] * 3)
    ws = [space(ops.attention_paged_workspace(h, 3, H)) for _ in q]
    torch.cuda.synchronize()
    for _ in range(20):
        for x, o, w, s in zip(q, out, ws, streams):
            ops.attention_paged(Buf(x), H * hd, h, 0, Buf(off), 3, H, 0.1, Buf(o), H * hd, Buf(w), stream=s.cuda_stream)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, out))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("scale", [1e-38, 1e-6, 20.0])
def test_scales(ops, dtype, scale):
    """Scales that make all weights alike, and that leave one."""
    rows, H, G, hd = [70, 300], 4, 2, 64
    x = normal((sum(rows), (H + 2 * G) * hd), dtype, seed=5).cuda()
    check_packed(x, run_packed(ops, x, rows, H, G, hd, scale), rows, H, G, hd, scale, dtype)
    c = R.Cache([900, 40], 16, G, hd, dtype)
    _, h = device_cache(ops, c)
    q = normal((2, H * hd), dtype, 3).cuda()
    check_paged(c, q, run_paged(ops, h, q, [1, 1], H, scale), [1, 1], H, scale)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_scores_of_minus_infinity(ops, dtype):
    """Keys whose score is -inf have no weight; a row that sees only such keys is no number, as a
    softmax of them is; values past f32's parts are what they are."""
    H, G, hd, n = 2, 1, 64, 200
    x = normal((n, (H + 2 * G) * hd), dtype, 7).abs()
    x[:, :H * hd] += 0.5                       # positive queries
    x[:40, H * hd:(H + 1) * hd] = -math.inf    # and keys of -inf: every score with them is -inf
    out = run_packed(ops, x.cuda(), [n], H, G, hd, 0.1).cpu().reshape(n, H, hd)
    assert bool(torch.isnan(out[:40].float()).all())
    q, k, v = (x[:, a * hd:b * hd].reshape(n, b - a, hd) for a, b in ((0, H), (H, H + G), (H + G, H + 2 * G)))
    ref, mass, top = R.attend(q[40:], k[40:], v[40:], 0, 0.1)
    close(out[40:], ref, R.bound(dtype, ref, mass, top, hd, n))


def all_or_none(out, want):
    """Rows of which a True in want says that they are no numbers throughout, and the others' rows."""
    nan = torch.isnan(out.float().cpu()).reshape(out.shape[0], -1, want.shape[-1])
    assert bool((nan.all(2) == want.all(2)).all()) and bool((nan.any(2) == want.any(2)).all()), (nan.sum(2), want.sum(2))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("form", ["packed", "tokens", "prefix-few", "prefix-tiles"])
def test_keys_without_a_number_fill_a_part(ops, dtype, form):
    """Keys cut into parts, of which one holds no score that is a number: rows that see it are NaN."""
    H, G, hd, n = 6, 2, 64, 1100
    for first in (512, 1024):
        if form == "packed":
            x = normal((n, (H + 2 * G) * hd), dtype, seed=n)
            x[first:, H * hd:(H + 1) * hd] = math.nan
            out = run_packed(ops, x.cuda(), [n], H, G, hd, 0.1)
            want = torch.zeros(n, H, hd, dtype=torch.bool)
            want[first:, :3] = True
            all_or_none(out, want)
            continue
        seqs = 24 if form == "prefix-tiles" else 3
        lengths = [n + 20 - 9 * s for s in range(seqs - 1)] + [first]
        c = R.Cache(lengths, 16, G, hd, dtype, seed=2)
        for s, m in enumerate(lengths):
            for pool in (c.k, c.v):
                x = c.rows(pool, 0, s, m).clone()
                shared = min(m, n)
                x[:shared] = c.rows(pool, 0, 0, shared)
                if pool is c.k:
                    x[first:n, 0] = math.nan
                c.write(pool, 0, s, x)
        _, h = device_cache(ops, c)
        q = normal((seqs, H * hd), dtype, seed=3).cuda()
        prefix = n if form.startswith("prefix") else 0
        out = run_prefix(ops, h, q, prefix, H, 0.12, c.table[0].clone().cuda()) if prefix else run_paged(ops, h, q, [1] * seqs, H, 0.12)
        want = torch.zeros(seqs, H, hd, dtype=torch.bool)
        want[[s for s, m in enumerate(lengths) if m > first], :3] = True
        all_or_none(out, want)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("form", ["packed", "rows", "drafts", "prefix-few", "prefix-tiles"])
def test_parts_a_row_does_not_see(ops, dtype, form):
    """Values that are no numbers in a part of the keys of which a row sees none."""
    H, G, hd, n = 6, 2, 64, 1100
    for first in (512, 1024):
        if form == "packed":
            x = normal((n, (H + 2 * G) * hd), dtype, seed=n)
            x[first:, (H + G) * hd:(H + G + 1) * hd] = math.nan
            out = run_packed(ops, x.cuda(), [n], H, G, hd, 0.1)
            want = torch.zeros(n, H, hd, dtype=torch.bool)
            want[first:, :3] = True
            all_or_none(out, want)
            continue
        seqs = 24 if form == "prefix-tiles" else 3
        rows = {"rows": [60] * seqs, "drafts": [5] * seqs}.get(form, [1] * seqs)
        lengths = [n - 9 * s for s in range(seqs - 1)] + [first] if form.startswith("prefix") else [first + 4, first + 1, first + 30]
        c = R.Cache(lengths, 16, G, hd, dtype, seed=2)
        for s, m in enumerate(lengths):
            for pool in (c.k, c.v):
                x = c.rows(pool, 0, s, m).clone()
                if form.startswith("prefix"):
                    x[:] = c.rows(pool, 0, 0, m)
                if pool is c.v:
                    x[first:, 0] = math.nan
                c.write(pool, 0, s, x)
        _, h = device_cache(ops, c)
        q = normal((sum(rows), H * hd), dtype, seed=3).cuda()
        out = run_prefix(ops, h, q, n, H, 0.12, c.table[0].clone().cuda()) if form.startswith("prefix") else run_paged(ops, h, q, rows, H, 0.12)
        want = torch.zeros(sum(rows), H, hd, dtype=torch.bool)
        at = 0
        for s, r in enumerate(rows):
            for i in range(r):
                want[at + i, :3] = lengths[s] - r + i >= first
            at += r
        all_or_none(out, want)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows", [4, 9, 80])
def test_rows_without_a_position(ops, dtype, rows):
    """Rows in front of a sequence's first position are zeros, whatever its keys and values hold."""
    H, G, hd, length = 6, 2, 64, rows - 2
    c = R.Cache([length], 16, G, hd, dtype, seed=6)
    for pool in (c.k, c.v):
        x = c.rows(pool, 0, 0, length).clone()
        x[1, 0] = math.nan
        c.write(pool, 0, 0, x)
    _, h = device_cache(ops, c)
    q = normal((rows, H * hd), dtype, seed=3).cuda()
    out = run_paged(ops, h, q, [rows], H, 0.12).cpu().reshape(rows, H, hd)
    assert bool((out[:2] == 0).all())
    want = torch.zeros(rows, H, hd, dtype=torch.bool)
    want[3:, :3] = True
    all_or_none(out, want)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows", [1, 30])
def test_values_without_a_number_at_weight_zero(ops, dtype, rows):
    """Keys whose score is -inf have weight 0, and 0 times a NaN value is NaN in its dimension."""
    H, G, hd, n = 6, 2, 64, 1100
    c = R.Cache([n], 16, G, hd, dtype, seed=6)
    k, v = c.rows(c.k, 0, 0, n).abs(), c.rows(c.v, 0, 0, n).clone()
    k[:700] = -math.inf
    v[40, 0, 9] = v[600, 1, 11] = math.nan
    c.write(c.k, 0, 0, k)
    c.write(c.v, 0, 0, v)
    _, h = device_cache(ops, c)
    q = (normal((rows, H * hd), dtype, seed=3).abs() + 0.5).cuda()  # positive queries
    out = run_paged(ops, h, q, [rows], H, 0.12)
    nan = torch.zeros(rows, H, hd, dtype=torch.bool)
    nan[:, :3, 9] = nan[:, 3:, 11] = True
    assert torch.equal(torch.isnan(out.cpu().float()).reshape(rows, H, hd), nan)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("seqs", [257, 600, 1100])
def test_tokens_of_many_sequences(ops, dtype, seqs):
    """One token each of some hundred sequences: over their own pages, some idle, and after a prefix."""
    H, G, hd, prefix = 6, 2, 32, 20
    lengths = [prefix + (s * 13) % 50 for s in range(seqs)]
    c = R.Cache(lengths, 16, G, hd, dtype, seed=seqs)
    for s in range(1, seqs):
        for pool in (c.k, c.v):
            c.write(pool, 0, s, c.rows(pool, 0, 0, prefix).clone())
    _, h = device_cache(ops, c)
    q = normal((seqs, H * hd), dtype, seed=3).cuda()
    out = run_prefix(ops, h, q, prefix, H, 0.2, c.table[0].clone().cuda())
    check_paged(c, q, out, [1] * seqs, H, 0.2)
    rows = [int(s % 3 != 0) for s in range(seqs)]
    check_paged(c, q[:sum(rows)], run_paged(ops, h, q[:sum(rows)], rows, H, 0.2), rows, H, 0.2)
