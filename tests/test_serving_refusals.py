"""What the serving operators refuse: argument checks that end before any launch, so
they run without a GPU, on addresses that are never read."""
import ctypes

import pytest

A = 1 << 20  # an address for arguments that are not the one under test


class Mem:
    def __init__(self, ptr=A, nbytes=1 << 60):
        self.ptr, self.nbytes = ptr, nbytes


@pytest.fixture
def ops():
    from gaje_hip import ops
    return ops


def cache(ops, **change):
    a = dict(k=Mem(), v=Mem(), table=Mem(16 * A), length=Mem(32 * A), ref=Mem(48 * A), n_layer=2, n_pages=10, page=16, n_seq=3,
             max_pages=4, n_head_kv=2, head_dim=64, dtype="f16")
    a.update(change)
    return ops.kv_pages(a.pop("k"), a.pop("v"), a.pop("table"), a.pop("length"), a.pop("ref"), **a)


def refused(text, call, *args, **kw):
    from gaje_hip import GajeError
    with pytest.raises(GajeError) as e:
        call(*args, **kw)
    assert text in str(e.value), str(e.value)


BAD_CACHES = [(dict(page=12), "page of 12"), (dict(page=4), "page of 4"), (dict(page=2048), "page of 2048"),
              (dict(head_dim=60), "head_dim 60"), (dict(head_dim=264), "head_dim 264"), (dict(head_dim=0), "head_dim 0"),
              (dict(n_head_kv=0), "heads"), (dict(k=Mem(A + 8)), "16-byte aligned"), (dict(table=Mem(0)), "lacks an array"),
              (dict(n_pages=(1 << 26) + 1), "pages"), (dict(n_seq=0), "sequences"), (dict(n_seq=65537), "sequences"), (dict(max_pages=0), "pages"),
              (dict(n_layer=0), "layers"), (dict(max_pages=1 << 27), "pages")]


@pytest.mark.parametrize("change,text", BAD_CACHES)
def test_caches(ops, change, text):
    c = cache(ops, **change)
    m = Mem()
    refused(text, ops.kv_update, c, Mem(64 * A), Mem(65 * A), Mem(66 * A), m, m)
    refused(text, ops.kv_compact, c, Mem(64 * A), Mem(66 * A), m, m)
    refused(text, ops.kv_append, c, 0, m, 128, m, 128, m, 5)
    refused(text, ops.attention_paged, m, 256, c, 0, m, 3, 4, 0.1, m, 256, m)
    refused(text, ops.attention_prefix, m, 256, c, 0, m, 16, 4, 0.1, m, 256, m)
    for size in (ops.kv_workspace(c), ops.attention_paged_workspace(c, 3, 4), ops.attention_prefix_workspace(c, 16, 4)):
        assert size == -1


def test_small_buffers(ops):
    with pytest.raises(ValueError):
        cache(ops, v=Mem(nbytes=2 * 10 * 16 * 2 * 64 * 2 - 1))
    with pytest.raises(ValueError):
        cache(ops, table=Mem(nbytes=4 * 3 * 4 - 1))


def test_pages(ops):
    c, m = cache(ops), Mem()
    own = [Mem(16 * A), Mem(32 * A + 8), Mem(48 * A - 4)]  # the cache's arrays, or partly so
    good = [Mem(64 * A), Mem(65 * A), Mem(66 * A)]
    for i in range(3):
        for bad in own:
            new = list(good)
            new[i] = bad
            refused("not the cache's own", ops.kv_update, c, *new, m, m)
    refused("null", ops.kv_update, c, Mem(0), good[1], good[2], m, m)
    refused("null", ops.kv_update, c, *good, Mem(0), m)
    refused("workspace", ops.kv_update, c, *good, m, Mem(A, ops.kv_workspace(c) - 1))
    refused("workspace", ops.kv_update, c, *good, m, Mem(A + 4))
    refused("not the cache's own", ops.kv_compact, c, own[0], good[2], m, m)
    refused("not the cache's own", ops.kv_compact, c, good[0], own[2], m, m)
    refused("workspace", ops.kv_compact, c, good[0], good[2], m, Mem(0))
    for layer in (-1, 2):
        refused("layer", ops.kv_append, c, layer, m, 128, m, 128, m, 5)
    refused("multiple of 8", ops.kv_append, c, 0, m, 132, m, 128, m, 5)
    refused("multiple of 8", ops.kv_append, c, 0, m, 128, m, 120, m, 5)
    refused("16-byte aligned", ops.kv_append, c, 0, Mem(A + 4), 128, m, 128, m, 5)
    refused("dtype", ops.kv_append, c, 0, m, 128, m, 128, m, 5, source="bf16")
    refused("null seq_off", ops.kv_append, c, 0, m, 128, m, 128, Mem(0), 5)
    refused("rows", ops.kv_append, c, 0, m, 128, m, 128, m, -1)
    ops.kv_append(c, 0, m, 128, m, 128, m, 0)  # nothing to do


def packed(ops, **change):
    a = dict(q=Mem(), ldq=256, k=Mem(), ldk=128, v=Mem(), ldv=128, seq_off=Mem(), n_seq=3, T=9, n_head=4, n_head_kv=2,
             head_dim=64, scale=0.1, out=Mem(), ldo=256, workspace=Mem())
    a.update(change)
    return ops.attention_packed(**a)


@pytest.mark.parametrize("change,text", [
    (dict(n_head=5), "heads"), (dict(n_head=0), "heads"), (dict(head_dim=68), "head_dim"), (dict(head_dim=-8), "head_dim"),
    (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"), (dict(scale=float("nan")), "scale"),
    (dict(scale=float("inf")), "scale"), (dict(q=Mem(A + 2)), "16-byte"), (dict(q=Mem(0)), "null q"),
    (dict(out=Mem(0)), "null out"), (dict(ldq=248), "leading"), (dict(ldk=130), "leading"), (dict(ldv=64), "leading"),
    (dict(ldo=-256), "leading"), (dict(seq_off=Mem(0)), "null seq_off"), (dict(n_seq=-1), "sequences"), (dict(n_seq=65537), "sequences"), (dict(T=1 << 24, n_head=128, ldq=8192, ldo=8192), "heads (2^30"),
    (dict(T=-1), "rows"), (dict(T=(1 << 24) + 1), "rows")])
def test_packed(ops, change, text):
    refused(text, packed, ops, **change)


def test_empty_packed(ops):
    packed(ops, T=0)
    packed(ops, n_seq=0)


def test_cached(ops):
    c, m = cache(ops), Mem()
    for args, text in [((m, 256, c, 2, m, 3, 4, 0.1, m, 256, m), "layer"), ((m, 256, c, 0, m, 3, 3, 0.1, m, 256, m), "heads"),
                       ((m, 256, c, 0, m, 3, 4, 0.0, m, 256, m), "scale"), ((m, 200, c, 0, m, 3, 4, 0.1, m, 256, m), "leading"),
                       ((m, 256, c, 0, Mem(0), 3, 4, 0.1, m, 256, m), "null seq_off"),
                       ((m, 256, c, 0, m, 3, 4, 0.1, Mem(A + 1), 256, m), "16-byte")]:
        refused(text, ops.attention_paged, *args)
    ops.attention_paged(m, 256, c, 0, m, 0, 4, 0.1, m, 256, m)  # no rows
    for n in (-1, 4 * 16 + 1):
        refused("prefix of", ops.attention_prefix, m, 256, c, 0, m, n, 4, 0.1, m, 256, m)
        assert ops.attention_prefix_workspace(c, n, 4) == -1
    refused("prefix of", ops.attention_prefix, m, 256, c, 0, Mem(0), 16, 4, 0.1, m, 256, m)
    refused("layer", ops.attention_prefix, m, 256, c, -1, m, 16, 4, 0.1, m, 256, m)
    refused("scale", ops.attention_prefix, m, 256, c, 0, m, 16, 4, -0.1, m, 256, m)


@pytest.mark.parametrize("T,n_seq,heads,kv,hd", [(1, 1, 14, 2, 64), (4000, 3, 12, 2, 128), (8190, 1, 32, 8, 128), (64, 64, 9, 3, 256)])
def test_workspace_too_small(ops, T, n_seq, heads, kv, hd):
    """Each call refuses less than its _workspace() bytes, where that is any."""
    need = ops.attention_packed_workspace(T, n_seq, heads, kv, hd)
    assert need >= 0
    c = cache(ops, n_pages=40000, n_seq=n_seq, max_pages=300, n_head_kv=kv, head_dim=hd, table=Mem(1 << 40), length=Mem(1 << 41),
              ref=Mem(1 << 42))
    m = Mem()
    for dtype in ("f16",):
        n = ops.attention_paged_workspace(c, T, heads)
        if n > 0:
            refused("workspace", ops.attention_paged, m, heads * hd, c, 0, m, T, heads, 0.1, m, heads * hd, Mem(A, n - 1))
        n = ops.attention_prefix_workspace(c, 3000, heads)
        if n > 0:
            refused("workspace", ops.attention_prefix, m, heads * hd, c, 0, m, 3000, heads, 0.1, m, heads * hd, Mem(A, n - 1))


def test_struct_layout(tmp_path):
    """gaje_hip_kv_pages as a C compiler lays it out."""
    import os
    import subprocess
    from conftest import REPO
    from gaje_hip import _lib
    names = [f for f, _ in _lib.KvPages._fields_]
    src = '#include <stdio.h>\n#include <stddef.h>\n#include "gaje_hip.h"\nint main(void) {\n'
    src += 'printf("%zu", sizeof(gaje_hip_kv_pages));\n'
    src += "".join(f'printf(" %zu", offsetof(gaje_hip_kv_pages, {f}));\n' for f in names) + "return 0; }\n"
    (tmp_path / "l.c").write_text(src)
    subprocess.run(["gcc", "-std=c11", "-I", os.path.join(REPO, "include"), str(tmp_path / "l.c"), "-o", str(tmp_path / "l")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "l")], check=True, capture_output=True, text=True).stdout.split()]
    assert got == [ctypes.sizeof(_lib.KvPages)] + [getattr(_lib.KvPages, f).offset for f in names]


def test_arguments_that_may_be_missing(ops):
    """No workspace where none is needed, no prefix table without a prefix; refused where they are."""
    from gaje_hip import GajeError
    c, m = cache(ops), Mem()
    packed(ops, T=0, workspace=None)
    ops.attention_paged(m, 256, c, 0, m, 0, 4, 0.1, m, 256, None)
    assert ops.attention_packed_workspace(8190, 1, 4, 2, 64) > 0
    refused("workspace", packed, ops, T=8190, n_seq=1, workspace=None, dtype="f16")
    refused("workspace", ops.kv_update, c, Mem(64 * A), Mem(65 * A), Mem(66 * A), m, None)
    refused("workspace", ops.kv_compact, c, Mem(64 * A), Mem(66 * A), m, None)
    refused("prefix of", ops.attention_prefix, m, 256, c, 0, None, 16, 4, 0.1, m, 256, m)
    with pytest.raises(GajeError, match="null q"):
        ops.attention_prefix(Mem(0), 256, c, 0, None, 0, 4, 0.1, m, 256, m)
