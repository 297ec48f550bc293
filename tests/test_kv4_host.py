"""The 4-bit cache's C ABI without a GPU: exported symbols and argument checks."""
import os
import re

from gcnasm_b200 import capi

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "b2g", "kv4.h")


def test_exports_every_declared_symbol():
    decl = set(re.findall(r"\b(b2g_kv4_\w+)\s*\(", re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)))
    assert decl == set(capi.KV4_EXPORTS)
    for s in decl:
        assert hasattr(capi.lib(), s), s


def cache(**k):
    a = dict(k=1 << 20, v=2 << 20, k_scale=3 << 20, v_scale=4 << 20, pages=8, kv_heads=2, page_size=16, head_dim=64) | k
    return capi.Kv4Cache(*a.values())


def batch(**k):
    a = dict(table=5 << 20, lens=6 << 20, cu=7 << 20, seqs=2, table_width=2, rows=4, max_new=2) | k
    return capi.Kv4Batch(*a.values())


def read(c, b, start=8 << 20, k=9 << 20, v=10 << 20):
    return capi.lib().b2g_kv4_read(c, b, start, k, v, None)


def test_arguments_are_refused_without_a_gpu():
    """Each is found before the device is asked for, so the addresses are never used."""
    for got, want in [
        (read(None, batch()), capi.B2G_ERR_INVALID_ARG),
        (read(cache(), None), capi.B2G_ERR_INVALID_ARG),
        (read(cache(), batch(), start=None), capi.B2G_ERR_INVALID_ARG),
        (read(cache(), batch(), k=8), capi.B2G_ERR_ALIGNMENT),
        (read(cache(k=None), batch()), capi.B2G_ERR_INVALID_ARG),
        (read(cache(v_scale=8), batch()), capi.B2G_ERR_ALIGNMENT),
        (read(cache(head_dim=96), batch()), capi.B2G_ERR_UNSUPPORTED),
        (read(cache(page_size=24), batch()), capi.B2G_ERR_UNSUPPORTED),
        (read(cache(page_size=8), batch()), capi.B2G_ERR_UNSUPPORTED),
        (read(cache(page_size=2048), batch()), capi.B2G_ERR_UNSUPPORTED),
        (read(cache(kv_heads=0), batch()), capi.B2G_ERR_UNSUPPORTED),
        (read(cache(pages=0), batch()), capi.B2G_ERR_INVALID_ARG),
        (read(cache(), batch(table=None)), capi.B2G_ERR_INVALID_ARG),
        (read(cache(), batch(seqs=0)), capi.B2G_ERR_UNSUPPORTED),
        (read(cache(), batch(seqs=8193)), capi.B2G_ERR_UNSUPPORTED),
        (read(cache(), batch(table_width=0)), capi.B2G_ERR_UNSUPPORTED),
        (read(cache(page_size=1024), batch(table_width=1 << 21)), capi.B2G_ERR_UNSUPPORTED),
        (read(cache(), batch(rows=-1)), capi.B2G_ERR_INVALID_ARG),
        (read(cache(), batch(cu=None)), capi.B2G_ERR_INVALID_ARG),
    ]:
        assert got == want, capi.lib().b2g_last_error()
    L = capi.lib()
    one = 1 << 20
    assert L.b2g_kv4_append(cache(), batch(), one, one, 5, 128, 64, 128, 64, None, None) == capi.B2G_ERR_INVALID_ARG
    assert L.b2g_kv4_append(cache(), batch(), one, None, 0, 128, 64, 128, 64, None, None) == capi.B2G_ERR_INVALID_ARG
    assert L.b2g_kv4_append(cache(), batch(), one, one, 0, 128, 60, 128, 64, None, None) == capi.B2G_ERR_ALIGNMENT
    assert L.b2g_kv4_append(cache(), batch(), one, one, 1, 128, 64, 126, 64, None, None) == capi.B2G_ERR_ALIGNMENT
    assert L.b2g_kv4_append(cache(), batch(lens=None), one, one, 0, 128, 64, 128, 64, None, None) == capi.B2G_ERR_INVALID_ARG
    assert L.b2g_kv4_workspace_bytes(96) < 0
