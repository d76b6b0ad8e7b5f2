"""CPU tests of the paged-cache entry points: what they refuse, before anything
reaches a device."""
import ctypes as C

import pytest

from tests.vox_testlib import cuda_available, vox


@pytest.fixture(scope="module")
def V():
    return vox()


OUT = 1 << 21  # another made-up address: results must not replace their queries


def descs(V, **kw):
    """A valid cache, batch, prefix and row set on made-up addresses (never read here)."""
    a = 1 << 20
    c = dict(device=0, dtype=8, keys=a, values=a, n_pages=10, page_size=16, n_kv_heads=2, head_dim=64, page_stride=0,
             head_stride=0, slot_stride=0)
    b = dict(n_seqs=2, n_tokens=3, max_q_len=2, max_kv_len=40, table_width=3, table_stride=3, q_start=a, kv_len=a,
             page_table=a, first_pos=None, status=None)
    p = dict(pages=a, len=a, n_pages=4, max_len=64)
    q = dict(ptr=a, token_stride=0, head_stride=0)
    out = []
    for cls, d, key in ((V.PagedCacheDesc, c, "cache"), (V.PagedBatchDesc, b, "batch"), (V.PagedPrefixDesc, p, "prefix"),
                        (V.Rows, q, "rows")):
        d.update(kw.get(key, {}))
        out.append(cls(*[d[n] for n, _ in cls._fields_]))
    return out


CACHE = [
    (dict(dtype=9), "ERR_UNSUPPORTED", "dtype"), (dict(dtype=3), "ERR_UNSUPPORTED", "dtype"),
    (dict(keys=None), "ERR_INVALID_ARG", "null"), (dict(values=None), "ERR_INVALID_ARG", "null"),
    (dict(keys=(1 << 20) + 1), "ERR_INVALID_ARG", "aligned"),
    (dict(n_pages=0), "ERR_INVALID_ARG", "n_pages"), (dict(n_pages=1 << 30), "ERR_INVALID_ARG", "n_pages"),
    (dict(n_kv_heads=0), "ERR_INVALID_ARG", "n_kv_heads"),
    (dict(page_size=0), "ERR_UNSUPPORTED", "page_size"), (dict(page_size=24), "ERR_UNSUPPORTED", "page_size"),
    (dict(page_size=2048), "ERR_UNSUPPORTED", "page_size"),
    (dict(head_dim=0), "ERR_UNSUPPORTED", "head_dim"), (dict(head_dim=63), "ERR_UNSUPPORTED", "head_dim"),
    (dict(head_dim=258), "ERR_UNSUPPORTED", "head_dim"),
    (dict(slot_stride=32, head_stride=1024, page_stride=2048), "ERR_SHAPE", "strides"),
    (dict(slot_stride=64), "ERR_SHAPE", "strides"),
]
BATCH = [
    (dict(q_start=None), "ERR_INVALID_ARG", "null"), (dict(kv_len=None), "ERR_INVALID_ARG", "null"),
    (dict(page_table=None), "ERR_INVALID_ARG", "null"),
    (dict(max_q_len=0), "ERR_SHAPE", "max_q_len"), (dict(max_q_len=4), "ERR_SHAPE", "max_q_len"),
    (dict(max_kv_len=49), "ERR_SHAPE", "max_kv_len"), (dict(table_stride=2), "ERR_SHAPE", "table_stride"),
    (dict(n_tokens=1 << 31), "ERR_UNSUPPORTED", "batch sizes"), (dict(n_seqs=1 << 40), "ERR_UNSUPPORTED", "batch sizes"),
    (dict(max_kv_len=1 << 31), "ERR_UNSUPPORTED", "batch sizes"),
]


def refused(V, rc, code, word):
    assert rc == getattr(V, code), (rc, V.last_error())
    assert word in V.last_error()


@pytest.mark.parametrize("key,change,code,word", [("cache", *x) for x in CACHE] + [("batch", *x) for x in BATCH])
def test_descriptions_are_checked_by_every_call(V, key, change, code, word):
    c, b, p, r = (C.byref(x) for x in descs(V, **{key: change}))
    L, n = V.lib(), C.c_size_t()
    refused(V, L.vox_paged_append_rope(c, b, r, r, 1e4, 4, r, r, None), code, word)
    refused(V, L.vox_paged_attention(c, b, r, 4, 0, 0, 0.0, r, None, 0, None), code, word)
    refused(V, L.vox_paged_prefix_attention(c, b, p, r, 4, 0, 0, 0.0, r, None, 0, None), code, word)
    refused(V, L.vox_paged_attention_workspace(c, b, 4, 0, 0, C.byref(n)), code, word)
    refused(V, L.vox_paged_prefix_attention_workspace(c, b, p, 4, 0, 0, C.byref(n)), code, word)


def test_null_arguments(V):
    c, b, p, r = (C.byref(x) for x in descs(V))
    L, n = V.lib(), C.c_size_t()
    for rc in (L.vox_paged_append_rope(None, b, r, r, 1e4, 4, r, r, None),
               L.vox_paged_append_rope(c, None, r, r, 1e4, 4, r, r, None),
               L.vox_paged_append_rope(c, b, None, r, 1e4, 4, r, r, None),
               L.vox_paged_append_rope(c, b, r, None, 1e4, 4, r, r, None),
               L.vox_paged_append_rope(c, b, r, r, 1e4, 4, r, None, None),
               L.vox_paged_attention(c, b, None, 4, 0, 0, 0.0, r, None, 0, None),
               L.vox_paged_attention(c, b, r, 4, 0, 0, 0.0, None, None, 0, None),
               L.vox_paged_prefix_attention(c, b, None, r, 4, 0, 0, 0.0, r, None, 0, None),
               L.vox_paged_prefix_attention_workspace(c, b, None, 4, 0, 0, C.byref(n)),
               L.vox_paged_attention_workspace(c, b, 4, 0, 0, None)):
        refused(V, rc, "ERR_INVALID_ARG", "null")


@pytest.mark.parametrize("theta", [-1.0, 0.5, float("inf"), float("nan")])
def test_append_refuses_thetas(V, theta):
    c, b, _, r = (C.byref(x) for x in descs(V))
    refused(V, V.lib().vox_paged_append_rope(c, b, r, r, theta, 4, r, r, None), "ERR_INVALID_ARG", "rope_theta")


@pytest.mark.parametrize("heads", [0, 3, 1 << 17])
def test_attention_refuses_head_counts(V, heads):
    c, b, _, r = (C.byref(x) for x in descs(V))
    refused(V, V.lib().vox_paged_attention(c, b, r, heads, 0, 0, 0.0, r, None, 0, None), "ERR_INVALID_ARG", "n_heads")


@pytest.mark.parametrize("scale", [-0.1, float("inf"), float("nan")])
def test_attention_refuses_scales(V, scale):
    c, b, _, r = (C.byref(x) for x in descs(V))
    refused(V, V.lib().vox_paged_attention(c, b, r, 4, 0, 0, scale, r, None, 0, None), "ERR_INVALID_ARG", "scale")


def test_rows_are_checked(V):
    L = V.lib()
    for change, code, word in ((dict(ptr=(1 << 20) + 1), "ERR_INVALID_ARG", "aligned"),
                               (dict(token_stride=1 << 41, head_stride=64), "ERR_SHAPE", "strides"),
                               (dict(token_stride=256, head_stride=32), "ERR_SHAPE", "strides")):
        c, b, _, r = (C.byref(x) for x in descs(V))
        bad = C.byref(descs(V, rows=change)[3])
        refused(V, L.vox_paged_attention(c, b, r, 4, 0, 0, 0.0, bad, None, 0, None), code, word)
        refused(V, L.vox_paged_append_rope(c, b, r, r, 1e4, 4, r, bad, None), code, word)


def test_results_must_not_replace_the_queries(V):
    c, b, p, r = (C.byref(x) for x in descs(V))
    L = V.lib()
    refused(V, L.vox_paged_attention(c, b, r, 4, 0, 0, 0.0, r, None, 0, None), "ERR_INVALID_ARG", "out must not be q")
    refused(V, L.vox_paged_prefix_attention(c, b, p, r, 4, 0, 0, 0.0, r, None, 0, None), "ERR_INVALID_ARG", "out must not be q")


def test_prefix_is_checked(V):
    L = V.lib()
    for change, code in ((dict(len=None), "ERR_INVALID_ARG"), (dict(pages=None), "ERR_INVALID_ARG"),
                         (dict(max_len=65), "ERR_SHAPE"), (dict(n_pages=1 << 30), "ERR_UNSUPPORTED")):
        c, b, p, r = (C.byref(x) for x in descs(V, prefix=change))
        refused(V, L.vox_paged_prefix_attention(c, b, p, r, 4, 0, 0, 0.0, r, None, 0, None), code, "")


def test_empty_batches_need_no_device(V):
    for change in (dict(n_seqs=0), dict(n_tokens=0)):
        c, b, p, r = (C.byref(x) for x in descs(V, batch=change))
        L, n = V.lib(), C.c_size_t(7)
        assert L.vox_paged_append_rope(c, b, r, r, 1e4, 4, r, r, None) == 0
        assert L.vox_paged_attention(c, b, r, 4, 0, 0, 0.0, r, None, 0, None) == 0
        assert L.vox_paged_prefix_attention_workspace(c, b, p, 4, 0, 0, C.byref(n)) == 0 and n.value == 0


def test_workspace_is_asked_for(V):
    """A prefix long enough to be read once for all sequences leaves partial results."""
    c, b, p, r = (C.byref(x) for x in descs(V, prefix=dict(n_pages=2100, max_len=33000)))
    L, n = V.lib(), C.c_size_t()
    o = C.byref(descs(V, rows=dict(ptr=OUT))[3])
    assert L.vox_paged_prefix_attention_workspace(c, b, p, 4, 0, 0, C.byref(n)) == 0 and n.value > 0
    refused(V, L.vox_paged_prefix_attention(c, b, p, r, 4, 0, 0, 0.0, o, None, 0, None), "ERR_INVALID_ARG", "workspace")
    refused(V, L.vox_paged_prefix_attention(c, b, p, r, 4, 0, 0, 0.0, o, (1 << 20) + 8, 1 << 30, None),
            "ERR_INVALID_ARG", "workspace")


@pytest.mark.skipif(cuda_available(), reason="checks the no-GPU error path")
def test_without_a_gpu_the_calls_fail_loudly(V):
    c, b, _, r = (C.byref(x) for x in descs(V))
    assert V.lib().vox_paged_append_rope(c, b, r, r, 1e4, 4, r, r, None) == V.ERR_CUDA


def test_python_front_end_refuses(V):
    torch = pytest.importorskip("torch")
    k = torch.zeros(3, 2, 16, 64)
    for bad in ((k, k), (k, torch.zeros(3, 2, 16, 32)), (k[0], k[0]), (k, k.transpose(0, 1)), (k, k.half())):
        with pytest.raises(ValueError):
            V.PagedKvCache(*bad)
    i32 = torch.int32
    ok = dict(q_start=torch.zeros(3, dtype=i32), kv_len=torch.zeros(2, dtype=i32),
              page_table=torch.zeros(2, 4, dtype=i32), n_tokens=2, max_q_len=1)
    for change in (dict(q_start=torch.zeros(2, dtype=i32)), dict(kv_len=torch.zeros(2)), dict(first_pos=torch.zeros(2)),
                   dict(page_table=torch.zeros(3, 4, dtype=i32)), dict(status=torch.zeros(2, dtype=i32)), {}):
        with pytest.raises(ValueError):  # the last one: not CUDA tensors
            V.PagedBatch(**dict(ok, **change))
