"""CPU tests of the paged-cache entry points among other calls: errors that one
call leaves for the next, layouts whose rows overlap, arguments at their limits."""
import ctypes as C

import pytest

from tests.test_paged_host import OUT, descs, refused
from tests.vox_testlib import cuda_available, vox


@pytest.fixture(scope="module")
def V():
    return vox()


@pytest.mark.skipif(cuda_available(), reason="needs a call that fails without a GPU")
def test_an_error_that_was_reported_is_not_reported_again(V):
    c, b, _, r = (C.byref(x) for x in descs(V))
    cfg = V.DecoderConfig(dim=8, hidden_dim=16, n_heads=2, n_kv_heads=1, head_dim=4, sliding_window=4, norm_eps=1e-5,
                          rope_theta=1e4)
    for _ in range(2):
        with pytest.raises(V.VoxError) as e:
            V.Context(cfg)
        assert e.value.code == V.ERR_CUDA
        assert V.lib().vox_paged_append_rope(c, b, r, r, 1e4, 4, r, r, None) == V.ERR_CUDA
        assert "cannot use device" in V.last_error()


def test_rows_that_are_written_must_not_overlap(V):
    """3 tokens of 4 heads of 64."""
    L = V.lib()
    c, b, _, r = (C.byref(x) for x in descs(V))
    for token, head in ((64, 64), (255, 64), (64, 191), (256, 63), (100, 100)):
        out = C.byref(descs(V, rows=dict(ptr=OUT, token_stride=token, head_stride=head))[3])
        refused(V, L.vox_paged_attention(c, b, r, 4, 0, 0, 0.0, out, None, 0, None), "ERR_SHAPE", "strides")
        refused(V, L.vox_paged_append_rope(c, b, r, r, 1e4, 4, r, out, None), "ERR_SHAPE", "strides")
    for token, head in ((256, 64), (64, 192), (1000, 100), (1 << 40, 64)):
        out = C.byref(descs(V, rows=dict(ptr=OUT, token_stride=token, head_stride=head))[3])
        if not cuda_available():  # (made-up addresses: past the checks there is only the missing device)
            assert L.vox_paged_attention(c, b, r, 4, 0, 0, 0.0, out, None, 0, None) == V.ERR_CUDA
            assert L.vox_paged_append_rope(c, b, r, r, 1e4, 4, r, out, None) == V.ERR_CUDA


def test_a_pool_that_is_written_must_not_overlap(V):
    """10 pages of 2 heads of 16 slots of 64."""
    L = V.lib()
    for page, head, slot in ((64, 64, 64), (2047, 1024, 64), (2048, 64, 64), (2048, 1023, 64), (2048, 64, 127),
                             (1024, 1024, 64), (64, 640, 640)):
        c, b, _, r = (C.byref(x) for x in descs(V, cache=dict(page_stride=page, head_stride=head, slot_stride=slot)))
        refused(V, L.vox_paged_append_rope(c, b, r, r, 1e4, 4, r, r, None), "ERR_SHAPE", "strides")
    for page, head, slot in ((2048, 1024, 64), (2048, 64, 128), (4096, 1024, 64), (64, 10240, 640), (64, 640, 1280)):
        c, b, _, r = (C.byref(x) for x in descs(V, cache=dict(page_stride=page, head_stride=head, slot_stride=slot)))
        if not cuda_available():
            assert L.vox_paged_append_rope(c, b, r, r, 1e4, 4, r, r, None) == V.ERR_CUDA


def test_queries_in_place_keep_their_strides(V):
    L = V.lib()
    c, b, _, r = (C.byref(x) for x in descs(V))
    wide = C.byref(descs(V, rows=dict(token_stride=512, head_stride=64))[3])
    for q, out in ((r, wide), (wide, r)):
        refused(V, L.vox_paged_append_rope(c, b, r, r, 1e4, 4, q, out, None), "ERR_SHAPE", "strides")
    if not cuda_available():
        assert L.vox_paged_append_rope(c, b, r, r, 1e4, 4, wide, wide, None) == V.ERR_CUDA


def test_negative_windows_and_sinks_are_refused(V):
    for kw in (dict(sliding_window=-1), dict(n_sinks=-3)):
        with pytest.raises(ValueError, match="sliding_window and n_sinks"):
            V.paged_attention(None, None, None, **kw)


def test_scales_that_overflow_are_refused(V):
    """The kernels work in powers of two: scale times log2(e) has to be finite."""
    c, b, p, r = (C.byref(x) for x in descs(V))
    L = V.lib()
    refused(V, L.vox_paged_attention(c, b, r, 4, 0, 0, 3e38, r, None, 0, None), "ERR_INVALID_ARG", "scale")
    refused(V, L.vox_paged_prefix_attention(c, b, p, r, 4, 0, 0, 3e38, r, None, 0, None), "ERR_INVALID_ARG", "scale")


def test_append_refuses_rotated_queries_without_queries(V):
    c, b, _, r = (C.byref(x) for x in descs(V))
    refused(V, V.lib().vox_paged_append_rope(c, b, r, r, 1e4, 4, None, r, None), "ERR_INVALID_ARG", "q_out")
    with pytest.raises(ValueError, match="q_out needs q"):
        V.paged_append_rope(None, None, None, None, 1e4, q_out=object())
