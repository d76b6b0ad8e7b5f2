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
