"""What becomes of a wait of the latent attention that runs out, as far as it shows without a GPU: the cache's status, and what
the C ABI refuses."""
import ctypes

import pytest
import torch

from fleet import mk
from fleet.latent import LatentCache

P = 1 << 20             # an aligned address that nothing reads


def test_status_and_reset():
    cache = LatentCache(2, 16, 64, 16, device="cpu")
    assert cache.status() == {"error": 0}
    cache.error.fill_(1)
    assert cache.status(raise_on_error=False) == {"error": 1}
    with pytest.raises(mk.MkError) as e:
        cache.status()
    assert e.value.code == mk.MK_EDEVICE and e.value.status == {"error": 1}
    cache.reset()
    assert cache.status() == {"error": 0}


def test_limits():
    assert LatentCache(2, 16, 64, 16, device="cpu").wait_ns == 2 * 10 ** 9
    assert LatentCache(2, 16, 64, 16, device="cpu", wait_timeout_s=1e-9).wait_ns == 1
    for s in (0, -1, 1e-12, 1e30, float("inf"), float("nan")):
        with pytest.raises(ValueError):
            LatentCache(2, 16, 64, 16, device="cpu", wait_timeout_s=s)


def test_abi():
    if not mk.LIB_PATH.exists():
        pytest.skip("library not built")
    l, b = mk.MkLatent(P, P, P, 4, 64, 512, 64), mk.MkLatentBatch(P, P, None, 2, 3, 2)

    def call(error=None, wait_ns=0, rows=3, n=3):
        b.n = n
        return mk.lib().mk_latent_attend_status(ctypes.addressof(l), ctypes.addressof(b), P, 9216, 576, rows, 16, 0, 1.0, P, 8192, 512,
                                                None, P, 1 << 40, error, wait_ns, None)
    for bad in (dict(wait_ns=-1), dict(error=P + 2)):
        assert call(**bad) == mk.MK_EINVAL, bad
    assert call(error=P, wait_ns=1, rows=0, n=0) == mk.MK_OK


def test_only_the_softmax_says_that_its_segment_is_lost():
    """All softmax threads leave a segment or none does, by a word that each reads behind a barrier: no other warp may write it, which
    could come between two readings."""
    text = (mk.PKG / "csrc" / "mk_latent_attend.cu").read_text()
    kernel = text[text.index("void __launch_bounds__(THREADS, 1) attend_kernel"):text.index("// The groups that several blocks' runs share")]
    others, softmax = kernel.split("    // ---- softmax:")
    assert "sh.lost = 1" not in others and softmax.count("sh.lost = 1") == 3 and others.count("sh.late = 1") == 3
