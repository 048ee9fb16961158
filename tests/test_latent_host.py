"""What the latent attention's operators refuse, without a GPU: the Python objects' checks, and the C ABI's over
pointers that are never followed."""
import ctypes

import pytest
import torch

from fleet import mk
from fleet.latent import LatentBatch, LatentCache, _beside
from fleet.rope import Rope, _apart, overlap

P = 1 << 20             # an aligned address that nothing reads


@pytest.fixture(scope="module")
def lib():
    if not mk.LIB_PATH.exists():
        pytest.skip("library not built")
    return mk.lib()


def test_rope_is_refused():
    f = torch.ones(32, dtype=torch.float64)
    for bad in (torch.ones(2, 2, dtype=torch.float64), torch.ones(0), torch.ones(257), torch.ones(4).half(), torch.ones(4).long()):
        with pytest.raises(ValueError):
            Rope(bad)
    with pytest.raises(ValueError):
        Rope(f, layout="pairs")
    with pytest.raises(ValueError):
        Rope(f, scale=float("inf"))
    with pytest.raises(mk.MkError):       # no fallback
        Rope(f)(torch.zeros(1, 1, 64).bfloat16(), torch.zeros(1, dtype=torch.int64))
    with pytest.raises(mk.MkError):
        Rope(f)(torch.zeros(1, 1, 64).bfloat16(), torch.zeros(1, dtype=torch.int64), stream=0)
    given = torch.ones(4)
    rope = Rope(given)
    given.zero_()                         # the object's frequencies are its own
    assert rope.dim == 8 and rope.inv_freq.dtype == torch.float64 and rope.inv_freq.all()


def test_cache_is_refused():
    for args in ((0, 64, 512, 64), (4, 48, 512, 64), (4, 64, 520, 64), (4, 64, 12, 64), (4, 64, 512, 72), (4, 64, 512, 0),
                 (4, 64, 0, 64), (2 ** 25, 64, 8, 8)):
        with pytest.raises(ValueError):
            LatentCache(*args, device="meta")
    cache = LatentCache(3, 16, 200, 24, device="cpu")
    assert cache.c_codes.shape == (3, 16, 200) and cache.c_codes.stride() == (16 * 256, 256, 1) and cache.r_codes.shape == (3, 16, 24)
    batch = LatentBatch(torch.zeros(2, 1, dtype=torch.int32), torch.zeros(2, dtype=torch.int32))
    for call in (lambda: cache.append(torch.zeros(2, 200).half(), torch.zeros(2, 24).half(), batch), lambda: cache.read(batch, 2),
                 lambda: cache.attend(torch.zeros(2, 4, 224).half(), batch, 1.0)):
        with pytest.raises(mk.MkError):   # no fallback
            call()


def test_batch_is_refused():
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    LatentBatch(i(3, 2), i(3), i(4))
    LatentBatch(i(3, 9)[:, :2], i(3))
    for args in ((i(3, 2).long(), i(3)), (i(3, 2), i(3).long()), (i(2, 2), i(3)), (i(3, 0), i(3)), (i(6), i(3)), (i(2, 3).T, i(3)),
                 (i(3, 2), i(3, 1)), (i(3, 2), i(6)[::2]), (i(3, 2), i(3), i(3)), (i(3, 2), i(3), i(4).long()), (i(3, 2), i(3), i(8)[::2])):
        with pytest.raises(ValueError):
            LatentBatch(*args)


def test_overlaps():
    z = torch.zeros(10, 600)
    assert _beside(z[:, :512], z[:, 512:576]) and _beside(z[:, 64:576], z[:, :64]) and _beside(z[:5, :64], z[5:, 64:576])
    assert not _beside(z[:, :512], z[:, 511:575]) and not _beside(z[:, :512], z[:, :64])
    assert overlap(z[:, :512], z[:, 511:575]) and not overlap(z[:5], z[5:])
    assert _apart((3, 4, 64), (256, 64, 1)) and _apart((3, 4, 64), (64, 192, 1)) and _apart((1, 4, 64), (0, 64, 1))
    assert not _apart((3, 4, 64), (0, 64, 1)) and not _apart((3, 4, 64), (256, 63, 1)) and not _apart((3, 4, 64), (128, 64, 1))


def rope(lib, dim=64, layout=0, dtype=0, pos64=1, inv=P, pos=P, t=2, x=P, heads=2, width=64, start=0, out=2 * P):
    r = mk.MkRope(inv, dim, layout, dtype, pos64, 1.0, 0)
    return lib.mk_rope(ctypes.addressof(r), pos, t, x, 128, 64, heads, width, start, out, 128, 64, None)


def test_rope_abi(lib):
    assert lib.mk_rope(None, P, 1, P, 1, 1, 1, 64, 0, P, 1, 1, None) == mk.MK_EINVAL
    for bad in (dict(dim=0), dict(dim=63), dict(dim=514, width=600), dict(layout=3), dict(layout=-1), dict(dtype=2), dict(t=-1),
                dict(heads=-1), dict(start=1), dict(start=-1), dict(width=62), dict(heads=2 ** 26), dict(inv=None), dict(inv=P + 4),
                dict(pos=None), dict(pos=P + 4), dict(pos=P + 2, pos64=0), dict(x=None), dict(x=P + 1), dict(out=None), dict(out=P + 1)):
        assert rope(lib, **bad) == mk.MK_EINVAL, bad
    assert rope(lib, t=0) == mk.MK_OK and rope(lib, heads=0) == mk.MK_OK


def structs(c=P, r=P, scales=P, pages=4, page=64, d_c=512, d_r=64, table=P, lens=P, starts=None, ldt=2, n=3, width=2):
    return mk.MkLatent(c, r, scales, pages, page, d_c, d_r), mk.MkLatentBatch(table, lens, starts, ldt, n, width)


BAD = [dict(c=None), dict(c=P + 64), dict(r=None), dict(r=P + 64), dict(scales=None), dict(scales=P + 4), dict(pages=0), dict(page=48),
       dict(pages=2 ** 25), dict(d_c=0), dict(d_c=520), dict(d_c=20), dict(d_r=0), dict(d_r=72), dict(d_r=12), dict(table=None), dict(table=P + 2),
       dict(lens=None), dict(lens=P + 2), dict(starts=P + 2), dict(ldt=-1), dict(n=-1), dict(width=0), dict(width=2 ** 25)]


def test_latent_abi(lib):
    def append(rows=3, dtype=0, xc=P, xr=P, **kw):
        l, b = structs(**kw)
        return lib.mk_latent_append(ctypes.addressof(l), ctypes.addressof(b), xc, 512, xr, 64, rows, dtype, None)

    def read(rows=3, dtype=0, xc=P, xr=P, **kw):
        l, b = structs(**kw)
        return lib.mk_latent_read(ctypes.addressof(l), ctypes.addressof(b), xc, 512, xr, 64, rows, dtype, 0, None)

    def attend(rows=3, dtype=0, heads=16, q=P, out=P, lse=None, ws=P, nbytes=1 << 40, scale=1.0, **kw):
        l, b = structs(**kw)
        return lib.mk_latent_attend(ctypes.addressof(l), ctypes.addressof(b), q, 9216, 576, rows, heads, dtype, scale, out, 8192, 512, lse, ws,
                                    nbytes, None)
    for call in (append, read, attend):
        for bad in BAD + [dict(rows=-1), dict(rows=2), dict(dtype=2), dict(dtype=-1)]:
            assert call(**bad) == mk.MK_EINVAL, (call.__name__, bad)
        assert call(n=0, rows=0) == mk.MK_OK and call(n=0, rows=0, table=None, lens=None) == mk.MK_OK
        assert call(rows=0, starts=P) == mk.MK_OK
    for call in (append, read):
        for bad in (dict(xc=None), dict(xr=None), dict(xc=P + 1), dict(xr=P + 1)):
            assert call(**bad) == mk.MK_EINVAL, (call.__name__, bad)
    for bad in (dict(heads=0), dict(heads=-1), dict(heads=1025), dict(q=None), dict(q=P + 1), dict(out=None), dict(out=P + 1), dict(lse=P + 2)):
        assert attend(**bad) == mk.MK_EINVAL, bad
    l, _ = structs()
    need = ctypes.c_int64()
    for args in ((None, 3, 3, 16, ctypes.byref(need)), (ctypes.addressof(l), -1, 3, 16, ctypes.byref(need)),
                 (ctypes.addressof(l), 3, -1, 16, ctypes.byref(need)), (ctypes.addressof(l), 3, 3, 0, ctypes.byref(need)), (ctypes.addressof(l), 3, 3, 16, None)):
        assert lib.mk_latent_attend_workspace(*args) == mk.MK_EINVAL
    assert lib.mk_latent_attend_workspace(ctypes.addressof(l), 3, 3, 16, ctypes.byref(need)) == mk.MK_OK
