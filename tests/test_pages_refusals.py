"""uwc_amd.pages and its C-ABI refuse what they cannot take before any GPU work (no GPU needed)."""
import ctypes

import pytest
import torch


def cpu(pages=4, Hkv=2, hd=64, page=16):
    from uwc_amd import kv
    return kv.new_cache(pages, Hkv, hd, page, "cpu")


def i(*s, dt=torch.int32):
    return torch.zeros(s, dtype=dt)


@pytest.mark.parametrize("change,msg", [
    (dict(caches=[]), "no caches"), (dict(caches=[cpu(), cpu(pages=5)]), "one shape"), (dict(caches=[cpu(), cpu(hd=32)]), "one shape"),
    (dict(caches=[(i(2), i(2), i(2), i(2))]), "unpack"), (dict(table=i(2, 3, dt=torch.int64)), "page table"), (dict(table=i(3)), "page table"),
    (dict(table=i(4097, 1), lens=i(4097)), "4097 rows"), (dict(refs=i(3)), "refs must be"), (dict(refs=i(4, dt=torch.int64)), "refs must be"),
    ({}, "must be on a GPU"),
])
def test_both_refuse(change, msg):
    from uwc_amd import pages
    a = dict(caches=[cpu(), cpu()], table=i(2, 3), lens=i(2), refs=i(4), parents=i(2))
    a.update(change)
    with pytest.raises((AssertionError, ValueError), match=msg):
        pages.fork(**a)
    with pytest.raises((AssertionError, ValueError), match=msg):
        pages.compact(a["caches"], a["table"], a["refs"])


def test_fork_refuses_negative_room():
    from uwc_amd import pages
    with pytest.raises(AssertionError, match="room=-1"):
        pages.fork([cpu()], i(2, 3), i(2), i(4), i(2), room=-1)


FAKE, ODD = 1 << 20, (1 << 20) + 8


def call(name, caches=(FAKE,) * 8, **change):
    from uwc_amd import _lib
    L = _lib.lib()
    a = dict(layers=len(caches) // 4, caches=(ctypes.c_void_p * len(caches))(*caches), pages=4, page=16, Hkv=2, hd=64, table=FAKE, stride=3,
             width=3, lens=FAKE, B=2, refs=FAKE, parents=FAKE, R=2, room=1, new_table=FAKE, new_lens=FAKE, new_refs=FAKE, missing=FAKE,
             scratch=FAKE, bytes=1 << 20, stream=None)
    a.update(change)
    if name == "uwc_kv_compact":
        for k in ("lens", "parents", "R", "room", "new_lens", "missing"):
            del a[k]
    return getattr(L, name)(*a.values()), L.uwc_last_error().decode()


@pytest.mark.parametrize("change,msg", [
    (dict(layers=-1), "layers"), (dict(caches=(FAKE, FAKE, None, FAKE)), "null cache"), (dict(caches=(ODD, FAKE, FAKE, FAKE)), "aligned"),
    (dict(caches=(FAKE, ODD, FAKE, FAKE)), "aligned"), (dict(pages=0), "pages"), (dict(pages=(1 << 21) + 1), "pages"), (dict(Hkv=0), "Hkv"),
    (dict(Hkv=65536), "Hkv"), (dict(page=24), "page 24"), (dict(hd=96), "head_dim"), (dict(width=-1), "bad width"), (dict(B=-1), "rows"),
    (dict(B=4097), "rows"), (dict(width=1 << 22, B=1000), "2^31"), (dict(stride=-1), "bad width"), (dict(table=None), "null"), (dict(refs=None), "null"),
    (dict(scratch=None), "null"), (dict(bytes=100), "scratch"), (dict(scratch=ODD), "scratch"), (dict(new_table=None), "null"),
    (dict(new_refs=None), "null"),
])
def test_the_library_refuses(change, msg):
    for name in ("uwc_kv_fork", "uwc_kv_compact"):
        st, err = call(name, **change)
        assert st == -1 and name in err and msg in err


@pytest.mark.parametrize("change,msg", [
    (dict(R=-1), "rows"), (dict(R=4097), "rows"), (dict(room=-1), "room"), (dict(lens=None), "null"), (dict(parents=None), "null"),
    (dict(new_lens=None), "null"), (dict(missing=None), "null"), (dict(width=1 << 28), "2^31"),
])
def test_fork_of_the_library_refuses(change, msg):
    st, err = call("uwc_kv_fork", **change)
    assert st == -1 and msg in err


def test_scratch_bytes():
    from uwc_amd import _lib
    f = _lib.lib().uwc_kv_pages_scratch_bytes
    assert f(0, 5) == 0 and f(5, -1) == 0
    assert f(1, 0) == f(1024, 0) == 132 and f(1025, 3) == 2 * 132 + 48


def test_short_way_declines_other_forms():
    from uwc_amd import _lib
    k = _lib.kv()
    assert k.fork([cpu()], i(2, 3), i(2), i(4), i(2), 0, 0) is None and k.fork() is None and k.fork((), 1, 2, 3, 4, 5, 6) is None
    assert k.compact([cpu()], i(2, 3), i(4), 0) is None and k.compact([1], i(2, 3), i(4), 0) is None
    assert k.linear(torch.zeros((1, 32)), i(2, 16, dt=torch.uint8), i(2, 1, dt=torch.uint8), None, 0) is None and k.linear(1, 2, 3, 4, 5) is None
    assert k.gated(torch.zeros((1, 32)), i(2, 16, dt=torch.uint8), i(2, 1, dt=torch.uint8), 0) is None
