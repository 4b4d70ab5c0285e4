"""uwc_amd.kv and its C-ABI refuse what they cannot take before any GPU work (no GPU needed)."""
import ctypes

import pytest
import torch

BF = torch.bfloat16


def cpu_cache(pages=4, Hkv=2, hd=64, page=16):
    from uwc_amd import kv
    return kv.new_cache(pages, Hkv, hd, page, "cpu")


@pytest.mark.parametrize("kwargs", [dict(page=48), dict(page=8), dict(hd=96), dict(hd=256), dict(pages=0), dict(Hkv=0)])
def test_new_cache_refuses(kwargs):
    with pytest.raises(AssertionError, match="new_cache"):
        cpu_cache(**kwargs)


def test_cache_must_be_of_one_layout():
    from uwc_amd import kv
    k, v, ks, vs = cpu_cache()
    q, table, lens = torch.zeros((1, 4, 64), dtype=BF), torch.zeros((1, 2), dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    for bad in ((k, k, ks, vs), (k.float(), v, ks, vs), (k, v, ks.double(), vs), (k, v, ks, vs[:2]), (k, v[:2], ks, vs)):
        with pytest.raises(AssertionError, match="the cache is int8"):
            kv.attend(bad, q, table, lens)
    with pytest.raises(AssertionError, match="contiguous"):
        kv.attend((k.transpose(2, 3).contiguous().transpose(2, 3), v, ks, vs), q, table, lens)


@pytest.mark.parametrize("change,msg", [
    (dict(q=torch.zeros((1, 3, 64), dtype=BF)), "multiple of 2"),
    (dict(q=torch.zeros((1, 4, 32), dtype=BF)), "q must be"),
    (dict(q=torch.zeros((1, 0, 64), dtype=BF)), "q must be"),
    (dict(q=torch.zeros((4, 64), dtype=BF)), "q must be"),
    (dict(q=torch.zeros((1, 4, 64))), "bfloat16 or float16"),
    (dict(q=torch.zeros((2, 4, 64), dtype=BF)), "one row"),
    (dict(table=torch.zeros((1, 2), dtype=torch.int64)), "page table"),
    (dict(table=torch.zeros(2, dtype=torch.int32)), "page table"),
    (dict(lens=torch.ones(2, dtype=torch.int32)), "lens must be"),
    (dict(lens=torch.ones(1)), "lens must be"),
    (dict(cu=torch.zeros(1, dtype=torch.int32)), "cu must be"),
    (dict(cu=torch.zeros(2, dtype=torch.int64)), "cu must be"),
    (dict(window=-1), "window"),
    (dict(sinks=4), "sinks need a window"),
    (dict(window=8, sinks=-1), "sinks"),
])
def test_attend_refuses(change, msg):
    from uwc_amd import kv
    a = dict(q=torch.zeros((1, 4, 64), dtype=BF), table=torch.zeros((1, 2), dtype=torch.int32), lens=torch.ones(1, dtype=torch.int32))
    a.update(change)
    with pytest.raises(AssertionError, match=msg):
        kv.attend(cpu_cache(), **a)


@pytest.mark.parametrize("change,msg", [
    (dict(qkv=torch.zeros((1, 8 * 64 + 8), dtype=BF)), "whole q heads"),
    (dict(qkv=torch.zeros((1, 3 * 64), dtype=BF)), "whole q heads"),
    (dict(qkv=torch.zeros((1, 8, 64), dtype=BF)), "qkv must be"),
    (dict(qkv=torch.zeros((1, 8 * 64))), "bfloat16 or float16"),
    (dict(qkv=torch.zeros((3, 8 * 64), dtype=BF)), "one row"),
    (dict(ctx=torch.zeros(1, dtype=torch.int64)), "ctx must be"),
    (dict(cos=torch.zeros((4, 32))), "cos must be"),
    (dict(sin=torch.zeros((5, 64))), "sin must be"),
    (dict(cos=torch.zeros((4, 64), dtype=torch.float64)), "cos must be"),
    (dict(q_norm=torch.zeros(32)), "q_norm must be"),
    (dict(k_norm=torch.zeros(64, dtype=BF)), "k_norm must be"),
    (dict(cu=torch.zeros(3, dtype=torch.int32)), "cu must be"),
])
def test_append_refuses(change, msg):
    from uwc_amd import kv
    a = dict(qkv=torch.zeros((1, 8 * 64), dtype=BF), table=torch.zeros((1, 2), dtype=torch.int32), ctx=torch.zeros(1, dtype=torch.int32),
             cos=torch.zeros((4, 64)), sin=torch.zeros((4, 64)))
    a.update(change)
    with pytest.raises(AssertionError, match=msg):
        kv.append(cpu_cache(), **a)


def test_read_refuses():
    from uwc_amd import kv
    table, one, cu = torch.zeros((1, 2), dtype=torch.int32), torch.zeros(1, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    for args, kw, msg in (((table, one, cu, -1), {}, "rows"), ((table, one, cu, 1), dict(dtype=torch.float32), "dtype"),
                          ((table, one, one, 1), {}, "cu must be"), ((table, cu, cu, 1), {}, "start must be")):
        with pytest.raises(AssertionError, match=msg):
            kv.read(cpu_cache(), *args, **kw)


FAKE = ctypes.c_void_p(1 << 20)  # aligned, never dereferenced: validation fails first
ODD = ctypes.c_void_p((1 << 20) + 8)


def attend_call(**change):
    from uwc_amd import _lib
    a = dict(k=FAKE, v=FAKE, ks=FAKE, vs=FAKE, pages=4, page=16, Hkv=2, hd=64, q=FAKE, q_stride=256, dtype=0, T=1, H=4, table=FAKE,
             table_stride=2, width=2, lens=FAKE, cu=None, B=1, max_new=1, max_len=32, window=0, sinks=0, scale=1.0, scratch=None,
             scratch_bytes=0, o=FAKE, stream=None)
    a.update(change)
    st = _lib.lib().uwc_kv_attend(*a.values())
    return st, _lib.lib().uwc_last_error().decode()


@pytest.mark.parametrize("change,msg", [
    (dict(k=None), "null cache"), (dict(q=None), "null"), (dict(pages=0), "bad pages"), (dict(page=24), "page 24"),
    (dict(hd=80), "head_dim 80"), (dict(dtype=2), "unknown dtype"), (dict(H=5), "no multiple"), (dict(T=2), "one row"),
    (dict(q_stride=252), "16-byte aligned"), (dict(q=ODD), "16-byte aligned"), (dict(o=ODD), "16-byte aligned"),
    (dict(sinks=3), "sinks"), (dict(window=-2), "window"), (dict(T=-1), "bad T"),
    (dict(T=1 << 30, cu=FAKE, H=8), "too many"), (dict(max_len=1 << 20), "scratch holds 0 bytes"),
])
def test_attend_entry_refuses(change, msg):
    st, err = attend_call(**change)
    assert st == -1 and "uwc_kv_attend" in err and msg in err


def test_attend_scratch_one_byte_short():
    from uwc_amd import _lib
    need = _lib.lib().uwc_kv_attend_scratch_bytes(1, 1, 0, 4, 2, 64, 1, 1 << 20, 0, 0)
    assert need > 0
    st, err = attend_call(max_len=1 << 20, scratch=FAKE, scratch_bytes=need - 1)
    assert st == -1 and f"scratch holds {need - 1} bytes, {need} needed" in err
    assert _lib.lib().uwc_kv_attend_scratch_bytes(0, 1, 0, 4, 2, 64, 1, 1 << 20, 0, 0) == 0


def test_other_entries_refuse():
    from uwc_amd import _lib
    L = _lib.lib()

    def append(**change):
        a = dict(qkv=FAKE, stride=512, dtype=0, T=1, B=1, cu=None, ctx=FAKE, table=FAKE, table_stride=2, width=2, cos=FAKE, sin=FAKE,
                 positions=4, qn=None, kn=None, eps=1e-6, H=4, Hkv=2, hd=64, page=16, pages=4, k=FAKE, v=FAKE, ks=FAKE, vs=FAKE,
                 q=FAKE, stream=None)
        a.update(change)
        return L.uwc_kv_append(*a.values()), L.uwc_last_error().decode()

    for change, msg in ((dict(qkv=None), "null"), (dict(qkv=ODD), "aligned"), (dict(stride=508), "aligned"), (dict(k=ODD), "aligned"),
                        (dict(T=3), "one row"), (dict(positions=0), "empty"), (dict(page=17), "page 17"), (dict(H=-1), "bad T"),
                        (dict(T=1 << 30, cu=FAKE), "too many")):
        st, err = append(**change)
        assert st == -1 and "uwc_kv_append" in err and msg in err, change

    def read(**change):
        a = dict(k=FAKE, v=FAKE, ks=FAKE, vs=FAKE, pages=4, page=16, Hkv=2, hd=64, table=FAKE, table_stride=2, width=2, start=FAKE,
                 cu=FAKE, B=1, rows=1, dtype=0, ko=FAKE, vo=FAKE, stream=None)
        a.update(change)
        return L.uwc_kv_read(*a.values()), L.uwc_last_error().decode()

    for change, msg in ((dict(cu=None), "null"), (dict(vo=ODD), "aligned"), (dict(rows=-1), "bad rows"), (dict(vs=None), "null cache"),
                        (dict(rows=1 << 30, Hkv=64), "too many")):
        st, err = read(**change)
        assert st == -1 and "uwc_kv_read" in err and msg in err, change


def test_short_way_is_built_from_this_header_and_declines_other_forms(monkeypatch):
    """_kv.so carries the header's stamp, returns None for what is not of the usual form (here: not on a GPU) or
    not as many arguments as it takes, and is refused when it was built from another header."""
    from uwc_amd import _lib
    k = _lib.kv()
    assert k.header_sha() == _lib.lib().uwc_header_sha().decode()
    cache = cpu_cache()
    q, table, lens = torch.zeros((1, 4, 64), dtype=BF), torch.zeros((1, 2), dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    assert k.attend(*cache, q, table, lens, None, None, None, 0, 0, None, 0) is None
    assert k.attend(*cache, q) is None and k.attend() is None
    assert k.append(1, 2, 3, 4, 5, 6, 7, 8, 9, None, None, None, 1e-6, 0) is None
    assert k.read(*cache, table, lens, lens, 1, False, 0) is None
    with pytest.raises(TypeError):
        k.bind(1)

    class Other:
        header_sha = staticmethod(lambda: "0" * 16)

    import sys
    import uwc_amd
    monkeypatch.setattr(_lib, "_KV", None)
    monkeypatch.setitem(sys.modules, "uwc_amd._kv", Other)
    monkeypatch.setattr(uwc_amd, "_kv", Other, raising=False)
    with pytest.raises(ImportError, match="different include/uwc.h"):
        _lib.kv()
