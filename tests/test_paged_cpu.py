"""What the paged cache's entry points and the prompt attention refuse, without a GPU: a call with
a bad argument is PF_ERR_INVALID before a device is looked for."""
import ctypes as C

import pytest

import pocketforge_b200 as pf
from pocketforge_b200 import _lib

INVALID = _lib.PF_ERR_INVALID
A = 1 << 20  # an aligned address that nothing reads: every call here is refused


def cache(**kw):
    d = dict(dtype=_lib.PF_I8, n_layers=2, n_kv_heads=2, head_dim=64, page_size=16, n_pages=32, max_seqs=4,
             max_pages=8, k=A, v=A, k_scale=A, v_scale=A, table=A, lens=A, refs=A, work=A)
    d.update(kw)
    return _lib.PagedCacheC(**d)


def refused(name, *args):
    st = getattr(_lib.lib(), name)(*args)
    assert st == INVALID, (name, st)
    assert name.encode() in _lib.lib().pf_last_error()


BAD = [dict(dtype=_lib.PF_F32), dict(dtype=7), dict(head_dim=96), dict(head_dim=0), dict(page_size=8),
       dict(page_size=48), dict(page_size=256), dict(n_layers=0), dict(n_kv_heads=0), dict(n_pages=0),
       dict(n_pages=-3), dict(max_seqs=0), dict(max_pages=0), dict(max_pages=1 << 30, page_size=128), dict(k=None),
       dict(v=None), dict(k_scale=None), dict(v_scale=None), dict(table=None), dict(lens=None), dict(refs=None),
       dict(k=A + 8), dict(v=A + 4), dict(k_scale=A + 4), dict(n_layers=1 << 20, n_kv_heads=1 << 14)]


@pytest.mark.parametrize("bad", BAD, ids=str)
def test_every_call_refuses_a_bad_cache(bad):
    c = C.byref(cache(**bad))
    refused("pf_paged_reserve", c, A, A, 1, None)
    refused("pf_paged_free", c, A, 1, None)
    refused("pf_paged_fork", c, A, A, 1, None)
    refused("pf_paged_copy", c, A, A, 1, None)
    refused("pf_paged_compact", c, None)
    refused("pf_paged_store", c, 0, A, 128, A, 128, _lib.PF_F32, A, 1, 1, None)
    refused("pf_paged_attention", c, 0, A, 256, A, 256, _lib.PF_F32, 1, 1, 4, 0.125, A, 1 << 30, None)


def test_null_cache():
    refused("pf_paged_reserve", None, A, A, 1, None)
    refused("pf_paged_store", None, 0, A, 128, A, 128, _lib.PF_F32, A, 1, 1, None)
    assert _lib.lib().pf_paged_work_bytes(None) == 0
    assert _lib.lib().pf_paged_attention_work_bytes(None, 1, 1, 4) == 0


def test_page_operations_need_work_and_a_list_that_fits():
    for w in (None, A + 4):
        c = C.byref(cache(work=w))
        refused("pf_paged_reserve", c, A, A, 1, None)
        refused("pf_paged_fork", c, A, A, 1, None)
        refused("pf_paged_compact", c, None)
    c = C.byref(cache())
    for n in (-1, 5):
        refused("pf_paged_reserve", c, A, A, n, None)
        refused("pf_paged_free", c, A, n, None)
        refused("pf_paged_fork", c, A, A, n, None)
    refused("pf_paged_copy", c, A, A, -1, None)
    refused("pf_paged_copy", c, A, A, 33, None)


@pytest.mark.parametrize("bad", [dict(layer=-1), dict(layer=2), dict(ks=120), dict(vs=127), dict(ks=130), dict(k=A + 4),
                                 dict(v=A + 8), dict(dtype=_lib.PF_I8), dict(dtype=9), dict(seqs=-1), dict(seqs=5),
                                 dict(tokens=-1)], ids=str)
def test_store_refusals(bad):
    d = dict(layer=0, k=A, ks=128, v=A, vs=128, dtype=_lib.PF_F32, seqs=2, tokens=3)
    d.update(bad)
    refused("pf_paged_store", C.byref(cache()), d["layer"], d["k"], d["ks"], d["v"], d["vs"], d["dtype"], A, d["seqs"],
            d["tokens"], None)


def test_store_types():
    for cd, rd in ((_lib.PF_BF16, _lib.PF_F16), (_lib.PF_F16, _lib.PF_BF16), (_lib.PF_F16, _lib.PF_I8)):
        refused("pf_paged_store", C.byref(cache(dtype=cd)), 0, A, 128, A, 128, rd, A, 1, 1, None)


@pytest.mark.parametrize("bad", [dict(layer=-1), dict(layer=2), dict(qs=252), dict(os=255), dict(qs=258), dict(q=A + 4),
                                 dict(out=A + 8), dict(dtype=_lib.PF_I8), dict(dtype=9), dict(seqs=-1), dict(seqs=5),
                                 dict(rows=0), dict(rows=9), dict(heads=0), dict(heads=3), dict(heads=-2),
                                 dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")),
                                 dict(bytes=0), dict(work=A + 4)], ids=str)
def test_attention_refusals(bad):
    d = dict(layer=0, q=A, qs=256, out=A, os=256, dtype=_lib.PF_F32, seqs=2, rows=1, heads=4, scale=0.125, work=A,
             bytes=1 << 30)
    d.update(bad)
    refused("pf_paged_attention", C.byref(cache()), d["layer"], d["q"], d["qs"], d["out"], d["os"], d["dtype"],
            d["seqs"], d["rows"], d["heads"], d["scale"], d["work"], d["bytes"], None)


def test_attention_types():
    for cd, rd in ((_lib.PF_BF16, _lib.PF_F16), (_lib.PF_F16, _lib.PF_F32), (_lib.PF_BF16, _lib.PF_F32)):
        refused("pf_paged_attention", C.byref(cache(dtype=cd)), 0, A, 256, A, 256, rd, 1, 1, 4, 0.125, A, 1 << 30, None)


@pytest.mark.parametrize("bad", [dict(dtype=_lib.PF_F32), dict(dtype=_lib.PF_I8), dict(dim=32), dict(dim=256),
                                 dict(heads=0), dict(heads=5), dict(kv=0), dict(kv=-1), dict(seqs=-1), dict(tokens=-1),
                                 dict(qs=248), dict(ks=120), dict(vs=120), dict(os=248), dict(qs=260), dict(os=257),
                                 dict(q=A + 8), dict(k=A + 2), dict(v=A + 4), dict(out=A + 8), dict(scale=0.0),
                                 dict(scale=float("nan")), dict(scale=float("inf")), dict(scale=-0.5)], ids=str)
def test_prompt_refusals(bad):
    d = dict(q=A, qs=256, k=A, ks=128, v=A, vs=128, out=A, os=256, dtype=_lib.PF_BF16, seqs=1, tokens=5, heads=4, kv=2,
             dim=64, scale=0.125)
    d.update(bad)
    refused("pf_prompt_attention", d["q"], d["qs"], d["k"], d["ks"], d["v"], d["vs"], d["out"], d["os"], d["dtype"], A,
            d["seqs"], d["tokens"], d["heads"], d["kv"], d["dim"], d["scale"], None)


def test_a_good_call_needs_a_device():
    if pf.device_count() > 0:
        pytest.skip("a device is present")
    L = _lib.lib()
    c = C.byref(cache())
    none = _lib.PF_ERR_NO_DEVICE
    assert L.pf_paged_reserve(c, A, A, 1, None) == none
    assert L.pf_paged_free(c, A, 1, None) == none
    assert L.pf_paged_fork(c, A, A, 1, None) == none
    assert L.pf_paged_copy(c, A, A, 1, None) == none
    assert L.pf_paged_compact(c, None) == none
    assert L.pf_paged_store(c, 0, A, 128, A, 128, _lib.PF_F32, A, 1, 1, None) == none
    assert L.pf_paged_attention(c, 0, A, 256, A, 256, _lib.PF_F32, 1, 1, 4, 0.125, A, 1 << 30, None) == none
    assert L.pf_prompt_attention(A, 256, A, 128, A, 128, A, 256, _lib.PF_BF16, A, 1, 5, 4, 2, 64, 0.125, None) == none


def test_calls_too_large_to_count():
    refused("pf_paged_store", C.byref(cache()), 0, A, 128, A, 128, _lib.PF_F32, A, 1, (1 << 30) + 1, None)
    for seqs, tokens in (((1 << 20) + 1, 5), (1, (1 << 30) + 1)):
        refused("pf_prompt_attention", A, 256, A, 128, A, 128, A, 256, _lib.PF_BF16, A, seqs, tokens, 4, 2, 64, 0.125, None)
    assert _lib.lib().pf_paged_work_bytes(C.byref(cache(n_pages=(1 << 28) + 1))) == 0
    assert _lib.lib().pf_paged_work_bytes(C.byref(cache(max_seqs=(1 << 20) + 1))) == 0


def test_work_sizes():
    L = _lib.lib()
    assert L.pf_paged_work_bytes(C.byref(cache())) >= 4 * (3 * 32 + 2 * 4)
    assert L.pf_paged_work_bytes(C.byref(cache(n_pages=0))) == 0
    assert L.pf_paged_attention_work_bytes(C.byref(cache()), 4, 8, 4) > 0
    for bad in ((-1, 1, 4), (1, 0, 4), (1, 9, 4), (1, 1, 0), (1, 1, 3)):
        assert L.pf_paged_attention_work_bytes(C.byref(cache()), *bad) == 0


@pytest.mark.parametrize("off", [1, 2, 3])
def test_lists_that_are_not_aligned(off):
    """Arrays of 32-bit integers begin at a multiple of 4 bytes."""
    for name in ("table", "lens", "refs"):
        c = C.byref(cache(**{name: A + off}))
        refused("pf_paged_reserve", c, A, A, 1, None)
        refused("pf_paged_free", c, A, 1, None)
        refused("pf_paged_fork", c, A, A, 1, None)
        refused("pf_paged_copy", c, A, A, 1, None)
        refused("pf_paged_compact", c, None)
        refused("pf_paged_store", c, 0, A, 128, A, 128, _lib.PF_F32, A, 1, 1, None)
        refused("pf_paged_attention", c, 0, A, 256, A, 256, _lib.PF_F32, 1, 1, 4, 0.125, A, 1 << 30, None)
    c = C.byref(cache())
    for a, b in ((A + off, A), (A, A + off)):
        refused("pf_paged_reserve", c, a, b, 1, None)
        refused("pf_paged_fork", c, a, b, 1, None)
        refused("pf_paged_copy", c, a, b, 1, None)
    refused("pf_paged_free", c, A + off, 1, None)
    refused("pf_paged_store", c, 0, A, 128, A, 128, _lib.PF_F32, A + off, 1, 1, None)
    refused("pf_prompt_attention", A, 256, A, 128, A, 128, A, 256, _lib.PF_BF16, A + off, 1, 5, 4, 2, 64, 0.125, None)


def test_scales_whose_log2_units_are_no_number():
    """Scores are taken to log2 units by scale * log2 e: a scale that has none there is refused."""
    for scale in (2.4e38, 3.4e38):
        refused("pf_paged_attention", C.byref(cache()), 0, A, 256, A, 256, _lib.PF_F32, 1, 1, 4, scale, A, 1 << 30, None)
        refused("pf_prompt_attention", A, 256, A, 128, A, 128, A, 256, _lib.PF_BF16, A, 1, 5, 4, 2, 64, scale, None)


SIZES = [dict(dtype=_lib.PF_F32), dict(dtype=7), dict(head_dim=96), dict(page_size=48), dict(n_layers=0), dict(n_kv_heads=0),
         dict(n_pages=-3), dict(max_seqs=0), dict(max_pages=0), dict(max_pages=1 << 30, page_size=128),
         dict(n_layers=1 << 20, n_kv_heads=1 << 14)]


@pytest.mark.parametrize("bad", SIZES, ids=str)
def test_no_work_size_for_sizes_that_are_refused(bad):
    c = C.byref(cache(**bad))
    assert _lib.lib().pf_paged_work_bytes(c) == 0
    assert _lib.lib().pf_paged_attention_work_bytes(c, 2, 1, 4) == 0


def test_no_work_size_for_heads_that_are_refused():
    """65,536 heads and more; the columns of 2^31 - 2 of them, 8 rows each, would pass 32 bits."""
    for heads in (65_536, (1 << 31) - 2):
        assert _lib.lib().pf_paged_attention_work_bytes(C.byref(cache()), 2, 8, heads) == 0
    assert _lib.lib().pf_paged_attention_work_bytes(C.byref(cache(n_kv_heads=1)), 2, 8, 65_535) > 0


def test_work_sizes_need_no_pointers():
    """The size is asked for before there is a cache."""
    c = cache(k=None, v=None, k_scale=None, v_scale=None, table=None, lens=None, refs=None, work=None)
    assert _lib.lib().pf_paged_work_bytes(C.byref(c)) == _lib.lib().pf_paged_work_bytes(C.byref(cache())) > 0
    assert _lib.lib().pf_paged_attention_work_bytes(C.byref(c), 2, 1, 4) > 0
