"""Host-side behaviour of the prompt entry points and the block-scaled decode at
the edges of their contracts (no GPU, no kernel launch)."""

from types import SimpleNamespace

import pytest

from persistentkv_attention_b200.serving import NativeEngine
from tests.test_prompt_abi import decode, slots, write


# ------------------------------------------------------------------ nothing to do
@pytest.mark.parametrize("fp8", [False, True])
def test_write_of_no_tokens_needs_no_tokens(lib, fp8):
    assert write(lib, fp8, T=0, k=None, v=None, slots=None) == 0
    for kw, msg in ((dict(kp=None), b"k_pages"), (dict(dtype=7), b"dtype"), (dict(d=64), b"d=128")):
        assert write(lib, fp8, T=0, k=None, v=None, slots=None, **kw) != 0
        assert msg in lib.pkv_last_error_message()


def test_block_decode_of_no_rows_needs_no_rows(lib):
    none = dict(B=0, q=None, bt=None, sl=None, out=None, ws=None, wsb=0, qr=0, orow=0)
    assert decode(lib, **none) == 0
    for kw, msg in ((dict(ks=None), b"k_scales"), (dict(k=None), b"k_pages"),
                    (dict(dtype=3), b"dtype"), (dict(Hq=24), b"G=3"), (dict(block=8), b"of 16")):
        assert decode(lib, **{**none, **kw}) != 0
        assert msg in lib.pkv_last_error_message()


# ------------------------------------------------------------------ overlaps
# 4 rows of 8 pages, 64 slots, a stack of 32: each buffer on a page of its own
APART = dict(cached=1 << 20, new=2 << 20, table=3 << 20, slots=4 << 20, cu=5 << 20, seq=6 << 20,
             free=7 << 20, count=8 << 20, left=9 << 20, ctr=10 << 20)


@pytest.mark.parametrize("kw", [
    dict(seq=(1 << 20) + 4), dict(seq=(1 << 20) - 12), dict(cu=(2 << 20) - 16),
    dict(slots=(1 << 20) - 252), dict(slots=(2 << 20) + 12), dict(table=(1 << 20) - 124),
    dict(seq=(3 << 20) + 124), dict(cu=(4 << 20) + 252), dict(cu=6 << 20), dict(seq=7 << 20),
    dict(table=(7 << 20) + 124), dict(slots=8 << 20), dict(left=(7 << 20) + 4),
    dict(left=(4 << 20) + 252), dict(ctr=9 << 20), dict(ctr=8 << 20), dict(left=6 << 20),
    dict(left=8 << 20, ctr=8 << 20), dict(left=8 << 20, slots=(8 << 20) - 252),
    dict(free=None, count=None, left=None, ctr=None, seq=(3 << 20) + 4)])
def test_slots_refuses_overlaps(lib, kw):
    assert slots(lib, **{**APART, **kw}) == 1
    assert b"must not overlap" in lib.pkv_last_error_message()


# ------------------------------------------------------------------ prefill
def prefill(lib, **kw):
    """40 tokens of 32 / 8 heads, 64 pages of 16: each operand 256 MB from the next."""
    a = dict(q=1 << 28, k=2 << 28, v=3 << 28, out=4 << 28, lse=5 << 28, kp=6 << 28, vp=7 << 28,
             ks=None, vs=None, B=2, T=40, Hq=32, Hkv=8, d=128, qt=4096, qh=128, kt=1024, kh=128,
             vt=1024, vh=128, P=64, page=16, block=0, dtype=0)
    assert set(kw) <= set(a)
    a.update(kw)
    return lib.pkv_prefill_check(*a.values())


SCALED = dict(ks=8 << 28, vs=9 << 28, block=16)


@pytest.mark.parametrize("scaled", [False, True])
@pytest.mark.parametrize("kw,status,msg", [
    (dict(), 0, ""), (dict(lse=None), 0, ""), (dict(T=0, q=None, k=None, v=None, out=None), 0, ""),
    (dict(qt=4100), 3, "q strides"), (dict(kt=1028), 3, "k strides"), (dict(vh=-128), 3, "v strides"),
    (dict(k=(2 << 28) + 2), 3, "16-byte"), (dict(q=(1 << 28) + 8), 3, "16-byte"),
    (dict(out=(4 << 28) + 4), 3, "16-byte"), (dict(out=1 << 28), 1, "output must not overlap"),
    (dict(lse=(4 << 28) + 4), 1, "lse must not overlap"), (dict(k=6 << 28), 1, "must not overlap"),
    (dict(vp=6 << 28), 1, "must not overlap"), (dict(Hq=24), 2, "G=3"), (dict(d=64), 2, "d=128"),
    (dict(P=1 << 28), 2, "32-bit slots"), (dict(dtype=4), 2, "dtype"), (dict(kp=None), 1, "k_pages"),
    (dict(out=(6 << 28) + 4096), 1, "overlap the cache"), (dict(lse=7 << 28), 1, "overlap the cache"),
    (dict(T=1 << 30, Hq=8, Hkv=1, qt=8, kt=8, vt=8), 1, "must not overlap")])
def test_prefill_check(lib, scaled, kw, status, msg):
    assert prefill(lib, **{**(SCALED if scaled else {}), **kw}) == status
    assert msg in lib.pkv_last_error_message().decode()


@pytest.mark.parametrize("kw,status,msg", [
    (dict(vs=None), 1, "k_scales and v_scales"), (dict(block=8), 2, "multiple of 16"),
    (dict(vs=8 << 28), 1, "must not overlap"), (dict(ks=(6 << 28) + 64), 1, "must not overlap"),
    (dict(lse=8 << 28), 1, "overlap the cache"),
    (dict(Hkv=1 << 18, Hq=1 << 18), 2, "too many heads")])
def test_prefill_check_of_block_scales(lib, kw, status, msg):
    assert prefill(lib, **{**SCALED, **kw}) == status
    assert msg in lib.pkv_last_error_message().decode()


# ------------------------------------------------------------------ native host step
def test_native_step_refuses_e4m3_caches(monkeypatch):
    """Its kernels would read an e4m3 pool as one of 16-bit values, past its end."""
    from persistentkv_attention_b200 import _native

    monkeypatch.setattr(_native, "load", lambda: pytest.fail("the library was reached"))
    with pytest.raises(RuntimeError, match="16-bit K/V caches"):
        NativeEngine(SimpleNamespace(kv8=True), 4, 8)
