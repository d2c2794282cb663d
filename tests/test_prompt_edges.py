"""Host-side behaviour of the prompt entry points and the block-scaled decode at
the edges of their contracts (no GPU, no kernel launch)."""

import pytest

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
