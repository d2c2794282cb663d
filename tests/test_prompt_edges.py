"""Host-side behaviour of the prompt entry points and the block-scaled decode at
the edges of their contracts (no GPU, no kernel launch)."""

import pytest

from tests.test_prompt_abi import decode, write


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
