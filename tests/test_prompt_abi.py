"""Host-side refusals of the prompt entry points and the block-scaled decode
(no GPU, no kernel launch)."""

import pytest
import torch

from persistentkv_attention_b200 import _native, ops

FAKE = 0x10000  # never dereferenced: every call below fails validation first
FAKE2 = 0x20000


def slots(lib, **kw):
    a = dict(cached=FAKE, new=FAKE2, table=FAKE, slots=FAKE, cu=0x30000, seq=0x40000, free=FAKE,
             count=FAKE, left=FAKE, ctr=FAKE, B=4, maxp=8, page=16, n=64, cap=32, stream=None)
    a.update(kw)
    return lib.pkv_prompt_slots(*a.values())


@pytest.mark.parametrize("kw,status,msg", [
    (dict(cached=None), 1, "cached_lens"),
    (dict(table=None), 1, "block_table"),
    (dict(slots=None), 1, "slots must be"),
    (dict(count=None), 1, "free_count"),
    (dict(left=None), 1, "free_left"),
    (dict(ctr=None), 1, "zeroed counters"),
    (dict(seq=FAKE), 1, "must not be the tensors"),
    (dict(seq=FAKE2), 1, "must not be the tensors"),
    (dict(cu=FAKE), 1, "must not be the tensors"),
    (dict(page=0), 1, "invalid slot map shape"),
    (dict(B=-1), 1, "invalid slot map shape"),
    (dict(maxp=1 << 27), 2, "32-bit positions"),
    (dict(maxp=178956970, page=12), 2, "32-bit positions"),  # 2^31 - 8: rounded up, too many
])
def test_slots_validation(lib, kw, status, msg):
    assert slots(lib, **kw) == status
    assert msg in lib.pkv_last_error_message().decode()


def write(lib, fp8=False, **kw):
    a = dict(k=FAKE, v=FAKE, kp=FAKE, vp=FAKE)
    if fp8:
        a.update(ks=FAKE, vs=FAKE)
    a.update(slots=FAKE, T=4, Hkv=8, d=128, kt=1024, kh=128, vt=1024, vh=128, P=64, page=16)
    if fp8:
        a.update(block=16)
    a.update(dtype=0, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return (lib.pkv_kv_write_fp8_block if fp8 else lib.pkv_kv_write)(*a.values())


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("kw,status,msg", [
    (dict(k=None), 1, "k and v"),
    (dict(vp=None), 1, "k_pages and v_pages"),
    (dict(slots=None), 1, "slots"),
    (dict(dtype=5), 2, "wrong dtype"),
    (dict(d=64), 2, "d=128"),
    (dict(T=-1), 1, "invalid write shape"),
    (dict(P=1 << 28), 2, "32-bit slots"),
    (dict(kt=1028), 3, "k strides"),
    (dict(vh=-128), 3, "v strides"),
    (dict(k=FAKE + 2), 3, "16-byte aligned"),
])
def test_write_validation(lib, fp8, kw, status, msg):
    assert write(lib, fp8, **kw) == status
    assert msg in lib.pkv_last_error_message().decode()


@pytest.mark.parametrize("kw,status,msg", [
    (dict(ks=None), 1, "k_scales"),
    (dict(block=8), 2, "multiple of 16"),
    (dict(block=0), 2, "multiple of 16"),
    (dict(block=32), 2, "divides the page"),
    (dict(page=48, block=32), 2, "divides the page"),
])
def test_block_write_validation(lib, kw, status, msg):
    assert write(lib, True, **kw) == status
    assert msg in lib.pkv_last_error_message().decode()


def prompt(lib, **kw):
    a = dict(q=FAKE, k=FAKE, v=FAKE, cq=FAKE, ck=FAKE, out=FAKE, lse=None, B=2, Tq=40, Tk=40,
             Hq=32, Hkv=8, d=128, qt=4096, qh=128, kt=1024, kh=128, vt=1024, vh=128, dtype=0,
             stream=None)
    a.update(kw)
    return lib.pkv_prompt_attention(*a.values())


@pytest.mark.parametrize("kw,status,msg", [
    (dict(q=None), 1, "q and output"),
    (dict(v=None), 1, "k and v"),
    (dict(cq=None), 1, "cu_seqlens_q"),
    (dict(dtype=2), 2, "wrong dtype"),
    (dict(d=96), 2, "d=128"),
    (dict(Hkv=0), 1, "Hkv must be positive"),
    (dict(Hq=30), 1, "divisible"),
    (dict(Hq=24), 2, "G=3"),
    (dict(B=-1), 1, "invalid prompt shape"),
    (dict(Tk=-1), 1, "invalid prompt shape"),
    (dict(qt=4100), 3, "q strides"),
    (dict(kh=-128), 3, "k strides"),
    (dict(out=FAKE + 8), 3, "16-byte aligned"),
])
def test_prompt_validation(lib, kw, status, msg):
    assert prompt(lib, **kw) == status
    assert msg in lib.pkv_last_error_message().decode()


@pytest.mark.parametrize("kw", [
    dict(), dict(vp=FAKE + (1 << 20), k=FAKE2), dict(kp=FAKE2, vp=FAKE + 4096),
    dict(kp=FAKE - 4096, vp=FAKE2 + (1 << 24))])
@pytest.mark.parametrize("fp8", [False, True])
def test_write_refuses_overlaps(lib, fp8, kw):
    # pools of 2 MB (1 MB of e4m3), tokens of 8 KB at FAKE
    assert write(lib, fp8, **kw) == 1
    assert b"overlap" in lib.pkv_last_error_message()


@pytest.mark.parametrize("kw", [
    dict(), dict(q=FAKE - 16, k=1 << 30, v=1 << 30), dict(q=1 << 30, k=FAKE + 1024, v=1 << 30),
    dict(q=1 << 30, k=1 << 30, out=1 << 24, v=(1 << 24) - 80 * 1024 + 16)])
def test_prompt_refuses_overlaps(lib, kw):
    assert prompt(lib, **kw) == 1
    assert b"output must not overlap" in lib.pkv_last_error_message()


@pytest.mark.parametrize("lse", [1 << 24, (1 << 30) + 40 * 8192 - 16, (1 << 31) - 16, 1 << 32])
def test_prompt_refuses_an_lse_in_its_operands(lib, lse):
    kw = dict(out=1 << 24, q=1 << 30, k=1 << 31, v=1 << 32, lse=lse)
    assert prompt(lib, **kw) == 1
    assert b"lse must not overlap" in lib.pkv_last_error_message()


@pytest.mark.parametrize("ks,vs,msg", [
    (1 << 34, (1 << 34) + 2044, b"k_scales and v_scales"),  # 64 pages x 8 heads: 2 KB
    (1 << 30, 1 << 34, b"the scales"), (1 << 34, (1 << 31) - 4, b"the scales"),
    ((1 << 32) + 8000, 1 << 34, b"the scales"), (1 << 34, (1 << 33) - 4, b"the scales")])
def test_block_write_refuses_scales_in_its_operands(lib, ks, vs, msg):
    kw = dict(kp=1 << 30, vp=1 << 31, k=1 << 32, v=1 << 33, ks=ks, vs=vs)
    assert write(lib, True, **kw) == 1
    assert msg in lib.pkv_last_error_message()


def test_nothing_to_do_is_no_error(lib):
    assert prompt(lib, B=0) == 0
    assert prompt(lib, q=None, out=None, Tq=0) == 0
    assert write(lib, T=0) == 0
    assert write(lib, True, T=0) == 0


def decode(lib, **kw):
    a = dict(q=FAKE, k=FAKE, v=FAKE, ks=FAKE, vs=FAKE, bt=FAKE, sl=FAKE, qi=None, oi=None,
             out=FAKE, ws=FAKE, wsb=1 << 30, ctr=None, B=1, qr=1, orow=1, Hq=32, Hkv=8, d=128,
             P=64, page=16, maxp=8, block=16, dtype=0, stream=None)
    a.update(kw)
    return lib.pkv_paged_attention_auto_fp8_block(*a.values())


@pytest.mark.parametrize("kw,status,msg", [
    (dict(ks=None), 1, "k_scales and v_scales"),
    (dict(block=8), 2, "multiple of 16"),
    (dict(page=8, block=8), 2, "multiple of 16"),
    (dict(block=32), 2, "divides the page"),
    (dict(out=None), 1, "output"),
    (dict(page=0), 1, "page_size"),
    (dict(d=64), 2, "d=128"),
    (dict(Hq=24), 2, "G=3"),
    (dict(dtype=3), 2, "wrong dtype"),
    (dict(sl=None), 1, "seq_lens"),
    (dict(k=FAKE + 8), 3, "16-byte aligned"),
])
def test_block_decode_validation(lib, kw, status, msg):
    assert decode(lib, **kw) == status
    assert msg in lib.pkv_last_error_message().decode()


def test_torch_surface_refuses_host_tensors():
    i = torch.zeros(1, dtype=torch.int32)
    x = torch.zeros(1, 8, 128, dtype=torch.float16)
    pool = torch.zeros(4, 8, 16, 128, dtype=torch.float16)
    pool8 = pool.to(torch.float8_e4m3fn)
    sc = torch.ones(4, 8, 1)
    with pytest.raises(RuntimeError, match="cached_lens must be a CUDA tensor"):
        ops.prompt_slots(i, i, i[None], i, i, i, i, i, i, i, 16)
    with pytest.raises(RuntimeError, match="k must be a CUDA tensor"):
        ops.kv_write(x, x, pool, pool, i)
    with pytest.raises(RuntimeError, match="k must be a CUDA tensor"):
        ops.kv_write_fp8_block(x, x, pool8, pool8, sc, sc, i)
    with pytest.raises(RuntimeError, match="q must be a CUDA tensor"):
        ops.prompt_attention(x, x, x, i, None, x)
    with pytest.raises(RuntimeError, match="q_source must be a CUDA tensor"):
        ops.paged_attention_auto_fp8_block(x, pool8, pool8, sc, sc, i[None], i, x, sc)


class _Fake:
    """A tensor's face, for checks that come before any use of its memory."""

    is_cuda = True

    def __init__(self, *shape, dtype=torch.float16, device=0, stride=None):
        self.t = torch.empty(*shape, dtype=dtype, device="meta")
        if stride is not None:
            self.t = torch.empty_strided(shape, stride, dtype=dtype, device="meta")
        self.device_index = device

    def __getattr__(self, name):
        return getattr(self.t, name)

    def get_device(self):
        return self.device_index

    def data_ptr(self):
        return FAKE


def test_torch_surface_refuses_shapes_and_devices(monkeypatch):
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    F, I = _Fake, lambda *s, **kw: _Fake(*s, dtype=torch.int32, **kw)  # noqa: E741
    q, kv = F(5, 8, 128), F(5, 4, 128)

    def prompt_call(q=q, k=kv, v=kv, cq=I(3), ck=None, out=F(5, 8, 128), lse=None):
        return lambda: ops.prompt_attention(q, k, v, cq, ck, out, lse)

    f8 = lambda *s: _Fake(*s, dtype=torch.float8_e4m3fn)  # noqa: E731
    f32 = lambda *s: _Fake(*s, dtype=torch.float32)  # noqa: E731
    pool = f8(4, 4, 32, 128)

    def write8(k=kv, v=kv, pool=pool, ks=f32(4, 4, 2), vs=f32(4, 4, 2), slots=I(5)):
        return lambda: ops.kv_write_fp8_block(k, v, pool, pool, ks, vs, slots)

    def decode8(q=F(2, 8, 128), ks=f32(4, 4, 2), bt=I(2, 3), sl=I(2), out=F(2, 8, 128), ws=f32(9),
                qi=None, ctr=None):
        return lambda: ops.paged_attention_auto_fp8_block(q, pool, pool, ks, ks, bt, sl, out, ws,
                                                          qi, None, ctr)

    for call, msg in [
        (prompt_call(q=F(5, 8, 128, dtype=torch.float32)), "q has wrong dtype"),
        (prompt_call(k=F(5, 4, 128, dtype=torch.bfloat16)), "k has wrong dtype"),
        (prompt_call(q=F(5, 8, 64)), "d=128"),
        (prompt_call(q=F(5, 8, 128, stride=(2048, 256, 2))), "contiguous in its last"),
        (prompt_call(v=F(6, 4, 128)), "v shape must match k"),
        (prompt_call(out=F(4, 8, 128)), "output shape must match q"),
        (prompt_call(ck=I(4)), "cu_seqlens_k batch"),
        (prompt_call(cq=I(0)), r"B \+ 1"),
        (prompt_call(lse=f32(8, 5)), "lse must have shape"),
        (prompt_call(k=F(5, 3, 128), v=F(5, 3, 128)), "divisible"),
        (prompt_call(k=F(5, 4, 128, device=1)), "current device"),
        (write8(slots=I(4)), "one value per token"),
        (write8(ks=f32(4, 4, 4), vs=f32(4, 4, 4)), "multiple of 16"),
        (write8(ks=f32(4, 2, 2)), "k_scales / v_scales shape"),
        (write8(k=F(5, 8, 128), v=F(5, 8, 128)), "matching the pools"),
        (write8(slots=I(5, device=1)), "current device"),
        (decode8(sl=I(3)), "seq_lens batch"),
        (decode8(q=F(1, 8, 128)), "a row per block_table row"),
        (decode8(out=F(1, 8, 128)), "a row per block_table row"),
        (decode8(qi=I(3)), "q_indices batch"),
        (decode8(ctr=I(2, 3)), "merge_counters shape"),
        (decode8(ks=f32(4, 4, 0)), "multiple of 16"),
        (decode8(ws=_Fake(9, dtype=torch.float32, device=1)), "current device"),
        (lambda: ops.prompt_slots(I(2), I(2), I(2, 3), I(9), I(2), I(2), None, None, None, None,
                                  16), r"B \+ 1"),
        (lambda: ops.prompt_slots(I(2), I(3), I(2, 3), I(9), I(3), I(2), None, None, None, None,
                                  16), "batch mismatch"),
        (lambda: ops.prompt_slots(I(2), I(2), I(2, 3), I(9), I(3), I(2), I(4), I(1), None, None,
                                  16), "free_left"),
        (lambda: ops.prompt_slots(I(2), I(2), I(2, 3), I(9), I(3), I(2), I(4), I(1), I(0), I(1),
                                  16), "must hold one value"),
        (lambda: ops.kv_write(kv, kv, F(4, 4, 16, 128, dtype=torch.bfloat16),
                              F(4, 4, 16, 128, dtype=torch.bfloat16), I(5)), "k_pages has wrong"),
    ]:
        with pytest.raises(RuntimeError, match=msg):
            call()
    assert issubclass(_native.PkvError, RuntimeError)
