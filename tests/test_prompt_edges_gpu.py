"""The prompt operators and the block-scaled cache where their contracts are
widest: block and page sizes, values that are not finite, scales far apart,
nothing to do."""

import numpy as np
import pytest
import torch

from persistentkv_attention_b200 import _native, ops
from persistentkv_attention_b200.serving import DecodeEngine, PageStack
from tests.test_prompt_gpu import (DT, check_block_write, check_decode, decode_case, empty_cache,
                                   i32, no_error, run_decode, run_slots, slots_of)

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _clean_error_word():
    _native.device_error(clear=True)
    yield


# ------------------------------------------------------------------ block and page sizes
def scale_blocks_apart(kp, ks, vp, vs):
    """Neighbouring blocks of a page at scales 8 times apart, K and V in turn."""
    factor = torch.tensor([1.0, 8.0], device="cuda").repeat(ks.shape[2])[:ks.shape[2]]
    return kp, ks * factor / 8, vp, vs * factor


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("page,block", [(96, 48), (160, 80), (288, 48), (288, 144), (224, 112),
                                        (192, 96), (48, 48), (80, 80), (96, 96), (64, 32)])
def test_decode_reads_every_token_at_its_blocks_scale(page, block, dtype):
    """Blocks that end inside a copy of 32 tokens, and ones that do not."""
    lens = [page, 2 * page + block + 5, 900, 33]
    q, *cache, table = decode_case(lens, 8, 2, page, block, dtype, seed=page + block)
    c = (q, *scale_blocks_apart(*cache), table)
    check_decode(run_decode(*c, lens), *c, lens, dtype)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("page,block", [(96, 48), (160, 80), (144, 144)])
def test_block_write_of_blocks_of_odd_multiples(page, block, dtype):
    """Whole prompts, then chunks that go on inside a block."""
    rows, hkv, steps = 3, 2, [70, 1, 33, 130, 2]
    total = sum(steps)
    all_slots, pool = slots_of([total] * rows, page, seed=block)
    all_slots = all_slots.reshape(rows, total)
    gen = torch.Generator().manual_seed(block)
    kp, ks = empty_cache(pool, hkv, page, block)
    vp, vs = empty_cache(pool, hkv, page, block)
    at = 0
    for i, n in enumerate(steps):
        x = torch.randn(rows * n, 2 * hkv, 128, generator=gen)
        x *= torch.exp(torch.randn(rows * n, 2 * hkv, 1, generator=gen)) * 4.0 ** ((2 * i) % 3 - 1)
        x = x.to(DT[dtype]).cuda()
        check_block_write(x[:, :hkv], x[:, hkv:], all_slots[:, at:at + n].reshape(-1), kp, vp, ks, vs)
        at += n


# ------------------------------------------------------------------ scales far apart
@pytest.mark.parametrize("fused", [True, False])
@pytest.mark.parametrize("far", [(100, None), (None, 100), (120, -24), (-24, 120), (90, -130, 3),
                                 (None, -140, None), (126, 0, None, -148, 60)])
def test_decode_v_scales_any_powers_of_two_apart(far, fused):
    """Blocks whose V scales are 2^a, 2^b, ... in turn (None: a block of zeros),
    beyond fp32's exponents apart, every token about as likely as the others: each
    counts in the sum.  Rows in one piece, in pieces of a few blocks, and blocks
    in runs, so that pieces and warps hold scales of one kind."""
    lens, page = [16 * 3 + 5, 16 * 40, 16 * 200 + 9, 7], 16
    for run in (1, 2, 25):
        q, kp, ks, vp, vs, table = decode_case(lens, 4, 1, page, 16, "bf16", seed=11, spread=0.0)
        codes = vp.view(torch.uint8)
        codes[(codes & 127) == 127] = 0      # (slots of no token)
        vs.fill_(1.0)
        for b, n in enumerate(lens):
            for j in range(-(-n // page)):
                power = far[(j // run) % len(far)]
                vs[table[b, j], 0, 0] = 0.0 if power is None else 2.0 ** power
        vs = vs.contiguous()
        got = run_decode(q, kp, ks, vp, vs, table, lens, fused=fused)
        check_decode(got, q, kp, ks, vp, vs, table, lens, "bf16")


def test_decode_v_scales_all_small_or_large():
    """A common power of two of all V scales is one of the output."""
    lens = [16 * 30 + 3, 9]
    q, kp, ks, vp, vs, table = decode_case(lens, 4, 2, 16, 16, "bf16", seed=12)
    for power in (-140, -100, -60, 60, 110):
        got = run_decode(q, kp, ks, vp, (vs.double() * 2.0 ** power).float(), table, lens)
        if power == -140:      # (scales and outputs near fp32's least)
            assert got.isfinite().all() and (got.double().abs() <= 2.0 ** -110).all()
            continue
        back = (got.double() * 2.0 ** -power).to(torch.bfloat16)
        check_decode(back, q, kp, ks, vp, vs, table, lens, "bf16")


# ------------------------------------------------------------------ nothing there
@pytest.mark.parametrize("in_place", [False, True])
def test_slots_of_an_empty_stack(in_place):
    """A free list of no pages serves no row that needs one, whatever the table
    holds; rows that need none go on."""
    cached, new = [0, 5, 16, 0], [3, 11, 1, 0]
    table = np.arange(4)[:, None] * np.ones((1, 3), np.int64)
    d, left, code = run_slots(cached, new, table, 16, 16, [], 0, in_place)
    assert code == 0x80 and left == 0
    assert d["s"].tolist() == [-1] * 3 + list(range(16 + 5, 32)) + [-1] * 2
    assert d["seq"].tolist() == [0, 16, 16, 0] and np.array_equal(d["t"].cpu().numpy(), table)
    # one that claims pages it cannot hold
    d, left, code = run_slots(cached, new, table, 16, 16, [], 7, in_place)
    assert code == 0x80 | 0x10 and left == 0 and (d["s"][:3] == -1).all()


def test_slots_of_a_full_stack_of_no_pages():
    stack = PageStack.full(0, "cuda")
    s, cu, seq, table = i32([5, 5]), i32([0, 0]), i32([9]), i32([[0]])
    ops.prompt_slots(i32([0]), i32([2]), table, s, cu, seq, stack.free_pages, stack.free_count,
                     stack.free_count, stack.counters, 16)
    torch.cuda.synchronize()
    assert _native.device_error(clear=True) == 0x80
    assert s.tolist() == [-1, -1] and seq.tolist() == [0] and stack.free_count.item() == 0


def test_append_to_an_empty_stack():
    """A token that opens a page finds none; one inside a page is written."""
    kp = torch.zeros(2, 1, 16, 128, dtype=torch.float16, device="cuda")
    vp, table = torch.zeros_like(kp), i32([[0, 0], [1, 0]])
    x = torch.ones(2, 1, 128, dtype=torch.float16, device="cuda")
    stack = PageStack.full(0, "cuda")
    ops.kv_append(x, x, kp, vp, table, i32([16, 3]), stack.free_pages, stack.free_count,
                  stack.counters)
    torch.cuda.synchronize()
    assert _native.device_error(clear=True) == 0x80
    assert not kp[0].any() and kp[1, 0, 3].all() and kp.sum() == 128 and torch.equal(kp, vp)
    assert stack.free_count.item() == 0 and stack.counters.item() == 0
    assert table.tolist() == [[0, 0], [1, 0]]


@pytest.mark.parametrize("cache", ["f16", "block"])
def test_no_tokens_and_no_rows(cache):
    """Writes of no tokens, a decode of no rows and a prefill of empty prompts do
    nothing."""
    f16 = torch.float16
    k, q = (torch.empty(0, h, 128, dtype=f16, device="cuda") for h in (2, 4))
    kp, ks = empty_cache(4, 2, 16, 16)
    vp, vs = empty_cache(4, 2, 16, 16)
    stack, table = PageStack.full(4, "cuda"), i32([[-1, -1]])
    if cache == "block":
        ops.kv_write_fp8_block(k, k, kp, vp, ks, vs, i32([]))
        ops.paged_attention_auto_fp8_block(q, kp, vp, ks, vs, i32(np.zeros((0, 2))), i32([]), q,
                                           torch.empty(0, device="cuda"))
        engine = DecodeEngine(kp, vp, 4, kv_block_scales=(ks, vs))
    else:
        kp, vp = (torch.full((4, 2, 16, 128), 7.0, dtype=f16, device="cuda") for _ in range(2))
        ops.kv_write(k, k, kp, vp, i32([]))
        engine = DecodeEngine(kp, vp, 4)
    seq = engine.prefill(q, k, k, i32([0]), table, q, stack)
    no_error()
    assert seq.tolist() == [0] and stack.free_count.item() == 4 and table.tolist() == [[-1, -1]]
    for t in (kp, vp):
        assert (t == 7).all() if cache == "f16" else (t.view(torch.uint8) == 255).all()


# ------------------------------------------------------------------ overlaps
def test_slots_from_parts_of_one_buffer():
    """Buffers that only touch, lengths that share their memory, and a stack
    lowered in place are fine."""
    buf = torch.zeros(200, dtype=torch.int32, device="cuda")
    lens, cu, seq, slots = buf[0:2], buf[2:5], buf[5:7], buf[7:27]
    table, free, count, ctr = buf[27:35].view(2, 4), buf[35:43], buf[43:44], buf[44:45]
    lens.copy_(i32([7, 3])), free.copy_(i32(range(8))), count.fill_(8), buf[45:].fill_(9)
    ops.prompt_slots(lens, lens, table, slots, cu, seq, free, count, count, ctr, 8)
    no_error()
    assert lens.tolist() == [7, 3] and cu.tolist() == [0, 7, 10] and seq.tolist() == [14, 6]
    assert slots.tolist() == [7] + [56 + i for i in range(6)] + [3, 4, 5] + [-1] * 10
    assert table.tolist() == [[0, 7, 0, 0], [0, 0, 0, 0]] and count.item() == 7
    assert free.tolist() == list(range(8)) and ctr.item() == 0 and (buf[45:] == 9).all()
    with pytest.raises(RuntimeError, match="must not overlap"):
        ops.prompt_slots(lens, lens, table, buf[8:28], cu, seq, free, count, count, ctr, 8)


# ------------------------------------------------------------------ prefill
@pytest.mark.parametrize("cache", ["f16", "block"])
def test_prefill_takes_no_pages_for_what_it_refuses(cache):
    """Strides, alignment, overlaps and scales that only the calls behind the slot
    map would refuse."""
    f16 = torch.float16
    if cache == "block":
        kp, ks = empty_cache(4, 2, 16, 16)
        vp, vs = empty_cache(4, 2, 16, 16)
        scales = dict(kv_block_scales=(ks, vs))
    else:
        kp, vp = (torch.zeros(4, 2, 16, 128, dtype=f16, device="cuda") for _ in range(2))
        scales = {}
    engine = DecodeEngine(kp, vp, 4, **scales)
    q, k, v = (torch.randn(20, h, 128, device="cuda").to(f16) for h in (4, 2, 2))
    out, lse = torch.zeros_like(q), torch.zeros(20, 4, device="cuda")
    flat = torch.zeros(1 << 16, dtype=f16, device="cuda")
    odd = flat.as_strided((20, 2, 128), (260, 128, 1))
    off = flat.as_strided((20, 2, 128), (256, 128, 1), 4)
    whole = kp.view(torch.uint8).view(-1).view(f16)      # the pool's memory
    stack, table, new = PageStack.full(4, "cuda"), i32([[-1, -1]]), i32([20])
    bad = [(engine, a) for a in (
        (q, odd, v, out, None), (q, k, off, out, None), (q, k, v, q, None), (q[:19], k, v, out[:19], None),
        (flat.as_strided((20, 4, 128), (516, 128, 1)), k, v, out, None),
        (q, k, v, out, out.view(-1)[:160].view(torch.float32).view(20, 4)),
        (q, whole[:5120].view(20, 2, 128), v, out, None),
        (q, k, v, whole[:8192].view(16, 4, 128), None),
        (q[:16], k[:16], v[:16], whole[:8192].view(16, 4, 128), None))]
    if cache == "block":
        for a, b in ((ks, ks), (ks, torch.zeros(4, 2, 2, device="cuda")), (ks.half(), vs.half()),
                     (ks[:3], vs[:3])):
            bad.append((DecodeEngine(kp, vp, 4, kv_block_scales=(a, b)), (q, k, v, out, None)))
    else:
        bad.append((DecodeEngine(kp, kp, 4), (q, k, v, out, None)))
        bad.append((DecodeEngine(kp, vp[:3], 4), (q, k, v, out, None)))
    kept = [t.view(torch.uint8).clone() for t in (kp, vp)]
    for eng, (a, b, c, o, l) in bad:
        with pytest.raises(RuntimeError):
            eng.prefill(a, b, c, new, table, o, stack, l)
        assert stack.free_count.item() == 4 and table.tolist() == [[-1, -1]]
    no_error()
    for t, was in zip((kp, vp), kept):
        assert torch.equal(t.view(torch.uint8), was)
    assert engine.prefill(q, k, v, new, table, out, stack, lse).tolist() == [20]
    no_error()
    assert stack.free_count.item() == 2 and table.tolist() == [[0, 1]]
