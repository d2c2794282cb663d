"""The prompt operators and the block-scaled cache where their contracts are
widest: block and page sizes, values that are not finite, scales far apart,
nothing to do."""

import numpy as np
import pytest
import torch

from oracle import prompt_oracle as pr
from persistentkv_attention_b200 import _native, ops
from persistentkv_attention_b200.serving import DecodeEngine, PageStack
from tests.test_prompt_gpu import (DT, check_block_write, check_close, check_decode, check_lse,
                                   check_prompt, decode_case, empty_cache, i32, no_error, packed,
                                   run_decode, run_prompt, run_slots, slots_of)

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


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_block_write_into_a_block_of_zeros(dtype):
    """A block of scale 0 is zeros whatever its codes; a token that joins it leaves
    the earlier ones zeros."""
    kp, ks = empty_cache(2, 1, 32, 32)      # codes that are all NaN
    vp, vs = empty_cache(2, 1, 32, 32)
    ks.zero_(), vs.zero_()
    x = torch.randn(3, 2, 128).to(DT[dtype]).cuda()
    ops.kv_write_fp8_block(x[:, :1], x[:, 1:], kp, vp, ks, vs, i32([5, 6, 32 + 31]))
    no_error()
    for t, (p, s) in enumerate(((kp, ks), (vp, vs))):
        got = pr.dequantised(p.view(torch.uint8).cpu().numpy(), s.cpu().numpy())[:, 0]
        assert (got[0, :5] == 0).all() and (got[1, :31] == 0).all()
        new = np.stack([got[0, 5], got[0, 6], got[1, 31]])
        want = x[:, t].double().cpu().numpy()
        # half a step of e4m3, or of its least value at a scale of at most 2^-6
        assert (np.abs(new - want) <= 2.0 ** -4 * np.abs(want) + 2.0 ** -16).all()


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


# ------------------------------------------------------------------ values that are not finite
def visible(row, cq, ck):
    """(first key, end of keys) that a packed query row sees."""
    b = int(np.searchsorted(cq, row, side="right")) - 1
    return ck[b], max(ck[b], ck[b] + row - cq[b] + 1 + (ck[b + 1] - ck[b]) - (cq[b + 1] - cq[b]))


def check_bad_values(lq, lk, hq, hkv, dtype, places, seed):
    """V holds `places` (sequence, key, dim, value), by KV head alike: an output is
    not finite where its row sees one, of the sign of those it sees, and every
    other output is that of V without them."""
    q, k, v, cq, ck = packed(lq, lk, hq, hkv, dtype, seed=seed, tail=3)
    bad = v.clone()
    v = v.clone()
    bad[ck[-1]:] = float("nan")
    for b, key, dim, value in places:
        bad[ck[b] + key, :, dim] = value
        v[ck[b] + key, :, dim] = 0.0
    got, ls = run_prompt(q, k, bad, cq, ck)
    want, lse, mag, size = pr.prompt_attention(q.double().numpy(), k.double().numpy(),
                                               v.double().numpy(), cq, ck)
    check_lse(ls, lse, size)
    g = got.double().cpu().numpy()
    for row in range(cq[-1]):
        lo, hi = visible(row, np.asarray(cq), np.asarray(ck))
        for dim in {d for _, _, d, _ in places}:
            seen = {x for b, key, d, x in places if d == dim and lo <= ck[b] + key < hi}
            if not seen:
                continue
            if len(seen) == 1 and seen <= {float("inf"), float("-inf")}:
                # (a weight that the type rounds to zero makes a NaN of it)
                ok = (g[row, :, dim] == seen.pop()) | np.isnan(g[row, :, dim])
            else:
                ok = np.isnan(g[row, :, dim])
            assert ok.all()
            want[row, :, dim] = np.nan
    check_close(got, want, np.nan_to_num(mag), size, 1e3, dtype)


INF, NAN = float("inf"), float("nan")


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("hq,hkv", [(4, 1), (2, 2)])
@pytest.mark.parametrize("lq,lk,places", [
    ([300], [300], [(0, 0, 3, NAN)]),
    ([300], [300], [(0, 0, 3, INF), (0, 130, 3, -INF), (0, 131, 9, INF), (0, 299, 0, NAN)]),
    ([300, 200], [300, 200], [(0, 255, 1, INF), (0, 256, 2, -INF), (1, 127, 127, NAN),
                              (1, 128, 64, INF), (1, 199, 65, -INF)]),
    ([1], [77], [(0, 76, 5, INF), (0, 3, 6, NAN)]),
    ([700, 9], [700, 140], [(0, 40 * i, 7 + i, INF) for i in range(17)] + [(1, 131, 0, NAN)]),
    ([100], [300], [(0, 201, 3, INF), (0, 250, 3, INF), (0, 220, 4, NAN)]),
    ([300], [40], [(0, 0, 1, INF), (0, 39, 2, NAN)]),
    ([640], [640], [(0, 511, 11, INF), (0, 512, 12, -INF), (0, 639, 13, INF)])])
def test_prompt_values_that_are_not_finite(lq, lk, places, hq, hkv, dtype):
    check_bad_values(lq, lk, hq, hkv, dtype, places, seed=sum(lq))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("hq,hkv", [(4, 1), (2, 2)])
@pytest.mark.parametrize("lq,lk,places", [
    ([6], [4500], [(0, 4495, 3, INF), (0, 4497, 3, -INF), (0, 4499, 4, NAN), (0, 100, 5, INF)]),
    ([300], [4400], [(0, 4100, 3, INF), (0, 4101, 9, INF), (0, 4352, 3, -INF), (0, 4399, 4, NAN)]),
    ([1], [4097], [(0, 4096, 0, INF), (0, 0, 1, -INF)]),
    ([130, 2], [2100, 2051], [(0, 2047, 2, INF), (0, 2099, 3, NAN), (1, 2050, 4, INF)])])
def test_prompt_split_values_that_are_not_finite(lq, lk, places, hq, hkv, dtype):
    """The same where a cluster's CTAs share the keys."""
    check_bad_values(lq, lk, hq, hkv, dtype, places, seed=sum(lk))


@pytest.mark.parametrize("hq,hkv", [(4, 1), (3, 3)])
def test_prompt_values_that_are_not_finite_among_many_items(hq, hkv):
    """Several items a CTA, some of whose tiles hold such values: they stay with
    their own rows."""
    lens = [(37 * i) % 290 + 1 for i in range(330)]
    places = [(b, (11 * b) % lens[b], b % 128, (INF, -INF, NAN)[b % 3])
              for b in range(0, 330, 3) if b % 4]
    check_bad_values(lens, lens, hq, hkv, "bf16", places, seed=3)


def test_prompt_values_that_are_not_finite_in_a_graph():
    """Replays over other values, and two calls at once, know nothing of one another."""
    lens = [150, 129, 400]
    q, k, v, cq, _ = packed(lens, lens, 4, 2, "f16", seed=8)
    dq, dk, dv, c = q.cuda(), k.cuda(), v.cuda(), i32(cq)
    want, _ = run_prompt(q, k, v, cq, None)
    bad = dv.clone()
    bad[cq[1] + 100, :, 7] = NAN
    out = torch.zeros_like(dq)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.prompt_attention(dq, dk, dv, c, None, out)
    clean = dv.clone()
    for values in (bad, clean, bad):
        dv.copy_(values)
        graph.replay()
        no_error()
        is_nan = torch.zeros_like(out, dtype=torch.bool)
        if values is bad:
            is_nan[cq[1] + 100:cq[2], :, 7] = True
        assert torch.equal(out.isnan(), is_nan) and torch.equal(out[~is_nan], want[~is_nan])
    outs = [torch.zeros_like(out) for _ in range(12)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for i, o in enumerate(outs):
        with torch.cuda.stream(streams[i % 2]):
            ops.prompt_attention(dq, dk, (bad, clean)[i % 2], c, None, o)
    no_error()
    for i, o in enumerate(outs):
        keep = ~is_nan if i % 2 == 0 else torch.ones_like(is_nan)
        assert torch.equal(o[keep], want[keep]) and (i % 2 or o.isnan().equal(is_nan))


@pytest.mark.parametrize("power", [-78, -60, 60, 100, 112])
def test_prompt_large_and_small_values(power):
    """Values of bf16's range pass through 32-bit sums of weights of at most 1 (3000
    values of 3 * 2^112: below 2^126): a common power of two of V is one of the
    output."""
    for lq, lk in (([300], [300]), ([5], [3000])):
        q, k, v, cq, ck = packed(lq, lk, 4, 2, "bf16", seed=power, spread=3.0)
        v = v.clamp(-3, 3)
        got, ls = run_prompt(q, k, (v.double() * 2.0 ** power).to(torch.bfloat16), cq, ck)
        back = (got.double() * 2.0 ** -power).to(torch.bfloat16)
        check_prompt(q, k, v, cq, ck, "bf16", back, ls)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_prompt_log_sums_are_exact_to_their_own_rounding(dtype):
    """Scores of no size: the log-sum of n keys is ln n, up to the rounding of one
    logarithm (2^-22 of it) and of sums of n ones."""
    for lq, lk in ((300, 300), (3, 5000)):
        q, k, v, cq, ck = packed([lq], [lk], 2, 1, dtype, seed=2)
        _, ls = run_prompt(q, torch.zeros_like(k), v, cq, ck)
        want = np.log(np.arange(lq) + 1.0 + lk - lq)[:, None]
        assert (np.abs(ls.double().cpu().numpy() - want) <= 2.0 ** -22 * (want + 2)).all()


def test_prompt_of_bad_values_takes_no_longer():
    """One NaN at the first key, or nothing but NaN: the tensor cores still do the
    work (a row computed on its own would take a hundred times as long)."""
    n, hq, hkv = 4096, 8, 2
    q, k, v, cq, _ = packed([n], [n], hq, hkv, "bf16", seed=1)
    q, k, v, c = q.cuda(), k.cuda(), v.cuda(), i32(cq)
    out = torch.empty_like(q)

    def took(values):
        times = []
        for _ in range(4):
            a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            a.record()
            ops.prompt_attention(q, k, values, c, None, out)
            b.record()
            b.synchronize()
            times.append(a.elapsed_time(b))
        return min(times)

    one, last, every = v.clone(), v.clone(), torch.full_like(v, NAN)
    one[0, :, 5] = NAN
    last[127::128] = INF
    usual = took(v)
    for values in (one, last, every):
        assert took(values) < 10 * usual
    no_error()


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
