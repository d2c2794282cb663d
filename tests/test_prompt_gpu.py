"""The prompt operators and the block-scaled e4m3 cache on the GPU, against the
64-bit oracle.

Error bounds.  u is half a step of the output type (bf16 2^-8, fp16 2^-11), A
the weighted sum of |v| of a row.  A weight is rounded to 16 bits once (u of
its type, and 2^-25 absolute where fp16 leaves its normal range; the weights
sum to at least 1 before the division, so A_abs = sum |v| 2^-25 bounds it).  A
score is a sum of 128 products in 32 bits: off by at most 130 * 2^-24 of its
sum of |q k|, which moves every weight by that factor twice (numerator and
denominator).  exp2 and the running rescales stay below 2^-18 of a weight.
"""

import numpy as np
import pytest
import torch

from oracle import prompt_oracle as pr
from persistentkv_attention_b200 import _native, ops
from persistentkv_attention_b200.serving import DecodeEngine, PageStack

pytestmark = pytest.mark.gpu

DT = {"f16": torch.float16, "bf16": torch.bfloat16}
U = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}


@pytest.fixture(autouse=True)
def _clean_error_word():
    _native.device_error(clear=True)
    yield


def i32(x):
    return torch.as_tensor(np.asarray(x, np.int32), device="cuda")


def no_error():
    torch.cuda.synchronize()
    code = _native.device_error(clear=True)
    assert code == 0, _native.describe_device_error(code)


def check_close(got, want, mag, size, v_abs, dtype, p_dtype=None):
    """got within the bound above of want, wherever want is a number."""
    real = ~np.isnan(want)
    g = got.double().cpu().numpy()
    u, up = U[dtype], U[p_dtype or dtype]
    move = np.exp(2 * 130 * 2.0 ** -24 * size) - 1 + 2.0 ** -18
    tol = u * np.abs(want) + (up + move[..., None]) * mag + 2.0 ** -25 * (v_abs + 1)
    assert np.isfinite(tol[real]).all()
    # a value that may round beyond the type's largest may be the infinity of
    # its sign, and one that must is
    top = torch.finfo(got.dtype).max
    inf = np.isinf(g) & (np.sign(g) == np.sign(want)) & (np.abs(want) + tol > top)
    assert (inf | (np.abs(want) - tol <= top * (1 + u)))[real].all()
    real &= ~inf
    assert np.isfinite(g[real]).all()
    worst = np.max((np.abs(g - want) / tol)[real], initial=0.0)
    assert worst <= 1.0, f"off by {worst:.2f} of the bound"


def check_lse(got, want, size):
    g = got.double().cpu().numpy()
    real = ~np.isnan(want)
    empty = np.isneginf(want)
    assert np.isneginf(g[real & empty]).all()
    there = real & ~empty
    want = np.where(there, want, 0.0)
    tol = 130 * 2.0 ** -24 * size + 2.0 ** -18 + 2.0 ** -22 * np.abs(want)
    assert (np.abs(np.where(there, g, 0.0) - want) <= tol).all()


# ------------------------------------------------------------------ attention
def packed(lq, lk, hq, hkv, dtype, seed, tail=0, spread=1.0):
    gen = torch.Generator().manual_seed(seed)
    r = lambda n, h, s=1.0: (torch.randn(n, h, 128, generator=gen) * s).to(DT[dtype])  # noqa: E731
    cq, ck = np.cumsum([0] + lq), np.cumsum([0] + lk)
    return r(cq[-1] + tail, hq), r(ck[-1] + tail, hkv, spread), r(ck[-1] + tail, hkv), cq, ck


def run_prompt(q, k, v, cq, ck, lse=True):
    dev = [t.cuda() if not t.is_cuda else t for t in (q, k, v)]
    out = torch.full(q.shape, 7.0, dtype=q.dtype, device="cuda")
    ls = torch.full(q.shape[:2], 7.0, device="cuda") if lse else None
    ops.prompt_attention(*dev, i32(cq), None if ck is None else i32(ck), out, lse=ls)
    no_error()
    return out, ls


def check_prompt(q, k, v, cq, ck, dtype, out, ls):
    want, lse, mag, size = pr.prompt_attention(q.double().numpy(), k.double().numpy(),
                                               v.double().numpy(), cq, ck)
    rows = ~np.isnan(lse)
    v_abs = np.nansum(np.abs(v.double().numpy()))  # over all keys: an upper bound
    check_close(out, want, mag, size, min(v_abs, 1e3), dtype)
    check_lse(ls, lse, size)
    # rows of no sequence are left as they were
    assert (out.double().cpu().numpy()[~rows] == 7.0).all()
    assert (ls.cpu().numpy()[~rows] == 7.0).all()


LENGTHS = [
    ([1], [1]), ([17], [17]), ([64, 64], [64, 64]), ([127, 1, 128], [127, 1, 128]),
    ([129], [129]), ([256, 0, 3], [256, 0, 3]), ([300, 511], [300, 511]),
    ([5, 130], [400, 131]), ([1, 1, 1], [1, 200, 129]),
    ([200, 40], [70, 0]), ([0, 0], [0, 3]), ([260], [1]), ([640], [640]),
]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("lq,lk", LENGTHS)
def test_prompt_lengths(lq, lk, dtype):
    q, k, v, cq, ck = packed(lq, lk, 4, 2, dtype, seed=len(lq) + sum(lq), tail=3)
    check_prompt(q, k, v, cq, ck, dtype, *run_prompt(q, k, v, cq, ck))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("hq,hkv", [(1, 1), (3, 3), (2, 1), (6, 3), (4, 1), (8, 2), (8, 1), (16, 2)])
def test_prompt_heads(hq, hkv, dtype):
    q, k, v, cq, ck = packed([150, 33], [170, 33], hq, hkv, dtype, seed=hq)
    check_prompt(q, k, v, cq, ck, dtype, *run_prompt(q, k, v, cq, ck))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("lq,lk,hq,hkv", [
    ([1], [600], 2, 1), ([3], [4000], 2, 1), ([1], [2049], 2, 2), ([130], [3000], 4, 2),
    ([257], [2300], 3, 3), ([200, 7], [70, 5000], 2, 1), ([16, 16], [2048, 2048], 8, 1),
    ([700], [1100], 2, 2), ([300], [2200], 1, 1),
    ([2], [4500], 2, 1), ([9], [4097], 1, 1)])
def test_prompt_few_rows_many_keys(lq, lk, hq, hkv, dtype):
    """Key blocks shared by the CTAs of a cluster, some of which get none."""
    q, k, v, cq, ck = packed(lq, lk, hq, hkv, dtype, seed=sum(lk), tail=2)
    check_prompt(q, k, v, cq, ck, dtype, *run_prompt(q, k, v, cq, ck))
    a, _ = run_prompt(q, k, v, cq, ck, lse=False)
    b, _ = run_prompt(q, k, v, cq, ck)
    assert torch.equal(a, b)


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_prompt_few_rows_ignore_what_they_do_not_see(bad):
    lq, lk = [40, 20], [1500, 1500]
    q, k, v, cq, ck = packed(lq, lk, 2, 1, "bf16", seed=3, tail=9)
    want, _ = run_prompt(q, k, v, cq, ck)
    k2, v2 = k.clone(), v.clone()
    for t in (k2, v2):
        t[ck[2]:] = bad
        t[ck[2] - 5:ck[2]] = bad       # the last keys: rows before them do not see them
    got, _ = run_prompt(q, k2, v2, cq, ck)
    seen = list(range(55))
    _, _, mag, size = pr.prompt_attention(q.double().numpy(), k.double().numpy(),
                                          v.double().numpy(), cq, ck)
    w = np.full(want.shape, np.nan)
    w[seen] = want.double().cpu().numpy()[seen]
    check_close(got, w, 2 * np.nan_to_num(mag), size, 1e3, "bf16")
    assert not torch.isfinite(got[55:60].float()).all(-1).any()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_prompt_many_short_sequences(dtype):
    lens = [(7 * i) % 23 for i in range(300)]
    q, k, v, cq, ck = packed(lens, lens, 2, 2, dtype, seed=4, tail=1)
    out, ls = run_prompt(q, k, v, cq, None)   # keys as the queries
    check_prompt(q, k, v, cq, cq, dtype, out, ls)


def test_prompt_thousands_of_sequences():
    """Many more items than CTAs, most of the grid without a tile of its own."""
    lens = [1 + (i % 3) for i in range(4000)] + [0] * 90 + [150]
    q, k, v, cq, ck = packed(lens, lens, 4, 4, "f16", seed=5)
    check_prompt(q, k, v, cq, ck, "f16", *run_prompt(q, k, v, cq, ck))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_prompt_large_scores(dtype):
    """Scores of hundreds: the running maximum moves far, later and earlier."""
    q, k, v, cq, ck = packed([300], [420], 2, 1, dtype, seed=8, spread=12.0)
    check_prompt(q, k, v, cq, ck, dtype, *run_prompt(q, k, v, cq, ck))
    k = k.flip(0).contiguous() * torch.linspace(0.05, 2.0, 420)[:, None, None].to(k.dtype)
    check_prompt(q, k, v, cq, ck, dtype, *run_prompt(q, k, v, cq, ck))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_prompt_ignores_what_it_does_not_see(dtype, bad):
    """Keys and values of other sequences, of later positions and behind the
    last sequence do not reach a row, whatever they hold."""
    lens = [140, 77, 200]
    q, k, v, cq, ck = packed(lens, lens, 4, 2, dtype, seed=11, tail=40)
    want, ls0 = run_prompt(q, k, v, cq, ck)
    k2, v2 = k.clone(), v.clone()
    for t in (k2, v2):
        t[ck[1]:ck[2]] = bad                # the middle sequence
        t[ck[2] + 60:ck[2] + 64] = bad      # some later positions of the last one
        t[ck[3]:] = bad                     # behind it
    q2 = q.clone()
    q2[cq[3]:] = bad
    got, ls = run_prompt(q2, k2, v2, cq, ck)
    seen = list(range(cq[1])) + list(range(cq[2], cq[2] + 60))
    # a row that is told apart by what it must not see is computed another
    # way, so it agrees within the bound, not bit for bit
    _, _, mag, size = pr.prompt_attention(q.double().numpy(), k.double().numpy(),
                                          v.double().numpy(), cq, ck)
    w = np.full(want.shape, np.nan)
    w[seen] = want.double().cpu().numpy()[seen]
    check_close(got, w, 2 * np.nan_to_num(mag), size, 1e3, dtype)
    assert (got[cq[3]:] == 7.0).all()
    torch.testing.assert_close(ls[seen], ls0[seen], rtol=1e-5, atol=1e-5)
    # rows that see them say so
    assert not torch.isfinite(got[cq[2] + 64:cq[3]].float()).all(-1).any()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("hkv", [1, 4])
def test_prompt_split_keys_pass_nan_on(dtype, hkv):
    """Rows whose keys are split among CTAs: a NaN that a row sees reaches it,
    one in a part of its own, in one key or in the query."""
    lq, lk = 6, 4500
    q, k, v, cq, ck = packed([lq], [lk], 4, hkv, dtype, seed=21)
    nan = float("nan")
    want, lse = run_prompt(q, k, v, cq, ck)
    assert want.isfinite().all()
    for lo, hi in ((0, 2000), (777, 778), (4000, 4494), (0, lk)):
        k2 = k.clone()
        k2[lo:hi, 0] = nan
        got, ls = run_prompt(q, k2, v, cq, ck)
        g = 4 // hkv  # the heads that read KV head 0
        assert got[:, :g].isnan().all() and ls[:, :g].isnan().all()
        assert torch.equal(got[:, g:], want[:, g:]) and torch.equal(ls[:, g:], lse[:, g:])
    q2 = q.clone()
    q2[2] = nan
    got, ls = run_prompt(q2, k, v, cq, ck)
    rest = [0, 1, 3, 4, 5]
    assert got[2].isnan().all() and ls[2].isnan().all()
    assert torch.equal(got[rest], want[rest]) and torch.equal(ls[rest], lse[rest])
    # the keys of the last position, which only the last row sees
    k2, v2 = k.clone(), v.clone()
    k2[-1] = v2[-1] = nan
    got, ls = run_prompt(q, k2, v2, cq, ck)
    assert got[-1].isnan().all() and ls[-1].isnan().all()
    w = np.full(want.shape, np.nan)
    w[:-1] = want.double().cpu().numpy()[:-1]
    _, _, mag, size = pr.prompt_attention(q.double().numpy(), k.double().numpy(),
                                          v.double().numpy(), cq, ck)
    check_close(got, w, 2 * mag, size, 1e3, dtype)


def test_prompt_split_keys_in_a_graph():
    """The split is chosen by shapes; a replay follows the lengths on the device,
    down to none."""
    q, k, v, cq, ck = packed([6], [4500], 4, 1, "bf16", seed=31)
    dev = [t.cuda() for t in (q, k, v)]
    c, d, out = i32([0, 6]), i32([0, 4500]), torch.zeros_like(dev[0])
    ls = torch.zeros(6, 4, device="cuda")
    ops.prompt_attention(*dev, c, d, out, lse=ls)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.prompt_attention(*dev, c, d, out, lse=ls)
    for cq, ck in (([0, 6], [0, 4500]), ([1, 4], [100, 130]), ([0, 6], [7, 7]), ([2, 2], [0, 4500]),
                   ([0, 5], [0, 4499]), ([0, 6], [4490, 4500])):
        c.copy_(i32(cq)), d.copy_(i32(ck))
        out.fill_(7.0), ls.fill_(7.0)
        graph.replay()
        no_error()
        check_prompt(q, k, v, cq, ck, "bf16", out, ls)
    # two at once, on two streams
    c.copy_(i32([0, 6])), d.copy_(i32([0, 4500]))
    want = out.clone()
    ops.prompt_attention(*dev, c, d, want)
    outs = [torch.zeros_like(out) for _ in range(8)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for i, o in enumerate(outs):
        with torch.cuda.stream(streams[i % 2]):
            ops.prompt_attention(*dev, c, d, o)
    no_error()
    assert all(torch.equal(o, want) for o in outs)


def test_prompt_strided_operands():
    """Slices of one fused projection: token strides beyond heads * 128, and
    head-major storage."""
    gen = torch.Generator().manual_seed(3)
    fused = torch.randn(210, (8 + 2 + 2) * 128, generator=gen).half().cuda()
    q = fused[:, :1024].view(210, 8, 128)
    k = fused[:, 1024:1280].view(210, 2, 128)
    v = fused[:, 1280:].view(210, 2, 128)
    out, ls = run_prompt(q, k, v, [0, 90, 210], None)
    want, ls2 = run_prompt(q.contiguous(), k.contiguous(), v.contiguous(), [0, 90, 210], None)
    assert torch.equal(out, want) and torch.equal(ls, ls2)
    by_head = k.permute(1, 0, 2).contiguous().permute(1, 0, 2)
    got, _ = run_prompt(q, by_head, v, [0, 90, 210], None)
    assert torch.equal(got, want)
    # one key, and strides that no operand of its size has
    one = torch.randn(1, 2, 128).half().cuda()
    odd = one.as_strided((1, 2, 128), (12, 128, 1))
    q1 = torch.randn(1, 8, 128).half().cuda()
    a, _ = run_prompt(q1, odd, one, [0, 1], None)
    b, _ = run_prompt(q1, one, one, [0, 1], None)
    assert torch.equal(a, b)


def test_prompt_without_lse_and_repeated():
    q, k, v, cq, ck = packed([333], [333], 8, 2, "bf16", seed=5)
    a, _ = run_prompt(q, k, v, cq, ck)
    b, _ = run_prompt(q, k, v, cq, ck, lse=False)
    assert torch.equal(a, b)


def test_prompt_refuses_bad_ranges_on_the_device():
    q, k, v, cq, ck = packed([40, 30], [40, 30], 2, 1, "f16", seed=5)
    dev = [t.cuda() for t in (q, k, v)]
    for bq, bk in (([0, 40, 71], [0, 40, 70]), ([0, 40, 70], [0, 40, 71]),
                   ([0, 40, 70], [0, 40, 30]), ([0, 40, 20], [0, 40, 70]),
                   ([0, 40, 70], [0, -1, 70])):
        out = torch.full(q.shape, 7.0, dtype=q.dtype, device="cuda")
        ops.prompt_attention(*dev, i32(bq), i32(bk), out)
        torch.cuda.synchronize()
        assert _native.device_error(clear=True) == 0x10
        if bk[1] >= 0:
            assert (out[40:] == 7.0).all()


def test_prompt_on_another_stream_and_in_a_graph():
    q, k, v, cq, ck = packed([190, 65], [190, 65], 4, 2, "bf16", seed=6)
    want, _ = run_prompt(q, k, v, cq, ck)
    dq, dk, dv, c = q.cuda(), k.cuda(), v.cuda(), i32(cq)
    out = torch.zeros_like(dq)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.prompt_attention(dq, dk, dv, c, None, out)
    side.synchronize()
    assert torch.equal(out, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.prompt_attention(dq, dk, dv, c, None, out)
    for seed in (1, 2):
        q2, k2, v2, _, _ = packed([190, 65], [190, 65], 4, 2, "bf16", seed=seed)
        dq.copy_(q2), dk.copy_(k2), dv.copy_(v2)
        graph.replay()
        torch.cuda.synchronize()
        again, _ = run_prompt(q2, k2, v2, cq, ck)
        assert torch.equal(out, again)
    # the lengths live on the device: a replay follows them
    c.copy_(i32([0, 100, 255]))
    graph.replay()
    torch.cuda.synchronize()
    again, _ = run_prompt(q2, k2, v2, [0, 100, 255], None)
    assert torch.equal(out, again)


# ------------------------------------------------------------------ slots
def run_slots(cached, new, table, num_slots, page, free, count, in_place=False):
    d = dict(t=i32(table), s=torch.full((num_slots,), 5, dtype=torch.int32, device="cuda"),
             cu=i32(np.zeros(len(cached) + 1)), seq=i32(np.zeros(len(cached))), ctr=i32([0]))
    fp = None if free is None else i32(free)
    fc = None if free is None else i32([count])
    left = None if free is None else (fc if in_place else i32([0]))
    ops.prompt_slots(i32(cached), i32(new), d["t"], d["s"], d["cu"], d["seq"], fp, fc, left,
                     None if free is None else d["ctr"], page)
    torch.cuda.synchronize()
    code = _native.device_error(clear=True)
    assert d["ctr"].item() == 0
    if free is not None and not in_place:
        assert fc.item() == count
    return d, (None if free is None else left.item()), code


def slots_case(b, page, cached_hi, new_hi, seed, spare=0):
    gen = np.random.default_rng(seed)
    cached = gen.integers(0, cached_hi + 1, b)
    new = gen.integers(0, new_hi + 1, b)
    width = max(1, -(-int((cached + new).max(initial=1)) // page)) + 1
    pool = b * width + 50
    perm = gen.permutation(pool)
    table = perm[:b * width].reshape(b, width)
    need = sum(-(-(c + n) // page) - -(-c // page) for c, n in zip(cached, new))
    return cached, new, table, perm[::-1][:max(1, need + spare)], need


@pytest.mark.parametrize("b,page,cached_hi,new_hi", [
    (1, 16, 0, 1), (1, 16, 40, 3000), (8, 16, 100, 50), (5, 8, 0, 40), (64, 24, 64, 1),
    (256, 16, 700, 60), (257, 64, 9, 9), (700, 16, 30, 20), (3, 1, 5, 5), (2, 16, 100000, 20000)])
@pytest.mark.parametrize("in_place", [False, True])
def test_slots_match_oracle(b, page, cached_hi, new_hi, in_place):
    cached, new, table, free, need = slots_case(b, page, cached_hi, new_hi, b + page, spare=3)
    n = int(new.sum()) + 9
    d, left, code = run_slots(cached, new, table, n, page, free, len(free), in_place)
    assert code == 0
    t, s, cu, seq, want_left, bad = pr.prompt_slots(cached, new, table, n, page, free, len(free))
    assert not bad and left == want_left == len(free) - need
    for got, want in ((d["t"], t), (d["s"], s), (d["cu"], cu), (d["seq"], seq)):
        assert np.array_equal(got.cpu().numpy(), want)


@pytest.mark.parametrize("b", [4, 300])
@pytest.mark.parametrize("share", [0.0, 0.4, 0.9])
def test_slots_when_the_stack_runs_out(b, share):
    cached, new, table, free, need = slots_case(b, 16, 50, 90, b, spare=0)
    count = int(need * share)
    n = int(new.sum())
    d, left, code = run_slots(cached, new, table, n, 16, free, count)
    t, s, cu, seq, want_left, bad = pr.prompt_slots(cached, new, table, n, 16, free, count)
    assert bad and code == 0x80 and left == want_left
    for got, want in ((d["t"], t), (d["s"], s), (d["cu"], cu), (d["seq"], seq)):
        assert np.array_equal(got.cpu().numpy(), want)


def test_slots_without_a_stack_and_with_bad_rows():
    cached, new, table, _, _ = slots_case(6, 16, 60, 40, 1)
    n = int(new.sum())
    d, _, code = run_slots(cached, new, table, n, 16, None, 0)
    t, s, cu, seq, _, _ = pr.prompt_slots(cached, new, table, n, 16)
    assert code == 0
    for got, want in ((d["t"], t), (d["s"], s), (d["cu"], cu), (d["seq"], seq)):
        assert np.array_equal(got.cpu().numpy(), want)
    # too long, negative, and a stack that claims more than it holds
    cached, new = [0, -3, 5, 2 ** 31 - 1, 0], [7, 4, 1000, 5, -2]
    free = list(range(100, 120))
    d, left, code = run_slots(cached, new, np.zeros((5, 4)), 1030, 16, free, 20)
    want = pr.prompt_slots(cached, new, np.zeros((5, 4)), 1030, 16, free, 20)
    assert code == 0x2 and left == want[4]
    for got, w in zip((d["t"], d["s"], d["cu"], d["seq"]), want):
        assert np.array_equal(got.cpu().numpy(), w)
    d, left, code = run_slots([0], [20], np.zeros((1, 4)), 20, 16, free, 999)
    assert code == 0x10 and left == 18 and d["t"][0, :2].tolist() == [119, 118]
    # fewer places than tokens: the row that does not fit is not served; a page id
    # that cannot be a slot
    cached, new = [0, 0, 3], [7, 20, 0]
    d, left, code = run_slots(cached, new, np.zeros((3, 4)), 12, 16, free, 20)
    want = pr.prompt_slots(cached, new, np.zeros((3, 4)), 12, 16, free, 20)
    assert code == 0x8 and left == want[4] == 19 and want[5] == [1]
    for got, w in zip((d["t"], d["s"], d["cu"], d["seq"]), want):
        assert np.array_equal(got.cpu().numpy(), w)
    d, left, code = run_slots([0], [20], np.zeros((1, 4)), 20, 16, [-1, 3], 2)
    assert code == 0x4 >> 2 and d["s"].tolist() == [48 + i for i in range(16)] + [-1] * 4


@pytest.mark.parametrize("page", [1, 16])
def test_slots_of_lengths_that_hold_anything(page):
    """Sums of lengths beyond 32 bits, in one chunk of rows and over all: what comes
    before them is served, no token behind them is."""
    big = 2 ** 31 - 1
    new = [5, 3] + [big] * 9 + [4, 0, 2] + [big - 7] * 260 + [6, 0]
    cached = [0, 2] + [0, 9, 0, -1, 0, 0, 3, 0, 0] + [1, 2, 3] + [0] * 260 + [0, 1]
    width = 64
    free = list(range(50))
    table = np.arange(len(new) * width).reshape(len(new), width) % 40
    for stack, count in ((free, 50), (None, 0)):
        d, left, code = run_slots(cached, new, table, 1500, page, stack, count)
        want = pr.prompt_slots(cached, new, table, 1500, page, stack, count)
        assert code == 0x2 | 0x8 and (stack is None or left == want[4])
        assert np.array_equal(d["cu"].cpu().numpy(), np.minimum(want[2], big))
        for got, w in ((d["t"], want[0]), (d["s"], want[1]), (d["seq"], want[3])):
            assert np.array_equal(got.cpu().numpy(), w)


def test_slots_of_no_rows():
    d, left, code = run_slots([], [], np.zeros((0, 3)), 5, 16, [4, 5], 2)
    assert code == 0 and left == 2 and d["s"].tolist() == [-1] * 5 and d["cu"].tolist() == [0]


def test_slots_in_a_graph_pop_the_stack_each_time():
    table, free = i32(np.zeros((2, 8))), i32(range(40))
    count, ctr = i32([40]), i32([0])
    cached, new = i32([0, 3]), i32([5, 17])
    s, cu, seq = i32(np.zeros(30)), i32(np.zeros(3)), i32(np.zeros(2))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.prompt_slots(cached, new, table, s, cu, seq, free, count, count, ctr, 16)
    for want in (38, 36, 34):
        graph.replay()
        torch.cuda.synchronize()
        assert count.item() == want and table[0, 0].item() == want + 1
    new.copy_(i32([0, 0]))
    graph.replay()
    torch.cuda.synchronize()
    assert count.item() == 34 and s.tolist() == [-1] * 30


# ------------------------------------------------------------------ writes
def slots_of(lens, page, seed, starts=None):
    """Slot map of rows over a shuffled pool; returns (slots, pool pages)."""
    gen = np.random.default_rng(seed)
    starts = [0] * len(lens) if starts is None else starts
    pages = [-(-(s + n) // page) for s, n in zip(starts, lens)]
    perm = gen.permutation(sum(pages) + 5)
    out, at = [], 0
    for s, n, p in zip(starts, lens, pages):
        row = perm[at:at + p]
        at += p
        out += [int(row[i // page]) * page + i % page for i in range(s, s + n)]
    return np.asarray(out, np.int32), sum(pages) + 5


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("lens,hkv,page", [([1], 1, 8), ([37], 8, 16), ([5, 0, 130], 2, 24),
                                           ([700, 3], 3, 64)])
def test_kv_write(lens, hkv, page, dtype):
    slots, pool = slots_of(lens, page, seed=hkv)
    slots[len(slots) // 2] = -1 if len(slots) > 1 else slots[0]
    gen = torch.Generator().manual_seed(1)
    fused = torch.randn(len(slots), 2 * hkv + 1, 128, generator=gen).to(DT[dtype]).cuda()
    k, v = fused[:, :hkv], fused[:, hkv:2 * hkv]
    kp = torch.randn(pool, hkv, page, 128, generator=gen).to(DT[dtype]).cuda()
    vp = torch.randn(pool, hkv, page, 128, generator=gen).to(DT[dtype]).cuda()
    wants = [pr.kv_write(x.float().cpu().numpy(), p.float().cpu().numpy(), slots)
             for x, p in ((k, kp), (v, vp))]
    ops.kv_write(k, v, kp, vp, i32(slots))
    no_error()
    for got, want in zip((kp, vp), wants):
        assert np.array_equal(got.float().cpu().numpy(), want)
    bad = slots.copy()
    bad[-1] = pool * page
    ops.kv_write(k, v, kp, vp, i32(bad))
    torch.cuda.synchronize()
    assert _native.device_error(clear=True) == 0x8
    for got, want in zip((kp, vp), wants):
        assert np.array_equal(got.float().cpu().numpy(), want)


def empty_cache(pool, hkv, page, block):
    """Pools and scales as an allocator leaves them: NaN codes, NaN scales."""
    p = torch.full((pool, hkv, page, 128), 255, dtype=torch.uint8, device="cuda")
    s = torch.full((pool, hkv, page // block), float("nan"), device="cuda")
    return p.view(torch.float8_e4m3fn), s


def check_block_write(k, v, slots, kp, vp, ks, vs):
    wants = [pr.kv_write_fp8_block(x.double().cpu().numpy(), p.view(torch.uint8).cpu().numpy(),
                                   s.cpu().numpy(), slots) for x, p, s in ((k, kp, ks), (v, vp, vs))]
    ops.kv_write_fp8_block(k, v, kp, vp, ks, vs, i32(slots))
    no_error()
    for (codes, scales), p, s in zip(wants, (kp, vp), (ks, vs)):
        assert np.array_equal(s.cpu().numpy().astype(np.float64), scales, equal_nan=True)
        got = p.view(torch.uint8).cpu().numpy()
        nan = (got & 127) == 127
        assert np.array_equal(nan, (codes & 127) == 127)
        assert np.array_equal(got[~nan], codes[~nan])


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("lens,starts,hkv,page,block", [
    ([1], [0], 1, 16, 16), ([37], [0], 8, 16, 16), ([5, 0, 130], [0, 0, 0], 2, 32, 16),
    ([200, 3, 70], [0, 0, 0], 3, 64, 64), ([150], [0], 2, 48, 16), ([300], [0], 1, 128, 128)])
def test_block_write_of_prompts(lens, starts, hkv, page, block, dtype):
    slots, pool = slots_of(lens, page, seed=hkv, starts=starts)
    gen = torch.Generator().manual_seed(page)
    x = torch.randn(len(slots), 2 * hkv, 128, generator=gen)
    x *= torch.exp(2 * torch.randn(len(slots), 2 * hkv, 1, generator=gen))
    x = x.to(DT[dtype]).cuda()
    kp, ks = empty_cache(pool, hkv, page, block)
    vp, vs = empty_cache(pool, hkv, page, block)
    check_block_write(x[:, :hkv], x[:, hkv:], slots, kp, vp, ks, vs)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("page,block", [(16, 16), (64, 32)])
def test_block_write_continues_a_block(page, block, dtype):
    """Chunks and single tokens that go on inside a block, of magnitudes that
    grow and shrink."""
    gen = torch.Generator().manual_seed(block)
    rows, hkv, step = 3, 2, [5, 1, 1, 1, 9, 1, 30, 1, 1, 64, 1]
    total = sum(step)
    all_slots, pool = slots_of([total] * rows, page, seed=block)
    all_slots = all_slots.reshape(rows, total)
    kp, ks = empty_cache(pool, hkv, page, block)
    vp, vs = empty_cache(pool, hkv, page, block)
    at = 0
    for i, n in enumerate(step):
        x = torch.randn(rows * n, 2 * hkv, 128, generator=gen) * 4.0 ** ((3 * i) % 5 - 2)
        x = x.to(DT[dtype]).cuda()
        slots = all_slots[:, at:at + n].reshape(-1)
        check_block_write(x[:, :hkv], x[:, hkv:], slots, kp, vp, ks, vs)
        at += n


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_block_write_of_extreme_values(dtype):
    top = torch.finfo(DT[dtype]).max
    tiny = torch.finfo(DT[dtype]).tiny
    rows = [0.0, top, -top, tiny, 448.0, 449.0, float("inf"), -float("inf"), float("nan"), 1e-7]
    n = 16 * len(rows)
    slots, pool = slots_of([n], 16, seed=2)
    x = torch.zeros(n, 2, 128)
    for i, r in enumerate(rows):   # one block each
        x[16 * i + 3, :, 5] = r
    x[16 * 6 + 4, :, 9] = 2.5      # a finite value beside an infinity
    x = x.to(DT[dtype]).cuda()
    kp, ks = empty_cache(pool, 1, 16, 16)
    vp, vs = empty_cache(pool, 1, 16, 16)
    check_block_write(x[:, :1], x[:, 1:], slots, kp, vp, ks, vs)


def test_block_write_skips_padding_and_refuses_bad_slots():
    slots, pool = slots_of([40], 16, seed=9)
    slots[16:20] = -1
    slots = np.concatenate([[-1, -1], slots, [-1] * 20]).astype(np.int32)
    x = torch.randn(len(slots), 4, 128).half().cuda()
    kp, ks = empty_cache(pool, 2, 16, 16)
    vp, vs = empty_cache(pool, 2, 16, 16)
    check_block_write(x[:, :2], x[:, 2:], slots, kp, vp, ks, vs)
    before = kp.view(torch.uint8).clone()
    bad = torch.full((len(slots),), pool * 16 + 3, dtype=torch.int32, device="cuda")
    ops.kv_write_fp8_block(x[:, :2], x[:, 2:], kp, vp, ks, vs, bad)
    torch.cuda.synchronize()
    assert _native.device_error(clear=True) == 0x8
    assert torch.equal(before, kp.view(torch.uint8))


# ------------------------------------------------------------------ decode
def decode_case(lens, hq, hkv, page, block, dtype, seed, spread=0.6):
    """A cache whose unused places (slots past a row's end, their scales, pages
    of no row) hold NaN."""
    slots, pool = slots_of(lens, page, seed)
    gen = torch.Generator().manual_seed(seed)
    kp, ks = empty_cache(pool, hkv, page, block)
    vp, vs = empty_cache(pool, hkv, page, block)
    x = torch.randn(len(slots), 2 * hkv, 128, generator=gen)
    x *= torch.exp(spread * torch.randn(len(slots), 2 * hkv, 1, generator=gen))
    x = x.to(DT[dtype]).cuda()
    if len(slots):
        ops.kv_write_fp8_block(x[:, :hkv], x[:, hkv:], kp, vp, ks, vs, i32(slots))
    width = max(1, max(-(-n // page) for n in lens))
    table, at = np.full((len(lens), width), pool - 1, np.int32), 0
    for b, n in enumerate(lens):
        for j in range(-(-n // page)):
            table[b, j] = slots[at + j * page] // page
        at += n
    q = torch.randn(len(lens), hq, 128, generator=gen).to(DT[dtype])
    return q, kp, ks, vp, vs, table


def run_decode(q, kp, ks, vp, vs, table, lens, fused=True, qi=None, oi=None, out=None):
    b, hq, hkv = table.shape[0], q.shape[1], kp.shape[1]
    if out is None:
        out = torch.full((b, hq, 128), 7.0, dtype=q.dtype, device="cuda")
    ws = torch.full((ops.auto_workspace_bytes(b, hq, hkv) // 4,), float("nan"), device="cuda")
    ctr = torch.zeros(b, hkv, dtype=torch.int32, device="cuda") if fused else None
    ops.paged_attention_auto_fp8_block(q.cuda(), kp, vp, ks, vs, i32(table), i32(lens), out, ws,
                                       qi, oi, ctr)
    no_error()
    if fused:
        assert not ctr.any()
    return out


def check_decode(got, q, kp, ks, vp, vs, table, lens, dtype, qi=None, oi=None):
    kd = pr.dequantised(kp.view(torch.uint8).cpu().numpy(), ks.cpu().numpy())
    vd = pr.dequantised(vp.view(torch.uint8).cpu().numpy(), vs.cpu().numpy())
    # weights are rounded to fp16 with the V scale in their exponent: one below
    # fp16's normal range is off by 2^-25 of the largest weight * V scale
    want, mag, size, unit = pr.paged_decode(q.double().numpy(), kd, vd, vs.cpu().numpy(), table,
                                            lens, qi, oi, got.shape[0])
    check_close(got, want, mag, size, unit[..., None], dtype, "f16")


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("lens", [[1], [0], [15, 16, 17], [31, 33, 0, 64], [65, 1, 300],
                                  [1000, 5], [4097]])
def test_decode_lengths(lens, dtype):
    c = decode_case(lens, 8, 2, 16, 16, dtype, seed=sum(lens))
    check_decode(run_decode(*c, lens), *c, lens, dtype)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("hq,hkv", [(1, 1), (3, 3), (4, 2), (4, 1), (8, 1), (16, 2), (32, 8)])
def test_decode_heads(hq, hkv, dtype):
    lens = [130, 700]
    c = decode_case(lens, hq, hkv, 32, 16, dtype, seed=hq)
    check_decode(run_decode(*c, lens), *c, lens, dtype)


@pytest.mark.parametrize("fused", [True, False])
@pytest.mark.parametrize("page,block", [(16, 16), (32, 16), (32, 32), (48, 16), (64, 64),
                                        (128, 32), (256, 256)])
def test_decode_pages(page, block, fused):
    lens = [page, page + 1, 3 * page - 1, 2000, 0]
    c = decode_case(lens, 8, 2, page, block, "f16", seed=page)
    check_decode(run_decode(*c, lens, fused=fused), *c, lens, "f16")


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_decode_indexed_rows(dtype):
    lens = [200, 0, 77]
    c = decode_case(lens, 4, 2, 16, 16, dtype, seed=1)
    q = torch.randn(6, 4, 128).to(DT[dtype])
    qi, oi = [5, 0, 2], [1, 4, 0]
    out = torch.full((5, 4, 128), 7.0, dtype=DT[dtype], device="cuda")
    got = run_decode(q, *c[1:], lens, qi=i32(qi), oi=i32(oi), out=out)
    check_decode(got, q, *c[1:], lens, dtype, qi, oi)
    assert (got[[2, 3]] == 7.0).all()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_decode_scales_far_apart(dtype):
    """Blocks at magnitudes from 2^-24 to 2^20, blocks of zeros with scale zero,
    and queries that look only at a small one."""
    lens = [16 * 12 + 7]
    q, kp, ks, vp, vs, table = decode_case(lens, 4, 1, 16, 16, dtype, seed=5, spread=0.0)
    for j in range(13):
        vs[table[0, j], 0, 0] *= 2.0 ** [-16, 20, 0, -12, 14][j % 5]
    vs[table[0, 4], 0, 0] = 0.0
    ks[table[0, 7], 0, 0] = 0.0
    c = (q, kp, ks, vp, vs, table)
    check_decode(run_decode(*c, lens), *c, lens, dtype)
    # all weight on one block of small values among large ones
    kp.view(torch.uint8)[table[0, 0].item()] = 0x38          # 1.0
    ks[table[0, 0], 0, 0] = 30.0
    q = q.abs() * 0 + 1
    c = (q, kp, ks, vp, vs, table)
    check_decode(run_decode(*c, lens), *c, lens, dtype)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_decode_zero_blocks_count_in_the_sum(dtype):
    """Most blocks are zeros of scale 0 with codes that mean nothing, under large V
    scales: their weights still share the sum."""
    lens = [16 * 40]
    q, kp, ks, vp, vs, table = decode_case(lens, 4, 1, 16, 16, dtype, seed=6, spread=0.0)
    vs *= 2.0 ** 12
    for j in range(40):
        if j % 8 != 3:
            vs[table[0, j], 0, 0] = 0.0
    vp_nan = vp.view(torch.uint8).clone()
    zero = (vs[:, 0, 0] == 0).nonzero()[:, 0]
    vp_nan[zero] = 0x7f
    got = run_decode(q, kp, ks, vp_nan.view(torch.float8_e4m3fn), vs, table, lens)
    vp.view(torch.uint8)[zero] = 0
    check_decode(got, q, kp, ks, vp, vs, table, lens, dtype)


def test_decode_bf16_queries_beyond_fp16():
    lens = [100]
    q, kp, ks, vp, vs, table = decode_case(lens, 4, 1, 16, 16, "bf16", seed=5)
    for f in (1e6, 1e-12):
        q2 = (q.float() * f).to(torch.bfloat16)
        ks2 = ks / f
        c = (q2, kp, ks2, vp, vs, table)
        check_decode(run_decode(*c, lens), *c, lens, "bf16")


def test_decode_flags_bad_pages_and_indices():
    lens = [50, 40]
    q, kp, ks, vp, vs, table = decode_case(lens, 4, 1, 16, 16, "f16", seed=5)
    ws = torch.empty(ops.auto_workspace_bytes(2, 4, 1) // 4, device="cuda")
    out = torch.zeros(2, 4, 128, dtype=torch.float16, device="cuda")
    bad = table.copy()
    bad[0, 1] = kp.shape[0]
    ops.paged_attention_auto_fp8_block(q.cuda(), kp, vp, ks, vs, i32(bad), i32(lens), out, ws)
    torch.cuda.synchronize()
    assert _native.device_error(clear=True) == 0x1
    ops.paged_attention_auto_fp8_block(q.cuda(), kp, vp, ks, vs, i32(table), i32([50, 900]), out,
                                       ws)
    torch.cuda.synchronize()
    assert _native.device_error(clear=True) == 0x2
    ops.paged_attention_auto_fp8_block(q.cuda(), kp, vp, ks, vs, i32(table), i32(lens), out, ws,
                                       i32([0, 9]))
    torch.cuda.synchronize()
    assert _native.device_error(clear=True) == 0x10


def test_decode_in_two_graphs_with_their_own_workspaces():
    lens = [900, 30, 2000]
    c = decode_case(lens, 16, 2, 16, 16, "bf16", seed=3)
    q, kp, ks, vp, vs, table = c
    want = run_decode(*c, lens)
    dq, t, sl = q.cuda(), i32(table), i32(lens)
    graphs = []
    for _ in range(2):
        out = torch.zeros(3, 16, 128, dtype=torch.bfloat16, device="cuda")
        ws = torch.empty(ops.auto_workspace_bytes(3, 16, 2) // 4, device="cuda")
        ctr = torch.zeros(3, 2, dtype=torch.int32, device="cuda")
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            ops.paged_attention_auto_fp8_block(dq, kp, vp, ks, vs, t, sl, out, ws,
                                               merge_counters=ctr)
        graphs.append((g, out, ws, ctr))
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(5):
        for (g, *_), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for _, out, _, _ in graphs:
        assert torch.equal(out, want)


# ------------------------------------------------------------------ together
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_prompt_then_decode_over_one_cache(dtype):
    """Two prompts enter the cache in two chunks and are attended to; then tokens
    are decoded one by one, each step's K/V appended through the same calls."""
    hq, hkv, page, width = 8, 2, 16, 24
    gen = torch.Generator().manual_seed(7)
    new = lambda n, h: torch.randn(n, h, 128, generator=gen).to(DT[dtype])  # noqa: E731
    pool = 60
    kp, ks = empty_cache(pool, hkv, page, page)
    vp, vs = empty_cache(pool, hkv, page, page)
    table = torch.full((2, width), -1, dtype=torch.int32, device="cuda")
    free, count, ctr = i32(np.random.default_rng(1).permutation(pool)), i32([pool]), i32([0])
    lens, cu, after = i32([0, 0]), i32([0, 0, 0]), i32([0, 0])
    history = [(new(0, hkv), new(0, hkv)) for _ in range(2)]
    ws = torch.empty(ops.auto_workspace_bytes(2, hq, hkv) // 4, device="cuda")
    mc = torch.zeros(2, hkv, dtype=torch.int32, device="cuda")
    for step, n in enumerate([(70, 5), (40, 133), (1, 1), (1, 1), (1, 1)]):
        total = sum(n)
        q, k, v = new(total, hq), new(total, hkv), new(total, hkv)
        slots = torch.empty(total, dtype=torch.int32, device="cuda")
        ops.prompt_slots(lens, i32(n), table, slots, cu, after, free, count, count, ctr, page)
        ops.kv_write_fp8_block(k.cuda(), v.cuda(), kp, vp, ks, vs, slots)
        parts = k.split(n), v.split(n)
        history = [(torch.cat([h[0], parts[0][i]]), torch.cat([h[1], parts[1][i]]))
                   for i, h in enumerate(history)]
        lens.copy_(after)
        assert lens.tolist() == [len(h[0]) for h in history]
        if step < 2:
            # a chunk sees its own keys and the earlier ones
            ck = np.cumsum([0] + [len(h[0]) for h in history])
            k_all = torch.cat([h[0] for h in history])
            v_all = torch.cat([h[1] for h in history])
            out, ls = run_prompt(q, k_all, v_all, cu.tolist(), ck)
            check_prompt(q, k_all, v_all, cu.tolist(), ck, dtype, out, ls)
        else:
            out = torch.empty(2, hq, 128, dtype=DT[dtype], device="cuda")
            ops.paged_attention_auto_fp8_block(q.cuda(), kp, vp, ks, vs, table.clamp_min(0), lens,
                                               out, ws, merge_counters=mc)
            no_error()
            c = (q, kp, ks, vp, vs, table.clamp_min(0).cpu().numpy())
            check_decode(out, *c, lens.tolist(), dtype)
            # and the cache holds the tokens: e4m3's half step of each block's largest
            for b, (hk, _) in enumerate(history):
                kd = pr.dequantised(kp.view(torch.uint8).cpu().numpy(), ks.cpu().numpy())
                pages = table[b].tolist()[:-(-len(hk) // page)]
                got = kd[pages].transpose(0, 2, 1, 3).reshape(-1, hkv, 128)[:len(hk)]
                off = np.abs(got - hk.double().numpy())
                assert (off <= 2.0 ** -4 * np.abs(hk.double().numpy()) + 2.0 ** -9).all()
    no_error()


@pytest.mark.parametrize("cache", ["f16", "bf16", "block-f16", "block-bf16"])
def test_engine_prefill_then_steps(cache):
    """The engine's own path: prompts through ``prefill``, then decode steps over
    what it wrote, for 16-bit caches and e4m3 ones with block scales."""
    dtype = cache.rsplit("-")[-1]
    hq, hkv, page, pool, width = 16, 4, 32, 40, 12
    gen = torch.Generator().manual_seed(9)
    new = lambda n, h: torch.randn(n, h, 128, generator=gen).to(DT[dtype])  # noqa: E731
    if cache.startswith("block"):
        kp, ks = empty_cache(pool, hkv, page, 16)
        vp, vs = empty_cache(pool, hkv, page, 16)
        engine = DecodeEngine(kp, vp, hq, kv_block_scales=(ks, vs), q_dtype=DT[dtype])
    else:
        kp = torch.zeros(pool, hkv, page, 128, dtype=DT[dtype], device="cuda")
        vp = torch.zeros_like(kp)
        engine = DecodeEngine(kp, vp, hq)
    stack = PageStack.full(pool, "cuda")
    lens = [130, 1, 300, 0]
    total, pad = sum(lens), 9
    q, k, v = new(total + pad, hq), new(total + pad, hkv), new(total + pad, hkv)
    table = torch.zeros(4, width, dtype=torch.int32, device="cuda")
    out = torch.full((total + pad, hq, 128), 7.0, dtype=DT[dtype], device="cuda")
    lse = torch.full((total + pad, hq), 7.0, device="cuda")
    seq = engine.prefill(q.cuda(), k.cuda(), v.cuda(), i32(lens), table, out, stack, lse)
    no_error()
    assert seq.tolist() == lens and stack.free_count.item() == pool - 5 - 1 - 10
    cu = np.cumsum([0] + lens)
    check_prompt(q, k, v, cu, cu, dtype, out, lse)
    plan = engine.upload(engine.plan_step(lens, table.cpu().numpy()))
    dq = new(4, hq)
    step = torch.zeros(4, hq, 128, dtype=DT[dtype], device="cuda")
    engine.run(plan, dq.cuda(), step)
    no_error()
    t = table.cpu().numpy()
    if cache.startswith("block"):
        check_decode(step, dq, kp, ks, vp, vs, t, lens, dtype)
    else:
        one = np.ones((pool, hkv, 1))
        want, mag, size, _ = pr.paged_decode(dq.double().numpy(), kp.double().cpu().numpy(),
                                             vp.double().cpu().numpy(), one, t, lens)
        check_close(step, want, mag, size, 1e3, dtype)


def test_engine_refuses_caches_it_cannot_fill():
    p8, s8 = empty_cache(4, 2, 16, 16)
    p16 = torch.zeros(4, 2, 16, 128, dtype=torch.float16, device="cuda")
    with pytest.raises(RuntimeError, match="kv_scales or kv_block_scales"):
        DecodeEngine(p8, p8, 4)
    with pytest.raises(RuntimeError, match="kv_scales or kv_block_scales"):
        DecodeEngine(p8, p8, 4, kv_scales=(1.0, 1.0), kv_block_scales=(s8, s8))
    with pytest.raises(RuntimeError, match="belong to an e4m3"):
        DecodeEngine(p16, p16, 4, kv_block_scales=(s8, s8))
    x = torch.zeros(3, 2, 128, dtype=torch.float16, device="cuda")
    q = torch.zeros(3, 4, 128, dtype=torch.float16, device="cuda")
    with pytest.raises(RuntimeError, match="prefill writes"):
        DecodeEngine(p8, p8, 4, kv_scales=(1.0, 1.0)).prefill(
            q, x, x, i32([3]), i32([[0]]), torch.empty_like(q))


def test_engine_refuses_before_it_takes_pages():
    p8, s8 = empty_cache(4, 2, 16, 16)
    p16 = torch.zeros(4, 2, 16, 128, dtype=torch.float16, device="cuda")
    x = torch.zeros(3, 2, 128, dtype=torch.float16, device="cuda")
    q = torch.zeros(3, 4, 128, dtype=torch.float16, device="cuda")
    stack, table, new = PageStack.full(4, "cuda"), i32([[-1]]), i32([3])
    good = DecodeEngine(p16, p16.clone(), 4)
    block = DecodeEngine(p8, p8.clone(), 4, kv_block_scales=(s8, s8.clone()))
    for engine, args in (
            (DecodeEngine(p8, p8, 4, kv_scales=(1.0, 1.0)), (q, x, x, new, table, q.clone())),
            (good, (q, x, x[:2], new, table, q.clone())), (good, (q, x, x, new, table, q[:2])),
            (good, (q.bfloat16(), x.bfloat16(), x.bfloat16(), new, table, q.bfloat16())),
            (block, (q, x[:, :1], x[:, :1], new, table, q.clone()))):
        with pytest.raises(RuntimeError):
            engine.prefill(*args, stack)
    torch.cuda.synchronize()
    assert stack.free_count.item() == 4 and table.tolist() == [[-1]]
    good.prefill(q, x, x, new, table, q.clone(), stack)
    no_error()
    assert stack.free_count.item() == 3 and table.tolist() == [[0]]


# ------------------------------------------------------------------ offsets past 32 bits
def test_prompt_beyond_4gb():
    """Strided operands and packed rows whose bytes lie past 2^32."""
    gap, n = 1 << 22, 600                     # elements between tokens: 8 MB
    big = torch.empty(gap * n, dtype=torch.bfloat16, device="cuda")
    q, k, v, cq, ck = packed([n], [n], 2, 1, "bf16", seed=12)
    views, at = [], 0
    for t in (q, k, v):
        view = big.as_strided((n, t.shape[1], 128), (gap, 128, 1), at)
        view.copy_(t)
        views.append(view)
        at += t.shape[1] * 128
    out = torch.full(q.shape, 7.0, dtype=q.dtype, device="cuda")
    ls = torch.full(q.shape[:2], 7.0, device="cuda")
    ops.prompt_attention(*views, i32(cq), None, out, lse=ls)
    no_error()
    check_prompt(q, k, v, cq, ck, "bf16", out, ls)
    del big, views
    # the last rows of a long packed batch; nobody's rows before them
    rows = (1 << 32) // (8 * 256) + 70
    dq = torch.zeros(rows, 8, 128, dtype=torch.float16, device="cuda")
    out = torch.zeros_like(dq)
    q, k, v, cq, ck = packed([60], [60], 8, 2, "f16", seed=13)
    dq[-60:] = q.cuda()
    ops.prompt_attention(dq, k.cuda(), v.cuda(), i32([rows - 60, rows]), i32([0, 60]), out)
    no_error()
    small, _ = run_prompt(q, k, v, cq, ck)
    assert torch.equal(out[-60:], small) and not out[:-60].any()


@pytest.mark.parametrize("cache", ["f16", "block"])
def test_pools_beyond_4gb(cache):
    """Writes to and decode from the last pages of pools past 2^32 bytes."""
    hq, hkv, page = 8, 4, 16
    elem = 2 if cache == "f16" else 1
    pool = (1 << 32) // (hkv * page * 128 * elem) + 9
    n = 100
    pages = np.arange(pool - 1, pool - 8, -1)
    slots = np.concatenate([p * page + np.arange(page) for p in pages])[:n].astype(np.int32)
    gen = torch.Generator().manual_seed(4)
    k, v = (torch.randn(n, hkv, 128, generator=gen).half() for _ in range(2))
    q = torch.randn(1, hq, 128, generator=gen).half()
    table, lens = pages[None], [n]
    near = np.arange(7)[None]               # the same rows in a pool of 7 pages
    local = np.arange(n, dtype=np.int32)
    if cache == "f16":
        outs = []
        for size, s, t in ((pool, slots, table), (7, local, near)):
            kp = torch.zeros(size, hkv, page, 128, dtype=torch.float16, device="cuda")
            vp = torch.zeros_like(kp)
            ops.kv_write(k.cuda(), v.cuda(), kp, vp, i32(s))
            engine = DecodeEngine(kp, vp, hq)
            out = torch.zeros(1, hq, 128, dtype=torch.float16, device="cuda")
            engine.run(engine.upload(engine.plan_step(lens, t.astype(np.int32))), q.cuda(), out)
            no_error()
            outs.append((kp[torch.as_tensor(t[0]).cuda()], vp[torch.as_tensor(t[0]).cuda()], out))
            del kp, vp, engine
    else:
        outs = []
        for size, s, t in ((pool, slots, table), (7, local, near)):
            kp = torch.zeros(size, hkv, page, 128, dtype=torch.uint8, device="cuda")
            kp = kp.view(torch.float8_e4m3fn)
            vp = torch.zeros_like(kp.view(torch.uint8)).view(torch.float8_e4m3fn)
            ks = torch.zeros(size, hkv, 1, device="cuda")
            vs = torch.zeros_like(ks)
            ops.kv_write_fp8_block(k.cuda(), v.cuda(), kp, vp, ks, vs, i32(s))
            out = run_decode(q, kp, ks, vp, vs, t, lens)
            no_error()
            at = torch.as_tensor(t[0]).cuda()
            outs.append((kp.view(torch.uint8)[at], vp.view(torch.uint8)[at], ks[at], vs[at], out))
            del kp, vp, ks, vs
    for a, b in zip(*outs):
        assert torch.equal(a, b)
    assert outs[0][-1].any()
