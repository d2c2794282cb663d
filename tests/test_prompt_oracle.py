"""The prompt oracle against independent statements of the same things (CPU)."""

import numpy as np
import pytest
import torch

from oracle import prompt_oracle as pr


def test_e4m3_codes_match_torch():
    codes = np.arange(256, dtype=np.uint8)
    mine = pr.e4m3_decode(codes)
    theirs = torch.from_numpy(codes).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(mine, theirs, equal_nan=True)
    gen = np.random.default_rng(0)
    x = np.concatenate([gen.normal(0, s, 4000) for s in (1e-3, 0.05, 1, 100)])
    x = x[np.abs(x) <= 448].astype(np.float32)
    # midpoints of neighbouring values: ties go to the even code
    pos = mine[:127]
    x = np.concatenate([x, ((pos[1:] + pos[:-1]) / 2).astype(np.float32), [0.0, -0.0, 448, -448]])
    want = torch.from_numpy(x.astype(np.float32)).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(pr.e4m3_encode(x), want)
    assert pr.e4m3_encode([np.inf, -np.inf, 1e6]).tolist() == [126, 254, 126]


@pytest.mark.parametrize("amax,scale", [
    (0.0, 2.0 ** -24), (448.0, 1.0), (448.1, 2.0), (224.0, 0.5), (1.0, 2.0 ** -8),
    (1e-9, 2.0 ** -24), (1.75, 2.0 ** -8), (1.76, 2.0 ** -7), (3e38, 2.0 ** 120)])
def test_least_scale(amax, scale):
    assert pr.least_scale(amax) == scale


def test_attention_matches_softmax():
    gen = torch.Generator().manual_seed(3)
    q = torch.randn(7, 4, 128, generator=gen, dtype=torch.float64)
    k = torch.randn(9, 2, 128, generator=gen, dtype=torch.float64)
    v = torch.randn(9, 2, 128, generator=gen, dtype=torch.float64)
    out, lse, _, _ = pr.prompt_attention(q, k, v, [0, 7], [0, 9])
    s = torch.einsum("qhd,khd->hqk", q, k.repeat_interleave(2, 1)) / 128 ** 0.5
    s = s.masked_fill(torch.ones(7, 9, dtype=torch.bool).triu(3), -torch.inf)
    want = torch.einsum("hqk,khd->qhd", s.softmax(-1), v.repeat_interleave(2, 1))
    assert np.abs(out - want.numpy()).max() < 1e-13
    assert np.abs(lse - torch.logsumexp(s, -1).T.numpy()).max() < 1e-13
    # more queries than keys: the first rows see nothing
    out, lse, _, _ = pr.prompt_attention(q, k[:3], v[:3], [0, 7], [0, 3])
    assert (out[:4] == 0).all() and np.isneginf(lse[:4]).all() and np.isfinite(lse[4:]).all()


def test_appends_token_by_token_keep_the_block_readable():
    """Growing scales move the earlier tokens: each stays within half a step of
    e4m3 per move (2^-4 relative) of what was written."""
    gen = np.random.default_rng(5)
    codes = np.full((1, 1, 16, 128), 255, np.uint8)
    scales = np.full((1, 1, 1), np.nan)
    x = gen.normal(size=(16, 1, 128)) * (2.0 ** np.arange(16))[:, None, None]
    for t in range(16):
        codes, scales = pr.kv_write_fp8_block(x[t:t + 1], codes, scales, [t])
    got = pr.dequantised(codes, scales)[0, 0]
    assert scales[0, 0, 0] == pr.least_scale(np.abs(x).max())
    step = scales[0, 0, 0] * 2.0 ** -9     # e4m3's smallest step at the final scale
    assert (np.abs(got - x[:, 0]) <= np.abs(x[:, 0]) * 2.0 ** -4 + step).all()


def test_slots_by_hand():
    table = np.zeros((3, 4), np.int64)
    table[1, 0] = 9
    table, slots, cu, seq, left, bad = pr.prompt_slots(
        [0, 3, 0], [5, 2, 4], table, 12, 4, free=[20, 21, 22, 23], free_count=3)
    # row 0 takes 22, 21; row 1 continues page 9 and takes 20; row 2 finds nothing
    assert table[0, :2].tolist() == [22, 21] and table[1, :2].tolist() == [9, 20]
    assert slots.tolist() == [88, 89, 90, 91, 84, 39, 80, -1, -1, -1, -1, -1]
    assert cu.tolist() == [0, 5, 7, 11] and seq.tolist() == [5, 5, 0] and left == 0 and bad == [2]
