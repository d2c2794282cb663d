"""The prompt operators and the block-scaled cache where their contracts are
widest: block and page sizes, values that are not finite, scales far apart,
nothing to do."""

import pytest
import torch

from persistentkv_attention_b200 import _native
from tests.test_prompt_gpu import (DT, check_block_write, check_decode, decode_case, empty_cache,
                                   run_decode, slots_of)

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
