"""A planned decode whose schedule has groups without a row piece."""

import numpy as np
import pytest
import torch

from persistentkv_attention_b200 import _native
from persistentkv_attention_b200.serving import DecodeEngine
from tests.helpers import assert_close, make_case


@pytest.mark.gpu
@pytest.mark.parametrize("lens,groups", [([130, 1, 0], 19), ([1], 37), ([0, 40], 8)])
def test_more_groups_than_tiles_is_no_error(lens, groups):
    c = make_case(lens, hq=8, hkv=2, page_size=32)
    d = c.cuda()
    _native.device_error(clear=True)
    engine = DecodeEngine(d["k_pages"], d["v_pages"], c.hq, groups=groups)
    out = torch.full((len(lens), c.hq, 128), float("nan"), dtype=torch.float16, device="cuda")
    engine.run(engine.upload(engine.plan_step(lens, c.block_table)), d["q_source"], out)
    torch.cuda.synchronize()
    assert _native.device_error(clear=True) == 0
    want = np.nan_to_num(c.oracle())
    assert_close(out, want, "f16")
