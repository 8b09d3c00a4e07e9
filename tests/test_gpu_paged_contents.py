"""What mgpu_paged_attention and mgpu_kv_append find in a batch's buffers: every page outside the cache that a
key needs is reported, whatever its bits, and the other sequences have their results."""
import numpy as np
import pytest
import torch

import mvlm_b200 as mg
from tests.paged import Pool, assert_within, from_bits, to_bits

pytestmark = pytest.mark.gpu


def reported(dev):
    with pytest.raises(mg.MgpuError) as e:
        dev.finish()
    assert e.value.code == mg.ERR_INVALID_ARG
    dev.finish()  # once


@pytest.mark.parametrize("page", [-1, -2, -3, -2 ** 31, 2 ** 31 - 1])
@pytest.mark.parametrize("n", [1, 150])
def test_every_page_outside_the_cache_is_reported(dev, n, page):
    pool = Pool(dev, [n, 2], [200, 90], 2, 64, 16, mg.F16)
    q = torch.randn(pool.tokens, 4, 64, generator=pool.g).half()
    want, tol = pool.attention(q, 4, 0.125)
    src, dst = dev.array(to_bits(q, mg.F16), mg.F16), dev.empty(pool.tokens * 256, mg.F16)
    for at in (0, 3, 12):  # 12: the last, which ends inside a block
        table = pool.table.copy()
        table[0, at] = page
        pool.buffers[2].write(table)
        mg.paged_attention(pool.cache, pool.batch, src, dst, 4)
        reported(dev)
        got = from_bits(dst.read(np.uint16), mg.F16).view(-1, 4, 64)
        assert_within(got[n:], want[n:], tol[n:], f"page {page} at {at}")
