"""The device's status word with two kinds of report: an expired wait, whose output is invalid, is never
hidden by contents that another call skipped, nor by the clearing of an earlier report."""
import numpy as np
import pytest
import torch

import mvlm_b200 as mg
from tests.paged import Pool, assert_within, from_bits, to_bits

pytestmark = pytest.mark.gpu


def wrong_page(dev):
    pool = Pool(dev, [1], [40], 2, 64, 16, mg.F16)
    pool.buffers[2].write(np.array([-7], np.int32), offset=4)
    q, out = dev.array(np.zeros(256, np.uint16), mg.F16), dev.empty(256, mg.F16)
    ev = mg.paged_attention(pool.cache, pool.batch, q, out, 4)
    return ev, (pool, q, out)


def code_of(call):
    with pytest.raises(mg.MgpuError) as e:
        call()
    return e.value.code


def still_right(dev):
    pool = Pool(dev, [200, 1], [3000, 70], 2, 128, 16, mg.BF16)
    q = torch.randn(pool.tokens, 8, 128, generator=pool.g).bfloat16()
    out = dev.empty(pool.tokens * 1024, mg.BF16)
    want, tol = pool.attention(q, 8, 128 ** -0.5)
    for _ in range(2):
        mg.paged_attention(pool.cache, pool.batch, dev.array(to_bits(q, mg.BF16), mg.BF16), out, 8)
        dev.finish()
        assert_within(from_bits(out.read(np.uint16), mg.BF16).view(want.shape), want, tol)


@pytest.mark.parametrize("wait_first", [True, False])
def test_an_expired_wait_has_the_word(dev, wait_first):
    dev.finish()
    keep = None
    for wait in (wait_first, not wait_first):
        if wait:
            dev.selftest_bounded_wait(2_000_000)
        else:
            keep = wrong_page(dev)
    assert code_of(dev.finish) == mg.ERR_DEVICE_TIMEOUT
    dev.finish()
    still_right(dev)
    del keep


def test_a_report_is_not_cleared_with_the_one_before(dev):
    dev.finish()
    keep = wrong_page(dev)
    dev.selftest_bounded_wait(200_000_000)  # still waiting when the first report is read
    assert code_of(keep[0].wait) == mg.ERR_INVALID_ARG
    assert code_of(dev.finish) == mg.ERR_DEVICE_TIMEOUT
    dev.finish()
    still_right(dev)
