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


def test_append_reports_a_start_before_the_rows(dev):
    pool = Pool(dev, [2, 3], [10, 20], 2, 64, 16, mg.F16, max_q_len=2 ** 31 - 1)
    x = dev.array(np.ones((5, 128), np.float32), mg.F32)
    for start in (-1, -2 ** 31, -2 ** 31 + 1):
        pool.buffers[0].write(np.array([start, 2, 5], np.int32))
        mg.kv_append(pool.cache, pool.batch, None, x, x, None, 0)
        reported(dev)
        k = from_bits(pool.cache.k.read(np.uint16), mg.F16).view(pool.k.shape)
        want = pool.k.clone()
        for p in range(17, 20):
            want[pool.table[1, p // 16], :, p % 16] = 1.0
        assert torch.equal(k, want), start


def test_more_values_of_a_token_than_are_counted(dev):
    pool = Pool(dev, [1], [10], 2, 64, 16, mg.F16)
    x, q = dev.array(np.ones((1, 128), np.float32), mg.F32), dev.empty(256, mg.F16)
    for heads, code in ((2 ** 24 - 3, mg.ERR_UNSUPPORTED), (2 ** 31 - 1, mg.ERR_UNSUPPORTED), (2 ** 24 - 4, mg.ERR_INVALID_ARG), (5, mg.ERR_INVALID_ARG)):
        with pytest.raises(mg.MgpuError) as e:  # the last two fit, but q does not hold them
            mg.kv_append(pool.cache, pool.batch, q, x, x, dev.empty(256, mg.F16), heads)
        assert e.value.code == code, heads
    dev.finish()


def test_append_reports_negative_lengths_under_a_wide_table(dev):
    # 2.2e9 places in the table: an index that wrapped around would find a page there
    page, wide = 1000, 2_200_000
    cache = mg.KVCache(dev, 2, page, 1, 8, mg.F16)
    x = dev.array(np.ones((2, 8), np.float32), mg.F32)
    lens = dev.array(np.array([0], np.int32), mg.F32)
    batch = mg.PagedBatch(dev.array(np.array([0, 2], np.int32), mg.F32), lens, dev.array(np.zeros(wide, np.int32), mg.F32), 1, 2, 2, wide)
    for kv in (-2 ** 31, -2 ** 31 + 1, -1, 0, 1):
        lens.write(np.array([kv], np.int32))
        mg.kv_append(cache, batch, None, x, x, None, 0)
        reported(dev)
        k = from_bits(cache.k.read(np.uint16), mg.F16).view(2, page, 8)
        assert bool((k[:, 1:] == 0).all()) and bool((k[1] == 0).all()), kv
        assert bool((k[0, 0] == (1.0 if kv == 1 else 0.0)).all()), kv  # of two tokens, the second has a place


def test_sequences_that_share_rows(dev):
    # cu_q descends: more new tokens in all than there are rows, which the counts of items do not allow for
    n = 300
    pool = Pool(dev, [n, 0, n], [400, 400, 500], 2, 64, 16, mg.F16)
    pool.tokens = pool.batch.c.n_tokens = n
    pool.buffers[0].write(np.array([0, n, 0, n], np.int32))
    src, dst = dev.array(np.zeros(n * 256, np.uint16), mg.F16), dev.array(np.full(n * 256, 0x4000, np.uint16), mg.F16)
    mg.paged_attention(pool.cache, pool.batch, src, dst, 4)
    reported(dev)
    assert bool((dst.read(np.uint16) == 0x4000).all())
