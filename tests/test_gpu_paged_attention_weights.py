"""The weights of mgpu_paged_attention: what their 16 bits leave out.

Few rows to a key head: a weight and its rest are multiplied, so that the result has the error of fp32
scores, exponentials and sums (2^-13 of its terms, as in test_gpu_paged_attention.py; the rest itself is
2^-17 of a weight or less) and one rounding to the cache's type.  Many rows: one rounding of a weight
more.  Small weights count in fp16 too: its spacing, 2^-24, stands for 2^-31 of the greatest weight."""
import numpy as np
import pytest
import torch

import mvlm_b200 as mg
from tests.paged import UNIT, Pool, assert_within, from_bits, ints, to_bits
from tests.test_gpu_paged_attention import attend

pytestmark = pytest.mark.gpu


def bound(pool, q, q_heads, scale, want, weights_rounded=False, **mask):
    """One rounding of the result, 2^-13 of the terms' magnitudes, 2^-32 of each value that is seen."""
    v = pool.v
    pool.v = torch.nan_to_num(v, 0.0, 0.0, 0.0).abs()
    terms, _ = pool.attention(q, q_heads, scale, **mask)
    pool.v = v
    most = float(pool.v.nan_to_num(0.0, 0.0, 0.0).abs().max())
    u = UNIT[pool.t]
    return u * want.abs().nan_to_num(0.0, 0.0, 0.0) + (2.0 ** -13 + (u if weights_rounded else 0.0)) * terms.abs() + 2.0 ** -32 * max(pool.kv) * most


@pytest.mark.parametrize("t", [mg.F16, mg.BF16])
@pytest.mark.parametrize("new,kv,hq,hk,d", [([1], [300], 8, 2, 128), ([1], [9000], 4, 1, 64), ([1, 2, 4], [40, 700, 65], 8, 2, 128),
                                           ([16, 1], [500, 2000], 2, 2, 64), ([1], [150], 16, 1, 80)])
@pytest.mark.parametrize("spread", [0.3, 2.5, 8.0])
def test_few_rows_round_once(dev, t, new, kv, hq, hk, d, spread):
    pool = Pool(dev, new, kv, hk, d, 16, t, seed=4, fill=float("nan"))
    q = (torch.randn(pool.tokens, hq, d, generator=pool.g) * spread).to(pool.k.dtype)
    got = attend(dev, pool, q, hq)
    want, _ = pool.attention(q, hq, d ** -0.5)
    assert_within(got, want, bound(pool, q, hq, d ** -0.5, want), f"{new} {kv} {spread}")


@pytest.mark.parametrize("n", [1, 3, 40])
@pytest.mark.parametrize("at", [5, 25000])
def test_small_weights_count(dev, n, at):
    """One key of weight 1 and value 0, 50,000 of weight 2^-25.5 and value 1: the result is their share of the
    sum, 1e-3.  160 sequences, so that a CTA takes about one of them whole; two pages hold all keys there are."""
    seqs, kv, page = 160, 50000, 64
    k, v = torch.zeros(2, 1, page, 64), torch.ones(2, 1, page, 64)
    k[1, 0, at % page, 0], v[1, 0, at % page] = 17.671875, 0.0
    cache = mg.KVCache(dev, 2, page, 1, 64, mg.F16, k=dev.array(to_bits(k, mg.F16), mg.F16), v=dev.array(to_bits(v, mg.F16), mg.F16))
    table = np.zeros((seqs, -(-kv // page)), np.int32)
    table[:, at // page] = 1
    batch = mg.PagedBatch(ints(dev, np.arange(seqs + 1) * n), ints(dev, np.full(seqs, kv)), ints(dev, table), seqs, seqs * n, n, table.shape[1])
    q = torch.zeros(seqs * n, 4, 64)
    q[..., 0] = 1.0
    out = dev.empty(seqs * n * 256, mg.F16)
    mg.paged_attention(cache, batch, dev.array(to_bits(q, mg.F16), mg.F16), out, 4, scale=1.0)
    dev.finish()
    got = from_bits(out.read(np.uint16), mg.F16).view(seqs, n, 256)
    rest = (torch.arange(kv - n, kv).double() * np.exp(-17.671875))[None, :, None]  # of the keys up to a token, but one
    want = (rest / (rest + 1.0)).expand(got.shape)
    # the result's rounding, 2^-13 for fp32 scores, exponentials and sums, and half of 2^-31 for each weight
    assert_within(got, want, (UNIT[mg.F16] + 2.0 ** -13) * want + kv * 2.0 ** -32, f"at {at}")


@pytest.mark.parametrize("t", [mg.F16, mg.BF16])
@pytest.mark.parametrize("new,kv,hq,window", [([1], [300], 4, 0), ([1], [9000], 4, 0), ([4, 1], [200, 70], 4, 0), ([3], [900], 2, 130)])
def test_odd_values_that_are_seen(dev, t, new, kv, hq, window):
    inf, nan = float("inf"), float("nan")
    pool = Pool(dev, new, kv, 1, 64, 16, t, seed=8, fill=nan)
    for at, dim, x in ((3, 0, inf), (10, 1, -inf), (40, 2, nan), (50, 3, inf), (60, 3, -inf), (64, 4, inf), (kv[0] - 1, 5, inf),
                       (kv[0] - 100, 6, inf), (kv[0] - 101, 7, -inf), (kv[0] - 131, 63, nan)):
        if 0 <= at < kv[0]:
            pool.v[pool.table[0, at // 16], 0, at % 16, dim] = x
    pool.cache.v.write(to_bits(pool.v, t))
    # scores that spread by 8: some weights are far below fp32's smallest value beside the greatest
    q = (torch.randn(pool.tokens, hq, 64, generator=pool.g) * 30.0).to(pool.k.dtype)
    got = attend(dev, pool, q, hq, window=window)
    want, _ = pool.attention(q, hq, 0.125, window=window)
    # (scores of some hundred: their fp32 error is in every weight)
    assert_within(got, want, 4 * bound(pool, q, hq, 0.125, want, window=window), f"{new} {kv}")


def test_odd_values_among_a_million_keys(dev):
    # 16 rows, each of whose values is looked up again, by one CTA or another; the two pages hold all keys there are
    kv, page, n, hq = 1000000, 16, 2, 8
    g = torch.Generator().manual_seed(3)
    k, v = torch.randn(2, 1, page, 64, generator=g).half(), torch.randn(2, 1, page, 64, generator=g).half()
    v[1, 0, 5, ::2], v[1, 0, 6, 3], v[1, 0, 7, 7] = float("inf"), -float("inf"), float("nan")
    v[1, 0, 8, 0] = -float("inf")
    cache = mg.KVCache(dev, 2, page, 1, 64, mg.F16, k=dev.array(to_bits(k, mg.F16), mg.F16), v=dev.array(to_bits(v, mg.F16), mg.F16))
    table = np.zeros((3, kv // page), np.int32)
    table[:, 7] = table[1, -1] = 1
    lens = np.array([kv, kv - 3, kv], np.int32)
    batch = mg.PagedBatch(ints(dev, np.arange(4) * n), ints(dev, lens), ints(dev, table), 3, 3 * n, n, table.shape[1])
    q = torch.randn(3 * n, hq, 64, generator=g).half()
    out = dev.empty(3 * n * hq * 64, mg.F16)
    mg.paged_attention(cache, batch, dev.array(to_bits(q, mg.F16), mg.F16), out, hq)
    dev.finish()
    got = from_bits(out.read(np.uint16), mg.F16).view(3 * n, hq, 64)
    want = torch.zeros(64)
    want[::2], want[3], want[7], want[0] = float("inf"), -float("inf"), float("nan"), float("nan")
    odd = ~torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), (~odd).expand(got.shape))
    torch.testing.assert_close(got[..., odd].float(), want[odd].expand(3 * n, hq, -1), equal_nan=True)
