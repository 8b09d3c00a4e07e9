"""Captured graphs and the device's scratch: a graph keeps the tickets and partials of the arena that it
was captured with, so later calls that need a larger one must leave that one in place.  A replayed step
has to give the bits of the same call made directly."""
import numpy as np
import pytest
import torch

import mvlm_b200 as mg
from tests.paged import Pool, assert_within, from_bits, ints, to_bits

pytestmark = pytest.mark.gpu


@pytest.fixture()
def fresh():
    """A device whose scratch nothing has grown yet."""
    d = mg.Device(0)
    d.set_event_mode(0)
    yield d
    d.finish()


def chunk(dev, seed=9):
    """A call whose rows many CTAs share: its pieces take some 40 MB."""
    pool = Pool(dev, [300], [4000], 2, 128, 16, mg.BF16, seed)
    q = torch.randn(300, 8, 128, generator=pool.g).bfloat16()
    out = dev.empty(300 * 8 * 128, mg.BF16)
    mg.paged_attention(pool.cache, pool.batch, dev.array(to_bits(q, mg.BF16), mg.BF16), out, 8)
    dev.finish()
    want, tol = pool.attention(q, 8, 128 ** -0.5)
    assert_within(from_bits(out.read(np.uint16), mg.BF16).view(300, 8, 128), want, tol)


def test_a_captured_decode_step_outlives_larger_calls(fresh):
    pool = Pool(fresh, [1, 1, 1], [9000, 70, 2500], 2, 64, 16, mg.F16)
    q = torch.randn(3, 8, 64, generator=pool.g).half()
    src, dst = fresh.array(to_bits(q, mg.F16), mg.F16), fresh.empty(3 * 512, mg.F16)
    mg.paged_attention(pool.cache, pool.batch, src, dst, 8)
    fresh.finish()
    first = dst.read(np.uint16)
    want, tol = pool.attention(q, 8, 0.125)
    assert_within(from_bits(first, mg.F16).view(3, 8, 64), want, tol)
    fresh.capture_begin()
    mg.paged_attention(pool.cache, pool.batch, src, dst, 8)
    graph = fresh.capture_end()
    for _ in range(3):
        chunk(fresh)
        # what a freed arena's place would be given to
        other = [fresh.array(np.full(1 << 19, 0xFFFF, np.uint16), mg.F16) for _ in range(8)]
        dst.write(np.zeros(3 * 512, np.uint16))
        graph.launch()
        fresh.finish()
        np.testing.assert_array_equal(dst.read(np.uint16), first)
        assert all((o.read(np.uint16) == 0xFFFF).all() for o in other)
    mg.paged_attention(pool.cache, pool.batch, src, dst, 8)  # with the arena of now
    fresh.finish()
    np.testing.assert_array_equal(dst.read(np.uint16), first)


def test_captured_logit_rules_outlive_larger_calls(fresh):
    rows, n = 3, 51200
    x = np.random.RandomState(2).randn(rows, n).astype(np.float32)
    logits, best = fresh.array(x, mg.F32), fresh.create_buffer(8 * rows)
    hist = np.ascontiguousarray(np.argsort(-x, 1)[:, :2], np.int32)
    rules = mg.LogitRules(history=ints(fresh, hist), history_lens=ints(fresh, [2] * rows), history_ld=2,
                          penalties=fresh.array(np.tile(np.array([1.0, 100.0, 0.0], np.float32), (rows, 1)), mg.F32))
    want = np.argsort(-x, 1)[:, 2]
    mg.logits_process(fresh, logits, None, rows, n, rules, best)
    fresh.finish()
    fresh.capture_begin()
    mg.logits_process(fresh, logits, None, rows, n, rules, best)
    graph = fresh.capture_end()
    for _ in range(3):
        chunk(fresh)
        best.write(np.full(2 * rows, -1, np.int32))
        graph.launch()
        fresh.finish()
        np.testing.assert_array_equal(best.read(np.int32).reshape(rows, 2)[:, 0], want)
