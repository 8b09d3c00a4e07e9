"""The serving operators refuse results that would lie in what other CTAs of the call still read."""
import numpy as np
import pytest

import mvlm_b200 as mg
from tests.paged import Pool, ints

pytestmark = pytest.mark.gpu


def refused(call):
    with pytest.raises(mg.MgpuError) as e:
        call()
    assert e.value.code == mg.ERR_INVALID_ARG


def inside(buf, at, nbytes):
    return buf.view(at, nbytes).set_format(mg.F32)


def test_logit_rules(dev):
    rows, n = 4, 1000
    size = rows * n * 4
    x, out, best = dev.empty(rows * n, mg.F32), dev.empty(rows * n, mg.F32), dev.create_buffer(8 * rows)
    pens = dev.array(np.ones(12, np.float32), mg.F32)
    lens, offsets, words = ints(dev, np.zeros(4)), ints(dev, np.zeros(5)), ints(dev, np.full((rows, 32), -1))
    hist, tokens, values = ints(dev, np.zeros((rows, 7))), ints(dev, np.zeros(3)), dev.array(np.zeros(3, np.float32), mg.F32)
    every = dict(history=hist, history_lens=lens, prompt_lens=lens, history_ld=7, penalties=pens, bias_offsets=offsets, bias_tokens=tokens,
                 bias_values=values, allowed=words)
    need = dict(history=112, history_lens=16, prompt_lens=16, penalties=48, bias_offsets=20, bias_tokens=12, bias_values=12, allowed=512)
    for name, nbytes in need.items():
        for where in (out, best) if nbytes <= best.nbytes else (out,):
            for at in (0, where.nbytes - nbytes):
                kw = every | {name: inside(where, at, nbytes)}
                refused(lambda: mg.logits_process(dev, x, out, rows, n, mg.LogitRules(**kw), best))
        # in place: the logits' own places
        kw = every | {name: inside(x, size - nbytes, nbytes)}
        refused(lambda: mg.logits_process(dev, x, x, rows, n, mg.LogitRules(**kw), best))
    for b in (inside(x, 16, 32), inside(out, size - 32, 32)):
        refused(lambda: mg.logits_process(dev, x, out, rows, n, mg.LogitRules(**every), b))
    refused(lambda: mg.logits_process(dev, x, None, rows, n, mg.LogitRules(**every), inside(x, 0, 32)))
    # neighbours are fine
    whole = dev.create_buffer(2 * size + 64)
    x2, out2, best2 = inside(whole, 0, size), inside(whole, size, size), inside(whole, 2 * size, 32)
    kw = every | dict(history_lens=inside(whole, 2 * size + 32, 16), prompt_lens=inside(whole, 2 * size + 48, 16))
    whole.write(np.zeros(2 * size // 4 + 16, np.int32))
    mg.logits_process(dev, x2, out2, rows, n, mg.LogitRules(**kw), best2)
    dev.finish()


def test_paged_cache(dev):
    pool = Pool(dev, [2, 3], [10, 20], 2, 64, 16, mg.F16)
    T, c, b = pool.tokens, pool.cache, pool.buffers
    q, out = dev.empty(T * 256, mg.F16), dev.empty(T * 256, mg.F16)
    kv = dev.empty(T * 128, mg.F16)
    sizes = (12, 8, 4 * 2 * pool.max_pages)
    table = mg.rope_table(dev, 4, 8)
    for i in range(3):
        for where in (out, c.k, c.v):
            bufs = list(b)
            bufs[i] = inside(where, where.nbytes - sizes[i], sizes[i])
            batch = mg.PagedBatch(*bufs, 2, T, 3, pool.max_pages)
            refused(lambda: mg.kv_append(c, batch, q, kv, kv, out, 4))
            if where is out:
                refused(lambda: mg.paged_attention(c, batch, q, out, 4))
    for where in (out, c.k, c.v):
        refused(lambda: mg.kv_append(c, pool.batch, q, kv, kv, out, 4, mg.Rope(inside(where, 0, 4 * 8 * 4), 4, 8)))
        refused(lambda: mg.kv_append(c, pool.batch, q, kv, kv, out, 4, mg.Rope(table, 4, 8, positions=inside(where, 0, 4 * T))))
    dev.finish()


def test_queries_in_place_beside_keys_and_values(dev):
    pool = Pool(dev, [2, 3], [10, 20], 2, 64, 16, mg.F16)
    T, c, b = pool.tokens, pool.cache, pool.batch
    ld = 256 + 128 + 128
    qkv = dev.array(np.zeros(T * ld + ld, np.uint16), mg.F16)

    def view(column, row=0, pitch=ld):
        at = 2 * (row * ld + column)
        return qkv.view(at, qkv.nbytes - at).set_format(mg.F16, ld=pitch)

    q = view(0)
    for k, v in ((view(256), view(384)), (view(384), view(256)), (view(256, 1), view(384, 1))):
        mg.kv_append(c, b, q, k, v, q, 4)
    mg.kv_append(c, b, view(256), view(0, 1), view(128, 1), view(256), 4)  # queries at the end of the rows
    for k, v in ((view(255), view(384)), (view(256), view(0)), (view(256), view(385)), (view(100), view(384)), (view(256, 0, ld + 8), view(384)),
                 (view(256), view(384, 0, 128)), (view(384).view(0, T * ld).set_format(mg.BF16, ld=ld), view(384))):
        refused(lambda: mg.kv_append(c, b, q, k, v, q, 4))
    dev.finish()
