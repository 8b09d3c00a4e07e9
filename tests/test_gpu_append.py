"""GPU parity of mgpu_kv_append and mgpu_rope_table (dispatch_rope_apply and kv_cache_append of the
reference, src/models/moondream2.cpp:302-314, :406-420, over a paged cache) with 64-bit
restatements.  Values that are not rotated have to be the rounded inputs bit for bit; a rotated one
is a sum of two products in fp32, rounded once."""
import numpy as np
import pytest
import torch

import mvlm_b200 as mg
from tests.paged import TINY, TORCH, UNIT, Pool, assert_within, from_bits, ints, to_bits

pytestmark = pytest.mark.gpu


def rotated(x, angle, interleaved):
    """x [tokens][heads][dim] (64 bits), angle {cos, sin} [tokens][pairs][2]; and the bound's magnitudes."""
    rot = 2 * angle.shape[1]
    c, s = angle[:, None, :, 0], angle[:, None, :, 1]
    a, b = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
    y, size = x.clone(), torch.zeros_like(x)
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., a] * s + x[..., b] * c
    size[..., a] = size[..., b] = x[..., a].abs() + x[..., b].abs()
    return y, size


def append_case(dev, new, kv, hq, hk, d, page, t, src, rot, interleaved=False, axes=1, positions=False, pitch=0, offset=0,
                in_place=False, seed=1, pad_tokens=0):
    pool = Pool(dev, new, kv, hk, d, page, t, seed, pad_tokens=pad_tokens)
    g, T = pool.g, pool.tokens
    x, bufs = {}, {}
    for name, heads in (("q", hq), ("k", hk), ("v", hk)):
        x[name] = torch.randn(T, heads * d, generator=g).to(TORCH[src])
        ld = heads * d + pitch
        host = torch.full((T * ld + offset,), 7.0).to(TORCH[src])
        host[offset:].view(T, ld)[:, : heads * d] = x[name]
        whole = dev.array(to_bits(host, src), src)
        es = mg.TYPE_SIZE[src]
        bufs[name] = whole.view(offset * es, T * ld * es).set_format(src, ld=ld)
        bufs[name]._whole = whole
    most = max(kv + [1]) + 5
    pairs = rot // 2
    sections = [pairs] if axes == 1 else [pairs // 2, pairs - pairs // 2] if axes == 2 else [pairs // 4, pairs // 3, pairs - pairs // 4 - pairs // 3]
    place = torch.cat([torch.arange(k - n, k) for n, k in zip(new, kv)] + [torch.zeros(pad_tokens, dtype=torch.long)])
    pos = torch.stack([place] * axes)
    if positions:
        pos = torch.randint(0, most, (axes, T), generator=g)
    rope, angle = None, torch.zeros(T, 0, 2, dtype=torch.float64)
    if rot:
        table = mg.rope_table(dev, most, rot, 10000.0)
        host = torch.from_numpy(table.read(np.float32)).view(most, pairs, 2).double()
        axis = torch.repeat_interleave(torch.arange(axes), torch.tensor(sections))
        angle = host[pos[axis].T, torch.arange(pairs)]
        rope = mg.Rope(table, most, rot, interleaved, sections, ints(dev, pos.numpy()) if positions else None)
    qt = src if in_place else t
    q_out = bufs["q"] if in_place else dev.array(to_bits(torch.full((T, hq * d), 3.0), qt), qt)
    mg.kv_append(pool.cache, pool.batch, bufs["q"], bufs["k"], bufs["v"], q_out, hq, rope)
    dev.finish()

    covered = sum(new)
    what = f"new={new} kv={kv} hq={hq} hk={hk} d={d} rot={rot} t={t} src={src}"
    # queries: the first `covered` rows
    want, size = rotated(x["q"].double().view(T, hq, d), angle, interleaved)
    if in_place:
        got = from_bits(q_out._whole.read(mg.NP_DTYPE[qt]), qt)[offset:].view(T, -1)[:, : hq * d].view(T, hq, d)
    else:
        got = from_bits(q_out.read(mg.NP_DTYPE[qt]), qt).view(T, hq, d)
    bound = UNIT[qt] * want.abs() + (1 + UNIT[qt]) * 2.0 ** -22 * size + TINY[qt]
    assert_within(got[:covered], want[:covered], bound[:covered], "q " + what)
    assert torch.equal(got[:covered, :, rot:], x["q"].view(T, hq, d)[:covered, :, rot:].float().to(TORCH[qt])), "q rest " + what
    if pad_tokens and not in_place:
        assert bool((got[covered:] == 3.0).all()), "rows of no sequence " + what
    # the cache: each new token's slot, and nothing else
    kw, ks = rotated(x["k"].double().view(T, hk, d), angle, interleaved)
    k_old, v_old = pool.k.clone(), pool.v.clone()
    kc = from_bits(pool.cache.k.read(np.uint16), t).view(pool.k.shape)
    vc = from_bits(pool.cache.v.read(np.uint16), t).view(pool.k.shape)
    i = 0
    for b, n in enumerate(new):
        for p in range(kv[b] - n, kv[b]):
            at = (int(pool.table[b, p // page]), slice(None), p % page)
            bound = UNIT[t] * kw[i].abs() + (1 + UNIT[t]) * 2.0 ** -22 * ks[i] + TINY[t]
            assert_within(kc[at], kw[i], bound, "k " + what)
            assert torch.equal(kc[at][:, rot:], x["k"][i].view(hk, d)[:, rot:].float().to(TORCH[t])), "k rest " + what
            assert torch.equal(vc[at], x["v"][i].view(hk, d).float().to(TORCH[t])), "v " + what
            k_old[at], v_old[at] = kc[at], vc[at]
            i += 1
    assert torch.equal(kc, k_old) and torch.equal(vc, v_old), "places of no new token were written: " + what


@pytest.mark.parametrize("t", [mg.F16, mg.BF16])
@pytest.mark.parametrize("src", [mg.F32, mg.F16, mg.BF16])
def test_types(dev, t, src):
    append_case(dev, [1, 5], [9, 37], 8, 2, 64, 16, t, src, 64)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,rot", [(64, 32), (64, 64), (128, 128), (128, 96), (80, 80), (72, 24), (8, 4), (40, 2), (128, 126), (64, 0)])
def test_head_dims_and_partial_rotation(dev, interleaved, d, rot):
    append_case(dev, [3, 1], [20, 1], 6, 3, d, 8, mg.F16, mg.F32, rot, interleaved)


@pytest.mark.parametrize("axes", [1, 2, 3])
@pytest.mark.parametrize("interleaved", [False, True])
def test_positions_of_several_axes(dev, axes, interleaved):
    append_case(dev, [40], [40], 4, 4, 64, 16, mg.F16, mg.F16, 64, interleaved, axes, positions=True)


@pytest.mark.parametrize("page", [8, 24, 64, 200])
def test_pages_and_ragged_sequences(dev, page):
    append_case(dev, [1, 0, 61, 7, 1], [1, 30, 100, 7, 200], 4, 1, 64, page, mg.BF16, mg.BF16, 64)


@pytest.mark.parametrize("seqs", [31, 32, 33, 70, 1025])
def test_many_sequences(dev, seqs):
    append_case(dev, [1 if b % 7 else 0 for b in range(seqs)], [b % 19 + 1 for b in range(seqs)], 2, 1, 8, 8, mg.F16, mg.F32, 8)


@pytest.mark.parametrize("pitch,offset", [(64, 0), (8, 8), (1, 0), (0, 1), (3, 5)])
@pytest.mark.parametrize("src", [mg.F32, mg.F16])
def test_pitches_and_alignment(dev, pitch, offset, src):
    append_case(dev, [9, 1], [12, 5], 4, 2, 64, 16, mg.F16, src, 32, pitch=pitch, offset=offset)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("pitch", [0, 1])
def test_queries_in_place(dev, interleaved, pitch):
    append_case(dev, [9, 1], [12, 5], 4, 2, 64, 16, mg.F16, mg.F32, 32, interleaved, pitch=pitch, in_place=True)


def test_rows_of_no_sequence_are_left_alone(dev):
    append_case(dev, [2, 1], [5, 9], 4, 2, 64, 16, mg.F16, mg.F32, 64, pad_tokens=4)


def test_rope_table(dev):
    most, rot = 70001, 64
    got = torch.from_numpy(mg.rope_table(dev, most, rot, 1e6).read(np.float32)).view(most, rot // 2, 2).double()
    angle = torch.arange(most, dtype=torch.float64)[:, None] * 1e6 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    want = torch.stack([angle.cos(), angle.sin()], -1)
    # one rounding to fp32, and the angle's own rounding in fp64 (7e4 * 2^-51)
    assert bool(((got - want).abs() <= 2.0 ** -24 * want.abs() + 1e-10).all())


def test_contents_that_do_not_fit_are_reported(dev):
    for spoil in ("page", "negative page", "length", "too many new", "before the start", "position"):
        pool = Pool(dev, [2, 3], [10, 20], 2, 64, 16, mg.F16, max_q_len=3)
        T = pool.tokens
        x = dev.array(np.ones((T, 128), np.float32), mg.F32)
        table = mg.rope_table(dev, 32, 64)
        positions = np.zeros((1, T), np.int32)
        if spoil == "page":
            pool.buffers[2].write(np.array([pool.k.shape[0]], np.int32))
        elif spoil == "negative page":
            pool.buffers[2].write(np.array([-1], np.int32))
        elif spoil == "length":
            pool.buffers[1].write(np.array([2 ** 31 - 1], np.int32))
        elif spoil == "too many new":
            pool.batch.c.max_q_len = 1
        elif spoil == "before the start":
            pool.buffers[1].write(np.array([1], np.int32))
        else:
            positions[0, 0] = 32
        rope = mg.Rope(table, 32, 64, positions=ints(dev, positions))
        mg.kv_append(pool.cache, pool.batch, None, x, x, None, 0, rope)
        with pytest.raises(mg.MgpuError) as e:
            dev.finish()
        assert e.value.code == mg.ERR_INVALID_ARG, spoil
        dev.finish()  # the status was consumed
        if spoil == "too many new":
            continue
        vc = from_bits(pool.cache.v.read(np.uint16), mg.F16).view(pool.v.shape)  # the other sequence's tokens are there
        for p in range(17, 20):
            assert bool((vc[pool.table[1, p // 16], :, p % 16] == 1.0).all()), spoil


def test_refusals(dev):
    pool = Pool(dev, [2, 3], [10, 20], 2, 64, 16, mg.F16)
    T = pool.tokens
    kv = dev.array(np.ones((T, 128), np.float32), mg.F32)
    q = dev.array(np.ones((T, 256), np.float32), mg.F32)
    table = mg.rope_table(dev, 32, 64)

    def refused(fn, code=mg.ERR_INVALID_ARG):
        with pytest.raises(mg.MgpuError) as e:
            fn()
        assert e.value.code == code

    b, c = pool.batch, pool.cache
    refused(lambda: mg.kv_append(c, b, q, kv, kv, None, 4))
    refused(lambda: mg.kv_append(c, b, q, kv, kv, dev.empty(T * 256 - 1, mg.F16), 4))
    refused(lambda: mg.kv_append(c, b, q, kv, kv, q, 0))
    refused(lambda: mg.kv_append(c, b, None, kv.view(0, kv.nbytes - 4).set_format(mg.F32), kv, None, 0))
    refused(lambda: mg.kv_append(c, b, None, kv, kv.view(0, kv.nbytes).set_format(mg.Q8_0, mg.LAYOUT_NK), None, 0))
    refused(lambda: mg.kv_append(c, b, q, kv, kv, q.view(4, q.nbytes - 4).set_format(mg.F32), 2))  # overlaps q
    refused(lambda: mg.kv_append(c, b, None, c.k, kv, None, 0))  # the cache as a source
    refused(lambda: mg.kv_append(c, b, None, kv, kv, None, 0, mg.Rope(table, 33, 64)))
    refused(lambda: mg.kv_append(c, b, None, kv, kv, None, 0, mg.Rope(table, 32, 63)))
    refused(lambda: mg.kv_append(c, b, None, kv, kv, None, 0, mg.Rope(table, 16, 128)))
    refused(lambda: mg.kv_append(c, b, None, kv, kv, None, 0, mg.Rope(table, 32, 64, sections=[16, 15])))
    refused(lambda: mg.kv_append(c, b, None, kv, kv, None, 0, mg.Rope(table, 32, 64, sections=[-1, 33])))
    refused(lambda: mg.Rope(table, 32, 64, sections=[8, 8, 8, 8]))
    refused(lambda: mg.kv_append(c, b, None, kv, kv, None, 0, mg.Rope(table, 32, 64, positions=ints(dev, np.zeros(T - 1)))))
    bad = mg.PagedBatch(*pool.buffers, 3, T, 3, pool.max_pages)
    refused(lambda: mg.kv_append(c, bad, None, kv, kv, None, 0))
    bad = mg.PagedBatch(pool.buffers[0], None, pool.buffers[2], 2, T, 3, pool.max_pages)
    refused(lambda: mg.kv_append(c, bad, None, kv, kv, None, 0))
    for args in ((4, 12, 2, 64, mg.F16), (4, 16, 2, 60, mg.F16), (4, 16, 2, 64, mg.F32), (0, 16, 2, 64, mg.F16), (4, 16, 0, 64, mg.F16)):
        refused(lambda: mg.KVCache(dev, *args))
    refused(lambda: mg.KVCache(dev, 4, 16, 2, 256, mg.F16), mg.ERR_UNSUPPORTED)
    refused(lambda: mg.KVCache(dev, 4, 16, 2, 64, mg.F16, k=kv))
    refused(lambda: mg.KVCache(dev, 400, 16, 2, 64, mg.F16, k=kv, v=q))
    dev.finish()
