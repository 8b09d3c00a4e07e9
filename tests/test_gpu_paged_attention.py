"""GPU parity of mgpu_paged_attention (the reference's dispatch_attention_decode / _prefill,
src/models/moondream2.cpp:424-430, over a paged cache and for ragged batches) with a 64-bit
restatement, within bounds that follow from the roundings the header states."""
import numpy as np
import pytest
import torch

import mvlm_b200 as mg
from tests.paged import TORCH, Pool, assert_within, from_bits, ints, to_bits

pytestmark = pytest.mark.gpu


def attend(dev, pool, q, hq, scale=0.0, causal=True, window=0, pitch=0, offset=0, out_pitch=0, out_offset=0):
    """Runs the kernel on q [tokens][heads][dim]; returns out like it (rows of no sequence: 5)."""
    t, T, width = pool.t, q.shape[0], hq * pool.d
    ld, ldo = width + pitch, width + out_pitch
    host = torch.full((T * ld + offset,), 9.0).to(TORCH[t])
    host[offset:].view(T, ld)[:, :width] = q.reshape(T, width)
    whole = dev.array(to_bits(host, t), t)
    src = whole.view(2 * offset, T * ld * 2).set_format(t, ld=ld)
    back = dev.array(to_bits(torch.full((T * ldo + out_offset,), 5.0), t), t)
    dst = back.view(2 * out_offset, T * ldo * 2).set_format(t, ld=ldo)
    mg.paged_attention(pool.cache, pool.batch, src, dst, hq, scale, causal, window)
    dev.finish()
    res = from_bits(back.read(np.uint16), t)
    assert bool((res[:out_offset] == 5.0).all())
    res = res[out_offset:].view(T, ldo)
    assert bool((res[:, width:] == 5.0).all()), "written beyond its rows"
    return res[:, :width].view(T, hq, pool.d)


def check(dev, new, kv, hq, hk, d, page, t, causal=True, window=0, scale=0.0, spread=2.5, fill=float("nan"), pad_tokens=0, seed=3,
          max_q_len=None, **kw):
    pool = Pool(dev, new, kv, hk, d, page, t, seed, fill=fill, pad_tokens=pad_tokens, max_q_len=max_q_len)
    q = (torch.randn(pool.tokens, hq, d, generator=pool.g) * spread).to(TORCH[t])
    got = attend(dev, pool, q, hq, scale, causal, window, **kw)
    want, tol = pool.attention(q, hq, scale or d ** -0.5, causal, window)
    n = sum(new)
    assert_within(got[:n], want[:n], tol[:n], f"new={new} kv={kv} heads={hq}/{hk} d={d} page={page} t={t} causal={causal} window={window}")
    assert bool((got[n:] == 5.0).all()), "rows of no sequence were written"
    return got


LENGTHS = [1, 2, 7, 8, 63, 64, 65, 127, 128, 129, 255, 257, 700]


@pytest.mark.parametrize("t", [mg.F16, mg.BF16])
@pytest.mark.parametrize("kv", LENGTHS)
def test_single_tokens(dev, t, kv):
    check(dev, [1], [kv], 8, 2, 64, 16, t)


@pytest.mark.parametrize("t", [mg.F16, mg.BF16])
@pytest.mark.parametrize("n,kv", [(1, 1), (2, 2), (5, 5), (16, 20), (17, 17), (63, 64), (64, 64), (65, 70), (128, 128), (129, 300),
                                  (200, 201), (257, 257), (300, 1000), (513, 600)])
def test_chunks(dev, t, n, kv):
    check(dev, [n], [kv], 4, 2, 128, 16, t)


@pytest.mark.parametrize("d", [8, 16, 40, 64, 72, 80, 96, 104, 128])
@pytest.mark.parametrize("n,kv", [(1, 150), (3, 9), (140, 300)])
def test_head_dims(dev, d, n, kv):
    check(dev, [n, 1], [kv, 77], 6, 2, d, 16, mg.F16)


@pytest.mark.parametrize("hq,hk", [(1, 1), (5, 5), (3, 1), (14, 2), (12, 2), (8, 1), (16, 1), (24, 1), (48, 2), (64, 1), (96, 1), (128, 1), (130, 13)])
@pytest.mark.parametrize("n,kv", [(1, 130), (6, 70), (45, 140)])
def test_shared_heads(dev, hq, hk, n, kv):
    check(dev, [n, 2], [kv, 33], hq, hk, 64, 16, mg.BF16)


@pytest.mark.parametrize("page", [8, 16, 24, 40, 48, 64, 72, 128, 136, 256, 1000])
@pytest.mark.parametrize("n", [1, 90])
def test_pages(dev, page, n):
    check(dev, [n, 1, 1], [371, 1, 129], 4, 2, 64, page, mg.F16)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("window", [0, 1, 5, 64, 100, 1000])
@pytest.mark.parametrize("n,kv", [(1, 300), (4, 300), (170, 300), (170, 170)])
def test_masks(dev, causal, window, n, kv):
    check(dev, [n, 1], [kv, 40], 4, 1, 64, 16, mg.F16, causal, window)


def test_ragged_batches(dev):
    check(dev, [1, 33, 0, 1, 200, 1, 2, 0, 1], [50, 400, 12, 1, 200, 777, 2, 0, 300], 8, 2, 128, 16, mg.BF16)
    check(dev, [1] * 70, [13 * b % 500 + 1 for b in range(70)], 4, 4, 64, 16, mg.F16)
    check(dev, [1 if b % 3 else 0 for b in range(1100)], [b % 37 + 1 for b in range(1100)], 2, 1, 64, 8, mg.F16)


@pytest.mark.parametrize("hq,hk,d,kv", [(8, 1, 128, 20011), (1, 1, 64, 40009), (4, 4, 64, 9001)])
def test_long_contexts(dev, hq, hk, d, kv):
    check(dev, [1], [kv], hq, hk, d, 64, mg.BF16)
    check(dev, [1, 1, 1], [kv, 5, kv // 3], hq, hk, d, 16, mg.F16, window=kv // 2)
    check(dev, [9], [kv], hq, hk, d, 32, mg.F16)


def test_rows_that_see_nothing(dev):
    # more new tokens than the sequence is long: the first ones stand before its start
    pool = Pool(dev, [1], [0], 2, 64, 16, mg.F16)
    got = attend(dev, pool, torch.ones(1, 4, 64).half(), 4)
    assert bool((got == 0).all())
    for causal in (True, False):
        pool = Pool(dev, [40, 1], [10, 30], 2, 64, 16, mg.F16, fill=float("nan"))
        q = torch.randn(41, 4, 64, generator=pool.g).half()
        got = attend(dev, pool, q, 4, causal=causal)
        want, tol = pool.attention(q, 4, 0.125, causal)
        assert_within(got, want, tol)
        if causal:
            assert bool((got[:30] == 0).all())


@pytest.mark.parametrize("fill", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("n,kv", [(1, 100), (5, 100), (150, 150), (300, 410)])
def test_odd_values_where_nothing_is_seen(dev, fill, n, kv):
    """NaN and Inf in keys and values reach the tokens that see them, and no other."""
    for which, at in (("k", kv - 1), ("v", kv - 1), ("v", kv - n), ("v", max(0, kv - n // 2 - 1))):
        pool = Pool(dev, [n], [kv], 1, 64, 16, mg.F16, fill=fill)
        x = getattr(pool, which)
        if which == "k":
            fill_at = slice(None)
            if n == 1:
                continue  # the token's own key: everything is NaN or one-hot by definition
        else:
            fill_at = slice(3, 6)
        x[pool.table[0, at // 16], 0, at % 16, fill_at] = fill
        (pool.cache.k if which == "k" else pool.cache.v).write(to_bits(x, mg.F16))
        q = torch.randn(n, 4, 64, generator=pool.g).half()
        got = attend(dev, pool, q, 4)
        want, tol = pool.attention(q, 4, 0.125)
        sees = torch.arange(kv - n, kv) >= at
        rows = ~sees if which == "k" else slice(None)
        assert_within(got[rows], want[rows], tol[rows], f"{which} {at}")


def test_odd_values_outside_a_window(dev):
    pool = Pool(dev, [3], [500], 2, 64, 16, mg.BF16, fill=float("inf"))
    for x in range(440):
        pool.v[pool.table[0, x // 16], :, x % 16] = float("nan")
        pool.k[pool.table[0, x // 16], :, x % 16] = float("nan")
    pool.cache.k.write(to_bits(pool.k, mg.BF16))
    pool.cache.v.write(to_bits(pool.v, mg.BF16))
    q = torch.randn(3, 2, 64, generator=pool.g).bfloat16()
    got = attend(dev, pool, q, 2, window=50)
    want, tol = pool.attention(q, 2, 0.125, window=50)
    assert_within(got, want, tol)


@pytest.mark.parametrize("n,kv", [(1, 200), (150, 200)])
def test_scores_of_any_size(dev, n, kv):
    # one key far above the rest, ever larger maxima along the sequence, all scores equal
    check(dev, [n], [kv], 4, 2, 64, 16, mg.F16, spread=60.0)
    check(dev, [n], [kv], 4, 2, 64, 16, mg.BF16, spread=0.0)
    pool = Pool(dev, [n], [kv], 1, 64, 16, mg.F16)
    for x in range(kv):
        pool.k[pool.table[0, x // 16], 0, x % 16] = 0.01 * x
    pool.cache.k.write(to_bits(pool.k, mg.F16))
    for sign in (1.0, -1.0):
        q = torch.full((n, 2, 64), 4.0 * sign).half()
        want, tol = pool.attention(q, 2, 0.125)
        # scores of about 64: their fp32 error, 2^-18, is in every weight
        assert_within(attend(dev, pool, q, 2), want, tol)


@pytest.mark.parametrize("n,kv", [(1, 90), (140, 150)])
@pytest.mark.parametrize("pitch,offset,out_pitch,out_offset", [(512, 0, 0, 0), (8, 8, 8, 8), (1, 0, 1, 0), (0, 1, 0, 3), (2, 2, 4, 4)])
def test_pitches_and_alignment(dev, n, kv, pitch, offset, out_pitch, out_offset):
    check(dev, [n, 1], [kv, 20], 4, 2, 64, 16, mg.F16, pitch=pitch, offset=offset, out_pitch=out_pitch, out_offset=out_offset)


def test_scale_and_padding_rows(dev):
    check(dev, [1, 2], [80, 90], 4, 2, 64, 16, mg.F16, scale=0.3, pad_tokens=5)
    check(dev, [130, 2], [180, 90], 4, 2, 64, 16, mg.BF16, scale=0.05, pad_tokens=200, max_q_len=400)
    check(dev, [1, 1], [80, 90], 4, 2, 64, 16, mg.F16, max_q_len=300)  # the host's bound may be loose


def test_same_bits_every_time(dev):
    for new, kv in (([1, 1, 1], [5000, 64, 900]), ([200, 1], [3000, 70])):
        pool = Pool(dev, new, kv, 2, 128, 16, mg.BF16)
        q = torch.randn(pool.tokens, 8, 128, generator=pool.g).bfloat16()
        first = attend(dev, pool, q, 8)
        for _ in range(5):
            assert torch.equal(attend(dev, pool, q, 8), first)


def test_offsets_beyond_32_bits(dev):
    """A cache of more than 2^32 bytes and 2^31 elements a side, a sequence in its last pages."""
    pages, page, hk, d = 131073 + 8, 16, 8, 128
    side = dev.create_buffer(pages * hk * page * d * 2)
    cache = mg.KVCache(dev, pages, page, hk, d, mg.F16, k=side, v=dev.create_buffer(pages * hk * page * d * 2))
    for n, kv in ((1, 100), (100, 100)):
        g = torch.Generator().manual_seed(n)
        table = np.arange(pages - 7, pages, dtype=np.int32)[::-1].copy()
        batch = mg.PagedBatch(ints(dev, [0, kv]), ints(dev, [kv]), ints(dev, table), 1, kv, kv, 7)
        x = [torch.randn(kv, hk * d, generator=g).half() for _ in range(2)]
        mg.kv_append(cache, batch, None, *[dev.array(to_bits(y, mg.F16), mg.F16) for y in x], None, 0)
        q = torch.randn(n, 16 * d, generator=g).half()
        out = dev.empty(n * 16 * d, mg.F16)
        batch = mg.PagedBatch(ints(dev, [0, n]), ints(dev, [kv]), ints(dev, table), 1, n, n, 7)
        mg.paged_attention(cache, batch, dev.array(to_bits(q, mg.F16), mg.F16), out, 16)
        dev.finish()
        k, v = (y.view(kv, hk, d).double().repeat_interleave(2, 1) for y in x)
        s = torch.einsum("thd,jhd->htj", q.view(n, 16, d).double(), k) * d ** -0.5
        seen = torch.arange(kv) <= torch.arange(kv - n, kv)[:, None]
        w = torch.softmax(s.masked_fill(~seen, -torch.inf), -1)
        want = torch.einsum("htj,jhd->thd", w, v)
        tol = (2.0 ** -10 + 2.0 ** -13) * torch.einsum("htj,jhd->thd", w, v.abs()) + 2.0 ** -24 * v.abs().sum(0)
        assert_within(from_bits(out.read(np.uint16), mg.F16).view(n, 16, d), want, tol)


def test_another_stream_and_a_captured_graph(dev):
    import torch as th
    pool = Pool(dev, [1, 1], [300, 40], 2, 64, 16, mg.F16)
    q = torch.randn(2, 4, 64, generator=pool.g).half()
    src, dst = dev.array(to_bits(q, mg.F16), mg.F16), dev.empty(2 * 256, mg.F16)
    stream = th.cuda.Stream()
    dev.set_stream(stream.cuda_stream)
    try:
        mg.paged_attention(pool.cache, pool.batch, src, dst, 4)
        dev.finish()
        want, tol = pool.attention(q, 4, 0.125)
        assert_within(from_bits(dst.read(np.uint16), mg.F16).view(2, 4, 64), want, tol)
    finally:
        dev.set_stream(None)
    dev.capture_begin()
    mg.paged_attention(pool.cache, pool.batch, src, dst, 4)
    graph = dev.capture_end()
    for kv in ([299, 1], [17, 40], [300, 39]):  # the graph follows the lengths
        pool.kv = kv
        pool.buffers[1].write(np.array(kv, np.int32))
        graph.launch()
        dev.finish()
        want, tol = pool.attention(q, 4, 0.125)
        assert_within(from_bits(dst.read(np.uint16), mg.F16).view(2, 4, 64), want, tol)


@pytest.mark.parametrize("n", [1, 150])
def test_contents_that_do_not_fit_are_reported(dev, n):
    for spoil in ("page", "negative page", "length", "negative length", "too many new", "rows"):
        pool = Pool(dev, [n, 2], [200, 90], 2, 64, 16, mg.F16)
        q = torch.randn(pool.tokens, 4, 64, generator=pool.g).half()
        want, tol = pool.attention(q, 4, 0.125)
        if spoil == "page":
            pool.buffers[2].write(np.array([pool.k.shape[0]], np.int32), offset=12)
        elif spoil == "negative page":
            pool.buffers[2].write(np.array([-7], np.int32), offset=12)
        elif spoil == "length":
            pool.buffers[1].write(np.array([2 ** 31 - 1], np.int32))
        elif spoil == "negative length":
            pool.buffers[1].write(np.array([-1], np.int32))
        elif spoil == "too many new":
            pool.buffers[0].write(np.array([0, n + 1 if n == 1 else 0, pool.tokens], np.int32))
            pool.batch.c.max_q_len = 1
        else:
            pool.buffers[0].write(np.array([0, n, n + 3], np.int32))
        src, dst = dev.array(to_bits(q, mg.F16), mg.F16), dev.empty(pool.tokens * 256, mg.F16)
        mg.paged_attention(pool.cache, pool.batch, src, dst, 4)
        with pytest.raises(mg.MgpuError) as e:
            dev.finish()
        assert e.value.code == mg.ERR_INVALID_ARG, spoil
        dev.finish()
        if spoil not in ("too many new", "rows"):  # the other sequence has its result
            got = from_bits(dst.read(np.uint16), mg.F16).view(-1, 4, 64)
            assert_within(got[n:], want[n:], tol[n:], spoil)


def test_refusals(dev):
    pool = Pool(dev, [2, 3], [10, 20], 2, 64, 16, mg.F16)
    T = pool.tokens
    q, out = dev.empty(T * 256, mg.F16), dev.empty(T * 256, mg.F16)

    def refused(q=q, out=out, heads=4, code=mg.ERR_INVALID_ARG, batch=pool.batch, **kw):
        with pytest.raises(mg.MgpuError) as e:
            mg.paged_attention(pool.cache, batch, q, out, heads, **kw)
        assert e.value.code == code

    refused(heads=3)
    refused(heads=0)
    refused(heads=8)  # q too small
    refused(heads=2 * 129, code=mg.ERR_UNSUPPORTED)
    refused(q=dev.empty(T * 256, mg.BF16))
    refused(out=dev.empty(T * 256, mg.F32))
    refused(out=q)
    refused(out=pool.cache.k, heads=2)
    refused(out=dev.empty(T * 256 - 1, mg.F16))
    refused(q=None)
    refused(window=-1)
    refused(scale=-1.0)
    refused(scale=float("nan"))
    b = pool.buffers
    refused(batch=mg.PagedBatch(*b, 2, 0, 3, pool.max_pages))
    refused(batch=mg.PagedBatch(*b, 3, T, 3, pool.max_pages))
    refused(batch=mg.PagedBatch(b[0], b[1], None, 2, T, 3, pool.max_pages))
    refused(batch=mg.PagedBatch(*b, 2, T, 0, pool.max_pages))
    refused(batch=mg.PagedBatch(*b, 2, T, 3, pool.max_pages + 1))
    dev.finish()
