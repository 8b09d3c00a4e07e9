"""GPU parity of mgpu_logits_process with a 64-bit restatement: one rounding per operation (four at
most) and one to the logits' type; counts, masks and the maximum's index are exact."""
import numpy as np
import pytest
import torch

import mvlm_b200 as mg
from tests.paged import TINY, TORCH, UNIT, assert_within, from_bits, ints, to_bits

pytestmark = pytest.mark.gpu


def rules_case(dev, rows, n, t, history=0, prompt=True, bias=0, grammar=False, in_place=False, pitch=0, offset=0, best=True,
               out=True, seed=0, allowed=None, x=None, ids=None):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, n, generator=g) * 4.0 if x is None else x).to(TORCH[t])
    want = x.double()
    size = want.abs()
    lens = torch.randint(0, history + 1, (rows,), generator=g)
    lens[0] = history
    kw = {}
    if history:
        if ids is None:
            ids = (torch.rand(rows, history, generator=g) ** 2 * (n + 4)).int() - 2  # some of no token
        pens = torch.stack([0.7 + torch.rand(rows, generator=g), torch.rand(rows, generator=g) - 0.3, torch.rand(rows, generator=g) - 0.3], 1)
        kw |= dict(history=ints(dev, ids.numpy()), history_lens=ints(dev, lens.numpy()), history_ld=history,
                   penalties=dev.array(pens.numpy(), mg.F32))
        prompts = torch.randint(0, history + 1, (rows,), generator=g) if prompt else torch.zeros(rows, dtype=torch.long)
        if prompt:
            kw["prompt_lens"] = ints(dev, prompts.numpy())
        for r in range(rows):
            h = ids[r, : int(lens[r])].long()
            keep = (h >= 0) & (h < n)
            used = torch.bincount(h[keep], minlength=n) > 0
            after = torch.arange(len(h)) >= prompts[r]
            count = torch.bincount(h[keep & after], minlength=n).double()
            again, often, present = (float(v) for v in pens[r])
            want[r] = torch.where(used, torch.where(want[r] > 0, want[r] / again, want[r] * again), want[r])
            size[r] = want[r].abs() + abs(often) * count + abs(present) * (count > 0)
            want[r] = want[r] - often * count - present * (count > 0)
    if bias:
        entries = [int(v) for v in torch.randint(0, bias + 1, (rows,), generator=g)]
        offsets = np.concatenate([[0], np.cumsum(entries)])
        tokens = torch.randint(-1, n + 1, (max(1, int(offsets[-1])),), generator=g)  # some of no token, some twice
        values = torch.randn(len(tokens), generator=g) * 3.0
        kw |= dict(bias_offsets=ints(dev, offsets), bias_tokens=ints(dev, tokens.numpy()), bias_values=dev.array(values.numpy(), mg.F32))
        for r in range(rows):
            last = {int(tokens[i]): float(values[i]) for i in range(offsets[r], offsets[r + 1])}
            for k, v in last.items():
                if 0 <= k < n:
                    want[r, k] += v
                    size[r, k] += abs(v)
    words = (n + 31) // 32
    if grammar or allowed is not None:
        if allowed is None:
            allowed = torch.rand(rows, n, generator=g) < 0.4
        bits = np.zeros((rows, words * 32), np.uint8)
        bits[:, :n] = allowed.numpy()
        bits[:, n:] = np.random.RandomState(seed).randint(0, 2, bits[:, n:].shape)  # bits of no token
        kw["allowed"] = dev.array(np.packbits(bits, axis=1, bitorder="little").view(np.uint32), mg.F32)
        want = want.masked_fill(~allowed, -torch.inf)
    ld, es = n + pitch, mg.TYPE_SIZE[t]
    host = torch.full((rows * ld + offset,), 9.0).to(TORCH[t])
    host[offset:].view(rows, ld)[:, :n] = x
    whole = dev.array(to_bits(host, t), t)
    src = whole.view(offset * es, rows * ld * es).set_format(t, ld=ld)
    dst = src if in_place else dev.empty(rows * n, t) if out else None
    top = dev.create_buffer(rows * 8, np.full(rows * 2, -5, np.int32)) if best else None
    mg.logits_process(dev, src, dst, rows, n, mg.LogitRules(**kw), top)
    dev.finish()
    what = f"rows={rows} n={n} t={t} history={history} bias={bias} grammar={grammar}"
    got = None
    if in_place:
        back = from_bits(whole.read(mg.NP_DTYPE[t]), t)
        assert bool((back[offset:].view(rows, ld)[:, n:] == 9.0).all()) and bool((back[:offset] == 9.0).all()), what
        got = back[offset:].view(rows, ld)[:, :n]
    elif out:
        got = from_bits(dst.read(mg.NP_DTYPE[t]), t).view(rows, n)
    if got is not None:
        assert_within(got, want, UNIT[t] * want.abs().nan_to_num(0, 0, 0) + (1 + UNIT[t]) * 4 * 2.0 ** -24 * size.nan_to_num(0, 0, 0) + TINY[t], what)
    if best:
        pairs = top.read(np.int32).reshape(rows, 2)
        if got is not None:  # what argmax_rows finds in the result, bit for bit
            flat = dev.array(to_bits(got.contiguous(), t), t)
            again = dev.create_buffer(rows * 8)
            mg.argmax_rows(dev, flat, rows, n, n, again)
            dev.finish()
            np.testing.assert_array_equal(pairs, again.read(np.int32).reshape(rows, 2), what)
    return got, (pairs if best else None)


@pytest.mark.parametrize("t", [mg.F32, mg.F16, mg.BF16])
@pytest.mark.parametrize("rows,n", [(1, 1), (1, 31), (3, 257), (2, 51200), (5, 4097), (300, 1000), (1, 200003)])
def test_all_rules(dev, t, rows, n):
    rules_case(dev, rows, n, t, history=77, bias=9, grammar=True)


@pytest.mark.parametrize("t", [mg.F32, mg.F16])
@pytest.mark.parametrize("rules", [{}, dict(history=50), dict(history=50, prompt=False), dict(bias=20), dict(grammar=True),
                                   dict(history=50, grammar=True), dict(history=1), dict(history=5000), dict(bias=300)])
def test_groups_of_rules(dev, t, rules):
    rules_case(dev, 4, 3001, t, **rules)


@pytest.mark.parametrize("t", [mg.F32, mg.BF16])
@pytest.mark.parametrize("pitch,offset", [(0, 0), (8, 0), (1, 0), (0, 1), (5, 3)])
@pytest.mark.parametrize("in_place", [False, True])
def test_pitches_and_alignment(dev, t, pitch, offset, in_place):
    rules_case(dev, 7, 1003, t, history=40, bias=5, grammar=True, in_place=in_place, pitch=pitch, offset=offset)


def test_a_vocabulary_beyond_one_piece(dev):
    # more tokens to a CTA than its shared words: several rounds over the history
    rules_case(dev, 2, 400001, mg.F16, history=3000, bias=50, grammar=True)


def test_one_token_many_times(dev):
    rules_case(dev, 2, 500, mg.F32, history=20000, ids=torch.full((2, 20000), 123, dtype=torch.int32))


def test_only_the_maximum(dev):
    a = rules_case(dev, 3, 5000, mg.F32, history=60, bias=4, grammar=True, seed=3)[1]
    b = rules_case(dev, 3, 5000, mg.F32, history=60, bias=4, grammar=True, seed=3, out=False)[1]
    c = rules_case(dev, 3, 5000, mg.F32, history=60, bias=4, grammar=True, seed=3, best=False)[0]
    np.testing.assert_array_equal(a, b)
    assert c is not None


@pytest.mark.parametrize("t", [mg.F32, mg.F16])
def test_masks_that_leave_nothing_and_odd_values(dev, t):
    n = 700
    allowed = torch.ones(4, n, dtype=torch.bool)
    allowed[0] = False
    allowed[1, 1:] = False
    x = torch.randn(4, n, generator=torch.Generator().manual_seed(5))
    x[2, 5:9] = torch.tensor([float("inf"), -float("inf"), float("nan"), 0.0])
    x[3] = 2.0  # a tie
    allowed[3, :10] = False
    allowed[0, 3], x[0, 3] = False, float("nan")
    got, pairs = rules_case(dev, 4, n, t, allowed=allowed, x=x)
    assert bool((got[0] == -torch.inf).all()) and pairs[0, 0] == 0
    assert pairs[1, 0] == 0 and pairs[3, 0] == 10


def test_refusals(dev):
    x, other = dev.empty(4 * 100, mg.F32), dev.empty(4 * 100, mg.F16)
    small = ints(dev, np.zeros(3))
    four, five = ints(dev, np.zeros(4)), ints(dev, np.zeros(5))
    pens = dev.array(np.ones(12, np.float32), mg.F32)
    hist = ints(dev, np.zeros((4, 7)))

    def refused(out=x, best=None, rows=4, n=100, logits=x, **kw):
        with pytest.raises(mg.MgpuError) as e:
            mg.logits_process(dev, logits, out, rows, n, mg.LogitRules(**kw), best)
        assert e.value.code == mg.ERR_INVALID_ARG

    refused(out=None)
    refused(out=other)
    refused(rows=0)
    refused(n=0)
    refused(rows=5)
    refused(n=101)
    refused(out=x.view(4, x.nbytes - 4).set_format(mg.F32), rows=3)  # overlaps
    refused(best=dev.create_buffer(24))
    refused(history=hist, history_ld=7, penalties=pens)
    refused(history=hist, history_ld=8, history_lens=four, penalties=pens)
    refused(history=hist, history_ld=7, history_lens=small, penalties=pens)
    refused(history=hist, history_ld=7, history_lens=four, penalties=four)
    refused(history=hist, history_ld=7, history_lens=four, penalties=pens, prompt_lens=small)
    refused(penalties=pens)
    refused(bias_offsets=four, bias_tokens=four, bias_values=pens)
    refused(bias_offsets=five)
    refused(bias_tokens=four, bias_values=pens)
    refused(allowed=five)
    mg.logits_process(dev, x, x, 4, 100, mg.LogitRules(), None)
    dev.finish()
