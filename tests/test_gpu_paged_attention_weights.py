"""The weights of mgpu_paged_attention: what their 16 bits leave out.  Small weights count in fp16 too, whose
spacing, 2^-24, stands for 2^-31 of the greatest weight."""
import numpy as np
import pytest
import torch

import mvlm_b200 as mg
from tests.paged import UNIT, assert_within, from_bits, ints, to_bits

pytestmark = pytest.mark.gpu


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
