"""The limits of mgpu_logits_process: rows beyond one launch's, more marked tokens than a round lists,
histories and biases beyond what a token's word counts.  Values against the restatement of
test_gpu_logit_rules.py, with its tolerances."""
import numpy as np
import pytest
import torch

import mvlm_b200 as mg
from tests.paged import ints
from tests.test_gpu_logit_rules import rules_case

pytestmark = pytest.mark.gpu


def test_more_rows_than_one_launch_takes(dev):
    rules_case(dev, 8203, 37, mg.F16, history=5, bias=3, grammar=True)


@pytest.mark.parametrize("t", [mg.F32, mg.BF16])
def test_more_marked_tokens_than_a_round_lists(dev, t):
    # a CTA's range of some 7500 tokens, most of which the history holds
    ids = torch.stack([torch.randperm(30000, generator=torch.Generator().manual_seed(r))[:25000] for r in range(200)]).int()
    rules_case(dev, 200, 30000, t, history=25000, bias=7, grammar=True, ids=ids)


def test_most_biases_of_a_row(dev):
    # 2047 entries are a row's most: the rest is skipped and reported, other rows keep theirs
    n = 4000
    counts = [2047, 2060, 3]
    offsets = np.concatenate([[0], np.cumsum(counts)])
    tokens = np.concatenate([np.arange(c) for c in counts])
    x, best = dev.array(np.zeros(3 * n, np.float32), mg.F32), dev.create_buffer(24)
    rules = mg.LogitRules(bias_offsets=ints(dev, offsets), bias_tokens=ints(dev, tokens),
                          bias_values=dev.array((1.0 + np.arange(len(tokens))).astype(np.float32), mg.F32))
    out = dev.empty(3 * n, mg.F32)
    mg.logits_process(dev, x, out, 3, n, rules, best)
    with pytest.raises(mg.MgpuError) as e:
        dev.finish()
    assert e.value.code == mg.ERR_INVALID_ARG
    dev.finish()  # reported once
    got = out.read(np.float32).reshape(3, n)
    want = np.zeros((3, n), np.float32)
    for r in range(3):
        k = min(counts[r], 2047)
        want[r, :k] = 1.0 + offsets[r] + np.arange(k)
    np.testing.assert_array_equal(got, want)
    np.testing.assert_array_equal(best.read(np.int32).reshape(3, 2)[:, 0], [2046, 2046, 2])


def test_histories_too_long_to_count(dev):
    x, lens, pens = dev.empty(100, mg.F32), ints(dev, np.zeros(1)), dev.array(np.ones(3, np.float32), mg.F32)
    hist = dev.create_buffer(4 << 20)
    with pytest.raises(mg.MgpuError) as e:
        mg.logits_process(dev, x, x, 1, 100, mg.LogitRules(history=hist, history_lens=lens, history_ld=1 << 20, penalties=pens))
    assert e.value.code == mg.ERR_UNSUPPORTED
    mg.logits_process(dev, x, x, 1, 100, mg.LogitRules(history=hist, history_lens=lens, history_ld=(1 << 20) - 1, penalties=pens))
    dev.finish()
