"""What mgpu_logits_process makes of bias offsets that do not fit: no access leaves the buffers, a row whose
end comes before its start has no biases, and other rows keep theirs."""
import numpy as np
import pytest

import mvlm_b200 as mg
from tests.paged import ints

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("offsets,rows_with", [
    ([5, -2 ** 31, 3, 7], {1: (0, 3), 2: (3, 7)}),
    ([-2 ** 31, 4, -5, 2 ** 31 - 1], {0: (0, 4), 2: (0, 9)}),
    ([2 ** 31 - 1, -2 ** 31, 2 ** 31 - 1, 0], {1: (0, 9)}),
    ([9, 8, 1, 1], {}),
])
def test_bias_offsets_that_do_not_fit(dev, offsets, rows_with):
    n, rows = 4000, 3
    x, out, best = dev.array(np.zeros(rows * n, np.float32), mg.F32), dev.empty(rows * n, mg.F32), dev.create_buffer(8 * rows)
    tokens, values = np.arange(9) * 400 + 7, (1.0 + np.arange(9)).astype(np.float32)
    rules = mg.LogitRules(bias_offsets=ints(dev, np.array(offsets, np.int64).astype(np.int32)), bias_tokens=ints(dev, tokens),
                          bias_values=dev.array(values, mg.F32))
    mg.logits_process(dev, x, out, rows, n, rules, best)
    dev.finish()
    want = np.zeros((rows, n), np.float32)
    for r, (a, b) in rows_with.items():
        want[r, tokens[a:b]] = values[a:b]
    np.testing.assert_array_equal(out.read(np.float32).reshape(rows, n), want)
    np.testing.assert_array_equal(best.read(np.int32).reshape(rows, 2)[:, 0], want.argmax(1))
