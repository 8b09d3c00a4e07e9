"""mgpu_paged_attention beyond what one launch or one table of items holds, with the bounds of
test_gpu_paged_attention.py."""
import pytest

import mvlm_b200 as mg
from tests.test_gpu_paged_attention import check

pytestmark = pytest.mark.gpu


def test_more_chunks_than_one_launch_takes(dev):
    # 1024 sequences to a launch; some of one token and some of none between the chunks
    check(dev, [(0, 1, 9, 20)[b % 4] for b in range(1300)], [20 + b % 23 for b in range(1300)], 2, 1, 32, 8, mg.F16)


@pytest.mark.parametrize("causal", [True, False])
def test_more_items_than_the_table_has_entries(dev, causal):
    # two tokens to an item at 128 rows a token: some 3000 items, several to an entry of the table
    check(dev, [5 + b % 3 for b in range(900)], [5 + b % 29 + b % 3 for b in range(900)], 128, 1, 16, 8, mg.BF16, causal=causal)
