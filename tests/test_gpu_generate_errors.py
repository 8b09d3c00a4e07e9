"""A session of mvlm_b200.generate goes on after a step without a free page: what it then says is what a
session that never failed says."""
import numpy as np
import pytest

import mvlm_b200 as mg
from mvlm_b200 import generate as G
from tests.numerics import TOL_16, rel_err

pytestmark = pytest.mark.gpu


def test_goes_on_after_running_out_of_pages(dev):
    decoder = G.Decoder(dev, G.Config(layers=1, num_pages=6), seed=7)
    rng = np.random.RandomState(1)
    ids = rng.randint(0, 1000, 45)
    session = G.Session(decoder, chunk=40)
    first, second = session.add(ids), session.add(rng.randint(0, 1000, 60))
    session.step()  # three pages each; the next has room for the first alone
    with pytest.raises(mg.MgpuError) as e:
        session.step()
    assert e.value.code == mg.ERR_OUT_OF_MEMORY
    session.release(second)
    (s, _), = session.step()[0]
    out, logits = session.step()
    assert s is first and out[0][0] is first and len(first.ids) == 47
    row = logits.read(np.float32)
    session.release(first)
    again = G.Session(decoder, chunk=512)
    whole = again.add(first.ids[:46])
    whole.prompt = 45
    out, logits = again.step()
    assert rel_err(row, logits.read(np.float32)) <= TOL_16
