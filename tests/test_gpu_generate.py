"""The decoder of mvlm_b200.generate: the cache, the attention over it and the logit rules as they run
together.  A prompt taken in chunks, mixed with other sequences' tokens, has to give what one pass over
the whole sequence gives, within the error of its 16-bit activations, and the greedy tokens have to be
the maxima of the processed logits."""
import numpy as np
import pytest

import mvlm_b200 as mg
from mvlm_b200 import generate as G
from tests.numerics import TOL_16, rel_err

pytestmark = pytest.mark.gpu


def test_chunks_and_single_tokens_agree_with_one_pass(dev):
    cfg = G.Config()
    decoder = G.Decoder(dev, cfg)
    rng = np.random.RandomState(3)
    prompts = [(rng.randint(0, cfg.vocab, n), p) for n, p in ((5, None), (93, G.image_positions(9, 9, 12)), (200, None))]
    session = G.Session(decoder, chunk=37, penalties=(1.3, 0.2, 0.1))
    seqs = [session.add(ids, p) for ids, p in prompts]
    last = {}
    for _ in range(12):
        out, logits = session.step()
        if logits is not None:
            values = logits.read(np.float32).reshape(len(out), -1)
            for (s, token), row in zip(out, values):
                assert token == int(np.argmax(row))
                last[id(s)] = row
    assert all(len(s.ids) > s.prompt for s in seqs)
    for s in seqs:  # the same ids at once, without rules on the way
        whole = G.Session(decoder, chunk=512, penalties=(1.3, 0.2, 0.1))
        whole.free = list(range(cfg.num_pages // 2, cfg.num_pages))
        one = whole.add(s.ids[:-1], s.positions[:, :-1])
        one.prompt = s.prompt
        out, logits = whole.step()
        row = logits.read(np.float32)
        assert rel_err(last[id(s)], row) <= TOL_16
    for s in list(seqs):
        session.release(s)
    assert sorted(session.free) == list(range(cfg.num_pages))


def test_grammar_mask_and_repetition(dev):
    cfg = G.Config(layers=1)
    decoder = G.Decoder(dev, cfg, seed=5)
    allowed = np.zeros(cfg.vocab, bool)
    allowed[[7, 70, 700]] = True
    session = G.Session(decoder, penalties=(1.0, 1000.0, 0.0), allowed=allowed)
    s = session.add(np.arange(50) * 7 % cfg.vocab)
    for _ in range(6):
        session.step()
    said = s.ids[s.prompt:]
    assert len(said) == 6 and set(said) == {7, 70, 700}
    # a heavy frequency penalty takes turns among the three
    assert sorted(said[:3]) == sorted(said[3:]) == [7, 70, 700]


def test_no_free_page_is_an_error(dev):
    decoder = G.Decoder(dev, G.Config(layers=1, num_pages=3))
    session = G.Session(decoder)
    session.add(np.zeros(49, int))
    with pytest.raises(mg.MgpuError) as e:
        session.step()
    assert e.value.code == mg.ERR_OUT_OF_MEMORY
