"""The bookkeeping of mvlm_b200.generate.Session on the host, with a decoder that computes nothing: a step
that fails leaves the session as it was, and every token of every sequence is taken exactly once."""
import types

import numpy as np
import pytest

import mvlm_b200 as mg
from mvlm_b200 import generate as G


class Stub:
    """Records what each sequence's pages would hold, as kv_append would write it; row r's token is r."""

    def __init__(self, monkeypatch, **cfg):
        self.cfg = G.Config(**cfg)
        self.dev = types.SimpleNamespace(array=lambda a, t: np.array(a), create_buffer=lambda n: Stub.Best(n // 8))
        self.held, self.fail = {}, False
        monkeypatch.setattr(mg, "PagedBatch", lambda *a: types.SimpleNamespace(args=a))
        monkeypatch.setattr(mg, "LogitRules", lambda **kw: kw)
        monkeypatch.setattr(mg, "logits_process", self.rules)
        self.fail_rules = False

    class Best:
        def __init__(self, rows):
            self.rows = rows

        def read(self, t):
            return np.stack([np.arange(self.rows), np.zeros(self.rows, int)], 1).astype(t).reshape(-1)

    def rules(self, *a):
        if self.fail_rules:
            raise mg.MgpuError(mg.ERR_CUDA, "stub")

    def step(self, ids, positions, batch, last_rows):
        starts, lens, table, n_seqs, n_tokens, most, width = batch.args
        assert n_tokens == len(ids) <= self.cfg.max_tokens and positions.shape == (3, n_tokens)
        assert (np.diff(starts) > 0).all() and most == np.diff(starts).max() and table.shape == (n_seqs, width)
        if self.fail:
            raise mg.MgpuError(mg.ERR_CUDA, "stub")
        for b in range(n_seqs):
            for i in range(starts[b], starts[b + 1]):
                x = lens[b] - starts[b + 1] + i
                self.held[int(table[b, x // self.cfg.page_size]), int(x % self.cfg.page_size)] = ids[i]
        return object()


def cached(stub, s):
    return [stub.held.get((s.pages[x // stub.cfg.page_size], x % stub.cfg.page_size)) for x in range(s.cached)]


def state(session):
    return sorted(session.free), [(list(s.ids), s.cached, list(s.pages), s.positions.shape) for s in session.sequences]


def test_no_free_page_loses_no_token(monkeypatch):
    stub = Stub(monkeypatch, num_pages=4, page_size=16)
    session = G.Session(stub, chunk=20)
    a, b = session.add(range(1, 26)), session.add(range(100, 140))
    session.step()  # two pages each; the next has room for the first alone
    before = state(session)
    with pytest.raises(mg.MgpuError) as e:
        session.step()
    assert e.value.code == mg.ERR_OUT_OF_MEMORY and state(session) == before
    session.release(b)
    while a.cached < 40:
        session.step()
    assert cached(stub, a) == a.ids[:a.cached] and a.ids[:25] == list(range(1, 26))
    assert sorted(session.free + a.pages) == [0, 1, 2, 3]


@pytest.mark.parametrize("what", ["fail", "fail_rules"])
def test_a_step_that_fails_can_be_taken_again(monkeypatch, what):
    stub = Stub(monkeypatch)
    session = G.Session(stub, chunk=7)
    seqs = [session.add(range(n)) for n in (3, 20, 7)]
    for _ in range(6):
        before = state(session)
        setattr(stub, what, True)
        if what == "fail" or any(len(s.ids) - s.cached <= 7 for s in seqs):
            with pytest.raises(mg.MgpuError):
                session.step()
            assert state(session) == before
        setattr(stub, what, False)
        session.step()
    for s in seqs:
        assert s.cached == len(s.ids) - 1 and cached(stub, s) == s.ids[:s.cached]


def test_as_many_sequences_as_rows(monkeypatch):
    stub = Stub(monkeypatch, max_tokens=4, num_pages=64)
    session = G.Session(stub)
    seqs = [session.add(range(9)) for _ in range(4)]
    with pytest.raises(mg.MgpuError):
        session.add(range(9))
    for _ in range(12):
        session.step()
    for s in seqs:
        assert s.cached == 12 and cached(stub, s) == s.ids[:12]


def test_refusals(monkeypatch):
    stub = Stub(monkeypatch)
    with pytest.raises(mg.MgpuError):
        G.Session(stub, chunk=0)
    session = G.Session(stub)
    for args in (([],), ([-1],), ([stub.cfg.vocab],), ([1, 2], np.zeros((3, 1), np.int32)), ([1], np.zeros((1, 1), np.int32))):
        with pytest.raises(mg.MgpuError) as e:
            session.add(*args)
        assert e.value.code == mg.ERR_INVALID_ARG
    assert session.step() == ([], None) and not session.sequences
