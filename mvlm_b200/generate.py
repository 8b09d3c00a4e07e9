"""A small decoder on the library's operators: batched generation over a paged KV cache.

    python -m mvlm_b200.generate                 # four prompts, one of them with an image's positions

``Decoder`` runs the layers of a Phi-like language model with random Q8_0 weights (RMSNorm, rotary
attention with shared key heads, SiLU-gated MLP): the loop of the reference's moondream2_forward
(src/models/moondream2.cpp:321-549) for a batch of sequences of which each step may bring a chunk of a
prompt or one new token.  ``Session`` holds the sequences: their pages, ids and positions.  A step is

    embeddings -> [norm, qkv, kv_append, paged_attention, out + residual, norm, MLP + residual] x layers
               -> norm, lm_head -> logits_process (penalties, mask, the greedy token)

in which the cache, the attention and the choice of the token stay on the device; eight bytes a
sequence come back.  Embeddings are looked up on the host.
"""
from __future__ import annotations

import argparse
from dataclasses import dataclass, field

import numpy as np

import mvlm_b200 as mg


@dataclass
class Config:
    layers: int = 2
    hidden: int = 512
    heads: int = 8
    kv_heads: int = 4
    head_dim: int = 64
    mlp: int = 1024
    vocab: int = 1000
    sections: tuple = (8, 12, 12)  # pairs that turn by time, height and width
    page_size: int = 16
    num_pages: int = 512
    max_tokens: int = 512  # activation rows of a step
    max_pos: int = 4096
    eps: float = 1e-5


@dataclass
class Sequence:
    ids: list
    positions: np.ndarray  # [3][len(ids)]
    pages: list = field(default_factory=list)
    cached: int = 0  # tokens whose keys and values are in the cache
    prompt: int = 0

    def append(self, token: int):
        self.ids.append(int(token))
        self.positions = np.concatenate([self.positions, np.full((3, 1), self.positions.max() + 1, np.int32)], 1)


class Decoder:
    def __init__(self, dev: mg.Device, cfg: Config, seed: int = 1):
        self.dev, self.cfg, c = dev, cfg, cfg
        if c.heads % c.kv_heads or sum(c.sections) * 2 > c.head_dim:
            raise mg.MgpuError(mg.ERR_INVALID_ARG, "generate: heads or rotary sections do not fit")
        self._seed = seed
        qkv = (c.heads + 2 * c.kv_heads) * c.head_dim
        width = c.heads * c.head_dim
        self.layers = [dict(qkv=self._weight(qkv, c.hidden), out=self._weight(c.hidden, width), up=self._weight(c.mlp, c.hidden),
                            gate=self._weight(c.mlp, c.hidden, dense=True), down=self._weight(c.hidden, c.mlp),
                            norm1=self._ones(c.hidden), norm2=self._ones(c.hidden),
                            cache=mg.KVCache(dev, c.num_pages, c.page_size, c.kv_heads, c.head_dim, mg.F16))
                       for _ in range(c.layers)]
        self.norm, self.head = self._ones(c.hidden), self._weight(c.vocab, c.hidden)
        self.embedding = (np.random.RandomState(seed).randn(c.vocab, c.hidden) * 0.5).astype(np.float16)
        self.rope_table = mg.rope_table(dev, c.max_pos, 2 * sum(c.sections))
        T = c.max_tokens
        self.buf = {k: dev.empty(T * n, mg.F16) for k, n in dict(x=c.hidden, norm=c.hidden, qkv=qkv, q=width, att=width, up=c.mlp).items()}

    def _ones(self, n):
        return self.dev.array(np.ones(n, np.float16).view(np.uint16), mg.F16)

    def _weight(self, rows, cols, dense=False):
        """Random [rows][cols], GGUF Q8_0 blocks (fp16 where the GEMM's epilogue wants a dense operand)."""
        self._seed += 1
        full = self.dev.empty(rows * cols, mg.F32)
        self.dev.fill_normal(full, rows * cols, self._seed, cols ** -0.5)
        if dense:
            w = self.dev.empty(rows * cols, mg.F16)
            self.dev.convert(full, w, rows * cols)
            return w.set_format(mg.F16, mg.LAYOUT_NK, rows, cols, cols)
        w = self.dev.create_buffer(rows * mg.row_bytes(mg.Q8_0, cols), None, mg.Q8_0, mg.LAYOUT_NK, rows, cols)
        self.dev.quantize(full, w, rows * cols, mg.Q8_0)
        return w

    def step(self, ids, positions, batch: mg.PagedBatch, last_rows) -> mg.Buffer:
        """The logits (fp32 [len(last_rows)][vocab]) of the step's rows `last_rows`."""
        c, dev, b, T = self.cfg, self.dev, self.buf, len(ids)
        x = self._rows("x", T, c.hidden)
        x.write(self.embedding[np.asarray(ids)].view(np.uint16))
        norm, up = self._rows("norm", T, c.hidden), self._rows("up", T, c.mlp)
        width, kv = c.heads * c.head_dim, c.kv_heads * c.head_dim
        ld = width + 2 * kv
        qkv = self._rows("qkv", T, ld)
        q, k, v = (b["qkv"].view(2 * at, 2 * (T * ld - at)).set_format(mg.F16, ld=ld) for at in (0, width, width + kv))
        q_rot, att = self._rows("q", T, width), self._rows("att", T, width)
        rope = mg.Rope(self.rope_table, c.max_pos, 2 * sum(c.sections), False, c.sections,
                       dev.array(np.ascontiguousarray(positions, np.int32), mg.F32))
        for w in self.layers:
            mg.dispatch_rms_norm(dev, None, x, norm, w["norm1"], T, c.hidden, c.eps)
            mg.gemm_q(dev, norm, w["qkv"], qkv, T, ld, c.hidden, mg.Q8_0)
            mg.kv_append(w["cache"], batch, q, k, v, q_rot, c.heads, rope)
            mg.paged_attention(w["cache"], batch, q_rot, att, c.heads)
            mg.gemm_fused(dev, att, w["out"], x, T, c.hidden, width, residual=x)
            mg.dispatch_rms_norm(dev, None, x, norm, w["norm2"], T, c.hidden, c.eps)
            mg.gemm_q(dev, norm, w["up"], up, T, c.mlp, c.hidden, mg.Q8_0)
            mg.gemm_silu_gate(dev, norm, w["gate"], up, up, T, c.mlp, c.hidden)
            mg.gemm_fused(dev, up, w["down"], x, T, c.hidden, c.mlp, residual=x)
        S = len(last_rows)
        rows = dev.empty(S * c.hidden, mg.F16)
        for i, r in enumerate(last_rows):
            if mg.lib().mgpu_buf_copy_async(rows.h, i * c.hidden * 2, x.h, int(r) * c.hidden * 2, c.hidden * 2) != mg.OK:
                raise mg.MgpuError(*mg.last_error())
        normed, logits = dev.empty(S * c.hidden, mg.F16), dev.empty(S * c.vocab, mg.F32)
        mg.dispatch_rms_norm(dev, None, rows, normed, self.norm, S, c.hidden, c.eps)
        mg.gemm_q(dev, normed, self.head, logits, S, c.vocab, c.hidden, mg.Q8_0)
        dev.finish()  # the step's own buffers live until here
        return logits

    def _rows(self, name, rows, width):
        return self.buf[name].view(0, rows * width * 2).set_format(mg.F16)


class Session:
    """Sequences in the decoder's cache; ``step`` advances each by a chunk of its prompt or one token."""

    def __init__(self, decoder: Decoder, chunk: int = 128, penalties=(1.1, 0.1, 0.0), allowed: np.ndarray | None = None):
        if chunk < 1:
            raise mg.MgpuError(mg.ERR_INVALID_ARG, f"generate: chunks of {chunk} tokens")
        self.d, self.chunk, self.penalties, self.sequences = decoder, chunk, penalties, []
        self.free = list(range(decoder.cfg.num_pages))[::-1]
        self.allowed = None if allowed is None else np.packbits(
            np.pad(np.asarray(allowed, bool), (0, -len(allowed) % 32)), bitorder="little").view(np.uint32)

    def add(self, ids, positions=None) -> Sequence:
        """A prompt; positions [3][len(ids)] (time, height, width), by default 0, 1, 2, ... on every axis."""
        c, ids = self.d.cfg, [int(i) for i in ids]
        if not ids or min(ids) < 0 or max(ids) >= c.vocab:
            raise mg.MgpuError(mg.ERR_INVALID_ARG, "generate: an empty prompt, or ids outside the vocabulary")
        if len(self.sequences) >= c.max_tokens:
            raise mg.MgpuError(mg.ERR_INVALID_ARG, f"generate: more sequences than a step's {c.max_tokens} rows")
        if positions is None:
            positions = np.tile(np.arange(len(ids), dtype=np.int32), (3, 1))
        positions = np.asarray(positions, np.int32)
        if positions.shape != (3, len(ids)):
            raise mg.MgpuError(mg.ERR_INVALID_ARG, f"generate: positions {positions.shape} of {len(ids)} ids")
        s = Sequence(ids, positions, prompt=len(ids))
        self.sequences.append(s)
        return s

    def release(self, s: Sequence):
        self.free += s.pages
        self.sequences.remove(s)

    def _plan(self):
        """[(sequence, its tokens of this step, its pages with them)] and the pages then left."""
        c, free, plan = self.d.cfg, list(self.free), []
        room = c.max_tokens - len(self.sequences)
        for s in self.sequences:
            n = min(len(s.ids) - s.cached, self.chunk, 1 + room)
            room -= n - 1
            more = -(-(s.cached + n) // c.page_size) - len(s.pages)
            if more > len(free):
                raise mg.MgpuError(mg.ERR_OUT_OF_MEMORY, "generate: no free page")
            plan.append((s, n, s.pages + [free.pop() for _ in range(more)]))
        return plan, free

    def step(self):
        """One step over all sequences; [(sequence, its next token)] for those whose prompts are done, and
        the processed logits, a row for each of them (None where there is none).  An error leaves the
        session as it was: the step may be taken again, for instance after a sequence was released."""
        if not self.sequences:
            return [], None
        c, dev = self.d.cfg, self.d.dev
        plan, free = self._plan()
        ids, positions, starts, lens, done = [], [], [0], [], []
        for s, n, _ in plan:
            ids += s.ids[s.cached:s.cached + n]
            positions.append(s.positions[:, s.cached:s.cached + n])
            starts.append(starts[-1] + n)
            lens.append(s.cached + n)
            if lens[-1] == len(s.ids):
                done.append((s, starts[-1] - 1))
        width = max(len(pages) for _, _, pages in plan)
        table = np.zeros((len(plan), width), np.int32)
        for i, (_, _, pages) in enumerate(plan):
            table[i, :len(pages)] = pages
        batch = mg.PagedBatch(*(dev.array(np.asarray(a, np.int32), mg.F32) for a in (starts, lens, table)), len(lens), len(ids),
                              int(max(np.diff(starts))), width)
        logits = self.d.step(ids, np.concatenate(positions, 1), batch, [r for _, r in done] or [len(ids) - 1])
        out = [(s, t) for (s, _), t in zip(done, self._tokens([s for s, _ in done], logits))]
        # everything is in the cache, and nothing failed
        self.free = free
        for s, n, pages in plan:
            s.cached += n
            s.pages = pages
        for s, t in out:
            s.append(t)
        return out, logits if done else None

    def _tokens(self, sequences, logits):
        """The sequences' greedy tokens, from their rows of the logits, which the rules change in place."""
        rows, c, dev = len(sequences), self.d.cfg, self.d.dev
        if not rows:
            return []
        most = max(len(s.ids) for s in sequences)
        history = np.full((rows, most), -1, np.int32)
        for i, s in enumerate(sequences):
            history[i, :len(s.ids)] = s.ids
        ints = [dev.array(np.asarray(a, np.int32), mg.F32) for a in (history, [len(s.ids) for s in sequences], [s.prompt for s in sequences])]
        rules = mg.LogitRules(history=ints[0], history_lens=ints[1], prompt_lens=ints[2], history_ld=most,
                              penalties=dev.array(np.tile(np.asarray(self.penalties, np.float32), (rows, 1)), mg.F32),
                              allowed=None if self.allowed is None else dev.array(np.tile(self.allowed, (rows, 1)), mg.F32))
        best = dev.create_buffer(8 * rows)
        mg.logits_process(dev, logits, logits, rows, c.vocab, rules, best)
        return [int(t) for t in best.read(np.int32).reshape(rows, 2)[:, 0]]


def image_positions(rows: int, cols: int, text: int) -> np.ndarray:
    """Positions of an image's patches, row by row at one time, and of the words after it."""
    t = np.zeros(rows * cols, np.int32)
    y, x = np.divmod(np.arange(rows * cols, dtype=np.int32), cols)
    after = np.tile(max(rows, cols) + np.arange(text, dtype=np.int32), (3, 1))
    return np.concatenate([np.stack([t, y, x]), after], 1)


def main():
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--tokens", type=int, default=16)
    ap.add_argument("--layers", type=int, default=2)
    ap.add_argument("--seed", type=int, default=1)
    a = ap.parse_args()
    dev = mg.Device(0)
    dev.set_event_mode(0)
    session = Session(Decoder(dev, Config(layers=a.layers), a.seed))
    rng = np.random.RandomState(a.seed)
    prompts = [session.add(rng.randint(0, 1000, n)) for n in (5, 40, 300)]
    prompts.append(session.add(rng.randint(0, 1000, 27 * 27 // 9 + 12), image_positions(9, 9, 12)))
    for _ in range(a.tokens + 3):
        session.step()
    for s in prompts:
        print(f"prompt of {s.prompt}: {s.ids[s.prompt:]}")


if __name__ == "__main__":
    main()
