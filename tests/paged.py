"""What the tests of the paged cache share: a random pool of pages, a ragged batch over it, and the
operators restated in 64 bits."""
import numpy as np
import torch

import mvlm_b200 as mg

TORCH = {mg.F16: torch.float16, mg.BF16: torch.bfloat16, mg.F32: torch.float32}
# Unit roundoff: half the spacing of the type's values, relative.
UNIT = {mg.F16: 2.0 ** -11, mg.BF16: 2.0 ** -8, mg.F32: 2.0 ** -24}
TINY = {mg.F16: 2.0 ** -25, mg.BF16: 2.0 ** -134, mg.F32: 2.0 ** -150}  # half the smallest subnormal


def to_bits(x: torch.Tensor, t: int) -> np.ndarray:
    x = x.to(TORCH[t]).contiguous()
    return x.numpy() if t == mg.F32 else x.view(torch.int16).numpy().view(np.uint16)


def from_bits(a: np.ndarray, t: int) -> torch.Tensor:
    a = torch.from_numpy(np.ascontiguousarray(a).copy() if t == mg.F32 else np.ascontiguousarray(a).view(np.int16).copy())
    return a if t == mg.F32 else a.view(TORCH[t])


def ints(dev, a):
    return dev.array(np.ascontiguousarray(a, np.int32), mg.F32)


class Pool:
    """Sequences of new[b] tokens at the end of kv[b], their pages scattered over a pool."""

    def __init__(self, dev, new, kv, kv_heads, dim, page, t, seed=0, spare=3, fill=None, pad_tokens=0, max_q_len=None):
        g = torch.Generator().manual_seed(seed)
        self.dev, self.new, self.kv, self.hk, self.d, self.page, self.t, self.g = dev, list(new), list(kv), kv_heads, dim, page, t, g
        need = [-(-max(k, 0) // page) for k in kv]
        pool = sum(need) + spare
        self.max_pages = max(need + [1])
        order = torch.randperm(pool, generator=g)
        # entries that no token needs are as bad as they can be
        self.table = np.full((len(kv), self.max_pages), 0x7FFFFFF0, np.int32)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = order[at:at + n].numpy()
            at += n
        shape = (pool, kv_heads, page, dim)
        self.k = torch.randn(shape, generator=g).to(TORCH[t])
        self.v = torch.randn(shape, generator=g).to(TORCH[t])
        if fill is not None:  # what the places of no token hold
            held = torch.zeros(pool, page, dtype=torch.bool)
            for b in range(len(kv)):
                for x in range(kv[b]):
                    held[self.table[b, x // page], x % page] = True
            blank = ~held[:, None, :, None].expand(shape)
            self.k[blank] = fill
            self.v[blank] = fill
        self.cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        self.tokens = max(1, int(self.cu[-1]) + pad_tokens)
        self.cache = mg.KVCache(dev, pool, page, kv_heads, dim, t, k=dev.array(to_bits(self.k, t), t), v=dev.array(to_bits(self.v, t), t))
        self.buffers = [ints(dev, self.cu), ints(dev, np.array(kv)), ints(dev, self.table)]
        self.batch = mg.PagedBatch(*self.buffers, len(kv), self.tokens, max_q_len or max(list(new) + [1]), self.max_pages)

    def keys(self, b, which):
        """Sequence b's [kv][heads][dim] in 64 bits."""
        n = self.kv[b]
        pages = torch.from_numpy(self.table[b, : -(-n // self.page)].astype(np.int64))
        return which[pages].transpose(1, 2).reshape(-1, self.hk, self.d)[:n].double()

    def attention(self, q, q_heads, scale, causal=True, window=0):
        """The result in 64 bits and the bound on a kernel's error, for q [tokens][heads][dim]."""
        q = q.double()
        out, tol = torch.zeros_like(q), torch.zeros_like(q)
        u, group = UNIT[self.t], q_heads // self.hk
        for b, n in enumerate(self.new):
            k, v = self.keys(b, self.k), self.keys(b, self.v)
            p = torch.arange(self.kv[b] - n, self.kv[b])[:, None]
            j = torch.arange(self.kv[b])
            seen = torch.ones(n, self.kv[b], dtype=torch.bool)
            if causal:
                seen &= j <= p
            if window:
                seen &= p - j < window
            for h in range(q_heads):
                rows = slice(int(self.cu[b]), int(self.cu[b]) + n)
                s = (q[rows, h] @ torch.nan_to_num(k[:, h // group], 0.0, 0.0, 0.0).T) * scale
                w = torch.softmax(s.masked_fill(~seen, -torch.inf), -1)
                w[~seen.any(-1)] = 0.0
                fine = torch.nan_to_num(v[:, h // group], 0.0, 0.0, 0.0)
                out[rows, h] = w @ fine
                # a key's Inf or NaN reaches exactly the tokens that see it
                odd = v[:, h // group] - fine
                if not bool((odd == 0).all()):
                    for i in range(n):
                        out[rows.start + i, h] += odd[seen[i]].sum(0)
                # weights rounded to the cache's type, the result rounded once more, fp32 scores, exponentials and
                # sums (2^-13 of the result's terms), weights below the type's smallest value
                tol[rows, h] = (2 * u + 2.0 ** -13) * (w @ fine.abs()) + 2.0 ** -24 * (seen.double() @ fine.abs())
        return out, tol


def assert_within(got, want, tol, what=""):
    got, want = got.double(), want.double()
    odd = ~torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN in other places"
    assert torch.equal(got[odd & ~torch.isnan(want)], want[odd & ~torch.isnan(want)]), f"{what}: other infinities"
    err = (got - want).abs()[~odd]
    over = err > tol[~odd]
    assert not bool(over.any()), f"{what}: {int(over.sum())} of {over.numel()} values off, worst {float((err - tol[~odd]).max()):.3e} over its bound"
