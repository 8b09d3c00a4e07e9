"""The serving operators around the matmul path, as they are measured: appending a step's keys and
values to a paged cache with the position rotation, attention of new tokens over that cache, and
the rules (penalties, biases, grammar masks) applied to the logits before a token is chosen.

``listed()`` and ``draw()`` give cases, ``prepare()`` what a program holds before a call, ``run()``
one pass: in plain torch, or through the package where ``own`` is true.  ``exact()`` restates each
operator in 64 bits.
"""
import math
import random

import torch

own = False

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
SIZE = {"f16": 2, "bf16": 2, "f32": 4}


def listed():
    return [
        # One decode step of the repository's own language model (32 heads of 64, half of each head
        # rotated) after a 760-token prompt: the projections' fp32 outputs go into an fp16 cache.
        dict(name="append 1 token", op="append", dtype="f16", src="f32", seqs=1, new=1, past=760, q_heads=32, kv_heads=32,
             dim=64, rot=32, interleaved=False, axes=1, page=16),
        # The same model's image prompt, 729 patches and 32 words, positions along time, height and width.
        dict(name="append image prompt", op="append", dtype="f16", src="f16", seqs=1, new=761, past=0, q_heads=32,
             kv_heads=32, dim=64, rot=64, interleaved=False, axes=3, page=16),
        # A prefill step of a serving engine: five prompts, shared key heads, pairs side by side.
        dict(name="append 5 prompts", op="append", dtype="bf16", src="bf16", seqs=5, new=4096, past=500, q_heads=32,
             kv_heads=8, dim=128, rot=128, interleaved=True, axes=1, page=64),
        # The decode step's attention for one sequence of the repository's model: latency.
        dict(name="decode 1 sequence", op="attend", dtype="f16", seqs=1, new=1, chunks=0, past=900, q_heads=32, kv_heads=32,
             dim=64, page=16, causal=True, window=0),
        # A serving batch of 64 conversations of different lengths, one new token each.
        dict(name="decode 64 sequences", op="attend", dtype="bf16", seqs=64, new=1, chunks=0, past=4097, q_heads=32,
             kv_heads=8, dim=128, page=16, causal=True, window=0),
        # One new token at the end of a very long document.
        dict(name="decode long context", op="attend", dtype="bf16", seqs=1, new=1, chunks=0, past=131001, q_heads=32,
             kv_heads=8, dim=128, page=64, causal=True, window=0),
        # The image prompt of the repository's model, all 761 tokens new.
        dict(name="prompt 761", op="attend", dtype="f16", seqs=1, new=761, chunks=1, past=0, q_heads=32, kv_heads=32, dim=64,
             page=16, causal=True, window=0),
        # A chunk of a long prompt over what earlier chunks left in the cache; seven queries to a key head.
        dict(name="chunk 512 over 16K", op="attend", dtype="bf16", seqs=1, new=512, chunks=1, past=16001, q_heads=28,
             kv_heads=4, dim=128, page=32, causal=True, window=0),
        # A step of an engine that mixes chunks of new prompts with running conversations.
        dict(name="mixed batch", op="attend", dtype="f16", seqs=24, new=300, chunks=4, past=4000, q_heads=32, kv_heads=8,
             dim=128, page=16, causal=True, window=0),
        # A long prompt's second half in one chunk: the largest amount of arithmetic.
        dict(name="chunk 4096 over 4096", op="attend", dtype="bf16", seqs=1, new=4096, chunks=1, past=4096, q_heads=32,
             kv_heads=8, dim=128, page=64, causal=True, window=0),
        # The rules on one sequence's logits over the repository's vocabulary: latency.
        dict(name="rules 1 row", op="rules", dtype="f32", rows=1, vocab=51200, history=400, bias=0, grammar=False),
        # A large batch, each row with its history, its biases and its grammar's mask.
        dict(name="rules 256 rows", op="rules", dtype="f32", rows=256, vocab=51200, history=2048, bias=16, grammar=True),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    while True:
        case = _draw(rng)
        w = work(case)
        # no dearer than the largest listed cases, the plain form's padded score matrix included
        if w["bytes"] > 6e8 or w["flops"] > 4e11:
            continue
        if case["op"] == "attend":
            q, kv = _lengths(case)
            if len(q) * max(q) * max(kv) * case["q_heads"] > 1.1e9 or len(q) * max(kv) * case["kv_heads"] * case["dim"] > 3e8:
                continue
        return case


def _draw(rng):
    op = rng.choice(["append", "attend", "attend", "attend", "rules"])
    dtype = rng.choice(["f16", "bf16"])
    if op == "rules":
        return dict(op=op, dtype=rng.choice(["f16", "bf16", "f32"]), rows=_log(rng, 1, 256), vocab=_log(rng, 8000, 200000),
                    history=_log(rng, 1, 8000), bias=rng.choice([0, _log(rng, 1, 300)]), grammar=rng.random() < 0.5)
    kv_heads, group = rng.choice([(32, 1), (8, 4), (4, 7), (4, 8), (2, 6), (1, 16), (8, 1), (16, 2)])
    dim, page = rng.choice([64, 64, 80, 96, 128, 128, 128]), rng.choice([8, 16, 16, 32, 48, 64, 128])
    heads = dict(q_heads=kv_heads * group, kv_heads=kv_heads, dim=dim, page=page)
    if op == "append":
        rot = rng.choice([dim, dim // 2])
        return dict(op=op, dtype=dtype, src=rng.choice([dtype, "f32"]), seqs=_log(rng, 1, 64), new=_log(rng, 1, 4096),
                    past=_log(rng, 1, 2000), rot=rot, interleaved=rng.random() < 0.5, axes=rng.choice([1, 3]), **heads)
    kind = rng.choice(["decode", "chunk", "mixed"])
    window = rng.choice([0, 0, 0, _log(rng, 64, 4096)])
    if kind == "decode":
        return dict(op=op, dtype=dtype, seqs=_log(rng, 1, 128), new=1, chunks=0, past=_log(rng, 1, 131072), causal=True,
                    window=window, **heads)
    if kind == "chunk":
        return dict(op=op, dtype=dtype, seqs=1, new=_log(rng, 2, 4096), chunks=1, past=_log(rng, 1, 32768),
                    causal=rng.random() < 0.8, window=window, **heads)
    seqs = _log(rng, 2, 32)
    return dict(op=op, dtype=dtype, seqs=seqs, new=_log(rng, 2, 1024), chunks=max(1, seqs // 4), past=_log(rng, 1, 8192),
                causal=True, window=window, **heads)


def _lengths(case):
    """The sequences' new tokens and their lengths with them: ragged, the same for every seed."""
    rng = random.Random(97)
    new, kv = [], []
    for i in range(case["seqs"]):
        full = i == 0  # the first has the case's own sizes
        n = case["new"] if case["op"] == "append" or i < case["chunks"] else 1
        n = n if full else max(1, int(n * rng.uniform(0.1, 1.0)))
        p = case["past"] if full else int(case["past"] * rng.uniform(0.05, 1.0))
        new.append(n)
        kv.append(p + n)
    return new, kv


def _histories(case):
    rng = random.Random(53)
    return [case["history"]] + [int(case["history"] * rng.uniform(0.0, 1.0)) for _ in range(case["rows"] - 1)]


def _pairs_seen(n, kv, causal, window):
    """Scores that one head needs for n new tokens at the end of kv: keys j <= p, and p - j < window."""
    if not causal and not window:
        return n * kv
    total = 0
    for p in range(kv - n, kv):
        last = p if causal else kv - 1
        total += last + 1 - (max(0, p - window + 1) if window else 0)
    return total


def work(case):
    """Each input read once, each output written once; the arithmetic of the definition."""
    e = SIZE[case["dtype"]]
    if case["op"] == "rules":
        n, rows = case["vocab"], case["rows"]
        data = 2 * rows * n * e + 4 * sum(_histories(case)) + 8 * rows * case["bias"] + (rows * ((n + 31) // 32) * 4 if case["grammar"] else 0)
        return {"bytes": data, "flops": rows * n}
    new, kv = _lengths(case)
    tokens, d = sum(new), case["dim"]
    if case["op"] == "append":
        elems = tokens * (case["q_heads"] + 2 * case["kv_heads"]) * d
        table = tokens * case["rot"] * 4
        return {"bytes": elems * (SIZE[case["src"]] + e) + table + 4 * tokens, "flops": 3 * tokens * (case["q_heads"] + case["kv_heads"]) * case["rot"]}
    seen = [k if not case["window"] else min(k, n - 1 + case["window"]) for n, k in zip(new, kv)]
    scores = sum(_pairs_seen(n, k, case["causal"], case["window"]) for n, k in zip(new, kv))
    return {"bytes": 2 * tokens * case["q_heads"] * d * e + 2 * sum(seen) * case["kv_heads"] * d * e,
            "flops": 4 * scores * case["q_heads"] * d}


# ---------------------------------------------------------------------------- inputs
def _paged(case, g):
    """A pool of pages with what earlier steps left in it, and a batch's view of it."""
    dev, t = "cuda", TYPES[case["dtype"]]
    new, kv = _lengths(case)
    page = case["page"]
    need = [-(-k // page) for k in kv]
    pool, widest = sum(need) + 3, max(need)
    shape = (pool, case["kv_heads"], page, case["dim"])
    order = torch.randperm(pool, generator=g, device=dev).to(torch.int32)
    table = torch.zeros(len(new), widest, dtype=torch.int32, device=dev)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    return dict(case=case, k_cache=torch.randn(shape, generator=g, device=dev, dtype=t),
                v_cache=torch.randn(shape, generator=g, device=dev, dtype=t), table=table,
                cu_q=torch.tensor(starts, dtype=torch.int32, device=dev), kv_lens=torch.tensor(kv, dtype=torch.int32, device=dev),
                tokens=starts[-1], most_new=max(new), most_kv=max(kv))


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    state = {"append": _prepare_append, "attend": _prepare_attend, "rules": _prepare_rules}[case["op"]](case, g)
    if own:
        _handles(state)
    return state


def _sections(case):
    pairs = case["rot"] // 2
    if case["axes"] == 1:
        return [pairs]
    return [pairs // 4, (pairs - pairs // 4) // 2, pairs - pairs // 4 - (pairs - pairs // 4) // 2]


def _prepare_append(case, g):
    s = _paged(case, g)
    src, d, tokens = TYPES[case["src"]], case["dim"], s["tokens"]
    for name, heads in (("q", case["q_heads"]), ("k", case["kv_heads"]), ("v", case["kv_heads"])):
        s[name] = torch.randn(tokens, heads * d, generator=g, device="cuda", dtype=torch.float32).to(src)
    most = s["most_kv"] + 64
    rate = 10000.0 ** (-torch.arange(0, case["rot"], 2, dtype=torch.float64, device="cuda") / case["rot"])
    angle = torch.arange(most, dtype=torch.float64, device="cuda")[:, None] * rate
    s["rope"] = torch.stack([angle.cos(), angle.sin()], -1).float().contiguous()  # [positions][pairs][2]
    place = torch.cat([torch.arange(k - n, k, device="cuda") for n, k in zip(*_lengths(case))])
    if case["axes"] == 3:  # an image's rows of 27 patches: time stands still, height and width run
        s["positions"] = torch.stack([place // 729, place % 729 // 27, place % 27]).to(torch.int32)
    else:
        s["positions"] = place.to(torch.int32)[None]
    return s


def _prepare_attend(case, g):
    s = _paged(case, g)
    # trained heads attend sharply: scores spread by about 2.5
    s["q"] = (torch.randn(s["tokens"], case["q_heads"] * case["dim"], generator=g, device="cuda") * 2.5).to(TYPES[case["dtype"]])
    return s


def _prepare_rules(case, g):
    rows, n = case["rows"], case["vocab"]
    lens = _histories(case)
    s = dict(case=case, logits=(torch.randn(rows, n, generator=g, device="cuda") * 3.0).to(TYPES[case["dtype"]]))
    # texts repeat themselves: ids crowd at the low end
    s["history"] = (torch.rand(rows, max(lens + [1]), generator=g, device="cuda") ** 3 * n).to(torch.int32).clamp_(max=n - 1)
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    s["prompts"] = (s["lens"] // 2).to(torch.int32)
    u = torch.rand(rows, 3, generator=g, device="cuda")
    s["penalties"] = torch.stack([1.0 + 0.3 * u[:, 0], 0.5 * u[:, 1], 0.5 * u[:, 2]], 1).contiguous()
    if case["bias"]:
        b = case["bias"]
        s["bias_offsets"] = torch.arange(0, (rows + 1) * b, b, dtype=torch.int32, device="cuda")
        step = max(1, n // b)  # a row's tokens differ
        jump = (torch.rand(rows, b, generator=g, device="cuda") * step).to(torch.int32)
        s["bias_tokens"] = (torch.arange(b, dtype=torch.int32, device="cuda") * step + jump).reshape(-1).contiguous()
        s["bias_values"] = torch.randn(rows * b, generator=g, device="cuda") * 5.0
    if case["grammar"]:  # one token in eight or so may come next
        words = (rows, (n + 31) // 32)
        s["allowed"] = torch.full(words, -1, dtype=torch.int32, device="cuda")
        for _ in range(3):
            s["allowed"] &= torch.randint(-2**31, 2**31, words, generator=g, device="cuda").to(torch.int32)
    return s


# ---------------------------------------------------------------------------- through the package
_device = None


def _handles(s):
    """The handles that a serving program makes once and keeps beside its buffers."""
    global _device
    import mvlm_b200 as mg
    if _device is None:
        _device = mg.Device(0)
        _device.set_event_mode(0)
        _device.set_stream(torch.cuda.current_stream().cuda_stream or 1)  # 1: the legacy default stream
    d, case, kinds = _device, s["case"], {torch.float16: mg.F16, torch.bfloat16: mg.BF16, torch.float32: mg.F32}

    def wrap(x, type_=None, ld=0):
        return d.wrap(x.data_ptr(), x.numel() * x.element_size(), kinds.get(x.dtype, mg.F32) if type_ is None else type_, ld=ld)

    if case["op"] == "rules":
        rows = case["rows"]
        s["out"] = torch.empty_like(s["logits"])
        s["best"] = torch.empty(rows, 2, dtype=torch.int32, device="cuda")
        bias = dict(bias_offsets=wrap(s["bias_offsets"]), bias_tokens=wrap(s["bias_tokens"]), bias_values=wrap(s["bias_values"])) if case["bias"] else {}
        rules = mg.LogitRules(history=wrap(s["history"]), history_lens=wrap(s["lens"]), prompt_lens=wrap(s["prompts"]),
                              history_ld=s["history"].shape[1], penalties=wrap(s["penalties"]),
                              allowed=wrap(s["allowed"]) if case["grammar"] else None, **bias)
        s["call"] = (d, wrap(s["logits"]), wrap(s["out"]), rows, case["vocab"], rules, wrap(s["best"]))
        return
    cache = mg.KVCache(d, s["k_cache"].shape[0], case["page"], case["kv_heads"], case["dim"], kinds[s["k_cache"].dtype],
                       k=wrap(s["k_cache"]), v=wrap(s["v_cache"]))
    batch = mg.PagedBatch(cu_q=wrap(s["cu_q"]), kv_lens=wrap(s["kv_lens"]), page_table=wrap(s["table"]), n_seqs=case["seqs"],
                          n_tokens=s["tokens"], max_q_len=s["most_new"], max_pages=s["table"].shape[1])
    s["out"] = torch.empty(s["tokens"], case["q_heads"] * case["dim"], dtype=TYPES[case["dtype"]], device="cuda")
    if case["op"] == "append":
        rope = mg.Rope(table=wrap(s["rope"]), max_pos=s["rope"].shape[0], rot_dim=case["rot"], interleaved=case["interleaved"],
                       sections=_sections(case), positions=wrap(s["positions"]))
        s["call"] = (cache, batch, wrap(s["q"]), wrap(s["k"]), wrap(s["v"]), wrap(s["out"]), case["q_heads"], rope)
    else:
        s["call"] = (cache, batch, wrap(s["q"]), wrap(s["out"]), case["q_heads"], case["dim"] ** -0.5, case["causal"], case["window"])


def run(state):
    op = state["case"]["op"]
    if own:
        import mvlm_b200 as mg
        if op == "append":
            mg.kv_append(*state["call"])
            return {"q": state["out"], "k_cache": state["k_cache"], "v_cache": state["v_cache"]}
        if op == "attend":
            mg.paged_attention(*state["call"])
            return {"out": state["out"]}
        mg.logits_process(*state["call"])
        return {"logits": state["out"], "token": state["best"][:, 0]}
    return {"append": _append, "attend": _attend, "rules": _rules}[op](state)


# ---------------------------------------------------------------------------- plain forms
def _places(s):
    """Sequence and index of every new token, and its slot in the cache."""
    t = torch.arange(s["tokens"], device="cuda")
    seq = torch.searchsorted(s["cu_q"].long(), t, right=True) - 1
    starts, ends = s["cu_q"].long()[seq], s["cu_q"].long()[seq + 1]
    index = s["kv_lens"].long()[seq] - (ends - starts) + t - starts
    return seq, index, t - starts


def _rotate(x, cos, sin, rot, interleaved):
    """x [tokens][heads][dim]; cos, sin [tokens][1][rot / 2]."""
    r = x[..., :rot]
    a, b = (r[..., 0::2], r[..., 1::2]) if interleaved else (r[..., : rot // 2], r[..., rot // 2:])
    y, z = a * cos - b * sin, a * sin + b * cos
    r = torch.stack([y, z], -1).flatten(-2) if interleaved else torch.cat([y, z], -1)
    return torch.cat([r, x[..., rot:]], -1)


def _append(s):
    case, t, d = s["case"], TYPES[s["case"]["dtype"]], s["case"]["dim"]
    axis = torch.repeat_interleave(torch.arange(case["axes"], device="cuda"), torch.tensor(_sections(case), device="cuda"), output_size=case["rot"] // 2)
    at = s["positions"].long()[axis].T  # [tokens][pairs]
    angle = s["rope"][at, torch.arange(case["rot"] // 2, device="cuda")]
    cos, sin = angle[..., 0][:, None], angle[..., 1][:, None]
    q = _rotate(s["q"].float().view(s["tokens"], -1, d), cos, sin, case["rot"], case["interleaved"])
    k = _rotate(s["k"].float().view(s["tokens"], -1, d), cos, sin, case["rot"], case["interleaved"])
    seq, index, _ = _places(s)
    page, slot = s["table"].long()[seq, index // case["page"]], index % case["page"]
    s["k_cache"][page, :, slot] = k.to(t)
    s["v_cache"][page, :, slot] = s["v"].float().view(s["tokens"], -1, d).to(t)
    return {"q": q.reshape(s["tokens"], -1).to(t), "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _attend(s):
    case, d = s["case"], s["case"]["dim"]
    b, hk, group, most, kv = case["seqs"], case["kv_heads"], case["q_heads"] // case["kv_heads"], s["most_new"], s["most_kv"]
    pages = s["table"].long()
    k = s["k_cache"][pages].float().transpose(1, 2).reshape(b, hk, -1, d)[:, :, :kv]
    v = s["v_cache"][pages].float().transpose(1, 2).reshape(b, hk, -1, d)[:, :, :kv]
    seq, index, row = _places(s)
    q = torch.zeros(b, most, hk, group, d, device="cuda")
    q[seq, row] = s["q"].float().view(-1, hk, group, d)
    scores = (q.permute(0, 2, 3, 1, 4).reshape(b, hk, group * most, d) @ k.transpose(2, 3)).mul_(d ** -0.5).view(b, hk, group, most, kv)
    j = torch.arange(kv, device="cuda")
    lens = s["kv_lens"].long()[:, None, None]
    p = lens - (s["cu_q"][1:] - s["cu_q"][:-1]).long()[:, None, None] + torch.arange(most, device="cuda")[:, None]
    seen = j < lens
    if case["causal"]:
        seen = seen & (j <= p)
    if case["window"]:
        seen = seen & (p - j < case["window"])
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True).clamp_(min=-3e38)
    scores = scores.sub_(top).exp_()
    out = scores.view(b, hk, group * most, kv) @ v
    out = out / scores.sum(-1).view(b, hk, group * most, 1)
    out = out.view(b, hk, group, most, d).permute(0, 3, 1, 2, 4)[seq, row]
    return {"out": out.reshape(s["tokens"], -1).to(TYPES[case["dtype"]])}


def _rules(s):
    case, x = s["case"], s["logits"].float()
    rows, n = case["rows"], case["vocab"]
    i = torch.arange(s["history"].shape[1], device="cuda")
    ids = s["history"].long()
    said = torch.zeros(rows, n, device="cuda").scatter_add_(1, ids, (i < s["lens"][:, None]).float())
    count = torch.zeros(rows, n, device="cuda").scatter_add_(1, ids, ((i < s["lens"][:, None]) & (i >= s["prompts"][:, None])).float())
    again, often, present = s["penalties"][:, :1], s["penalties"][:, 1:2], s["penalties"][:, 2:]
    x = torch.where(said > 0, torch.where(x > 0, x / again, x * again), x)
    x = x - often * count - present * (count > 0)
    if case["bias"]:
        x = x.scatter_add(1, s["bias_tokens"].long().view(rows, -1), s["bias_values"].view(rows, -1))
    if case["grammar"]:
        bits = (s["allowed"][:, :, None] >> torch.arange(32, device="cuda", dtype=torch.int32)) & 1
        x = torch.where(bits.view(rows, -1)[:, :n] > 0, x, -math.inf)
    x = x.to(TYPES[case["dtype"]])
    best = x == x.amax(1, keepdim=True)  # a tie goes to the lowest index
    token = torch.where(best, torch.arange(n, device="cuda"), n).amin(1)
    return {"logits": x, "token": token.to(torch.int32)}


# ---------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    global own
    kept, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = kept
    return {"append": _exact_append, "attend": _exact_attend, "rules": _exact_rules}[case["op"]](s)


def _exact_append(s):
    """Each pair (a, b) of a head becomes (a + ib) e^(i angle), sequence by sequence."""
    case, d, rot = s["case"], s["case"]["dim"], s["case"]["rot"]
    kc, vc = s["k_cache"].double(), s["v_cache"].double()
    turn = torch.view_as_complex(s["rope"].double())
    parts, first = [], 0
    for a, size in enumerate(_sections(case)):
        parts.append(turn[s["positions"][a].long()][:, first:first + size])
        first += size
    turn = torch.cat(parts, 1)[:, None]

    def turned(x):
        y = x.double().view(s["tokens"], -1, d).clone()
        even, odd = (slice(0, rot, 2), slice(1, rot, 2)) if case["interleaved"] else (slice(0, rot // 2), slice(rot // 2, rot))
        z = torch.complex(y[..., even].contiguous(), y[..., odd].contiguous()) * turn
        y[..., even], y[..., odd] = z.real, z.imag
        return y

    q, k, v = turned(s["q"]), turned(s["k"]), s["v"].double().view(s["tokens"], -1, d)
    at = 0
    for b, (n, kv) in enumerate(zip(*_lengths(case))):
        index = torch.arange(kv - n, kv, device="cuda")
        page = s["table"][b].long()[index // case["page"]]
        kc[page, :, index % case["page"]] = k[at:at + n]
        vc[page, :, index % case["page"]] = v[at:at + n]
        at += n
    return {"q": q.reshape(s["tokens"], -1), "k_cache": kc, "v_cache": vc}


def _exact_attend(s):
    """softmax(q . k) v by its definition, one sequence and one key head at a time."""
    case, d = s["case"], s["case"]["dim"]
    group = case["q_heads"] // case["kv_heads"]
    out = torch.zeros(s["tokens"], case["q_heads"], d, dtype=torch.float64, device="cuda")
    at = 0
    for b, (n, kv) in enumerate(zip(*_lengths(case))):
        pages = s["table"][b, : -(-kv // case["page"])].long()
        place = torch.arange(kv - n, kv, device="cuda")[:, None]
        key = torch.arange(kv, device="cuda")
        hidden = torch.zeros(n, kv, dtype=torch.bool, device="cuda")
        if case["causal"]:
            hidden |= key > place
        if case["window"]:
            hidden |= key <= place - case["window"]
        for h in range(case["kv_heads"]):
            k = s["k_cache"][pages, h].reshape(-1, d)[:kv].double()
            v = s["v_cache"][pages, h].reshape(-1, d)[:kv].double()
            for g in range(group):
                q = s["q"][at:at + n, (h * group + g) * d:(h * group + g + 1) * d].double()
                w = torch.softmax((q @ k.T / math.sqrt(d)).masked_fill(hidden, -math.inf), -1)
                out[at:at + n, h * group + g] = w @ v
        at += n
    return {"out": out.view(s["tokens"], -1)}


def _exact_rules(s):
    case, rows = s["case"], []
    for r in range(case["rows"]):
        x = s["logits"][r].double()
        n = int(s["lens"][r])
        ids = s["history"][r, :n].long()
        again, often, present = (float(p) for p in s["penalties"][r])
        used = torch.bincount(ids, minlength=case["vocab"]) > 0
        x = torch.where(used, torch.where(x > 0, x / again, x * again), x)
        count = torch.bincount(ids[int(s["prompts"][r]):], minlength=case["vocab"])
        x = x - often * count - present * (count > 0).double()
        if case["bias"]:
            b = slice(r * case["bias"], (r + 1) * case["bias"])
            x[s["bias_tokens"][b].long()] += s["bias_values"][b].double()
        if case["grammar"]:
            word = s["allowed"][r].long() & 0xFFFFFFFF
            ok = (word[:, None] >> torch.arange(32, device="cuda")) & 1
            x = x.masked_fill(ok.view(-1)[: case["vocab"]] == 0, -math.inf)
        rows.append(x)
    return {"logits": torch.stack(rows), "token": None}
