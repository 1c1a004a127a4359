"""Attention over packed sequences, attention of new tokens over a paged cache,
and the log probabilities of given tokens: measurable cases, in plain form and
through the library.

  packed    causal attention over sequences of different lengths laid one after
            another in the token rows, with grouped heads; training adds the
            gradients of q, k and v
  paged     new tokens of each sequence attend over a paged cache and
            themselves, and their keys and values are stored into the pages
  logprobs  log probability of each row's target, entropy, and the most likely
            alternatives; training adds the gradient of the logits

`run` computes the plain form in FP32 with elementary torch operations, or
(own) makes the library's calls. `exact` restates each operator in FP64.
"""

import math
import random

import torch

own = False


def listed():
    return [
        # Five short prompts scored together: 64-wide heads, latency counts.
        dict(name="packed-eval-200", kind="packed", tokens=200, sequences=5, mix=1, spare=0,
             heads=12, kv_heads=12, head_width=64, train=False),
        # A training batch of the GPT-2 124M heads: 8,192 tokens of documents
        # of very different lengths instead of 8 rows of 1,024.
        dict(name="packed-train-8192", kind="packed", tokens=8192, sequences=24, mix=2, spare=0,
             heads=12, kv_heads=12, head_width=64, train=True),
        # Grouped heads of width 128 on an odd number of tokens, the batch
        # padded by rows that belong to no sequence.
        dict(name="packed-train-grouped", kind="packed", tokens=4133, sequences=9, mix=3, spare=91,
             heads=16, kv_heads=2, head_width=128, train=True),
        # One long document and a few short ones behind it, grouped heads.
        dict(name="packed-eval-long", kind="packed", tokens=16384, sequences=4, mix=2, spare=0,
             heads=12, kv_heads=4, head_width=64, train=False),
        # Generation of one sequence, one token at a time: latency.
        dict(name="paged-decode-1", kind="paged", sequences=1, new=1, cached=777, mix=1, heads=12,
             kv_heads=12, head_width=64, page_size=16),
        # A serving batch: 64 sequences of different lengths, grouped heads of
        # width 128, one token each.
        dict(name="paged-decode-64", kind="paged", sequences=64, new=1, cached=8192, mix=2,
             heads=32, kv_heads=8, head_width=128, page_size=64),
        # Few sequences with very long caches, one token each.
        dict(name="paged-decode-long", kind="paged", sequences=3, new=1, cached=131072, mix=3,
             heads=12, kv_heads=12, head_width=64, page_size=32),
        # Chunks of prompts over what is cached of them, odd lengths.
        dict(name="paged-chunk-500", kind="paged", sequences=4, new=500, cached=4096, mix=4,
             heads=12, kv_heads=4, head_width=64, page_size=16),
        # The last rows of a sampling step: log probabilities with the five
        # most likely alternatives at GPT-2's vocabulary.
        dict(name="logprobs-eval-16", kind="logprobs", rows=16, vocab=50257, cols=50304, top=5,
             scale=1.0, train=False),
        # A character-sized vocabulary, odd rows, at a temperature.
        dict(name="logprobs-train-777x997", kind="logprobs", rows=777, vocab=997, cols=1000, top=20,
             scale=0.8, train=True),
        # A training batch's policy gradient with an entropy term at GPT-2's
        # vocabulary.
        dict(name="logprobs-train-8192", kind="logprobs", rows=8192, vocab=50257, cols=50304, top=0,
             scale=1.0, train=True),
        # The same batch scored, with twenty alternatives a token.
        dict(name="logprobs-eval-8192", kind="logprobs", rows=8192, vocab=50257, cols=50304, top=20,
             scale=1.0, train=False),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["packed", "packed", "paged", "paged", "logprobs"])
    if kind == "logprobs":
        vocab = rng.choice([_log_int(rng, 100, 50257), 50257])
        pad = rng.choice([8, 64, 128])
        return dict(kind=kind, rows=_log_int(rng, 1, 8192), vocab=vocab,
                    cols=(vocab + pad - 1) // pad * pad, top=rng.choice([0, 1, 5, 20, 64]),
                    scale=rng.choice([1.0, 1.0, 0.7, 1.5]), train=rng.random() < 0.5)
    kv_heads = rng.randint(1, 8)
    heads = kv_heads * rng.choice([1, 1, 2, 3, 4, 8])
    while heads > 16:
        heads -= kv_heads
    width = rng.choice([64, 64, 128])
    if kind == "packed":
        tokens = _log_int(rng, 1, 8192)
        case = dict(kind=kind, tokens=tokens, sequences=_log_int(rng, 1, min(64, tokens)),
                    mix=rng.randrange(1 << 16), spare=rng.choice([0, 0, _log_int(rng, 1, 200)]),
                    heads=heads, kv_heads=kv_heads, head_width=width, train=rng.random() < 0.6)
        most = max(work(c)["flops"] for c in listed() if c["kind"] == kind)
        while work(case)["flops"] > most:
            case["tokens"] = case["tokens"] * 3 // 4
        return case
    mode = rng.random()
    if mode < 0.5:
        new, sequences, cached = 1, _log_int(rng, 1, 64), _log_int(rng, 1, 8192)
    elif mode < 0.65:
        new, sequences, cached = 1, rng.randint(1, 2), _log_int(rng, 8192, 131072)
    else:
        new, sequences, cached = _log_int(rng, 2, 600), _log_int(rng, 1, 4), _log_int(rng, 1, 4096)
    return dict(kind=kind, sequences=sequences, new=new, cached=cached, mix=rng.randrange(1 << 16),
                heads=heads, kv_heads=kv_heads, head_width=width,
                page_size=rng.choice([8, 16, 32, 64, 128]))


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return dict(_PREPARE[case["kind"]](case, g), case=case)


def run(state):
    return _RUN[state["case"]["kind"]](state["case"], state)


def exact(case, seed):
    return _EXACT[case["kind"]](case, prepare(case, seed))


def work(case):
    return _WORK[case["kind"]](case)


# ------------------------------------------------------------------ inputs
_library = None


def _flint():
    global _library
    if _library is None:
        from flint_amd.flint_lib import Flint

        _library = Flint()
    return _library


def _normal(g, shape, std=1.0, dtype=torch.float16):
    return (torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * std).to(dtype)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _offsets(lengths):
    out = [0]
    for n in lengths:
        out.append(out[-1] + n)
    return out


def _bytes(n):
    return torch.empty(max(int(n), 16), dtype=torch.uint8, device="cuda")


def _once(state, name, make):
    """What a program makes once beside its tensors (shapes, workspaces)."""
    if name not in state:
        state[name] = make()
    return state[name]


# ------------------------------------------------------------------ packed
def _lengths(case):
    """The sequences' lengths: a document mix whose lengths spread over their
    logarithm, summing to the case's tokens; some may be empty."""
    rng = random.Random(case["mix"])
    weights = [math.exp(rng.gauss(0.0, 1.3)) for _ in range(case["sequences"])]
    cuts, at = [], 0.0
    for w in weights:
        at += w
        cuts.append(int(round(case["tokens"] * at / sum(weights))))
    cuts[-1] = case["tokens"]
    return [b - a for a, b in zip([0] + cuts[:-1], cuts)]


def _packed_inputs(case, g):
    H, Hk, w = case["heads"], case["kv_heads"], case["head_width"]
    rows = case["tokens"] + case["spare"]
    lengths = _lengths(case)
    # q, k and v are column slices of one projection, as a model has them.
    qkv = _normal(g, (rows, (H + 2 * Hk) * w))
    s = dict(qkv=qkv, q=qkv[:, :H * w], k=qkv[:, H * w:(H + Hk) * w], v=qkv[:, (H + Hk) * w:],
             offsets=_ints(_offsets(lengths)), longest=max(lengths), scale=1.0 / math.sqrt(w),
             o=torch.zeros((rows, H * w), dtype=torch.float16, device="cuda"),
             lse=torch.zeros((H, rows), device="cuda"))
    if case["train"]:
        s.update(dout=_normal(g, (rows, H * w), 1e-2), dqkv=torch.zeros_like(qkv))
    return s


def _packed_run(case, s):
    return _packed_own(case, s) if own else _packed_plain(case, s)


def _packed_own(case, s):
    f = _flint()
    H, Hk, w = case["heads"], case["kv_heads"], case["head_width"]
    rows, wide = s["qkv"].shape
    shape = _once(s, "shape", lambda: f.packed_shape(rows, case["sequences"], H, Hk, w, wide, wide,
                                                      H * w))
    plan = _once(s, "plan", lambda: _bytes(f.attention_packed_plan_bytes(shape)))
    f.attention_packed_plan(plan, s["offsets"], shape)
    f.attention_packed_forward(s["o"], s["lse"], s["q"], s["k"], s["v"], plan, shape, s["scale"])
    if not case["train"]:
        return dict(o=s["o"], lse=s["lse"])
    ws = _once(s, "ws", lambda: _bytes(f.attention_packed_backward_workspace(shape)))
    d = s["dqkv"]
    f.attention_packed_backward(d[:, :H * w], d[:, H * w:(H + Hk) * w], d[:, (H + Hk) * w:],
                                s["dout"], s["q"], s["k"], s["v"], s["o"], s["lse"], plan, shape,
                                s["scale"], ws)
    return dict(o=s["o"], lse=s["lse"], dqkv=d)


def _packed_plain(case, s):
    H, Hk, w = case["heads"], case["kv_heads"], case["head_width"]
    S, T, L, G = case["sequences"], case["tokens"], s["longest"], H // Hk
    rows = s["qkv"].shape[0]
    ends = s["offsets"].long()
    token = torch.arange(rows, device="cuda")
    inside = (token < ends[-1])[:, None]
    seq = torch.searchsorted(ends, token, right=True).clamp_(max=S) - 1
    # Sequences side by side, padded to the longest; or, where that is more,
    # all of them in one row of the batch, kept apart by the mask.
    if S * L * L <= T * T:
        at = ends[:-1, None] + torch.arange(L, device="cuda")
        of = torch.where(at < ends[1:, None], torch.arange(S, device="cuda")[:, None], -1)
        back = seq * L + token - ends[seq]
    else:
        L, at, of, back = T, token[None, :T], seq[None, :T], token
    at = at.clamp(max=T - 1)
    back = back.clamp(max=at.numel() - 1)

    def padded(x, heads):
        return x[at].float().view(at.shape[0], L, heads, w).transpose(1, 2)

    def rows_of(x):
        return x.transpose(1, 2).reshape(at.numel(), -1)[back]

    t = torch.arange(L, device="cuda")
    seen = ((of[:, :, None] == of[:, None, :]) & (t[None, :, None] >= t[None, None, :])
            & (of[:, None, :] >= 0))[:, None]
    q = padded(s["q"], H)
    k = padded(s["k"], Hk).repeat_interleave(G, 1)
    v = padded(s["v"], Hk).repeat_interleave(G, 1)
    p = (q @ k.transpose(2, 3)).mul_(s["scale"]).masked_fill_(~seen, -math.inf)
    m = p.amax(-1, keepdim=True).clamp_(min=-3e38)
    p.sub_(m).exp_()
    total = p.sum(-1, keepdim=True)
    total = total + (total == 0)
    p.div_(total)
    o = p @ v
    lse = rows_of(m + total.log()).T
    s["o"].copy_(torch.where(inside, rows_of(o), s["o"].float()))
    s["lse"].copy_(torch.where(inside.T, lse, s["lse"]))
    if not case["train"]:
        return dict(o=s["o"], lse=s["lse"])
    do = padded(s["dout"], H)
    do = torch.where((of >= 0)[:, None, :, None], do, 0.0)
    dv = p.transpose(2, 3) @ do
    dp = do @ v.transpose(2, 3)
    dp.sub_((do * o).sum(-1, keepdim=True)).mul_(p).mul_(s["scale"])
    dq = dp @ k
    dk = dp.transpose(2, 3) @ q

    def shared(x):
        return x.reshape(x.shape[0], Hk, G, L, w).sum(2)

    got = torch.cat([rows_of(dq), rows_of(shared(dk)), rows_of(shared(dv))], 1)
    s["dqkv"].copy_(torch.where(inside, got, s["dqkv"].float()))
    return dict(o=s["o"], lse=s["lse"], dqkv=s["dqkv"])


def _packed_exact(case, s):
    H, Hk, w = case["heads"], case["kv_heads"], case["head_width"]
    out = dict(o=s["o"].double(), lse=s["lse"].double())
    if case["train"]:
        out["dqkv"] = torch.zeros_like(s["qkv"], dtype=torch.float64)
    at = _offsets(_lengths(case))
    for first, end in zip(at, at[1:]):
        hidden = torch.ones(end - first, end - first, dtype=torch.bool, device="cuda").triu_(1)
        for h in range(H if end > first else 0):
            j = h // (H // Hk)
            cq, ck, cv = (slice(c * w, c * w + w) for c in (h, H + j, H + Hk + j))
            q, k, v = (s["qkv"][first:end, c].double() for c in (cq, ck, cv))
            x = torch.matmul(q, k.T.contiguous()) * s["scale"]
            x[hidden] = -math.inf
            lse = torch.logsumexp(x, 1)
            p = torch.exp_(x - lse[:, None])
            o = torch.matmul(p, v)
            out["o"][first:end, h * w:h * w + w] = o
            out["lse"][h, first:end] = lse
            if case["train"]:
                do = s["dout"][first:end, h * w:h * w + w].double()
                ds = torch.matmul(do, v.T.contiguous())
                ds = p * (ds - (do * o).sum(1, keepdim=True)) * s["scale"]
                out["dqkv"][first:end, cq] = torch.matmul(ds, k)
                out["dqkv"][first:end, ck] += torch.matmul(ds.T.contiguous(), q)
                out["dqkv"][first:end, cv] += torch.matmul(p.T.contiguous(), do)
    return out


def _packed_work(case):
    H, Hk, w, n = case["heads"], case["kv_heads"], case["head_width"], case["tokens"]
    product = sum(2 * w * H * (x * (x + 1) // 2) for x in _lengths(case))
    read, written = n * (H + 2 * Hk) * w * 2, n * H * (2 * w + 4)
    if not case["train"]:
        return dict(flops=2 * product, bytes=read + written)
    # Forward, then dout read and the three gradients written.
    return dict(flops=7 * product, bytes=2 * read + written + n * H * w * 2)


# ------------------------------------------------------------------- paged
def _chunks(case):
    """(cached, new) of each sequence: caches from an eighth of the case's
    length to all of it, new tokens from half of the chunk to all of it."""
    rng = random.Random(case["mix"])
    n, c = case["new"], case["cached"]
    return [(c if i == 0 else rng.randint((c + 7) // 8, c), n if i == 0 else rng.randint((n + 1) // 2, n))
            for i in range(case["sequences"])]


def _paged_inputs(case, g):
    H, Hk, w, size = case["heads"], case["kv_heads"], case["head_width"], case["page_size"]
    chunks = _chunks(case)
    need = [-(-(c + n) // size) for c, n in chunks]
    pages, width = sum(need) + 3, max(need) + 1
    # Pages are handed out in no order; entries past a sequence's last hold -1.
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(chunks), width), -1, dtype=torch.int32, device="cuda")
    for i, (a, n) in enumerate(zip(_offsets(need), need)):
        table[i, :n] = order[a:a + n]
    tokens = sum(n for _, n in chunks)
    qkv = _normal(g, (tokens, (H + 2 * Hk) * w))
    pool = (pages, Hk, size, w)
    return dict(qkv=qkv, q=qkv[:, :H * w], k=qkv[:, H * w:(H + Hk) * w], v=qkv[:, (H + Hk) * w:],
                k_pages=_normal(g, pool), v_pages=_normal(g, pool), table=table,
                offsets=_ints(_offsets([n for _, n in chunks])), cached=_ints([c for c, _ in chunks]),
                scale=1.0 / math.sqrt(w), o=torch.empty((tokens, H * w), dtype=torch.float16,
                                                        device="cuda"))


def _paged_run(case, s):
    return _paged_own(case, s) if own else _paged_plain(case, s)


def _paged_own(case, s):
    f = _flint()
    H, Hk, w = case["heads"], case["kv_heads"], case["head_width"]
    tokens, wide = s["qkv"].shape
    shape = _once(s, "shape", lambda: f.paged_shape(
        tokens, case["sequences"], case["new"], H, Hk, w, wide, wide, H * w,
        s["k_pages"].shape[0], case["page_size"], s["table"].shape[1]))
    ws = _once(s, "ws", lambda: _bytes(f.attention_paged_workspace(shape)))
    f.attention_paged(s["o"], s["k_pages"], s["v_pages"], s["q"], s["k"], s["v"], s["offsets"],
                      s["cached"], s["table"], shape, s["scale"], ws)
    return dict(o=s["o"], k_pages=s["k_pages"], v_pages=s["v_pages"])


def _paged_plain(case, s):
    H, Hk, w, size = case["heads"], case["kv_heads"], case["head_width"], case["page_size"]
    S, N, G = case["sequences"], case["new"], H // Hk
    tokens = s["qkv"].shape[0]
    first = s["offsets"].long()
    cached = s["cached"].long()
    token = torch.arange(tokens, device="cuda")
    seq = torch.searchsorted(first, token, right=True) - 1
    place = token - first[seq]
    position = cached[seq] + place
    page = s["table"][seq, position // size].long()
    s["k_pages"][page, :, position % size] = s["k"].view(tokens, Hk, w)
    s["v_pages"][page, :, position % size] = s["v"].view(tokens, Hk, w)

    table = s["table"].clamp(min=0)
    k = s["k_pages"][table].transpose(1, 2).reshape(S, Hk, -1, w).float()
    v = s["v_pages"][table].transpose(1, 2).reshape(S, Hk, -1, w).float()
    at = (first[:-1, None] + torch.arange(N, device="cuda")).clamp_(max=tokens - 1)
    q = s["q"][at].float().view(S, N, Hk, G, w).permute(0, 2, 3, 1, 4).reshape(S, Hk, G * N, w)
    last = (cached[:, None] + torch.arange(N, device="cuda")).repeat(1, G)
    seen = torch.arange(k.shape[2], device="cuda") <= last[:, :, None]
    # Rows past a sequence's keys may hold anything (a page handed out and not
    # written yet): out of the sums, not times 0.
    held = torch.arange(k.shape[2], device="cuda") < (cached + first[1:] - first[:-1])[:, None]
    v = torch.where(held[:, None, :, None], v, 0.0)
    p = (q @ k.transpose(2, 3)).mul_(s["scale"]).masked_fill_(~seen[:, None], -math.inf)
    p.sub_(p.amax(-1, keepdim=True)).exp_()
    p.div_(p.sum(-1, keepdim=True))
    o = (p @ v).view(S, Hk, G, N, w).permute(0, 3, 1, 2, 4).reshape(S, N, H * w)
    s["o"].copy_(o[seq, place])
    return dict(o=s["o"], k_pages=s["k_pages"], v_pages=s["v_pages"])


def _paged_exact(case, s):
    H, Hk, w, size = case["heads"], case["kv_heads"], case["head_width"], case["page_size"]
    out = torch.zeros_like(s["o"], dtype=torch.float64)
    # The pages move values and round none: the caches as they are stored.
    pages = dict(k=s["k_pages"].clone(), v=s["v_pages"].clone())
    table = s["table"].tolist()
    t = 0
    for i, (c, n) in enumerate(_chunks(case)):
        chosen = table[i][:-(-(c + n) // size)]
        whole = {}
        for name in "kv":
            new = s[name][t:t + n].reshape(n, Hk, w)
            rows = pages[name][chosen].transpose(1, 2).reshape(-1, Hk, w)
            rows[c:c + n] = new
            pages[name][chosen] = rows.view(len(chosen), size, Hk, w).transpose(1, 2).contiguous()
            whole[name] = rows[:c + n]
        hidden = torch.arange(c + n, device="cuda") > torch.arange(c, c + n, device="cuda")[:, None]
        for h in range(H):
            j = h // (H // Hk)
            q = s["q"][t:t + n, h * w:h * w + w].double()
            x = torch.matmul(q, whole["k"][:, j].double().T.contiguous()) * s["scale"]
            x[hidden] = -math.inf
            p = torch.exp_(x - torch.logsumexp(x, 1)[:, None])
            out[t:t + n, h * w:h * w + w] = torch.matmul(p, whole["v"][:, j].double())
        t += n
    return dict(o=out, k_pages=pages["k"], v_pages=pages["v"])


def _paged_work(case):
    H, Hk, w = case["heads"], case["kv_heads"], case["head_width"]
    chunks = _chunks(case)
    pairs = sum(n * c + n * (n + 1) // 2 for c, n in chunks)
    new = sum(n for _, n in chunks)
    # The cached rows read; the new rows of q, k and v read, of o, k and v
    # written.
    row = 2 * Hk * w * 2
    return dict(flops=4 * w * H * pairs,
                bytes=sum(c for c, _ in chunks) * row + 2 * new * (row + H * w * 2))


# ---------------------------------------------------------------- logprobs
def _logprobs_inputs(case, g):
    rows, vocab, cols = case["rows"], case["vocab"], case["cols"]
    # A language model's logits: a spread of a few, some words far likelier;
    # the target one of the likely words in most rows.
    logits = _normal(g, (rows, cols), 2.0)
    likely = torch.randint(0, vocab, (rows, 8), generator=g, device="cuda")
    rise = torch.rand((rows, 8), generator=g, device="cuda") * 12.0
    logits.scatter_add_(1, likely, rise.half())
    targets = torch.where(torch.rand(rows, generator=g, device="cuda") < 0.8, likely[:, 0],
                          torch.randint(0, vocab, (rows,), generator=g, device="cuda"))
    s = dict(logits=logits, targets=targets.to(torch.int32).to(torch.int16),
             logprob=torch.empty(rows, device="cuda"), entropy=torch.empty(rows, device="cuda"),
             stats=torch.empty((rows, 2), device="cuda"), ids=None, values=None)
    if case["top"]:
        s.update(ids=torch.empty((rows, case["top"]), dtype=torch.int32, device="cuda"),
                 values=torch.empty((rows, case["top"]), device="cuda"))
    if case["train"]:
        s.update(dlogprob=_normal(g, (rows,), dtype=torch.float32),
                 dentropy=torch.full((rows,), -0.01, device="cuda"),
                 dlogits=torch.empty((rows, cols), dtype=torch.float16, device="cuda"))
    return s


def _logprobs_run(case, s):
    return _logprobs_own(case, s) if own else _logprobs_plain(case, s)


def _logprobs_own(case, s):
    f = _flint()
    rows, vocab, cols = case["rows"], case["vocab"], case["cols"]
    f.logprobs_forward(s["logprob"], s["entropy"], s["stats"], s["ids"], s["values"], s["logits"],
                       s["targets"], case["scale"], rows, vocab, cols, case["top"])
    out = dict(logprob=s["logprob"], entropy=s["entropy"])
    if case["top"]:
        out.update(ids=s["ids"], values=s["values"])
    if case["train"]:
        f.logprobs_backward(s["dlogits"], s["dlogprob"], s["dentropy"], s["logits"], s["targets"],
                            s["entropy"], s["stats"], case["scale"], rows, vocab, cols)
        out["dlogits"] = s["dlogits"]
    return out


def _logprobs_plain(case, s):
    rows, vocab, cols = case["rows"], case["vocab"], case["cols"]
    target = (s["targets"].long() & 0xFFFF)[:, None]
    x = s["logits"][:, :vocab].float()
    x = x.sub_(x.amax(1, keepdim=True)).mul_(case["scale"])
    p = x.exp()
    total = p.sum(1, keepdim=True)
    x.sub_(total.log())            # every word's log probability
    p.div_(total)
    entropy = -(p * x.clamp(min=-3e38)).sum(1)
    out = dict(logprob=x.gather(1, target)[:, 0], entropy=entropy)
    if case["top"]:
        # Distinct whole numbers in the order of the values, the lower index
        # first among equal ones.
        bits = (s["logits"][:, :vocab] + 0.0).view(torch.int16).int()
        order = torch.where(bits < 0, -32768 - bits - 1, bits)
        order = order * 65536 + (65535 - torch.arange(vocab, device="cuda", dtype=torch.int32))
        ids = order.topk(case["top"], dim=1).indices
        out.update(ids=ids.int(), values=x.gather(1, ids))
    if case["train"]:
        x.clamp_(min=-3e38).add_(entropy[:, None]).mul_(s["dentropy"][:, None])
        x.add_(s["dlogprob"][:, None]).mul_(p).neg_()
        x.scatter_add_(1, target, s["dlogprob"][:, None])
        x.mul_(case["scale"])
        s["dlogits"][:, :vocab] = x
        s["dlogits"][:, vocab:] = 0
        out["dlogits"] = s["dlogits"]
    return out


def _logprobs_exact(case, s):
    rows, vocab, cols = case["rows"], case["vocab"], case["cols"]
    step = max(1, (1 << 26) // cols)
    parts = []
    for a in range(0, rows, step):
        b = min(rows, a + step)
        target = s["targets"][a:b].long() & 0xFFFF
        logp = s["logits"][a:b, :vocab].double() * case["scale"]
        logp = logp - torch.logsumexp(logp, 1)[:, None]
        p = torch.exp(logp)
        row = torch.arange(b - a, device="cuda")
        part = dict(logprob=logp[row, target], entropy=-(p * logp).sum(1))
        if case["top"]:
            at = torch.sort(s["logits"][a:b, :vocab].double(), dim=1, descending=True,
                            stable=True).indices[:, :case["top"]]
            part.update(ids=at.int(), values=logp[row[:, None], at])
        if case["train"]:
            d = torch.zeros((b - a, cols), dtype=torch.float64, device="cuda")
            dl, dh = s["dlogprob"][a:b, None].double(), s["dentropy"][a:b, None].double()
            d[:, :vocab] = -p * (dl + dh * (logp + part["entropy"][:, None]))
            d[row, target] += dl[:, 0]
            part["dlogits"] = d * case["scale"]
        parts.append(part)
    return {name: torch.cat([p[name] for p in parts]) for name in parts[0]}


def _logprobs_work(case):
    rows, vocab, top = case["rows"], case["vocab"], case["top"]
    read = rows * vocab * 2
    small = rows * (2 + 8 + 8 * top)
    if not case["train"]:
        return dict(flops=0, bytes=read + small)
    # Backward reads the logits again (they do not fit on the chip) and writes
    # their gradient.
    return dict(flops=0, bytes=2 * read + rows * case["cols"] * 2 + small + rows * 24)


_PREPARE = dict(packed=_packed_inputs, paged=_paged_inputs, logprobs=_logprobs_inputs)
_RUN = dict(packed=_packed_run, paged=_paged_run, logprobs=_logprobs_run)
_EXACT = dict(packed=_packed_exact, paged=_paged_exact, logprobs=_logprobs_exact)
_WORK = dict(packed=_packed_work, paged=_paged_work, logprobs=_logprobs_work)
