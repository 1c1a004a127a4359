"""The packed and the paged attention and the log probabilities used together: one
attention layer and an output head that generates from a cache, scores what it
generated in one packed batch, and takes a policy gradient step's gradients.

Bounds. u = 2^-11 is half a step of FP16. Between the FP16 inputs and a weight
gradient lie ten roundings to FP16 (qkv, P, o, logits, dlogits, do, P again, dS,
dqkv, and for the head's gradient fewer), each relative to the value, and a
logit's enters its probability times the logit, at most 5 here. As 2-norms they
add up to at most (9 + 5) u; 16 u covers the products of small terms."""

import math

import pytest
import torch

from attention_bounds import U, attend, causal, worst
from inputs import normal

pytestmark = pytest.mark.gpu

HEADS, KV, HD, VOCAB, COLS = 4, 2, 64, 501, 504
WIDTH = HEADS * HD
QKV = (HEADS + 2 * KV) * HD


class Layer:
    def __init__(self, flint, cuda, seed=1):
        self.f, self.cuda = flint, cuda
        self.w_qkv = normal((QKV, WIDTH), seed, 0.06, torch.float16)
        self.w_head = normal((COLS, WIDTH), seed + 1, 0.12, torch.float16)
        self.dev = [w.to(cuda) for w in (self.w_qkv, self.w_head)]

    def half(self, *shape):
        return torch.empty(shape, dtype=torch.float16, device=self.cuda)

    def project(self, h):
        qkv = self.half(h.shape[0], QKV)
        self.f.gemm_nt(qkv, h, self.dev[0], h.shape[0], QKV, WIDTH)
        return qkv

    def head(self, o):
        logits = self.half(o.shape[0], COLS)
        self.f.gemm_nt(logits, o, self.dev[1], o.shape[0], COLS, WIDTH)
        return logits

    def split(self, qkv):
        return qkv[:, :WIDTH], qkv[:, WIDTH:WIDTH + KV * HD], qkv[:, WIDTH + KV * HD:]

    def logprobs(self, logits, targets, top=0):
        n = logits.shape[0]
        one = lambda *s: torch.empty(s, device=self.cuda)   # noqa: E731
        out = dict(logprob=one(n), entropy=one(n), stats=one(n, 2), ids=None, values=None)
        if top:
            out.update(ids=torch.empty((n, top), dtype=torch.int32, device=self.cuda),
                       values=one(n, top))
        self.f.logprobs_forward(out["logprob"], out["entropy"], out["stats"], out["ids"],
                                out["values"], logits, targets, 1.0, n, VOCAB, COLS, top)
        return out

    def packed(self, qkv, offsets, sequences):
        n = qkv.shape[0]
        shape = self.f.packed_shape(n, sequences, HEADS, KV, HD, QKV, QKV, WIDTH)
        plan = torch.empty(self.f.attention_packed_plan_bytes(shape), dtype=torch.uint8,
                           device=self.cuda)
        o, lse = self.half(n, WIDTH), torch.empty((HEADS, n), device=self.cuda)
        self.f.attention_packed_plan(plan, offsets, shape)
        self.f.attention_packed_forward(o, lse, *self.split(qkv), plan, shape, HD ** -0.5)
        return o, lse, plan, shape


def generate(layer, h, lengths, chunks, page_size=16):
    """Feeds each sequence's rows of h chunk by chunk (chunks: a list of row
    counts a call takes of every sequence, as far as it has them) over a paged
    cache; returns o in the packed order."""
    f, cuda, S = layer.f, layer.cuda, len(lengths)
    columns = max(-(-n // page_size) for n in lengths)
    pages = S * columns
    table = torch.randperm(pages, generator=torch.Generator().manual_seed(3)).to(torch.int32)
    table = table.view(S, columns).to(cuda)
    pool = torch.full((2, pages, KV, page_size, HD), float("nan"), dtype=torch.float16, device=cuda)
    starts = [sum(lengths[:i]) for i in range(S)]
    done = [0] * S
    out = layer.half(sum(lengths), WIDTH)
    for size in chunks:
        take = [min(size, n - d) for n, d in zip(lengths, done)]
        rows = [r for s, t in enumerate(take) for r in range(starts[s] + done[s],
                                                              starts[s] + done[s] + t)]
        qkv = layer.project(h[rows].contiguous())
        offsets = torch.tensor([sum(take[:i]) for i in range(S + 1)], dtype=torch.int32, device=cuda)
        cached = torch.tensor(done, dtype=torch.int32, device=cuda)
        o = layer.half(len(rows), WIDTH)
        shape = f.paged_shape(len(rows), S, max(take), HEADS, KV, HD, QKV, QKV, WIDTH, pages,
                              page_size, columns)
        f.attention_paged(o, pool[0], pool[1], *layer.split(qkv), offsets, cached, table, shape,
                          HD ** -0.5)
        out[rows] = o
        done = [d + t for d, t in zip(done, take)]
    assert done == list(lengths)
    return out


def test_cache_and_packed_batch_agree_and_score(flint, cuda):
    layer = Layer(flint, cuda)
    lengths = [70, 1, 33, 120]
    n = sum(lengths)
    h = normal((n, WIDTH), 5, 1.0, torch.float16).to(cuda)
    offsets = [sum(lengths[:i]) for i in range(len(lengths) + 1)]
    qkv = layer.project(h)
    o, _, _, _ = layer.packed(qkv, torch.tensor(offsets, dtype=torch.int32, device=cuda), len(lengths))
    # A prompt in chunks, then one token at a time.
    paged = generate(layer, h, lengths, [40, 17] + [1] * 63)
    torch.cuda.synchronize()
    # Both against float64 attention of the same projected rows.
    q, k, v = layer.split(qkv.cpu())
    for a, b in zip(offsets, offsets[1:]):
        for head in range(HEADS):
            j = head // (HEADS // KV)
            ref = attend(q[a:b, head * HD:head * HD + HD], k[a:b, j * HD:j * HD + HD],
                         v[a:b, j * HD:j * HD + HD], HD ** -0.5, causal(b - a))["o"]
            for got in (o, paged):
                assert worst(got[a:b, head * HD:head * HD + HD].cpu(), *ref) <= 1.0
    # Scored from either, the alternatives' values agree to the logits' rounding
    # (|logit| below 8: 8 u each way, twice over for the sum of the others).
    targets = torch.zeros(n, dtype=torch.int16, device=cuda)
    one, two = (layer.logprobs(layer.head(x), targets, top=5) for x in (o, paged))
    torch.cuda.synchronize()
    assert float((one["values"] - two["values"]).abs().max()) <= 32 * U
    assert float((one["logprob"] - two["logprob"]).abs().max()) <= 32 * U


def test_policy_gradient_of_a_packed_batch(flint, cuda):
    layer = Layer(flint, cuda, seed=9)
    f, lengths = flint, [37, 2, 90, 1, 64]
    n = sum(lengths)
    h = normal((n, WIDTH), 11, 1.0, torch.float16)
    targets = torch.randint(0, VOCAB, (n,), generator=torch.Generator().manual_seed(12))
    advantage = normal((n,), 13, 1.0)
    bonus = 0.05
    offsets = [sum(lengths[:i]) for i in range(len(lengths) + 1)]

    hd = h.to(cuda)
    t16 = targets.to(torch.int32).to(torch.int16).to(cuda)
    qkv = layer.project(hd)
    o, lse, plan, shape = layer.packed(qkv, torch.tensor(offsets, dtype=torch.int32, device=cuda),
                                       len(lengths))
    logits = layer.head(o)
    lp = layer.logprobs(logits, t16)
    dlogits = torch.empty_like(logits)
    f.logprobs_backward(dlogits, advantage.to(cuda), torch.full((n,), bonus, device=cuda), logits,
                        t16, lp["entropy"], lp["stats"], 1.0, n, VOCAB, COLS)
    do, dqkv, dh = layer.half(n, WIDTH), layer.half(n, QKV), layer.half(n, WIDTH)
    dw_head = torch.empty((COLS, WIDTH), device=cuda)
    dw_qkv = torch.empty((QKV, WIDTH), device=cuda)
    f.gemm_nn(do, dlogits, layer.dev[1], n, WIDTH, COLS)
    f.gemm_tn(dw_head, dlogits, o, COLS, WIDTH, n)
    f.attention_packed_backward(*layer.split(dqkv), do, *layer.split(qkv), o, lse, plan, shape,
                                HD ** -0.5)
    f.gemm_tn(dw_qkv, dqkv, hd, QKV, WIDTH, n)
    f.gemm_nn(dh, dqkv, layer.dev[0], n, WIDTH, QKV)
    torch.cuda.synchronize()

    # The same in float64 by automatic differentiation.
    x, wq, wh = (t.double().requires_grad_(True) for t in (h, layer.w_qkv, layer.w_head))
    q, k, v = ((x @ wq.T)[:, c] for c in (slice(0, WIDTH), slice(WIDTH, WIDTH + KV * HD),
                                          slice(WIDTH + KV * HD, None)))
    rows = []
    for a, b in zip(offsets, offsets[1:]):
        heads = []
        for head in range(HEADS):
            c = slice(head // (HEADS // KV) * HD, head // (HEADS // KV) * HD + HD)
            s = q[a:b, head * HD:head * HD + HD] @ k[a:b, c].T * HD ** -0.5
            s = s.masked_fill(~causal(b - a), -math.inf)
            heads.append(torch.softmax(s, 1) @ v[a:b, c])
        rows.append(torch.cat(heads, 1))
    logp = torch.log_softmax((torch.cat(rows) @ wh.T)[:, :VOCAB], 1)
    entropy = -(logp.exp() * logp).sum(1)
    (advantage.double() * logp[torch.arange(n), targets] + bonus * entropy).sum().backward()
    for name, got, ref in (("dw_head", dw_head, wh.grad), ("dw_qkv", dw_qkv, wq.grad),
                           ("dh", dh, x.grad)):
        off = float(torch.linalg.vector_norm(got.cpu().double() - ref) / torch.linalg.vector_norm(ref))
        print(f"{name}: {off / U:.2f} u")
        assert off <= 16 * U, name
