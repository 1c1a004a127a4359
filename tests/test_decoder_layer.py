"""A decoder layer with grouped heads, rotary positions and a gated feed-forward block
through the library's functions, as a program would run it: trained on packed
sequences, and served from a paged cache of 8-bit values.

Training is compared with float64 autograd in the 2-norm. Every stored value is
rounded once to FP16, at most 2^-11 of itself, so of the tensor in the norm; 14
roundings stand before the last gradient. A random matrix passes a random relative error
on as it is, the softmax multiplies one of the scores (of size about 1) by them, twice
in the gradient: a factor of 4 for it. 14 x 4 x 2^-11 < 2^-5."""

import math

import pytest
import torch

from attention_bounds import attend, worst
from inputs import normal
from test_paged8 import value_of
from test_rotary import frequencies, reference as rotary_reference

WIDTH, HIDDEN, HEADS, KV_HEADS, HEAD = 128, 328, 4, 2, 64
QW, KW = HEADS * HEAD, KV_HEADS * HEAD
SCALE = 1.0 / math.sqrt(HEAD)


def weights():
    def make(rows, cols, seed):
        return normal((rows, cols), seed, cols ** -0.5, torch.float16)

    return dict(qkv=make(QW + 2 * KW, WIDTH, 1), out=make(WIDTH, QW, 2),
                gate_up=make(2 * HIDDEN, WIDTH, 3), down=make(WIDTH, HIDDEN, 4))


def turned(x, positions, heads):
    """Rotary positions of x (tokens x heads x HEAD) in float64, halves."""
    angle = positions.double()[:, None] * frequencies(HEAD, 10000.0)
    c, s = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
    a, b = x[..., :HEAD // 2], x[..., HEAD // 2:]
    return torch.cat([a * c - b * s, a * s + b * c], -1)


def exact_layer(x, w, lengths, positions):
    """float64, differentiable: the layer's output and what it keeps."""
    qkv = x @ w["qkv"].T
    n = len(x)
    q = turned(qkv[:, :QW].reshape(n, HEADS, HEAD), positions, HEADS)
    k = turned(qkv[:, QW:QW + KW].reshape(n, KV_HEADS, HEAD), positions, KV_HEADS)
    v = qkv[:, QW + KW:].reshape(n, KV_HEADS, HEAD)
    group = HEADS // KV_HEADS
    rows, at = [], 0
    for length in lengths:
        s = slice(at, at + length)
        at += length
        scores = SCALE * torch.einsum("thd,uhd->htu", q[s], k[s].repeat_interleave(group, 1))
        hidden = torch.ones(length, length, dtype=torch.bool).triu(1)
        p = torch.softmax(scores.masked_fill(hidden, -math.inf), -1)
        rows.append(torch.einsum("htu,uhd->thd", p, v[s].repeat_interleave(group, 1)))
    o = torch.cat(rows).reshape(n, QW)
    mid = o @ w["out"].T
    pre = mid @ w["gate_up"].T
    h = torch.nn.functional.silu(pre[:, :HIDDEN]) * pre[:, HIDDEN:]
    return h @ w["down"].T


def halves(cuda, *shape):
    return torch.empty(shape, dtype=torch.float16, device=cuda)


@pytest.mark.gpu
def test_trained_on_packed_sequences(flint, cuda):
    lengths = [70, 1, 130, 55]
    n = sum(lengths)
    x = normal((n, WIDTH), 5, 1.0, torch.float16)
    dout = normal((n, WIDTH), 6, 1.0, torch.float16)
    positions = torch.cat([torch.arange(m) for m in lengths]).int()
    w = weights()

    leaves = {name: t.double().requires_grad_(True) for name, t in dict(w, x=x).items()}
    out = exact_layer(leaves["x"], leaves, lengths, positions)
    out.backward(dout.double())

    d = {name: t.to(cuda) for name, t in dict(w, x=x, dout=dout, positions=positions).items()}
    wide = QW + 2 * KW
    plan = torch.empty(flint.rotary_plan_bytes(HEAD), dtype=torch.uint8, device=cuda)
    flint.rotary_plan(plan, flint.rotary_angles(HEAD))
    turn = flint.rotary_shape(n, HEADS, KV_HEADS, HEAD, HEAD, False, wide, wide)
    qkv, o, mid = halves(cuda, n, wide), halves(cuda, n, QW), halves(cuda, n, WIDTH)
    h, pre, y = halves(cuda, n, HIDDEN), halves(cuda, n, 2 * HIDDEN), halves(cuda, n, WIDTH)
    lse = torch.empty((HEADS, n), device=cuda)

    def parts(t):
        return t[:, :QW], t[:, QW:QW + KW], t[:, QW + KW:]

    flint.gemm_nt(qkv, d["x"], d["qkv"], n, wide, WIDTH)
    q, k, v = parts(qkv)
    flint.rotary(q, k, q, k, d["positions"], plan, turn)
    offsets = torch.tensor([0, *torch.tensor(lengths).cumsum(0)], dtype=torch.int32, device=cuda)
    shape = flint.packed_shape(n, len(lengths), HEADS, KV_HEADS, HEAD, wide, wide, QW)
    blocks = torch.empty(flint.attention_packed_plan_bytes(shape), dtype=torch.uint8, device=cuda)
    flint.attention_packed_plan(blocks, offsets, shape)
    flint.attention_packed_forward(o, lse, q, k, v, blocks, shape, SCALE)
    flint.gemm_nt(mid, o, d["out"], n, WIDTH, QW)
    flint.gemm_nt_gated(h, pre, mid, d["gate_up"], None, n, HIDDEN, WIDTH, "silu")
    flint.gemm_nt(y, h, d["down"], n, WIDTH, HIDDEN)

    grads = {name: torch.empty(t.shape, device=cuda) for name, t in w.items()}
    dpre, dmid, do = halves(cuda, n, 2 * HIDDEN), halves(cuda, n, WIDTH), halves(cuda, n, QW)
    dqkv, dx = halves(cuda, n, wide), halves(cuda, n, WIDTH)
    flint.gemm_tn(grads["down"], d["dout"], h, WIDTH, HIDDEN, n)
    flint.gemm_nn_dgated(dpre, d["dout"], d["down"], pre, n, HIDDEN, WIDTH, "silu")
    flint.gemm_tn(grads["gate_up"], dpre, mid, 2 * HIDDEN, WIDTH, n)
    flint.gemm_nn(dmid, dpre, d["gate_up"], n, WIDTH, 2 * HIDDEN)
    flint.gemm_tn(grads["out"], dmid, o, WIDTH, QW, n)
    flint.gemm_nn(do, dmid, d["out"], n, QW, WIDTH)
    dq, dk, dv = parts(dqkv)
    flint.attention_packed_backward(dq, dk, dv, do, q, k, v, o, lse, blocks, shape, SCALE)
    flint.rotary(dq, dk, dq, dk, d["positions"], plan, turn, backward=True)
    flint.gemm_tn(grads["qkv"], dqkv, d["x"], wide, WIDTH, n)
    flint.gemm_nn(dx, dqkv, d["qkv"], n, WIDTH, wide)

    got = dict(grads, x=dx, out_rows=y)
    want = {name: t.grad for name, t in leaves.items()}
    want["out_rows"] = out.detach()
    for name, g in got.items():
        off = (g.cpu().double() - want[name]).norm() / want[name].norm()
        assert float(off) <= 2.0 ** -5, (name, float(off))


class Server:
    """One layer over a paged 8-bit cache: a step takes each sequence's new tokens."""

    def __init__(self, flint, cuda, sequences, block, page_size=16, columns=12):
        self.flint, self.cuda, self.block, self.page_size = flint, cuda, block, page_size
        self.w = {name: t.to(cuda) for name, t in weights().items()}
        pages = sequences * columns
        order = torch.randperm(pages, generator=torch.Generator().manual_seed(9))
        self.table = order.view(sequences, columns).int().to(cuda)
        pool = (pages, KV_HEADS, page_size, HEAD)
        self.codes = [torch.full(pool, 0x7F, dtype=torch.uint8, device=cuda) for _ in "kv"]
        self.scales = [torch.zeros(pool[:2] + (page_size // block,), dtype=torch.uint8, device=cuda)
                       for _ in "kv"]
        self.cached = torch.zeros(sequences, dtype=torch.int32, device=cuda)
        self.plan = torch.empty(flint.rotary_plan_bytes(HEAD), dtype=torch.uint8, device=cuda)
        flint.rotary_plan(self.plan, flint.rotary_angles(HEAD))

    def step(self, x, counts):
        f, n, wide = self.flint, len(x), QW + 2 * KW
        qkv, o = halves(self.cuda, n, wide), halves(self.cuda, n, QW)
        mid, h, y = (halves(self.cuda, n, c) for c in (WIDTH, HIDDEN, WIDTH))
        offsets = torch.tensor([0, *torch.tensor(counts).cumsum(0)], dtype=torch.int32,
                               device=self.cuda)
        positions = torch.cat([c + torch.arange(m, device=self.cuda)
                               for c, m in zip(self.cached, counts)]).int()
        f.gemm_nt(qkv, x, self.w["qkv"], n, wide, WIDTH)
        q, k, v = qkv[:, :QW], qkv[:, QW:QW + KW], qkv[:, QW + KW:]
        f.rotary(q, k, q, k, positions, self.plan,
                 f.rotary_shape(n, HEADS, KV_HEADS, HEAD, HEAD, False, wide, wide))
        shape = f.paged_shape(n, len(counts), max(counts), HEADS, KV_HEADS, HEAD, wide, wide, QW,
                              len(self.codes[0]), self.page_size, self.table.shape[1])
        before = self.values()
        f.attention_paged8(o, self.codes[0], self.scales[0], self.codes[1], self.scales[1], q, k, v,
                           offsets, self.cached, self.table, shape, self.block, SCALE)
        f.gemm_nt(mid, o, self.w["out"], n, WIDTH, QW)
        f.gemm_nt_gated(h, None, mid, self.w["gate_up"], None, n, HIDDEN, WIDTH, "silu")
        f.gemm_nt(y, h, self.w["down"], n, WIDTH, HIDDEN)
        was = self.cached.tolist()
        self.cached += torch.tensor(counts, dtype=torch.int32, device=self.cuda)
        return y, qkv, o, before, was, positions

    def values(self):
        """[k, v][page, head, row, column] that the cache stands for, float64."""
        return [value_of(c.cpu(), s.cpu(), self.block) for c, s in zip(self.codes, self.scales)]


@pytest.mark.gpu
@pytest.mark.parametrize("block", [1, 8, 16])
def test_served_from_an_8_bit_cache(flint, cuda, block):
    """Prompts, a chunk and single tokens. Every step's attention is checked against the
    values that the cache held before it, and the block's output against that attention;
    the cache afterwards against the rows given: e4m3 rounds to 2^-4 of a value, or to
    2^-10 of the block's scale among the subnormals, once more where a scale grew."""
    server = Server(flint, cuda, 3, block)
    rows = [[], [], []]     # the sequences' keys and values as given
    for step, counts in enumerate([[40, 1, 17], [1, 1, 1], [1, 30, 2], [1, 1, 1], [1, 1, 1]]):
        x = normal((sum(counts), WIDTH), 20 + step, 1.0, torch.float16).to(cuda)
        y, qkv, o, before, was, positions = server.step(x, counts)
        table, at = server.table.cpu(), 0
        for s, n in enumerate(counts):
            new = qkv[at:at + n].cpu()
            p = torch.arange(was[s])
            page, row = table[s][p // 16].long(), p % 16
            for j in range(KV_HEADS):
                kv = []
                for which in range(2):
                    first = QW + which * KW + j * HEAD
                    kv.append(torch.cat([before[which][page, j, row],
                                         new[:, first:first + HEAD].double()]))
                visible = torch.arange(was[s] + n)[None] <= torch.arange(was[s], was[s] + n)[:, None]
                for h in range(2 * j, 2 * j + 2):
                    value, bound = attend(new[:, h * HEAD:(h + 1) * HEAD], *kv, SCALE, visible)["o"]
                    got = o[at:at + n, h * HEAD:(h + 1) * HEAD].cpu()
                    assert worst(got, value, bound) <= 1.0
            rows[s].append(new[:, QW:].double())
            at += n
        # Keys as they are: turned by their positions.
        plain = x.double().cpu() @ server.w["qkv"].double().cpu().T
        k, bound = rotary_reference(plain[:, QW:QW + KW].half(), positions.cpu(),
                                    frequencies(HEAD, 10000.0), KV_HEADS, HEAD, HEAD, False)
        # (plain's rounding to FP16 may differ from the product's by a step: 2^-10.)
        assert torch.all((qkv[:, QW:QW + KW].cpu().double() - k).abs()
                         <= bound + 2.0 ** -9 * plain[:, QW:QW + KW].abs().amax())
        w = {name: t.double().cpu() for name, t in server.w.items()}
        pre = o.cpu().double() @ w["out"].T @ w["gate_up"].T
        want = (torch.nn.functional.silu(pre[:, :HIDDEN]) * pre[:, HIDDEN:]) @ w["down"].T
        # mid, h and y are rounded; an error of mid reaches h through gate and up.
        assert float((y.cpu().double() - want).norm() / want.norm()) <= 4 * 2.0 ** -11 * 2
    after = server.values()
    table = server.table.cpu()
    for s in range(3):
        given = torch.cat(rows[s])
        p = torch.arange(len(given))
        assert len(given) == int(server.cached[s])
        for which in range(2):
            for j in range(KV_HEADS):
                first = which * KW + j * HEAD
                want = given[:, first:first + HEAD]
                got = after[which][table[s][p // 16].long(), j, p % 16]
                top = after[which].nan_to_num(0.0).abs().amax()
                assert torch.all((got - want).abs() <= 2.0 ** -4 * want.abs() * 1.07
                                 + 2 * 2.0 ** -10 * 2.0 ** math.ceil(math.log2(float(top) / 448.0) + 1))
