"""Attention of new tokens over a paged cache of 8-bit values
(include/flint/flint_paged8.h) against float64 on the values that the cache holds,
within bounds counted in rounding steps (attention_bounds.py: decoding is exact, so
they are the FP16 cache's); the bytes it stores, and what it leaves; its refusals."""

import ctypes
import math

import pytest
import torch

from attention_bounds import attend, worst
from flint_amd import flint_lib
from inputs import gen, normal

SENTINEL = 7.25
NAN = float("nan")
NAN_CODE = 0x7F


def value_of(codes, scale_bytes, block):
    """[..., rows, width] codes and [..., rows / block] bytes -> float64 values."""
    e = scale_bytes.int().clamp(112, 135) - 127
    x = codes.view(torch.float8_e4m3fn).double()
    return torch.ldexp(x, e.repeat_interleave(block, -1)[..., None])


def exponent_of(x):
    """The least e in -15 .. 8 with every finite |x| at most 448 2^e."""
    x = x[torch.isfinite(x)].abs()
    most = float(x.max()) if len(x) else 0.0
    e = -15
    while e < 8 and most > 448.0 * 2.0 ** e:
        e += 1
    return e


def code_of(x, e):
    """float64 values -> e4m3 codes at 2^e, nearest even, within FP16's range."""
    most = 240.0 if e == 8 else 448.0
    y = (x * 2.0 ** -e)
    return torch.where(torch.isfinite(x), y.clamp(-most, most), NAN).float().to(
        torch.float8_e4m3fn).view(torch.uint8)


class Cache:
    """Sequences with cached positions and new tokens, on the CPU. Every cache row that
    holds no position is NaN, and a block without one has a scale byte of 255."""

    def __init__(self, cached, new, heads, kv_heads, width, page_size, block, seed=1, max_new=None,
                 spare_columns=1, after=0, scale=None, shared=0, dropped=(), spread=1.0, grow=1.0):
        self.cached, self.new, self.block = cached, new, block
        self.heads, self.kv_heads, self.width, self.page_size = heads, kv_heads, width, page_size
        self.scale = 1.0 / math.sqrt(width) if scale is None else scale
        self.max_new = max(new) if max_new is None else max_new
        S = len(cached)
        need = [-(-(c + n) // page_size) for c, n in zip(cached, new)]
        self.pages = sum(need) - shared * (S - 1) + 2
        order = torch.randperm(self.pages, generator=gen(seed)).tolist()
        self.table = torch.full((S, max(max(need) + spare_columns, 1)), -1, dtype=torch.int32)
        for s, n in enumerate(need):
            for i in range(shared if s else 0, min(n, self.table.shape[1])):
                self.table[s, i] = order.pop()
            if s:   # the first pages are the first sequence's own: a shared prefix
                self.table[s, :shared] = self.table[0, :shared]
        for s, i, entry in dropped:
            self.table[s, i] = entry
        pool = (self.pages, kv_heads, page_size, width)
        self.codes = [torch.full(pool, NAN_CODE, dtype=torch.uint8) for _ in "kv"]
        self.bytes = [torch.full((self.pages, kv_heads, page_size // block), 255, dtype=torch.uint8)
                      for _ in "kv"]
        fill = normal((2,) + pool, seed + 1, spread, torch.float16).double()
        for s, c in enumerate(cached):
            for p in range(0, c, block):
                page = self.page(s, p)
                if page is None:
                    continue
                at, rows = p % page_size, min(block, c - p)
                for which in range(2):
                    for head in range(kv_heads):
                        x = fill[which, page, head, at:at + rows]
                        e = exponent_of(x)
                        self.codes[which][page, head, at:at + rows] = code_of(x, e)
                        self.bytes[which][page, head, at // block] = e + 127
        self.offsets = [0]
        for n in new:
            self.offsets.append(self.offsets[-1] + n)
        self.tokens = self.offsets[-1] + after
        self.qkv = normal((self.tokens, (heads + 2 * kv_heads) * width), seed + 2, 1.0,
                          torch.float16)
        self.qkv[:, heads * width:] *= grow
        self.qkv[self.offsets[-1]:] = NAN

    def page(self, s, p):
        column = p // self.page_size
        if column >= self.table.shape[1]:
            return None
        page = int(self.table[s, column])
        return page if 0 <= page < self.pages else None

    def parts(self, qkv):
        hw, kw = self.heads * self.width, self.kv_heads * self.width
        return qkv[:, :hw], qkv[:, hw:hw + kw], qkv[:, hw + kw:]

    def reference(self):
        """(o, bound) as tokens x (heads x width), the codes and bytes after the call,
        and which rows of o are written."""
        H, Hk, w, B = self.heads, self.kv_heads, self.width, self.block
        q, k, v = self.parts(self.qkv)
        o = torch.zeros(self.tokens, H * w, dtype=torch.float64)
        bound = torch.zeros_like(o)
        done = torch.zeros(self.tokens, dtype=torch.bool)
        codes, scales = [x.clone() for x in self.codes], [x.clone() for x in self.bytes]
        values = [value_of(c, b, B) for c, b in zip(self.codes, self.bytes)]
        most = self.table.shape[1] * self.page_size
        for s in range(len(self.cached)):
            c, n = min(max(self.cached[s], 0), most), min(self.new[s], self.max_new)
            at = self.offsets[s]
            if n == 0:
                continue
            done[at:at + n] = True
            kept = [(p, self.page(s, p)) for p in range(c)]
            kept = [(p, page) for p, page in kept if page is not None]
            rows = torch.tensor([page for _, page in kept], dtype=torch.long)
            ins = torch.tensor([p % self.page_size for p, _ in kept], dtype=torch.long)
            for j in range(Hk):
                whole = []
                for which, x in enumerate((k, v)):
                    old = values[which][rows, j, ins]
                    whole.append(torch.cat([old, x[at:at + n, j * w:j * w + w].double()]))
                visible = torch.cat([torch.ones(n, len(kept), dtype=torch.bool),
                                     torch.ones(n, n, dtype=torch.bool).tril()], 1)
                for h in range(j * (H // Hk), (j + 1) * (H // Hk)):
                    got = attend(q[at:at + n, h * w:h * w + w], *whole, self.scale, visible)["o"]
                    o[at:at + n, h * w:h * w + w], bound[at:at + n, h * w:h * w + w] = got
            for p0 in range(c // B * B, c + n, B):
                page = self.page(s, p0)
                if page is None:
                    continue
                i0, old, end = p0 % self.page_size, max(0, min(c - p0, B)), min(c + n - p0, B)
                fresh = slice(at + p0 + old - c, at + p0 + end - c)
                for which, x in enumerate((k, v)):
                    for j in range(Hk):
                        new = x[fresh, j * w:j * w + w].double()
                        e = exponent_of(new)
                        if old:
                            was = min(max(int(scales[which][page, j, i0 // B]), 112), 135) - 127
                            if e > was:
                                codes[which][page, j, i0:i0 + old] = code_of(
                                    values[which][page, j, i0:i0 + old], e)
                            e = max(e, was)
                        codes[which][page, j, i0 + old:i0 + end] = code_of(new, e)
                        scales[which][page, j, i0 // B] = e + 127
        return o, bound, codes, scales, done


class Run:
    """A call on the GPU over a Cache's values."""

    def __init__(self, flint, cuda, c, qkv_columns=0, guard=64):
        self.flint, self.c = flint, c
        wide = c.qkv.shape[1] + qkv_columns
        self.qkv = torch.full((c.tokens, wide), NAN, dtype=torch.float16, device=cuda)
        self.qkv[:, :c.qkv.shape[1]] = c.qkv.to(cuda)
        self.codes, self.bytes = ([x.to(cuda) for x in y] for y in (c.codes, c.bytes))
        self.offsets = torch.tensor(c.offsets, dtype=torch.int32, device=cuda)
        self.cached = torch.tensor(c.cached, dtype=torch.int32, device=cuda)
        self.table = c.table.to(cuda)
        hw = c.heads * c.width
        self.o = torch.full((c.tokens, hw + 8), SENTINEL, dtype=torch.float16, device=cuda)
        self.shape = flint.paged_shape(c.tokens, len(c.cached), c.max_new, c.heads, c.kv_heads,
                                       c.width, wide, wide, hw + 8, c.pages, c.page_size,
                                       c.table.shape[1])
        self.need = flint.attention_paged8_workspace(self.shape, c.block)
        self.ws = torch.full((self.need + guard,), 0xA5, dtype=torch.uint8, device=cuda)

    def run(self, stream=None):
        q, k, v = self.c.parts(self.qkv)
        self.flint.attention_paged8(self.o, self.codes[0], self.bytes[0], self.codes[1],
                                    self.bytes[1], q, k, v, self.offsets, self.cached, self.table,
                                    self.shape, self.c.block, self.c.scale, self.ws,
                                    workspace_bytes=self.need, stream=stream)
        return self


def check(run, ref=None):
    c = run.c
    o, bound, codes, scales, done = ref or c.reference()
    hw = c.heads * c.width
    got = run.o.cpu()
    assert torch.all(got[:, hw:] == SENTINEL)
    assert torch.all(got[~done] == SENTINEL)
    assert worst(got[done][:, :hw], o[done], bound[done]) <= 1.0
    for name, want, have in (("k codes", codes[0], run.codes[0]), ("v codes", codes[1], run.codes[1]),
                             ("k scales", scales[0], run.bytes[0]),
                             ("v scales", scales[1], run.bytes[1])):
        # A NaN's sign is any.
        a, b = want, have.cpu()
        if "codes" in name:
            a, b = (torch.where((x & 0x7F) == NAN_CODE, NAN_CODE, x) for x in (a, b))
        assert torch.equal(a, b), name
    assert torch.all(run.ws[run.need:] == 0xA5)


# cached, new, heads, kv_heads, width, page_size, block
SHAPES = [
    ([0], [1], 1, 1, 64, 8, 1),
    ([0], [1], 4, 2, 128, 16, 16),
    ([1], [1], 2, 1, 64, 8, 8),
    ([31, 32, 33], [1, 1, 1], 4, 4, 64, 16, 4),
    ([777], [1], 12, 12, 64, 16, 16),
    ([300, 0, 5, 1000], [1, 1, 1, 1], 8, 2, 128, 32, 8),
    ([500, 64], [1, 1], 32, 1, 64, 24, 8),
    ([65, 200], [1, 1], 16, 1, 128, 40, 1),
    ([90, 7, 0], [3, 1, 2], 6, 2, 64, 8, 2),
    ([100, 0, 33], [32, 9, 17], 2, 2, 128, 64, 64),
    ([0, 70], [40, 100], 2, 1, 64, 16, 8),
    ([500, 129, 0, 63], [130, 1, 77, 64], 4, 4, 64, 16, 16),
    ([130, 1], [65, 200], 8, 2, 128, 128, 128),
    ([260, 12], [33, 129], 3, 1, 128, 8, 4),
    ([4000], [1], 2, 1, 64, 32, 32),
    ([3000, 50], [1, 1], 4, 1, 128, 16, 16),
    ([40, 100], [20, 7], 1, 1, 64, 16, 4),
    ([77, 400], [6, 1], 4, 1, 128, 8, 1),
    ([200, 3], [2, 2], 8, 1, 128, 65536, 128),
    ([1000], [1], 1, 1, 64, 8, 8),
]


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SHAPES, ids=[str(i) for i in range(len(SHAPES))])
def test_against_float64(flint, cuda, shape):
    check(Run(flint, cuda, Cache(*shape, seed=3, after=2), qkv_columns=8).run())


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 70])
@pytest.mark.parametrize("width", [64, 128])
def test_many_parts(flint, cuda, width, new):
    check(Run(flint, cuda, Cache([9000, 40, 2000], [new, 1, new], 4, 2, width, 32, 32, seed=5)).run())


@pytest.mark.gpu
@pytest.mark.parametrize("kv_heads,width", [(32, 64), (16, 128)])
def test_two_rounds_of_parts(flint, cuda, kv_heads, width):
    """Six blocks of rows of 102 tiles for 16 workgroups: 12 parts, or 30 in two rounds."""
    check(Run(flint, cuda, Cache([5800], [700], kv_heads, kv_heads, width, 64, 64, seed=29)).run())


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 40])
def test_many_sequences(flint, cuda, new):
    """More than one step of the search over sequences, some of them empty."""
    g = gen(6)
    cached = torch.randint(0, 120, (150,), generator=g).tolist()
    news = torch.randint(0, new + 1, (150,), generator=g).tolist()
    check(Run(flint, cuda, Cache(cached, news, 2, 1, 64, 16, 8, seed=7, max_new=new, after=3)).run())


@pytest.mark.gpu
@pytest.mark.parametrize("block,page_size", [(1, 8), (8, 16), (32, 32)])
def test_one_prompt_among_many_single_tokens(flint, cuda, block, page_size):
    """More slots for blocks than tokens: the blocks are found token by token."""
    cached = [(37 * i) % 90 for i in range(20)]
    new = [100 if i == 7 else i % 3 for i in range(20)]
    check(Run(flint, cuda, Cache(cached, new, 4, 2, 64, page_size, block, seed=23, after=1)).run())


@pytest.mark.gpu
def test_single_tokens_and_a_prompt_called_apart(flint, cuda):
    """Two calls over one cache and one set of rows, each with its own sequences: what one
    call gives, and neither touches the other's rows or blocks."""
    c = Cache([700, 33, 0, 129, 64, 300], [1, 1, 1, 1, 70, 41], 8, 2, 64, 16, 16, seed=30, after=1)
    ref = c.reference()
    r = Run(flint, cuda, c)
    for first, last, most in ((0, 4, 1), (4, 6, 70)):
        before = r.o.clone()
        part = slice(first, last)
        # (Clones of their own: a slice may begin off 16 bytes.)
        offsets, cached, table = (x.clone() for x in (r.offsets[first:last + 1], r.cached[part],
                                                      r.table[part]))
        s = flint.paged_shape(c.tokens, last - first, most, c.heads, c.kv_heads, c.width,
                              r.shape.q_stride, r.shape.kv_stride, r.shape.o_stride, c.pages,
                              c.page_size, c.table.shape[1])
        q, k, v = c.parts(r.qkv)
        flint.attention_paged8(r.o, r.codes[0], r.bytes[0], r.codes[1], r.bytes[1], q, k, v,
                               offsets, cached, table, s, c.block, c.scale)
        mine = torch.zeros(c.tokens, dtype=torch.bool)
        mine[c.offsets[first]:c.offsets[last]] = True
        assert torch.equal(r.o[~mine.to(cuda)], before[~mine.to(cuda)])
    check(r, ref)


@pytest.mark.gpu
@pytest.mark.parametrize("grow", [1e-4, 30.0, 6e4])
@pytest.mark.parametrize("block", [1, 16])
def test_scales_that_grow_and_extreme_rows(flint, cuda, grow, block):
    """New rows far smaller and far larger than the cached ones (overflowing to infinity
    here and there at 6e4): the older rows of their block are rounded again."""
    c = Cache([37, 16, 5], [1, 2, 30], 4, 2, 64, 16, block, seed=8, grow=1.0, scale=2.0 ** -12)
    kv = c.qkv[:, c.heads * c.width:]
    kv.copy_((kv.float() * grow).clamp(-65504, 65504).half())
    check(Run(flint, cuda, c).run())


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [3.0, -3.0, 0.0, 1e-30])
@pytest.mark.parametrize("heads,new,width", [(4, 1, 64), (32, 1, 128), (24, 1, 64), (4, 70, 128)])
def test_scales_of_the_scores(flint, cuda, heads, new, width, scale):
    """Scores of deviation 24 and more move the softmax's reference again and again."""
    check(Run(flint, cuda, Cache([700, 33], [new, 1], heads, 1, width, 16, 16, seed=24,
                                 scale=scale)).run())


@pytest.mark.gpu
def test_pages_past_4_gib(flint, cuda):
    """The last pages of a pool of 5 GB, of K and of V."""
    c = Cache([150, 64], [1, 3], 8, 8, 128, 64, 32, seed=25)
    per = c.kv_heads * c.page_size * c.width
    shift = (5 << 30) // per
    small = Run(flint, cuda, c)
    big = Run(flint, cuda, c)
    for name in ("codes", "bytes"):
        pools = []
        for x in getattr(small, name):
            pool = torch.zeros((shift + len(x),) + x.shape[1:], dtype=torch.uint8, device=cuda)
            pool[shift:] = x
            pools.append(pool)
        setattr(big, name, pools)
    big.table = torch.where(small.table >= 0, small.table + shift, -1)
    big.shape.pages = shift + c.pages
    small.run()
    big.run()
    check(small)
    assert torch.equal(big.o, small.o)
    for a, b in zip(big.codes + big.bytes, small.codes + small.bytes):
        assert torch.equal(a[shift:], b)
        assert int(a[:shift].count_nonzero()) == 0


@pytest.mark.gpu
def test_zero_rows_and_largest_values(flint, cuda):
    c = Cache([20, 9], [1, 1], 2, 1, 64, 16, 16, seed=9, scale=1e-3)
    w, hw = c.width, c.heads * c.width
    c.qkv[0, hw:hw + w] = 0.0
    c.qkv[1, hw:hw + w] = torch.tensor([65504.0, -65504.0, 61440.0, 57344.0, 448.0, 464.0, 0.0, -0.0] * 8)
    c.qkv[1, hw + w:] = torch.tensor([2.0 ** -24, 2.0 ** -14, -2.0 ** -20, 1.75 * 2.0 ** -7] * 16)
    check(Run(flint, cuda, c).run())


@pytest.mark.gpu
def test_every_code_and_scale_is_read(flint, cuda):
    """o of a token that sees one cached position nearly alone is that position's v."""
    codes = torch.arange(256, dtype=torch.uint8)
    codes = torch.where((codes & 0x7F) == NAN_CODE, 0x38, codes)
    for width in (64, 128):
        for byte in (0, 112, 120, 127, 134, 135, 255):
            c = Cache([32], [1], 1, 1, width, 32, 32, seed=10, scale=1.0)
            most = 240 if byte >= 135 else 448
            x = codes.view(torch.float8_e4m3fn).float()
            fit = torch.where(x.abs() > most, 0x38, codes)
            page = int(c.table[0, 0])
            c.codes[1][page, 0] = fit[torch.arange(32 * width) % 256].view(32, width)
            c.bytes[1][page, 0, 0] = byte
            c.codes[0][page, 0] = 0
            c.codes[0][page, 0, 13] = 0x7E          # 448 in every column of position 13
            c.bytes[0][page, 0, 0] = 127
            c.qkv[:, :width] = 1.0
            check(Run(flint, cuda, c).run())


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 33])
def test_pages_that_are_none(flint, cuda, new):
    """Entries outside the pool: their positions are not seen, new rows there not
    stored."""
    dropped = [(0, 1, -1), (0, 5, 1 << 30), (1, 0, -7)]
    check(Run(flint, cuda, Cache([100, 20], [new, new], 4, 2, 64, 16, 8, seed=11,
                                 dropped=dropped)).run())
    c = Cache([16], [1], 1, 1, 64, 16, 16, seed=12, dropped=[(0, 0, -1), (0, 1, -1)])
    check(Run(flint, cuda, c).run())


@pytest.mark.gpu
def test_lengths_past_the_table(flint, cuda):
    c = Cache([60, 30], [3, 2], 2, 1, 64, 16, 16, seed=13, spare_columns=0)
    c.cached = [64, 1 << 30]     # past the columns: taken into them, and no page for new rows
    for which in range(2):       # what is then read holds values
        c.codes[which][(c.codes[which] & 0x7F) == NAN_CODE] = 0x30
        c.bytes[which][c.bytes[which] == 255] = 127
    c.table[c.table < 0] = 0
    check(Run(flint, cuda, c).run())


@pytest.mark.gpu
def test_new_tokens_past_max_new_are_left(flint, cuda):
    check(Run(flint, cuda, Cache([50, 8], [9, 3], 2, 1, 128, 8, 8, seed=14, max_new=4)).run())


@pytest.mark.gpu
def test_shared_prefix(flint, cuda):
    check(Run(flint, cuda, Cache([64, 70, 90], [1, 1, 5], 4, 2, 64, 16, 16, seed=15, shared=2)).run())


@pytest.mark.gpu
def test_a_sequence_that_is_not_finite_leaves_the_others(flint, cuda):
    base = Cache([40, 50, 33], [1, 2, 1], 2, 1, 64, 16, 8, seed=16)
    clean = Run(flint, cuda, base).run()
    c = Cache([40, 50, 33], [1, 2, 1], 2, 1, 64, 16, 8, seed=16)
    c.qkv[1, c.heads * c.width + 3] = float("inf")       # a key of sequence 1
    c.codes[1][c.page(1, 17), 0, 1, 5] = NAN_CODE        # a cached value of it
    r = Run(flint, cuda, c).run()
    for at in (0, 3):
        assert torch.equal(r.o[at], clean.o[at])
    assert not torch.isfinite(r.o[1:3, :128]).all()
    stored = r.codes[0][c.page(1, 50), 0, 50 % 16].cpu()
    assert int(stored[3]) & 0x7F == NAN_CODE
    _, _, codes, scales, _ = c.reference()
    assert torch.equal(r.bytes[0].cpu(), scales[0]) and torch.equal(r.bytes[1].cpu(), scales[1])


@pytest.mark.gpu
def test_token_by_token_is_the_cache_of_the_chunk(flint, cuda):
    """Blocks of one position: the bytes do not depend on how the rows came, and equal
    those of one call."""
    n, H, Hk, w, size = 41, 4, 2, 64, 16
    qkv = normal((n, (H + 2 * Hk) * w), 17, 1.0, torch.float16).to(cuda)
    q, k, v = qkv[:, :H * w], qkv[:, H * w:(H + Hk) * w], qkv[:, (H + Hk) * w:]
    table = torch.tensor([[2, 0, 3]], dtype=torch.int32, device=cuda)

    def pools():
        return ([torch.zeros((4, Hk, size, w), dtype=torch.uint8, device=cuda) for _ in "kv"],
                [torch.zeros((4, Hk, size), dtype=torch.uint8, device=cuda) for _ in "kv"])

    def call(pool, first, count):
        (kp, vp), (ks, vs) = pool
        o = torch.empty((count, H * w), dtype=torch.float16, device=cuda)
        shape = flint.paged_shape(count, 1, count, H, Hk, w, *[qkv.shape[1]] * 2, H * w, 4, size, 3)
        rows = slice(first, first + count)
        flint.attention_paged8(o, kp, ks, vp, vs, q[rows], k[rows], v[rows],
                               torch.tensor([0, count], dtype=torch.int32, device=cuda),
                               torch.tensor([first], dtype=torch.int32, device=cuda), table, shape,
                               1, 0.125)
        return o

    one, steps = pools(), pools()
    call(one, 0, n)
    for t in range(n):
        call(steps, t, 1)
    for a, b in zip(one[0] + one[1], steps[0] + steps[1]):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_two_runs_are_bit_identical(flint, cuda):
    c = Cache([3000, 100, 800], [1, 1, 1], 8, 2, 128, 16, 16, seed=18)
    one, two = Run(flint, cuda, c).run(), Run(flint, cuda, c).run()
    assert torch.equal(one.o, two.o) and torch.equal(one.codes[0], two.codes[0])


@pytest.mark.gpu
def test_captured_and_replayed_with_other_lengths(flint, cuda):
    """Two graphs over one workspace; lengths change between replays."""
    runs = [Run(flint, cuda, Cache([2000, 40], [1, 1], 4, 2, 64, 16, 16, seed=19)),
            Run(flint, cuda, Cache([300, 900], [50, 1], 4, 2, 64, 16, 8, seed=20))]
    size = max(r.ws.numel() for r in runs)
    ws = torch.full((size,), 0xA5, dtype=torch.uint8, device=cuda)
    stream = torch.cuda.Stream()
    graphs, refs, before = [], [], []
    for r in runs:
        r.ws = ws
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            r.run()
        graphs.append(graph)
        refs.append(r.c.reference())
        before.append([x.clone() for x in r.codes + r.bytes])
    for _ in range(3):
        for r, g, old in zip(runs, graphs, before):
            for x, y in zip(r.codes + r.bytes, old):
                x.copy_(y)
            r.o.fill_(SENTINEL)
            g.replay()
        for r, ref in zip(runs, refs):
            hw = r.c.heads * r.c.width
            assert worst(r.o.cpu()[:, :hw], ref[0], ref[1]) <= 1.0
            for want, have in zip(ref[2] + ref[3], r.codes + r.bytes):
                assert torch.equal(want, have.cpu())
    c = runs[0].c
    c.cached = [77, 39]
    runs[0].cached.copy_(torch.tensor(c.cached, dtype=torch.int32))
    c.codes, c.bytes = ([x.cpu() for x in y] for y in (runs[0].codes, runs[0].bytes))
    runs[0].need = runs[0].ws.numel()
    ref = c.reference()
    graphs[0].replay()
    check(runs[0], ref)


@pytest.mark.gpu
def test_on_another_stream(flint, cuda):
    r = Run(flint, cuda, Cache([500, 20], [1, 1], 4, 2, 64, 16, 16, seed=21))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    r.run(stream=stream)
    stream.synchronize()
    check(r)


@pytest.mark.gpu
def test_offsets_that_decrease_stay_inside(flint, cuda):
    """Nothing outside the outputs is written, whatever the offsets are."""
    c = Cache([40, 40, 40], [4, 4, 4], 4, 2, 64, 16, 8, seed=22)
    r = Run(flint, cuda, c)
    r.offsets.copy_(torch.tensor([8, 3, 12, -5], dtype=torch.int32))
    r.run()
    torch.cuda.synchronize()
    assert torch.all(r.ws[r.need:] == 0xA5)
    assert torch.all(r.o[:, c.heads * c.width:] == SENTINEL)


# ------------------------------------------------------------------ refusals

A = 0x1000000   # a 16-byte-aligned fake device address: refusals never read it


def fails(flint, fn, *args, message):
    status = getattr(flint.lib, fn)(*args)
    assert status == flint_lib.ERROR_INVALID_ARGUMENT
    assert message in flint.last_error(), flint.last_error()


def shape_of(flint, **changes):
    s = flint.paged_shape(3, 2, 2, 4, 2, 64, 256, 128, 256, 20, 16, 9)
    for name, value in changes.items():
        setattr(s, name, value)
    return s


@pytest.mark.parametrize("changes,block,message", [
    (dict(head_width=80), 8, "head_width (80) must be 64 or 128"),
    (dict(kv_heads=3), 8, "kv_heads (3) must divide heads (4)"),
    (dict(page_size=12), 4, "page_size (12) must be a multiple of 8"),
    (dict(q_stride=250), 8, "q_stride (250) must be a multiple of 8 from 256"),
    (dict(), 0, "block (0) must be a power of two up to 128 that divides page_size (16)"),
    (dict(), 3, "block (3) must be a power of two"),
    (dict(), 32, "block (32) must be a power of two up to 128 that divides page_size (16)"),
    (dict(page_size=24), 16, "block (16) must be a power of two up to 128 that divides page_size (24)"),
    (dict(page_size=256), 256, "block (256) must be a power of two up to 128"),
])
def test_shapes_refused(flint, changes, block, message):
    s = shape_of(flint, **changes)
    fails(flint, "flint_attention_paged8_workspace", s, block, ctypes.c_size_t(0),
          message=f"flint_attention_paged8_workspace: {message}")
    fails(flint, "flint_attention_paged8", *[(i + 1) * A for i in range(11)], s, block,
          ctypes.c_float(0.1), 12 * A, 1 << 20, None, message=f"flint_attention_paged8: {message}")


def test_buffers_refused(flint):
    s = shape_of(flint)
    f = ctypes.c_float(0.125)
    fn = "flint_attention_paged8"
    good = [(i + 1) * A for i in range(11)]
    names = ("o", "k_pages", "k_scales", "v_pages", "v_scales", "q", "k", "v", "offsets", "cached",
             "table")
    for i, name in enumerate(names):
        bad = list(good)
        bad[i] = None
        fails(flint, fn, *bad, s, 8, f, 12 * A, 1 << 24, None, message=f"{fn}: {name} is null")
        bad[i] = good[i] + 4
        fails(flint, fn, *bad, s, 8, f, 12 * A, 1 << 24, None,
              message=f"{name} is not 16-byte aligned")
        for j in range(i + 1, 11):
            if i < 5:
                bad = list(good)
                bad[j] = bad[i]
                fails(flint, fn, *bad, s, 8, f, 12 * A, 1 << 24, None,
                      message=f"{names[i]} and {names[j]} overlap")
    need = flint.attention_paged8_workspace(s, 8)
    assert need > 0
    for at in good:
        fails(flint, fn, *good, s, 8, f, at, need, None, message="workspace and")
    fails(flint, fn, *good, s, 8, f, None, 0, None, message=f"needs {need} bytes of workspace")
    fails(flint, fn, *good, s, 8, f, 12 * A, need - 1, None, message=f"needs {need} bytes")
    fails(flint, fn, *good, s, 8, ctypes.c_float(float("nan")), 12 * A, need, None,
          message="scale (nan) must be finite")
    fails(flint, fn, *good, s, 8, ctypes.c_float(1e30), 12 * A, need, None,
          message="scale (1e+30) can be up to 1.84467e+19 in size")
    fails(flint, fn, *good, None, 8, f, 12 * A, need, None, message="shape is null")


def test_nothing_to_do(flint):
    f = ctypes.c_float(0.125)
    for none in (dict(tokens=0), dict(sequences=0), dict(max_new=0)):
        s = shape_of(flint, **none)
        assert flint.lib.flint_attention_paged8(*[None] * 11, s, 8, f, None, 0, None) == 0
        out = ctypes.c_size_t(5)
        assert flint.lib.flint_attention_paged8_workspace(s, 8, out) == 0 and out.value == 0


def test_the_codes_of_the_tests_are_the_formats():
    """e4m3 as torch has it: 1 sign, 4 exponent (bias 7), 3 mantissa bits."""
    codes = torch.arange(127, dtype=torch.uint8)
    want = [m / 8.0 * 2.0 ** -6 if e == 0 else (1 + m / 8.0) * 2.0 ** (e - 7)
            for e in range(16) for m in range(8)][:127]
    assert codes.view(torch.float8_e4m3fn).double().tolist() == want
    assert code_of(torch.tensor([464.0, 1e9, -1e9], dtype=torch.float64), 0).tolist() == [
        0x7E, 0x7E, 0xFE]
    assert [exponent_of(torch.tensor([x])) for x in (0.0, 448.0, 449.0, 57344.0, 65504.0)] == [
        -15, 0, 1, 7, 8]
