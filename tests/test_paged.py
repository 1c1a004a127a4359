"""Attention of new tokens over a paged cache (include/flint/flint_paged.h)
against float64, within bounds counted in rounding steps
(attention_bounds.py); what it stores and what it leaves; its refusals."""

import ctypes
import math

import pytest
import torch

from attention_bounds import Z, attend, worst
from flint_amd import flint_lib
from inputs import gen, normal

SENTINEL = 7.25
NAN = float("nan")


class Cache:
    """Sequences with cached positions and new tokens, on the CPU. Every cache
    row that holds no position is NaN."""

    def __init__(self, cached, new, heads, kv_heads, width, page_size, seed=1, max_new=None,
                 spare_columns=1, after=0, scale=None, shared=0, dropped=()):
        self.cached, self.new = cached, new
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
        self.k_pages = torch.full(pool, NAN, dtype=torch.float16)
        self.v_pages = torch.full(pool, NAN, dtype=torch.float16)
        fill = normal((2,) + pool, seed + 1, 1.0, torch.float16)
        for s, c in enumerate(cached):
            for p in range(0, c, page_size):
                page = self.page(s, p)
                if page is not None:
                    rows = min(page_size, c - p)
                    self.k_pages[page, :, :rows] = fill[0, page, :, :rows]
                    self.v_pages[page, :, :rows] = fill[1, page, :, :rows]
        self.offsets = [0]
        for n in new:
            self.offsets.append(self.offsets[-1] + n)
        self.tokens = self.offsets[-1] + after
        self.qkv = normal((self.tokens, (heads + 2 * kv_heads) * width), seed + 2, 1.0,
                          torch.float16)
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
        """(o, bound) as tokens x (heads x width), the pages after the call, and
        which rows of o are written."""
        H, Hk, w = self.heads, self.kv_heads, self.width
        q, k, v = self.parts(self.qkv)
        o = torch.zeros(self.tokens, H * w, dtype=torch.float64)
        bound = torch.zeros_like(o)
        done = torch.zeros(self.tokens, dtype=torch.bool)
        kp, vp = self.k_pages.clone(), self.v_pages.clone()
        for s, (c, n) in enumerate(zip(self.cached, self.new)):
            n, t = min(n, self.max_new), self.offsets[s]
            places = [(self.page(s, p), p % self.page_size) for p in range(c + n)]
            held = [i for i in range(c) if places[i][0] is not None]
            for i in range(n):
                page, row = places[c + i]
                if page is not None:
                    kp[page, :, row] = k[t + i].view(Hk, w)
                    vp[page, :, row] = v[t + i].view(Hk, w)
            done[t:t + n] = True
            visible = torch.cat([torch.ones(n, len(held), dtype=torch.bool),
                                 torch.ones(n, n, dtype=torch.bool).tril()], 1)
            for h in range(H if n else 0):
                j = h // (H // Hk)
                keys, values = (
                    torch.cat([pool[[places[i][0] for i in held], j, [places[i][1] for i in held]],
                               new[t:t + n, j * w:j * w + w]])
                    for pool, new in ((self.k_pages, k), (self.v_pages, v)))
                got = attend(q[t:t + n, h * w:h * w + w], keys, values, self.scale, visible)["o"]
                o[t:t + n, h * w:h * w + w], bound[t:t + n, h * w:h * w + w] = got
        return o, bound, kp, vp, done


class Run:
    def __init__(self, flint, cuda, c):
        self.flint, self.c = flint, c
        self.qkv = c.qkv.to(cuda)
        self.q, self.k, self.v = c.parts(self.qkv)
        self.k_pages, self.v_pages = c.k_pages.to(cuda), c.v_pages.to(cuda)
        self.table = c.table.to(cuda)
        self.offsets = torch.tensor(c.offsets, dtype=torch.int32, device=cuda)
        self.cached = torch.tensor(c.cached, dtype=torch.int32, device=cuda)
        self.o = torch.full((c.tokens, c.heads * c.width), SENTINEL, dtype=torch.float16,
                            device=cuda)
        wide = self.qkv.shape[1]
        self.shape = flint.paged_shape(c.tokens, len(c.cached), c.max_new, c.heads, c.kv_heads,
                                       c.width, wide, wide, c.heads * c.width, c.pages,
                                       c.page_size, c.table.shape[1])
        self.ws = torch.full((max(16, flint.attention_paged_workspace(self.shape)),), 0xFF,
                             dtype=torch.uint8, device=cuda)

    def run(self, stream=None):
        self.flint.attention_paged(self.o, self.k_pages, self.v_pages, self.q, self.k, self.v,
                                   self.offsets, self.cached, self.table, self.shape,
                                   self.c.scale, self.ws, stream=stream)
        return self


def same_bits(a, b):
    return torch.equal(a.cpu().view(torch.int16), b.cpu().view(torch.int16))


def check(run, reference=None):
    torch.cuda.synchronize()
    o, bound, kp, vp, done = run.c.reference() if reference is None else reference
    got = run.o.cpu()
    if bool(done.any()):
        off = worst(got[done], o[done], bound[done])
        print(f"o: {off:.2f} of the bound")
        assert off <= 1.0
    assert bool((got[~done] == SENTINEL).all())
    assert same_bits(run.k_pages, kp) and same_bits(run.v_pages, vp)


@pytest.mark.gpu
@pytest.mark.parametrize("width", [64, 128])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (3, 3), (6, 2), (9, 1)])
@pytest.mark.parametrize("cached,page_size", [([0], 8), ([1], 16), ([63, 64, 65], 16),
                                              ([200, 0, 7, 129], 24), ([700], 64), ([31, 300], 128)])
def test_single_tokens(flint, cuda, cached, page_size, heads, kv_heads, width):
    check(Run(flint, cuda, Cache(cached, [1] * len(cached), heads, kv_heads, width, page_size,
                                 seed=sum(cached) + heads)).run())


@pytest.mark.gpu
@pytest.mark.parametrize("width", [64, 128])
@pytest.mark.parametrize("heads,kv_heads", [(2, 2), (6, 2), (8, 1)])
@pytest.mark.parametrize("cached,new", [([0], [5]), ([3, 64], [64, 1]), ([100, 0, 31], [33, 130, 2]),
                                        ([500], [200])])
def test_chunks(flint, cuda, cached, new, heads, kv_heads, width):
    check(Run(flint, cuda, Cache(cached, new, heads, kv_heads, width, 16,
                                 seed=sum(cached) + sum(new))).run())


@pytest.mark.gpu
@pytest.mark.parametrize("width", [64, 128])
def test_many_rows_in_several_parts(flint, cuda, width):
    """More than 4,096 rows of o whose sequences are cut into parts."""
    check(Run(flint, cuda, Cache([900, 1300], [290, 230], 8, 2, width, 32, seed=21)).run())
    check(Run(flint, cuda, Cache([2000], [600], 7, 1, width, 16, seed=22)).run())


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 9])
def test_more_sequences_than_a_wave_has_lanes(flint, cuda, new):
    cached = [(i * 37) % 400 for i in range(150)]
    chunk = [(i * 5) % (new + 1) if new > 1 else 1 for i in range(150)]
    check(Run(flint, cuda, Cache(cached, chunk, 4, 1, 64, 16, seed=23)).run())


@pytest.mark.gpu
def test_one_long_sequence_in_many_parts(flint, cuda):
    check(Run(flint, cuda, Cache([60000], [1], 2, 1, 64, 64, seed=24)).run())
    check(Run(flint, cuda, Cache([30000], [40], 1, 1, 128, 128, seed=25)).run())


@pytest.mark.gpu
def test_so_many_tiles_that_the_parts_take_two_rounds(flint, cuda):
    """64 tiles for each of the 16 items that one of 64 heads of K and V gets."""
    c = Cache([2100 - 3 * s for s in range(16)], [1] * 16, 64, 64, 64, 64, seed=30, shared=32)
    check(Run(flint, cuda, c).run())


@pytest.mark.gpu
def test_a_long_cache_and_an_empty_one(flint, cuda):
    check(Run(flint, cuda, Cache([9000, 0, 4097], [1, 1, 1], 4, 2, 64, 32, seed=4)).run())
    check(Run(flint, cuda, Cache([5000, 3], [7, 2], 4, 4, 128, 64, seed=5)).run())


@pytest.mark.gpu
def test_sequences_without_new_tokens_and_rows_behind_the_last(flint, cuda):
    check(Run(flint, cuda, Cache([40, 90, 17], [3, 0, 2], 4, 2, 64, 16, seed=6, after=9)).run())


@pytest.mark.gpu
@pytest.mark.parametrize("entry", [-1, -2 ** 31, 1 << 20])
def test_positions_without_a_page(flint, cuda, entry):
    """Dropped pages in the middle, at the front and where new rows would go."""
    c = Cache([200, 70, 33], [4, 1, 16], 4, 2, 64, 16, seed=7,
              dropped=[(0, 0, entry), (0, 5, entry), (1, 1, entry), (2, 2, entry)])
    check(Run(flint, cuda, c).run())


@pytest.mark.gpu
def test_every_cached_page_dropped(flint, cuda):
    c = Cache([64, 2000], [1, 3], 2, 1, 64, 32, seed=8,
              dropped=[(0, i, -1) for i in range(2)] + [(1, i, -1) for i in range(62)])
    check(Run(flint, cuda, c).run())


@pytest.mark.gpu
def test_a_table_too_short_for_the_new_tokens(flint, cuda):
    check(Run(flint, cuda, Cache([30], [40], 2, 2, 64, 16, seed=9, spare_columns=-2)).run())


@pytest.mark.gpu
def test_tokens_past_max_new_are_ignored(flint, cuda):
    check(Run(flint, cuda, Cache([50, 20], [9, 3], 4, 2, 64, 16, seed=10, max_new=5)).run())


@pytest.mark.gpu
def test_a_shared_prefix(flint, cuda):
    check(Run(flint, cuda, Cache([160, 150, 129], [1, 6, 2], 4, 4, 64, 32, seed=11, shared=4)).run())


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [-0.2, 0.0, 1.0])
def test_any_finite_scale(flint, cuda, scale):
    check(Run(flint, cuda, Cache([300, 10], [1, 40], 2, 1, 64, 16, seed=12, scale=scale)).run())


@pytest.mark.gpu
@pytest.mark.parametrize("width", [64, 128])
@pytest.mark.parametrize("new", [1, 40])
def test_a_key_that_outweighs_the_others_by_far(flint, cuda, new, width):
    """The first key is 2^25 to 2^27 times as likely as each other one and its
    value is 0: o is what the others add up to. Probabilities are rounded at 2^5
    times their size, so half a step among FP16's subnormals is 2^-30."""
    n = 250
    c = Cache([n], [new], 1, 1, width, 64, seed=33, scale=8.0 / width)   # scores: 8 k
    spread = torch.rand(n + new, generator=gen(34)) * -0.09
    spread[0] = 2.21
    q, k, v = c.parts(c.qkv)
    q[:], k[:], v[:] = 1.0, spread[n:, None], 64.0
    for p in range(n):
        c.k_pages[c.page(0, p), :, p % 64] = spread[p]
        c.v_pages[c.page(0, p), :, p % 64] = 64.0 if p else 0.0
    o, bound, kp, vp, done = c.reference()
    reach = 64.0 * torch.arange(n, n + new, dtype=torch.float64)[:, None]
    check(Run(flint, cuda, c).run(), (o, bound - 1.05 * (Z - 2.0 ** -30) * reach, kp, vp, done))


@pytest.mark.gpu
def test_a_long_group_of_heads(flint, cuda):
    check(Run(flint, cuda, Cache([100, 700], [1, 3], 48, 1, 64, 16, seed=13)).run())


@pytest.mark.gpu
def test_cache_offsets_past_32_bits(flint, cuda):
    """Pages whose values lie past 2^32 bytes in their tensor."""
    width, size, heads = 128, 256, 2
    pages = (1 << 32) // (heads * size * width * 2) + 40
    k_pages = torch.zeros((pages, heads, size, width), dtype=torch.float16, device=cuda)
    v_pages = torch.zeros_like(k_pages)
    c = Cache([700, 300], [1, 2], heads, heads, width, size, seed=14)
    ref = c.reference()
    c.table = torch.where(c.table >= 0, c.table + pages - c.pages, -1).to(torch.int32)
    k_pages[-c.pages:], v_pages[-c.pages:] = c.k_pages.to(cuda), c.v_pages.to(cuda)
    small, c.pages = c.pages, pages
    r = Run(flint, cuda, c)
    r.k_pages, r.v_pages = k_pages, v_pages
    r.run()
    assert not bool(k_pages[:-small].any()) and not bool(v_pages[:-small].any())
    r.k_pages, r.v_pages = k_pages[-small:], v_pages[-small:]
    check(r, ref)


@pytest.mark.gpu
def test_step_after_step_matches_one_chunk(flint, cuda):
    """Tokens taken one at a time, each call storing for the next, against the
    same tokens in one chunk."""
    c = Cache([37], [12], 4, 2, 64, 16, seed=15)
    check(Run(flint, cuda, c).run())
    r = Run(flint, cuda, c)
    shape = flint.paged_shape(1, 1, 1, c.heads, c.kv_heads, c.width, *[r.qkv.shape[1]] * 2,
                              c.heads * c.width, c.pages, c.page_size, c.table.shape[1])
    offsets = torch.tensor([0, 1], dtype=torch.int32, device=cuda)
    for t in range(12):
        flint.attention_paged(r.o[t], r.k_pages, r.v_pages, r.q[t], r.k[t], r.v[t], offsets,
                              r.cached, r.table, shape, c.scale)
        r.cached += 1
    check(r)


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 30])
def test_offsets_that_decrease_stay_inside(flint, cuda, new):
    c = Cache([500, 40, 3000, 7], [new] * 4, 4, 2, 64, 16, seed=31, after=9)
    r = Run(flint, cuda, c)
    n = 4 * new
    r.offsets = torch.tensor([n, 0, n, -5, n], dtype=torch.int32, device=cuda)
    r.run()
    torch.cuda.synchronize()
    assert torch.all(r.o[n:] == SENTINEL)


@pytest.mark.gpu
def test_offsets_that_decrease_stay_inside_the_workspace(flint, cuda):
    """Five times the same 100 tokens: 60 parts, where 48 is the most."""
    c = Cache([700] * 10, [10] * 10, 3, 1, 64, 16, seed=32, max_new=100)
    r = Run(flint, cuda, c)
    need = flint.attention_paged_workspace(r.shape)
    r.ws = torch.full((need + (1 << 20),), 0x5A, dtype=torch.uint8, device=cuda)
    r.offsets = torch.tensor([0, 100] * 5 + [0], dtype=torch.int32, device=cuda)
    flint.attention_paged(r.o, r.k_pages, r.v_pages, r.q, r.k, r.v, r.offsets, r.cached, r.table,
                          r.shape, c.scale, r.ws, workspace_bytes=need)
    torch.cuda.synchronize()
    assert torch.all(r.ws[need:] == 0x5A)


@pytest.mark.gpu
@pytest.mark.parametrize("word", [0x3F800000, 0x00000002, 0x7FFFFFFF])
def test_offsets_that_decrease_past_the_grid_join_inside_the_workspace(flint, cuda, word):
    """3,968 blocks a head of K and V for 1,014 workgroups: the last sequence gets
    none, so its entry in the workspace is the word that lay there."""
    heads, S, n = 64, 999, 1000
    qkv = normal((n, 3 * heads * 64), 35, 1.0, torch.float16).to(cuda)
    q, k, v = (qkv[:, i * heads * 64:(i + 1) * heads * 64] for i in range(3))
    pages = torch.zeros((2, 70, heads, 16, 64), dtype=torch.float16, device=cuda)
    table = torch.arange(70, dtype=torch.int32, device=cuda).repeat(S, 1)
    shape = flint.paged_shape(n, S, n, heads, heads, 64, *[qkv.shape[1]] * 2, heads * 64, 70, 16, 70)
    offsets = torch.tensor([0, n] * 496 + [0] * 7 + [n], dtype=torch.int32, device=cuda)
    need = flint.attention_paged_workspace(shape)
    assert need > 0
    ws = torch.full((need // 4 + (1 << 18),), word, dtype=torch.int32, device=cuda)
    o = torch.full((n + 8, heads * 64), SENTINEL, dtype=torch.float16, device=cuda)
    flint.attention_paged(o, pages[0], pages[1], q, k, v, offsets,
                          torch.zeros(S, dtype=torch.int32, device=cuda), table, shape, 0.125, ws,
                          workspace_bytes=need)
    torch.cuda.synchronize()
    assert torch.all(ws[need // 4:] == word)
    assert torch.all(o[n:] == SENTINEL)


@pytest.mark.gpu
def test_two_runs_are_bit_identical(flint, cuda):
    c = Cache([3000, 100, 800], [1, 1, 1], 8, 2, 128, 16, seed=16)
    one, two = Run(flint, cuda, c).run().o, Run(flint, cuda, c).run().o
    assert same_bits(one, two)


@pytest.mark.gpu
def test_captured_and_replayed_with_other_lengths(flint, cuda):
    """Two graphs over one workspace; lengths and tables change between
    replays."""
    runs = [Run(flint, cuda, Cache([2000, 40], [1, 1], 4, 2, 64, 16, seed=17)),
            Run(flint, cuda, Cache([300, 900], [1, 1], 4, 2, 64, 16, seed=18, spare_columns=69))]
    size = max(r.ws.numel() for r in runs)
    ws = torch.empty(size, dtype=torch.uint8, device=cuda)
    stream = torch.cuda.Stream()
    graphs = []
    for r in runs:
        r.ws = ws
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            r.run()
        graphs.append(graph)
    refs = [r.c.reference() for r in runs]
    for _ in range(3):
        for r, g in zip(runs, graphs):
            r.o.fill_(SENTINEL)
            g.replay()
        for r, ref in zip(runs, refs):
            check(r, ref)
    # The first graph on a shorter cache in its own buffers.
    c = runs[0].c
    c.cached = [77, 39]
    runs[0].cached.copy_(torch.tensor(c.cached, dtype=torch.int32))
    c.k_pages, c.v_pages = runs[0].k_pages.cpu(), runs[0].v_pages.cpu()
    ref = c.reference()
    graphs[0].replay()
    check(runs[0], ref)


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


@pytest.mark.parametrize("changes,message", [
    (dict(head_width=80), "head_width (80) must be 64 or 128"),
    (dict(heads=1025), "heads (1025) must be from 1 to 1024"),
    (dict(kv_heads=3), "kv_heads (3) must divide heads (4)"),
    (dict(tokens=(1 << 20) + 1), "tokens (1048577) can be up to 1048576"),
    (dict(sequences=65536), "sequences (65536) can be up to 65535"),
    (dict(max_new=(1 << 20) + 1), "max_new (1048577) can be up to 1048576"),
    (dict(page_size=0), "page_size (0) must be a multiple of 8 from 8 to 65536"),
    (dict(page_size=12), "page_size (12) must be a multiple of 8"),
    (dict(pages=0), "pages (0) must be from 1 to 2147483647"),
    (dict(max_pages=0), "max_pages (0) must be from 1 to 67108864"),
    (dict(max_pages=(1 << 26) + 1), "max_pages (67108865) must be from 1 to 67108864"),
    (dict(q_stride=250), "q_stride (250) must be a multiple of 8 from 256"),
    (dict(kv_stride=64), "kv_stride (64) must be a multiple of 8 from 128"),
    (dict(o_stride=0), "o_stride (0) must be a multiple of 8 from 256"),
])
def test_shapes_refused(flint, changes, message):
    s = shape_of(flint, **changes)
    fails(flint, "flint_attention_paged_workspace", s, ctypes.c_size_t(0), message=message)
    fails(flint, "flint_attention_paged", *[(i + 1) * A for i in range(9)], s,
          ctypes.c_float(0.1), 10 * A, 1 << 20, None, message=message)


def test_buffers_refused(flint):
    s = shape_of(flint)
    f = ctypes.c_float(0.125)
    fn = "flint_attention_paged"
    good = [(i + 1) * A for i in range(9)]
    names = ("o", "k_pages", "v_pages", "q", "k", "v", "offsets", "cached", "table")
    for i, name in enumerate(names):
        bad = list(good)
        bad[i] = None
        fails(flint, fn, *bad, s, f, 10 * A, 1 << 24, None, message=f"{fn}: {name} is null")
        bad[i] = good[i] + 4
        fails(flint, fn, *bad, s, f, 10 * A, 1 << 24, None, message=f"{name} is not 16-byte aligned")
    same = list(good)
    same[2] = same[1]
    fails(flint, fn, *same, s, f, 10 * A, 1 << 24, None, message="k_pages and v_pages overlap")
    same = list(good)
    same[4] = same[1] + 64
    fails(flint, fn, *same, s, f, 10 * A, 1 << 24, None, message="k_pages and k overlap")
    fails(flint, fn, *good, s, ctypes.c_float(float("inf")), 10 * A, 1 << 24, None,
          message="scale (inf) must be finite")
    fails(flint, fn, *good, None, f, 10 * A, 1 << 24, None, message="shape is null")


@pytest.mark.parametrize("scale", [1e30, -3.4e38])
def test_scales_whose_scores_pass_fp32_are_refused(flint, scale):
    f = ctypes.c_float(scale)
    fails(flint, "flint_attention_paged", *[(i + 1) * A for i in range(9)], shape_of(flint), f, 10 * A,
          1 << 24, None, message=f"scale ({f.value:g}) can be up to 1.84467e+19 in size")


def test_a_pool_past_the_addresses_is_refused(flint):
    """Sizes whose bytes pass 2^64: nothing would be left for the overlap checks."""
    s = shape_of(flint, pages=(1 << 31) - 1, page_size=65536, heads=1024, kv_heads=1024,
                 head_width=128, q_stride=131072, kv_stride=131072, o_stride=131072, max_pages=1)
    fails(flint, "flint_attention_paged_workspace", s, ctypes.c_size_t(0),
          message="pages (2147483647) x page_size x kv_heads x head_width can be up to 70368744177664")
    s = shape_of(flint, pages=(1 << 31) - 1)
    assert flint.lib.flint_attention_paged_workspace(s, ctypes.c_size_t(0)) == 0


def test_nothing_to_do(flint):
    f = ctypes.c_float(0.125)
    for none in (dict(tokens=0), dict(sequences=0), dict(max_new=0)):
        s = shape_of(flint, **none)
        assert flint.lib.flint_attention_paged(*[None] * 9, s, f, None, 0, None) == 0
        out = ctypes.c_size_t(5)
        assert flint.lib.flint_attention_paged_workspace(s, out) == 0 and out.value == 0
