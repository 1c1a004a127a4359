"""Log probabilities of given tokens, entropy, top alternatives and the gradient
of the logits (include/flint/flint_logprobs.h) against float64; refusals.

Bounds. w = 2^-24 is half a step of FP32. g = scale (l - max) is two rounded
operations: 2 w |g| off; its exponential a further 4 w (the hardware's 2^x and
its argument, log2(e) g, rounded twice: 2 w |g| more). With G = the largest |g|
that matters (terms with g < -110 are below 2^-158 of the sum), an exponential
is off by e = (4 G + 4) w relative, the sum by that and the additions' own: FP32
partial sums of at most 512 terms a lane and 16 merges, 528 w. log S takes the
sum's relative error, s = e + 528 w, and half a step of itself."""

import ctypes
import math

import pytest
import torch

from flint_amd import flint_lib
from inputs import gen, normal

W, U, Z = 2.0 ** -24, 2.0 ** -11, 2.0 ** -25
SENTINEL = 7.25


def reference(logits, targets, vocab, scale, top, dlp=None, dh=None):
    x = scale * logits[:, :vocab].double()
    # log1p of the sum without the largest term: of a word 40 above the others
    # log p is -4e-15, half a step of float64 at 40.
    rest = torch.exp(x - x.amax(1, keepdim=True))
    rest[torch.arange(x.shape[0]), x.argmax(1)] -= 1.0
    lp = (x - x.amax(1, keepdim=True)) - torch.log1p(rest.sum(1, keepdim=True))
    p = torch.exp(lp)
    plp = torch.where(p > 0, p * lp, torch.where(p == 0, 0.0, p))
    entropy = -plp.sum(1)
    row = torch.arange(x.shape[0])
    has = targets < vocab
    logprob = torch.where(has, lp[row, targets.clamp(max=vocab - 1)], 0.0)
    ids = torch.sort(logits[:, :vocab].double() + 0.0, dim=1, descending=True,
                     stable=True).indices[:, :top]
    out = dict(logprob=logprob, entropy=entropy, ids=ids, values=lp.gather(1, ids))
    if dlp is not None:
        dlp = torch.where(has, dlp.double(), 0.0)[:, None]
        dh = torch.zeros_like(dlp) if dh is None else dh.double()[:, None]
        d = -torch.where(p > 0, p * (dlp + dh * (lp + entropy[:, None])), torch.where(p == 0, 0.0, p))
        d[row[has], targets[has]] += dlp[has, 0]
        out["d"] = torch.zeros(logits.shape, dtype=torch.float64)
        out["d"][:, :vocab] = scale * d
    # Bounds.
    g = (x - x.amax(1, keepdim=True)).nan_to_num(0.0, 0.0, 0.0).abs()
    near = torch.where(g < 110, g, 0.0)
    s = (4 * near.amax(1) + 532) * W
    logsum = (torch.logsumexp(x, 1) - x.amax(1)).nan_to_num(0.0)
    fixed = s + W * logsum
    out["logprob_bound"] = 1.05 * (fixed + 3 * W * g[row, targets.clamp(max=vocab - 1)]
                                   + 2 * W * logprob.abs().nan_to_num(0.0, 0.0, 0.0)) + 1e-38
    out["values_bound"] = 1.05 * (fixed[:, None] + 3 * W * g.gather(1, ids)
                                  + 2 * W * out["values"].abs().nan_to_num(0.0, 0.0, 0.0)) + 1e-38
    spread = (p * near).sum(1)   # -sum g p
    out["entropy_bound"] = 1.05 * (fixed + (2 * s + 532 * W) * spread + 4 * W * entropy.abs()) + 1e-38
    if dlp is not None:
        # log p is off by t, p by that relative and the exponential's 4 w, and
        # the entropy by its own bound; then the FP16 rounding.
        t = fixed[:, None] + 6 * W * near + 4 * W
        part = p * (dlp.abs() + dh.abs() * (near + logsum[:, None] + entropy[:, None].abs()))
        out["d_bound"] = U * out["d"].abs() + Z
        out["d_bound"][:, :vocab] += 1.05 * scale * (
            (t + 8 * W) * part + p * dh.abs() * (t + out["entropy_bound"][:, None])
            + 4 * W * d.abs())
    return out


class Rows:
    def __init__(self, cuda, rows, vocab, cols, top, seed, spread=3.0, scale=1.0):
        self.rows, self.vocab, self.cols, self.top, self.scale = rows, vocab, cols, top, scale
        self.logits = normal((rows, cols), seed, spread, torch.float16)
        self.targets = torch.randint(0, vocab, (rows,), generator=gen(seed + 1))
        self.dlp = normal((rows,), seed + 2, 1.0)
        self.dh = normal((rows,), seed + 3, 0.3)
        self.cuda = cuda

    def run(self, flint, entropy_gradient=True, in_place=False, stream=None):
        c, n = self.cuda, self.rows
        self.dev = self.logits.to(c)
        t16 = self.targets.to(torch.int32).to(torch.int16).to(c)
        one = lambda *size: torch.full(size, SENTINEL, device=c)   # noqa: E731
        self.out = dict(logprob=one(n), entropy=one(n), stats=one(n, 2))
        ids = values = None
        if self.top:
            ids = self.out["ids"] = torch.full((n, self.top), -1, dtype=torch.int32, device=c)
            values = self.out["values"] = one(n, self.top)
        flint.logprobs_forward(self.out["logprob"], self.out["entropy"], self.out["stats"], ids,
                               values, self.dev, t16, self.scale, n, self.vocab, self.cols,
                               self.top, stream=stream)
        d = self.dev if in_place else torch.full_like(self.dev, SENTINEL)
        flint.logprobs_backward(d, self.dlp.to(c), self.dh.to(c) if entropy_gradient else None,
                                self.dev, t16, self.out["entropy"] if entropy_gradient else None,
                                self.out["stats"], self.scale, n, self.vocab, self.cols,
                                stream=stream)
        self.out["d"] = d
        torch.cuda.synchronize()
        return {name: t.cpu() for name, t in self.out.items()}

    def reference(self, entropy_gradient=True):
        return reference(self.logits, self.targets, self.vocab, self.scale, self.top, self.dlp,
                         self.dh if entropy_gradient else None)


def check(got, ref, names=("logprob", "entropy", "values", "d")):
    for name in names:
        if name not in got:
            continue
        value, bound = ref[name], ref[name + "_bound"]
        g = got[name].double()
        nan = torch.isnan(value)
        assert torch.equal(torch.isnan(g), nan), name
        infinite = torch.isinf(value)
        assert torch.equal(g[infinite], value[infinite]), name
        fine = ~nan & ~infinite
        off = float(((g - value).abs() / bound)[fine].max()) if bool(fine.any()) else 0.0
        print(f"{name}: {off:.2f} of the bound")
        assert off <= 1.0, (name, off)
    if "ids" in got:
        assert torch.equal(got["ids"].long(), ref["ids"])


@pytest.mark.gpu
@pytest.mark.parametrize("rows,vocab,cols,top", [
    (1, 1, 8, 1), (3, 5, 8, 5), (7, 64, 64, 64), (5, 97, 104, 20), (33, 997, 1000, 20),
    (4, 2048, 2048, 64), (3, 2049, 2056, 7), (5, 8200, 8200, 1), (3, 16391, 16392, 40),
    (6, 50257, 50304, 20), (2, 50257, 50304, 0), (2, 65536, 65536, 64), (3, 65535, 65536, 3)])
def test_matches_float64(flint, cuda, rows, vocab, cols, top):
    r = Rows(cuda, rows, vocab, cols, top, seed=rows + vocab)
    check(r.run(flint), r.reference())


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [0.3, 1.0, 2.5, 1e-3])
@pytest.mark.parametrize("vocab", [300, 12000])
def test_scales(flint, cuda, scale, vocab):
    r = Rows(cuda, 9, vocab, vocab + 8 - vocab % 8, 10, seed=vocab, scale=scale)
    check(r.run(flint), r.reference())


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [1e5, 1e8, 1e9, 1e30, 3e38])
@pytest.mark.parametrize("vocab", [300, 12000])
def test_scales_that_leave_the_largest_words_alone(flint, cuda, vocab, scale):
    """1 / scale is a temperature near 0: one word, or equal ones, take the row.
    What passes FP32 (a log probability) or FP16 (a gradient) is infinite."""
    r = Rows(cuda, 60, vocab, vocab + 8 - vocab % 8, 10, seed=vocab, scale=scale)
    r.logits[20:40] -= 40                   # negative maxima
    r.logits[40:45] *= 1e-3                 # around 0, close together
    r.logits[45] = 0.0
    r.logits[46] = -65504.0
    r.logits[47] = 65504.0
    r.logits[48, 7] = r.logits[48, 90] = 30.0
    r.logits[49, 5:] = float("-inf")
    r.dh[:] = 0.0       # of equal words log p + entropy is 0, and scale times float64's roundings
    r.targets[:10] = r.logits[:10, :vocab].float().argmax(1)
    r.targets[48], r.targets[49] = 90, 2
    got, ref = r.run(flint), r.reference()
    for name, kind in (("logprob", torch.float32), ("values", torch.float32), ("d", torch.float16)):
        past = ref[name].abs() > torch.finfo(kind).max
        ref[name] = torch.where(past, ref[name] * math.inf, ref[name])
    check(got, ref)


@pytest.mark.gpu
def test_many_rows(flint, cuda):
    r = Rows(cuda, 3001, 250, 256, 5, seed=5)
    check(r.run(flint), r.reference())


@pytest.mark.gpu
@pytest.mark.parametrize("vocab,top", [(3000, 64), (9000, 5), (30000, 33), (50257, 64), (65536, 1)])
def test_many_rows_of_long_ones(flint, cuda, vocab, top):
    """More rows than the GPU has compute units: other workgroup sizes."""
    r = Rows(cuda, 300, vocab, (vocab + 7) // 8 * 8, top, seed=vocab)
    r.logits[7] = 0.25          # equal logits: the lowest columns
    r.logits[8, 40:] = float("-inf")
    r.logits[9] = (r.logits[9] * 0.3).round()
    r.targets[8] = 39
    check(r.run(flint), r.reference())


@pytest.mark.gpu
@pytest.mark.parametrize("vocab,top", [(33000, 7), (51208, 3)])
def test_more_long_rows_than_four_a_compute_unit(flint, cuda, vocab, top):
    r = Rows(cuda, 1026, vocab, vocab, top, seed=vocab)
    r.logits[1020] = -2.0
    check(r.run(flint), r.reference())


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [500, 1000, 2000, 9000, 50257])
@pytest.mark.parametrize("top", [40, 41, 64])
def test_many_alternatives(flint, cuda, vocab, top):
    """On both sides of the finer groups, for each size of workgroup."""
    r = Rows(cuda, 40, vocab, (vocab + 7) // 8 * 8, top, seed=vocab + top)
    r.logits[3, 50:] = float("-inf")
    r.targets[3] = 49
    check(r.run(flint), r.reference())


@pytest.mark.gpu
@pytest.mark.parametrize("vocab,period", [(50257, 1024), (2000, 64), (12000, 256)])
def test_largest_words_close_together(flint, cuda, vocab, period):
    """The largest words in half the threads' columns: the groups' maxima say
    little, and more words pass the border than are listed."""
    r = Rows(cuda, 4, vocab, (vocab + 7) // 8 * 8, 40, seed=vocab)
    chunk = torch.arange(r.cols) // 8 % period
    r.logits[:, chunk >= period // 2] -= 30
    check(r.run(flint), r.reference())


@pytest.mark.gpu
@pytest.mark.parametrize("left", [1, 3, 39])
@pytest.mark.parametrize("vocab", [997, 9000, 50257])
def test_a_mask_that_leaves_fewer_words_than_asked(flint, cuda, left, vocab):
    r = Rows(cuda, 5, vocab, (vocab + 7) // 8 * 8, 40, seed=vocab + left)
    keep = torch.randperm(vocab, generator=torch.Generator().manual_seed(left))[:left]
    masked = torch.full_like(r.logits, float("-inf"))
    masked[:, keep] = r.logits[:, keep]
    masked[4, :] = -1.0
    r.logits[:] = masked
    r.targets[:] = int(keep[0])
    check(r.run(flint), r.reference())


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [900, 20000])
@pytest.mark.parametrize("kind", ["equal", "zeros", "few values", "lowest", "masked", "ramp", "ends"])
def test_ties_and_masks(flint, cuda, kind, vocab):
    """Equal logits go to the lower column, -0 with +0; the type's lowest value
    and -inf as masks, also with fewer words left than alternatives asked."""
    r = Rows(cuda, 4, vocab, (vocab + 7) // 8 * 8, 33, seed=7)
    column = torch.arange(r.cols)
    if kind == "equal":
        r.logits[:] = 1.5
    elif kind == "zeros":
        r.logits[:] = torch.where(column % 3 == 0, -0.0, 0.0).half()
        r.logits[:, 700] = 1.0
    elif kind == "few values":
        r.logits[:] = (r.logits * 0.5).round()
    elif kind == "lowest":
        r.logits[:, 10:] = -65504.0
    elif kind == "masked":
        r.logits[:, 10:] = float("-inf")
        r.dh[:] = torch.tensor([3.0, -40.0, 1e4, 0.0])
        r.targets[0] = 20          # a target of probability 0
    elif kind == "ramp":
        r.logits[:] = (column.float() / r.cols * 10).half()
    else:
        r.logits[:, :] = -3.0
        r.logits[:, -1 - (r.cols - vocab)] = 4.0
        r.logits[:, 0] = 4.0
    ref = r.reference()
    if kind == "masked":
        # dlogprob of a target of probability 0 reaches its column as it is.
        assert bool(torch.isinf(ref["logprob"][0]))
    check(r.run(flint), ref)


@pytest.mark.gpu
def test_peaked_rows_keep_their_small_values(flint, cuda):
    """A word far above the others: logprob and entropy are tiny and still right
    relative to themselves (log1p of the rest of the sum)."""
    r = Rows(cuda, 6, 1000, 1000, 2, seed=8, spread=0.5)
    lead = torch.tensor([6.0, 10.0, 14.0, 18.0, 24.0, 40.0])
    r.logits[torch.arange(6), r.targets] = lead.half()
    got, ref = r.run(flint), r.reference()
    check(got, ref)
    for name in ("logprob", "entropy"):
        off = ((got[name].double() - ref[name]) / ref[name]).abs()
        # e, twice over for the product with g, and the sums' own roundings.
        bound = (10 * lead.double() + 1100) * W
        assert bool((off <= bound).all()), (name, off / bound)


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [1000, 30000])
def test_peaked_rows_keep_their_gradient(flint, cuda, vocab):
    """dlogprob (1 - p) at a target of probability near 1, right relative to
    itself: log p's relative error, two steps of FP32 for 1 - p, and FP16's."""
    r = Rows(cuda, 7, vocab, vocab, 0, seed=18, spread=0.5)
    lead = torch.tensor([8.0, 12.0, 16.0, 18.0, 20.0, 24.0, 30.0]) + math.log(vocab / 1000)
    r.logits[torch.arange(7), r.targets] = lead.half()
    r.dlp[:] = 6e4 * torch.tensor([1.0, -1.0, 1.0, 1.0, -1.0, 1.0, 1.0])
    got, ref = r.run(flint, entropy_gradient=False), r.reference(entropy_gradient=False)
    check(got, ref)
    at = torch.arange(7), r.targets
    # 1 - p from the sum of the others' exponentials: float64 keeps it whole.
    others = r.logits.double()
    others = torch.exp(others - others[at][:, None])
    others[at] = 0.0
    others = others.sum(1)
    want = r.dlp.double() * others / (1 + others)
    bound = ((10 * lead.double() + 1110) * W + U) * want.abs() + Z
    off = (got["d"][at].double() - want).abs()
    assert bool((off <= bound).all()), off / bound


@pytest.mark.gpu
def test_not_a_number_and_infinity(flint, cuda):
    r = Rows(cuda, 5, 700, 704, 4, seed=9)
    r.logits[1, 13] = float("nan")
    r.logits[2, 500] = float("inf")
    r.logits[3, :] = float("-inf")
    got, ref = r.run(flint), r.reference()
    for name in ("logprob", "entropy", "values"):
        assert bool(torch.isnan(got[name][1:4]).all()), name
    assert bool(torch.isnan(got["d"][1:4, :700]).all())
    assert bool((got["d"][:, 700:] == 0).all())
    assert int(got["ids"][1, 0]) == 13 and int(got["ids"][2, 0]) == 500
    assert got["ids"][3].tolist() == [0, 1, 2, 3]
    for name in ("logprob", "entropy", "values", "d"):
        for row in (0, 4):
            off = (got[name][row].double() - ref[name][row]).abs() / ref[name + "_bound"][row]
            assert float(off.max()) <= 1.0, name


@pytest.mark.gpu
def test_padding_columns_do_not_count(flint, cuda):
    r = Rows(cuda, 4, 1001, 1064, 12, seed=10)
    want = r.run(flint)
    r.logits[:, 1001:] = float("nan")
    got = r.run(flint)
    for name in want:
        assert torch.equal(got[name], want[name]), name
    assert bool((got["d"][:, 1001:] == 0).all())


@pytest.mark.gpu
def test_rows_without_a_target(flint, cuda):
    r = Rows(cuda, 6, 500, 504, 3, seed=11)
    r.targets[1], r.targets[4] = 500, 65535
    got, ref = r.run(flint), r.reference()
    check(got, ref)
    assert float(got["logprob"][1]) == 0.0 and float(got["logprob"][4]) == 0.0


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [997, 50257])
def test_without_an_entropy_gradient_and_in_place(flint, cuda, vocab):
    r = Rows(cuda, 5, vocab, (vocab + 63) // 64 * 64, 0, seed=12)
    got = r.run(flint, entropy_gradient=False)
    check(got, r.reference(entropy_gradient=False))
    assert torch.equal(r.run(flint, entropy_gradient=False, in_place=True)["d"], got["d"])


@pytest.mark.gpu
def test_agrees_with_the_cross_entropy(flint, cuda):
    """row_loss is -logprob, and dlogits of sum(-logprob) the loss's gradient."""
    r = Rows(cuda, 40, 3000, 3008, 0, seed=13)
    r.dlp[:] = -1.0
    got, ref = r.run(flint, entropy_gradient=False), r.reference(entropy_gradient=False)
    d = torch.empty((40, 3008), dtype=torch.float16, device=cuda)
    loss = torch.empty(40, device=cuda)
    flint.softmax_cross_entropy(d, loss, r.logits.to(cuda),
                                r.targets.to(torch.int32).to(torch.int16).to(cuda), 1.0, 40, 3000,
                                3008)
    torch.cuda.synchronize()
    assert bool(((loss.cpu() + got["logprob"]).abs().double() <= 2 * ref["logprob_bound"]).all())
    assert bool(((d.cpu() - got["d"]).abs().double() <= 2 * ref["d_bound"]).all())


@pytest.mark.gpu
def test_gradient_against_differences(flint, cuda):
    r = Rows(cuda, 4, 60, 64, 0, seed=14, scale=0.7)
    got, ref = r.run(flint), r.reference()
    move = normal((4, 64), 15, 1.0, torch.float64)
    step = 1e-4

    def loss(sign):
        out = reference(r.logits.double() + sign * step * move, r.targets, 60, 0.7, 0)
        return float((r.dlp.double() * out["logprob"] + r.dh.double() * out["entropy"]).sum())

    slope = (loss(1) - loss(-1)) / (2 * step)
    along = float((got["d"].double() * move).sum())
    assert abs(slope - along) <= float((ref["d_bound"] * move.abs()).sum()) + 1e-6


@pytest.mark.gpu
def test_two_runs_are_bit_identical(flint, cuda):
    r = Rows(cuda, 20, 50257, 50304, 20, seed=16)
    one, two = r.run(flint), r.run(flint)
    for name in one:
        assert torch.equal(one[name], two[name]), name


@pytest.mark.gpu
def test_captured_and_replayed(flint, cuda):
    r = Rows(cuda, 12, 5000, 5000, 8, seed=17)
    want = r.run(flint)
    logits, t16 = r.logits.to(cuda), r.targets.to(torch.int32).to(torch.int16).to(cuda)
    dlp, dh = r.dlp.to(cuda), r.dh.to(cuda)
    d, out = torch.empty_like(logits), {n: torch.empty_like(t) for n, t in r.out.items()}
    stream = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        flint.logprobs_forward(out["logprob"], out["entropy"], out["stats"], out["ids"],
                               out["values"], logits, t16, 1.0, 12, 5000, 5000, 8)
        flint.logprobs_backward(d, dlp, dh, logits, t16, out["entropy"], out["stats"], 1.0, 12,
                                5000, 5000)
    for _ in range(3):
        d.fill_(SENTINEL)
        for t in out.values():
            t.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(d.cpu(), want["d"])
        for name in ("logprob", "entropy", "ids", "values"):
            assert torch.equal(out[name].cpu(), want[name]), name


# ------------------------------------------------------------------ refusals

A = 0x1000000   # a 16-byte-aligned fake device address: refusals never read it
ONE = ctypes.c_float(1.0)


def fails(flint, fn, *args, message):
    status = getattr(flint.lib, fn)(*args)
    assert status == flint_lib.ERROR_INVALID_ARGUMENT
    assert message in flint.last_error(), flint.last_error()


@pytest.mark.parametrize("scale,rows,vocab,cols,message", [
    (1.0, 4, 10, 12, "cols (12) must be a multiple of 8 from 8 to 65536"),
    (1.0, 4, 0, 16, "vocab (0) must be from 1 to cols (16)"),
    (1.0, 4, 17, 16, "vocab (17) must be from 1 to cols (16)"),
    (0.0, 4, 16, 16, "scale (0) must be positive and finite"),
    (-1.0, 4, 16, 16, "scale (-1) must be positive and finite"),
    (math.nan, 4, 16, 16, "scale (nan) must be positive and finite"),
    (math.inf, 4, 16, 16, "scale (inf) must be positive and finite"),
    (1.0, 1 << 40, 16, 16, "rows (1099511627776) can be up to"),
])
def test_sizes_refused(flint, scale, rows, vocab, cols, message):
    args = [(i + 1) * A for i in range(7)]
    fails(flint, "flint_logprobs_forward", *args, ctypes.c_float(scale), rows, vocab, cols, 2, None,
          message=message)
    fails(flint, "flint_logprobs_backward", *args, ctypes.c_float(scale), rows, vocab, cols, None,
          message=message)


def test_buffers_refused(flint):
    good = [(i + 1) * A for i in range(7)]
    fn = "flint_logprobs_forward"
    fails(flint, fn, *good, ONE, 4, 16, 16, 17, None, message="top (17) can be up to 64 and up to vocab (16)")
    fails(flint, fn, *good, ONE, 4, 100, 104, 65, None, message="top (65) can be up to 64")
    for i, name in enumerate(("logprob", "entropy", "stats", "top_ids", "top_logprobs", "logits",
                              "targets")):
        bad = list(good)
        bad[i] = None
        fails(flint, fn, *bad, ONE, 4, 16, 16, 2, None, message=f"{fn}: {name} is null")
        bad[i] = good[i] + 2
        fails(flint, fn, *bad, ONE, 4, 16, 16, 2, None, message=f"{name} is not 16-byte aligned")
    bad = list(good)
    bad[2] = good[5] + 16
    fails(flint, fn, *bad, ONE, 4, 16, 16, 2, None, message="stats and logits overlap")
    fn = "flint_logprobs_backward"
    for i, name in ((0, "dlogits"), (1, "dlogprob"), (3, "logits"), (4, "targets"), (5, "entropy"),
                    (6, "stats")):
        bad = list(good)
        bad[i] = None
        fails(flint, fn, *bad, ONE, 4, 16, 16, None, message=f"{fn}: {name} is null")
    bad = list(good)
    bad[3] = bad[0] + 16
    fails(flint, fn, *bad, ONE, 4, 16, 16, None, message="dlogits and logits overlap")
    bad = list(good)
    bad[6] = bad[0]
    fails(flint, fn, *bad, ONE, 4, 16, 16, None, message="dlogits and stats overlap")


def test_no_rows(flint):
    assert flint.lib.flint_logprobs_forward(*[None] * 7, ONE, 0, 16, 16, 2, None) == 0
    assert flint.lib.flint_logprobs_backward(*[None] * 7, ONE, 0, 16, 16, None) == 0
