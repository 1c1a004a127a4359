"""Causal attention over packed sequences (include/flint/flint_packed.h) against
float64, within bounds counted in rounding steps (attention_bounds.py); its
refusals; and what it leaves alone."""

import ctypes
import math

import pytest
import torch

from attention_bounds import Z, attend, causal, worst
from flint_amd import flint_lib
from inputs import normal

SENTINEL = 7.25


class Batch:
    """A batch on the CPU: q, k, v and dout as column slices or tensors of their
    own, and the offsets."""

    def __init__(self, lengths, heads, kv_heads, width, seed=1, sliced=True, before=0, after=0,
                 scale=None):
        self.lengths, self.heads, self.kv_heads, self.width = lengths, heads, kv_heads, width
        self.scale = 1.0 / math.sqrt(width) if scale is None else scale
        self.offsets = [before]
        for n in lengths:
            self.offsets.append(self.offsets[-1] + n)
        self.tokens = self.offsets[-1] + after
        rows, hw, kw = self.tokens, heads * width, kv_heads * width
        self.sliced = sliced
        self.qkv = normal((rows, hw + 2 * kw), seed, 1.0, torch.float16)
        self.dout = normal((rows, hw), seed + 1, 0.5, torch.float16)

    def parts(self, qkv):
        hw, kw = self.heads * self.width, self.kv_heads * self.width
        parts = qkv[:, :hw], qkv[:, hw:hw + kw], qkv[:, hw + kw:]
        return parts if self.sliced else tuple(p.contiguous() for p in parts)

    def shape(self, flint):
        if not self.sliced:
            return flint.packed_shape(self.tokens, len(self.lengths), self.heads, self.kv_heads,
                                      self.width)
        wide = self.qkv.shape[1]
        return flint.packed_shape(self.tokens, len(self.lengths), self.heads, self.kv_heads,
                                  self.width, wide, wide, self.heads * self.width)

    def reference(self, backward=True):
        """name -> (value, bound), laid out as the kernels' outputs."""
        H, Hk, w, n = self.heads, self.kv_heads, self.width, self.tokens
        q, k, v = self.parts(self.qkv)
        sizes = dict(o=(n, H, w), lse=(n, H), dq=(n, H, w), dk=(n, Hk, w), dv=(n, Hk, w))
        out = {name: (torch.zeros(size, dtype=torch.float64), torch.zeros(size, dtype=torch.float64))
               for name, size in sizes.items()}
        for a, b in zip(self.offsets, self.offsets[1:]):
            for h in range(H if b > a else 0):
                j = h // (H // Hk)
                got = attend(q[a:b, h * w:h * w + w], k[a:b, j * w:j * w + w],
                             v[a:b, j * w:j * w + w], self.scale, causal(b - a),
                             self.dout[a:b, h * w:h * w + w] if backward else None)
                for name, pair in got.items():
                    at = j if name in ("dk", "dv") else h
                    for total, part in zip(out[name], pair):
                        total[a:b, at] += part
        return {name: (v.flatten(1), b.flatten(1)) for name, (v, b) in out.items()}


class Run:
    """A batch on the GPU and its outputs, filled with a sentinel."""

    def __init__(self, flint, cuda, batch):
        self.flint, self.b = flint, batch
        self.shape = batch.shape(flint)
        self.qkv = batch.qkv.to(cuda)
        self.q, self.k, self.v = batch.parts(self.qkv)
        self.dout = batch.dout.to(cuda)
        self.offsets = torch.tensor(batch.offsets, dtype=torch.int32, device=cuda)
        self.o = torch.full_like(self.dout, SENTINEL)
        self.lse = torch.full((batch.heads, batch.tokens), SENTINEL, device=cuda)
        self.dqkv = torch.full_like(self.qkv, SENTINEL)
        self.dq, self.dk, self.dv = batch.parts(self.dqkv)
        self.plan = torch.empty(flint.attention_packed_plan_bytes(self.shape), dtype=torch.uint8,
                                device=cuda)
        self.ws = torch.empty(max(16, flint.attention_packed_backward_workspace(self.shape)),
                              dtype=torch.uint8, device=cuda)

    def run(self, backward=True, stream=None):
        f = self.flint
        f.attention_packed_plan(self.plan, self.offsets, self.shape, stream=stream)
        f.attention_packed_forward(self.o, self.lse, self.q, self.k, self.v, self.plan, self.shape,
                                   self.b.scale, stream=stream)
        if backward:
            f.attention_packed_backward(self.dq, self.dk, self.dv, self.dout, self.q, self.k,
                                        self.v, self.o, self.lse, self.plan, self.shape,
                                        self.b.scale, self.ws, stream=stream)
        return self

    def outputs(self):
        torch.cuda.synchronize()
        return dict(o=self.o.cpu(), lse=self.lse.T.cpu(), dq=self.dq.cpu(), dk=self.dk.cpu(),
                    dv=self.dv.cpu())


def check(run, names=("o", "lse", "dq", "dk", "dv"), reference=None):
    b = run.b
    got = run.outputs()
    ref = b.reference("dq" in names) if reference is None else reference
    inside = torch.zeros(b.tokens, dtype=torch.bool)
    inside[b.offsets[0]:b.offsets[-1]] = True
    for name in names:
        off = worst(got[name][inside], *(t[inside] for t in ref[name]))
        print(f"{name}: {off:.2f} of the bound")
        assert off <= 1.0, (name, off)
        assert bool((got[name][~inside] == SENTINEL).all()), name


@pytest.mark.gpu
@pytest.mark.parametrize("width", [64, 128])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (3, 3), (4, 2), (6, 1)])
@pytest.mark.parametrize("lengths", [[1], [2, 1, 3], [64], [31, 65, 0, 127], [128, 129], [200, 300]])
def test_matches_float64(flint, cuda, lengths, heads, kv_heads, width):
    check(Run(flint, cuda, Batch(lengths, heads, kv_heads, width, seed=sum(lengths))).run())


@pytest.mark.gpu
@pytest.mark.parametrize("width", [64, 128])
def test_long_and_short_together(flint, cuda, width):
    check(Run(flint, cuda, Batch([1500, 1, 0, 77, 640], 2, 1, width, seed=5)).run())


@pytest.mark.gpu
def test_tensors_of_their_own_and_rows_of_no_sequence(flint, cuda):
    """Contiguous q, k, v; rows before, and after the last sequence, hold NaN:
    read into nothing, and their outputs stay."""
    b = Batch([70, 0, 133], 4, 2, 64, sliced=False, before=5, after=200)
    for t in (b.qkv, b.dout):
        t[:5] = float("nan")
        t[b.offsets[-1]:] = float("nan")
    check(Run(flint, cuda, b).run())


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [-0.125, 0.0, 2.0])
def test_any_finite_scale(flint, cuda, scale):
    check(Run(flint, cuda, Batch([150, 90], 2, 2, 64, scale=scale, seed=9)).run())


@pytest.mark.gpu
def test_many_short_sequences(flint, cuda):
    lengths = [(i * 7) % 5 for i in range(2500)]
    check(Run(flint, cuda, Batch(lengths, 2, 1, 64, seed=3)).run())


@pytest.mark.gpu
@pytest.mark.parametrize("lengths", [[1] * 200, [3, 1] * 60 + [65], [900, 1, 2, 30]])
def test_large_groups_of_heads(flint, cuda, lengths):
    """The heads of a group go into parts for dK and dV, and join."""
    check(Run(flint, cuda, Batch(lengths, 32, 1, 64, seed=28)).run())


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv_heads,width", [(1, 1, 64), (2, 1, 128), (3, 3, 64)])
def test_one_sequence_much_longer(flint, cuda, heads, kv_heads, width):
    check(Run(flint, cuda, Batch([5, 2300, 64, 130], heads, kv_heads, width, seed=29)).run())


@pytest.mark.gpu
def test_more_blocks_than_the_plan_has_buckets(flint, cuda):
    """Places go two to a bucket from 1,024 blocks on: every block is listed
    once, the longest bucket first, and rows along the long sequence are right."""
    lengths = [700, 140000, 0, 260, 5000]
    b = Batch(lengths, 1, 1, 64, seed=38, scale=0.125)
    r = Run(flint, cuda, b).run(backward=False)
    got = r.outputs()
    plan = r.plan.view(torch.int32).view(-1, 4).cpu()
    listed = plan[plan[:, 1] > plan[:, 0], :3].tolist()
    blocks = [[a, e, i] for a, e in zip(b.offsets, b.offsets[1:]) for i in range(-(-(e - a) // 128))]
    assert sorted(listed) == sorted(blocks)
    places = [i // 2 for _, _, i in listed]
    assert places == sorted(places, reverse=True)
    q, k, v = b.parts(b.qkv)
    first, end = b.offsets[1], b.offsets[2]
    for row in (first, first + 131071, first + 70001, end - 1):
        seen = torch.ones(1, row + 1 - first, dtype=torch.bool)
        ref = attend(q[row:row + 1], k[first:row + 1], v[first:row + 1], b.scale, seen)
        assert worst(got["o"][row:row + 1], *ref["o"]) <= 1.0
        assert worst(got["lse"][row], *ref["lse"]) <= 1.0


@pytest.mark.gpu
def test_a_sequence_keeps_its_non_finite_values(flint, cuda):
    b = Batch([100, 90, 130], 2, 2, 64, seed=12)
    clean = Run(flint, cuda, b).run().outputs()
    b.qkv[100:190] = float("nan")
    b.dout[100:190] = float("inf")
    got = Run(flint, cuda, b).run().outputs()
    for name, value in clean.items():
        for rows in (slice(0, 100), slice(190, 320)):
            assert torch.equal(got[name][rows], value[rows]), name


@pytest.mark.gpu
def test_large_scores(flint, cuda):
    """Scores of some hundred: one key takes a row, in whatever tile it lies."""
    b = Batch([300], 1, 1, 64, seed=14, scale=1.0)
    b.qkv[:, :128] *= 4.0
    check(Run(flint, cuda, b).run(backward=False), names=("o", "lse"))


@pytest.mark.gpu
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("width", [64, 128])
def test_scores_of_millions_stay_finite(flint, cuda, width, sign):
    """Scores around 2^24.9, where FP32 is 2 apart: what weights they give is
    rounding, but o lies among the values and lse beside the scores."""
    b = Batch([300, 70], 2, 1, width, seed=37, scale=sign * 1.0)
    q, k, v = b.parts(b.qkv)
    q[:], k[:] = 700.0, (2.0 ** 24.9 / (700.0 * width)) * (1 + 1e-3 * k.float()).half()
    got = Run(flint, cuda, b).run(backward=False).outputs()
    most = v.float().abs().amax(0).repeat(2) * (1 + 2.0 ** -10)   # P's rounding and o's
    assert bool((got["o"].float().abs() <= most).all())
    assert bool((got["lse"] * sign > 2.0 ** 24.8).all() and (got["lse"] * sign < 2.0 ** 25).all())


@pytest.mark.gpu
@pytest.mark.parametrize("width", [64, 128])
def test_a_key_that_outweighs_the_others_by_far(flint, cuda, width):
    """The first key is 2^25 to 2^27 times as likely as each other one and its
    value is 0: o is what the others add up to. Probabilities are rounded at 2^5
    times their size, so half a step among FP16's subnormals is 2^-30."""
    b = Batch([600, 90], 2, 1, width, seed=35, scale=8.0 / width)   # scores: 8 k
    q, k, v = b.parts(b.qkv)
    q[:] = 1.0
    k[:] = -0.09 * torch.rand(k.shape[0], 1, generator=torch.Generator().manual_seed(36))
    v[:] = 64.0
    for first in b.offsets[:-1]:
        k[first], v[first] = 2.21, 0.0
    ref = b.reference(backward=False)
    for first, end in zip(b.offsets, b.offsets[1:]):
        reach = v[first:end].double().cumsum(0).repeat(1, 2)
        ref["o"][1][first:end] -= 1.05 * (Z - 2.0 ** -30) * reach
    check(Run(flint, cuda, b).run(backward=False), names=("o", "lse"), reference=ref)


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv_heads,width,size", [(2, 2, 64, 400.0), (4, 1, 128, 400.0),
                                                       (4, 2, 64, 2e-4)])
def test_large_and_small_gradients(flint, cuda, heads, kv_heads, width, size):
    """dS past what FP16 holds at 2^8 times its size, and far below its normal
    values."""
    b = Batch([300, 65, 700], heads, kv_heads, width, seed=20)
    b.dout = (b.dout.float() * (2 * size)).half()
    check(Run(flint, cuda, b).run())


@pytest.mark.gpu
def test_offsets_outside_the_tokens_are_taken_inside(flint, cuda):
    b = Batch([40, 60], 2, 2, 64, seed=15)
    r = Run(flint, cuda, b)
    r.offsets = torch.tensor([-7, 40, 1 << 30], dtype=torch.int32, device=cuda)
    check(r.run())


@pytest.mark.gpu
def test_offsets_that_decrease_make_no_more_blocks_than_the_plan_holds(flint, cuda):
    """20 sequences of the same 512 tokens: 80 blocks, where 44 is the most."""
    b = Batch([512] + [0] * 39, 2, 2, 64, seed=19)
    r = Run(flint, cuda, b)
    r.offsets = torch.tensor([0, 512] * 20 + [0], dtype=torch.int32, device=cuda)
    for name, got in r.run().outputs().items():
        assert torch.all(got == SENTINEL), name


@pytest.mark.gpu
def test_two_runs_are_bit_identical(flint, cuda):
    b = Batch([500, 33, 700], 4, 2, 128, seed=16)
    one, two = Run(flint, cuda, b).run().outputs(), Run(flint, cuda, b).run().outputs()
    for name in one:
        assert torch.equal(one[name], two[name]), name


@pytest.mark.gpu
@pytest.mark.parametrize("width", [64, 128])
def test_outputs_do_not_depend_on_what_ran_before(flint, cuda, width):
    """Workgroups find in LDS what others left there: zeros, or NaN. Sequences of
    up to 64 tokens have a tile for the first of two groups of waves only; their
    dS is below FP16's normal values, so a second walk without the factor 2^8
    shows."""
    b = Batch([40, 64, 1, 17, 50], 2, 2, width, seed=33)
    b.dout = (b.dout.float() * 1e-4).half()
    r = Run(flint, cuda, b)
    before = Run(flint, cuda, Batch([512] * 64, 8, 8, width, seed=34))
    got = []
    for fill in (0.0, float("nan")):
        before.qkv.fill_(fill)
        before.dout.fill_(fill)
        before.run(backward=False)
        r.run(backward=False)
        before.run()
        flint.attention_packed_backward(r.dq, r.dk, r.dv, r.dout, r.q, r.k, r.v, r.o, r.lse, r.plan,
                                        r.shape, b.scale, r.ws)
        got.append(r.outputs())
    for name, value in got[0].items():
        assert torch.equal(got[1][name], value), name
    check(r)


@pytest.mark.gpu
def test_captured_and_replayed_on_a_stream_of_its_own(flint, cuda):
    """Two graphs share the plan and the workspace; each replay reads the inputs
    and offsets that the tensors hold then."""
    first, second = Batch([90, 200], 2, 1, 64, seed=20), Batch([200, 90], 2, 1, 64, seed=22)
    runs = [Run(flint, cuda, b) for b in (first, second)]
    runs[1].plan, runs[1].ws = runs[0].plan, runs[0].ws
    want = [Run(flint, cuda, b).run().outputs() for b in (first, second)]
    stream = torch.cuda.Stream()
    graphs = []
    for r in runs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            r.run()
        graphs.append(graph)
    for _ in range(3):
        for r in runs:
            for t in (r.o, r.lse, r.dqkv):
                t.fill_(SENTINEL)
        for g in graphs:
            g.replay()
        for r, w in zip(runs, want):
            for name, value in r.outputs().items():
                assert torch.equal(value, w[name]), name
    runs[0].qkv.copy_(runs[1].qkv)
    runs[0].dout.copy_(runs[1].dout)
    runs[0].offsets.copy_(runs[1].offsets)
    graphs[0].replay()
    for name, value in runs[0].outputs().items():
        assert torch.equal(value, want[1][name]), name


@pytest.mark.gpu
def test_equal_lengths_agree_with_the_batched_attention(flint, cuda):
    """Sequences of one length and a head each: flint_attention_forward and
    _backward's case, within both kernels' distance from float64."""
    batches, length = 3, 200
    b = Batch([length] * batches, 1, 1, 64, seed=24, sliced=False)
    r = Run(flint, cuda, b).run()
    ref = b.reference()
    o, lse = torch.empty_like(r.o), torch.empty_like(r.lse)
    grads = [torch.empty_like(r.q) for _ in range(3)]
    flint.attention_forward(o, lse, r.q, r.k, r.v, batches, length, 64, b.scale)
    flint.attention_backward(*grads, r.dout, r.q, r.k, r.v, o, lse, batches, length, 64, b.scale)
    got = r.outputs()
    for name, other in zip(("o", "dq", "dk", "dv"), [o] + grads):
        assert worst(got[name], other.cpu().double(), 2 * ref[name][1]) <= 1.0, name


@pytest.mark.gpu
def test_gradients_against_differences(flint, cuda):
    """The change of sum(dout * o) along a direction, from float64 attention of
    moved inputs, against the gradients' product with it."""
    b = Batch([37, 90], 4, 2, 64, seed=26)
    got = Run(flint, cuda, b).run().outputs()
    ref = b.reference()
    d = normal(b.qkv.shape, 27, 1.0, torch.float64)
    base = b.qkv
    step = 1e-4

    def loss(sign):
        b.qkv = base.double() + sign * step * d
        o = b.reference(backward=False)["o"][0]
        b.qkv = base
        return float((o * b.dout.double()).sum())

    slope = (loss(1) - loss(-1)) / (2 * step)
    dq, dk, dv = b.parts(d)
    along = sum(float((got[n].double() * t).sum()) for n, t in (("dq", dq), ("dk", dk), ("dv", dv)))
    slack = sum(float((ref[n][1] * t.abs()).sum()) for n, t in (("dq", dq), ("dk", dk), ("dv", dv)))
    # Central differences: step^2 / 6 of the third derivative, below 1e-6 of
    # the slope's scale here; the gradients' own bounds cover the rest.
    assert abs(slope - along) <= slack + 1e-5 * abs(slope)


# ------------------------------------------------------------------ refusals

A = 0x100000   # a 16-byte-aligned fake device address: refusals never read it


def fails(flint, fn, *args, message):
    status = getattr(flint.lib, fn)(*args)
    assert status == flint_lib.ERROR_INVALID_ARGUMENT
    assert message in flint.last_error(), flint.last_error()


def shape_of(flint, **changes):
    s = flint.packed_shape(64, 2, 4, 2, 64)
    for name, value in changes.items():
        setattr(s, name, value)
    return s


@pytest.mark.parametrize("changes,message", [
    (dict(head_width=96), "head_width (96) must be 64 or 128"),
    (dict(heads=0), "heads (0) must be from 1 to 1024"),
    (dict(kv_heads=3), "kv_heads (3) must divide heads (4)"),
    (dict(kv_heads=0), "kv_heads (0) must divide heads (4)"),
    (dict(tokens=(1 << 26) + 1), "tokens (67108865) can be up to 67108864"),
    (dict(sequences=(1 << 20) + 1), "sequences (1048577) can be up to 1048576"),
    (dict(tokens=1 << 26, sequences=1 << 20, heads=1024, q_stride=65536, o_stride=65536),
     "(tokens / 128 + sequences) x heads"),
    (dict(q_stride=260), "q_stride (260) must be a multiple of 8 from 256"),
    (dict(kv_stride=120), "kv_stride (120) must be a multiple of 8 from 128"),
    (dict(o_stride=1 << 24), "o_stride (16777216) must be a multiple of 8 from 256 to 8388608"),
])
def test_shapes_refused(flint, changes, message):
    s = shape_of(flint, **changes)
    out = ctypes.c_size_t(0)
    f = ctypes.c_float(0.125)
    fails(flint, "flint_attention_packed_plan_bytes", s, out, message=message)
    fails(flint, "flint_attention_packed_backward_workspace", s, out, message=message)
    fails(flint, "flint_attention_packed_plan", A, 2 * A, s, None, message=message)
    fails(flint, "flint_attention_packed_forward", *[(i + 1) * A for i in range(6)], s, f, None,
          message=message)
    fails(flint, "flint_attention_packed_backward", *[(i + 1) * A for i in range(10)], s, f, 11 * A,
          1 << 20, None, message=message)


def test_buffers_refused(flint):
    s = shape_of(flint)
    f = ctypes.c_float(0.125)
    fn = "flint_attention_packed_forward"
    good = [(i + 1) * A for i in range(6)]
    for i, name in enumerate(("o", "lse", "q", "k", "v", "plan")):
        bad = list(good)
        bad[i] = None
        fails(flint, fn, *bad, s, f, None, message=f"{fn}: {name} is null")
        bad[i] = good[i] + 8
        fails(flint, fn, *bad, s, f, None, message=f"{name} is not 16-byte aligned")
    fails(flint, fn, A, 2 * A, A + 1024, 4 * A, 5 * A, 6 * A, s, f, None, message="o and q overlap")
    fails(flint, fn, *good, s, ctypes.c_float(float("nan")), None, message="must be finite")
    fails(flint, fn, *good, None, f, None, message="shape is null")
    fails(flint, "flint_attention_packed_plan", A, A, s, None, message="plan and offsets overlap")
    fn = "flint_attention_packed_backward"
    good = [(i + 1) * A for i in range(10)]
    need = ctypes.c_size_t(0)
    assert flint.lib.flint_attention_packed_backward_workspace(s, need) == 0 and need.value >= 1024
    fails(flint, fn, *good, s, f, 11 * A, 100, None,
          message=f"needs {need.value} bytes of workspace, given 100")
    fails(flint, fn, A, A + 64, *good[2:], s, f, 11 * A, 1 << 20, None, message="dq and dk overlap")


@pytest.mark.parametrize("scale", [1e30, -3.4e38, 2.0 ** 64 * 1.001])
def test_scales_whose_scores_pass_fp32_are_refused(flint, scale):
    s, f = shape_of(flint), ctypes.c_float(scale)
    message = f"scale ({f.value:g}) can be up to 1.84467e+19 in size"
    fails(flint, "flint_attention_packed_forward", *[(i + 1) * A for i in range(6)], s, f, None,
          message=message)
    fails(flint, "flint_attention_packed_backward", *[(i + 1) * A for i in range(10)], s, f, 11 * A,
          1 << 20, None, message=message)


def test_column_slices_of_one_tensor_do_not_overlap(flint):
    """dq, dk and dv beside each other in rows of 512 values pass that check (the
    next one fails: a null plan); one column more of overlap does not."""
    s = shape_of(flint, q_stride=512, kv_stride=512)
    f = ctypes.c_float(0.125)
    rest = [(i + 4) * A for i in range(6)]
    fn = "flint_attention_packed_backward"
    fails(flint, fn, A, A + 512, A + 768, *rest, None, s, f, 11 * A, 1 << 20, None,
          message="plan is null")
    fails(flint, fn, A, A + 512, A + 768, *rest, A + 768, s, f, 11 * A, 1 << 20, None,
          message="dq and plan overlap")
    fails(flint, fn, A, A + 496, A + 768, *rest, 12 * A, s, f, 11 * A, 1 << 20, None,
          message="dq and dk overlap")
    fails(flint, fn, A, A + 512, A + 752, *rest, 12 * A, s, f, 11 * A, 1 << 20, None,
          message="dk and dv overlap")
    # dv running past the row's end meets the next row's dq.
    fails(flint, fn, A, A + 512, A + 784, *rest, 12 * A, s, f, 11 * A, 1 << 20, None,
          message="dq and dv overlap")


def test_nothing_to_do(flint):
    s = shape_of(flint, tokens=0)
    f = ctypes.c_float(0.125)
    assert flint.lib.flint_attention_packed_plan(None, None, s, None) == 0
    assert flint.lib.flint_attention_packed_forward(*[None] * 6, s, f, None) == 0
    assert flint.lib.flint_attention_packed_backward(*[None] * 10, s, f, None, 0, None) == 0
