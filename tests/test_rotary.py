"""Rotary positions (include/flint/flint_rotary.h) against float64, what is
copied and what is left alone, the gradient against differences, captured and
replayed; its refusals.

How far a correct kernel may be: the angle in turns, below 1/2, is rounded to FP32
(2^-26 turns, 2^-23.3 radians), sine and cosine are off by at most 4 steps of FP32
(2^-22 each, relative to 1) with the magnitude, the two products and their sum by
3 x 2^-24: together under 2^-20 m (|a| + |b|). Then RN16: 2^-11 of the value, 2^-25
among the subnormals."""

import ctypes
import math

import pytest
import torch

from flint_amd import flint_lib
from inputs import normal

SENTINEL = 7.25
LOW, HIGH = 1.0, 32.0


def frequencies(width, base, factor=1.0, original=0.0, low=LOW, high=HIGH):
    out = []
    for i in range(width // 2):
        f = base ** (-2.0 * i / width)
        keep = 0.0
        if original:
            keep = min(max((original * f / (2 * math.pi) - low) / (high - low), 0.0), 1.0)
        out.append(f * (keep + (1.0 - keep) / factor))
    return torch.tensor(out, dtype=torch.float64)


def reference(x, positions, f, heads, head_width, width, pairs, magnitude=1.0, backward=False):
    """x: tokens x (heads x head_width) -> (value, bound), float64."""
    x = x.double().reshape(x.shape[0], heads, head_width)
    value, bound = x.clone(), torch.zeros_like(x)
    angle = positions.double()[:, None] * f
    c = (magnitude * torch.cos(angle))[:, None]
    s = (magnitude * torch.sin(angle) * (-1.0 if backward else 1.0))[:, None]
    first = torch.arange(0, width, 2) if pairs else torch.arange(width // 2)
    second = first + (1 if pairs else width // 2)
    a, b = x[:, :, first], x[:, :, second]
    for at, v in ((first, a * c - b * s), (second, a * s + b * c)):
        value[:, :, at] = v
        bound[:, :, at] = (2.0 ** -11 * v.abs() + 2.0 ** -25
                           + 2.0 ** -20 * abs(magnitude) * (a.abs() + b.abs()))
    return value.reshape(len(x), -1), bound.reshape(len(x), -1)


def make_plan(flint, cuda, width, base=10000.0, factor=1.0, original=0.0, magnitude=1.0):
    plan = torch.full((1 + width // 2 + 2,), SENTINEL, dtype=torch.float64, device=cuda)
    assert flint.rotary_plan_bytes(width) == 8 * (1 + width // 2)
    flint.rotary_plan(plan, flint.rotary_angles(width, base, factor, original, LOW, HIGH,
                                                magnitude))
    return plan


def close(got, ref):
    value, bound = ref
    diff = (got.cpu().double() - value).abs()
    assert torch.all(diff <= bound), float((diff - bound).max())


@pytest.mark.gpu
@pytest.mark.parametrize("width,base,factor,original,magnitude", [
    (64, 10000.0, 1.0, 0.0, 1.0), (128, 500000.0, 8.0, 8192.0, 1.2), (2, 2.0, 4.0, 0.0, 1.0),
    (1024, 10000.0, 0.5, 100.0, 0.0)])
def test_plan(flint, cuda, width, base, factor, original, magnitude):
    plan = make_plan(flint, cuda, width, base, factor, original, magnitude).cpu()
    want = frequencies(width, base, factor, original) / (2 * math.pi)
    n = width // 2
    assert float(plan[0]) == magnitude
    assert torch.allclose(plan[1:1 + n], want, rtol=1e-13, atol=0.0)
    assert torch.all(plan[1 + n:] == SENTINEL)


SHAPES = [
    # tokens, heads, kv_heads, head_width, width, pairs
    (1, 1, 1, 64, 64, False), (1, 32, 8, 128, 128, True), (17, 12, 12, 64, 64, False),
    (5, 4, 2, 128, 64, True), (130, 4, 1, 80, 20, False), (33, 3, 3, 80, 40, False),
    (9, 2, 2, 96, 24, False), (7, 3, 1, 64, 6, True), (7, 3, 1, 64, 2, False), (3, 1, 1, 8, 8, True),
    (3, 2, 1, 1024, 1024, False), (2, 2, 1, 1024, 510, True), (2100, 4, 2, 64, 32, False),
    (1025, 3, 1, 128, 128, False), (40, 3, 0, 64, 64, True), (40, 0, 3, 64, 48, False),
]


@pytest.mark.gpu
@pytest.mark.parametrize("backward", [False, True])
@pytest.mark.parametrize("tokens,heads,kv_heads,head_width,width,pairs", SHAPES)
def test_against_float64(flint, cuda, tokens, heads, kv_heads, head_width, width, pairs, backward):
    """q and k column slices of one projection; rows and columns beside them stay."""
    qw, kw = heads * head_width, kv_heads * head_width
    wide, wide_out = qw + kw + 8, qw + kw + 24
    x = normal((tokens, wide), 1, 1.0, torch.float16)
    positions = torch.randint(0, 1 << 20, (tokens,), generator=torch.Generator().manual_seed(2),
                              dtype=torch.int32)
    positions[0] = 0
    plan = make_plan(flint, cuda, width, 10000.0, 4.0, 2048.0, 1.1)
    f = frequencies(width, 10000.0, 4.0, 2048.0)
    shape = flint.rotary_shape(tokens, heads, kv_heads, head_width, width, pairs, wide, wide,
                               wide_out, wide_out)
    out = torch.full((tokens + 2, wide_out), SENTINEL, dtype=torch.float16, device=cuda)
    d = x.to(cuda)
    flint.rotary(out[:, :qw], out[:, qw + 8:], d[:, :qw], d[:, qw:], positions.to(cuda), plan,
                 shape, backward)
    if qw:
        close(out[:tokens, :qw], reference(x[:, :qw], positions, f, heads, head_width, width,
                                           pairs, 1.1, backward))
    if kw:
        close(out[:tokens, qw + 8:qw + 8 + kw],
              reference(x[:, qw:qw + kw], positions, f, kv_heads, head_width, width, pairs, 1.1,
                        backward))
    assert torch.all(out[tokens:] == SENTINEL)
    assert torch.all(out[:, qw:qw + 8] == SENTINEL)
    assert torch.all(out[:, qw + 8 + kw:] == SENTINEL)
    assert torch.equal(d.cpu(), x)
    # In place: the same bits, and nothing else touched.
    shape = flint.rotary_shape(tokens, heads, kv_heads, head_width, width, pairs, wide, wide)
    flint.rotary(d[:, :qw], d[:, qw:], d[:, :qw], d[:, qw:], positions.to(cuda), plan, shape,
                 backward)
    assert torch.equal(d[:, :qw], out[:tokens, :qw])
    assert torch.equal(d[:, qw:qw + kw], out[:tokens, qw + 8:qw + 8 + kw])
    assert torch.equal(d[:, qw + kw:].cpu(), x[:, qw + kw:])


@pytest.mark.gpu
@pytest.mark.parametrize("position", [0, 1, -1, 131071, -131071, 2 ** 31 - 1, -2 ** 31])
def test_far_and_negative_positions(flint, cuda, position):
    x = normal((3, 128), 3, 1.0, torch.float16)
    positions = torch.tensor([position] * 3, dtype=torch.int32)
    plan = make_plan(flint, cuda, 128)
    out = torch.empty((3, 128), dtype=torch.float16, device=cuda)
    shape = flint.rotary_shape(3, 1, 0, 128, 128, False, 128, 0)
    flint.rotary(out, None, x.to(cuda), None, positions.to(cuda), plan, shape)
    # p f to 2^-53 of itself, in FP64 here and there: 2^31 2^-53 radians beside the
    # bound's 2^-20 are nothing.
    close(out, reference(x, positions, frequencies(128, 10000.0), 1, 128, 128, False))
    if position == 0:
        assert torch.equal(out.cpu(), x)


@pytest.mark.gpu
def test_rows_past_2_to_the_32_values(flint, cuda):
    """Rows as far apart as they may be, in place; the values beside them stay."""
    tokens, stride = 520, 1 << 23
    x = torch.empty((tokens, stride), dtype=torch.float16, device=cuda)
    x[:, :136] = SENTINEL
    rows = normal((tokens, 128), 5, 1.0, torch.float16)
    x[:, :128] = rows.to(cuda)
    positions = torch.arange(tokens, dtype=torch.int32) * 1000
    plan = make_plan(flint, cuda, 64)
    shape = flint.rotary_shape(tokens, 1, 1, 64, 64, False, stride, stride)
    flint.rotary(x, x[:, 64:], x, x[:, 64:], positions.to(cuda), plan, shape)
    close(x[:, :128], reference(rows, positions, frequencies(64, 10000.0), 2, 64, 64, False))
    assert torch.all(x[:, 128:136] == SENTINEL)


@pytest.mark.gpu
def test_non_finite_values_stay_in_their_pair(flint, cuda):
    x = normal((4, 2 * 64), 4, 1.0, torch.float16)
    clean = x.clone()
    x[1, 5], x[2, 64 + 40] = float("nan"), float("inf")
    positions = torch.arange(4, dtype=torch.int32, device=cuda) + 3
    plan = make_plan(flint, cuda, 64)
    shape = flint.rotary_shape(4, 2, 0, 64, 64, False, 128, 0)
    outs = []
    for v in (x, clean):
        out = torch.empty((4, 128), dtype=torch.float16, device=cuda)
        flint.rotary(out, None, v.to(cuda), None, positions, plan, shape)
        outs.append(out.cpu())
    touched = torch.zeros(4, 128, dtype=torch.bool)
    touched[1, [5, 37]] = True
    touched[2, [64 + 8, 64 + 40]] = True
    assert torch.equal(outs[0][~touched], outs[1][~touched])
    assert not torch.isfinite(outs[0][touched]).any()


@pytest.mark.gpu
def test_backward_is_the_gradient(flint, cuda):
    """<dy, f(x + h e) - f(x - h e)> / 2h is <dx, e>; f is linear, so h is 1 and only
    roundings differ: each value of both sides is off by at most 2^-11 of itself
    and the 2^-20 of the sums, on 2 x 256 values."""
    n, w = 6, 128
    x, e, dy = (normal((n, 2 * w), s, 1.0, torch.float16) for s in (5, 6, 7))
    positions = torch.tensor([0, 3, 777, 70000, 12, 5], dtype=torch.int32, device=cuda)
    plan = make_plan(flint, cuda, 64, magnitude=1.3)
    shape = flint.rotary_shape(n, 2, 0, w, 64, True, 2 * w, 0)

    def turned(v, backward=False):
        out = torch.empty((n, 2 * w), dtype=torch.float16, device=cuda)
        flint.rotary(out, None, v.to(cuda), None, positions, plan, shape, backward)
        return out.cpu().double()

    up, down = turned(x + e), turned(x - e)
    exact_up, exact_down = (x + e), (x - e)        # as FP16 holds them
    step = (exact_up.double() - exact_down.double()) / 2
    left = (dy.double() * (up - down) / 2)
    dx = turned(dy, True)
    right = dx * step
    tol = (2.0 ** -10 * (dy.double().abs() * (up.abs() + down.abs()) / 2 + right.abs())).sum()
    assert abs(float(left.sum() - right.sum())) <= float(tol)


@pytest.mark.gpu
def test_captured_and_on_another_stream(flint, cuda):
    """One plan for two graphs; positions change between replays."""
    T, H, w = 300, 4, 64
    x = normal((T, H * w), 8, 1.0, torch.float16).to(cuda)
    positions = torch.arange(T, dtype=torch.int32, device=cuda)
    plan = make_plan(flint, cuda, w)
    shape = flint.rotary_shape(T, H, 0, w, w, False, H * w, 0)
    outs = [torch.empty_like(x) for _ in range(2)]
    stream = torch.cuda.Stream()
    graphs = []
    for backward, out in enumerate(outs):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            flint.rotary(out, None, x, None, positions, plan, shape, bool(backward))
        graphs.append(graph)
    f = frequencies(w, 10000.0)
    for shift in (0, 1000, 5):
        positions.add_(shift)
        for g in graphs:
            g.replay()
        for backward, out in enumerate(outs):
            close(out, reference(x.cpu(), positions.cpu(), f, H, w, w, False, 1.0, bool(backward)))
            out.fill_(SENTINEL)


# ------------------------------------------------------------------ refusals

A = 0x1000000   # a 16-byte-aligned fake device address: refusals never read it


def fails(flint, fn, *args, message):
    status = getattr(flint.lib, fn)(*args)
    assert status == flint_lib.ERROR_INVALID_ARGUMENT
    assert message in flint.last_error(), flint.last_error()


def shape_of(flint, **changes):
    s = flint.rotary_shape(3, 4, 2, 64, 64, False, 384, 384, 256, 128)
    for name, value in changes.items():
        setattr(s, name, value)
    return s


@pytest.mark.parametrize("changes,message", [
    (dict(head_width=60), "head_width (60) must be a multiple of 8 from 8 to 1024"),
    (dict(head_width=1032), "head_width (1032) must be a multiple of 8 from 8 to 1024"),
    (dict(width=0), "width (0) must be even, from 2 to 1024"),
    (dict(width=33), "width (33) must be even"),
    (dict(width=66), "width (66) can be up to head_width (64)"),
    (dict(layout=2), "layout (2) must be 0 or 1"),
    (dict(tokens=(1 << 26) + 1), "tokens (67108865) can be up to 67108864"),
    (dict(heads=1025), "heads (1025) can be up to 1024"),
    (dict(kv_heads=1025), "kv_heads (1025) can be up to 1024"),
    (dict(q_stride=250), "q_stride (250) must be a multiple of 8 from 256"),
    (dict(k_stride=120), "k_stride (120) must be a multiple of 8 from 128"),
    (dict(q_out_stride=0), "q_out_stride (0) must be a multiple of 8 from 256"),
    (dict(k_out_stride=(1 << 23) + 8), "k_out_stride (8388616) must be a multiple of 8 from 128"),
])
def test_shapes_refused(flint, changes, message):
    fails(flint, "flint_rotary", *[(i + 1) * A for i in range(6)], shape_of(flint, **changes), 0,
          None, message=f"flint_rotary: {message}")


def test_buffers_refused(flint):
    s = shape_of(flint)
    fn = "flint_rotary"
    good = [(i + 1) * A for i in range(6)]
    for i, name in enumerate(("q_out", "k_out", "q", "k", "positions", "plan")):
        bad = list(good)
        bad[i] = None
        fails(flint, fn, *bad, s, 0, None, message=f"{fn}: {name} is null")
        bad[i] = good[i] + 4
        fails(flint, fn, *bad, s, 0, None, message=f"{name} is not 16-byte aligned")
    for i, j, message in ((0, 1, "q_out and k_out overlap"), (0, 2, "q_out and q overlap"),
                          (0, 3, "q_out and k overlap"), (1, 2, "k_out and q overlap"),
                          (1, 3, "k_out and k overlap"), (0, 4, "q_out and positions overlap"),
                          (1, 5, "k_out and plan overlap")):
        bad = list(good)
        bad[i] = bad[j] + (0 if j > 3 else 32)
        fails(flint, fn, *bad, s, 0, None, message=message)
    # The same start with another stride is not in place.
    bad = list(good)
    bad[0] = bad[2]
    fails(flint, fn, *bad, s, 0, None, message="q_out and q overlap")
    fails(flint, fn, *good, None, 0, None, message="shape is null")


@pytest.mark.parametrize("changes,message", [
    (dict(width=7), "width (7) must be even"), (dict(base=1.0), "base (1) must be finite and above 1"),
    (dict(base=float("nan")), "base (nan)"), (dict(factor=0.0), "factor (0) must be positive"),
    (dict(factor=float("inf")), "factor (inf)"), (dict(original=-1.0), "original (-1) must be 0 or"),
    (dict(original=10.0, low=2.0, high=2.0), "low (2) must be below high (2)"),
    (dict(magnitude=float("inf")), "magnitude (inf) must be finite")])
def test_angles_refused(flint, changes, message):
    a = flint.rotary_angles(64)
    for name, value in changes.items():
        setattr(a, name, value)
    fails(flint, "flint_rotary_plan", A, a, None, message=f"flint_rotary_plan: {message}")


def test_plans_refused(flint):
    a = flint.rotary_angles(64)
    fails(flint, "flint_rotary_plan", None, a, None, message="plan is null")
    fails(flint, "flint_rotary_plan", A + 8, a, None, message="plan is not 16-byte aligned")
    fails(flint, "flint_rotary_plan", A, None, None, message="angles is null")
    fails(flint, "flint_rotary_plan_bytes", 64, None, message="bytes is null")
    fails(flint, "flint_rotary_plan_bytes", 0, ctypes.c_size_t(0), message="width (0) must be even")


def test_nothing_to_do(flint):
    for none in (dict(tokens=0), dict(heads=0, kv_heads=0)):
        assert flint.lib.flint_rotary(*[None] * 6, shape_of(flint, **none), 0, None) == 0
