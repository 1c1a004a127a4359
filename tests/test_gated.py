"""The gated feed-forward product and its gradient (include/flint/flint_gated.h)
against float64, on every kernel and tile; refusals.

How far a correct kernel may be, with w = 2^-24 half a step of FP32, u = 2^-11 and z =
2^-25 of FP16:
  - a sum of k products: (k + 2) w of the terms' magnitudes |x| |w| (+ |bias|);
  - the activation s sigma(a), a the argument of the exponential: sigma moves by
    sigma (1 - sigma) times the error of a, at most |a| 2^-22 with the hardware's
    2^x, and by 2^-22 of itself for the quotient. x e^-x is at most 0.37, so sigma is
    off by less than 2^-22 and s sigma by 2^-21 max(1, |s|), 2^-20 counted. The slope
    sigma + s sigma (1 - sigma) z' adds |s z'| sigma (1 - sigma) (|a| 2^-22 + 2^-22),
    and |s z' a| e^-|a| is below 3: 2^-20, 2^-19 counted;
  - |act'| <= 1.13, so the activation passes an error of s on 1.13 times;
  - the product and the output: 2 w and u of the value, z."""

import ctypes
import math

import pytest
import torch

from flint_amd import flint_lib
from inputs import normal

SENTINEL = 7.25
W, U, Z16 = 2.0 ** -24, 2.0 ** -11, 2.0 ** -25


def slope_argument(g, act):
    """z'(g) / 1 and z(g): sigma's argument and its derivative."""
    if act == "silu":
        return torch.ones_like(g), g
    c = 2.0 * math.sqrt(2.0 / math.pi)
    return c * (1.0 + 3.0 * 0.044715 * g * g), c * (g + 0.044715 * g ** 3)


def activation(g, act):
    """(value, slope), float64."""
    dz, z = slope_argument(g, act)
    sigma = torch.sigmoid(z)
    return g * sigma, sigma + g * sigma * torch.sigmoid(-z) * dz


def forward_reference(x, w, bias, act):
    """(y, bound, pre, bound) in float64."""
    x, w = x.double(), w.double()
    n, k = w.shape[0] // 2, w.shape[1]
    pre, terms = x @ w.T, x.abs() @ w.abs().T
    if bias is not None:
        pre, terms = pre + bias.double(), terms + bias.double().abs()
    err = (k + 2) * W * terms
    g, u = pre[:, :n], pre[:, n:]
    a, _ = activation(g, act)
    a_err = 1.13 * err[:, :n] + 2.0 ** -20 * g.abs().clamp(min=1.0)
    y = a * u
    y_bound = (a_err * u.abs() + (a.abs() + a_err) * err[:, n:] + (U + 2 * W) * y.abs() + Z16)
    return y, 1.01 * y_bound, pre, 1.01 * (err + U * pre.abs() + Z16)


def backward_reference(dout, w, pre, act):
    """(dpre, bound) in float64."""
    dout, w, pre = dout.double(), w.double(), pre.double()
    k, n = w.shape
    s, err = dout @ w, (k + 2) * W * (dout.abs() @ w.abs())
    g, u = pre[:, :n], pre[:, n:]
    a, d = activation(g, act)
    a_err = 2.0 ** -20 * g.abs().clamp(min=1.0)
    dg, du = s * u * d, s * a
    dg_bound = err * (u * d).abs() + (s.abs() + err) * u.abs() * 2.0 ** -19
    du_bound = err * a.abs() + (s.abs() + err) * a_err
    bound = torch.cat([dg_bound + (U + 4 * W) * dg.abs(), du_bound + (U + 4 * W) * du.abs()], 1)
    return torch.cat([dg, du], 1), 1.01 * (bound + Z16)


def close(got, value, bound):
    diff = (got.double().cpu() - value.cpu()).abs()
    assert torch.isfinite(got).all()
    assert torch.all(diff <= bound.cpu()), float((diff - bound.cpu()).max())


def forward_inputs(m, n, k, bias, seed=1):
    return (normal((m, k), seed, 1.0, torch.float16),
            normal((2 * n, k), seed + 1, k ** -0.5, torch.float16),
            normal((2 * n,), seed + 2, 0.3) if bias else None)


def run_forward(flint, cuda, x, w, bias, act, keep, guard=3):
    """y and pre with `guard` rows of the sentinel behind them."""
    m, k = x.shape
    n = w.shape[0] // 2
    y = torch.full((m + guard, n), SENTINEL, dtype=torch.float16, device=cuda)
    pre = torch.full((m + guard, 2 * n), SENTINEL, dtype=torch.float16, device=cuda)
    flint.gemm_nt_gated(y, pre if keep else None, x.to(cuda), w.to(cuda),
                        None if bias is None else bias.to(cuda), m, n, k, act)
    assert torch.all(y[m:] == SENTINEL)
    assert torch.all(pre[m if keep else 0:] == SENTINEL)
    return y[:m], pre[:m] if keep else None


def run_backward(flint, cuda, dout, w, pre, act, guard=3):
    m, k = dout.shape
    n = w.shape[1]
    dpre = torch.full((m + guard, 2 * n), SENTINEL, dtype=torch.float16, device=cuda)
    flint.gemm_nn_dgated(dpre, dout.to(cuda), w.to(cuda), pre.to(cuda), m, n, k, act)
    assert torch.all(dpre[m:] == SENTINEL)
    return dpre[:m]


SIZES = [(1, 8, 8), (1, 16, 768), (3, 24, 40), (5, 2048, 64), (32, 72, 128), (64, 704, 256),
         (129, 200, 136), (300, 1000, 72), (257, 264, 1600), (1000, 136, 320), (2000, 512, 96),
         (2100, 2056, 128)]


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_forward(flint, cuda, m, n, k, act):
    for bias in (False, True):
        x, w, b = forward_inputs(m, n, k, bias)
        y_ref, y_bound, pre_ref, pre_bound = forward_reference(x, w, b, act)
        y, pre = run_forward(flint, cuda, x, w, b, act, True)
        close(y, y_ref, y_bound)
        close(pre, pre_ref, pre_bound)
        alone, _ = run_forward(flint, cuda, x, w, b, act, False)
        assert torch.equal(alone, y)


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_backward(flint, cuda, m, n, k, act):
    dout = normal((m, k), 4, 0.5, torch.float16)
    w = normal((k, n), 5, k ** -0.5, torch.float16)
    pre = normal((m, 2 * n), 6, 2.0, torch.float16)
    close(run_backward(flint, cuda, dout, w, pre, act),
          *backward_reference(dout, w, pre, act))


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_backward_is_the_gradient(flint, cuda, act):
    """Against differences of y(pre) = act(g) u in float64, of a step 2^-10: the third
    derivative of the activation is below 3, so they are off by 2^-20 u s."""
    m, n, k, h = 9, 40, 16, 2.0 ** -10
    dout = normal((m, k), 7, 0.5, torch.float16)
    w = normal((k, n), 8, 0.25, torch.float16)
    pre = normal((m, 2 * n), 9, 1.5, torch.float16)
    s = dout.double() @ w.double()
    g, u = pre[:, :n].double(), pre[:, n:].double()

    def y(g, u):
        return activation(g, act)[0] * u

    dg = s * (y(g + h, u) - y(g - h, u)) / (2 * h)
    du = s * (y(g, u + h) - y(g, u - h)) / (2 * h)
    _, bound = backward_reference(dout, w, pre, act)
    off = 2.0 ** -20 * (s * u).abs()
    close(run_backward(flint, cuda, dout, w, pre, act), torch.cat([dg, du], 1),
          bound + torch.cat([off, off], 1))


PIPE = ["256,192,4", "128,192,4", "128,192,3,64", "256,128,3,64", "256,192,2,64",
        "128,192,3,64,4,1", "256,128,3,64,4,1"]
SMALL = ["32,32,5,8,2", "32,64,4,6,2", "64,64,8,6,2", "64,64,4,4,1", "128,64,8,3,1"]


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(130, 72, 192), (300, 456, 64), (520, 1032, 128)])
def test_every_kernel_gives_the_same_bits(flint, cuda, tune, m, n, k):
    x, w, b = forward_inputs(m, n, k, True)
    dout = normal((m, k), 4, 0.5, torch.float16)
    wd = normal((k, n), 5, k ** -0.5, torch.float16)
    pre_in = normal((m, 2 * n), 6, 2.0, torch.float16)

    def all_of():
        out = [*run_forward(flint, cuda, x, w, b, "silu", True)]
        out += [run_forward(flint, cuda, x, w, None, "gelu", False)[0]]
        return out + [run_backward(flint, cuda, dout, wd, pre_in, a) for a in ("silu", "gelu")]

    want = None
    for name, plans in (("gemm_pipe", PIPE), ("gemm_small", SMALL)):
        for plan in plans:
            tune(name, plan)
            got = all_of()
            tune(name, None)
            want = want or got
            for i, (a, b_) in enumerate(zip(got, want)):
                assert torch.equal(a, b_), (name, plan, i)
    y_ref, y_bound, pre_ref, pre_bound = forward_reference(x, w, b, "silu")
    close(want[0], y_ref, y_bound)
    close(want[1], pre_ref, pre_bound)


@pytest.mark.gpu
def test_with_the_other_kernels_turned_off(flint, cuda, tune):
    """There is none behind these: a size that the pipeline does not take runs anyway."""
    x, w, b = forward_inputs(33, 40, 72, True)
    want, _ = run_forward(flint, cuda, x, w, b, "silu", False)
    for name in ("gemm_pipe", "gemm_small"):
        tune(name, "0")
        got, _ = run_forward(flint, cuda, x, w, b, "silu", False)
        assert torch.equal(got, want)
        tune(name, None)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(8, 16384, 65536), (70000, 4096, 8)])
def test_past_the_pipelines_sizes(flint, cuda, m, n, k):
    """Weights of 2^32 bytes, and projections of over 2^30 bytes; some columns looked
    at."""
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn((m, k), generator=g, device=cuda, dtype=torch.float16)
    w = torch.randn((2 * n, k), generator=g, device=cuda, dtype=torch.float16) * k ** -0.5
    y = torch.empty((m, n), dtype=torch.float16, device=cuda)
    pre = torch.empty((m, 2 * n), dtype=torch.float16, device=cuda)
    flint.gemm_nt_gated(y, pre, x, w, None, m, n, k, "silu")
    cols = [0, 15, 16, 31, n // 2 + 7, n - 17, n - 16, n - 1]
    rows = [0, m // 3, m - 1]
    at = torch.tensor(cols + [n + c for c in cols], device=cuda)
    y_ref, y_bound, pre_ref, pre_bound = forward_reference(x[rows].cpu(), w[at].cpu(), None, "silu")
    close(y[rows][:, at[:len(cols)]], y_ref, y_bound)
    close(pre[rows][:, at], pre_ref, pre_bound)
    # The gradient: w (2^31 bytes) as k x n.
    wd = w.view(-1)[:k * n].view(k, n)
    dpre = torch.empty((m, 2 * n), dtype=torch.float16, device=cuda)
    flint.gemm_nn_dgated(dpre, x, wd, pre, m, n, k, "silu")
    ref = backward_reference(x[rows].cpu(), wd[:, at[:len(cols)]].cpu(), pre[rows][:, at].cpu(), "silu")
    close(dpre[rows][:, at], *ref)


def check_rows(y, pre, dpre, x, w, dout, wd, pre_in, rows, act):
    """Whole rows of either pass against float64."""
    x, dout, w, wd = x[rows].cpu(), dout[rows].cpu(), w.cpu(), wd.cpu()
    y_ref, y_bound, pre_ref, pre_bound = forward_reference(x, w, None, act)
    close(y[rows], y_ref, y_bound)
    close(pre[rows], pre_ref, pre_bound)
    close(dpre[rows], *backward_reference(dout, wd, pre_in[rows].cpu(), act))


@pytest.mark.gpu
@pytest.mark.parametrize("k", [320, 328])
def test_several_tiles_a_workgroup_of_several_steps(flint, cuda, tune, k):
    """25 x 22 tiles of 256 x 192 for 256 CUs, and more of every other tile, of 5 steps and
    more: a workgroup's second and third tiles begin under the stores of the one before.
    Whole outputs are the same bits from every tile (k = 328 on the tile that takes partial
    steps), with the projections' stores through L2 and past it."""
    m, n, nd, act = 6151, 2056, 4104, "silu"
    g = torch.Generator(device="cuda").manual_seed(5)

    def random(rows, columns, std=1.0):
        return (torch.randn((rows, columns), generator=g, device=cuda) * std).half()

    x, w = random(m, k), random(2 * n, k, k ** -0.5)
    dout, wd, pre_in = random(m, k, 0.5), random(k, nd, k ** -0.5), random(m, 2 * nd, 2.0)
    rows = [0, 1, 31, 127, 128, 255, 256, 2999, m // 2, 4095, 4096, m - 9, m - 8, m - 7, m - 2, m - 1]

    def all_of():
        y, pre = run_forward(flint, cuda, x, w, None, act, True)
        alone, _ = run_forward(flint, cuda, x, w, None, act, False)
        return y, pre, alone, run_backward(flint, cuda, dout, wd, pre_in, act)

    want = all_of()
    check_rows(want[0], want[1], want[3], x, w, dout, wd, pre_in, rows, act)
    assert torch.equal(want[0], want[2])
    for name, plans in (("gemm_pipe", PIPE if k % 64 == 0 else ["128,192,3,64"]),
                        ("gemm_small", SMALL[3:])):
        for plan in plans:
            tune(name, plan)
            got = all_of()
            tune(name, None)
            for i, (a, b) in enumerate(zip(got, want)):
                assert torch.equal(a, b), (name, plan, i)


@pytest.mark.gpu
def test_outputs_past_the_pipelines_in_several_steps(flint, cuda):
    """Projections and gradients of 2.3 GB, past the pipeline's 2^31 bytes, k a whole step
    and a partial one: the first, middle and last rows."""
    m, n, k, act = 70001, 8192, 72, "gelu"
    assert m * 2 * n * 2 >= 1 << 31
    g = torch.Generator(device="cuda").manual_seed(6)
    x, dout = (torch.randn((m, k), generator=g, device=cuda, dtype=torch.float16) for _ in range(2))
    w = torch.randn((2 * n, k), generator=g, device=cuda, dtype=torch.float16) * k ** -0.5
    wd = w.view(-1)[:k * n].view(k, n)
    y, pre = run_forward(flint, cuda, x, w, None, act, True)
    dpre = run_backward(flint, cuda, dout, wd, pre, act)
    rows = [0, m // 2, m // 2 + 1, m - 2, m - 1]
    check_rows(y, pre, dpre, x, w, dout, wd, pre, rows, act)


@pytest.mark.gpu
def test_projections_past_2_to_the_32_values(flint, cuda):
    """The last rows of 550,000 x 8,192 projections, and of their gradients."""
    m, n, k = 550000, 4096, 8
    g = torch.Generator(device="cuda").manual_seed(4)
    x = torch.randn((m, k), generator=g, device=cuda, dtype=torch.float16)
    w = torch.randn((2 * n, k), generator=g, device=cuda, dtype=torch.float16) * k ** -0.5
    y = torch.empty((m, n), dtype=torch.float16, device=cuda)
    pre = torch.empty((m, 2 * n), dtype=torch.float16, device=cuda)
    flint.gemm_nt_gated(y, pre, x, w, None, m, n, k, "gelu")
    wd = w.view(-1)[:k * n].view(k, n)
    dpre = torch.empty((m, 2 * n), dtype=torch.float16, device=cuda)
    flint.gemm_nn_dgated(dpre, x, wd, pre, m, n, k, "gelu")
    for rows in (slice(0, 2), slice(m // 2, m // 2 + 2), slice(m - 2, m)):
        y_ref, y_bound, pre_ref, pre_bound = forward_reference(x[rows].cpu(), w.cpu(), None, "gelu")
        close(y[rows], y_ref, y_bound)
        close(pre[rows], pre_ref, pre_bound)
        close(dpre[rows], *backward_reference(x[rows].cpu(), wd.cpu(), pre[rows].cpu(), "gelu"))


@pytest.mark.gpu
def test_non_finite_values_stay_in_their_rows_and_columns(flint, cuda):
    m, n, k = 40, 48, 64
    x, w, _ = forward_inputs(m, n, k, False)
    clean, clean_pre = run_forward(flint, cuda, x, w, None, "silu", True)
    x[7, 3], w[5, 9], w[n + 20, 1] = float("nan"), float("inf"), float("nan")
    y, pre = run_forward(flint, cuda, x, w, None, "silu", True)
    keep = torch.ones(m, n, dtype=torch.bool, device=cuda)
    keep[7] = False
    keep[:, 5] = False
    keep[:, 20] = False
    assert torch.equal(y[keep], clean[keep])
    assert torch.isnan(y[7]).all() and torch.isnan(y[:, 20]).all()
    assert torch.isnan(pre[7]).all()
    assert torch.equal(pre[:, :5][:7], clean_pre[:, :5][:7])


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_projections_that_overflowed(flint, cuda, act):
    """act and act' are 0 at -inf, act' is 1 at +inf; large finite values likewise."""
    m, n, k = 2, 8, 8
    inf = float("inf")
    dout, w = torch.ones(m, k).half(), torch.ones(k, n).half() * 0.125      # s = 1
    pre = torch.zeros(m, 2 * n).half()
    pre[0, :n] = torch.tensor([-inf, inf, -65504.0, 65504.0, float("nan"), 0.0, -30.0, 30.0])
    pre[0, n:] = 2.0
    dpre = run_backward(flint, cuda, dout, w, pre, act).cpu()
    dg, du = dpre[0, :n], dpre[0, n:]
    assert dg[[0, 2]].tolist() == [0.0, 0.0] and dg[[1, 3]].tolist() == [2.0, 2.0]
    assert du[[0, 2]].tolist() == [0.0, 0.0] and du[[1, 3]].tolist() == [inf, 65504.0]
    assert torch.isnan(dg[4]) and torch.isnan(du[4])
    assert dg[5] == 1.0 and du[5] == 0.0
    assert torch.isfinite(dpre[0, [6, 7, n + 6, n + 7]]).all()
    assert torch.all(dpre[1, :n] == 0.0)


@pytest.mark.gpu
def test_large_sums_stay_finite(flint, cuda):
    """A bias of 1e30 on the gate: act(g) = g, and s^2 overflows FP32."""
    x, w = torch.zeros(1, 8).half(), torch.zeros(16, 8).half()
    bias = torch.zeros(16)
    bias[0], bias[1], bias[8:] = 1e30, -1e30, 1e-30
    for act in ("silu", "gelu"):
        y, _ = run_forward(flint, cuda, x, w, bias, act, False)
        assert abs(float(y[0, 0]) - 1.0) <= 2.0 ** -10
        assert float(y[0, 1]) == 0.0


@pytest.mark.gpu
def test_captured_and_on_another_stream(flint, cuda):
    m, n, k = 70, 136, 128
    x, w, b = (t.to(cuda) for t in forward_inputs(m, n, k, True))
    dout = normal((m, k), 4, 0.5, torch.float16).to(cuda)
    wd = normal((k, n), 5, k ** -0.5, torch.float16).to(cuda)
    y = torch.empty((m, n), dtype=torch.float16, device=cuda)
    pre, dpre = (torch.empty((m, 2 * n), dtype=torch.float16, device=cuda) for _ in range(2))
    stream = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        flint.gemm_nt_gated(y, pre, x, w, b, m, n, k, "gelu")
        flint.gemm_nn_dgated(dpre, dout, wd, pre, m, n, k, "gelu")
    for i in range(3):
        x.mul_(0.5 if i else 1.0)
        graph.replay()
        y_ref, y_bound, pre_ref, pre_bound = forward_reference(x.cpu(), w.cpu(), b.cpu(), "gelu")
        close(y, y_ref, y_bound)
        close(pre, pre_ref, pre_bound)
        close(dpre, *backward_reference(dout.cpu(), wd.cpu(), pre.cpu(), "gelu"))
        for t in (y, pre, dpre):
            t.fill_(SENTINEL)


# ------------------------------------------------------------------ refusals

A = 0x1000000   # a 16-byte-aligned fake device address: refusals never read it


def fails(flint, fn, *args, message):
    status = getattr(flint.lib, fn)(*args)
    assert status == flint_lib.ERROR_INVALID_ARGUMENT
    assert message in flint.last_error(), flint.last_error()


SIZE_REFUSALS = [
    ((4, 8, 12, 0), "k (12) must be a positive multiple of 8"),
    ((4, 8, 0, 0), "k (0) must be a positive multiple of 8"),
    ((4, 12, 8, 0), "n (12) must be a multiple of 8"),
    ((4, 8, 8, 2), "activation (2) must be 0 or 1"),
    ((4, 8, 1 << 17, 0), "4 x 8 x 131072 is too large"),
    ((4, 65535 * 64 + 8, 8, 0), "is too large: m can be up to 8388480, n up to 4194240, m n up to "
                                "17179869184, and k up to 65536"),
    ((1 << 21, 1 << 14, 8, 0), "2097152 x 16384 x 8 is too large"),
]


@pytest.mark.parametrize("sizes,message", SIZE_REFUSALS)
def test_sizes_refused(flint, sizes, message):
    m, n, k, act = sizes
    fails(flint, "flint_gemm_nt_gated", A, 2 * A, 3 * A, 4 * A, None, m, n, k, act, None,
          message=f"flint_gemm_nt_gated: {message}" if message[0] != "i" else message)
    fails(flint, "flint_gemm_nn_dgated", A, 2 * A, 3 * A, 4 * A, m, n, k, act, None,
          message=f"flint_gemm_nn_dgated: {message}" if message[0] != "i" else message)


def test_buffers_refused(flint):
    fn = "flint_gemm_nt_gated"
    good = [A, 2 * A, 3 * A, 4 * A, 5 * A]
    for i, name in ((0, "y"), (2, "x"), (3, "w")):
        bad = list(good)
        bad[i] = None
        fails(flint, fn, *bad, 4, 8, 8, 0, None, message=f"{fn}: {name} is null")
    for i, name in enumerate(("y", "pre", "x", "w", "bias")):
        bad = list(good)
        bad[i] += 8
        fails(flint, fn, *bad, 4, 8, 8, 0, None, message=f"{fn}: {name} is not 16-byte aligned")
    for i, j, message in ((0, 2, "y and x overlap"), (0, 3, "y and w overlap"),
                          (0, 4, "y and bias overlap"), (1, 0, "pre and y overlap"),
                          (1, 2, "pre and x overlap"), (1, 3, "pre and w overlap"),
                          (1, 4, "pre and bias overlap")):
        bad = list(good)
        bad[i] = bad[j] + 16
        fails(flint, fn, *bad, 4, 8, 8, 0, None, message=f"{fn}: {message}")
    fn = "flint_gemm_nn_dgated"
    good = good[:4]
    for i, name in enumerate(("dpre", "x", "w", "pre")):
        bad = list(good)
        bad[i] = None
        fails(flint, fn, *bad, 4, 8, 8, 0, None, message=f"{fn}: {name} is null")
        bad[i] = good[i] + 8
        fails(flint, fn, *bad, 4, 8, 8, 0, None, message=f"{fn}: {name} is not 16-byte aligned")
        if i:
            bad[i] = good[0] + 16
            fails(flint, fn, *bad, 4, 8, 8, 0, None, message=f"{fn}: dpre and {name} overlap")


def test_nothing_to_do(flint):
    for m, n in ((0, 8), (8, 0)):
        assert flint.lib.flint_gemm_nt_gated(*[None] * 5, m, n, 3, 9, None) == 0
        assert flint.lib.flint_gemm_nn_dgated(*[None] * 4, m, n, 3, 9, None) == 0
    with pytest.raises(ctypes.ArgumentError):
        flint.gemm_nt_gated(A, None, A, A, None, 1, 8, 8, "relu", stream=0)
