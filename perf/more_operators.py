"""Rotary positions, the gated feed-forward product with its gradient, and the
attention of new tokens over a paged cache of 8-bit values: measurable cases, in
plain form and through the library.

  rotary   each head's pairs of values of q and k turned by their token's position
           (frequencies scaled for long contexts, a part of the head, pairs of
           halves or of neighbours); training adds the turn back of the gradients
  gated    activation(gate) * up of both projections of x; training keeps the
           projections for the gradient
  dgated   the projections' gradient from the output's, through the down
           projection, the product and the activation
  paged8   new tokens of each sequence attend over a paged cache in e4m3 with a
           power of two a block of positions and head, and are stored into it

`run` computes the plain form in FP32 with elementary torch operations, or
(own) makes the library's calls. `exact` restates each operator in FP64.
"""

import math
import random

import torch

own = False


def listed():
    return [
        # A serving step's 64 tokens at far positions, grouped heads of 128, the
        # slow frequencies scaled for eight times the trained length: latency.
        dict(name="rotary-decode-64", kind="rotary", tokens=64, mix=1, far=131071, heads=32,
             kv_heads=8, head_width=128, width=128, pairs=False, base=500000.0, factor=8.0,
             original=8192, train=False),
        # A training batch of packed documents at the GPT-2 124M heads, with the
        # gradients turned back.
        dict(name="rotary-train-8192", kind="rotary", tokens=8192, mix=2, far=2047, heads=12,
             kv_heads=12, head_width=64, width=64, pairs=False, base=10000.0, factor=1.0,
             original=0, train=True),
        # A long prompt of an odd length, half of each head turned in pairs of
        # neighbours.
        dict(name="rotary-prompt-16411", kind="rotary", tokens=16411, mix=3, far=16410, heads=32,
             kv_heads=8, head_width=128, width=64, pairs=True, base=10000.0, factor=4.0,
             original=4096, train=False),
        # One token of a generation at GPT-2 124M's width: latency.
        dict(name="gated-decode-1", kind="gated", m=1, n=2048, k=768, act="silu", bias=False,
             train=False),
        # A serving batch's step on a wide layer: reading the weights.
        dict(name="gated-decode-64", kind="gated", m=64, n=5504, k=2048, act="silu", bias=False,
             train=False),
        # Prompts of odd lengths, GELU and a bias, a ragged width.
        dict(name="gated-eval-1000", kind="gated", m=1000, n=4264, k=1600, act="gelu", bias=True,
             train=False),
        # A training batch's forward pass: the projections kept.
        dict(name="gated-train-8192", kind="gated", m=8192, n=2048, k=768, act="silu", bias=False,
             train=True),
        # The same batch's gradient of the projections.
        dict(name="dgated-train-8192", kind="dgated", m=8192, n=2048, k=768, act="silu"),
        # A wide layer's, on an odd number of tokens.
        dict(name="dgated-train-2053", kind="dgated", m=2053, n=5504, k=2048, act="gelu"),
        # Generation of one sequence, one token at a time: latency.
        dict(name="paged8-decode-1", kind="paged8", sequences=1, new=1, cached=777, mix=1,
             heads=12, kv_heads=12, head_width=64, page_size=16, block=16),
        # A serving batch: 64 sequences of different lengths, grouped heads of
        # width 128, one token each.
        dict(name="paged8-decode-64", kind="paged8", sequences=64, new=1, cached=8192, mix=2,
             heads=32, kv_heads=8, head_width=128, page_size=64, block=32),
        # Chunks of prompts over what is cached of them, odd lengths.
        dict(name="paged8-chunk-500", kind="paged8", sequences=4, new=500, cached=4096, mix=4,
             heads=12, kv_heads=4, head_width=64, page_size=16, block=8),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _heads(rng):
    kv_heads = rng.randint(1, 8)
    heads = kv_heads * rng.choice([1, 1, 2, 3, 4, 8])
    while heads > 32:
        heads -= kv_heads
    return heads, kv_heads


def draw(rng):
    kind = rng.choice(["rotary", "gated", "gated", "dgated", "paged8", "paged8"])
    if kind == "rotary":
        heads, kv_heads = _heads(rng)
        head_width = rng.choice([64, 64, 80, 96, 128, 128, 256])
        case = dict(kind=kind, tokens=_log_int(rng, 1, 16384), mix=rng.randrange(1 << 16),
                    far=_log_int(rng, 16, 1 << 20), heads=heads, kv_heads=kv_heads,
                    head_width=head_width,
                    width=rng.choice([head_width, head_width, head_width // 2, head_width // 4]),
                    pairs=rng.random() < 0.5, base=rng.choice([10000.0, 500000.0]),
                    factor=rng.choice([1.0, 2.0, 8.0]), original=rng.choice([0, 2048, 8192]),
                    train=rng.random() < 0.4)
        most = max(work(c)["bytes"] for c in listed() if c["kind"] == kind)
        while work(case)["bytes"] > most:
            case["tokens"] = case["tokens"] * 3 // 4
        return case
    if kind in ("gated", "dgated"):
        case = dict(kind=kind, m=_log_int(rng, 1, 8192), n=8 * _log_int(rng, 8, 688),
                    k=8 * _log_int(rng, 8, 256), act=rng.choice(["silu", "gelu"]))
        if kind == "gated":
            case.update(bias=rng.random() < 0.3, train=rng.random() < 0.5)
        most = max(work(c)["flops"] for c in listed() if c["kind"] == kind)
        while work(case)["flops"] > most:
            case["m"] = case["m"] * 3 // 4
        return case
    heads, kv_heads = _heads(rng)
    mode = rng.random()
    if mode < 0.5:
        new, sequences, cached = 1, _log_int(rng, 1, 64), _log_int(rng, 1, 8192)
    elif mode < 0.65:
        new, sequences, cached = 1, rng.randint(1, 2), _log_int(rng, 8192, 131072)
    else:
        new, sequences, cached = _log_int(rng, 2, 600), _log_int(rng, 1, 4), _log_int(rng, 1, 4096)
    page_size = rng.choice([8, 16, 32, 64, 128])
    return dict(kind=kind, sequences=sequences, new=new, cached=cached, mix=rng.randrange(1 << 16),
                heads=heads, kv_heads=kv_heads, head_width=rng.choice([64, 64, 128]),
                page_size=page_size,
                block=rng.choice([b for b in (1, 4, 8, 16, 32, 64, 128) if b <= page_size]))


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
    """What a program makes once beside its tensors (shapes, plans, workspaces)."""
    if name not in state:
        state[name] = make()
    return state[name]


# ------------------------------------------------------------------ rotary
# Turns that a pair makes over the trained length: under the first its frequency
# is divided by the factor, over the second it is kept.
LOW, HIGH = 1.0, 32.0


def _magnitude(case):
    return 0.1 * math.log(case["factor"]) + 1.0


def _rotary_inputs(case, g):
    T, H, Hk, w = case["tokens"], case["heads"], case["kv_heads"], case["head_width"]
    if case["tokens"] <= 256:      # tokens of many sequences, anywhere in them
        positions = torch.randint(0, case["far"] + 1, (T,), generator=g, device="cuda",
                                  dtype=torch.int32)
    else:                          # documents one after another
        positions = torch.arange(T, device="cuda", dtype=torch.int32) % (case["far"] + 1)
    # q, k and v are column slices of one projection, as a model has them.
    wide = (H + 2 * Hk) * w
    qkv = _normal(g, (T, wide))
    s = dict(qkv=qkv, q=qkv[:, :H * w], k=qkv[:, H * w:(H + Hk) * w], positions=positions,
             q_out=torch.empty((T, H * w), dtype=torch.float16, device="cuda"),
             k_out=torch.empty((T, Hk * w), dtype=torch.float16, device="cuda"))
    if case["train"]:
        s.update(dq_out=_normal(g, (T, H * w), 1e-2), dk_out=_normal(g, (T, Hk * w), 1e-2),
                 dqkv=torch.zeros_like(qkv))
    return s


def _rotary_run(case, s):
    return _rotary_own(case, s) if own else _rotary_plain(case, s)


def _rotary_own(case, s):
    f = _flint()
    T, H, Hk, w = case["tokens"], case["heads"], case["kv_heads"], case["head_width"]
    wide = s["qkv"].shape[1]

    def plan():
        p = _bytes(f.rotary_plan_bytes(case["width"]))
        f.rotary_plan(p, f.rotary_angles(case["width"], case["base"], case["factor"],
                                         case["original"], LOW, HIGH, _magnitude(case)))
        return p

    p = _once(s, "plan", plan)
    shape = _once(s, "shape", lambda: f.rotary_shape(T, H, Hk, w, case["width"], case["pairs"],
                                                      wide, wide, H * w, Hk * w))
    f.rotary(s["q_out"], s["k_out"], s["q"], s["k"], s["positions"], p, shape)
    if not case["train"]:
        return dict(q=s["q_out"], k=s["k_out"])
    back = _once(s, "back", lambda: f.rotary_shape(T, H, Hk, w, case["width"], case["pairs"],
                                                    H * w, Hk * w, wide, wide))
    d = s["dqkv"]
    f.rotary(d[:, :H * w], d[:, H * w:(H + Hk) * w], s["dq_out"], s["dk_out"], s["positions"], p,
             back, backward=True)
    return dict(q=s["q_out"], k=s["k_out"], dqkv=d)


def _rotary_plain(case, s):
    T, w, width = case["tokens"], case["head_width"], case["width"]
    # Angles in 64 bits: at position 100,000 one in 32 is off by a hundredth.
    f = case["base"] ** (torch.arange(0, width, 2, device="cuda", dtype=torch.float64) / -width)
    keep = ((f * (case["original"] / (2 * math.pi)) - LOW) / (HIGH - LOW)).clamp_(0.0, 1.0)
    f = f * (keep + (1.0 - keep) / case["factor"])
    angle = s["positions"].double()[:, None] * f
    cos = (angle.cos() * _magnitude(case)).float()[:, None]
    sin = (angle.sin() * _magnitude(case)).float()[:, None]

    def turned(x, sin):
        x = x.float().reshape(T, -1, w)
        out = x.clone()
        a, b = ((slice(0, width, 2), slice(1, width, 2)) if case["pairs"]
                else (slice(0, width // 2), slice(width // 2, width)))
        out[:, :, a] = x[:, :, a] * cos - x[:, :, b] * sin
        out[:, :, b] = x[:, :, a] * sin + x[:, :, b] * cos
        return out.reshape(T, -1)

    s["q_out"].copy_(turned(s["q"], sin))
    s["k_out"].copy_(turned(s["k"], sin))
    if not case["train"]:
        return dict(q=s["q_out"], k=s["k_out"])
    nq, nk = s["q_out"].shape[1], s["k_out"].shape[1]
    s["dqkv"][:, :nq] = turned(s["dq_out"], -sin)
    s["dqkv"][:, nq:nq + nk] = turned(s["dk_out"], -sin)
    return dict(q=s["q_out"], k=s["k_out"], dqkv=s["dqkv"])


def _rotary_exact(case, s):
    T, w, width = case["tokens"], case["head_width"], case["width"]
    position = s["positions"].double()
    out = dict(q=s["q"].double(), k=s["k"].double())
    if case["train"]:
        out["dqkv"] = torch.zeros_like(s["qkv"], dtype=torch.float64)
        nq, nk = s["dq_out"].shape[1], s["dk_out"].shape[1]
        out["dqkv"][:, :nq] = s["dq_out"]
        out["dqkv"][:, nq:nq + nk] = s["dk_out"]
    out = {name: x.clone() for name, x in out.items()}
    for i in range(width // 2):
        f = math.exp(-2.0 * i / width * math.log(case["base"]))
        r = case["original"] * f / (2.0 * math.pi)
        keep = min(1.0, max(0.0, (r - LOW) / (HIGH - LOW)))
        turn = torch.polar(torch.full_like(position, _magnitude(case)),
                           position * (f * keep + f * (1.0 - keep) / case["factor"]))
        a, b = (2 * i, 2 * i + 1) if case["pairs"] else (i, i + width // 2)
        for name, x in out.items():
            heads = (case["heads"] + case["kv_heads"]) if name == "dqkv" else x.shape[1] // w
            x = x[:, :heads * w].view(T, heads, w) if name != "dqkv" else \
                x.view(T, -1, w)[:, :heads]
            z = torch.complex(x[:, :, a], x[:, :, b]) * (
                turn.conj() if name == "dqkv" else turn)[:, None]
            x[:, :, a], x[:, :, b] = z.real, z.imag
    return out


def _rotary_work(case):
    values = case["tokens"] * (case["heads"] + case["kv_heads"]) * case["head_width"]
    passes = 2 if case["train"] else 1
    return dict(flops=passes * 3 * values, bytes=passes * (4 * values + 4 * case["tokens"]))


# ------------------------------------------------------------------- gated
def _gated_inputs(case, g):
    m, n, k = case["m"], case["n"], case["k"]
    s = dict(x=_normal(g, (m, k)), w=_normal(g, (2 * n, k), k ** -0.5), bias=None, pre=None,
             y=torch.empty((m, n), dtype=torch.float16, device="cuda"))
    if case["bias"]:
        s["bias"] = _normal(g, (2 * n,), 0.2, torch.float32)
    if case["train"]:
        s["pre"] = torch.empty((m, 2 * n), dtype=torch.float16, device="cuda")
    return s


def _activation(case, g):
    if case["act"] == "silu":
        return g / (1.0 + torch.exp(-g))
    # 0.5 g (1 + tanh u) without the difference: g / (1 + exp(-2 u)).
    return g / (1.0 + torch.exp(-2.0 * math.sqrt(2.0 / math.pi) * (g + 0.044715 * g * g * g)))


def _gated_run(case, s):
    return _gated_own(case, s) if own else _gated_plain(case, s)


def _gated_own(case, s):
    f = _flint()
    f.gemm_nt_gated(s["y"], s["pre"], s["x"], s["w"], s["bias"], case["m"], case["n"], case["k"],
                    case["act"])
    return dict(y=s["y"], pre=s["pre"]) if case["train"] else dict(y=s["y"])


def _gated_plain(case, s):
    n = case["n"]
    pre = s["x"].float() @ s["w"].float().T
    if case["bias"]:
        pre += s["bias"]
    s["y"].copy_(_activation(case, pre[:, :n]) * pre[:, n:])
    if not case["train"]:
        return dict(y=s["y"])
    s["pre"].copy_(pre)
    return dict(y=s["y"], pre=s["pre"])


def _gated_exact(case, s):
    n = case["n"]
    pre = torch.matmul(s["x"].double(), s["w"].double().T.contiguous())
    if case["bias"]:
        pre = pre + s["bias"].double()
    gate, up = pre[:, :n], pre[:, n:]
    if case["act"] == "silu":
        y = gate * torch.special.expit(gate) * up
    else:
        y = torch.nn.functional.gelu(gate, approximate="tanh") * up
    return dict(y=y, pre=pre) if case["train"] else dict(y=y)


def _gated_work(case):
    m, n, k = case["m"], case["n"], case["k"]
    return dict(flops=4 * m * n * k,
                bytes=2 * (m * k + 2 * n * k + m * n + (2 * m * n if case["train"] else 0))
                + (8 * n if case["bias"] else 0))


# ------------------------------------------------------------------ dgated
def _dgated_inputs(case, g):
    m, n, k = case["m"], case["n"], case["k"]
    return dict(dout=_normal(g, (m, k), 1e-1), w=_normal(g, (k, n), k ** -0.5),
                pre=_normal(g, (m, 2 * n)),
                dpre=torch.empty((m, 2 * n), dtype=torch.float16, device="cuda"))


def _dgated_run(case, s):
    return _dgated_own(case, s) if own else _dgated_plain(case, s)


def _dgated_own(case, s):
    _flint().gemm_nn_dgated(s["dpre"], s["dout"], s["w"], s["pre"], case["m"], case["n"],
                            case["k"], case["act"])
    return dict(dpre=s["dpre"])


def _dgated_plain(case, s):
    n = case["n"]
    d = s["dout"].float() @ s["w"].float()
    gate, up = s["pre"][:, :n].float(), s["pre"][:, n:].float()
    if case["act"] == "silu":
        e = torch.exp(-gate)
        sigma = 1.0 / (1.0 + e)
        slope = sigma * (1.0 + gate * (e * sigma))
    else:
        c = 2.0 * math.sqrt(2.0 / math.pi)
        e = torch.exp(-c * (gate + 0.044715 * gate * gate * gate))
        sigma = 1.0 / (1.0 + e)
        slope = sigma * (1.0 + gate * (e * sigma) * c * (1.0 + 3 * 0.044715 * gate * gate))
    s["dpre"][:, :n] = d * up * slope
    s["dpre"][:, n:] = d * _activation(case, gate)
    return dict(dpre=s["dpre"])


def _dgated_exact(case, s):
    n = case["n"]
    d = torch.matmul(s["dout"].double(), s["w"].double())
    gate = s["pre"][:, :n].double().requires_grad_(True)
    with torch.enable_grad():
        act = (torch.nn.functional.silu(gate) if case["act"] == "silu"
               else torch.nn.functional.gelu(gate, approximate="tanh"))
        (slope,) = torch.autograd.grad(act.sum(), gate)
    return dict(dpre=torch.cat([d * s["pre"][:, n:].double() * slope, d * act.detach()], 1))


def _dgated_work(case):
    m, n, k = case["m"], case["n"], case["k"]
    return dict(flops=2 * m * n * k, bytes=2 * (m * k + k * n + 4 * m * n))


# ------------------------------------------------------------------ paged8
# e4m3's largest value, and the exponents of a block's scale (stored plus 127).
MOST, LEAST_E, MOST_E = 448.0, -15, 8


def _chunks(case):
    """(cached, new) of each sequence: caches from an eighth of the case's
    length to all of it, new tokens from half of the chunk to all of it."""
    rng = random.Random(case["mix"])
    n, c = case["new"], case["cached"]
    return [(c if i == 0 else rng.randint((c + 7) // 8, c),
             n if i == 0 else rng.randint((n + 1) // 2, n)) for i in range(case["sequences"])]


def _exponent(largest):
    """The least e at which largest <= MOST 2^e, within its range."""
    f, x = torch.frexp(largest)
    return (x - 9 + (f > 0.875).int()).clamp_(LEAST_E, MOST_E)


def _coded(x, e):
    """x 2^-e in e4m3, to the nearest value that FP16 holds times 2^e."""
    most = torch.where(e == MOST_E, 240.0, MOST)
    return torch.ldexp(x, -e).clamp(-most, most).to(torch.float8_e4m3fn)


def _paged8_pool(g, pages, kv_heads, page_size, width, block):
    x = _normal(g, (pages, kv_heads, page_size // block, block, width), 1.0, torch.float32)
    e = _exponent(x.abs().amax((3, 4)))
    coded = _coded(x, e[..., None, None]).view(torch.uint8)
    return coded.view(pages, kv_heads, page_size, width), (e + 127).to(torch.uint8)


def _paged8_inputs(case, g):
    H, Hk, w, size = case["heads"], case["kv_heads"], case["head_width"], case["page_size"]
    chunks = _chunks(case)
    need = [-(-(c + n) // size) for c, n in chunks]
    pages, columns = sum(need) + 3, max(need) + 1
    # Pages are handed out in no order; entries past a sequence's last hold -1.
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(chunks), columns), -1, dtype=torch.int32, device="cuda")
    for i, (a, n) in enumerate(zip(_offsets(need), need)):
        table[i, :n] = order[a:a + n]
    tokens = sum(n for _, n in chunks)
    qkv = _normal(g, (tokens, (H + 2 * Hk) * w))
    k_pages, k_scales = _paged8_pool(g, pages, Hk, size, w, case["block"])
    v_pages, v_scales = _paged8_pool(g, pages, Hk, size, w, case["block"])
    return dict(qkv=qkv, q=qkv[:, :H * w], k=qkv[:, H * w:(H + Hk) * w], v=qkv[:, (H + Hk) * w:],
                k_pages=k_pages, k_scales=k_scales, v_pages=v_pages, v_scales=v_scales,
                table=table, offsets=_ints(_offsets([n for _, n in chunks])),
                cached=_ints([c for c, _ in chunks]), scale=1.0 / math.sqrt(w),
                o=torch.empty((tokens, H * w), dtype=torch.float16, device="cuda"))


def _paged8_outputs(s):
    # The values that the pages stand for: e4m3 numbers, in units of their block's
    # power of two.
    return dict(o=s["o"], k_pages=s["k_pages"].view(torch.float8_e4m3fn), k_scales=s["k_scales"],
                v_pages=s["v_pages"].view(torch.float8_e4m3fn), v_scales=s["v_scales"])


def _paged8_run(case, s):
    return _paged8_own(case, s) if own else _paged8_plain(case, s)


def _paged8_own(case, s):
    f = _flint()
    H, Hk, w = case["heads"], case["kv_heads"], case["head_width"]
    tokens, wide = s["qkv"].shape
    shape = _once(s, "shape", lambda: f.paged_shape(
        tokens, case["sequences"], case["new"], H, Hk, w, wide, wide, H * w,
        s["k_pages"].shape[0], case["page_size"], s["table"].shape[1]))
    ws = _once(s, "ws", lambda: _bytes(f.attention_paged8_workspace(shape, case["block"])))
    f.attention_paged8(s["o"], s["k_pages"], s["k_scales"], s["v_pages"], s["v_scales"], s["q"],
                       s["k"], s["v"], s["offsets"], s["cached"], s["table"], shape, case["block"],
                       s["scale"], ws)
    return _paged8_outputs(s)


def _paged8_plain(case, s):
    H, Hk, w, size = case["heads"], case["kv_heads"], case["head_width"], case["page_size"]
    S, N, G, B = case["sequences"], case["new"], H // Hk, case["block"]
    tokens = s["qkv"].shape[0]
    first = s["offsets"].long()
    cached = s["cached"].long()
    count = first[1:] - first[:-1]
    token = torch.arange(tokens, device="cuda")
    seq = torch.searchsorted(first, token, right=True) - 1
    place = token - first[seq]

    # The new rows as given, the cached ones as they are stored.
    at = (first[:-1, None] + torch.arange(N, device="cuda")).clamp_(max=tokens - 1)
    q = s["q"][at].float().view(S, N, Hk, G, w).permute(0, 2, 3, 1, 4).reshape(S, Hk, G * N, w)
    table = s["table"].clamp(min=0)

    def held(name):
        e = s[name + "_scales"][table].int() - 127
        x = s[name + "_pages"][table].view(torch.float8_e4m3fn).float()
        x = torch.ldexp(x, e.repeat_interleave(B, -1)[..., None])
        x = x.transpose(1, 2).reshape(S, Hk, -1, w)
        p = torch.arange(x.shape[2], device="cuda")
        x = torch.where((p < cached[:, None])[:, None, :, None], x, 0.0)
        x[seq, :, cached[seq] + place] = s[name].view(tokens, Hk, w).float()
        return x

    k, v = held("k"), held("v")
    last = (cached[:, None] + torch.arange(N, device="cuda")).repeat(1, G)
    seen = torch.arange(k.shape[2], device="cuda") <= last[:, :, None]
    p = (q @ k.transpose(2, 3)).mul_(s["scale"]).masked_fill_(~seen[:, None], -math.inf)
    p.sub_(p.amax(-1, keepdim=True)).exp_()
    p.div_(p.sum(-1, keepdim=True))
    o = (p @ v).view(S, Hk, G, N, w).permute(0, 3, 1, 2, 4).reshape(S, N, H * w)
    s["o"].copy_(o[seq, place])

    # Every block that holds a new row, whole: [sequence, block, row].
    row = (cached // B)[:, None] + torch.arange((N - 1) // B + 2, device="cuda")
    row = (row * B)[:, :, None] + torch.arange(B, device="cuda")
    new = (row >= cached[:, None, None]) & (row < (cached + count)[:, None, None])
    s_at, b_at = new.any(2).nonzero(as_tuple=True)
    row, new = row[s_at, b_at], new[s_at, b_at]
    old = (row < cached[s_at, None])[:, None, :, None]
    page = s["table"][s_at, row[:, 0] // size].long()
    inside = row % size
    source = (first[s_at, None] + row - cached[s_at, None]).clamp_(0, tokens - 1)
    fresh = new[:, None, :, None]
    some_old = old.any(2)[:, :, 0]
    for name in ("k", "v"):
        x = s[name].view(tokens, Hk, w)[source].transpose(1, 2).float()
        codes = s[name + "_pages"].view(-1, Hk, size // B, B, w)
        scales = s[name + "_scales"]
        was = scales[page, :, inside[:, 0] // B].int() - 127
        kept = codes[page, :, inside[:, 0] // B]
        e = _exponent(torch.where(fresh, x, 0.0).abs().amax((2, 3)))
        e = torch.where(some_old, torch.maximum(e, was), e)
        values = torch.ldexp(kept.view(torch.float8_e4m3fn).float(), was[:, :, None, None])
        put = _coded(torch.where(fresh, x, values), e[:, :, None, None]).view(torch.uint8)
        codes[page, :, inside[:, 0] // B] = torch.where(fresh | old, put, kept)
        scales[page, :, inside[:, 0] // B] = (e + 127).to(torch.uint8)
    return _paged8_outputs(s)


def _paged8_exact(case, s):
    H, Hk, w, size = case["heads"], case["kv_heads"], case["head_width"], case["page_size"]
    B = case["block"]
    out = torch.zeros_like(s["o"], dtype=torch.float64)
    # Pages after the call, in units of their blocks' scales, not rounded.
    stored = {}
    for name in "kv":
        stored[name] = s[name + "_pages"].view(torch.float8_e4m3fn).double()
        stored[name + "e"] = s[name + "_scales"].int() - 127
    table = s["table"].tolist()
    t = 0
    for i, (c, n) in enumerate(_chunks(case)):
        chosen = table[i][:-(-(c + n) // size)]
        whole = {}
        for name in "kv":
            codes = stored[name][chosen].transpose(1, 2).reshape(-1, Hk, w)
            power = torch.pow(2.0, stored[name + "e"][chosen].double())
            power = power.repeat_interleave(B, -1).transpose(1, 2).reshape(-1, Hk)
            rows = codes * power[:, :, None]
            rows[c:c + n] = s[name][t:t + n].reshape(n, Hk, w).double()
            whole[name] = rows[:c + n].clone()
            b0, b1 = c // B, (c + n - 1) // B + 1
            block = rows[b0 * B:b1 * B].view(b1 - b0, B, Hk, w)
            place = torch.arange(b0 * B, b1 * B, device="cuda").view(b1 - b0, B)
            block = torch.where((place < c + n)[:, :, None, None], block, 0.0)
            fresh = torch.where((place >= c)[:, :, None, None], block, 0.0).abs().amax((1, 3))
            e = torch.ceil(torch.log2(fresh.clamp(min=1e-30) / 448.0)).clamp(-15, 8)
            if c % B:
                e[0] = torch.maximum(e[0], torch.log2(power[c - 1]))
            scaled = rows[b0 * B:b1 * B].view(b1 - b0, B, Hk, w) / torch.pow(2.0, e)[:, None, :, None]
            live = (place < c + n)[:, :, None, None]
            codes = codes.clone()
            kept = codes[b0 * B:b1 * B].view(b1 - b0, B, Hk, w)
            codes[b0 * B:b1 * B] = torch.where(live, scaled, kept).reshape(-1, Hk, w)
            stored[name][chosen] = codes.view(len(chosen), size, Hk, w).transpose(1, 2).contiguous()
        hidden = torch.arange(c + n, device="cuda") > torch.arange(c, c + n, device="cuda")[:, None]
        for h in range(H):
            j = h // (H // Hk)
            q = s["q"][t:t + n, h * w:h * w + w].double()
            x = torch.matmul(q, whole["k"][:, j].T.contiguous()) * s["scale"]
            x[hidden] = -math.inf
            p = torch.exp_(x - torch.logsumexp(x, 1)[:, None])
            out[t:t + n, h * w:h * w + w] = torch.matmul(p, whole["v"][:, j])
        t += n
    return dict(o=out, k_pages=stored["k"], k_scales=None, v_pages=stored["v"], v_scales=None)


def _paged8_work(case):
    H, Hk, w = case["heads"], case["kv_heads"], case["head_width"]
    chunks = _chunks(case)
    pairs = sum(n * c + n * (n + 1) // 2 for c, n in chunks)
    new = sum(n for _, n in chunks)
    # The cached rows and their blocks' scales read; the new rows of q, k and v
    # read, of o, k and v written.
    cached = sum(c * w + -(-c // case["block"]) for c, _ in chunks) * Hk * 2
    return dict(flops=4 * w * H * pairs,
                bytes=cached + new * (4 * H * w + 4 * Hk * w + 2 * Hk * w))


_PREPARE = dict(rotary=_rotary_inputs, gated=_gated_inputs, dgated=_dgated_inputs,
                paged8=_paged8_inputs)
_RUN = dict(rotary=_rotary_run, gated=_gated_run, dgated=_dgated_run, paged8=_paged8_run)
_EXACT = dict(rotary=_rotary_exact, gated=_gated_exact, dgated=_dgated_exact,
              paged8=_paged8_exact)
_WORK = dict(rotary=_rotary_work, gated=_gated_work, dgated=_dgated_work, paged8=_paged8_work)
