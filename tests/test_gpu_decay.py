"""Linear attention with a decay per head (kernels.decay_linear_attn, decay_decode_step) against its
definition in 64 bits.

Tolerances, elementwise, with A the sum of the magnitudes of an output's terms (the definition on
absolute values).  Inputs are what the kernel reads, so only its own roundings count:
* bf16 inputs: scores and states enter products as two bf16 terms, 2^-16 of a term at most each, and the
  powers g^n = 2^(n log2 g) have a relative error of at most about 4 |n ln g| 2^-24, at most 2^-17 of any term that
  is not below 2^-45 of its undecayed self: 2^-15 A in all, and half a step of the output, 2^-8 |y|.
* fp32 inputs, and states of either: every term is rounded at most three times and passes at most
  d + N additions: (d + N + 64) 2^-24 A, which leaves 64 for powers and products, and 2^-24 |y|.
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32


def _K():
    import kernels
    return kernels


def definition(q, k, v, g, scale, state=None, lengths=None):
    """y and the last state, dense, in the inputs' precision (64 bits), on the inputs' device."""
    b, h, n, d = q.shape
    last = torch.full((b,), n, device=q.device) if lengths is None else lengths.to(q.device).long().clamp(0, n)
    t = torch.arange(n, device=q.device)
    there = (t < last.view(-1, 1)).view(b, 1, n, 1)
    q, k, v = (torch.where(there, x, torch.zeros_like(x)) for x in (q, k, v))
    gap = t[:, None] - t[None, :]
    lg = g.double().clamp(min=-1e30).view(1, h, 1, 1)
    w = torch.exp(lg * gap.clamp(min=0)) * (gap >= 0)
    y = torch.matmul(torch.matmul(q, k.transpose(-1, -2).contiguous()) * w, v)
    m = last.view(b, 1, 1, 1)
    to_end = torch.exp(lg * (m - 1 - t.view(1, 1, n, 1)).clamp(min=0)) * there
    st = torch.matmul((k * to_end).transpose(-1, -2).contiguous(), v)
    if state is not None:
        y = y + torch.matmul(q, state) * torch.exp(lg * (t + 1).view(1, 1, n, 1))
        st = st + state * torch.exp(lg * m)
    return y * scale, st


def close(y, want, mag, dtype, terms, what=""):
    assert y.shape == want.shape, what
    unit = 2.0 ** -8 if y.dtype == BF else 2.0 ** -24
    rel = 2.0 ** -15 if dtype == BF else (terms + 64) * 2.0 ** -24
    bound = unit * want.abs() + rel * mag + 1e-30
    worst = float(((y.double() - want).abs() / bound).max()) if y.numel() else 0.0
    assert worst <= 1.0, f"{what}: {worst} of its bound"


def make(B, H, N, d, dv, dtype, seed, lengths=False, state=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    x = dict(q=r(B, H, N, d).to(dtype), k=r(B, H, N, d).to(dtype), v=r(B, H, N, dv).to(dtype), dy=r(B, H, N, dv).to(dtype))
    decays = torch.tensor([-0.05, 0.0, -3.0, float("-inf"), -1e-4, -0.3], device="cuda")
    x["g"] = decays[(torch.arange(H, device="cuda") + seed) % 6].contiguous()
    x["state"] = r(B, H, d, dv) * 3 if state else None
    x["dstate"] = r(B, H, d, dv) if state else None
    x["lengths"] = torch.randint(0, N + 1, (B,), generator=g, device="cuda", dtype=torch.int32) if lengths else None
    return x


SHAPES = [(1, 1, 1, 16, 16), (2, 3, 63, 16, 64), (1, 2, 64, 64, 64), (1, 6, 65, 64, 32), (2, 2, 130, 32, 128),
          (1, 3, 200, 128, 128), (1, 2, 300, 24, 40), (1, 1, 129, 7, 5), (1, 2, 700, 64, 64), (2, 6, 1100, 17, 128),
          (1, 1, 2000, 128, 24), (1, 1, 5, 1, 1)]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("extra", ["plain", "states", "ragged"])
@pytest.mark.parametrize("B,H,N,d,dv", SHAPES)
def test_forward(B, H, N, d, dv, extra, dtype):
    x = make(B, H, N, d, dv, dtype, N + d, lengths=extra == "ragged", state=extra != "plain")
    if x["lengths"] is not None:      # rows behind a sequence hold anything
        behind = torch.arange(N, device="cuda").view(1, 1, N, 1) >= x["lengths"].view(B, 1, 1, 1)
        clean = {n: x[n].clone() for n in ("q", "k", "v")}
        for n, bad in (("q", float("nan")), ("k", float("inf")), ("v", float("nan"))):
            x[n] = x[n].masked_fill(behind, bad)
    else:
        clean = x
    y, st = _K().decay_linear_attn(x["q"], x["k"], x["v"], x["g"], state_in=x["state"], return_state=True,
                                   lengths=x["lengths"])
    assert y.dtype == dtype and st.dtype == F32
    args = [clean[n].double() for n in ("q", "k", "v")]
    s0 = None if x["state"] is None else x["state"].double()
    scale = 1 / math.sqrt(d)
    want, wst = definition(*args, x["g"], scale, s0, x["lengths"])
    mag, mst = definition(*(a.abs() for a in args), x["g"], scale, None if s0 is None else s0.abs(), x["lengths"])
    close(y, want, mag, dtype, d + N, "y")
    close(st, wst, mst, F32, N, "state")
    if x["lengths"] is not None:
        assert not y.masked_select(behind).any()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("extra", ["plain", "states", "ragged"])
@pytest.mark.parametrize("B,H,N,d,dv", SHAPES)
def test_gradients(B, H, N, d, dv, extra, dtype):
    x = make(B, H, N, d, dv, dtype, N + d + 1, lengths=extra == "ragged", state=extra != "plain")
    names = ["q", "k", "v"] + (["state"] if extra != "plain" else [])
    leaves = [x[n].clone().requires_grad_() for n in names]
    st_in = leaves[3] if extra != "plain" else None
    y, st = _K().decay_linear_attn(*leaves[:3], x["g"], state_in=st_in, return_state=True, lengths=x["lengths"])
    outs, cot = ([y, st], [x["dy"], x["dstate"]]) if extra != "plain" else ([y], [x["dy"]])
    got = torch.autograd.grad(outs, leaves, cot)
    scale = 1 / math.sqrt(d)

    def formula(f):
        w = [f(x[n].double()).requires_grad_() for n in names]
        yy, ss = definition(*w[:3], x["g"], scale, w[3] if extra != "plain" else None, x["lengths"])
        o, c = ([yy, ss], [f(t.double()) for t in cot]) if extra != "plain" else ([yy], [f(x["dy"].double())])
        return torch.autograd.grad(o, w, c)

    for n, a, want, mag in zip(names, got, formula(lambda t: t.clone()), formula(torch.abs)):
        assert a.dtype == x[n].dtype
        close(a, want, mag, F32 if n == "state" else dtype, d + dv + N, "d" + n)


@pytest.mark.parametrize("N,d,dv", [(1, 16, 16), (150, 40, 64), (640, 64, 32)])
def test_gradients_by_differences(N, d, dv):
    """y and the state are linear in q, in v and in the first state, and in k: the difference of two calls at
    x + u and x - u is twice the gradient's product with u, up to the calls' own roundings.  fp32."""
    K = _K()
    x = make(1, 3, N, d, dv, F32, N, state=True)
    names = ["q", "k", "v", "state"]

    def loss(t):
        y, st = K.decay_linear_attn(t["q"], t["k"], t["v"], x["g"], state_in=t["state"], return_state=True)
        return float((y.double() * x["dy"]).sum() + (st.double() * x["dstate"]).sum()), float(
            (y.double() * x["dy"]).abs().sum() + (st.double() * x["dstate"]).abs().sum())

    leaves = [x[n].clone().requires_grad_() for n in names]
    y, st = K.decay_linear_attn(*leaves[:3], x["g"], state_in=leaves[3], return_state=True)
    grads = torch.autograd.grad([y, st], leaves, [x["dy"], x["dstate"]])
    for n, gr in zip(names, grads):
        u = torch.randn_like(x[n])
        (up, m1), (down, m2) = loss({**x, n: x[n] + u}), loss({**x, n: x[n] - u})
        # sums of magnitudes bound what 2^-24 per addition can do in either call; x +- u is itself rounded
        bound = (d + dv + N + 64) * 2.0 ** -24 * (m1 + m2 + float((gr.double() * u).abs().sum())) * 4
        assert abs((up - down) / 2 - float((gr.double() * u).sum())) <= bound, n


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("B,H,d,dv", [(1, 1, 1, 1), (2, 16, 64, 64), (3, 5, 17, 33), (2, 6, 128, 128), (1, 2, 100, 6), (70, 16, 16, 24)])
def test_step(B, H, d, dv, dtype):
    x = make(B, H, 1, d, dv, dtype, B + d, state=True)
    st = x["state"].clone()
    y = _K().decay_decode_step(x["q"], x["k"], x["v"], x["g"], st)
    args = [x[n].double() for n in ("q", "k", "v")]
    # one token after the state: y is of the new state, which is the definition's for one token
    want, wst = definition(*args, x["g"], 1 / math.sqrt(d), x["state"].double())
    mag, mst = definition(*(a.abs() for a in args), x["g"], 1 / math.sqrt(d), x["state"].double().abs())
    assert y.shape == x["v"].shape and y.dtype == dtype
    close(y, want, mag, F32, d, "y")
    close(st, wst, mst, F32, 0, "state")
    st3 = x["state"].clone()
    y3 = _K().decay_decode_step(x["q"][:, :, 0], x["k"][:, :, 0], x["v"][:, :, 0], x["g"], st3)
    assert torch.equal(y3, y[:, :, 0]) and torch.equal(st3, st)


def test_prompt_in_pieces_then_tokens():
    """A ragged batch of prompts in two pieces, then token by token, equals one call on all of it."""
    K = _K()
    B, H, d, dv = 3, 4, 64, 64
    x = make(B, H, 700, d, dv, BF, 5)
    cut = torch.tensor([0, 130, 200], dtype=torch.int32, device="cuda")
    rest = torch.tensor([300, 64, 496], dtype=torch.int32, device="cuda")
    steps = 3
    _, st = K.decay_linear_attn(*(x[n][:, :, :200] for n in "qkv"), x["g"], return_state=True, lengths=cut)
    second = [torch.stack([x[n][i, :, c:c + 496] if c + 496 <= 700 else torch.nn.functional.pad(x[n][i, :, c:], (0, 0, 0, c + 496 - 700))
                           for i, c in enumerate(cut.tolist())]) for n in "qkv"]
    y2, st = K.decay_linear_attn(*second, x["g"], return_state=True, state_in=st, lengths=rest)
    total = (cut + rest).tolist()
    ys = []
    for i in range(steps):
        tok = [torch.stack([x[n][j, :, m + i] for j, m in enumerate(total)]) for n in "qkv"]
        ys.append(K.decay_decode_step(*tok, x["g"], st))
    for j, (c, m) in enumerate(zip(cut.tolist(), total)):
        a = [x[n][j:j + 1, :, :m + steps].double() for n in "qkv"]
        want, wst = definition(*a, x["g"], 1 / math.sqrt(d))
        mag, mst = definition(*(t.abs() for t in a), x["g"], 1 / math.sqrt(d))
        close(y2[j:j + 1, :, :m - c], want[:, :, c:m], mag[:, :, c:m], BF, 0, "second piece")
        close(torch.stack([y[j] for y in ys], 1).unsqueeze(0), want[:, :, m:], mag[:, :, m:], BF, 0, "tokens")
        close(st[j:j + 1], wst, mst, F32, m + steps, "state")


@pytest.mark.parametrize("g", [0.01, 0.5])
def test_growth(g):
    """Logarithms above 0: the same formula, while its numbers stay finite.  Powers of up to 2^92 have arguments that are
    rounded once more, by 92 2^-24 of a power: 2^-17, in the state as in the outputs."""
    x = make(1, 2, 128, 32, 32, F32, 2)
    lg = torch.full((2,), g, device="cuda")
    y, st = _K().decay_linear_attn(x["q"], x["k"], x["v"], lg, return_state=True)
    want, wst = definition(*(x[n].double() for n in "qkv"), lg, 1 / math.sqrt(32))
    mag, mst = definition(*(x[n].double().abs() for n in "qkv"), lg, 1 / math.sqrt(32))
    assert float(((y - want).abs() / mag).max()) <= 2.0 ** -15 and float(((st - wst).abs() / mst).max()) <= 2.0 ** -15


def test_backward_without_the_forward_states():
    """la_decay_bwd computes the segments' states itself when the forward call's workspace is not given: same gradients,
    to the bit."""
    K = _K()
    x = make(1, 3, 900, 64, 64, BF, 3, state=True, lengths=True)
    leaves = [x[n].clone().requires_grad_() for n in ("q", "k", "v", "state")]
    y = K.decay_linear_attn(*leaves[:3], x["g"], state_in=leaves[3], lengths=x["lengths"])
    node = y.grad_fn
    assert node.segments is not None
    want = torch.autograd.grad(y, leaves, x["dy"], retain_graph=True)
    node.segments = None
    got = torch.autograd.grad(y, leaves, x["dy"])
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_step_is_seen_by_autograd():
    """A state that a differentiable call has saved and a step then changes: its gradient raises instead of being wrong."""
    K = _K()
    x = make(1, 2, 10, 16, 16, F32, 3, state=True)
    q = x["q"].clone().requires_grad_()
    y = K.decay_linear_attn(q, x["k"], x["v"], x["g"], state_in=x["state"])
    K.decay_decode_step(x["q"][:, :, 0], x["k"][:, :, 0], x["v"][:, :, 0], x["g"], x["state"])
    with pytest.raises(RuntimeError):
        torch.autograd.grad(y, q, x["dy"])


def test_no_decay_is_the_identity_map():
    K = _K()
    x = make(2, 3, 500, 32, 64, BF, 1)
    y = K.decay_linear_attn(x["q"], x["k"], x["v"], torch.zeros(3, device="cuda"), out_dtype=F32)
    z = K.identity_linear_attn(x["q"], x["k"], x["v"], out_dtype=F32)
    mag, _ = definition(*(x[n].double().abs() for n in "qkv"), torch.zeros(3, device="cuda"), 1 / math.sqrt(32))
    assert float(((y - z).abs() / mag).max()) <= 2.0 ** -14     # 2^-15 each


@pytest.mark.parametrize("dtype", [BF, F32])
def test_strides_and_alignment(dtype):
    """Heads inside a token's row, a start off 16 bytes, strides that no 16-byte load fits, expanded heads."""
    K = _K()
    B, N, H, d = 2, 200, 3, 64
    row = torch.randn(B, N, 3, H, d, device="cuda").to(dtype)
    q, k, v = row.permute(2, 0, 3, 1, 4).unbind(0)
    g = torch.tensor([-0.1, -0.01, 0.0], device="cuda")
    want = K.decay_linear_attn(q.contiguous(), k.contiguous(), v.contiguous(), g)
    assert torch.equal(K.decay_linear_attn(q, k, v, g), want)
    odd = torch.randn(B, H, N, d + 1, device="cuda").to(dtype)
    for w in (odd[..., 1:], odd[..., :d], odd.flip(2)[..., 1:], odd.transpose(2, 3)[:, :, :d, :].contiguous().transpose(2, 3)):
        assert torch.equal(K.decay_linear_attn(w, k, v, g), K.decay_linear_attn(w.clone(memory_format=torch.contiguous_format), k, v, g))
    one = torch.randn(B, 1, N, d, device="cuda").to(dtype).requires_grad_()
    qq = q.detach().clone().requires_grad_()
    y = K.decay_linear_attn(qq, one.expand(B, H, N, d), v, g)
    dy = torch.randn(B, N, H, d, device="cuda").to(dtype).transpose(1, 2)      # a cotangent with its own strides
    dq, dk = torch.autograd.grad(y, (qq, one), dy)
    full = one.detach().expand(B, H, N, d).clone().requires_grad_()
    yf = K.decay_linear_attn(qq, full, v, g)
    dqf, dkf = torch.autograd.grad(yf, (qq, full), dy.contiguous())
    assert torch.equal(dq, dqf)
    want = dkf.double().sum(1, keepdim=True)
    assert bool(((dk.double() - want).abs() <= 2.0 ** -7 * dkf.double().abs().sum(1, keepdim=True)).all())


@pytest.mark.parametrize("dtype", [BF, F32])
def test_expanded_tokens(dtype):
    """One row for all tokens (stride 0), at a length that no chunk divides: rows behind it are no tokens."""
    K = _K()
    x = make(1, 3, 70, 64, 64, dtype, 8)
    for n in "qkv":
        one = {m: x[m].clone() for m in "qkv"}
        one[n] = x[n][:, :, :1].expand(-1, -1, 70, -1)
        y, st = K.decay_linear_attn(*(one[m] for m in "qkv"), x["g"], return_state=True)
        one[n] = one[n].contiguous()
        want, wst = K.decay_linear_attn(*(one[m] for m in "qkv"), x["g"], return_state=True)
        assert torch.equal(y, want) and torch.equal(st, wst)


def test_second_derivatives_are_refused():
    K = _K()
    x = make(1, 2, 20, 16, 16, F32, 3)
    q = x["q"].requires_grad_()
    y = K.decay_linear_attn(q, x["k"], x["v"], x["g"])
    dq, = torch.autograd.grad(y, q, x["dy"], create_graph=True)
    assert torch.equal(dq, torch.autograd.grad(K.decay_linear_attn(q, x["k"], x["v"], x["g"]), q, x["dy"])[0])
    with pytest.raises(RuntimeError):
        torch.autograd.grad(dq.sum(), q)


def test_types_through_fp32():
    K = _K()
    x = make(1, 2, 100, 16, 16, F32, 3)
    for dt in (torch.float16, torch.float64):
        a = [x[n].to(dt).requires_grad_() for n in "qkv"]
        y = K.decay_linear_attn(*a, x["g"])
        assert y.dtype == dt
        want = K.decay_linear_attn(*(t.detach().float() for t in a), x["g"])
        assert torch.equal(y, want.to(dt))
        assert all(t.dtype == dt for t in torch.autograd.grad(y, a, torch.ones_like(y)))
    assert K.decay_linear_attn(x["q"].bfloat16(), x["k"].bfloat16(), x["v"].bfloat16(), x["g"], out_dtype=F32).dtype == F32


def test_empty():
    K = _K()
    g = torch.zeros(2, device="cuda")
    q = torch.zeros(1, 2, 0, 16, device="cuda", requires_grad=True)
    st = torch.randn(1, 2, 16, 16, device="cuda", requires_grad=True)
    y, s = K.decay_linear_attn(q, q, q, g, state_in=st, return_state=True)
    assert y.shape == (1, 2, 0, 16) and torch.equal(s, st)
    dst = torch.randn_like(st)
    assert torch.equal(torch.autograd.grad(s, st, dst)[0], dst)
    z = torch.zeros(0, 2, 5, 16, device="cuda")
    assert K.decay_linear_attn(z, z, z, g).shape == z.shape
    # sequences of no tokens keep their state, and give no gradients
    x = make(2, 2, 70, 16, 16, BF, 9, state=True)
    none = torch.zeros(2, dtype=torch.int32, device="cuda")
    q = x["q"].clone().requires_grad_()
    y, s = K.decay_linear_attn(q, x["k"], x["v"], g, state_in=x["state"], return_state=True, lengths=none)
    assert not y.any() and torch.equal(s, x["state"])
    assert not torch.autograd.grad(y, q, x["dy"])[0].any()


def test_refusals():
    K = _K()
    x = make(1, 2, 10, 16, 16, BF, 2, state=True)
    q, k, v, g = x["q"], x["k"], x["v"], x["g"]
    bad = [dict(q=q.cpu()), dict(k=k[:, :, :5]), dict(v=v.float()), dict(log_decay=g[:1]), dict(log_decay=g.double()),
           dict(log_decay=g.clone().requires_grad_()), dict(lengths=torch.ones(1, device="cuda")),
           dict(lengths=torch.ones(2, dtype=torch.int32, device="cuda")), dict(state_in=x["state"][..., :8]),
           dict(state_in=x["state"].bfloat16()), dict(scale=-1.0), dict(scale=float("nan")), dict(log_decay=g.cpu())]
    for b in bad:
        with pytest.raises(RuntimeError):
            K.decay_linear_attn(**{**dict(q=q, k=k, v=v, log_decay=g), **b})
    wide = torch.zeros(1, 2, 4, 129, device="cuda", dtype=BF)
    with pytest.raises(RuntimeError):
        K.decay_linear_attn(wide, wide, wide, g)
    t = [x[n][:, :, 0] for n in "qkv"]
    for b in (dict(state=x["state"].transpose(2, 3)), dict(state=x["state"].double()), dict(q=t[0][:, :, None]),
              dict(q=x["q"], k=x["k"], v=x["v"]), dict(state=x["state"].clone().requires_grad_()), dict(scale=0.0)):
        with pytest.raises(RuntimeError):
            K.decay_decode_step(**{**dict(q=t[0], k=t[1], v=t[2], log_decay=g, state=x["state"]), **b})


def _captured(fn):
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        fn()
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = fn()
    return g, out


def test_graphs():
    """Forward, gradients and a step captured; every replay gives the eager call's bits."""
    K = _K()
    x = make(1, 4, 1000, 64, 64, BF, 4, state=True, lengths=True)
    tok = [x[n][:, :, 0] for n in "qkv"]
    step_state = x["state"].clone()

    def calls():
        leaves = [x[n].detach().requires_grad_() for n in ("q", "k", "v", "state")]
        y, st = K.decay_linear_attn(*leaves[:3], x["g"], state_in=leaves[3], return_state=True, lengths=x["lengths"])
        grads = torch.autograd.grad([y, st], leaves, [x["dy"], x["dstate"]])
        return (y.detach(), st.detach(), *grads, K.decay_decode_step(*tok, x["g"], step_state))

    want = [t.clone() for t in calls()]
    g, outs = _captured(calls)
    for _ in range(3):
        K.sliding_window_attn(x["q"], x["k"], x["v"], window_size=33)
        step_state.copy_(x["state"])
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        for a, w in zip(outs, want):
            assert torch.equal(a, w)


def test_other_stream():
    K = _K()
    x = make(1, 2, 600, 64, 64, BF, 6)
    want = K.decay_linear_attn(x["q"], x["k"], x["v"], x["g"])
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        y = K.decay_linear_attn(x["q"], x["k"], x["v"], x["g"])
    s.synchronize()
    assert torch.equal(y, want)


def test_offsets_beyond_32_bits():
    """One sequence of more than 2^31 elements: with g = e^-0.5 rows near an end see nothing of the other end (e^-128),
    so that both ends are the definition's on 512 rows; outputs and gradients of the rows that lie in their inner half."""
    N, d, cut = (1 << 24) + 77, 128, 512
    g = torch.Generator(device="cuda").manual_seed(11)
    q, k, v, dy = (torch.randn(1, 1, N, d, generator=g, device="cuda", dtype=BF) for _ in range(4))
    lg = torch.tensor([-0.5], device="cuda")
    leaves = [x.requires_grad_() for x in (q, k, v)]
    y, st = _K().decay_linear_attn(*leaves, lg, return_state=True)
    grads = [x.detach() for x in torch.autograd.grad(y, leaves, dy)]
    y, st = y.detach(), st.detach()
    for rows, half in ((slice(N - cut, N), slice(cut // 2, cut)), (slice(0, cut), slice(0, cut // 2))):
        def formula(f):
            w = [f(x.detach()[:, :, rows].double()).requires_grad_() for x in leaves]
            yy, ss = definition(*w, lg, 1 / math.sqrt(d))
            return [yy.detach(), ss.detach()] + list(torch.autograd.grad(yy, w, f(dy[:, :, rows].double())))
        want, mag = formula(lambda t: t.clone()), formula(torch.abs)
        at_end = rows.stop == N
        names = ["y", "dq"] if at_end else ["y", "dq", "dk", "dv"]      # dk and dv look ahead
        for n, a, w, m in zip(["y", "dq", "dk", "dv"], [y] + grads, want[:1] + want[2:], mag[:1] + mag[2:]):
            if n in names:
                close(a[:, :, rows][:, :, half], w[:, :, half], m[:, :, half], BF, d, n)
        if at_end:
            close(st, want[1], mag[1], F32, cut, "state")


@pytest.mark.parametrize("dtype,d,dv", [(BF, 100, 60), (BF, 6, 34), (BF, 62, 128), (F32, 63, 5), (F32, 101, 127), (BF, 33, 64)])
def test_rows_of_words_and_of_elements(dtype, d, dv):
    """Widths that are no whole 16-byte pieces, and a start in the middle of one: with zeros behind each row up to whole
    pieces the terms are the same, and so are the bits of outputs, states and gradients."""
    K, P = _K(), torch.nn.functional.pad
    B, H, N = 2, 3, 333
    x = make(B, H, N, d, dv, dtype, d, lengths=True, state=True)
    pd, pv = -d % 8, -dv % 8
    wide = {n: P(x[n], (0, pd if n in "qk" else pv)) for n in ("q", "k", "v", "dy")}
    wide.update({n: P(x[n], (0, pv, 0, pd)) for n in ("state", "dstate")})

    def call(t):
        leaves = [t[n].detach().requires_grad_() for n in ("q", "k", "v", "state")]
        y, st = K.decay_linear_attn(*leaves[:3], x["g"], scale=0.3, state_in=leaves[3], return_state=True, lengths=x["lengths"])
        return [y, st] + list(torch.autograd.grad([y, st], leaves, [t["dy"], t["dstate"]]))

    want = call(wide)
    shifted = dict(x)      # rows of two elements more, from the second on
    for n in ("q", "k", "v", "dy"):
        shifted[n] = P(x[n], (2, 0))[..., 2:]
    for t in (x, shifted):
        for n, a, w in zip(("y", "state", "dq", "dk", "dv", "dstate"), call(t), want):
            assert torch.equal(a.detach(), w.detach()[tuple(slice(0, s) for s in a.shape)]), n
