"""The 8-bit cache (kernels.sliding_cache, sliding_cache_append) and one-token attention over it
(sliding_decode_step), against a token-by-token model of the cache and softmax in 64 bits.

Codes and scales are equal to the model's.  Attention is held to the definition on the values that the codes
stand for, elementwise, with A = sum p |v| / sum p and S the largest sum of magnitudes of a score's terms:
* a score is off by at most (d + 8) 2^-24 S, and so a weight relative to another by twice that;
* weights, products and sums over n tokens: (n + 64) 2^-24 A; bf16 inputs take P as two bf16 terms, 2^-16 A,
  doubled for the sum it is divided by;
* the output's rounding, half a step: 2^-8 |y| in bf16, 2^-24 |y| in fp32.
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32
E4 = torch.float8_e4m3fn


def _K():
    import kernels
    return kernels


def scale_of(x):
    """The smallest power of two, 2^-100 at the least, with |x| <= 448 of it, over finite entries of x (.., n)."""
    a = torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x)).amax(-1).double()
    m, e = torch.frexp(a)      # a = m 2^e, m in [1/2, 1); 448 = 7/8 2^9
    e = torch.where(a > 0, e - 9 + (m > 0.875), torch.full_like(e, -100)).clamp(min=-100)
    return (e.long() + 1023 << 52).view(torch.float64)


def encode(x):
    x = torch.where(torch.isinf(x), torch.full_like(x, float("nan")), x)
    return x.float().to(E4).double()


class Model:
    """The cache, a token at a time, on the CPU in 64 bits: codes by place and scales by block.  A piece of several
    tokens of a block is rounded once, under the piece's scale."""

    def __init__(self, b, hk, blocks, d, dv):
        self.k, self.v = torch.zeros(b, hk, blocks, 64, d).double(), torch.zeros(b, hk, blocks, 64, dv).double()
        self.ks, self.vs = torch.zeros(b, hk, blocks).double(), torch.zeros(b, hk, blocks).double()
        self.blocks = blocks

    def append(self, k, v, start, lengths):
        for i, (p, n) in enumerate(zip(start, lengths)):
            while n > 0:
                m = min(n, 64 - p % 64)
                for codes, scales, x in ((self.k, self.ks, k), (self.v, self.vs, v)):
                    rows = x[i, :, p - start[i]:p - start[i] + m].double().cpu()
                    j, at = p // 64 % self.blocks, p % 64
                    s = scale_of(rows.flatten(1))
                    if at == 0:
                        codes[i, :, j] = 0
                    else:
                        s = torch.maximum(s, scales[i, :, j])
                        codes[i, :, j, :at] = encode(codes[i, :, j, :at] * (scales[i, :, j] / s)[:, None, None])
                        codes[i, :, j, at:] = 0
                    codes[i, :, j, at:at + m] = encode(rows / s[:, None, None])
                    scales[i, :, j] = s
                p, n = p + m, n - m

    def check(self, cache):
        got = cache.k.float().double().cpu()
        assert torch.equal(torch.nan_to_num(got[..., :cache.d], nan=999.0), torch.nan_to_num(self.k, nan=999.0)), "keys"
        got = cache.v.float().double().cpu().transpose(3, 4)
        assert torch.equal(torch.nan_to_num(got[..., :cache.dv], nan=999.0), torch.nan_to_num(self.v, nan=999.0)), "values"
        assert not cache.k[..., cache.d:].float().any() and not cache.v[..., cache.dv:, :].float().any()
        assert torch.equal(cache.k_scale.double().cpu(), self.ks) and torch.equal(cache.v_scale.double().cpu(), self.vs)


def attention(q, cache, length, window, scale):
    """Softmax attention in 64 bits over a sequence's last positions, from the values the cache stands for; and A, S."""
    k, v = (x.double().cpu() for x in cache.values())
    b, hk, cap, _ = k.shape
    h = q.shape[1]
    q = q.double().cpu()
    y, A, S = torch.zeros(b, h, cache.dv).double(), torch.zeros(b, h, cache.dv).double(), torch.zeros(b, h, 1).double()
    for i in range(b):
        n = int(length[i])
        if n <= 0:
            continue
        first = max(0, ((n - 1) // 64 + 1) * 64 - cap)
        if window:
            first = max(first, n - window)
        at = torch.arange(first, n) % cap
        for j in range(h):
            kk, vv = k[i, j // (h // hk), at], v[i, j // (h // hk), at]
            p = torch.softmax(kk @ q[i, j] * scale, 0)
            y[i, j], A[i, j], S[i, j] = p @ vv, p @ vv.abs(), (kk.abs() @ q[i, j].abs() * scale).max()
    return y, A, S


def close(y, want, A, S, dtype, d, n):
    unit = 2.0 ** -8 if y.dtype == BF else 2.0 ** -24
    rel = (n + 64) * 2.0 ** -24 + (2.0 ** -15 if dtype == BF else 0.0) + 2 * (d + 8) * 2.0 ** -24 * S
    worst = float(((y.double().cpu() - want).abs() / (unit * want.abs() + rel * A + 1e-30)).max())
    assert worst <= 1.0, f"{worst} of its bound"


def ints(*x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("hk,t,d,dv,blocks,start,lengths", [
    (1, 1, 16, 16, 1, (0,), (1,)), (2, 64, 64, 64, 2, (0,), (64,)), (3, 65, 64, 32, 2, (0,), (65,)),
    (2, 300, 128, 128, 6, (0, 10, 64), (300, 0, 299)), (2, 100, 24, 40, 4, (63, 130), (100, 1)),
    (1, 500, 7, 5, 3, (0, 37), (500, 400)), (2, 130, 100, 1, 64, (1000, 64), (130, 77)),
    (16, 33, 32, 80, 2, (90, 95, 96), (33, 32, 31))])
def test_append(hk, t, d, dv, blocks, start, lengths, dtype):
    """Pieces at any start, ragged, longer than the ring; rows behind a sequence hold NaN."""
    K = _K()
    b = len(start)
    g = torch.Generator(device="cuda").manual_seed(t + d)
    cache, model = K.sliding_cache(b, hk, 64 * blocks, d, dv), Model(b, hk, blocks, d, dv)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda") * torch.exp(3 * torch.randn(s[0], s[1], 1, 1, generator=g, device="cuda"))  # noqa: E731
    if any(start):      # what lies before: from each sequence's block's first place
        k0, v0 = r(b, hk, 64, d).to(dtype), r(b, hk, 64, dv).to(dtype)
        s0, n0 = [p // 64 * 64 for p in start], [p % 64 for p in start]
        K.sliding_cache_append(cache, k0, v0, start=ints(*s0), lengths=ints(*n0))
        model.append(k0, v0, s0, n0)
        model.check(cache)
    k, v = r(b, hk, t, d).to(dtype), r(b, hk, t, dv).to(dtype)
    model.append(k, v, list(start), list(lengths))
    behind = torch.arange(t, device="cuda").view(1, 1, t, 1) >= ints(*lengths).view(b, 1, 1, 1)
    k, v = k.masked_fill(behind, float("nan")), v.masked_fill(behind, float("inf"))
    K.sliding_cache_append(cache, k, v, start=ints(*start), lengths=ints(*lengths))
    model.check(cache)


def test_codes_over_the_whole_range():
    """Every magnitude: zeros, what rounds to zero and to the smallest codes, ties, the largest, 32-bit extremes,
    infinities and NaN; a later token that raises the scale by 2^20."""
    K = _K()
    e = torch.arange(-130, 127).float()
    x = torch.cat([torch.tensor([1.0, 1.0625, 1.1875, 1.25, 1.75, 1.8125, 1.875, 1.9375, 1.9999])[:, None] * torch.exp2(e)], 0).flatten()
    x = torch.cat([x, -x])
    x = torch.nn.functional.pad(x, (0, -x.numel() % 64)).view(1, 1, -1, 64).cuda()
    t = x.shape[2]
    for y in (x, x.flip(2), x[..., torch.randperm(64, generator=torch.Generator().manual_seed(1)).cuda()]):
        cache, model = K.sliding_cache(1, 1, t, 64), Model(1, 1, -(-t // 64), 64, 64)
        K.sliding_cache_append(cache, y, y.flip(3))
        model.append(y, y.flip(3), [0], [t])
        model.check(cache)
    cache, model = K.sliding_cache(1, 1, 64, 64), Model(1, 1, 1, 64, 64)
    small = torch.randn(1, 1, 5, 64, device="cuda")
    odd = torch.randn(1, 1, 2, 64, device="cuda") * 2 ** 12
    odd[0, 0, 0, 3], odd[0, 0, 0, 4], odd[0, 0, 1, 5], odd[0, 0, 1, 6] = float("inf"), float("nan"), -float("inf"), 0.0
    p = 0
    for y in (torch.zeros(1, 1, 2, 64, device="cuda"), small, small * 2.0 ** -30, odd, small * 2 ** 20):
        K.sliding_cache_append(cache, y, y, start=ints(p))
        model.append(y, y, [p], [y.shape[2]])
        model.check(cache)
        p += y.shape[2]


CASES = [  # b, h, hk, d, dv, blocks, window, lengths
    (1, 1, 1, 16, 16, 1, None, (1,)), (2, 16, 16, 64, 64, 2, 64, (300, 64)), (3, 4, 2, 128, 128, 8, None, (512, 1, 385)),
    (2, 8, 1, 64, 32, 40, None, (2560, 1300)), (2, 40, 2, 24, 40, 5, 100, (301, 99)), (4, 6, 3, 80, 128, 3, 1, (200, 65, 64, 0)),
    (2, 2, 1, 32, 7, 4, 193, (1000, 257)), (1, 5, 5, 5, 96, 3, None, (1000,)), (2, 33, 1, 128, 64, 33, 2000, (2112, 2047))]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("b,h,hk,d,dv,blocks,window,lengths", CASES)
def test_step(b, h, hk, d, dv, blocks, window, lengths, dtype):
    """After the prompts are appended, one token: the cache is the model's, the output the definition's.  Stale codes in
    places that the window does not reach are NaN."""
    K = _K()
    g = torch.Generator(device="cuda").manual_seed(h + d)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda").to(dtype)  # noqa: E731
    cache, model = K.sliding_cache(b, hk, 64 * blocks, d, dv), Model(b, hk, blocks, d, dv)
    t = max(lengths)
    kp, vp = r(b, hk, t, d), r(b, hk, t, dv)
    if window:      # behind every window
        for i, n in enumerate(lengths):
            kp[i, :, :max(0, n - window)] = float("nan")
            vp[i, :, :max(0, n - window)] = float("nan")
    past = [max(0, n - 1) for n in lengths]
    K.sliding_cache_append(cache, kp, vp, lengths=ints(*past))
    model.append(kp, vp, [0] * b, past)
    q, k, v = r(b, h, d), r(b, hk, d), r(b, hk, dv)
    y = K.sliding_decode_step(q, k, v, cache, ints(*lengths), window_size=window)
    assert y.dtype == dtype and y.shape == (b, h, dv)
    model.append(k.unsqueeze(2), v.unsqueeze(2), past, [int(n > 0) for n in lengths])
    model.check(cache)
    want, A, S = attention(q, cache, lengths, window or 0, 1 / math.sqrt(d))
    close(y, want, A, S, dtype, d, t)
    for i, n in enumerate(lengths):
        assert n > 0 or not y[i].any()
    # again, with the token in a third dimension and another scale
    y = K.sliding_decode_step(q.unsqueeze(2), k.unsqueeze(2), v.unsqueeze(2), cache, ints(*lengths), window_size=window, scale=0.5)
    want, A, S = attention(q, cache, lengths, window or 0, 0.5)
    close(y.squeeze(2), want, A, S, dtype, d, t)


def test_large_scores():
    """Scores of thousands, of either sign: the running maximum holds across blocks, waves and splits."""
    K = _K()
    b, hk, d, n = 1, 2, 64, 5000
    g = torch.Generator(device="cuda").manual_seed(3)
    k, v = torch.randn(b, hk, n, d, generator=g, device="cuda") * 30, torch.randn(b, hk, n, d, generator=g, device="cuda")
    cache = K.sliding_cache(b, hk, n, d)
    K.sliding_cache_append(cache, k, v, lengths=ints(n - 1))
    for sign in (30.0, -30.0):
        q = torch.randn(b, 4, d, generator=g, device="cuda") * sign
        y = K.sliding_decode_step(q, k[:, :, -1], v[:, :, -1], cache, ints(n))
        want, A, S = attention(q, cache, [n], 0, 1 / math.sqrt(d))
        close(y, want, A, S, F32, d, n)


def test_rolling_decode_matches_the_window_kernel():
    """A prompt, then 200 tokens through a ring of little more than the window: every step equals
    sliding_window_attn on the values that were cached, at positions that cross blocks and laps of the ring."""
    K = _K()
    b, h, d, window, n0, steps = 2, 4, 64, 100, 150, 200
    g = torch.Generator(device="cuda").manual_seed(11)
    # whole numbers up to 15 are e4m3 values under any scale from 2^-4 to 1: the cache holds them exactly
    q, k, v = (torch.randint(-15, 16, (b, h, n0 + steps, d), generator=g, device="cuda").to(BF) for _ in range(3))
    cache = K.sliding_cache(b, h, window + 63, d)
    K.sliding_cache_append(cache, k[:, :, :n0], v[:, :, :n0])
    want = K.sliding_window_attn(q.float(), k.float(), v.float(), window_size=window, scale=0.02)
    mag = K.sliding_window_attn(q.float(), k.float(), v.float().abs(), window_size=window, scale=0.02)
    lengths = ints(n0, n0)
    for t in range(n0, n0 + steps):
        lengths += 1
        y = K.sliding_decode_step(q[:, :, t], k[:, :, t], v[:, :, t], cache, lengths, window_size=window, scale=0.02)
        # 2^-8 |y| for the output, 2^-15 A for P, and 2^-14 A for scores of up to 300 in either kernel's fp32
        assert bool(((y.float() - want[:, :, t]).abs() <= 2.0 ** -8 * want[:, :, t].abs() + 2.0 ** -13 * mag[:, :, t]).all()), t


def test_layer_decode():
    """The two branches of a layer together, prompt then tokens: decay state and cache side by side, in one captured
    graph that is replayed for every token."""
    K = _K()
    b, h, d, window, n0 = 2, 4, 64, 64, 129
    g = torch.Generator(device="cuda").manual_seed(12)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda").to(BF)  # noqa: E731
    q, k, v = r(b, h, n0 + 70, d), r(b, h, n0 + 70, d), r(b, h, n0 + 70, d)
    ld = torch.tensor([-0.5, -0.1, -0.01, 0.0], device="cuda")

    def prompt():
        cache = K.sliding_cache(b, h, window + 63, d)
        K.sliding_cache_append(cache, k[:, :, :n0], v[:, :, :n0])
        _, st = K.decay_linear_attn(q[:, :, :n0], k[:, :, :n0], v[:, :, :n0], ld, return_state=True)
        return cache, st, ints(n0, n0)

    def step(tok, cache, st, lengths):
        lengths += 1
        return K.decay_decode_step(*tok, ld, st) + K.sliding_decode_step(*tok, cache, lengths, window_size=window)

    cache, st, lengths = prompt()
    want = [step([x[:, :, t].contiguous() for x in (q, k, v)], cache, st, lengths) for t in range(n0, n0 + 70)]
    cache2, st2, lengths2 = prompt()
    tok = [x[:, :, n0].contiguous() for x in (q, k, v)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        scratch = [x.clone() for x in cache2[:4]]
        step(tok, K.SlidingCache(*scratch, d, d), st2.clone(), lengths2.clone())
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(tok, cache2, st2, lengths2)
    for i, t in enumerate(range(n0, n0 + 70)):
        for x, y in zip(tok, (q, k, v)):
            x.copy_(y[:, :, t])
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[i]), t
    assert torch.equal(st, st2) and all(torch.equal(a.view(torch.uint8), c.view(torch.uint8)) for a, c in zip(cache[:4], cache2[:4]))


def test_strides_and_types():
    K = _K()
    b, t, hk, d = 2, 200, 3, 64
    row = torch.randn(b, t, 2, hk, d, device="cuda").to(BF)
    k, v = row.permute(2, 0, 3, 1, 4).unbind(0)
    odd = torch.randn(b, hk, t, d + 1, device="cuda").to(BF)[..., 1:]
    for kk, vv in ((k, v), (odd, v), (k, odd), (k.double(), v.double()), (k.half(), odd.half())):
        one, two = K.sliding_cache(b, hk, t, d), K.sliding_cache(b, hk, t, d)
        K.sliding_cache_append(one, kk, vv)
        K.sliding_cache_append(two, kk.contiguous(), vv.contiguous())
        for a, c in zip(one[:4], two[:4]):
            assert torch.equal(a.view(torch.uint8), c.view(torch.uint8))
        q = torch.randn(b, d, 6, device="cuda").to(kk.dtype).transpose(1, 2)
        y = K.sliding_decode_step(q, kk[:, :, 7], vv[:, :, 7], one, ints(150, t))
        z = K.sliding_decode_step(q.contiguous(), kk[:, :, 7].contiguous(), vv[:, :, 7].contiguous(), two, ints(150, t))
        assert torch.equal(y, z) and y.dtype == kk.dtype


def test_refusals():
    K = _K()
    b, h, hk, d = 2, 4, 2, 64
    cache = K.sliding_cache(b, hk, 128, d)
    r = lambda *s: torch.randn(*s, device="cuda").to(BF)  # noqa: E731
    q, k, v, n = r(b, h, d), r(b, hk, d), r(b, hk, d), ints(3, 4)
    for bad in (dict(q=r(b, 3, d)), dict(q=q.float()), dict(k=r(b, h, d)), dict(v=r(b, hk, 32)), dict(lengths=n.long()), dict(lengths=n[:1]),
                dict(window_size=0), dict(window_size=66), dict(scale=-1.0), dict(q=q.unsqueeze(2)), dict(k=k.cpu()),
                dict(lengths=n.cpu()), dict(cache=cache._replace(k=cache.k.float())), dict(cache=cache._replace(d=32)),
                dict(cache=cache._replace(v=cache.v.transpose(3, 4))), dict(cache=cache._replace(k_scale=cache.k_scale[:, :, :1])),
                dict(q=q.clone().requires_grad_())):
        with pytest.raises(RuntimeError):
            K.sliding_decode_step(**{**dict(q=q, k=k, v=v, cache=cache, lengths=n), **bad})
    kp, vp = r(b, hk, 10, d), r(b, hk, 10, d)
    for bad in (dict(k=kp[:1]), dict(v=vp.float()), dict(k=kp[..., :32]), dict(v=vp[:, :, :5]), dict(start=n.long()), dict(lengths=n[:1]),
                dict(k=kp.cpu()), dict(cache=cache._replace(v=cache.v[:, :1]))):
        with pytest.raises(RuntimeError):
            K.sliding_cache_append(**{**dict(cache=cache, k=kp, v=vp), **bad})
    for bad in (dict(d=129), dict(d=0), dict(dv=200), dict(tokens=0)):
        with pytest.raises(RuntimeError):
            K.sliding_cache(**{**dict(b=1, heads=1, tokens=64, d=64), **bad})
    assert not cache.k.float().any() and not cache.k_scale.any()


def test_empty_batches():
    K = _K()
    cache = K.sliding_cache(0, 2, 64, 16)
    z = torch.zeros(0, 2, 16, device="cuda")
    assert K.sliding_decode_step(z, z, z, cache, ints()).shape == (0, 2, 16)
    K.sliding_cache_append(cache, z.unsqueeze(2), z.unsqueeze(2))
    cache = K.sliding_cache(2, 2, 64, 16)
    z = torch.zeros(2, 2, 0, 16, device="cuda")
    K.sliding_cache_append(cache, z, z)
    q = torch.randn(2, 2, 16, device="cuda")
    y = K.sliding_decode_step(q, q, q, cache, ints(0, -5))
    assert not y.any() and not cache.k.float().any() and not cache.k_scale.any()


def test_offsets_beyond_32_bits():
    """Positions around 2^25, where the codes lie 2^32 bytes from the first ones: the last blocks are the model's, the step
    the definition's on them."""
    K = _K()
    lo, n, d, w = (1 << 19) - 2, 329, 128, 190      # from block lo on: 328 tokens, then one
    g = torch.Generator(device="cuda").manual_seed(4)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda").to(BF)  # noqa: E731
    cache, model = K.sliding_cache(1, 1, 64 * (lo + 6), d), Model(1, 1, 6, d, d)
    k, v = r(1, 1, n - 1, d), r(1, 1, n - 1, d)
    K.sliding_cache_append(cache, k, v, start=ints(64 * lo))
    model.append(k, v, [0], [n - 1])
    q, k, v = r(1, 2, d), r(1, 1, d), r(1, 1, d)
    y = K.sliding_decode_step(q, k, v, cache, ints(64 * lo + n), window_size=w)
    model.append(k.unsqueeze(2), v.unsqueeze(2), [n - 1], [1])
    tail = K.SlidingCache(*(x[:, :, lo:].contiguous() for x in cache[:4]), d, d)
    assert not cache.k_scale[:, :, :lo].any() and not cache.v_scale[:, :, :lo].any()
    del cache
    model.check(tail)
    want, A, S = attention(q, tail, (n,), w, 1 / math.sqrt(d))
    close(y, want, A, S, BF, d, w)


@pytest.mark.parametrize("dtype,d,dv", [(BF, 100, 60), (BF, 6, 34), (BF, 62, 128), (F32, 63, 5), (F32, 101, 127), (BF, 33, 64)])
def test_rows_of_words_and_of_elements(dtype, d, dv):
    """Widths that are no whole 16-byte pieces, in rows that start in the middle of one."""
    K = _K()
    g = torch.Generator(device="cuda").manual_seed(d)
    b, hk, t, start, lengths = 2, 3, 200, (0, 64), (130, 200)
    rows = [torch.randn(b, hk, t, w + 2, generator=g, device="cuda").to(dtype) for w in (d, dv)]
    behind = torch.arange(t, device="cuda").view(1, 1, t, 1) >= ints(*lengths).view(b, 1, 1, 1)
    for shift in (0, 2):
        k, v = (x[..., shift:x.shape[3] - 2 + shift] for x in rows)
        if not shift:
            k, v = k.contiguous(), v.contiguous()
        cache, model = K.sliding_cache(b, hk, 320, d, dv), Model(b, hk, 5, d, dv)
        model.append(k, v, list(start), list(lengths))
        for x in (k, v):      # in place: a view stays one
            x.masked_fill_(behind, float("nan"))
        K.sliding_cache_append(cache, k, v, start=ints(*start), lengths=ints(*lengths))
        model.check(cache)
