"""Linear attention with a decay for each head, and one-token attention over an 8-bit cache, as measured.

``run`` computes each operator in its plain form: elementary torch operations in 32 bits, rounded once at
the end.  With ``own`` true it makes the calls of the ``kernels`` package instead.  ``exact`` is the same
function in 64 bits, written from the definition.

The kinds (b sequences, h heads, g_h = exp(log_decay_h) <= 1, s = 1 / sqrt(d)):

* ``forward`` -- ``decay_linear_attn``: y_t = s sum_{u <= t} g^(t - u) (q_t . k_u) v_u; with ``states`` also
  the state S = sum_u g^(N - 1 - u) k_u v_u^T, and an earlier state that these tokens follow; with ``ragged``
  prompts padded on the right to one length.
* ``train``   -- the same and its gradients by q, k, v (and by the first state with ``states``).
* ``step``    -- ``decay_decode_step``: S <- g S + k v^T in place, y = s q^T S; one token for each sequence.
* ``append``  -- ``sliding_cache_append``: keys and values into an 8-bit cache (blocks of 64 tokens, a
  power-of-two scale for each block and head).
* ``sliding`` -- ``sliding_decode_step``: one token into that cache, and its softmax attention over the
  cache's last ``window`` tokens (0: all of them); h query heads share hk cached ones.
"""

import math
import os
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
E4M3 = torch.float8_e4m3fn
BLOCK = 64           # tokens of a cache block
LEAST_SCALE = -100   # exponent of the smallest block scale


def _kernels():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "trainium-linear-attention_amd")
    if pkg not in sys.path:
        sys.path.insert(1, pkg)
    import kernels
    return kernels


def listed():
    return [
        # the smallest benchmark forward, 32-bit
        dict(name="forward_f32_b1h4n1024", kind="forward", b=1, h=4, n=1024, d=16, dv=64, dtype="f32", states=False,
             ragged=False),
        # an ordinary training-length forward
        dict(name="forward_b2h16n2048", kind="forward", b=2, h=16, n=2048, d=64, dv=64, dtype="bf16", states=False,
             ragged=False),
        # the next pieces of a few prompts of unlike lengths, wide heads, a length that no tile divides
        dict(name="forward_ragged_b4h8n3001", kind="forward", b=4, h=8, n=3001, d=128, dv=128, dtype="bf16", states=True,
             ragged=True),
        # a long prompt
        dict(name="forward_b1h16n65536", kind="forward", b=1, h=16, n=65536, d=64, dv=64, dtype="bf16", states=False,
             ragged=False),
        # a training step at an ordinary length
        dict(name="train_b2h16n2048", kind="train", b=2, h=16, n=2048, d=64, dv=64, dtype="bf16", states=False,
             ragged=False),
        # a training step at the headline length
        dict(name="train_b2h16n8192", kind="train", b=2, h=16, n=8192, d=64, dv=64, dtype="bf16", states=False,
             ragged=False),
        # one token of a small batch: latency
        dict(name="step_b2h16", kind="step", b=2, h=16, d=64, dv=64, dtype="bf16"),
        # one token of a serving batch: the states' bytes
        dict(name="step_b64h16", kind="step", b=64, h=16, d=128, dv=128, dtype="bf16"),
        # two prompts into the cache, at the softmax companion's benchmark shape
        dict(name="append_b2h16n4096", kind="append", b=2, hk=16, n=4096, d=64, dv=64, dtype="bf16", past=0, cap=4160),
        # pieces of long prompts, starting inside a block
        dict(name="append_b8h8n8200", kind="append", b=8, hk=8, n=8200, d=128, dv=128, dtype="bf16", past=1000, cap=9280),
        # one token with the companion's window: latency
        dict(name="sliding_w64_b2h16", kind="sliding", b=2, h=16, hk=16, d=64, dv=64, dtype="bf16", length=300, cap=128,
             window=64),
        # one token of a serving batch over all of its long contexts, four query heads for each cached one
        dict(name="sliding_b8h32n32768", kind="sliding", b=8, h=32, hk=8, d=128, dv=128, dtype="bf16", length=32768,
             cap=32768, window=0),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _cost(c):
    # what the plain form works through, roughly: bytes in 32 bits
    if c["kind"] in ("forward", "train"):
        return c["b"] * c["h"] * c["n"] * (c["d"] + c["dv"] + 128) * (3 if c["kind"] == "train" else 1)
    if c["kind"] == "step":
        return c["b"] * c["h"] * c["d"] * c["dv"]
    return c["b"] * c["hk"] * c["cap"] * (c["d"] + c["dv"])


def draw(rng):
    """One more case: any kind, over the listed cases' ranges of batches, heads, lengths, dims and types."""
    kind = rng.choice(["forward", "forward", "train", "train", "step", "append", "sliding", "sliding"])
    c = dict(kind=kind, b=_log_int(rng, 1, 16), dtype=rng.choice(["bf16", "bf16", "bf16", "f32"]))
    dims = [16, 24, 32, 40, 64, 64, 64, 80, 96, 128, 128]
    c["d"] = rng.choice(dims)
    c["dv"] = c["d"] if rng.random() < 0.6 else rng.choice(dims)
    if kind in ("forward", "train"):
        c.update(h=rng.choice([1, 2, 4, 8, 12, 16, 16, 32]), n=_log_int(rng, 1, 65536 if kind == "forward" else 16384),
                 states=rng.random() < 0.5, ragged=rng.random() < 0.4)
        if rng.random() < 0.4 and c["n"] > 256:
            c["n"] -= c["n"] % 64
    elif kind == "step":
        c.update(b=_log_int(rng, 1, 64), h=rng.choice([2, 4, 8, 16, 16, 24, 32]))
    else:
        c["hk"] = rng.choice([1, 2, 4, 8, 8, 16])
        n = _log_int(rng, 1, 32768)
        if kind == "append":
            c.update(n=n, past=rng.choice([0, 0, 64 * rng.randint(1, 20), rng.randint(1, 1000)]))
            c["cap"] = -(-(c["past"] + n) // BLOCK) * BLOCK + BLOCK * rng.randint(0, 8)
        else:
            c.update(b=_log_int(rng, 1, 64), h=c["hk"] * rng.choice([1, 1, 2, 4, 8]), length=n, window=0)
            c["cap"] = -(-n // BLOCK) * BLOCK
            if rng.random() < 0.5:   # a ring of little more than the window
                c["window"] = _log_int(rng, 1, 4096)
                c["cap"] = min(c["cap"] + BLOCK, -(-(c["window"] + BLOCK - 1) // BLOCK) * BLOCK)
                c["window"] = min(c["window"], c["cap"] - BLOCK + 1)
    most = max(_cost(x) for x in listed() if x["kind"] == kind)
    while _cost(c) > most:
        if c["b"] > 1:
            c["b"] = (c["b"] + 1) // 2
        elif kind in ("forward", "train") and c["n"] > 1:
            c["n"] = c["n"] * 2 // 3 + 1
        elif "h" in c and "hk" not in c:
            c["h"] = max(1, c["h"] // 2)
        else:
            c["hk"] = max(1, c["hk"] // 2)
            if "h" in c:
                c["h"] = c["hk"]
    return c


# ---- inputs

def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _log_decay(h):
    """From exp(-2^(-8 / h)) for the first head to exp(-1 / 256) for the last, the usual geometric spread."""
    return -(2.0 ** (-8.0 * torch.arange(1, h + 1, device="cuda", dtype=torch.float64) / h)).float()


def _codes(g, c, lengths):
    """The cache after lengths[i] - 1 tokens of N(0, 1) in sequence i: codes where a token is held, zeros elsewhere."""
    b, hk, cap, dp, dvp = c["b"], c["hk"], c["cap"], _padded(c["d"]), _padded(c["dv"])
    k = torch.zeros(b, hk, cap, dp, dtype=E4M3, device="cuda")
    v = torch.zeros(b, hk, cap // BLOCK, dvp, BLOCK, dtype=E4M3, device="cuda")
    last = lengths.long().view(b, 1) - 1
    at = last - (last - torch.arange(cap, device="cuda")) % cap      # the position that a place of the ring holds
    there = (at >= 0) & (at < last) & (at >= last // BLOCK * BLOCK - cap + BLOCK)
    for i in range(b):    # a sequence at a time: 32-bit numbers of the whole cache would be four times its size
        k[i, :, :, :c["d"]] = torch.where(there[i].view(1, cap, 1), _randn(g, hk, cap, c["d"]) * 64, 0.0).clamp_(-448, 448).to(E4M3)
        x = torch.where(there[i].view(1, cap, 1), _randn(g, hk, cap, c["dv"]) * 64, 0.0).clamp_(-448, 448)
        v[i, :, :, :c["dv"]] = x.view(hk, cap // BLOCK, BLOCK, c["dv"]).transpose(2, 3).to(E4M3)
    scale = torch.where(there.view(b, 1, -1, BLOCK).any(-1), 2.0 ** -6, 0.0).expand(b, hk, -1)
    return {"k": k.view(b, hk, -1, BLOCK, dp), "v": v, "k_scale": scale.clone(), "v_scale": scale.clone()}


def _padded(d):
    return 32 if d <= 32 else 64 if d <= 64 else 128


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dt, b, d, dv = DTYPES[c["dtype"]], c["b"], c["d"], c["dv"]
    s = {"case": c}
    if c["kind"] in ("forward", "train"):
        h, n = c["h"], c["n"]
        s.update(q=_randn(g, b, h, n, d).to(dt), k=_randn(g, b, h, n, d).to(dt), v=_randn(g, b, h, n, dv).to(dt),
                 log_decay=_log_decay(h), state=None, lengths=None)
        if c["states"]:
            s["state"] = _randn(g, b, h, d, dv) * 4
        if c["ragged"]:
            s["lengths"] = torch.randint(0, n + 1, (b,), generator=g, device="cuda", dtype=torch.int32)
            s["lengths"][0] = n
        if c["kind"] == "train":
            for x in ("q", "k", "v") + (("state",) if c["states"] else ()):
                s[x].requires_grad_()
            s["dy"] = _randn(g, b, h, n, dv).to(dt)
    elif c["kind"] == "step":
        h = c["h"]
        s.update(q=_randn(g, b, h, d).to(dt), k=_randn(g, b, h, d).to(dt), v=_randn(g, b, h, dv).to(dt),
                 log_decay=_log_decay(h), state=_randn(g, b, h, d, dv) * 4)
    elif c["kind"] == "append":
        s.update(k=_randn(g, b, c["hk"], c["n"], d).to(dt), v=_randn(g, b, c["hk"], c["n"], dv).to(dt),
                 start=torch.full((b,), c["past"], dtype=torch.int32, device="cuda"))
        s["cache"] = _codes(g, c, s["start"] + 1)
    else:
        s.update(q=_randn(g, b, c["h"], d).to(dt), k=_randn(g, b, c["hk"], d).to(dt), v=_randn(g, b, c["hk"], dv).to(dt))
        # sequences of unlike lengths, the longest as long as the case says
        s["lengths"] = torch.randint((c["length"] + 1) // 2, c["length"] + 1, (b,), generator=g, device="cuda",
                                     dtype=torch.int32)
        s["lengths"][0] = c["length"]
        s["cache"] = _codes(g, c, s["lengths"])
    return s


# ---- plain forms

def _powers(log_decay, n):
    """exp(log_decay_h n) for whole n of any shape, (h, *n.shape), in 32 bits from 64-bit exponents."""
    return torch.exp(log_decay.double().view(-1, *([1] * n.dim())) * n.double()).float()


def _plain_attn(q, k, v, log_decay, scale, state, lead):
    """s sum_{u <= t} g^(t - u) (q_t . k_u) v_u + s g^(t + lead) q_t S, 32-bit (b, h, n, .), by chunks of 256 tokens:
    pairs inside a chunk, and the state before each chunk as a decayed sum of the chunks' own."""
    b, h, n, d = q.shape
    dv, cs = v.shape[-1], min(256, n)
    nc = -(-n // cs)
    q, k, v = (torch.nn.functional.pad(x, (0, 0, 0, nc * cs - n)).view(b, h, nc, cs, -1) for x in (q, k, v))
    i = torch.arange(cs, device=q.device)
    gap = i[:, None] - i[None, :]
    inside = torch.where(gap >= 0, _powers(log_decay, gap.clamp(min=0)), 0.0).view(1, h, 1, cs, cs)
    y = torch.matmul(torch.matmul(q, k.transpose(-1, -2)) * inside, v)
    to_end = _powers(log_decay, cs - 1 - i).view(1, h, 1, cs, 1)
    own_states = torch.matmul((k * to_end).transpose(-1, -2), v)                        # (b, h, nc, d, dv)
    j = torch.arange(nc, device=q.device)
    gap = j[:, None] - j[None, :] - 1
    carry = torch.where(gap >= 0, _powers(log_decay, cs * gap.clamp(min=0)), 0.0)       # (h, nc, nc)
    before = torch.matmul(carry, own_states.reshape(b, h, nc, d * dv)).view(b, h, nc, d, dv)
    y = y + torch.matmul(q, before) * _powers(log_decay, i + 1).view(1, h, 1, cs, 1)
    y = y.reshape(b, h, nc * cs, dv)[:, :, :n]
    if state is not None:
        far = _powers(log_decay, torch.arange(n, device=q.device) + lead).view(1, h, n, 1)
        y = y + torch.matmul(q.reshape(b, h, nc * cs, d)[:, :, :n], state) * far
    return y * scale


def _plain_state(k, v, log_decay, last, state, shift=0):
    """sum_u g^(last - 1 - u + shift) k_u v_u^T + g^last S; last (b,) tokens of each sequence."""
    n = k.shape[2]
    gap = last.view(-1, 1) - 1 - torch.arange(n, device=k.device) + shift
    w = torch.exp(log_decay.double().view(1, -1, 1) * gap.clamp(min=0).double().unsqueeze(1)).float()
    out = torch.matmul((k * w.unsqueeze(-1)).transpose(-1, -2), v)
    if state is not None:
        out = out + state * torch.exp(log_decay.double() * last.double().view(-1, 1)).float()[..., None, None]
    return out


def _reversed(x, last):
    """Row t of a sequence of ``last`` tokens at row last - 1 - t; rows behind the sequence are zero either way."""
    n = x.shape[2]
    t = last.view(-1, 1) - 1 - torch.arange(n, device=x.device)
    at = t.clamp(min=0).view(-1, 1, n, 1).expand(-1, x.shape[1], -1, x.shape[3])
    return torch.gather(x, 2, at) * (t >= 0).view(-1, 1, n, 1)


def _plain_forward(s, x):
    c, g = s["case"], s["log_decay"]
    q, k, v, last = x
    state = None if s["state"] is None else s["state"].detach()
    y = _plain_attn(q, k, v, g, 1.0 / math.sqrt(c["d"]), state, 1)
    return y.to(s["q"].dtype)


def _plain_inputs(s):
    """q, k, v in 32 bits with zeros behind each sequence, and the sequences' lengths."""
    n, b = s["case"]["n"], s["case"]["b"]
    last = s["lengths"] if s["lengths"] is not None else torch.full((b,), n, dtype=torch.int32, device="cuda")
    there = (torch.arange(n, device="cuda") < last.view(-1, 1)).view(b, 1, n, 1)
    return [torch.where(there, s[x].detach().float(), 0.0) for x in ("q", "k", "v")] + [last]


def _plain_train(s):
    c, g, scale = s["case"], s["log_decay"], 1.0 / math.sqrt(s["case"]["d"])
    x = _plain_inputs(s)
    q, k, v, last = x
    out = {"y": _plain_forward(s, x)}
    n, b = c["n"], c["b"]
    there = (torch.arange(n, device="cuda") < last.view(-1, 1)).view(b, 1, n, 1)
    dy = torch.where(there, s["dy"].float(), 0.0)
    state = None if s["state"] is None else s["state"].detach().transpose(-1, -2).contiguous()
    # dq_t = s sum_{u <= t} g^(t - u) (dy_t . v_u) k_u + s g^(t + 1) S dy_t: the same sums with other operands; dk and
    # dv are such sums from the other end
    out["dq"] = _plain_attn(dy, v, k, g, scale, state, 1).to(s["q"].dtype)
    rq, rk, rv, rdy = (_reversed(t, last) for t in (q, k, v, dy))
    out["dk"] = _reversed(_plain_attn(rv, rdy, rq, g, scale, None, 0), last).to(s["q"].dtype)
    out["dv"] = _reversed(_plain_attn(rk, rq, rdy, g, scale, None, 0), last).to(s["q"].dtype)
    if state is not None:
        # the first state's gradient: s sum_t g^(t + 1) q_t dy_t^T
        out["dstate"] = _plain_state(rq, rdy, g, last, None, 1) * scale
    return out


def _plain_step(s):
    g, st = torch.exp(s["log_decay"]).view(1, -1, 1, 1), s["state"]
    st.copy_(st * g + s["k"].float().unsqueeze(-1) * s["v"].float().unsqueeze(-2))
    y = torch.matmul(s["q"].float().unsqueeze(-2), st).squeeze(-2) / math.sqrt(s["case"]["d"])
    return {"y": y.to(s["q"].dtype), "state": st}


def _scale_for(amax):
    """The smallest power of two (2^-100 at the least) that brings amax to 448, e4m3's largest number, or below."""
    m, e = torch.frexp(amax)
    e = torch.where(amax > 0, e - 9 + (m > 0.875), LEAST_SCALE).clamp(min=LEAST_SCALE)
    return (e.int() + 127 << 23).view(torch.float32)


def _plain_append_rows(cache, name, x, past):
    """Rows x (b, hk, n, d) as tokens past, past + 1, ..: whole blocks, the first joined with what it holds already."""
    codes, scales, (b, hk, n, d) = cache[name], cache[name + "_scale"], x.shape
    first, end = past // BLOCK, -(-(past + n) // BLOCK)      # the blocks that are written
    rows = codes if name == "k" else codes.transpose(-1, -2)
    x = torch.nn.functional.pad(x.float(), (0, rows.shape[-1] - d, past - BLOCK * first, BLOCK * end - past - n))
    x = x.view(b, hk, end - first, BLOCK, -1)
    scale = _scale_for(x.abs().amax((-1, -2)))
    if past % BLOCK:
        scale[:, :, 0] = torch.maximum(scale[:, :, 0], scales[:, :, first])
        kept = torch.arange(BLOCK, device="cuda").view(-1, 1) < past % BLOCK
        x[:, :, 0] += torch.where(kept, rows[:, :, first].float() * scales[:, :, first, None, None], 0.0)
    new = (x / scale[..., None, None]).to(E4M3)
    codes[:, :, first:end] = new if name == "k" else new.transpose(-1, -2)
    scales[:, :, first:end] = scale


def _plain_append(s):
    _plain_append_rows(s["cache"], "k", s["k"], s["case"]["past"])
    _plain_append_rows(s["cache"], "v", s["v"], s["case"]["past"])
    return s["cache"]


def _plain_append_token(cache, name, x, last):
    """Rows x (b, hk, d), one each, as the tokens at positions last (b,) of a ring of blocks."""
    codes, scales, b = cache[name], cache[name + "_scale"], x.shape[0]
    i, blk, slot = torch.arange(b, device="cuda"), last // BLOCK % codes.shape[2], last % BLOCK
    place = torch.arange(BLOCK, device="cuda").view(1, 1, -1, 1)
    rows = codes[i, :, blk].float() if name == "k" else codes[i, :, blk].float().transpose(-1, -2)
    old = scales[i, :, blk] * (slot > 0).view(-1, 1)
    x = torch.nn.functional.pad(x.float(), (0, rows.shape[-1] - x.shape[-1]))
    scale = torch.maximum(old, _scale_for(x.abs().amax(-1)))
    value = torch.where(place < slot.view(b, 1, 1, 1), rows * old[..., None, None], 0.0)
    value = torch.where(place == slot.view(b, 1, 1, 1), x.unsqueeze(-2), value)
    new = (value / scale[..., None, None]).to(E4M3)
    codes[i, :, blk] = new if name == "k" else new.transpose(-1, -2)
    scales[i, :, blk] = scale


def _plain_sliding(s):
    c, cache, q = s["case"], s["cache"], s["q"]
    b, h, hk, d, dv, cap = (c[x] for x in ("b", "h", "hk", "d", "dv", "cap"))
    last = s["lengths"].long() - 1
    _plain_append_token(cache, "k", s["k"], last)
    _plain_append_token(cache, "v", s["v"], last)
    # positions that the ring's places hold, and those of the window
    at = last.view(-1, 1) - (last.view(-1, 1) - torch.arange(cap, device="cuda")) % cap
    seen = (at >= 0) & ((at > last.view(-1, 1) - c["window"]) if c["window"] else (at >= 0))
    k = (cache["k"].float() * cache["k_scale"][..., None, None]).view(b, hk, cap, -1)[..., :d]
    v = (cache["v"].float() * cache["v_scale"][..., None, None]).transpose(-1, -2).reshape(b, hk, cap, -1)[..., :dv]
    p = torch.matmul(q.float().view(b, hk, h // hk, d), k.transpose(-1, -2)) / math.sqrt(d)
    p = torch.where(seen.view(b, 1, 1, cap), p, float("-inf"))
    p = torch.exp(p - p.amax(-1, keepdim=True))
    y = torch.matmul(p, v) / p.sum(-1, keepdim=True)
    return {"y": y.view(b, h, dv).to(q.dtype), **cache}


# ---- the calls

def run(state):
    s, c = state, state["case"]
    kind = c["kind"]
    if own:
        K = _kernels()
        if kind == "forward":
            if not c["states"]:
                return {"y": K.decay_linear_attn(s["q"], s["k"], s["v"], s["log_decay"], lengths=s["lengths"])}
            y, st = K.decay_linear_attn(s["q"], s["k"], s["v"], s["log_decay"], state_in=s["state"], return_state=True,
                                        lengths=s["lengths"])
            return {"y": y, "state": st}
        if kind == "train":
            y = K.decay_linear_attn(s["q"], s["k"], s["v"], s["log_decay"], state_in=s["state"], lengths=s["lengths"])
            names = ["q", "k", "v"] + (["state"] if c["states"] else [])
            grads = torch.autograd.grad(y, [s[x] for x in names], s["dy"])
            return {"y": y.detach(), **{"d" + x: t for x, t in zip(names, grads)}}
        if kind == "step":
            return {"y": K.decay_decode_step(s["q"], s["k"], s["v"], s["log_decay"], s["state"]), "state": s["state"]}
        cache = K.SlidingCache(**s["cache"], d=c["d"], dv=c["dv"])
        if kind == "append":
            K.sliding_cache_append(cache, s["k"], s["v"], start=s["start"])
            return s["cache"]
        y = K.sliding_decode_step(s["q"], s["k"], s["v"], cache, s["lengths"], window_size=c["window"] or None)
        return {"y": y, **s["cache"]}
    with torch.no_grad():
        if kind == "forward":
            x = _plain_inputs(s)
            out = {"y": _plain_forward(s, x)}
            if c["states"]:
                out["state"] = _plain_state(x[1], x[2], s["log_decay"], x[3], s["state"])
            return out
        return {"train": _plain_train, "step": _plain_step, "append": _plain_append, "sliding": _plain_sliding}[kind](s)


# ---- the same in 64 bits

def _exact_attn(s):
    """The recurrence, 128 tokens at a time: y and the state after each sequence's last token."""
    c = s["case"]
    b, h, n, d, dv = (c[x] for x in ("b", "h", "n", "d", "dv"))
    g = s["log_decay"].double().view(1, h, 1, 1)
    last = (s["lengths"] if s["lengths"] is not None else torch.full((b,), n, device="cuda")).long().view(b, 1, 1, 1)
    st = torch.zeros(b, h, d, dv, dtype=torch.float64, device="cuda") if s["state"] is None else s["state"].double()
    ys = []
    for t0 in range(0, n, 128):
        t1 = min(n, t0 + 128)
        t = torch.arange(t0, t1, device="cuda")
        there = t.view(1, 1, -1, 1) < last
        q, k, v = (torch.where(there, s[x][:, :, t0:t1].double(), 0.0) for x in ("q", "k", "v"))
        gap = (t[:, None] - t[None, :]).double()
        p = torch.matmul(q, k.transpose(-1, -2).contiguous()) * torch.exp(torch.where(gap >= 0, g * gap, float("-inf")))
        ys.append((torch.matmul(p, v) + torch.matmul(q, st) * torch.exp(g * (t - t0 + 1).view(1, 1, -1, 1))) / math.sqrt(d))
        m = (last - t0).clamp(0, t1 - t0)                       # tokens of each sequence in this piece
        w = torch.where(there, torch.exp(g * (m - 1 - (t - t0).view(1, 1, -1, 1)).clamp(min=0)), 0.0)
        st = st * torch.exp(g * m) + torch.matmul((k * w).transpose(-1, -2).contiguous(), v)
    return torch.cat(ys, 2), st


def _pow2(e):
    return (e.long() + 1023 << 52).view(torch.float64)


def _exact_codes(x, scale):
    """Rows over a power-of-two scale, rounded to e4m3 (nearest, ties to even), in 64 bits."""
    r = x / scale
    e = torch.frexp(r)[1].clamp(min=-5)                         # 4 significant bits, down to 2^-9
    step = _pow2(e - 4)
    return torch.round(r / step) * step


def _exact_scale(amax):
    e = torch.ceil(torch.log2(amax.clamp(min=1e-300) / 448)).clamp(min=LEAST_SCALE)
    e = torch.where(448 * _pow2(e - 1) >= amax, e - 1, e).clamp(min=LEAST_SCALE)   # where log2 rounded up
    return _pow2(torch.where(448 * _pow2(e) < amax, e + 1, e))


def _exact_cache(s, x, name, positions):
    """The cache's codes and scales with rows x (b, hk, m, d) at the given positions (b, m), block by block."""
    codes, scales = s["cache"][name].double(), s["cache"][name + "_scale"].double()
    codes = codes.clone() if name == "k" else codes.transpose(-1, -2).clone()
    scales, nb = scales.clone(), codes.shape[2]
    for i in range(x.shape[0]):
        at, blocks = positions[i], torch.unique(positions[i] // BLOCK).tolist()
        lo, hi = int(at[0]), int(at[-1])
        for j in blocks:
            a, e = max(lo, j * BLOCK), min(hi + 1, (j + 1) * BLOCK)
            rows = torch.zeros_like(codes[i, :, 0])
            kept = a - j * BLOCK
            scale = _exact_scale(x[i, :, a - lo:e - lo].abs().amax((-1, -2)))
            if kept:
                scale = torch.maximum(scale, scales[i, :, j % nb])
                rows[:, :kept] = codes[i, :, j % nb, :kept] * scales[i, :, j % nb, None, None]
            rows[:, kept:e - j * BLOCK, :x.shape[-1]] = x[i, :, a - lo:e - lo]
            codes[i, :, j % nb] = _exact_codes(rows, scale[:, None, None])
            scales[i, :, j % nb] = scale
    return codes, scales


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["kind"] == "forward":
        y, st = _exact_attn(s)
        return {"y": y, "state": st} if c["states"] else {"y": y}
    if c["kind"] == "train":
        names = ["q", "k", "v"] + (["state"] if c["states"] else [])
        for x in names:
            s[x] = s[x].detach().double().requires_grad_()
        y, _ = _exact_attn(s)
        grads = torch.autograd.grad(y, [s[x] for x in names], s["dy"].double())
        return {"y": y.detach(), **{"d" + x: t for x, t in zip(names, grads)}}
    if c["kind"] == "step":
        q, k, v = (s[x].double() for x in ("q", "k", "v"))
        st = s["state"].double() * torch.exp(s["log_decay"].double()).view(1, -1, 1, 1) + k.unsqueeze(-1) * v.unsqueeze(-2)
        return {"y": (q.unsqueeze(-1) * st).sum(-2) / math.sqrt(c["d"]), "state": st}
    b, hk, d, dv = c["b"], c["hk"], c["d"], c["dv"]
    if c["kind"] == "append":
        if b * (c["n"] // BLOCK + 2) > 4096:
            return None
        at = c["past"] + torch.arange(c["n"], device="cuda").expand(b, -1)
        kc, ks = _exact_cache(s, s["k"].double(), "k", at)
        vc, vs = _exact_cache(s, s["v"].double(), "v", at)
        return {"k": kc, "v": vc.transpose(-1, -2), "k_scale": ks, "v_scale": vs}
    last = s["lengths"].long() - 1
    at = last.view(b, 1)
    kc, ks = _exact_cache(s, s["k"].double().unsqueeze(2), "k", at)
    vc, vs = _exact_cache(s, s["v"].double().unsqueeze(2), "v", at)
    y = torch.zeros(b, c["h"], dv, dtype=torch.float64, device="cuda")
    for i in range(b):
        p1 = int(last[i])
        p0 = max(0, p1 + 1 - c["window"]) if c["window"] else 0
        pos = torch.arange(p0, p1 + 1, device="cuda")
        blk, slot = pos // BLOCK % kc.shape[2], pos % BLOCK
        k = kc[i, :, blk, slot, :d] * ks[i, :, blk].unsqueeze(-1)
        v = vc[i, :, blk, slot, :dv] * vs[i, :, blk].unsqueeze(-1)
        p = torch.softmax(torch.matmul(s["q"][i].double().view(hk, -1, d), k.transpose(1, 2).contiguous()) / math.sqrt(d), -1)
        y[i] = torch.matmul(p, v).reshape(c["h"], dv)
    return {"y": y, "k": kc, "v": vc.transpose(-1, -2), "k_scale": ks, "v_scale": vs}


# ---- what a call cannot do without

def work(case):
    c = case
    b, d, dv, e = c["b"], c["d"], c["dv"], (2 if c["dtype"] == "bf16" else 4)
    if c["kind"] in ("forward", "train"):
        rows, state = b * c["h"] * c["n"], 4 * b * c["h"] * d * dv
        # a token's pairs in a chunk of 64, and its part of the state's product and update
        flops = rows * (65 * (d + dv) + 4 * d * dv)
        if c["kind"] == "forward":
            return {"bytes": e * rows * 2 * (d + dv) + (2 * state if c["states"] else 0), "flops": flops}
        # q, k, v and dy in, y and three gradients out; the pairs' two products and three gradients, two states
        return {"bytes": e * rows * 4 * (d + dv) + (2 * state if c["states"] else 0),
                "flops": flops + rows * (65 * (3 * d + 2 * dv) + 8 * d * dv)}
    if c["kind"] == "step":
        bh = b * c["h"]
        return {"bytes": bh * (8 * d * dv + e * 2 * (d + dv)), "flops": bh * 5 * d * dv}
    if c["kind"] == "append":
        rows = b * c["hk"] * c["n"]
        return {"bytes": rows * (e + 1) * (d + dv) + rows // 64 * 8, "flops": rows * 2 * (d + dv)}
    # lengths are spread evenly from half of the longest on
    seen = min(c["window"] or c["length"], (0.75 if b > 1 else 1.0) * c["length"])
    return {"bytes": b * c["hk"] * seen * (d + dv) + e * b * (c["h"] + c["hk"]) * (d + dv),
            "flops": 2 * b * c["h"] * seen * (d + dv)}
