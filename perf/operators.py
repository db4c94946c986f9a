"""Measured cases of the attention-side operators: the per-head norm and position rotation of queries and keys (forward
and backward), the append to a paged 8-bit key/value cache, and the attention that reads that cache.

A case is a dict of plain values.  `prepare` makes what a program holds before the call, `run` makes one call: with
`own` false in elementary torch operations in 32 bits (angles, and sums over all tokens, in 64), with `own` true
through `dfdx_b200.Cuda`.  `exact` computes the same from the definitions in 64 bits.
"""
from __future__ import annotations

import functools
import math

import torch

own = False

EPS = 1e-6
E4M3_MAX = 448.0
MIN_SCALE = 2.0 ** -60          # the smallest scale of a cache block: blocks of zeros carry it
_DTYPES = {"f16": torch.float16, "f32": torch.float32}


# ----------------------------------------------------------------------------------------------- cases
def _rot(name, kind, dtype, batch, tokens, q_heads, k_heads, d, rotated, axes=1, interleaved=False, norm=True, first=0):
    return dict(name=name, kind=kind, dtype=dtype, batch=batch, tokens=tokens, q_heads=q_heads, k_heads=k_heads,
                head_dim=d, rotated=rotated, axes=axes, interleaved=interleaved, norm=norm, first=first)


def _app(name, dtype, seqs, new, past, page, q_heads, k_heads, d, rotated, norm=True, interleaved=False):
    return dict(name=name, kind="append", dtype=dtype, seqs=seqs, new_min=new[0], new_max=new[1], past_min=past[0],
                past_max=past[1], page=page, q_heads=q_heads, k_heads=k_heads, head_dim=d, rotated=rotated, axes=1,
                interleaved=interleaved, norm=norm)


def _att(name, seqs, new, past, page, q_heads, k_heads, d, window=0):
    return dict(name=name, kind="attention", dtype="f16", seqs=seqs, new_min=new[0], new_max=new[1], past_min=past[0],
                past_max=past[1], page=page, q_heads=q_heads, k_heads=k_heads, head_dim=d, window=window)


def listed():
    return [
        # a handful of new tokens far into a context: what one decoding step of a small model norms and rotates
        _rot("rotary few tokens", "rotary", "f16", 1, 7, 16, 4, 128, 128, first=70001),
        # a training batch with shared key heads, straight out of the fused projection
        _rot("rotary training batch", "rotary", "f16", 8, 2048, 32, 8, 128, 128),
        # the attention benchmark's batch x heads x length, without shared heads
        _rot("rotary grad 16x512x16x64", "rotary_grad", "f16", 16, 512, 16, 16, 64, 64),
        # f32 training on video tokens: time, height and width rotate a share of the pairs each; odd extents
        _rot("rotary grad video f32", "rotary_grad", "f32", 2, 2475, 12, 12, 96, 96, axes=3),
        # the largest backward: long sequences, shared key heads, adjacent pairs, a part of each head rotated
        _rot("rotary grad long", "rotary_grad", "f16", 2, 8192, 32, 4, 128, 64, interleaved=True),
        # one token for each of 64 running sequences
        _app("append decode 64", "f16", 64, (1, 1), (100, 8000), 64, 32, 8, 128, 128),
        # prompts of several lengths arriving together, some behind a cached prefix
        _app("append prompts", "f16", 9, (130, 1900), (0, 700), 64, 32, 8, 128, 128),
        # one sequence, one token: the latency of a decoding step
        _att("attend one sequence", 1, (1, 1), (900, 900), 64, 16, 4, 64),
        # a serving batch of ragged lengths
        _att("attend batch 48", 48, (1, 1), (200, 12000), 64, 32, 8, 128),
        # one very long context
        _att("attend long context", 1, (1, 1), (131000, 131000), 128, 32, 8, 128),
        # drafts of a few tokens to verify at once, small pages, a sliding window
        _att("attend drafts window", 24, (2, 5), (50, 6000), 16, 24, 6, 96, window=1024),
        # prompts taken in chunks behind cached prefixes: bound by the products
        _att("attend prompt chunks", 3, (511, 1024), (0, 6000), 64, 32, 8, 128),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(("rotary", "rotary_grad", "append", "attention", "attention"))
    d = rng.choice((64, 96, 128))
    k_heads = rng.choice((1, 2, 4, 8))
    q_heads = k_heads * rng.choice((1, 2, 3, 4, 8) if k_heads < 8 else (1, 2, 4))
    page = rng.choice((16, 32, 64, 128))
    if kind in ("rotary", "rotary_grad"):
        batch = log(1, 8)
        tokens = max(1, min(log(1, 9000), 600000 // (batch * (q_heads + k_heads))))
        axes = rng.choice((1, 1, 2, 3))
        dtype = rng.choice(("f16", "f16", "f32"))
        return {k: v for k, v in _rot("", kind, dtype, batch, tokens, q_heads, k_heads, d, rng.choice((d, d, d // 2)), axes,
                                      rng.random() < 0.3, rng.random() < 0.8, rng.choice((0, 0, 5000, 900000))).items()
                if k != "name"}
    if kind == "append":
        seqs = log(1, 100)
        new = log(1, max(1, 8000 // seqs)) if rng.random() < 0.6 else 1
        return {k: v for k, v in _app("", rng.choice(("f16", "f16", "f32")), seqs, (max(1, new // 3), new),
                                      (rng.choice((0, 17)), log(17, 9000)), page, q_heads, k_heads, d,
                                      rng.choice((d, d // 2)), rng.random() < 0.5, rng.random() < 0.3).items() if k != "name"}
    shape = rng.choice(("decode", "decode", "drafts", "chunk"))
    seqs = log(1, 60) if shape == "decode" else log(1, 20) if shape == "drafts" else log(1, 4)
    new = 1 if shape == "decode" else rng.randint(2, 6) if shape == "drafts" else log(100, 1024 // (1 + seqs // 3))
    past = log(20, max(40, min(120000, 250000 // seqs))) if shape != "chunk" else log(20, 5000)
    window = rng.choice((0, 0, 0, 700))
    return {k: v for k, v in _att("", seqs, (max(1, new // 2), new), (past // 8, past), page, q_heads, k_heads, d,
                                  window).items() if k != "name"}


def _spread(lo, hi, n, phase):
    """n whole numbers in [lo, hi], the ends among them where n allows: a fixed ragged pattern."""
    out = [lo + int((hi - lo + 1) * ((i * 0.6180339887498949 + phase) % 1.0)) for i in range(n)]
    out[0] = hi
    if n > 1:
        out[-1] = lo
    return out


def _lengths(c):
    new = _spread(c["new_min"], c["new_max"], c["seqs"], 0.25)
    past = _spread(c["past_min"], c["past_max"], c["seqs"], 0.0)
    return new, past


def _visible(c):
    """(key rows that some query of the sequence sees, query-key pairs) over all sequences."""
    rows = pairs = 0
    w = c["window"]
    for m, p in zip(*_lengths(c)):
        first = max(0, p + 1 - w) if w else 0
        rows += p + m - first
        pairs += sum(min(p + j + 1, w) if w else p + j + 1 for j in range(m))
    return rows, pairs


def work(c):
    es, d, hq, hk = (2 if c["dtype"] == "f16" else 4), c["head_dim"], c["q_heads"], c["k_heads"]
    if c["kind"] in ("rotary", "rotary_grad"):
        n = c["batch"] * c["tokens"] * (hq + hk) * d
        grad = c["kind"] == "rotary_grad"
        return {"bytes": n * es * (3 if grad else 2) + 4 * c["axes"] * c["batch"] * c["tokens"] + 2 * d * es * (3 if grad else 1),
                "flops": n * (14 if grad else 7)}
    new, past = _lengths(c)
    if c["kind"] == "append":
        t, touched = sum(new), sum(_touched(c, m, p) for m, p in zip(new, past))
        block = hk * c["page"] * d
        # the rows in, the queries out, the codes; and the touched blocks read back as f16 values
        return {"bytes": t * (2 * hq + 2 * hk) * d * es + 2 * t * hk * d + 2 * touched * block * 3,
                "flops": t * (hq + 2 * hk) * d * 8 + 2 * touched * block}
    rows, pairs = _visible(c)
    t = sum(new)
    return {"bytes": rows * hk * (2 * d + 8.0 / c["page"]) + 2 * t * hq * d * 2 + 4 * t * hq, "flops": 4 * d * hq * pairs}


def _touched(c, m, p):
    return (p + m - 1) // c["page"] - p // c["page"] + 1


# --------------------------------------------------------------------------------------------- inputs
def _axis_pairs(c):
    pairs, axes = c["rotated"] // 2, c["axes"]
    each = pairs // axes
    return (pairs - each * (axes - 1),) + (each,) * (axes - 1)


def _frequencies(c, dev):
    """Radians per position of every rotated pair: base 10000, counted from the start on each axis."""
    parts = [10000.0 ** (-torch.arange(n, dtype=torch.float64, device=dev) / max(n, 1)) for n in _axis_pairs(c)]
    return torch.cat(parts)


def _grid_positions(c, dev):
    """(axes, batch, tokens) positions: the token's index, or its place in a video of square frames."""
    i = torch.arange(c["tokens"], device=dev)
    side = max(2, int(round(c["tokens"] ** (1.0 / 3.0))))
    axes = {1: [i], 2: [i // side, i % side], 3: [i // (side * side), i // side % side, i % side]}[c["axes"]]
    p = torch.stack(axes).to(torch.int32) + c["first"]
    return p[:, None, :].expand(-1, c["batch"], -1).contiguous()


def _projection(c, rows, g, dev, dt):
    """q, k, v views of one fused projection's output; the keys have a few strong channels, as trained ones have."""
    hq, hk, d = c["q_heads"], c["k_heads"], c["head_dim"]
    x = torch.randn(*rows, (hq + 2 * hk) * d, generator=g, device=dev, dtype=torch.float32)
    strong = 1.0 + 7.0 * (torch.rand(hk * d, generator=g, device=dev) < 0.02)
    x[..., hq * d:(hq + hk) * d] *= strong
    x = x.to(dt)
    return (x[..., :hq * d].unflatten(-1, (hq, d)), x[..., hq * d:(hq + hk) * d].unflatten(-1, (hk, d)),
            x[..., (hq + hk) * d:].unflatten(-1, (hk, d)))


def _gain(c, g, dev, dt):
    return (1.0 + 0.2 * torch.randn(c["head_dim"], generator=g, device=dev)).to(dt) if c["norm"] else None


def _cache(c, g, dev, pages):
    """A cache of `pages` pages that earlier sequences have filled: codes and the scales of their blocks."""
    hk, d, page = c["k_heads"], c["head_dim"], c["page"]
    out = {}
    for name in ("k", "v"):
        x = torch.randn(pages, hk, page, d, generator=g, device=dev)
        if name == "k":
            x *= 1.0 + 7.0 * (torch.rand(hk, 1, d, generator=g, device=dev) < 0.02)
        scale = _plain_scale(x.abs().amax((2, 3)))
        out[name] = (x / scale[:, :, None, None]).to(torch.float8_e4m3fn)
        out[name + "_scale"] = scale
    return out


def prepare(c, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = _DTYPES[c["dtype"]]
    s = {"case": c}
    if c["kind"] in ("rotary", "rotary_grad"):
        rows = (c["batch"], c["tokens"])
        s["q"], s["k"], _ = _projection(c, rows, g, dev, dt)
        s["frequencies"], s["positions"] = _frequencies(c, dev), _grid_positions(c, dev)
        s["q_gain"], s["k_gain"] = _gain(c, g, dev, dt), _gain(c, g, dev, dt)
        if c["kind"] == "rotary_grad":
            for n in ("q", "k"):
                s["g" + n] = torch.randn(s[n].shape, generator=g, device=dev).to(dt)
        return s
    new, past = _lengths(c)
    total = [m + p for m, p in zip(new, past)]
    need = [-(-t // c["page"]) for t in total]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=g, device=dev).to(torch.int32)
    owner = torch.arange(c["seqs"], device=dev).repeat_interleave(torch.tensor(need, device=dev), output_size=sum(need))
    ends = torch.tensor([0] + need, device=dev).cumsum(0)
    column = torch.arange(sum(need), device=dev) - ends[owner]
    table = torch.full((c["seqs"], max(need)), -1, dtype=torch.int32, device=dev)
    table[owner, column] = order[:sum(need)]
    s["page_table"] = table
    s["cu_tokens"] = torch.tensor([0] + new, device=dev).cumsum(0).to(torch.int32)
    s["seq_lens"] = torch.tensor(total, dtype=torch.int32, device=dev)
    s["max_new"] = max(new)
    s.update(_cache(c, g, dev, pages))
    t = sum(new)
    s["q"], s["k_new"], s["v_new"] = _projection(c, (t,), g, dev, dt)
    if c["kind"] == "append":
        s["frequencies"] = _frequencies(c, dev)
        s["q_gain"], s["k_gain"] = _gain(c, g, dev, dt), _gain(c, g, dev, dt)
        # the pages that this call writes into, as the program's page allocator knows them
        first = torch.tensor(past, device=dev) // c["page"]
        s["touched"] = table[owner, column][column >= first[owner]].contiguous()
    return s


# ------------------------------------------------------------------------------------------ the plain forms
def _plain_scale(absmax):
    """The smallest power of two that brings absmax to at most E4M3_MAX."""
    m, e = torch.frexp(absmax.double() / E4M3_MAX)
    e = torch.where(m == 0.5, e - 1, e)
    return torch.where(absmax > 0, torch.exp2(e.double()), torch.zeros_like(absmax, dtype=torch.float64)) \
        .clamp_min(MIN_SCALE).float()


def _plain_angles(c, positions, frequencies):
    """cos and sin (..., 1, pairs) in 32 bits of positions (axes, ...), the angles in 64."""
    axis = torch.repeat_interleave(torch.arange(c["axes"], device=positions.device),
                                   torch.tensor(_axis_pairs(c), device=positions.device), output_size=c["rotated"] // 2)
    angle = positions.double()[axis].movedim(0, -1) * frequencies
    return angle.cos().float().unsqueeze(-2), angle.sin().float().unsqueeze(-2)


def _plain_rotate(c, x, cos, sin):
    n, p = c["rotated"], c["rotated"] // 2
    if c["interleaved"]:
        a, b = x[..., 0:n:2], x[..., 1:n:2]
        y = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = x[..., :p], x[..., p:n]
        y = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((y, x[..., n:]), -1)


def _plain_norm(c, x, gain):
    if not c["norm"]:
        return x
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * gain.float()


def _plain_grad(c, x, gain, grad, cos, sin):
    """The gradients of x and of the gain of rotate(norm(x) * gain)."""
    h = _plain_rotate(c, grad, cos, -sin)
    if not c["norm"]:
        return h, None
    r = torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
    xhat, hg = x * r, h * gain.float()
    return r * (hg - xhat * (hg * xhat).mean(-1, keepdim=True)), (h * xhat).flatten(0, -2).sum(0, dtype=torch.float64).float()


def _plain_owner(s):
    """For every new token: its sequence, and its slot in that sequence."""
    cu, lens = s["cu_tokens"].long(), s["seq_lens"].long()
    t = torch.arange(s["q"].shape[0], device=cu.device)
    owner = torch.searchsorted(cu, t, right=True) - 1
    return owner, lens[owner] - cu[owner + 1] + t


def _plain_append(s):
    c = s["case"]
    owner, slot = _plain_owner(s)
    cos, sin = _plain_angles(c, slot[None], s["frequencies"])
    q = _plain_rotate(c, _plain_norm(c, s["q"].float(), s["q_gain"]), cos, sin).to(s["q"].dtype)
    k = _plain_rotate(c, _plain_norm(c, s["k_new"].float(), s["k_gain"]), cos, sin)
    page = s["page_table"][owner, slot // c["page"]].long()
    row = slot % c["page"]
    fresh = torch.zeros(s["k"].shape[0], dtype=torch.bool, device=page.device)
    fresh[page[row == 0]] = True
    pages = s["touched"].long()
    for_page = torch.zeros(s["k"].shape[0], dtype=torch.long, device=page.device)
    for_page[pages] = torch.arange(pages.numel(), device=page.device)
    out = [q]
    for x, code, scale in ((k, s["k"], s["k_scale"]), (s["v_new"].float(), s["v"], s["v_scale"])):
        old = torch.where(fresh[pages, None], torch.zeros_like(scale[pages]), scale[pages])
        top = torch.zeros_like(old).index_reduce_(0, for_page[page], x.abs().amax(-1), "amax")
        now = torch.maximum(old, _plain_scale(top))
        held = code[pages].float()
        moved = (held * (scale[pages] / now)[:, :, None, None]).to(torch.float8_e4m3fn)
        keep = (old == now) | fresh[pages, None]
        blocks = torch.where(keep[:, :, None, None], code[pages].view(torch.uint8), moved.view(torch.uint8))
        blocks[for_page[page], :, row] = (x / now[for_page[page]][:, :, None]).to(torch.float8_e4m3fn).view(torch.uint8)
        code.view(torch.uint8)[pages] = blocks
        scale[pages] = now
        out.append((blocks.view(torch.float8_e4m3fn).float() * now[:, :, None, None]).half())
    return out


def _plain_attention(s):
    c = s["case"]
    hq, hk, d, page = c["q_heads"], c["k_heads"], c["head_dim"], c["page"]
    n, m = s["seq_lens"].numel(), s["max_new"]
    owner, slot = _plain_owner(s)
    t = torch.arange(owner.numel(), device=owner.device) - s["cu_tokens"].long()[owner]
    q = torch.zeros(n, m, hq, d, device=owner.device)
    q[owner, t] = s["q"].float()
    at = torch.full((n, m), -1, dtype=torch.long, device=owner.device)
    at[owner, t] = slot
    pages = s["page_table"].long().clamp_min(0)
    k = (s["k"][pages].float() * s["k_scale"][pages][..., None, None]).permute(0, 2, 1, 3, 4).reshape(n, hk, -1, d)
    v = (s["v"][pages].float() * s["v_scale"][pages][..., None, None]).permute(0, 2, 1, 3, 4).reshape(n, hk, -1, d)
    q = q.reshape(n, m, hk, hq // hk, d).permute(0, 2, 3, 1, 4).reshape(n, hk, -1, d)
    scores = (q @ k.transpose(2, 3)).unflatten(2, (hq // hk, m)) * (1.0 / math.sqrt(d))
    j = torch.arange(k.shape[2], device=owner.device)
    seen = j <= at[..., None]
    if c["window"]:
        seen &= j > at[..., None] - c["window"]
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True).clamp_min(-3e38)
    p = (scores - top).exp()
    total = p.sum(-1, keepdim=True)
    out = ((p / total).flatten(2, 3) @ v).unflatten(2, (hq // hk, m))
    lse = (total.log() + top).squeeze(-1)
    return [out.permute(0, 3, 1, 2, 4).reshape(n, m, hq, d)[owner, t].half(), lse.permute(0, 3, 1, 2).reshape(n, m, hq)[owner, t]]


def _plain(s):
    c = s["case"]
    if c["kind"] == "append":
        return _plain_append(s)
    if c["kind"] == "attention":
        return _plain_attention(s)
    cos, sin = _plain_angles(c, s["positions"], s["frequencies"])
    if c["kind"] == "rotary":
        return [_plain_rotate(c, _plain_norm(c, s[n].float(), s[n + "_gain"]), cos, sin).to(s[n].dtype) for n in ("q", "k")]
    dq, dqg = _plain_grad(c, s["q"].float(), s["q_gain"], s["gq"].float(), cos, sin)
    dk, dkg = _plain_grad(c, s["k"].float(), s["k_gain"], s["gk"].float(), cos, sin)
    out = [dq.to(s["q"].dtype), dk.to(s["k"].dtype)]
    return out + [dqg, dkg] if c["norm"] else out


# ------------------------------------------------------------------------------------------ the framework's calls
@functools.lru_cache(maxsize=1)
def _device():
    import dfdx_b200
    return dfdx_b200.Cuda(torch.cuda.current_device())


def _own(s):
    import dfdx_b200
    c, dev = s["case"], _device()
    if c["kind"] == "attention":
        cache = dfdx_b200.KvCache(s["k"], s["v"], s["k_scale"], s["v_scale"])
        return list(dev.kv_cache_attention(cache, s["q"], s["cu_tokens"], s["seq_lens"], s["page_table"], s["max_new"],
                                           1.0 / math.sqrt(c["head_dim"]), window=c["window"], want_lse=True))
    rotary = dfdx_b200.Rotary(s["frequencies"], _axis_pairs(c), c["interleaved"])
    if c["kind"] == "append":
        cache = dfdx_b200.KvCache(s["k"], s["v"], s["k_scale"], s["v_scale"])
        q = dev.kv_cache_append(cache, s["k_new"], s["v_new"], s["cu_tokens"], s["seq_lens"], s["page_table"], s["max_new"],
                                q=s["q"], rotary=rotary, norm=c["norm"], q_gain=s["q_gain"], k_gain=s["k_gain"], eps=EPS)
        return [q, *dev.kv_cache_read(cache, s["touched"], torch.float16)]
    if c["kind"] == "rotary":
        return list(dev.qk_norm_rotary_forward(s["q"], s["k"], rotary, s["positions"], norm=c["norm"], q_gain=s["q_gain"],
                                               k_gain=s["k_gain"], eps=EPS))
    out = dev.qk_norm_rotary_backward(s["q"], s["k"], s["gq"], s["gk"], rotary, s["positions"], norm=c["norm"],
                                      q_gain=s["q_gain"], k_gain=s["k_gain"], eps=EPS)
    return list(out) if c["norm"] else list(out[:2])


def run(s):
    return _own(s) if own else _plain(s)


# --------------------------------------------------------------------------------------------- in 64 bits
def _exact_turn(c, positions, frequencies):
    """exp(i * angle), (..., 1, pairs), of positions (axes, ...)."""
    parts, at = [], 0
    for a, n in enumerate(_axis_pairs(c)):
        parts.append(positions[a].double()[..., None] * frequencies[at:at + n])
        at += n
    angle = torch.cat(parts, -1)
    return torch.polar(torch.ones_like(angle), angle).unsqueeze(-2)


def _exact_transform(c, x, gain, turn):
    x = x.double() if x.dtype != torch.float64 else x
    if c["norm"]:
        x = x / (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt() * gain
    n = c["rotated"]
    r = x[..., :n]
    z = torch.view_as_complex(r.unflatten(-1, (n // 2, 2)).contiguous()) if c["interleaved"] \
        else torch.complex(r[..., :n // 2].contiguous(), r[..., n // 2:].contiguous())
    z = z * turn
    y = torch.view_as_real(z).flatten(-2) if c["interleaved"] else torch.cat((z.real, z.imag), -1)
    return torch.cat((y, x[..., n:]), -1)


def _exact_e4m3(x):
    """The nearest e4m3 value, ties to the even code: 3 bits behind the leading one, steps of 2^-9 below 2^-6."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -6))) - 3)
    return torch.round(x / step) * step


def _exact_append(s):
    c = s["case"]
    cu, lens, table = s["cu_tokens"].tolist(), s["seq_lens"].tolist(), s["page_table"].tolist()
    place = {p: i for i, p in enumerate(s["touched"].tolist())}
    slots = torch.cat([torch.arange(n - (e - b), n) for b, e, n in zip(cu, cu[1:], lens)]).to(s["q"].device)
    turn = _exact_turn(c, slots[None], s["frequencies"])
    wide = [None if s[n] is None else s[n].double() for n in ("q_gain", "k_gain")]
    q = _exact_transform(c, s["q"], wide[0], turn)
    k = _exact_transform(c, s["k_new"], wide[1], turn)
    out = [q]
    for x, code, scale in ((k, s["k"], s["k_scale"]), (s["v_new"].double(), s["v"], s["v_scale"])):
        held = code[s["touched"].long()].double() * scale[s["touched"].long()].double()[..., None, None]
        for i, (b, e, n) in enumerate(zip(cu, cu[1:], lens)):
            at = n - (e - b)
            while at < n:
                row = at % c["page"]
                m = min(c["page"] - row, n - at)
                w = place[table[i][at // c["page"]]]
                rows = x[b:b + m].transpose(0, 1)                       # (heads, m, d)
                top = rows.abs().amax((1, 2))
                need = torch.exp2(torch.ceil(torch.log2(top / E4M3_MAX))).clamp_min(MIN_SCALE)
                if row:
                    need = torch.maximum(need, scale[table[i][at // c["page"]]].double())
                grown = need > scale[table[i][at // c["page"]]].double()
                need = need[:, None, None]
                if row:
                    held[w] = torch.where(grown[:, None, None], _exact_e4m3(held[w] / need) * need, held[w])
                else:                                                   # what a fresh block holds behind its rows: codes, unread
                    held[w] = code[table[i][at // c["page"]]].double() * need
                held[w][:, row:row + m] = _exact_e4m3(rows / need) * need
                b, at = b + m, at + m
        out.append(held)
    return out


def _exact_attention(s):
    c = s["case"]
    hk, d, w = c["k_heads"], c["head_dim"], c["window"]
    group = c["q_heads"] // hk
    cu, lens = s["cu_tokens"].tolist(), s["seq_lens"].tolist()
    outs, lses = [], []
    for i, (b, e, n) in enumerate(zip(cu, cu[1:], lens)):
        pages = s["page_table"][i, :-(-n // c["page"])].long()
        k, v = ((s[x][pages].double() * s[x + "_scale"][pages].double()[..., None, None]).transpose(0, 1).flatten(1, 2)[:, :n]
                for x in ("k", "v"))
        at, j = torch.arange(n - (e - b), n, device=k.device)[:, None], torch.arange(n, device=k.device)
        mask = (j > at) | (j <= at - w) if w else j > at
        out, lse = [], []
        for h in range(hk):
            q = s["q"][b:e, h * group:(h + 1) * group].double().transpose(0, 1)
            x = (torch.einsum("gmd,nd->gmn", q, k[h]) / d ** 0.5).masked_fill(mask, -math.inf)
            lse.append(torch.logsumexp(x, -1))
            out.append(torch.softmax(x, -1) @ v[h])
        outs.append(torch.cat(out).transpose(0, 1))
        lses.append(torch.cat(lse).transpose(0, 1))
    return [torch.cat(outs), torch.cat(lses)]


def exact(c, seed):
    s = prepare(c, seed)
    if c["kind"] == "append":
        return _exact_append(s)
    if c["kind"] == "attention":
        return _exact_attention(s)
    turn = _exact_turn(c, s["positions"], s["frequencies"])
    if c["kind"] == "rotary":
        return [_exact_transform(c, s[n], None if s[n + "_gain"] is None else s[n + "_gain"].double(), turn) for n in ("q", "k")]
    grads, gains = [], []
    for n in ("q", "k"):
        x = s[n].double().requires_grad_()
        gain = s[n + "_gain"].double().requires_grad_() if c["norm"] else None
        _exact_transform(c, x, gain, turn).backward(s["g" + n].double())
        grads.append(x.grad)
        gains.append(gain.grad if c["norm"] else None)
    return grads + gains if c["norm"] else grads
