"""Per-head norm and rotation of queries and keys, the paged 8-bit cache, and the attention over it, against their
definitions in 64 bits (tests/heads_reference.py).

Tolerances, with u = 2^-24 (f32) and h = half a step of the output's type relative to the value (f16 2^-11, f32 u):
  transform   the row's mean square, reciprocal root, gain, sine and cosine and the pair's two products each lose a few
              u; 64 u = 2^-18 of the row's largest normed magnitude covers them, plus h of the value.
  backward    the same for each factor of r (h g - xhat mean): 2^-17 of the bound below, which adds magnitudes where
              the formula adds values; gains' sums over n rows: (n + 64) u of the sum of magnitudes.
  codes       half an e4m3 step of the exact value (2^-4 of it, 2^-10 of the scale below 2^-6), plus the transform's.
  attention   probabilities rounded to f16 (2^-11 of each), scores wrong by d u alpha sum |q k| and exponentials by
              2^-21: that share of sum w |v|; plus 2^-11 of the value for the output.  A probability p' is held as
              2^14 at the running maximum p'* (which counts its block's value scale in); one below 2^-14 is rounded to
              steps of 2^-24: off by 2^-25 2^-14 p'*.  It meets a code of at most 448 and the sum l >= p'* / sv*, so n
              slots add at most n 2^-39 448 sv* with sv* the largest scale among the visible blocks, itself at most
              2 / 448 of their largest value: n 2^-38 max |v|.
"""
import math

import pytest
import torch

import dfdx_b200
import heads_reference as ref
from dfdx_b200 import _lib

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {torch.float16: 2.0 ** -11, torch.float32: U}
TINY = {torch.float16: 2.0 ** -25, torch.float32: 0.0}
F16, F32 = torch.float16, torch.float32


def gen(seed):
    return torch.Generator().manual_seed(seed)


def within(got, want, tol, what):
    got, tol = got.detach().cpu().double(), torch.as_tensor(tol, dtype=torch.float64)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.equal(got.isnan(), want.isnan()), what
    bad = (got - want).abs() > tol
    bad &= ~(got == want)
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} outside; worst " \
        f"{float((((got - want).abs() / tol.clamp_min(1e-300))[bad]).max()):.3g} times the tolerance"


def out_tol(want, dtype, scale):
    return HALF[dtype] * want.abs() + TINY[dtype] + scale


# ------------------------------------------------------------------------------------------- norm and rotation
# (dtype, batch, tokens, q_heads, k_heads, d, axis_pairs, interleaved, norm, gains, layout)
ROT = [
    (F16, 1, 1, 1, 1, 64, (32,), False, True, True, "fused"),
    (F16, 2, 5, 8, 2, 128, (64,), False, True, True, "fused"),
    (F32, 1, 37, 3, 1, 96, (16, 16, 16), False, True, True, "fused"),
    (F16, 3, 33, 4, 4, 128, (32,), False, True, False, "fused"),        # half of each head rotates
    (F16, 1, 130, 12, 4, 64, (32,), True, True, True, "bhsd"),
    (F32, 2, 9, 2, 2, 256, (128,), True, False, False, "fused"),
    (F16, 2, 11, 5, 1, 80, (20, 20), False, False, False, "fused"),
    (F16, 1, 7, 2, 2, 48, (7, 5), False, True, True, "fused"),          # pairs no multiple of 4: element access
    (F32, 1, 6, 3, 2, 30, (15,), False, True, True, "odd"),             # rows that no vector fits
    (F16, 1, 19, 2, 3, 10, (3,), True, True, True, "odd"),
    (F16, 1, 300, 16, 16, 8, (4,), False, True, True, "fused"),
    (F16, 4, 700, 6, 2, 128, (), False, True, True, "fused"),           # norm alone
    (F32, 1, 2100, 1, 1, 64, (10, 11, 11), False, True, True, "fused"),
    (F16, 1, 16, 4, 0, 64, (32,), False, True, True, "fused"),          # queries alone
]


def rot_inputs(case, seed):
    dtype, b, s, hq, hk, d, axis_pairs, inter, norm, gains, layout = case
    g = gen(seed)
    w = (hq + hk) * d + (1 if layout == "odd" else 0)
    x = torch.randn(b, s, w, generator=g, dtype=torch.float64)
    x = (x * torch.exp(torch.randn(b, s, 1, generator=g, dtype=torch.float64))).to(dtype).cuda()
    if layout == "odd":
        x = x[..., 1:]
    q, k = x[..., :hq * d].unflatten(-1, (hq, d)), x[..., hq * d:].unflatten(-1, (hk, d)) if hk else x[..., :0].reshape(b, s, 0, d)
    if layout == "bhsd":
        q, k = (t.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3) for t in (q, k))
    pos = torch.randint(-50, 1 << 21, (max(len(axis_pairs), 1), b, s), generator=g, dtype=torch.int32)
    f = torch.rand(sum(axis_pairs), generator=g, dtype=torch.float64)
    qg, kg = ((1 + 0.3 * torch.randn(d, generator=g, dtype=torch.float64)).to(dtype).cuda() if gains else None for _ in range(2))
    rotary = dfdx_b200.Rotary(f.cuda(), axis_pairs, inter) if axis_pairs else None
    return q, k, pos, f, qg, kg, rotary, g


def exact_rot(case, x, gain, pos, f):
    _, _, _, _, _, _, axis_pairs, inter, norm, _, _ = case
    a = ref.angles(pos, f, axis_pairs) if axis_pairs else None
    return ref.transform(x, gain, norm, 1e-6, a, inter)


@pytest.mark.parametrize("case", ROT, ids=lambda c: "-".join(str(x).replace("torch.", "") for x in c))
def test_norm_rotary_forward_and_backward(cuda_dev, case):
    dtype, b, s, hq, hk, d, axis_pairs, inter, norm, gains, layout = case
    dev = cuda_dev
    q, k, pos, f, qg, kg, rotary, g = rot_inputs(case, 11)
    dpos = pos.cuda() if rotary is not None else None
    kw = dict(rotary=rotary, positions=dpos, norm=norm, q_gain=qg, k_gain=kg)
    yq, yk = dev.qk_norm_rotary_forward(q, k, **kw)
    goq = torch.randn(q.shape, generator=g, dtype=torch.float64).to(dtype).cuda()
    gok = torch.randn(k.shape, generator=g, dtype=torch.float64).to(dtype).cuda()
    dq, dk, dqg, dkg = dev.qk_norm_rotary_backward(q, k, goq, gok, **kw)
    dev.synchronize()
    for what, x, gain, y, go, dx, dg in (("q", q, qg, yq, goq, dq, dqg), ("k", k, kg, yk, gok, dk, dkg)):
        x64 = x.cpu().double().requires_grad_()
        g64 = torch.ones(d, dtype=torch.float64) if gain is None else gain.cpu().double()
        g64.requires_grad_()
        want = exact_rot(case, x64, g64 if norm else None, pos, f)
        if x.shape[2] == 0:
            assert y.shape == x.shape and (not norm or not bool(dg.any()))
            continue
        size = ref.transform(x64, g64, norm, 1e-6, None, False).detach().abs().amax(-1, keepdim=True)
        within(y, want.detach(), out_tol(want.detach(), dtype, 2.0 ** -18 * size), what)
        want.backward(go.cpu().double())
        go64 = go.cpu().double().abs().amax(-1, keepdim=True) * 1.4143
        r = 1 / (x64.detach().square().mean(-1, keepdim=True) + 1e-6).sqrt() if norm else torch.ones_like(go64)
        xh = (x64.detach() * r).abs().amax(-1, keepdim=True)
        bound = r * go64 * (g64.detach().abs().max() if norm else 1.0) * ((1 + xh * xh) if norm else 1.0)
        within(dx, x64.grad, out_tol(x64.grad, dtype, 2.0 ** -17 * bound), "d" + what)
        if norm:
            sums = (go64 * xh).sum()
            n = b * s * x.shape[2]
            within(dg, g64.grad, ((n + 64) * U + 2.0 ** -18) * sums * torch.ones(d, dtype=torch.float64), f"d{what}_gain")
        else:
            assert dg is None


def test_norm_rotary_gradient_by_differences(cuda_dev):
    """The backward against central differences of the forward, both on the device in f32."""
    dev = cuda_dev
    g = gen(5)
    q, k = (torch.randn(1, 3, h, 32, generator=g).cuda() for h in (2, 1))
    gain = (1 + 0.3 * torch.randn(32, generator=g)).cuda()
    rotary = dfdx_b200.Rotary(dev.rotary_frequencies((8, 4)), (8, 4))
    pos = torch.tensor([[[0, 1, 2]], [[5, 0, 9]]], dtype=torch.int32).cuda()
    w = [torch.randn(t.shape, generator=g).cuda() for t in (q, k)]

    def loss(q_, k_, gain_):
        y = dev.qk_norm_rotary_forward(q_, k_, rotary, pos, q_gain=gain_, k_gain=gain_)
        return sum(float((a.double() * b.double()).sum()) for a, b in zip(y, w))

    dq, dk, dqg, dkg = dev.qk_norm_rotary_backward(q, k, w[0], w[1], rotary, pos, q_gain=gain, k_gain=gain)
    step = 2.0 ** -7
    for t, grad in ((q, dq), (k, dk), (gain, dqg + dkg)):
        for i in range(0, t.numel(), 7):
            hi, lo = t.clone(), t.clone()
            hi.view(-1)[i] += step
            lo.view(-1)[i] -= step
            args = [(hi if t is x else x, lo if t is x else x) for x in (q, k, gain)]
            got = (loss(*(a for a, _ in args)) - loss(*(b for _, b in args))) / (2 * step)
            # second-order differences leave step^2 / 6 of a third derivative of order one, f32 outputs 96 u of sums of 4 / step
            assert abs(got - float(grad.view(-1)[i])) <= 2.0 ** -14 * 16 + 288 * 4 * U / step


def test_norm_rotary_default_positions_in_place_and_broadcast(cuda_dev):
    dev = cuda_dev
    g = gen(6)
    q, k = torch.randn(2, 9, 4, 64, generator=g).half().cuda(), torch.randn(2, 9, 2, 64, generator=g).half().cuda()
    rotary = dfdx_b200.Rotary(dev.rotary_frequencies((32,)), (32,))
    pos = torch.arange(9, dtype=torch.int32).expand(1, 2, 9).contiguous().cuda()
    want = dev.qk_norm_rotary_forward(q, k, rotary, pos)
    assert all(torch.equal(a, b) for a, b in zip(want, dev.qk_norm_rotary_forward(q, k, rotary)))
    shared = k[:, :, :1].expand(2, 9, 4, 64)                             # a broadcast view: one stored head
    y, _ = dev.qk_norm_rotary_forward(shared, k, rotary)
    assert torch.equal(y, want[1][:, :, :1].expand_as(y))
    go = torch.randn(2, 9, 4, 64, generator=g).half().cuda()
    gk = torch.zeros_like(k)
    dense = dev.qk_norm_rotary_backward(shared.contiguous(), k, go, gk, rotary)
    view = dev.qk_norm_rotary_backward(shared, k, go, gk, rotary)
    assert torch.equal(dense[0], view[0]) and torch.equal(dense[2], view[2])
    with pytest.raises(dfdx_b200.B200Error) as e:
        dev.qk_norm_rotary_forward(q, k, rotary, out=(k[:, :, :1].expand(2, 9, 4, 64), k))
    assert e.value.status == _lib.ERR_STRIDE
    a, b = q.clone(), k.clone()
    dev.qk_norm_rotary_forward(a, b, rotary, out=(a, b))
    assert torch.equal(a, want[0]) and torch.equal(b, want[1])
    into = torch.ones(64, device="cuda"), torch.full((64,), 2.0, device="cuda")
    fresh = dev.qk_norm_rotary_backward(q, k, go, gk + 1, rotary)
    again = dev.qk_norm_rotary_backward(q, k, go, gk + 1, rotary, gain_grads=into)
    assert torch.equal(again[2], fresh[2] + 1) and torch.equal(again[3], fresh[3] + 2)


def test_norm_rotary_inf_and_empty(cuda_dev):
    dev = cuda_dev
    x = torch.ones(1, 2, 1, 32).cuda()
    x[0, 0, 0, 31] = math.inf                                            # among elements that pass through
    rotary = dfdx_b200.Rotary(dev.rotary_frequencies((4,)), (4,))
    y, _ = dev.qk_norm_rotary_forward(x, x, rotary, norm=False)
    assert bool(y[0, 0, 0, :31].isfinite().all()) and math.isinf(float(y[0, 0, 0, 31]))
    z = torch.zeros(1, 2, 1, 32).cuda()
    assert not bool(dev.qk_norm_rotary_forward(z, z, rotary)[0].any())   # a row of zeros: eps keeps it finite
    e = torch.empty(0, 5, 2, 32).cuda()
    out = dev.qk_norm_rotary_backward(e, e, e, e, rotary)
    assert out[0].shape == e.shape and not bool(out[2].any()) and not bool(out[3].any())   # sums over nothing


# --------------------------------------------------------------------------------------------------- the cache
class Serving:
    """Sequences in a cache, their pages dealt out of order, stale pages full of NaN."""

    def __init__(self, dev, lens, new, page, heads, d, seed, spare=2):
        self.dev, self.page, self.g = dev, page, gen(seed)
        need = [-(-n // page) for n in lens]
        pages = sum(need) + spare
        self.cache = dev.kv_cache(pages, page, heads, d)
        for t in self.cache[:2]:
            t.view(torch.uint8).fill_(0x7F)
        for t in self.cache[2:]:
            t.fill_(math.nan)
        order = torch.randperm(pages, generator=self.g).tolist()
        self.table = torch.full((len(lens), max(need + [1])), -7, dtype=torch.int32)
        for s, n in enumerate(need):
            self.table[s, :n] = torch.tensor([order.pop() for _ in range(n)], dtype=torch.int32)
        self.lens, self.new = list(lens), list(new)

    def args(self):
        cu = torch.tensor([0] + self.new).cumsum(0).to(torch.int32).cuda()
        return cu, torch.tensor(self.lens, dtype=torch.int32).cuda(), self.table.cuda(), max(self.new + [0])

    def fill(self, lens):
        """Puts random earlier tokens into the cache, through an append."""
        n = sum(lens)
        heads, d = self.cache.k.shape[1], self.cache.k.shape[3]
        if n:
            k, v = (torch.randn(n, heads, d, generator=self.g).half().cuda() for _ in range(2))
            keep = self.lens, self.new
            self.lens, self.new = list(lens), list(lens)
            self.dev.kv_cache_append(self.cache, k, v, *self.args())
            self.lens, self.new = keep

    def rows(self, s, n):
        """The first n slots of sequence s: (n, heads, d) keys and values in f64."""
        pages = self.table[s, :-(-n // self.page)].long()
        out = []
        for code, scale in ((self.cache.k, self.cache.k_scale), (self.cache.v, self.cache.v_scale)):
            x = code.cpu()[pages].double() * scale.cpu()[pages].double()[..., None, None]
            out.append(x.transpose(1, 2).flatten(0, 1)[:n])
        return out


APPEND = [  # dtype, page, heads, q_heads, d, past, new, pairs, interleaved, norm
    (F16, 16, 1, 1, 32, [0], [1], 16, False, True),
    (F16, 64, 8, 32, 128, [63, 64, 65, 0, 1000], [1, 1, 1, 1, 1], 64, False, True),
    (F32, 32, 2, 6, 96, [0, 5, 31, 32], [70, 1, 33, 0], 24, True, True),
    (F16, 128, 4, 4, 64, [0, 100, 127, 3], [300, 28, 2, 129], 32, False, False),
    (F16, 16, 3, 3, 128, [7, 0, 15, 16, 17], [0, 0, 40, 16, 3], 0, False, False),
    (F32, 64, 2, 4, 128, [10], [200], 30, False, True),                  # pairs no multiple of 4
    (F16, 16, 5, 10, 64, [7 * i % 50 for i in range(100)], [1] * 100, 32, False, True),            # several heads a CTA, the
    (F16, 16, 7, 7, 96, [5 * i % 33 for i in range(60)], [1 + 11 * i % 37 for i in range(60)], 48, False, True),  # last fewer
    (F32, 32, 3, 3, 64, [3 * i % 40 for i in range(70)], [1 + 13 * i % 50 for i in range(70)], 16, True, False),
]


@pytest.mark.parametrize("case", APPEND, ids=lambda c: "-".join(str(x).replace("torch.", "") for x in c)[:80])
def test_append(cuda_dev, case):
    dtype, page, heads, hq, d, past, new, pairs, inter, norm = case
    dev = cuda_dev
    lens = [a + b for a, b in zip(past, new)]
    sv = Serving(dev, lens, new, page, heads, d, 21)
    sv.fill(past)
    before = [sv.rows(s, p) for s, p in enumerate(past)]
    scales = [t.cpu().double() for t in sv.cache[2:]]
    held = [t.view(torch.uint8).cpu() for t in sv.cache[:2]]
    g, t = sv.g, sum(new)
    grow = torch.exp(2 * torch.randn(t, 1, 1, generator=g))              # some rows far larger than what the block holds
    q, k, v = ((torch.randn(t, h, d, generator=g) * grow).to(dtype).cuda() for h in (hq, heads, heads))
    qg, kg = ((1 + 0.3 * torch.randn(d, generator=g)).to(dtype).cuda() if norm else None for _ in range(2))
    f = torch.rand(pairs, generator=g, dtype=torch.float64)
    rotary = dfdx_b200.Rotary(f.cuda(), (pairs,), inter) if pairs else None
    y = dev.kv_cache_append(sv.cache, k, v, *sv.args(), q=q, rotary=rotary, norm=norm, q_gain=qg, k_gain=kg)
    dev.synchronize()
    slots = torch.cat([torch.arange(p, p + m) for p, m in zip(past, new)])
    angle = ref.angles(slots[None], f, (pairs,)) if pairs else None

    def exact(x, gain):
        return ref.transform(x.cpu().double(), None if gain is None else gain.cpu().double(), norm, 1e-6, angle, inter)

    wq, wk, wv = exact(q, qg), exact(k, kg), v.cpu().double()
    size = ref.transform(q.cpu().double(), None if qg is None else qg.cpu().double(), norm, 1e-6, None, False).abs().amax(-1, keepdim=True)
    within(y, wq, out_tol(wq, dtype, 2.0 ** -18 * size), "q")
    at = 0
    touched = set()
    for s, (p, m) in enumerate(zip(past, new)):
        after = sv.rows(s, p + m)
        for c, want in enumerate((wk, wv)):
            scale = sv.cache[2 + c].cpu().double()
            for col in range(p // page, -(-(p + m) // page) if m else 0):
                pid, a, b = int(sv.table[s, col]), max(p, col * page), min(p + m, (col + 1) * page)
                touched.add(pid)
                rows = want[at + a - p:at + b - p]
                old = scales[c][pid] if a % page else torch.zeros(heads, dtype=torch.float64)
                top, now = rows.abs().amax((0, 2)), scale[pid]
                lo, hi = (torch.maximum(old, ref.scale_for(top * (1 + sgn * 2.0 ** -18))) for sgn in (-1, 1))
                assert bool(((now == lo) | (now == hi)).all()), (s, c, col)
                got = after[c][a:b]
                tol = torch.maximum(2.0 ** -4 * rows.abs(), 2.0 ** -10 * now[None, :, None]) * (1 + 2.0 ** -18) \
                    + 2.0 ** -18 * rows.abs().amax(-1, keepdim=True)
                within(got, rows, tol, f"codes {s} {c} {col}")
                if a % page:                                             # earlier rows of the block: exactly moved
                    first = col * page
                    kept = before[s][c][first:a]
                    want_old = torch.where((now > old)[None, :, None], ref.e4m3(kept / now[None, :, None]) * now[None, :, None], kept)
                    assert torch.equal(after[c][first:a], want_old)
        first = min(p // page * page, p)
        for c in range(2):
            assert torch.equal(after[c][:first], before[s][c][:first])
        at += m
    for c in range(2):                                                   # pages that no new token lies in are untouched
        same = torch.tensor([i not in touched for i in range(sv.cache.k.shape[0])])
        assert torch.equal(sv.cache[c].view(torch.uint8).cpu()[same], held[c][same])
    assert dev.device_status() == 0


def test_read_gives_codes_times_scales(cuda_dev):
    dev = cuda_dev
    sv = Serving(dev, [100, 33], [0, 0], 32, 3, 96, 31, spare=0)
    sv.fill([100, 33])
    pages = torch.tensor([5, 0, 0, 3], dtype=torch.int32)
    for dtype in (F16, F32):
        got = dev.kv_cache_read(sv.cache, pages.cuda(), dtype)
        for c in range(2):
            want = (sv.cache[c].cpu()[pages.long()].float() * sv.cache[2 + c].cpu()[pages.long()][..., None, None]).to(dtype)
            assert torch.equal(got[c].cpu().nan_to_num(7.0), want.nan_to_num(7.0))
    assert dev.device_status() == 0


def test_append_with_positions_of_three_axes(cuda_dev):
    """Positions given by the caller, and cu_tokens, seq_lens and a page table that are views."""
    dev = cuda_dev
    sv = Serving(dev, [20, 7], [13, 7], 16, 2, 64, 42)
    sv.fill([7, 0])
    g = sv.g
    q, k, v = (torch.randn(20, h, 64, generator=g).half().cuda() for h in (4, 2, 2))
    pos = torch.randint(-9, 5000, (3, 20), generator=g, dtype=torch.int32)
    f = torch.rand(30, generator=g, dtype=torch.float64)
    rotary = dfdx_b200.Rotary(f.cuda(), (12, 10, 8), True)
    cu, lens, table, most = sv.args()
    wide = torch.full((2, table.shape[1] + 3), -1, dtype=torch.int32, device="cuda")
    wide[:, 2:2 + table.shape[1]] = table
    y = dev.kv_cache_append(sv.cache, k, v, torch.cat([cu, cu])[:3], torch.cat([lens, lens])[2:], wide[:, 2:2 + table.shape[1]], most,
                            q=q, rotary=rotary, positions=pos.cuda())
    angle = ref.angles(pos, f, (12, 10, 8))
    size = lambda x: x.abs().amax(-1, keepdim=True) * 1.4143
    q64, k64 = q.cpu().double(), k.cpu().double()
    want = ref.transform(q64, None, False, 0.0, angle, True)
    within(y, want, out_tol(want, F16, 2.0 ** -18 * size(q64)), "q")
    want = ref.transform(k64, None, False, 0.0, angle, True)
    scale = sv.cache.k_scale.cpu().double()
    for s, (a, b, n) in enumerate(((0, 13, 20), (13, 20, 7))):
        got = sv.rows(s, n)[0][n - (b - a):]
        blocks = torch.stack([scale[int(sv.table[s, i // 16])] for i in range(n - (b - a), n)])[..., None]
        tol = torch.maximum(2.0 ** -4 * want[a:b].abs(), 2.0 ** -10 * blocks) * (1 + 2.0 ** -18) + 2.0 ** -18 * size(k64[a:b])
        within(got, want[a:b], tol, f"codes {s}")
    assert dev.device_status() == 0


def test_append_padded_batches_of_single_tokens(cuda_dev):
    """Sequences without a new token before those with one, tokens of no sequence behind: as many tokens as sequences."""
    dev = cuda_dev
    sv = Serving(dev, [5, 40, 17, 3, 64, 9], [0, 1, 1, 0, 1, 1], 16, 2, 64, 47)
    sv.fill([5, 39, 16, 3, 63, 8])
    q = torch.randn(6, 4, 64, generator=sv.g).half().cuda()
    k, v = (torch.randn(6, 2, 64, generator=sv.g).half().cuda() for _ in range(2))
    rotary = dfdx_b200.Rotary(dev.rotary_frequencies((32,)), (32,))
    out = torch.full_like(q, 7.0)
    dev.kv_cache_append(sv.cache, k, v, *sv.args(), q=q, rotary=rotary, q_out=out)
    assert bool((out[4:] == 7.0).all())
    pos = torch.tensor([[39, 16, 63, 8]], dtype=torch.int32).cuda()[:, None]
    want, _ = dev.qk_norm_rotary_forward(q[None, :4], k[None, :4], rotary, pos, norm=False)
    assert torch.equal(out[:4], want[0])
    for s, tok in ((1, 0), (2, 1), (4, 2), (5, 3)):
        got = sv.rows(s, sv.lens[s])[1][-1]
        held = sv.cache.v_scale.cpu().double()[int(sv.table[s, (sv.lens[s] - 1) // 16])]
        within(got, v[tok].cpu().double(), torch.maximum(2.0 ** -4 * v[tok].cpu().double().abs(), 2.0 ** -10 * held[:, None]), f"values {s}")
    assert dev.device_status() == 0


def test_append_reports_bounds_that_do_not_fit(cuda_dev):
    dev = cuda_dev
    sv = Serving(dev, [10, 10, 10], [2, 2, 2], 16, 1, 32, 43)
    sv.fill([8, 8, 8])
    cu, lens, table, most = sv.args()
    x = torch.randn(6, 1, 32, generator=sv.g).half().cuda()
    good = torch.full_like(x, 7.0)
    for bad_cu, bad_lens in (([0, 2, 1, 6], None), ([0, 2, 9, 6], None), ([-1, 2, 4, 6], None), (None, [10, 1, 10]), (None, [10, 17, 10]), (None, [10, -3, 10])):
        held = [t.view(torch.uint8).clone() for t in sv.cache[:2]]
        c = torch.tensor(bad_cu, dtype=torch.int32).cuda() if bad_cu else cu
        n = torch.tensor(bad_lens, dtype=torch.int32).cuda() if bad_lens else lens
        dev.kv_cache_append(sv.cache, x, x, c, n, table, most, q=x, q_out=good)
        assert dev.device_status() == _lib.ERR_INDEX
        if bad_lens:                                                      # the other sequences' pages are written, this one's not
            page = int(sv.table[1, 0])
            assert all(torch.equal(a[page], b.view(torch.uint8)[page]) for a, b in zip(held, sv.cache[:2]))
    dev.kv_cache_append(sv.cache, x, x, cu, lens, table, most)
    assert dev.device_status() == 0


def test_append_infinities_nan_zeros(cuda_dev):
    """An infinity is held as the block's largest code and does not set its scale, NaN stays NaN, zeros get the least scale."""
    dev = cuda_dev
    sv = Serving(dev, [3, 1], [3, 1], 16, 1, 32, 41)
    k = torch.zeros(4, 1, 32)
    k[0, 0, :4] = torch.tensor([1.0, math.inf, -math.inf, math.nan])
    k[1, 0, :2] = torch.tensor([3.5, -448.0])
    dev.kv_cache_append(sv.cache, k.cuda(), torch.zeros(4, 1, 32).cuda(), *sv.args())
    rows = sv.rows(0, 3)[0][:, 0]
    assert rows[0, :3].tolist() == [1.0, 448.0, -448.0] and math.isnan(rows[0, 3]) and rows[1, :2].tolist() == [3.5, -448.0]
    assert float(sv.cache.k_scale[int(sv.table[0, 0]), 0]) == 1.0
    assert float(sv.cache.k_scale[int(sv.table[1, 0]), 0]) == ref.MIN_SCALE
    assert float(sv.cache.v_scale[int(sv.table[0, 0]), 0]) == ref.MIN_SCALE


def check_attention(dev, sv, q, out, lse, alpha, causal=True, window=0):
    at = 0
    d = q.shape[2]
    for s, (n, m) in enumerate(zip(sv.lens, sv.new)):
        if m == 0:
            continue
        k, v = sv.rows(s, n)
        pos = torch.arange(n - m, n)[:, None]
        j = torch.arange(n)[None]
        vis = (j <= pos) if causal else torch.ones(m, n, dtype=torch.bool)
        if window:
            vis = vis & (j > pos - window)
        q64 = q[at:at + m].cpu().double()
        want, wlse, size = ref.attention(q64, k, v, alpha, vis)
        score = abs(alpha) * d * U * (q64.abs().amax((0, 2)).max() * (k.nan_to_num(0.0).abs().sum(-1).max() if n else 0.0)) / math.sqrt(d) * 8
        big = v.nan_to_num(0.0).abs().max() if n else 0.0
        tol = (2.0 ** -11 + 2 * score + 2.0 ** -20) * size + 2.0 ** -11 * want.abs() + n * 2.0 ** -38 * big + 2.0 ** -25
        within(out[at:at + m], want, tol, f"sequence {s}")
        if lse is not None:
            within(lse[at:at + m], wlse, 2 * score + 2.0 ** -19 + 4 * U * wlse.abs().nan_to_num(0, 0, 0), f"lse {s}")
        at += m


ATT = [  # page, heads, q_heads, d, past, new, causal, window
    (16, 1, 1, 32, [0], [1], True, 0),
    (64, 2, 8, 64, [899, 0, 63, 64, 15], [1, 1, 1, 1, 1], True, 0),
    (64, 8, 32, 128, [2000, 1, 130, 555], [1, 1, 1, 1], True, 0),
    (16, 2, 8, 96, [40, 300, 7, 0], [3, 5, 1, 2], True, 0),
    (32, 1, 20, 128, [257, 1000], [1, 2], True, 0),                      # more rows than one matrix tile
    (16, 2, 8, 64, [400, 20, 1500, 0], [4, 3, 1, 2], True, 33),
    (128, 2, 4, 128, [700, 100], [0, 5], True, 128),
    (64, 4, 4, 64, [100, 0, 300], [7, 20, 0], False, 0),
    (64, 1, 4, 128, [0, 200], [150, 301], True, 0),                      # prompts
    (16, 2, 12, 96, [37], [203], True, 50),
    (32, 3, 6, 32, [0, 64, 5], [129, 64, 40], True, 0),
    (128, 1, 8, 128, [9000], [1], True, 0),
    (16, 2, 8, 64, [500, 0, 77, 1200], [1, 300, 9, 5], True, 0),         # few and many rows in one batch
    (64, 1, 8, 128, [9000, 3], [40, 33], True, 0),                       # many rows over ranges that are joined
    (32, 1, 16, 96, [6000], [60], True, 2500),
    (128, 2, 32, 64, [3000, 5000], [3, 40], False, 0),
    (16, 8, 32, 32, [100, 5, 700, 0], [900, 3, 500, 0], True, 0),        # more row tiles than SMs, of uneven length
    (64, 1, 40, 32, [300], [1], True, 0),                                # one token, more heads than a small tile's rows
]


@pytest.mark.parametrize("case", ATT, ids=lambda c: "-".join(map(str, c)))
def test_attention(cuda_dev, case):
    page, heads, hq, d, past, new, causal, window = case
    dev = cuda_dev
    sv = Serving(dev, [a + b for a, b in zip(past, new)], new, page, heads, d, 51)
    sv.fill(sv.lens)
    q = torch.randn(sum(new) + 3, hq, d, generator=sv.g).half().cuda()    # rows behind the last sequence
    out = torch.full_like(q, 7.0)
    alpha = 1.0 / math.sqrt(d)
    _, lse = dev.kv_cache_attention(sv.cache, q, *sv.args(), alpha, causal=causal, window=window, out=out, want_lse=True)
    dev.synchronize()
    check_attention(dev, sv, q, out, lse, alpha, causal, window)
    assert bool((out[sum(new):] == 7.0).all())
    again, lse2 = dev.kv_cache_attention(sv.cache, q, *sv.args(), alpha, causal=causal, window=window, want_lse=True)
    assert torch.equal(again[:sum(new)], out[:sum(new)]) and torch.equal(lse2[:sum(new)], lse[:sum(new)])
    assert dev.device_status() == 0


@pytest.mark.parametrize("new", [1, 40])
def test_attention_scores_far_apart_and_scales_far_apart(cuda_dev, new):
    """Scores of several hundred, and blocks whose value scales differ by 2^30: the running maximum carries both."""
    dev = cuda_dev
    sv = Serving(dev, [200, 100], [0, 0], 16, 2, 64, 61)
    k = (8 * torch.randn(300, 2, 64, generator=sv.g)).half().cuda()
    size = torch.exp2(torch.randint(-15, 16, (300, 1, 1), generator=sv.g).float().repeat_interleave(16, 0)[:300])
    v = (torch.randn(300, 2, 64, generator=sv.g) * size).cuda()
    sv.new = [200, 100]
    dev.kv_cache_append(sv.cache, k.float(), v, *sv.args())
    sv.new = [new, new]
    q = (4 * torch.randn(2 * new, 4, 64, generator=sv.g)).half().cuda()
    for alpha in (0.125, 1.0, -0.5):
        out, lse = dev.kv_cache_attention(sv.cache, q, *sv.args(), alpha, want_lse=True)
        at = 0
        for s in range(2):
            n = sv.lens[s]
            kk, vv = sv.rows(s, n)
            vis = torch.arange(n)[None] <= torch.arange(n - new, n)[:, None]
            want, wlse, sz = ref.attention(q[at:at + new].cpu().double(), kk, vv, alpha, vis)
            # scores reach 64 * 32 * 40 alpha: 64 u of that is their error, and e^error the weights'
            err = 64 * U * abs(alpha) * float((q.cpu().double().abs().amax() * kk.abs().sum(-1).amax()))
            fine = want.abs() < 60000
            within(torch.where(fine, out[at:at + new].cpu().double(), 0.0), torch.where(fine, want, 0.0),
                   (2.0 ** -11 + 2 * err) * sz + 2.0 ** -11 * want.abs() + 2.0 ** -25 + n * 2.0 ** -38 * float(vv.abs().max()), f"{alpha} {s}")
            within(lse[at:at + new], wlse, 2 * err + 2.0 ** -19 + 4 * U * wlse.abs(), f"lse {alpha} {s}")
            at += new
    assert dev.device_status() == 0


@pytest.mark.parametrize("new", [3, 45])
def test_attention_nan_in_slots_that_a_row_does_not_see(cuda_dev, new):
    """NaN keys and values at a late slot reach the rows that see them and no others."""
    dev = cuda_dev
    n = 100 + new
    sv = Serving(dev, [n], [n], 16, 1, 64, 71)
    k, v = (torch.randn(n, 1, 64, generator=sv.g) for _ in range(2))
    v[n - 2, 0, 5] = math.nan
    k[n - 1, 0, 3] = math.nan
    dev.kv_cache_append(sv.cache, k.cuda(), v.cuda(), *sv.args())
    sv.new = [new]
    q = torch.randn(new, 2, 64, generator=sv.g).half().cuda()
    out, lse = dev.kv_cache_attention(sv.cache, q, *sv.args(), 0.125, want_lse=True)
    out, lse = out.cpu(), lse.cpu()
    assert bool(out[:new - 2].isfinite().all()) and bool(lse[:new - 1].isfinite().all())
    nan = out[new - 2].isnan()
    assert bool(nan[:, 5].all()) and int(nan.sum()) == 2                  # the column whose value is NaN
    assert bool(out[new - 1].isnan().all()) and bool(lse[new - 1].isnan().all())


@pytest.mark.parametrize("new", [(3, 43, 20), (0, 2, 48), (16, 17, 50)])
def test_attention_of_a_padded_batch(cuda_dev, new):
    """As many tokens as sequences of the longest length would have, though some are short: the rest belongs to none."""
    dev = cuda_dev
    sv = Serving(dev, [a + b for a, b in zip((70, 5, 200), new)], new, 16, 2, 64, 57)
    sv.fill(sv.lens)
    q = torch.randn(3 * max(new), 4, 64, generator=sv.g).half().cuda()
    out = torch.full_like(q, 7.0)
    _, lse = dev.kv_cache_attention(sv.cache, q, *sv.args(), 0.125, out=out, want_lse=True)
    check_attention(dev, sv, q, out, lse, 0.125)
    assert bool((out[sum(new):] == 7.0).all())
    assert dev.device_status() == 0


def test_lengths_above_the_limit_are_reported(cuda_dev):
    dev = cuda_dev
    cache = dev.kv_cache(1, 128, 1, 32)
    x = torch.ones(1, 1, 32).half().cuda()
    table = torch.zeros(1, (1 << 23) + 2, dtype=torch.int32, device="cuda")
    cu, one, long = (torch.tensor(t, dtype=torch.int32).cuda() for t in ([0, 1], [1], [(1 << 30) + 1]))
    dev.kv_cache_append(cache, x, x, cu, one, table, 1)
    assert dev.device_status() == 0
    out = torch.full_like(x, 7.0)
    dev.kv_cache_append(cache, x + 1, x, cu, long, table, 1)
    assert dev.device_status() == _lib.ERR_INDEX
    dev.kv_cache_attention(cache, x, cu, long, table, 1, 1.0, window=16, out=out)
    assert dev.device_status() == _lib.ERR_INDEX and bool((out == 7.0).all())
    dev.kv_cache_attention(cache, x, cu, one, table, 1, 1.0, out=out)
    assert dev.device_status() == 0 and bool((out == 1.0).all())


def test_attention_strides_and_empty_rows(cuda_dev):
    dev = cuda_dev
    sv = Serving(dev, [0, 50, 0], [2, 3, 0], 16, 2, 64, 81)              # two queries before anything is in the cache
    sv.fill([0, 50, 0])
    x = torch.randn(5, 9, 80, generator=sv.g).half().cuda()
    q = x[:, 1:9, 8:72]
    buf = torch.full((8, 5, 72), 3.0, dtype=F16, device="cuda")
    out = buf.permute(1, 0, 2)[..., :64]
    _, lse = dev.kv_cache_attention(sv.cache, q, *sv.args(), 0.125, out=out, want_lse=True)
    assert not bool(out[:2].any()) and bool((lse[:2] == -math.inf).all())
    sv.lens, sv.new = [50], [3]
    sv.table = sv.table[1:2]
    check_attention(dev, sv, q[2:], out[2:], lse[2:], 0.125)
    assert bool((buf[..., 64:] == 3.0).all())
    assert dev.device_status() == 0


def test_bad_pages_and_lengths_are_skipped_and_reported(cuda_dev):
    """What the device arrays hold is checked where it is read: nothing out of range is touched, the others' results stand."""
    dev = cuda_dev
    sv = Serving(dev, [40, 40, 40], [1, 1, 1], 16, 1, 64, 91)
    sv.fill([40, 40, 40])
    q = torch.randn(3, 2, 64, generator=sv.g).half().cuda()
    good, _ = dev.kv_cache_attention(sv.cache, q, *sv.args(), 0.125)
    assert dev.device_status() == 0
    held = [t.view(torch.uint8).clone() for t in sv.cache[:2]]
    cu, lens, table, m = sv.args()
    for page in (-1, 1 << 20, -(1 << 31)):
        bad = table.clone()
        bad[1, 2] = page
        out, _ = dev.kv_cache_attention(sv.cache, q, cu, lens, bad, m, 0.125)
        assert dev.device_status() == _lib.ERR_INDEX
        assert torch.equal(out[0], good[0]) and torch.equal(out[2], good[2])
        x = torch.randn(3, 1, 64).half().cuda()
        only = torch.tensor([0, 0, 1, 1], dtype=torch.int32).cuda()
        dev.kv_cache_append(sv.cache, x, x, only, lens, bad, m)
        assert dev.device_status() == _lib.ERR_INDEX
        assert all(torch.equal(a, b.view(torch.uint8)) for a, b in zip(held, sv.cache[:2]))
        k, _ = dev.kv_cache_read(sv.cache, torch.tensor([page], dtype=torch.int32).cuda())
        assert dev.device_status() == _lib.ERR_INDEX and not bool(k.any())
    for bad_lens, bad_cu in (([40, 49, 40], None), ([40, -1, 40], None), (None, [0, 1, 5, 3]), (None, [0, 1, -4, 3]), (None, [0, 1, 3, 3])):
        l2 = torch.tensor(bad_lens, dtype=torch.int32).cuda() if bad_lens else lens
        c2 = torch.tensor(bad_cu, dtype=torch.int32).cuda() if bad_cu else cu
        out, _ = dev.kv_cache_attention(sv.cache, q, c2, l2, table, m, 0.125)
        assert dev.device_status() == _lib.ERR_INDEX
        assert torch.equal(out[0], good[0])
    assert dev.device_status() == 0


def test_cache_larger_than_32_bit_offsets(cuda_dev):
    dev = cuda_dev
    pages = (1 << 31) // (8 * 128 * 128) + 40
    cache = dev.kv_cache(pages, 128, 8, 128)
    n, g = 300, gen(101)
    k, v = (torch.randn(n, 8, 128, generator=g).half().cuda() for _ in range(2))
    table = torch.tensor([[pages - 1, 0, pages - 3]], dtype=torch.int32).cuda()
    cu, lens = torch.tensor([0, n], dtype=torch.int32).cuda(), torch.tensor([n], dtype=torch.int32).cuda()
    dev.kv_cache_append(cache, k, v, cu, lens, table, n)
    q = torch.randn(1, 16, 128, generator=g).half().cuda()
    one = torch.tensor([0, 1], dtype=torch.int32).cuda()
    out, _ = dev.kv_cache_attention(cache, q, one, lens, table, 1, 0.1)
    small = dev.kv_cache(3, 128, 8, 128)
    near = torch.tensor([[0, 1, 2]], dtype=torch.int32).cuda()
    dev.kv_cache_append(small, k, v, cu, lens, near, n)
    want, _ = dev.kv_cache_attention(small, q, one, lens, near, 1, 0.1)
    assert torch.equal(out, want)
    a, b = dev.kv_cache_read(cache, table[0]), dev.kv_cache_read(small, near[0])
    for x, y in zip(a, b):                                               # 300 slots: the third page holds 44
        assert torch.equal(x[:2], y[:2]) and torch.equal(x[2, :, :44], y[2, :, :44])
    assert dev.device_status() == 0


def test_refusals_of_the_python_layer(cuda_dev):
    dev = cuda_dev
    sv = Serving(dev, [40], [1], 16, 2, 64, 111)
    q = torch.zeros(1, 4, 64, dtype=F16, device="cuda")
    k = torch.zeros(1, 2, 64, dtype=F16, device="cuda")
    cu, lens, table, m = sv.args()
    for error, call in (
            (dfdx_b200.ShapeMismatch, lambda: dev.kv_cache_attention(sv.cache, q[:, :3], cu, lens, table, m, 1.0)),
            (dfdx_b200.B200Error, lambda: dev.kv_cache_attention(sv.cache, q.float(), cu, lens, table, m, 1.0)),
            (TypeError, lambda: dev.kv_cache_attention(sv.cache, q, cu.long(), lens, table, m, 1.0)),
            (dfdx_b200.ShapeMismatch, lambda: dev.kv_cache_attention(sv.cache, q, cu[:1], lens, table, m, 1.0)),
            (ValueError, lambda: dev.kv_cache_attention(sv.cache, q, cu.cpu(), lens, table, m, 1.0)),
            (dfdx_b200.B200Error, lambda: dev.kv_cache_attention(sv.cache, q, cu, lens, table, m, 1.0, causal=False, window=4)),
            (dfdx_b200.ShapeMismatch, lambda: dev.kv_cache_append(sv.cache, q, q, cu, lens, table, m)),
            (TypeError, lambda: dev.kv_cache_append(sv.cache, k, k.float(), cu, lens, table, m)),
            (ValueError, lambda: dev.kv_cache_append(sv.cache, k, k, cu, lens, table, m, k_gain=k[0, 0])),
            (TypeError, lambda: dev.kv_cache_append(sv.cache, k, k, cu, lens, table, m, rotary=dfdx_b200.Rotary(torch.zeros(4, device="cuda"), (4,)))),
            (dfdx_b200.ShapeMismatch, lambda: dev.kv_cache_append(sv.cache, k, k, cu, lens, table, m,
                                                                  rotary=dfdx_b200.Rotary(dev.rotary_frequencies((4,)), (3,)))),
            (TypeError, lambda: dev.kv_cache_read(sv.cache, table[0], torch.float64)),
            (dfdx_b200.ShapeMismatch, lambda: dev.qk_norm_rotary_forward(q[None], k[None, :, :, :32])),
            (TypeError, lambda: dev.qk_norm_rotary_forward(q[None].double(), k[None].double())),
    ):
        with pytest.raises(error):
            call()
    assert dev.device_status() == 0


# ------------------------------------------------------------------------------------------------- together
def test_a_step_of_serving(cuda_dev):
    """Prompts, then two decoded tokens each: projection, append with norm and rotation, attention, as a decoder's layer
    runs them, with the decoding step captured once and replayed with the next lengths."""
    dev = cuda_dev
    g = gen(121)
    hq, hk, d, width = 8, 2, 64, 256
    prompts = [70, 5, 129]
    w = (torch.randn((hq + 2 * hk) * d, width, generator=g) / 16).half().cuda()
    gain = (1 + 0.2 * torch.randn(d, generator=g)).half().cuda()
    rotary = dfdx_b200.Rotary(dev.rotary_frequencies((32,)), (32,))
    sv = Serving(dev, [n + 2 for n in prompts], prompts, 16, hk, d, 122)

    def step(x, cu, lens, table, most):
        y = dev.linear_forward(x[None], w.permute(1, 0))[0]
        q, k, v = y[:, :hq * d].unflatten(1, (hq, d)), y[:, hq * d:(hq + hk) * d].unflatten(1, (hk, d)), y[:, (hq + hk) * d:].unflatten(1, (hk, d))
        q = dev.kv_cache_append(sv.cache, k, v, cu, lens, table, most, q=q, rotary=rotary, norm=True, q_gain=gain, k_gain=gain)
        return q, *dev.kv_cache_attention(sv.cache, q, cu, lens, table, most, 0.125, want_lse=True)

    sv.lens = list(prompts)
    q, out, lse = step(torch.randn(sum(prompts), width, generator=g).half().cuda(), *sv.args())
    dev.synchronize()
    check_attention(dev, sv, q, out, lse, 0.125)
    sv.new = [1, 1, 1]
    sv.lens = [n + 1 for n in prompts]
    x = torch.randn(3, width, generator=g).half().cuda()
    cu, lens, table, most = sv.args()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(x, cu, lens, table, most)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q, out, lse = step(x, cu, lens, table, most)
    for extra in (1, 2):
        sv.lens = [n + extra for n in prompts]
        lens.copy_(torch.tensor(sv.lens, dtype=torch.int32))
        x.copy_(torch.randn(3, width, generator=g).half())
        graph.replay()
        dev.synchronize()
        check_attention(dev, sv, q, out, lse, 0.125)
    assert dev.device_status() == 0


def test_calls_on_two_streams_and_in_two_graphs(cuda_dev):
    """Calls that run at the same time, and graphs that are replayed in turn, each have their own partial results."""
    dev = cuda_dev
    cases = []
    for seed, (page, heads, hq, d, past, new) in enumerate(((64, 2, 8, 128, [6000], [1]), (16, 2, 8, 64, [700, 4000], [40, 50]), (32, 1, 4, 96, [5000], [3]))):
        sv = Serving(dev, [a + b for a, b in zip(past, new)], new, page, heads, d, 140 + seed)
        sv.fill(sv.lens)
        cases.append((sv, torch.randn(sum(new), hq, d, generator=sv.g).half().cuda(), sv.args()))
    q, k = torch.randn(4, 200, 6, 64).half().cuda(), torch.randn(4, 200, 2, 64).half().cuda()
    rotary = dfdx_b200.Rotary(dev.rotary_frequencies((32,)), (32,))

    def run(i):
        if i == 3:
            return dev.qk_norm_rotary_backward(q, k, q, k, rotary)
        sv, x, args = cases[i]
        return dev.kv_cache_attention(sv.cache, x, *args, 0.1, want_lse=True)

    want = [run(i) for i in range(4)]
    dev.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    got = [[] for _ in range(4)]
    for _ in range(8):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(run(i))
    torch.cuda.synchronize()
    for i in range(4):
        for g in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(g, want[i]))
    graphs, outs = [], []
    for i in range(4):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(run(i))
        graphs.append(gr)
    for i in (0, 1, 2, 3, 3, 2, 1, 0, 2, 0, 3, 1):
        graphs[i].replay()
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert all(torch.equal(a, b) for a, b in zip(o, w))
    assert dev.device_status() == 0


def test_a_step_of_training(cuda_dev, oracle):
    """Norm and rotation in front of the fused attention, forward and backward, against autograd in 64 bits."""
    dev = cuda_dev
    g = gen(131)
    b, s, h, d = 2, 150, 4, 64
    x = torch.randn(b, s, 3 * h * d, generator=g).half().cuda()
    q, k, v = (x[..., i * h * d:(i + 1) * h * d].unflatten(-1, (h, d)) for i in range(3))
    gain = (1 + 0.2 * torch.randn(2, d, generator=g)).half().cuda()
    rotary = dfdx_b200.Rotary(dev.rotary_frequencies((32,)), (32,))
    yq, yk = dev.qk_norm_rotary_forward(q, k, rotary, q_gain=gain[0], k_gain=gain[1])
    views = yq.permute(0, 2, 1, 3), yk.permute(0, 2, 3, 1), v.permute(0, 2, 1, 3)
    out, lse = dev.attention_forward(*views, 0.125, want_lse=True)
    go = torch.randn(b, s, h, d, generator=g).half().cuda().permute(0, 2, 1, 3)
    gx = torch.empty_like(x)
    into = gx.unflatten(-1, (3, h, d))
    dyq, dyk = torch.empty_like(yq), torch.empty_like(yk)
    dev.attention_backward(*views, 0.125, out, lse, go,
                           write_into=(dyq.permute(0, 2, 1, 3), dyk.permute(0, 2, 3, 1), into[:, :, 2].permute(0, 2, 1, 3)))
    _, _, gq, gk = dev.qk_norm_rotary_backward(q, k, dyq, dyk, rotary, q_gain=gain[0], k_gain=gain[1], out=(into[:, :, 0], into[:, :, 1]))
    dev.synchronize()
    x64, g64 = x.cpu().double().requires_grad_(), gain.cpu().double().requires_grad_()
    a = ref.angles(torch.arange(s).expand(1, b, s), rotary.frequencies.cpu(), (32,))
    q64, k64, v64 = x64.unflatten(-1, (3, h, d)).unbind(2)
    q64, k64 = ref.transform(q64, g64[0], True, 1e-6, a, False), ref.transform(k64, g64[1], True, 1e-6, a, False)
    w = torch.softmax(torch.einsum("bihd,bjhd->bhij", q64, k64) * 0.125, -1)
    torch.einsum("bhij,bjhd->bhid", w, v64).backward(go.cpu().double())
    # five f16 roundings between input and gradient, each 2^-11 of the value at most, meet in norms over thousands of
    # values: the attention's own bound of 4e-3 for its gradients, twice for the two stages
    for got, want in ((gx, x64.grad), (gq, g64.grad[0]), (gk, g64.grad[1])):
        assert oracle.rel_frobenius(got, want) <= 8e-3
    assert dev.device_status() == 0
