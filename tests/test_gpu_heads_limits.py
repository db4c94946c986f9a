"""Limits of the per-head norm and rotation, the 8-bit cache and the attention over it: factors of zero, positions at the
ends of 32 bits, strides that no address depends on, many sequences, the forms of the append that single tokens take.

Definitions: tests/heads_reference.py; tolerances as in tests/test_gpu_heads.py unless a test derives its own.
"""
import math
from fractions import Fraction

import pytest
import torch

import dfdx_b200
import heads_reference as ref
from dfdx_b200 import _lib
from test_gpu_heads import F16, F32, U, Serving, check_attention, gen, within
from test_gpu_heads import test_append as check_append

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("window", [0, 21])
@pytest.mark.parametrize("new", [3, 45])
def test_attention_with_a_factor_of_zero(cuda_dev, new, window):
    """alpha = 0, or so small that its product with a block's scale is 0 in f32, takes the mean of the visible values: with
    blocks of zero keys (the least scale, 2^-60) on both sides of the causal edge and of the window's, and a block of keys
    of about 2^100.  In sequences of few and of many rows, alone and in one batch."""
    dev = cuda_dev
    for lens, news in (([100 + new], [new]), ([20 + new, 64, 70], [new, 1, min(new, 64)])):
        sv = Serving(dev, lens, lens, 16, 1, 64, 73)
        n = sum(lens)
        k, v = (torch.randn(n, 1, 64, generator=sv.g) for _ in range(2))
        at = 0
        for m in lens:
            slot = torch.arange(m)
            k[at:at + m][slot // 16 % 3 == 0] = 0.0
            k[at:at + m][slot >= m - new] = 0.0                           # the edge of all rows lies among zero keys
            k[at:at + m][slot // 16 == 1] *= 2.0 ** 100
            at += m
        dev.kv_cache_append(sv.cache, k.cuda(), v.cuda(), *sv.args())
        assert float(sv.cache.k_scale[int(sv.table[0, 0]), 0]) == ref.MIN_SCALE
        sv.new = news
        q = torch.randn(sum(news), 2, 64, generator=sv.g).half().cuda()
        for alpha in (0.0, -0.0, 1e-40, 2.0 ** -100, -2.0 ** -100, 2.0 ** -126):
            out, lse = dev.kv_cache_attention(sv.cache, q, *sv.args(), alpha, window=window, want_lse=True)
            assert bool(out.isfinite().all()) and bool(lse.isfinite().all()), alpha
            check_attention(dev, sv, q, out, lse, alpha, True, window)
    assert dev.device_status() == 0


@pytest.mark.parametrize("new", [3, 45])
def test_log_sum_exp_beside_values_of_another_size(cuda_dev, new):
    """Value scales 2^116 apart, the most that is promised: a block of zeros (2^-60) whose slots weigh 2^-20 to 2^100 times as
    much as those of blocks of values up to 448 * 2^56.  (The outputs are no matter here: values of 2^65 and scores that differ by up to 2^60 leave f16.)"""
    dev = cuda_dev
    n = 32 + new
    sv = Serving(dev, [n], [n], 16, 1, 64, 97)
    k, v = (torch.randn(n, 1, 64, generator=sv.g) for _ in range(2))
    v = v.clamp(-1, 1) * 448 * 2.0 ** 56
    v[16:, 0, 0] = 448 * 2.0 ** 56
    v[:16] = 0.0
    k[:, 0, 0] = 0.0
    k[:16, 0, 0] = 1.0
    dev.kv_cache_append(sv.cache, k.cuda(), v.cuda(), *sv.args())
    scales = sv.cache.v_scale.cpu()[sv.table[0].long(), 0]
    assert float(scales[0]) == ref.MIN_SCALE and bool((scales[1:] == 2.0 ** 56).all())
    sv.new = [new]
    heads = (-20, 0, 10, 50, 100)
    q = torch.randn(new, len(heads), 64, generator=sv.g)
    q[..., 0] = torch.tensor(heads, dtype=torch.float32)
    q = q.half().cuda()
    alpha = math.log(2.0)
    _, lse = dev.kv_cache_attention(sv.cache, q, *sv.args(), alpha, want_lse=True)
    kk, vv = sv.rows(0, n)
    vis = torch.arange(n)[None] <= torch.arange(n - new, n)[:, None]
    _, want, _ = ref.attention(q.cpu().double(), kk, vv, alpha, vis)
    # a score of 64 products in f32: off by 64 u of the sum of their magnitudes, 100 + 64 * 5 * 5 at most
    assert float(q[..., 1:].abs().max()) < 5 and float(k.abs().max()) < 5
    within(lse, want, 2 * 64 * U * alpha * (100 + 64 * 25) + 2.0 ** -19 + 4 * U * want.abs(), "lse")
    assert dev.device_status() == 0


def test_a_wait_that_ran_out_is_reported_before_a_bad_index(cuda_dev):
    """Both happened: the kernel that gave up on a wait left an output that does not hold, whichever came first."""
    dev = cuda_dev
    cache = dev.kv_cache(1, 16, 1, 32)
    for t in cache:
        t.zero_() if t.dtype is F32 else t.view(torch.uint8).zero_()
    bad = torch.tensor([5], dtype=torch.int32).cuda()

    def wait():
        assert dev.lib.b200_selftest_bounded_wait(200000, None, dev._stream()) == 0

    for calls in ((wait, lambda: dev.kv_cache_read(cache, bad)), (lambda: dev.kv_cache_read(cache, bad), wait)):
        assert dev.device_status() == 0
        for call in calls:
            call()
        assert dev.device_status() == _lib.ERR_DEVICE_TIMEOUT
    dev.kv_cache_read(cache, bad)
    assert dev.device_status() == _lib.ERR_INDEX                          # and by itself a bad index is reported as before
    assert dev.device_status() == 0


def test_strides_of_axes_of_one_element(cuda_dev):
    """No address depends on the stride of an axis of extent 1: one token, one head or one batch entry may have any."""
    dev = cuda_dev
    g = gen(93)
    rotary = dfdx_b200.Rotary(dev.rotary_frequencies((32,)), (32,))

    def odd(t, axis, stride):
        """t with another stride on an axis of extent 1."""
        assert t.shape[axis] == 1
        s = list(t.stride())
        s[axis] = stride
        return t.as_strided(t.shape, s)

    sv = Serving(dev, [50], [1], 16, 1, 64, 94)
    sv.fill([50])
    for hq, axis in ((4, 0), (1, 0), (1, 1)):
        t = 1 if axis == 0 else 5
        sv.new = [t]
        q = torch.randn(t, hq, 64, generator=g).half().cuda()
        want, wlse = dev.kv_cache_attention(sv.cache, q, *sv.args(), 0.125, want_lse=True)
        for stride in (0, 515, (1 << 31) + 1, 1 << 41):
            out = torch.zeros_like(q)
            _, lse = dev.kv_cache_attention(sv.cache, odd(q, axis, stride), *sv.args(), 0.125, out=odd(out, axis, stride), want_lse=True)
            assert torch.equal(out, want) and torch.equal(lse, wlse)
            a, b = dev.kv_cache(4, 16, 1, 64), dev.kv_cache(4, 16, 1, 64)
            k, v = (torch.randn(t, 1, 64, generator=g).half().cuda() for _ in range(2))
            cu, lens, table, most = torch.tensor([0, t], dtype=torch.int32).cuda(), torch.tensor([t], dtype=torch.int32).cuda(), sv.table[:, :1].cuda() * 0, t
            wq = dev.kv_cache_append(a, k, v, cu, lens, table, most, q=q, rotary=rotary)
            gq = torch.zeros_like(q)
            dev.kv_cache_append(b, odd(k, axis, stride), odd(v, axis, stride), cu, lens, table, most, q=odd(q, axis, stride), rotary=rotary,
                                q_out=odd(gq, axis, stride))
            assert torch.equal(gq, wq)
            for x, y in zip(a[:2], b[:2]):
                assert torch.equal(x[0, :, :t].view(torch.uint8), y[0, :, :t].view(torch.uint8))
            assert torch.equal(a.k_scale[0], b.k_scale[0]) and torch.equal(a.v_scale[0], b.v_scale[0])
            x4, k4 = q[None], k[None]
            wy = dev.qk_norm_rotary_forward(x4, k4, rotary)
            wd = dev.qk_norm_rotary_backward(x4, k4, x4, k4, rotary)
            for ax in (0, axis + 1):
                o = [torch.zeros_like(x) for x in (x4, k4, x4, k4)]
                xs, ks = odd(x4, ax, stride), odd(k4, ax, stride)
                dev.qk_norm_rotary_forward(xs, ks, rotary, out=(odd(o[0], ax, stride), odd(o[1], ax, stride)))
                d = dev.qk_norm_rotary_backward(xs, ks, xs, ks, rotary, out=(odd(o[2], ax, stride), odd(o[3], ax, stride)))
                assert all(torch.equal(x, y) for x, y in zip((*o[:2], *d), (*wy, *wd)))
    assert dev.device_status() == 0


TWO_PI = Fraction("6.28318530717958647692528676655900576839433879875021164194988918461563281257241799726")


def exact_angles(positions, frequencies):
    """position * frequency less its whole turns, (positions, pairs), from exact products and 80 digits of 2 pi."""
    def angle(p, f):
        turns = Fraction(p) * Fraction(f) / TWO_PI
        return float((turns - round(turns)) * TWO_PI)
    return torch.tensor([[angle(p, f) for f in frequencies] for p in positions], dtype=torch.float64)


@pytest.mark.parametrize("inter", [False, True])
def test_rotation_at_the_ends_of_32_bits(cuda_dev, inter):
    """Positions up to +-2^31 at frequencies of 2^-12 to 2^10 radians are as exact as position 0.

    Tolerance: the remainder in turns, at most 1/2, is rounded to f32 (2^-25: pi u of angle, u = 2^-24), sine and cosine
    are within an ulp (at most 2 u), the first product is rounded (u) and the sum (u of |a| + |b| at most): 8 u (|a| + |b|)
    covers their 3.15 + 2 + 1 + 1."""
    dev = cuda_dev
    g = gen(91)
    pos = [0, 1, -1, 1 << 20, (1 << 27) + 1, (1 << 30) - 1, -(1 << 30) - 7, (1 << 31) - 1, -(1 << 31), 2147480001, -2000000011]
    f = torch.exp2(22 * torch.rand(16, generator=g, dtype=torch.float64) - 12)
    f[0], f[1] = 1.0, 1024.0
    want_angle = exact_angles(pos, f.tolist())
    n = len(pos)
    q, k = (torch.randn(n, h, 32, generator=g) for h in (3, 2))
    rotary = dfdx_b200.Rotary(f.cuda(), (16,), inter)
    p = torch.tensor(pos, dtype=torch.int64).to(torch.int32).cuda()
    yq, yk = dev.qk_norm_rotary_forward(q.cuda()[None], k.cuda()[None], rotary, p[None, None], norm=False)
    dq, dk, _, _ = dev.qk_norm_rotary_backward(q.cuda()[None], k.cuda()[None], q.cuda()[None], k.cuda()[None], rotary, p[None, None], norm=False)
    cache = dev.kv_cache(1, 16, 2, 32)
    cu, lens, table = (torch.tensor(t, dtype=torch.int32).cuda() for t in ([0, n], [n], [[0]]))
    aq = dev.kv_cache_append(cache, k.cuda(), k.cuda(), cu, lens, table, n, q=q.cuda(), rotary=rotary, positions=p[None])
    for x, sign, got in ((q, 1, yq[0]), (k, 1, yk[0]), (q, -1, dq[0]), (k, -1, dk[0]), (q, 1, aq)):
        want = ref.transform(x.double(), None, False, 0.0, sign * want_angle, inter)
        size = x.double().abs()
        size = size[..., 0::2] + size[..., 1::2] if inter else size[..., :16] + size[..., 16:]
        size = size.repeat_interleave(2, -1) if inter else torch.cat((size, size), -1)
        within(got, want, 8 * U * size, "rotated")
    assert dev.device_status() == 0


def test_sines_and_cosines(cuda_dev):
    """A pair (1, 0) turns into its cosine and sine themselves.  They are CUDA's of the angle's f32 part, within an ulp (2^-24
    below 1), plus the rest's share, rounded once (half an ulp): 1.5 u."""
    dev = cuda_dev
    g = gen(92)
    f = torch.exp2(-12 * torch.rand(16, generator=g, dtype=torch.float64))
    pos = torch.randint(-(1 << 31), 1 << 31, (400,), generator=g)
    pos = torch.where(torch.arange(400) % 2 == 0, pos, pos % 9000)
    angle = exact_angles(pos.tolist(), f.tolist())
    want = torch.cat((angle.cos(), angle.sin()), -1)[:, None]
    x = torch.cat((torch.ones(400, 1, 16), torch.zeros(400, 1, 16)), -1)
    p = pos.to(torch.int32).cuda()
    y, _ = dev.qk_norm_rotary_forward(x.cuda()[None], x[:, :0].cuda()[None], dfdx_b200.Rotary(f.cuda(), (16,)), p[None, None], norm=False)
    within(y[0], want, 1.5 * U, "cosine and sine")


@pytest.mark.parametrize("seqs", [40, 991, 993, 2500])
@pytest.mark.parametrize("most", [1, 3])
def test_append_of_many_sequences(cuda_dev, seqs, most):
    """More sequences than one look of a warp, or two, narrows down to one; runs of sequences without new tokens, tokens of
    no sequence in front and behind."""
    dev = cuda_dev
    g = gen(95 + seqs)
    new = torch.randint(0, most + 1, (seqs,), generator=g)
    new[seqs // 3:seqs // 3 + 35] = 0
    new[:2] = 0
    new[-3:-1] = 0
    past = torch.randint(0, 40, (seqs,), generator=g)
    lead, tail, page = 5, 9, 16
    t = lead + int(new.sum()) + tail
    lens = past + new
    table = torch.randperm(4 * seqs + 7, generator=g)[:4 * seqs].view(seqs, 4)
    cache = dev.kv_cache(4 * seqs + 7, page, 2, 32)
    cu = lead + torch.cat([torch.zeros(1, dtype=torch.int64), new.cumsum(0)])
    on = lambda x: x.to(torch.int32).cuda()
    for x in cache[:2]:
        x.view(torch.uint8).fill_(0x7F)
    # the earlier slots, through appends of at most 20 sequences
    for s0 in range(0, seqs, 20):
        p = past[s0:s0 + 20]
        c = torch.cat([torch.zeros(1, dtype=torch.int64), p.cumsum(0)])
        if int(c[-1]):
            old = torch.zeros(int(c[-1]), 2, 32).half().cuda()
            dev.kv_cache_append(cache, old, old, on(c), on(p), on(table[s0:s0 + 20]), int(p.max()))
    held = [x.view(torch.uint8).cpu() for x in cache[:2]]
    q, k, v = (torch.randn(t, h, 32, generator=g).half().cuda() for h in (3, 2, 2))
    rotary = dfdx_b200.Rotary(dev.rotary_frequencies((16,)), (16,))
    out = torch.full_like(q, 7.0)
    dev.kv_cache_append(cache, k, v, on(cu), on(lens), on(table), most, q=q, rotary=rotary, q_out=out)
    assert dev.device_status() == 0
    owner = torch.arange(seqs).repeat_interleave(new)
    slot = torch.cat([torch.arange(int(p), int(p + m)) for p, m in zip(past, new)])
    mine = slice(lead, t - tail)
    wq, wk = dev.qk_norm_rotary_forward(q[None, mine], k[None, mine], rotary, on(slot)[None, None], norm=False)
    assert torch.equal(out[mine], wq[0]) and bool((out[:lead] == 7.0).all()) and bool((out[t - tail:] == 7.0).all())
    ids, row = table[owner, slot // page], slot % page
    for c, want in enumerate((wk[0], v[mine])):
        want = want.cpu().double()
        scale = cache[2 + c].cpu().double()[ids][..., None]
        got = cache[c].cpu()[ids, :, row].double() * scale
        # half a code; the keys' want is itself rounded to f16
        within(got, want, torch.maximum(2.0 ** -4 * want.abs(), 2.0 ** -10 * scale) * (1 + 2.0 ** -6) + 2.0 ** -10 * want.abs(), f"codes {c}")
        same = torch.ones(held[c].shape[0], page, dtype=torch.bool)
        same[ids, row] = False
        same[ids[row > 0]] = False                                        # blocks whose scale may have grown under zeros
        fresh = same[:, :, None].expand(-1, -1, 2).transpose(1, 2)
        assert torch.equal(cache[c].view(torch.uint8).cpu()[fresh], held[c][fresh])


def test_append_leaves_what_does_not_fit_untouched(cuda_dev):
    """Bounds that do not fit: the sequences' tokens, pages and the rows around the buffers stay as they were."""
    dev = cuda_dev
    sv = Serving(dev, [10, 10, 10], [2, 2, 2], 16, 1, 32, 96)
    sv.fill([8, 8, 8])
    cu, lens, table, most = sv.args()
    x = torch.randn(10, 1, 32, generator=sv.g).half().cuda()[2:8]
    owned = {int(p) for p in sv.table.flatten()}
    spare = [i for i in range(sv.cache.k.shape[0]) if i not in owned]
    assert spare
    for bad_cu, bad_lens, skipped in (([0, 2, 1, 6], None, (1, 2)), ([0, 2, 9, 6], None, (1, 2)), ([-1, 2, 4, 6], None, (0,)), ([0, 2, 4, 7], None, (2,)),
                                      ([0, 2, 4, 1 << 30], None, (2,)), (None, [10, 1, 10], (1,)), (None, [10, 17, 10], (1,)), (None, [10, -3, 10], (1,))):
        held = [t.view(torch.uint8).clone() for t in sv.cache]
        buf = torch.full((12, 1, 32), 7.0, dtype=F16, device="cuda")
        c = torch.tensor(bad_cu, dtype=torch.int32).cuda() if bad_cu else cu
        n = torch.tensor(bad_lens, dtype=torch.int32).cuda() if bad_lens else lens
        dev.kv_cache_append(sv.cache, x, x, c, n, table, most, q=x, q_out=buf[3:9])
        assert dev.device_status() == _lib.ERR_INDEX
        assert bool((buf[:3] == 7.0).all()) and bool((buf[9:] == 7.0).all())
        out = buf[3:9]
        falling = bad_cu is not None and sorted(bad_cu) != bad_cu          # then other sequences' tokens may be skipped too
        for s in range(3):
            rows = slice(2 * s, 2 * s + 2)
            done = (out[rows] == x[rows]).all(-1)
            left = (out[rows] == 7.0).all(-1)
            assert bool((done | left).all())
            assert falling or bool((left if s in skipped else done).all()), (bad_cu, bad_lens, s)
            if s in skipped:
                for was, now in zip(held, sv.cache):
                    p = int(sv.table[s, 0])
                    assert torch.equal(was[p], now.view(torch.uint8)[p]), (bad_cu, bad_lens, s)
        for was, now in zip(held, sv.cache):
            assert torch.equal(was[spare], now.view(torch.uint8)[spare])
    dev.kv_cache_append(sv.cache, x, x, cu, lens, table, most)
    assert dev.device_status() == 0


APPEND = [  # dtype, page, heads, q_heads, d, past, new, pairs, interleaved, norm: forms that the cases of test_gpu_heads.py leave out
    (F32, 64, 2, 4, 128, [63, 64, 0, 5], [1, 1, 1, 1], 64, False, True),              # single tokens: f32,
    (F32, 16, 3, 6, 64, [15, 16, 0, 33, 7], [1, 1, 1, 1, 0], 32, True, True),         # adjacent pairs, an empty sequence,
    (F16, 32, 2, 6, 96, [31, 0, 40], [1, 1, 1], 48, True, False),
    (F32, 128, 1, 5, 96, [127, 3, 200], [1, 1, 1], 30, False, True),                  # pairs no multiple of 4: element access,
    (F16, 16, 5, 5, 32, [9, 0, 15], [1, 1, 1], 7, True, True),
    (F32, 16, 7, 7, 64, [5 * i % 50 for i in range(90)], [1] * 90, 16, True, False),  # several heads a CTA
    (F32, 128, 2, 2, 128, [0, 100, 127], [300, 28, 2], 64, True, True),               # f32 with the largest pages
    (F32, 128, 1, 3, 64, [60, 0], [140, 257], 32, False, True),
    (F32, 128, 2, 2, 96, [1, 130], [129, 90], 25, False, True),
    (F16, 128, 3, 3, 128, [5], [300], 13, True, True),
]


@pytest.mark.parametrize("case", APPEND, ids=lambda c: "-".join(str(x).replace("torch.", "") for x in c)[:80])
def test_append_forms(cuda_dev, case):
    check_append(cuda_dev, case)
