"""GPU tests of the 4-bit KV cache. Codes, scales and zero points are compared
bit for bit with the format's formula run in fp32 on the CPU, values read back
with (code - zero) * scale rounded once. Attention over the cache is compared
with softmax(q k^T scale) v in 64 bits on the values the codes stand for, with
the tolerance: u|out| for the output's rounding (u = 2^-8 bf16, 2^-11 fp16);
2^-11 sum p|v| for weights held in 11 bits; a score, scale * s (q.c - z sum q),
is an fp32 sum of D terms no larger than 30 s |q|, off by at most
e = (D + 16) 2^-24 scale 30 s sum|q|, which moves each p within exp(+-2e); the
fp32 exponential, sums and products add at most 2^-16 sum p 15 s."""

from __future__ import annotations

import pytest
import torch

from tritonforge_b200 import kernels
from tritonforge_b200.kernels import KV4Cache

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
SHAPES = [(2, 64, 64), (4, 128, 64), (8, 128, 128), (1, 128, 64), (3, 64, 64)]


def cu(lens):
    return torch.tensor([0] + list(lens)).cumsum(0).to(torch.int32).cuda()


def i32(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def quantize(x, group):
    """The format on the CPU, in fp32: (codes [.., D/2] uint8, parameters [.., D/g, 2] of x's dtype)."""
    xg = x.cpu().float().unflatten(-1, (-1, group))
    lo, hi = xg.amin(-1, keepdim=True).clamp(max=0), xg.amax(-1, keepdim=True).clamp(min=0)
    rng = hi - lo
    scale = (rng / torch.full_like(rng, 15.0)).clamp(min=1e-8)
    zero = ((0 - lo) / scale).round().clamp(0, 15)
    code = (xg / scale + zero).round().clamp(0, 15)
    bad = ~torch.isfinite(rng)
    scale, zero = torch.where(bad, torch.nan, scale), torch.where(bad, 0.0, zero)
    code = torch.where(bad, 0.0, code).to(torch.uint8).flatten(-2)
    return code[..., 0::2] | (code[..., 1::2] << 4), torch.cat([scale, zero], -1).to(x.dtype)


def values(codes, params):
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).float()
    p = params.float()
    return ((c.unflatten(-1, (p.shape[-2], -1)) - p[..., 1:]) * p[..., :1]).flatten(-2)


def same_bits(a, b):
    a, b = a.cpu(), b.cpu()
    if a.dtype != torch.uint8:
        nan = torch.isnan(a.float())
        return bool(torch.equal(nan, torch.isnan(b.float())) and
                    torch.equal(a.view(torch.int16)[~nan], b.view(torch.int16)[~nan]))
    return torch.equal(a, b)


def tokens(t, h, d, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + t)
    spread = 1 + 4 * (torch.rand(d, device="cuda", generator=g) < 0.1)
    return [(torch.randn(t, h, d, device="cuda", generator=g) * spread + o).to(dtype) for o in (0.5, 0.0)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("h,d,g", SHAPES)
@pytest.mark.parametrize("lens,start,slots", [([1], None, None), ([5, 0, 19, 1], [0, 3, 7, 0], None),
                                              ([33, 2], [4, 60], [2, 0]), ([200], [3], [1])])
def test_write_and_read(h, d, g, lens, start, slots, dtype):
    t_max, b = 224, max(len(lens), 3)
    cache = KV4Cache.empty(b, h, t_max, d, g, dtype)
    for x in cache:
        x.view(torch.uint8).fill_(0x5A)  # what is not written stays
    before = [x.clone() for x in cache]
    k, v = tokens(sum(lens), h, d, dtype)
    st = None if start is None else i32(*start)
    sl = None if slots is None else i32(*slots)
    kernels.kv4_write(k, v, cache, cu(lens), st, sl)
    want = [x.cpu() for x in before]
    i = 0
    for s, n in enumerate(lens):
        p0, row = (start or [0] * len(lens))[s], (slots or list(range(len(lens))))[s]
        for side, x in ((0, k), (2, v)):
            c, p = quantize(x[i:i + n], g)
            want[side][row, :, p0:p0 + n] = c.transpose(0, 1)
            want[side + 1][row, :, p0:p0 + n] = p.transpose(0, 1)
        i += n
    for name, a, w in zip(KV4Cache._fields, cache, want):
        assert same_bits(a, w), name
    kr, vr = kernels.kv4_read(cache, cu(lens), sum(lens), st, sl)
    for x, got in ((k, kr), (v, vr)):
        assert torch.equal(got.cpu(), values(*quantize(x, g)).to(dtype))


def test_group_edges():
    """Zero groups, one sign, tiny and huge ranges, halves of a code, NaN and infinities."""
    d, g = 128, 64
    rows = torch.zeros(14, 1, d)
    rows[1, 0, :64] = 10.5
    rows[2, 0, :64] = -3.25
    rows[3, 0, 5] = 1e-9
    rows[4, 0, 64:] = torch.linspace(-6e4, 6e4, 64)
    rows[5, 0, :64] = torch.arange(64) * 0.5 - 7.5  # halves between codes
    rows[6, 0, 3] = float("nan")
    rows[7, 0, 70] = float("inf")
    rows[8, 0, 2] = -float("inf")
    rows[9, 0] = -0.0
    rows[10, 0, :64] = torch.linspace(1.0, 1.001, 64)
    rows[11, 0, 10], rows[11, 0, 11] = float("inf"), -float("inf")
    rows[12, 0, :64] = torch.arange(64) / 64 * 15 + 0.5
    rows[13, 0, 0], rows[13, 0, 1] = 6e-8, -6e-8
    for dtype in (torch.float16, torch.bfloat16):
        x = rows.to(dtype).cuda()
        cache = KV4Cache.empty(1, 1, 16, d, g, dtype)
        kernels.kv4_write(x, -x, cache, cu([14]))
        for side, y in ((0, x), (2, -x)):
            c, p = quantize(y, g)
            assert same_bits(cache[side][0, :, :14], c.transpose(0, 1)), dtype
            assert same_bits(cache[side + 1][0, :, :14], p.transpose(0, 1)), dtype
        kr, _ = kernels.kv4_read(cache, cu([14]), 14)
        nan = torch.isnan(kr.float()).cpu()[:, 0]
        want = torch.zeros(14, d, dtype=torch.bool)
        for r, half in ((6, 0), (7, 1), (8, 0), (11, 0)):
            want[r, 64 * half:64 * half + 64] = True
        assert torch.equal(nan, want)
        assert float(kr[1, 0, 0]) == pytest.approx(10.5, rel=0.01)


def test_positions_outside_the_cache():
    """Tokens whose position or slot is outside are left out; they read as zeros."""
    cache = KV4Cache.empty(2, 2, 32, 64, 64, torch.float16)
    k, v = tokens(12, 2, 64, torch.float16)
    lens, start, slots = [4, 4, 4], i32(30, -2, 0), i32(0, 1, 2)
    kernels.kv4_write(k, v, cache, cu(lens), start, slots)
    kr, vr = kernels.kv4_read(cache, cu(lens), 12, start, slots)
    keep = torch.zeros(12, dtype=torch.bool, device="cuda")
    keep[[0, 1, 6, 7]] = True
    for x, got in ((k, kr), (v, vr)):
        assert torch.equal(got[keep].cpu(), values(*quantize(x[keep], 64)).half())
        assert (got[~keep] == 0).all()
    used = torch.zeros(2, 2, 32, dtype=torch.bool, device="cuda")
    used[0, :, 30:] = True
    used[1, :, :2] = True
    assert (cache.k_params[~used] == 0).all() and (cache.v[~used] == 0).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hq,h,d,g", [(14, 2, 64, 64), (28, 4, 128, 64), (8, 8, 128, 128), (3, 1, 64, 64)])
def test_rope_write(hq, h, d, g, dtype):
    """q and k rotated in place with transformers' roundings, the cache as kv4_write of the rotated keys."""
    lens, start, t_max = [9, 1, 30], [0, 17, 2], 48
    t = sum(lens)
    gen = torch.Generator().manual_seed(d + hq)
    rows = torch.randn(t, (hq + 2 * h) * d + 8, generator=gen).to(dtype).cuda()
    qkv = rows[:, :-8]
    ang = torch.rand(t_max, d // 2, generator=gen) * 6
    cos, sin = (torch.cat([f(ang), f(ang)], -1).to(dtype).cuda() for f in (torch.cos, torch.sin))
    before = rows.clone()
    pos = torch.cat([torch.arange(n) + s for n, s in zip(lens, start)]).cuda()

    def turn(x):
        half = x.shape[-1] // 2
        return x * cos[pos][:, None] + torch.cat((-x[..., half:], x[..., :half]), -1) * sin[pos][:, None]

    n = (hq + h) * d
    heads = turn(before[:, :n].view(t, hq + h, d))
    k, v = heads[:, hq:], before[:, n:n + h * d].view(t, h, d)
    want = KV4Cache.empty(3, h, t_max, d, g, dtype)
    got = KV4Cache.empty(3, h, t_max, d, g, dtype)
    kernels.kv4_write(k, v, want, cu(lens), i32(*start))
    kernels.rope_kv4_write(qkv, hq, cos, sin, got, cu(lens), i32(*start))
    assert torch.equal(rows[:, :n].view(t, hq + h, d), heads)
    assert torch.equal(rows[:, n:], before[:, n:])
    for name, a, b in zip(KV4Cache._fields, got, want):
        assert same_bits(a, b), name


def random_cache(b, h, t_max, d, g, dtype, seed=0, v_size=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed + t_max)
    cache = KV4Cache.empty(b, h, t_max, d, g, dtype)
    t_max = cache.k.shape[2]
    k = torch.randn(b * t_max, h, d, device="cuda", generator=gen) + 0.3
    v = torch.randn(b * t_max, h, d, device="cuda", generator=gen) * v_size
    kernels.kv4_write(k.to(dtype), v.to(dtype), cache, cu([t_max] * b))
    return cache


def check_decode(got, q, cache, lens, scale=None):
    b, hq, d = q.shape
    h, r = cache.k.shape[1], hq // cache.k.shape[1]
    scale = d ** -0.5 if scale is None else scale
    g = d // cache.k_params.shape[3]
    for i, n in enumerate(lens):
        n = max(0, min(n, cache.k.shape[2]))
        if n == 0:
            assert (got[i] == 0).all()
            continue
        k = values(cache.k[i, :, :n], cache.k_params[i, :, :n]).double()
        v = values(cache.v[i, :, :n], cache.v_params[i, :, :n]).double()
        qi = q[i].double().view(h, r, d)
        p = torch.softmax(qi @ k.transpose(1, 2) * scale, -1)
        want = p @ v
        ks = cache.k_params[i, :, :n, :, 0].double().amax((1, 2))
        e = (d + 16) * 2.0 ** -24 * scale * 30 * ks[:, None] * qi.abs().sum(-1)
        e = torch.expm1(2 * e)[..., None]
        s15 = p @ (15 * cache.v_params[i, :, :n, :, 0].double().repeat_interleave(g, -1))
        tol = U[q.dtype] * want.abs() + (2.0 ** -11 + e) * (p @ v.abs()) + 2.0 ** -16 * s15
        if q.dtype == torch.float16:
            tol = tol + 2.0 ** -25  # half a subnormal step
        bad = (got[i].double().view(h, r, d) - want).abs() > tol
        assert not bad.any(), (f"sequence {i} ({n} positions): {int(bad.sum())} off, first {bad.nonzero()[0].tolist()},"
                               f" worst {float(((got[i].double().view(h, r, d) - want).abs() / tol).max()):.2f} x")


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hq,h,d,g", [(14, 2, 64, 64), (28, 4, 128, 64), (64, 8, 128, 128), (64, 8, 128, 64),
                                      (8, 8, 64, 64), (3, 3, 128, 128), (20, 2, 128, 64), (40, 1, 64, 64)])
@pytest.mark.parametrize("t_max,lens", [(16, [1]), (336, [0, 1, 2, 15, 16, 17, 300]), (1040, [1040, 5, 63, 64, 65]),
                                        (5008, [5001, 129])])
def test_decode_attention(hq, h, d, g, t_max, lens, dtype):
    cache = random_cache(len(lens), h, t_max, d, g, dtype)
    gen = torch.Generator(device="cuda").manual_seed(hq + t_max)
    q = torch.randn(len(lens), hq, d, device="cuda", generator=gen).to(dtype)
    got = kernels.kv4_decode_attention(q, cache, i32(*lens))
    check_decode(got, q, cache, lens)
    assert torch.equal(got, kernels.kv4_decode_attention(q, cache, i32(*lens))), "two runs differ"


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("qs,vs", [(1e-4, 1.0), (30.0, 1e-3), (1.0, 200.0), (3.0, 1e-5)])
def test_decode_magnitudes(qs, vs, dtype):
    """Queries and values far from 1: weights and codes keep their precision."""
    lens = [700, 33]
    cache = random_cache(2, 4, 704, 128, 64, dtype, v_size=vs)
    q = (torch.randn(2, 28, 128, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)) * qs).to(dtype)
    check_decode(kernels.kv4_decode_attention(q, cache, i32(*lens)), q, cache, lens)


def test_decode_mixed_value_scales():
    """Values whose scale grows and shrinks by orders of magnitude along the context."""
    n, dtype = 900, torch.bfloat16
    cache = KV4Cache.empty(1, 2, 912, 128, 64, dtype)
    gen = torch.Generator(device="cuda").manual_seed(9)
    k = torch.randn(n, 2, 128, device="cuda", generator=gen)
    ramp = 10.0 ** torch.linspace(-4, 4, n, device="cuda")
    for v in (ramp, ramp.flip(0)):
        vals = torch.randn(n, 2, 128, device="cuda", generator=gen) * v[:, None, None]
        kernels.kv4_write(k.to(dtype), vals.to(dtype), cache, cu([n]))
        q = torch.randn(1, 14, 128, device="cuda", generator=gen).to(dtype)
        check_decode(kernels.kv4_decode_attention(q, cache, i32(n)), q, cache, [n])


def test_decode_ignores_what_lies_past_the_length():
    """Parameters past the length may be anything (NaN here), and a length past the cache is the cache's."""
    cache = random_cache(2, 2, 96, 64, 64, torch.float16)
    q = torch.randn(2, 14, 64, device="cuda").half()
    want = kernels.kv4_decode_attention(q, cache, i32(41, 96))
    cache.k_params[0, :, 41:] = float("nan")
    cache.v_params[0, :, 41:] = float("inf")
    assert torch.equal(kernels.kv4_decode_attention(q, cache, i32(41, 1000)), want)
    assert (kernels.kv4_decode_attention(q, cache, i32(-3, 0)) == 0).all()
    # a cached NaN shows in the heads that read it, and only there
    cache.v_params[1, 1, 7, :, 0] = float("nan")
    got = kernels.kv4_decode_attention(q, cache, i32(41, 96))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1, :7], want[1, :7])
    assert torch.isnan(got[1, 7:].float()).all()


def test_decode_scale_and_out():
    cache = random_cache(3, 4, 128, 128, 64, torch.bfloat16)
    q = torch.randn(3, 28, 128, device="cuda").bfloat16()
    out = torch.empty_like(q)
    lens = [100, 1, 128]
    assert kernels.kv4_decode_attention(q, cache, i32(*lens), scale=0.3, out=out) is out
    check_decode(out, q, cache, lens, scale=0.3)
    s = torch.cuda.Stream()
    n = i32(*lens)
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = kernels.kv4_decode_attention(q, cache, n, scale=0.3)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, out)


def test_offsets_past_32_bits():
    """A cache of more than 2^31 codes: the last sequence's rows are found."""
    b, h, d = 9, 8, 128
    t_max = 466_048  # 9 x 8 x 466048 x 64 bytes = 2.15e9
    cache = KV4Cache.empty(b, h, t_max, d, 128, torch.bfloat16)
    k, v = tokens(600, h, d, torch.bfloat16)
    start, slots = i32(t_max - 600), i32(b - 1)
    kernels.kv4_write(k, v, cache, cu([600]), start, slots)
    kr, vr = kernels.kv4_read(cache, cu([600]), 600, start, slots)
    assert torch.equal(kr.cpu(), values(*quantize(k, 128)).bfloat16())
    assert torch.equal(vr.cpu(), values(*quantize(v, 128)).bfloat16())
    q = torch.randn(b, 64, d, device="cuda").bfloat16()
    lens = torch.zeros(b, dtype=torch.int32, device="cuda")
    lens[-1] = t_max
    got = kernels.kv4_decode_attention(q, cache, lens)
    # all but the last 600 positions hold zeros: score 0, value 0. A sum of 466048 weights in parts
    # of at most 1/16 of them adds 29128 x 2^-24 < 2^-9 to the weights' 2^-11; scores as in check_decode
    kv, vv = (values(*quantize(x, 128)).double().cuda() for x in (k, v))
    q64 = q[-1].double().view(h, 8, d)
    e = (d + 16) * 2.0 ** -24 * d ** -0.5 * 30 * float(cache.k_params[-1, :, -600:, :, 0].max()) * q64.abs().sum(-1)
    s = (q64 @ kv.permute(1, 2, 0)).reshape(64, 600) * d ** -0.5
    p = torch.softmax(torch.cat([torch.zeros(64, t_max - 600, dtype=torch.float64, device="cuda"), s], 1), -1)
    p = p[:, -600:].view(h, 8, 600)
    want, av = p @ vv.transpose(0, 1), p @ vv.abs().transpose(0, 1)
    tol = 2.0 ** -8 * want.abs() + (2.0 ** -11 + 2.0 ** -9 + torch.expm1(2 * e)[..., None]) * av
    assert (got[:-1] == 0).all()
    assert ((got[-1].double().view(h, 8, d) - want).abs() <= tol).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hq,h,d,g,t_max,pos", [(14, 2, 64, 64, 336, [0, 31, 32, 127, 300]), (28, 4, 128, 64, 1040, [1039, 0, 513]),
                                                (64, 8, 128, 128, 144, [128, 143]), (20, 1, 64, 64, 80, [63, 64]),
                                                (28, 4, 128, 128, 5008, [4999])])
def test_fused_step(hq, h, d, g, t_max, pos, dtype):
    """kv4_decode_attention_rope equals rope_kv4_write then kv4_decode_attention bit for bit, cache included;
    the projection rows are only read, positions outside the cache write nothing and give zeros."""
    pos = pos + [-1, t_max]
    b = len(pos)
    cache = random_cache(b, h, t_max, d, g, dtype)
    gen = torch.Generator(device="cuda").manual_seed(hq + t_max)
    rows = torch.randn(b, (hq + 2 * h) * d + 8, device="cuda", generator=gen).to(dtype)
    ang = torch.rand(t_max, d // 2, device="cuda", generator=gen) * 6
    cos, sin = (torch.cat([f(ang), f(ang)], -1).to(dtype) for f in (torch.cos, torch.sin))
    other = KV4Cache(*[x.clone() for x in cache])
    before = rows.clone()
    got = kernels.kv4_decode_attention_rope(rows[:, :-8], hq, cos, sin, cache, i32(*pos))
    assert torch.equal(rows, before)
    kernels.rope_kv4_write(rows[:, :-8], hq, cos, sin, other, cu([1] * b), i32(*pos))
    lens = [p + 1 if 0 <= p < t_max else 0 for p in pos]
    want = kernels.kv4_decode_attention(rows[:, :hq * d].view(b, hq, d), other, i32(*lens))
    for name, x, y in zip(KV4Cache._fields, cache, other):
        assert same_bits(x, y), name
    assert torch.equal(got, want)
    assert (got[-2:] == 0).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_codes_at_and_around_halves(dtype):
    """Rows built so that many quotients fall on, and next to, a half between two codes; random exponents."""
    gen = torch.Generator().manual_seed(4)
    n, d = 4000, 64
    x = torch.randint(-255, 256, (n, 1, d), generator=gen).float()
    x[: n // 2, 0, 0] = -torch.randint(0, 121, (n // 2,), generator=gen).float()
    x[: n // 2, 0, 1] = x[: n // 2, 0, 0] + 30 * torch.randint(1, 9, (n // 2,), generator=gen)  # range / 15 is even
    x[: n // 2] = x[: n // 2].clamp(x[: n // 2, :, :1], x[: n // 2, :, 1:2])
    x = torch.ldexp(x, torch.randint(-12, 6, (n, 1, 1), generator=gen))
    x[n // 2:] += torch.randn(n // 2, 1, d, generator=gen) * x[n // 2:].abs() * 2.0 ** -7
    x = x.to(dtype).cuda()
    cache = KV4Cache.empty(1, 1, n, d, 64, dtype)
    kernels.kv4_write(x, -x, cache, cu([n]))
    for side, y in ((0, x), (2, -x)):
        c, p = quantize(y, 64)
        assert same_bits(cache[side][0, 0, :n], c[:, 0])
        assert same_bits(cache[side + 1][0, 0, :n], p[:, 0])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_one_token_or_one_head_of_odd_strides(dtype):
    """An axis of one element may have any stride, as in a row cut from a wider one."""
    h, hq, d, g = 2, 4, 64, 64
    k, v = tokens(1, h, d, dtype)

    def one(x):  # heads 72 apart, the token 147 from a next one
        buf = torch.zeros(h * (d + 8), device="cuda", dtype=dtype)
        return torch.as_strided(buf, (1, h, d), (h * (d + 8) + 3, d + 8, 1)).copy_(x)

    want, got = (KV4Cache.empty(1, h, 32, d, g, dtype) for _ in range(2))
    kernels.kv4_write(k, v, want, cu([1]), i32(5))
    kernels.kv4_write(one(k), one(v), got, cu([1]), i32(5))
    assert all(same_bits(a, b) for a, b in zip(got, want))
    for x, y in zip(kernels.kv4_read(got, cu([1]), 1, i32(5), out=(one(k), one(v))),
                    kernels.kv4_read(got, cu([1]), 1, i32(5))):
        assert torch.equal(x, y)
    # the projection row of one token
    width = (hq + 2 * h) * d
    row = torch.randn(1, width, device="cuda", generator=torch.Generator("cuda").manual_seed(1)).to(dtype)
    whole, qkv = row.clone(), torch.as_strided(row, (1, width), (width + 3, 1))
    ang = torch.rand(32, d // 2, device="cuda", generator=torch.Generator("cuda").manual_seed(2)) * 6
    cos, sin = (torch.cat([f(ang), f(ang)], -1).to(dtype) for f in (torch.cos, torch.sin))
    a = kernels.kv4_decode_attention_rope(qkv, hq, cos, sin, got, i32(6))
    b = kernels.kv4_decode_attention_rope(whole, hq, cos, sin, want, i32(6))
    assert torch.equal(a, b) and all(same_bits(x, y) for x, y in zip(got, want))
    kernels.rope_kv4_write(qkv, hq, cos, sin, got, cu([1]), i32(7))
    kernels.rope_kv4_write(whole, hq, cos, sin, want, cu([1]), i32(7))
    assert torch.equal(qkv, whole) and all(same_bits(x, y) for x, y in zip(got, want))
    # several tokens of one head
    k1, v1 = tokens(5, 1, d, dtype)

    def many(x):
        return torch.as_strided(torch.zeros(5 * 72, device="cuda", dtype=dtype), x.shape, (72, 3, 1)).copy_(x)

    want, got = (KV4Cache.empty(1, 1, 16, d, g, dtype) for _ in range(2))
    kernels.kv4_write(k1, v1, want, cu([5]))
    kernels.kv4_write(many(k1), many(v1), got, cu([5]))
    assert all(same_bits(x, y) for x, y in zip(got, want))


def test_tokens_in_no_sequence():
    """Rows before cu[0] and from cu[S] on (padding to a fixed size) belong to nobody: not written, not
    rotated, read as zeros."""
    h, hq, d, dtype = 2, 4, 64, torch.bfloat16
    offs, start = i32(2, 5, 9), i32(4, 10)
    k, v = tokens(12, h, d, dtype)
    want, got = (KV4Cache.empty(2, h, 32, d, 64, dtype) for _ in range(2))
    kernels.kv4_write(k[2:9], v[2:9], want, cu([3, 4]), start)
    kernels.kv4_write(k, v, got, offs, start)
    assert all(same_bits(a, b) for a, b in zip(got, want))
    for x, y in zip(kernels.kv4_read(random_cache(2, h, 32, d, 64, dtype), offs, 12, start),
                    kernels.kv4_read(random_cache(2, h, 32, d, 64, dtype), cu([3, 4]), 7, start)):
        assert torch.equal(x[2:9], y) and (x[:2] == 0).all() and (x[9:] == 0).all()
    gen = torch.Generator("cuda").manual_seed(3)
    rows = torch.randn(12, (hq + 2 * h) * d, device="cuda", generator=gen).to(dtype)
    ang = torch.rand(32, d // 2, device="cuda", generator=gen) * 6
    cos, sin = (torch.cat([f(ang), f(ang)], -1).to(dtype) for f in (torch.cos, torch.sin))
    some, every = rows[2:9].clone(), rows.clone()
    kernels.rope_kv4_write(some, hq, cos, sin, want, cu([3, 4]), start)
    kernels.rope_kv4_write(every, hq, cos, sin, got, offs, start)
    assert all(same_bits(a, b) for a, b in zip(got, want))
    assert torch.equal(every, torch.cat([rows[:2], some, rows[9:]]))


def check_finite(got, q, cache, lens):
    """check_decode, where a NaN (its difference is not above a tolerance either) fails too."""
    assert torch.isfinite(got.float()).all(), f"{int((~torch.isfinite(got.float())).sum())} of {got.numel()} not finite"
    check_decode(got, q, cache, lens)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d,g", [(64, 64), (128, 64), (128, 128)])
@pytest.mark.parametrize("qs,vs", [(1e-4, 1.0), (30.0, 1e-3), (1.0, 200.0), (3.0, 1e-5), (2e3, 3e3), (0.0, 1.0), (1.0, 0.0)])
def test_decode_magnitudes_stay_finite(qs, vs, d, g, dtype):
    """Queries and values far from 1, all zero among them: finite results of the same precision."""
    lens = [700, 33]
    cache = random_cache(2, 4, 704, d, g, dtype, v_size=vs)
    gen = torch.Generator(device="cuda").manual_seed(3)
    q = (torch.randn(2, 28, d, device="cuda", generator=gen) * qs).to(dtype)
    check_finite(kernels.kv4_decode_attention(q, cache, i32(*lens)), q, cache, lens)


@pytest.mark.parametrize("up", [True, False])
def test_decode_mixed_value_scales_stay_finite(up):
    """Value scales over eight orders of magnitude along the context, growing and shrinking."""
    n, dtype = 900, torch.bfloat16
    cache = KV4Cache.empty(1, 2, 912, 128, 64, dtype)
    gen = torch.Generator(device="cuda").manual_seed(10)
    ramp = 10.0 ** torch.linspace(-4, 4, n, device="cuda")
    k = torch.randn(n, 2, 128, device="cuda", generator=gen)
    vals = torch.randn(n, 2, 128, device="cuda", generator=gen) * (ramp if up else ramp.flip(0))[:, None, None]
    kernels.kv4_write(k.to(dtype), vals.to(dtype), cache, cu([n]))
    q = torch.randn(1, 14, 128, device="cuda", generator=gen).to(dtype)
    check_finite(kernels.kv4_decode_attention(q, cache, i32(n)), q, cache, [n])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d,g", [(64, 64), (128, 64), (128, 128)])
@pytest.mark.parametrize("n", [8, 900])
def test_small_weights_beside_a_large_one(n, d, g, dtype):
    """One position takes nearly all of the weight, and all but two values of a group are zero there (their
    codes the zero point); the others weigh e^-11.5 to e^-13.5 each, with the largest code. Their sum must
    not drown in the products of the first with its codes, which the zero points take away again."""
    h = 16
    gen = torch.Generator(device="cuda").manual_seed(d + g)
    q = torch.randn(1, h, d, device="cuda", generator=gen).to(dtype)
    gap = torch.linspace(11.5, 13.5, h, device="cuda")[:, None]
    k = torch.zeros(n, h, d, device="cuda")
    k[5] = q[0].float() * gap * d ** 0.5 / q[0].float().pow(2).sum(-1, keepdim=True)
    v = torch.full((n, h, d), 63.0, device="cuda")  # groups of scale 126 / 15, zero point 8
    v[5] = 0
    v[:, :, ::g], v[:, :, 1::g] = -63, 63
    cache = KV4Cache.empty(1, h, n, d, g, dtype)
    kernels.kv4_write(k.to(dtype), v.to(dtype), cache, cu([n]))
    check_finite(kernels.kv4_decode_attention(q, cache, i32(n)), q, cache, [n])
