"""GPU tests of prompt_attention against softmax(q k^T scale) v in 64 bits, one
sequence at a time. Tolerance: with u the unit roundoff of the type (2^-8 bf16,
2^-11 fp16), probabilities rounded to the type move an output by at most u
sum p|v|, the rounded output by u|out|; a score is a D-term fp32 dot product,
off by at most e = (D + 4) 2^-24 scale sum|q k|, which moves each p by a factor
within exp(+-2e), and the fp32 exponential, sum and product add at most
2^-16 sum p|v| (256 roundings of 2^-24)."""

from __future__ import annotations

import pytest
import torch

from tritonforge_b200 import _lib, kernels

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def cu(lens):
    return torch.tensor([0] + list(lens)).cumsum(0).to(torch.int32).cuda()


def reference(q, k, v, lq, lk, causal, scale):
    """(out, tolerance) in fp64; masked positions take no part whatever they hold."""
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    u = U[q.dtype]
    hq, hkv, d = q.shape[1], k.shape[1], q.shape[2]
    i = j = 0
    for n, m in zip(lq, lk):
        for a in range(0, n, 512):
            b = min(n, a + 512)
            hi = min(m, b + m - n) if causal else m
            if hi <= 0:
                continue
            qs = q[i + a:i + b].double().transpose(0, 1)
            ks = k[j:j + hi].double().transpose(0, 1).repeat_interleave(hq // hkv, 0)
            vs = v[j:j + hi].double().transpose(0, 1).repeat_interleave(hq // hkv, 0)
            see = torch.ones(b - a, hi, dtype=torch.bool, device=q.device)
            if causal:
                see = torch.arange(hi, device=q.device)[None] <= torch.arange(a, b, device=q.device)[:, None] + m - n
            s = torch.where(see, qs @ ks.transpose(1, 2) * scale, -torch.inf)
            e = torch.where(see, qs.abs() @ ks.abs().transpose(1, 2) * scale, 0).amax(-1, keepdim=True)
            e = torch.expm1(2 * (d + 4) * 2.0 ** -24 * e)
            mx = s.amax(-1, keepdim=True)
            p = torch.exp(s - torch.where(mx == -torch.inf, 0, mx))
            p = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
            # a query at a time where masked values are not finite: 0 x NaN must not enter
            clean = torch.isfinite(vs).all() and torch.isfinite(ks).all()
            if clean:
                o, av = p @ vs, p @ vs.abs()
            else:
                w = torch.where((see & torch.ones_like(p, dtype=torch.bool))[..., None], p[..., None] * vs[:, None], 0)
                o, av = w.sum(-2), w.abs().sum(-2)
            o, av = (torch.where(see.any(-1)[None, :, None], t, 0) for t in (o, av))
            out[i + a:i + b] = o.transpose(0, 1)
            tol[i + a:i + b] = (u * o.abs() + (u + 2.0 ** -16 + e) * av).transpose(0, 1)
        i, j = i + n, j + m
    return out, tol


def check(got, q, k, v, lq, lk, causal=True, scale=None):
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    want, tol = reference(q, k, v, lq, lk, causal, scale)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), "NaN in other places"
    bad = (got.double() - want).abs() > tol + 1e-30
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, first at {bad.nonzero()[0].tolist()}"


def inputs(tq, tk, hq, hkv, d, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + tq * 3 + tk + hq)
    q = torch.randn(tq, hq, d, device="cuda", generator=g).to(dtype)
    k = (torch.randn(tk, hkv, d, device="cuda", generator=g) * 1.5).to(dtype)
    v = torch.randn(tk, hkv, d, device="cuda", generator=g).to(dtype)
    return q, k, v


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hq,hkv,d", [(14, 2, 64), (28, 4, 128), (64, 8, 128), (8, 8, 64), (10, 2, 128), (16, 1, 64)])
@pytest.mark.parametrize("lens", [[1], [37], [128, 1, 0, 129], [0, 3, 260, 17, 0], [511], [700, 1, 1, 300]])
def test_packed_causal(hq, hkv, d, lens, dtype):
    q, k, v = inputs(sum(lens), sum(lens), hq, hkv, d, dtype)
    got = kernels.prompt_attention(q, k, v, cu(lens))
    check(got, q, k, v, lens, lens)
    assert torch.equal(got, kernels.prompt_attention(q, k, v, cu(lens))), "two runs differ"


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hq,hkv,d", [(14, 2, 64), (28, 4, 128), (32, 8, 128)])
@pytest.mark.parametrize("lq,lk", [([1, 1, 1], [1, 500, 2049]), ([5, 64, 33], [5, 1000, 128 + 33]),
                                   ([130], [4001]), ([20, 7], [4, 0]), ([300, 2], [290, 600]), ([1], [30000])])
def test_earlier_positions(hq, hkv, d, lq, lk, dtype):
    """More keys than queries (a later chunk, single tokens), and fewer: queries that see nothing give zeros."""
    q, k, v = inputs(sum(lq), sum(lk), hq, hkv, d, dtype)
    got = kernels.prompt_attention(q, k, v, cu(lq), cu(lk))
    check(got, q, k, v, lq, lk)
    if lq[0] > lk[0]:
        assert (got[:lq[0] - lk[0]] == 0).all()


@pytest.mark.parametrize("lq,lk", [([40, 200], [40, 200]), ([1, 150, 9], [700, 0, 130])])
@pytest.mark.parametrize("hq,hkv,d", [(28, 4, 128), (8, 8, 64)])
def test_not_causal(hq, hkv, d, lq, lk):
    q, k, v = inputs(sum(lq), sum(lk), hq, hkv, d, torch.bfloat16)
    check(kernels.prompt_attention(q, k, v, cu(lq), cu(lk), causal=False), q, k, v, lq, lk, causal=False)


def test_long_prompt():
    q, k, v = inputs(5003, 5003, 14, 2, 64, torch.bfloat16)
    check(kernels.prompt_attention(q, k, v, cu([5003])), q, k, v, [5003], [5003])


def test_views_of_the_projection_and_out():
    """q, k, v as views of fused q|k|v rows, an output with padded rows, another scale."""
    hq, hkv, d, lens = 28, 4, 128, [70, 333]
    t = sum(lens)
    g = torch.Generator(device="cuda").manual_seed(5)
    qkv = torch.randn(t, (hq + 2 * hkv) * d + 16, device="cuda", generator=g).bfloat16()
    q = qkv[:, :hq * d].view(t, hq, d)
    k = qkv[:, hq * d:(hq + hkv) * d].view(t, hkv, d)
    v = qkv[:, (hq + hkv) * d:(hq + 2 * hkv) * d].view(t, hkv, d)
    buf = torch.full((t, hq, d + 8), 7.0, device="cuda", dtype=torch.bfloat16)
    got = kernels.prompt_attention(q, k, v, cu(lens), scale=0.2, out=buf[..., :d])
    check(got, q, k, v, lens, lens, scale=0.2)
    assert (buf[..., d:] == 7).all()
    # heads before tokens in memory, and rows off a 16-byte boundary
    kt, vt = k.transpose(0, 1).contiguous().transpose(0, 1), v.transpose(0, 1).contiguous().transpose(0, 1)
    odd = torch.empty(t * hq * d + 1, device="cuda", dtype=torch.bfloat16)[1:].view(t, hq, d).copy_(q)
    assert torch.equal(kernels.prompt_attention(odd, kt, vt, cu(lens), scale=0.2), got)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_masked_places_may_hold_anything(bad, d):
    """Non-finite keys and values touch only the queries that see them: not
    earlier queries of their sequence, nor other sequences in the same tile."""
    lens = [50, 90, 30]
    q, k, v = inputs(170, 170, 8, 2, d, torch.bfloat16)
    want = kernels.prompt_attention(q, k, v, cu(lens))
    v2, k2 = v.clone(), k.clone()
    v2[100] = bad  # position 50 of the second sequence
    got = kernels.prompt_attention(q, k, v2, cu(lens))
    ok = torch.ones(170, dtype=torch.bool, device="cuda")
    ok[100:140] = False
    assert torch.equal(got[ok], want[ok])
    assert not torch.isfinite(got[100:140].float()).any()
    check(got, q, k, v2, lens, lens)
    k2[100] = bad
    got = kernels.prompt_attention(q, k2, v, cu(lens))
    assert torch.equal(got[ok], want[ok])


def test_extreme_scores():
    """Scores far apart and far from zero: the running maximum carries them."""
    lens = [400]
    q, k, v = inputs(400, 400, 7, 1, 128, torch.float16)
    k = (k * torch.linspace(0.1, 20, 400, device="cuda")[:, None, None]).half()
    check(kernels.prompt_attention(q * 4, k, v, cu(lens)), q * 4, k, v, lens, lens)
    check(kernels.prompt_attention(q * 4, -k.flip(0), v, cu(lens)), q * 4, -k.flip(0), v, lens, lens)


def test_no_tokens_and_side_stream():
    q, k, v = inputs(0, 0, 8, 2, 64, torch.float16)
    assert kernels.prompt_attention(q, k, v, cu([])).shape == (0, 8, 64)
    assert kernels.prompt_attention(q, k, v, cu([0, 0])).shape == (0, 8, 64)
    q, k, v = inputs(200, 200, 8, 2, 64, torch.float16)
    want = kernels.prompt_attention(q, k, v, cu([200]))
    offs = cu([200])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = kernels.prompt_attention(q, k, v, offs)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)


@pytest.mark.parametrize("d", [64, 128])
def test_masked_places_of_split_keys(d):
    """The same where the keys of a few queries are split between CTAs."""
    lq, lk = [3, 5, 40], [4000, 3000, 2500]
    q, k, v = inputs(sum(lq), sum(lk), 8, 2, d, torch.float16)
    cuq, cuk = cu(lq), cu(lk)
    want = kernels.prompt_attention(q, k, v, cuq, cuk)
    check(want, q, k, v, lq, lk)
    v2 = v.clone()
    v2[6998] = float("nan")  # the last but one position of the second sequence: its last two queries see it
    got = kernels.prompt_attention(q, k, v2, cuq, cuk)
    seen = torch.zeros(48, dtype=torch.bool, device="cuda")
    seen[6:8] = True
    assert torch.isnan(got[seen].float()).all()
    check(got, q, k, v2, lq, lk)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hq,hkv,d,lq,lk", [
    (64, 8, 128, [610], [5003]),                                          # a few pairs more than SMs
    (64, 8, 128, [242, 69, 390], [2595, 3091, 3313]),
    (64, 8, 128, [3] * 40, [2000 + 17 * i for i in range(40)]),           # more than a warp of sequences
    (64, 8, 128, [0, 200, 0, 0, 390, 5], [0, 4100, 900, 0, 3, 4090]),     # pairs fewer than their bound, keys fewer than queries
    (28, 4, 128, [1500], [4000]),
    (14, 2, 64, [3000, 10], [9100, 2300]),
])
def test_pairs_beyond_whole_rounds(hq, hkv, d, lq, lk, dtype):
    """Pairs of tiles for a little more than one or two rounds of the SMs: the rest is cut into ranges of keys."""
    q, k, v = inputs(sum(lq), sum(lk), hq, hkv, d, dtype)
    got = kernels.prompt_attention(q, k, v, cu(lq), cu(lk))
    check(got, q, k, v, lq, lk)
    assert torch.equal(got, kernels.prompt_attention(q, k, v, cu(lq), cu(lk))), "two runs differ"


def test_masked_places_beyond_whole_rounds():
    """The last key's value is NaN: it shows in the last query alone, cut pairs and whole ones alike."""
    q, k, v = inputs(610, 5003, 64, 8, 128, torch.bfloat16)
    v[-1] = 0
    want = v.clone()
    v[-1] = float("nan")
    got = kernels.prompt_attention(q, k, v, cu([610]), cu([5003]))
    assert torch.isnan(got[-1]).all()
    check(got[:-1], q[:-1], k[:-1], want[:-1], [609], [5002])


def test_a_nan_in_every_pair():
    """12000 prompts of two tokens, a pair of tiles each, with a NaN in one channel
    of every second token's value: each of a CTA's 81 or more pairs meets it. The
    first tokens see their own value alone, so they return it exactly."""
    n, h, d = 12000, 128, 64
    q, k, v = inputs(2 * n, 2 * n, h, 1, d, torch.bfloat16)
    v[1::2, :, 5] = float("nan")
    got = kernels.prompt_attention(q, k, v, cu([2] * n))
    assert torch.equal(got[0::2], v[0::2].expand(n, h, d))
    assert torch.isnan(got[1::2, :, 5]).all()
    keep = [c for c in range(d) if c != 5]
    for a in range(0, n, 1000):  # the second tokens: two weights each
        qs = q[2 * a + 1:2 * a + 2001:2].double()
        ks, vs = (t[2 * a:2 * a + 2000].double().view(1000, 2, d) for t in (k, v))
        p = torch.softmax(qs @ ks.transpose(1, 2) * d ** -0.5, -1)
        e = (qs.abs() @ ks.abs().transpose(1, 2) * d ** -0.5).amax(-1, keepdim=True)
        e = torch.expm1(2 * (d + 4) * 2.0 ** -24 * e)
        vs = vs[..., keep]
        want, av = p @ vs, p @ vs.abs()
        off = (got[2 * a + 1:2 * a + 2001:2][..., keep].double() - want).abs()
        u = U[torch.bfloat16]
        assert (off <= u * want.abs() + (u + 2.0 ** -16 + e) * av).all()
    assert _lib.prompt_workspaces.errors() == 0


def poison(v, places):
    """v with (key, channels, value) set in every head; the channels that stay as they were."""
    v, d = v.clone(), v.shape[2]
    for key, channels, x in places:
        v[key, :, channels] = x
    bad = {c for _, channels, _ in places for c in channels}
    return v, [c for c in range(d) if c not in bad]


INF, NAN = float("inf"), float("nan")


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hq,hkv,d,lq,lk", [
    (8, 2, 64, 6000, 6000), (14, 2, 64, 6000, 6000), (8, 2, 128, 3001, 6000), (64, 8, 128, 610, 6000),
    (8, 2, 64, 16, 70000), (8, 8, 128, 40, 70000)])
def test_values_that_are_not_finite_stay_in_their_channel(hq, hkv, d, lq, lk, dtype):
    """Single values that are infinite or NaN, seen by nearly every query, by some and
    by none: a query's output is the infinity, or NaN where it sees both signs or a
    NaN, in these channels alone; all else comes out bit for bit as without them."""
    q, k, v = inputs(lq, lk, hq, hkv, d, dtype)
    late = lk - lq // 2 - 3
    places = [(3, [7], NAN), (10, [9], INF), (late, [9], -INF), (lk // 2, [1], -INF), (late, [40], INF),
              (lk - 1, [d - 1, 33], NAN), (5, [33], INF)]
    bad, same = poison(v, places)
    want = kernels.prompt_attention(q, k, v, cu([lq]), cu([lk]))
    got = kernels.prompt_attention(q, k, bad, cu([lq]), cu([lk]))
    assert torch.equal(got[..., same], want[..., same])
    pos = torch.arange(lk - lq, lk, device="cuda")[:, None].expand(lq, hq)
    for c in sorted(set(range(d)) - set(same)):
        seen = {s: torch.zeros(lq, hq, dtype=torch.bool, device="cuda") for s in ("nan", "up", "down")}
        for key, channels, x in places:
            if c in channels:
                seen["nan" if x != x else "up" if x > 0 else "down"] |= pos >= key
        nan = seen["nan"] | (seen["up"] & seen["down"])
        expect = torch.where(seen["up"], INF, torch.where(seen["down"], -INF, want[..., c].float()))
        assert torch.equal(torch.isnan(got[..., c]), nan), c
        assert torch.equal(got[..., c].float()[~nan], expect[~nan]), c
    assert _lib.prompt_workspaces.errors() == 0


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lq,lk", [([700, 300], [700, 300]), ([9, 4], [9000, 5000])])
def test_keys_and_queries_that_are_not_finite(lq, lk, d):
    """NaN in a key: the whole rows that see it are NaN, also where a value is infinite; NaN in a query: its row."""
    q, k, v = inputs(sum(lq), sum(lk), 8, 2, d, torch.bfloat16)
    want = kernels.prompt_attention(q, k, v, cu(lq), cu(lk))
    k[lk[0] - 5, 1, 3] = NAN  # kv head 1 (query heads 4 to 7): the first sequence's last five queries
    v[2, 1, 6] = INF
    q[-2, 2, 0] = NAN
    got = kernels.prompt_attention(q, k, v, cu(lq), cu(lk))
    nan = torch.zeros_like(got, dtype=torch.bool)
    nan[lq[0] - 5:lq[0], 4:] = True
    nan[-2, 2] = True
    inf = torch.zeros_like(nan)
    inf[max(0, 2 - lk[0] + lq[0]):lq[0], 4:, 6] = True
    inf &= ~nan
    assert torch.equal(torch.isnan(got), nan)
    assert (got[inf] == INF).all()
    assert torch.equal(got[~(nan | inf)], want[~(nan | inf)])


def test_not_causal_values_that_are_not_finite():
    """Every query of the sequence sees the value, no query of the other does."""
    lens = [130, 70]
    q, k, v = inputs(200, 200, 28, 4, 128, torch.float16)
    want = kernels.prompt_attention(q, k, v, cu(lens), causal=False)
    v[150, 1, 77] = NAN
    got = kernels.prompt_attention(q, k, v, cu(lens), causal=False)
    nan = torch.zeros_like(got, dtype=torch.bool)
    nan[130:, 7:14, 77] = True
    assert torch.equal(torch.isnan(got), nan) and torch.equal(got[~nan], want[~nan])
