"""GPU tests of token_logprobs against float64.

Tolerances: a term's exponent (x - m) / T is rounded twice (2^-23 relative) and meets v_exp_f32
(2^-23), so a term is off by (|z| + 1) 2^-22 with e^z: at most 2^-21 of itself after weighting (z e^z
is at most 0.37). Threads, waves and chunks add up to 2^12 terms in turn and then 9 levels: (128 + 9)
2^-24 at most of the positive sum: 2^-16.9, typically its square root. ln s: that, absolute, so
2e-5 at most against |lp| of order 1 to 30, whose own (x - m) / T adds 2^-23 |lp|. Near 0 the sum without
the largest entry is all of lp: relative 2e-5. Entropy: the same sums and |t| / s, 4e-5 (1 + H)."""
from __future__ import annotations

import math

import pytest
import torch

from gpu_util import note

pytestmark = pytest.mark.gpu

INF = float("inf")
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def ctx(wrs):
    c = wrs.Context(0)
    c.use_torch_stream()
    yield c
    torch.cuda.synchronize()
    c.close()


def logits_of(n, v, dtype, seed, sigma=3.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, v, generator=g) * sigma
    hot = torch.randint(v, (n, 3), generator=g)
    x.scatter_add_(1, hot, torch.rand(n, 3, generator=g) * 15)
    return x.to(DT[dtype]).cuda()


def score(wrs, ctx, x, tokens, k, allowed=None, temperature=1.0):
    n = x.shape[0]
    lp, h = torch.full((n,), 9.0, device="cuda"), torch.full((n,), 9.0, device="cuda")
    ids = torch.full((n, k), 9, dtype=torch.int32, device="cuda") if k else None
    top = torch.full((n, k), 9.0, device="cuda") if k else None
    wrs.token_logprobs(x, tokens, lp, entropy=h, top_ids=ids, top_logprobs=top, allowed=allowed,
                       temperature=temperature, ctx=ctx)
    torch.cuda.synchronize()
    return lp, h, ids, top


def expect(x, tokens, k, allowed=None, temperature=1.0):
    x = x.double()
    if allowed is not None:
        x = torch.where(allowed.bool(), x, -INF)
    z = x / temperature
    m = z.amax(1, keepdim=True)
    # ln s as log1p of the sum without the largest entry
    first = (z == m).int().argmax(1, keepdim=True)
    rest = torch.exp(z - m).scatter(1, first, 0.0).sum(1, keepdim=True)
    lse = torch.log1p(rest)
    lp = z - m - lse
    p = torch.exp(lp)
    h = -torch.where(p > 0, p * lp, 0.0).sum(1)
    ok = (tokens >= 0) & (tokens < x.shape[1])
    got = lp.gather(1, tokens.long().clamp(0, x.shape[1] - 1)[:, None])[:, 0]
    lp_t = torch.where(ok, got, -INF)
    order = torch.sort(x, dim=1, descending=True, stable=True)[1][:, :k]
    return lp_t, h, order, lp.gather(1, order)


def close(got, want):
    both = torch.isinf(want) & (got.double() == want)
    return (both | ((got.double() - want).abs() <= 2e-5 * torch.minimum(
        torch.ones_like(want), want.abs()) + 2.0 ** -22 * want.abs())).all()


def check(wrs, ctx, x, tokens, k, allowed=None, temperature=1.0):
    lp, h, ids, top = score(wrs, ctx, x, tokens, k, allowed, temperature)
    w_lp, w_h, w_ids, w_top = expect(x, tokens, k, allowed, temperature)
    assert close(lp, w_lp), (lp.double() - w_lp).abs().max()
    assert ((h.double() - w_h).abs() <= 4e-5 * torch.minimum(w_h + 1e-30, 1 + w_h)).all() or \
        ((h.double() - w_h).abs() <= 4e-5 * w_h + 1e-37).all()
    if k:
        fine = w_top > -INF
        assert torch.equal(ids[fine].long(), w_ids[fine])
        assert (ids[~fine] == -1).all() and (top[~fine] == -INF).all()
        assert close(top, w_top)


def some_tokens(n, v, seed):
    return torch.randint(v, (n,), generator=torch.Generator().manual_seed(seed)).int().cuda()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,v,k", [(1, 51865, 5), (5, 51866, 10), (3, 51864, 32), (130, 51865, 1),
                                   (600, 4099, 7), (2, 1, 1), (3, 2, 2), (4, 7, 7), (2, 31, 31),
                                   (2, 64, 32), (9, 513, 32), (2, 4096, 3), (2, 4097, 3),
                                   (1, 65536, 32), (700, 130, 4), (1, 8191, 2), (1, 8193, 2)])
def test_scores(wrs, ctx, dtype, n, v, k):
    note(f"score {dtype} {n} {v} {k}")
    x = logits_of(n, v, dtype, seed=n + v)
    check(wrs, ctx, x, some_tokens(n, v, 1), k)


@pytest.mark.parametrize("n,v", [(1, 65537), (3, 200_003), (1, 1 << 22), (520, 66_000)])
def test_rows_longer_than_a_workgroup_takes(wrs, ctx, n, v):
    note(f"long rows {n} {v}")
    x = logits_of(n, v, "f16", seed=v)
    check(wrs, ctx, x, some_tokens(n, v, 2), 9)


def test_more_rows_than_a_grid_is_wide(wrs, ctx):
    note("70001 rows")
    x = logits_of(70001, 33, "f16", seed=3)
    check(wrs, ctx, x, some_tokens(70001, 33, 4), 3)


@pytest.mark.parametrize("temperature", [0.2, 0.4, 0.7, 1.0, 3.0, 1e-6, 1e6])
def test_temperature(wrs, ctx, temperature):
    note(f"temperature {temperature}")
    x = logits_of(6, 5000, "f32", seed=3)
    t = float(torch.tensor(temperature, dtype=torch.float32))
    check(wrs, ctx, x, some_tokens(6, 5000, 3), 5, temperature=t)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("kind", ["bool", "uint8"])
@pytest.mark.parametrize("shared", [True, False])
def test_allowed(wrs, ctx, dtype, kind, shared):
    n, v = 12, 51865
    x = logits_of(n, v, dtype, seed=4)
    g = torch.Generator().manual_seed(6)
    ok = torch.rand(1 if shared else n, v, generator=g) < 0.3
    if not shared:
        ok[3] = False        # nothing
        ok[4] = False
        ok[4, 77] = True     # one entry
        ok[5] = False
        ok[5, -2:] = True    # two, for five alternatives
    ok = ok.cuda()
    mask = ok if kind == "bool" else ok.to(torch.uint8) * 200
    tokens = some_tokens(n, v, 5)
    tokens[4] = 77
    note(f"allowed {dtype} {kind} {shared}")
    if shared:
        check(wrs, ctx, x, tokens, 5, allowed=mask)
        return
    full = torch.tensor([i != 3 for i in range(n)], device="cuda")
    lp, h, ids, top = score(wrs, ctx, x, tokens, 5, allowed=mask)
    w = expect(x[full], tokens[full], 5, mask[full])
    assert close(lp[full], w[0]) and close(top[full], w[3])
    assert lp[3] == -INF and h[3] == 0 and (ids[3] == -1).all() and (top[3] == -INF).all()
    assert lp[4] == 0 and h[4] == 0 and ids[4].tolist() == [77, -1, -1, -1, -1]
    assert (ids[5] >= v - 2).sum() == 2 and (ids[5, 2:] == -1).all()
    # the same through wider rows of the mask at an odd address
    wide = torch.zeros(n, v + 3, dtype=mask.dtype, device="cuda")
    wide[:, 1:v + 1] = mask
    again = score(wrs, ctx, x, tokens, 5, allowed=wide[:, 1:v + 1])
    for a, b in zip((lp, h, ids, top), again):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_equal_logits_and_ties(wrs, ctx, dtype):
    v = 51865
    x = torch.zeros(4, v, dtype=DT[dtype], device="cuda")
    x[1, 1::2] = 1.0           # half of them tie at the top
    x[2] = -torch.arange(v, device="cuda").clamp(max=100).to(DT[dtype])
    x[3, ::3] = -0.0           # zeros of both signs are equal
    note(f"ties {dtype}")
    tokens = torch.tensor([5, 1, 3, v - 1], dtype=torch.int32, device="cuda")
    check(wrs, ctx, x, tokens, 32)
    for n in (1, 600):  # split over workgroups, and whole
        check(wrs, ctx, x[:1].expand(n, v).contiguous(), torch.zeros(n, dtype=torch.int32).cuda(), 32)
    up = torch.arange(v, device="cuda").float()[None].repeat(3, 1).to(DT[dtype]) / 512
    check(wrs, ctx, up, some_tokens(3, v, 8), 32)  # rising rows: a thread's entries all count
    check(wrs, ctx, up.flip(1).contiguous(), some_tokens(3, v, 8), 32)


@pytest.mark.parametrize("n", [1, 700])
def test_values_that_are_no_numbers(wrs, ctx, n):
    v = 9001
    x = logits_of(n, v, "f32", seed=7)
    low = torch.finfo(torch.float32).min
    x[0, 4000:] = -INF
    note(f"odd values {n}")
    check(wrs, ctx, x, some_tokens(n, v, 9), 4)
    x[0, 3:] = low  # a mask of the type's lowest value
    check(wrs, ctx, x, some_tokens(n, v, 9), 4)
    x[0] = low      # all of them: an even distribution
    lp, h, ids, top = score(wrs, ctx, x, some_tokens(n, v, 9), 4)
    assert abs(lp[0].item() + math.log(v)) < 1e-4 and abs(h[0].item() - math.log(v)) < 1e-4
    assert ids[0].tolist() == [0, 1, 2, 3]
    x[0] = -INF
    lp, h, ids, top = score(wrs, ctx, x, some_tokens(n, v, 9), 4)
    assert lp[0] == -INF and h[0] == 0 and (ids[0] == -1).all() and (top[0] == -INF).all()
    for bad in (math.nan, INF):
        for at in (0, 8999):
            x[0] = 1.0
            x[0, at] = bad
            lp, h, ids, top = score(wrs, ctx, x, some_tokens(n, v, 9), 4)
            assert lp[0].isnan() and h[0].isnan() and (ids[0] == -1).all() and top[0].isnan().all()
            assert n == 1 or lp[1:].isfinite().all()
            # hidden, it does not count
            ok = torch.ones(1, v, dtype=torch.bool, device="cuda")
            ok[0, at] = False
            check(wrs, ctx, x[:1], some_tokens(1, v, 9), 4, allowed=ok)


def rows_of_many_candidates(v, dtype):
    """Rows of which many entries lie close to the best ones or equal them."""
    i = torch.arange(v, device="cuda")
    g = torch.Generator().manual_seed(13)
    noise = torch.randint(0, 40, (v,), generator=g).cuda()
    ulp = {"f32": 2.0 ** -23, "f16": 2.0 ** -10, "bf16": 2.0 ** -7}[dtype]
    low = -65504.0
    rows = [
        torch.ones(v, device="cuda"),
        1 + noise * ulp,                                    # a narrow band
        (noise % 3).float(),                                # three values
        torch.where(i % 2048 < 128, 5 + (i % 7) * ulp, 0),  # all entries of some threads, f32
        torch.where(i % 4096 < 200, 5.0, low),
        torch.where(i < min(1501, v), noise * 0.125, low),  # the others held down
        torch.where(i >= v - 9, i % 5, low),                # fewer than are asked for, then equal ones
        torch.where(i == v // 2, 1.0, low),
        -(i // 64).float(),                                 # falling steps
        (i // 600).float(),                                 # rising ones
    ]
    return torch.stack([r.float() for r in rows]).to(DT[dtype])


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("v", [300, 2049, 4096, 4097, 8191, 51865, 262144])
@pytest.mark.parametrize("k", [1, 5, 32])
def test_many_candidates(wrs, ctx, dtype, v, k):
    x = rows_of_many_candidates(v, dtype)
    n = x.shape[0]
    note(f"many candidates {dtype} {v} {k}")
    ok = torch.rand(n, v, generator=torch.Generator().manual_seed(v)) < 0.6
    for copies in (1, 30):  # rows split over workgroups where they are long, and whole
        rows = x.repeat(copies, 1)
        tokens = some_tokens(n * copies, v, 3)
        check(wrs, ctx, rows, tokens, k)
        if copies == 1:
            check(wrs, ctx, rows, tokens, k, allowed=ok.cuda())
            for row in range(n):
                check(wrs, ctx, rows[row:row + 1], tokens[row:row + 1], k)


def time_of(call):
    """The least of several means over queued calls, in us."""
    for _ in range(3):
        call()
    best = float("inf")
    for _ in range(5):
        a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        a.record()
        for _ in range(20):
            call()
        b.record()
        torch.cuda.synchronize()
        best = min(best, a.elapsed_time(b) * 50)
    return best


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("n,v,k", [(5, 51866, 10), (1, 51866, 32), (600, 4096, 7), (1, 262144, 32),
                                   (130, 51865, 32)])
def test_time_does_not_depend_on_values(wrs, ctx, dtype, n, v, k):
    """Rows of many candidates take no more than three times what random ones do (ranked one against all
    the others they took up to two hundred times that)."""
    outs = [torch.zeros(n, k, dtype=torch.int32, device="cuda"), torch.zeros(n, k, device="cuda")]
    h = torch.zeros(n, device="cuda")

    def took(x):
        return time_of(lambda: wrs.token_logprobs(x, entropy=h, top_ids=outs[0], top_logprobs=outs[1],
                                                  ctx=ctx))
    note(f"times {dtype} {n} {v} {k}")
    usual = took(logits_of(n, v, dtype, seed=1))
    for i, row in enumerate(rows_of_many_candidates(v, dtype)):
        us = took(row.repeat(n, 1))
        assert us <= 3 * usual, f"row {i}: {us:.1f} us, random values {usual:.1f}"


def check_far(wrs, ctx, x, tokens, k, allowed=None, temperature=1.0):
    """check(), of rows whose smallest terms may lie below 2^-126: those come as zero, which is off by
    v 2^-126 < 1e-33 in the sum and 88 times that in the entropy. Log probabilities past f32's range are
    -infinity."""
    lp, h, ids, top = score(wrs, ctx, x, tokens, k, allowed, temperature)
    w_lp, w_h, w_ids, w_top = expect(x, tokens, k, allowed, temperature)
    most = torch.finfo(torch.float32).max
    for got, want in ((lp, w_lp), (top, w_top)):
        want = torch.where(want < -most, -INF, want)
        small = (want.abs() < 1e-27) & ((got.double() - want).abs() <= 1e-33 + 2e-5 * want.abs())
        assert close(torch.where(small, 0.0, got), torch.where(small, 0.0, want))
    assert ((h.double() - w_h).abs() <= 4e-5 * w_h + 1e-31).all()
    assert torch.equal(ids.long(), w_ids)


def far_rows(dtype, far):
    """Rows with entries far from zero, or far from each other, all finite in `dtype`."""
    v = 51865
    x = logits_of(6, v, "f32", seed=5)
    x[0, 1501:] = far          # all but the first ones held down by a finite mask
    x[1, :v - 9] = far         # all but the last ones
    x[2] += far                # every entry there
    x[3, 1::2] = far
    x[4] = far                 # all equal
    x[5, 100:200] -= far / 2   # some far up
    return x.to(DT[dtype])


@pytest.mark.parametrize("dtype,far", [
    *(("f32", f) for f in (-1e7, -1e9, -3e9, -1e10, -2e10, -5e10, -1e12, -3e15, -1e20, -1e25, -9e29, -1e32)),
    ("bf16", -1e10), ("bf16", -3e15), ("bf16", -1e29), ("f16", -65504.0)])
@pytest.mark.parametrize("copies", [1, 60])
def test_entries_far_from_zero(wrs, ctx, dtype, far, copies):
    """Masks of any finite value, rows split over workgroups and whole."""
    x = far_rows(dtype, far).repeat(copies, 1)
    tokens = some_tokens(x.shape[0], x.shape[1], 11)
    ok = torch.ones(1, x.shape[1], dtype=torch.bool, device="cuda")
    for temperature in (1.0, 0.7):
        note(f"far entries {dtype} {far} {copies} {temperature}")
        t = float(torch.tensor(temperature, dtype=torch.float32))
        check_far(wrs, ctx, x, tokens, 5, temperature=t)
        check_far(wrs, ctx, x, tokens, 5, allowed=ok, temperature=t)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("temperature", [1e-7, 1e-8, 1e-9, 3e-10, 1e-11, 1e-20, 1e-30, 1e-37])
@pytest.mark.parametrize("n", [3, 300])
def test_temperatures_next_to_zero(wrs, ctx, dtype, temperature, n):
    note(f"cold {dtype} {temperature} {n}")
    x = logits_of(n, 9001, dtype, seed=8)
    x[0, 100:] = x[0, 0]
    x[1] = x[1, 0]  # all equal
    t = float(torch.tensor(temperature, dtype=torch.float32))
    check_far(wrs, ctx, x, some_tokens(n, 9001, 12), 5, temperature=t)


def test_confident_rows_keep_their_precision(wrs, ctx):
    """Log probabilities close to 0, with the likeliest entry anywhere."""
    v = 51865
    for n, at in ((4, 0), (4, 51864), (4, 12345), (600, 30000)):
        x = torch.full((n, v), -30.0, device="cuda")
        x[:, 7] = -5.0
        x[:, at] = 9.0
        note(f"confident {n} {at}")
        lp = score(wrs, ctx, x, torch.full((n,), at, dtype=torch.int32, device="cuda"), 1)[0]
        w = expect(x, torch.full((n,), at, device="cuda"), 1)[0]
        assert ((lp.double() - w).abs() <= 2e-5 * w.abs()).all() and (w.abs() < 1e-5).all()


def test_tokens_that_are_no_entries(wrs, ctx):
    x = logits_of(4, 100, "f32", seed=2)
    t = torch.tensor([-1, 100, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32, device="cuda")
    note("no entries")
    assert (score(wrs, ctx, x, t, 0)[0] == -INF).all()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_strided_rows_at_odd_places(wrs, ctx, dtype):
    n, v = 6, 5003
    x = logits_of(n, v, dtype, seed=5)
    wide = torch.full((n, v + 9), 99.0, dtype=DT[dtype], device="cuda")
    note(f"strides {dtype}")
    want = score(wrs, ctx, x, some_tokens(n, v, 1), 6)
    for off in (1, 2, 3, 5):
        wide.fill_(99.0)
        wide[:, off:off + v] = x
        for a, b in zip(want, score(wrs, ctx, wide[:, off:off + v], some_tokens(n, v, 1), 6)):
            assert torch.equal(a, b)


def test_outputs_that_are_left_out(wrs, ctx):
    n, v = 3, 3000
    x, t = logits_of(n, v, "f32", seed=1), some_tokens(n, v, 1)
    lp, h, ids, top = score(wrs, ctx, x, t, 4)
    note("left out")
    only = torch.zeros(n, device="cuda")
    wrs.token_logprobs(x, t, only, ctx=ctx)
    assert torch.equal(only, lp)
    only = torch.zeros(n, device="cuda")
    wrs.token_logprobs(x, entropy=only, ctx=ctx)
    assert torch.equal(only, h)
    i = torch.zeros(n, 4, dtype=torch.int32, device="cuda")
    wrs.token_logprobs(x, top_ids=i, ctx=ctx)
    assert torch.equal(i, ids)
    p = torch.zeros(n, 4, device="cuda")
    wrs.token_logprobs(x, top_logprobs=p, ctx=ctx)
    assert torch.equal(p, top)


def test_captured_scores_replay(wrs):
    """A captured call replays on new logits, unsplit where it was captured first, and split."""
    stream = torch.cuda.Stream()
    c = wrs.Context(0)
    n, v, k = 3, 51865, 8
    with torch.cuda.stream(stream):
        c.use_torch_stream()
        x = logits_of(n, v, "f32", seed=1)
        t = some_tokens(n, v, 1)
        lp, h, top = (torch.zeros(s, device="cuda") for s in ((n,), (n,), (n, k)))
        ids = torch.zeros(n, k, dtype=torch.int32, device="cuda")
        stream.synchronize()
        graphs = []
        for eager_first in (False, True):
            note(f"captured score {eager_first}")
            if eager_first:
                score(wrs, c, x, t, k)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=stream):
                wrs.token_logprobs(x, t, lp, entropy=h, top_ids=ids, top_logprobs=top, ctx=c)
            graphs.append(g)
        for turn in range(4):
            for g in graphs:
                x.copy_(logits_of(n, v, "f32", seed=10 + turn))
                g.replay()
                stream.synchronize()
                w = expect(x, t, k)
                assert close(lp, w[0]) and close(top, w[3]) and torch.equal(ids.long(), w[2])
                check(wrs, c, x, t, k)
        long = logits_of(1, 70_000, "f16", seed=1)
        one = torch.zeros(1, device="cuda")
        fresh = wrs.Context(0)
        fresh.use_torch_stream()
        g = torch.cuda.CUDAGraph()
        stream.synchronize()
        with torch.cuda.graph(g, stream=stream):
            with pytest.raises(RuntimeError, match="reserve"):
                wrs.token_logprobs(long, entropy=one, ctx=fresh)
            one.zero_()
        g.replay()
        fresh.reserve(n_heads=1, decode_rows=1, decode_keys=1)
        g2 = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g2, stream=stream):
            wrs.token_logprobs(long, entropy=one, ctx=fresh)
        g2.replay()
        stream.synchronize()
        w = expect(long, torch.zeros(1, device="cuda"), 1)[1]
        assert abs(one.item() - w.item()) < 4e-5 * (1 + w.item())
        del graphs, g, g2
    torch.cuda.synchronize()


def test_repeated_calls_give_the_same_bits(wrs, ctx):
    for n in (1, 5, 600):
        x = logits_of(n, 51865, "f16", seed=n)
        first = score(wrs, ctx, x, some_tokens(n, 51865, 1), 10)
        note(f"repeat {n}")
        for _ in range(4):
            for a, b in zip(first, score(wrs, ctx, x, some_tokens(n, 51865, 1), 10)):
                assert torch.equal(a, b)


def test_refusals(wrs, ctx):
    x = logits_of(3, 100, "f32", seed=1)
    t, lp = some_tokens(3, 100, 1), torch.full((3,), 5.0, device="cuda")
    ids = torch.zeros(3, 33, dtype=torch.int32, device="cuda")
    note("score refusals")
    bad = [dict(temperature=0.0), dict(temperature=-1.0), dict(temperature=math.nan),
           dict(temperature=INF), dict(temperature=1e-39)]
    for b in bad:
        with pytest.raises(AssertionError):
            wrs.token_logprobs(x, t, lp, ctx=ctx, **b)
    with pytest.raises(AssertionError):
        wrs.token_logprobs(x, ctx=ctx)
    with pytest.raises(AssertionError):
        wrs.token_logprobs(x, t, ctx=ctx)
    with pytest.raises(AssertionError):
        wrs.token_logprobs(x, t[:2], lp[:2], ctx=ctx)
    with pytest.raises(AssertionError):
        wrs.token_logprobs(x[:, :0], t, lp, ctx=ctx)
    with pytest.raises(RuntimeError):
        wrs.token_logprobs(x, top_ids=ids, ctx=ctx)  # more than 32
    with pytest.raises(RuntimeError):
        wrs.token_logprobs(x[:, :4], top_ids=ids[:, :5].contiguous(), ctx=ctx)
    with pytest.raises(TypeError):
        wrs.token_logprobs(x, t.long(), lp, ctx=ctx)
    with pytest.raises(TypeError):
        wrs.token_logprobs(x, t, lp.half(), ctx=ctx)
    with pytest.raises(TypeError):
        wrs.token_logprobs(x.cpu(), t, lp, ctx=ctx)
    with pytest.raises(TypeError):
        wrs.token_logprobs(x.T, t, lp, ctx=ctx)
    with pytest.raises(TypeError):
        wrs.token_logprobs(x, t, lp, allowed=torch.ones(3, 100, device="cuda"), ctx=ctx)
    with pytest.raises(AssertionError):
        wrs.token_logprobs(x, t, lp, allowed=torch.ones(2, 100, dtype=torch.bool).cuda(), ctx=ctx)
    lib = ctx._lib
    p = x.data_ptr()

    def raw(dtype=0, ptr=p, length=300, rs=100, n=3, v=100, ok=None, ok_len=0, ok_rs=0, tp=t.data_ptr(),
            out=lp.data_ptr(), k=0, i=None):
        return lib.wrs_token_logprobs(ctx.handle, dtype, ptr, length, rs, n, v, ok, ok_len, ok_rs, 1.0,
                                      tp, out, None, k, i, None)
    m = torch.ones(300, dtype=torch.uint8, device="cuda").data_ptr()
    for b, rc in ((dict(dtype=3), wrs._lib.WRS_EUNSUPPORTED), (dict(ptr=None), -1),
                  (dict(length=299), -1), (dict(rs=99), -1), (dict(rs=-100), -1),
                  (dict(rs=2 ** 62), -1), (dict(ptr=p + 2), -1), (dict(tp=t.data_ptr() + 1), -1),
                  (dict(tp=None), -1), (dict(out=None), -1), (dict(v=0), -1),
                  (dict(ok=m, ok_len=299, ok_rs=100), -1), (dict(ok=m, ok_len=300, ok_rs=50), -1),
                  (dict(ok=m, ok_len=99), -1), (dict(k=2), -1), (dict(i=ids.data_ptr()), -1)):
        assert raw(**b) == rc, b
    torch.cuda.synchronize()
    assert (lp == 5.0).all()
    assert raw(n=0) == 0 and raw(ok=m, ok_len=100) == 0
    torch.cuda.synchronize()
