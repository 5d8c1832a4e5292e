"""GPU tests of window attention over the KV arena and of attention over 8-bit arenas, against a
float64 softmax over the values that the arena holds.

Tolerances. With S the largest sum of |q_i k_i| / 8 over a visible pair: a score is off by the
split of q (2^-22 of each product) and the f32 sums of 64 products on the matrix pipe (8
roundings, 2^-21), so by (2^-22 + 2^-21 + 2^-23) S at most, scaling and powers of two being exact
but for the factor of q (2^-24, within the last term). A weight is off by that, by v_exp_f32
(2^-23 and the 2^-24 of its argument's rounding at up to 2^5: 2^-19) and by its parts: 2^-22 for
f16 ones, 0 for f32. An output is a mean with these weights on both
sides of a quotient: 2 dw max|v|, and its f32 sums of n keys, added 32 at a time on four waves,
(n / 128 + 12) 2^-24 max|v|."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from gpu_util import note

pytestmark = pytest.mark.gpu

D = 64
INF = float("inf")


def _dtype(wrs, name):
    return {"f16": wrs.WRS_F16, "f32": wrs.WRS_F32, "i8": wrs.WRS_I8}[name]


@pytest.fixture(scope="module")
def ctx(wrs):
    c = wrs.Context(0)
    c.use_torch_stream()
    yield c
    torch.cuda.synchronize()
    c.close()


def stored(x, name):
    """What an arena keeps of f32 rows, in float64."""
    if name == "f32":
        return x.double()
    if name == "f16":
        return x.half().double()
    b = x.double().reshape(-1, D)
    top = b.abs().amax(1, keepdim=True)
    e = torch.frexp(top)[1].double() - 7
    e = torch.where(top * torch.exp2(-e) >= 127.5, e + 1, e).clamp(-126, 121)
    out = torch.round(b * torch.exp2(-e)).clamp(-127, 127) * torch.exp2(e)
    out[~b.isfinite().all(1)] = math.nan
    return out.reshape(x.shape)


def normal(*shape, seed, sigma=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * sigma).cuda()


def attend64(q, k, v, hide):
    """softmax(q k^T / 8) v per head over what is not hidden, and the tolerance of its rows."""
    heads = q.shape[1] // D
    out = torch.empty(q.shape, dtype=torch.float64, device="cuda")
    worst = torch.zeros((), dtype=torch.float64, device="cuda")
    q = q.double()
    for h in range(heads):
        c = slice(h * D, (h + 1) * D)
        vis = (~hide).any(0)
        kk = torch.where(vis[:, None], k[:, c], 0.0)
        vv = torch.where(vis[:, None], v[:, c], 0.0)
        s = q[:, c] @ kk.T.contiguous() / 8
        s = torch.where(hide, -INF, s)
        p = torch.exp(s - s.amax(1, keepdim=True))
        p = torch.where(hide, 0.0, p)
        odd = ~vv.isfinite()
        o = p @ torch.where(odd, 0.0, vv)
        for j in odd.any(1).nonzero()[:, 0].tolist():  # added where the row sees the key
            x = torch.where(odd[j], p[:, j:j + 1] * vv[j], 0.0)
            o += torch.where(hide[:, j:j + 1], 0.0, x)
        out[:, c] = o / p.sum(1, keepdim=True)
        big = q[:, c].abs() @ kk.abs().T.contiguous() / 8
        worst = torch.maximum(worst, torch.where(hide, 0.0, big).max())
    return out, worst.item()


def tolerance(name, worst, v, n):
    parts = {"f16": 2.0 ** -22, "i8": 2.0 ** -22, "f32": 0.0}[name]
    dw = worst * (2.0 ** -22 + 2.0 ** -21 + 2.0 ** -23) + 2.0 ** -19 + parts
    vmax = v[v.isfinite()].abs().max().item()
    return vmax * (2 * dw + (n / 128 + 12) * 2.0 ** -24)


def hidden(past, n, window, sinks):
    at = past + torch.arange(n, device="cuda")[:, None]
    j = torch.arange(past + n, device="cuda")[None]
    return (j > at) | ((j <= at - window) & (j >= sinks))


class Session:
    """An arena of one type whose slots hold `pasts` rows and `counts` new ones, in layer 1 of 2."""

    def __init__(self, wrs, ctx, name, heads, pasts, counts, seed, spoil=None, sigma=1.0, room=0):
        self.name, self.heads, self.pasts, self.counts = name, heads, pasts, counts
        d = heads * D
        most = max(p + n for p, n in zip(pasts, counts)) + room
        self.arena = wrs.KvArena(2, len(pasts), heads, most, 0, ctx=ctx, dtype=_dtype(wrs, name))
        self.rows = []
        for i, (p, n) in enumerate(zip(pasts, counts)):
            k = normal(p + n, d, seed=seed + 3 * i, sigma=sigma)
            v = normal(p + n, d, seed=seed + 3 * i + 1, sigma=sigma)
            if spoil:
                spoil(i, k, v)
            self.rows.append((k, v))
        fill = [p + n for p, n in zip(pasts, counts)]
        self.arena.append_rows(1, list(range(len(pasts))), fill, torch.cat([k for k, _ in self.rows]),
                               torch.cat([v for _, v in self.rows]))
        for i, p in enumerate(pasts):
            self.arena.advance(i, p)
        self.q = normal(sum(counts), d, seed=seed + 2)

    def expect(self, window, sinks, which=None):
        outs, tol, row = [], 0.0, 0
        for i, (p, n) in enumerate(zip(self.pasts, self.counts)):
            if n == 0:
                continue
            k, v = (stored(x, self.name) for x in self.rows[i])
            hide = hidden(p, n, window, sinks)
            o, worst = attend64(self.q[row:row + n], k, v, hide)
            seen = min(p + n, window + n + sinks)
            tol = max(tol, tolerance(self.name, worst, v, seen))
            outs.append(o)
            row += n
        return torch.cat(outs), tol

    def run(self, window, sinks, q=None, out=None):
        q = self.q if q is None else q
        out = torch.full(self.q.shape, 7.0, device="cuda") if out is None else out
        self.arena.window_self(1, list(range(len(self.pasts))), self.counts, window, sinks, q, out)
        torch.cuda.synchronize()
        return out

    def check(self, window, sinks):
        want, tol = self.expect(window, sinks)
        got = self.run(window, sinks)
        err = (got.double() - want).abs().max().item()
        assert err <= tol, f"{err} > {tol}"


CASES = [
    # heads, pasts, counts, window, sinks
    (6, [441], [1], 128, 4),
    (1, [0], [1], 1, 0),
    (2, [0], [5], 1, 0),
    (2, [1], [1], 1, 1),
    (2, [31], [1], 32, 0),
    (2, [32], [1], 32, 0),
    (2, [33], [2], 32, 1),
    (3, [63, 0, 7], [1, 1, 1], 5, 2),
    (2, [100], [16], 16, 3),
    (2, [100], [17], 17, 33),
    (2, [95], [33], 31, 32),
    (2, [96], [40], 33, 64),
    (2, [500, 3, 77], [31, 64, 1], 47, 5),
    (1, [700], [130], 64, 200),
    (2, [900], [1], 2000, 4),
    (2, [900], [3], 300, 900),
    (4, [5000], [1], 4096, 4),
    (2, [5003], [19], 2048, 16),
    (1, [9000], [2], 9001, 0),
    (2, [2900, 2897, 2894], [33, 28, 30], 448, 1),
    (4, [6000, 5000, 4100], [3, 1, 17], 5000, 4),
    (4, [8000, 10, 0], [1, 40, 9], 5000, 4),
    (2, [4000] * 9 + [30], [1] * 9 + [200], 3000, 5),
]


@pytest.mark.parametrize("name", ["f16", "f32", "i8"])
@pytest.mark.parametrize("heads,pasts,counts,window,sinks", CASES)
def test_windows(wrs, ctx, name, heads, pasts, counts, window, sinks):
    note(f"window {name} {heads} {pasts} {counts} {window} {sinks}")
    Session(wrs, ctx, name, heads, pasts, counts, seed=11).check(window, sinks)


@pytest.mark.parametrize("name", ["f16", "f32", "i8"])
def test_every_edge_of_a_step(wrs, ctx, name):
    """Windows, sinks and positions around the 16- and 32-key borders."""
    s = Session(wrs, ctx, name, 1, [70], [21], seed=5)
    for window in (1, 2, 15, 16, 17, 31, 32, 33, 38, 39, 40, 63, 64, 65, 90, 91, 92):
        for sinks in (0, 1, 31, 32, 33, 64, 91, 200):
            note(f"edge {name} {window} {sinks}")
            s.check(window, sinks)


@pytest.mark.parametrize("name", ["f16", "f32", "i8"])
@pytest.mark.parametrize("rows", [1, 2, 15, 16, 17, 31, 32, 33, 47, 64, 65, 129])
def test_row_counts(wrs, ctx, name, rows):
    note(f"rows {name} {rows}")
    s = Session(wrs, ctx, name, 2, [50], [rows], seed=rows)
    s.check(30, 2)
    s.check(10 ** 6, 0)


@pytest.mark.parametrize("name", ["f16", "f32", "i8"])
def test_many_slots(wrs, ctx, name):
    """More sequences than one launch takes, some of them without rows."""
    n = 70
    pasts = [(37 * i) % 101 for i in range(n)]
    counts = [(i % 4) * (i % 3 > 0) for i in range(n)]
    note(f"slots {name}")
    Session(wrs, ctx, name, 1, pasts, counts, seed=9).check(20, 3)


@pytest.mark.parametrize("name", ["f16", "f32", "i8"])
def test_strides_and_what_is_left_alone(wrs, ctx, name):
    """Rows in wider rows at any dword; memory between and behind the rows stays."""
    s = Session(wrs, ctx, name, 2, [200, 90], [20, 3], seed=3)
    want, tol = s.expect(64, 4)
    n, d = s.q.shape
    qw = torch.full((n, 3 * d + 1), 5.0, device="cuda")
    qw[:, 1:d + 1] = s.q
    ow = torch.full((n + 1, 2 * d + 3), -3.0, device="cuda")
    note(f"strides {name}")
    s.run(64, 4, q=qw[:, 1:d + 1], out=ow[:n, 3:d + 3])
    got = ow[:n, 3:d + 3]
    assert (got.double() - want).abs().max().item() <= tol
    rest = ow.clone()
    rest[:n, 3:d + 3] = -3.0
    assert (rest == -3.0).all()
    assert torch.equal(got, s.run(64, 4))


@pytest.mark.parametrize("bad", [math.nan, INF, -INF])
@pytest.mark.parametrize("name", ["f16", "f32", "i8"])
def test_hidden_values_never_reach_a_row(wrs, ctx, name, bad):
    """Infinities and NaN in keys that no row, or only some rows, see."""
    def spoil(i, k, v):
        for j in (3, 40, 41, 95):
            k[j, j % 64] = bad
            v[j, ::7] = bad
    rows = 30  # positions 150..179, window 50: row 0 sees 101.., the sinks 0..2
    note(f"hidden {name} {bad}")
    s = Session(wrs, ctx, name, 2, [150], [rows], seed=21, spoil=spoil)
    want, tol = s.expect(50, 3)
    assert want.isfinite().all()
    got = s.run(50, 3)
    assert (got.double() - want).abs().max().item() <= tol
    # the same just inside the windows of the first rows only: 92 + 8 > j > 91 ...
    s = Session(wrs, ctx, name, 1, [90], [40], seed=22,
                spoil=lambda i, k, v: (k[60].fill_(0.5), v[60, 5:6].fill_(bad)))
    want, tol = s.expect(35, 0)
    got = s.run(35, 0)
    clean = torch.arange(40) + 90 - 35 >= 60  # rows that do not see key 60
    assert (got.double() - want)[clean.cuda()].abs().max().item() <= tol
    assert not got[~clean.cuda(), 5].isfinite().any()
    if name != "i8":  # an 8-bit row is NaN as a whole
        other = torch.arange(64, device="cuda") != 5
        d = (got.double() - want)[~clean.cuda()][:, other]
        assert d.abs().max().item() <= tol


@pytest.mark.parametrize("name", ["f16", "f32"])
def test_rows_whose_scores_are_all_minus_infinity(wrs, ctx, name):
    def spoil(i, k, v):
        k[20:, 0] = -INF
    s = Session(wrs, ctx, name, 1, [40], [2], seed=4, spoil=spoil)
    s.q[:, :] = 1.0
    note(f"all -inf {name}")
    got = s.run(8, 0)
    assert (got == 0).all()
    s.q[1, 0] = math.nan
    got = s.run(8, 0)
    assert (got[0] == 0).all() and got[1].isnan().all()


@pytest.mark.parametrize("name", ["f16", "f32", "i8"])
@pytest.mark.parametrize("sigma", [1e-4, 1.0, 30.0])
def test_scales(wrs, ctx, name, sigma):
    s = Session(wrs, ctx, name, 2, [300], [20], seed=8, sigma=sigma)
    s.q /= max(sigma, 1e-3)
    note(f"scale {name} {sigma}")
    s.check(128, 4)


def test_8_bit_rows_of_any_scale_in_one_sum(wrs, ctx):
    """Value rows 2^-60 to 2^60: a tiny weight of a huge row counts, a huge row without a weight
    does not disturb the others."""
    def spoil(i, k, v):
        v *= torch.exp2(((torch.arange(v.shape[0]) * 13) % 121 - 60.0).cuda())[:, None]
        v[7] = 0.0
        k[7] = 0.0
    s = Session(wrs, ctx, "i8", 1, [100], [4], seed=14, spoil=spoil)
    note("8-bit scales")
    want, _ = s.expect(10 ** 6, 0)
    got = s.run(10 ** 6, 0).double()
    # each row is a sum dominated by its largest terms: relative to the sum of magnitudes
    k, v = (stored(x, "i8") for x in s.rows[0])
    sc = s.q.double() @ k.T.contiguous() / 8
    sc = torch.where(hidden(100, 4, 10 ** 6, 0), -INF, sc)
    scale = torch.softmax(sc, 1) @ v.abs()
    assert ((got - want).abs() <= scale * 1.2e-4).all()  # 2 dw with S below 12, as above
    # one key takes the whole weight against huge values elsewhere, before and behind it
    for past, at, rows in ((100, 50, 2), (2000, 1900, 1), (2000, 70, 20), (400, 300, 40)):
        def far(i, k, v):
            k.zero_()
            k[:, 0] = -80.0
            k[at, 0] = 80.0
            v *= 2.0 ** 40
            v[at] = v[at] * 2.0 ** -40
        s = Session(wrs, ctx, "i8", 1, [past], [rows], seed=15, spoil=far)
        s.q.zero_()
        s.q[:, 0] = 8.0  # scores 80 and -80: the others weigh e^-160
        got = s.run(10 ** 6, 0).double()
        want = stored(s.rows[0][1], "i8")[at]
        assert (got - want).abs().max().item() <= want.abs().max().item() * 2.0 ** -17
    # scores that rise from key to key, values that fall
    def ramp(i, k, v):
        k.zero_()
        k[:, 0] = torch.arange(k.shape[0], device="cuda") * 0.25 - 100.0
        v *= torch.exp2(100.0 - torch.arange(v.shape[0], device="cuda") * 0.2)[:, None]
    s = Session(wrs, ctx, "i8", 1, [900], [33], seed=17, spoil=ramp)
    s.q.zero_()
    s.q[:, 0] = 4.0
    want, _ = s.expect(10 ** 6, 0)
    got = s.run(10 ** 6, 0).double()
    k, v = (stored(x, "i8") for x in s.rows[0])
    sc = torch.where(hidden(900, 33, 10 ** 6, 0), -INF, s.q.double() @ k.T.contiguous() / 8)
    # scores of up to 66 (S above): 2 dw = 2 (66 (2^-22 + 2^-21 + 2^-23) + 2^-18 + 2^-22)
    assert ((got - want).abs() <= torch.softmax(sc, 1) @ v.abs() * 1.3e-4).all()


@pytest.mark.parametrize("name", ["f16", "i8"])
@pytest.mark.parametrize("past,rows,window", [(399, 1, 10 ** 6), (384, 16, 10 ** 6), (4000, 1, 3000)])
def test_errors_do_not_add_up(wrs, ctx, name, past, rows, window):
    """Over outputs, the errors' root mean square. Of even weights it is that of a weight's: an
    exponent of up to 2^4 rounds to 2^-21 at most (2^-21 / sqrt(3) ln 2 = 1.9e-7 on average),
    the score before it to 3 products' 2^-23 of its own 2^2 (1.4e-7), v_exp_f32 and the parts add
    2^-23 each: 3e-7 together, and twice that for whatever lies together unluckily."""
    s = Session(wrs, ctx, name, 20, [past], [rows], seed=33)
    note(f"root mean square {name} {past} {rows}")
    want, _ = s.expect(window, 0)
    got = s.run(window, 0).double()
    assert (got - want).norm().item() <= 6e-7 * want.norm().item()


@pytest.mark.parametrize("name", ["f16", "i8"])
@pytest.mark.parametrize("window,sinks", [(200, 5), (10 ** 6, 0), (33, 130)])
def test_many_rows(wrs, ctx, name, window, sinks):
    """Enough rows for tiles, sequences of a few rows among them."""
    rows = 1500 if name == "f16" else 3300
    note(f"many rows {name} {window}")
    Session(wrs, ctx, name, 16, [37, 300, 0, 513], [rows, 3, 0, 70], seed=41).check(window, sinks)


@pytest.mark.parametrize("bad", [math.nan, INF, -INF])
@pytest.mark.parametrize("name", ["f16", "i8"])
def test_hidden_values_of_many_rows(wrs, ctx, name, bad):
    rows = 1030 if name == "f16" else 2600
    hit = (5, 64, 200, 777)  # of rows on; row r sees keys r - 39 to r and the first two

    def spoil(i, k, v):
        for j in hit:
            k[j] = 0.5
            v[j, ::7] = bad
    note(f"hidden, many rows {name} {bad}")
    s = Session(wrs, ctx, name, 16, [0], [rows], seed=42, spoil=spoil)
    want, tol = s.expect(40, 2)
    got = s.run(40, 2).double()
    r = torch.arange(rows, device="cuda")[:, None]
    sees = torch.zeros(rows, 1, dtype=torch.bool, device="cuda")
    for j in hit:
        sees |= (r >= j) & (r < j + 40)
    col = torch.arange(16 * D, device="cuda")[None]
    # an 8-bit row of a head is NaN as a whole, and every head has some of the columns
    odd = sees & ((col % 7 == 0) | (name == "i8"))
    assert not got[odd].isfinite().any()
    assert (got - want)[~odd].abs().max().item() <= tol


def test_wide_range_of_values_f16(wrs, ctx):
    """Weights far below the largest keep their precision next to it."""
    def spoil(i, k, v):
        v[:60] *= 2.0 ** 14
        v[60:] *= 2.0 ** -10
    s = Session(wrs, ctx, "f16", 1, [120], [3], seed=16, spoil=spoil)
    note("f16 range")
    s.check(40, 2)


# ---- the calls that f16 arenas have, over 8-bit ones --------------------------------------------


def cross_expect(q, k, v):
    kk, vv = stored(k, "i8"), stored(v, "i8")
    hide = torch.zeros(q.shape[0], k.shape[0], dtype=torch.bool, device="cuda")
    want, worst = attend64(q, kk, vv, hide)
    return want, tolerance("i8", worst, vv, k.shape[0])


@pytest.mark.parametrize("frames", [1, 31, 32, 33, 257, 1500])
@pytest.mark.parametrize("rows", [1, 5, 8, 9, 33, 223])
def test_cross_rows_8_bit(wrs, ctx, rows, frames):
    heads, d = 3, 3 * D
    ar = wrs.KvArena(2, 1, heads, 1, 1500, ctx=ctx, dtype=wrs.WRS_I8)
    k, v = normal(frames, d, seed=1), normal(frames, d, seed=2)
    ar.set_cross(1, k, v)
    q = normal(rows, d, seed=rows)
    want, tol = cross_expect(q, k, v)
    out = torch.zeros_like(q)
    note(f"cross i8 {rows} {frames}")
    ar.prefill_cross(1, q, out)
    assert (out.double() - want).abs().max().item() <= tol
    again = torch.zeros_like(q)
    ar.decode_cross(1, q, again)
    assert torch.equal(out, again)
    ar.prefill_cross(0, q, out)  # a layer without frames
    assert (out == 0).all()


@pytest.mark.parametrize("frames", [1, 64, 100])
def test_many_cross_rows_8_bit(wrs, ctx, frames):
    """Tiles whose rows all see every key."""
    heads, rows = 16, 2600
    d = heads * D
    ar = wrs.KvArena(1, 1, heads, 8, 100, ctx=ctx, dtype=wrs.WRS_I8)
    k, v = normal(frames, d, seed=46), normal(frames, d, seed=47)
    ar.set_cross(0, k, v)
    q, out = normal(rows, d, seed=48), torch.zeros(rows, d, device="cuda")
    note(f"many cross rows {frames}")
    ar.prefill_cross(0, q, out)
    torch.cuda.synchronize()
    kk, vv = stored(k, "i8"), stored(v, "i8")
    hide = torch.zeros(rows, frames, dtype=torch.bool, device="cuda")
    want, worst = attend64(q, kk, vv, hide)
    assert (out.double() - want).abs().max().item() <= tolerance("i8", worst, vv, frames)


@pytest.mark.parametrize("past", [0, 1, 31, 223, 600, 4000])
def test_self_rows_8_bit(wrs, ctx, past):
    note(f"self i8 {past}")
    s = Session(wrs, ctx, "i8", 4, [past, max(0, past - 3), past // 2], [1, 1, 1], seed=past)
    want, tol = s.expect(10 ** 7, 0)
    out = torch.zeros_like(s.q)
    s.arena.decode_self(1, [0, 1, 2], s.q, out)
    assert (out.double() - want).abs().max().item() <= tol
    assert torch.equal(out, s.run(10 ** 7, 0))
    s = Session(wrs, ctx, "i8", 2, [past], [37], seed=past + 1)
    want, tol = s.expect(10 ** 7, 0)
    out = torch.zeros_like(s.q)
    s.arena.prefill_self(1, 0, s.q, out)
    assert (out.double() - want).abs().max().item() <= tol
    assert torch.equal(out, s.run(None, 0))


def test_cross_projection_into_an_8_bit_arena(wrs, ctx):
    heads, frames, layers = 2, 70, 3
    d = heads * D
    enc = normal(frames, d, seed=1)
    wk = [normal(d, d, seed=2 + i, sigma=d ** -0.5).half() for i in range(layers)]
    wv = [normal(d, d, seed=9 + i, sigma=d ** -0.5).half() for i in range(layers)]
    bv = [normal(d, seed=20 + i) for i in range(layers)]
    a8 = wrs.KvArena(layers, 1, heads, 1, frames, ctx=ctx, dtype=wrs.WRS_I8)
    a32 = wrs.KvArena(layers, 1, heads, 1, frames, ctx=ctx, dtype=wrs.WRS_F32)
    note("cross proj i8")
    a8.set_cross_proj(enc, wk, wv, bv)
    a32.set_cross_proj(enc, wk, wv, bv)
    for layer in range(layers):
        k8, v8, k32, v32 = (torch.zeros(frames, d, device="cuda") for _ in range(4))
        a8.read_cross(layer, 0, k8, v8)
        a32.read_cross(layer, 0, k32, v32)
        assert a8.cross_len(layer) == frames
        for x, y in ((k8, k32), (v8, v32)):  # the same f32 products, rounded
            assert torch.equal(x.double(), stored(y, "i8"))


# ---- streams, graphs, contexts ----------------------------------------------------------------


@pytest.mark.parametrize("name", ["f16", "f32", "i8"])
def test_captured_steps_replay(wrs, name):
    """A captured step (append, window attention) replays on new rows, between eager calls of the
    same context; captured before the context has scratch it runs unsplit."""
    stream = torch.cuda.Stream()
    c = wrs.Context(0)
    with torch.cuda.stream(stream):
        c.use_torch_stream()
        s = Session(wrs, c, name, 2, [3000], [1], seed=31)
        d = 2 * D
        k, v = normal(1, d, seed=40), normal(1, d, seed=41)
        out = torch.zeros(1, d, device="cuda")
        stream.synchronize()
        graphs = []
        for eager_first in (False, True):
            note(f"capture {name} {eager_first}")
            if eager_first:
                s.run(2048, 4)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=stream):
                s.arena.append_rows(1, [0], [1], k, v)
                s.arena.window_self(1, [0], [1], 2048, 4, s.q, out)
            graphs.append(g)
        for turn in range(4):
            for g in graphs:
                k.copy_(normal(1, d, seed=50 + turn))
                v.copy_(normal(1, d, seed=60 + turn))
                s.q.copy_(normal(1, d, seed=70 + turn))
                s.rows[0][0][-1:] = k
                s.rows[0][1][-1:] = v
                out.zero_()
                g.replay()
                stream.synchronize()
                want, tol = s.expect(2048, 4)
                assert (out.double() - want).abs().max().item() <= tol
                # the program's own work between the replays
                assert torch.allclose(s.run(2048, 4), out, atol=tol)
        del graphs
    torch.cuda.synchronize()


def test_two_contexts_at_once(wrs):
    """Two contexts on streams of their own, split launches in flight together."""
    streams = [torch.cuda.Stream() for _ in range(2)]
    sessions, outs, wants = [], [[], []], []
    for i, st in enumerate(streams):
        with torch.cuda.stream(st):
            c = wrs.Context(0)
            c.use_torch_stream()
            s = Session(wrs, c, "i8", 4, [6000 + 50 * i], [1], seed=80 + i)
            st.synchronize()
            sessions.append(s)
            wants.append(s.expect(5000, 4))
    torch.cuda.synchronize()
    note("two contexts")
    for _ in range(8):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                out = torch.empty(1, 4 * D, device="cuda")
                sessions[i].arena.window_self(1, [0], [1], 5000, 4, sessions[i].q, out)
                outs[i].append(out)
    torch.cuda.synchronize()
    for i in range(2):
        want, tol = wants[i]
        for o in outs[i]:
            assert torch.equal(o, outs[i][0])
            assert (o.double() - want).abs().max().item() <= tol


def test_repeated_calls_give_the_same_bits(wrs, ctx):
    for name in ("f16", "f32", "i8"):
        s = Session(wrs, ctx, name, 4, [7000], [2], seed=90)
        first = s.run(6000, 8)
        note(f"repeat {name}")
        for _ in range(5):
            assert torch.equal(first, s.run(6000, 8))


# ---- refusals ---------------------------------------------------------------------------------


def test_refusals(wrs, ctx):
    heads, d = 2, 2 * D
    ar = wrs.KvArena(1, 2, heads, 16, 4, ctx=ctx, dtype=wrs.WRS_I8)
    ar.advance(0, 10)
    q, out = torch.zeros(3, d, device="cuda"), torch.full((3, d), 2.0, device="cuda")
    good = (0, [0], [3], 4, 0, q, out)

    def call(*args):
        ar.window_self(*args)
    note("refusals")
    call(*good)
    torch.cuda.synchronize()
    out.fill_(2.0)
    with pytest.raises(AssertionError):
        call(0, [0], [3], 0, 0, q, out)  # no window
    with pytest.raises(AssertionError):
        call(0, [0], [2], 4, 0, q, out)  # counts and rows differ
    with pytest.raises(AssertionError):
        call(0, [0, 1], [3], 4, 0, q, out)
    with pytest.raises(AssertionError):
        call(0, [0], [3], 4, 0, q[:, :64], out)
    with pytest.raises(TypeError):
        call(0, [0], [3], 4, 0, q.half(), out)
    with pytest.raises(TypeError):
        call(0, [0], [3], 4, 0, q.cpu(), out)
    with pytest.raises(RuntimeError):
        call(1, [0], [3], 4, 0, q, out)  # layer
    with pytest.raises(RuntimeError):
        call(0, [2], [3], 4, 0, q, out)  # slot
    seven = torch.zeros(7, d, device="cuda")
    with pytest.raises(RuntimeError):
        call(0, [0], [7], 4, 0, seven, seven)  # past max_ctx
    lib, sz = ar._lib, wrs._lib.ctypes.c_size_t
    one, three = (sz * 1)(0), (sz * 1)(3)

    def raw(window=4, q_len=3 * d, q_rs=d, o_len=3 * d, o_rs=d, qp=q.data_ptr(), op=out.data_ptr()):
        return lib.wrs_attn_window_self(ctx.handle, ar.handle, 0, one, three, 1, window, 0, qp,
                                        q_len, q_rs, op, o_len, o_rs)
    assert raw() == 0
    torch.cuda.synchronize()
    out.fill_(2.0)
    for bad in (dict(window=0), dict(q_len=3 * d - 1), dict(q_rs=d - 1), dict(o_len=3 * d - 1),
                dict(o_rs=0), dict(q_rs=-d), dict(qp=None), dict(op=None),
                dict(qp=q.data_ptr() + 2), dict(q_rs=2 ** 62)):
        assert raw(**bad) == wrs.WRS_EINVAL, bad
    torch.cuda.synchronize()
    assert (out == 2.0).all()
    parents = torch.full((3,), -1, dtype=torch.int32, device="cuda")
    with pytest.raises(RuntimeError, match="unsupported"):
        ar.tree_self(0, [0], [3], parents, q, out)
    ar.set_cross(0, torch.zeros(4, d, device="cuda"), torch.zeros(4, d, device="cuda"))
    with pytest.raises(RuntimeError, match="unsupported"):
        ar.decode_cross_noalloc(0, q, out)
    with pytest.raises(RuntimeError, match="unsupported"):
        ar.prefill_cross(0, q, out, lse=torch.zeros(2 * heads * 3, device="cuda"))
    with pytest.raises(RuntimeError, match="unsupported"):
        ar.capture_cross_heads(0, q, [(0, 0)], 1, 0, torch.zeros(3 * 4, device="cuda"))
    with pytest.raises(RuntimeError, match="unsupported"):
        wrs.KvArena(1, 1, 1, 2 ** 24 - 4000, 0, ctx=ctx, dtype=wrs.WRS_I8)
    torch.cuda.synchronize()
    assert (out == 2.0).all()
