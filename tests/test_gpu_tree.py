"""Attention of drafted trees over the KV arena (wrs_attn_tree_self) and the move of
an accepted path (wrs_kv_keep_rows), against plain float64 attention over the rows
that each drafted row sees, and a whole verification step of a small decoder with
MXFP4 projections against decoding the accepted tokens one by one."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from gpu_util import dev, host, note

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24  # half a step of f32, relative


@pytest.fixture(scope="module")
def ctx(wrs):
    c = wrs.Context(0)
    c.use_torch_stream()
    return c


def make_parents(rng, n, shape):
    i = np.arange(n)
    if shape == "chain":
        return i - 1
    if shape == "roots":
        return np.full(n, -1)
    if shape == "star":
        return np.where(i == 0, -1, 0)
    return np.floor(rng.random(n) * (i + 1)).astype(np.int64) - 1


def ancestors(parents):
    """seen[i, j]: row i of the tree sees row j."""
    n = len(parents)
    seen = np.zeros((n, n), bool)
    for i in range(n):
        a = i
        while a >= 0:
            seen[i, a] = True
            p = int(parents[a])
            a = p if 0 <= p < a else -1
    return seen


def tree_f64(q, k, v, parents, past, heads):
    """Outputs of one tree and how far f32 arithmetic may be off, [n][heads * 64]:
    scores are sums of at most 3 * 64 products (operands in up to three parts), off by
    200 u of their absolute sum, and once more by the exponential's argument; a relative
    error of the weights enters the result twice, the sums over the keys once each."""
    n = len(parents)
    q, k, v = (np.asarray(x, np.float64).reshape(len(x), heads, 64) for x in (q, k, v))
    seen = np.ones((n, past + n), bool)
    seen[:, past:] = ancestors(parents)
    out, tol = np.zeros((n, heads, 64)), np.zeros((n, heads, 64))
    for i in range(n):
        kk, vv = k[:past + n][seen[i]], v[:past + n][seen[i]]
        s = np.einsum("hd,jhd->hj", q[i], kk) / 8
        mag = np.einsum("hd,jhd->hj", np.abs(q[i]), np.abs(kk)).max(axis=1) / 8
        p = np.exp(s - s.max(axis=1, keepdims=True))
        p /= p.sum(axis=1, keepdims=True)
        out[i] = np.einsum("hj,jhd->hd", p, vv)
        rel = 2 * (200 * U32 * mag + 8 * U32 * (1 + np.abs(s).max(axis=1))) + 2 * len(kk) * U32
        tol[i] = rel[:, None] * np.einsum("hj,jhd->hd", p, np.abs(vv)) + 1e-30
    return out.reshape(n, heads * 64), tol.reshape(n, heads * 64)


def store_type(x, wrs, dtype):
    return x.astype(np.float16).astype(np.float32) if dtype == wrs.WRS_F16 else x


class Trees:
    """An arena with histories and drafted rows of several slots, and its host copy."""

    def __init__(self, wrs, ctx, dtype, heads, pasts, counts, shape, seed, max_ctx=None):
        rng = np.random.default_rng(seed)
        self.heads, self.pasts, self.counts = heads, pasts, counts
        d = heads * 64
        most = max_ctx or max(p + n for p, n in zip(pasts, counts))
        self.arena = wrs.KvArena(2, len(pasts), heads, most, 0, ctx=ctx, dtype=dtype)
        self.k, self.v, self.parents = [], [], []
        for s, (p, n) in enumerate(zip(pasts, counts)):
            k, v = (store_type(rng.standard_normal((p + n, d)).astype(np.float32), wrs, dtype)
                    for _ in range(2))
            self.k.append(k)
            self.v.append(v)
            self.parents.append(make_parents(rng, n, shape))
            if p + n:
                self.arena.append(1, s, dev(k), dev(v))
            self.arena.advance(s, p)
        self.q = rng.standard_normal((sum(counts), d)).astype(np.float32)

    def device_parents(self):
        return torch.from_numpy(np.concatenate(self.parents).astype(np.int32)).cuda()

    def run(self, q=None, out=None, parents=None):
        q = dev(self.q) if q is None else q
        out = torch.full(tuple(q.shape), float("nan"), device="cuda") if out is None else out
        parents = self.device_parents() if parents is None else parents
        self.arena.tree_self(1, list(range(len(self.counts))), self.counts, parents, q, out)
        return out

    def check(self, got):
        row = 0
        for s, (p, n) in enumerate(zip(self.pasts, self.counts)):
            ref, tol = tree_f64(self.q[row:row + n], self.k[s], self.v[s], self.parents[s], p,
                                self.heads)
            err = np.abs(got[row:row + n].astype(np.float64) - ref)
            assert np.all(err <= tol), (s, float((err - tol).max()), float(err.max()))
            row += n


CASES = [
    # heads, pasts, counts, shape
    (1, [0], [1], "tree"),
    (6, [60], [8], "tree"),
    (2, [0, 1, 5], [3, 1, 17], "tree"),
    (3, [15, 16, 17, 31, 33], [16, 17, 15, 1, 32], "chain"),
    (2, [127, 128, 129], [33, 64, 31], "tree"),
    (1, [500], [256], "chain"),
    (2, [447], [255], "tree"),
    (2, [40, 0, 40], [0, 5, 0], "roots"),
    (1, [2000], [9], "star"),
    (20, [223, 220, 217, 214, 222], [26, 21, 23, 25, 20], "tree"),
    (2, [5000], [40], "tree"),
]


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_trees_match_float64(wrs, ctx, case, dtype):
    heads, pasts, counts, shape = CASES[case]
    note(f"tree_self {dtype} heads={heads} pasts={pasts} counts={counts} {shape}")
    t = Trees(wrs, ctx, getattr(wrs, "WRS_" + dtype.upper()), heads, pasts, counts, shape,
              100 + case)
    t.check(host(t.run()))
    t.arena.close()


def test_more_trees_than_a_launch_takes(wrs, ctx):
    note("tree_self over 70 slots")
    pasts = [(7 * i) % 90 for i in range(70)]
    counts = [(3 * i) % 6 for i in range(70)]
    t = Trees(wrs, ctx, wrs.WRS_F16, 2, pasts, counts, "tree", 7)
    t.check(host(t.run()))
    t.arena.close()


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_chain_matches_prefill_self(wrs, ctx, dtype):
    # a chain is the cached prompt that wrs_attn_prefill_self runs
    note(f"tree_self chain against prefill_self {dtype}")
    t = Trees(wrs, ctx, getattr(wrs, "WRS_" + dtype.upper()), 4, [300], [24], "chain", 11)
    other = torch.empty_like(dev(t.q))
    got = host(t.run())
    t.arena.prefill_self(1, 0, dev(t.q), other)
    _, tol = tree_f64(t.q, t.k[0], t.v[0], t.parents[0], 300, 4)
    # the reference's rule drops weights below 1e-7 on f32 arenas: up to 1e-7 per key
    # times the largest value
    extra = 324 * 1e-7 * np.abs(t.v[0]).max() if dtype == "f32" else 0.0
    assert np.all(np.abs(got.astype(np.float64) - host(other)) <= 2 * tol + extra)
    t.arena.close()


def test_two_trees_of_one_slot(wrs, ctx):
    note("two trees over one slot's drafted rows")
    t = Trees(wrs, ctx, wrs.WRS_F16, 2, [50], [12], "tree", 13)
    q = dev(np.concatenate([t.q, t.q]))
    out = torch.full_like(q, float("nan"))
    par = torch.cat([t.device_parents(), t.device_parents()])
    t.arena.tree_self(1, [0, 0], [12, 12], par, q, out)
    a = host(out)
    t.check(a[:12])
    assert np.array_equal(a[:12], a[12:])
    t.arena.close()


def test_strided_rows_and_untouched_neighbours(wrs, ctx):
    # q in place in fused [n][3 d] rows, out into wider rows
    note("tree_self on strided rows")
    t = Trees(wrs, ctx, wrs.WRS_F16, 3, [70, 9], [10, 19], "tree", 17)
    d = 192
    wide = torch.randn((29, 3 * d + 1), device="cuda")
    wide[:, d + 1:2 * d + 1] = dev(t.q)
    out = torch.full((31, d + 8), 7.0, device="cuda")
    t.run(q=wide[:, d + 1:2 * d + 1], out=out[1:30, 4:4 + d])
    got = host(out)
    t.check(got[1:30, 4:4 + d])
    got[1:30, 4:4 + d] = 7.0
    assert np.all(got == 7.0)
    t.arena.close()


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_bad_parents_hang_from_the_root(wrs, ctx, dtype):
    note("tree_self with parents out of range")
    t = Trees(wrs, ctx, getattr(wrs, "WRS_" + dtype.upper()), 2, [21], [20], "tree", 19)
    bad = t.parents[0].copy()
    bad[[2, 5, 9, 19]] = [2, 1000, -7, 2 ** 31 - 1]
    t.parents[0] = bad
    t.check(host(t.run()))
    t.arena.close()


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf"), 3.0e38])
def test_hidden_rows_never_reach_a_result(wrs, ctx, dtype, bad):
    # drafted rows 3 and 20 are leaves: only they see themselves; rows behind the tree and
    # rows past the history hold the same
    note(f"tree_self with {bad} in hidden rows, {dtype}")
    heads, past, n = 2, 37, 24
    dt = getattr(wrs, "WRS_" + dtype.upper())
    t = Trees(wrs, ctx, dt, heads, [past], [n], "tree", 23, max_ctx=past + n + 40)
    par = np.minimum(t.parents[0], 2)  # nothing hangs from a row above 2
    t.parents[0] = par
    k, v = t.k[0].copy(), t.v[0].copy()
    for r in (3, 20):
        k[past + r] = bad
        v[past + r] = bad
    junk = np.full((40, heads * 64), bad, np.float32)
    t.arena.set_len(0, 0)
    t.arena.append(1, 0, dev(np.concatenate([k, junk])), dev(np.concatenate([v, junk])))
    t.arena.advance(0, past)
    got = host(t.run())
    ref, tol = tree_f64(t.q, t.k[0], t.v[0], par, past, heads)
    clean = [i for i in range(n) if i not in (3, 20)]
    assert np.all(np.abs(got[clean].astype(np.float64) - ref[clean]) <= tol[clean])
    if bad != bad:
        assert np.all(np.isnan(got[[3, 20]]))
    t.arena.close()


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_infinite_values_of_seen_rows(wrs, ctx, dtype):
    # an infinity in a value that rows see with positive weight is their result; a NaN
    # among a row's scores makes the row NaN and no other
    note(f"tree_self with visible infinities, {dtype}")
    dt = getattr(wrs, "WRS_" + dtype.upper())
    t = Trees(wrs, ctx, dt, 1, [20], [6], "chain", 29)
    v = t.v[0].copy()
    v[20 + 3, 7] = np.inf   # seen by rows 3, 4, 5
    v[4, 9] = -np.inf       # of the history: seen by all
    k = t.k[0].copy()
    k[20 + 5, 0] = np.nan   # seen by row 5 alone
    t.arena.set_len(0, 0)
    t.arena.append(1, 0, dev(k), dev(v))
    t.arena.advance(0, 20)
    got = host(t.run())
    ref, tol = tree_f64(t.q, t.k[0], t.v[0], t.parents[0], 20, 1)
    assert np.all(got[3:5, 7] == np.inf) and np.all(got[:5, 9] == -np.inf)
    assert np.all(np.isnan(got[5]))
    ok = np.ones((6, 64), bool)
    ok[3:, 7] = ok[:, 9] = ok[5] = False
    assert np.all((np.abs(got.astype(np.float64) - ref) <= tol)[ok])
    t.arena.close()


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_infinite_keys(wrs, ctx, dtype):
    # a key of -infinity where q > 0: the score is -infinity and the key drops out; rows
    # that see nothing else are zero
    note(f"tree_self with infinite keys, {dtype}")
    dt = getattr(wrs, "WRS_" + dtype.upper())
    t = Trees(wrs, ctx, dt, 1, [0], [3], "roots", 31)
    t.q = np.abs(t.q)
    k = t.k[0].copy()
    k[1, 5] = -np.inf
    t.arena.set_len(0, 0)
    t.arena.append(1, 0, dev(k), dev(t.v[0]))
    got = host(t.run())
    assert np.all(got[1] == 0.0)
    for r in (0, 2):
        assert np.all(np.abs(got[r] - t.v[0][r]) <= 4 * U32 * np.abs(t.v[0][r]))
    t.arena.close()


def test_large_scores(wrs, ctx):
    # scores of several hundred: the maximum is taken off before the exponential
    note("tree_self with large scores")
    t = Trees(wrs, ctx, wrs.WRS_F32, 2, [100], [10], "tree", 37)
    t.q *= 100.0
    t.check(host(t.run()))
    t.arena.close()


def test_nothing_to_do(wrs, ctx):
    t = Trees(wrs, ctx, wrs.WRS_F16, 1, [4], [2], "chain", 41)
    none = torch.empty((0, 64), device="cuda")
    t.arena.tree_self(0, [], [], torch.empty(0, dtype=torch.int32, device="cuda"), none, none)
    t.arena.tree_self(0, [0], [0], torch.empty(0, dtype=torch.int32, device="cuda"), none, none)
    t.arena.close()


def test_refusals(wrs, ctx):
    note("tree_self and keep_rows refusals (no launch)")
    ar = wrs.KvArena(1, 2, 2, 300, 0, ctx=ctx)
    ar.advance(0, 100)
    q = torch.zeros((4, 128), device="cuda")
    par = torch.zeros(4, dtype=torch.int32, device="cuda")
    with pytest.raises(RuntimeError):  # layer
        ar.tree_self(1, [0], [4], par, q, q)
    with pytest.raises(RuntimeError):  # slot
        ar.tree_self(0, [2], [4], par, q, q)
    with pytest.raises(AssertionError):  # a parent per row
        ar.tree_self(0, [0], [4], par[:3], q, q)
    with pytest.raises(AssertionError):  # rows and counts
        ar.tree_self(0, [0], [3], par, q, q)
    with pytest.raises(AssertionError):  # width
        ar.tree_self(0, [0], [4], par, q[:, :64], q[:, :64])
    with pytest.raises(TypeError):
        ar.tree_self(0, [0], [4], par.long(), q, q)
    with pytest.raises(TypeError):
        ar.tree_self(0, [0], [4], par, q.half(), q)
    with pytest.raises(TypeError):
        ar.tree_self(0, [0], [4], par.cpu(), q, q)
    with pytest.raises(TypeError):
        ar.tree_self(0, [0], [4], par, q.cpu(), q)
    with pytest.raises(TypeError):
        ar.tree_self(0, [0], [4], par, torch.zeros((128, 4), device="cuda").T, q)
    big = torch.zeros((257, 128), device="cuda")
    with pytest.raises(RuntimeError):  # nodes of one tree
        ar.tree_self(0, [1], [257], torch.zeros(257, dtype=torch.int32, device="cuda"), big, big)
    with pytest.raises(RuntimeError):  # past max_ctx
        ar.tree_self(0, [0], [201], torch.zeros(201, dtype=torch.int32, device="cuda"),
                     big[:201], big[:201])
    with pytest.raises(AssertionError):  # rows on top of each other
        ar.tree_self(0, [0], [4], par, q, torch.zeros(128, device="cuda").expand(4, -1))

    with pytest.raises(RuntimeError):  # slot
        ar.keep_rows([2], [1], [0])
    with pytest.raises(AssertionError):  # twice
        ar.keep_rows([0, 0], [1, 1], [1, 2])
    with pytest.raises(AssertionError):  # falling
        ar.keep_rows([0], [2], [3, 3])
    with pytest.raises(AssertionError):  # too few
        ar.keep_rows([0], [2], [3])
    with pytest.raises(AssertionError):  # too many
        ar.keep_rows([0], [1], [3, 4])
    with pytest.raises(RuntimeError):  # past max_ctx
        ar.keep_rows([0], [1], [200])
    with pytest.raises((OverflowError, RuntimeError)):  # negative
        ar.keep_rows([0], [1], [-1])
    assert ar.slot_len(0) == 100
    ar.close()


def _planes(wrs, arena, dtype, shape):
    class Span:
        def __init__(self, ptr):
            self.__cuda_array_interface__ = {"shape": shape, "typestr": dtype,
                                             "data": (ptr, False), "version": 2}
    return [torch.as_tensor(Span(p), device="cuda") for p in arena.plane_pointers()[:2]]


@pytest.mark.parametrize("dtype,typestr", [("f16", "<f2"), ("f32", "<f4")])
def test_keep_rows_moves_the_path_and_nothing_else(wrs, ctx, dtype, typestr):
    note(f"keep_rows {dtype}")
    layers, slots, heads, most = 3, 4, 5, 400
    ar = wrs.KvArena(layers, slots, heads, most, 0, ctx=ctx,
                     dtype=getattr(wrs, "WRS_" + dtype.upper()))
    planes = _planes(wrs, ar, typestr, (layers, slots, heads, most, 64))
    rng = np.random.default_rng(3)
    pasts = [0, 17, 130, 60]
    rows = [[0, 1, 5, 6, 40], sorted(rng.choice(380, 300, replace=False).tolist()), [],
            list(range(12)) + [339]]
    ref = []
    for p in planes:
        p.copy_(torch.randn(p.shape, device="cuda"))
        x = p.clone()
        for s, r in enumerate(rows):
            if r:
                src = torch.tensor([pasts[s] + i for i in r], device="cuda")
                x[:, s, :, pasts[s]:pasts[s] + len(r)] = p[:, s][:, :, src]
        ref.append(x)
    for s, n in enumerate(pasts):
        ar.advance(s, n)
    torch.cuda.synchronize()
    order = [3, 1, 2, 0]
    ar.keep_rows(order, [len(rows[s]) for s in order], sum((rows[s] for s in order), []))
    for p, x in zip(planes, ref):
        assert torch.equal(p, x)
    assert [ar.slot_len(s) for s in range(slots)] == pasts
    ar.close()


def test_keep_rows_longer_than_a_launch(wrs, ctx):
    # every row of a path of 2000 moves by one or more: several launches in order
    note("keep_rows of 2000 rows")
    ar = wrs.KvArena(1, 2, 1, 4100, 0, ctx=ctx)
    planes = _planes(wrs, ar, "<f2", (1, 2, 1, 4100, 64))
    for p in planes:
        p.copy_(torch.randn(p.shape, device="cuda"))
    ar.advance(1, 3)
    rows = [2 * i + 1 for i in range(2000)]
    ref = [p.clone() for p in planes]
    for p, x in zip(planes, ref):
        x[0, 1, 0, 3:2003] = p[0, 1, 0, 4:4004:2]
    torch.cuda.synchronize()
    ar.keep_rows([1], [2000], rows)
    for p, x in zip(planes, ref):
        assert torch.equal(p, x)
    ar.close()


def test_results_do_not_depend_on_the_run(wrs, ctx):
    # split caches merge in chunk order, whichever workgroup is the last
    note("tree_self repeated")
    t = Trees(wrs, ctx, wrs.WRS_F16, 4, [3000, 1500], [30, 7], "tree", 43)
    first = t.run()
    for _ in range(5):
        assert torch.equal(t.run(), first)
    t.arena.close()


def test_captured_and_replayed_with_new_trees(wrs):
    # parents and q are read at replay: one captured step takes new trees, with eager calls
    # of the same context between the replays
    note("tree_self captured and replayed")
    c = wrs.Context(0)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        c.use_torch_stream()
        c.reserve(n_heads=4, decode_rows=8, decode_keys=1500)
        t = Trees(wrs, c, wrs.WRS_F16, 4, [1500, 700], [16, 9], "tree", 47)
        q, par = dev(t.q), t.device_parents()
        out = torch.full_like(q, float("nan"))
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            t.run(q=q, out=out, parents=par)
        for seed in range(4):
            rng = np.random.default_rng(seed)
            t.parents = [make_parents(rng, n, "tree") for n in t.counts]
            t.q = rng.standard_normal(t.q.shape).astype(np.float32)
            q.copy_(dev(t.q))
            par.copy_(t.device_parents())
            out.fill_(float("nan"))
            g.replay()
            side.synchronize()
            t.check(host(out))
            assert torch.equal(t.run(), out)
            side.synchronize()
        t.arena.close()
    c.close()


def test_captured_without_scratch_runs_unsplit(wrs):
    note("tree_self captured on a fresh context")
    c = wrs.Context(0)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        c.use_torch_stream()
        t = Trees(wrs, c, wrs.WRS_F16, 2, [900], [12], "tree", 53)
        q, par = dev(t.q), t.device_parents()
        out = torch.full_like(q, float("nan"))
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            t.run(q=q, out=out, parents=par)
        for _ in range(3):
            out.fill_(float("nan"))
            g.replay()
            side.synchronize()
            t.check(host(out))
            t.check(host(t.run()))
        t.arena.close()
    c.close()


def test_two_contexts_at_once(wrs):
    # contexts on streams of their own, each with its own scratch
    note("tree_self from two contexts on two streams")
    made = []
    for i in range(2):
        c = wrs.Context(0)
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            c.use_torch_stream()
            t = Trees(wrs, c, wrs.WRS_F16, 4, [2500], [20], "tree", 60 + i)
            made.append((c, s, t, dev(t.q), t.device_parents(),
                         [torch.full((20, 256), float("nan"), device="cuda") for _ in range(6)]))
    torch.cuda.synchronize()
    for j in range(6):
        for c, s, t, q, par, outs in made:
            t.run(q=q, out=outs[j], parents=par)
    torch.cuda.synchronize()
    for c, s, t, q, par, outs in made:
        for o in outs:
            t.check(host(o))
        t.arena.close()
        c.close()


def test_verification_step_equals_decoding_the_path(wrs, ctx):
    """Two decoder layers with MXFP4 projections: a drafted tree is checked in one pass,
    its path kept, and the next token decoded; against a second slot that decodes the same
    tokens one at a time. Projections see the same rows, so each layer differs by f32
    rounding alone (f16 cache rows may then round the other way: half an f16 step)."""
    note("verification step: linear_mx4, append, tree_self, keep_rows, decode_self")
    heads, layers, past = 4, 2, 30
    d = heads * 64
    rng = np.random.default_rng(71)
    g = [[wrs.mx4_quantize(dev((rng.standard_normal((o, i)) * i ** -0.5).astype(np.float32)),
                           ctx=ctx)
          for o, i in ((d, d), (d, d), (d, d), (d, d), (4 * d, d), (d, 4 * d))]
         for _ in range(layers)]
    gam, bet = dev(np.ones(d, np.float32)), dev(np.zeros(d, np.float32))
    ar = wrs.KvArena(layers, 2, heads, 64, 0, ctx=ctx, dtype=wrs.WRS_F32)
    for layer in range(layers):
        k, v = (dev(rng.standard_normal((past, d)).astype(np.float32)) for _ in range(2))
        for s in range(2):
            ar.append(layer, s, k, v)
    for s in range(2):
        ar.advance(s, past)

    def step(x, slot, attend):
        n = x.shape[0]
        for layer, (wq, wk, wv, wo, w0, w2) in enumerate(g):
            h, q, k, v, att, y = (torch.empty((n, d), device="cuda") for _ in range(6))
            m = torch.empty((n, 4 * d), device="cuda")
            wrs.layer_norm(x, gam, bet, 1e-5, h, ctx=ctx)
            wrs.linear_mx4(h, [wq, wk, wv], None, [q, k, v], ctx=ctx)
            ar.append(layer, slot, k, v)
            attend(layer, q, att)
            wrs.linear_mx4(att, [wo], None, [y], ctx=ctx)
            x = x + y
            wrs.layer_norm(x, gam, bet, 1e-5, h, ctx=ctx)
            wrs.linear_mx4(h, [w0], None, [m], act="gelu", ctx=ctx)
            wrs.linear_mx4(m, [w2], None, [y], ctx=ctx)
            x = x + y
        return x

    parents = np.array([-1, -1, 0, 1, 1, 3, 4, 4, 7, 2], np.int32)
    path = [1, 4, 7, 8]
    tokens = dev(rng.standard_normal((len(parents), d)).astype(np.float32))
    par = torch.from_numpy(parents).cuda()
    drafted = host(step(tokens, 0, lambda layer, q, o: ar.tree_self(
        layer, [0], [len(parents)], par, q, o)))
    ar.keep_rows([0], [len(path)], path)
    ar.advance(0, len(path))
    after = dev(rng.standard_normal((1, d)).astype(np.float32))
    one = lambda slot: lambda layer, q, o: ar.decode_self(layer, [slot], q, o)  # noqa: E731
    singles = []
    for t in path:
        singles.append(host(step(tokens[t:t + 1].contiguous(), 1, one(1))))
        ar.advance(1, 1)
    last = [host(step(after, s, one(s))) for s in range(2)]
    # Two layers of sums of at most 1024 products, values of order 1 to 10: rounding of
    # f32 sums, 1024 u each way, through norms of gain 1, and the decode's dropped weights
    # (34 keys of up to 1e-7).
    bar = 40 * 1024 * U32 * 0.1
    assert np.abs(drafted[path] - np.concatenate(singles)).max() <= bar
    assert np.abs(last[0] - last[1]).max() <= bar
    ar.close()


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("octaves", [14, 20, 26])
def test_weights_far_below_the_largest(wrs, ctx, dtype, octaves):
    """One key takes nearly all of the softmax and its value is 0: the outputs are what the
    weights 2^-octaves of the largest carry."""
    note(f"tree_self with weights 2^-{octaves} of the largest, {dtype}")
    dt = getattr(wrs, "WRS_" + dtype.upper())
    t = Trees(wrs, ctx, dt, 2, [300], [20], "tree", 43)
    t.q *= 0.25
    t.q.reshape(20, 2, 64)[:, :, 7] = 8 * octaves * np.log(2)
    k, v = t.k[0].reshape(-1, 2, 64), t.v[0].reshape(-1, 2, 64)
    k[:, :, 7], k[77, :, 7] = 0, 1
    v[77] = 0
    t.arena.set_len(0, 0)
    t.arena.append(1, 0, dev(t.k[0]), dev(t.v[0]))
    t.arena.advance(0, 300)
    t.check(host(t.run()))
    t.arena.close()


def head_f64(q, k, v, parents, past):
    """tree_f64 of one head, all rows at once: outputs and tolerances [n][64]."""
    n = len(parents)
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    seen = np.ones((n, past + n), bool)
    seen[:, past:] = ancestors(parents)
    k, v = k[:past + n], v[:past + n]
    s = np.where(seen, q @ k.T / 8, -np.inf)
    mag = np.where(seen, np.abs(q) @ np.abs(k).T / 8, 0.0).max(axis=1)
    largest = np.where(seen, np.abs(s), 0.0).max(axis=1)
    p = np.exp(s - s.max(axis=1, keepdims=True))
    p /= p.sum(axis=1, keepdims=True)
    rel = (2 * (200 * U32 * mag + 8 * U32 * (1 + largest)) + 2 * seen.sum(axis=1) * U32)
    return p @ v, rel[:, None] * (p @ np.abs(v)) + 1e-30


class LargeTrees:
    """Caches past the size from which blocks of 32 rows run (128 MB of f16 K and V, 384 of f32,
    and an even number of three or more blocks of 16 rows in the largest tree), drawn on the GPU;
    some (slot, head) pairs are checked. From head 10 on the history's values are 2^-14 of the
    drafted rows', so that the outputs are the drafted rows' and one seen too many or too few
    stands out (of 40000 equal weights one is 2.5e-5, f32 sums of as many may be off by 5e-3)."""

    heads = 20

    def __init__(self, wrs, ctx, dtype, pasts, counts, seed):
        size, least = (2, 128 << 20) if dtype == "f16" else (4, 384 << 20)
        blocks = (max(counts) + 15) // 16
        assert max(counts) > 32 and blocks % 2 == 0
        assert sum(p + n for p, n in zip(pasts, counts)) * self.heads * 64 * 2 * size >= least
        gen = torch.Generator(device="cuda").manual_seed(seed)
        rng = np.random.default_rng(seed)
        d = self.heads * 64
        self.pasts, self.counts = pasts, counts
        self.arena = wrs.KvArena(1, len(pasts), self.heads,
                                 max(p + n for p, n in zip(pasts, counts)) + 8, 0, ctx=ctx,
                                 dtype=getattr(wrs, "WRS_" + dtype.upper()))
        store = torch.float16 if dtype == "f16" else torch.float32
        self.kv = []
        for s, (p, n) in enumerate(zip(pasts, counts)):
            k, v = (torch.randn((p + n, d), generator=gen, device="cuda") for _ in range(2))
            v[:p, 640:] *= 2.0 ** -14
            k, v = (x.to(store).float() for x in (k, v))
            self.kv.append((k, v))
            self.arena.append(0, s, k, v)
            self.arena.advance(s, pasts[s])
        self.q = torch.randn((sum(counts), d), generator=gen, device="cuda")
        self.new_trees(rng)
        torch.cuda.synchronize()

    def new_trees(self, rng):
        self.parents = [make_parents(rng, n, rng.choice(["tree", "tree", "chain", "star"]))
                        for n in self.counts]

    def device_parents(self):
        return torch.from_numpy(np.concatenate(self.parents).astype(np.int32)).cuda()

    def run(self, out=None, parents=None):
        out = torch.full_like(self.q, float("nan")) if out is None else out
        parents = self.device_parents() if parents is None else parents
        self.arena.tree_self(0, list(range(len(self.counts))), self.counts, parents, self.q, out)
        return out

    def check(self, out, pairs, rows=None):
        starts = np.concatenate([[0], np.cumsum(self.counts)])
        for s, h in pairs:
            at = slice(64 * h, 64 * h + 64)
            r = slice(int(starts[s]), int(starts[s + 1]))
            k, v = (x[:, at].cpu().numpy() for x in self.kv[s])
            ref, tol = head_f64(self.q[r, at].cpu().numpy(), k, v, self.parents[s], self.pasts[s])
            err = np.abs(host(out[r, at]).astype(np.float64) - ref)
            if rows is not None:
                err, tol = err[rows], tol[rows]
            assert np.all(err <= tol), (s, h, float((err / tol).max()))


LARGE = {  # pasts and counts of the slots
    # one long history: masks in registers, and (250 nodes) walks in LDS
    "one_64": lambda f32: ([39400 if f32 else 27000], [64]),
    "one_250": lambda f32: ([39500 if f32 else 26219], [250]),
    # ragged trees over many short histories
    "many": lambda f32: ([1000 - 7 * i for i in range(46 if f32 else 32)],
                         [(64, 17, 40, 1, 50, 33)[i % 6] for i in range(46 if f32 else 32)]),
    # large trees beside small ones
    "both": lambda f32: ([30000 if f32 else 20000, 12000, 0], [96, 64, 255]),
}


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("case", sorted(LARGE))
def test_large_caches_match_float64(wrs, ctx, case, dtype):
    note(f"tree_self, blocks of 32 rows, {case} {dtype}")
    pasts, counts = LARGE[case](dtype == "f32")
    t = LargeTrees(wrs, ctx, dtype, pasts, counts, 81)
    first = t.run()
    some = sorted({0, 1, 2, 3, len(counts) // 2, len(counts) - 1} & set(range(len(counts))))
    t.check(first, [(s, h) for s in some for h in (0, 7, 12, 19)])
    assert bool(torch.isfinite(first).all())
    for _ in range(3):  # and the same bits each time
        assert torch.equal(t.run(), first)
    t.arena.close()


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("nodes", [64, 122])
def test_large_caches_hide_what_a_row_does_not_see(wrs, ctx, nodes, bad, dtype):
    """Leaves of either half of a block hold non-finite keys and values; other rows never see
    them, nor rows behind the tree. A value that rows see is their result."""
    note(f"tree_self, blocks of 32 rows, {bad} in hidden rows, {nodes} nodes {dtype}")
    past = 39400 if dtype == "f32" else 26300
    t = LargeTrees(wrs, ctx, dtype, [past], [nodes], 83)
    par = np.minimum(make_parents(np.random.default_rng(84), nodes, "tree"), 2)
    par[nodes - 1] = 40  # a deeper path, through the second half of a block
    t.parents = [par]
    leaves = [3, 20, 33, nodes - 2]
    k, v = (x.clone() for x in t.kv[0])
    for x in (k, v):
        x[[past + r for r in leaves]] = bad
    junk = torch.full((8, t.heads * 64), bad, device="cuda")
    v[past + 40, 5] = float("inf")  # of head 0, seen by row 40 and the last
    t.arena.set_len(0, 0)
    t.arena.append(0, 0, torch.cat([k, junk]), torch.cat([v, junk]))
    t.arena.advance(0, past)
    out = t.run()
    clean = [i for i in range(nodes) if i not in leaves]
    t.check(out, [(0, 1), (0, 19)], rows=clean)
    t.check(out, [(0, 0)], rows=[i for i in clean if i not in (40, nodes - 1)])
    got = host(out)
    assert np.all(got[[40, nodes - 1], 5] == np.inf)
    if bad != bad:
        assert np.all(np.isnan(got[leaves]))
    t.arena.close()


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("reserved", [True, False])
def test_large_caches_captured(wrs, reserved, dtype):
    """Captured with the scratch (chunks) and without (whole), replayed with new trees, eager
    calls of the same context between the replays."""
    note(f"tree_self, blocks of 32 rows, captured, reserved {reserved}, {dtype}")
    c = wrs.Context(0)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        c.use_torch_stream()
        if reserved:
            c.reserve(n_heads=20, decode_rows=8, decode_keys=1500)
        t = LargeTrees(wrs, c, dtype, [27000 if dtype == "f32" else 18000, 13000], [64, 39], 85)
        par, out = t.device_parents(), torch.full_like(t.q, float("nan"))
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            t.run(out=out, parents=par)
        for seed in range(3):
            t.new_trees(np.random.default_rng(seed))
            t.q.copy_(torch.randn(t.q.shape))
            par.copy_(t.device_parents())
            out.fill_(float("nan"))
            g.replay()
            side.synchronize()
            some = [(0, 3), (0, 18), (1, 9), (1, 10)]
            t.check(out, some)
            eager = t.run()
            side.synchronize()
            t.check(eager, some)
            if reserved:
                assert torch.equal(eager, out)
        t.arena.close()
    c.close()


def norm_bound(keys):
    """How far the norm of the outputs' error may be off, of the outputs' norm: roundings of
    random terms add in squares. A score of size 1 is off by 64 sums and products, the maximum
    and the exponential, 8 u in all, and so is its weight; a sum over n keys of either sign by
    sqrt(n / 6) u, one of weights by sqrt(n / 9) u. Twice that (q in one f16 part alone leaves
    about 1e-4)."""
    return 2 * U32 * np.sqrt(64 + keys / 6 + keys / 9)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("case", [i for i, c in enumerate(CASES) if max(c[1]) >= 100])
def test_norm_of_the_error(wrs, ctx, case, dtype):
    heads, pasts, counts, shape = CASES[case]
    note(f"tree_self {dtype}, norm of the error, heads={heads} pasts={pasts} counts={counts}")
    t = Trees(wrs, ctx, getattr(wrs, "WRS_" + dtype.upper()), heads, pasts, counts, shape,
              200 + case)
    got, row = host(t.run()).astype(np.float64), 0
    for s, (p, n) in enumerate(zip(pasts, counts)):
        ref, _ = tree_f64(t.q[row:row + n], t.k[s], t.v[s], t.parents[s], p, heads)
        off = np.linalg.norm(got[row:row + n] - ref) / np.linalg.norm(ref)
        assert off <= norm_bound(p + n), (s, off)
        row += n
    t.arena.close()


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("case", sorted(LARGE))
def test_norm_of_the_error_of_large_caches(wrs, ctx, case, dtype):
    note(f"tree_self, blocks of 32 rows, norm of the error, {case} {dtype}")
    pasts, counts = LARGE[case](dtype == "f32")
    t = LargeTrees(wrs, ctx, dtype, pasts, counts, 87)
    out, starts = t.run(), np.concatenate([[0], np.cumsum(counts)])
    for s in sorted({0, 1, len(counts) - 1} & set(range(len(counts)))):
        for h in (1, 9):
            at, r = slice(64 * h, 64 * h + 64), slice(int(starts[s]), int(starts[s + 1]))
            k, v = (x[:, at].cpu().numpy() for x in t.kv[s])
            ref, _ = head_f64(t.q[r, at].cpu().numpy(), k, v, t.parents[s], pasts[s])
            off = np.linalg.norm(host(out[r, at]) - ref) / np.linalg.norm(ref)
            assert off <= norm_bound(pasts[s] + counts[s]), (s, h, off)
    t.arena.close()


def test_reserved_scratch_is_what_trees_can_use(wrs):
    """Reserving decode rows gives a context the scratch of split caches: partial rows of as many
    workgroups as a launch splits into (512 of 32 rows of 66 floats, 4.3 MB), no more."""
    note("reserve of eight contexts (no launch)")
    made = [wrs.Context(0) for _ in range(8)]
    torch.cuda.synchronize()
    before = torch.cuda.mem_get_info(0)[0]
    for c in made:
        c.reserve(n_heads=1, decode_rows=1, decode_keys=64)
    taken = before - torch.cuda.mem_get_info(0)[0]
    for c in made:
        c.close()
    assert taken <= 8 * 7 * 2 ** 20, taken / 8


def test_drafts_of_several_slots_from_one_projection(wrs, ctx):
    """One projection makes q, k and v of every drafted row; each slot's rows are appended from
    it, one call attends them all, and the accepted paths are kept and taken in."""
    note("linear_mx4, append per slot, tree_self, keep_rows over three slots")
    heads, pasts, counts = 3, [20, 0, 41], [7, 12, 5]
    d, slots, total = heads * 64, [2, 0, 1], sum(counts)
    rng = np.random.default_rng(91)
    w_qkv = [dev((rng.standard_normal((d, d)) * d ** -0.5).astype(np.float32)).half()
             for _ in range(3)]
    b_q, b_v = (dev(rng.standard_normal(d).astype(np.float32)) for _ in range(2))
    ar = wrs.KvArena(1, 3, heads, 64, 0, ctx=ctx, dtype=wrs.WRS_F32)
    old = [tuple(dev(rng.standard_normal((p, d)).astype(np.float32)) for _ in range(2))
           for p in pasts]
    for s, p, (k, v) in zip(slots, pasts, old):
        if p:
            ar.append(0, s, k, v)
            ar.advance(s, p)
    x = dev(rng.standard_normal((total, d)).astype(np.float32))
    q, k, v, att = (torch.full((total, d), float("nan"), device="cuda") for _ in range(4))
    trees = [make_parents(rng, n, "tree") for n in counts]
    parents = torch.from_numpy(np.concatenate(trees).astype(np.int32)).cuda()

    w_q, w_k, w_v = (wrs.mx4_quantize(w, ctx=ctx) for w in w_qkv)
    wrs.linear_mx4(x, [w_q, w_k, w_v], [b_q, None, b_v], [q, k, v], ctx=ctx)
    r0 = 0
    for s, n in zip(slots, counts):
        ar.append(0, s, k[r0:r0 + n], v[r0:r0 + n])
        r0 += n
    ar.tree_self(0, slots, counts, parents, q, att)
    paths = [[0, 3, 6], [], [1, 4]]
    ar.keep_rows(slots, [len(p) for p in paths], [r for p in paths for r in p])
    for s, p in zip(slots, paths):
        ar.advance(s, len(p))

    kh, vh, qh, got, r0 = host(k), host(v), host(q), host(att), 0
    kp, vp = _planes(wrs, ar, "<f4", (1, 3, heads, 64, 64))
    for s, p, n, par, path, (k0, v0) in zip(slots, pasts, counts, trees, paths, old):
        kk, vv = (np.concatenate([host(a), b[r0:r0 + n]]) for a, b in ((k0, kh), (v0, vh)))
        ref, tol = tree_f64(qh[r0:r0 + n], kk, vv, par, p, heads)
        assert np.all(np.abs(got[r0:r0 + n] - ref) <= tol)
        assert ar.slot_len(s) == p + len(path)
        for plane, rows in ((kp, kk), (vp, vv)):
            want = np.concatenate([rows[:p], rows[p:][path]]).reshape(-1, heads, 64)
            kept = plane[0, s].transpose(0, 1)[:p + len(path)].cpu().numpy()
            assert np.array_equal(kept, want)
        r0 += n
    ar.close()


def test_keep_rows_captured(wrs):
    """A replayed graph makes the moves it was captured with, whatever the rows hold by then;
    eager calls of the same arena run between the replays."""
    note("keep_rows captured and replayed")
    c = wrs.Context(0)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        c.use_torch_stream()
        ar = wrs.KvArena(2, 3, 2, 64, 0, ctx=c)
        planes = _planes(wrs, ar, "<f2", (2, 3, 2, 64, 64))
        for s, n in enumerate((5, 0, 30)):
            ar.advance(s, n)
        moves = {0: [1, 4, 9], 1: [], 2: [0, 2, 3, 33]}
        side.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            ar.keep_rows(list(moves), [len(r) for r in moves.values()], sum(moves.values(), []))
        for _ in range(4):
            for p in planes:
                p.copy_(torch.randn(p.shape, device="cuda"))
            want = [p.clone() for p in planes]
            for p, x in zip(planes, want):
                for s, past in ((0, 5), (2, 30)):
                    x[:, s, :, past:past + len(moves[s])] = \
                        p[:, s][:, :, torch.tensor(moves[s], device="cuda") + past]
            g.replay()
            side.synchronize()
            assert all(torch.equal(p, x) for p, x in zip(planes, want))
            ar.keep_rows([1], [1], [7])
            for x in want:
                x[:, 1, :, 0] = x[:, 1, :, 7]
            side.synchronize()
            assert all(torch.equal(p, x) for p, x in zip(planes, want))
        ar.close()
    c.close()


def test_nothing_kept(wrs, ctx):
    note("keep_rows of empty paths")
    ar = wrs.KvArena(1, 2, 2, 32, 0, ctx=ctx)
    ar.keep_rows([], [], [])
    ar.keep_rows([0, 1], [0, 0], [])
    ar.keep_rows([1], [3], [0, 1, 2])  # in place already
    ar.close()


def test_another_context_than_the_arenas(wrs, ctx):
    """A context of the same device attends an arena that another one made, on its own stream."""
    note("wrs_attn_tree_self from a second context")
    t = Trees(wrs, ctx, wrs.WRS_F16, 2, [1400, 70], [20, 9], "tree", 95)
    q, par = dev(t.q), t.device_parents()
    out = torch.full_like(q, float("nan"))
    want = t.run()
    torch.cuda.synchronize()
    c = wrs.Context(0)
    size = lambda *v: (ctypes.c_size_t * len(v))(*v)  # noqa: E731
    rc = c._lib.wrs_attn_tree_self(c.handle, t.arena.handle, 1, size(0, 1), size(20, 9), 2,
                                   par.data_ptr(), par.numel(), q.data_ptr(), 128, out.data_ptr(),
                                   128)
    assert rc == 0
    c.synchronize()
    assert torch.equal(out, want)
    c.close()
    t.check(host(out))
    t.arena.close()


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("past", [60, 3000])
def test_queries_of_any_size(wrs, ctx, past, dtype):
    """Rows of q from 2^-60 to 2^8 of the others' size: each row has a scale of its own."""
    note(f"tree_self over {past} keys, rows of q of very different size, {dtype}")
    t = Trees(wrs, ctx, getattr(wrs, "WRS_" + dtype.upper()), 2, [past], [33], "tree", 97)
    t.q *= np.exp2(np.linspace(-60, 8, 33)).astype(np.float32)[:, None]
    t.q[7] = 0.0
    t.check(host(t.run()))
    t.arena.close()
