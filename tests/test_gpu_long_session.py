"""GPU tests of the long-session calls used together, as a decoder's step uses them: projections,
append_rows, window attention (or an 8-bit arena's own decode calls), the vocabulary and the scores
of its tokens, eager and captured; and of what the calls of one context share."""
from __future__ import annotations

import pytest
import torch

from gpu_util import note
from test_gpu_window import D, Session, _dtype, hidden, normal, stored

pytestmark = pytest.mark.gpu

HEADS, VOCAB = 4, 997  # entries of the vocabulary that are tokens, of 1000 that it is padded to
DM = HEADS * D


class Model:
    """One attention layer between two projections, f16 weights, and a vocabulary."""

    def __init__(self, wrs, ctx, seed):
        def w(n, m, i):
            return (normal(n, m, seed=seed + i) * m ** -0.5).half()
        self.wrs, self.ctx = wrs, ctx
        self.w_qkv, self.w_o, self.w_v = w(3 * DM, DM, 0), w(DM, DM, 1), w(1000, DM, 2) * 4

    def step(self, arena, slots, counts, window, sinks, x, room, tokens):
        """Rows x [n][DM] of the slots, appended and not advanced. room: a dict of outputs."""
        wrs, c = self.wrs, self.ctx
        qkv = room["qkv"]
        wrs.linear(x, self.w_qkv, None, qkv, ctx=c)
        arena.append_rows(0, slots, counts, qkv[:, DM:2 * DM], qkv[:, 2 * DM:])
        arena.window_self(0, slots, counts, window, sinks, qkv[:, :DM], room["att"])
        wrs.linear(room["att"], self.w_o, None, room["y"], ctx=c)
        wrs.linear(room["y"], self.w_v, None, room["padded"], ctx=c)
        wrs.token_logprobs(room["logits"], tokens, room["lp"], entropy=room["h"],
                           top_ids=room["ids"], top_logprobs=room["best"], ctx=c)

    def room(self, n):
        f = {"qkv": 3 * DM, "att": DM, "y": DM, "padded": 1000, "best": 5}
        r = {k: torch.zeros(n, m, device="cuda") for k, m in f.items()}
        r.update(logits=r["padded"][:, :VOCAB], lp=torch.zeros(n, device="cuda"), h=torch.zeros(n, device="cuda"),
                 ids=torch.zeros(n, 5, dtype=torch.int32, device="cuda"))
        return r


def attend(name, past, rows, window, sinks):
    """past: a slot's stored (k, v); rows: its new (q, k, v). In 64 bits, with the keys seen."""
    q, k, v = rows
    keys = torch.cat([past[0], stored(k.contiguous(), name)])
    vals = torch.cat([past[1], stored(v.contiguous(), name)])
    hide = hidden(past[0].shape[0], q.shape[0], window, sinks)
    out = []
    for h in range(HEADS):
        c = slice(h * D, (h + 1) * D)
        s = q[:, c].double() @ keys[:, c].T.contiguous() / 8
        out.append(torch.softmax(torch.where(hide, -torch.inf, s), 1) @ vals[:, c])
    return torch.cat(out, 1), (keys, vals)


def check_scores(room, tokens):
    lp = torch.log_softmax(room["logits"].double(), 1)
    n = lp.shape[0]
    at = lp[torch.arange(n, device="cuda"), tokens.long()]
    # a log probability: the largest logit's rounding to 24 bits before the exponent, sums of 997
    tol = 2.0 ** -20 * (1 + room["logits"].abs().max().item())
    assert (room["lp"].double() - at).abs().max().item() <= tol
    best, ids = lp.topk(5, 1)
    assert torch.equal(room["ids"].long(), ids)
    assert (room["best"].double() - best).abs().max().item() <= tol
    assert (room["h"].double() + (lp.exp() * lp).sum(1)).abs().max().item() <= 8 * tol


@pytest.mark.parametrize("name", ["f16", "f32", "i8"])
def test_a_session_of_steps(wrs, name):
    """Ragged texts, then single tokens of three slots past their window, then another text."""
    c = wrs.Context(0)
    c.use_torch_stream()
    m = Model(wrs, c, seed=3)
    slots, window, sinks = [2, 0, 3], 40, 3
    ar = wrs.KvArena(1, 4, HEADS, 160, 0, ctx=c, dtype=_dtype(wrs, name))
    past = [(torch.empty(0, DM, dtype=torch.float64, device="cuda"),) * 2 for _ in slots]
    seed = 100
    for counts in [[70, 1, 33]] + [[1, 1, 1]] * 6 + [[5, 0, 40]] + [[1, 1, 1]] * 2:
        note(f"session {name} {counts}")
        n = sum(counts)
        seed += 1
        x, tokens = normal(n, DM, seed=seed), (torch.arange(n, device="cuda") * 7 % VOCAB).int()
        room = m.room(n)
        m.step(ar, slots, counts, window, sinks, x, room, tokens)
        torch.cuda.synchronize()
        q, k, v = room["qkv"].split(DM, 1)
        row = 0
        for i, cnt in enumerate(counts):
            if cnt == 0:
                continue
            r = slice(row, row + cnt)
            want, past[i] = attend(name, past[i], (q[r], k[r], v[r]), window, sinks)
            # sums of |q k| / 8 below 9: a weight to 9 (2^-22 + 2^-21 + 2^-23) + 2^-19 + 2^-22 of itself,
            # below 2^-16, on both sides of the quotient
            tol = 2.0 ** -15 * past[i][1].abs().max().item()
            assert (room["att"][r].double() - want).abs().max().item() <= tol
            row += cnt
            ar.advance(slots[i], cnt)
        check_scores(room, tokens)
    ar.close()
    c.close()


@pytest.mark.parametrize("name", ["f16", "i8"])
def test_a_captured_step(wrs, name):
    """A whole step in one graph, replayed on new rows, with the program's own steps of other slots
    between the replays."""
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        c = wrs.Context(0)
        c.use_torch_stream()
        m = Model(wrs, c, seed=9)
        slots, counts = [0, 1], [1, 1]
        ar = wrs.KvArena(1, 3, HEADS, 2200, 0, ctx=c, dtype=_dtype(wrs, name))
        hist = [(normal(2000 + 100 * i, DM, seed=60 + i), normal(2000 + 100 * i, DM, seed=70 + i))
                for i in range(2)]
        ar.append_rows(0, slots, [2000, 2100], *(torch.cat([h[j] for h in hist]) for j in (0, 1)))
        for i in range(2):
            ar.advance(i, 2000 + 100 * i)
        past = [tuple(stored(t, name) for t in h) for h in hist]
        x, tokens = normal(2, DM, seed=80), torch.tensor([3, 996], device="cuda").int()
        room, other = m.room(2), m.room(3)
        m.step(ar, slots, counts, 1500, 4, x, room, tokens)  # scratch, and the eager form
        stream.synchronize()
        note(f"captured step {name}")
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            m.step(ar, slots, counts, 1500, 4, x, room, tokens)
        for turn in range(4):
            x.copy_(normal(2, DM, seed=90 + turn))
            for t in room.values():
                t.zero_()
            g.replay()
            m.step(ar, [2], [3], 64, 1, normal(3, DM, seed=95 + turn), other,
                   torch.tensor([1, 2, 3], device="cuda").int())
            stream.synchronize()
            q, k, v = room["qkv"].split(DM, 1)
            for i in range(2):
                r = slice(i, i + 1)
                want, _ = attend(name, past[i], (q[r], k[r], v[r]), 1500, 4)
                tol = 2.0 ** -15 * past[i][1].abs().max().item()
                assert (room["att"][r].double() - want).abs().max().item() <= tol
            check_scores(room, tokens)
            check_scores(other, torch.tensor([1, 2, 3], device="cuda"))
            eager = m.room(2)
            m.step(ar, slots, counts, 1500, 4, x, eager, tokens)
            stream.synchronize()
            for k_, t in eager.items():
                assert torch.equal(t, room[k_]), k_
        del g
        ar.close()
        c.close()


def test_kinds_that_share_a_context(wrs):
    """Trees, windows of each arena type and scores, all split over workgroups, in turn on one
    context and recorded into one graph: what each gives alone."""
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        c = wrs.Context(0)
        c.use_torch_stream()
        runs, sessions = [], []
        for name in ("f16", "f32", "i8"):
            s = Session(wrs, c, name, 2, [3000], [1], seed=15)
            sessions.append(s)
            o = torch.zeros(1, 2 * D, device="cuda")
            runs.append((lambda s=s, o=o: s.arena.window_self(1, [0], [1], 2500, 4, s.q, o), [o]))
            if name != "i8":
                t = torch.zeros(1, 2 * D, device="cuda")
                par = torch.full((1,), -1, dtype=torch.int32, device="cuda")
                runs.append((lambda s=s, t=t, par=par: s.arena.tree_self(1, [0], [1], par, s.q, t),
                             [t]))
        x = normal(3, 51865, seed=4)
        lp, h = torch.zeros(3, device="cuda"), torch.zeros(3, device="cuda")
        tok = torch.tensor([5, 50000, 77], device="cuda").int()
        ids = torch.zeros(3, 7, dtype=torch.int32, device="cuda")
        runs.append((lambda: wrs.token_logprobs(x, tok, lp, entropy=h, top_ids=ids, ctx=c),
                     [lp, h, ids]))
        alone = []
        for f, outs in runs:
            note("alone")
            f()
            f()
            stream.synchronize()
            alone.append([o.clone() for o in outs])
        note("one graph of all kinds")
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            for _ in range(2):
                for f, _o in runs:
                    f()
        for turn in range(4):
            for _, outs in runs:
                for o in outs:
                    o.zero_()
            if turn % 2:
                for f, _o in reversed(runs):
                    f()
            else:
                g.replay()
            stream.synchronize()
            for (_, outs), want in zip(runs, alone):
                for o, w in zip(outs, want):
                    assert torch.equal(o, w)
        del g
        for s in sessions:
            s.arena.close()
        c.close()


def test_a_stream_of_the_contexts_own(wrs):
    """A context keeps its own stream until it is given another: inputs are ready before, outputs
    after its synchronize(), whatever stream torch works on."""
    c = wrs.Context(0)
    s = Session(wrs, c, "i8", 3, [700], [2], seed=6)  # torch made the rows on its stream
    torch.cuda.synchronize()
    s.arena.append_rows(1, [0], [0], s.q[:0], s.q[:0])  # nothing to do
    k, v = s.rows[0]
    s.arena.set_len(0, 0)
    s.arena.append_rows(1, [0], [702], k, v)
    s.arena.advance(0, 700)
    out = torch.zeros(2, 3 * D, device="cuda")
    lp = torch.zeros(2, device="cuda")
    ids = torch.zeros(2, 3, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    note("own stream")
    s.arena.window_self(1, [0], [2], 300, 2, s.q, out)
    wrs.token_logprobs(out, torch.tensor([1, 2]).int().cuda(), lp, top_ids=ids, ctx=c)
    c.synchronize()
    want, tol = s.expect(300, 2)
    assert (out.double() - want).abs().max().item() <= tol
    assert torch.equal(ids.long(), out.topk(3, 1)[1])
    s.arena.close()
    c.close()


@pytest.mark.parametrize("name", ["f16", "f32", "i8"])
@pytest.mark.parametrize("window", [None, 2 ** 40, 1])
def test_the_widest_and_the_narrowest_window(wrs, name, window):
    c = wrs.Context(0)
    c.use_torch_stream()
    s = Session(wrs, c, name, 2, [130], [3], seed=12)
    note(f"window {name} {window}")
    for sinks in (0, 10 ** 15):
        out = torch.zeros(3, 2 * D, device="cuda")
        s.arena.window_self(1, [0], [3], window, sinks, s.q, out)
        torch.cuda.synchronize()
        want, tol = s.expect(1 if window == 1 else 10 ** 6, min(sinks, 10 ** 6))
        assert (out.double() - want).abs().max().item() <= tol
    with pytest.raises(AssertionError):
        s.arena.window_self(1, [-1], [3], window, 0, s.q, out)
    with pytest.raises(AssertionError):
        s.arena.window_self(1, [0, 0], [4, -1], window, 0, s.q, out)
    # the same slot twice: its rows attend twice
    q2 = torch.cat([s.q, s.q])
    two = torch.zeros(6, 2 * D, device="cuda")
    s.arena.window_self(1, [0, 0], [3, 3], window, 10 ** 15, q2, two)
    torch.cuda.synchronize()
    assert torch.equal(two[:3], two[3:]) and torch.equal(two[:3], out)
    # in place
    s.arena.window_self(1, [0], [3], window, 10 ** 15, s.q, s.q)
    torch.cuda.synchronize()
    assert torch.equal(s.q, out)
    s.arena.close()
    c.close()


@pytest.mark.parametrize("name", ["f16", "f32", "i8"])
def test_windows_past_64_bits(wrs, name):
    """Counts of keys that no size_t holds are all of the keys."""
    c = wrs.Context(0)
    c.use_torch_stream()
    s = Session(wrs, c, name, 2, [130], [3], seed=13)
    note(f"huge windows {name}")
    outs = []
    for window, sinks in ((None, 0), (2 ** 64, 0), (2 ** 64 + 3, 0), (2, 2 ** 64), (5, 2 ** 70 + 1)):
        out = torch.zeros(3, 2 * D, device="cuda")
        s.arena.window_self(1, [0], [3], window, sinks, s.q, out)
        outs.append(out)
    torch.cuda.synchronize()
    want, tol = s.expect(10 ** 6, 0)
    for out in outs:
        assert (out.double() - want).abs().max().item() <= tol
    s.arena.close()
    c.close()


@pytest.mark.parametrize("name,rows", [("f32", 9_000_000), ("f16", 16_000_000), ("i8", 16_000_000)])
def test_far_rows_of_a_long_cache(wrs, name, rows):
    """Planes of gigabytes: rows behind 2^31 bytes of their plane, planes behind 2^32 bytes."""
    c = wrs.Context(0)
    c.use_torch_stream()
    heads, n, new = 5, 100, 3
    d = heads * D
    note(f"far rows {name}")
    ar = wrs.KvArena(1, 1, heads, rows, 0, ctx=c, dtype=_dtype(wrs, name))
    past = rows - n
    ar.set_len(0, 0)
    ar.advance(0, past)
    k, v, q = (normal(n, d, seed=s) for s in (1, 2, 3))
    ar.append_rows(0, [0], [n], k, v)
    ar.advance(0, n - new)
    gk, gv = torch.zeros_like(k), torch.zeros_like(v)
    ar.read_rows(0, [0], [past], [n], gk, gv)
    out = torch.zeros(new, d, device="cuda")
    ar.window_self(0, [0], [new], 60, 0, q[:new], out)
    torch.cuda.synchronize()
    kk, vv = stored(k, name), stored(v, name)
    assert torch.equal(gk.double(), kk) and torch.equal(gv.double(), vv)
    hide = hidden(n - new, new, 60, 0)
    for h in range(heads):
        at = slice(h * D, (h + 1) * D)
        s = torch.where(hide, -torch.inf, q[:new, at].double() @ kk[:, at].T.contiguous() / 8)
        want = torch.softmax(s, 1) @ vv[:, at]
        # weights to 2^-16 of themselves (sums of |q k| / 8 below 9), on both sides
        assert (out[:, at].double() - want).abs().max().item() <= 2.0 ** -15 * vv.abs().max().item()
    ar.close()
    c.close()


def test_logits_rows_far_apart(wrs):
    c = wrs.Context(0)
    c.use_torch_stream()
    stride, v = 1_200_000_000, 5000
    note("far logits")
    x = torch.empty(3, stride, dtype=torch.float16, device="cuda")[:, :v]
    x.copy_(normal(3, v, seed=5))
    tokens = torch.tensor([0, 2500, 4999], device="cuda").int()
    lp, ids = torch.zeros(3, device="cuda"), torch.zeros(3, 1, dtype=torch.int32, device="cuda")
    wrs.token_logprobs(x, tokens, lp, top_ids=ids, ctx=c)
    torch.cuda.synchronize()
    want = torch.log_softmax(x.double(), 1)
    # exponents below 2^4: 2^-20; the sum's logarithm 2^-22
    assert (lp.double() - want[torch.arange(3), tokens.long()]).abs().max().item() <= 2.0 ** -19
    assert torch.equal(ids[:, 0].long(), want.argmax(1))
    c.close()


def test_a_cache_of_too_many_keys_is_refused(wrs):
    c = wrs.Context(0)
    c.use_torch_stream()
    note("too many keys")
    ar = wrs.KvArena(1, 1, 1, 2 ** 24 + 10, 0, ctx=c)
    q, out = torch.zeros(1, D, device="cuda"), torch.full((1, D), 3.0, device="cuda")
    ar.advance(0, 2 ** 24 - 4096)
    with pytest.raises(RuntimeError, match="too long"):
        ar.window_self(0, [0], [1], 5, 0, q, out)
    ar.set_len(0, 2 ** 24 - 4097)
    ar.append_rows(0, [0], [1], q + 1.0, q + 2.0)
    torch.cuda.synchronize()
    assert (out == 3.0).all()
    ar.window_self(0, [0], [1], 1, 0, q, out)  # the last key there is room for, alone
    torch.cuda.synchronize()
    assert (out == 2.0).all()
    with pytest.raises(RuntimeError, match="too long"):
        wrs.KvArena(1, 1, 1, 2 ** 24, 0, ctx=c, dtype=wrs.WRS_I8)
    ar.close()
    c.close()
