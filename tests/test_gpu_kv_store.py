"""GPU tests of rows stored for several slots at once, of reading them back, and of the row moves of
8-bit arenas. What an arena holds is compared exactly: storing rounds once, by a rule."""
from __future__ import annotations

import math

import pytest
import torch

from gpu_util import note
from test_gpu_window import D, _dtype, normal, stored

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx(wrs):
    c = wrs.Context(0)
    c.use_torch_stream()
    yield c
    torch.cuda.synchronize()
    c.close()


def read(ar, layer, slot, first, n):
    k, v = (torch.zeros(n, ar.d_model, device="cuda") for _ in range(2))
    ar.read_rows(layer, [slot], [first], [n], k, v)
    torch.cuda.synchronize()
    return k, v


def same(x, want):
    return torch.equal(torch.nan_to_num(x.double(), 123.0), torch.nan_to_num(want, 123.0))


@pytest.mark.parametrize("name", ["f16", "f32", "i8"])
@pytest.mark.parametrize("counts", [[1, 1, 1, 1, 1], [3, 0, 7], [1], [70, 1, 33]])
def test_append_rows_and_read(wrs, ctx, name, counts):
    heads = 3
    d = heads * D
    n = sum(counts)
    ar = wrs.KvArena(2, len(counts) + 1, heads, 100, 0, ctx=ctx, dtype=_dtype(wrs, name))
    pasts = [(5 * i) % 11 for i in range(len(counts))]
    slots = [len(counts) - i for i in range(len(counts))]  # not in order, slot 0 unused
    for s, p in zip(slots, pasts):
        ar.advance(s, p)
    qkv = normal(n, 3 * d, seed=n)
    k, v = qkv[:, d:2 * d], qkv[:, 2 * d:]
    note(f"append_rows {name} {counts}")
    ar.append_rows(1, slots, counts, k, v)
    row = 0
    for s, p, c in zip(slots, pasts, counts):
        if c:
            gk, gv = read(ar, 1, s, p, c)
            assert same(gk, stored(k[row:row + c].contiguous(), name))
            assert same(gv, stored(v[row:row + c].contiguous(), name))
        row += c
    # all slots in one call, into wider rows; what lies between stays
    wide = torch.full((n, 2 * d + 5), -3.0, device="cuda")
    ar.read_rows(1, slots, pasts, counts, wide[:, :d], wide[:, d + 1:2 * d + 1])
    torch.cuda.synchronize()
    assert same(wide[:, :d], stored(k.contiguous(), name))
    assert same(wide[:, d + 1:2 * d + 1], stored(v.contiguous(), name))
    assert (wide[:, d] == -3.0).all() and (wide[:, 2 * d + 1:] == -3.0).all()
    assert ar.slot_len(slots[0]) == pasts[0]  # not advanced


@pytest.mark.parametrize("name", ["f16", "f32", "i8"])
def test_append_rows_equals_append(wrs, ctx, name):
    heads, n = 2, 45
    d = heads * D
    k, v = normal(n, d, seed=1), normal(n, d, seed=2)
    ar = wrs.KvArena(1, 2, heads, 64, 0, ctx=ctx, dtype=_dtype(wrs, name))
    note(f"append {name}")
    ar.append(0, 0, k, v)
    ar.append_rows(0, [1], [n], k, v)
    for a, b in zip(read(ar, 0, 0, 0, n), read(ar, 0, 1, 0, n)):
        assert torch.equal(a, b)
    host = wrs.KvArena(1, 1, heads, 64, 0, ctx=ctx, dtype=_dtype(wrs, name))
    host.append(0, 0, k.cpu().numpy(), v.cpu().numpy())
    for a, b in zip(read(ar, 0, 0, 0, n), read(host, 0, 0, 0, n)):
        assert torch.equal(a, b)


def test_8_bit_rounding(wrs, ctx):
    """Ties, the step where a larger power is taken, zeros, the smallest and largest values, and
    values that are no numbers."""
    f = torch.zeros(14, D)
    f[0, :4] = torch.tensor([64.0, 0.5, 1.5, 2.5])       # codes of 1: ties to even
    f[1, :3] = torch.tensor([127.4999, 0.5, -1.5])       # the largest that a power keeps
    f[2, :3] = torch.tensor([127.5, 1.0, 3.0])           # rounds past 127: the next power
    f[3, :3] = torch.tensor([-128.0, 127.0, 1.0])
    f[5, :2] = torch.tensor([1e-45, -1e-45])             # below every code
    f[6, :3] = torch.tensor([2.0 ** -126, 2.0 ** -127, 1.5 * 2.0 ** -126])
    f[7, :2] = torch.tensor([3.4028235e38, -3.4028235e38])
    f[8, 5] = math.nan
    f[9, 6] = math.inf
    f[10, 63] = -math.inf
    f[11] = torch.linspace(-1, 1, D)
    f[12] = 2.0 ** torch.linspace(-20, 3, D)
    f[13] = -0.0
    f = f.cuda()
    ar = wrs.KvArena(1, 1, 1, 16, 0, ctx=ctx, dtype=wrs.WRS_I8)
    note("8-bit rounding")
    ar.append_rows(0, [0], [14], f, f)
    k, v = read(ar, 0, 0, 0, 14)
    want = stored(f, "i8")
    assert same(k, want) and same(v, want)
    assert k[8:11].isnan().all() and k[:8].isfinite().all()
    # off by at most half a code; the largest, which a smaller power would put past 127.5 codes,
    # is at least 63.75 of them (127.5 itself becomes 63.75): 0.5 / 63.75 = 1 / 127.5
    ok = [0, 1, 2, 3, 11, 12]
    err = (k.double() - f.double())[ok].abs().amax(1)
    assert (err <= f[ok].double().abs().amax(1) / 127.5).all()
    # values that were read back are stored as they are
    ar.append_rows(0, [0], [14], k, v)
    again, _ = read(ar, 0, 0, 0, 14)
    assert same(again, k.double())


def test_long_rows_of_many_slots(wrs, ctx):
    """More than 64 slots, and rows that fill several workgroups."""
    heads, n = 2, 70
    d = heads * D
    counts = [1 + (7 * i) % 5 for i in range(n)]
    counts[3] = 700
    ar = wrs.KvArena(1, n, heads, 700, 0, ctx=ctx, dtype=wrs.WRS_I8)
    k, v = normal(sum(counts), d, seed=5), normal(sum(counts), d, seed=6)
    note("many slots")
    ar.append_rows(0, list(range(n)), counts, k, v)
    gk, gv = torch.zeros_like(k), torch.zeros_like(v)
    ar.read_rows(0, list(range(n)), [0] * n, counts, gk, gv)
    torch.cuda.synchronize()
    assert same(gk, stored(k, "i8")) and same(gv, stored(v, "i8"))


@pytest.mark.parametrize("name", ["f16", "f32", "i8"])
@pytest.mark.parametrize("heads,counts", [(3, [16, 1, 0, 15]), (5, [64, 65, 1]), (1, [129, 63]),
                                          (8, [33000, 100])])
def test_many_rows_of_a_slot(wrs, ctx, name, heads, counts):
    """Blocks of rows of a head, the longest ones read past the caches; from odd rows on, in wider
    rows at an odd dword; what lies around stays."""
    d, n, slots = heads * D, sum(counts), len(counts)
    note(f"rows of a head {name} {heads} {counts}")
    ar = wrs.KvArena(1, slots, heads, max(counts) + 4, 0, ctx=ctx, dtype=_dtype(wrs, name))
    before = normal(3 * slots, d, seed=50)
    ar.append_rows(0, list(range(slots)), [3] * slots, before, before)
    for i in range(slots):
        ar.advance(i, 3)
    wide = normal(n, 2 * d + 3, seed=51)
    k, v = wide[:, 1:d + 1], wide[:, d + 3:]
    ar.append_rows(0, list(range(slots)), counts, k, v)
    out = torch.full((n + 2, 2 * d + 3), 9.0, device="cuda")
    gk, gv = out[1:-1, 2:d + 2], out[1:-1, d + 2:2 * d + 2]
    for i, c in enumerate(counts):
        ar.advance(i, c)
    ar.read_rows(0, list(range(slots)), [3] * slots, counts, gk, gv)
    old_k, old_v = torch.zeros_like(before), torch.zeros_like(before)
    ar.read_rows(0, list(range(slots)), [0] * slots, [3] * slots, old_k, old_v)
    torch.cuda.synchronize()
    assert same(gk, stored(k.contiguous(), name)) and same(gv, stored(v.contiguous(), name))
    assert same(old_k, stored(before, name)) and same(old_v, stored(before, name))
    gk.fill_(9.0)
    gv.fill_(9.0)
    assert (out == 9.0).all()


def fill(wrs, ctx, layers, slots, heads, rows, max_ctx, seed=0):
    ar = wrs.KvArena(layers, slots, heads, max_ctx, 0, ctx=ctx, dtype=wrs.WRS_I8)
    data = {}
    for layer in range(layers):
        for s in range(slots):
            k = normal(rows, heads * D, seed=seed + 100 * layer + 10 * s)
            v = normal(rows, heads * D, seed=seed + 100 * layer + 10 * s + 1, sigma=3.0)
            ar.append(layer, s, k, v)
            data[layer, s] = (stored(k, "i8"), stored(v, "i8"))
    return ar, data


def test_rows_from_the_host(wrs, ctx):
    heads, n = 2, 37
    ar = wrs.KvArena(2, 2, heads, 40, 40, ctx=ctx, dtype=wrs.WRS_I8)
    k, v = normal(n, heads * D, seed=61), normal(n, heads * D, seed=62)
    note("rows from the host")
    ar.append(1, 1, k.cpu().numpy(), v.cpu().numpy())
    ar.advance(1, n)
    ar.set_cross(1, v.cpu().numpy(), k.cpu().numpy())
    gk, gv = torch.zeros_like(k), torch.zeros_like(v)
    ar.read_rows(1, [1], [0], [n], gk, gv)
    ck, cv = torch.zeros_like(k), torch.zeros_like(v)
    ar.read_cross(1, 0, ck, cv)
    torch.cuda.synchronize()
    assert same(gk, stored(k, "i8")) and same(gv, stored(v, "i8"))
    assert same(ck, stored(v, "i8")) and same(cv, stored(k, "i8"))


@pytest.mark.parametrize("rows", [1, 63, 257, 600])
def test_copy_slot_8_bit(wrs, ctx, rows):
    ar, data = fill(wrs, ctx, 2, 3, 2, rows, 601)
    mark = normal(1, 2 * D, seed=77)
    ar.set_len(2, 0)
    ar.advance(2, rows)  # a row behind the copied ones
    ar.append(0, 2, mark, mark)
    ar.set_len(2, 0)
    ar.advance(0, rows)
    note(f"copy {rows}")
    ar.copy_slot(2, 0)
    assert ar.slot_len(2) == rows
    for layer in range(2):
        for got, want in zip(read(ar, layer, 2, 0, rows), data[layer, 0]):
            assert same(got, want)
        for got, want in zip(read(ar, layer, 1, 0, rows), data[layer, 1]):
            assert same(got, want)
    assert same(read(ar, 0, 2, rows, 1)[0], stored(mark, "i8"))


@pytest.mark.parametrize("rows,drop", [(10, 1), (64, 63), (300, 5), (600, 256), (600, 259), (9, 9)])
def test_slide_8_bit(wrs, ctx, rows, drop):
    ar, data = fill(wrs, ctx, 2, 2, 2, rows, 600)
    for s in range(2):
        ar.advance(s, rows)
    note(f"slide {rows} {drop}")
    pos = ar.slide_to_fit(1, drop, rows)
    assert pos == rows - drop == ar.slot_len(1)
    for layer in range(2):
        if pos:
            for got, want in zip(read(ar, layer, 1, 0, pos), data[layer, 1]):
                assert same(got, want[drop:])
        for got, want in zip(read(ar, layer, 0, 0, rows), data[layer, 0]):
            assert same(got, want)


@pytest.mark.parametrize("slots,most", [(1, 5), (3, 9), (20, 30)])
def test_keep_rows_8_bit(wrs, ctx, slots, most):
    rows, past = 90, 20
    ar, data = fill(wrs, ctx, 2, slots, 3, rows, 128)
    g = torch.Generator().manual_seed(slots)
    counts, picks = [], []
    for s in range(slots):
        ar.advance(s, past - s % 3)
        n = int(torch.randint(0, most + 1, (1,), generator=g))
        counts.append(n)
        picks.append(sorted(torch.randperm(60, generator=g)[:n].tolist()))
    note(f"keep {slots} {most}")
    ar.keep_rows(list(range(slots)), counts, [r for p in picks for r in p])
    for layer in range(2):
        for s in range(slots):
            at = past - s % 3
            for got, want in zip(read(ar, layer, s, 0, at + counts[s]), data[layer, s]):
                moved = torch.cat([want[:at], want[[at + r for r in picks[s]]]])
                assert same(got, moved)


def test_ensure_slots_8_bit(wrs, ctx):
    ar, data = fill(wrs, ctx, 3, 2, 2, 33, 40)
    note("grow")
    ar.ensure_slots(5)
    for (layer, s), kv in data.items():
        for got, want in zip(read(ar, layer, s, 0, 33), kv):
            assert same(got, want)
    k = normal(4, 2 * D, seed=3)
    ar.append_rows(2, [4], [4], k, k)
    assert same(read(ar, 2, 4, 0, 4)[0], stored(k, "i8"))


def test_cut_and_written_again(wrs, ctx):
    """A cut history takes other rows; rows before the cut are as they were."""
    ar, data = fill(wrs, ctx, 1, 1, 2, 30, 64)
    ar.advance(0, 30)
    ar.set_len(0, 13)
    k = normal(6, 2 * D, seed=3, sigma=100.0)
    note("cut")
    ar.append(0, 0, k, k)
    got = read(ar, 0, 0, 0, 30)[0]
    want = torch.cat([data[0, 0][0][:13], stored(k, "i8"), data[0, 0][0][19:]])
    assert same(got, want)


@pytest.mark.parametrize("name", ["f16", "f32", "i8"])
def test_read_cross(wrs, ctx, name):
    heads, d = 2, 2 * D
    ar = wrs.KvArena(2, 1, heads, 1, 70, ctx=ctx, dtype=_dtype(wrs, name))
    k, v = normal(50, d, seed=1), normal(50, d, seed=2)
    note(f"read_cross {name}")
    ar.set_cross(1, k, v)
    for first, n in ((0, 50), (7, 20), (49, 1), (50, 0)):
        gk, gv = torch.zeros(n, d, device="cuda"), torch.zeros(n, d, device="cuda")
        ar.read_cross(1, first, gk, gv)
        torch.cuda.synchronize()
        assert same(gk, stored(k, name)[first:first + n])
        assert same(gv, stored(v, name)[first:first + n])
    x = torch.zeros(2, d, device="cuda")
    with pytest.raises(RuntimeError):
        ar.read_cross(1, 49, x, x)
    with pytest.raises(RuntimeError):
        ar.read_cross(0, 0, x, x)  # never set


def test_captured_append_rows(wrs):
    stream = torch.cuda.Stream()
    c = wrs.Context(0)
    with torch.cuda.stream(stream):
        c.use_torch_stream()
        ar = wrs.KvArena(1, 3, 2, 32, 0, ctx=c, dtype=wrs.WRS_I8)
        k, v = normal(4, 2 * D, seed=1), normal(4, 2 * D, seed=2)
        gk, gv = torch.zeros_like(k), torch.zeros_like(v)
        stream.synchronize()
        note("captured append")
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            ar.append_rows(0, [2, 0], [1, 3], k, v)
            ar.read_rows(0, [2, 0], [0, 0], [1, 3], gk, gv)
        for turn in range(4):
            k.copy_(normal(4, 2 * D, seed=10 + turn))
            v.copy_(normal(4, 2 * D, seed=20 + turn))
            g.replay()
            stream.synchronize()
            assert same(gk, stored(k, "i8")) and same(gv, stored(v, "i8"))
            ar.append(0, 1, k, v)  # eager work between the replays
        del g
    torch.cuda.synchronize()


def test_refusals(wrs, ctx):
    heads, d = 2, 2 * D
    ar = wrs.KvArena(1, 3, heads, 16, 0, ctx=ctx, dtype=wrs.WRS_I8)
    base, _ = normal(16, d, seed=1), None
    ar.append(0, 0, base, base)
    ar.advance(0, 10)
    x = normal(3, d, seed=2)
    note("store refusals")
    before = read(ar, 0, 0, 0, 16)[0]
    for args in ((0, [0, 0], [1, 2], x, x),):
        with pytest.raises(AssertionError):
            ar.append_rows(*args)  # a slot twice
    with pytest.raises(AssertionError):
        ar.append_rows(0, [0], [2], x, x)
    with pytest.raises(AssertionError):
        ar.append_rows(0, [0], [3], x, x[:2])
    with pytest.raises(AssertionError):
        ar.append_rows(0, [0], [3], x[:, :64], x[:, :64])
    with pytest.raises(TypeError):
        ar.append_rows(0, [0], [3], x.half(), x)
    with pytest.raises(TypeError):
        ar.append_rows(0, [0], [3], x.cpu(), x)
    with pytest.raises(RuntimeError):
        ar.append_rows(1, [0], [3], x, x)
    with pytest.raises(RuntimeError):
        ar.append_rows(0, [3], [3], x, x)
    seven = normal(7, d, seed=3)
    with pytest.raises(RuntimeError):
        ar.append_rows(0, [1, 0], [0, 7], seven, seven)  # past max_ctx
    with pytest.raises(RuntimeError):
        ar.read_rows(0, [0], [14], [3], x, x)
    with pytest.raises(RuntimeError):
        ar.read_rows(0, [0], [2 ** 63], [3], x, x)
    sz = wrs._lib.ctypes.c_size_t
    zero, three = (sz * 1)(0), (sz * 1)(3)
    p = x.data_ptr()
    for k, kl, kr, v, vl, vr in ((p, 3 * d - 1, d, p, 3 * d, d), (p, 3 * d, d, p, 3 * d - 1, d),
                                 (p, 3 * d, d - 1, p, 3 * d, d), (p, 3 * d, d, p, 3 * d, -1),
                                 (None, 3 * d, d, p, 3 * d, d), (p, 3 * d, d, None, 3 * d, d),
                                 (p + 2, 3 * d, d, p, 3 * d, d)):
        assert ar._lib.wrs_kv_append_rows(ar.handle, 0, zero, three, 1, k, kl, kr, v, vl,
                                          vr) == wrs.WRS_EINVAL
        assert ar._lib.wrs_kv_read_rows(ar.handle, 0, zero, zero, three, 1, k, kl, kr, v, vl,
                                        vr) == wrs.WRS_EINVAL
    assert torch.equal(before, read(ar, 0, 0, 0, 16)[0])


# ---- cross projections: their f32 rows pass through memory that the context keeps ----------------


def projections(layers, d, seed):
    wk = [normal(d, d, seed=seed + i, sigma=d ** -0.5).half() for i in range(layers)]
    wv = [normal(d, d, seed=seed + 20 + i, sigma=d ** -0.5).half() for i in range(layers)]
    bv = [normal(d, seed=seed + 40 + i) for i in range(layers)]
    return wk, wv, bv


def cross(ar, layer, frames):
    k, v = (torch.zeros(frames, ar.d_model, device="cuda") for _ in range(2))
    ar.read_cross(layer, 0, k, v)
    return k, v


@pytest.mark.parametrize("ready", ["eager", "reserved"])
def test_a_captured_cross_projection_keeps_its_rows(wrs, ready):
    """A projection captured for a few frames replays after eager ones of more frames and of wider
    arenas on the same context."""
    heads, frames, layers = 2, 40, 2
    d = heads * D
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        c = wrs.Context(0)
        c.use_torch_stream()
        small = wrs.KvArena(layers, 1, heads, 1, frames, ctx=c, dtype=wrs.WRS_I8)
        plain = wrs.KvArena(layers, 1, heads, 1, frames, ctx=c, dtype=wrs.WRS_F32)
        wide = wrs.KvArena(1, 1, 20, 1, 1500, ctx=c, dtype=wrs.WRS_I8)
        ws, wide_ws = projections(layers, d, 1), projections(1, 20 * D, 100)
        enc, wide_enc = normal(frames, d, seed=7).half(), normal(1500, 20 * D, seed=8).half()
        stream.synchronize()
        note(f"captured cross projection {ready}")
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            with pytest.raises(RuntimeError, match="reserve"):
                small.set_cross_proj(enc, *ws)
            enc.mul_(1.0)
        if ready == "eager":
            small.set_cross_proj(enc, *ws)
        else:
            c.reserve(linear_tokens=frames, linear_n_in=d)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            small.set_cross_proj(enc, *ws)
        wide.set_cross_proj(wide_enc, *wide_ws)
        before = [t.clone() for t in cross(wide, 0, 1500)]
        others = torch.full((4, 4 << 20), 7.0, device="cuda")  # 64 MB that take what was freed
        for turn in range(4):
            enc.copy_(normal(frames, d, seed=60 + turn))
            g.replay()
            if turn % 2:
                wide.set_cross_proj(wide_enc, *wide_ws)
            plain.set_cross_proj(enc, *ws)
            for layer in range(layers):
                for x, y in zip(cross(small, layer, frames), cross(plain, layer, frames)):
                    assert torch.equal(x.double(), stored(y, "i8"))
            for x, y in zip(before, cross(wide, 0, 1500)):
                assert torch.equal(x, y)
            stream.synchronize()
            assert (others == 7.0).all()
        del g
        for ar in (small, plain, wide):
            ar.close()
        c.close()


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("frames", [512, 517, 1100])
def test_a_cross_projection_of_many_pieces(wrs, ctx, dtype, frames):
    """64 heads: 512 rows at a time. A stored value is off by half a code, at most 1/127.5 of its row's
    largest, and by the product's own error. That is at most (4096 + 4) 2^-24 of the terms' absolute sum,
    which for these terms is below 64 |largest| / 1.5: below 2^-6.5, and as a walk of rounded sums rather
    its square root's share, 64 2^-24 times 43: 2^-12."""
    heads = 64
    d = heads * D
    wk, wv, bv = projections(1, d, 3)
    wide = normal(frames, d + 8, seed=frames).to(dtype)
    enc = wide[:, :d]
    ar = wrs.KvArena(1, 1, heads, 1, frames + 3, ctx=ctx, dtype=wrs.WRS_I8)
    note(f"cross projection in pieces {dtype} {frames}")
    ar.set_cross_proj(enc, wk, wv, bv)
    torch.cuda.synchronize()
    assert ar.cross_len(0) == frames
    k, v = cross(ar, 0, frames)
    torch.cuda.synchronize()
    for got, w, b in ((k, wk[0], 0.0), (v, wv[0], bv[0].double())):
        want = (enc.double() @ w.double().T.contiguous() + b).reshape(frames, heads, D)
        largest = want.abs().amax(2, keepdim=True)
        err = (got.double().reshape(frames, heads, D) - want).abs()
        assert (err <= largest * (1 / 127.5 + 2.0 ** -10)).all()
    ar.close()


# ---- slots of unlike lengths -----------------------------------------------------------------


@pytest.mark.parametrize("name", ["f16", "f32", "i8"])
@pytest.mark.parametrize("counts", [[1] * 40 + [500], [500] + [1] * 69, [1] * 7 + [500],
                                    [300] + [1] * 15, [i * 7 % 97 for i in range(70)], [15, 1, 2, 9],
                                    [0, 16, 0, 1, 33, 0], [2] * 63 + [65, 1]])
def test_unlike_slots_in_one_call(wrs, ctx, name, counts):
    heads = 7
    d, n, n_slots = heads * D, sum(counts), len(counts)
    ar = wrs.KvArena(1, n_slots, heads, 512, 0, ctx=ctx, dtype=_dtype(wrs, name))
    slots = [(11 * i + 3) % n_slots if n_slots % 11 else n_slots - 1 - i for i in range(n_slots)]
    pasts = [i % 12 for i in range(n_slots)]
    guard = torch.full((512, d), 2.0, device="cuda")
    for s, p in zip(slots, pasts):
        ar.append_rows(0, [s], [512], guard, guard)
        ar.advance(s, p)
    k, v = normal(n, d, seed=n), normal(n, d, seed=n + 1)
    note(f"unlike {name} {counts[:4]}")
    ar.append_rows(0, slots, counts, k, v)
    row = 0
    for s, p, c in zip(slots, pasts, counts):
        gk, gv = read(ar, 0, s, 0, 512)
        for got, x in ((gk, k), (gv, v)):
            want = guard.double()
            want[p:p + c] = stored(x[row:row + c].contiguous(), name) if c else want[p:p + c]
            assert same(got, want)
        row += c
    gk, gv = (torch.zeros(n, d, device="cuda") for _ in range(2))
    ar.read_rows(0, slots, pasts, counts, gk, gv)
    torch.cuda.synchronize()
    assert same(gk, stored(k, name)) and same(gv, stored(v, name))
    ar.close()


@pytest.mark.parametrize("name", ["f16", "i8"])
def test_single_tokens_beside_a_text_cost_little(wrs, ctx, name):
    heads, text, singles = 20, 8191, 15
    d = heads * D
    ar = wrs.KvArena(1, singles + 1, heads, text, 0, ctx=ctx, dtype=_dtype(wrs, name))
    k, v = (torch.randn(text + singles, d, device="cuda") for _ in range(2))

    def took(call):
        for _ in range(3):
            call()
        best = math.inf
        for _ in range(5):
            a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            a.record()
            for _ in range(20):
                call()
            b.record()
            torch.cuda.synchronize()
            best = min(best, a.elapsed_time(b) * 50)
        return best

    note(f"mixed append {name}")
    alone = took(lambda: ar.append_rows(0, [0], [text], k[:text], v[:text]))
    slots, counts = list(range(singles + 1)), [text] + [1] * singles
    mixed = took(lambda: ar.append_rows(0, slots, counts, k, v))
    assert mixed <= 1.8 * alone, (mixed, alone)
    ar.close()
