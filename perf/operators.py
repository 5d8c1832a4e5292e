"""Timed cases of the operators that verify drafted tokens under 4-bit weights.

Tree attention over the KV arena, the move of an accepted path's cache rows,
MXFP4 quantisation and the projections with MXFP4 weights. Every case is one
call (or one call and its inverse) as a decoder, a loader or a batch encoder
makes it; widths are those of the workloads in this repository (heads of 64, 6
to 20 of them, 1500 encoder frames, vocabularies around 51865). Inputs are drawn
on the GPU from the case's seed.
"""
from __future__ import annotations

import importlib.util
import math
import sys
from pathlib import Path

import numpy as np
import torch

own = False

D = 64  # head width
BLOCK = 32  # values that share an MX scale
MOST_NODES = 256  # of one tree
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
MODELS = ((6, 4), (8, 6), (12, 12), (16, 24), (20, 32))  # (heads, layers)
# The eight magnitudes of a 4-bit e2m1 code; bit 3 is the sign.
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


# --------------------------------------------------------------------------
# the cases
# --------------------------------------------------------------------------

def listed():
    return [
        # The smallest call: a greedy whisper-tiny decoder checks one small draft.
        {"name": "tree_f16_tiny", "op": "tree", "heads": 6, "slots": 1, "past": 60, "nodes": 8,
         "shape": "tree", "dtype": "f16"},
        # Five beams of a large decoder, each with a draft of its own, ragged.
        {"name": "tree_f16_large_beam5", "op": "tree", "heads": 20, "slots": 5, "past": 223,
         "nodes": 26, "shape": "tree", "dtype": "f16"},
        # One long session (an arena far over 448 positions), a wide draft.
        {"name": "tree_f16_long", "op": "tree", "heads": 20, "slots": 1, "past": 65471,
         "nodes": 64, "shape": "tree", "dtype": "f16"},
        # Drafted chains over the f32 cache of a small decoder, four streams.
        {"name": "tree_f32_small_x4", "op": "tree", "heads": 12, "slots": 4, "past": 430,
         "nodes": 13, "shape": "chain", "dtype": "f32"},
        # The accepted path of one large stream: five of its drafted rows.
        {"name": "keep_f16_large", "op": "keep", "heads": 20, "layers": 32, "slots": 1,
         "past": 223, "width": 6, "kept": 5, "dtype": "f16"},
        # The same for sixteen f32 streams of a small decoder.
        {"name": "keep_f32_small_x16", "op": "keep", "heads": 12, "layers": 12, "slots": 16,
         "past": 200, "width": 9, "kept": 7, "dtype": "f32"},
        # Loading: a large vocabulary matrix from f16 weights.
        {"name": "round_f16_vocab", "op": "round", "rows": 51866, "cols": 1280, "dtype": "f16"},
        # Activations of one window, f32 rows of a ragged length.
        {"name": "round_f32_window", "op": "round", "rows": 1311, "cols": 1280, "dtype": "f32"},
        # A beam-5 step's vocabulary projection: the 4-bit weight stream.
        {"name": "linear_f32_vocab_beam5", "op": "linear", "rows": 5, "n_in": 1280,
         "n_out": 51866, "groups": 1, "x": "f32", "out": "f32", "act": False},
        # Query, key and value rows of five drafted trees.
        {"name": "linear_f32_qkv_trees", "op": "linear", "rows": 130, "n_in": 1280,
         "n_out": 1280, "groups": 3, "x": "f32", "out": "f32", "act": False},
        # The second MLP matrix for sixteen windows of a batch encoder.
        {"name": "linear_f16_mlp_x16", "op": "linear", "rows": 24000, "n_in": 5120,
         "n_out": 1280, "groups": 1, "x": "f16", "out": "f16", "act": False},
        # The first one with its activations rounded to 4 bits on the way in.
        {"name": "linear_mx4_mlp_x16", "op": "linear", "rows": 24000, "n_in": 1280,
         "n_out": 5120, "groups": 1, "x": "mx4", "out": "f16", "act": True},
    ]


def _length(rng, lo, hi):
    """A length spread over the logarithm of [lo, hi]; odd ones among them."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    most = [work(c) for c in listed()]
    top_bytes, top_flops = (max(w[k] for w in most) for k in ("bytes", "flops"))
    while True:
        op = rng.choice(["tree", "tree", "keep", "round", "linear", "linear"])
        heads, layers = rng.choice(MODELS)
        if op == "tree":
            c = {"op": op, "heads": heads, "slots": _length(rng, 1, 16),
                 "past": rng.choice([0, _length(rng, 1, 448), _length(rng, 1, 65536)]),
                 "nodes": _length(rng, 1, MOST_NODES), "shape": rng.choice(["tree", "chain"]),
                 "dtype": rng.choice(["f16", "f16", "f32"])}
            if c["slots"] * (c["past"] + c["nodes"]) * heads > 1_400_000:
                continue
            if c["slots"] * c["nodes"] * (c["past"] + c["nodes"]) * heads > 90_000_000:
                continue  # what the plain form's scores may take
        elif op == "keep":
            c = {"op": op, "heads": heads, "layers": layers, "slots": _length(rng, 1, 16),
                 "past": rng.choice([0, _length(rng, 1, 400)]), "kept": _length(rng, 1, 12),
                 "dtype": rng.choice(["f16", "f32"])}
            c["width"] = c["kept"] + rng.randint(0, 6)
            if layers * heads * c["slots"] * (c["past"] + c["kept"] * c["width"]) > 1_200_000:
                continue
        elif op == "round":
            c = {"op": op, "rows": _length(rng, 1, 52000), "cols": 32 * _length(rng, 1, 160),
                 "dtype": rng.choice(["f16", "bf16", "f32"])}
        else:
            c = {"op": op, "rows": _length(rng, 1, 24000), "n_in": 64 * _length(rng, 1, 80),
                 "n_out": _length(rng, 1, 52000), "groups": rng.choice([1, 1, 3]),
                 "x": rng.choice(["f32", "f16", "bf16", "mx4"]),
                 "out": rng.choice(["f32", "f16", "bf16"]), "act": rng.random() < 0.3}
            if c["rows"] * c["n_out"] * c["groups"] > 130_000_000:
                continue
        w = work(c)
        if w["bytes"] <= top_bytes and w["flops"] <= top_flops:
            return c


def _counts(case):
    """Drafted nodes of each slot: drafts differ by a few."""
    return [max(1, case["nodes"] - (5 * i) % 7) for i in range(case["slots"])]


def _pasts(case):
    """Cached rows of each slot: histories differ by a few tokens."""
    return [max(0, case["past"] - (3 * i) % 11) for i in range(case["slots"])]


def work(case):
    op = case["op"]
    size = {"f32": 4, "f16": 2, "bf16": 2, "mx4": 17 / 32}
    if op == "tree":
        d = case["heads"] * D
        b = f = 0
        for n, p in zip(_counts(case), _pasts(case)):
            b += 2 * (p + n) * d * size[case["dtype"]] + 8 * n * d + 4 * n
            f += 4 * n * (p + 1) * d
    elif op == "keep":
        rows = case["slots"] * case["kept"]
        b = 2 * 2 * rows * case["layers"] * case["heads"] * D * size[case["dtype"]]
        f = 0
    elif op == "round":
        n = case["rows"] * case["cols"]
        b = n * (2 * size[case["dtype"]] + size["mx4"])
        f = 4 * n
    else:
        r, i, o, g = case["rows"], case["n_in"], case["n_out"], case["groups"]
        x = size["f16"] if case["x"] == "mx4" else size[case["x"]]
        b = r * i * x + g * (i * o * size["mx4"] + 4 * o + r * o * size[case["out"]])
        f = 2 * r * i * o * g
    return {"bytes": int(b), "flops": int(f)}


# --------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------

class _Draw:
    """Seeded normal tensors on the GPU."""

    def __init__(self, seed):
        self.gen = torch.Generator(device="cuda").manual_seed(int(seed) & 0x7FFFFFFF)

    def __call__(self, *shape, sigma=1.0):
        return torch.randn(shape, generator=self.gen, device="cuda").mul_(sigma)


def _tree_inputs(case, seed):
    """Cache and drafted rows ([row][heads * 64] f32 per slot), q, and parents."""
    r = _Draw(seed)
    d = case["heads"] * D
    counts, pasts = _counts(case), _pasts(case)
    rows = [(r(p + n, d), r(p + n, d)) for p, n in zip(pasts, counts)]
    q = r(sum(counts), d)
    g = np.random.default_rng(seed)
    parents = []
    for n in counts:
        i = np.arange(n)
        # a node hangs from the root or from an earlier node; a chain's from the one before
        parents.append(i - 1 if case["shape"] == "chain"
                       else np.floor(g.random(n) * (i + 1)).astype(np.int64) - 1)
    return rows, q, parents


def _keep_rows(case, seed):
    """The accepted row of every level of each slot's draft, as offsets past its history.

    Levels are at least as wide as the path is long and the first pick is not one of
    the rows that the path moves to, so that a second pass finds what the first found."""
    g = np.random.default_rng(seed)
    w, m = case["width"], case["kept"]
    picks = g.integers(0, w, size=(case["slots"], m))
    if m > 1:
        picks[:, 0] = np.where(picks[:, 0] < m, 0, picks[:, 0])
    return picks + w * np.arange(m)


def _keep_planes(case, seed):
    """K and V planes [layer][slot][head][row][64]."""
    r = _Draw(seed)
    rows = case["past"] + case["kept"] * case["width"]
    shape = (case["layers"], case["slots"], case["heads"], rows, D)
    return [r(*shape).to(DTYPES[case["dtype"]]) for _ in range(2)]


def _blocks(x):
    return x.reshape(*x.shape[:-1], x.shape[-1] // BLOCK, BLOCK)


def _scale_exponents(blocks):
    """floor(log2(largest magnitude)) - 2 of every block; -127 for a block of zeros."""
    top = blocks.abs().amax(dim=-1, keepdim=True)
    return torch.where(top > 0, torch.frexp(top)[1] - 3, -127).clamp(-127, 127)


def _nearest(y):
    """Magnitudes up to 8 to the nearest e2m1 value, ties to the even code, 6 the largest."""
    step = torch.where(y < 2, 0.5, torch.where(y < 4, 1.0, 2.0))
    return (torch.round(y / step) * step).clamp(max=6.0)


def _mx4_values(x):
    """x rounded to MXFP4, as the values that the codes and scales stand for."""
    b = _blocks(x.float())
    e = _scale_exponents(b)
    y = _nearest(torch.ldexp(b.abs(), -e))
    return torch.copysign(torch.ldexp(y, e), b).reshape(x.shape)


def _mx4_pack(x):
    """x as MXFP4: codes two to a byte (the even column in the low half) and scale bytes."""
    b = _blocks(x.float())
    e = _scale_exponents(b)
    y = _nearest(torch.ldexp(b.abs(), -e))
    edges = torch.tensor([(a + c) / 2 for a, c in zip(E2M1, E2M1[1:])], device=x.device)
    code = torch.bucketize(y, edges).to(torch.uint8) + 8 * torch.signbit(b).to(torch.uint8)
    code = code.reshape(x.shape)
    return ((code[:, 0::2] | (code[:, 1::2] << 4)).contiguous(),
            (e + 127).to(torch.uint8).squeeze(-1).contiguous())


def _mx4_unpack(codes, scales):
    """The f32 values of packed codes and scales (bytes)."""
    table = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=codes.device)
    both = torch.stack([codes & 15, codes >> 4], dim=-1).reshape(codes.shape[0], -1).int()
    e = scales.int().unsqueeze(-1) - 127
    return torch.ldexp(_blocks(table[both]), e).reshape(codes.shape[0], -1)


def _linear_inputs(case, seed):
    r = _Draw(seed)
    n_in, n_out = case["n_in"], case["n_out"]
    x = r(case["rows"], n_in)
    x = x.to(DTYPES["f16" if case["x"] == "mx4" else case["x"]])
    ws = [_mx4_pack(r(n_out, n_in, sigma=n_in ** -0.5).half()) for _ in range(case["groups"])]
    bs = [r(n_out, sigma=0.1) for _ in range(case["groups"])]
    return x, ws, bs


# --------------------------------------------------------------------------
# what a program has in hand
# --------------------------------------------------------------------------

def _package():
    """This repository's package (its folder's name is not an identifier)."""
    if "wrs_amd" in sys.modules:
        return sys.modules["wrs_amd"]
    root = Path.cwd() / "whisper.rs_amd"
    spec = importlib.util.spec_from_file_location(
        "wrs_amd", root / "__init__.py", submodule_search_locations=[str(root)])
    mod = importlib.util.module_from_spec(spec)
    sys.modules["wrs_amd"] = mod
    spec.loader.exec_module(mod)
    return mod


_worker = []


def _context():
    """The context of a worker of a serving program, on torch's stream."""
    if not _worker:
        _worker.append(_package().Context(0))
    _worker[0].use_torch_stream()
    return _worker[0]


def _empty(*shape, dtype=torch.float32):
    return torch.empty(shape, dtype=dtype, device="cuda")


class _DeviceSpan:
    """Device memory owned by an arena, for torch.as_tensor."""

    def __init__(self, ptr, shape, dtype, owner):
        self.owner = owner
        self.__cuda_array_interface__ = {
            "shape": shape, "typestr": {"f16": "<f2", "f32": "<f4"}[dtype],
            "data": (ptr, False), "version": 2}


def _arena(case, layers, rows):
    wrs = _package()
    return wrs.KvArena(layers, case["slots"], case["heads"], rows, 0, ctx=_context(),
                       dtype={"f16": wrs.WRS_F16, "f32": wrs.WRS_F32}[case["dtype"]])


def _tree_state(case, seed):
    rows, q, parents = _tree_inputs(case, seed)
    counts, pasts = _counts(case), _pasts(case)
    most = max(p + n for p, n in zip(pasts, counts))
    s = {"q": q, "slots": list(range(case["slots"])), "counts": counts,
         "parents": torch.from_numpy(np.concatenate(parents).astype(np.int32)).cuda(),
         "heads": case["heads"]}
    if own:
        s["arena"] = arena = _arena(case, 1, most)
        for slot, (k, v) in enumerate(rows):
            arena.append(0, slot, k, v)
            arena.advance(slot, pasts[slot])
        s["out"] = _empty(*q.shape)
    else:
        shape = (case["slots"], case["heads"], most, D)
        s["planes"] = planes = [torch.zeros(shape, dtype=DTYPES[case["dtype"]], device="cuda")
                                for _ in range(2)]
        for slot, kv in enumerate(rows):
            for plane, x in zip(planes, kv):
                plane[slot, :, :x.shape[0]] = x.view(-1, case["heads"], D).transpose(0, 1)
        s["pasts"] = torch.tensor(pasts, device="cuda")
        s["lengths"] = torch.tensor(counts, device="cuda")
        s["tree_of"] = torch.repeat_interleave(torch.arange(len(counts), device="cuda"),
                                               s["lengths"])
        s["node_of"] = torch.cat([torch.arange(n, device="cuda") for n in counts])
    return s


def _keep_state(case, seed):
    planes = _keep_planes(case, seed)
    pasts, picks = _pasts(case), _keep_rows(case, seed)
    m = case["kept"]
    s = {"slots": list(range(case["slots"])), "counts": [m] * case["slots"],
         "rows": [int(i) for i in picks.reshape(-1)]}
    if own:
        s["arena"] = arena = _arena(case, case["layers"], planes[0].shape[3])
        spans = [torch.as_tensor(_DeviceSpan(p, tuple(x.shape), case["dtype"], arena),
                                 device="cuda")
                 for p, x in zip(arena.plane_pointers()[:2], planes)]
        for span, x in zip(spans, planes):
            span.copy_(x)
        torch.cuda.synchronize()
        for slot, n in enumerate(pasts):
            arena.advance(slot, n)
        planes = spans
    s["planes"] = planes
    past = torch.tensor(pasts, device="cuda")[:, None]
    s["slot_of"] = torch.arange(case["slots"], device="cuda")[:, None].expand(-1, m)
    s["to"] = past + torch.arange(m, device="cuda")
    s["from"] = past + torch.from_numpy(picks).cuda()
    s["kept"] = [[x[:, i, :, p:p + m] for i, p in enumerate(pasts)] for x in planes]
    return s


def _round_state(case, seed):
    x = _Draw(seed)(case["rows"], case["cols"]).to(DTYPES[case["dtype"]])
    s = {"x": x}
    if own:
        wrs = _package()
        s.update(ctx=_context(), packed=wrs.Mx4.empty(case["rows"], case["cols"]),
                 values=torch.empty_like(x))
    return s


def _linear_state(case, seed):
    x, ws, bs = _linear_inputs(case, seed)
    s = {"x": x, "ws": ws, "bs": bs, "act": case["act"], "both": case["x"] == "mx4",
         "out": DTYPES[case["out"]]}
    if own:
        wrs = _package()
        s["ctx"] = _context()
        s["ws"] = [wrs.Mx4(codes, scales) for codes, scales in ws]
        s["outs"] = [_empty(case["rows"], case["n_out"], dtype=s["out"]) for _ in ws]
        s["packed"] = wrs.Mx4.empty(*x.shape) if s["both"] else None
    return s


def prepare(case, seed):
    state = {"tree": _tree_state, "keep": _keep_state, "round": _round_state,
             "linear": _linear_state}[case["op"]](case, seed)
    state["op"] = case["op"]
    return state


# --------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------

def _tree_plain(s):
    """Scores of every node against its slot's whole plane, hidden keys at -infinity."""
    h, n_most = s["heads"], max(s["counts"])
    tree, node = s["tree_of"], s["node_of"]
    n_trees, keys = len(s["counts"]), s["planes"][0].shape[2]
    q = torch.zeros(n_trees, n_most, h * D, device="cuda")
    q[tree, node] = s["q"]
    q = q.view(n_trees, n_most, h, D).transpose(1, 2).contiguous()
    # ancestors: the inverse of (1 - parent matrix), a sum of its powers
    step = torch.zeros(n_trees, n_most, n_most + 1, device="cuda")
    step[tree, node, s["parents"].long() + 1] = 1.0
    eye = torch.eye(n_most, device="cuda").expand(n_trees, -1, -1)
    above = torch.linalg.solve_triangular(eye - step[:, :, 1:], eye, upper=False,
                                          unitriangular=True) > 0.5
    at = torch.arange(keys, device="cuda")[None] - s["pasts"][:, None]
    drafted = (at >= 0) & (at < s["lengths"][:, None])
    seen = above.gather(2, at.clamp(0, n_most - 1)[:, None].expand(-1, n_most, -1))
    seen = (seen & drafted[:, None]) | (at < 0)[:, None]
    k, v = (x.float() for x in s["planes"])
    scores = torch.matmul(q, k.transpose(2, 3).contiguous()) * D ** -0.5
    scores.masked_fill_(~seen[:, None], -math.inf)
    p = torch.exp(scores - scores.amax(dim=-1, keepdim=True))
    out = torch.matmul(p, v) / p.sum(dim=-1, keepdim=True)
    return out.transpose(1, 2).reshape(n_trees, n_most, h * D)[tree, node]


def _gelu(x):
    return 0.5 * x * (1.0 + torch.tanh(0.7978846 * x * (1.0 + 0.044715 * x * x)))


def _linear_plain(s):
    x = _mx4_values(s["x"]) if s["both"] else s["x"].float()
    ys = [torch.addmm(b, x, _mx4_unpack(*w).T) for w, b in zip(s["ws"], s["bs"])]
    return [(_gelu(y) if s["act"] else y).to(s["out"]) for y in ys]


def run(state):
    s = state
    op = s["op"]
    if op == "tree":
        if own:
            s["arena"].tree_self(0, s["slots"], s["counts"], s["parents"], s["q"], s["out"])
            return s["out"]
        return _tree_plain(s)
    if op == "keep":
        if own:
            s["arena"].keep_rows(s["slots"], s["counts"], s["rows"])
        else:
            k, v = s["planes"]
            k[:, s["slot_of"], :, s["to"]] = k[:, s["slot_of"], :, s["from"]]
            v[:, s["slot_of"], :, s["to"]] = v[:, s["slot_of"], :, s["from"]]
        return s["kept"]
    if op == "round":
        if own:
            wrs = _package()
            wrs.mx4_quantize(s["x"], s["packed"], ctx=s["ctx"])
            wrs.mx4_dequantize(s["packed"], s["values"], ctx=s["ctx"])
            return s["values"]
        return _mx4_values(s["x"]).to(s["x"].dtype)
    if own:
        wrs = _package()
        x = s["x"]
        if s["both"]:
            wrs.mx4_quantize(x, s["packed"], ctx=s["ctx"])
            x = s["packed"]
        wrs.linear_mx4(x, s["ws"], s["bs"], s["outs"], act="gelu" if s["act"] else None,
                       ctx=s["ctx"])
        return s["outs"]
    return _linear_plain(s)


# --------------------------------------------------------------------------
# the same from the definitions, in 64 bits
# --------------------------------------------------------------------------

def _tree_exact(case, seed):
    rows, q, parents = _tree_inputs(case, seed)
    outs, row = [], 0
    for (k, v), tree, past in zip(rows, parents, _pasts(case)):
        n = len(tree)
        seen = torch.zeros(n, past + n, dtype=torch.bool)
        seen[:, :past] = True
        for i in range(n):
            a = i
            while a >= 0:
                seen[i, past + a] = True
                a = int(tree[a])
        hide = ~seen.cuda()
        k, v = (x.to(DTYPES[case["dtype"]]).double() for x in (k, v))
        qs = q[row:row + n].double()
        out = torch.empty_like(qs)
        for h in range(case["heads"]):
            c = slice(h * D, (h + 1) * D)
            sc = (qs[:, c] @ k[:, c].T.contiguous()) / 8.0
            out[:, c] = torch.softmax(sc.masked_fill_(hide, -math.inf), dim=1) @ v[:, c]
        outs.append(out)
        row += n
    return torch.cat(outs)


def _keep_exact(case, seed):
    planes = [x.double() for x in _keep_planes(case, seed)]
    picks = _keep_rows(case, seed)
    return [[x[:, i, :, [p + int(r) for r in picks[i]]] for i, p in enumerate(_pasts(case))]
            for x in planes]


def _mx4_exact(x):
    """Nearest e2m1 value of every element in units of its block's scale, in 64 bits."""
    b = x.double().reshape(-1, BLOCK)
    top = b.abs().amax(dim=1, keepdim=True)
    unit = torch.where(top > 0, torch.exp2(torch.floor(torch.log2(top)) - 2), 2.0 ** -127)
    unit = torch.where(2 * unit * 4 <= top, 2 * unit, unit)  # log2 rounded across a power of two
    unit = torch.where(unit * 4 > top, unit / 2, unit).clamp(min=2.0 ** -127)
    y = b.abs() / unit
    values = torch.tensor(E2M1, dtype=torch.float64, device=x.device)
    low = (torch.searchsorted(values, y.clamp(max=6.0).contiguous(), right=True) - 1).clamp(0, 6)
    up = y - values[low] - (values[low + 1] - y)
    low = low + ((up > 0) | ((up == 0) & (low % 2 == 1))).long()
    return torch.copysign(values[low] * unit, b).reshape(x.shape)


def _linear_exact(case, seed):
    x, ws, bs = _linear_inputs(case, seed)
    x = _mx4_exact(x) if case["x"] == "mx4" else x.double()
    ys = []
    for (codes, scales), b in zip(ws, bs):
        code = torch.stack([codes & 15, codes >> 4], dim=2).reshape(codes.shape[0], -1).long()
        values = torch.tensor(E2M1 + tuple(-v for v in E2M1), dtype=torch.float64, device="cuda")
        w = values[code] * torch.exp2(scales.double() - 127).repeat_interleave(BLOCK, dim=1)
        y = x @ w.T.contiguous() + b.double()
        if case["act"]:
            y = 0.5 * y * (1.0 + torch.tanh(0.7978846 * y * (1.0 + 0.044715 * y * y)))
        ys.append(y)
    return ys


def exact(case, seed):
    if case["op"] == "tree":
        return _tree_exact(case, seed)
    if case["op"] == "keep":
        return _keep_exact(case, seed)
    if case["op"] == "round":
        return _mx4_exact(_Draw(seed)(case["rows"], case["cols"]).to(DTYPES[case["dtype"]]))
    return _linear_exact(case, seed)
