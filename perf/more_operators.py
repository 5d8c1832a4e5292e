"""Timed cases of the operators of long sessions: an 8-bit cache, windows, scores.

Storing rows in a cache of 8-bit codes with a scale for each row and head (and
reading them back), attention over such a cache, attention that sees a sliding
window and the first tokens, and the log probabilities of given tokens with
entropy and the likeliest alternatives. Every case is one call (or one call and
its inverse) as a decoder or a scorer makes it; widths are those of the
workloads in this repository (heads of 64, 6 to 20 of them, 1500 encoder frames,
vocabularies around 51865). Inputs are drawn on the GPU from the case's seed.
"""
from __future__ import annotations

import importlib.util
import math
import sys
from pathlib import Path

import torch

own = False

D = 64  # head width
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
MODELS = ((6, 4), (8, 6), (12, 12), (16, 24), (20, 32))  # (heads, layers)
MOST_TOP = 32  # alternatives of one row


# --------------------------------------------------------------------------
# the cases
# --------------------------------------------------------------------------

def listed():
    return [
        # One step of five beams of a large decoder: a new row for each.
        {"name": "store_i8_beam5", "op": "store", "heads": 20, "slots": 5, "rows": 1, "past": 223},
        # Four long sessions of a small decoder come back into the cache.
        {"name": "store_i8_sessions", "op": "store", "heads": 12, "slots": 4, "rows": 11003,
         "past": 0},
        # The self-attention of a beam-5 step of a small decoder.
        {"name": "attend_i8_self_beam5", "op": "attend", "heads": 12, "slots": 5, "rows": 1,
         "past": 223, "cross": False},
        # The cross-attention of a beam-5 step of a large one: its frames are shared.
        {"name": "attend_i8_cross_beam5", "op": "attend", "heads": 20, "slots": 1, "rows": 5,
         "past": 1500, "cross": True},
        # A whole prompt of the previous text over the encoder's frames.
        {"name": "attend_i8_cross_prompt", "op": "attend", "heads": 20, "slots": 1, "rows": 223,
         "past": 1500, "cross": True},
        # The smallest step: a greedy tiny decoder with a window over its 448 positions.
        {"name": "window_f16_tiny", "op": "window", "heads": 6, "slots": 1, "rows": 1, "past": 441,
         "window": 128, "sinks": 4, "dtype": "f16"},
        # Sixteen long sessions of a large decoder, one token each, 8-bit cache.
        {"name": "window_i8_streams", "op": "window", "heads": 20, "slots": 16, "rows": 1,
         "past": 30011, "window": 8192, "sinks": 16, "dtype": "i8"},
        # A long text goes in behind a prompt: every row has its own window.
        {"name": "window_f16_prompt", "op": "window", "heads": 20, "slots": 1, "rows": 8191,
         "past": 500, "window": 1024, "sinks": 4, "dtype": "f16"},
        # Short ragged pieces of four small streams over an f32 cache.
        {"name": "window_f32_small_x4", "op": "window", "heads": 12, "slots": 4, "rows": 33,
         "past": 2900, "window": 448, "sinks": 1, "dtype": "f32"},
        # A beam-5 step: suppressed tokens, ten continuations for each beam.
        {"name": "score_f32_beam5", "op": "score", "rows": 5, "vocab": 51866, "top": 10,
         "dtype": "f32", "allowed": "shared", "temperature": 1.0},
        # Five drafted trees of a step, each row with its own permitted tokens.
        {"name": "score_f32_drafts", "op": "score", "rows": 130, "vocab": 51865, "top": 1,
         "dtype": "f32", "allowed": "rows", "temperature": 0.4},
        # Sixteen full transcripts scored at once from f16 logits.
        {"name": "score_f16_transcripts", "op": "score", "rows": 7168, "vocab": 51865, "top": 5,
         "dtype": "f16", "allowed": "none", "temperature": 1.0},
    ]


def _length(rng, lo, hi):
    """A length spread over the logarithm of [lo, hi]; odd ones among them."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    most = [work(c) for c in listed()]
    top_bytes, top_flops = (max(w[k] for w in most) for k in ("bytes", "flops"))
    while True:
        op = rng.choice(["store", "attend", "attend", "window", "window", "score", "score"])
        heads, _ = rng.choice(MODELS)
        if op == "store":
            c = {"op": op, "heads": heads, "slots": _length(rng, 1, 16),
                 "rows": rng.choice([1, _length(rng, 1, 20000)]),
                 "past": rng.choice([0, _length(rng, 1, 2000)])}
        elif op == "attend":
            cross = rng.random() < 0.5
            c = {"op": op, "heads": heads, "slots": 1 if cross else _length(rng, 1, 16),
                 "rows": _length(rng, 1, 448), "past": _length(rng, 1, 1500 if cross else 65536),
                 "cross": cross}
            if c["slots"] > 1:
                c["rows"] = 1  # a step; prompts come one slot at a time
        elif op == "window":
            c = {"op": op, "heads": heads, "slots": _length(rng, 1, 16),
                 "rows": rng.choice([1, _length(rng, 1, 8192)]),
                 "past": rng.choice([0, _length(rng, 1, 448), _length(rng, 1, 65536)]),
                 "window": _length(rng, 1, 16384), "sinks": rng.choice([0, _length(rng, 1, 64)]),
                 "dtype": rng.choice(["f16", "f32", "i8", "i8"])}
        else:
            vocab = rng.choice([51864, 51865, 51866, _length(rng, 40, 65536)])
            c = {"op": op, "rows": _length(rng, 1, 8192), "vocab": vocab,
                 "top": rng.randint(1, min(MOST_TOP, vocab // 8)),
                 "dtype": rng.choice(["f32", "f16", "bf16"]),
                 "allowed": rng.choice(["none", "shared", "rows"]),
                 "temperature": rng.choice([1.0, 1.0, 0.2, 0.4, 0.6, 0.8])}
        if op in ("attend", "window"):
            keys = c["past"] + (0 if op == "attend" and c["cross"] else c["rows"])
            if c["slots"] * keys * heads > 9_700_000:
                continue
            if c["slots"] * c["rows"] * keys * heads > 1_430_000_000:
                continue  # what the plain form's scores may take
        w = work(c)
        if w["bytes"] <= top_bytes and w["flops"] <= top_flops:
            return c


def _counts(case):
    """New rows of each slot: pieces of text differ by a few tokens."""
    return [max(1, case["rows"] - (5 * i) % 7) for i in range(case["slots"])]


def _pasts(case):
    """Cached rows of each slot: histories differ by a few tokens."""
    return [max(0, case["past"] - (3 * i) % 11) for i in range(case["slots"])]


def work(case):
    op = case["op"]
    size = {"f32": 4, "f16": 2, "bf16": 2, "i8": 1 + 1 / D}
    b = f = 0
    if op == "store":
        n = sum(_counts(case)) * case["heads"] * D
        b = 2 * n * (4 + size["i8"] + 4)  # rows in, the cache, the values it stands for
        f = 2 * n * 4
    elif op == "attend" and case["cross"]:
        d = case["heads"] * D
        b = 2 * case["past"] * d * size["i8"] + 8 * case["rows"] * d
        f = 4 * case["rows"] * case["past"] * d
    elif op in ("attend", "window"):
        d = case["heads"] * D
        window = case.get("window", 1 << 40)
        sinks = case.get("sinks", 0)
        for n, p in zip(_counts(case), _pasts(case)):
            span = min(p + n, window + n - 1)  # keys that some row's window holds
            keys = span + min(sinks, p + n - span)
            b += 2 * keys * d * size[case.get("dtype", "i8")] + 8 * n * d
            for at in (p, p + n - 1):  # the rows' visible keys, between the first and the last
                seen = min(at + 1, window) + min(sinks, max(0, at + 1 - window))
                f += 2 * n * seen * d
    else:
        r, v = case["rows"], case["vocab"]
        b = r * v * size[case["dtype"]] + {"none": 0, "shared": 1, "rows": r}[case["allowed"]] * v
        b += r * (4 + 4 + 4 + 8 * case["top"])
        f = 5 * r * v
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

    def whole(self, most, *shape):
        return torch.randint(most, shape, generator=self.gen, device="cuda")


def _kv_rows(r, n, d):
    """K and V rows; a few channels of K are large, as a decoder's are."""
    k, v = r(n, d), r(n, d)
    k[:, ::47] *= 6.0
    return k, v


def _store_inputs(case, seed):
    """K and V rows, as two thirds of a fused projection's rows ([row][q, k, v])."""
    r = _Draw(seed)
    d = case["heads"] * D
    qkv = r(sum(_counts(case)), 3 * d)
    qkv[:, d::47] *= 6.0
    return qkv


def _attend_inputs(case, seed):
    """Rows of each slot's cache ((k, v), [row][heads * 64] f32) and q."""
    r = _Draw(seed)
    d = case["heads"] * D
    if case["op"] == "attend" and case["cross"]:
        rows = [_kv_rows(r, case["past"], d)]
        return rows, r(case["rows"], d)
    counts, pasts = _counts(case), _pasts(case)
    rows = [_kv_rows(r, p + n, d) for p, n in zip(pasts, counts)]
    # the queries lie in a fused projection's rows ([row][q, k, v]) where the call takes strides
    q = r(sum(counts), 3 * d)[:, :d] if case["op"] == "window" else r(sum(counts), d)
    return rows, q


def _score_inputs(case, seed):
    """Logits with a few likely tokens a row, the tokens to score and the permitted ones."""
    r = _Draw(seed)
    n, v = case["rows"], case["vocab"]
    logits = torch.empty(n, v, dtype=DTYPES[case["dtype"]], device="cuda")
    likely = r.whole(v, n, 8)
    lift = r(n, 8).abs_().mul_(5.0)
    for a in range(0, n, 512):
        x = r(min(512, n - a), v, sigma=2.2)
        x.scatter_add_(1, likely[a:a + 512], lift[a:a + 512])
        logits[a:a + 512] = x.to(logits.dtype)
    # two in three scored tokens are likely ones
    some = torch.arange(n, device="cuda") % 3
    tokens = torch.where(some < 2, likely.gather(1, some[:, None].clamp(max=1))[:, 0],
                         r.whole(v, n)).int()
    allowed = None
    if case["allowed"] == "shared":
        allowed = r.whole(500, 1, v) > 0
        allowed[0, tokens.long()] = True
    elif case["allowed"] == "rows":
        allowed = r.whole(3, n, v) > 0
        allowed.scatter_(1, tokens.long()[:, None], True)
    return logits, tokens, allowed


def _codes(x):
    """[...][64] f32 as 8-bit codes and the power of two of each 64, nearest, ties to even.

    The power is the least that leaves no code past 127."""
    top = x.abs().amax(dim=-1, keepdim=True)
    e = torch.frexp(top)[1] - 7  # the largest comes to [64, 128)
    e = torch.where(torch.ldexp(top, -e) >= 127.5, e + 1, e).clamp(-126, 121)
    return torch.round(torch.ldexp(x, -e)).clamp(-127, 127).to(torch.int8), e


def _values(codes, e):
    return torch.ldexp(codes.float(), e)


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


def _arena(slots, heads, rows, frames, dtype):
    wrs = _package()
    return wrs.KvArena(1, slots, heads, max(rows, 1), frames, ctx=_context(),
                       dtype={"f16": wrs.WRS_F16, "f32": wrs.WRS_F32, "i8": wrs.WRS_I8}[dtype])


def _store_state(case, seed):
    d = case["heads"] * D
    counts, pasts = _counts(case), _pasts(case)
    qkv = _store_inputs(case, seed)
    s = {"k": qkv[:, d:2 * d], "v": qkv[:, 2 * d:], "heads": case["heads"],
         "slots": list(range(case["slots"])), "counts": counts, "pasts": pasts}
    if own:
        most = max(p + n for p, n in zip(pasts, counts))
        s["arena"] = arena = _arena(case["slots"], case["heads"], most, 0, "i8")
        for slot, n in enumerate(pasts):
            arena.advance(slot, n)
        n = sum(counts)
        s["out"] = [_empty(n, d), _empty(n, d)]
    return s


def _attend_state(case, seed):
    rows, q = _attend_inputs(case, seed)
    dtype = case.get("dtype", "i8")
    cross = case["op"] == "attend" and case["cross"]
    counts, pasts = _counts(case), _pasts(case)
    lengths = [k.shape[0] for k, _ in rows]
    h = case["heads"]
    s = {"q": q, "heads": h, "cross": cross, "slots": list(range(case["slots"])),
         "counts": [case["rows"]] if cross else counts, "window": case.get("window"),
         "sinks": case.get("sinks", 0)}
    if own:
        frames = lengths[0] if cross else 0
        s["arena"] = arena = _arena(case["slots"], h, 0 if cross else max(lengths), frames, dtype)
        for slot, (k, v) in enumerate(rows):
            if cross:
                arena.set_cross(0, k, v)
            else:
                arena.append(0, slot, k, v)
                arena.advance(slot, pasts[slot])
        s["out"] = _empty(*q.shape)
        return s
    most = max(lengths)
    shape = (case["slots"], h, most, D)
    planes = []
    for i in range(2):
        x = torch.zeros(shape, device="cuda")
        for slot, kv in enumerate(rows):
            x[slot, :, :lengths[slot]] = kv[i].view(-1, h, D).transpose(0, 1)
        planes.append(_codes(x) if dtype == "i8" else x.to(DTYPES[dtype]))
    s["planes"] = planes
    s["past"] = torch.tensor(pasts, device="cuda")
    s["slot_of"] = torch.repeat_interleave(torch.arange(len(s["counts"]), device="cuda"),
                                           torch.tensor(s["counts"], device="cuda"))
    s["row_of"] = torch.cat([torch.arange(n, device="cuda") for n in s["counts"]])
    return s


def _score_state(case, seed):
    logits, tokens, allowed = _score_inputs(case, seed)
    s = {"logits": logits, "tokens": tokens, "allowed": allowed, "top": case["top"],
         "temperature": case["temperature"]}
    if own:
        n, k = case["rows"], case["top"]
        s["ctx"] = _context()
        s["outs"] = [_empty(n), _empty(n), _empty(n, k, dtype=torch.int32), _empty(n, k)]
    return s


def prepare(case, seed):
    state = {"store": _store_state, "attend": _attend_state, "window": _attend_state,
             "score": _score_state}[case["op"]](case, seed)
    state["op"] = case["op"]
    return state


# --------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------

def _attend_plain(s):
    """Scores of every row against its slot's whole plane, hidden keys at -infinity."""
    h, slots, most = s["heads"], len(s["counts"]), max(s["counts"])
    slot, row = s["slot_of"], s["row_of"]
    q = torch.zeros(slots, most, h * D, device="cuda")
    q[slot, row] = s["q"]
    q = q.view(slots, most, h, D).transpose(1, 2).contiguous()
    k, v = (_values(*x) if isinstance(x, tuple) else x.float() for x in s["planes"])
    scores = torch.matmul(q, k.transpose(2, 3).contiguous()) * D ** -0.5
    if not s["cross"]:
        key = torch.arange(k.shape[2], device="cuda")
        at = (s["past"][:, None] + torch.arange(most, device="cuda"))[:, :, None]
        hidden = key > at
        if s["window"] is not None:
            hidden |= (key <= at - s["window"]) & (key >= s["sinks"])
        scores.masked_fill_(hidden[:, None], -math.inf)
    scores -= scores.amax(dim=-1, keepdim=True)
    scores.exp_()
    out = torch.matmul(scores, v) / scores.sum(dim=-1, keepdim=True)
    return out.transpose(1, 2).reshape(slots, most, h * D)[slot, row]


def _score_plain(s):
    x = s["logits"].float()
    if s["allowed"] is not None:
        x = x.masked_fill(~s["allowed"], -math.inf)
    # likeliest first, the lowest index among equals; by parts, for the sort's memory
    best = [torch.sort(part, dim=1, descending=True, stable=True)[1][:, :s["top"]].clone()
            for part in x.split(1024)]
    ids = torch.cat(best)
    z = x / s["temperature"]
    z -= z.amax(dim=1, keepdim=True)
    p = z.exp()
    total = p.sum(dim=1)
    lse = total.log()
    entropy = lse - torch.where(p > 0, p * z, 0.0).sum(dim=1) / total
    at = z.gather(1, s["tokens"].long()[:, None])[:, 0]
    return [at - lse, entropy, ids.int(), z.gather(1, ids) - lse[:, None]]


def run(state):
    s = state
    op = s["op"]
    if op == "store":
        if own:
            k, v = s["out"]
            s["arena"].append_rows(0, s["slots"], s["counts"], s["k"], s["v"])
            s["arena"].read_rows(0, s["slots"], s["pasts"], s["counts"], k, v)
            return s["out"]
        return [_values(*_codes(x.reshape(x.shape[0], s["heads"], D))).reshape(x.shape)
                for x in (s["k"], s["v"])]
    if op == "score":
        if not own:
            return _score_plain(s)
        logprobs, entropy, ids, top = s["outs"]
        _package().token_logprobs(s["logits"], s["tokens"], logprobs, entropy=entropy,
                                  top_ids=ids, top_logprobs=top, allowed=s["allowed"],
                                  temperature=s["temperature"], ctx=s["ctx"])
        return s["outs"]
    if not own:
        return _attend_plain(s)
    arena, q, out = s["arena"], s["q"], s["out"]
    if op == "window":
        arena.window_self(0, s["slots"], s["counts"], s["window"], s["sinks"], q, out)
    elif s["cross"]:
        (arena.decode_cross if q.shape[0] <= 8 else arena.prefill_cross)(0, q, out)
    elif s["counts"] == [1] * len(s["counts"]):
        arena.decode_self(0, s["slots"], q, out)
    else:
        arena.prefill_self(0, 0, q, out)
    return out


# --------------------------------------------------------------------------
# the same from the definitions, in 64 bits
# --------------------------------------------------------------------------

def _stored_exact(x):
    """The values that 8-bit codes of x's blocks of 64 stand for."""
    b = x.double().reshape(-1, D)
    top = b.abs().amax(dim=1, keepdim=True)
    unit = torch.exp2(torch.floor(torch.log2(top.clamp(min=2.0 ** -120))) - 7)
    for _ in range(3):  # the least power of two whose codes end at 127
        unit = torch.where(top >= 127.5 * unit, 2 * unit, unit)
    unit = unit.clamp(min=2.0 ** -126)
    n = torch.floor(b / unit)
    rest = b / unit - n
    up = (rest > 0.5) | ((rest == 0.5) & (torch.remainder(n, 2) == 1))
    return ((n + up) * unit).reshape(x.shape)


def _store_exact(case, seed):
    d = case["heads"] * D
    qkv = _store_inputs(case, seed)
    return [_stored_exact(qkv[:, a:a + d]) for a in (d, 2 * d)]


def _attend_exact(case, seed):
    rows, q = _attend_inputs(case, seed)
    cross = case["op"] == "attend" and case["cross"]
    counts = [case["rows"]] if cross else _counts(case)
    dtype = case.get("dtype", "i8")
    window, sinks = case.get("window", 1 << 40), case.get("sinks", 0)
    out, first = torch.empty(q.shape, dtype=torch.float64, device="cuda"), 0
    for (k, v), n in zip(rows, counts):
        k, v = (_stored_exact(x) if dtype == "i8" else x.to(DTYPES[dtype]).double()
                for x in (k, v))
        hide = torch.zeros(n, k.shape[0], dtype=torch.bool, device="cuda")
        if not cross:
            ahead = (torch.arange(k.shape[0] - n, k.shape[0], device="cuda")[:, None]
                     - torch.arange(k.shape[0], device="cuda")[None])  # tokens back from the row
            hide = (ahead < 0) | ((ahead >= window)
                                  & (torch.arange(k.shape[0], device="cuda")[None] >= sinks))
        qs = q[first:first + n].double()
        for c in (slice(i * D, (i + 1) * D) for i in range(case["heads"])):
            sc = (qs[:, c] @ k[:, c].T.contiguous()) / 8.0
            out[first:first + n, c] = torch.softmax(sc.masked_fill_(hide, -math.inf), 1) @ v[:, c]
        first += n
    return out


def _score_exact(case, seed):
    logits, tokens, allowed = _score_inputs(case, seed)
    parts = []
    for a in range(0, case["rows"], 256):
        x = logits[a:a + 256].double()
        if allowed is not None:
            ok = allowed if allowed.shape[0] == 1 else allowed[a:a + 256]
            x = torch.where(ok, x, -math.inf)
        lp = torch.log_softmax(x / case["temperature"], dim=1)
        h = -torch.where(lp > -math.inf, lp.exp() * lp, 0.0).sum(dim=1)
        t = tokens[a:a + 256].long()
        left, best = lp.clone(), []
        for _ in range(case["top"]):
            m = left.amax(dim=1, keepdim=True)
            best.append(m)
            first = (left == m).int().argmax(dim=1, keepdim=True)
            left.scatter_(1, first, -math.inf)
        parts.append((lp.gather(1, t[:, None])[:, 0], h, torch.cat(best, dim=1)))
    lp, h, top = (torch.cat(x) for x in zip(*parts))
    return [lp, h, None, top]


def exact(case, seed):
    return {"store": _store_exact, "attend": _attend_exact, "window": _attend_exact,
            "score": _score_exact}[case["op"]](case, seed)
