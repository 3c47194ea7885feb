"""The operators that serve several requests on one resident model, and what they are measured on.

Three groups, each reached through llm_accel.Accelerator:

  attention  the rows of a batch whose sequences share a long prefix (one copy of it, in the
             context's cache) and continue it each in K/V rows of its own
  adapted    a resident projection with a low-rank adapter of each row's own request
  probs      the target's next-token probabilities of hidden rows, through the LM head
  verify     the drafted tokens of several requests, tested against those probabilities with
             random numbers that the caller gives, and the token after the accepted ones

All values are fixed point, all results whole numbers (raw Q8.8 rows, Q0.32 probabilities,
token ids), so both forms have to agree bit for bit.
"""
import math
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.join(os.getcwd(), "llm-accel_amd"))

import llm_accel  # noqa: E402

own = False

# hidden, intermediate, query heads, KV heads
SHAPES = {
    "small": (256, 688, 4, 2),
    "mid": (896, 4864, 14, 2),
    "odd": (480, 1300, 10, 2),       # head_dim 48, nothing a multiple of 128
    "large": (2048, 11008, 16, 2),
}
# operator -> (outputs, inputs) of the projection as keys of _dims()
PROJECTIONS = {"q": ("h", "h"), "k": ("c", "h"), "v": ("c", "h"), "o": ("h", "h"),
               "gate": ("i", "h"), "up": ("i", "h"), "down": ("h", "i")}
OPS = {"q": 1, "k": 2, "v": 3, "o": 4, "gate": 5, "up": 6, "down": 7}


def listed():
    return [
        # Two answers to one short question: launches are all of it.
        {"name": "attention_small", "kind": "attention", "shape": "small", "sequences": 2,
         "prefix": 40, "own": 8, "outliers": False},
        # A handful of continuations of a chat, of ragged lengths, on 7 query heads a group.
        {"name": "attention_chat", "kind": "attention", "shape": "mid", "sequences": 5,
         "prefix": 1003, "own": 200, "outliers": False},
        # Eight continuations of a long document.
        {"name": "attention_long", "kind": "attention", "shape": "large", "sequences": 8,
         "prefix": 16000, "own": 300, "outliers": False},
        # A wide batch over one long system prompt; keys with outlier channels past Q4.12.
        {"name": "attention_wide", "kind": "attention", "shape": "large", "sequences": 32,
         "prefix": 8100, "own": 600, "outliers": True},
        # One decode row under one request's adapter.
        {"name": "adapted_row", "kind": "adapted", "shape": "large", "proj": "q", "rows": 1,
         "adapters": 1, "rank": 16},
        # Five requests under three small adapters of odd rank, one row without any.
        {"name": "adapted_mixed", "kind": "adapted", "shape": "mid", "proj": "up", "rows": 5,
         "adapters": 3, "rank": 13},
        # A full block, every row under an adapter of its own, over the long input side.
        {"name": "adapted_block", "kind": "adapted", "shape": "large", "proj": "down",
         "rows": 8, "adapters": 8, "rank": 64},
        # Next-token probabilities of one decode row over the whole vocabulary (a sampler's
        # or drafter's step).
        {"name": "probs_row", "kind": "probs", "shape": "large", "rows": 1, "vocab": 151936},
        # The same of a block on a small model of no round vocabulary.
        {"name": "probs_block", "kind": "probs", "shape": "mid", "rows": 8, "vocab": 32011},
        # One request's three looked-up drafts on a small model.
        {"name": "verify_small", "kind": "verify", "shape": "small", "requests": 1, "rows": 4,
         "vocab": 1024, "sampled": False},
        # Three requests of ragged draft lengths, drafts looked up in their own texts.
        {"name": "verify_ragged", "kind": "verify", "shape": "mid", "requests": 3, "rows": 8,
         "vocab": 32011, "sampled": False},
        # Seven drafts sampled from a draft model over the whole vocabulary.
        {"name": "verify_block", "kind": "verify", "shape": "large", "requests": 1, "rows": 8,
         "vocab": 151936, "sampled": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attention", "attention", "attention", "adapted", "adapted", "probs",
                       "verify", "verify"])
    shape = rng.choice(["small", "mid", "odd", "large", "large"])
    if kind == "attention":
        sequences = _log(rng, 1, 32)
        prefix = _log(rng, 1, min(16000, 260000 // sequences)) - rng.choice([0, 1])
        return {"kind": kind, "shape": shape, "sequences": sequences, "prefix": prefix,
                "own": _log(rng, 1, 600), "outliers": rng.random() < 0.3}
    if kind == "adapted":
        rows = rng.randint(1, 8)
        return {"kind": kind, "shape": shape, "proj": rng.choice(sorted(PROJECTIONS)),
                "rows": rows, "adapters": rng.randint(1, rows), "rank": _log(rng, 1, 64)}
    rows = rng.randint(1, 8)
    vocab = _log(rng, 1000, 151936)
    if kind == "probs":
        return {"kind": kind, "shape": shape, "rows": rows, "vocab": vocab}
    return {"kind": kind, "shape": shape, "requests": rng.randint(1, rows), "rows": rows,
            "vocab": vocab, "sampled": rng.random() < 0.5}


def _dims(case):
    h, i, heads, kv_heads = SHAPES[case["shape"]]
    return {"h": h, "i": i, "heads": heads, "kv": kv_heads, "group": heads // kv_heads,
            "d": h // heads, "c": kv_heads * (h // heads)}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _generator(seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return gen


def _whole(gen, limit, *shape):
    """Whole numbers spread evenly over [-limit, limit]."""
    return torch.randint(-limit, limit + 1, shape, generator=gen, device="cuda",
                         dtype=torch.int16)


def _normal(gen, sigma, *shape):
    """Q8.8 values of a normal distribution cut at four sigmas."""
    x = torch.randn(shape, generator=gen, device="cuda").clamp_(-4, 4)
    return (x * (sigma * 256)).round_().to(torch.int16)


def _uniforms(gen, n):
    """32-bit uniform numbers, as a host program's generator gives them."""
    return [int(u) for u in torch.randint(0, 1 << 32, (n,), generator=gen, device="cuda",
                                          dtype=torch.int64).cpu()]


def _split(rng, total, parts):
    """`total` rows over `parts` requests, at least one each."""
    cuts = sorted(rng.choice(np.arange(1, total), parts - 1, replace=False).tolist())
    return [b - a for a, b in zip([0] + cuts, cuts + [total])]


def _inputs(case, seed):
    """The tensors and numbers of a case, without any handle."""
    gen, rng, n = _generator(seed), np.random.default_rng([7, seed]), _dims(case)
    kind, s = case["kind"], {"case": case}
    if kind == "attention":
        t, p, cap, kv, d = case["sequences"], case["prefix"], case["own"], n["kv"], n["d"]
        # rotated queries and keys whose scores spread as a trained model's do: few of the
        # positions hold most of the weight
        s["q"] = _normal(gen, 2.0, t, n["heads"], d)
        s["k"], s["v"] = _normal(gen, 1.5, kv, p, d), _normal(gen, 0.5, kv, p, d)
        s["k_own"], s["v_own"] = (_normal(gen, x, t, kv, cap, d) for x in (1.5, 0.5))
        if case["outliers"]:  # one channel of the keys lies far out, as projections' do
            for k in (s["k"], s["k_own"]):
                k[..., 5] = (k[..., 5].int() * 8 + 1800).clamp_(-32768, 32767).to(torch.int16)
        # positions that each sequence has generated so far
        s["lengths"] = torch.from_numpy(rng.integers(0, cap + 1, t).astype(np.int32)).cuda()
        s["out"] = torch.zeros((t, n["heads"], d), dtype=torch.int16, device="cuda")
    elif kind == "adapted":
        rows, count, rank = case["rows"], case["adapters"], case["rank"]
        outs, ins = (n[x] for x in PROJECTIONS[case["proj"]])
        s["w"] = _whole(gen, 512, outs, ins)
        s["x"] = _normal(gen, 1.0, rows, ins)
        # each adapter's factors, A [rank][inputs] and B [rank][outputs], and alpha / rank
        s["a"] = _whole(gen, 300, count, rank, ins)
        s["b"] = _whole(gen, 300, count, rank, outs)
        s["ranks"] = [rank if j == 0 else int(rng.integers(1, rank + 1)) for j in range(count)]
        for j, r in enumerate(s["ranks"]):  # what a smaller adapter does not have
            s["a"][j, r:], s["b"][j, r:] = 0, 0
        s["scales"] = [int(x) for x in rng.integers(1 << 13, 1 << 17, count)]
        # every adapter has a row; the rows left over take any, or none
        more = rng.integers(-1, count, rows - count).tolist()
        s["of_row"] = [int(x) for x in rng.permutation(list(range(count)) + more)]
        s["out"] = torch.zeros((rows, outs), dtype=torch.int16, device="cuda")
    else:
        rows, vocab = case["rows"], case["vocab"]
        s["head"] = _whole(gen, 512, vocab, n["h"])
        s["x"] = _normal(gen, 1.5, rows, n["h"])
        if kind == "probs":
            s["temperatures"] = [float(x) for x in rng.uniform(0.5, 1.2, rows)]
            s["out"] = torch.zeros((rows, vocab), dtype=torch.int32, device="cuda")
        else:
            held = _split(rng, rows, case["requests"])
            s["counts"] = [x - 1 for x in held]
            s["temperatures"] = [float(x) for x in rng.uniform(0.5, 1.2, case["requests"])]
            of_row = torch.tensor(np.repeat(s["temperatures"], held), device="cuda")
            # the draft model: the same head on rows that are off by some noise
            noisy = (s["x"] + _normal(gen, 0.12, rows, n["h"])).float()
            p = torch.empty((rows, vocab), dtype=torch.float64, device="cuda")
            for at in range(0, vocab, 16384):
                p[:, at:at + 16384] = noisy @ s["head"][at:at + 16384].float().T
            p = torch.softmax(p / 2.0 ** 20 / of_row[:, None], dim=1)
            drafting = [r for r, last in enumerate(_last_rows(s["counts"])) if not last]
            p = p[drafting]
            if case["sampled"]:
                u = torch.rand((len(drafting), 1), generator=gen, device="cuda",
                               dtype=torch.float64)
                tokens = (p.cumsum(1) < u).sum(1).clamp_(max=vocab - 1)
                # probabilities in the Q0.32 that lm_head_probs gives them in
                q = (p * 2.0 ** 32).floor().clamp_(max=2.0 ** 32 - 1).to(torch.int64)
                s["q"] = torch.where(q >= 1 << 31, q - (1 << 32), q).to(torch.int32)
            else:
                tokens, s["q"] = p.argmax(1), None
            s["drafts"] = [int(x) for x in tokens.cpu()]
            s["accept_u"] = _uniforms(gen, len(drafting))
            s["sample_u"] = _uniforms(gen, case["requests"])
    return s


def _last_rows(counts):
    """For every row, whether it is its request's last (the one after its drafts)."""
    return [j == c for c in counts for j in range(c + 1)]


def prepare(case, seed):
    s, n, kind = _inputs(case, seed), _dims(case), case["kind"]
    room = case["prefix"] if kind == "attention" else 0
    acc = llm_accel.Accelerator(llm_accel.Shape(
        case.get("vocab", 1024), n["h"], n["i"], 1, n["heads"], n["kv"], room + 64, 1e6))
    if kind == "attention":
        if room:
            for head in range(n["kv"]):
                acc.kv_write(0, head, 0, s["k"][head].cpu().numpy(), s["v"][head].cpu().numpy())
        steps = torch.arange(-2048, 1, dtype=torch.float64) / 256
        s["exp14"] = (torch.exp(steps) * 16384).floor().to(torch.int64).cuda()
    elif kind == "adapted":
        acc.load_projection(0, OPS[case["proj"]] - 1, s["w"].cpu().numpy())
    else:
        acc.load_lm_head(s["head"].cpu().numpy())
        acc.upload(0, s["x"].cpu().numpy())
        s["exp2"] = [x.cuda() for x in _exp2_tables()]
    s["acc"] = acc
    return s


def _exp2_tables():
    """2^-(i / 2^10) and 2^-(j / 2^20), i, j < 1024, in units of 2^-30."""
    i = torch.arange(1024, dtype=torch.float64)
    return [torch.floor(torch.exp2(30 - i / 2.0 ** bits) + 0.5).to(torch.int64)
            for bits in (10, 20)]


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------

def _sat16(x):
    return x.clamp(-32768, 32767)


def _sat32(x):
    return x.clamp(-(1 << 31), (1 << 31) - 1)


def _round(x, bits):
    return (x + (1 << (bits - 1))) >> bits


def _product(a, b):
    """a @ b of whole numbers whose sums stay below 2^53."""
    return (a.double() @ b.double().contiguous()).long()


def _scores(q, k, d):
    """Q8.8 scores of queries [..., m, d] and keys [..., n, d]: products with keys clamped to
    Q4.12's range, in four saturating sums by the element's index modulo 4."""
    clamped = k.clamp(-2048, 2048)
    far = (k >= 2048).to(torch.int16)           # there the clamped factor is 8 - 2^-12
    less = (8 - q.int()) >> 4
    total = sum(_sat32(_product(q[..., b::4], clamped[..., b::4].transpose(-1, -2)) +
                       _product(less[..., b::4], far[..., b::4].transpose(-1, -2)))
                for b in range(4))
    scale = int(math.floor(256.0 / math.sqrt(d) + 0.5)) << 8
    return _sat16(_round(_sat32(_round(_sat32(total) * scale, 16)), 8))


def _values(p, v):
    """Q8.8 values of Q2.14 probabilities [..., m, 64] over one tile's V rows [..., 64, d]."""
    far = (v >= 2048).to(torch.int16)
    total = _product(p, v.clamp(-2048, 2048)) + _product((8 - p) >> 4, far)
    return _sat16(_round(_round(_sat32(total) * 1024, 16), 8))


def _plain_attention(s):
    case, n = s["case"], _dims(s["case"])
    t, p, cap, kv, g, d = (case["sequences"], case["prefix"], case["own"], n["kv"], n["group"],
                           n["d"])
    tiles, whole = -(-(p + cap) // 64), p // 64   # 64-position tiles; those of the prefix alone
    q = s["q"].reshape(t, kv, g, d)
    # scores over the prefix for all rows at once, over each sequence's own rows apart
    shared = _scores(q.permute(1, 0, 2, 3).reshape(kv, t * g, d), s["k"], d)
    shared = shared.reshape(kv, t, g, p).permute(1, 0, 2, 3)
    sc = torch.cat([shared, _scores(q, s["k_own"], d)], -1)
    sc = torch.nn.functional.pad(sc, (0, tiles * 64 - p - cap))
    ends = p + s["lengths"].long().clamp(0, cap)
    there = (torch.arange(tiles * 64, device="cuda")[None] < ends[:, None])[:, None, None]
    sc = torch.where(there, sc, -32768).reshape(t, kv, g, tiles, 64)
    # the running maximum after each tile, and the factor by which it shrinks what was before
    top = torch.cummax(sc.amax(-1), -1).values
    before = torch.nn.functional.pad(top[..., :-1], (1, 0), value=-32768)
    exp14 = lambda x: s["exp14"][x.clamp(-2048, 0) + 2048]  # noqa: E731
    old = exp14(before - top) << 2
    prob = torch.where(there.reshape(t, 1, 1, tiles, 64), exp14(sc - top[..., None]), 0)
    sums = prob.sum(-1) << 2
    # each tile's values: the whole prefix tiles for all rows at once, the others by sequence
    first = prob[..., :whole, :].permute(1, 3, 0, 2, 4).reshape(kv, whole, t * g, 64)
    first = _values(first, s["v"][:, :whole * 64].reshape(kv, whole, 64, d))
    first = first.reshape(kv, whole, t, g, d).permute(2, 0, 3, 1, 4)
    rest = torch.cat([s["v"][:, whole * 64:].expand(t, kv, -1, d), s["v_own"]], 2)
    rest = torch.nn.functional.pad(rest, (0, 0, 0, tiles * 64 - p - cap))
    rest = _values(prob[..., whole:, :].transpose(2, 3),
                   rest.reshape(t, kv, tiles - whole, 64, d)).transpose(2, 3)
    tile = torch.cat([first, rest], 3)
    # the recurrence over the tiles rounds at each of them: it has no closed form
    total = torch.zeros((t, kv, g), dtype=torch.int64, device="cuda")
    acc = torch.zeros((t, kv, g, d), dtype=torch.int64, device="cuda")
    for j in range(tiles):
        total = _sat32(_round(total * old[..., j] + (sums[..., j] << 16), 16))
        acc = _sat32(_sat32(_round(acc * old[..., j, None], 16)) + tile[..., j, :] * 256)
    inverse = _sat16(_round((1 << 32) // total.clamp(min=16), 8))
    return _sat16(_round(acc * inverse[..., None], 16)).to(torch.int16).reshape(t, -1, d)


def _plain_adapted(s):
    x, of_row = s["x"], torch.tensor(s["of_row"], device="cuda")
    base = _product(x, s["w"].T)                                 # 20 bits after the point
    held = of_row.clamp(min=0)
    scale = torch.tensor(s["scales"], device="cuda")[held] * (of_row >= 0)
    t = _sat32(_round(_product(s["a"][held], x[..., None]), 4))  # 16 bits after the point
    more = _product(t.transpose(1, 2), s["b"][held])[:, 0]       # 28
    base += _round(_sat32(_round(more, 12)) * scale[:, None], 12)
    return _sat16(_round(_sat32(_round(base, 4)), 8)).to(torch.int16)


def _plain_probs(s, temperatures):
    """Q0.32 probabilities [rows][vocab] as int64."""
    scores = _product(s["x"], s["head"].T)                       # 20 bits after the point
    c = torch.tensor([_inverse(t) for t in temperatures], device="cuda")
    below = (scores.amax(1, keepdim=True) - scores).clamp(max=1 << 31)
    y = (below * c[:, None]) >> 24                               # octaves, 20 bits
    high, low = s["exp2"]
    w = ((high[(y >> 10) & 1023] * low[y & 1023]) >> 30) >> (y >> 20).clamp(max=31)
    return ((w << 32) // w.sum(1, keepdim=True)).clamp(max=(1 << 32) - 1)


def _inverse(temperature):
    """log2(e) / temperature in units of 2^-24."""
    return int(math.floor(math.log2(math.e) / temperature * 16777216.0 + 0.5))


def _scaled(u, total):
    """floor(u * total / 2^32) of 32-bit u and totals up to 2^33, within 64 bits."""
    return ((u >> 16) * total + (((u & 65535) * total) >> 16)) >> 16


def _plain_verify(s):
    counts = s["counts"]
    p = _plain_probs(s, np.repeat(s["temperatures"], [c + 1 for c in counts]))
    rows, vocab = p.shape
    last = torch.tensor(_last_rows(counts), device="cuda")
    drafts = torch.zeros(rows, dtype=torch.int64, device="cuda")
    drafts[~last] = torch.tensor(s["drafts"], dtype=torch.int64, device="cuda")
    u = torch.zeros(rows, dtype=torch.int64, device="cuda")
    u[~last] = torch.tensor(s["accept_u"], dtype=torch.int64, device="cuda")
    # the drafter's probabilities: given, or all of it on the drafted token
    q = torch.zeros((rows, vocab), dtype=torch.int64, device="cuda")
    if s["q"] is not None:
        q[~last] = s["q"].long() & 0xffffffff
    else:
        q[~last] = torch.nn.functional.one_hot(drafts[~last], vocab) * ((1 << 32) - 1)
    of = drafts[:, None]
    p_draft = p.gather(1, of)[:, 0]
    # u < p / q: the draft of this row is taken
    taken = ~last & (_scaled(u, q.gather(1, of)[:, 0]) < p_draft)
    row = torch.arange(rows, device="cuda")
    request = torch.tensor(np.repeat(np.arange(len(counts)), [c + 1 for c in counts]),
                           device="cuda")
    # each request's first row whose draft is not taken: there the next token is drawn
    at = torch.full((len(counts),), rows, dtype=torch.int64, device="cuda").scatter_reduce(
        0, request, torch.where(taken, rows, row), "amin")
    first = torch.tensor(np.cumsum([0] + [c + 1 for c in counts[:-1]]), device="cuda")
    left = (p - q)[at].clamp(min=0)
    left = torch.where(left.sum(1, keepdim=True) > 0, left, p[at])
    drawn = _scaled(torch.tensor(s["sample_u"], device="cuda"), left.sum(1))
    tokens = (left.cumsum(1) <= drawn[:, None]).sum(1)
    p_row = p_draft.clone()
    p_row[last] = p[at].gather(1, tokens[:, None])[:, 0]
    return {"accepted": at - first, "tokens": tokens, "probs": p_row}


# ---------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------

def _own(s):
    case, acc = s["case"], s["acc"]
    kind = case["kind"]
    if kind == "attention":
        acc.attention_shared(0, case["prefix"], case["sequences"], s["q"].data_ptr(),
                             s["k_own"].data_ptr(), s["v_own"].data_ptr(),
                             s["lengths"].data_ptr(), case["own"], s["out"].data_ptr())
        return s["out"]
    if kind == "adapted":
        adapters = [(s["a"][j].data_ptr(), s["b"][j].data_ptr(), r, scale)
                    for j, (r, scale) in enumerate(zip(s["ranks"], s["scales"]))]
        acc.op_adapted(OPS[case["proj"]], 0, s["of_row"], adapters, s["x"].data_ptr(),
                       s["out"].data_ptr())
        return s["out"]
    if kind == "probs":
        acc.lm_head_probs(0, 0, s["temperatures"], s["out"].data_ptr())
        return s["out"]
    accepted, tokens, probs = acc.lm_head_verify(
        0, 0, s["counts"], s["drafts"], s["accept_u"], s["sample_u"], s["temperatures"],
        draft_probs=s["q"].data_ptr() if s["q"] is not None else None)
    return {"accepted": np.array(accepted, np.int64), "tokens": np.array(tokens, np.int64),
            "probs": np.array(probs, np.int64)}


def run(state):
    if own:
        return _own(state)
    kind = state["case"]["kind"]
    if kind == "attention":
        return _plain_attention(state)
    if kind == "adapted":
        return _plain_adapted(state)
    if kind == "probs":
        p = _plain_probs(state, state["temperatures"])
        return torch.where(p >= 1 << 31, p - (1 << 32), p).to(torch.int32)  # the 32 bits
    return {k: v.cpu().numpy() for k, v in _plain_verify(state).items()}


def work(case):
    """Each input read once and each output written once: K/V rows, weights and the LM head
    in the 16 bits that the framework is given them in."""
    n, kind = _dims(case), case["kind"]
    if kind == "attention":
        t, p, cap = case["sequences"], case["prefix"], case["own"]
        rows = p + t * cap / 2.0            # half of the own rows are there, on average
        return {"bytes": 2.0 * (2 * n["c"] * rows + 2 * t * n["h"]),
                "flops": 4.0 * n["h"] * t * (p + cap / 2.0)}
    if kind == "adapted":
        outs, ins = (n[x] for x in PROJECTIONS[case["proj"]])
        factors = case["rank"] * (outs + ins)
        return {"bytes": 2.0 * (outs * ins + case["adapters"] * factors +
                                case["rows"] * (outs + ins)),
                "flops": 2.0 * case["rows"] * (outs * ins + factors)}
    rows, vocab, h = case["rows"], case["vocab"], n["h"]
    size = 2.0 * h * (vocab + rows)
    if kind == "probs":
        size += 4.0 * rows * vocab
    elif case["sampled"]:
        size += 4.0 * vocab * case["requests"]  # the rows that a token is drawn in
    return {"bytes": size, "flops": 2.0 * h * vocab * rows}


# ---------------------------------------------------------------------------
# the definitions, in 64 bits on the host
# ---------------------------------------------------------------------------

def _host(t):
    return t.cpu().numpy().astype(np.int64)


def _half_up(x, bits):
    return np.floor_divide(x + 2 ** (bits - 1), 2 ** bits)


def _cut(x, bits):
    return np.clip(x, -2 ** (bits - 1), 2 ** (bits - 1) - 1)


def _matmul(a, b):
    return np.rint(a.astype(np.float64) @ b.astype(np.float64)).astype(np.int64)


def _exact_attention(case, s):
    """Row by row and tile by tile, as the recurrence is written."""
    n = _dims(case)
    d, g = n["d"], n["group"]
    q, k, v, ko, vo = (_host(s[x]) for x in ("q", "k", "v", "k_own", "v_own"))
    lengths, scale = _host(s["lengths"]), int(math.floor(256 / math.sqrt(d) + 0.5)) * 256
    table = np.array([math.floor(math.exp(x / 256) * 16384) for x in range(-2048, 1)], np.int64)
    exp14 = lambda x: table[np.clip(x, -2048, 0) + 2048]  # noqa: E731
    out = np.zeros(q.shape, np.int16)
    for t in range(case["sequences"]):
        for h in range(n["kv"]):
            rows = q[t, h * g:(h + 1) * g]
            keys = np.concatenate([k[h], ko[t, h, :lengths[t]]])
            vals = np.concatenate([v[h], vo[t, h, :lengths[t]]])
            top = np.full((g, 1), -32768)
            total, acc = np.zeros((g, 1), np.int64), np.zeros((g, d), np.int64)
            for at in range(0, len(keys), 64):
                kt, vt = (np.minimum(x[at:at + 64] * 16, 32767).clip(-32768) for x in
                          (keys, vals))
                # sum over elements of floor(x y / 16 + 1/2): x y / 16 is whole but for 32767
                term = lambda x, y: _matmul(x, np.where(y == 32767, 2048, y // 16)) + _matmul(  # noqa: E731
                    (8 - x) // 16, y == 32767)
                sc = sum(_cut(term(rows[:, b::4], kt[:, b::4].T), 32) for b in range(4))
                sc = _cut(_half_up(_cut(_half_up(_cut(sc, 32) * scale, 16), 32), 8), 16)
                new = np.maximum(top, sc.max(1, keepdims=True))
                old, p = exp14(top - new) * 4, exp14(sc - new)
                top = new
                total = _cut(_half_up(total * old + p.sum(1, keepdims=True) * 4 * 65536, 16), 32)
                val = _cut(_half_up(_cut(_half_up(_cut(term(p, vt), 32) * 1024, 16), 32), 8), 16)
                acc = _cut(_cut(_half_up(acc * old, 16), 32) + val * 256, 32)
            inv = _cut(_half_up(2 ** 32 // np.maximum(total, 16), 8), 16)
            out[t, h * g:(h + 1) * g] = _cut(_half_up(acc * inv, 16), 16)
    return out


def _exact_adapted(s):
    x, w = _host(s["x"]), _host(s["w"])
    out = _matmul(x, w.T)
    for r, j in enumerate(s["of_row"]):
        if j >= 0:
            t = _cut(_half_up(_matmul(_host(s["a"][j]), x[r]), 4), 32)
            m = _cut(_half_up(_matmul(t, _host(s["b"][j])), 12), 32)
            out[r] += _half_up(m * s["scales"][j], 12)
    return _cut(_half_up(_cut(_half_up(out, 4), 32), 8), 16).astype(np.int16)


def _exact_probs(s, temperatures):
    head, x = s["head"].cpu().numpy(), _host(s["x"])
    scores = np.concatenate([_matmul(head[a:a + 8192], x.T) for a in range(0, len(head), 8192)])
    out = []
    for r, temperature in enumerate(temperatures):
        c = math.floor(math.log2(math.e) / temperature * 2 ** 24 + 0.5)
        y = np.minimum(scores[:, r].max() - scores[:, r], 2 ** 31) * c // 2 ** 24
        part = [np.floor(np.exp2(30 - np.arange(1024) / 2.0 ** b) + 0.5).astype(np.int64)
                for b in (10, 20)]
        w = part[0][y // 1024 % 1024] * part[1][y % 1024] // 2 ** 30 // 2 ** np.minimum(
            y // 2 ** 20, 31)
        out.append(np.minimum(w * 2 ** 32 // w.sum(), 2 ** 32 - 1))
    return out


def _exact_verify(s):
    p = _exact_probs(s, np.repeat(s["temperatures"], [c + 1 for c in s["counts"]]))
    accepted, tokens, probs, row, d = [], [], [], 0, 0
    for j, count in enumerate(s["counts"]):
        q = []
        for e in range(d, d + count):
            one = np.zeros(len(p[0]), np.int64)
            one[s["drafts"][e]] = 2 ** 32 - 1
            q.append(one if s["q"] is None else _host(s["q"][e]) % 2 ** 32)
        a = 0
        while a < count:
            x = s["drafts"][d + a]
            if not s["accept_u"][d + a] * int(q[a][x]) < int(p[row + a][x]) * 2 ** 32:
                break
            a += 1
        left = np.maximum(p[row + a] - q[a], 0) if a < count else p[row + a]
        left = left if left.sum() else p[row + a]
        drawn = s["sample_u"][j] * int(left.sum()) // 2 ** 32
        token = int(np.searchsorted(left.cumsum(), drawn, side="right"))
        probs += [int(p[row + e][s["drafts"][d + e]]) for e in range(count)]
        probs.append(int(p[row + a][token]))
        accepted.append(a)
        tokens.append(token)
        row, d = row + count + 1, d + count
    return {"accepted": np.array(accepted), "tokens": np.array(tokens), "probs": np.array(probs)}


def exact(case, seed):
    s = _inputs(case, seed)
    if case["kind"] == "attention":
        return _exact_attention(case, s)
    if case["kind"] == "adapted":
        return _exact_adapted(s)
    if case["kind"] == "probs":
        p = np.stack(_exact_probs(s, s["temperatures"]))
        return p.astype(np.uint32).view(np.int32)
    return _exact_verify(s)
