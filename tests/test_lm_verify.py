"""Next-token probabilities and draft verification (llm_lm_head_probs,
llm_lm_head_verify) against the definitions in Python integers and 64-bit
floating point."""
import ctypes
import math

import numpy as np
import pytest

import llm_accel
from hipmem import Hip

FULL = (1 << 32) - 1
# hidden, intermediate, heads, KV heads: one and several k-steps, one that is
# no multiple of 128, and one past the matrix-core scores' width
SHAPES = {128: (128, 64, 2, 1), 256: (256, 688, 4, 2), 480: (480, 1300, 10, 2),
          4096: (4096, 512, 32, 2)}


def _accelerator(hidden, vocab):
    h, i, heads, kv = SHAPES[hidden]
    return llm_accel.Accelerator(llm_accel.Shape(vocab, h, i, 1, heads, kv, 64, 1e6))


# --- the definitions ------------------------------------------------------

def _scores(rows, table):
    # |sums| <= 2^30 hidden < 2^53: exact
    return (rows.astype(np.float64) @ table.astype(np.float64).T).astype(np.int64)


_E = [[math.floor(2 ** (30 - i / 2 ** b) + 0.5) for i in range(1024)] for b in (10, 20)]


def _probs_row(scores, temperature):
    """Q0.32 of one row, in Python integers per distinct score."""
    c = math.floor(math.log2(math.e) / temperature * 2 ** 24 + 0.5)
    top = int(scores.max())
    below, back = np.unique(top - scores, return_inverse=True)
    w = []
    for d in below.tolist():
        y = min(d, 1 << 31) * c >> 24
        w.append((_E[0][y >> 10 & 1023] * _E[1][y & 1023] >> 30) >> min(y >> 20, 99))
    z = sum(int(x) * int(n) for x, n in zip(w, np.bincount(back.reshape(-1))))
    return np.array([min((x << 32) // z, FULL) for x in w], np.uint64)[back.reshape(-1)]


def _verify(p, counts, drafts, accept_u, sample_u, q):
    """accepted, tokens, probs from the rows' probabilities."""
    accepted, tokens, probs, row, d = [], [], [], 0, 0
    for j, count in enumerate(counts):
        def drafter(i):
            if q is not None:
                return [int(x) for x in q[d + i]]
            return [FULL if v == drafts[d + i] else 0 for v in range(p.shape[1])]
        a = 0
        while a < count:
            x = drafts[d + a]
            if not accept_u[d + a] * drafter(a)[x] < int(p[row + a][x]) << 32:
                break
            a += 1
        left = [int(x) for x in p[row + a]]
        if a < count:
            above = [max(x - y, 0) for x, y in zip(left, drafter(a))]
            left = above if sum(above) else left
        t, token = sample_u[j] * sum(left) >> 32, 0
        while t >= left[token]:
            t -= left[token]
            token += 1
        accepted.append(a)
        tokens.append(token)
        probs += [int(p[row + i][drafts[d + i]]) for i in range(count)] + [int(p[row + a][token])]
        row, d = row + count + 1, d + count
    return accepted, tokens, probs


def _table(rng, vocab, hidden, limit=600):
    return rng.integers(-limit, limit + 1, (vocab, hidden)).astype(np.int16)


def _rows(rng, n, hidden, sigma=1.5):
    return np.clip(np.round(rng.standard_normal((n, hidden)) * 256 * sigma), -32768,
                   32767).astype(np.int16)


# --- probabilities --------------------------------------------------------

def _device_probs(acc, hip, rows, temperatures, vocab, row0=0, pair=0):
    out = hip.put(np.full((len(temperatures) + 1, vocab), 0xabcdef01, np.uint32))
    acc.upload(pair, rows)
    acc.lm_head_probs(pair, row0, temperatures, out)
    acc.sync()
    got = hip.get(out, (len(temperatures) + 1, vocab), np.uint32)
    assert (got[-1] == 0xabcdef01).all()  # what lies behind the rows
    return got[:-1]


@pytest.mark.gpu
@pytest.mark.parametrize("hidden,vocab,rows", [
    (128, 1, 1), (128, 2, 3), (256, 15, 2), (256, 2048, 1), (256, 2049, 8), (480, 4099, 5),
    (256, 33000, 8), (480, 33001, 3), (128, 70001, 2), (4096, 1030, 1), (4096, 1030, 2),
    (4096, 1030, 4), (4096, 1030, 8)])
def test_probabilities_are_the_definition(hidden, vocab, rows):
    rng = np.random.default_rng([1, hidden, vocab, rows])
    table, x = _table(rng, vocab, hidden), _rows(rng, rows, hidden)
    temperatures = [float(t) for t in rng.choice([1 / 64, 0.3, 0.7, 1.0, 1.7, 64.0], rows)]
    with _accelerator(hidden, vocab) as acc, Hip() as hip:
        acc.load_lm_head(table)
        got = _device_probs(acc, hip, x, temperatures, vocab)
        scores = _scores(x, table)
        for r in range(rows):
            assert np.array_equal(got[r], _probs_row(scores[r], temperatures[r])), r
        # the argmax's keys are as an argmax expects them
        toks, best = acc.lm_head_argmax(0, 0, rows)
        assert toks == scores.argmax(1).tolist() and best == scores.max(1).tolist()


@pytest.mark.gpu
def test_probabilities_near_the_softmax():
    """Against the softmax in 64 bits.  y is short of its value by less than
    2^-20 (its floor) and off by at most y / (2 c) for the rounding of c, at
    most 31 octaves / 2^24.5 here; a table entry is off by 2^-30 of its value
    and the two floors take less than 2 2^-30 of the largest weight.  So a
    weight is w (1 + e) - d with |e| < ln 2 (2^-20 + 2^-20.5) + 2^-28 <
    2^-19.7 and 0 <= d < 2^-29; the sum, at least the largest weight, is off
    by e and V d; the quotient's floor takes 2^-32."""
    rng = np.random.default_rng(2)
    vocab, hidden = 5003, 256
    table, x = _table(rng, vocab, hidden), _rows(rng, 4, hidden, 3.0)
    temperatures = [0.5, 0.8, 1.0, 1.3]
    with _accelerator(hidden, vocab) as acc, Hip() as hip:
        acc.load_lm_head(table)
        got = _device_probs(acc, hip, x, temperatures, vocab) / 2.0 ** 32
    z = _scores(x, table) / 2.0 ** 20 / np.array(temperatures)[:, None]
    p = np.exp(z - z.max(1, keepdims=True))
    p /= p.sum(1, keepdims=True)
    e, d = 2 ** -19.7, 2.0 ** -29
    assert (abs(got - p) <= p * (2 * e + vocab * d) + d + 2.0 ** -32).all()


@pytest.mark.gpu
def test_probabilities_of_extreme_rows():
    """Scores as far apart as they come, all scores equal, one score above the
    rest, and rows of a pair from row0 on."""
    vocab, hidden = 3000, 256
    rng = np.random.default_rng(3)
    table = _table(rng, vocab, hidden)
    table[70] = table[2990] = -32768
    table[5] = 32767
    x = np.zeros((8, hidden), np.int16)
    x[0], x[1] = -32768, 32767
    x[3, 0], x[4] = 1, _rows(rng, 1, hidden)[0]
    temperatures = [64.0, 1 / 64, 1.0, 1.0, 0.9]
    with _accelerator(hidden, vocab) as acc, Hip() as hip:
        acc.load_lm_head(table)
        got = _device_probs(acc, hip, x, temperatures, vocab)
        scores = _scores(x, table)
        for r, t in enumerate(temperatures):
            assert np.array_equal(got[r], _probs_row(scores[r], t)), r
        assert (got[2] == (1 << 32) // vocab).all()  # a row of zeros
        got = _device_probs(acc, hip, x, temperatures[3:], vocab, row0=3, pair=1)
        for r, t in enumerate(temperatures[3:]):
            assert np.array_equal(got[r], _probs_row(scores[3 + r], t)), r


@pytest.mark.gpu
def test_probabilities_captured_and_replayed():
    vocab, hidden = 4100, 256
    rng = np.random.default_rng(4)
    tables = [_table(rng, vocab, hidden) for _ in range(1)]
    with _accelerator(hidden, vocab) as acc, Hip() as hip:
        acc.load_lm_head(tables[0])
        x = _rows(rng, 3, hidden)
        temperatures = [0.7, 1.0, 1.2]
        acc.upload(0, x)
        out = hip.put(np.zeros((3, vocab), np.uint32))
        acc.lm_head_probs(0, 0, temperatures, out)  # allocates
        acc.sync()
        stream = llm_accel.lib().llm_stream(acc._ctx)
        graph = hip.capture(stream, lambda: acc.lm_head_probs(0, 0, temperatures, out))
        for _ in range(4):
            x = _rows(rng, 3, hidden)
            acc.upload(0, x)
            hip.put(np.zeros((3, vocab), np.uint32), to=out)
            hip.replay(graph, stream)
            acc.sync()
            scores = _scores(x, tables[0])
            got = hip.get(out, (3, vocab), np.uint32)
            for r, t in enumerate(temperatures):
                assert np.array_equal(got[r], _probs_row(scores[r], t))
            # an eager verification between the replays
            a = acc.lm_head_verify(0, 0, [2], [1, 2], [0, 0], [1 << 31], [1.0])
            p = np.stack([_probs_row(s, 1.0) for s in scores])
            assert a == _verify(p, [2], [1, 2], [0, 0], [1 << 31], None)


# --- verification ---------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("hidden,vocab,counts", [
    (128, 1, [0]), (128, 3, [2]), (256, 15, [0, 0, 0]), (256, 2048, [7]), (256, 2049, [3, 0, 2]),
    (480, 4099, [0] * 8), (480, 6001, [1, 1, 1, 1]), (256, 33000, [4]), (4096, 1030, [2, 1])])
@pytest.mark.parametrize("sampled", [False, True])
def test_verification_is_the_definition(hidden, vocab, counts, sampled):
    rng = np.random.default_rng([5, hidden, vocab, len(counts), sampled])
    table = _table(rng, vocab, hidden)
    n, nd = sum(counts) + len(counts), sum(counts)
    drafting = [r for r, last in enumerate(i == c for c in counts for i in range(c + 1))
                if not last]
    with _accelerator(hidden, vocab) as acc, Hip() as hip:
        acc.load_lm_head(table)
        for trial in range(6):
            x = _rows(rng, n, hidden, 0.7)
            temperatures = [float(t) for t in rng.uniform(0.4, 2.0, len(counts))]
            scores = _scores(x, table)
            p = np.stack([_probs_row(scores[r], t) for r, t in enumerate(
                np.repeat(temperatures, [c + 1 for c in counts]))])
            # likely drafts, the drafter's distribution near the target's
            drafts = [int(rng.choice(np.argsort(p[r])[-3:])) for r in drafting]
            q = None
            if sampled:
                q = np.minimum(p[drafting] * rng.uniform(0.3, 1.5, (nd, vocab)), FULL).astype(
                    np.uint32)
            accept_u = [int(u) for u in rng.integers(0, 1 << 32, nd)]
            sample_u = [int(u) for u in rng.integers(0, 1 << 32, len(counts))]
            if trial == 4:
                accept_u, sample_u = [0] * nd, [0] * len(counts)
            if trial == 5:
                accept_u, sample_u = [FULL] * nd, [FULL] * len(counts)
            acc.upload(0, x)
            got = acc.lm_head_verify(0, 0, counts, drafts, accept_u, sample_u, temperatures,
                                     hip.put(q) if sampled and nd else None)
            assert got == _verify(p, counts, drafts, accept_u, sample_u, q), trial
        toks, _ = acc.lm_head_argmax(0, 0, n)
        assert toks == scores.argmax(1).tolist()


@pytest.mark.gpu
def test_verification_where_distributions_meet():
    """Q equal to P (nothing above it: the draw falls back to P), Q above P
    everywhere but at one token, Q and P both 0 at the draft, the same draft
    twice, and Q the whole mass on another token."""
    vocab, hidden = 2500, 256
    rng = np.random.default_rng(6)
    table, x = _table(rng, vocab, hidden), _rows(rng, 5, hidden, 2.0)
    scores = _scores(x, table)
    t = 0.5  # some tokens weigh nothing
    p = np.stack([_probs_row(s, t) for s in scores])
    least = int(p[0].argmin())
    assert p[0][least] == 0
    best = int(p[0].argmax())
    equal = p[:4].astype(np.uint32)
    above = np.full((4, vocab), FULL, np.uint32)
    above[:, 7] = 0
    other = np.zeros((4, vocab), np.uint32)
    other[:, least] = FULL
    with _accelerator(hidden, vocab) as acc, Hip() as hip:
        acc.load_lm_head(table)
        acc.upload(0, x)
        for q in (equal, above, other):
            for first in (least, best, 7):
                for u in (0, 1, 1 << 31, FULL):
                    args = ([4], [first, first, best, 0], [u] * 4, [u])
                    got = acc.lm_head_verify(0, 0, *args, [t], hip.put(q))
                    assert got == _verify(p, *args, q), (first, u)


@pytest.mark.gpu
def test_verified_tokens_follow_the_target():
    """Over all pairs of an even grid of random numbers the token after a draft
    sampled from Q is distributed as P.  The draft's choice is exact here (each
    x weighed by Q_x), the grids of n points put every probability off by at
    most 1 / n each: |difference| <= 2 / n per token."""
    vocab, hidden, n = 5, 128, 24
    rng = np.random.default_rng(8)
    table, x = _table(rng, vocab, hidden), _rows(rng, 2, hidden, 0.3)
    scores = _scores(x, table)
    p = _probs_row(scores[0], 1.0) / 2.0 ** 32
    q = rng.dirichlet(np.ones(vocab))
    grid = [int((i + 0.5) / n * 2 ** 32) for i in range(n)]
    seen = np.zeros(vocab)
    with _accelerator(hidden, vocab) as acc, Hip() as hip:
        acc.load_lm_head(table)
        acc.upload(0, x)
        dq = hip.put(np.floor(q * 2 ** 32).astype(np.uint32))
        for draft in range(vocab):
            for u in grid:
                for v in grid:
                    accepted, token, _ = acc.lm_head_verify(0, 0, [1], [draft], [u], [v], [1.0],
                                                            dq)
                    seen[draft if accepted[0] else token[0]] += q[draft] / n ** 2
    assert (abs(seen - p) <= 2.0 / n).all()


@pytest.mark.gpu
def test_a_larger_head_and_a_smaller_one():
    """The scores' memory grows with the vocabulary and serves smaller ones."""
    hidden = 256
    rng = np.random.default_rng(9)
    x = _rows(rng, 2, hidden)
    with _accelerator(hidden, 5000) as acc, Hip() as hip:
        for vocab in (700, 5000, 700):
            table = _table(rng, vocab, hidden)
            acc.load_lm_head(table)
            got = _device_probs(acc, hip, x, [1.0, 0.5], vocab)
            s = _scores(x, table)
            assert np.array_equal(got[0], _probs_row(s[0], 1.0))
            assert np.array_equal(got[1], _probs_row(s[1], 0.5))
            args = ([1], [3], [1 << 30], [1 << 31])
            p = np.stack([_probs_row(r, 1.0) for r in s])
            assert acc.lm_head_verify(0, 0, *args, [1.0]) == _verify(p, *args, None)


# --- refusals --------------------------------------------------------------

def test_every_export_has_its_argument_types():
    lib = llm_accel.lib()
    for name in llm_accel.EXPORTS:
        assert getattr(lib, name).argtypes is not None, name


def test_refusals_without_a_context():
    lib = llm_accel.lib()
    one = (ctypes.c_uint32 * 1)(0)
    t = (ctypes.c_double * 1)(1.0)
    assert lib.llm_lm_head_probs(None, 0, 0, 1, t, 1 << 20) == -1
    assert lib.llm_lm_head_verify(None, 0, 0, 1, one, one, one, one, t, None, one, one, one) == -1


def test_mismatched_requests_are_refused_on_the_host():
    acc = object.__new__(llm_accel.Accelerator)
    acc._ctx = ctypes.c_void_p()
    for args in (([1], [], [], [0], [1.0]), ([0], [1], [1], [0], [1.0]),
                 ([1], [1], [], [0], [1.0]), ([0, 0], [], [], [0], [1.0, 1.0]),
                 ([0], [], [], [0], [])):
        with pytest.raises(llm_accel.AccelError):
            acc.lm_head_verify(0, 0, *args)


@pytest.mark.gpu
def test_refusals_of_a_context():
    vocab, hidden = 100, 128
    with _accelerator(hidden, vocab) as acc, Hip() as hip:
        out = hip.alloc(8 * vocab * 4)
        with pytest.raises(llm_accel.AccelError, match="not loaded"):
            acc.lm_head_probs(0, 0, [1.0], out)
        with pytest.raises(llm_accel.AccelError, match="not loaded"):
            acc.lm_head_verify(0, 0, [0], [], [], [0], [1.0])
        acc.load_lm_head(_table(np.random.default_rng(0), vocab, hidden))
        for args in ((4, 0, [1.0], out), (0, 8, [1.0], out), (0, 0xffffffff, [1.0] * 2, out),
                     (0, 1, [1.0] * 8, out), (0, 0, [], out), (0, 0, [1.0] * 9, out),
                     (0, 0, [1.0], None), (0, 0, [1.0], out + 2), (0, 0, [0.0], out),
                     (0, 0, [float("nan")], out), (0, 0, [-1.0], out), (0, 0, [65.0], out)):
            with pytest.raises(llm_accel.AccelError):
                acc.lm_head_probs(*args)
        for args in ((4, 0, [0], [], [], [0], [1.0]), (0, 8, [0], [], [], [0], [1.0]),
                     (0, 0, [8], [0] * 8, [0] * 8, [0], [1.0]),
                     (0, 1, [7], [0] * 7, [0] * 7, [0], [1.0]),
                     (0, 0, [3, 4], [0] * 7, [0] * 7, [0] * 2, [1.0] * 2),
                     (0, 0, [0] * 9, [], [], [0] * 9, [1.0] * 9), (0, 0, [], [], [], [], []),
                     (0, 0, [1], [vocab], [0], [0], [1.0]),
                     (0, 0, [0, 0], [], [], [0, 0], [1.0, float("inf")])):
            with pytest.raises(llm_accel.AccelError):
                acc.lm_head_verify(*args)
        with pytest.raises(llm_accel.AccelError):
            acc.lm_head_verify(0, 0, [1], [1], [0], [0], [1.0], out + 1)


@pytest.mark.gpu
@pytest.mark.parametrize("hidden,heads,vocab,rows", [
    (2048, 16, 40001, 8), (2048, 16, 40001, 3), (2816, 22, 9000, 5), (2944, 23, 32770, 8),
    (3840, 30, 33003, 3), (3968, 31, 2050, 8)])
def test_probabilities_of_wide_heads(hidden, heads, vocab, rows):
    """Every way that the scores are computed in: groups shared with four steps
    ahead, a group per wavefront, and no matrix cores."""
    rng = np.random.default_rng([9, hidden, vocab, rows])
    table, x = _table(rng, vocab, hidden), _rows(rng, rows, hidden)
    table[vocab // 3], x[rows - 1] = -32768, -32768
    temperatures = [float(t) for t in rng.choice([0.7, 20.0, 64.0], rows)]
    with llm_accel.Accelerator(llm_accel.Shape(vocab, hidden, 128, 1, heads, heads, 64,
                                               1e6)) as acc, Hip() as hip:
        acc.load_lm_head(table)
        got = _device_probs(acc, hip, x, temperatures, vocab)
        scores = _scores(x, table)
        for r in range(rows):
            assert np.array_equal(got[r], _probs_row(scores[r], temperatures[r])), r
        toks, best = acc.lm_head_argmax(0, 0, rows)
        assert toks == scores.argmax(1).tolist() and best == scores.max(1).tolist()
