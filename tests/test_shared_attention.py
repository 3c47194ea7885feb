"""Attention of a batch that shares a prefix (llm_attention_shared), bit for bit
against the oracle's attention over each sequence's concatenated positions,
and against operator 17 on a cache that holds them."""
import numpy as np
import pytest

import llm_accel
from helpers import first_mismatch
from hipmem import Hip
from oracle import orc

GUARD = 0x1234


def _accelerator(heads, kv, d, max_seq, layers=1):
    return llm_accel.Accelerator(llm_accel.Shape(64, heads * d, 64, layers, heads, kv, max_seq,
                                                 1e6))


def _normal(rng, sigma, *shape):
    return np.clip(np.round(rng.standard_normal(shape) * 256 * sigma), -32768,
                   32767).astype(np.int16)


def _full(rng, *shape):
    """The whole 16-bit range, its ends and the edges of Q4.12 among them."""
    x = rng.integers(-32768, 32768, shape)
    edges = np.array([-32768, 32767, 2047, 2048, 2049, -2047, -2048, -2049, 0])
    return np.where(rng.random(shape) < 0.2, rng.choice(edges, shape), x).astype(np.int16)


def _fill(acc, layer, k, v):
    for h in range(k.shape[0]):
        if k.shape[1]:
            acc.kv_write(layer, h, 0, k[h], v[h])


def _call(acc, hip, prefix, q, ko, vo, lengths, layer=0):
    """The entry point on fresh device buffers; what lies behind every buffer
    and the own rows themselves are as they were."""
    t, heads, d = q.shape
    cap = ko.shape[2]
    pad = lambda a: np.concatenate([a.reshape(-1), np.full(64, GUARD, np.int16)])  # noqa: E731
    dk, dv = hip.put(pad(ko)), hip.put(pad(vo))
    dout = hip.put(np.full(q.size + 64, GUARD, np.int16))
    acc.attention_shared(layer, prefix, t, hip.put(q), dk if cap else None, dv if cap else None,
                         hip.put(np.asarray(lengths, np.uint32)) if cap else None, cap, dout)
    acc.sync()
    out = hip.get(dout, q.size + 64, np.int16)
    assert (out[q.size:] == GUARD).all()
    assert np.array_equal(hip.get(dk, ko.size + 64, np.int16), pad(ko))
    assert np.array_equal(hip.get(dv, vo.size + 64, np.int16), pad(vo))
    return out[:q.size].reshape(q.shape)


def _expected(q, k, v, ko, vo, lengths, prefix):
    t, heads, d = q.shape
    kv = k.shape[0]
    g = heads // kv
    out = np.zeros_like(q)
    for s in range(t):
        n = min(int(lengths[s]), ko.shape[2])
        for h in range(kv):
            kk = np.concatenate([k[h, :prefix], ko[s, h, :n]])
            vv = np.concatenate([v[h, :prefix], vo[s, h, :n]])
            if len(kk):
                out[s, h * g:(h + 1) * g] = orc.attention(q[s, h * g:(h + 1) * g], kk, vv)
    return out


def _case(rng, heads, kv, d, seqs, cached, cap, values):
    gen = (lambda s, *sh: _normal(rng, s, *sh)) if values == "normal" else (
        lambda s, *sh: _full(rng, *sh))
    if values == "far":   # saturating keys and values among ordinary ones
        gen = lambda s, *sh: np.where(rng.random(sh) < 0.02, 3000, _normal(rng, s, *sh)).astype(  # noqa: E731,E501
            np.int16)
    q = gen(2.0, seqs, heads, d)
    k, v = gen(1.5, kv, cached, d), gen(0.5, kv, cached, d)
    ko, vo = gen(1.5, seqs, kv, cap, d), gen(0.5, seqs, kv, cap, d)
    return q, k, v, ko, vo


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv,d,seqs", [
    (2, 1, 16, 1), (4, 2, 64, 2), (14, 2, 64, 5), (10, 2, 48, 3), (16, 1, 128, 2), (3, 3, 80, 4),
    (16, 2, 128, 8), (4, 4, 96, 9), (14, 2, 128, 13), (2, 2, 32, 64), (8, 1, 112, 33)])
@pytest.mark.parametrize("prefix,cap", [
    (0, 1), (1, 0), (5, 3), (63, 2), (64, 0), (64, 65), (65, 7), (127, 130), (200, 64)])
def test_rows_are_the_oracles(heads, kv, d, seqs, prefix, cap):
    rng = np.random.default_rng([heads, kv, d, seqs, prefix, cap])
    cached = prefix + 37  # what lies behind the prefix is another's
    with _accelerator(heads, kv, d, cached) as acc, Hip() as hip:
        for values in ("normal", "far", "full"):
            q, k, v, ko, vo = _case(rng, heads, kv, d, seqs, cached, cap, values)
            _fill(acc, 0, k, v)
            lengths = rng.integers(0, cap + 1, seqs)
            lengths[0] = cap
            lengths[-1] = min(lengths[-1], 1) if seqs > 1 else lengths[-1]
            got = _call(acc, hip, prefix, q, ko, vo, lengths)
            want = _expected(q, k, v, ko, vo, lengths, prefix)
            assert np.array_equal(got, want), (values, first_mismatch(got, want))


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv,d,seqs,prefix,cap", [
    (16, 2, 128, 8, 1500, 200), (14, 2, 64, 20, 2500, 100), (4, 1, 128, 3, 20000, 70),
    (8, 2, 128, 64, 640, 30), (6, 2, 48, 2, 70, 1500)])
def test_long_contexts(heads, kv, d, seqs, prefix, cap):
    rng = np.random.default_rng([7, heads, d, seqs, prefix])
    q, k, v, ko, vo = _case(rng, heads, kv, d, seqs, prefix, cap, "normal")
    lengths = rng.integers(0, cap + 1, seqs)
    lengths[0] = cap
    with _accelerator(heads, kv, d, prefix) as acc, Hip() as hip:
        _fill(acc, 0, k, v)
        got = _call(acc, hip, prefix, q, ko, vo, lengths)
        want = _expected(q, k, v, ko, vo, lengths, prefix)
        assert np.array_equal(got, want), first_mismatch(got, want)
        assert (got != 0).mean() > 0.5


@pytest.mark.gpu
def test_banks_that_reach_their_limit():
    """d = 128: 32 products of -32768 and -2048 in a bank are 2^31, one past
    what it holds; in all four banks, in one, and in rows beside ordinary
    ones, over prefix tiles and own ones."""
    heads, kv, d, seqs, prefix, cap = 4, 1, 128, 5, 150, 20
    rng = np.random.default_rng(11)
    q, k, v, ko, vo = _case(rng, heads, kv, d, seqs, prefix, cap, "normal")
    q[0], q[2, 1] = -32768, -32768
    q[3, :, 1::4] = -32768
    q[4, 2, 3::4] = -32768
    for x in (k, ko):
        x[..., 3, :] = -2048
        x[..., 9, :] = -32768
        x[..., 11, 1::4] = -2048
    k[0, 140] = -2500
    with _accelerator(heads, kv, d, prefix) as acc, Hip() as hip:
        _fill(acc, 0, k, v)
        lengths = [20, 4, 10, 20, 12]
        got = _call(acc, hip, prefix, q, ko, vo, lengths)
        want = _expected(q, k, v, ko, vo, lengths, prefix)
        assert np.array_equal(got, want), first_mismatch(got, want)


@pytest.mark.gpu
def test_largest_values_and_sums():
    """Probabilities of one in every position, V at both ends."""
    heads, kv, d, seqs, prefix, cap = 4, 2, 64, 3, 700, 40
    q = np.zeros((seqs, heads, d), np.int16)
    rng = np.random.default_rng(12)
    for fill in (-32768, 32767, -2048, 2048):
        k = _normal(rng, 1, kv, prefix, d)
        ko = _normal(rng, 1, seqs, kv, cap, d)
        v, vo = np.full_like(k, fill), np.full_like(ko, fill)
        with _accelerator(heads, kv, d, prefix) as acc, Hip() as hip:
            _fill(acc, 0, k, v)
            got = _call(acc, hip, prefix, q, ko, vo, [40, 0, 7])
            assert np.array_equal(got, _expected(q, k, v, ko, vo, [40, 0, 7], prefix))


@pytest.mark.gpu
def test_sequences_without_positions_and_lengths_past_the_rows():
    heads, kv, d, seqs, cap = 4, 2, 64, 6, 70
    rng = np.random.default_rng(13)
    q, k, v, ko, vo = _case(rng, heads, kv, d, seqs, 10, cap, "normal")
    lengths = np.array([0, 70, 71, 0xffffffff, 0, 64], np.uint32)
    with _accelerator(heads, kv, d, 10) as acc, Hip() as hip:
        got = _call(acc, hip, 0, q, ko, vo, lengths)
        want = _expected(q, k, v, ko, vo, lengths, 0)
        assert np.array_equal(got, want)
        assert (got[0] == 0).all() and (got[4] == 0).all() and (got[1] != 0).any()
        # no rows anywhere
        got = _call(acc, hip, 0, q, ko[:, :, :0], vo[:, :, :0], [0] * seqs)
        assert (got == 0).all()


@pytest.mark.gpu
def test_rows_are_operator_17s():
    """The same positions in one cache, read by the prefill attention block;
    another layer's cache, and results in the queries' place."""
    heads, kv, d, prefix, cap = 16, 2, 128, 333, 90
    rng = np.random.default_rng(14)
    q, k, v, ko, vo = _case(rng, heads, kv, d, 3, prefix, cap, "normal")
    lengths = [90, 1, 51]
    with _accelerator(heads, kv, d, prefix + cap, layers=2) as acc, Hip() as hip:
        _fill(acc, 1, k, v)
        dq = hip.put(q)
        args = (hip.put(ko), hip.put(vo), hip.put(np.array(lengths, np.uint32)), cap)
        acc.attention_shared(1, prefix, 3, dq, *args, dq)
        acc.sync()
        got = hip.get(dq, q.shape, np.int16)
        for s, n in enumerate(lengths):
            for h in range(kv):
                acc.kv_write(1, h, prefix, ko[s, h, :n], vo[s, h, :n])
            block = q[s].reshape(kv, 1, heads // kv, d)
            want, _ = acc.run_prefill_attention_block(block, prefix + n - 1, 1, layer=1)
            assert np.array_equal(got[s].reshape(want.shape), want), s


@pytest.mark.gpu
def test_captured_and_replayed_with_growing_sequences():
    """Lengths are read when the work runs: a graph captured once serves a
    decode loop.  Larger eager calls between replays grow the context's
    scratch, the graph keeps its own."""
    heads, kv, d, seqs, prefix, cap = 8, 2, 64, 4, 130, 100
    rng = np.random.default_rng(15)
    q, k, v, ko, vo = _case(rng, heads, kv, d, seqs, 1000, cap, "normal")
    with _accelerator(heads, kv, d, 1000) as acc, Hip() as hip:
        _fill(acc, 0, k, v)
        dq, dk, dv, dn = (hip.put(x) for x in (q, ko, vo, np.zeros(seqs, np.uint32)))
        dout = hip.alloc(q.nbytes)
        call = lambda: acc.attention_shared(0, prefix, seqs, dq, dk, dv, dn, cap, dout)  # noqa: E731
        call()
        acc.sync()
        stream = llm_accel.lib().llm_stream(acc._ctx)
        graph = hip.capture(stream, call)
        for step, lengths in enumerate(([1, 2, 3, 4], [0, 0, 0, 0], [100, 1, 62, 63],
                                        [64, 65, 99, 0])):
            hip.put(np.array(lengths, np.uint32), to=dn)
            q = _normal(rng, 2.0, seqs, heads, d)
            hip.put(q, to=dq)
            hip.put(np.zeros_like(q), to=dout)
            hip.replay(graph, stream)
            acc.sync()
            got = hip.get(dout, q.shape, np.int16)
            assert np.array_equal(got, _expected(q, k, v, ko, vo, lengths, prefix)), step
            more = prefix + 250 * (step + 1) if step < 3 else 0
            got = _call(acc, hip, more, q, ko, vo, lengths)
            assert np.array_equal(got, _expected(q, k, v, ko, vo, lengths, more)), step


def test_refusals_without_a_context():
    lib = llm_accel.lib()
    p = 1 << 20
    assert lib.llm_attention_shared(None, 0, 0, 1, p, p, p, p, 1, p) == -1


@pytest.mark.gpu
def test_refusals():
    with _accelerator(4, 2, 64, 100) as acc, Hip() as hip:
        p = hip.alloc(1 << 20)
        good = (0, 64, 2, p, p, p, p, 8, p)
        for at, bad in ((0, 1), (1, 101), (1, 0xffffffff), (2, 0), (2, 65), (3, None), (3, p + 8),
                        (4, None), (4, p + 2), (5, None), (5, p + 8), (6, None), (6, p + 2),
                        (7, (1 << 20) + 1), (7, 0xffffffff), (8, None), (8, p + 4)):
            args = list(good)
            args[at] = bad
            with pytest.raises(llm_accel.AccelError):
                acc.attention_shared(*args)
        hip.put(np.zeros(1 << 18, np.uint32), to=p)
        acc.attention_shared(*good)
        acc.attention_shared(0, 100, 2, p, None, None, None, 0, p)
        acc.sync()


@pytest.mark.gpu
def test_refuses_more_tiles_than_a_launch_counts():
    """16 KV heads, 64 sequences of up to 2^20 positions: 2^24 tiles.  The
    buffers are never reached; 63 sequences of 2^14 positions are fine."""
    with _accelerator(16, 16, 16, 64) as acc, Hip() as hip:
        p = hip.alloc(1 << 20)
        with pytest.raises(llm_accel.AccelError, match="tiles"):
            acc.attention_shared(0, 0, 64, p, p, p, p, 1 << 20, p)
        hip.put(np.zeros(64, np.uint32), to=p)  # no sequence has a position
        out = hip.put(np.full(63 * 16 * 16, 5, np.int16))
        acc.attention_shared(0, 0, 63, out, p, p, p, 1 << 14, out)
        acc.sync()
        assert not hip.get(out, 63 * 16 * 16, np.int16).any()


@pytest.mark.gpu
def test_nothing_to_attend_to():
    """No prefix and no own rows at all: zeros, and nothing behind them."""
    with _accelerator(6, 3, 48, 64) as acc, Hip() as hip:
        rng = np.random.default_rng(3)
        q = _full(rng, 5, 6, 48)
        none = np.zeros((5, 3, 0, 48), np.int16)
        assert not _call(acc, hip, 0, q, none, none, [0] * 5).any()


@pytest.mark.gpu
def test_two_contexts_and_calls_of_changing_sizes():
    """Calls of two contexts in turn, none waited for, larger and smaller ones
    over the same scratch: each finds its own."""
    rng = np.random.default_rng(21)
    heads, kv, d, cached = 14, 2, 64, 1400
    sizes = [(1400, 9, 200), (130, 3, 5), (700, 20, 90), (0, 2, 700), (1400, 1, 0), (64, 33, 257)]
    with _accelerator(heads, kv, d, cached) as a0, _accelerator(heads, kv, d, cached) as a1, \
            Hip() as hip:
        accs, caches, calls = (a0, a1), [], []
        for acc in accs:
            k, v = _normal(rng, 1.5, kv, cached, d), _normal(rng, 0.5, kv, cached, d)
            _fill(acc, 0, k, v)
            caches.append((k, v))
        for prefix, seqs, cap in sizes:
            for i in (0, 1):
                q, ko, vo = (_normal(rng, s, *sh) for s, sh in (
                    (2.0, (seqs, heads, d)), (1.5, (seqs, kv, cap, d)), (0.5, (seqs, kv, cap, d))))
                lengths = rng.integers(0, cap + 1, seqs).astype(np.uint32)
                calls.append((i, prefix, q, ko, vo, lengths, hip.put(q), hip.put(ko), hip.put(vo),
                              hip.put(lengths), hip.alloc(q.nbytes)))
        for _ in range(2):
            for i, prefix, q, ko, vo, lengths, dq, dk, dv, dl, out in calls:
                accs[i].attention_shared(0, prefix, len(q), dq, dk, dv, dl, ko.shape[2], out)
        a0.sync(), a1.sync()
        for i, prefix, q, ko, vo, lengths, *_, out in calls:
            want = _expected(q, *caches[i], ko, vo, lengths, prefix)
            got = hip.get(out, q.shape, np.int16)
            assert np.array_equal(got, want), (i, prefix, first_mismatch(got, want))
