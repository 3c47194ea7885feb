"""Projections with low-rank adapters (llm_op_adapted) against the definition
in 64-bit whole numbers."""
import ctypes

import numpy as np
import pytest

import llm_accel
import workloads
from helpers import accel_shape
from hipmem import Hip

ODD = workloads.ShapeSpec("odd", 512, 480, 1300, 1, 10, 2, 64, 0.25, 0.5)
MID = workloads.ShapeSpec("mid", 512, 896, 4864, 1, 14, 2, 64, 0.125, 0.5)
SPECS = {"A": workloads.CONFIG_A, "odd": ODD, "mid": MID}


def _half_up(x, bits):
    return (x + (1 << (bits - 1))) >> bits


def _cut(x, bits):
    return np.clip(x, -(1 << (bits - 1)), (1 << (bits - 1)) - 1)


def _matmul(a, b):
    """Exact: the factors in 16-bit halves where products pass 2^53."""
    a, b = np.asarray(a, np.int64), np.asarray(b, np.int64)
    hi, lo = a >> 16, a & 0xffff
    f = lambda x, y: (x.astype(np.float64) @ y.astype(np.float64)).astype(np.int64)  # noqa: E731
    return (f(hi, b) << 16) + f(lo, b)


def _expected(x, w, adapters, row_adapter):
    out = _matmul(x, w.T)
    for r, j in enumerate(row_adapter):
        if j >= 0:
            a, b, scale = adapters[j]
            t = _cut(_half_up(_matmul(x[r:r + 1], a.T), 4), 32)
            m = _cut(_half_up(_matmul(t, b), 12), 32)
            out[r] += _half_up(m[0] * scale, 12)
    return _cut(_half_up(_cut(_half_up(out, 4), 32), 8), 16).astype(np.int16)


def _adapter(rng, rank, ins, outs, limit=400, scale=None):
    return (rng.integers(-limit, limit + 1, (rank, ins)).astype(np.int16),
            rng.integers(-limit, limit + 1, (rank, outs)).astype(np.int16),
            int(rng.integers(-1 << 18, 1 << 18)) if scale is None else scale)


def _run(acc, hip, op, x, adapters, row_adapter, outs, in_place=False):
    dev = [(hip.put(a), hip.put(b), a.shape[0], s) for a, b, s in adapters]
    n = len(x) * outs
    pad = max(n, x.size) + 64
    buf = np.full(pad, 0x5a5a, np.int16)
    dout = hip.put(buf)
    if in_place:
        buf[:x.size] = x.reshape(-1)
        hip.put(buf, to=dout)
    st = acc.op_adapted(op, 0, row_adapter, dev, dout if in_place else hip.put(x), dout)
    acc.sync()
    assert st.code == 0 and st.op == op and st.token_count == len(x)
    got = hip.get(dout, pad, np.int16)
    assert (got[max(n, x.size if in_place else 0):] == 0x5a5a).all()
    return got[:n].reshape(len(x), outs)


def _model(spec, wide=0, seed=1):
    synth = workloads.SyntheticModel(spec, seed=seed, layers=1)
    rng = np.random.default_rng(seed)
    for w in synth._w[0]:
        if wide == 1:      # a few weights outside 12 bits: corrections
            w[rng.integers(0, w.shape[0], 40), rng.integers(0, w.shape[1], 40)] = 4000
        elif wide == 2:    # many: 16-bit copies
            w[rng.random(w.shape) < 0.02] *= 9
    return synth


ROWS = {1: [0], 2: [1, -1], 3: [0, 0, 0], 5: [2, -1, 0, 2, 1], 8: [3, 1, 1, 1, -1, 1, 1, 0]}


@pytest.mark.gpu
@pytest.mark.parametrize("shape,wide", [("A", 0), ("odd", 0), ("mid", 0), ("A", 1), ("odd", 2)])
def test_every_projection_and_row_count(shape, wide):
    spec = SPECS[shape]
    synth = _model(spec, wide)
    rng = np.random.default_rng(2)
    with llm_accel.Accelerator(accel_shape(spec, layers=1)) as acc, Hip() as hip:
        acc.load_model(synth)
        for op in range(1, 8):
            w = synth.weight(0, op - 1)
            outs, ins = w.shape
            adapters = [_adapter(rng, rank, ins, outs) for rank in (1, 13, 16, 64)]
            for rows, of_row in ROWS.items():
                x = rng.integers(-2000, 2001, (rows, ins)).astype(np.int16)
                got = _run(acc, hip, op, x, adapters, of_row, outs)
                assert np.array_equal(got, _expected(x, w, adapters, of_row)), (op, rows)
                plain = acc.run_feature(op, x)
                for r, j in enumerate(of_row):
                    if j < 0:
                        assert np.array_equal(got[r], plain[r])


@pytest.mark.gpu
def test_every_row_its_own_adapter_and_all_the_same():
    spec = MID
    synth = _model(spec)
    rng = np.random.default_rng(3)
    with llm_accel.Accelerator(accel_shape(spec, layers=1)) as acc, Hip() as hip:
        acc.load_model(synth)
        for op in (2, 5, 7):
            w = synth.weight(0, op - 1)
            outs, ins = w.shape
            adapters = [_adapter(rng, int(r), ins, outs) for r in rng.integers(1, 65, 8)]
            adapters.append(_adapter(rng, 512, ins, outs, 60))
            x = rng.integers(-1500, 1501, (8, ins)).astype(np.int16)
            for of_row in (list(range(8)), list(range(7, -1, -1)), [8] * 8, [-1] * 8,
                           [8, 0, 8, 1, 8, 2, 8, 3]):
                got = _run(acc, hip, op, x, adapters, of_row, outs)
                assert np.array_equal(got, _expected(x, w, adapters, of_row)), (op, of_row)


@pytest.mark.gpu
def test_saturated_values():
    """x A^T past 32 bits, t B past 32 bits, results past 16, the ends of the
    scale, and operands whose products are the largest."""
    spec = SPECS["A"]
    synth = _model(spec)
    h, i = spec.hidden, spec.inter
    lo, hi = -32768, 32767
    full = lambda v, *s: np.full(s, v, np.int16)  # noqa: E731
    with llm_accel.Accelerator(accel_shape(spec, layers=1)) as acc, Hip() as hip:
        acc.load_model(synth)
        for op, ins, outs in ((1, h, h), (7, i, h)):
            w = synth.weight(0, op - 1)
            adapters = [(full(a, 3, ins), full(b, 3, outs), s)
                        for a, b, s in ((lo, lo, 1 << 16), (hi, lo, -1 << 31), (lo, hi, (1 << 31) - 1),
                                        (1, 1, 1), (lo, 1, 3), (1, lo, -5))]
            x = np.stack([full(v, ins) for v in (lo, hi, lo, hi, -1, 1)])
            for shift in range(6):
                of_row = [(r + shift) % 6 for r in range(6)]
                got = _run(acc, hip, op, x, adapters, of_row, outs)
                assert np.array_equal(got, _expected(x, w, adapters, of_row)), (op, shift)


@pytest.mark.gpu
def test_rows_and_results_in_one_place():
    spec = ODD
    synth = _model(spec)
    rng = np.random.default_rng(5)
    with llm_accel.Accelerator(accel_shape(spec, layers=1)) as acc, Hip() as hip:
        acc.load_model(synth)
        for op in (1, 2, 5, 7):
            w = synth.weight(0, op - 1)
            outs, ins = w.shape
            adapters = [_adapter(rng, 9, ins, outs)]
            x = rng.integers(-900, 901, (4, ins)).astype(np.int16)
            got = _run(acc, hip, op, x, adapters, [0, -1, 0, 0], outs, in_place=True)
            assert np.array_equal(got, _expected(x, w, adapters, [0, -1, 0, 0]))
            # the context's own ports
            acc.port_write(llm_accel.PORT_IN, x)
            dev = [(hip.put(a), hip.put(b), a.shape[0], s) for a, b, s in adapters]
            acc.op_adapted(op, 0, [0, 0, 0, -1], dev)
            got = acc.port_read(llm_accel.PORT_OUT, 4 * outs).reshape(4, outs)
            assert np.array_equal(got, _expected(x, w, adapters, [0, 0, 0, -1]))


@pytest.mark.gpu
def test_captured_and_replayed():
    spec = SPECS["A"]
    synth = _model(spec)
    rng = np.random.default_rng(6)
    w = synth.weight(0, 6)
    outs, ins = w.shape
    adapters = [_adapter(rng, 16, ins, outs), _adapter(rng, 5, ins, outs)]
    of_row = [1, 0, -1, 0, 1]
    with llm_accel.Accelerator(accel_shape(spec, layers=1)) as acc, Hip() as hip:
        acc.load_model(synth)
        dev = [(hip.put(a), hip.put(b), a.shape[0], s) for a, b, s in adapters]
        x = rng.integers(-900, 901, (5, ins)).astype(np.int16)
        din, dout = hip.put(x), hip.alloc(5 * outs * 2)
        call = lambda: acc.op_adapted(7, 0, of_row, dev, din, dout)  # noqa: E731
        call()
        acc.sync()
        stream = llm_accel.lib().llm_stream(acc._ctx)
        graph = hip.capture(stream, call)
        for _ in range(4):
            x = rng.integers(-900, 901, (5, ins)).astype(np.int16)
            hip.put(x, to=din)
            hip.put(np.zeros((5, outs), np.int16), to=dout)
            hip.replay(graph, stream)
            acc.sync()
            want = _expected(x, w, adapters, of_row)
            assert np.array_equal(hip.get(dout, (5, outs), np.int16), want)
            got = _run(acc, hip, 7, x, adapters, [0] * 5, outs)  # eager, between replays
            assert np.array_equal(got, _expected(x, w, adapters, [0] * 5))


def test_refusals_without_a_context():
    lib = llm_accel.lib()
    ad = (llm_accel.Adapter * 1)(llm_accel.Adapter(1 << 20, 1 << 20, 4, 1))
    one = (ctypes.c_int32 * 1)(0)
    assert lib.llm_op_adapted(None, 1, 0, 1, 1 << 20, 1 << 20, ad, 1, one, None) == -1


@pytest.mark.gpu
def test_refusals_and_status_codes():
    spec = SPECS["A"]
    with llm_accel.Accelerator(accel_shape(spec, layers=1)) as acc, Hip() as hip:
        p = hip.alloc(1 << 20)
        good = (p, p, 4, 1)
        with pytest.raises(llm_accel.AccelError, match="not loaded"):
            acc.op_adapted(1, 0, [0], [good], p, p)
        acc.load_model(workloads.SyntheticModel(spec, layers=1))
        for op in (0, 8, 14, 18, 21):
            with pytest.raises(llm_accel.AccelError, match="not a projection"):
                acc.op_adapted(op, 0, [0], [good], p, p)
        for bad in ((None, p, 4, 1), (p, None, 4, 1), (p, p, 0, 1), (p, p, 513, 1),
                    (p + 2, p, 4, 1), (p, p + 4, 4, 1)):
            with pytest.raises(llm_accel.AccelError, match="adapter 1"):
                acc.op_adapted(1, 0, [0, 1], [good, bad], p, p)
            acc.op_adapted(1, 0, [0, 0], [good, bad], p, p)  # no row names it
        for of_row in ([1], [-2], [0, 7], [1 << 30]):
            with pytest.raises(llm_accel.AccelError, match="names no adapter"):
                acc.op_adapted(1, 0, of_row, [good], p, p)
        with pytest.raises(llm_accel.AccelError, match="8-byte"):
            acc.op_adapted(1, 0, [0], [good], p + 4, p)
        st = acc.op_adapted(1, 0, [0] * 9, [good], p, p)
        assert st.code == llm_accel.BAD_TOKEN_COUNT
        st = acc.op_adapted(1, 1, [0], [good], p, p)
        assert st.code == llm_accel.BAD_LAYER
        st = acc.op_adapted(1, 0, [], [], p, p)
        assert st.code == llm_accel.STATUS_OK
        want = acc.op(1, token_count=3, lhs=np.zeros((3, spec.hidden), np.int16))[1]
        assert acc.op_adapted(1, 0, [0, -1, 0], [good], p, p).as_tuple() == want.as_tuple()
        acc.sync()
