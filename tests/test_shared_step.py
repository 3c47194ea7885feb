"""A decoding step made of the operators for batches, as a serving program
runs it: requests that share a prompt, each under an adapter of its own or
none, their drafted tokens verified in the same step.  Every value against the
oracle's operators and the tests' definitions."""
import numpy as np
import pytest

import llm_accel
import workloads
from helpers import accel_shape, first_mismatch
from hipmem import Hip
from oracle import orc
from test_lm_verify import _probs_row, _scores, _verify
from test_op_adapted import _adapter
from test_op_adapted import _expected as adapted

SPEC = workloads.ShapeSpec("step", 1000, 256, 688, 2, 8, 2, 32, 0.25, 0.5)


def _layer(spec, synth, layer, x, pos, of_row, adapters, table, prefix, own):
    """One decoder layer on rows x by the definitions; own: per row its K / V
    before this step, to which the rows of its request add theirs."""
    heads, kv, d = spec.heads, spec.kv_heads, spec.hidden // spec.heads
    norms = synth.norms()
    w = lambda p: synth.weight(layer, p)  # noqa: E731
    run = lambda p, v: adapted(v, w(p), adapters[layer][p], of_row)  # noqa: E731
    n1 = orc.rmsnorm(x, norms[2 * layer])
    q, k, v = (run(p, n1) for p in range(3))
    q = np.stack([orc.rope_apply(r, heads, d, table[p]) for r, p in zip(q, pos)])
    k = np.stack([orc.rope_apply(r, kv, d, table[p]) for r, p in zip(k, pos)])
    o = np.zeros_like(q)
    for r in range(len(x)):
        ko, vo = own(r, k, v)
        for h in range(kv):
            g = heads // kv
            o[r].reshape(heads, d)[h * g:(h + 1) * g] = orc.attention(
                q[r].reshape(heads, d)[h * g:(h + 1) * g],
                np.concatenate([prefix[0][layer, h], ko[:, h]]),
                np.concatenate([prefix[1][layer, h], vo[:, h]]))
    x = orc.residual(x, run(3, o))
    n2 = orc.rmsnorm(x, norms[2 * layer + 1])
    return orc.residual(x, run(6, orc.silu_mul(run(4, n2), run(5, n2)))), k, v


@pytest.mark.gpu
@pytest.mark.parametrize("plen", [0, 100, 700])
def test_steps_of_requests_that_share_a_prompt(plen):
    spec, layers, cap, steps = SPEC, 2, 24, 3
    hid, heads, kv, d = spec.hidden, spec.heads, spec.kv_heads, spec.hidden // spec.heads
    rng = np.random.default_rng([5, plen])
    synth = workloads.SyntheticModel(spec, seed=4, layers=layers)
    norms, emb, lm = synth.norms(), synth.embedding(), synth.lm_head()
    table = orc.rope_table(plen + cap + 1, d)
    # request j: its adapter, and its drafts per step
    of_request, counts = [0, -1, 1], [2, 1, 0]
    request = [j for j, c in enumerate(counts) for _ in range(c + 1)]
    rows = len(request)
    of_row = [of_request[j] for j in request]
    adapters = [[[_adapter(rng, rank, *synth.weight(la, p).shape[::-1], limit=300, scale=8000)
                  for rank in (8, 20)] for p in range(7)] for la in range(layers)]
    norm16 = lambda s, *sh: np.round(rng.standard_normal(sh) * 256 * s).astype(np.int16)  # noqa: E731,E501
    prefix = norm16(1.0, layers, kv, plen, d), norm16(0.5, layers, kv, plen, d)
    temperatures = [30.0, 64.0, 40.0]  # the synthetic head's scores spread over 100 and more
    # what each request has generated: K / V per layer [n][kv][d], last token
    past = [[(np.zeros((0, kv, d), np.int16),) * 2 for _ in range(layers)] for _ in counts]
    last = rng.integers(0, spec.vocab, len(counts)).tolist()
    op, taken = llm_accel, 0
    with llm_accel.Accelerator(accel_shape(spec, max_seq=plen + cap)) as acc, Hip() as hip:
        acc.load_model(synth)
        acc.load_lm_head(lm)
        for la in range(layers):
            for h in range(kv):
                if plen:
                    acc.kv_write(la, h, 0, prefix[0][la, h], prefix[1][la, h])
        dev = [[[(hip.put(a), hip.put(b), len(a), s) for a, b, s in ads] for ads in per]
               for per in adapters]
        dnorm = [hip.put(n) for n in norms]
        buf = lambda n: hip.alloc(2 * rows * n)  # noqa: E731
        dx, dn, dq, dk, dv, do = buf(hid), buf(hid), buf(hid), buf(hid), buf(hid), buf(hid)
        dg, du = buf(spec.inter), buf(spec.inter)
        own_n = rows * kv * cap * d
        dko, dvo, dlen = hip.alloc(2 * own_n), hip.alloc(2 * own_n), hip.alloc(4 * rows)
        for step in range(steps):
            drafts = [rng.integers(0, spec.vocab, c).tolist() for c in counts]
            tokens = [t for j in range(len(counts)) for t in [last[j]] + drafts[j]]
            back = [i for c in counts for i in range(c + 1)]  # the row's place in its request
            pos = [plen + len(past[j][0][0]) + i for j, i in zip(request, back)]
            x = emb[tokens]
            # --- the step on the device ---
            hip.put(x, to=dx)
            hip.put(np.array([p + 1 - plen for p in pos], np.uint32), to=dlen)
            for la in range(layers):
                def project(p, src, dst):
                    st = acc.op_adapted(p + 1, la, of_row, dev[la][p], src, dst)
                    assert st.code == 0
                acc.op(op.OP_RMSNORM, 0, rows, in_ptr=dx, aux_ptr=dnorm[2 * la], out_ptr=dn,
                       sync=False)
                for p, dst in ((0, dq), (1, dk), (2, dv)):
                    project(p, dn, dst)
                acc.sync()
                # rotation and the rows' places on the host
                q, k, v = (hip.get(a, (rows, n, d), np.int16)
                           for a, n in ((dq, heads), (dk, kv), (dv, kv)))
                q = np.stack([orc.rope_apply(r, heads, d, table[p]) for r, p in zip(q, pos)])
                k = np.stack([orc.rope_apply(r, kv, d, table[p]) for r, p in zip(k, pos)])
                ko, vo = rng.integers(-9999, 9999, (2, rows, kv, cap, d)).astype(np.int16)
                for r, j in enumerate(request):
                    for into, old, new in ((ko, past[j][la][0], k), (vo, past[j][la][1], v)):
                        mine = np.concatenate([old, new.reshape(rows, kv, d)[r - back[r]:r + 1]])
                        into[r, :, :len(mine)] = mine.transpose(1, 0, 2)
                hip.put(q, to=dq), hip.put(ko, to=dko), hip.put(vo, to=dvo)
                acc.attention_shared(la, plen, rows, dq, dko, dvo, dlen, cap, do)
                project(3, do, dn)
                acc.op(op.OP_RESIDUAL_ADD, 0, rows, in_ptr=dx, aux_ptr=dn, out_ptr=dx, sync=False)
                acc.op(op.OP_RMSNORM, 0, rows, in_ptr=dx, aux_ptr=dnorm[2 * la + 1], out_ptr=dn,
                       sync=False)
                project(4, dn, dg)
                project(5, dn, du)
                acc.op(op.OP_SILU_MUL, 0, rows, in_ptr=dg, aux_ptr=du, out_ptr=dg, sync=False)
                project(6, dg, dn)
                acc.op(op.OP_RESIDUAL_ADD, 0, rows, in_ptr=dx, aux_ptr=dn, out_ptr=dx, sync=False)
            acc.op(op.OP_RMSNORM, 0, rows, in_ptr=dx, aux_ptr=dnorm[2 * layers], out_ptr=dn)
            final = hip.get(dn, (rows, hid), np.int16)
            acc.upload(1, final)
            flat = sum(drafts, [])
            accept, sample = (rng.integers(0, 1 << 32, n).tolist() for n in (len(flat), 3))
            if step != 1:  # a draft of any probability is taken
                accept = [0] * len(flat)
            got = acc.lm_head_verify(1, 0, counts, flat, accept, sample, temperatures)
            # --- and by the definitions ---
            want, kvs = x, []
            for la in range(layers):
                def own(r, k, v):
                    j = request[r]
                    return [np.concatenate([o, n.reshape(rows, kv, d)[r - back[r]:r + 1]])
                            for o, n in zip(past[j][la], (k, v))]
                want, k, v = _layer(spec, synth, la, want, pos, of_row, adapters, table, prefix,
                                    own)
                kvs.append((k.reshape(rows, kv, d), v.reshape(rows, kv, d)))
            want = orc.rmsnorm(want, norms[2 * layers])
            assert np.array_equal(final, want), first_mismatch(final, want)
            scores = _scores(want, lm)
            p = np.stack([_probs_row(s, temperatures[j]) for s, j in zip(scores, request)])
            expect = _verify(p, counts, flat, accept, sample, None)
            assert [list(g) for g in got] == [list(e) for e in expect]
            taken += sum(got[0])
            # the taken rows join their request's past
            first = 0
            for j, c in enumerate(counts):
                n = got[0][j] + 1
                past[j] = [tuple(np.concatenate([o, a[first:first + n]])
                                 for o, a in zip(past[j][la], kvs[la])) for la in range(layers)]
                last[j] = got[1][j]
                first += c + 1
        assert taken > 0


def test_the_step_by_definitions_moves_with_its_adapters():
    """The definitions themselves: rows under an adapter differ from those
    without, and rows of equal adapters and inputs are equal."""
    spec = SPEC
    synth = workloads.SyntheticModel(spec, seed=4, layers=1)
    rng = np.random.default_rng(6)
    adapters = [[[_adapter(rng, 8, *synth.weight(0, p).shape[::-1], limit=300, scale=8000)]
                 for p in range(7)]]
    d, kv = spec.hidden // spec.heads, spec.kv_heads
    empty = np.zeros((1, kv, 0, d), np.int16), np.zeros((1, kv, 0, d), np.int16)
    x = np.repeat(synth.embedding()[5:6], 3, 0)
    own = lambda r, k, v: (k[r:r + 1].reshape(1, kv, d), v[r:r + 1].reshape(1, kv, d))  # noqa: E731
    y, _, _ = _layer(spec, synth, 0, x, [3, 3, 3], [0, -1, 0], adapters, orc.rope_table(8, d),
                     empty, own)
    assert np.array_equal(y[0], y[2]) and not np.array_equal(y[0], y[1])
