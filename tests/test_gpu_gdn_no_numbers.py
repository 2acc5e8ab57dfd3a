"""Rows that hold no number: they spoil the rows behind them in their own sequence, and those of their block or pass, and nothing else."""
import numpy as np
import pytest

import turbospark_amd as ts
from tests.gdn_common import Dev, Layer, from_bits, offsets_of, strided, to_bits
from tests.test_gpu_gdn import Prompt, Step, _results, _ring

pytestmark = pytest.mark.gpu
BF, HF = ts.BF16, ts.F16
NAN, INF = {BF: 0x7FC1, HF: 0x7E01}, {BF: 0x7F80, HF: 0x7C00}


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("bits", [NAN, INF])
def test_in_a_convolution(dtype, bits):
    rng = np.random.default_rng(41)
    ly = Layer(rng, 1, 2, 64, 32, 4, dtype)
    lengths, base = [20, 40, 7], [3, 64, 0]
    off, T = offsets_of(lengths), sum(lengths)
    x, a = to_bits(rng.standard_normal((T, ly.C)), dtype), to_bits(rng.standard_normal((T, 2)), dtype)
    ring = _ring(rng, ly, 3, base)
    got = []
    for bad in (False, True):
        y = x.copy()
        if bad:
            y[off[1] + 21] = bits[dtype]
            y[off[1] + 39] = bits[dtype]
        dx, da, dr, dbase, out = Dev(y), Dev(a), Dev(ring), Dev(np.array(base, np.int64)), Dev(np.zeros_like(x))
        g, be = Dev(np.zeros((T, 2), np.float32)), Dev(np.zeros((T, 2), np.float32))
        ly.gpu.conv(ly.gpu.batch(off, dbase.ptr), ts.GdnConv(qkv=dx.ptr, qkv_stride=ly.C, a=da.ptr, b=da.ptr, gate_stride=2, ring=dr.ptr, out=out.ptr,
                                                             out_stride=ly.C, g=g.ptr, beta=be.ptr))
        got.append((out.get(), dr.get(), g.get(), be.get()))
    (rows, ring_a, g_a, be_a), (spoilt, ring_b, g_b, be_b) = got
    touched = [off[1] + r for r in (21, 22, 23, 24, 39)]                # four taps
    sound = [r for r in range(T) if r not in touched]
    assert np.array_equal(rows[sound], spoilt[sound]) and np.array_equal(g_a, g_b) and np.array_equal(be_a, be_b)
    assert np.isnan(from_bits(spoilt[off[1] + 21], dtype)).any()
    assert np.array_equal(ring_a[[0, 2]], ring_b[[0, 2]])


@pytest.mark.parametrize("hk,hv,dk,dv,lengths,bad_row", [
    (2, 4, 64, 64, [200, 130, 64], 100),
    (1, 3, 128, 48, [200, 130, 64], 199),            # the last row, which the rows behind the sequence's end are taken from
    (1, 2, 64, 32, [2100, 130, 0], 1500),            # in segments
    (4, 8, 128, 128, [70] * 8, 66),                  # two column tiles a workgroup
    (16, 32, 64, 16, [130, 70] * 8, 65),             # several value heads a workgroup
])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("where", ["q", "k", "v", "g", "beta", "z", "v inf"])
def test_in_a_prompt(hk, hv, dk, dv, lengths, bad_row, dtype, where):
    rng = np.random.default_rng(dk + dv)
    p = Prompt(rng, Layer(rng, hk, hv, dk, dv, 4, dtype), lengths, [s % 3 for s in range(len(lengths))], gated=True)
    p.ly.gpu.prefill(p.batch, p.io)
    rows, S = p.check()
    if where in ("g", "beta"):
        buf, dev = (p.g, p.dg) if where == "g" else (p.beta, p.db)
        buf = buf.copy()
        buf[bad_row] = np.nan
        dev.put(np.concatenate([buf, np.full((1, hv), np.nan, np.float32)]))
    else:
        buf, dev, stride = {"q": (p.q, p.dq, p.io.q_stride), "k": (p.k, p.dk_, p.io.k_stride), "v": (p.v, p.dv_, p.io.v_stride), "z": (p.z, p.dz, p.io.z_stride)}[where[0]]
        buf = buf.copy()
        buf[bad_row] = (INF if "inf" in where else NAN)[dtype]
        dev.put(strided(buf, stride))
    p.out.put(np.full_like(p.out.a, 0x1234))
    p.ly.gpu.prefill(p.batch, p.io)
    spoilt, T = p.out.get(), p.dout.get()
    block = bad_row // 64 * 64
    assert np.array_equal(spoilt[:block], rows[:block]) and np.array_equal(spoilt[lengths[0]:], rows[lengths[0]:])
    assert np.array_equal(T[1:], S[1:])
    assert np.isnan(from_bits(spoilt[bad_row, :hv * dv], dtype)).any()
    if where in ("q", "z"):                          # neither goes into the state
        assert np.array_equal(T[0], S[0])
    if where == "z":
        sound = [r for r in range(p.T) if r != bad_row]
        assert np.array_equal(spoilt[sound], rows[sound])


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("lengths", [[5, 16, 2], [1, 1, 1]])
@pytest.mark.parametrize("where", ["x", "a", "b", "z", "state"])
def test_in_a_step_and_its_commit(dtype, lengths, where):
    got = []
    for bad in (False, True):
        rng = np.random.default_rng(43)
        ly = Layer(rng, 2, 4, 64, 32, 4, dtype)
        p = Step(rng, ly, lengths, [7, 31, 2])
        if bad and where == "state":
            p.state[1, 1, 3, 5] = np.nan
            p.din.put(p.state)
        elif bad:
            buf, dev, stride = {"x": (p.x, p.dx, p.io.qkv_stride), "a": (p.a, p.da, p.io.gate_stride), "b": (p.b, p.db, p.io.gate_stride), "z": (p.z, p.dz, p.io.z_stride)}[where]
            buf[p.off[2] - 1] = NAN[dtype]           # the second sequence's last row
            dev.put(strided(buf, stride))
        p.io.record, p.io.state_out = p.record.ptr, p.dnew.ptr
        ly.gpu.step(p.batch, p.io)
        final = p.dnew.get()
        res = _results([list(range(m)) for m in lengths])
        ly.gpu.commit(p.batch, ts.GdnCommit(n_layers=1, results=res.ptr, record=p.record.ptr, ring_in=p.dring.ptr, ring_out=p.dring.ptr,
                                            state_in=p.din.ptr, state_out=p.din.ptr))
        got.append((p.out.get(), final, p.din.get(), p.off))
    (rows, final_a, kept_a, off), (spoilt, final_b, kept_b, _) = got
    sound = [r for r in range(off[-1]) if not off[1] <= r < off[2]]
    assert np.array_equal(rows[sound], spoilt[sound])
    for a, b in ((final_a, final_b), (kept_a, kept_b)):
        assert np.array_equal(a[[0, 2]], b[[0, 2]]) and np.isfinite(b[[0, 2]]).all()
    assert np.isnan(from_bits(spoilt[off[1]:off[2], :128], dtype)).any()


def test_rows_that_were_not_kept_do_not_reach_the_state():
    """A record of rejected rows that hold no number: the commit reads the kept ones alone."""
    rng = np.random.default_rng(44)
    ly = Layer(rng, 2, 4, 64, 32, 4, BF)
    p = Step(rng, ly, [9, 5], [7, 0], tree=True)
    res = _results([[0, 1, 5, 6, 7], [0, 2]])
    rec = rng.standard_normal(p.record.a.shape).astype(np.float32)
    a, b = p.T * 128, p.T * 128
    rec[a + b:a + b + p.T * 4] = -np.abs(rec[a + b:a + b + p.T * 4])
    want = None
    for bad in (False, True):
        r = rec.copy()
        if bad:
            for row in (2, 3, 4, 8, 9 + 1, 9 + 4):
                r[row * 128:(row + 1) * 128] = np.nan
                r[a + row * 128:a + (row + 1) * 128] = np.inf
                r[a + b + row * 4:a + b + row * 4 + 4] = np.nan
        p.record.put(r)
        ly.gpu.commit(p.batch, ts.GdnCommit(n_layers=1, results=res.ptr, record=p.record.ptr, ring_in=p.dring.ptr, ring_out=p.dring.ptr,
                                            state_in=p.din.ptr, state_out=p.dnew.ptr))
        S = p.dnew.get()
        assert np.isfinite(S).all()
        want = S if want is None else want
        assert np.array_equal(S, want)
