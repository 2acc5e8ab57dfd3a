"""The recurrent mixer (tsv_gdn_*) against the recurrence row after row in 64 bits.

Tolerances.  A result rounded to the rows' type is off by half a step, 2^-8 (bf16) or 2^-11 (fp16) of the value.  Operands of the
matrix products are two bf16 terms (2^-18 of the value at most) and the product of the two lower terms is left out (2^-18): of what a
product adds at most 3 * 2^-18 is lost.  The state passes through three such products a block (k S, T r, k^T u), 9 * 2^-18 < 2^-14 at
worst; the recurrence contracts (|1 - beta k k^T| <= 1, e^g <= 1), so that blocks do not add up beyond the state's own size.  In the
2-norm, where these errors are of all signs, half of that is allowed: 2^-15.  The rows of a prompt take u and P rounded to bf16 once
for bf16 rows (two more half steps; fp16 rows: two terms), then the result's rounding, and under a gate the norm's rounding
after that of o: 3 and 4 half steps.  f32 sums of at most 256 products: 2^-16 and less."""
import ctypes as C

import numpy as np
import pytest

import turbospark_amd as ts
from turbospark_amd import ffi, hip
from tests.gdn_common import RING, TREE16, Dev, Layer, chain, from_bits, half_step, offsets_of, rel2, strided, to_bits

pytestmark = pytest.mark.gpu
BF, HF = ts.BF16, ts.F16
STATE = 2.0 ** -15


def _ring(rng, ly, n, base):
    """Rings of n sequences; slots that hold no position yet are no numbers."""
    r = to_bits(rng.standard_normal((n, RING, ly.C)), ly.dtype)
    for s in range(n):
        for slot in range(RING):
            if base[s] < RING and slot >= base[s]:
                r[s, slot] = 0x7FC1
    return r


# ---- the convolution ----------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("hk,hv,dk,dv,taps,dtype,lengths,base", [
    (2, 4, 64, 64, 4, HF, [1], [0]),
    (2, 4, 64, 64, 4, BF, [2, 0, 3, 1], [1, 5, 2, 31]),
    (1, 3, 128, 48, 4, BF, [15, 16, 17], [0, 100, 30]),
    (4, 8, 64, 128, 4, HF, [33, 32], [31, 3]),
    (16, 16, 128, 128, 4, BF, [70], [4000000000]),
    (1, 1, 256, 16, 3, BF, [40], [29]),
    (2, 2, 64, 80, 2, HF, [31, 1], [2, 0]),
    (1, 2, 64, 16, 1, BF, [5], [3]),
])
def test_convolution_rows_gates_and_ring(hk, hv, dk, dv, taps, dtype, lengths, base):
    rng = np.random.default_rng(hk * 1000 + dv + taps)
    ly = Layer(rng, hk, hv, dk, dv, taps, dtype)
    off, n, T = offsets_of(lengths), len(lengths), sum(lengths)
    x, a, b = (to_bits(rng.standard_normal(s), dtype) for s in ((T, ly.C), (T, hv), (T, hv)))
    ring = _ring(rng, ly, n, base)
    stride, gs = ly.C + 24, hv + 1
    dx, da, db, dring = Dev(strided(x, stride), lead=16), Dev(strided(a, gs)), Dev(strided(b, gs)), Dev(ring)
    out = Dev(np.full((T + 1, ly.C + 8), 0x1234, np.uint16))
    g, be = Dev(np.full((T + 1, hv), 7.0, np.float32)), Dev(np.full((T + 1, hv), 7.0, np.float32))
    dbase = Dev(np.array(base, np.int64))
    io = ts.GdnConv(qkv=dx.ptr, qkv_stride=stride, a=da.ptr, b=db.ptr, gate_stride=gs, ring_in=dring.ptr, ring_out=dring.ptr, out=out.ptr, out_stride=ly.C + 8,
                    g=g.ptr, beta=be.ptr)
    ly.gpu.conv(ly.gpu.batch(off, dbase.ptr), io)
    rows, got_g, got_b, got_ring = out.get(), g.get(), be.get(), dring.get()
    assert (rows[T] == 0x1234).all() and (rows[:, ly.C:] == 0x1234).all() and (got_g[T] == 7).all() and (got_b[T] == 7).all()
    want_ring = ring.copy()
    for s in range(n):
        lo, hi = off[s], off[s + 1]
        q, k, v = ly.convolved(from_bits(x[lo:hi], dtype), from_bits(ring[s], dtype), base[s], chain(hi - lo))
        want = np.concatenate([t.reshape(hi - lo, t.shape[1] * t.shape[2]) for t in (q, k, v)], axis=1)
        err = np.abs(from_bits(rows[lo:hi, :ly.C], dtype) - want)
        # the f32 sums and exponentials of values up to a few: 2^-20; fp16 has no steps finer than 2^-25 below 2^-14
        assert (err <= half_step(dtype) * np.abs(want) * (1 + 2.0 ** -6) + 2.0 ** -20).all(), err.max()
        wg, wb = ly.gates(from_bits(a[lo:hi], dtype), from_bits(b[lo:hi], dtype))
        assert np.allclose(got_g[lo:hi], wg, rtol=2.0 ** -19, atol=0) and np.allclose(got_b[lo:hi], wb, rtol=2.0 ** -20, atol=0)
        for i in range(max(0, hi - lo - (taps - 1)), hi - lo):
            want_ring[s, (base[s] + i) % RING] = x[lo + i]
    assert np.array_equal(got_ring, want_ring)


def test_convolution_of_128_sequences():
    rng = np.random.default_rng(5)
    ly = Layer(rng, 1, 1, 64, 16, 4, BF)
    lengths = [int(v) for v in rng.integers(0, 40, 128)]
    off, T = offsets_of(lengths), sum(lengths)
    x, a = to_bits(rng.standard_normal((T, ly.C)), BF), to_bits(rng.standard_normal((T, 1)), BF)
    base = [int(v) for v in rng.integers(0, 100, 128)]
    ring = _ring(rng, ly, 128, base)
    dx, da, dring, out = Dev(x), Dev(a), Dev(ring), Dev(np.zeros_like(x))
    g, be, dbase = Dev(np.zeros((T, 1), np.float32)), Dev(np.zeros((T, 1), np.float32)), Dev(np.array(base, np.int64))
    ly.gpu.conv(ly.gpu.batch(off, dbase.ptr), ts.GdnConv(qkv=dx.ptr, qkv_stride=ly.C, a=da.ptr, b=da.ptr, gate_stride=1, ring_in=dring.ptr, ring_out=dring.ptr,
                                                         out=out.ptr, out_stride=ly.C, g=g.ptr, beta=be.ptr))
    rows = from_bits(out.get(), BF)
    for s in range(128):
        lo, hi = off[s], off[s + 1]
        q, k, v = ly.convolved(from_bits(x[lo:hi], BF), from_bits(ring[s], BF), base[s], chain(hi - lo))
        want = np.concatenate([t.reshape(hi - lo, t.shape[1] * t.shape[2]) for t in (q, k, v)], axis=1)
        assert (np.abs(rows[lo:hi] - want) <= 2.0 ** -8 * np.abs(want) * (1 + 2.0 ** -6) + 2.0 ** -20).all(), s


def test_a_convolution_made_again_from_the_same_rings():
    """With a ring_out of its own a pass leaves what it read: lengths whose last rows go to the very slots that the first ones read."""
    rng = np.random.default_rng(9)
    ly = Layer(rng, 1, 2, 64, 32, 4, HF)
    lengths, base = [30, 31, 32, 33, 34, 62, 1, 0], [31, 64, 3, 100, 7, 31, 40, 12]
    off, n, T = offsets_of(lengths), len(lengths), sum(lengths)
    x, a = to_bits(rng.standard_normal((T, ly.C)), HF), to_bits(rng.standard_normal((T, 2)), HF)
    ring = _ring(rng, ly, n, base)
    dx, da, din, dout, out = Dev(x), Dev(a), Dev(ring), Dev(np.full_like(ring, 0x1234)), Dev(np.zeros_like(x))
    g, be, dbase = Dev(np.zeros((T, 2), np.float32)), Dev(np.zeros((T, 2), np.float32)), Dev(np.array(base, np.int64))
    io = ts.GdnConv(qkv=dx.ptr, qkv_stride=ly.C, a=da.ptr, b=da.ptr, gate_stride=2, ring_in=din.ptr, ring_out=dout.ptr, out=out.ptr,
                    out_stride=ly.C, g=g.ptr, beta=be.ptr)
    want_ring = np.full_like(ring, 0x1234)
    for s in range(n):
        for i in range(max(0, lengths[s] - 3), lengths[s]):
            want_ring[s, (base[s] + i) % RING] = x[off[s] + i]
    for _ in range(2):
        out.put(np.zeros_like(x))
        ly.gpu.conv(ly.gpu.batch(off, dbase.ptr), io)
        rows = from_bits(out.get(), HF)
        for s in range(n):
            lo, hi = off[s], off[s + 1]
            q, k, v = ly.convolved(from_bits(x[lo:hi], HF), from_bits(ring[s], HF), base[s], chain(hi - lo))
            want = np.concatenate([t.reshape(hi - lo, t.shape[1] * t.shape[2]) for t in (q, k, v)], axis=1)
            assert (np.abs(rows[lo:hi] - want) <= half_step(HF) * np.abs(want) * (1 + 2.0 ** -6) + 2.0 ** -20).all(), s
        assert np.array_equal(dout.get(), want_ring) and np.array_equal(din.get(), ring)


# ---- the rule over prompts ------------------------------------------------------------------------------------------------

class Prompt:
    """Rows of a prompt and the buffers of one prefill call."""

    def __init__(self, rng, ly, lengths, base, keys="random", decay="usual", gated=True, pad=0):
        self.ly, self.lengths, self.base = ly, lengths, base
        self.off, self.n, T = offsets_of(lengths), len(lengths), sum(lengths)
        unit = lambda t: t / np.linalg.norm(t, axis=-1, keepdims=True)  # noqa: E731
        q, k = (unit(rng.standard_normal((T, ly.hk, ly.dk))) for _ in range(2))
        if keys == "same":
            k = np.broadcast_to(unit(rng.standard_normal((1, ly.hk, ly.dk))), k.shape)
        self.q, self.k, self.v = (to_bits(t.reshape(T, t.shape[1] * t.shape[2]), ly.dtype) for t in (q, k, rng.standard_normal((T, ly.hv, ly.dv))))
        g = -0.1 * rng.random((T, ly.hv))
        if decay == "wild":          # resets, no decay at all, a value above 0 (counts as 0), ordinary rows
            pick = rng.integers(0, 6, g.shape)
            g = np.select([pick == 0, pick == 1, pick == 2, pick == 3], [-np.inf, -1000.0, 0.0, 0.5], g)
        self.g = g.astype(np.float32)
        self.beta = (np.ones_like(g) if keys == "same" else rng.random(g.shape)).astype(np.float32)
        self.z = to_bits(rng.standard_normal((T, ly.hv * ly.dv)), ly.dtype) if gated else None
        self.state = (0.3 * rng.standard_normal((self.n, ly.hv, ly.dv, ly.dk))).astype(np.float32)
        given = self.state.copy()
        for s in range(self.n):
            if base[s] == 0:
                given[s] = np.nan
        qs, ks, vs = ly.hk * ly.dk + pad, ly.hk * ly.dk + 2 * pad, ly.hv * ly.dv + 3 * pad
        self.T, self.width = T, ly.hv * ly.dv + pad
        self.dq, self.dk_, self.dv_ = Dev(strided(self.q, qs)), Dev(strided(self.k, ks), lead=16), Dev(strided(self.v, vs))
        self.dg = Dev(np.concatenate([self.g, np.full((1, ly.hv), np.nan, np.float32)]))
        self.db = Dev(np.concatenate([self.beta, np.full((1, ly.hv), np.nan, np.float32)]))
        self.dz = Dev(strided(self.z, vs)) if gated else None
        self.dbase, self.din, self.dout = Dev(np.array(base, np.int64)), Dev(given), Dev(np.full_like(given, 3.0))
        self.out = Dev(np.full((T + 1, self.width), 0x1234, np.uint16))
        self.batch = ly.gpu.batch(self.off, self.dbase.ptr)
        self.ws = hip.DeviceBuffer(ly.gpu.prefill_workspace(self.batch))
        self.io = ts.GdnPrefill(q=self.dq.ptr, k=self.dk_.ptr, v=self.dv_.ptr, q_stride=qs, k_stride=ks, v_stride=vs, g=self.dg.ptr,
                                beta=self.db.ptr, z=self.dz.ptr if gated else None, z_stride=vs if gated else 0, state_in=self.din.ptr,
                                state_out=self.dout.ptr, out=self.out.ptr, out_stride=self.width, workspace=self.ws.ptr,
                                workspace_bytes=self.ws.nbytes)

    def want(self):
        ly = self.ly
        S = self.state.astype(np.float64)
        o = np.zeros((self.T, ly.hv, ly.dv))
        q, k, v = (from_bits(t, ly.dtype) for t in (self.q, self.k, self.v))
        q, k, v = q.reshape(-1, ly.hk, ly.dk), k.reshape(-1, ly.hk, ly.dk), v.reshape(-1, ly.hv, ly.dv)
        g, beta = np.minimum(self.g.astype(np.float64), 0), self.beta.astype(np.float64)
        for s in range(self.n):
            if self.base[s] == 0:
                S[s] = 0
            for i in range(self.off[s], self.off[s + 1]):
                S[s], _, o[i] = ly.row(S[s], q[i], k[i], v[i], g[i], beta[i])
        if self.z is not None:
            o = ly.gate(o, from_bits(self.z, ly.dtype))
        return o.reshape(self.T, ly.hv * ly.dv), S

    def check(self, state=None):
        ly = self.ly
        got, S = self.out.get(), (state or self.dout).get()
        want, want_S = self.want()
        assert (got[self.T] == 0x1234).all() and (got[:, ly.hv * ly.dv:] == 0x1234).all()
        for s in range(self.n):
            assert rel2(S[s], want_S[s]) <= STATE, (s, rel2(S[s], want_S[s]))
            assert np.abs(S[s] - want_S[s]).max() <= 2.0 ** -12 * max(np.abs(want_S[s]).max(), 2.0 ** -20)
        rows = from_bits(got[:self.T, :ly.hv * ly.dv], ly.dtype)
        steps = 4 if self.z is not None else 3
        if self.T:
            assert rel2(rows, want) <= steps * half_step(ly.dtype), rel2(rows, want)
            size = np.abs(want).reshape(self.T, ly.hv, ly.dv).max(-1).repeat(ly.dv, -1)
            assert (np.abs(rows - want) <= 4 * steps * half_step(ly.dtype) * size + 2.0 ** -20).all()
        return got, S


@pytest.mark.parametrize("hk,hv,dk,dv,dtype,lengths,base,pad", [
    (1, 1, 64, 16, BF, [1], [0], 0),
    (1, 1, 64, 16, HF, [1], [9], 8),
    (2, 4, 64, 64, HF, [65], [777], 0),
    (2, 4, 64, 64, BF, [63, 64, 65, 0, 1], [0, 5, 0, 7, 3], 8),
    (1, 3, 128, 48, BF, [130], [1], 0),
    (2, 2, 128, 128, BF, [300], [0], 16),
    (1, 4, 128, 128, HF, [17, 100], [2, 0], 0),
    (2, 2, 128, 80, HF, [0, 0], [0, 4], 0),
    (1, 2, 256, 32, BF, [129], [6], 8),
    (1, 1, 256, 256, HF, [70], [0], 0),
    (8, 24, 64, 32, BF, [31], [1], 0),
    (3, 9, 64, 96, BF, [127, 2], [0, 1], 0),
])
@pytest.mark.parametrize("gated", [True, False])
def test_prompt_blocks(hk, hv, dk, dv, dtype, lengths, base, pad, gated):
    rng = np.random.default_rng(dk + dv + len(lengths))
    p = Prompt(rng, Layer(rng, hk, hv, dk, dv, 4, dtype), lengths, base, gated=gated, pad=pad)
    p.ly.gpu.prefill(p.batch, p.io)
    p.check()


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("keys,decay", [("same", "usual"), ("random", "wild"), ("same", "wild")])
def test_prompt_with_alike_keys_and_wild_decays(dtype, keys, decay):
    """Keys that are all the same with beta 1 (the inverse's powers would cancel), decays that wipe the state, none at all."""
    rng = np.random.default_rng(11)
    p = Prompt(rng, Layer(rng, 2, 4, 128, 64, 4, dtype, scale=0.25), [200, 64], [3, 0], keys=keys, decay=decay, gated=False)
    p.ly.gpu.prefill(p.batch, p.io)
    p.check()


@pytest.mark.parametrize("hk,hv,dk,dv,dtype,lengths,base,decay", [
    (1, 1, 64, 64, BF, [2600], [0], "usual"),
    (1, 2, 128, 128, BF, [2049], [7], "usual"),
    (1, 1, 128, 48, HF, [2111], [0], "usual"),
    (1, 1, 256, 32, BF, [2200], [3], "usual"),
    (1, 2, 64, 32, BF, [2100, 70, 0, 2500], [5, 0, 4, 0], "usual"),
    (1, 1, 64, 32, HF, [2300], [9], "wild"),
])
def test_long_prompts_of_few_heads(hk, hv, dk, dv, dtype, lengths, base, decay):
    """Prompts that are walked in segments side by side and put together."""
    rng = np.random.default_rng(dk + dv + len(lengths))
    p = Prompt(rng, Layer(rng, hk, hv, dk, dv, 4, dtype), lengths, base, gated=False, decay=decay)
    p.ly.gpu.prefill(p.batch, p.io)
    rows, S = p.check()
    p.io.state_out = p.io.state_in               # in place: to the same bits
    p.ly.gpu.prefill(p.batch, p.io)
    assert np.array_equal(p.out.get(), rows) and np.array_equal(p.din.get(), S)


@pytest.mark.parametrize("size", [1e-12, 1e12])
def test_prompt_states_of_any_size(size):
    """Values and state far outside fp16's range: the operands' terms are bf16."""
    rng = np.random.default_rng(12)
    p = Prompt(rng, Layer(rng, 1, 2, 128, 32, 4, BF), [100], [5], gated=False)
    p.v = to_bits(from_bits(p.v, BF) * size, BF)
    p.state = (p.state * size).astype(np.float32)
    p.dv_.put(strided(p.v, 64))
    p.din.put(p.state)
    p.ly.gpu.prefill(p.batch, p.io)
    got, S = p.out.get(), p.dout.get()
    want, want_S = p.want()
    assert rel2(S, want_S) <= STATE and rel2(from_bits(got[:100, :64], BF), want) <= 3 * 2.0 ** -8


def test_prompt_in_place_and_in_two_calls():
    """A prompt in two calls, the state in place: as in one call, up to the two forms' own roundings; rows that share a buffer."""
    rng = np.random.default_rng(13)
    ly = Layer(rng, 2, 4, 64, 64, 4, BF)
    p = Prompt(rng, ly, [150], [0], gated=False)
    ly.gpu.prefill(p.batch, p.io)
    p.check()
    whole = p.out.get()
    p.io.state_out = p.io.state_in
    first = ly.gpu.batch([0, 90], p.dbase.ptr)
    ly.gpu.prefill(first, p.io)
    p.dbase.put(np.array([90], np.int64))
    at = lambda ptr, stride: ptr + 2 * 90 * stride  # noqa: E731
    p.io.q, p.io.k, p.io.v = at(p.io.q, p.io.q_stride), at(p.io.k, p.io.k_stride), at(p.io.v, p.io.v_stride)
    p.io.g, p.io.beta, p.io.out = p.dg.ptr + 4 * 90 * 4, p.db.ptr + 4 * 90 * 4, at(p.out.ptr, p.width)
    ly.gpu.prefill(ly.gpu.batch([0, 60], p.dbase.ptr), p.io)
    got, S = p.check(state=p.din)
    assert rel2(from_bits(got[:150], BF), from_bits(whole[:150], BF)) <= 4 * 2.0 ** -8


def test_prompt_calls_repeat_bit_for_bit_also_in_a_graph_and_beside_each_other():
    """Two calls at once on two streams with a workspace each, and a captured call replayed with other inputs: same bits as alone."""
    rng = np.random.default_rng(14)
    ly = Layer(rng, 2, 4, 128, 64, 4, BF)
    calls = [Prompt(rng, ly, [130, 70], [0, 4]) for _ in range(2)]
    alone = []
    for p in calls:
        ly.gpu.prefill(p.batch, p.io)
        alone.append(p.check())
        p.out.put(np.full_like(p.out.a, 0x1234))
    streams = [hip.Stream(), hip.Stream()]
    for _ in range(4):
        for p, st in zip(calls, streams):
            ly.gpu.prefill(p.batch, p.io, st.h)
    for p, st, (rows, S) in zip(calls, streams, alone):
        st.sync()
        assert np.array_equal(p.out.get(), rows) and np.array_equal(p.dout.get(), S)
    a, b = calls
    graph = hip.CapturedGraph(streams[0], lambda s: ly.gpu.prefill(a.batch, a.io, s.h))
    for source in (b, a, b):
        for dst, src in ((a.dq, source.q), (a.dv_, source.v)):
            dst.put(strided(src, src.shape[1]))
        a.dk_.put(strided(source.k, source.k.shape[1]))
        a.dg.put(np.concatenate([source.g, np.zeros((1, 4), np.float32)]))
        a.db.put(np.concatenate([source.beta, np.zeros((1, 4), np.float32)]))
        a.dz.put(strided(source.z, source.z.shape[1]))
        state = source.state.copy()
        state[0] = np.nan
        a.din.put(state)
        graph.launch()
        streams[0].sync()
        rows, S = alone[0] if source is a else alone[1]
        assert np.array_equal(a.out.get()[:200], rows[:200]) and np.array_equal(a.dout.get(), S)
        ly.gpu.prefill(b.batch, b.io)        # the program's own eager work between the replays
        hip.check(hip.rt().hipDeviceSynchronize(), "sync")


# ---- the step of a few rows ---------------------------------------------------------------------------------------------------

class Step:
    def __init__(self, rng, ly, lengths, base, tree=False, gated=True, pad=0, parents=None):
        self.ly, self.base, self.lengths = ly, base, lengths
        self.off, self.n, self.T = offsets_of(lengths), len(lengths), sum(lengths)
        self.parents = parents if parents is not None else [TREE16[:m] if tree else chain(m) for m in lengths]
        self.x, self.a, self.b = (to_bits(rng.standard_normal(s), ly.dtype) for s in ((self.T, ly.C), (self.T, ly.hv), (self.T, ly.hv)))
        self.z = to_bits(rng.standard_normal((self.T, ly.hv * ly.dv)), ly.dtype) if gated else None
        self.ring = _ring(rng, ly, self.n, base)
        self.state = (0.3 * rng.standard_normal((self.n, ly.hv, ly.dv, ly.dk))).astype(np.float32)
        given = self.state.copy()
        for s in range(self.n):
            if base[s] == 0:
                given[s] = np.nan
        stride, gs, self.width = ly.C + pad, ly.hv + (pad > 0), ly.hv * ly.dv + pad
        self.dx, self.da, self.db = Dev(strided(self.x, stride)), Dev(strided(self.a, gs)), Dev(strided(self.b, gs))
        self.dz = Dev(strided(self.z, self.width)) if gated else None
        self.dring, self.din, self.dnew = Dev(self.ring), Dev(given), Dev(np.full_like(given, 3.0))
        self.dbase = Dev(np.array(base, np.int64))
        self.dpar = Dev(np.array([q for p in self.parents for q in p] or [0], np.int32))
        self.out = Dev(np.full((self.T + 1, self.width), 0x1234, np.uint16))
        self.row = ly.hv * ly.dv + ly.hk * ly.dk + ly.hv
        assert ly.gpu.record_bytes(self.T) == 4 * self.T * self.row
        self.record = Dev(np.full((self.T * self.row + 8,), 5.0, np.float32))
        self.batch = ly.gpu.batch(self.off, self.dbase.ptr, self.dpar.ptr if tree or parents is not None else None)
        self.io = ts.GdnStep(qkv=self.dx.ptr, qkv_stride=stride, a=self.da.ptr, b=self.db.ptr, gate_stride=gs,
                             z=self.dz.ptr if gated else None, z_stride=self.width if gated else 0, ring=self.dring.ptr,
                             state_in=self.din.ptr, out=self.out.ptr, out_stride=self.width)

    def want(self):
        ly = self.ly
        o, u, ks, gs, ends, ring = np.zeros((self.T, ly.hv, ly.dv)), np.zeros((self.T, ly.hv, ly.dv)), [], [], [], self.ring.copy()
        self.off_by = np.zeros_like(o)
        for s, m in enumerate(self.lengths):
            lo = self.off[s]
            rows = slice(lo, lo + m)
            q, k, v = ly.convolved(from_bits(self.x[rows], ly.dtype), from_bits(self.ring[s], ly.dtype), self.base[s], self.parents[s])
            g, beta = ly.gates(from_bits(self.a[rows], ly.dtype), from_bits(self.b[rows], ly.dtype))
            at = {-1: np.zeros_like(self.state[s], np.float64) if self.base[s] == 0 else self.state[s].astype(np.float64)}
            for i in range(m):
                at[i], u[lo + i], o[lo + i] = ly.row(at[self.parents[s][i]], q[i], k[i], v[i], g[i], beta[i])
                ring[s, (self.base[s] + i) % RING] = self.x[lo + i]
            if m:
                self.off_by[rows] = self._bound(self.parents[s], at[-1], q, k, v, g, beta, u[rows])
            ks.append(k)
            gs.append(g)
            ends.append(at[m - 1])
        if self.z is not None:
            z, raw = from_bits(self.z, ly.dtype), o
            o = ly.gate(raw, z)
            # y = o / r * w with r the root of the mean square: dy <= (do + |o| dr / r) / r |w|, dr <= the root of the mean of do^2
            r = np.sqrt((raw ** 2).mean(-1, keepdims=True) + 1e-6)
            dr = np.sqrt((self.off_by ** 2).mean(-1, keepdims=True))
            w = np.abs(ly.norm * z.reshape(raw.shape) / (1 + np.exp(-z.reshape(raw.shape))))
            self.off_by = (self.off_by + np.abs(raw) * dr / r) / r * w + 2.0 ** -19 * np.abs(o)
        return o.reshape(self.T, -1), u, np.concatenate(ks), np.concatenate(gs), np.stack(ends), ring

    def _bound(self, parent, S, q, k, v, g, beta, u):
        """How far o may be off before its rounding, value by value.  A product with the state loses 3 * 2^-18 < 2^-16 of its absolute
        sum, which is |S_c| at most for a unit row; what u is off by passes to later rows through k_i.k_j and q_i.k_j as u itself
        does; f32 sums of up to 256 terms and the exponentials lose 2^-19 of their absolute sums."""
        ly, m = self.ly, len(q)
        q, k = np.repeat(q, ly.rep, 1), np.repeat(k, ly.rep, 1)
        size = np.linalg.norm(S, axis=-1)
        du, do = np.zeros_like(u), np.zeros_like(u)
        for i in range(m):
            line, decay = [], np.zeros(ly.hv)            # (ancestor, e^{sum of g behind it}), the row itself first
            at = i
            while at >= 0:
                line.append((at, np.exp(decay)))
                decay = decay + g[at]
                at = parent[at]
            held = np.exp(decay)[:, None] * size
            du[i] = 2.0 ** -16 * held + 2.0 ** -19 * (np.abs(v[i]) + held)
            for j, d in line[1:]:
                c = (d * np.abs((k[i] * k[j]).sum(-1)) + 2.0 ** -16 * d)[:, None]
                du[i] += c * du[j] + (2.0 ** -16 * d)[:, None] * np.abs(u[j]) + 2.0 ** -19 * c * np.abs(u[j])
            du[i] *= beta[i][:, None]
            do[i] = 2.0 ** -16 * held
            for j, d in line:
                c = (d * np.abs((q[i] * k[j]).sum(-1)) + 2.0 ** -16 * d)[:, None]
                do[i] += c * du[j] + (2.0 ** -16 * d)[:, None] * np.abs(u[j]) + 2.0 ** -19 * c * np.abs(u[j])
        return ly.scale * do

    def check(self, final=False, record=False):
        ly, T = self.ly, self.T
        o, u, k, g, ends, ring = self.want()
        got = self.out.get()
        assert (got[T] == 0x1234).all() and (got[:, ly.hv * ly.dv:] == 0x1234).all()
        rows = from_bits(got[:T, :ly.hv * ly.dv], ly.dtype)
        if T:
            assert rel2(rows, o) <= half_step(ly.dtype) + STATE, rel2(rows, o)
            # (fp16 has no steps finer than 2^-25 below 2^-14)
            assert (np.abs(rows - o) <= half_step(ly.dtype) * np.abs(o) * 1.01 + 1.01 * self.off_by.reshape(T, -1) + 2.0 ** -25).all()
        assert np.array_equal(self.dring.get(), ring)
        if final:
            S = self.dnew.get() if final == "new" else self.din.get()
            for s in range(self.n):
                assert rel2(S[s], ends[s]) <= STATE, (s, rel2(S[s], ends[s]))
        rec = self.record.get()
        assert (rec[T * self.row:] == 5.0).all()
        if record:
            a, b = T * ly.hv * ly.dv, T * ly.hk * ly.dk
            assert rel2(rec[:a], u.reshape(-1)) <= STATE
            assert rel2(rec[a:a + b], k.reshape(-1)) <= 2.0 ** -20 and rel2(rec[a + b:a + b + T * ly.hv], g.reshape(-1)) <= 2.0 ** -20
        else:
            assert (rec == 5.0).all()


SHAPES = [(1, 1, 64, 16, BF), (2, 4, 64, 64, HF), (1, 3, 128, 48, BF), (2, 4, 128, 128, BF), (1, 2, 256, 32, HF), (1, 2, 64, 256, BF),
          (1, 1, 256, 256, BF), (2, 2, 128, 80, HF)]


@pytest.mark.parametrize("hk,hv,dk,dv,dtype", SHAPES)
@pytest.mark.parametrize("lengths,base,tree", [
    ([1], [0], False), ([1, 1, 1], [1, 2, 64], False), ([5], [777], False), ([16, 3], [0, 31], False), ([16], [30], True),
    ([16, 1, 9], [0, 5, 2], True), ([13], [5000000000], True),
])
def test_rows_under_verification(hk, hv, dk, dv, dtype, lengths, base, tree):
    rng = np.random.default_rng(dk + dv + sum(lengths))
    p = Step(rng, Layer(rng, hk, hv, dk, dv, 4, dtype), lengths, base, tree, gated=dv != 48, pad=8 if dv == 64 else 0)
    p.io.record = p.record.ptr
    before = p.din.get()
    p.ly.gpu.step(p.batch, p.io)
    p.check(record=True)
    assert np.array_equal(p.din.get().view(np.uint32), before.view(np.uint32))      # nothing is final yet


@pytest.mark.parametrize("hk,hv,dk,dv,dtype", SHAPES)
@pytest.mark.parametrize("lengths,base,in_place", [([1], [0], False), ([1, 1, 1], [1, 2, 64], True), ([5, 16], [777, 0], False), ([3, 4, 2], [1, 0, 8], True)])
def test_final_rows(hk, hv, dk, dv, dtype, lengths, base, in_place):
    rng = np.random.default_rng(dk + dv + sum(lengths) + 1)
    p = Step(rng, Layer(rng, hk, hv, dk, dv, 4, dtype), lengths, base, gated=True)
    p.io.state_out = p.io.state_in if in_place else p.dnew.ptr
    p.ly.gpu.step(p.batch, p.io)
    p.check(final="in place" if in_place else "new")


@pytest.mark.parametrize("lengths,base", [([1, 1], [0, 9]), ([4, 1], [70, 0])])
@pytest.mark.parametrize("final,record", [(True, True), (False, False)])
def test_new_state_and_record_or_neither(lengths, base, final, record):
    rng = np.random.default_rng(8)
    p = Step(rng, Layer(rng, 2, 4, 128, 64, 4, BF), lengths, base, gated=True)
    if final:
        p.io.state_out = p.dnew.ptr
    if record:
        p.io.record = p.record.ptr
    before = p.din.get()
    p.ly.gpu.step(p.batch, p.io)
    p.check(final="new" if final else None, record=record)
    assert np.array_equal(p.din.get().view(np.uint32), before.view(np.uint32))


@pytest.mark.parametrize("dtype", [BF, HF])
def test_wider_passes_behind_narrow_ones(dtype):
    """The widest heads, more shared memory from pass to pass."""
    for rows in (2, 11, 14, 16):
        rng = np.random.default_rng(rows)
        p = Step(rng, Layer(rng, 1, 1, 256, 256, 4, dtype), [rows], [3])
        p.io.record = p.record.ptr
        p.ly.gpu.step(p.batch, p.io)
        p.check(record=True)


@pytest.mark.parametrize("taps", [1, 2, 3])
def test_fewer_taps_through_a_tree(taps):
    rng = np.random.default_rng(taps)
    p = Step(rng, Layer(rng, 2, 2, 64, 32, taps, BF), [16, 5], [1, 40], tree=True)
    p.io.record = p.record.ptr
    p.ly.gpu.step(p.batch, p.io)
    p.check(record=True)


def test_sequences_without_rows_keep_their_state():
    rng = np.random.default_rng(3)
    ly = Layer(rng, 1, 2, 64, 32, 4, BF)
    p = Step(rng, ly, [1, 1, 1], [4, 6, 0])
    p.io.state_out = p.dnew.ptr
    ly.gpu.step(ly.gpu.batch([0, 1, 1, 1], p.dbase.ptr), p.io)
    S, rows = p.dnew.get(), p.out.get()
    assert np.array_equal(S[1], p.state[1]) and (S[2] == 0).all()                   # a base of 0: nothing yet
    assert (rows[1:] == 0x1234).all()
    ring = p.dring.get()
    assert np.array_equal(ring[1:], p.ring[1:])


def test_malformed_parents_count_as_none():
    rng = np.random.default_rng(4)
    p = Step(rng, Layer(rng, 1, 2, 64, 32, 4, BF), [6, 4], [20, 3], parents=[[-7, 0, 2, 9, 1, 1 << 30], [3, -1, 1, -(1 << 31)]])
    p.io.record = p.record.ptr
    p.ly.gpu.step(p.batch, p.io)
    p.parents = [[-1, 0, -1, -1, 1, -1], [-1, -1, 1, -1]]
    p.check(record=True)


def test_a_step_is_the_prompt_continued():
    """The same rows as a prompt and as steps of one row: the prompt's rows are rounded once on the way (unit q, unit k, v), so the two
    agree to that rounding: a half step of each of q, k and v and those of the results."""
    rng = np.random.default_rng(6)
    ly = Layer(rng, 2, 4, 128, 64, 4, HF)
    n = 12
    p = Step(rng, ly, [n], [0])
    g, be, out = Dev(np.zeros((n, 4), np.float32)), Dev(np.zeros((n, 4), np.float32)), Dev(np.zeros((n, ly.C), np.uint16))
    ring = Dev(p.ring)
    batch = ly.gpu.batch([0, n], p.dbase.ptr)
    ly.gpu.conv(batch, ts.GdnConv(qkv=p.io.qkv, qkv_stride=p.io.qkv_stride, a=p.io.a, b=p.io.b, gate_stride=p.io.gate_stride, ring_in=ring.ptr, ring_out=ring.ptr,
                                  out=out.ptr, out_stride=ly.C, g=g.ptr, beta=be.ptr))
    rows, S = Dev(np.zeros((n, ly.hv * ly.dv), np.uint16)), Dev(np.zeros_like(p.state))
    ws = hip.DeviceBuffer(ly.gpu.prefill_workspace(batch))
    kd = 2 * ly.hk * ly.dk
    ly.gpu.prefill(batch, ts.GdnPrefill(q=out.ptr, k=out.ptr + kd, v=out.ptr + 2 * kd, q_stride=ly.C, k_stride=ly.C, v_stride=ly.C, g=g.ptr,
                                        beta=be.ptr, z=p.io.z, z_stride=p.io.z_stride, state_in=S.ptr, state_out=S.ptr, out=rows.ptr,
                                        out_stride=ly.hv * ly.dv, workspace=ws.ptr, workspace_bytes=ws.nbytes))
    prompt, end = rows.get(), S.get()
    p.io.state_out = p.io.state_in
    for i in range(n):
        p.dbase.put(np.array([i], np.int64))
        io = ts.GdnStep(qkv=p.io.qkv + 2 * i * p.io.qkv_stride, qkv_stride=p.io.qkv_stride, a=p.io.a + 2 * i * ly.hv, b=p.io.b + 2 * i * ly.hv,
                        gate_stride=ly.hv, z=p.io.z + 2 * i * p.io.z_stride, z_stride=p.io.z_stride, ring=p.io.ring, state_in=p.io.state_in,
                        state_out=p.io.state_in, out=p.out.ptr + 2 * i * p.width, out_stride=p.width)
        ly.gpu.step(ly.gpu.batch([0, 1], p.dbase.ptr), io)
    steps = p.out.get()[:n, :ly.hv * ly.dv]
    assert rel2(p.din.get(), end) <= 4 * 2.0 ** -11
    assert rel2(from_bits(steps, HF), from_bits(prompt, HF)) <= 8 * 2.0 ** -11
    o, _, _, _, ends, _ = p.want()
    assert rel2(from_bits(steps, HF), o) <= 2.0 ** -11 + STATE and rel2(p.din.get()[0], ends[0]) <= STATE


# ---- accepted rows into the state ----------------------------------------------------------------------------------------------

def _results(paths, committed=None):
    out = (ffi.RoundResultC * len(paths))()
    for s, p in enumerate(paths):
        out[s].path_len = len(p)
        out[s].committed = len(p) - 1 if committed is None else committed[s]
        for i, slot in enumerate(p):
            out[s].path[i] = slot
    return Dev(np.frombuffer(bytes(out), np.int32).copy())


@pytest.mark.parametrize("hk,hv,dk,dv,dtype", [(1, 1, 64, 16, BF), (2, 4, 128, 128, BF), (1, 3, 64, 80, HF), (2, 2, 256, 48, BF), (1, 2, 128, 256, HF)])
@pytest.mark.parametrize("layers,in_place", [(1, True), (3, False), (2, True)])
def test_commit_of_paths(hk, hv, dk, dv, dtype, layers, in_place):
    rng = np.random.default_rng(dk + dv + layers)
    ly = Layer(rng, hk, hv, dk, dv, 4, dtype)
    lengths, base = [16, 5, 1, 7, 16, 4, 3, 6], [0, 31, 9, 100, 6000000000, 2, 8, 50]
    paths = [[0, 2, 8, 9, 10], [0, 1, 2], [0], [], list(range(16)), [0, 2, 2, 3], [0, 7], [1, -1, 2]]
    committed = [4, 2, 0, -1, 1 << 30, 3, 5, 2]
    kept = [[0, 2, 8, 9, 10], [0, 1, 2], [0], [], list(range(16)), [0, 2], [0], [1]]
    paths.append([0, 1, 2, 3])                    # a stop: fewer committed than accepted
    lengths.append(5), base.append(12), committed.append(1), kept.append([0, 1])
    off, n, T = offsets_of(lengths), len(lengths), sum(lengths)
    row = hv * dv + hk * dk + hv
    rec_stride, ring_stride, state_stride = T * row + 3, n * RING * ly.C + 8, n * hv * dv * dk + 4
    record = rng.standard_normal((layers, rec_stride)).astype(np.float32)
    a, b = T * hv * dv, T * hk * dk
    record[:, a + b:a + b + T * hv] = -rng.random((layers, T * hv))
    record[:, a + b] = -np.inf                    # row 0 of sequence 0 forgets everything
    ring = to_bits(rng.standard_normal((layers, ring_stride)), dtype)
    state = rng.standard_normal((layers, state_stride)).astype(np.float32)
    state[:, :hv * dv * dk] = np.nan              # sequence 0 stands at base 0
    dres, drec, dring, dstate, dbase = _results(paths, committed), Dev(record), Dev(ring), Dev(state), Dev(np.array(base, np.int64))
    dring2, dstate2 = (dring, dstate) if in_place else (Dev(np.full_like(ring, 0x1234)), Dev(np.full_like(state, 3.0)))
    io = ts.GdnCommit(n_layers=layers, results=dres.ptr, record=drec.ptr, record_stride=4 * rec_stride, ring_in=dring.ptr, ring_out=dring2.ptr,
                      ring_stride=ring_stride, state_in=dstate.ptr, state_out=dstate2.ptr, state_stride=state_stride)
    ly.gpu.commit(ly.gpu.batch(off, dbase.ptr), io)
    got, got_ring = dstate2.get(), dring2.get()
    want_ring = ring.copy() if in_place else np.full_like(ring, 0x1234)
    for l in range(layers):
        for s in range(n):
            S = state[l, :n * hv * dv * dk].reshape(n, hv, dv, dk)[s].astype(np.float64)
            if base[s] == 0:
                S = np.zeros_like(S)
            for p in kept[s]:
                r = off[s] + p
                u, k, g = record[l, :a].reshape(T, hv, dv)[r], record[l, a:a + b].reshape(T, hk, dk)[r], record[l, a + b:a + b + T * hv].reshape(T, hv)[r]
                S = np.exp(g.astype(np.float64))[:, None, None] * S + u[:, :, None].astype(np.float64) * np.repeat(k, ly.rep, 0)[:, None, :]
            have = got[l, :n * hv * dv * dk].reshape(n, hv, dv, dk)[s]
            assert np.abs(have - S).max() <= 2.0 ** -19 * max(1.0, np.abs(S).max()), (l, s)   # f32 sums of up to 17 products
            rows_in, rows_out = (t[l, :n * RING * ly.C].reshape(n, RING, ly.C)[s] for t in (ring, want_ring))
            for i, p in enumerate(kept[s]):
                rows_out[(base[s] + i) % RING] = rows_in[(base[s] + p) % RING]
        tail = got[l, n * hv * dv * dk:]
        assert np.array_equal(tail, state[l, n * hv * dv * dk:] if in_place else np.full_like(tail, 3.0))
    assert np.array_equal(got_ring, want_ring)


# ---- together --------------------------------------------------------------------------------------------------------------------

def test_a_verify_loop_of_two_layers_in_one_graph():
    """Prompt (convolution, blocks), then rounds of: a tree step in two recurrent layers, the greedy acceptance of one target's logits,
    one commit for both layers along the acceptance's result -- the rounds as one captured graph, replayed -- against the recurrence
    over the accepted rows alone."""
    rng = np.random.default_rng(21)
    layers = [Layer(rng, 2, 4, 64, 32, 4, BF) for _ in range(2)]
    ly, n0, m, vocab = layers[0], 70, 9, 256
    parent = TREE16[:m]
    prompt = [to_bits(rng.standard_normal((n0, ly.C)), BF) for _ in layers]
    gates = [[to_bits(rng.standard_normal((n0, 4)), BF) for _ in range(2)] for _ in layers]
    per_state, per_ring = 4 * 32 * 64, RING * ly.C
    state, ring = Dev(np.zeros((2, per_state), np.float32)), Dev(np.zeros((2, per_ring), np.uint16))
    base = Dev(np.array([0], np.int64))
    pb = ly.gpu.batch([0, n0], base.ptr)
    ws = hip.DeviceBuffer(ly.gpu.prefill_workspace(pb))
    keep = []
    for i, l in enumerate(layers):
        x, a, b = Dev(prompt[i]), Dev(gates[i][0]), Dev(gates[i][1])
        rows, g, be, out = Dev(np.zeros_like(prompt[i])), Dev(np.zeros((n0, 4), np.float32)), Dev(np.zeros((n0, 4), np.float32)), Dev(np.zeros((n0, 128), np.uint16))
        l.gpu.conv(pb, ts.GdnConv(qkv=x.ptr, qkv_stride=ly.C, a=a.ptr, b=b.ptr, gate_stride=4, ring_in=ring.ptr + 2 * per_ring * i, ring_out=ring.ptr + 2 * per_ring * i, out=rows.ptr,
                                  out_stride=ly.C, g=g.ptr, beta=be.ptr))
        s = state.ptr + 4 * per_state * i
        l.gpu.prefill(pb, ts.GdnPrefill(q=rows.ptr, k=rows.ptr + 256, v=rows.ptr + 512, q_stride=ly.C, k_stride=ly.C, v_stride=ly.C, g=g.ptr,
                                        beta=be.ptr, state_in=s, state_out=s, out=out.ptr, out_stride=128, workspace=ws.ptr, workspace_bytes=ws.nbytes))
        keep += [x, a, b, rows, g, be, out]
    # what the recurrence makes of the prompt
    want, hist = [], []
    for i, l in enumerate(layers):
        S = np.zeros((4, 32, 64))
        x = from_bits(prompt[i], BF)
        q, k, v = l.convolved(x, np.zeros((RING, ly.C)), 0, chain(n0))
        g, be = l.gates(from_bits(gates[i][0], BF), from_bits(gates[i][1], BF))
        for r in range(n0):
            S, _, _ = l.row(S, q[r], k[r], v[r], g[r], be[r])
        got = state.get()[i].reshape(S.shape)
        assert rel2(got, S) <= 4 * 2.0 ** -8             # (unit q, unit k and v were rounded to bf16 on the way)
        want.append(got.astype(np.float64))              # the rounds are judged from the state that is there
        hist.append([x[r] for r in range(n0)])
    # the round's buffers
    stream = hip.Stream()
    x, a, b = (Dev(np.zeros((2, m, w), np.uint16)) for w in (ly.C, 4, 4))
    out, logits = Dev(np.zeros((2, m, 128), np.uint16)), Dev(np.zeros((m, vocab), np.uint16))
    dpar = Dev(np.array(parent, np.int32))
    rec_bytes = ly.gpu.record_bytes(m)
    record, result = Dev(np.zeros((2, rec_bytes // 4), np.float32)), Dev(np.zeros((28,), np.int32))
    batch = ly.gpu.batch([0, m], base.ptr, dpar.ptr)
    feed, par = np.arange(m, dtype=np.int32), np.array(parent, np.int32)
    steps = [ts.GdnStep(qkv=x.ptr + 2 * m * ly.C * i, qkv_stride=ly.C, a=a.ptr + 8 * m * i, b=b.ptr + 8 * m * i, gate_stride=4,
                        ring=ring.ptr + 2 * per_ring * i, state_in=state.ptr + 4 * per_state * i, record=record.ptr + rec_bytes * i,
                        out=out.ptr + 256 * m * i, out_stride=128) for i in range(2)]
    commit = ts.GdnCommit(n_layers=2, results=result.ptr, record=record.ptr, record_stride=rec_bytes, ring_in=ring.ptr, ring_out=ring.ptr,
                          ring_stride=per_ring, state_in=state.ptr, state_out=state.ptr, state_stride=per_state)

    def round_(s):
        for l, io in zip(layers, steps):
            l.gpu.step(batch, io, s.h)
        ffi.check(ffi.lib().tsv_accept_greedy_noalloc(s.h, logits.ptr, vocab, feed.ctypes.data, par.ctypes.data, m, 0, None, 0, 0, 0, result.ptr))
        ly.gpu.commit(batch, commit, s.h)

    scores = np.zeros((m, vocab), np.float16)
    # the acceptance's first call on a device asks for an address, outside capture
    ffi.check(ffi.lib().tsv_accept_greedy_noalloc(None, logits.ptr, vocab, feed.ctypes.data, par.ctypes.data, m, 0, None, 0, 0, 0, result.ptr))
    hip.check(hip.rt().hipDeviceSynchronize(), "sync")
    graph = hip.CapturedGraph(stream, round_)
    position = n0
    for turn, path in enumerate([[0, 1, 5, 6, 7], [0], [0, 2, 8], [0, 3], [0, 4]]):
        fresh = [to_bits(rng.standard_normal((2, m, w)), BF) for w in (ly.C, 4, 4)]
        for d, f in zip((x, a, b), fresh):
            d.put(f)
        base.put(np.array([position], np.int64))
        scores[:] = 0
        for slot in range(m):
            scores[slot, vocab - 1] = 1.0                # no child is wanted ..
        for here, there in zip(path, path[1:]):
            scores[here, feed[there]] = 2.0              # .. but along the path
        logits.put(scores.view(np.uint16))
        graph.launch()
        stream.sync()
        got, rows, kept = state.get(), out.get(), result.get()
        assert list(kept[6:6 + kept[23]]) == path, (turn, list(kept))
        for i, l in enumerate(layers):
            xs = from_bits(fresh[0][i], BF)
            ringed = np.zeros((RING, ly.C))
            for back in range(1, 4):
                ringed[(position - back) % RING] = hist[i][position - back]
            q, k, v = l.convolved(xs, ringed, position, parent)
            g, be = l.gates(from_bits(fresh[1][i], BF), from_bits(fresh[2][i], BF))
            at = {-1: want[i]}
            for slot in range(m):
                at[slot], _, o = l.row(at[parent[slot]], q[slot], k[slot], v[slot], g[slot], be[slot])
                assert rel2(from_bits(rows[i, slot], BF), o.reshape(-1)) <= 2.0 ** -8 + STATE, (turn, i, slot)
            want[i] = at[path[-1]]
            assert rel2(got[i].reshape(want[i].shape), want[i]) <= STATE * (turn + 1), (turn, i)
            hist[i] += [xs[slot] for slot in path]
        position += len(path)
