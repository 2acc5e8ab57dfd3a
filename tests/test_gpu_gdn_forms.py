"""The recurrent mixer (tsv_gdn_*) at the shapes that its launch rules set apart: several value heads a workgroup, two column tiles,
segments of either, tiles of 32 rows, a norm of several launches.  Each test says by the rule that its shape is on that side."""
import ctypes as C

import numpy as np
import pytest

import turbospark_amd as ts
from turbospark_amd import hip
from tests.gdn_common import RING, Dev, Layer, chain, from_bits, half_step, offsets_of, to_bits
from tests.test_gpu_gdn import Prompt, _ring

pytestmark = pytest.mark.gpu
BF, HF = ts.BF16, ts.F16


def blocks_of(lengths):
    return [-(-n // 64) for n in lengths]


def several_heads_a_workgroup(ly, lengths):
    return ly.rep > 1 and sum(blocks_of(lengths)) * ly.hk >= 512


def two_column_tiles(ly, segments):
    return ly.dk < 256 and ly.dv % 32 == 0 and segments * ly.hv * ly.dv // 32 >= 256


def _ragged(seed, n, most):
    """n lengths from none to `most`, whole blocks and one row more or less among them."""
    rng = np.random.default_rng(seed)
    out = [int(v) for v in rng.integers(0, most + 1, n)]
    out[:6] = [0, 1, 63, 64, 65, most]
    return out


@pytest.mark.parametrize("hk,hv,dk,dv,dtype,lengths", [
    (16, 32, 64, 16, BF, _ragged(1, 45, 70)),
    (16, 48, 64, 16, HF, _ragged(2, 45, 66)),
    (16, 48, 128, 16, BF, _ragged(3, 40, 130)),
    (32, 64, 128, 16, HF, _ragged(4, 25, 66)),
    (16, 32, 256, 16, BF, _ragged(5, 40, 66)),
    (16, 80, 64, 16, BF, [2049]),
])
@pytest.mark.parametrize("gated", [True, False])
def test_several_value_heads_a_workgroup(hk, hv, dk, dv, dtype, lengths, gated):
    rng = np.random.default_rng(hv + dk)
    ly = Layer(rng, hk, hv, dk, dv, 4, dtype)
    assert several_heads_a_workgroup(ly, lengths)
    p = Prompt(rng, ly, lengths, [int(v) for v in rng.integers(0, 3, len(lengths))], gated=gated, pad=8)
    ly.gpu.prefill(p.batch, p.io)
    rows, S = p.check()
    p.io.state_out = p.io.state_in
    ly.gpu.prefill(p.batch, p.io)
    assert np.array_equal(p.out.get(), rows) and np.array_equal(p.din.get(), S)


@pytest.mark.parametrize("hk,hv,dk,dv,dtype,lengths", [
    (4, 8, 64, 32, BF, _ragged(6, 32, 140)),
    (4, 12, 64, 96, HF, _ragged(7, 8, 70)),
    (8, 16, 128, 64, BF, _ragged(8, 8, 200)),
    (4, 4, 128, 128, HF, _ragged(9, 16, 66)),
    (1, 2, 128, 32, BF, _ragged(10, 128, 65)),
    (2, 32, 64, 256, BF, [130]),
])
@pytest.mark.parametrize("gated", [True, False])
def test_two_column_tiles_a_workgroup(hk, hv, dk, dv, dtype, lengths, gated):
    rng = np.random.default_rng(hv + dv)
    ly = Layer(rng, hk, hv, dk, dv, 4, dtype)
    assert two_column_tiles(ly, len(lengths))
    p = Prompt(rng, ly, lengths, [int(v) for v in rng.integers(0, 3, len(lengths))], gated=gated, pad=8)
    ly.gpu.prefill(p.batch, p.io)
    rows, S = p.check()
    p.io.state_out = p.io.state_in
    ly.gpu.prefill(p.batch, p.io)
    assert np.array_equal(p.out.get(), rows) and np.array_equal(p.din.get(), S)


@pytest.mark.parametrize("hk,hv,dk,dv,dtype,rows,base,gated", [
    (8, 32, 64, 32, BF, 4097, 0, True),
    (8, 16, 64, 64, HF, 4500, 9, False),
    (4, 8, 128, 128, BF, 4200, 1, True),
])
def test_segments_with_two_column_tiles(hk, hv, dk, dv, dtype, rows, base, gated):
    """Eight segments of at least eight blocks each: a prompt alone, its 64 column tiles on a quarter of the compute units."""
    rng = np.random.default_rng(dk + dv)
    ly = Layer(rng, hk, hv, dk, dv, 4, dtype)
    assert hv * dv // 16 == 64 and blocks_of([rows])[0] >= 64 and two_column_tiles(ly, 8)
    p = Prompt(rng, ly, [rows], [base], gated=gated)
    ly.gpu.prefill(p.batch, p.io)
    got, S = p.check()
    p.io.state_out = p.io.state_in
    ly.gpu.prefill(p.batch, p.io)
    assert np.array_equal(p.out.get(), got) and np.array_equal(p.din.get(), S)


@pytest.mark.parametrize("hk,hv,dk,dv,taps,dtype,lengths,base", [
    (1, 3, 64, 16, 4, BF, [9001, 1, 0, 31, 33, 7400, 32, 2], [31, 7, 3, 0, 100, 1, 64, 2]),
    (1, 1, 128, 16, 3, HF, [16387], [5000000000]),
    (2, 6, 256, 256, 4, HF, [4101, 4099], [0, 30]),
])
def test_convolution_in_tiles_of_32_rows(hk, hv, dk, dv, taps, dtype, lengths, base):
    rng = np.random.default_rng(dk + taps)
    ly = Layer(rng, hk, hv, dk, dv, taps, dtype)
    off, n, T = offsets_of(lengths), len(lengths), sum(lengths)
    assert T * -(-ly.C // 2048) >= 32 * 512          # a workgroup has 2048 channels
    x, a, b = (to_bits(rng.standard_normal(s, np.float32), dtype) for s in ((T, ly.C), (T, hv), (T, hv)))
    ring = _ring(rng, ly, n, base)
    dx, da, db, dring, dbase = Dev(x), Dev(a), Dev(b), Dev(ring), Dev(np.array(base, np.int64))
    out, g, be = Dev(np.full((T + 1, ly.C), 0x1234, np.uint16)), Dev(np.full((T + 1, hv), 7.0, np.float32)), Dev(np.full((T + 1, hv), 7.0, np.float32))
    ly.gpu.conv(ly.gpu.batch(off, dbase.ptr), ts.GdnConv(qkv=dx.ptr, qkv_stride=ly.C, a=da.ptr, b=db.ptr, gate_stride=hv, ring=dring.ptr,
                                                         out=out.ptr, out_stride=ly.C, g=g.ptr, beta=be.ptr))
    rows, got_g, got_b, want_ring = out.get(), g.get(), be.get(), ring.copy()
    assert (rows[T] == 0x1234).all() and (got_g[T] == 7).all() and (got_b[T] == 7).all()
    for s in range(n):
        lo, hi = off[s], off[s + 1]
        q, k, v = ly.convolved(from_bits(x[lo:hi], dtype), from_bits(ring[s], dtype), base[s], chain(hi - lo))
        at = 0
        for t in (q, k, v):
            want = t.reshape(hi - lo, t.shape[1] * t.shape[2])
            err = np.abs(from_bits(rows[lo:hi, at:at + want.shape[1]], dtype) - want)
            # the f32 sums and exponentials of values up to a few: 2^-20; fp16 has no steps finer than 2^-25 below 2^-14
            assert (err <= half_step(dtype) * np.abs(want) * (1 + 2.0 ** -6) + 2.0 ** -20).all(), (s, err.max())
            at += want.shape[1]
        wg, wb = ly.gates(from_bits(a[lo:hi], dtype), from_bits(b[lo:hi], dtype))
        assert np.allclose(got_g[lo:hi], wg, rtol=2.0 ** -19, atol=0) and np.allclose(got_b[lo:hi], wb, rtol=2.0 ** -20, atol=0)
        for i in range(max(0, hi - lo - (taps - 1)), hi - lo):
            want_ring[s, (base[s] + i) % RING] = x[lo + i]
    assert np.array_equal(dring.get(), want_ring)


def test_a_norm_of_several_launches():
    """More than 2^26 heads' rows: every row keeps the state (beta 0) and reads it with a q of its own, so that each row behind the first
    launch's last is known by itself.  Value rows are not read for anything (beta 0) but are there; z is the same everywhere."""
    rng = np.random.default_rng(15)
    hv, dk, dv, extra = 1024, 64, 16, 70
    T = (1 << 26) // hv + extra
    ly = Layer(rng, 1, hv, dk, dv, 4, HF)
    q = rng.standard_normal((T, dk))
    q = to_bits(q / np.linalg.norm(q, axis=-1, keepdims=True), HF)
    state = (0.3 * rng.standard_normal((1, hv, dv, dk))).astype(np.float32)
    zero = {}
    for name, nbytes, byte in (("v", 2 * T * hv * dv, 0), ("g", 4 * T * hv, 0), ("beta", 4 * T * hv, 0), ("z", 2 * T * hv * dv, 0x3C), ("out", 2 * T * hv * dv, 0x11)):
        zero[name] = hip.DeviceBuffer(nbytes)
        hip.check(hip.rt().hipMemset(zero[name].ptr, C.c_int(byte), C.c_size_t(nbytes)), "memset")
    dq, dstate, dbase = Dev(q), Dev(state), Dev(np.array([5], np.int64))
    batch = ly.gpu.batch([0, T], dbase.ptr)
    ws = hip.DeviceBuffer(ly.gpu.prefill_workspace(batch))
    w = hv * dv
    ly.gpu.prefill(batch, ts.GdnPrefill(q=dq.ptr, k=dq.ptr, v=zero["v"].ptr.value, q_stride=dk, k_stride=dk, v_stride=w, g=zero["g"].ptr.value, beta=zero["beta"].ptr.value,
                                        z=zero["z"].ptr.value, z_stride=w, state_in=dstate.ptr, state_out=dstate.ptr, out=zero["out"].ptr.value, out_stride=w,
                                        workspace=ws.ptr, workspace_bytes=ws.nbytes))
    hip.check(hip.rt().hipDeviceSynchronize(), "sync")
    z = from_bits(np.full((1, w), 0x3C3C, np.uint16), HF)
    for row in (0, 63, T - extra - 1, T - extra, T - extra + 1, T - 1):
        got = np.empty(w, np.uint16)
        hip.check(hip.rt().hipMemcpy(got.ctypes.data, zero["out"].ptr.value + 2 * row * w, 2 * w, 2), "D2H")
        o = ly.scale * np.einsum("hcd,d->hc", state[0].astype(np.float64), from_bits(q[row], HF))
        want = ly.gate(o[None], z).reshape(-1)
        assert np.linalg.norm(from_bits(got, HF) - want) <= 4 * half_step(HF) * np.linalg.norm(want), row
    assert np.array_equal(dstate.get(), state)


@pytest.mark.parametrize("lengths", [[1, 2100, 0], [0, 0, 2049, 64, 1, 65, 3]])
def test_a_long_prompt_in_segments_beside_short_ones(lengths):
    rng = np.random.default_rng(len(lengths))
    ly = Layer(rng, 2, 8, 64, 128, 4, BF)
    assert len(lengths) * ly.hv * ly.dv // 16 > 64 >= ly.hv * ly.dv // 16 and max(blocks_of(lengths)) >= 32
    p = Prompt(rng, ly, lengths, [3 * (s % 2) for s in range(len(lengths))], gated=True)
    ly.gpu.prefill(p.batch, p.io)
    got, S = p.check()
    p.io.state_out = p.io.state_in
    ly.gpu.prefill(p.batch, p.io)
    assert np.array_equal(p.out.get(), got) and np.array_equal(p.din.get(), S)


@pytest.mark.parametrize("gated", [True, False])
def test_blocks_brought_into_the_cache_ahead(gated):
    """fp16 rows of k_dim 128 whose blocks' matrices are 128 MB and more: the walk has a ninth wave."""
    rng = np.random.default_rng(16)
    ly = Layer(rng, 32, 32, 128, 16, 4, HF)
    lengths = [900, 1300, 1, 64, 0]
    per_block = 32 * 3 * 128 // 8 * 2 * 1024 + 32 * 22 * 1024
    assert sum(blocks_of(lengths)) * per_block >= 128 << 20
    p = Prompt(rng, ly, lengths, [0, 3, 2, 0, 1], gated=gated)
    ly.gpu.prefill(p.batch, p.io)
    rows, S = p.check()
    p.io.state_out = p.io.state_in
    ly.gpu.prefill(p.batch, p.io)
    assert np.array_equal(p.out.get(), rows) and np.array_equal(p.din.get(), S)


@pytest.mark.parametrize("hk,hv,dk,dv,dtype,lengths", [
    (2, 8, 64, 128, BF, [1, 2100, 0]),              # segments, then the norm
    (4, 8, 64, 32, HF, _ragged(6, 32, 140)),        # two column tiles
])
def test_captured_calls_of_these_forms_replay(hk, hv, dk, dv, dtype, lengths):
    """Replayed with other inputs, the program's own calls between: the same bits as without a graph."""
    rng = np.random.default_rng(17)
    ly = Layer(rng, hk, hv, dk, dv, 4, dtype)
    base = [3 * (s % 2) for s in range(len(lengths))]
    a, b = (Prompt(rng, ly, lengths, base) for _ in range(2))
    alone = []
    for p in (a, b):
        ly.gpu.prefill(p.batch, p.io)
        alone.append((p.out.get(), p.dout.get()))
    stream = hip.Stream()
    graph = hip.CapturedGraph(stream, lambda s: ly.gpu.prefill(a.batch, a.io, s.h))
    for source in (b, a, b, b):
        for dst, src in ((a.dq, source.dq), (a.dk_, source.dk_), (a.dv_, source.dv_), (a.dg, source.dg), (a.db, source.db), (a.dz, source.dz), (a.din, source.din)):
            dst.put(src.a)
        graph.launch()
        stream.sync()
        rows, S = alone[0] if source is a else alone[1]
        assert np.array_equal(a.out.get(), rows) and np.array_equal(a.dout.get(), S)
        a.out.put(np.full_like(a.out.a, 0x1234))
        ly.gpu.prefill(b.batch, b.io)
        hip.check(hip.rt().hipDeviceSynchronize(), "sync")
