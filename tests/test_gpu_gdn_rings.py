"""Rings in two buffers: a ring_out that holds a copy of ring_in before a call serves the next call as one updated in place does."""
import numpy as np
import pytest

import turbospark_amd as ts
from tests.gdn_common import Dev, Layer, from_bits, half_step, offsets_of, rel2, to_bits
from tests.test_gpu_gdn import Step, _results, _ring

pytestmark = pytest.mark.gpu
BF, HF = ts.BF16, ts.F16


def _next_step(rng, ly, base, ring):
    """A step of two rows a sequence from a ring in device memory: its rows, and what the recurrence makes of the ring's rows."""
    p = Step(rng, ly, [2] * len(base), base, gated=False)
    p.ring = ring.get().copy()
    p.io.ring = ring.ptr
    p.io.record = p.record.ptr
    ly.gpu.step(p.batch, p.io)
    return from_bits(p.out.get()[:p.T, :ly.hv * ly.dv], ly.dtype), p.want()[0]


@pytest.mark.parametrize("dtype", [BF, HF])
def test_short_prompts_into_another_ring(dtype):
    lengths, base = [0, 1, 2, 3, 5, 0], [7, 40, 31, 1, 100, 0]
    steps = []
    for in_place in (True, False):
        rng = np.random.default_rng(31)
        ly = Layer(rng, 1, 2, 64, 32, 4, dtype)
        off, n, T = offsets_of(lengths), len(lengths), sum(lengths)
        x, a = to_bits(rng.standard_normal((T, ly.C)), dtype), to_bits(rng.standard_normal((T, 2)), dtype)
        ring = _ring(rng, ly, n, base)
        dx, da, din, dbase = Dev(x), Dev(a), Dev(ring), Dev(np.array(base, np.int64))
        dout = din if in_place else Dev(ring)
        out, g, be = Dev(np.zeros_like(x)), Dev(np.zeros((T, 2), np.float32)), Dev(np.zeros((T, 2), np.float32))
        ly.gpu.conv(ly.gpu.batch(off, dbase.ptr), ts.GdnConv(qkv=dx.ptr, qkv_stride=ly.C, a=da.ptr, b=da.ptr, gate_stride=2, ring_in=din.ptr,
                                                             ring_out=dout.ptr, out=out.ptr, out_stride=ly.C, g=g.ptr, beta=be.ptr))
        if not in_place:
            assert np.array_equal(din.get(), ring)
        behind = [b + m for b, m in zip(base, lengths)]
        steps.append(_next_step(rng, ly, behind, dout))
        # the recurrence from the rows themselves, not from what the ring holds
        want = ring.copy()
        for s in range(n):
            for i in range(lengths[s]):
                want[s, (base[s] + i) % 32] = x[off[s] + i]
        got = dout.get()
        for s in range(n):
            for back in range(1, min(3, behind[s]) + 1):
                assert np.array_equal(got[s, (behind[s] - back) % 32], want[s, (behind[s] - back) % 32]), (s, back)
    (rows, o), (other, _) = steps
    assert np.array_equal(rows, other) and rel2(rows, o) <= half_step(dtype) + 2.0 ** -15


@pytest.mark.parametrize("paths", [[[0], [0], [0]], [[0, 2, 8], [], [0, 1]]])
def test_a_round_with_few_kept_rows_into_another_ring(paths):
    """The rows behind the kept ones, which the next step reads, lie in ring_out too."""
    steps = []
    for in_place in (True, False):
        rng = np.random.default_rng(32)
        ly = Layer(rng, 2, 4, 64, 32, 4, HF)
        base = [9, 64, 31]
        p = Step(rng, ly, [9, 5, 3], base, tree=True, gated=False)
        p.io.record = p.record.ptr
        ly.gpu.step(p.batch, p.io)
        before = p.dring.get().copy()
        dout, res = p.dring if in_place else Dev(before), _results(paths)
        ly.gpu.commit(p.batch, ts.GdnCommit(n_layers=1, results=res.ptr, record=p.record.ptr, ring_in=p.dring.ptr, ring_out=dout.ptr,
                                            state_in=p.din.ptr, state_out=p.dnew.ptr))
        behind = [b + len(q) for b, q in zip(base, paths)]
        ring = dout.get()
        for s in range(3):
            rows = [before[s, (base[s] - j) % 32] for j in (3, 2, 1)] + [p.x[p.off[s] + i] for i in paths[s]]
            for back in range(1, 4):
                assert np.array_equal(ring[s, (behind[s] - back) % 32], rows[-back]), (s, back)
        steps.append(_next_step(rng, ly, behind, dout))
    (rows, o), (other, _) = steps
    assert np.array_equal(rows, other) and rel2(rows, o) <= half_step(HF) + 2.0 ** -15
