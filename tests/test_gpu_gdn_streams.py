"""The recurrent operators on every kind of stream handle that HIP has."""
import numpy as np
import pytest

import turbospark_amd as ts
from turbospark_amd import hip
from tests.gdn_common import Dev, Layer, to_bits
from tests.test_gpu_gdn import Prompt, Step, _results

pytestmark = pytest.mark.gpu
LEGACY, PER_THREAD = 1, 2


@pytest.mark.parametrize("handle", [LEGACY, PER_THREAD])
def test_the_runtimes_own_stream_handles(handle):
    rng = np.random.default_rng(51)
    ly = Layer(rng, 1, 2, 64, 32, 4, ts.BF16)
    x, a = to_bits(rng.standard_normal((5, ly.C)), ts.BF16), to_bits(rng.standard_normal((5, 2)), ts.BF16)
    p, q = Prompt(rng, ly, [70, 3], [0, 4]), Step(rng, ly, [5, 2], [9, 0])
    q.io.record = q.record.ptr
    res, base = _results([[0, 1], [0]]), Dev(np.array([3], np.int64))
    got = []
    for stream in (None, handle):
        dx, da, dr, out = Dev(x), Dev(a), Dev(np.zeros((1, 32, ly.C), np.uint16)), Dev(np.zeros_like(x))
        g, be, ring = Dev(np.zeros((5, 2), np.float32)), Dev(np.zeros((5, 2), np.float32)), Dev(q.ring)
        q.io.ring = ring.ptr
        hip.check(hip.rt().hipDeviceSynchronize(), "sync")
        ly.gpu.conv(ly.gpu.batch([0, 5], base.ptr), ts.GdnConv(qkv=dx.ptr, qkv_stride=ly.C, a=da.ptr, b=da.ptr, gate_stride=2, ring=dr.ptr,
                                                               out=out.ptr, out_stride=ly.C, g=g.ptr, beta=be.ptr), stream)
        ly.gpu.prefill(p.batch, p.io, stream)
        ly.gpu.step(q.batch, q.io, stream)
        ly.gpu.commit(q.batch, ts.GdnCommit(n_layers=1, results=res.ptr, record=q.record.ptr, ring_in=ring.ptr, ring_out=ring.ptr, state_in=q.din.ptr,
                                            state_out=q.dnew.ptr), stream)
        hip.check(hip.rt().hipDeviceSynchronize(), "sync")
        got.append([d.get() for d in (out, g, be, dr, p.out, p.dout, q.out, q.record, ring, q.dnew)])
        p.out.put(np.full_like(p.out.a, 0x1234))
        q.out.put(np.full_like(q.out.a, 0x1234))
    for first, second in zip(*got):
        assert np.array_equal(first, second)
