"""What tsv_gdn_* refuse before any device call, and their host arithmetic: no GPU needed."""
import ctypes as C

import numpy as np
import pytest

import turbospark_amd as ts
from turbospark_amd import ffi

P = 1 << 20          # stands for a device address: nothing here gets as far as reading it
INVALID, UNSUPPORTED = -1, -3


def _layer(**over):
    f = dict(n_k_heads=2, n_v_heads=4, k_dim=64, v_dim=32, conv_width=4, dtype=ts.BF16, scale=0.0, l2_eps=1e-6, norm_eps=1e-6,
             conv=P, a_log=P, dt_bias=P, norm=P)
    f.update(over)
    return ffi.GdnLayer(**f)


def _batch(offsets=(0, 3), **over):
    off = (C.c_int32 * len(offsets))(*offsets)
    f = dict(n_seq=len(offsets) - 1, offsets=off, base=P, parent=None)
    f.update(over)
    b = ffi.GdnBatch(**f)
    b.keep = off
    return b


CH = 2 * 2 * 64 + 4 * 32
IO = {
    "conv": lambda: ffi.GdnConv(qkv=P, qkv_stride=CH, a=P, b=P, gate_stride=4, ring_in=P, ring_out=P, out=2 * P, out_stride=CH, g=P, beta=P),
    "prefill": lambda: ffi.GdnPrefill(q=P, k=P, v=P, q_stride=128, k_stride=128, v_stride=128, g=P, beta=P, z=P, z_stride=128,
                                      state_in=P, state_out=P, out=2 * P, out_stride=128, workspace=P, workspace_bytes=1 << 30),
    "step": lambda: ffi.GdnStep(qkv=P, qkv_stride=CH, a=P, b=P, gate_stride=4, z=P, z_stride=128, ring=P, state_in=P, state_out=P,
                                record=P, out=2 * P, out_stride=128),
    "commit": lambda: ffi.GdnCommit(n_layers=2, results=P, record=P, record_stride=1 << 20, ring_in=P, ring_out=P, ring_stride=1 << 20,
                                    state_in=P, state_out=P, state_stride=1 << 20),
}


def _call(what, layer=None, batch=None, io=None):
    ref = lambda x: C.byref(x) if x is not None else None  # noqa: E731
    return getattr(ffi.lib(), "tsv_gdn_" + what)(None, ref(layer), ref(batch), ref(io))


@pytest.mark.parametrize("what", sorted(IO))
def test_descriptions_are_refused_by_name(what):
    refused = [
        (INVALID, "null", dict(layer=None)), (INVALID, "null", dict(batch=None)), (INVALID, "null", dict(io=None)),
        (INVALID, "heads", dict(layer=_layer(n_v_heads=3))), (INVALID, "heads", dict(layer=_layer(n_k_heads=0))),
        (INVALID, "heads", dict(layer=_layer(n_k_heads=2, n_v_heads=2048))),
        (UNSUPPORTED, "k_dim", dict(layer=_layer(k_dim=96))), (UNSUPPORTED, "v_dim", dict(layer=_layer(v_dim=24))),
        (UNSUPPORTED, "v_dim", dict(layer=_layer(v_dim=272))), (UNSUPPORTED, "rows", dict(layer=_layer(dtype=ts.F32))),
        (UNSUPPORTED, "taps", dict(layer=_layer(conv_width=5))), (UNSUPPORTED, "taps", dict(layer=_layer(conv_width=0))),
        (INVALID, "epsilon", dict(layer=_layer(l2_eps=float("nan")))), (INVALID, "epsilon", dict(layer=_layer(norm_eps=-1.0))),
        (INVALID, "batch", dict(batch=_batch(base=None))), (INVALID, "batch", dict(batch=_batch(offsets=(0, 3), base=P + 4))),
        (INVALID, "256 sequences", dict(batch=_batch(n_seq=0))), (INVALID, "256 sequences", dict(batch=_batch(offsets=[0] * 258))),
        (INVALID, "start at 0", dict(batch=_batch(offsets=(1, 3)))), (INVALID, "decrease", dict(batch=_batch(offsets=(0, 3, 2)))),
    ]
    for code, text, over in refused:
        given = dict(layer=_layer(), batch=_batch(), io=IO[what]())
        given.update(over)
        assert _call(what, **given) == code, (text, over)
        assert text in ffi.last_error() and "gdn_" + what in ffi.last_error(), ffi.last_error()


@pytest.mark.parametrize("what,fields", [
    ("conv", dict(qkv=None)), ("conv", dict(qkv=P + 8)), ("conv", dict(qkv_stride=CH - 8)), ("conv", dict(qkv_stride=CH + 4)),
    ("conv", dict(out=P)), ("conv", dict(out_stride=8)), ("conv", dict(ring_in=None)), ("conv", dict(ring_out=None)),
    ("conv", dict(ring_in=P + 2)), ("conv", dict(ring_out=P + 2)), ("conv", dict(ring_out=P + 64)), ("conv", dict(gate_stride=3)),
    ("conv", dict(a=None)), ("conv", dict(g=None)), ("conv", dict(beta=None)),
    ("prefill", dict(q=None)), ("prefill", dict(k=P + 2)), ("prefill", dict(v_stride=120)), ("prefill", dict(out=P)),
    ("prefill", dict(state_in=None)), ("prefill", dict(state_out=P + 64)), ("prefill", dict(workspace=None)),
    ("prefill", dict(workspace_bytes=100)), ("prefill", dict(workspace=P + 4)), ("prefill", dict(z_stride=4)), ("prefill", dict(g=None)),
    ("step", dict(qkv=None)), ("step", dict(out=2 * P + 2)), ("step", dict(state_in=None)), ("step", dict(state_out=P + 64)),
    ("step", dict(z=P + 4)), ("step", dict(ring=None)), ("step", dict(b=None)), ("step", dict(record=P + 2)),
    ("commit", dict(n_layers=0)), ("commit", dict(results=None)), ("commit", dict(results=P + 4)), ("commit", dict(record=None)),
    ("commit", dict(ring_out=P + 64)), ("commit", dict(state_out=P + 64)), ("commit", dict(state_stride=8)), ("commit", dict(ring_stride=8)),
    ("commit", dict(record_stride=16)), ("commit", dict(record_stride=(1 << 20) + 2)), ("commit", dict(state_in=None)),
])
def test_buffers_are_refused_by_name(what, fields):
    io = IO[what]()
    for k, v in fields.items():
        setattr(io, k, v)
    assert _call(what, _layer(), _batch(), io) == INVALID
    assert "gdn_" + what in ffi.last_error()


def test_rows_beyond_a_pass_and_trees_out_of_place_are_refused():
    assert _call("step", _layer(), _batch(offsets=(0, 17)), IO["step"]()) == INVALID and "16 rows" in ffi.last_error()
    assert _call("commit", _layer(), _batch(offsets=(0, 4, 21)), IO["commit"]()) == INVALID and "16 rows" in ffi.last_error()
    assert _call("step", _layer(), _batch(parent=P), IO["step"]()) == INVALID and "tree" in ffi.last_error()
    for what in ("conv", "prefill"):
        assert _call(what, _layer(), _batch(parent=P), IO[what]()) == INVALID and "chains" in ffi.last_error()
    for what in ("conv", "step"):
        assert _call(what, _layer(conv=None), _batch(), IO[what]()) == INVALID and "null" in ffi.last_error()
    for what in ("prefill", "step"):
        assert _call(what, _layer(norm=None), _batch(), IO[what]()) == INVALID and "null" in ffi.last_error()


def test_sizes_of_workspace_and_record():
    L = ffi.lib()
    one = L.tsv_gdn_prefill_workspace(C.byref(_layer()), C.byref(_batch(offsets=(0, 64))))
    assert one > 0
    assert L.tsv_gdn_prefill_workspace(C.byref(_layer()), C.byref(_batch(offsets=(0, 65)))) == 2 * one
    assert L.tsv_gdn_prefill_workspace(C.byref(_layer()), C.byref(_batch(offsets=(0, 1, 1, 2)))) == 2 * one
    assert L.tsv_gdn_prefill_workspace(C.byref(_layer()), C.byref(_batch(offsets=(0, 0)))) > 0
    assert L.tsv_gdn_prefill_workspace(C.byref(_layer(k_dim=65)), C.byref(_batch())) == -1 and "k_dim" in ffi.last_error()
    # beyond 32 bits: a long prompt of many heads
    many = _layer(n_k_heads=64, n_v_heads=64, k_dim=256)
    assert L.tsv_gdn_prefill_workspace(C.byref(many), C.byref(_batch(offsets=(0, 1 << 22)))) > 1 << 34
    assert L.tsv_gdn_record_bytes(C.byref(_layer()), 5) == 4 * 5 * (4 * 32 + 2 * 64 + 4)
    assert L.tsv_gdn_record_bytes(C.byref(_layer()), -1) == -1
    with pytest.raises(ffi.TsvError):
        ts.GatedDelta(2, 3, 64, 32, 4, ts.BF16).record_bytes(1)
    with pytest.raises(ValueError):
        ts.GatedDelta(2, 4, 64, 32, 4, ts.BF16).batch([0], P)


def test_struct_layouts_match_the_header():
    assert C.sizeof(ffi.GdnLayer) == 9 * 4 + 4 + 4 * 8 and C.sizeof(ffi.GdnBatch) == 4 * 8
    assert (C.sizeof(ffi.GdnConv), C.sizeof(ffi.GdnPrefill), C.sizeof(ffi.GdnStep), C.sizeof(ffi.GdnCommit)) == (88, 128, 104, 80)
    assert np.dtype(np.int32).itemsize * 28 == C.sizeof(ffi.RoundResultC)


def test_one_ring_stands_for_both():
    """A convolution that updates its ring in place names it once; what names one and both at once is refused."""
    io = ffi.GdnConv(qkv=P, ring=3 * P, out=2 * P)
    assert io.ring_in == io.ring_out == io.ring == 3 * P and io.qkv == P and io.out == 2 * P
    io.ring = 4 * P
    assert io.ring_in == io.ring_out == 4 * P
    io.ring_out = 5 * P
    assert io.ring is None and io.ring_in == 4 * P
    for twice in (dict(ring_in=P), dict(ring_out=P)):
        with pytest.raises(TypeError):
            ffi.GdnConv(ring=P, **twice)
    whole = IO["conv"]()
    whole.ring = P + 2
    assert _call("conv", _layer(), _batch(), whole) == INVALID and "rings" in ffi.last_error()
    whole.ring = None
    assert _call("conv", _layer(), _batch(), whole) == INVALID and "null" in ffi.last_error()


def test_offsets_are_whole_numbers_that_fit():
    """What int32 cannot hold is refused, not taken for another row."""
    layer = ts.GatedDelta(2, 4, 64, 32, 4, ts.BF16)
    for good in ([0, 3, 3], (0, 5), np.array([0, 7], np.int64), np.array([0, 7], np.uint8), np.array([0.0, 3.0])):
        b = layer.batch(good, P)
        assert [b.c.offsets[i] for i in range(len(good))] == list(good) and b.rows == good[-1]
    for bad in (np.array([0, (1 << 32) + 3]), np.array([0, 1 << 31]), [0, 1 << 40], [0.0, 2.5], [0.0, float("nan")], [0.0, float("inf")], [0, True, None], np.array([[0, 3]]),
                np.array([0, (1 << 64) - 1], np.uint64), [], 3):
        with pytest.raises(ValueError):
            layer.batch(bad, P)


def _segments(layer, offsets):
    """How many segments a batch is walked in, from what the workspace has beside its blocks' part: 0 where sequences are walked whole."""
    L = ffi.lib()
    size = lambda off: L.tsv_gdn_prefill_workspace(C.byref(layer), C.byref(_batch(offsets=off)))  # noqa: E731
    blocks = sum(-(-(b - a) // 64) for a, b in zip(offsets, offsets[1:]))
    more = size(offsets) - blocks * size((0, 64))
    state = 4 * layer.n_v_heads * layer.v_dim * layer.k_dim
    segment = 4 * layer.n_v_heads * (layer.v_dim + layer.k_dim) * layer.k_dim
    n = len(offsets) - 1                          # a sequence's last segment leaves nothing for others
    return (more - n * state) / segment + n if more else 0


def test_segments_go_by_the_long_sequences():
    few = _layer(n_k_heads=4, n_v_heads=8, k_dim=128, v_dim=128)
    assert _segments(few, (0, 32768)) == 8
    # short sequences beside the long one do not take it out of its segments
    assert _segments(few, (0, 32768, 32769)) == 9 and _segments(few, (0, 0, 0, 32768, 32768)) == 11
    assert _segments(few, (0, 130, 32768 + 130, 32768 + 200)) == 10
    # as many long ones as fill the compute units do, and so do more heads
    assert _segments(few, (0, 32768, 65536)) == 0 and _segments(few, (0, 32768, 32768 + 20000)) == 0
    assert _segments(_layer(n_k_heads=4, n_v_heads=16, k_dim=128, v_dim=128), (0, 32768)) == 0
    assert _segments(few, (0, 64 * 31)) == 0 and _segments(few, (0, 64 * 31 + 1)) > 0
    # one narrow head: no more segments than putting them together is worth
    narrow = _layer(n_k_heads=1, n_v_heads=1, k_dim=128, v_dim=16)
    assert 32 <= _segments(narrow, (0, 1 << 18)) <= 64
    assert _segments(narrow, (0, 4096)) <= 8
