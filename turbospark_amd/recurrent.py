"""The mixer of a recurrent (gated delta rule) layer: the host mirror of tsv_gdn_*.

Like the C entry points, these calls take device addresses of the caller's memory and the caller's stream (None: the default
stream) and return as soon as the work is enqueued.  A call's buffers and strides are a GdnConv / GdnPrefill / GdnStep /
GdnCommit, which a program with buffers of its own fills once and passes again."""
import ctypes as C

import numpy as np

from . import ffi


class Batch:
    """The rows of a call: sequence s owns rows [offsets[s], offsets[s + 1]); `base` (int64 per sequence) and `parent` (int32 per
    row, None: chains) are device addresses."""

    def __init__(self, offsets, base, parent=None):
        given = np.asarray(offsets)
        if given.ndim != 1 or given.size < 2:
            raise ValueError("offsets: one entry per sequence and one behind the last")
        if given.dtype.kind not in "iuf" or not all(-(1 << 31) <= x < 1 << 31 and x == int(x) for x in given.tolist()):
            raise ValueError("offsets: whole numbers of 32 bits")
        self._offsets = np.ascontiguousarray(given, np.int32)
        self.c = ffi.GdnBatch(self._offsets.size - 1, self._offsets.ctypes.data_as(C.POINTER(C.c_int32)), base, parent)
        self._ref = C.byref(self.c)
        self.rows = int(self._offsets[-1])


class GatedDelta:
    """One layer's head counts, widths and weights (device addresses of f32 vectors).  `dtype` (BF16 or F16) is that of all rows."""

    def __init__(self, k_heads, v_heads, k_dim, v_dim, conv_width, dtype, conv=None, a_log=None, dt_bias=None, norm=None, scale=0.0,
                 l2_eps=1e-6, norm_eps=1e-6):
        self.c = ffi.GdnLayer(k_heads, v_heads, k_dim, v_dim, conv_width, dtype, scale, l2_eps, norm_eps, conv, a_log, dt_bias, norm)
        self._ref = C.byref(self.c)
        self._lib = ffi.lib()
        self.channels = 2 * k_heads * k_dim + v_heads * v_dim

    def batch(self, offsets, base, parent=None):
        return Batch(offsets, base, parent)

    def conv(self, batch, io, stream=None):
        """Prompt rows through the convolution, SiLU and the unit vectors; their decays and betas; the rings' new rows."""
        ffi.check(self._lib.tsv_gdn_conv(stream, self._ref, batch._ref, C.byref(io)))

    def prefill_workspace(self, batch):
        """Bytes of workspace that prefill needs for this batch."""
        n = self._lib.tsv_gdn_prefill_workspace(self._ref, batch._ref)
        if n < 0:
            raise ffi.TsvError(-1, ffi.last_error())
        return n

    def prefill(self, batch, io, stream=None):
        """The delta rule over the prompts' rows, blocks of 64 at a time."""
        ffi.check(self._lib.tsv_gdn_prefill(stream, self._ref, batch._ref, C.byref(io)))

    def record_bytes(self, rows):
        """Bytes of the record that a verify step of `rows` rows leaves for commit."""
        n = self._lib.tsv_gdn_record_bytes(self._ref, rows)
        if n < 0:
            raise ffi.TsvError(-1, ffi.last_error())
        return n

    def step(self, batch, io, stream=None):
        """The whole mixer for up to sixteen rows a sequence: final rows (io.state_out) or rows under verification (io.record)."""
        ffi.check(self._lib.tsv_gdn_step(stream, self._ref, batch._ref, C.byref(io)))

    def commit(self, batch, io, stream=None):
        """commit_pending: the rows the acceptance kept go into the state, in all of io.n_layers layers."""
        ffi.check(self._lib.tsv_gdn_commit(stream, self._ref, batch._ref, C.byref(io)))
