"""The recurrent mixer row after row in 64 bits, and a layer with its buffers on the device, for the tests of tsv_gdn_*."""
import numpy as np

import turbospark_amd as ts
from turbospark_amd import hip

RING = 32
TREE16 = [-1, 0, 0, 0, 0, 1, 5, 6, 2, 8, 9, 3, 11, 12, 4, 14]


def to_bits(x, dtype):
    x = np.ascontiguousarray(x, np.float32)
    if dtype == ts.F16:
        return x.astype(np.float16).view(np.uint16)
    b = x.view(np.uint32)
    return ((b + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint16)


def from_bits(b, dtype):
    b = np.ascontiguousarray(b, np.uint16)
    if dtype == ts.F16:
        return b.view(np.float16).astype(np.float64)
    return (b.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def half_step(dtype):
    """The most a rounding to the rows' type is off, relative to the value."""
    return 2.0 ** -11 if dtype == ts.F16 else 2.0 ** -8


def rel2(got, want):
    return float(np.linalg.norm(got - want) / max(np.linalg.norm(want), 1e-300))


class Dev:
    """A numpy array's copy in device memory, `lead` bytes behind the start of its allocation."""

    def __init__(self, a, lead=0):
        self.a = np.ascontiguousarray(a)
        self.lead = lead
        self.buf = hip.DeviceBuffer(max(16, self.a.nbytes + lead))
        self.put(self.a)

    def put(self, a):
        a = np.ascontiguousarray(a)
        assert a.dtype == self.a.dtype and a.size == self.a.size
        if a.nbytes:
            hip.check(hip.rt().hipMemcpy(self.ptr, a.ctypes.data, a.nbytes, 1), "H2D")
        return self

    @property
    def ptr(self):
        return self.buf.ptr.value + self.lead

    def get(self):
        hip.check(hip.rt().hipDeviceSynchronize(), "sync")
        out = np.empty_like(self.a)
        if out.nbytes:
            hip.check(hip.rt().hipMemcpy(out.ctypes.data, self.ptr, out.nbytes, 2), "D2H")
        return out


def silu(x):
    return x / (1.0 + np.exp(-x))


def softplus(x):
    return np.logaddexp(x, 0.0)


class Layer:
    """Sizes and weights of one mixer, on the host and on the device."""

    def __init__(self, rng, hk, hv, dk, dv, taps=4, dtype=ts.BF16, scale=0.0):
        self.hk, self.hv, self.dk, self.dv, self.taps, self.dtype = hk, hv, dk, dv, taps, dtype
        self.C = 2 * hk * dk + hv * dv
        self.rep = hv // hk
        self.scale = scale if scale > 0 else dk ** -0.5
        self.conv = (0.5 * rng.standard_normal((self.C, taps))).astype(np.float32)
        self.a_log = np.log(1 + 15 * rng.random(hv)).astype(np.float32)
        self.dt_bias = (-4 + 2 * rng.random(hv)).astype(np.float32)
        self.norm = (1 + 0.1 * rng.standard_normal(dv)).astype(np.float32)
        self.dev = [Dev(x) for x in (self.conv, self.a_log, self.dt_bias, self.norm)]
        self.gpu = ts.GatedDelta(hk, hv, dk, dv, taps, dtype, *[d.ptr for d in self.dev], scale=scale)

    def heads(self, rows):
        kd = self.hk * self.dk
        return (rows[:, :kd].reshape(-1, self.hk, self.dk), rows[:, kd:2 * kd].reshape(-1, self.hk, self.dk),
                rows[:, 2 * kd:].reshape(-1, self.hv, self.dv))

    def convolved(self, x, ring, base, parent):
        """x: the raw rows of one sequence (f64), ring: its 32 rows.  Unit q, unit k, v."""
        y = np.zeros_like(x)
        for i in range(len(x)):
            at = i
            for j in range(self.taps):
                if at >= 0:
                    row = x[at]
                elif base + at >= 0:
                    row = ring[(base + at) % RING]
                else:
                    row = 0.0
                y[i] += row * self.conv[:, self.taps - 1 - j].astype(np.float64)
                at = parent[at] if at >= 0 else at - 1
        q, k, v = self.heads(silu(y))
        return tuple(t / np.sqrt((t * t).sum(-1, keepdims=True) + 1e-6) for t in (q, k)) + (v,)

    def gates(self, a, b):
        return -np.exp(self.a_log.astype(np.float64)) * softplus(a + self.dt_bias.astype(np.float64)), 1 / (1 + np.exp(-b))

    def row(self, S, q, k, v, g, beta):
        """One row through every head.  S: [hv][dv][dk].  The new state, u, o."""
        k, q = np.repeat(k, self.rep, 0), np.repeat(q, self.rep, 0)
        S = np.exp(g)[:, None, None] * S
        u = beta[:, None] * (v - np.einsum("hcd,hd->hc", S, k))
        S = S + u[:, :, None] * k[:, None, :]
        return S, u, self.scale * np.einsum("hcd,hd->hc", S, q)

    def gate(self, o, z):
        z = z.reshape(o.shape)
        return o / np.sqrt((o * o).mean(-1, keepdims=True) + 1e-6) * self.norm.astype(np.float64) * silu(z)


def chain(n):
    return list(range(-1, n - 1))


def offsets_of(lengths):
    return np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32)


def strided(rows, stride, fill=0x7FC1):
    """Rows in a wider buffer whose other values are no numbers, with one more row behind."""
    out = np.full((rows.shape[0] + 1, stride), fill, np.uint16)
    out[:-1, :rows.shape[1]] = rows
    return out
