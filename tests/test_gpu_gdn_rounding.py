"""What the prompts' rule (tsv_gdn_prefill) loses beside the one rounding of its results.

A result rounded once lies within half a step of the rows' type of what was rounded; how much further from the 64-bit recurrence it lies
(`excess`) is at most what the value was off before.  Of what a product of two-term operands adds at most 3 * 2^-18 is lost (2^-18 of
either operand and of the product of the two lower terms); three products one behind the other (k S, T r, P u) make 9 * 2^-18, and in the
2-norm, where these are of all signs, half of that: 2^-15 of a row's o at the most.  Under a gate y = o / r * w: o and the root r of its
mean square both, 2^-14; f32 sums and exponentials stay below 2^-17.  2^-13 is allowed, an eighth of what fp16 rows lose to a rounding of o
before the norm at the worst, 2^-11."""
import numpy as np
import pytest

import turbospark_amd as ts
from tests.gdn_common import Dev, Layer, from_bits, strided, to_bits
from tests.test_gpu_gdn import Prompt

pytestmark = pytest.mark.gpu
BF, HF = ts.BF16, ts.F16


def excess(got, want, dtype):
    """How far got lies from want beyond half a step of the rows' type."""
    bits, least = (11, -14) if dtype == HF else (8, -126)
    size = np.maximum(np.maximum(np.abs(got), np.abs(want)), 2.0 ** least)
    half = 2.0 ** (np.floor(np.log2(size)) - bits)
    return np.maximum(np.abs(got - want) - half, 0.0)


def sized(p, size):
    """The prompt's values and state, `size` times as large."""
    p.v = to_bits(from_bits(p.v, p.ly.dtype) * size, p.ly.dtype)
    p.state = (p.state * size).astype(np.float32)
    p.dv_.put(strided(p.v, p.io.v_stride))
    given = p.state.copy()
    for s in range(p.n):
        if p.base[s] == 0:
            given[s] = np.nan
    p.din.put(given)


def rows_of(p):
    p.ly.gpu.prefill(p.batch, p.io)
    width = p.ly.hv * p.ly.dv
    return from_bits(p.out.get()[:p.T, :width], p.ly.dtype), p.want()[0]


@pytest.mark.parametrize("hk,hv,dk,dv,lengths,size,scale", [
    (2, 4, 64, 64, [130, 65], 1.0, 0.0),
    (1, 2, 128, 48, [200], 4000.0, 64.0),         # o far above 65504
    (1, 2, 128, 48, [200], 2.0 ** -13, 0.0),      # o of fp16's subnormal numbers
    (2, 4, 64, 32, [2100], 4000.0, 64.0),         # in segments
    (4, 8, 128, 128, [70] * 8, 2.0 ** -13, 0.0),  # two column tiles a workgroup
    (1, 1, 256, 256, [70], 4000.0, 64.0),
])
def test_the_norm_takes_o_as_it_is(hk, hv, dk, dv, lengths, size, scale):
    rng = np.random.default_rng(dk + dv)
    p = Prompt(rng, Layer(rng, hk, hv, dk, dv, 4, HF, scale=scale), lengths, [s for s in range(len(lengths))], gated=True, pad=8)
    sized(p, size)
    rows, want = rows_of(p)
    assert np.isfinite(rows).all()
    off = excess(rows, want, HF)
    assert np.linalg.norm(off) <= 2.0 ** -13 * np.linalg.norm(want), np.linalg.norm(off) / np.linalg.norm(want)


def test_a_layer_without_norm_weights_needs_no_room_for_the_norm():
    rng = np.random.default_rng(1)
    ly = Layer(rng, 1, 2, 64, 32, 4, BF)
    p = Prompt(rng, ly, [200], [3], gated=False)
    bare = ts.GatedDelta(1, 2, 64, 32, 4, BF)
    room = bare.prefill_workspace(p.batch)
    assert room == ly.gpu.prefill_workspace(p.batch) - 4 * 64 * 2 * 32 * 4
    ly.gpu.prefill(p.batch, p.io)
    rows, S = p.check()
    p.ws = Dev(np.full(room // 4 + 4, 7.0, np.float32))
    p.io.workspace, p.io.workspace_bytes = p.ws.ptr, room
    p.out.put(np.full_like(p.out.a, 0x1234))
    bare.prefill(p.batch, p.io)
    assert np.array_equal(p.out.get(), rows) and np.array_equal(p.dout.get(), S) and (p.ws.get()[room // 4:] == 7).all()


@pytest.mark.parametrize("hk,hv,dk,dv,lengths,dtype", [
    (2, 4, 64, 64, [130, 65], BF),
    (1, 3, 128, 48, [200, 1, 64], BF),
    (2, 4, 128, 128, [300], HF),
    (1, 2, 64, 32, [2100], BF),                   # in segments
    (4, 8, 128, 128, [70] * 8, BF),               # two column tiles a workgroup
    (16, 80, 64, 16, [600], BF),                  # several value heads a workgroup
    (1, 1, 256, 256, [70], BF),
])
@pytest.mark.parametrize("gated", [True, False])
def test_rows_are_rounded_once(hk, hv, dk, dv, lengths, dtype, gated):
    rng = np.random.default_rng(dk + dv + 1)
    p = Prompt(rng, Layer(rng, hk, hv, dk, dv, 4, dtype), lengths, [s for s in range(len(lengths))], gated=gated, pad=8)
    rows, want = rows_of(p)
    off = excess(rows, want, dtype)
    assert np.linalg.norm(off) <= 2.0 ** -13 * np.linalg.norm(want), np.linalg.norm(off) / np.linalg.norm(want)


@pytest.mark.parametrize("hk,hv,dk,dv,lengths,dtype", [
    (2, 4, 64, 64, [130, 65], BF),
    (2, 4, 64, 64, [130, 65], HF),
    (1, 3, 128, 48, [700, 1, 64], BF),
    (1, 2, 128, 128, [300], HF),
    (1, 2, 64, 32, [2100], BF),                   # in segments
    (1, 1, 128, 48, [2111], HF),
    (1, 1, 256, 32, [2200], BF),
    (4, 8, 128, 128, [70] * 8, BF),               # two column tiles a workgroup
    (16, 80, 64, 16, [600], HF),                  # several value heads a workgroup
    (1, 1, 256, 256, [170], HF),
])
@pytest.mark.parametrize("decay", [0.1, 0.002])
def test_states_are_those_of_32_bits(hk, hv, dk, dv, lengths, dtype, decay):
    """What a block adds to the state in f32 is off by its sums of 64 to 256 products (2^-24 of what they have reached, of all signs: 16 *
    2^-25 = 2^-21 in the 2-norm), three one behind the other, by the inverse and by the exponentials (2^-22 each): 2^-20 together.  Blocks
    add up where nothing decays, but of all signs too, and the recurrence only contracts: 2^-20 is allowed.  Operands of two bf16 terms,
    2^-18 each, do not keep to it."""
    rng = np.random.default_rng(dk + dv + 2)
    p = Prompt(rng, Layer(rng, hk, hv, dk, dv, 4, dtype), lengths, [s for s in range(len(lengths))], gated=False)
    p.g = (-decay * rng.random(p.g.shape)).astype(np.float32)
    p.dg.put(np.concatenate([p.g, np.full((1, hv), np.nan, np.float32)]))
    p.ly.gpu.prefill(p.batch, p.io)
    S, want = p.dout.get(), p.want()[1]
    for s in range(p.n):
        off = np.linalg.norm(S[s] - want[s]) / np.linalg.norm(want[s])
        print("state off by 2^%.2f" % np.log2(off))
        assert off <= 2.0 ** -20, (s, off)
