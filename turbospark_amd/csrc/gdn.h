// What the kernels of a recurrent layer's mixer share: gdn.hip (convolution, few-row step, commit, the entry points) and
// gdn_prefill.hip (the rule over prompts).
#pragma once
#include "tsv_internal.h"

namespace tsv {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float gf4 __attribute__((ext_vector_type(4)));
typedef float uf4 __attribute__((ext_vector_type(4), aligned(4)));  // where only the 4-byte values are aligned

// The batch as a kernel gets it: the offsets by value, so that a launch needs no copy and no host memory.
struct GdnBatch {
    int32_t n_seq;
    const int64_t* base;
    const int32_t* parent;
    int32_t off[TSV_GDN_MAX_SEQ + 1];
};

struct GdnShape {
    int32_t hk, hv, rep, dv, taps, channels;
    float scale, l2_eps, norm_eps;
    const float *conv, *a_log, *dt_bias, *norm;
};

int gdn_check(const char* who, void* stream, const tsv_gdn_layer* l, const tsv_gdn_batch* b, int max_rows, GdnShape* sh, GdnBatch* kb);
int gdn_check_layer(const char* who, const tsv_gdn_layer* l, GdnShape* sh);
int gdn_refuse(const char* who, const char* what);
// The default stream's other handle (hipStreamLegacy) as the runtime's calls take it: hipStreamGetDevice reads through what it is given.
inline hipStream_t gdn_stream(void* stream) { return (hipStream_t)stream == hipStreamLegacy ? nullptr : (hipStream_t)stream; }
bool gdn_rows_ok(const void* p, int64_t stride, int64_t width);
bool gdn_overlap(const void* a, const void* b, size_t bytes);

// One row value: bf16 and fp16 bits to f32 and back (to nearest even).
template <bool F16>
__device__ __forceinline__ float row_f32(uint16_t b) {
    if constexpr (F16) return (float)__builtin_bit_cast(_Float16, b);
    return __uint_as_float((uint32_t)b << 16);
}
template <bool F16>
__device__ __forceinline__ uint16_t row_bits(float x) {
    if constexpr (F16) return __builtin_bit_cast(uint16_t, (_Float16)x);
    return __builtin_bit_cast(uint16_t, (__bf16)x);
}
template <bool F16>
__device__ __forceinline__ uint32_t row_pair(float x, float y) {
    typedef float f2 __attribute__((ext_vector_type(2)));
    if constexpr (F16) {
        typedef _Float16 h2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2{x, y}), h2));
    } else {
        typedef __bf16 b2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2{x, y}), b2));
    }
}
template <bool F16>
__device__ __forceinline__ void row8_f32(const uint4& u, float* x) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        x[2 * i] = row_f32<F16>((uint16_t)w[i]);
        x[2 * i + 1] = row_f32<F16>((uint16_t)(w[i] >> 16));
    }
}

// x as two bf16 terms: x - hi - lo is at most 2^-18 of x.  Products of two such pairs without the lo * lo part are 2^-16 to 2^-17
// off at the very most and 2^-19 on average (one term: 2^-9).  Of results that are rounded to 11 bits and fewer that leaves nothing; u and the
// state of a few-row step are 3e-7 to 1e-6 off by it, where three terms would leave 1e-7 and cost 0.5 us of 8.6.
__device__ __forceinline__ void split2(float x, __bf16& hi, __bf16& lo) {
    hi = (__bf16)x;
    lo = (__bf16)(x - (float)hi);
}

// two values at once: bits of (hi of x, hi of y) and of (lo of x, lo of y)
__device__ __forceinline__ void split2(float x, float y, uint32_t& hi, uint32_t& lo) {
    hi = row_pair<false>(x, y);
    lo = row_pair<false>(x - __uint_as_float(hi << 16), y - __uint_as_float(hi & 0xFFFF0000u));
}

// ... as three: what they leave out is 2^-27 of the value at most, less than f32 itself holds.  What a prompt's
// state is made of, block after block.
__device__ __forceinline__ void split3(float x, float y, uint32_t& hi, uint32_t& mid, uint32_t& lo) {
    hi = row_pair<false>(x, y);
    split2(x - __uint_as_float(hi << 16), y - __uint_as_float(hi & 0xFFFF0000u), mid, lo);
}

// a store that does not stay in the L2: it is on its way to memory while the kernel runs, not when it ends
__device__ __forceinline__ void store_through(void* to, gf4 x) { __builtin_nontemporal_store(x, (gf4*)to); }

__device__ __forceinline__ gf4 mfma_bf16(bf16x8 a, bf16x8 b, gf4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ gf4 mfma_f32(float a, float b, gf4 c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }

__device__ __forceinline__ float silu_f32(float x) { return x * __builtin_amdgcn_rcpf(1.0f + __expf(-x)); }
__device__ __forceinline__ float sigmoid_f32(float x) { return __builtin_amdgcn_rcpf(1.0f + __expf(-x)); }
// g = -e^a_log softplus(x), softplus(x) = max(x, 0) + log(1 + e^-|x|); log(1 + t) = 2 artanh(t / (2 + t)), whose series at t / (2 + t)
// <= 1/3 is 2^-24 off behind its seventh term: small t keep their bits and the code stays short
__device__ __forceinline__ float decay_of(float a_log, float x) {
    const float t = __expf(-fabsf(x)), s = t * __builtin_amdgcn_rcpf(2.0f + t), q = s * s;
    float y = fmaf(q, 1.0f / 13.0f, 1.0f / 11.0f);
    y = fmaf(q, y, 1.0f / 9.0f);
    y = fmaf(q, y, 1.0f / 7.0f);
    y = fmaf(q, y, 1.0f / 5.0f);
    y = fmaf(q, y, 1.0f / 3.0f);
    y = fmaf(q, y, 1.0f);
    return -__expf(a_log) * fmaf(2.0f * s, y, fmaxf(x, 0.0f));
}

// The sum of x over LANES neighbouring lanes (4, 8, 16 or 32), in all of them: lanes 1, 2, 7 - i and 15 - i apart, without LDS.
template <int LANES>
__device__ __forceinline__ float sum_lanes(float x) {
    x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0xB1, 0xF, 0xF, true));  // quad_perm 1 0 3 2
    x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x4E, 0xF, 0xF, true));  // quad_perm 2 3 0 1
    if constexpr (LANES >= 8) x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x141, 0xF, 0xF, true));   // row_half_mirror
    if constexpr (LANES >= 16) x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x140, 0xF, 0xF, true));  // row_mirror
    if constexpr (LANES >= 32) x += __shfl_xor(x, 16);
    return x;
}

// Two values to be summed over pairs of lanes 16 or 32 apart: the sum of x in the lower lane of the pair, that of y in the upper.
__device__ __forceinline__ float lane_pairs_by_16(float x, float y) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(y), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float lane_pairs_by_32(float x, float y) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(y), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// orders a wave's own LDS writes before its own later reads, where no other wave is involved
__device__ __forceinline__ void wave_lds_fence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// (I + A)^-1 of a strictly lower 16 x 16 matrix by one wave, both in LDS with rows of a multiple of four floats: the 8 x 8 halves on the
// diagonal row by row, a column a lane, both in the same instructions; then the block below, -T2 A21 T1, as two products of the f32
// instruction, whose D layout is its B operand's when the contraction takes rows 4 gq + r in step r.  second: whether rows 8 to 15 hold anything.
__device__ __forceinline__ void invert_lower16(const float* A, int as, float* T, int ts, int l16, int gq, bool second = true) {
    const int b = l16 & 8;
    const float* a = A + b * as + b;
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
        float v = i == (l16 & 7) ? 1.0f : 0.0f;
#pragma unroll
        for (int j = 0; j < i; j++) v = fmaf(-a[i * as + j], x[j], v);
        x[i] = v;
    }
    if (gq < 2) {
#pragma unroll
        for (int i = 0; i < 8; i++) T[((gq ? 8 - b : b) + i) * ts + l16] = gq ? 0.0f : x[i];
    }
    wave_lds_fence();
    if (!second) return;
    float4 r = *(const float4*)(A + l16 * as + 4 * gq);
    if (l16 < 8 || gq > 1) r = make_float4(0, 0, 0, 0);
    const float4 n = *(const float4*)(T + l16 * ts + 4 * gq);
    gf4 t, p = {0, 0, 0, 0}, y = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 4; i++) t[i] = T[(4 * gq + i) * ts + l16];
    p = mfma_f32(r.x, t[0], p);
    p = mfma_f32(r.y, t[1], p);
    p = mfma_f32(r.z, t[2], p);
    p = mfma_f32(r.w, t[3], p);
    y = mfma_f32(n.x, p[0], y);
    y = mfma_f32(n.y, p[1], y);
    y = mfma_f32(n.z, p[2], y);
    y = mfma_f32(n.w, p[3], y);
    if (gq > 1) {
#pragma unroll
        for (int i = 0; i < 4; i++) T[(4 * gq + i) * ts + l16] = t[i] - y[i];
    }
}

}  // namespace tsv
