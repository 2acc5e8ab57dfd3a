// The mixer of a gated-delta-rule layer: the prompt's short convolution, the step of a few rows (decode and verify passes) and the
// commit of accepted rows; entry points and argument checks of those and of the rule over prompts (gdn_prefill.hip).  Formulas:
// include/tsverify.h.
#include "gdn.h"

#include <cstring>

namespace tsv {

// ---- the short convolution of prompt rows ---------------------------------------------------------------------------------
// A thread owns 8 neighbouring channels and walks a tile of rows, four at a time with the next four under way and the taps' rows in
// registers: every row is read once, conv_width - 1 of them again per tile.  The k_dim / 8 threads of a head are neighbours in a wave
// and sum its squares by lane moves.  Bound by memory (4 bytes a channel) and, close behind, by the exponential and the reciprocal of
// each SiLU.  Tiles have 32 rows, or 4 where 32 would leave compute units without a workgroup.  8192 rows of 8192 channels: 57 us, 4.7
// TB/s (60 where the rows stay in the L2 as they are stored); 299 rows of 1024: 4.8 us, the chain of loads.
constexpr int CONV_THREADS = 256;

struct ConvArgs {
    const uint16_t* qkv;
    int64_t qkv_stride;
    const uint16_t *a, *b;
    int64_t gate_stride;
    const uint16_t* ring_in;
    uint16_t* ring_out;
    uint16_t* out;
    int64_t out_stride;
    float *g, *beta;
    int32_t tile_of[TSV_GDN_MAX_SEQ + 1];  // first row tile of every sequence
    int32_t channel_blocks, tile_rows;
};

template <int DK, bool F16>
__global__ __launch_bounds__(CONV_THREADS) void k_gdn_conv(GdnShape sh, GdnBatch bt, ConvArgs p) {
    int lo = 0, hi = bt.n_seq;  // the sequence of this tile: the last one that starts at or before it
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (p.tile_of[mid] <= (int)blockIdx.x) lo = mid;
        else hi = mid;
    }
    const int s = lo, first = bt.off[s], n = bt.off[s + 1] - first, r0 = ((int)blockIdx.x - p.tile_of[s]) * p.tile_rows;
    const int rows = min(p.tile_rows, n - r0);
    if ((int)blockIdx.y == p.channel_blocks) {  // the gates' block
        for (int i = threadIdx.x; i < rows * sh.hv; i += CONV_THREADS) {
            const int r = i / sh.hv, h = i - r * sh.hv;
            const int64_t row = first + r0 + r;
            p.g[row * sh.hv + h] = decay_of(sh.a_log[h], row_f32<F16>(p.a[row * p.gate_stride + h]) + sh.dt_bias[h]);
            p.beta[row * sh.hv + h] = sigmoid_f32(row_f32<F16>(p.b[row * p.gate_stride + h]));
        }
        return;
    }
    const int c = ((int)blockIdx.y * CONV_THREADS + threadIdx.x) * 8;
    if (c >= sh.channels) return;  // (a head's threads stay or leave together: head widths are multiples of 16 channels)
    const int taps = sh.taps;
    const uint16_t* in = p.qkv + (int64_t)(first + r0) * p.qkv_stride + c;
    uint16_t* out = p.out + (int64_t)(first + r0) * p.out_stride + c;
    uint4 ahead[4];
#pragma unroll
    for (int r = 0; r < 4; r++) ahead[r] = *(const uint4*)(in + min(r, rows - 1) * p.qkv_stride);
    float w[4][8], x[7][8];  // w[j]: j rows back; x[3 - j]: the row j before the four in hand
    if (taps == 4) {
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const uf4 t = *(const uf4*)(sh.conv + (int64_t)(c + e) * 4);
#pragma unroll
            for (int j = 0; j < 4; j++) w[j][e] = t[3 - j];
        }
    } else {
#pragma unroll
        for (int j = 0; j < 4; j++)
#pragma unroll
            for (int e = 0; e < 8; e++) w[j][e] = j < taps ? sh.conv[(int64_t)(c + e) * taps + taps - 1 - j] : 0.0f;
    }
    const int64_t ring = (int64_t)s * TSV_GDN_RING * sh.channels + c;
    const int64_t base = r0 == 0 ? bt.base[s] : 0;
#pragma unroll
    for (int j = 1; j < 4; j++) {
        uint4 u = make_uint4(0, 0, 0, 0);
        if (j < taps) {
            if (r0 - j >= 0) u = *(const uint4*)(in - j * p.qkv_stride);
            else if (base - j >= 0) u = *(const uint4*)(p.ring_in + ring + ((base - j) & (TSV_GDN_RING - 1)) * sh.channels);
        }
        row8_f32<F16>(u, x[3 - j]);
    }
    const bool unit = c < 2 * sh.hk * DK;
    for (int r = 0; r < rows; r += 4) {
#pragma unroll
        for (int i = 0; i < 4; i++) row8_f32<F16>(ahead[i], x[3 + i]);
        if (r + 4 < rows) {
#pragma unroll
            for (int i = 0; i < 4; i++) ahead[i] = *(const uint4*)(in + min(r + 4 + i, rows - 1) * p.qkv_stride);
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            float y[8], sum = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                float v = x[3 + i][e] * w[0][e];
#pragma unroll
                for (int j = 1; j < 4; j++) v = fmaf(x[3 + i - j][e], w[j][e], v);
                y[e] = silu_f32(v);
            }
            if (unit) {
#pragma unroll
                for (int e = 0; e < 8; e++) sum = fmaf(y[e], y[e], sum);
                const float f = rsqrtf(sum_lanes<DK / 8>(sum) + sh.l2_eps);
#pragma unroll
                for (int e = 0; e < 8; e++) y[e] *= f;
            }
            if (r + i < rows)
                store_through(out + (r + i) * p.out_stride, __builtin_bit_cast(gf4, make_uint4(row_pair<F16>(y[0], y[1]), row_pair<F16>(y[2], y[3]),
                                                                                             row_pair<F16>(y[4], y[5]), row_pair<F16>(y[6], y[7]))));
        }
#pragma unroll
        for (int j = 0; j < 3; j++)
#pragma unroll
            for (int e = 0; e < 8; e++) x[j][e] = x[4 + j][e];
    }
    // the ring's new rows, by the thread that has read the old ones of these channels
    if (r0 == 0)
        for (int j = 1; j < taps && j <= n; j++)
            *(uint4*)(p.ring_out + ring + ((base + n - j) & (TSV_GDN_RING - 1)) * sh.channels) = *(const uint4*)(p.qkv + (int64_t)(first + n - j) * p.qkv_stride + c);
}

// ---- the step of a few rows -------------------------------------------------------------------------------------------------
// One workgroup per (value head, sequence), a wave per 16 value channels.  A wave's part of the state (16 x k_dim f32) is asked
// for first and stays in registers.  Meanwhile every thread takes 8 channels of one row through the convolution (the taps' rows come
// straight from the rows and the ring), k_dim / 8 neighbours make a unit vector of them and store it as two bf16 terms in operand
// order; the last wave makes D_ij = exp(sum of g from j, exclusive, to i) along the root paths.  From D and the products k_i.k_j,
// q_i.k_j the first two waves make the 16 x 16 matrices
//     T = (I + A)^-1,  A_ij = beta_i D_ij k_i.k_j (j a strict ancestor of i),    P_ij = D_ij q_i.k_j (j an ancestor or i)
// while the others go on to KS = k S, QS = q S (three bf16 products each: 2^-17, see split2).  Then, for all rows at once,
// u = T beta (v - e^G KS), o = e^G QS + P u, and for final rows S <- e^G_end S + sum_i D_end,i k_i u_i (f32 matrix instructions).
// With one sequence the chain of loads and three barriers bounds it (32 heads of 128, a call among others: 5 rows 8.6 us; 16-row trees of 4
// sequences 12.6), with many the state's bytes.
// Operand order of the contraction over k_dim: lane group gq of the 16x16x32 instruction takes elements 4 gq .. + 3 of both
// 16-wide halves of its 32, so that two neighbouring D tiles of the f32 update are exactly one B operand.

struct StepArgs {
    const uint16_t* qkv;
    int64_t qkv_stride;
    const uint16_t *a, *b;
    int64_t gate_stride;
    const uint16_t* z;
    int64_t z_stride;
    uint16_t* ring;
    const float* state_in;
    float* state_out;
    float* record;
    uint16_t* out;
    int64_t out_stride;
    int32_t total_rows, max_rows;
    uint32_t inv_pv;
};

// the weights of 8 channels, w[..][3 - j] that of the row j back
__device__ __forceinline__ void step_weights(const float* conv, int ch, int taps, uf4* w) {
    if (taps == 4) {
#pragma unroll
        for (int e = 0; e < 8; e++) w[e] = *(const uf4*)(conv + (int64_t)(ch + e) * 4);
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++) {
            w[e] = uf4{0, 0, 0, 0};
            const float* from = conv + (int64_t)(ch + e) * taps + taps;
            w[e][3] = from[-1];
            if (taps > 1) w[e][2] = from[-2];
            if (taps > 2) w[e][1] = from[-3];
        }
    }
}
template <bool F16>
__device__ __forceinline__ void step_convolve(const uint4* raw, const uf4* w, float* y) {
#pragma unroll
    for (int e = 0; e < 8; e++) y[e] = 0.0f;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        float x[8];
        row8_f32<F16>(raw[j], x);
#pragma unroll
        for (int e = 0; e < 8; e++) y[e] = fmaf(x[e], w[e][3 - j], y[e]);
    }
#pragma unroll
    for (int e = 0; e < 8; e++) y[e] = silu_f32(y[e]);
}
// 8 values of a head's vector, its others in the DK / 8 lanes around, to unit length
template <int DK>
__device__ __forceinline__ void step_unit(float* y, float eps) {
    float sum = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; e++) sum = fmaf(y[e], y[e], sum);
    const float f = rsqrtf(sum_lanes<DK / 8>(sum) + eps);
#pragma unroll
    for (int e = 0; e < 8; e++) y[e] *= f;
}

template <int DK>
constexpr int step_lds = 16 * (DK / 32 * 64) + 256 + 3 * 320 + 2 * 16;  // floats beside k, v and the sums of squares

template <int DK, bool F16, int THREADS>
__global__ __launch_bounds__(THREADS, DK == 256 ? 2 : 4) void k_gdn_step(GdnShape sh, StepArgs p, GdnBatch bt) {
    extern __shared__ uint4 lds4[];
    // all arguments asked for together: each trip to them takes about 0.2 us
    asm volatile("" ::"s"(sh.hk), "s"(sh.hv), "s"(sh.rep), "s"(sh.dv), "s"(sh.taps), "s"(sh.channels), "s"(sh.conv), "s"(sh.a_log), "s"(sh.dt_bias), "s"(sh.norm));
    asm volatile("" ::"s"(p.qkv), "s"(p.qkv_stride), "s"(p.a), "s"(p.b), "s"(p.gate_stride), "s"(p.z), "s"(p.z_stride), "s"(p.ring), "s"(p.state_in), "s"(p.state_out),
                 "s"(p.record), "s"(p.out), "s"(p.out_stride), "s"(p.total_rows), "s"(p.max_rows), "s"(p.inv_pv), "s"(bt.base), "s"(bt.parent));
    const int hk = blockIdx.y, h = hk * sh.rep + blockIdx.x, s = blockIdx.z, dv = sh.dv, nt = dv * 4, tid = threadIdx.x;
    const int first = bt.off[s], m = bt.off[s + 1] - first, taps = sh.taps;
    const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l16 = lane & 15, gq = lane >> 4, waves = dv >> 4;
    const int64_t base = bt.base[s];
    const float a_log = sh.a_log[h], dt_bias = sh.dt_bias[h];
    const size_t at = ((size_t)s * sh.hv + h) * dv * DK + (size_t)(16 * wave + l16) * DK + 4 * gq;
    constexpr int NT = DK / 16;
    float4 S[NT];
#pragma unroll
    for (int t = 0; t < NT; t++) S[t] = *(const float4*)(p.state_in + at + 16 * t);
    if (m <= 0) {  // no rows: the state stays
        if (p.state_out) {
#pragma unroll
            for (int t = 0; t < NT; t++) *(float4*)(p.state_out + at + 16 * t) = base == 0 ? make_float4(0, 0, 0, 0) : S[t];
        }
        return;
    }
    const int col = 16 * wave + l16;  // this lane's value channel; its rows are 4 gq .. + 3
    uint16_t zr[4];
    float nw = 0.0f;
    if (p.z) {
#pragma unroll
        for (int r = 0; r < 4; r++) zr[r] = p.z[(int64_t)(first + min(4 * gq + r, m - 1)) * p.z_stride + h * dv + col];
        nw = sh.norm[col];
    }
    constexpr int FR = DK / 32 * 64;
    uint4* kf = lds4;                 // operand fragments [q, k][hi, lo][DK / 32][lane]
    float* D = (float*)(kf + 4 * FR);  // [16][16], zero where j is no ancestor of i
    float* A = D + 256;               // [16][20]
    float* T = A + 320;
    float* P = T + 320;
    float* beta = P + 320;
    float* eG = beta + 16;
    float* kv = eG + 16;              // k as f32 [m][DK], v [m][dv]
    float* vv = kv + p.max_rows * DK;
    float* red = vv + p.max_rows * dv;  // [row][16]: a wave's sum of squares each
    // every wave knows the rows' parents, each sixteen lanes again
    int par = l16 - 1;
    if (bt.parent) {
        par = l16 < m ? bt.parent[first + l16] : -1;
        if (par >= l16) par = -1;
    }
    if (par < 0) par = -1;
    if (wave == waves - 1) {
        float g = 0.0f, be = 0.0f;
        if (l16 < m) {
            const int64_t row = first + l16;
            g = decay_of(a_log, row_f32<F16>(p.a[row * p.gate_stride + h]) + dt_bias);
            be = sigmoid_f32(row_f32<F16>(p.b[row * p.gate_stride + h]));
            if (p.record && gq == 0) p.record[(size_t)p.total_rows * (sh.hv * dv + sh.hk * DK) + (size_t)row * sh.hv + h] = g;
        }
        // the rows on row l16's root path, as bits: in each round the path doubles
        uint32_t on = 1u << l16;
        int up = par;
        if (!bt.parent) {
            on = (2u << l16) - 1;
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const uint32_t more = __shfl(on, up & 15, 16);
                const int next = __shfl(up, up & 15, 16);
                if (up >= 0) {
                    on |= more;
                    up = next;
                }
            }
        }
        float sum[4] = {}, all = 0.0f;  // of g over the rows behind ancestor 4 gq + r, and over the whole path
        uint32_t path[4];
#pragma unroll
        for (int r = 0; r < 4; r++) path[r] = on & ~__shfl(on, 4 * gq + r, 16);
#pragma unroll 1
        for (int t = 0; t < m; t++) {  // (not unrolled: code that runs once is paid by its length)
            const float gt = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(g), t));
            const uint32_t bit = 1u << t;
            all += on & bit ? gt : 0.0f;
#pragma unroll
            for (int r = 0; r < 4; r++) sum[r] += path[r] & bit ? gt : 0.0f;
        }
#pragma unroll
        for (int r = 0; r < 4; r++) D[l16 * 16 + 4 * gq + r] = on >> (4 * gq + r) & 1 ? __expf(sum[r]) : 0.0f;
        if (gq == 0) {
            beta[l16] = be;
            eG[l16] = __expf(all);
        }
    }
    // the convolution: items of 8 channels of a row, all rows' q, then k, then v
    constexpr int pk = DK / 8;
    const int pv = dv >> 3, items = m * (2 * pk + pv);
    const uint32_t inv_pv = p.inv_pv;  // 65536 / pv, up: exact for the up to 512 items of v
    uint16_t* ring = p.ring + (int64_t)s * TSV_GDN_RING * sh.channels;
    for (int i0 = 64 * wave; i0 < items; i0 += nt) {
        const int i = min(i0 + lane, items - 1);  // (lanes behind the last item do it again: the parents are read across lanes)
        const int kind = i < m * pk ? 0 : i < 2 * m * pk ? 1 : 2, left = i - min(kind, 2) * m * pk;
        const int row = kind < 2 ? left / pk : (int)(((uint32_t)left * inv_pv) >> 16), c = (left - row * (kind < 2 ? pk : pv)) * 8;
        const int ch = kind == 0 ? hk * DK + c : kind == 1 ? (sh.hk + hk) * DK + c : 2 * sh.hk * DK + h * dv + c;
        uf4 w[8];
        step_weights(sh.conv, ch, taps, w);
        uint4 raw[4];
        int q = row;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const uint16_t* from = q >= 0 ? p.qkv + (int64_t)(first + q) * p.qkv_stride : ring + ((base + q) & (TSV_GDN_RING - 1)) * sh.channels;
            raw[j] = *(const uint4*)(from + ch);  // (every slot can be read; those of no position do not count)
            if (j >= taps || base + q < 0) raw[j] = make_uint4(0, 0, 0, 0);
            const int next = bt.parent ? __shfl(par, q & 15, 16) : q - 1;
            q = q >= 0 ? next : q - 1;
        }
        float y[8];
        step_convolve<F16>(raw, w, y);
        if (kind == 2 || blockIdx.x == 0) *(uint4*)(ring + ((base + row) & (TSV_GDN_RING - 1)) * sh.channels + ch) = raw[0];
        if (kind == 2) {
            *(float4*)(vv + row * dv + c) = make_float4(y[0], y[1], y[2], y[3]);
            *(float4*)(vv + row * dv + c + 4) = make_float4(y[4], y[5], y[6], y[7]);
        } else {
            step_unit<DK>(y, sh.l2_eps);
            if (kind == 1) {
                *(float4*)(kv + row * DK + c) = make_float4(y[0], y[1], y[2], y[3]);
                *(float4*)(kv + row * DK + c + 4) = make_float4(y[4], y[5], y[6], y[7]);
                if (p.record && blockIdx.x == 0) {
                    float* to = p.record + (size_t)p.total_rows * sh.hv * dv + ((size_t)(first + row) * sh.hk + hk) * DK + c;
                    *(uf4*)to = uf4{y[0], y[1], y[2], y[3]};
                    *(uf4*)(to + 4) = uf4{y[4], y[5], y[6], y[7]};
                }
            }
            uint2* f2 = (uint2*)(kf + kind * 2 * FR);
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const int o = (c & 31) + 4 * e, to = ((c >> 5) * 64 + ((o & 15) >> 2) * 16 + row) * 2 + (o >> 4);
                uint2 hi, lo;
                split2(y[4 * e], y[4 * e + 1], hi.x, lo.x);
                split2(y[4 * e + 2], y[4 * e + 3], hi.y, lo.y);
                f2[to] = hi;
                f2[2 * FR + to] = lo;
            }
        }
    }
    for (int i = tid; i < 256; i += nt)  // waves and rows there are not
        if ((i & 15) >= waves) red[i] = 0.0f;
    for (int i = tid; i < 4 * FR; i += nt)
        if ((i & 15) >= m) kf[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    const uint4 *qh = kf, *ql = kf + FR, *kh = kf + 2 * FR, *kl = kf + 3 * FR;
    for (int which = wave; which < 2; which += waves) {  // 0: k.k -> A, T;  1: q.k -> P
        gf4 acc = {0, 0, 0, 0}, acc2 = {0, 0, 0, 0};
#pragma unroll
        for (int t = 0; t < DK / 32; t++) {
            const bf16x8 bh = __builtin_bit_cast(bf16x8, kh[t * 64 + lane]), bl = __builtin_bit_cast(bf16x8, kl[t * 64 + lane]);
            const bf16x8 ah = __builtin_bit_cast(bf16x8, (which ? qh : kh)[t * 64 + lane]);
            const bf16x8 al = __builtin_bit_cast(bf16x8, (which ? ql : kl)[t * 64 + lane]);
            acc = mfma_bf16(ah, bh, acc);
            acc2 = mfma_bf16(ah, bl, acc2);
            acc2 = mfma_bf16(al, bh, acc2);
        }
        acc += acc2;
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const int i = 4 * gq + r;
            const float d = D[i * 16 + l16];
            if (which) P[i * 20 + l16] = d * acc[r];
            else A[i * 20 + l16] = i == l16 ? 0.0f : beta[i] * d * acc[r];
        }
        if (which == 0) {
            wave_lds_fence();
            invert_lower16(A, 20, T, 20, l16, gq, m > 8);
        }
    }
    if (base == 0) {
#pragma unroll
        for (int t = 0; t < NT; t++) S[t] = make_float4(0, 0, 0, 0);
    }
    gf4 ks = {0, 0, 0, 0}, qs = {0, 0, 0, 0}, ks2 = {0, 0, 0, 0}, qs2 = {0, 0, 0, 0};
#pragma unroll
    for (int t = 0; t < DK / 32; t++) {
        uint4 sh8, sl8;
        split2(S[2 * t].x, S[2 * t].y, sh8.x, sl8.x);
        split2(S[2 * t].z, S[2 * t].w, sh8.y, sl8.y);
        split2(S[2 * t + 1].x, S[2 * t + 1].y, sh8.z, sl8.z);
        split2(S[2 * t + 1].z, S[2 * t + 1].w, sh8.w, sl8.w);
        const bf16x8 s0 = __builtin_bit_cast(bf16x8, sh8), s1 = __builtin_bit_cast(bf16x8, sl8);
        const bf16x8 k0 = __builtin_bit_cast(bf16x8, kh[t * 64 + lane]), k1 = __builtin_bit_cast(bf16x8, kl[t * 64 + lane]);
        const bf16x8 q0 = __builtin_bit_cast(bf16x8, qh[t * 64 + lane]), q1 = __builtin_bit_cast(bf16x8, ql[t * 64 + lane]);
        ks = mfma_bf16(k0, s0, ks);
        qs = mfma_bf16(q0, s0, qs);
        ks2 = mfma_bf16(k0, s1, ks2);
        qs2 = mfma_bf16(q0, s1, qs2);
        ks2 = mfma_bf16(k1, s0, ks2);
        qs2 = mfma_bf16(q1, s0, qs2);
    }
    float r4[4];
    gf4 u = {0, 0, 0, 0}, o;
#pragma unroll
    for (int r = 0; r < 4; r++) {
        const int i = 4 * gq + r;
        const float v = vv[min(i, m - 1) * dv + col], e = eG[i];  // (beta is 0 in rows there are not)
        r4[r] = beta[i] * fmaf(-e, ks[r] + ks2[r], v);
        o[r] = e * (qs[r] + qs2[r]);
    }
    __syncthreads();
    const float4 t4 = *(const float4*)(T + l16 * 20 + 4 * gq), p4 = *(const float4*)(P + l16 * 20 + 4 * gq);
    const float tt[4] = {t4.x, t4.y, t4.z, t4.w}, pp[4] = {p4.x, p4.y, p4.z, p4.w};
#pragma unroll
    for (int r = 0; r < 4; r++) u = mfma_f32(tt[r], r4[r], u);
#pragma unroll
    for (int r = 0; r < 4; r++) o = mfma_f32(pp[r], u[r], o);
    o *= sh.scale;
    if (p.z) {
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const float q = sum_lanes<16>(o[r] * o[r]);
            if (l16 == 0) red[(4 * gq + r) * 16 + wave] = q;
        }
    }
    if (p.record) {
#pragma unroll
        for (int r = 0; r < 4; r++)
            if (4 * gq + r < m) p.record[((size_t)(first + 4 * gq + r) * sh.hv + h) * dv + col] = u[r];
    }
    if (p.z) {
        __syncthreads();
#pragma unroll
        for (int r = 0; r < 4; r++) {
            float sum = 0.0f;
#pragma unroll
            for (int w = 0; w < THREADS / 256; w++) {
                const float4 t = *(const float4*)(red + (4 * gq + r) * 16 + 4 * w);
                sum += (t.x + t.y) + (t.z + t.w);
            }
            o[r] *= rsqrtf(sum / (float)dv + sh.norm_eps) * nw * silu_f32(row_f32<F16>(zr[r]));
        }
    }
#pragma unroll
    for (int r = 0; r < 4; r++)
        if (4 * gq + r < m) p.out[(int64_t)(first + 4 * gq + r) * p.out_stride + h * dv + col] = row_bits<F16>(o[r]);
    // (last: the stores of a whole head hold a compute unit's write path for a while)
    if (p.state_out) {
        const float end = eG[m - 1];
#pragma unroll
        for (int t = 0; t < NT; t++) S[t] = make_float4(S[t].x * end, S[t].y * end, S[t].z * end, S[t].w * end);
#pragma unroll
        for (int r = 0; r < 4; r++) {
            if (r >= m) break;  // (rows 4, 8 and 12 ride in the same instructions as row 0)
            const int i = 4 * gq + r;
            const float uw = u[r] * D[(m - 1) * 16 + i];  // (u is 0 in rows there are not)
            const float* k = kv + min(i, m - 1) * DK + l16;
#pragma unroll
            for (int t = 0; t < NT; t++) {
                const gf4 acc = mfma_f32(k[16 * t], uw, gf4{S[t].x, S[t].y, S[t].z, S[t].w});
                S[t] = make_float4(acc[0], acc[1], acc[2], acc[3]);
            }
        }
#pragma unroll
        for (int t = 0; t < NT; t++) *(float4*)(p.state_out + at + 16 * t) = S[t];
    }
}

// The same for one row a sequence, plain decoding: u = beta (v - e^g k S), o = e^g q S + (q.k) u, S <- e^g S + k u^T need no
// 16 x 16 matrices and no operand fragments; the products with the state are f32 dot products over the k_dim / 4 neighbouring lanes of a
// channel.  A wave's 16 channels x k_dim are one run of memory, taken 1 KiB an instruction: whole lines in and out (lanes that held k_dim
// / 4 values of one channel, 64 bytes of 16 lines an instruction, took 7.4 us where this takes 5.2, and 124 where this takes 101).  Two
// barriers.  32 heads of 128: one sequence 5.2 us, 128 sequences 101 us for 537 MB of state (5.3 TB/s; 107 with stores that stay in the
// L2).

// sums over the DK / 4 lanes of each of the NT x 256 / DK channels that the lanes' x belong to: x[0 .. 3] become the sums of channels
// 4 j + one_row_channel, the same in all lanes of a row of sixteen
template <int DK>
__device__ __forceinline__ void one_row_sums(float* x) {
    if constexpr (DK == 256) {
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = lane_pairs_by_32(x[2 * i], x[2 * i + 1]);
    }
    if constexpr (DK >= 128) {
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = lane_pairs_by_16(x[2 * i], x[2 * i + 1]);
    }
#pragma unroll
    for (int i = 0; i < 4; i++) x[i] = sum_lanes<16>(x[i]);
}
template <int DK>
__device__ __forceinline__ int one_row_channel(int row) {
    return DK == 64 ? row : 2 * (row & 1) + (row >> 1);
}
// the other way: u, which lane j of every four holds for channel 4 j + one_row_channel, to the channels of x[NT]
template <int DK>
__device__ __forceinline__ void one_row_spread(float u, float* x) {
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int v = __float_as_int(u);
        const float w = __int_as_float(j == 0   ? __builtin_amdgcn_update_dpp(0, v, 0x00, 0xF, 0xF, true)
                                       : j == 1 ? __builtin_amdgcn_update_dpp(0, v, 0x55, 0xF, 0xF, true)
                                       : j == 2 ? __builtin_amdgcn_update_dpp(0, v, 0xAA, 0xF, 0xF, true)
                                                : __builtin_amdgcn_update_dpp(0, v, 0xFF, 0xF, 0xF, true));
        if constexpr (DK == 64) x[j] = w;
        if constexpr (DK == 128) {
            const float2 r = lanes_by_16(w);
            x[2 * j] = r.x, x[2 * j + 1] = r.y;
        }
        if constexpr (DK == 256) {
            const float2 r = lanes_by_16(w), a = lanes_by_32(r.x), b = lanes_by_32(r.y);
            x[4 * j] = a.x, x[4 * j + 1] = a.y, x[4 * j + 2] = b.x, x[4 * j + 3] = b.y;
        }
    }
}

template <int DK, bool F16, int THREADS>
__global__ __launch_bounds__(THREADS, DK == 256 ? 2 : 4) void k_gdn_step_one(GdnShape sh, StepArgs p, GdnBatch bt) {
    __shared__ float4 q4[DK / 4], k4[DK / 4];
    __shared__ float vv[256], red[16], gate[2];
    asm volatile("" ::"s"(sh.hk), "s"(sh.hv), "s"(sh.rep), "s"(sh.dv), "s"(sh.taps), "s"(sh.channels), "s"(sh.conv), "s"(sh.a_log), "s"(sh.dt_bias), "s"(sh.norm));
    asm volatile("" ::"s"(p.qkv), "s"(p.qkv_stride), "s"(p.a), "s"(p.b), "s"(p.gate_stride), "s"(p.z), "s"(p.z_stride), "s"(p.ring), "s"(p.state_in), "s"(p.state_out),
                 "s"(p.record), "s"(p.out), "s"(p.out_stride), "s"(p.total_rows), "s"(bt.base));
    const int hk = blockIdx.y, h = hk * sh.rep + blockIdx.x, s = blockIdx.z, dv = sh.dv, tid = threadIdx.x;
    const int row = bt.off[s], m = bt.off[s + 1] - row, taps = sh.taps;
    const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), waves = dv >> 4;
    const int64_t base = bt.base[s];
    const size_t at = ((size_t)s * sh.hv + h) * dv * DK + (size_t)(16 * wave * DK + 4 * lane);
    constexpr int NT = DK / 16;
    float4 S[NT];
#pragma unroll
    for (int t = 0; t < NT; t++) S[t] = *(const float4*)(p.state_in + at + 256 * t);
    if (m <= 0) {  // no row: the state stays
        if (p.state_out) {
#pragma unroll
            for (int t = 0; t < NT; t++) *(float4*)(p.state_out + at + 256 * t) = base == 0 ? make_float4(0, 0, 0, 0) : S[t];
        }
        return;
    }
    const int col = 16 * wave + 4 * (lane & 3) + one_row_channel<DK>(lane >> 4);  // the value channel whose u and o this lane makes
    uint16_t zr = 0;
    float nw = 0.0f;
    if (p.z) {
        zr = p.z[(int64_t)row * p.z_stride + h * dv + col];
        nw = sh.norm[col];
    }
    if (tid == 64 * (waves - 1)) {
        const float g = decay_of(sh.a_log[h], row_f32<F16>(p.a[row * p.gate_stride + h]) + sh.dt_bias[h]);
        gate[0] = __expf(g);
        gate[1] = sigmoid_f32(row_f32<F16>(p.b[row * p.gate_stride + h]));
        if (p.record) p.record[(size_t)p.total_rows * (sh.hv * dv + sh.hk * DK) + (size_t)row * sh.hv + h] = g;
    }
    if (tid < 16) red[tid] = 0.0f;
    constexpr int pk = DK / 8;
    const int items = 2 * pk + (dv >> 3);
    uint16_t* ring = p.ring + (int64_t)s * TSV_GDN_RING * sh.channels;
    for (int i = tid; i < items; i += 4 * dv) {
        const int kind = i < pk ? 0 : i < 2 * pk ? 1 : 2, c = (i - kind * pk) * 8;
        const int ch = kind == 0 ? hk * DK + c : kind == 1 ? (sh.hk + hk) * DK + c : 2 * sh.hk * DK + h * dv + c;
        uf4 w[8];
        step_weights(sh.conv, ch, taps, w);
        uint4 raw[4];
        raw[0] = *(const uint4*)(p.qkv + (int64_t)row * p.qkv_stride + ch);
#pragma unroll
        for (int j = 1; j < 4; j++) {
            raw[j] = *(const uint4*)(ring + ((base - j) & (TSV_GDN_RING - 1)) * sh.channels + ch);  // (every slot can be read; those of no position do not count)
            if (j >= taps || base < j) raw[j] = make_uint4(0, 0, 0, 0);
        }
        float y[8];
        step_convolve<F16>(raw, w, y);
        if (kind == 2 || blockIdx.x == 0) *(uint4*)(ring + (base & (TSV_GDN_RING - 1)) * sh.channels + ch) = raw[0];
        if (kind < 2) step_unit<DK>(y, sh.l2_eps);
        float4* to = kind == 0 ? q4 + c / 4 : kind == 1 ? k4 + c / 4 : (float4*)vv + c / 4;
        to[0] = make_float4(y[0], y[1], y[2], y[3]);
        to[1] = make_float4(y[4], y[5], y[6], y[7]);
        if (kind == 1 && p.record && blockIdx.x == 0) {
            float* rec = p.record + (size_t)p.total_rows * sh.hv * dv + ((size_t)row * sh.hk + hk) * DK + c;
            *(uf4*)rec = uf4{y[0], y[1], y[2], y[3]};
            *(uf4*)(rec + 4) = uf4{y[4], y[5], y[6], y[7]};
        }
    }
    __syncthreads();
    if (base == 0) {
#pragma unroll
        for (int t = 0; t < NT; t++) S[t] = make_float4(0, 0, 0, 0);
    }
    const float4 k = k4[lane & (DK / 4 - 1)], q = q4[lane & (DK / 4 - 1)];
    float ks4[NT], qs4[NT];
#pragma unroll
    for (int t = 0; t < NT; t++) {
        ks4[t] = fmaf(k.x, S[t].x, fmaf(k.y, S[t].y, fmaf(k.z, S[t].z, k.w * S[t].w)));
        qs4[t] = fmaf(q.x, S[t].x, fmaf(q.y, S[t].y, fmaf(q.z, S[t].z, q.w * S[t].w)));
    }
    one_row_sums<DK>(ks4);
    one_row_sums<DK>(qs4);
    float2 r;
    float qk = sum_lanes<16>(fmaf(q.x, k.x, fmaf(q.y, k.y, fmaf(q.z, k.z, q.w * k.w))));
    if constexpr (DK >= 128) r = lanes_by_16(qk), qk = r.x + r.y;
    if constexpr (DK == 256) r = lanes_by_32(qk), qk = r.x + r.y;
    const float ks = lane & 2 ? (lane & 1 ? ks4[3] : ks4[2]) : lane & 1 ? ks4[1] : ks4[0];
    const float qs = lane & 2 ? (lane & 1 ? qs4[3] : qs4[2]) : lane & 1 ? qs4[1] : qs4[0];
    const float e = gate[0], u = gate[1] * fmaf(-e, ks, vv[col]);
    float o = sh.scale * fmaf(qk, u, e * qs);
    if (p.z) {
        float sq = sum_lanes<4>(o * o);
        r = lanes_by_16(sq), sq = r.x + r.y;
        r = lanes_by_32(sq), sq = r.x + r.y;
        if (lane == 0) red[wave] = sq;
        __syncthreads();
        float sum = 0.0f;
#pragma unroll
        for (int w = 0; w < THREADS / 64; w += 4) {
            const float4 t = *(const float4*)(red + w);
            sum += (t.x + t.y) + (t.z + t.w);
        }
        o *= rsqrtf(sum / (float)dv + sh.norm_eps) * nw * silu_f32(row_f32<F16>(zr));
    }
    if ((lane & 12) == 0) {
        p.out[(int64_t)row * p.out_stride + h * dv + col] = row_bits<F16>(o);
        if (p.record) p.record[((size_t)row * sh.hv + h) * dv + col] = u;
    }
    if (p.state_out) {
        float us[NT];
        one_row_spread<DK>(u, us);
#pragma unroll
        for (int t = 0; t < NT; t++)
            store_through(p.state_out + at + 256 * t, gf4{fmaf(us[t], k.x, e * S[t].x), fmaf(us[t], k.y, e * S[t].y), fmaf(us[t], k.z, e * S[t].z), fmaf(us[t], k.w, e * S[t].w)});
    }
}

// ---- accepted rows into the state -----------------------------------------------------------------------------------------------
// S <- e^{g_1 + .. + g_n} S + sum_i e^{g_{i+1} + .. + g_n} k_i u_i^T over the kept path.  A thread keeps four state values of
// COMMIT_PIECES neighbouring value channels; the path, the same for a workgroup, goes through scalar registers, and from it four rows'
// k and u at a time are under way.  One pass over the state, which is what bounds it: three rows of one sequence in 24 layers of 32 heads
// of 128, 101 MB of state, 19 us (5.2 TB/s; 26 where the stores stay in the L2); trees of 16 rows of 32 sequences, 134 MB, 25 us (31).
// (Steps of all those layers right behind it take 0.4 us more each, which find the state in the L2 else; a model's products between them
// would have emptied it.)
// The last workgroups of a (sequence, layer) move the ring's rows: slot i takes the row of slot path[i] >= i, in ascending order by one
// thread.
constexpr int COMMIT_THREADS = 256, COMMIT_PIECES = 4;

struct CommitArgs {
    const tsv_round_result* results;
    const float* record;
    int64_t record_stride;  // floats
    const uint16_t* ring_in;
    uint16_t* ring_out;
    int64_t ring_stride;
    const float* state_in;
    float* state_out;
    int64_t state_stride;
    int32_t total_rows, state_blocks, blocks;  // workgroups of all heads' state, and of a head's
};

template <int DK>
__global__ __launch_bounds__(COMMIT_THREADS) void k_gdn_commit(GdnShape sh, CommitArgs p, GdnBatch bt) {
    asm volatile("" ::"s"(sh.hk), "s"(sh.hv), "s"(sh.rep), "s"(sh.dv), "s"(sh.channels), "s"(p.results), "s"(p.record), "s"(p.record_stride), "s"(p.ring_in),
                 "s"(p.ring_out), "s"(p.ring_stride), "s"(p.state_in), "s"(p.state_out), "s"(p.state_stride), "s"(p.total_rows), "s"(p.state_blocks), "s"(p.blocks),
                 "s"(bt.base));
    const int s = blockIdx.y, layer = blockIdx.z, tid = threadIdx.x, first = bt.off[s], m = min(bt.off[s + 1] - first, TSV_MAX_ROWS);
    const auto* said = uniform_memory(p.results + s);
    const int64_t base = bt.base[s];
    constexpr int PER_ROW = DK / 4, CH = COMMIT_THREADS / PER_ROW * COMMIT_PIECES;  // value channels of a workgroup
    const bool of_ring = (int)blockIdx.x >= p.state_blocks;
    const int h = of_ring ? 0 : (int)blockIdx.x / p.blocks, c0 = ((int)blockIdx.x - h * p.blocks) * CH + tid / PER_ROW * COMMIT_PIECES;
    const bool in = !of_ring && c0 < sh.dv;  // (v_dim is a multiple of 16: a thread's channels are all there or none)
    const int kq = (tid % PER_ROW) * 4;
    const size_t at = (size_t)((int64_t)layer * p.state_stride) + (((size_t)s * sh.hv + h) * sh.dv + c0) * DK + kq;
    float4 S[COMMIT_PIECES];
#pragma unroll
    for (int i = 0; i < COMMIT_PIECES; i++) {
        S[i] = make_float4(0, 0, 0, 0);
        if (in) S[i] = *(const float4*)(p.state_in + at + i * DK);
    }
    // the path as far as it names rows of the sequence in ascending order
    int path[TSV_MAX_ROWS], n = 0;
    {
        const int kept = said->committed < m ? said->committed + 1 : m, len = said->path_len, want = min(kept, len);
        int before = -1;
        bool on = true;
#pragma unroll
        for (int i = 0; i < TSV_MAX_ROWS; i++) {
            const int row = said->path[i];
            on = on && i < want && row > before && row < m;
            path[i] = on ? row : 0;  // (behind the path: a row that there is, with no weight)
            n += on;
            before = row;
        }
    }
    if (of_ring) {
        const int c = (((int)blockIdx.x - p.state_blocks) * COMMIT_THREADS + tid) * 8;
        if (c >= sh.channels) return;
        const int64_t to = (int64_t)layer * p.ring_stride + (int64_t)s * TSV_GDN_RING * sh.channels + c;
#pragma unroll
        for (int i = 0; i < TSV_MAX_ROWS; i++) {
            if (i >= n) break;
            if (path[i] == i && p.ring_in == p.ring_out) continue;
            *(uint4*)(p.ring_out + to + ((base + i) & (TSV_GDN_RING - 1)) * sh.channels) =
                *(const uint4*)(p.ring_in + to + ((base + path[i]) & (TSV_GDN_RING - 1)) * sh.channels);
        }
        return;
    }
    if (!in) return;
    const float* rec = p.record + (int64_t)layer * p.record_stride;
    const float* rec_k = rec + (size_t)p.total_rows * sh.hv * sh.dv + ((size_t)first * sh.hk + h / sh.rep) * DK + kq;
    const float* rec_u = rec + ((size_t)first * sh.hv + h) * sh.dv + c0;
    const auto* rec_g = uniform_memory(rec + (size_t)p.total_rows * (sh.hv * sh.dv + sh.hk * DK) + (size_t)first * sh.hv + h);
    float w[TSV_MAX_ROWS], sum = 0.0f;
    if (n > 0) {  // (a sequence may have no rows at all)
#pragma unroll
        for (int i = 0; i < TSV_MAX_ROWS; i++) w[i] = i < n ? rec_g[path[i] * sh.hv] : 0.0f;
    }
#pragma unroll
    for (int i = TSV_MAX_ROWS - 1; i >= 0; i--) {
        const float g = n > 0 ? w[i] : 0.0f;
        w[i] = i < n ? __expf(sum) : 0.0f;
        sum += g;
    }
    const float end = __expf(sum);
#pragma unroll
    for (int i = 0; i < COMMIT_PIECES; i++) {
        if (base == 0) S[i] = make_float4(0, 0, 0, 0);  // (what the buffer holds may be no number)
        S[i].x *= end;
        S[i].y *= end;
        S[i].z *= end;
        S[i].w *= end;
    }
#pragma unroll
    for (int j = 0; j < TSV_MAX_ROWS; j += 4) {
        if (j >= n) break;
        uf4 k[4], u[4];
#pragma unroll
        for (int r = 0; r < 4; r++) {
            k[r] = *(const uf4*)(rec_k + (size_t)path[j + r] * sh.hk * DK);
            u[r] = *(const uf4*)(rec_u + (size_t)path[j + r] * sh.hv * sh.dv);
        }
#pragma unroll
        for (int r = 0; r < 4; r++) {
            if (j + r >= n) break;
#pragma unroll
            for (int i = 0; i < COMMIT_PIECES; i++) {
                const float x = w[j + r] * u[r][i];
                S[i].x = fmaf(x, k[r].x, S[i].x);
                S[i].y = fmaf(x, k[r].y, S[i].y);
                S[i].z = fmaf(x, k[r].z, S[i].z);
                S[i].w = fmaf(x, k[r].w, S[i].w);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < COMMIT_PIECES; i++) store_through(p.state_out + at + i * DK, __builtin_bit_cast(gf4, S[i]));
}

// ---- arguments ----------------------------------------------------------------------------------------------------------------

int gdn_refuse(const char* who, const char* what) {
    set_error(std::string(who) + ": " + what);
    return TSV_ERR_INVALID;
}

bool gdn_rows_ok(const void* p, int64_t stride, int64_t width) {
    return p && ((uintptr_t)p & 15) == 0 && (stride & 7) == 0 && stride >= width && stride <= (int64_t)1 << 22;
}

bool gdn_overlap(const void* a, const void* b, size_t bytes) {
    return a != b && (uintptr_t)a < (uintptr_t)b + bytes && (uintptr_t)b < (uintptr_t)a + bytes;
}

int gdn_check_layer(const char* who, const tsv_gdn_layer* l, GdnShape* sh) {
    if (!l) return gdn_refuse(who, "null layer");
    if (l->n_k_heads < 1 || l->n_v_heads < 1 || l->n_v_heads % l->n_k_heads || l->n_v_heads > 1024)
        return gdn_refuse(who, "1..1024 value heads, a multiple of the key heads");
    if ((l->k_dim != 64 && l->k_dim != 128 && l->k_dim != 256) || l->v_dim < 16 || l->v_dim > 256 || l->v_dim % 16) {
        set_error(std::string(who) + ": k_dim must be 64, 128 or 256, v_dim a multiple of 16 up to 256");
        return TSV_ERR_UNSUPPORTED;
    }
    if (l->dtype != TSV_BF16 && l->dtype != TSV_F16) {
        set_error(std::string(who) + ": rows are bf16 or fp16");
        return TSV_ERR_UNSUPPORTED;
    }
    if (l->conv_width < 1 || l->conv_width > 4) {
        set_error(std::string(who) + ": 1..4 convolution taps");
        return TSV_ERR_UNSUPPORTED;
    }
    if (!(l->l2_eps >= 0.0f) || !(l->norm_eps >= 0.0f) || !(l->scale == l->scale)) return gdn_refuse(who, "a negative or undefined epsilon or scale");
    sh->hk = l->n_k_heads;
    sh->hv = l->n_v_heads;
    sh->rep = l->n_v_heads / l->n_k_heads;
    sh->dv = l->v_dim;
    sh->taps = l->conv_width;
    sh->channels = 2 * l->n_k_heads * l->k_dim + l->n_v_heads * l->v_dim;
    sh->scale = l->scale > 0.0f ? l->scale : 1.0f / sqrtf((float)l->k_dim);
    sh->l2_eps = l->l2_eps;
    sh->norm_eps = l->norm_eps;
    sh->conv = l->conv;
    sh->a_log = l->a_log;
    sh->dt_bias = l->dt_bias;
    sh->norm = l->norm;
    return TSV_OK;
}

int gdn_check(const char* who, void* stream, const tsv_gdn_layer* l, const tsv_gdn_batch* b, int max_rows, GdnShape* sh, GdnBatch* kb) {
    const int rc = gdn_check_layer(who, l, sh);
    if (rc) return rc;
    if (!b || !b->offsets || !b->base || ((uintptr_t)b->base & 7) || ((uintptr_t)b->parent & 3)) return gdn_refuse(who, "null or misaligned batch");
    if (b->n_seq < 1 || b->n_seq > TSV_GDN_MAX_SEQ) return gdn_refuse(who, "1..256 sequences");
    if (b->offsets[0] != 0) return gdn_refuse(who, "offsets start at 0");
    for (int s = 0; s < b->n_seq; s++) {
        if (b->offsets[s + 1] < b->offsets[s]) return gdn_refuse(who, "offsets decrease");
        if (max_rows && b->offsets[s + 1] - b->offsets[s] > max_rows) return gdn_refuse(who, "at most 16 rows a sequence");
    }
    if (b->offsets[b->n_seq] > 1 << 28) return gdn_refuse(who, "more than 2^28 rows");
    kb->n_seq = b->n_seq;
    kb->base = b->base;
    kb->parent = b->parent;
    std::memcpy(kb->off, b->offsets, sizeof(int32_t) * (b->n_seq + 1));
    if (const hipStream_t st = gdn_stream(stream)) {  // launches go to the current device
        int current = 0;
        hipDevice_t of = 0;
        TSV_HIP(hipGetDevice(&current));
        TSV_HIP(hipStreamGetDevice(st, &of));
        if ((int)of != current) return gdn_refuse(who, "the stream belongs to another device than the current one");
    }
    return TSV_OK;
}

namespace {

template <int DK, bool F16>
int launch_conv(hipStream_t st, const GdnShape& sh, const GdnBatch& bt, const ConvArgs& p, int tiles) {
    hipLaunchKernelGGL((k_gdn_conv<DK, F16>), dim3(tiles, p.channel_blocks + 1), dim3(CONV_THREADS), 0, st, sh, bt, p);
    TSV_HIP(hipGetLastError());
    return TSV_OK;
}

template <int DK, bool F16, int THREADS>
int launch_step(hipStream_t st, const GdnShape& sh, const GdnBatch& bt, const StepArgs& p) {
    const int waves = sh.dv / 16;
    if (p.max_rows == 1) {  // (a row of 128 conversations: see k_gdn_step_one)
        hipLaunchKernelGGL((k_gdn_step_one<DK, F16, THREADS>), dim3(sh.rep, sh.hk, bt.n_seq), dim3(64 * waves), 0, st, sh, p, bt);
        TSV_HIP(hipGetLastError());
        return TSV_OK;
    }
    auto bytes = [](int rows, int dv) { return sizeof(float) * (size_t)(step_lds<DK> + rows * (DK + dv) + 256); };
    const size_t lds = bytes(p.max_rows, sh.dv);
    static OncePerDevice once;  // (asked for once: for the most that a call can need)
    const int rc = allow_lds((const void*)k_gdn_step<DK, F16, THREADS>, bytes(TSV_MAX_ROWS, THREADS / 4), once);
    if (rc) return rc;
    hipLaunchKernelGGL((k_gdn_step<DK, F16, THREADS>), dim3(sh.rep, sh.hk, bt.n_seq), dim3(64 * waves), lds, st, sh, p, bt);
    TSV_HIP(hipGetLastError());
    return TSV_OK;
}

template <int DK>
int launch_commit(hipStream_t st, const GdnShape& sh, const GdnBatch& bt, CommitArgs& p, int layers) {
    constexpr int CH = COMMIT_THREADS / (DK / 4) * COMMIT_PIECES;
    p.blocks = (sh.dv + CH - 1) / CH;
    p.state_blocks = sh.hv * p.blocks;
    const int ring_blocks = (sh.channels / 8 + COMMIT_THREADS - 1) / COMMIT_THREADS;
    hipLaunchKernelGGL((k_gdn_commit<DK>), dim3(p.state_blocks + ring_blocks, bt.n_seq, layers), dim3(COMMIT_THREADS), 0, st, sh, p, bt);
    TSV_HIP(hipGetLastError());
    return TSV_OK;
}

}  // namespace

}  // namespace tsv

using namespace tsv;

extern "C" int32_t tsv_gdn_conv(void* stream, const tsv_gdn_layer* layer, const tsv_gdn_batch* batch, const tsv_gdn_conv_io* io) {
    const char* who = "gdn_conv";
    GdnShape sh;
    GdnBatch bt;
    const int rc = gdn_check(who, stream, layer, batch, 0, &sh, &bt);
    if (rc) return rc;
    if (!io || !io->a || !io->b || !io->ring_in || !io->ring_out || !io->g || !io->beta || !sh.conv || !sh.a_log || !sh.dt_bias) return gdn_refuse(who, "null argument");
    if (batch->parent) return gdn_refuse(who, "prompt rows are chains");
    if (!gdn_rows_ok(io->qkv, io->qkv_stride, sh.channels) || !gdn_rows_ok(io->out, io->out_stride, sh.channels) || ((uintptr_t)io->ring_in & 15) || ((uintptr_t)io->ring_out & 15) ||
        io->gate_stride < sh.hv || ((uintptr_t)io->g & 3) || ((uintptr_t)io->beta & 3))
        return gdn_refuse(who, "rows, rings and strides: 16-byte aligned, multiples of 8, as wide as a row");
    if (io->out == io->qkv) return gdn_refuse(who, "out may not be the input rows");
    if (gdn_overlap(io->ring_in, io->ring_out, 2 * (size_t)bt.n_seq * TSV_GDN_RING * sh.channels)) return gdn_refuse(who, "ring_out overlaps ring_in");
    ConvArgs p;
    p.qkv = (const uint16_t*)io->qkv;
    p.qkv_stride = io->qkv_stride;
    p.a = (const uint16_t*)io->a;
    p.b = (const uint16_t*)io->b;
    p.gate_stride = io->gate_stride;
    p.ring_in = (const uint16_t*)io->ring_in;
    p.ring_out = (uint16_t*)io->ring_out;
    p.out = (uint16_t*)io->out;
    p.out_stride = io->out_stride;
    p.g = io->g;
    p.beta = io->beta;
    p.tile_of[0] = 0;
    p.channel_blocks = (sh.channels / 8 + CONV_THREADS - 1) / CONV_THREADS;
    p.tile_rows = (int64_t)bt.off[bt.n_seq] * p.channel_blocks >= 32 * 512 ? 32 : 4;
    for (int s = 0; s < bt.n_seq; s++) p.tile_of[s + 1] = p.tile_of[s] + (bt.off[s + 1] - bt.off[s] + p.tile_rows - 1) / p.tile_rows;
    const int tiles = p.tile_of[bt.n_seq];
    if (!tiles) return TSV_OK;
    const hipStream_t st = gdn_stream(stream);
    const bool f16 = layer->dtype == TSV_F16;
    if (layer->k_dim == 64) return f16 ? launch_conv<64, true>(st, sh, bt, p, tiles) : launch_conv<64, false>(st, sh, bt, p, tiles);
    if (layer->k_dim == 128) return f16 ? launch_conv<128, true>(st, sh, bt, p, tiles) : launch_conv<128, false>(st, sh, bt, p, tiles);
    return f16 ? launch_conv<256, true>(st, sh, bt, p, tiles) : launch_conv<256, false>(st, sh, bt, p, tiles);
}

extern "C" int64_t tsv_gdn_record_bytes(const tsv_gdn_layer* layer, int64_t rows) {
    GdnShape sh;
    if (gdn_check_layer("gdn_record_bytes", layer, &sh)) return -1;
    if (rows < 0 || rows > 1 << 28) {
        gdn_refuse("gdn_record_bytes", "0..2^28 rows");
        return -1;
    }
    return 4 * rows * (int64_t)(sh.hv * sh.dv + sh.hk * layer->k_dim + sh.hv);
}

extern "C" int32_t tsv_gdn_step(void* stream, const tsv_gdn_layer* layer, const tsv_gdn_batch* batch, const tsv_gdn_step_io* io) {
    const char* who = "gdn_step";
    GdnShape sh;
    GdnBatch bt;
    const int rc = gdn_check(who, stream, layer, batch, TSV_MAX_ROWS, &sh, &bt);
    if (rc) return rc;
    if (!io || !io->a || !io->b || !io->ring || !io->state_in || !sh.conv || !sh.a_log || !sh.dt_bias || (io->z && !sh.norm)) return gdn_refuse(who, "null argument");
    if (!gdn_rows_ok(io->qkv, io->qkv_stride, sh.channels) || !gdn_rows_ok(io->out, io->out_stride, (int64_t)sh.hv * sh.dv) ||
        (io->z && !gdn_rows_ok(io->z, io->z_stride, (int64_t)sh.hv * sh.dv)) || ((uintptr_t)io->ring & 15) || io->gate_stride < sh.hv ||
        ((uintptr_t)io->state_in & 15) || ((uintptr_t)io->state_out & 15) || ((uintptr_t)io->record & 3))
        return gdn_refuse(who, "rows, rings, states, record and strides: 16-byte aligned, multiples of 8, as wide as a row");
    if (io->state_out && batch->parent) return gdn_refuse(who, "rows of a tree are not final: no state_out");
    if (io->state_out && gdn_overlap(io->state_in, io->state_out, sizeof(float) * (size_t)bt.n_seq * sh.hv * sh.dv * layer->k_dim))
        return gdn_refuse(who, "state_out overlaps state_in");
    StepArgs p;
    p.qkv = (const uint16_t*)io->qkv;
    p.qkv_stride = io->qkv_stride;
    p.a = (const uint16_t*)io->a;
    p.b = (const uint16_t*)io->b;
    p.gate_stride = io->gate_stride;
    p.z = (const uint16_t*)io->z;
    p.z_stride = io->z_stride;
    p.ring = (uint16_t*)io->ring;
    p.state_in = io->state_in;
    p.state_out = io->state_out;
    p.record = io->record;
    p.out = (uint16_t*)io->out;
    p.out_stride = io->out_stride;
    p.total_rows = bt.off[bt.n_seq];
    p.max_rows = 1;
    p.inv_pv = (65536 + sh.dv / 8 - 1) / (sh.dv / 8);
    for (int s = 0; s < bt.n_seq; s++) p.max_rows = std::max(p.max_rows, bt.off[s + 1] - bt.off[s]);
    const hipStream_t st = gdn_stream(stream);
    const bool f16 = layer->dtype == TSV_F16, wide = sh.dv > 128;
#define TSV_GDN_STEP(DK)                                                                                                   \
    (wide ? (f16 ? launch_step<DK, true, 1024>(st, sh, bt, p) : launch_step<DK, false, 1024>(st, sh, bt, p))              \
          : (f16 ? launch_step<DK, true, 512>(st, sh, bt, p) : launch_step<DK, false, 512>(st, sh, bt, p)))
    if (layer->k_dim == 64) return TSV_GDN_STEP(64);
    if (layer->k_dim == 128) return TSV_GDN_STEP(128);
    return TSV_GDN_STEP(256);
#undef TSV_GDN_STEP
}

extern "C" int32_t tsv_gdn_commit(void* stream, const tsv_gdn_layer* layer, const tsv_gdn_batch* batch, const tsv_gdn_commit_io* io) {
    const char* who = "gdn_commit";
    GdnShape sh;
    GdnBatch bt;
    const int rc = gdn_check(who, stream, layer, batch, TSV_MAX_ROWS, &sh, &bt);
    if (rc) return rc;
    if (!io || !io->results || !io->record || !io->ring_in || !io->ring_out || !io->state_in || !io->state_out) return gdn_refuse(who, "null argument");
    if (io->n_layers < 1 || io->n_layers > 65535) return gdn_refuse(who, "1..65535 layers");
    const int64_t state = (int64_t)bt.n_seq * sh.hv * sh.dv * layer->k_dim, ring = (int64_t)bt.n_seq * TSV_GDN_RING * sh.channels;
    const int64_t rec = tsv_gdn_record_bytes(layer, bt.off[bt.n_seq]);
    if (((uintptr_t)io->results & 7) || ((uintptr_t)io->record & 3) || ((uintptr_t)io->ring_in & 15) || ((uintptr_t)io->ring_out & 15) ||
        ((uintptr_t)io->state_in & 15) || ((uintptr_t)io->state_out & 15))
        return gdn_refuse(who, "misaligned argument");
    if (io->n_layers > 1 && (io->record_stride < rec || io->record_stride & 3 || io->ring_stride < ring || io->ring_stride & 7 ||
                             io->state_stride < state || io->state_stride & 3))
        return gdn_refuse(who, "a layer's stride is shorter than a layer or misaligned");
    const int64_t more = io->n_layers - 1;
    if (gdn_overlap(io->state_in, io->state_out, sizeof(float) * (size_t)(more * io->state_stride + state)) ||
        gdn_overlap(io->ring_in, io->ring_out, 2 * (size_t)(more * io->ring_stride + ring)))
        return gdn_refuse(who, "state_out overlaps state_in, or ring_out ring_in");
    CommitArgs p;
    p.results = io->results;
    p.record = io->record;
    p.record_stride = more ? io->record_stride / 4 : 0;
    p.ring_in = (const uint16_t*)io->ring_in;
    p.ring_out = (uint16_t*)io->ring_out;
    p.ring_stride = more ? io->ring_stride : 0;
    p.state_in = io->state_in;
    p.state_out = io->state_out;
    p.state_stride = more ? io->state_stride : 0;
    p.total_rows = bt.off[bt.n_seq];
    const hipStream_t st = gdn_stream(stream);
    if (layer->k_dim == 64) return launch_commit<64>(st, sh, bt, p, io->n_layers);
    if (layer->k_dim == 128) return launch_commit<128>(st, sh, bt, p, io->n_layers);
    return launch_commit<256>(st, sh, bt, p, io->n_layers);
}
