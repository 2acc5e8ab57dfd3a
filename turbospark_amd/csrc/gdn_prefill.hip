// The gated delta rule over prompts, in blocks of 64 rows.  Inside a block, with G the running sum of g, D_ij = e^{G_i - G_j} (j <= i)
// and S the state before it, the recurrence solves to
//     u = T diag(beta) (v - e^G (k S)),   T = (I + A)^-1,   A_ij = beta_i D_ij k_i.k_j  (j < i)
//     o = scale (e^G (q S) + P u),        P_ij = D_ij q_i.k_j                            (j <= i)
//     S <- e^{G_end} S + sum_j e^{G_end - G_j} k_j u_j^T.
// k_gdn_blocks makes T diag(beta), P, k transposed and the decays of every block at once, k_gdn_walk goes through the blocks of a
// sequence with 16 NT columns of one head's state in registers, k_gdn_norm is the gated norm of the result.
//
// Precision: the state is f32 and never rounded; as operands of the bf16 matrix instruction the state, T, u and the difference
// v - e^G kS are two bf16 terms each (2^-18, split2), k and q the rows' own bits (fp16 rows: two terms, exact).  P u, which ends in
// a rounding to the rows' type, is one term by one for bf16 rows and two by two for fp16.  T's inverse is f32 throughout, the running
// sum of g 64 bits, since differences of a long sum are what the decays are made of.
#include "gdn.h"

#include <algorithm>

namespace tsv {

constexpr int BLK = 64, MS = 68;  // rows of a block; row stride (floats) of the 64 x 64 matrices in LDS
constexpr int TFRAGS = 6;         // 16 x 32 fragments of a 64 x 64 lower triangle: row tile w has w / 2 + 1

struct PrefillArgs {
    const uint16_t *q, *k, *v;
    int64_t q_stride, k_stride, v_stride;
    const float *g, *beta;
    const float* state_in;
    float* state_out;
    uint16_t* out;
    int64_t out_stride;
    uint4 *kt, *tp;  // workspace: k transposed per (block, key head); T and P fragments per (block, value head)
    float* gates;    // ... and e^G, e^{G_end - G}
    int32_t tiles;   // column tiles of a head in the walk
    int32_t block_of[TSV_GDN_MAX_SEQ + 1];
};

__device__ __host__ constexpr int tfrag(int w, int ks) { return w < 2 ? w : 2 * w - 2 + ks; }

// eight row values as one bf16 operand, or (fp16) two that sum to them exactly
template <bool F16>
__device__ __forceinline__ void row_terms(const uint4& u, bf16x8* t) {
    if constexpr (!F16) {
        t[0] = __builtin_bit_cast(bf16x8, u);
    } else {
        float x[8];
        row8_f32<true>(u, x);
#pragma unroll
        for (int e = 0; e < 8; e++) {
            __bf16 hi, lo;
            split2(x[e], hi, lo);
            t[0][e] = hi;
            t[1][e] = lo;
        }
    }
}

// c += a b over terms: (1, 1), (1, 2) and (2, 1) whole, (2, 2) without lo * lo
template <int TA, int TB>
__device__ __forceinline__ gf4 mfma_terms(const bf16x8* a, const bf16x8* b, gf4 c) {
    c = mfma_bf16(a[0], b[0], c);
    if constexpr (TB == 2) c = mfma_bf16(a[0], b[1], c);
    if constexpr (TA == 2) c = mfma_bf16(a[1], b[0], c);
    return c;
}

__device__ __forceinline__ int sequence_of(const int32_t* starts, int n, int at) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (starts[mid] <= at) lo = mid;
        else hi = mid;
    }
    return lo;
}

// ---- the blocks' matrices ---------------------------------------------------------------------------------------------------------
// One workgroup per (block, key head), wave w owning rows 16 w ..; the products k.k and q.k are made once and shared by the key head's
// value heads, whose decays make A and P of them.  The inverse: each wave inverts its 16 x 16 diagonal block row by row, a column a
// lane; then wave j does the blocks under diagonal block j, T_ij = -T_ii sum_l A_il T_lj, on the f32 matrix instruction, whose D layout
// is its B operand's when the contraction takes rows 4 gq + r in step r.
template <int DK, bool F16>
__global__ __launch_bounds__(256) void k_gdn_blocks(GdnShape sh, GdnBatch bt, PrefillArgs p) {
    constexpr int TR = F16 ? 2 : 1, KS = DK / 32;
    extern __shared__ uint4 lds[];
    uint4* kf = lds;                                   // [row tile][k step][term][lane]
    float* A = (float*)(kf + 4 * KS * TR * 64);        // [64][MS]
    float* T = A + BLK * MS;
    float* P = T + BLK * MS;
    double* G = (double*)(P + BLK * MS);               // [64]
    float* be = (float*)(G + BLK);                     // [64]
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, l16 = lane & 15, gq = lane >> 4, hk = blockIdx.y;
    const int blk = blockIdx.x, s = sequence_of(p.block_of, bt.n_seq, blk);
    const int r0 = (blk - p.block_of[s]) * BLK, n = min(BLK, bt.off[s + 1] - bt.off[s] - r0);
    const int64_t row0 = bt.off[s] + r0;
    const int mine = 16 * w + l16;
    bf16x8 kr[KS][TR], qr[KS][TR];
#pragma unroll
    for (int t = 0; t < KS; t++) {
        uint4 a = make_uint4(0, 0, 0, 0), b = a;
        if (mine < n) {
            a = *(const uint4*)(p.k + (row0 + mine) * p.k_stride + hk * DK + 32 * t + 8 * gq);
            b = *(const uint4*)(p.q + (row0 + mine) * p.q_stride + hk * DK + 32 * t + 8 * gq);
        }
        row_terms<F16>(a, kr[t]);
        row_terms<F16>(b, qr[t]);
#pragma unroll
        for (int e = 0; e < TR; e++) kf[((w * KS + t) * TR + e) * 64 + lane] = __builtin_bit_cast(uint4, kr[t][e]);
    }
    __syncthreads();
    gf4 kk[4], qk[4];
#pragma unroll
    for (int c = 0; c < 4; c++) {
        kk[c] = qk[c] = gf4{0, 0, 0, 0};
        if (c > w) continue;
#pragma unroll
        for (int t = 0; t < KS; t++) {
            bf16x8 b[TR];
#pragma unroll
            for (int e = 0; e < TR; e++) b[e] = __builtin_bit_cast(bf16x8, kf[((c * KS + t) * TR + e) * 64 + lane]);
            kk[c] = mfma_terms<TR, TR>(kr[t], b, kk[c]);
            qk[c] = mfma_terms<TR, TR>(qr[t], b, qk[c]);
        }
    }
    // k transposed, as the operand of the state's update: rows k_dim, eight block rows a lane
    {
        const uint16_t* kh = (const uint16_t*)kf;
        uint4* to = p.kt + ((int64_t)blk * sh.hk + hk) * (DK / 16 * 2 * TR * 64);
        for (int f = w; f < DK / 16 * 2 * TR; f += 4) {
            const int e = f % TR, ks = f / TR % 2, d = 16 * (f / TR / 2) + l16;
            uint16_t x[8];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const int row = 32 * ks + 8 * gq + i;
                x[i] = kh[((((row >> 4) * KS + (d >> 5)) * TR + e) * 64 + ((d & 31) >> 3) * 16 + (row & 15)) * 8 + (d & 7)];
            }
            to[f * 64 + lane] = make_uint4(x[0] | (uint32_t)x[1] << 16, x[2] | (uint32_t)x[3] << 16, x[4] | (uint32_t)x[5] << 16, x[6] | (uint32_t)x[7] << 16);
        }
    }
    for (int h = hk * sh.rep; h < (hk + 1) * sh.rep; h++) {
        if (w == 0) {
            float g = 0.0f, b = 0.0f;
            if (lane < n) {
                g = p.g[(row0 + lane) * sh.hv + h];
                b = p.beta[(row0 + lane) * sh.hv + h];
                g = g > 0.0f ? 0.0f : g < -1e4f ? -1e4f : g;  // (e^-1e4 is 0; a sum of infinities has no differences)
            }
            double sum = g;
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                const double up = __shfl_up(sum, d);
                if (lane >= d) sum += up;
            }
            G[lane] = sum;
            be[lane] = b;
            const double end = __shfl(sum, 63);
            float* to = p.gates + ((int64_t)blk * sh.hv + h) * 128;
            to[lane] = __expf((float)sum);
            to[64 + lane] = __expf((float)(end - sum));
        }
        __syncthreads();
#pragma unroll
        for (int c = 0; c < 4; c++) {
            if (c > w) continue;
            const int j = 16 * c + l16;
            const double gj = G[j];
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int i = 16 * w + 4 * gq + r;
                const float d = j <= i ? __expf((float)(G[i] - gj)) : 0.0f;
                A[i * MS + j] = j < i ? be[i] * d * kk[c][r] : 0.0f;
                P[i * MS + j] = j <= i ? d * qk[c][r] : 0.0f;
            }
        }
        wave_lds_fence();
        {
            float x[16];  // column l16 of the diagonal block's inverse
            const float* a = A + 16 * w * MS + 16 * w;
#pragma unroll
            for (int i = 0; i < 16; i++) {
                float v = i == l16 ? 1.0f : 0.0f;
#pragma unroll
                for (int j = 0; j < i; j++) v = fmaf(-a[i * MS + j], x[j], v);
                x[i] = v;
                if (gq == 0) T[(16 * w + i) * MS + 16 * w + l16] = v;
            }
        }
        __syncthreads();
        {
            gf4 col[4];  // T_lw, l = w ..
#pragma unroll
            for (int r = 0; r < 4; r++) {
#pragma unroll
                for (int l = 0; l < 4; l++)
                    if (l == w) col[l][r] = T[(16 * w + 4 * gq + r) * MS + 16 * w + l16];
            }
#pragma unroll
            for (int i = 1; i < 4; i++) {
                if (i <= w) continue;
                gf4 x = {0, 0, 0, 0}, y = {0, 0, 0, 0};
#pragma unroll
                for (int l = 0; l < i; l++) {
                    if (l < w) continue;
                    const float4 a = *(const float4*)(A + (16 * i + l16) * MS + 16 * l + 4 * gq);
                    x = mfma_f32(a.x, col[l][0], x);
                    x = mfma_f32(a.y, col[l][1], x);
                    x = mfma_f32(a.z, col[l][2], x);
                    x = mfma_f32(a.w, col[l][3], x);
                }
                const float4 a = *(const float4*)(T + (16 * i + l16) * MS + 16 * i + 4 * gq);
                y = mfma_f32(-a.x, x[0], y);
                y = mfma_f32(-a.y, x[1], y);
                y = mfma_f32(-a.z, x[2], y);
                y = mfma_f32(-a.w, x[3], y);
                col[i] = y;
#pragma unroll
                for (int r = 0; r < 4; r++) T[(16 * i + 4 * gq + r) * MS + 16 * w + l16] = y[r];
            }
        }
        __syncthreads();
        uint4* to = p.tp + ((int64_t)blk * sh.hv + h) * (TFRAGS * (2 + TR) * 64);
#pragma unroll
        for (int ks = 0; ks < 2; ks++) {
            if (ks > w / 2) continue;
            const int f = tfrag(w, ks), j0 = 32 * ks + 8 * gq, row = 16 * w + l16;
            bf16x8 th, tl, ph, pl;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const bool in = j0 + e <= row;  // above the diagonal nothing has been written
                __bf16 hi, lo;
                split2(in ? T[row * MS + j0 + e] * be[j0 + e] : 0.0f, hi, lo);
                th[e] = hi;
                tl[e] = lo;
                split2(in ? P[row * MS + j0 + e] : 0.0f, hi, lo);
                ph[e] = hi;
                pl[e] = lo;
            }
            to[(2 * f) * 64 + lane] = __builtin_bit_cast(uint4, th);
            to[(2 * f + 1) * 64 + lane] = __builtin_bit_cast(uint4, tl);
            to[(2 * TFRAGS + TR * f) * 64 + lane] = __builtin_bit_cast(uint4, ph);
            if constexpr (TR == 2) to[(2 * TFRAGS + TR * f + 1) * 64 + lane] = __builtin_bit_cast(uint4, pl);
        }
        __syncthreads();
    }
}

// ---- the walk through a sequence's blocks --------------------------------------------------------------------------------------------
// One workgroup of four waves per (sequence, value head, 16 NT value channels).  Wave w owns rows 16 w .. of the block and k_dim / 4
// rows of the state, which stay in the accumulators; the state, v - e^G kS and u pass between the waves through LDS as bf16 terms in
// operand order, three barriers a block.  Everything a block reads is asked for one block ahead, into the registers just used.  The
// column tiles of a head read the same k, q, T and P: workgroups are numbered so that they share an XCD's L2.
template <int DK, bool F16, int NT>
__global__ __launch_bounds__(256) void k_gdn_walk(GdnShape sh, GdnBatch bt, PrefillArgs p) {
    constexpr int TR = F16 ? 2 : 1, KS = DK / 32, SD = DK / 64;
    extern __shared__ uint4 lds[];
    uint4* sf = lds;                        // state: [k step][nt][term][lane]
    uint4* rf = sf + KS * NT * 2 * 64;      // v - e^G kS: [k step][nt][term][lane]
    uint4* uf = rf + 2 * NT * 2 * 64;       // u for the output: [k step][nt][term TR][lane]
    uint4* df = uf + 2 * NT * TR * 64;      // u decayed to the block's end, for the state: [k step][nt][term][lane]
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, l16 = lane & 15, gq = lane >> 4;
    const int y = blockIdx.x >> 3, tile = y % p.tiles, hs = y / p.tiles * 8 + (blockIdx.x & 7);
    if (hs >= bt.n_seq * sh.hv) return;
    const int s = hs / sh.hv, h = hs - s * sh.hv, hk = h / sh.rep, first = bt.off[s], rows = bt.off[s + 1] - first;
    const int blocks = p.block_of[s + 1] - p.block_of[s], col0 = tile * 16 * NT + l16;
    const size_t at = ((size_t)hs * sh.dv + col0) * DK + 16 * SD * w + 4 * gq;
    const bool fresh = bt.base[s] == 0;
    gf4 S[SD][NT];
#pragma unroll
    for (int d = 0; d < SD; d++)
#pragma unroll
        for (int t = 0; t < NT; t++) {
            S[d][t] = *(const gf4*)(p.state_in + at + (size_t)16 * t * DK + 16 * d);
            if (fresh) S[d][t] = gf4{0, 0, 0, 0};
        }
    const uint16_t* kp = p.k + (int64_t)first * p.k_stride + hk * DK + 8 * gq;
    const uint16_t* qp = p.q + (int64_t)first * p.q_stride + hk * DK + 8 * gq;
    const uint16_t* vp = p.v + (int64_t)first * p.v_stride + h * sh.dv + col0;
    const int64_t b0 = p.block_of[s];
    const uint4* ktp = p.kt + (b0 * sh.hk + hk) * (DK / 16 * 2 * TR * 64) + SD * w * 2 * TR * 64 + lane;
    const uint4* tpp = p.tp + (b0 * sh.hv + h) * (TFRAGS * (2 + TR) * 64) + lane;
    const float* gp = p.gates + (b0 * sh.hv + h) * 128 + 16 * w + 4 * gq;
    const int64_t kt_step = (int64_t)sh.hk * (DK / 16 * 2 * TR * 64), tp_step = (int64_t)sh.hv * (TFRAGS * (2 + TR) * 64), g_step = (int64_t)sh.hv * 128;
    const int nks = w / 2 + 1, f0 = tfrag(w, 0);

    uint4 kr[KS], qr[KS], ktr[SD][2][TR], tr[2][2], pr[2][TR];
    uint16_t vr[NT][4];
    gf4 eg, ed;
    float e_end;
    auto ask_kq = [&](int b) {
        const int row = min(b * BLK + 16 * w + l16, rows - 1);  // (rows behind the sequence's last: T and k transposed are 0 there)
#pragma unroll
        for (int t = 0; t < KS; t++) kr[t] = *(const uint4*)(kp + row * p.k_stride + 32 * t);
#pragma unroll
        for (int t = 0; t < KS; t++) qr[t] = *(const uint4*)(qp + row * p.q_stride + 32 * t);
    };
    auto ask_v = [&](int b) {
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const int row = min(b * BLK + 16 * w + 4 * gq + r, rows - 1);
#pragma unroll
            for (int t = 0; t < NT; t++) vr[t][r] = vp[row * p.v_stride + 16 * t];
        }
        eg = *(const gf4*)(gp + b * g_step);
    };
    auto ask_t = [&](int b) {
#pragma unroll
        for (int ks = 0; ks < 2; ks++)
            if (ks < nks) {
#pragma unroll
                for (int e = 0; e < 2; e++) tr[ks][e] = tpp[b * tp_step + (2 * (f0 + ks) + e) * 64];
            }
        ed = *(const gf4*)(gp + b * g_step + 64);
    };
    auto ask_kt = [&](int b) {
#pragma unroll
        for (int d = 0; d < SD; d++)
#pragma unroll
            for (int ks = 0; ks < 2; ks++)
#pragma unroll
                for (int e = 0; e < TR; e++) ktr[d][ks][e] = ktp[b * kt_step + ((d * 2 + ks) * TR + e) * 64];
        e_end = p.gates[((b0 + b) * sh.hv + h) * 128 + 63];
    };
    auto ask_p = [&](int b) {
#pragma unroll
        for (int ks = 0; ks < 2; ks++)
            if (ks < nks) {
#pragma unroll
                for (int e = 0; e < TR; e++) pr[ks][e] = tpp[b * tp_step + (2 * TFRAGS + TR * (f0 + ks) + e) * 64];
            }
    };
    // four consecutive contraction indices of one column, as two terms, where the B operand's lane finds its eight
    auto put = [&](uint4* to, int step, int t, int terms, int group, float x0, float x1, float x2, float x3) {
        const float x[4] = {x0, x1, x2, x3};
        __bf16 hi[4], lo[4];
#pragma unroll
        for (int i = 0; i < 4; i++) split2(x[i], hi[i], lo[i]);
        uint2* f = (uint2*)(to + (step * NT + t) * terms * 64) + (group * 16 + l16) * 2 + (gq & 1);
        f[0] = *(uint2*)hi;
        if (terms == 2) f[128] = *(uint2*)lo;
    };
    auto get = [&](const uint4* from, int step, int t, int terms, bf16x8* x) {
#pragma unroll
        for (int e = 0; e < terms; e++) x[e] = __builtin_bit_cast(bf16x8, from[((step * NT + t) * terms + e) * 64 + lane]);
    };
    auto put_state = [&]() {
#pragma unroll
        for (int d = 0; d < SD; d++) {
            const int tile16 = SD * w + d;
#pragma unroll
            for (int t = 0; t < NT; t++) put(sf, tile16 >> 1, t, 2, 2 * (tile16 & 1) + (gq >> 1), S[d][t][0], S[d][t][1], S[d][t][2], S[d][t][3]);
        }
    };
    if (blocks > 0) {
        ask_kq(0);
        ask_v(0);
        ask_t(0);
        ask_kt(0);
        ask_p(0);
        put_state();
    }
    for (int b = 0; b < blocks; b++) {
        const int next = min(b + 1, blocks - 1);
        __syncthreads();
        gf4 ks_[NT], o[NT];
#pragma unroll
        for (int t = 0; t < NT; t++) ks_[t] = o[t] = gf4{0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < KS; i++) {
            bf16x8 kt_[TR], qt_[TR];
            row_terms<F16>(kr[i], kt_);
            row_terms<F16>(qr[i], qt_);
#pragma unroll
            for (int t = 0; t < NT; t++) {
                bf16x8 x[2];
                get(sf, i, t, 2, x);
                ks_[t] = mfma_terms<TR, 2>(kt_, x, ks_[t]);
                o[t] = mfma_terms<TR, 2>(qt_, x, o[t]);
            }
        }
        ask_kq(next);
#pragma unroll
        for (int t = 0; t < NT; t++) {
            float x[4];
#pragma unroll
            for (int r = 0; r < 4; r++) {
                x[r] = fmaf(-eg[r], ks_[t][r], row_f32<F16>(vr[t][r]));
                o[t][r] *= eg[r];
            }
            put(rf, w >> 1, t, 2, 2 * (w & 1) + (gq >> 1), x[0], x[1], x[2], x[3]);
        }
        ask_v(next);
        __syncthreads();
        gf4 u[NT];
#pragma unroll
        for (int t = 0; t < NT; t++) u[t] = gf4{0, 0, 0, 0};
#pragma unroll
        for (int ks = 0; ks < 2; ks++)
            if (ks < nks) {
                const bf16x8 a[2] = {__builtin_bit_cast(bf16x8, tr[ks][0]), __builtin_bit_cast(bf16x8, tr[ks][1])};
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    bf16x8 x[2];
                    get(rf, ks, t, 2, x);
                    u[t] = mfma_terms<2, 2>(a, x, u[t]);
                }
            }
#pragma unroll
        for (int t = 0; t < NT; t++) {
            put(uf, w >> 1, t, TR, 2 * (w & 1) + (gq >> 1), u[t][0], u[t][1], u[t][2], u[t][3]);
            put(df, w >> 1, t, 2, 2 * (w & 1) + (gq >> 1), ed[0] * u[t][0], ed[1] * u[t][1], ed[2] * u[t][2], ed[3] * u[t][3]);
        }
        ask_t(next);
        __syncthreads();
#pragma unroll
        for (int d = 0; d < SD; d++)
#pragma unroll
            for (int t = 0; t < NT; t++) S[d][t] *= e_end;
#pragma unroll
        for (int ks = 0; ks < 2; ks++)
#pragma unroll
            for (int t = 0; t < NT; t++) {
                bf16x8 x[2];
                get(df, ks, t, 2, x);
#pragma unroll
                for (int d = 0; d < SD; d++) {
                    bf16x8 a[TR];
#pragma unroll
                    for (int e = 0; e < TR; e++) a[e] = __builtin_bit_cast(bf16x8, ktr[d][ks][e]);
                    S[d][t] = mfma_terms<TR, 2>(a, x, S[d][t]);
                }
            }
        ask_kt(next);
        put_state();
#pragma unroll
        for (int ks = 0; ks < 2; ks++)
            if (ks < nks) {
                bf16x8 a[TR];
#pragma unroll
                for (int e = 0; e < TR; e++) a[e] = __builtin_bit_cast(bf16x8, pr[ks][e]);
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    bf16x8 x[TR];
                    get(uf, ks, t, TR, x);
                    o[t] = mfma_terms<TR, TR>(a, x, o[t]);
                }
            }
        ask_p(next);
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const int row = b * BLK + 16 * w + 4 * gq + r;
            if (row < rows) {
#pragma unroll
                for (int t = 0; t < NT; t++) p.out[(int64_t)(first + row) * p.out_stride + h * sh.dv + col0 + 16 * t] = row_bits<F16>(sh.scale * o[t][r]);
            }
        }
    }
#pragma unroll
    for (int d = 0; d < SD; d++)
#pragma unroll
        for (int t = 0; t < NT; t++) *(gf4*)(p.state_out + at + (size_t)16 * t * DK + 16 * d) = S[d][t];
}

// ---- the gated norm, in place --------------------------------------------------------------------------------------------------------
// v_dim / 8 of GROUP neighbouring lanes hold a head's row.
template <bool F16>
__global__ __launch_bounds__(256) void k_gdn_norm(GdnShape sh, uint16_t* out, int64_t out_stride, const uint16_t* z, int64_t z_stride, int64_t heads, int group) {
    const int64_t at = ((int64_t)blockIdx.x * 256 + threadIdx.x) / group;
    const int c = (threadIdx.x & (group - 1)) * 8;
    const bool in = at < heads && c < sh.dv;
    const int64_t row = at / sh.hv;
    const int h = (int)(at - row * sh.hv);
    uint16_t* o = out + row * out_stride + h * sh.dv + c;
    float x[8] = {}, y[8] = {}, sum = 0.0f;
    if (in) {
        row8_f32<F16>(*(const uint4*)o, x);
        row8_f32<F16>(*(const uint4*)(z + row * z_stride + h * sh.dv + c), y);
    }
#pragma unroll
    for (int e = 0; e < 8; e++) sum = fmaf(x[e], x[e], sum);
    for (int d = 1; d < group; d <<= 1) sum += __shfl_xor(sum, d);
    if (!in) return;
    const float f = rsqrtf(sum / (float)sh.dv + sh.norm_eps);
    uint32_t b[8];
#pragma unroll
    for (int e = 0; e < 8; e++) b[e] = row_bits<F16>(x[e] * f * sh.norm[c + e] * silu_f32(y[e]));
    *(uint4*)o = make_uint4(b[0] | b[1] << 16, b[2] | b[3] << 16, b[4] | b[5] << 16, b[6] | b[7] << 16);
}

namespace {

struct Sizes {
    int64_t kt, tp, gates, total;  // bytes
};

Sizes workspace_of(const GdnShape& sh, int dk, bool f16, int64_t blocks) {
    const int tr = f16 ? 2 : 1;
    Sizes z;
    z.kt = blocks * sh.hk * (dk / 16 * 2 * tr * 1024);
    z.tp = blocks * sh.hv * (TFRAGS * (2 + tr) * 1024);
    z.gates = blocks * sh.hv * 512;
    z.total = z.kt + z.tp + z.gates;
    return z;
}

int64_t blocks_of(const GdnBatch& bt) {
    int64_t n = 0;
    for (int s = 0; s < bt.n_seq; s++) n += (bt.off[s + 1] - bt.off[s] + BLK - 1) / BLK;
    return n;
}

template <int DK, bool F16>
int launch_blocks(hipStream_t st, const GdnShape& sh, const GdnBatch& bt, const PrefillArgs& p, int blocks) {
    constexpr int TR = F16 ? 2 : 1;
    const size_t lds = (size_t)4 * (DK / 32) * TR * 1024 + 3 * BLK * MS * 4 + BLK * 12;
    static OncePerDevice once;
    const int rc = allow_lds((const void*)k_gdn_blocks<DK, F16>, lds, once);
    if (rc) return rc;
    hipLaunchKernelGGL((k_gdn_blocks<DK, F16>), dim3(blocks, sh.hk), dim3(256), lds, st, sh, bt, p);
    TSV_HIP(hipGetLastError());
    return TSV_OK;
}

template <int DK, bool F16, int NT>
int launch_walk(hipStream_t st, const GdnShape& sh, const GdnBatch& bt, PrefillArgs& p) {
    constexpr int TR = F16 ? 2 : 1;
    const size_t lds = (size_t)(DK / 32 * 2 + 2 * 2 + 2 * TR + 2 * 2) * NT * 1024;
    static OncePerDevice once;
    const int rc = allow_lds((const void*)k_gdn_walk<DK, F16, NT>, lds, once);
    if (rc) return rc;
    p.tiles = sh.dv / (16 * NT);
    const int heads = bt.n_seq * sh.hv;
    hipLaunchKernelGGL((k_gdn_walk<DK, F16, NT>), dim3((heads + 7) / 8 * 8 * p.tiles), dim3(256), lds, st, sh, bt, p);
    TSV_HIP(hipGetLastError());
    return TSV_OK;
}

template <int DK, bool F16>
int launch_prefill(hipStream_t st, const GdnShape& sh, const GdnBatch& bt, PrefillArgs& p, int blocks) {
    if (blocks > 0) {
        const int rc = launch_blocks<DK, F16>(st, sh, bt, p, blocks);
        if (rc) return rc;
    }
    if (sh.dv % 32 == 0) return launch_walk<DK, F16, 2>(st, sh, bt, p);
    return launch_walk<DK, F16, 1>(st, sh, bt, p);
}

}  // namespace

}  // namespace tsv

using namespace tsv;

extern "C" int64_t tsv_gdn_prefill_workspace(const tsv_gdn_layer* layer, const tsv_gdn_batch* batch) {
    GdnShape sh;
    GdnBatch bt;
    if (gdn_check("gdn_prefill_workspace", nullptr, layer, batch, 0, &sh, &bt)) return -1;
    return std::max<int64_t>(16, workspace_of(sh, layer->k_dim, layer->dtype == TSV_F16, blocks_of(bt)).total);
}

extern "C" int32_t tsv_gdn_prefill(void* stream, const tsv_gdn_layer* layer, const tsv_gdn_batch* batch, const tsv_gdn_prefill_io* io) {
    const char* who = "gdn_prefill";
    GdnShape sh;
    GdnBatch bt;
    const int rc = gdn_check(who, stream, layer, batch, 0, &sh, &bt);
    if (rc) return rc;
    if (!io || !io->g || !io->beta || !io->state_in || !io->state_out || !io->workspace || (io->z && !sh.norm)) return gdn_refuse(who, "null argument");
    if (batch->parent) return gdn_refuse(who, "prompt rows are chains");
    const int dk = layer->k_dim;
    const int64_t kw = (int64_t)sh.hk * dk, vw = (int64_t)sh.hv * sh.dv;
    if (!gdn_rows_ok(io->q, io->q_stride, kw) || !gdn_rows_ok(io->k, io->k_stride, kw) || !gdn_rows_ok(io->v, io->v_stride, vw) ||
        !gdn_rows_ok(io->out, io->out_stride, vw) || (io->z && !gdn_rows_ok(io->z, io->z_stride, vw)) || ((uintptr_t)io->state_in & 15) ||
        ((uintptr_t)io->state_out & 15) || ((uintptr_t)io->workspace & 15) || ((uintptr_t)io->g & 3) || ((uintptr_t)io->beta & 3))
        return gdn_refuse(who, "rows, states, workspace and strides: 16-byte aligned, multiples of 8, as wide as a row");
    if (io->out == io->q || io->out == io->k || io->out == io->v || io->out == io->z) return gdn_refuse(who, "out may not be the input rows");
    if (gdn_overlap(io->state_in, io->state_out, sizeof(float) * (size_t)(bt.n_seq * vw * dk))) return gdn_refuse(who, "state_out overlaps state_in");
    const bool f16 = layer->dtype == TSV_F16;
    const int64_t blocks = blocks_of(bt);
    const Sizes z = workspace_of(sh, dk, f16, blocks);
    if (io->workspace_bytes < z.total) return gdn_refuse(who, "the workspace is smaller than tsv_gdn_prefill_workspace says");
    PrefillArgs p;
    p.q = (const uint16_t*)io->q;
    p.k = (const uint16_t*)io->k;
    p.v = (const uint16_t*)io->v;
    p.q_stride = io->q_stride;
    p.k_stride = io->k_stride;
    p.v_stride = io->v_stride;
    p.g = io->g;
    p.beta = io->beta;
    p.state_in = io->state_in;
    p.state_out = io->state_out;
    p.out = (uint16_t*)io->out;
    p.out_stride = io->out_stride;
    uint8_t* ws = (uint8_t*)io->workspace;
    p.kt = (uint4*)ws;
    p.tp = (uint4*)(ws + z.kt);
    p.gates = (float*)(ws + z.kt + z.tp);
    p.block_of[0] = 0;
    for (int s = 0; s < bt.n_seq; s++) p.block_of[s + 1] = p.block_of[s] + (bt.off[s + 1] - bt.off[s] + BLK - 1) / BLK;
    const hipStream_t st = (hipStream_t)stream;
    int done;
    if (dk == 64) done = f16 ? launch_prefill<64, true>(st, sh, bt, p, (int)blocks) : launch_prefill<64, false>(st, sh, bt, p, (int)blocks);
    else if (dk == 128) done = f16 ? launch_prefill<128, true>(st, sh, bt, p, (int)blocks) : launch_prefill<128, false>(st, sh, bt, p, (int)blocks);
    else done = f16 ? launch_prefill<256, true>(st, sh, bt, p, (int)blocks) : launch_prefill<256, false>(st, sh, bt, p, (int)blocks);
    if (done || !io->z || !bt.off[bt.n_seq]) return done;
    int group = 2;
    while (group * 8 < sh.dv) group *= 2;
    const int64_t heads = (int64_t)bt.off[bt.n_seq] * sh.hv, wgs = (heads * group + 255) / 256;
    if (f16) hipLaunchKernelGGL((k_gdn_norm<true>), dim3((uint32_t)wgs), dim3(256), 0, st, sh, p.out, p.out_stride, (const uint16_t*)io->z, io->z_stride, heads, group);
    else hipLaunchKernelGGL((k_gdn_norm<false>), dim3((uint32_t)wgs), dim3(256), 0, st, sh, p.out, p.out_stride, (const uint16_t*)io->z, io->z_stride, heads, group);
    TSV_HIP(hipGetLastError());
    return TSV_OK;
}
