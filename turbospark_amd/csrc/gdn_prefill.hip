// The gated delta rule over prompts, in blocks of 64 rows.  Inside a block, with G the running sum of g, D_ij = e^{G_i - G_j} (j <= i)
// and S the state before it, the recurrence solves to
//     u = T diag(beta) (v - e^G (k S)),   T = (I + A)^-1,   A_ij = beta_i D_ij k_i.k_j  (j < i)
//     o = scale (e^G (q S) + P u),        P_ij = D_ij q_i.k_j                            (j <= i)
//     S <- e^{G_end} S + sum_j e^{G_end - G_j} k_j u_j^T.
// k_gdn_blocks makes T diag(beta), P, k transposed and the decays of every block at once, k_gdn_walk goes through the blocks of a
// sequence with 16 NT columns of one head's state in registers, k_gdn_norm is the gated norm of the result.
//
// Precision: the state is f32 and never rounded.  In what makes it, k S and k^T u, it and u are three bf16 terms each (2^-27, split3), k the
// rows' own bits (fp16 rows: two terms, exact); k k^T is made of the rows' bits as they are, T (v - e^G kS) by the f32 instruction from f32
// operands.  The state is then as far off as one of plain 32-bit sums, 1.2e-7 to 1.5e-7 of its norm (two terms throughout: 5e-6).
// What only goes to the output, q S and P u, has two terms by two (2^-18, split2), so that the rows' own rounding is what a result is off by
// (P u one term by one left bf16 rows 2.6e-3 off for their rounding's 1.7e-3).  T's inverse is f32 throughout, the running sum of g 64 bits,
// since differences of a long sum are what the decays are made of.  The gated norm reads o in f32 from the workspace: rounded to the rows'
// type before, fp16 rows had no o above 65504 and no bits in a small one, and the result of bf16 rows was half a step further off.
#include "gdn.h"

#include <algorithm>
#include <cmath>

namespace tsv {

constexpr int BLK = 64, MS = 68;  // rows of a block; row stride (floats) of the 64 x 64 matrices in LDS
constexpr int TFRAGS = 6;         // 16 x 32 fragments of a 64 x 64 lower triangle: row tile w has w / 2 + 1
constexpr int TTILES = 10;        // 16 x 16 tiles of it: row tile w has w + 1
constexpr int TP_UNITS = (TTILES + 2 * TFRAGS) * 64;  // 16-byte units of T in f32 tiles and P in fragments of two terms, of a (block, value head)

struct PrefillArgs {
    const uint16_t *q, *k, *v;
    int64_t q_stride, k_stride, v_stride;
    const float *g, *beta;
    const float* state_in;
    float* state_out;
    uint16_t* out;
    int64_t out_stride;
    uint4 *kt, *tp;  // workspace: k, q and k transposed per (block, key head); T and P fragments per (block, value head)
    float* gates;    // ... and e^G, e^{G_end - G}
    float* ends;     // ... and per (segment but a sequence's last, value head) what a segment does to a state: [v_dim][k_dim] from nothing, then [k_dim][k_dim]
    float* starts;   // ... and the states that sequences of several segments start from: state_out may be state_in
    float* o32;      // ... and the rows of o that the gated norm reads
    int32_t tiles;   // column tiles of a head in the walk
    int32_t bring;   // the walk has a wave that brings data into the L2
    int32_t split;   // the blocks' matrices: a workgroup per value head
    int32_t seg_blocks;  // blocks of a segment, the last of a sequence may have fewer
    int32_t block_of[TSV_GDN_MAX_SEQ + 1], seg_of[TSV_GDN_MAX_SEQ + 1];  // first block and first segment of every sequence
};

// fragments (1 KiB: a wave's 16 bytes a lane) of a (block, key head): k and q by row tile, k transposed by 16 of k_dim
template <int DK, int TR>
constexpr int KFRAGS = 4 * (DK / 32) * TR;

__device__ __host__ constexpr int tfrag(int w, int ks) { return w < 2 ? w : 2 * w - 2 + ks; }
__device__ __host__ constexpr int ttile(int w, int j) { return w * (w + 1) / 2 + j; }

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

// c += a b over terms, without those products of two terms that are 2^-9 and less of the operands' own last terms
template <int TA, int TB>
__device__ __forceinline__ gf4 mfma_terms(const bf16x8* a, const bf16x8* b, gf4 c) {
    constexpr int MOST = TA > TB ? TA : TB;
#pragma unroll
    for (int i = 0; i < TA; i++)
#pragma unroll
        for (int j = 0; j < TB; j++)
            if (i + j < MOST) c = mfma_bf16(a[i], b[j], c);
    return c;
}

// the product of the rows' own bits
template <bool F16>
__device__ __forceinline__ gf4 mfma_rows(const uint4& a, const uint4& b, gf4 c) {
    typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
    if constexpr (F16) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else return mfma_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c);
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
// value heads, whose decays make A and P of them.  The inverse: each wave inverts its 16 x 16 diagonal block; then wave j does the blocks
// under diagonal block j, T_ij = -T_ii sum_l A_il T_lj, on the f32 matrix instruction, whose D layout is its B operand's when the
// contraction takes rows 4 gq + r in step r.  8192 rows, 16 key and 32 value heads of 128: 78 us for 69 MB read and 195 MB written
// (3.4 TB/s); the waits of one workgroup, three on a compute unit, bound it.  Few blocks have a workgroup per value head instead
// (split), each making the products again: the whole call with 65 rows, 8 heads over 4, 17.8 us against 21.1; 1024 rows, 32 over 16, 43.7
// against 45.0; 700 and 800 rows of heads of their own the same.
// Where P's value (i, j) lies in LDS: rows of 64 values, whose eight 16-byte units take turns from row to row (a column of them, as the
// fragments are read, would else lie in two banks)
__device__ __forceinline__ int p_at(int i, int j) { return i * BLK + (((j >> 3) ^ (i & 7)) << 3) + (j & 7); }
// 16-byte units of LDS that hold k's rows, then P
template <int DK>
constexpr int blocks_operands = DK > 2 * BLK ? BLK * DK / 8 : 2 * BLK * BLK / 8;

// What a head's decays are in a block.  e^{G_i - G_j} of rows in different row tiles is made of three factors of at most 1: from j to its
// tile's end, the tiles between, and from the start of i's tile to i; inside a tile it is one exponential of a 64-bit difference.
// (Two heads' at a time, without what can be made of the others: three workgroups fit a compute unit's LDS.)
struct BlockGates {
    double G[BLK];
    float beta[BLK], from_start[BLK], to_end[BLK];
};
constexpr int GATE_HEADS = 2;

template <int DK, bool F16>
__global__ __launch_bounds__(256, 3) void k_gdn_blocks(GdnShape sh, GdnBatch bt, PrefillArgs p) {
    constexpr int TR = F16 ? 2 : 1, KS = DK / 32;
    extern __shared__ uint4 lds[];
    uint4* kf = lds;                                   // [row tile][k step][lane], as the rows have them
    uint16_t* P = (uint16_t*)lds;                      // [term][64][64], where the operands were
    float* A = (float*)(lds + blocks_operands<DK>);  // [64][MS]
    float* T = A + BLK * MS;
    BlockGates* gates = (BlockGates*)(T + BLK * MS);   // of GATE_HEADS heads
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), l16 = lane & 15, gq = lane >> 4;
    const int hk = p.split ? blockIdx.y / sh.rep : blockIdx.y, h0 = p.split ? blockIdx.y : hk * sh.rep, h1 = p.split ? h0 + 1 : h0 + sh.rep;
    const bool writes = h0 == hk * sh.rep;  // k, q and k transposed, for all of the key head's value heads
    const int blk = blockIdx.x, s = sequence_of(p.block_of, bt.n_seq, blk);
    const int r0 = (blk - p.block_of[s]) * BLK, n = min(BLK, bt.off[s + 1] - bt.off[s] - r0);
    const int64_t row0 = bt.off[s] + r0;
    const int mine = 16 * w + l16;
    float next_g = 0.0f, next_b = 0.0f;  // of the head this wave makes the decays of
    auto ask_gates = [&](int h) {
        const int64_t at = (row0 + min(lane, n - 1)) * sh.hv + min(h, h1 - 1);
        next_g = p.g[at];
        next_b = p.beta[at];
    };
    ask_gates(h0 + w);
    uint4 kr[KS], qr[KS];
    uint4* rows_out = p.kt + ((int64_t)blk * sh.hk + hk) * (3 * KFRAGS<DK, TR> * 64);
#pragma unroll
    for (int t = 0; t < KS; t++) {
        kr[t] = qr[t] = make_uint4(0, 0, 0, 0);
        if (mine < n) {
            kr[t] = *(const uint4*)(p.k + (row0 + mine) * p.k_stride + hk * DK + 32 * t + 8 * gq);
            qr[t] = *(const uint4*)(p.q + (row0 + mine) * p.q_stride + hk * DK + 32 * t + 8 * gq);
        }
        kf[(w * KS + t) * 64 + lane] = kr[t];
        if (!writes) continue;
        bf16x8 k[TR], q[TR];
        row_terms<F16>(kr[t], k);
        row_terms<F16>(qr[t], q);
#pragma unroll
        for (int e = 0; e < TR; e++) {
            const int f = (w * KS + t) * TR + e;
            rows_out[f * 64 + lane] = __builtin_bit_cast(uint4, k[e]);
            rows_out[(KFRAGS<DK, TR> + f) * 64 + lane] = __builtin_bit_cast(uint4, q[e]);
        }
    }
    __syncthreads();
    gf4 kk[4], qk[4];  // of the rows' own bits: exact products
#pragma unroll
    for (int c = 0; c < 4; c++) {
        kk[c] = qk[c] = gf4{0, 0, 0, 0};
        if (c > w) continue;
#pragma unroll
        for (int t = 0; t < KS; t++) {
            const uint4 b = kf[(c * KS + t) * 64 + lane];
            kk[c] = mfma_rows<F16>(kr[t], b, kk[c]);
            qk[c] = mfma_rows<F16>(qr[t], b, qk[c]);
        }
    }
    // k transposed, as the operand of the state's update: rows k_dim, eight block rows a lane
    if (writes) {
        const uint16_t* kh = (const uint16_t*)kf;
        uint4* to = rows_out + 2 * KFRAGS<DK, TR> * 64;
        for (int f = w; f < DK / 16 * 2; f += 4) {
            const int ks = f % 2, d = 16 * (f / 2) + l16;
            uint16_t x[8];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const int row = 32 * ks + 8 * gq + i;
                x[i] = kh[(((row >> 4) * KS + (d >> 5)) * 64 + ((d & 31) >> 3) * 16 + (row & 15)) * 8 + (d & 7)];
            }
            bf16x8 k[TR];
            row_terms<F16>(make_uint4(x[0] | (uint32_t)x[1] << 16, x[2] | (uint32_t)x[3] << 16, x[4] | (uint32_t)x[5] << 16, x[6] | (uint32_t)x[7] << 16), k);
#pragma unroll
            for (int e = 0; e < TR; e++) to[(f * TR + e) * 64 + lane] = __builtin_bit_cast(uint4, k[e]);
        }
    }
    for (int h = h0; h < h1; h++) {
        const int turn = (h - h0) % GATE_HEADS;
        if (turn == 0) {  // the next heads, one a wave
            if (w < GATE_HEADS && h + w < h1) {
                const float b = lane < n ? next_b : 0.0f;
                float g = next_g > 0.0f ? 0.0f : next_g < -1e4f ? -1e4f : next_g;  // (e^-1e4 is 0; a sum of infinities has no differences)
                if (lane >= n) g = 0.0f;
                double sum = g;
#pragma unroll
                for (int d = 1; d < 64; d <<= 1) {
                    const double up = __shfl_up(sum, d);
                    if (lane >= d) sum += up;
                }
                double end[4];  // at the row tiles' ends
#pragma unroll
                for (int t = 0; t < 4; t++) end[t] = __shfl(sum, 16 * t + 15);
                const double before = gq == 0 ? 0.0 : gq == 1 ? end[0] : gq == 2 ? end[1] : end[2];
                const double mine_end = gq == 0 ? end[0] : gq == 1 ? end[1] : gq == 2 ? end[2] : end[3];
                BlockGates& o = gates[w];
                o.G[lane] = sum;
                o.beta[lane] = b;
                o.from_start[lane] = __expf((float)(sum - before));
                o.to_end[lane] = __expf((float)(mine_end - sum));
                float* to = p.gates + ((int64_t)blk * sh.hv + h + w) * 128;
                to[lane] = __expf((float)sum);
                to[64 + lane] = __expf((float)(end[3] - sum));
            }
            ask_gates(h + GATE_HEADS + w);
            __syncthreads();
        }
        const BlockGates& gt = gates[turn];
        {
            const float4 be4 = *(const float4*)(gt.beta + 16 * w + 4 * gq), st4 = *(const float4*)(gt.from_start + 16 * w + 4 * gq);
            const float be[4] = {be4.x, be4.y, be4.z, be4.w}, st[4] = {st4.x, st4.y, st4.z, st4.w};
            auto put_p = [&](int i, int j, float x) {
                __bf16 hi, lo;
                split2(x, hi, lo);
                P[p_at(i, j)] = __builtin_bit_cast(uint16_t, hi);
                P[BLK * BLK + p_at(i, j)] = __builtin_bit_cast(uint16_t, lo);
            };
#pragma unroll
            for (int c = 0; c < 3; c++) {
                if (c >= w) continue;
                const int j = 16 * c + l16;
                float x = gt.to_end[j];
                if (w - c > 1) x *= __expf((float)(gt.G[16 * w - 1] - gt.G[16 * c + 15]));
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const int i = 16 * w + 4 * gq + r;
                    const float d = st[r] * x;
                    A[i * MS + j] = be[r] * d * kk[c][r];
                    put_p(i, j, d * qk[c][r]);
                }
            }
            const int j = 16 * w + l16;
            const double gj = gt.G[j];
            gf4 kd, qd;
#pragma unroll
            for (int c = 0; c < 4; c++)
                if (c == w) kd = kk[c], qd = qk[c];
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int i = 16 * w + 4 * gq + r;
                const float d = j <= i ? __expf((float)(gt.G[i] - gj)) : 0.0f;
                A[i * MS + j] = j < i ? be[r] * d * kd[r] : 0.0f;
                put_p(i, j, j <= i ? d * qd[r] : 0.0f);
            }
        }
        wave_lds_fence();
        invert_lower16(A + 16 * w * MS + 16 * w, MS, T + 16 * w * MS + 16 * w, MS, l16, gq);
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
        uint4* to = p.tp + ((int64_t)blk * sh.hv + h) * TP_UNITS;
        const int row = 16 * w + l16;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            if (j > w) continue;
            const int j0 = 16 * j + 4 * gq;
            float4 x = *(const float4*)(T + row * MS + j0);  // (above the diagonal nothing has been written)
            const float4 be = *(const float4*)(gt.beta + j0);
            x.x = j0 <= row ? x.x * be.x : 0.0f;
            x.y = j0 + 1 <= row ? x.y * be.y : 0.0f;
            x.z = j0 + 2 <= row ? x.z * be.z : 0.0f;
            x.w = j0 + 3 <= row ? x.w * be.w : 0.0f;
            to[ttile(w, j) * 64 + lane] = __builtin_bit_cast(uint4, x);
        }
#pragma unroll
        for (int ks = 0; ks < 2; ks++) {
            if (ks > w / 2) continue;
            const int f = tfrag(w, ks), j0 = 32 * ks + 8 * gq;
            const bool zero = 32 * ks + 8 * gq >= 16 * (w + 1);  // (columns of row tiles behind this one)
#pragma unroll
            for (int e = 0; e < 2; e++) to[(TTILES + 2 * f + e) * 64 + lane] = zero ? make_uint4(0, 0, 0, 0) : *(const uint4*)(P + e * BLK * BLK + p_at(row, j0));
        }
        __syncthreads();
    }
}

// ---- the walk through a sequence's blocks --------------------------------------------------------------------------------------------
// One workgroup of eight waves per (sequence, value head, 16 NT value channels).  Waves 0 to 3 take the state from block to block:
// wave w owns rows 16 w .. of the block and k_dim / 4 rows of the state, which stay in its accumulators; the state and u pass between
// them through LDS as bf16 terms in operand order, v - e^G kS as the f32 instruction takes it, three barriers a block.  Waves 4 to 7, one
// beside each of them on a SIMD, make the output rows from the same LDS (q S behind the first barrier, P u behind the third) and hand the
// others v, transposed, and the decays through LDS: a load or store of any width holds the CU's address unit for 16 cycles, which bounds a block (12 and 11 of
// them a wave here), so two-byte ones are taken together.  Everything a block reads is asked for one block ahead, into the registers
// just used: the scheduling fences keep the compiler from asking earlier, which would take copies and, with them, waits.  The column
// tiles of a head read the same k, q, T and P: workgroups are numbered so that they share an XCD's L2.
// Where few heads leave most of the chip idle a sequence is cut into segments.  A block takes every column of the state alike, S -> M S + c
// with M the same for all, so a first launch (ENDS) walks all segments but the last at once, from nothing with the rows' v and from the
// unit matrix with v = 0; the walk of segment n then begins with n products M S + c of its own 16 NT columns.
// 8192 rows of 32 heads of 128, one column tile on each compute unit: 200 us, 1.6 us a block: the three hand-overs through LDS that follow
// each other, 0.6 of it the address unit's 92 loads and stores.  235 where o goes out in f32 for the norm (twice the bytes).  Of two
// column tiles the output's waves make the second's u: T r takes 4 to 16 f32 products a row tile, and a SIMD whose two waves have row tiles
// w and 3 - w has 20 of the 80 (segments of 32768 rows: 238 us where the state's waves make them all, 219 so).
#define GDN_FENCE __builtin_amdgcn_sched_barrier(0)
// all loads have arrived, and the compiler knows: what is under way before a loop would else count in every wait inside it
#define GDN_ARRIVED                            \
    GDN_FENCE;                                 \
    __builtin_amdgcn_s_waitcnt(0x0F70);        \
    GDN_FENCE
// The wave that brings data into the L2 pays where one workgroup has a compute unit and reads what the last-level cache may not hold any
// more: of fp16 rows, whose k and q are two terms each, from 128 MB of matrices on (16 / 32 heads of 128: 3000 rows, 105 MB, 116 us with it
// and 109 without; 5000, 176 MB, 201 and 212; 8192, 288 MB, 355 and 398).  bf16 rows are 2 to 5% faster without it at every length, heads
// of 64 up to 12%; k_dim 256 has no registers for it.
template <int DK, bool F16, int NT>
constexpr int walk_threads = NT == 1 && F16 && DK == 128 ? 576 : 512;
constexpr int64_t BRING_FROM = 128 << 20;

template <int DK, bool F16, int NT>
struct Walk {
    static constexpr int TR = F16 ? 2 : 1, KS = DK / 32, SD = DK / 64;
    // LDS, in operand order [k step][nt][term][lane], but for the difference v - e^G kS, in f32 [row tile][nt][lane]
    static constexpr int S_AT = 0, R_AT = KS * NT * 3 * 64, U_AT = R_AT + 4 * NT * 64, D_AT = U_AT + 2 * NT * 2 * 64;
    // v as [column][VS], the decays e^G and e^{G_end - G}, and the output rows on their way out, a region per wave (f32 rows of OS values)
    static constexpr int V_AT = D_AT + 2 * NT * 3 * 64, VS = 72, G_AT = V_AT + 16 * NT * VS / 8, O_AT = G_AT + 32, OS = 16 * NT + 4, LDS = O_AT + 64 * OS / 4;
    uint4* lds;
    int lane, w, l16, gq;

    // four consecutive contraction indices of one column, as two or three terms, where the B operand's lane finds its eight
    template <int TERMS>
    __device__ __forceinline__ void put(int to, int step, int t, int group, gf4 x) const {
        uint2* f = (uint2*)(lds + to + (step * NT + t) * TERMS * 64) + (group * 16 + l16) * 2 + (gq & 1);
#pragma unroll
        for (int e = 0; e < TERMS; e++) {
            const uint2 two = make_uint2(row_pair<false>(x[0], x[1]), row_pair<false>(x[2], x[3]));
            f[128 * e] = two;
            x -= gf4{__uint_as_float(two.x << 16), __uint_as_float(two.x & 0xFFFF0000u), __uint_as_float(two.y << 16), __uint_as_float(two.y & 0xFFFF0000u)};
        }
    }
    // the same in f32, a tile of a product as it comes: one that the f32 instruction's contraction takes in rows 4 gq + r
    __device__ __forceinline__ void put_f32(int to, int t, gf4 x) const { lds[to + (w * NT + t) * 64 + lane] = __builtin_bit_cast(uint4, x); }
    // the first READ of an operand's terms
    template <int TERMS, int READ = TERMS>
    __device__ __forceinline__ void get(int from, int step, int t, bf16x8* x) const {
#pragma unroll
        for (int e = 0; e < READ; e++) x[e] = __builtin_bit_cast(bf16x8, lds[from + ((step * NT + t) * TERMS + e) * 64 + lane]);
    }
};

// What a walk is for: o in the rows' type, o in f32 for the norm behind it, or what the segments do to a state.
enum WalkFor { ROWS, NORM, SEGMENTS };

template <int DK, bool F16, int NT, WalkFor FOR>
__global__ __launch_bounds__((walk_threads<DK, F16, NT>), 2) void k_gdn_walk(GdnShape sh, GdnBatch bt, PrefillArgs p) {
    typedef Walk<DK, F16, NT> W;
    constexpr bool ENDS = FOR == SEGMENTS;
    constexpr int TR = W::TR, KS = W::KS, SD = W::SD;
    extern __shared__ uint4 lds[];
    const int tid = threadIdx.x, lane = tid & 63, w8 = __builtin_amdgcn_readfirstlane(tid >> 6), w = w8 & 3, l16 = lane & 15, gq = lane >> 4;
    const W x{lds, lane, w, l16, gq};
    // a key head's workgroups, its value heads' column tiles, are 8 apart: the same XCD
    const int y = blockIdx.x >> 3, of = p.tiles * sh.rep, ks_ = y / of * 8 + (blockIdx.x & 7), tile = y % p.tiles;
    const int segs = p.seg_of[bt.n_seq];
    if (ks_ >= segs * sh.hk) return;
    const int seg_at = ks_ / sh.hk, hk = ks_ - seg_at * sh.hk, h = hk * sh.rep + y % of / p.tiles;
    const int s = sequence_of(p.seg_of, bt.n_seq, seg_at), seg = seg_at - p.seg_of[s], hs = s * sh.hv + h;
    const bool last = seg_at + 1 == p.seg_of[s + 1];
    const bool whole = seg == 0 && last;
    if (ENDS && last) return;
    const int skip = seg * p.seg_blocks, first = bt.off[s] + skip * BLK;
    const int rows = last ? bt.off[s + 1] - first : p.seg_blocks * BLK, blocks = (rows + BLK - 1) / BLK;
    const int64_t b0 = p.block_of[s] + skip;
    const bool unit = ENDS && tile * 16 * NT >= sh.dv;  // columns of the unit matrix, not of the rows' v
    const float* ends = p.ends + ((int64_t)(p.seg_of[s] - s) * sh.hv + h) * (sh.dv + DK) * DK;  // of the sequence's first segment
    const int64_t ends_step = (int64_t)sh.hv * (sh.dv + DK) * DK;
    // uniform addresses of the block asked for, and what a lane adds to them (in bytes)
    const char* tpp = (const char*)(p.tp + (b0 * sh.hv + h) * TP_UNITS);
    const char* gp = (const char*)(p.gates + (b0 * sh.hv + h) * 128);
    const int64_t tp_step = (int64_t)sh.hv * (TP_UNITS * 16), g_step = (int64_t)sh.hv * 512;
    const uint32_t lane16 = lane * 16;
    // (waves of rows 0 and 16 have one fragment of T and P where the others have two: they ask for theirs twice and clear the copy, so
    // that every wave has the same loads under way and a wait is for the ones it needs)
    const uint32_t second = w < 2 ? 0u : 0xFFFFFFFFu;
    const int f0 = tfrag(w, 0), f1 = w < 2 ? f0 : f0 + 1;
    auto fragment = [&](const uint4& f, int ks) {
        if (ks == 0) return __builtin_bit_cast(bf16x8, f);
        return __builtin_bit_cast(bf16x8, make_uint4(f.x & second, f.y & second, f.z & second, f.w & second));
    };
    // u = T (v - e^G kS) of row tile i, columns of tile t, on the f32 instruction, and what is read of it
    auto ask_t = [&](uint4* tr, int i) {  // (as many for every wave: row tile i has i + 1 tiles)
#pragma unroll
        for (int j = 0; j < 4; j++) tr[j] = *(const uint4*)(tpp + ttile(i, min(j, i)) * 1024 + lane16);
    };
    auto solve = [&](const uint4* tr, int i, int t) {
        gf4 d[4];
#pragma unroll
        for (int j = 0; j < 4; j++) d[j] = __builtin_bit_cast(gf4, lds[W::R_AT + (j * NT + t) * 64 + lane]);
        const gf4 ed = *(const gf4*)((const float*)(lds + W::G_AT) + 64 + 16 * i + 4 * gq);
        GDN_FENCE;
        gf4 u = {0, 0, 0, 0}, u2 = u;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            if (j > i) break;
            const gf4 a = __builtin_bit_cast(gf4, tr[j]);
            u = mfma_f32(a[0], d[j][0], u);
            u2 = mfma_f32(a[1], d[j][1], u2);
            u = mfma_f32(a[2], d[j][2], u);
            u2 = mfma_f32(a[3], d[j][3], u2);
        }
        u += u2;
        x.template put<3>(W::D_AT, i >> 1, t, 2 * (i & 1) + (gq >> 1), ed * u);
        if constexpr (!ENDS) x.template put<2>(W::U_AT, i >> 1, t, 2 * (i & 1) + (gq >> 1), u);
    };
    if (walk_threads<DK, F16, NT> > 512 && w8 == 8) {  // ---- the wave that brings what is four blocks ahead into the XCD's L2, this workgroup's share of it
        constexpr int AHEAD = 4, LINES = 3 * KFRAGS<DK, TR> * 8 + TP_UNITS / 8, SHARE = 3;
        const char* kreg = (const char*)(p.kt + (b0 * sh.hk + hk) * (3 * KFRAGS<DK, TR> * 64));
        const int64_t k_step = (int64_t)sh.hk * (3 * KFRAGS<DK, TR> * 1024);
        const char* vreg = (const char*)(p.v + (int64_t)first * p.v_stride + h * sh.dv + (unit ? 0 : tile * 16 * NT));
        uint32_t got[AHEAD][SHARE + 1] = {};
        if constexpr (!ENDS)
            for (int q = 0; q < 2 * seg; q++) __builtin_amdgcn_s_barrier();
        for (int b = 0; b < blocks; b += AHEAD)
#pragma unroll
            for (int j = 0; j < AHEAD; j++) {
                if (b + j >= blocks) break;
                const int at = min(b + j + AHEAD, blocks - 1);
#pragma unroll
                for (int i = 0; i < SHARE + 1; i++) asm volatile("" ::"v"(got[j][i]));  // what was asked for AHEAD blocks ago is there
#pragma unroll
                for (int i = 0; i < SHARE; i++) {
                    const int line = min((i * p.tiles + tile) * 64 + lane, LINES - 1) * 128;
                    constexpr int KB = 3 * KFRAGS<DK, TR> * 1024;
                    got[j][i] = *(const uint32_t*)(line < KB ? kreg + at * k_step + line : tpp + at * tp_step + (line - KB));
                }
                got[j][SHARE] = *(const uint32_t*)(vreg + (int64_t)min(at * BLK + lane, rows - 1) * (2 * p.v_stride));
                __builtin_amdgcn_s_barrier();
                __builtin_amdgcn_s_barrier();
                __builtin_amdgcn_s_barrier();
            }
        return;
    }
    if (w8 >= 4) {  // ---- the output's waves
        const char* qp = (const char*)(p.kt + ((b0 * sh.hk + hk) * 3 + 1) * (KFRAGS<DK, TR> * 64) + w * KS * TR * 64);
        const int64_t q_step = (int64_t)sh.hk * (3 * KFRAGS<DK, TR> * 1024);
        uint4 qr[KS][TR], pr[2][2], tr[4];  // (tr: of the row tile that this SIMD's other wave has least of)
        auto ask_q = [&]() {
#pragma unroll
            for (int t = 0; t < KS; t++)
#pragma unroll
                for (int e = 0; e < TR; e++) qr[t][e] = *(const uint4*)(qp + (t * TR + e) * 1024 + lane16);
        };
        auto ask_p = [&]() {
#pragma unroll
            for (int e = 0; e < 2; e++) {
                pr[0][e] = *(const uint4*)(tpp + (TTILES + 2 * f0 + e) * 1024 + lane16);
                pr[1][e] = *(const uint4*)(tpp + (TTILES + 2 * f1 + e) * 1024 + lane16);
            }
        };
        // a lane's piece of the rows: a quarter of row lane / 4 of the wave's sixteen
        typedef uint32_t piece __attribute__((ext_vector_type(2 * NT)));
        const int prow = 16 * w + (lane >> 2), pcol = (lane & 3) * 4 * NT;
        const uint16_t* vp = p.v + (int64_t)first * p.v_stride + h * sh.dv + (unit ? 0 : tile * 16 * NT) + pcol;
        constexpr int OB = FOR == NORM ? 4 : 2;  // bytes of a value of o
        const int64_t o_stride = FOR == NORM ? sh.hv * sh.dv : p.out_stride;
        char* op = (FOR == NORM ? (char*)p.o32 : (char*)p.out) + OB * ((int64_t)first * o_stride + h * sh.dv + tile * 16 * NT);
        const int64_t o_step = o_stride * (OB * BLK);
        const uint32_t o_off = prow * (uint32_t)(OB * o_stride) + OB * pcol;
        uint16_t* vt = (uint16_t*)(lds + W::V_AT);
        uint16_t* ot = (uint16_t*)(lds + W::O_AT) + w * 16 * 16 * NT;
        float* of = (float*)(lds + W::O_AT) + w * 16 * W::OS;
        piece vr;
        float2 gr;
        auto ask_v = [&](int b) {  // (rows behind the sequence's last are taken from it: T is 0 there)
            b = min(b, blocks - 1);
            vr = *(const piece*)(vp + min(b * BLK + prow, rows - 1) * p.v_stride);
            gr = *(const float2*)(gp + b * g_step + 8 * lane);
        };
        auto put_v = [&]() {
#pragma unroll
            for (int i = 0; i < 2 * NT; i++) {
                const uint32_t two = ENDS && unit ? 0 : vr[i];
                vt[(pcol + 2 * i) * W::VS + prow] = (uint16_t)two;
                vt[(pcol + 2 * i + 1) * W::VS + prow] = (uint16_t)(two >> 16);
            }
            if (w == 0) ((float2*)(lds + W::G_AT))[lane] = gr;
        };
        if constexpr (!ENDS)
            for (int q = 0; q < 2 * seg; q++) __syncthreads();
        if (blocks > 0) {
            ask_v(0);
            if constexpr (!ENDS) {
                ask_q();
                ask_p();
            }
            if constexpr (NT == 2) ask_t(tr, 3 - w);
            put_v();
            ask_v(1);
            GDN_ARRIVED;
        }
        for (int b = 0; b < blocks; b++) {
            const bool more = b + 1 < blocks;  // (behind the last block the same one is asked for again)
            qp += more ? q_step : 0;
            tpp += more ? tp_step : 0;
            __syncthreads();
            if constexpr (ENDS) {  // no rows go out: v and the decays alone
                __syncthreads();
                if constexpr (NT == 2) {
                    solve(tr, 3 - w, 1);
                    GDN_FENCE;
                    ask_t(tr, 3 - w);
                }
                __syncthreads();
                GDN_FENCE;
                put_v();
                GDN_FENCE;
                ask_v(b + 2);
                continue;
            }
            bf16x8 st[KS][NT][2];
#pragma unroll
            for (int i = 0; i < KS; i++)
#pragma unroll
                for (int t = 0; t < NT; t++) x.template get<3, 2>(W::S_AT, i, t, st[i][t]);
            const gf4 eg = *(const gf4*)((const float*)(lds + W::G_AT) + 16 * w + 4 * gq);
            GDN_FENCE;
            gf4 o[NT], o2[NT];
#pragma unroll
            for (int t = 0; t < NT; t++) o[t] = o2[t] = gf4{0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < KS; i++) {
                bf16x8 a[TR];
#pragma unroll
                for (int e = 0; e < TR; e++) a[e] = __builtin_bit_cast(bf16x8, qr[i][e]);
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    o[t] = mfma_bf16(a[0], st[i][t][0], o[t]);
                    o2[t] = mfma_bf16(a[0], st[i][t][1], o2[t]);
                    if constexpr (TR == 2) o2[t] = mfma_bf16(a[1], st[i][t][0], o2[t]);
                }
            }
#pragma unroll
            for (int t = 0; t < NT; t++) o[t] = (o[t] + o2[t]) * eg;
            GDN_FENCE;
            __syncthreads();
            ask_q();
            if constexpr (NT == 2) {
                solve(tr, 3 - w, 1);
                GDN_FENCE;
                ask_t(tr, 3 - w);
            }
            __syncthreads();
            bf16x8 u[2][NT][2];
#pragma unroll
            for (int ks = 0; ks < 2; ks++)
#pragma unroll
                for (int t = 0; t < NT; t++) x.template get<2>(W::U_AT, ks, t, u[ks][t]);
            put_v();  // (the others are done with this block's)
            GDN_FENCE;
            ask_v(b + 2);
            gf4 o3[NT];
#pragma unroll
            for (int t = 0; t < NT; t++) o2[t] = o3[t] = gf4{0, 0, 0, 0};
#pragma unroll
            for (int ks = 0; ks < 2; ks++) {
                const bf16x8 a0 = fragment(pr[ks][0], ks), a1 = fragment(pr[ks][1], ks);
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    o[t] = mfma_bf16(a0, u[ks][t][0], o[t]);
                    o2[t] = mfma_bf16(a0, u[ks][t][1], o2[t]);
                    o3[t] = mfma_bf16(a1, u[ks][t][0], o3[t]);
                }
            }
#pragma unroll
            for (int t = 0; t < NT; t++) o[t] += o2[t] + o3[t];
            GDN_FENCE;
            ask_p();
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    if constexpr (FOR == NORM) of[(4 * gq + r) * W::OS + 16 * t + l16] = sh.scale * o[t][r];
                    else ot[(4 * gq + r) * 16 * NT + 16 * t + l16] = row_bits<F16>(sh.scale * o[t][r]);
                }
            wave_lds_fence();
            // (a buffer's end at the sequence's last row: stores behind it are dropped by the hardware, without a branch)
            const auto rsrc = __builtin_amdgcn_make_buffer_rsrc(op, 0, ((uint32_t)min(rows - b * BLK, BLK) - 1) * (uint32_t)(OB * o_stride) + 16 * OB * NT, 0x00027000);
            if constexpr (FOR == NORM) {
                typedef uint32_t four __attribute__((ext_vector_type(4)));
#pragma unroll
                for (int t = 0; t < NT; t++) __builtin_amdgcn_raw_buffer_store_b128(*(const four*)(of + (lane >> 2) * W::OS + pcol + 4 * t), rsrc, o_off, 16 * t, 0);
            } else {
                const piece out = *(const piece*)(ot + (lane >> 2) * 16 * NT + pcol);
                if constexpr (NT == 1) __builtin_amdgcn_raw_buffer_store_b64(out, rsrc, o_off, 0, 0);
                else __builtin_amdgcn_raw_buffer_store_b128(out, rsrc, o_off, 0, 0);
            }
            op += o_step;
        }
        return;
    }
    // ---- the state's waves
    const int64_t at = ((int64_t)hs * sh.dv + tile * 16 * NT + l16) * DK + 16 * SD * w + 4 * gq;
    const bool fresh = bt.base[s] == 0;
    gf4 S[SD][NT];
#pragma unroll
    for (int d = 0; d < SD; d++)
#pragma unroll
        for (int t = 0; t < NT; t++) {
            if constexpr (ENDS) {
                // (the last segment writes state_out while others may still have to read theirs: they read a copy)
                if (seg == 0 && !unit) *(gf4*)(p.starts + at + (int64_t)16 * t * DK + 16 * d) = *(const gf4*)(p.state_in + at + (int64_t)16 * t * DK + 16 * d);
                S[d][t] = gf4{0, 0, 0, 0};
                const int on = tile * 16 * NT - sh.dv + 16 * t + l16 - (16 * (SD * w + d) + 4 * gq);  // the row of this lane's four that is 1
                if (unit && on >= 0 && on < 4) S[d][t] = gf4{on == 0 ? 1.0f : 0.0f, on == 1 ? 1.0f : 0.0f, on == 2 ? 1.0f : 0.0f, on == 3 ? 1.0f : 0.0f};
            } else {
                S[d][t] = *(const gf4*)((whole ? p.state_in : p.starts) + at + (int64_t)16 * t * DK + 16 * d);
                if (fresh) S[d][t] = gf4{0, 0, 0, 0};
            }
        }
    const char* kp = (const char*)(p.kt + (b0 * sh.hk + hk) * (3 * KFRAGS<DK, TR> * 64) + w * KS * TR * 64);
    const char* ktp = (const char*)(p.kt + ((b0 * sh.hk + hk) * 3 + 2) * (KFRAGS<DK, TR> * 64) + SD * w * 2 * TR * 64);
    const int64_t k_step = (int64_t)sh.hk * (3 * KFRAGS<DK, TR> * 1024);
    uint4 kr[KS][TR], ktr[SD][2][TR], tr[4];
    const uint16_t* vt = (const uint16_t*)(lds + W::V_AT) + l16 * W::VS + 16 * w + 4 * gq;
    const float* gates = (const float*)(lds + W::G_AT);
    auto ask_k = [&]() {
#pragma unroll
        for (int t = 0; t < KS; t++)
#pragma unroll
            for (int e = 0; e < TR; e++) kr[t][e] = *(const uint4*)(kp + (t * TR + e) * 1024 + lane16);
    };
    auto ask_kt = [&]() {
#pragma unroll
        for (int d = 0; d < SD; d++)
#pragma unroll
            for (int ks = 0; ks < 2; ks++)
#pragma unroll
                for (int e = 0; e < TR; e++) ktr[d][ks][e] = *(const uint4*)(ktp + ((d * 2 + ks) * TR + e) * 1024 + lane16);
    };
    auto put_state = [&]() {
#pragma unroll
        for (int d = 0; d < SD; d++)
#pragma unroll
            for (int t = 0; t < NT; t++) x.template put<3>(W::S_AT, (SD * w + d) >> 1, t, 2 * ((SD * w + d) & 1) + (gq >> 1), S[d][t]);
    };
    if constexpr (!ENDS)
        for (int q = 0; q < seg; q++) {  // the segments before this one: S <- M S + c
            const float* c = ends + q * ends_step;
            const float* M = c + (int64_t)sh.dv * DK;
            put_state();
            __syncthreads();
#pragma unroll
            for (int d = 0; d < SD; d++) {
                float4 m[KS][2];
#pragma unroll
                for (int i = 0; i < KS; i++)
#pragma unroll
                    for (int e = 0; e < 2; e++) m[i][e] = *(const float4*)(M + (16 * (SD * w + d) + l16) * DK + 32 * i + 8 * gq + 4 * e);
#pragma unroll
                for (int t = 0; t < NT; t++) S[d][t] = *(const gf4*)(c + (int64_t)(tile * 16 * NT + 16 * t + l16) * DK + 16 * (SD * w + d) + 4 * gq);
#pragma unroll
                for (int i = 0; i < KS; i++) {
                    uint4 m3[3];
                    split3(m[i][0].x, m[i][0].y, m3[0].x, m3[1].x, m3[2].x);
                    split3(m[i][0].z, m[i][0].w, m3[0].y, m3[1].y, m3[2].y);
                    split3(m[i][1].x, m[i][1].y, m3[0].z, m3[1].z, m3[2].z);
                    split3(m[i][1].z, m[i][1].w, m3[0].w, m3[1].w, m3[2].w);
                    const bf16x8 a[3] = {__builtin_bit_cast(bf16x8, m3[0]), __builtin_bit_cast(bf16x8, m3[1]), __builtin_bit_cast(bf16x8, m3[2])};
#pragma unroll
                    for (int t = 0; t < NT; t++) {
                        bf16x8 st[3];
                        x.template get<3>(W::S_AT, i, t, st);
                        S[d][t] = mfma_terms<3, 3>(a, st, S[d][t]);
                    }
                }
            }
            __syncthreads();
        }
    if (blocks > 0) {
        ask_k();
        ask_t(tr, w);
        ask_kt();
        put_state();
        GDN_ARRIVED;
    }
    for (int b = 0; b < blocks; b++) {
        const bool more = b + 1 < blocks;
        kp += more ? k_step : 0;
        ktp += more ? k_step : 0;
        tpp += more ? tp_step : 0;
        __syncthreads();
        {
            uint2 v4[NT];
#pragma unroll
            for (int t = 0; t < NT; t++) v4[t] = *(const uint2*)(vt + 16 * t * W::VS);
            const gf4 eg = *(const gf4*)(gates + 16 * w + 4 * gq);
            gf4 c[NT], c2[NT];
#pragma unroll
            for (int t = 0; t < NT; t++) c[t] = c2[t] = gf4{0, 0, 0, 0};
            constexpr int PART = KS > 4 ? KS / 2 : KS;  // (k_dim 256 has no registers for all of the state's terms at once)
#pragma unroll
            for (int i0 = 0; i0 < KS; i0 += PART) {
                bf16x8 st[PART][NT][3];
#pragma unroll
                for (int i = 0; i < PART; i++)
#pragma unroll
                    for (int t = 0; t < NT; t++) x.template get<3>(W::S_AT, i0 + i, t, st[i][t]);
                GDN_FENCE;
#pragma unroll
                for (int i = 0; i < PART; i++) {
                    bf16x8 a[TR];
#pragma unroll
                    for (int e = 0; e < TR; e++) a[e] = __builtin_bit_cast(bf16x8, kr[i0 + i][e]);
#pragma unroll
                    for (int t = 0; t < NT; t++) {
                        c[t] = mfma_bf16(a[0], st[i][t][0], c[t]);
                        c2[t] = mfma_bf16(a[0], st[i][t][1], c2[t]);
                        c2[t] = mfma_bf16(a[0], st[i][t][2], c2[t]);
                        if constexpr (TR == 2) {
                            c2[t] = mfma_bf16(a[1], st[i][t][0], c2[t]);
                            c2[t] = mfma_bf16(a[1], st[i][t][1], c2[t]);
                        }
                    }
                }
            }
#pragma unroll
            for (int t = 0; t < NT; t++) {
                gf4 d;
#pragma unroll
                for (int r = 0; r < 4; r++) d[r] = fmaf(-eg[r], c[t][r] + c2[t][r], row_f32<F16>((uint16_t)((r & 2 ? v4[t].y : v4[t].x) >> (16 * (r & 1)))));
                x.put_f32(W::R_AT, t, d);
            }
        }
        __syncthreads();
        {
            const float e_end = gates[63];
            ask_k();
            GDN_FENCE;
            // (two column tiles: the second's is the other wave's of a SIMD, row tiles the other way round, so that every SIMD has as many products)
            solve(tr, w, 0);
#pragma unroll
            for (int i = 0; i < SD; i++)
#pragma unroll
                for (int t = 0; t < NT; t++) S[i][t] *= e_end;
        }
        __syncthreads();
        {
            bf16x8 d[2][NT][3];
#pragma unroll
            for (int ks = 0; ks < 2; ks++)
#pragma unroll
                for (int t = 0; t < NT; t++) x.template get<3>(W::D_AT, ks, t, d[ks][t]);
            GDN_FENCE;
            ask_t(tr, w);
            GDN_FENCE;
#pragma unroll
            for (int ks = 0; ks < 2; ks++)
#pragma unroll
                for (int i = 0; i < SD; i++) {
                    bf16x8 a[TR];
#pragma unroll
                    for (int e = 0; e < TR; e++) a[e] = __builtin_bit_cast(bf16x8, ktr[i][ks][e]);
#pragma unroll
                    for (int t = 0; t < NT; t++) S[i][t] = mfma_terms<TR, 3>(a, d[ks][t], S[i][t]);
                }
        }
        ask_kt();
        put_state();
    }
    if constexpr (ENDS) {
        float* to = p.ends + ((int64_t)(seg_at - s) * sh.hv + h) * (sh.dv + DK) * DK;
#pragma unroll
        for (int d = 0; d < SD; d++)
#pragma unroll
            for (int t = 0; t < NT; t++) {
                const int row = 16 * (SD * w + d) + 4 * gq, col = tile * 16 * NT + 16 * t + l16;
                if (!unit) {
                    *(gf4*)(to + (int64_t)col * DK + row) = S[d][t];
                } else {
#pragma unroll
                    for (int r = 0; r < 4; r++) to[(int64_t)sh.dv * DK + (row + r) * DK + col - sh.dv] = S[d][t][r];
                }
            }
    } else if (last) {
#pragma unroll
        for (int d = 0; d < SD; d++)
#pragma unroll
            for (int t = 0; t < NT; t++) *(gf4*)(p.state_out + at + (int64_t)16 * t * DK + 16 * d) = S[d][t];
    }
}
#undef GDN_FENCE
#undef GDN_ARRIVED

// ---- the gated norm ----------------------------------------------------------------------------------------------------------------------
// v_dim / 8 of GROUP neighbouring lanes hold a head's row.  Bound by memory: 8192 rows of 32 heads of 128, 268 MB, 46 us (5.8 TB/s).
template <bool F16>
__global__ __launch_bounds__(256) void k_gdn_norm(GdnShape sh, const float* o, uint16_t* out, int64_t out_stride, const uint16_t* z, int64_t z_stride, uint32_t heads, int group) {
    const uint32_t at = (blockIdx.x * 256 + threadIdx.x) / group, row = at / sh.hv, h = at - row * sh.hv;
    const int c = (threadIdx.x & (group - 1)) * 8;
    const bool in = at < heads && c < sh.dv;
    float x[8] = {}, y[8] = {}, sum = 0.0f;
    if (in) {
        const float4* from = (const float4*)(o + (int64_t)at * sh.dv + c);
        const float4 a = from[0], b = from[1];
        x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
        row8_f32<F16>(*(const uint4*)(z + (int64_t)row * z_stride + h * sh.dv + c), y);
    }
#pragma unroll
    for (int e = 0; e < 8; e++) sum = fmaf(x[e], x[e], sum);
    for (int d = 1; d < group; d <<= 1) sum += __shfl_xor(sum, d);
    if (!in) return;
    const float f = rsqrtf(sum / (float)sh.dv + sh.norm_eps);
#pragma unroll
    for (int e = 0; e < 8; e++) x[e] = x[e] * f * sh.norm[c + e] * silu_f32(y[e]);
    *(uint4*)(out + (int64_t)row * out_stride + h * sh.dv + c) = make_uint4(row_pair<F16>(x[0], x[1]), row_pair<F16>(x[2], x[3]), row_pair<F16>(x[4], x[5]), row_pair<F16>(x[6], x[7]));
}

namespace {

int64_t blocks_of(const GdnBatch& bt, int s) { return (bt.off[s + 1] - bt.off[s] + BLK - 1) / BLK; }

// How many blocks a segment has, INT32_MAX: whole sequences.  In segments a sequence's columns are walked twice and the k_dim columns of the
// unit matrix once, so that it pays where at most a quarter of the compute units would have a workgroup: 32768 rows of 8 heads of 128
// (64 column tiles) take 817 us whole, 515 in 4 segments, 465 in 8 and 515 in 16.  Sequences count by their length beside the longest: short
// ones are done early (one row beside those 32768: 457 us in 8 segments, 819 whole).  Segments of fewer than 8 blocks gain nothing over
// what putting them together takes, and since each puts together all before it, which takes as long as a block or two, there are no more
// than the square root of the blocks (262144 rows of one head of 16: 601 us in 64, 2274 in 512).
int segment_blocks(const GdnShape& sh, const GdnBatch& bt) {
    int64_t longest = 0, all = 0;
    for (int s = 0; s < bt.n_seq; s++) {
        longest = std::max(longest, blocks_of(bt, s));
        all += blocks_of(bt, s);
    }
    if (longest < 32) return INT32_MAX;
    const int64_t tiles = (2 * all + longest) / (2 * longest) * sh.hv * (sh.dv / 16);
    if (tiles > 64) return INT32_MAX;
    const int64_t segs = std::min({512 / tiles, longest / 8, (int64_t)sqrt((double)longest)});
    return (int)((longest + segs - 1) / segs);
}

struct Sizes {
    int64_t kt, tp, gates, ends, starts, o32, total;  // bytes
    int64_t blocks, segments;
    int seg_blocks;
};

Sizes workspace_of(const GdnShape& sh, const GdnBatch& bt, int dk, bool f16) {
    const int tr = f16 ? 2 : 1;
    Sizes z;
    z.blocks = z.segments = 0;
    z.seg_blocks = segment_blocks(sh, bt);
    for (int s = 0; s < bt.n_seq; s++) {
        z.blocks += blocks_of(bt, s);
        z.segments += std::max<int64_t>(1, (blocks_of(bt, s) + z.seg_blocks - 1) / z.seg_blocks);
    }
    z.kt = z.blocks * sh.hk * (3 * (dk / 8) * tr * 1024);
    z.tp = z.blocks * sh.hv * (TP_UNITS * 16);
    z.gates = z.blocks * sh.hv * 512;
    z.ends = z.seg_blocks == INT32_MAX ? 0 : (z.segments - bt.n_seq) * sh.hv * (sh.dv + dk) * dk * 4;
    z.starts = z.seg_blocks == INT32_MAX ? 0 : (int64_t)bt.n_seq * sh.hv * sh.dv * dk * 4;
    z.o32 = sh.norm ? z.blocks * BLK * sh.hv * sh.dv * 4 : 0;  // (without norm weights a layer has no gated norm)
    z.total = z.kt + z.tp + z.gates + z.ends + z.starts + z.o32;
    return z;
}

template <int DK, bool F16>
int launch_blocks(hipStream_t st, const GdnShape& sh, const GdnBatch& bt, PrefillArgs& p, int blocks) {
    const size_t lds = (size_t)blocks_operands<DK> * 16 + 2 * BLK * MS * 4 + GATE_HEADS * sizeof(BlockGates);
    static OncePerDevice once;
    const int rc = allow_lds((const void*)k_gdn_blocks<DK, F16>, lds, once);
    if (rc) return rc;
    p.split = sh.rep > 1 && (int64_t)blocks * sh.hk < 512;
    hipLaunchKernelGGL((k_gdn_blocks<DK, F16>), dim3(blocks, p.split ? sh.hv : sh.hk), dim3(256), lds, st, sh, bt, p);
    TSV_HIP(hipGetLastError());
    return TSV_OK;
}

template <int DK, bool F16, int NT, WalkFor FOR>
int launch_walk(hipStream_t st, const GdnShape& sh, const GdnBatch& bt, PrefillArgs& p) {
    const size_t lds = (size_t)Walk<DK, F16, NT>::LDS * 16;
    static OncePerDevice once;
    const int rc = allow_lds((const void*)k_gdn_walk<DK, F16, NT, FOR>, lds, once);
    if (rc) return rc;
    p.tiles = (sh.dv + (FOR == SEGMENTS ? DK : 0)) / (16 * NT);
    const int heads = p.seg_of[bt.n_seq] * sh.hk;
    hipLaunchKernelGGL((k_gdn_walk<DK, F16, NT, FOR>), dim3((heads + 7) / 8 * 8 * sh.rep * p.tiles), dim3(p.bring ? walk_threads<DK, F16, NT> : 512), lds, st, sh, bt, p);
    TSV_HIP(hipGetLastError());
    return TSV_OK;
}

template <int DK, bool F16, WalkFor FOR>
int launch_rows(hipStream_t st, const GdnShape& sh, const GdnBatch& bt, PrefillArgs& p) {
    // Two column tiles a workgroup where that still gives every compute unit one: they share what a block reads (prompts of 1 to 2049 rows, 6
    // sequences, 32 heads of 128: 157 us in all against 189); else one, for the shorter way through a block (8192 rows, 32 heads: 279 us
    // against 342).  k_dim 256 has no registers for two.
    if constexpr (DK < 256)
        if (sh.dv % 32 == 0 && (int64_t)p.seg_of[bt.n_seq] * sh.hv * (sh.dv / 32) >= 256) return launch_walk<DK, F16, 2, FOR>(st, sh, bt, p);
    return launch_walk<DK, F16, 1, FOR>(st, sh, bt, p);
}

template <int DK, bool F16>
int launch_prefill(hipStream_t st, const GdnShape& sh, const GdnBatch& bt, PrefillArgs& p, int blocks) {
    if (blocks > 0) {
        const int rc = launch_blocks<DK, F16>(st, sh, bt, p, blocks);
        if (rc) return rc;
    }
    if (p.seg_of[bt.n_seq] > bt.n_seq) {
        int rc;
        if constexpr (DK < 256) rc = sh.dv % 32 == 0 ? launch_walk<DK, F16, 2, SEGMENTS>(st, sh, bt, p) : launch_walk<DK, F16, 1, SEGMENTS>(st, sh, bt, p);
        else rc = launch_walk<DK, F16, 1, SEGMENTS>(st, sh, bt, p);
        if (rc) return rc;
    }
    return p.o32 ? launch_rows<DK, F16, NORM>(st, sh, bt, p) : launch_rows<DK, F16, ROWS>(st, sh, bt, p);
}

}  // namespace

}  // namespace tsv

using namespace tsv;

extern "C" int64_t tsv_gdn_prefill_workspace(const tsv_gdn_layer* layer, const tsv_gdn_batch* batch) {
    GdnShape sh;
    GdnBatch bt;
    if (gdn_check("gdn_prefill_workspace", nullptr, layer, batch, 0, &sh, &bt)) return -1;
    return std::max<int64_t>(16, workspace_of(sh, bt, layer->k_dim, layer->dtype == TSV_F16).total);
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
    const Sizes z = workspace_of(sh, bt, dk, f16);
    const int64_t blocks = z.blocks;
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
    p.ends = (float*)(ws + z.kt + z.tp + z.gates);
    p.starts = (float*)(ws + z.kt + z.tp + z.gates + z.ends);
    p.o32 = io->z ? (float*)(ws + z.kt + z.tp + z.gates + z.ends + z.starts) : nullptr;
    p.bring = z.kt + z.tp >= BRING_FROM;
    p.seg_blocks = z.seg_blocks;
    p.block_of[0] = p.seg_of[0] = 0;
    for (int s = 0; s < bt.n_seq; s++) {
        p.block_of[s + 1] = p.block_of[s] + (int32_t)blocks_of(bt, s);
        p.seg_of[s + 1] = p.seg_of[s] + (int32_t)std::max<int64_t>(1, (blocks_of(bt, s) + z.seg_blocks - 1) / z.seg_blocks);
    }
    const hipStream_t st = gdn_stream(stream);
    int done;
    if (dk == 64) done = f16 ? launch_prefill<64, true>(st, sh, bt, p, (int)blocks) : launch_prefill<64, false>(st, sh, bt, p, (int)blocks);
    else if (dk == 128) done = f16 ? launch_prefill<128, true>(st, sh, bt, p, (int)blocks) : launch_prefill<128, false>(st, sh, bt, p, (int)blocks);
    else done = f16 ? launch_prefill<256, true>(st, sh, bt, p, (int)blocks) : launch_prefill<256, false>(st, sh, bt, p, (int)blocks);
    if (done || !io->z || !bt.off[bt.n_seq]) return done;
    int group = 2;
    while (group * 8 < sh.dv) group *= 2;
    const int rows = bt.off[bt.n_seq], at_once = (1 << 26) / sh.hv;  // (a launch has 2^32 threads at most)
    for (int r = 0; r < rows; r += at_once) {
        const uint32_t heads = (uint32_t)std::min(at_once, rows - r) * sh.hv, wgs = (uint32_t)(((uint64_t)heads * group + 255) / 256);
        const float* o = p.o32 + (int64_t)r * sh.hv * sh.dv;
        uint16_t* out = p.out + (int64_t)r * p.out_stride;
        const uint16_t* gate = (const uint16_t*)io->z + (int64_t)r * io->z_stride;
        if (f16) hipLaunchKernelGGL((k_gdn_norm<true>), dim3(wgs), dim3(256), 0, st, sh, o, out, p.out_stride, gate, io->z_stride, heads, group);
        else hipLaunchKernelGGL((k_gdn_norm<false>), dim3(wgs), dim3(256), 0, st, sh, o, out, p.out_stride, gate, io->z_stride, heads, group);
    }
    TSV_HIP(hipGetLastError());
    return TSV_OK;
}
