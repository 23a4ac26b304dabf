// Epilogues of the 256x256 GEMM kernel (gemm_w4m.hip) for the loss of a language-model head whose logits are never kept
// (linear_ce.hip).  Four products of it run on that kernel; a wave owns 128 x 128 of a tile and sends it as eight 32 x 64 groups
// through its LDS patch (gemm_common.h), so that in a row pass eight lanes hold 8 consecutive columns each of one row:
//   LSE     z = s x W^T: per row and 128-column strip (max, sum exp(z - max)) -> part[strip][row]; the label's z -> zlab[row], all in units
//           of log 2.  Statistics in fp32 straight from the fp32 accumulators: a logit is never rounded to bf16.
//   DLOGIT  the same product again: D = exp(z - lse[row]) - [column == label], times the row's upstream gradient where rows have one of
//           their own, stored as bf16 (the operand type of the two products behind it; half a unit of 2^-8 of each entry at most).  A
//           scalar upstream gradient is NOT in D -- it multiplies the fp32 sums of those products instead, so that -1 + p keeps its bits.
//   EARLY   the product once for both, where the table's gradient is not wanted: E = exp(z - c[row]) as bf16, 0 at the label, and its fp32 sum
//           per row and 128-column strip (the label's included) -> part[strip][row]; the label's z -> zlab[row].  c, the label's logit from a
//           dot product of its own, is never above the log-sum-exp, and E overflows only where a row's loss is above 80 (linear_ce.hip)
//   DX      dx_acc (fp32) = beta dx_acc + D W over the pieces of the vocabulary; with few tiles (few rows) the piece is split along the
//           vocabulary into of_ce_splits parts, each with a dx_acc of its own
//   DW      dW (bf16) = scale D^T x
// Rows are the compacted ones (labels that count), padded to 256; the vocabulary's last tile hangs over the table's end: its rows
// read as zeros (of_buf_make_n), its columns are masked here.
#pragma once
#include "gemm_tile256.h"

enum { OF_EPI_CE_LSE = 16, OF_EPI_CE_DLOGIT = 17, OF_EPI_CE_DX = 18, OF_EPI_CE_DW = 19, OF_EPI_CE_EARLY = 20 };      // internal: of_gemm refuses them
OF_HOSTDEV constexpr bool of_epi_is_ce(int epi) { return epi >= OF_EPI_CE_LSE; }

struct OfCeGemmArgs : OfGemmArgs {      // M, N, K: the padded extents of the launch (of_gemm's layout rules)
    const int* count;        // device: rows with a label that counts; live rows = count rounded up to 256, at least 256 (M, or K of DW)
    long b_bytes;            // bytes of the B matrix from args.B to the end of its last row
    int n_valid;             // columns that exist (LSE, DLOGIT: vocabulary of the piece; DX, DW: d)
    int m_valid;             // DW: rows that exist (vocabulary of the piece)
    int col0;                // vocabulary index of column 0 of the piece (labels count from the table's first row; EARLY's strips too)
    const int* lab;          // [row] label, -1 for rows behind `count`
    const int* gate;         // device flag or NULL: nothing is done where it is 0
    const float* lse;        // [row] in units of log 2, +inf for rows behind `count` (EARLY: c)
    const float* grow;       // [row] upstream gradient of its own, or NULL
    float* part;             // LSE: [strip][row][2]; EARLY: [strip][row]
    float* zlab;             // LSE, EARLY: [row]
    long part_ld;            // rows of one strip
    const float* gscale;     // DW: scalar upstream gradient or NULL (1)
    int by_count;            // DW: divide by `count`
    int split_stages;        // DX: 64-deep stages of a whole piece (the same for every piece: of_ce_splits)
};
int of_gemm_w4m_ce(const OfCeGemmArgs& a, of_stream_t s);      // gemm_w4m.hip: a.epi selects the product

template <int EPI>
struct OfEpiArgs { typedef OfGemmArgs type; };
template <> struct OfEpiArgs<OF_EPI_CE_LSE> { typedef OfCeGemmArgs type; };
template <> struct OfEpiArgs<OF_EPI_CE_DLOGIT> { typedef OfCeGemmArgs type; };
template <> struct OfEpiArgs<OF_EPI_CE_EARLY> { typedef OfCeGemmArgs type; };
template <> struct OfEpiArgs<OF_EPI_CE_DX> { typedef OfCeGemmArgs type; };
template <> struct OfEpiArgs<OF_EPI_CE_DW> { typedef OfCeGemmArgs type; };

// rows a launch works on: at least one tile, so that every product, sum and gradient of a batch without a single label is written (as zeros)
OF_HOSTDEV int of_ce_live_rows(int count) { return count > 0 ? (count + 255) & ~255 : 256; }
// Parts a dx product is split into along the vocabulary, so that few rows fill the chip too: 1024 rows x d = 2560 are 40 tiles on 256
// CUs, 443 us a piece of 32768; as 6 parts 151 us.  A part keeps at least 4 stages of 64.
constexpr int CE_PART_STAGES = 4;
OF_HOSTDEV int of_ce_splits(int tiles, int stages) {
    int s = OF_NUM_CUS / tiles;
    const int most = stages / CE_PART_STAGES;
    if (s > most) s = most;
    return s < 1 ? 1 : s;
}
// the scalar that multiplies both gradients: upstream / number of labels (mean), upstream (sum), 1 (rows have their own)
OF_DEV float of_ce_scale(const float* gscale, int by_count, const int* count) {
    if (by_count && *count == 0) return 0.f;
    const float g = gscale ? *gscale : 1.0f;
    return by_count ? g / (float)*count : g;
}

namespace oft {

constexpr float CE_LOG2E = 1.4426950408889634f;
constexpr float CE_LN2 = 0.69314718055994531f;
constexpr float CE_LOWEST = -3.0e38f;      // the running maximum of nothing: below every finite logit, and no NaN in differences

// LSE straight from the accumulators: lane l of a 16 x 16 fragment holds row l & 15, columns 4 (l >> 4) + 0..3, so that a lane owns 32 of
// a row's 128 columns in the eight fragments of a row block and the four lanes of a row meet in two register exchanges -- no LDS patch
// (through it a tile's epilogue took 5 us more of one wave's issue slots).  frag(b) = the row block's fragment of columns 16 b..
template <class Frag>
OF_DEV void ce_lse_rows(const OfCeGemmArgs& p, Frag frag, int m_base, int n_base, int lane) {
    const int m = m_base + (lane & 15), n0 = n_base + 4 * (lane >> 4);
    const bool edge = n_base + 128 > p.n_valid;
    const int at = p.lab[m] - p.col0 - n0;            // the label's place counted from this lane's first column
    const float sc = p.alpha * CE_LOG2E;              // base-2 logits: exp(z - max) is one subtraction and one v_exp_f32
    float top = CE_LOWEST;
    f32x4 z[8];
#pragma unroll
    for (int b = 0; b < 8; ++b) {
        z[b] = frag(b);
#pragma unroll
        for (int e = 0; e < 4; ++e) z[b][e] *= sc;         // (rounded here: DLOGIT rounds the same product)
        if (edge) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (n0 + 16 * b + e >= p.n_valid) z[b][e] = -__builtin_inff();
        }
        top = of_max(of_max(top, of_max(z[b][0], z[b][1])), of_max(z[b][2], z[b][3]));
    }
    top = of_rows_max(top);
    float s = 0.f;
#pragma unroll
    for (int b = 0; b < 8; ++b) s += (of_exp2(z[b][0] - top) + of_exp2(z[b][1] - top)) + (of_exp2(z[b][2] - top) + of_exp2(z[b][3] - top));
    s = of_rows_sum(s);
    if (at >= 0 && at < 116 && (at & 15) < 4) {       // one lane of the row, in one strip
#pragma unroll
        for (int b = 0; b < 8; ++b)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (at == 16 * b + e) p.zlab[m] = z[b][e];
    }
    if (lane < 16) *(f32x2*)(p.part + ((size_t)(n_base >> 7) * p.part_ld + m) * 2) = f32x2{top, s};
}

// the row passes of one 32 x 64 group (accumulators in the patch)
template <int EPI>
OF_DEV void ce_group_rows(const OfCeGemmArgs& p, char* patch, int m_base, int n_base, int lane, float sc, float (&sum)[4]) {
    constexpr bool SPLIT = EPI == OF_EPI_CE_DX;          // fp32 output: columns 4j.. and 32 + 4j.. (gemm_common.h, epi_split_cols)
    const int hi = SPLIT ? 32 : 4;
    const int rd_row = lane >> 3, rd_col = (lane & 7) * (SPLIT ? 4 : 8);
    of_wave_sync();
#pragma unroll
    for (int it = 0; it < 4; ++it) {
        const int r = it * 8 + rd_row, m = m_base + r, n = n_base + rd_col;
        const f32x4 v0 = *(const f32x4*)(patch + r * ofg::PATCH_PITCH + rd_col * 4), v1 = *(const f32x4*)(patch + r * ofg::PATCH_PITCH + (rd_col + hi) * 4);
        float a[8] = {v0[0], v0[1], v0[2], v0[3], v1[0], v1[1], v1[2], v1[3]};
        if constexpr (EPI == OF_EPI_CE_EARLY) {
            const int at = p.lab[m] - p.col0 - n;
            const float c = p.lse[m];
            float o[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e] = of_exp2(__builtin_fmaf(a[e], sc, -c));
            if (n_base + 64 > p.n_valid) {
#pragma unroll
                for (int e = 0; e < 8; ++e) o[e] = n + e < p.n_valid ? o[e] : 0.f;
            }
            sum[it] += ((o[0] + o[1]) + (o[2] + o[3])) + ((o[4] + o[5]) + (o[6] + o[7]));
            if ((unsigned)at < 8u) {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (e == at) {
                        p.zlab[m] = a[e] * sc;
                        o[e] = 0.f;
                    }
            }
            *(u32x4*)((bf16_t*)p.C + (size_t)m * p.ldc + n) = ofg::pack8(o);
        } else if constexpr (EPI == OF_EPI_CE_DLOGIT) {
            // what few elements need (the label's, columns behind the vocabulary) sits in branches
            const int at = p.lab[m] - p.col0 - n;         // the label's place among this lane's eight columns, if 0 <= at < 8
            const float l = p.lse[m];
            float o[8];
            {
                // the logit as LSE rounded it, then the difference: the same two roundings, so that a row with one class left has p = 1
                // exactly and no gradient (a fused multiply-add would leave the rounding of lse's own logit in p)
#pragma clang fp contract(off)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float z = a[e] * sc;
                    o[e] = of_exp2(z - l);
                }
            }
            if ((unsigned)at < 8u) {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (e == at) o[e] -= 1.0f;
            }
            if (p.grow) {
                const float g = p.grow[m];
#pragma unroll
                for (int e = 0; e < 8; ++e) o[e] *= g;
            }
            if (n_base + 64 > p.n_valid) {
#pragma unroll
                for (int e = 0; e < 8; ++e) o[e] = n + e < p.n_valid ? o[e] : 0.f;
            }
            *(u32x4*)((bf16_t*)p.C + (size_t)m * p.ldc + n) = ofg::pack8(o);
        } else if constexpr (EPI == OF_EPI_CE_DX) {
            float* c = (float*)p.C + (size_t)m * p.ldc + n;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if (n + h * 32 >= p.n_valid) continue;
                f32x4 o = {a[4 * h], a[4 * h + 1], a[4 * h + 2], a[4 * h + 3]};
                if (p.beta != 0.f) {
                    const f32x4 old = *(const f32x4*)(c + h * 32);
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[e] += old[e];
                }
                *(f32x4*)(c + h * 32) = o;
            }
        } else {
            if (m < p.m_valid && n < p.n_valid) {
                float o[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) o[e] = sc * a[e];
                *(u32x4*)((bf16_t*)p.C + (size_t)m * p.ldc + n) = ofg::pack8(o);
            }
        }
        of_sched_fence();
    }
    of_wave_sync();
}

template <int EPI, class ToPatch>
OF_DEV void w4_epilogue_ce(const OfCeGemmArgs& p, ToPatch to_patch, char* smem, int m0, int n0, int wm, int wn, int wave, int lane) {
    char* patch = smem + wave * ofg::PATCH_BYTES;
    float sc = p.alpha;
    if (EPI == OF_EPI_CE_DLOGIT || EPI == OF_EPI_CE_EARLY) sc *= CE_LOG2E;
    if (EPI == OF_EPI_CE_DW) sc *= of_ce_scale(p.gscale, p.by_count, p.count);
    float sum[4];
#pragma unroll
    for (int g = 0; g < 8; ++g) {
        if (!(g & 1)) sum[0] = sum[1] = sum[2] = sum[3] = 0.f;
        to_patch(g, patch);
        ce_group_rows<EPI>(p, patch, m0 + wm * 128 + (g >> 1) * 32, n0 + wn * 128 + (g & 1) * 64, lane, sc, sum);
        if constexpr (EPI == OF_EPI_CE_EARLY) {
            if (g & 1) {          // the strip's 128 columns of a row sit in eight lanes
#pragma unroll
                for (int it = 0; it < 4; ++it) {
                    float s = sum[it];
#pragma unroll
                    for (int o = 4; o >= 1; o >>= 1) s += of_shfl_xor(s, o);
                    const int m = m0 + wm * 128 + (g >> 1) * 32 + it * 8 + (lane >> 3);
                    if ((lane & 7) == 0) p.part[((size_t)((p.col0 + n0) >> 7) + wn) * p.part_ld + m] = s;
                }
            }
        }
    }
}

}  // namespace oft
