// Softmax cross entropy of a language-model head whose logits are never kept (gfx950):  z = s x W^T over a vocabulary of ~50 000,
// loss_r = log sum_v exp z_rv - z_r,label, and its gradients dx = s g D W, dW = s g D^T x with D = softmax(z) - onehot(label).
//
// Materialised (loss.hip behind a vendor GEMM) the logits of 8192 rows are 826 MB in bf16, written once and read twice, and rounded
// to 8 bits of mantissa in front of the exponential.  Here:
//   forward   rows whose label counts are gathered (an ignored row costs nothing behind this point), then ONE product whose epilogue
//             keeps (max, sum exp) per row and 128 columns, from fp32 accumulators; a small launch joins the ~400 strips of a row;
//   backward  the vocabulary in pieces: the product again -> D of the piece (bf16; 128 MB, so that it stays in the 256-MB Infinity Cache
//             between the three products that touch it; never under 256 table rows, i.e. 512 bytes a row of the batch: 512 MB at 2^20
//             rows) -> dx += D W_piece in fp32, dW_piece = D^T x.
//   frozen table   without dW the forward forms dx as well and the backward has no product left (two instead of three): E = exp(z - c) with
//             c = the label's logit needs no maximum, dx = s g (exp(c - lse) E W + (p_label - 1) w_label).  lse - c is the row's loss; only a
//             loss above 80 (in units of log 2) could overflow, and then a flag on the device lets the forms above run behind it.
// All products run on the 256x256 MFMA kernel (gemm_w4m.hip) with the epilogues of gemm_ce_epi.h: they are bound by its K loop, i.e. by
// the chip's power budget, 2 R V d operations forward and 6 R V d backward (a third of them the second logits product).
// Measured (8192 rows, 7361 count, d = 2048, vocabulary 50435; kernel times and calls of one profiled run): loss and both gradients 4.97 ms =
// four products of 1.52 TFLOP at 1235 TFLOP/s (1.10 ms statistics, 1.31 logits again, 1.34 dx, 1.18 dW; a library product of that shape reaches
// 1282) and 60 us in the small launches; d = 4096, 9 of 10 and more count: 9.88 ms, 1310 TFLOP/s.  Frozen table, 1999 rows (1013 count), d = 2560:
// 0.56 ms (0.26 EARLY, 0.26 dx); 1032 that count are a fifth tile of rows: 0.66.  One row: 47 us, 207 MB at 4.8 TB/s.
// No atomics; every sum has a fixed order.
#include "gemm_ce_epi.h"

namespace {

constexpr float CE_FAR = 80.f;             // E <= 2^80: finite in bf16, and in fp32 sums of it
constexpr int CE_THREADS = 512;          // of the launches that are one workgroup

struct CeRowsArgs {
    const long long* labels; long long ignore_index;
    long rows; int vocab;
    int* count; int* slot_of; int* row_of; int* lab;
    float* lse; float* loss_rows;
    const bf16_t* x; long ldx; bf16_t* xc; long ldxc; int d, d_pad;
    const float* part; const float* zlab; long part_ld; int strips;
    float* loss; int mean;
    const float* grad; int by_count; float logit_scale; const float* acc; int split_stages; bf16_t* dx; long lddx;
    float* grow;
    const int* gate;                           // device flag or NULL: nothing is done where it is 0
    float* ref; int* far; float sc2;           // EARLY: c by place, "some loss is above CE_FAR", logit_scale * log2 e
    const bf16_t* w; long ldw; bf16_t* wc; long ldwc; long w_rows;
};

// EARLY's c: the label's logit in units of log 2, a dot product by the wave that gathers the row
OF_DEV void ce_reference(const CeRowsArgs& a, const bf16_t* x, int lab, long i, int lane) {
    const bf16_t* w = a.w + (size_t)lab * a.ldw;
    float s = 0.f;
    for (int c = lane * 8; c < a.d; c += 512) {
        const u32x4 u = *(const u32x4*)(x + c), v = *(const u32x4*)(w + c);
#pragma unroll
        for (int e = 0; e < 4; ++e) s = of_dot2_bf16(u[e], v[e], s);
    }
    s = of_wave_sum(s);
    if (lane == 0) a.ref[i] = s * a.sc2;
}

// One workgroup: the rows whose label counts, in order.  slot_of[row] = place among them or -1, row_of its inverse, lab by place;
// loss_rows of the others is final here: 0 for ignored rows, NaN for a label outside the vocabulary (a caller's mistake that has to
// surface in the loss; such a row has no gradient).  A wave owns consecutive 64s of rows: it counts them with one ballot each, the waves'
// counts are joined, and a second walk over the (cached) labels places them.
OF_GLOBAL void OF_BOUNDS(CE_THREADS, 1) ce_index_kernel(CeRowsArgs a) {
    int* cum = (int*)of_smem();
    constexpr int WAVES = CE_THREADS / 64;
    const int tid = of_tid(), lane = tid & 63, wave = tid >> 6;
    const long per = ((a.rows + WAVES * 64 - 1) / (WAVES * 64)) * 64, lo = wave * per, hi = lo + per < a.rows ? lo + per : a.rows;
    auto counts = [&](long r) OF_INLINE_LAMBDA -> bool {
        if (r >= hi) return false;
        const long long l = a.labels[r];
        return l != a.ignore_index && l >= 0 && l < a.vocab;
    };
    int n = 0;
    for (long r0 = lo; r0 < lo + per; r0 += 256) {
        bool c[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) c[u] = counts(r0 + u * 64 + lane);
#pragma unroll
        for (int u = 0; u < 4; ++u) n += __builtin_popcountll(of_ballot(c[u]));
    }
    if (lane == 0) cum[wave] = n;
    of_sync();
    int at = 0, total = 0;
    for (int w = 0; w < WAVES; ++w) {
        if (w < wave) at += cum[w];
        total += cum[w];
    }
    for (long r0 = lo; r0 < lo + per; r0 += 256) {
        long long l[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) l[u] = r0 + u * 64 + lane < hi ? a.labels[r0 + u * 64 + lane] : a.ignore_index;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const long r = r0 + u * 64 + lane;
            const bool c = r < hi && l[u] != a.ignore_index && l[u] >= 0 && l[u] < a.vocab;
            const unsigned long long all = of_ballot(c);
            const int slot = at + __builtin_popcountll(all & ((1ull << lane) - 1));
            at += __builtin_popcountll(all);
            if (r >= hi) continue;
            a.slot_of[r] = c ? slot : -1;
            if (c) {
                a.row_of[slot] = (int)r;
                a.lab[slot] = (int)l[u];
            } else {
                a.loss_rows[r] = l[u] == a.ignore_index ? 0.f : __builtin_nanf("");
            }
        }
    }
    if (tid == 0) {
        *a.count = total;
        if (a.far) *a.far = 0;
    }
    for (int i = total + tid; i < of_ce_live_rows(total); i += CE_THREADS) a.lab[i] = -1;
}

// xc[place] = x[row_of[place]], zeros in the columns behind d and in the rows behind `count` up to the next 256: the products then
// need no row or depth edges.  One wave per row.
OF_GLOBAL void OF_BOUNDS(256, 4) ce_gather_kernel(CeRowsArgs a) {
    const int lane = of_tid() & 63, count = *a.count;
    const long i = (long)of_bid_x() * 4 + (of_tid() >> 6);
    if (i >= of_ce_live_rows(count)) return;
    const bf16_t* src = i < count ? a.x + (size_t)a.row_of[i] * a.ldx : nullptr;
    if (a.ref) {
        if (src) ce_reference(a, src, a.lab[i], i, lane);
        else if (lane == 0) a.ref[i] = 0.f;
    }
    bf16_t* dst = a.xc + (size_t)i * a.ldxc;
    for (int c = lane * 8; c < a.d_pad; c += 512) {
        u32x4 v = {0u, 0u, 0u, 0u};
        if (src && c < a.d) v = *(const u32x4*)(src + c);
        *(u32x4*)(dst + c) = v;
    }
}

// Both of the above in one launch for at most 1024 rows: every wave finds its place's row by counting the labels itself (16 ballots), the
// first workgroup also writes the lists.
constexpr int CE_FEW_ROWS = 1024;
OF_GLOBAL void OF_BOUNDS(256, 4) ce_index_gather_kernel(CeRowsArgs a) {
    const int lane = of_tid() & 63, wave = of_tid() >> 6, rows = (int)a.rows;
    const int i = of_bid_x() * 4 + wave;
    int at = 0, mine = -1;
    for (int r0 = 0; r0 < rows; r0 += 256) {
        long long l[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) l[u] = r0 + u * 64 + lane < rows ? a.labels[r0 + u * 64 + lane] : a.ignore_index;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int r = r0 + u * 64 + lane;
            const bool c = l[u] != a.ignore_index && l[u] >= 0 && l[u] < a.vocab;
            const unsigned long long all = of_ballot(c);
            const int slot = at + __builtin_popcountll(all & ((1ull << lane) - 1));
            const unsigned long long hit = of_ballot(c && slot == i);
            if (hit) mine = r0 + u * 64 + __builtin_ctzll(hit);
            at += __builtin_popcountll(all);
            if (of_bid_x() == 0 && wave == 0 && r < rows) {
                a.slot_of[r] = c ? slot : -1;
                if (c) {
                    a.row_of[slot] = r;
                    a.lab[slot] = (int)l[u];
                } else {
                    a.loss_rows[r] = l[u] == a.ignore_index ? 0.f : __builtin_nanf("");
                }
            }
        }
    }
    const int live = of_ce_live_rows(at);
    if (of_bid_x() == 0 && wave == 0) {
        if (lane == 0) {
            *a.count = at;
            if (a.far) *a.far = 0;
        }
        for (int k = at + lane; k < live; k += 64) a.lab[k] = -1;
    }
    if (i >= live) return;
    const bf16_t* src = mine >= 0 ? a.x + (size_t)mine * a.ldx : nullptr;
    if (a.ref) {
        if (src) ce_reference(a, src, (int)a.labels[mine], i, lane);
        else if (lane == 0) a.ref[i] = 0.f;
    }
    bf16_t* dst = a.xc + (size_t)i * a.ldxc;
    for (int c = lane * 8; c < a.d_pad; c += 512) {
        u32x4 v = {0u, 0u, 0u, 0u};
        if (src && c < a.d) v = *(const u32x4*)(src + c);
        *(u32x4*)(dst + c) = v;
    }
}

// the table with its rows padded to a multiple of 64 columns by zeros (only where d is none)
OF_GLOBAL void OF_BOUNDS(256, 4) ce_pad_table_kernel(CeRowsArgs a) {
    const int lane = of_tid() & 63;
    for (long i = (long)of_bid_x() * 4 + (of_tid() >> 6); i < a.w_rows; i += (long)of_gdim_x() * 4)
        for (int c = lane * 8; c < a.d_pad; c += 512) {
            u32x4 v = {0u, 0u, 0u, 0u};
            if (c < a.d) v = *(const u32x4*)(a.w + (size_t)i * a.ldw + c);
            *(u32x4*)(a.wc + (size_t)i * a.ldwc + c) = v;
        }
}

// 16 rows a workgroup, 16 lanes a row: lane j joins strips j, j + 16, ... of its row, then the 16 lanes in a fixed order (base-2 logits)
OF_GLOBAL void OF_BOUNDS(256, 2) ce_finish_kernel(CeRowsArgs a) {
    float* red = (float*)of_smem();          // [16 groups][16 rows][2]
    const int tid = of_tid(), r = tid & 15, j = tid >> 4, count = *a.count;
    if (a.gate && *a.gate == 0) return;
    const long i0 = (long)of_bid_x() * 16;
    if (i0 >= of_ce_live_rows(count)) return;
    const long i = i0 + r;
    float m = oft::CE_LOWEST, s = 0.f;
    if (a.ref) {
#pragma unroll 4
        for (int t = j; t < a.strips; t += 16) s += a.part[(size_t)t * a.part_ld + i];
        m = a.ref[i];
    } else
#pragma unroll 4
    for (int t = j; t < a.strips; t += 16) {
        const f32x2 q = *(const f32x2*)(a.part + ((size_t)t * a.part_ld + i) * 2);
        const float top = of_max(m, q[0]);
        s = s * of_exp2(m - top) + q[1] * of_exp2(q[0] - top);
        m = top;
    }
    red[(j * 16 + r) * 2] = m;
    red[(j * 16 + r) * 2 + 1] = s;
    of_sync();
    if (j == 0) {
        float top = red[r * 2];
        for (int k = 1; k < 16; ++k) top = of_max(top, red[(k * 16 + r) * 2]);
        float sum = 0.f;
        for (int k = 0; k < 16; ++k) sum += red[(k * 16 + r) * 2 + 1] * of_exp2(red[(k * 16 + r) * 2] - top);
        const float lse = top + of_log2(sum);
        a.lse[i] = i < count ? lse : __builtin_inff();          // behind `count`: exp(z - inf) = 0, rows of D that are zero
        if (i < count) {
            a.loss_rows[a.row_of[i]] = (lse - a.zlab[i]) * oft::CE_LN2;
            if (a.far && lse - a.ref[i] > CE_FAR) *a.far = 1;
        }
    }
}

// one workgroup: the sum of the rows' losses, divided by the number of labels for a mean (0 / 0 = NaN without any, as torch has it)
OF_GLOBAL void OF_BOUNDS(CE_THREADS, 1) ce_reduce_kernel(CeRowsArgs a) {
    float* red = (float*)of_smem();
    const int tid = of_tid();
    float s = 0.f;
    for (long r = tid; r < a.rows; r += CE_THREADS) s += a.loss_rows[r];
    red[tid] = s;
    of_sync();
    for (int o = CE_THREADS / 2; o >= 1; o >>= 1) {
        if (tid < o) red[tid] += red[tid + o];
        of_sync();
    }
    if (tid == 0) *a.loss = a.mean ? red[0] / (float)*a.count : red[0];
}

// both of the above in one workgroup where there is little to join
constexpr int CE_FEW_PARTS = 1 << 14;
OF_GLOBAL void OF_BOUNDS(CE_THREADS, 1) ce_finish_reduce_kernel(CeRowsArgs a) {
    float* red = (float*)of_smem();
    const int tid = of_tid(), count = *a.count, live = of_ce_live_rows(count);
    float sum = 0.f;
    for (int i = tid; i < live; i += CE_THREADS) {
        float m = oft::CE_LOWEST, s = 0.f;
#pragma unroll 4
        for (int t = 0; t < a.strips; ++t) {
            const f32x2 q = *(const f32x2*)(a.part + ((size_t)t * a.part_ld + i) * 2);
            const float top = of_max(m, q[0]);
            s = s * of_exp2(m - top) + q[1] * of_exp2(q[0] - top);
            m = top;
        }
        const float lse = m + of_log2(s);
        a.lse[i] = i < count ? lse : __builtin_inff();
        if (i < count) {
            const float l = (lse - a.zlab[i]) * oft::CE_LN2;
            a.loss_rows[a.row_of[i]] = l;
            sum += l;
        }
    }
    if (!a.loss) return;
    for (long r = tid; r < a.rows; r += CE_THREADS)
        if (a.slot_of[r] < 0) sum += a.loss_rows[r];          // zeros, and the NaN of a label outside the vocabulary
    red[tid] = sum;
    of_sync();
    for (int o = CE_THREADS / 2; o >= 1; o >>= 1) {
        if (tid < o) red[tid] += red[tid + o];
        of_sync();
    }
    if (tid == 0) *a.loss = a.mean ? red[0] / (float)count : red[0];
}

// ------------------------------------------------------------------------------------------------ a handful of rows, no gradient
// Scoring the next token of up to 16 sequences: the table is read once and nothing else counts (206 MB at 50435 x 2048: 40 us at the
// rate of a large copy), while a 256-row MFMA tile would be 1/16 ... 1/256 full.  A wave takes four table rows at a time, 16 bytes a lane and
// row, against the rows of x in LDS (v_dot2, fp32); a halving butterfly leaves every (row, table row) product in a lane of its own, which
// keeps that pair's running maximum and sum.
constexpr int FEW_WAVES = 4, FEW_R = 4, FEW_WG = 512;
struct CeFewArgs {
    const bf16_t* x; long ldx; const bf16_t* w; long ldw; const long long* labels; long long ignore_index;
    int rows, vocab, d; float scale;          // scale: logit_scale * log2 e
    float* part; float* zlab; float* loss_rows; float* loss; int mean;
};
template <int MT>
OF_GLOBAL void OF_BOUNDS(FEW_WAVES * 64, 2) ce_few_kernel(CeFewArgs a) {
    constexpr int V = MT * FEW_R;
    const int tid = of_tid(), lane = tid & 63, wave = tid >> 6;
    bf16_t* xs = (bf16_t*)of_smem();                                   // [MT][d]
    float* red = (float*)(of_smem() + (((size_t)MT * a.d * 2 + 15) & ~(size_t)15));      // [FEW_WAVES][V][2]
    for (int i = tid * 8; i < MT * a.d; i += FEW_WAVES * 64 * 8) {
        const int m = i / a.d, k = i - m * a.d;
        *(u32x4*)(xs + i) = m < a.rows ? *(const u32x4*)(a.x + (size_t)m * a.ldx + k) : u32x4{0u, 0u, 0u, 0u};
    }
    of_sync();
    // the pair this lane ends up with (the same every time) and its label
    int pair = 0;
    {
        int live = V;
#pragma unroll
        for (int s = 0; s < 6; ++s)
            if (live > 1) {
                live >>= 1;
                pair += ((lane >> s) & 1) * live;
            }
    }
    const int m = pair / FEW_R;
    const long long lab = m < a.rows ? a.labels[m] : -1;
    float top = oft::CE_LOWEST, sum = 0.f;
    const int groups = (a.vocab + FEW_R - 1) / FEW_R;
    for (int g = of_bid_x() * FEW_WAVES + wave; g < groups; g += FEW_WG * FEW_WAVES) {
        const int n0 = g * FEW_R;
        float acc[V];
#pragma unroll
        for (int i = 0; i < V; ++i) acc[i] = 0.f;
#pragma unroll 4
        for (int k = lane * 8; k < a.d; k += 512) {
            u32x4 w[FEW_R];
#pragma unroll
            for (int r = 0; r < FEW_R; ++r) {
                const int n = n0 + r < a.vocab ? n0 + r : a.vocab - 1;          // (computed and dropped)
                w[r] = *(const u32x4*)(a.w + (size_t)n * a.ldw + k);
            }
#pragma unroll
            for (int mm = 0; mm < MT; ++mm) {
                const u32x4 x = *(const u32x4*)(xs + mm * a.d + k);
#pragma unroll
                for (int r = 0; r < FEW_R; ++r)
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[mm * FEW_R + r] = of_dot2_bf16(x[e], w[r][e], acc[mm * FEW_R + r]);
            }
        }
        int live = V;
#pragma unroll
        for (int s = 0; s < 6; ++s) {
            const int bit = (lane >> s) & 1;
            if (live > 1) {
                live >>= 1;
#pragma unroll
                for (int i = 0; i < V / 2; ++i)
                    if (i < live) {
                        const float lo = acc[i], hi = acc[i + live];
                        acc[i] = (bit ? hi : lo) + of_shfl_xor(bit ? lo : hi, 1 << s);
                    }
            } else {
                acc[0] += of_shfl_xor(acc[0], 1 << s);
            }
        }
        const int n = n0 + pair % FEW_R;
        if (n < a.vocab) {
            const float z = acc[0] * a.scale, t = of_max(top, z);
            sum = sum * of_exp2(top - t) + of_exp2(z - t);
            top = t;
            if (n == lab) a.zlab[m] = z;
        }
    }
    if (lane < V) {
        red[(wave * V + pair) * 2] = top;
        red[(wave * V + pair) * 2 + 1] = sum;
    }
    of_sync();
    if (tid < a.rows) {
        float t = oft::CE_LOWEST, s = 0.f;
        for (int i = 0; i < FEW_WAVES * FEW_R; ++i) {
            const float* q = red + ((i / FEW_R) * V + tid * FEW_R + i % FEW_R) * 2;
            const float u = of_max(t, q[0]);
            s = s * of_exp2(t - u) + q[1] * of_exp2(q[0] - u);
            t = u;
        }
        *(f32x2*)(a.part + ((size_t)tid * FEW_WG + of_bid_x()) * 2) = f32x2{t, s};
    }
}
// one workgroup, a wave at a time per row: the 512 partial results of a row, its loss, and their sum
OF_GLOBAL void OF_BOUNDS(256, 1) ce_few_finish_kernel(CeFewArgs a) {
    float* red = (float*)of_smem();
    const int tid = of_tid(), lane = tid & 63, wave = tid >> 6;
    for (int m = wave; m < a.rows; m += 4) {
        f32x2 q[FEW_WG / 64];
#pragma unroll
        for (int u = 0; u < FEW_WG / 64; ++u) q[u] = *(const f32x2*)(a.part + ((size_t)m * FEW_WG + u * 64 + lane) * 2);
        float top = oft::CE_LOWEST;
#pragma unroll
        for (int u = 0; u < FEW_WG / 64; ++u) top = of_max(top, q[u][0]);
        top = of_wave_max(top);
        float s = 0.f;
#pragma unroll
        for (int u = 0; u < FEW_WG / 64; ++u) s += q[u][1] * of_exp2(q[u][0] - top);
        s = of_wave_sum(s);
        if (lane == 0) {
            const long long l = a.labels[m];
            const float lse = top + of_log2(s);
            const float loss = l == a.ignore_index ? 0.f : l >= 0 && l < a.vocab ? (lse - a.zlab[m]) * oft::CE_LN2 : __builtin_nanf("");
            a.loss_rows[m] = loss;
            red[m] = loss;
        }
    }
    of_sync();
    if (tid == 0 && a.loss) {
        float sum = 0.f;
        int n = 0;
        for (int m = 0; m < a.rows; ++m) {
            sum += red[m];
            n += a.labels[m] != a.ignore_index;
        }
        *a.loss = a.mean ? sum / (float)n : sum;
    }
}

// upstream gradients of the rows, by place
OF_GLOBAL void OF_BOUNDS(256, 4) ce_row_grads_kernel(CeRowsArgs a) {
    const long i = (long)of_bid_x() * 256 + of_tid();
    const int count = *a.count;
    if (i < of_ce_live_rows(count)) a.grow[i] = i < count ? a.grad[a.row_of[i]] : 0.f;
}

// dx[row] = bf16(logit_scale * scale * the sum of acc's parts), zeros for rows without a label; one wave per row.  EARLY: acc is E W, and
// the row's own factor and the label's part join here, in fp32.
OF_GLOBAL void OF_BOUNDS(256, 4) ce_scatter_kernel(CeRowsArgs a) {
    const int lane = of_tid() & 63;
    const long r = (long)of_bid_x() * 4 + (of_tid() >> 6);
    if (r >= a.rows) return;
    const int i = a.slot_of[r], live = of_ce_live_rows(*a.count);
    const int parts = of_ce_splits((live >> 8) * ((a.d + 255) >> 8), a.split_stages);
    const size_t part = (size_t)live * a.d;
    float sc = a.logit_scale * (a.grow ? a.grow[r] : of_ce_scale(a.grad, a.by_count, a.count));
    float own = 0.f;
    const bf16_t* w = a.w;
    if (a.far && i >= 0 && *a.far == 0) {
        const float lse = a.lse[i];
        own = sc * (of_exp2(a.zlab[i] - lse) - 1.0f);
        sc *= of_exp2(a.ref[i] - lse);
        w += (size_t)a.lab[i] * a.ldw;
    } else {
        w = nullptr;
    }
    const float* src = i < 0 ? nullptr : a.acc + (size_t)i * a.d;
    bf16_t* dst = a.dx + (size_t)r * a.lddx;
    for (int c = lane * 8; c < a.d; c += 512) {
        float o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (src) {
            for (int k = 0; k < parts; ++k) {
                const f32x4 v0 = *(const f32x4*)(src + k * part + c), v1 = *(const f32x4*)(src + k * part + c + 4);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    o[e] += v0[e];
                    o[4 + e] += v1[e];
                }
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e] *= sc;
            if (w) {
                float x[8];
                ofg::unpack8(*(const u32x4*)(w + c), x);
#pragma unroll
                for (int e = 0; e < 8; ++e) o[e] += own * x[e];
            }
        }
        *(u32x4*)(dst + c) = ofg::pack8(o);
    }
}

size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }
long rows_padded(long rows) { return rows > 0 ? (rows + 255) & ~255l : 256; }
int depth_padded(int d) { return (d + 63) & ~63; }

// Vocabulary rows of one backward piece.  D (rows x piece, bf16) is written once and read twice: up to 128 MB it stays in the Infinity
// Cache; a larger piece saves passes over the fp32 sums of dx.
int ce_piece(const OfLinearCeArgs& a) {
    long p = a.piece;
    if (p <= 0) p = (128l << 20) / (2 * rows_padded(a.rows));
    // ... and the products' byte offsets are 32-bit: a piece of the table and a piece of D both stay below 4 GiB
    const long wide = a.ldw > depth_padded(a.d) ? a.ldw : depth_padded(a.d), tall = rows_padded(a.rows);
    const long most = ((1l << 31) - 1) / (wide > tall ? wide : tall);
    if (p > most) p = most;
    p &= ~255l;
    const long all = (a.vocab + 255l) & ~255l;
    if (p < 256) p = 256;
    return (int)(p < all ? p : all);
}
// fp32 sums of dx: rows x d, or the parts of fewer rows (of_ce_splits: parts x tiles <= the chip's CUs)
size_t ce_acc_bytes(const OfLinearCeArgs& a) {
    const long rp = rows_padded(a.rows), nt = (a.d + 255) >> 8, most = ce_piece(a) / 64 / CE_PART_STAGES;
    long rows = OF_NUM_CUS / nt * 256;
    if (rows > most * rp) rows = most * rp;
    return up256((size_t)(rows > rp ? rows : rp) * a.d * 4);
}
// what the forward leaves for the backward
struct CeState {
    int *count, *far, *slot_of, *row_of, *lab;
    float *lse, *ref, *zlab, *acc;          // (the last three: EARLY)
    bf16_t* xc;
    size_t bytes;
};
CeState ce_state(const OfLinearCeArgs& a) {
    const size_t rp = (size_t)rows_padded(a.rows);
    char* at = (char*)a.state;
    CeState s{};
    auto take = [&](size_t n) {
        char* p = at;
        at += up256(n);
        return p;
    };
    s.count = (int*)take(8);
    s.far = s.count + 1;
    s.slot_of = (int*)take(rp * 4);
    s.row_of = (int*)take(rp * 4);
    s.lab = (int*)take(rp * 4);
    s.lse = (float*)take(rp * 4);
    s.xc = (bf16_t*)take(rp * depth_padded(a.d) * 2);
    if (a.early_dx) {
        s.ref = (float*)take(rp * 4);
        s.zlab = (float*)take(rp * 4);
        s.acc = (float*)take(ce_acc_bytes(a));
    }
    s.bytes = (size_t)(at - (char*)a.state);
    return s;
}

size_t ce_table_bytes(const OfLinearCeArgs& a) { return depth_padded(a.d) != a.d ? up256((size_t)a.vocab * depth_padded(a.d) * 2) : 0; }

bool ce_few(long rows, int d) { return rows > 0 && rows <= 16 && d > 0 && (d & 7) == 0 && rows * d <= 1 << 15; }          // (rounded up: 128 KB of x in LDS at most)

int ce_check(const OfLinearCeArgs* args, bool few = false) {
    if (!args) return OF_E_ARG;
    const OfLinearCeArgs& a = *args;
    if (!a.x || !a.w || !a.labels || (!a.state && !few) || !a.workspace) return OF_E_ARG;
    if (a.rows <= 0 || a.vocab <= 0 || a.d <= 0 || a.ldx < a.d || a.ldw < a.d || a.piece < 0) return OF_E_ARG;
    if (a.reduction < OF_CE_NONE || a.reduction > OF_CE_SUM) return OF_E_ARG;
    if ((a.d & 7) || a.rows > (1l << 30) || a.vocab > (1 << 30)) return OF_E_SHAPE;
    if ((a.ldx & 7) || (a.ldw & 7) || ((uintptr_t)a.x & 15) || ((uintptr_t)a.w & 15) || ((uintptr_t)a.state & 15) || ((uintptr_t)a.workspace & 15))
        return OF_E_ALIGN;
    if (few) return 0;
    if (a.state_bytes < of_linear_ce_state_bytes(args)) return OF_E_WORKSPACE;
    // byte offsets inside a tile's operand windows are 32-bit (gemm_w4m.hip); the weight gradient walks all rows of D and of xc
    const unsigned long long lim = 1ull << 32;
    if (2ull * 256 * (unsigned long long)a.ldw >= lim || 2ull * 256 * (unsigned long long)rows_padded(a.rows) >= lim || 2ull * (unsigned long long)rows_padded(a.rows) * depth_padded(a.d) >= lim) return OF_E_SHAPE;
    return 0;
}

// the table the products read: the caller's, or its copy with padded rows at the start of the workspace
int ce_table(const OfLinearCeArgs& a, of_stream_t s, const bf16_t*& w, long& ldw, char*& ws) {
    w = a.w;
    ldw = a.ldw;
    ws = (char*)a.workspace;
    if (depth_padded(a.d) == a.d) return 0;
    CeRowsArgs r{};
    r.w = a.w; r.ldw = a.ldw; r.w_rows = a.vocab; r.d = a.d; r.d_pad = depth_padded(a.d);
    r.wc = (bf16_t*)ws; r.ldwc = r.d_pad;
    w = r.wc;
    ldw = r.ldwc;
    ws += ce_table_bytes(a);
    const long wg = (a.vocab + 3l) / 4;
    return of_launch(ce_pad_table_kernel, of_dim3{(unsigned)(wg < 4096 ? wg : 4096), 1, 1}, 256, 0, s, r);
}

// the logits product of table rows [v0, v0 + n): A = the gathered rows, B = the table
OfCeGemmArgs ce_logits_args(const OfLinearCeArgs& a, const CeState& st, const bf16_t* w, long ldw, int v0, int n) {
    OfCeGemmArgs g{};
    const int dp = depth_padded(a.d);
    g.A = st.xc; g.lda = dp;
    g.B = w + (size_t)v0 * ldw; g.ldb = (int)ldw;
    g.M = (int)rows_padded(a.rows); g.N = (n + 255) & ~255; g.K = dp;
    g.alpha = a.logit_scale;
    g.count = st.count;
    g.b_bytes = ((long)(n - 1) * ldw + dp) * 2;
    g.n_valid = n; g.col0 = v0;
    g.lab = st.lab; g.lse = st.lse;
    return g;
}

// dx_acc += D W of table rows [v0, v0 + n)
OfCeGemmArgs ce_dx_args(const OfLinearCeArgs& a, const CeState& st, const bf16_t* w, long ldw, int v0, int n, const bf16_t* D, float* acc) {
    OfCeGemmArgs q{};
    const int piece = ce_piece(a);
    q.epi = OF_EPI_CE_DX;
    q.A = D; q.lda = piece;
    q.B = w + (size_t)v0 * ldw; q.ldb = (int)ldw; q.b_trans = 1;
    q.b_bytes = ((long)(n - 1) * ldw + depth_padded(a.d)) * 2;
    q.M = (int)rows_padded(a.rows); q.N = (a.d + 255) & ~255; q.K = (n + 63) & ~63;
    q.C = acc; q.ldc = a.d; q.beta = v0 ? 1.f : 0.f; q.alpha = 1.f;
    q.count = st.count; q.n_valid = a.d; q.split_stages = piece / 64;
    return q;
}

}  // namespace

extern "C" size_t of_linear_ce_state_bytes(const OfLinearCeArgs* args) {
    if (!args || args->rows <= 0 || args->vocab <= 0 || args->d <= 0) return 0;
    OfLinearCeArgs a = *args;
    a.state = nullptr;
    return ce_state(a).bytes;
}

extern "C" int of_linear_ce_stateless(long rows, int d) { return ce_few(rows, d); }

extern "C" size_t of_linear_ce_workspace_bytes(const OfLinearCeArgs* args, int backward) {
    if (!args || args->rows <= 0 || args->vocab <= 0 || args->d <= 0) return 0;
    const OfLinearCeArgs& a = *args;
    const size_t rp = (size_t)rows_padded(a.rows);
    if (!backward && !a.state && ce_few(a.rows, a.d)) return (size_t)a.rows * FEW_WG * 8 + 256;
    const size_t strips = (size_t)((a.vocab + 255l) / 256) * 2, D = up256(rp * (size_t)ce_piece(a) * 2);
    if (!backward) return ce_table_bytes(a) + up256(strips * rp * 8) + (a.early_dx ? D : up256(rp * 4));
    return ce_table_bytes(a) + D + (a.dx && !a.early_dx ? ce_acc_bytes(a) : 0) + (a.reduction == OF_CE_NONE && !a.early_dx ? up256(rp * 4) : 0);
}

template <int MT>
static int ce_few_launch(const CeFewArgs& f, of_stream_t s) {
    const size_t lds = (((size_t)MT * f.d * 2 + 15) & ~(size_t)15) + FEW_WAVES * MT * FEW_R * 2 * sizeof(float);
    const int rc = of_launch(ce_few_kernel<MT>, of_dim3{FEW_WG, 1, 1}, FEW_WAVES * 64, lds, s, f);
    return rc ? rc : of_launch(ce_few_finish_kernel, of_dim3{1, 1, 1}, 256, 16 * sizeof(float), s, f);
}

extern "C" int of_linear_ce_fwd(const OfLinearCeArgs* args, void* stream) {
    const bool few = args && !args->state && ce_few(args->rows, args->d);
    const int bad = ce_check(args, few);
    if (bad) return bad;
    const OfLinearCeArgs& a = *args;
    if (few) {
        if (!a.loss_rows || (a.reduction != OF_CE_NONE && !a.loss)) return OF_E_ARG;
        if (a.workspace_bytes < of_linear_ce_workspace_bytes(args, 0)) return OF_E_WORKSPACE;
        CeFewArgs f{a.x, a.ldx, a.w, a.ldw, a.labels, a.ignore_index, (int)a.rows, a.vocab, a.d, a.logit_scale * oft::CE_LOG2E, (float*)((char*)a.workspace + 256),
                    (float*)a.workspace, a.loss_rows, a.reduction == OF_CE_NONE ? nullptr : a.loss, a.reduction == OF_CE_MEAN};
        of_stream_t s = (of_stream_t)stream;
        if (a.rows <= 1) return ce_few_launch<1>(f, s);
        if (a.rows <= 2) return ce_few_launch<2>(f, s);
        if (a.rows <= 4) return ce_few_launch<4>(f, s);
        if (a.rows <= 8) return ce_few_launch<8>(f, s);
        return ce_few_launch<16>(f, s);
    }
    if (!a.loss_rows || (a.reduction != OF_CE_NONE && !a.loss)) return OF_E_ARG;
    if (a.workspace_bytes < of_linear_ce_workspace_bytes(args, 0)) return OF_E_WORKSPACE;
    of_stream_t s = (of_stream_t)stream;
    const CeState st = ce_state(a);
    const long rp = rows_padded(a.rows);
    const bf16_t* w;
    long ldw;
    char* ws;
    int rc = ce_table(a, s, w, ldw, ws);
    if (rc) return rc;

    CeRowsArgs r{};
    r.labels = a.labels; r.ignore_index = a.ignore_index; r.rows = a.rows; r.vocab = a.vocab;
    r.count = st.count; r.slot_of = st.slot_of; r.row_of = st.row_of; r.lab = st.lab; r.lse = st.lse;
    r.loss_rows = a.loss_rows; r.loss = a.reduction == OF_CE_NONE ? nullptr : a.loss; r.mean = a.reduction == OF_CE_MEAN;
    r.x = a.x; r.ldx = a.ldx; r.xc = st.xc; r.ldxc = depth_padded(a.d); r.d = a.d; r.d_pad = depth_padded(a.d);
    if (a.early_dx) {
        r.ref = st.ref; r.far = st.far; r.sc2 = a.logit_scale * oft::CE_LOG2E;
        r.w = w; r.ldw = ldw;
    }
    if (a.rows <= CE_FEW_ROWS) {
        rc = of_launch(ce_index_gather_kernel, of_dim3{(unsigned)(rp / 4), 1, 1}, 256, 0, s, r);
    } else {
        rc = of_launch(ce_index_kernel, of_dim3{1, 1, 1}, CE_THREADS, CE_THREADS / 64 * sizeof(int), s, r);
        if (rc) return rc;
        rc = of_launch(ce_gather_kernel, of_dim3{(unsigned)(rp / 4), 1, 1}, 256, 0, s, r);
    }
    if (rc) return rc;

    r.strips = (int)((a.vocab + 255l) / 256) * 2;
    r.part_ld = rp;
    r.part = (float*)ws;
    if (a.early_dx) {
        bf16_t* D = (bf16_t*)(ws + up256((size_t)r.strips * rp * 8));
        r.zlab = st.zlab;
        const int piece = ce_piece(a);
        for (int v0 = 0; v0 < a.vocab; v0 += piece) {
            const int n = a.vocab - v0 < piece ? a.vocab - v0 : piece;
            OfCeGemmArgs g = ce_logits_args(a, st, w, ldw, v0, n);
            g.epi = OF_EPI_CE_EARLY;
            g.lse = st.ref; g.C = D; g.ldc = piece;
            g.part = (float*)ws; g.part_ld = rp; g.zlab = st.zlab;
            rc = of_gemm_w4m_ce(g, s);
            if (rc) return rc;
            rc = of_gemm_w4m_ce(ce_dx_args(a, st, w, ldw, v0, n, D, st.acc), s);
            if (rc) return rc;
        }
    } else {
        OfCeGemmArgs g = ce_logits_args(a, st, w, ldw, 0, a.vocab);
        g.epi = OF_EPI_CE_LSE;
        g.part = (float*)ws; g.part_ld = rp;
        g.zlab = (float*)(ws + up256((size_t)r.strips * rp * 8));
        r.zlab = g.zlab;
        rc = of_gemm_w4m_ce(g, s);
        if (rc) return rc;
    }
    if (!a.early_dx && rp * r.strips <= CE_FEW_PARTS) return of_launch(ce_finish_reduce_kernel, of_dim3{1, 1, 1}, CE_THREADS, CE_THREADS * sizeof(float), s, r);
    const of_dim3 grid{(unsigned)(rp / 16), 1, 1};
    const size_t lds = 16 * 16 * 2 * sizeof(float);
    rc = of_launch(ce_finish_kernel, grid, 256, lds, s, r);
    if (rc) return rc;
    if (a.early_dx) {          // some loss above CE_FAR: the statistics with a maximum, for every row
        OfCeGemmArgs g = ce_logits_args(a, st, w, ldw, 0, a.vocab);
        g.epi = OF_EPI_CE_LSE;
        g.part = (float*)ws; g.part_ld = rp; g.zlab = st.zlab;
        g.gate = r.gate = st.far;
        rc = of_gemm_w4m_ce(g, s);
        if (rc) return rc;
        r.ref = nullptr; r.far = nullptr;
        rc = of_launch(ce_finish_kernel, grid, 256, lds, s, r);
        if (rc) return rc;
    }
    if (a.reduction == OF_CE_NONE) return 0;
    return of_launch(ce_reduce_kernel, of_dim3{1, 1, 1}, CE_THREADS, CE_THREADS * sizeof(float), s, r);
}

extern "C" int of_linear_ce_bwd(const OfLinearCeArgs* args, void* stream) {
    const int bad = ce_check(args);
    if (bad) return bad;
    const OfLinearCeArgs& a = *args;
    if (!a.grad || (!a.dx && !a.dw) || (a.early_dx && (!a.dx || a.dw))) return OF_E_ARG;
    if ((a.dx && a.lddx < a.d) || (a.dw && a.lddw < a.d)) return OF_E_ARG;
    if ((a.lddx & 7) || (a.lddw & 7) || ((uintptr_t)a.dx & 15) || ((uintptr_t)a.dw & 15)) return OF_E_ALIGN;
    if (a.workspace_bytes < of_linear_ce_workspace_bytes(args, 1)) return OF_E_WORKSPACE;
    of_stream_t s = (of_stream_t)stream;
    const CeState st = ce_state(a);
    const long rp = rows_padded(a.rows);
    const int piece = ce_piece(a), dp = depth_padded(a.d), d256 = (a.d + 255) & ~255;
    const bf16_t* w;
    long ldw;
    char* ws;
    int rc = ce_table(a, s, w, ldw, ws);
    if (rc) return rc;
    bf16_t* D = (bf16_t*)ws;
    ws += up256((size_t)rp * piece * 2);
    float* acc = st.acc;
    if (a.dx && !acc) {
        acc = (float*)ws;
        ws += ce_acc_bytes(a);
    }

    CeRowsArgs r{};
    r.rows = a.rows; r.count = st.count; r.slot_of = st.slot_of; r.row_of = st.row_of;
    r.d = a.d; r.acc = acc; r.split_stages = piece / 64; r.dx = a.dx; r.lddx = a.lddx;
    float* grow = nullptr;
    if (a.early_dx) {          // the rows' own gradients join at the end
        r.far = st.far; r.ref = st.ref; r.zlab = st.zlab; r.lse = st.lse; r.lab = st.lab; r.w = w; r.ldw = ldw;
        if (a.reduction == OF_CE_NONE) r.grow = const_cast<float*>(a.grad);
    } else if (a.reduction == OF_CE_NONE) {
        r.grad = a.grad;
        r.grow = grow = (float*)ws;
        rc = of_launch(ce_row_grads_kernel, of_dim3{(unsigned)((rp + 255) / 256), 1, 1}, 256, 0, s, r);
        if (rc) return rc;
        r.grow = nullptr;
    }
    const float* gscale = a.reduction == OF_CE_NONE ? nullptr : a.grad;
    const int by_count = a.reduction == OF_CE_MEAN;

    for (int v0 = 0; v0 < a.vocab; v0 += piece) {
        const int n = a.vocab - v0 < piece ? a.vocab - v0 : piece;
        OfCeGemmArgs g = ce_logits_args(a, st, w, ldw, v0, n);
        g.epi = OF_EPI_CE_DLOGIT;
        g.C = D; g.ldc = piece; g.grow = grow;
        if (a.early_dx) g.gate = st.far;
        rc = of_gemm_w4m_ce(g, s);
        if (rc) return rc;
        if (a.dx) {
            OfCeGemmArgs q = ce_dx_args(a, st, w, ldw, v0, n, D, acc);
            if (a.early_dx) q.gate = st.far;
            rc = of_gemm_w4m_ce(q, s);
            if (rc) return rc;
        }
        if (a.dw) {
            OfCeGemmArgs q{};
            q.epi = OF_EPI_CE_DW;
            q.A = D; q.lda = piece; q.a_trans = 1;
            q.B = st.xc; q.ldb = dp; q.b_trans = 1;
            q.b_bytes = rp * dp * 2;
            q.M = (n + 255) & ~255; q.N = d256; q.K = (int)rp;
            q.C = a.dw + (size_t)v0 * a.lddw; q.ldc = (int)a.lddw;
            q.alpha = a.logit_scale;
            q.count = st.count; q.n_valid = a.d; q.m_valid = n;
            q.gscale = gscale; q.by_count = by_count;
            rc = of_gemm_w4m_ce(q, s);
            if (rc) return rc;
        }
    }
    if (!a.dx) return 0;
    r.grad = gscale; r.by_count = by_count; r.logit_scale = a.logit_scale;
    return of_launch(ce_scatter_kernel, of_dim3{(unsigned)((a.rows + 3) / 4), 1, 1}, 256, 0, s, r);
}
