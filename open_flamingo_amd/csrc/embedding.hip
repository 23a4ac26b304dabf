// Lookup in a vocabulary table with a scale, and its gradient by sorted tokens (gfx950, HBM-bound).
//   y[i] = scale * W[id_i]                       one wave per position, 16-byte loads and stores
//   dW[v] = scale * sum over {i: id_i = v} dy[i]   in fp32, positions in ascending order; rows without a token are zeros
// The gradient has to read dy once (n x d) and to write the table once (vocabulary x d).  Scattered with atomics into a zeroed table it would
// depend on their order, and round behind every addition where the table is bf16.  Here, without floating-point atomics:
//   sort     (id, position) by id, stable: radix passes of 9 bits.  Up to 16384 positions ONE workgroup sorts in LDS while the
//            others of the same launch clear the table; more positions take two launches a pass (counts, placement), from 2^22 + 1 on a
//            third that adds the counts up.
//            Ids that have no gradient (padding_idx, ids outside the table) sort behind all others.
//   sum      a workgroup takes a chunk of the sorted list and 256 vectors of columns and walks the chunk with the running sum in
//            registers.  A token whose positions lie inside the chunk is finished there; the two that cross its ends leave fp32
//            partial rows in the workspace;
//   join     the chunk in which a crossing token begins adds the partial rows of the chunks behind it, in order.
// The same ids and gradients give the same bits on every run.
// Measured: 8192 tokens of a 50435 x 2048 fp32 table, forward and gradient 134 us (lookup 39, sort beside the clearing of 413 MB 58, sums 33, join
// 5; 614 MB); 32768 tokens, 4096 columns of bf16, skewed ids: 309 us (lookup 85, the rest 222).  Waited for one by one 181 and 347 us; torch's
// embedding module takes 323 and 1310 (the second with its scaling as a pass of its own), and 34 and 93 against 36 and 100 forward alone.
#include "gemm_common.h"

namespace {

constexpr int RB = 9, BINS = 1 << RB;            // two passes up to a vocabulary of 2^18 - 1
constexpr int SMALL_MAX = 16384;                 // positions one workgroup sorts in LDS
constexpr int SMALL_THREADS = 1024;
constexpr int TILE = 4096, TILE_THREADS = 512;   // positions per workgroup of a pass over more
constexpr int SCAN_TILES = 1024;                 // up to this many tiles each adds their counts up for itself: a launch less per pass (32768
                                                 // positions x 4096, gradient: 234 -> 218 us with 8 tiles; 1048576 x 64: 431 -> 380 with 256; 4000000: 1537 -> 1347)
constexpr int VEC_THREADS = 256;

struct EmbArgs {
    const long long* ids; long n; int vocab; int d; long long padding_idx;
    const void* table; long ldt; int f32; int vec; float scale;
    void* y; long ldy;
    const void* dy; long lddy; void* dw; long lddw;
    unsigned *key_in, *pos_in, *key_out, *pos_out; int shift; int from_ids; int nb;
    int* hist;
    const unsigned *key, *pos; int chunk; long chunks; float* part;
    int passes; int cap;
};

OF_DEV unsigned emb_key(const EmbArgs& a, long i) {
    const long long id = a.ids[i];
    return id < 0 || id >= a.vocab || id == a.padding_idx ? (unsigned)a.vocab : (unsigned)id;
}

// ------------------------------------------------------------------------------------------------ forward
// one wave per position; `vec`: rows of whole 16-byte vectors at 16-byte addresses
OF_GLOBAL void OF_BOUNDS(256, 4) emb_fwd_kernel(EmbArgs a) {
    const int lane = of_tid() & 63;
    const long i = (long)of_bid_x() * 4 + (of_tid() >> 6);
    if (i >= a.n) return;
    const long long id = a.ids[i];
    const bool inside = id >= 0 && id < a.vocab;
    const float bad = __builtin_nanf("");          // an id outside the table: a caller's mistake, read nowhere, visible everywhere
    const size_t src = inside ? (size_t)id * a.ldt : 0, dst = (size_t)i * a.ldy;
    if (a.vec && inside) {          // eight 16-byte loads of a lane in flight
        const int per = a.d / (a.f32 ? 4 : 8);
        const u32x4* t = (const u32x4*)((const char*)a.table + src * (a.f32 ? 4 : 2));
        u32x4* o = (u32x4*)((char*)a.y + dst * (a.f32 ? 4 : 2));
        for (int c0 = 0; c0 < per; c0 += 512) {
            u32x4 v[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const int c = c0 + u * 64 + lane;
                if (c < per) v[u] = t[c];
            }
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const int c = c0 + u * 64 + lane;
                if (c >= per) break;
                if (a.scale != 1.0f) {
                    if (a.f32) {
                        const f32x4 x = __builtin_bit_cast(f32x4, v[u]);
                        v[u] = __builtin_bit_cast(u32x4, f32x4{a.scale * x[0], a.scale * x[1], a.scale * x[2], a.scale * x[3]});
                    } else {
                        float x[8];
                        ofg::unpack8(v[u], x);
#pragma unroll
                        for (int e = 0; e < 8; ++e) x[e] *= a.scale;
                        v[u] = ofg::pack8(x);
                    }
                }
                o[c] = v[u];
            }
        }
        return;
    }
    for (int c = lane; c < a.d; c += 64) {
        if (a.f32) ((float*)a.y)[dst + c] = inside ? a.scale * ((const float*)a.table)[src + c] : bad;
        else ((bf16_t*)a.y)[dst + c] = inside ? of_f32_to_bf16(a.scale * of_bf16_to_f32(((const bf16_t*)a.table)[src + c])) : of_f32_to_bf16(bad);
    }
}

// ------------------------------------------------------------------------------------------------ sort
// The lanes of the wave that hold the same digit as this one (dead lanes match nobody)
OF_DEV unsigned long long emb_match(unsigned digit, bool live) {
    unsigned long long m = of_ballot(live);
#pragma unroll
    for (int b = 0; b < RB; ++b) {
        const unsigned long long one = of_ballot((digit >> b) & 1);
        m &= (digit >> b) & 1 ? one : ~one;
    }
    return m;
}
OF_DEV int emb_below(unsigned long long m, int lane) { return __builtin_popcountll(m & ((1ull << lane) - 1)); }

// running sums over the bins, in place; every thread of the workgroup calls it
OF_DEV void emb_scan_bins(int* cum, int tid) {
    for (int o = 1; o < BINS; o <<= 1) {
        const int v = tid < BINS && tid >= o ? cum[tid - o] : 0;
        of_sync();
        if (tid < BINS) cum[tid] += v;
        of_sync();
    }
}

// Turns cnt[wave][digit] (how often each wave met each digit) into the place of the wave's first such element: in a tile that is all there
// is (given = false), or from `at`, the place of the tile's first element of digit `tid`.  The waves hold consecutive parts of the tile: the order stays.  LDS: cnt, cum[BINS];
// every thread of the workgroup calls.
template <class CNT>
OF_DEV void emb_offsets(CNT* cnt, int* cum, int waves, int tid, bool given, int at) {
    of_sync();
    int total = 0;
    if (tid < BINS) {
        for (int w = 0; w < waves; ++w) total += cnt[w * BINS + tid];
        cum[tid] = total;
    }
    of_sync();
    if (!given) {
        emb_scan_bins(cum, tid);
        at = tid < BINS ? cum[tid] - total : 0;
    }
    if (tid < BINS)
        for (int w = 0; w < waves; ++w) {
            const int c = cnt[w * BINS + tid];
            cnt[w * BINS + tid] = (CNT)at;
            at += c;
        }
    of_sync();
}

// zeros in the whole of dw
OF_DEV void emb_fill(const EmbArgs& a, long block, long blocks, int tid, int nthreads) {
    const int es = a.f32 ? 4 : 2;
    if (a.vec && a.lddw == a.d) {
        const long per = (long)a.vocab * a.d * es / 16;
        for (long i = block * nthreads + tid; i < per; i += blocks * nthreads) *(u32x4*)((char*)a.dw + i * 16) = u32x4{0u, 0u, 0u, 0u};
        return;
    }
    for (long r = block; r < a.vocab; r += blocks)
        for (int c = tid; c < a.d; c += nthreads) {
            if (a.f32) ((float*)a.dw)[(size_t)r * a.lddw + c] = 0.f;
            else ((bf16_t*)a.dw)[(size_t)r * a.lddw + c] = 0;
        }
}

// Workgroup 0 sorts all positions (at most SMALL_MAX) in LDS: two lists of key << 14 | position (a key has 18 bits at most: larger
// vocabularies take the launches below), 16-bit counters of every wave (a place is below 16384), the scan.  The others clear the table.
constexpr int SMALL_WAVES = SMALL_THREADS / 64, SMALL_ITERS = SMALL_MAX / SMALL_THREADS;
OF_GLOBAL void OF_BOUNDS(SMALL_THREADS, 1) emb_sort_small_kernel(EmbArgs a) {
    const int tid = of_tid(), lane = tid & 63, wave = tid >> 6;
    if (of_bid_x() > 0) {
        emb_fill(a, of_bid_x() - 1, of_gdim_x() - 1, tid, SMALL_THREADS);
        return;
    }
    unsigned* from = (unsigned*)of_smem();
    unsigned* to = from + a.cap;
    unsigned short* cnt = (unsigned short*)(to + a.cap);
    int* cum = (int*)(cnt + SMALL_WAVES * BINS);
    const int n = (int)a.n;
    const int iters = (n + SMALL_THREADS - 1) / SMALL_THREADS;          // 64 elements of every wave at a time; a wave's part is consecutive
    const int lo = wave * iters * 64;
    for (int i = tid; i < n; i += SMALL_THREADS) from[i] = emb_key(a, i) << 14 | (unsigned)i;
    for (int p = 0; p < a.passes; ++p) {
        for (int i = tid; i < SMALL_WAVES * BINS; i += SMALL_THREADS) cnt[i] = 0;
        of_sync();
        unsigned short* mine = cnt + wave * BINS;
        int rank[SMALL_ITERS];
#pragma unroll
        for (int it = 0; it < SMALL_ITERS; ++it) {
            if (it < iters) {
                const int i = lo + it * 64 + lane;
                const bool live = i < n;
                const unsigned digit = live ? (from[i] >> (14 + p * RB)) & (BINS - 1) : 0;
                const unsigned long long same = emb_match(digit, live);
                const int before = emb_below(same, lane);
                if (live) rank[it] = mine[digit] + before;
                of_wave_sync();
                if (live && before == 0) mine[digit] += (unsigned short)__builtin_popcountll(same);
                of_wave_sync();
            }
        }
        emb_offsets(cnt, cum, SMALL_WAVES, tid, false, 0);
#pragma unroll
        for (int it = 0; it < SMALL_ITERS; ++it) {
            if (it < iters) {
                const int i = lo + it * 64 + lane;
                if (i < n) {
                    const unsigned e = from[i];
                    to[mine[(e >> (14 + p * RB)) & (BINS - 1)] + rank[it]] = e;
                }
            }
        }
        of_sync();
        unsigned* t = from;
        from = to;
        to = t;
    }
    for (int i = tid; i < n; i += SMALL_THREADS) {
        a.key_out[i] = from[i] >> 14;
        a.pos_out[i] = from[i] & 16383u;
    }
}

// ---- more positions: two or three launches a pass.  key / position i of the pass's input (the first pass reads the ids)
OF_DEV unsigned emb_in_key(const EmbArgs& a, long i) { return a.from_ids ? emb_key(a, i) : a.key_in[i]; }

// counts of the digits of every tile: hist[tile][digit]; workgroups behind the tiles clear the table
OF_GLOBAL void OF_BOUNDS(TILE_THREADS, 2) emb_count_kernel(EmbArgs a) {
    const int tid = of_tid();
    if (of_bid_x() >= a.nb) {
        emb_fill(a, of_bid_x() - a.nb, of_gdim_x() - a.nb, tid, TILE_THREADS);
        return;
    }
    int* cnt = (int*)of_smem();
    cnt[tid] = 0;
    of_sync();
    const long first = (long)of_bid_x() * TILE;
    for (long i = first + tid; i < first + TILE && i < a.n; i += TILE_THREADS) of_lds_count(cnt + ((emb_in_key(a, i) >> a.shift) & (BINS - 1)), 1);
    of_sync();
    a.hist[(size_t)of_bid_x() * BINS + tid] = cnt[tid];
}
// hist -> the place of every (digit, tile)'s first element; one workgroup, a thread per digit
OF_GLOBAL void OF_BOUNDS(BINS, 1) emb_scan_kernel(EmbArgs a) {
    int* cum = (int*)of_smem();
    const int tid = of_tid();
    int* mine = a.hist + tid;
    int total = 0;
    for (int b = 0; b < a.nb; ++b) total += mine[(size_t)b * BINS];
    cum[tid] = total;
    of_sync();
    emb_scan_bins(cum, tid);
    int at = cum[tid] - total;
    for (int b = 0; b < a.nb; ++b) {
        const int c = mine[(size_t)b * BINS];
        mine[(size_t)b * BINS] = at;
        at += c;
    }
}
constexpr int TILE_WAVES = TILE_THREADS / 64, TILE_ITERS = TILE / TILE_THREADS;
OF_GLOBAL void OF_BOUNDS(TILE_THREADS, 2) emb_place_kernel(EmbArgs a) {
    const int tid = of_tid(), lane = tid & 63, wave = tid >> 6;
    int* cnt = (int*)of_smem();
    int* cum = cnt + TILE_WAVES * BINS;
    int* mine = cnt + wave * BINS;
    for (int i = tid; i < TILE_WAVES * BINS; i += TILE_THREADS) cnt[i] = 0;
    of_sync();
    int total = 0, earlier = 0;          // of digit `tid`: in all tiles, in those in front of this one
    if (a.nb <= SCAN_TILES)
        for (int b = 0; b < a.nb; ++b) {
            const int c = a.hist[(size_t)b * BINS + tid];
            total += c;
            if (b < of_bid_x()) earlier += c;
        }
    const long lo = (long)of_bid_x() * TILE + wave * TILE_ITERS * 64;
    int rank[TILE_ITERS];
    unsigned key[TILE_ITERS], pos[TILE_ITERS];
#pragma unroll
    for (int it = 0; it < TILE_ITERS; ++it) {
        const long i = lo + it * 64 + lane;
        key[it] = i < a.n ? emb_in_key(a, i) : 0;
        pos[it] = i < a.n ? (a.from_ids ? (unsigned)i : a.pos_in[i]) : 0;
    }
#pragma unroll
    for (int it = 0; it < TILE_ITERS; ++it) {
        const bool live = lo + it * 64 + lane < a.n;
        const unsigned digit = (key[it] >> a.shift) & (BINS - 1);
        const unsigned long long same = emb_match(digit, live);
        const int before = emb_below(same, lane);
        if (live) rank[it] = mine[digit] + before;
        of_wave_sync();
        if (live && before == 0) mine[digit] += __builtin_popcountll(same);
        of_wave_sync();
    }
    int at = 0;          // place of this tile's first element of digit `tid`
    if (a.nb > SCAN_TILES) {
        at = a.hist[(size_t)of_bid_x() * BINS + tid];
    } else {
        cum[tid] = total;
        of_sync();
        emb_scan_bins(cum, tid);
        at = cum[tid] - total + earlier;
    }
    emb_offsets(cnt, cum, TILE_WAVES, tid, true, at);
#pragma unroll
    for (int it = 0; it < TILE_ITERS; ++it) {
        if (lo + it * 64 + lane < a.n) {
            const int at = mine[(key[it] >> a.shift) & (BINS - 1)] + rank[it];
            a.key_out[at] = key[it];
            a.pos_out[at] = pos[it];
        }
    }
}

// ------------------------------------------------------------------------------------------------ sums
// the columns one thread owns: a 16-byte vector of dy, or one element
template <bool F32, bool VEC>
struct EmbVec {
    static constexpr int W = VEC ? (F32 ? 4 : 8) : 1;
};
// as it lies in memory (so that loads stay in flight), and added to a sum
template <bool F32, bool VEC>
OF_DEV u32x4 emb_raw(const void* base, size_t at) {
    if constexpr (VEC) return *(const u32x4*)((const char*)base + at * (F32 ? 4 : 2));
    else return u32x4{F32 ? ((const unsigned*)base)[at] : (unsigned)((const bf16_t*)base)[at], 0u, 0u, 0u};
}
template <bool F32, bool VEC>
OF_DEV void emb_add(u32x4 v, float (&s)[8]) {
    if constexpr (!VEC) s[0] += F32 ? __builtin_bit_cast(float, v[0]) : of_bf16_to_f32((bf16_t)v[0]);
    else if constexpr (F32) {
        const f32x4 x = __builtin_bit_cast(f32x4, v);
#pragma unroll
        for (int e = 0; e < 4; ++e) s[e] += x[e];
    } else {
        float x[8];
        ofg::unpack8(v, x);
#pragma unroll
        for (int e = 0; e < 8; ++e) s[e] += x[e];
    }
}
template <bool F32, bool VEC>
OF_DEV void emb_store(void* base, size_t at, const float (&x)[8], float sc) {
    if constexpr (!VEC) {
        if (F32) ((float*)base)[at] = sc * x[0];
        else ((bf16_t*)base)[at] = of_f32_to_bf16(sc * x[0]);
    } else if constexpr (F32) *(f32x4*)((float*)base + at) = f32x4{sc * x[0], sc * x[1], sc * x[2], sc * x[3]};
    else {
        float o[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = sc * x[e];
        *(u32x4*)((bf16_t*)base + at) = ofg::pack8(o);
    }
}

constexpr int AHEAD = 8;          // rows of dy in flight per thread

// grid (chunks, column blocks).  part[chunk][0]: the sum of a token that began in an earlier chunk, [1]: of one that begins here and
// goes on behind this chunk's end (a token that fills the whole chunk and does both counts as [0]).  64 entries of the list at a time sit
// in a register, one a lane: the walk reads them with v_readlane.
template <bool F32, bool VEC>
OF_GLOBAL void OF_BOUNDS(VEC_THREADS, 4) emb_sum_kernel(EmbArgs a) {
    typedef EmbVec<F32, VEC> V;
    const long chunk = of_bid_x(), lo = chunk * a.chunk, hi = lo + a.chunk < a.n ? lo + a.chunk : a.n;
    const int lane = of_tid() & 63;
    const int col = (of_bid_y() * VEC_THREADS + of_tid()) * V::W;
    const bool mine = col < a.d;
    const unsigned none = (unsigned)a.vocab;
    const unsigned before = lo > 0 ? a.key[lo - 1] : none, behind = hi < a.n ? a.key[hi] : none;
    unsigned cur = a.key[lo];
    bool head = lo > 0 && before == cur;
    float s[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    auto flush = [&](bool goes_on) OF_INLINE_LAMBDA {
        if (cur == none || !mine) return;
        if (head || goes_on) {
            float* p = a.part + ((size_t)chunk * 2 + (head ? 0 : 1)) * a.d + col;
#pragma unroll
            for (int e = 0; e < V::W; ++e) p[e] = s[e];
        } else {
            emb_store<F32, VEC>(a.dw, (size_t)cur * a.lddw + col, s, a.scale);
        }
    };
    for (long i0 = lo; i0 < hi; i0 += 64) {
        const int len = hi - i0 < 64 ? (int)(hi - i0) : 64;
        const long at = i0 + (lane < len ? lane : len - 1);
        const unsigned key = a.key[at], pos = a.pos[at];
        for (int i = 0; i < len; i += AHEAD) {
            if (of_readlane(key, i) == none) break;          // sorted: nothing but positions without a gradient from here on
            u32x4 x[AHEAD];
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) {
                const size_t row = of_readlane(pos, i + u < len ? i + u : len - 1);
                x[u] = emb_raw<F32, VEC>(a.dy, row * a.lddy + (mine ? col : 0));
            }
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) {
                const unsigned k = of_readlane(key, i + u < len ? i + u : len - 1);
                if (i + u < len) {
                    if (k != cur) {
                        flush(false);
                        cur = k;
                        head = false;
#pragma unroll
                        for (int e = 0; e < V::W; ++e) s[e] = 0.f;
                    }
                    emb_add<F32, VEC>(x[u], s);
                }
            }
        }
        if (of_readlane(key, len - 1) == none && cur != none) {          // the last token of the list ended in these 64
            flush(false);
            cur = none;
        }
        if (cur == none) return;
    }
    flush(behind == cur);
}

// grid (chunks, column blocks): the chunk whose last token begins there and goes on adds what the following chunks hold of it
template <bool F32, bool VEC>
OF_GLOBAL void OF_BOUNDS(VEC_THREADS, 4) emb_join_kernel(EmbArgs a) {
    typedef EmbVec<F32, VEC> V;
    const long chunk = of_bid_x(), lo = chunk * a.chunk, hi = lo + a.chunk;
    if (hi >= a.n) return;
    const unsigned cur = a.key[hi];
    if (cur == (unsigned)a.vocab || a.key[hi - 1] != cur) return;          // nothing crosses this chunk's end
    if (a.key[lo] == cur && lo > 0 && a.key[lo - 1] == cur) return;        // it began earlier
    const int col = (of_bid_y() * VEC_THREADS + of_tid()) * V::W;
    if (col >= a.d) return;
    float s[8];
    const float* own = a.part + ((size_t)chunk * 2 + 1) * a.d + col;
#pragma unroll
    for (int e = 0; e < V::W; ++e) s[e] = own[e];
    long end = chunk + 1, behind = a.chunks;          // the token is the first of the chunks up to `end`: the list is sorted
    while (end + 1 < behind) {
        const long mid = (end + behind) >> 1;
        if (a.key[mid * a.chunk] == cur) end = mid;
        else behind = mid;
    }
    for (long c = chunk + 1; c <= end; c += AHEAD) {
        float x[AHEAD][8];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const float* p = a.part + (size_t)(c + u <= end ? c + u : end) * 2 * a.d + col;
#pragma unroll
            for (int e = 0; e < V::W; ++e) x[u][e] = p[e];
        }
#pragma unroll
        for (int u = 0; u < AHEAD; ++u)
            if (c + u <= end)
#pragma unroll
                for (int e = 0; e < V::W; ++e) s[e] += x[u][e];
    }
    emb_store<F32, VEC>(a.dw, (size_t)cur * a.lddw + col, s, a.scale);
}

// At most 64 positions: every wave holds all ids, one a lane, and the ballot of the lanes that hold a row's id says which rows of dy make
// it up, in ascending order.  One launch in place of sort, sum and join, and no row is written twice.  All positions on one row cost a
// workgroup 64 rows of dy, AHEAD in flight.
constexpr int FEW = 64;
template <bool F32, bool VEC>
OF_DEV void emb_few_sum(const EmbArgs& a, unsigned long long who, int col, float (&s)[8]) {
    while (who) {
        u32x4 x[AHEAD];
        int many = 0;
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            if (!who) break;
            x[u] = emb_raw<F32, VEC>(a.dy, (size_t)__builtin_ctzll(who) * a.lddy + col);
            who &= who - 1;
            many = u + 1;
        }
#pragma unroll
        for (int u = 0; u < AHEAD; ++u)
            if (u < many) emb_add<F32, VEC>(x[u], s);
    }
}
// any strides and widths: a row of the table per workgroup
template <bool F32, bool VEC>
OF_GLOBAL void OF_BOUNDS(VEC_THREADS, 4) emb_few_kernel(EmbArgs a) {
    typedef EmbVec<F32, VEC> V;
    const int tid = of_tid(), lane = tid & 63;
    const int key = lane < a.n ? (int)emb_key(a, lane) : a.vocab;
    for (long r = of_bid_x(); r < a.vocab; r += of_gdim_x()) {
        const unsigned long long who = of_ballot(key == r);
        for (int col = tid * V::W; col < a.d; col += VEC_THREADS * V::W) {
            float s[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
            emb_few_sum<F32, VEC>(a, who, col, s);
            emb_store<F32, VEC>(a.dw, (size_t)r * a.lddw + col, s, who ? a.scale : 0.f);
        }
    }
}
// The table without gaps, in whole vectors: one vector per thread, 4 KB per workgroup, whatever the rows' ends.  Almost every workgroup finds
// no position in its rows and writes zeros, at the rate of a fill: 50434 x 2048 fp32 in 61 us (61 for the fill alone; 74 with 16 KB per
// workgroup), 47771 x 4008 in 120 (112; 138 by sort and sum, 156 with a row of the table per workgroup, two of which share a cache line),
// 3461 x 2560 in 9 (17 by sort and sum).
template <bool F32>
OF_GLOBAL void OF_BOUNDS(VEC_THREADS, 4) emb_few_flat_kernel(EmbArgs a) {
    typedef EmbVec<F32, true> V;
    const int tid = of_tid(), lane = tid & 63, per = a.d / V::W;
    const int key = lane < a.n ? (int)emb_key(a, lane) : a.vocab;
    const long total = (long)a.vocab * per, lo = (long)of_bid_x() * VEC_THREADS, hi = lo + VEC_THREADS < total ? lo + VEC_THREADS : total, i = lo + tid;
    unsigned long long left = of_ballot(key < a.vocab && key >= lo / per && key <= (hi - 1) / per);
    float s[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    bool any = false;
    if (left) {          // (no lane has left: all of them hold ids)
        const int r = (int)(i / per), col = (int)(i - (long)r * per) * V::W;
        while (left) {
            const int k = (int)of_readlane((unsigned)key, __builtin_ctzll(left));
            const unsigned long long who = of_ballot(key == k);
            left &= ~who;
            if (r == k) {
                emb_few_sum<F32, true>(a, who, col, s);
                any = true;
            }
        }
    }
    if (i < hi) emb_store<F32, true>(a.dw, (size_t)i * V::W, s, any ? a.scale : 0.f);
}

size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }
bool emb_small(long n, int vocab) { return n <= SMALL_MAX && vocab < (1 << 18); }
int emb_passes(int vocab) {
    int bits = 1;
    while ((vocab >> bits) != 0) ++bits;
    return (bits + RB - 1) / RB;
}
// Positions per chunk of the sums: enough chunks to fill the chip, few enough that joining one token that fills them all stays short.  32768
// positions of 4096 columns: 259 us in all with chunks of 8, 242 / 236 / 228 / 226 with 16 / 32 / 64 / 128; 2048 positions of 2048: 84, 84, 92, 109 with 8, 16, 64, 128
int emb_chunk(long n) {
    long c = n / 512 < 64 ? n / 512 : n / 1024 < 64 ? 64 : n / 1024;
    return (int)(c < 16 ? 16 : c > 4096 ? 4096 : (c + AHEAD - 1) / AHEAD * AHEAD);
}
int emb_dtype_ok(int f32) { return f32 == 0 || f32 == 1; }
bool emb_vec(const void* p, long ld, int d, int f32) { const int w = f32 ? 4 : 8; return d % w == 0 && ld % w == 0 && !((uintptr_t)p & 15); }

template <bool F32, bool VEC>
int emb_sums(const EmbArgs& a, of_stream_t s) {
    if (a.n <= FEW) {
        if constexpr (VEC) {
            const long total = (long)a.vocab * (a.d / EmbVec<F32, VEC>::W);
            if (a.lddw == a.d && total < (1l << 31)) return of_launch(emb_few_flat_kernel<F32>, of_dim3{(unsigned)((total + VEC_THREADS - 1) / VEC_THREADS), 1, 1}, VEC_THREADS, 0, s, a);
        }
        return of_launch(emb_few_kernel<F32, VEC>, of_dim3{(unsigned)(a.vocab < 16384 ? a.vocab : 16384), 1, 1}, VEC_THREADS, 0, s, a);
    }
    const of_dim3 grid{(unsigned)a.chunks, (unsigned)((a.d + VEC_THREADS * EmbVec<F32, VEC>::W - 1) / (VEC_THREADS * EmbVec<F32, VEC>::W)), 1};
    const int rc = of_launch(emb_sum_kernel<F32, VEC>, grid, VEC_THREADS, 0, s, a);
    if (rc || a.chunks == 1) return rc;
    return of_launch(emb_join_kernel<F32, VEC>, grid, VEC_THREADS, 0, s, a);
}
}  // namespace

extern "C" int of_embedding_fwd(const long long* ids, long n, const void* table, int f32, long ldt, int vocab, int d, float scale, void* y, long ldy,
                                void* stream) {
    if (!ids || !table || !y || n <= 0 || vocab <= 0 || d <= 0 || ldt < d || ldy < d || !emb_dtype_ok(f32)) return OF_E_ARG;
    if (n > (1l << 31) - 8 || vocab > (1 << 30)) return OF_E_SHAPE;
    EmbArgs a{};
    a.ids = ids; a.n = n; a.vocab = vocab; a.d = d; a.table = table; a.ldt = ldt; a.f32 = f32; a.scale = scale; a.y = y; a.ldy = ldy;
    a.vec = emb_vec(table, ldt, d, f32) && emb_vec(y, ldy, d, f32);
    return of_launch(emb_fwd_kernel, of_dim3{(unsigned)((n + 3) / 4), 1, 1}, 256, 0, (of_stream_t)stream, a);
}

extern "C" size_t of_embedding_bwd_workspace_bytes(long n, int vocab, int d) {
    if (n <= FEW || vocab <= 0 || d <= 0) return 0;
    const long nb = (n + TILE - 1) / TILE, chunks = (n + emb_chunk(n) - 1) / emb_chunk(n);
    return 4 * up256((size_t)n * 4) + up256((size_t)BINS * nb * 4) + up256((size_t)chunks * 2 * d * 4);
}

extern "C" int of_embedding_bwd(const long long* ids, long n, const void* dy, int f32, long lddy, int vocab, int d, float scale, long long padding_idx,
                                void* dw, long lddw, void* workspace, size_t workspace_bytes, void* stream) {
    if (!ids || !dy || !dw || (!workspace && n > FEW) || n <= 0 || vocab <= 0 || d <= 0 || lddy < d || lddw < d || !emb_dtype_ok(f32)) return OF_E_ARG;
    if (n > (1l << 31) - 2 * TILE || vocab > (1 << 30)) return OF_E_SHAPE;
    if ((uintptr_t)workspace & 15) return OF_E_ALIGN;
    if (workspace_bytes < of_embedding_bwd_workspace_bytes(n, vocab, d)) return OF_E_WORKSPACE;
    of_stream_t s = (of_stream_t)stream;
    EmbArgs a{};
    a.ids = ids; a.n = n; a.vocab = vocab; a.d = d; a.padding_idx = padding_idx; a.f32 = f32; a.scale = scale;
    a.dy = dy; a.lddy = lddy; a.dw = dw; a.lddw = lddw;
    a.vec = emb_vec(dy, lddy, d, f32) && emb_vec(dw, lddw, d, f32);
    if (n > FEW) {
        char* ws = (char*)workspace;
        auto take = [&](size_t bytes) {
            char* p = ws;
            ws += up256(bytes);
            return p;
        };
        unsigned* key[2];
        unsigned* pos[2];
        for (int i = 0; i < 2; ++i) {
            key[i] = (unsigned*)take((size_t)n * 4);
            pos[i] = (unsigned*)take((size_t)n * 4);
        }
        a.nb = (int)((n + TILE - 1) / TILE);
        a.hist = (int*)take((size_t)BINS * a.nb * 4);
        a.chunk = emb_chunk(n);
        a.chunks = (n + a.chunk - 1) / a.chunk;
        a.part = (float*)take((size_t)a.chunks * 2 * d * 4);
        a.passes = emb_passes(vocab);
        const int fill = vocab < 2048 ? vocab : 2048;
        int rc, in = 0;
        if (emb_small(n, vocab)) {
            a.key_out = key[0]; a.pos_out = pos[0];
            a.cap = (int)(n + 63) / 64 * 64;
            const size_t lds = 2 * (size_t)a.cap * 4 + SMALL_WAVES * BINS * 2 + BINS * 4;
            // 256 workgroups sweep the table in windows of 4 MB: the gradient of 65 positions of a 766-MB table takes 139 us (a fill alone 113);
            // 255, 511 and 1022 of them, whose windows do not end at a power of two, take 167, 156 and 169, 512 (two to a compute unit) 159
            rc = of_launch(emb_sort_small_kernel, of_dim3{(unsigned)(1 + (fill < 256 ? fill : 256)), 1, 1}, SMALL_THREADS, lds, s, a);
            if (rc) return rc;
        } else {
            for (int p = 0; p < a.passes; ++p) {
                const int out = p & 1;
                in = out ^ 1;
                a.key_in = key[in]; a.pos_in = pos[in]; a.key_out = key[out]; a.pos_out = pos[out];
                a.shift = p * RB;
                a.from_ids = p == 0;
                rc = of_launch(emb_count_kernel, of_dim3{(unsigned)(a.nb + (p == 0 ? fill : 0)), 1, 1}, TILE_THREADS, BINS * sizeof(int), s, a);
                if (rc) return rc;
                if (a.nb > SCAN_TILES) rc = of_launch(emb_scan_kernel, of_dim3{1, 1, 1}, BINS, BINS * sizeof(int), s, a);
                if (rc) return rc;
                rc = of_launch(emb_place_kernel, of_dim3{(unsigned)a.nb, 1, 1}, TILE_THREADS, (TILE_WAVES + 1) * BINS * sizeof(int), s, a);
                if (rc) return rc;
                in = out;
            }
        }
        a.key = key[in]; a.pos = pos[in];
    }
    if (f32) return a.vec ? emb_sums<true, true>(a, s) : emb_sums<true, false>(a, s);
    return a.vec ? emb_sums<false, true>(a, s) : emb_sums<false, false>(a, s);
}
