// AdamW over many tensors at once (gfx950, HBM-bound), moments in fp32 or in 8 bits; the clip by the global norm is part of the step.
//   g' = g min(1, max_norm / (|g| + 1e-6));   m = b1 m + (1 - b1) g';   v = b2 v + (1 - b2) g'^2
//   p  = p (1 - lr wd) - lr / (1 - b1^t)  m / (sqrt(v / (1 - b2^t)) + eps)
// An element costs 28 bytes of traffic with fp32 moments and gradients, 16 with 8-bit moments, and 4 more for the norm.  One launch takes
// up to 48 tensors (their pointers travel in the kernel arguments: nothing to keep in step on the device, safe to capture); a
// workgroup takes 4096 elements of one tensor.  Measured (160 tensors, 120 million elements, fp32 gradients, with the clip): 760 us with fp32
// moments = 3.84 GB at 5.05 TB/s, a large copy's rate (update 620, norm 125 us); 492 us with 8-bit moments = 2.40 GB at 4.9 TB/s.
//
// 8-bit moments: e4m3 codes with one fp32 scale (largest magnitude / 448) per 256 consecutive elements of a tensor.
//   * The first moment is rounded to the nearest code: it moves by a tenth of its distance to g' every step, and stands still where that is
//     less than half a code (1/32 ... 1/16 of it), i.e. within 0.3 ... 0.6 of it from g'.
//   * The second moment is held as its square root, which halves the range of exponents a code has to cover.  It moves by a thousandth
//     (b2 = 0.999) of its distance to g'^2 a step, far less than half a code: rounded to the nearest it would stand still.  It is rounded up
//     or down at random in proportion, so that the ROOT's expectation is the unrounded one's (the second moment itself gains the rounding's
//     variance); the 20 random bits are a hash of (tensor, element, step): the same call gives the same bits.  From above zero it never goes
//     to zero (m / (0 + eps) would explode).
//   * What that comes to beside 32 bits, 1000 to 20000 steps of noisy gradients of a fixed mean (8192 elements, b = 0.9, 0.999): the second
//     moment 3 to 7 % high, its root between -24 % and +31 % (5th to 95th percentile), the first moment 4 to 5 % off (rms); the sum of the
//     updates has a cosine of 0.994 and more with that of 32 bits and is 1 % longer.  None of it grows with the steps.
//   * The parameter's own update uses the moments in fp32, before they are rounded.
#include "of_platform.h"
#include "../../include/of_hip.h"

namespace {

constexpr int MT_MAX = 48;                  // tensors per launch: 48 x 72 bytes of descriptors in the kernel arguments
constexpr int MT_CHUNK = 4096;              // elements per workgroup = 16 blocks of 256, four for each wave
constexpr int MT_PARTS = 1024;              // partial sums of squares per launch of the norm
constexpr int BLOCK = OF_ADAMW_BLOCK;

struct MtTensor {
    float* p; const void* g; void* m; void* v; float* ms; float* vs;
    long n;
    float lr, wd;
    int flags;                              // 1: bf16 gradient, 2: all pointers aligned for four elements at a time
    int ordinal;
};
// what the step's launches share, on the device
struct MtStep {
    float coef;                             // gradient factor of the clip; negative: a squared norm that is not finite, the step is left out
    float inv_sqrt_bc2, inv_bc1;
    int t;
};
struct MtArgs {
    int n;
    int chunk_end[MT_MAX];                  // cumulative chunks
    float beta1, omb1, beta2, omb2, eps;
    MtStep* step;
    MtTensor t[MT_MAX];
};
constexpr int MT_NORM_CHUNK = 8192;
constexpr int MT_NORM_MAX = 196;            // the norm needs less of a tensor: more of them per launch
struct MtNormArgs {
    int n;
    int chunk_end[MT_NORM_MAX];
    double* parts;
    unsigned long long g[MT_NORM_MAX];      // address, plus 1 for bf16
    long count[MT_NORM_MAX];
};
static_assert(sizeof(MtArgs) <= 4096 && sizeof(MtNormArgs) <= 4096, "kernel arguments");
struct MtBeginArgs {
    const double* parts; long count;
    float max_norm; double beta1, beta2;
    int step; int* applied;
    MtStep* out; float* sumsq;
};

// the tensor a chunk belongs to (branches are uniform; the table sits in the kernel arguments)
OF_DEV int mt_find(const MtArgs& a, int chunk, int& first) {
    int lo = 0, hi = a.n - 1;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (chunk < a.chunk_end[mid]) hi = mid;
        else lo = mid + 1;
    }
    lo = of_uniform(lo);
    first = lo ? a.chunk_end[lo - 1] : 0;
    return lo;
}

// four elements at i of a float / bf16 array; zeros behind n
OF_DEV f32x4 mt_load(const void* base, int bf16, bool vec, long i, long n) {
    f32x4 r = {0.f, 0.f, 0.f, 0.f};
    if (vec && i + 4 <= n) {
        if (!bf16) return *(const f32x4*)((const float*)base + i);
        const u32x2 u = *(const u32x2*)((const bf16_t*)base + i);
        return f32x4{of_bf16_to_f32((bf16_t)(u[0] & 0xffff)), of_bf16_to_f32((bf16_t)(u[0] >> 16)), of_bf16_to_f32((bf16_t)(u[1] & 0xffff)),
                     of_bf16_to_f32((bf16_t)(u[1] >> 16))};
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (i + e < n) r[e] = bf16 ? of_bf16_to_f32(((const bf16_t*)base)[i + e]) : ((const float*)base)[i + e];
    return r;
}
OF_DEV void mt_store(float* base, bool vec, long i, long n, f32x4 x) {
    if (vec && i + 4 <= n) {
        *(f32x4*)(base + i) = x;
        return;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (i + e < n) base[i + e] = x[e];
}
OF_DEV unsigned mt_load_codes(const void* base, bool vec, long i, long n) {
    if (vec && i + 4 <= n) return *(const unsigned*)((const unsigned char*)base + i);
    unsigned u = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (i + e < n) u |= (unsigned)((const unsigned char*)base)[i + e] << (8 * e);
    return u;
}
OF_DEV void mt_store_codes(void* base, bool vec, long i, long n, unsigned u) {
    if (vec && i + 4 <= n) {
        *(unsigned*)((unsigned char*)base + i) = u;
        return;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (i + e < n) ((unsigned char*)base)[i + e] = (unsigned char)(u >> (8 * e));
}

// ------------------------------------------------------------------------------------------------ the norm
// 256 lanes' values in a fixed order, the result in thread 0
OF_DEV double mt_sum64(double s, double* red, int tid) {
    red[tid] = s;
    of_sync();
    for (int o = 128; o >= 1; o >>= 1) {
        if (tid < o) red[tid] += red[tid + o];
        of_sync();
    }
    return red[0];
}
// The sum of squares in 64 bits: the pass waits for memory, and the clip factor then does not depend on how the elements are cut into
// workgroups (8-bit moments make a rounding of the factor visible: one code in a few million).
// Workgroup b of MT_PARTS takes chunks b, b + MT_PARTS, ... (32 KB each: the grid as a whole walks memory front to back -- with a long run of
// its own for every workgroup the same pass read 3.6 TB/s); which slot sums which elements depends on the sizes alone
OF_GLOBAL void OF_BOUNDS(256, 4) mt_sumsq_kernel(MtNormArgs a) {
    double* red = (double*)of_smem();
    const int tid = of_tid(), all = a.chunk_end[a.n - 1];
    int k = 0;
    double s = 0.0, s2 = 0.0;
    for (int c = of_bid_x(); c < all; c += MT_PARTS) {
        while (a.chunk_end[k] <= c) ++k;
        const unsigned long long at = a.g[k];
        const int bf16 = (int)(at & 1);          // (gradients are at even addresses: the lowest bit tells the type)
        const void* g0 = (const void*)(at & ~1ull);
        const bool vec = !(at & (bf16 ? 6 : 14));
        const long i = (long)(c - (k ? a.chunk_end[k - 1] : 0)) * MT_NORM_CHUNK + tid * 4, n = a.count[k];
        f32x4 g[8];          // eight loads of a lane in flight
#pragma unroll
        for (int u = 0; u < 8; ++u) g[u] = mt_load(g0, bf16, vec, i + u * 1024, n);
#pragma unroll
        for (int u = 0; u < 8; u += 2)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const double x = (double)g[u][e], y = (double)g[u + 1][e];
                s = __builtin_fma(x, x, s);
                s2 = __builtin_fma(y, y, s2);
            }
    }
    s = mt_sum64(s + s2, red, tid);
    if (tid == 0) a.parts[of_bid_x()] = s;
}

// one workgroup: the partial sums in a fixed order, then everything a step needs once -- bias corrections in 64 bits (1 - 0.999^t loses
// four digits in 32 at small t).  `applied` counts the steps that were not left out.
OF_GLOBAL void OF_BOUNDS(256, 1) mt_begin_kernel(MtBeginArgs a) {
    double* red = (double*)of_smem();
    const int tid = of_tid();
    double s = 0.0;
    for (long i = tid; i < a.count; i += 256) s += a.parts[i];
    s = mt_sum64(s, red, tid);
    if (tid == 0) {
        const float sum = (float)s, norm = (float)sqrt(s);
        // the SQUARED norm has to be an fp32 value: no element's second moment then leaves the range (one that did would make its block's
        // scale infinite, and with it every 8-bit code of the block NaN), and the caller sees from *sumsq that the step was left out
        const bool finite = sum < 3.0e38f;
        *a.sumsq = sum;
        int t = a.step;
        if (a.applied) {
            t = *a.applied + 1;
            if (finite) *a.applied = t;
        }
        float coef = a.max_norm > 0.f ? 1.0f / (norm + 1e-6f) * a.max_norm : 1.0f;
        if (!(coef < 1.0f)) coef = 1.0f;
        a.out->coef = finite ? coef : -1.0f;
        a.out->t = t;
        a.out->inv_bc1 = (float)(1.0 / (1.0 - pow(a.beta1, (double)t)));
        a.out->inv_sqrt_bc2 = (float)(1.0 / sqrt(1.0 - pow(a.beta2, (double)t)));
    }
}

// ------------------------------------------------------------------------------------------------ the update
// 20 random bits of (tensor, element, step): multiplications by odd constants and shifts, every input bit reaches every output bit
OF_DEV unsigned mt_random20(unsigned key, long i) {
    unsigned x = ((unsigned)i ^ key) * 0x9E3779B1u;
    x = (x ^ (x >> 15)) * 0x85157AF5u;
    x = (x ^ (x >> 13)) * 0x9E3779B1u;
    return (x ^ (x >> 16)) & 0xFFFFFu;
}
// q in [0, 448] to a neighbouring e4m3 value, the upper one with the probability of q's place between the two (u: 20 random bits);
// above zero stays above zero
OF_DEV float mt_round_random(float q, unsigned u) {
    // from 2^-6, the smallest normal value, 20 of the 23 mantissa bits go; below, values are 2^-9 apart
    const float n = of_min(__builtin_bit_cast(float, (__builtin_bit_cast(unsigned, q) + u) & 0xFFF00000u), 448.0f);
    const float d = of_max(floorf(q * 512.0f + (float)u * 0x1p-20f) * (1.0f / 512.0f), 1.0f / 512.0f);
    return q >= 0.015625f ? n : q > 0.f ? d : 0.f;
}

struct MtHyper {
    float coef, step_size, inv_sqrt_bc2, decay, beta1, omb1, beta2, omb2, eps;
};
// r receives the square root of the second moment.  Moments, root and everything that 8-bit codes are made of take one IEEE rounding per
// written operation, in this order: where a value lies between two codes then does not depend on how the compiler joins operations.
// The parameter's update goes into no later step: a 1-ulp reciprocal there (2e-7 of an update) saves its division.
OF_DEV void mt_update(const MtHyper& h, f32x4& p, f32x4 g, f32x4& m, f32x4& v, f32x4& r) {
#pragma clang fp contract(off)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float ge = g[e] * h.coef;
        m[e] = m[e] * h.beta1 + ge * h.omb1;
        v[e] = v[e] * h.beta2 + ge * h.omb2 * ge;
        r[e] = sqrtf(v[e]);
        p[e] = p[e] * h.decay - h.step_size * (m[e] * of_rcp(r[e] * h.inv_sqrt_bc2 + h.eps));
    }
}

template <int BITS>
OF_GLOBAL void OF_BOUNDS(256, 4) mt_adamw_kernel(MtArgs a) {
    const MtStep st = *a.step;
    if (st.coef < 0.f) return;
    int first;
    const MtTensor& t = a.t[mt_find(a, of_bid_x(), first)];
    const int tid = of_tid(), lane = tid & 63, wave = tid >> 6, bf16 = t.flags & 1;
    const bool vec = t.flags & 2;
    const long n = t.n, base = (long)(of_bid_x() - first) * MT_CHUNK + wave * (4 * BLOCK) + lane * 4;
    const MtHyper h{st.coef, t.lr * st.inv_bc1, st.inv_sqrt_bc2, 1.0f - t.lr * t.wd, a.beta1, a.omb1, a.beta2, a.omb2, a.eps};
    f32x4 p[4], g[4], m[4], v[4];
    unsigned mc[4], vc[4];
    float ms[4], vs[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        const long i = base + u * BLOCK;
        p[u] = mt_load(t.p, 0, vec, i, n);
        g[u] = mt_load(t.g, bf16, vec, i, n);
        if (BITS == 32) {
            m[u] = mt_load(t.m, 0, vec, i, n);
            v[u] = mt_load(t.v, 0, vec, i, n);
        } else {
            mc[u] = mt_load_codes(t.m, vec, i, n);
            vc[u] = mt_load_codes(t.v, vec, i, n);
            const long b = i / BLOCK;           // the wave's block
            ms[u] = i - lane * 4 < n ? t.ms[b] : 0.f;
            vs[u] = i - lane * 4 < n ? t.vs[b] : 0.f;
        }
    }
    const unsigned key = (unsigned)st.t * 0x9E3779B1u + (unsigned)t.ordinal * 0x85157AF5u;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        const long i = base + u * BLOCK;
        if (BITS == 32) {
            f32x4 r;
            mt_update(h, p[u], g[u], m[u], v[u], r);
            mt_store(t.p, vec, i, n, p[u]);
            mt_store((float*)t.m, vec, i, n, m[u]);
            mt_store((float*)t.v, vec, i, n, v[u]);
        } else {
            m[u] = of_fp8x4_to_f32(mc[u]);
            v[u] = of_fp8x4_to_f32(vc[u]);
            float tm = 0.f, tr = 0.f;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                m[u][e] *= ms[u];
                v[u][e] *= vs[u];
                v[u][e] *= v[u][e];
            }
            f32x4 r;
            mt_update(h, p[u], g[u], m[u], v[u], r);
            mt_store(t.p, vec, i, n, p[u]);
            if (i + 4 > n) {          // behind the tensor's end: zeros, which no block's largest is
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (i + e >= n) m[u][e] = r[e] = 0.f;
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                tm = of_max(tm, __builtin_fabsf(m[u][e]));
                tr = of_max(tr, r[e]);
            }
            tm = of_wave_max(tm);
            tr = of_wave_max(tr);
            const float im = 1.0f / of_max(tm, 1e-30f) * 448.0f, ir = 1.0f / of_max(tr, 1e-30f) * 448.0f;          // (IEEE: once a block)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                m[u][e] = of_max(of_min(m[u][e] * im, 448.0f), -448.0f);
                r[e] = mt_round_random(of_min(r[e] * ir, 448.0f), mt_random20(key, i + e));
            }
            mt_store_codes(t.m, vec, i, n, of_f32_to_fp8x4(m[u]));
            mt_store_codes(t.v, vec, i, n, of_f32_to_fp8x4(r));
            if (lane == 0 && i < n) {
                t.ms[i / BLOCK] = tm * (1.0f / 448.0f);
                t.vs[i / BLOCK] = tr * (1.0f / 448.0f);
            }
        }
    }
}

int mt_launches(int n, int per) { return (n + per - 1) / per; }
size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }
}  // namespace

extern "C" size_t of_adamw_multi_workspace_bytes(int n) { return n > 0 ? up256(sizeof(MtStep)) + (size_t)mt_launches(n, MT_NORM_MAX) * MT_PARTS * sizeof(double) : 0; }

extern "C" int of_adamw_multi(const OfAdamwTensor* tensors, int n, int bits, double beta1, double beta2, double eps, double max_norm, int step, int* applied_steps,
                              float* sumsq, void* workspace, size_t workspace_bytes, void* stream) {
    if (!tensors || n <= 0 || (bits != 8 && bits != 32) || !sumsq || !workspace || (step <= 0 && !applied_steps)) return OF_E_ARG;
    if (!(beta1 >= 0.0 && beta1 < 1.0) || !(beta2 >= 0.0 && beta2 < 1.0) || !(eps >= 0.0)) return OF_E_ARG;
    if (workspace_bytes < of_adamw_multi_workspace_bytes(n)) return OF_E_WORKSPACE;
    if ((uintptr_t)workspace & 15) return OF_E_ALIGN;
    for (int i = 0; i < n; ++i) {
        const OfAdamwTensor& t = tensors[i];
        if (!t.p || !t.g || !t.m || !t.v || t.n <= 0 || (bits == 8 && (!t.m_scale || !t.v_scale))) return OF_E_ARG;
        if (((uintptr_t)t.p & 3) || ((uintptr_t)t.g & (t.g_bf16 ? 1 : 3)) || (bits == 32 && (((uintptr_t)t.m & 3) || ((uintptr_t)t.v & 3))) || ((uintptr_t)t.m_scale & 3) || ((uintptr_t)t.v_scale & 3))
            return OF_E_ALIGN;
        if (t.n > (long)MT_CHUNK << 24) return OF_E_SHAPE;      // 2^36 elements of one tensor
    }
    of_stream_t s = (of_stream_t)stream;
    MtStep* st = (MtStep*)workspace;
    double* parts = (double*)((char*)workspace + up256(sizeof(MtStep)));
    const int launches = mt_launches(n, MT_MAX), norms = mt_launches(n, MT_NORM_MAX);
    auto chunks = [](long elements, int chunk) { return (elements + chunk - 1) / chunk; };
    auto pack = [&](int l, MtArgs& a) {
        a = MtArgs{};
        long end = 0;
        for (int i = l * MT_MAX; i < n && i < (l + 1) * MT_MAX; ++i) {
            const OfAdamwTensor& t = tensors[i];
            MtTensor& d = a.t[a.n];
            d.p = t.p; d.g = t.g; d.m = t.m; d.v = t.v; d.ms = t.m_scale; d.vs = t.v_scale; d.n = t.n; d.lr = t.lr; d.wd = t.weight_decay;
            const uintptr_t wide = (uintptr_t)t.p | (t.g_bf16 ? (uintptr_t)t.g << 1 : (uintptr_t)t.g);
            const uintptr_t state = (uintptr_t)t.m | (uintptr_t)t.v;
            d.flags = (t.g_bf16 ? 1 : 0) | (!(wide & 15) && !(state & (bits == 32 ? 15 : 3)) ? 2 : 0);
            d.ordinal = i;
            end += chunks(t.n, MT_CHUNK);
            a.chunk_end[a.n++] = (int)end;
        }
        a.beta1 = (float)beta1; a.omb1 = (float)(1.0 - beta1); a.beta2 = (float)beta2; a.omb2 = (float)(1.0 - beta2); a.eps = (float)eps;
        a.step = st;
        return end;
    };
    long most = 0;
    for (int l = 0; l < norms; ++l) {
        long end = 0;
        for (int i = l * MT_NORM_MAX; i < n && i < (l + 1) * MT_NORM_MAX; ++i) end += chunks(tensors[i].n, MT_CHUNK);
        if (end > most) most = end;
    }
    if (most >= 1l << 31) return OF_E_SHAPE;          // (the updates' launches hold fewer tensors)
    int rc = 0;
    for (int l = 0; l < norms && !rc; ++l) {
        MtNormArgs a{};
        long end = 0;
        for (int i = l * MT_NORM_MAX; i < n && i < (l + 1) * MT_NORM_MAX; ++i) {
            end += chunks(tensors[i].n, MT_NORM_CHUNK);
            a.g[a.n] = (unsigned long long)(uintptr_t)tensors[i].g | (tensors[i].g_bf16 ? 1 : 0);
            a.count[a.n] = tensors[i].n;
            a.chunk_end[a.n++] = (int)end;
        }
        a.parts = parts + (size_t)l * MT_PARTS;
        rc = of_launch(mt_sumsq_kernel, of_dim3{MT_PARTS, 1, 1}, 256, 256 * sizeof(double), s, a);
    }
    if (rc) return rc;
    const MtBeginArgs b{parts, (long)norms * MT_PARTS, (float)max_norm, beta1, beta2, step, applied_steps, st, sumsq};
    rc = of_launch(mt_begin_kernel, of_dim3{1, 1, 1}, 256, 256 * sizeof(double), s, b);
    // last tensors first: the norm's launch read their gradients last, up to 256 MB of them are still in the Infinity Cache
    for (int l = launches - 1; l >= 0 && !rc; --l) {
        MtArgs a;
        const unsigned grid = (unsigned)pack(l, a);
        rc = bits == 8 ? of_launch(mt_adamw_kernel<8>, of_dim3{grid, 1, 1}, 256, 0, s, a) : of_launch(mt_adamw_kernel<32>, of_dim3{grid, 1, 1}, 256, 0, s, a);
    }
    return rc;
}
