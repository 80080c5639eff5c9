// s2k_kv8_attn.cu -- attention of few query rows over the 8-bit paged KV cache
// (decode steps, drafted tokens, short prompts); s2k_kv8_prompt.cu has the rest.
//
//   o = sum_j w_j v_j,  w = softmax over the visible keys of scale * q.k_j
// Row i of a sequence sits at position p = past + i and sees key j iff
//   j <= p  and  (window == 0  or  j > p - window  or  j < sinks).
// A row that sees nothing (a sequence whose pages are all bad) is zero.
//
// Bound by the cache's bytes: 2 * head_dim bytes per key and kv head, read
// once for a tile of slots, a slot being one (row, query head) pair of the kv
// head.  At HBM's rate a page (16 keys, 4 KB at head_dim 128) leaves an SM ~700
// issue slots, which FMAs on 4 query heads (512 per lane and page with the
// conversions) do not fit.  So the products run on the tensor cores, and on
// integers: the cache is int8, and a query or a weight is written in digits of
// base 256, each a row of the left operand of mma.sync m16n8k32.
//   S = Q K^T  rows: the digits of the slots' queries, columns: keys
//   O = P V    rows: the digits of the slots' weights, columns: dimensions
// 16 rows are 4 slots of 4 digits (30 bits: f32's accuracy), or for f16 and bf16
// rows of which there are more 8 slots of 2 digits: weights have 15 bits of the
// largest one, queries 30 bits of the row's largest element in two products (a
// few large dimensions must not cost the others their bits; with one product a
// score was off by up to 2^-16 * max|q| * sum |k|, and 8 slots took 7 to 12 %
// less time).  Keys and values go from shared memory into the products as they
// are, and the integer sums are exact.  The same kernel with
// f16 products (int8 -> f16, halves of q and p) took 573 instructions per page
// and warp, this one ~220; mma.sync does int8 at twice the rate of f16 (both 2
// cycles per instruction and SM, measured).  tcgen05 has 128 rows: 16 of them
// would be used, and its operands would need a pass through shared memory.
//
// Weights are taken relative to the largest of two pages (32 keys) with the
// blocks' value scales in them: digits of p * v_scale / W, W the pages' largest
// such product.  The f32 factors (W, the running maximum) multiply the sums,
// which are in units of a power of two, that of the largest value scale that the
// warp met: scales may be anything that f32 holds, and no sum passes it on the
// way.  A product below 2^-90 of that unit has fewer bits.
//
// The order of dimensions within a product is free as long as both operands
// agree.  Lane (i, c) = (lane / 4, lane % 4) takes dims 16c .. 16c+15 (and 64
// more for head_dim 128) of a key as 16-byte words, and tokens 4c .. 4c+3 of a
// value's dimension as one 4-byte word; the keys' columns are ordered so that
// the weights leave S in the lane that needs them for P.
//
// One warp walks its own pairs of pages through its own ring of 16-byte
// asynchronous copies with a running maximum, sum and output; no barrier inside
// the loop.  The pages of a (tile, kv head, sequence) are split over the CTAs of
// a cluster when there are few of them, and joined through distributed shared
// memory: no workspace, one launch, and the same order of sums every time.
#include "s2k_common.cuh"
#include "s2k_kv8.h"

#include <algorithm>
#include <atomic>

namespace s2k {

// Three CTAs of four warps per SM: a warp's step (a pair of pages) is a chain
// of ~2000 cycles, so it takes twelve of them to keep HBM busy.  16 KB of pages
// in flight per warp.  Twelve warps in one CTA per SM were as fast or slower
// (a CTA's start is then hidden by no other) but for one sequence of 32768
// tokens (22.6 against 24.7 us when it was compared), which cannot fill the
// machine from clusters.  Now, with the call and cold caches: 64 bf16 sequences
// of up to 2523 tokens 43.7 us (4.25 TB/s), one of 32768 26.6 us, one of 512
// 13.5 us.
constexpr int kDWarps = 4;
constexpr int kDThreads = kDWarps * 32;
template <int HD>
constexpr int kDStages = HD == 128 ? 2 : 4;
// D = A B + D, or + kMagic's bits: int8 digits, int32 sums.  Not volatile: the
// order among them is the compiler's.
__device__ __forceinline__ void imma(int (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void imma0(int (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "r"(0x4b400000));
}

// Integers below 2^22 as f32 and back by adding 1.5 * 2^23, whose low mantissa
// bits then are the integer: conversions run at a quarter of an addition's
// rate and took a third of the loop.
constexpr float kMagic = 12582912.f;

// How the 16 rows of a product are shared out.  Rows i and i + 8 are the upper
// and lower digit of one 16-bit integer.  4 slots (wide): rows i < 4 hold the
// high part h and rows i >= 4 the low part of x = h * 2^15 + low, |h| <= 32512,
// |low| <= 2^14, of slot i % 4.  8 slots: a row per slot i, weights x = h; the
// queries' low parts are in a second product.
constexpr float kHigh = 32768.f;  // what an upper part's unit is worth
// the largest integers written: digits in [-128, 127] reach 127 * 257
constexpr float kQUnit = 32512.f * kHigh;
constexpr float kQOne = 1073741824.f;  // 2^30, what the products with queries are divided by
// the upper or the lower part of round(x), |x| <= kQUnit, in the low 16 bits
__device__ __forceinline__ uint32_t split_part(float x, bool low) {
    const float h = fmaf(x, 1.f / kHigh, kMagic);
    return __float_as_uint(low ? fmaf(h - kMagic, -kHigh, x) + kMagic : h);
}
template <int SLOTS>
struct Digits {
    static constexpr bool wide = SLOTS == 4;
    static constexpr int slots = SLOTS;
    static constexpr float unit = wide ? 32512.f * kHigh : 32512.f;  // of the weights
    static __device__ __forceinline__ int slot(int i) { return i % slots; }
    // the lane's part of round(x), a weight's, in the low 16 bits
    static __device__ __forceinline__ uint32_t part(float x, bool low) {
        return wide ? split_part(x, low) : __float_as_uint(x + kMagic);
    }
    // Four parts -> the words of their upper and lower digits.  The digits of
    // n are the bytes of n + 0x8080, less 128 each.
    static __device__ __forceinline__ void words(const uint32_t (&n)[4], uint32_t &a, uint32_t &b) {
        const uint32_t s = __byte_perm(n[0] + 0x8080u, n[1] + 0x8080u, 0x4051);  // (upper, upper, lower, lower)
        const uint32_t t = __byte_perm(n[2] + 0x8080u, n[3] + 0x8080u, 0x4051);
        a = __byte_perm(s, t, 0x5410) ^ 0x80808080u;
        b = __byte_perm(s, t, 0x7632) ^ 0x80808080u;
    }
};

template <int HD, int SLOTS>
struct DecodeSmem {
    static constexpr int kRow = HD + 8;  // eight rows' stores meet different banks
    union {
        alignas(128) int8_t ring[kDWarps][kDStages<HD>][2][2][kPage * HD];  // page of the pair, keys / values
        float o[kDWarps][SLOTS][kRow];                                      // after the loop: each warp's output
    };
    uint32_t q[SLOTS][4][HD / 4 + 4];  // digit words of the queries, upper first
    float qmul[SLOTS];
    float m[kDWarps][SLOTS], l[kDWarps][SLOTS];
    int unit[kDWarps];  // exponents of the outputs' units
    // what the cluster's CTAs send: their outputs for this CTA's share, (maximum, sum) and unit
    float4 from[SLOTS * HD / 4 + kMaxCluster];
    float2 ml[kMaxCluster][SLOTS];
    float un[kMaxCluster];
};

// Where byte x (16-byte aligned) of a page's keys lies in shared memory: rows
// of 128 bytes swap their halves in odd tokens, so that the 16-byte reads of
// two tokens' 64 bytes meet all banks.
template <int HD>
__device__ __forceinline__ int key_at(int x) {
    return HD == 128 ? x ^ ((x & 128) >> 1) : x;
}

// Powers of two by their exponents as f32 holds them (1 .. 254); 2^(a - b), a <= b, 0 from 2^-127 on.
__device__ __forceinline__ float pow2(int e) { return __int_as_float(e << 23); }
__device__ __forceinline__ float pow2_of(int a, int b) { return __int_as_float(max(127 + a - b, 0) << 23); }

template <int HD, int TYPE, int SLOTS>
__global__ void __launch_bounds__(kDThreads, 3)
    kv8_decode_kernel(Kv8 c, Kv8Rows r, Kv8Attn a, int cs, float inv_group, int vec) {
    using T = typename OType<TYPE>::T;
    using Dg = Digits<SLOTS>;
    constexpr int STAGES = kDStages<HD>;
    constexpr int KV = HD / 32;  // k steps of Q K^T
    constexpr int NU = HD / 8;   // column tiles of P V
    constexpr unsigned kAll = 0xffffffffu;
    extern __shared__ uint8_t raw[];
    auto &sm = *reinterpret_cast<DecodeSmem<HD, SLOTS> *>((reinterpret_cast<uintptr_t>(raw) + 127) & ~uintptr_t(127));
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, li = lane >> 2, lc = lane & 3;
    const int b = blockIdx.x / cs, rank = blockIdx.x - b * cs;  // clusters lie along x
    const int kvh = blockIdx.y, tile = blockIdx.z;
    const int G = a.n_heads / c.n_kv_heads;
    int row0, n, past;
    // the same for every CTA of the cluster: none is left waiting
    if (!kv8_seq(r, b, row0, n, past) || tile * SLOTS >= n * G) return;

    // the lane's slot; the quotient is exact below 2^20 slots
    auto row_of = [&](int slot) { return (int)(((float)slot + 0.5f) * inv_group); };
    const int nslots = min(SLOTS, n * G - tile * SLOTS);
    const int ls = Dg::slot(li);
    const int slot = tile * SLOTS + min(ls, nslots - 1);
    const int pos = past + row_of(slot);
    // the tile's positions, and the logical pages that one of them sees: sink
    // pages [0, ns), then window pages [fw, ...]
    const int pos_lo = past + row_of(tile * SLOTS), pos_hi = past + row_of(tile * SLOTS + nslots - 1);
    const int wlo = a.window ? max(pos_lo - a.window + 1, 0) : 0;
    const int fw = wlo / kPage;
    const int ns = min((int)(((long long)a.sinks + kPage - 1) / kPage), fw);
    const int total = ns + pos_hi / kPage - fw + 1;
    // this CTA's pages, in pairs; pair k of the warp is pages 2 * (warp + k * kDWarps) and the next
    const int pairs = (total + 1) / 2;
    const int each = pairs / cs, more = pairs - each * cs;  // the first `more` CTAs have one more
    const int first = each * rank + min(rank, more), last = first + each + (rank < more);
    const int mine = last - first > warp ? (last - first - warp + kDWarps - 1) / kDWarps : 0;
    if (cs > 1) cluster_arrive();  // this CTA runs: others may store into its shared memory
    // lanes 2k and 2k + 1 hold pair k of the warp's current 16 pairs, and of the next 16: the physical page, or -1,
    // and its first token, behind every position where there is no page
    constexpr int kNone = 0x7fffff00;
    int page, next, p0s, next_p0;
    auto page_of = [&](int k, int &pg, int &p0) {
        const int x = 2 * (first + warp + k * kDWarps) + (lane & 1);
        const bool in = k < mine && x < total;
        const int lg = x < ns ? x : x - ns + fw;
        pg = in ? kv8_page(c, r, b, lg) : -1;
        p0 = pg >= 0 ? lg * kPage : kNone;
    };
    page_of(lane >> 1, page, p0s);
    page_of(16 + (lane >> 1), next, next_p0);
    // pair k into its stage: every lane 16-byte pieces of both pages, one group per pair (empty behind the last)
    auto issue = [&](int k, int pg) {
        if (k < mine) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int p = __shfl_sync(kAll, pg, 2 * (k & 15) + e);
                if (p < 0) continue;
                const size_t at = c.block(p, kvh) * (kPage * HD) + lane * 16;
                int8_t *kd = sm.ring[warp][k % STAGES][e][0], *vd = sm.ring[warp][k % STAGES][e][1];
#pragma unroll
                for (int x = 0; x < HD / 32; ++x) {
                    cp16(kd + key_at<HD>(lane * 16 + x * 512), c.k + at + x * 512);
                    cp16(vd + lane * 16 + x * 512, c.v + at + x * 512);
                }
            }
        }
        cp_commit();
    };
#pragma unroll
    for (int k = 0; k < STAGES - 1; ++k) issue(k, page);

    // queries in digits, a warp a slot at a time: lane l dims [l * E, l * E + E)
    {
        constexpr int E = HD / 32;
        for (int sl = warp; sl < SLOTS; sl += kDWarps) {
            const int st = tile * SLOTS + min(sl, nslots - 1), row = row_of(st);
            float x[E];
            load_n<E>(reinterpret_cast<const T *>(a.q.p) + (long long)(row0 + row) * a.q.row_stride +
                          (long long)(kvh * G + st - row * G) * a.q.head_stride + lane * E,
                      vec, x);
            unsigned top = 0;
#pragma unroll
            for (int e = 0; e < E; ++e) top = max(top, __float_as_uint(x[e]) & 0x7fffffffu);
            top = __reduce_max_sync(kAll, top);
            // the row's largest element becomes kQUnit; far down, both sides by 2^64, exactly, so that the factor is finite
            const float pre = top < 0x20000000u ? 18446744073709551616.f : 1.f;  // below 2^-63
            const float amax = __uint_as_float(top);
            const float up = __fdiv_rn(kQUnit, fmaxf(amax * pre, 8.0779356694631609e-28f));  // a row of zeros: 2^-90
            // takes the scores, in units of 2^30, to base-2 logarithms
            if (lane == 0) sm.qmul[sl] = top >= 0x7f800000u ? NAN : a.scale * 1.44269504f * (amax * (kQOne / kQUnit));
            uint32_t v[4] = {}, w[4];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int e = 0; e < E; ++e) v[e] = split_part(x[e] * pre * up, h);
                Dg::words(v, w[2 * h], w[2 * h + 1]);
            }
#pragma unroll
            for (int d = 0; d < 4; ++d) {
                if (E == 4) sm.q[sl][d][lane] = w[d];
                else reinterpret_cast<uint16_t *>(sm.q[sl][d])[lane] = (uint16_t)w[d];
            }
        }
    }
    __syncthreads();
    uint32_t q[KV][4];
    const float smul = sm.qmul[ls];
    // the queries' digits d0 and d0 + 1 as k steps' left operands
    auto load_q = [&](uint32_t (&t)[KV][4], int d0) {
#pragma unroll
        for (int j = 0; j < KV / 2; ++j)
#pragma unroll
            for (int d = 0; d < 2; ++d) {
                const uint4 w = *reinterpret_cast<const uint4 *>(&sm.q[ls][d0 + d][16 * j + 4 * lc]);
                t[2 * j][d] = w.x;
                t[2 * j][2 + d] = w.y;
                t[2 * j + 1][d] = w.z;
                t[2 * j + 1][2 + d] = w.w;
            }
    };
    load_q(q, Dg::wide && li >= 4 ? 2 : 0);
    uint32_t q2[KV][4];
    if (!Dg::wide) load_q(q2, 2);
    float m = -INFINITY, l = 0.f;  // l: this lane's tokens only
    float o[NU][2];
#pragma unroll
    for (int u = 0; u < NU; ++u) o[u][0] = o[u][1] = 0.f;
    float ks = 0.f, vs = 0.f;
    int unit = 1;      // o is in units of 2^(unit - 127): the exponent of the largest value scale met, as f32 holds it
    float grow = 1.f;  // and is to be multiplied by this
    for (int k = 0; k < mine; ++k) {
        if (k % 16 == 0) {
            if (k) {
                page = next;
                p0s = next_p0;
                page_of(k + 16 + (lane >> 1), next, next_p0);
            }
            ks = vs = 0.f;
            if (page >= 0) {  // wanted only once the page itself has come
                ks = c.k_scale[c.block(page, kvh)];
                vs = c.v_scale[c.block(page, kvh)];
            }
        }
        const int s = k % STAGES, from = 2 * (k & 15);
        __syncwarp();  // every lane has read the stage that comes next
        const int ahead = k + STAGES - 1;
        issue(ahead, (ahead >> 4) == (k >> 4) ? page : next);
        cp_wait<STAGES - 1>();
        __syncwarp();  // the pair has arrived for every lane
        // scores of the pair: x[4 e + t] is token 4 lc + t of page e
        float x[8], pm[2], f[2];
        int p0[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int8_t *kp = sm.ring[warp][s][e][0];
            const float pks = __shfl_sync(kAll, ks, from + e) * smul;
            p0[e] = __shfl_sync(kAll, p0s, from + e);
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                int acc[4], low[4];
                const int tok = 4 * (li >> 1) + 2 * t + (li & 1);
#pragma unroll
                for (int j = 0; j < KV / 2; ++j) {
                    const uint4 w = *reinterpret_cast<const uint4 *>(kp + key_at<HD>(tok * HD + 64 * j + 16 * lc));
                    if (j == 0) imma0(acc, q[0], w.x, w.y);
                    else imma(acc, q[2 * j], w.x, w.y);
                    imma(acc, q[2 * j + 1], w.z, w.w);
                    if (!Dg::wide) {
                        if (j == 0) imma0(low, q2[0], w.x, w.y);
                        else imma(low, q2[2 * j], w.x, w.y);
                        imma(low, q2[2 * j + 1], w.z, w.w);
                    }
                }
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    // digit by digit, the result in units of 2^30
                    auto two = [](int hi, int lo) {
                        return fmaf(__int_as_float(hi) - kMagic, 256.f / kQOne, fmaf(__int_as_float(lo), 1.f / kQOne, -kMagic / kQOne));
                    };
                    float y = two(acc[h], acc[2 + h]);
                    if (Dg::wide) {
                        const float other = __shfl_xor_sync(kAll, y, 16);
                        y = li < 4 ? fmaf(y, kHigh, other) : fmaf(other, kHigh, y);
                    } else {
                        y = fmaf(y, kHigh, two(low[h], low[2 + h]));
                    }
                    x[4 * e + 2 * t + h] = y * pks;
                }
            }
        }
        if (k % 16 == 0) {
            // the unit that these pairs' scales need, and they in it: below 2, but for the last powers (after the products:
            // the scales are still on their way before them)
            const int e = __float_as_int(vs) >> 23, most = max(min(__reduce_max_sync(kAll, e < 255 ? e : 0), 252), unit);
            grow = pow2_of(unit, most);
            unit = most;
            vs *= pow2(254 - unit);
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) f[e] = __shfl_sync(kAll, vs, from + e);
        // a page at the edge of what the slots see, or none
        const int p_lo = min(p0[0], p0[1]), p_hi = max(p0[0], p0[1]);
        if (p_hi + kPage - 1 > pos_lo || (a.window && p_lo <= pos_hi - a.window && p_hi + kPage > a.sinks)) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                if (!(p0[e] <= pos && (!a.window || p0[e] + kPage - 1 > pos - a.window || p0[e] < a.sinks)))
                    f[e] = 0.f;  // a hidden block's scale may be NaN
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    const int j = p0[e] + 4 * lc + t;
                    if (j > pos || (a.window && j <= pos - a.window && j >= a.sinks)) x[4 * e + t] = -INFINITY;
                }
            }
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            float t = fmaxf(fmaxf(x[4 * e], x[4 * e + 1]), fmaxf(x[4 * e + 2], x[4 * e + 3]));
            t = fmaxf(t, __shfl_xor_sync(kAll, t, 1));
            pm[e] = fmaxf(t, __shfl_xor_sync(kAll, t, 2));
        }
        const float both = fmaxf(pm[0], pm[1]);
        const float ref = both == -INFINITY ? 0.f : both;
        const float m2 = fmaxf(m, both);
        if (__any_sync(kAll, m2 > m || grow != 1.f)) {
            const float alpha = m == m2 ? 1.f : ex2(m - m2);  // 0 for the slot's first pair
            l *= alpha;
#pragma unroll
            for (int u = 0; u < NU; ++u) o[u][0] *= alpha * grow, o[u][1] *= alpha * grow;
            m = m2;
            grow = 1.f;
        }
        const float f0 = both == -INFINITY ? 0.f : ex2(ref - m2);
        float p[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) p[e] = ex2(x[e] - ref);
        l += f0 * (((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7])));
        // weights times value scales, relative to the pair's largest; a NaN scale has to reach the sum by `down`: integers
        // do not carry it
        const float W = fmaxf(fmaxf(ex2(pm[0] - ref) * f[0], ex2(pm[1] - ref) * f[1]), 8.0779356694631609e-28f);  // 2^-90
        const float up = __fdividef(Dg::unit, W);
        const float down = f0 * (W * (1.f / Dg::unit)) + 0.f * (f[0] + f[1]);
        const float mul = Dg::wide && li < 4 ? down * kHigh : down;
        uint32_t pa[4];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            uint32_t v[4];
            const float g = f[e] * up;
#pragma unroll
            for (int t = 0; t < 4; ++t) v[t] = Dg::part(p[4 * e + t] * g, li >= 4);
            Dg::words(v, pa[2 * e], pa[2 * e + 1]);
        }
        const int8_t *v0 = sm.ring[warp][s][0][1] + lane * 4, *v1 = sm.ring[warp][s][1][1] + lane * 4;
#pragma unroll
        for (int u = 0; u < NU; ++u) {
            int d[4];
            imma0(d, pa, *reinterpret_cast<const uint32_t *>(v0 + u * 128), *reinterpret_cast<const uint32_t *>(v1 + u * 128));
            float y[4] = {__int_as_float(d[0]), __int_as_float(d[1]), __int_as_float(d[2]), __int_as_float(d[3])};
            add2(y[0], y[1], -kMagic);
            add2(y[2], y[3], -kMagic);
            fma2(o[u], mul * 256.f, y[0], y[1]);
            fma2(o[u], mul, y[2], y[3]);
        }
    }
    l += __shfl_xor_sync(kAll, l, 1);
    l += __shfl_xor_sync(kAll, l, 2);
    if (Dg::wide) {  // upper and lower digits
#pragma unroll
        for (int u = 0; u < NU; ++u) {
            o[u][0] += __shfl_xor_sync(kAll, o[u][0], 16);
            o[u][1] += __shfl_xor_sync(kAll, o[u][1], 16);
        }
    }

    // join the warps, in order: outputs relative to the CTA's maximum
    if (li < SLOTS && lc == 0) sm.m[warp][ls] = m;
    if (lane == 0) sm.unit[warp] = unit;
    cp_wait<0>();
    __syncthreads();  // the maxima are there, and the ring is read
    float top = sm.m[0][ls];
    int most = sm.unit[0];
#pragma unroll
    for (int w = 1; w < kDWarps; ++w) top = fmaxf(top, sm.m[w][ls]), most = max(most, sm.unit[w]);
    const float g = m == -INFINITY ? 0.f : ex2(m - top), go = g * pow2_of(unit, most);
    if (li < SLOTS) {
#pragma unroll
        for (int u = 0; u < NU; ++u)
            *reinterpret_cast<float2 *>(&sm.o[warp][ls][8 * u + 2 * lc]) = make_float2(go * o[u][0], go * o[u][1]);
        if (lc == 0) sm.l[warp][ls] = g * l;  // NaN scores leave m at -inf and l NaN: 0 * NaN is NaN
    }
    __syncthreads();
    constexpr int kItems = SLOTS * HD / 4;  // of 4 dims; with a cluster each CTA joins a share of them
    const int share = (kItems + cs - 1) / cs;
    auto put = [&](int item, float sum, float4 v, float un) {
        const int st = tile * SLOTS + item / (HD / 4);
        if (item / (HD / 4) >= nslots) return;
        const int row = row_of(st);
        const float inv = sum == 0.f ? 0.f : __fdiv_rn(1.f, sum);
        const float y[4] = {v.x * inv * un, v.y * inv * un, v.z * inv * un, v.w * inv * un};
        store_n<4>(reinterpret_cast<T *>(a.out.p) + (long long)(row0 + row) * a.out.row_stride +
                       (long long)(kvh * G + st - row * G) * a.out.head_stride + item % (HD / 4) * 4,
                   vec, y);
    };
    if (cs > 1) cluster_wait();
    for (int item = tid; item < kItems; item += kDThreads) {
        const int sl = item / (HD / 4), d = item % (HD / 4) * 4;
        float4 v = *reinterpret_cast<const float4 *>(&sm.o[0][sl][d]);
        float sum = sm.l[0][sl];
#pragma unroll
        for (int w = 1; w < kDWarps; ++w) {
            const float4 t = *reinterpret_cast<const float4 *>(&sm.o[w][sl][d]);
            v = make_float4(v.x + t.x, v.y + t.y, v.z + t.z, v.w + t.w);
            sum += sm.l[w][sl];
        }
        if (cs == 1) put(item, sum, v, pow2(most));
        else {
            const int owner = item / share;
            st_cluster(in_cta(&sm.from[rank * share + item - owner * share], owner), v);
        }
    }
    if (cs == 1) return;
    for (int x = tid; x < SLOTS * cs; x += kDThreads) {
        const int sl = x % SLOTS;
        float mm = sm.m[0][sl], sum = sm.l[0][sl];
#pragma unroll
        for (int w = 1; w < kDWarps; ++w) mm = fmaxf(mm, sm.m[w][sl]), sum += sm.l[w][sl];
        st_cluster(in_cta(&sm.ml[rank][sl], x / SLOTS), mm, sum);
        if (sl == 0) st_cluster(in_cta(&sm.un[rank], x / SLOTS), pow2(most));
    }
    cluster_arrive();
    cluster_wait();  // from here no CTA reaches into another's shared memory
    for (int x = tid; x < min(share, kItems - rank * share); x += kDThreads) {
        const int item = rank * share + x, sl = item / (HD / 4);
        float mm = -INFINITY, sum = 0.f, un = 0.f;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (int k = 0; k < cs; ++k) mm = fmaxf(mm, sm.ml[k][sl].x), un = fmaxf(un, sm.un[k]);
#pragma unroll 4
        for (int k = 0; k < cs; ++k) {
            const float2 ml = sm.ml[k][sl];
            const float4 t = sm.from[k * share + x];
            const float gk = ml.x == -INFINITY ? 0.f : ex2(ml.x - mm);
            sum += gk * ml.y;
            const float go = gk * pow2_of(__float_as_int(sm.un[k]) >> 23, __float_as_int(un) >> 23);
            v = make_float4(v.x + go * t.x, v.y + go * t.y, v.z + go * t.z, v.w + go * t.w);
        }
        put(item, sum, v, un);
    }
}

// What a device allows, looked up once.
struct DecodeDevice {
    std::atomic<int> ready{0};
    int sms = 148;
};
static DecodeDevice g_decode[64];

thread_local int g_kv8_attend_kernel = 0;

template <int HD, int SLOTS>
static constexpr int decode_smem() {
    constexpr int n = (int)sizeof(DecodeSmem<HD, SLOTS>) + 128;
    static_assert(3 * (n + 1024) <= 228 * 1024, "three CTAs per SM");
    return n;
}

template <int HD, int TYPE, int SLOTS>
static cudaError_t decode_setup() {
    const auto f = kv8_decode_kernel<HD, TYPE, SLOTS>;
    cudaError_t e = cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, decode_smem<HD, SLOTS>());
    return e != cudaSuccess ? e : cudaFuncSetAttribute(f, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
}

template <int HD, int TYPE, int SLOTS>
static cudaError_t decode_launch(const Kv8 &c, const Kv8Rows &r, const Kv8Attn &a, int cs, int tiles,
                                 cudaStream_t st) {
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cs;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)r.n_seqs * cs, c.n_kv_heads, tiles);
    cfg.blockDim = dim3(kDThreads);
    cfg.dynamicSmemBytes = decode_smem<HD, SLOTS>();
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = cs > 1 ? 1 : 0;
    const float inv_group = 1.0f / (float)(a.n_heads / c.n_kv_heads);
    const int vec = rows_vec(a.q, 4) && rows_vec(a.out, 4);
    return cudaLaunchKernelEx(&cfg, kv8_decode_kernel<HD, TYPE, SLOTS>, c, r, a, cs, inv_group, vec);
}

cudaError_t launch_kv8_attend(const Kv8 &c, const Kv8Rows &r, const Kv8Attn &a, cudaStream_t st) {
    if (r.n_seqs == 0 || r.max_rows == 0) return cudaSuccess;
    const int G = a.n_heads / c.n_kv_heads;
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= 64) return cudaErrorInvalidDevice;
    DecodeDevice &d = g_decode[dev];
    if (!d.ready.load(std::memory_order_acquire)) {
        // idempotent: threads that meet here set the same values
        int sms = 0;
        if ((e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev))) return e;
        for (int hd : {64, 128})
            for (int type : {OT_F32, OT_F16, OT_BF16})
                if ((e = kv8_dispatch(hd, type, [&](auto h, auto t) {
                         cudaError_t e4 = decode_setup<h, t, 4>();
                         if constexpr (t != OT_F32)
                             if (e4 == cudaSuccess) e4 = decode_setup<h, t, 8>();
                         return e4;
                     })))
                    return e;
        d.sms = sms;
        d.ready.store(1, std::memory_order_release);
    }
    // tiles of `per` slots of a (sequence, kv head), and the pages that one of them sees at most
    auto tiles_of = [&](long long per) { return ((long long)r.max_rows * G + per - 1) / per; };
    auto pages_of = [&](long long per) {
        const long long rows = std::min<long long>(r.max_rows, per / G + 2);
        const long long seen = a.window ? ((long long)a.window + rows + a.sinks) / kPage + 3 : r.table_ld;
        return std::min<long long>(seen, r.table_ld);
    };
    // 16-bit rows: 8 slots a tile, but 4 where no sequence has more, with one product in place of two (4 query heads a kv
    // head: 64 bf16 sequences of up to 2523 tokens 43.2 us in fours, 46.5 in eights; one f16 of 32768 25.0 and 28.6)
    const bool four = a.q.type == OT_F32 || (long long)r.max_rows * G <= 4;
    const long long slots = four ? 4 : 8;
    const long long tiles = tiles_of(slots), pages = pages_of(slots);
    const long long groups = (long long)c.n_kv_heads * r.n_seqs, units = tiles * groups;
    // Which kernel.  Here every tile of 4 or 8 slots walks the pages, spread over the SMs: a page of a tile is the unit
    // of time, a tile's start about 30 of them.  The prompt kernel walks them once for 128 or 256 slots, one CTA per SM:
    // wave by wave a page takes 3 units, its start and end about 80 pages.  The wrong one is up
    // to 17 times slower (one f32 sequence of 16000 tokens, 64 slots, 8 heads: 104 us here, 275 there; 64 sequences of 2500:
    // 780 and 286; of 8 slots: 115 and 266; one of 100 with 64 slots: 4.5 and 12.7).  Over 920 calls of both kernels with
    // tables as wide as the longest sequence the choice is 0.3 % from the better one on average and 23 % at most.  Without
    // a window the table's width stands for the lengths, which the host does not know: 64 bf16 sequences of 100 tokens
    // take 9.0 us with a table of their width or 8 times that, 49 with one of 64 times, whose clusters find no pages; 8
    // f32 ones of 3000 14.5 and 28.7; a prompt of 60 f32 rows 7.4 and 24.7.
    const long long prompt_slots = kv8_prompt_slots(a.q.type);
    const long long waves = (tiles_of(prompt_slots) * groups + d.sms - 1) / d.sms;
    if (tiles > 65535 || (double)units * (pages + 30) > 3.0 * d.sms * waves * (pages_of(prompt_slots) + 80)) {
        g_kv8_attend_kernel = 2;
        return launch_kv8_prompt(c, r, a, st);
    }
    g_kv8_attend_kernel = 1;
    // CTAs per unit.  A CTA's start and its join cost about as much as 40 pages: pieces of about 64 pages are best
    // where the machine is full (64 sequences of up to 2523 tokens: 46 us whole, 43.6 halved, 48 in thirds; 8 of up
    // to 6095: 20.6 in fourths, 18.9 in sixths, 24.2 in sevenths; 16 of 4000 visible ones: 18.4 in thirds, 16.4 in
    // fourths, 22.5 in sixths).  With SMs left over, down to a pair of pages per warp (one sequence of 512 tokens:
    // 6.7 us in the kernel whole, 5.1 in pieces, replayed one after another).
    long long want = (pages + 32) / 64;
    if (units * want < d.sms) want = std::min(d.sms / units, pages / (2 * kDWarps));
    const int cs = (int)std::min<long long>(std::max<long long>(want, 1), kMaxCluster);
    if ((long long)r.n_seqs * cs > 0x7fffffffLL) return cudaErrorInvalidValue;
    count_launch();
    return kv8_dispatch(c.head_dim, a.q.type, [&](auto hd, auto type) {
        if constexpr (type != OT_F32)
            if (!four) return decode_launch<hd, type, 8>(c, r, a, cs, (int)tiles, st);
        return decode_launch<hd, type, 4>(c, r, a, cs, (int)tiles, st);
    });
}

}  // namespace s2k
