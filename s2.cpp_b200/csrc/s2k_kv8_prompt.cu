// s2k_kv8_prompt.cu -- attention of many query rows (prompts) over the 8-bit
// paged KV cache, on the tensor cores (tcgen05).
//
// The same sums as s2k_kv8_attn.cu; here a kv head's pages are read for 128 or
// 256 slots at once (a slot is one (row, query head) pair of the kv head), so
// the products are the bound: 4 * head_dim operations per slot and visible key
// at the f16 rate, and one exponential per slot and key, which at 16 per cycle
// and SM takes as long as the products at head_dim 128 and twice as long at 64.
//
// One CTA per tile of slots; a step is 128 keys (8 pages):
//   warps 0-3    producers: int8 pages -> f16 operands in shared memory, two
//                steps deep (128-byte swizzled rows, K-major: keys [key][dim],
//                values [dim][key], which is how the cache holds them).  Every
//                int8 is exact in f16; the blocks' scales stay apart.
//   warp 4       one lane issues the products: S = Q K^T (128 x 128, f32 in
//                TMEM), O += P V with P from TMEM.
//   warps 8-11, 12-15   two groups of one row per thread: softmax of S, P as f16
//                over S's own columns, the output.
// The groups take turns: while one forms its weights, the other's products
// run.  f16 / bf16 rows: 256 slots, 128 per group, every step.  A last tile of
// up to 128 slots, and f32 rows: both groups have the same 128 slots and take
// alternate steps.
//
// Rounding, f16 / bf16 rows.  Q is used as it is, with K in its type (int8,
// and int8 times a power of two, are exact in bf16 too).  P is f16: a weight
// times its block's value scale, relative to a power of two within 2^7 of the
// row's largest such product (of the largest scale, a block of large values and
// next to no weight cost the others their bits), 2^15 at most, with f16's full
// precision down to 2^-20 of the largest.  O stays in TMEM (f32) and is rescaled
// only when that reference moves: in a row's first steps and rarely after.
//
// f32 rows.  Q (after a power of two per slot) and P are two f16 operands each,
// rounded and left over: twice the products for 22 bits.  Sums in TMEM lose a
// little at every addition (they are cut, not rounded), which over a long
// context would show in f32: each step's O is taken out and added in registers,
// half of the dimensions by each group, with the step's own largest weight and
// product as its references.
//
// Measured: 2 x 4096 bf16 rows, 32 / 8 heads of 128: 322 us, 607 TFLOP/s; 8191
// f16 rows under a window of 1000, 16 / 4 heads of 64: 133 us, 248 TFLOP/s; 1024
// f32 rows, 32 / 8 heads of 128: 52 us, 166 TFLOP/s.  With weights relative to the
// largest scale these took 318, 129 and 50.  A step of both groups takes ~4800
// cycles (stamped in a build at 312 us): a group's scores, weights and products
// wait for one another.
#include "s2k_common.cuh"
#include "s2k_kv8.h"
#include "s2k_tc.cuh"

#include <algorithm>
#include <atomic>

namespace s2k {

constexpr int kPM = 128;        // slots of a group, keys of a step
constexpr int kPPages = kPM / kPage;
constexpr int kPThreads = 512;  // warps 5-7 only make the register shares whole groups of four warps
constexpr int kPMeta = 4;       // steps whose scales and positions are held
// All log2.  A weight * value scale at its reference is 2^kPTop of P, or 2^kPStepTop for f32 rows, whose reference is the
// step's own; how far the largest product may pass its reference, and the running maximum of the scores its own; and how
// far the product's reference is kept above a scale in view (its factor has to be finite).
constexpr float kPTop = 7.f, kPStepTop = 14.f, kPSlack = 7.f, kPScoreSlack = 8.f, kPBelow = 100.f;
constexpr float kPFar = 1048576.f;  // sums of scores from here on with a scale's exponent lose bits that matter
constexpr float kPRound = 12582912.f;  // 1.5 * 2^23: an integer added to it is in its low bits
constexpr int kPNone = 0x7fffff00;  // "first token" of no page: behind every position

template <int HD>
struct PromptSmem {
    static constexpr int NC = HD / 64;
    alignas(1024) uint8_t q[2][NC][kPM * 128];  // f32: rounded, left over; else the groups'
    alignas(1024) uint8_t k[2][NC][kPM * 128];
    alignas(1024) uint8_t v[2][2][HD * 128];
    float qmul[kPM];
    struct Meta {
        // a value scale is between 2^ve and twice that; vb: its bits, but with an exponent of any size (0: far below)
        float ks[kPPages], ve[kPPages];
        int vb[kPPages];
        int p0[kPPages];
    };
    alignas(16) Meta meta[kPMeta];
    float join[3][kPM];
    float4 stat[kPMeta][kPM];  // f32 rows: a step's reference, sum and its products' reference
    uint64_t kfull[2], kempty[2], vfull[2], vempty[2], mfull[kPMeta], sfull[2], pfull[2][2], odone[2];
    uint64_t tfull[kPMeta], ofree[2], qfull, drained;
    uint32_t tmem;
};

// kind::f16: D f32, A and B f16 (or both bf16), K-major, M = 128
template <int N, bool BF16 = false>
constexpr uint32_t prompt_idesc() {
    return (1u << 4) | (BF16 ? 1u << 7 | 1u << 10 : 0) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(kPM >> 4) << 24);
}
// An operand's descriptor (sw128_desc) by its low word: the high word is the
// same for all, and 64-bit sums per product kept the issuing lane behind the
// tensor cores.
constexpr uint32_t kDescHigh = (uint32_t)((1024 >> 4) | (1u << 14) | (2u << 29));
__device__ __forceinline__ uint32_t desc_low(const void *p) { return ((smem_u32(p) >> 4) & 0x3fff) | 1u << 16; }
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, int acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\tsetp.ne.b32 p, %4, 0;\n\tmov.b64 a, {%1, %5};\n\t"
        "mov.b64 b, {%2, %5};\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t}" ::"r"(d),
        "r"(a), "r"(b), "r"(idesc), "r"(acc), "n"(kDescHigh)
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, int acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\tsetp.ne.b32 p, %4, 0;\n\tmov.b64 b, {%2, %5};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t}" ::"r"(d),
        "r"(a), "r"(b), "r"(idesc), "r"(acc), "n"(kDescHigh)
        : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(
            taddr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
        "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
        : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Four int8 (one word) -> two f16 pairs, exactly: q + 128 in the low bits of
// 1024's mantissa, minus 1152.
__device__ __forceinline__ void cvt_i8x4(uint32_t w, uint32_t &a, uint32_t &b) {
    w ^= 0x80808080u;
    const __half2 bias = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));
    uint32_t lo = __byte_perm(w, 0x64646464u, 0x4140), hi = __byte_perm(w, 0x64646464u, 0x4342);
    const __half2 l = __hsub2(*reinterpret_cast<__half2 *>(&lo), bias);
    const __half2 h = __hsub2(*reinterpret_cast<__half2 *>(&hi), bias);
    a = *reinterpret_cast<const uint32_t *>(&l);
    b = *reinterpret_cast<const uint32_t *>(&h);
}
// The same to bf16, times 2^-16: 128 products with the largest bf16 then stay within f32 (as they are, queries from 2.7e36
// on gave infinite scores).  With m = q mod 128, 128 + m has all its bits in bf16, and q is that less 128, or less 256 where
// q is negative: 128 with q's sign bit as its lowest exponent bit.
constexpr float kBf16Keys = 65536.f;
__device__ __forceinline__ void cvt_i8x4_bf16(uint32_t w, uint32_t &a, uint32_t &b) {
    const uint32_t m = w & 0x7f7f7f7fu, n = w & 0x80808080u;
    // 0x3b00 is 128 * 2^-16
    uint32_t x[4] = {__byte_perm(m, 0x3b3b3b3bu, 0x4140), __byte_perm(n, 0x3b3b3b3bu, 0x4140),
                     __byte_perm(m, 0x3b3b3b3bu, 0x4342), __byte_perm(n, 0x3b3b3b3bu, 0x4342)};
    const __nv_bfloat162 l = __hsub2(*reinterpret_cast<__nv_bfloat162 *>(&x[0]), *reinterpret_cast<__nv_bfloat162 *>(&x[1]));
    const __nv_bfloat162 h = __hsub2(*reinterpret_cast<__nv_bfloat162 *>(&x[2]), *reinterpret_cast<__nv_bfloat162 *>(&x[3]));
    a = *reinterpret_cast<const uint32_t *>(&l);
    b = *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t half2_bits(float x, float y) {
    const __half2 h = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t *>(&h);
}
// what rounding (x, y) to the f16 pair h left over
__device__ __forceinline__ uint32_t left_over(float x, float y, uint32_t h) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&h));
    return half2_bits(x - f.x, y - f.y);
}
// byte offset of 16-byte piece `piece` of row `row` in a 128-byte swizzled operand
__device__ __forceinline__ int swz(int row, int piece) { return row * 128 + ((piece ^ (row & 7)) << 4); }

template <int HD, int TYPE>
__global__ void __launch_bounds__(kPThreads, 1) kv8_prompt_kernel(Kv8 c, Kv8Rows r, Kv8Attn a, int vec_q, int vec_out) {
    using T = typename OType<TYPE>::T;
    using Sm = PromptSmem<HD>;
    constexpr bool wide = TYPE == OT_F32;
    constexpr int NC = Sm::NC, SLOTS = kv8_prompt_slots(TYPE);
    static_assert(SLOTS == (wide ? kPM : 2 * kPM), "groups of kPM slots");
    constexpr unsigned kAll = 0xffffffffu;
    extern __shared__ uint8_t raw[];
    Sm &sm = *reinterpret_cast<Sm *>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    // later tiles see more keys: they start first
    const int b = blockIdx.x % r.n_seqs, tile = gridDim.x / r.n_seqs - 1 - blockIdx.x / r.n_seqs, kvh = blockIdx.y;
    const int G = a.n_heads / c.n_kv_heads;
    int row0, n, past;
    if (!kv8_seq(r, b, row0, n, past) || (long long)tile * SLOTS >= (long long)n * G) return;
    // a slot's row: exact in f32 below 2^20 slots
    const bool few = (long long)n * G < 1 << 20;
    const float inv_group = 1.f / (float)G;
    auto row_of = [&](int slot) { return few ? (int)(((float)slot + 0.5f) * inv_group) : slot / G; };
    const int slot0 = tile * SLOTS, nslots = (int)min((long long)SLOTS, (long long)n * G - slot0);
    const bool split = wide || nslots <= kPM;  // the groups share the slots and alternate in steps
    const int pos_lo = past + row_of(slot0), pos_hi = past + row_of(slot0 + nslots - 1);
    const int wlo = a.window ? max(pos_lo - a.window + 1, 0) : 0;
    const int fw = wlo / kPage;
    const int ns = min((int)(((long long)a.sinks + kPage - 1) / kPage), fw);
    const int total = ns + pos_hi / kPage - fw + 1;
    const int steps = (total + kPPages - 1) / kPPages;
    const int jobs = split ? steps : 2 * steps;  // job g: group g % 2, step g or g / 2

    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&sm.kfull[i], 4);
            mbar_init(&sm.vfull[i], 4);
            mbar_init(&sm.kempty[i], 1);
            mbar_init(&sm.vempty[i], 1);
            mbar_init(&sm.sfull[i], 1);
            mbar_init(&sm.pfull[i][0], kPM);
            mbar_init(&sm.pfull[i][1], kPM);
            mbar_init(&sm.odone[i], 1);
            mbar_init(&sm.ofree[i], 2 * kPM);
        }
        mbar_init(&sm.qfull, 8);
        mbar_init(&sm.drained, 1);
        for (int i = 0; i < kPMeta; ++i) {
            mbar_init(&sm.mfull[i], 4);
            mbar_init(&sm.tfull[i], kPM);
        }
        fence_mbar_init();
    }
    if (warp == 4) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&sm.tmem))
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sm.tmem;
    bool ok = true;

    // registers: 512 threads start with 128 each, and 2 * 168 + 96 + 72 <= 4 * 128
    if (warp < 4) {
        // ---------------- producers: two pages of each step per warp ----------------
        asm volatile("setmaxnreg.dec.sync.aligned.u32 96;");
        const int pw = warp;
        constexpr int U = HD / 32;  // 16-byte pieces per lane and page
        uint4 kr[2][U], vr[2][U];
        // lanes 0 and 1 look up the warp's two pages, a step before anything depends on them
        auto first_token = [&](int t) {
            const int x = t * kPPages + 2 * pw + (lane & 1);
            return t < steps && x < total ? (x < ns ? x : x - ns + fw) * kPage : kPNone;
        };
        auto look_up = [&](int t) {
            const int p0 = first_token(t);
            return lane < 2 && p0 != kPNone ? kv8_page(c, r, b, p0 / kPage) : -1;
        };
        auto scales = [&](int page, float &ks, float &vs) {
            ks = vs = 0.f;
            if (page >= 0) {
                ks = c.k_scale[c.block(page, kvh)];
                vs = c.v_scale[c.block(page, kvh)];
            }
        };
        // where there is no page, page 0's: its tokens are behind every position, so nothing of them is used
        // (loads under a condition were waited for one by one, 4400 cycles a step)
        auto fetch = [&](const int8_t *src, const int (&pg)[2], uint4 (&x)[2][U]) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const uint4 *p = reinterpret_cast<const uint4 *>(src + c.block(max(pg[e], 0), kvh) * (kPage * HD)) + lane;
#pragma unroll
                for (int u = 0; u < U; ++u) x[e][u] = __ldg(p + u * 32);
            }
        };
        auto put = [&](uint8_t *buf, int row, int piece, uint32_t w0, uint32_t w1, bool bf16 = false) {
            uint4 h;
            if (bf16) {
                cvt_i8x4_bf16(w0, h.x, h.y);
                cvt_i8x4_bf16(w1, h.z, h.w);
            } else {
                cvt_i8x4(w0, h.x, h.y);
                cvt_i8x4(w1, h.z, h.w);
            }
            *reinterpret_cast<uint4 *>(buf + swz(row, piece)) = h;
        };
        int pg[2], own = look_up(0), next = look_up(1), later;
        float ks, vs;
        pg[0] = __shfl_sync(kAll, own, 0);
        pg[1] = __shfl_sync(kAll, own, 1);
        fetch(c.k, pg, kr);
        scales(own, ks, vs);
        for (int t = 0; t < steps && ok; ++t) {
            const int s = t & 1;
            fetch(c.v, pg, vr);
            later = look_up(t + 2);
            if (t >= 2) ok = kv8_wait(r, &sm.kempty[s], ((t >> 1) - 1) & 1, ERR_WAIT_EMPTY);
            if (!(ok = __all_sync(kAll, ok))) break;
            if (lane < 2) {
                typename Sm::Meta &m = sm.meta[t % kPMeta];
                m.ks[2 * pw + lane] = ks;
                // subnormal scales by way of 2^32; a block with an infinite or NaN one is NaN to whoever sees it
                const bool sub = vs < 1.17549435e-38f, none = vs == 0.f;
                const int bits = __float_as_int(sub ? vs * 4294967296.f : vs), e = bits >> 23 & 255;
                if (e == 255) m.ks[2 * pw + lane] = NAN;
                m.vb[2 * pw + lane] = none || e == 255 ? -(1 << 30) : bits - (sub ? 32 << 23 : 0);
                m.ve[2 * pw + lane] = none || e == 255 ? -200.f : (float)(e - (sub ? 159 : 127));
                m.p0[2 * pw + lane] = own >= 0 ? first_token(t) : kPNone;
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&sm.mfull[t % kPMeta]);
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    // piece x of a key's 16-dim pieces; lanes of the upper 64 dims store their halves in the other
                    // order, so that eight lanes meet all banks
                    const int id = u * 32 + lane, row = (2 * pw + e) * kPage + id / (HD / 16), x = id % (HD / 16);
                    uint8_t *buf = sm.k[s][x / 4];
                    const int flip = x / 4 & 1;
                    const uint4 w = kr[e][u];
                    put(buf, row, 2 * (x % 4) + flip, flip ? w.z : w.x, flip ? w.w : w.y, TYPE == OT_BF16);
                    put(buf, row, 2 * (x % 4) + 1 - flip, flip ? w.x : w.z, flip ? w.y : w.w, TYPE == OT_BF16);
                }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sm.kfull[s]);
            own = next;
            next = later;
            pg[0] = __shfl_sync(kAll, own, 0);
            pg[1] = __shfl_sync(kAll, own, 1);
            fetch(c.k, pg, kr);
            scales(own, ks, vs);
            if (t >= 2) ok = kv8_wait(r, &sm.vempty[s], ((t >> 1) - 1) & 1, ERR_WAIT_EMPTY);
            if (!(ok = __all_sync(kAll, ok))) break;
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int d = u * 32 + lane, page = 2 * pw + e;
                    uint8_t *buf = sm.v[s][page / 4];
                    const uint4 w = vr[e][u];
                    put(buf, d, 2 * (page % 4), w.x, w.y);
                    put(buf, d, 2 * (page % 4) + 1, w.z, w.w);
                }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sm.vfull[s]);
        }
    } else if (warp < 8) {
        // ---------------- products ----------------
        asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        if (warp == 4 && lane == 0) {
            // an operand's next 16 columns of K are 32 bytes on, the next 64 a chunk
            const uint32_t q0 = desc_low(sm.q[0][0]), q1 = desc_low(sm.q[1][0]);
            auto at = [](int x, int chunk) { return (uint32_t)(2 * (x % 4) + (x / 4) * (chunk >> 4)); };
            auto qk = [&](int g) {
                const int t = split ? g : g >> 1, w = g & 1, s = t & 1;
                if (!kv8_wait(r, &sm.kfull[s], (t >> 1) & 1, ERR_WAIT_FULL)) return false;
                tc_fence_after();
                const uint32_t d = tmem + w * kPM;
                const uint32_t q = !split && w ? q1 : q0, k = desc_low(sm.k[s][0]);
#pragma unroll
                for (int x = 0; x < 4 * NC; ++x) mma_ss(d, q + at(x, kPM * 128), k + at(x, kPM * 128), prompt_idesc<kPM, TYPE == OT_BF16>(), x != 0);
                if (wide) {
#pragma unroll
                    for (int x = 0; x < 4 * NC; ++x) mma_ss(d, q1 + at(x, kPM * 128), k + at(x, kPM * 128), prompt_idesc<kPM, TYPE == OT_BF16>(), 1);
                }
                mma_commit(&sm.sfull[w]);
                if (split || w) mma_commit(&sm.kempty[s]);
                return true;
            };
            ok = kv8_wait(r, &sm.qfull, 0, ERR_WAIT_FULL) && qk(0);
            if (ok && jobs > 1) ok = qk(1);
            for (int g = 0; g < jobs && ok; ++g) {
                const int t = split ? g : g >> 1, w = g & 1, s = t & 1;
                const uint32_t d = tmem + 2 * kPM + w * kPM, p = tmem + w * kPM;
                const uint32_t v = desc_low(sm.v[s][0]);
                ok = kv8_wait(r, &sm.vfull[s], (t >> 1) & 1, ERR_WAIT_FULL);
                // f32 rows: the output of two steps ago has been taken
                if (ok && wide && g > 1) ok = kv8_wait(r, &sm.ofree[w], ((g >> 1) - 1) & 1, ERR_WAIT_EMPTY);
                for (int h = 0; h < 2 && ok; ++h) {  // 64 keys each
                    if (!(ok = kv8_wait(r, &sm.pfull[w][h], (g >> 1) & 1, ERR_WAIT_FULL))) break;
                    tc_fence_after();
#pragma unroll
                    for (int y = 0; y < 4; ++y) {
                        const uint32_t vx = v + at(y, 0) + h * (HD * 128 >> 4);
                        const uint32_t px = p + 64 * h + 32 * (y / 2) + 8 * (y % 2);
                        mma_ts(d, px, vx, prompt_idesc<HD>(), (!wide && g > 1) || h > 0 || y > 0);
                        if (wide) mma_ts(d, px + 16, vx, prompt_idesc<HD>(), 1);
                    }
                }
                if (!ok) break;
                if (split || w) mma_commit(&sm.vempty[s]);
                if (wide || g + 2 >= jobs) mma_commit(&sm.odone[w]);
                if (g + 2 < jobs) ok = qk(g + 2);
            }
            if (!ok) {
                // a wait ran out: the products that were issued end before the CTA gives its memory back (they wait for
                // nothing, so this takes them microseconds)
                mma_commit(&sm.drained);
                mbar_wait(&sm.drained, 0, nullptr, ERR_WAIT_FULL);
            }
        }
    } else {
        // ---------------- softmax: one row per thread ----------------
        asm volatile("setmaxnreg.inc.sync.aligned.u32 168;");
        // queries: a lane eight dims, LR lanes a slot
        {
            constexpr int LR = HD / 8, RW = 32 / LR;
            const int dim = lane % LR * 8, all = nslots > kPM ? 2 * kPM : kPM;
            auto from = [&](int s) {
                const int st = slot0 + min(s, nslots - 1), row = row_of(st);
                return reinterpret_cast<const T *>(a.q.p) + (long long)(row0 + row) * a.q.row_stride +
                       (long long)(kvh * G + st - row * G) * a.q.head_stride + dim;
            };
            if constexpr (!wide) {  // as they are
                for (int s = (warp - 8) * RW + lane / LR; s < all; s += 8 * RW) {
                    uint8_t *to = &sm.q[s / kPM][dim / 64][swz(s % kPM, dim % 64 / 8)];
                    const T *p = from(s);
                    if (vec_q) {
                        cp16(to, p);
                    } else {
                        Vec<T, 8> u;
#pragma unroll
                        for (int e = 0; e < 8; ++e) u.v[e] = p[e];
                        *reinterpret_cast<Vec<T, 8> *>(to) = u;
                    }
                }
                cp_commit();
                cp_wait<0>();
            } else {  // -> f16 and what that leaves over
                constexpr int B = 4;
#pragma unroll 1
                for (int s0 = (warp - 8) * RW * B + lane / LR; s0 < all; s0 += 8 * RW * B) {
                    Vec<T, 8> raw8[B];
                    // one branch around all loads: with one around each they are waited for one by one
                    if (vec_q) {
#pragma unroll
                        for (int i = 0; i < B; ++i) load_raw(from(s0 + i * RW), raw8[i]);
                    } else {
#pragma unroll
                        for (int i = 0; i < B; ++i)
#pragma unroll
                            for (int e = 0; e < 8; ++e) raw8[i].v[e] = from(s0 + i * RW)[e];
                    }
#pragma unroll
                    for (int i = 0; i < B; ++i) {
                        const int s = s0 + i * RW;
                        unsigned top = 0;  // NaN and infinity order above as integers
#pragma unroll
                        for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(to_f(raw8[i].v[e])) & 0x7fffffffu);
#pragma unroll
                        for (int o = 1; o < LR; o <<= 1) top = max(top, __shfl_xor_sync(kAll, top, o));
                        // 2^-e brings the slot's largest to 2^13 .. 2^14
                        const int e2 = max((int)(top >> 23) - 127, -112) - 13;
                        const float down = __int_as_float((127 - e2) << 23);
                        if (dim == 0)
                            sm.qmul[s] = top >= 0x7f800000u ? NAN : a.scale * 1.44269504f * __int_as_float((e2 + 127) << 23);
                        uint32_t h[4], lo[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float x0 = to_f(raw8[i].v[2 * e]) * down, x1 = to_f(raw8[i].v[2 * e + 1]) * down;
                            h[e] = half2_bits(x0, x1);
                            lo[e] = left_over(x0, x1, h[e]);
                        }
                        const int at = swz(s, dim % 64 / 8);
                        *reinterpret_cast<uint4 *>(&sm.q[0][dim / 64][at]) = make_uint4(h[0], h[1], h[2], h[3]);
                        *reinterpret_cast<uint4 *>(&sm.q[1][dim / 64][at]) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                    }
                }
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sm.qfull);
            ok = kv8_wait(r, &sm.qfull, 0, ERR_WAIT_FULL);
        }
        const int w = (warp >> 2) - 2, row = tid & (kPM - 1), ls = (split ? 0 : w * kPM) + row;
        const int pos = past + row_of(slot0 + min(ls, nslots - 1));
        // positions of the warp's rows
        const int s_lo = slot0 + min(ls - lane, nslots - 1), s_hi = slot0 + min(ls - lane + 31, nslots - 1);
        const int p_min = past + row_of(s_lo), p_max = past + row_of(s_hi);
        const int wlo_row = a.window ? max(pos - a.window + 1, 0) : 0;  // the first position in the row's window
        const float smul = wide ? sm.qmul[row] : a.scale * 1.44269504f * (TYPE == OT_BF16 ? kBf16Keys : 1.f);
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t S = tmem + lanes + w * kPM, O = tmem + lanes + 2 * kPM + w * kPM;
        // log2 of the weights' reference (an integer), and of the products' relative to it
        float ref = -INFINITY, l = 0.f, vr = -INFINITY;
        // f32 rows: this group's half of the output
        constexpr int HALF = wide ? HD / 2 : 1;
        float acc[HALF];
#pragma unroll
        for (int i = 0; i < HALF; ++i) acc[i] = 0.f;
        float top_ref = -INFINITY, top_vr = -INFINITY, sum = 0.f;
        auto take = [&](int t) {  // f32 rows: adds step t's output
            bool fine = kv8_wait(r, &sm.tfull[t % kPMeta], (t / kPMeta) & 1, ERR_WAIT_FULL) &&
                        kv8_wait(r, &sm.odone[t & 1], (t >> 1) & 1, ERR_WAIT_FULL);
            if (!__all_sync(kAll, fine)) return false;
            tc_fence_after();
            const float4 z = sm.stat[t % kPMeta][row];
            const float r2 = fmaxf(top_ref, z.x);
            const float d0 = top_ref == r2 ? 0.f : top_ref - r2, d1 = z.x == r2 ? 0.f : z.x - r2;
            const float e0 = top_vr + d0, e1 = z.z + d1, v2 = fmaxf(e0, e1);
            const float f0 = e0 == v2 ? 1.f : ex2(e0 - v2), mul = z.z == -INFINITY ? 0.f : ex2(e1 - v2 - kPStepTop);
            sum = sum * ex2(d0) + (z.x == -INFINITY ? 0.f * z.y : z.y * ex2(d1));
            top_ref = r2;
            top_vr = v2;
            const uint32_t from = tmem + lanes + 2 * kPM + (t & 1) * kPM + w * HALF;
#pragma unroll
            for (int ch = 0; ch < (HALF + 15) / 16; ++ch) {
                int x[16];
                tmem_ld16(from + 16 * ch, x);
#pragma unroll
                for (int i = 0; i < 16 && 16 * ch + i < HALF; ++i)
                    acc[16 * ch + i] = fmaf(mul, __int_as_float(x[i]), acc[16 * ch + i] * f0);
            }
            tc_fence_before();
            mbar_arrive(&sm.ofree[t & 1]);
            return true;
        };
        int done = 0;  // this group's jobs so far
        for (int g = wide ? 0 : w; g < jobs && ok; g += wide ? 1 : 2) {
            if (wide && (g & 1) != w) {  // the other group's step
                if (g > 0) ok = take(g - 1);
                continue;
            }
            const int t = split ? g : g >> 1;
            ok = kv8_wait(r, &sm.mfull[t % kPMeta], (t / kPMeta) & 1, ERR_WAIT_FULL) &&
                 kv8_wait(r, &sm.sfull[w], done & 1, ERR_WAIT_FULL);
            if (!(ok = __all_sync(kAll, ok))) break;
            tc_fence_after();
            const typename Sm::Meta &m = sm.meta[t % kPMeta];
            int lo = m.p0[0], hi = m.p0[0];
            float vl = m.ve[0];  // the largest value scale that the row sees
#pragma unroll
            for (int i = 1; i < kPPages; ++i) {
                lo = min(lo, m.p0[i]);
                hi = max(hi, m.p0[i]);
                vl = fmaxf(vl, m.ve[i]);
            }
            const bool edge = hi + kPage - 1 > p_min || (a.window && lo <= p_max - a.window && hi + kPage > a.sinks) || a.scale < 0.f;
            // bit i: the row sees token i of page pg
            auto below = [](int n) { return 0xffffu >> (kPage - min(max(n, 0), kPage)); };
            auto seen = [&](int pg) {
                const int p0 = m.p0[pg];
                return below(pos + 1 - p0) & (~below(wlo_row - p0) | below(a.sinks - p0));
            };
            // the step's largest score, and log2 of its largest product over b.  Loops stay rolled: unrolled, with the next
            // columns' loads ahead, they took twice as long (the instruction cache serves ten warps in five places).
            float mx = -INFINITY, us = -INFINITY, b = ref == -INFINITY ? 0.f : ref;
            uint32_t any = 0;
            auto page_max = [&](int pg, float t) {
                mx = fmaxf(mx, t);
                us = fmaxf(us, (t - b) + m.ve[pg]);
            };
            auto whole_max = [&](int ch, const int(&y)[32], float k0, float k1) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float t0 = -INFINITY, t1 = -INFINITY;
#pragma unroll
                    for (int i = 0; i < kPage; i += 4) {
                        t0 = fmaxf(fmaxf(t0, __int_as_float(y[16 * e + i])), __int_as_float(y[16 * e + i + 1]));
                        t1 = fmaxf(fmaxf(t1, __int_as_float(y[16 * e + i + 2])), __int_as_float(y[16 * e + i + 3]));
                    }
                    page_max(2 * ch + e, fmaxf(t0, t1) * (e ? k1 : k0));
                }
            };
            bool large, careful;
#pragma unroll 1
            for (bool last = false;; last = true) {
                if (!edge) {
#pragma unroll 1
                    for (int ch = 0; ch < 4; ++ch) {
                        int y[32];
                        tmem_ld32(S + 32 * ch, y);
                        whole_max(ch, y, m.ks[2 * ch] * smul, m.ks[2 * ch + 1] * smul);
                    }
                    any = 1;
                } else {
                    vl = -INFINITY;
#pragma unroll 1
                    for (int ch = 0; ch < 4; ++ch) {
                        int y[32];
                        tmem_ld32(S + 32 * ch, y);
                        const float k0 = m.ks[2 * ch] * smul, k1 = m.ks[2 * ch + 1] * smul;
                        const uint32_t b0 = seen(2 * ch), b1 = seen(2 * ch + 1), bits = b0 | b1 << 16;
                        any |= bits;
                        if (b0) vl = fmaxf(vl, m.ve[2 * ch]);
                        if (b1) vl = fmaxf(vl, m.ve[2 * ch + 1]);
                        if (__all_sync(kAll, bits == 0)) continue;
                        // the largest product is the largest score's unless the scale is negative
                        if (__all_sync(kAll, bits == ~0u) && a.scale >= 0.f) {
                            whole_max(ch, y, k0, k1);
                            continue;
                        }
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            float t0 = -INFINITY;
#pragma unroll
                            for (int i = 0; i < kPage; ++i)
                                t0 = fmaxf(t0, bits >> (16 * e + i) & 1 ? __int_as_float(y[16 * e + i]) * (e ? k1 : k0) : -INFINITY);
                            page_max(2 * ch + e, t0);
                        }
                    }
                }
                // scores so large that they swallow a scale's exponent, unless b is next to them: once more
                large = fabsf(mx) > kPFar && fabsf(mx) < INFINITY;
                careful = __any_sync(kAll, large);
                if (last || !careful) break;
                if (large) b = ceilf(mx);
                us = -INFINITY;
            }
            // keys in view and no number among their scores: an infinite or NaN query or scale
            const float odd = any && mx == -INFINITY ? NAN : 0.f;
            const bool far = wide || mx > ref + kPScoreSlack;  // true for the first finite one
            const float r2 = far ? ceilf(mx) : ref, moved = far && r2 != ref ? r2 - ref : 0.f;
            // the products' reference that this step asks for, relative to r2
            const float need = fmaxf(r2 == -INFINITY ? us : us - (r2 - b), vl - kPBelow);
            if (wide) {
                ref = r2;
                vr = any ? ceilf(need) : -INFINITY;
            } else {
                const float old = vr - moved;
                const bool grow = need > old + kPSlack;
                if (__any_sync(kAll, far || grow)) {
                    if (far) l *= ex2(-moved);
                    vr = grow ? ceilf(need) : old;
                    if (done && __any_sync(kAll, grow)) {
                        const float f = grow ? ex2(old - vr) : 1.f;
#pragma unroll 2
                        for (int ch = 0; ch < HD / 16; ++ch) {
                            int z[16];
                            uint32_t y[16];
                            tmem_ld16(O + 16 * ch, z);
#pragma unroll
                            for (int i = 0; i < 16; ++i) y[i] = __float_as_uint(__int_as_float(z[i]) * f);
                            tmem_st16(O + 16 * ch, y);
                        }
                    }
                    ref = r2;
                }
            }
            // what is taken from the scores: large ones are rounded first like the maximum, which they must not pass
            const float base = ref == -INFINITY ? 0.f : ref, fused = large ? 0.f : -base, apart = large ? -base : 0.f;
            // a page's scale times 2^(top - vr) by its bits; 0 where that is below every normal number
            const int vc = __float_as_int(kPRound + (wide ? kPStepTop : kPTop) - vr) << 23;
            auto scale_of = [&](int pg) { return __int_as_float(__viaddmax_s32(m.vb[pg], vc, 0)); };
            float l0 = odd, l1 = 0.f;
            // masked: some keys are hidden, or scores are large
            auto weights = [&](int ch, const int(&y)[32], auto masked) {
                uint32_t hi16[16], lo16[16];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float ks = m.ks[2 * ch + e] * smul, vs = scale_of(2 * ch + e);
                    const uint32_t bits = masked ? seen(2 * ch + e) : 0;
#pragma unroll
                    for (int i = 0; i < kPage; i += 2) {
                        float p[2] = {fused, fused};
                        fma2(p, ks, __int_as_float(y[16 * e + i]), __int_as_float(y[16 * e + i + 1]));
                        if (masked) add2(p[0], p[1], apart);
                        p[0] = ex2(p[0]);
                        p[1] = ex2(p[1]);
                        if (masked) {  // a hidden block's scales may be NaN
                            p[0] = bits >> i & 1 ? p[0] : 0.f;
                            p[1] = bits >> (i + 1) & 1 ? p[1] : 0.f;
                        }
                        l0 += p[0];
                        l1 += p[1];
                        mul2(p, vs);
                        if (masked) {
                            p[0] = bits >> i & 1 ? p[0] : 0.f;
                            p[1] = bits >> (i + 1) & 1 ? p[1] : 0.f;
                        }
                        hi16[8 * e + i / 2] = half2_bits(p[0], p[1]);
                        if (wide) lo16[8 * e + i / 2] = left_over(p[0], p[1], hi16[8 * e + i / 2]);
                    }
                }
                tmem_st16(S + 32 * ch, hi16);
                if (wide) tmem_st16(S + 32 * ch + 16, lo16);
            };
            auto half_done = [&](int h) {  // its products may start
                tmem_wait_st();
                tc_fence_before();
                mbar_arrive(&sm.pfull[w][h]);
            };
            if (!edge && !careful) {
#pragma unroll 1
                for (int ch = 0; ch < 4; ++ch) {
                    int y[32];
                    tmem_ld32(S + 32 * ch, y);
                    weights(ch, y, std::false_type());
                    if (ch & 1) half_done(ch / 2);
                }
            } else {
#pragma unroll 1
                for (int ch = 0; ch < 4; ++ch) {
                    const uint32_t bits = seen(2 * ch) | seen(2 * ch + 1) << 16;
                    if (__all_sync(kAll, bits == 0)) {  // nothing of it in the warp's view
                        const uint32_t none[16] = {};
                        tmem_st16(S + 32 * ch, none);
                        if (wide) tmem_st16(S + 32 * ch + 16, none);
                    } else {
                        int y[32];
                        tmem_ld32(S + 32 * ch, y);
                        if (__all_sync(kAll, bits == ~0u) && !careful) weights(ch, y, std::false_type());
                        else weights(ch, y, std::true_type());
                    }
                    if (ch & 1) half_done(ch / 2);
                }
            }
            if (wide) {
                sm.stat[t % kPMeta][row] = make_float4(ref, l0 + l1, vr, 0.f);
                mbar_arrive(&sm.tfull[t % kPMeta]);
                if (g > 0) ok = take(g - 1);
            } else {
                l += l0 + l1;
            }
            ++done;
        }
        // The group's outputs go out by way of its half of Q's memory (the products are done with it), so that a warp
        // stores whole rows: pieces of 16 bytes, a row's pieces exchanged by its number to meet all banks.
        constexpr int E = 16 / sizeof(T), PIECES = (wide ? HD / 2 : HD) / E;
        uint8_t *stage = sm.q[w][0];
        auto piece_at = [&](int rr, int piece) { return stage + (rr * PIECES + (piece ^ (rr & 7))) * 16; };
        auto lay = [&](int first, const float (&z)[16]) {  // 16 dims of the thread's row
#pragma unroll
            for (int p = 0; p < 16 / E; ++p) {
                Vec<T, E> u;
#pragma unroll
                for (int e = 0; e < E; ++e) u.v[e] = from_f<T>(z[p * E + e]);
                *reinterpret_cast<Vec<T, E> *>(piece_at(row, first / E + p)) = u;
            }
        };
        auto store_rows = [&](int dim0) {  // the warp's 32 rows, dims from dim0 on
            __syncwarp();
            constexpr int RPI = 32 / PIECES;  // rows per access
#pragma unroll 4
            for (int rr = 0; rr < 32; rr += RPI) {
                const int rl = row - lane + rr + lane / PIECES, sl = ls - lane + rr + lane / PIECES, p = lane % PIECES;
                if (sl >= nslots) break;
                const int s2 = slot0 + sl, t2 = row_of(s2);
                T *y = reinterpret_cast<T *>(a.out.p) + (long long)(row0 + t2) * a.out.row_stride +
                       (long long)(kvh * G + s2 - t2 * G) * a.out.head_stride + dim0 + p * E;
                const Vec<T, E> u = *reinterpret_cast<const Vec<T, E> *>(piece_at(rl, p));
                if (vec_out) {
                    *reinterpret_cast<Vec<T, E> *>(y) = u;
                } else {
#pragma unroll
                    for (int e = 0; e < E; ++e) y[e] = u.v[e];
                }
            }
        };
        // f times 2^e as f * rest: 2^e may be subnormal
        auto in_two = [](float e, float &f, float &rest) {
            if (e == -INFINITY) e = 0.f;
            f *= ex2(fmaxf(e, -64.f));
            rest = ex2(fminf(e + 64.f, 0.f));
        };
        if (wide) {
            if (ok) ok = take(jobs - 1);
            if (!__all_sync(kAll, ok)) sum = NAN;  // a wait ran out: the result says so
            float inv = sum == 0.f ? 0.f : __fdiv_rn(1.f, sum), rest;
            in_two(top_vr, inv, rest);
#pragma unroll
            for (int i = 0; i < HALF; i += 16) {
                float z[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) z[e] = acc[(i + e) % HALF] * inv * rest;
                lay(i, z);
            }
            store_rows(w * HALF);
        } else {
            if (ok && done) ok = kv8_wait(r, &sm.odone[w], 0, ERR_WAIT_FULL);
            if (ok && split && w) ok = kv8_wait(r, &sm.odone[0], 0, ERR_WAIT_FULL);  // it stores where V was
            ok = __all_sync(kAll, ok);
            if (!ok) l = NAN;
            tc_fence_after();
            float *xch = reinterpret_cast<float *>(sm.k);  // [kPM][HD + 4], over K and V
            if (split) {
                if (w == 1) {
#pragma unroll 1
                    for (int ch = 0; ch < HD / 16; ++ch) {
                        int x[16] = {};
                        if (done) tmem_ld16(O + 16 * ch, x);
#pragma unroll
                        for (int i = 0; i < 16; i += 4)
                            *reinterpret_cast<int4 *>(&xch[row * (HD + 4) + 16 * ch + i]) = make_int4(x[i], x[i + 1], x[i + 2], x[i + 3]);
                    }
                    sm.join[0][row] = ref;
                    sm.join[1][row] = l;
                    sm.join[2][row] = vr;
                }
                named_sync(1, 2 * kPM);
            }
            if ((!split || w == 0) && ls - lane < nslots) {
                float f0 = 1.f, f1 = 0.f;  // the groups' outputs to the larger of their units
                if (split) {
                    const float ref1 = sm.join[0][row], top = fmaxf(ref, ref1);
                    const float d0 = ref == top ? 0.f : ref - top, d1 = ref1 == top ? 0.f : ref1 - top;
                    const float e0 = vr + d0, e1 = sm.join[2][row] + d1;
                    l = (ref == -INFINITY ? 0.f * l : ex2(d0) * l) + (ref1 == -INFINITY ? 0.f * sm.join[1][row] : ex2(d1) * sm.join[1][row]);
                    vr = fmaxf(e0, e1);
                    f0 = e0 == vr ? 1.f : ex2(e0 - vr);
                    f1 = e1 == vr ? 1.f : ex2(e1 - vr);
                }
                float inv = l == 0.f ? 0.f : __fdiv_rn(1.f, l), rest;
                in_two(vr - kPTop, inv, rest);
                f0 *= inv;
                f1 *= inv;
#pragma unroll 1
                for (int ch = 0; ch < HD / 16; ++ch) {
                    int x[16];
                    tmem_ld16(O + 16 * ch, x);
                    float z[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) z[i] = __int_as_float(x[i]) * f0;
                    if (split) {
#pragma unroll
                        for (int i = 0; i < 16; i += 4) {
                            const float4 o1 = *reinterpret_cast<const float4 *>(&xch[row * (HD + 4) + 16 * ch + i]);
                            z[i] += f1 * o1.x, z[i + 1] += f1 * o1.y, z[i + 2] += f1 * o1.z, z[i + 3] += f1 * o1.w;
                        }
                    }
#pragma unroll
                    for (int i = 0; i < 16; ++i) z[i] *= rest;
                    lay(16 * ch, z);
                }
                store_rows(0);
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 4) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
}

// More than half of an SM's: a CTA holds all of its TMEM, a second one would only wait for it.
template <int HD>
constexpr int prompt_smem() {
    return std::max((int)sizeof(PromptSmem<HD>) + 1024, 120 * 1024);
}

static std::atomic<int> g_prompt_ready[64];

cudaError_t launch_kv8_prompt(const Kv8 &c, const Kv8Rows &r, const Kv8Attn &a, cudaStream_t st) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= 64) return cudaErrorInvalidDevice;
    if (!g_prompt_ready[dev].load(std::memory_order_acquire)) {
        for (int hd : {64, 128})
            for (int type : {OT_F32, OT_F16, OT_BF16})
                if ((e = kv8_dispatch(hd, type, [&](auto h, auto t) {
                         return cudaFuncSetAttribute(kv8_prompt_kernel<h, t>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                     prompt_smem<h>());
                     })))
                    return e;
        g_prompt_ready[dev].store(1, std::memory_order_release);
    }
    const long long slots = (long long)r.max_rows * (a.n_heads / c.n_kv_heads);
    const int per = kv8_prompt_slots(a.q.type);
    const long long tiles = (slots + per - 1) / per;
    if (slots > 0x7fffffffLL || tiles * r.n_seqs > 0x7fffffffLL) return cudaErrorInvalidValue;
    const dim3 grid((unsigned)(tiles * r.n_seqs), c.n_kv_heads);
    const int vec_q = rows_vec(a.q, a.q.type == OT_F32 ? 4 : 8), vec_out = rows_vec(a.out, a.out.type == OT_F32 ? 4 : 8);
    count_launch();
    return kv8_dispatch(c.head_dim, a.q.type, [&](auto h, auto t) {
        kv8_prompt_kernel<h, t><<<grid, kPThreads, prompt_smem<h>(), st>>>(c, r, a, vec_q, vec_out);
        return cudaGetLastError();
    });
}

}  // namespace s2k
