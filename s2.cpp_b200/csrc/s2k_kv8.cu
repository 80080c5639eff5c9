// s2k_kv8.cu -- storing into and reading from the 8-bit paged KV cache.
//
// Quantisation of one block (16 tokens of one kv head, keys or values):
//   s = max |x| / 127 over the block's tokens, held in f32
//   q = x / s rounded to the nearest integer, ties to even
// A block that fills over several calls keeps one scale: it only grows, and
// when it does, what the block holds is rounded again, q' = (q * s) / s'.
// Each such step adds at most half of s', and a block of 16 tokens sees few
// (the running maximum of 16 values changes about 3.4 times on average).
//
// The quotient is rounded exactly: the product with 1/s is within 127 * 2^-23 =
// 1.5e-5 of it, so its nearest integer n is right or one off, and the remainder
// e = x - n s tells: n is right iff |e| < s/2 (or = and n is even).  One fma
// gives e exactly: it is a multiple of s's last place (for n = 0 it is x) and
// not larger than about s/2, so it fits 24 bits.  The stored integers are then a
// function of the inputs alone, whatever computes them.
//
// int8 with a block's scale rather than an 8-bit float: over a block of normal
// values the uniform step's error is about a third of e4m3's, and every
// integer up to 127 is exact in f16, which the attention's products use.
//
// A block with a NaN or an infinity gets a NaN scale: it reads as NaN.
//
// Measured: eight prompts of up to 4096 f32 rows, 8 heads of 128, stored and read
// back: 91 us (5.1 TB/s), 49 us and 40 us in the kernels.  One token: 2.7 and 2.4
// us in the kernels, replayed one after another.
#include "s2k_common.cuh"
#include "s2k_kv8.h"

namespace s2k {

constexpr int kKv8Warps = 4;

// Adding 1.5 * 2^23 rounds to an integer, ties to even, and leaves it in the low mantissa bits: the conversion and
// rounding instructions run at a quarter of an addition's rate.
constexpr float kRound = 12582912.f;

// round(x / s) in the low byte, inv = 1 / s; s >= 2^-110 or s = x = 0
__device__ __forceinline__ unsigned q8(float x, float s, float inv) {
    const float t = __fadd_rn(__fmul_rn(x, inv), kRound);
    const int n = __float_as_int(t), e = __float_as_int(fmaf(-__fsub_rn(t, kRound), s, x));
    // |e| > s/2, or = and n is odd, in the order of their bits
    return (e & 0x7fffffff) + (n & 1) > __float_as_int(0.5f * s) ? n + (e >> 31 | 1) : n;
}
// round(q * was / s) for an older token's q, ratio = was / s: near a half it is divided in double, where a 31-bit by
// 24-bit quotient that is no half stays at least 2^-33 away from one
__device__ __forceinline__ unsigned q8_again(float q, float was, float s, float ratio) {
    const float r = __fmul_rn(q, ratio), t = __fadd_rn(r, kRound);
    if (s >= 1.17549435e-38f && fabsf(__fsub_rn(r, __fsub_rn(t, kRound))) <= 0.49998f) return __float_as_uint(t);
    return (unsigned)(int)fmin(fmax(rint((double)q * (double)was / (double)s), -127.0), 127.0);
}

// the low bytes of four words
__device__ __forceinline__ unsigned low_bytes(unsigned a, unsigned b, unsigned c, unsigned d) {
    return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}
// the first n bytes of a word
__device__ __forceinline__ unsigned byte_mask(int n) { return n <= 0 ? 0u : n >= 4 ? ~0u : (1u << (8 * n)) - 1u; }
// byte i of w as a number, exactly: 128 + q under 2^23's exponent
__device__ __forceinline__ float byte_value(unsigned w, int i) {
    return __uint_as_float(__byte_perm(w ^ 0x80808080u, 0x4b000000u, 0x7440 + i)) - 8388736.f;
}

// One warp per (sequence, page, kv head, keys or values): lane l holds dims
// [l*D, l*D + D) of the page's 16 tokens, so the block's maximum is one warp
// reduction and nothing is read twice.  Bound by the rows' bytes for prompts,
// by the chain of dependent loads for a single token.  Five CTAs per SM (96
// registers, a few of them spilled): 8 x 4096 f32 rows of 8 heads of 128 take 60
// us (5.6 TB/s), bf16 ones 57; with the compiler's choice of 168, 72 and 71.  One
// token 3.0 us against 2.6, one of 64 sequences 3.7, of 256 6.7 against 8.0.
template <int HD, int TYPE, bool VEC>
__global__ void __launch_bounds__(kKv8Warps * 32, 5) kv8_append_kernel(Kv8 c, Kv8Rows r, Rows k, Rows v,
                                                                      int pages_per_seq) {
    using T = typename OType<TYPE>::T;
    constexpr int D = HD / 32;
    const int lane = threadIdx.x & 31;
    const int unit = blockIdx.y * kKv8Warps + (threadIdx.x >> 5);
    const int b = blockIdx.x / pages_per_seq, pi = blockIdx.x % pages_per_seq;
    int row0, n, past;
    if (!kv8_seq(r, b, row0, n, past) || n == 0 || unit >= 2 * c.n_kv_heads) return;
    const bool is_v = unit >= c.n_kv_heads;
    const int head = is_v ? unit - c.n_kv_heads : unit;
    const int pg = past / kPage + pi, p0 = pg * kPage;
    if (p0 >= past + n) return;
    const int lo = max(past - p0, 0), hi = min(past + n - p0, kPage);  // slots [lo, hi) are new, [0, lo) older
    const Rows &src = is_v ? v : k;
    const T *x0 = reinterpret_cast<const T *>(src.p) + (long long)head * src.head_stride + lane * D;
    float x[kPage][D];
    unsigned top = 0;  // |x| as integers: NaN and infinity order above every finite value
    // slots without a new token load a neighbour's: a condition around a load would be waited for
#pragma unroll
    for (int t = 0; t < kPage; ++t)
        load_n<D>(x0 + (long long)(row0 + p0 + min(max(t, lo), hi - 1) - past) * src.row_stride, VEC, x[t]);
    const int page = kv8_page(c, r, b, pg);
    if (page < 0) return;
    const size_t blk = c.block(page, head);
    float *scale = (is_v ? c.v_scale : c.k_scale) + blk;
    int8_t *dst = (is_v ? c.v : c.k) + blk * (kPage * HD);
#pragma unroll
    for (int t = 0; t < kPage; ++t)
#pragma unroll
        for (int d = 0; d < D; ++d) top = max(top, __float_as_uint(x[t][d]) & 0x7fffffffu);
    const float was = lo > 0 ? *scale : 0.f;
    top = __reduce_max_sync(0xffffffffu, top);
    const float amax = __uint_as_float(top);
    const bool bad = top >= 0x7f800000u || was != was;
    const float fresh = __fdiv_rn(amax, 127.f);
    const float s = bad ? __int_as_float(0x7fc00000) : fmaxf(fresh, was);
    const bool zero = bad || s == 0.f, tiny = s < 7.8886091e-31f;  // 2^-100
    const float su = zero ? 0.f : tiny ? s * 18446744073709551616.f : s;
    if (zero || tiny) {
        // a NaN or an infinity would stay one; far down, both sides by 2^64, exactly.  A subnormal scale is so coarse that
        // a quotient can pass 127.
        const float most = 127.f * su;
#pragma unroll
        for (int t = 0; t < kPage; ++t)
#pragma unroll
            for (int d = 0; d < D; ++d)
                x[t][d] = zero ? 0.f : fminf(fmaxf(x[t][d] * 18446744073709551616.f, -most), most);
    }
    const float inv = zero ? 0.f : __fdiv_rn(1.f, su);
    if (lo > 0 && s != was && !zero) {  // the older tokens' scale grew: 4 or 16 bytes at a time, rarely and compactly
        const float ratio = __fdiv_rn(was, s);
        auto again = [&](unsigned w) {
            unsigned y = 0;
#pragma unroll 1
            for (int i = 0; i < 4; ++i) y = __funnelshift_r(y, q8_again(byte_value(w, i), was, s, ratio), 8);
            return y;
        };
        if (!is_v) {
            // a lane's D bytes of a key; the two of head_dim 64 as the low half of a word
#pragma unroll 1
            for (int t = 0; t < lo; ++t) {
                unsigned char *at = reinterpret_cast<unsigned char *>(dst + t * HD + lane * D);
                if (D == 4) *reinterpret_cast<unsigned *>(at) = again(*reinterpret_cast<const unsigned *>(at));
                else *reinterpret_cast<uint16_t *>(at) = (uint16_t)again(*reinterpret_cast<const uint16_t *>(at));
            }
        } else {
#pragma unroll 1
            for (int g = 0; g < 4 * D; ++g) {  // four tokens of a dimension; those behind lo are new or unused
                if (g % 4 * 4 >= lo) continue;
                unsigned *at = reinterpret_cast<unsigned *>(dst + (lane * D + g / 4) * kPage) + g % 4;
                const unsigned w = *at, m = byte_mask(lo - g % 4 * 4);
                *at = (again(w) & m) | (w & ~m);
            }
        }
    }
    if (!is_v) {
#pragma unroll
        for (int t = 0; t < kPage; ++t) {
            if (t < lo || t >= hi) continue;
            unsigned char *at = reinterpret_cast<unsigned char *>(dst + t * HD + lane * D);
            unsigned q[D];
#pragma unroll
            for (int d = 0; d < D; ++d) q[d] = q8(x[t][d], su, inv);
            if (D == 4) *reinterpret_cast<unsigned *>(at) = low_bytes(q[0], q[1], q[D - 2], q[D - 1]);
            else *reinterpret_cast<uint16_t *>(at) = (uint16_t)low_bytes(q[0], q[1], 0u, 0u);
        }
    } else {
        // 16 bytes of a dimension: four words of four tokens
        if (lo == 0 && hi == kPage) {
#pragma unroll
            for (int d = 0; d < D; ++d) {
                unsigned w[4];
#pragma unroll
                for (int g = 0; g < 4; ++g)
                    w[g] = low_bytes(q8(x[4 * g][d], su, inv), q8(x[4 * g + 1][d], su, inv), q8(x[4 * g + 2][d], su, inv),
                                     q8(x[4 * g + 3][d], su, inv));
                *reinterpret_cast<uint4 *>(dst + (lane * D + d) * kPage) = make_uint4(w[0], w[1], w[2], w[3]);
            }
            if (lane == 0) *scale = s;
            return;
        }
        // part of a page: bytes [lo, hi) are new, the others stay
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const unsigned m = byte_mask(hi - 4 * g) & ~byte_mask(lo - 4 * g);
            if (!m) continue;
#pragma unroll
            for (int d = 0; d < D; ++d) {
                unsigned *at = reinterpret_cast<unsigned *>(dst + (lane * D + d) * kPage) + g;
                unsigned q[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) q[e] = q8(x[4 * g + e][d], su, inv);
                const unsigned w = low_bytes(q[0], q[1], q[2], q[3]);
                *at = (w & m) | (*at & ~m);
            }
        }
    }
    if (lane == 0 && (lo == 0 || s != was)) *scale = s;
}

// The values the pages stand for: the same split, one warp per block.
template <int HD, int TYPE, bool VEC>
__global__ void __launch_bounds__(kKv8Warps * 32) kv8_read_kernel(Kv8 c, Kv8Rows r, Rows k, Rows v,
                                                                 int pages_per_seq) {
    using T = typename OType<TYPE>::T;
    constexpr int D = HD / 32;
    const int lane = threadIdx.x & 31;
    const int unit = blockIdx.y * kKv8Warps + (threadIdx.x >> 5);
    const int b = blockIdx.x / pages_per_seq, pi = blockIdx.x % pages_per_seq;
    int row0, n, past;
    if (!kv8_seq(r, b, row0, n, past) || n == 0 || unit >= 2 * c.n_kv_heads) return;
    const bool is_v = unit >= c.n_kv_heads;
    const int head = is_v ? unit - c.n_kv_heads : unit;
    const int pg = past / kPage + pi, p0 = pg * kPage;
    if (p0 >= past + n) return;
    const int lo = max(past - p0, 0), hi = min(past + n - p0, kPage);
    const int page = kv8_page(c, r, b, pg);
    if (page < 0) return;
    const Rows &dst = is_v ? v : k;
    T *y0 = reinterpret_cast<T *>(dst.p) + (long long)head * dst.head_stride + lane * D;
    const size_t blk = c.block(page, head);
    const float s = (is_v ? c.v_scale : c.k_scale)[blk];
    const int8_t *src = (is_v ? c.v : c.k) + blk * (kPage * HD);
    // one 4-byte word (keys) or 16 bytes (values) per lane and row or dimension, all on their way at once
    unsigned w[kPage];
    if (is_v) {
#pragma unroll
        for (int d = 0; d < D; ++d) {
            const uint4 o = *reinterpret_cast<const uint4 *>(src + (lane * D + d) * kPage);
            w[4 * d] = o.x, w[4 * d + 1] = o.y, w[4 * d + 2] = o.z, w[4 * d + 3] = o.w;
        }
    } else {
#pragma unroll
        for (int t = 0; t < kPage; ++t)
            w[t] = D == 4 ? *reinterpret_cast<const unsigned *>(src + t * HD + lane * D)
                          : *reinterpret_cast<const uint16_t *>(src + t * HD + lane * D);
    }
#pragma unroll
    for (int t = 0; t < kPage; ++t) {
        if (t < lo || t >= hi) continue;
        float y[D];
#pragma unroll
        for (int d = 0; d < D; ++d)
            y[d] = __fmul_rn(is_v ? byte_value(w[4 * d + t / 4], t % 4) : byte_value(w[t], d), s);
        store_n<D>(y0 + (long long)(row0 + p0 + t - past) * dst.row_stride, VEC, y);
    }
}

cudaError_t launch_kv8_append(const Kv8 &c, const Kv8Rows &r, const Rows &k, const Rows &v, cudaStream_t st) {
    if (r.n_seqs == 0 || r.max_rows == 0) return cudaSuccess;
    const int pages = (r.max_rows + kPage - 2) / kPage + 1;  // most pages that max_rows tokens touch
    const dim3 grid((unsigned)(r.n_seqs * (long long)pages), (2 * c.n_kv_heads + kKv8Warps - 1) / kKv8Warps);
    const int vec = rows_vec(k, c.head_dim / 32) && rows_vec(v, c.head_dim / 32);
    count_launch();
    return kv8_dispatch(c.head_dim, k.type, [&](auto hd, auto type) {
        if (vec) kv8_append_kernel<hd, type, true><<<grid, kKv8Warps * 32, 0, st>>>(c, r, k, v, pages);
        else kv8_append_kernel<hd, type, false><<<grid, kKv8Warps * 32, 0, st>>>(c, r, k, v, pages);
        return cudaGetLastError();
    });
}

cudaError_t launch_kv8_read(const Kv8 &c, const Kv8Rows &r, const Rows &k, const Rows &v, cudaStream_t st) {
    if (r.n_seqs == 0 || r.max_rows == 0) return cudaSuccess;
    const int pages = (r.max_rows + kPage - 2) / kPage + 1;
    const dim3 grid((unsigned)(r.n_seqs * (long long)pages), (2 * c.n_kv_heads + kKv8Warps - 1) / kKv8Warps);
    const int vec = rows_vec(k, c.head_dim / 32) && rows_vec(v, c.head_dim / 32);
    count_launch();
    return kv8_dispatch(c.head_dim, k.type, [&](auto hd, auto type) {
        if (vec) kv8_read_kernel<hd, type, true><<<grid, kKv8Warps * 32, 0, st>>>(c, r, k, v, pages);
        else kv8_read_kernel<hd, type, false><<<grid, kKv8Warps * 32, 0, st>>>(c, r, k, v, pages);
        return cudaGetLastError();
    });
}

}  // namespace s2k
