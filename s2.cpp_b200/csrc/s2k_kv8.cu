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
// The quotient is rounded exactly: the product with 1/s is within 127 * 2^-23
// of it, so only a result that near to a half is divided again, in double
// (where a 24-bit by 24-bit quotient that is no half stays at least 2^-33
// away from one).  The stored integers are then a function of the inputs
// alone, whatever computes them.
//
// int8 with a block's scale rather than an 8-bit float: over a block of normal
// values the uniform step's error is about a third of e4m3's, and every
// integer up to 127 is exact in f16, which the attention's products use.
//
// A block with a NaN or an infinity gets a NaN scale: it reads as NaN.
#include "s2k_common.cuh"
#include "s2k_kv8.h"

namespace s2k {

constexpr int kKv8Warps = 4;

// q = round(x / s): r is the quotient to 127 * 2^-23, exact() the same in double
template <class F>
__device__ __forceinline__ int q8_round(float r, bool tiny, F exact) {
    float n = rintf(r);
    if (tiny || fabsf(fabsf(r - n) - 0.5f) < 1e-4f) n = (float)rint(exact());
    return (int)fminf(fmaxf(n, -127.f), 127.f);
}

__device__ __forceinline__ unsigned pack4(int a, int b, int c, int d) {
    return (unsigned)(a & 255) | (unsigned)(b & 255) << 8 | (unsigned)(c & 255) << 16 | (unsigned)(d & 255) << 24;
}

// One warp per (sequence, page, kv head, keys or values): lane l holds dims
// [l*D, l*D + D) of the page's 16 tokens, so the block's maximum is one warp
// reduction and nothing is read twice.  Bound by the rows' bytes for prompts,
// by the chain of dependent loads for a single token.
template <int HD, int TYPE, bool VEC>
__global__ void __launch_bounds__(kKv8Warps * 32) kv8_append_kernel(Kv8 c, Kv8Rows r, Rows k, Rows v,
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
    const int page = kv8_page(c, r, b, pg);
    if (page < 0) return;
    const Rows &src = is_v ? v : k;
    const T *x0 = reinterpret_cast<const T *>(src.p) + (long long)head * src.head_stride + lane * D;
    const size_t blk = c.block(page, head);
    float *scale = (is_v ? c.v_scale : c.k_scale) + blk;
    int8_t *dst = (is_v ? c.v : c.k) + blk * (kPage * HD);
    float x[kPage][D];
    unsigned top = 0;  // |x| as integers: NaN and infinity order above every finite value
    // slots without a new token load a neighbour's: a condition around a load would be waited for
#pragma unroll
    for (int t = 0; t < kPage; ++t)
        load_n<D>(x0 + (long long)(row0 + p0 + min(max(t, lo), hi - 1) - past) * src.row_stride, VEC, x[t]);
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
    const bool zero = bad || s == 0.f, tiny = s < 1.17549435e-38f;
    const float inv = zero ? 0.f : __fdiv_rn(1.f, s);
    const bool again = lo > 0 && s != was && !zero;  // the older tokens' scale grew
    const float ratio = again ? __fdiv_rn(was, s) : 1.f;
    auto quant = [&](float y) {
        return zero ? 0 : q8_round(__fmul_rn(y, inv), tiny, [&] { return (double)y / (double)s; });
    };
    auto requant = [&](int q) {
        return q8_round(__fmul_rn((float)q, ratio), tiny, [&] { return (double)q * (double)was / (double)s; });
    };
    if (!is_v) {
#pragma unroll
        for (int t = 0; t < kPage; ++t) {
            Vec<int8_t, D> *at = reinterpret_cast<Vec<int8_t, D> *>(dst + t * HD + lane * D);
            if (t >= lo && t < hi) {
                Vec<int8_t, D> u;
#pragma unroll
                for (int d = 0; d < D; ++d) u.v[d] = (int8_t)quant(x[t][d]);
                *at = u;
            } else if (t < lo && again) {
                Vec<int8_t, D> u = *at;
#pragma unroll
                for (int d = 0; d < D; ++d) u.v[d] = (int8_t)requant(u.v[d]);
                *at = u;
            }
        }
    } else {
#pragma unroll
        for (int d = 0; d < D; ++d) {
            uint4 *at = reinterpret_cast<uint4 *>(dst + (lane * D + d) * kPage);
            Vec<int8_t, kPage> u = {};
            if (lo > 0 || hi < kPage) u = *reinterpret_cast<const Vec<int8_t, kPage> *>(at);
#pragma unroll
            for (int t = 0; t < kPage; ++t) {
                if (t >= lo && t < hi) u.v[t] = (int8_t)quant(x[t][d]);
                else if (t < lo && again) u.v[t] = (int8_t)requant(u.v[t]);
            }
            *at = *reinterpret_cast<const uint4 *>(&u);
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
    Vec<int8_t, kPage> col[D];
    if (is_v) {
#pragma unroll
        for (int d = 0; d < D; ++d) col[d] = *reinterpret_cast<const Vec<int8_t, kPage> *>(src + (lane * D + d) * kPage);
    }
#pragma unroll
    for (int t = 0; t < kPage; ++t) {
        if (t < lo || t >= hi) continue;
        float y[D];
        if (is_v) {
#pragma unroll
            for (int d = 0; d < D; ++d) y[d] = __fmul_rn((float)col[d].v[t], s);
        } else {
            const Vec<int8_t, D> u = *reinterpret_cast<const Vec<int8_t, D> *>(src + t * HD + lane * D);
#pragma unroll
            for (int d = 0; d < D; ++d) y[d] = __fmul_rn((float)u.v[d], s);
        }
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
