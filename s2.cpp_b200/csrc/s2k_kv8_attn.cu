// s2k_kv8_attn.cu -- attention of query rows over the 8-bit paged KV cache.
//
//   o = sum_j w_j v_j,  w = softmax over the visible keys of scale * q.k_j
// Row i of a sequence sits at position p = past + i and sees key j iff
//   j <= p  and  (window == 0  or  j > p - window  or  j < sinks).
// A row that sees nothing (a sequence whose pages are all bad) is zero.
#include "s2k_common.cuh"
#include "s2k_kv8.h"

#include <type_traits>

namespace s2k {

// One warp per (row, query head), one page of keys at a time with a running
// maximum and sum.
template <int HD, int TYPE>
__global__ void __launch_bounds__(128) kv8_attn_simple_kernel(Kv8 c, Kv8Rows r, Kv8Attn a) {
    using T = typename OType<TYPE>::T;
    constexpr int D = HD / 32;
    const int lane = threadIdx.x & 31;
    const int i = blockIdx.x, b = blockIdx.z;
    const int h = blockIdx.y * 4 + (threadIdx.x >> 5);
    int row0, n, past;
    if (!kv8_seq(r, b, row0, n, past) || i >= n || h >= a.n_heads) return;
    const int head = h / (a.n_heads / c.n_kv_heads);
    const int pos = past + i;
    float q[D], o[D] = {};
    load_n<D>(reinterpret_cast<const T *>(a.q.p) + (long long)(row0 + i) * a.q.row_stride +
                  (long long)h * a.q.head_stride + lane * D,
              false, q);
    float m = -INFINITY, l = 0.f;
    for (int pg = 0; pg * kPage <= pos; ++pg) {
        const int p0 = pg * kPage;
        if (a.window && p0 + kPage - 1 <= pos - a.window && p0 >= a.sinks) continue;
        const int page = kv8_page(c, r, b, pg);
        if (page < 0) continue;
        const size_t blk = c.block(page, head);
        const float ks = c.k_scale[blk] * a.scale, vs = c.v_scale[blk];
        const int8_t *kp = c.k + blk * (kPage * HD) + lane * D, *vp = c.v + blk * (kPage * HD) + lane * D * kPage;
        float s[kPage], top = -INFINITY;
#pragma unroll
        for (int t = 0; t < kPage; ++t) {
            float acc = 0.f;
#pragma unroll
            for (int d = 0; d < D; ++d) acc += q[d] * (float)kp[t * HD + d];
            acc = warp_sum(acc) * ks;
            const int j = p0 + t;
            const bool seen = j <= pos && (!a.window || j > pos - a.window || j < a.sinks);
            s[t] = seen ? acc : -INFINITY;
            top = fmaxf(top, s[t]);
        }
        const float m2 = fmaxf(m, top);
        if (m2 == -INFINITY) {
            // nothing seen yet, or only NaN scores: those reach the sum below
            bool nan = false;
#pragma unroll
            for (int t = 0; t < kPage; ++t) nan |= s[t] != s[t];
            if (nan) l = NAN;
            continue;
        }
        const float alpha = exp2f((m - m2) * 1.44269504f);
        l *= alpha;
#pragma unroll
        for (int d = 0; d < D; ++d) o[d] *= alpha;
#pragma unroll
        for (int t = 0; t < kPage; ++t) {
            if (s[t] == -INFINITY) continue;
            const float p = exp2f((s[t] - m2) * 1.44269504f);
            l += p;
#pragma unroll
            for (int d = 0; d < D; ++d) o[d] += p * vs * (float)vp[d * kPage + t];
        }
        m = m2;
    }
    const float inv = l != 0.f ? 1.f / l : 0.f;
#pragma unroll
    for (int d = 0; d < D; ++d) o[d] *= inv;
    store_n<D>(reinterpret_cast<T *>(a.out.p) + (long long)(row0 + i) * a.out.row_stride +
                   (long long)h * a.out.head_stride + lane * D,
               false, o);
}

cudaError_t launch_kv8_attend(const Kv8 &c, const Kv8Rows &r, const Kv8Attn &a, cudaStream_t st) {
    if (r.n_seqs == 0 || r.max_rows == 0) return cudaSuccess;
    const dim3 grid(r.max_rows, (a.n_heads + 3) / 4, r.n_seqs);
    count_launch();
    switch (c.head_dim * 100 + a.q.type) {
        case 12800 + OT_F32: kv8_attn_simple_kernel<128, OT_F32><<<grid, 128, 0, st>>>(c, r, a); break;
        case 12800 + OT_F16: kv8_attn_simple_kernel<128, OT_F16><<<grid, 128, 0, st>>>(c, r, a); break;
        case 12800 + OT_BF16: kv8_attn_simple_kernel<128, OT_BF16><<<grid, 128, 0, st>>>(c, r, a); break;
        case 6400 + OT_F32: kv8_attn_simple_kernel<64, OT_F32><<<grid, 128, 0, st>>>(c, r, a); break;
        case 6400 + OT_F16: kv8_attn_simple_kernel<64, OT_F16><<<grid, 128, 0, st>>>(c, r, a); break;
        case 6400 + OT_BF16: kv8_attn_simple_kernel<64, OT_BF16><<<grid, 128, 0, st>>>(c, r, a); break;
        default: return cudaErrorInvalidValue;
    }
    return cudaGetLastError();
}

}  // namespace s2k
