// s2k_logprobs.cu -- log probabilities of given tokens, entropy and top
// alternatives of rows of logits.
//
// With M = max x, c = how many values equal M, d = the sum of e^(x-M) over the
// others:  log S = log c + log1p(d / c)
//   log p_i = (x_i - M) - log S
//   H       = log S - (sum (x-M) e^(x-M)) / (c + d)
// The largest values' ones are counted apart from d because a sure row has
// d ~ 1e-6 and smaller: added to 1 in 32 bits it would be lost, and with it
// the entropy and the target's log probability, both about d.  Both terms of
// H are >= 0, so nothing cancels.
#include "s2k_common.cuh"
#include "s2k_kv8.h"

namespace s2k {

constexpr int kLpThreads = 512;

// A value and its index as one number: larger values first, then lower
// indexes.  NaN orders below every number.
__device__ __forceinline__ unsigned long long lp_key(float x, int i) {
    x = __fadd_rn(x, 0.f);  // -0 and +0 are equal
    const unsigned b = __float_as_uint(x);
    const unsigned o = x != x ? 0u : (b & 0x80000000u) ? ~b : b | 0x80000000u;
    return (unsigned long long)o << 32 | (unsigned)~i;
}
__device__ __forceinline__ float lp_value(unsigned long long key) {
    const unsigned o = (unsigned)(key >> 32);
    if (o == 0) return NAN;
    return __uint_as_float((o & 0x80000000u) ? o & 0x7fffffffu : ~o);
}

template <int TYPE>
__global__ void __launch_bounds__(kLpThreads) logprobs_simple_kernel(LogprobArgs a) {
    using T = typename OType<TYPE>::T;
    __shared__ float red[3][kLpThreads / 32];
    __shared__ unsigned long long redk[kLpThreads / 32];
    const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const T *x = reinterpret_cast<const T *>(a.x) + (long long)row * a.ld;
    float mx = -INFINITY;
    for (int i = tid; i < a.n; i += kLpThreads) mx = fmaxf(mx, to_f(x[i]));
    mx = warp_max(mx);
    if (lane == 0) red[0][warp] = mx;
    __syncthreads();
    mx = red[0][0];
    for (int w = 1; w < kLpThreads / 32; ++w) mx = fmaxf(mx, red[0][w]);
    __syncthreads();
    const bool masked = mx == -INFINITY;  // no token allowed (or NaN only): take 0, so that -inf gives e = 0, not NaN
    if (masked) mx = 0.f;
    float cnt = 0.f, d = 0.f, t = 0.f;
    for (int i = tid; i < a.n; i += kLpThreads) {
        const float z = to_f(x[i]) - mx;
        const float e = exp2f(z * 1.44269504f);
        if (z == 0.f) cnt += 1.f;
        else {
            d += e;
            if (e != 0.f) t += z * e;
        }
    }
    cnt = warp_sum(cnt), d = warp_sum(d), t = warp_sum(t);
    if (lane == 0) red[0][warp] = cnt, red[1][warp] = d, red[2][warp] = t;
    __syncthreads();
    cnt = d = t = 0.f;
    for (int w = 0; w < kLpThreads / 32; ++w) cnt += red[0][w], d += red[1][w], t += red[2][w];
    const bool none = masked && d == 0.f;  // every token masked (a NaN reaches d)
    const float ls = logf(cnt) + log1pf(d / cnt);
    if (tid == 0) {
        const int y = a.targets ? a.targets[row] : -1;
        if (a.logprob) a.logprob[row] = y < 0 || y >= a.n ? NAN : none ? -INFINITY : (to_f(x[y]) - mx) - ls;
        if (a.entropy) a.entropy[row] = none ? 0.f : ls - t / (cnt + d);
    }
    unsigned long long last = ~0ull;
    for (int k = 0; k < a.n_top; ++k) {
        unsigned long long best = 0;
        for (int i = tid; i < a.n; i += kLpThreads) {
            const unsigned long long key = lp_key(to_f(x[i]), i);
            if (key < last && key > best) best = key;
        }
        for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
        __syncthreads();
        if (lane == 0) redk[warp] = best;
        __syncthreads();
        for (int w = 0; w < kLpThreads / 32; ++w) best = max(best, redk[w]);
        last = best;
        if (tid == 0) {
            a.top_ids[(size_t)row * a.n_top + k] = (int)~(unsigned)best;
            a.top_logprob[(size_t)row * a.n_top + k] = none ? -INFINITY : (lp_value(best) - mx) - ls;
        }
    }
}

cudaError_t launch_logprobs(const LogprobArgs &a, cudaStream_t st) {
    if (a.rows == 0) return cudaSuccess;
    count_launch();
    switch (a.type) {
        case OT_F32: logprobs_simple_kernel<OT_F32><<<a.rows, kLpThreads, 0, st>>>(a); break;
        case OT_F16: logprobs_simple_kernel<OT_F16><<<a.rows, kLpThreads, 0, st>>>(a); break;
        case OT_BF16: logprobs_simple_kernel<OT_BF16><<<a.rows, kLpThreads, 0, st>>>(a); break;
        default: return cudaErrorInvalidValue;
    }
    return cudaGetLastError();
}

}  // namespace s2k
