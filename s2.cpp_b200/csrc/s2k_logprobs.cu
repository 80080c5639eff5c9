// s2k_logprobs.cu -- log probabilities of given tokens, entropy and top
// alternatives of rows of logits, in one pass over the logits.
//
// With M = max x, c = how many values equal M, d = the sum of e^(x-M) over the
// others and t that of (x-M) e^(x-M):  log S = log c + log1p(d / c),
//   log p_i = (x_i - M) - log S        H = log S - t / (c + d)
// The largest values' ones are counted apart from d because a sure row has
// d ~ 1e-6 and smaller: added to 1 in 32 bits it would be lost, and with it
// the entropy and the target's log probability, both about d.  Both terms of
// H are >= 0, so nothing cancels.
//
// Bound by the logits' bytes.  A CTA takes tiles of 8192 logits, 32 per thread
// in registers with the next 32 on their way, and each thread keeps (M, c, d,
// t) of its own and the maximum of each of its tiles: no exchange and no
// barrier inside the loop, one ex2 and eight other instructions a logit (HBM's
// rate leaves room for 21 in f32, 10 in 16 bits).  A row's CTAs are a cluster
// and send what they found to its first.
//
// Top alternatives.  A logit and its index are one 64-bit key (ties to the
// lowest index).  After the loop, the k-th largest of the 64 maxima of four
// threads each bounds the k-th largest logit from below; only the (thread,
// tile) pairs whose maximum reaches it, little more than k, are read again, a
// warp a pair.  Rows with so many ties that the pairs or the candidates do not
// fit go tile by tile instead, with the bound raised by each tile's own maxima
// and the list of candidates cut to its best k.  (Looking for candidates inside
// the loop took 124 us for 512 rows of 155648 f32 logits: barriers.)
// -inf and NaN are no candidates; a row with fewer than k others is filled up
// with them at the end.
//
// Measured, top 8: 512 rows of 155648 f32 logits 65-66 us (4.9 TB/s), f16 53.5 and
// bf16 53.9 (3.0 TB/s: the instructions are the same for half the bytes); one row
// of f32 16.6 us with the call, 11.2 in the kernel with cold caches, and replayed
// one after another 8.5, f16 8.2, bf16 7.8.
#include "s2k_common.cuh"
#include "s2k_kv8.h"

#include <algorithm>
#include <atomic>

namespace s2k {

constexpr int kLpThreads = 256;
constexpr int kLpItems = 32;                        // logits per thread and tile
constexpr int kLpTile = kLpThreads * kLpItems;      // 8192
constexpr int kLpGroups = 64;                       // of 4 threads
constexpr int kLpCap = 1024;                        // candidates
constexpr int kLpPairs = 512;                       // (thread, record) pairs read again at once
constexpr int kLpRecords = 16;                      // maxima a thread keeps, of one or more tiles
constexpr int kLpTop = 32;                          // S2K_LOGPROBS_MAX_TOP
using lp_key_t = unsigned long long;

// Of a finite or infinite x: larger values first, then lower indexes.  0: none.
__device__ __forceinline__ lp_key_t lp_key(float x, int i) {
    const unsigned b = __float_as_uint(__fadd_rn(x, 0.f));  // -0 and +0 are equal
    return (lp_key_t)((b & 0x80000000u) ? ~b : b | 0x80000000u) << 32 | (unsigned)~i;
}
__device__ __forceinline__ float lp_value(lp_key_t key) {
    const unsigned o = (unsigned)(key >> 32);
    return __uint_as_float((o & 0x80000000u) ? o & 0x7fffffffu : ~o);
}

// Maximum, how many equal it, and the others' sums relative to it.
struct alignas(16) LpSums {
    float m = -INFINITY, c = 0.f, d = 0.f, t = 0.f;
    // the same relative to M >= m
    __device__ void shift(float M) {
        if (m == M) return;
        const float z = m - M;  // -inf where nothing was summed: m = -inf has c = 0 and d = 0 (or NaN)
        const float e = ex2(z * 1.44269504f);
        const float s = c + d;
        t = e == 0.f && s == s ? 0.f : e * fmaf(z, s, t);
        d = s == s ? e * s : s;
        c = 0.f;
        m = M;
    }
    __device__ void join(LpSums o) {
        const float M = fmaxf(m, o.m);
        shift(M);
        o.shift(M);
        c += o.c, d += o.d, t += o.t;
    }
};

// Joins the lanes' sums, groups of `width` lanes (a power of two) each.
__device__ void lp_join_lanes(LpSums &s, int width) {
    for (int o = width >> 1; o > 0; o >>= 1) {
        LpSums q;
        q.m = __shfl_xor_sync(0xffffffffu, s.m, o);
        q.c = __shfl_xor_sync(0xffffffffu, s.c, o);
        q.d = __shfl_xor_sync(0xffffffffu, s.d, o);
        q.t = __shfl_xor_sync(0xffffffffu, s.t, o);
        s.join(q);
    }
}

struct LpSmem {
    LpSums warp[kLpThreads / 32];
    LpSums row[kMaxCluster];             // the cluster's CTAs, in its first
    lp_key_t top[kMaxCluster][kLpTop];   // and their best keys
    alignas(16) lp_key_t cand[kLpCap];
    lp_key_t best[kLpTop], group[kLpGroups];
    lp_key_t tau;
    int count, pairs;
    uint16_t pair[kLpPairs];  // record * kLpThreads + thread
    float rec[kLpRecords][kLpThreads];
    float fill[kLpThreads / 32];
};

// The k largest of keys[0..n) in order to out (0 where there are fewer): each key's rank by counting.  Zeroes keys up
// to a multiple of 4; all threads, ends with a barrier.
__device__ void lp_select(lp_key_t *keys, int n, int k, lp_key_t *out) {
    const int padded = (n + 3) & ~3;
    if (threadIdx.x < k) out[threadIdx.x] = 0;
    if (threadIdx.x < padded - n) keys[n + threadIdx.x] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kLpThreads) {
        const lp_key_t mine = keys[i];
        int rank = 0;
#pragma unroll 2
        for (int j = 0; j < padded; j += 4) {
            const ulonglong2 u = *reinterpret_cast<const ulonglong2 *>(keys + j);
            const ulonglong2 w = *reinterpret_cast<const ulonglong2 *>(keys + j + 2);
            rank += (u.x > mine) + (u.y > mine) + (w.x > mine) + (w.y > mine);
        }
        if (rank < k && mine) out[rank] = mine;
    }
    __syncthreads();
}

// Raises tau to the k-th largest of the groups' keys (kept bits of it): so many logits reach it.  All threads, ends
// with a barrier.
__device__ void lp_raise(LpSmem &sm, int k, lp_key_t kept) {
    if (threadIdx.x < kLpGroups) {
        const lp_key_t g = sm.group[threadIdx.x];
        int r = 0;
#pragma unroll 8
        for (int j = 0; j < kLpGroups; ++j) r += sm.group[j] > g;
        if (r == k - 1 && (g & kept) > sm.tau) sm.tau = g & kept;  // keys differ: one thread at most
    }
    __syncthreads();
}

// Fills out[have..k) with the row's first masked (-inf) and then its first NaN logits; all threads, ends with a barrier.
template <class T>
__device__ void lp_fill(const T *x, int n, int have, int k, int *ids, float *logprob, float *scratch) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int nan = 0; nan < 2; ++nan)
        for (int base = 0; base < n && have < k; base += kLpThreads) {
            const int i = base + threadIdx.x;
            const float y = i < n ? to_f(x[i]) : 0.f;
            const bool hit = nan ? y != y : y == -INFINITY;
            const unsigned ballot = __ballot_sync(0xffffffffu, hit);
            if (lane == 0) scratch[warp] = (float)__popc(ballot);
            __syncthreads();
            int before = have + __popc(ballot & ((1u << lane) - 1)), all = 0;
            for (int w = 0; w < kLpThreads / 32; ++w) {
                if (w < warp) before += (int)scratch[w];
                all += (int)scratch[w];
            }
            if (hit && before < k) {
                ids[before] = i;
                logprob[before] = y;
            }
            have += all;
            __syncthreads();
        }
}

template <int TYPE>
__global__ void __launch_bounds__(kLpThreads, 2) logprobs_kernel(LogprobArgs a, int cs_log2) {
    using T = typename OType<TYPE>::T;
    constexpr int E = 16 / sizeof(T), V = kLpItems / E;  // logits of a 16-byte access, accesses of a tile
    __shared__ LpSmem sm;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int cs = 1 << cs_log2, rank = blockIdx.x & (cs - 1);
    const long long row = blockIdx.x >> cs_log2;
    const T *x = reinterpret_cast<const T *>(a.x) + row * a.ld;
    const int k = a.n_top;
    if (cs > 1) cluster_arrive();
    if (tid == 0) sm.tau = 0, sm.count = sm.pairs = 0;
    // the row in 16-byte pieces of aligned memory: piece g holds logits g * E - shift ..
    const int shift = (int)(((uintptr_t)x & 15) / sizeof(T));
    const int pieces = (a.n + shift + E - 1) / E;
    // this CTA's tiles: a contiguous run
    const int tiles = (pieces + kLpThreads * V - 1) / (kLpThreads * V);
    const int t0 = (int)((long long)tiles * rank >> cs_log2), t1 = (int)((long long)tiles * (rank + 1) >> cs_log2);
    const int R = (t1 - t0 + kLpRecords - 1) / kLpRecords;  // tiles of a record
    float rec = -INFINITY;
    uint4 next[V];
    auto fetch = [&](int tile) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int g = tile * (kLpThreads * V) + v * kLpThreads + tid, i = g * E - shift;
            if (i >= 0 && i <= a.n - E) {
                next[v] = __ldcs(reinterpret_cast<const uint4 *>(x + i));
            } else {  // the row's ends: what is not there counts as masked
                alignas(16) T y[E];
#pragma unroll
                for (int e = 0; e < E; ++e) y[e] = i + e >= 0 && i + e < a.n ? x[i + e] : from_f<T>(-INFINITY);
                next[v] = *reinterpret_cast<const uint4 *>(y);
            }
        }
    };
    LpSums s;
    if (t0 < t1) fetch(t0);
    for (int tile = t0; tile < t1; ++tile) {
        float y[kLpItems];
#pragma unroll
        for (int v = 0; v < V; ++v)
#pragma unroll
            for (int e = 0; e < E; ++e) y[v * E + e] = to_f(reinterpret_cast<const T *>(&next[v])[e]);
        if (tile + 1 < t1) fetch(tile + 1);
        float top = y[0];
#pragma unroll
        for (int i = 1; i < kLpItems; ++i) top = fmaxf(top, y[i]);
        if (top > s.m) s.shift(top);
        const float m = s.m == -INFINITY ? 0.f : s.m;
        // (x - M) e^(x-M): -inf * 0 is NaN, and e is 0 from -150 on.  e rounds to 1 only next to the maximum.
        float d0 = 0.f, d1 = 0.f, u0 = 0.f, u1 = 0.f, c0 = 0.f, c1 = 0.f;
#pragma unroll
        for (int i = 0; i < kLpItems; i += 2) {
            float z0 = y[i], z1 = y[i + 1];
            add2(z0, z1, -m);
            const float e0 = ex2(z0 * 1.44269504f), e1 = ex2(z1 * 1.44269504f);
            if (e0 >= 1.f) c0 += 1.f;
            else d0 += e0;
            if (e1 >= 1.f) c1 += 1.f;
            else d1 += e1;
            u0 = fmaf(fmaxf(z0, -1000.f), e0, u0), u1 = fmaf(fmaxf(z1, -1000.f), e1, u1);
        }
        s.c += c0 + c1;
        s.d += d0 + d1;
        s.t += u0 + u1;
        rec = fmaxf(rec, top);
        if ((tile + 1 - t0) % R == 0 || tile + 1 == t1) {
            sm.rec[(tile - t0) / R][tid] = rec;
            rec = -INFINITY;
        }
    }
    if (k) {
        const int records = t1 > t0 ? (t1 - t0 + R - 1) / R : 0;
        float best = fmaxf(s.m, __shfl_xor_sync(0xffffffffu, s.m, 1));
        best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, 2));
        if ((tid & 3) == 0) sm.group[tid >> 2] = best > -INFINITY ? lp_key(best, tid) : 0;
        __syncthreads();
        lp_raise(sm, k, 0xffffffff00000000ull);
        // the row's logits of tile `tile` that `thread` had, one a lane
        auto item = [&](int tile, int thread, int &at) {
            at = (tile * (kLpThreads * V) + lane / E * kLpThreads + thread) * E - shift + lane % E;
            return at >= 0 && at < a.n ? to_f(x[at]) : -INFINITY;
        };
        lp_key_t tau = sm.tau;
        const float bound = tau ? lp_value(tau) : -INFINITY;
        for (int r = 0; r < records; ++r) {
            const float mx = sm.rec[r][tid];
            if (mx >= bound && mx > -INFINITY) {
                const int slot = atomicAdd(&sm.pairs, 1);
                if (slot < kLpPairs) sm.pair[slot] = (uint16_t)(r * kLpThreads + tid);
            }
        }
        __syncthreads();
        int pairs = sm.pairs;
        if (pairs <= kLpPairs) {
            for (int p = warp; p < pairs; p += kLpThreads / 32) {
                const int r = sm.pair[p] / kLpThreads, thread = sm.pair[p] % kLpThreads;
                for (int tile = t0 + r * R; tile < min(t0 + (r + 1) * R, t1); ++tile) {
                    int at;
                    const float y = item(tile, thread, at);
                    if (y >= bound && y > -INFINITY) {
                        const int slot = atomicAdd(&sm.count, 1);
                        if (slot < kLpCap) sm.cand[slot] = lp_key(y, at);
                    }
                }
            }
            __syncthreads();
        }
        if (pairs > kLpPairs || sm.count > kLpCap) {
            // tile by tile
            __syncthreads();
            if (tid == 0) sm.count = 0;
            for (int tile = t0; tile < t1; ++tile) {
                lp_key_t mine = 0;
                for (int v = 0; v < V; ++v)
                    for (int e = 0; e < E; ++e) {
                        const int at = (tile * (kLpThreads * V) + v * kLpThreads + tid) * E - shift + e;
                        const float y = at >= 0 && at < a.n ? to_f(x[at]) : -INFINITY;
                        if (y > -INFINITY) mine = max(mine, lp_key(y, at));
                    }
                lp_key_t g = max(mine, __shfl_xor_sync(0xffffffffu, mine, 1));
                g = max(g, __shfl_xor_sync(0xffffffffu, g, 2));
                if ((tid & 3) == 0) sm.group[tid >> 2] = g;
                __syncthreads();
                lp_raise(sm, k, ~0ull);
                unsigned left = mine && mine >= sm.tau ? ~0u : 0u;  // logits not dealt with
                for (;;) {
                    tau = sm.tau;
                    if (left)
                        for (int i = 0; i < kLpItems; ++i) {
                            if (!(left >> i & 1)) continue;
                            const int at = (tile * (kLpThreads * V) + i / E * kLpThreads + tid) * E - shift + i % E;
                            const float y = at >= 0 && at < a.n ? to_f(x[at]) : -INFINITY;
                            const lp_key_t key = y > -INFINITY ? lp_key(y, at) : 0;
                            const int slot = key && key >= tau ? atomicAdd(&sm.count, 1) : 0;
                            if (slot >= kLpCap) continue;
                            if (key && key >= tau) sm.cand[slot] = key;
                            left &= ~(1u << i);
                        }
                    const bool more = __syncthreads_or(left != 0);
                    const int n = min(sm.count, kLpCap);
                    lp_select(sm.cand, n, k, sm.best);
                    if (tid < k) sm.cand[tid] = sm.best[tid];
                    if (tid == 0) {
                        sm.count = min(n, k);
                        if (n >= k && sm.best[k - 1] > sm.tau) sm.tau = sm.best[k - 1];
                    }
                    __syncthreads();
                    if (!more) break;
                }
            }
        }
    }

    // join the threads, the warps, then the cluster's CTAs
    lp_join_lanes(s, 32);
    if (lane == 0) sm.warp[warp] = s;
    __syncthreads();
    if (k) lp_select(sm.cand, min(sm.count, kLpCap), k, sm.best);
    if (cs > 1) cluster_wait();
    if (warp == 0) {
        s = sm.warp[lane % (kLpThreads / 32)];
        lp_join_lanes(s, kLpThreads / 32);
        if (lane == 0) {
            if (cs > 1) st_cluster(in_cta(&sm.row[rank], 0), make_float4(s.m, s.c, s.d, s.t));
            else sm.row[0] = s;
        }
    }
    if (cs > 1) {
        if (tid < k) {
            const float2 w = *reinterpret_cast<const float2 *>(&sm.best[tid]);
            st_cluster(in_cta(&sm.top[rank][tid], 0), w.x, w.y);
        }
        cluster_arrive();
        cluster_wait();
        if (rank) return;
        if (warp == 0) {
            s = lane < cs ? sm.row[lane] : LpSums();
            lp_join_lanes(s, kMaxCluster);
            // k keys of one CTA reach its last one: smaller ones are none of the row's
            lp_key_t last = k && lane < cs ? sm.top[lane][k - 1] : 0;
#pragma unroll
            for (int o = kMaxCluster / 2; o > 0; o >>= 1) last = max(last, __shfl_xor_sync(0xffffffffu, last, o));
            __syncwarp();
            if (lane == 0) {
                sm.row[0] = s;
                sm.tau = last;
                sm.count = 0;
            }
        }
        __syncthreads();
        if (k) {
            for (int i = tid; i < cs * k; i += kLpThreads) {
                const lp_key_t key = sm.top[i / k][i % k];
                if (key && key >= sm.tau) sm.cand[atomicAdd(&sm.count, 1)] = key;
            }
            __syncthreads();
            lp_select(sm.cand, sm.count, k, sm.best);
        }
    } else {
        __syncthreads();
    }
    s = sm.row[0];
    if (s.m == INFINITY) s.d = NAN;
    const bool none = s.m == -INFINITY && s.d == 0.f;  // every token masked (a NaN reaches d)
    const float M = s.m == -INFINITY ? 0.f : s.m;
    const float ls = logf(s.c) + log1pf(s.d / s.c);
    if (tid == 0) {
        const int y = a.targets ? a.targets[row] : -1;
        if (a.logprob) a.logprob[row] = y < 0 || y >= a.n ? NAN : none ? -INFINITY : (to_f(x[y]) - M) - ls;
        if (a.entropy) a.entropy[row] = none ? 0.f : ls - s.t / (s.c + s.d);
    }
    if (k == 0) return;
    const lp_key_t key = tid < k ? sm.best[tid] : 1;
    if (key && tid < k) {
        a.top_ids[row * k + tid] = (int)~(unsigned)key;
        a.top_logprob[row * k + tid] = (lp_value(key) - M) - ls;
    }
    const int have = k - __syncthreads_count(key == 0);
    if (have < k) lp_fill(x, a.n, have, k, a.top_ids + row * k, a.top_logprob + row * k, sm.fill);
    if (s.d != s.d && tid >= have && tid < k) a.top_logprob[row * k + tid] = NAN;
}

template <int TYPE>
static cudaError_t lp_launch(const LogprobArgs &a, int cs_log2, cudaStream_t st) {
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 1u << cs_log2;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)a.rows << cs_log2);
    cfg.blockDim = dim3(kLpThreads);
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = cs_log2 > 0 ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, logprobs_kernel<TYPE>, a, cs_log2);
}

cudaError_t launch_logprobs(const LogprobArgs &a, cudaStream_t st) {
    if (a.rows == 0) return cudaSuccess;
    static std::atomic<int> sms_of[64];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= 64) return cudaErrorInvalidDevice;
    int sms = sms_of[dev].load(std::memory_order_acquire);
    if (!sms) {
        if ((e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev))) return e;
        for (auto f : {logprobs_kernel<OT_F32>, logprobs_kernel<OT_F16>, logprobs_kernel<OT_BF16>})
            if ((e = cudaFuncSetAttribute(f, cudaFuncAttributeNonPortableClusterSizeAllowed, 1))) return e;
        sms_of[dev].store(sms, std::memory_order_release);
    }
    // CTAs per row: one where the rows fill the device (512 rows of 155648 f32 logits: 65.6 us, 81.9 in halves), else
    // as many as fit at once, each with a tile at least
    int cs = 0;
    while (cs < 4 && ((long long)a.rows << (cs + 1)) <= 2LL * sms && a.n > kLpTile << cs) ++cs;
    count_launch();
    switch (a.type) {
        case OT_F32: return lp_launch<OT_F32>(a, cs, st);
        case OT_F16: return lp_launch<OT_F16>(a, cs, st);
        case OT_BF16: return lp_launch<OT_BF16>(a, cs, st);
        default: return cudaErrorInvalidValue;
    }
}

}  // namespace s2k
