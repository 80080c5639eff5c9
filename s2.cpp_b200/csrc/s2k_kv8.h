// s2k_kv8.h -- the 8-bit paged KV cache as its kernels see it, and the
// launchers of its operators (internal).
//
// A page holds 16 tokens of every (layer, kv head): keys as int8
// [16][head_dim], values transposed as int8 [head_dim][16], and one f32 scale
// for each of the two.  A value stands for q * scale, q in [-127, 127].
// Values are transposed because the product with the weights sums over
// tokens: four tokens of one dimension are then one aligned 4-byte word, the
// operand the tensor cores take.
#pragma once

#include "s2k_common.cuh"
#include "s2k_kernels.h"

#include <cuda_bf16.h>
#include <stdint.h>
#include <type_traits>

namespace s2k {

// Element types of operator tensors (S2K_TYPE_F32 / F16 / BF16).
enum : int { OT_F32 = 0, OT_F16 = 1, OT_BF16 = 30 };

struct Kv8 {
    int8_t *k = nullptr, *v = nullptr;
    float *k_scale = nullptr, *v_scale = nullptr;  // [page][layer][kv_head]
    int n_pages = 0, n_layers = 0, n_kv_heads = 0, head_dim = 0;
    int layer = 0;
    // (page, layer, kv head) block: index of its scale; its int8 values start
    // at index * 16 * head_dim
    __host__ __device__ size_t block(int page, int head) const {
        return ((size_t)page * n_layers + layer) * n_kv_heads + head;
    }
};

// The rows of a call: sequence b owns rows [row0, row0 + T) at positions
// past[b] .. past[b] + T - 1 and the pages table[b][*].
struct Kv8Rows {
    int n_seqs = 0, n_rows = 0, max_rows = 0, table_ld = 0;
    const int *past = nullptr;       // [n_seqs]
    const int *row_start = nullptr;  // [n_seqs + 1], null: max_rows rows each
    const int *table = nullptr;      // [n_seqs][table_ld]
    int *err = nullptr;              // optional error word
    int *block = nullptr;            // a model's error block (its wait limit), where the call is one of a model's
    const int *done = nullptr;       // optional: nothing is done once it is set (frame loop)
};

struct Rows {
    void *p = nullptr;
    int type = OT_F32;
    long long row_stride = 0, head_stride = 0;  // elements
};

#ifdef __CUDACC__
// Sequence b's rows, false (and an error bit) when what the device arrays say
// does not fit the call: nothing of that sequence is then read or written.
__device__ __forceinline__ bool kv8_seq(const Kv8Rows &r, int b, int &row0, int &T, int &past) {
    if (r.done && __ldcg(r.done)) return false;
    row0 = r.row_start ? r.row_start[b] : b * r.max_rows;
    T = r.row_start ? r.row_start[b + 1] - row0 : r.max_rows;
    past = r.past[b];
    const bool ok = T >= 0 && T <= r.max_rows && row0 >= 0 && row0 <= r.n_rows - T && past >= 0 &&
                    past <= r.table_ld * kPage - T;
    if (!ok && r.err && threadIdx.x == 0) atomicOr(r.err, ERR_BAD_POS);
    return ok;
}

// Bounded wait on an mbarrier phase; the caller's error word has no wait limit behind it, a model's block does.
__device__ __forceinline__ bool kv8_wait(const Kv8Rows &r, uint64_t *bar, uint32_t parity, int code) {
    if (mbar_wait(bar, parity, r.block, code)) return true;
    if (r.err) atomicOr(r.err, code);
    return false;
}

// Physical page of logical page pg, -1 (and an error bit) when the table
// names none of the cache's pages.
__device__ __forceinline__ int kv8_page(const Kv8 &c, const Kv8Rows &r, int b, int pg) {
    const int p = r.table[(size_t)b * r.table_ld + pg];
    if ((unsigned)p < (unsigned)c.n_pages) return p;
    if (r.err) atomicOr(r.err, ERR_BAD_POS);
    return -1;
}

template <int TYPE>
struct OType {
    using T = float;
};
template <>
struct OType<OT_F16> {
    using T = __half;
};
template <>
struct OType<OT_BF16> {
    using T = __nv_bfloat16;
};
__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
template <class T>
__device__ __forceinline__ T from_f(float x);
template <>
__device__ __forceinline__ float from_f<float>(float x) {
    return x;
}
template <>
__device__ __forceinline__ __half from_f<__half>(float x) {
    return __float2half_rn(x);
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float x) {
    return __float2bfloat16_rn(x);
}

// 2^x; subnormal results are zero
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// 16 bytes global -> shared, past L1
__device__ __forceinline__ void cp16(void *dst, const void *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// all but the last N groups of this thread have arrived
template <int N>
__device__ __forceinline__ void cp_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Most CTAs of a cluster that the operators use (more than 8 is opt-in).
constexpr int kMaxCluster = 16;

// The cluster's barrier in two halves: memory before the arrival is seen after the wait.
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// Address of `p` of this CTA's shared memory in CTA `rank` of the cluster, and stores to it.
__device__ __forceinline__ uint32_t in_cta(const void *p, uint32_t rank) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
    return a;
}
__device__ __forceinline__ void st_cluster(uint32_t a, float x, float y) {
    asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(a), "f"(x), "f"(y) : "memory");
}
__device__ __forceinline__ void st_cluster(uint32_t a, float x) {
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(a), "f"(x) : "memory");
}
__device__ __forceinline__ void st_cluster(uint32_t a, float4 v) {
    asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(a), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w)
                 : "memory");
}

// (a, b) += m * (x, y) as packed f32 pairs
__device__ __forceinline__ void fma2(float (&o)[2], float m, float x, float y) {
    asm("{\n\t.reg .b64 d, a, b;\n\tmov.b64 d, {%0, %1};\n\tmov.b64 a, {%2, %2};\n\tmov.b64 b, {%3, %4};\n\t"
        "fma.rn.f32x2 d, a, b, d;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "+f"(o[0]), "+f"(o[1])
        : "f"(m), "f"(x), "f"(y));
}
__device__ __forceinline__ void mul2(float (&o)[2], float m) {
    asm("{\n\t.reg .b64 d, a;\n\tmov.b64 d, {%0, %1};\n\tmov.b64 a, {%2, %2};\n\tmul.rn.f32x2 d, d, a;\n\t"
        "mov.b64 {%0, %1}, d;\n\t}"
        : "+f"(o[0]), "+f"(o[1])
        : "f"(m));
}
__device__ __forceinline__ void add2(float &x, float &y, float v) {
    asm("{\n\t.reg .b64 d, a;\n\tmov.b64 d, {%0, %1};\n\tmov.b64 a, {%2, %2};\n\tadd.rn.f32x2 d, d, a;\n\t"
        "mov.b64 {%0, %1}, d;\n\t}"
        : "+f"(x), "+f"(y)
        : "f"(v));
}

template <class T, int N>
struct alignas(sizeof(T) * N) Vec {
    T v[N];
};

// Eight elements from 16-byte aligned memory, 16 bytes an access.
template <class T>
__device__ __forceinline__ void load_raw(const T *p, Vec<T, 8> &x) {
    constexpr int E = 16 / sizeof(T);
#pragma unroll
    for (int i = 0; i < 8 / E; ++i)
        *reinterpret_cast<Vec<T, E> *>(&x.v[i * E]) = *reinterpret_cast<const Vec<T, E> *>(p + i * E);
}

// N consecutive elements, as one access where the rows' alignment allows it
// (vec: base and strides are multiples of N elements).
template <int N, class T>
__device__ __forceinline__ void load_n(const T *p, bool vec, float (&x)[N]) {
    if (vec) {
        const Vec<T, N> u = *reinterpret_cast<const Vec<T, N> *>(p);
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = to_f(u.v[i]);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = to_f(p[i]);
    }
}
template <int N, class T>
__device__ __forceinline__ void store_n(T *p, bool vec, const float (&x)[N]) {
    if (vec) {
        Vec<T, N> u;
#pragma unroll
        for (int i = 0; i < N; ++i) u.v[i] = from_f<T>(x[i]);
        *reinterpret_cast<Vec<T, N> *>(p) = u;
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) p[i] = from_f<T>(x[i]);
    }
}
#endif

// Whether rows of `t` may be accessed n elements at a time.
inline bool rows_vec(const Rows &t, int n) {
    const int es = t.type == OT_F32 ? 4 : 2;
    return (uintptr_t)t.p % (size_t)(n * es) == 0 && t.row_stride % n == 0 && t.head_stride % n == 0;
}

// f(head_dim, type) as constants
template <class F>
cudaError_t kv8_dispatch(int hd, int type, F f) {
    switch (hd * 100 + type) {
        case 12800 + OT_F32: return f(std::integral_constant<int, 128>(), std::integral_constant<int, OT_F32>());
        case 12800 + OT_F16: return f(std::integral_constant<int, 128>(), std::integral_constant<int, OT_F16>());
        case 12800 + OT_BF16: return f(std::integral_constant<int, 128>(), std::integral_constant<int, OT_BF16>());
        case 6400 + OT_F32: return f(std::integral_constant<int, 64>(), std::integral_constant<int, OT_F32>());
        case 6400 + OT_F16: return f(std::integral_constant<int, 64>(), std::integral_constant<int, OT_F16>());
        case 6400 + OT_BF16: return f(std::integral_constant<int, 64>(), std::integral_constant<int, OT_BF16>());
        default: return cudaErrorInvalidValue;
    }
}

struct Kv8Attn {
    Rows q, out;
    int n_heads = 0;
    float scale = 1.f;
    int window = 0, sinks = 0;
};

cudaError_t launch_kv8_append(const Kv8 &c, const Kv8Rows &r, const Rows &k, const Rows &v, cudaStream_t st);
cudaError_t launch_kv8_read(const Kv8 &c, const Kv8Rows &r, const Rows &k, const Rows &v, cudaStream_t st);
// slots of a CTA of the prompt kernel
constexpr int kv8_prompt_slots(int type) { return type == OT_F32 ? 128 : 256; }
cudaError_t launch_kv8_attend(const Kv8 &c, const Kv8Rows &r, const Kv8Attn &a, cudaStream_t st);

// this thread's last launch_kv8_attend: 1 the kernel of few rows, 2 that of many
extern thread_local int g_kv8_attend_kernel;

// the same for calls of many rows per sequence
cudaError_t launch_kv8_prompt(const Kv8 &c, const Kv8Rows &r, const Kv8Attn &a, cudaStream_t st);

struct LogprobArgs {
    const void *x = nullptr;
    int type = OT_F32;
    int rows = 0, n = 0;
    long long ld = 0;
    const int *targets = nullptr;
    int n_top = 0;
    float *logprob = nullptr, *entropy = nullptr;
    int *top_ids = nullptr;
    float *top_logprob = nullptr;
};
cudaError_t launch_logprobs(const LogprobArgs &a, cudaStream_t st);

}  // namespace s2k
