// kv8.cuh -- what the files of the paged 8-bit cache share: the record of a page, rows of activations of three types, the step's sequences.
#pragma once
#include "../../include/b200_kv8.h"
#include "ops_util.cuh"
#include <cuda_bf16.h>

namespace b200 {
namespace kv8 {

// offsets within a page's record
__host__ __device__ inline size_t v_at(const b200_kv8_cache &c) { return (size_t)c.n_head_kv * c.page_size * c.dim; }
__host__ __device__ inline size_t scales_at(const b200_kv8_cache &c) { return (size_t)c.n_head_kv * c.page_size * (c.dim + c.vdim); }
__host__ __device__ inline size_t record_bytes(const b200_kv8_cache &c) { return (scales_at(c) + (size_t)c.n_head_kv * 8 + 127) / 128 * 128; }

struct Step {  // a step's sequences and the table, as kernels take them
    const int32_t *info, *table;
    int64_t table_stride;
    int32_t n_rows, n_seq, n_tokens, n_pages, page_size;
};
struct Seq { int first, count, row, held; };
// sequence s as far as it can be: a row that is none, or tokens outside the batch, leave a count of 0
__device__ __forceinline__ Seq seq_of(const Step &st, const int32_t *info, int s) {
    Seq q = {info[s], info[st.n_seq + s], info[2 * st.n_seq + s], info[3 * st.n_seq + s]};
    const bool none = q.first < 0 || q.first >= st.n_tokens || q.row < 0 || q.row >= st.n_rows || q.held < 0 || q.count < 0;
    if (none) q.first = q.held = 0;
    q.count = none ? 0 : min(q.count, min(st.n_tokens - q.first, 0x7fffffff - q.held));
    return q;
}
// page number `at` of a row, or -1
__device__ __forceinline__ int page_of(const Step &st, const int32_t *table, int row, int at) {
    if (at >= st.table_stride) return -1;
    const int p = table[(int64_t)row * st.table_stride + at];
    return p >= 0 && p < st.n_pages ? p : -1;
}
// The last sequence s with begin(its first token, s) <= j, and what is known of it, by a whole warp (begin does not fall with s; sequence 0 begins at or below j): 32 of them at a
// time, the last 32 with all that a step says of them.
template <typename F>
__device__ __forceinline__ Seq find_seq(const Step &st, const int32_t *info, int j, int &s, F begin) {
    const int lane = threadIdx.x & 31, n_seq = st.n_seq;
    int lo = 0, n = n_seq;  // the answer is in [lo, lo + n)
    while (n > 32) {
        const int step = (n + 31) / 32, at = lo + lane * step;
        const unsigned yes = __ballot_sync(0xffffffffu, lane * step < n && begin(info[min(at, n_seq - 1)], at) <= j);
        const int k = yes ? 31 - __clz(yes) : 0;
        lo += k * step;
        n = min(step, n - k * step);
    }
    const int at = min(lo + lane, n_seq - 1);
    Seq q = seq_of(st, info, at);
    const int first = info[at];
    const unsigned yes = __ballot_sync(0xffffffffu, lane < n && begin(first, lo + lane) <= j);
    const int k = yes ? 31 - __clz(yes) : 0;
    s = lo + k;
    return Seq{__shfl_sync(0xffffffffu, q.first, k), __shfl_sync(0xffffffffu, q.count, k), __shfl_sync(0xffffffffu, q.row, k), __shfl_sync(0xffffffffu, q.held, k)};
}

// 16 consecutive values of a row as they lie there, without a conversion; VEC: the row's pieces of 16 values are 16-byte aligned
template <typename T> struct Raw16 { uint4 u[sizeof(T)]; };
template <typename T, bool VEC>
__device__ __forceinline__ void load_raw16(const T *p, Raw16<T> &r) {
    if constexpr (VEC) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T); i++) r.u[i] = reinterpret_cast<const uint4 *>(p)[i];
    } else {
        __align__(16) T v[16];
#pragma unroll
        for (int i = 0; i < 16; i++) v[i] = p[i];
#pragma unroll
        for (int i = 0; i < (int)sizeof(T); i++) r.u[i] = reinterpret_cast<const uint4 *>(v)[i];
    }
}
template <typename T>
__device__ __forceinline__ float raw_value(const Raw16<T> &r, int i) {  // (i known when compiled)
    const uint4 u = r.u[i * (int)sizeof(T) / 16];
    const int word = i * (int)sizeof(T) / 4 % 4;
    const unsigned w = word == 0 ? u.x : word == 1 ? u.y : word == 2 ? u.z : u.w;
    if constexpr (sizeof(T) == 4) return __uint_as_float(w);
    else if constexpr (std::is_same<T, __half>::value) return h2f((unsigned short)(w >> (16 * (i & 1))));
    else return __uint_as_float(i & 1 ? w & 0xffff0000u : w << 16);
}

// 16 consecutive values of a row of activations as f32; VEC: the row's pieces of 16 values are 16-byte aligned
template <typename T, bool VEC>
__device__ __forceinline__ void load16(const T *p, float (&x)[16]) {
    if constexpr (!VEC) {
#pragma unroll
        for (int i = 0; i < 16; i++) {
            if constexpr (sizeof(T) == 4) x[i] = p[i];
            else if constexpr (std::is_same<T, __half>::value) x[i] = __half2float(p[i]);
            else x[i] = __bfloat162float(p[i]);
        }
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float4 f = *reinterpret_cast<const float4 *>(p + 4 * i);
            x[4 * i] = f.x; x[4 * i + 1] = f.y; x[4 * i + 2] = f.z; x[4 * i + 3] = f.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const uint4 u = *reinterpret_cast<const uint4 *>(p + 8 * i);
            const unsigned w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int j = 0; j < 4; j++) {
                if constexpr (std::is_same<T, __half>::value) {
                    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[j]));
                    x[8 * i + 2 * j] = f.x; x[8 * i + 2 * j + 1] = f.y;
                } else {
                    x[8 * i + 2 * j] = __uint_as_float(w[j] << 16);
                    x[8 * i + 2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
                }
            }
        }
    }
}
template <typename T> __device__ __forceinline__ T to_row(float x) {
    if constexpr (sizeof(T) == 4) return x;
    else if constexpr (std::is_same<T, __half>::value) return __float2half_rn(x);
    else return __float2bfloat16_rn(x);
}
template <typename T, bool VEC>
__device__ __forceinline__ void store16(T *p, const float (&x)[16]) {
    if constexpr (!VEC) {
#pragma unroll
        for (int i = 0; i < 16; i++) p[i] = to_row<T>(x[i]);
    } else {
        constexpr int N = 16 / sizeof(T);  // values of 16 bytes
#pragma unroll
        for (int i = 0; i < 16 / N; i++) {
            __align__(16) T v[N];
#pragma unroll
            for (int j = 0; j < N; j++) v[j] = to_row<T>(x[N * i + j]);
            *reinterpret_cast<uint4 *>(p + N * i) = *reinterpret_cast<const uint4 *>(v);
        }
    }
}

// ---------------------------------------------------------------- host side
inline bool type_ok(int t) { return t == B200_TYPE_F32 || t == B200_TYPE_F16 || t == B200_TYPE_BF16; }
inline size_t type_size(int t) { return t == B200_TYPE_F32 ? 4 : 2; }
// rows whose pieces of 16 bytes all begin on 16 bytes
inline bool rows_aligned(const void *p, int64_t stride, int type) { return (uintptr_t)p % 16 == 0 && stride * (int64_t)type_size(type) % 16 == 0; }
// pointers to values of so many bytes (NULL too)
inline bool aligned_to(size_t size, const void *a, const void *b = nullptr, const void *c = nullptr) { return ((uintptr_t)a | (uintptr_t)b | (uintptr_t)c) % size == 0; }
int check_cache(const b200_kv8_cache *c, const char *who);
int check_step(const b200_kv8_cache *c, const int32_t *seq_info, const int32_t *table, int64_t table_stride, int32_t n_rows, int32_t n_seq, int32_t n_tokens, int32_t type, const char *who);

}  // namespace kv8
}  // namespace b200
