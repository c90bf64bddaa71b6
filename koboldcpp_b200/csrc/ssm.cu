// ssm.cu -- selective state space scan and the short causal convolution in front of it (include/b200_state.h: b200_op_ssm_conv, b200_op_ssm_scan).  A batch names its sequences
// through seq_info (first row, count, state slot, begins) like the mixers of recur.cu; rows are f32, f16 or bf16, states and sums f32.
// Semantics of the reference's form (all sequences of one length, f32): ggml_compute_forward_ssm_conv_f32 / _ssm_scan_f32, ggml.c.
#include <cuda_bf16.h>

#include "../../include/b200_state.h"
#include "ops_util.cuh"

namespace b200 {
namespace ssm {

struct Seq { int first, count, slot; bool begins; };
// what a step's sequences are made of, as kernels take it
struct Step {
    const int32_t *info;
    int32_t n_seq, n_slots, n_tokens, max_new;
};
// sequence s as far as it can be: a slot that is none, or rows outside the batch, leave a count of 0
__device__ __forceinline__ Seq seq_of(const Step &st, int s) {
    if (!st.info) {
        const int each = st.n_tokens / st.n_seq;
        return {s * each, min(each, st.max_new), s, false};
    }
    Seq q = {st.info[s], st.info[st.n_seq + s], st.info[2 * st.n_seq + s], st.info[3 * st.n_seq + s] != 0};
    if (q.first < 0 || q.first >= st.n_tokens || q.slot < 0 || q.slot >= st.n_slots || q.count < 0) q.count = 0;
    else q.count = min(min(q.count, st.max_new), st.n_tokens - q.first);
    return q;
}

template <typename T> __device__ __forceinline__ float wide(T x) {
    if constexpr (sizeof(T) == 4) return x;
    else if constexpr (std::is_same<T, __half>::value) return __half2float(x);
    else return __bfloat162float(x);
}
template <typename T> __device__ __forceinline__ T narrow(float x) {
    if constexpr (sizeof(T) == 4) return x;
    else if constexpr (std::is_same<T, __half>::value) return __float2half_rn(x);
    else return __float2bfloat16_rn(x);
}
// V consecutive values, in one access where they lie on a boundary of their size
template <typename T, int V> struct __align__(sizeof(T) * V) Pack { T v[V]; };

// y * sigmoid(y); one exponential and one reciprocal of the special function unit (2^-22 each)
__device__ __forceinline__ float silu(float y) { return __fdividef(y, 1.0f + __expf(-y)); }

// ------------------------------------------------------------------------------------------------ short convolution
// A thread takes V channels of CONV_ROWS rows of one sequence and keeps the last K - 1 inputs in registers.  The CTAs that hold a sequence's first rows read its tail, and they alone
// write it (each channel by one thread), so that nobody reads what another has rewritten.  K: taps, or the next of 8 and 16, whose products of taps that are not there are left out.
constexpr int CONV_ROWS = 16, CONV_AHEAD = 8, CONV_THREADS = 128;
struct ConvArgs {
    Step step;
    const void *x; int64_t x_stride;
    const float *w, *bias;
    float *tail; int64_t slot_stride;
    void *dst; int64_t dst_stride;
    int32_t channels, taps, silu;
};
template <typename T, int K, int V, bool EXACT>
__global__ void __launch_bounds__(CONV_THREADS) ssm_conv_kernel(const ConvArgs a) {
    pdl_enter();
    const int c = (blockIdx.x * CONV_THREADS + threadIdx.x) * V, t0 = blockIdx.y * CONV_ROWS;
    const Seq q = seq_of(a.step, blockIdx.z);
    if (c >= a.channels || t0 >= q.count) return;
    const int nt = min(CONV_ROWS, q.count - t0), skip = EXACT ? 0 : K - a.taps;  // taps that are not there
    const T *x = (const T *)a.x + (int64_t)q.first * a.x_stride + c;
    float *tail = a.tail + (int64_t)q.slot * a.slot_stride + c;
    using P = Pack<T, V>;
    float w[K][V], bias[V], win[K][V];  // win[K - 1]: the newest input
#pragma unroll
    for (int e = 0; e < V; e++) {
        bias[e] = a.bias ? a.bias[c + e] : 0.f;
#pragma unroll
        for (int j = 0; j < K; j++) w[j][e] = EXACT || j >= skip ? a.w[(int64_t)(c + e) * a.taps + j - skip] : 0.f;
    }
#pragma unroll
    for (int j = 1; j < K; j++) {  // win[j]: the input of row t0 - K + j
        const int i = t0 - K + j;
        if (i >= 0) {
            const P p = *reinterpret_cast<const P *>(x + (int64_t)i * a.x_stride);
#pragma unroll
            for (int e = 0; e < V; e++) win[j][e] = wide(p.v[e]);
        } else {
            const int at = a.taps - 1 + i;
#pragma unroll
            for (int e = 0; e < V; e++) win[j][e] = at >= 0 && !q.begins ? tail[(int64_t)at * a.channels + e] : 0.f;
        }
    }
    T *dst = (T *)a.dst + (int64_t)(q.first + t0) * a.dst_stride + c;
    x += (int64_t)t0 * a.x_stride;
    for (int b = 0; b < nt; b += CONV_AHEAD) {
        P in[CONV_AHEAD];
#pragma unroll
        for (int u = 0; u < CONV_AHEAD; u++) {
            if (b + u < nt) in[u] = *reinterpret_cast<const P *>(x + (int64_t)(b + u) * a.x_stride);
        }
#pragma unroll
        for (int u = 0; u < CONV_AHEAD; u++) {
            if (b + u >= nt) break;
            P out;
#pragma unroll
            for (int e = 0; e < V; e++) {
#pragma unroll
                for (int j = 0; j < K - 1; j++) win[j][e] = win[j + 1][e];
                win[K - 1][e] = wide(in[u].v[e]);
                float y = bias[e];
#pragma unroll
                for (int j = 0; j < K; j++) if (EXACT || j >= skip) y = fmaf(w[j][e], win[j][e], y);
                out.v[e] = narrow<T>(a.silu ? silu(y) : y);
            }
            *reinterpret_cast<P *>(dst + (int64_t)(b + u) * a.dst_stride) = out;
        }
    }
    if (t0 == 0) {
        // entry j of the new tail is the input of row count - taps + 1 + j: all of them are in the window, or behind the rows of this CTA
#pragma unroll
        for (int j = 1; j < K; j++) {
            if (!EXACT && j <= skip) continue;
            const int i = q.count - K + j;
            float *to = tail + (int64_t)(j - 1 - skip) * a.channels;
            if (q.count <= CONV_ROWS) {
#pragma unroll
                for (int e = 0; e < V; e++) to[e] = win[j][e];
            } else {
                const P p = *reinterpret_cast<const P *>(x + (int64_t)i * a.x_stride);
#pragma unroll
                for (int e = 0; e < V; e++) to[e] = wide(p.v[e]);
            }
        }
    }
}
static_assert(CONV_ROWS >= 15, "a sequence of more rows than a CTA takes has all the new tail's inputs among its rows");

template <typename T, int K, int V, bool EXACT>
static int launch_conv(const ConvArgs &a, cudaStream_t st) {
    const int each = CONV_THREADS * V;
    const dim3 grid((unsigned)((a.channels + each - 1) / each), (unsigned)((a.step.max_new + CONV_ROWS - 1) / CONV_ROWS), (unsigned)a.step.n_seq);
    B200_CUDA_TRY(launch_chained(ssm_conv_kernel<T, K, V, EXACT>, grid, CONV_THREADS, 0, st, a));
    return B200_OK;
}
template <typename T, int V>
static int launch_conv_taps(const ConvArgs &a, cudaStream_t st) {
    switch (a.taps) {
        case 1: return launch_conv<T, 1, V, true>(a, st);
        case 2: return launch_conv<T, 2, V, true>(a, st);
        case 3: return launch_conv<T, 3, V, true>(a, st);
        case 4: return launch_conv<T, 4, V, true>(a, st);
        default: return a.taps <= 8 ? launch_conv<T, 8, V < 4 ? V : 4, false>(a, st) : launch_conv<T, 16, V < 2 ? V : 2, false>(a, st);
    }
}

// ------------------------------------------------------------------------------------------------ scan
struct ScanArgs {
    Step step;
    const void *x, *dt, *b, *c, *z;
    int64_t x_stride, dt_stride, b_stride, c_stride, z_stride;
    const float *a, *dt_bias, *d;
    const float *from; int64_t from_stride;
    float *state; int64_t slot_stride;
    void *dst; int64_t dst_stride;
    int32_t channels, d_state, per_group, softplus;
    // stretches: rows of one, how many a sequence may have; where their end states and sums of d wait
    int32_t stretch, n_stretch;
    float *ends, *sums;
};

constexpr float LOG2E = 1.4426950408889634f;
__device__ __forceinline__ float ex2(float x) { float r; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x)); return r; }
// ln(1 + e^x) without overflow for large x and without cancellation for very negative x
__device__ __forceinline__ float softplus(float x) { return fmaxf(x, 0.f) + log1pf(__expf(-fabsf(x))); }

// Four neighbouring states of a channel; numbers behind d_state count as zeros
template <bool VEC>
__device__ __forceinline__ float4 load_states(const float *row, int n0, int d_state) {
    if constexpr (VEC) return n0 < d_state ? *reinterpret_cast<const float4 *>(row + n0) : make_float4(0.f, 0.f, 0.f, 0.f);
    float4 r;
    r.x = n0 < d_state ? row[n0] : 0.f;
    r.y = n0 + 1 < d_state ? row[n0 + 1] : 0.f;
    r.z = n0 + 2 < d_state ? row[n0 + 2] : 0.f;
    r.w = n0 + 3 < d_state ? row[n0 + 3] : 0.f;
    return r;
}
template <bool VEC>
__device__ __forceinline__ void store_states(float *row, int n0, int d_state, float4 v) {
    if constexpr (VEC) {
        if (n0 < d_state) *reinterpret_cast<float4 *>(row + n0) = v;
    } else {
        if (n0 < d_state) row[n0] = v.x;
        if (n0 + 1 < d_state) row[n0 + 1] = v.y;
        if (n0 + 2 < d_state) row[n0 + 2] = v.z;
        if (n0 + 3 < d_state) row[n0 + 3] = v.w;
    }
}
template <typename T>
__device__ __forceinline__ float4 load_row4(const T *row, int n0, int d_state) {
    float4 r;
    r.x = n0 < d_state ? wide(row[n0]) : 0.f;
    r.y = n0 + 1 < d_state ? wide(row[n0 + 1]) : 0.f;
    r.z = n0 + 2 < d_state ? wide(row[n0 + 2]) : 0.f;
    r.w = n0 + 3 < d_state ? wide(row[n0 + 3]) : 0.f;
    return r;
}

// ===== one row a sequence.  A warp takes 32 channels; L lanes share a channel, a lane four of its states, so that a load of the warp is 512 consecutive bytes of the state.  What a channel
// needs by itself (d, d x, z) is made by one lane and handed to the other L - 1; the sums of L channels are exchanged so that each lane ends up with one of them.
constexpr int STEP_WARPS = 2;
template <typename T, int L, bool VEC>
__global__ void __launch_bounds__(32 * STEP_WARPS) ssm_step_kernel(const ScanArgs a) {
    constexpr int G = 32 / L, U = L < 4 ? L : 4;  // channels of a round; rounds whose loads travel together
    pdl_enter();
    const int lane = threadIdx.x & 31, p = lane % L, g = lane / L;
    const int c0 = (blockIdx.x * STEP_WARPS + (threadIdx.x >> 5)) * 32;
    const Seq q = seq_of(a.step, blockIdx.y);
    if (c0 >= a.channels || q.count == 0) return;
    const int64_t row = q.first;
    const int mine = c0 + G * p + g;  // the channel that is this lane's by itself
    const bool ok = mine < a.channels;
    float d = 0.f, x = 0.f;
    if (ok) {
        d = wide(((const T *)a.dt)[row * a.dt_stride + mine]) + (a.dt_bias ? a.dt_bias[mine] : 0.f);
        x = wide(((const T *)a.x)[row * a.x_stride + mine]);
        if (a.softplus) d = softplus(d);
    }
    const float dx = d * x;
    const float *from = a.from + (int64_t)q.slot * a.from_stride;
    float *state = a.state + (int64_t)q.slot * a.slot_stride;
    float sum[L];
#pragma unroll
    for (int i0 = 0; i0 < L; i0 += U) {
        float4 h[U], rate[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int c = c0 + G * (i0 + u) + g;
            h[u] = rate[u] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (c < a.channels) {
                rate[u] = load_states<VEC>(a.a + (int64_t)c * a.d_state, 4 * p, a.d_state);
                if (!q.begins) h[u] = load_states<VEC>(from + (int64_t)c * a.d_state, 4 * p, a.d_state);
            }
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int c = c0 + G * (i0 + u) + g, at = min(c, a.channels - 1) / a.per_group * a.d_state;
            const float4 b = load_row4((const T *)a.b + row * a.b_stride + at, 4 * p, a.d_state), cc = load_row4((const T *)a.c + row * a.c_stride + at, 4 * p, a.d_state);
            const float dc = LOG2E * __shfl_sync(0xffffffffu, d, g * L + i0 + u), dxc = __shfl_sync(0xffffffffu, dx, g * L + i0 + u);
            float4 s = h[u];
            s.x = fmaf(ex2(dc * rate[u].x), s.x, dxc * b.x);
            s.y = fmaf(ex2(dc * rate[u].y), s.y, dxc * b.y);
            s.z = fmaf(ex2(dc * rate[u].z), s.z, dxc * b.z);
            s.w = fmaf(ex2(dc * rate[u].w), s.w, dxc * b.w);
            if (c < a.channels) store_states<VEC>(state + (int64_t)c * a.d_state, 4 * p, a.d_state, s);
            sum[i0 + u] = fmaf(cc.x, s.x, fmaf(cc.y, s.y, fmaf(cc.z, s.z, cc.w * s.w)));
        }
    }
    // sum i of the lanes of a channel ends up in lane i of them
#pragma unroll
    for (int n = L / 2; n >= 1; n /= 2) {
        const bool upper = (p & n) != 0;
#pragma unroll
        for (int i = 0; i < n; i++) {
            const float send = upper ? sum[i] : sum[i + n], keep = upper ? sum[i + n] : sum[i];
            sum[i] = keep + __shfl_xor_sync(0xffffffffu, send, n);
        }
    }
    if (ok) {
        float y = sum[0];
        if (a.d) y = fmaf(a.d[mine], x, y);
        if (a.z) y *= silu(wide(((const T *)a.z)[row * a.z_stride + mine]));
        ((T *)a.dst)[row * a.dst_stride + mine] = narrow<T>(y);
    }
}

// ===== several rows a sequence
constexpr int SCAN_WARPS = 4, SCAN_THREADS = 32 * SCAN_WARPS;
// the three things that a CTA can be there for: a whole sequence; the state at the end of a stretch as if it began from nothing (the first one: from the sequence's state), and the sum of
// its d; a stretch's rows, from the states and sums of those before it
enum Pass { WHOLE, ENDS, ROWS };
template <typename T, int L, int CI>
struct ScanSizes {
    static constexpr int G = 32 / L, WC = G * CI, CB = SCAN_WARPS * WC, NP = 4 * L;
    static constexpr int TC = CB >= 64 ? 16 : 1024 / CB;          // rows of a chunk
    static constexpr int PIECES = TC * CB / 4 / SCAN_THREADS;     // pieces of four channels of one row that a thread stages
    static constexpr int RAW = TC * CB * (int)sizeof(T), RAW_BC = TC * NP * (int)sizeof(T);
    static constexpr int BUF = 3 * RAW + 2 * RAW_BC;              // x, dt, z, b, c as they lie in memory
    static constexpr int SMEM = 2 * BUF + 4 * (2 * TC * CB + 2 * TC * NP);
    static_assert(PIECES >= 1 && TC % 4 == 0, "every thread stages the same number of pieces");
};
template <typename T, int L, int CI, bool VEC, int PASS>
__global__ void __launch_bounds__(SCAN_THREADS) ssm_scan_kernel(const ScanArgs a) {
    using Z = ScanSizes<T, L, CI>;
    constexpr int G = Z::G, CB = Z::CB, NP = Z::NP, TC = Z::TC, C4 = CB / 4;
    extern __shared__ __align__(16) unsigned char ssm_shared[];
    pdl_enter();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, p = lane % L, g = lane / L;
    const Seq q = seq_of(a.step, blockIdx.z);
    const int N = a.d_state, blocks = (a.per_group + CB - 1) / CB, group = blockIdx.x / blocks, in_group = (blockIdx.x - group * blocks) * CB;
    const int c0 = group * a.per_group + in_group, nc = min(CB, a.per_group - in_group);  // channels of the CTA
    const int stretch = PASS == WHOLE ? 0 : blockIdx.y, begin = PASS == WHOLE ? 0 : stretch * a.stretch, end = PASS == WHOLE ? q.count : min(q.count, begin + a.stretch);
    if (begin >= end) return;
    if (PASS == ENDS && end == q.count && stretch > 0) return;  // nobody asks for the last one's
    unsigned char *raw = ssm_shared;
    float *sd = (float *)(ssm_shared + 2 * Z::BUF), *sx = sd + TC * CB, *sb = sx + TC * CB, *sc = sb + TC * NP;
    const int64_t first = q.first + begin;
    const T *px = (const T *)a.x + first * a.x_stride + c0, *pdt = (const T *)a.dt + first * a.dt_stride + c0, *pz = a.z ? (const T *)a.z + first * a.z_stride + c0 : nullptr;
    const T *pb = (const T *)a.b + first * a.b_stride + (int64_t)group * N, *pc = (const T *)a.c + first * a.c_stride + (int64_t)group * N;
    T *pd = (T *)a.dst + first * a.dst_stride + c0;
    const int rows = end - begin, chunks = (rows + TC - 1) / TC;
    auto copy4 = [&](T *to, const T *row, int c) {  // (four channels; those behind the CTA's last are nobody's)
        if constexpr (VEC) {
            if constexpr (sizeof(T) == 4) cp_async16(to, row + c);
            else cp_async8(to, row + c);
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++) to[e] = c + e < nc ? row[c + e] : narrow<T>(0.f);
        }
    };
    auto fetch = [&](int chunk) {
        T *x = (T *)(raw + (chunk & 1) * Z::BUF), *dt = x + TC * CB, *z = dt + TC * CB, *b = z + TC * CB, *c = b + TC * NP;
        const int r0 = chunk * TC, nt = min(TC, rows - r0);
#pragma unroll
        for (int k = 0; k < Z::PIECES; k++) {
            const int i = tid + k * SCAN_THREADS, t = i / C4, ch = i % C4 * 4;
            if (t < nt && ch < nc) {
                copy4(x + t * CB + ch, px + (r0 + t) * a.x_stride, ch);
                copy4(dt + t * CB + ch, pdt + (r0 + t) * a.dt_stride, ch);
                if (PASS != ENDS && pz) copy4(z + t * CB + ch, pz + (r0 + t) * a.z_stride, ch);
            }
        }
        for (int i = tid; i < nt * N; i += SCAN_THREADS) {
            const int t = i / N, n = i - t * N;
            b[t * NP + n] = pb[(r0 + t) * a.b_stride + n];
            if (PASS != ENDS) c[t * NP + n] = pc[(r0 + t) * a.c_stride + n];
        }
        cp_async_commit();
    };
    fetch(0);
    // ===== the states
    const int cl = warp * Z::WC + g * CI;  // the lane's channels, counted from c0
    float h[CI][4], rate[CI][4], total[CI];
    const bool pieces = (N & 3) == 0 && ((a.slot_stride | a.from_stride) & 3) == 0 && (((uintptr_t)a.state | (uintptr_t)a.from | (uintptr_t)a.a) & 15) == 0;
    const int64_t ends_row = (int64_t)a.channels * N;  // floats of a stretch's end states; the stretch in front of a sequence's first is its state
    float *ends = a.ends + ((int64_t)blockIdx.z * (a.n_stretch + 1) + 1) * ends_row, *sums = a.sums + (int64_t)blockIdx.z * a.n_stretch * a.channels;
#pragma unroll
    for (int ci = 0; ci < CI; ci++) {
        const int c = c0 + cl + ci;
        float4 r = make_float4(0.f, 0.f, 0.f, 0.f), s = r;
        total[ci] = 0.f;
        if (cl + ci < nc) {
            const float *pa = a.a + (int64_t)c * N;
            r = pieces ? load_states<true>(pa, 4 * p, N) : load_states<false>(pa, 4 * p, N);
            if (PASS != ROWS && stretch == 0 && !q.begins) {
                const float *from = a.from + (int64_t)q.slot * a.from_stride + (int64_t)c * N;
                s = pieces ? load_states<true>(from, 4 * p, N) : load_states<false>(from, 4 * p, N);
            }
            if (PASS == ENDS && stretch == 0) store_states<false>(ends - ends_row + (int64_t)c * N, 4 * p, N, s);
            r.x *= LOG2E; r.y *= LOG2E; r.z *= LOG2E; r.w *= LOG2E;
            if (PASS == ROWS) {
                s = load_states<false>(ends + (stretch > 0 ? 0 : -ends_row) + (int64_t)c * N, 4 * p, N);
                for (int j = 1; j < stretch; j++) {
                    const float4 e = load_states<false>(ends + j * ends_row + (int64_t)c * N, 4 * p, N);
                    const float d = sums[(int64_t)j * a.channels + c];
                    s.x = fmaf(ex2(d * r.x), s.x, e.x);
                    s.y = fmaf(ex2(d * r.y), s.y, e.y);
                    s.z = fmaf(ex2(d * r.z), s.z, e.z);
                    s.w = fmaf(ex2(d * r.w), s.w, e.w);
                }
            }
        }
        rate[ci][0] = r.x; rate[ci][1] = r.y; rate[ci][2] = r.z; rate[ci][3] = r.w;
        h[ci][0] = s.x; h[ci][1] = s.y; h[ci][2] = s.z; h[ci][3] = s.w;
    }
    for (int i = tid; i < TC * NP; i += SCAN_THREADS) {  // (numbers behind d_state stay zeros)
        sb[i] = 0.f;
        sc[i] = 0.f;
    }
    for (int chunk = 0; chunk < chunks; chunk++) {
        const int r0 = chunk * TC, nt = min(TC, rows - r0);
        const T *x = (const T *)(raw + (chunk & 1) * Z::BUF), *dt = x + TC * CB, *z = dt + TC * CB, *b = z + TC * CB, *c = b + TC * NP;
        cp_async_wait<0>();
        __syncthreads();
        if (chunk + 1 < chunks) fetch(chunk + 1);
        // ===== d and d x.  Rows behind the last and channels behind the CTA's leave states as they are
#pragma unroll
        for (int k = 0; k < Z::PIECES; k++) {
            const int i = tid + k * SCAN_THREADS, t = i / C4, ch = i % C4 * 4;
            float4 d4 = make_float4(0.f, 0.f, 0.f, 0.f), x4 = d4;
            if (t < nt && ch < nc) {
                const Pack<T, 4> pdt4 = *reinterpret_cast<const Pack<T, 4> *>(dt + t * CB + ch), px4 = *reinterpret_cast<const Pack<T, 4> *>(x + t * CB + ch);
                float dv[4], xv[4];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const bool there = VEC || ch + e < nc;
                    float d = there ? wide(pdt4.v[e]) + (a.dt_bias ? a.dt_bias[c0 + ch + e] : 0.f) : 0.f;
                    if (a.softplus && there) d = softplus(d);
                    dv[e] = d;
                    xv[e] = there ? d * wide(px4.v[e]) : 0.f;
                }
                d4 = make_float4(dv[0], dv[1], dv[2], dv[3]);
                x4 = make_float4(xv[0], xv[1], xv[2], xv[3]);
            }
            *reinterpret_cast<float4 *>(sd + t * CB + ch) = d4;
            *reinterpret_cast<float4 *>(sx + t * CB + ch) = x4;
        }
        for (int i = tid; i < nt * N; i += SCAN_THREADS) {
            const int t = i / N, n = i - t * N;
            sb[t * NP + n] = wide(b[t * NP + n]);
            if (PASS != ENDS) sc[t * NP + n] = wide(c[t * NP + n]);
        }
        __syncthreads();
        // ===== the rows, four at a time
#pragma unroll 1
        for (int t0 = 0; t0 < nt; t0 += 4) {
            float y[4][CI];
#pragma unroll
            for (int u = 0; u < 4; u++) {
                const int t = t0 + u;
                const float4 b4 = *reinterpret_cast<const float4 *>(sb + t * NP + 4 * p);
                const float4 c4 = PASS == ENDS ? b4 : *reinterpret_cast<const float4 *>(sc + t * NP + 4 * p);
                const Pack<float, CI> d = *reinterpret_cast<const Pack<float, CI> *>(sd + t * CB + cl), dx = *reinterpret_cast<const Pack<float, CI> *>(sx + t * CB + cl);
                const float bv[4] = {b4.x, b4.y, b4.z, b4.w}, cv[4] = {c4.x, c4.y, c4.z, c4.w};
#pragma unroll
                for (int ci = 0; ci < CI; ci++) {
                    if (PASS == ENDS) total[ci] += d.v[ci];
#pragma unroll
                    for (int n = 0; n < 4; n++) {
                        h[ci][n] = fmaf(ex2(d.v[ci] * rate[ci][n]), h[ci][n], dx.v[ci] * bv[n]);
                        if (PASS != ENDS) y[u][ci] = n == 0 ? cv[0] * h[ci][0] : fmaf(cv[n], h[ci][n], y[u][ci]);
                    }
                }
            }
            if (PASS != ENDS) {
                // sums over the channel's lanes: those of one half keep rows 2 and 3, then a quarter one row each
                const bool hi = (p & (L / 2)) != 0, odd = (p & (L / 4)) != 0;
                float v[CI];
#pragma unroll
                for (int ci = 0; ci < CI; ci++) {
                    const float s0 = hi ? y[0][ci] : y[2][ci], s1 = hi ? y[1][ci] : y[3][ci], k0 = hi ? y[2][ci] : y[0][ci], k1 = hi ? y[3][ci] : y[1][ci];
                    const float w0 = k0 + __shfl_xor_sync(0xffffffffu, s0, L / 2), w1 = k1 + __shfl_xor_sync(0xffffffffu, s1, L / 2);
                    const float s = odd ? w0 : w1, k = odd ? w1 : w0;
                    v[ci] = k + __shfl_xor_sync(0xffffffffu, s, L / 4);
                }
#pragma unroll
                for (int n = L / 8; n >= 1; n /= 2) {
#pragma unroll
                    for (int ci = 0; ci < CI; ci++) v[ci] += __shfl_xor_sync(0xffffffffu, v[ci], n);
                }
                __syncwarp();  // the warp has read these rows of its channels in sd: their results take the place
                if ((p & (L / 4 - 1)) == 0) {
                    Pack<float, CI> out;
#pragma unroll
                    for (int ci = 0; ci < CI; ci++) out.v[ci] = v[ci];
                    *reinterpret_cast<Pack<float, CI> *>(sd + (t0 + 2 * hi + odd) * CB + cl) = out;
                }
            }
        }
        if (PASS == ENDS) continue;
        __syncthreads();
#pragma unroll
        for (int k = 0; k < Z::PIECES; k++) {
            const int i = tid + k * SCAN_THREADS, t = i / C4, ch = i % C4 * 4;
            if (t < nt && ch < nc) {
                const float4 y4 = *reinterpret_cast<const float4 *>(sd + t * CB + ch);
                float y[4] = {y4.x, y4.y, y4.z, y4.w};
                if (a.d) {
                    const Pack<T, 4> px4 = *reinterpret_cast<const Pack<T, 4> *>(x + t * CB + ch);
#pragma unroll
                    for (int e = 0; e < 4; e++) if (VEC || ch + e < nc) y[e] = fmaf(a.d[c0 + ch + e], wide(px4.v[e]), y[e]);
                }
                if (a.z) {
                    const Pack<T, 4> pz4 = *reinterpret_cast<const Pack<T, 4> *>(z + t * CB + ch);
#pragma unroll
                    for (int e = 0; e < 4; e++) y[e] *= silu(wide(pz4.v[e]));
                }
                T *to = pd + (r0 + t) * a.dst_stride + ch;
                if constexpr (VEC) {
                    Pack<T, 4> out;
#pragma unroll
                    for (int e = 0; e < 4; e++) out.v[e] = narrow<T>(y[e]);
                    *reinterpret_cast<Pack<T, 4> *>(to) = out;
                } else {
#pragma unroll
                    for (int e = 0; e < 4; e++) if (ch + e < nc) to[e] = narrow<T>(y[e]);
                }
            }
        }
    }
    // ===== where the states go: the stretch's place, or the slot
#pragma unroll
    for (int ci = 0; ci < CI; ci++) {
        if (cl + ci >= nc) continue;
        const int c = c0 + cl + ci;
        const float4 s = make_float4(h[ci][0], h[ci][1], h[ci][2], h[ci][3]);
        if (PASS == ENDS) {
            store_states<false>(ends + stretch * ends_row + (int64_t)c * N, 4 * p, N, s);
            if (p == 0) sums[(int64_t)stretch * a.channels + c] = total[ci];
        } else if (end == q.count) {
            float *to = a.state + (int64_t)q.slot * a.slot_stride + (int64_t)c * N;
            if (pieces) store_states<true>(to, 4 * p, N, s);
            else store_states<false>(to, 4 * p, N, s);
        }
    }
}

// ------------------------------------------------------------------------------------------------ host side
static inline bool type_ok(int t) { return t == B200_TYPE_F32 || t == B200_TYPE_F16 || t == B200_TYPE_BF16; }
static inline size_t type_size(int t) { return t == B200_TYPE_F32 ? 4 : 2; }
static inline bool on(size_t size, std::initializer_list<const void *> ps) {
    for (const void *p : ps) if ((uintptr_t)p % size) return false;
    return true;
}

// How a call's work is laid out.
struct ScanPlan {
    int lanes, per_lane;          // lanes of a channel, channels of a lane
    int stretch, n_stretch;       // 0, 1: no stretches
    bool step;                    // one row a sequence
};
static int max_new_of(const b200_ssm_scan_args *a) { return a->max_new > 0 && a->max_new < a->n_tokens ? a->max_new : a->n_tokens; }
static ScanPlan plan_of(const b200_ssm_scan_args *a) {
    ScanPlan p = {};
    const int longest = a->seq_info ? max_new_of(a) : (a->n_seq > 0 ? a->n_tokens / a->n_seq : 0);
    p.lanes = a->d_state <= 16 ? 4 : a->d_state <= 32 ? 8 : a->d_state <= 64 ? 16 : 32;
    p.step = longest <= 1;
    p.per_lane = 4;
    p.n_stretch = 1;
    const int block = SCAN_WARPS * 32 / p.lanes * p.per_lane, per_group = a->channels / a->groups;
    const int64_t ctas = (int64_t)((per_group + block - 1) / block) * a->groups * a->n_seq;
    const int want = 3 * sm_count();
    if (!p.step && ctas < want / 2 && longest >= 128) {
        int n = (int)(want / ctas);
        if (n > 32) n = 32;
        if (n > longest / 64) n = longest / 64;
        if (n > 1) {
            p.stretch = ((longest + n - 1) / n + 31) / 32 * 32;
            p.n_stretch = (longest + p.stretch - 1) / p.stretch;
            if (p.n_stretch < 2) p.n_stretch = 1;
        }
    }
    return p;
}
static size_t scan_room(const b200_ssm_scan_args *a, const ScanPlan &p) {
    if (p.n_stretch < 2) return 0;
    return 4 * (size_t)a->n_seq * ((size_t)(p.n_stretch + 1) * a->channels * a->d_state + (size_t)p.n_stretch * a->channels);
}

template <typename T, int L, bool VEC, int PASS>
static int launch_scan(const ScanArgs &a, cudaStream_t st) {
    using Z = ScanSizes<T, L, 4>;
    const auto kern = ssm_scan_kernel<T, L, 4, VEC, PASS>;
    if (Z::SMEM > 48 * 1024) {
        static bool attr_set_dev[16] = {};  // cudaFuncSetAttribute is per device
        int dev = 0;
        B200_CUDA_TRY(cudaGetDevice(&dev));
        if (dev > 15 || !attr_set_dev[dev]) {
            B200_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Z::SMEM));
            if (dev <= 15) attr_set_dev[dev] = true;
        }
    }
    const int groups = a.channels / a.per_group;
    const dim3 grid((unsigned)((a.per_group + Z::CB - 1) / Z::CB * groups), (unsigned)(PASS == WHOLE ? 1 : a.n_stretch), (unsigned)a.step.n_seq);
    B200_CUDA_TRY(launch_chained(kern, grid, SCAN_THREADS, Z::SMEM, st, a));
    return B200_OK;
}
template <typename T, int L>
static int launch_scan_lanes(const ScanArgs &a, const ScanPlan &p, bool vec, bool states16, cudaStream_t st) {
    if (p.step) {
        const dim3 grid((unsigned)((a.channels + 32 * STEP_WARPS - 1) / (32 * STEP_WARPS)), (unsigned)a.step.n_seq);
        B200_CUDA_TRY(launch_chained(states16 ? ssm_step_kernel<T, L, true> : ssm_step_kernel<T, L, false>, grid, 32 * STEP_WARPS, 0, st, a));
        return B200_OK;
    }
    if (p.n_stretch < 2) return vec ? launch_scan<T, L, true, WHOLE>(a, st) : launch_scan<T, L, false, WHOLE>(a, st);
    const int rc = vec ? launch_scan<T, L, true, ENDS>(a, st) : launch_scan<T, L, false, ENDS>(a, st);
    if (rc != B200_OK) return rc;
    return vec ? launch_scan<T, L, true, ROWS>(a, st) : launch_scan<T, L, false, ROWS>(a, st);
}
template <typename T>
static int launch_scan_type(const ScanArgs &a, const ScanPlan &p, bool vec, bool states16, cudaStream_t st) {
    switch (p.lanes) {
        case 4: return launch_scan_lanes<T, 4>(a, p, vec, states16, st);
        case 8: return launch_scan_lanes<T, 8>(a, p, vec, states16, st);
        case 16: return launch_scan_lanes<T, 16>(a, p, vec, states16, st);
        default: return launch_scan_lanes<T, 32>(a, p, vec, states16, st);
    }
}

static int check_step(const int32_t *seq_info, int32_t n_seq, int32_t n_slots, int32_t n_tokens, int32_t max_new, int32_t type, const char *who) {
    OPX_REQUIRE(type_ok(type), B200_ERR_UNSUPPORTED, "%s: rows of type %d", who, type);
    OPX_REQUIRE(n_seq >= 0 && n_seq <= 65535 && n_slots >= 0 && n_tokens >= 0 && max_new >= 0, B200_ERR_INVALID, "%s: %d sequences, %d slots, %d rows, %d new ones at most", who, n_seq, n_slots,
                n_tokens, max_new);
    OPX_REQUIRE((uintptr_t)seq_info % 4 == 0, B200_ERR_INVALID, "%s: seq_info at an odd place", who);
    OPX_REQUIRE(seq_info || (n_seq <= n_slots && (n_seq == 0 ? n_tokens == 0 : n_tokens % n_seq == 0)), B200_ERR_INVALID, "%s: without seq_info, %d rows are not %d sequences of one length in %d slots",
                who, n_tokens, n_seq, n_slots);
    return B200_OK;
}

int ssm_scan_check(const b200_ssm_scan_args *a) {
    const char *who = "b200_op_ssm_scan";
    OPX_REQUIRE(a, B200_ERR_INVALID, "%s: NULL arguments", who);
    const int rc = check_step(a->seq_info, a->n_seq, a->n_slots, a->n_tokens, a->max_new, a->type, who);
    if (rc != B200_OK) return rc;
    OPX_REQUIRE(a->channels > 0 && a->d_state > 0 && a->groups > 0 && a->channels % a->groups == 0, B200_ERR_INVALID, "%s: %d channels in %d groups, %d states", who, a->channels, a->groups, a->d_state);
    OPX_REQUIRE(a->d_state <= 128, B200_ERR_UNSUPPORTED, "%s: %d states a channel, 128 at most", who, a->d_state);
    if (a->n_seq == 0 || a->n_tokens == 0) return B200_OK;
    OPX_REQUIRE(a->x && a->dt && a->b && a->c && a->a && a->state && a->dst, B200_ERR_INVALID, "%s: NULL argument", who);
    const int64_t states = (int64_t)a->channels * a->d_state, bc = (int64_t)a->groups * a->d_state;
    OPX_REQUIRE(a->x_stride >= a->channels && a->dt_stride >= a->channels && a->dst_stride >= a->channels && (!a->z || a->z_stride >= a->channels) && a->b_stride >= bc && a->c_stride >= bc,
                B200_ERR_INVALID, "%s: rows overlap", who);
    OPX_REQUIRE(a->slot_stride >= states && (!a->from || a->from_stride >= states), B200_ERR_INVALID, "%s: slots overlap", who);
    OPX_REQUIRE(on(type_size(a->type), {a->x, a->dt, a->b, a->c, a->z, a->dst}) && on(4, {a->a, a->dt_bias, a->d, a->state, a->from}), B200_ERR_INVALID, "%s: a pointer is not aligned to its type", who);
    OPX_REQUIRE(a->dst != a->b && a->dst != a->c, B200_ERR_INVALID, "%s: dst is b or c, which other channels read", who);
    return B200_OK;
}

}  // namespace ssm
}  // namespace b200

using namespace b200;
using namespace b200::ssm;

extern "C" {

int b200_op_ssm_conv(const b200_ssm_conv_args *a, b200_stream_t stream) {
    const char *who = "b200_op_ssm_conv";
    OPX_REQUIRE(a, B200_ERR_INVALID, "%s: NULL arguments", who);
    const int rc = check_step(a->seq_info, a->n_seq, a->n_slots, a->n_tokens, a->max_new, a->type, who);
    if (rc != B200_OK) return rc;
    OPX_REQUIRE(a->channels > 0 && a->taps >= 1, B200_ERR_INVALID, "%s: %d channels, %d taps", who, a->channels, a->taps);
    OPX_REQUIRE(a->taps <= 16, B200_ERR_UNSUPPORTED, "%s: %d taps, 16 at most", who, a->taps);
    if (a->n_seq == 0 || a->n_tokens == 0) return B200_OK;
    OPX_REQUIRE(a->x && a->w && a->dst && (a->tail || a->taps == 1), B200_ERR_INVALID, "%s: NULL argument", who);
    OPX_REQUIRE(a->x_stride >= a->channels && a->dst_stride >= a->channels, B200_ERR_INVALID, "%s: rows overlap", who);
    OPX_REQUIRE(a->slot_stride >= (int64_t)(a->taps - 1) * a->channels, B200_ERR_INVALID, "%s: slots overlap", who);
    OPX_REQUIRE(on(type_size(a->type), {a->x, a->dst}) && on(4, {a->w, a->bias, a->tail}), B200_ERR_INVALID, "%s: a pointer is not aligned to its type", who);
    OPX_REQUIRE(a->x != a->dst, B200_ERR_INVALID, "%s: not in place", who);
    const int each = a->seq_info ? a->n_tokens : a->n_tokens / a->n_seq, longest = a->max_new > 0 && a->max_new < each ? a->max_new : each;
    OPX_REQUIRE((longest + CONV_ROWS - 1) / CONV_ROWS <= 65535, B200_ERR_UNSUPPORTED, "%s: at most %d rows of a sequence", who, 65535 * CONV_ROWS);
    const ConvArgs c = {{a->seq_info, a->n_seq, a->n_slots, a->n_tokens, longest}, a->x, a->x_stride, a->w, a->bias, a->tail, a->slot_stride, a->dst, a->dst_stride, a->channels, a->taps, a->silu};
    const cudaStream_t st = (cudaStream_t)stream;
    const int v = a->type == B200_TYPE_F32 ? 4 : 8;
    const bool vec = on(16, {a->x, a->dst}) && ((a->x_stride | a->dst_stride | a->channels) & (v - 1)) == 0;
    if (a->type == B200_TYPE_F32) return vec ? launch_conv_taps<float, 4>(c, st) : launch_conv_taps<float, 1>(c, st);
    if (a->type == B200_TYPE_F16) return vec ? launch_conv_taps<__half, 8>(c, st) : launch_conv_taps<__half, 1>(c, st);
    return vec ? launch_conv_taps<__nv_bfloat16, 8>(c, st) : launch_conv_taps<__nv_bfloat16, 1>(c, st);
}

size_t b200_ssm_scan_workspace_bytes(const b200_ssm_scan_args *a) {
    if (!a || a->n_seq <= 0 || a->n_tokens <= 0 || a->channels <= 0 || a->groups <= 0 || a->channels % a->groups || a->d_state <= 0 || a->d_state > 128) return 0;
    return scan_room(a, plan_of(a));
}

int b200_op_ssm_scan(const b200_ssm_scan_args *a, void *workspace, size_t workspace_bytes, b200_stream_t stream) {
    const char *who = "b200_op_ssm_scan";
    const int rc = ssm_scan_check(a);
    if (rc != B200_OK || a->n_seq == 0 || a->n_tokens == 0) return rc;
    const ScanPlan p = plan_of(a);
    const size_t need = scan_room(a, p);
    OPX_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && (uintptr_t)workspace % 16 == 0), B200_ERR_INVALID, "%s: workspace of %zu bytes, 16-byte aligned", who, need);
    const int per_group = a->channels / a->groups, each = a->seq_info ? a->n_tokens : a->n_tokens / a->n_seq, longest = a->max_new > 0 && a->max_new < each ? a->max_new : each;
    float *ends = (float *)workspace;
    const ScanArgs s = {{a->seq_info, a->n_seq, a->n_slots, a->n_tokens, longest}, a->x, a->dt, a->b, a->c, a->z, a->x_stride, a->dt_stride, a->b_stride, a->c_stride, a->z_stride, a->a, a->dt_bias, a->d,
                        a->from ? a->from : a->state, a->from ? a->from_stride : a->slot_stride, a->state, a->slot_stride, a->dst, a->dst_stride, a->channels, a->d_state, per_group, a->softplus,
                        p.stretch, p.n_stretch, ends, ends ? ends + (size_t)a->n_seq * (p.n_stretch + 1) * a->channels * a->d_state : nullptr};
    const size_t four = 4 * type_size(a->type);
    const bool vec = per_group % 4 == 0 && on(four, {a->x, a->dt, a->z, a->dst}) && ((a->x_stride | a->dt_stride | a->dst_stride | (a->z ? a->z_stride : 0)) & 3) == 0;
    const bool states16 = (a->d_state & 3) == 0 && ((s.slot_stride | s.from_stride) & 3) == 0 && on(16, {s.state, s.from, a->a});
    const cudaStream_t st = (cudaStream_t)stream;
    if (a->type == B200_TYPE_F32) return launch_scan_type<float>(s, p, vec, states16, st);
    if (a->type == B200_TYPE_F16) return launch_scan_type<__half>(s, p, vec, states16, st);
    return launch_scan_type<__nv_bfloat16>(s, p, vec, states16, st);
}

}  // extern "C"
