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
// two values at once
template <typename T> __device__ __forceinline__ void narrow2(T *to, float lo, float hi) {
    if constexpr (std::is_same<T, __half>::value) *reinterpret_cast<__half2 *>(to) = __floats2half2_rn(lo, hi);
    else if constexpr (sizeof(T) == 2) *reinterpret_cast<__nv_bfloat162 *>(to) = __floats2bfloat162_rn(lo, hi);
    else { to[0] = lo; to[1] = hi; }
}
// V consecutive values, in one access where they lie on a boundary of their size
template <typename T, int V> struct __align__(sizeof(T) * V) Pack { T v[V]; };

constexpr float LOG2E = 1.4426950408889634f;
// 2^x and 1 / x of the special function unit, off by 2^-22 and 2^-23; numbers below 2^-126 are zeros
__device__ __forceinline__ float ex2(float x) { float r; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x)); return r; }
__device__ __forceinline__ float rcp(float x) { float r; asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x)); return r; }
// y * sigmoid(y) (where e^-y is more than f32 holds, -0)
__device__ __forceinline__ float silu(float y) { return y * rcp(1.0f + ex2(-LOG2E * y)); }

// two floats that are worked on by one instruction
using Two = unsigned long long;
__device__ __forceinline__ Two two(float lo, float hi) { Two r; asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi)); return r; }
__device__ __forceinline__ float2 each(Two x) { float2 r; asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(x)); return r; }
__device__ __forceinline__ Two fma2(Two x, Two y, Two z) { Two r; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(x), "l"(y), "l"(z)); return r; }
__device__ __forceinline__ Two mul2(Two x, Two y) { Two r; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y)); return r; }

// ------------------------------------------------------------------------------------------------ short convolution
// A thread takes V channels of `rows` rows of one sequence and keeps the last K - 1 inputs in registers; rows travel in groups, asynchronously to a ring in shared memory.  The CTAs that hold a
// sequence's first rows read its tail, and they alone write it (each channel by one thread), so that nobody reads what another has rewritten.  K: taps, or the next of 8 and 16, whose products of
// taps that are not there are left out.  Weights and biases do not depend on the sequence: they are asked for before it is known.
constexpr int CONV_THREADS = 128, CONV_GROUP = 4, CONV_GROUPS = 4, CONV_ROWS_MIN = 16, CONV_ROWS_MAX = 64;
struct ConvArgs {
    Step step;
    const void *x; int64_t x_stride;
    const float *w, *bias;
    float *tail; int64_t slot_stride;
    void *dst; int64_t dst_stride;
    int32_t channels, taps, silu, rows;
};
template <typename T, int K, int V, bool EXACT, bool RING>
__global__ void __launch_bounds__(CONV_THREADS) ssm_conv_kernel(const ConvArgs a) {
    pdl_enter();
    const int c = (blockIdx.x * CONV_THREADS + threadIdx.x) * V, t0 = blockIdx.y * a.rows;
    const int skip = EXACT ? 0 : K - a.taps;  // taps that are not there
    if (c >= a.channels) return;
    float w[K][V], bias[V], win[K][V];  // win[K - 1]: the newest input
    const float *pw = a.w + (int64_t)c * a.taps;
    if (K == 4 && EXACT && ((uintptr_t)a.w & 15) == 0) {
#pragma unroll
        for (int e = 0; e < V; e++) {
            const float4 v = reinterpret_cast<const float4 *>(pw)[e];
            w[0][e] = v.x; w[1 % K][e] = v.y; w[2 % K][e] = v.z; w[3 % K][e] = v.w;
        }
    } else {
#pragma unroll
        for (int e = 0; e < V; e++) {
#pragma unroll
            for (int j = 0; j < K; j++) w[j][e] = EXACT || j >= skip ? pw[e * a.taps + j - skip] : 0.f;
        }
    }
#pragma unroll
    for (int e = 0; e < V; e++) bias[e] = a.bias ? a.bias[c + e] : 0.f;
    const Seq q = seq_of(a.step, blockIdx.z);
    if (t0 >= q.count) return;
    const int nt = min(a.rows, q.count - t0);
    const T *x = (const T *)a.x + (int64_t)q.first * a.x_stride + c;
    float *tail = a.tail + (int64_t)q.slot * a.slot_stride + c;
    using P = Pack<T, V>;
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
    const T *in_row = x + (int64_t)t0 * a.x_stride;
    auto turn = [&](const P &in) {  // the next row
        P out;
#pragma unroll
        for (int e = 0; e < V; e++) {
#pragma unroll
            for (int j = 0; j < K - 1; j++) win[j][e] = win[j + 1][e];
            win[K - 1][e] = wide(in.v[e]);
        }
#pragma unroll
        for (int e = 0; e < V; e += 2) {
            float y[2];
            if constexpr (V >= 2) {
                Two s = two(bias[e], bias[e + 1]);
#pragma unroll
                for (int j = 0; j < K; j++) if (EXACT || j >= skip) s = fma2(two(w[j][e], w[j][e + 1]), two(win[j][e], win[j][e + 1]), s);
                y[0] = each(s).x; y[1] = each(s).y;
            } else {
                y[0] = bias[e];
#pragma unroll
                for (int j = 0; j < K; j++) if (EXACT || j >= skip) y[0] = fmaf(w[j][e], win[j][e], y[0]);
            }
            if (a.silu) {
                y[0] = silu(y[0]);
                if (V >= 2) y[1] = silu(y[1]);
            }
            if constexpr (V >= 2) narrow2<T>(out.v + e, y[0], y[1]);
            else out.v[e] = narrow<T>(y[0]);
        }
        *reinterpret_cast<P *>(dst) = out;
        dst += a.dst_stride;
    };
    if constexpr (RING) {
        // (of the ring every thread reads only what it has asked for)
        __shared__ __align__(16) P ring[CONV_GROUPS][CONV_GROUP][CONV_THREADS];
        auto fetch = [&](int g) {
#pragma unroll
            for (int u = 0; u < CONV_GROUP; u++) {
                if (g * CONV_GROUP + u < nt) {
                    if constexpr (sizeof(P) == 16) cp_async16(&ring[g % CONV_GROUPS][u][threadIdx.x], in_row);
                    else cp_async8(&ring[g % CONV_GROUPS][u][threadIdx.x], in_row);
                }
                in_row += a.x_stride;
            }
            cp_async_commit();
        };
#pragma unroll
        for (int g = 0; g < CONV_GROUPS - 1; g++) fetch(g);
        for (int g = 0; g * CONV_GROUP < nt; g++) {
            cp_async_wait<CONV_GROUPS - 2>();
#pragma unroll
            for (int u = 0; u < CONV_GROUP; u++) {
                if (g * CONV_GROUP + u < nt) turn(ring[g % CONV_GROUPS][u][threadIdx.x]);
            }
            fetch(g + CONV_GROUPS - 1);
        }
        cp_async_wait<0>();
    } else {
        for (int b = 0; b < nt; b += CONV_GROUP) {
            P in[CONV_GROUP];
#pragma unroll
            for (int u = 0; u < CONV_GROUP; u++) {
                if (b + u < nt) in[u] = *reinterpret_cast<const P *>(in_row);
                in_row += a.x_stride;
            }
#pragma unroll
            for (int u = 0; u < CONV_GROUP; u++) {
                if (b + u < nt) turn(in[u]);
            }
        }
    }
    if (t0 == 0) {
        // entry j of the new tail is the input of row count - taps + 1 + j: all of them are in the window, or among x's rows
#pragma unroll
        for (int j = 1; j < K; j++) {
            if (!EXACT && j <= skip) continue;
            const int i = q.count - K + j;
            float *to = tail + (int64_t)(j - 1 - skip) * a.channels;
            if (q.count <= a.rows) {
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
static_assert(CONV_ROWS_MIN >= 15, "a sequence of more rows than a CTA takes has all the new tail's inputs among its rows");

template <typename T, int K, int V, bool EXACT>
static int launch_conv(ConvArgs a, cudaStream_t st) {
    // rows of a CTA: as many as leave every SM eight of them (each one reads its weights and the taps - 1 rows in front)
    const unsigned across = (unsigned)((a.channels + CONV_THREADS * V - 1) / (CONV_THREADS * V));
    a.rows = CONV_ROWS_MAX;
    while (a.rows > CONV_ROWS_MIN && (int64_t)across * ((a.step.n_tokens + a.rows - 1) / a.rows) < 8 * (int64_t)sm_count()) a.rows /= 2;
    const dim3 grid(across, (unsigned)((a.step.max_new + a.rows - 1) / a.rows), (unsigned)a.step.n_seq);
    // the ring pays where there is something to wait for: 64 sequences of one row, f32: 4.5 us with it, 3.8 without; 5330 rows, bf16: 40 and 46 us
    const bool ring = V * sizeof(T) >= 8 && a.step.max_new > 2 * CONV_GROUP;
    B200_CUDA_TRY(launch_chained(ring ? ssm_conv_kernel<T, K, V, EXACT, (V * sizeof(T) >= 8)> : ssm_conv_kernel<T, K, V, EXACT, false>, grid, CONV_THREADS, 0, st, a));
    return B200_OK;
}
template <typename T, int V>
static int launch_conv_taps(const ConvArgs &a, cudaStream_t st) {
    switch (a.taps) {
        case 1: return launch_conv<T, 1, V, true>(a, st);
        case 2: return launch_conv<T, 2, V, true>(a, st);
        case 3: return launch_conv<T, 3, V, true>(a, st);
        case 4: return launch_conv<T, 4, V, true>(a, st);
        default: return a.taps <= 8 ? launch_conv<T, 8, V, false>(a, st) : launch_conv<T, 16, V, false>(a, st);
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
    int32_t channels, d_state, per_group, softplus, bc_pieces;  // bc_pieces: b and c can be read four numbers at a time
    // stretches: rows of one, how many a sequence may have; where their end states and sums of d wait
    int32_t stretch, n_stretch;
    float *ends, *sums;
};

// ln(1 + e^x) = max(x, 0) + ln(1 + e^-|x|), and ln(1 + e) = e P(e) on [0, 1] with a polynomial whose relative error is smallest at its largest (fitted by weighted least squares on
// Chebyshev points; 1.8e-7 with the roundings of f32): one exponential on the special function unit and nothing else there, no overflow, no cancellation.
__device__ __forceinline__ float2 softplus2(float2 x) {
    const Two e = two(ex2(-LOG2E * fabsf(x.x)), ex2(-LOG2E * fabsf(x.y)));
    auto both = [](float v) { return two(v, v); };
    Two p = both(0.0052326764f);
    p = fma2(p, e, both(-0.0295051672f));
    p = fma2(p, e, both(0.0782258362f));
    p = fma2(p, e, both(-0.136632353f));
    p = fma2(p, e, both(0.191060022f));
    p = fma2(p, e, both(-0.248429805f));
    p = fma2(p, e, both(0.333190978f));
    p = fma2(p, e, both(-0.499994934f));
    return each(fma2(fma2(p, e, both(1.0f)), e, two(fmaxf(x.x, 0.f), fmaxf(x.y, 0.f))));
}
__device__ __forceinline__ float softplus(float x) { return softplus2(make_float2(x, x)).x; }

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
// A CTA takes CB channels.  L lanes share CI of them, a lane four states of each: the loads of b and c serve CI channels, and a warp's chains are 4 CI exponentials and multiply-adds a lane
// wide.  Rows come in chunks of TC.  While the warps walk chunk k, chunk k + 1 is made ready (d and d x), the results of chunk k - 1 go out and chunk k + 2 travels: one barrier a chunk.  Every thread
// stages, and later sends off, the same pieces of a chunk, so what lies in memory's form between its arrival and the end is nobody else's.
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
    static constexpr int BUF = 3 * RAW + 2 * RAW_BC;              // x, dt, z, b, c as they lie in memory: three chunks
    static constexpr int READY = 4 * (2 * TC * CB + 2 * TC * NP); // d (later y), d x, b, c in f32: two chunks
    static constexpr int SMEM = 3 * BUF + 2 * READY;
    static_assert(PIECES >= 1 && TC % 4 == 0 && SCAN_THREADS % (CB / 4) == 0 && 2 * TC * L % SCAN_THREADS == 0, "every thread stages the same number of pieces, of one place in the rows");
};
template <typename T, int L, int CI, bool VEC, int PASS>
__global__ void __launch_bounds__(SCAN_THREADS) ssm_scan_kernel(const ScanArgs a) {
    using Z = ScanSizes<T, L, CI>;
    constexpr int G = Z::G, CB = Z::CB, NP = Z::NP, TC = Z::TC, C4 = CB / 4, TB = CI == 2 ? 16 : 8;
    extern __shared__ __align__(16) unsigned char ssm_shared[];
    pdl_wait();  // (the kernel behind is let in at the end: CTAs of it that wait would take places in an order that leaves SMs unequal, 520 -> 610 us for four long prompts)
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, p = lane % L, g = lane / L;
    const Seq q = seq_of(a.step, blockIdx.z);
    const int N = a.d_state, blocks = (a.per_group + CB - 1) / CB, group = blockIdx.x / blocks, in_group = (blockIdx.x - group * blocks) * CB;
    const int c0 = group * a.per_group + in_group, nc = min(CB, a.per_group - in_group);  // channels of the CTA
    const int stretch = PASS == WHOLE ? 0 : blockIdx.y, begin = PASS == WHOLE ? 0 : stretch * a.stretch, end = PASS == WHOLE ? q.count : min(q.count, begin + a.stretch);
    if (begin >= end) return;
    if (PASS == ENDS && end == q.count && stretch > 0) return;  // nobody asks for the last one's
    const int64_t first = q.first + begin;
    const T *px = (const T *)a.x + first * a.x_stride + c0, *pdt = (const T *)a.dt + first * a.dt_stride + c0, *pz = a.z ? (const T *)a.z + first * a.z_stride + c0 : nullptr;
    const T *pb = (const T *)a.b + first * a.b_stride + (int64_t)group * N, *pc = (const T *)a.c + first * a.c_stride + (int64_t)group * N;
    T *pd = (T *)a.dst + first * a.dst_stride + c0;
    const int rows = end - begin, chunks = (rows + TC - 1) / TC;
    // chunk k as it lies in memory, and made ready
    auto raw = [&](int k) { return (T *)(ssm_shared + k % 3 * Z::BUF); };                  // x, dt, z [TC][CB], b, c [TC][NP]
    auto ready = [&](int k) { return (float *)(ssm_shared + 3 * Z::BUF + (k & 1) * Z::READY); };  // d, d x [TC][CB], b, c [TC][NP]
    // the thread's pieces: four channels from ch on of the rows t1, t1 + TR, ..; four of the numbers of b or c
    constexpr int TR = SCAN_THREADS / C4, BC = 2 * TC * L / SCAN_THREADS;
    const int ch = tid % C4 * 4, t1 = tid / C4;
    const bool mine = ch < nc;
    float bias[4], skip[4];
#pragma unroll
    for (int e = 0; e < 4; e++) {
        bias[e] = a.dt_bias && ch + e < nc ? a.dt_bias[c0 + ch + e] : 0.f;
        skip[e] = PASS != ENDS && a.d && ch + e < nc ? a.d[c0 + ch + e] : 0.f;
    }
    px += t1 * a.x_stride + ch;
    pdt += t1 * a.dt_stride + ch;
    pd += t1 * a.dst_stride + ch;
    if (pz) pz += t1 * a.z_stride + ch;
    auto copy4 = [&](T *to, const T *row) {  // (four channels; those behind the CTA's last are nobody's)
        if constexpr (VEC) {
            if constexpr (sizeof(T) == 4) cp_async16(to, row);
            else cp_async8(to, row);
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++) to[e] = ch + e < nc ? row[e] : narrow<T>(0.f);
        }
    };
    auto fetch = [&](int k) {  // called for 0, 1, 2, ..
        if (k < chunks) {
            T *x = raw(k) + t1 * CB + ch;
            const int nt = min(TC, rows - k * TC);
            if (mine) {
#pragma unroll
                for (int j = 0; j < Z::PIECES; j++) {
                    if (t1 + j * TR < nt) {
                        copy4(x + j * TR * CB, px + j * TR * a.x_stride);
                        copy4(x + (TC + j * TR) * CB, pdt + j * TR * a.dt_stride);
                        if (PASS != ENDS && pz) copy4(x + (2 * TC + j * TR) * CB, pz + j * TR * a.z_stride);
                    }
                }
            }
            px += TC * a.x_stride;
            pdt += TC * a.dt_stride;
            if (pz) pz += TC * a.z_stride;
            T *b = raw(k) + 3 * TC * CB;
#pragma unroll
            for (int j = 0; j < BC; j++) {
                const int i = tid + j * SCAN_THREADS, r = i / L, n = i % L * 4, t = r % TC;
                if (t < nt && n < N && (PASS != ENDS || r < TC)) {
                    const T *row = (r < TC ? pb + (k * TC + t) * a.b_stride : pc + (k * TC + t) * a.c_stride) + n;
                    if (a.bc_pieces) {
                        if constexpr (sizeof(T) == 4) cp_async16(b + 4 * i, row);
                        else cp_async8(b + 4 * i, row);
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; e++) b[4 * i + e] = n + e < N ? row[e] : narrow<T>(0.f);
                    }
                }
            }
        }
        cp_async_commit();
    };
    // d and d x, b and c.  Rows behind the last and channels behind the CTA's leave states as they are
    auto stage = [&](int k) {
        if (k >= chunks) return;
        const T *x = raw(k) + t1 * CB + ch, *b = raw(k) + 3 * TC * CB;
        float *sd = ready(k) + t1 * CB + ch, *sb = ready(k) + 2 * TC * CB;
        const int nt = min(TC, rows - k * TC);
#pragma unroll
        for (int j = 0; j < Z::PIECES; j++) {
            float4 d = make_float4(0.f, 0.f, 0.f, 0.f), dx = d;
            if (mine && t1 + j * TR < nt) {
                const Pack<T, 4> x4 = *reinterpret_cast<const Pack<T, 4> *>(x + j * TR * CB), dt4 = *reinterpret_cast<const Pack<T, 4> *>(x + (TC + j * TR) * CB);
                float2 lo = make_float2(wide(dt4.v[0]) + bias[0], wide(dt4.v[1]) + bias[1]), hi = make_float2(wide(dt4.v[2]) + bias[2], wide(dt4.v[3]) + bias[3]);
                if (a.softplus) {
                    lo = softplus2(lo);
                    hi = softplus2(hi);
                }
                d = make_float4(lo.x, lo.y, hi.x, hi.y);
                if (!VEC) {
                    if (ch + 1 >= nc) d.y = 0.f;
                    if (ch + 2 >= nc) d.z = 0.f;
                    if (ch + 3 >= nc) d.w = 0.f;
                }
                dx = make_float4(d.x * wide(x4.v[0]), d.y * wide(x4.v[1]), d.z * wide(x4.v[2]), d.w * wide(x4.v[3]));
            }
            *reinterpret_cast<float4 *>(sd + j * TR * CB) = d;
            *reinterpret_cast<float4 *>(sd + (TC + j * TR) * CB) = dx;
        }
#pragma unroll
        for (int j = 0; j < BC; j++) {
            const int i = tid + j * SCAN_THREADS, r = i / L, n = i % L * 4, t = r % TC;
            if (PASS == ENDS && r >= TC) break;
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
            if (t < nt && n < N) {
                const Pack<T, 4> b4 = *reinterpret_cast<const Pack<T, 4> *>(b + 4 * i);
                v = make_float4(wide(b4.v[0]), wide(b4.v[1]), wide(b4.v[2]), wide(b4.v[3]));
            }
            *reinterpret_cast<float4 *>(sb + 4 * i) = v;
        }
    };
    // the rows of chunk k that have been walked: skip, gate, out
    auto send = [&](int k) {  // called for 0, 1, 2, ..
        const T *x = raw(k) + t1 * CB + ch;
        const float *sd = ready(k) + t1 * CB + ch;
        const int nt = min(TC, rows - k * TC);
        if (mine) {
#pragma unroll
            for (int j = 0; j < Z::PIECES; j++) {
                if (t1 + j * TR >= nt) break;
                const float4 y4 = *reinterpret_cast<const float4 *>(sd + j * TR * CB);
                float y[4] = {y4.x, y4.y, y4.z, y4.w};
                if (a.d) {
                    const Pack<T, 4> x4 = *reinterpret_cast<const Pack<T, 4> *>(x + j * TR * CB);
#pragma unroll
                    for (int e = 0; e < 4; e++) if (VEC || ch + e < nc) y[e] = fmaf(skip[e], wide(x4.v[e]), y[e]);
                }
                if (pz) {
                    const Pack<T, 4> z4 = *reinterpret_cast<const Pack<T, 4> *>(x + (2 * TC + j * TR) * CB);
#pragma unroll
                    for (int e = 0; e < 4; e++) y[e] *= silu(wide(z4.v[e]));
                }
                T *to = pd + j * TR * a.dst_stride;
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
        pd += TC * a.dst_stride;
    };
    fetch(0);
    fetch(1);
    // ===== the states
    const int cl = warp * Z::WC + g * CI;  // the lane's channels, counted from c0
    Two h[CI][2], rate[CI][2];
    float total[CI];
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
        rate[ci][0] = two(r.x, r.y); rate[ci][1] = two(r.z, r.w);
        h[ci][0] = two(s.x, s.y); h[ci][1] = two(s.z, s.w);
    }
    // ===== chunk k's rows, all of them (those behind the last change nothing), in blocks of up to 16 whose loads can go ahead of the chains: results are written behind the block
    auto walk = [&](int k) {
        float *sd = ready(k);
        const float *sx = sd + TC * CB, *sb = sx + TC * CB, *sc = sb + TC * NP;
#pragma unroll 1
        for (int tb = 0; tb < TC; tb += TB) {
            float v[TB / 4][CI];
            const bool hi = (p & (L / 2)) != 0, odd = (p & (L / 4)) != 0;
#pragma unroll
            for (int t0 = 0; t0 < TB; t0 += 4) {
                float y[4][CI];
#pragma unroll
                for (int u = 0; u < 4; u++) {
                    const int t = tb + t0 + u;
                    const ulonglong2 b2 = *reinterpret_cast<const ulonglong2 *>(sb + t * NP + 4 * p);
                    const ulonglong2 c2 = PASS == ENDS ? b2 : *reinterpret_cast<const ulonglong2 *>(sc + t * NP + 4 * p);
                    const Pack<float, CI> d = *reinterpret_cast<const Pack<float, CI> *>(sd + t * CB + cl), dx = *reinterpret_cast<const Pack<float, CI> *>(sx + t * CB + cl);
#pragma unroll
                    for (int ci = 0; ci < CI; ci++) {
                        if (PASS == ENDS) total[ci] += d.v[ci];
                        const Two dd = two(d.v[ci], d.v[ci]), xx = two(dx.v[ci], dx.v[ci]);
                        const float2 e0 = each(mul2(dd, rate[ci][0])), e1 = each(mul2(dd, rate[ci][1]));
                        h[ci][0] = fma2(two(ex2(e0.x), ex2(e0.y)), h[ci][0], mul2(xx, b2.x));
                        h[ci][1] = fma2(two(ex2(e1.x), ex2(e1.y)), h[ci][1], mul2(xx, b2.y));
                        if (PASS != ENDS) {
                            const float2 s = each(fma2(c2.y, h[ci][1], mul2(c2.x, h[ci][0])));
                            y[u][ci] = s.x + s.y;
                        }
                    }
                }
                if (PASS != ENDS) {
                    // sums over the channel's lanes: those of one half keep rows 2 and 3, then a quarter one row each
#pragma unroll
                    for (int ci = 0; ci < CI; ci++) {
                        const float s0 = hi ? y[0][ci] : y[2][ci], s1 = hi ? y[1][ci] : y[3][ci], k0 = hi ? y[2][ci] : y[0][ci], k1 = hi ? y[3][ci] : y[1][ci];
                        const float w0 = k0 + __shfl_xor_sync(0xffffffffu, s0, L / 2), w1 = k1 + __shfl_xor_sync(0xffffffffu, s1, L / 2);
                        const float s = odd ? w0 : w1, kk = odd ? w1 : w0;
                        v[t0 / 4][ci] = kk + __shfl_xor_sync(0xffffffffu, s, L / 4);
                    }
#pragma unroll
                    for (int n = L / 8; n >= 1; n /= 2) {
#pragma unroll
                        for (int ci = 0; ci < CI; ci++) v[t0 / 4][ci] += __shfl_xor_sync(0xffffffffu, v[t0 / 4][ci], n);
                    }
                }
            }
            if (PASS != ENDS) {
                __syncwarp();  // the warp has read these rows of its channels in sd: their results take the place
                if ((p & (L / 4 - 1)) == 0) {
#pragma unroll
                    for (int i = 0; i < TB / 4; i++) {
                        Pack<float, CI> out;
#pragma unroll
                        for (int ci = 0; ci < CI; ci++) out.v[ci] = v[i][ci];
                        *reinterpret_cast<Pack<float, CI> *>(sd + (tb + 4 * i + 2 * hi + odd) * CB + cl) = out;
                    }
                }
            }
        }
    };
    cp_async_wait<1>();
    stage(0);
    __syncthreads();
    for (int k = 0; k < chunks; k++) {
        if (PASS != ENDS && k > 0) send(k - 1);
        fetch(k + 2);
        cp_async_wait<1>();
        stage(k + 1);
        walk(k);
        __syncthreads();
    }
    pdl_trigger();
    if (PASS != ENDS) send(chunks - 1);
    // ===== where the states go: the stretch's place, or the slot
#pragma unroll
    for (int ci = 0; ci < CI; ci++) {
        if (cl + ci >= nc) continue;
        const int c = c0 + cl + ci;
        const float2 s0 = each(h[ci][0]), s1 = each(h[ci][1]);
        const float4 s = make_float4(s0.x, s0.y, s1.x, s1.y);
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
    p.per_lane = p.lanes == 4 ? 2 : p.lanes == 32 ? 4 : 4;
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
    constexpr int CI = L == 4 ? 2 : 4;
    using Z = ScanSizes<T, L, CI>;
    const auto kern = ssm_scan_kernel<T, L, CI, VEC, PASS>;
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
    OPX_REQUIRE((longest + CONV_ROWS_MIN - 1) / CONV_ROWS_MIN <= 65535, B200_ERR_UNSUPPORTED, "%s: at most %d rows of a sequence", who, 65535 * CONV_ROWS_MIN);
    const ConvArgs c = {{a->seq_info, a->n_seq, a->n_slots, a->n_tokens, longest}, a->x, a->x_stride, a->w, a->bias, a->tail, a->slot_stride, a->dst, a->dst_stride, a->channels, a->taps, a->silu, 0};
    const cudaStream_t st = (cudaStream_t)stream;
    constexpr int CV = 4;
    const bool vec = on(CV * type_size(a->type), {a->x, a->dst}) && ((a->x_stride | a->dst_stride | a->channels) & (CV - 1)) == 0;
    if (a->type == B200_TYPE_F32) return vec ? launch_conv_taps<float, CV>(c, st) : launch_conv_taps<float, 1>(c, st);
    if (a->type == B200_TYPE_F16) return vec ? launch_conv_taps<__half, CV>(c, st) : launch_conv_taps<__half, 1>(c, st);
    return vec ? launch_conv_taps<__nv_bfloat16, CV>(c, st) : launch_conv_taps<__nv_bfloat16, 1>(c, st);
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
    const size_t four = 4 * type_size(a->type);
    const bool bc_pieces = on(four, {a->b, a->c}) && ((a->b_stride | a->c_stride | a->d_state) & 3) == 0;
    const ScanArgs s = {{a->seq_info, a->n_seq, a->n_slots, a->n_tokens, longest}, a->x, a->dt, a->b, a->c, a->z, a->x_stride, a->dt_stride, a->b_stride, a->c_stride, a->z_stride, a->a, a->dt_bias, a->d,
                        a->from ? a->from : a->state, a->from ? a->from_stride : a->slot_stride, a->state, a->slot_stride, a->dst, a->dst_stride, a->channels, a->d_state, per_group, a->softplus, bc_pieces,
                        p.stretch, p.n_stretch, ends, ends ? ends + (size_t)a->n_seq * (p.n_stretch + 1) * a->channels * a->d_state : nullptr};
    const bool vec = per_group % 4 == 0 && on(four, {a->x, a->dt, a->z, a->dst}) && ((a->x_stride | a->dt_stride | a->dst_stride | (a->z ? a->z_stride : 0)) & 3) == 0;
    const bool states16 = (a->d_state & 3) == 0 && ((s.slot_stride | s.from_stride) & 3) == 0 && on(16, {s.state, s.from, a->a});
    const cudaStream_t st = (cudaStream_t)stream;
    if (a->type == B200_TYPE_F32) return launch_scan_type<float>(s, p, vec, states16, st);
    if (a->type == B200_TYPE_F16) return launch_scan_type<__half>(s, p, vec, states16, st);
    return launch_scan_type<__nv_bfloat16>(s, p, vec, states16, st);
}

}  // extern "C"
