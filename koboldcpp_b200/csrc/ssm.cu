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
// y * sigmoid(y): relative error 2^-21, and |y| 2^-23 more below 0 by the exponent's rounding; -0 below -87, where e^-y or its reciprocal leaves f32's normal numbers
__device__ __forceinline__ float silu(float y) { return y * rcp(1.0f + ex2(-LOG2E * y)); }

// two floats that are worked on by one instruction
using Two = unsigned long long;
__device__ __forceinline__ Two two(float lo, float hi) { Two r; asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi)); return r; }
__device__ __forceinline__ float2 each(Two x) { float2 r; asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(x)); return r; }
__device__ __forceinline__ Two fma2(Two x, Two y, Two z) { Two r; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(x), "l"(y), "l"(z)); return r; }
__device__ __forceinline__ Two add2(Two x, Two y) { Two r; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y)); return r; }
__device__ __forceinline__ Two mul2(Two x, Two y) { Two r; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y)); return r; }

// silu of two values
__device__ __forceinline__ Two silu2(Two z) {
    const float2 turn = each(mul2(z, two(-LOG2E, -LOG2E))), all = each(add2(two(ex2(turn.x), ex2(turn.y)), two(1.0f, 1.0f)));
    return mul2(z, two(rcp(all.x), rcp(all.y)));
}

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
            const int left = nt - g * CONV_GROUP;
            P *to = &ring[g % CONV_GROUPS][0][threadIdx.x];
#pragma unroll
            for (int u = 0; u < CONV_GROUP; u++) {
                if (u < left) {
                    if constexpr (sizeof(P) == 16) cp_async16(to + u * CONV_THREADS, in_row + u * a.x_stride);
                    else cp_async8(to + u * CONV_THREADS, in_row + u * a.x_stride);
                }
            }
            in_row += CONV_GROUP * a.x_stride;
            cp_async_commit();
        };
#pragma unroll
        for (int g = 0; g < CONV_GROUPS - 1; g++) fetch(g);
        for (int g = 0; g * CONV_GROUP < nt; g++) {
            cp_async_wait<CONV_GROUPS - 2>();
            const P *from = &ring[g % CONV_GROUPS][0][threadIdx.x];
            if ((g + 1) * CONV_GROUP <= nt) {
#pragma unroll
                for (int u = 0; u < CONV_GROUP; u++) turn(from[u * CONV_THREADS]);
            } else {
                for (int u = 0; g * CONV_GROUP + u < nt; u++) turn(from[u * CONV_THREADS]);
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
    // the ring pays where there is something to wait for (5330 rows, bf16: 36 us with it, 51 without); for 64 sequences of one or three rows it is 4.2 to 4.4 us either way, and shared memory is left alone
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
    // stretches: rows of one, how many a sequence may have; where end states and sums of d wait, and the states of sequences that are cut, which the last of their stretches overwrites.  A stretch's
    // place is its first row / stretch: those that have a place are whole, so no two share one, and there are n_tokens / stretch of them whatever the number of sequences.
    int32_t stretch, n_stretch;
    float *ends, *starts, *sums;
};

// -|x|, and -128 below it (e^-128 is zero here; NaN stays)
__device__ __forceinline__ float down(float x) {
    float r;
    asm("max.NaN.f32 %0, %1, 0fC3000000;" : "=f"(r) : "f"(-fabsf(x)));
    return r;
}
// ln(1 + e^x) = max(x, 0) + ln(1 + e^-|x|), and ln(1 + e) = e P(e) on [0, 1] with a polynomial whose relative error is smallest at its largest (fitted by weighted least squares on
// Chebyshev points; 1.8e-7 with the roundings of f32): one exponential on the special function unit and nothing else there, no overflow, no cancellation.  What the exponential's argument loses, its
// rounding and what LOG2E has not of log2 e, is made good to first order: where e is small all of the result is e, and such steps are the usual ones of a trained layer.  (Relative error for x of
// -12 .. -6: 2.6e-7 at most, 7.0e-8 root mean square, -5e-8 in the mean; without it 8.9e-7, 2.5e-7 and +7e-8, and more further out.  Four prompts of 2048 rows: 448 -> 455 us.)
__device__ __forceinline__ float2 softplus2(float2 x) {
    auto both = [](float v) { return two(v, v); };
    const Two far = two(down(x.x), down(x.y)), turn = mul2(far, both(LOG2E));
    const float2 v = each(turn);
    Two e = two(ex2(v.x), ex2(v.y));
    e = fma2(e, fma2(turn, both(1.90465421e-9f), fma2(turn, both(-0x1.62e430p-1f), far)), e);
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
// .. of one value.  (Not as one of two: with that the compiler gives the kernel of single rows 64 registers and lets it ask for its states later, 25.5 -> 28.4 us for 96 rows of 8192 channels.)
__device__ __forceinline__ float softplus(float x) {
    const float far = down(x), turn = far * LOG2E;
    float e = ex2(turn);
    e = fmaf(e, fmaf(turn, 1.90465421e-9f, fmaf(turn, -0x1.62e430p-1f, far)), e);
    float p = 0.0052326764f;
    p = fmaf(p, e, -0.0295051672f);
    p = fmaf(p, e, 0.0782258362f);
    p = fmaf(p, e, -0.136632353f);
    p = fmaf(p, e, 0.191060022f);
    p = fmaf(p, e, -0.248429805f);
    p = fmaf(p, e, 0.333190978f);
    p = fmaf(p, e, -0.499994934f);
    return fmaf(fmaf(p, e, 1.0f), e, fmaxf(x, 0.f));
}

// Rates of -inf and +inf count as the largest numbers of f32, so that a row with d = 0 (and those behind a sequence's last, which are walked as such) leaves their states as they are.  NaN stays.
__device__ __forceinline__ float finite(float x) {
    float r;
    asm("max.NaN.f32 %0, %1, 0fFF7FFFFF;" : "=f"(r) : "f"(x));
    asm("min.NaN.f32 %0, %0, 0f7F7FFFFF;" : "+f"(r));
    return r;
}

// 2^(2 half) * s + e for two states.  In two steps, since a stretch over which states grow has a factor that f32 may not hold, and what it meets may be zero or small enough to stay in range.
// (The bounds keep zeros and infinities what they are; a normal number is infinite behind the upper one, and below 2^-124 behind the lower.)
__device__ __forceinline__ Two carried(Two half, Two s, Two e) {
    const float2 v = each(half);
    const Two f = two(ex2(fmaxf(fminf(v.x, 127.f), -126.f)), ex2(fmaxf(fminf(v.y, 127.f), -126.f)));
    return fma2(f, mul2(f, s), e);
}

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
__device__ __forceinline__ float4 load_row4(const T *row, int n0, int d_state, bool pieces) {
    if (pieces) {
        if (n0 >= d_state) return make_float4(0.f, 0.f, 0.f, 0.f);
        const Pack<T, 4> v = *reinterpret_cast<const Pack<T, 4> *>(row + n0);
        return make_float4(wide(v.v[0]), wide(v.v[1]), wide(v.v[2]), wide(v.v[3]));
    }
    float4 r;
    r.x = n0 < d_state ? wide(row[n0]) : 0.f;
    r.y = n0 + 1 < d_state ? wide(row[n0 + 1]) : 0.f;
    r.z = n0 + 2 < d_state ? wide(row[n0 + 2]) : 0.f;
    r.w = n0 + 3 < d_state ? wide(row[n0 + 3]) : 0.f;
    return r;
}

// ===== one row a sequence.  A warp takes 32 channels; L lanes share a channel, a lane four of its states, so that a load of the warp is 512 consecutive bytes of the state.  What a channel
// needs by itself (d, d x, z) is made by one lane and handed to the other L - 1; the sums of L channels are exchanged so that each lane ends up with one of them.  What takes longest is asked for
// first.  What bounds it is waiting for memory with 38 % of an SM's warps there (96 sequences of 8192 channels, 16 states: 25.5 us, 4.2 TB/s;
// half of the cycles between two instructions of a warp are waits for loads, instructions are issued 58 % of the time); sequences one after the other in a warp, whose rates would stay, are 45 us.
constexpr int STEP_WARPS = 2;
template <typename T, int L, bool VEC>
__global__ void __launch_bounds__(32 * STEP_WARPS) ssm_step_kernel(const ScanArgs a) {
    constexpr int G = 32 / L, U = 4;  // channels of a round; rounds whose loads travel together
    pdl_enter();
    const int lane = threadIdx.x & 31, p = lane % L, g = lane / L;
    const int c0 = (blockIdx.x * STEP_WARPS + (threadIdx.x >> 5)) * 32, left = a.channels - c0;  // (left > 31: no channel has to be asked for)
    const Seq q = seq_of(a.step, blockIdx.y);
    if (left <= 0 || q.count == 0) return;
    const int64_t row = q.first;
    // the lane's first piece of the states and rates, and how far the next channel's is
    const int64_t at = (int64_t)(c0 + g) * a.d_state;
    const int step = G * a.d_state;
    const float *from = a.from + (int64_t)q.slot * a.from_stride + at, *rates = a.a + at;
    float *state = a.state + (int64_t)q.slot * a.slot_stride + at;
    float4 h[U], rate[U];
    auto load = [&](int i0) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            h[u] = rate[u] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (left > 31 || G * (i0 + u) + g < left) {
                if (!q.begins) h[u] = load_states<VEC>(from + (i0 + u) * step, 4 * p, a.d_state);
                rate[u] = load_states<VEC>(rates + (i0 + u) * step, 4 * p, a.d_state);
            }
        }
    };
    load(0);
    // b and c of the warp's channels, which are of one group as a rule
    const bool groups = a.per_group < a.channels;
    const int group0 = groups ? c0 / a.per_group : 0;
    const bool one_group = !groups || min(c0 + 31, a.channels - 1) < (group0 + 1) * a.per_group;
    const T *pb = (const T *)a.b + row * a.b_stride, *pc = (const T *)a.c + row * a.c_stride;
    float4 b = load_row4(pb + (int64_t)group0 * a.d_state, 4 * p, a.d_state, a.bc_pieces), cc = load_row4(pc + (int64_t)group0 * a.d_state, 4 * p, a.d_state, a.bc_pieces);
    const int mine = c0 + G * p + g;  // the channel that is this lane's by itself
    const bool ok = mine < a.channels;
    float d = 0.f, x = 0.f, z = 0.f, skip = 0.f;
    if (ok) {
        if (a.z) z = wide(((const T *)a.z)[row * a.z_stride + mine]);
        if (a.d) skip = a.d[mine];
        d = wide(((const T *)a.dt)[row * a.dt_stride + mine]) + (a.dt_bias ? a.dt_bias[mine] : 0.f);
        x = wide(((const T *)a.x)[row * a.x_stride + mine]);
        if (a.softplus) d = softplus(d);
    }
    const float dx = d * x;
    d *= LOG2E;
    float sum[L];
#pragma unroll
    for (int i0 = 0; i0 < L; i0 += U) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (!one_group) {
                const int64_t of = (int64_t)(min(c0 + G * (i0 + u) + g, a.channels - 1) / a.per_group) * a.d_state;
                b = load_row4(pb + of, 4 * p, a.d_state, a.bc_pieces);
                cc = load_row4(pc + of, 4 * p, a.d_state, a.bc_pieces);
            }
            const float dc = __shfl_sync(0xffffffffu, d, g * L + i0 + u), dxc = __shfl_sync(0xffffffffu, dx, g * L + i0 + u);
            const Two dd = two(dc, dc), xx = two(dxc, dxc);
            const float2 e0 = each(mul2(dd, two(finite(rate[u].x), finite(rate[u].y)))), e1 = each(mul2(dd, two(finite(rate[u].z), finite(rate[u].w))));
            const Two s0 = fma2(two(ex2(e0.x), ex2(e0.y)), two(h[u].x, h[u].y), mul2(xx, two(b.x, b.y))), s1 = fma2(two(ex2(e1.x), ex2(e1.y)), two(h[u].z, h[u].w), mul2(xx, two(b.z, b.w)));
            float2 v0 = each(s0), v1 = each(s1);
            if (left > 31 || G * (i0 + u) + g < left) store_states<VEC>(state + (i0 + u) * step, 4 * p, a.d_state, make_float4(v0.x, v0.y, v1.x, v1.y));
            // numbers behind d_state are no part of the sum (0 times an infinite d x is no number)
            if constexpr (!VEC) {
                if (4 * p + 1 >= a.d_state) v0.y = 0.f;
                if (4 * p + 2 >= a.d_state) v1.x = 0.f;
                if (4 * p + 3 >= a.d_state) v1.y = 0.f;
            }
            const float2 y = each(fma2(two(cc.x, cc.y), two(v0.x, v0.y), mul2(two(cc.z, cc.w), two(v1.x, v1.y))));
            sum[i0 + u] = 4 * p < a.d_state ? y.x + y.y : 0.f;
        }
        if (i0 + U < L) load(i0 + U);
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
        if (a.d) y = fmaf(skip, x, y);
        if (a.z) y *= silu(z);
        ((T *)a.dst)[row * a.dst_stride + mine] = narrow<T>(y);
    }
}

// ===== several rows a sequence
// A channel is L lanes, NS of its states each: with 16 states a lane is a channel.  What belongs to a channel alone (dt, x, z, the result) then never leaves the lane's registers, and the 16 exponentials
// and multiply-adds of a row are chains that run side by side.  b and c of a chunk of rows wait in shared memory, where all lanes read the same words.  Rows go in groups of TG; lane p of a channel makes d and d x of the group's rows p, p + L, ..,
// and sends off their results; the next group's rows are loaded meanwhile.
// What bounds it: exponentials, d_state + 3 for each row and channel at 16 a cycle and SM (four prompts of 2048 rows x 8192 channels: 283 us), and that 1024 warps make two on some schedulers and one
// on others: 455 us, 445 cycles a row, of which the unit has 304 to do where there are two.  Some of the exponentials made by multiply-adds (two or four of 16 as polynomials) gave nothing: the other instructions, 100 a row in all, fill up what that leaves.
constexpr int SCAN_WARPS = 4, SCAN_THREADS = 32 * SCAN_WARPS;
// the things that a CTA can be there for: a whole sequence, with few CTAs or with many; the state at the end of a stretch as if it began from nothing (the first one: from the sequence's state), and the sum of
// its d; a stretch's rows, from the states and sums of those before it
enum Pass { WHOLE, MANY, ENDS, ROWS };
template <int L, int NS>
struct ScanSizes {
    static constexpr int CB = SCAN_THREADS / L, NP = NS * L;       // channels of a CTA; states of a channel, those behind d_state included
    static constexpr int TC = NP <= 16 ? 32 : 16;                  // rows of a chunk
    static constexpr int PIECES = (2 * TC * NP / 4 + SCAN_THREADS - 1) / SCAN_THREADS;  // pieces of four numbers of b or c that a thread fetches
};
// Rows of a group, and CTAs that an SM is to hold.  A lane that is a channel, in few CTAs: long groups in the order that the compiler gives them with 255 registers (four long prompts, 1.7 CTAs
// an SM: 16 rows 455 us, 8 rows 462).  Where there are CTAs for every place that an SM has, more places are worth more: short groups, four CTAs (128 sequences of
// 48 rows, 8192 channels: 287 us, 357 the other way; of 5 rows, where a long group would also walk what is not there, 81 and 187).  Stretches stay with the first: one prompt of 4096 rows of 2048
// channels 100 us, 122 the other way; of 5120 channels 250 and 259; of 8192 channels 405 and 378, where the other way would be the better one.  With exchanges between lanes there is one way, four CTAs
// and groups of 8 rows (64 states: 189 us, with three CTAs 300).
constexpr int SCAN_SHORT = 32;  // rows up to which sequences take the second way whatever the number of CTAs
constexpr int scan_rows(int lanes, int pass) { return lanes > 1 ? 8 : pass == MANY ? 4 : 16; }
constexpr int scan_ctas(int lanes, int pass) { return lanes > 1 || pass == MANY ? 4 : 2; }
// PADS: lanes have numbers behind d_state, which results must not see.  (Kernels of their own: the second way through a group of rows that this takes would make the others 2 to 7 % longer, one prompt of
// 4096 rows of 2048 channels and 16 states 101 -> 107 us; with 9 to 14 states it is 2 to 5 % longer than without, with 5 states 10 %.)
template <typename T, int L, int NS, int PASS, bool PADS>
__global__ void __launch_bounds__(SCAN_THREADS, scan_ctas(L, PASS)) ssm_scan_kernel(const ScanArgs a) {
    using Z = ScanSizes<L, NS>;
    constexpr int CB = Z::CB, NP = Z::NP, TC = Z::TC, NQ = NS / 4, TG = scan_rows(L, PASS), MT = TG / L;  // TG: rows of a group; MT: those that a lane makes ready
    __shared__ __align__(16) float sbc[2][2][TC][NP];  // [chunk & 1][b, c]
    pdl_wait();  // (the kernel behind is let in at the end: its CTAs would wait in places of this one's.  Four long prompts 455 us, let in at the beginning 456)
    const int tid = threadIdx.x, lane = tid & 31, p = lane % L;
    const Seq q = seq_of(a.step, blockIdx.z);
    const int N = a.d_state, blocks = (a.per_group + CB - 1) / CB, group = blockIdx.x / blocks, in_group = (blockIdx.x - group * blocks) * CB + tid / L;
    const bool mine = in_group < a.per_group;
    const int c = group * a.per_group + min(in_group, a.per_group - 1);  // the lane's channel (those behind the group's last walk along with it and leave nothing)
    constexpr bool ALL = PASS == WHOLE || PASS == MANY;
    // what is done to every row by itself is done to two at a time: one prompt of 4096 rows of 2048 channels 103 -> 100 us, six ragged ones 273 -> 270; short groups are better off without (128 sequences of 48
    // rows 287 -> 291)
    constexpr bool PAIRS = MT > 1 && PASS != MANY;
    const int stretch = ALL ? 0 : blockIdx.y, begin = ALL ? 0 : stretch * a.stretch, end = ALL ? q.count : min(q.count, begin + a.stretch);
    if (begin >= end) return;
    const bool last = end == q.count;
    if (PASS == ENDS && last) return;  // (nobody asks for its end)
    const int64_t first = q.first + begin;
    const int rows = end - begin;
    const T *pb = (const T *)a.b + first * a.b_stride + (int64_t)group * N, *pc = (const T *)a.c + first * a.c_stride + (int64_t)group * N;
    // ===== b and c of a chunk: to registers, then to shared memory, zeros behind d_state and behind the last row
    Pack<T, 4> held[Z::PIECES];
    auto fetch = [&](int r0) {
#pragma unroll
        for (int j = 0; j < Z::PIECES; j++) {
            const int i = tid + j * SCAN_THREADS, r = i / (NP / 4), n = i % (NP / 4) * 4, t = r % TC;
            if (r >= (PASS == ENDS ? TC : 2 * TC) || r0 + t >= rows) continue;
            const T *row = (r < TC ? pb + (r0 + t) * a.b_stride : pc + (r0 + t) * a.c_stride) + n;
            if (a.bc_pieces) {
                if (n < N) held[j] = *reinterpret_cast<const Pack<T, 4> *>(row);
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++) held[j].v[e] = n + e < N ? row[e] : narrow<T>(0.f);
            }
        }
    };
    auto keep = [&](int r0, int buf) {
#pragma unroll
        for (int j = 0; j < Z::PIECES; j++) {
            const int i = tid + j * SCAN_THREADS, r = i / (NP / 4), n = i % (NP / 4) * 4, t = r % TC;
            if (r >= (PASS == ENDS ? TC : 2 * TC)) continue;
            const bool there = r0 + t < rows && n < N;
            *reinterpret_cast<float4 *>(&sbc[buf][0][0][0] + 4 * i) =
                there ? make_float4(wide(held[j].v[0]), wide(held[j].v[1]), wide(held[j].v[2]), wide(held[j].v[3])) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
    };
    // ===== the channel's rows: lane p has rows p, p + L, .. of a group
    const T *px = (const T *)a.x + (first + p) * a.x_stride + c, *pdt = (const T *)a.dt + (first + p) * a.dt_stride + c, *pz = a.z ? (const T *)a.z + (first + p) * a.z_stride + c : nullptr;
    T *pd = (T *)a.dst + (first + p) * a.dst_stride + c;
    const float bias = a.dt_bias ? a.dt_bias[c] : 0.f, skip = PASS != ENDS && a.d ? a.d[c] : 0.f;
    T nx[MT], ndt[MT], nz[MT];
    auto load = [&](int r0) {
        if (r0 + TG <= rows) {
#pragma unroll
            for (int j = 0; j < MT; j++) {
                nx[j] = px[j * L * a.x_stride];
                ndt[j] = pdt[j * L * a.dt_stride];
                if (PASS != ENDS && pz) nz[j] = pz[j * L * a.z_stride];
            }
        } else {
#pragma unroll
            for (int j = 0; j < MT; j++) {
                const bool there = r0 + j * L + p < rows;
                nx[j] = there ? px[j * L * a.x_stride] : narrow<T>(0.f);
                ndt[j] = there ? pdt[j * L * a.dt_stride] : narrow<T>(0.f);
                if (PASS != ENDS && pz) nz[j] = there ? pz[j * L * a.z_stride] : narrow<T>(0.f);
            }
        }
        px += TG * a.x_stride;
        pdt += TG * a.dt_stride;
        if (pz) pz += TG * a.z_stride;
    };
    fetch(0);
    load(0);
    // ===== the states
    Two h[NS / 2], rate[NS / 2];
    double total = 0.0;  // (a stretch may be long: terms of one size would all be rounded the same way)
    const bool pieces = (N & 3) == 0 && ((a.slot_stride | a.from_stride) & 3) == 0 && (((uintptr_t)a.state | (uintptr_t)a.from | (uintptr_t)a.a) & 15) == 0;
    // they lie as [d_state][channels], so that neighbouring lanes read neighbouring words
    const int64_t ends_row = (int64_t)a.channels * N;
    const int place = ALL ? 0 : (int)(q.first / a.stretch);  // of the sequence's first stretch; the others' places follow it
    auto load_end = [&](const float *from, int n) {
        const float *q4 = from + (int64_t)n * a.channels;
        return make_float4(n < N ? q4[0] : 0.f, n + 1 < N ? q4[a.channels] : 0.f, n + 2 < N ? q4[2 * (int64_t)a.channels] : 0.f, n + 3 < N ? q4[3 * (int64_t)a.channels] : 0.f);
    };
    auto store_end = [&](float *to, int n, float4 v) {
        float *q4 = to + (int64_t)n * a.channels;
        if (n < N) q4[0] = v.x;
        if (n + 1 < N) q4[a.channels] = v.y;
        if (n + 2 < N) q4[2 * (int64_t)a.channels] = v.z;
        if (n + 3 < N) q4[3 * (int64_t)a.channels] = v.w;
    };
    float *ends = a.ends + place * ends_row + c, *starts = a.starts + place * ends_row + c, *sums = a.sums + (int64_t)place * a.channels + c;
#pragma unroll
    for (int i = 0; i < NQ; i++) {
        const int n = 4 * (i * L + p);  // (the channel's lanes side by side: their loads of b and c too)
        const float *pa = a.a + (int64_t)c * N;
        float4 r = pieces ? load_states<true>(pa, n, N) : load_states<false>(pa, n, N), s = make_float4(0.f, 0.f, 0.f, 0.f);
        if (stretch == 0 && !q.begins && (PASS != ROWS || last)) {
            const float *from = a.from + (int64_t)q.slot * a.from_stride + (int64_t)c * N;
            s = pieces ? load_states<true>(from, n, N) : load_states<false>(from, n, N);
        }
        if (PASS == ENDS && stretch == 0 && mine) store_end(starts, n, s);
        r.x = finite(r.x * LOG2E); r.y = finite(r.y * LOG2E); r.z = finite(r.z * LOG2E); r.w = finite(r.w * LOG2E);
        if (PASS == ROWS && !(stretch == 0 && last)) {
            s = load_end(stretch > 0 ? ends : starts, n);
            Two lo = two(s.x, s.y), hi = two(s.z, s.w);
#pragma unroll 4
            for (int j = 1; j < stretch; j++) {
                const float4 e = load_end(ends + j * ends_row, n);
                const float d = 0.5f * sums[(int64_t)j * a.channels];
                lo = carried(mul2(two(d, d), two(r.x, r.y)), lo, two(e.x, e.y));
                hi = carried(mul2(two(d, d), two(r.z, r.w)), hi, two(e.z, e.w));
            }
            s = make_float4(each(lo).x, each(lo).y, each(hi).x, each(hi).y);
            // (numbers behind d_state: 0 times what an infinite sum of d makes of them is none)
            if (PADS && n + 3 >= N) s = make_float4(n < N ? s.x : 0.f, n + 1 < N ? s.y : 0.f, n + 2 < N ? s.z : 0.f, 0.f);
        }
        rate[2 * i] = two(r.x, r.y); rate[2 * i + 1] = two(r.z, r.w);
        h[2 * i] = two(s.x, s.y); h[2 * i + 1] = two(s.z, s.w);
    }
    keep(0, 0);
    __syncthreads();
    for (int r0 = 0, buf = 0; r0 < rows; r0 += TC, buf ^= 1) {
        if (r0 + TC < rows) fetch(r0 + TC);
#pragma unroll 1
        for (int tg = 0; tg < TC && r0 + tg < rows; tg += TG) {
            float d[MT], x[MT], dx[MT], z[MT];
#pragma unroll
            for (int j = 0; j < MT; j++) {
                x[j] = wide(nx[j]);
                if (PASS != ENDS) z[j] = wide(nz[j]);
                d[j] = wide(ndt[j]);
            }
            if constexpr (!PAIRS) {
#pragma unroll
                for (int j = 0; j < MT; j++) d[j] += bias;
            } else {
#pragma unroll
                for (int j = 0; j < MT; j += 2) {
                    const float2 v = each(add2(two(d[j], d[j + 1]), two(bias, bias)));
                    d[j] = v.x; d[j + 1] = v.y;
                }
            }
            if (a.softplus) {
                if constexpr (MT == 1) {
                    d[0] = softplus(d[0]);
                } else {
#pragma unroll
                    for (int j = 0; j < MT; j += 2) {
                        const float2 s = softplus2(make_float2(d[j], d[j + 1]));
                        d[j] = s.x; d[j + 1] = s.y;
                    }
                }
            }
            const bool full = r0 + tg + TG <= rows;
            if (!full) {  // rows behind the last leave the states as they are
#pragma unroll
                for (int j = 0; j < MT; j++) if (r0 + tg + j * L + p >= rows) d[j] = 0.f;
            }
            if constexpr (!PAIRS) {
#pragma unroll
                for (int j = 0; j < MT; j++) dx[j] = d[j] * x[j];
            } else {
#pragma unroll
                for (int j = 0; j < MT; j += 2) {
                    const float2 v = each(mul2(two(d[j], d[j + 1]), two(x[j], x[j + 1])));
                    dx[j] = v.x; dx[j + 1] = v.y;
                }
            }
            if (PASS == ENDS) {
                float some = d[0];
#pragma unroll
                for (int j = 1; j < MT; j++) some += d[j];
                total += some;
            }
            load(r0 + tg + TG);
            float ds[TG], dxs[TG];  // of all the group's rows
#pragma unroll
            for (int t = 0; t < TG; t++) {
                ds[t] = L == 1 ? d[t / L] : __shfl_sync(0xffffffffu, d[t / L], lane - p + t % L);
                dxs[t] = L == 1 ? dx[t / L] : __shfl_sync(0xffffffffu, dx[t / L], lane - p + t % L);
            }
            float y[TG];
            auto walk = [&](int t, float d_row, float dx_row, auto whole) {  // row t of the group; whole: numbers behind d_state are treated as all others
                const ulonglong2 *b2 = reinterpret_cast<const ulonglong2 *>(&sbc[buf][0][tg + t][4 * p]), *c2 = reinterpret_cast<const ulonglong2 *>(&sbc[buf][1][tg + t][4 * p]);
                Two sum = 0;
#pragma unroll
                for (int i = 0; i < NQ; i++) {
                    const ulonglong2 bv = b2[i * L];
                    const int n = 4 * (i * L + p);
                    auto pair = [&](float v, int k) { return whole ? two(v, v) : two(n + k < N ? v : 0.f, n + k + 1 < N ? v : 0.f); };
                    const float2 e0 = each(mul2(pair(d_row, 0), rate[2 * i])), e1 = each(mul2(pair(d_row, 2), rate[2 * i + 1]));
                    h[2 * i] = fma2(two(ex2(e0.x), ex2(e0.y)), h[2 * i], mul2(pair(dx_row, 0), bv.x));
                    h[2 * i + 1] = fma2(two(ex2(e1.x), ex2(e1.y)), h[2 * i + 1], mul2(pair(dx_row, 2), bv.y));
                    if (PASS != ENDS) {
                        const ulonglong2 cv = c2[i * L];
                        sum = i == 0 ? mul2(cv.x, h[0]) : fma2(cv.x, h[2 * i], sum);
                        sum = fma2(cv.y, h[2 * i + 1], sum);
                    }
                }
                const float2 s = each(sum);
                return s.x + s.y;
            };
            bool odd = false;  // the group has a row that the states behind d_state must not see: an infinite d x times their b of 0 is no number
            if constexpr (PADS) {
                float most = 0.f;
#pragma unroll
                for (int t = 0; t < TG; t++) most = fmaxf(most, fabsf(dxs[t]));
                odd = most == INFINITY;
            }
            if (!PADS || !odd) {
#pragma unroll
                for (int t = 0; t < TG; t++) y[t] = walk(t, ds[t], dxs[t], std::true_type{});
            } else if constexpr (PADS) {
#pragma unroll 1
                for (int t = 0; t < TG; t++) {
                    float d_row = 0.f, dx_row = 0.f;
#pragma unroll
                    for (int k = 0; k < TG; k++) if (k == t) { d_row = ds[k]; dx_row = dxs[k]; }
                    const float v = walk(t, d_row, dx_row, std::false_type{});
#pragma unroll
                    for (int k = 0; k < TG; k++) if (k == t) y[k] = v;
                }
            }
            if (PASS == ENDS) continue;
            // sums over the channel's lanes: lane p ends up with the rows p, p + L, ..
#pragma unroll
            for (int n = L / 2; n >= 1; n /= 2) {
#pragma unroll
                for (int t = 0; t < TG; t++) {
                    if ((t & n) || (t & (L - 1)) >= 2 * n) continue;  // (rows that are still there: t < 2 n modulo L)
                    const float send = p & n ? y[t] : y[t + n], kept = p & n ? y[t + n] : y[t];
                    y[t] = kept + __shfl_xor_sync(0xffffffffu, send, n);
                }
            }
            // (0 times an x that is not finite would be no number: no skip is no product)
            if (a.d) {
                if constexpr (!PAIRS) {
#pragma unroll
                    for (int j = 0; j < MT; j++) y[j * L] = fmaf(skip, x[j], y[j * L]);
                } else {
#pragma unroll
                    for (int j = 0; j < MT; j += 2) {
                        const float2 v = each(fma2(two(skip, skip), two(x[j], x[j + 1]), two(y[j * L], y[j * L + L])));
                        y[j * L] = v.x; y[j * L + L] = v.y;
                    }
                }
            }
            if (pz) {
                if constexpr (!PAIRS) {
#pragma unroll
                    for (int j = 0; j < MT; j++) y[j * L] *= silu(z[j]);
                } else {
#pragma unroll
                    for (int j = 0; j < MT; j += 2) {
                        const float2 v = each(mul2(two(y[j * L], y[j * L + L]), silu2(two(z[j], z[j + 1]))));
                        y[j * L] = v.x; y[j * L + L] = v.y;
                    }
                }
            }
            if (mine && full) {
#pragma unroll
                for (int j = 0; j < MT; j++) pd[j * L * a.dst_stride] = narrow<T>(y[j * L]);
            } else if (mine) {
#pragma unroll
                for (int j = 0; j < MT; j++) if (r0 + tg + j * L + p < rows) pd[j * L * a.dst_stride] = narrow<T>(y[j * L]);
            }
            pd += TG * a.dst_stride;
        }
        if (r0 + TC < rows) {
            keep(r0 + TC, buf ^ 1);
            __syncthreads();
        }
    }
    pdl_trigger();
    // ===== where the states go: the stretch's place, or the slot
    if constexpr (PASS == ENDS && L > 1) {
#pragma unroll
        for (int n = L / 2; n >= 1; n /= 2) total += __shfl_xor_sync(0xffffffffu, total, n);
    }
    if (!mine) return;
#pragma unroll
    for (int i = 0; i < NQ; i++) {
        const int n = 4 * (i * L + p);
        const float2 s0 = each(h[2 * i]), s1 = each(h[2 * i + 1]);
        const float4 s = make_float4(s0.x, s0.y, s1.x, s1.y);
        if (PASS == ENDS) {
            store_end(ends + stretch * ends_row, n, s);
        } else if (last) {
            float *to = a.state + (int64_t)q.slot * a.slot_stride + (int64_t)c * N;
            if (pieces) store_states<true>(to, n, N, s);
            else store_states<false>(to, n, N, s);
        }
    }
    if (PASS == ENDS && p == 0) sums[(int64_t)stretch * a.channels] = (float)total;
}

// ------------------------------------------------------------------------------------------------ convolution as a graph node has it
// The inputs of a channel lie side by side (the last ones of the sequence in front, made so by a CONCAT), the results channel by channel: a CTA turns a tile of NODE_CHANNELS channels and
// NODE_ROWS rows over in shared memory.
constexpr int NODE_CHANNELS = 32, NODE_ROWS = 64, NODE_WARPS = 8, NODE_TAPS = 16;
__global__ void __launch_bounds__(32 * NODE_WARPS) ssm_conv_nodes_kernel(const char *sx, int64_t nb1, int64_t nb2, const float *w, float *dst, int channels, int rows, int taps) {
    __shared__ float in[NODE_CHANNELS][NODE_ROWS + NODE_TAPS + 1];  // (a stride without common factors with the banks)
    pdl_enter();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c0 = blockIdx.x * NODE_CHANNELS, t0 = blockIdx.y * NODE_ROWS;
    const int nt = min(NODE_ROWS, rows - t0), nc = min(NODE_CHANNELS, channels - c0);
    sx += blockIdx.z * nb2;
    dst += (int64_t)blockIdx.z * rows * channels;
    for (int c = warp; c < nc; c += NODE_WARPS) {
        const float *row = (const float *)(sx + (c0 + c) * nb1) + t0;
        for (int t = lane; t < nt + taps - 1; t += 32) in[c][t] = row[t];
    }
    __syncthreads();
    if (lane >= nc) return;
    float k[NODE_TAPS];
#pragma unroll
    for (int j = 0; j < NODE_TAPS; j++) k[j] = j < taps ? w[(int64_t)(c0 + lane) * taps + j] : 0.f;
    for (int t = warp; t < nt; t += NODE_WARPS) {
        float y = 0.f;
#pragma unroll
        for (int j = 0; j < NODE_TAPS; j++) if (j < taps) y = fmaf(k[j], in[lane][t + j], y);
        dst[(int64_t)(t0 + t) * channels + c0 + lane] = y;
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
    int stretch, n_stretch;       // rows of a stretch, stretches of the longest sequence; n_stretch 1: no stretches
    bool step;                    // one row a sequence
    bool many;                    // whole sequences in many CTAs, or short ones
};
static int max_new_of(const b200_ssm_scan_args *a) {
    const int each = a->seq_info || a->n_seq <= 0 ? a->n_tokens : a->n_tokens / a->n_seq;
    return a->max_new > 0 && a->max_new < each ? a->max_new : each;
}
static int lanes_of(int d_state) { return d_state <= 16 ? 1 : d_state <= 32 ? 2 : d_state <= 64 ? 4 : 8; }
static ScanPlan plan_of(const b200_ssm_scan_args *a) {
    ScanPlan p = {0, 1, false, false};
    const int longest = max_new_of(a), block = SCAN_THREADS / lanes_of(a->d_state), per_group = a->channels / a->groups;
    p.step = longest <= 1;
    if (p.step) return p;
    // CTAs that are there on average while the longest sequence lasts
    const double ctas = (double)((per_group + block - 1) / block) * a->groups * a->n_tokens / longest;
    p.many = longest <= SCAN_SHORT || ctas >= 3.0 * sm_count();
    if (ctas < 1.25 * sm_count() && longest >= 128) {
        // One sequence: as many CTAs as are there at once (4096 rows of 2048 channels: 100 us, twice as many 126; of 5120 channels 250 and 272; of 8192 channels
        // 405 and 375, where more would be better).  Several: four an SM, which pays where they end at different times and there is enough
        // of them (six of 37 to 1501 rows of 5120 channels: 270 us, 306 with two), is little either way for prompts of one length (two of 2048 rows: of 2048 channels 115 and 112, of 5120 256 and
        // 260) and loses where channels are few (three of 100 to 2000 rows of 2048 channels: 103 and 86; three of 4096 rows of 512: 112 and 91).
        const double n = (double)(a->n_seq > 1 ? 4 : scan_ctas(lanes_of(a->d_state), ENDS)) * sm_count() / ctas;
        const int rows = (int)(longest / (n < 32 ? n : 32));
        p.stretch = ((rows < 64 ? 64 : rows) + 7) / 8 * 8;
        p.n_stretch = (longest + p.stretch - 1) / p.stretch;
    }
    return p;
}
// At most (4 SMs + blocks) / blocks places, of fewer than 1.25 SMs blocks of 128 / lanes channels: 13 MB.
static size_t scan_places(const b200_ssm_scan_args *a, const ScanPlan &p) { return ((size_t)a->n_tokens + p.stretch - 1) / p.stretch; }
static size_t scan_room(const b200_ssm_scan_args *a, const ScanPlan &p) {
    return p.n_stretch < 2 ? 0 : 4 * scan_places(a, p) * a->channels * (2 * (size_t)a->d_state + 1);
}

template <typename T, int L, int NS, int PASS>
static int launch_scan(const ScanArgs &a, cudaStream_t st) {
    constexpr int CB = ScanSizes<L, NS>::CB;
    const dim3 grid((unsigned)((a.per_group + CB - 1) / CB * (a.channels / a.per_group)), (unsigned)(PASS == WHOLE || PASS == MANY ? 1 : a.n_stretch), (unsigned)a.step.n_seq);
    const bool pads = PASS != ENDS && a.d_state < NS * L;  // (the ends of stretches are stored without them)
    B200_CUDA_TRY(launch_chained(pads ? ssm_scan_kernel<T, L, NS, PASS, PASS != ENDS> : ssm_scan_kernel<T, L, NS, PASS, false>, grid, SCAN_THREADS, 0, st, a));
    return B200_OK;
}
template <typename T, int L, int NS>
static int launch_scan_rows(const ScanArgs &a, const ScanPlan &p, cudaStream_t st) {
    if (p.n_stretch < 2) return L == 1 && p.many ? launch_scan<T, L, NS, L == 1 ? MANY : WHOLE>(a, st) : launch_scan<T, L, NS, WHOLE>(a, st);
    const int rc = launch_scan<T, L, NS, ENDS>(a, st);
    return rc != B200_OK ? rc : launch_scan<T, L, NS, ROWS>(a, st);
}
template <typename T, int L>
static int launch_step(const ScanArgs &a, bool states16, cudaStream_t st) {
    const dim3 grid((unsigned)((a.channels + 32 * STEP_WARPS - 1) / (32 * STEP_WARPS)), (unsigned)a.step.n_seq);
    B200_CUDA_TRY(launch_chained(states16 ? ssm_step_kernel<T, L, true> : ssm_step_kernel<T, L, false>, grid, 32 * STEP_WARPS, 0, st, a));
    return B200_OK;
}
template <typename T>
static int launch_scan_type(const ScanArgs &a, const ScanPlan &p, bool states16, cudaStream_t st) {
    const int n = a.d_state;
    if (p.step) return n <= 16 ? launch_step<T, 4>(a, states16, st) : n <= 32 ? launch_step<T, 8>(a, states16, st) : n <= 64 ? launch_step<T, 16>(a, states16, st) : launch_step<T, 32>(a, states16, st);
    if (n <= 4) return launch_scan_rows<T, 1, 4>(a, p, st);
    if (n <= 8) return launch_scan_rows<T, 1, 8>(a, p, st);
    if (n <= 16) return launch_scan_rows<T, 1, 16>(a, p, st);
    if (n <= 32) return launch_scan_rows<T, 2, 16>(a, p, st);
    if (n <= 64) return launch_scan_rows<T, 4, 16>(a, p, st);
    return launch_scan_rows<T, 8, 16>(a, p, st);
}

static int check_step(const int32_t *seq_info, int32_t n_seq, int32_t n_slots, int32_t n_tokens, int32_t max_new, int32_t channels, int32_t type, const char *who) {
    OPX_REQUIRE(type_ok(type), B200_ERR_UNSUPPORTED, "%s: rows of type %d", who, type);
    OPX_REQUIRE(n_seq >= 0 && n_seq <= 65535 && n_slots >= 0 && n_tokens >= 0 && max_new >= 0, B200_ERR_INVALID, "%s: %d sequences, %d slots, %d rows, %d new ones at most", who, n_seq, n_slots,
                n_tokens, max_new);
    OPX_REQUIRE(n_tokens <= B200_STATE_MAX_INDEX && channels <= B200_STATE_MAX_INDEX, B200_ERR_UNSUPPORTED, "%s: %d rows of %d channels, %d of either at most", who, n_tokens, channels, B200_STATE_MAX_INDEX);
    OPX_REQUIRE((uintptr_t)seq_info % 4 == 0, B200_ERR_INVALID, "%s: seq_info at an odd place", who);
    OPX_REQUIRE(seq_info || (n_seq <= n_slots && (n_seq == 0 ? n_tokens == 0 : n_tokens % n_seq == 0)), B200_ERR_INVALID, "%s: without seq_info, %d rows are not %d sequences of one length in %d slots",
                who, n_tokens, n_seq, n_slots);
    return B200_OK;
}

int ssm_scan_check(const b200_ssm_scan_args *a) {
    const char *who = "b200_op_ssm_scan";
    OPX_REQUIRE(a, B200_ERR_INVALID, "%s: NULL arguments", who);
    const int rc = check_step(a->seq_info, a->n_seq, a->n_slots, a->n_tokens, a->max_new, a->channels, a->type, who);
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
    OPX_REQUIRE((a->dst != a->x || a->dst_stride == a->x_stride) && (a->dst != a->dt || a->dst_stride == a->dt_stride) && (a->dst != a->z || a->dst_stride == a->z_stride), B200_ERR_INVALID,
                "%s: dst is an input at another stride", who);
    OPX_REQUIRE(a->from != a->state || a->from_stride == a->slot_stride, B200_ERR_INVALID, "%s: from is state at another stride", who);
    return B200_OK;
}

}  // namespace ssm

// whether the calls take tensors of these shapes (their memory apart): what supports_op asks
static bool dense(const b200_tensor *t) {
    int64_t nb = 4;
    for (int i = 0; i < 4; i++) {
        if (t->ne[i] != 1 && (int64_t)t->nb[i] != nb) return false;
        nb *= t->ne[i];
    }
    return t->type == B200_TYPE_F32;
}
bool ssm_conv_nodes_ok(const b200_tensor *sx, const b200_tensor *c, const b200_tensor *dst) {
    return sx && c && dst && sx->type == B200_TYPE_F32 && sx->nb[0] == 4 && sx->nb[1] % 4 == 0 && sx->nb[2] % 4 == 0 && dense(c) && dense(dst) && c->ne[0] >= 1 && c->ne[0] <= ssm::NODE_TAPS &&
           c->ne[2] == 1 && c->ne[3] == 1 && sx->ne[3] == 1 && dst->ne[3] == 1 && sx->ne[0] == dst->ne[1] + c->ne[0] - 1 && sx->ne[1] == dst->ne[0] && c->ne[1] == dst->ne[0] &&
           sx->ne[2] == dst->ne[2] && dst->ne[0] <= 0x7fffffff && dst->ne[1] <= 65535 * (int64_t)ssm::NODE_ROWS && dst->ne[2] <= 65535;
}
bool ssm_scan_nodes_ok(const b200_tensor *s, const b200_tensor *x, const b200_tensor *dt, const b200_tensor *a, const b200_tensor *b, const b200_tensor *c, const b200_tensor *dst) {
    if (!s || !x || !dt || !a || !b || !c || !dst || !dense(s) || !dense(x) || !dense(dt) || !dense(a) || !dense(dst)) return false;
    const int64_t n = s->ne[0], ch = s->ne[1], seqs = s->ne[2], rows = x->ne[1];
    for (const b200_tensor *t : {b, c}) {
        if (t->type != B200_TYPE_F32 || t->nb[0] != 4 || t->nb[1] % 4 || t->ne[0] != n || t->ne[1] != rows || t->ne[2] != seqs || t->ne[3] != 1) return false;
        if ((rows > 1 || seqs > 1) && t->nb[1] < 4 * (size_t)n) return false;
        if (seqs > 1 && t->nb[2] != t->nb[1] * (size_t)rows) return false;
    }
    return n >= 1 && n <= 128 && ch >= 1 && seqs >= 1 && seqs <= 65535 && rows >= 1 && s->ne[3] == 1 && x->ne[0] == ch && x->ne[2] == seqs && x->ne[3] == 1 && a->ne[0] == n && a->ne[1] == ch &&
           a->ne[2] == 1 && a->ne[3] == 1 && dt->ne[0] == ch && dt->ne[1] == rows && dt->ne[2] == seqs && dt->ne[3] == 1 && rows <= B200_STATE_MAX_INDEX && rows * seqs <= B200_STATE_MAX_INDEX && ch <= B200_STATE_MAX_INDEX &&
           opx::nelements(dst) == opx::nelements(x) + opx::nelements(s);
}
namespace ssm {
static void scan_node_sizes(const b200_tensor *s, const b200_tensor *x, b200_ssm_scan_args *a) {
    a->d_state = (int32_t)s->ne[0];
    a->channels = (int32_t)s->ne[1];
    a->n_seq = a->n_slots = (int32_t)s->ne[2];
    a->n_tokens = (int32_t)(x->ne[1] * s->ne[2]);
    a->groups = 1;
    a->type = B200_TYPE_F32;
}
}  // namespace ssm
}  // namespace b200

using namespace b200;
using namespace b200::ssm;

extern "C" {

int b200_op_ssm_conv(const b200_ssm_conv_args *a, b200_stream_t stream) {
    const char *who = "b200_op_ssm_conv";
    OPX_REQUIRE(a, B200_ERR_INVALID, "%s: NULL arguments", who);
    const int rc = check_step(a->seq_info, a->n_seq, a->n_slots, a->n_tokens, a->max_new, a->channels, a->type, who);
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
    if (!a || a->n_seq <= 0 || a->n_tokens <= 0 || a->n_tokens > B200_STATE_MAX_INDEX || a->channels <= 0 || a->channels > B200_STATE_MAX_INDEX || a->groups <= 0 || a->channels % a->groups || a->d_state <= 0 || a->d_state > 128) return 0;
    return scan_room(a, plan_of(a));
}

int b200_op_ssm_scan(const b200_ssm_scan_args *a, void *workspace, size_t workspace_bytes, b200_stream_t stream) {
    const char *who = "b200_op_ssm_scan";
    const int rc = ssm_scan_check(a);
    if (rc != B200_OK || a->n_seq == 0 || a->n_tokens == 0) return rc;
    const ScanPlan p = plan_of(a);
    const size_t need = scan_room(a, p);
    OPX_REQUIRE(need <= B200_SSM_SCAN_WORKSPACE_MAX, B200_ERR_UNSUPPORTED, "%s: %zu bytes of workspace", who, need);  // (what the header promises)
    OPX_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && (uintptr_t)workspace % 16 == 0), B200_ERR_INVALID, "%s: workspace of %zu bytes, 16-byte aligned", who, need);
    const int per_group = a->channels / a->groups, each = a->seq_info ? a->n_tokens : a->n_tokens / a->n_seq, longest = a->max_new > 0 && a->max_new < each ? a->max_new : each;
    float *ends = need ? (float *)workspace : nullptr;
    const size_t places = need ? scan_places(a, p) * a->channels * a->d_state : 0;
    const size_t four = 4 * type_size(a->type);
    const bool bc_pieces = on(four, {a->b, a->c}) && ((a->b_stride | a->c_stride | a->d_state) & 3) == 0;
    const ScanArgs s = {{a->seq_info, a->n_seq, a->n_slots, a->n_tokens, longest}, a->x, a->dt, a->b, a->c, a->z, a->x_stride, a->dt_stride, a->b_stride, a->c_stride, a->z_stride, a->a, a->dt_bias, a->d,
                        a->from ? a->from : a->state, a->from ? a->from_stride : a->slot_stride, a->state, a->slot_stride, a->dst, a->dst_stride, a->channels, a->d_state, per_group, a->softplus, bc_pieces,
                        p.stretch, p.n_stretch, ends, ends + places, ends + 2 * places};
    const bool states16 = (a->d_state & 3) == 0 && ((s.slot_stride | s.from_stride) & 3) == 0 && on(16, {s.state, s.from, a->a});
    const cudaStream_t st = (cudaStream_t)stream;
    if (a->type == B200_TYPE_F32) return launch_scan_type<float>(s, p, states16, st);
    if (a->type == B200_TYPE_F16) return launch_scan_type<__half>(s, p, states16, st);
    return launch_scan_type<__nv_bfloat16>(s, p, states16, st);
}

int b200_op_concat(const b200_tensor *a, const b200_tensor *b, const b200_tensor *dst, int dim, b200_stream_t stream) {
    const char *who = "b200_op_concat";
    OPX_REQUIRE(a && b && dst && dim >= 0 && dim < 4, B200_ERR_INVALID, "%s: NULL argument or no such dimension", who);
    OPX_REQUIRE(a->type == B200_TYPE_F32 && b->type == B200_TYPE_F32 && dst->type == B200_TYPE_F32, B200_ERR_UNSUPPORTED, "%s: f32 only", who);
    for (int i = 0; i < 4; i++) {
        OPX_REQUIRE(i == dim ? dst->ne[i] == a->ne[i] + b->ne[i] : dst->ne[i] == a->ne[i] && dst->ne[i] == b->ne[i], B200_ERR_INVALID, "%s: shapes do not fit", who);
    }
    b200_tensor part = *dst;
    for (const b200_tensor *s : {a, b}) {
        part.ne[dim] = s->ne[dim];
        const int rc = opx::nelements(s) > 0 ? b200_op_cpy(s, &part, stream) : B200_OK;
        if (rc != B200_OK) return rc;
        part.data = (char *)part.data + s->ne[dim] * dst->nb[dim];
    }
    return B200_OK;
}

int b200_op_ssm_conv_nodes(const b200_tensor *sx, const b200_tensor *c, const b200_tensor *dst, b200_stream_t stream) {
    const char *who = "b200_op_ssm_conv_nodes";
    OPX_REQUIRE(ssm_conv_nodes_ok(sx, c, dst), B200_ERR_UNSUPPORTED, "%s: f32, one row in front for every tap but one, at most %d taps", who, NODE_TAPS);
    if (opx::nelements(dst) == 0) return B200_OK;
    OPX_REQUIRE(sx->data && c->data && dst->data, B200_ERR_INVALID, "%s: NULL argument", who);
    const int channels = (int)dst->ne[0], rows = (int)dst->ne[1];
    const dim3 grid((unsigned)((channels + NODE_CHANNELS - 1) / NODE_CHANNELS), (unsigned)((rows + NODE_ROWS - 1) / NODE_ROWS), (unsigned)dst->ne[2]);
    B200_CUDA_TRY(launch_chained(ssm_conv_nodes_kernel, grid, 32 * NODE_WARPS, 0, (cudaStream_t)stream, (const char *)sx->data, (int64_t)sx->nb[1], (int64_t)sx->nb[2], (const float *)c->data,
                                 (float *)dst->data, channels, rows, (int)c->ne[0]));
    return B200_OK;
}

size_t b200_op_ssm_scan_nodes_workspace_bytes(const b200_tensor *s, const b200_tensor *x) {
    b200_ssm_scan_args a = {};
    if (!s || !x || s->ne[1] > B200_STATE_MAX_INDEX || s->ne[2] > 65535 || x->ne[1] > B200_STATE_MAX_INDEX || x->ne[1] * s->ne[2] > B200_STATE_MAX_INDEX) return 0;
    scan_node_sizes(s, x, &a);
    return b200_ssm_scan_workspace_bytes(&a);
}

int b200_op_ssm_scan_nodes(const b200_tensor *s, const b200_tensor *x, const b200_tensor *dt, const b200_tensor *a, const b200_tensor *b, const b200_tensor *c, const b200_tensor *dst,
                           void *workspace, size_t workspace_bytes, b200_stream_t stream) {
    const char *who = "b200_op_ssm_scan_nodes";
    OPX_REQUIRE(ssm_scan_nodes_ok(s, x, dt, a, b, c, dst), B200_ERR_UNSUPPORTED, "%s: f32, contiguous but for b and c, at most 128 states", who);
    b200_ssm_scan_args n = {};
    scan_node_sizes(s, x, &n);
    n.x = x->data; n.dt = dt->data; n.x_stride = n.dt_stride = n.dst_stride = n.channels;
    const bool one = n.n_tokens == 1;  // (what a single row's stride says is nothing to go by)
    n.b = b->data; n.b_stride = one ? n.d_state : (int64_t)(b->nb[1] / 4);
    n.c = c->data; n.c_stride = one ? n.d_state : (int64_t)(c->nb[1] / 4);
    n.a = (const float *)a->data;
    n.from = (const float *)s->data;
    n.dst = dst->data;
    n.state = (float *)dst->data + (int64_t)n.n_tokens * n.channels;
    n.slot_stride = n.from_stride = (int64_t)n.channels * n.d_state;
    n.softplus = 1;
    return b200_op_ssm_scan(&n, workspace, workspace_bytes, stream);
}

}  // extern "C"
