// beam.cu -- beam search (include/b200_state.h): the best successors over all beams and tokens of a request (b200_op_beam_select), and slots that become what other slots
// held (b200_op_state_reorder).
#include <cuda_bf16.h>

#include "../../include/b200_state.h"
#include "ops_util.cuh"

namespace b200 {
namespace beam {

// ------------------------------------------------------------------------------------------------ selection
// Two launches.  The first reads the logits once: of every piece of PIECE tokens of a row (or a power of two of them) it keeps the largest, of every share of a row the sum of exponentials.
// The second, a CTA a request, knows the logarithms of the sums then, and so every piece's best score.  The n_keep best successors all lie in the n_keep pieces whose best come first
// (a successor elsewhere comes behind the best of each of these), so it reads those pieces again and nothing else.
// What bounds it: the first launch instructions (12.4 a token of 16 bits at odd places, issued 65 % of the time), the second the way from one result to the next: barriers, and code that is run once.
// (The second launch is a chain of instructions, 7000 a warp of eight for 32 beams of 151936 tokens and 64 results, and its loads hide none of it: 49 us for both launches with 256 threads, 34 with 512,
// 28 with 1024, whose 64 registers are too few for rows at odd places; four beams of 32000 tokens 10.4, 10.5 and 10.8.)
constexpr int PIECE = 512, ROW_WARPS = 8, PICK_THREADS = 512, PICK_WARPS = PICK_THREADS / 32;
constexpr int MOST_PIECES = 4096;  // of a request: what the second launch looks through
constexpr int LIST = 512;          // candidates that are ranked by counting; where ties make them more, the best are taken out one after the other
struct SelectArgs {
    const void *logits; int64_t logits_stride;
    const float *score;
    const int32_t *ended, *slot;
    float *to_score; int32_t *to_beam, *to_token, *to_slot;
    int32_t beams, vocab, keep, end_token;
    // layout: tokens of a piece, pieces of a row, pieces of a share, shares of a row
    int32_t piece, n_pieces, share, n_shares;
    unsigned by_pieces;  // ceil(2^32 / n_pieces): i / n_pieces is the upper half of its product with i < MOST_PIECES (n_pieces > 1)
    float *tops;         // [rows][n_pieces]: the largest logit, -inf where there is none
    double *sums;        // [rows][n_shares]: sum of exp(logit - ref) ..
    float *refs;         // .. and its ref: the largest logit, rounded up to a whole number
};
constexpr float NEG_INF = -INFINITY;
constexpr float LOG2E = 1.4426950408889634f;
__device__ __forceinline__ float ex2(float x) { float r; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x)); return r; }
using Two = unsigned long long;
__device__ __forceinline__ Two two(float lo, float hi) { Two r; asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi)); return r; }
__device__ __forceinline__ float2 each(Two x) { float2 r; asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(x)); return r; }
__device__ __forceinline__ Two add2(Two x, Two y) { Two r; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y)); return r; }
__device__ __forceinline__ Two mul2(Two x, Two y) { Two r; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y)); return r; }

// A sum of exponentials that refers to `from` as one that refers to the larger `to`.  References are whole numbers where f32 has a choice, so that few larger logits move them, and the
// largest logits' exponents are small numbers, whose product with log2 e is off by little.
__device__ __noinline__ double less(double sum, double by) { return sum * exp(-by); }  // (once in the code: it is seldom wanted, and a short kernel waits for every line that it fetches)
__device__ __forceinline__ double follow(double sum, float from, float to) { return from == to ? sum : from == NEG_INF ? 0.0 : less(sum, (double)to - (double)from); }
// the largest of a warp's, NaN apart; -inf where all are NaN
__device__ __forceinline__ float largest(float x) { float r; asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(x)); return r != r ? NEG_INF : r; }

// a logit as it counts: NaN is none
__device__ __forceinline__ float counted(float x) { return x != x ? NEG_INF : x; }
template <typename T> __device__ __forceinline__ float value_at(const T *p) {
    if constexpr (sizeof(T) == 4) return *p;
    else if constexpr (std::is_same<T, __half>::value) return __half2float(*p);
    else return __bfloat162float(*p);
}
// the two values of a word of 16-bit logits
template <typename T> __device__ __forceinline__ float2 both(unsigned w) {
    if constexpr (std::is_same<T, __half>::value) return __half22float2(*reinterpret_cast<const __half2 *>(&w));
    else return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}

// PIECE tokens of a row from token t0 on, 16 a lane, those behind the vocabulary -inf.  Which token a lane gets does not depend on where the row lies (WIDE is the same for all rows of
// a call): rows with the same logits have the same sums, bit by bit.
template <typename T, bool WIDE>
__device__ __forceinline__ int token_of(int i, int lane) {  // number i of a lane, counted from t0
    if constexpr (sizeof(T) == 4) return WIDE ? 128 * (i / 4) + 4 * lane + i % 4 : 32 * i + lane;
    else return WIDE ? 256 * (i / 8) + 8 * lane + i % 8 : 64 * (i / 2) + 2 * lane + i % 2;
}
// .. as they lie in memory: words of one or two logits
template <typename T>
struct Raw {
    static constexpr int N = 4 * (int)sizeof(T);  // 16 or 8
    unsigned v[N + 1];
    bool odd;  // 16 bits: the row begins in the middle of a word, so a lane's tokens are the upper half of its word and the lower half of the next lane's
};
template <typename T, bool WIDE>
__device__ __forceinline__ void load_raw(const T *row, int t0, int vocab, int lane, Raw<T> &r) {
    r.odd = false;
    if (t0 + PIECE + 2 > vocab) {
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const int t = t0 + token_of<T, WIDE>(i, lane);
            if constexpr (sizeof(T) == 4) {
                r.v[i] = t < vocab ? __float_as_uint(row[t]) : __float_as_uint(NEG_INF);
            } else {
                const unsigned none = std::is_same<T, __half>::value ? 0xfc00u : 0xff80u, h = t < vocab ? reinterpret_cast<const unsigned short *>(row)[t] : none;
                r.v[i / 2] = i & 1 ? r.v[i / 2] | h << 16 : h;
            }
        }
    } else if constexpr (WIDE) {
#pragma unroll
        for (int i = 0; i < Raw<T>::N / 4; i++) {
            const uint4 v = *reinterpret_cast<const uint4 *>(row + t0 + token_of<T, true>(4 * i * (4 / (int)sizeof(T)), lane));
            r.v[4 * i] = v.x; r.v[4 * i + 1] = v.y; r.v[4 * i + 2] = v.z; r.v[4 * i + 3] = v.w;
        }
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 16; i++) r.v[i] = __float_as_uint(row[t0 + 32 * i + lane]);
    } else {
        r.odd = ((uintptr_t)row & 2) != 0;
        const unsigned *w = reinterpret_cast<const unsigned *>(row + t0 - r.odd);
        r.v[0] = t0 > 0 || !r.odd || lane > 0 ? w[lane] : (unsigned)*reinterpret_cast<const unsigned short *>(row) << 16;  // (nothing in front of the row is read)
#pragma unroll
        for (int i = 1; i < 8; i++) r.v[i] = w[32 * i + lane];
        r.v[8] = r.odd && lane == 0 ? w[256] : 0;
    }
}
template <typename T>
__device__ __forceinline__ void values_of(Raw<T> &r, int lane, float (&x)[16]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 16; i++) x[i] = __uint_as_float(r.v[i]);
    } else {
        if (r.odd) {
#pragma unroll
            for (int i = 0; i < 8; i++) r.v[i] = __funnelshift_r(r.v[i], __shfl_sync(0xffffffffu, lane == 0 ? r.v[i + 1] : r.v[i], lane + 1), 16);
        }
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float2 f = both<T>(r.v[i]);
            x[2 * i] = f.x; x[2 * i + 1] = f.y;
        }
    }
}

// the sum over a lane's 16 logits of exp(x - ref)
__device__ __forceinline__ float sum_of(const float (&x)[16], float ref) {
    Two s = 0;
#pragma unroll
    for (int i = 0; i < 16; i += 2) {
        const float2 e = each(mul2(add2(two(x[i], x[i + 1]), two(-ref, -ref)), two(LOG2E, LOG2E)));
        s = add2(s, two(ex2(e.x), ex2(e.y)));
    }
    return each(s).x + each(s).y;
}

template <typename T, bool WIDE>
__global__ void __launch_bounds__(32 * ROW_WARPS) beam_rows_kernel(const SelectArgs a) {
    __shared__ double s_sum[ROW_WARPS];
    __shared__ float s_ref[ROW_WARPS];
    pdl_enter();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t r = blockIdx.y;
    const T *row = (const T *)a.logits + r * a.logits_stride;
    const int p0 = blockIdx.x * a.share, p1 = min(a.n_pieces, p0 + a.share);
    const bool unwanted = (a.ended && a.ended[r]) || !(a.score[r] > NEG_INF);  // a beam that nobody asks for the successors of
    double sum = 0.0;
    float ref = NEG_INF;
    // (the next PIECE tokens travel while these are added up; the first ones before it is known whether they are wanted)
    Raw<T> next;
    int p = p0 + warp, t0 = p * a.piece;
    if (p < p1) load_raw<T, WIDE>(row, t0, a.vocab, lane, next);
    if (unwanted) return;
    while (p < p1) {
        float top = NEG_INF;
        for (const int end = min(a.vocab, (p + 1) * a.piece); t0 < end;) {
            Raw<T> now_here = next;
            t0 += PIECE;
            const int ahead = t0 < end ? t0 : (p + ROW_WARPS) * a.piece;
            if (t0 < end || p + ROW_WARPS < p1) load_raw<T, WIDE>(row, ahead, a.vocab, lane, next);
            float x[16];
            values_of<T>(now_here, lane, x);
            float m = x[0];
#pragma unroll
            for (int i = 1; i < 16; i++) m = fmaxf(m, x[i]);  // (a NaN loses)
            m = largest(m);
            if (m == NEG_INF) continue;
            top = fmaxf(top, m);
            const float now = fmaxf(ref, ceilf(m));
            if (now != ref) {
                sum = follow(sum, ref, now);
                ref = now;
            }
            float part = 0.f;
            if (ref < INFINITY) {
                part = sum_of(x, ref);
                if (__any_sync(0xffffffffu, part != part)) {
#pragma unroll
                    for (int i = 0; i < 16; i++) x[i] = counted(x[i]);
                    part = sum_of(x, ref);
                }
            } else {
#pragma unroll
                for (int i = 0; i < 16; i++) part += x[i] == INFINITY ? 1.f : 0.f;
            }
            sum += part;
        }
        if (lane == 0) a.tops[r * a.n_pieces + p] = top;
        p += ROW_WARPS;
        t0 = p * a.piece;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) { s_sum[warp] = sum; s_ref[warp] = ref; }
    __syncthreads();
    if (warp == 0) {
        ref = warp_max(lane < ROW_WARPS ? s_ref[lane] : NEG_INF);
        sum = lane < ROW_WARPS ? follow(s_sum[lane], s_ref[lane], ref) : 0.0;
#pragma unroll
        for (int o = ROW_WARPS / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0) {
            a.sums[r * a.n_shares + blockIdx.x] = sum;
            a.refs[r * a.n_shares + blockIdx.x] = ref;
        }
    }
}

// A successor: its score and its place beam * vocab + token in the request.  Whether x comes before y:
struct Cand { double score; int64_t at; };
__device__ __forceinline__ bool before(const Cand &x, const Cand &y) { return x.score > y.score || (x.score == y.score && x.at < y.at); }
__device__ __forceinline__ Cand shuffled(const Cand &x, int off) { return {__shfl_xor_sync(0xffffffffu, x.score, off), __shfl_xor_sync(0xffffffffu, x.at, off)}; }
// numbers whose order as unsigned ones is that of the floats; 0 is behind all of them
__device__ __forceinline__ unsigned ordered(float f) {
    const unsigned u = __float_as_uint(f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float unordered(unsigned u) { return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u); }

struct PickShared {
    double base[B200_BEAM_MAX];     // a beam's score (base_of)
    double ref[B200_BEAM_MAX], norm[B200_BEAM_MAX];  // what is taken off its logits, one after the other
    int ended[B200_BEAM_MAX];
    Cand list[LIST];
    Cand best[B200_BEAM_KEEP];      // first the pieces, then the successors
    Cand warps[PICK_WARPS];
    unsigned low[PICK_WARPS], high[PICK_WARPS];
    int piece[B200_BEAM_KEEP];      // where the successors are looked for
    int n[2];                       // candidates of the pieces, of the successors: a count each, so that none is reset while a warp has still to read it
};

// A beam's score as its successors have it; ref: its row's largest logit.  -inf: it has none.  +inf counts as the largest number of 64 bits, which is +inf again once it is rounded to f32: beside a
// logit of +inf it would make sums that are no numbers, and these have no rank.
__device__ __forceinline__ double base_of(float s, bool ended, float ref) {
    return s != s || (!ended && ref == NEG_INF) ? -(double)INFINITY : s == INFINITY ? 0x1.fffffffffffffp1023 : (double)s;
}
// The score of a logit of beam b.  With a reference of +inf the tokens of +inf share evenly, the others have none.
__device__ __forceinline__ double score_of(const PickShared &sh, int b, float x) {
    if (x == NEG_INF || sh.base[b] == -(double)INFINITY) return -(double)INFINITY;
    if (x == INFINITY) return sh.base[b] - sh.norm[b];
    return sh.base[b] + (((double)x - sh.ref[b]) - sh.norm[b]);
}

// The `keep` first of the candidates that each(thread's function) names, in order, to sh.best; returns how many there are.  each(f) calls f(candidate) for all candidates of the calling
// thread, whatever their order, and always for the same ones; `floor`: candidates with smaller scores can be left aside (at least `keep` have a score of that or more, or it is -inf).
// (sh.n[phase] is 0 and everybody knows; no two calls share a phase.)
template <typename F>
__device__ __forceinline__ int first_of(PickShared &sh, int phase, int keep, double floor, F each) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    each([&](const Cand &c) {
        if (c.score == -(double)INFINITY || c.score < floor) return;
        const int i = atomicAdd(&sh.n[phase], 1);
        if (i < LIST) sh.list[i] = c;
    });
    __syncthreads();
    const int n = sh.n[phase];  // (nothing changes it from here on)
    if (n <= LIST) {
        // a candidate's rank is the number of those before it: the list's own order, which is that of arrival, does not matter
        for (int i = tid; i < n; i += PICK_THREADS) {
            const Cand c = sh.list[i];
            int rank = 0;
#pragma unroll 8
            for (int j = 0; j < n; j++) rank += before(sh.list[j], c);
            if (rank < keep) sh.best[rank] = c;
        }
    } else {
        // one after the other: the first of those behind the last one found
        Cand last = {INFINITY, -1};
        for (int k = 0; k < keep; k++) {
            Cand mine = {-(double)INFINITY, 0x7fffffffffffffffLL};
            each([&](const Cand &c) { if (c.score >= floor && before(last, c) && before(c, mine)) mine = c; });
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                const Cand other = shuffled(mine, o);
                if (before(other, mine)) mine = other;
            }
            if (lane == 0) sh.warps[warp] = mine;
            __syncthreads();
            mine = sh.warps[0];
            for (int w = 1; w < PICK_WARPS; w++) if (before(sh.warps[w], mine)) mine = sh.warps[w];
            if (tid == 0) sh.best[k] = mine;
            last = mine;
            __syncthreads();
        }
    }
    __syncthreads();
    return min(n, keep);
}

template <typename T, bool WIDE>
__global__ void __launch_bounds__(PICK_THREADS) beam_pick_kernel(const SelectArgs a) {
    __shared__ PickShared sh;
    __shared__ float tops[MOST_PIECES];
    pdl_enter();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t r0 = (int64_t)blockIdx.x * a.beams;
    const int total = a.beams * a.n_pieces;
    for (int i = tid; i < total; i += PICK_THREADS) cp_async4(&tops[i], a.tops + r0 * a.n_pieces + i);
    cp_async_commit();
    // ===== the logarithms of the sums, a warp a beam
    if (tid < 2) sh.n[tid] = 0;
    for (int b = warp; b < a.beams; b += PICK_WARPS) {
        const double *sums = a.sums + (r0 + b) * a.n_shares;
        const float *refs = a.refs + (r0 + b) * a.n_shares;
        const float s = a.score[r0 + b];
        const bool ended = a.ended && a.ended[r0 + b];
        float ref = NEG_INF;
        for (int i = lane; i < a.n_shares; i += 32) ref = fmaxf(ref, refs[i]);
        ref = warp_max(ref);
        double all = 0.0;
        for (int i = lane; i < a.n_shares; i += 32) all += follow(sums[i], refs[i], ref);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
        if (lane == 0) {
            sh.base[b] = base_of(s, ended, ref);  // (of a beam whose row was not read ref and sum are anything, and its score -inf)
            sh.ref[b] = (double)ref;
            sh.norm[b] = log(all);
            sh.ended[b] = ended;
        }
    }
    cp_async_wait<0>();
    __syncthreads();
    // ===== the pieces: candidates are their best scores, at beam * n_pieces + piece.  An ended beam is one piece of one successor
    auto beam_of = [&](int i) { return a.n_pieces == 1 ? i : (int)__umulhi((unsigned)i, a.by_pieces); };
    auto pieces = [&](auto &&f) {
#pragma unroll 4
        for (int i = tid; i < total; i += PICK_THREADS) {
            const int b = beam_of(i);
            const double s = sh.ended[b] ? (i == b * a.n_pieces ? sh.base[b] : -(double)INFINITY) : score_of(sh, b, tops[i]);
            f(Cand{s, i});
        }
    };
    // a score that `keep` threads' best reach at least, by halving between the smallest and the largest of these: what lies below can be left aside
    double floor = -(double)INFINITY;
    if (total > 64) {
        float top = NEG_INF;
        pieces([&](const Cand &c) { top = fmaxf(top, __double2float_rd(c.score)); });
        const unsigned key = top == NEG_INF ? 0 : ordered(top);
        const unsigned lo = __reduce_min_sync(0xffffffffu, key ? key : 0xffffffffu), hi = __reduce_max_sync(0xffffffffu, key);
        if (lane == 0) { sh.low[warp] = lo; sh.high[warp] = hi; }
        const int n_there = __syncthreads_count(key != 0);
        if (n_there >= a.keep) {
            unsigned low = sh.low[0], high = sh.high[0];
            for (int w = 1; w < PICK_WARPS; w++) {
                low = min(low, sh.low[w]);
                high = max(high, sh.high[w]);
            }
            for (int k = 0; k < 9 && low < high; k++) {
                const unsigned at = low + (high - low + 1) / 2;
                if (__syncthreads_count(key >= at) >= a.keep) low = at;
                else high = at - 1;
            }
            floor = (double)unordered(low);
        }
    }
    const int n_best = first_of(sh, 0, a.keep, floor, pieces);
    // ===== the successors in those pieces, a warp a piece
    for (int k = tid; k < n_best; k += PICK_THREADS) sh.piece[k] = (int)sh.best[k].at;
    floor = n_best == a.keep ? sh.best[a.keep - 1].score : -(double)INFINITY;
    __syncthreads();
    auto successors = [&](auto &&f) {
#pragma unroll 1
        for (int k = warp; k < n_best; k += PICK_WARPS) {
            const int piece = sh.piece[k], b = beam_of(piece), t1 = (piece - b * a.n_pieces) * a.piece;
            if (sh.ended[b]) {
                if (lane == 0) f(Cand{sh.base[b], (int64_t)b * a.vocab + a.end_token});
                continue;
            }
            const T *row = (const T *)a.logits + (r0 + b) * a.logits_stride;
            // (a logit below this has a score below the floor: 2^-20 of what its terms may be is more than their roundings)
            const double at = (floor - sh.base[b]) + sh.norm[b] + sh.ref[b];
            const float least = __double2float_rd(at - 0x1p-20 * (fabs(floor) + fabs(sh.base[b]) + fabs(sh.norm[b]) + fabs(sh.ref[b])));
#pragma unroll 1
            for (int t0 = t1; t0 < min(a.vocab, t1 + a.piece); t0 += PIECE) {
                Raw<T> raw;
                float x[16];
                load_raw<T, WIDE>(row, t0, a.vocab, lane, raw);
                values_of<T>(raw, lane, x);
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    if (!(x[i] < least) && x[i] > NEG_INF) f(Cand{score_of(sh, b, x[i]), (int64_t)b * a.vocab + t0 + token_of<T, WIDE>(i, lane)});
                }
            }
        }
    };
    const int n = first_of(sh, 1, a.keep, floor, successors);
    for (int i = tid; i < a.keep; i += PICK_THREADS) {
        const int64_t to = (int64_t)blockIdx.x * a.keep + i;
        const bool there = i < n;
        const int b = there ? (int)(sh.best[i].at / a.vocab) : -1;
        a.to_score[to] = there ? (float)sh.best[i].score : NEG_INF;
        a.to_beam[to] = b;
        a.to_token[to] = there ? (int)(sh.best[i].at - (int64_t)b * a.vocab) : -1;
        if (a.to_slot) a.to_slot[to] = there && a.slot ? a.slot[r0 + b] : -1;
    }
}

struct SelectPlan { int piece, n_pieces, share, n_shares; };
static SelectPlan select_plan(const b200_beam_select_args *a) {
    SelectPlan p;
    p.piece = PIECE;
    while ((int64_t)a->n_beams * ((a->n_vocab + p.piece - 1) / p.piece) > MOST_PIECES) p.piece *= 2;
    p.n_pieces = (a->n_vocab + p.piece - 1) / p.piece;
    // a piece a warp until every SM has its CTAs, then up to four: fewer and longer ones
    const int64_t rows = (int64_t)a->n_requests * a->n_beams, ctas = rows * ((p.n_pieces + ROW_WARPS - 1) / ROW_WARPS);
    p.share = ROW_WARPS * (ctas >= 64 * (int64_t)sm_count() ? 8 : ctas >= 32 * (int64_t)sm_count() ? 4 : ctas >= 16 * (int64_t)sm_count() ? 2 : 1);
    p.n_shares = (p.n_pieces + p.share - 1) / p.share;
    return p;
}
static size_t select_room(const b200_beam_select_args *a, const SelectPlan &p) {
    const size_t rows = (size_t)a->n_requests * a->n_beams;
    return rows * ((size_t)p.n_shares * 12 + (size_t)p.n_pieces * 4);
}
static int check_select_sizes(const b200_beam_select_args *a, const char *who) {
    OPX_REQUIRE(a, B200_ERR_INVALID, "%s: NULL arguments", who);
    OPX_REQUIRE(a->type == B200_TYPE_F32 || a->type == B200_TYPE_F16 || a->type == B200_TYPE_BF16, B200_ERR_UNSUPPORTED, "%s: logits of type %d", who, a->type);
    OPX_REQUIRE(a->n_requests >= 0 && a->n_beams > 0 && a->n_vocab > 0 && a->n_keep > 0, B200_ERR_INVALID, "%s: %d requests of %d beams, %d tokens, %d to keep", who, a->n_requests, a->n_beams, a->n_vocab,
                a->n_keep);
    OPX_REQUIRE(a->n_beams <= B200_BEAM_MAX && a->n_keep <= B200_BEAM_KEEP && a->n_vocab <= B200_BEAM_VOCAB, B200_ERR_UNSUPPORTED, "%s: %d beams (%d at most), %d to keep (%d), %d tokens (%d)", who, a->n_beams,
                B200_BEAM_MAX, a->n_keep, B200_BEAM_KEEP, a->n_vocab, B200_BEAM_VOCAB);
    OPX_REQUIRE((int64_t)a->n_requests * a->n_beams <= 65535 && (int64_t)a->n_requests * a->n_keep <= 0x7fffffff, B200_ERR_UNSUPPORTED, "%s: %d requests of %d beams, 65535 rows at most", who,
                a->n_requests, a->n_beams);
    return B200_OK;
}

template <typename T>
static int launch_select(const SelectArgs &a, int rows, bool wide, cudaStream_t st) {
    const dim3 grid((unsigned)a.n_shares, (unsigned)rows);
    B200_CUDA_TRY(launch_chained(wide ? beam_rows_kernel<T, true> : beam_rows_kernel<T, false>, grid, 32 * ROW_WARPS, 0, st, a));
    B200_CUDA_TRY(launch_chained(wide ? beam_pick_kernel<T, true> : beam_pick_kernel<T, false>, (unsigned)(rows / a.beams), PICK_THREADS, 0, st, a));
    return B200_OK;
}

// ------------------------------------------------------------------------------------------------ reordering
// A CTA takes the same bytes of all slots that move, a column: it reads them all into shared memory before it writes any, so nothing is overwritten that is still wanted, whatever cycles
// the moves make.  Columns do not touch one another.
constexpr int REORDER_THREADS = 256, REORDER_STATES = 128, COLUMNS_BYTES = 32 * 1024;
constexpr int64_t MOST_COLUMNS = 0x7fffffff - 0x10000;  // of a launch: a CTA's next column is one grid further, and grids are below 2^16
constexpr int REORDER_MOST = COLUMNS_BYTES + 4 * (B200_STATE_MAX_SLOTS + 2 * B200_STATE_MAX_MOVES);
struct ReorderArgs {
    char *base[REORDER_STATES];
    int64_t stride[REORDER_STATES], bytes[REORDER_STATES];
    int32_t first[REORDER_STATES + 1];  // number of a state's first column
    uint8_t unit_log2[REORDER_STATES];  // bytes of an access: 16, 8 or 4
    int32_t n_states, n, n_slots, width, width_log2;  // width: bytes of a column
    const int32_t *src, *dst;
    int32_t *refused;
};
template <int LOG2>
__device__ __forceinline__ void move_column(unsigned char *column, char *base, int64_t stride, const int *from, const int *to, int n, int width_log2, int bytes) {
    const int shift = width_log2 - LOG2, last = bytes >> LOG2;
#pragma unroll 4
    for (int i = threadIdx.x; i < n << shift; i += REORDER_THREADS) {
        const int k = i >> shift, u = i & ((1 << shift) - 1);
        if (u < last) {
            void *in = column + ((size_t)i << LOG2);
            const char *out = base + from[k] * stride + (u << LOG2);
            if constexpr (LOG2 == 4) cp_async16(in, out);
            else if constexpr (LOG2 == 3) cp_async8(in, out);
            else cp_async4(in, out);
        }
    }
    cp_async_commit();
    cp_async_wait<0>();
    __syncthreads();
#pragma unroll 4
    for (int i = threadIdx.x; i < n << shift; i += REORDER_THREADS) {
        const int k = i >> shift, u = i & ((1 << shift) - 1);
        if (u < last) {
            const unsigned char *in = column + ((size_t)i << LOG2);
            char *out = base + to[k] * stride + (u << LOG2);
            if constexpr (LOG2 == 4) *reinterpret_cast<uint4 *>(out) = *reinterpret_cast<const uint4 *>(in);
            else if constexpr (LOG2 == 3) *reinterpret_cast<uint2 *>(out) = *reinterpret_cast<const uint2 *>(in);
            else *reinterpret_cast<unsigned *>(out) = *reinterpret_cast<const unsigned *>(in);
        }
    }
    __syncthreads();
}
__global__ void __launch_bounds__(REORDER_THREADS, 8) state_reorder_kernel(const ReorderArgs a) {
    extern __shared__ __align__(16) unsigned char column[];  // [n][width], then the moves
    int *claim = (int *)(column + (size_t)a.n * a.width), *from = claim + a.n_slots, *to = from + a.n;
    __shared__ int n_moves, n_refused;
    pdl_wait();  // (the kernel behind is let in by CTAs that are done: one that took places early would leave SMs unequal)
    const int tid = threadIdx.x;
    if (tid == 0) n_moves = n_refused = 0;
    for (int i = tid; i < a.n_slots; i += REORDER_THREADS) claim[i] = 0x7fffffff;
    __syncthreads();
    for (int i = tid; i < a.n; i += REORDER_THREADS) {
        const int s = a.src[i], d = a.dst[i];
        if (s >= 0 && s < a.n_slots && d >= 0 && d < a.n_slots) atomicMin(&claim[d], i);
    }
    __syncthreads();
    for (int i = tid; i < a.n; i += REORDER_THREADS) {
        const int s = a.src[i], d = a.dst[i];
        if (s < 0 || s >= a.n_slots || d < 0 || d >= a.n_slots || claim[d] != i) {
            atomicAdd(&n_refused, 1);
        } else if (s != d) {
            const int k = atomicAdd(&n_moves, 1);
            from[k] = s;
            to[k] = d;
        }
    }
    __syncthreads();
    if (a.refused && blockIdx.x == 0 && tid == 0 && n_refused) atomicAdd(a.refused, n_refused);  // (calls on other streams may raise the same number)
    const int n = n_moves;
    if (n == 0) return;
    for (int item = blockIdx.x; item < a.first[a.n_states]; item += gridDim.x) {
        int lo = 0, hi = a.n_states - 1;  // the last state whose first column is not behind this one
        while (lo < hi) {
            const int mid = (lo + hi + 1) / 2;
            if (a.first[mid] <= item) lo = mid;
            else hi = mid - 1;
        }
        const int64_t at = (int64_t)(item - a.first[lo]) * a.width, stride = a.stride[lo];
        char *base = a.base[lo] + at;
        const int here = (int)min((int64_t)a.width, a.bytes[lo] - at);
        if (a.unit_log2[lo] == 4) move_column<4>(column, base, stride, from, to, n, a.width_log2, here);
        else if (a.unit_log2[lo] == 3) move_column<3>(column, base, stride, from, to, n, a.width_log2, here);
        else move_column<2>(column, base, stride, from, to, n, a.width_log2, here);
    }
}

}  // namespace beam
}  // namespace b200

using namespace b200;
using namespace b200::beam;

extern "C" {

size_t b200_beam_select_workspace_bytes(const b200_beam_select_args *a) {
    if (check_select_sizes(a, "b200_beam_select_workspace_bytes") != B200_OK) return 0;
    return select_room(a, select_plan(a));
}

int b200_op_beam_select(const b200_beam_select_args *a, void *workspace, size_t workspace_bytes, b200_stream_t stream) {
    const char *who = "b200_op_beam_select";
    const int rc = check_select_sizes(a, who);
    if (rc != B200_OK || a->n_requests == 0) return rc;
    OPX_REQUIRE(a->logits && a->score && a->to_score && a->to_beam && a->to_token, B200_ERR_INVALID, "%s: NULL argument", who);
    OPX_REQUIRE(!a->to_slot || a->slot, B200_ERR_INVALID, "%s: to_slot without slot", who);
    OPX_REQUIRE(a->logits_stride >= a->n_vocab, B200_ERR_INVALID, "%s: rows overlap (stride %lld, %d tokens)", who, (long long)a->logits_stride, a->n_vocab);
    OPX_REQUIRE(!a->ended || (a->end_token >= 0 && a->end_token < a->n_vocab), B200_ERR_INVALID, "%s: end token %d of %d", who, a->end_token, a->n_vocab);
    const size_t size = a->type == B200_TYPE_F32 ? 4 : 2;
    OPX_REQUIRE((uintptr_t)a->logits % size == 0 && (((uintptr_t)a->score | (uintptr_t)a->ended | (uintptr_t)a->slot | (uintptr_t)a->to_score | (uintptr_t)a->to_beam | (uintptr_t)a->to_token |
                (uintptr_t)a->to_slot) & 3) == 0, B200_ERR_INVALID, "%s: a pointer is not aligned to its type", who);
    const SelectPlan p = select_plan(a);
    const size_t need = select_room(a, p), rows = (size_t)a->n_requests * a->n_beams;
    // (a request's results are written while others' inputs are still read)
    for (const void *in : {(const void *)a->score, (const void *)a->ended, (const void *)a->slot}) {
        for (const void *out : {(const void *)a->to_score, (const void *)a->to_beam, (const void *)a->to_token, (const void *)a->to_slot}) {
            const uintptr_t i = (uintptr_t)in, o = (uintptr_t)out;
            OPX_REQUIRE(!in || !out || i + 4 * rows <= o || o + 4 * (size_t)a->n_requests * a->n_keep <= i, B200_ERR_INVALID, "%s: not in place", who);
        }
    }
    OPX_REQUIRE(workspace && workspace_bytes >= need && (uintptr_t)workspace % 8 == 0, B200_ERR_INVALID, "%s: workspace of %zu bytes, 8-byte aligned", who, need);
    double *sums = (double *)workspace;
    float *refs = (float *)(sums + rows * p.n_shares);
    const SelectArgs s = {a->logits, a->logits_stride, a->score, a->ended, a->slot, a->to_score, a->to_beam, a->to_token, a->to_slot, a->n_beams, a->n_vocab, a->n_keep, a->end_token,
                          p.piece, p.n_pieces, p.share, p.n_shares, (unsigned)(((1ull << 32) + p.n_pieces - 1) / p.n_pieces), refs + rows * p.n_shares, sums, refs};
    const bool wide = (uintptr_t)a->logits % 16 == 0 && a->logits_stride * (int64_t)size % 16 == 0;
    const cudaStream_t st = (cudaStream_t)stream;
    if (a->type == B200_TYPE_F32) return launch_select<float>(s, (int)rows, wide, st);
    if (a->type == B200_TYPE_F16) return launch_select<__half>(s, (int)rows, wide, st);
    return launch_select<__nv_bfloat16>(s, (int)rows, wide, st);
}

int b200_op_state_reorder(const b200_slot_state *states, int32_t n_states, const int32_t *src, const int32_t *dst, int32_t n, int32_t n_slots, int32_t *refused, b200_stream_t stream) {
    const char *who = "b200_op_state_reorder";
    OPX_REQUIRE(n_states >= 0 && n >= 0 && n_slots >= 0, B200_ERR_INVALID, "%s: %d states, %d moves, %d slots", who, n_states, n, n_slots);
    OPX_REQUIRE(n <= B200_STATE_MAX_MOVES && n_slots <= B200_STATE_MAX_SLOTS, B200_ERR_UNSUPPORTED, "%s: %d moves (%d at most), %d slots (%d)", who, n, B200_STATE_MAX_MOVES, n_slots, B200_STATE_MAX_SLOTS);
    if (n == 0) return B200_OK;
    OPX_REQUIRE(src && dst && (states || n_states == 0), B200_ERR_INVALID, "%s: NULL argument", who);
    OPX_REQUIRE((((uintptr_t)src | (uintptr_t)dst | (uintptr_t)refused) & 3) == 0, B200_ERR_INVALID, "%s: a list at an odd place", who);
    for (int i = 0; i < n_states; i++) {
        const b200_slot_state &s = states[i];
        OPX_REQUIRE(s.bytes >= 0 && s.stride >= s.bytes && (s.base || s.bytes == 0), B200_ERR_INVALID, "%s: state %d: %lld bytes of a slot every %lld", who, i, (long long)s.bytes, (long long)s.stride);
        OPX_REQUIRE((((uintptr_t)s.base | (uint64_t)s.stride | (uint64_t)s.bytes) & 3) == 0, B200_ERR_INVALID, "%s: state %d is not a multiple of 4 bytes", who, i);
    }
    // as wide a column as the moves leave room for
    int log2 = 5;  // (COLUMNS_BYTES / B200_STATE_MAX_MOVES)
    while (log2 < 12 && n << (log2 + 1) <= COLUMNS_BYTES) log2++;
    const int width = 1 << log2;
    const size_t smem = (size_t)n * width + 4 * ((size_t)n_slots + 2 * n);
    if (smem > 48 * 1024) B200_CUDA_TRY(cudaFuncSetAttribute(state_reorder_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, REORDER_MOST));  // (the same for all calls: they may be in several threads)
    int at = 0;
    do {  // (without states too: refused moves are counted)
        ReorderArgs r = {};
        int64_t columns = 0;
        while (at < n_states && r.n_states < REORDER_STATES && columns + (states[at].bytes + width - 1) / width <= MOST_COLUMNS) {
            const b200_slot_state &s = states[at++];
            r.base[r.n_states] = (char *)s.base;
            r.stride[r.n_states] = s.stride;
            r.bytes[r.n_states] = s.bytes;
            const uint64_t all = (uintptr_t)s.base | (uint64_t)s.stride | (uint64_t)s.bytes;
            r.unit_log2[r.n_states] = all % 16 == 0 ? 4 : all % 8 == 0 ? 3 : 2;
            r.first[r.n_states++] = (int32_t)columns;
            columns += (s.bytes + width - 1) / width;
        }
        OPX_REQUIRE(r.n_states > 0 || n_states == 0, B200_ERR_UNSUPPORTED, "%s: a state of %lld bytes a slot", who, (long long)states[at].bytes);
        r.first[r.n_states] = (int32_t)columns;
        r.n = n; r.n_slots = n_slots; r.width = width; r.width_log2 = log2; r.src = src; r.dst = dst;
        r.refused = at >= n_states ? refused : nullptr;
        const int64_t most = (int64_t)(smem < 27 * 1024 ? 8 : smem < 36 * 1024 ? 6 : 4) * sm_count();  // as many as an SM holds, by threads or by shared memory
        const unsigned grid = (unsigned)(columns < 1 ? 1 : columns < most ? columns : most);
        B200_CUDA_TRY(launch_chained(state_reorder_kernel, grid, REORDER_THREADS, smem, (cudaStream_t)stream, r));
    } while (at < n_states);
    return B200_OK;
}

}  // extern "C"
