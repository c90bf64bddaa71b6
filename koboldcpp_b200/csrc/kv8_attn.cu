// kv8_attn.cu -- attention over the paged 8-bit cache (include/b200_kv8.h: b200_op_kv8_attn).
#include <algorithm>
#include <cfloat>
#include <type_traits>

#include "kv8.cuh"
#include "tcgen05.cuh"

namespace b200 {
namespace kv8 {

// ------------------------------------------------------------------------------------------------ shared by the kernels
__device__ __forceinline__ float ex2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ float pow2i(int e) { return __int_as_float((e + 127) << 23); }  // -126 <= e <= 127
// tanh(x) of a score over its cap.  1 - 2 / (1 + e^(2x)) is off by about 2^-22 of 1, whatever the result: 7e-6 of a score under a cap of 30, enough where queries are rounded to f16 or results
// to 16 bits.  Rows of full precision take tanhf, off by two units in the last place of the result (2048 tokens behind 2048 under a
// cap, f32: 318 -> 348 us).
template <bool EXACT> __device__ __forceinline__ float cap_tanh(float x) {
    if constexpr (EXACT) return tanhf(x);
    else return 1.0f - __fdividef(2.0f, 1.0f + ex2(x * 2.8853900817779268f));
}
// x < 2^e for the magnitude with these bits, e >= -100
__device__ __forceinline__ int exponent_above(unsigned bits) { return max((int)(bits >> 23) - 126, -100); }
__device__ __forceinline__ unsigned pack_half(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const unsigned *>(&h);
}
// what the f16 pair `hi` leaves over of (a, b), as another pair
__device__ __forceinline__ unsigned pack_rest(float a, float b, unsigned hi) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&hi));
    return pack_half(a - f.x, b - f.y);
}
// Four int8 as f16, exactly: a byte with its sign flipped is x + 128, behind 0x64 it is the f16 1024 + 128 + x.
__device__ __forceinline__ unsigned less_1152(unsigned u) {
    const unsigned c = 0x64806480u;
    const __half2 r = __hsub2(*reinterpret_cast<const __half2 *>(&u), *reinterpret_cast<const __half2 *>(&c));
    return *reinterpret_cast<const unsigned *>(&r);
}
__device__ __forceinline__ void int4_to_half(unsigned w, unsigned &lo, unsigned &hi) {
    w ^= 0x80808080u;
    lo = less_1152(prmt(w, 0x64646464u, 0x4140));
    hi = less_1152(prmt(w, 0x64646464u, 0x4342));
}
// value i of two words as a pair, i = 0 .. 3: the k side of an MMA's second operand runs along the keys, which lie in different rows
__device__ __forceinline__ void pairs_to_half(unsigned a, unsigned b, unsigned (&p)[4]) {
    const unsigned lo = prmt(a, b, 0x5140) ^ 0x80808080u, hi = prmt(a, b, 0x7362) ^ 0x80808080u;
    p[0] = less_1152(prmt(lo, 0x64646464u, 0x4140));
    p[1] = less_1152(prmt(lo, 0x64646464u, 0x4342));
    p[2] = less_1152(prmt(hi, 0x64646464u, 0x4140));
    p[3] = less_1152(prmt(hi, 0x64646464u, 0x4342));
}
__device__ __forceinline__ void mma_f16(float (&d)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// 16 values of a row of q or dst, whose type is an argument
template <bool VEC>
__device__ __forceinline__ void row_load16_(const void *row, int type, int64_t at, float (&x)[16]) {
    if (type == B200_TYPE_F32) load16<float, VEC>(reinterpret_cast<const float *>(row) + at, x);
    else if (type == B200_TYPE_F16) load16<__half, VEC>(reinterpret_cast<const __half *>(row) + at, x);
    else load16<__nv_bfloat16, VEC>(reinterpret_cast<const __nv_bfloat16 *>(row) + at, x);
}
__device__ __forceinline__ void row_load16(const void *row, int type, int64_t at, bool vec, float (&x)[16]) { vec ? row_load16_<true>(row, type, at, x) : row_load16_<false>(row, type, at, x); }
__device__ __forceinline__ void row_put(void *row, int type, int64_t at, float x) {
    if (type == B200_TYPE_F32) reinterpret_cast<float *>(row)[at] = x;
    else if (type == B200_TYPE_F16) reinterpret_cast<__half *>(row)[at] = __float2half_rn(x);
    else reinterpret_cast<__nv_bfloat16 *>(row)[at] = __float2bfloat16_rn(x);
}
__device__ __forceinline__ void row_store4(void *row, int type, int64_t at, bool vec, float4 y) {
    if (!vec) {
        row_put(row, type, at, y.x); row_put(row, type, at + 1, y.y); row_put(row, type, at + 2, y.z); row_put(row, type, at + 3, y.w);
    } else if (type == B200_TYPE_F32) {
        *reinterpret_cast<float4 *>(reinterpret_cast<float *>(row) + at) = y;
    } else if (type == B200_TYPE_F16) {
        *reinterpret_cast<uint2 *>(reinterpret_cast<__half *>(row) + at) = make_uint2(pack_half(y.x, y.y), pack_half(y.z, y.w));
    } else {
        const __nv_bfloat162 a = __floats2bfloat162_rn(y.x, y.y), b = __floats2bfloat162_rn(y.z, y.w);
        *reinterpret_cast<uint2 *>(reinterpret_cast<__nv_bfloat16 *>(row) + at) = make_uint2(*reinterpret_cast<const unsigned *>(&a), *reinterpret_cast<const unsigned *>(&b));
    }
}
// bits below n of 32
__device__ __forceinline__ unsigned below(int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1; }
// Which of the 32 keys from `key` on a query sees: those up to its own position, and of them those within the window or among the first that stay.  `there`:
// bits 0 and 1, whether the pages of the two 16s are there.
__device__ __forceinline__ unsigned seen_keys(int key, int pos, int there, int window, int keep_first) {
    unsigned seen = below(pos + 1 - key);
    if (window > 0) seen &= ~below(pos + 1 - window - key) | below(keep_first - key);
    return seen & ((there & 1 ? 0xffffu : 0u) | (there & 2 ? 0xffff0000u : 0u));
}

constexpr float LOG2E = 1.4426950408889634f;
// Weights enter the second product times 2^HEAD (f16 holds 2^-24 .. 2^16); the maximum that the exponent subtracts follows the true one only when that
// has grown by more than SLACK, so a weight is below 2^(HEAD + SLACK).
constexpr int HEAD = 6;
constexpr float SLACK = 8.0f;

struct AttnArgs {
    b200_kv8_attn_args a;
    Step step;
    int *counters;    // one per CTA, zero between calls (the prompt kernel's: which of its places are taken)
    float *partials;  // two per CTA
    int group;        // query heads per kv head
    unsigned group_div;  // ceil(2^32 / group): __umulhi(x, group_div) = x / group for x < 2^32 / group
    int table_tokens; // tokens that the table has entries for, at least 1: nobody has to look behind them
    int places;       // for rows that a CTA of the prompt kernel folds (kt_take)
    int splits;       // a prompt's block of rows may be shared by so many CTAs, each with a stretch of its tiles
    int rows_most;    // sequences with more query rows a kv head (tokens times group) are the prompt kernel's; negative: there is none
};

// ------------------------------------------------------------------------------------------------ few query rows a sequence
// The rows of a kv head (tokens times the query heads that share it) come in blocks of R; a block against UNIT keys is a unit of work.  The units of all
// sequences, heads and blocks are numbered, and each CTA takes an equal run of them, whatever the sequences' lengths.  Within a unit each of four
// warps takes 32 keys of its own: pages come by cp.async, one tile ahead, 16-byte pieces exchanged within a row so that both products read
// them without conflicts; int8 becomes f16 in registers, in the layout of the MMA's second operand.  R = 8 rows of f32 fill the 16 rows of the MMA as
// two f16 each (the upper halves and what those leave over), so full precision costs nothing; with one f16 a value R is 16.
// Warps keep maximum, sum and result of their own and meet in shared memory at the end of a run of units of one block; runs of one block in
// several CTAs meet in global memory, where the last one to arrive adds them in the order of the CTAs.
// Scales: a key's joins its score; a value's joins its weight, relative to the power of two above the largest one that the row has seen.
// Measured (heads of 128, 32 query heads over 8, f32): one token behind 131,000: 268 MB in 70.7 us, 3.8 TB/s; 64 sequences of 129 to 4096 tokens: 280 MB in 75.4 us; behind 511: 9.9 us.
// What it spends its time on is instructions, about 1150 a warp for 32 keys (350 of them turn int8 into f16), issued in 59% of the cycles by three warps a scheduler, which wait for one another's
// results in the others; registers (168) allow no fourth.  Short blocks (drafts, f16: 45 MB in 40.5 us) are two thirds loop, 3.5 us for 128 keys, 4.5 us beginning and 7 us end.
constexpr int RW_WARPS = 4, RW_TILE = 32, RW_UNIT = RW_WARPS * RW_TILE, RW_THREADS = RW_WARPS * 32;
constexpr int RW_STAGES = 2, RW_PARTS = 128;
constexpr int RW_BEGIN = 2;  // to begin and end a block costs a CTA about as much as two units: they are counted with each block's
template <int C> constexpr int rw_stage_bytes() { return RW_TILE * 2 * C + 32; }  // keys, values, 2 scales of each, which pages are there
template <int C> constexpr int rw_per_sm() { return C == 64 ? 4 : C == 128 ? 3 : 1; }
template <int C> constexpr int rw_fixed() { return RW_WARPS * RW_STAGES * rw_stage_bytes<C>() + C * 32; }  // stages; q as operands of the first product
template <int C> constexpr int rw_row() { return C + 16; }  // of a warp's results in shared memory, floats: two neighbouring rows fall on the two halves of the banks

// where piece c (16 bytes) of row r of a tile lies
template <int C>
__device__ __forceinline__ int rw_piece(int r, int c) {
    if constexpr (C == 64) return (r >> 1) * 128 + ((((r & 1) << 2 | c) ^ ((r >> 1 & 3) << 1)) << 4);
    else return r * C + (((c & ~7) | ((c & 7) ^ ((r & 1) << 2 | (r >> 1 & 3)))) << 4);
}

template <int C, int TERMS, bool REST>
__global__ void __launch_bounds__(RW_THREADS, rw_per_sm<C>()) kv8_attn_rows_kernel(const __grid_constant__ AttnArgs args, bool vec) {
    pdl_enter();
    constexpr int R = 16 / TERMS, NR = 2 / TERMS;  // rows of a block; a thread's rows in the MMA's result
    constexpr int NT = C / 8, STAGE = rw_stage_bytes<C>(), ROW = rw_row<C>();
    static_assert(RW_WARPS == 4 && RW_PARTS * R * 4 <= RW_WARPS * RW_STAGES * STAGE, "the parts' shares too");
    static_assert(RW_WARPS * R * ROW * 4 <= RW_WARPS * RW_STAGES * STAGE, "the warps' results lie where the stages were");
    extern __shared__ __align__(16) unsigned char smem[];
    uint4 *q_s = reinterpret_cast<uint4 *>(smem + RW_WARPS * RW_STAGES * STAGE);                 // [step of 16 dims][lane]
    long long *sum_s = reinterpret_cast<long long *>(smem + rw_fixed<C>());                      // units of the sequences up to this one
    __shared__ long long warp_sum_s[RW_WARPS];
    __shared__ float top_s[RW_WARPS][16], total_s[RW_WARPS][16], fac_s[RW_WARPS][16], share_s[16], scale_s[16], sink_s[16];
    __shared__ int power_s[RW_WARPS][16], most_s[RW_WARPS], last_s;
    const b200_kv8_attn_args &a = args.a;
    const b200_kv8_cache &c = a.cache;
    const Step &st = args.step;
    const int32_t *info = behind(st.info), *table = behind(st.table);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, tg = lane & 3;
    const int ps = c.page_size, ps_shift = 31 - __clz(ps), group = args.group;
    const size_t record = record_bytes(c);

    struct Span { int keep, first, units, blocks; };  // units of kept first tokens; number of the first unit behind them; units; blocks of rows
    auto span_of = [&](const Seq &q) {
        Span s;
        s.first = a.window > 0 ? max(0, q.held + 1 - a.window) / RW_UNIT : 0;
        s.keep = a.window > 0 ? min((int)(((int64_t)max(a.keep_first, 0) + RW_UNIT - 1) / RW_UNIT), s.first) : 0;
        s.units = s.keep + max((int)((unsigned)(min(q.held + q.count, args.table_tokens) + RW_UNIT - 1) / RW_UNIT) - s.first, 1);
        const int64_t rows = (int64_t)q.count * group;
        s.blocks = args.rows_most >= 0 && rows > args.rows_most ? 0 : (int)((rows + R - 1) / R);
        return s;
    };
    // ---- all sequences' units, summed up
    {
        const int each = (st.n_seq + RW_THREADS - 1) / RW_THREADS, s0 = tid * each;
        long long mine = 0;
        int most = 1;
        for (int s = s0; s < min(s0 + each, st.n_seq); s++) {
            const Seq q = seq_of(st, info, s);
            const Span sp = span_of(q);
            mine += (long long)(sp.units + RW_BEGIN) * sp.blocks * c.n_head_kv;
            most = max(most, sp.blocks > 0 ? sp.units + RW_BEGIN : 1);
            sum_s[s] = mine;
        }
        long long inc = mine;
#pragma unroll
        for (int o = 1; o < 32; o *= 2) { const long long y = __shfl_up_sync(0xffffffffu, inc, o); if (lane >= o) inc += y; }
        most = (int)__reduce_max_sync(0xffffffffu, (unsigned)most);
        if (lane == 31) { warp_sum_s[warp] = inc; most_s[warp] = most; }
        __syncthreads();
        long long before = inc - mine;
        for (int w = 0; w < warp; w++) before += warp_sum_s[w];
        for (int s = s0; s < min(s0 + each, st.n_seq); s++) sum_s[s] += before;
        __syncthreads();
    }
    const long long all = sum_s[st.n_seq - 1];
    // (no block in more than RW_PARTS parts: what one CTA adds up at the end)
    const long long ctas = min(min((long long)gridDim.x, all), max(1ll, (RW_PARTS - 2) * all / max(max(most_s[0], most_s[1]), max(most_s[2], most_s[3]))));
    if ((long long)blockIdx.x >= ctas) return;
    const long long u_end = all * (blockIdx.x + 1) / ctas;

    for (long long u = all * blockIdx.x / ctas; u < u_end;) {
        int s = 0;
        for (int lo = 0, n = st.n_seq; n > 0;) {  // the first sequence whose sum is above u
            const int half = n / 2;
            if (sum_s[lo + half] > u) n = half; else { lo += half + 1; n -= half + 1; }
            s = lo;
        }
        const Seq q = seq_of(st, info, s);
        const Span sp = span_of(q);
        const long long rem = u - (s ? sum_s[s - 1] : 0);
        const unsigned each = (unsigned)(sp.units + RW_BEGIN);
        const int item = rem >> 32 ? (int)(rem / each) : (int)((unsigned)rem / each);
        const int at = (int)(rem - (long long)item * each);  // where in the block this CTA's run of it begins, what RW_BEGIN stands for in front of its units
        const int unit0 = max(at - RW_BEGIN, 0), n_here = (int)min((long long)sp.units, u_end - u + at - RW_BEGIN) - unit0;
        const long long begin = u - at, end = begin + each;
        u = min(end, u_end);
        if (n_here <= 0) continue;  // (the next CTA begins it)
        const int h = item / sp.blocks, row0 = (item - h * sp.blocks) * R, n_rows = min(R, q.count * group - row0);
        const int len = q.held + q.count;
        // row r of the block is query head head0 + r - token(r) * group of token tok0 + token(r)
        const int tok0 = row0 / group, head0 = row0 - tok0 * group;
        auto token = [&](int r) { return group == 1 ? r : (int)__umulhi((unsigned)(head0 + r), args.group_div); };
        const int pos_lo = q.held + tok0, pos_hi = pos_lo + token(n_rows - 1);

        // ---- q: pieces of 16 dims of the block's rows, on their way
        constexpr int PIECES = C / 16, Q_EACH = (R * PIECES + RW_THREADS - 1) / RW_THREADS;
        float x[Q_EACH][16];
#pragma unroll
        for (int i = 0; i < Q_EACH; i++) {
            const int at = tid + i * RW_THREADS, r = at / PIECES, piece = at % PIECES;
#pragma unroll
            for (int e = 0; e < 16; e++) x[i][e] = 0.f;
            if (r < n_rows && piece * 16 < c.dim) {
                const int tok = token(r);
                row_load16(behind(a.q), a.type, (int64_t)(q.first + tok0 + tok) * a.q_stride + (int64_t)(h * group + head0 + r - tok * group) * c.dim + piece * 16, vec, x[i]);
            }
        }

        // ---- stages of pages
        unsigned char *mine = smem + (size_t)warp * RW_STAGES * STAGE;
        auto key_of = [&](int t) {  // the first of this warp's keys of unit t of the run
            const int n = unit0 + t;
            return (n < sp.keep ? n : n - sp.keep + sp.first) * RW_UNIT + warp * RW_TILE;
        };
        auto fetch = [&](int t) {  // lanes 0 and 1: the pages of the two 16s of keys
            const int key = key_of(t) + lane * 16;
            return lane < 2 && t < n_here && key < len ? page_of(st, table, q.row, key >> ps_shift) : -1;
        };
        auto issue = [&](int t, int pages) {
            if (t < n_here) {
                unsigned char *stage = mine + (t % RW_STAGES) * STAGE;
                const int key = key_of(t);
                constexpr int PER_ROW = C / 16, ROWS = 32 / PER_ROW;  // lanes of a row, rows at once
                const int piece = lane % PER_ROW;
                int there = 0;
#pragma unroll
                for (int half = 0; half < 2; half++) {
                    const int page = __shfl_sync(0xffffffffu, pages, half);
                    if (page < 0) continue;
                    there |= 1 << half;
                    const unsigned char *at_page = reinterpret_cast<const unsigned char *>(c.pages) + (size_t)page * record;
                    const unsigned row = (unsigned)(h * ps + ((key + 16 * half) & (ps - 1)));
                    const unsigned char *kp = at_page + row * (unsigned)c.dim + piece * 16, *vp = at_page + v_at(c) + row * (unsigned)c.vdim + piece * 16;
#pragma unroll
                    for (int i = 0; i < 16 / ROWS; i++) {
                        const int r = lane / PER_ROW + i * ROWS, at = rw_piece<C>(16 * half + r, piece);
                        if (piece * 16 < c.dim) cp_async16(stage + at, kp + r * c.dim);
                        if (piece * 16 < c.vdim) cp_async16(stage + RW_TILE * C + at, vp + r * c.vdim);
                    }
                    if (lane < 2) cp_async4(stage + RW_TILE * 2 * C + 8 * half + 4 * lane, at_page + scales_at(c) + (unsigned)(lane * c.n_head_kv + h) * 4);
                }
                if (lane == 0) *reinterpret_cast<int *>(stage + RW_TILE * 2 * C + 16) = there;
            }
            cp_async_commit();
        };
        if (tid < n_rows) sink_s[tid] = a.sink ? a.sink[h * group + head0 + tid - token(tid) * group] * LOG2E : -INFINITY;
        static_assert(RW_STAGES == 2, "one tile on its way, one in use");
        int next_pages = fetch(1);
        issue(0, fetch(0));

        // ---- q as the first operand, each row relative to the power of two above its largest value: in step 4 (piece / 4) + j thread tg holds the dims 4 j .. 4 j + 3 of
        // its piece, as the keys' do
#pragma unroll
        for (int i = 0; i < Q_EACH; i++) {
            const int at = tid + i * RW_THREADS, r = at / PIECES, piece = at % PIECES;
            unsigned loud = 0;
#pragma unroll
            for (int e = 0; e < 16; e++) loud = max(loud, __float_as_uint(x[i][e]) & 0x7fffffffu);
#pragma unroll
            for (int off = 1; off < PIECES; off *= 2) loud = max(loud, __shfl_xor_sync(0xffffffffu, loud, off));
            const int e_q = exponent_above(loud);
            const float down = pow2i(min(14 - e_q, 126));
            if (r >= R) continue;
            if (piece == 0) scale_s[r] = loud >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : a.scale * pow2i(max(e_q - 14, -126)) * (a.softcap > 0.f ? 1.0f / a.softcap : LOG2E);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float x0 = x[i][4 * j] * down, x1 = x[i][4 * j + 1] * down, x2 = x[i][4 * j + 2] * down, x3 = x[i][4 * j + 3] * down;
                const unsigned lo = pack_half(x0, x1), hi = pack_half(x2, x3);
                uint4 *to = q_s + (piece / 4 * 4 + j) * 32 + (r % 8) * 4 + piece % 4;
                if constexpr (TERMS == 2) {
                    *to = make_uint4(lo, pack_rest(x0, x1, lo), hi, pack_rest(x2, x3, hi));
                } else {
                    unsigned *w = reinterpret_cast<unsigned *>(to) + r / 8;
                    w[0] = lo;
                    w[2] = hi;
                }
            }
        }
        __syncthreads();
        float row_scale[NR];
        int pos[NR];
#pragma unroll
        for (int r = 0; r < NR; r++) {
            row_scale[r] = scale_s[g + 8 * r];
            pos[r] = g + 8 * r < n_rows ? pos_lo + token(g + 8 * r) : -1;  // (no such row: sees nothing)
        }

        float o[NT][4], m[NR], l[NR];
        int power[NR];  // the scales of the values that a row has seen are below 2^power
#pragma unroll
        for (int i = 0; i < NT; i++) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
#pragma unroll
        for (int r = 0; r < NR; r++) { m[r] = -INFINITY; l[r] = 0.f; power[r] = -100; }

        for (int t = 0; t < n_here; t++) {
            cp_async_wait<0>();
            __syncwarp();
            issue(t + 1, next_pages);
            next_pages = fetch(t + 2);
            const unsigned char *stage = mine + (t % RW_STAGES) * STAGE;
            const int key0 = key_of(t);
            const int there = *reinterpret_cast<const volatile int *>(stage + RW_TILE * 2 * C + 16);
            if (key0 > pos_hi || there == 0) continue;
            // ---- scores
            float sc[4][4];
#pragma unroll
            for (int n = 0; n < 4; n++) sc[n][0] = sc[n][1] = sc[n][2] = sc[n][3] = 0.f;
#pragma unroll
            for (int hf = 0; hf < C / 64; hf++) {
                if (hf * 64 >= c.dim) break;
                uint4 w[4];
#pragma unroll
                for (int n = 0; n < 4; n++) w[n] = *reinterpret_cast<const uint4 *>(stage + rw_piece<C>(8 * n + g, tg + 4 * hf));
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const uint4 qv = q_s[(hf * 4 + j) * 32 + lane];
                    const unsigned qf[4] = {qv.x, qv.y, qv.z, qv.w};
#pragma unroll
                    for (int n = 0; n < 4; n++) {
                        unsigned b0, b1;
                        int4_to_half(j == 0 ? w[n].x : j == 1 ? w[n].y : j == 2 ? w[n].z : w[n].w, b0, b1);
                        mma_f16(sc[n], qf, b0, b1);
                    }
                }
            }
            const float4 scales = *reinterpret_cast<const float4 *>(stage + RW_TILE * 2 * C);  // keys, values of the first 16, then of the others
            float p[NR][8];
#pragma unroll
            for (int n = 0; n < 4; n++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const float ks = n < 2 ? scales.x : scales.z;
                    if constexpr (TERMS == 2) p[0][2 * n + e] = (sc[n][e] + sc[n][2 + e]) * (row_scale[0] * ks);
                    else { p[0][2 * n + e] = sc[n][e] * (row_scale[0] * ks); p[NR - 1][2 * n + e] = sc[n][2 + e] * (row_scale[NR - 1] * ks); }
                }
            if (a.softcap > 0.f) {
                const float cap_log2 = a.softcap * LOG2E;
#pragma unroll
                for (int r = 0; r < NR; r++)
#pragma unroll
                    for (int i = 0; i < 8; i++) p[r][i] = cap_log2 * cap_tanh<TERMS == 2>(p[r][i]);
            }
            const bool whole = there == 3 && n_rows == R && key0 + RW_TILE - 1 <= pos_lo && (a.window <= 0 || pos_hi - key0 < a.window);
            unsigned seen[NR];
#pragma unroll
            for (int r = 0; r < NR; r++) {
                seen[r] = whole ? 0xffffffffu : seen_keys(key0, pos[r], there, a.window, a.keep_first);
                if (whole) continue;
                const unsigned own = seen[r] >> (2 * tg);
#pragma unroll
                for (int i = 0; i < 8; i++) p[r][i] = own >> (8 * (i / 2) + i % 2) & 1u ? p[r][i] : -INFINITY;
            }
            // ---- maxima, weights
            float corr[NR], common[NR];
            bool grown = false;
#pragma unroll
            for (int r = 0; r < NR; r++) {
                float top = fmaxf(fmaxf(fmaxf(p[r][0], p[r][1]), fmaxf(p[r][2], p[r][3])), fmaxf(fmaxf(p[r][4], p[r][5]), fmaxf(p[r][6], p[r][7])));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                corr[r] = common[r] = 1.0f;
                if (top > m[r] + SLACK) {  // (m = -inf: as soon as a key is seen)
                    corr[r] = ex2(m[r] - top);
                    m[r] = top;
                    grown = true;
                }
            }
            // the values' scales that a row sees: a new largest one moves its accumulators' power of two
            float vs[NR][2];
#pragma unroll
            for (int r = 0; r < NR; r++) {
                vs[r][0] = seen[r] & 0xffffu ? scales.y : 0.f;
                vs[r][1] = seen[r] & 0xffff0000u ? scales.w : 0.f;
                // a row that sees a page whose scale is NaN: its sum becomes NaN, and with it the row, whatever that page's values are
                const float broken = 0.f * (vs[r][0] + vs[r][1]);
                l[r] += broken;
                if (!(broken == 0.f)) vs[r][0] = vs[r][1] = 0.f;
                const int now = exponent_above(__float_as_uint(fmaxf(vs[r][0], vs[r][1])) & 0x7fffffffu);
                if (now > power[r]) {
                    common[r] = pow2i(max(power[r] - now, -126));
                    power[r] = now;
                    grown = true;
                }
            }
            if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
                for (int r = 0; r < NR; r++) { l[r] *= corr[r]; corr[r] *= common[r]; }
#pragma unroll
                for (int i = 0; i < NT; i++) { o[i][0] *= corr[0]; o[i][1] *= corr[0]; o[i][2] *= corr[NR - 1]; o[i][3] *= corr[NR - 1]; }
            }
            unsigned rest[2][4];  // REST: what f16 leaves over of them
            unsigned pf[2][4];  // the weights as the second product's first operand, for the two 16s of keys
#pragma unroll
            for (int r = 0; r < NR; r++) {
                const float mb = m[r] == -INFINITY ? 0.f : m[r], unit = pow2i(HEAD - power[r]), vs0 = vs[r][0] * unit, vs1 = vs[r][1] * unit;
                float w[8];
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    p[r][i] = ex2(p[r][i] - mb);
                    w[i] = p[r][i] * (i < 4 ? vs0 : vs1);
                }
                l[r] += ((p[r][0] + p[r][1]) + (p[r][2] + p[r][3])) + ((p[r][4] + p[r][5]) + (p[r][6] + p[r][7]));  // (one rounding of the running sum a tile)
#pragma unroll
                for (int half = 0; half < 2; half++) {
                    const unsigned x = pack_half(w[4 * half], w[4 * half + 1]), y = pack_half(w[4 * half + 2], w[4 * half + 3]);
                    pf[half][r] = x;
                    pf[half][2 + r] = y;
                    if constexpr (REST) {
                        rest[half][r] = pack_rest(w[4 * half], w[4 * half + 1], x);
                        rest[half][2 + r] = pack_rest(w[4 * half + 2], w[4 * half + 3], y);
                    }
                    if constexpr (TERMS == 2) {
                        pf[half][1] = pack_rest(w[4 * half], w[4 * half + 1], x);
                        pf[half][3] = pack_rest(w[4 * half + 2], w[4 * half + 3], y);
                    }
                }
            }
            // ---- weights times values: thread g brings the dims of its own 8 (C = 64) or 16 bytes (and those 128 further on) of keys 2 tg, 2 tg + 1, 2 tg + 8, 2 tg + 9
            // The tensor cores cut their sums off instead of rounding them, which a long sum shows as a drift (every addition takes up to 2^-23 of what has been summed up): the products of 16 keys
            // begin at 0, and what they come to is added to o by f32 additions.  (One-term rows of 128 and more dims: one half's code for both, or registers spill, 63.7 us for 60.9 of a
            // serving step; the others lose 2 to 3% by that.)
            const unsigned char *sv = stage + RW_TILE * C;
            constexpr int BYTES = C == 64 ? 8 : 16;
#pragma unroll(C >= 128 && TERMS == 1 && !REST ? 1 : 2)
            for (int half = 0; half < 2; half++) {
                const unsigned pw[4] = {half ? pf[1][0] : pf[0][0], half ? pf[1][1] : pf[0][1], half ? pf[1][2] : pf[0][2], half ? pf[1][3] : pf[0][3]};
#pragma unroll
                for (int cb = 0; cb < (C == 256 ? 2 : 1); cb++) {
                    const int piece = C == 64 ? g >> 1 : (g >> 1 | (g & 1) << 2) + 8 * cb, inside = C == 64 ? (g & 1) * 8 : 0;
                    unsigned wv[4][BYTES / 4];
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const unsigned char *at = sv + rw_piece<C>(16 * half + 2 * tg + (k & 1) + (k >> 1) * 8, piece) + inside;
                        if constexpr (C == 64) {
                            const uint2 v = *reinterpret_cast<const uint2 *>(at);
                            wv[k][0] = v.x; wv[k][1] = v.y;
                        } else {
                            const uint4 v = *reinterpret_cast<const uint4 *>(at);
                            wv[k][0] = v.x; wv[k][1] = v.y; wv[k][2] = v.z; wv[k][3] = v.w;
                        }
                    }
#pragma unroll
                    for (int w = 0; w < BYTES / 4; w++) {
                        unsigned b0[4], b1[4];
                        pairs_to_half(wv[0][w], wv[1][w], b0);
                        pairs_to_half(wv[2][w], wv[3][w], b1);
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            float d[4] = {0.f, 0.f, 0.f, 0.f};
                            if constexpr (REST) mma_f16(d, rest[half], b0[j], b1[j]);
                            mma_f16(d, pw, b0[j], b1[j]);
                            float(&to)[4] = o[16 * cb + 4 * w + j];
                            const float2 x = ft_add2(make_float2(to[0], to[1]), make_float2(d[0], d[1])), y = ft_add2(make_float2(to[2], to[3]), make_float2(d[2], d[3]));
                            to[0] = x.x; to[1] = x.y; to[2] = y.x; to[3] = y.y;
                        }
                    }
                }
            }
        }
        cp_async_wait<0>();
        __syncthreads();

        // ---- the warps meet: rows [warp][R][ROW] where the stages were.  Piece p (4 dims) of a row's 16 dims number n is at p ^ n: thread tg's pieces of the same number
        // fall on different banks
        float *so = reinterpret_cast<float *>(smem);
        auto place = [&](int d) { return C == 64 ? d : (d & ~15) | (((d >> 2 & 3) ^ (d >> 4 & 3)) << 2); };  // (d a multiple of 4)
#pragma unroll
        for (int r = 0; r < NR; r++) {
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
            if (tg == 0) { top_s[warp][g + 8 * r] = m[r]; total_s[warp][g + 8 * r] = l[r]; power_s[warp][g + 8 * r] = power[r]; }
        }
#pragma unroll
        for (int i = 0; i < NT; i += 4) {
            // (columns 2 tg and 2 tg + 1 of tiles i .. i + 3)
            const int d0 = C == 64 ? 16 * tg + i : 128 * (i / 16) + 16 * tg + i % 16, d1 = C == 64 ? d0 + 8 : d0 + 64;
            float *at = so + (warp * R + g) * ROW;
            if constexpr (TERMS == 2) {
                *reinterpret_cast<float4 *>(at + place(d0)) = make_float4(o[i][0] + o[i][2], o[i + 1][0] + o[i + 1][2], o[i + 2][0] + o[i + 2][2], o[i + 3][0] + o[i + 3][2]);
                *reinterpret_cast<float4 *>(at + place(d1)) = make_float4(o[i][1] + o[i][3], o[i + 1][1] + o[i + 1][3], o[i + 2][1] + o[i + 2][3], o[i + 3][1] + o[i + 3][3]);
            } else {
                *reinterpret_cast<float4 *>(at + place(d0)) = make_float4(o[i][0], o[i + 1][0], o[i + 2][0], o[i + 3][0]);
                *reinterpret_cast<float4 *>(at + place(d1)) = make_float4(o[i][1], o[i + 1][1], o[i + 2][1], o[i + 3][1]);
                *reinterpret_cast<float4 *>(at + 8 * ROW + place(d0)) = make_float4(o[i][2], o[i + 1][2], o[i + 2][2], o[i + 3][2]);
                *reinterpret_cast<float4 *>(at + 8 * ROW + place(d1)) = make_float4(o[i][3], o[i + 1][3], o[i + 2][3], o[i + 3][3]);
            }
        }
        // the factor that takes a row's results relative to maximum `top` to the row: 1 / (sum and sink)
        auto finish = [&](int r, float top, float total) {
            const float sink = sink_s[r], mm = fmaxf(top, sink);
            const float f = top == -INFINITY ? (total == 0.f ? 0.f : 1.0f) : ex2(top - mm);
            const float sum = total * f + (sink == -INFINITY ? 0.f : ex2(sink - mm));
            return sum == 0.f ? 0.f : f / sum;
        };
        const bool whole_block = n_here == sp.units;
        __syncthreads();
        if (tid < R) {
            float top = -INFINITY, total = 0.f;
#pragma unroll
            for (int w = 0; w < RW_WARPS; w++) top = fmaxf(top, top_s[w][tid]);
            float f[RW_WARPS];
#pragma unroll
            for (int w = 0; w < RW_WARPS; w++) {
                f[w] = top_s[w][tid] == -INFINITY ? (total_s[w][tid] == 0.f ? 0.f : 1.0f) : ex2(top_s[w][tid] - top);  // (a sum without a maximum is NaN: it stays)
                total += total_s[w][tid] * f[w];
            }
            const float share = whole_block && tid < n_rows ? finish(tid, top, total) : 1.0f;
#pragma unroll
            for (int w = 0; w < RW_WARPS; w++) fac_s[w][tid] = f[w] * pow2i(power_s[w][tid] - HEAD) * share;
            top_s[0][tid] = top;
            total_s[0][tid] = total;
        }
        __syncthreads();
        const int quads = c.vdim / 4, quads_shift = 32 - __clz(quads - 1);  // 4 dims a thread; rows 2^quads_shift apart
        auto sum_of = [&](int r, int d) {
            float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < RW_WARPS; w++) {
                const float4 z = *reinterpret_cast<const float4 *>(so + (w * R + r) * ROW + place(d));
                const float f = fac_s[w][r];
                y = make_float4(y.x + z.x * f, y.y + z.y * f, y.z + z.z * f, y.w + z.w * f);
            }
            return y;
        };
        auto put = [&](int r, int d, float4 y) {
            const int tok = token(r);
            row_store4(a.dst, a.type, (int64_t)(q.first + tok0 + tok) * a.dst_stride + (int64_t)(h * group + head0 + r - tok * group) * c.vdim + d, vec, y);
        };
        if (whole_block) {
            for (int i = tid; i < n_rows << quads_shift; i += RW_THREADS) {
                const int r = i >> quads_shift, d = (i & ((1 << quads_shift) - 1)) * 4;
                if (d < c.vdim) put(r, d, sum_of(r, d));
            }
        } else {
            // ---- part of a block: what began in an earlier CTA is this one's partial 0, what it begins itself its partial 1
            auto cta_of = [&](long long unit) { return (int)(((unit + 1) * ctas - 1) / all); };
            const int c0 = cta_of(begin + RW_BEGIN), parts = cta_of(end - 1) - c0 + 1;
            constexpr int PART = R * (C + 2);
            auto part_at = [&](int k) { return args.partials + ((size_t)(c0 + k) * 2 + (k == 0 ? 1 : 0)) * PART; };
            float *out = part_at((int)blockIdx.x - c0);
            if (tid < R) { out[tid] = top_s[0][tid]; out[R + tid] = total_s[0][tid]; }
            for (int i = tid; i < R << quads_shift; i += RW_THREADS) {
                const int r = i >> quads_shift, d = (i & ((1 << quads_shift) - 1)) * 4;
                if (d < c.vdim) *reinterpret_cast<float4 *>(out + 2 * R + r * C + d) = sum_of(r, d);
            }
            __syncthreads();
            if (tid == 0) {
                __threadfence();  // (what the CTA wrote, the barrier in front)
                last_s = atomicAdd(&args.counters[c0], 1) == parts - 1;
                if (last_s) args.counters[c0] = 0;
                __threadfence();
            }
            __syncthreads();
            if (last_s) {
                // maxima and sums of all parts: LANES threads a row
                float *fac = so;  // [part][R]
                constexpr int LANES = RW_THREADS / R, EACH = RW_PARTS / LANES;
                const int r = tid / LANES, j = tid % LANES;
                float mk[EACH], lk[EACH], top = -INFINITY, total = 0.f;
#pragma unroll
                for (int i = 0; i < EACH; i++) {
                    const int k = j + i * LANES;
                    mk[i] = -INFINITY;
                    lk[i] = 0.f;
                    if (k < parts) { mk[i] = __ldcg(part_at(k) + r); lk[i] = __ldcg(part_at(k) + R + r); }
                    top = fmaxf(top, mk[i]);
                }
#pragma unroll
                for (int off = 1; off < LANES; off *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
#pragma unroll
                for (int i = 0; i < EACH; i++) {
                    const int k = j + i * LANES;
                    const float f = mk[i] == -INFINITY ? (lk[i] == 0.f ? 0.f : 1.0f) : ex2(mk[i] - top);
                    if (k < parts) fac[k * R + r] = f;
                    total += lk[i] * f;
                }
#pragma unroll
                for (int off = 1; off < LANES; off *= 2) total += __shfl_xor_sync(0xffffffffu, total, off);
                if (j == 0) share_s[r] = r < n_rows ? finish(r, top, total) : 0.f;
                __syncthreads();
                // all of a thread's pieces side by side: a part's loads then take their way to L2 and back once
                constexpr int PIECES_EACH = (R * C / 4 + RW_THREADS - 1) / RW_THREADS;
                float4 y[PIECES_EACH];
#pragma unroll
                for (int i = 0; i < PIECES_EACH; i++) y[i] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll(PIECES_EACH >= 8 ? 1 : 8 / PIECES_EACH)
                for (int k = 0; k < parts; k++) {
                    const float *at = part_at(k) + 2 * R, *f = fac + k * R;
#pragma unroll
                    for (int i = 0; i < PIECES_EACH; i++) {
                        const int e = tid + i * RW_THREADS, row = e >> quads_shift, d = (e & ((1 << quads_shift) - 1)) * 4;
                        if (row >= n_rows || d >= c.vdim) continue;
                        const float4 z = __ldcg(reinterpret_cast<const float4 *>(at + row * C + d));
                        const float w = f[row];
                        y[i] = make_float4(y[i].x + z.x * w, y[i].y + z.y * w, y[i].z + z.z * w, y[i].w + z.w * w);
                    }
                }
#pragma unroll
                for (int i = 0; i < PIECES_EACH; i++) {
                    const int e = tid + i * RW_THREADS, row = e >> quads_shift, d = (e & ((1 << quads_shift) - 1)) * 4;
                    if (row >= n_rows || d >= c.vdim) continue;
                    const float w = share_s[row];
                    put(row, d, make_float4(y[i].x * w, y[i].y * w, y[i].z * w, y[i].w * w));
                }
            }
        }
        __syncthreads();  // (the stages are free again)
    }
}

}  // namespace kv8
}  // namespace b200

#include "kv8_attn_tc.cuh"

namespace b200 {
namespace kv8 {

static int attn_class(const b200_kv8_cache &c) { const int d = c.dim > c.vdim ? c.dim : c.vdim; return d <= 64 ? 64 : d <= 128 ? 128 : 256; }
static int rows_grid(const b200_kv8_cache &c) {
    const int k = attn_class(c);
    return sm_count() * (k == 64 ? rw_per_sm<64>() : k == 128 ? rw_per_sm<128>() : rw_per_sm<256>());
}
// counters in front of the partial results: as many for heads of all sizes, so that none lies where a call before left partial results
static size_t rows_counter_bytes() { return ((size_t)sm_count() * rw_per_sm<64>() * 4 + 255) / 256 * 256; }
template <int C, int TERMS, bool REST>
static int launch_rows(const AttnArgs &args, bool vec, cudaStream_t st) {
    static bool done[16] = {};  // cudaFuncSetAttribute is per device
    int dev = 0;
    B200_CUDA_TRY(cudaGetDevice(&dev));
    if (dev >= 16 || !done[dev]) {
        B200_CUDA_TRY(cudaFuncSetAttribute(kv8_attn_rows_kernel<C, TERMS, REST>, cudaFuncAttributeMaxDynamicSharedMemorySize, rw_fixed<C>() + 8 * B200_KV8_MAX_SEQ));
        if (dev < 16) done[dev] = true;
    }
    B200_CUDA_TRY(launch_chained(kv8_attn_rows_kernel<C, TERMS, REST>, (unsigned)rows_grid(args.a.cache), RW_THREADS, (size_t)rw_fixed<C>() + 8 * (size_t)args.a.n_seq, st, args, vec));
    return B200_OK;
}

static int check_attn(const b200_kv8_attn_args *a, const char *who) {
    OPX_REQUIRE(a, B200_ERR_INVALID, "%s: NULL arguments", who);
    const int rc = check_step(&a->cache, a->seq_info, a->table, a->table_stride, a->n_rows, a->n_seq, a->n_tokens, a->type, who);
    if (rc != B200_OK) return rc;
    const b200_kv8_cache &c = a->cache;
    OPX_REQUIRE(a->n_head > 0 && a->n_head % c.n_head_kv == 0, B200_ERR_INVALID, "%s: %d query heads over %d kv heads", who, a->n_head, c.n_head_kv);
    OPX_REQUIRE((int64_t)a->n_tokens * a->n_head <= INT32_MAX, B200_ERR_UNSUPPORTED, "%s: %d tokens of %d query heads", who, a->n_tokens, a->n_head);
    OPX_REQUIRE(a->window >= 0 && a->keep_first >= 0, B200_ERR_INVALID, "%s: window %d, keep_first %d", who, a->window, a->keep_first);
    OPX_REQUIRE(a->scale == a->scale && a->softcap >= 0.0f && a->softcap <= FLT_MAX, B200_ERR_INVALID, "%s: scale or softcap", who);
    if (a->n_tokens == 0 || a->n_seq == 0) return B200_OK;
    OPX_REQUIRE(a->q && a->dst, B200_ERR_INVALID, "%s: NULL q or dst", who);
    OPX_REQUIRE(a->q_stride >= (int64_t)a->n_head * c.dim && a->dst_stride >= (int64_t)a->n_head * c.vdim, B200_ERR_INVALID, "%s: rows of q or dst overlap (strides %lld, %lld)", who,
                (long long)a->q_stride, (long long)a->dst_stride);
    OPX_REQUIRE(aligned_to(type_size(a->type), a->q, a->dst) && aligned_to(4, a->sink), B200_ERR_INVALID, "%s: q, dst or sink is not aligned to its type", who);
    return B200_OK;
}
// Where a step has PROMPT_ROWS query rows over all heads (rows of two terms count twice), its sequences of more than ROWS_MOST rows a kv head are the prompt kernel's, if the
// heads are of its sizes.  What a call costs without a past, behind 1000 and behind 8000 tokens, heads of 128 (us, this file's other kernel : the prompt kernel's launches):
//   bf16, 1 sequence, 32 query heads over 8:   64 tokens  8.6 : 19.5, 22.4 : 28.9,  71 :  47   128 tokens 10 : 21, 32 : 31, 130 :  67   256 tokens 22 : 23, 52 : 35, 246 :  90
//   f32, the same:                             33 tokens  7.6 : 21.0, 20.4 : 30.0,  67 :  48    64 tokens  9 : 21, 29 : 30, 116 :  53   128 tokens 13 : 22, 44 : 33, 219 :  77
//   bf16, 4 sequences:                         17 tokens  9.0 : 18.6, 23.3 : 30.2,  88 :  74    33 tokens  9 : 20, 34 : 34, 146 : 102    64 tokens 14 : 19, 49 : 34, 240 : 144
//   bf16, 16 sequences:                         5 tokens  9.3 : 18.9, 29.7 : 36.8, 136 : 192     9 tokens 10 : 18, 38 : 35, 195 : 183    17 tokens 15 : 18, 56 : 36, 310 : 185
//   bf16, 1 sequence, 8 query heads over 1:   128 tokens  8.9 : 21.0, 18.0 : 29.1,  44 :  41   256 tokens 14 : 22, 23 : 30,  74 :  45
//   f32, the same:                             64 tokens  7.4 : 20.0, 15.6 : 27.3,  39 :  37   128 tokens  8 : 22, 20 : 31,  65 :  44   256 tokens 13 : 24, 29 : 32, 119 : 49
// A border at half of PROMPT_ROWS would win up to 45 us behind 8000 tokens and lose 6 to 14 without a past or behind 1000: steps of a chat begin with little.
// (how long the past is, only the device knows; 5 tokens of 4 heads are 20 rows, 9 are 36)
constexpr int ROWS_MOST = 32, PROMPT_ROWS = 4096;
// queries as one f16 (rows of 16 bits: exactly, but for values far below a row's largest), weights as one (no more bits are asked for than bf16 has, or f16_products allows: 2048 tokens behind
// 2048 take 154 us with one, 171 with two, and results in bf16 are off by 1.67e-3 and 1.66e-3, root mean square)
static bool one_term(const b200_kv8_attn_args *a) { return a->type != B200_TYPE_F32 || a->f16_products != 0; }
static bool one_weight(const b200_kv8_attn_args *a) { return a->type == B200_TYPE_BF16 || a->f16_products != 0; }

// whether some sequences of a step can be the prompt kernel's (which sequences have how many tokens is known on the device only)
static bool has_prompts(const b200_kv8_attn_args *a) {
    const int64_t group = a->n_head / a->cache.n_head_kv, longest = a->max_new > 0 && a->max_new < a->n_tokens ? a->max_new : a->n_tokens;
    return attn_class(a->cache) <= 128 && longest * group > ROWS_MOST && (int64_t)a->n_tokens * a->n_head * (one_term(a) ? 1 : 2) >= PROMPT_ROWS;
}
// The prompt kernel's plan.  256 rows a CTA (keys are converted once for all of them) where blocks of 128 would be more than the SMs, sequences being of one length for all that is
// known here: 32 query heads over 8, bf16, behind 1000: 4 sequences of 256 tokens 67.0 us with 128 rows, 45.0 with 256; of 128 tokens 34.9 and 42.0.  Where blocks are fewer than
// the SMs, several CTAs share a block's tiles: one sequence of 128 tokens behind 8000 took 129 us with one CTA a block.
struct PromptPlan { bool two; int splits; };
static PromptPlan prompt_plan(const b200_kv8_attn_args *a) {
    const int64_t rows = (int64_t)a->n_tokens * (a->n_head / a->cache.n_head_kv), each = (rows + a->n_seq - 1) / a->n_seq;
    const int64_t ctas = a->n_seq * ((each + KT_ROWS - 1) / KT_ROWS) * a->cache.n_head_kv;
    return {ctas > sm_count(), (int)std::max<int64_t>(1, std::min<int64_t>(sm_count() / ctas, KT_SPLITS))};
}
template <int C, int GROUPS>
static int launch_prompt_terms(const AttnArgs &args, bool vec, long long limit, cudaStream_t st) {
    if (!one_term(&args.a)) return launch_tc<C, GROUPS, 2, 2>(args, vec, limit, st);
    return one_weight(&args.a) ? launch_tc<C, GROUPS, 1, 1>(args, vec, limit, st) : launch_tc<C, GROUPS, 1, 2>(args, vec, limit, st);
}
static int launch_prompt(AttnArgs &args, bool vec, int k, long long limit, cudaStream_t st) {
    const PromptPlan plan = prompt_plan(&args.a);
    const bool two = plan.two;
    args.splits = plan.splits;
    if (k == 64) return two ? launch_prompt_terms<64, 2>(args, vec, limit, st) : launch_prompt_terms<64, 1>(args, vec, limit, st);
    return two ? launch_prompt_terms<128, 2>(args, vec, limit, st) : launch_prompt_terms<128, 1>(args, vec, limit, st);
}

}  // namespace kv8

int kv8_attn_check(const b200_kv8_attn_args *a, size_t workspace_bytes) {
    const int rc = kv8::check_attn(a, "b200_op_kv8_attn");
    if (rc != B200_OK || a->n_tokens == 0 || a->n_seq == 0) return rc;
    OPX_REQUIRE(workspace_bytes >= b200_kv8_attn_workspace_bytes(a), B200_ERR_INVALID, "b200_op_kv8_attn: workspace of %zu bytes", b200_kv8_attn_workspace_bytes(a));
    return B200_OK;
}
int kv8_attn_launches(const b200_kv8_attn_args *a) {
    if (a->n_tokens == 0 || a->n_seq == 0) return 0;
    return !kv8::has_prompts(a) ? 1 : kv8::prompt_plan(a).splits > 1 ? 3 : 2;
}

}  // namespace b200

using namespace b200;
using namespace b200::kv8;

extern "C" {

size_t b200_kv8_attn_workspace_bytes(const b200_kv8_attn_args *a) {
    if (!a || b200_kv8_page_bytes(a->cache.page_size, a->cache.n_head_kv, a->cache.dim, a->cache.vdim) == 0) return 0;
    const int grid = rows_grid(a->cache), k = attn_class(a->cache);
    // (the two kernels' partial results are not there at the same time; the prompt kernel's are those of twice the blocks that its plan counts, or as many places of up to 256 rows as SMs)
    const size_t rows = (size_t)grid * 2 * (one_term(a) ? 16 : 8) * (k + 2) * 4, prompts = k <= 128 ? (size_t)2 * sm_count() * KT_ROWS * (k + 2) * 4 : 0;
    return rows_counter_bytes() + (rows > prompts ? rows : prompts);
}

int b200_op_kv8_attn(const b200_kv8_attn_args *a, void *workspace, size_t workspace_bytes, b200_stream_t stream) {
    return b200_op_kv8_attn_wait(a, workspace, workspace_bytes, PAIR_WAIT_LIMIT, stream);
}

int b200_op_kv8_attn_wait(const b200_kv8_attn_args *a, void *workspace, size_t workspace_bytes, int64_t wait_cycles, b200_stream_t stream) {
    const char *who = "b200_op_kv8_attn";
    OPX_REQUIRE(wait_cycles >= 0, B200_ERR_INVALID, "%s: limit below zero", who);
    const int rc = check_attn(a, who);
    if (rc != B200_OK || a->n_tokens == 0 || a->n_seq == 0) return rc;
    OPX_REQUIRE(workspace && workspace_bytes >= b200_kv8_attn_workspace_bytes(a) && (uintptr_t)workspace % 16 == 0, B200_ERR_INVALID, "%s: workspace of %zu bytes, 16-byte aligned", who,
                b200_kv8_attn_workspace_bytes(a));
    const b200_kv8_cache &c = a->cache;
    AttnArgs args = {*a, {a->seq_info, a->table, a->table_stride, a->n_rows, a->n_seq, a->n_tokens, c.n_pages, c.page_size}, (int *)workspace,
                     (float *)((char *)workspace + rows_counter_bytes()), a->n_head / c.n_head_kv, 0, std::max(1, (int)a->table_stride * c.page_size), sm_count(), 1, -1};
    args.group_div = (unsigned)(((1ull << 32) + args.group - 1) / args.group);
    const cudaStream_t st = (cudaStream_t)stream;
    const int k = attn_class(c);
    const bool vec = rows_aligned(a->q, a->q_stride, a->type) && rows_aligned(a->dst, a->dst_stride, a->type);
    if (has_prompts(a)) {
        args.rows_most = ROWS_MOST;
        const int rc2 = launch_prompt(args, vec, k, wait_cycles, st);
        if (rc2 != B200_OK) return rc2;
    }
    if (!one_term(a)) return k == 64 ? launch_rows<64, 2, false>(args, vec, st) : k == 128 ? launch_rows<128, 2, false>(args, vec, st) : launch_rows<256, 2, false>(args, vec, st);
    if (one_weight(a)) return k == 64 ? launch_rows<64, 1, false>(args, vec, st) : k == 128 ? launch_rows<128, 1, false>(args, vec, st) : launch_rows<256, 1, false>(args, vec, st);
    return k == 64 ? launch_rows<64, 1, true>(args, vec, st) : k == 128 ? launch_rows<128, 1, true>(args, vec, st) : launch_rows<256, 1, true>(args, vec, st);
}

}  // extern "C"
