// kv8_attn_tc.cuh -- attention of many new tokens over the paged 8-bit cache on the 5th-generation tensor cores (heads of up to 128).  Included by kv8_attn.cu.
//
// A CTA serves GROUPS times 128 query rows of one kv head (tokens times the query heads that share it) and walks over tiles of 64 keys:
//   S = Q . K^T      tcgen05, both operands in shared memory as f16, into TMEM
//   P = 2^(c S - m)  a thread a row, no exchange between lanes; P goes back to TMEM as f16, in place of S
//   O += P . V       A = P from TMEM, B = V as it lies in the page (keys are the strided side), O stays in TMEM
// Eight warps turn int8 keys and values into f16 once for all the CTA's rows: pieces of 16 bytes come from the pages into registers a tile ahead, and leave for
// shared memory in the 128-byte swizzle that the products read.  int8 is exact in f16, so only Q (TERMS = 2) and P (WEIGHTS = 2) have to be taken apart (upper
// halves and what those leave over, a second product each) for results as f32 gives them, rows of f16 only P; 64 columns of S are just two times 32 of P.
// Softmax: four warps a group of 128 rows.  The maximum that the exponent subtracts follows the true one only when that has grown by SLACK, so O is hardly
// ever rescaled.  A key's scale joins its score, a value's its weight, relative to the power of two above the largest that the row has seen.
// Every S has two buffers a group: products run while the softmax is busy with the tile before.
// Measured (heads of 128, 32 query heads over 8, bf16): 2048 tokens behind 2048 in 154 us, 668 TFLOP/s; 7 ragged prompts of up to 700 tokens, 32 heads with keys of their own, f32,
// in 98 us.  A tile of 64 keys and 256 rows takes 1.45 us where its products take 0.75 and its exponentials 0.55: the four phases of a softmax warp's tile (scores, maximum,
// exponentials, weights) follow one another and two such warps share a scheduler, whose issue is at 54%.  A CTA takes 6.5 us to its first tile and 4.5 after its last.
// With few rows behind many keys, several CTAs (of one group) share a block's tiles; kv8_attn_join_kernel adds their results up.
// Waits have a limit, as in the prompt GEMM: a role that gives up sets `failed`, the others follow, and the status word is set.
#pragma once
#include "tcgen05.cuh"

namespace b200 {
namespace kv8 {

constexpr int KT_ROWS = 128, KT_KEYS = 64;
constexpr int KT_SPLITS = 16, KT_SPLIT_TILES = 4;  // CTAs that share a block of rows at most; tiles that each of them has at least
constexpr int KT_RING = 8;  // scales of so many tiles: a tile's are written when the weights of the tile NB + 2 before it have been used
constexpr int KT_Q_PANEL = KT_ROWS * 128, KT_PANEL = KT_KEYS * 128;  // panels of 64 values, 128 bytes a row
template <int GROUPS> constexpr int kt_threads() { return (GROUPS * 4 + 4 + 8) * 32; }  // softmax; products (one warp a group and product); conversion of keys and of values
template <int GROUPS, int TERMS> constexpr int kt_buffers() { return GROUPS * TERMS == 4 ? 3 : 4; }  // of K and V
template <int C, int GROUPS, int TERMS> constexpr size_t kt_smem() {
    return 1024 + (size_t)GROUPS * TERMS * (C / 64) * KT_Q_PANEL + (size_t)kt_buffers<GROUPS, TERMS>() * 2 * (C / 64) * KT_PANEL;
}
// f16 operands, f32 results, 128 rows
__device__ __forceinline__ unsigned kt_idesc(int n, bool b_mn) { return (1u << 4) | (b_mn ? 1u << 16 : 0u) | ((unsigned)(n >> 3) << 17) | ((unsigned)(KT_ROWS >> 4) << 24); }
// CTAs that share a block of so many tiles
__device__ __forceinline__ int kt_splits(int tiles, int most) { return max(1, min(most, tiles / KT_SPLIT_TILES)); }
template <int C> constexpr size_t kt_part() { return (size_t)KT_ROWS * (C + 2); }  // maxima, sums, rows
// A block of rows at positions pos_lo .. pos_hi: its tiles are those of the kept first tokens, then from the window's on (of which the table has entries for).
struct Tiles { int keep, first, all; };
__device__ __forceinline__ Tiles kt_tiles(const AttnArgs &args, int pos_lo, int pos_hi) {
    const b200_kv8_attn_args &a = args.a;
    Tiles t;
    t.first = a.window > 0 ? max(0, pos_lo + 1 - a.window) / KT_KEYS : 0;
    t.keep = a.window > 0 ? min((int)(((int64_t)max(a.keep_first, 0) + KT_KEYS - 1) / KT_KEYS), t.first) : 0;
    t.all = t.keep + max(min(pos_hi, args.table_tokens - 1) / KT_KEYS + 1 - t.first, 1);
    return t;
}
__device__ __forceinline__ float2 mul2(float2 x, float2 y) {
    float2 r;
    asm("{\n.reg .b64 a, b;\nmov.b64 a, {%2, %3};\nmov.b64 b, {%4, %5};\nmul.rn.f32x2 a, a, b;\nmov.b64 {%0, %1}, a;\n}\n" : "=f"(r.x), "=f"(r.y) : "f"(x.x), "f"(x.y), "f"(y.x), "f"(y.y));
    return r;
}
__device__ __forceinline__ float max3(float x, float y, float z) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(x), "f"(y), "f"(z));
    return r;
}
// accumulators of a row times alpha
template <int C>
__device__ __noinline__ void kt_rescale(unsigned o_at, float alpha) {
#pragma unroll 1
    for (int ch = 0; ch < C / 32; ch++) {
        float v[32];
        unsigned x[32];
        tmem_ld32(o_at + 32 * ch, v);
#pragma unroll
        for (int i = 0; i < 32; i++) x[i] = __float_as_uint(v[i] * alpha);
        tmem_st32(o_at + 32 * ch, x);
    }
}
// 4 values of a row that this thread has written
__device__ __forceinline__ float4 row_load4(const float *p, bool vec) {
    if (vec) return *reinterpret_cast<const float4 *>(p);
    return make_float4(p[0], p[1], p[2], p[3]);
}
// The tensor cores cut their sums off below the last place instead of rounding them: an addition takes up to 2^-23 of what has been summed up, half a last place on average, and a sum that is
// kept in TMEM drifts (values around a mean: 1.7e-6 of the result after 81 additions, 7.4e-6 after 270, 1.5e-4 after 3800).  So after kt_fold_every additions the accumulators go to
// memory, where f32 additions round, and begin at 0 again: to the rows of dst if they are f32, to this CTA's share of the partial results if several share a block, or to a place
// that the CTA takes from the workspace for as long as it runs.  Rows of full precision 128 additions: 2.8e-6 of a result that grows evenly (measured, 30,000 keys), 2^-17 of any, 15% of a prompt's
// time at 2000 to 16,000 keys (64: half of the error, 31%; 256: twice, 6%).  Where queries are one f16, or results have 16 bits, 512: 1.1e-5 and 2^-15, where half a step of f16 is 2.4e-4 or more.
template <int TERMS> constexpr int kt_fold_every() { return TERMS == 2 ? 128 : 512; }
// A place for GROUPS times 128 rows: there are as many as SMs, which run one CTA each (registers), so one is free.  -1: none was.
__device__ __forceinline__ int kt_take(int *places, int n) {
    for (int k = 0; k < 64 * n; k++) {
        const int i = (int)((blockIdx.x + (unsigned)k) % (unsigned)n);
        if (atomicCAS(places + i, 0, 1) == 0) {
            __threadfence();
            return i;
        }
    }
    return -1;
}
// A thread's row of accumulators times `unit`, and what lies at base + at times beta (0: nothing does), to base + at (at < 0: no such row).  Eight lanes exchange their rows' pieces of
// 16 bytes, so that each row's 32 columns are stored side by side (a lane a row took 75% of a prompt's time, 16,000 keys).
template <int C>
__device__ __noinline__ void kt_fold(unsigned o_at, float *base, int64_t at, bool vec, int vdim, float unit, float beta) {
    const int lane = threadIdx.x & 31;
    int64_t rows[8];
    float betas[8];
#pragma unroll
    for (int j = 0; j < 8; j++) {
        rows[j] = __shfl_sync(0xffffffffu, (long long)at, (lane & 24) + j);
        betas[j] = __shfl_sync(0xffffffffu, beta, (lane & 24) + j);
    }
#pragma unroll 1
    for (int ch = 0; ch < vdim; ch += 32) {
        float v[32];
        tmem_ld32(o_at + ch, v);
#pragma unroll
        for (int i = 0; i < 32; i++) v[i] *= unit;
#pragma unroll
        for (int s = 1; s < 8; s *= 2) {
            const bool upper = (lane & s) != 0;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                if (i & s) continue;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    float &a = v[4 * i + e], &b = v[4 * (i | s) + e];
                    const float got = __shfl_xor_sync(0xffffffffu, upper ? a : b, s);
                    a = upper ? got : a;
                    b = upper ? b : got;
                }
            }
        }
        // now piece j is number lane % 8 of row lane / 8 * 8 + j
        const int col = ch + 4 * (lane & 7);
        if (col >= vdim) continue;
        float4 z[8];
#pragma unroll
        for (int j = 0; j < 8; j++) z[j] = rows[j] >= 0 && betas[j] != 0.f ? row_load4(base + rows[j] + col, vec) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (rows[j] >= 0)
                row_store4(base, B200_TYPE_F32, rows[j] + col, vec,
                           make_float4(fmaf(z[j].x, betas[j], v[4 * j]), fmaf(z[j].y, betas[j], v[4 * j + 1]), fmaf(z[j].z, betas[j], v[4 * j + 2]), fmaf(z[j].w, betas[j], v[4 * j + 3])));
    }
}
// Rows that kt_fold has put together at base + at go to dst + to in their type; a thread reads what it has written itself.
__device__ __noinline__ void kt_put(const float *base, int64_t at, void *dst, int type, int64_t to, bool vec, int vdim) {
    const int lane = threadIdx.x & 31;
#pragma unroll 1
    for (int j = 0; j < 8; j++) {
        const int64_t from = __shfl_sync(0xffffffffu, (long long)at, (lane & 24) + j), out = __shfl_sync(0xffffffffu, (long long)to, (lane & 24) + j);
        if (from < 0) continue;
        for (int col = 4 * (lane & 7); col < vdim; col += 32) row_store4(dst, type, out + col, vec, row_load4(base + from + col, true));
    }
}
// A thread's registers from here on, by groups of four warps.  A launch has 96 a thread for 20 warps, 61,440 in all: 8 softmax warps of 144, 8 converting ones of 72
// and 4 of 48 take just those (with one group of rows 16 warps are launched with 128 each, 65,536 in all, of which 4 of 144, 8 of 72 and 4 of 48 take 43,008).
constexpr int KT_REGS_SOFTMAX = 144, KT_REGS_CONVERT = 72, KT_REGS_PRODUCTS = 48;
template <int N, bool MORE>
__device__ __forceinline__ void kt_registers() {
    if constexpr (MORE) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
    else asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
// a whole warp waits
template <int SLEEP>
__device__ __forceinline__ bool kt_wait(unsigned long long *bar, int parity, volatile int *failed, long long limit) {
    return __all_sync(0xffffffffu, pair_wait<SLEEP>(smem_u32(bar), (unsigned)parity, failed, limit));
}

// 8 values of a row as they lie there (16 bits: in the first of the two); zeros where there are none
__device__ __forceinline__ void row_load8(const void *row, int type, int64_t at, bool there, bool vec, uint4 (&u)[2]) {
    u[0] = u[1] = make_uint4(0u, 0u, 0u, 0u);
    if (!there) return;
    const unsigned char *p = reinterpret_cast<const unsigned char *>(row) + at * (type == B200_TYPE_F32 ? 4 : 2);
    if (vec) {
        u[0] = reinterpret_cast<const uint4 *>(p)[0];
        if (type == B200_TYPE_F32) u[1] = reinterpret_cast<const uint4 *>(p)[1];
    } else if (type == B200_TYPE_F32) {
        const unsigned *f = reinterpret_cast<const unsigned *>(p);
        u[0] = make_uint4(f[0], f[1], f[2], f[3]);
        u[1] = make_uint4(f[4], f[5], f[6], f[7]);
    } else {
        const unsigned short *f = reinterpret_cast<const unsigned short *>(p);
        u[0] = make_uint4(f[0] | (unsigned)f[1] << 16, f[2] | (unsigned)f[3] << 16, f[4] | (unsigned)f[5] << 16, f[6] | (unsigned)f[7] << 16);
    }
}
__device__ __forceinline__ void row_values8(const uint4 (&u)[2], int type, float (&x)[8]) {
    const unsigned w[8] = {u[0].x, u[0].y, u[0].z, u[0].w, u[1].x, u[1].y, u[1].z, u[1].w};
    if (type == B200_TYPE_F32) {
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = __uint_as_float(w[e]);
    } else if (type == B200_TYPE_F16) {
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = h2f((unsigned short)(w[e / 2] >> (16 * (e & 1))));
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = __uint_as_float(e & 1 ? w[e / 2] & 0xffff0000u : w[e / 2] << 16);
    }
}
template <int C, int GROUPS, int TERMS, int WEIGHTS>
__global__ void __launch_bounds__(kt_threads<GROUPS>(), 1) kv8_attn_tc_kernel(const __grid_constant__ AttnArgs args, bool vec, long long limit, int *timeout) {
    constexpr int NB = kt_buffers<GROUPS, TERMS>(), PANELS = C / 64, BLOCK = GROUPS * KT_ROWS, SOFTMAX = GROUPS * 4, CONVERT = SOFTMAX + 4;
    constexpr int TILE = PANELS * KT_PANEL;
    extern __shared__ unsigned char smem_raw[];
    unsigned char *smem = reinterpret_cast<unsigned char *>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    __shared__ __align__(8) unsigned long long k_full[NB], k_free[NB], v_full[NB], v_free[NB], s_full[GROUPS][2], p_full[GROUPS][2], o_done[GROUPS][2];
    __shared__ unsigned tmem_base_s;
    __shared__ float row_scale_s[BLOCK];
    __shared__ __align__(16) float scales_s[KT_RING][8];  // of a tile's four 16s of keys: the keys', the values'
    __shared__ int there_s[KT_RING];                      // bit i: their page is there
    __shared__ __align__(8) unsigned long long scales_full[KT_RING];
    __shared__ volatile int failed;
    __shared__ int place_s;
    const b200_kv8_attn_args &a = args.a;
    const b200_kv8_cache &c = a.cache;
    const Step &st = args.step;
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    const int group = args.group, ps = c.page_size, h = (int)(blockIdx.x / (unsigned)args.splits % (unsigned)c.n_head_kv);
    pdl_enter();
    const int32_t *info = behind(st.info), *table = behind(st.table);
    // block j of rows belongs to the sequence s with first_s group / BLOCK + s <= j (long causal walks first, of all heads)
    const int j = (int)((gridDim.x - 1 - blockIdx.x) / (unsigned)(args.splits * c.n_head_kv));
    auto first_block = [&](int first, int s) { return (int)((int64_t)first * group / BLOCK) + s; };
    int s;
    const Seq q = find_seq(st, info, j, s, first_block);
    const int64_t row0_64 = (int64_t)(j - first_block(q.first, s)) * BLOCK, rows_64 = (int64_t)q.count * group;
    if (rows_64 <= args.rows_most || row0_64 < 0 || row0_64 >= rows_64) return;  // (another kernel's, or no block)
    const int row0 = (int)row0_64, n_rows = (int)min((int64_t)BLOCK, rows_64 - row0_64);
    const int pos_lo = q.held + row0 / group, pos_hi = q.held + (row0 + n_rows - 1) / group;
    // local row r is query head head0 + r - token(r) * group of token tok0 + token(r)
    const int tok0 = row0 / group, head0 = row0 - tok0 * group;
    auto token = [&](int r) { return group == 1 ? r : (int)__umulhi((unsigned)(head0 + r), args.group_div); };
    const Tiles tiles_of = kt_tiles(args, pos_lo, pos_hi);
    // this CTA's stretch of them
    const int splits = kt_splits(tiles_of.all, args.splits), z = (int)(blockIdx.x % (unsigned)args.splits);
    if (z >= splits) return;
    const int t_begin = (int)((int64_t)tiles_of.all * z / splits), n_tiles = (int)((int64_t)tiles_of.all * (z + 1) / splits) - t_begin;
    auto key_of = [&](int t) { return (t + t_begin < tiles_of.keep ? t + t_begin : t + t_begin - tiles_of.keep + tiles_of.first) * KT_KEYS; };
    constexpr int fold = kt_fold_every<TERMS>() / (4 * WEIGHTS);  // tiles between two folds, a power of two
    const bool whole_block = splits == 1, folded = n_tiles > fold, placed = folded && whole_block && a.type != B200_TYPE_F32;
    unsigned char *sq = smem, *sk = sq + GROUPS * TERMS * PANELS * KT_Q_PANEL, *sv = sk + NB * TILE;

    if (tid == 0) {
        for (int i = 0; i < NB; i++) { mbar_init(&k_full[i], 4); mbar_init(&k_free[i], GROUPS); mbar_init(&v_full[i], 4); mbar_init(&v_free[i], GROUPS); }
        for (int i = 0; i < KT_RING; i++) mbar_init(&scales_full[i], 1);
        for (int i = 0; i < 2 * GROUPS; i++) { mbar_init(&s_full[i >> 1][i & 1], 1); mbar_init(&p_full[i >> 1][i & 1], 4); mbar_init(&o_done[i >> 1][i & 1], 1); }
        mbar_fence_init();
        place_s = placed ? kt_take(args.counters, args.places) : 0;
        failed = place_s < 0;
    }
    constexpr unsigned TMEM = GROUPS == 2 ? 512 : 256;  // S: two buffers of 64 columns a group; then O
    if (warp == SOFTMAX) tmem_alloc(&tmem_base_s, TMEM);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const unsigned tmem = tmem_base_s, tmem_o = tmem + GROUPS * 2 * KT_KEYS;

    if (warp < SOFTMAX) {
        kt_registers<KT_REGS_SOFTMAX, true>();
        // ===== Q as f16, a row relative to the power of two above its largest value: a thread takes 8 dims, piece number `piece` of a row, of every ROWS-th row
        const int w = warp >> 2, quarter = warp & 3, r = quarter * 32 + lane, row = w * KT_ROWS + r;
        {
            constexpr int PIECES = C / 8, ROWS = SOFTMAX * 32 / PIECES, AT_ONCE = 8;
            const int piece = tid % PIECES;
            const bool there = piece * 8 < c.dim;
            const void *qp = behind(a.q);
            unsigned char *at = sq + piece / 8 * KT_Q_PANEL;
#pragma unroll 1
            for (int r0 = tid / PIECES; r0 < BLOCK; r0 += AT_ONCE * ROWS) {
                uint4 raw[AT_ONCE][2];
#pragma unroll
                for (int k = 0; k < AT_ONCE; k++) {
                    const int rr = r0 + k * ROWS, tok = token(rr);
                    row_load8(qp, a.type, (int64_t)(q.first + tok0 + tok) * a.q_stride + (int64_t)(h * group + head0 + rr - tok * group) * c.dim + piece * 8, rr < n_rows && there, vec, raw[k]);
                }
#pragma unroll
                for (int k = 0; k < AT_ONCE; k++) {
                    const int rr = r0 + k * ROWS, rw = rr % KT_ROWS;
                    float x[8];
                    row_values8(raw[k], a.type, x);
                    unsigned loud = 0;
#pragma unroll
                    for (int e = 0; e < 8; e++) loud = max(loud, __float_as_uint(x[e]) & 0x7fffffffu);
#pragma unroll
                    for (int o = 1; o < PIECES; o *= 2) loud = max(loud, __shfl_xor_sync(0xffffffffu, loud, o));
                    const int e_q = exponent_above(loud);
                    const float down = pow2i(min(14 - e_q, 126));
                    if (piece == 0)
                        row_scale_s[rr] = loud >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : a.scale * pow2i(max(e_q - 14, -126)) * (a.softcap > 0.f ? 1.0f / a.softcap : LOG2E);
                    unsigned hi[4];
#pragma unroll
                    for (int e = 0; e < 4; e++) hi[e] = pack_half(x[2 * e] *= down, x[2 * e + 1] *= down);
                    unsigned char *to = at + rr / KT_ROWS * (TERMS * PANELS * KT_Q_PANEL) + rw * 128 + (((piece % 8) ^ (rw & 7)) << 4);
                    *reinterpret_cast<uint4 *>(to) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                    if constexpr (TERMS == 2)
                        *reinterpret_cast<uint4 *>(to + PANELS * KT_Q_PANEL) = make_uint4(pack_rest(x[0], x[1], hi[0]), pack_rest(x[2], x[3], hi[1]), pack_rest(x[4], x[5], hi[2]),
                                                                                        pack_rest(x[6], x[7], hi[3]));
                }
            }
        }
        fence_proxy_async_smem();
        asm volatile("bar.arrive 2, %0;" ::"n"((SOFTMAX + GROUPS) * 32) : "memory");
        asm volatile("bar.sync 3, %0;" ::"n"(SOFTMAX * 32) : "memory");  // (the rows' scales)

        const bool mine = row < n_rows;
        const int i_tok = tok0 + (mine ? token(row) : 0), head = h * group + (mine ? head0 + row - token(row) * group : 0);
        const float row_scale = row_scale_s[row];
        const int pos = mine ? q.held + i_tok : -1;
        // positions of this warp's rows (none: pos_hi_w < pos_lo_w)
        const int w0 = w * KT_ROWS + quarter * 32, w1 = min(w0 + 31, n_rows - 1);
        const int pos_lo_w = w0 < n_rows ? q.held + (row0 + w0) / group : 0, pos_hi_w = w0 < n_rows ? q.held + (row0 + w1) / group : -1;
        const bool all_rows = w0 + 31 < n_rows;
        const unsigned lanes = (unsigned)(quarter * 32) << 16, o_at = tmem_o + (unsigned)(w * C) + lanes;
        float m = -INFINITY, l = 0.f, m_fold = -INFINITY;
        int power = -100;
        bool ok = place_s >= 0;
        auto part_at = [&]() { return args.partials + ((size_t)(j * c.n_head_kv + h) * args.splits + z) * kt_part<C>(); };
        auto row_at = [&]() { return (int64_t)(q.first + i_tok) * a.dst_stride + (int64_t)head * c.vdim; };  // in dst
        // where rows are folded: dst, this CTA's place or its share of the partial results
        auto fold_base = [&]() { return placed ? args.partials + (size_t)place_s * (BLOCK * C) : whole_block ? reinterpret_cast<float *>(a.dst) : part_at(); };
        auto fold_at = [&]() { return !mine ? -1 : placed ? (int64_t)row * C : whole_block ? row_at() : 2 * KT_ROWS + (int64_t)row * C; };
        auto fold_rows = [&](float unit, float beta) { kt_fold<C>(o_at, fold_base(), fold_at(), vec || placed || !whole_block, c.vdim, unit, beta); };
#pragma unroll 1
        for (int t0 = 0; t0 < n_tiles && ok; t0 += fold) {
        if (t0 > 0) {
            ok = kt_wait<20>(&o_done[w][1], ((t0 - 1) >> 1) & 1, &failed, limit);
            if (!ok) break;
            tc_fence_after();
            fold_rows(pow2i(power - HEAD), t0 == fold ? 0.f : m == m_fold ? 1.0f : ex2(m_fold - m));
            m_fold = m;
        }
        const int t1 = min(t0 + fold, n_tiles);
#pragma unroll 1
        for (int t = t0; t < t1; t++) {
            const int b = t & 1, key0 = key_of(t);
            const unsigned s_at = tmem + (unsigned)((w * 2 + b) * KT_KEYS) + lanes;
            ok = kt_wait<0>(&scales_full[t % KT_RING], (t / KT_RING) & 1, &failed, limit);
            if (!ok) break;
            const int there = there_s[t % KT_RING];
            const float4 k4 = *reinterpret_cast<const float4 *>(&scales_s[t % KT_RING][0]), v4 = *reinterpret_cast<const float4 *>(&scales_s[t % KT_RING][4]);
            float ks[4] = {k4.x * row_scale, k4.y * row_scale, k4.z * row_scale, k4.w * row_scale}, vs[4] = {v4.x, v4.y, v4.z, v4.w};
            ok = kt_wait<20>(&s_full[w][b], (t >> 1) & 1, &failed, limit);
            if (!ok) break;
            tc_fence_after();
            unsigned x[32];
            const bool hidden = there == 0 || key0 > pos_hi_w || (a.window > 0 && pos_lo_w - (key0 + KT_KEYS - 1) >= a.window && key0 >= a.keep_first);
            if (hidden) {
#pragma unroll
                for (int i = 0; i < 32; i++) x[i] = 0u;
                tmem_st32(s_at, x);
                if constexpr (WEIGHTS == 2) tmem_st32(s_at + 32, x);
            } else {
                float v[64];
                tmem_ld32_async(s_at, v);
                tmem_ld32_async(s_at + 32, v + 32);
                const bool whole = there == 15 && all_rows && key0 + KT_KEYS - 1 <= pos_lo_w && (a.window <= 0 || pos_hi_w - key0 < a.window);
                tmem_wait_ld(v);
                unsigned seen[2] = {0xffffffffu, 0xffffffffu};
                // the common tile keeps the raw products; ks takes them to scores times log2 e
                if (!whole || a.softcap > 0.f || !(a.scale > 0.f)) {
#pragma unroll
                    for (int i = 0; i < 64; i++) v[i] *= ks[i / 16];
                    if (a.softcap > 0.f) {
                        const float cap_log2 = a.softcap * LOG2E;
#pragma unroll
                        for (int i = 0; i < 64; i++) v[i] = cap_log2 * cap_tanh<TERMS == 2>(v[i]);
                    }
                    if (!whole) {
                        seen[0] = seen_keys(key0, pos, there, a.window, a.keep_first);
                        seen[1] = seen_keys(key0 + 32, pos, there >> 2, a.window, a.keep_first);
#pragma unroll
                        for (int i = 0; i < 64; i++) v[i] = seen[i / 32] >> (i % 32) & 1u ? v[i] : -INFINITY;
                    }
#pragma unroll
                    for (int i = 0; i < 4; i++) ks[i] = 1.0f;
                }
                float top = -INFINITY, loudest = 0.f;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    float t0 = max3(v[16 * i], v[16 * i + 1], v[16 * i + 2]), t1 = max3(v[16 * i + 3], v[16 * i + 4], v[16 * i + 5]);
                    t0 = max3(t0, v[16 * i + 6], v[16 * i + 7]);
                    t1 = max3(t1, v[16 * i + 8], v[16 * i + 9]);
                    t0 = max3(t0, v[16 * i + 10], v[16 * i + 11]);
                    t1 = max3(t1, v[16 * i + 12], v[16 * i + 13]);
                    top = fmaxf(top, fmaxf(max3(t0, v[16 * i + 14], v[16 * i + 15]), t1) * ks[i]);
                    vs[i] = seen[i / 2] >> (16 * (i & 1)) & 0xffffu ? vs[i] : 0.f;
                    loudest = fmaxf(loudest, vs[i]);  // (passes over NaN)
                }
                // a row that sees a page whose scale is NaN: its sum becomes NaN, and with it the row, whatever that page's values are
                const float broken = 0.f * ((vs[0] + vs[1]) + (vs[2] + vs[3]));
                l += broken;
                if (!(broken == 0.f)) vs[0] = vs[1] = vs[2] = vs[3] = 0.f;
                const bool grown = top > m + SLACK;  // (m = -inf: as soon as a key is seen)
                const int now = exponent_above(__float_as_uint(loudest));
                if (__any_sync(0xffffffffu, grown || now > power)) {
                    float alpha = grown ? ex2(m - top) : 1.0f;
                    if (grown) { m = top; l *= alpha; }
                    if (now > power) { alpha *= pow2i(max(power - now, -126)); power = now; }
                    if (t > t0) {
                        ok = kt_wait<20>(&o_done[w][b ^ 1], ((t - 1) >> 1) & 1, &failed, limit);  // (the second product of the tile before may be under way)
                        if (!ok) break;
                        tc_fence_after();
                        kt_rescale<C>(o_at, alpha);
                    }
                }
                const float mb = m == -INFINITY ? 0.f : m, unit = pow2i(HEAD - power);
                float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
                for (int i = 0; i < 64; i += 2) {
                    const float2 e = ft_fma2(make_float2(v[i], v[i + 1]), make_float2(ks[i / 16], ks[i / 16]), make_float2(-mb, -mb));
                    v[i] = ex2(e.x);
                    v[i + 1] = ex2(e.y);
                    sum[i / 2 & 1] = ft_add2(sum[i / 2 & 1], make_float2(v[i], v[i + 1]));
                }
                l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
                unsigned y[32];
#pragma unroll
                for (int i = 0; i < 64; i += 2) {
                    const float f = vs[i / 16] * unit;
                    const float2 e = mul2(make_float2(v[i], v[i + 1]), make_float2(f, f));
                    x[i / 2] = pack_half(e.x, e.y);
                    if constexpr (WEIGHTS == 2) y[i / 2] = pack_rest(e.x, e.y, x[i / 2]);
                }
                tmem_st32(s_at, x);  // (over scores that have been read)
                if constexpr (WEIGHTS == 2) tmem_st32(s_at + 32, y);
            }
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_full[w][b]);
        }
        }
        // ===== results
        ok = ok && kt_wait<20>(&o_done[w][(n_tiles - 1) & 1], ((n_tiles - 1) >> 1) & 1, &failed, limit);
        tc_fence_after();
        float *part = part_at();
        __syncwarp();
        if (!ok && mine) {  // given up: NaN rows rather than what an earlier call or this one left there
            const float nan = __uint_as_float(0x7fc00000u);
            if (!whole_block) { part[row] = -INFINITY; part[KT_ROWS + row] = nan; }
            else if (folded && !placed) for (int e = 0; e < c.vdim; e++) reinterpret_cast<float *>(a.dst)[(int64_t)(q.first + i_tok) * a.dst_stride + (int64_t)head * c.vdim + e] = nan;
        }
        if (ok) {
            const float sink = a.sink ? a.sink[head] * LOG2E : -INFINITY;
            const float mm = fmaxf(m, sink), f = m == -INFINITY ? (l == 0.f ? 0.f : 1.0f) : ex2(m - mm);
            const float sum = l * f + (sink == -INFINITY ? 0.f : ex2(sink - mm));
            const float inv = sum == 0.f ? 0.f : f / sum, back = pow2i(power - HEAD);
            // (a stretch of the tiles: relative to its own maximum, which goes with its sum to where kv8_attn_join_kernel finds it)
            const float all = whole_block ? inv : 1.0f, share = all * back;
            const float beta = m == m_fold ? all : all * ex2(m_fold - m);
            if (!whole_block && mine) { part[row] = m; part[KT_ROWS + row] = l; }
            if (folded) fold_rows(share, beta);
            if (placed) kt_put(fold_base(), fold_at(), a.dst, a.type, row_at(), vec, c.vdim);
            // 32 columns at a time through shared memory (where this warp's rows of Q were), so that a row's stores lie side by side
            unsigned char *stage = sq + w * TERMS * PANELS * KT_Q_PANEL + quarter * 4096;
            const int e = lane & 7;
            int64_t at[8];  // where this lane's part of the rows 4 k + lane / 8 goes; -1: no such row
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const int rb = w0 + 4 * k + (lane >> 3), tok = token(rb);
                const int64_t row_at = whole_block ? (int64_t)(q.first + tok0 + tok) * a.dst_stride + (int64_t)(h * group + head0 + rb - tok * group) * c.vdim : 2 * KT_ROWS + (int64_t)rb * C;
                at[k] = rb < n_rows ? row_at + 4 * e : -1;
            }
#pragma unroll 1
            for (int ch = folded ? c.vdim : 0; ch < c.vdim; ch += 32) {
                float v[32];
                tmem_ld32(o_at + ch, v);
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    float4 y = make_float4(v[4 * i] * share, v[4 * i + 1] * share, v[4 * i + 2] * share, v[4 * i + 3] * share);
                    if (share == 0.f) y = make_float4(0.f, 0.f, 0.f, 0.f);  // (nothing was seen)
                    *reinterpret_cast<float4 *>(stage + lane * 128 + ((i ^ (lane & 7)) << 4)) = y;
                }
                __syncwarp();
                if (ch + 4 * e < c.vdim) {
#pragma unroll
                    for (int k = 0; k < 8; k++) {
                        const int rr = 4 * k + (lane >> 3);
                        const float4 y = *reinterpret_cast<const float4 *>(stage + rr * 128 + ((e ^ (rr & 7)) << 4));
                        if (at[k] >= 0) whole_block ? row_store4(a.dst, a.type, at[k] + ch, vec, y) : row_store4(part, B200_TYPE_F32, at[k] + ch, true, y);
                    }
                }
                __syncwarp();
            }
        }
    } else if (warp >= CONVERT) {
        // ===== int8 to f16, four warps for the keys and four for the values: of a tile's rows (keys), PIECES pieces of 16 values each
        kt_registers<KT_REGS_CONVERT, false>();
        // (8 neighbouring lanes bring half a panel's row each of two keys: their stores fall on all banks)
        constexpr int U = 2 * PANELS;  // pieces of a thread: keys id / 4 and 32 further on, of every panel
        const bool is_v = warp >= CONVERT + 4;
        const int id = tid & 127, piece = id & 3, row = id >> 2, size = is_v ? c.vdim : c.dim;
        const size_t record = record_bytes(c);
        const unsigned char *base = reinterpret_cast<const unsigned char *>(c.pages), *from = base + (is_v ? v_at(c) : 0) + ((size_t)h * ps + row % 16) * size + piece * 16;
        unsigned char *tiles = is_v ? sv : sk;
        unsigned long long *full = is_v ? v_full : k_full, *free = is_v ? v_free : k_free;
        const int shift = 31 - __clz(ps);
        auto pages_ahead = [&](int t) {  // lane & 3: the pages of a tile's 16s of keys
            const int key = t < n_tiles ? key_of(t) + 16 * (lane & 3) : 0x7fffffff;
            return key <= pos_hi ? page_of(st, table, q.row, key >> shift) : -1;
        };
        // (first warp of the keys') lanes 0 .. 3 the keys' scales of a tile's 16s, 4 .. 7 the values'
        const bool scales = warp == CONVERT;
        auto scale_ahead = [&](int page) {
            if (lane >= 8 || page < 0) return 0.f;
            const volatile float *at = reinterpret_cast<const volatile float *>(base + (size_t)page * record + scales_at(c));
            return at[(lane >> 2) * c.n_head_kv + h];
        };
        uint4 raw[U];
        auto fetch = [&](int t, int pages) {  // pages that are not there: zeros
            const int key0 = t < n_tiles ? key_of(t) : 0;
#pragma unroll
            for (int half = 0; half < 2; half++) {
                const int sixteen = (row >> 4) + 2 * half, page = __shfl_sync(0xffffffffu, pages, sixteen);
                const unsigned char *at = from + (size_t)max(page, 0) * record + (unsigned)(((key0 + 16 * sixteen) & (ps - 1)) * size);
#pragma unroll
                for (int p = 0; p < PANELS; p++) {
                    raw[2 * p + half] = make_uint4(0u, 0u, 0u, 0u);
                    if (page >= 0 && 64 * p + piece * 16 < size) raw[2 * p + half] = ld_behind(reinterpret_cast<const uint4 *>(at + 64 * p));
                }
            }
        };
        int pages = pages_ahead(0);
        fetch(0, pages);
        float scale = 0.f;
        int there = 0;
        if (scales) {
            scale = scale_ahead(pages);
            there = (int)(__ballot_sync(0xffffffffu, pages >= 0) & 15u);
        }
        pages = pages_ahead(1);
        unsigned char *at0 = tiles + row * 128 + (((piece * 2) ^ (row & 7)) << 4);
        for (int t = 0; t < n_tiles; t++) {
            const int nb = t % NB;
            if (t >= NB && !kt_wait<200>(&free[nb], ((t / NB) & 1) ^ 1, &failed, limit)) break;
            if (scales) {
                if (lane < 8) scales_s[t % KT_RING][lane] = scale;
                if (lane == 0) there_s[t % KT_RING] = there;
            }
#pragma unroll
            for (int u = 0; u < U; u++) {
                const unsigned w[4] = {raw[u].x, raw[u].y, raw[u].z, raw[u].w};
                unsigned f[8];
#pragma unroll
                for (int e = 0; e < 4; e++) int4_to_half(w[e], f[2 * e], f[2 * e + 1]);
                unsigned char *at = at0 + nb * TILE + u / 2 * KT_PANEL + u % 2 * (32 * 128);
                *reinterpret_cast<uint4 *>(at) = make_uint4(f[0], f[1], f[2], f[3]);
                *reinterpret_cast<uint4 *>((unsigned char *)((uintptr_t)at ^ 16)) = make_uint4(f[4], f[5], f[6], f[7]);
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&full[nb]);
                if (scales) mbar_arrive(&scales_full[t % KT_RING]);
            }
            fetch(t + 1, pages);
            if (scales) {
                scale = scale_ahead(pages);
                there = (int)(__ballot_sync(0xffffffffu, pages >= 0) & 15u);
            }
            pages = pages_ahead(t + 2);
        }
        __syncwarp();
    } else {
        kt_registers<KT_REGS_PRODUCTS, false>();
        if (warp < SOFTMAX + GROUPS) {
            // ===== first products of a group
            const int w = warp - SOFTMAX;
            asm volatile("bar.sync 2, %0;" ::"n"((SOFTMAX + GROUPS) * 32) : "memory");
            const bool elected = elect_lane();
            const unsigned long long qd = umma_desc_sw128(smem_u32(sq)) + (unsigned)(w * TERMS * PANELS * (KT_Q_PANEL >> 4)), kd0 = umma_desc_sw128(smem_u32(sk));
            const int steps = c.dim / 16, walk = limit > 0 ? n_tiles : 0;
            if (limit <= 0) failed = 1;  // (a try of a barrier takes microseconds, longer than any wait of a short call: this warp gives up without one)
            for (int t = 0; t < walk; t++) {
                const int b = t & 1, nb = t % NB;
                if (!kt_wait<40>(&k_full[nb], (t / NB) & 1, &failed, limit)) break;
                if (t >= 2 && !kt_wait<40>(&o_done[w][b], ((t >> 1) & 1) ^ 1, &failed, limit)) break;  // the weights of tile t - 2 have been used
                tc_fence_after();
                if (elected) {
                    const unsigned sd = tmem + (unsigned)((w * 2 + b) * KT_KEYS);
                    const unsigned long long kd = kd0 + (unsigned)(nb * (TILE >> 4));
                    if (steps == C / 16) {
#pragma unroll
                        for (int term = TERMS - 1; term >= 0; term--)  // (small products first: less is cut off)
#pragma unroll
                            for (int k = 0; k < C / 16; k++)
                                tc_mma_bf16(sd, qd + (unsigned)((term * PANELS + k / 4) * (KT_Q_PANEL >> 4) + 2 * (k % 4)), kd + (unsigned)(k / 4 * (KT_PANEL >> 4) + 2 * (k % 4)), kt_idesc(KT_KEYS, false), term != TERMS - 1 || k != 0);
                    } else {
#pragma unroll 1
                        for (int i = 0; i < TERMS * steps; i++) {
                            const int term = TERMS - 1 - (i >= steps), k = i >= steps ? i - steps : i;
                            tc_mma_bf16(sd, qd + (unsigned)((term * PANELS + k / 4) * (KT_Q_PANEL >> 4) + 2 * (k % 4)), kd + (unsigned)(k / 4 * (KT_PANEL >> 4) + 2 * (k % 4)), kt_idesc(KT_KEYS, false), i != 0);
                        }
                    }
                    tc_commit(&s_full[w][b]);
                    tc_commit(&k_free[nb]);
                }
                __syncwarp();
            }
            __syncwarp();
        } else if (warp < SOFTMAX + 2 * GROUPS) {
            // ===== second products of a group
            const int w = warp - SOFTMAX - GROUPS;
            const bool elected = elect_lane();
            const unsigned long long vd0 = umma_desc_mn_sw128(smem_u32(sv), KT_PANEL);
            const unsigned idesc = kt_idesc(c.vdim, true), out = tmem_o + (unsigned)(w * C);
            for (int t = 0; t < n_tiles; t++) {
                const int b = t & 1, nb = t % NB;
                if (!kt_wait<40>(&v_full[nb], (t / NB) & 1, &failed, limit)) break;
                if (!kt_wait<40>(&p_full[w][b], (t >> 1) & 1, &failed, limit)) break;
                tc_fence_after();
                if (elected) {
                    const unsigned pd = tmem + (unsigned)((w * 2 + b) * KT_KEYS);
                    const unsigned long long vd = vd0 + (unsigned)(nb * (TILE >> 4));
#pragma unroll
                    for (int term = 0; term < WEIGHTS; term++)
#pragma unroll
                        for (int k = 0; k < KT_KEYS / 16; k++) ft_mma_ts(out, pd + 32 * term + 8 * k, vd + (unsigned)(k * (2048 >> 4)), idesc, (t & (fold - 1)) + term + k != 0);
                    tc_commit(&o_done[w][b]);
                    tc_commit(&v_free[nb]);
                }
                __syncwarp();
            }
            __syncwarp();
        }
    }
    __syncwarp();
    __syncthreads();
    if (failed) {  // MMAs that were requested end within this time
        if (tid == 0) atomicExch(timeout, 1);
        for (const long long t0 = clock64(); clock64() - t0 < 4000000LL;) {}
    }
    tc_fence_before();
    __syncthreads();
    if (tid == 0 && placed && place_s >= 0) {
        __threadfence();  // (what the CTA wrote there, the barrier in front)
        atomicExch(&args.counters[place_s], 0);
    }
    if (warp == SOFTMAX) {
        tc_fence_after();
        tmem_dealloc(tmem, TMEM);
    }
}

// Rows of blocks that several CTAs shared: their stretches' results, in the order of the tiles.  A warp a row.
constexpr int KJ_ROWS = 16;  // rows of a CTA
template <int C>
__global__ void __launch_bounds__(256) kv8_attn_join_kernel(const __grid_constant__ AttnArgs args, bool vec) {
    pdl_enter();
    const b200_kv8_attn_args &a = args.a;
    const b200_kv8_cache &c = a.cache;
    const Step &st = args.step;
    const int group = args.group, lane = threadIdx.x & 31, h = (int)(blockIdx.x % (unsigned)c.n_head_kv), j = (int)(blockIdx.x / (unsigned)c.n_head_kv);
    const int32_t *info = behind(st.info);
    auto first_block = [&](int first, int s) { return (int)((int64_t)first * group / KT_ROWS) + s; };
    int s;
    const Seq q = find_seq(st, info, j, s, first_block);
    const int64_t row0 = (int64_t)(j - first_block(q.first, s)) * KT_ROWS, rows = (int64_t)q.count * group;
    if (rows <= args.rows_most || row0 < 0 || row0 >= rows) return;
    const int n_rows = (int)min((int64_t)KT_ROWS, rows - row0), tok0 = (int)(row0 / group), head0 = (int)(row0 - (int64_t)tok0 * group);
    const int pos_lo = q.held + tok0, pos_hi = q.held + (int)((row0 + n_rows - 1) / group);
    const int splits = kt_splits(kt_tiles(args, pos_lo, pos_hi).all, args.splits);
    if (splits == 1) return;  // (stored by its one CTA)
    const float *part = behind(args.partials) + (size_t)(j * c.n_head_kv + h) * args.splits * kt_part<C>();
    for (int r = blockIdx.y * KJ_ROWS + (threadIdx.x >> 5); r < min((int)(blockIdx.y + 1) * KJ_ROWS, n_rows); r += 8) {
        const int tok = (head0 + r) / group, head = h * group + head0 + r - tok * group;
        const float mine = lane < splits ? __ldcg(part + (size_t)lane * kt_part<C>() + r) : -INFINITY, sum_of = lane < splits ? __ldcg(part + (size_t)lane * kt_part<C>() + KT_ROWS + r) : 0.f;
        const float sink = a.sink ? a.sink[head] * LOG2E : -INFINITY, top = fmaxf(warp_max(mine), sink);
        const float f = mine == -INFINITY ? (sum_of == 0.f ? 0.f : 1.0f) : ex2(mine - top);
        const float sum = warp_sum(sum_of * f) + (sink == -INFINITY ? 0.f : ex2(sink - top));
        const float share = sum == 0.f ? 0.f : f / sum;
        float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (int k = 0; k < splits; k++) {
            const float w = __shfl_sync(0xffffffffu, share, k);
            if (4 * lane >= c.vdim) continue;
            const float4 v = __ldcg(reinterpret_cast<const float4 *>(part + (size_t)k * kt_part<C>() + 2 * KT_ROWS + (size_t)r * C) + lane);
            y = make_float4(y.x + v.x * w, y.y + v.y * w, y.z + v.z * w, y.w + v.w * w);
        }
        if (4 * lane < c.vdim) row_store4(a.dst, a.type, (int64_t)(q.first + tok0 + tok) * a.dst_stride + (int64_t)head * c.vdim + 4 * lane, vec, y);
    }
}

template <int C, int GROUPS, int TERMS, int WEIGHTS>
static int launch_tc(const AttnArgs &args, bool vec, long long limit, cudaStream_t st) {
    int *status = nullptr;
    const int rc = gemm_status_word(&status);
    if (rc != B200_OK) return rc;
    static bool done[16] = {};  // cudaFuncSetAttribute is per device
    int dev = 0;
    B200_CUDA_TRY(cudaGetDevice(&dev));
    if (dev >= 16 || !done[dev]) {
        B200_CUDA_TRY(cudaFuncSetAttribute(kv8_attn_tc_kernel<C, GROUPS, TERMS, WEIGHTS>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kt_smem<C, GROUPS, TERMS>()));
        if (dev < 16) done[dev] = true;
    }
    const unsigned blocks = (unsigned)(((int64_t)args.a.n_tokens * args.group / (GROUPS * KT_ROWS) + args.a.n_seq) * args.a.cache.n_head_kv);
    B200_CUDA_TRY(launch_chained(kv8_attn_tc_kernel<C, GROUPS, TERMS, WEIGHTS>, blocks * (unsigned)args.splits, kt_threads<GROUPS>(), kt_smem<C, GROUPS, TERMS>(), st, args, vec, limit, status));
    if (args.splits > 1) B200_CUDA_TRY(launch_chained(kv8_attn_join_kernel<C>, dim3(blocks, KT_ROWS / KJ_ROWS), 256, 0, st, args, vec));
    return B200_OK;
}

}  // namespace kv8
}  // namespace b200
