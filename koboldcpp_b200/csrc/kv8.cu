// kv8.cu -- the paged 8-bit cache of keys and values: what writes it, what reads it back, and what manages its pages (include/b200_kv8.h).
#include <cfloat>
#include <type_traits>

#include "kv8.cuh"

namespace b200 {
namespace kv8 {

int check_cache(const b200_kv8_cache *c, const char *who) {
    OPX_REQUIRE(c->pages != nullptr, B200_ERR_INVALID, "%s: the cache has no pages", who);
    OPX_REQUIRE((uintptr_t)c->pages % 16 == 0, B200_ERR_INVALID, "%s: pages must be 16-byte aligned", who);
    OPX_REQUIRE(c->n_pages > 0, B200_ERR_INVALID, "%s: n_pages %d", who, c->n_pages);
    OPX_REQUIRE(b200_kv8_page_bytes(c->page_size, c->n_head_kv, c->dim, c->vdim) > 0, B200_ERR_UNSUPPORTED,
                "%s: page_size %d (16, 32, 64 or 128), n_head_kv %d (1 to 1024), dim %d, vdim %d (multiples of 16, at most 256)", who, c->page_size, c->n_head_kv, c->dim, c->vdim);
    return B200_OK;
}
int check_step(const b200_kv8_cache *c, const int32_t *seq_info, const int32_t *table, int64_t table_stride, int32_t n_rows, int32_t n_seq, int32_t n_tokens, int32_t type,
               const char *who) {
    const int rc = check_cache(c, who);
    if (rc != B200_OK) return rc;
    OPX_REQUIRE(type_ok(type), B200_ERR_UNSUPPORTED, "%s: type %d of the rows (f32, f16 or bf16)", who, type);
    OPX_REQUIRE(n_seq >= 0 && n_tokens >= 0 && n_rows >= 0 && table_stride >= 0, B200_ERR_INVALID, "%s: negative sizes", who);
    OPX_REQUIRE(n_seq <= B200_KV8_MAX_SEQ, B200_ERR_UNSUPPORTED, "%s: %d sequences in a step, at most %d", who, n_seq, B200_KV8_MAX_SEQ);
    OPX_REQUIRE(table_stride <= 0x7fffffff / c->page_size, B200_ERR_UNSUPPORTED, "%s: rows of more than 2^31 tokens", who);
    OPX_REQUIRE(n_tokens == 0 || n_seq == 0 || (seq_info != nullptr && table != nullptr), B200_ERR_INVALID, "%s: NULL seq_info or table", who);
    OPX_REQUIRE(aligned_to(4, seq_info, table), B200_ERR_INVALID, "%s: seq_info or table at an odd place", who);
    return B200_OK;
}

// ------------------------------------------------------------------------------------------------ store
// Quotients x / s are rounded exactly (to the nearest integer, ties to even), |x| <= 127 s and a little.  MAGIC + x (1 / s) rounds to an integer in the lowest bits, the right one or
// its neighbour; d = x less r s is exact in f32 (both are multiples of the finer of their last places, and the difference is below 2^24 of those; where |x| < s, r is 0 or +-1 and
// the difference is Sterbenz's), and so is 2 d - s beside a tie: comparisons of 2 d with s tell whether r is the right one (s / 2 is no f32 where s is below 2^-125).  It hardly ever is not: put()
// asks whether a piece has such a value, mend() moves it.
constexpr float MAGIC = 12582912.0f;  // 1.5 2^23
__device__ __forceinline__ float rest(float x, float t, float s) { return fmaf(-(t - MAGIC), s, x); }
__device__ __forceinline__ float mend(float t, float d, float below, float above) {  // below: of 2 d - s, above: of 2 d + s, their signs
    const bool odd = (__float_as_uint(t) & 1u) != 0;
    if (below > 0.f || (below == 0.f && odd)) return t + 1.0f;
    if (above < 0.f || (above == 0.f && odd)) return t - 1.0f;
    return t;
}
// lowest bytes of four
__device__ __forceinline__ unsigned pack4(float a, float b, float c, float d) {
    return prmt(prmt(__float_as_uint(a), __float_as_uint(b), 0x0040), prmt(__float_as_uint(c), __float_as_uint(d), 0x0040), 0x5410);
}
__device__ __forceinline__ float max_nan(float x, float y, float z) {  // NaN if one is
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(x), "f"(y), "f"(z));
    return r;
}

// One CTA per (page that gets new tokens, head), half of its threads for the keys and half for the values: the largest magnitude of the new values, the scale, what was there
// before if the scale grew, the new values.  The values wait in registers as they came (KEEP pieces of 16 a thread; of a page with more they are read twice).
// Item j of the grid is a page of sequence s where first_s / page_size + 2 s <= j: a sequence of n tokens touches n / page_size + 2 pages at most, so
// the items of the sequences do not overlap and nothing has to be summed up beforehand.
// Measured: prompts of 3 sequences, 32 heads of 128, bf16, 377 MB (with reading back) in 83 us, 4.5 TB/s (instructions are issued in 65% of the cycles: 3 rounds of arithmetic a value, of
// which two check the rounding; warps wait for their rows in the rest); one token each of 64 sequences, 8 heads, f32: 10 us, of which two ways to memory (the step, then the page and the rows) and their launch are nearly all.
constexpr int ST_THREADS = 128;
struct StoreArgs {
    b200_kv8_cache cache;
    Step step;
    const void *k, *v;
    int64_t k_stride, v_stride;
};
template <typename T, bool VEC>
__global__ void __launch_bounds__(2 * ST_THREADS, 4) kv8_store_kernel(const StoreArgs a) {
    pdl_enter();
    constexpr int KEEP = 16 / sizeof(T) / 2;  // f32: 2, else 4
    __shared__ float top[2 * ST_THREADS / 32];
    const b200_kv8_cache &c = a.cache;
    const Step &st = a.step;
    const int j = blockIdx.x, ps = c.page_size, ps_shift = 31 - __clz(ps), h = blockIdx.y, tid = threadIdx.x % ST_THREADS;
    const bool is_v = threadIdx.x >= ST_THREADS;
    const int32_t *info = behind(st.info), *table = behind(st.table);
    int s;
    const Seq q = find_seq(st, info, j, s, [&](int first, int i) { return (first >> ps_shift) + 2 * i; });
    const int at = (q.held >> ps_shift) + (j - ((q.first >> ps_shift) + 2 * s));
    if (q.count == 0 || at < q.held >> ps_shift || (int64_t)at * ps >= (int64_t)q.held + q.count) return;
    const int page = page_of(st, table, q.row, at);
    if (page < 0) return;
    const int begin = max(q.held, at * ps), used = begin - at * ps, n = (int)min((int64_t)q.held + q.count, (int64_t)(at + 1) * ps) - begin;
    const int size = is_v ? c.vdim : c.dim, pieces = size / 16, total = n * pieces;
    const int64_t stride = is_v ? a.v_stride : a.k_stride;
    const T *src = behind(reinterpret_cast<const T *>(is_v ? a.v : a.k)) + (int64_t)(q.first + begin - q.held) * stride + h * size;
    unsigned char *record = reinterpret_cast<unsigned char *>(c.pages) + (size_t)page * record_bytes(c);
    unsigned char *ints = record + (is_v ? v_at(c) : 0) + (size_t)h * ps * size;
    float *scale = reinterpret_cast<float *>(record + scales_at(c)) + (is_v ? c.n_head_kv : 0) + h;
    const float before = used > 0 ? *scale : 0.f;

    Raw16<T> x[KEEP];
    const unsigned per = (65536u + (unsigned)pieces - 1) / (unsigned)pieces;  // i / pieces = i per >> 16 (i < 2048, pieces <= 16)
    auto fetch = [&](int i, Raw16<T> &y) {
        const int row = (int)((unsigned)i * per >> 16);
        load_raw16<T, VEC>(src + (int64_t)row * stride + (i - row * pieces) * 16, y);
    };
    float loud = 0.f;  // NaN stays
    auto magnitude = [&](const Raw16<T> &y) {
#pragma unroll
        for (int e = 0; e < 16; e += 2) loud = max_nan(loud, fabsf(raw_value(y, e)), fabsf(raw_value(y, e + 1)));
    };
#pragma unroll
    for (int u = 0; u < KEEP; u++) if (tid + u * ST_THREADS < total) fetch(tid + u * ST_THREADS, x[u]);
#pragma unroll
    for (int u = 0; u < KEEP; u++) if (tid + u * ST_THREADS < total) magnitude(x[u]);
    for (int i = tid + KEEP * ST_THREADS; i < total; i += ST_THREADS) {
        Raw16<T> y;
        fetch(i, y);
        magnitude(y);
    }
    // (magnitudes compare like their bits, NaN above all)
    loud = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(loud) & 0x7fffffffu));
    if ((threadIdx.x & 31) == 0) top[threadIdx.x >> 5] = loud;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < ST_THREADS / 32; w++) loud = max_nan(loud, top[(is_v ? ST_THREADS / 32 : 0) + w], 0.f);
    float want = __fdiv_rn(loud, 127.0f), now;
    want = want < FLT_MIN ? 0.f : want;
    const bool broken = !(loud <= FLT_MAX) || !(fabsf(before) <= FLT_MAX);
    if (broken) now = __uint_as_float(0x7fc00000u);
    else if (used == 0) now = want;
    else now = want <= before ? before : fmaxf(want, __fmul_rn(1.25f, before));
    __syncthreads();  // (every thread has read the scale)
    if (tid == 0) *scale = now;
    const float inv = now > 0.f ? __fdiv_rn(1.0f, now) : 0.f;  // (NaN, 0: all values become 0)

    if (used > 0 && !broken && now != before) {  // a scale of 0 in front of one that is not: all of them are 0
        for (int i = tid; i < used * pieces; i += ST_THREADS) {
            uint4 *p = reinterpret_cast<uint4 *>(ints) + i;
            const uint4 u = *p;
            unsigned w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int e = 0; e < 4; e++) {
                float f[4];
#pragma unroll
                for (int b = 0; b < 4; b++) {
                    // q before = hi + lo exactly; with d = hi - r now exact, as above, the signs of 2 (d + lo) -+ now are those of (2 d -+ now) + 2 lo
                    const float qf = (float)(signed char)(w[e] >> (8 * b)), hi = __fmul_rn(qf, before), lo = fmaf(qf, before, -hi);
                    const float t = fmaf(hi, inv, MAGIC), d = rest(hi, t, now);
                    f[b] = mend(t, d, fmaf(2.0f, d, -now) + 2.0f * lo, fmaf(2.0f, d, now) + 2.0f * lo);
                }
                w[e] = pack4(f[0], f[1], f[2], f[3]);
            }
            *p = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
    auto put = [&](int i, const Raw16<T> &y) {
        unsigned w[4];
        float off = 0.f;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            float t[4];
#pragma unroll
            for (int b = 0; b < 4; b++) {
                const float v = raw_value(y, 4 * e + b);
                t[b] = fmaf(v, inv, MAGIC);
                off = fmaxf(off, fabsf(rest(v, t[b], now)));
            }
            w[e] = pack4(t[0], t[1], t[2], t[3]);
        }
        if (!(off + off < now)) {  // a tie, or beside one (or a scale that is 0 or no number)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                float t[4];
#pragma unroll
                for (int b = 0; b < 4; b++) {
                    const float v = raw_value(y, 4 * e + b), t0 = fmaf(v, inv, MAGIC), d = rest(v, t0, now);
                    t[b] = inv > 0.f ? mend(t0, d, fmaf(2.0f, d, -now), fmaf(2.0f, d, now)) : MAGIC;
                }
                w[e] = pack4(t[0], t[1], t[2], t[3]);
            }
        }
        reinterpret_cast<uint4 *>(ints + (size_t)used * size)[i] = make_uint4(w[0], w[1], w[2], w[3]);
    };
#pragma unroll
    for (int u = 0; u < KEEP; u++) if (tid + u * ST_THREADS < total) put(tid + u * ST_THREADS, x[u]);
    for (int i = tid + KEEP * ST_THREADS; i < total; i += ST_THREADS) {
        Raw16<T> y;
        fetch(i, y);
        put(i, y);
    }
}

// ------------------------------------------------------------------------------------------------ load
// One CTA per token: its page once, then pieces of 16 values of all heads, keys before values.  Bound by memory; meant for looking at a cache, and for carrying it elsewhere.
constexpr int LD_THREADS = 256;
struct LoadArgs {
    b200_kv8_cache cache;
    Step step;
    void *k, *v;
    int64_t k_stride, v_stride;
};
template <typename T, bool VEC>
__global__ void __launch_bounds__(LD_THREADS) kv8_load_kernel(const LoadArgs a) {
    pdl_enter();
    const b200_kv8_cache &c = a.cache;
    const Step &st = a.step;
    const int t = blockIdx.x, ps = c.page_size;
    const int32_t *info = behind(st.info), *table = behind(st.table);
    int s;
    const Seq q = find_seq(st, info, t, s, [](int first, int) { return first; });
    if (t < q.first || t - q.first >= q.count) return;
    const int pos = q.held + t - q.first, page = page_of(st, table, q.row, pos / ps), slot = pos % ps;
    const unsigned char *record = behind(reinterpret_cast<const unsigned char *>(c.pages)) + (size_t)max(page, 0) * record_bytes(c);
    const float *scales = reinterpret_cast<const float *>(record + scales_at(c));
    const int nk = a.k ? c.n_head_kv * (c.dim / 16) : 0, nv = a.v ? c.n_head_kv * (c.vdim / 16) : 0;
    for (int i = threadIdx.x; i < nk + nv; i += LD_THREADS) {
        const bool is_v = i >= nk;
        const int size = is_v ? c.vdim : c.dim, e = is_v ? i - nk : i, h = e / (size / 16), piece = e % (size / 16);
        float y[16];
        if (page < 0) {
#pragma unroll
            for (int b = 0; b < 16; b++) y[b] = 0.f;
        } else {
            const uint4 u = *reinterpret_cast<const uint4 *>(record + (is_v ? v_at(c) : 0) + ((size_t)h * ps + slot) * size + piece * 16);
            const float f = scales[(is_v ? c.n_head_kv : 0) + h];
            const unsigned w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int b = 0; b < 16; b++) y[b] = (float)(signed char)(w[b / 4] >> (8 * (b % 4))) * f;
        }
        T *out = reinterpret_cast<T *>(is_v ? a.v : a.k) + (int64_t)t * (is_v ? a.v_stride : a.k_stride) + e * 16;
        store16<T, VEC>(out, y);
    }
}

// ------------------------------------------------------------------------------------------------ pages
struct Records { unsigned char *pages[B200_KV8_MAX_CACHES]; unsigned bytes[B200_KV8_MAX_CACHES]; };  // of up to so many caches, as a kernel's argument

// 16 bytes a thread and round, four rounds in flight.  Copies of pages are bound by memory: in compaction (32 layers, half of the pages live) 526 MB in 88 us of 108, 6 TB/s; the
// rest are counting and ranking, 10 us each.  16 continuations of 4 prompts that grow, 32 layers: 135 MB in 27 us, 10 of them growing.
constexpr int CP_THREADS = 256;
__device__ __forceinline__ void copy_record(unsigned char *base, unsigned bytes, int src, int dst) {
    const uint4 *from = reinterpret_cast<const uint4 *>(base + (size_t)src * bytes);
    uint4 *to = reinterpret_cast<uint4 *>(base + (size_t)dst * bytes);
    const int n = (int)(bytes / 16);
    int i = threadIdx.x;
    for (; i + 3 * CP_THREADS < n; i += 4 * CP_THREADS) {
        uint4 v[4];
#pragma unroll
        for (int u = 0; u < 4; u++) v[u] = from[i + u * CP_THREADS];
#pragma unroll
        for (int u = 0; u < 4; u++) to[i + u * CP_THREADS] = v[u];
    }
    for (; i < n; i += CP_THREADS) to[i] = from[i];
}
// pair i of a list of pages, or of a list of (from, to); a page outside the pool, or -1: no pair
__global__ void __launch_bounds__(CP_THREADS) kv8_copy_kernel(const __grid_constant__ Records r, const int32_t *__restrict__ src, const int32_t *__restrict__ dst, int step, int n_pages) {
    pdl_enter(src, dst);
    const int from = src[(int64_t)blockIdx.x * step], to = dst[(int64_t)blockIdx.x * step];
    if (from < 0 || to < 0 || from >= n_pages || to >= n_pages || from == to) return;
    copy_record(r.pages[blockIdx.y], r.bytes[blockIdx.y], from, to);
}

struct Map { int32_t *table, *len, *refs; int64_t stride; int32_t n_rows, n_pages, page_size; };
__device__ __forceinline__ int pages_for(int tokens, int ps) { return tokens / ps + (tokens % ps != 0); }
// whether one of list[0 .. n) is x, asked by a whole block
__device__ __forceinline__ bool named(const int32_t *list, int n, int x) {
    int hit = 0;
    for (int i = threadIdx.x; i < n; i += blockDim.x) hit |= list[i] == x;
    return __syncthreads_or(hit) != 0;
}

// a CTA per row
__global__ void __launch_bounds__(128) kv8_cut_kernel(const Map m, const int32_t *__restrict__ rows, const int32_t *__restrict__ keep) {
    pdl_enter(rows, keep);
    const int i = blockIdx.x, row = rows[i];
    const bool again = named(rows, i, row);
    if (row < 0 || row >= m.n_rows || again) return;
    const int had = max(m.len[row], 0), left = min(had, keep ? max(keep[i], 0) : 0);
    int32_t *entry = m.table + (int64_t)row * m.stride;
    const int last = (int)min((int64_t)pages_for(had, m.page_size), m.stride);
    for (int e = pages_for(left, m.page_size) + threadIdx.x; e < last; e += blockDim.x) {
        const int p = entry[e];
        if (p >= 0 && p < m.n_pages) atomicSub(&m.refs[p], 1);
        entry[e] = -1;
    }
    __syncthreads();  // (all have read the length)
    if (threadIdx.x == 0) m.len[row] = left;
}

// a CTA per pair
__global__ void __launch_bounds__(128) kv8_fork_kernel(const Map m, const int32_t *__restrict__ src, const int32_t *__restrict__ dst, int n, int32_t *refused) {
    pdl_enter(src, dst);
    const int i = blockIdx.x, from = src[i], to = dst[i];
    const bool again = named(dst, i, to), moving = named(dst, n, from);
    bool ok = !again && !moving && from >= 0 && from < m.n_rows && to >= 0 && to < m.n_rows;
    ok = ok && m.len[to] == 0;  // (only this CTA writes it: any other pair with this dst is refused)
    __syncthreads();
    if (!ok) {
        if (threadIdx.x == 0 && refused) atomicAdd(refused, 1);
        return;
    }
    const int held = max(m.len[from], 0), last = (int)min((int64_t)pages_for(held, m.page_size), m.stride);
    for (int e = threadIdx.x; e < last; e += blockDim.x) {
        const int p = m.table[(int64_t)from * m.stride + e];
        if (p >= 0 && p < m.n_pages) atomicAdd(&m.refs[p], 1);
        m.table[(int64_t)to * m.stride + e] = p;
    }
    if (threadIdx.x == 0) m.len[to] = held;
}

// sum of x over the threads before this one, and over all; 1024 threads, sh: 32 ints.  Begins with a barrier: what the threads did with sh before is over.
__device__ __forceinline__ int scan_1024(int x, int *sh, int &all) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int inc = x;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) { const int y = __shfl_up_sync(0xffffffffu, inc, o); if (lane >= o) inc += y; }
    __syncthreads();
    if (lane == 31) sh[warp] = inc;
    __syncthreads();
    int w = sh[lane];
#pragma unroll
    for (int o = 1; o < 32; o *= 2) { const int y = __shfl_up_sync(0xffffffffu, w, o); if (lane >= o) w += y; }
    all = __shfl_sync(0xffffffffu, w, 31);
    return __shfl_sync(0xffffffffu, w, (warp + 31) & 31) * (warp > 0) + inc - x;
}

// The same of two values at a time, neither below 0; sums stay at 2^31 - 1 once they come to it.
__device__ __forceinline__ int add_up(int a, int b) { return (int)min((unsigned)a + (unsigned)b, 0x7fffffffu); }
__device__ __forceinline__ int2 scan2_1024(int2 x, int2 *sh, int2 &all) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    auto up = [](int2 v, int o) { return make_int2(__shfl_up_sync(0xffffffffu, v.x, o), __shfl_up_sync(0xffffffffu, v.y, o)); };
    auto add = [](int2 a, int2 b) { return make_int2(add_up(a.x, b.x), add_up(a.y, b.y)); };
    int2 inc = x;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) { const int2 y = up(inc, o); if (lane >= o) inc = add(inc, y); }
    __syncthreads();
    if (lane == 31) sh[warp] = inc;
    __syncthreads();
    int2 w = sh[lane], before = up(inc, 1);
#pragma unroll
    for (int o = 1; o < 32; o *= 2) { const int2 y = up(w, o); if (lane >= o) w = add(w, y); }
    all = make_int2(__shfl_sync(0xffffffffu, w.x, 31), __shfl_sync(0xffffffffu, w.y, 31));
    const int2 warps = make_int2(__shfl_sync(0xffffffffu, w.x, (warp + 31) & 31), __shfl_sync(0xffffffffu, w.y, (warp + 31) & 31));
    if (lane == 0) before = make_int2(0, 0);
    return warp > 0 ? add(before, warps) : before;
}

// One CTA, a thread per row of the list: what each needs, sums before it, then the free pages in ascending order, each to the row whose share
// it falls in.  The free pages are counted first (as many as are asked for), because a row that does not get all it needs gets nothing.
// One CTA, because rows are served in order and free pages by number; 48 rows take 9.6 us, all of it latency (8192 entries of refs a round, most often the only one).
constexpr int GR_EACH = 8;  // neighbouring entries of refs a thread looks at per round
__global__ void __launch_bounds__(1024) kv8_grow_kernel(const Map m, const int32_t *__restrict__ rows, const int32_t *__restrict__ n_new, int n, int32_t *__restrict__ seq_info, int32_t *refused,
                                                        int32_t *__restrict__ pairs) {
    pdl_enter(rows, n_new, pairs);
    __shared__ __align__(16) int row_s[1024];
    __shared__ int2 sum_sh[32];
    __shared__ int sh[32], start_s[1024], first_s[1024], short_s;  // start: pages of the rows before; first: table entry of a row's first page
    const int i = threadIdx.x, ps = m.page_size;
    const int row = i < n ? rows[i] : -1, asked = i < n ? n_new[i] : 0;
    row_s[i] = row;
    if (i == 0) short_s = 0;
    __syncthreads();
    bool ok = i < n && row >= 0 && row < m.n_rows && asked >= 0;
    if (i < n) {
        bool again = false;
        for (int j = 0; j < i; j += 4) {
            const int4 r = *reinterpret_cast<const int4 *>(row_s + j);
            again |= r.x == row || (r.y == row && j + 1 < i) || (r.z == row && j + 2 < i) || (r.w == row && j + 3 < i);
        }
        ok = ok && !again;
    }
    const int held = ok ? max(m.len[row], 0) : 0;
    ok = ok && (int64_t)held + asked <= min(m.stride * ps, (int64_t)0x7fffffff);
    const int begin = pages_for(held, ps), more = ok ? pages_for(held + asked, ps) - begin : 0;
    int tail = -1;
    if (ok && asked > 0 && held % ps != 0) {
        const int p = m.table[(int64_t)row * m.stride + held / ps];
        if (p >= 0 && p < m.n_pages && m.refs[p] > 1) tail = p;
    }
    const int need = more + (tail >= 0);
    int n_free = 0;
    int2 sums;
    const int2 sum = scan2_1024(make_int2(need, i < n ? max(asked, 0) : 0), sum_sh, sums);
    const int start = sum.x, total = sums.x, first_token = sum.y;
    ok = ok && (!seq_info || (unsigned)first_token + (unsigned)asked <= 0x7fffffffu);  // (no step has room for it, nor for those behind it)
    start_s[i] = start;
    first_s[i] = begin - (tail >= 0);
    auto free_pages = [&](int base) {
        unsigned mask = 0;
#pragma unroll
        for (int u = 0; u < GR_EACH; u++) { const int p = base + i * GR_EACH + u; if (p < m.n_pages && m.refs[p] == 0) mask |= 1u << u; }
        return mask;
    };
    unsigned first_mask = 0;  // of the first round, which is most often the only one: it need not be asked for twice
    int first_rank = 0, first_all = 0;
    for (int base = 0; base < m.n_pages && n_free < total; base += 1024 * GR_EACH) {
        const unsigned mask = free_pages(base);
        int all;
        const int rank = scan_1024(__popc(mask), sh, all);
        if (base == 0) { first_mask = mask; first_rank = rank; first_all = all; }
        n_free += all;
    }
    ok = ok && (need == 0 || (unsigned)start + (unsigned)need <= (unsigned)n_free);
    if (i < n && !ok) atomicAdd(&short_s, 1);
    row_s[i] = ok ? row : -1;
    __syncthreads();
    int before = 0;
    for (int base = 0; base < m.n_pages && before < min(total, n_free); base += 1024 * GR_EACH) {
        unsigned free_mask = first_mask;
        int all = first_all, rank = first_rank;
        if (base > 0) {
            free_mask = free_pages(base);
            rank = before + scan_1024(__popc(free_mask), sh, all);
        }
        while (free_mask && rank < total) {
            const int p = base + i * GR_EACH + __ffs(free_mask) - 1;
            free_mask &= free_mask - 1;
            int lo = 0, hi = n;  // the last row that starts at or below rank: the one with pages there (rows that need none start where the next does)
            while (hi - lo > 1) { const int mid = (lo + hi) / 2; if (start_s[mid] <= rank) lo = mid; else hi = mid; }
            if (row_s[lo] >= 0) {
                m.table[(int64_t)row_s[lo] * m.stride + first_s[lo] + rank - start_s[lo]] = p;
                m.refs[p] = 1;
            }
            rank++;
        }
        before += all;
    }
    __syncthreads();  // (the table's new entries are there)
    if (i < n) {
        const bool copied = ok && tail >= 0;
        pairs[2 * i] = copied ? tail : -1;
        pairs[2 * i + 1] = copied ? m.table[(int64_t)row * m.stride + first_s[i]] : -1;
        if (copied) atomicSub(&m.refs[tail], 1);
        if (ok) m.len[row] = held + asked;
        if (seq_info) {
            seq_info[i] = first_token;
            seq_info[n + i] = ok ? asked : 0;
            seq_info[2 * n + i] = row;
            seq_info[3 * n + i] = held;
        }
    }
    if (i == 0 && refused && short_s) atomicAdd(refused, short_s);
}

// compaction: counts of live pages per stretch; then, with those, every page's place among the live and the free ones; then the moves.
constexpr int CM_THREADS = 256, CM_EACH = 16, CM_STRETCH = CM_THREADS * CM_EACH;
struct Compact { int32_t *head, *counts, *holes, *movers, *rank; };  // head: live pages, moves
__device__ __forceinline__ int block_total(int x, int *sh) {  // (256 threads)
    x = (int)__reduce_add_sync(0xffffffffu, (unsigned)x);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = x;
    __syncthreads();
    int s = 0;
#pragma unroll
    for (int w = 0; w < CM_THREADS / 32; w++) s += sh[w];
    return s;
}
__device__ __forceinline__ unsigned live_mask(const int32_t *refs, int base, int n_pages) {
    unsigned live = 0;
#pragma unroll
    for (int u = 0; u < CM_EACH; u++) if (base + u < n_pages && refs[base + u] > 0) live |= 1u << u;
    return live;
}
__global__ void __launch_bounds__(CM_THREADS) kv8_count_kernel(const int32_t *__restrict__ refs, int n_pages, int32_t *counts) {
    pdl_enter(refs);
    __shared__ int sh[CM_THREADS / 32];
    const int s = block_total(__popc(live_mask(refs, blockIdx.x * CM_STRETCH + threadIdx.x * CM_EACH, n_pages)), sh);
    if (threadIdx.x == 0) counts[blockIdx.x] = s;
}
__global__ void __launch_bounds__(CM_THREADS) kv8_rank_kernel(const int32_t *__restrict__ refs, int n_pages, const Compact w, int32_t *n_live) {
    pdl_enter(refs);
    __shared__ int sh[CM_THREADS / 32], part[CM_THREADS / 32];
    const int32_t *counts = behind(w.counts);
    const int n = (n_pages + CM_STRETCH - 1) / CM_STRETCH, mine = blockIdx.x;
    int below = 0, all = 0;
    for (int b = threadIdx.x; b < n; b += CM_THREADS) { const int x = counts[b]; all += x; below += b < mine ? x : 0; }
    const int before = block_total(below, sh), live_total = block_total(all, sh);
    const int at = mine * CM_STRETCH + threadIdx.x * CM_EACH;
    const unsigned live = live_mask(refs, at, n_pages);
    // live pages below page `live_total`: those of whole stretches, and of the stretch that it lies in
    const int edge = live_total / CM_STRETCH;
    int under = 0;
    for (int b = threadIdx.x; b < edge; b += CM_THREADS) under += counts[b];
    {
        const int e = edge * CM_STRETCH + threadIdx.x * CM_EACH, left = live_total - e;
        const unsigned x = live_mask(refs, e, n_pages);
        under += __popc(left <= 0 ? 0u : left >= CM_EACH ? x : x & ((1u << left) - 1));
    }
    const int stay = block_total(under, sh);
    // live pages in front of this thread's
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int inc = __popc(live);
#pragma unroll
    for (int o = 1; o < 32; o *= 2) { const int y = __shfl_up_sync(0xffffffffu, inc, o); if (lane >= o) inc += y; }
    if (lane == 31) part[warp] = inc;
    __syncthreads();
    int rank = before + inc - __popc(live);
    for (int i = 0; i < warp; i++) rank += part[i];
#pragma unroll
    for (int u = 0; u < CM_EACH; u++) {
        const int p = at + u;
        if (p >= n_pages) break;
        const bool is_live = live >> u & 1u;
        if (!is_live && p < live_total) w.holes[p - rank] = p;
        if (is_live && p >= live_total) { w.movers[rank - stay] = p; w.rank[p] = rank - stay; }
        rank += is_live;
    }
    if (mine == 0 && threadIdx.x == 0) {
        w.head[0] = live_total;
        w.head[1] = live_total - stay;
        if (n_live) *n_live = live_total;
    }
}
__global__ void __launch_bounds__(CM_THREADS) kv8_move_kernel(const __grid_constant__ Records r, int n_caches, const Map m, const Compact w, bool last) {
    pdl_enter();
    static_assert(CM_THREADS == CP_THREADS, "copy_record");
    const int32_t *head = behind(w.head), *holes = behind(w.holes), *movers = behind(w.movers), *rank = behind(w.rank);
    const int live = head[0], moves = head[1];
    for (int64_t i = blockIdx.x; i < (int64_t)moves * n_caches; i += gridDim.x) {
        const int c = (int)(i / moves), k = (int)(i % moves);
        copy_record(r.pages[c], r.bytes[c], movers[k], holes[k]);
    }
    if (!last) return;  // (of several launches, for more caches than one takes)
    const int64_t me = (int64_t)blockIdx.x * CM_THREADS + threadIdx.x, all = (int64_t)gridDim.x * CM_THREADS;
    for (int64_t e = me; e < (int64_t)m.n_rows * m.stride; e += all) {
        const int p = m.table[e];
        if (p < live || p >= m.n_pages) continue;
        const int k = rank[p];
        if (k >= 0 && k < moves && movers[k] == p) m.table[e] = holes[k];  // (an entry that refs knows nothing of stays)
    }
    for (int64_t k = me; k < moves; k += all) {
        m.refs[holes[k]] = m.refs[movers[k]];
        m.refs[movers[k]] = 0;
    }
}

static int check_map(const b200_kv8_map *m, const char *who) {
    OPX_REQUIRE(m && m->table && m->len && m->refs, B200_ERR_INVALID, "%s: NULL map, table, len or refs", who);
    OPX_REQUIRE(m->n_rows > 0 && m->n_pages > 0 && m->table_stride > 0, B200_ERR_INVALID, "%s: n_rows %d, n_pages %d, table_stride %lld", who, m->n_rows, m->n_pages, (long long)m->table_stride);
    OPX_REQUIRE(m->page_size == 16 || m->page_size == 32 || m->page_size == 64 || m->page_size == 128, B200_ERR_UNSUPPORTED, "%s: page_size %d (16, 32, 64 or 128)", who, m->page_size);
    OPX_REQUIRE(m->table_stride <= 0x7fffffff / m->page_size, B200_ERR_UNSUPPORTED, "%s: rows of more than 2^31 tokens", who);
    return B200_OK;
}
static int check_list(int32_t n, const char *who) {
    OPX_REQUIRE(n >= 0, B200_ERR_INVALID, "%s: a list of %d", who, n);
    OPX_REQUIRE(n <= B200_KV8_MAX_SEQ, B200_ERR_UNSUPPORTED, "%s: a list of %d rows, at most %d", who, n, B200_KV8_MAX_SEQ);
    return B200_OK;
}
static int check_caches(const b200_kv8_cache *caches, int32_t n_caches, int32_t n_pages, int32_t page_size, const char *who) {
    OPX_REQUIRE(n_caches >= 0 && (n_caches == 0 || caches), B200_ERR_INVALID, "%s: NULL caches, or %d of them", who, n_caches);
    OPX_REQUIRE(n_caches <= 65535, B200_ERR_UNSUPPORTED, "%s: %d caches", who, n_caches);
    for (int i = 0; i < n_caches; i++) {
        const int rc = check_cache(&caches[i], who);
        if (rc != B200_OK) return rc;
        OPX_REQUIRE(caches[i].n_pages >= n_pages && (page_size == 0 || caches[i].page_size == page_size), B200_ERR_INVALID, "%s: cache %d has %d pages of %d tokens, the map %d of %d", who, i,
                    caches[i].n_pages, caches[i].page_size, n_pages, page_size);
        OPX_REQUIRE(record_bytes(caches[i]) < ((size_t)1 << 31), B200_ERR_UNSUPPORTED, "%s: pages of 2 GB", who);
    }
    return B200_OK;
}
// up to B200_KV8_MAX_CACHES of them from number `at` on
static int take_records(Records &r, const b200_kv8_cache *caches, int at, int n) {
    const int k = n - at < B200_KV8_MAX_CACHES ? n - at : B200_KV8_MAX_CACHES;
    for (int i = 0; i < k; i++) { r.pages[i] = (unsigned char *)caches[at + i].pages; r.bytes[i] = (unsigned)record_bytes(caches[at + i]); }
    return k;
}
static int launch_copies(const b200_kv8_cache *caches, int n_caches, const int32_t *src, const int32_t *dst, int step, int n, int n_pages, cudaStream_t st) {
    for (int at = 0; at < n_caches; at += B200_KV8_MAX_CACHES) {
        Records r = {};
        const int k = take_records(r, caches, at, n_caches);
        B200_CUDA_TRY(launch_chained(kv8_copy_kernel, dim3((unsigned)n, (unsigned)k), CP_THREADS, 0, st, r, src, dst, step, n_pages));
    }
    return B200_OK;
}
static Map map_of(const b200_kv8_map *m) { return Map{m->table, m->len, m->refs, m->table_stride, m->n_rows, m->n_pages, m->page_size}; }

template <typename T>
static int launch_store(const StoreArgs &s, bool vec, dim3 grid, cudaStream_t st) {
    B200_CUDA_TRY(vec ? launch_chained(kv8_store_kernel<T, true>, grid, 2 * ST_THREADS, 0, st, s) : launch_chained(kv8_store_kernel<T, false>, grid, 2 * ST_THREADS, 0, st, s));
    return B200_OK;
}
template <typename T>
static int launch_load(const LoadArgs &s, bool vec, unsigned grid, cudaStream_t st) {
    B200_CUDA_TRY(vec ? launch_chained(kv8_load_kernel<T, true>, grid, LD_THREADS, 0, st, s) : launch_chained(kv8_load_kernel<T, false>, grid, LD_THREADS, 0, st, s));
    return B200_OK;
}

static int check_store(const b200_kv8_store_args *a, const char *who) {
    const int rc = check_step(&a->cache, a->seq_info, a->table, a->table_stride, a->n_rows, a->n_seq, a->n_tokens, a->type, who);
    if (rc != B200_OK || a->n_tokens == 0 || a->n_seq == 0) return rc;
    const b200_kv8_cache &c = a->cache;
    OPX_REQUIRE(a->k && a->v, B200_ERR_INVALID, "%s: NULL k or v", who);
    OPX_REQUIRE(a->k_stride >= (int64_t)c.n_head_kv * c.dim && a->v_stride >= (int64_t)c.n_head_kv * c.vdim, B200_ERR_INVALID, "%s: rows of k or v overlap (strides %lld, %lld)", who,
                (long long)a->k_stride, (long long)a->v_stride);
    OPX_REQUIRE(aligned_to(type_size(a->type), a->k, a->v), B200_ERR_INVALID, "%s: k or v is not aligned to its type", who);
    return B200_OK;
}

}  // namespace kv8

int kv8_store_check(const b200_kv8_store_args *a) { return kv8::check_store(a, "b200_op_kv8_store"); }

}  // namespace b200

using namespace b200;
using namespace b200::kv8;

extern "C" {

size_t b200_kv8_page_bytes(int32_t page_size, int32_t n_head_kv, int32_t dim, int32_t vdim) {
    if (page_size != 16 && page_size != 32 && page_size != 64 && page_size != 128) return 0;
    if (n_head_kv < 1 || n_head_kv > 1024 || dim < 16 || dim > 256 || dim % 16 || vdim < 16 || vdim > 256 || vdim % 16) return 0;
    b200_kv8_cache c = {nullptr, 0, page_size, n_head_kv, dim, vdim, 0};
    return record_bytes(c);
}

int b200_op_kv8_store(const b200_kv8_store_args *a, b200_stream_t stream) {
    const char *who = "b200_op_kv8_store";
    OPX_REQUIRE(a, B200_ERR_INVALID, "%s: NULL arguments", who);
    const int rc = check_store(a, who);
    if (rc != B200_OK || a->n_tokens == 0 || a->n_seq == 0) return rc;
    const b200_kv8_cache &c = a->cache;
    const StoreArgs s = {c, {a->seq_info, a->table, a->table_stride, a->n_rows, a->n_seq, a->n_tokens, c.n_pages, c.page_size}, a->k, a->v, a->k_stride, a->v_stride};
    const dim3 grid((unsigned)(a->n_tokens / c.page_size + 2 * a->n_seq), (unsigned)c.n_head_kv);
    const bool vec = rows_aligned(a->k, a->k_stride, a->type) && rows_aligned(a->v, a->v_stride, a->type);
    const cudaStream_t st = (cudaStream_t)stream;
    return a->type == B200_TYPE_F32 ? launch_store<float>(s, vec, grid, st) : a->type == B200_TYPE_F16 ? launch_store<__half>(s, vec, grid, st) : launch_store<__nv_bfloat16>(s, vec, grid, st);
}

int b200_op_kv8_load(const b200_kv8_load_args *a, b200_stream_t stream) {
    const char *who = "b200_op_kv8_load";
    OPX_REQUIRE(a, B200_ERR_INVALID, "%s: NULL arguments", who);
    const int rc = check_step(&a->cache, a->seq_info, a->table, a->table_stride, a->n_rows, a->n_seq, a->n_tokens, a->type, who);
    if (rc != B200_OK) return rc;
    if (a->n_tokens == 0 || a->n_seq == 0 || (!a->k && !a->v)) return B200_OK;
    const b200_kv8_cache &c = a->cache;
    OPX_REQUIRE((!a->k || a->k_stride >= (int64_t)c.n_head_kv * c.dim) && (!a->v || a->v_stride >= (int64_t)c.n_head_kv * c.vdim), B200_ERR_INVALID, "%s: rows of k or v overlap (strides %lld, %lld)",
                who, (long long)a->k_stride, (long long)a->v_stride);
    OPX_REQUIRE(aligned_to(type_size(a->type), a->k, a->v), B200_ERR_INVALID, "%s: k or v is not aligned to its type", who);
    const LoadArgs s = {c, {a->seq_info, a->table, a->table_stride, a->n_rows, a->n_seq, a->n_tokens, c.n_pages, c.page_size}, a->k, a->v, a->k_stride, a->v_stride};
    const bool vec = (!a->k || rows_aligned(a->k, a->k_stride, a->type)) && (!a->v || rows_aligned(a->v, a->v_stride, a->type));
    const unsigned grid = (unsigned)a->n_tokens;
    const cudaStream_t st = (cudaStream_t)stream;
    return a->type == B200_TYPE_F32 ? launch_load<float>(s, vec, grid, st) : a->type == B200_TYPE_F16 ? launch_load<__half>(s, vec, grid, st) : launch_load<__nv_bfloat16>(s, vec, grid, st);
}

int b200_op_kv8_cut(const b200_kv8_map *m, const int32_t *rows, const int32_t *keep, int32_t n, b200_stream_t stream) {
    const char *who = "b200_op_kv8_cut";
    int rc = check_map(m, who);
    if (rc == B200_OK) rc = check_list(n, who);
    if (rc != B200_OK || n == 0) return rc;
    OPX_REQUIRE(rows, B200_ERR_INVALID, "%s: NULL rows", who);
    B200_CUDA_TRY(launch_chained(kv8_cut_kernel, (unsigned)n, 128, 0, (cudaStream_t)stream, map_of(m), rows, keep));
    return B200_OK;
}

int b200_op_kv8_fork(const b200_kv8_map *m, const int32_t *src, const int32_t *dst, int32_t n, int32_t *refused, b200_stream_t stream) {
    const char *who = "b200_op_kv8_fork";
    int rc = check_map(m, who);
    if (rc == B200_OK) rc = check_list(n, who);
    if (rc != B200_OK || n == 0) return rc;
    OPX_REQUIRE(src && dst, B200_ERR_INVALID, "%s: NULL src or dst", who);
    B200_CUDA_TRY(launch_chained(kv8_fork_kernel, (unsigned)n, 128, 0, (cudaStream_t)stream, map_of(m), src, dst, (int)n, refused));
    return B200_OK;
}

size_t b200_kv8_grow_workspace_bytes(int32_t n) { return n > 0 ? (size_t)n * 8 : 0; }

int b200_op_kv8_grow(const b200_kv8_map *m, const b200_kv8_cache *caches, int32_t n_caches, const int32_t *rows, const int32_t *n_new, int32_t n, int32_t *seq_info, int32_t *refused,
                     void *workspace, size_t workspace_bytes, b200_stream_t stream) {
    const char *who = "b200_op_kv8_grow";
    int rc = check_map(m, who);
    if (rc == B200_OK) rc = check_list(n, who);
    if (rc == B200_OK) rc = check_caches(caches, n_caches, m->n_pages, m->page_size, who);
    if (rc != B200_OK || n == 0) return rc;
    OPX_REQUIRE(rows && n_new, B200_ERR_INVALID, "%s: NULL rows or n_new", who);
    OPX_REQUIRE(workspace && workspace_bytes >= b200_kv8_grow_workspace_bytes(n) && (uintptr_t)workspace % 8 == 0, B200_ERR_INVALID, "%s: workspace of %zu bytes, 8-byte aligned", who,
                b200_kv8_grow_workspace_bytes(n));
    int32_t *pairs = (int32_t *)workspace;
    B200_CUDA_TRY(launch_chained(kv8_grow_kernel, 1, 1024, 0, (cudaStream_t)stream, map_of(m), rows, n_new, (int)n, seq_info, refused, pairs));
    return launch_copies(caches, n_caches, pairs, pairs + 1, 2, n, m->n_pages, (cudaStream_t)stream);
}

static size_t compact_layout(int32_t n_pages, Compact *w, void *workspace) {
    const size_t stretches = ((size_t)n_pages + CM_STRETCH - 1) / CM_STRETCH, half = (size_t)n_pages / 2 + 1;
    int32_t *p = (int32_t *)workspace;
    if (w) *w = {p, p + 4, p + 4 + stretches, p + 4 + stretches + half, p + 4 + stretches + 2 * half};
    return 4 * (4 + stretches + 2 * half + (size_t)n_pages);
}
size_t b200_kv8_compact_workspace_bytes(int32_t n_pages) { return n_pages > 0 ? compact_layout(n_pages, nullptr, nullptr) : 0; }

int b200_op_kv8_compact(const b200_kv8_map *m, const b200_kv8_cache *caches, int32_t n_caches, int32_t *n_live, void *workspace, size_t workspace_bytes, b200_stream_t stream) {
    const char *who = "b200_op_kv8_compact";
    int rc = check_map(m, who);
    if (rc == B200_OK) rc = check_caches(caches, n_caches, m->n_pages, m->page_size, who);
    if (rc != B200_OK) return rc;
    OPX_REQUIRE(workspace && workspace_bytes >= b200_kv8_compact_workspace_bytes(m->n_pages) && (uintptr_t)workspace % 4 == 0, B200_ERR_INVALID, "%s: workspace of %zu bytes, 4-byte aligned", who,
                b200_kv8_compact_workspace_bytes(m->n_pages));
    Compact w;
    compact_layout(m->n_pages, &w, workspace);
    const cudaStream_t st = (cudaStream_t)stream;
    const unsigned stretches = (unsigned)((m->n_pages + CM_STRETCH - 1) / CM_STRETCH);
    const int32_t *refs = m->refs;
    B200_CUDA_TRY(launch_chained(kv8_count_kernel, stretches, CM_THREADS, 0, st, refs, (int)m->n_pages, w.counts));
    B200_CUDA_TRY(launch_chained(kv8_rank_kernel, stretches, CM_THREADS, 0, st, refs, (int)m->n_pages, w, n_live));
    int at = 0;
    do {
        Records r = {};
        const int k = take_records(r, caches, at, n_caches);
        at += k;
        B200_CUDA_TRY(launch_chained(kv8_move_kernel, (unsigned)(8 * sm_count()), CM_THREADS, 0, st, r, k, map_of(m), w, at >= n_caches));
    } while (at < n_caches);
    return B200_OK;
}

int b200_op_kv8_copy_pages(const b200_kv8_cache *caches, int32_t n_caches, const int32_t *src, const int32_t *dst, int32_t n, b200_stream_t stream) {
    const char *who = "b200_op_kv8_copy_pages";
    OPX_REQUIRE(n >= 0, B200_ERR_INVALID, "%s: %d pairs", who, n);
    int32_t n_pages = 0x7fffffff;
    for (int i = 0; caches && i < n_caches; i++) n_pages = caches[i].n_pages < n_pages ? caches[i].n_pages : n_pages;
    const int rc = check_caches(caches, n_caches, 0, 0, who);
    if (rc != B200_OK || n == 0 || n_caches == 0) return rc;
    OPX_REQUIRE(src && dst, B200_ERR_INVALID, "%s: NULL src or dst", who);
    return launch_copies(caches, n_caches, src, dst, 1, n, n_pages, (cudaStream_t)stream);
}

}  // extern "C"
