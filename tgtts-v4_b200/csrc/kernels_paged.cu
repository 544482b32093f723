// A paged batch's bookkeeping and elementwise kernels: page_plan (block tables and slot maps from
// request lengths), rope_pages (rotary embedding with the append of keys and values into pages) and
// logits_pick (penalties, biases and grammar masks on logits, with the greedy choice). All three are
// bound by memory or by their launch: one launch each, every input read once from HBM.
#include <cooperative_groups.h>

#include <type_traits>

#include "tg_common.cuh"
#include "tg_internal.h"

namespace tg {

namespace {

constexpr uint32_t SPARE = TG_SPARE;

// Division by a number the host knows: n / d = (mulhi(n, mul) + n) >> shift for every 32-bit n
// (Granlund and Montgomery, "Division by invariant integers using multiplication").
struct Divisor {
    uint32_t d, mul, shift;
    explicit Divisor(uint32_t by) : d(by), shift(0) {
        while ((1ull << shift) < by) shift++;
        mul = (uint32_t)(((1ull << 32) * ((1ull << shift) - by)) / by + 1);
    }
    TG_DEVICE uint32_t div(uint32_t n) const { return (uint32_t)(((uint64_t)__umulhi(n, mul) + n) >> shift); }
};

// ---- page_plan -------------------------------------------------------------------------------------
// With o_s = ceil(held / page) and w_s = ceil((held + fresh) / page) - o_s, request s's rows start at
// sum_{t < s} fresh_t and its new pages at free[sum_{t < s} w_t]. Every block takes both sums over
// all requests into shared memory (a block-wide scan: seqs x 8 bytes from L2, so that the blocks
// need nothing of one another), then writes its share of the rows, of the new table entries and of
// the requests' words; a row finds its request by bisection of the sums. All requests up to the first
// one that does not fit are served, so the sums over served requests are the sums over all.
// Latency-bound: a load of the requests' words (all in flight at once), the scan, the bisection and a row's load of
// its page's number follow one another. 2048 requests with 82,000 rows: 7.4 us of a run of launches (twice as many
// blocks 8.5, a quarter 9.5: they read the same words); 8 requests 3.0, about an empty launch.
constexpr int PLAN_THREADS = 512;
constexpr int PLAN_ROWS = 1024;  // rows a block, up to PLAN_BLOCKS blocks
constexpr uint32_t PLAN_BLOCKS = 148;

TG_DEVICE uint64_t warp_scan(uint64_t v) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint64_t u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
    }
    return v;
}

// The last of n ascending sums that is at most `x` (sums[0] = 0).
TG_DEVICE uint32_t find_sum(const uint32_t *sums, uint32_t n, uint32_t x) {
    uint32_t lo = 0, hi = n;
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if (sums[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

__global__ void __launch_bounds__(PLAN_THREADS)
    page_plan_kernel(tg_params p, Divisor by_page, const uint32_t *__restrict__ held, const uint32_t *__restrict__ fresh,
                     const uint32_t *__restrict__ free, uint32_t *table, uint32_t *__restrict__ at,
                     uint32_t *__restrict__ place, uint32_t *__restrict__ starts, uint32_t *__restrict__ next,
                     uint32_t *__restrict__ counts, uint32_t *err) {
    extern __shared__ uint32_t plan_smem[];
    uint32_t *row0 = plan_smem, *page0 = plan_smem + p.seqs + 1, *held_s = page0 + p.seqs + 1;
    constexpr int WARPS = PLAN_THREADS / 32;
    __shared__ uint64_t warp_rows[WARPS], warp_pages[WARPS];
    __shared__ uint32_t first_bad;
    const uint32_t n = p.seqs, page = p.capacity, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid == 0) first_bad = n;
    pdl_launch_dependents();
    pdl_wait();
    // All loads of the requests' words at once; row0 holds fresh until the sums take its place.
#pragma unroll 4
    for (uint32_t s = tid; s < n; s += PLAN_THREADS) {
        held_s[s] = held[s];
        row0[s] = fresh[s];
    }
    __syncthreads();
    const uint32_t each = (n + PLAN_THREADS - 1) / PLAN_THREADS, s0 = min(n, tid * each), s1 = min(n, s0 + each);
    auto pages_of = [page, by_page](uint64_t positions) {
        if (positions > SPARE) return (positions + page - 1) / page;
        return (uint64_t)(positions ? by_page.div((uint32_t)positions - 1) + 1 : 0);
    };
    uint64_t rows = 0, pages = 0;
    for (uint32_t s = s0; s < s1; s++) {
        const uint64_t h = held_s[s], f = row0[s];
        rows += f;
        pages += pages_of(h + f) - pages_of(h);
    }
    uint64_t r = warp_scan(rows), g = warp_scan(pages);
    if (lane == 31) {
        warp_rows[warp] = r;
        warp_pages[warp] = g;
    }
    __syncthreads();
    uint64_t all_pages = 0;
#pragma unroll
    for (uint32_t w = 0; w < WARPS; w++) {
        if (w < warp) {
            r += warp_rows[w];
            g += warp_pages[w];
        }
        all_pages += warp_pages[w];
    }
    r -= rows;
    g -= pages;
    for (uint32_t s = s0; s < s1; s++) {
        const uint64_t h = held_s[s], f = row0[s], w = pages_of(h + f) - pages_of(h);
        row0[s] = (uint32_t)min(r, (uint64_t)SPARE);
        page0[s] = (uint32_t)min(g, (uint64_t)SPARE);
        r += f;
        g += w;
        if (r > p.rows || g > p.n || pages_of(h + f) > p.stride || p.first + h + f >= SPARE) {
            atomicMin(&first_bad, s);
            break;  // the ones behind it are not served either
        }
        if (s == n - 1) {
            row0[n] = (uint32_t)r;
            page0[n] = (uint32_t)g;
        }
    }
    __syncthreads();
    const uint32_t served = first_bad, total = row0[served], taken = page0[served];
    const uint32_t stride = gridDim.x * PLAN_THREADS, t0 = blockIdx.x * PLAN_THREADS + tid;
    bool bad = false;
    for (uint32_t i = t0; i < p.rows; i += stride) {
        uint32_t pos = SPARE, seq = SPARE, to = SPARE;
        if (i < total) {
            seq = find_sum(row0, served, i);
            const uint32_t h = held_s[seq], at_own = h + (i - row0[seq]), j = by_page.div(at_own), old = (uint32_t)pages_of(h);
            const uint32_t id = j < old ? table[(size_t)seq * p.stride + j] : free[page0[seq] + (j - old)];
            pos = p.first + at_own;
            if (id < p.slots) to = id * page + (at_own - j * page);
            else bad = true;
        }
        at[i] = pos;
        at[p.rows + i] = seq;
        place[i] = to;
    }
    for (uint32_t i = t0; i < taken; i += stride) {
        const uint32_t seq = find_sum(page0, served, i);
        table[(size_t)seq * p.stride + (uint32_t)pages_of(held_s[seq]) + (i - page0[seq])] = free[i];
    }
    for (uint32_t s = t0; s < n; s += stride) {
        starts[s] = s < served ? row0[s] : total;
        next[s] = s < served ? held_s[s] + fresh[s] : held_s[s];
    }
    if (t0 == 0) {
        starts[n] = total;
        counts[0] = taken;
        counts[1] = total;
        counts[2] = served;
        counts[3] = (uint32_t)min(all_pages, (uint64_t)SPARE);
    }
    if (bad) atomicExch(err, ERR_BAD_INDEX);
}

// ---- rope_pages ------------------------------------------------------------------------------------
// A pair (a, b) of a head at a row's position turns by its table's angle: a cos - b sin, b cos + a sin
// (rope_rows' products and their order, so the same bits for the half layout over the whole head).
// HBM-bound: c is read once, q and the pages written once; the tables' rows come from L2.

// Four consecutive values as f32.
template <typename C>
TG_DEVICE float4 load4(const C *p);
template <>
TG_DEVICE float4 load4<float>(const float *p) { return __ldcs(reinterpret_cast<const float4 *>(p)); }
template <>
TG_DEVICE float4 load4<bf16>(const bf16 *p) {
    const uint2 r = __ldcs(reinterpret_cast<const uint2 *>(p));
    return make_float4(__uint_as_float(r.x << 16), __uint_as_float(r.x & 0xffff0000u), __uint_as_float(r.y << 16),
                       __uint_as_float(r.y & 0xffff0000u));
}
TG_DEVICE void put4(float *o, float4 v) { *reinterpret_cast<float4 *>(o) = v; }
TG_DEVICE void put4(bf16 *o, float4 v) {
    const __nv_bfloat162 lo = __floats2bfloat162_rn(v.x, v.y), hi = __floats2bfloat162_rn(v.z, v.w);
    *reinterpret_cast<uint2 *>(o) =
        make_uint2(*reinterpret_cast<const uint32_t *>(&lo), *reinterpret_cast<const uint32_t *>(&hi));
}
// Two consecutive values, at an even place.
template <typename C>
TG_DEVICE float2 load2(const C *p);
template <>
TG_DEVICE float2 load2<float>(const float *p) { return __ldcs(reinterpret_cast<const float2 *>(p)); }
template <>
TG_DEVICE float2 load2<bf16>(const bf16 *p) {
    const uint32_t r = __ldcs(reinterpret_cast<const uint32_t *>(p));
    return make_float2(__uint_as_float(r << 16), __uint_as_float(r & 0xffff0000u));
}
TG_DEVICE void put2(float *o, float2 v) { *reinterpret_cast<float2 *>(o) = v; }
TG_DEVICE void put2(bf16 *o, float2 v) { *reinterpret_cast<__nv_bfloat162 *>(o) = __floats2bfloat162_rn(v.x, v.y); }
TG_DEVICE void turn(float &a, float &b, float co, float si) {
    const float na = __fmaf_rn(a, co, -__fmul_rn(b, si));
    b = __fmaf_rn(b, co, __fmul_rn(a, si));
    a = na;
}

// False for a row that writes nothing.
TG_DEVICE bool rope_row(const tg_params &p, uint32_t pos, uint32_t to, uint32_t *err) {
    if (pos == SPARE) return false;
    if ((p.rope && pos >= p.n) || (to != SPARE && to >= p.slots * p.capacity)) {
        atomicExch(err, ERR_BAD_INDEX);
        return false;
    }
    return true;
}

// For a rotated part that is a multiple of 8: a thread takes eight dimensions of two heads (h and h + half the heads,
// which turn by the same angles), rotated ones as four pairs (in the half layout two runs of four, each a warp's
// whole sectors), of every gridDim-th group of rows: where they lie in a row is worked out once. All of a
// row's loads of c leave before it is known whether the row is spare. 32768 rows of 20 heads of 64, f32 to bf16 (253
// MB): 46.4 us, 5.4 TB/s; 2047 rows of 48 heads of 128 (50 MB, not in L2): 13.9 us, 3.7 TB/s.
constexpr int ROPE_THREADS = 256;

template <typename T, typename C, bool INTER, int HD>
__global__ void __launch_bounds__(ROPE_THREADS)
    rope_pages_kernel(tg_params p, Divisor page, uint32_t units, uint32_t row_units, uint32_t block_rows,
                      const uint32_t *__restrict__ at, const uint32_t *__restrict__ place, const C *__restrict__ c,
                      const float *__restrict__ cosv, const float *__restrict__ sinv, T *__restrict__ q, T *__restrict__ k,
                      T *__restrict__ v, uint32_t *err) {
    // A block's `units` threads of a row, from unit blockIdx.y x units on, times block_rows rows.
    const uint32_t heads = p.heads + 2 * p.kv_heads, apart = (heads + 1) / 2, half = p.k / 2;
    const uint32_t sub = threadIdx.x / units, unit = blockIdx.y * units + threadIdx.x % units;
    const uint32_t head0 = unit / (HD / 8), head1 = head0 + apart, u = unit % (HD / 8);
    const bool here[2] = {unit < row_units, unit < row_units && head1 < heads};
    const bool rotated = p.rope && u < p.k / 8;
    const bool turned[2] = {rotated && head0 < p.heads + p.kv_heads, rotated && head1 < p.heads + p.kv_heads};
    uint32_t d0[2], d1[2];
#pragma unroll
    for (int n = 0; n < 2; n++) {
        d0[n] = (turned[n] && !INTER) ? 4 * u : 8 * u;
        d1[n] = (turned[n] && !INTER) ? half + 4 * u : 8 * u + 4;
    }
    const C *x[2] = {c + (size_t)head0 * HD, c + (size_t)head1 * HD};
    const size_t row_values = (size_t)heads * HD;
    pdl_launch_dependents();
    pdl_wait();
    const uint32_t step = gridDim.x * block_rows;
    for (uint32_t row = blockIdx.x * block_rows + sub; row < p.rows; row += step) {
        float4 a[2], b[2];
#pragma unroll
        for (int n = 0; n < 2; n++) {
            if (!here[n]) continue;
            a[n] = load4(x[n] + row * row_values + d0[n]);
            b[n] = load4(x[n] + row * row_values + d1[n]);
        }
        const uint32_t pos = at[row], to = place[row];
        if (!rope_row(p, pos, to, err)) continue;
        const uint32_t id = page.div(to), off = to - id * p.capacity;
        float4 co, si;
        if (turned[0] || turned[1]) {
            co = __ldg(reinterpret_cast<const float4 *>(cosv + (size_t)pos * half) + u);
            si = __ldg(reinterpret_cast<const float4 *>(sinv + (size_t)pos * half) + u);
        }
#pragma unroll
        for (int n = 0; n < 2; n++) {
            const uint32_t head = n ? head1 : head0;
            if (!here[n] || (head >= p.heads && to == SPARE)) continue;
            const bool value = head >= p.heads + p.kv_heads;
            T *o = head < p.heads
                       ? q + ((size_t)row * p.heads + head) * HD
                       : (value ? v : k) + (((size_t)id * p.kv_heads + (head - p.heads - (value ? p.kv_heads : 0))) * p.capacity + off) * HD;
            if (turned[n]) {
                if (INTER) {
                    turn(a[n].x, a[n].y, co.x, si.x);
                    turn(a[n].z, a[n].w, co.y, si.y);
                    turn(b[n].x, b[n].y, co.z, si.z);
                    turn(b[n].z, b[n].w, co.w, si.w);
                } else {
                    turn(a[n].x, b[n].x, co.x, si.x);
                    turn(a[n].y, b[n].y, co.y, si.y);
                    turn(a[n].z, b[n].z, co.z, si.z);
                    turn(a[n].w, b[n].w, co.w, si.w);
                }
            }
            put4(o + d0[n], a[n]);
            put4(o + d1[n], b[n]);
        }
    }
}

// Any other even rotated part, where fours of the two halves or of the tables' rows do not lie on 16 bytes: a thread takes
// pair u of ROPE_PAIRS heads (apart by a ROPE_PAIRS-th of the heads), in the same order of rows. 2047 rows of 48 heads of 128, 100 turned:
// 33 us (4 heads 37, 8 45), against 14 where a thread takes eight dimensions: the few bytes of a thread's loads in
// flight bound it.
constexpr int ROPE_PAIRS = 2;

template <typename T, typename C>
__global__ void __launch_bounds__(ROPE_THREADS)
    rope_pages_any_kernel(tg_params p, Divisor page, uint32_t units, uint32_t row_units, uint32_t block_rows,
                          const uint32_t *__restrict__ at, const uint32_t *__restrict__ place, const C *__restrict__ c,
                          const float *__restrict__ cosv, const float *__restrict__ sinv, T *__restrict__ q, T *__restrict__ k,
                          T *__restrict__ v, uint32_t *err) {
    const uint32_t hd = p.head_dim, heads = p.heads + 2 * p.kv_heads, apart = (heads + ROPE_PAIRS - 1) / ROPE_PAIRS, half = p.k / 2;
    const uint32_t sub = threadIdx.x / units, unit = blockIdx.y * units + threadIdx.x % units;
    const uint32_t head0 = unit / (hd / 2), u = unit % (hd / 2);
    const bool rotated = p.rope && u < half;
    // Of each head: where its first value lies in a row of c, where its pair's do in q's row or a page's position, and
    // the pair: dimensions 2 u and 2 u + 1, or u and u + half of a head that turns in the half layout.
    const C *x[ROPE_PAIRS];
    T *o[ROPE_PAIRS];
    bool here[ROPE_PAIRS], paged[ROPE_PAIRS], turned[ROPE_PAIRS], halves[ROPE_PAIRS];
#pragma unroll
    for (int n = 0; n < ROPE_PAIRS; n++) {
        const uint32_t head = head0 + n * apart;
        here[n] = unit < row_units && head < heads;
        paged[n] = head >= p.heads;
        turned[n] = rotated && head < p.heads + p.kv_heads;
        halves[n] = turned[n] && !(p.flags & 1);
        const uint32_t in = halves[n] ? u : 2 * u;
        x[n] = c + (size_t)head * hd + in;
        T *cache = head < p.heads + p.kv_heads ? k + (size_t)(head - p.heads) * p.capacity * hd
                                               : v + (size_t)(head - p.heads - p.kv_heads) * p.capacity * hd;
        o[n] = (paged[n] ? cache : q + (size_t)head * hd) + in;
    }
    pdl_launch_dependents();
    pdl_wait();
    const size_t row_values = (size_t)heads * hd, row_q = (size_t)p.heads * hd, page_values = (size_t)p.kv_heads * p.capacity * hd;
    const uint32_t step = gridDim.x * block_rows;
    for (uint32_t row = blockIdx.x * block_rows + sub; row < p.rows; row += step) {
        float a[ROPE_PAIRS], b[ROPE_PAIRS];
#pragma unroll
        for (int n = 0; n < ROPE_PAIRS; n++) {
            if (!here[n]) continue;
            const C *from = x[n] + row * row_values;
            if (halves[n]) {
                a[n] = to_f32<C>(from[0]);
                b[n] = to_f32<C>(from[half]);
            } else {
                const float2 two = load2<C>(from);
                a[n] = two.x;
                b[n] = two.y;
            }
        }
        const uint32_t pos = at[row], to = place[row];
        if (!rope_row(p, pos, to, err)) continue;
        const float co = rotated ? __ldg(cosv + (size_t)pos * half + u) : 1.0f, si = rotated ? __ldg(sinv + (size_t)pos * half + u) : 0.0f;
        const uint32_t id = page.div(to);
        const size_t at_q = row * row_q, at_page = id * page_values + (size_t)(to - id * p.capacity) * hd;
#pragma unroll
        for (int n = 0; n < ROPE_PAIRS; n++) {
            if (!here[n] || (paged[n] && to == SPARE)) continue;
            T *out = o[n] + (paged[n] ? at_page : at_q);
            if (turned[n]) turn(a[n], b[n], co, si);
            if (halves[n]) {
                out[0] = from_f32<T>(a[n]);
                out[half] = from_f32<T>(b[n]);
            } else
                put2(out, make_float2(a[n], b[n]));
        }
    }
}

// ---- logits_pick -----------------------------------------------------------------------------------
// A cluster of blocks to a row, every ranks-th tile of PICK_TILE tokens to each (a history holds many low
// tokens: in ranges the first block had most of the counting). A block marks its touched tokens (in
// the history or the biases) in a bit map and numbers them by its running bit counts; their occurrences are
// added, and a token's last bias entry found, atomically on whole numbers, so that no order shows. The
// touched logits are then done a thread to a token, and the others pass through without a barrier, four
// or eight to a 16-byte load and store (one by one in rows that 16 bytes do not divide); the touched ones' values
// overwrite what the stream left. The row's greedy choice is joined over the cluster in distributed shared memory.
// HBM-bound where there are rows enough: each logit is read and written once. 128 rows of 128,000 tokens in f32
// (131 MB, not in L2): 28.3 us without controls, 4.6 TB/s; 38.5 us with histories of 4096 tokens and 64 biases, whose two
// passes come before the stream (under them the logits come into L2). One row of 32,000 with a history of 700: 6.2 us,
// the passes' latencies. Counting inside the stream, a table of counts to a tile, took twice the time for the 128 rows.
// A run in which more than PICK_TOUCHED different tokens are touched is cut to that many tokens, and the history is read
// again for each: 64 rows with histories to 20,000 52.5 us, to 4000 20.1.
constexpr int PICK_THREADS = 512;
constexpr uint32_t PICK_TILE = 1024, PICK_AHEAD = 64 * PICK_TILE;
constexpr uint32_t PICK_RUN = 65536;     // the most tokens whose bits are held at once
constexpr uint32_t PICK_TOUCHED = 4096;  // the most touched tokens whose words are held at once
constexpr size_t PICK_SMEM = (PICK_RUN / 32 + 2 * PICK_TOUCHED) * sizeof(uint32_t) + (PICK_TOUCHED + PICK_RUN / 32) * sizeof(uint16_t);
// A count word: the prompt holds the token; a bias names it; below, its generated occurrences.
constexpr uint32_t IN_PROMPT = 1u << 31, BIASED = 1u << 30;

struct Best {
    float value;
    uint32_t token;
};
TG_DEVICE void better(Best &a, float value, uint32_t token) {
    if (value > a.value || (value == a.value && token < a.token)) a = Best{value, token};
}

// VEC consecutive logits to one load: 16 bytes, or one logit for rows that are not 16-byte aligned.
template <typename T, int VEC>
__global__ void __launch_bounds__(PICK_THREADS, 2)
    logits_pick_kernel(tg_params p, const T *logits, const uint32_t *__restrict__ seen,
                       const uint32_t *__restrict__ spans, const float *__restrict__ penalties,
                       const uint32_t *__restrict__ bias_ids, const float *__restrict__ bias,
                       const uint32_t *__restrict__ masks, T *out, uint32_t *__restrict__ pick, uint32_t *err) {
    namespace cg = cooperative_groups;
    using Raw = typename std::conditional<VEC == 1, T, typename Vec<T>::Raw>::type;
    constexpr int EACH = VEC == 1 ? 8 : 4;  // loads of a thread in flight
    constexpr uint32_t STEP = PICK_THREADS * VEC * EACH, ALL = (1u << VEC) - 1;
    extern __shared__ __align__(16) uint32_t pick_smem[];
    uint32_t *touched = pick_smem, *count = touched + PICK_RUN / 32, *biased = count + PICK_TOUCHED;
    uint16_t *token = reinterpret_cast<uint16_t *>(biased + PICK_TOUCHED);  // the touched tokens in order
    uint16_t *before = reinterpret_cast<uint16_t *>(token + PICK_TOUCHED);
    __shared__ Best warp_best[PICK_THREADS / 32], block_best[8];  // the first block's: of every block
    __shared__ uint32_t warp_bits[PICK_THREADS / 32];
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, ranks = cluster.num_blocks(), rank = cluster.block_rank();
    const uint32_t row = blockIdx.x / ranks, n = p.n;
    cluster.sync();  // every block has started before its shared memory is written
    pdl_launch_dependents();
    pdl_wait();
    const uint32_t *span = spans + (size_t)row * 6;
    const uint32_t begin = span[0], prompt = span[1], made = span[2], bias0 = span[3], biases = span[4], mask = span[5];
    // The same words for the whole cluster: all of its blocks leave here, or none.
    if ((uint64_t)begin + prompt + made > p.k || (uint64_t)bias0 + biases > p.k1 || (mask != SPARE && mask >= p.m)) {
        if (tid == 0 && rank == 0) atomicExch(err, ERR_BAD_INDEX);
        return;
    }
    const uint32_t history = prompt + made;
    const float repetition = penalties[(size_t)row * 3], presence = penalties[(size_t)row * 3 + 1], frequency = penalties[(size_t)row * 3 + 2];
    const uint32_t *bits = mask == SPARE ? nullptr : masks + (size_t)mask * ((n + 31) / 32);
    const T *x = logits + (size_t)row * p.stride;
    T *y = out + (size_t)row * p.stride;
    Best best{-INFINITY, SPARE}, other{-INFINITY, SPARE};  // of the untouched tokens, and of the touched ones
    const bool controls = history || biases;
    const uint32_t rank_bits = 31 - __clz(ranks);  // ranks is a power of two
    // The block's tokens in ascending order, as numbers l of its own: the token of l, and a token's l (none: past all).
    const uint32_t tiles = (n + PICK_TILE - 1) / PICK_TILE, mine = tiles > rank ? (tiles - rank + ranks - 1) / ranks * PICK_TILE : 0;
    auto token_of = [&](uint32_t l) { return (l / PICK_TILE * ranks + rank) * PICK_TILE + l % PICK_TILE; };
    auto local_of = [&](uint32_t t) {
        const uint32_t tile = t / PICK_TILE;
        return t < n && (tile & (ranks - 1)) == rank ? (tile >> rank_bits) * PICK_TILE + t % PICK_TILE : SPARE;
    };
    constexpr int H = 8;  // entries of a thread in flight
    auto history_at = [&](uint32_t i0, uint32_t(&e)[H]) {
#pragma unroll
        for (int h = 0; h < H; h++) e[h] = i0 + h * PICK_THREADS < history ? __ldg(seen + begin + i0 + h * PICK_THREADS) : SPARE;
    };
    for (uint32_t l0 = 0, end; l0 < mine; l0 = end) {
        end = min(mine, l0 + PICK_RUN);
        Raw raw[EACH];
        auto load = [&](uint32_t at) {
#pragma unroll
            for (int j = 0; j < EACH; j++) {
                const uint32_t t = token_of(at + (j * PICK_THREADS + tid) * VEC);
                if (t + VEC <= n) raw[j] = __ldcs(reinterpret_cast<const Raw *>(x + t));
            }
        };
        uint32_t total = 0;  // touched tokens
        auto allow = [&](uint32_t t) { return bits ? __ldg(bits + t / 32) >> (t % 32) : 0xffffffffu; };
        auto hits = [&](uint32_t in) { return controls ? touched[in / 32] >> (in % 32) & ALL : 0u; };
        if (controls) {
            // A thread's first entries stay with it for both passes; a token past the vocabulary where there is none.
            uint32_t first_entries[H];
            history_at(tid, first_entries);
            const uint32_t first_bias = tid < biases ? __ldg(bias_ids + bias0 + tid) : SPARE;
            auto entries = [&](auto in_history, auto in_biases) {
                auto all = [&](const uint32_t(&e)[H], uint32_t i0) {
#pragma unroll
                    for (int h = 0; h < H; h++) {
                        const uint32_t in = local_of(e[h]) - l0;
                        if (in < end - l0) in_history(in, i0 + h * PICK_THREADS);
                    }
                };
                all(first_entries, tid);
                for (uint32_t i0 = tid + PICK_THREADS * H; i0 < history; i0 += PICK_THREADS * H) {
                    uint32_t e[H];
                    history_at(i0, e);
                    all(e, i0);
                }
                for (uint32_t i = tid; i < biases; i += PICK_THREADS) {
                    const uint32_t in = local_of(i == tid ? first_bias : bias_ids[bias0 + i]) - l0;
                    if (in < end - l0) in_biases(in, i);
                }
            };
            constexpr uint32_t LINE = 128 / sizeof(T);
            constexpr uint32_t W = PICK_RUN / 32 / PICK_THREADS;  // words of the bit map to a thread
            uint32_t upto, marks[W];
            while (true) {
                __syncthreads();  // the run before is done with the words
#pragma unroll
                for (uint32_t i = 0; i < W; i++) touched[tid + i * PICK_THREADS] = 0;
                __syncthreads();
                auto touch = [&](uint32_t in, uint32_t) {
                    if (!(touched[in / 32] >> (in % 32) & 1)) atomicOr(touched + in / 32, 1u << (in % 32));
                };
                entries(touch, touch);
                // The history is here: while it is counted the run's first logits come into L2. (Before it, their traffic
                // held it up.)
                for (uint32_t l = l0 + tid * LINE; l < min(end, l0 + PICK_AHEAD); l += PICK_THREADS * LINE)
                    if (token_of(l) < n) asm volatile("prefetch.global.L2 [%0];" ::"l"(x + token_of(l)) : "memory");
                __syncthreads();
                uint32_t sum = 0;
#pragma unroll
                for (uint32_t i = 0; i < W; i++) {
                    marks[i] = touched[tid * W + i];
                    sum += __popc(marks[i]);
                }
                upto = sum;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const uint32_t u = __shfl_up_sync(0xffffffffu, upto, o);
                    if (lane >= (uint32_t)o) upto += u;
                }
                if (lane == 31) warp_bits[warp] = upto;
                __syncthreads();
                total = 0;
                for (uint32_t w = 0; w < PICK_THREADS / 32; w++) {
                    if (w < warp) upto += warp_bits[w];
                    total += warp_bits[w];
                }
                upto -= sum;
                if (total <= PICK_TOUCHED) break;
                end = l0 + PICK_TOUCHED;  // of so many tokens no more can be touched
            }
#pragma unroll
            for (uint32_t i = 0; i < W; i++) {
                before[tid * W + i] = upto;
                upto += __popc(marks[i]);
            }
            for (uint32_t i = tid; i < total; i += PICK_THREADS) count[i] = biased[i] = 0;
            __syncthreads();
            // (The entries of a token all write the same number of it.)
            auto add = [&](uint32_t in, uint32_t i, uint32_t first) {
                const uint32_t at = before[in / 32] + __popc(touched[in / 32] & ((1u << (in % 32)) - 1));
                if (first == 1) atomicAdd(count + at, 1u);
                else atomicOr(count + at, first);
                if (first == BIASED) atomicMax(biased + at, i + 1);
                token[at] = (uint16_t)in;
            };
            entries([&](uint32_t in, uint32_t i) { add(in, i, i < prompt ? IN_PROMPT : 1u); }, [&](uint32_t in, uint32_t i) { add(in, i, BIASED); });
            __syncthreads();
            constexpr int F = 4;  // touched logits of a thread in flight
            for (uint32_t i0 = tid; i0 < total; i0 += PICK_THREADS * F) {
                T value[F];
                uint32_t all[F];
#pragma unroll
                for (int k = 0; k < F; k++) {
                    const uint32_t i = i0 + k * PICK_THREADS;
                    if (i >= total) continue;
                    const uint32_t t = token_of(l0 + token[i]);
                    value[k] = x[t];
                    all[k] = allow(t);
                }
#pragma unroll
                for (int k = 0; k < F; k++) {
                    const uint32_t i = i0 + k * PICK_THREADS;
                    if (i >= total) continue;
                    const uint32_t t = token_of(l0 + token[i]), c = count[i], b = biased[i], made = c & (BIASED - 1);
                    float f = to_f32<T>(value[k]);
                    if (c & ~BIASED) {
                        f = f > 0.0f ? __fdiv_rn(f, repetition) : f * repetition;
                        f = f - (float)made * frequency;
                        if (made) f = f - presence;
                    }
                    if (b) f = f + bias[bias0 + b - 1];
                    const float stored = to_f32<T>(from_f32<T>(all[k] & 1 ? f : -INFINITY));
                    biased[i] = __float_as_uint(stored);  // stored behind the stream
                    if (stored > -INFINITY) better(other, stored, t);
                }
            }
        }
        // The stream: logits masked, stored and, untouched ones, compared with the best so far. A thread meets its
        // tokens in ascending order, so that the first of equal values stays.
        for (uint32_t at = l0; at < end; at += STEP) {
            load(at);
#pragma unroll
            for (int j = 0; j < EACH; j++) {
                const uint32_t l = at + (j * PICK_THREADS + tid) * VEC, t = token_of(l);
                if (l >= end || t + VEC > n) break;
                const uint32_t hit = hits(l - l0), allowed = allow(t) & ALL;
                __align__(16) T value[VEC];
                *reinterpret_cast<Raw *>(value) = raw[j];
                if (allowed != ALL)
#pragma unroll
                    for (int e = 0; e < VEC; e++) value[e] = allowed >> e & 1 ? value[e] : from_f32<T>(-INFINITY);
                __stcs(reinterpret_cast<Raw *>(y + t), *reinterpret_cast<const Raw *>(value));
                if (hit)
#pragma unroll
                    for (int e = 0; e < VEC; e++) value[e] = hit >> e & 1 ? from_f32<T>(-INFINITY) : value[e];
#pragma unroll
                for (int e = 0; e < VEC; e++)
                    if (to_f32<T>(value[e]) > best.value) best = Best{to_f32<T>(value[e]), t + e};
            }
        }
        // The row's last tokens, past its whole vectors.
        if (VEC > 1 && tid < n % VEC) {
            const uint32_t t = n / VEC * VEC + tid, l = local_of(t);
            if (l >= l0 && l < end && !(hits(l - l0) & 1)) {
                const T value = allow(t) & 1 ? x[t] : from_f32<T>(-INFINITY);
                y[t] = value;
                if (to_f32<T>(value) > best.value) best = Best{to_f32<T>(value), t};
            }
        }
        if (controls) {
            __syncthreads();  // the touched tokens' logits over what the stream left there
            for (uint32_t i = tid; i < total; i += PICK_THREADS) y[token_of(l0 + token[i])] = from_f32<T>(__uint_as_float(biased[i]));
        }
    }
    better(best, other.value, other.token);
    auto warp_join = [&](Best v) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
            better(v, __shfl_xor_sync(0xffffffffu, v.value, o), __shfl_xor_sync(0xffffffffu, v.token, o));
        return v;
    };
    best = warp_join(best);
    if (lane == 0) warp_best[warp] = best;
    __syncthreads();
    if (warp == 0) {
        best = warp_join(lane < PICK_THREADS / 32 ? warp_best[lane] : Best{-INFINITY, SPARE});
        if (lane == 0) *cluster.map_shared_rank(block_best + rank, 0) = best;
    }
    cluster.sync();
    if (rank == 0 && warp == 0) {
        best = warp_join(lane < ranks ? block_best[lane] : Best{-INFINITY, SPARE});
        if (lane == 0) pick[row] = best.token;
    }
}

template <typename T, int VEC>
cudaError_t pick_t(const tg_params &p, const void *logits, const uint32_t *seen, const uint32_t *spans, const float *pen,
                   const uint32_t *ids, const float *bias, const uint32_t *masks, void *out, uint32_t *pick, uint32_t *err,
                   cudaStream_t s) {
    // Blocks of 1024 tokens at least; the most to a row that run at once (two an SM), up to eight. Of 128,000 tokens
    // with 8, 4 and 2 blocks a row: 1 row 6.8, 8.9, 13.0 us; 32 rows 10.8, 13.2, 18.5; 64 rows 20.3, 16.8, 21.9; 128
    // rows 39, 31, 28 (without controls; with histories to 4096 55, 42, 39).
    uint32_t ranks = p.rows <= 32 ? 8 : p.rows <= 64 ? 4 : 2;
    while (ranks > 1 && p.n <= ranks / 2 * PICK_TILE) ranks /= 2;
    cudaError_t e = with_smem(logits_pick_kernel<T, VEC>, PICK_SMEM);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(p.rows * ranks);
    cfg.blockDim = dim3(PICK_THREADS);
    cfg.dynamicSmemBytes = PICK_SMEM;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = ranks;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, logits_pick_kernel<T, VEC>, p, (const T *)logits, seen, spans, pen, ids, bias, masks,
                              (T *)out, pick, err);
}

template <typename T, typename C>
cudaError_t rope_t(const tg_params &p, const uint32_t *at, const uint32_t *place, const void *c, const float *cs,
                   const float *sn, void *q, void *k, void *v, uint32_t *err, cudaStream_t s) {
    const uint32_t heads = p.heads + 2 * p.kv_heads;
    const Divisor page(p.capacity);
    // A row's units over gridDim.y blocks of about equal width; as many rows to a block as fit; no more blocks than
    // four waves of four an SM (more rows to a thread then: 46.5 us for 32768 rows of 20 heads of 64; sixteen waves or a
    // thread a row 50.2 and 51.5, one wave 57.9).
    const bool eights = p.k % 8 == 0;
    const uint32_t row_units = eights ? (heads + 1) / 2 * (p.head_dim / 8) : (heads + ROPE_PAIRS - 1) / ROPE_PAIRS * (p.head_dim / 2), ny = (row_units + ROPE_THREADS - 1) / ROPE_THREADS;
    const uint32_t units = (row_units + ny - 1) / ny, block_rows = ROPE_THREADS / units;
    const uint32_t nx = min((p.rows + block_rows - 1) / block_rows, 4u * 4 * 148 / ny + 1);
    auto run = [&](auto kern) {
        return launch_pdl(kern, dim3(nx, ny), dim3(units * block_rows), 0, s, p, page, units, row_units, block_rows, at, place, (const C *)c, cs, sn,
                          (T *)q, (T *)k, (T *)v, err);
    };
    if (!eights) return run(rope_pages_any_kernel<T, C>);
    if (p.head_dim == 64) return p.flags & 1 ? run(rope_pages_kernel<T, C, true, 64>) : run(rope_pages_kernel<T, C, false, 64>);
    return p.flags & 1 ? run(rope_pages_kernel<T, C, true, 128>) : run(rope_pages_kernel<T, C, false, 128>);
}

}  // namespace

cudaError_t launch_page_plan(const tg_params &p, const uint32_t *held, const uint32_t *fresh, const uint32_t *free,
                             uint32_t *table, uint32_t *at, uint32_t *place, uint32_t *starts, uint32_t *next,
                             uint32_t *counts, uint32_t *err, cudaStream_t s) {
    const size_t smem = (3 * (size_t)p.seqs + 2) * sizeof(uint32_t);
    cudaError_t e = with_smem(page_plan_kernel, smem);
    if (e != cudaSuccess) return e;
    const uint32_t blocks = min((p.rows + PLAN_ROWS - 1) / PLAN_ROWS, PLAN_BLOCKS);
    return launch_pdl(page_plan_kernel, dim3(blocks), dim3(PLAN_THREADS), smem, s, p, Divisor(p.capacity), held, fresh, free, table, at, place,
                      starts, next, counts, err);
}

cudaError_t launch_rope_pages(const tg_params &p, const uint32_t *at, const uint32_t *place, const void *c,
                              const float *cs, const float *sn, void *q, void *k, void *v, uint32_t *err, cudaStream_t s) {
    const bool c16 = p.flags & 2;
    if (p.dtype == TG_BF16)
        return c16 ? rope_t<bf16, bf16>(p, at, place, c, cs, sn, q, k, v, err, s)
                   : rope_t<bf16, float>(p, at, place, c, cs, sn, q, k, v, err, s);
    return rope_t<float, float>(p, at, place, c, cs, sn, q, k, v, err, s);
}

cudaError_t launch_logits_pick(const tg_params &p, const void *logits, const uint32_t *seen, const uint32_t *spans,
                               const float *pen, const uint32_t *ids, const float *bias, const uint32_t *masks, void *out,
                               uint32_t *pick, uint32_t *err, cudaStream_t s) {
    if (p.dtype == TG_BF16)
        return p.stride % 8 ? pick_t<bf16, 1>(p, logits, seen, spans, pen, ids, bias, masks, out, pick, err, s)
                            : pick_t<bf16, 8>(p, logits, seen, spans, pen, ids, bias, masks, out, pick, err, s);
    return p.stride % 4 ? pick_t<float, 1>(p, logits, seen, spans, pen, ids, bias, masks, out, pick, err, s)
                        : pick_t<float, 4>(p, logits, seen, spans, pen, ids, bias, masks, out, pick, err, s);
}

}  // namespace tg
