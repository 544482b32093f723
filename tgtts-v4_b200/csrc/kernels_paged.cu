// A paged batch's bookkeeping and elementwise kernels: page_plan (block tables and slot maps from
// request lengths), rope_pages (rotary embedding with the append of keys and values into pages) and
// logits_pick (penalties, biases and grammar masks on logits, with the greedy choice). All three are
// bound by memory or by their launch: one launch each, every input read once from HBM.
#include <cooperative_groups.h>

#include "tg_common.cuh"
#include "tg_internal.h"

namespace tg {

namespace {

constexpr uint32_t SPARE = TG_SPARE;

// ---- page_plan -------------------------------------------------------------------------------------
// With o_s = ceil(held / page) and w_s = ceil((held + fresh) / page) - o_s, request s's rows start at
// sum_{t < s} fresh_t and its new pages at free[sum_{t < s} w_t]. Every block takes both sums over
// all requests into shared memory (a block-wide scan: seqs x 8 bytes from L2, so that the blocks
// need nothing of one another), then writes its share of the rows, of the new table entries and of
// the requests' words; a row finds its request by bisection of the sums. All requests up to the first
// one that does not fit are served, so the sums over served requests are the sums over all.
constexpr int PLAN_THREADS = 512;
constexpr int PLAN_ROWS = 2048;  // rows a block

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
    page_plan_kernel(tg_params p, const uint32_t *__restrict__ held, const uint32_t *__restrict__ fresh,
                     const uint32_t *__restrict__ free, uint32_t *table, uint32_t *__restrict__ at,
                     uint32_t *__restrict__ place, uint32_t *__restrict__ starts, uint32_t *__restrict__ next,
                     uint32_t *__restrict__ counts, uint32_t *err) {
    extern __shared__ uint32_t plan_smem[];
    uint32_t *row0 = plan_smem, *page0 = plan_smem + p.seqs + 1;
    __shared__ uint64_t warp_rows[32], warp_pages[32];
    __shared__ uint32_t first_bad;
    const uint32_t n = p.seqs, page = p.capacity, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid == 0) first_bad = n;
    pdl_launch_dependents();
    pdl_wait();
    const uint32_t each = (n + blockDim.x - 1) / blockDim.x, s0 = min(n, tid * each), s1 = min(n, s0 + each);
    auto pages_of = [page](uint64_t positions) { return (positions + page - 1) / page; };
    uint64_t rows = 0, pages = 0;
    for (uint32_t s = s0; s < s1; s++) {
        const uint64_t h = held[s], f = fresh[s];
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
    for (uint32_t w = 0; w < blockDim.x / 32; w++) {
        if (w < warp) {
            r += warp_rows[w];
            g += warp_pages[w];
        }
        all_pages += warp_pages[w];
    }
    r -= rows;
    g -= pages;
    for (uint32_t s = s0; s < s1; s++) {
        const uint64_t h = held[s], f = fresh[s], w = pages_of(h + f) - pages_of(h);
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
    const uint32_t stride = gridDim.x * blockDim.x, t0 = blockIdx.x * blockDim.x + tid;
    bool bad = false;
    for (uint32_t i = t0; i < p.rows; i += stride) {
        uint32_t pos = SPARE, seq = SPARE, to = SPARE;
        if (i < total) {
            seq = find_sum(row0, served, i);
            const uint32_t h = held[seq], at_own = h + (i - row0[seq]), j = at_own / page, old = (uint32_t)pages_of(h);
            const uint32_t id = j < old ? table[(size_t)seq * p.stride + j] : free[page0[seq] + (j - old)];
            pos = p.first + at_own;
            if (id < p.slots) to = id * page + at_own % page;
            else bad = true;
        }
        at[i] = pos;
        at[p.rows + i] = seq;
        place[i] = to;
    }
    for (uint32_t i = t0; i < taken; i += stride) {
        const uint32_t seq = find_sum(page0, served, i);
        table[(size_t)seq * p.stride + (uint32_t)pages_of(held[seq]) + (i - page0[seq])] = free[i];
    }
    for (uint32_t s = t0; s < n; s += stride) {
        starts[s] = s < served ? row0[s] : total;
        next[s] = s < served ? held[s] + fresh[s] : held[s];
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
TG_DEVICE void turn(float &a, float &b, float co, float si) {
    const float na = __fmaf_rn(a, co, -__fmul_rn(b, si));
    b = __fmaf_rn(b, co, __fmul_rn(a, si));
    a = na;
}

// Where a row's head is stored: null when the row does not write it.
template <typename T>
TG_DEVICE T *rope_out(const tg_params &p, int row, int head, uint32_t to, T *q, T *k, T *v) {
    if (head < (int)p.heads) return q + ((size_t)row * p.heads + head) * p.head_dim;
    if (to == SPARE) return nullptr;
    const int h = head - (int)p.heads;
    T *cache = h < (int)p.kv_heads ? k : v;
    const uint32_t page = to / p.capacity, off = to % p.capacity;
    return cache + (((size_t)page * p.kv_heads + h % (int)p.kv_heads) * p.capacity + off) * p.head_dim;
}

// A row's position and place; false when it writes nothing.
TG_DEVICE bool rope_row(const tg_params &p, const uint32_t *at, const uint32_t *place, int row, uint32_t &pos,
                        uint32_t &to, uint32_t *err) {
    pos = at[row];
    to = place[row];
    if (pos == SPARE) return false;
    if ((p.rope && pos >= p.n) || (to != SPARE && to >= p.slots * p.capacity)) {
        atomicExch(err, ERR_BAD_INDEX);
        return false;
    }
    return true;
}

// Eight dimensions of a head to a thread, for a rotated part that is a multiple of 8: rotated ones as
// four pairs (in the half layout two runs of four, each a warp's whole sectors).
template <typename T, typename C, bool INTER>
__global__ void __launch_bounds__(256)
    rope_pages_kernel(tg_params p, const uint32_t *__restrict__ at, const uint32_t *__restrict__ place,
                      const C *__restrict__ c, const float *__restrict__ cosv, const float *__restrict__ sinv,
                      T *__restrict__ q, T *__restrict__ k, T *__restrict__ v, uint32_t *err) {
    pdl_launch_dependents();
    pdl_wait();
    const uint32_t units = p.head_dim / 8, heads = p.heads + 2 * p.kv_heads, row_units = units * heads;
    const uint64_t i = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= (uint64_t)p.rows * row_units) return;
    const uint32_t row = (uint32_t)(i / row_units), in_row = (uint32_t)(i % row_units), head = in_row / units, u = in_row % units;
    uint32_t pos, to;
    if (!rope_row(p, at, place, row, pos, to, err)) return;
    T *o = rope_out(p, row, head, to, q, k, v);
    if (!o) return;
    const C *x = c + ((size_t)row * heads + head) * p.head_dim;
    const bool turned = p.rope && head < p.heads + p.kv_heads && u < p.k / 8;
    const uint32_t d0 = (turned && !INTER) ? 4 * u : 8 * u, d1 = (turned && !INTER) ? p.k / 2 + 4 * u : 8 * u + 4;
    float4 a = load4(x + d0), b = load4(x + d1);
    if (turned) {
        const float4 co = __ldg(reinterpret_cast<const float4 *>(cosv + (size_t)pos * (p.k / 2)) + u);
        const float4 si = __ldg(reinterpret_cast<const float4 *>(sinv + (size_t)pos * (p.k / 2)) + u);
        if (INTER) {
            turn(a.x, a.y, co.x, si.x);
            turn(a.z, a.w, co.y, si.y);
            turn(b.x, b.y, co.z, si.z);
            turn(b.z, b.w, co.w, si.w);
        } else {
            turn(a.x, b.x, co.x, si.x);
            turn(a.y, b.y, co.y, si.y);
            turn(a.z, b.z, co.z, si.z);
            turn(a.w, b.w, co.w, si.w);
        }
    }
    put4(o + d0, a);
    put4(o + d1, b);
}

// Any even rotated part: a pair to a thread.
template <typename T, typename C>
__global__ void __launch_bounds__(256)
    rope_pages_any_kernel(tg_params p, const uint32_t *__restrict__ at, const uint32_t *__restrict__ place,
                          const C *__restrict__ c, const float *__restrict__ cosv, const float *__restrict__ sinv,
                          T *__restrict__ q, T *__restrict__ k, T *__restrict__ v, uint32_t *err) {
    pdl_launch_dependents();
    pdl_wait();
    const uint32_t units = p.head_dim / 2, heads = p.heads + 2 * p.kv_heads, row_units = units * heads;
    const uint64_t i = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= (uint64_t)p.rows * row_units) return;
    const uint32_t row = (uint32_t)(i / row_units), in_row = (uint32_t)(i % row_units), head = in_row / units, u = in_row % units;
    uint32_t pos, to;
    if (!rope_row(p, at, place, row, pos, to, err)) return;
    T *o = rope_out(p, row, head, to, q, k, v);
    if (!o) return;
    const C *x = c + ((size_t)row * heads + head) * p.head_dim;
    const bool turned = p.rope && head < p.heads + p.kv_heads && u < p.k / 2;
    const bool half = turned && !(p.flags & 1);
    const uint32_t d0 = half ? u : 2 * u, d1 = half ? p.k / 2 + u : 2 * u + 1;
    float a = to_f32<C>(x[d0]), b = to_f32<C>(x[d1]);
    if (turned) turn(a, b, __ldg(cosv + (size_t)pos * (p.k / 2) + u), __ldg(sinv + (size_t)pos * (p.k / 2) + u));
    o[d0] = from_f32<T>(a);
    o[d1] = from_f32<T>(b);
}

// ---- logits_pick -----------------------------------------------------------------------------------
// A cluster of blocks to a row, each block a run of PICK_SLICE-token slices: the slice's occurrences
// counted in shared memory (every entry of the row's history is looked at, whole numbers added
// atomically: no order shows), then its logits streamed through once. The row's greedy choice is
// joined over the cluster in distributed shared memory. HBM-bound: each logit read and written once.
constexpr int PICK_THREADS = 512, PICK_SLICE = 4096, PICK_EACH = PICK_SLICE / PICK_THREADS;
constexpr uint32_t IN_PROMPT = 1u << 31;  // a slice word: the prompt holds the token; below, its generated occurrences

struct Best {
    float value;
    uint32_t token;
};
TG_DEVICE void better(Best &a, float value, uint32_t token) {
    if (value > a.value || (value == a.value && token < a.token)) a = Best{value, token};
}

// VEC consecutive logits to one 16-byte load (1: rows that are not 16-byte aligned).
template <typename T, int VEC>
__global__ void __launch_bounds__(PICK_THREADS)
    logits_pick_kernel(tg_params p, const T *logits, const uint32_t *__restrict__ seen,
                       const uint32_t *__restrict__ spans, const float *__restrict__ penalties,
                       const uint32_t *__restrict__ bias_ids, const float *__restrict__ bias,
                       const uint32_t *__restrict__ masks, T *out, uint32_t *__restrict__ pick, uint32_t *err) {
    namespace cg = cooperative_groups;
    __shared__ __align__(16) uint32_t count[PICK_SLICE], biased[PICK_SLICE];
    __shared__ Best warp_best[PICK_THREADS / 32], block_best;
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t tid = threadIdx.x, ranks = cluster.num_blocks(), rank = cluster.block_rank();
    const uint32_t row = blockIdx.x / ranks, n = p.n;
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
    const uint32_t *bits = masks + (size_t)(mask == SPARE ? 0 : mask) * ((n + 31) / 32);
    const T *x = logits + (size_t)row * p.stride;
    T *y = out + (size_t)row * p.stride;
    Best best{-INFINITY, SPARE};
    const uint32_t slices = (n + PICK_SLICE - 1) / PICK_SLICE;
    for (uint32_t slice = rank; slice < slices; slice += ranks) {
        const uint32_t t0 = slice * PICK_SLICE;
        // The slice's logits are on their way while its history is counted.
        float v[PICK_EACH];
#pragma unroll
        for (int j = 0; j < PICK_EACH / VEC; j++) {
            const uint32_t t = t0 + (j * PICK_THREADS + tid) * VEC;
            if constexpr (VEC > 1) {
                if (t + VEC <= n) {
                    typename Vec<T>::Raw raw = __ldcs(reinterpret_cast<const typename Vec<T>::Raw *>(x + t));
                    float f[Vec<T>::N];
                    Vec<T>::unpack(raw, f);
#pragma unroll
                    for (int e = 0; e < VEC; e++) v[j * VEC + e] = f[e];
                    continue;
                }
            }
#pragma unroll
            for (int e = 0; e < VEC; e++) v[j * VEC + e] = t + e < n ? to_f32<T>(x[t + e]) : 0.0f;
        }
        const bool controls = history || biases;
        if (controls) {
            __syncthreads();  // the slice before is done with the words
            for (uint32_t i = tid; i < PICK_SLICE / 4; i += PICK_THREADS) {
                reinterpret_cast<uint4 *>(count)[i] = make_uint4(0, 0, 0, 0);
                reinterpret_cast<uint4 *>(biased)[i] = make_uint4(0, 0, 0, 0);
            }
            __syncthreads();
            for (uint32_t i = tid; i < history; i += PICK_THREADS) {
                const uint32_t t = seen[begin + i] - t0;
                if (t < PICK_SLICE) {
                    if (i < prompt) atomicOr(count + t, IN_PROMPT);
                    else atomicAdd(count + t, 1u);
                }
            }
            for (uint32_t i = tid; i < biases; i += PICK_THREADS) {
                const uint32_t t = bias_ids[bias0 + i] - t0;
                if (t < PICK_SLICE) atomicMax(biased + t, i + 1);
            }
            __syncthreads();
        }
#pragma unroll
        for (int j = 0; j < PICK_EACH / VEC; j++) {
            const uint32_t in = (j * PICK_THREADS + tid) * VEC, t = t0 + in;
            if (t >= n) break;
            uint32_t allowed = 0xffffffffu;
            if (mask != SPARE) allowed = __ldg(bits + t / 32) >> (t % 32);
            __align__(16) T stored[VEC];
#pragma unroll
            for (int e = 0; e < VEC; e++) {
                float f = v[j * VEC + e];
                if (controls) {
                    const uint32_t c = count[in + e], b = biased[in + e];
                    if (c) {
                        const float m = (float)(c & ~IN_PROMPT);
                        f = f > 0.0f ? __fdiv_rn(f, repetition) : f * repetition;
                        f = f - m * frequency;
                        if (c & ~IN_PROMPT) f = f - presence;
                    }
                    if (b) f = f + bias[bias0 + b - 1];
                }
                if (!(allowed >> e & 1)) f = -INFINITY;
                stored[e] = from_f32<T>(f);
                // A thread meets its tokens in ascending order: the first of equal values stays.
                const float s = to_f32<T>(stored[e]);
                if (t + e < n && s > best.value) best = Best{s, t + e};
            }
            if (VEC > 1 && t + VEC <= n) {
                *reinterpret_cast<typename Vec<T>::Raw *>(y + t) = *reinterpret_cast<const typename Vec<T>::Raw *>(stored);
            } else {
#pragma unroll
                for (int e = 0; e < VEC; e++)
                    if (t + e < n) y[t + e] = stored[e];
            }
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        better(best, __shfl_xor_sync(0xffffffffu, best.value, o), __shfl_xor_sync(0xffffffffu, best.token, o));
    if ((tid & 31) == 0) warp_best[tid >> 5] = best;
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < PICK_THREADS / 32; w++) better(best, warp_best[w].value, warp_best[w].token);
        block_best = best;
    }
    cluster.sync();
    if (rank == 0 && tid == 0) {
        for (uint32_t b = 1; b < ranks; b++) {
            const Best o = *cluster.map_shared_rank(&block_best, b);
            better(best, o.value, o.token);
        }
        pick[row] = best.token;
    }
    cluster.sync();  // no block ends while its choice is read
}

template <typename T, int VEC>
cudaError_t pick_t(const tg_params &p, const void *logits, const uint32_t *seen, const uint32_t *spans, const float *pen,
                   const uint32_t *ids, const float *bias, const uint32_t *masks, void *out, uint32_t *pick, uint32_t *err,
                   cudaStream_t s) {
    const uint32_t slices = (p.n + PICK_SLICE - 1) / PICK_SLICE;
    uint32_t ranks = p.rows <= 64 ? 8 : 4;
    while (ranks > 1 && ranks / 2 >= slices) ranks /= 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(p.rows * ranks);
    cfg.blockDim = dim3(PICK_THREADS);
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
    const bool wide = p.k % 8 == 0;
    const uint64_t threads = (uint64_t)p.rows * (p.heads + 2 * p.kv_heads) * (p.head_dim / (wide ? 8 : 2));
    const uint64_t blocks = (threads + 255) / 256;
    if (blocks > 0x7fffffffu) return cudaErrorNotSupported;
    const dim3 grid((unsigned)blocks);
    auto run = [&](auto kern) {
        return launch_pdl(kern, grid, dim3(256), 0, s, p, at, place, (const C *)c, cs, sn, (T *)q, (T *)k, (T *)v, err);
    };
    if (!wide) return run(rope_pages_any_kernel<T, C>);
    return p.flags & 1 ? run(rope_pages_kernel<T, C, true>) : run(rope_pages_kernel<T, C, false>);
}

}  // namespace

cudaError_t launch_page_plan(const tg_params &p, const uint32_t *held, const uint32_t *fresh, const uint32_t *free,
                             uint32_t *table, uint32_t *at, uint32_t *place, uint32_t *starts, uint32_t *next,
                             uint32_t *counts, uint32_t *err, cudaStream_t s) {
    const size_t smem = 2 * ((size_t)p.seqs + 1) * sizeof(uint32_t);
    cudaError_t e = with_smem(page_plan_kernel, smem);
    if (e != cudaSuccess) return e;
    const uint32_t blocks = min((p.rows + PLAN_ROWS - 1) / PLAN_ROWS, 128u);
    return launch_pdl(page_plan_kernel, dim3(blocks), dim3(PLAN_THREADS), smem, s, p, held, fresh, free, table, at, place,
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
