// Decode attention over pages for a batch that shares a long prefix. A row's keys are cut into pieces:
// the shared prefix's (of a length that depends on the prefix alone) and its own positions' (of a
// fixed length), so that a row's sums are the same bits whatever rows run beside it. Each piece gives
// a partial: the largest scaled score m, the sum l of e^(s - m), and o = sum e^(s - m) v; a last
// kernel joins a row's partials: M = max m, out = sum o e^(m - M) / sum l e^(m - M).
#include "mma_common.cuh"
#include "tg_internal.h"

namespace tg {

namespace {

constexpr uint32_t SPARE = TG_SPARE;
constexpr int CHUNK = 128;  // positions a block takes at once

// Own positions of a piece.
__host__ __device__ constexpr uint32_t own_piece(uint32_t hd) { return 16384 / hd; }
// Shared positions of a piece: at most 16 pieces, each whole chunks.
__host__ __device__ inline uint32_t shared_piece(uint32_t first) {
    const uint32_t even = (first + 15) / 16;
    return even <= CHUNK ? CHUNK : (even + CHUNK - 1) / CHUNK * CHUNK;
}
__host__ __device__ inline uint32_t shared_pieces(uint32_t first) { return (first + shared_piece(first) - 1) / shared_piece(first); }
__host__ __device__ inline uint64_t all_pieces(const tg_params &p) {
    return shared_pieces(p.first) + ((uint64_t)p.stride * p.capacity + own_piece(p.head_dim) - 1) / own_piece(p.head_dim);
}

// The partials in the work buffer: o f32 [rows][heads][pieces][hd], then m, l f32 [rows][heads][pieces][2].
struct Partials {
    float *o, *ml;
};

// A row's own length and request; false for a row that computes nothing.
TG_DEVICE bool paged_row(const tg_params &p, const uint32_t *at, int row, uint32_t &length, uint32_t &seq, uint32_t *err) {
    const uint32_t pos = at[row];
    seq = at[p.rows + row];
    if (pos == SPARE) return false;
    length = pos - p.first + 1;
    if (pos < p.first || (uint64_t)length > (uint64_t)p.stride * p.capacity || seq >= p.seqs) {
        if (err) atomicExch(err, ERR_BAD_INDEX);
        return false;
    }
    return true;
}

// A piece of a row for one KV head, on the CUDA cores: a thread to a position for the scores, to a
// dimension for the output, chunk by chunk with a running maximum.
template <typename T, int HD>
__global__ void __launch_bounds__(CHUNK)
    pieces_kernel(tg_params p, const T *__restrict__ q, const T *__restrict__ k, const T *__restrict__ v,
                  const uint32_t *__restrict__ at, const uint32_t *__restrict__ table, const uint32_t *__restrict__ shared,
                  Partials out, uint32_t np, uint32_t pieces, uint32_t *err) {
    constexpr int G = MAX_GROUP, HALVES = CHUNK / HD;
    __shared__ __align__(16) float qs[G][HD];
    __shared__ float es[G][CHUNK], red[G][CHUNK / 32], mrun[G], lrun[G], alpha[G];
    __shared__ uint64_t from[CHUNK];
    __shared__ float add[HALVES > 1 ? G : 1][HD];
    pdl_launch_dependents();
    pdl_wait();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, row = blockIdx.z, kv = blockIdx.y, piece = blockIdx.x;
    const int heads = p.heads, kvh = p.kv_heads, group = heads / kvh;
    uint32_t length, seq;
    if (!paged_row(p, at, row, length, seq, kv == 0 && piece == 0 && tid == 0 ? err : nullptr)) return;
    const bool own = piece >= (int)np;
    const uint32_t size = own ? own_piece(HD) : shared_piece(p.first), n = own ? length : p.first;
    const uint64_t begin = (uint64_t)(own ? piece - np : piece) * size;
    if (begin >= n) return;
    const uint32_t stop = (uint32_t)min((uint64_t)n, begin + size);
    const uint32_t *list = own ? table + (size_t)seq * p.stride : shared;
    const float scale = 1.0f / sqrtf((float)HD);
    for (int i = tid; i < group * HD; i += CHUNK) qs[i / HD][i % HD] = to_f32<T>(q[((size_t)row * heads + kv * group) * HD + i]) * scale;
    if (tid < G) {
        mrun[tid] = -INFINITY;
        lrun[tid] = 0.0f;
    }
    float acc[G];
#pragma unroll
    for (int g = 0; g < G; g++) acc[g] = 0.0f;
    for (uint32_t c0 = (uint32_t)begin; c0 < stop; c0 += CHUNK) {
        __syncthreads();
        const uint32_t pos = c0 + tid;
        const bool live = pos < stop;
        float s[G];
#pragma unroll
        for (int g = 0; g < G; g++) s[g] = live ? 0.0f : -INFINITY;
        if (live) {
            uint32_t id = list[pos / p.capacity];
            if (id >= p.slots) {
                atomicExch(err, ERR_BAD_INDEX);
                id = 0;
            }
            from[tid] = (((uint64_t)id * kvh + kv) * p.capacity + pos % p.capacity) * HD;
            const typename Vec<T>::Raw *kr = reinterpret_cast<const typename Vec<T>::Raw *>(k + from[tid]);
#pragma unroll 4
            for (int d = 0; d < HD / Vec<T>::N; d++) {
                float f[Vec<T>::N];
                Vec<T>::unpack(__ldg(kr + d), f);
#pragma unroll
                for (int g = 0; g < G; g++)
                    if (g < group)
#pragma unroll
                        for (int e = 0; e < Vec<T>::N; e++) s[g] = __fmaf_rn(f[e], qs[g][d * Vec<T>::N + e], s[g]);
            }
        }
#pragma unroll
        for (int g = 0; g < G; g++) {
            const float m = warp_max(s[g]);
            if (lane == 0) red[g][warp] = m;
        }
        __syncthreads();
        if (tid < G) {
            float m = mrun[tid];
            for (int w = 0; w < CHUNK / 32; w++) m = fmaxf(m, red[tid][w]);
            alpha[tid] = mrun[tid] == -INFINITY ? 0.0f : expf(mrun[tid] - m);
            mrun[tid] = m;
        }
        __syncthreads();
#pragma unroll
        for (int g = 0; g < G; g++) {
            const float e = s[g] == -INFINITY ? 0.0f : expf(s[g] - mrun[g]);
            es[g][tid] = e;
            const float l = warp_sum(e);
            if (lane == 0) red[g][warp] = l;
        }
        __syncthreads();
        if (tid < G) {
            float l = lrun[tid] * alpha[tid];
            for (int w = 0; w < CHUNK / 32; w++) l += red[tid][w];
            lrun[tid] = l;
        }
        const int d = tid % HD, half = tid / HD, count = (int)min((uint32_t)CHUNK, stop - c0);
#pragma unroll
        for (int g = 0; g < G; g++) acc[g] *= alpha[g];
        for (int i = half; i < count; i += HALVES) {
            const float x = to_f32<T>(v[from[i] + d]);
#pragma unroll
            for (int g = 0; g < G; g++) acc[g] = __fmaf_rn(es[g][i], x, acc[g]);
        }
    }
    if (HALVES > 1) {
        __syncthreads();
        if (tid >= HD)
#pragma unroll
            for (int g = 0; g < G; g++) add[g][tid - HD] = acc[g];
        __syncthreads();
        if (tid < HD)
#pragma unroll
            for (int g = 0; g < G; g++) acc[g] += add[g][tid];
    }
    __syncthreads();
#pragma unroll
    for (int g = 0; g < G; g++) {
        if (g >= group) break;
        const size_t to = ((size_t)row * heads + kv * group + g) * pieces + piece;
        if (tid < HD) out.o[to * HD + tid] = acc[g];
        if (tid == 0) *reinterpret_cast<float2 *>(out.ml + to * 2) = make_float2(mrun[g], lrun[g]);
    }
}

// Joins a row's partials, a warp to a head, in piece order.
template <typename T, int HD>
__global__ void __launch_bounds__(128)
    join_kernel(tg_params p, const uint32_t *__restrict__ at, Partials in, uint32_t np, uint32_t pieces, T *__restrict__ out) {
    constexpr int D = HD / 32;
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31;
    const uint64_t item = (uint64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (item >= (uint64_t)p.rows * p.heads) return;
    const int row = (int)(item / p.heads);
    uint32_t length, seq;
    if (!paged_row(p, at, row, length, seq, nullptr)) return;
    const uint32_t n = np + (length + own_piece(HD) - 1) / own_piece(HD);
    const float2 *ml = reinterpret_cast<const float2 *>(in.ml) + item * pieces;
    const float *o = in.o + item * pieces * HD + lane * D;
    float m = -INFINITY;
    for (uint32_t i = lane; i < n; i += 32) m = fmaxf(m, ml[i].x);
    m = warp_max(m);
    float l = 0.0f, acc[D];
#pragma unroll
    for (int d = 0; d < D; d++) acc[d] = 0.0f;
    for (uint32_t i = 0; i < n; i++) {
        const float2 part = ml[i];
        const float e = part.x == -INFINITY ? 0.0f : expf(part.x - m);
        l = __fmaf_rn(part.y, e, l);
#pragma unroll
        for (int d = 0; d < D; d++) acc[d] = __fmaf_rn(o[(size_t)i * HD + d], e, acc[d]);
    }
#pragma unroll
    for (int d = 0; d < D; d++) out[item * HD + lane * D + d] = from_f32<T>(__fdiv_rn(acc[d], l));
}

template <typename T, int HD>
cudaError_t attend(const tg_params &p, const void *q, const void *k, const void *v, const uint32_t *at, const uint32_t *table,
                   const uint32_t *shared, void *work, void *out, uint32_t *err, cudaStream_t s) {
    const uint64_t pieces = all_pieces(p), items = (uint64_t)p.rows * p.heads;
    if (pieces > 0x7fffffffu || p.kv_heads > 65535) return cudaErrorNotSupported;
    Partials part{static_cast<float *>(work), static_cast<float *>(work) + items * pieces * HD};
    const uint32_t np = shared_pieces(p.first);
    cudaError_t e = launch_pdl(pieces_kernel<T, HD>, dim3((unsigned)pieces, p.kv_heads, p.rows), dim3(CHUNK), 0, s, p, (const T *)q,
                               (const T *)k, (const T *)v, at, table, shared, part, np, (uint32_t)pieces, err);
    if (e != cudaSuccess) return e;
    return launch_pdl(join_kernel<T, HD>, dim3((unsigned)((items + 3) / 4)), dim3(128), 0, s, p, at, part, np, (uint32_t)pieces, (T *)out);
}

}  // namespace

uint64_t attention_pages_work(const tg_params &p) {
    if (p.head_dim == 0 || p.head_dim > 16384) return 0;
    return (uint64_t)p.rows * p.heads * all_pieces(p) * (p.head_dim + 2) * sizeof(float);
}

cudaError_t launch_attention_pages(const tg_params &p, const void *q, const void *k, const void *v, const uint32_t *at,
                                   const uint32_t *table, const uint32_t *shared, void *work, void *out, uint32_t *err,
                                   cudaStream_t s) {
    if (p.dtype == TG_BF16)
        return p.head_dim == 64 ? attend<bf16, 64>(p, q, k, v, at, table, shared, work, out, err, s)
                                : attend<bf16, 128>(p, q, k, v, at, table, shared, work, out, err, s);
    return p.head_dim == 64 ? attend<float, 64>(p, q, k, v, at, table, shared, work, out, err, s)
                            : attend<float, 128>(p, q, k, v, at, table, shared, work, out, err, s);
}

}  // namespace tg
