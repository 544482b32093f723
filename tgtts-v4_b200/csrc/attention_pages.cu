// Decode attention over pages for a batch that shares a long prefix. A row's keys are cut into pieces:
// the shared prefix's (of a length that depends on the prefix alone) and its own positions' (of a
// fixed length), so that a row's sums are the same bits whatever rows run beside it. Each piece gives
// a partial: a reference m near the largest scaled score, the sum l of e^(s - m), and
// o = sum e^(s - m) v; a last kernel joins a row's partials: M = max m,
// out = sum o e^(m - M) / sum l e^(m - M).
//
// For bf16 the shared pieces run on tcgen05 (prefix_kernel): the rows of all requests, times the query
// heads of one KV head, are the 128 rows of its products, so that a tile of keys and values is read
// once for 128 queries. The own pieces, which no other row shares, run on mma.sync
// (own_kernel), bound by the caches' bytes. f32 runs on the CUDA cores (f32_kernel, for both kinds of piece).
#include <algorithm>

#include "mma_common.cuh"
#include "tc_common.cuh"

namespace tg {

namespace {

constexpr uint32_t SPARE = TG_SPARE;

// Own positions of a piece.
constexpr uint32_t OWN_PIECE = 128;
// n / d, rounded up.
__host__ __device__ inline uint32_t shares(uint32_t n, uint32_t d) { return n / d + (n % d != 0); }
// Shared positions of a piece, whole tiles of 128: at most 16 pieces; 8 while those are at most 512 and at most 64 x KV
// heads long, as the KV heads make units too. (Rows of one own position behind 4096, 8 KV heads of 128,
// pieces of 512 against 256: one row 17.3 us against 17.0, 32 rows 20.3 against 20.5, 64 rows 23.0 against 26.7, 128 rows
// 34 against 41. Behind 16384 pieces of 2048 against 1024: one row 33 against 25, 32 rows 36 against 29, 64 rows 39 against
// 42, 128 rows 64 against 70. Behind 8191, 2 KV heads of 64, pieces of 1024 against 512: 128 rows 31 against 24.)
__host__ __device__ inline uint32_t shared_piece(const tg_params &p) {
    const uint32_t most = p.kv_heads < 8 ? 64 * p.kv_heads : 512, even = shares(p.first, 8);
    const uint32_t longer = even < most ? even : most, size = longer > shares(p.first, 16) ? longer : shares(p.first, 16);
    return size ? shares(size, 128) * 128 : 128;
}
__host__ __device__ inline uint32_t shared_pieces(const tg_params &p) { return shares(p.first, shared_piece(p)); }
__host__ __device__ inline uint64_t all_pieces(const tg_params &p) {
    return shared_pieces(p) + ((uint64_t)p.stride * p.capacity + OWN_PIECE - 1) / OWN_PIECE;
}

// The partials in the work buffer, from its first 256-byte boundary: o f32 [rows][heads][pieces][hd], then
// m, l f32 [rows][heads][pieces][2].
struct Partials {
    float *o, *ml;
};
constexpr uint32_t OWN_ROWS = 512;  // rows whose own pieces are listed at once

// A row's own length, of its position and request; false for a row that computes nothing.
TG_DEVICE bool paged_words(const tg_params &p, uint32_t pos, uint32_t seq, uint32_t &length, uint32_t *err) {
    if (pos == SPARE) return false;
    length = pos - p.first + 1;
    if (pos < p.first || (uint64_t)length > (uint64_t)p.stride * p.capacity || seq >= p.seqs) {
        if (err) atomicExch(err, ERR_BAD_INDEX);
        return false;
    }
    return true;
}
TG_DEVICE bool paged_row(const tg_params &p, const uint32_t *at, int row, uint32_t &length, uint32_t &seq, uint32_t *err) {
    const uint32_t pos = at[row];
    seq = at[p.rows + row];
    return paged_words(p, pos, seq, length, err);
}

// ---- f32, on the CUDA cores ----------------------------------------------------------------------------
// A block to a piece for one KV head and up to QN queries: of a row's own positions for the heads of the row, of
// the shared prefix for the heads of as many rows as fit, so that its keys and values are read once for them.
// Chunks of keys in shared memory (32 KB of them, and of values); a thread to a key and a share of the queries for
// the scores, to a dimension and a share of the queries for the output, with a running maximum over the chunks.
// Products, sums and statistics in f32; the references are natural.
// Bound by the shared memory reads that feed the multiply-adds (three of 16 bytes to 32 of those). One launch for
// both kinds of piece: two cost 5 us more in a call of 10 rows. 32 queries a block against one row's heads:
// 128 rows of 16 heads over 2 at head dim 64 behind 4096 shared positions in 118 us against 211, 18 TFLOP/s.
constexpr int F32_THREADS = 256, F32_QUERIES = 32;
template <int HD, int QN>
struct F32 {
    static constexpr int CHUNK = 8192 / HD;  // keys at once
    static constexpr int KROW = HD + 4;  // floats of a key: eight keys' same 16 bytes lie in all banks
    static constexpr int V = CHUNK * KROW, Q = V + CHUNK * HD, E = Q + QN * HD, FLOATS = E + QN * CHUNK;
};

template <int HD, int QN, bool SHARED>
__device__ __forceinline__ void f32_piece(const tg_params &p, const float *__restrict__ q, const float *__restrict__ k,
                                          const float *__restrict__ v, const uint32_t *__restrict__ at, const uint32_t *__restrict__ table,
                                          const uint32_t *__restrict__ shared, const Partials &out, uint32_t index, uint32_t kv, uint32_t tile,
                                          uint32_t np, uint32_t pieces, uint32_t *err) {
    using C = F32<HD, QN>;
    constexpr int CHUNK = C::CHUNK, PARTS = F32_THREADS / HD, QH = QN * CHUNK / F32_THREADS, QP = QN / PARTS;
    static_assert(QH >= 1 && QP >= 1 && QN % PARTS == 0, "threads");
    extern __shared__ __align__(16) float f32_mem[];
    float *ks = f32_mem, *vs = f32_mem + C::V, *qs = f32_mem + C::Q, *es = f32_mem + C::E;
    __shared__ float mrun[QN], lrun[QN], keep_s[QN];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, heads = p.heads, kvh = p.kv_heads, group = heads / kvh;
    const int rows = SHARED ? QN / group : 1, row0 = tile * rows, queries = min(rows, (int)p.rows - row0) * group;
    uint32_t length = p.first, seq = 0;
    const uint32_t size = SHARED ? shared_piece(p) : OWN_PIECE;
    const uint64_t begin = (uint64_t)index * size;
    if ((!SHARED && !paged_row(p, at, row0, length, seq, kv == 0 && index == 0 && tid == 0 ? err : nullptr)) || begin >= length) return;
    const uint32_t stop = (uint32_t)min((uint64_t)length, begin + size);
    const uint32_t *list = SHARED ? shared : table + (size_t)seq * p.stride;
    const float scale = 1.0f / sqrtf((float)HD);
    auto head_of = [&](int j) { return ((size_t)(row0 + j / group) * heads + (size_t)kv * group + j % group); };
    for (int i = tid; i < QN * (HD / 4); i += F32_THREADS) {
        const int j = i / (HD / 4), d = i % (HD / 4) * 4;
        float4 x = j < queries ? *reinterpret_cast<const float4 *>(q + head_of(j) * HD + d) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        *reinterpret_cast<float4 *>(qs + j * HD + d) = make_float4(x.x * scale, x.y * scale, x.z * scale, x.w * scale);
    }
    if (tid < QN) {
        mrun[tid] = -INFINITY;
        lrun[tid] = 0.0f;
    }
    float acc[QP];
#pragma unroll
    for (int j = 0; j < QP; j++) acc[j] = 0.0f;
    const int d = tid % HD, part = tid / HD;
    for (uint32_t c0 = (uint32_t)begin; c0 < stop; c0 += CHUNK) {
        const int live = (int)min(stop - c0, (uint32_t)CHUNK);
        __syncthreads();  // the chunk before is done with
        for (int i = tid; i < CHUNK * (HD / 4); i += F32_THREADS) {
            const int r = i / (HD / 4), x = i % (HD / 4) * 4;
            const uint32_t pos = c0 + min(r, live - 1);
            uint32_t id = __ldg(list + pos / p.capacity);
            if (id >= p.slots) {
                atomicExch(err, ERR_BAD_INDEX);
                id = 0;
            }
            const size_t from = (((size_t)id * kvh + kv) * p.capacity + pos % p.capacity) * HD + x;
            fa::cp_async16(ks + r * C::KROW + x, k + from, r < live);
            fa::cp_async16(vs + r * HD + x, v + from, r < live);  // zero past the piece: 0 x NaN is NaN
        }
        fa::cp_async_commit();
        fa::cp_async_wait<0>();
        __syncthreads();
        {
            const int key = tid % CHUNK, half = tid / CHUNK;
            float s[QH];
#pragma unroll
            for (int j = 0; j < QH; j++) s[j] = 0.0f;
#pragma unroll 4
            for (int x = 0; x < HD; x += 4) {
                const float4 kx = *reinterpret_cast<const float4 *>(ks + key * C::KROW + x);
#pragma unroll
                for (int j = 0; j < QH; j++) {
                    const float4 qx = *reinterpret_cast<const float4 *>(qs + (half * QH + j) * HD + x);
                    s[j] = __fmaf_rn(kx.w, qx.w, __fmaf_rn(kx.z, qx.z, __fmaf_rn(kx.y, qx.y, __fmaf_rn(kx.x, qx.x, s[j]))));
                }
            }
#pragma unroll
            for (int j = 0; j < QH; j++) es[(half * QH + j) * CHUNK + key] = key < live ? s[j] : -INFINITY;
        }
        __syncthreads();
        for (int j = warp; j < queries; j += F32_THREADS / 32) {
            float e[CHUNK / 32], top = -INFINITY, sum = 0.0f;
#pragma unroll
            for (int i = 0; i < CHUNK / 32; i++) top = fmaxf(top, e[i] = es[j * CHUNK + i * 32 + lane]);
            const float m0 = mrun[j], l0 = lrun[j], m = fmaxf(m0, warp_max(top));
#pragma unroll
            for (int i = 0; i < CHUNK / 32; i++) {
                const float x = e[i] == -INFINITY ? 0.0f : expf(e[i] - m);
                es[j * CHUNK + i * 32 + lane] = x;
                sum += x;
            }
            const float l = warp_sum(sum), keep = m0 == -INFINITY ? 0.0f : expf(m0 - m);
            if (lane == 0) {
                mrun[j] = m;
                lrun[j] = __fmaf_rn(l0, keep, l);
                keep_s[j] = keep;
            }
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < QP; j++)
            if (part * QP + j < queries) acc[j] *= keep_s[part * QP + j];
#pragma unroll 2
        for (int x = 0; x < CHUNK; x += 4) {
            const float v0 = vs[x * HD + d], v1 = vs[(x + 1) * HD + d], v2 = vs[(x + 2) * HD + d], v3 = vs[(x + 3) * HD + d];
#pragma unroll
            for (int j = 0; j < QP; j++) {
                const float4 e = *reinterpret_cast<const float4 *>(es + (part * QP + j) * CHUNK + x);
                acc[j] = __fmaf_rn(e.w, v3, __fmaf_rn(e.z, v2, __fmaf_rn(e.y, v1, __fmaf_rn(e.x, v0, acc[j]))));
            }
        }
    }
    const uint32_t piece = SHARED ? index : np + index;
#pragma unroll
    for (int j = 0; j < QP; j++) {
        const int x = part * QP + j;
        if (x < queries) out.o[(head_of(x) * pieces + piece) * HD + d] = acc[j];
    }
    if (tid < queries) *reinterpret_cast<float2 *>(out.ml + (head_of(tid) * pieces + piece) * 2) = make_float2(mrun[tid], lrun[tid]);
}

// Blocks of the shared pieces first (they take longer), then those of the rows' own; a block to a KV head in y.
template <int HD>
__global__ void __launch_bounds__(F32_THREADS)
    f32_kernel(tg_params p, const float *__restrict__ q, const float *__restrict__ k, const float *__restrict__ v,
               const uint32_t *__restrict__ at, const uint32_t *__restrict__ table, const uint32_t *__restrict__ shared, Partials out,
               uint32_t np, uint32_t pieces, uint32_t far, uint32_t *err) {
    pdl_wait();
    pdl_launch_dependents();
    if (blockIdx.x < far)
        f32_piece<HD, F32_QUERIES, true>(p, q, k, v, at, table, shared, out, blockIdx.x % np, blockIdx.y, blockIdx.x / np, np, pieces, err);
    else {
        const uint32_t b = blockIdx.x - far, own = pieces - np;
        f32_piece<HD, MAX_GROUP, false>(p, q, k, v, at, table, shared, out, b % own, blockIdx.y, b / own, np, pieces, err);
    }
}

// ---- tcgen05 parts ------------------------------------------------------------------------------------
// How far (base 2) a maximum may pass a query's reference before O and l are rescaled.
constexpr float MOVE_PAST = 8.0f;

// 2^x by the hardware's base-2 exponential (relative error about 2^-22); 2^-inf = 0.
TG_DEVICE float hw_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Brings a copy's descriptor near before its first use.
TG_DEVICE void prefetch_map(const CUtensorMap *map) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory");
}
// A tile [keys][64 to a chunk] read with its 64-dimension chunks (`chunk` bytes apart) as M or N and its keys as K: atoms of
// 8 keys x 128 bytes, 1024 bytes apart.
TG_DEVICE uint64_t mn_desc(uint32_t addr, uint32_t chunk) {
    return (uint64_t)((addr >> 4) & 0x3fff) | ((uint64_t)(chunk >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
           ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}

// ---- own pieces, bf16 ---------------------------------------------------------------------------------
// A warp to a piece of a row's own positions for one KV head, in chunks of own_chunk positions: the group's
// query heads, at most 8, are the columns of mma.sync.m16n8k16 (S^T = K q^T, O^T = V^T e^T with e split
// into bf16 hi + lo, against a reference that moves as prefix_kernel's), keys and values gathered from their
// pages by cp.async, OWN_STAGES - 1 chunks ahead of the products. e keeps 16 bits because a row's own positions are
// few and may carry its whole sum; the second product costs nothing here, as the caches' bytes bound the
// kernel: a head reads 4 hd bytes a position for 4 hd x group operations. What is needed is bytes in flight: 11
// one-warp blocks an SM of two 8 KB stages each hold 90 KB of them. 64 rows of up to 1024, 8 KV
// heads of 128 (143 MB, not in L2): 34.8 us with the join, 4.1 TB/s; 128 rows (268 MB) 62 us, 4.3 TB/s (four warps to a
// block: 36.3 and 59 us; 64 rows behind 16384 shared positions 70 with one, 72 with four). Pieces of 128
// positions, so that the longest row is no one warp's.
constexpr int OWN_WARPS = 1, OWN_STAGES = 2;
constexpr int own_chunk(int hd) { return 2048 / hd; }
constexpr int OWN_STAGE = 2 * 2048;  // bf16 of a chunk's keys and values
constexpr int OWN_SMEM = OWN_WARPS * OWN_STAGES * OWN_STAGE * 2 + (int)OWN_ROWS * 4;
constexpr int OWN_BLOCKS = 11;  // an SM's, by their shared memory
// 16 bytes c of row r of a chunk, as an element: the rows' pieces turned so that eight rows' same piece lie in all banks.
template <int HD>
TG_DEVICE int own_at(int r, int c) { return r * HD + ((c ^ (r & 7)) << 3); }

// An 8 x 8 block of 16-bit values over a warp (lane 4 r + c: columns 2 c and 2 c + 1 of row r), transposed.
TG_DEVICE uint32_t turn8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

template <int HD>
__global__ void __launch_bounds__(OWN_WARPS * 32)
    own_kernel(tg_params p, const bf16 *__restrict__ q, const bf16 *__restrict__ k, const bf16 *__restrict__ v,
               const uint32_t *__restrict__ at, const uint32_t *__restrict__ table, Partials out, uint32_t np,
               uint32_t pieces, uint32_t *err) {
    using namespace fa;
    extern __shared__ __align__(128) unsigned char own_mem[];
    __shared__ uint32_t total_s;
    constexpr int CH = own_chunk(HD), VECS = HD / 8, G16 = CH / 16, ROWS = 32 / VECS;
    // Every block waits, behind prefix_kernel too: the rows' words, the table and the pages may be the stores of kernels
    // before both, and this wait alone makes them visible here. (Run under prefix_kernel without it, 64 rows behind 1024 positions
    // took 13 us against 22, 64 behind 16384 55 against 70, but nothing ordered the loads behind those stores.)
    pdl_wait();
    pdl_launch_dependents();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3, mi = lane >> 3, rr = lane & 7;
    const int heads = p.heads, kvh = p.kv_heads, group = heads / kvh;
    bf16 *stages = reinterpret_cast<bf16 *>(own_mem) + warp * OWN_STAGES * OWN_STAGE;
    uint32_t *first_piece = reinterpret_cast<uint32_t *>(own_mem + OWN_WARPS * OWN_STAGES * OWN_STAGE * 2);
    const float scale2 = 1.4426950408889634f / sqrtf((float)HD);
    for (uint32_t row0 = 0; row0 < p.rows; row0 += OWN_ROWS) {
        // The pieces of rows row0 .. before each of them.
        const uint32_t rows = min(OWN_ROWS, p.rows - row0);
        __syncthreads();  // the rows before are done with their list
        if (warp == 0) {
            uint32_t total = 0;
            constexpr int AT_ONCE = 4;  // loads of 32 rows' words in flight
            for (uint32_t r0 = 0; r0 < rows; r0 += 32 * AT_ONCE) {
                uint32_t pos[AT_ONCE], seq[AT_ONCE];
#pragma unroll
                for (int i = 0; i < AT_ONCE; i++) {
                    const uint32_t r = r0 + 32 * i + lane;
                    pos[i] = r < rows ? at[row0 + r] : SPARE;
                    seq[i] = r < rows ? at[p.rows + row0 + r] : 0;
                }
#pragma unroll
                for (int i = 0; i < AT_ONCE; i++) {
                    const uint32_t r = r0 + 32 * i + lane;
                    uint32_t length, n = 0;
                    if (paged_words(p, pos[i], seq[i], length, blockIdx.x == 0 ? err : nullptr)) n = (length + OWN_PIECE - 1) / OWN_PIECE;
                    uint32_t upto = n;
#pragma unroll
                    for (int o = 1; o < 32; o <<= 1) {
                        const uint32_t u = __shfl_up_sync(0xffffffffu, upto, o);
                        if (lane >= o) upto += u;
                    }
                    if (r < rows) first_piece[r] = total + upto - n;
                    total += __shfl_sync(0xffffffffu, upto, 31);
                }
            }
            if (lane == 0) total_s = total;
        }
        __syncthreads();
        // (Fewer than 2^32: each has partials of 264 bytes or more in the work buffer.)
        const uint32_t tasks = total_s * kvh, step = gridDim.x * OWN_WARPS;
        // A task, and the words that lead to its pages: they are on their way while the one before is computed.
        uint32_t row_n, piece_n, pos_n, seq_n, id_n = 0;
        auto find = [&](uint32_t task) {
            if (task >= tasks) return;
            const uint32_t u = task / kvh;
            uint32_t lo = 0, hi = rows;  // the row with first_piece at most u, its next above
            while (hi - lo > 1) {
                const uint32_t mid = (lo + hi) / 2;
                if (first_piece[mid] <= u) lo = mid;
                else hi = mid;
            }
            row_n = row0 + lo;
            piece_n = u - first_piece[lo];
            pos_n = at[row_n];
            seq_n = at[p.rows + row_n];
        };
        auto live_of = [&](uint32_t pos, uint32_t piece) { return (int)min(pos - p.first + 1 - piece * OWN_PIECE, OWN_PIECE); };
        // Positions piece x OWN_PIECE + 16 i .. share a page: lane i < 8.
        auto place_of = [&](uint32_t piece, int live) { return piece * OWN_PIECE + min(16 * (lane & 7), (live - 1) & ~15); };
        auto fetch = [&](uint32_t task) {
            if (task < tasks) id_n = __ldg(table + (size_t)seq_n * p.stride + place_of(piece_n, live_of(pos_n, piece_n)) / p.capacity);
        };
        const uint32_t task0 = blockIdx.x * OWN_WARPS + warp;
        find(task0);
        fetch(task0);
        for (uint32_t task = task0; task < tasks; task += step) {
            const int kv = (int)(task % kvh);
            const uint32_t row = row_n, piece = piece_n;
            const int live = live_of(pos_n, piece_n), chunks = (live + CH - 1) / CH;
            uint64_t from;
            {
                uint32_t id = id_n;
                if (id >= p.slots) {
                    atomicExch(err, ERR_BAD_INDEX);
                    id = 0;
                }
                from = (((uint64_t)id * kvh + kv) * p.capacity + place_of(piece, live) % p.capacity) * HD;
            }
            const int in_row = lane % VECS, in_group = lane / VECS;
            auto gather = [&](int c) {
                bf16 *ks = stages + (c % OWN_STAGES) * OWN_STAGE, *vs = ks + CH * HD;
#pragma unroll
                for (int i = 0; i < G16; i++) {
                    const uint64_t src = __shfl_sync(0xffffffffu, from, c * G16 + i) + in_group * HD + in_row * 8;
#pragma unroll
                    for (int j = 0; j < 16 / ROWS; j++) {
                        const int r = 16 * i + ROWS * j + in_group, d = own_at<HD>(r, in_row);
                        const bool ok = c * CH + r < live;
                        const uint64_t at_src = ok ? src + ROWS * j * HD : src - in_group * HD;  // a page's first position is there
                        cp_async16(ks + d, k + at_src, ok);
                        cp_async16(vs + d, v + at_src, ok);
                    }
                }
            };
#pragma unroll
            for (int c = 0; c < OWN_STAGES - 1; c++) {
                if (c < chunks) gather(c);
                cp_async_commit();
            }
            find(task + step);
            // q of the group's heads as columns g < group of the products (those past it zero).
            uint32_t qf[HD / 16][2];
            const bf16 *qg = q + ((size_t)row * heads + kv * group + g) * HD + 2 * t4;
#pragma unroll
            for (int s = 0; s < HD / 16; s++) {
                qf[s][0] = g < group ? __ldg(reinterpret_cast<const uint32_t *>(qg + 16 * s)) : 0u;
                qf[s][1] = g < group ? __ldg(reinterpret_cast<const uint32_t *>(qg + 16 * s + 8)) : 0u;
            }
            // A lane's heads 2 t4 and 2 t4 + 1: references, sums, and dimensions g and g + 8 of each 16 of O^T.
            float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f}, o[HD / 16][4];
#pragma unroll
            for (int j = 0; j < HD / 16; j++) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.0f;
            for (int c = 0; c < chunks; c++) {
                cp_async_wait<OWN_STAGES - 2>();
                __syncwarp();  // the chunk is in, and every lane is done with the one before
                if (c + OWN_STAGES - 1 < chunks) gather(c + OWN_STAGES - 1);
                cp_async_commit();
                if (c == 0) fetch(task + step);
                const bf16 *ks = stages + (c % OWN_STAGES) * OWN_STAGE, *vs = ks + CH * HD;
                float sc[G16][4];  // positions g and g + 8 of each 16, the lane's two heads
                const int left = live - c * CH - g;
#pragma unroll
                for (int j = 0; j < G16; j++) {
                    float odd[4] = {0.0f, 0.0f, 0.0f, 0.0f};  // two sums, for two chains of products
                    sc[j][0] = sc[j][1] = sc[j][2] = sc[j][3] = 0.0f;
#pragma unroll
                    for (int s = 0; s < HD / 16; s++) {
                        uint32_t ka[4];
                        ldmatrix_x4(ka, ks + own_at<HD>(16 * j + (mi & 1) * 8 + rr, 2 * s + (mi >> 1)));
                        mma_bf16(s & 1 ? odd : sc[j], ka, qf[s][0], qf[s][1]);
                    }
#pragma unroll
                    for (int e = 0; e < 4; e++) sc[j][e] = 16 * j + 8 * (e >> 1) < left ? (sc[j][e] + odd[e]) * scale2 : -INFINITY;
                }
                float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
                for (int j = 0; j < G16; j++)
#pragma unroll
                    for (int e = 0; e < 4; e++) mx[e & 1] = fmaxf(mx[e & 1], sc[j][e]);
                // Mostly no score passes its reference by MOVE_PAST, and then nobody need know the maximum.
                if (__any_sync(0xffffffffu, mx[0] > m[0] + MOVE_PAST || mx[1] > m[1] + MOVE_PAST)) {
#pragma unroll
                    for (int x = 4; x < 32; x <<= 1) {
                        mx[0] = fmaxf(mx[0], __shfl_xor_sync(0xffffffffu, mx[0], x));
                        mx[1] = fmaxf(mx[1], __shfl_xor_sync(0xffffffffu, mx[1], x));
                    }
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        if (!(mx[e] > m[e] + MOVE_PAST)) continue;
                        const float keep = m[e] == -INFINITY ? 0.0f : hw_exp2(m[e] - mx[e]);
                        m[e] = mx[e];
                        l[e] *= keep;
#pragma unroll
                        for (int j = 0; j < HD / 16; j++) {
                            o[j][e] *= keep;
                            o[j][2 + e] *= keep;
                        }
                    }
                }
                const float nm[2] = {m[0] == -INFINITY ? 0.0f : m[0], m[1] == -INFINITY ? 0.0f : m[1]};  // every score -inf: e 0
#pragma unroll
                for (int j = 0; j < G16; j++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        sc[j][e] = hw_exp2(sc[j][e] - nm[e & 1]);
                        l[e & 1] += sc[j][e];  // the lane's positions' alone
                    }
#pragma unroll
                for (int s = 0; s < G16; s++) {
                    // e^T as the second operand: each 8 x 8 block turned over among the lanes.
                    uint32_t h0, h1, l0, l1;
                    split_pack(sc[s][0], sc[s][1], h0, l0);
                    split_pack(sc[s][2], sc[s][3], h1, l1);
                    h0 = turn8(h0);
                    h1 = turn8(h1);
                    l0 = turn8(l0);
                    l1 = turn8(l1);
#pragma unroll
                    for (int j = 0; j < HD / 16; j++) {
                        uint32_t va[4];
                        ldmatrix_x4_trans(va, vs + own_at<HD>(16 * s + (mi >> 1) * 8 + rr, 2 * j + (mi & 1)));
                        mma_bf16(o[j], va, h0, h1);
                        mma_bf16(o[j], va, l0, l1);
                    }
                }
            }
            __syncwarp();  // the next piece's copies go into the same stages
#pragma unroll
            for (int e = 0; e < 2; e++) {
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) l[e] += __shfl_xor_sync(0xffffffffu, l[e], x);
                const int head = 2 * t4 + e;
                if (head >= group) continue;
                const size_t to = ((size_t)row * heads + kv * group + head) * pieces + np + piece;
#pragma unroll
                for (int j = 0; j < HD / 16; j++) {
                    out.o[to * HD + 16 * j + g] = o[j][e];
                    out.o[to * HD + 16 * j + 8 + g] = o[j][2 + e];
                }
                if (g == 0) *reinterpret_cast<float2 *>(out.ml + to * 2) = make_float2(m[e], l[e]);
            }
        }
    }
}

// ---- shared pieces, bf16 ------------------------------------------------------------------------------
// A block an SM, over units of a piece, a KV head and NT tiles of up to 128 queries, query m of a tile being
// head m % group of row m / group of the tile's rows, against the piece's
// keys in tiles of 128. Twelve warps (eight for one tile; warp 3 has no part):
//   warps 0 and 2  TMA: Q and the K tiles, and the V tiles, page by page (boxes of the largest of
//              128, 64, 32 and 16 positions that divides a page) into STAGES stages of
//              128-byte-swizzled halves of 64 dimensions; values past the prefix in its last tile set to
//              zero (0 x NaN is NaN). Two warps, as a copy's issue takes about 110 clocks: 16 to a tile
//              of K or V for pages of 16 (8 KiB of HD = 128 each);
//   warp 1     TMEM and the MMAs: S_j = Q K_j^T (M = 128, N = 128), O += P_j V_j (N = HD; P in TMEM, V
//              read MN-major), the tile's next S ahead of its PV so that the softmax runs under it;
//   warps 4-7  (and 8-11)  the softmax of a tile, a thread to a query: P_j = 2^(S_j scale - mref) as bf16
//              into TMEM against a reference that moves only when a tile's maximum passes it by 2^8 (O
//              then rescaled in place), the same pass as the prefill's attention kernel. P is rounded to
//              bf16 for the product (by 2^-8 of its value at most; the errors of many keys average out);
//              its sum l is of the f32 values.
// HD = 64: two tiles, which share the keys' copies, each with S, P and O in 256 columns. HD = 128: one tile
// with two S buffers (S 2 x 128, P 64, O 128), as two tiles do not fit TMEM's 512 columns.
// The softmax warps take registers from the first four (setmaxnreg).
// A tile of 128 keys takes about 2400 clocks (hd 64: 3400 for two tiles of queries), of which a softmax thread's
// exponentials and sums are 1400, its waits and TMEM's loads and stores the rest. No unit is near its rate: hd 128 (hd 64)
// has the tensor cores busy 22% (11%) of the time, the exponentials' pipe 31% (34%), L2 at 21% (7%) and
// HBM at 25% (3%) of theirs. The chain of S, softmax, P and PV with its waits bounds a tile. Storing a unit's partials
// takes 5000 clocks. Alone, from cold caches: 128 rows of 16 heads over 2 of 64 behind 8191 positions 18.1 us, 64 rows
// of 32 over 8 of 128 behind 16384 35.6 us (256 units over 148 SMs: two rounds, the second for 108).
// Every wait is bounded (the context's error word, then the block runs out).
template <int HD>
struct Pfx {
    static constexpr int NT = HD == 64 ? 2 : 1, HALVES = HD / 64, STAGES = HD == 64 ? 3 : 2;
    static constexpr int THREADS = 128 + 128 * NT, SB = HD == 64 ? 1 : 2;
    // Registers a thread: at launch, of warps 0-3 and of the softmax warps (the same sum).
    static constexpr int REGS = HD == 64 ? 136 : 144, FEW = 72, MANY = HD == 64 ? 168 : 216;
    static_assert(FEW + NT * MANY == (1 + NT) * REGS, "setmaxnreg draws on the launch's registers");
    static constexpr uint32_t HALF = 128 * 64 * 2, TILE = HALF * HALVES;  // 128 rows x 64 dimensions; x HD
    static constexpr uint32_t Q = 0, K = NT * TILE, V = K + STAGES * TILE, STAGE = V + STAGES * TILE;  // STAGE: 4 KiB a softmax warp
    static constexpr uint32_t SMEM = STAGE + NT * 4 * 4096 + 1024;
    static constexpr TG_DEVICE uint32_t s_col(int h, int j) { return NT == 2 ? 256 * h : 128 * (j & 1); }
    static constexpr TG_DEVICE uint32_t p_col(int h) { return NT == 2 ? 256 * h + 128 : 256; }
    static constexpr TG_DEVICE uint32_t o_col(int h) { return NT == 2 ? 256 * h + 192 : 320; }
};
// Two f32 fused multiply-adds, or adds, in one issue.
TG_DEVICE float2 fma2(float2 a, float2 b, float2 c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;"
        : "=l"(d)
        : "l"(*reinterpret_cast<const uint64_t *>(&a)), "l"(*reinterpret_cast<const uint64_t *>(&b)),
          "l"(*reinterpret_cast<const uint64_t *>(&c)));
    return *reinterpret_cast<const float2 *>(&d);
}
TG_DEVICE float2 add2(float2 a, float2 b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;"
        : "=l"(d)
        : "l"(*reinterpret_cast<const uint64_t *>(&a)), "l"(*reinterpret_cast<const uint64_t *>(&b)));
    return *reinterpret_cast<const float2 *>(&d);
}
TG_DEVICE float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
template <int HD>
__global__ void __launch_bounds__(Pfx<HD>::THREADS) __maxnreg__(Pfx<HD>::REGS)
    prefix_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                  const __grid_constant__ CUtensorMap vmap, tg_params p, const uint32_t *__restrict__ at,
                  const uint32_t *__restrict__ shared, Partials out, uint32_t pieces, uint32_t box, uint32_t *err) {
    using C = Pfx<HD>;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const uint32_t base = smem_u32(smem);
    __shared__ __align__(8) uint64_t bq_full, bq_empty, bk_full[C::STAGES], bk_empty[C::STAGES], bv_full[C::STAGES], bv_empty[C::STAGES];
    __shared__ __align__(8) uint64_t bs_full[C::NT * C::SB], bp_full[C::NT], bo_full[C::NT], bv_clear;
    __shared__ uint32_t tmem_slot;
    __shared__ int gave_up;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, tid = threadIdx.x;
    const int heads = p.heads, kvh = p.kv_heads, group = heads / kvh, tile_rows = 128 / group;
    const int tiles = ((int)p.rows + tile_rows - 1) / tile_rows, pairs = (tiles + C::NT - 1) / C::NT;
    const uint32_t size = shared_piece(p), np = shared_pieces(p), units = np * pairs * kvh;
    auto B = [](uint64_t &b) { return smem_u32(&b); };

    if (tid == 0) {
        gave_up = 0;
        mbar_init(B(bq_full), 1);
        mbar_init(B(bq_empty), 1);
        for (int i = 0; i < C::STAGES; i++) {
            mbar_init(B(bk_full[i]), 1);
            mbar_init(B(bk_empty[i]), 1);
            mbar_init(B(bv_full[i]), 1);
            mbar_init(B(bv_empty[i]), 1);
        }
        for (int i = 0; i < C::NT * C::SB; i++) mbar_init(B(bs_full[i]), 1);
        for (int i = 0; i < C::NT; i++) {
            mbar_init(B(bp_full[i]), 128);  // P_j in TMEM, S_j read and O rescaled
            mbar_init(B(bo_full[i]), 1);
        }
        mbar_init(B(bv_clear), 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (tid == 32) {
        prefetch_map(&kmap);
        prefetch_map(&qmap);
        prefetch_map(&vmap);
    }
    // The rows of a Q tile that no query fills (a group that does not divide 128) are zero.
    const int blank = 128 - tile_rows * group;
    for (int i = tid; i < C::NT * C::HALVES * blank * 8; i += C::THREADS)
        *reinterpret_cast<uint4 *>(smem + C::Q + i / (blank * 8) * C::HALF + (tile_rows * group + i / 8 % blank) * 128 + (i % 8) * 16) =
            make_uint4(0u, 0u, 0u, 0u);
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)),
                     "r"(512u)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    pdl_wait();
    pdl_launch_dependents();

    // A unit: a piece of the prefix, a KV head, NT tiles of queries. The roles walk the block's units each by itself;
    // `t` counts the tiles of keys over all of them (stages, and their barriers' phases).
    struct Unit {
        uint32_t piece, begin, keys;
        int kv, tile0, nt, n;
    };
    auto unit = [&](uint32_t u) {
        Unit x;
        x.piece = u % np;
        x.tile0 = (int)(u / np % pairs) * C::NT;
        x.kv = (int)(u / np / pairs);
        x.nt = min(C::NT, tiles - x.tile0);
        x.begin = x.piece * size;
        x.keys = min(size, p.first - x.begin);
        x.n = (int)((x.keys + 127) / 128);
        return x;
    };
    const bool values = warp == 2;
    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::FEW));
        if (warp == 0 || values) {
            // A lane to a copy: one half of the dimensions, one box of positions; the pages' numbers a tile ahead.
            const int boxes = 128 / (int)box, seg = lane % boxes, half = lane / boxes;
            uint64_t *full = values ? bv_full : bk_full, *empty = values ? bv_empty : bk_empty;
            const CUtensorMap *map = values ? &vmap : &kmap;
            int t = 0, done = 0, last_clear = -1;  // last_clear: the tile whose values were last cleared
            for (uint32_t u = blockIdx.x; u < units; u += gridDim.x, done++) {
                const Unit x = unit(u);
                auto page_of = [&](int j) {
                    const uint32_t in = j * 128 + seg * box;
                    uint32_t id = in < x.keys ? __ldg(shared + (x.begin + in) / p.capacity) : 0u;
                    if (id >= p.slots) {
                        atomicExch(err, ERR_BAD_INDEX);
                        id = 0;
                    }
                    return id;
                };
                uint32_t id = page_of(0);
                for (int j = 0; j < x.n; j++, t++) {
                    const int b = t % C::STAGES, live = min(128, (int)x.keys - j * 128), segs = (live + (int)box - 1) / (int)box;
                    const uint32_t pos = x.begin + j * 128 + seg * box, next = page_of(j + 1);
                    mbar_wait(B(empty[b]), ((t / C::STAGES) & 1) ^ 1, err, &gave_up);
                    if (lane == 0) mbar_arrive_expect_tx(B(full[b]), C::HALVES * segs * box * 128);
                    __syncwarp();
                    if (half < C::HALVES && seg < segs)
                        tma_load_3d(base + (values ? C::V : C::K) + b * C::TILE + half * C::HALF + seg * box * 128, map, half * 64,
                                    (int)(pos % p.capacity), (int)(id * kvh + x.kv), B(full[b]));
                    id = next;
                    if (warp == 0 && j == 0) {
                        // Q, once the unit before has all of its S.
                        mbar_wait(B(bq_empty), (done & 1) ^ 1, err, &gave_up);
                        if (lane == 0) {
                            mbar_arrive_expect_tx(B(bq_full), x.nt * C::HALVES * tile_rows * group * 128);
                            for (int h = 0; h < x.nt; h++)
                                for (int c = 0; c < C::HALVES; c++)
                                    tma_load_3d(base + C::Q + h * C::TILE + c * C::HALF, &qmap, c * 64, x.kv * group, (x.tile0 + h) * tile_rows, B(bq_full));
                        }
                        __syncwarp();
                    }
                }
                if (values && x.keys % 128) {
                    const int b = (t - 1) % C::STAGES, keep = (int)(x.keys % 128);
                    mbar_wait(B(bv_full[b]), ((t - 1) / C::STAGES) & 1, err, &gave_up);
                    // The clear before has been used: its stage's next copy waited for that, or else this does.
                    if (last_clear >= 0 && t - 1 < last_clear + C::STAGES)
                        mbar_wait(B(bv_empty[last_clear % C::STAGES]), (last_clear / C::STAGES) & 1, err, &gave_up);
                    last_clear = t - 1;
                    uint8_t *vt = smem + C::V + b * C::TILE;
                    for (int i = lane; i < C::HALVES * (128 - keep) * 8; i += 32) {
                        const int c = i / ((128 - keep) * 8), r = keep + i / 8 % (128 - keep);  // a swizzled row is 128 whole bytes
                        *reinterpret_cast<uint4 *>(vt + c * C::HALF + r * 128 + (i % 8) * 16) = make_uint4(0u, 0u, 0u, 0u);
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // for the tensor cores' reads
                    __syncwarp();
                    if (lane == 0) mbar_arrive(B(bv_clear));
                }
            }
            // Every copy has landed before the block can end.
            for (int i = t > C::STAGES ? t - C::STAGES : 0; i < t; i++) mbar_wait(B(full[i % C::STAGES]), (i / C::STAGES) & 1, err, &gave_up);
            if (warp == 0) mbar_wait(B(bq_full), (done - 1) & 1, err, &gave_up);
        } else if (warp == 1) {
            if (lane == 0) {
                constexpr uint32_t idesc_s = bf16_idesc(128, 128);
                constexpr uint32_t idesc_o = bf16_idesc(128, HD) | (1u << 16);  // B (V) MN-major
                int t0 = 0, done = 0, cleared = 0, seen[2] = {0, 0};  // seen: the tiles of keys each tile of queries has had
                for (uint32_t u = blockIdx.x; u < units; u += gridDim.x, done++) {
                    const Unit x = unit(u);
                    auto issue_s = [&](int j, int h) {
                        const uint32_t kt = base + C::K + ((t0 + j) % C::STAGES) * C::TILE, qt = base + C::Q + h * C::TILE;
                        const int at_s = seen[h] + j;
#pragma unroll
                        for (int i = 0; i < HD / 16; i++)
                            tc_mma(tmem + C::s_col(h, at_s), sw128_desc(qt + (i / 4) * C::HALF + (i % 4) * 32),
                                   sw128_desc(kt + (i / 4) * C::HALF + (i % 4) * 32), idesc_s, i > 0 ? 1u : 0u);
                        tc_commit(B(bs_full[h * C::SB + (C::SB - 1) * (at_s & 1)]));
                    };
                    auto wait_k = [&](int j) {
                        mbar_wait(B(bk_full[(t0 + j) % C::STAGES]), ((t0 + j) / C::STAGES) & 1, err, &gave_up);
                        tc_fence_after();
                    };
                    mbar_wait(B(bq_full), done & 1, err, &gave_up);
                    // S_j is issued: its keys, and after the last one the queries, may be overwritten once it is done.
                    auto issued_s = [&](int j) {
                        tc_commit(B(bk_empty[(t0 + j) % C::STAGES]));
                        if (j == x.n - 1) tc_commit(B(bq_empty));
                    };
                    for (int j = 0; j < C::SB && j < x.n; j++) {
                        wait_k(j);
                        for (int h = 0; h < x.nt; h++) issue_s(j, h);
                        issued_s(j);
                    }
                    for (int j = 0; j < x.n; j++) {
                        const int b = (t0 + j) % C::STAGES, next = j + C::SB;  // the S whose buffer S_j leaves free
                        const uint32_t v = base + C::V + b * C::TILE;
                        for (int h = 0; h < x.nt; h++) {
                            // P_j in TMEM, S_j read, and O rescaled to the query's reference (or the unit's before stored).
                            mbar_wait(B(bp_full[h]), (seen[h] + j) & 1, err, &gave_up);
                            tc_fence_after();
                            if (C::SB == 1 && next < x.n) {
                                if (h == 0) wait_k(next);
                                issue_s(next, h);
                                if (h == x.nt - 1) issued_s(next);
                            }
                            if (h == 0) {
                                mbar_wait(B(bv_full[b]), ((t0 + j) / C::STAGES) & 1, err, &gave_up);
                                if (j == x.n - 1 && x.keys % 128) mbar_wait(B(bv_clear), cleared++ & 1, err, &gave_up);
                                tc_fence_after();
                            }
#pragma unroll
                            for (int i = 0; i < 8; i++)
                                tc_mma_ts(tmem + C::o_col(h), tmem + C::p_col(h) + 8 * i, mn_desc(v + i * 2048, C::HALF), idesc_o,
                                          (j > 0 || i > 0) ? 1u : 0u);
                            tc_commit(B(bo_full[h]));
                        }
                        tc_commit(B(bv_empty[b]));
                        if (C::SB == 2 && next < x.n) {
                            wait_k(next);
                            issue_s(next, 0);
                            issued_s(next);
                        }
                    }
                    t0 += x.n;
                    for (int h = 0; h < x.nt; h++) seen[h] += x.n;
                }
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::MANY));
        const int h = warp / 4 - 1, quad = warp & 3, m = quad * 32 + lane;
        const uint32_t lanes = tmem + ((uint32_t)(quad * 32) << 16);
        const float scale2 = 1.4426950408889634f / sqrtf((float)HD);  // log2(e) / sqrt(hd)
        int t = 0;  // the tiles of keys this tile of queries has had
        for (uint32_t u = blockIdx.x; u < units; u += gridDim.x) {
            const Unit x = unit(u);
            if (h < x.nt) {
                float mref = -INFINITY, l = 0.0f;
                // 64 scores of S_j, past the prefix -inf.
                auto scores = [&](int j, int c, float (&sv)[64]) {
                    uint32_t r[4][16];
#pragma unroll
                    for (int i = 0; i < 4; i++) tmem_ld16_nowait(lanes + C::s_col(h, t) + (uint32_t)(c + 16 * i), r[i]);
                    tmem_wait_ld();
#pragma unroll
                    for (int i = 0; i < 64; i++) sv[i] = __uint_as_float(r[i / 16][i % 16]);
                    const int live = (int)x.keys - j * 128 - c;
                    if (live < 64) {
#pragma unroll
                        for (int i = 0; i < 64; i++)
                            if (i >= live) sv[i] = -INFINITY;
                    }
                };
                for (int j = 0; j < x.n; j++, t++) {
                    mbar_wait(B(bs_full[h * C::SB + (C::SB - 1) * (t & 1)]), (t / C::SB) & 1, err, &gave_up);
                    tc_fence_after();
                    // P_j against mref into TMEM with its sum, the tile's raw maximum alongside; P_j takes P_{j-1}'s place once
                    // PV_{j-1} has read it. (The first tile's first half of keys gives the first reference.) Where the maximum
                    // has passed a reference by MOVE_PAST, O (with PV_{j-1} in it) is rescaled, a query that keeps its
                    // reference times 1, and the warp's pass runs again from S_j.
                    float a = 1.0f, sum;
                    for (bool again = false;; again = true) {
                        float2 sums[4];
#pragma unroll
                        for (int i = 0; i < 4; i++) sums[i] = make_float2(0.0f, 0.0f);
                        float mx[2] = {-INFINITY, -INFINITY};
                        const float2 scale22 = make_float2(scale2, scale2);
#pragma unroll
                        for (int c = 0; c < 128; c += 64) {
                            float sv[64];
                            scores(j, c, sv);
                            if (c == 0 && j == 0 && !again) {
                                float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                                for (int i = 0; i < 64; i += 2) top[(i / 2) % 4] = max3(top[(i / 2) % 4], sv[i], sv[i + 1]);
                                mref = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * scale2;
                            }
                            const float nm = mref != -INFINITY ? -mref : -INFINITY;  // every score -inf: P comes out 0
                            const float2 neg_m = make_float2(nm, nm);
                            uint32_t pk[2][16];
#pragma unroll
                            for (int i = 0; i < 64; i += 2) {
                                mx[(i / 2) % 2] = max3(mx[(i / 2) % 2], sv[i], sv[i + 1]);
                                const float2 e = fma2(make_float2(sv[i], sv[i + 1]), scale22, neg_m);
                                const float p0 = hw_exp2(e.x), p1 = hw_exp2(e.y);
                                sums[(i / 2) % 4] = add2(sums[(i / 2) % 4], make_float2(p0, p1));
                                pk[i / 32][(i / 2) % 16] = fa::pack_bf16(p0, p1);
                            }
                            if (c == 0 && !again && j > 0) {
                                mbar_wait(B(bo_full[h]), (t - 1) & 1, err, &gave_up);
                                tc_fence_after();
                            }
                            tmem_st16(lanes + C::p_col(h) + (uint32_t)(c / 2), pk[0]);
                            tmem_st16(lanes + C::p_col(h) + (uint32_t)(c / 2) + 16, pk[1]);
                        }
                        sum = ((sums[0].x + sums[0].y) + (sums[1].x + sums[1].y)) + ((sums[2].x + sums[2].y) + (sums[3].x + sums[3].y));
                        const float m_tile = fmaxf(mx[0], mx[1]) * scale2;
                        const bool move = m_tile > mref + MOVE_PAST;
                        if (again || !__any_sync(0xffffffffu, move)) break;
                        a = move && mref != -INFINITY ? hw_exp2(mref - m_tile) : 1.0f;
                        if (move) mref = m_tile;
                        tmem_wait_st();
#pragma unroll 1
                        for (int c = 0; c < HD && j > 0; c += 16) {
                            uint32_t o[16];
                            tmem_ld16_nowait(lanes + C::o_col(h) + c, o);
                            tmem_wait_ld();
#pragma unroll
                            for (int e = 0; e < 16; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * a);
                            tmem_st16(lanes + C::o_col(h) + c, o);
                        }
                        tmem_wait_st();
                    }
                    tmem_wait_st();
                    tc_fence_before();
                    l = __fmaf_rn(l, a, sum);
                    mbar_arrive(B(bp_full[h]));
                }
                mbar_wait(B(bo_full[h]), (t - 1) & 1, err, &gave_up);
                tc_fence_after();
                // The partials, where a query is one: O as it stands in TMEM by way of shared memory, so that a store covers
                // whole lines of four queries; references and sums. A row of the stage is 32 values, its 16-byte pieces
                // turned by the row.
                const int row = (x.tile0 + h) * tile_rows + m / group;
                const bool real = m < tile_rows * group && row < (int)p.rows;
                const uint64_t to = real ? ((uint64_t)row * heads + x.kv * group + m % group) * pieces + x.piece : ~0ull;
                float4 *stage = reinterpret_cast<float4 *>(smem + C::STAGE + (warp - 4) * 4096);
                float4 *dst[8];
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const uint64_t q = __shfl_sync(0xffffffffu, to, 4 * i + lane / 8);
                    dst[i] = q != ~0ull ? reinterpret_cast<float4 *>(out.o + q * HD) + lane % 8 : nullptr;
                }
                uint32_t o[2][16];
                tmem_ld16_nowait(lanes + C::o_col(h), o[0]);
                tmem_ld16_nowait(lanes + C::o_col(h) + 16, o[1]);
#pragma unroll
                for (int c = 0; c < HD; c += 32) {
                    tmem_wait_ld();
#pragma unroll
                    for (int e = 0; e < 8; e++)
                        stage[lane * 8 + (e ^ (lane & 7))] =
                            make_float4(__uint_as_float(o[e / 4][e % 4 * 4]), __uint_as_float(o[e / 4][e % 4 * 4 + 1]),
                                        __uint_as_float(o[e / 4][e % 4 * 4 + 2]), __uint_as_float(o[e / 4][e % 4 * 4 + 3]));
                    if (c + 32 < HD) {
                        tmem_ld16_nowait(lanes + C::o_col(h) + c + 32, o[0]);
                        tmem_ld16_nowait(lanes + C::o_col(h) + c + 48, o[1]);
                    }
                    __syncwarp();
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const int q = 4 * i + lane / 8;
                        if (dst[i]) dst[i][c / 4] = stage[q * 8 + (lane % 8 ^ (q & 7))];
                    }
                    __syncwarp();
                }
                if (real) *reinterpret_cast<float2 *>(out.ml + to * 2) = make_float2(mref, l);
                tc_fence_before();
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
}

// Joins the partials of a row's head, a block to it: 16 bytes of a piece's o to a lane, the pieces over the
// block's groups of HD / 4 lanes, all loads of a row of up to JOIN_DEEP pieces a group in flight at once; the
// groups' sums are then added in order. References are in base 2 for bf16, natural for f32. Latency-bound, then by
// the partials' bytes: from cold caches 2048 heads of 16 + up to 6 pieces of 64 (10 MB) 10.2 us, of 16 + up to 8 of 128 (22 MB) 11.2.
constexpr int JOIN_THREADS = 128, JOIN_DEEP = 8;

template <typename T, int HD>
__global__ void __launch_bounds__(JOIN_THREADS)
    join_kernel(tg_params p, const uint32_t *__restrict__ at, Partials in, uint32_t np, uint32_t pieces, T *__restrict__ out) {
    constexpr int LANES = HD / 4, GROUPS = JOIN_THREADS / LANES;
    __shared__ __align__(16) float4 acc_s[GROUPS][LANES];
    __shared__ float m_s[GROUPS], l_s[GROUPS];
    pdl_launch_dependents();
    pdl_wait();
    const uint64_t item = blockIdx.x;
    const int group = threadIdx.x / LANES, d = threadIdx.x % LANES;
    uint32_t length, seq;
    if (!paged_row(p, at, (int)(item / p.heads), length, seq, nullptr)) return;
    const uint32_t n = np + (length + OWN_PIECE - 1) / OWN_PIECE;
    const float2 *ml = reinterpret_cast<const float2 *>(in.ml) + item * pieces;
    const float4 *o = reinterpret_cast<const float4 *>(in.o + item * pieces * HD) + d;
    auto power = [](float x) { return sizeof(T) == 2 ? exp2f(x) : expf(x); };
    float m = -INFINITY, l = 0.0f;
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (uint32_t i0 = group; i0 < n; i0 += GROUPS * JOIN_DEEP) {
        float2 part[JOIN_DEEP];
        float4 x[JOIN_DEEP];
#pragma unroll
        for (int i = 0; i < JOIN_DEEP; i++) {
            const uint32_t piece = i0 + i * GROUPS;
            part[i] = piece < n ? ml[piece] : make_float2(-INFINITY, 0.0f);
            x[i] = piece < n ? o[(size_t)piece * LANES] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
        float next = m;
#pragma unroll
        for (int i = 0; i < JOIN_DEEP; i++) next = fmaxf(next, part[i].x);
        const float keep = m == -INFINITY ? 0.0f : power(m - next);
        m = next;
        l *= keep;
        acc = make_float4(acc.x * keep, acc.y * keep, acc.z * keep, acc.w * keep);
#pragma unroll
        for (int i = 0; i < JOIN_DEEP; i++) {
            const float e = part[i].x == -INFINITY ? 0.0f : power(part[i].x - m);
            l = __fmaf_rn(part[i].y, e, l);
            acc = make_float4(__fmaf_rn(x[i].x, e, acc.x), __fmaf_rn(x[i].y, e, acc.y), __fmaf_rn(x[i].z, e, acc.z), __fmaf_rn(x[i].w, e, acc.w));
        }
    }
    // The groups' references joined, then their sums.
    if (d == 0) m_s[group] = m;
    __syncthreads();
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < GROUPS; i++) top = fmaxf(top, m_s[i]);
    const float e = m == -INFINITY ? 0.0f : power(m - top);
    if (d == 0) l_s[group] = l * e;
    acc_s[group][d] = make_float4(acc.x * e, acc.y * e, acc.z * e, acc.w * e);
    __syncthreads();
    if (group) return;
    l = 0.0f;
    acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < GROUPS; i++) {
        const float4 x = acc_s[i][d];
        l += l_s[i];
        acc = make_float4(acc.x + x.x, acc.y + x.y, acc.z + x.z, acc.w + x.w);
    }
    T *dst = out + item * HD + 4 * d;
    const float4 r = make_float4(__fdiv_rn(acc.x, l), __fdiv_rn(acc.y, l), __fdiv_rn(acc.z, l), __fdiv_rn(acc.w, l));
    if constexpr (sizeof(T) == 2)
        *reinterpret_cast<uint2 *>(dst) = make_uint2(fa::pack_bf16(r.x, r.y), fa::pack_bf16(r.z, r.w));
    else
        *reinterpret_cast<float4 *>(dst) = r;
}

// A 3-D map over bf16 [outer][rows][hd]: boxes of 64 dimensions x `box_rows` x `box_outer` in the 128-byte
// swizzle; what lies past the tensor reads as zero.
bool map_heads(CUtensorMap *map, const void *ptr, uint64_t rows, uint64_t outer, uint64_t hd, uint32_t box_rows, uint32_t box_outer) {
    EncodeTiledFn fn = encode_fn();
    if (!fn) return false;
    cuuint64_t dims[3] = {hd, rows, outer}, strides[2] = {hd * 2, rows * hd * 2};
    cuuint32_t box[3] = {64, box_rows, box_outer}, steps[3] = {1, 1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void *>(ptr), dims, strides, box, steps,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Opts a kernel into its shared memory with all of an SM's as shared memory, so that blocks of the next kernel, which
// start under it and wait, find room there.
template <typename F>
cudaError_t with_all_smem(F kernel, size_t bytes) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    return e != cudaSuccess ? e : cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
}

template <typename T, int HD>
cudaError_t attend(const tg_params &p, const void *q_, const void *k_, const void *v_, const uint32_t *at, const uint32_t *table,
                   const uint32_t *shared, void *work, void *out_, uint32_t *err, int sm_count, Enqueue &run) {
    const uint64_t all = all_pieces(p), items = (uint64_t)p.rows * p.heads;
    if (all > 0x7fffffffu || p.kv_heads > 65535) return cudaErrorNotSupported;
    const T *q = static_cast<const T *>(q_), *k = static_cast<const T *>(k_), *v = static_cast<const T *>(v_);
    T *out = static_cast<T *>(out_);
    float *o = reinterpret_cast<float *>((reinterpret_cast<uintptr_t>(work) + 255) & ~uintptr_t(255));
    const Partials part{o, o + items * all * HD};
    const uint32_t np = shared_pieces(p), pieces = (uint32_t)all;
    auto join = [=](cudaStream_t s) {
        return launch_pdl(join_kernel<T, HD>, dim3((unsigned)items), dim3(JOIN_THREADS), 0, s, p, at, part, np, pieces, out);
    };
    if constexpr (sizeof(T) == 4) {
        auto kernel = f32_kernel<HD>;
        constexpr int SMEM = F32<HD, F32_QUERIES>::FLOATS * sizeof(float);
        static_assert(SMEM >= F32<HD, MAX_GROUP>::FLOATS * sizeof(float), "the own pieces' too");
        const cudaError_t e = with_all_smem(kernel, SMEM);
        if (e != cudaSuccess) return e;
        const uint32_t tile_rows = F32_QUERIES / (p.heads / p.kv_heads), far = np * ((p.rows + tile_rows - 1) / tile_rows);
        const uint64_t blocks = far + (uint64_t)p.rows * (pieces - np);
        run = [=](cudaStream_t s) {
            const cudaError_t e = launch_pdl(kernel, dim3((unsigned)blocks, p.kv_heads), dim3(F32_THREADS), SMEM, s, p, q, k, v, at, table,
                                             shared, part, np, pieces, far, err);
            return e != cudaSuccess ? e : join(s);
        };
    } else {
        using C = Pfx<HD>;
        cudaError_t e = with_all_smem(own_kernel<HD>, OWN_SMEM);
        if (e != cudaSuccess) return e;
        const uint64_t most = ((uint64_t)p.rows * p.kv_heads * (pieces - np) + OWN_WARPS - 1) / OWN_WARPS;
        const unsigned own_blocks = (unsigned)std::min<uint64_t>(most, (uint64_t)sm_count * OWN_BLOCKS);
        auto own = [=](cudaStream_t s) {
            const cudaError_t e = launch_pdl(own_kernel<HD>, dim3(own_blocks), dim3(OWN_WARPS * 32), OWN_SMEM, s, p, q, k, v, at, table, part, np,
                                             pieces, err);
            return e != cudaSuccess ? e : join(s);
        };
        if (np == 0) {
            run = own;
            return cudaSuccess;
        }
        const uint32_t group = p.heads / p.kv_heads, tile_rows = 128 / group;
        const uint32_t box = p.capacity % 128 == 0 ? 128 : p.capacity % 64 == 0 ? 64 : p.capacity % 32 == 0 ? 32 : 16;
        CUtensorMap qm, km, vm;
        if (!map_heads(&qm, q, p.heads, p.rows, HD, group, tile_rows) ||
            !map_heads(&km, k, p.capacity, (uint64_t)p.slots * p.kv_heads, HD, box, 1) ||
            !map_heads(&vm, v, p.capacity, (uint64_t)p.slots * p.kv_heads, HD, box, 1))
            return cudaErrorInvalidValue;
        e = with_all_smem(prefix_kernel<HD>, C::SMEM);
        if (e != cudaSuccess) return e;
        // Its setmaxnreg counts on the launch's registers: fewer would be waited for without end.
        cudaFuncAttributes a;
        e = cudaFuncGetAttributes(&a, prefix_kernel<HD>);
        if (e != cudaSuccess) return e;
        if (a.numRegs != C::REGS) return cudaErrorInvalidConfiguration;
        const uint64_t tiles = (p.rows + tile_rows - 1) / tile_rows, units = np * ((tiles + C::NT - 1) / C::NT) * p.kv_heads;
        if (units > 0x7fffffffu) return cudaErrorNotSupported;
        const unsigned blocks = (unsigned)std::min<uint64_t>(units, (uint64_t)sm_count);
        run = [=](cudaStream_t s) {
            const cudaError_t e = launch_pdl(prefix_kernel<HD>, dim3(blocks), dim3(C::THREADS), C::SMEM, s, qm, km, vm, p, at, shared, part, pieces,
                                             box, err);
            return e != cudaSuccess ? e : own(s);
        };
    }
    return cudaSuccess;
}

}  // namespace

uint64_t attention_pages_work(const tg_params &p) {
    return (uint64_t)p.rows * p.heads * all_pieces(p) * (p.head_dim + 2) * sizeof(float) + 256;
}

cudaError_t make_attention_pages(const tg_params &p, const void *q, const void *k, const void *v, const uint32_t *at,
                                 const uint32_t *table, const uint32_t *shared, void *work, void *out, uint32_t *err,
                                 int sm_count, Enqueue &run) {
    if (p.dtype == TG_BF16)
        return p.head_dim == 64 ? attend<bf16, 64>(p, q, k, v, at, table, shared, work, out, err, sm_count, run)
                                : attend<bf16, 128>(p, q, k, v, at, table, shared, work, out, err, sm_count, run);
    return p.head_dim == 64 ? attend<float, 64>(p, q, k, v, at, table, shared, work, out, err, sm_count, run)
                            : attend<float, 128>(p, q, k, v, at, table, shared, work, out, err, sm_count, run);
}

}  // namespace tg
