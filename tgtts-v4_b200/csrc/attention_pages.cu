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
// (own_kernel), bound by the caches' bytes. f32 runs on the CUDA cores (pieces_kernel).
#include "mma_common.cuh"
#include "tc_common.cuh"

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

// The partials in the work buffer, from its first 256-byte boundary: o f32 [rows][heads][pieces][hd], then
// m, l f32 [rows][heads][pieces][2].
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

// ---- own pieces, bf16 ---------------------------------------------------------------------------------
// A block to a piece of a row's own positions for one KV head, a quarter of it to each of four warps:
// the group's query heads are the rows of mma.sync.m16n8k16 (S = q K^T, O = e V with e split into bf16
// hi + lo), keys and values gathered from their pages into the warp's shared memory by cp.async, all in
// flight at once. The block joins its warps' partials in shared memory. References are in base 2.
constexpr int OWN_WARPS = 4;
constexpr int own_row(int hd) { return hd + fa::PAD; }  // bf16 of a shared row
constexpr int own_smem(int hd) { return 2 * (int)own_piece(hd) * own_row(hd) * 2; }

template <int HD>
__global__ void __launch_bounds__(OWN_WARPS * 32)
    own_kernel(tg_params p, const bf16 *__restrict__ q, const bf16 *__restrict__ k, const bf16 *__restrict__ v,
               const uint32_t *__restrict__ at, const uint32_t *__restrict__ table, Partials out, uint32_t np,
               uint32_t pieces, uint32_t *err) {
    using namespace fa;
    extern __shared__ __align__(128) unsigned char own_mem[];
    constexpr int W = own_piece(HD) / OWN_WARPS, ROW = own_row(HD), NT = W / 8, DT = HD / 8, VECS = HD / 8;
    // Behind prefix_kernel this one starts under it: that kernel lets it go once what comes before both has
    // ended (its own wait), and the two share nothing. A block still waits before it ends, for the join.
    if (np == 0) pdl_wait();
    pdl_launch_dependents();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
    const int kv = blockIdx.y, row = blockIdx.z, heads = p.heads, kvh = p.kv_heads, group = heads / kvh;
    uint32_t length, seq;
    if (!paged_row(p, at, row, length, seq, kv == 0 && blockIdx.x == 0 && threadIdx.x == 0 ? err : nullptr) ||
        (uint64_t)blockIdx.x * own_piece(HD) >= length) {
        pdl_wait();
        return;
    }
    bf16 *ks = reinterpret_cast<bf16 *>(own_mem) + (size_t)warp * 2 * W * ROW, *vs = ks + W * ROW;
    const uint32_t start = blockIdx.x * own_piece(HD) + warp * W;
    const int live = start < length ? (int)min(length - start, (uint32_t)W) : 0;  // positions of this warp
    float m = -INFINITY, l = 0.0f, o[DT][4];
#pragma unroll
    for (int j = 0; j < DT; j++) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.0f;
    if (live) {
        uint64_t from[W / 32];  // where positions lane, lane + 32, .. lie in the caches
#pragma unroll
        for (int i = 0; i < W / 32; i++) {
            const uint32_t pos = start + min(lane + 32 * i, live - 1);
            uint32_t id = __ldg(table + (size_t)seq * p.stride + pos / p.capacity);
            if (id >= p.slots) {
                atomicExch(err, ERR_BAD_INDEX);
                id = 0;
            }
            from[i] = (((uint64_t)id * kvh + kv) * p.capacity + pos % p.capacity) * HD;
        }
        auto gather = [&](bf16 *to, const bf16 *cache) {
#pragma unroll
            for (int i = 0; i < W * VECS / 32; i++) {
                const int r = i * (32 / VECS) + lane / VECS, c = lane % VECS;
                uint64_t src = __shfl_sync(0xffffffffu, from[(i * (32 / VECS)) / 32], r % 32);
                cp_async16(to + r * ROW + c * 8, cache + src + c * 8, r < live);
            }
            cp_async_commit();
        };
        gather(ks, k);
        gather(vs, v);
        // q of the group's heads: rows g < group of the products (rows past it, and 8 to 15, zero).
        uint32_t qf[HD / 16][4];
        const bf16 *qg = q + ((size_t)row * heads + kv * group + g) * HD + 2 * t4;
#pragma unroll
        for (int s = 0; s < HD / 16; s++) {
            qf[s][0] = g < group ? __ldg(reinterpret_cast<const uint32_t *>(qg + 16 * s)) : 0u;
            qf[s][2] = g < group ? __ldg(reinterpret_cast<const uint32_t *>(qg + 16 * s + 8)) : 0u;
            qf[s][1] = qf[s][3] = 0u;
        }
        cp_async_wait<1>();
        __syncwarp();
        const int mi = lane >> 3, rr = lane & 7;
        float sc[NT][4];
#pragma unroll
        for (int j = 0; j < NT; j++) sc[j][0] = sc[j][1] = sc[j][2] = sc[j][3] = 0.0f;
#pragma unroll
        for (int s = 0; s < HD / 16; s++)
#pragma unroll
            for (int j = 0; j < NT; j += 2) {
                uint32_t kb[4];
                ldmatrix_x4(kb, ks + (8 * j + (mi >> 1) * 8 + rr) * ROW + s * 16 + (mi & 1) * 8);
                mma_bf16(sc[j], qf[s], kb[0], kb[1]);
                mma_bf16(sc[j + 1], qf[s], kb[2], kb[3]);
            }
        const float scale2 = 1.4426950408889634f / sqrtf((float)HD);
#pragma unroll
        for (int j = 0; j < NT; j++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                sc[j][e] = 8 * j + 2 * t4 + e < live ? sc[j][e] * scale2 : -INFINITY;
                m = fmaxf(m, sc[j][e]);
            }
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
#pragma unroll
        for (int j = 0; j < NT; j++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                sc[j][e] = sc[j][e] == -INFINITY ? 0.0f : exp2f(sc[j][e] - m);
                l += sc[j][e];
            }
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
        cp_async_wait<0>();
        __syncwarp();
#pragma unroll
        for (int s = 0; s < W / 16; s++) {
            uint32_t ph[4], pl[4];
            split_pack(sc[2 * s][0], sc[2 * s][1], ph[0], pl[0]);
            split_pack(sc[2 * s + 1][0], sc[2 * s + 1][1], ph[2], pl[2]);
            ph[1] = ph[3] = pl[1] = pl[3] = 0u;
#pragma unroll
            for (int j = 0; j < DT; j += 2) {
                uint32_t vb[4];
                ldmatrix_x4_trans(vb, vs + (16 * s + (mi & 1) * 8 + rr) * ROW + 8 * j + (mi >> 1) * 8);
                mma_bf16(o[j], ph, vb[0], vb[1]);
                mma_bf16(o[j], pl, vb[0], vb[1]);
                mma_bf16(o[j + 1], ph, vb[2], vb[3]);
                mma_bf16(o[j + 1], pl, vb[2], vb[3]);
            }
        }
    }
    // The warps' partials joined in warp order (a warp past the row's length: m -inf, o zero).
    constexpr int G = MAX_GROUP;
    float *red = reinterpret_cast<float *>(own_mem);  // [OWN_WARPS][G][HD], then [OWN_WARPS][G][2]
    float *red_ml = red + OWN_WARPS * G * HD;
    __syncthreads();  // every warp is done with its keys and values
    if (g < group) {
        float *dst = red + (warp * G + g) * HD + 2 * t4;
#pragma unroll
        for (int j = 0; j < DT; j++) *reinterpret_cast<float2 *>(dst + 8 * j) = make_float2(o[j][0], o[j][1]);
        if (t4 == 0) *reinterpret_cast<float2 *>(red_ml + (warp * G + g) * 2) = make_float2(m, l);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < group * (HD / 4); i += OWN_WARPS * 32) {
        const int h = i / (HD / 4), d = 4 * (i % (HD / 4));
        float mx = -INFINITY, sum = 0.0f;
        float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int w = 0; w < OWN_WARPS; w++) mx = fmaxf(mx, red_ml[(w * G + h) * 2]);
#pragma unroll
        for (int w = 0; w < OWN_WARPS; w++) {
            const float mw = red_ml[(w * G + h) * 2], e = mw == -INFINITY ? 0.0f : exp2f(mw - mx);
            const float4 x = *reinterpret_cast<const float4 *>(red + (w * G + h) * HD + d);
            sum = __fmaf_rn(red_ml[(w * G + h) * 2 + 1], e, sum);
            acc = make_float4(__fmaf_rn(x.x, e, acc.x), __fmaf_rn(x.y, e, acc.y), __fmaf_rn(x.z, e, acc.z), __fmaf_rn(x.w, e, acc.w));
        }
        const size_t to = ((size_t)row * heads + kv * group + h) * pieces + np + blockIdx.x;
        *reinterpret_cast<float4 *>(out.o + to * HD + d) = acc;
        if (d == 0) *reinterpret_cast<float2 *>(out.ml + to * 2) = make_float2(mx, sum);
    }
    pdl_wait();
}

// ---- shared pieces, bf16 ------------------------------------------------------------------------------
// Block (piece, t, kv): NT tiles of up to 128 queries, query m of a tile being head m % group of row
// m / group of the tile's rows, against the piece's keys in tiles of 128. Ten warps (six for one tile):
//   warp 0     TMA: Q, then K and V tiles page by page (boxes of the largest of 128, 64, 32 and 16
//              positions that divides a page) into STAGES stages of 128-byte-swizzled halves of 64
//              dimensions; values past the prefix in its last tile set to zero (0 x NaN is NaN);
//   warp 1     TMEM and the MMAs: S_j = Q K_j^T (M = 128, N = 128), O += P_j V_j (N = HD; P in TMEM, V
//              read MN-major), the tile's next S ahead of its PV so that the softmax runs under it;
//   warps 2-5  (and 6-9) the softmax of a tile, a thread to a query: P_j = 2^(S_j scale - mref) as bf16
//              into TMEM against a reference that moves only when a tile's maximum passes it by 2^8 (O
//              then rescaled in place), the same pass as the prefill's attention kernel.
// HD = 64: two tiles, which share the keys' copies, each with S, P and O in 256 columns. HD = 128: one tile
// with two S buffers (S 2 x 128, P 64, O 128), as two tiles do not fit TMEM's 512 columns.
// Every wait is bounded (the context's error word, then the block runs out).
template <int HD>
struct Pfx {
    static constexpr int NT = HD == 64 ? 2 : 1, HALVES = HD / 64, STAGES = HD == 64 ? 3 : 2;
    static constexpr int THREADS = 64 + 128 * NT, SB = HD == 64 ? 1 : 2;
    static constexpr uint32_t HALF = 128 * 64 * 2, TILE = HALF * HALVES;  // 128 rows x 64 dimensions; x HD
    static constexpr uint32_t Q = 0, K = NT * TILE, V = K + STAGES * TILE, SMEM = V + STAGES * TILE + 1024;
    static constexpr TG_DEVICE uint32_t s_col(int h, int j) { return NT == 2 ? 256 * h : 128 * (j & 1); }
    static constexpr TG_DEVICE uint32_t p_col(int h) { return NT == 2 ? 256 * h + 128 : 256; }
    static constexpr TG_DEVICE uint32_t o_col(int h) { return NT == 2 ? 256 * h + 192 : 320; }
};
// How far (base 2) a tile's maximum may pass a query's reference before O and l are rescaled.
constexpr float MOVE_PAST = 8.0f;

// 2^x by the hardware's base-2 exponential (relative error about 2^-22); 2^-inf = 0.
TG_DEVICE float hw_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
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
// V's tile [keys][HD] as B = V^T: N along a row in chunks of 64 dimensions `chunk` bytes apart, K = keys
// down the rows in atoms of 8 keys x 128 bytes, 1024 bytes apart.
TG_DEVICE uint64_t mn_desc(uint32_t addr, uint32_t chunk) {
    return (uint64_t)((addr >> 4) & 0x3fff) | ((uint64_t)(chunk >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
           ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}

// 32 aligned bytes in one store: a whole sector.
TG_DEVICE void store8(float *dst, const uint32_t *v) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(dst), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]),
                 "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
}

template <int HD>
__global__ void __launch_bounds__(Pfx<HD>::THREADS, 1)
    prefix_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                  const __grid_constant__ CUtensorMap vmap, tg_params p, const uint32_t *__restrict__ at,
                  const uint32_t *__restrict__ shared, Partials out, uint32_t pieces, uint32_t box, uint32_t *err) {
    using C = Pfx<HD>;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const uint32_t base = smem_u32(smem);
    __shared__ __align__(8) uint64_t bq, bk_full[C::STAGES], bk_empty[C::STAGES], bv_full[C::STAGES], bv_empty[C::STAGES];
    __shared__ __align__(8) uint64_t bs_full[C::NT * C::SB], bp_full[C::NT], bo_full[C::NT], bv_clear;
    __shared__ uint32_t tmem_slot;
    __shared__ int gave_up;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, tid = threadIdx.x;
    const int kv = blockIdx.z, heads = p.heads, kvh = p.kv_heads, group = heads / kvh;
    const int tile_rows = 128 / group, tiles = ((int)p.rows + tile_rows - 1) / tile_rows;
    const int tile0 = blockIdx.y * C::NT, nt = min(C::NT, tiles - tile0);
    const uint32_t begin = blockIdx.x * shared_piece(p.first), keys = min(shared_piece(p.first), p.first - begin);
    const int n = (int)((keys + 127) / 128);
    const bool clear_v = keys % 128 != 0;
    auto B = [](uint64_t &b) { return smem_u32(&b); };

    if (tid == 0) {
        gave_up = 0;
        mbar_init(B(bq), 1);
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
    // The rows of a Q tile that no query fills (a group that does not divide 128) are zero.
    for (int i = tid; i < C::NT * C::HALVES * (128 - tile_rows * group) * 8; i += C::THREADS) {
        const int part = i / ((128 - tile_rows * group) * 8), r = tile_rows * group + i / 8 % (128 - tile_rows * group);
        *reinterpret_cast<uint4 *>(smem + C::Q + part * C::HALF + r * 128 + (i % 8) * 16) = make_uint4(0u, 0u, 0u, 0u);
    }
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

    if (warp == 0) {
        if (lane == 0) {
            mbar_arrive_expect_tx(B(bq), nt * C::HALVES * tile_rows * group * 128);
            for (int h = 0; h < nt; h++)
                for (int c = 0; c < C::HALVES; c++)
                    tma_load_3d(base + C::Q + h * C::TILE + c * C::HALF, &qmap, c * 64, kv * group, (tile0 + h) * tile_rows, B(bq));
        }
        // A lane to a copy: one half of the dimensions, one box of positions. Keys run a tile ahead of
        // values, as their stages come free earlier, and the pages' numbers a tile ahead of the keys.
        const int boxes = 128 / (int)box, seg = lane % boxes, half = lane / boxes;
        auto page_of = [&](int j) {
            const uint32_t in = j * 128 + seg * box;
            uint32_t id = in < keys ? __ldg(shared + (begin + in) / p.capacity) : 0u;
            if (id >= p.slots) {
                atomicExch(err, ERR_BAD_INDEX);
                id = 0;
            }
            return id;
        };
        auto load = [&](int j, uint32_t id, uint32_t dst, const CUtensorMap *map, uint64_t *full, uint64_t *empty) {
            const int b = j % C::STAGES, live = min(128, (int)keys - j * 128), segs = (live + (int)box - 1) / (int)box;
            const uint32_t pos = begin + j * 128 + seg * box;
            mbar_wait(B(empty[b]), ((j / C::STAGES) & 1) ^ 1, err, &gave_up);
            if (lane == 0) mbar_arrive_expect_tx(B(full[b]), C::HALVES * segs * box * 128);
            __syncwarp();
            if (half < C::HALVES && seg < segs)
                tma_load_3d(base + dst + b * C::TILE + half * C::HALF + seg * box * 128, map, half * 64, (int)(pos % p.capacity),
                            (int)(id * kvh + kv), B(full[b]));
        };
        uint32_t id = page_of(0), id1 = page_of(1);
        load(0, id, C::K, &kmap, bk_full, bk_empty);
        for (int j = 0; j < n; j++) {
            const uint32_t id2 = page_of(j + 2);
            if (j + 1 < n) load(j + 1, id1, C::K, &kmap, bk_full, bk_empty);
            load(j, id, C::V, &vmap, bv_full, bv_empty);
            id = id1;
            id1 = id2;
        }
        // Every copy has landed before the block can end.
        for (int j = n > C::STAGES ? n - C::STAGES : 0; j < n; j++) {
            mbar_wait(B(bk_full[j % C::STAGES]), (j / C::STAGES) & 1, err, &gave_up);
            mbar_wait(B(bv_full[j % C::STAGES]), (j / C::STAGES) & 1, err, &gave_up);
        }
        mbar_wait(B(bq), 0, err, &gave_up);
        if (clear_v) {
            uint8_t *vt = smem + C::V + ((n - 1) % C::STAGES) * C::TILE;
            const int keep = (int)(keys % 128);
            for (int i = lane; i < C::HALVES * (128 - keep) * 8; i += 32) {
                const int c = i / ((128 - keep) * 8), r = keep + i / 8 % (128 - keep);  // a swizzled row is 128 whole bytes
                *reinterpret_cast<uint4 *>(vt + c * C::HALF + r * 128 + (i % 8) * 16) = make_uint4(0u, 0u, 0u, 0u);
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // for the tensor cores' reads
            __syncwarp();
            if (lane == 0) mbar_arrive(B(bv_clear));
        }
    } else if (warp == 1) {
        if (lane == 0) {
            constexpr uint32_t idesc_s = bf16_idesc(128, 128);
            constexpr uint32_t idesc_o = bf16_idesc(128, HD) | (1u << 16);  // B (V) MN-major
            auto issue_s = [&](int j, int h) {
                const uint32_t kt = base + C::K + (j % C::STAGES) * C::TILE, qt = base + C::Q + h * C::TILE;
#pragma unroll
                for (int i = 0; i < HD / 16; i++)
                    tc_mma(tmem + C::s_col(h, j), sw128_desc(qt + (i / 4) * C::HALF + (i % 4) * 32),
                           sw128_desc(kt + (i / 4) * C::HALF + (i % 4) * 32), idesc_s, i > 0 ? 1u : 0u);
                tc_commit(B(bs_full[h * C::SB + (C::SB - 1) * (j & 1)]));
            };
            auto wait_k = [&](int j) {
                mbar_wait(B(bk_full[j % C::STAGES]), (j / C::STAGES) & 1, err, &gave_up);
                tc_fence_after();
            };
            mbar_wait(B(bq), 0, err, &gave_up);
            for (int j = 0; j < C::SB && j < n; j++) {
                wait_k(j);
                for (int h = 0; h < nt; h++) issue_s(j, h);
                tc_commit(B(bk_empty[j % C::STAGES]));
            }
            for (int j = 0; j < n; j++) {
                const int b = j % C::STAGES, next = j + C::SB;  // the S whose buffer S_j leaves free
                const uint32_t v = base + C::V + b * C::TILE;
                for (int h = 0; h < nt; h++) {
                    // P_j in TMEM, S_j read, and O rescaled to the query's reference.
                    mbar_wait(B(bp_full[h]), j & 1, err, &gave_up);
                    tc_fence_after();
                    if (C::SB == 1 && next < n) {
                        if (h == 0) wait_k(next);
                        issue_s(next, h);
                        if (h == nt - 1) tc_commit(B(bk_empty[next % C::STAGES]));
                    }
                    if (h == 0) {
                        mbar_wait(B(bv_full[b]), (j / C::STAGES) & 1, err, &gave_up);
                        if (clear_v && j == n - 1) mbar_wait(B(bv_clear), 0, err, &gave_up);
                        tc_fence_after();
                    }
#pragma unroll
                    for (int i = 0; i < 8; i++)
                        tc_mma_ts(tmem + C::o_col(h), tmem + C::p_col(h) + 8 * i, mn_desc(v + i * 2048, C::HALF), idesc_o,
                                  (j > 0 || i > 0) ? 1u : 0u);
                    tc_commit(B(bo_full[h]));
                }
                tc_commit(B(bv_empty[b]));
                if (C::SB == 2 && next < n) {
                    wait_k(next);
                    issue_s(next, 0);
                    tc_commit(B(bk_empty[next % C::STAGES]));
                }
            }
        }
    } else if ((warp - 2) / 4 < nt) {
        const int h = (warp - 2) / 4, quad = warp & 3, m = quad * 32 + lane;
        const uint32_t lanes = tmem + ((uint32_t)(quad * 32) << 16);
        const float scale2 = 1.4426950408889634f / sqrtf((float)HD);  // log2(e) / sqrt(hd)
        float mref = -INFINITY, l = 0.0f;
        for (int j = 0; j < n; j++) {
            mbar_wait(B(bs_full[h * C::SB + (C::SB - 1) * (j & 1)]), (j / C::SB) & 1, err, &gave_up);
            tc_fence_after();
            const int live = (int)keys - j * 128;
            // P_j against mref into TMEM with its sum, the tile's raw maximum alongside; P_j takes
            // P_{j-1}'s place once PV_{j-1} has read it, which the first pass waits for.
            auto p_pass = [&](float &mx, bool first) {
                float2 sum4[4];
#pragma unroll
                for (int e = 0; e < 4; e++) sum4[e] = make_float2(0.0f, 0.0f);
                float mxs[2] = {-INFINITY, -INFINITY};
                const float nm = mref != -INFINITY ? -mref : -INFINITY;  // every score -inf: P comes out 0
                const float2 scale22 = make_float2(scale2, scale2), neg_m = make_float2(nm, nm);
#pragma unroll
                for (int c2 = 0; c2 < 2; c2++) {
                    uint32_t r[4][16];
#pragma unroll
                    for (int c = 0; c < 4; c++) tmem_ld16_nowait(lanes + C::s_col(h, j) + (uint32_t)(c2 * 64 + c * 16), r[c]);
                    tmem_wait_ld();
                    float sv[64];
#pragma unroll
                    for (int c = 0; c < 64; c++) sv[c] = __uint_as_float(r[c / 16][c % 16]);
                    if (c2 * 64 + 64 > live) {
#pragma unroll
                        for (int c = 0; c < 64; c++)
                            if (c2 * 64 + c >= live) sv[c] = -INFINITY;
                    }
                    uint32_t pk[2][16];
#pragma unroll
                    for (int c = 0; c < 64; c += 2) {
                        mxs[(c / 2) % 2] = max3(mxs[(c / 2) % 2], sv[c], sv[c + 1]);
                        const float2 x = fma2(make_float2(sv[c], sv[c + 1]), scale22, neg_m);
                        const float p0 = hw_exp2(x.x), p1 = hw_exp2(x.y);
                        sum4[(c % 8) / 2] = add2(sum4[(c % 8) / 2], make_float2(p0, p1));
                        pk[c / 32][(c / 2) % 16] = fa::pack_bf16(p0, p1);
                    }
                    if (c2 == 0 && first && j > 0) {
                        mbar_wait(B(bo_full[h]), (j - 1) & 1, err, &gave_up);
                        tc_fence_after();
                    }
                    tmem_st16(lanes + C::p_col(h) + 32 * c2, pk[0]);
                    tmem_st16(lanes + C::p_col(h) + 32 * c2 + 16, pk[1]);
                }
                mx = fmaxf(mxs[0], mxs[1]);
                return ((sum4[0].x + sum4[0].y) + (sum4[1].x + sum4[1].y)) +
                       ((sum4[2].x + sum4[2].y) + (sum4[3].x + sum4[3].y));
            };
            if (j == 0) {  // no reference yet: the tile's maximum first
                float mxs[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int c4 = 0; c4 < 2; c4++) {
                    uint32_t r[4][16];
#pragma unroll
                    for (int c = 0; c < 4; c++) tmem_ld16_nowait(lanes + C::s_col(h, 0) + (uint32_t)(c4 * 64 + c * 16), r[c]);
                    tmem_wait_ld();
                    const int in = min(live - c4 * 64, 64);
#pragma unroll
                    for (int c = 0; c < 64; c += 2)
                        mxs[(c / 2) % 4] = max3(mxs[(c / 2) % 4], c < in ? __uint_as_float(r[c / 16][c % 16]) : -INFINITY,
                                                c + 1 < in ? __uint_as_float(r[c / 16][c % 16 + 1]) : -INFINITY);
                }
                mref = fmaxf(fmaxf(mxs[0], mxs[1]), fmaxf(mxs[2], mxs[3])) * scale2;
            }
            float a = 1.0f, mx;
            float sum = p_pass(mx, true);
            const float m_tile = mx * scale2;
            const bool move = m_tile > mref + MOVE_PAST;
            if (__any_sync(0xffffffffu, move)) {
                // A query of the warp moves: O (with PV_{j-1} in it) rescaled, a query that keeps its
                // reference times 1, then the warp's P_j again from S_j, still in TMEM.
                a = move && mref != -INFINITY ? hw_exp2(mref - m_tile) : 1.0f;
                if (move) mref = m_tile;
                tmem_wait_st();
#pragma unroll
                for (int c = 0; c < HD / 16; c++) {
                    uint32_t o[16];
                    tmem_ld16_nowait(lanes + C::o_col(h) + c * 16, o);
                    tmem_wait_ld();
#pragma unroll
                    for (int e = 0; e < 16; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * a);
                    tmem_st16(lanes + C::o_col(h) + c * 16, o);
                }
                tmem_wait_st();
                sum = p_pass(mx, false);
            }
            tmem_wait_st();
            tc_fence_before();
            l = __fmaf_rn(l, a, sum);
            mbar_arrive(B(bp_full[h]));
        }
        mbar_wait(B(bo_full[h]), (n - 1) & 1, err, &gave_up);
        tc_fence_after();
        // The partial of query m, where it is one: O as it stands in TMEM, and its reference and sum.
        const int row = (tile0 + h) * tile_rows + m / group;
        const bool real = m < tile_rows * group && row < (int)p.rows;
        const size_t to = (((size_t)(real ? row : 0) * heads + kv * group + m % group) * pieces + blockIdx.x);
#pragma unroll
        for (int c = 0; c < HD / 16; c++) {
            uint32_t o[16];
            tmem_ld16_nowait(lanes + C::o_col(h) + c * 16, o);
            tmem_wait_ld();
            if (real) {
                store8(out.o + to * HD + c * 16, o);
                store8(out.o + to * HD + c * 16 + 8, o + 8);
            }
        }
        if (real) *reinterpret_cast<float2 *>(out.ml + to * 2) = make_float2(mref, l);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
}

// Joins a row's partials, a warp to a head, in piece order. References are in base 2 for bf16, natural for f32.
// A lane takes four dimensions of every LANES-th piece, so that a warp has several pieces' loads in flight; the
// lanes' sums are added by a butterfly.
template <typename T, int HD>
__global__ void __launch_bounds__(128)
    join_kernel(tg_params p, const uint32_t *__restrict__ at, Partials in, uint32_t np, uint32_t pieces, T *__restrict__ out) {
    constexpr int LANES = 32 / (HD / 4);  // pieces at once
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31, d = 4 * (lane % (HD / 4)), of = lane / (HD / 4);
    const uint64_t item = (uint64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (item >= (uint64_t)p.rows * p.heads) return;
    uint32_t length, seq;
    if (!paged_row(p, at, (int)(item / p.heads), length, seq, nullptr)) return;
    const uint32_t n = np + (length + own_piece(HD) - 1) / own_piece(HD);
    const float2 *ml = reinterpret_cast<const float2 *>(in.ml) + item * pieces;
    const float *o = in.o + item * pieces * HD + d;
    float m = -INFINITY, l = 0.0f;
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    auto power = [](float x) { return sizeof(T) == 2 ? exp2f(x) : expf(x); };
    for (uint32_t i0 = 0; i0 < n; i0 += 32) {
        // 32 pieces at once: a lane holds one's reference and sum.
        const float2 part = i0 + lane < n ? ml[i0 + lane] : make_float2(-INFINITY, 0.0f);
        const float next = fmaxf(m, warp_max(part.x)), keep = m == -INFINITY ? 0.0f : power(m - next);
        const float e = part.x == -INFINITY ? 0.0f : power(part.x - next);
        m = next;
        l = __fmaf_rn(l, keep, warp_sum(part.y * e));
        acc = make_float4(acc.x * keep, acc.y * keep, acc.z * keep, acc.w * keep);
        const uint32_t count = min(n - i0, 32u);
#pragma unroll 4
        for (uint32_t i = 0; i < count; i += LANES) {
            const float w = __shfl_sync(0xffffffffu, e, (i + of) & 31);
            if (i + of >= count) continue;
            const float4 x = *reinterpret_cast<const float4 *>(o + (size_t)(i0 + i + of) * HD);
            acc = make_float4(__fmaf_rn(x.x, w, acc.x), __fmaf_rn(x.y, w, acc.y), __fmaf_rn(x.z, w, acc.z), __fmaf_rn(x.w, w, acc.w));
        }
    }
    if (LANES > 1) {
        acc.x += __shfl_xor_sync(0xffffffffu, acc.x, 16);
        acc.y += __shfl_xor_sync(0xffffffffu, acc.y, 16);
        acc.z += __shfl_xor_sync(0xffffffffu, acc.z, 16);
        acc.w += __shfl_xor_sync(0xffffffffu, acc.w, 16);
    }
    if (of) return;
    T *dst = out + item * HD + d;
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

template <typename T, int HD>
cudaError_t attend(const tg_params &p, const void *q, const void *k, const void *v, const uint32_t *at, const uint32_t *table,
                   const uint32_t *shared, void *work, void *out, uint32_t *err, cudaStream_t s) {
    const uint64_t pieces = all_pieces(p), items = (uint64_t)p.rows * p.heads;
    if (pieces > 0x7fffffffu || p.kv_heads > 65535) return cudaErrorNotSupported;
    float *o = reinterpret_cast<float *>((reinterpret_cast<uintptr_t>(work) + 255) & ~uintptr_t(255));
    Partials part{o, o + items * pieces * HD};
    const uint32_t np = shared_pieces(p.first);
    cudaError_t e = cudaSuccess;
    if constexpr (sizeof(T) == 2) {
        using C = Pfx<HD>;
        if (np) {
            const uint32_t group = p.heads / p.kv_heads, tile_rows = 128 / group;
            const uint32_t box = p.capacity % 128 == 0 ? 128 : p.capacity % 64 == 0 ? 64 : p.capacity % 32 == 0 ? 32 : 16;
            CUtensorMap qm, km, vm;
            if (!map_heads(&qm, q, p.heads, p.rows, HD, group, tile_rows) ||
                !map_heads(&km, k, p.capacity, (uint64_t)p.slots * p.kv_heads, HD, box, 1) ||
                !map_heads(&vm, v, p.capacity, (uint64_t)p.slots * p.kv_heads, HD, box, 1))
                return cudaErrorInvalidValue;
            e = with_smem(prefix_kernel<HD>, C::SMEM);
            if (e != cudaSuccess) return e;
            const uint32_t tiles = (p.rows + tile_rows - 1) / tile_rows;
            e = launch_pdl(prefix_kernel<HD>, dim3(np, (tiles + C::NT - 1) / C::NT, p.kv_heads), dim3(C::THREADS), C::SMEM, s, qm, km,
                           vm, p, at, shared, part, (uint32_t)pieces, box, err);
            if (e != cudaSuccess) return e;
        }
        e = with_smem(own_kernel<HD>, own_smem(HD));
        if (e != cudaSuccess) return e;
        e = launch_pdl(own_kernel<HD>, dim3((unsigned)(pieces - np), p.kv_heads, p.rows), dim3(OWN_WARPS * 32), own_smem(HD), s, p,
                       (const T *)q, (const T *)k, (const T *)v, at, table, part, np, (uint32_t)pieces, err);
    } else {
        e = launch_pdl(pieces_kernel<T, HD>, dim3((unsigned)pieces, p.kv_heads, p.rows), dim3(CHUNK), 0, s, p, (const T *)q, (const T *)k,
                       (const T *)v, at, table, shared, part, np, (uint32_t)pieces, err);
    }
    if (e != cudaSuccess) return e;
    return launch_pdl(join_kernel<T, HD>, dim3((unsigned)((items + 3) / 4)), dim3(128), 0, s, p, at, part, np, (uint32_t)pieces, (T *)out);
}

}  // namespace

uint64_t attention_pages_work(const tg_params &p) {
    if (p.head_dim == 0 || p.head_dim > 16384) return 0;
    return (uint64_t)p.rows * p.heads * all_pieces(p) * (p.head_dim + 2) * sizeof(float) + 256;
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
