// adapters.hip — low-rank adapters of many requests at once beside a shared projection (rows_gemm.hip's dense layers), forward and
// backward, on rows of float32, bfloat16 or float16.
//
//     t[r]   = A_a x[r]                                  (rank)           a = the adapter of row r
//     out[r] = base[r] + s_a B_a t[r]                    (n)              rows without an adapter: out = base, t = 0
// and for the gradients, with u[r] = B_a^T dy[r]:
//     dx[r]  = base[r] + s_a A_a^T u[r]                  the forward on (dy, B^T, A^T): one kernel serves both
//     dA_a   = s_a sum over the rows of a of u[r] x[r]^T,   dB_a = s_a sum dy[r] t[r]^T
// t, u and every sum are float32; base + s B t is rounded once.
//
// The rows of an adapter are found by a plan in device memory (a stable counting sort of the rows by adapter, built by three small
// kernels, one for up to PL_ROWS rows; the host never learns the counts): tiles of 16 rows and chunks of AD_CHUNK rows, each of one
// adapter.
#include "jm_elem.h"
#include "jm_rows.h"

namespace jm {

// ------------------------------------------------------------------------------------------------ plan
constexpr int PL_ROWS = 4096;        // rows of a counting block
constexpr int PL_THREADS = 1024;
constexpr int PL_MAX_ADAPTERS = 1023;        // + the rows without an adapter: one counter a thread
constexpr int AD_TILE = 16;          // rows of a tile
constexpr int AD_CHUNK = 1024;       // rows of a chunk (weight gradients)
constexpr int AD_MAX_ROWS = 1 << 30, AD_MAX_WIDTH = 1 << 20;        // tile counts, grids and per-adapter element counts stay in range

struct PlanLayout {                  // offsets in ints; header: [0] tiles, [1] chunks
    size_t order, tiles, chunks, chunk_first, hist, total;
    int max_tiles, max_chunks, blocks;
};
static PlanLayout plan_layout(int m, int adapters) {
    PlanLayout l;
    l.blocks = divup(m, PL_ROWS);
    l.max_tiles = divup(m, AD_TILE) + (adapters + 1 < m ? adapters + 1 : m);
    l.max_chunks = divup(m, AD_CHUNK) + (adapters < m ? adapters : m);
    l.order = 4;
    l.tiles = align_up(l.order + (size_t)m, 4);
    l.chunks = l.tiles + 4 * (size_t)l.max_tiles;
    l.chunk_first = l.chunks + 4 * (size_t)l.max_chunks;
    l.hist = align_up(l.chunk_first + (size_t)adapters + 1, 4);
    l.total = l.hist + (size_t)l.blocks * (size_t)(adapters + 1);
    return l;
}

__device__ __forceinline__ int plan_bucket(const int* ids, long long row, int adapters) {
    const int id = ids[row];
    return (id >= 0 && id < adapters) ? id : adapters;          // the last bucket: rows without an adapter
}

// exclusive prefix sums over the block's threads of three counters at once
__device__ __forceinline__ void plan_scan3(int (&v)[3], int (*wave_tot)[3]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int incl[3];
#pragma unroll
    for (int q = 0; q < 3; ++q) incl[q] = wave_incl_scan_i32_dpp(v[q]);
    if (lane == 63)
#pragma unroll
        for (int q = 0; q < 3; ++q) wave_tot[wave][q] = incl[q];
    __syncthreads();
#pragma unroll
    for (int q = 0; q < 3; ++q) {
        int before = 0;
        for (int w = 0; w < wave; ++w) before += wave_tot[w][q];
        v[q] = before + incl[q] - v[q];
    }
    __syncthreads();
}

// bucket counts -> starts, and the tables of tiles and chunks.  `count`: this thread's bucket count (thread = bucket).
// first[b] = {row start, first tile, first chunk} of bucket b, first[adapters + 1] = the totals.
__device__ void plan_tables(int count, int adapters, int (*first)[3], int (*wave_tot)[3], int* __restrict__ plan, size_t o_tiles, size_t o_chunks,
                            size_t o_chunk_first) {
    const int b = threadIdx.x;
    int v[3] = {count, (count + AD_TILE - 1) / AD_TILE, b < adapters ? (count + AD_CHUNK - 1) / AD_CHUNK : 0};
    const int mine[3] = {v[0], v[1], v[2]};
    plan_scan3(v, wave_tot);
    if (b <= adapters)
#pragma unroll
        for (int q = 0; q < 3; ++q) {
            first[b][q] = v[q];
            if (b == adapters) first[b + 1][q] = v[q] + mine[q];
        }
    __syncthreads();
    if (b <= adapters) plan[o_chunk_first + b] = first[b][2];
    const int nt = first[adapters + 1][1], nc = first[adapters + 1][2];
    if (b == 0) { plan[0] = nt; plan[1] = nc; plan[2] = 0; plan[3] = 0; }
    // a table entry finds its bucket by bisection: the last bucket whose first tile is <= t
    for (int t = b; t < nt; t += PL_THREADS) {
        int lo = 0, hi = adapters;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (first[mid][1] <= t) lo = mid; else hi = mid - 1;
        }
        const int start = first[lo][0] + (t - first[lo][1]) * AD_TILE;
        *reinterpret_cast<int4*>(plan + o_tiles + 4 * (size_t)t) = make_int4(lo < adapters ? lo : -1, start, min(AD_TILE, first[lo + 1][0] - start), 0);
    }
    for (int t = b; t < nc; t += PL_THREADS) {
        int lo = 0, hi = adapters - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (first[mid][2] <= t) lo = mid; else hi = mid - 1;
        }
        const int start = first[lo][0] + (t - first[lo][2]) * AD_CHUNK;
        *reinterpret_cast<int4*>(plan + o_chunks + 4 * (size_t)t) = make_int4(lo, start, min(AD_CHUNK, first[lo + 1][0] - start), 0);
    }
}

// rows row0 .. row0 + rows - 1 to their places, in row order within a bucket: next[b] = the bucket's next place.  A wave ranks its 64
// rows by matching ids, the waves' counts (bytes: at most 64) are added in wave order.
__device__ void plan_scatter(const int* __restrict__ ids, long long row0, int rows, int adapters, int* next, unsigned char (*wcnt)[PL_THREADS],
                             int* __restrict__ order) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int r = 0; r < rows; r += PL_THREADS) {
        __syncthreads();
        for (int q = threadIdx.x; q < 16 * PL_THREADS / 4; q += PL_THREADS) reinterpret_cast<unsigned*>(wcnt)[q] = 0u;
        __syncthreads();
        const bool ok = r + (int)threadIdx.x < rows;
        const int b = ok ? plan_bucket(ids, row0 + r + threadIdx.x, adapters) : -1;
        int rank = 0;
        unsigned long long left = __ballot(ok);
        while (left) {
            const int lead = __shfl(b, (int)__builtin_ctzll(left));
            const unsigned long long same = __ballot(b == lead) ;
            if (b == lead) rank = mbcnt(same);
            if (lane == 0) wcnt[wave][lead] = (unsigned char)__popcll(same);
            left &= ~same;
        }
        __syncthreads();
        if (ok) {
            int at = next[b] + rank;
            for (int w = 0; w < wave; ++w) at += wcnt[w][b];
            order[at] = (int)(row0 + r + threadIdx.x);
        }
        __syncthreads();
        if ((int)threadIdx.x <= adapters) {
            int add = 0;
#pragma unroll
            for (int w = 0; w < 16; ++w) add += wcnt[w][threadIdx.x];
            next[threadIdx.x] += add;
        }
    }
}

// ids of one counting block counted in LDS; whole: the block is all there is and the plan is finished here (one launch)
template <bool WHOLE>
__global__ void __launch_bounds__(PL_THREADS)
adapter_plan_count_kernel(int m, int adapters, const int* __restrict__ ids, int* __restrict__ plan, size_t o_order, size_t o_tiles, size_t o_chunks,
                          size_t o_chunk_first, size_t o_hist) {
    __shared__ int cnt[PL_THREADS];
    __shared__ int first[WHOLE ? PL_THREADS + 2 : 1][3], wave_tot[16][3];
    __shared__ __attribute__((aligned(4))) unsigned char wcnt[WHOLE ? 16 : 1][PL_THREADS];
    cnt[threadIdx.x] = 0;
    __syncthreads();
    const long long row0 = (long long)blockIdx.x * PL_ROWS;
    const int rows = (int)min((long long)PL_ROWS, m - row0);
    for (int r = threadIdx.x; r < rows; r += PL_THREADS) atomicAdd(&cnt[plan_bucket(ids, row0 + r, adapters)], 1);
    __syncthreads();
    if constexpr (WHOLE) {
        plan_tables(cnt[threadIdx.x], adapters, first, wave_tot, plan, o_tiles, o_chunks, o_chunk_first);
        __syncthreads();
        if ((int)threadIdx.x <= adapters) cnt[threadIdx.x] = first[threadIdx.x][0];
        plan_scatter(ids, 0, rows, adapters, cnt, wcnt, plan + o_order);
    } else {
        if ((int)threadIdx.x <= adapters) plan[o_hist + (size_t)blockIdx.x * (adapters + 1) + threadIdx.x] = cnt[threadIdx.x];
    }
}

// the blocks' counts -> every block's first place of every bucket (in place), and the tables
__global__ void __launch_bounds__(PL_THREADS)
adapter_plan_tables_kernel(int blocks, int adapters, int* __restrict__ plan, size_t o_tiles, size_t o_chunks, size_t o_chunk_first, size_t o_hist) {
    __shared__ int first[PL_THREADS + 2][3], wave_tot[16][3];
    const int b = threadIdx.x;
    int total = 0;
    if (b <= adapters)
        for (int k = 0; k < blocks; ++k) total += plan[o_hist + (size_t)k * (adapters + 1) + b];
    plan_tables(total, adapters, first, wave_tot, plan, o_tiles, o_chunks, o_chunk_first);
    if (b <= adapters) {
        int at = first[b][0];
        for (int k = 0; k < blocks; ++k) {
            int* h = plan + o_hist + (size_t)k * (adapters + 1) + b;
            const int c = *h;
            *h = at;
            at += c;
        }
    }
}

__global__ void __launch_bounds__(PL_THREADS)
adapter_plan_scatter_kernel(int m, int adapters, const int* __restrict__ ids, int* __restrict__ plan, size_t o_order, size_t o_hist) {
    __shared__ int next[PL_THREADS];
    __shared__ __attribute__((aligned(4))) unsigned char wcnt[16][PL_THREADS];
    if ((int)threadIdx.x <= adapters) next[threadIdx.x] = plan[o_hist + (size_t)blockIdx.x * (adapters + 1) + threadIdx.x];
    const long long row0 = (long long)blockIdx.x * PL_ROWS;
    plan_scatter(ids, row0, (int)min((long long)PL_ROWS, m - row0), adapters, next, wcnt, plan + o_order);
}

// ------------------------------------------------------------------------------------------------ the product
struct Adapt {
    int m, k, n, rank;
    const int* plan; size_t o_order, o_tiles;
    const void* x; long long ldx;
    const void* a; const void* b;        // (adapters, rank, k), (adapters, n, rank)
    const float* scales;
    const void* base; long long ldb;     // NULL: zero
    void* out; long long ldo;
    float* t;                            // (m, rank) or NULL
    int copy;                            // base and out are not the same rows: rows without an adapter are copied
};

// A wave owns a tile of 16 rows.  First t (rank x 16 rows) = A x^T over k, 32 elements a step, both operands straight from memory into
// the registers of the 16 x 16 products; t crosses the lanes through LDS; then out (n x 16 rows), 64 channels at a time: the rows of B
// are permuted so that a lane ends up with 16 consecutive channels of its row.
// t enters the second product as the sum of two values of the 16-bit type (16 significant bits in bfloat16, 22 in float16, where the
// row is scaled by a power of two first: t may leave float16's range although out does not); as it is in float32.
template <int TY, int RB>
__global__ void __launch_bounds__(64)
adapter_rows_kernel(Adapt p) {
    typedef typename Elem<TY>::T T;
    typedef typename Elem<TY>::V8 V8;
    constexpr int RS = (RB * 16 + 31) / 32;              // 32-wide steps over the rank
    constexpr int LD = RS * 32 + 4;
    __shared__ __attribute__((aligned(16))) float ts[16][LD];
    if ((int)blockIdx.x >= p.plan[0]) return;
    const int4 tile = *reinterpret_cast<const int4*>(p.plan + p.o_tiles + 4 * (size_t)blockIdx.x);
    const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
    const int ad = tile.x, count = tile.z;
    const bool live = i < count;
    const size_t row = (size_t)p.plan[p.o_order + tile.y + min(i, count - 1)];
    const T* base = p.base ? (const T*)p.base + row * p.ldb : nullptr;
    T* out = (T*)p.out + row * p.ldo;
    if (ad < 0) {                                        // rows without an adapter
        if (!live) return;
        if (p.copy)
            for (int c = g; c < p.n; c += 4) out[c] = base ? base[c] : (T)0.f;
        if (p.t)
            for (int c = g; c < p.rank; c += 4) p.t[row * p.rank + c] = 0.f;
        return;
    }
    const T* x = (const T*)p.x + row * p.ldx;
    const T* A = (const T*)p.a + (size_t)ad * p.rank * p.k;
    const T* B = (const T*)p.b + (size_t)ad * p.n * p.rank;
    const float scale = p.scales[ad];

    f32x4 acc[RB];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) acc[rb] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int k0 = 0; k0 < p.k; k0 += 32) {
        const int kk = k0 + 8 * g, left = p.k - kk;
        const V8 xv = load8_upto<V8>(x + kk, left);
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
            const V8 av = load8_upto<V8>(A + (size_t)min(rb * 16 + i, p.rank - 1) * p.k + kk, left);
            acc[rb] = mma16(acc[rb], av, xv);            // D: column = row i of the tile, rows = rank index 4 g + q
        }
    }
    // rank indices beyond the rank hold copies of the last one: zeroed, so that the second product contracts zeros there
#pragma unroll
    for (int rb = 0; rb < 2 * RS; ++rb) {
        f32x4 v = f32x4{0.f, 0.f, 0.f, 0.f};
        if (rb < RB)
#pragma unroll
            for (int q = 0; q < 4; ++q) v[q] = rb * 16 + 4 * g + q < p.rank ? acc[rb < RB ? rb : 0][q] : 0.f;
        *reinterpret_cast<f32x4*>(&ts[i][rb * 16 + 4 * g]) = v;
    }
    __syncthreads();
    if (p.t && live)
        for (int c = g; c < p.rank; c += 4) p.t[row * p.rank + c] = ts[i][c];

    float back = scale;
    V8 hi[RS], lo[RS];
    float fit = 1.f;
    if constexpr (TY == JM_F16) {
        float top = 0.f;
#pragma unroll
        for (int s = 0; s < RS; ++s)
#pragma unroll
            for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(ts[i][s * 32 + 8 * g + e]));
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        const int ex = min(max((int)(__float_as_uint(top) >> 23) - 127, -100), 126);      // the row's values become less than 2
        fit = __uint_as_float((unsigned)(127 - ex) << 23);
        back = scale * __uint_as_float((unsigned)(127 + ex) << 23);
    }
#pragma unroll
    for (int s = 0; s < RS; ++s)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float v = ts[i][s * 32 + 8 * g + e] * fit;
            const T h = (T)v;
            hi[s][e] = h;
            if constexpr (TY != JM_F32) lo[s][e] = (T)(fabsf((float)h) < __builtin_inff() ? v - (float)h : 0.f);
        }

    for (int n0 = 0; n0 < p.n; n0 += 64) {
        f32x4 d[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            d[j] = f32x4{0.f, 0.f, 0.f, 0.f};
            const T* Br = B + (size_t)min(n0 + (i >> 2) * 16 + j * 4 + (i & 3), p.n - 1) * p.rank;
#pragma unroll
            for (int s = 0; s < RS; ++s) {
                const int r0 = s * 32 + 8 * g;
                const V8 bv = load8_upto<V8>(Br + r0, p.rank - r0);
                d[j] = mma16(d[j], bv, hi[s]);
                if constexpr (TY != JM_F32) d[j] = mma16(d[j], bv, lo[s]);
            }
        }
        if (live) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int c = n0 + 16 * g + 4 * j + q;
                    if (c < p.n) out[c] = (T)((base ? (float)base[c] : 0.f) + back * d[j][q]);
                }
        }
    }
}

// (count, rows, cols) -> (count, cols, rows)
template <typename T>
__global__ void __launch_bounds__(256)
adapter_transpose_kernel(int rows, int cols, const T* __restrict__ src, T* __restrict__ dst) {
    __shared__ T tile[32][33];
    const size_t off = (size_t)blockIdx.z * rows * cols;
    const int c0 = blockIdx.x * 32, r0 = blockIdx.y * 32, tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    for (int q = ty; q < 32; q += 8)
        if (r0 + q < rows && c0 + tx < cols) tile[q][tx] = src[off + (size_t)(r0 + q) * cols + c0 + tx];
    __syncthreads();
    for (int q = ty; q < 32; q += 8)
        if (c0 + q < cols && r0 + tx < rows) dst[off + (size_t)(c0 + q) * rows + r0 + tx] = tile[tx][q];
}

// ------------------------------------------------------------------------------------------------ gradients of A and B
struct AdaptGrad {
    int m, k, n, rank, adapters;
    const int* plan; size_t o_order, o_chunks, o_chunk_first;
    const void* x; long long ldx;
    const unsigned char* codes; int ldc; const unsigned char* exps; int blocks;      // x kept in 8 bits (x NULL)
    const void* dy; long long lddy;
    const float *t, *u;                  // (m, rank)
    const float* scales;
    float* part;                         // per chunk: (rank, k) of dA, then (n, rank) of dB
    void *da, *db;
};

// 4 consecutive channels of a row, zeros beyond the width
template <int TY, bool KEPT>
__device__ __forceinline__ f32x4 grad_load4(const AdaptGrad& p, const void* src, long long ld, size_t row, int c, int width) {
    f32x4 v;
    if (KEPT) {
        const float s = __uint_as_float((unsigned)p.exps[row * p.blocks + min(c, width - 1) / 32] << 23);       // scale bytes: 27 .. 247
        unsigned w = 0;
        if (c < width) w = *reinterpret_cast<const unsigned*>(p.codes + row * p.ldc + c);
        const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false);
        const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
        v = f32x4{lo[0] * s, lo[1] * s, hi[0] * s, hi[1] * s};
    } else {
        const typename Elem<TY>::T* q = (const typename Elem<TY>::T*)src + row * ld + c;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = c + e < width ? (float)q[e] : 0.f;
    }
    return v;
}

// Workgroup = (chunk of one adapter's rows) x (64 channels of x, then of dy) x (64 rank indices); its four waves take every fourth group
// of four rows, 16 x 16 x 4 float32 products of T (t or u: rank) with X (channels), and add their tiles in wave order through LDS.
template <int TY, bool KEPT, int RB>
__global__ void __launch_bounds__(256)
adapter_wgrad_kernel(AdaptGrad p) {
    __shared__ f32x4 red[3][RB * 4][64];
    if ((int)blockIdx.x >= p.plan[1]) return;
    const int4 chunk = *reinterpret_cast<const int4*>(p.plan + p.o_chunks + 4 * (size_t)blockIdx.x);
    const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4, wave = threadIdx.x >> 6;
    const int tk = (p.k + 63) / 64;
    const bool isA = (int)blockIdx.y < tk;
    const int c0 = (isA ? (int)blockIdx.y : (int)blockIdx.y - tk) * 64, width = isA ? p.k : p.n, r0 = blockIdx.z * 64;
    const float* T = isA ? p.u : p.t;
    f32x4 acc[RB][4];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[rb][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int q = wave * 4; q < chunk.z; q += 16) {
        const bool ok = q + g < chunk.z;
        const size_t row = (size_t)p.plan[p.o_order + chunk.y + min(q + g, chunk.z - 1)];
        f32x4 xv;
        if (isA) xv = grad_load4<TY, KEPT>(p, p.x, p.ldx, row, c0 + 4 * i, width);
        else xv = grad_load4<TY, false>(p, p.dy, p.lddy, row, c0 + 4 * i, width);
#pragma unroll
        for (int e = 0; e < 4; ++e) xv[e] = ok ? xv[e] : 0.f;
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
            const float tv = ok ? T[row * p.rank + min(r0 + rb * 16 + i, p.rank - 1)] : 0.f;
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[rb][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(tv, xv[j], acc[rb][j], 0, 0, 0);
        }
    }
    if (wave > 0)
#pragma unroll
        for (int rb = 0; rb < RB; ++rb)
#pragma unroll
            for (int j = 0; j < 4; ++j) red[wave - 1][rb * 4 + j][lane] = acc[rb][j];
    __syncthreads();
    if (wave > 0) return;
#pragma unroll
    for (int w = 0; w < 3; ++w)
#pragma unroll
        for (int rb = 0; rb < RB; ++rb)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[rb][j] += red[w][rb * 4 + j][lane];
    // D: rows = rank index 4 g + q, column i = channel c0 + 4 i + j
    float* part = p.part + (size_t)blockIdx.x * p.rank * (p.k + p.n);
#pragma unroll
    for (int rb = 0; rb < RB; ++rb)
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int r = r0 + rb * 16 + 4 * g + q, c = c0 + 4 * i + j;
                if (r < p.rank && c < width) {
                    if (isA) part[(size_t)r * p.k + c] = acc[rb][j][q];
                    else part[(size_t)p.rank * p.k + (size_t)c * p.rank + r] = acc[rb][j][q];
                }
            }
}

// dA, dB of an adapter = s times the sum of its chunks' partials, in chunk order (zero without rows)
template <typename T>
__global__ void __launch_bounds__(256)
adapter_wgrad_reduce_kernel(AdaptGrad p) {
    const int per = p.rank * (p.k + p.n);
    const int e = blockIdx.x * 256 + threadIdx.x, ad = blockIdx.y;
    if (e >= per) return;
    const int c_begin = p.plan[p.o_chunk_first + ad], c_end = p.plan[p.o_chunk_first + ad + 1];
    float s = 0.f;
    for (int c = c_begin; c < c_end; ++c) s += p.part[(size_t)c * per + e];
    s *= p.scales[ad];
    const int na = p.rank * p.k;
    if (c_begin == c_end) s = 0.f;
    if (e < na) ((T*)p.da)[(size_t)ad * na + e] = (T)s;
    else ((T*)p.db)[(size_t)ad * p.rank * p.n + (e - na)] = (T)s;
}

static size_t elem_size(int type) { return type == JM_F32 ? 4 : 2; }

template <int TY>
static void launch_rows(const Adapt& p, int tiles, hipStream_t s) {
    const dim3 grid((unsigned)tiles), block(64);
    if (p.rank <= 16) hipLaunchKernelGGL((adapter_rows_kernel<TY, 1>), grid, block, 0, s, p);
    else if (p.rank <= 32) hipLaunchKernelGGL((adapter_rows_kernel<TY, 2>), grid, block, 0, s, p);
    else if (p.rank <= 64) hipLaunchKernelGGL((adapter_rows_kernel<TY, 4>), grid, block, 0, s, p);
    else hipLaunchKernelGGL((adapter_rows_kernel<TY, 8>), grid, block, 0, s, p);
}
static void launch_rows(int type, const Adapt& p, int tiles, hipStream_t s) {
    if (type == JM_F32) launch_rows<JM_F32>(p, tiles, s);
    else if (type == JM_BF16) launch_rows<JM_BF16>(p, tiles, s);
    else launch_rows<JM_F16>(p, tiles, s);
}

template <int TY, bool KEPT>
static void launch_wgrad(const AdaptGrad& p, int chunks, hipStream_t s) {
    const dim3 grid((unsigned)chunks, (unsigned)(divup(p.k, 64) + divup(p.n, 64)), (unsigned)divup(p.rank, 64)), block(256);
    if (p.rank <= 16) hipLaunchKernelGGL((adapter_wgrad_kernel<TY, KEPT, 1>), grid, block, 0, s, p);
    else if (p.rank <= 32) hipLaunchKernelGGL((adapter_wgrad_kernel<TY, KEPT, 2>), grid, block, 0, s, p);
    else hipLaunchKernelGGL((adapter_wgrad_kernel<TY, KEPT, 4>), grid, block, 0, s, p);
}

struct GradLayout { size_t at, bt, u, part, total; };        // bytes
static GradLayout grad_layout(int m, int k, int n, int rank, int adapters, int type) {
    const PlanLayout l = plan_layout(m, adapters);
    GradLayout g;
    g.at = 0;
    g.bt = align_up(g.at + (size_t)adapters * k * rank * elem_size(type), 256);
    g.u = align_up(g.bt + (size_t)adapters * n * rank * elem_size(type), 256);
    g.part = align_up(g.u + (size_t)m * rank * 4, 256);
    g.total = g.part + (size_t)l.max_chunks * rank * ((size_t)k + n) * 4;
    return g;
}

static int adapter_check(const char* what, int m, int k, int n, int rank, int adapters, int type) {
    JM_REQUIRE(m >= 0 && m <= AD_MAX_ROWS && k > 0 && k <= AD_MAX_WIDTH && n > 0 && n <= AD_MAX_WIDTH && type >= JM_F32 && type <= JM_F16, "%s: m %d, k %d, n %d, type %d", what, m, k, n, type);
    JM_REQUIRE(rank > 0 && rank <= JM_ADAPTER_MAX_RANK && adapters > 0 && adapters <= PL_MAX_ADAPTERS, "%s: rank %d of 1 .. %d, %d adapters of 1 .. %d", what, rank,
               JM_ADAPTER_MAX_RANK, adapters, PL_MAX_ADAPTERS);
    return JM_OK;
}

}  // namespace jm

using namespace jm;

extern "C" {

size_t jm_adapter_plan_elems(int m, int adapters) {
    if (m < 0 || m > AD_MAX_ROWS || adapters <= 0 || adapters > PL_MAX_ADAPTERS) return 0;
    return plan_layout(m, adapters).total;
}

int jm_adapter_plan(int m, int adapters, const int* ids, int* plan, jm_stream_t stream) {
    JM_REQUIRE(m >= 0 && m <= AD_MAX_ROWS && adapters > 0 && adapters <= PL_MAX_ADAPTERS, "adapter_plan: m %d, %d adapters of 1 .. %d", m, adapters, PL_MAX_ADAPTERS);
    JM_REQUIRE(plan && ((uintptr_t)plan & 15) == 0 && (m == 0 || ids), "adapter_plan: NULL or unaligned buffers");
    const PlanLayout l = plan_layout(m, adapters);
    hipStream_t s = (hipStream_t)stream;
    if (l.blocks <= 1) {
        hipLaunchKernelGGL((adapter_plan_count_kernel<true>), dim3(1), dim3(PL_THREADS), 0, s, m, adapters, ids, plan, l.order, l.tiles, l.chunks, l.chunk_first, l.hist);
        return check_launch("adapter_plan");
    }
    hipLaunchKernelGGL((adapter_plan_count_kernel<false>), dim3((unsigned)l.blocks), dim3(PL_THREADS), 0, s, m, adapters, ids, plan, l.order, l.tiles, l.chunks,
                       l.chunk_first, l.hist);
    hipLaunchKernelGGL(adapter_plan_tables_kernel, dim3(1), dim3(PL_THREADS), 0, s, l.blocks, adapters, plan, l.tiles, l.chunks, l.chunk_first, l.hist);
    hipLaunchKernelGGL(adapter_plan_scatter_kernel, dim3((unsigned)l.blocks), dim3(PL_THREADS), 0, s, m, adapters, ids, plan, l.order, l.hist);
    return check_launch("adapter_plan");
}

int jm_adapter_forward(int m, int k, int n, int rank, int adapters, int type, const void* x, long long ldx, const void* a, const void* b,
                       const float* scales, const int* plan, const void* base, long long ldb, void* out, long long ldo, float* t, jm_stream_t stream) {
    if (int e = adapter_check("adapter_forward", m, k, n, rank, adapters, type)) return e;
    JM_REQUIRE(ldx >= k && ldo >= n && (!base || ldb >= n), "adapter_forward: ldx %lld, ldb %lld, ldo %lld for k %d, n %d", ldx, ldb, ldo, k, n);
    if (m == 0) return JM_OK;
    JM_REQUIRE(x && a && b && scales && plan && out, "adapter_forward: NULL buffers");
    const PlanLayout l = plan_layout(m, adapters);
    Adapt p{};
    p.m = m; p.k = k; p.n = n; p.rank = rank; p.plan = plan; p.o_order = l.order; p.o_tiles = l.tiles; p.x = x; p.ldx = ldx; p.a = a; p.b = b;
    p.scales = scales; p.base = base; p.ldb = ldb; p.out = out; p.ldo = ldo; p.t = t; p.copy = base != out;
    launch_rows(type, p, l.max_tiles, (hipStream_t)stream);
    return check_launch("adapter_forward");
}

size_t jm_adapter_grad_workspace_bytes(int m, int k, int n, int rank, int adapters, int type) {
    if (m < 0 || m > AD_MAX_ROWS || k <= 0 || k > AD_MAX_WIDTH || n <= 0 || n > AD_MAX_WIDTH || rank <= 0 || rank > JM_ADAPTER_MAX_RANK || adapters <= 0 || adapters > PL_MAX_ADAPTERS) return 0;
    return grad_layout(m, k, n, rank, adapters, type).total;
}

int jm_adapter_grad(int m, int k, int n, int rank, int adapters, int type, const void* dy, long long lddy, const void* x, long long ldx,
                    const unsigned char* codes, int ldc, const unsigned char* exps, const float* t, const void* a, const void* b, const float* scales,
                    const int* plan, const void* base, long long ldb, void* dx, long long lddx, void* da, void* db, void* ws, size_t ws_bytes,
                    jm_stream_t stream) {
    if (int e = adapter_check("adapter_grad", m, k, n, rank, adapters, type)) return e;
    JM_REQUIRE(lddy >= n && lddx >= k && (!base || ldb >= k), "adapter_grad: lddy %lld, ldb %lld, lddx %lld for k %d, n %d", lddy, ldb, lddx, k, n);
    JM_REQUIRE(x ? ldx >= k : (m == 0 || (codes && exps && ldc >= k && ldc % 16 == 0 && ((uintptr_t)codes & 15) == 0)),
               "adapter_grad: x or its kept rows are needed (ldx %lld, ldc %d, k %d)", ldx, ldc, k);
    JM_REQUIRE(a && b && scales && plan && da && db && (m == 0 || (dy && t && dx)), "adapter_grad: NULL buffers");
    const GradLayout gl = grad_layout(m, k, n, rank, adapters, type);
    if (!ws || ws_bytes < gl.total || ((uintptr_t)ws & 15)) {
        set_error("adapter_grad: workspace of %zu bytes (16-byte aligned), need %zu", ws_bytes, gl.total);
        return JM_EWORKSPACE;
    }
    hipStream_t s = (hipStream_t)stream;
    const PlanLayout l = plan_layout(m, adapters);
    char* w = (char*)ws;
    AdaptGrad q{};
    q.m = m; q.k = k; q.n = n; q.rank = rank; q.adapters = adapters; q.plan = plan; q.o_order = l.order; q.o_chunks = l.chunks;
    q.o_chunk_first = l.chunk_first; q.x = x; q.ldx = ldx; q.codes = codes; q.ldc = ldc; q.exps = exps; q.blocks = divup(k, 32);
    q.dy = dy; q.lddy = lddy; q.t = t; q.u = (const float*)(w + gl.u); q.scales = scales; q.part = (float*)(w + gl.part); q.da = da; q.db = db;
    if (m > 0) {
        const dim3 ga((unsigned)divup(k, 32), (unsigned)divup(rank, 32), (unsigned)adapters), gb((unsigned)divup(rank, 32), (unsigned)divup(n, 32), (unsigned)adapters);
        if (type == JM_F32) {
            hipLaunchKernelGGL((adapter_transpose_kernel<float>), ga, dim3(256), 0, s, rank, k, (const float*)a, (float*)(w + gl.at));
            hipLaunchKernelGGL((adapter_transpose_kernel<float>), gb, dim3(256), 0, s, n, rank, (const float*)b, (float*)(w + gl.bt));
        } else {
            typedef unsigned short u16;
            hipLaunchKernelGGL((adapter_transpose_kernel<u16>), ga, dim3(256), 0, s, rank, k, (const u16*)a, (u16*)(w + gl.at));
            hipLaunchKernelGGL((adapter_transpose_kernel<u16>), gb, dim3(256), 0, s, n, rank, (const u16*)b, (u16*)(w + gl.bt));
        }
        Adapt p{};
        p.m = m; p.k = n; p.n = k; p.rank = rank; p.plan = plan; p.o_order = l.order; p.o_tiles = l.tiles; p.x = dy; p.ldx = lddy;
        p.a = w + gl.bt; p.b = w + gl.at; p.scales = scales; p.base = base; p.ldb = ldb; p.out = dx; p.ldo = lddx; p.t = (float*)(w + gl.u);
        p.copy = base != dx;
        launch_rows(type, p, l.max_tiles, s);
        if (x) {
            if (type == JM_F32) launch_wgrad<JM_F32, false>(q, l.max_chunks, s);
            else if (type == JM_BF16) launch_wgrad<JM_BF16, false>(q, l.max_chunks, s);
            else launch_wgrad<JM_F16, false>(q, l.max_chunks, s);
        } else {
            if (type == JM_F32) launch_wgrad<JM_F32, true>(q, l.max_chunks, s);
            else if (type == JM_BF16) launch_wgrad<JM_BF16, true>(q, l.max_chunks, s);
            else launch_wgrad<JM_F16, true>(q, l.max_chunks, s);
        }
    }
    const dim3 gr((unsigned)divup(rank * (k + n), 256), (unsigned)adapters);
    if (type == JM_F32) hipLaunchKernelGGL((adapter_wgrad_reduce_kernel<float>), gr, dim3(256), 0, s, q);
    else if (type == JM_BF16) hipLaunchKernelGGL((adapter_wgrad_reduce_kernel<__bf16>), gr, dim3(256), 0, s, q);
    else hipLaunchKernelGGL((adapter_wgrad_reduce_kernel<_Float16>), gr, dim3(256), 0, s, q);
    return check_launch("adapter_grad");
}

}  // extern "C"
