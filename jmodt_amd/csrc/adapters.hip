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
// The rows of an adapter are found by a plan in device memory (a stable counting sort of the rows by adapter, built by two small
// kernels, one for up to PL_ROWS rows; the host never learns the counts): tiles of 16 or 32 rows and chunks of 128 to 512 rows, each of
// one adapter.
#include "jm_elem.h"
#include "jm_rows.h"
#include <type_traits>

namespace jm {

// ------------------------------------------------------------------------------------------------ plan
constexpr int PL_ROWS = 4096, PL_BLOCKS = 256;        // a counting block has a multiple of PL_ROWS rows, so that there are at most PL_BLOCKS
constexpr int PL_THREADS = 1024;
constexpr int PL_MAX_ADAPTERS = 1023;        // + the rows without an adapter: one counter a thread
constexpr int AD_WIDE_ROWS = 16384;
// rows of a tile: 16 while that leaves CUs idle, 32 where there are enough tiles (A and B are read once a tile).  Forward, k = n = 512, 16 | 32
// rows: 4096 rows float32 rank 16 10.2 | 14.4 us, 8192 bfloat16 8.7 | 9.4; 16384 rank 64 47 | 43 and 24 | 20; 65536 rank 16 108 | 98, 40 | 38.
// With tiles of 16 the backward gathers A and B transposed, with 32 a kernel transposes them first (gather | transpose, float32 rank 16:
// 512 rows 11.0 | 15.1 us, 4096 rows 28.8 | 32.8, 8192 rows 35.4 | 38.6).
static __host__ __device__ __forceinline__ int ad_tile(int m) { return m < AD_WIDE_ROWS ? 16 : 32; }
constexpr int AD_CHUNK = 512;
// rows of a chunk (weight gradients).  Up to AD_CHUNK rows an adapter is one chunk and its workgroups write the gradients themselves (512 rows of
// four adapters, float32 rank 16: 12.0 us for the backward, 14.0 with chunks of 128 and a second kernel; of a single adapter 19.4 | 14.9).
// Beyond that small chunks fill the CUs, large ones write fewer partials (chunks of 128 | 256 | 512, float32 rank 16: 1024 rows of one
// adapter 14.6 | 17.6 | 22 us; 4096 rows of eight 24.3 | 24.1 | 28.7; 8192 rows, rank 64: 58 | 53 | 62; 16383 rows, rank 64: 98 | 87 | 82).
static __host__ __device__ __forceinline__ int ad_chunk(int m) { return m <= AD_CHUNK || m > 8192 ? AD_CHUNK : (m <= 4096 ? 128 : 256); }
constexpr int AD_MAX_ROWS = 1 << 28, AD_MAX_WIDTH = 1 << 20;        // grids (2^32 threads) and per-adapter element counts stay in range

struct PlanLayout {                  // offsets in ints; header: [0] tiles, [1] chunks
    size_t order, tiles, chunks, chunk_first, hist, total;
    int max_tiles, max_chunks, blocks, block_rows;
};
static PlanLayout plan_layout(int m, int adapters) {
    PlanLayout l;
    l.block_rows = PL_ROWS * imax(1, divup(m, PL_ROWS * PL_BLOCKS));
    l.blocks = divup(m, l.block_rows);
    l.max_tiles = divup(m, ad_tile(m)) + (adapters + 1 < m ? adapters + 1 : m);
    l.max_chunks = divup(m, ad_chunk(m)) + (adapters < m ? adapters : m);
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

// bucket counts -> starts, and the tables of tiles and chunks (entries part, part + parts, ... of every PL_THREADS).  `count`: this
// thread's bucket count (thread = bucket).  first[b] = {row start, first tile, first chunk} of bucket b, first[adapters + 1] = the totals.
__device__ void plan_tables(int count, int adapters, int tile_rows, int chunk_rows, int part, int parts, int (*first)[3], int (*wave_tot)[3], int* __restrict__ plan, size_t o_tiles,
                            size_t o_chunks, size_t o_chunk_first) {
    const int b = threadIdx.x;
    int v[3] = {count, (count + tile_rows - 1) / tile_rows, b < adapters ? (count + chunk_rows - 1) / chunk_rows : 0};
    const int mine[3] = {v[0], v[1], v[2]};
    plan_scan3(v, wave_tot);
    if (b <= adapters)
#pragma unroll
        for (int q = 0; q < 3; ++q) {
            first[b][q] = v[q];
            if (b == adapters) first[b + 1][q] = v[q] + mine[q];
        }
    __syncthreads();
    if (part == 0 && b <= adapters) plan[o_chunk_first + b] = first[b][2];
    const int nt = first[adapters + 1][1], nc = first[adapters + 1][2];
    if (part == 0 && b == 0) { plan[0] = nt; plan[1] = nc; plan[2] = 0; plan[3] = 0; }
    // a table entry finds its bucket by bisection: the last bucket whose first tile is <= t
    for (int t = part * PL_THREADS + b; t < nt; t += parts * PL_THREADS) {
        int lo = 0, hi = adapters;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (first[mid][1] <= t) lo = mid; else hi = mid - 1;
        }
        const int start = first[lo][0] + (t - first[lo][1]) * tile_rows;
        *reinterpret_cast<int4*>(plan + o_tiles + 4 * (size_t)t) = make_int4(lo < adapters ? lo : -1, start, min(tile_rows, first[lo + 1][0] - start), 0);
    }
    for (int t = part * PL_THREADS + b; t < nc; t += parts * PL_THREADS) {
        int lo = 0, hi = adapters - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (first[mid][2] <= t) lo = mid; else hi = mid - 1;
        }
        const int start = first[lo][0] + (t - first[lo][2]) * chunk_rows;
        *reinterpret_cast<int4*>(plan + o_chunks + 4 * (size_t)t) = make_int4(lo, start, min(chunk_rows, first[lo + 1][0] - start), 0);
    }
}

// rows row0 .. row0 + rows - 1 to their places, in row order within a bucket: next[b] = the bucket's next place.  A wave ranks its 64
// rows among those of the same id, the waves' counts (bytes: at most 64) are added in wave order.
__device__ void plan_scatter(const int* __restrict__ ids, long long row0, int rows, int adapters, int* next, unsigned char (*wcnt)[PL_THREADS],
                             int* __restrict__ order) {
    const int wave = threadIdx.x >> 6;
    for (int r = 0; r < rows; r += PL_THREADS) {
        __syncthreads();
        for (int q = threadIdx.x; q < 16 * PL_THREADS / 4; q += PL_THREADS) reinterpret_cast<unsigned*>(wcnt)[q] = 0u;
        __syncthreads();
        const bool ok = r + (int)threadIdx.x < rows;
        const int b = ok ? plan_bucket(ids, row0 + r + threadIdx.x, adapters) : -1;
        unsigned long long same = __ballot(ok);              // the lanes of this wave with the same id, bit by bit of it
        for (int bit = 1; bit <= adapters; bit <<= 1) {
            const unsigned long long set = __ballot((b & bit) != 0);
            same &= (b & bit) ? set : ~set;
        }
        const int rank = mbcnt(same);
        if (ok && rank == 0) wcnt[wave][b] = (unsigned char)__popcll(same);
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

// The plan reads ids twice and writes 4 bytes a row; launches and one block's barriers bound it: 4096 rows 10 us in one launch, 65536 rows
// 15 us (4 adapters) and 13 us (64 in mixed order) in two, 2^20 rows 25 us.
// ids of one counting block counted in LDS; whole: the block is all there is and the plan is finished here (one launch)
template <bool WHOLE>
__global__ void __launch_bounds__(PL_THREADS)
adapter_plan_count_kernel(int m, int block_rows, int adapters, const int* __restrict__ ids, int* __restrict__ plan, size_t o_order, size_t o_tiles, size_t o_chunks,
                          size_t o_chunk_first, size_t o_hist) {
    __shared__ int cnt[PL_THREADS];
    __shared__ int first[WHOLE ? PL_THREADS + 2 : 1][3], wave_tot[16][3];
    __shared__ __attribute__((aligned(4))) unsigned char wcnt[WHOLE ? 16 : 1][PL_THREADS];
    cnt[threadIdx.x] = 0;
    __syncthreads();
    const long long row0 = (long long)blockIdx.x * block_rows;
    const int rows = (int)min((long long)block_rows, m - row0);
    for (int r = threadIdx.x; r < rows; r += PL_THREADS) atomicAdd(&cnt[plan_bucket(ids, row0 + r, adapters)], 1);
    __syncthreads();
    if constexpr (WHOLE) {
        plan_tables(cnt[threadIdx.x], adapters, ad_tile(m), ad_chunk(m), 0, 1, first, wave_tot, plan, o_tiles, o_chunks, o_chunk_first);
        __syncthreads();
        if ((int)threadIdx.x <= adapters) cnt[threadIdx.x] = first[threadIdx.x][0];
        plan_scatter(ids, 0, rows, adapters, cnt, wcnt, plan + o_order);
    } else {
        if ((int)threadIdx.x <= adapters) plan[o_hist + (size_t)blockIdx.x * (adapters + 1) + threadIdx.x] = cnt[threadIdx.x];
    }
}

// the rows to their places: every block adds up the counts of the blocks before it (and of all, for the starts of the buckets) and writes
// its share of the tables
__global__ void __launch_bounds__(PL_THREADS)
adapter_plan_scatter_kernel(int m, int block_rows, int adapters, const int* __restrict__ ids, int* __restrict__ plan, size_t o_order, size_t o_tiles, size_t o_chunks,
                            size_t o_chunk_first, size_t o_hist) {
    __shared__ int next[PL_THREADS];
    __shared__ int first[PL_THREADS + 2][3], wave_tot[16][3];
    __shared__ __attribute__((aligned(4))) unsigned char wcnt[16][PL_THREADS];
    const int b = threadIdx.x;
    const int* hist = plan + o_hist + b;
    int total = 0, before = 0;
    if (b <= adapters)
#pragma unroll 8
        for (int k = 0; k < (int)gridDim.x; ++k) {
            const int c = hist[k * (adapters + 1)];
            total += c;
            before += k < (int)blockIdx.x ? c : 0;
        }
    plan_tables(total, adapters, ad_tile(m), ad_chunk(m), blockIdx.x, gridDim.x, first, wave_tot, plan, o_tiles, o_chunks, o_chunk_first);
    if (b <= adapters) next[b] = first[b][0] + before;
    const long long row0 = (long long)blockIdx.x * block_rows;
    plan_scatter(ids, row0, (int)min((long long)block_rows, m - row0), adapters, next, wcnt, plan + o_order);
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

// 16 consecutive channels of a row
template <int TY>
struct Run16 {
    typedef typename Elem<TY>::T T;
    typedef typename Elem<TY>::V8 V8;
    V8 v[2];
    __device__ __forceinline__ void load(const T* p, int n) {
        if (n >= 16) { v[0] = load8<V8>(p); v[1] = load8<V8>(p + 8); }
        else { v[0] = load8_upto<V8>(p, n); v[1] = load8_upto<V8>(p + 8, n - 8); }
    }
    __device__ __forceinline__ void store(T* p, int n) const {
        if (n >= 16) { store8(p, v[0]); store8(p + 8, v[1]); return; }
#pragma unroll
        for (int e = 0; e < 16; ++e)
            if (e < n) p[e] = v[e >> 3][e & 7];
    }
};

// A workgroup owns a tile of 16 MB rows of one adapter (and every gridDim.y-th group of four 64-channel blocks of out: with few rows the
// workgroups of one tile each make t again, which costs less than a CU left idle).
//   1  t (rank x rows) = A x^T: the four waves take a quarter of k each, 32 elements a step, both operands straight from memory into the
//      registers of the 16 x 16 products (lane: 8 consecutive elements of one row), UK steps in flight; the quarters are added through LDS.
//   2  out (channels x rows) = base + s B t^T: a wave takes 64 channels; the rows of B are permuted so that a lane ends up with 16
//      consecutive channels of its row, which it reads from base and writes to out.
// t enters the second product as it is in float32, as the sum of three values in bfloat16 (8 + 8 + 8 bits: all of float32's) and of two in
// float16 (11 + 11 bits and the signs: 2^-23 of the row's largest value; the row is scaled by a power of two first, as t may leave float16's
// range although out does not).  With two values in bfloat16, too (2^-17 of t), 0.1 % of the outputs rounded to the neighbouring value, and
// where base and the adapter cancel it was more than out's own rounding.  With a rank of up to 16 two values share one product: the contraction
// is 32 long, [hi | lo] times [B | B].
// WT: A and B are given transposed, (k, rank) and (rank, n) — the backward on B and A as they are: their elements are gathered one by one,
// which few tiles can afford and many cannot (there a kernel of its own transposes them first).
// Bound by memory with many rows (x and base read, out written once: 65536 x 256 x 256 bfloat16, rank 32, t written: 30 us, 3.7 TB/s;
// 65536 x 512 x 512 float32, t written, rank 16: 105 us, 3.9 TB/s, rank 64: 184 us — there the float32 pipe has 56 us of it), by the chain of loads
// through both products with few (1024 x 512 x 512 float32, rank 16: 7.4 us).
template <int TY, int RB, int MB, bool WT>
__global__ void __launch_bounds__(256)
adapter_rows_kernel(Adapt p) {
    typedef typename Elem<TY>::T T;
    typedef typename Elem<TY>::V8 V8;
    constexpr int RP = RB * 16, LD = RP + 4, ROWS = 16 * MB;
    constexpr int UK = (TY == JM_F32 ? 4 : 8) / (RB < 2 ? 1 : (RB < 8 ? RB / 2 * MB : 8 / (TY == JM_F32 ? 2 : 1)));
    constexpr bool PAIR = TY != JM_F32 && RB == 1;       // hi and lo in one contraction
    constexpr int RS = TY == JM_F32 ? RB : (RB + 1) / 2; // contraction steps over the rank: 16 long in float32, 32 otherwise
    __shared__ __attribute__((aligned(16))) float ts[2][ROWS][LD];
    if ((int)blockIdx.x >= p.plan[0]) return;
    const int4 tile = *reinterpret_cast<const int4*>(p.plan + p.o_tiles + 4 * (size_t)blockIdx.x);
    const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int ad = tile.x, count = tile.z;
    const int* order = p.plan + p.o_order + tile.y;
    size_t row[MB];
    bool live[MB];
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) {
        live[mb] = mb * 16 + i < count;
        row[mb] = (size_t)order[min(mb * 16 + i, count - 1)];
    }
    const int nblocks = (p.n + 63) / 64;
    const T* const base = (const T*)p.base;
    T* const out = (T*)p.out;
    if (ad < 0) {                                        // rows without an adapter
        if (p.copy)
            for (int nb = blockIdx.y * 4 + wave; nb < nblocks; nb += gridDim.y * 4)
#pragma unroll
                for (int mb = 0; mb < MB; ++mb)
                    if (live[mb]) {
                        const int c = nb * 64 + 16 * g;
                        Run16<TY> v;
                        if (base) v.load(base + row[mb] * p.ldb + c, p.n - c);
                        else
#pragma unroll
                            for (int e = 0; e < 16; ++e) v.v[e >> 3][e & 7] = (T)0.f;
                        v.store(out + row[mb] * p.ldo + c, p.n - c);
                    }
        if (p.t && blockIdx.y == 0)
            for (int e = threadIdx.x; e < count * p.rank; e += 256) p.t[(size_t)order[e / p.rank] * p.rank + e % p.rank] = 0.f;
        return;
    }
    const T* A = (const T*)p.a + (size_t)ad * p.rank * p.k;
    const T* B = (const T*)p.b + (size_t)ad * p.n * p.rank;
    const float scale = p.scales[ad];

    {
        const T *xr[MB], *ar[RB];
#pragma unroll
        for (int mb = 0; mb < MB; ++mb) xr[mb] = (const T*)p.x + row[mb] * p.ldx + 8 * g;
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
            const int r = min(rb * 16 + i, p.rank - 1);
            ar[rb] = WT ? A + (size_t)(8 * g) * p.rank + r : A + (size_t)r * p.k + 8 * g;
        }
        // elements 0 .. left - 1 (of 8) of step s; WT: A lies as (k, rank)
        auto load_a = [&](const T* q, int s, int left) __attribute__((always_inline)) {
            if constexpr (WT) {
                V8 v;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    T t = (T)0.f;
                    if (e < left) t = q[(size_t)(32 * s + e) * p.rank];
                    v[e] = t;
                }
                return v;
            } else {
                return load8_upto<V8>(q + 32 * s, left);
            }
        };
        f32x4 acc[MB][RB];
#pragma unroll
        for (int mb = 0; mb < MB; ++mb)
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) acc[mb][rb] = f32x4{0.f, 0.f, 0.f, 0.f};
        const int nk = (p.k + 31) / 32, per = (nk + 3) / 4;
        int s = wave * per;
        const int s_end = min(nk, s + per), s_full = min(s_end, p.k / 32);
        auto batch = [&](auto n_) __attribute__((always_inline)) {
            constexpr int U = decltype(n_)::value;
            V8 xv[U][MB], av[U][RB];
#pragma unroll
            for (int u = 0; u < U; ++u) {
#pragma unroll
                for (int mb = 0; mb < MB; ++mb) xv[u][mb] = load8<V8>(xr[mb] + 32 * (s + u));
#pragma unroll
                for (int rb = 0; rb < RB; ++rb) av[u][rb] = load_a(ar[rb], s + u, 8);
            }
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int mb = 0; mb < MB; ++mb)
#pragma unroll
                    for (int rb = 0; rb < RB; ++rb) acc[mb][rb] = mma16(acc[mb][rb], av[u][rb], xv[u][mb]);
            s += U;
        };
        while (s + UK <= s_full) batch(std::integral_constant<int, UK>{});
        if constexpr (UK > 4) { if (s + 4 <= s_full) batch(std::integral_constant<int, 4>{}); }
        if constexpr (UK > 2) { if (s + 2 <= s_full) batch(std::integral_constant<int, 2>{}); }
        if constexpr (UK > 1) { if (s + 1 <= s_full) batch(std::integral_constant<int, 1>{}); }
        for (; s < s_end; ++s) {
            const int left = p.k - 32 * s - 8 * g;
            V8 xv[MB];
#pragma unroll
            for (int mb = 0; mb < MB; ++mb) xv[mb] = load8_upto<V8>(xr[mb] + 32 * s, left);
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) {
                const V8 av = load_a(ar[rb], s, left);
#pragma unroll
                for (int mb = 0; mb < MB; ++mb) acc[mb][rb] = mma16(acc[mb][rb], av, xv[mb]);
            }
        }
        // D: column = row i of the block, rows = rank index 4 g + q
        if (wave < 2)
#pragma unroll
            for (int mb = 0; mb < MB; ++mb)
#pragma unroll
                for (int rb = 0; rb < RB; ++rb) *reinterpret_cast<f32x4*>(&ts[wave][mb * 16 + i][rb * 16 + 4 * g]) = acc[mb][rb];
        __syncthreads();
        if (wave >= 2)
#pragma unroll
            for (int mb = 0; mb < MB; ++mb)
#pragma unroll
                for (int rb = 0; rb < RB; ++rb) {
                    f32x4* q = reinterpret_cast<f32x4*>(&ts[wave - 2][mb * 16 + i][rb * 16 + 4 * g]);
                    *q = *q + acc[mb][rb];
                }
        __syncthreads();
    }
    if (p.t && blockIdx.y == 0)
        for (int e = threadIdx.x; e < count * p.rank; e += 256) {
            const int r = e / p.rank, c = e - r * p.rank;
            p.t[(size_t)order[r] * p.rank + c] = ts[0][r][c] + ts[1][r][c];
        }
    if (blockIdx.y * 4 + wave >= nblocks) return;

    // this lane's part of t; rank indices beyond the rank (copies of the last one) are zeros
    auto tval = [&](int mb, int r) { return r < p.rank ? ts[0][mb * 16 + i][r] + ts[1][mb * 16 + i][r] : 0.f; };
    float back[MB];
    f32x4 t32[TY == JM_F32 ? MB : 1][RS];
    constexpr bool THREE = TY == JM_BF16;
    V8 hi[MB][RS], lo[MB][RS], rest[THREE ? MB : 1][RS];
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) {
        back[mb] = scale;
        if constexpr (TY == JM_F32) {
#pragma unroll
            for (int s = 0; s < RS; ++s)
#pragma unroll
                for (int e = 0; e < 4; ++e) t32[mb][s][e] = tval(mb, s * 16 + 4 * g + e);
        } else {
            float v[RS][8], fit = 1.f, top = 0.f;
#pragma unroll
            for (int s = 0; s < RS; ++s)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    v[s][e] = tval(mb, PAIR ? 8 * (g & 1) + e : s * 32 + 8 * g + e);
                    top = fmaxf(top, fabsf(v[s][e]));
                }
            if constexpr (TY == JM_F16) {
                top = fmaxf(top, __shfl_xor(top, 16));
                top = fmaxf(top, __shfl_xor(top, 32));
                const int ex = min(max((int)(__float_as_uint(top) >> 23) - 127, -100), 126);      // the row's values become less than 4
                fit = __uint_as_float((unsigned)(127 - ex) << 23);
                back[mb] = scale * __uint_as_float((unsigned)(127 + ex) << 23);
            }
#pragma unroll
            for (int s = 0; s < RS; ++s)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float f = v[s][e] * fit;
                    const T h = (T)f;
                    const float left = fabsf((float)h) < __builtin_inff() ? f - (float)h : 0.f;
                    const T r = (T)left;
                    hi[mb][s][e] = (PAIR && g >= 2) ? r : h;
                    lo[mb][s][e] = r;
                    if constexpr (THREE) rest[mb][s][e] = (PAIR && g >= 2) ? (T)0.f : (T)(left - (float)r);
                }
        }
    }

    for (int nb = blockIdx.y * 4 + wave; nb < nblocks; nb += gridDim.y * 4) {
        const int n0 = nb * 64, c = n0 + 16 * g;
        Run16<TY> bv[MB];
#pragma unroll
        for (int mb = 0; mb < MB; ++mb) {
            if (base) bv[mb].load(base + row[mb] * p.ldb + c, p.n - c);
            else
#pragma unroll
                for (int e = 0; e < 16; ++e) bv[mb].v[e >> 3][e & 7] = (T)0.f;
        }
        f32x4 d[MB][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int bc = min(n0 + (i >> 2) * 16 + j * 4 + (i & 3), p.n - 1);
            const T* Br = WT ? B + bc : B + (size_t)bc * p.rank;           // WT: B lies as (rank, n)
#pragma unroll
            for (int mb = 0; mb < MB; ++mb) d[mb][j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int s = 0; s < RS; ++s) {
                if constexpr (TY == JM_F32) {
                    const int r0 = s * 16 + 4 * g;
                    f32x4 b4;
                    if (!WT && r0 + 4 <= p.rank) __builtin_memcpy(&b4, Br + r0, 16);
                    else
#pragma unroll
                        for (int e = 0; e < 4; ++e) b4[e] = r0 + e < p.rank ? (WT ? Br[(size_t)(r0 + e) * p.n] : Br[r0 + e]) : 0.f;
#pragma unroll
                    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
                        for (int e = 0; e < 4; ++e) d[mb][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(b4[e], t32[mb][s][e], d[mb][j], 0, 0, 0);
                } else {
                    const int r0 = PAIR ? 8 * (g & 1) : s * 32 + 8 * g;
                    V8 b8;
                    if constexpr (WT) {
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            T t = (T)0.f;
                            if (r0 + e < p.rank) t = Br[(size_t)(r0 + e) * p.n];
                            b8[e] = t;
                        }
                    } else {
                        b8 = load8_upto<V8>(Br + r0, p.rank - r0);
                    }
#pragma unroll
                    for (int mb = 0; mb < MB; ++mb) {
                        d[mb][j] = mma16(d[mb][j], b8, hi[mb][s]);
                        if constexpr (!PAIR) d[mb][j] = mma16(d[mb][j], b8, lo[mb][s]);
                        if constexpr (THREE) d[mb][j] = mma16(d[mb][j], b8, rest[mb][s]);
                    }
                }
            }
        }
#pragma unroll
        for (int mb = 0; mb < MB; ++mb)
            if (live[mb]) {
                Run16<TY> o;
#pragma unroll
                for (int e = 0; e < 16; ++e) o.v[e >> 3][e & 7] = (T)((float)bv[mb].v[e >> 3][e & 7] + back[mb] * d[mb][e >> 2][e & 3]);
                o.store(out + row[mb] * p.ldo + c, p.n - c);
            }
    }
}

// (adapters, rank, k) -> (adapters, k, rank) and (adapters, n, rank) -> (adapters, rank, n): blockIdx.x walks the 32 x 32 tiles of both.  A launch's
// latency: 4.2 us for four adapters of 512 x 256, rank 16.
template <typename T>
__global__ void __launch_bounds__(256)
adapter_transpose_kernel(int rank, int k, int n, const T* __restrict__ a, T* __restrict__ at, const T* __restrict__ b, T* __restrict__ bt) {
    __shared__ T tile[32][33];
    const int tr = (rank + 31) / 32, ta = ((k + 31) / 32) * tr;
    const bool isA = (int)blockIdx.x < ta;
    const int id = isA ? blockIdx.x : blockIdx.x - ta;
    const int rows = isA ? rank : n, cols = isA ? k : rank;
    const int r0 = (isA ? id % tr : id / tr) * 32, c0 = (isA ? id / tr : id % tr) * 32, tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    const size_t off = (size_t)blockIdx.y * rows * cols;
    const T* src = (isA ? a : b) + off;
    T* dst = (isA ? at : bt) + off;
    for (int q = ty; q < 32; q += 8)
        if (r0 + q < rows && c0 + tx < cols) tile[q][tx] = src[(size_t)(r0 + q) * cols + c0 + tx];
    __syncthreads();
    for (int q = ty; q < 32; q += 8)
        if (c0 + q < cols && r0 + tx < rows) dst[(size_t)(c0 + q) * rows + r0 + tx] = tile[tx][q];
}

// ------------------------------------------------------------------------------------------------ gradients of A and B
struct AdaptGrad {
    int m, k, n, rank, adapters, direct;
    const int* plan; size_t o_order, o_chunks, o_chunk_first;
    const void* x; long long ldx;
    const unsigned char* codes; int ldc; const unsigned char* exps; int lde;      // x kept in 8 bits (x NULL)
    const void* dy; long long lddy;
    const float *t, *u;                  // (m, rank)
    const float* scales;
    float* part;                         // per chunk: (rank, k) of dA, then (n, rank) of dB
    void *da, *db;
};

// CW consecutive channels of a row as they are stored (kept: e4m3 codes and the scale of their block), zeros beyond the width
template <int TY, bool KEPT, int CW>
struct GradRun {
    typedef typename Elem<TY>::T T;
    typedef T V __attribute__((ext_vector_type(CW)));
    V v;
    unsigned w[CW / 4], e;
    // scale: kept rows, the scale byte of the row and the channels' block
    __device__ __forceinline__ void load(const AdaptGrad& p, const void* src, long long ld, size_t row, int c, int width, const unsigned char* scale) {
        if constexpr (KEPT) {
            e = *scale;
            const unsigned* q = reinterpret_cast<const unsigned*>(p.codes + row * p.ldc + c);
#pragma unroll
            for (int h = 0; h < CW / 4; ++h) w[h] = 0u;
            if (c + CW <= p.ldc)
#pragma unroll
                for (int h = 0; h < CW / 4; ++h) w[h] = q[h];
        } else {
            const T* q = (const T*)src + row * ld + c;
            if (c + CW <= width) {
                __builtin_memcpy(&v, q, sizeof(V));
            } else {
#pragma unroll
                for (int j = 0; j < CW; ++j) {
                    T t = (T)0.f;
                    if (c + j < width) t = q[j];
                    v[j] = t;
                }
            }
        }
    }
    // channels 2 h, 2 h + 1 as two bfloat16 (rows of bfloat16, kept rows)
    __device__ __forceinline__ unsigned pair(int h) const {
        unsigned o;
        if constexpr (KEPT) {
            const float s = __uint_as_float(e << 23);
            const auto d = (h & 1) ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)w[h / 2], s, true) : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)w[h / 2], s, false);
            __builtin_memcpy(&o, &d, 4);
        } else {
            typedef T V2 __attribute__((ext_vector_type(2)));
            const V2 d = {v[2 * h], v[2 * h + 1]};
            __builtin_memcpy(&o, &d, 4);
        }
        return o;
    }
    __device__ __forceinline__ float get(int j) const {
        if constexpr (KEPT) {
            const auto d = (j & 2) ? __builtin_amdgcn_cvt_pk_f32_fp8((int)w[j / 4], true) : __builtin_amdgcn_cvt_pk_f32_fp8((int)w[j / 4], false);
            return d[j & 1] * __uint_as_float(e << 23);      // scale bytes: 27 .. 247
        } else {
            return (float)v[j];
        }
    }
};

// the four waves' tiles through LDS, added in wave order, to their place; 32 KB of LDS at a time (with 64 KB a CU
// holds two workgroups, too few loads in flight)
constexpr int ad_finish(int rb, int cw) { return rb * cw > 8 ? 8 / cw : rb; }
template <int TY, int RB, int CW>
__device__ __forceinline__ void adapter_wgrad_finish(const AdaptGrad& p, float* lds, float* part, int4 chunk, int ad, bool isA, int c0, int r0, const f32x4 (&acc)[RB][CW]) {
    constexpr int FB = ad_finish(RB, CW), TR = 16 * FB, TC = 16 * CW;
    const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4, wave = threadIdx.x >> 6, width = isA ? p.k : p.n;
    // D: rows = rank index 4 g + q, column i = channel CW i + j of the tile.  Row r of a tile is turned by 4 r columns, so that it can be read
    // down the ranks, too (dB) without its lanes meeting in one bank
    float* const mine = lds + wave * TR * TC;
    auto place = [&](int r, int c) { return r * TC + ((c + 4 * r) & (TC - 1)); };
    typedef typename Elem<TY>::T E;
    const float scale = p.direct ? p.scales[ad] : 1.f;
#pragma unroll
    for (int f = 0; f < RB; f += FB) {
        __syncthreads();
#pragma unroll
        for (int rb = 0; rb < FB; ++rb)
#pragma unroll
            for (int q = 0; q < 4; ++q)
#pragma unroll
                for (int j = 0; j < CW; j += 4) {
                    const f32x4* a = acc[f + rb];
                    *reinterpret_cast<f32x4*>(mine + place(rb * 16 + 4 * g + q, CW * i + j)) = f32x4{a[j][q], a[j + 1][q], a[j + 2][q], a[j + 3][q]};
                }
        __syncthreads();
        for (int e = threadIdx.x; e < TR * TC; e += 256) {   // (dA runs along the channels, dB along the rank)
            const int rt = isA ? e / TC : e % TR, ct = isA ? e % TC : e / TR, r = r0 + 16 * f + rt, c = c0 + ct;
            if (r >= p.rank || c >= width) continue;
            const float* v = lds + place(rt, ct);
            const float sum = (v[0] + v[TR * TC]) + (v[2 * TR * TC] + v[3 * TR * TC]);
            const size_t at = isA ? (size_t)r * p.k + c : (size_t)c * p.rank + r;
            if (p.direct) ((E*)(isA ? p.da : p.db))[(size_t)ad * p.rank * width + at] = (E)(chunk.z > 0 ? scale * sum : 0.f);
            else part[(isA ? 0 : (size_t)p.rank * p.k) + at] = sum;
        }
    }
}

// Workgroup = (chunk of one adapter's rows) x (16 CW channels of x, then of dy) x (16 RB rank indices); its four waves take every fourth
// group of four rows, 16 x 16 x 4 float32 products of T (t or u: rank) with X (CW channels a lane), UR groups in flight while UR are
// multiplied, and add their tiles in wave order through LDS.  Bound by the loads' latency with few rows (512 x 512 x 512, rank 16, four
// adapters: 6.4 us), by the memory and the float32 pipe together with many (65536 x 512 x 512, rank 16: 63 us of 268 MB, 4.3 TB/s).
// With at most one chunk an adapter (direct) the workgroups are the adapters' and write dA and dB themselves.
template <int TY, bool KEPT, int RB, int CW>
__device__ __forceinline__ void adapter_wgrad_tile(const AdaptGrad& p, float* lds, float* part, int4 chunk, int ad, bool isA, int c0, int r0) {
    constexpr int UR = 4;
    int* const rows = reinterpret_cast<int*>(lds);
    const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4, wave = threadIdx.x >> 6;
    const int width = isA ? p.k : p.n;
    const void* src = isA ? p.x : p.dy;
    const long long ld = isA ? p.ldx : p.lddy;
    const float* T = isA ? p.u : p.t;
    // the chunk's rows, and of kept rows the scales of the tile's blocks of 32 channels, once for all batches
    unsigned char* const scales = reinterpret_cast<unsigned char*>(rows + AD_CHUNK);
    for (int q = threadIdx.x; q < chunk.z; q += 256) {
        const int row = p.plan[p.o_order + chunk.y + q];
        rows[q] = row;
        if constexpr (KEPT) {
#pragma unroll
            for (int b = 0; b < CW / 2; ++b) scales[b * AD_CHUNK + q] = p.exps[(size_t)min(c0 / 32 + b, (width - 1) / 32) * p.lde + row];
        }
    }
    __syncthreads();
    const unsigned char* const scale = scales + (CW * i / 32) * AD_CHUNK;
    f32x4 acc[RB][CW];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb)
#pragma unroll
        for (int j = 0; j < CW; ++j) acc[rb][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    struct Batch {
        GradRun<TY, KEPT, CW> x[UR];
        float t[UR][RB];
    };
    auto fetch = [&](Batch& b, int q0) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < UR; ++u) {                       // (rows beyond the chunk: the last one, counted as zeros)
            const int at = min(q0 + 16 * u + g, chunk.z - 1);
            const size_t row = (size_t)rows[at];
            b.x[u].load(p, src, ld, row, c0 + CW * i, width, scale + at);
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) b.t[u][rb] = T[row * p.rank + min(r0 + rb * 16 + i, p.rank - 1)];
        }
    };
    auto multiply = [&](const Batch& b, int q0) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < UR; ++u) {
            const bool ok = q0 + 16 * u + g < chunk.z;
            float xv[CW];
#pragma unroll
            for (int j = 0; j < CW; ++j) xv[j] = ok ? b.x[u].get(j) : 0.f;
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) {
                const float t = ok ? b.t[u][rb] : 0.f;
#pragma unroll
                for (int j = 0; j < CW; ++j) acc[rb][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(t, xv[j], acc[rb][j], 0, 0, 0);
            }
        }
    };
    if (chunk.z > 0) {
        constexpr int ST = 16 * UR;                          // rows of a batch of the four waves
        Batch b[2];
        int q = wave * 4;
        fetch(b[0], q);
        for (; q < chunk.z; q += 2 * ST) {
            if (q + ST < chunk.z) fetch(b[1], q + ST);
            multiply(b[0], q);
            if (q + 2 * ST < chunk.z) fetch(b[0], q + 2 * ST);
            if (q + ST < chunk.z) multiply(b[1], q + ST);
        }
    }
    adapter_wgrad_finish<TY, RB, CW>(p, lds, part, chunk, ad, isA, c0, r0, acc);
}

// The same tile on the bf16 matrix pipe, for channels that are exact in bfloat16 (bfloat16 rows, kept rows): T enters as three bfloat16
// pieces that add up to it (rows8.hip's cut), so products are exact and only the float32 additions round — at a third of sixteen times the
// float32 rate.  A lane's 8 contraction elements are 8 rows; it holds 8 channels of each and turns the 8 x 8 block over in its registers.
// One batch in flight a wave and many waves: 65536 rows, kept x of 512, dy of 256, rank 16: 18 us of 76 MB, 4.2 TB/s; 131072 x 512 x 512,
// rank 64: 119 us, the loads of the few workgroups that fit (147 registers a lane).
template <bool KEPT, int RB>
__device__ __forceinline__ void adapter_wgrad_tile_bf16(const AdaptGrad& p, float* lds, float* part, int4 chunk, int ad, bool isA, int c0, int r0) {
    constexpr int CW = 8, STEP = 4 * 32;
    int* const rows = reinterpret_cast<int*>(lds);
    const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4, wave = threadIdx.x >> 6;
    const int width = isA ? p.k : p.n;
    const void* src = isA ? p.x : p.dy;
    const long long ld = isA ? p.ldx : p.lddy;
    const float* T = isA ? p.u : p.t;
    // the chunk's rows, and of kept rows the scales of the tile's blocks of 32 channels, once for all batches
    unsigned char* const scales = reinterpret_cast<unsigned char*>(rows + AD_CHUNK);
    for (int q = threadIdx.x; q < chunk.z; q += 256) {
        const int row = p.plan[p.o_order + chunk.y + q];
        rows[q] = row;
        if constexpr (KEPT) {
#pragma unroll
            for (int b = 0; b < CW / 2; ++b) scales[b * AD_CHUNK + q] = p.exps[(size_t)min(c0 / 32 + b, (width - 1) / 32) * p.lde + row];
        }
    }
    __syncthreads();
    const unsigned char* const scale = scales + (CW * i / 32) * AD_CHUNK;
    f32x4 acc[RB][CW];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb)
#pragma unroll
        for (int j = 0; j < CW; ++j) acc[rb][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    struct Batch {
        GradRun<JM_BF16, KEPT, CW> x[8];
        float t[RB][8];
    };
    auto fetch = [&](Batch& b, int q0) __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {                        // (rows beyond the chunk: the last one, counted as zeros)
            const int at = min(q0 + 8 * g + e, chunk.z - 1);
            const size_t row = (size_t)rows[at];
            b.x[e].load(p, src, ld, row, c0 + CW * i, width, scale + at);
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) b.t[rb][e] = T[row * p.rank + min(r0 + rb * 16 + i, p.rank - 1)];
        }
    };
    auto multiply = [&](const Batch& b, int q0) __attribute__((always_inline)) {
        unsigned xw[8][4];                                   // two channels a word
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const bool ok = q0 + 8 * g + e < chunk.z;
#pragma unroll
            for (int h = 0; h < 4; ++h) xw[e][h] = ok ? b.x[e].pair(h) : 0u;
        }
        bf16x8 xf[CW];
#pragma unroll
        for (int j = 0; j < CW; ++j) {
            u32x4 w;
#pragma unroll
            for (int h = 0; h < 4; ++h) w[h] = (j & 1) ? pack_hi(xw[2 * h][j / 2], xw[2 * h + 1][j / 2]) : pack_lo(xw[2 * h][j / 2], xw[2 * h + 1][j / 2]);
            xf[j] = __builtin_bit_cast(bf16x8, w);
        }
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
            u32x4 piece[3];
#pragma unroll
            for (int h = 0; h < 4; ++h) {
                unsigned a = q0 + 8 * g + 2 * h < chunk.z ? __float_as_uint(b.t[rb][2 * h]) : 0u;
                unsigned c = q0 + 8 * g + 2 * h + 1 < chunk.z ? __float_as_uint(b.t[rb][2 * h + 1]) : 0u;
#pragma unroll
                for (int s = 0; s < 3; ++s) {
                    piece[s][h] = pack_hi(a, c);
                    if (s < 2) {                             // what the cut left; of an infinity nothing, of a NaN a NaN
                        const float fa = __uint_as_float(a), fc = __uint_as_float(c);
                        a = __builtin_isinf(fa) ? 0u : __float_as_uint(fa - __uint_as_float(a & 0xffff0000u));
                        c = __builtin_isinf(fc) ? 0u : __float_as_uint(fc - __uint_as_float(c & 0xffff0000u));
                    }
                }
            }
#pragma unroll
            for (int s = 2; s >= 0; --s) {
                const bf16x8 tf = __builtin_bit_cast(bf16x8, piece[s]);
#pragma unroll
                for (int j = 0; j < CW; ++j) acc[rb][j] = mma16(acc[rb][j], tf, xf[j]);
            }
        }
    };
    if (chunk.z > 0) {
        for (int q = wave * 32; q < chunk.z; q += STEP) {
            Batch b;
            fetch(b, q);
            multiply(b, q);
        }
    }
    adapter_wgrad_finish<JM_BF16, RB, CW>(p, lds, part, chunk, ad, isA, c0, r0, acc);
}

template <int TY, bool KEPT, int RB, int CW>
__global__ void __launch_bounds__(256)
adapter_wgrad_kernel(AdaptGrad p) {
    __shared__ __attribute__((aligned(16))) float lds[4 * 16 * ad_finish(RB, CW) * 16 * CW];       // the rows of the chunk, then the waves' tiles
    static_assert(sizeof(lds) >= AD_CHUNK * (sizeof(int) + CW / 2), "the row list and the scales are kept there");
    // workgroups are dealt to the 8 XCDs in turn: each takes an eighth of the (chunk, channels, ranks) list, so that the workgroups that read
    // one chunk's rows share an L2
    const int tk = (p.k + 16 * CW - 1) / (16 * CW), ny = tk + (p.n + 16 * CW - 1) / (16 * CW), per = ny * ((p.rank + 16 * RB - 1) / (16 * RB));
    const int total = (p.direct ? p.adapters : p.plan[1]) * per, share = (total + 7) / 8;
    const int item = (int)(blockIdx.x & 7) * share + (int)(blockIdx.x >> 3);
    if ((int)(blockIdx.x >> 3) >= share || item >= total) return;
    const int index = item / per, tile = item % per, r0 = tile / ny * 16 * RB;
    const bool isA = tile % ny < tk;
    const int c0 = (tile % ny - (isA ? 0 : tk)) * 16 * CW;
    int ad = 0;
    int4 chunk;
    if (p.direct) {
        ad = index;
        const int c = p.plan[p.o_chunk_first + ad];
        chunk = make_int4(ad, 0, 0, 0);
        if (p.plan[p.o_chunk_first + ad + 1] > c) chunk = *reinterpret_cast<const int4*>(p.plan + p.o_chunks + 4 * (size_t)c);
    } else {
        chunk = *reinterpret_cast<const int4*>(p.plan + p.o_chunks + 4 * (size_t)index);
    }
    float* const part = p.part + (size_t)index * p.rank * ((size_t)p.k + p.n);
    if constexpr (TY == JM_BF16 && CW == 8) {
        if (KEPT && isA) adapter_wgrad_tile_bf16<KEPT, RB>(p, lds, part, chunk, ad, true, c0, r0);
        else adapter_wgrad_tile_bf16<false, RB>(p, lds, part, chunk, ad, isA, c0, r0);
    } else {
        if (KEPT && isA) adapter_wgrad_tile<TY, KEPT, RB, CW>(p, lds, part, chunk, ad, true, c0, r0);
        else adapter_wgrad_tile<TY, false, RB, CW>(p, lds, part, chunk, ad, isA, c0, r0);
    }
}

// dA, dB of an adapter = s times the sum of its chunks' partials, in chunk order (zero without rows): 4.3 us for four adapters of 32 chunks
template <typename T>
__global__ void __launch_bounds__(256)
adapter_wgrad_reduce_kernel(AdaptGrad p) {
    const int per = p.rank * (p.k + p.n);
    const int e = blockIdx.x * 256 + threadIdx.x, ad = blockIdx.y;
    if (e >= per) return;
    const int c_begin = p.plan[p.o_chunk_first + ad], c_end = p.plan[p.o_chunk_first + ad + 1];
    float s[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};   // eight chains: the loads of consecutive chunks are in flight together
    int c = c_begin;
    for (; c + 8 <= c_end; c += 8)
#pragma unroll
        for (int u = 0; u < 8; ++u) s[u] += p.part[(size_t)(c + u) * per + e];
    for (; c < c_end; ++c) s[0] += p.part[(size_t)c * per + e];
    float v = (((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7]))) * p.scales[ad];
    const int na = p.rank * p.k;
    if (c_begin == c_end) v = 0.f;
    if (e < na) ((T*)p.da)[(size_t)ad * na + e] = (T)v;
    else ((T*)p.db)[(size_t)ad * p.rank * p.n + (e - na)] = (T)v;
}

static size_t elem_size(int type) { return type == JM_F32 ? 4 : 2; }

template <int TY, int RB>
static void launch_rows(const Adapt& p, bool wt, dim3 grid, hipStream_t s) {
    if (wt) hipLaunchKernelGGL((adapter_rows_kernel<TY, RB, 1, true>), grid, dim3(256), 0, s, p);
    else if (ad_tile(p.m) == 16) hipLaunchKernelGGL((adapter_rows_kernel<TY, RB, 1, false>), grid, dim3(256), 0, s, p);
    else hipLaunchKernelGGL((adapter_rows_kernel<TY, RB, 2, false>), grid, dim3(256), 0, s, p);
}
template <int TY>
static void launch_rows(const Adapt& p, bool wt, dim3 grid, hipStream_t s) {
    if (p.rank <= 16) launch_rows<TY, 1>(p, wt, grid, s);
    else if (p.rank <= 32) launch_rows<TY, 2>(p, wt, grid, s);
    else if (p.rank <= 64) launch_rows<TY, 4>(p, wt, grid, s);
    else launch_rows<TY, 8>(p, wt, grid, s);
}
static void launch_rows(int type, const Adapt& p, bool wt, int tiles, hipStream_t s) {
    // few tiles: several workgroups a tile, as far as there are channel blocks and idle CUs
    const int y = imax(1, (int)((long long)divup(p.n, 256) < 256 / tiles ? divup(p.n, 256) : 256 / tiles));
    const dim3 grid((unsigned)tiles, (unsigned)y);
    if (type == JM_F32) launch_rows<JM_F32>(p, wt, grid, s);
    else if (type == JM_BF16) launch_rows<JM_BF16>(p, wt, grid, s);
    else launch_rows<JM_F16>(p, wt, grid, s);
}

// rank indices and channels of a workgroup: 16 x 128, 32 x 128, 64 x 64 (accumulators of a wave: 32, 64, 64 registers); on the bf16 pipe, whose
// operands take more registers, 32 x 128 beyond a rank of 32 too
template <int TY, bool KEPT>
static void launch_wgrad(const AdaptGrad& p, int groups, hipStream_t s) {
    const bool wide = p.rank <= 32 || TY == JM_BF16;
    const int cw = wide ? 128 : 64, rw = p.rank <= 16 ? 16 : (wide ? 32 : 64);
    const dim3 grid((unsigned)(divup(groups * (divup(p.k, cw) + divup(p.n, cw)) * divup(p.rank, rw), 8) * 8)), block(256);
    if (p.rank <= 16) hipLaunchKernelGGL((adapter_wgrad_kernel<TY, KEPT, 1, 8>), grid, block, 0, s, p);
    else if (wide) hipLaunchKernelGGL((adapter_wgrad_kernel<TY, KEPT, 2, 8>), grid, block, 0, s, p);
    else if constexpr (TY != JM_BF16) hipLaunchKernelGGL((adapter_wgrad_kernel<TY, KEPT, 4, 4>), grid, block, 0, s, p);
}

// at, bt: the transposed weights, where they are transposed (tiles of 32 rows); part: the chunks' partials, where there are any
struct GradLayout { size_t at, bt, u, part, total; };        // bytes
static GradLayout grad_layout(int m, int k, int n, int rank, int adapters, int type) {
    const PlanLayout l = plan_layout(m, adapters);
    const size_t transposed = ad_tile(m) == 32 ? (size_t)adapters * rank * elem_size(type) : 0, chunks = m > AD_CHUNK ? l.max_chunks : 0;
    GradLayout g;
    g.at = 0;
    g.bt = align_up(g.at + transposed * k, 256);
    g.u = align_up(g.bt + transposed * n, 256);
    g.part = align_up(g.u + (size_t)imax(m, 1) * rank * 4, 256);
    g.total = g.part + chunks * rank * ((size_t)k + n) * 4;
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
        hipLaunchKernelGGL((adapter_plan_count_kernel<true>), dim3(1), dim3(PL_THREADS), 0, s, m, l.block_rows, adapters, ids, plan, l.order, l.tiles, l.chunks,
                           l.chunk_first, l.hist);
    } else {
        hipLaunchKernelGGL((adapter_plan_count_kernel<false>), dim3((unsigned)l.blocks), dim3(PL_THREADS), 0, s, m, l.block_rows, adapters, ids, plan, l.order, l.tiles,
                           l.chunks, l.chunk_first, l.hist);
        hipLaunchKernelGGL(adapter_plan_scatter_kernel, dim3((unsigned)l.blocks), dim3(PL_THREADS), 0, s, m, l.block_rows, adapters, ids, plan, l.order, l.tiles,
                           l.chunks, l.chunk_first, l.hist);
    }
    return check_launch("adapter_plan");
}

int jm_adapter_forward(int m, int k, int n, int rank, int adapters, int type, const void* x, long long ldx, const void* a, const void* b,
                       const float* scales, const int* plan, const void* base, long long ldb, void* out, long long ldo, float* t, jm_stream_t stream) {
    if (int e = adapter_check("adapter_forward", m, k, n, rank, adapters, type)) return e;
    JM_REQUIRE(ldx >= k && ldo >= n && (!base || ldb >= n), "adapter_forward: ldx %lld, ldb %lld, ldo %lld for k %d, n %d", ldx, ldb, ldo, k, n);
    JM_REQUIRE(m <= 1 || !base || base != out || ldb == ldo, "adapter_forward: in place with rows %lld and %lld apart", ldb, ldo);
    if (m == 0) return JM_OK;
    JM_REQUIRE(x && a && b && scales && plan && out, "adapter_forward: NULL buffers");
    const PlanLayout l = plan_layout(m, adapters);
    Adapt p{};
    p.m = m; p.k = k; p.n = n; p.rank = rank; p.plan = plan; p.o_order = l.order; p.o_tiles = l.tiles; p.x = x; p.ldx = ldx; p.a = a; p.b = b;
    p.scales = scales; p.base = base; p.ldb = ldb; p.out = out; p.ldo = ldo; p.t = t; p.copy = base != out;
    launch_rows(type, p, false, l.max_tiles, (hipStream_t)stream);
    return check_launch("adapter_forward");
}

size_t jm_adapter_grad_workspace_bytes(int m, int k, int n, int rank, int adapters, int type) {
    if (m < 0 || m > AD_MAX_ROWS || k <= 0 || k > AD_MAX_WIDTH || n <= 0 || n > AD_MAX_WIDTH || rank <= 0 || rank > JM_ADAPTER_MAX_RANK || adapters <= 0 || adapters > PL_MAX_ADAPTERS) return 0;
    return grad_layout(m, k, n, rank, adapters, type).total;
}

int jm_adapter_grad_select(int results, int m, int k, int n, int rank, int adapters, int type, const void* dy, long long lddy, const void* x, long long ldx,
                           const unsigned char* codes, int ldc, const unsigned char* exps, int lde, const float* t, const void* a, const void* b, const float* scales,
                           const int* plan, const void* base, long long ldb, void* dx, long long lddx, void* da, void* db, void* ws, size_t ws_bytes,
                           jm_stream_t stream) {
    if (int e = adapter_check("adapter_grad", m, k, n, rank, adapters, type)) return e;
    JM_REQUIRE(results >= 0 && results <= (JM_ADAPTER_DX | JM_ADAPTER_DA | JM_ADAPTER_DB), "adapter_grad: results %d", results);
    const bool want_dx = results & JM_ADAPTER_DX, want_da = results & JM_ADAPTER_DA, want_db = results & JM_ADAPTER_DB;
    JM_REQUIRE(lddy >= n && (!want_dx || (lddx >= k && (!base || ldb >= k))), "adapter_grad: lddy %lld, ldb %lld, lddx %lld for k %d, n %d", lddy, ldb, lddx, k, n);
    JM_REQUIRE(m <= 1 || !want_dx || !base || base != dx || ldb == lddx, "adapter_grad: in place with rows %lld and %lld apart", ldb, lddx);
    JM_REQUIRE(!want_da || (x ? ldx >= k : (m == 0 || (codes && exps && ldc >= k && ldc % 16 == 0 && lde >= m && lde % 16 == 0 && (((uintptr_t)codes | (uintptr_t)exps) & 15) == 0))),
               "adapter_grad: x or its kept rows are needed (ldx %lld, ldc %d, k %d)", ldx, ldc, k);
    JM_REQUIRE(a && b && scales && plan && (!want_da || da) && (!want_db || db) && (m == 0 || (dy && (!want_db || t) && (!want_dx || dx))), "adapter_grad: NULL buffers");
    const GradLayout gl = grad_layout(m, k, n, rank, adapters, type);
    if (!ws || ws_bytes < gl.total || ((uintptr_t)ws & 15)) {
        set_error("adapter_grad: workspace of %zu bytes (16-byte aligned), need %zu", ws_bytes, gl.total);
        return JM_EWORKSPACE;
    }
    hipStream_t s = (hipStream_t)stream;
    const PlanLayout l = plan_layout(m, adapters);
    char* w = (char*)ws;
    AdaptGrad q{};
    // (a weight gradient that is not wanted is a matrix without channels)
    q.m = m; q.k = want_da ? k : 0; q.n = want_db ? n : 0; q.rank = rank; q.adapters = adapters; q.plan = plan; q.o_order = l.order; q.o_chunks = l.chunks;
    q.o_chunk_first = l.chunk_first; q.x = x; q.ldx = ldx; q.codes = codes; q.ldc = ldc; q.exps = exps; q.lde = lde;
    q.dy = dy; q.lddy = lddy; q.t = t; q.u = (const float*)(w + gl.u); q.scales = scales; q.part = (float*)(w + gl.part); q.direct = m > 0 && m <= AD_CHUNK; q.da = da; q.db = db;
    const int groups = q.direct ? adapters : l.max_chunks;
    JM_REQUIRE((long long)groups * (divup(k, 64) + divup(n, 64)) * divup(rank, 16) < 1 << 24, "adapter_grad: too many (chunk, tile) pairs (m %d, k %d, n %d, rank %d)", m, k, n, rank);
    if (m > 0 && (want_dx || want_da)) {
        const bool wt = ad_tile(m) == 16;
        if (!wt) {
            const dim3 gt((unsigned)((divup(k, 32) + divup(n, 32)) * divup(rank, 32)), (unsigned)adapters);
            if (type == JM_F32) {
                hipLaunchKernelGGL((adapter_transpose_kernel<float>), gt, dim3(256), 0, s, rank, k, n, (const float*)a, (float*)(w + gl.at), (const float*)b, (float*)(w + gl.bt));
            } else {
                typedef unsigned short u16;
                hipLaunchKernelGGL((adapter_transpose_kernel<u16>), gt, dim3(256), 0, s, rank, k, n, (const u16*)a, (u16*)(w + gl.at), (const u16*)b, (u16*)(w + gl.bt));
            }
        }
        // (without dx: outputs without channels, u only)
        Adapt p{};
        p.m = m; p.k = n; p.n = want_dx ? k : 0; p.rank = rank; p.plan = plan; p.o_order = l.order; p.o_tiles = l.tiles; p.x = dy; p.ldx = lddy;
        p.a = wt ? b : w + gl.bt; p.b = wt ? a : w + gl.at; p.scales = scales; p.base = base; p.ldb = ldb; p.out = dx; p.ldo = lddx;
        p.t = want_da ? (float*)(w + gl.u) : nullptr;
        p.copy = want_dx && base != dx;
        launch_rows(type, p, wt, l.max_tiles, s);
    }
    if (!want_da && !want_db) return check_launch("adapter_grad");
    if (m > 0) {
        if (x || !want_da) {
            if (type == JM_F32) launch_wgrad<JM_F32, false>(q, groups, s);
            else if (type == JM_BF16) launch_wgrad<JM_BF16, false>(q, groups, s);
            else launch_wgrad<JM_F16, false>(q, groups, s);
        } else {
            if (type == JM_F32) launch_wgrad<JM_F32, true>(q, groups, s);
            else if (type == JM_BF16) launch_wgrad<JM_BF16, true>(q, groups, s);
            else launch_wgrad<JM_F16, true>(q, groups, s);
        }
    }
    if (q.direct) return check_launch("adapter_grad");
    const dim3 gr((unsigned)divup(rank * (q.k + q.n), 256), (unsigned)adapters);
    if (type == JM_F32) hipLaunchKernelGGL((adapter_wgrad_reduce_kernel<float>), gr, dim3(256), 0, s, q);
    else if (type == JM_BF16) hipLaunchKernelGGL((adapter_wgrad_reduce_kernel<__bf16>), gr, dim3(256), 0, s, q);
    else hipLaunchKernelGGL((adapter_wgrad_reduce_kernel<_Float16>), gr, dim3(256), 0, s, q);
    return check_launch("adapter_grad");
}

int jm_adapter_grad(int m, int k, int n, int rank, int adapters, int type, const void* dy, long long lddy, const void* x, long long ldx,
                    const unsigned char* codes, int ldc, const unsigned char* exps, int lde, const float* t, const void* a, const void* b, const float* scales,
                    const int* plan, const void* base, long long ldb, void* dx, long long lddx, void* da, void* db, void* ws, size_t ws_bytes,
                    jm_stream_t stream) {
    return jm_adapter_grad_select(JM_ADAPTER_DX | JM_ADAPTER_DA | JM_ADAPTER_DB, m, k, n, rank, adapters, type, dy, lddy, x, ldx, codes, ldc, exps, lde, t, a, b, scales,
                                  plan, base, ldb, dx, lddx, da, db, ws, ws_bytes, stream);
}

}  // extern "C"
