// rows8.hip — activations kept in 8 bits between the forward and the backward pass of the row layers (rows_gemm.hip), and their use in
// the backward pass.
//
// Format.  A row tensor X (m, c) is kept as e4m3 codes (m, ldc) plus one scale byte per 32 consecutive channels of a row:
//     amax  = the largest finite |x| of the block;  2^e = the smallest power of two with amax <= 448 2^e, e >= -100 (empty block: -100)
//     code  = x / 2^e rounded to the nearest e4m3 value, ties to even;  scale byte = e + 127
// (the scale bytes of one block of channels lie together, (blocks, lde >= m): the scales of many rows are one load for the weight gradient)
// with two exceptions: a value that is not zero never becomes zero (it takes the smallest code of its sign, 2^-9 2^e, so that the sign
// pattern — a ReLU's mask — survives), and a value that is not finite becomes the NaN code 0x7f (e4m3 has no infinity).
// Why e4m3 with power-of-two scales: the division is exact, so the codes are a defined rounding of the input (half a step, 2^-4
// relative, within 2^14 of the block's maximum) whatever computes them; and a kept value, 4 significant bits times a power of two, is
// exact in bfloat16, so the backward's products run on the bf16 matrix pipe without another rounding of X.
// 1.03 bytes per element instead of 4 (float32) or 2.
#include "jm_elem.h"
#include "jm_rows.h"
#include <type_traits>

namespace jm {

constexpr int R8_BLOCK = 32;         // channels per scale
constexpr int R8_MAX_ROWS = 1 << 30, R8_MAX_WIDTH = 1 << 22;        // (32-bit row counters, and offsets of up to 128 rows of codes)
constexpr long long R8_MAX_LD = 1 << 22;      // (128 rows of it are addressed by 32-bit offsets there)
constexpr int R8_GRID = 4096;         // workgroups of the element-wise kernels: 16 a CU, then they walk
constexpr int R8_EMIN = -100;        // least scale exponent: 2^e and the smallest code 2^(e - 9) stay normal in float32 and bfloat16

__device__ __forceinline__ float exp2i(int e) { return __uint_as_float((unsigned)(e + 127) << 23); }      // -126 <= e <= 127
__device__ __forceinline__ bool finite_bits(unsigned b) { return (b & 0x7f800000u) != 0x7f800000u; }

// the scale exponent of a block from the bits of its largest finite |x|
__device__ __forceinline__ int r8_exponent(unsigned amax_bits) {
    const int e = (int)(amax_bits >> 23) - 127 - 8 + ((amax_bits & 0x7fffffu) > 0x600000u ? 1 : 0);      // 448 = 1.75 x 2^8
    return max(e, R8_EMIN);
}

// a thread's walk over the (row, 8 channels) items of a matrix in memory order, `step` items at a time: one division at the start
struct R8Walk {
    long long row;
    int grp;
    __device__ __forceinline__ R8Walk(long long it, int groups) : row(it <= 0x7fffffffll ? (long long)((unsigned)it / (unsigned)groups) : it / groups) {
        grp = (int)(it - row * groups);
    }
    __device__ __forceinline__ void advance(long long rows, int grps, int groups) {
        row += rows;
        grp += grps;
        if (grp >= groups) { grp -= groups; ++row; }
    }
};

// Four lanes hold a block, 8 channels each; the block's maximum by two quad permutations.  One read of X, one write of the codes: bound
// by memory.  A value's smallest magnitude is raised to the smallest code before the conversion (zeros keep zero); values that are not
// finite are looked for once a wave.  65536 x 128 float32: 9 us (4.7 TB/s); 100003 x 196 bfloat16: 17 us (3.6 TB/s).
template <int TY>
__global__ void __launch_bounds__(256)
rows8_pack_kernel(int m, int lde, int c, int groups, const typename Elem<TY>::T* __restrict__ x, long long ldx, unsigned char* __restrict__ codes, int ldc,
                  unsigned char* __restrict__ exps) {
    typedef typename Elem<TY>::V8 V8;
    const long long step = gridDim.x * 256ll, rows = step / groups;
    const int grps = (int)(step - rows * groups);
    for (R8Walk w(blockIdx.x * 256ll + threadIdx.x, groups); w.row < m; w.advance(rows, grps, groups)) {
        const int left = c - w.grp * 8;
        const typename Elem<TY>::T* src = x + w.row * ldx + w.grp * 8;
        V8 raw;
        if (left > 0 && (long long)(m - 1 - w.row) * ldx + left >= 8) {      // (behind a row's end what lies there inside X is read and not used)
            raw = load8<V8>(src);
#pragma unroll
            for (int e = 1; e < 8; ++e) raw[e] = e < left ? raw[e] : (typename Elem<TY>::T)0.f;
        } else {
            raw = load8_tail<V8>(src, left);
        }
        float v[8];
        unsigned top = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            v[e] = (float)raw[e];
            top = max(top, __float_as_uint(v[e]) & 0x7fffffffu);
        }
        unsigned bad = 0;                                    // bit e: element e is not finite
        if (__ballot(top >= 0x7f800000u)) {
            top = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const unsigned b = __float_as_uint(v[e]) & 0x7fffffffu;
                if (b >= 0x7f800000u) { bad |= 1u << e; v[e] = 0.f; }
                else top = max(top, b);
            }
        }
        top = max(top, (unsigned)__builtin_amdgcn_update_dpp(0, (int)top, JM_DPP_XOR1, 0xf, 0xf, true));
        top = max(top, (unsigned)__builtin_amdgcn_update_dpp(0, (int)top, JM_DPP_XOR2, 0xf, 0xf, true));
        const int e2 = r8_exponent(top);
        const float inv = exp2i(-e2);
        float f[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = copysignf(fmaxf(fabsf(v[e] * inv), v[e] != 0.f ? 0x1p-9f : 0.f), v[e]);
        unsigned o[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            int p = __builtin_amdgcn_cvt_pk_fp8_f32(f[4 * h], f[4 * h + 1], 0, false);
            o[h] = (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(f[4 * h + 2], f[4 * h + 3], p, true);
        }
        if (bad)
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (bad >> e & 1u) o[e >> 2] = (o[e >> 2] & ~(0xffu << (8 * (e & 3)))) | (0x7fu << (8 * (e & 3)));
        if (w.grp * 8 < ldc) *reinterpret_cast<uint2*>(codes + w.row * ldc + w.grp * 8) = make_uint2(o[0], o[1]);
        if ((w.grp & 3) == 0) exps[(size_t)(w.grp >> 2) * lde + w.row] = (unsigned char)(e2 + 127);
    }
}

__device__ __forceinline__ void r8_decode4(unsigned w, float scale, float (&v)[4]) {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false);
    const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    v[0] = lo[0] * scale; v[1] = lo[1] * scale; v[2] = hi[0] * scale; v[3] = hi[1] * scale;
}

// One read of the codes, one write of the values: bound by memory.  65536 x 128 float32: 10.6 us (4 TB/s); 100003 x 196 bfloat16: 12 us (5 TB/s).
template <int TY>
__global__ void __launch_bounds__(256)
rows8_restore_kernel(int m, int lde, int c, int groups, const unsigned char* __restrict__ codes, int ldc, const unsigned char* __restrict__ exps,
                     typename Elem<TY>::T* __restrict__ out, long long ldo) {
    typedef typename Elem<TY>::T T;
    typedef typename Elem<TY>::V8 V8;
    const long long step = gridDim.x * 256ll, rows = step / groups;
    const int grps = (int)(step - rows * groups);
    for (R8Walk at(blockIdx.x * 256ll + threadIdx.x, groups); at.row < m; at.advance(rows, grps, groups)) {
        const long long row = at.row;
        const int grp = at.grp;
        const uint2 w = *reinterpret_cast<const uint2*>(codes + row * ldc + grp * 8);
        const float scale = exp2i((int)exps[(size_t)(grp >> 2) * lde + row] - 127);
        float v[8];
        r8_decode4(w.x, scale, *reinterpret_cast<float (*)[4]>(&v[0]));
        r8_decode4(w.y, scale, *reinterpret_cast<float (*)[4]>(&v[4]));
        V8 o;
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = (T)v[e];
        T* dst = out + row * ldo + grp * 8;
        const int n = c - grp * 8;
        if (n >= 8) {
            store8(dst, o);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (e < n) dst[e] = o[e];
        }
    }
}

// out = (the kept value > 0) ? dy : 0 — the gradient through a ReLU whose output was kept.  A ReLU's output is never negative, so the code of
// values that are not finite stands for +infinity there and counts as positive.  out may be dy.  Four channels a lane, 9 bytes
// moved an element: bound by memory.  65536 x 128: 12 us (6.2 TB/s), 131072 x 512: 115 us (5.2 TB/s); 512 x 512: 2.6 us.
__global__ void __launch_bounds__(256)
rows8_relu_mask_kernel(int m, int c, int groups, const float* dy, long long ldd, const unsigned char* __restrict__ codes, int ldc, float* out, long long ldo) {
    const long long step = gridDim.x * 256ll, rows = step / groups;
    const int grps = (int)(step - rows * groups);
    for (R8Walk at(blockIdx.x * 256ll + threadIdx.x, groups); at.row < m; at.advance(rows, grps, groups)) {
        const int c0 = at.grp * 4;
        const unsigned w = *reinterpret_cast<const unsigned*>(codes + at.row * ldc + c0);
        const float* src = dy + at.row * ldd + c0;
        float* dst = out + at.row * ldo + c0;
        auto on = [&](int q) { const unsigned b = (w >> (8 * q)) & 0xffu; return b != 0u && b < 0x80u; };
        if (c0 + 4 <= c) {
            f32x4 v;
            __builtin_memcpy(&v, src, 16);
#pragma unroll
            for (int q = 0; q < 4; ++q) v[q] = on(q) ? v[q] : 0.f;
            __builtin_memcpy(dst, &v, 16);
        } else {
            for (int q = 0; c0 + q < c; ++q) dst[q] = on(q) ? src[q] : 0.f;
        }
    }
}

// ------------------------------------------------------------------------------------------------ weight gradient from kept rows
// dW (n, k) = dY (m, n)^T X (m, k), db (n) = column sums of dY.
//
// On the bf16 matrix pipe although dW is a float32 result: a kept value is exact in bfloat16, and a gradient is the sum of bfloat16
// pieces without any rounding — a float32 value of three (24 significant bits = 8 + 8 + 8, cut off, not rounded), a float16 value of two, a
// bfloat16 value of one — so every product is exact and only the float32 additions round, as on the float32 pipe, at a third of sixteen
// times its rate.
//
// Workgroup = a 128 x 128 (64 x 64) tile of dW over one split of the rows, 64 (128) rows a step.  A thread fetches 8 rows x 4 columns of both
// operands, cuts and converts them, and stores 8 rows of one column as 16 bytes: the contraction index becomes the fast one on the way
// into LDS, and a matrix operand (8 rows of a column) is one 16-byte read.  In LDS column 4 i + q of a tile sits in slot (T / 4) q + i:
// writes and reads of a wave are contiguous.
// Two groups of four waves take the steps in turn: while one cuts and stores its step (about 250 vector instructions a wave in float32),
// the other multiplies its own (48 matrix instructions of 32 x 32 x 16 a wave) and asks for its next rows between them; their sums are
// added through LDS at the end, so a CU writes one partial tile.  The splits' partials are added in split order by the second kernel (no
// float atomics: the same bits every time).
// Measured (float32 | bfloat16 gradients, both kernels, alone and on inputs that change from call to call): 65536 x 256 x 256 41 | 28 us, 131072 x
// 512 x 512 249 | 127 us; calls one behind the other 37 us for the first and 108 for the last (93 on the same inputs again, which the caches then
// hold in part) — 0.7 and 0.63 PFLOP/s on the bf16 pipe, where a library product of 8192^3 reaches 1.4; 512 x 512 x 512 9.7 | 7.5 us.  No one unit
// bounds it: copies of the kernel with only the staging and LDS reads, only the products or only the loads took 70, 57 and 56 us of the 97 that
// the whole took then on the same inputs; what is lost is their overlap.  (Two steps between barriers: 2 % less; a tile of 128 x 256: registers spill.)
constexpr int W8_SLAB = 8192;          // elements of one operand piece of a step: 64 rows x 128 columns or 128 x 64

struct Wgrad8 {
    int m, n, k, splits, rows_per;       // rows_per: rows of a split, a multiple of a step's
    const void* dy; long long lddy;
    const unsigned char* codes; int ldc; const unsigned char* exps; int lde, blocks;
    float *dw, *db;                      // (splits, n, k) and (splits, n) partials, or the results when splits == 1
    long long lddw;
};

// four consecutive columns of a row.  The columns of a group that lies outside the matrix are whatever lies inside (they only reach
// outputs that are never stored); a group that straddles the edge (`ragged`, widths that are no multiple of 4) is read from width - 4 and shifted
// (16-bit rows of an odd width in rows of an even stride: that read starts 2 bytes off a word and is exact, the bits of the column-by-column route)
template <int TY> struct Quad;
template <> struct Quad<JM_F32> {
    f32x4 v;
    __device__ __forceinline__ void load(const float* p) { __builtin_memcpy(&v, p, 16); }
    __device__ __forceinline__ void shift(int n) {
        if (n & 1) { v[0] = v[1]; v[1] = v[2]; v[2] = v[3]; }
        if (n & 2) { v[0] = v[2]; v[1] = v[3]; }
    }
    __device__ __forceinline__ void zero() { v = f32x4{0.f, 0.f, 0.f, 0.f}; }
    __device__ __forceinline__ float get(int q) const { return v[q]; }
};
template <int TY> struct Quad16 {
    unsigned v[2];
    __device__ __forceinline__ void load(const typename Elem<TY>::T* p) { __builtin_memcpy(v, p, 8); }
    __device__ __forceinline__ void shift(int n) {
        if (n & 1) { v[0] = (v[0] >> 16) | (v[1] << 16); v[1] >>= 16; }
        if (n & 2) v[0] = v[1];
    }
    __device__ __forceinline__ void zero() { v[0] = v[1] = 0u; }
    template <typename V2> __device__ __forceinline__ void set(const V2& w) { v[0] = w[0]; v[1] = w[1]; }
    __device__ __forceinline__ unsigned word(int q) const { return v[q >> 1]; }
    __device__ __forceinline__ float get(int q) const {
        const unsigned short h = (unsigned short)(v[q >> 1] >> (16 * (q & 1)));
        typename Elem<TY>::T t;
        __builtin_memcpy(&t, &h, 2);
        return (float)t;
    }
};
template <> struct Quad<JM_BF16> : Quad16<JM_BF16> {};
template <> struct Quad<JM_F16> : Quad16<JM_F16> {};

template <int TY, bool SMALL, int W8_T>
__global__ void __launch_bounds__(512, 1)
rows8_wgrad_kernel(Wgrad8 p) {
    typedef typename Elem<TY>::T T;
    constexpr int W8_R = W8_SLAB / W8_T, G = W8_T / 4, BL = W8_T / 64;          // rows of a step; column groups; 32-wide blocks of a wave a side
    constexpr int P = TY == JM_F32 ? 3 : (TY == JM_F16 ? 2 : 1);                  // pieces of a gradient
    typedef __bf16 frag_t __attribute__((ext_vector_type(8)));
    typedef float f32x16 __attribute__((ext_vector_type(16)));
    extern __shared__ __attribute__((aligned(16))) unsigned short lds_all[];
    constexpr int BUF = (P + 1) * W8_SLAB;                   // one step's operands; two buffers
    const int grp = __builtin_amdgcn_readfirstlane(threadIdx.x >> 8);
    const int tid = threadIdx.x & 255, lane = tid & 63, wave = tid >> 6;
    // workgroups are dealt to the 8 XCDs in turn: each XCD takes an eighth of the (split, tile) list, so that the tiles of one split, which
    // read the same rows, share an L2
    const int tk = (p.k + W8_T - 1) / W8_T, tiles = ((p.n + W8_T - 1) / W8_T) * tk, total = tiles * p.splits;
    const int item = (int)(blockIdx.x & 7) * ((total + 7) / 8) + (int)(blockIdx.x >> 3);
    if ((int)(blockIdx.x >> 3) >= (total + 7) / 8 || item >= total) return;
    const int split = item / tiles, tile = item % tiles;
    const int n0 = (tile / tk) * W8_T, k0 = (tile % tk) * W8_T;
    const int r_begin = (int)min((long long)split * p.rows_per, (long long)p.m), r_end = (int)min((long long)p.m, (long long)r_begin + p.rows_per);

    // fetch: rows 8 oct .. + 7 of the 64, columns 4 l .. + 3 of both tiles
    const int l = tid % G, oct = tid / G;
    const int cy = n0 + 4 * l, cx = min(k0 + 4 * l, p.ldc - 4);
    const int ylast = p.n - 4;
    const int ysh = (!SMALL && cy < p.n) ? max(0, cy - ylast) : 0;
    const bool ragged = !SMALL && (p.n & 3) != 0 && n0 + W8_T > p.n;
    const int ycol = min(cy, max(ylast, 0));
    struct Rows {
        Quad<TY> y[8];
        unsigned x[8];
        unsigned long long e;                                // the rows' scales
    };
    Rows rows;
    const unsigned char* const ep = p.exps + (size_t)min(cx / R8_BLOCK, p.blocks - 1) * p.lde;
    const unsigned yo = ((unsigned)(8 * oct) * (unsigned)p.lddy + (unsigned)ycol) * (unsigned)sizeof(T), xo = (unsigned)(8 * oct) * (unsigned)p.ldc + (unsigned)cx;
    // rows q0 .. q1 - 1 of the lane's eight of the step at row r; rows behind the split are read as zeros (bounds of the buffers)
    auto fetch = [&](Rows& d, int r, int q0, int q1) __attribute__((always_inline)) {
        const int left = min(W8_R, r_end - r);
        if (q0 == 0) d.e = *reinterpret_cast<const unsigned long long*>(ep + min(r + 8 * oct, p.lde - 8));
        const unsigned char* xr = p.codes + (long long)r * p.ldc;
        const auto xbuf = __builtin_amdgcn_make_buffer_rsrc((void*)xr, 0, (unsigned)left * (unsigned)p.ldc, 0x00020000);
        const T* yr = (const T*)p.dy + (long long)r * p.lddy;
        const auto ybuf = __builtin_amdgcn_make_buffer_rsrc((void*)yr, 0, ((unsigned)(left - 1) * (unsigned)p.lddy + (unsigned)p.n) * (unsigned)sizeof(T), 0x00020000);
#pragma unroll
        for (int q = 0; q < 8; ++q) {
            if (q < q0 || q >= q1) continue;
            d.x[q] = __builtin_amdgcn_raw_buffer_load_b32(xbuf, xo + (unsigned)(q * p.ldc), 0, 0);
            if constexpr (SMALL) {                           // fewer than 4 columns, or rows that are not aligned to 4 bytes
                const T* dy = yr + (long long)min(8 * oct + q, left - 1) * p.lddy;
                T t[4];
#pragma unroll
                for (int c = 0; c < 4; ++c) t[c] = dy[min(cy + c, p.n - 1)];
                d.y[q].load(t);
                if (8 * oct + q >= left) d.y[q].zero();
            } else if constexpr (TY == JM_F32) {
                d.y[q].v = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(ybuf, yo + (unsigned)(q * (int)p.lddy * 4), 0, 0));
            } else {
                d.y[q].set(__builtin_amdgcn_raw_buffer_load_b64(ybuf, yo + (unsigned)(q * (int)p.lddy * 2), 0, 0));
            }
        }
    };
    float bs[4] = {0.f, 0.f, 0.f, 0.f};
    // the bias sums of a split's rows: step i is the tile column i mod tk's, so that no workgroup has all of them (one split: its first column's)
    const int kt = tile % tk;
    const bool do_bias = p.db != nullptr && (p.splits > 1 || kt == 0);
    // before a step's rows are staged: rows behind the split count as zeros on both sides, columns that straddle the edge, the bias sums.
    // Returns whether the wave holds an infinity (looked for once: its rest must be nothing, inf - inf would be NaN; a NaN's rest is a NaN).
    auto prepare = [&](Rows& d, int r) __attribute__((always_inline)) -> bool {
        Quad<TY>(&y)[8] = d.y;
        if (r + W8_R > r_end) {                              // (the scales behind the matrix are not written: any power of two for the zeros there)
#pragma unroll
            for (int q = 0; q < 8; ++q)
                if (r + 8 * oct + q >= r_end) d.e = (d.e & ~(0xffull << (8 * q))) | (127ull << (8 * q));
        }
        if (ragged) {
#pragma unroll
            for (int q = 0; q < 8; ++q) y[q].shift(ysh);
        }
        if (do_bias && (p.splits == 1 || ((r - r_begin) / W8_R) % tk == kt)) {
#pragma unroll
            for (int c = 0; c < 4; ++c)                      // (pairs of pairs: an addition rounds at most 3 times before the step's sum)
                bs[c] += ((y[0].get(c) + y[1].get(c)) + (y[2].get(c) + y[3].get(c))) + ((y[4].get(c) + y[5].get(c)) + (y[6].get(c) + y[7].get(c)));
        }
        if constexpr (P > 1) {
            float top = 0.f;
#pragma unroll
            for (int q = 0; q < 8; ++q)
#pragma unroll
                for (int c = 0; c < 4; c += 2) asm("v_max3_f32 %0, |%1|, |%2|, %0" : "+v"(top) : "v"(y[q].get(c)), "v"(y[q].get(c + 1)));
            return __ballot(top == __builtin_inff()) != 0ull;
        }
        return false;
    };
    auto stage = [&](auto special_, Rows& d, unsigned short* lds) __attribute__((always_inline)) {
        Quad<TY>(&y)[8] = d.y;
        u32x4* Y = reinterpret_cast<u32x4*>(lds) + oct * W8_T + l;          // 16 bytes = 8 rows of a slot
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            u32x4 w[P];
#pragma unroll
            for (int h = 0; h < 4; ++h) {
                if constexpr (TY == JM_BF16) {
                    w[0][h] = (c & 1) ? pack_hi(y[2 * h].word(c), y[2 * h + 1].word(c)) : pack_lo(y[2 * h].word(c), y[2 * h + 1].word(c));
                } else {
                    unsigned a = __float_as_uint(y[2 * h].get(c)), b = __float_as_uint(y[2 * h + 1].get(c));
#pragma unroll
                    for (int s = 0; s < P; ++s) {
                        w[s][h] = pack_hi(a, b);
                        if (s + 1 < P) {
                            const float fa = __uint_as_float(a), fb = __uint_as_float(b);
                            const float ra = fa - __uint_as_float(a & 0xffff0000u), rb = fb - __uint_as_float(b & 0xffff0000u);
                            a = (decltype(special_)::value && __builtin_isinf(fa)) ? 0u : __float_as_uint(ra);
                            b = (decltype(special_)::value && __builtin_isinf(fb)) ? 0u : __float_as_uint(rb);
                        }
                    }
                }
            }
#pragma unroll
            for (int s = 0; s < P; ++s) Y[s * (W8_SLAB / 8) + c * G] = w[s];
        }
        // kept values: codes of a row share a scale within the four columns
        unsigned v0[8], v1[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) {
            const unsigned half = (unsigned)(d.e >> (q < 4 ? 0 : 32));
            const float sc = __uint_as_float(((half >> (8 * (q & 3))) & 0xffu) << 23);
            const auto lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)d.x[q], sc, false);
            const auto hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)d.x[q], sc, true);
            __builtin_memcpy(&v0[q], &lo, 4);
            __builtin_memcpy(&v1[q], &hi, 4);
        }
        u32x4* X = Y + P * (W8_SLAB / 8);
        u32x4 w0, w1, w2, w3;
#pragma unroll
        for (int h = 0; h < 4; ++h) {
            w0[h] = pack_lo(v0[2 * h], v0[2 * h + 1]);
            w1[h] = pack_hi(v0[2 * h], v0[2 * h + 1]);
            w2[h] = pack_lo(v1[2 * h], v1[2 * h + 1]);
            w3[h] = pack_hi(v1[2 * h], v1[2 * h + 1]);
        }
        X[0] = w0; X[G] = w1; X[2 * G] = w2; X[3 * G] = w3;
    };

    const int wn = wave >> 1, wk = wave & 1, lr = lane & 31, lk = lane >> 5;
    f32x16 acc[BL][BL];
#pragma unroll
    for (int a = 0; a < BL; ++a)
#pragma unroll
        for (int b = 0; b < BL; ++b)
#pragma unroll
            for (int q = 0; q < 16; ++q) acc[a][b][q] = 0.f;
    // one step's products, and the next one's rows asked for in between: a load waits for its turn at the L1's port, and a wave that waits
    // there in one go leaves the matrix pipe idle
    auto multiply = [&](unsigned short* lds, Rows& d, int r) __attribute__((always_inline)) {
        const u32x4* Y = reinterpret_cast<const u32x4*>(lds);
        const u32x4* X = Y + P * (W8_SLAB / 8);
        frag_t xb[2][BL], ya[2][P][BL];
        auto read = [&](int s) __attribute__((always_inline)) {
            const int at = (2 * s + lk) * W8_T + lr;
#pragma unroll
            for (int b = 0; b < BL; ++b) xb[s & 1][b] = __builtin_bit_cast(frag_t, X[at + (BL * wk + b) * 32]);
#pragma unroll
            for (int c = P - 1; c >= 0; --c)
#pragma unroll
                for (int a = 0; a < BL; ++a) ya[s & 1][c][a] = __builtin_bit_cast(frag_t, Y[c * (W8_SLAB / 8) + at + (BL * wn + a) * 32]);
        };
        constexpr int KS = W8_R / 16;
        const bool more = r < r_end;
        read(0);
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            if (s + 1 < KS) read(s + 1);                     // the next operands are on their way while these are multiplied
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int c = P - 1; c >= 0; --c)
#pragma unroll
                for (int a = 0; a < BL; ++a)
#pragma unroll
                    for (int b = 0; b < BL; ++b) acc[a][b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ya[s & 1][c][a], xb[s & 1][b], acc[a][b], 0, 0, 0);
            if (more) fetch(d, r, s * 8 / KS, (s + 1) * 8 / KS);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    const int steps = (r_end - r_begin + W8_R - 1) / W8_R;
    // group g takes the steps g, g + 2, ...; the barriers put one group's staging beside the other's products (2 turns + 1 for both;
    // lds_barrier leaves loads in flight)
    const int first = r_begin + grp * W8_R, turns = (steps + 1) / 2;
    unsigned short* lds = lds_all + grp * BUF;
    if (first < r_end) fetch(rows, first, 0, 8);
    auto put = [&](int r) __attribute__((always_inline)) {
        if (r >= r_end) return;
        if (prepare(rows, r)) stage(std::true_type{}, rows, lds);
        else stage(std::false_type{}, rows, lds);
    };
    if (grp == 0) {
        put(first);
        lds_barrier();
        for (int t = 0; t < turns; ++t) {
            multiply(lds, rows, first + (t + 1) * 2 * W8_R);
            lds_barrier();
            put(first + (t + 1) * 2 * W8_R);
            lds_barrier();
        }
    } else {
        lds_barrier();
        for (int t = 0; t < turns; ++t) {
            const int r = first + t * 2 * W8_R;
            put(r);
            lds_barrier();
            if (r < r_end) multiply(lds, rows, r + 2 * W8_R);
            lds_barrier();
        }
    }
    float* red = reinterpret_cast<float*>(lds_all);
    if (grp == 1) {
#pragma unroll
        for (int a = 0; a < BL; ++a)
#pragma unroll
            for (int b = 0; b < BL; ++b)
#pragma unroll
                for (int q = 0; q < 16; ++q) red[((a * BL + b) * 16 + q) * 256 + tid] = acc[a][b][q];
    }
    __syncthreads();
    if (grp == 0) {
#pragma unroll
        for (int a = 0; a < BL; ++a)
#pragma unroll
            for (int b = 0; b < BL; ++b)
#pragma unroll
                for (int q = 0; q < 16; ++q) acc[a][b][q] += red[((a * BL + b) * 16 + q) * 256 + tid];
    }

    float* dw = p.dw + (p.splits > 1 ? (size_t)split * p.n * p.k : 0);
    auto column = [&](int slot) { return 4 * (slot % G) + slot / G; };
    if (grp == 0) {
#pragma unroll
        for (int a = 0; a < BL; ++a)
#pragma unroll
            for (int q = 0; q < 16; ++q) {
                const int n = n0 + column((BL * wn + a) * 32 + (q & 3) + 8 * (q >> 2) + 4 * lk);
                if (n < p.n) {
#pragma unroll
                    for (int b = 0; b < BL; ++b) {
                        const int k = k0 + column((BL * wk + b) * 32 + lr);
                        if (k < p.k) dw[(size_t)n * p.lddw + k] = acc[a][b][q];
                    }
                }
            }
    }
    if (do_bias) {                                           // the row groups' sums, in order
        f32x4* sums = reinterpret_cast<f32x4*>(lds_all);
        __syncthreads();
        sums[threadIdx.x] = f32x4{bs[0], bs[1], bs[2], bs[3]};       // (oct * G + l)
        __syncthreads();
        if (grp == 0 && tid < G) {
            f32x4 part[4] = {sums[tid], sums[G + tid], sums[2 * G + tid], sums[3 * G + tid]};
            for (int o = 4; o < 512 / G; o += 4)
#pragma unroll
                for (int u = 0; u < 4; ++u) part[u] += sums[(o + u) * G + tid];
            const f32x4 s = (part[0] + part[1]) + (part[2] + part[3]);
            float* db = p.db + (p.splits > 1 ? ((size_t)split * tk + kt) * p.n : 0);
#pragma unroll
            for (int c = 0; c < 4; ++c)
                if (n0 + 4 * tid + c < p.n) db[n0 + 4 * tid + c] = s[c];
        }
    }
}

// out = the sum of the splits' partials: first dW's n k, then db's n, V consecutive values a lane.  G groups of 512 / G lanes take every
// G-th split on four chains, their sums are added in order through LDS (no float atomics: the same bits every time).  Four values a
// lane and few groups for large results (4096 x 512 x 512, 4 splits, whole call in bfloat16: 15.3 us, with one value and 16 groups 19.5), one value and
// up to 16 groups for small ones, where lanes are what is short (65536 x 64 x 64, 256 splits: 10.4 us, with four 11.4).
template <int V, int G>
__global__ void __launch_bounds__(512)
rows8_wgrad_reduce_kernel(int n, int k, int splits_w, int splits_b, const float* __restrict__ part_w, const float* __restrict__ part_b,
                          float* __restrict__ dw, long long lddw, float* __restrict__ db) {
    __shared__ float red[512][V];
    constexpr int lanes = 512 / G;
    const int lane = threadIdx.x & (lanes - 1), grp = threadIdx.x / lanes;
    const long long nk = (long long)n * k, items = (nk + V - 1) / V, item = (long long)blockIdx.x * lanes + lane;
    const bool w = item < items;
    const long long i = V * (w ? item : item - items), len = w ? nk : n;
    const int left = (w || db) && i < len ? (int)min((long long)V, len - i) : 0, splits = w ? splits_w : splits_b;
    const float* src = (w ? part_w : part_b) + i;
    float s[4][V];
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int e = 0; e < V; ++e) s[u][e] = 0.f;
    auto add = [&](float (&to)[V], int t) {
        float v[V];
        __builtin_memcpy(v, src + (size_t)t * len, sizeof(v));
#pragma unroll
        for (int e = 0; e < V; ++e) to[e] += v[e];
    };
    if (left == V) {
        int t = grp;
        for (; t + 3 * G < splits; t += 4 * G)
#pragma unroll
            for (int u = 0; u < 4; ++u) add(s[u], t + u * G);
        for (; t < splits; t += G) add(s[0], t);
    } else if (left > 0) {
        for (int t = grp; t < splits; t += G)
#pragma unroll
            for (int e = 0; e < V; ++e) s[0][e] += e < left ? src[(size_t)t * len + e] : 0.f;
    }
#pragma unroll
    for (int e = 0; e < V; ++e) s[0][e] = (s[0][e] + s[1][e]) + (s[2][e] + s[3][e]);
    if constexpr (G > 1) {
#pragma unroll
        for (int e = 0; e < V; ++e) red[threadIdx.x][e] = s[0][e];
        __syncthreads();
        if (grp > 0) return;
#pragma unroll
        for (int g = 1; g < G; ++g)
#pragma unroll
            for (int e = 0; e < V; ++e) s[0][e] += red[g * lanes + lane][e];
    }
    long long r = w ? i / k : 0;
    int c = w ? (int)(i - r * k) : 0;
#pragma unroll
    for (int e = 0; e < V; ++e) {
        if (e < left) (w ? dw[r * lddw + c] : db[i + e]) = s[0][e];
        if (++c == k) { c = 0; ++r; }
    }
}

// The tile and the number of splits (up to one workgroup a CU) by the time they take: 1 us a step of a workgroup for every type (measured 1.05 in
// float32, 0.6 in bfloat16, at either tile: in bfloat16 the rule counts steps too dear and splits early), 3.6 us more for the larger tile's
// longer start and end, and for splits 2.5 us and 0.9 us a MB of partials, written and read again.  What that decides, both sides measured in float32: 1024 x 512 x 512, 64 x 64, 1 | 4 splits: 13.3 | 14.0 us;
// 2048 rows: 21.5 | 16.4; 4096 x 1024 x 1024, 64 x 64 and 1 split | 128 x 128 and 4: 41.5 | 42.5 (bfloat16 26.5 | 33.3), 8192 rows: 76 | 64; 16384 x
// 512 x 512, 64 x 64 and 4 | 128 x 128 and 16: 47.7 | 41.1; 65536 x 256 x 256, 16 | 64: 47.8 | 40.7.
struct Wgrad8Plan { int tile, splits; };
static Wgrad8Plan wgrad8_plan(int m, int n, int k) {
    Wgrad8Plan p{64, 1};
    float best = 0.f;
    for (int tile = 64; tile <= (n > 64 && k > 64 ? 128 : 64); tile *= 2) {
        const int steps = imax(1, divup(m, W8_SLAB / tile));
        const long long tiles = (long long)divup(n, tile) * divup(k, tile);
        const float start = tile == 64 ? 0.f : 3.6f, rounds = (float)((tiles + 255) / 256);
        for (long long s = imax(1, (int)(256 / tiles)); s > 0; s /= 2) {
            const int t = (int)(s > steps ? steps : s);
            const float us = start + rounds * (float)divup(steps, t) + (t > 1 ? 2.5f + 3.6e-6f * (float)t * (float)n * (float)k : 0.f);
            if (best == 0.f || us < best) { best = us; p = {tile, t}; }
        }
    }
    return p;
}

}  // namespace jm

using namespace jm;

extern "C" {

int jm_rows8_pack(int m, int c, int type, const void* x, long long ldx, unsigned char* codes, int ldc, unsigned char* exps, int lde,
                  jm_stream_t stream) {
    JM_REQUIRE(m >= 0 && m <= R8_MAX_ROWS && c > 0 && c <= R8_MAX_WIDTH && type >= JM_F32 && type <= JM_F16, "rows8_pack: m %d, c %d, type %d", m, c, type);
    JM_REQUIRE(ldc >= c && ldc % 16 == 0 && lde >= m && lde % 16 == 0 && ldx >= c, "rows8_pack: codes and scales in multiples of 16 bytes (ldc %d, c %d, lde %d, m %d, ldx %lld)", ldc,
               c, lde, m, ldx);
    if (m == 0) return JM_OK;
    JM_REQUIRE(x && codes && exps && (((uintptr_t)codes | (uintptr_t)exps) & 15) == 0, "rows8_pack: NULL or unaligned buffers");
    const int groups = divup(c, R8_BLOCK) * 4;
    const dim3 grid((unsigned)grid_for((long long)m * groups, 256, R8_GRID)), block(256);
    hipStream_t s = (hipStream_t)stream;
    if (type == JM_F32) hipLaunchKernelGGL((rows8_pack_kernel<JM_F32>), grid, block, 0, s, m, lde, c, groups, (const float*)x, ldx, codes, ldc, exps);
    else if (type == JM_BF16) hipLaunchKernelGGL((rows8_pack_kernel<JM_BF16>), grid, block, 0, s, m, lde, c, groups, (const __bf16*)x, ldx, codes, ldc, exps);
    else hipLaunchKernelGGL((rows8_pack_kernel<JM_F16>), grid, block, 0, s, m, lde, c, groups, (const _Float16*)x, ldx, codes, ldc, exps);
    return check_launch("rows8_pack");
}

int jm_rows8_restore(int m, int c, int type, const unsigned char* codes, int ldc, const unsigned char* exps, int lde, void* out, long long ldo,
                     jm_stream_t stream) {
    JM_REQUIRE(m >= 0 && m <= R8_MAX_ROWS && c > 0 && c <= R8_MAX_WIDTH && type >= JM_F32 && type <= JM_F16, "rows8_restore: m %d, c %d, type %d", m, c, type);
    JM_REQUIRE(ldc >= c && ldc % 16 == 0 && lde >= m && lde % 16 == 0 && ldo >= c, "rows8_restore: codes and scales in multiples of 16 bytes (ldc %d, c %d, lde %d, m %d, ldo %lld)",
               ldc, c, lde, m, ldo);
    if (m == 0) return JM_OK;
    JM_REQUIRE(codes && exps && out && (((uintptr_t)codes | (uintptr_t)exps) & 15) == 0, "rows8_restore: NULL or unaligned buffers");
    const int groups = divup(c, 8);
    const dim3 grid((unsigned)grid_for((long long)m * groups, 256, R8_GRID)), block(256);
    hipStream_t s = (hipStream_t)stream;
    if (type == JM_F32) hipLaunchKernelGGL((rows8_restore_kernel<JM_F32>), grid, block, 0, s, m, lde, c, groups, codes, ldc, exps, (float*)out, ldo);
    else if (type == JM_BF16) hipLaunchKernelGGL((rows8_restore_kernel<JM_BF16>), grid, block, 0, s, m, lde, c, groups, codes, ldc, exps, (__bf16*)out, ldo);
    else hipLaunchKernelGGL((rows8_restore_kernel<JM_F16>), grid, block, 0, s, m, lde, c, groups, codes, ldc, exps, (_Float16*)out, ldo);
    return check_launch("rows8_restore");
}

int jm_rows8_relu_mask(int m, int c, const float* dy, long long ldd, const unsigned char* codes, int ldc, float* out, long long ldo,
                       jm_stream_t stream) {
    JM_REQUIRE(m >= 0 && m <= R8_MAX_ROWS && c > 0 && c <= R8_MAX_WIDTH && ldd >= c && ldo >= c && ldc >= c && ldc % 16 == 0,
               "rows8_relu_mask: m %d, c %d, ldd %lld, ldc %d, ldo %lld", m, c, ldd, ldc, ldo);
    JM_REQUIRE(m <= 1 || !dy || dy != out || ldd == ldo, "rows8_relu_mask: in place with rows %lld and %lld apart", ldd, ldo);
    if (m == 0) return JM_OK;
    JM_REQUIRE(dy && codes && out && ((uintptr_t)codes & 15) == 0, "rows8_relu_mask: NULL or unaligned buffers");
    const int groups = divup(c, 4);
    hipLaunchKernelGGL(rows8_relu_mask_kernel, dim3((unsigned)grid_for((long long)m * groups, 256, R8_GRID)), dim3(256), 0, (hipStream_t)stream, m, c, groups, dy, ldd,
                       codes, ldc, out, ldo);
    return check_launch("rows8_relu_mask");
}

size_t jm_rows8_wgrad_workspace_bytes(int m, int n, int k) {
    if (m <= 0 || m > R8_MAX_ROWS || n <= 0 || n > R8_MAX_WIDTH || k <= 0 || k > R8_MAX_WIDTH) return 0;
    const Wgrad8Plan p = wgrad8_plan(m, n, k);               // per split dW, then per split and tile column the bias sums
    return p.splits > 1 ? (size_t)p.splits * ((size_t)n * (size_t)k + (size_t)divup(k, p.tile) * n) * sizeof(float) : 0;
}

int jm_rows8_linear_wgrad(int m, int n, int k, int type, const void* dy, long long lddy, const unsigned char* codes, int ldc, const unsigned char* exps,
                          int lde, float* dw, long long lddw, float* dbias, void* ws, size_t ws_bytes, jm_stream_t stream) {
    JM_REQUIRE(m >= 0 && m <= R8_MAX_ROWS && n > 0 && n <= R8_MAX_WIDTH && k > 0 && k <= R8_MAX_WIDTH && type >= JM_F32 && type <= JM_F16 && dw, "rows8_linear_wgrad: m %d, n %d, k %d, type %d", m, n, k, type);
    JM_REQUIRE(lddy >= n && lddy <= R8_MAX_LD && ldc >= k && ldc <= R8_MAX_LD && ldc % 16 == 0 && lde >= m && lde % 16 == 0 && lddw >= k,
               "rows8_linear_wgrad: lddy %lld, ldc %d, lde %d, lddw %lld for m %d, n %d, k %d", lddy, ldc, lde, lddw, m, n, k);
    JM_REQUIRE(m == 0 || (dy && codes && exps && (((uintptr_t)codes | (uintptr_t)exps) & 15) == 0), "rows8_linear_wgrad: NULL or unaligned buffers");
    const Wgrad8Plan plan = wgrad8_plan(m, n, k);
    const int splits = plan.splits, step = W8_SLAB / plan.tile;
    if (splits > 1 && (!ws || ws_bytes < jm_rows8_wgrad_workspace_bytes(m, n, k))) {
        set_error("rows8_linear_wgrad: workspace of %zu bytes, need %zu", ws_bytes, jm_rows8_wgrad_workspace_bytes(m, n, k));
        return JM_EWORKSPACE;
    }
    hipStream_t s = (hipStream_t)stream;
    Wgrad8 p{};
    p.m = m; p.n = n; p.k = k; p.splits = splits; p.rows_per = m > 0 ? ((m - 1) / splits / step + 1) * step : step;
    p.dy = dy; p.lddy = lddy; p.codes = codes; p.ldc = ldc; p.exps = exps; p.lde = lde; p.blocks = divup(k, R8_BLOCK);
    float* part_b = (float*)ws + (size_t)splits * n * k;
    if (splits > 1) { p.dw = (float*)ws; p.lddw = k; p.db = dbias ? part_b : nullptr; }
    else { p.dw = dw; p.lddw = lddw; p.db = dbias; }
    const long long wgs = ((long long)divup(n, plan.tile) * divup(k, plan.tile) * splits + 7) / 8 * 8;
    JM_REQUIRE(wgs <= 0x7fffffffll, "rows8_linear_wgrad: n %d, k %d", n, k);
    const dim3 grid((unsigned)wgs), block(512);
    const unsigned lds = 2u * (type == JM_F32 ? 4u : (type == JM_F16 ? 3u : 2u)) * W8_SLAB * 2u;
    auto run = [&](auto kernel) {
        (void)hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        hipLaunchKernelGGL(kernel, grid, block, lds, s, p);
    };
    auto tile = [&](auto type_, auto small_) {
        constexpr int TY = decltype(type_)::value;
        constexpr bool S = decltype(small_)::value;
        if (plan.tile == 64) run(rows8_wgrad_kernel<TY, S, 64>);
        else if constexpr (!S || TY != JM_F32) run(rows8_wgrad_kernel<TY, S, 128>);        // (n < 4 has small tiles)
    };
    const bool small = n < 4 || (type != JM_F32 && (((uintptr_t)dy & 3) || (lddy & 1)));
    auto pick = [&](auto type_) { small ? tile(type_, std::true_type{}) : tile(type_, std::false_type{}); };
    if (type == JM_F32) pick(std::integral_constant<int, JM_F32>{});
    else if (type == JM_BF16) pick(std::integral_constant<int, JM_BF16>{});
    else pick(std::integral_constant<int, JM_F16>{});
    if (splits > 1) {
        auto reduce = [&](auto v_, auto g_) {
            constexpr int V = decltype(v_)::value, G = decltype(g_)::value;
            const long long items = ((long long)n * k + V - 1) / V + (dbias ? divup(n, V) : 0);
            hipLaunchKernelGGL((rows8_wgrad_reduce_kernel<V, G>), dim3((unsigned)((items + 512 / G - 1) / (512 / G))), dim3(512), 0, s, n, k, splits,
                               splits * divup(k, plan.tile), (const float*)ws, (const float*)part_b, dw, lddw, dbias);
        };
        if ((long long)n * k < (1 << 17)) reduce(std::integral_constant<int, 1>{}, std::integral_constant<int, 16>{});
        else if (splits > 4) reduce(std::integral_constant<int, 4>{}, std::integral_constant<int, 4>{});
        else reduce(std::integral_constant<int, 4>{}, std::integral_constant<int, 1>{});
    }
    return check_launch("rows8_linear_wgrad");
}

}  // extern "C"
