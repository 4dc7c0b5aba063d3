// rows8.hip — activations kept in 8 bits between the forward and the backward pass of the row layers (rows_gemm.hip), and their use in
// the backward pass.
//
// Format.  A row tensor X (m, c) is kept as e4m3 codes (m, ldc) plus one scale byte per 32 consecutive channels of a row:
//     amax  = the largest finite |x| of the block;  2^e = the smallest power of two with amax <= 448 2^e, e >= -100 (empty block: -100)
//     code  = x / 2^e rounded to the nearest e4m3 value, ties to even;  scale byte = e + 127
// with two exceptions: a value that is not zero never becomes zero (it takes the smallest code of its sign, 2^-9 2^e, so that the sign
// pattern — a ReLU's mask — survives), and a value that is not finite becomes the NaN code (e4m3 has no infinity).
// Why e4m3 with power-of-two scales: the division is exact, so the codes are a defined rounding of the input (half a step, 2^-4
// relative, within 2^14 of the block's maximum) whatever computes them; and a kept value, 4 significant bits times a power of two, is
// exact in bfloat16, so the backward's products run on the bf16 matrix pipe without another rounding of X.
// 1.03 bytes per element instead of 4 (float32) or 2.
#include "jm_elem.h"
#include "jm_rows.h"
#include <type_traits>

namespace jm {

constexpr int R8_BLOCK = 32;         // channels per scale
constexpr int R8_MAX_ROWS = 1 << 30;        // (row counters of the weight gradient are 32 bits wide)
constexpr int R8_EMIN = -100;        // least scale exponent: 2^e and the smallest code 2^(e - 9) stay normal in float32 and bfloat16

__device__ __forceinline__ float exp2i(int e) { return __uint_as_float((unsigned)(e + 127) << 23); }      // -126 <= e <= 127
__device__ __forceinline__ bool finite_bits(unsigned b) { return (b & 0x7f800000u) != 0x7f800000u; }

// the scale exponent of a block from the bits of its largest finite |x|
__device__ __forceinline__ int r8_exponent(unsigned amax_bits) {
    const int e = (int)(amax_bits >> 23) - 127 - 8 + ((amax_bits & 0x7fffffu) > 0x600000u ? 1 : 0);      // 448 = 1.75 x 2^8
    return max(e, R8_EMIN);
}

// Four lanes hold a block, 8 channels each; the block's maximum by two quad permutations.  One read of X, one write of the codes: bound
// by memory.  Threads walk (row, 8 channels) in memory order.
template <int TY>
__global__ void __launch_bounds__(256)
rows8_pack_kernel(long long items, int c, int groups, const typename Elem<TY>::T* __restrict__ x, long long ldx, unsigned char* __restrict__ codes,
                  int ldc, unsigned char* __restrict__ exps) {
    typedef typename Elem<TY>::V8 V8;
    for (long long it = blockIdx.x * 256ll + threadIdx.x; it < items; it += gridDim.x * 256ll) {
        long long row;
        int grp;
        if (items <= 0x7fffffffll) {
            row = (unsigned)it / (unsigned)groups;
            grp = (int)((unsigned)it - (unsigned)row * (unsigned)groups);
        } else {
            row = it / groups;
            grp = (int)(it - row * groups);
        }
        const V8 raw = load8_upto<V8>(x + row * ldx + grp * 8, c - grp * 8);
        float v[8];
        unsigned top = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            v[e] = (float)raw[e];
            const unsigned b = __float_as_uint(v[e]) & 0x7fffffffu;
            top = max(top, finite_bits(b) ? b : 0u);
        }
        top = max(top, (unsigned)__builtin_amdgcn_update_dpp(0, (int)top, JM_DPP_XOR1, 0xf, 0xf, true));
        top = max(top, (unsigned)__builtin_amdgcn_update_dpp(0, (int)top, JM_DPP_XOR2, 0xf, 0xf, true));
        const int e2 = r8_exponent(top);
        const float inv = exp2i(-e2);
        unsigned w[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            int p = 0;
            // (values that are not finite are converted as zero and replaced below)
            float f[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) f[q] = finite_bits(__float_as_uint(v[4 * h + q])) ? v[4 * h + q] * inv : 0.f;
            p = __builtin_amdgcn_cvt_pk_fp8_f32(f[0], f[1], p, false);
            p = __builtin_amdgcn_cvt_pk_fp8_f32(f[2], f[3], p, true);
            unsigned u = (unsigned)p;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const unsigned b = __float_as_uint(v[4 * h + q]);
                const unsigned code = (u >> (8 * q)) & 0xffu;
                unsigned fixed = code;
                if ((code & 0x7fu) == 0u && (b & 0x7fffffffu) != 0u) fixed = (b >> 31) ? 0x81u : 0x01u;
                if (!finite_bits(b)) fixed = 0x7fu;
                u = (u & ~(0xffu << (8 * q))) | (fixed << (8 * q));
            }
            w[h] = u;
        }
        if (grp * 8 < ldc) *reinterpret_cast<uint2*>(codes + row * ldc + grp * 8) = make_uint2(w[0], w[1]);
        if ((grp & 3) == 0) exps[row * (groups >> 2) + (grp >> 2)] = (unsigned char)(e2 + 127);
    }
}

__device__ __forceinline__ void r8_decode4(unsigned w, float scale, float (&v)[4]) {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false);
    const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    v[0] = lo[0] * scale; v[1] = lo[1] * scale; v[2] = hi[0] * scale; v[3] = hi[1] * scale;
}

template <int TY>
__global__ void __launch_bounds__(256)
rows8_restore_kernel(long long items, int c, int groups, const unsigned char* __restrict__ codes, int ldc, const unsigned char* __restrict__ exps,
                     typename Elem<TY>::T* __restrict__ out, long long ldo) {
    typedef typename Elem<TY>::T T;
    typedef typename Elem<TY>::V8 V8;
    const int blocks = (c + R8_BLOCK - 1) / R8_BLOCK;
    for (long long it = blockIdx.x * 256ll + threadIdx.x; it < items; it += gridDim.x * 256ll) {
        long long row;
        int grp;
        if (items <= 0x7fffffffll) {
            row = (unsigned)it / (unsigned)groups;
            grp = (int)((unsigned)it - (unsigned)row * (unsigned)groups);
        } else {
            row = it / groups;
            grp = (int)(it - row * groups);
        }
        const uint2 w = *reinterpret_cast<const uint2*>(codes + row * ldc + grp * 8);
        const float scale = exp2i((int)exps[row * blocks + (grp >> 2)] - 127);
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

// out = (the kept value > 0) ? dy : 0 — the gradient through a ReLU whose output was kept.  out may be dy.
__global__ void __launch_bounds__(256)
rows8_relu_mask_kernel(long long items, int c, int groups, const float* dy, int ldd, const unsigned char* __restrict__ codes, int ldc, float* out, int ldo) {
    for (long long it = blockIdx.x * 256ll + threadIdx.x; it < items; it += gridDim.x * 256ll) {
        const long long row = it / groups;
        const int c0 = (int)(it - row * groups) * 4;
        const unsigned w = *reinterpret_cast<const unsigned*>(codes + row * ldc + c0);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const unsigned b = (w >> (8 * q)) & 0xffu;
            if (c0 + q < c) out[row * ldo + c0 + q] = (b != 0u && b < 0x7fu) ? dy[row * ldd + c0 + q] : 0.f;
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
// Workgroup = a 128 x 128 tile of dW over one split of the rows, 64 rows at a time.  A thread fetches 8 rows x 4 columns of both
// operands (the next 64 rows' while this one's are multiplied), cuts and converts them, and stores 8 rows of one column as 16 bytes: the
// contraction index becomes the fast one on the way into LDS, and a matrix operand (8 rows of a column) is one 16-byte read.  In LDS column
// 4 i + q of a tile sits in slot 32 q + i: writes and reads of a wave are contiguous.  Four waves of 64 x 64 (2 x 2 products of
// 32 x 32 x 16), two workgroups a CU: one stores while the other multiplies.
// The splits' partial tiles are added in split order by the second kernel (no float atomics: the same bits every time).
constexpr int W8_SLAB = 8192;          // elements of one operand piece of a step: 64 rows x 128 columns or 128 x 64

struct Wgrad8 {
    int m, n, k, splits, rows_per;       // rows_per: rows of a split, a multiple of a step's
    const void* dy; long long lddy;
    const unsigned char* codes; int ldc; const unsigned char* exps; int blocks;
    float *dw, *db;                      // (splits, n, k) and (splits, n) partials, or the results when splits == 1
    long long lddw;
};

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

// four consecutive columns of a row.  The columns of a group that lies outside the matrix are whatever lies inside (they only reach
// outputs that are never stored); a group that straddles the edge (`ragged`, widths that are no multiple of 4) is read from width - 4 and shifted
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
    unsigned long long v;
    __device__ __forceinline__ void load(const typename Elem<TY>::T* p) { __builtin_memcpy(&v, p, 8); }
    __device__ __forceinline__ void shift(int n) { v >>= 16 * n; }
    __device__ __forceinline__ void zero() { v = 0; }
    __device__ __forceinline__ unsigned bits(int q) const { return (unsigned)(v >> (16 * q)) & 0xffffu; }
    __device__ __forceinline__ float get(int q) const {
        const unsigned short h = (unsigned short)bits(q);
        typename Elem<TY>::T t;
        __builtin_memcpy(&t, &h, 2);
        return (float)t;
    }
};
template <> struct Quad<JM_BF16> : Quad16<JM_BF16> {};
template <> struct Quad<JM_F16> : Quad16<JM_F16> {};

// the upper halves of two words as one: (hi half of a) | (hi half of b) << 16
__device__ __forceinline__ unsigned pack_hi(unsigned a, unsigned b) { return __builtin_amdgcn_perm(b, a, 0x07060302u); }

template <int TY, bool SMALL, int W8_T>
__global__ void __launch_bounds__(256, 2)
rows8_wgrad_kernel(Wgrad8 p) {
    typedef typename Elem<TY>::T T;
    constexpr int W8_R = W8_SLAB / W8_T, G = W8_T / 4, BL = W8_T / 64;          // rows of a step; column groups; 32-wide blocks of a wave a side
    constexpr int P = TY == JM_F32 ? 3 : (TY == JM_F16 ? 2 : 1);                  // pieces of a gradient
    typedef __bf16 frag_t __attribute__((ext_vector_type(8)));
    typedef float f32x16 __attribute__((ext_vector_type(16)));
    __shared__ __attribute__((aligned(16))) unsigned short lds[(P + 1) * W8_SLAB];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    // workgroups are dealt to the 8 XCDs in turn: the tiles of one split, which read the same rows, stay on one of them
    const int tk = (p.k + W8_T - 1) / W8_T, tiles = ((p.n + W8_T - 1) / W8_T) * tk;
    const int xcd = blockIdx.x & 7, local = blockIdx.x >> 3;
    const int split = (local / tiles) * 8 + xcd, tile = local % tiles;
    if (split >= p.splits) return;
    const int n0 = (tile / tk) * W8_T, k0 = (tile % tk) * W8_T;
    const int r_begin = min((long long)split * p.rows_per, (long long)p.m), r_end = min(p.m, r_begin + p.rows_per);

    // fetch: rows 8 oct .. + 7 of the 64, columns 4 l .. + 3 of both tiles
    const int l = tid % G, oct = tid / G;
    const int cy = n0 + 4 * l, cx = min(k0 + 4 * l, p.ldc - 4);
    const int ylast = p.n - 4;
    const int ysh = (!SMALL && cy < p.n) ? max(0, cy - ylast) : 0;
    const bool ragged = !SMALL && (p.n & 3) != 0 && n0 + W8_T > p.n;
    const T* dyp = (const T*)p.dy + (SMALL ? 0 : min(cy, ylast));
    const unsigned char* xp = p.codes + cx;
    const unsigned char* ep = p.exps + min(cx / R8_BLOCK, p.blocks - 1);
    struct Rows {
        Quad<TY> y[8];
        unsigned x[8], e[8];
    };
    Rows rows[2];
    // the last octet of the matrix is read from row m - 8 on: rows before its own first one count as zeros (stage)
    auto first_row = [&](int r) { return SMALL ? r + 8 * oct : min(r + 8 * oct, p.m - 8); };
    auto fetch = [&](Rows& d, int r) __attribute__((always_inline)) {
        const int at = first_row(r);
        const T* py = dyp + (long long)at * p.lddy;
        const unsigned char* px = xp + (long long)at * p.ldc;
        const unsigned char* pe = ep + (long long)at * p.blocks;
#pragma unroll
        for (int q = 0; q < 8; ++q) {
            if constexpr (SMALL) {                           // fewer than 8 rows or 4 columns: element by element
                const long long row = min(at + q, p.m - 1);
                T t[4];
#pragma unroll
                for (int c = 0; c < 4; ++c) t[c] = dyp[row * p.lddy + min(cy + c, p.n - 1)];
                d.y[q].load(t);
                d.x[q] = *reinterpret_cast<const unsigned*>(xp + row * p.ldc);
                d.e[q] = ep[row * p.blocks];
            } else {
                d.y[q].load(py + q * p.lddy);
                d.x[q] = *reinterpret_cast<const unsigned*>(px + q * (long long)p.ldc);
                d.e[q] = pe[q * (long long)p.blocks];
            }
        }
    };
    float bs[4] = {0.f, 0.f, 0.f, 0.f};
    const bool do_bias = p.db != nullptr && k0 == 0;
    auto stage = [&](Rows& d, int r) __attribute__((always_inline)) {
        Quad<TY>(&y)[8] = d.y;
        unsigned(&x)[8] = d.x;
        unsigned(&e)[8] = d.e;
        if (r + W8_R > r_end) {                              // rows outside this step's own count as zeros on both sides
            const int at = first_row(r);
#pragma unroll
            for (int q = 0; q < 8; ++q)
                if (at + q >= r_end || at + q < r + 8 * oct) { y[q].zero(); x[q] = 0u; e[q] = 127u; }
        }
        if (ragged) {
#pragma unroll
            for (int q = 0; q < 8; ++q) y[q].shift(ysh);
        }
        if (do_bias) {
#pragma unroll
            for (int q = 0; q < 8; ++q)
#pragma unroll
                for (int c = 0; c < 4; ++c) bs[c] += y[q].get(c);
        }
        // an infinity leaves no rest (inf - inf would be NaN), a NaN leaves a NaN: looked for once for the whole wave
        bool inf_seen = false;
        if constexpr (P > 1) {
            float z = 0.f;
#pragma unroll
            for (int q = 0; q < 8; ++q)
#pragma unroll
                for (int c = 0; c < 4; ++c) z = __builtin_fmaf(y[q].get(c), 0.f, z);
            inf_seen = __ballot(z != z) != 0ull;
        }
        u32x4* Y = reinterpret_cast<u32x4*>(lds) + oct * W8_T + l;          // 16 bytes = 8 rows of a slot
        auto cut = [&](auto special_) __attribute__((always_inline)) {
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                u32x4 w[P];
#pragma unroll
                for (int h = 0; h < 4; ++h) {
                    if constexpr (TY == JM_BF16) {
                        w[0][h] = y[2 * h].bits(c) | (y[2 * h + 1].bits(c) << 16);
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
        };
        if (P > 1 && inf_seen) cut(std::true_type{});
        else cut(std::false_type{});
        // kept values: codes of a row share a scale within the four columns
        unsigned v0[8], v1[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) {
            const float sc = __uint_as_float(e[q] << 23);
            const auto lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)x[q], sc, false);
            const auto hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)x[q], sc, true);
            __builtin_memcpy(&v0[q], &lo, 4);
            __builtin_memcpy(&v1[q], &hi, 4);
        }
        u32x4* X = reinterpret_cast<u32x4*>(lds + P * W8_SLAB) + oct * W8_T + l;
        u32x4 w0, w1, w2, w3;
#pragma unroll
        for (int h = 0; h < 4; ++h) {
            w0[h] = __builtin_amdgcn_perm(v0[2 * h + 1], v0[2 * h], 0x05040100u);
            w1[h] = pack_hi(v0[2 * h], v0[2 * h + 1]);
            w2[h] = __builtin_amdgcn_perm(v1[2 * h + 1], v1[2 * h], 0x05040100u);
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
    auto step = [&](Rows& d, int r) __attribute__((always_inline)) {
        stage(d, r);
        __syncthreads();
        if (r + 2 * W8_R < r_end) fetch(d, r + 2 * W8_R);    // two steps ahead
        const u32x4* Y = reinterpret_cast<const u32x4*>(lds);
        const u32x4* X = reinterpret_cast<const u32x4*>(lds + P * W8_SLAB);
#pragma unroll
        for (int s = 0; s < W8_R / 16; ++s) {
            const int at = (2 * s + lk) * W8_T + lr;
            frag_t xb[BL], ya[P][BL];
#pragma unroll
            for (int b = 0; b < BL; ++b) xb[b] = __builtin_bit_cast(frag_t, X[at + (BL * wk + b) * 32]);
#pragma unroll
            for (int c = 0; c < P; ++c)
#pragma unroll
                for (int a = 0; a < BL; ++a) ya[c][a] = __builtin_bit_cast(frag_t, Y[c * (W8_SLAB / 8) + at + (BL * wn + a) * 32]);
#pragma unroll
            for (int c = P - 1; c >= 0; --c)
#pragma unroll
                for (int a = 0; a < BL; ++a)
#pragma unroll
                    for (int b = 0; b < BL; ++b) acc[a][b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ya[c][a], xb[b], acc[a][b], 0, 0, 0);
        }
        __syncthreads();
    };
    if (r_begin < r_end) fetch(rows[0], r_begin);
    if (r_begin + W8_R < r_end) fetch(rows[1], r_begin + W8_R);
    for (int r = r_begin; r < r_end; r += 2 * W8_R) {
        step(rows[0], r);
        if (r + W8_R < r_end) step(rows[1], r + W8_R);
    }

    float* dw = p.dw + (p.splits > 1 ? (size_t)split * p.n * p.k : 0);
    auto column = [&](int slot) { return 4 * (slot % G) + slot / G; };
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
    if (do_bias) {                                           // the row groups' sums, in order
        f32x4* red = reinterpret_cast<f32x4*>(lds);
        red[oct * G + l] = f32x4{bs[0], bs[1], bs[2], bs[3]};
        __syncthreads();
        if (tid < G) {
            f32x4 s = red[tid];
            for (int o = 1; o < 256 / G; ++o) s += red[o * G + tid];
            float* db = p.db + (p.splits > 1 ? (size_t)split * p.n : 0);
#pragma unroll
            for (int c = 0; c < 4; ++c)
                if (n0 + 4 * tid + c < p.n) db[n0 + 4 * tid + c] = s[c];
        }
    }
}

// out = the sum of the splits' partials: items 0 .. n k - 1 are dW, then n of db.  A workgroup takes 32 items (a cache line of every
// partial); its 16 groups of 32 lanes sum every 16th split on four chains, the groups are added in order through LDS.
__global__ void __launch_bounds__(512)
rows8_wgrad_reduce_kernel(int n, int k, int splits, const float* __restrict__ part_w, const float* __restrict__ part_b, float* __restrict__ dw,
                          long long lddw, float* __restrict__ db) {
    __shared__ float red[16][32];
    const long long nk = (long long)n * k;
    const int lane = threadIdx.x & 31, grp = threadIdx.x >> 5;
    const long long i = blockIdx.x * 32ll + lane;
    const bool w = i < nk, ok = i < nk + (db ? n : 0);
    const float* src = w ? part_w + i : part_b + (ok ? i - nk : 0);
    const size_t step = w ? (size_t)nk : (size_t)n;
    float s0 = 0.f, s1 = 0.f, s2 = 0.f, s3 = 0.f;
    if (ok) {
        int t = grp;
        for (; t + 48 < splits; t += 64) {
            s0 += src[(size_t)t * step];        s1 += src[(size_t)(t + 16) * step];
            s2 += src[(size_t)(t + 32) * step]; s3 += src[(size_t)(t + 48) * step];
        }
        for (; t < splits; t += 16) s0 += src[(size_t)t * step];
    }
    red[grp][lane] = (s0 + s1) + (s2 + s3);
    __syncthreads();
    if (grp > 0 || !ok) return;
    float s = red[0][lane];
#pragma unroll
    for (int g = 1; g < 16; ++g) s += red[g][lane];
    if (w) dw[(i / k) * lddw + i % k] = s;
    else db[i - nk] = s;
}

// Tiles of 128 x 128 halve what is read from the L2 and feed the matrix pipe best, but there have to be enough of them: with at least 4096
// (tile, 64 rows) steps and both sides wider than 64 (65536 x 256 x 256: 47 us against 52; 16384 x 1024 x 1024: 144 against 338); 64 x 64
// otherwise (65536 x 64 x 64: 13 us against 18; 4096 x 512 x 512: 26 against 33).  Splits: up to two workgroups a CU; what a split saves
// in steps (about 1.5 us each where the CU has nothing else to do) is weighed against the partials it writes and the second kernel reads.
struct Wgrad8Plan { int tile, splits; };
static Wgrad8Plan wgrad8_plan(int m, int n, int k) {
    Wgrad8Plan p;
    const bool wide = n > 64 && k > 64 && (long long)divup(n, 128) * divup(k, 128) * (m / 64) >= 4096;
    p.tile = wide ? 128 : 64;
    const int steps = imax(1, m / (W8_SLAB / p.tile));
    const long long tiles = (long long)divup(n, p.tile) * divup(k, p.tile);
    p.splits = 1;
    float best = 1.5f * (float)steps;
    for (long long s = 512 / tiles; s > 1; s /= 2) {
        const int t = (int)(s > 256 ? 256 : (s > steps ? steps : s));
        const float us = 1.5f * (float)divup(steps, t) + 3.f + 2.f * (float)t * (float)n * (float)k * 1e-6f;
        if (t > 1 && us < best) { best = us; p.splits = t; }
    }
    return p;
}

}  // namespace jm

using namespace jm;

extern "C" {

int jm_rows8_pack(int m, int c, int type, const void* x, long long ldx, unsigned char* codes, int ldc, unsigned char* exps, jm_stream_t stream) {
    JM_REQUIRE(m >= 0 && c > 0 && type >= JM_F32 && type <= JM_F16, "rows8_pack: m %d, c %d, type %d", m, c, type);
    JM_REQUIRE(ldc >= c && ldc % 16 == 0 && ldx >= c, "rows8_pack: codes in rows of a multiple of 16 bytes (ldc %d, c %d, ldx %lld)", ldc, c, ldx);
    if (m == 0) return JM_OK;
    JM_REQUIRE(x && codes && exps && ((uintptr_t)codes & 15) == 0, "rows8_pack: NULL or unaligned buffers");
    const int groups = divup(c, R8_BLOCK) * 4;
    const long long items = (long long)m * groups;
    const dim3 grid((unsigned)grid_for(items, 256, JM_EGRID)), block(256);
    hipStream_t s = (hipStream_t)stream;
    if (type == JM_F32) hipLaunchKernelGGL((rows8_pack_kernel<JM_F32>), grid, block, 0, s, items, c, groups, (const float*)x, ldx, codes, ldc, exps);
    else if (type == JM_BF16) hipLaunchKernelGGL((rows8_pack_kernel<JM_BF16>), grid, block, 0, s, items, c, groups, (const __bf16*)x, ldx, codes, ldc, exps);
    else hipLaunchKernelGGL((rows8_pack_kernel<JM_F16>), grid, block, 0, s, items, c, groups, (const _Float16*)x, ldx, codes, ldc, exps);
    return check_launch("rows8_pack");
}

int jm_rows8_restore(int m, int c, int type, const unsigned char* codes, int ldc, const unsigned char* exps, void* out, long long ldo, jm_stream_t stream) {
    JM_REQUIRE(m >= 0 && c > 0 && type >= JM_F32 && type <= JM_F16, "rows8_restore: m %d, c %d, type %d", m, c, type);
    JM_REQUIRE(ldc >= c && ldc % 16 == 0 && ldo >= c, "rows8_restore: codes in rows of a multiple of 16 bytes (ldc %d, c %d, ldo %lld)", ldc, c, ldo);
    if (m == 0) return JM_OK;
    JM_REQUIRE(codes && exps && out && ((uintptr_t)codes & 15) == 0, "rows8_restore: NULL or unaligned buffers");
    const int groups = divup(c, 8);
    const long long items = (long long)m * groups;
    const dim3 grid((unsigned)grid_for(items, 256, JM_EGRID)), block(256);
    hipStream_t s = (hipStream_t)stream;
    if (type == JM_F32) hipLaunchKernelGGL((rows8_restore_kernel<JM_F32>), grid, block, 0, s, items, c, groups, codes, ldc, exps, (float*)out, ldo);
    else if (type == JM_BF16) hipLaunchKernelGGL((rows8_restore_kernel<JM_BF16>), grid, block, 0, s, items, c, groups, codes, ldc, exps, (__bf16*)out, ldo);
    else hipLaunchKernelGGL((rows8_restore_kernel<JM_F16>), grid, block, 0, s, items, c, groups, codes, ldc, exps, (_Float16*)out, ldo);
    return check_launch("rows8_restore");
}

int jm_rows8_relu_mask(int m, int c, const float* dy, int ldd, const unsigned char* codes, int ldc, float* out, int ldo, jm_stream_t stream) {
    JM_REQUIRE(m >= 0 && c > 0 && ldd >= c && ldo >= c && ldc >= c && ldc % 16 == 0, "rows8_relu_mask: m %d, c %d, ldd %d, ldc %d, ldo %d", m, c, ldd, ldc, ldo);
    if (m == 0) return JM_OK;
    JM_REQUIRE(dy && codes && out && ((uintptr_t)codes & 15) == 0, "rows8_relu_mask: NULL or unaligned buffers");
    const int groups = divup(c, 4);
    const long long items = (long long)m * groups;
    hipLaunchKernelGGL(rows8_relu_mask_kernel, dim3((unsigned)grid_for(items, 256, JM_EGRID)), dim3(256), 0, (hipStream_t)stream, items, c, groups, dy, ldd,
                       codes, ldc, out, ldo);
    return check_launch("rows8_relu_mask");
}

size_t jm_rows8_wgrad_workspace_bytes(int m, int n, int k) {
    if (m <= 0 || n <= 0 || k <= 0) return 0;
    const size_t s = (size_t)wgrad8_plan(m, n, k).splits;
    return s > 1 ? s * ((size_t)n * (size_t)k + (size_t)n) * sizeof(float) : 0;
}

int jm_rows8_linear_wgrad(int m, int n, int k, int type, const void* dy, long long lddy, const unsigned char* codes, int ldc, const unsigned char* exps,
                          float* dw, long long lddw, float* dbias, void* ws, size_t ws_bytes, jm_stream_t stream) {
    JM_REQUIRE(m >= 0 && m <= R8_MAX_ROWS && n > 0 && k > 0 && type >= JM_F32 && type <= JM_F16 && dw, "rows8_linear_wgrad: m %d, n %d, k %d, type %d", m, n, k, type);
    JM_REQUIRE(lddy >= n && ldc >= k && ldc % 16 == 0 && lddw >= k, "rows8_linear_wgrad: lddy %lld, ldc %d, lddw %lld for n %d, k %d", lddy, ldc, lddw, n, k);
    JM_REQUIRE(m == 0 || (dy && codes && exps && ((uintptr_t)codes & 15) == 0), "rows8_linear_wgrad: NULL or unaligned buffers");
    const Wgrad8Plan plan = wgrad8_plan(m, n, k);
    const int splits = plan.splits, step = W8_SLAB / plan.tile;
    if (splits > 1 && (!ws || ws_bytes < jm_rows8_wgrad_workspace_bytes(m, n, k))) {
        set_error("rows8_linear_wgrad: workspace of %zu bytes, need %zu", ws_bytes, jm_rows8_wgrad_workspace_bytes(m, n, k));
        return JM_EWORKSPACE;
    }
    hipStream_t s = (hipStream_t)stream;
    Wgrad8 p{};
    p.m = m; p.n = n; p.k = k; p.splits = splits; p.rows_per = m > 0 ? ((m - 1) / splits / step + 1) * step : step;
    p.dy = dy; p.lddy = lddy; p.codes = codes; p.ldc = ldc; p.exps = exps; p.blocks = divup(k, R8_BLOCK);
    float* part_b = (float*)ws + (size_t)splits * n * k;
    if (splits > 1) { p.dw = (float*)ws; p.lddw = k; p.db = dbias ? part_b : nullptr; }
    else { p.dw = dw; p.lddw = lddw; p.db = dbias; }
    const long long wgs = (long long)divup(n, plan.tile) * divup(k, plan.tile) * (divup(splits, 8) * 8);
    JM_REQUIRE(wgs <= 0x7fffffffll, "rows8_linear_wgrad: n %d, k %d", n, k);
    const dim3 grid((unsigned)wgs), block(256);
    auto run = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, block, 0, s, p); };
    auto pick = [&](auto small_, auto tile_) {
        constexpr bool S = decltype(small_)::value;
        constexpr int W = decltype(tile_)::value;
        run(type == JM_F32 ? rows8_wgrad_kernel<JM_F32, S, W> : (type == JM_BF16 ? rows8_wgrad_kernel<JM_BF16, S, W> : rows8_wgrad_kernel<JM_F16, S, W>));
    };
    if (m < 8 || n < 4) pick(std::true_type{}, std::integral_constant<int, 64>{});
    else if (plan.tile == 64) pick(std::false_type{}, std::integral_constant<int, 64>{});
    else pick(std::false_type{}, std::integral_constant<int, 128>{});
    if (splits > 1) {
        const long long items = (long long)n * k + (dbias ? n : 0);
        hipLaunchKernelGGL(rows8_wgrad_reduce_kernel, dim3((unsigned)((items + 31) / 32)), dim3(512), 0, s, n, k, splits, (const float*)ws,
                           (const float*)part_b, dw, lddw, dbias);
    }
    return check_launch("rows8_linear_wgrad");
}

}  // extern "C"
