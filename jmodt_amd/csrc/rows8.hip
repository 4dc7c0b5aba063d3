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

namespace jm {

constexpr int R8_BLOCK = 32;         // channels per scale
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
// dW (n, k) = dY (m, n)^T X (m, k), db (n) = column sums of dY.  Workgroup = a 64 x 64 tile of dW over one split of the rows, 32 rows of
// both operands at a time through LDS as float32, four waves of 16 x 64, 16 x 16 x 4 float32 products; the splits' partial tiles are
// added in split order by the second kernel (no float atomics: the same bits every time).
constexpr int W8_T = 64, W8_R = 32, W8_LD = W8_T + 4;

struct Wgrad8 {
    int m, n, k, splits, rows_per;       // rows_per: rows of a split
    const void* dy; long long lddy;
    const unsigned char* codes; int ldc; const unsigned char* exps; int blocks;
    float *dw, *db;                      // (splits, n, k) and (splits, n) partials, or the results when splits == 1
    long long lddw;
};

template <int TY>
__global__ void __launch_bounds__(256)
rows8_wgrad_kernel(Wgrad8 p) {
    typedef typename Elem<TY>::T T;
    __shared__ float Ys[W8_R][W8_LD], Xs[W8_R][W8_LD];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, i = lane & 15, g = lane >> 4;
    const int tk = (p.k + W8_T - 1) / W8_T;
    const int n0 = (int)(blockIdx.x / tk) * W8_T, k0 = (int)(blockIdx.x % tk) * W8_T;
    const long long r_begin = (long long)blockIdx.y * p.rows_per, r_end = min((long long)p.m, r_begin + p.rows_per);
    const T* dy = (const T*)p.dy;
    f32x4 acc[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
    float bsum = 0.f;
    const int col = tid & 63, r0 = tid >> 6;
    for (long long r = r_begin; r < r_end; r += W8_R) {
        __syncthreads();
#pragma unroll
        for (int q = 0; q < W8_R / 4; ++q) {
            const long long row = r + r0 + 4 * q;
            const bool ok = row < r_end;
            Ys[r0 + 4 * q][col] = (ok && n0 + col < p.n) ? (float)dy[row * p.lddy + n0 + col] : 0.f;
            float x = 0.f;
            if (ok && k0 + col < p.k)
                x = __builtin_amdgcn_cvt_pk_f32_fp8((int)p.codes[row * p.ldc + k0 + col], false)[0] *
                    exp2i((int)p.exps[row * p.blocks + (k0 + col) / R8_BLOCK] - 127);
            Xs[r0 + 4 * q][col] = x;
        }
        __syncthreads();
        if (k0 == 0 && wave == 0)
            for (int q = 0; q < W8_R; ++q) bsum += Ys[q][col];
#pragma unroll
        for (int q = 0; q < W8_R; q += 4) {
            const float a = Ys[q + g][wave * 16 + i];
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(a, Xs[q + g][j * 16 + i], acc[j], 0, 0, 0);
        }
    }
    float* dw = p.dw + (p.splits > 1 ? (size_t)blockIdx.y * p.n * p.k : 0);
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int n = n0 + wave * 16 + 4 * g + q, k = k0 + j * 16 + i;
            if (n < p.n && k < p.k) dw[(size_t)n * p.lddw + k] = acc[j][q];
        }
    if (k0 == 0 && wave == 0 && p.db != nullptr && n0 + col < p.n) p.db[(p.splits > 1 ? (size_t)blockIdx.y * p.n : 0) + n0 + col] = bsum;
}

// out[i] = the sum of the splits' partials in split order: items 0 .. n k - 1 are dW, then n of db
__global__ void __launch_bounds__(256)
rows8_wgrad_reduce_kernel(int n, int k, int splits, const float* __restrict__ part_w, const float* __restrict__ part_b, float* __restrict__ dw,
                          long long lddw, float* __restrict__ db) {
    const long long nk = (long long)n * k;
    const long long i = blockIdx.x * 256ll + threadIdx.x;
    if (i >= nk + (db ? n : 0)) return;
    const bool w = i < nk;
    const float* src = w ? part_w + i : part_b + (i - nk);
    const size_t step = w ? (size_t)nk : (size_t)n;
    float s0 = 0.f, s1 = 0.f, s2 = 0.f, s3 = 0.f;
    int t = 0;
    for (; t + 4 <= splits; t += 4) {
        s0 += src[(size_t)t * step];       s1 += src[(size_t)(t + 1) * step];
        s2 += src[(size_t)(t + 2) * step]; s3 += src[(size_t)(t + 3) * step];
    }
    for (; t < splits; ++t) s0 += src[(size_t)t * step];
    const float s = (s0 + s1) + (s2 + s3);
    if (w) dw[(i / k) * lddw + i % k] = s;
    else db[i - nk] = s;
}

static int wgrad8_splits(int m, int n, int k) {
    const long long tiles = (long long)divup(n, W8_T) * divup(k, W8_T);
    long long s = (1024 + tiles - 1) / tiles;
    const int cap = imax(1, m / 256);
    if (s > cap) s = cap;
    return (int)s;
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
    const size_t s = (size_t)wgrad8_splits(m, n, k);
    return s > 1 ? s * ((size_t)n * (size_t)k + (size_t)n) * sizeof(float) : 0;
}

int jm_rows8_linear_wgrad(int m, int n, int k, int type, const void* dy, long long lddy, const unsigned char* codes, int ldc, const unsigned char* exps,
                          float* dw, long long lddw, float* dbias, void* ws, size_t ws_bytes, jm_stream_t stream) {
    JM_REQUIRE(m >= 0 && n > 0 && k > 0 && type >= JM_F32 && type <= JM_F16 && dw, "rows8_linear_wgrad: m %d, n %d, k %d, type %d", m, n, k, type);
    JM_REQUIRE(lddy >= n && ldc >= k && ldc % 16 == 0 && lddw >= k, "rows8_linear_wgrad: lddy %lld, ldc %d, lddw %lld for n %d, k %d", lddy, ldc, lddw, n, k);
    JM_REQUIRE(m == 0 || (dy && codes && exps && ((uintptr_t)codes & 15) == 0), "rows8_linear_wgrad: NULL or unaligned buffers");
    const int splits = m > 0 ? wgrad8_splits(m, n, k) : 1;
    if (splits > 1 && (!ws || ws_bytes < jm_rows8_wgrad_workspace_bytes(m, n, k))) {
        set_error("rows8_linear_wgrad: workspace of %zu bytes, need %zu", ws_bytes, jm_rows8_wgrad_workspace_bytes(m, n, k));
        return JM_EWORKSPACE;
    }
    hipStream_t s = (hipStream_t)stream;
    Wgrad8 p{};
    p.m = m; p.n = n; p.k = k; p.splits = splits; p.rows_per = divup(divup(m, splits), W8_R) * W8_R;
    p.dy = dy; p.lddy = lddy; p.codes = codes; p.ldc = ldc; p.exps = exps; p.blocks = divup(k, R8_BLOCK);
    float* part_b = (float*)ws + (size_t)splits * n * k;
    if (splits > 1) { p.dw = (float*)ws; p.lddw = k; p.db = dbias ? part_b : nullptr; }
    else { p.dw = dw; p.lddw = lddw; p.db = dbias; }
    const dim3 grid((unsigned)(divup(n, W8_T) * divup(k, W8_T)), (unsigned)splits), block(256);
    if (type == JM_F32) hipLaunchKernelGGL((rows8_wgrad_kernel<JM_F32>), grid, block, 0, s, p);
    else if (type == JM_BF16) hipLaunchKernelGGL((rows8_wgrad_kernel<JM_BF16>), grid, block, 0, s, p);
    else hipLaunchKernelGGL((rows8_wgrad_kernel<JM_F16>), grid, block, 0, s, p);
    if (splits > 1) {
        const long long items = (long long)n * k + (dbias ? n : 0);
        hipLaunchKernelGGL(rows8_wgrad_reduce_kernel, dim3((unsigned)((items + 255) / 256)), block, 0, s, n, k, splits, (const float*)ws,
                           (const float*)part_b, dw, lddw, dbias);
    }
    return check_launch("rows8_linear_wgrad");
}

}  // extern "C"
