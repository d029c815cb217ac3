// Matrices held in 8-bit floating point with one scale per block of 128 (cp_blocks), the cast that makes them and their product.
#include <cfloat>

#include "cp_common.h"
#include "nt_mfma.h"

namespace {

using nt::f4;

constexpr float kTiny = 7.888609052210118e-31f;   // 2^-100: a block's largest magnitude counts as at least this
constexpr int64_t kMaxLd = int64_t(1) << 22;
constexpr int64_t kMaxRows = int64_t(1) << 30;

int check_blocks(cp_ctx *ctx, const cp_blocks *m, const char *name) {
    if (!m) return cp_set_error(ctx, CP_ERR_ARG, "%s: null description", name);
    if (m->fmt != CP_E4M3 && m->fmt != CP_E5M2) return cp_set_error(ctx, CP_ERR_ARG, "%s: fmt %d is not an 8-bit type", name, m->fmt);
    if (m->tile != 1 && m->tile != 128) return cp_set_error(ctx, CP_ERR_ARG, "%s: %d rows to a scale (1 or 128)", name, m->tile);
    if (m->rows < 0 || m->cols < 0 || m->rows > kMaxRows) return cp_set_error(ctx, CP_ERR_ARG, "%s: rows, cols out of range", name);
    if (m->ld % 128 != 0 || m->ld < m->cols || m->ld >= kMaxLd)
        return cp_set_error(ctx, CP_ERR_ARG, "%s: row stride %lld (a multiple of 128, >= cols, < 2^22)", name, (long long)m->ld);
    if (m->lds < (m->tile == 1 ? m->rows : (m->rows + 127) / 128) || m->lds > kMaxRows)
        return cp_set_error(ctx, CP_ERR_ARG, "%s: scale stride %lld", name, (long long)m->lds);
    if (m->rows && m->cols && (!m->q || !m->scale)) return cp_set_error(ctx, CP_ERR_ARG, "%s: null pointer", name);
    if (uintptr_t(m->q) % 16 || uintptr_t(m->scale) % 4) return cp_set_error(ctx, CP_ERR_ARG, "%s: alignment", name);
    return CP_OK;
}

// ---- the cast ------------------------------------------------------------------------------------------------------------
// One workgroup takes a 128 x 128 tile: exactly one block column of the matrix and, transposed, one of out_t.  A thread keeps
// an 8 x 8 patch in registers, so x is read once for both orientations; a wave's patches form 64 x 64, which makes the
// segments that it writes 64 bytes long in either.  Bound by HBM.
struct Held {
    uint8_t *q;
    float *scale;
    int64_t ld, lds;
    int fmt, tile;
};

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(double v) { return float(v); }
__device__ __forceinline__ float to_float(__bf16 v) { return float(v); }
__device__ __forceinline__ float to_float(_Float16 v) { return float(v); }

__device__ __forceinline__ float finite_abs(float v) {
    const float a = fabsf(v);
    return a <= FLT_MAX ? a : 0.f;
}

// a block's scale and the factor that its elements are cast with
__device__ __forceinline__ void scale_of(float amax, int fmt, bool pow2, float &scale, float &inv) {
    const float top = fmt == CP_E4M3 ? 448.f : 57344.f;
    amax = fmaxf(amax, kTiny);
    scale = amax / top;
    if (pow2) {
        const uint32_t b = __float_as_uint(scale), e = (b >> 23) + ((b & 0x7fffffu) != 0);   // scale is a normal number
        scale = __uint_as_float(e << 23);
        inv = __uint_as_float((254u - e) << 23);
    } else {
        inv = top / amax;
    }
}

__device__ __forceinline__ float cut(float x, float inv, float top) {
    const float y = __builtin_amdgcn_fmed3f(x * inv, -top, top);
    return fabsf(x) <= FLT_MAX ? y : __uint_as_float(0x7fc00000u);
}

__device__ __forceinline__ uint32_t pack4(const float (&y)[4], int fmt) {
    int w = 0;
    if (fmt == CP_E4M3) {
        w = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], w, false);
        w = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], w, true);
    } else {
        w = __builtin_amdgcn_cvt_pk_bf8_f32(y[0], y[1], w, false);
        w = __builtin_amdgcn_cvt_pk_bf8_f32(y[2], y[3], w, true);
    }
    return uint32_t(w);
}

template <typename T>
__global__ void __launch_bounds__(256) k_quant_blocks(const T *__restrict__ x, int64_t rows, int64_t cols, int64_t ldx, int vec,
                                                      int pow2, Held o, Held t) {
    __shared__ float rmax[2][128], cmax[2][128];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int lr = (wave >> 1) * 64 + (lane >> 3) * 8, lc = (wave & 1) * 64 + (lane & 7) * 8;
    const int64_t r0 = int64_t(blockIdx.y) * 128, c0 = int64_t(blockIdx.x) * 128;
    const int64_t row = r0 + lr, col = c0 + lc;

    float v[8][8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const T *p = x + (row + i) * ldx + col;
        if (vec && row + i < rows && col + 8 <= cols) {
            struct alignas(16) Eight {
                T e[8];
            };
            const Eight e = *reinterpret_cast<const Eight *>(p);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[i][j] = to_float(e.e[j]);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[i][j] = row + i < rows && col + j < cols ? to_float(p[j]) : 0.f;
        }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        float m = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) m = fmaxf(m, finite_abs(v[i][j]));
        for (int s = 1; s < 8; s <<= 1) m = fmaxf(m, __shfl_xor(m, s));
        if ((lane & 7) == 0) rmax[wave & 1][lr + i] = m;
    }
    if (t.q) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            float m = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) m = fmaxf(m, finite_abs(v[i][j]));
            for (int s = 8; s < 64; s <<= 1) m = fmaxf(m, __shfl_xor(m, s));
            if (lane < 8) cmax[wave >> 1][lc + j] = m;
        }
    }
    __syncthreads();
    float whole = 0.f;
    if ((o.q && o.tile != 1) || (t.q && t.tile != 1)) {
        whole = fmaxf(fmaxf(rmax[0][lane], rmax[1][lane]), fmaxf(rmax[0][lane + 64], rmax[1][lane + 64]));
        for (int s = 1; s < 64; s <<= 1) whole = fmaxf(whole, __shfl_xor(whole, s));
    }
    float scale, inv;
    if (o.q) {
        const float top = o.fmt == CP_E4M3 ? 448.f : 57344.f;
        float *sp = o.scale + blockIdx.x * o.lds;
        if (o.tile != 1) {
            scale_of(whole, o.fmt, pow2, scale, inv);
            if (tid == 0) sp[blockIdx.y] = scale;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (row + i >= rows) break;
            if (o.tile == 1) {
                scale_of(fmaxf(rmax[0][lr + i], rmax[1][lr + i]), o.fmt, pow2, scale, inv);
                if (lc == 0) sp[row + i] = scale;
            }
            uint32_t w[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float y[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) y[e] = cut(v[i][4 * h + e], inv, top);
                w[h] = pack4(y, o.fmt);
            }
            *reinterpret_cast<uint2 *>(o.q + (row + i) * o.ld + col) = make_uint2(w[0], w[1]);
        }
    }
    if (t.q) {
        const float top = t.fmt == CP_E4M3 ? 448.f : 57344.f;
        float *sp = t.scale + blockIdx.y * t.lds;
        if (t.tile != 1) {
            scale_of(whole, t.fmt, pow2, scale, inv);
            if (tid == 0) sp[blockIdx.x] = scale;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if (col + j >= cols) break;
            if (t.tile == 1) {
                scale_of(fmaxf(cmax[0][lc + j], cmax[1][lc + j]), t.fmt, pow2, scale, inv);
                if (lr == 0) sp[col + j] = scale;
            }
            uint32_t w[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float y[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) y[e] = cut(v[4 * h + e][j], inv, top);
                w[h] = pack4(y, t.fmt);
            }
            *reinterpret_cast<uint2 *>(t.q + (col + j) * t.ld + row) = make_uint2(w[0], w[1]);
        }
    }
}

Held held(const cp_blocks *m) {
    Held h = {};
    if (m) h = {static_cast<uint8_t *>(m->q), m->scale, m->ld, m->lds, m->fmt, m->tile};
    return h;
}

template <typename T>
void launch_quant(cp_ctx *ctx, const void *x, int64_t rows, int64_t cols, int64_t ldx, int flags, const cp_blocks *out,
                  const cp_blocks *out_t) {
    const int vec = uintptr_t(x) % 16 == 0 && size_t(ldx) * sizeof(T) % 16 == 0;
    const dim3 grid(uint32_t((cols + 127) / 128), uint32_t((rows + 127) / 128));
    k_quant_blocks<T><<<grid, 256, 0, ctx->stream>>>(static_cast<const T *>(x), rows, cols, ldx, vec, flags & CP_QUANT_POW2,
                                                     held(out), held(out_t));
}

// ---- the product ---------------------------------------------------------------------------------------------------------
struct Product {
    const char *a, *b;
    const float *sa, *sb, *bias;
    void *c;
    int64_t sa_step, sb_step, ldc;   // scale strides per block column
    uint32_t lda, ldb;
    int M, N, steps, tiles_m, tiles_n;
    int a_shift, b_shift;            // row -> scale: 0 (one per row) or 7
    int c_dtype, c_vec;
};

__device__ __forceinline__ void store_c(const Product &p, int64_t i, int j, f4 v) {
    if (p.bias) {
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (j + r < p.N) v[r] += p.bias[j + r];
    }
    const int64_t at = i * p.ldc + j;
    if (p.c_vec && j + 4 <= p.N) {
        if (p.c_dtype == CP_F32) {
            *reinterpret_cast<f4 *>(static_cast<float *>(p.c) + at) = v;
        } else if (p.c_dtype == CP_BF16) {
            typedef __bf16 b4 __attribute__((ext_vector_type(4)));
            *reinterpret_cast<b4 *>(static_cast<__bf16 *>(p.c) + at) = __builtin_convertvector(v, b4);
        } else {
            *reinterpret_cast<nt::h4 *>(static_cast<_Float16 *>(p.c) + at) = __builtin_convertvector(v, nt::h4);
        }
        return;
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        if (j + r >= p.N) return;
        if (p.c_dtype == CP_F32) static_cast<float *>(p.c)[at + r] = v[r];
        else if (p.c_dtype == CP_BF16) static_cast<__bf16 *>(p.c)[at + r] = __bf16(v[r]);
        else static_cast<_Float16 *>(p.c)[at + r] = _Float16(v[r]);
    }
}

template <int BM, int BN, int NWM, int NWN, int FA, int FB, bool COMMON, bool WIDE>
__global__ void __launch_bounds__(64 * NWM * NWN) k_matmul_blocks(Product p) {
    constexpr int T = 64 * NWM * NWN, WI = BM / NWM / 16, WJ = BN / NWN / 16;
    static_assert((BM + BN) / 64 == NWM * NWN, "one wave per 64 scales");
    static_assert(!COMMON || (128 % (16 * WJ) == 0 && BN % 128 == 0), "a wave's columns share their scale");
    __shared__ alignas(1024) char a0[BM * 128], a1[BM * 128], b0[BN * 128], b1[BN * 128];
    __shared__ alignas(1024) float s0[BM + BN], s1[BM + BN];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave / NWN, wn = wave % NWN;
    const int tile = nt::xcd_order(blockIdx.x, p.tiles_m * p.tiles_n);
    const int tm = tile % p.tiles_m, tn = tile / p.tiles_m;
    const int i0 = tm * BM, j0 = tn * BN;

    nt::Loader<BM, T> la;
    nt::Loader<BN, T> lb;
    la.init(p.a + int64_t(i0) * p.lda, p.lda, p.M - i0, tid);
    lb.init(p.b + int64_t(j0) * p.ldb, p.ldb, p.N - j0, tid);
    const bool for_a = wave < BM / 64;
    const float *sp;
    int64_t s_step;
    if (for_a) {
        const int r = i0 + wave * 64 + lane;
        sp = p.sa + ((r < p.M ? r : p.M - 1) >> p.a_shift);
        s_step = p.sa_step;
    } else {
        const int r = j0 + (wave - BM / 64) * 64 + lane;
        sp = p.sb + ((r < p.N ? r : p.N - 1) >> p.b_shift);
        s_step = p.sb_step;
    }
    f4 acc[WI][WJ];
#pragma unroll
    for (int i = 0; i < WI; ++i)
#pragma unroll
        for (int j = 0; j < WJ; ++j) acc[i][j] = f4{0.f, 0.f, 0.f, 0.f};
    const int ra = wm * WI * 16, rb = wn * WJ * 16;

    auto fetch = [&](int k, char *a, char *b, float *s) {
        la.issue(k, a, wave);
        lb.issue(k, b, wave);
        nt::load_lds4(sp + k * s_step, s + wave * 64);
    };
    auto compute = [&](const char *a, const char *b, const float *s) {
        nt::products8<WI, WJ, FA, FB, COMMON, WIDE>(a + ra * 128, b + rb * 128, s + ra, s + BM + rb, lane, acc);
    };
    if (p.steps > 0) fetch(0, a0, b0, s0);
    for (int k = 0; k < p.steps; k += 2) {
        nt::stage_barrier();
        if (k + 1 < p.steps) fetch(k + 1, a1, b1, s1);
        compute(a0, b0, s0);
        if (k + 1 >= p.steps) break;
        nt::stage_barrier();
        if (k + 2 < p.steps) fetch(k + 2, a0, b0, s0);
        compute(a1, b1, s1);
    }
#pragma unroll
    for (int i = 0; i < WI; ++i) {
        const int row = i0 + ra + i * 16 + (lane & 15);
        if (row >= p.M) continue;
#pragma unroll
        for (int j = 0; j < WJ; ++j) store_c(p, row, j0 + rb + j * 16 + (lane >> 4) * 4, acc[i][j]);
    }
}

int check_product(cp_ctx *ctx, const cp_blocks *A, const cp_blocks *B, int c_dtype, int64_t ldc) {
    CP_TRY(check_blocks(ctx, A, "A"));
    CP_TRY(check_blocks(ctx, B, "B"));
    if (A->cols != B->cols)
        return cp_set_error(ctx, CP_ERR_ARG, "A has %lld columns, B %lld", (long long)A->cols, (long long)B->cols);
    if (c_dtype != CP_F32 && c_dtype != CP_BF16 && c_dtype != CP_F16) return cp_set_error(ctx, CP_ERR_ARG, "c_dtype %d", c_dtype);
    if (ldc < B->rows) return cp_set_error(ctx, CP_ERR_ARG, "ldc %lld < %lld", (long long)ldc, (long long)B->rows);
    if (((A->rows + 127) / 128) * ((B->rows + 127) / 128) >= (int64_t(1) << 31))
        return cp_set_error(ctx, CP_ERR_UNSUPPORTED, "C is too large");
    return CP_OK;
}

template <int FA, int FB, bool COMMON, bool WIDE>
void launch_product(cp_ctx *ctx, const Product &p) {
    k_matmul_blocks<128, 128, 2, 2, FA, FB, COMMON, WIDE><<<p.tiles_m * p.tiles_n, 256, 0, ctx->stream>>>(p);
}

template <int FA, int FB>
void launch_product(cp_ctx *ctx, const Product &p) {
    const bool wide = p.c_dtype != CP_BF16;   // what the 8-bit matrix instructions drop is below bfloat16's rounding only
    if (p.b_shift) wide ? launch_product<FA, FB, true, true>(ctx, p) : launch_product<FA, FB, true, false>(ctx, p);
    else wide ? launch_product<FA, FB, false, true>(ctx, p) : launch_product<FA, FB, false, false>(ctx, p);
}

}  // namespace

extern "C" int cp_blocks_check(const cp_blocks *m) { return check_blocks(nullptr, m, "matrix"); }

extern "C" int cp_quant_blocks(cp_ctx *ctx, const void *x, int x_dtype, int64_t rows, int64_t cols, int64_t ldx, int flags,
                               const cp_blocks *out, const cp_blocks *out_t) {
    if (!ctx) return CP_ERR_ARG;
    if (x_dtype != CP_F32 && x_dtype != CP_F64 && x_dtype != CP_BF16 && x_dtype != CP_F16)
        return cp_set_error(ctx, CP_ERR_ARG, "x_dtype %d", x_dtype);
    if (rows < 0 || cols < 0 || ldx < cols) return cp_set_error(ctx, CP_ERR_ARG, "rows, cols, ldx");
    if (flags & ~CP_QUANT_POW2) return cp_set_error(ctx, CP_ERR_ARG, "flags %d", flags);
    if (!out && !out_t) return cp_set_error(ctx, CP_ERR_ARG, "no output");
    if (out) {
        CP_TRY(check_blocks(ctx, out, "out"));
        if (out->rows != rows || out->cols != cols) return cp_set_error(ctx, CP_ERR_ARG, "out is not [rows, cols]");
    }
    if (out_t) {
        CP_TRY(check_blocks(ctx, out_t, "out_t"));
        if (out_t->rows != cols || out_t->cols != rows) return cp_set_error(ctx, CP_ERR_ARG, "out_t is not [cols, rows]");
    }
    if (out && out_t && out->q == out_t->q && out->q) return cp_set_error(ctx, CP_ERR_ARG, "out and out_t are the same memory");
    if (!rows || !cols) return CP_OK;
    const size_t size = x_dtype == CP_F64 ? 8 : x_dtype == CP_F32 ? 4 : 2;
    if (!x || uintptr_t(x) % size) return cp_set_error(ctx, CP_ERR_ARG, "x is null or misaligned");
    if ((rows + 127) / 128 > 65535) return cp_set_error(ctx, CP_ERR_UNSUPPORTED, "more than 65535 * 128 rows");
    CP_HIP(ctx, hipSetDevice(ctx->device));
    switch (x_dtype) {
        case CP_F32: launch_quant<float>(ctx, x, rows, cols, ldx, flags, out, out_t); break;
        case CP_F64: launch_quant<double>(ctx, x, rows, cols, ldx, flags, out, out_t); break;
        case CP_BF16: launch_quant<__bf16>(ctx, x, rows, cols, ldx, flags, out, out_t); break;
        default: launch_quant<_Float16>(ctx, x, rows, cols, ldx, flags, out, out_t); break;
    }
    CP_LAUNCH_CHECK(ctx);
    return CP_OK;
}

extern "C" int cp_matmul_blocks_workspace(const cp_blocks *A, const cp_blocks *B, int c_dtype, int64_t ldc, size_t *bytes) {
    if (!bytes) return CP_ERR_ARG;
    CP_TRY(check_product(nullptr, A, B, c_dtype, ldc));
    *bytes = 0;
    return CP_OK;
}

extern "C" int cp_matmul_blocks(cp_ctx *ctx, const cp_blocks *A, const cp_blocks *B, const float *bias, void *C, int c_dtype,
                                int64_t ldc, void *ws, size_t ws_bytes) {
    if (!ctx) return CP_ERR_ARG;
    CP_TRY(check_product(ctx, A, B, c_dtype, ldc));
    if (!A->rows || !B->rows) return CP_OK;
    const size_t size = c_dtype == CP_F32 ? 4 : 2;
    if (!C || uintptr_t(C) % size || uintptr_t(bias) % 4) return cp_set_error(ctx, CP_ERR_ARG, "C is null or misaligned");
    (void)ws, (void)ws_bytes;
    CP_HIP(ctx, hipSetDevice(ctx->device));
    Product p = {};
    p.a = static_cast<const char *>(A->q);
    p.b = static_cast<const char *>(B->q);
    p.sa = A->scale;
    p.sb = B->scale;
    p.sa_step = A->lds;
    p.sb_step = B->lds;
    p.bias = bias;
    p.c = C;
    p.ldc = ldc;
    p.lda = uint32_t(A->ld);
    p.ldb = uint32_t(B->ld);
    p.M = int(A->rows);
    p.N = int(B->rows);
    p.steps = int((A->cols + 127) / 128);
    p.tiles_m = (p.M + 127) / 128;
    p.tiles_n = (p.N + 127) / 128;
    p.a_shift = A->tile == 1 ? 0 : 7;
    p.b_shift = B->tile == 1 ? 0 : 7;
    p.c_dtype = c_dtype;
    p.c_vec = ldc % 4 == 0 && uintptr_t(C) % (4 * size) == 0;
    const bool a5 = A->fmt == CP_E5M2, b5 = B->fmt == CP_E5M2;
    if (a5 && b5) launch_product<1, 1>(ctx, p);
    else if (a5) launch_product<1, 0>(ctx, p);
    else if (b5) launch_product<0, 1>(ctx, p);
    else launch_product<0, 0>(ctx, p);
    CP_LAUNCH_CHECK(ctx);
    return CP_OK;
}
