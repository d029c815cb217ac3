// Matrices held in 8-bit floating point with one scale per block of 128 (cp_blocks), the cast that makes them and their product.
#include <algorithm>
#include <cfloat>
#include <cmath>

#include "cp_common.h"
#include "nt_mfma.h"

namespace {

using nt::f4;

constexpr float kTiny = 7.888609052210118e-31f;   // 2^-100: a block's largest magnitude counts as at least this
constexpr int64_t kMaxLd = int64_t(1) << 22;
constexpr int64_t kMaxRows = int64_t(1) << 30;
constexpr int64_t kMaxThreads = (int64_t(1) << 32) - 1;   // of a launch

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
// segments that it writes 64 bytes long in either.  Bound by HBM, as long as the arithmetic stays short: the largest magnitudes
// are found on the bit patterns; a thread makes the factors of one row or column, not of its patch's sixteen; and what only
// infinities and NaN need is done in tiles that hold one.  f32 [20000, 4608] both ways: 106 us for 559 MB (5.2 TB/s; adding two large
// float32 matrices, which also reads two bytes for each that it writes, reaches 5.7, a copy 4.97), bf16 [4096, 25088]: 87 us for 411 MB,
// bf16 [20000, 4005], whose rows begin anywhere: 82 us for 324 MB; the same on six inputs in turn, none of which is in a cache.
// (No cut to +-fmax is needed: a finite x times the inverse exceeds fmax by two roundings at most, and rounds to it.)
struct Held {
    uint8_t *q;
    float *scale;
    int64_t rows, ld, lds;
    int fmt, tile;
};

// eight neighbours, at any element's address
__device__ __forceinline__ void load8(const float *p, float (&v)[8]) {
    const f4 a = *reinterpret_cast<const nt::f4u *>(p), b = *reinterpret_cast<const nt::f4u *>(p + 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = a[e], v[e + 4] = b[e];
}
__device__ __forceinline__ void load8(const double *p, float (&v)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = float(p[e]);
}
__device__ __forceinline__ void load8(const __bf16 *p, float (&v)[8]) {
    const nt::b8 a = *reinterpret_cast<const nt::b8u *>(p);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = float(a[e]);
}
__device__ __forceinline__ void load8(const _Float16 *p, float (&v)[8]) {
    const nt::h8 a = *reinterpret_cast<const nt::h8u *>(p);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = float(a[e]);
}

constexpr uint32_t kInf = 0x7f800000u;
// |v| as an integer of the same order; FINITE: zero for what is not
template <bool FINITE>
__device__ __forceinline__ uint32_t magnitude(float v) {
    const uint32_t b = __float_as_uint(v) & 0x7fffffffu;
    return FINITE && b >= kInf ? 0u : b;
}

template <int CTRL>
__device__ __forceinline__ uint32_t max_with(uint32_t v) {
    return max(v, uint32_t(__builtin_amdgcn_update_dpp(0, int(v), CTRL, 0xf, 0xf, true)));
}

// The largest magnitudes into LDS: of the rows over this wave's 64 columns, of the columns over this thread's eight rows
// (group: which eight of the tile).  Returns the thread's largest.
template <bool FINITE>
__device__ __forceinline__ uint32_t maxima(const float (&v)[8][8], uint32_t *rmax, uint32_t *cmax, bool columns, int lr, int lane) {
    uint32_t all = 0, rm[8], cm[8] = {};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        rm[i] = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint32_t m = magnitude<FINITE>(v[i][j]);
            rm[i] = max(rm[i], m);
            cm[j] = max(cm[j], m);
        }
        all = max(all, rm[i]);
        NT_STAY();   // one row after the other: all magnitudes at once would take as many registers again
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) rm[i] = max_with<0x141>(max_with<0x4E>(max_with<0xB1>(rm[i])));   // over eight neighbouring lanes
    if ((lane & 7) == 0) {
        *reinterpret_cast<uint4 *>(rmax + lr) = make_uint4(rm[0], rm[1], rm[2], rm[3]);
        *reinterpret_cast<uint4 *>(rmax + lr + 4) = make_uint4(rm[4], rm[5], rm[6], rm[7]);
    }
    if (columns) {
        *reinterpret_cast<uint4 *>(cmax) = make_uint4(cm[0], cm[1], cm[2], cm[3]);
        *reinterpret_cast<uint4 *>(cmax + 4) = make_uint4(cm[4], cm[5], cm[6], cm[7]);
    }
    return all;
}

// a block's scale and the factor that its elements are cast with
__device__ __forceinline__ void scale_of(uint32_t largest, int fmt, bool pow2, float &scale, float &inv) {
    const float top = fmt == CP_E4M3 ? 448.f : 57344.f, amax = fmaxf(__uint_as_float(largest), kTiny);
    scale = amax / top;
    if (pow2) {
        const uint32_t b = __float_as_uint(scale), e = (b >> 23) + ((b & 0x7fffffu) != 0);   // scale is a normal number
        scale = __uint_as_float(e << 23);
        inv = __uint_as_float((254u - e) << 23);
    } else {
        inv = top / amax;
    }
}

// four numbers times their factor, in 8 bits; SPECIAL: what is not finite becomes NaN
template <int FMT, bool SPECIAL>
__device__ __forceinline__ uint32_t pack4(float x0, float x1, float x2, float x3, float inv) {
    const float x[4] = {x0, x1, x2, x3};
    float y[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        y[e] = x[e] * inv;
        if (SPECIAL && magnitude<false>(x[e]) >= kInf) y[e] = __uint_as_float(0x7fc00000u);
    }
    int w = 0;
    if (FMT == CP_E4M3) {
        w = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], w, false);
        w = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], w, true);
    } else {
        w = __builtin_amdgcn_cvt_pk_bf8_f32(y[0], y[1], w, false);
        w = __builtin_amdgcn_cvt_pk_bf8_f32(y[2], y[3], w, true);
    }
    return uint32_t(w);
}

// a thread's patch into its eight rows of a matrix (TURN: of the transpose), `at`: the first's place, n: how many there are
template <int FMT, bool SPECIAL, bool TURN>
__device__ __forceinline__ void write_patch(const float (&v)[8][8], const float *inverse, uint8_t *at, int64_t ld, int64_t n) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if (i >= n) break;
        const float f = inverse[i];
        uint2 w;
        w.x = TURN ? pack4<FMT, SPECIAL>(v[0][i], v[1][i], v[2][i], v[3][i], f) : pack4<FMT, SPECIAL>(v[i][0], v[i][1], v[i][2], v[i][3], f);
        w.y = TURN ? pack4<FMT, SPECIAL>(v[4][i], v[5][i], v[6][i], v[7][i], f) : pack4<FMT, SPECIAL>(v[i][4], v[i][5], v[i][6], v[i][7], f);
        *reinterpret_cast<uint2 *>(at) = w;
        at += ld;
        NT_STAY();   // row after row, in few registers
    }
}
template <bool TURN>
__device__ __forceinline__ void write_patch(const float (&v)[8][8], const float *inverse, const Held &h, int64_t row, int64_t col, bool special) {
    uint8_t *at = h.q + row * h.ld + col;
    const int64_t n = h.rows - row;
    if (h.fmt == CP_E4M3) special ? write_patch<CP_E4M3, true, TURN>(v, inverse, at, h.ld, n) : write_patch<CP_E4M3, false, TURN>(v, inverse, at, h.ld, n);
    else special ? write_patch<CP_E5M2, true, TURN>(v, inverse, at, h.ld, n) : write_patch<CP_E5M2, false, TURN>(v, inverse, at, h.ld, n);
}

template <typename T>
__global__ void __launch_bounds__(256) k_quant_blocks(const T *__restrict__ x, int64_t rows, int64_t cols, int64_t ldx, int tiles_c, int pow2,
                                                      Held o, Held t) {
    __shared__ alignas(16) uint32_t rmax[2][128], cmax[16][128];
    __shared__ float inverse[2][128];   // of the tile's rows and columns
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int lr = (wave >> 1) * 64 + (lane >> 3) * 8, lc = (wave & 1) * 64 + (lane & 7) * 8;
    // neighbours in a row on one XCD: where rows begin inside a line, they share it in that XCD's L2
    const int tile = nt::xcd_runs(blockIdx.x, gridDim.x), tr = tile / tiles_c, tc = tile % tiles_c;
    const int64_t r0 = int64_t(tr) * 128, c0 = int64_t(tc) * 128;
    const int64_t row = r0 + lr, col = c0 + lc;

    float v[8][8];
    const T *p = x + row * ldx + col;
    if (r0 + 128 <= rows && c0 + 128 <= cols) {
#pragma unroll
        for (int i = 0; i < 8; ++i) load8(p + i * ldx, v[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i, p += ldx) {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[i][j] = 0.f;
            if (row + i < rows) {
                if (col + 8 <= cols) {
                    load8(p, v[i]);
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (col + j < cols) v[i][j] = float(p[j]);
                }
            }
            NT_STAY();   // the edge's rows one after the other, in few registers
        }
    }
    const uint32_t mine = maxima<false>(v, rmax[wave & 1], cmax[lr >> 3] + lc, t.q, lr, lane);
    const bool special = __syncthreads_or(mine >= kInf);
    if (special) {
        // (to the compiler these are new numbers: it would keep 64 magnitudes in registers for this rare path)
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) asm volatile("" : "+v"(v[i][j]));
        maxima<true>(v, rmax[wave & 1], cmax[lr >> 3] + lc, t.q, lr, lane);
        __syncthreads();
    }
    // thread k < 128: row k of the tile; 128 + k: column k
    {
        const bool is_col = tid >= 128;
        const int k = tid & 127;
        const Held &h = is_col ? t : o;
        if (h.q) {
            uint32_t m = max(rmax[0][k], rmax[1][k]);
            if (is_col) {
                m = 0;
#pragma unroll
                for (int g = 0; g < 16; ++g) m = max(m, cmax[g][k]);
            }
            if (h.tile != 1) {
                m = max(max(rmax[0][lane], rmax[1][lane]), max(rmax[0][lane + 64], rmax[1][lane + 64]));
#pragma unroll
                for (int s = 1; s < 64; s <<= 1) m = max(m, uint32_t(__shfl_xor(int(m), s)));
            }
            float scale;
            scale_of(m, h.fmt, pow2, scale, inverse[is_col][k]);
            float *sp = is_col ? t.scale + tr * t.lds : o.scale + tc * o.lds;
            const int64_t at = (is_col ? c0 : r0) + k, n = is_col ? cols : rows;
            if (h.tile == 1 ? at < n : k == 0) sp[h.tile == 1 ? at : at / 128] = scale;
        }
    }
    __syncthreads();
    if (o.q) write_patch<false>(v, inverse[0] + lr, o, row, col, special);
    if (t.q) write_patch<true>(v, inverse[1] + lc, t, col, row, special);
}

Held held(const cp_blocks *m) {
    Held h = {};
    if (m) h = {static_cast<uint8_t *>(m->q), m->scale, m->rows, m->ld, m->lds, m->fmt, m->tile};
    return h;
}

template <typename T>
void launch_quant(cp_ctx *ctx, const void *x, int64_t rows, int64_t cols, int64_t ldx, int flags, const cp_blocks *out,
                  const cp_blocks *out_t) {
    const int64_t tiles_c = (cols + 127) / 128, tiles_r = (rows + 127) / 128;
    k_quant_blocks<T><<<uint32_t(tiles_c * tiles_r), 256, 0, ctx->stream>>>(static_cast<const T *>(x), rows, cols, ldx, int(tiles_c),
                                                                            flags & CP_QUANT_POW2, held(out), held(out_t));
}

// ---- the product ---------------------------------------------------------------------------------------------------------
struct Product {
    const char *a, *b;
    const float *sa, *sb, *bias;
    void *c;
    int64_t sa_step, sb_step, ldc;   // scale strides per block column
    uint32_t lda, ldb;
    int M, N, steps, tiles_m, tiles_n, pieces;
    int a_shift, b_shift;            // row -> scale: 0 (one per row) or 7
    int c_dtype;
    float *parts;
    int *counts;
};

__device__ __forceinline__ void store4(const Product &p, int64_t i, int j, f4 v) {
    const int64_t at = i * p.ldc + j;
    if (p.c_dtype == CP_F32) {
        *reinterpret_cast<nt::f4u *>(static_cast<float *>(p.c) + at) = v;
    } else if (p.c_dtype == CP_BF16) {
        *reinterpret_cast<nt::b4u *>(static_cast<__bf16 *>(p.c) + at) = __builtin_convertvector(v, nt::b4);
    } else {
        *reinterpret_cast<nt::h4u *>(static_cast<_Float16 *>(p.c) + at) = __builtin_convertvector(v, nt::h4);
    }
}
__device__ __forceinline__ void store1(const Product &p, int64_t i, int j, float v) {
    const int64_t at = i * p.ldc + j;
    if (p.c_dtype == CP_F32) static_cast<float *>(p.c)[at] = v;
    else if (p.c_dtype == CP_BF16) static_cast<__bf16 *>(p.c)[at] = __bf16(v);
    else static_cast<_Float16 *>(p.c)[at] = _Float16(v);
}

__device__ __forceinline__ void store8(const Product &p, int64_t i, int j, const float (&v)[8]) {
    const int64_t at = i * p.ldc + j;
    if (p.c_dtype == CP_BF16) {
        nt::b8 q;
#pragma unroll
        for (int e = 0; e < 8; ++e) q[e] = __bf16(v[e]);
        *reinterpret_cast<nt::b8u *>(static_cast<__bf16 *>(p.c) + at) = q;
    } else {
        nt::h8 q;
#pragma unroll
        for (int e = 0; e < 8; ++e) q[e] = _Float16(v[e]);
        *reinterpret_cast<nt::h8u *>(static_cast<_Float16 *>(p.c) + at) = q;
    }
}

// A wave's part of C [16 WI rows from i0, 16 WJ columns from j0]
template <int WI, int WJ>
__device__ __forceinline__ void write_c(const Product &p, const f4 (&acc)[WI][WJ], int i0, int j0, const nt::Patch<WI, WJ> &patch) {
    typedef nt::Patch<WI, WJ> Patch;
    const int each = p.c_dtype == CP_F32 ? 4 : 8, mine = j0 + patch.lane % (Patch::COLS / each) * each;
    float bias[8];   // a lane's columns are the same in all of its groups
#pragma unroll
    for (int e = 0; e < 8; ++e) bias[e] = p.bias && mine + e < p.N ? p.bias[mine + e] : 0.f;
#pragma unroll
    for (int pass = 0; pass < Patch::PASSES; ++pass) {
        const int ip = i0 + pass * Patch::ROWS;
        if (ip >= p.M) break;
        patch.put(acc, pass, 1.f);
        if (p.c_dtype == CP_F32) {
#pragma unroll
            for (int u = 0; u < 2 * Patch::EIGHTS; ++u) {
                int i, j;
                const f4 v = patch.four_of_row(u, i, j) + f4{bias[0], bias[1], bias[2], bias[3]};
                i += ip;
                j += j0;
                if (i >= p.M) continue;
                if (j + 4 <= p.N) {
                    store4(p, i, j, v);
                } else {
#pragma unroll
                    for (int e = 0; e < 3; ++e)
                        if (j + e < p.N) store1(p, i, j + e, v[e]);
                }
            }
            continue;
        }
#pragma unroll
        for (int u = 0; u < Patch::EIGHTS; ++u) {
            int i, j;
            float v[8];
            patch.of_row(u, i, j, v);
            i += ip;
            j += j0;
            if (i >= p.M) continue;
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] += bias[e];
            if (j + 8 <= p.N) {
                store8(p, i, j, v);
            } else {
#pragma unroll
                for (int e = 0; e < 7; ++e)
                    if (j + e < p.N) store1(p, i, j + e, v[e]);
            }
        }
    }
}

// One tile of C, or a piece of k of it, to a workgroup.  COMMON: B's rows share their scales in blocks of 128 (weights), so that a
// wave's sums take a row's factor; else a row's and a column's.  Beside the matrix instructions a step has those
// factors in a fused add for every number of the tile (and a product): bound by both together.  8192^3, every row with its own scales: 527 us, 2.09
// PFLOP/s (a library product without any scales 358), common scales 439; those, 20000 x 512 x 4005: 70 us, 1.17 (its
// 80 MB come from HBM one step ahead of their use).  WIDE (float32 and fp16 results):
// the operands are widened in registers and go through the fp16 instructions, twice as many: 512 x 4005 x 20000, 112 us, 0.73
// PFLOP/s (104 if the conversions cost nothing); 256 x 256 tiles would need more registers than there are.
template <class CFG, int FA, int FB, bool COMMON, bool WIDE>
__global__ void __launch_bounds__(CFG::T) k_matmul_blocks(Product p) {
    constexpr int BM = CFG::BM, BN = CFG::BN, T = CFG::T, WI = CFG::WI, WJ = CFG::WJ;
    static_assert((BM + BN) / 64 <= CFG::NWM * CFG::NWN, "one wave per 64 scales");
    static_assert(!COMMON || 128 % (16 * WJ) == 0, "a wave's columns share their scale");
    NT_STAGES(st, CFG::STAGES, CFG::STAGE + (BM + BN) * 4);
    __shared__ int flag;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave / CFG::NWN, wn = wave % CFG::NWN;
    const int at = nt::xcd_order(blockIdx.x, gridDim.x), tiles = p.tiles_m * p.tiles_n, piece = at / tiles, tile = at % tiles;
    const int k0 = int(int64_t(p.steps) * piece / p.pieces), k1 = int(int64_t(p.steps) * (piece + 1) / p.pieces);
    int tm, tn;
    nt::tile_at(tile, p.tiles_m, p.tiles_n, tm, tn);
    const int i0 = tm * BM, j0 = tn * BN;

    nt::Loader<BM, T> la;
    nt::Loader<BN, T> lb;
    la.init(p.a + int64_t(i0) * p.lda + int64_t(k0) * 128, p.lda, p.M - i0, tid);
    lb.init(p.b + int64_t(j0) * p.ldb + int64_t(k0) * 128, p.ldb, p.N - j0, tid);
    // the step's scales, 64 to a wave; waves without any load the last ones again (every wave waits for as many loads)
    const int sw = wave < (BM + BN) / 64 ? wave : (BM + BN) / 64 - 1;
    const float *sp;
    int64_t s_step;
    if (sw < BM / 64) {
        const int r = i0 + sw * 64 + lane;
        sp = p.sa + ((r < p.M ? r : p.M - 1) >> p.a_shift);
        s_step = p.sa_step;
    } else {
        const int r = j0 + (sw - BM / 64) * 64 + lane;
        sp = p.sb + ((r < p.N ? r : p.N - 1) >> p.b_shift);
        s_step = p.sb_step;
    }
    sp += k0 * s_step;
    f4 acc[WI][WJ];
#pragma unroll
    for (int i = 0; i < WI; ++i)
#pragma unroll
        for (int j = 0; j < WJ; ++j) acc[i][j] = f4{0.f, 0.f, 0.f, 0.f};
    const int ra = wm * WI * 16, rb = wn * WJ * 16;
    if (k1 > k0) nt::pipeline<CFG::STAGES, CFG::LOADS + 1, CFG::PARTS>(
        st, k1 - k0,
        [&](int k, char *s, int part, int parts) {
            if (part == 0) nt::load_lds4(sp + k * s_step, reinterpret_cast<float *>(s + CFG::STAGE) + sw * 64);
            la.issue(k, s, wave, part, parts);
            lb.issue(k, s + BM * 128, wave, part, parts);
        },
        [&](const char *s, auto between) {
            const float *sc = reinterpret_cast<const float *>(s + CFG::STAGE);
            nt::products8<WI, WJ, FA, FB, COMMON, WIDE>(s + ra * 128, s + (BM + rb) * 128, sc + ra, sc + BM + rb, lane, acc, between);
        });
    if (p.pieces > 1 && !nt::join<T>(acc, piece, p.pieces, p.parts + int64_t(tile) * (BM * BN), tiles, p.counts + tile, &flag, tid)) return;
    write_c<WI, WJ>(p, acc, i0 + ra, j0 + rb, nt::Patch<WI, WJ>::template of<CFG>(st, wave, lane));
}

// Few rows of A: bound by reading B once.  A workgroup takes sixteen rows of B and its eight waves an eighth of k each, straight
// from memory into the matrix instruction's registers (a lane holds 32 bytes of one row: the K order within a block is the same
// for A and B, and that is all that a sum needs); their sums are added in the order of k.  Up to 128 rows (the waves' sums take 64 KB
// of LDS then), while the tiles' launch costs more (form_of): one row by 4096 x 4096 takes 5.6 us (17 MB), a call of it 7.3 -- in 64 x 64 tiles, most of whose rows
// would be padding, 12.
template <int MT, int FA, int FB, bool COMMON, bool WIDE>
__global__ void __launch_bounds__(512) k_matmul_blocks_rows(Product p) {
    __shared__ alignas(16) float sum[8][MT][64][4];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int j0 = blockIdx.x * 16, jr = j0 + (lane & 15), o = (lane >> 4) * 16;
    const char *b = p.b + int64_t(jr < p.N ? jr : p.N - 1) * p.ldb + o;
    const char *a[MT];
    const float *sa[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        const int i = min(m * 16 + (lane & 15), p.M - 1);
        a[m] = p.a + int64_t(i) * p.lda + o;
        sa[m] = p.sa + (i >> p.a_shift);
    }
    const float *sb[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) sb[r] = p.sb + (min(j0 + (lane >> 4) * 4 + r, p.N - 1) >> p.b_shift);
    const int k0 = p.steps * wave / 8, k1 = p.steps * (wave + 1) / 8;
    f4 acc[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[m] = f4{0.f, 0.f, 0.f, 0.f};
    constexpr int U = MT == 1 ? 4 : MT == 2 ? 2 : 1;   // blocks whose loads are under way together
    for (int k = k0; k < k1; k += U) {
        nt::i4v qb[U][2], qa[U][MT][2];
        float sj[U][4], si[U][MT];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t kb = k + u < k1 ? k + u : k1 - 1;
#pragma unroll
            for (int h = 0; h < 2; ++h) qb[u][h] = *reinterpret_cast<const nt::i4v *>(b + kb * 128 + h * 64);
#pragma unroll
            for (int r = 0; r < (COMMON ? 1 : 4); ++r) sj[u][r] = sb[r][kb * p.sb_step];
#pragma unroll
            for (int m = 0; m < MT; ++m) {
#pragma unroll
                for (int h = 0; h < 2; ++h) qa[u][m][h] = *reinterpret_cast<const nt::i4v *>(a[m] + kb * 128 + h * 64);
                si[u][m] = sa[m][kb * p.sa_step];
            }
        }
        NT_STAY();
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (k + u >= k1) break;
            nt::Frag8<FB, WIDE> fb;
            fb.set(qb[u][0], qb[u][1]);
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                nt::Frag8<FA, WIDE> fa;
                fa.set(qa[u][m][0], qa[u][m][1]);
                const f4 t = nt::block_product<FA, FB, WIDE>(fa, fb);
#pragma unroll
                for (int r = 0; r < 4; ++r) acc[m][r] = fmaf(t[r] * si[u][m], sj[u][COMMON ? 0 : r], acc[m][r]);
            }
        }
    }
#pragma unroll
    for (int m = 0; m < MT; ++m) *reinterpret_cast<f4 *>(sum[wave][m][lane]) = acc[m];
    __syncthreads();
    for (int u = tid; u < MT * 64; u += 512) {
        const int m = u >> 6, l = u & 63, i = m * 16 + (l & 15), j = j0 + (l >> 4) * 4;
        f4 v = *reinterpret_cast<const f4 *>(sum[0][m][l]);
        for (int w = 1; w < 8; ++w) v += *reinterpret_cast<const f4 *>(sum[w][m][l]);
        if (i >= p.M) continue;
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (p.bias && j + r < p.N) v[r] += p.bias[j + r];
        if (j + 4 <= p.N) store4(p, i, j, v);
        else
            for (int r = 0; r < 4; ++r)
                if (j + r < p.N) store1(p, i, j + r, v[r]);
    }
}

bool wide_form(int c_dtype) { return c_dtype != CP_BF16; }   // what the 8-bit matrix instructions drop is below bfloat16's rounding only

int check_product(cp_ctx *ctx, const cp_blocks *A, const cp_blocks *B, int c_dtype, int64_t ldc) {
    CP_TRY(check_blocks(ctx, A, "A"));
    CP_TRY(check_blocks(ctx, B, "B"));
    if (A->cols != B->cols)
        return cp_set_error(ctx, CP_ERR_ARG, "A has %lld columns, B %lld", (long long)A->cols, (long long)B->cols);
    if (c_dtype != CP_F32 && c_dtype != CP_BF16 && c_dtype != CP_F16) return cp_set_error(ctx, CP_ERR_ARG, "c_dtype %d", c_dtype);
    if (ldc < B->rows) return cp_set_error(ctx, CP_ERR_ARG, "ldc %lld < %lld", (long long)ldc, (long long)B->rows);
    const bool wide = wide_form(c_dtype);
    const int64_t edge = wide ? nt::Medium::BM : nt::Large::BM;
    if (((A->rows + edge - 1) / edge) * ((B->rows + edge - 1) / edge) * (wide ? nt::Medium::T : nt::Large::T) > kMaxThreads)
        return cp_set_error(ctx, CP_ERR_UNSUPPORTED, "C is too large");
    return CP_OK;
}

// How a product is formed: by its shape, its types and C's type alone
struct Form {
    int cfg;             // 0 Large, 1 Medium, 2 Small, 3 Flat, 4 few rows
    int tiles_m, tiles_n, pieces;
    size_t counts, parts;   // bytes
};
constexpr int kMaxJoined = 16384;   // workgroups of a launch that joins pieces
constexpr int kRowGroups = 8;        // of sixteen rows of A, for k_matmul_blocks_rows
constexpr int kChip = 256;          // CUs that a split is planned for

Form form_of(const cp_blocks *A, const cp_blocks *B, int c_dtype) {
    // us per step and workgroup on a full chip / with at most one to a CU, beside the steps, for a join and for every piece that it
    // adds; [wide][cfg].  Fitted to 172 shapes (33..20000 x 64..8192 x 128..16384): off by 4 to 9 % (root mean square), and the
    // rule's choice takes 1.01 of the time of the best shape of tile.
    static const double full[2][4] = {{1.67, 1.04, 0.38, 1.24}, {0, 1.82, 0.69, 0}}, alone[2][4] = {{1.31, 0.68, 0.265, 1.14}, {0, 1.2, 0.51, 0}};
    static const double extra[4] = {6.3, 4.5, 2.2, 6.2}, joined[4] = {16.0, 7.0, 1.2, 15.0}, piece[4] = {1.7, 0.5, 0.5, 1.35};
    static const int rows_of[4] = {nt::Large::BM, nt::Medium::BM, nt::Small::BM, nt::Flat::BM};
    static const int cols_of[4] = {nt::Large::BN, nt::Medium::BN, nt::Small::BN, nt::Flat::BN};
    const int64_t steps = (A->cols + 127) / 128;
    const bool wide = wide_form(c_dtype);
    Form best = {};
    const bool few = A->rows <= 16 * kRowGroups && B->rows <= kMaxThreads / 512 * 16;
    int forced = cp_knob(CP_KNOB_NT_TILE);
    if (forced == 5 && !few) forced = 0;
    double least = 1e300;
    if (few && (!forced || forced == 5)) {
        // sixteen rows of B to a workgroup: rounds of 256, each a part of a us per step.  us for 16, 32, 64, 80, 96, 128 rows, against
        // 64 x 64 tiles:  4096 x 512 bfloat16 4.3 4.2 4.7 4.3 4.4 5.0, 4.5-4.6;  1000 x 2048 float32 5.6 5.0 7.1 8.0 9.1 11.0, 8.5-9.6;
        // 4096 x 2048 float32 5.7 5.2 7.2 8.3 9.3 11.3, 10.5-13.1;  bfloat16 5.2 5.0 7.0 8.1 9.1 11.1, 7.6-8.0;
        // 4096 x 8192 bfloat16 9.7 13 21 24 28 35, 11-15.  Over 576 shapes the choice takes 1.01 of the better form's time.
        best = {4, 0, 0, 1, 0, 0};
        least = double((B->rows + 4095) / 4096) * steps * (0.07 + 0.0032 * A->rows) + 1.0;
        // (no tile costs less than a 64 x 64 one in one piece, or in pieces of four steps)
        const double one = std::min(steps * alone[wide][2], 4 * alone[wide][2] + joined[2] + 2 * piece[2]);
        if (forced || least <= extra[2] + one) return best;
    }
    for (int cfg = 0; cfg < 4; ++cfg) {
        const bool alone_on_cu = cfg == 0 || cfg == 3;
        if (wide && alone_on_cu) continue;
        if (forced && forced - 1 != cfg && !(wide && cfg == 1 && (forced == 1 || forced == 4))) continue;
        const int64_t tm = (A->rows + rows_of[cfg] - 1) / rows_of[cfg], tn = (B->rows + cols_of[cfg] - 1) / cols_of[cfg];
        if (tm * tn * (alone_on_cu ? nt::Large::T : nt::Medium::T) > kMaxThreads) continue;   // (the largest tile's count is checked)
        for (int p = 1; p <= 32 && (p == 1 || (steps / p >= 4 && tm * tn * p <= kMaxJoined)); ++p) {
            const int64_t groups = tm * tn * p, slots = alone_on_cu ? kChip : 2 * kChip, rest = groups % slots;
            const double beside = extra[cfg] + (p > 1 ? joined[cfg] + p * piece[cfg] : 0.0);
            const double most = (steps + p - 1) / p * full[wide][cfg] + beside, least_of = (steps + p - 1) / p * alone[wide][cfg] + beside;
            const double cost = double(groups / slots) * most + (rest > slots / 2 ? most : rest ? least_of : 0.0);
            if (cost < 0.97 * least) {
                least = cost;
                best = {cfg, int(tm), int(tn), p, 0, 0};
                if (p > 1) {
                    best.counts = cp_align_up(size_t(tm * tn) * sizeof(int), 256);
                    best.parts = size_t(tm * tn * p) * rows_of[cfg] * cols_of[cfg] * sizeof(float);
                }
            }
        }
    }
    return best;
}

__global__ void __launch_bounds__(256) k_zero(int *p, int n) {
    for (int i = blockIdx.x * 256 + threadIdx.x; i < n; i += gridDim.x * 256) p[i] = 0;
}

// the least number of row groups that holds A
template <int MT, int FA, int FB, bool COMMON, bool WIDE>
void launch_rows(cp_ctx *ctx, const Product &p) {
    if constexpr (MT > 1)
        if (p.M <= 16 * (MT - 1)) return launch_rows<MT - 1, FA, FB, COMMON, WIDE>(ctx, p);
    k_matmul_blocks_rows<MT, FA, FB, COMMON, WIDE><<<(p.N + 15) / 16, 512, 0, ctx->stream>>>(p);
}

template <int FA, int FB, bool COMMON, bool WIDE>
void launch_product(cp_ctx *ctx, const Product &p, const Form &f) {
    const int n = f.tiles_m * f.tiles_n * f.pieces;
    if (f.cfg == 4) {
        return launch_rows<kRowGroups, FA, FB, COMMON, WIDE>(ctx, p);
    }
    if constexpr (!WIDE) {   // the widened fragments of 256 x 256 do not fit into registers
        if (f.cfg == 0) return (void)(k_matmul_blocks<nt::Large, FA, FB, COMMON, WIDE><<<n, nt::Large::T, 0, ctx->stream>>>(p));
        if (f.cfg == 3) return (void)(k_matmul_blocks<nt::Flat, FA, FB, COMMON, WIDE><<<n, nt::Flat::T, 0, ctx->stream>>>(p));
    }
    if (f.cfg <= 1) k_matmul_blocks<nt::Medium, FA, FB, COMMON, WIDE><<<n, nt::Medium::T, 0, ctx->stream>>>(p);
    else k_matmul_blocks<nt::Small, FA, FB, COMMON, WIDE><<<n, nt::Small::T, 0, ctx->stream>>>(p);
}

template <int FA, int FB>
void launch_product(cp_ctx *ctx, const Product &p, const Form &f) {
    const bool wide = wide_form(p.c_dtype);
    if (p.b_shift) wide ? launch_product<FA, FB, true, true>(ctx, p, f) : launch_product<FA, FB, true, false>(ctx, p, f);
    else wide ? launch_product<FA, FB, false, true>(ctx, p, f) : launch_product<FA, FB, false, false>(ctx, p, f);
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
    if (out && out_t && out->q == out_t->q && out->q && rows && cols) return cp_set_error(ctx, CP_ERR_ARG, "out and out_t are the same memory");
    if (!rows || !cols) return CP_OK;
    const size_t size = x_dtype == CP_F64 ? 8 : x_dtype == CP_F32 ? 4 : 2;
    if (!x || uintptr_t(x) % size) return cp_set_error(ctx, CP_ERR_ARG, "x is null or misaligned");
    if (((rows + 127) / 128) * ((cols + 127) / 128) * 256 > kMaxThreads) return cp_set_error(ctx, CP_ERR_UNSUPPORTED, "x is too large");
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
    const Form f = form_of(A, B, c_dtype);
    *bytes = f.counts + f.parts;
    return CP_OK;
}

extern "C" int cp_matmul_blocks(cp_ctx *ctx, const cp_blocks *A, const cp_blocks *B, const float *bias, void *C, int c_dtype,
                                int64_t ldc, void *ws, size_t ws_bytes) {
    if (!ctx) return CP_ERR_ARG;
    CP_TRY(check_product(ctx, A, B, c_dtype, ldc));
    if (!A->rows || !B->rows) return CP_OK;
    const size_t size = c_dtype == CP_F32 ? 4 : 2;
    if (!C || uintptr_t(C) % size || uintptr_t(bias) % 4) return cp_set_error(ctx, CP_ERR_ARG, "C is null or misaligned");
    CP_HIP(ctx, hipSetDevice(ctx->device));
    const Form f = form_of(A, B, c_dtype);
    char *scratch = nullptr;
    if (f.pieces > 1) {
        CP_TRY(cp_scratch(ctx, ws, ws_bytes, f.counts + f.parts, &scratch));
        if (!ws && !ctx->nt_cnt) {   // the context's own counters are zero between launches
            int *c = nullptr;
            CP_HIP(ctx, hipMalloc(reinterpret_cast<void **>(&c), kMaxJoined * sizeof(int)));
            k_zero<<<16, 256, 0, ctx->stream>>>(c, kMaxJoined);
            ctx->nt_cnt = c;
        }
        if (ws) k_zero<<<1, 256, 0, ctx->stream>>>(reinterpret_cast<int *>(scratch), f.tiles_m * f.tiles_n);
    }
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
    p.tiles_m = f.tiles_m;
    p.tiles_n = f.tiles_n;
    p.pieces = f.pieces;
    p.counts = ws ? reinterpret_cast<int *>(scratch) : ctx->nt_cnt;
    p.parts = reinterpret_cast<float *>(scratch + f.counts);
    p.a_shift = A->tile == 1 ? 0 : 7;
    p.b_shift = B->tile == 1 ? 0 : 7;
    p.c_dtype = c_dtype;
    const bool a5 = A->fmt == CP_E5M2, b5 = B->fmt == CP_E5M2;
    if (a5 && b5) launch_product<1, 1>(ctx, p, f);
    else if (a5) launch_product<1, 0>(ctx, p, f);
    else if (b5) launch_product<0, 1>(ctx, p, f);
    else launch_product<0, 0>(ctx, p, f);
    CP_LAUNCH_CHECK(ctx);
    return CP_OK;
}
