// Orthogonalised updates: Newton-Schulz products on a set of matrices, and the optimiser step around them.
//
// X = U / (|U|_F + eps) lies with its short side m first (a tall matrix is taken transposed).  Every step is three products
//     A = X X^T,   B = a I + b A + c A A,   X <- B X
// the first two symmetric: only the tiles on and below the diagonal are computed, and mirrored.
//
// Numbers.  Singular values stay in [0, u_k] with bounds u_k that the host derives from the coefficients, so every entry of X,
// A and B is bounded too, and a power of two per step and matrix puts that bound at 2^14: fp16's whole range is used, with
// headroom of four.  Numbers are carried as pairs of fp16 (22 bits) and three products instead of one; the pair's dropped
// low * low term is below its rounding.  Only where G and the result are both bf16 they are one fp16 each (11 bits, where bf16
// would hold 8, at the same rate): a step amplifies what is lost in a small singular direction up to 3.44 times, so that the
// 11 bits cost 0.5, 4 and 7 % of O where a rank-4 part is 10, 100 and 1000 times as strong as the rest (256 x 576) -- an eighth of
// what G's own rounding to bf16 has cost there (3, 26 and 46 %).  float32, fp16 and the step's momentum have not lost that: they
// get pairs (3e-5 in the worst of these), whatever the result's type.
// Sums are float32 in the accumulators, |U|_F is summed in float64.
#include <algorithm>
#include <cfloat>
#include <cmath>

#include "cp_common.h"
#include "nt_mfma.h"

namespace {

using nt::f4;
using nt::h4;
using nt::h8;
using nt::put_to;
using nt::take_from;

constexpr int kJobs = 20;        // jobs whose records one launch carries in its arguments (4 KB)
constexpr int kMaxSteps = 32;
constexpr int kCus = 256;        // the chip's CUs: what the split of a launch is planned for (results do not depend on the real number)
constexpr int kPartials = 512;   // partial sums of |U|_F^2 per job, at most
constexpr int kPad = 64;         // both sides are padded to this (and the tiles' loads repeat the last row beyond it)
constexpr double kDefault[3] = {3.4445, -4.7750, 2.0315};

struct Job {
    const void *G;
    float *M;                    // momentum (cp_ortho_step), else null
    void *out;                   // O, or W
    char *x, *xt0, *xt1, *a, *b; // X [mp][np], X^T [np][mp] twice, A and B [mp][mp]
    double *part;
    int64_t ldg, ldm, ldo;
    int64_t sum_cols;            // |U|: a row's length, the whole matrix' where it is contiguous
    uint32_t ldn, lds;           // bytes of a row of np / of mp numbers
    int rows, cols, mp, np;
    int sum_rows, rows_per, width, chunks;   // |U|: rows, and rows, columns that a workgroup sums, chunks of columns
    int16_t g_dtype, o_dtype;
    float lr;                    // lr * gamma
};

// The phases' launches: job k's first workgroup of each, and how the products' tiles are shared: the pieces of k that they are cut
// into (at most 16, in the low bits) and, where there are several, the job's first slot among the launch's partial sums and counters
// (LAST: the last step's third product, which writes O or W)
enum { LOAD, GRAM, POLY, APPLY, LAST, PHASES };
constexpr int kShareBits = 5;
struct Place {
    int first[PHASES];
    int share[PHASES - 1];
    int pieces(int phase) const { return share[phase - 1] & ((1 << kShareBits) - 1); }
};

// A call's jobs in its workspace.  The first kernel carries them in its arguments and writes them there.
struct Table {
    Job *job;
    int *first[PHASES];
    int *share[PHASES - 1];
    int n;
};

struct Jobs {
    int n, base;                 // job[0] is the call's job `base`
    int first[kJobs];            // this job's first workgroup of the launch
    Place place[kJobs];
    Job job[kJobs];
};
static_assert(sizeof(Jobs) <= 3900, "kernel arguments");

// the job whose workgroups include `at`; every wave looks for itself
__device__ __forceinline__ int find_job(const int *first, int n, int at) {
    int k = 0;
    for (int i = threadIdx.x & 63; i - int(threadIdx.x & 63) < n; i += 64) k += __popcll(__ballot(i < n && first[i] <= at));
    return __builtin_amdgcn_readfirstlane(k - 1);
}

__device__ __forceinline__ float load_as_float(const void *p, int dtype, int64_t at) {
    if (dtype == CP_F32) return take_from<float>(static_cast<const float *>(p) + at);
    if (dtype == CP_BF16) return float(take_from<__bf16>(static_cast<const __bf16 *>(p) + at));
    return float(take_from<_Float16>(static_cast<const _Float16 *>(p) + at));
}
__device__ __forceinline__ void store_as(void *p, int dtype, int64_t at, float v) {
    if (dtype == CP_F32) put_to(static_cast<float *>(p) + at, v);
    else if (dtype == CP_BF16) put_to(static_cast<__bf16 *>(p) + at, __bf16(v));
    else put_to(static_cast<_Float16 *>(p) + at, _Float16(v));
}
__device__ __forceinline__ f4 load4_as_float(const void *p, int dtype, int64_t at) {
    if (dtype == CP_F32) return take_from<nt::f4u>(static_cast<const float *>(p) + at);
    if (dtype == CP_BF16) return __builtin_convertvector(take_from<nt::b4u>(static_cast<const __bf16 *>(p) + at), f4);
    return __builtin_convertvector(take_from<nt::h4u>(static_cast<const _Float16 *>(p) + at), f4);
}
__device__ __forceinline__ void store4_as(void *p, int dtype, int64_t at, f4 v) {
    if (dtype == CP_F32) put_to<nt::f4u>(static_cast<float *>(p) + at, v);
    else if (dtype == CP_BF16) put_to<nt::b4u>(static_cast<__bf16 *>(p) + at, __builtin_convertvector(v, nt::b4));
    else put_to<nt::h4u>(static_cast<_Float16 *>(p) + at, __builtin_convertvector(v, h4));
}

// eight numbers of a row from column c, zero from `cols` on
__device__ __forceinline__ void load8(const void *row, int dtype, int c, int cols, float (&v)[8]) {
    if (c + 8 <= cols) {
        if (dtype == CP_F32) {
            const float *p = static_cast<const float *>(row) + c;
            const f4 a = take_from<nt::f4u>(p), b = take_from<nt::f4u>(p + 4);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = a[e], v[e + 4] = b[e];
        } else if (dtype == CP_BF16) {
            const nt::b8 a = take_from<nt::b8u>(static_cast<const __bf16 *>(row) + c);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = float(a[e]);
        } else {
            const h8 a = take_from<nt::h8u>(static_cast<const _Float16 *>(row) + c);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = float(a[e]);
        }
        return;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = c + e < cols ? load_as_float(row, dtype, c + e) : 0.f;
}

// eight numbers of a row from column c, those before `cols`
__device__ __forceinline__ void store8(void *row, int dtype, int c, int cols, const float (&v)[8]) {
    if (c + 8 <= cols) {
        store4_as(row, dtype, c, f4{v[0], v[1], v[2], v[3]});
        store4_as(row, dtype, c + 4, f4{v[4], v[5], v[6], v[7]});
        return;
    }
#pragma unroll
    for (int e = 0; e < 7; ++e)
        if (c + e < cols) store_as(row, dtype, c + e, v[e]);
}

__device__ __forceinline__ const void *row_of(const void *p, int dtype, int64_t at) {
    return static_cast<const char *>(p) + at * (dtype == CP_F32 ? 4 : 2);
}

// One number for all of its uses.  The compiler may fuse a product with its rounding to fp16, but not with the difference from
// that rounding: the halves of a pair would belong to different numbers.
__device__ __forceinline__ float settled(float v) {
    asm("" : "+v"(v));
    return v;
}
__device__ __forceinline__ f4 settled(f4 v) { return f4{settled(v[0]), settled(v[1]), settled(v[2]), settled(v[3])}; }

__device__ __forceinline__ double wave_sum(double v) {
    for (int s = 32; s; s >>= 1) v += __shfl_xor(v, s);
    return v;
}

// scale / (|U|_F + eps), which may lie outside float32 where its products with U do not: as a mantissa and an exponent
struct Inverse {
    float mantissa;
    int exponent;
    __device__ __forceinline__ Inverse(double sum, double eps, double scale) {
        const double norm = sqrt(sum) + eps, inv = norm > 0.0 || norm != norm ? scale / norm : 0.0;
        mantissa = float(__builtin_amdgcn_frexp_mant(inv));
        exponent = __builtin_amdgcn_frexp_exp(inv);
    }
    __device__ __forceinline__ float times(float v) const {
        return settled(ldexpf(v, exponent) * mantissa);
    }
};

// ---- |U|_F, and the momentum: one pass over G (and M), bound by HBM -----------------------------------------------------------
// (12.8 M numbers, G and M float32: 28.5 us for 153 MB, 5.4 TB/s, and 29.5 on six sets of layers in turn, 5.2; adding two large
// matrices reaches 5.7.  67 M in bfloat16: 39 us for 134 MB; reading alone, a large maximum takes 3.7 TB/s.)
// A workgroup sums rows_per rows of a chunk of `width` columns; the partial sums are added in one order by whoever needs the
// norm.  Contiguous matrices are one row: their own rows' lengths would leave most of them unaligned.
__global__ void __launch_bounds__(256) k_ortho_norm(Jobs js, Table t, float momentum, int nesterov, int *counts, int n_counts) {
    int which = 0;
#pragma unroll
    for (int i = 1; i < kJobs; ++i) which += i < js.n && js.first[i] <= int(blockIdx.x);
    const Job &j = js.job[which];
    const int id = blockIdx.x - js.first[which];
    if (id == 0) {   // this job's record, for the kernels that follow
        const int *from = reinterpret_cast<const int *>(&j);
        int *to = reinterpret_cast<int *>(t.job + js.base + which);
        for (int i = threadIdx.x; i < int(sizeof(Job) / 4); i += 256) to[i] = from[i];
        if (threadIdx.x < PHASES) t.first[threadIdx.x][js.base + which] = js.place[which].first[threadIdx.x];
        if (threadIdx.x < PHASES - 1) t.share[threadIdx.x][js.base + which] = js.place[which].share[threadIdx.x];
    }
    for (int i = blockIdx.x * 256 + threadIdx.x; i < n_counts; i += gridDim.x * 256) counts[i] = 0;
    const int r0 = id / j.chunks * j.rows_per, rows = min(r0 + j.rows_per, j.sum_rows) - r0;
    const int64_t c0 = int64_t(id % j.chunks) * j.width;
    const int wide = int(min(j.sum_cols - c0, int64_t(j.width))), eights = wide / 8, tail = wide & 7, n = rows * eights;
    double sum = 0.0;
    auto momentum_of = [&](float &m, float &v) {
        m = fmaf(momentum, m, v);
        v = nesterov ? fmaf(momentum, m, v) : m;
    };
    // whole groups of eight, AT_ONCE loads of a thread under way together (beyond the end the last group's again, for nothing)
    auto groups = [&](auto type) {
        typedef decltype(type) V;   // eight numbers, at any element's address
        constexpr int AT_ONCE = 4, SIZE = int(sizeof(V) / 8);
        for (int u0 = threadIdx.x; u0 < n; u0 += 256 * AT_ONCE) {
            int64_t r[AT_ONCE];
            int c[AT_ONCE];
            V v[AT_ONCE];
            f4 m[AT_ONCE][2];
#pragma unroll
            for (int q = 0; q < AT_ONCE; ++q) {
                const int u = min(u0 + q * 256, n - 1), k = rows > 1 ? u / eights : 0;
                r[q] = r0 + k;
                c[q] = (u - k * eights) * 8;
                v[q] = take_from<V>(static_cast<const char *>(j.G) + (r[q] * j.ldg + c0 + c[q]) * SIZE);
            }
            if (j.M) {
#pragma unroll
                for (int q = 0; q < AT_ONCE; ++q)
#pragma unroll
                    for (int h = 0; h < 2; ++h) m[q][h] = take_from<nt::f4u>(j.M + r[q] * j.ldm + c0 + c[q] + 4 * h);
            }
#pragma unroll
            for (int q = 0; q < AT_ONCE; ++q) {
                if (u0 + q * 256 >= n) break;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    float x = float(v[q][e]);
                    if (j.M) {
                        float y = m[q][e >> 2][e & 3];
                        momentum_of(y, x);
                        m[q][e >> 2][e & 3] = y;
                    }
                    sum = fma(double(x), double(x), sum);
                }
                if (j.M) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) put_to<nt::f4u>(j.M + r[q] * j.ldm + c0 + c[q] + 4 * h, m[q][h]);
                }
            }
        }
    };
    typedef float f8u __attribute__((ext_vector_type(8), aligned(4)));
    if (j.g_dtype == CP_F32) groups(f8u());
    else if (j.g_dtype == CP_BF16) groups(nt::b8u());
    else groups(nt::h8u());
    for (int u = threadIdx.x; u < rows * tail; u += 256) {   // the rows' ends
        const int64_t r = r0 + u / tail, c = c0 + eights * 8 + u % tail;
        float x = load_as_float(j.G, j.g_dtype, r * j.ldg + c);
        if (j.M) {
            float y = load_as_float(j.M, CP_F32, r * j.ldm + c);
            momentum_of(y, x);
            store_as(j.M, CP_F32, r * j.ldm + c, y);
        }
        sum = fma(double(x), double(x), sum);
    }
    __shared__ double s[4];
    sum = wave_sum(sum);
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = sum;
    __syncthreads();
    if (threadIdx.x == 0) j.part[id] = (s[0] + s[1]) + (s[2] + s[3]);
}

// eight numbers of a row, from column k (a multiple of 8), as fp16 or as pairs
template <bool SPLIT>
__device__ __forceinline__ void store8(char *row, int k, const float *v) {
    char *p = row + (SPLIT ? (k >> 5) * 128 + (k & 31) * 2 : k * 2);
    h8 hi, lo;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float x = SPLIT ? settled(v[e]) : v[e];
        hi[e] = _Float16(x);
        lo[e] = _Float16(x - float(hi[e]));
    }
    put_to(p, hi);
    if (SPLIT) put_to(p + 64, lo);
}
template <bool SPLIT>
__device__ __forceinline__ void load8(const char *row, int k, float (&v)[8]) {
    const char *p = row + (SPLIT ? (k >> 5) * 128 + (k & 31) * 2 : k * 2);
    const h8 hi = take_from<h8>(p);
    h8 lo = {};
    if (SPLIT) lo = take_from<h8>(p + 64);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = SPLIT ? float(hi[e]) + float(lo[e]) : float(hi[e]);
}

// ---- X = U / (|U|_F + eps) in both orientations, zero in the padding: one 64 x 64 tile of G to a workgroup --------------------
// Bound by HBM: 4096 x 16384 in bfloat16 90 us for 403 MB, 12.8 M numbers in float32 40 us for 204 MB.
// sixteen numbers of a tile's row
__device__ __forceinline__ void load_tile(const void *p, int dtype, int64_t ld, const Job &j, int r, int c, float (&v)[16]) {
    float a[8] = {}, b[8] = {};
    if (r < j.rows) {
        load8(row_of(p, dtype, r * ld), dtype, c, j.cols, a);
        load8(row_of(p, dtype, r * ld), dtype, c + 8, j.cols, b);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = a[e], v[e + 8] = b[e];
}

template <bool SPLIT>
__global__ void __launch_bounds__(256) k_ortho_load(Table tab, float momentum, int nesterov, double eps, float x_scale) {
    const int at = nt::xcd_runs(blockIdx.x, gridDim.x), which = find_job(tab.first[LOAD], tab.n, at);
    const Job j = tab.job[which];
    const bool tall = j.rows > j.cols;
    const int id = at - tab.first[LOAD][which], tiles_c = (tall ? j.mp : j.np) / 64;
    const int r0 = id / tiles_c * 64, c0 = id % tiles_c * 64;
    __shared__ double s[4];
    __shared__ float t[64][65];
    const int tid = threadIdx.x, line = tid >> 2, k = (tid & 3) * 16;
    float v[16];
    if (j.M) {
        load_tile(j.M, CP_F32, j.ldm, j, r0 + line, c0 + k, v);
        if (nesterov) {
            float u[16];
            load_tile(j.G, j.g_dtype, j.ldg, j, r0 + line, c0 + k, u);
#pragma unroll
            for (int e = 0; e < 16; ++e) v[e] = fmaf(momentum, v[e], u[e]);
        }
    } else {
        load_tile(j.G, j.g_dtype, j.ldg, j, r0 + line, c0 + k, v);
    }
    const int n_part = (j.sum_rows + j.rows_per - 1) / j.rows_per * j.chunks;
    double part = 0.0;
    for (int i = tid; i < n_part; i += 256) part += take_from<double>(j.part + i);
    part = wave_sum(part);
    if ((tid & 63) == 0) s[tid >> 6] = part;
    __syncthreads();
    const Inverse inv((s[0] + s[1]) + (s[2] + s[3]), eps, x_scale);
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        v[e] = inv.times(v[e]);
        t[line][k + e] = v[e];
    }
    char *n = tall ? j.xt0 : j.x, *o = tall ? j.x : j.xt0;
    const uint32_t ldn = tall ? j.lds : j.ldn, ldo = tall ? j.ldn : j.lds;
    store8<SPLIT>(n + int64_t(r0 + line) * ldn, c0 + k, v);
    store8<SPLIT>(n + int64_t(r0 + line) * ldn, c0 + k + 8, v + 8);
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 16; ++e) v[e] = t[k + e][line];
    store8<SPLIT>(o + int64_t(c0 + line) * ldo, r0 + k, v);
    store8<SPLIT>(o + int64_t(c0 + line) * ldo, r0 + k + 8, v + 8);
}

// ---- the products ------------------------------------------------------------------------------------------------------------
// All jobs' tiles of one of a step's three products in one launch.  Bound by the matrix instructions where matrices are large (4096 x
// 16384 in fp16: first product 305 us, 0.90 PFLOP/s of the half that is formed -- 136 tiles of 256 x 256 divide badly over 256
// CUs --, second 110, third 480, 1.15 PFLOP/s), by a launch's fixed costs where they are many and small (the 40 layers of a
// pruned resnet50, 8.5 M numbers in pairs: 25, 13 and 41 us).
struct Factors {
    float acc, a, diag;   // what the accumulator, A's entry and the diagonal count for in the result
    float keep;           // LAST: 1 - lr * weight_decay (cp_ortho_step)
    int xt;               // which X^T is read
};

template <int PHASE, bool SPLIT, class CFG>
__global__ void __launch_bounds__(CFG::T) k_ortho_product(Table tab, Factors f, float *parts, int *counts) {
    constexpr int BM = CFG::BM, BN = CFG::BN, T = CFG::T, WI = CFG::WI, WJ = CFG::WJ;
    constexpr bool SYM = PHASE == GRAM || PHASE == POLY;
    NT_STAGES(st, CFG::STAGES, CFG::STAGE);
    __shared__ int flag;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave / CFG::NWN, wn = wave % CFG::NWN;
    const int ra = wm * WI * 16, rb = wn * WJ * 16;
    const int at = nt::xcd_order(blockIdx.x, gridDim.x), which = find_job(tab.first[PHASE], tab.n, at);
    const Job j = tab.job[which];
    const int first = tab.first[PHASE][which], share = tab.share[PHASE - 1][which];
    const int pieces = share & ((1 << kShareBits) - 1), slot = share >> kShareBits;
    const bool tall = j.rows > j.cols;
    const bool swap = PHASE == LAST && tall;   // the result's rows are G's rows: four consecutive numbers lie in one of them
    const char *xt = f.xt ? j.xt1 : j.xt0;
    const char *pa = PHASE == GRAM ? j.x : PHASE == POLY ? j.a : swap ? xt : j.b;
    const char *pb = PHASE == GRAM ? j.x : PHASE == POLY ? j.a : swap ? j.b : xt;
    const uint32_t ld = PHASE == GRAM ? j.ldn : j.lds;
    const int rows_a = swap ? j.np : j.mp, rows_b = SYM || swap ? j.mp : j.np;
    const int tiles_m = (rows_a + BM - 1) / BM, tiles_n = (rows_b + BN - 1) / BN;
    const int tiles = SYM ? tiles_m * (tiles_m + 1) / 2 : tiles_m * tiles_n;
    const int piece = (at - first) / tiles, tile = (at - first) % tiles;
    const int steps = int(ld >> 7), k0 = steps * piece / pieces, k1 = steps * (piece + 1) / pieces;
    int tm, tn;
    if (SYM) nt::lower_tile_at(tile, tiles_m, tm, tn);
    else nt::tile_at(tile, tiles_m, tiles_n, tm, tn);
    const int i0 = tm * BM, j0 = tn * BN;
    nt::Loader<BM, T> la;
    nt::Loader<BN, T> lb;
    la.init(pa + int64_t(i0) * ld + k0 * 128, ld, rows_a - i0, tid);
    lb.init(pb + int64_t(j0) * ld + k0 * 128, ld, rows_b - j0, tid);
    f4 acc[WI][WJ];
#pragma unroll
    for (int i = 0; i < WI; ++i)
#pragma unroll
        for (int k = 0; k < WJ; ++k) acc[i][k] = f4{0.f, 0.f, 0.f, 0.f};
    nt::pipeline<CFG::STAGES, CFG::LOADS, CFG::PARTS>(
        st, k1 - k0,
        [&](int k, char *s, int part, int parts) {
            la.issue(k, s, wave, part, parts);
            lb.issue(k, s + BM * 128, wave, part, parts);
        },
        [&](const char *s, auto between) {
            nt::products16<WI, WJ, SPLIT>(s + ra * 128, s + (BM + rb) * 128, lane, acc, between);
        });
    if (pieces > 1 && !nt::join<T>(acc, piece, pieces, parts + int64_t(slot + tile) * (BM * BN), tiles, counts + slot + tile, &flag, tid))
        return;
    typedef nt::Patch<WI, WJ> Patch;
    const Patch patch = Patch::template of<CFG>(st, wave, lane);
#pragma unroll
    for (int pass = 0; pass < Patch::PASSES; ++pass) {
        const int ip = i0 + ra + pass * Patch::ROWS, jp = j0 + rb;
        // what lies beyond the padding is not there (both sides are multiples of 64: a pass is all in or all out)
        if (ip >= rows_a || jp >= rows_b) break;
        patch.put(acc, pass, f.acc);
        auto finish = [&](int i, int c, float (&v)[8]) {   // eight neighbours of row i, or, as B is symmetric, of column i
            if (PHASE != POLY) return;
            float a[8];
            load8<SPLIT>(j.a + int64_t(i) * j.lds, c, a);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                v[e] = fmaf(a[e], f.a, v[e]);
                if (c + e == i) v[e] += f.diag;
            }
        };
        constexpr int AT_ONCE = Patch::PASSES == 1 ? 8 : 4;
        if (PHASE == LAST && SPLIT && j.o_dtype == CP_F32) {
#pragma unroll AT_ONCE
            for (int u = 0; u < 2 * Patch::EIGHTS; ++u) {
                int i, c;
                f4 v = patch.four_of_row(u, i, c);
                i += ip;
                c += jp;
                if (i >= j.rows || c >= j.cols) continue;
                const int64_t o = i * j.ldo + c;
                if (c + 4 <= j.cols) {
                    if (j.M) v = load4_as_float(j.out, CP_F32, o) * f.keep - v * j.lr;
                    store4_as(j.out, CP_F32, o, v);
                } else {
#pragma unroll
                    for (int r = 0; r < 3; ++r) {
                        if (c + r >= j.cols) break;
                        float y = v[r];
                        if (j.M) y = f.keep * load_as_float(j.out, CP_F32, o + r) - j.lr * y;
                        store_as(j.out, CP_F32, o + r, y);
                    }
                }
            }
            continue;
        }
#pragma unroll AT_ONCE
        for (int u = 0; u < Patch::EIGHTS; ++u) {
            int i, c;
            float v[8];
            patch.of_row(u, i, c, v);
            i += ip;
            c += jp;
            finish(i, c, v);
            if (PHASE != LAST) {
                char *out = PHASE == GRAM ? j.a : PHASE == POLY ? j.b : j.x;
                store8<SPLIT>(out + int64_t(i) * (SYM ? j.lds : j.ldn), c, v);
            } else if (i < j.rows && c < j.cols) {
                void *row = const_cast<void *>(row_of(j.out, j.o_dtype, i * j.ldo));
                if (j.M) {
                    float w[8];
                    load8(row, j.o_dtype, c, j.cols, w);
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] = f.keep * w[e] - j.lr * v[e];
                }
                store8(row, j.o_dtype, c, j.cols, v);
            }
        }
        if (PHASE != LAST && (!SYM || tm != tn)) {
#pragma unroll 4
            for (int u = 0; u < Patch::EIGHTS; ++u) {
                int i, c;
                float v[8];
                patch.of_column(u, i, c, v);
                i += ip;
                c += jp;
                finish(c, i, v);
                char *out_t = PHASE == GRAM ? j.a : PHASE == POLY ? j.b : f.xt ? j.xt0 : j.xt1;
                store8<SPLIT>(out_t + int64_t(c) * j.lds, i, v);
            }
        }
    }
}

// ---- small matrices: the whole step in one workgroup ---------------------------------------------------------------------------
// Where the short side fits 64 rows and the long side the registers of eight waves, seventeen launches of 4.3 us each do 1 us
// of arithmetic.  Here a workgroup keeps X in registers from the first product to the last (64 x 576 in bfloat16: 29 us, of which
// 3.3 a step; 73 with the launches above).  Bound by the latency of a step's chain: a product, a sum over the waves through LDS, a
// product of 64 x 64, a product.
// A wave owns CT tiles of 16 columns, in the two forms that the matrix instruction's operands need: by columns (lane: column
// j, eight rows; K = rows, for B X) and by rows (lane: row i, eight columns; K = columns, for X X^T).  The result of a product
// IS such an operand (lane: column, four consecutive rows; or, with the operands exchanged, row and four columns) once K's
// order within a block of 32 is taken as (4 g .. 4 g + 3, 16 + 4 g .. 16 + 4 g + 3) for lane group g: B X comes out in one form, a
// product with the unit matrix turns it, exactly, into the other, and nothing of X passes through LDS.  Only A and B do.
constexpr int kSmallWaves = 8;
constexpr int kSmallJobs = 24;
constexpr int kSmallTiles[2] = {6, 4};   // column tiles of a wave at most: one fp16 a number, pairs

struct SmallJob {
    const void *G;
    float *M;
    void *out;
    int64_t ldg, ldm, ldo;
    int rows, cols;
    int g_dtype, o_dtype;
    float lr;
};
struct StepFactors {
    float gram, poly, a, diag, apply;   // what a step's accumulators, A's entry and the diagonal count for
};
struct SmallJobs {
    SmallJob job[kSmallJobs];
    StepFactors step[kMaxSteps];
    double eps, x_scale;
    float momentum, keep;
    int nesterov, steps;
};
static_assert(sizeof(SmallJobs) <= 3900, "kernel arguments");

template <bool SPLIT>
struct Op {   // an operand: eight numbers of a lane, as fp16 or as pairs
    h8 v[SPLIT ? 2 : 1];
    __device__ __forceinline__ void set(int half, f4 x) {
        if (SPLIT) x = settled(x);
        const h4 hi = __builtin_convertvector(x, h4);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[0][4 * half + e] = hi[e];
        if constexpr (SPLIT) {
            const h4 lo = __builtin_convertvector(x - __builtin_convertvector(hi, f4), h4);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[1][4 * half + e] = lo[e];
        }
    }
};
template <bool SPLIT>
__device__ __forceinline__ f4 multiply(const Op<SPLIT> &a, const Op<SPLIT> &b, f4 acc) {
    if constexpr (SPLIT) {
        acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(a.v[1], b.v[0], acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(a.v[0], b.v[1], acc, 0, 0, 0);
    }
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a.v[0], b.v[0], acc, 0, 0, 0);
}

template <bool SPLIT, int CT, bool TALL>
__global__ void __launch_bounds__(64 * kSmallWaves) k_ortho_small(SmallJobs js) {
    constexpr int N = SPLIT ? 2 : 1, T = 64 * kSmallWaves, LONG = CT * kSmallWaves * 16;
    constexpr int LD = 72;   // a row of A or B: 64 numbers, and eight that keep rows off one bank
    // LDS: first X as it comes (G's rows); then the waves' shares of A, and A and B; last O's rows, half of the column tiles at a time
    constexpr int R = TALL ? LONG : 64, C = TALL ? 64 : LONG, LDX = C + 8;   // G's padded shape
    constexpr int RO = TALL ? LONG / 2 : 64, CO = TALL ? 64 : LONG / 2, LDO = CO + 4;
    constexpr int PARTS = kSmallWaves * 10 * 64 * 16, MATS = N * 64 * LD * 2, XS = N * R * LDX * 2, OS = RO * LDO * 4;
    constexpr int BYTES = (PARTS + 2 * MATS > XS ? PARTS + 2 * MATS : XS) > OS ? (PARTS + 2 * MATS > XS ? PARTS + 2 * MATS : XS) : OS;
    __shared__ alignas(16) char lds[BYTES];
    __shared__ double sums[kSmallWaves];
    auto part = reinterpret_cast<float(*)[10][64][4]>(lds);
    auto as = reinterpret_cast<_Float16(*)[64][LD]>(lds + PARTS), bs = reinterpret_cast<_Float16(*)[64][LD]>(lds + PARTS + MATS);
    auto xs = reinterpret_cast<_Float16(*)[R][LDX]>(lds);
    auto os = reinterpret_cast<float(*)[LDO]>(lds);
    const SmallJob &j = js.job[blockIdx.x];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 15, g = lane >> 4;

    // U, eight neighbours to a unit, all of a thread's loads under way at once: whole units, then the rows' ends
    constexpr int UNITS = R * (C / 8) / T, ENDS = (R + T - 1) / T;
    static_assert(R * (C / 8) % T == 0, "");
    float u[UNITS + ENDS][8];
    auto place = [&](int k, int &r, int &c) {   // a unit's row and column; false: there is none
        const int i = k * T + tid;
        if (k < UNITS) {
            r = i / (C / 8);
            c = i % (C / 8) * 8;
            return r < j.rows && c + 8 <= j.cols;
        }
        r = (k - UNITS) * T + tid;
        c = j.cols & ~7;
        return r < j.rows && c < j.cols;
    };
    auto load = [&](const void *p, int dtype, int64_t ld, float(&v)[UNITS + ENDS][8]) {
        auto whole = [&](auto type) {
            typedef decltype(type) V;   // eight numbers
#pragma unroll
            for (int k = 0; k < UNITS; ++k) {
                int r, c;
                const bool in = place(k, r, c);
                V q = {};
                if (in) __builtin_memcpy(&q, static_cast<const char *>(p) + (r * ld + c) * int(sizeof(V) / 8), sizeof(V));
#pragma unroll
                for (int e = 0; e < 8; ++e) v[k][e] = float(q[e]);
            }
            if constexpr (sizeof(V) > 16) return;   // (float32 needs no conversion, for which each load would be waited for)
            if (j.cols < 8) return;
            // the rows' last eight, of which the units have had some
            const int had = -j.cols & 7;
#pragma unroll
            for (int k = UNITS; k < UNITS + ENDS; ++k) {
                int r, c;
                const bool in = place(k, r, c);
                V q = {};
                if (in) __builtin_memcpy(&q, static_cast<const char *>(p) + (r * ld + j.cols - 8) * int(sizeof(V) / 8), sizeof(V));
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    v[k][e] = 0.f;
#pragma unroll
                    for (int h = 1; h < 8; ++h)
                        if (e + h < 8) v[k][e] = had == h ? float(q[e + h]) : v[k][e];
                }
            }
        };
        typedef float f8 __attribute__((ext_vector_type(8)));
        if (dtype == CP_F32) whole(f8());
        else if (dtype == CP_BF16) whole(nt::b8());
        else whole(h8());
        if (j.cols >= 8 && dtype != CP_F32) return;
#pragma unroll
        for (int k = UNITS; k < UNITS + ENDS; ++k) {
            int r, c;
            const bool in = place(k, r, c);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[k][e] = in && c + e < j.cols ? load_as_float(p, dtype, r * ld + c + e) : 0.f;
        }
    };
    load(j.G, j.g_dtype, j.ldg, u);
    double sum = 0.0;
    if (j.M) {
        float m[UNITS + ENDS][8];
        load(j.M, CP_F32, j.ldm, m);
#pragma unroll
        for (int k = 0; k < UNITS + ENDS; ++k) {
            int r, c;
            const bool in = place(k, r, c);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                m[k][e] = fmaf(js.momentum, m[k][e], u[k][e]);
                u[k][e] = js.nesterov ? fmaf(js.momentum, m[k][e], u[k][e]) : m[k][e];
            }
            if (!in) continue;
            float *row = j.M + r * j.ldm + c;
            if (k < UNITS) {
                *reinterpret_cast<nt::f4u *>(row) = f4{m[k][0], m[k][1], m[k][2], m[k][3]};
                *reinterpret_cast<nt::f4u *>(row + 4) = f4{m[k][4], m[k][5], m[k][6], m[k][7]};
            } else {
#pragma unroll
                for (int e = 0; e < 7; ++e)
                    if (c + e < j.cols) row[e] = m[k][e];
            }
        }
    }
#pragma unroll
    for (int k = 0; k < UNITS + ENDS; ++k)
#pragma unroll
        for (int e = 0; e < 8; ++e) sum = fma(double(u[k][e]), double(u[k][e]), sum);
    sum = wave_sum(sum);
    if (lane == 0) sums[wave] = sum;
    __syncthreads();
    sum = 0.0;
#pragma unroll
    for (int w = 0; w < kSmallWaves; ++w) sum += sums[w];
    const Inverse inv(sum, js.eps, js.x_scale);
    // X into LDS, zero in the padding; then the rows' ends
    auto put = [&](int k, int r, int c) {
        h8 hi, lo;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float x = inv.times(u[k][e]);
            hi[e] = _Float16(x);
            lo[e] = _Float16(x - float(hi[e]));
        }
        *reinterpret_cast<h8 *>(&xs[0][r][c]) = hi;
        if constexpr (SPLIT) *reinterpret_cast<h8 *>(&xs[N - 1][r][c]) = lo;
    };
#pragma unroll
    for (int k = 0; k < UNITS; ++k) put(k, (k * T + tid) / (C / 8), (k * T + tid) % (C / 8) * 8);
    __syncthreads();
#pragma unroll
    for (int k = UNITS; k < UNITS + ENDS; ++k) {
        int r, c;
        if (place(k, r, c)) put(k, r, c);
    }
    __syncthreads();

    // X by columns, xc[c][h] (rows 32 h ..), and by rows, xr[t][p] (tiles 2 p, 2 p + 1).  G's rows give one form; a product with
    // the unit matrix gives the other, exactly
    Op<SPLIT> xc[CT][2], xr[4][CT / 2];
    h8 unit[2];
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int e = 0; e < 8; ++e) unit[s][e] = _Float16((e >> 2) == s && 4 * g + (e & 3) == n ? 1.f : 0.f);
#pragma unroll
    for (int c = 0; c < CT; ++c)
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int s = 0; s < N; ++s) {
                const int tile = (wave * CT + c) * 16, row = TALL ? tile + n : t * 16 + n, col = (TALL ? t * 16 : tile) + g * 4;
                const h4 x = *reinterpret_cast<const h4 *>(&xs[s][row][col]);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (TALL) xc[c][t >> 1].v[s][4 * (t & 1) + e] = x[e];
                    else xr[t][c >> 1].v[s][4 * (c & 1) + e] = x[e];
                }
            }
    auto turn = [&](int c) {   // the other form of a column tile
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int s = 0; s < N; ++s) {
                const f4 z = {0.f, 0.f, 0.f, 0.f};
                const f4 y = TALL ? __builtin_amdgcn_mfma_f32_16x16x32_f16(xc[c][t >> 1].v[s], unit[t & 1], z, 0, 0, 0)
                                  : __builtin_amdgcn_mfma_f32_16x16x32_f16(xr[t][c >> 1].v[s], unit[c & 1], z, 0, 0, 0);
                const h4 q = __builtin_convertvector(y, h4);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (TALL) xr[t][c >> 1].v[s][4 * (c & 1) + e] = q[e];
                    else xc[c][t >> 1].v[s][4 * (t & 1) + e] = q[e];
                }
            }
    };
#pragma unroll
    for (int c = 0; c < CT; ++c) turn(c);
    __syncthreads();   // X has left LDS

    const int long_side = TALL ? j.rows : j.cols, shares = min(kSmallWaves, (long_side + CT * 16 - 1) / (CT * 16));   // waves with columns
    // a step's B, in fragments
    Op<SPLIT> bf[4][2];
    auto make_b = [&](const StepFactors &f) {
        if (wave < shares) {   // this wave's share of A = X X^T: tile (a, b) as (lane: row of a, four rows of b)
            int k = 0;
#pragma unroll
            for (int a = 0; a < 4; ++a)
#pragma unroll
                for (int b = 0; b <= a; ++b, ++k) {
                    f4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int p = 0; p < CT / 2; ++p) acc = multiply<SPLIT>(xr[b][p], xr[a][p], acc);
                    *reinterpret_cast<f4 *>(part[wave][k][lane]) = acc;
                }
        }
        __syncthreads();
        for (int i = tid; i < 640; i += T) {
            const int k = i >> 6, l = i & 63;
            const int a = k >= 6 ? 3 : k >= 3 ? 2 : k >= 1 ? 1 : 0, b = k - a * (a + 1) / 2;
            f4 v = *reinterpret_cast<const f4 *>(part[0][k][l]);
            for (int w = 1; w < shares; ++w) v += *reinterpret_cast<const f4 *>(part[w][k][l]);
            v = settled(v * f.gram);
            const int row = a * 16 + (l & 15), col = b * 16 + (l >> 4) * 4;
            const h4 hi = __builtin_convertvector(v, h4);
            *reinterpret_cast<h4 *>(&as[0][row][col]) = hi;
            h4 lo;
            if constexpr (SPLIT) {
                lo = __builtin_convertvector(v - __builtin_convertvector(hi, f4), h4);
                *reinterpret_cast<h4 *>(&as[N - 1][row][col]) = lo;
            }
            if (a != b) {
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    as[0][col + r][row] = hi[r];
                    if constexpr (SPLIT) as[N - 1][col + r][row] = lo[r];
                }
            }
        }
        __syncthreads();
        auto fragment = [&](const _Float16(*m)[64][LD], int t, int h) {   // rows 16 t .. of A or B, K = 32 h ..
            Op<SPLIT> q;
#pragma unroll
            for (int s = 0; s < N; ++s) {
                const h4 x = *reinterpret_cast<const h4 *>(&m[s][t * 16 + n][h * 32 + g * 4]);
                const h4 y = *reinterpret_cast<const h4 *>(&m[s][t * 16 + n][h * 32 + 16 + g * 4]);
                q.v[s] = __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
            }
            return q;
        };
        // B = a I + b A + c A A, two tiles to a wave
#pragma unroll
        for (int q = 0; q < 16 / kSmallWaves; ++q) {
            const int a = (wave * (16 / kSmallWaves) + q) >> 2, b = (wave * (16 / kSmallWaves) + q) & 3;
            f4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int h = 0; h < 2; ++h) v = multiply<SPLIT>(fragment(as, b, h), fragment(as, a, h), v);
            const int row = a * 16 + n, col = b * 16 + g * 4;
            f4 at = __builtin_convertvector(*reinterpret_cast<const h4 *>(&as[0][row][col]), f4);
            if constexpr (SPLIT) at += __builtin_convertvector(*reinterpret_cast<const h4 *>(&as[N - 1][row][col]), f4);
            v = v * f.poly + at * f.a;
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (col + r == row) v[r] += f.diag;
            v = settled(v);
            const h4 hi = __builtin_convertvector(v, h4);
            *reinterpret_cast<h4 *>(&bs[0][row][col]) = hi;
            if constexpr (SPLIT) *reinterpret_cast<h4 *>(&bs[N - 1][row][col]) = __builtin_convertvector(v - __builtin_convertvector(hi, f4), h4);
        }
        __syncthreads();
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int h = 0; h < 2; ++h) bf[t][h] = fragment(bs, t, h);
    };
    for (int step = 0; step + 1 < js.steps; ++step) {
        const StepFactors f = js.step[step];
        make_b(f);
        // X <- B X in G's form, and turned.  (B carries the factor: the accumulators are X's next numbers as they are.)
#pragma unroll
        for (int c = 0; c < CT; ++c) {
            f4 y[4];
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                y[t] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int h = 0; h < 2; ++h) y[t] = TALL ? multiply<SPLIT>(bf[t][h], xc[c][h], y[t]) : multiply<SPLIT>(xc[c][h], bf[t][h], y[t]);
            }
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                if (TALL) xc[c][t >> 1].set(t & 1, y[t]);
                else xr[t][c >> 1].set(c & 1, y[t]);
            }
            turn(c);
            NT_STAY();
        }
    }
    const StepFactors last = js.step[js.steps - 1];
    make_b(last);
    // O in the form whose four numbers lie in a row of G, through LDS, so that one short loop writes it
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        __syncthreads();
#pragma unroll
        for (int c = 0; c < CT / 2; ++c)
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const int tile = (wave * (CT / 2) + c) * 16, row = TALL ? tile + n : t * 16 + n, col = (TALL ? t * 16 : tile) + g * 4;
                f4 y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const Op<SPLIT> &x = xc[half * (CT / 2) + c][h];
                    y = TALL ? multiply<SPLIT>(bf[t][h], x, y) : multiply<SPLIT>(x, bf[t][h], y);
                }
                *reinterpret_cast<f4 *>(&os[row][col]) = y * last.apply;
            }
        __syncthreads();
        constexpr int FOURS = RO * (CO / 4) / T, AT_ONCE = FOURS % 4 ? 2 : 4;   // of a thread; W's loads that are under way at once
        static_assert(RO * (CO / 4) % T == 0 && FOURS % AT_ONCE == 0, "");
        auto write = [&](auto type) {
            typedef decltype(type) V;   // four numbers, at any element's address
            for (int i0 = 0; i0 < FOURS; i0 += AT_ONCE) {
                f4 v[AT_ONCE];
                V w[AT_ONCE];
                int row[AT_ONCE], col[AT_ONCE];
#pragma unroll
                for (int q = 0; q < AT_ONCE; ++q) {
                    const int i = (i0 + q) * T + tid, r = i / (CO / 4), c = i % (CO / 4) * 4;
                    // place in the long side: wave's tiles of this half
                    const int l = TALL ? r : c, at = (l / (CT * 8) * CT + half * (CT / 2)) * 16 + l % (CT * 8);
                    row[q] = TALL ? at : r;
                    col[q] = TALL ? c : at;
                    v[q] = *reinterpret_cast<const f4 *>(&os[r][c]);
                    w[q] = V{};
                    if (j.M && row[q] < j.rows && col[q] + 4 <= j.cols)
                        w[q] = take_from<V>(static_cast<const char *>(j.out) + (row[q] * j.ldo + col[q]) * int(sizeof(V) / 4));
                }
#pragma unroll
                for (int q = 0; q < AT_ONCE; ++q) {
                    if (row[q] >= j.rows || col[q] >= j.cols) continue;
                    const int64_t to = row[q] * j.ldo + col[q];
                    if (col[q] + 4 <= j.cols) {
                        const f4 o = j.M ? __builtin_convertvector(w[q], f4) * js.keep - v[q] * j.lr : v[q];
                        put_to<V>(static_cast<char *>(j.out) + to * int(sizeof(V) / 4), __builtin_convertvector(o, V));
                    } else {
                        for (int e = 0; col[q] + e < j.cols; ++e) {
                            const float o = e == 0 ? v[q][0] : e == 1 ? v[q][1] : v[q][2];
                            store_as(j.out, j.o_dtype, to + e, j.M ? js.keep * load_as_float(j.out, j.o_dtype, to + e) - j.lr * o : o);
                        }
                    }
                }
            }
        };
        if (!SPLIT || j.o_dtype == CP_BF16) write(nt::b4u());
        else if (j.o_dtype == CP_F32) write(nt::f4u());
        else write(nt::h4u());
    }
}

// a copy of G's rows (of `size` bytes a number), without gaps
struct CopyJob {
    const char *from;
    char *to;
    int64_t ld;
    int rows, cols, size;
};
__global__ void __launch_bounds__(256) k_ortho_copy(CopyJob j) {
    const int64_t n = int64_t(j.rows) * j.cols;
    for (int64_t i = blockIdx.x * 256 + threadIdx.x; i < n; i += int64_t(gridDim.x) * 256) {
        const int64_t at = i / j.cols * j.ld + i % j.cols;
        if (j.size == 4) reinterpret_cast<uint32_t *>(j.to)[i] = reinterpret_cast<const uint32_t *>(j.from)[at];
        else reinterpret_cast<uint16_t *>(j.to)[i] = reinterpret_cast<const uint16_t *>(j.from)[at];
    }
}

// ---- host --------------------------------------------------------------------------------------------------------------------
struct Plan {
    int steps = 0;
    double coef[kMaxSteps][3];
    double sx[kMaxSteps + 1], sa[kMaxSteps], sb[kMaxSteps];   // scales of X before step k, of A and B in it
};

// the power of two that puts a bound at 2^14 (what shrinks below 2^-86 is below float32's numbers after a step or two)
double scale_for(double bound) {
    int e;
    std::frexp(std::max(bound, 1e-60), &e);
    return std::ldexp(1.0, std::min(14 - e, 100));
}

// largest |p(x)| on [0, u], p(x) = x^odd (a + b x^2 + c x^4): at an end or where the derivative, a quadratic in x^2, is zero
double largest(double a, double b, double c, int odd, double u) {
    auto p = [&](double x) { return std::fabs((odd ? x : 1.0) * (a + x * x * (b + c * x * x))); };
    double best = std::max(p(0.0), p(u));
    const double qa = odd ? 5 * c : 2 * c, qb = odd ? 3 * b : b, qc = odd ? a : 0.0;   // qa y^2 + qb y + qc = 0, y = x^2
    double root[2];
    int n = 0;
    if (qa != 0.0) {
        const double d = qb * qb - 4 * qa * qc;
        if (d >= 0) {
            root[n++] = (-qb + std::sqrt(d)) / (2 * qa);
            root[n++] = (-qb - std::sqrt(d)) / (2 * qa);
        }
    } else if (qb != 0.0) {
        root[n++] = -qc / qb;
    }
    for (int i = 0; i < n; ++i)
        if (root[i] > 0 && root[i] < u * u) best = std::max(best, p(std::sqrt(root[i])));
    return best;
}

int make_plan(cp_ctx *ctx, int steps, const double *coef, double eps, Plan &pl) {
    if (steps < 1 || steps > kMaxSteps) return cp_set_error(ctx, CP_ERR_ARG, "steps %d (1..%d)", steps, kMaxSteps);
    if (!(eps >= 0) || !std::isfinite(eps)) return cp_set_error(ctx, CP_ERR_ARG, "eps");
    pl.steps = steps;
    double u = 1.0;
    pl.sx[0] = scale_for(u);
    for (int k = 0; k < steps; ++k) {
        const double *q = coef ? coef + 3 * k : kDefault;
        for (int i = 0; i < 3; ++i) {
            if (!std::isfinite(q[i])) return cp_set_error(ctx, CP_ERR_ARG, "coef of step %d is not finite", k);
            pl.coef[k][i] = q[i];
        }
        pl.sa[k] = scale_for(u * u);
        const double b = largest(q[0], q[1], q[2], 0, u);
        u = largest(q[0], q[1], q[2], 1, u);
        if (!(b < 4096) || !(u < 16)) return cp_set_error(ctx, CP_ERR_ARG, "coef of step %d lets singular values grow to %g", k, u);
        pl.sb[k] = scale_for(b);
        pl.sx[k + 1] = scale_for(u);
    }
    return CP_OK;
}

bool ortho_type(int d) { return d == CP_F32 || d == CP_BF16 || d == CP_F16; }
size_t type_size(int d) { return d == CP_F32 ? 4 : 2; }

// one matrix of the call, for the overlap check
struct Region {
    uintptr_t at;
    int64_t ld, rows, cols;
    size_t size;
    size_t job;
    bool read;   // G
    int64_t width() const { return cols * int64_t(size); }
    uintptr_t end() const { return at + (size_t(rows - 1) * ld + cols) * size; }
};

// whether two matrices share a byte
bool overlap(const Region &p, const Region &q) {
    if (p.at >= q.end() || q.at >= p.end()) return false;
    if (p.ld == q.ld && p.size == q.size) {   // rows of one stride interleave as column ranges of one wider matrix do
        const Region &lo = p.at <= q.at ? p : q, &hi = p.at <= q.at ? q : p;
        const int64_t stride = lo.ld * int64_t(lo.size), d = int64_t(hi.at - lo.at) % stride;   // hi's first byte, counted from a row of lo
        return d < lo.width() || d + hi.width() > stride;
    }
    // every row of the one with fewer against the first row of the other that ends behind its begin
    const Region &few = p.rows <= q.rows ? p : q, &many = p.rows <= q.rows ? q : p;
    const int64_t stride = many.ld * int64_t(many.size);
    for (int64_t i = 0; i < few.rows; ++i) {
        const int64_t begin = int64_t(few.at) + i * few.ld * int64_t(few.size) - int64_t(many.at);
        const int64_t row = begin < many.width() ? 0 : (begin - many.width()) / stride + 1;
        if (row < many.rows && row * stride < begin + few.width()) return true;
    }
    return false;
}

struct Request {
    const void *G;
    float *M;
    void *out;
    int64_t ldg, ldm, ldo;
    int rows, cols, g_dtype, o_dtype;
    double gamma;
};

// `crossed`: whether an output shares memory with another job's G.  The products' path reads every G before it writes, but a
// small matrix is read and written by one kernel: such a call's G are copied first.
int check_requests(cp_ctx *ctx, const std::vector<Request> &rq, bool step, bool &crossed) {
    std::vector<Region> w;
    for (size_t k = 0; k < rq.size(); ++k) {
        const Request &r = rq[k];
        if (r.rows < 0 || r.cols < 0 || r.rows > (1 << 20) || r.cols > (1 << 20))
            return cp_set_error(ctx, CP_ERR_ARG, "job %d: rows, cols (0..2^20)", int(k));
        if (!ortho_type(r.g_dtype) || !ortho_type(r.o_dtype)) return cp_set_error(ctx, CP_ERR_ARG, "job %d: type", int(k));
        if (r.ldg < r.cols || r.ldo < r.cols || (step && r.ldm < r.cols))
            return cp_set_error(ctx, CP_ERR_ARG, "job %d: row stride below cols", int(k));
        if (step && !std::isfinite(r.gamma)) return cp_set_error(ctx, CP_ERR_ARG, "job %d: gamma", int(k));
        if (!r.rows || !r.cols) continue;
        if (!r.G || !r.out || (step && !r.M)) return cp_set_error(ctx, CP_ERR_ARG, "job %d: null pointer", int(k));
        if (uintptr_t(r.G) % type_size(r.g_dtype) || uintptr_t(r.out) % type_size(r.o_dtype) || uintptr_t(r.M) % 4)
            return cp_set_error(ctx, CP_ERR_ARG, "job %d: alignment", int(k));
        if (std::min(r.rows, r.cols) > 65536)
            return cp_set_error(ctx, CP_ERR_UNSUPPORTED, "job %d: shorter side above 65536", int(k));
        w.push_back({uintptr_t(r.G), r.ldg, r.rows, r.cols, type_size(r.g_dtype), k, true});
        w.push_back({uintptr_t(r.out), r.ldo, r.rows, r.cols, type_size(r.o_dtype), k, false});
        if (step) w.push_back({uintptr_t(r.M), r.ldm, r.rows, r.cols, 4, k, false});
    }
    std::sort(w.begin(), w.end(), [](const Region &p, const Region &q) { return p.at < q.at; });
    crossed = false;
    for (size_t i = 0; i < w.size(); ++i)
        for (size_t k = i + 1; k < w.size() && w[k].at < w[i].end(); ++k) {
            const Region &p = w[i], &q = w[k];
            if ((p.read && q.read) || !overlap(p, q)) continue;
            if (!p.read && !q.read) return cp_set_error(ctx, CP_ERR_ARG, "two outputs of the call overlap");
            if (step)   // the momentum is written while other jobs' gradients are still to be read
                return cp_set_error(ctx, CP_ERR_ARG, "job %d's G overlaps job %d's M or W", int((p.read ? p : q).job), int((p.read ? q : p).job));
            crossed |= p.job != q.job;
        }
    return CP_OK;
}

// whether a job's numbers are carried as pairs: see the head of this file
bool is_split(const Request &r) { return r.M || r.g_dtype != CP_BF16 || r.o_dtype != CP_BF16; }

int64_t padded(int64_t v) { return (v + kPad - 1) / kPad * kPad; }

size_t job_bytes(const Request &r) {
    if (!r.rows || !r.cols) return 0;
    const size_t e = is_split(r) ? 4 : 2;
    const size_t mp = padded(std::min(r.rows, r.cols)), np = padded(std::max(r.rows, r.cols));
    return cp_align_up(kPartials * sizeof(double) + e * (3 * mp * np + 2 * mp * mp), 256);
}

// One launch of a product over a class's jobs: its shape of tile, and the pieces that each job's tiles are cut into
struct Choice {
    int cfg;           // 0 Large, 1 Medium, 2 Small
    int grid;
    int slots;         // of partial sums: the workgroups of the jobs whose tiles are cut
};

// The jobs of one class (one fp16 a number, or pairs)
struct Class {
    bool split;
    std::vector<Job> jobs;
    std::vector<Place> places;
    std::vector<int> sum_groups;   // workgroups of k_ortho_norm
    Table table;
    int64_t loads = 0;
    Choice gram, poly, apply, last;
};

constexpr int kEdge[3] = {256, 128, 64};
constexpr int64_t kMaxThreads = (int64_t(1) << 32) - 1;   // of a launch

int64_t tiles_of(const Job &j, int phase, int edge) {
    const int64_t m = (j.mp + edge - 1) / edge, n = (j.np + edge - 1) / edge;
    return phase == APPLY || phase == LAST ? m * n : m * (m + 1) / 2;
}
int64_t steps_of(const Job &j, int phase) { return (phase == GRAM ? j.ldn : j.lds) / 128; }

// What a launch costs in us, from its number of workgroups, their K steps in all and the longest's.
// Measured: us per step and workgroup where a CU holds as many as fit (Large one, the others two), and where there is at most
// one to a CU; what a workgroup costs beside its steps (first loads, stores: twice as many where numbers are pairs); a join; and
// what it costs to read and write W.
double cost_of(int cfg, bool split, bool weights, int64_t groups, int64_t total, int64_t longest, bool joins) {
    static const double full[2][3] = {{1.55, 1.04, 0.33}, {2.25, 1.35, 0.37}}, alone[2][3] = {{1.35, 0.60, 0.20}, {2.0, 0.75, 0.28}};
    static const double extra[2][3] = {{14.0, 6.0, 3.0}, {19.0, 11.0, 4.0}}, joined[3] = {14.0, 5.0, 3.0}, update[3] = {20.0, 13.0, 2.2};
    const int slots = cfg == 0 ? kCus : 2 * kCus;
    const double step = groups > kCus ? full[split][cfg] : alone[split][cfg];
    const double more = extra[split][cfg] + (joins ? joined[cfg] : 0.0) + (weights ? update[cfg] : 0.0);
    const double mean = double(total) / groups * step + more, most = longest * step + more, rounds = double(groups) / slots;
    // equal workgroups end together; others fill each other's gaps
    return std::max(most, mean * (total == longest * groups ? std::ceil(rounds) : rounds + 0.3));
}

constexpr int kLeast = 32;   // K steps of a piece, at least

// into how many pieces of k a job's tiles are cut: as if it were alone, so that its sums do not depend on the call's other jobs
int pieces_of(const Job &j, int phase, bool split) {
    const int64_t steps = steps_of(j, phase);
    double least = 1e30;
    int best = 1;
    for (int cfg = 0; cfg < 3; ++cfg) {
        const int64_t tiles = tiles_of(j, phase, kEdge[cfg]);
        for (int p = 1; p <= 16 && (p == 1 || steps / p >= kLeast); ++p) {
            const double c = cost_of(cfg, split, phase == LAST && j.M, tiles * p, tiles * steps, (steps + p - 1) / p, p > 1);
            if (c < 0.97 * least) {
                least = c;
                best = p;
            }
        }
    }
    return best;
}

bool choose(Class &cl, int phase, Choice &best) {
    double least = 1e300;
    const int knob = cp_knob(CP_KNOB_NT_TILE), forced = knob > 3 ? 0 : knob;   // (the others are the 8-bit products')
    for (int cfg = 0; cfg < 3; ++cfg) {
        if (forced && forced - 1 != cfg) continue;
        int64_t groups = 0, total = 0, longest = 0;
        bool joins = false;
        for (size_t k = 0; k < cl.jobs.size(); ++k) {
            const int64_t tiles = tiles_of(cl.jobs[k], phase, kEdge[cfg]), steps = steps_of(cl.jobs[k], phase);
            const int p = cl.places[k].pieces(phase);
            joins |= p > 1;
            groups += tiles * p;
            total += tiles * steps;
            longest = std::max(longest, (steps + p - 1) / p);
        }
        if (groups * (cfg == 0 ? nt::Large::T : nt::Medium::T) > kMaxThreads) continue;
        const double cost = cost_of(cfg, cl.split, phase == LAST && cl.jobs[0].M, groups, total, longest, joins);
        if (cost < least) {
            least = cost;
            best = {cfg, int(groups), 0};
        }
    }
    if (least == 1e300) return false;
    int at = 0;
    for (size_t k = 0; k < cl.jobs.size(); ++k) {
        Place &p = cl.places[k];
        const int pieces = p.pieces(phase), groups = int(tiles_of(cl.jobs[k], phase, kEdge[best.cfg])) * pieces;
        p.first[phase] = at;
        at += groups;
        if (pieces == 1) continue;
        p.share[phase - 1] = pieces | best.slots << kShareBits;
        best.slots += groups;
    }
    return true;
}

// The layout of a call in its workspace: | arrival counters | pieces of tiles | tables | the jobs' matrices |
struct Layout {
    size_t counts = 0, parts = 0, tables = 0, jobs = 0, copies = 0;   // bytes
    Class cls[2];
    std::vector<SmallJob> small[2][2][4];   // [class][tall][column tiles of a wave / 2]
    std::vector<CopyJob> copied;
    size_t all() const { return (jobs ? counts + parts + tables + jobs : 0) + copies; }
};

// column tiles that each of eight waves takes of a small matrix (an even number), or 0 where the matrix is not small
int small_tiles(const Request &r) {
    const bool split = is_split(r);
    const int tiles = (std::max(r.rows, r.cols) + 15) / 16, each = (tiles + kSmallWaves - 1) / kSmallWaves;
    return std::min(r.rows, r.cols) <= 64 && each <= kSmallTiles[split] ? (each + 1) / 2 * 2 : 0;
}

size_t table_bytes(size_t n) { return cp_align_up(n * (sizeof(Job) + (2 * PHASES - 1) * sizeof(int)), 256); }

int lay_out(cp_ctx *ctx, const std::vector<Request> &rq, bool crossed, double lr, Layout &lay) {
    lay.cls[0].split = false;
    lay.cls[1].split = true;
    bool small = !cp_knob(CP_KNOB_NT_TILE);   // beside larger matrices, small ones cost next to nothing in the products' launches
    for (const Request &r : rq) small &= !r.rows || !r.cols || small_tiles(r) > 0;
    const bool copy = small && crossed;
    for (const Request &r : rq) {
        if (!r.rows || !r.cols) continue;
        if (small) {
            const int ct = small_tiles(r);
            SmallJob j = {r.G, r.M, r.out, r.ldg, r.ldm, r.ldo, r.rows, r.cols, r.g_dtype, r.o_dtype, float(lr * r.gamma)};
            if (copy) {
                const size_t size = type_size(r.g_dtype);
                lay.copied.push_back({static_cast<const char *>(r.G), reinterpret_cast<char *>(lay.copies), r.ldg, r.rows, r.cols, int(size)});
                j.G = reinterpret_cast<const void *>(lay.copies);   // offsets so far
                j.ldg = r.cols;
                lay.copies += cp_align_up(size_t(r.rows) * r.cols * size, 256);
            }
            lay.small[is_split(r)][r.rows > r.cols][ct / 2].push_back(j);
            continue;
        }
        Class &cl = lay.cls[is_split(r)];
        const size_t e = cl.split ? 4 : 2;
        const size_t mp = padded(std::min(r.rows, r.cols)), np = padded(std::max(r.rows, r.cols));
        Job j = {};
        j.G = r.G;
        j.M = r.M;
        j.out = r.out;
        j.ldg = r.ldg;
        j.ldm = r.ldm;
        j.ldo = r.ldo;
        j.rows = r.rows;
        j.cols = r.cols;
        j.mp = int(mp);
        j.np = int(np);
        j.ldn = uint32_t(np * e);
        j.lds = uint32_t(mp * e);
        j.g_dtype = int16_t(r.g_dtype);
        j.o_dtype = int16_t(r.o_dtype);
        j.lr = float(lr * r.gamma);
        const bool flat = r.ldg == r.cols && (!r.M || r.ldm == r.cols);
        j.sum_rows = flat ? 1 : r.rows;
        j.sum_cols = flat ? int64_t(r.rows) * r.cols : r.cols;
        j.width = flat ? int(std::max<int64_t>(4096, (j.sum_cols / kPartials + 2048) / 2048 * 2048)) : 4096;
        j.chunks = int((j.sum_cols + j.width - 1) / j.width);
        j.rows_per = int(std::max<int64_t>(1, 4096 / std::min<int64_t>(j.sum_cols, 4096)));
        while (int64_t((j.sum_rows + j.rows_per - 1) / j.rows_per) * j.chunks > kPartials) j.rows_per *= 2;
        j.part = reinterpret_cast<double *>(lay.jobs);   // an offset so far
        lay.jobs += job_bytes(r);
        Place p = {};
        p.first[LOAD] = int(cl.loads);
        cl.loads += int64_t(mp / 64) * int64_t(np / 64);
        for (int phase = GRAM; phase < PHASES; ++phase) p.share[phase - 1] = pieces_of(j, phase, cl.split);
        cl.sum_groups.push_back((j.sum_rows + j.rows_per - 1) / j.rows_per * j.chunks);
        cl.jobs.push_back(j);
        cl.places.push_back(p);
    }
    for (Class &cl : lay.cls) {
        if (cl.jobs.empty()) continue;
        if (cl.loads * 256 > kMaxThreads || !choose(cl, GRAM, cl.gram) || !choose(cl, POLY, cl.poly) || !choose(cl, APPLY, cl.apply) || !choose(cl, LAST, cl.last))
            return cp_set_error(ctx, CP_ERR_UNSUPPORTED, "matrices of a call too large for one launch");
        for (const Choice *c : {&cl.gram, &cl.poly, &cl.apply, &cl.last})
            if (c->slots) {
                lay.counts = std::max(lay.counts, cp_align_up(size_t(c->slots) * sizeof(int), 256));
                lay.parts = std::max(lay.parts, size_t(c->slots) * kEdge[c->cfg] * kEdge[c->cfg] * sizeof(float));
            }
        lay.tables += table_bytes(cl.jobs.size());
    }
    return CP_OK;
}

// the offsets become pointers into the workspace
void place(Layout &lay, char *ws) {
    char *tables = ws + lay.counts + lay.parts, *jobs = tables + lay.tables;
    if (!lay.copied.empty()) {
        char *copies = jobs + lay.jobs;
        for (CopyJob &c : lay.copied) c.to = copies + reinterpret_cast<size_t>(c.to);
        for (auto &of : lay.small)
            for (auto &way : of)
                for (auto &list : way)
                    for (SmallJob &j : list) j.G = copies + reinterpret_cast<size_t>(j.G);
    }
    for (Class &cl : lay.cls) {
        const size_t n = cl.jobs.size();
        if (!n) continue;
        cl.table.n = int(n);
        cl.table.job = reinterpret_cast<Job *>(tables);
        int *p = reinterpret_cast<int *>(tables + n * sizeof(Job));
        for (int k = 0; k < PHASES; ++k) cl.table.first[k] = p + k * n;
        for (int k = 0; k < PHASES - 1; ++k) cl.table.share[k] = p + (PHASES + k) * n;
        tables += table_bytes(n);
        for (Job &j : cl.jobs) {
            const size_t mn = size_t(j.mp) * j.ldn, mm = size_t(j.mp) * j.lds;
            char *q = jobs + reinterpret_cast<size_t>(j.part);
            j.part = reinterpret_cast<double *>(q);
            j.x = q + kPartials * sizeof(double);
            j.xt0 = j.x + mn;
            j.xt1 = j.xt0 + mn;
            j.a = j.xt1 + mn;
            j.b = j.a + mm;
        }
    }
}

StepFactors step_factors(const Plan &pl, int k) {
    const double sx = pl.sx[k], sa = pl.sa[k], sb = pl.sb[k];
    return {float(sa / (sx * sx)), float(pl.coef[k][2] * sb / (sa * sa)), float(pl.coef[k][1] * sb / sa), float(pl.coef[k][0] * sb),
            float((k + 1 < pl.steps ? pl.sx[k + 1] : 1.0) / (sb * sx))};
}

struct Call {
    hipStream_t st;
    const Layout &lay;
    char *ws;
    int *counts() const { return reinterpret_cast<int *>(ws); }
    float *parts() const { return reinterpret_cast<float *>(ws + lay.counts); }
};

template <int PHASE, bool SPLIT>
void launch_product(const Call &call, const Table &t, const Choice &c, const Factors &f) {
    if (c.cfg == 0) k_ortho_product<PHASE, SPLIT, nt::Large><<<c.grid, nt::Large::T, 0, call.st>>>(t, f, call.parts(), call.counts());
    else if (c.cfg == 1) k_ortho_product<PHASE, SPLIT, nt::Medium><<<c.grid, nt::Medium::T, 0, call.st>>>(t, f, call.parts(), call.counts());
    else k_ortho_product<PHASE, SPLIT, nt::Small><<<c.grid, nt::Small::T, 0, call.st>>>(t, f, call.parts(), call.counts());
}

template <bool SPLIT>
void launch_steps(const Call &call, const Class &cl, const Plan &pl, float keep) {
    for (int k = 0; k < pl.steps; ++k) {
        const StepFactors q = step_factors(pl, k);
        Factors f = {};
        f.xt = k & 1;
        f.acc = q.gram;
        launch_product<GRAM, SPLIT>(call, cl.table, cl.gram, f);
        f.acc = q.poly;
        f.a = q.a;
        f.diag = q.diag;
        launch_product<POLY, SPLIT>(call, cl.table, cl.poly, f);
        f.acc = q.apply;
        f.keep = keep;
        if (k + 1 < pl.steps) launch_product<APPLY, SPLIT>(call, cl.table, cl.apply, f);
        else launch_product<LAST, SPLIT>(call, cl.table, cl.last, f);
    }
}

template <bool SPLIT, bool TALL>
void launch_small(hipStream_t st, const std::vector<SmallJob> &jobs, SmallJobs &js, int ct) {
    const int T = 64 * kSmallWaves;
    for (size_t base = 0; base < jobs.size(); base += kSmallJobs) {
        const int n = int(std::min<size_t>(kSmallJobs, jobs.size() - base));
        std::copy(jobs.begin() + base, jobs.begin() + base + n, js.job);
        if (ct == 1) k_ortho_small<SPLIT, 2, TALL><<<n, T, 0, st>>>(js);
        else if (ct == 2) k_ortho_small<SPLIT, 4, TALL><<<n, T, 0, st>>>(js);
        if constexpr (!SPLIT) {
            if (ct == 3) k_ortho_small<SPLIT, 6, TALL><<<n, T, 0, st>>>(js);
        }
    }
}

int run(cp_ctx *ctx, const std::vector<Request> &rq, bool crossed, const Plan &pl, double lr, double momentum, int nesterov, double decay,
        double eps, void *given, size_t given_bytes) {
    // (no more than that: lr, decay and gamma are finite, so that a NaN is not among them)
    bool fits = std::fabs(momentum) <= FLT_MAX && std::fabs(1.0 - lr * decay) <= FLT_MAX;
    for (const Request &r : rq) fits &= std::fabs(lr * r.gamma) <= FLT_MAX;
    if (!fits) return cp_set_error(ctx, CP_ERR_ARG, "momentum, 1 - lr weight_decay or lr gamma is past float32");
    Layout lay;
    CP_TRY(lay_out(ctx, rq, crossed, lr, lay));
    CP_HIP(ctx, hipSetDevice(ctx->device));
    char *ws = nullptr;
    if (lay.all()) {
        CP_TRY(cp_scratch(ctx, given, given_bytes, lay.all(), &ws));
        place(lay, ws);
    }
    const Call call = {ctx->stream, lay, ws};
    const float mu = float(momentum), keep = float(1.0 - lr * decay), sx = float(pl.sx[0]);
    // every job's G is read (or copied) before any output is written: an output may be another job's G
    for (const CopyJob &c : lay.copied)
        k_ortho_copy<<<int(std::min<int64_t>(256, (int64_t(c.rows) * c.cols + 255) / 256)), 256, 0, call.st>>>(c);
    for (const Class &cl : lay.cls)
        for (size_t base = 0; base < cl.jobs.size(); base += kJobs) {
            Jobs js = {};
            js.base = int(base);
            int groups = 0;
            for (; js.n < kJobs && base + js.n < cl.jobs.size(); ++js.n) {
                js.first[js.n] = groups;
                js.job[js.n] = cl.jobs[base + js.n];
                js.place[js.n] = cl.places[base + js.n];
                groups += cl.sum_groups[base + js.n];
            }
            k_ortho_norm<<<groups, 256, 0, call.st>>>(js, cl.table, mu, nesterov, call.counts(), int(lay.counts / sizeof(int)));
        }
    for (const Class &cl : lay.cls) {
        if (cl.jobs.empty()) continue;
        if (cl.split) k_ortho_load<true><<<uint32_t(cl.loads), 256, 0, call.st>>>(cl.table, mu, nesterov, eps, sx);
        else k_ortho_load<false><<<uint32_t(cl.loads), 256, 0, call.st>>>(cl.table, mu, nesterov, eps, sx);
    }
    SmallJobs js = {};
    js.eps = eps;
    js.x_scale = pl.sx[0];
    js.momentum = mu;
    js.keep = keep;
    js.nesterov = nesterov;
    js.steps = pl.steps;
    for (int k = 0; k < pl.steps; ++k) {
        StepFactors q = step_factors(pl, k);
        if (k + 1 < pl.steps) {   // B takes X from its scale to the next step's
            q.poly *= q.apply;
            q.a *= q.apply;
            q.diag *= q.apply;
            q.apply = 1.f;
        }
        js.step[k] = q;
    }
    for (int ct = 1; ct <= 3; ++ct) {
        launch_small<false, false>(call.st, lay.small[0][0][ct], js, ct);
        launch_small<false, true>(call.st, lay.small[0][1][ct], js, ct);
        if (ct > 2) continue;
        launch_small<true, false>(call.st, lay.small[1][0][ct], js, ct);
        launch_small<true, true>(call.st, lay.small[1][1][ct], js, ct);
    }
    for (const Class &cl : lay.cls) {
        if (cl.jobs.empty()) continue;
        if (cl.split) launch_steps<true>(call, cl, pl, keep);
        else launch_steps<false>(call, cl, pl, keep);
    }
    CP_LAUNCH_CHECK(ctx);
    return CP_OK;
}

int take_jobs(cp_ctx *ctx, int n, const cp_ortho_job *jobs, std::vector<Request> &rq, bool &crossed) {
    if (n < 0 || (n && !jobs)) return cp_set_error(ctx, CP_ERR_ARG, "jobs");
    for (int i = 0; i < n; ++i) {
        const cp_ortho_job &q = jobs[i];
        rq.push_back({q.G, nullptr, q.O, q.ldg, 0, q.ldo, q.rows, q.cols, q.g_dtype, q.o_dtype, 1.0});
    }
    return check_requests(ctx, rq, false, crossed);
}

int take_jobs(cp_ctx *ctx, int n, const cp_ortho_step_job *jobs, std::vector<Request> &rq, bool &crossed) {
    if (n < 0 || (n && !jobs)) return cp_set_error(ctx, CP_ERR_ARG, "jobs");
    for (int i = 0; i < n; ++i) {
        const cp_ortho_step_job &q = jobs[i];
        rq.push_back({q.G, q.M, q.W, q.ldg, q.ldm, q.ldw, q.rows, q.cols, q.g_dtype, q.w_dtype, q.gamma});
    }
    return check_requests(ctx, rq, true, crossed);
}

template <typename J>
int workspace(int n, const J *jobs, int steps, const double *coef, double eps, size_t *bytes) {
    if (!bytes) return CP_ERR_ARG;
    try {
        Plan pl;
        std::vector<Request> rq;
        bool crossed = false;
        CP_TRY(make_plan(nullptr, steps, coef, eps, pl));
        CP_TRY(take_jobs(nullptr, n, jobs, rq, crossed));
        Layout lay;
        CP_TRY(lay_out(nullptr, rq, crossed, 0.0, lay));
        *bytes = lay.all();
        return CP_OK;
    } catch (...) {
        return CP_ERR_NOMEM;
    }
}

}  // namespace

extern "C" int cp_orthogonalise_workspace(int n_jobs, const cp_ortho_job *jobs, int steps, const double *coef, double eps,
                                          size_t *bytes) {
    return workspace(n_jobs, jobs, steps, coef, eps, bytes);
}

extern "C" int cp_ortho_step_workspace(int n_jobs, const cp_ortho_step_job *jobs, int steps, const double *coef, double eps,
                                       size_t *bytes) {
    return workspace(n_jobs, jobs, steps, coef, eps, bytes);
}

extern "C" int cp_orthogonalise(cp_ctx *ctx, int n_jobs, const cp_ortho_job *jobs, int steps, const double *coef, double eps,
                                void *ws, size_t ws_bytes) {
    if (!ctx) return CP_ERR_ARG;
    try {
        Plan pl;
        std::vector<Request> rq;
        bool crossed = false;
        CP_TRY(make_plan(ctx, steps, coef, eps, pl));
        CP_TRY(take_jobs(ctx, n_jobs, jobs, rq, crossed));
        return run(ctx, rq, crossed, pl, 0.0, 0.0, 0, 0.0, eps, ws, ws_bytes);
    } catch (...) {
        return cp_set_error(ctx, CP_ERR_NOMEM, "host memory");
    }
}

extern "C" int cp_ortho_step(cp_ctx *ctx, int n_jobs, const cp_ortho_step_job *jobs, double lr, double momentum, int nesterov,
                             double weight_decay, int steps, const double *coef, double eps, void *ws, size_t ws_bytes) {
    if (!ctx) return CP_ERR_ARG;
    if (!std::isfinite(lr) || !std::isfinite(momentum) || !std::isfinite(weight_decay))
        return cp_set_error(ctx, CP_ERR_ARG, "lr, momentum or weight_decay is not finite");
    try {
        Plan pl;
        std::vector<Request> rq;
        bool crossed = false;
        CP_TRY(make_plan(ctx, steps, coef, eps, pl));
        CP_TRY(take_jobs(ctx, n_jobs, jobs, rq, crossed));
        return run(ctx, rq, crossed, pl, lr, momentum, nesterov != 0, weight_decay, eps, ws, ws_bytes);
    } catch (...) {
        return cp_set_error(ctx, CP_ERR_NOMEM, "host memory");
    }
}
