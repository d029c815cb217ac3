// Orthogonalised updates: Newton-Schulz products on a set of matrices, and the optimiser step around them.
//
// X = U / (|U|_F + eps) lies with its short side m first (a tall matrix is taken transposed).  Every step is three products
//     A = X X^T,   B = a I + b A + c A A,   X <- B X
// the first two symmetric: only the tiles on and below the diagonal are computed, and mirrored.
//
// Numbers.  Singular values stay in [0, u_k] with bounds u_k that the host derives from the coefficients, so every entry of X,
// A and B is bounded too, and a power of two per step and matrix puts that bound at 2^14: fp16's whole range is used, with
// headroom of four.  fp16 then holds 11 bits of an entry where bf16 would hold 8, at the same rate.  Results of 24 or 11 bits
// carry a pair of fp16 (22 bits) and three products instead of one; the pair's dropped low * low term is below its rounding.
// Sums are float32 in the accumulators, |U|_F is summed in float64.
#include <algorithm>
#include <cmath>

#include "cp_common.h"
#include "nt_mfma.h"

namespace {

using nt::f4;
using nt::h4;
using nt::h8;

constexpr int kJobs = 24;        // jobs of one launch: their table travels in the kernel's arguments (4 KB)
constexpr int kMaxSteps = 32;
constexpr int kPartials = 256;   // partial sums of |U|_F^2 per job
constexpr int kTile = 128;
constexpr double kDefault[3] = {3.4445, -4.7750, 2.0315};

struct Job {
    const void *G;
    float *M;                    // momentum (cp_ortho_step), else null
    void *out;                   // O, or W
    char *x, *xt0, *xt1, *a, *b; // X [mp][np], X^T [np][mp] twice, A and B [mp][mp]
    double *part;
    int64_t ldg, ldm, ldo;
    uint32_t ldn, lds;           // bytes of a row of np / of mp numbers
    int rows, cols, mp, np;
    int g_dtype, o_dtype;
    float lr;                    // lr * gamma
    int first_sym, first_apply, first_load;   // this job's first workgroup of the phase
};

struct Jobs {
    int n, total_sym, total_apply, total_load;
    Job job[kJobs];
};
static_assert(sizeof(Jobs) <= 3900, "kernel arguments");

__device__ __forceinline__ float load_as_float(const void *p, int dtype, int64_t at) {
    if (dtype == CP_F32) return static_cast<const float *>(p)[at];
    if (dtype == CP_BF16) return float(static_cast<const __bf16 *>(p)[at]);
    return float(static_cast<const _Float16 *>(p)[at]);
}
__device__ __forceinline__ void store_as(void *p, int dtype, int64_t at, float v) {
    if (dtype == CP_F32) static_cast<float *>(p)[at] = v;
    else if (dtype == CP_BF16) static_cast<__bf16 *>(p)[at] = __bf16(v);
    else static_cast<_Float16 *>(p)[at] = _Float16(v);
}

__device__ __forceinline__ double wave_sum(double v) {
    for (int s = 32; s; s >>= 1) v += __shfl_xor(v, s);
    return v;
}

// ---- |U|_F, and the momentum -----------------------------------------------------------------------------------------------
__global__ void __launch_bounds__(256) k_ortho_norm(Jobs js, float momentum, int nesterov) {
    const Job &j = js.job[blockIdx.y];
    double sum = 0.0;
    for (int r = blockIdx.x; r < j.rows; r += kPartials)
        for (int c = threadIdx.x; c < j.cols; c += 256) {
            float u = load_as_float(j.G, j.g_dtype, r * j.ldg + c);
            if (j.M) {
                float *m = j.M + r * j.ldm + c;
                const float v = fmaf(momentum, *m, u);
                *m = v;
                u = nesterov ? fmaf(momentum, v, u) : v;
            }
            sum += double(u) * double(u);
        }
    __shared__ double s[4];
    sum = wave_sum(sum);
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = sum;
    __syncthreads();
    if (threadIdx.x == 0) j.part[blockIdx.x] = (s[0] + s[1]) + (s[2] + s[3]);
}

__device__ __forceinline__ int find_job(const Jobs &js, int id, int Job::*first) {
    int k = js.n - 1;
    while (k > 0 && js.job[k].*first > id) --k;
    return k;
}

// sixteen numbers of a row, from column k (a multiple of 16), as fp16 or as pairs
template <bool SPLIT>
__device__ __forceinline__ void store16(char *row, int k, const float (&v)[16]) {
    char *p = row + (SPLIT ? (k >> 5) * 128 + (k & 31) * 2 : k * 2);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        h8 hi, lo;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            hi[e] = _Float16(v[8 * h + e]);
            lo[e] = _Float16(v[8 * h + e] - float(hi[e]));
        }
        *reinterpret_cast<h8 *>(p + 16 * h) = hi;
        if (SPLIT) *reinterpret_cast<h8 *>(p + 64 + 16 * h) = lo;
    }
}

// four numbers of a row, from column k (a multiple of 4)
template <bool SPLIT>
__device__ __forceinline__ void store4(char *row, int k, f4 v) {
    char *p = row + (SPLIT ? (k >> 5) * 128 + (k & 31) * 2 : k * 2);
    const h4 hi = __builtin_convertvector(v, h4);
    *reinterpret_cast<h4 *>(p) = hi;
    if (SPLIT) *reinterpret_cast<h4 *>(p + 64) = __builtin_convertvector(v - __builtin_convertvector(hi, f4), h4);
}
template <bool SPLIT>
__device__ __forceinline__ void store1(char *row, int k, float v) {
    char *p = row + (SPLIT ? (k >> 5) * 128 + (k & 31) * 2 : k * 2);
    const _Float16 hi = _Float16(v);
    *reinterpret_cast<_Float16 *>(p) = hi;
    if (SPLIT) *reinterpret_cast<_Float16 *>(p + 64) = _Float16(v - float(hi));
}
template <bool SPLIT>
__device__ __forceinline__ f4 load4(const char *row, int k) {
    const char *p = row + (SPLIT ? (k >> 5) * 128 + (k & 31) * 2 : k * 2);
    f4 v = __builtin_convertvector(*reinterpret_cast<const h4 *>(p), f4);
    if (SPLIT) v += __builtin_convertvector(*reinterpret_cast<const h4 *>(p + 64), f4);
    return v;
}

// ---- X = U / (|U|_F + eps) in both orientations, zero outside ---------------------------------------------------------------
template <bool SPLIT>
__global__ void __launch_bounds__(256) k_ortho_load(Jobs js, float momentum, int nesterov, double eps, float x_scale) {
    const Job &j = js.job[find_job(js, blockIdx.x, &Job::first_load)];
    const bool tall = j.rows > j.cols;
    const int pr = tall ? j.np : j.mp, pc = tall ? j.mp : j.np;   // padded rows / columns of G as it lies
    const int id = blockIdx.x - j.first_load, tiles_c = pc / 64;
    const int r0 = id / tiles_c * 64, c0 = id % tiles_c * 64;
    (void)pr;
    __shared__ double s[4];
    __shared__ float t[64][65];
    const int tid = threadIdx.x;
    const double part = wave_sum(j.part[tid]);
    if ((tid & 63) == 0) s[tid >> 6] = part;
    __syncthreads();
    const double norm = sqrt((s[0] + s[1]) + (s[2] + s[3])) + eps;
    const double inv = norm > 0.0 || norm != norm ? double(x_scale) / norm : 0.0;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const int r = i * 4 + (tid >> 6), c = tid & 63;
        float v = 0.f;
        if (r0 + r < j.rows && c0 + c < j.cols) {
            float u = load_as_float(j.G, j.g_dtype, int64_t(r0 + r) * j.ldg + c0 + c);
            if (j.M) {
                const float m = j.M[int64_t(r0 + r) * j.ldm + c0 + c];
                u = nesterov ? fmaf(momentum, m, u) : m;
            }
            v = float(double(u) * inv);
        }
        t[r][c] = v;
    }
    __syncthreads();
    char *n = tall ? j.xt0 : j.x, *o = tall ? j.x : j.xt0;
    const uint32_t ldn = tall ? j.lds : j.ldn, ldo = tall ? j.ldn : j.lds;
    const int line = tid >> 2, k = (tid & 3) * 16;
    float v[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) v[e] = t[line][k + e];
    store16<SPLIT>(n + int64_t(r0 + line) * ldn, c0 + k, v);
#pragma unroll
    for (int e = 0; e < 16; ++e) v[e] = t[k + e][line];
    store16<SPLIT>(o + int64_t(c0 + line) * ldo, r0 + k, v);
}

// ---- the products ------------------------------------------------------------------------------------------------------------
enum { GRAM, POLY, APPLY, LAST };

struct Factors {
    float acc, a, diag;   // what the accumulator, A's entry and the diagonal count for in the result
    float keep;           // LAST: 1 - lr * weight_decay (cp_ortho_step)
    int xt;               // which X^T is read
};

template <int PHASE, bool SPLIT>
__global__ void __launch_bounds__(256) k_ortho_product(Jobs js, Factors f) {
    constexpr int BM = kTile, BN = kTile, T = 256, WI = 4, WJ = 4;
    constexpr bool SYM = PHASE == GRAM || PHASE == POLY;
    __shared__ alignas(1024) char a0[BM * 128], a1[BM * 128], b0[BN * 128], b1[BN * 128];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave >> 1, wn = wave & 1;
    const int id = nt::xcd_order(blockIdx.x, SYM ? js.total_sym : js.total_apply);
    const Job &j = js.job[find_job(js, id, SYM ? &Job::first_sym : &Job::first_apply)];
    const bool tall = j.rows > j.cols;
    const bool swap = PHASE == LAST && tall;   // the result's rows are G's rows: four consecutive numbers lie in one of them
    const char *xt = f.xt ? j.xt1 : j.xt0;
    const char *pa = PHASE == GRAM ? j.x : PHASE == POLY ? j.a : swap ? xt : j.b;
    const char *pb = PHASE == GRAM ? j.x : PHASE == POLY ? j.a : swap ? j.b : xt;
    const uint32_t ld = PHASE == GRAM ? j.ldn : j.lds;
    const int steps = int(ld >> 7);
    int tm, tn;
    if (SYM) {
        const int t = id - j.first_sym;
        tm = int((sqrtf(8.f * t + 1.f) - 1.f) * 0.5f);
        while (tm * (tm + 1) / 2 > t) --tm;
        while ((tm + 1) * (tm + 2) / 2 <= t) ++tm;
        tn = t - tm * (tm + 1) / 2;
    } else {
        const int t = id - j.first_apply, tiles_m = (swap ? j.np : j.mp) / BM;
        tm = t % tiles_m;
        tn = t / tiles_m;
    }
    const int i0 = tm * BM, j0 = tn * BN;
    nt::Loader<BM, T> la;
    nt::Loader<BN, T> lb;
    la.init(pa + int64_t(i0) * ld, ld, BM, tid);
    lb.init(pb + int64_t(j0) * ld, ld, BN, tid);
    f4 acc[WI][WJ];
#pragma unroll
    for (int i = 0; i < WI; ++i)
#pragma unroll
        for (int k = 0; k < WJ; ++k) acc[i][k] = f4{0.f, 0.f, 0.f, 0.f};
    const int ra = wm * WI * 16, rb = wn * WJ * 16;
    auto fetch = [&](int k, char *a, char *b) {
        la.issue(k, a, wave);
        lb.issue(k, b, wave);
    };
    fetch(0, a0, b0);
    for (int k = 0; k < steps; k += 2) {
        nt::stage_barrier();
        if (k + 1 < steps) fetch(k + 1, a1, b1);
        nt::products16<WI, WJ>(a0 + ra * 128, b0 + rb * 128, lane, acc, SPLIT);
        if (k + 1 >= steps) break;
        nt::stage_barrier();
        if (k + 2 < steps) fetch(k + 2, a0, b0);
        nt::products16<WI, WJ>(a1 + ra * 128, b1 + rb * 128, lane, acc, SPLIT);
    }
#pragma unroll
    for (int wi = 0; wi < WI; ++wi) {
        const int i = i0 + ra + wi * 16 + (lane & 15);
#pragma unroll
        for (int wj = 0; wj < WJ; ++wj) {
            const int c = j0 + rb + wj * 16 + (lane >> 4) * 4;
            f4 v = acc[wi][wj] * f.acc;
            if (PHASE == POLY) {
                v += load4<SPLIT>(j.a + int64_t(i) * j.lds, c) * f.a;
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (c + r == i) v[r] += f.diag;
            }
            if (SYM) {
                char *out = PHASE == GRAM ? j.a : j.b;
                store4<SPLIT>(out + int64_t(i) * j.lds, c, v);
                if (tm != tn) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) store1<SPLIT>(out + int64_t(c + r) * j.lds, i, v[r]);
                }
            } else if (PHASE == APPLY) {
                store4<SPLIT>(j.x + int64_t(i) * j.ldn, c, v);
                char *out = f.xt ? j.xt0 : j.xt1;
#pragma unroll
                for (int r = 0; r < 4; ++r) store1<SPLIT>(out + int64_t(c + r) * j.lds, i, v[r]);
            } else if (i < j.rows) {
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    if (c + r >= j.cols) break;
                    const int64_t at = i * j.ldo + c + r;
                    float o = v[r];
                    if (j.M) o = f.keep * load_as_float(j.out, j.o_dtype, at) - j.lr * o;
                    store_as(j.out, j.o_dtype, at, o);
                }
            }
        }
    }
}

// ---- host --------------------------------------------------------------------------------------------------------------------
struct Plan {
    int steps = 0;
    double coef[kMaxSteps][3];
    double sx[kMaxSteps + 1], sa[kMaxSteps], sb[kMaxSteps];   // scales of X before step k, of A and B in it
};

// the power of two that puts a bound at 2^14
double scale_for(double bound) {
    int e;
    std::frexp(std::max(bound, 1e-30), &e);
    return std::ldexp(1.0, std::min(14 - e, 30));
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

// one matrix that is written, for the overlap check
struct Written {
    uintptr_t at;
    int64_t ld, rows, cols;
    size_t size;
    uintptr_t end() const { return at + (size_t(rows - 1) * ld + cols) * size; }
};

// whether two matrices share an element: rows of one stride interleave as column ranges of one wider matrix do
bool overlap(const Written &p, const Written &q) {
    if (p.at >= q.end() || q.at >= p.end()) return false;
    if (p.ld != q.ld || p.size != q.size) return true;
    const Written &lo = p.at <= q.at ? p : q, &hi = p.at <= q.at ? q : p;
    if ((hi.at - lo.at) % lo.size) return true;
    const int64_t d = int64_t((hi.at - lo.at) / lo.size) % lo.ld;   // hi's first column, counted from lo's
    return d < lo.cols || d + hi.cols > lo.ld;
}

struct Request {
    const void *G;
    float *M;
    void *out;
    int64_t ldg, ldm, ldo;
    int rows, cols, g_dtype, o_dtype;
    double gamma;
};

int check_requests(cp_ctx *ctx, const std::vector<Request> &rq, bool step) {
    std::vector<Written> w;
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
        if (int64_t(std::min(r.rows, r.cols) + 127) / 128 > 512)
            return cp_set_error(ctx, CP_ERR_UNSUPPORTED, "job %d: shorter side above 65536", int(k));
        w.push_back({uintptr_t(r.out), r.ldo, r.rows, r.cols, type_size(r.o_dtype)});
        const Written g = {uintptr_t(r.G), r.ldg, r.rows, r.cols, type_size(r.g_dtype)};
        if (step) {
            w.push_back({uintptr_t(r.M), r.ldm, r.rows, r.cols, 4});
            if (overlap(g, w.back()) || overlap(g, w[w.size() - 2]))
                return cp_set_error(ctx, CP_ERR_ARG, "job %d: G overlaps M or W", int(k));
        }
    }
    std::sort(w.begin(), w.end(), [](const Written &p, const Written &q) { return p.at < q.at; });
    for (size_t i = 0; i < w.size(); ++i)
        for (size_t k = i + 1; k < w.size() && w[k].at < w[i].end(); ++k)
            if (overlap(w[i], w[k])) return cp_set_error(ctx, CP_ERR_ARG, "two outputs of the call overlap");
    return CP_OK;
}

bool is_split(const Request &r) { return r.o_dtype != CP_BF16; }

int64_t padded(int v) { return (int64_t(v) + kTile - 1) / kTile * kTile; }

size_t job_bytes(const Request &r) {
    if (!r.rows || !r.cols) return 0;
    const size_t e = is_split(r) ? 4 : 2;
    const size_t mp = padded(std::min(r.rows, r.cols)), np = padded(std::max(r.rows, r.cols));
    return cp_align_up(kPartials * sizeof(double) + e * (3 * mp * np + 2 * mp * mp), 256);
}

size_t call_bytes(const std::vector<Request> &rq) {
    size_t b = 0;
    for (const Request &r : rq) b += job_bytes(r);
    return b;
}

// the scratch of a call: the caller's, or the context's own (which a captured call must not use: the graph outlives it)
int scratch(cp_ctx *ctx, void *ws, size_t ws_bytes, size_t need, char **out) {
    if (ws) {
        if (uintptr_t(ws) % 256) return cp_set_error(ctx, CP_ERR_ARG, "workspace is not 256-byte aligned");
        if (ws_bytes < need) return cp_set_error(ctx, CP_ERR_ARG, "workspace of %zu bytes, %zu needed", ws_bytes, need);
        *out = static_cast<char *>(ws);
        return CP_OK;
    }
    hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
    CP_HIP(ctx, hipStreamIsCapturing(ctx->stream, &st));
    if (st != hipStreamCaptureStatusNone)
        return cp_set_error(ctx, CP_ERR_ARG, "a captured call needs a workspace of its own (%zu bytes)", need);
    CP_TRY(cp_arena_reserve(ctx, need));
    *out = static_cast<char *>(cp_arena_take(ctx, need));
    return *out ? CP_OK : cp_set_error(ctx, CP_ERR_NOMEM, "arena");
}

template <bool SPLIT>
void launch_all(cp_ctx *ctx, const std::vector<Jobs> &launches, const Plan &pl, float momentum, int nesterov, double eps,
                float keep) {
    hipStream_t st = ctx->stream;
    for (int k = 0; k < pl.steps; ++k) {
        const double a = pl.coef[k][0], b = pl.coef[k][1], c = pl.coef[k][2];
        const double sx = pl.sx[k], sa = pl.sa[k], sb = pl.sb[k];
        Factors f = {};
        f.xt = k & 1;
        for (const Jobs &js : launches) {
            f.acc = float(sa / (sx * sx));
            k_ortho_product<GRAM, SPLIT><<<js.total_sym, 256, 0, st>>>(js, f);
        }
        for (const Jobs &js : launches) {
            f.acc = float(c * sb / (sa * sa));
            f.a = float(b * sb / sa);
            f.diag = float(a * sb);
            k_ortho_product<POLY, SPLIT><<<js.total_sym, 256, 0, st>>>(js, f);
        }
        for (const Jobs &js : launches) {
            if (k + 1 < pl.steps) {
                f.acc = float(pl.sx[k + 1] / (sb * sx));
                k_ortho_product<APPLY, SPLIT><<<js.total_apply, 256, 0, st>>>(js, f);
            } else {
                f.acc = float(1.0 / (sb * sx));
                f.keep = keep;
                k_ortho_product<LAST, SPLIT><<<js.total_apply, 256, 0, st>>>(js, f);
            }
        }
    }
}

int run(cp_ctx *ctx, const std::vector<Request> &rq, const Plan &pl, double lr, double momentum, int nesterov, double decay,
        double eps, void *ws, size_t ws_bytes) {
    const size_t need = call_bytes(rq);
    if (!need) return CP_OK;
    CP_HIP(ctx, hipSetDevice(ctx->device));
    char *at = nullptr;
    CP_TRY(scratch(ctx, ws, ws_bytes, need, &at));
    std::vector<Jobs> launches[2];
    for (const Request &r : rq) {
        if (!r.rows || !r.cols) continue;
        std::vector<Jobs> &ls = launches[is_split(r)];
        if (ls.empty() || ls.back().n == kJobs) ls.push_back(Jobs());
        Jobs &js = ls.back();
        Job &j = js.job[js.n++];
        j = {};
        const size_t e = is_split(r) ? 4 : 2;
        const size_t mp = padded(std::min(r.rows, r.cols)), np = padded(std::max(r.rows, r.cols));
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
        j.g_dtype = r.g_dtype;
        j.o_dtype = r.o_dtype;
        j.lr = float(lr * r.gamma);
        j.part = reinterpret_cast<double *>(at);
        j.x = at + kPartials * sizeof(double);
        j.xt0 = j.x + mp * np * e;
        j.xt1 = j.xt0 + mp * np * e;
        j.a = j.xt1 + mp * np * e;
        j.b = j.a + mp * mp * e;
        at += job_bytes(r);
        const int tm = int(mp / kTile), tn = int(np / kTile);
        j.first_sym = js.total_sym;
        js.total_sym += tm * (tm + 1) / 2;
        j.first_apply = js.total_apply;
        js.total_apply += tm * tn;
        j.first_load = js.total_load;
        js.total_load += int((mp / 64) * (np / 64));
    }
    for (int s = 0; s < 2; ++s)
        for (const Jobs &js : launches[s])
            k_ortho_norm<<<dim3(kPartials, js.n), 256, 0, ctx->stream>>>(js, float(momentum), nesterov);
    for (const Jobs &js : launches[0])
        k_ortho_load<false><<<js.total_load, 256, 0, ctx->stream>>>(js, float(momentum), nesterov, eps, float(pl.sx[0]));
    for (const Jobs &js : launches[1])
        k_ortho_load<true><<<js.total_load, 256, 0, ctx->stream>>>(js, float(momentum), nesterov, eps, float(pl.sx[0]));
    const float keep = float(1.0 - lr * decay);
    launch_all<false>(ctx, launches[0], pl, float(momentum), nesterov, eps, keep);
    launch_all<true>(ctx, launches[1], pl, float(momentum), nesterov, eps, keep);
    CP_LAUNCH_CHECK(ctx);
    return CP_OK;
}

int take_jobs(cp_ctx *ctx, int n, const cp_ortho_job *jobs, std::vector<Request> &rq) {
    if (n < 0 || (n && !jobs)) return cp_set_error(ctx, CP_ERR_ARG, "jobs");
    for (int i = 0; i < n; ++i) {
        const cp_ortho_job &q = jobs[i];
        rq.push_back({q.G, nullptr, q.O, q.ldg, 0, q.ldo, q.rows, q.cols, q.g_dtype, q.o_dtype, 1.0});
    }
    return check_requests(ctx, rq, false);
}

int take_jobs(cp_ctx *ctx, int n, const cp_ortho_step_job *jobs, std::vector<Request> &rq) {
    if (n < 0 || (n && !jobs)) return cp_set_error(ctx, CP_ERR_ARG, "jobs");
    for (int i = 0; i < n; ++i) {
        const cp_ortho_step_job &q = jobs[i];
        rq.push_back({q.G, q.M, q.W, q.ldg, q.ldm, q.ldw, q.rows, q.cols, q.g_dtype, q.w_dtype, q.gamma});
    }
    return check_requests(ctx, rq, true);
}

template <typename J>
int workspace(int n, const J *jobs, int steps, const double *coef, double eps, size_t *bytes) {
    if (!bytes) return CP_ERR_ARG;
    try {
        Plan pl;
        std::vector<Request> rq;
        CP_TRY(make_plan(nullptr, steps, coef, eps, pl));
        CP_TRY(take_jobs(nullptr, n, jobs, rq));
        *bytes = call_bytes(rq);
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
        CP_TRY(make_plan(ctx, steps, coef, eps, pl));
        CP_TRY(take_jobs(ctx, n_jobs, jobs, rq));
        return run(ctx, rq, pl, 0.0, 0.0, 0, 0.0, eps, ws, ws_bytes);
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
        CP_TRY(make_plan(ctx, steps, coef, eps, pl));
        CP_TRY(take_jobs(ctx, n_jobs, jobs, rq));
        return run(ctx, rq, pl, lr, momentum, nesterov != 0, weight_decay, eps, ws, ws_bytes);
    } catch (...) {
        return cp_set_error(ctx, CP_ERR_NOMEM, "host memory");
    }
}
