// The tile loop that the 16-bit and 8-bit matrix products share (ortho.hip, blocks8.hip; gfx950).
//
// C[i, j] = sum_k A[i, k] B[j, k]: both operands hold k contiguously ("NT").  A K step is always 128 BYTES of every row,
// whatever the type: 64 fp16 numbers, 32 fp16 pairs (32 high parts, then their 32 low parts), or 128 8-bit numbers -- one
// block of a common scale.  So one loader, one LDS layout and one schedule serve all three.
//
// LDS: a row's 128 bytes are eight 16-byte chunks, and chunk c of row r is kept at place c ^ (r & 7): the sixteen lanes that
// read one chunk column of sixteen rows then hit all banks evenly, with no padding -- which the direct global -> LDS loads
// could not write (their destination is linear in the lane).  The swizzle is applied to the SOURCE address instead.
//
// The accumulators come out of the matrix instruction as (four consecutive rows, one column) per lane, so B feeds its row side
// and A its column side: a lane then owns four consecutive j of one i, a vector store in row-major C.
//
// STAGES LDS stages, each in its own __shared__ array so that the compiler can tell a load into one from reads of the others
// (and inserts no wait between them); one barrier per K step, behind which the loads of a step STAGES - 1 ahead are issued.
// A tile that fills the chip alone needs two stages (a step of 256 x 256 takes 3500 cycles, a load from a cold L2 2000); small
// tiles take four.  128 x 128 with four stages and one workgroup to a CU instead of two with two: no faster where tiles are few
// (8-bit 5000 x 512 x 4005: 28.1 against 29.4 us), slower where there are many (20000 x 4005 x 512: 152 against 109).
//
// What bounds it: the matrix instructions.  A 256 x 256 step of fp16 takes 1.55-1.7 us with its loads, 1.49 without any (1440
// TFLOP/s of the chip, which lowers its clock under such a load; a large library product reaches 1570-1590), the loads alone
// 0.96.  128 x 128 takes 0.52 (a third more for its part of 256 x 256: the same LDS reads feed half the products), 64 x 64 0.18.
//
// A tile with a long k and few tiles beside it is cut into pieces of k (their number follows from the product's shape alone)
// that several workgroups form; the one that arrives last adds them in the order of k.  The result does not depend on who
// that is, and nobody waits for anybody.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

namespace nt {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef int i8v __attribute__((ext_vector_type(8)));
typedef int i4v __attribute__((ext_vector_type(4)));

// the same, at any element's address: the vector loads and stores of this chip take any alignment
typedef __bf16 b4 __attribute__((ext_vector_type(4)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef f4 f4u __attribute__((aligned(4)));
typedef h4 h4u __attribute__((aligned(2)));
typedef h8 h8u __attribute__((aligned(2)));
typedef b4 b4u __attribute__((aligned(2)));
typedef b8 b8u __attribute__((aligned(2)));

// Access through a pointer that was itself read from memory: for all that the compiler knows it could point into LDS, and such
// an access would count, and be waited for, as one of LDS too.
template <class V>
__device__ __forceinline__ V take_from(const void *p) {
    return *(const __attribute__((address_space(1))) V *)p;
}
template <class V>
__device__ __forceinline__ void put_to(void *p, V v) {
    *(__attribute__((address_space(1))) V *)p = v;
}

__device__ __forceinline__ void load_lds16(const char *g, char *l) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)g,
                                     (__attribute__((address_space(3))) void *)l, 16, 0, 0);
}
__device__ __forceinline__ void load_lds4(const float *g, float *l) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)g,
                                     (__attribute__((address_space(3))) void *)l, 4, 0, 0);
}

// at most N of this wave's loads are still under way, its LDS reads are done, and both hold for the other waves
template <int N>
__device__ __forceinline__ void stage_barrier() {
    static_assert(N < 64, "vmcnt has six bits");
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0070 | (N & 15) | ((N >> 4) << 14));   // vmcnt(N) lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}
template <int STAGES, int U, class Step>
__device__ __forceinline__ void rest(int n, Step step) {
    if constexpr (U < STAGES - 1) {
        if (n <= U) return;
        step(std::integral_constant<int, U>());
        rest<STAGES, U + 1>(n, step);
    }
}

// `steps` K steps: fetch(k, stage, part, parts) issues a share of a step's loads (LOADS per thread in all), compute(stage,
// between) uses a step's and calls between(i) among its products, where the first PARTS calls issue the shares.  Ends with a barrier.
// Every path through the loop issues the same loads (the last step's again where there is no further one): the compiler
// counts them along paths, not values, and would wait for all of them otherwise.
template <int STAGES, int LOADS, int PARTS, class Fetch, class Compute>
__device__ __forceinline__ void pipeline(char *const (&st)[8], int steps, Fetch fetch, Compute compute) {
    const int last = steps - 1;
    auto step = [&](int k, int u) {
        stage_barrier<LOADS *(STAGES - 2)>();
        const int next = k + STAGES - 1, n = next < last ? next : last;
        compute(st[u], [&](int i) { if (i < PARTS) fetch(n, st[(u + STAGES - 1) % STAGES], i, PARTS); });
    };
#pragma unroll
    for (int u = 0; u < STAGES - 1; ++u) fetch(u < last ? u : last, st[u], 0, 1);
    int k = 0;
    // whole rounds of the stages, then the rest: a loop that can be left in its middle keeps the accumulators twice
    for (; k + STAGES <= steps; k += STAGES) {
#pragma unroll
        for (int u = 0; u < STAGES; ++u) step(k + u, u);
    }
    rest<STAGES, 0>(steps - k, [&](auto u) { step(k + u.value, u.value); });
    stage_barrier<0>();
}
// the stages' arrays, `bytes` each
#define NT_STAGES(name, n, bytes)                                                                                        \
    __shared__ alignas(1024) char name##0[bytes], name##1[(n) > 1 ? (bytes) : 16], name##2[(n) > 2 ? (bytes) : 16],      \
        name##3[(n) > 3 ? (bytes) : 16], name##4[(n) > 4 ? (bytes) : 16], name##5[(n) > 5 ? (bytes) : 16],               \
        name##6[(n) > 6 ? (bytes) : 16], name##7[(n) > 7 ? (bytes) : 16];                                                \
    char *const name[8] = {name##0, name##1, name##2, name##3, name##4, name##5, name##6, name##7}

// A tile shape: BM x BN by NWM x NWN waves
template <int BM_, int BN_, int NWM_, int NWN_, int STAGES_>
struct Tile {
    static constexpr int BM = BM_, BN = BN_, NWM = NWM_, NWN = NWN_, STAGES = STAGES_;
    static constexpr int T = 64 * NWM * NWN, WI = BM / NWM / 16, WJ = BN / NWN / 16;
    static constexpr int STAGE = (BM + BN) * 128, LOADS = STAGE / 16 / T;
    static constexpr int PARTS = WI >= 6 ? 4 : 1;
};
typedef Tile<256, 256, 2, 4, 2> Large;    // 132 KB of LDS, one workgroup to a CU
typedef Tile<192, 256, 2, 4, 2> Flat;     // 112 KB, one: where tiles of 256 leave many CUs idle
typedef Tile<128, 128, 2, 2, 2> Medium;   // 64 KB, two
typedef Tile<64, 64, 2, 2, 4> Small;      // 64 KB, two

// One operand's share of the loads: ROWS rows of 128 bytes by THREADS threads, 16 bytes each
template <int ROWS, int THREADS>
struct Loader {
    static constexpr int N = ROWS * 8 / THREADS;
    const char *base;
    uint32_t off[N];
    // g: row 0 of the tile; rows from `valid` on are not there (their places repeat the last one; the caller drops what
    // they give).  255 * ld < 2^32 by the callers' limits on ld.
    __device__ __forceinline__ void init(const char *g, uint32_t ld, int valid, int tid) {
        base = g;
        const int chunk = (tid & 7) ^ ((tid >> 3) & 7);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            int r = i * (THREADS / 8) + (tid >> 3);
            r = r < valid ? r : valid - 1;
            off[i] = uint32_t(r) * ld + chunk * 16;
        }
    }
    // the part-th of `parts` shares of a step's loads
    __device__ __forceinline__ void issue(int64_t step, char *lds, int wave, int part, int parts) const {
        const char *g = base + step * 128;
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (i * parts / N == part) load_lds16(g + off[i], lds + (i * THREADS + wave * 64) * 16);
    }
};

// per-lane byte offset of chunk (lane >> 4) + 4 h of row (lane & 15) of a 16-row group
__device__ __forceinline__ int frag_off(int lane, int h) { return (lane & 15) * 128 + ((((lane >> 4) + 4 * h) ^ (lane & 7)) << 4); }

// A step's products.  A row group's fragments are read one group ahead of their use, and the next step's loads are issued
// among the products (`between`): the barriers of the compiler's scheduler keep both where they stand, or it gathers the reads
// at the top of the step, where both waves of a SIMD then wait for them at once (4096 x 16384 times 4096^2 in fp16: 480 us with
// them, 568 without).
#define NT_STAY() __builtin_amdgcn_sched_barrier(0)

template <int WI, int WJ, bool SPLIT, class Between>
__device__ __forceinline__ void products16(const char *a, const char *b, int lane, f4 (&acc)[WI][WJ], Between between) {
    const int o0 = frag_off(lane, 0), o1 = frag_off(lane, 1);
    h8 b0[WJ], b1[WJ], a0[2], a1[2];
    a0[0] = *reinterpret_cast<const h8 *>(a + o0);
    a1[0] = *reinterpret_cast<const h8 *>(a + o1);
#pragma unroll
    for (int j = 0; j < WJ; ++j) {
        b0[j] = *reinterpret_cast<const h8 *>(b + j * 2048 + o0);
        b1[j] = *reinterpret_cast<const h8 *>(b + j * 2048 + o1);
    }
    NT_STAY();
#pragma unroll
    for (int i = 0; i < WI; ++i) {
        const int u = i & 1;
        if (i + 1 < WI) {
            a0[u ^ 1] = *reinterpret_cast<const h8 *>(a + (i + 1) * 2048 + o0);
            a1[u ^ 1] = *reinterpret_cast<const h8 *>(a + (i + 1) * 2048 + o1);
        }
        between(i);
        NT_STAY();
        if (SPLIT) {   // (high + low) (high + low) without low * low, which is below the pair's own rounding
#pragma unroll
            for (int j = 0; j < WJ; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(b1[j], a0[u], acc[i][j], 0, 0, 0);
#pragma unroll
            for (int j = 0; j < WJ; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(b0[j], a1[u], acc[i][j], 0, 0, 0);
#pragma unroll
            for (int j = 0; j < WJ; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(b0[j], a0[u], acc[i][j], 0, 0, 0);
        } else {
#pragma unroll
            for (int j = 0; j < WJ; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(b0[j], a0[u], acc[i][j], 0, 0, 0);
#pragma unroll
            for (int j = 0; j < WJ; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(b1[j], a1[u], acc[i][j], 0, 0, 0);
        }
        NT_STAY();
    }
}

// sixteen 8-bit numbers as fp16, which holds either type's values exactly
template <int FMT>
__device__ __forceinline__ void widen(i4v q, h8 (&w)[2]) {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int d = 0; d < 4; ++d)
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            h2 p;
            if (FMT == 0) p = s ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(q[d], 1.f, true) : __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(q[d], 1.f, false);
            else p = s ? __builtin_amdgcn_cvt_scalef32_pk_f16_bf8(q[d], 1.f, true) : __builtin_amdgcn_cvt_scalef32_pk_f16_bf8(q[d], 1.f, false);
            w[d >> 1][(d & 1) * 4 + s * 2] = p[0];
            w[d >> 1][(d & 1) * 4 + s * 2 + 1] = p[1];
        }
}

// One block of 128 of sixteen rows as a lane holds it: two chunks of 8-bit numbers, or the same widened
template <int FMT, bool WIDE>
struct Frag8 {
    i8v v;
    h8 w[4];
    __device__ __forceinline__ void load(const char *rows, int o0, int o1) {
        set(*reinterpret_cast<const i4v *>(rows + o0), *reinterpret_cast<const i4v *>(rows + o1));
    }
    __device__ __forceinline__ void set(i4v c0, i4v c1) {
        if (WIDE) {
            widen<FMT>(c0, reinterpret_cast<h8(&)[2]>(w[0]));
            widen<FMT>(c1, reinterpret_cast<h8(&)[2]>(w[2]));
        } else {
            v = __builtin_shufflevector(c0, c1, 0, 1, 2, 3, 4, 5, 6, 7);
        }
    }
};

// a scale as a power of two, in the form of the matrix instruction's own scales, and the rest (a user's scale may be anything)
__device__ __forceinline__ float part_of(float scale, int &power) {
    const uint32_t e = __float_as_uint(scale) >> 23 & 0xff;
    power = int(min(max(e, 1u), 254u));
    return ldexpf(scale, 127 - power);
}

// the products of one block of sixteen rows of A and of B, from zero.  SCALED: times 2^(power - 127)
template <int FA, int FB, bool WIDE, bool SCALED = false>
__device__ __forceinline__ f4 block_product(const Frag8<FA, WIDE> &a, const Frag8<FB, WIDE> &b, int power = 127) {
    f4 z = {0.f, 0.f, 0.f, 0.f};
    if (WIDE) {
#pragma unroll
        for (int h = 0; h < 4; ++h) z = __builtin_amdgcn_mfma_f32_16x16x32_f16(b.w[h], a.w[h], z, 0, 0, 0);
    } else if constexpr (SCALED) {
        z = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b.v, a.v, z, FB, FA, 0, power, 0, 127);
    } else {
        z = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b.v, a.v, z, FB, FA, 0, 0, 0, 0);
    }
    return z;
}

// The 8-bit step: the products of one block of 128 start from zero and join the accumulators times both blocks' scales.
// sa [16 WI] and sb ([16 WJ], or one value where COMMON) are this wave's scales of the step.  The product of two scales may lie
// outside float32 where the result does not (operands of 1e-19; blocks of 1e30 and 1e14 that share no column): a sum is taken
// times one, then times the other.  COMMON on the 8-bit instructions has no time for a second product (8192^3: 505 us instead of 430): there the
// instruction takes the power of two of B's scale, and what is left of it joins A's (439 us).
// WIDE: the 8-bit matrix instructions align the eight products of a group to the largest and drop what lies below 2^-13 of
// its power of two (measured: 2^16 + 4 gives 2^16 within a group, 2^16 + 8 is exact, and across groups all of float32 counts).
// A bfloat16 result rounds off 2^-8 and takes them as they are; float32 and fp16 results are formed with the fp16
// instructions, which keep float32's bits at half the rate.
template <int WI, int WJ, int FA, int FB, bool COMMON, bool WIDE, class Between>
__device__ __forceinline__ void products8(const char *a, const char *b, const float *sa, const float *sb, int lane,
                                          f4 (&acc)[WI][WJ], Between between) {
    const int o0 = frag_off(lane, 0), o1 = frag_off(lane, 1);
    Frag8<FB, WIDE> bf[WJ];
    Frag8<FA, WIDE> af[2];
    f4 sj[WJ], t[2][WJ];
    float si[2];
    constexpr bool SCALED = COMMON && !WIDE;
    int power = 127;
    float common = COMMON ? sb[0] : 1.f;
    if constexpr (SCALED) common = part_of(common, power);
    auto join = [&](int i, int j) {   // a row group's products join the accumulators while the next one's are formed
#pragma unroll
        for (int r = 0; r < 4; ++r)
            acc[i][j][r] = SCALED ? fmaf(t[i & 1][j][r], si[i & 1], acc[i][j][r])
                                  : fmaf(t[i & 1][j][r] * si[i & 1], COMMON ? common : sj[j][r], acc[i][j][r]);
    };
    af[0].load(a, o0, o1);
    si[0] = sa[lane & 15] * (SCALED ? common : 1.f);
#pragma unroll
    for (int j = 0; j < WJ; ++j) {
        bf[j].load(b + j * 2048, o0, o1);
        if (!COMMON) sj[j] = *reinterpret_cast<const f4 *>(sb + j * 16 + (lane >> 4) * 4);
    }
    NT_STAY();
#pragma unroll
    for (int i = 0; i < WI; ++i) {
        const int u = i & 1;
        float next = 0.f;
        if (i + 1 < WI) {
            af[u ^ 1].load(a + (i + 1) * 2048, o0, o1);
            if (COMMON) next = sa[(i + 1) * 16 + (lane & 15)];   // (registers are short where every column has its scale)
        }
        between(i);
        NT_STAY();
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int j = 0; j < WJ; ++j) {
            t[u][j] = block_product<FA, FB, WIDE, SCALED>(af[u], bf[j], power);
            if (i > 0) join(i - 1, j);
            // a matrix instruction, then the vector instructions that fit beside it
            __builtin_amdgcn_sched_group_barrier(0x008, WIDE ? 4 : 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x002, SCALED ? 4 : 8, 0);
        }
        __builtin_amdgcn_s_setprio(0);
        if (i + 1 < WI) si[u ^ 1] = COMMON ? next * (SCALED ? common : 1.f) : sa[(i + 1) * 16 + (lane & 15)];
        NT_STAY();
    }
#pragma unroll
    for (int j = 0; j < WJ; ++j) join(WI - 1, j);
}

// ---- tiles that several workgroups share ---------------------------------------------------------------------------------
// Parts are stored through to where every XCD sees them (sc1), waited for, and announced by a relaxed counter; the last to
// arrive reads them the same way.  No fence is needed around these.
typedef unsigned int u4v __attribute__((ext_vector_type(4)));
constexpr int kSc1 = 16;
__device__ __forceinline__ __amdgpu_buffer_rsrc_t slot_of(float *p, int bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(p, 0, bytes, 0x00027000);
}
__device__ __forceinline__ void put(__amdgpu_buffer_rsrc_t slot, int at, f4 v) {
    u4v q;
    __builtin_memcpy(&q, &v, 16);
    __builtin_amdgcn_raw_buffer_store_b128(q, slot, at, 0, kSc1);
}
__device__ __forceinline__ f4 take(__amdgpu_buffer_rsrc_t slot, int at) {
    const u4v q = __builtin_amdgcn_raw_buffer_load_b128(slot, at, 0, kSc1);
    f4 v;
    __builtin_memcpy(&v, &q, 16);
    return v;
}

// This workgroup's acc is one of n pieces of a tile; piece q's slot lies at parts + q * apart tiles' sizes.  Returns whether
// this workgroup holds the whole tile in acc now.  `flag`: one int of LDS, `count`: the tile's counter, zero before and after.
template <int T, int WI, int WJ>
__device__ __forceinline__ bool join(f4 (&acc)[WI][WJ], int piece, int n, float *parts, int64_t apart, int *count, int *flag, int tid) {
    constexpr int SLOT = T * WI * WJ * 4;   // numbers
    const __amdgpu_buffer_rsrc_t mine = slot_of(parts + piece * apart * SLOT, SLOT * 4);
#pragma unroll
    for (int i = 0; i < WI; ++i)
#pragma unroll
        for (int j = 0; j < WJ; ++j) put(mine, ((i * WJ + j) * T + tid) * 16, acc[i][j]);
    stage_barrier<0>();
    if (tid == 0) {
        const int seen = __hip_atomic_fetch_add(count, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        const bool last = seen == n - 1;
        if (last) __hip_atomic_store(count, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        *flag = last;
    }
    __syncthreads();
    const bool last = *flag != 0;
    __syncthreads();
    if (!last) return false;
    for (int q = 0; q < n; ++q) {
        const __amdgpu_buffer_rsrc_t p = slot_of(parts + q * apart * SLOT, SLOT * 4);
#pragma unroll
        for (int i = 0; i < WI; ++i)
#pragma unroll
            for (int j = 0; j < WJ; ++j) {
                const f4 v = take(p, ((i * WJ + j) * T + tid) * 16);
                acc[i][j] = q == 0 ? v : acc[i][j] + v;
            }
    }
    return true;
}

// ---- results ---------------------------------------------------------------------------------------------------------------
// A lane's accumulators are four numbers of one row: written from there, a row gets 32 or 64 bytes at a time, which costs twice
// what whole lines cost.  So a wave passes its part of the tile through the LDS that the stages have left (12 or 16 KB a wave, its
// own: no barrier), up to 64 x 64 float32 at a time, and reads it back as eight neighbours of a row or of a column.  The
// 16-byte chunks of row r lie at chunk ^ key(r), so that writes and both kinds of reads hit all banks evenly.
template <int WI, int WJ>
struct Patch {
    static constexpr int COLS = WJ * 16, ROWS = WI % 4 == 0 ? 64 : WI % 3 == 0 ? 48 : WI * 16, PASSES = WI * 16 / ROWS;
    static constexpr int EACH_WAVE = ROWS * COLS * 4 <= 12288 ? 12288 : 16384;   // bytes of LDS
    static constexpr int EIGHTS = ROWS * COLS / 512;   // groups of eight numbers to a lane
    static_assert(ROWS * COLS * 4 <= EACH_WAVE && ROWS * PASSES == WI * 16 && ROWS * COLS % 512 == 0, "");
    char *lds;
    int lane;
    template <class CFG>
    __device__ __forceinline__ static Patch of(char *const (&st)[8], int wave, int lane) {
        constexpr int EACH = CFG::NWM * CFG::NWN / CFG::STAGES;
        static_assert(CFG::STAGE >= EACH * EACH_WAVE, "");
        typedef __attribute__((address_space(3))) char *Lds;
        uint32_t from = 0;
#pragma unroll
        for (int k = 0; k < CFG::STAGES; ++k) {
            uint32_t s = uint32_t(uintptr_t(Lds(st[k])));
            asm("" : "+s"(s));   // (the compiler would look these up in a table, which it cannot place)
            from = wave / EACH == k ? s : from;
        }
        return {(char *)(Lds(uintptr_t(from + wave % EACH * EACH_WAVE))), lane};
    }
    __device__ __forceinline__ static void order() {   // a wave's LDS accesses run in order: only the compiler has to be told
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
    __device__ __forceinline__ char *at(int r, int chunk) const { return lds + r * COLS * 4 + ((chunk ^ ((r ^ (r >> 3)) & (COLS / 4 - 1))) << 4); }
    // rows ROWS * pass .. of the wave's part, times a factor
    __device__ __forceinline__ void put(const f4 (&acc)[WI][WJ], int pass, float factor) const {
        order();
#pragma unroll
        for (int i = 0; i < ROWS / 16; ++i)
#pragma unroll
            for (int j = 0; j < WJ; ++j)
                *reinterpret_cast<f4 *>(at(i * 16 + (lane & 15), j * 4 + (lane >> 4))) = acc[pass * (ROWS / 16) + i][j] * factor;
        order();
    }
    // four numbers of row r from column c (u < 2 EIGHTS): float32 results, 16 bytes a lane
    __device__ __forceinline__ f4 four_of_row(int u, int &r, int &c) const {
        r = (u * 64 + lane) / (COLS / 4);
        c = (u * 64 + lane) % (COLS / 4) * 4;
        return *reinterpret_cast<const f4 *>(at(r, c / 4));
    }
    // group u: eight numbers of row r from column c, or of column c from row r
    __device__ __forceinline__ void of_row(int u, int &r, int &c, float (&v)[8]) const {
        r = (u * 64 + lane) / (COLS / 8);
        c = (u * 64 + lane) % (COLS / 8) * 8;
        const f4 a = *reinterpret_cast<const f4 *>(at(r, c / 4)), b = *reinterpret_cast<const f4 *>(at(r, c / 4 + 1));
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = a[e], v[e + 4] = b[e];
    }
    __device__ __forceinline__ void of_column(int u, int &r, int &c, float (&v)[8]) const {
        c = (u * 64 + lane) / (ROWS / 8);
        r = (u * 64 + lane) % (ROWS / 8) * 8;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = *reinterpret_cast<const float *>(at(r + e, c >> 2) + (c & 3) * 4);
    }
};

// ---- the order of tiles --------------------------------------------------------------------------------------------------
// Neighbours in the order share operand rows in their XCD's L2: bands of eight tile rows, column by column
__device__ __forceinline__ void tile_at(int t, int tiles_m, int tiles_n, int &tm, int &tn) {
    const int band = t / (8 * tiles_n), first = band * 8, h = tiles_m - first < 8 ? tiles_m - first : 8;
    const int r = t - first * tiles_n;
    tm = first + r % h;
    tn = r / h;
}
// the tiles on and below the diagonal: bands of four rows, column by column.  Band b begins at tile 8 b^2 + 2 b.
__device__ __forceinline__ void lower_tile_at(int t, int tiles, int &tm, int &tn) {
    int b = int((sqrtf(8.f * t + 1.f) - 1.f) * 0.125f);
    while (b > 0 && 8 * b * b + 2 * b > t) --b;
    while (8 * (b + 1) * (b + 1) + 2 * (b + 1) <= t) ++b;
    const int first = 4 * b, h = tiles - first < 4 ? tiles - first : 4;
    int r = t - (8 * b * b + 2 * b);
    if (r < first * h) {
        tm = first + r % h;
        tn = r / h;
        return;
    }
    r -= first * h;
    int c = 0;
    while (r >= h - c) r -= h - c++;
    tn = first + c;
    tm = tn + r;
}

// Workgroups are handed to the eight XCDs in turn; this maps the launch order so that each XCD works on a run of
// consecutive tiles (whose operands its own L2 then holds).
__device__ __forceinline__ int xcd_order(int id, int n) {
    const int q = n >> 3, r = n & 7, x = id & 7;
    return (x < r ? x * (q + 1) : r * (q + 1) + (x - r) * q) + (id >> 3);
}

// The same in runs of 32, for kernels that stream: neighbours share the lines between them in one L2, while all XCDs work on
// one region of memory.
__device__ __forceinline__ int xcd_runs(int id, int n) {
    const int block = id & ~255;
    return block + 256 <= n ? block | (id & 7) << 5 | (id >> 3 & 31) : id;
}

}  // namespace nt
