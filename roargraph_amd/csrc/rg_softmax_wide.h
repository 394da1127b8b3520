// rg_softmax_wide.h -- the pass of the softmax operators for many stationary rows: bound by the matrix cores (rg_softmax_pass.h has the
// mathematics, the operand layouts and the LDS swizzle; rg_softmax_thin.h the form for few rows, bound by memory).
//
// Streamed rows arrive as 16-bit planes (16-bit rows where they lie, or what rg_softmax_planes_kernel wrote: rows padded to the
// instantiation's width, fp32 as two halves) and go from memory to LDS without passing registers (global_load_lds, 16 bytes a lane) into
// a ring of as many tile buffers as fit, so that 50 - 100 KB per CU are on their way at any time.
//
// Two waves per SIMD, so that the weights of one are taken while the products of the other run.  (One wave per SIMD with 512 registers and a
// loop over three tiles, which does the same within a wave, took 4.5 ms where this takes 3.0: half the registers can only be moved to, not used.)
// Every LDS operand read feeds NX products.  Wide rows, of which a wave's 256 registers do not hold one, are shared by KQ waves: each has a
// part of the dimensions, they add up their products in LDS, and each takes the weights of all rows y for its own part of the output.
#pragma once
#include <type_traits>

#include "rg_softmax_pass.h"

namespace rg {

// A workgroup of eight waves, two per SIMD.  KQ waves share each of its 8 / KQ groups of 16 NX rows x, a KQ-th of the dimensions each.
struct WideChoice {
    int nx, kq;
};
// Measured (2000 queries, 30M elements of base, training step; with spills: the form whose registers were not enough): fp32 x 512 one wave a row
// 1.82 ms, two 1.57 ms; x 768 four waves, 16 rows each 2.31 ms, 32 rows (spills) 2.80 ms, one wave (spills) 6.07 ms; fp16 x 512 one wave, 16 rows
// 0.62 ms, two waves, 32 rows (spills) 1.10 ms; x 1024 four waves 0.93 ms, one (spills) 5.59 ms.  Statistics alone: fp16 x 768 one wave 0.14 ms,
// four 0.26 ms; fp32 x 768 four waves, 32 rows 0.56 ms, one 0.93 ms.
constexpr WideChoice softmax_wide_cfg(int dt, int ks, int mode) {
    const bool f32 = dt == RG_DTYPE_F32;
    if (mode == kStats && f32) return ks <= 4 ? WideChoice{3, 1} : ks <= 7 ? WideChoice{2, 1} : ks <= 16 ? WideChoice{1, 1} : ks <= 24 ? WideChoice{2, 4} : WideChoice{1, 4};
    if (mode == kStats) return {ks <= 7 ? 4 : ks <= 8 ? 3 : ks <= 16 ? 2 : 1, 1};
    const int kq = softmax_parts(dt, ks);
    if (f32) return {ks <= 4 ? 2 : 1, kq};
    return {ks <= 2 ? 4 : ks <= 4 ? 3 : ks <= 7 || (ks == 8 && mode == kMean) ? 2 : ks <= 16 ? 1 : ks <= 24 || mode == kMean ? 2 : 1, kq};
}

template <int DT, int KS, int MODE>
struct WideCfg {
    static constexpr bool F32 = DT == RG_DTYPE_F32;
    static constexpr int NP = F32 ? 2 : 1;
    static constexpr int NX = softmax_wide_cfg(DT, KS, MODE).nx, KQ = softmax_wide_cfg(DT, KS, MODE).kq;
    static constexpr int WAVES = 8, WPS = 2, NT = 64 * WAVES;
    static constexpr int KW = KS / KQ, OW = KS == 7 ? 13 : 2 * KW;   // steps of the first product and output blocks of a wave
    static constexpr int OB = KQ * OW;
    static constexpr int XT = 16 * NX * WAVES / KQ;
    static constexpr int TY = 32;
    static constexpr int PITCH = (KS * 64 + 255) / 256 * 256;
    static constexpr int PLANE = TY * PITCH;
    static constexpr int BUF = NP * PLANE;
    static constexpr bool INFO = F32 || MODE == kRows;
    static constexpr int NI = BUF / (16 * NT) + (INFO ? 1 : 0);      // loads of a tile, per wave
    static constexpr int PARTS = softmax_parts(DT, KS);
    static constexpr int EX = KQ > 1 ? WAVES * NX * 2 * 1024 : 0;    // where the waves of a group add up their products
    static constexpr int FIT = (160 * 1024 - EX) / (BUF + (INFO ? TY * 16 : 0));
    static constexpr int NBUF = FIT > 8 ? 8 : FIT;
    static constexpr int LDS = NBUF * (BUF + (INFO ? TY * 16 : 0)) + EX;
    static_assert((KQ == 1 || KQ == PARTS) && KS % PARTS == 0 && NBUF >= 1, "parts are whole steps, and a tile fits");
};

// 16 bytes a lane from base + off to LDS at `to` + 16 * lane.  Written as assembly because the compiler, which cannot tell the ring's buffers
// apart, makes every LDS read wait for all such loads; the waits are the kernel's own (`arrived`).  m0 holds the LDS address and is put back.
__device__ __forceinline__ void load_lds16(const void *base, uint32_t off, uint32_t to) {
    uint32_t m0;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2\n\ts_mov_b32 m0, %0" : "=&s"(m0) : "v"(off), "s"(base), "s"(to) : "memory");
}

template <int DT, int KS, int MODE>
__global__ void __launch_bounds__((WideCfg<DT, KS, MODE>::NT), (WideCfg<DT, KS, MODE>::WPS)) rg_softmax_wide_kernel(PassArgs A) {
    typedef WideCfg<DT, KS, MODE> C;
    typedef typename Frag<DT>::V V;
    constexpr int NP = C::NP, NX = C::NX, KQ = C::KQ, KW = C::KW, OW = C::OW, PITCH = C::PITCH, NBUF = C::NBUF;
    constexpr bool F32 = C::F32, INFO = C::INFO;
    constexpr bool TWO = F32 && MODE == kMean;      // weights of O carry the rows' scales: the sum l has a reference of its own
    constexpr bool BIAS = TWO || MODE == kRows;
    // (weights of kRows are at most |w| and bf16 has the range of fp32: a constant serves.  2^-16 keeps weights down to 2^-142 normal, and sums of weight times
    // query up to 2^111 finite; with 2^-60 those from 2^67 on were infinite.)
    constexpr bool NOREF = DT == RG_DTYPE_BF16 && MODE == kRows;
    constexpr float kTop = 15.0f, kStart = DT == RG_DTYPE_BF16 ? 0.0f : 7.0f;
    extern __shared__ char lds[];
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), n = lane & 15, g = lane >> 4;
    const uint32_t ntx = (A.nx + C::XT - 1) / C::XT;
    const uint32_t b = xcd_block(blockIdx.x, gridDim.x);
    const uint32_t xt = b % ntx;
    const uint32_t split = b / ntx, kq = wave % KQ;
    const uint32_t ybeg = min(A.ny, split * A.rows_per_split), yend = min(A.ny, ybeg + A.rows_per_split);
    const uint32_t ntiles = (yend - ybeg + 31) / 32;
    const uint32_t x0 = xt * C::XT + wave / KQ * 16 * NX;
    const bool live = x0 < A.nx;

    // tile t of this piece into its buffer: 16-byte slot q of a plane of the tile is (row, slot of the row).  Rows behind the last one are
    // loaded as the last (they take no part); chunks behind the rows' elements are not loaded and stay zero.
    constexpr int SR = PITCH / 16, PER = 32 * SR / C::NT;
    const uint32_t nchunks = A.ydim / 8, ystep = (uint32_t)A.ystride * 2;           // (32 rows' bytes fit 32 bits: the host's rule)
    const uint32_t ring = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)lds;
    auto offset = [&](int i, uint32_t rows, uint32_t thread) {
        const uint32_t q = i * C::NT + thread, r = q / SR, slot = q % SR;
        const uint32_t c = (slot & ~15u) | ((slot & 15) ^ swizzle(r));
        return c < nchunks ? min(r, rows - 1) * ystep + c * 16 : c < 4 * KS ? 0xffffffffu : min(r, rows - 1) * ystep;
    };
    constexpr bool KEPT = PER <= 6;                 // (more offsets than that are made anew for every tile: the registers are worth more)
    uint32_t off[KEPT ? PER : 1];
    if (KEPT)
#pragma unroll
        for (int i = 0; i < PER; ++i) off[i] = offset(i, 32, tid);
    const bool holes = nchunks < 4 * KS;
    if (holes) {                                    // what no load writes
        for (uint32_t i = tid; i < NBUF * C::BUF / 16; i += C::NT) reinterpret_cast<u32x4 *>(lds)[i] = u32x4{0, 0, 0, 0};
        __syncthreads();
    }
    auto load = [&](uint32_t t) {
        const uint32_t buf = t % NBUF, y0 = ybeg + 32 * t, to = __builtin_amdgcn_readfirstlane(ring + buf * C::BUF + wave * 1024);
        const char *first = static_cast<const char *>(A.y) + (size_t)y0 * A.ystride * 2;
        const uint32_t rows = min(yend - y0, 32u);
        uint32_t thread = tid;
        if (!KEPT) asm("" : "+v"(thread));
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const uint32_t o = !KEPT || rows < 32 ? offset(i, rows, thread) : off[i];
#pragma unroll
            for (int p = 0; p < NP; ++p)
                if (!holes || o != 0xffffffffu) load_lds16(first + p * (KS * 64), o, to + (p * PER + i) * (16 * C::NT));
        }
        constexpr uint32_t each = 32 / C::WAVES;    // lanes of a wave that load the tile's 512 bytes of info
        if (INFO && lane < each) load_lds16(A.yinfo + (size_t)y0 * 4 + wave * each * 4, lane * 16, __builtin_amdgcn_readfirstlane(ring + NBUF * C::BUF + buf * 512 + wave * each * 16));
    };
    // tile t has landed, for all waves; `newer` tiles may still be on their way (loads land in the order they were issued; near the end,
    // where fewer are, all are waited for)
    auto arrived = [&](uint32_t t, auto newer) {
        constexpr int N = decltype(newer)::value * C::NI;
        static_assert(N >= 0 && N < 64, "vmcnt");
        if (t + decltype(newer)::value < ntiles)
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
        else
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
    };
    if (ntiles)
        for (uint32_t t = 0; t + 1 < (NBUF > 1 ? NBUF : 2) && t < ntiles; ++t) load(t);

    V X[NX][KW][NP];
    float kx[NX];
    uint32_t target[NX];
#pragma unroll
    for (int j = 0; j < NX; ++j) {
        const uint32_t x = x0 + j * 16 + n;
        kx[j] = load_stationary<DT, KW, KQ>(A, x, g, X[j], kq);
        target[j] = kNoTarget;
        if (MODE != kRows && x < A.nx) {
            const uint32_t tg = A.targets[x];
            if (tg != kNoTarget && tg >= A.id_base && tg - A.id_base >= ybeg && tg - A.id_base < yend) target[j] = tg - A.id_base;
        }
    }
    __builtin_amdgcn_s_waitcnt(0x0f70);             // the compiler's own loads (vmcnt(0)): none of its waits is left for the loop
    f32x4 O[MODE == kStats ? 1 : OW][NX];
    constexpr bool SUM = softmax_sums_rounded(DT, MODE);
    float M[NX], l[NX], Ml[NX], R[NX];
#pragma unroll
    for (int j = 0; j < NX; ++j) {
        M[j] = NOREF ? -16.0f : kNothing;
        Ml[j] = kNothing;
        l[j] = R[j] = 0.0f;
        if (MODE != kStats)
#pragma unroll
            for (int ob = 0; ob < OW; ++ob) O[ob][j] = f32x4{0, 0, 0, 0};
    }

    if (MODE != kRows && A.resume) {
        take_up<DT, MODE, OW, NX>(A, x0, n, g, kq, split, M, Ml, l, R, O);
        __builtin_amdgcn_s_waitcnt(0x0f70);         // (as above)
    }

    // LDS operands are asked for AHEAD steps before the products that take them, and the compiler is kept from moving the reads back
    // (vector and scalar instructions may still move between the products)
    auto keep_order = [] { __builtin_amdgcn_sched_barrier(0x6); };
    typedef __attribute__((address_space(3))) const V LdsV;
    // an LDS address the compiler takes as it is: left to itself it splits these sums over the loop and folds no constant into the reads
    auto lds_at = [](uint32_t a) {
        asm("" : "+v"(a));
        return a;
    };
    // what a lane reads of a tile: chunks 4 ks + g of row n, and dims 4 (n % 4) of each block of rows 4 g + n / 4 (they repeat every 256 bytes)
    // -- where registers are few, all of them are made of the first, by its bits 5 - 7, for every read (a wave's part of a row starts with 256 bytes there):
    // mean of 2048 bf16 queries on 400k x 256 923 us, so 743 us; 2000 fp16 on 30k x 1024 492 us, so 414 us; but 4096 bf16 on 250k x 512, which fit, 1.74 ms, so 1.78
    constexpr bool MADE = softmax_sums_rounded(DT, MODE) && (KS == 8 || KS == 32);
    static_assert(!MADE || KQ == 1 || (KW % 4 == 0 && OW % 8 == 0), "parts start with 256 bytes");
    uint32_t first_at[MADE ? 1 : 4], second_at[MADE ? 1 : 8];
    auto chunk_at = [&](uint32_t row, uint32_t c) { return ring + row * PITCH + (c >> 4 << 8) + (((c & 15) ^ swizzle(row)) << 4); };
#pragma unroll
    for (int i = 0; i < (MADE ? 1 : 4); ++i) first_at[i] = chunk_at(n, 4 * (kq * KW + i) + g);
#pragma unroll
    for (int i = 0; i < (MADE ? 1 : 8); ++i) second_at[i] = chunk_at(4 * g + (n >> 2), 2 * (kq * OW + i) + (n >> 1 & 1)) + (n & 1) * 8;
    auto first_product = [&](uint32_t buf, f32x4 (&S)[NX][2]) {
        constexpr int AHEAD = 1;
        uint32_t at[MADE ? 1 : 4];
#pragma unroll
        for (int i = 0; i < (MADE ? 1 : 4); ++i) at[i] = lds_at(first_at[i] + buf * C::BUF);
        V a[AHEAD + 1][2][NP];
        auto read = [&](int ks) {
            const uint32_t from = MADE ? lds_at(at[0] ^ (uint32_t)(ks % 4 << 6)) : at[MADE ? 0 : ks % 4];
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int p = 0; p < NP; ++p) a[ks % (AHEAD + 1)][h][p] = *(LdsV *)(from + (uint32_t)(ks / 4 * 256 + h * 16 * PITCH + p * C::PLANE));
        };
#pragma unroll
        for (int j = 0; j < NX; ++j) S[j][0] = S[j][1] = f32x4{0, 0, 0, 0};
        constexpr int PART = KQ == 1 ? KS / C::PARTS : KW;      // steps of a part
        f32x4 sum[NX][2];
#pragma unroll
        for (int ks = 0; ks < AHEAD && ks < KW; ++ks) read(ks);
#pragma unroll
        for (int ks = 0; ks < KW; ++ks) {
            if (ks + AHEAD < KW) read(ks + AHEAD);
            keep_order();
            if (ks % PART == 0 && ks) {
#pragma unroll
                for (int j = 0; j < NX; ++j)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        sum[j][h] = ks == PART ? S[j][h] : sum[j][h] + S[j][h];
                        S[j][h] = f32x4{0, 0, 0, 0};
                    }
            }
            const V(&v)[2][NP] = a[ks % (AHEAD + 1)];
            if constexpr (F32) {
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int j = 0; j < NX; ++j) S[j][h] = mma(v[h][1], X[j][ks][0], S[j][h]);
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int j = 0; j < NX; ++j) S[j][h] = mma(v[h][0], X[j][ks][1], S[j][h]);
            }
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int j = 0; j < NX; ++j) S[j][h] = mma(v[h][0], X[j][ks][0], S[j][h]);
            keep_order();
        }
        if (PART < KW)
#pragma unroll
            for (int j = 0; j < NX; ++j)
#pragma unroll
                for (int h = 0; h < 2; ++h) S[j][h] = sum[j][h] + S[j][h];
    };
    // the products of the waves of a group, added up in one order by all of them
    f32x4 *const ex = reinterpret_cast<f32x4 *>(lds + C::LDS - C::EX);
    auto part_out = [&](const f32x4 (&S)[NX][2]) {
#pragma unroll
        for (int j = 0; j < NX; ++j)
#pragma unroll
            for (int h = 0; h < 2; ++h) ex[((wave * NX + j) * 2 + h) * 64 + lane] = S[j][h];
    };
    auto parts_in = [&](f32x4 (&S)[NX][2]) {
#pragma unroll
        for (int j = 0; j < NX; ++j)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                S[j][h] = ex[((wave / KQ * KQ * NX + j) * 2 + h) * 64 + lane];
#pragma unroll
                for (int q = 1; q < KQ; ++q) S[j][h] += ex[(((wave / KQ * KQ + q) * NX + j) * 2 + h) * 64 + lane];
            }
    };
    auto second_product = [&](uint32_t buf, const V (&W)[NX][NP]) {
        if constexpr (MODE != kStats) {
            typedef __attribute__((address_space(3))) s16x4 *tr_ptr;
            constexpr int AHEAD = 2;
            uint32_t at[MADE ? 1 : 8];
#pragma unroll
            for (int i = 0; i < (MADE ? 1 : 8); ++i) at[i] = lds_at(second_at[i] + buf * C::BUF);
            s16x4 a[AHEAD + 1][NP][2];
            auto read = [&](int ob) {
                const uint32_t from = MADE ? lds_at(at[0] ^ (uint32_t)(ob % 8 << 5)) : at[MADE ? 0 : ob % 8];
#pragma unroll
                for (int p = 0; p < NP; ++p)
#pragma unroll
                    for (int h = 0; h < 2; ++h) a[ob % (AHEAD + 1)][p][h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_ptr)(from + (uint32_t)(ob / 8 * 256 + p * C::PLANE + h * 16 * PITCH)));
            };
#pragma unroll
            for (int ob = 0; ob < AHEAD && ob < OW; ++ob) read(ob);
#pragma unroll
            for (int ob = 0; ob < OW; ++ob) {
                if (ob + AHEAD < OW) read(ob + AHEAD);
                keep_order();
                V v[NP];
#pragma unroll
                for (int p = 0; p < NP; ++p) v[p] = __builtin_bit_cast(V, __builtin_shufflevector(a[ob % (AHEAD + 1)][p][0], a[ob % (AHEAD + 1)][p][1], 0, 1, 2, 3, 4, 5, 6, 7));
                if constexpr (F32) {
#pragma unroll
                    for (int j = 0; j < NX; ++j) O[ob][j] = mma(v[1], W[j][0], O[ob][j]);
#pragma unroll
                    for (int j = 0; j < NX; ++j) O[ob][j] = mma(v[0], W[j][1], O[ob][j]);
                }
#pragma unroll
                for (int j = 0; j < NX; ++j) O[ob][j] = mma(v[0], W[j][0], O[ob][j]);
                keep_order();
            }
        }
    };

    // A query's own row gets most of its weight, and 8 bits of a weight are few: tiles that hold one are gone through twice, the second time for
    // what rounding left of the weights.  (A bf16 gradient's error then is that of its last rounding, 0.0017 of its norm instead of 0.0024.  A
    // second product in line instead kept O in two places: a step of 2048 queries on 1M x 200 took 10.5 ms, takes 2.9.)
    constexpr bool TWICE = DT == RG_DTYPE_BF16 && MODE == kRows;
    // a tile's rows: elements (h, i) of a lane are rows 16 h + 4 g + i
    struct Tile {
        uint32_t y0, slot;          // first row; where its info lies
        bool rare, neg;             // a target of these rows, or rows behind the last, lie in the tile; a weight is negative
        bool twice;                 // TWICE: a target of the workgroup's rows lies in the tile
    };
    enum { kFactor, kBias, kSign, kTarget };
    auto info = [&](const Tile &t, int what, uint32_t r) { return *reinterpret_cast<const float *>(lds + NBUF * C::BUF + t.slot * 512 + what * 128 + r * 4); };
    auto info4 = [&](const Tile &t, int what, int h) { return *reinterpret_cast<const f32x4 *>(lds + NBUF * C::BUF + t.slot * 512 + what * 128 + (16 * h + 4 * g) * 4); };
    auto look = [&](uint32_t t) {
        Tile k{ybeg + 32 * t, t % NBUF, false, false, false};
        bool met = false;
        if (MODE != kRows) {
#pragma unroll
            for (int j = 0; j < NX; ++j) met |= target[j] - k.y0 < 32;
        } else {
            const uint32_t at = __float_as_uint(info(k, kTarget, lane & 31));
            met = at - x0 < 16 * NX;
            if (TWICE) k.twice = __any(at - xt * C::XT < C::XT);
            k.neg = __any(info(k, kSign, lane & 31) < 0.0f);
        }
        k.rare = __any(met) || (MODE != kRows && k.y0 + 32 > yend);      // (kRows: rows behind the last have no weight as it is)
        return k;
    };
    // Rows read where they lie that take no part and hold an infinity or NaN (rare; planes of fp32 hold zeros there) become zeros: every wave
    // writes them before it reads the tile.
    auto blank = [&](uint32_t buf) {
        const float sign = *reinterpret_cast<const float *>(lds + NBUF * C::BUF + buf * 512 + kSign * 128 + (lane & 31) * 4);
        for (uint32_t m = (uint32_t)__ballot(sign == 0.0f); m; m &= m - 1)
            for (uint32_t c = lane; c < PITCH / 16; c += 64) reinterpret_cast<u32x4 *>(lds + buf * C::BUF + (__ffs(m) - 1) * PITCH)[c] = u32x4{0, 0, 0, 0};
    };
    // Rare: elements of a tile whose weight is not made of their product: bit 4 h + i of those that take no part (a target, whose logit is set aside;
    // rows behind the last), or in kRows of a query's own row, which has the logarithm of its weight, and whose sign turns.
    // (Every instruction here is fetched from memory when it comes to it: as 24 branches a tile it took a workgroup 25 us.)
    uint32_t off_bits[NX];
    auto special = [&](const Tile &k, const f32x4 (&S)[NX][2]) {
        auto bit_of = [&](uint32_t r) { return (r >> 2 & 3) == g ? 1u << (4 * (r >> 4) + (r & 3)) : 0u; };      // of row r < 32, where it lies in this lane
        if constexpr (MODE == kRows) {
#pragma unroll
            for (int j = 0; j < NX; ++j) off_bits[j] = 0;
            const uint32_t at = __float_as_uint(info(k, kTarget, lane & 31)) - x0;
            for (uint32_t m = (uint32_t)__ballot(at < 16 * NX); m; m &= m - 1) {
                const uint32_t r = __ffs(m) - 1, x = __builtin_amdgcn_readlane(at, r);
#pragma unroll
                for (int j = 0; j < NX; ++j) off_bits[j] |= x == 16 * j + n ? bit_of(r) : 0;
            }
        } else {
            uint32_t behind = 0;
            if (k.y0 + 32 > yend)
#pragma unroll
                for (int h = 0; h < 2; ++h) behind |= (15u << max(min((int)(yend - k.y0) - (int)(16 * h + 4 * g), 4), 0) & 15u) << (4 * h);
#pragma unroll
            for (int j = 0; j < NX; ++j) {
                const uint32_t r = target[j] - k.y0, mine = r < 32 ? bit_of(r) : 0;
                off_bits[j] = behind | mine;
                float z = 0.0f;
#pragma unroll
                for (int e = 0; e < 8; ++e) z = mine >> e & 1 ? S[j][e / 4][e % 4] : z;
                if (kq == 0 && mine) A.own2[x0 + 16 * j + n] = z * (INFO ? kx[j] * info(k, kFactor, r) : kx[j]);
            }
        }
    };
    // the exponent of a row y's own scale, which its weights carry in kRows (kMean: it is the bias).  It is taken from a reference first, which is
    // exact, so that a bias keeps its digits however large both are.
    auto exponent = [](float factor) { return (float)((int)(__float_as_uint(factor) >> 23) - 127); };
    constexpr bool SCALED = F32 && MODE == kRows;
    auto logits = [&](const Tile &k, const f32x4 (&S)[NX][2], bool biased, const float (&ref)[NX], float (&p)[NX][2][4]) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            f32x4 factor{1.0f, 1.0f, 1.0f, 1.0f}, bias{0.0f, 0.0f, 0.0f, 0.0f};
            if (F32) factor = info4(k, kFactor, h);
            if (BIAS) bias = info4(k, kBias, h);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float e = SCALED ? exponent(factor[i]) : 0.0f;
#pragma unroll
                for (int j = 0; j < NX; ++j) p[j][h][i] = fmaf(F32 ? S[j][h][i] * factor[i] : S[j][h][i], kx[j], SCALED ? bias[i] + (e - ref[j]) : biased ? bias[i] - ref[j] : -ref[j]);
            }
        }
        if (__builtin_expect(k.rare, 0))
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                f32x4 own{0.0f, 0.0f, 0.0f, 0.0f}, factor = own;
                if (MODE == kRows) own = *reinterpret_cast<const f32x4 *>(A.ytarget + (k.y0 + 16 * h + 4 * g));
                if (SCALED) factor = info4(k, kFactor, h);
#pragma unroll
                for (int j = 0; j < NX; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float v = MODE == kRows ? own[i] + ((SCALED ? exponent(factor[i]) : 0.0f) - ref[j]) : -INFINITY;
                        p[j][h][i] = off_bits[j] >> (4 * h + i) & 1 ? v : p[j][h][i];
                    }
            }
    };
    auto over = [&](const auto &p) {
        float top = kNothing;
#pragma unroll
        for (int j = 0; j < NX; ++j)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < 4; ++i) top = fmaxf(top, p[j][h][i]);
        return top > kTop;
    };
    // Rare: a logit p passes its reference by kTop.  The references of those rows move -- of those only, so that results do not depend on which rows
    // share a wave --, the logits are made anew, and `moved` multiplies what was summed under the old references.  (The loop leaves one copy of
    // the code; a first turn in it, for all tiles, cost 2 %: nothing moves between it and the products.)
    auto relocate = [&](const Tile &k, const f32x4 (&S)[NX][2], bool biased, float (&ref)[NX], float (&p)[NX][2][4], auto &&moved) {
        float under[NX], above[NX], old[NX];
        auto largest = [&](int j) {
            float z = kNothing;
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < 4; ++i) z = fmaxf(z, p[j][h][i]);
            z = fmaxf(z, __shfl_xor(z, 16));
            return fmaxf(z, __shfl_xor(z, 32));
        };
#pragma unroll
        for (int j = 0; j < NX; ++j) {
            above[j] = largest(j);
            under[j] = 0.0f;
            old[j] = 1.0f;
        }
#pragma clang loop unroll(disable)
        for (int turn = 0; turn < 2; ++turn) {
            logits(k, S, biased, under, p);
            if (turn == 0)
#pragma unroll
                for (int j = 0; j < NX; ++j) {
                    under[j] = above[j] > kTop ? largest(j) - kStart : ref[j];
                    old[j] = exp2_hw(ref[j] - under[j]);
                    ref[j] = under[j];
                }
        }
        moved(old);
    };
    auto sum = [&](const float (&p)[2][4]) { return ((p[0][0] + p[0][1]) + (p[0][2] + p[0][3])) + ((p[1][0] + p[1][1]) + (p[1][2] + p[1][3])); };
    auto exps = [&](auto &p) {
#pragma unroll
        for (int j = 0; j < NX; ++j)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < 4; ++i) p[j][h][i] = exp2_hw(p[j][h][i]);
    };
    auto pack = [&](const float (&p)[NX][2][4], V (&W)[NX][NP]) {
#pragma unroll
        for (int j = 0; j < NX; ++j)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if constexpr (DT == RG_DTYPE_BF16) {
                        W[j][0][4 * h + i] = (__bf16)p[j][h][i];
                    } else {
                        W[j][0][4 * h + i] = (_Float16)p[j][h][i];
                        if constexpr (F32) W[j][1][4 * h + i] = (_Float16)(p[j][h][i] - (float)W[j][0][4 * h + i]);
                    }
                }
    };
    auto signs = [&](const Tile &k, V (&W)[NX][NP]) {           // rare, kRows
        uint32_t minus[4] = {0, 0, 0, 0};
#pragma unroll
        for (int e = 0; e < 8; ++e) minus[e / 2] |= (__float_as_uint(info(k, kSign, 16 * (e / 4) + 4 * g + e % 4)) & 0x80000000u) >> (e % 2 ? 0 : 16);
#pragma unroll
        for (int j = 0; j < NX; ++j) {
            const uint32_t f = k.rare ? off_bits[j] : 0;
#pragma unroll
            for (int q = 0; q < NP; ++q) {
                u32x4 v = __builtin_bit_cast(u32x4, W[j][q]);
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] ^= minus[e] ^ ((f >> (2 * e) & 1) << 15 | (f >> (2 * e + 1) & 1) << 31);
                W[j][q] = __builtin_bit_cast(V, v);
            }
        }
    };
    // the weights of a tile, and their sums
    auto weights = [&](const Tile &k, const f32x4 (&S)[NX][2], float (&p)[NX][2][4]) {
        auto add = [&](const auto &v) {
#pragma unroll
            for (int j = 0; j < NX; ++j) l[j] += sum(v[j]);
        };
        auto scale_l = [&](const float (&old)[NX]) {
#pragma unroll
            for (int j = 0; j < NX; ++j) l[j] *= old[j];
        };
        float pl[TWO ? NX : 1][2][4];
        bool high = false;
        if constexpr (TWO) {
            logits(k, S, false, Ml, pl);
            high = over(pl);
        }
        logits(k, S, BIAS, M, p);
        if (!NOREF) high |= over(p);
        if (!NOREF && __builtin_expect(__any(high), 0)) {
            if constexpr (TWO) relocate(k, S, false, Ml, pl, scale_l);
            relocate(k, S, BIAS, M, p, [&](const float (&old)[NX]) {
                if (!TWO) scale_l(old);
                if (SUM)
#pragma unroll
                    for (int j = 0; j < NX; ++j) R[j] *= old[j];
                if (MODE != kStats)
#pragma unroll
                    for (int j = 0; j < NX; ++j)
#pragma unroll
                        for (int ob = 0; ob < OW; ++ob) O[ob][j] *= old[j];
            });
        }
        exps(p);
        if constexpr (TWO) {
            exps(pl);
            add(pl);
        } else if (MODE != kRows) {
            add(p);
        }
    };

    if (ntiles) {
        if constexpr (MODE == kStats && NBUF >= 3 && KQ == 1) {
            // first product of the next tile beside the weights of this one; tile t + NBUF - 1 takes the place of tile t - 1
            f32x4 S[NX][2], next[NX][2];
            arrived(0, std::integral_constant<int, NBUF - 2>{});
            if (live) first_product(0, S);
            for (uint32_t t = 0; t < ntiles; ++t) {
                arrived(t + 1, std::integral_constant<int, NBUF - 3>{});       // (every wave is through with tile t - 1)
                if (t + NBUF - 1 < ntiles) load(t + NBUF - 1);
                if (live) {
                    float p[NX][2][4];
                    const Tile k = look(t);
                    if (__builtin_expect(k.rare, 0)) special(k, S);
                    first_product((t + 1) % NBUF, next);                       // (behind the last tile: of old rows, for nobody)
                    weights(k, S, p);
#pragma unroll
                    for (int j = 0; j < NX; ++j) { S[j][0] = next[j][0]; S[j][1] = next[j][1]; }
                }
            }
        } else {
            f32x4 S[NX][2];
            V W[NX][NP];
            float p[NX][2][4];
            bool again = false;
            for (uint32_t t = 0; t < ntiles;) {
                if (TWICE && again) {
                    if (KQ > 1) __syncthreads();     // (every wave has read the parts)
                } else {
                    arrived(t, std::integral_constant<int, (NBUF > 1 ? NBUF - 2 : 0)>{});     // (every wave is through with tile t - 1)
                    if (NBUF > 1 && t + NBUF - 1 < ntiles) load(t + NBUF - 1);
                    if (MODE == kRows && !F32) blank(t % NBUF);
                }
                if (live) first_product(t % NBUF, S);
                if constexpr (KQ > 1) {
                    part_out(S);
                    __syncthreads();
                }
                Tile k;
                if (TWICE) k = look(t);              // (all waves: they turn together)
                if (live) {
                    if constexpr (KQ > 1) parts_in(S);
                    if (!TWICE) k = look(t);
                    if (__builtin_expect(k.rare, 0)) special(k, S);
                    weights(k, S, p);
                    if (MODE != kStats) {
                        if constexpr (TWICE)
                            if (__builtin_expect(again, 0))
#pragma unroll
                                for (int j = 0; j < NX; ++j)
#pragma unroll
                                    for (int h = 0; h < 2; ++h)
#pragma unroll
                                        for (int i = 0; i < 4; ++i) p[j][h][i] -= (float)(__bf16)p[j][h][i];
                        pack(p, W);
                        if constexpr (SUM)
#pragma unroll
                            for (int j = 0; j < NX; ++j) R[j] += sum_of(W[j][0]);
                        if (MODE == kRows && __builtin_expect(k.rare || k.neg, 0)) signs(k, W);
                        second_product(t % NBUF, W);
                    }
                }
                if constexpr (TWICE) {
                    again = !again && k.twice;
                    if (again) continue;
                }
                if (NBUF == 1 && t + 1 < ntiles) {
                    __syncthreads();
                    load(t + 1);
                }
                ++t;
            }
        }
    }
    finish<DT, MODE, OW, NX>(A, x0, n, g, kq, split, M, TWO ? Ml : M, l, R, O);
}

}  // namespace rg
