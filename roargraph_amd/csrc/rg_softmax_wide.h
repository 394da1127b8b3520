// rg_softmax_wide.h -- the pass of the softmax operators for many stationary rows: bound by the matrix cores (rg_softmax_pass.h has the
// mathematics, the operand layouts and the LDS swizzle; rg_softmax_thin.h the form for few rows, bound by memory).
//
// Streamed rows arrive as 16-bit planes (16-bit rows where they lie, or what rg_softmax_planes_kernel wrote: rows padded to the
// instantiation's width, fp32 as two halves) and go from memory to LDS without passing registers (global_load_lds, 16 bytes a lane) into
// a ring of as many tile buffers as fit, so that 50 - 100 KB per CU are on their way at any time.  One wave per SIMD, as many blocks of x
// as 512 registers hold: every LDS operand read feeds NX products.
//
// With a ring of six and more the loop runs three tiles at a time, so that matrix and vector units work side by side in one wave:
//     first product of tile t + 1   while  the logits of tile t are scaled and compared with the reference
//     second product of tile t - 1  while  the weights of tile t are taken (exp2, sums, rounding)
// A reference that moves (rare) first lets the pending second product go, then rescales.
#pragma once
#include <type_traits>

#include "rg_softmax_pass.h"

namespace rg {

template <int DT, int KS, int MODE>
struct WideCfg {
    static constexpr bool F32 = DT == RG_DTYPE_F32;
    static constexpr int NP = F32 ? 2 : 1;
    static constexpr int OB = KS == 7 ? 13 : F32 && KS == 32 ? 32 : 2 * KS;
    // registers of a lane: X 4 NP KS per block, O 4 OB, logits 16, weights 4 NP
    static constexpr int NX = MODE == kStats ? (F32 ? (KS <= 8 ? 4 : KS <= 12 ? 3 : KS <= 16 ? 2 : 1) : (KS <= 8 ? 6 : KS <= 12 ? 5 : KS <= 16 ? 4 : KS <= 24 ? 3 : 2))
                              : F32          ? (KS <= 4 ? 4 : KS <= 8 ? 2 : 1)
                                             : (KS <= 4 ? 4 : KS <= 7 ? 3 : KS <= 12 ? 2 : 1);
    static constexpr int XT = 64 * NX;
    static constexpr int TY = 32;
    static constexpr int PITCH = (KS * 64 + 255) / 256 * 256;
    static constexpr int PLANE = TY * PITCH;
    static constexpr int BUF = NP * PLANE;
    static constexpr bool INFO = F32 || MODE == kRows;
    static constexpr int NI = BUF / 4096 + (INFO ? 1 : 0);      // loads of a tile, per wave
    static constexpr int FIT = 160 * 1024 / (BUF + (INFO ? TY * 16 : 0));
    static constexpr int NBUF = FIT > 8 ? 8 : FIT;
    static constexpr bool PIPE = MODE != kStats && NBUF >= 6;
    static constexpr int LDS = NBUF * (BUF + (INFO ? TY * 16 : 0));
};

__device__ const u32x4 g_zero16 = {0, 0, 0, 0};

template <int DT, int KS, int MODE>
__global__ void __launch_bounds__(256, 1) rg_softmax_wide_kernel(PassArgs A) {
    typedef WideCfg<DT, KS, MODE> C;
    typedef typename Elem<DT>::T T;
    typedef typename Frag<DT>::V V;
    constexpr int NP = C::NP, NX = C::NX, OB = C::OB, PITCH = C::PITCH, NBUF = C::NBUF;
    constexpr bool F32 = C::F32, INFO = C::INFO;
    constexpr bool TWO = F32 && MODE == kMean;      // weights of O carry the rows' scales: the sum l has a reference of its own
    constexpr bool BIAS = TWO || MODE == kRows;
    // (weights of kRows are at most |w| and bf16 has the range of fp32: a constant serves, which keeps small ones normal)
    constexpr bool NOREF = DT == RG_DTYPE_BF16 && MODE == kRows;
    constexpr float kTop = 15.0f, kStart = DT == RG_DTYPE_BF16 ? 0.0f : 7.0f;
    extern __shared__ char lds[];
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), n = lane & 15, g = lane >> 4;
    const uint32_t ntx = (A.nx + C::XT - 1) / C::XT;
    uint32_t b = xcd_block(blockIdx.x, gridDim.x);
    const uint32_t xt = b % ntx;
    b /= ntx;
    const uint32_t slice = MODE == kStats ? 0 : b % A.nslices, split = MODE == kStats ? b : b / A.nslices;
    const uint32_t ybeg = min(A.ny, split * A.rows_per_split), yend = min(A.ny, ybeg + A.rows_per_split);
    const uint32_t ntiles = (yend - ybeg + 31) / 32;
    const uint32_t x0 = xt * C::XT + wave * 16 * NX;
    const bool live = x0 < A.nx;

    // tile t of this piece into buffer `buf`: 16-byte slot q of the tile is (plane, row, slot of the row)
    constexpr int SR = PITCH / 16;
    const uint32_t nchunks = A.ydim / 8;
    // (a tile behind the last is loaded as zeros, so that the number of loads on their way is always known)
    auto load = [&](uint32_t t) {
        const uint32_t buf = t % NBUF, y0 = ybeg + 32 * t, left = y0 < yend ? yend - y0 : 0;
        const char *first = static_cast<const char *>(A.y) + (size_t)y0 * A.ystride * 2;
#pragma unroll
        for (int i = 0; i < C::BUF / 4096; ++i) {
            const uint32_t q = i * 256 + tid, row = q / SR, slot = q % SR, r = row & 31, p = row >> 5;
            const uint32_t c = (slot & ~15u) | ((slot & 15) ^ (((r & 7) << 1) | (r >> 3 & 1)));
            const char *at = first + (size_t)r * A.ystride * 2 + p * (KS * 64) + c * 16;
            if (c >= nchunks || r >= left) at = reinterpret_cast<const char *>(&g_zero16);
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)at,
                                             (__attribute__((address_space(3))) void *)(lds + buf * C::BUF + (i * 256 + wave * 64) * 16), 16, 0, 0);
        }
        if (INFO && lane < 8) {
            const float4 *at = A.yinfo + (left ? y0 : ybeg) + wave * 8 + lane;
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)at, (__attribute__((address_space(3))) void *)(lds + NBUF * C::BUF + buf * 512 + wave * 128), 16, 0, 0);
        }
    };
    // all but the last `newer` tiles' loads have landed, for all waves (loads land in the order they were issued)
    auto arrived = [&](auto newer) {
        constexpr int N = decltype(newer)::value * C::NI;
        static_assert(N >= 0 && N < 64, "vmcnt");
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
        __syncthreads();
    };
    if (ntiles)
        for (uint32_t t = 0; t + 1 < (NBUF > 1 ? NBUF : 2); ++t) load(t);

    V X[NX][KS][NP];
    float kx[NX];
    uint32_t target[NX];
    const bool xvec = ((uintptr_t)A.x | A.xstride * sizeof(T)) % 16 == 0;
#pragma unroll
    for (int j = 0; j < NX; ++j) {
        const uint32_t x = x0 + j * 16 + n;
        kx[j] = load_stationary<DT, KS>(A, x, g, xvec, X[j]);
        target[j] = kNoTarget;
        if (MODE != kRows && x < A.nx) {
            const uint32_t tg = A.targets[x];
            if (tg != kNoTarget && tg >= A.id_base && tg - A.id_base >= ybeg && tg - A.id_base < yend) target[j] = tg - A.id_base;
        }
    }
    f32x4 O[MODE == kStats ? 1 : OB][NX];
    float M[NX], l[NX], Ml[NX];
#pragma unroll
    for (int j = 0; j < NX; ++j) {
        M[j] = NOREF ? -60.0f : kNothing;
        Ml[j] = kNothing;
        l[j] = 0.0f;
        if (MODE != kStats)
#pragma unroll
            for (int ob = 0; ob < OB; ++ob) O[ob][j] = f32x4{0, 0, 0, 0};
    }

    auto first_product = [&](uint32_t buf, f32x4 (&S)[NX][2]) {
        const char *row = lds + buf * C::BUF + n * PITCH;
        const uint32_t sw = ((n & 7) << 1) | (n >> 3);
#pragma unroll
        for (int j = 0; j < NX; ++j) S[j][0] = S[j][1] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const uint32_t c = 4 * ks + g;
            const char *at = row + (c & ~15u) * 16 + (((c & 15) ^ sw) << 4);
            V a[2][NP];
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int p = 0; p < NP; ++p) a[h][p] = *reinterpret_cast<const V *>(at + h * 16 * PITCH + p * C::PLANE);
            if constexpr (F32) {
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int j = 0; j < NX; ++j) S[j][h] = mma(a[h][1], X[j][ks][0], S[j][h]);
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int j = 0; j < NX; ++j) S[j][h] = mma(a[h][0], X[j][ks][1], S[j][h]);
            }
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int j = 0; j < NX; ++j) S[j][h] = mma(a[h][0], X[j][ks][0], S[j][h]);
        }
    };
    auto second_product = [&](uint32_t buf, const V (&W)[NX][NP]) {
        if constexpr (MODE != kStats) {
            typedef __attribute__((address_space(3))) s16x4 *tr_ptr;
            const uint32_t r = 4 * g + (n >> 2), sw = ((r & 7) << 1) | ((r >> 3) & 1);
            const char *row = lds + buf * C::BUF + r * PITCH + (n & 1) * 8;
#pragma unroll
            for (int ob = 0; ob < OB; ++ob) {
                const uint32_t c = 2 * (slice * OB + ob) + ((n >> 1) & 1);
                const char *at = row + (c & ~15u) * 16 + (((c & 15) ^ sw) << 4);
                V a[NP];
#pragma unroll
                for (int p = 0; p < NP; ++p) {
                    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_ptr)(const_cast<char *>(at) + p * C::PLANE));
                    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_ptr)(const_cast<char *>(at) + p * C::PLANE + 16 * PITCH));
                    a[p] = __builtin_bit_cast(V, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
                }
                if constexpr (F32) {
#pragma unroll
                    for (int j = 0; j < NX; ++j) O[ob][j] = mma(a[1], W[j][0], O[ob][j]);
#pragma unroll
                    for (int j = 0; j < NX; ++j) O[ob][j] = mma(a[0], W[j][1], O[ob][j]);
                }
#pragma unroll
                for (int j = 0; j < NX; ++j) O[ob][j] = mma(a[0], W[j][0], O[ob][j]);
            }
        }
    };

    // the logits of a tile, in units of log 2, minus a reference; elements (h, i) of a lane are rows 16 h + 4 g + i
    struct Tile {
        uint32_t y0, slot;          // first row; where its info lies
        bool met, neg, tail;        // a target of these rows lies in the tile; a weight is negative; rows behind the last
    };
    auto info = [&](const Tile &t, uint32_t r) { return *reinterpret_cast<const f32x4 *>(lds + NBUF * C::BUF + t.slot * 512 + r * 16); };
    auto look = [&](uint32_t t) {
        Tile k{ybeg + 32 * t, t % NBUF, false, false, false};
        k.tail = k.y0 + 32 > yend;
        if (MODE != kRows) {
            bool met = false;
#pragma unroll
            for (int j = 0; j < NX; ++j) met |= target[j] - k.y0 < 32;
            k.met = __any(met);
        } else {
            const f32x4 v = info(k, lane & 31);
            k.met = __any(__float_as_uint(v[3]) - x0 < 16 * NX);
            k.neg = __any(v[2] < 0.0f);
        }
        return k;
    };
    uint32_t dead[NX], hit[NX];     // rare: bits of the elements that take no part / that are a query's own row
    auto special = [&](const Tile &k, const f32x4 (&S)[NX][2]) {
#pragma unroll
        for (int j = 0; j < NX; ++j) {
            dead[j] = hit[j] = 0;
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t r = 16 * h + 4 * g + i, x = x0 + j * 16 + n;
                    if (MODE != kRows && k.y0 + r == target[j]) {
                        float z = S[j][h][i];
                        if (F32) z *= info(k, r)[0];
                        if (slice == 0) A.own2[x] = z * kx[j];
                        dead[j] |= 1u << (4 * h + i);
                    }
                    if (MODE == kRows && __float_as_uint(info(k, r)[3]) == x) hit[j] |= 1u << (4 * h + i);
                    if (k.y0 + r >= yend) dead[j] |= 1u << (4 * h + i);
                }
        }
    };
    auto fix = [&](const Tile &k, int j, int h, int i, float z, float ref) {
        if (MODE == kRows && (hit[j] >> (4 * h + i) & 1)) z = A.ytarget[k.y0 + 16 * h + 4 * g + i] - ref;
        return dead[j] >> (4 * h + i) & 1 ? -INFINITY : z;
    };
    auto logits = [&](const Tile &k, const f32x4 (&S)[NX][2], bool biased, const float (&ref)[NX], float (&p)[NX][2][4]) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                f32x4 v{1.0f, 0.0f, 0.0f, 0.0f};
                if (INFO) v = info(k, 16 * h + 4 * g + i);
#pragma unroll
                for (int j = 0; j < NX; ++j) p[j][h][i] = fmaf(F32 ? S[j][h][i] * v[0] : S[j][h][i], kx[j], biased ? v[1] - ref[j] : -ref[j]);
            }
        if (k.met || k.tail)
#pragma unroll
            for (int j = 0; j < NX; ++j)
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int i = 0; i < 4; ++i) p[j][h][i] = fix(k, j, h, i, p[j][h][i], ref[j]);
    };
    auto over = [&](const float (&p)[NX][2][4]) {
        float top = kNothing;
#pragma unroll
        for (int j = 0; j < NX; ++j)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < 4; ++i) top = fmaxf(top, p[j][h][i]);
        return __any(top > kTop);
    };
    // moves the references of the rows that need it; returns the logits minus the new ones, and what the sums so far are multiplied by
    auto move = [&](const Tile &k, const f32x4 (&S)[NX][2], bool biased, float (&ref)[NX], float (&p)[NX][2][4], float (&old)[NX]) {
        float zero[NX];
#pragma unroll
        for (int j = 0; j < NX; ++j) zero[j] = 0.0f;
        logits(k, S, biased, zero, p);
#pragma unroll
        for (int j = 0; j < NX; ++j) {
            float z = kNothing;
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < 4; ++i) z = fmaxf(z, p[j][h][i]);
            z = fmaxf(z, __shfl_xor(z, 16));
            z = fmaxf(z, __shfl_xor(z, 32));
            const float to = z - ref[j] > kTop ? z - kStart : ref[j];
            old[j] = exp2_hw(ref[j] - to);
            ref[j] = to;
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < 4; ++i) p[j][h][i] -= to;
        }
    };
    auto sum = [&](const float (&p)[2][4]) { return ((p[0][0] + p[0][1]) + (p[0][2] + p[0][3])) + ((p[1][0] + p[1][1]) + (p[1][2] + p[1][3])); };
    auto exps = [&](float (&p)[NX][2][4]) {
#pragma unroll
        for (int j = 0; j < NX; ++j)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < 4; ++i) p[j][h][i] = exp2_hw(p[j][h][i]);
    };
    auto pack = [&](const Tile &k, float (&p)[NX][2][4], V (&W)[NX][NP]) {
        if (MODE == kRows && (k.neg || k.met))
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float s = info(k, 16 * h + 4 * g + i)[2];
#pragma unroll
                    for (int j = 0; j < NX; ++j) p[j][h][i] *= k.met && (hit[j] >> (4 * h + i) & 1) ? -s : s;
                }
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
    // the weights of a tile; `pending`: what has to be added to O before it is rescaled
    auto weigh = [&](const Tile &k, const f32x4 (&S)[NX][2], auto &&pending, float (&p)[NX][2][4]) {
        if (k.met || k.tail) special(k, S);
        float old[NX];
        if constexpr (TWO) {
            logits(k, S, false, Ml, p);
            if (over(p)) {
                move(k, S, false, Ml, p, old);
#pragma unroll
                for (int j = 0; j < NX; ++j) l[j] *= old[j];
            }
            exps(p);
#pragma unroll
            for (int j = 0; j < NX; ++j) l[j] += sum(p[j]);
        }
        logits(k, S, BIAS, M, p);
        if (!NOREF && over(p)) {
            pending();
            move(k, S, BIAS, M, p, old);
#pragma unroll
            for (int j = 0; j < NX; ++j) {
                if (!TWO) l[j] *= old[j];
                if (MODE != kStats)
#pragma unroll
                    for (int ob = 0; ob < OB; ++ob) O[ob][j] *= old[j];
            }
        }
        exps(p);
        if (MODE != kRows && !TWO)
#pragma unroll
            for (int j = 0; j < NX; ++j) l[j] += sum(p[j]);
    };

    if (ntiles) {
        typedef std::integral_constant<int, 0> Zero;
        if constexpr (MODE == kStats && NBUF >= 3) {
            // first product of the next tile beside the weights of this one; tile t + NBUF - 1 takes the place of tile t - 1
            f32x4 S[NX][2], next[NX][2];
            arrived(std::integral_constant<int, NBUF - 2>{});
            if (live) first_product(0, S);
            for (uint32_t t = 0; t < ntiles; ++t) {
                arrived(std::integral_constant<int, NBUF - 3>{});      // tile t + 1; every wave is through with tile t - 1
                load(t + NBUF - 1);
                if (live) {
                    float p[NX][2][4];
                    first_product((t + 1) % NBUF, next);
                    weigh(look(t), S, [] {}, p);
#pragma unroll
                    for (int j = 0; j < NX; ++j) { S[j][0] = next[j][0]; S[j][1] = next[j][1]; }
                }
            }
        } else if constexpr (C::PIPE) {
            // tile t + NBUF - 2 takes the place of tile t - 2
            f32x4 S[NX][2], next[NX][2];
            V W[NX][NP];
#pragma unroll
            for (int j = 0; j < NX; ++j)
#pragma unroll
                for (int p = 0; p < NP; ++p) W[j][p] = __builtin_bit_cast(V, u32x4{0, 0, 0, 0});
            arrived(std::integral_constant<int, NBUF - 2>{});
            if (live) first_product(0, S);
            for (uint32_t t = 0; t < ntiles; ++t) {
                arrived(std::integral_constant<int, NBUF - 4>{});      // tile t + 1; every wave is through with tile t - 2
                if (t) load(t + NBUF - 2);
                if (live) {
                    float p[NX][2][4];
                    const Tile k = look(t);
                    // (the first time round the pending product is of no rows: weights of zero, and tile 0 so that no stale bits are read)
                    const uint32_t before = t ? (t - 1) % NBUF : 0;
                    first_product((t + 1) % NBUF, next);
                    weigh(k, S, [&] {
                        second_product(before, W);
#pragma unroll
                        for (int j = 0; j < NX; ++j)
#pragma unroll
                            for (int q = 0; q < NP; ++q) W[j][q] = __builtin_bit_cast(V, u32x4{0, 0, 0, 0});
                    }, p);
                    second_product(before, W);
                    pack(k, p, W);
#pragma unroll
                    for (int j = 0; j < NX; ++j) { S[j][0] = next[j][0]; S[j][1] = next[j][1]; }
                }
            }
            if (live) second_product((ntiles - 1) % NBUF, W);
        } else {
            f32x4 S[NX][2];
            V W[NX][NP];
            float p[NX][2][4];
            for (uint32_t t = 0; t < ntiles; ++t) {
                if constexpr (NBUF > 1) {
                    arrived(std::integral_constant<int, NBUF - 2>{});  // tile t; every wave is through with tile t - 1
                    load(t + NBUF - 1);
                } else {
                    arrived(Zero{});
                }
                if (live) {
                    const Tile k = look(t);
                    first_product(t % NBUF, S);
                    weigh(k, S, [] {}, p);
                    if (MODE != kStats) {
                        pack(k, p, W);
                        second_product(t % NBUF, W);
                    }
                }
                if (NBUF == 1 && t + 1 < ntiles) {
                    __syncthreads();
                    load(t + 1);
                }
            }
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");               // no load may write to LDS that is no longer ours
    }
    finish<DT, MODE, OB, NX>(A, x0, n, g, slice, split, M, TWO ? Ml : M, l, O);
}

}  // namespace rg
