// rg_softmax_thin.h -- the pass of the softmax operators for few stationary rows: bound by memory, so the streamed rows are
// read once for 64 of them, in the caller's type and layout, through registers (where fp32 rows are split), and every wave holds one block of 16 rows x.
// rg_softmax_pass.h has the mathematics, the operand layouts and the LDS swizzle.
#pragma once
#include "rg_softmax_pass.h"

namespace rg {

template <int DT, int KS>
struct ThinCfg {
    static constexpr int NP = DT == RG_DTYPE_F32 ? 2 : 1;
    static constexpr int OB = KS == 7 ? 13 : 2 * KS;
    static constexpr int XT = 64;
    static constexpr int TY = 32;
    static constexpr int PITCH = (KS * 64 + 255) / 256 * 256;
    static constexpr int PLANE = TY * PITCH;
    static constexpr int BUF = NP * PLANE;
    // tiles a turn: of short rows several, for the bytes that are on their way between two barriers (16 queries on 4M x 64, loss: fp16 one tile
    // 257 us, four 124 us; fp32 one 518 us, two 309 us; on 2M x 128 fp16 one 140 us, two 115 us)
    static constexpr int TURN = DT == RG_DTYPE_F32 ? (KS <= 4 ? 2 : 1) : KS <= 2 ? 4 : KS <= 4 ? 2 : 1;
    static constexpr int LPR = KS < 4 ? 4 * KS : 16;            // lanes that load a row
    static constexpr int ROWS = 256 / LPR, RPT = TURN * TY / ROWS;      // rows loaded at once, and by a thread
    static constexpr int NBUF = 2 * TURN * BUF <= 128 * 1024 ? 2 : 1;
    static constexpr int LDS = NBUF * TURN * (BUF + TY * 8);    // a factor and a bias per row
    static constexpr int WPS = (DT == RG_DTYPE_F32 ? KS <= 8 : KS <= 16) ? 2 : 1;
};

template <int DT, int KS, int MODE>
__global__ void __launch_bounds__(256, (ThinCfg<DT, KS>::WPS)) rg_softmax_thin_kernel(PassArgs A) {
    typedef ThinCfg<DT, KS> C;
    typedef typename Elem<DT>::T T;
    typedef typename Frag<DT>::V V;
    constexpr int NP = C::NP, NX = 1, OB = C::OB, PITCH = C::PITCH, CI = (KS + 3) / 4;
    constexpr bool F32 = DT == RG_DTYPE_F32;
    constexpr float kTop = 15.0f, kStart = DT == RG_DTYPE_BF16 ? 0.0f : 7.0f;   // a weight is at most 2^15; the first largest one 2^0 / 2^7
    extern __shared__ char lds[];
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = lane & 15, g = lane >> 4;
    const uint32_t ntx = (A.nx + C::XT - 1) / C::XT, b = xcd_block(blockIdx.x, gridDim.x), split = b / ntx;
    const uint32_t ybeg = min(A.ny, split * A.rows_per_split), yend = min(A.ny, ybeg + A.rows_per_split);
    const uint32_t x0 = b % ntx * C::XT + wave * 16;
    const bool live = x0 < A.nx;                                // waves behind the last row only help to load
    const uint32_t dim = A.dim;
    const size_t esz = sizeof(T);

    V X[NX][KS][NP];
    float kx[NX];
    uint32_t target[NX];
#pragma unroll
    for (int j = 0; j < NX; ++j) {
        const uint32_t x = x0 + j * 16 + n;
        kx[j] = load_stationary<DT, KS, 1>(A, x, g, X[j]);
        target[j] = kNoTarget;
        if (x < A.nx) {
            const uint32_t t = A.targets[x];
            if (t != kNoTarget && t >= A.id_base && t - A.id_base >= ybeg && t - A.id_base < yend) target[j] = t - A.id_base;
        }
    }

    f32x4 O[MODE == kStats ? 1 : OB][NX];
    // M: reference of the weights of O; with fp32 rows those carry the rows' scales, so that the sum l has a reference Ml of its own
    constexpr bool TWO = F32 && MODE == kMean;
    constexpr bool SUM = softmax_sums_rounded(DT, MODE);
    float M[NX], l[NX], Ml[NX], R[NX];
#pragma unroll
    for (int j = 0; j < NX; ++j) {
        M[j] = Ml[j] = kNothing;
        l[j] = R[j] = 0.0f;
        if (MODE != kStats)
#pragma unroll
            for (int ob = 0; ob < OB; ++ob) O[ob][j] = f32x4{0, 0, 0, 0};
    }

    if (A.resume) take_up<DT, MODE, OB, NX>(A, x0, n, g, 0, split, M, Ml, l, R, O);

    // streaming: LPR lanes per row, rows lr, lr + ROWS, .. per thread
    const uint32_t lr = tid / C::LPR, lc = tid % C::LPR;
    Chunk<DT> stage[C::RPT][CI];
    auto fetch = [&](uint32_t y0) {
#pragma unroll
        for (int h = 0; h < C::RPT; ++h) {
            const uint32_t y = y0 + lr + C::ROWS * h;
            const char *row = static_cast<const char *>(A.y) + (size_t)y * A.ystride * esz;
#pragma unroll
            for (int i = 0; i < CI; ++i) stage[h][i] = fetch_chunk<DT, KS <= 2>(row, 8 * (lc + 16 * i), dim, y < yend);
        }
    };
    auto commit = [&](uint32_t buf) {
#pragma unroll
        for (int h = 0; h < C::RPT; ++h) {
            const uint32_t r = (lr + C::ROWS * h) % C::TY, t = buf * C::TURN + (lr + C::ROWS * h) / C::TY, sw = swizzle(r);
            char *tile = lds + t * C::BUF;
            float *yv = reinterpret_cast<float *>(lds + C::NBUF * C::TURN * C::BUF) + t * C::TY * 2;
            if (ragged<KS <= 2>(dim))
#pragma unroll
                for (int i = 0; i < CI; ++i) stage[h][i] = settle<DT>(stage[h][i], 8 * (lc + 16 * i), dim);
            int e = 0;
            float top = 0.0f;
            if constexpr (F32) {
                uint32_t m = 0;
#pragma unroll
                for (int i = 0; i < CI; ++i) m = max(m, __float_as_uint(absmax(stage[h][i])));
#pragma unroll
                for (int d = 1; d < C::LPR; d <<= 1) m = max(m, (uint32_t)__shfl_xor((int)m, d));
                top = __uint_as_float(m);
                e = row_exponent(top);
            }
            const float s = F32 ? pow2(-e) : 1.0f;
#pragma unroll
            for (int i = 0; i < CI; ++i) {
                const uint32_t c = lc + 16 * i;
                if (KS * 4 % 16 == 0 || c < (uint32_t)KS * 4) {
                    char *at = tile + r * PITCH + i * 256 + ((lc ^ sw) << 4);
                    if constexpr (F32) {
                        half8 hi, lo;
                        split8(stage[h][i], top, s, hi, lo);
                        *reinterpret_cast<half8 *>(at) = hi;
                        *reinterpret_cast<half8 *>(at + C::PLANE) = lo;
                    } else {
                        *reinterpret_cast<u32x4 *>(at) = stage[h][i].v;
                    }
                }
            }
            if (F32 && lc == 0) {
                yv[r] = row_factor(top, e);
                yv[32 + r] = MODE == kMean ? row_bias(top, e) : 0.0f;
            }
        }
    };

    // Where registers are few, a lane's LDS addresses are made of one, by its bits 5 - 7, for every read, not kept over the tiles (mean of 20 fp16
    // queries on 500k x 509 304 us, so 236 us; statistics, which have registers to spare, 177 us, so 181 us).
    constexpr bool MADE = KS > 12 && MODE == kMean;
    auto compute = [&](uint32_t t, uint32_t y0) {
        const char *tile = lds + t * C::BUF;
        const float *yv = reinterpret_cast<const float *>(lds + C::NBUF * C::TURN * C::BUF) + t * C::TY * 2;
        f32x4 S[2][NX];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int j = 0; j < NX; ++j) S[h][j] = f32x4{0, 0, 0, 0};
        {
            const uint32_t sw = swizzle(n);                     // (row + 16: the same swizzle)
            const char *row = tile + n * PITCH;
            uint32_t first = t * C::BUF + n * PITCH + ((g ^ sw) << 4);
            if (MADE) asm("" : "+v"(first));
            constexpr int PART = KS / softmax_parts(DT, KS);
            f32x4 sum[2][NX];
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                if (ks % PART == 0 && ks) {
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int j = 0; j < NX; ++j) {
                            sum[h][j] = ks == PART ? S[h][j] : sum[h][j] + S[h][j];
                            S[h][j] = f32x4{0, 0, 0, 0};
                        }
                }
                const uint32_t c = 4 * ks + g;
                const char *at = MADE ? lds + (first ^ (uint32_t)(ks % 4 << 6)) + ks / 4 * 256 : row + (c & ~15u) * 16 + (((c & 15) ^ sw) << 4);
                V a[2][NP];
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int p = 0; p < NP; ++p) a[h][p] = *reinterpret_cast<const V *>(at + h * 16 * PITCH + p * C::PLANE);
                if constexpr (F32) {
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int j = 0; j < NX; ++j) S[h][j] = mma(a[h][1], X[j][ks][0], S[h][j]);
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int j = 0; j < NX; ++j) S[h][j] = mma(a[h][0], X[j][ks][1], S[h][j]);
                }
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int j = 0; j < NX; ++j) S[h][j] = mma(a[h][0], X[j][ks][0], S[h][j]);
            }
            if (PART < KS)
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int j = 0; j < NX; ++j) S[h][j] = sum[h][j] + S[h][j];
        }
        f32x4 ky[2], bias[2];
        if (F32)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                ky[h] = *reinterpret_cast<const f32x4 *>(yv + 16 * h + 4 * g);
                bias[h] = *reinterpret_cast<const f32x4 *>(yv + 32 + 16 * h + 4 * g);
            }
        const bool tail = y0 + 32 > yend;
        const bool met = __any(target[0] - y0 < 32);            // a target of these rows lies in the tile
#pragma unroll
        for (int j = 0; j < NX; ++j) {
            const uint32_t x = x0 + j * 16 + n;
            uint32_t dead = 0;                                  // bits of the elements (h, i) that take no part
            if (met || tail) {
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint32_t r = 16 * h + 4 * g + i;
                        if (y0 + r == target[j]) {
                            float z = S[h][j][i];
                            if (F32) z *= ky[h][i];
                            A.own2[x] = z * kx[j];
                            dead |= 1u << (4 * h + i);
                        }
                        if (y0 + r >= yend) dead |= 1u << (4 * h + i);
                    }
            }
            // the logit of element (h, i), in units of log 2, minus a reference
            auto logit = [&](int h, int i, bool biased, float ref) {
                float z = S[h][j][i];
                if (F32) z *= ky[h][i];
                z = fmaf(z, kx[j], biased ? bias[h][i] - ref : -ref);
                if (met || tail)
                    if (dead >> (4 * h + i) & 1) z = -INFINITY;
                return z;
            };
            // weights 2^(logit - ref) under a reference that moves where one would pass 2^kTop; true where it moved, by a factor `old`
            auto weigh = [&](bool biased, float &ref, float &old, float (&p)[2][4]) {
                float top = kNothing;
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        p[h][i] = logit(h, i, biased, ref);
                        top = fmaxf(top, p[h][i]);
                    }
                const bool move = __any(top > kTop);
                if (move) {                                     // (of the rows that need it, whatever the others do)
                    float z = kNothing;
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int i = 0; i < 4; ++i) z = fmaxf(z, logit(h, i, biased, 0.0f));
                    z = fmaxf(z, __shfl_xor(z, 16));
                    z = fmaxf(z, __shfl_xor(z, 32));
                    top = fmaxf(top, __shfl_xor(top, 16));
                    top = fmaxf(top, __shfl_xor(top, 32));
                    const float to = top > kTop ? z - kStart : ref;
                    old = exp2_hw(ref - to);
                    ref = to;
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int i = 0; i < 4; ++i) p[h][i] = logit(h, i, biased, ref);
                }
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int i = 0; i < 4; ++i) p[h][i] = exp2_hw(p[h][i]);
                return move;
            };
            float p[2][4], old = 1.0f;
            if (TWO) {
                if (weigh(false, Ml[j], old, p)) l[j] *= old;
                l[j] += ((p[0][0] + p[0][1]) + (p[0][2] + p[0][3])) + ((p[1][0] + p[1][1]) + (p[1][2] + p[1][3]));
            }
            if (weigh(TWO, M[j], old, p)) {
                if (!TWO) l[j] *= old;
                if (SUM) R[j] *= old;
                if (MODE != kStats)
#pragma unroll
                    for (int ob = 0; ob < OB; ++ob) O[ob][j] *= old;
            }
            if (!TWO) l[j] += ((p[0][0] + p[0][1]) + (p[0][2] + p[0][3])) + ((p[1][0] + p[1][1]) + (p[1][2] + p[1][3]));
            if constexpr (MODE != kStats) {
                V w, wl;
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if constexpr (DT == RG_DTYPE_BF16) {
                            w[4 * h + i] = (__bf16)p[h][i];
                        } else {
                            w[4 * h + i] = (_Float16)p[h][i];
                            if (F32) wl[4 * h + i] = (_Float16)(p[h][i] - (float)w[4 * h + i]);
                        }
                    }
                if constexpr (SUM) R[j] += sum_of(w);
                S[0][j] = __builtin_bit_cast(f32x4, w);
                if (F32) S[1][j] = __builtin_bit_cast(f32x4, wl);
            }
        }
        if constexpr (MODE != kStats) {
            // lane (n, g) reads 8 bytes of row 4 g + n / 4 (and + 16) at dims 4 (n % 4) of the block, and receives dim n of rows 4 g .. + 3
            typedef __attribute__((address_space(3))) s16x4 *tr_ptr;
            const uint32_t r = 4 * g + (n >> 2), sw = swizzle(r);     // (row + 16: the same swizzle)
            const char *row = tile + r * PITCH + (n & 1) * 8;
            uint32_t second = t * C::BUF + r * PITCH + (((n >> 1 & 1) ^ sw) << 4) + (n & 1) * 8;
            if (MADE) asm("" : "+v"(second));
#pragma unroll
            for (int ob = 0; ob < OB; ++ob) {
                const uint32_t c = 2 * ob + ((n >> 1) & 1);
                const char *at = MADE ? lds + (second ^ (uint32_t)(ob % 8 << 5)) + ob / 8 * 256 : row + (c & ~15u) * 16 + (((c & 15) ^ sw) << 4);
                V a[NP];
#pragma unroll
                for (int p = 0; p < NP; ++p) {
                    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_ptr)(const_cast<char *>(at) + p * C::PLANE));
                    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_ptr)(const_cast<char *>(at) + p * C::PLANE + 16 * PITCH));
                    a[p] = __builtin_bit_cast(V, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
                }
#pragma unroll
                for (int j = 0; j < NX; ++j) {
                    if constexpr (F32) {
                        O[ob][j] = mma(a[1], __builtin_bit_cast(V, S[0][j]), O[ob][j]);
                        O[ob][j] = mma(a[0], __builtin_bit_cast(V, S[1][j]), O[ob][j]);
                    }
                    O[ob][j] = mma(a[0], __builtin_bit_cast(V, S[0][j]), O[ob][j]);
                }
            }
        }
    };

    if (ybeg < yend) {
        constexpr uint32_t STEP = C::TURN * C::TY;
        auto turn = [&](uint32_t buf, uint32_t y0) {
            if (!live) return;
#pragma unroll 1
            for (uint32_t t = 0; t < C::TURN && y0 + t * C::TY < yend; ++t) compute(buf * C::TURN + t, y0 + t * C::TY);
        };
        if constexpr (C::NBUF == 2) {
            fetch(ybeg);
            commit(0);
            __syncthreads();
            uint32_t buf = 0;
            for (uint32_t y0 = ybeg; y0 < yend; y0 += STEP, buf ^= 1) {
                const bool more = y0 + STEP < yend;
                if (more) fetch(y0 + STEP);
                turn(buf, y0);
                if (more) commit(buf ^ 1);
                __syncthreads();
            }
        } else {
            for (uint32_t y0 = ybeg; y0 < yend; y0 += STEP) {
                fetch(y0);
                commit(0);
                __syncthreads();
                turn(0, y0);
                __syncthreads();
            }
        }
    }

    finish<DT, MODE, OB, NX>(A, x0, n, g, 0, split, M, TWO ? Ml : M, l, R, O);
}

}  // namespace rg
