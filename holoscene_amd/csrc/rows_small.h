// rows_small.h -- the forward products of the gated feed-forward block for few rows (serving; small_rows() in gated_mlp.h), where reading the weights once is all there is.
//
// A workgroup takes 16 rows of the weights (with EPI_GATE of both projections) and every row of x; its waves share K in turns of 128 elements, so that the
// workgroup streams whole stretches of each weight row, straight from global memory into the registers of the matrix instructions (a lane's fragment is 16
// consecutive bytes).  The weights are the instruction's A: a lane ends with four consecutive results of one row of x.  The waves' partial sums meet in
// LDS in the order of the waves.  Any row distance and alignment is read in place -- a copy of an unaligned weight would cost more than the product.
// fp32: each operand is split into its three planes in registers.
// Bound by reading the weights: 1 x 4 096 x 12 288 bf16 37.3 us (gate and up, 201 MB, 5.4 TB/s) and 20.2 us (down, 101 MB, 5.0 TB/s); 13 x 1 000 x 2 730 f16 6.1 and 5.8 us (16 MB: latency).
#pragma once
#include "rows_gemm.h"

namespace hs_gemm {

struct SmallArgs {
    const void *x, *w, *w1;          // x [M, K] (EPI_STORE: H, an operand with `plane`); w (gate or down), w1 (up) [N, K]
    int64_t ldx, ldw, ldw1;
    int32_t M, N, K;
    int32_t act;
    void *y;                         // EPI_STORE: [M, N], row distance ldy
    int64_t ldy;
    float *g, *u;                    // EPI_GATE: G, U (may be NULL) and H as an operand
    void *h;
    int64_t ldh, plane;
};

constexpr int kSmallTurn = 128;      // elements of K a wave takes at a time: four fragments

// P fragments (planes) of the 8 elements from k on; zeros behind K
template <typename T, typename U, int P> __device__ __forceinline__ void small_fragment(const U *row, int k, int K, i16x8 (&f)[P]) {
    Loose<U, 8> v;
    if (k + 8 <= K) v = *reinterpret_cast<const Loose<U, 8> *>(row + k);
    else
#pragma unroll
        for (int e = 0; e < 8; e++) v.v[e] = k + e < K ? row[k + e] : (U)0.f;
    if constexpr (sizeof(U) == 4) {
        Pack<bf16_t, 8> o[3];
#pragma unroll
        for (int e = 0; e < 8; e++) {
            bf16_t q[3];
            split3(v.v[e], q);
            o[0].v[e] = q[0]; o[1].v[e] = q[1]; o[2].v[e] = q[2];
        }
#pragma unroll
        for (int q = 0; q < P; q++) f[q] = __builtin_bit_cast(i16x8, o[q]);
    } else {
        f[0] = __builtin_bit_cast(i16x8, v);
    }
}

// c += the product, of several planes the smaller ones' to `low` (which is 2^-8 of c at most: c is rounded once)
template <typename T, int P, int PX> __device__ __forceinline__ void small_product(const i16x8 (&w)[P], const i16x8 (&x)[PX], f32x4 &c, f32x4 &low) {
    if constexpr (P == 1 && PX == 2) low = mfma<T>(w[0], x[1], low);
    if constexpr (P == 3) {
#pragma unroll
        for (int t = 0; t < 5; t++) low = plane_product<T, P>(t, w, x, low);
    }
    c = mfma<T>(w[0], x[0], c);
}

// the same of H as EPI_GATE left it: planes of whole fragments
template <typename U, int P> __device__ __forceinline__ void small_planes(const void *h, int64_t plane, int64_t at, i16x8 (&f)[P]) {
    using E = typename std::conditional<P == 3, bf16_t, U>::type;
#pragma unroll
    for (int q = 0; q < P; q++) f[q] = *reinterpret_cast<const i16x8 *>((const E *)h + q * plane + at);
}

// FINE: H in two planes of a 16-bit type
template <typename T, typename U, int TOK, int WAVES, int EPI, bool FINE>
__global__ __launch_bounds__(64 * WAVES) void k_rows_small(const SmallArgs p) {
    constexpr bool GATE = EPI == EPI_GATE;
    constexpr int P = sizeof(U) == 4 ? 3 : 1, PX = FINE && !GATE ? 2 : P, NW = GATE ? 2 : 1;
    __shared__ f32x4 join[WAVES][NW * TOK][64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r = lane & 15, q = lane >> 4;
    const int n0 = blockIdx.x * 16, n = n0 + r < p.N ? n0 + r : p.N - 1;         // (rows behind the last read it again; their results are not stored)
    const U *wrow[2] = {(const U *)p.w + (int64_t)n * p.ldw, (const U *)p.w1 + (int64_t)n * p.ldw1};
    int64_t xrow[TOK];
#pragma unroll
    for (int t = 0; t < TOK; t++) xrow[t] = (int64_t)(t * 16 + r < p.M ? t * 16 + r : p.M - 1) * p.ldx;
    auto load_x = [&](int t, int k, int K, i16x8 (&f)[PX]) {
        if constexpr (GATE) small_fragment<T, U, P>((const U *)p.x + xrow[t], k, K, f);
        else small_planes<U, PX>(p.x, p.plane, xrow[t] + k, f);
    };
    f32x4 acc[NW][TOK], low[NW][TOK];
#pragma unroll
    for (int w = 0; w < NW; w++)
#pragma unroll
        for (int t = 0; t < TOK; t++) acc[w][t] = low[w][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int k0 = wave * kSmallTurn; k0 < p.K; k0 += WAVES * kSmallTurn) {
        if (k0 + kSmallTurn <= p.K) {
            // (four groups of rows: half a turn's fragments at a time, or the registers leave one wave a SIMD: 50 x 4 096 x 12 288 fp32 463 -> 393 us)
            constexpr int HALF = TOK == 4 ? 2 : 4;
#pragma unroll
            for (int s0 = 0; s0 < 4; s0 += HALF) {
                i16x8 fw[NW][HALF][P];
#pragma unroll
                for (int s = 0; s < HALF; s++)
#pragma unroll
                    for (int w = 0; w < NW; w++) small_fragment<T, U, P>(wrow[w], k0 + 32 * (s0 + s) + 8 * q, 0x7fffffff, fw[w][s]);
#pragma unroll
                for (int s = 0; s < HALF; s++)
#pragma unroll
                    for (int t = 0; t < TOK; t++) {
                        i16x8 fx[PX];
                        load_x(t, k0 + 32 * (s0 + s) + 8 * q, 0x7fffffff, fx);
#pragma unroll
                        for (int w = 0; w < NW; w++) small_product<T, P, PX>(fw[w][s], fx, acc[w][t], low[w][t]);
                    }
            }
        } else {
            for (int s = 0; s < 4 && k0 + 32 * s < p.K; s++) {
                i16x8 fw[NW][P];
#pragma unroll
                for (int w = 0; w < NW; w++) small_fragment<T, U, P>(wrow[w], k0 + 32 * s + 8 * q, p.K, fw[w]);
#pragma unroll
                for (int t = 0; t < TOK; t++) {
                    i16x8 fx[PX];
                    if (k0 + 32 * s + 8 * q < p.K) load_x(t, k0 + 32 * s + 8 * q, p.K, fx);
                    else
#pragma unroll
                        for (int c = 0; c < PX; c++) fx[c] = i16x8{0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
                    for (int w = 0; w < NW; w++) small_product<T, P, PX>(fw[w], fx, acc[w][t], low[w][t]);
                }
            }
        }
    }
#pragma unroll
    for (int w = 0; w < NW; w++)
#pragma unroll
        for (int t = 0; t < TOK; t++) {
            if constexpr (P == 1 && PX == 2) {          // (an infinite weight times H's lower plane: any value, see rows_gemm.h)
#pragma unroll
                for (int e = 0; e < 4; e++) low[w][t][e] = finite_part(low[w][t][e]);
            }
            join[wave][w * TOK + t][lane] = PX > 1 ? acc[w][t] + low[w][t] : acc[w][t];
        }
    __syncthreads();
    // a wave per 16 rows of x: row t 16 + r, results n0 + 4 q ..
    for (int t = wave; t < TOK; t += WAVES) {
        f32x4 sum[NW];
#pragma unroll
        for (int w = 0; w < NW; w++) {
            sum[w] = join[0][w * TOK + t][lane];
            for (int o = 1; o < WAVES; o++) sum[w] += join[o][w * TOK + t][lane];
        }
        const int m = t * 16 + r, j = n0 + q * 4;
        if (m >= p.M) continue;
        if constexpr (GATE) {
            with_activation(p.act, [&](auto act) {
                float unused;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    if (j + e >= p.ldh) continue;
                    const bool in = j + e < p.N;                                 // (H, G, U: zeros up to ldh)
                    const float g = in ? sum[0][e] : 0.f, u = in ? sum[NW - 1][e] : 0.f, h = activation<decltype(act)::value, false>(g, unused) * u;
                    const int64_t at = (int64_t)m * p.ldh + j + e;
                    if (p.g) {
                        p.g[at] = g;
                        p.u[at] = u;
                    }
                    if constexpr (P == 3) {
                        bf16_t o[3];
                        split3(h, o);
#pragma unroll
                        for (int c = 0; c < 3; c++) ((bf16_t *)p.h)[c * p.plane + at] = o[c];
                    } else if constexpr (FINE) {
                        U o[2];
                        split2(h, o);
                        ((U *)p.h)[at] = o[0];
                        ((U *)p.h)[p.plane + at] = o[1];
                    } else {
                        ((U *)p.h)[at] = from_f32<U>(h);
                    }
                }
            });
        } else {
            U *y = (U *)p.y + (int64_t)m * p.ldy + j;
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (j + e < p.N) y[e] = from_f32<U>(sum[0][e]);
        }
    }
}

template <typename T, typename U, int EPI, bool FINE> inline int launch_small(const SmallArgs &p, hipStream_t s) {
    // (the down projection has few workgroups: 1 x 4 096 x 12 288 bf16 25.1 us with eight waves, 20.5 with 16; fp32 the same with either)
    constexpr int WAVES = EPI == EPI_GATE ? 4 : sizeof(U) == 2 ? 16 : 8;
    const int64_t cols = EPI == EPI_GATE ? p.ldh : p.N;
    const unsigned blocks = (unsigned)((cols + 15) / 16);
    if (p.M <= 16) k_rows_small<T, U, 1, WAVES, EPI, FINE><<<blocks, 64 * WAVES, 0, s>>>(p);
    else if (p.M <= 32) k_rows_small<T, U, 2, WAVES, EPI, FINE><<<blocks, 64 * WAVES, 0, s>>>(p);
    else if constexpr (sizeof(U) == 4) k_rows_small<T, U, 4, WAVES, EPI, FINE><<<blocks, 64 * WAVES, 0, s>>>(p);
    else return HS_ERR_ARG;
    return hipGetLastError() == hipSuccess ? HS_OK : HS_ERR_LAUNCH;
}

}  // namespace hs_gemm
