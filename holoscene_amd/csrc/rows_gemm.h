// rows_gemm.h -- the matrix products of the gated feed-forward block (gated_mlp_*.hip) on the 16-bit matrix cores.
//
//     C [I, J] = sum over segments of  A_s [I, K] . B_s [J, K]^T,   fp32 accumulators
//
// A segment is one pair of operands.  One: a plain product.  Two: gx = gg Wg + gu Wu in one pass.  Six: an fp32 product, whose operands
// are sums of three bf16 planes each (gemm_split.hip has the arithmetic: the plane products of combined weight >= 2^-16, smallest first).
// Either operand may have K as its contiguous index ([rows, K], ld) or as its strided one ([K, rows], ld); all four products of the
// block and its gradient are of that form, so nothing is ever transposed in memory.
//
// Workgroup = one BM x BN tile, K in steps of 64 through LDS, two buffers: step s + 1 is requested (LDS-DMA, 16 bytes a lane, no registers) before
// step s is multiplied.  Chunks of 16 bytes are permuted on their way in (the DMA's LDS addresses are fixed, the lane's global address is free)
// so that every fragment read is free of bank conflicts without padding: K-contiguous tiles [rows][64] exchange chunk c of row r with c ^ (r & 7);
// K-strided tiles [64][rows] exchange the 32-byte unit u of row k with u ^ (k & 3 | (k >> 3 & 1) << 2) and are read with the transposing
// ds_read_b64_tr_b16.  What lies outside an operand is requested at an address beyond the buffer descriptor, which reads as zero.
//
// The tile's orientation in the matrix instruction is C^T (its rows = J): a lane then holds four consecutive columns of one row of C.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <type_traits>

#include "holoscene_hip.h"
#include "launch_util.h"
#include "row_types.h"

namespace hs_gemm {

using namespace hs_row;

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(4))) int i32x4;
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef short i16x8 __attribute__((ext_vector_type(8)));

constexpr int BK = 64;
constexpr int kMaxSeg = 12;

struct Seg { const void *a, *b, *b1; };          // b1: the up projection's weights beside the gate's (EPI_GATE)

struct Args {
    Seg seg[2][kMaxSeg];                          // [problem][segment]
    int32_t n_seg;
    int64_t lda, ldb;                             // in elements, multiples of 8
    int64_t I;
    int32_t J, K;
    int32_t tiles_i, tiles_j, slices;
    // EPI_STORE
    void *out[2];                                 // per problem
    int64_t ldo;
    int64_t slice_stride;                         // elements between partial results (slices > 1: fp32)
    // gate epilogues: G, U [I, ldh] in the user's type; H or (gg, gu) as operands [planes][I][ldh]
    void *g, *u, *h, *gg, *gu;
    int64_t ldh, plane;                           // elements between planes
    int32_t act;
};

enum { EPI_STORE = 0, EPI_PARTIAL = 1, EPI_GATE = 2, EPI_GATE_BWD = 3 };

// ------------------------------------------------------------------------------------------------ activations (fp32)
// act(g) and, with `d`, act'(g).  expf / erff / tanhf are the library's fp32 functions.
__device__ __forceinline__ float activation(int act, float g, float *d) {
    if (act == HS_ACT_SILU || act == HS_ACT_SIGMOID) {
        const float s = 1.f / (1.f + expf(-g));
        if (act == HS_ACT_SIGMOID) {
            if (d) *d = s * (1.f - s);
            return s;
        }
        if (d) *d = s * (1.f + g * (1.f - s));
        return g * s;
    }
    if (act == HS_ACT_RELU) {
        if (d) *d = g > 0.f ? 1.f : 0.f;
        return g > 0.f ? g : (g == g ? 0.f : g);
    }
    if (act == HS_ACT_GELU) {
        const float c = 0.5f * (1.f + erff(g * 0.70710678118654752f));
        if (d) *d = c + g * expf(-0.5f * g * g) * 0.39894228040143268f;
        return g * c;
    }
    const float k = 0.79788456080286536f, t = tanhf(k * (g + 0.044715f * g * g * g));       // HS_ACT_GELU_TANH
    if (d) *d = 0.5f * (1.f + t) + 0.5f * g * (1.f - t * t) * k * (1.f + 0.134145f * g * g);
    return 0.5f * g * (1.f + t);
}

// ------------------------------------------------------------------------------------------------ three bf16 planes of an fp32 value
// v = p0 + p1 + p2 up to 2^-24 |v|.  A value that rounds to infinity is cut instead of rounded, an infinity or NaN stays in plane 0 alone.
__device__ __forceinline__ void split3(float v, bf16_t (&p)[3]) {
    const uint32_t bits = __float_as_uint(v);
    p[0] = (bf16_t)v;
    float r = (float)p[0];
    if (((bits >> 23) & 0xffu) == 0xffu) {
        p[1] = p[2] = (bf16_t)0.f;
        return;
    }
    if (((__float_as_uint(r) >> 23) & 0xffu) == 0xffu) {
        r = __uint_as_float(bits & 0xffff0000u);
        p[0] = (bf16_t)r;
    }
    v -= r;
    p[1] = (bf16_t)v;
    v -= (float)p[1];
    p[2] = (bf16_t)v;
}

// four consecutive elements of an operand that a later product reads: one plane in the 16-bit types, three for fp32
template <typename T, typename U> __device__ __forceinline__ void store_operand4(void *base, int64_t plane, int64_t at, const float (&v)[4]) {
    if constexpr (sizeof(U) == 4) {
        Pack<bf16_t, 4> o[3];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            bf16_t p[3];
            split3(v[e], p);
            o[0].v[e] = p[0]; o[1].v[e] = p[1]; o[2].v[e] = p[2];
        }
#pragma unroll
        for (int q = 0; q < 3; q++) *reinterpret_cast<Pack<bf16_t, 4> *>((bf16_t *)base + q * plane + at) = o[q];
    } else {
        Pack<U, 4> o;
#pragma unroll
        for (int e = 0; e < 4; e++) o.v[e] = from_f32<U>(v[e]);
        *reinterpret_cast<Pack<U, 4> *>((U *)base + at) = o;
    }
}

// ------------------------------------------------------------------------------------------------ the kernel
__device__ __forceinline__ uint32_t lds_addr(const void *p) { return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char *)p; }

// one LDS-DMA request: lane l's 16 bytes at base + voff land at lds + 16 l.  (The descriptor covers 2 GiB from the step's base; a lane with
// nothing to read passes kOutside and receives zeros.)  The compiler's own LDS-DMA builtin would wait for every request in front of
// the next LDS read (wgrad_pairs.hip); the waits are in wait_and_meet.
constexpr uint32_t kOutside = 0xfffffff0u, kDescBytes = 0x7fffffffu;
__device__ __forceinline__ i32x4 descriptor(const void *p) {
    const uint64_t a = (uint64_t)(uintptr_t)p;
    return i32x4{(int)__builtin_amdgcn_readfirstlane((int)(uint32_t)a), (int)__builtin_amdgcn_readfirstlane((int)((uint32_t)(a >> 32) & 0xffffu)), (int)kDescBytes, 0x00020000};
}
__device__ __forceinline__ void dma16(const i32x4 &desc, uint32_t voff, uint32_t to_lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(to_lds), "v"(voff), "s"(desc) : "memory");
}
__device__ __forceinline__ void wait_and_meet() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

template <typename T> __device__ __forceinline__ f32x4 mfma(i16x8 a, i16x8 b, f32x4 c) {
    if constexpr (__is_same(T, bf16_t)) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

typedef __attribute__((address_space(3))) const i16x8 *lds_frag_t;
typedef __attribute__((address_space(3))) i16x4 *lds_tr_t;

// One operand's side of a tile: R rows of C's index by 64 of K, WAVES waves requesting it, OWN units of 16 rows to a wave's products.
template <int R, bool KS, int WAVES, int OWN> struct Side {
    static constexpr int kBytes = R * BK * 2;
    static constexpr int kReq = kBytes / 1024 / WAVES;       // requests per wave and step
    static constexpr int kChunks = R / 8;                    // K-strided: 16-byte chunks of a row
    static constexpr int kUnits = R / 16;
    static_assert(kReq >= 1 && kBytes % (1024 * WAVES) == 0, "tile too small for its waves");
    uint32_t voff[kReq];
    int kpos[kReq];              // where along K this lane's chunk lies inside a step (first element)

    // rows: what is left of the operand from the tile's first row on (not clamped to R); second: a request of the tile's second half counts its rows from
    // the half's own start (two weights side by side)
    __device__ __forceinline__ void init(int wave, int lane, int64_t rows, int64_t ld, bool halves) {
#pragma unroll
        for (int q = 0; q < kReq; q++) {
            const int req = wave * kReq + q;
            if constexpr (!KS) {
                int row = req * 8 + (lane >> 3);
                const int chunk = (lane & 7) ^ (row & 7);
                if (halves && row >= R / 2) row -= R / 2;
                kpos[q] = chunk * 8;
                voff[q] = row < rows ? (uint32_t)(row * ld * 2 + chunk * 16) : kOutside;
            } else {
                const int k = req * (64 / kChunks) + lane / kChunks, slot = lane % kChunks;
                const int g = ((k & 3) | (((k >> 3) & 1) << 2)) & (kUnits - 1);
                const int chunk = (((slot >> 1) ^ g) << 1) | (slot & 1);
                kpos[q] = k;
                voff[q] = chunk * 8 < rows ? (uint32_t)(k * ld * 2 + chunk * 16) : kOutside;
            }
        }
    }
    // a step's requests; k_left = what is left of K from the step's start on
    __device__ __forceinline__ void request(int wave, const void *base, const void *base1, int64_t k_left, uint32_t to_lds) const {
        const i32x4 d0 = descriptor(base), d1 = descriptor(base1);
#pragma unroll
        for (int q = 0; q < kReq; q++) {
            const uint32_t v = kpos[q] < k_left ? voff[q] : kOutside;
            const bool upper = !KS && (wave * kReq + q) * 8 >= R / 2;
            const uint32_t at = __builtin_amdgcn_readfirstlane((int)(to_lds + (uint32_t)(wave * kReq + q) * 1024u));
            dma16(upper ? d1 : d0, v, at);
        }
    }
    // Fragments of 16 rows x 32 of K: lane l holds row (l & 15), K = 8 (l >> 4) .. + 7.  unit0: the first of the wave's units (16 rows each).
    static constexpr int kOwn = KS ? OWN : 2;
    uint32_t lane_at[kOwn];      // K-contiguous: by half of the step; K-strided: by unit
    __device__ __forceinline__ void init_frags(int lane, int unit0) {
        const int i = lane & 15, q = lane >> 4;
        if constexpr (!KS) {
#pragma unroll
            for (int ks = 0; ks < 2; ks++) lane_at[ks] = (uint32_t)(unit0 * 2048 + i * 128 + (((ks * 4 + q) ^ (i & 7)) * 16));
        } else {
            const int g = ((i >> 2) | ((q & 1) << 2)) & (kUnits - 1);
#pragma unroll
            for (int n = 0; n < OWN; n++)
                lane_at[n] = (uint32_t)((8 * q + (i >> 2)) * R * 2 + (((unit0 + n) ^ g) * 32) + (i & 3) * 8);       // (g < 8: changes the low bits only)
        }
    }
    // `own`: which of the wave's units; `ahead`: rows further on (compile-time constants)
    __device__ __forceinline__ i16x8 fragment(uint32_t buf, int own, int ks, uint32_t ahead = 0) const {
        if constexpr (!KS) {
            return *(lds_frag_t)(uintptr_t)(buf + lane_at[ks] + (uint32_t)own * 2048u + ahead * 128u);
        } else {
            const uint32_t at = buf + lane_at[own] + (uint32_t)ks * (32u * R * 2u);
            const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_tr_t)(uintptr_t)at);
            const i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_tr_t)(uintptr_t)(at + 4u * R * 2u));
            return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        }
    }
};

// T: the matrix instruction's type; U: the user's type (float: T = bf16, planes).
template <typename T, typename U, int BM, int BN, int WI, int WJ, bool AKS, bool BKS, int EPI>
__global__ __launch_bounds__(64 * WI * WJ) void k_rows_gemm(const Args p) {
    constexpr int WAVES = WI * WJ, MT = BM / WI / 16, NT = BN / WJ / 16;
    constexpr bool DUAL = EPI == EPI_GATE;
    constexpr int TJ = DUAL ? BN / 2 : BN;                   // columns of C per tile
    using SA = Side<BM, AKS, WAVES, MT>;
    using SB = Side<BN, BKS, WAVES, NT>;
    extern __shared__ __attribute__((aligned(1024))) char lds[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), wi = wave / WJ, wj = wave % WJ;
    // tiles: eight contiguous ranges, one per XCD (workgroups go round the XCDs), each walked in groups of 8 row tiles so that the tiles in flight
    // on an XCD share operands in its L2
    const int n_tiles = p.tiles_i * p.tiles_j, per_xcd = n_tiles / 8, rest = n_tiles % 8, xcd = blockIdx.x % 8, nth = blockIdx.x / 8;
    const int t = xcd * per_xcd + (xcd < rest ? xcd : rest) + nth;
    const int group = t / (8 * p.tiles_j), in_group = t - group * 8 * p.tiles_j, gi = p.tiles_i - group * 8 < 8 ? p.tiles_i - group * 8 : 8;
    const int64_t i0 = (int64_t)(group * 8 + in_group % gi) * BM;
    const int j0 = (in_group / gi) * TJ;
    const Seg *segs = p.seg[blockIdx.z];

    SA sa;
    SB sb;
    sa.init(wave, lane, p.I - i0, p.lda, false);
    sb.init(wave, lane, (int64_t)p.J - j0, p.ldb, DUAL);
    sa.init_frags(lane, wi * MT);
    sb.init_frags(lane, DUAL ? wj * (NT / 2) : wj * NT);
    const uint32_t lds0 = lds_addr(lds);
    const int steps_k = (p.K + BK - 1) / BK, steps = steps_k * p.n_seg;
    const int s_begin = (int)((int64_t)steps * blockIdx.y / p.slices), s_end = (int)((int64_t)steps * (blockIdx.y + 1) / p.slices);
    const int64_t a_step = AKS ? BK * p.lda * 2 : BK * 2, b_step = BKS ? BK * p.ldb * 2 : BK * 2;
    const int64_t a_tile = AKS ? i0 * 2 : i0 * p.lda * 2, b_tile = BKS ? (int64_t)j0 * 2 : (int64_t)j0 * p.ldb * 2;
    auto request = [&](int s, int buf) {
        const int sg = s / steps_k, kk = s - sg * steps_k;
        const char *a = (const char *)segs[sg].a + a_tile + kk * a_step, *b = (const char *)segs[sg].b + b_tile + kk * b_step;
        const char *b1 = DUAL ? (const char *)segs[sg].b1 + b_tile + kk * b_step : b;
        const int64_t left = p.K - (int64_t)kk * BK;
        const uint32_t at = lds0 + (uint32_t)buf * (SA::kBytes + SB::kBytes);
        sa.request(wave, a, a, left, at);
        sb.request(wave, b, b1, left, at + SA::kBytes);
    };
    f32x4 acc[MT][NT];
#pragma unroll
    for (int m = 0; m < MT; m++)
#pragma unroll
        for (int n = 0; n < NT; n++) acc[m][n] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (s_begin < s_end) request(s_begin, 0);
    int buf = 0;
    for (int s = s_begin; s < s_end; s++) {
        wait_and_meet();            // step s has landed for every wave; every wave is done with the other buffer
        if (s + 1 < s_end) request(s + 1, buf ^ 1);
        const uint32_t at = lds0 + (uint32_t)buf * (SA::kBytes + SB::kBytes);
#pragma unroll
        for (int ks = 0; ks < 2; ks++) {
            i16x8 fa[MT], fb[NT];
#pragma unroll
            for (int n = 0; n < NT; n++)         // (the tile's upper half: the up projection's rows)
                fb[n] = DUAL && n >= NT / 2 ? sb.fragment(at + SA::kBytes, n - NT / 2, ks, BN / 2) : sb.fragment(at + SA::kBytes, n, ks);
#pragma unroll
            for (int m = 0; m < MT; m++) fa[m] = sa.fragment(at, m, ks);
#pragma unroll
            for (int m = 0; m < MT; m++)
#pragma unroll
                for (int n = 0; n < NT; n++) acc[m][n] = mfma<T>(fb[n], fa[m], acc[m][n]);
        }
        buf ^= 1;
    }

    // ---- epilogue: acc[m][n][r] is row i0 + 16 (wi MT + m) + (lane & 15), column 16 unit + 4 (lane >> 4) + r
    const int li = lane & 15, lq = lane >> 4;
#pragma unroll
    for (int m = 0; m < MT; m++) {
        const int64_t i = i0 + (wi * MT + m) * 16 + li;
        if (i >= p.I) continue;
        if constexpr (EPI == EPI_STORE || EPI == EPI_PARTIAL) {
            using O = typename std::conditional<EPI == EPI_PARTIAL, float, U>::type;
            O *row = (O *)p.out[blockIdx.z] + (EPI == EPI_PARTIAL ? (int64_t)blockIdx.y * p.slice_stride : 0) + i * p.ldo;
            const bool wide = p.ldo % 4 == 0 && (uintptr_t)p.out[blockIdx.z] % (4 * sizeof(O)) == 0;
#pragma unroll
            for (int n = 0; n < NT; n++) {
                const int j = j0 + (wj * NT + n) * 16 + lq * 4;
                Pack<O, 4> o;
#pragma unroll
                for (int r = 0; r < 4; r++) o.v[r] = from_f32<O>(acc[m][n][r]);
                if (wide && j + 4 <= p.J) *reinterpret_cast<Pack<O, 4> *>(row + j) = o;
                else
#pragma unroll
                    for (int r = 0; r < 4; r++)
                        if (j + r < p.J) row[j + r] = o.v[r];
            }
        } else if constexpr (EPI == EPI_GATE) {
            // columns up to ldh are written: behind J both projections are zero (nothing was read), so the padding of G, U and H is zero
#pragma unroll
            for (int n = 0; n < NT / 2; n++) {
                const int j = j0 + (wj * (NT / 2) + n) * 16 + lq * 4;
                if (j >= p.ldh) continue;
                float h[4];
                Pack<U, 4> go, uo;
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const float g = acc[m][n][r], u = acc[m][n + NT / 2][r];
                    go.v[r] = from_f32<U>(g);
                    uo.v[r] = from_f32<U>(u);
                    h[r] = activation(p.act, g, nullptr) * u;
                }
                const int64_t at = i * p.ldh + j;
                if (p.g) {
                    *reinterpret_cast<Pack<U, 4> *>((U *)p.g + at) = go;
                    *reinterpret_cast<Pack<U, 4> *>((U *)p.u + at) = uo;
                }
                store_operand4<T, U>(p.h, p.plane, at, h);
            }
        } else {
#pragma unroll
            for (int n = 0; n < NT; n++) {
                const int j = j0 + (wj * NT + n) * 16 + lq * 4;
                if (j >= p.ldh) continue;
                const int64_t at = i * p.ldh + j;
                const Pack<U, 4> gi_ = *reinterpret_cast<const Pack<U, 4> *>((const U *)p.g + at), ui_ = *reinterpret_cast<const Pack<U, 4> *>((const U *)p.u + at);
                float gg[4], gu[4];
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    float d;
                    const float a = activation(p.act, to_f32(gi_.v[r]), &d), gh = acc[m][n][r];
                    gg[r] = gh * to_f32(ui_.v[r]) * d;
                    gu[r] = gh * a;
                }
                store_operand4<T, U>(p.gg, p.plane, at, gg);
                store_operand4<T, U>(p.gu, p.plane, at, gu);
            }
        }
    }
}

template <typename T, typename U, int BM, int BN, int WI, int WJ, bool AKS, bool BKS, int EPI>
inline int launch_tile(Args &p, int problems, hipStream_t s) {
    constexpr int TJ = EPI == EPI_GATE ? BN / 2 : BN;
    // the gate epilogues also write the padding columns up to ldh (< J + 8)
    const int64_t cols = EPI == EPI_GATE || EPI == EPI_GATE_BWD ? p.ldh : p.J;
    const int64_t ti = (p.I + BM - 1) / BM, tj = (cols + TJ - 1) / TJ;
    if (ti * tj > 0x7fffffff / 8 || p.slices > 65535) return HS_ERR_ARG;
    p.tiles_i = (int)ti;
    p.tiles_j = (int)tj;
    constexpr int lds = 2 * (BM + BN) * BK * 2;
    static hsLdsAttrOnce attr;
    const void *fn = (const void *)k_rows_gemm<T, U, BM, BN, WI, WJ, AKS, BKS, EPI>;
    attr.set(fn, lds);
    k_rows_gemm<T, U, BM, BN, WI, WJ, AKS, BKS, EPI><<<dim3((unsigned)(ti * tj), (unsigned)p.slices, (unsigned)problems), 64 * WI * WJ, lds, s>>>(p);
    return hipGetLastError() == hipSuccess ? HS_OK : HS_ERR_LAUNCH;
}

}  // namespace hs_gemm
