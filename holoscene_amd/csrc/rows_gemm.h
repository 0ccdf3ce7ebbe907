// rows_gemm.h -- the matrix products of the gated feed-forward block (gated_mlp_*.hip) on the 16-bit matrix cores.
//
//     C [I, J] = sum over segments of  A_s [I, K] . B_s [J, K]^T,   fp32 accumulators
//
// A segment is one pair of operands.  One: a plain product.  Two: gx = gg Wg + gu Wu in one pass.  An operand of the 16-bit types is one matrix; an fp32
// one is the sum of three bf16 planes, and its product six plane products (those of combined weight >= 2^-16, smallest first; gemm_split.hip has the
// arithmetic).  Small tiles have all planes in LDS together (P = 3): a step is 64 of K, each fragment takes part in up to three products.  The large tile has no
// room for that and takes the six as segments, one after the other (P = 1): it reads every plane twice, and still less per product.
// Either operand may have K as its contiguous index ([rows, K], ld) or as its strided one ([K, rows], ld); all four products of the
// block and its gradient are of that form, so nothing is ever transposed in memory.
//
// Workgroup = one BM x BN tile, K in steps of 64 through LDS, two to four buffers: one to three steps behind step s are requested (LDS-DMA, 16 bytes a lane, no
// registers) before step s is multiplied.  Chunks of 16 bytes are permuted on their way in (the DMA's LDS addresses are fixed, the lane's global address is free)
// so that every fragment read is free of bank conflicts without padding: K-contiguous tiles [rows][64] exchange chunk c of row r with c ^ (r & 7);
// K-strided tiles [64][rows] exchange the 32-byte unit u of row k with u ^ (k & 3 | (k >> 3 & 1) << 2) and are read with the transposing
// ds_read_b64_tr_b16.  What lies outside an operand is requested at an address beyond the buffer descriptor, which reads as zero.
//
// The tile's orientation in the matrix instruction is C^T (its rows = J): a lane then holds four consecutive columns of one row of C.
//
// Measured (medians of 30 passes), 8 192 x 4 096 x 12 288 bf16 (256 x 256 tiles): gate and up 1.41 ms (1.17 PFLOP/s, with act(G) U and G, U written), down 0.67 (1.23),
// gx 1.30 (1.27), gWg and gWu 1.37 (1.20), gWd 0.69 (1.20); the library's product of 8 192^3 reaches 1.40.  The matrix cores are busy 54 to 63 % of the cycles, the LDS 23 %, and the
// waves wait 30 % of theirs: what is left is the meeting of the waves at every step of 64.  At 131 072 x 256 x 1 024 a tile has four steps, and its beginning and end
// are half of it: gate 224 us (0.61 PFLOP/s), down 86, gx 162, gWg and gWu 144, gWd 100.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <type_traits>
#include <utility>

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
constexpr int64_t kMaxGrid = 0xffffffffll;        // threads along x in a launch

template <typename U> constexpr int planes() { return sizeof(U) == 4 ? 3 : 1; }

struct Seg { const void *a, *b, *b1; };          // b1: the up projection's weights beside the gate's (EPI_GATE)

struct Args {
    Seg seg[2][kMaxSeg];                          // [problem][segment]
    int32_t n_seg;
    int32_t low_seg;                              // how many of them, the first ones, are products of an operand's lower plane (16-bit types, fine() in gated_mlp.h)
    int64_t lda, ldb;                             // in elements, multiples of 8
    int64_t plane_a, plane_b;                     // bytes between planes
    int64_t I;
    int32_t J, K;                                 // K < 2^31 - BK (HS_GATED_MLP_MAX_ROWS): rounded up to whole steps in 32 bits
    int32_t tiles_i, tiles_j, problems, slices;
    // EPI_STORE
    void *out[2];                                 // per problem
    int64_t ldo;
    int64_t slice_stride;                         // elements between partial results (slices > 1: fp32)
    // gate kernels: G, U fp32 [I, ldh]; H or (gg, gu) as operands [planes][I][ldh]
    float *g, *u;
    void *h, *gg, *gu;
    int64_t ldh, plane;                           // plane: elements between planes
    int32_t act;
    // k_gate_bwd: the second product's operands are seg[1]
    int64_t lda2, ldb2, plane_a2, plane_b2;
};

// result; fp32 partial result; H (G, U); gg, gu from G, U; the last two with their results in two planes (16-bit types: fine() in gated_mlp.h)
enum { EPI_STORE = 0, EPI_PARTIAL = 1, EPI_GATE = 2, EPI_GATE_BWD = 3, EPI_GATE_FINE = 4, EPI_GATE_BWD_FINE = 5 };
constexpr bool gate_forward(int epi) { return epi == EPI_GATE || epi == EPI_GATE_FINE; }
constexpr bool gate_backward(int epi) { return epi == EPI_GATE_BWD || epi == EPI_GATE_BWD_FINE; }

// ------------------------------------------------------------------------------------------------ activations (fp32)
// act(g) and, with D, act'(g).  The logistic function is v_exp_f32 and v_rcp_f32 (one step each): its error is |g| 2^-24 relative to s (1 - s), below the
// rounding of g itself.  gelu_tanh: (1 + tanh z) / 2 is the logistic function of 2 z, so no difference of nearly equal numbers is formed.
__device__ __forceinline__ float logistic(float v) { return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(v * -1.4426950408889634f)); }

template <int ACT, bool D> __device__ __forceinline__ float activation(float g, float &d) {
    if constexpr (ACT == HS_ACT_SILU) {
        const float s = logistic(g);
        if constexpr (D) d = s * (1.f + g * (1.f - s));
        return g * s;
    } else if constexpr (ACT == HS_ACT_SIGMOID) {
        const float s = logistic(g);
        if constexpr (D) d = s * (1.f - s);
        return s;
    } else if constexpr (ACT == HS_ACT_RELU) {
        if constexpr (D) d = g > 0.f ? 1.f : 0.f;
        return g > 0.f ? g : (g == g ? 0.f : g);        // (a NaN stays one)
    } else if constexpr (ACT == HS_ACT_GELU) {
        const float c = 0.5f * (1.f + erff(g * 0.70710678118654752f));
        if constexpr (D) d = c + g * __builtin_amdgcn_exp2f(g * g * -0.72134752044448170f) * 0.39894228040143268f;
        return g * c;
    } else {                                            // HS_ACT_GELU_TANH: 2 sqrt(2 / pi) (g + 0.044715 g^3)
        const float s = logistic(1.5957691216057308f * (g + 0.044715f * g * g * g));
        const float t = s * (1.f - s);
        if constexpr (D) d = s + (t > 0.f ? g * t * 1.5957691216057308f * (1.f + 0.134145f * g * g) : 0.f);        // (t = 0: g^2 may be infinite)
        return g * s;
    }
}

// f(std::integral_constant<int, act>): the activation as a constant, one uniform branch for a whole epilogue
template <typename F> __device__ __forceinline__ void with_activation(int act, F f) {
    switch (act) {
        case HS_ACT_SILU: f(std::integral_constant<int, HS_ACT_SILU>{}); break;
        case HS_ACT_GELU: f(std::integral_constant<int, HS_ACT_GELU>{}); break;
        case HS_ACT_GELU_TANH: f(std::integral_constant<int, HS_ACT_GELU_TANH>{}); break;
        case HS_ACT_SIGMOID: f(std::integral_constant<int, HS_ACT_SIGMOID>{}); break;
        default: f(std::integral_constant<int, HS_ACT_RELU>{}); break;
    }
}

// ------------------------------------------------------------------------------------------------ three bf16 planes of an fp32 value
// v = p0 + p1 + p2 up to 2^-24 |v|.  A value that rounds to infinity is cut instead of rounded, an infinity or NaN stays in plane 0 alone.
__device__ __forceinline__ void split3(float v, bf16_t (&p)[3]) {
    const uint32_t bits = __float_as_uint(v);
    const bool finite = ((bits >> 23) & 0xffu) != 0xffu, big = (bits & 0x7fffffffu) >= 0x7f7f8000u;       // big: rounds to infinity (or is one)
    const float first = finite && big ? __uint_as_float(bits & 0xffff0000u) : v;
    p[0] = (bf16_t)first;
    const float r1 = finite ? v - (float)p[0] : 0.f;
    p[1] = (bf16_t)r1;
    p[2] = (bf16_t)(r1 - (float)p[1]);
}

// eight consecutive elements of an operand that a later product reads: one plane in the 16-bit types, three for fp32
template <typename U> __device__ __forceinline__ void store_operand8(void *base, int64_t plane, int64_t at, const float (&v)[8]) {
    if constexpr (sizeof(U) == 4) {
        Pack<bf16_t, 8> o[3];
#pragma unroll
        for (int e = 0; e < 8; e++) {
            bf16_t p[3];
            split3(v[e], p);
            o[0].v[e] = p[0]; o[1].v[e] = p[1]; o[2].v[e] = p[2];
        }
#pragma unroll
        for (int q = 0; q < 3; q++) *reinterpret_cast<Pack<bf16_t, 8> *>((bf16_t *)base + q * plane + at) = o[q];
    } else {
        Pack<U, 8> o;
#pragma unroll
        for (int e = 0; e < 8; e++) o.v[e] = from_f32<U>(v[e]);
        *reinterpret_cast<Pack<U, 8> *>((U *)base + at) = o;
    }
}

// eight consecutive floats
struct F8 { float v[8]; };
__device__ __forceinline__ F8 load8(const float *p) {
    const float4 a = reinterpret_cast<const float4 *>(p)[0], b = reinterpret_cast<const float4 *>(p)[1];
    return F8{{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w}};
}
// four elements of an operand of a 16-bit type in two planes, v = p0 + p1 up to the square of the type's rounding; an infinity or NaN stays in plane 0 alone
template <typename U> __device__ __forceinline__ void split2(float v, U (&p)[2]) {
    asm("" : "+v"(v));          // (both planes from this float: the compiler would round a product to float16 from its exact value in one place and from the float in another)
    p[0] = from_f32<U>(v);
    p[1] = __builtin_isfinite(to_f32(p[0])) ? from_f32<U>(v - to_f32(p[0])) : (U)0.f;
}
template <typename U> __device__ __forceinline__ void store_fine4(void *base, int64_t plane, int64_t at, const float (&v)[4]) {
    Pack<U, 4> o[2];
#pragma unroll
    for (int e = 0; e < 4; e++) {
        U p[2];
        split2(v[e], p);
        o[0].v[e] = p[0]; o[1].v[e] = p[1];
    }
#pragma unroll
    for (int q = 0; q < 2; q++) *reinterpret_cast<Pack<U, 4> *>((U *)base + q * plane + at) = o[q];
}
// the same of eight elements in LDS, rounded already
template <typename U> __device__ __forceinline__ void store_staged(void *base, int64_t plane, int64_t at, const U *s) {
    if constexpr (sizeof(U) == 4) store_operand8<U>(base, plane, at, load8(s).v);
    else *reinterpret_cast<Pack<U, 8> *>((U *)base + at) = *reinterpret_cast<const Pack<U, 8> *>(s);
}
__device__ __forceinline__ void store8(float *p, const F8 &f) {
    reinterpret_cast<float4 *>(p)[0] = make_float4(f.v[0], f.v[1], f.v[2], f.v[3]);
    reinterpret_cast<float4 *>(p)[1] = make_float4(f.v[4], f.v[5], f.v[6], f.v[7]);
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
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(to_lds), "v"(voff), "s"(desc) : "m0", "memory");
}
// everybody has this step's data (N of this wave's requests, for later steps, may still be under way) and is done with the previous step's
template <int N> __device__ __forceinline__ void wait_and_meet() { asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory"); }

__device__ __forceinline__ void meet() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }       // LDS only: stores to global memory stay in flight

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

// Which tile of which problem and slice a workgroup takes: eight contiguous ranges, one per XCD (workgroups go round the XCDs), the tiles of a slice next to each
// other, walked in groups of 8 row tiles, so that the tiles in flight on an XCD share operands in its L2.  (Slices spread over the XCDs, each of which then reads
// the whole of the smaller operand: gWd of 131 072 x 256 x 1 024 128 us against 99, gWg and gWu of 4 096 x 256 x 683 in fp32 29 against 23.)  Problems that are
// not sliced follow one another (blockIdx.y).
struct TilePlace { int i, j, problem, slice; };
__device__ __forceinline__ TilePlace tile_place(int tiles_i, int tiles_j, int problems, int slices) {      // problems: side by side in a slice
    const int tiles = tiles_i * tiles_j, n = tiles * problems * slices, per_xcd = n / 8, rest = n % 8, xcd = blockIdx.x % 8;
    const int t = xcd * per_xcd + (xcd < rest ? xcd : rest) + blockIdx.x / 8;
    const int which = t / tiles, at = t - which * tiles;
    const int group = at / (8 * tiles_j), in = at - group * 8 * tiles_j, rows = tiles_i - group * 8 < 8 ? tiles_i - group * 8 : 8;
    return TilePlace{group * 8 + in % rows, in / rows, which % problems + (int)blockIdx.y, which / problems};
}

// Results of the gate kernels through LDS: MP of each wave's MT row groups at a time (as many as MOST and the workgroup's LDS admit), COLS columns of U a row, items of
// 8 of the TJ result columns.
template <typename U, int COLS, int TJ, int MT, int WI, int WAVES, int MOST, int LDS> struct Staging {
    static constexpr int kPitch = COLS + 16 / (int)sizeof(U);
    static constexpr int bytes(int mp) { return WI * mp * 16 * kPitch * (int)sizeof(U); }
    static constexpr int most(int mp) { return mp > 1 && (mp > MOST || bytes(mp) > LDS) ? most(mp / 2) : mp; }
    static constexpr int MP = most(MT), kPasses = MT / MP, kLines = WI * MP * 16, kItems = kLines * (TJ / 8);
    static_assert(bytes(MP) <= LDS && MT % MP == 0, "the epilogue's tile must fit");
    // f(row of the tile (of pass 0), line of the stage, column) for this thread's items
    template <typename F> static __device__ __forceinline__ void copy_out(int tid, F f) {
#pragma unroll
        for (int k = 0; k < (kItems + 64 * WAVES - 1) / (64 * WAVES); k++) {
            const int item = tid + k * 64 * WAVES, line = item / (TJ / 8);
            if (kItems % (64 * WAVES) != 0 && item >= kItems) break;
            f(line / (MP * 16) * (MT * 16) + line % (MP * 16), line, item % (TJ / 8) * 8);
        }
    }
};

template <int... I, typename F> __device__ __forceinline__ void static_for(std::integer_sequence<int, I...>, F f) { (f(std::integral_constant<int, I>{}), ...); }

// c += the product of two fragments of P planes, the smallest plane products first
template <typename T, int P> __device__ __forceinline__ f32x4 plane_product(int term, const i16x8 (&w)[P], const i16x8 (&x)[P], f32x4 c) {
    constexpr int pw[6] = {0, 1, 2, 0, 1, 0}, px[6] = {2, 1, 0, 1, 0, 0};        // (which side is called the first does not matter)
    return P == 1 ? mfma<T>(w[0], x[0], c) : mfma<T>(w[pw[term]], x[px[term]], c);
}

// One step (64 of K) of a wave's products.  Fragments are requested PF groups of matrix instructions ahead of their use, and the order written here is pinned
// (sched_group_barrier: 0x100 LDS reads, 0x8 matrix instructions): left to itself the compiler puts every read directly in front of its use, with a wait for
// its whole latency between (8 192 x 4 096 x 12 288: 774 -> 699 us).  a(m, ks, plane), b(n, ks, plane): the fragments; RA, RB: LDS instructions of one.
// request(): the next step's LDS-DMA, issued while the first fragments are on their way.  P == 3: the five smaller plane products are summed in `low`, 2^-8 of acc at most,
// so that acc is rounded once in 32 of K and not six times (error of y against 64 bits at 3 033 x 2 016 x 64: 1.1e-6 -> 4.2e-7; fp32 library products 6.0e-7).
template <typename T, int MT, int NT, int P, int RA, int RB, typename A, typename B, typename R>
__device__ __forceinline__ void multiply_step(A a, B b, R request, f32x4 (&acc)[MT][NT], f32x4 (&low)[P == 3 ? MT : 1][NT]) {
    constexpr int G = 2 * MT, PF = P == 3 ? 1 : MT >= 4 ? 3 : 2, TERMS = P == 3 ? 6 : 1;
    i16x8 fa[G][P], fb[2][NT][P];
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int q = 0; q < P; q++) fb[0][n][q] = b(n, 0, q);
#pragma unroll
    for (int g = 0; g < PF; g++)
#pragma unroll
        for (int q = 0; q < P; q++) fa[g][q] = a(g % MT, g / MT, q);
    request();
    static_for(std::make_integer_sequence<int, G>{}, [&](auto group) {
        constexpr int g = decltype(group)::value, b0 = g < MT ? g * NT / MT : NT, b1 = g < MT ? (g + 1) * NT / MT : NT;
        constexpr int reads = P * ((g + PF < G ? RA : 0) + (b1 - b0) * RB);
        if constexpr (g + PF < G) {
#pragma unroll
            for (int q = 0; q < P; q++) fa[g + PF][q] = a((g + PF) % MT, (g + PF) / MT, q);
        }
#pragma unroll
        for (int n = b0; n < b1; n++)
#pragma unroll
            for (int q = 0; q < P; q++) fb[1][n][q] = b(n, 1, q);
#pragma unroll
        for (int t = 0; t < TERMS; t++)
#pragma unroll
            for (int n = 0; n < NT; n++) {
                f32x4 &to = P == 3 && t + 1 < TERMS ? low[P == 3 ? g % MT : 0][n] : acc[g % MT][n];
                to = plane_product<T, P>(t, fb[g / MT][n], fa[g], to);
            }
        if constexpr (reads > 0) __builtin_amdgcn_sched_group_barrier(0x100, reads, 0);
        __builtin_amdgcn_sched_group_barrier(0x8, NT * TERMS, 0);
    });
}

// Zeroes a wave's products of the columns from `left` on (counted from its unit 0): the padding columns of H, gg and gu, in the last tile of a row.  Their operand's
// rows were read as zeros, but zero times an infinity of x or gy is NaN, which the product after the gate would carry into the row's every result.
template <int MT, int NT> __device__ __forceinline__ void zero_columns(f32x4 (&acc)[MT][NT], int n0, int units, int left, int lq) {
#pragma unroll
    for (int n = 0; n < NT; n++) {
        if (n < n0 || n >= n0 + units) continue;
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
            for (int r = 0; r < 4; r++) acc[m][n][r] = (n - n0) * 16 + lq * 4 + r < left ? acc[m][n][r] : 0.f;
    }
}

__device__ __forceinline__ float finite_part(float v) { return __builtin_isfinite(v) ? v : 0.f; }
template <int MT, int NT> __device__ __forceinline__ void finite_part(f32x4 (&acc)[MT][NT]) {
#pragma unroll
    for (int m = 0; m < MT; m++)
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int r = 0; r < 4; r++) acc[m][n][r] = finite_part(acc[m][n][r]);
}

// T: the matrix instruction's type; U: the user's type (float: T = bf16, planes); P: planes in LDS.
template <typename T, typename U, int P, int BUFS, int BM, int BN, int WI, int WJ, bool AKS, bool BKS, int EPI>
__global__ __launch_bounds__(64 * WI * WJ) void k_rows_gemm(const Args p) {
    constexpr int WAVES = WI * WJ, MT = BM / WI / 16, NT = BN / WJ / 16;
    constexpr bool DUAL = gate_forward(EPI);
    constexpr int TJ = DUAL ? BN / 2 : BN;                   // columns of C per tile
    using SA = Side<BM, AKS, WAVES, MT>;
    using SB = Side<BN, BKS, WAVES, NT>;
    extern __shared__ __attribute__((aligned(1024))) char lds[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), wi = wave / WJ, wj = wave % WJ;
    const TilePlace t = tile_place(p.tiles_i, p.tiles_j, p.problems, p.slices);
    const int64_t i0 = (int64_t)t.i * BM;
    const int j0 = t.j * TJ;
    const Seg *segs = p.seg[t.problem];

    SA sa;
    SB sb;
    sa.init(wave, lane, p.I - i0, p.lda, false);
    sb.init(wave, lane, (int64_t)p.J - j0, p.ldb, DUAL);
    sa.init_frags(lane, wi * MT);
    sb.init_frags(lane, DUAL ? wj * (NT / 2) : wj * NT);
    constexpr uint32_t kBuf = P * (SA::kBytes + SB::kBytes);
    const uint32_t lds0 = lds_addr(lds);
    const int steps_k = (p.K + BK - 1) / BK, steps = steps_k * p.n_seg;
    const int s_begin = (int)((int64_t)steps * t.slice / p.slices), s_end = (int)((int64_t)steps * (t.slice + 1) / p.slices);
    const int64_t a_step = AKS ? BK * p.lda * 2 : BK * 2, b_step = BKS ? BK * p.ldb * 2 : BK * 2;
    const int64_t a_tile = AKS ? i0 * 2 : i0 * p.lda * 2, b_tile = BKS ? (int64_t)j0 * 2 : (int64_t)j0 * p.ldb * 2;
    int sg = s_begin / (steps_k ? steps_k : 1), kk = s_begin - sg * steps_k;       // the next request's segment and step, and its operands' addresses
    const char *pa, *pb, *pb1;
    auto point = [&]() {
        pa = (const char *)segs[sg].a + a_tile + kk * a_step;
        pb = (const char *)segs[sg].b + b_tile + kk * b_step;
        pb1 = DUAL ? (const char *)segs[sg].b1 + b_tile + kk * b_step : pb;
    };
    auto request = [&](int buf) {
        const int64_t left = p.K - (int64_t)kk * BK;
        const uint32_t at = lds0 + (uint32_t)buf * kBuf;
#pragma unroll
        for (int q = 0; q < P; q++) {
            const char *a = pa + q * p.plane_a, *b = pb + q * p.plane_b, *b1 = DUAL ? pb1 + q * p.plane_b : b;
            sa.request(wave, a, a, left, at + q * SA::kBytes);
            sb.request(wave, b, b1, left, at + P * SA::kBytes + q * SB::kBytes);
        }
        pa += a_step;
        pb += b_step;
        if constexpr (DUAL) pb1 += b_step;
        if (++kk == steps_k) {
            kk = 0;
            if (++sg < p.n_seg) point();
        }
    };
    f32x4 acc[MT][NT], low[P == 3 ? MT : 1][NT];
#pragma unroll
    for (int m = 0; m < MT; m++)
#pragma unroll
        for (int n = 0; n < NT; n++) {
            acc[m][n] = f32x4{0.f, 0.f, 0.f, 0.f};
            if (P == 3) low[P == 3 ? m : 0][n] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
    // BUFS buffers: a step's requests are made BUFS - 1 steps ahead, into the buffer that the step before the current one has just left
    if (s_begin < s_end) point();
#pragma unroll
    for (int b = 0; b < BUFS - 1; b++)
        if (s_begin + b < s_end) request(b);
    constexpr int kAhead = (BUFS - 2) * P * (SA::kReq + SB::kReq);       // a wave's requests for the steps after this one
    static_assert(kAhead < 64, "the wait counts to 63");
    int buf = 0;
    auto step = [&](int s) {
        if (s + BUFS - 2 < s_end) wait_and_meet<kAhead>();
        else wait_and_meet<0>();
        const uint32_t at = lds0 + (uint32_t)buf * kBuf, at_b = at + P * SA::kBytes;
        multiply_step<T, MT, NT, P, AKS ? 2 : 1, BKS ? 2 : 1>(
            [&](int m, int ks, int q) { return sa.fragment(at + q * SA::kBytes, m, ks); },
            [&](int n, int ks, int q) {         // (EPI_GATE: the tile's upper half is the up projection's rows)
                return DUAL && n >= NT / 2 ? sb.fragment(at_b + q * SB::kBytes, n - NT / 2, ks, BN / 2) : sb.fragment(at_b + q * SB::kBytes, n, ks);
            },
            [&]() { if (s + BUFS - 1 < s_end) request(buf == 0 ? BUFS - 1 : buf - 1); }, acc, low);
        buf = buf + 1 == BUFS ? 0 : buf + 1;
    };
    if constexpr ((EPI == EPI_STORE || EPI == EPI_PARTIAL) && sizeof(U) == 2) {
        // lower planes first; an infinity among the other operand's elements makes any value of theirs, zero among them: what is not finite then is left to the
        // upper planes, whose product says what it is
        const int low_end = p.low_seg * steps_k < s_end ? p.low_seg * steps_k : s_end;
        int s = s_begin;
#pragma unroll 1
        for (int part = low_end > s_begin ? 0 : 1; part < 2; part++) {
            const int stop = part == 0 ? low_end : s_end;
            for (; s < stop; s++) step(s);
            if (part == 0) finite_part(acc);
        }
    } else {
        for (int s = s_begin; s < s_end; s++) step(s);
    }
    if constexpr (P == 3) {
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
            for (int n = 0; n < NT; n++) acc[m][n] += low[m][n];
    }

    // ---- epilogue: acc[m][n][r] is row i0 + 16 (wi MT + m) + (lane & 15), column 16 unit + 4 (lane >> 4) + r
    const int li = lane & 15, lq = lane >> 4;
    if constexpr (EPI == EPI_STORE || EPI == EPI_PARTIAL) {
#pragma unroll
        for (int m = 0; m < MT; m++) {
            const int64_t i = i0 + (wi * MT + m) * 16 + li;
            if (i >= p.I) continue;
            using O = typename std::conditional<EPI == EPI_PARTIAL, float, U>::type;
            O *row = (O *)p.out[t.problem] + (EPI == EPI_PARTIAL ? (int64_t)t.slice * p.slice_stride : 0) + i * p.ldo;
            const bool wide = p.ldo % 4 == 0 && (uintptr_t)p.out[t.problem] % (4 * sizeof(O)) == 0;
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
        }
    } else {
        // A lane has both projections (EPI_GATE) of the same elements, or fetches G and U of its own: the elementwise part is done where the products are, rounded,
        // and only its results pass through LDS, so that full lines of global memory are written.  Columns up to ldh are written, zeros behind J.
        // (EPI_GATE_FINE and its like, few results: written from where they are, in two planes.)
        constexpr int COLS = DUAL ? TJ : 2 * TJ, N = DUAL ? NT / 2 : NT;
        if (j0 + TJ > p.J) {        // (uniform)
            zero_columns(acc, 0, N, p.J - j0 - wj * N * 16, lq);
            if constexpr (DUAL) zero_columns(acc, N, N, p.J - j0 - wj * N * 16, lq);
        }
        using St = Staging<U, COLS, TJ, MT, WI, WAVES, DUAL ? MT : 1, BUFS * P * (BM + BN) * BK * 2>;
        f32x4 gq[N], uq[N];
        auto place = [&](int m, int n) {                    // (clamped: nothing branches between the requests)
            int64_t i = i0 + (wi * MT + m) * 16 + li, j = j0 + (wj * N + n) * 16 + lq * 4;
            i = i < p.I ? i : p.I - 1;
            j = j < p.ldh ? j : p.ldh - 4;
            return i * p.ldh + j;
        };
        auto fetch = [&](int m) {
#pragma unroll
            for (int n = 0; n < N; n++) {
                gq[n] = *reinterpret_cast<const f32x4 *>(p.g + place(m, n));
                uq[n] = *reinterpret_cast<const f32x4 *>(p.u + place(m, n));
            }
        };
        if constexpr (EPI == EPI_GATE_FINE || EPI == EPI_GATE_BWD_FINE) {
            with_activation(p.act, [&](auto act) {
                constexpr int ACT = decltype(act)::value;
#pragma unroll
                for (int m = 0; m < MT; m++) {
                    if constexpr (!DUAL) fetch(m);
#pragma unroll
                    for (int n = 0; n < N; n++) {
                        if (i0 + (wi * MT + m) * 16 + li >= p.I || j0 + (wj * N + n) * 16 + lq * 4 >= p.ldh) continue;
                        const int64_t at = place(m, n);
                        float o[4], o1[4], d;
                        if constexpr (DUAL) {
                            const f32x4 g = acc[m][n], u = acc[m][n + N];
#pragma unroll
                            for (int r = 0; r < 4; r++) o[r] = activation<ACT, false>(g[r], d) * u[r];
                            if (p.g) {
                                *reinterpret_cast<f32x4 *>(p.g + at) = g;
                                *reinterpret_cast<f32x4 *>(p.u + at) = u;
                            }
                            store_fine4<U>(p.h, p.plane, at, o);
                        } else {
#pragma unroll
                            for (int r = 0; r < 4; r++) {
                                o1[r] = acc[m][n][r] * activation<ACT, true>(gq[n][r], d);
                                o[r] = acc[m][n][r] * uq[n][r] * d;
                            }
                            store_fine4<U>(p.gg, p.plane, at, o);
                            store_fine4<U>(p.gu, p.plane, at, o1);
                        }
                    }
                }
            });
            return;
        }
        if constexpr (EPI == EPI_GATE_BWD) fetch(0);
        U *stage = reinterpret_cast<U *>(lds);
        with_activation(p.act, [&](auto act) {
            constexpr int ACT = decltype(act)::value;
#pragma unroll
            for (int pass = 0; pass < St::kPasses; pass++) {
                meet();
#pragma unroll
                for (int mp = 0; mp < St::MP; mp++) {
                    const int m = pass * St::MP + mp;
#pragma unroll
                    for (int n = 0; n < N; n++) {
                        U *at = stage + ((wi * St::MP + mp) * 16 + li) * St::kPitch + (wj * N + n) * 16 + lq * 4;
                        Pack<U, 4> o, o1;
                        float d;
                        if constexpr (EPI == EPI_GATE) {
                            const f32x4 g = acc[m][n], u = acc[m][n + N];
#pragma unroll
                            for (int r = 0; r < 4; r++) o.v[r] = from_f32<U>(activation<ACT, false>(g[r], d) * u[r]);
                            if (p.g && i0 + (wi * MT + m) * 16 + li < p.I && j0 + (wj * N + n) * 16 + lq * 4 < p.ldh) {
                                *reinterpret_cast<f32x4 *>(p.g + place(m, n)) = g;
                                *reinterpret_cast<f32x4 *>(p.u + place(m, n)) = u;
                            }
                        } else {
#pragma unroll
                            for (int r = 0; r < 4; r++) {
                                o1.v[r] = from_f32<U>(acc[m][n][r] * activation<ACT, true>(gq[n][r], d));
                                o.v[r] = from_f32<U>(acc[m][n][r] * uq[n][r] * d);
                            }
                            *reinterpret_cast<Pack<U, 4> *>(at + TJ) = o1;
                        }
                        *reinterpret_cast<Pack<U, 4> *>(at) = o;
                    }
                }
                if constexpr (EPI == EPI_GATE_BWD) {
                    if (pass + 1 < St::kPasses) fetch(pass + 1);
                }
                meet();
                St::copy_out(tid, [&](int row, int line, int col) {
                    const int64_t i = i0 + row + pass * St::MP * 16, at = i * p.ldh + j0 + col;
                    if (i >= p.I || j0 + col >= p.ldh) return;
                    const U *s = stage + line * St::kPitch + col;
                    store_staged(EPI == EPI_GATE ? p.h : p.gg, p.plane, at, s);
                    if constexpr (EPI == EPI_GATE_BWD) store_staged(p.gu, p.plane, at, s + TJ);
                });
            }
        });
    }
}

constexpr int kPlaneA[6] = {0, 1, 2, 0, 1, 0}, kPlaneB[6] = {2, 1, 0, 1, 0, 0};      // the six plane products, smallest first

// every pair of fp32 operands as six pairs of planes
inline void as_segments(Args &p) {
    for (int z = 0; z < 2; z++)
        for (int s = p.n_seg - 1; s >= 0; s--) {
            const Seg pair = p.seg[z][s];
            const int64_t a = z && p.plane_a2 ? p.plane_a2 : p.plane_a, b = z && p.plane_b2 ? p.plane_b2 : p.plane_b;        // (k_gate_bwd's second product)
            for (int t = 0; t < 6; t++)
                p.seg[z][6 * s + t] = Seg{(const char *)pair.a + kPlaneA[t] * a, (const char *)pair.b + kPlaneB[t] * b, (const char *)pair.b1 + kPlaneB[t] * b};
        }
    p.n_seg *= 6;
}

template <typename T, typename U, int P, int BUFS, int BM, int BN, int WI, int WJ, bool AKS, bool BKS, int EPI>
inline int launch_tile(Args p, int problems, hipStream_t s) {
    constexpr int TJ = gate_forward(EPI) ? BN / 2 : BN;
    // the gate epilogues also write the padding columns up to ldh (< J + 8)
    const int64_t cols = gate_forward(EPI) || gate_backward(EPI) ? p.ldh : p.J;
    const int64_t ti = (p.I + BM - 1) / BM, tj = (cols + TJ - 1) / TJ;
    if (ti * tj > kMaxGrid / (64 * WI * WJ) / problems / p.slices) return HS_ERR_ARG;
    p.problems = p.slices > 1 ? problems : 1;
    p.tiles_i = (int)ti;
    p.tiles_j = (int)tj;
    if constexpr (planes<U>() != P) as_segments(p);
    constexpr int kBuffer = P * (BM + BN) * BK * 2;
    // no more buffers than a workgroup has steps (the gate's epilogue wants them all): products of one step have several workgroups a CU
    // then (forward of 131 072 x 32 x 16 fp32 44.8 -> 40.2 us)
    const int64_t steps = ((int64_t)(p.K + BK - 1) / BK * p.n_seg + p.slices - 1) / p.slices;
    const int lds = kBuffer * (int)((EPI == EPI_STORE || EPI == EPI_PARTIAL) && steps < BUFS ? steps : BUFS);
    static hsLdsAttrOnce attr;
    const void *fn = (const void *)k_rows_gemm<T, U, P, BUFS, BM, BN, WI, WJ, AKS, BKS, EPI>;
    attr.set(fn, kBuffer * BUFS);
    k_rows_gemm<T, U, P, BUFS, BM, BN, WI, WJ, AKS, BKS, EPI><<<dim3((unsigned)(ti * tj * p.problems * p.slices), (unsigned)(problems / p.problems)), 64 * WI * WJ, lds, s>>>(p);
    return hipGetLastError() == hipSuccess ? HS_OK : HS_ERR_LAUNCH;
}

// ------------------------------------------------------------------------------------------------ gg and gu without G and U
// gH = gy Wd, G = x Wg^T, U = x Wu^T over the same K = D in one workgroup: 4 D operations an element of H more than reading G and U back, 16 bytes less written
// and read (fp32: 16-bit G and U would add two roundings to every gradient).  Tile 128 x 64 of each of the three, four waves, two workgroups a CU
// (fp32: plane products as segments).  131 072 x 256 x 1 024: 389 us (0.53 PFLOP/s, median; least 361; matrix cores 25 % of the cycles, vector units 43 %, LDS 24 %).
// As least times: 370, without the stores 321.  Larger tiles read less and were slower: with K this short half the time is the beginnings and the ends of tiles, and a second workgroup
// is what fills them (128 x 128 435, 256 x 64 435, 256 x 128 413, 64 x 64 423; eight waves 366, no gain for twice the LDS reads).
constexpr int kAgainM = 128, kAgainJ = 64;

template <typename T, typename U, bool FINE>
__global__ __launch_bounds__(256) void k_gate_bwd(const Args p) {
    constexpr int BM = kAgainM, TJ = kAgainJ, WAVES = 4, WI = 2, WJ = 2, MT = BM / WI / 16, N2 = TJ / WJ / 16, N1 = 2 * N2;
    using SA = Side<BM, false, WAVES, MT>;
    using S1 = Side<2 * TJ, false, WAVES, N1>;
    using S2 = Side<TJ, true, WAVES, N2>;
    constexpr uint32_t kBuf = SA::kBytes + S1::kBytes;
    extern __shared__ __attribute__((aligned(1024))) char lds[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), wi = wave / WJ, wj = wave % WJ;
    const TilePlace t = tile_place(p.tiles_i, p.tiles_j, 1, 1);
    const int64_t i0 = (int64_t)t.i * BM;
    const int j0 = t.j * TJ;
    SA sx, sg;
    S1 s1;
    S2 s2;
    sx.init(wave, lane, p.I - i0, p.lda, false);
    sg.init(wave, lane, p.I - i0, p.lda2, false);
    s1.init(wave, lane, (int64_t)p.J - j0, p.ldb, true);
    s2.init(wave, lane, (int64_t)p.J - j0, p.ldb2, false);
    sx.init_frags(lane, wi * MT);
    s1.init_frags(lane, wj * N2);
    s2.init_frags(lane, wj * N2);
    const uint32_t lds0 = lds_addr(lds);
    const int steps_k = (p.K + BK - 1) / BK, steps = steps_k * p.n_seg;
    int sgm = 0, kk = 0;
    auto advance = [&]() { if (++kk == steps_k) { kk = 0; sgm++; } };
    auto request1 = [&](int buf) {
        const Seg &sg_ = p.seg[0][sgm];
        const int64_t left = p.K - (int64_t)kk * BK, b = (int64_t)j0 * p.ldb * 2 + kk * (BK * 2);
        const char *a = (const char *)sg_.a + i0 * p.lda * 2 + kk * (BK * 2);
        sx.request(wave, a, a, left, lds0 + buf * kBuf);
        s1.request(wave, (const char *)sg_.b + b, (const char *)sg_.b1 + b, left, lds0 + buf * kBuf + SA::kBytes);
        advance();
    };
    auto request2 = [&](int buf) {
        const Seg &sg_ = p.seg[1][sgm];
        const int64_t left = p.K - (int64_t)kk * BK;
        const char *a = (const char *)sg_.a + i0 * p.lda2 * 2 + kk * (BK * 2), *b = (const char *)sg_.b + (int64_t)j0 * 2 + kk * (BK * p.ldb2 * 2);
        sg.request(wave, a, a, left, lds0 + buf * kBuf);
        s2.request(wave, b, b, left, lds0 + buf * kBuf + SA::kBytes);
        advance();
    };
    f32x4 acc[MT][N1], acc2[MT][N2], none1[1][N1], none2[1][N2];
#pragma unroll
    for (int m = 0; m < MT; m++) {
#pragma unroll
        for (int n = 0; n < N1; n++) acc[m][n] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int n = 0; n < N2; n++) acc2[m][n] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    request1(0);
    int buf = 0;
    for (int s = 0; s < steps; s++) {
        wait_and_meet<0>();
        const uint32_t at = lds0 + buf * kBuf;
        multiply_step<T, MT, N1, 1, 1, 1>([&](int m, int ks, int) { return sx.fragment(at, m, ks); },
                                       [&](int n, int ks, int) { return n < N2 ? s1.fragment(at + SA::kBytes, n, ks) : s1.fragment(at + SA::kBytes, n - N2, ks, TJ); },
                                       [&]() {
                                           if (s + 1 < steps) request1(buf ^ 1);
                                           else {
                                               sgm = kk = 0;
                                               request2(buf ^ 1);
                                           }
                                       },
                                       acc, none1);
        buf ^= 1;
    }
    for (int s = 0; s < steps; s++) {
        wait_and_meet<0>();
        const uint32_t at = lds0 + buf * kBuf;
        multiply_step<T, MT, N2, 1, 1, 2>([&](int m, int ks, int) { return sx.fragment(at, m, ks); }, [&](int n, int ks, int) { return s2.fragment(at + SA::kBytes, n, ks); },
                                       [&]() { if (s + 1 < steps) request2(buf ^ 1); }, acc2, none2);
        buf ^= 1;
    }
    // A lane has G, U and gH of the same elements: gg and gu are computed where they are, rounded, and only then pass through LDS, so that full lines of global
    // memory are written (131 072 x 256 x 1 024, least times: 369 us; G, U and gH in fp32 through LDS: 381)
    using St = Staging<U, 2 * TJ, TJ, MT, WI, WAVES, MT, 2 * (int)kBuf>;
    const int li = lane & 15, lq = lane >> 4;
    if (j0 + TJ > p.J) {        // (uniform)
        const int left = p.J - j0 - wj * N2 * 16;
        zero_columns(acc, 0, N2, left, lq);
        zero_columns(acc, N2, N2, left, lq);
        zero_columns(acc2, 0, N2, left, lq);
    }
    if constexpr (FINE) {
        with_activation(p.act, [&](auto act) {
#pragma unroll
            for (int m = 0; m < MT; m++)
#pragma unroll
                for (int n = 0; n < N2; n++) {
                    const int64_t i = i0 + (wi * MT + m) * 16 + li, j = j0 + (wj * N2 + n) * 16 + lq * 4;
                    if (i >= p.I || j >= p.ldh) continue;
                    float gg[4], gu[4], d;
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        gu[r] = acc2[m][n][r] * activation<decltype(act)::value, true>(acc[m][n][r], d);
                        gg[r] = acc2[m][n][r] * acc[m][n + N2][r] * d;
                    }
                    store_fine4<U>(p.gg, p.plane, i * p.ldh + j, gg);
                    store_fine4<U>(p.gu, p.plane, i * p.ldh + j, gu);
                }
        });
        return;
    }
    U *stage = reinterpret_cast<U *>(lds);
    with_activation(p.act, [&](auto act) {
        constexpr int ACT = decltype(act)::value;
#pragma unroll
        for (int pass = 0; pass < St::kPasses; pass++) {
            meet();
#pragma unroll
            for (int m = 0; m < St::MP; m++)
#pragma unroll
                for (int n = 0; n < N2; n++) {
                    Pack<U, 4> gg, gu;
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        const float gh = acc2[pass * St::MP + m][n][r];
                        float d;
                        gu.v[r] = from_f32<U>(gh * activation<ACT, true>(acc[pass * St::MP + m][n][r], d));
                        gg.v[r] = from_f32<U>(gh * acc[pass * St::MP + m][n + N2][r] * d);
                    }
                    U *at = stage + ((wi * St::MP + m) * 16 + li) * St::kPitch + (wj * N2 + n) * 16 + lq * 4;
                    *reinterpret_cast<Pack<U, 4> *>(at) = gg;
                    *reinterpret_cast<Pack<U, 4> *>(at + TJ) = gu;
                }
            meet();
            St::copy_out(tid, [&](int row, int line, int col) {
                const int64_t i = i0 + row + pass * St::MP * 16, at = i * p.ldh + j0 + col;
                if (i >= p.I || j0 + col >= p.ldh) return;
                const U *s = stage + line * St::kPitch + col;
                store_staged(p.gg, p.plane, at, s);
                store_staged(p.gu, p.plane, at, s + TJ);
            });
        }
    });
}

template <typename T, typename U, bool FINE> inline int launch_gate_bwd(Args p, hipStream_t s) {
    constexpr int BM = kAgainM;
    if constexpr (planes<U>() == 3) as_segments(p);
    const int64_t ti = (p.I + BM - 1) / BM, tj = (p.ldh + kAgainJ - 1) / kAgainJ;
    if (ti * tj > kMaxGrid / 256) return HS_ERR_ARG;
    p.tiles_i = (int)ti;
    p.tiles_j = (int)tj;
    constexpr int lds = 2 * (BM + 2 * kAgainJ) * BK * 2;
    static hsLdsAttrOnce attr;
    attr.set((const void *)k_gate_bwd<T, U, FINE>, lds);
    k_gate_bwd<T, U, FINE><<<dim3((unsigned)(ti * tj)), 256, lds, s>>>(p);
    return hipGetLastError() == hipSuccess ? HS_OK : HS_ERR_LAUNCH;
}

}  // namespace hs_gemm
