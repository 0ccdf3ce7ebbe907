// gated_mlp.h -- the gated feed-forward block on rows_gemm.h, one instantiation per user type (gated_mlp_{bf16,f16,f32}.hip):
//     G = x Wg^T, U = x Wu^T, H = act(G) U (one launch), y = H Wd^T;
//     gH = gy Wd, gg = gH U act'(G), gu = gH act(G) (one launch), gx = gg Wg + gu Wu, gWg = gg^T x, gWu = gu^T x (one launch), gWd = gy^T H.
// Roundings besides the results' own: H, gg and gu to the operand type, because the matrix cores multiply 16-bit operands (fp32: as three bf16 planes,
// 24 bits; few results: two planes, fine()).  G and U are never rounded: the forward keeps them in fp32 for the backward pass, or the backward pass computes them again (k_gate_bwd) where that
// moves fewer bytes than it costs products.
#pragma once
#include "rows_gemm.h"
#include "rows_small.h"

namespace hs_gemm {

// An operand as the products read it: 16-byte aligned rows whose contiguous extent is a multiple of 8 (zeros behind the matrix's own), at most 2^21 elements
// apart (offsets inside a tile have 32 bits).
struct Operand {
    const void *p;
    int64_t ld, plane;
};

// Hands out pieces of the caller's work space; without one it only counts.
struct Arena {
    char *base;
    int64_t at = 0;
    void *take(int64_t bytes) {
        const int64_t r = at;
        at += (bytes + 255) / 256 * 256;
        return base ? base + r : nullptr;
    }
};

inline int64_t up8(int64_t n) { return (n + 7) / 8 * 8; }

// Operands that are not in that form, copied into it: src [rows, cols] -> dst [planes][rows][8 chunks], zeros behind cols.  All of a pass in one launch (fp32
// has every operand in it; a launch each cost more than the copies).  Bound by memory and its launch: 1 021 x 1 000 x 2 730 f16 4.7 us, the fp32 operands of a pass of
// 4 096 x 256 x 683 6.0 and 7.0 us.
constexpr int kMaxPack = 6;
struct PackJob { const void *src; void *dst; int64_t ld, rows, cols, chunks, plane; unsigned first; };      // first: the job's first workgroup
struct PackJobs { PackJob j[kMaxPack]; int n; unsigned blocks; };

template <typename U>
__global__ __launch_bounds__(256) void k_rows_pack(const PackJobs jobs) {
    int k = 0;
    while (k + 1 < jobs.n && blockIdx.x >= jobs.j[k + 1].first) k++;
    const PackJob &job = jobs.j[k];
    const int64_t id = (int64_t)(blockIdx.x - job.first) * 256 + threadIdx.x;
    if (id >= job.rows * job.chunks) return;
    const int64_t r = id / job.chunks, c = (id - r * job.chunks) * 8;
    const U *s = (const U *)job.src + r * job.ld + c;
    Loose<U, 8> v;
    if (c + 8 <= job.cols) v = *reinterpret_cast<const Loose<U, 8> *>(s);
    else
#pragma unroll
        for (int e = 0; e < 8; e++) v.v[e] = c + e < job.cols ? s[e] : (U)0.f;
    if constexpr (sizeof(U) == 4) {
        Pack<bf16_t, 8> o[3];
#pragma unroll
        for (int e = 0; e < 8; e++) {
            bf16_t q[3];
            split3(v.v[e], q);
            o[0].v[e] = q[0]; o[1].v[e] = q[1]; o[2].v[e] = q[2];
        }
#pragma unroll
        for (int q = 0; q < 3; q++) *reinterpret_cast<Pack<bf16_t, 8> *>((bf16_t *)job.dst + q * job.plane + id * 8) = o[q];
    } else {
        Pack<U, 8> o;
#pragma unroll
        for (int e = 0; e < 8; e++) o.v[e] = v.v[e];
        *reinterpret_cast<Pack<U, 8> *>((U *)job.dst + id * 8) = o;
    }
}

// out = sum of the slices' partial results, in the order of the slices: all results of a pass that were cut into slices, in one launch at its end (a launch
// each behind its product: 1 021 x 1 000 x 2 730 step, host 15 us more).  Bound by memory: 21 us for 32 slices of 2 x 1 024 x 256 and 32 of 256 x 1 024.
constexpr int kMaxReduce = 4;
struct ReduceJob { const float *parts; void *out; int64_t n, stride; int slices; unsigned first; };
struct ReduceJobs { ReduceJob j[kMaxReduce]; int n; unsigned blocks; };

template <typename U>
__global__ __launch_bounds__(256) void k_rows_reduce(const ReduceJobs jobs) {
    int k = 0;
    while (k + 1 < jobs.n && blockIdx.x >= jobs.j[k + 1].first) k++;
    const ReduceJob &job = jobs.j[k];
    const int64_t i = ((int64_t)(blockIdx.x - job.first) * 256 + threadIdx.x) * 4;
    if (i >= job.n) return;
    const float *p = job.parts + i;
    U *o = (U *)job.out + i;
    float4 v = *reinterpret_cast<const float4 *>(p);
    for (int s = 1; s < job.slices; s++) {
        const float4 t = *reinterpret_cast<const float4 *>(p + s * job.stride);
        v.x += t.x; v.y += t.y; v.z += t.z; v.w += t.w;
    }
    const float r[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int e = 0; e < 4; e++)
        if (i + e < job.n) o[e] = from_f32<U>(r[e]);
}

// ------------------------------------------------------------------------------------------------ products
// Which tile, and into how many slices K is cut, by what a step of 64 of K costs (microseconds, measured at 8 192 x 4 096 x 12 288 and 1 021 x 1 000 x 2 730):
// a lone workgroup on a CU waits for its requests (`first`), every further one of the `fit` that LDS admits adds its own work (`more`).  The 256 x 256
// tile reads the least per product and has the highest rate (1.2 PFLOP/s against 0.93 and 0.6); with few tiles of the result the smaller ones, or
// slices whose fp32 partial results are added up by another launch, fill the device.  E.g. 1 021 x 1 000 over K = 5 460: 52 us in 64 x 64 tiles,
// 72 in 128 x 128, 29 in 128 x 128 and four slices, 21 with the requests three steps ahead (eight waves, four buffers, so one workgroup a CU: with
// many tiles two workgroups of two buffers are faster, 231 us against 337 for G and U of 131 072 x 256 x 1 024, and 256 x 256 tiles 217).  fp32 (six plane products): the large tile in
// six passes, 200 TFLOP/s; small tiles with the planes in LDS, one workgroup a CU.
struct Plan { int tile, slices; };
struct TileCost { int rows, cols, fit; float first, more; };
constexpr TileCost kTiles16[4] = {{256, 256, 1, 1.9f, 0.f}, {128, 128, 2, 0.8f, 0.38f}, {64, 64, 5, 0.5f, 0.15f}, {128, 128, 1, 0.66f, 0.f}};
constexpr TileCost kTiles32[3] = {{256, 256, 1, 11.4f, 0.f}, {128, 64, 1, 1.75f, 0.f}, {64, 64, 1, 1.f, 0.f}};
constexpr int kSlices[] = {1, 2, 3, 4, 5, 6, 7, 8, 10, 12, 14, 16, 20, 24, 28, 32, 40, 48, 56, 64};
template <typename U> Plan plan_product(int64_t I, int64_t cols, int64_t steps, int problems, bool sliceable) {
    const TileCost *kinds = sizeof(U) == 4 ? kTiles32 : kTiles16;
    Plan best = {0, 1};
    float least = 0.f;
    // (fp32, one step: the large tile takes six, one a plane product -- forward of 113 397 x 502 x 13 372 us, without it 358)
    for (int k = sizeof(U) == 4 && steps == 1 ? 1 : 0; k < (sizeof(U) == 4 ? 3 : 4); k++) {
        const TileCost &t = kinds[k];
        const int64_t whole = ((I + t.rows - 1) / t.rows) * ((cols + t.cols - 1) / t.cols) * problems;
        for (int slices : kSlices) {
            if (slices > 1 && (!sliceable || steps < 4 * slices || whole > 1024)) break;
            const int64_t each = (whole * slices + 255) / 256, together = each < t.fit ? each : t.fit, rounds = (each + together - 1) / together;
            float us = (float)rounds * ((float)((steps + slices - 1) / slices) * (t.first + t.more * (float)(together - 1)) + 3.f);
            if (slices > 1) us += 4.f + (float)(I * cols * problems) * (float)slices * 2e-6f;        // partial results written and read at 4 TB/s, one launch more
            if (least == 0.f || us < least) {
                least = us;
                best = Plan{k, slices};
            }
        }
    }
    return best;
}

template <typename T, typename U, bool AKS, bool BKS, int EPI> int launch_product(Args &p, int tile, int problems, hipStream_t s) {
    constexpr int P = planes<U>();
    if (tile == 0) return launch_tile<T, U, 1, 2, 256, 256, 2, 4, AKS, BKS, EPI>(p, problems, s);
    // fp32, one workgroup a CU: eight waves, so that a wave's LDS reads pass beside another's products (128 x 64: 37 -> 30 us for G and U of 4 096 x 256 x 683)
    if (tile == 1) return launch_tile<T, U, P, 2, 128, P == 3 ? 64 : 128, P == 3 ? 4 : 2, 2, AKS, BKS, EPI>(p, problems, s);
    if constexpr (P == 1) {
        if (tile == 3) return launch_tile<T, U, P, 4, 128, 128, 2, 4, AKS, BKS, EPI>(p, problems, s);
    }
    return launch_tile<T, U, P, P == 3 ? 3 : 2, 64, 64, P == 3 ? 4 : 2, 2, AKS, BKS, EPI>(p, problems, s);
}

// Up to this D the backward pass computes G and U again: 4 D operations an element (fp32: six times that) against 16 bytes.  (At D = 256: 131 072 x 1 024 in
// bf16, forward and this part of the backward 660 us against 780 with G and U kept; 4 096 x 683 in fp32 77 us against 66.)
template <typename U> constexpr int64_t again_dim() { return sizeof(U) == 4 ? 128 : 768; }

// Up to this many rows the forward products read the weights in place (rows_small.h).  4 096 x 12 288 bf16: 105 us at 33 rows, 145 at 64, where the tiles take
// 104 at 65.  fp32, whose tiles need copies in planes: 4 096 x 12 288 368 us at 33 rows and 417 at 64 against 545 in tiles, but 1 000 x 2 730 52 and 60 against
// 45, and 239 and 36 at 32 rows: to 64 rows for large weights, to 32 for the others.
template <typename U> int64_t small_rows(int64_t D, int64_t F) { return sizeof(U) == 4 && D * F >= (1 << 23) ? 64 : 32; }

template <typename T, typename U> struct Block {
    const hsGatedMlp &a;
    Arena ws;
    hipStream_t s;
    bool run;
    int rc = HS_OK;
    int64_t M, D, F, ldh;

    Block(const hsGatedMlp &args, bool run_, hipStream_t stream) : a(args), ws{run_ ? (char *)args.ws : nullptr}, s(stream), run(run_), M(args.rows), D(args.dim), F(args.hidden),
                                                                  ldh(up8(args.hidden)) {}

    void check(int r) { if (rc == HS_OK) rc = r; }

    // H, gg and gu of the 16-bit types in one plane or two.  Rounded once they bring as much error into every result as its own rounding, 1.41 times in all; in two
    // planes nothing that shows (distance from 64 bits over that of one rounding: 1.41 and 1.00 at 300 x 256 x 1 024 and 2 000 x 512 x 1 500).  The products that read
    // them double.  bf16, one plane and two, forward and step in us: 8 192 x 4 096 x 12 288 1 912 / 3 830 and 6 182 / 12 514, 131 072 x 256 x 1 024 297 / 554 and
    // 1 083 / 1 820, 1 021 x 1 000 x 2 730 44 / 59 and 133 / 185.  The caller chooses (HS_GATED_ONE_PLANE, HS_GATED_TWO_PLANES); without a choice it is two where a
    // result has so few elements that their error is no average (32 of 1 x 32 x 2 976: anything from 1.2 to 1.8), and most such blocks are bound by the
    // host: 2 x 1 024 x 2 816 10.9 / 11.8 and 82.8 / 84.1, 2 000 x 46 x 44 13.5 / 12.8 and 90.8 / 90.5; with weights to read 1 x 2 048 x 12 288 33.5 / 36.8 and
    // 150 / 180; many narrow rows pay the most, 131 072 x 8 x 250 50 / 91 and 181 / 362.
    static constexpr int64_t kFineResults = 2048;
    bool fine() const {
        if (sizeof(U) == 4 || (a.activation & HS_GATED_ONE_PLANE)) return false;
        return (a.activation & HS_GATED_TWO_PLANES) || (M < F ? M : F) * D <= kFineResults;
    }
    int inner_planes() const { return fine() ? 2 : planes<U>(); }
    template <typename O> static const void *plane1(const O &o) { return (const char *)o.p + o.plane * 2; }        // (of an operand in two planes of 16 bits)

    // The operand itself, or the copy of it that the next pack() makes.
    PackJobs jobs = {};
    Operand operand(const void *p, int64_t ld, int64_t rows, int64_t cols, bool force = false) {
        if (sizeof(U) == 2 && !force && (uintptr_t)p % 16 == 0 && ld % 8 == 0 && cols % 8 == 0 && ld <= (1 << 21)) return Operand{p, ld, 0};
        const int64_t ldp = up8(cols), n = rows * ldp, blocks = (n / 8 + 255) / 256;
        void *dst = ws.take(n * 2 * planes<U>());
        if (jobs.n == kMaxPack || jobs.blocks + blocks > kMaxGrid / 256) check(HS_ERR_ARG);
        else {
            jobs.j[jobs.n++] = PackJob{p, dst, ld, rows, cols, ldp / 8, n, jobs.blocks};
            jobs.blocks += (unsigned)blocks;
        }
        return Operand{dst, ldp, n};
    }
    void pack() {
        if (run && rc == HS_OK && jobs.n > 0) {
            k_rows_pack<U><<<jobs.blocks, 256, 0, s>>>(jobs);
            check(hipGetLastError() == hipSuccess ? HS_OK : HS_ERR_LAUNCH);
        }
        jobs = {};
    }

    // both projections' weights with one row distance
    void projections(Operand &wg, Operand &wu) {
        const bool differ = a.ld_gate != a.ld_up;
        wg = operand(a.w_gate, a.ld_gate, F, D, differ);
        wu = operand(a.w_up, a.ld_up, F, D, differ);
        if (wg.ld != wu.ld) {        // (one needed a copy: so does the other)
            if (wg.ld == a.ld_gate && wg.p == a.w_gate) wg = operand(a.w_gate, a.ld_gate, F, D, true);
            else wu = operand(a.w_up, a.ld_up, F, D, true);
        }
    }

    // whether the backward pass computes G and U again instead of reading them
    bool again() const { return D <= again_dim<U>(); }

    struct Saved { float *g, *u; Operand h; int64_t bytes; };
    Saved saved_in(char *base) const {
        Saved v = {};
        const int64_t n = M * ldh, gu = again() ? 0 : (n * 4 + 255) / 256 * 256;
        v.g = gu ? (float *)base : nullptr;
        v.u = gu ? (float *)(base + gu) : nullptr;
        v.h = Operand{base + 2 * gu, ldh, n};
        v.bytes = 2 * gu + n * 2 * inner_planes();
        return v;
    }

    void fwd_small() {
        Saved sv = saved_in((char *)a.saved);
        if (!a.saved) {
            sv.g = sv.u = nullptr;
            sv.h = Operand{ws.take(M * ldh * 2 * inner_planes()), ldh, M * ldh};
        }
        if (!run || rc != HS_OK) return;
        SmallArgs p = {};
        p.x = a.x; p.w = a.w_gate; p.w1 = a.w_up; p.ldx = a.ldx; p.ldw = a.ld_gate; p.ldw1 = a.ld_up; p.M = (int)M; p.N = (int)F; p.K = (int)D; p.act = a.activation & 0xff;
        p.g = sv.g; p.u = sv.u; p.h = (void *)sv.h.p; p.ldh = ldh; p.plane = sv.h.plane;
        if constexpr (sizeof(U) == 2) {
            if (fine()) check(launch_small<T, U, EPI_GATE, true>(p, s));
            else check(launch_small<T, U, EPI_GATE, false>(p, s));
        } else check(launch_small<T, U, EPI_GATE, false>(p, s));
        SmallArgs q = {};
        q.x = sv.h.p; q.w = q.w1 = a.w_down; q.ldx = ldh; q.ldw = q.ldw1 = a.ld_down; q.M = (int)M; q.N = (int)D; q.K = (int)F; q.plane = sv.h.plane;
        q.y = a.y; q.ldy = D;
        if (rc != HS_OK) return;
        if constexpr (sizeof(U) == 2) {
            if (fine()) return check(launch_small<T, U, EPI_STORE, true>(q, s));
        }
        check(launch_small<T, U, EPI_STORE, false>(q, s));
    }

    void fwd() {
        if (M <= small_rows<U>(D, F)) return fwd_small();
        const Operand x = operand(a.x, a.ldx, M, D);
        Operand wg, wu;
        projections(wg, wu);
        const Operand wd = operand(a.w_down, a.ld_down, D, F);
        Saved sv = saved_in((char *)a.saved);
        if (!a.saved) {
            sv.g = sv.u = nullptr;
            sv.h = Operand{ws.take(M * ldh * 2 * inner_planes()), ldh, M * ldh};
        }
        pack();
        Args p = product(x, wg, M, F, D);
        p.seg[0][0].b1 = wu.p;
        p.g = sv.g; p.u = sv.u; p.h = (void *)sv.h.p; p.ldh = ldh; p.plane = sv.h.plane; p.act = a.activation & 0xff;
        if (run && rc == HS_OK) {
            if (!fine()) check(launch_product<T, U, false, false, EPI_GATE>(p, plan_product<U>(M, 2 * ldh, steps(D), 1, false).tile, 1, s));
            else if constexpr (sizeof(U) == 2) check(launch_tile<T, U, 1, 2, 64, 64, 2, 2, false, false, EPI_GATE_FINE>(p, 1, s));
        }
        Args q = product(sv.h, wd, M, D, F);
        if (fine()) {
            q.seg[0][1] = q.seg[0][0];
            q.seg[0][0].a = plane1(sv.h);        // (the smaller plane's product first)
            q.n_seg = 2;
            q.low_seg = 1;
        }
        result<false, false>(q, &a.y, 1);
        reduce();
    }

    static int64_t steps(int64_t k) { return (k + BK - 1) / BK; }

    // C [I, J] = a b^T over K, everything but where it goes
    static Args product(const Operand &a, const Operand &b, int64_t I, int64_t J, int64_t K) {
        Args p = {};
        p.seg[0][0] = Seg{a.p, b.p, nullptr};
        p.n_seg = 1;
        p.lda = a.ld; p.ldb = b.ld; p.plane_a = a.plane * 2; p.plane_b = b.plane * 2;
        p.I = I; p.J = (int)J; p.K = (int)K; p.slices = 1;
        return p;
    }

    // The results of up to two products of one shape (p holds everything but the outputs): out[z] [I, J], contiguous.
    template <bool AKS, bool BKS> void result(Args &p, void *const *out, int problems) {
        const int64_t n = p.I * p.J, stride = (n + 3) / 4 * 4;
        const Plan plan = plan_product<U>(p.I, p.J, steps(p.K) * p.n_seg, problems, true);
        float *parts = plan.slices > 1 ? (float *)ws.take(stride * 4 * plan.slices * problems) : nullptr;
        if (!run || rc != HS_OK) return;
        p.ldo = p.J;
        p.slices = plan.slices;
        p.slice_stride = stride;
        for (int z = 0; z < problems; z++) p.out[z] = parts ? (void *)(parts + z * plan.slices * stride) : out[z];
        if (!parts) {
            check(launch_product<T, U, AKS, BKS, EPI_STORE>(p, plan.tile, problems, s));
            return;
        }
        check(launch_product<T, U, AKS, BKS, EPI_PARTIAL>(p, plan.tile, problems, s));
        const int64_t blocks = (n + 1023) / 1024;
        for (int z = 0; z < problems; z++) {
            if (sums.n == kMaxReduce || sums.blocks + blocks > kMaxGrid / 256) return check(HS_ERR_ARG);
            sums.j[sums.n++] = ReduceJob{parts + z * plan.slices * stride, out[z], n, stride, plan.slices, sums.blocks};
            sums.blocks += (unsigned)blocks;
        }
    }
    ReduceJobs sums = {};
    void reduce() {
        if (!run || rc != HS_OK || sums.n == 0) return;
        k_rows_reduce<U><<<sums.blocks, 256, 0, s>>>(sums);
        check(hipGetLastError() == hipSuccess ? HS_OK : HS_ERR_LAUNCH);
    }

    // C_z [I, J] = A_z^T B over the rows; in_a: the two planes of fine() are A's, not B's
    void weight_gradient(const Operand *av, const Operand &b, void *const *out, int problems, int64_t I, int64_t J, bool in_a) {
        Args p = product(av[0], b, I, J, M);
        if (problems == 2) p.seg[1][0] = Seg{av[1].p, b.p, nullptr};
        if (fine()) {
            for (int z = 0; z < problems; z++) {
                p.seg[z][1] = p.seg[z][0];
                if (in_a) p.seg[z][0].a = plane1(av[z]);
                else p.seg[z][0].b = plane1(b);
            }
            p.n_seg = 2;
            p.low_seg = 1;
        }
        result<true, true>(p, out, problems);
    }

    void bwd() {
        const Saved sv = saved_in((char *)a.saved);
        const bool inner = a.gx || a.gw_gate || a.gw_up, xw = a.gw_gate || a.gw_up;
        const Operand gy = operand(a.grad, a.ld_grad, M, D);
        Operand wd, wg, wu, x;
        if (inner) wd = operand(a.w_down, a.ld_down, D, F);
        if (inner && (again() || a.gx)) projections(wg, wu);
        if (inner && (again() || xw)) x = operand(a.x, a.ldx, M, D);
        pack();
        if (inner) {
            const int64_t n = M * ldh;
            const Operand gg{ws.take(n * 2 * inner_planes()), ldh, n}, gu{ws.take(n * 2 * inner_planes()), ldh, n};
            if (run && rc == HS_OK) {
                Args p = again() ? product(x, wg, M, F, D) : product(gy, wd, M, F, D);
                p.g = sv.g; p.u = sv.u; p.gg = (void *)gg.p; p.gu = (void *)gu.p; p.ldh = ldh; p.plane = n; p.act = a.activation & 0xff;
                if (again()) {
                    p.seg[0][0].b1 = wu.p;
                    p.seg[1][0] = Seg{gy.p, wd.p, nullptr};
                    p.lda2 = gy.ld; p.ldb2 = wd.ld; p.plane_a2 = gy.plane * 2; p.plane_b2 = wd.plane * 2;
                    if (!fine()) check(launch_gate_bwd<T, U, false>(p, s));
                    else if constexpr (sizeof(U) == 2) check(launch_gate_bwd<T, U, true>(p, s));
                } else if (!fine()) {
                    check(launch_product<T, U, false, true, EPI_GATE_BWD>(p, plan_product<U>(M, ldh, steps(D), 1, false).tile, 1, s));
                } else if constexpr (sizeof(U) == 2) {
                    check(launch_tile<T, U, 1, 2, 64, 64, 2, 2, false, true, EPI_GATE_BWD_FINE>(p, 1, s));
                }
            }
            if (a.gx) {
                Args p = product(gg, wg, M, D, F);
                p.seg[0][1] = Seg{gu.p, wu.p, nullptr};
                p.n_seg = 2;
                if (fine()) {
                    for (int k = 0; k < 2; k++) p.seg[0][2 + k] = p.seg[0][k];
                    p.seg[0][0].a = plane1(gg);
                    p.seg[0][1].a = plane1(gu);
                    p.n_seg = 4;
                    p.low_seg = 2;
                }
                result<false, true>(p, &a.gx, 1);
            }
            if (xw) {
                const Operand av[2] = {a.gw_gate ? gg : gu, gu};
                void *const out[2] = {a.gw_gate ? a.gw_gate : a.gw_up, a.gw_up};
                weight_gradient(av, x, out, a.gw_gate && a.gw_up ? 2 : 1, F, D, true);
            }
        }
        if (a.gw_down) weight_gradient(&gy, sv.h, &a.gw_down, 1, D, F, false);
        reduce();
    }
};

template <typename T, typename U> int64_t block_call(const hsGatedMlp &a, int what, hipStream_t s) {
    if (what == 4) return Block<T, U>(a, false, s).saved_in(nullptr).bytes;
    Block<T, U> b(a, what < 2, s);
    if (what % 2 == 0) b.fwd(); else b.bwd();
    if (what >= 2) return b.ws.at;
    return b.rc;
}

// what: 0 forward, 1 backward, 2 / 3 their work spaces' bytes, 4 the saved buffer's bytes
int64_t gated_mlp_bf16(const hsGatedMlp &a, int what, hipStream_t s);
int64_t gated_mlp_f16(const hsGatedMlp &a, int what, hipStream_t s);
int64_t gated_mlp_f32(const hsGatedMlp &a, int what, hipStream_t s);

}  // namespace hs_gemm
