// holoscene_amd/csrc/embed_rows.hip -- learned codes looked up by index (gfx950):
//     out_i = scale * table[idx_i],          d table_v = scale * sum over {i : idx_i = v} of g_i.
// An index outside [0, V) reads a row of zeros and takes no gradient (as a point outside the hash grid's cube does), so no launch reads or writes
// outside the table whatever the indices hold; `padding` (or -1) is looked up like any other row and takes no gradient.
//
// The gradient sums each row's run in the order of the positions, so it is the same from run to run: (index, position) pairs are sorted by
// index with a stable counting sort, and the table's gradient is then written row by row, once, zeros included -- no fill, no atomics on it.
//   sort    N <= 4 096: one workgroup, the pairs in registers, one pass per <= 8 bits of the index through LDS (one launch);
//           longer: passes of <= 9 bits, two launches each (block histograms; ranks, every workgroup adding up the histograms itself).
//   chunks  sorted positions in chunks of 32: a chunk that lies inside one run is summed to fp32 partials (a run of one index may be the whole batch).
//   runs    the run of every row, by bisection in the sorted indices, in the same launch: lists of the long and of the short ones, a flag for the others.
//   rows    first the long runs (> 8 entries; a workgroup per run and block of columns: its head and tail from g and its whole chunks from the partials, joined
//           through LDS in a fixed order), then the short ones (a wave each), then the zeros of the rows without one: the reads are over before the stores
//           of the zeros, most of the bytes, fill the memory's queues.
// fp32 sums: 32 terms per chunk, then the partials; the last operation rounds to the table's type.
//
// Measured: 16 384 zipf-distributed rows of 2 048 bf16, table of 50 021: lookup 22.6 us (134 MB, 5.9 TB/s); gradient: sort 2 x (2.9 + 7.8), chunks and runs 13.6,
// rows 59 (205 MB of table written, 67 MB of gradient read: 54 us at the rate of a large copy).  131 072 rows of 32 fp32, 8 indices among 1 024: lookup 7.2, sort
// 4.8 + 18.7 (one pass), chunks 9.8, rows 4.8.  The lookup and the rows are bound by memory, the sort by its chains of dependent LDS operations and launches.
#include "holoscene_hip.h"
#include "launch_util.h"
#include "row_types.h"

namespace {

using namespace hs_row;

// ------------------------------------------------------------------------------------------------ lookup
// one thread per VEC elements of the output; `per_row` = D / VEC
template <typename T, typename O, typename I, int VEC>
__global__ __launch_bounds__(256) void k_embed_fwd(const I *__restrict__ idx, const T *__restrict__ table, int64_t ld, O *__restrict__ out, int64_t total,
                                                   uint32_t per_row, int64_t V, float scale) {
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (id >= total) return;
    int64_t row;
    uint32_t c;
    if (total <= 0xffffffffll) {        // (uniform: a 32-bit division is a tenth of the 64-bit one)
        row = (uint32_t)id / per_row;
        c = (uint32_t)id - (uint32_t)row * per_row;
    } else {
        row = id / per_row;
        c = (uint32_t)(id - row * per_row);
    }
    const int64_t v = (int64_t)idx[row];
    Pack<O, VEC> o;
    if (v >= 0 && v < V) {
        const Pack<T, VEC> t = *reinterpret_cast<const Pack<T, VEC> *>(table + v * ld + (int64_t)c * VEC);
#pragma unroll
        for (int e = 0; e < VEC; e++) o.v[e] = from_f32<O>(to_f32(t.v[e]) * scale);
    } else {
#pragma unroll
        for (int e = 0; e < VEC; e++) o.v[e] = from_f32<O>(0.f);
    }
    *reinterpret_cast<Pack<O, VEC> *>(out + id * VEC) = o;
}

// ------------------------------------------------------------------------------------------------ sort
// Keys: the index where it takes a gradient, V otherwise (sorted behind every row).
template <typename I> __device__ __forceinline__ uint32_t sort_key(const I *__restrict__ idx, int64_t i, int64_t V, int64_t padding) {
    const int64_t v = (int64_t)idx[i];
    return v >= 0 && v < V && v != padding ? (uint32_t)v : (uint32_t)V;
}

constexpr int kSortThreads = 1024, kSortWaves = kSortThreads / 64;
constexpr int kOneMax = 4096, kOneDigit = 8;        // the one-workgroup sort (16 384 pairs in it: 37 us, bound by one CU's vector instructions; over 16 CUs 24)
constexpr int kMultiDigit = 9, kOnlyDigit = 11;    // the multi-block sort: tiles of 1, 2 or 4 pairs per thread; up to 11 bits in a single pass (131 072 pairs: 23.8 us, in two of 9 bits 24.4 and two launches more)
constexpr int kMaxBlocks = 64;                      // workgroups of the multi-block sort (each adds up all their histograms)

// Lanes of this wave whose digit equals mine, among those with `on`.  (Per bit: a mask of the bit, a ballot, and the lanes that agree with it.)
__device__ __forceinline__ uint64_t same_digit(uint32_t digit, int bits, bool on) {
    const uint64_t all = __ballot(on);
    uint32_t lo = (uint32_t)all, hi = (uint32_t)(all >> 32);
#pragma unroll
    for (int b = 0; b < kOnlyDigit; b++) {
        if (b < bits) {         // (uniform)
            const uint32_t mine = (uint32_t)((int32_t)(digit << (31 - b)) >> 31);
            const uint64_t set = __ballot(mine != 0u);
            lo &= ~((uint32_t)set ^ mine);
            hi &= ~((uint32_t)(set >> 32) ^ mine);
        }
    }
    return ((uint64_t)hi << 32) | lo;
}

// Ranks of a tile's pairs among those of equal digit in front of them.  Wave w holds pairs [w * 64 * R, (w + 1) * 64 * R) of the tile, round r lane l
// the pair 64 r + l of them.  cnt [waves][bins] must be zero; afterwards it holds, per wave and digit, the pairs of that digit in earlier waves
// of the tile, and tile_total[digit] (may alias nothing) the tile's count.
template <int R> __device__ __forceinline__ void tile_ranks(const uint32_t (&digit)[R], const bool (&on)[R], uint32_t (&rank)[R], int bits, int bins, uint16_t *cnt,
                                                            uint32_t *tile_total) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    uint16_t *mine = cnt + wave * bins;
    const uint64_t below = (1ull << lane) - 1;
#pragma unroll
    for (int r = 0; r < R; r++) {
        const uint64_t peers = same_digit(digit[r], bits, on[r]);
        uint32_t base = 0;
        if (on[r]) {
            base = mine[digit[r]];
            rank[r] = base + __popcll(peers & below);
        }
        __builtin_amdgcn_wave_barrier();            // (a wave's LDS operations complete in order: every read above precedes the write below)
        if (on[r] && (peers & below) == 0) mine[digit[r]] = (uint16_t)(base + __popcll(peers));
        __builtin_amdgcn_wave_barrier();
    }
    __syncthreads();
    for (int d = tid; d < bins; d += kSortThreads) {
        uint32_t sum = 0;
#pragma unroll
        for (int w = 0; w < kSortWaves; w++) {
            const uint32_t c = cnt[w * bins + d];
            cnt[w * bins + d] = (uint16_t)sum;
            sum += c;
        }
        tile_total[d] = sum;
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < R; r++)
        if (on[r]) rank[r] += mine[digit[r]];
}

// exclusive scan of v[0, n) in place by the whole workgroup; n <= 2 * kSortThreads
__device__ __forceinline__ void scan_exclusive(uint32_t *v, int n, uint32_t *wave_sums) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const uint32_t a = 2 * tid < n ? v[2 * tid] : 0, b = 2 * tid + 1 < n ? v[2 * tid + 1] : 0;
    uint32_t s = a + b;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const uint32_t t = __shfl_up(s, off);
        if (lane >= off) s += t;
    }
    if (lane == 63) wave_sums[wave] = s;
    __syncthreads();
    uint32_t before = 0;
    for (int w = 0; w < wave; w++) before += wave_sums[w];
    const uint32_t ex = before + s - (a + b);
    if (2 * tid < n) v[2 * tid] = ex;
    if (2 * tid + 1 < n) v[2 * tid + 1] = ex + a;
    __syncthreads();
}

// All of it in one workgroup: R = pairs per thread (N <= 1024 R), `passes` passes of <= 8 bits, the pairs through LDS between passes.
template <typename I, int R>
__global__ __launch_bounds__(kSortThreads) void k_sort_one(const I *__restrict__ idx, int n, int64_t V, int64_t padding, int bits, int passes, uint32_t *__restrict__ keys,
                                                           uint32_t *__restrict__ pos, uint32_t *__restrict__ list_n) {
    extern __shared__ __attribute__((aligned(16))) uint32_t lds[];
    uint32_t *total = lds, *wave_sums = lds + 256;
    uint16_t *cnt = reinterpret_cast<uint16_t *>(lds + 256 + kSortWaves);
    uint32_t *lk = lds + 256 + kSortWaves + kSortWaves * 256 / 2, *lp = lk + 1024 * R;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    if (tid < 2) list_n[tid] = 0;              // (the next launch appends)
    uint32_t key[R], at[R], digit[R], rank[R];
    bool on[R];
#pragma unroll
    for (int r = 0; r < R; r++) {
        const int i = (wave * R + r) * 64 + lane;
        on[r] = i < n;
        key[r] = on[r] ? sort_key(idx, i, V, padding) : 0;
        at[r] = (uint32_t)i;
    }
    int shift = 0;
    for (int p = 0; p < passes; p++) {
        const int nb = (bits - shift + passes - p - 1) / (passes - p), bins = 1 << nb;
        for (int i = tid; i < kSortWaves * bins / 2; i += kSortThreads) reinterpret_cast<uint32_t *>(cnt)[i] = 0;
        __syncthreads();
#pragma unroll
        for (int r = 0; r < R; r++) digit[r] = (key[r] >> shift) & (uint32_t)(bins - 1);
        tile_ranks<R>(digit, on, rank, nb, bins, cnt, total);
        __syncthreads();
        scan_exclusive(total, bins, wave_sums);
#pragma unroll
        for (int r = 0; r < R; r++) {
            if (!on[r]) continue;
            const uint32_t to = total[digit[r]] + rank[r];
            lk[to] = key[r];
            lp[to] = at[r];
        }
        __syncthreads();
        if (p + 1 < passes) {
#pragma unroll
            for (int r = 0; r < R; r++) {
                const int i = (wave * R + r) * 64 + lane;
                if (on[r]) { key[r] = lk[i]; at[r] = lp[i]; }
            }
        } else {
            for (int i = tid; i < n; i += kSortThreads) {       // (from LDS: written where the ranks point, every store instruction would touch 64 lines)
                keys[i] = lk[i];
                pos[i] = lp[i];
            }
        }
        shift += nb;
    }
}

// Multi-block, first launch of a pass: hist[block][digit] over the block's `per` pairs.  keys_in == NULL: the first pass, from the indices.
template <typename I>
__global__ __launch_bounds__(kSortThreads) void k_sort_hist(const I *__restrict__ idx, const uint32_t *__restrict__ keys_in, int64_t n, int64_t per, int64_t V, int64_t padding,
                                                            int shift, int nb, uint32_t *__restrict__ hist, uint32_t *__restrict__ list_n) {
    __shared__ uint32_t h[1 << kOnlyDigit];
    const int tid = threadIdx.x, bins = 1 << nb;
    if (tid < 2 && blockIdx.x == 0) list_n[tid] = 0;
    for (int d = tid; d < bins; d += kSortThreads) h[d] = 0;
    __syncthreads();
    const int64_t begin = blockIdx.x * per, end = begin + per < n ? begin + per : n;
    for (int64_t i = begin + tid; i < end; i += kSortThreads) {
        const uint32_t k = keys_in ? keys_in[i] : sort_key(idx, i, V, padding);
        atomicAdd(&h[(k >> shift) & (uint32_t)(bins - 1)], 1u);        // (counts only: their order does not matter)
    }
    __syncthreads();
    for (int d = tid; d < bins; d += kSortThreads) hist[(size_t)blockIdx.x * bins + d] = h[d];
}

// second launch: ranks.  A workgroup's first place for a digit = all pairs of smaller digits + the pairs of this digit in earlier workgroups.
template <typename I, int R>
__global__ __launch_bounds__(kSortThreads) void k_sort_scatter(const I *__restrict__ idx, const uint32_t *__restrict__ keys_in, const uint32_t *__restrict__ pos_in, int64_t n,
                                                               int64_t per, int64_t V, int64_t padding, int shift, int nb, const uint32_t *__restrict__ hist,
                                                               uint32_t *__restrict__ keys, uint32_t *__restrict__ pos) {
    constexpr int kTile = R * kSortThreads;
    extern __shared__ __attribute__((aligned(16))) uint32_t lds[];
    const int bins = 1 << nb, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    uint32_t *place = lds, *tile_total = lds + bins, *tile_first = lds + 2 * bins, *wave_sums = lds + 3 * bins, *lk = wave_sums + kSortWaves, *lp = lk + kTile;
    uint16_t *cnt = reinterpret_cast<uint16_t *>(lp + kTile);
    // all pairs of a digit, and those in earlier workgroups: 2048 / bins threads a pair of digits, each a share of the workgroups' histograms
    uint32_t *before = tile_first;
    for (int d = tid; d < bins; d += kSortThreads) place[d] = before[d] = 0;
    __syncthreads();
    {
        const int half = bins / 2, d = tid % half, share = kSortThreads / half;
        uint2 all = make_uint2(0, 0), mine = all;
#pragma unroll 8
        for (int b = tid / half; b < (int)gridDim.x; b += share) {
            const uint2 c = reinterpret_cast<const uint2 *>(hist + (size_t)b * bins)[d];
            const bool earlier = b < (int)blockIdx.x;
            all.x += c.x;
            all.y += c.y;
            mine.x += earlier ? c.x : 0u;
            mine.y += earlier ? c.y : 0u;
        }
        if (tid / half < (int)gridDim.x) {
            atomicAdd(&place[2 * d], all.x);            // (counts in LDS: their order does not matter)
            atomicAdd(&place[2 * d + 1], all.y);
            atomicAdd(&before[2 * d], mine.x);
            atomicAdd(&before[2 * d + 1], mine.y);
        }
    }
    __syncthreads();
    scan_exclusive(place, bins, wave_sums);
    for (int d = tid; d < bins; d += kSortThreads) place[d] += before[d];
    __syncthreads();
    const int64_t begin = blockIdx.x * per, end = begin + per < n ? begin + per : n;
    for (int64_t t0 = begin; t0 < end; t0 += kTile) {
        for (int i = tid; i < kSortWaves * bins / 2; i += kSortThreads) reinterpret_cast<uint32_t *>(cnt)[i] = 0;
        uint32_t key[R], at[R], digit[R], rank[R];
        bool on[R];
#pragma unroll
        for (int r = 0; r < R; r++) {
            const int64_t i = t0 + (wave * R + r) * 64 + lane;
            on[r] = i < end;
            key[r] = on[r] ? (keys_in ? keys_in[i] : sort_key(idx, i, V, padding)) : 0;
            at[r] = on[r] && pos_in ? pos_in[i] : (uint32_t)i;
            digit[r] = (key[r] >> shift) & (uint32_t)(bins - 1);
        }
        __syncthreads();
        tile_ranks<R>(digit, on, rank, nb, bins, cnt, tile_total);
        // the tile in its own order through LDS, then out: neighbours go to neighbouring places
        for (int d = tid; d < bins; d += kSortThreads) tile_first[d] = tile_total[d];
        __syncthreads();
        scan_exclusive(tile_first, bins, wave_sums);
#pragma unroll
        for (int r = 0; r < R; r++) {
            if (!on[r]) continue;
            const uint32_t to = tile_first[digit[r]] + rank[r];
            lk[to] = key[r];
            lp[to] = at[r];
        }
        __syncthreads();
        const int in_tile = end - t0 < kTile ? (int)(end - t0) : kTile;
        for (int i = tid; i < in_tile; i += kSortThreads) {
            const uint32_t k = lk[i], d = (k >> shift) & (uint32_t)(bins - 1), to = place[d] + (uint32_t)i - tile_first[d];
            keys[to] = k;
            pos[to] = lp[i];
        }
        __syncthreads();
        for (int d = tid; d < bins; d += kSortThreads) place[d] += tile_total[d];
        __syncthreads();
    }
}

// ------------------------------------------------------------------------------------------------ sums
constexpr int kChunk = 32;
constexpr int kShort = 8, kWide = 2;        // runs up to kShort entries are summed by one group of lanes, kWide * VEC columns a lane at a time
constexpr int64_t kMaxGrid = 0xffffff;     // workgroups of 256 a launch takes: a grid has less than 2^32 threads
constexpr int kLongGroups = 256, kShortGroups = 8192;            // workgroups (per block of columns; in all) that share the long and the short runs

struct Run { uint32_t row, first, end, pos; };              // pos: of its first entry, a load less in front of the gradient
struct RunLists { Run *of_long, *of_short; uint32_t *n; uint8_t *used; };        // n: their lengths; used [V]: whether the row has a run

// acc += the entries first, first + step, .. < end, in that order.  row(j): where entry j's element `col` lies.  BATCH entries are requested together, the missing
// ones of the last batch at the first entry's address and not added (a branch between the requests would wait for each of them).
template <int BATCH, typename T, int VEC, typename R>
__device__ __forceinline__ void add_entries(int64_t first, int64_t end, int step, int cols, R row, float (&acc)[VEC]) {
    if (cols >= VEC) {
        for (int64_t j = first; j < end; j += BATCH * step) {
            Loose<T, VEC> t[BATCH];
#pragma unroll
            for (int b = 0; b < BATCH; b++) t[b] = *reinterpret_cast<const Loose<T, VEC> *>(row(j + b * step < end ? j + b * step : first));
#pragma unroll
            for (int b = 0; b < BATCH; b++)
#pragma unroll
                for (int e = 0; e < VEC; e++) acc[e] += j + b * step < end ? to_f32(t[b].v[e]) : 0.f;
        }
    } else {                    // a row's last columns
        for (int64_t j = first; j < end; j += step)
#pragma unroll
            for (int e = 0; e < VEC; e++)
                if (e < cols) acc[e] += to_f32(row(j)[e]);
    }
}

// First place in keys[0, n) that is >= v, by eights: seven loads that do not depend on each other a step, so the chain has a third of a bisection's loads.
__device__ __forceinline__ int64_t lower_bound(const uint32_t *__restrict__ keys, int64_t n, uint32_t v) {
    int64_t lo = 0, len = n;                    // the answer lies in [lo, lo + len]
    while (len > 0) {
        const int64_t step = len >= 8 ? len / 8 : 1;
        int smaller = 0;
#pragma unroll
        for (int j = 1; j < 8; j++) {
            const int64_t at = j * step <= len ? lo + j * step - 1 : lo + len - 1;
            smaller += keys[at] < v && j * step <= len;
        }
        lo += smaller * step;
        len = smaller == 7 ? len - 7 * step : step - 1;
    }
    return lo;
}

// Column layout of the two kernels below: a group of `lanes` (a power of two <= 64) covers lanes * VEC columns at a time; the 256 / lanes groups of a
// workgroup are slots that take entries (short runs: rows) in turn.  k_embed_chunks: blockIdx.y is the column block.

// Two jobs that only need the sorted pairs, in one launch: the first bound_blocks workgroups find the first entry of every row's run (a thread per row and a
// chain of ~log2 n dependent loads: as part of the rows' kernel it was most of its time), the others sum the chunks that lie inside one run.
template <typename T, int VEC>
__global__ __launch_bounds__(256) void k_embed_chunks(const uint32_t *__restrict__ keys, const uint32_t *__restrict__ pos, const T *__restrict__ grad, int64_t ldg,
                                                      int64_t n, uint32_t V, int D, int lanes, float *__restrict__ partial, RunLists lists, unsigned bound_blocks) {
    __shared__ float join[256 * VEC];
    const int tid = threadIdx.x;
    if (blockIdx.x < bound_blocks) {
        if (blockIdx.y != 0) return;
        __shared__ uint32_t first_of[257], part[2][4], base[2];        // one bound more than rows: the end of the last row's run
        const int lane = tid & 63, wave = tid >> 6;
        const int64_t v0 = (int64_t)blockIdx.x * 256, v = v0 + tid;
        for (int i = tid; i < 257; i += 256) first_of[i] = v0 + i <= V ? (uint32_t)lower_bound(keys, n, (uint32_t)(v0 + i)) : 0;
        __syncthreads();
        const uint32_t first = first_of[tid], end = v < V ? first_of[tid + 1] : first, len = end - first;
        const bool is_long = len > (uint32_t)kShort, is_short = len > 0 && !is_long;
        const uint64_t longs = __ballot(is_long), shorts = __ballot(is_short), below = (1ull << lane) - 1;
        if (lane == 0) {
            part[0][wave] = __popcll(longs);
            part[1][wave] = __popcll(shorts);
        }
        __syncthreads();
        if (tid < 2) base[tid] = atomicAdd(&lists.n[tid], part[tid][0] + part[tid][1] + part[tid][2] + part[tid][3]);        // (any order: each run is a sum of its own)
        __syncthreads();
        if (v < V) lists.used[v] = len > 0;
        if (len > 0) {
            uint32_t at = base[is_short] + __popcll((is_short ? shorts : longs) & below);
            for (int w = 0; w < wave; w++) at += part[is_short][w];
            (is_short ? lists.of_short : lists.of_long)[at] = Run{(uint32_t)v, first, end, pos[first]};
        }
        return;
    }
    const int64_t c = blockIdx.x - bound_blocks, c0 = c * kChunk;
    const uint32_t first = keys[c0];
    if (first == V || first != keys[c0 + kChunk - 1]) return;        // (uniform in the workgroup)
    const int col = ((int)blockIdx.y * lanes + (tid & (lanes - 1))) * VEC, slot = tid / lanes, slots = 256 / lanes;
    float acc[VEC];
#pragma unroll
    for (int e = 0; e < VEC; e++) acc[e] = 0.f;
    if (col < D) add_entries<8, T, VEC>(c0 + slot, c0 + kChunk, slots, D - col, [&](int64_t j) { return grad + (int64_t)pos[j] * ldg + col; }, acc);
#pragma unroll
    for (int e = 0; e < VEC; e++) join[e * 256 + tid] = acc[e];
    __syncthreads();
    if (slot != 0 || col >= D) return;
    for (int s = 1; s < slots; s++)
#pragma unroll
        for (int e = 0; e < VEC; e++) acc[e] += join[e * 256 + s * lanes + tid];
    float *out = partial + c * D + col;
#pragma unroll
    for (int e = 0; e < VEC; e++)
        if (col + e < D) out[e] = acc[e];
}

// The first long_groups * col_blocks workgroups: long runs; the next short_groups: short ones, a slot each; the others: a slot per row of the table, zeros where
// it has no run.
template <typename T, typename O, int VEC>
__global__ __launch_bounds__(256) void k_embed_rows(const RunLists lists, const uint32_t *__restrict__ pos, const T *__restrict__ grad, int64_t ldg, int64_t V, int D, int lanes,
                                                    const float *__restrict__ partial, float scale, O *__restrict__ gtable, unsigned long_groups, unsigned col_blocks,
                                                    unsigned short_groups) {
    __shared__ float join[256 * VEC];
    const int tid = threadIdx.x, lane = tid & (lanes - 1), slot = tid / lanes, slots = 256 / lanes;
    auto write = [&](int64_t row, int col, const float *acc) {
        O *out = gtable + row * D + col;
        Loose<O, VEC> o;
#pragma unroll
        for (int e = 0; e < VEC; e++) o.v[e] = from_f32<O>(acc[e] * scale);
        if (col + VEC <= D) *reinterpret_cast<Loose<O, VEC> *>(out) = o;
        else
#pragma unroll
            for (int e = 0; e < VEC; e++)
                if (col + e < D) out[e] = o.v[e];
    };
    if (blockIdx.x < long_groups * col_blocks) {
        const uint32_t n_long = lists.n[0];
        const int col = ((int)(blockIdx.x / long_groups) * lanes + lane) * VEC;
        for (uint32_t i = blockIdx.x % long_groups; i < n_long; i += long_groups) {
            const Run run = lists.of_long[i];
            const int64_t rs = run.first, re = run.end;
            const int64_t c_first = (rs + kChunk - 1) / kChunk, c_last = re / kChunk;      // whole chunks [c_first, c_last)
            const int64_t head = c_first < c_last ? c_first * kChunk : re, tail = c_first < c_last ? c_last * kChunk : re, skip = tail - head;
            float acc[VEC];
#pragma unroll
            for (int e = 0; e < VEC; e++) acc[e] = 0.f;
            if (col < D) {
                // head and tail as one sequence, then the chunks
                add_entries<4, T, VEC>(rs + slot, re - skip, slots, D - col, [&](int64_t j) { return grad + (int64_t)pos[j < head ? j : j + skip] * ldg + col; }, acc);
                add_entries<4, float, VEC>(c_first + slot, c_last, slots, D - col, [&](int64_t c) { return partial + c * D + col; }, acc);
            }
#pragma unroll
            for (int e = 0; e < VEC; e++) join[e * 256 + tid] = acc[e];
            __syncthreads();
            if (slot == 0 && col < D) {
                for (int o = 1; o < slots; o++)
#pragma unroll
                    for (int e = 0; e < VEC; e++) acc[e] += join[e * 256 + o * lanes + lane];
                write(run.row, col, acc);
            }
            __syncthreads();
        }
        return;
    }
    const unsigned group = blockIdx.x - long_groups * col_blocks;
    if (group < short_groups) {
        const uint32_t n_short = lists.n[1];
        for (uint32_t i = group * slots + slot; i < n_short; i += short_groups * slots) {
            const Run run = lists.of_short[i];
            const int len = (int)(run.end - run.first);
            uint32_t at[kShort];
            at[0] = run.pos;
#pragma unroll
            for (int j = 1; j < kShort; j++) at[j] = pos[j < len ? run.first + j : run.first];
            for (int c0 = lane * VEC; c0 < D; c0 += kWide * lanes * VEC) {
                float acc[kWide][VEC];
#pragma unroll
                for (int k = 0; k < kWide; k++)
#pragma unroll
                    for (int e = 0; e < VEC; e++) acc[k][e] = 0.f;
#pragma unroll
                for (int j = 0; j < kShort; j++) {
                    if (j >= len) break;
                    const T *row = grad + (int64_t)at[j] * ldg;
#pragma unroll
                    for (int k = 0; k < kWide; k++) {
                        const int col = c0 + k * lanes * VEC;
                        if (col + VEC <= D) {
                            const Loose<T, VEC> t = *reinterpret_cast<const Loose<T, VEC> *>(row + col);
#pragma unroll
                            for (int e = 0; e < VEC; e++) acc[k][e] += to_f32(t.v[e]);
                        } else {
#pragma unroll
                            for (int e = 0; e < VEC; e++)
                                if (col + e < D) acc[k][e] += to_f32(row[col + e]);
                        }
                    }
                }
#pragma unroll
                for (int k = 0; k < kWide; k++)
                    if (c0 + k * lanes * VEC < D) write(run.row, c0 + k * lanes * VEC, acc[k]);
            }
        }
        return;
    }
    const int64_t v = (int64_t)(group - short_groups) * slots + slot;
    if (v >= V || lists.used[v]) return;
    float zero[VEC];
#pragma unroll
    for (int e = 0; e < VEC; e++) zero[e] = 0.f;
    for (int col = lane * VEC; col < D; col += lanes * VEC) write(v, col, zero);
}

// ------------------------------------------------------------------------------------------------ host
struct BwdPlan {
    int bits, passes, nb_max, tile;
    int64_t blocks, per;            // multi-block sort
    int64_t off_keys[2], off_pos[2], off_hist, off_partial, off_used, off_long, off_short, off_n, bytes;
};

int64_t up256(int64_t b) { return (b + 255) / 256 * 256; }

BwdPlan plan_bwd(int64_t n, int64_t V, int64_t D) {        // (V > 0: at least one pass)
    BwdPlan p = {};
    while (p.bits < 32 && ((uint64_t)V >> p.bits) != 0) p.bits++;        // keys 0 .. V
    const bool one = n <= kOneMax;
    const int digit = one ? kOneDigit : p.bits <= kOnlyDigit ? kOnlyDigit : kMultiDigit;
    p.passes = (p.bits + digit - 1) / digit;
    p.nb_max = (p.bits + p.passes - 1) / p.passes;
    p.tile = kSortThreads * (n <= kMaxBlocks * 1024 ? 1 : n <= kMaxBlocks * 2048 ? 2 : 4);
    const int64_t tiles = (n + p.tile - 1) / p.tile;
    p.per = ((tiles + kMaxBlocks - 1) / kMaxBlocks) * p.tile;
    p.blocks = one ? 1 : (n + p.per - 1) / p.per;
    int64_t at = 0;
    auto take = [&](int64_t b) { const int64_t r = at; at += up256(b); return r; };
    const int copies = one || p.passes == 1 ? 1 : 2;
    for (int k = 0; k < 2; k++) {
        p.off_keys[k] = k < copies ? take(4 * n) : p.off_keys[0];
        p.off_pos[k] = k < copies ? take(4 * n) : p.off_pos[0];
    }
    p.off_hist = one ? 0 : take(p.blocks * 4ll << p.nb_max);
    p.off_partial = take((n / kChunk) * D * 4);
    p.off_used = take(V);
    p.off_long = take((int64_t)sizeof(Run) * (n / (kShort + 1)));
    p.off_short = take((int64_t)sizeof(Run) * (n < V ? n : V));
    p.off_n = take(8);
    p.bytes = at;
    return p;
}

template <typename I, int R>
void launch_one(const I *idx, int n, int64_t V, int64_t padding, const BwdPlan &p, uint32_t *keys, uint32_t *pos, uint32_t *list_n, hipStream_t s) {
    const int lds = 4 * (256 + kSortWaves + kSortWaves * 256 / 2 + 2 * 1024 * R);
    static hsLdsAttrOnce attr;
    attr.set((const void *)k_sort_one<I, R>, lds);
    k_sort_one<I, R><<<1, kSortThreads, lds, s>>>(idx, n, V, padding, p.bits, p.passes, keys, pos, list_n);
}

template <typename I, int R>
void launch_scatter(const I *idx, const uint32_t *k_in, const uint32_t *p_in, int64_t n, int64_t V, int64_t padding, const BwdPlan &p, int shift, int nb, const uint32_t *hist,
                    uint32_t *keys, uint32_t *pos, hipStream_t s) {
    auto lds = [](int bins) { return 4 * (3 * bins + kSortWaves + 2 * R * kSortThreads) + 2 * kSortWaves * bins; };
    static hsLdsAttrOnce attr;
    attr.set((const void *)k_sort_scatter<I, R>, lds(1 << kOnlyDigit));
    k_sort_scatter<I, R><<<(unsigned)p.blocks, kSortThreads, lds(1 << nb), s>>>(idx, k_in, p_in, n, p.per, V, padding, shift, nb, hist, keys, pos);
}

template <typename I>
void launch_sort(const I *idx, int64_t n, int64_t V, int64_t padding, const BwdPlan &p, char *ws, uint32_t *&keys, uint32_t *&pos, hipStream_t s) {
    uint32_t *list_n = (uint32_t *)(ws + p.off_n);
    if (n <= kOneMax) {
        keys = (uint32_t *)(ws + p.off_keys[0]);
        pos = (uint32_t *)(ws + p.off_pos[0]);
        if (n <= 1024) launch_one<I, 1>(idx, (int)n, V, padding, p, keys, pos, list_n, s);
        else launch_one<I, 4>(idx, (int)n, V, padding, p, keys, pos, list_n, s);
        return;
    }
    uint32_t *hist = (uint32_t *)(ws + p.off_hist), *k_in = nullptr, *p_in = nullptr;
    int shift = 0;
    for (int pass = 0; pass < p.passes; pass++) {
        const int nb = (p.bits - shift + p.passes - pass - 1) / (p.passes - pass);
        keys = (uint32_t *)(ws + p.off_keys[pass & 1]);
        pos = (uint32_t *)(ws + p.off_pos[pass & 1]);
        k_sort_hist<I><<<(unsigned)p.blocks, kSortThreads, 0, s>>>(idx, k_in, n, p.per, V, padding, shift, nb, hist, list_n);
        if (p.tile == 1024) launch_scatter<I, 1>(idx, k_in, p_in, n, V, padding, p, shift, nb, hist, keys, pos, s);
        else if (p.tile == 2048) launch_scatter<I, 2>(idx, k_in, p_in, n, V, padding, p, shift, nb, hist, keys, pos, s);
        else launch_scatter<I, 4>(idx, k_in, p_in, n, V, padding, p, shift, nb, hist, keys, pos, s);
        k_in = keys;
        p_in = pos;
        shift += nb;
    }
}

bool sizes_ok(int64_t n, int64_t V, int64_t D) { return n >= 0 && n <= 0x7fffffff && V >= 0 && V < 0x7fffffff && D >= 0 && D <= (1 << 20); }

int pow2_at_least(int v) { int p = 1; while (p < v) p <<= 1; return p; }

}  // namespace

extern "C" {

int hs_embed_fwd(const void *indices, int32_t index_bytes, const void *table, int64_t ld, void *out, int64_t n, int64_t V, int64_t D, float scale, int32_t table_dtype,
                 int32_t out_dtype, void *stream) {
    if (!sizes_ok(n, V, D) || (index_bytes != 4 && index_bytes != 8) || !known_dtype(table_dtype) || !known_dtype(out_dtype) || ld < D) return HS_ERR_ARG;
    if (n == 0 || D == 0) return HS_OK;
    if (!indices || !out || (V > 0 && !table)) return HS_ERR_NULL;
    const int tb = elem_bytes(table_dtype), ob = elem_bytes(out_dtype);
    // the widest group that the row starts of both sides allow
    int vec = 8;
    while (vec > 1 && (D % vec || ld % vec || (uintptr_t)table % (vec * tb < 16 ? vec * tb : 16) || (uintptr_t)out % (vec * ob < 16 ? vec * ob : 16))) vec >>= 1;
    if (vec == 2) vec = 1;
    const int64_t per_row = D / vec, piece = kMaxGrid * 256 / per_row;        // rows per launch (a grid has less than 2^32 threads)
    hipStream_t s = (hipStream_t)stream;
    for (int64_t r0 = 0; r0 < n; r0 += piece) {
        const int64_t total = (n - r0 < piece ? n - r0 : piece) * per_row, blocks = (total + 255) / 256;
        const char *idx = (const char *)indices + r0 * index_bytes;
        char *to = (char *)out + r0 * D * ob;
#define HS_EMBED_FWD(I, VEC)                                                                                                                                      \
    HS_BY_DTYPE(table_dtype, {                                                                                                                                    \
        using TT = T;                                                                                                                                             \
        HS_BY_DTYPE(out_dtype, (k_embed_fwd<TT, T, I, VEC><<<(unsigned)blocks, 256, 0, s>>>((const I *)idx, (const TT *)table, ld, (T *)to, total,                \
                                                                                           (uint32_t)per_row, V, scale)));                                       \
    })
        if (index_bytes == 8) {
            if (vec == 8) HS_EMBED_FWD(int64_t, 8); else if (vec == 4) HS_EMBED_FWD(int64_t, 4); else HS_EMBED_FWD(int64_t, 1);
        } else {
            if (vec == 8) HS_EMBED_FWD(int32_t, 8); else if (vec == 4) HS_EMBED_FWD(int32_t, 4); else HS_EMBED_FWD(int32_t, 1);
        }
        if (hipGetLastError() != hipSuccess) return HS_ERR_LAUNCH;
    }
    return HS_OK;
}

int64_t hs_embed_bwd_ws_bytes(int64_t n, int64_t V, int64_t D) { return !sizes_ok(n, V, D) ? HS_ERR_ARG : V > 0 && D > 0 ? plan_bwd(n, V, D).bytes : 0; }

int hs_embed_bwd(const void *indices, int32_t index_bytes, const void *grad, int64_t ldg, void *grad_table, int64_t n, int64_t V, int64_t D, float scale, int64_t padding,
                 int32_t grad_dtype, int32_t table_dtype, void *ws, int64_t ws_bytes, void *stream) {
    if (!sizes_ok(n, V, D) || (index_bytes != 4 && index_bytes != 8) || !known_dtype(grad_dtype) || !known_dtype(table_dtype) || ldg < D) return HS_ERR_ARG;
    if (V == 0 || D == 0) return HS_OK;
    if (!grad_table || !ws || (n > 0 && (!indices || !grad))) return HS_ERR_NULL;
    const BwdPlan p = plan_bwd(n, V, D);
    if (ws_bytes < p.bytes) return HS_ERR_ARG;
    hipStream_t s = (hipStream_t)stream;
    uint32_t *keys = nullptr, *pos = nullptr;
    float *partial = (float *)((char *)ws + p.off_partial);
    if (n > 0) {
        if (index_bytes == 8) launch_sort((const int64_t *)indices, n, V, padding, p, (char *)ws, keys, pos, s);
        else launch_sort((const int32_t *)indices, n, V, padding, p, (char *)ws, keys, pos, s);
    }
    const int VEC = grad_dtype == HS_F32 ? 4 : 8;
    int lanes = pow2_at_least((int)((D + VEC - 1) / VEC));
    lanes = lanes > 64 ? 64 : lanes;
    const unsigned col_blocks = (unsigned)((D + (int64_t)lanes * VEC - 1) / ((int64_t)lanes * VEC));
    const int64_t row_blocks = (V + 256 / lanes - 1) / (256 / lanes);
    const unsigned bound_blocks = (unsigned)(V / 256 + 1);
    const RunLists lists = {(Run *)((char *)ws + p.off_long), (Run *)((char *)ws + p.off_short), (uint32_t *)((char *)ws + p.off_n), (uint8_t *)ws + p.off_used};
    const int64_t most_long = n / (kShort + 1);
    const unsigned long_groups = (unsigned)(most_long < kLongGroups ? most_long : kLongGroups);
    const int64_t most_short = ((n < V ? n : V) + 256 / lanes - 1) / (256 / lanes);
    const unsigned short_groups = (unsigned)(most_short < kShortGroups ? most_short : kShortGroups);
    const int64_t chunks = n / kChunk, row_bytes = D * elem_bytes(table_dtype);
    HS_BY_DTYPE(grad_dtype, {
        using G = T;
        constexpr int W = sizeof(T) == 4 ? 4 : 8;
        // one launch each; more where a grid would pass 2^32 threads
        unsigned first = bound_blocks;
        for (int64_t c0 = 0; c0 == 0 || c0 < chunks;) {
            const int64_t take = chunks - c0 < kMaxGrid - first ? chunks - c0 : kMaxGrid - first;
            k_embed_chunks<G, W><<<dim3(first + (unsigned)take, col_blocks), 256, 0, s>>>(keys + c0 * kChunk, pos + c0 * kChunk, (const G *)grad, ldg, n, (uint32_t)V, (int)D, lanes,
                                                                                       partial + c0 * D, lists, first);
            first = 0;
            if (take == chunks - c0) break;
            c0 += take;
        }
        unsigned lead = long_groups * col_blocks + short_groups;
        for (int64_t b0 = 0; b0 < row_blocks;) {
            const int64_t take = row_blocks - b0 < kMaxGrid - lead ? row_blocks - b0 : kMaxGrid - lead, v0 = b0 * (256 / lanes);
            RunLists from = lists;
            from.used += v0;
            HS_BY_DTYPE(table_dtype, (k_embed_rows<G, T, W><<<lead + (unsigned)take, 256, 0, s>>>(from, pos, (const G *)grad, ldg, V - v0, (int)D, lanes, partial, scale,
                                                                                               (T *)((char *)grad_table + v0 * row_bytes), lead ? long_groups : 0u, col_blocks,
                                                                                               lead ? short_groups : 0u)));
            lead = 0;
            b0 += take;
        }
    });
    return hipGetLastError() == hipSuccess ? HS_OK : HS_ERR_LAUNCH;
}

}  // extern "C"
