// Attention weights of a prompt's queries, summed per token and kv head: what
// eviction by accumulated weight starts from.  Not in the reference.
//
//   weights[b, kv, j] = sum over the kv head's query heads and over queries
//                       i >= j (the last `last` of the sequence) of p_ij,
//   p_i = softmax over keys j <= i of scale q_i.k_j
//
// A weight needs its whole row's maximum and sum, so the scores are formed
// twice, each time by the same tile product on 32x32x16 MFMAs: 64 columns a
// wave (32 where there is little work) stay in registers, tiles of 64 rows pass
// through LDS.
//   * prompt_stats_kernel holds queries and streams the keys up to them: per
//     query the running maximum and the sum of exponentials.  A workgroup's four
//     waves hold consecutive (64 queries, head) chunks of one kv head, heads
//     fastest, so that they share the keys and end at the same diagonal.
//   * prompt_sums_kernel holds keys and streams the queries from them on, with
//     their maxima and 1 / sums: per key the sum of exp2(s - m) / l.  Heads and
//     ranges of queries are separate workgroups, whose sums
//   * prompt_join_kernel adds in a fixed order.
// Bound by the matrix cores and the exponentials: 2 * 2 D FLOP and two
// exponentials a score.  The maximum subtracted in the first pass is the one of
// the first tile unless a sum passes 2^100: sums are in fp32, whose exponent has
// room for the rest.
// A stage's products run beside the exponentials of the block before.  Measured,
// Hq=32, Hkv=8, D=128: 8192 tokens, all queries, about 670 us (the two passes 0.82
// PFLOP/s), 2.8 us a tile of 64 rows where two workgroups share a CU; the products
// alone are 1.0, the vector work alone 1.1, both with nothing to wait for 1.6; 1111 tokens 40 us (19 + 19 + 3, a chain
// of few tiles a workgroup); the last 64 queries of 12 prompts of 1110-4096 tokens 66.
#include <algorithm>
#include <numeric>

#include "attn_kernels.hpp"
#include "mxfp4.hpp"

namespace ak {

namespace {

constexpr int kWaves = 4, kThreads = kWaves * kWave;
template <int C>
constexpr int kCols = 32 * C;             // columns that a wave holds
template <int C>
constexpr int kHeld = kWaves * kCols<C>;  // of a workgroup
constexpr int kTile = 64;             // rows of a streamed tile
constexpr int kRing = 3;              // tiles in LDS: one in use, two on their way
constexpr int kRows = 512;            // queries whose maxima and sums a workgroup of the second pass has in LDS
// Wave tiles from which on a wave holds 64 columns.  Measured with 64 / 32 columns,
// us, Hq=32, Hkv=8, D=128, all queries: 512 tokens (1024 tiles) 29.1 / 23.9, 1111
// (5184) 44.8 / 42.0, 1500 (9216) 54.3 / 49.3, 2048 (16384) 83.5 / 85.0, 8192 (262144)
// 687 / 742; the last 64 of 12 prompts of 1110-4096 (17700) 89.5 / 95.0.
constexpr double kManyTiles = 14000;
constexpr float kLowest = -3.402823466e38f;

struct Params {
    const uint16_t *q, *k;
    const int* cu;
    float* weights;
    float *m, *l;          // [key splits, hq, total]
    float* partial;        // [items, hkv, total]; nullptr: one item, written to weights
    int64_t q_stride, k_stride, w_stride_b, w_stride_h;
    int total, hkv, group, max_seqlen, last, length;
    int key_range, key_splits, heads, items_h, row_range, ranges;
    int turn;             // sequences that a workgroup's rank among its pair's is turned by
    int held;             // keys of a workgroup of the second pass
    int pairs, key_tiles;  // (sequence, kv head) pairs, the fastest part of a workgroup's number: one's keys meet in one L2
    float sl2;
};

// The sequence of a workgroup.  An XCD's workgroups go to its four shader engines in
// turn, so one sequence's would all be on one of them where batch * hkv is a multiple
// of 32: the sequences take turns too, by a.turn, which keeps a pair on its XCD.  The
// last 64 queries of 12 prompts of 1110-4096 tokens, Hkv=8: first pass 46.5 -> 36.3 us.
__device__ __forceinline__ int batch_of(const Params& a, int pair, int index) {
    const int batch = a.pairs / a.hkv;
    return (pair / a.hkv + index % batch * a.turn) % batch;
}

struct Sequence {
    int start, n, first;  // rows in the packed tensors, tokens, first query that counts
};

__device__ __forceinline__ Sequence sequence(const Params& a, int b) {
    Sequence s;
    s.start = min(max(a.cu[b], 0), a.total);
    s.n = min(min(max(a.cu[b + 1], s.start), a.total) - s.start, a.max_seqlen);
    s.first = s.n - min(a.last, s.n);
    return s;
}

// Rows of one head: token i at p + i * stride elements.
struct Rows {
    const uint16_t* p;
    int64_t stride;
};

// 16-byte units of a row, and of a tile that one thread moves.
template <int D>
constexpr int kUnits = D / 8;
template <int D>
constexpr int kPer = kTile * kUnits<D> / kThreads;

// Where unit u of tile row r stands in LDS: 16 consecutive rows' same units
// are on 16 different places of the 256 bytes that one read group covers.
template <int D>
__device__ __forceinline__ int place(int r, int u) {
    return D == 128 ? r * 16 + (u ^ (r & 15)) : r * 8 + (u ^ (r >> 1 & 7));
}

// Starts rows i0 .. of `rows` (those past `end` as row end - 1) on their way
// into a tile, straight from memory: a wave's 64 lanes fill 1 KB of it, each
// lane with the unit that belongs to its place.  A tile of whole rows has a
// scalar base and the same 32-bit offsets every time.  In asm so that the
// compiler's waits for LDS reads do not wait for these too; tile_ready waits.
// s_nop 4: the wait states for a base that a vector instruction has just
// written (a spilled scalar's v_readlane), which the compiler cannot see in asm;
// they cover the write of M0 too.
template <int D>
__device__ __forceinline__ void load_tile(const Rows& rows, int i0, int end, u32x4* tile, int w, int lane) {
    const uint16_t* base = rows.p + (int64_t)i0 * rows.stride;
    const bool whole = i0 + kTile <= end;
#pragma unroll
    for (int j = 0; j < kPer<D>; ++j) {
        const int at = (j * kWaves + w) * kWave + lane, r = at / kUnits<D>, p = at % kUnits<D>;
        const int u = D == 128 ? p ^ (r & 15) : p ^ (r >> 1 & 7);
        typedef __attribute__((address_space(3))) void lds_void;
        const uint32_t l = __builtin_amdgcn_readfirstlane((uint32_t)(size_t)(lds_void*)(tile + (j * kWaves + w) * kWave));
        if (whole) {
            const uint32_t off = ((uint32_t)r * (uint32_t)rows.stride + u * 8) * 2;
            asm volatile("s_nop 4\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "{m0}"(l) : "memory");
        } else {
            const uint16_t* g = rows.p + (int64_t)min(i0 + r, end - 1) * rows.stride + u * 8;
            asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(g), "{m0}"(l) : "memory");
        }
    }
}

// Waits until the oldest tile is there, `later` tiles (at most kRing - 2) having
// been started after it, and until every wave is done with the one before.
template <int D>
__device__ __forceinline__ void tile_ready(int later) {
    static_assert(kRing == 3, "one tile may be on its way behind the one that is waited for");
    if (later > 0) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kPer<D>) : "memory");
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
}

// The score that is -infinity once it is scaled.
__device__ __forceinline__ float masked_score(float sl2) { return sl2 < 0.f ? INFINITY : -INFINITY; }

// The order of a stage's instructions (0x008 MFMA, 0x002 vector, 0x400
// exponentials, 0x100 LDS reads): the products of one block with an equal share
// of the other's exponentials and VALU vector instructions behind each.
template <int D, int C, int VALU>
__device__ __forceinline__ void interleave() {
    constexpr int N = C * D / 16;  // products
    __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x002, (VALU + N - 1) / N, 0);
        __builtin_amdgcn_sched_group_barrier(0x400, 16 * C / N, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
}

// Scores (unscaled) of the tile's rows 32 blk .. 32 blk + 31 against the held columns.
template <int D, class T, int C>
__device__ __forceinline__ void product(const u32x4* tile, int blk, const u32x4 (&held)[C][D / 16], int lane,
                                        f32x16 (&s)[C]) {
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[c][i] = 0.f;
#pragma unroll
    for (int k = 0; k < D / 16; ++k) {
        const u32x4 row = tile[place<D>(32 * blk + (lane & 31), 2 * k + (lane >> 5))];
#pragma unroll
        for (int c = 0; c < C; ++c) s[c] = Half<T>::mfma32(row, held[c][k], s[c]);
    }
}

// Starts the held columns' loads: rows i0 .. of `rows`, those past `end` as row end - 1.
// A product's operand is 16 of every 32 bytes of a lane's row; loaded so, four loads
// would meet each cache line, and all but the first would wait for it.  Instead a
// quad's lanes load each of their four rows' lines in turn, and trade in held_ready:
// the last 64 queries of 12 prompts of 1110-4096 tokens 68.6 -> 66.1 us.
template <int D, int C>
__device__ __forceinline__ void hold(const Rows& rows, int i0, int end, int lane, u32x4 (&held)[C][D / 16]) {
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
            const int i = min(i0 + 32 * c + (lane & 28) + k % 4, end - 1), of_line = lane & 3;
            held[c][k] = *reinterpret_cast<const u32x4*>(rows.p + i * rows.stride + 16 * (k / 4 * 4 + of_line) +
                                                         8 * (lane >> 5));
        }
}
template <int D, int C>
__device__ __forceinline__ void held_ready(u32x4 (&held)[C][D / 16], int lane) {
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
        for (int k = 0; k < D / 16; k += 4)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                uint32_t x[4] = {held[c][k][i], held[c][k + 1][i], held[c][k + 2][i], held[c][k + 3][i]};
                transpose_quad(x[0], x[1], x[2], x[3], lane);
#pragma unroll
                for (int j = 0; j < 4; ++j) held[c][k + j][i] = x[j];
            }
}

// The row of register r of a 32 x 32 product in this lane.
__device__ __forceinline__ int row_of(int r, int lane) { return 8 * (r / 4) + 4 * (lane >> 5) + r % 4; }

template <int D, class T, int C>
__global__ void __launch_bounds__(kThreads, C == 2 ? 2 : 3) prompt_stats_kernel(const Params a) {
    __shared__ u32x4 tiles[kRing][kTile * kUnits<D>];
    const int pair = blockIdx.x % a.pairs, kvh = pair % a.hkv, index = blockIdx.x / a.pairs;
    const int b = batch_of(a, pair, index);
    const int tid = threadIdx.x, lane = tid & 63, w = uniform(tid >> 6);
    const int G = a.group;
    const Sequence sq = sequence(a, b);
    const int R = sq.n - sq.first;
    const int chunks = (R + kCols<C> - 1) / kCols<C> * G;
    // The longest streams first: the last queries have the lowest workgroup numbers.
    const int groups = (chunks + kWaves - 1) / kWaves;
    const int part = index % a.key_splits, group = groups - 1 - index / a.key_splits;
    if (group < 0) return;
    const int chunk = min(group * kWaves + w, chunks - 1);
    const int h = kvh * G + chunk % G, q0 = sq.first + chunk / G * kCols<C>;  // position of the wave's first query
    const bool spare = group * kWaves + w >= chunks;
    const int last_chunk = min(group * kWaves + kWaves, chunks) - 1;
    const int begin = part * a.key_range;
    const int end = min(min(sq.first + (last_chunk / G + 1) * kCols<C>, sq.n), begin + a.key_range);
    const int count = begin < end ? (end - begin + kTile - 1) / kTile : 0;
    const Rows keys{a.k + (int64_t)sq.start * a.k_stride + kvh * D, a.k_stride};
    const Rows queries{a.q + (int64_t)sq.start * a.q_stride + h * D, a.q_stride};
    for (int t = 0; t < kRing - 1 && t < count; ++t) load_tile<D>(keys, begin + t * kTile, end, tiles[t], w, lane);
    u32x4 held[C][D / 16];
    hold<D, C>(queries, q0, sq.n, lane, held);

    const float lowest = masked_score(a.sl2);
    float m[C], l[C];
#pragma unroll
    for (int c = 0; c < C; ++c) {
        m[c] = kLowest;
        l[c] = 0.f;
    }
    // Adds the exponentials of a block's scores to sum.
    auto weigh = [&](const f32x16 (&x)[C], float (&sum)[C]) {
#pragma unroll
        for (int c = 0; c < C; ++c) {
            float t[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int r = 0; r < 16; ++r) t[r % 4] += exp2_fast(x[c][r] * a.sl2 - m[c]);
            sum[c] = l[c] + ((t[0] + t[1]) + (t[2] + t[3]));
        }
    };
    // One stage: the scores of rows kb .. (tile block blk) into x, while those of
    // the block before, y, become exponentials; live: the block before has any.
    bool live = false;
    auto stage = [&](const u32x4* tile, int blk, int kb, f32x16 (&x)[C], const f32x16 (&y)[C]) {
        const bool now = !spare && kb < end && kb < q0 + kCols<C>;  // a key that some query sees
        float sum[C];
        if (now && live) {
            product<D, T, C>(tile, blk, held, lane, x);
            weigh(y, sum);
            interleave<D, C, C * 36>();
        } else if (now) {
            product<D, T, C>(tile, blk, held, lane, x);
        } else if (live) {
            weigh(y, sum);
        }
        if (live) {
            // The maximum subtracted stays unless the sums pass 2^100 (as
            // against the lowest number at first); then the block is done again.
            float top = sum[0];
            if constexpr (C == 2) top += sum[1];
            if (__builtin_amdgcn_ballot_w64(!(top <= 0x1p100f))) {
#pragma unroll
                for (int c = 0; c < C; ++c) {
                    float mx = m[c];
#pragma unroll
                    for (int r = 0; r < 16; ++r) mx = fmaxf(mx, y[c][r] * a.sl2);
                    l[c] *= exp2_fast(m[c] - mx);
                    m[c] = mx;
                }
                weigh(y, sum);
            }
#pragma unroll
            for (int c = 0; c < C; ++c) l[c] = sum[c];
        }
        if (now && (kb + 31 > q0 || kb + 32 > end)) {  // keys after a query, or past the range
#pragma unroll
            for (int c = 0; c < C; ++c) {
                int limit = min(q0 + 32 * c + (lane & 31), end - 1) - kb;
                asm volatile("" : "+v"(limit));  // nothing of this is done ahead of the branch
#pragma unroll
                for (int r = 0; r < 16; ++r) x[c][r] = row_of(r, lane) > limit ? lowest : x[c][r];
            }
        }
        live = now;
    };
    held_ready<D, C>(held, lane);
    f32x16 x[C], y[C];
    for (int t = 0, cur = 0; t < count; ++t, cur = cur == kRing - 1 ? 0 : cur + 1) {
        const int k0 = begin + t * kTile;
        tile_ready<D>(count - 1 - t);
        if (t + kRing - 1 < count)
            load_tile<D>(keys, k0 + (kRing - 1) * kTile, end, tiles[cur == 0 ? kRing - 1 : cur - 1], w, lane);
        stage(tiles[cur], 0, k0, x, y);
        stage(tiles[cur], 1, k0 + 32, y, x);
    }
    stage(tiles[0], 0, end, x, y);  // the last block's exponentials
    if (spare) return;
    // A column's rows are in two lanes.
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const float m2 = __shfl_xor(m[c], 32, kWave), l2 = __shfl_xor(l[c], 32, kWave);
        const float mx = fmaxf(m[c], m2);
        const float sum = l[c] * exp2_fast(m[c] - mx) + l2 * exp2_fast(m2 - mx);
        const int i = q0 + 32 * c + (lane & 31);
        if (lane < 32 && i < sq.n) {
            const size_t at = ((size_t)part * a.hkv * G + h) * a.total + sq.start + i;
            a.m[at] = mx;
            a.l[at] = sum;
        }
    }
}

// Whether the queries of range j reach a tile of keys that begins with `key`.
__device__ __forceinline__ bool reaches(const Params& a, const Sequence& sq, int j, int key) {
    const int lo = sq.first + j * a.row_range, hi = min(sq.n, lo + a.row_range);
    return lo < hi && hi > key;
}

template <int D, class T, int C>
__global__ void __launch_bounds__(kThreads, C == 2 ? 2 : 3) prompt_sums_kernel(const Params a) {
    __shared__ u32x4 tiles[kRing][kTile * kUnits<D>];
    __shared__ f32x4 row_m[kRows / 4], row_w[kRows / 4];
    // The last ranges, which all keys stream, first.
    const int pair = blockIdx.x % a.pairs, kvh = pair % a.hkv;
    int index = blockIdx.x / a.pairs;
    const int b = batch_of(a, pair, index);
    const int part = index % a.items_h, head0 = part * a.heads;
    index /= a.items_h;
    const int kt = index % a.key_tiles, j = a.ranges - 1 - index / a.key_tiles, item = part * a.ranges + j;
    const int tid = threadIdx.x, lane = tid & 63, w = uniform(tid >> 6);
    const Sequence sq = sequence(a, b);
    const int k0 = kt * kHeld<C> + w * kCols<C>;
    // One item in all: its sums are the weights.
    float* const weights = a.partial ? nullptr : a.weights + b * a.w_stride_b + kvh * a.w_stride_h;
    if (kt * kHeld<C> >= sq.n || !reaches(a, sq, j, kt * kHeld<C>)) {
        if (weights && lane < kCols<C> && k0 + lane < a.length) weights[k0 + lane] = 0.f;
        return;
    }
    const int heads = min(a.heads, a.group - head0), h0 = kvh * a.group + head0;
    const int lo = sq.first + j * a.row_range, end = min(sq.n, lo + a.row_range);
    const int begin = lo + max(kt * kHeld<C> - lo, 0) / kTile * kTile;
    const int per_head = (end - begin + kTile - 1) / kTile, count = per_head * heads;
    const Rows keys{a.k + (int64_t)sq.start * a.k_stride + kvh * D, a.k_stride};
    Rows queries{a.q + (int64_t)sq.start * a.q_stride + (int64_t)h0 * D, a.q_stride};
    // Tiles go through the range's queries head by head; the loads run kRing - 1 tiles ahead.
    int ahead = 0;
    auto load_next = [&](int buf) {
        load_tile<D>(queries, begin + ahead * kTile, end, tiles[buf], w, lane);
        if (++ahead == per_head) {
            ahead = 0;
            queries.p += D;
        }
    };
    for (int t = 0; t < kRing - 1 && t < count; ++t) load_next(t);
    u32x4 held[C][D / 16];
    hold<D, C>(keys, k0, sq.n, lane, held);
    // Every row's maximum and 1 / sum over the key splits; rows past the end weigh nothing.
    for (int i = tid; i < count * kTile; i += kThreads) {
        const int head = i / (per_head * kTile), pos = begin + i % (per_head * kTile);
        float m = INFINITY, wgt = 0.f;
        if (pos < end) {
            const size_t step = (size_t)a.hkv * a.group * a.total;
            const size_t at = (size_t)(h0 + head) * a.total + sq.start + pos;
            float L = 0.f;
            m = kLowest;
            constexpr int kTogether = 8;  // splits whose loads are on their way together
            for (int p0 = 0; p0 < a.key_splits; p0 += kTogether) {
                float lp[kTogether] = {}, mp[kTogether] = {};
#pragma unroll
                for (int p = 0; p < kTogether; ++p)
                    if (p0 + p < a.key_splits) {
                        lp[p] = a.l[at + (p0 + p) * step];
                        mp[p] = a.m[at + (p0 + p) * step];
                    }
                float mx = m;
#pragma unroll
                for (int p = 0; p < kTogether; ++p) mx = lp[p] == 0.f ? mx : fmaxf(mx, mp[p]);
                L *= exp2_fast(m - mx);
#pragma unroll
                for (int p = 0; p < kTogether; ++p) L += lp[p] == 0.f ? 0.f : lp[p] * exp2_fast(mp[p] - mx);
                m = mx;
            }
            wgt = L == 0.f ? 0.f : 1.f / L;  // every score -inf: nothing
        }
        reinterpret_cast<float*>(row_m)[i] = m;
        reinterpret_cast<float*>(row_w)[i] = wgt;
    }
    const float lowest = masked_score(a.sl2);
    float sum[C][2] = {};
    // Adds a block's weights; its rows' numbers among row_m and row_w start at 32 at.
    auto weigh = [&](const f32x16 (&x)[C], int at) {
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
            const f32x4 m = row_m[8 * at + r / 2 + (lane >> 5)], wgt = row_w[8 * at + r / 2 + (lane >> 5)];
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    sum[c][i % 2] = fmaf(exp2_fast(x[c][r + i] * a.sl2 - m[i]), wgt[i], sum[c][i % 2]);
        }
    };
    // One stage, as in the first pass: rows ib .. , the at-th block.
    bool live = false;
    auto stage = [&](const u32x4* tile, int blk, int ib, int at, f32x16 (&x)[C], const f32x16 (&y)[C]) {
        const bool now = ib < end && ib + 32 > k0;  // a query that sees some key
        if (now && live) {
            product<D, T, C>(tile, blk, held, lane, x);
            weigh(y, at - 1);
            interleave<D, C, C * 32>();
        } else if (now) {
            product<D, T, C>(tile, blk, held, lane, x);
        } else if (live) {
            weigh(y, at - 1);
        }
        if (now && ib < k0 + kCols<C> - 1) {  // queries before a key
#pragma unroll
            for (int c = 0; c < C; ++c) {
                int limit = k0 + 32 * c + (lane & 31) - ib;
                asm volatile("" : "+v"(limit));  // nothing of this is done ahead of the branch
#pragma unroll
                for (int r = 0; r < 16; ++r) x[c][r] = row_of(r, lane) < limit ? lowest : x[c][r];
            }
        }
        live = now;
    };
    held_ready<D, C>(held, lane);
    f32x16 x[C], y[C];
    for (int t = 0, cur = 0, i0 = begin; t < count; ++t, cur = cur == kRing - 1 ? 0 : cur + 1) {
        tile_ready<D>(count - 1 - t);
        if (t + kRing - 1 < count) load_next(cur == 0 ? kRing - 1 : cur - 1);
        stage(tiles[cur], 0, i0, 2 * t, x, y);
        stage(tiles[cur], 1, i0 + 32, 2 * t + 1, y, x);
        i0 += kTile;
        if (i0 >= end) i0 = begin;
    }
    stage(tiles[0], 0, end, 2 * count, x, y);  // the last block's weights
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const float one = sum[c][0] + sum[c][1], both = one + __shfl_xor(one, 32, kWave);
        const int i = k0 + 32 * c + (lane & 31);
        if (lane >= 32) continue;
        if (weights && i < a.length) weights[i] = i < sq.n ? both : 0.f;
        if (!weights && i < sq.n) a.partial[((size_t)item * a.hkv + kvh) * a.total + sq.start + i] = both;
    }
}

__global__ void __launch_bounds__(kThreads) prompt_join_kernel(const Params a) {
    const int kvh = blockIdx.y, b = blockIdx.z, i = blockIdx.x * kThreads + threadIdx.x;
    if (i >= a.length) return;
    const Sequence sq = sequence(a, b);
    float sum = 0.f;
    if (i < sq.n) {
        // The ranges whose queries reach the token's tile are the last ones.
        const int used = (sq.n - sq.first + a.row_range - 1) / a.row_range, tile = i / a.held * a.held;
        const int j0 = min(max((tile - sq.first) / a.row_range, 0), used);
        const float* p = a.partial + (size_t)kvh * a.total + sq.start + i;
        const size_t step = (size_t)a.hkv * a.total;
        for (int item = 0; item < a.items_h; ++item)
#pragma unroll 8
            for (int j = j0; j < used; ++j) sum += p[(item * a.ranges + j) * step];
    }
    a.weights[b * a.w_stride_b + kvh * a.w_stride_h + i] = sum;
}

// How the work is cut.  A wave holds 64 columns (C = 2), or 32 where workgroups are
// few: more of them, and of fewer registers, then hide each other's latencies.
// First pass: keys are split where few queries count.  Second pass: an item is a
// range of at most kRows queries of one head, or several heads' queries where a
// head has few of them and enough workgroups are left.
struct Plan {
    int64_t columns;  // C
    int64_t key_range, key_splits, heads, items_h, row_range, ranges;
    int64_t key_tiles, stats_workgroups, sums_workgroups;
};

Plan make_plan(int64_t batch, int64_t total, int64_t hq, int64_t hkv, int64_t max_seqlen, int64_t last,
               int64_t length) {
    Plan p;
    const int64_t rows = std::min(last, max_seqlen), group = hq / hkv, pairs = batch * hkv;
    // Prompts of max_seqlen that hold as many tokens as there are.
    const double full = std::min((double)batch, (double)total / (double)max_seqlen);
    auto groups_of = [&](int64_t columns) {
        return ((rows + 32 * columns - 1) / (32 * columns) * group + kWaves - 1) / kWaves;
    };
    // Wave tiles of 64 columns and 64 rows.
    const double r = (double)((rows + 63) / 64), tiles = full * (double)hq * r * ((double)((max_seqlen + 63) / 64) - r / 2);
    p.columns = tiles >= kManyTiles ? 2 : 1;
    const int64_t slots = p.columns == 2 ? 512 : 768, groups = groups_of(p.columns);
    const int64_t most = (max_seqlen + 127) / 128;  // ranges of at least 128 keys
    // A sequence's last split is half empty on average.
    const double spare = (double)slots - 0.5 * (double)(groups * pairs);
    const int64_t want = std::max<int64_t>(1, std::min(most, (int64_t)(spare / (full * (double)(groups * hkv)))));
    p.key_range = ((max_seqlen + want - 1) / want + kTile - 1) / kTile * kTile;
    p.key_splits = (max_seqlen + p.key_range - 1) / p.key_range;
    p.row_range = kRows;
    p.ranges = (rows + kRows - 1) / kRows;
    p.heads = 1;
    const int64_t held = kWaves * 32 * p.columns, key_tiles = (max_seqlen + held - 1) / held;
    if (p.ranges == 1) {
        const int64_t padded = (rows + kTile - 1) / kTile * kTile;
        while (p.heads * 2 <= group && p.heads * 2 * padded <= kRows &&
               key_tiles * pairs * ((group + p.heads * 2 - 1) / (p.heads * 2)) >= slots)
            p.heads *= 2;
    }
    p.items_h = (group + p.heads - 1) / p.heads;
    // One item writes the weights itself, the zeros behind the longest prompt too.
    p.key_tiles = p.items_h * p.ranges == 1 ? (length + held - 1) / held : key_tiles;
    p.stats_workgroups = groups * p.key_splits * pairs;
    p.sums_workgroups = p.key_tiles * p.items_h * p.ranges * pairs;
    return p;
}

template <int D, class T, int C>
hipError_t launch(const PromptWeightsArgs& x, const Plan& plan) {
    Params p{};
    p.q = static_cast<const uint16_t*>(x.q);
    p.k = static_cast<const uint16_t*>(x.k);
    p.cu = x.cu;
    p.weights = x.weights;
    const size_t stats = (size_t)plan.key_splits * x.hq * x.total;
    p.m = static_cast<float*>(x.workspace);
    p.l = p.m + stats;
    const bool direct = plan.items_h * plan.ranges == 1;
    p.partial = direct ? nullptr : p.l + stats;
    p.q_stride = x.q_stride;
    p.k_stride = x.k_stride;
    p.w_stride_b = x.w_stride_b;
    p.w_stride_h = x.w_stride_h;
    p.total = (int)x.total;
    p.hkv = (int)x.hkv;
    p.group = (int)(x.hq / x.hkv);
    p.max_seqlen = (int)x.max_seqlen;
    p.last = (int)x.last;
    p.length = (int)x.length;
    p.key_range = (int)plan.key_range;
    p.key_splits = (int)plan.key_splits;
    p.heads = (int)plan.heads;
    p.items_h = (int)plan.items_h;
    p.row_range = (int)plan.row_range;
    p.ranges = (int)plan.ranges;
    p.sl2 = x.sl2;
    const int step = 8 / std::gcd(8, (int)x.hkv);
    p.turn = x.batch % step == 0 ? step : 0;
    p.held = kHeld<C>;
    p.pairs = (int)(x.batch * x.hkv);
    p.key_tiles = (int)plan.key_tiles;
    const auto stream = (hipStream_t)x.stream;
    hipLaunchKernelGGL((prompt_stats_kernel<D, T, C>), dim3((unsigned)plan.stats_workgroups), dim3(kThreads), 0, stream,
                       p);
    hipLaunchKernelGGL((prompt_sums_kernel<D, T, C>), dim3((unsigned)plan.sums_workgroups), dim3(kThreads), 0, stream, p);
    if (direct) return hipGetLastError();
    hipLaunchKernelGGL(prompt_join_kernel,
                       dim3((unsigned)((x.length + kThreads - 1) / kThreads), (unsigned)x.hkv, (unsigned)x.batch),
                       dim3(kThreads), 0, stream, p);
    return hipGetLastError();
}

template <int D, class T>
hipError_t launch_columns(const PromptWeightsArgs& x) {
    const Plan plan = make_plan(x.batch, x.total, x.hq, x.hkv, x.max_seqlen, x.last, x.length);
    return plan.columns == 2 ? launch<D, T, 2>(x, plan) : launch<D, T, 1>(x, plan);
}

}  // namespace

size_t prompt_weights_workspace(int64_t batch, int64_t total, int64_t hq, int64_t hkv, int64_t max_seqlen,
                                int64_t last) {
    const Plan p = make_plan(batch, total, hq, hkv, max_seqlen, last, max_seqlen);
    return sizeof(float) * (size_t)total * (size_t)(2 * p.key_splits * hq + hkv * p.items_h * p.ranges);
}

hipError_t prompt_weights_launch(const PromptWeightsArgs& x) {
    if (x.total == 0 || x.max_seqlen == 0) {  // no rows: zeros
        Params p{};
        p.cu = x.cu;
        p.weights = x.weights;
        p.length = (int)x.length;
        p.w_stride_b = x.w_stride_b;
        p.w_stride_h = x.w_stride_h;
        hipLaunchKernelGGL(prompt_join_kernel,
                           dim3((unsigned)((x.length + kThreads - 1) / kThreads), (unsigned)x.hkv, (unsigned)x.batch),
                           dim3(kThreads), 0, (hipStream_t)x.stream, p);
        return hipGetLastError();
    }
    if (x.d == 128) return x.bf16 ? launch_columns<128, bf16>(x) : launch_columns<128, f16>(x);
    return x.bf16 ? launch_columns<64, bf16>(x) : launch_columns<64, f16>(x);
}

bool prompt_weights_fits(const PromptWeightsArgs& x) {
    if (x.total == 0 || x.max_seqlen == 0) return true;
    const Plan p = make_plan(x.batch, x.total, x.hq, x.hkv, x.max_seqlen, x.last, x.length);
    return std::max(p.stats_workgroups, p.sums_workgroups) <= INT32_MAX;
}

}  // namespace ak
