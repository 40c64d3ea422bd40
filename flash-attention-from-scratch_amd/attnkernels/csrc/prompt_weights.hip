// Attention weights of a prompt's queries, summed per token and kv head: what
// eviction by accumulated weight starts from.  Not in the reference.
//
//   weights[b, kv, j] = sum over the kv head's query heads and over queries
//                       i >= j (the last `last` of the sequence) of p_ij,
//   p_i = softmax over keys j <= i of scale q_i.k_j
//
// A weight needs its whole row's maximum and sum, so the scores are formed
// twice, each time by the same tile product on 32x32x16 MFMAs: 64 columns a
// wave stay in registers, tiles of 64 rows pass through LDS.
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
// the first tile unless a sum passes 2^80: sums are in fp32, whose exponent has
// room for the rest.
#include <algorithm>

#include "attn_kernels.hpp"
#include "mxfp4.hpp"

namespace ak {

namespace {

constexpr int kWaves = 4, kThreads = kWaves * kWave;
constexpr int kCols = 64;             // columns that a wave holds
constexpr int kHeld = kWaves * kCols; // of a workgroup
constexpr int kTile = 64;             // rows of a streamed tile
constexpr float kLowest = -3.402823466e38f;

struct Params {
    const uint16_t *q, *k;
    const int* cu;
    float* weights;
    float *m, *l;          // [key splits, hq, total]
    float* partial;        // [items, hkv, total]
    int64_t q_stride, k_stride, w_stride_b, w_stride_h;
    int total, hkv, group, max_seqlen, last, length;
    int key_range, key_splits, row_range, ranges;
    float sl2;
};

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

template <int D>
struct Stream {
    static constexpr int UNITS = D / 8;                       // 16-byte units of a row
    static constexpr int PER = kTile * UNITS / kThreads;      // units of a thread
    u32x4 x[PER];

    // Where unit u of tile row r stands in LDS: 16 consecutive rows' same units
    // are on 16 different places of the 256 bytes that one read group covers.
    static __device__ __forceinline__ int place(int r, int u) {
        return D == 128 ? r * 16 + (u ^ (r & 15)) : r * 8 + (u ^ (r >> 1 & 7));
    }
    // Rows i0 + r, those past `end` as row end - 1.
    __device__ __forceinline__ void load(const Rows& rows, int i0, int end, int tid) {
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const int id = tid + j * kThreads, r = id / UNITS, u = id % UNITS;
            const int i = min(i0 + r, end - 1);
            x[j] = *reinterpret_cast<const u32x4*>(rows.p + i * rows.stride + u * 8);
        }
    }
    __device__ __forceinline__ void store(u32x4* tile, int tid) const {
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const int id = tid + j * kThreads;
            tile[place(id / UNITS, id % UNITS)] = x[j];
        }
    }
};

// Scores (unscaled) of the tile's rows 32 blk .. 32 blk + 31 against the held columns.
template <int D, class T>
__device__ __forceinline__ void product(const u32x4* tile, int blk, const u32x4 (&held)[2][D / 16], int lane,
                                        f32x16 (&s)[2]) {
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[c][i] = 0.f;
#pragma unroll
    for (int k = 0; k < D / 16; ++k) {
        const u32x4 row = tile[Stream<D>::place(32 * blk + (lane & 31), 2 * k + (lane >> 5))];
        s[0] = Half<T>::mfma32(row, held[0][k], s[0]);
        s[1] = Half<T>::mfma32(row, held[1][k], s[1]);
    }
}

template <int D>
__device__ __forceinline__ void hold(const Rows& rows, int i0, int end, int lane, u32x4 (&held)[2][D / 16]) {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        const int i = min(i0 + 32 * c + (lane & 31), end - 1);
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
            held[c][k] = *reinterpret_cast<const u32x4*>(rows.p + i * rows.stride + 16 * k + 8 * (lane >> 5));
    }
}

// Tiles of rows [begin, end) through LDS: use(tile, first row, rows' end) once for each, by every wave.
template <int D, class Use, class Stage>
__device__ __forceinline__ void stream(const Rows& rows, int begin, int end, u32x4 (&tiles)[2][kTile * D / 8], int tid,
                                       Stage stage, Use use) {
    Stream<D> next;
    next.load(rows, begin, end, tid);
    next.store(tiles[0], tid);
    stage(begin, 0);
    if (begin + kTile < end) next.load(rows, begin + kTile, end, tid);
    __syncthreads();
    int cur = 0;
    for (int i = begin; i < end; i += kTile, cur ^= 1) {
        if (i + kTile < end) {
            next.store(tiles[cur ^ 1], tid);
            stage(i + kTile, cur ^ 1);
            if (i + 2 * kTile < end) next.load(rows, i + 2 * kTile, end, tid);
        }
        use(tiles[cur], i, cur);
        __syncthreads();
    }
}

// The row of register r of a 32 x 32 product in this lane.
__device__ __forceinline__ int row_of(int r, int lane) { return 8 * (r / 4) + 4 * (lane >> 5) + r % 4; }

template <int D, class T>
__global__ void __launch_bounds__(kThreads) prompt_stats_kernel(const Params a) {
    __shared__ u32x4 tiles[2][kTile * D / 8];
    const int kvh = blockIdx.y, b = blockIdx.z;
    const int tid = threadIdx.x, lane = tid & 63, w = uniform(tid >> 6);
    const int G = a.group;
    const Sequence sq = sequence(a, b);
    const int R = sq.n - sq.first;
    const int chunks = (R + kCols - 1) / kCols * G;
    // The longest streams first: the last queries have the lowest workgroup numbers.
    const int groups = (chunks + kWaves - 1) / kWaves;
    const int part = blockIdx.x % a.key_splits, group = groups - 1 - (int)blockIdx.x / a.key_splits;
    if (group < 0) return;
    const int chunk = min(group * kWaves + w, chunks - 1);
    const int h = kvh * G + chunk % G, q0 = sq.first + chunk / G * kCols;  // position of the wave's first query
    const bool spare = group * kWaves + w >= chunks;
    const int last_chunk = min(group * kWaves + kWaves, chunks) - 1;
    const int k_begin = part * a.key_range;
    const int k_end = min(min(sq.first + (last_chunk / G + 1) * kCols, sq.n), k_begin + a.key_range);
    float m[2] = {kLowest, kLowest}, l[2] = {0.f, 0.f};
    if (k_begin < k_end) {
        const Rows keys{a.k + (int64_t)sq.start * a.k_stride + kvh * D, a.k_stride};
        const Rows queries{a.q + (int64_t)sq.start * a.q_stride + h * D, a.q_stride};
        u32x4 held[2][D / 16];
        hold<D>(queries, q0, sq.n, lane, held);
        stream<D>(keys, k_begin, k_end, tiles, tid, [](int, int) {}, [&](const u32x4* tile, int k0, int) {
            if (spare || k0 > q0 + kCols - 1) return;
#pragma unroll
            for (int blk = 0; blk < 2; ++blk) {
                const int kb = k0 + 32 * blk;
                f32x16 s[2];
                product<D, T>(tile, blk, held, lane, s);
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const int qc = q0 + 32 * c;
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[c][r] *= a.sl2;
                    if (kb + 31 > qc || kb + 32 > k_end) {  // keys after a query, or past the range
                        const int limit = min(qc + (lane & 31), k_end - 1) - kb;
#pragma unroll
                        for (int r = 0; r < 16; ++r) s[c][r] = row_of(r, lane) > limit ? -INFINITY : s[c][r];
                    }
                    auto sum = [&]() {
                        float t[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int r = 0; r < 16; ++r) t[r % 4] += exp2_fast(s[c][r] - m[c]);
                        return (t[0] + t[1]) + (t[2] + t[3]);
                    };
                    float add = sum();
                    if (__builtin_amdgcn_ballot_w64(!(add <= 0x1p80f))) {
                        float mx = m[c];
#pragma unroll
                        for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[c][r]);
                        l[c] *= exp2_fast(m[c] - mx);
                        m[c] = mx;
                        add = sum();
                    }
                    l[c] += add;
                }
            }
        });
    }
    if (spare) return;
    // A column's rows are in two lanes.
#pragma unroll
    for (int c = 0; c < 2; ++c) {
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

// Whether the queries of range j reach key tile kt (tiles of kHeld keys).
__device__ __forceinline__ bool reaches(const Params& a, const Sequence& sq, int j, int kt) {
    const int lo = sq.first + j * a.row_range, hi = min(sq.n, lo + a.row_range);
    return lo < hi && hi > kt * kHeld;
}

template <int D, class T>
__global__ void __launch_bounds__(kThreads) prompt_sums_kernel(const Params a) {
    __shared__ u32x4 tiles[2][kTile * D / 8];
    __shared__ f32x4 row_m[2][kTile / 4], row_w[2][kTile / 4];
    const int kt = blockIdx.x, kvh = blockIdx.y % a.hkv, b = blockIdx.z;
    const int item = blockIdx.y / a.hkv, head = item / a.ranges, j = item % a.ranges;
    const int tid = threadIdx.x, lane = tid & 63, w = uniform(tid >> 6);
    const Sequence sq = sequence(a, b);
    if (kt * kHeld >= sq.n || !reaches(a, sq, j, kt)) return;
    const int h = kvh * a.group + head;
    const int k0 = kt * kHeld + w * kCols;
    const int lo = sq.first + j * a.row_range, end = min(sq.n, lo + a.row_range);
    const int begin = lo + max(kt * kHeld - lo, 0) / kTile * kTile;
    const Rows keys{a.k + (int64_t)sq.start * a.k_stride + kvh * D, a.k_stride};
    const Rows queries{a.q + (int64_t)sq.start * a.q_stride + h * D, a.q_stride};
    u32x4 held[2][D / 16];
    hold<D>(keys, k0, sq.n, lane, held);
    float sum[2] = {0.f, 0.f};
    auto stage = [&](int i0, int buf) {  // the tile's rows: maximum and 1 / sum
        if (tid >= kTile) return;
        const int i = i0 + tid;
        float m = INFINITY, wgt = 0.f;  // past the end: weighs nothing
        if (i < end) {
            const size_t step = (size_t)a.hkv * a.group * a.total;
            const size_t at = (size_t)h * a.total + sq.start + i;
            float M = kLowest, L = 0.f;
            for (int p = 0; p < a.key_splits; ++p) {
                const float lp = a.l[at + p * step], mp = lp == 0.f ? kLowest : a.m[at + p * step];
                const float mx = fmaxf(M, mp);
                L = L * exp2_fast(M - mx) + lp * exp2_fast(mp - mx);
                M = mx;
            }
            m = M;
            wgt = L == 0.f ? 0.f : 1.f / L;  // every score -inf: nothing
        }
        reinterpret_cast<float*>(row_m[buf])[tid] = m;
        reinterpret_cast<float*>(row_w[buf])[tid] = wgt;
    };
    stream<D>(queries, begin, end, tiles, tid, stage, [&](const u32x4* tile, int i0, int buf) {
        if (i0 + kTile <= k0) return;  // every query before the wave's keys
#pragma unroll
        for (int blk = 0; blk < 2; ++blk) {
            const int ib = i0 + 32 * blk;
            f32x16 s[2];
            product<D, T>(tile, blk, held, lane, s);
            f32x4 m[4], wgt[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                m[r] = row_m[buf][8 * blk + 2 * r + (lane >> 5)];
                wgt[r] = row_w[buf][8 * blk + 2 * r + (lane >> 5)];
            }
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int kc = k0 + 32 * c;
                const bool cut = ib < kc + 31;  // queries before a key
                const int limit = kc + (lane & 31) - ib;
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    float x = s[c][r] * a.sl2 - m[r / 4][r % 4];
                    if (cut) x = row_of(r, lane) < limit ? -INFINITY : x;
                    sum[c] = fmaf(exp2_fast(x), wgt[r / 4][r % 4], sum[c]);
                }
            }
        }
    });
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        const float both = sum[c] + __shfl_xor(sum[c], 32, kWave);
        const int i = k0 + 32 * c + (lane & 31);
        if (lane < 32 && i < sq.n) a.partial[((size_t)item * a.hkv + kvh) * a.total + sq.start + i] = both;
    }
}

__global__ void __launch_bounds__(kThreads) prompt_join_kernel(const Params a) {
    const int kvh = blockIdx.y, b = blockIdx.z, i = blockIdx.x * kThreads + threadIdx.x;
    if (i >= a.length) return;
    const Sequence sq = sequence(a, b);
    float sum = 0.f;
    if (i < sq.n)
        for (int head = 0; head < a.group; ++head)
            for (int j = 0; j < a.ranges; ++j)
                if (reaches(a, sq, j, i / kHeld))
                    sum += a.partial[((size_t)(head * a.ranges + j) * a.hkv + kvh) * a.total + sq.start + i];
    a.weights[b * a.w_stride_b + kvh * a.w_stride_h + i] = sum;
}

// How the work is cut.  Key splits of the first pass: enough workgroups for two
// a CU where few queries count.  Ranges of the second: of at least 1024 queries.
struct Plan {
    int64_t rows, key_range, key_splits, row_range, ranges;
};

Plan make_plan(int64_t batch, int64_t hq, int64_t hkv, int64_t max_seqlen, int64_t last) {
    Plan p;
    p.rows = std::min(last, max_seqlen);
    const int64_t groups = ((p.rows + kCols - 1) / kCols * (hq / hkv) + kWaves - 1) / kWaves;
    const int64_t most = (max_seqlen + 255) / 256;  // ranges of at least 256 keys
    const int64_t want = std::max<int64_t>(1, std::min(most, 512 / std::max<int64_t>(1, groups * hkv * batch)));
    p.key_range = ((max_seqlen + want - 1) / want + kTile - 1) / kTile * kTile;
    p.key_splits = (max_seqlen + p.key_range - 1) / p.key_range;
    p.row_range = 1024;
    p.ranges = (p.rows + p.row_range - 1) / p.row_range;
    return p;
}

template <int D, class T>
hipError_t launch(const PromptWeightsArgs& x) {
    const Plan plan = make_plan(x.batch, x.hq, x.hkv, x.max_seqlen, x.last);
    Params p{};
    p.q = static_cast<const uint16_t*>(x.q);
    p.k = static_cast<const uint16_t*>(x.k);
    p.cu = x.cu;
    p.weights = x.weights;
    const size_t stats = (size_t)plan.key_splits * x.hq * x.total;
    p.m = static_cast<float*>(x.workspace);
    p.l = p.m + stats;
    p.partial = p.l + stats;
    p.q_stride = x.q_stride;
    p.k_stride = x.k_stride;
    p.w_stride_b = x.w_stride_b;
    p.w_stride_h = x.w_stride_h;
    p.total = (int)x.total;
    p.hkv = (int)x.hkv;
    p.group = (int)(x.hq / x.hkv);
    p.max_seqlen = (int)std::min(x.max_seqlen, x.total);
    p.last = (int)std::min(x.last, x.max_seqlen);
    p.length = (int)x.length;
    p.key_range = (int)plan.key_range;
    p.key_splits = (int)plan.key_splits;
    p.row_range = (int)plan.row_range;
    p.ranges = (int)plan.ranges;
    p.sl2 = x.sl2;
    const auto stream = (hipStream_t)x.stream;
    const unsigned hkv = (unsigned)x.hkv, batch = (unsigned)x.batch;
    const int64_t groups = ((plan.rows + kCols - 1) / kCols * p.group + kWaves - 1) / kWaves;
    hipLaunchKernelGGL((prompt_stats_kernel<D, T>), dim3((unsigned)(groups * plan.key_splits), hkv, batch),
                       dim3(kThreads), 0, stream, p);
    hipLaunchKernelGGL((prompt_sums_kernel<D, T>),
                       dim3((unsigned)((x.max_seqlen + kHeld - 1) / kHeld), (unsigned)(p.group * plan.ranges) * hkv, batch),
                       dim3(kThreads), 0, stream, p);
    hipLaunchKernelGGL(prompt_join_kernel, dim3((unsigned)((x.length + kThreads - 1) / kThreads), hkv, batch),
                       dim3(kThreads), 0, stream, p);
    return hipGetLastError();
}

}  // namespace

size_t prompt_weights_workspace(int64_t batch, int64_t total, int64_t hq, int64_t hkv, int64_t max_seqlen,
                                int64_t last) {
    const Plan p = make_plan(batch, hq, hkv, max_seqlen, last);
    return sizeof(float) * (size_t)total * (size_t)(2 * p.key_splits * hq + hq * p.ranges);
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
    if (x.d == 128) return x.bf16 ? launch<128, bf16>(x) : launch<128, f16>(x);
    return x.bf16 ? launch<64, bf16>(x) : launch<64, f16>(x);
}

}  // namespace ak
