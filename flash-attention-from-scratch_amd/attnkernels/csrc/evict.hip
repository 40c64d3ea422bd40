// Eviction from the paged KV cache by accumulated attention weight: of every
// sequence longer than a budget, each kv head keeps its last `recent` tokens and
// the others of the largest weight, and the kept rows move to the front of the
// sequence's pages in their order.  Not in the reference, which has no cache
// upkeep.
//
// evict_select_kernel, one workgroup per (sequence, kv head), bound by latency:
// the weights as integers that order as they do, 16 of each of 1024 threads in
// registers (longer contexts are read again in each pass); a radix select from the
// top bits down finds the key of the last one kept (LDS histograms of 2048 bins,
// three passes); then the tokens above it, and those equal to it (of which the
// first are kept), are counted in order of position: a kept token's new position
// is the number of kept ones before it.  Ballots count within a wave's 64 tokens,
// one scan over the waves' counts the rest.  16 sequences of 1487-8192 tokens, 8
// heads, to 2048: 13.4 us.
//
// evict_move_kernel, bound by memory: rows of the kept tokens are read and
// written once.  In place, row i becomes what row kept[i] >= i was: a workgroup
// owns a column of up to 128 bytes of one head's rows, so that no other touches
// its bytes, reads a batch of rows, waits until all of it is read, and writes it.
// Later batches only read rows behind what is written before them, so nothing else
// has to be ordered, and the next batch is on its way meanwhile.  The same batch in
// fp16, D = 128: 55 us, 4.3 TB/s read and written (a copy reaches 4.9); both kernels
// took 145 us when positions, pages and rows of a batch were not yet asked for together.
#include <algorithm>

#include "attn_kernels.hpp"
#include "wave.hpp"

namespace ak {

namespace {

constexpr int kSelectThreads = 1024, kSelectWaves = kSelectThreads / kWave;
constexpr int kKeys = 16;                          // of a thread, 1024 positions apart
constexpr int kSegment = kSelectThreads * kKeys;   // tokens at a time
constexpr int kBins = 2048;

// Larger weights are larger keys; -0 equals 0, every NaN is the largest.
__device__ __forceinline__ uint32_t order_key(float w) {
    if (w != w) return 0xffffffffu;
    const uint32_t u = __builtin_bit_cast(uint32_t, w + 0.f);  // -0 + 0 = +0
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

struct SelectParams {
    const float* weights;
    const int* ctx_lens;
    int* new_lens;
    float* new_weights;
    int* kept;
    int64_t w_stride_b, w_stride_h;
    int hkv, length, max_tok, budget, recent;
};

__global__ void __launch_bounds__(kSelectThreads) evict_select_kernel(const SelectParams a) {
    __shared__ int hist[kBins];
    __shared__ int wave_total[kSelectWaves];
    __shared__ int counts[kKeys * kSelectWaves];  // of 64 tokens each: above the key, and equal to it in the high half
    __shared__ int found_bin, found_above, segment_total;
    const int h = blockIdx.x, b = blockIdx.y;
    const int tid = threadIdx.x, lane = tid & 63, w = uniform(tid >> 6);
    const int n = max(min(a.ctx_lens[b], a.max_tok), 0);
    const float* wt = a.weights + b * a.w_stride_b + h * a.w_stride_h;
    float* new_wt = a.new_weights + ((size_t)b * a.hkv + h) * a.length;
    int* kept = a.kept + ((size_t)b * a.hkv + h) * a.budget;
    const int m = min(n, a.budget);
    float x[kKeys];
    uint32_t key[kKeys];
    auto some = [&](int base, int j) { return base + j * kSelectThreads < n; };  // whether any thread has a j-th token
    auto load = [&](int base) {
#pragma unroll
        for (int j = 0; j < kKeys; ++j) {
            const int i = base + j * kSelectThreads + tid;
            if (some(base, j)) x[j] = wt[min(i, n - 1)];
        }
#pragma unroll
        for (int j = 0; j < kKeys; ++j)
            if (some(base, j)) key[j] = order_key(x[j]);
    };
    load(0);
    if (h == 0 && tid == 0) a.new_lens[b] = m;
    for (int i = m + tid; i < a.length; i += kSelectThreads) new_wt[i] = 0.f;
    for (int i = m + tid; i < a.budget; i += kSelectThreads) kept[i] = -1;
    if (n <= a.budget) {
        for (int base = 0; base < n; base += kSegment) {
            if (base > 0) load(base);
#pragma unroll
            for (int j = 0; j < kKeys; ++j) {
                const int i = base + j * kSelectThreads + tid;
                if (i < n) {
                    kept[i] = i;
                    new_wt[i] = x[j];
                }
            }
        }
        return;
    }
    const bool once = n <= kSegment;  // the registers hold every token
    const int old = n - a.recent, want = a.budget - a.recent;  // 0 <= want < old
    // The key of the want-th largest of the first `old` tokens: `prefix` holds
    // its top bits, `above` of the tokens have larger ones.
    uint32_t prefix = 0xffffffffu;
    int above = 0;
    if (want > 0) {
        uint32_t known = 0;  // mask of the bits found
        prefix = 0;
        constexpr int kShift[3] = {21, 10, 0}, kBits[3] = {11, 11, 10};
#pragma unroll
        for (int pass = 0; pass < 3; ++pass) {
            const int shift = kShift[pass], bins = 1 << kBits[pass];
            for (int i = tid; i < bins; i += kSelectThreads) hist[i] = 0;
            __syncthreads();
            for (int base = 0; base < old; base += kSegment) {
                if (!once) load(base);
#pragma unroll
                for (int j = 0; j < kKeys; ++j) {
                    if (!some(base, j)) break;
                    const int i = base + j * kSelectThreads + tid;
                    if (i < old && (key[j] & known) == prefix) atomicAdd(&hist[key[j] >> shift & (bins - 1)], 1);
                }
            }
            __syncthreads();
            // Bins from the largest down, two of a thread: where the count passes want.
            const int hi = bins - 1 - 2 * tid;
            const int c0 = hi >= 0 ? hist[hi] : 0, c1 = hi >= 0 ? hist[hi - 1] : 0;
            const int inc = wave_inclusive_sum(c0 + c1);
            if (lane == kWave - 1) wave_total[w] = inc;
            __syncthreads();
            int before = above + inc - c0 - c1;
#pragma unroll
            for (int v = 0; v < kSelectWaves; ++v) before += v < w ? wave_total[v] : 0;
            if (before < want && want <= before + c0) {
                found_bin = hi;
                found_above = before;
            } else if (before + c0 < want && want <= before + c0 + c1) {
                found_bin = hi - 1;
                found_above = before + c0;
            }
            __syncthreads();
            prefix |= (uint32_t)found_bin << shift;
            known |= (uint32_t)(bins - 1) << shift;
            above = found_above;
        }
    }
    const int ties = want - above;  // tokens of that very key that are kept: the first ones (none where want is 0)
    int gt_before = 0, eq_before = 0;
    for (int base = 0; base < n; base += kSegment) {
        if (!once) load(base);
        uint64_t gt[kKeys], eq[kKeys];
#pragma unroll
        for (int j = 0; j < kKeys; ++j) {
            const int i = base + j * kSelectThreads + tid;
            const uint32_t k = key[j];
            gt[j] = eq[j] = 0;
            if (!some(base, j)) {
                if (lane == 0) counts[j * kSelectWaves + w] = 0;
                continue;
            }
            gt[j] = __builtin_amdgcn_ballot_w64(i < n && (i >= old || (want > 0 && k > prefix)));
            eq[j] = __builtin_amdgcn_ballot_w64(i < old && want > 0 && k == prefix);
            if (lane == 0) counts[j * kSelectWaves + w] = __popcll(gt[j]) | __popcll(eq[j]) << 16;
        }
        __syncthreads();
        if (w == 0) {  // exclusive sums over the 256 counts, four of a lane
            int c[4], sum = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) sum += c[i] = counts[4 * lane + i];
            int before = wave_inclusive_sum(sum) - sum;
            if (lane == kWave - 1) segment_total = before + sum;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                counts[4 * lane + i] = before;
                before += c[i];
            }
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < kKeys; ++j) {
            if (!some(base, j)) break;
            const int before = counts[j * kSelectWaves + w];
            const uint64_t below = (1ull << lane) - 1;
            const int g = gt_before + (before & 0xffff) + __popcll(gt[j] & below);
            const int e = eq_before + (before >> 16) + __popcll(eq[j] & below);
            if ((gt[j] >> lane & 1) || ((eq[j] >> lane & 1) && e < ties)) {
                const int to = g + min(e, ties);
                kept[to] = base + j * kSelectThreads + tid;
                new_wt[to] = x[j];
            }
        }
        gt_before += segment_total & 0xffff;
        eq_before += segment_total >> 16;
        if (!once) __syncthreads();  // counts are read before the next segment's
    }
}

struct MoveParams {
    char* rows[4];          // K, V and their scales
    int row_bytes[4], columns[4];
    const int *tables, *new_tables, *ctx_lens, *new_lens, *kept;
    int hkv, bs, bs_shift, max_blocks, new_max_blocks, num_blocks, max_tok, budget;
    bool in_place;
};

constexpr int kMoveThreads = 256;
constexpr int kBatch = 8;       // rows that a lane has in flight
constexpr int kColumn = 128;    // bytes of a row that a workgroup moves

// U: the bytes that a lane moves at a time.  POW2: pages of a power of two of tokens.
template <class U, bool POW2>
__device__ __forceinline__ void move_rows(const MoveParams& a, char* plane, int row_bytes, int column, int b, int h) {
    const int width = min(row_bytes - column * kColumn, kColumn) / (int)sizeof(U);  // lanes of a row
    const int tid = threadIdx.x, per_pass = kMoveThreads / width;
    const int lane_row = tid / width, offset = column * kColumn + tid % width * (int)sizeof(U);
    const bool idle = lane_row >= per_pass;
    const int m = a.new_lens[b];
    if (m == 0) return;
    const int* kept = a.kept + ((size_t)b * a.hkv + h) * a.budget;
    const int* from = a.tables + (size_t)b * a.max_blocks;
    const int* to = a.new_tables + (size_t)b * a.new_max_blocks;
    char* const base = plane + offset;
    auto page_index = [&](int i) { return POW2 ? i >> a.bs_shift : i / a.bs; };
    // Rows first, first + per_pass, ... of the batch; lanes without one take the last.
    auto row = [&](int first, int j) { return min(first + j * per_pass + lane_row, m - 1); };
    int src[kBatch];  // positions of the batch to be read next
    auto positions = [&](int first) {
#pragma unroll
        for (int j = 0; j < kBatch; ++j) src[j] = kept[row(first, j)];
    };
    const int step = kBatch * per_pass;
    struct Rows {
        U x[kBatch];
        char* dst[kBatch];  // null: nothing to write
    };
    auto read = [&](Rows& r, int first) {
        int sp[kBatch], dp[kBatch];
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            sp[j] = from[page_index(src[j])];
            dp[j] = to[page_index(row(first, j))];
        }
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            const int i = row(first, j);
            const bool fine = !idle && first + j * per_pass + lane_row < m && !(a.in_place && src[j] == i) &&
                              (unsigned)sp[j] < (unsigned)a.num_blocks && (unsigned)dp[j] < (unsigned)a.num_blocks;
            auto at = [&](int page, int token) {
                return base + (((size_t)page * a.hkv + h) * a.bs + (token - page_index(token) * a.bs)) * row_bytes;
            };
            r.x[j] = U{};
            if (fine) r.x[j] = *reinterpret_cast<const U*>(at(sp[j], src[j]));
            r.dst[j] = fine ? at(dp[j], i) : nullptr;
        }
        if (first + step < m) positions(first + step);
    };
    auto write = [&](const Rows& r) {
        // Every row of the batch has been read, by all waves, before one of them is
        // written: the use of r.x waits for this wave's (but not for the next batch's).
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            if constexpr (sizeof(U) < 4) asm volatile("" ::"v"((uint32_t)r.x[j]) : "memory");
            else asm volatile("" ::"v"(r.x[j]) : "memory");
        }
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
#pragma unroll
        for (int j = 0; j < kBatch; ++j)
            if (r.dst[j]) *reinterpret_cast<U*>(r.dst[j]) = r.x[j];
    };
    // A batch is read while the one before is written: what it reads lies behind
    // all that is written by then.
    Rows p, q;
    positions(0);
    read(p, 0);
    for (int first = 0;;) {
        if ((first += step) < m) read(q, first);
        write(p);
        if (first >= m) break;
        if ((first += step) < m) read(p, first);
        write(q);
        if (first >= m) break;
    }
}

template <bool POW2>
__global__ void __launch_bounds__(kMoveThreads) evict_move_kernel(const MoveParams a) {
    const int h = blockIdx.y, b = blockIdx.z;
    if (a.in_place && min(a.ctx_lens[b], a.max_tok) <= a.budget) return;  // every row stays
    int plane = 0, column = blockIdx.x;
    while (column >= a.columns[plane]) column -= a.columns[plane++];
    const int rb = a.row_bytes[plane];
    if (rb % 16 == 0) move_rows<u32x4, POW2>(a, a.rows[plane], rb, column, b, h);
    else if (rb % 4 == 0) move_rows<uint32_t, POW2>(a, a.rows[plane], rb, column, b, h);
    else move_rows<uint8_t, POW2>(a, a.rows[plane], rb, column, b, h);
}

}  // namespace

hipError_t evict_launch(const EvictArgs& x) {
    SelectParams s{};
    s.weights = x.weights;
    s.ctx_lens = x.context_lens;
    s.new_lens = x.new_lens;
    s.new_weights = x.new_weights;
    s.kept = x.kept;
    s.w_stride_b = x.w_stride_b;
    s.w_stride_h = x.w_stride_h;
    s.hkv = (int)x.hkv;
    s.length = (int)x.length;
    s.max_tok = (int)std::min(x.length, x.max_blocks * x.bs);
    s.budget = (int)x.budget;
    s.recent = (int)x.recent;
    hipLaunchKernelGGL(evict_select_kernel, dim3((unsigned)x.hkv, (unsigned)x.batch), dim3(kSelectThreads), 0,
                       (hipStream_t)x.stream, s);
    MoveParams m{};
    int columns = 0;
    for (int i = 0; i < 4 && x.rows[i]; ++i) {
        m.rows[i] = static_cast<char*>(x.rows[i]);
        m.row_bytes[i] = (int)x.row_bytes[i];
        m.columns[i] = (m.row_bytes[i] + kColumn - 1) / kColumn;
        columns += m.columns[i];
    }
    m.tables = x.block_tables;
    m.new_tables = x.new_block_tables ? x.new_block_tables : x.block_tables;
    m.in_place = !x.new_block_tables;
    m.ctx_lens = x.context_lens;
    m.max_tok = s.max_tok;
    m.new_lens = x.new_lens;
    m.kept = x.kept;
    m.hkv = (int)x.hkv;
    m.bs = (int)x.bs;
    m.bs_shift = (x.bs & (x.bs - 1)) == 0 ? __builtin_ctzll((unsigned long long)x.bs) : -1;
    m.max_blocks = (int)x.max_blocks;
    m.new_max_blocks = (int)(x.new_block_tables ? x.new_max_blocks : x.max_blocks);
    m.num_blocks = (int)x.num_blocks;
    m.budget = (int)x.budget;
    auto* move = m.bs_shift >= 0 ? evict_move_kernel<true> : evict_move_kernel<false>;
    hipLaunchKernelGGL(move, dim3((unsigned)columns, (unsigned)x.hkv, (unsigned)x.batch), dim3(kMoveThreads), 0,
                       (hipStream_t)x.stream, m);
    return hipGetLastError();
}

}  // namespace ak
