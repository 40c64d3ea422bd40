// Decode attention (one query token per sequence) over the 4-bit paged cache
// (MXFP4, mxfp4.hpp) and, where attention weights are summed per cached token,
// over fp16 and bf16 caches too.  Not in the reference, whose decode
// (attnkernels/csrc/paged_decode.cu) reads an fp16 cache and keeps no weights.
//
//   s_t = scale q.k_t,  p = softmax(s),  o = sum_t p_t v_t      per query head
//   weights[b, kv head, t] += sum over the kv head's G query heads of p_t
//
// Memory: 2 (D/2 + D/32) bytes a token and kv head in 4 bits (136 at D = 128,
// against 512 in fp16), 8 more for the weights.  Both products run on 16x16x32 MFMAs
// with the head group padded to 16 rows, for every G up to 16: the matrix cores have
// the time, and the vector work per byte does not grow with G.
//   * A wave takes 32 tokens per iteration, two blocks of 16.  S^T = K Q^T: lane
//     (n = l%16, g = l/16) holds token n of a block and D/4 of its channels.
//     In 4 bits that is one scale group (D = 128) or half of one (D = 64), so a
//     lane's codes have one scale, and the hardware's conversions turn a dword
//     of codes into the eight values of an operand in four instructions.
//   * The lane then holds the scores of query head n for tokens 4g..4g+3 of both
//     blocks, which is P as the operand of O += P V once rounded (to q's type: half
//     a step of each weight, as in the prefill).  V's operand for column n is the
//     D/16 channels D/16 n.. of those eight tokens; v_perm pairs the tokens.
//   * Loads are of whole cache lines, and lanes trade what is not theirs.  When each
//     lane read its own channels row by row, four loads met each line of V in 4 bits:
//     the first misses, the others wait for it and hold up all behind them.  8 x 32768
//     tokens, 32 heads of 64 took 165 us so, 137 with whole lines; 16 of 512-8192
//     tokens, Hq=64, Hkv=8, fp16 (two loads a line of K) 70 and 64.
//   * The registers of a tile's K and V take the next tile's loads as soon as its
//     products have read them, so three or four workgroups fit a CU.
//   * exp2 against a reference maximum that moves only when a score exceeds it
//     by more than 8, sums in fp32.
// The splits are cut by the kernel from the context lengths, of about equal size
// over the batch, unless the caller gives a size; the last split of a (sequence,
// kv head) to finish merges them.  With weights, the scores (scale * log2 e * q.k
// in fp32) go to a workspace, and a second kernel, which knows every split's maximum
// and sum, turns them into weights while it merges the splits' outputs.
// Measured: 16 x 8192 tokens, Hq=32, Hkv=8, D=128, 4 bits: 28.7 us, 5.0 TB/s, of which
// about 8 us are the first requests and the merge; 8 x 32768, 32 heads of 64 with
// weights: 134 us, 4.2 TB/s of cache, and 26 us for the second kernel (read scores,
// read and write weights: 3.9 TB/s); 16 of 512-8192, Hq=64, Hkv=8, fp16 with weights:
// 64 us, 4.9 TB/s, and 11; one of 1000 tokens: 8.7 us, a chain of round trips (length,
// page id, K and V, partial, counter, merge).
#include <algorithm>
#include <type_traits>

#include "attn_kernels.hpp"
#include "index_math.hpp"
#include "mxfp4.hpp"


namespace ak {

namespace {

constexpr int kWaves = 4, kThreads = kWaves * kWave;
constexpr int kTile = 32;           // tokens per wave iteration
constexpr int kMaxGroup = 16;       // query heads per kv head: rows of the MFMA
constexpr int kCut = kWaves * kTile; // splits start at multiples of it
constexpr int kMinSplit = 256;       // two tiles of a wave: less would not pay for its part of the merge
constexpr float kLowest = -3.402823466e38f;

struct Params {
    const void *q, *k, *v;
    const uint8_t *k_scales, *v_scales;
    const int *block_tables, *ctx_lens;
    void* out;
    float *o_part, *m_part, *l_part, *scores, *weights;
    int32_t* counters;
    int2* cuts;            // [batch]: a sequence's first slot and its splits, for the finishing kernel
    int64_t scores_stride, w_stride_b, w_stride_h;
    int batch, hkv, group, bs, bs_shift, max_blocks, num_blocks, max_tok;
    int partition;  // tokens per split; 0: cut evenly
    int slots;      // splits of a kv head over the whole batch, at most
    float sl2;
};

__device__ __forceinline__ void coherent_store(float* p, float v) {
    __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float coherent_load(const float* p) {
    return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

__device__ __forceinline__ f32x4 coherent_load4(const float* p) {  // 8-byte aligned
    const uint64_t a = __hip_atomic_load(reinterpret_cast<const uint64_t*>(p), __ATOMIC_RELAXED,
                                         __HIP_MEMORY_SCOPE_AGENT);
    const uint64_t b = __hip_atomic_load(reinterpret_cast<const uint64_t*>(p) + 1, __ATOMIC_RELAXED,
                                         __HIP_MEMORY_SCOPE_AGENT);
    const f32x2 x = __builtin_bit_cast(f32x2, a), y = __builtin_bit_cast(f32x2, b);
    return f32x4{x[0], x[1], y[0], y[1]};
}

// How a context is cut: ns splits (at least one) of `piece` tokens, the last one
// shorter.
struct Cut {
    int ns, piece;
};
__device__ __forceinline__ int parts(int len, int size, int max_tok) {
    return max_tok < 1 << 24 ? split_count(len, size, __builtin_amdgcn_rcpf((float)size)) : (len + size - 1) / size;
}
__device__ __forceinline__ Cut cut_context(int len, int size, int max_tok) {
    const int n = max(parts(len, size, max_tok), 1);
    Cut c;
    // At least ceil(len / n), or n would not do: the approximate quotient is off by 1.5 at most, its whole part by 2.5.
    const int each = max_tok < 1 << 24 ? (int)((float)len * __builtin_amdgcn_rcpf((float)n)) + 3 : (len + n - 1) / n;
    c.piece = max((min(each, size) + kCut - 1) / kCut * kCut, kCut);
    c.ns = max(parts(len, c.piece, max_tok), 1);
    return c;
}

__device__ __forceinline__ int context(const Params& a, int b) { return max(min(a.ctx_lens[b], a.max_tok), 0); }

__device__ __forceinline__ int wave_sum(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, true);  // row_shr:1, 2, 4, 8: a row's last lane has its sum
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, true);
    return __builtin_amdgcn_readlane(x, 15) + __builtin_amdgcn_readlane(x, 31) + __builtin_amdgcn_readlane(x, 47) +
           __builtin_amdgcn_readlane(x, 63);
}

// The split that slot `slot` holds.  b < 0: none.
struct Segment {
    int b, split, ns, piece, first, ctx;  // first: the sequence's first slot
};
__device__ __forceinline__ Segment segment(const Params& a, int slot, int lane) {
    // Contexts of 64 sequences a lane each; those of the first 64 are kept.
    const int ctx0 = lane < a.batch ? context(a, lane) : 0;
    auto ctx_of = [&](int b0) { return b0 == 0 ? ctx0 : b0 + lane < a.batch ? context(a, b0 + lane) : 0; };
    // Tokens per split.  Cut evenly: the smallest of five sizes whose splits fit the
    // slots; the last one always does: sum ceil(len / size) <= sum len / size + batch.
    int size = a.partition;
    if (size == 0 && a.slots <= a.batch) size = INT32_MAX / 4 / kCut * kCut;  // a split each
    if (size == 0) {
        float total = 0.f;  // in units of 64 tokens, rounded up, so that 64 of them fit an integer
        for (int b0 = 0; b0 < a.batch; b0 += kWave) total += (float)wave_sum((ctx_of(b0) + 63) / 64) * 64.f;
        for (int spare = 0;; ++spare) {
            const float of = fmaxf((float)a.slots - (float)a.batch * 0.25f * (float)spare, 1.f);
            if (spare == 4) {
                size = max(((int)fminf(total * 1.0005f / of, 0x1p29f) + kCut) / kCut * kCut, kMinSplit);
                break;
            }
            size = max(((int)fminf(total / of, 0x1p29f) + kCut - 1) / kCut * kCut, kMinSplit);
            int count = 0;
            for (int b0 = 0; b0 < a.batch; b0 += kWave) {
                const int ns = cut_context(ctx_of(b0), size, a.max_tok).ns;
                count += wave_sum(b0 + lane < a.batch ? ns : 0);
            }
            if (count <= a.slots) break;
        }
    }
    // Every wave counts the splits of the sequences in order.
    Segment s;
    s.b = -1;
    int before = 0;
    for (int b0 = 0; b0 < a.batch; b0 += kWave) {
        const int ctx = ctx_of(b0);
        const Cut c = cut_context(ctx, size, a.max_tok);
        const int sum = wave_inclusive_sum(b0 + lane < a.batch ? c.ns : 0);
        const uint64_t here = __builtin_amdgcn_ballot_w64(before + sum > slot);
        if (here != 0) {
            const int l = __builtin_ctzll(here);
            s.b = b0 + l;
            s.ns = __builtin_amdgcn_readlane(c.ns, l);
            s.piece = __builtin_amdgcn_readlane(c.piece, l);
            s.ctx = __builtin_amdgcn_readlane(ctx, l);
            s.first = before + __builtin_amdgcn_readlane(sum, l) - s.ns;
            s.split = slot - s.first;
            return s;
        }
        before += __builtin_amdgcn_readlane(sum, kWave - 1);
    }
    return s;
}

// The kv head (x) and slot (y) of a workgroup.  Workgroups go to the eight XCDs in
// turn.  Where there are slots for all of them, the heads of a slot go to one, whose
// L2 then has the cache lines that hold several heads' scales of a page: 16 x 8192
// tokens, 8 heads of 128 30.0 -> 28.9 us, 8 x 32768, 32 heads of 64 with weights
// 657 -> 558 MB read, 157.3 -> 156.4 us.
constexpr int kXcds = 8, kManySlots = 4 * kXcds;
__device__ __forceinline__ int2 place_of(const Params& a, int i) {
    if (a.slots < kManySlots) return int2{i % a.hkv, i / a.hkv};
    const int of_xcd = i / kXcds;
    return int2{of_xcd % a.hkv, of_xcd / a.hkv * kXcds + i % kXcds};
}

// Maximum and sum of one query row over its ns splits by 16 lanes, of which this
// is j; every lane gets them.  Splits without weight (l = 0) count nothing; a row
// without any has l = 0.
__device__ __forceinline__ void merge_stats(const float* mp, const float* lp, int ns, int j, float& m, float& l) {
    float M = kLowest, L = 0.f;
    for (int s = j; s < ns; s += 16) {
        const float ls = coherent_load(lp + s), ms = coherent_load(mp + s);
        const float mn = ls == 0.f ? M : fmaxf(M, ms);
        L = L * exp2_fast(M - mn) + (ls == 0.f ? 0.f : ls * exp2_fast(ms - mn));
        M = mn;
    }
    m = M;
#pragma unroll
    for (int d = 1; d < 16; d <<= 1) m = fmaxf(m, __shfl_xor(m, d, kWave));
    l = L * exp2_fast(M - m);
#pragma unroll
    for (int d = 1; d < 16; d <<= 1) l += __shfl_xor(l, d, kWave);
}

// Output rows head0, head0 + step, ... (count of them) of a sequence and kv head
// from their ns split partials, whose first is partial `first` of row `prow` on;
// row_m and row_l: their maxima and sums.  A thread has 4 channels of a row and
// every SG-th split.
template <int D, class T>
__device__ __forceinline__ void merge_rows(const Params& a, size_t row0, size_t prow0, int first, int ns, int head0,
                                           int step, int count, const float* row_m, const float* row_l, f32x4* part,
                                           int tid) {
    constexpr int UNITS = D / 4, ROWS = kThreads / UNITS;
    int rows = 1;  // at a time: a power of two
    while (rows < ROWS && rows < count) rows *= 2;
    const int SG = ROWS / rows, u = tid % UNITS, r = tid / UNITS % rows, sg = tid / UNITS / rows;
    for (int k0 = 0; k0 < count; k0 += rows) {
        const int k = k0 + r, h = head0 + k * step;
        f32x4 o = {0.f, 0.f, 0.f, 0.f};
        if (k < count && row_l[h] != 0.f) {
            const size_t at = (prow0 + h) * a.slots + first;
            const float m = row_m[h], inv = 1.f / row_l[h];
            for (int s0 = sg; s0 < ns; s0 += 4 * SG) {
                float ms[4], ls[4];
                f32x4 os[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {  // the loads of four splits together
                    const size_t from = at + min(s0 + i * SG, ns - 1);
                    ls[i] = s0 + i * SG < ns ? coherent_load(a.l_part + from) : 0.f;
                    ms[i] = coherent_load(a.m_part + from);
                    os[i] = coherent_load4(a.o_part + from * D + u * 4);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (ls[i] != 0.f) {
                        const float w = ls[i] * exp2_fast(ms[i] - m) * inv;
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[e] += w * os[i][e];
                    }
            }
        }
        if (SG > 1) {
            __syncthreads();  // the rows before may still be read
            part[tid] = o;
            __syncthreads();
            if (sg == 0)
                for (int i = 1; i < SG; ++i) o += part[tid + i * UNITS * rows];
        }
        if (sg == 0 && k < count) {
            uint32_t* dst = static_cast<uint32_t*>(a.out) + ((row0 + h) * D + u * 4) / 2;
            dst[0] = Half<T>::pack(o[0], o[1]);
            dst[1] = Half<T>::pack(o[2], o[3]);
        }
    }
}

// A register with x in its low bits and anything above.
__device__ __forceinline__ uint32_t loose(uint32_t x) { return x; }
__device__ __forceinline__ uint32_t loose(uint16_t x) {
    typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
    u16x2 y;
    y[0] = x;
    return __builtin_bit_cast(uint32_t, y);
}

template <int D, class T, bool MX>
struct Tile {
    static constexpr int KW = MX ? D / 32 : D / 8;    // dwords of K per block: a quarter row
    static constexpr int VW = MX ? D / 32 : D / 8;    // dwords of V per block: 4 bits, a quarter row; else D/16 channels of four
    // The two-byte words of D = 64 stay two bytes until they are used: widened
    // where they are loaded, the compiler would wait for them there.
    typedef std::conditional_t<MX && D == 64, uint16_t, uint32_t> word_t;
    uint32_t k[2][KW], v[2][VW];
    word_t ks[2];                     // a row's scales: 4 or 2 bytes
    uint32_t vs[2][MX ? D / 32 : 1];  // four rows' scales
};

template <int N>
__device__ __forceinline__ void load_words(uint32_t* to, const void* from) {
    typedef uint32_t vec __attribute__((ext_vector_type(N)));
    const vec y = __builtin_nontemporal_load(static_cast<const vec*>(from));
#pragma unroll
    for (int i = 0; i < N; ++i) to[i] = y[i];
}

// Lane j of a quad has token j's codes, a part for each of the four lanes (a dword
// in D = 128, half of one in D = 64); it gets its own part of all four tokens.
template <int D>
__device__ __forceinline__ void own_codes(const uint32_t (&in)[D / 32], uint32_t (&out)[D / 32], int lane) {
    if constexpr (D == 128) {
#pragma unroll
        for (int i = 0; i < 4; ++i) out[i] = in[i];
        transpose_quad(out[0], out[1], out[2], out[3], lane);
    } else {
        const bool odd = lane & 1, high = lane & 2;
        const uint32_t mine = odd ? 0x03020706u : 0x05040100u;  // (other's, own): halves of (token 0, token 1)
        const uint32_t pair[2] = {select(high, across2(in[1]), in[0]), select(high, in[1], across2(in[0]))};
#pragma unroll
        for (int i = 0; i < 2; ++i) out[i] = __builtin_amdgcn_perm(across1(pair[i]), pair[i], mine);
    }
}

template <int D, class T, bool MX, bool WEIGHTS>
__global__ void __launch_bounds__(kThreads, 3) decode_mx_kernel(const Params a) {
    using Tl = Tile<D, T, MX>;
    constexpr int DPL = D / 16;             // channels of a V row per lane = products per tile
    constexpr int KS = D / 32;              // products of S^T per block
    constexpr int KROW = MX ? D / 2 : 2 * D;  // bytes
    constexpr float kShift = 7.f, kPMax = 32768.f;
    __shared__ float red_acc[kWaves][kMaxGroup][D];
    __shared__ float red_m[kWaves][kMaxGroup], red_l[kWaves][kMaxGroup];
    __shared__ int last;

    const int2 place = place_of(a, blockIdx.x);
    const int kvh = place.x;
    const int G = a.group, hq = a.hkv * G;
    const int tid = threadIdx.x, lane = tid & 63, w = uniform(tid >> 6);
    const int n = lane & 15, g = lane >> 4;
    const Segment sg = segment(a, place.y, lane);
    if (sg.b < 0) return;
    const int b = sg.b, start = sg.split * sg.piece, end = min(sg.ctx, start + sg.piece);
    const size_t row0 = (size_t)b * hq + (size_t)kvh * G;
    const bool direct = !WEIGHTS && sg.ns == 1;
    if (a.cuts && sg.split == 0 && kvh == 0 && tid == 0) a.cuts[b] = int2{sg.first, sg.ns};
    if (start >= end) {  // an empty context
        if (direct)
            for (int i = tid; i < G * D / 2; i += kThreads) static_cast<uint32_t*>(a.out)[row0 * (D / 2) + i] = 0;
        return;
    }
    const int* bt = a.block_tables + (size_t)b * a.max_blocks;
    const int stride = kWaves * kTile;
    int t = start + w * kTile;

    // Q^T: head n (zeros past the group), the channels that the lane's K holds.
    u32x4 qf[KS];
#pragma unroll
    for (int i = 0; i < KS; ++i) {
        qf[i] = u32x4{0, 0, 0, 0};
        if (n < G) {
            const int ch = MX ? (D / 4) * g + 8 * i : 64 * (i / 2) + 16 * g + 8 * (i % 2);
            qf[i] = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(a.q) + (row0 + n) * D + ch);
        }
    }

    // What a lane loads of a block's rows: byte offsets from the block's first
    // row.  Of the scales it loads a row's (4 or 2 bytes) and shifts its group's.
    constexpr int SROW = D / 32;
    typedef typename Tl::word_t word_t;
    // One load reads whole cache lines of 128 bytes (a second one that meets a line on
    // its way waits for it); where those are not of the lane's own rows, lanes trade.
    // K in 16 bits: of each line of rows n & ~1 and n | 1 the 16 bytes 2g + n % 2; lanes
    // n and n ^ 1 trade.  V in 16 bits: D/16 channels of rows 4g .. 4g + 3.  V in 4 bits:
    // a quarter of row 4g + n % 4; the four lanes of a quad trade.
    constexpr int KE = MX ? 1 : 2;  // rows that a lane loads of K
    const uint32_t k_in = MX ? KROW / 4 * g : 32 * g + 16 * (n & 1), k_off = (MX ? n : n & ~1) * KROW + k_in;
    const uint32_t v_in = MX ? n / 4 * (KROW / 4) : KROW / 16 * n, v_off = (4 * g + (MX ? n % 4 : 0)) * KROW + v_in;
    // Right rotations that put the lane's scale where a float's exponent is: the
    // conversions read nothing else of it.
    const uint32_t k_turn = g / (4 / SROW) * 8 + 9, v_turn = n / (16 / SROW) * 8 + 9;
    auto load_k = [&](Tl& x, int blk, int e, const char* p) {
        if constexpr (MX) {
            load_words<Tl::KW>(x.k[blk], p);
        } else {
#pragma unroll
            for (int line = 0; line < KS / 2; ++line) load_words<4>(x.k[blk] + 4 * (2 * line + e), p + 128 * line);
        }
    };
    auto load_v = [&](Tl& x, int blk, int r, const char* p) {  // in 4 bits r is 0
        load_words<MX ? Tl::VW : Tl::VW / 4>(x.v[blk] + r * (Tl::VW / 4), p);
    };
    auto group_scale = [](uint32_t word, uint32_t turn) {
        return __builtin_bit_cast(float, __builtin_amdgcn_alignbit(word, word, turn));
    };
    // A tile each of whose two blocks is in one page: K's or V's loads at scalar
    // bases, pa and pb the pages.
    auto load_whole = [&](Tl& x, int tile, int pa, int pb, auto what) {
        constexpr bool V = decltype(what)::value;
        const char* cache = static_cast<const char*>(V ? a.v : a.k);
        const uint8_t* scales = V ? a.v_scales : a.k_scales;
#pragma unroll
        for (int blk = 0; blk < 2; ++blk) {
            const size_t row = ((size_t)(blk ? pb : pa) * a.hkv + kvh) * a.bs + ((tile + 16 * blk) & (a.bs - 1));
            const char* base = cache + row * KROW;
            const uint8_t* sbase = scales + row * SROW;
            if constexpr (V) {
#pragma unroll
                for (int r = 0; r < (MX ? 1 : 4); ++r) load_v(x, blk, r, base + v_off + r * KROW);
                if constexpr (MX) {
                    typedef uint32_t vec __attribute__((ext_vector_type(SROW)));
                    const vec y = *reinterpret_cast<const vec*>(sbase + (uint32_t)(4 * g * SROW));
#pragma unroll
                    for (int i = 0; i < SROW; ++i) x.vs[blk][i] = y[i];
                }
            } else {
#pragma unroll
                for (int e = 0; e < KE; ++e) load_k(x, blk, e, base + k_off + e * KROW);
                if constexpr (MX) x.ks[blk] = *reinterpret_cast<const word_t*>(sbase + (uint32_t)(n * SROW));
            }
        }
    };
    // Any tile: every token's row on its own; rows that are not read are zeros.
    // Returns a bit for each token that is read.
    auto load_rows = [&](Tl& x, int tile) {
        const int tok = tile + (lane & 31);
        const int index = a.bs_shift >= 0 ? tok >> a.bs_shift : tok / a.bs, in = tok - index * a.bs;
        const int pid = tok < end ? bt[index] : -1;
        const uint32_t valid = (uint32_t)__builtin_amdgcn_ballot_w64((unsigned)pid < (unsigned)a.num_blocks);
        auto row_of = [&](int i) {
            const int p = __shfl(pid, i, kWave), o = __shfl(in, i, kWave);
            return ((size_t)p * a.hkv + kvh) * a.bs + o;
        };
#pragma unroll
        for (int blk = 0; blk < 2; ++blk) {
            x.ks[blk] = 0;
#pragma unroll
            for (int i = 0; i < Tl::KW; ++i) x.k[blk][i] = 0;
#pragma unroll
            for (int e = 0; e < KE; ++e) {
                const int i = 16 * blk + (MX ? n : (n & ~1) + e);
                const size_t kr = row_of(i);
                if (!(valid >> i & 1)) continue;
                load_k(x, blk, e, static_cast<const char*>(a.k) + kr * KROW + k_in);
                if constexpr (MX) x.ks[blk] = *reinterpret_cast<const word_t*>(a.k_scales + kr * SROW);
            }
#pragma unroll
            for (int i = 0; i < Tl::VW; ++i) x.v[blk][i] = 0;
            if constexpr (MX) {
                const int i = 16 * blk + 4 * g + n % 4;
                const size_t vr = row_of(i);
                if (valid >> i & 1) load_v(x, blk, 0, static_cast<const char*>(a.v) + vr * KROW + v_in);
#pragma unroll
                for (int i = 0; i < SROW; ++i) x.vs[blk][i] = 0;
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int i = 16 * blk + 4 * g + r;
                const size_t vr = row_of(i);
                if (!(valid >> i & 1)) continue;
                if constexpr (MX)
                    x.vs[blk][r * SROW / 4] |= (uint32_t)*reinterpret_cast<const word_t*>(a.v_scales + vr * SROW)
                                               << r * SROW % 4 * 8;
                else
                    load_v(x, blk, r, static_cast<const char*>(a.v) + vr * KROW + v_in);
            }
        }
        return valid;
    };

    // Reference maximum of head n (the same in its four lanes), this lane's
    // share of l, and acc[j][r]: head 4g + r, channel DPL n + j.
    float m_own = kLowest, l_own = 0.f;
    f32x4 acc[DPL];
#pragma unroll
    for (int j = 0; j < DPL; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
    float* scores = WEIGHTS ? a.scores + (row0 + (n < G ? n : 0)) * a.scores_stride + 4 * g : nullptr;

    // One tile.  after_k and after_v run once the registers of its K, its V are free.
    auto step = [&](const Tl& x, int tile, uint32_t valid, auto masked, auto after_k, auto after_v) {
        f32x4 s[2];
#pragma unroll
        for (int blk = 0; blk < 2; ++blk) {
            s[blk] = f32x4{0.f, 0.f, 0.f, 0.f};
            if constexpr (MX) {
#pragma unroll
                for (int i = 0; i < KS; ++i)
                    s[blk] = Half<T>::mfma(mx_decode8<T>(x.k[blk][i], group_scale(loose(x.ks[blk]), k_turn)), qf[i], s[blk]);
            } else {
#pragma unroll
                for (int i = 0; i < KS; i += 2) {
                    u32x4 own[2];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint32_t even = x.k[blk][4 * i + j], odd = x.k[blk][4 * i + 4 + j];
                        own[0][j] = select(n & 1, across1(odd), even);
                        own[1][j] = select(n & 1, odd, across1(even));
                    }
                    s[blk] = Half<T>::mfma(own[0], qf[i], s[blk]);
                    s[blk] = Half<T>::mfma(own[1], qf[i + 1], s[blk]);
                }
            }
        }
        __builtin_amdgcn_sched_barrier(0);  // the next loads take these registers
        after_k();
#pragma unroll
        for (int blk = 0; blk < 2; ++blk)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                s[blk][r] *= a.sl2;
                if (decltype(masked)::value) s[blk][r] = valid >> (16 * blk + 4 * g + r) & 1 ? s[blk][r] : -INFINITY;
            }
        if constexpr (WEIGHTS) {
            if (n < G) {
                *reinterpret_cast<f32x4*>(scores + tile) = s[0];
                *reinterpret_cast<f32x4*>(scores + tile + 16) = s[1];
            }
        }
        float p[8], bias = kShift - m_own;
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = exp2_fast(s[i / 4][i % 4] + bias);
        const float top = fmaxf(fmaxf(fmaxf(p[0], p[1]), fmaxf(p[2], p[3])), fmaxf(fmaxf(p[4], p[5]), fmaxf(p[6], p[7])));
        if (__builtin_amdgcn_ballot_w64(top > kPMax)) {
            // Move the reference maximum of every head to its running maximum.
            float mx = m_own;
#pragma unroll
            for (int i = 0; i < 8; ++i) mx = fmaxf(mx, s[i / 4][i % 4]);
            mx = fmaxf(mx, __shfl_xor(mx, 16, kWave));
            mx = fmaxf(mx, __shfl_xor(mx, 32, kWave));
            const float alpha = exp2_fast(m_own - mx);
            l_own *= alpha;
            m_own = mx;
#pragma unroll
            for (int r = 0; r < 4; ++r) {  // accumulator row r is head 4g + r
                const float al = __shfl(alpha, 4 * g + r, kWave);
#pragma unroll
                for (int j = 0; j < DPL; ++j) acc[j][r] *= al;
            }
            bias = kShift - m_own;
#pragma unroll
            for (int i = 0; i < 8; ++i) p[i] = exp2_fast(s[i / 4][i % 4] + bias);
        }
        l_own += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
        u32x4 pf;
#pragma unroll
        for (int i = 0; i < 4; ++i) pf[i] = Half<T>::pack(p[2 * i], p[2 * i + 1]);
        // V: channels 2c, 2c + 1 of the lane's eight tokens, paired by tokens.
        auto channels = [&](const uint32_t (&v)[8], int c) {
#pragma unroll
            for (int o = 0; o < 2; ++o) {
                const uint32_t sel = o ? 0x07060302u : 0x05040100u;
                u32x4 f;
#pragma unroll
                for (int i = 0; i < 4; ++i) f[i] = __builtin_amdgcn_perm(v[2 * i + 1], v[2 * i], sel);
                acc[2 * c + o] = Half<T>::mfma(pf, f, acc[2 * c + o]);
            }
        };
        if constexpr (MX) {
            float sc[8];
            uint32_t v[8];
            // Tokens 4g + r of each block, D/16 channels: a dword, in D = 64 two tokens in one.
            uint32_t codes[2][Tl::VW];
#pragma unroll
            for (int blk = 0; blk < 2; ++blk) own_codes<D>(x.v[blk], codes[blk], lane);
#pragma unroll
            for (int i = 0; i < 8; ++i) sc[i] = group_scale(x.vs[i / 4][i % 4 * SROW / 4], v_turn + i % 4 * SROW % 4 * 8);
            auto decode = [&](auto byte) {  // channels 2 byte, 2 byte + 1
                constexpr int C = decltype(byte)::value;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const uint32_t word = codes[i / 4][i % 4 * SROW / 4];
                    if (D == 64 && i % 2) v[i] = Half<T>::template decode<(C + 2) % 4>(word, sc[i]);
                    else v[i] = Half<T>::template decode<C>(word, sc[i]);
                }
                channels(v, C);
            };
            decode(std::integral_constant<int, 0>{});
            decode(std::integral_constant<int, 1>{});
            if constexpr (D == 128) {
                decode(std::integral_constant<int, 2>{});
                decode(std::integral_constant<int, 3>{});
            }
        } else {
#pragma unroll
            for (int c = 0; c < DPL / 2; ++c) {
                uint32_t v[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = x.v[i / 4][i % 4 * (DPL / 2) + c];
                channels(v, c);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
        after_v();
    };

    // The wave's tiles.  While they are whole, a tile's K and V registers take the
    // next tile's loads as soon as they are free, and page ids come a tile earlier.
    Tl x;
    bool loaded = false;
    if (a.bs_shift >= 4) {
        // By scalar loads (nothing writes the table while the kernel runs): a vector
        // load's wait would be one for all the rows in flight.
        typedef const __attribute__((address_space(4))) int* scalar_ptr;
        const scalar_ptr table = (scalar_ptr)(uintptr_t)bt;
        auto page = [&](int tok) { return tok < end ? table[tok >> a.bs_shift] : -1; };
        auto whole = [&](int tile, int pa, int pb) {
            return tile + kTile <= end && (unsigned)pa < (unsigned)a.num_blocks && (unsigned)pb < (unsigned)a.num_blocks;
        };
        int pa = page(t), pb = page(t + 16);
        if (whole(t, pa, pb)) {
            load_whole(x, t, pa, pb, std::false_type{});
            load_whole(x, t, pa, pb, std::true_type{});
            loaded = true;
            pa = page(t + stride);
            pb = page(t + stride + 16);
            while (whole(t + stride, pa, pb)) {
                const int tn = t + stride, na = page(tn + stride), nb = page(tn + stride + 16);
                step(x, t, 0xffffffffu, std::false_type{}, [&] { load_whole(x, tn, pa, pb, std::false_type{}); },
                     [&] { load_whole(x, tn, pa, pb, std::true_type{}); });
                pa = na;
                pb = nb;
                t = tn;
            }
        }
    }
    // The last whole tile, and the rest: the context's end, pages outside the pool
    // or of other sizes.
    for (; t < end; t += stride) {
        const uint32_t valid = loaded ? 0xffffffffu : load_rows(x, t);
        loaded = false;
        step(x, t, valid, std::true_type{}, [] {}, [] {});
    }

    // Merge: l over the four lanes of each head, then the waves through LDS.
    l_own += __shfl_xor(l_own, 16, kWave);
    l_own += __shfl_xor(l_own, 32, kWave);
    if (g == 0) {
        red_m[w][n] = m_own;
        red_l[w][n] = l_own;
    }
#pragma unroll
    for (int r = 0; r < 4; ++r)
        if (4 * g + r < G) {
#pragma unroll
            for (int j = 0; j < DPL; ++j) red_acc[w][4 * g + r][DPL * n + j] = acc[j][r];
        }
    __syncthreads();
    for (int i = tid; i < G * D / 2; i += kThreads) {
        const int h = i / (D / 2), d = 2 * (i % (D / 2));
        float M = red_m[0][h];
#pragma unroll
        for (int v = 1; v < kWaves; ++v) M = fmaxf(M, red_m[v][h]);
        float L = 0.f, o0 = 0.f, o1 = 0.f;
#pragma unroll
        for (int v = 0; v < kWaves; ++v) {
            const float wv = exp2_fast(red_m[v][h] - M);
            L += red_l[v][h] * wv;
            o0 += red_acc[v][h][d] * wv;
            o1 += red_acc[v][h][d + 1] * wv;
        }
        const float inv = L == 0.f ? 0.f : 1.f / L;  // no token that counts: zeros
        const size_t slot = (size_t)(kvh * G + h) * a.slots + sg.first + sg.split;
        if (direct) {
            static_cast<uint32_t*>(a.out)[((row0 + h) * D + d) / 2] = Half<T>::pack(o0 * inv, o1 * inv);
        } else {
            coherent_store(a.o_part + slot * D + d, o0 * inv);
            coherent_store(a.o_part + slot * D + d + 1, o1 * inv);
            if (d == 0) {
                coherent_store(a.m_part + slot, M);
                coherent_store(a.l_part + slot, L * (1.f / 128.f));  // without the shift of P
            }
        }
    }
    if (WEIGHTS || direct || !a.counters) return;
    // The last split of the sequence and kv head to finish merges them all.
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    int32_t* cnt = a.counters + (size_t)b * a.hkv + kvh;
    if (tid == 0) last = __hip_atomic_fetch_add(cnt, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == sg.ns - 1;
    __syncthreads();
    if (!last) return;
    if (tid == 0) __hip_atomic_store(cnt, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    const size_t prow0 = (size_t)kvh * G;
    if (const int h = tid / 16; h < G) {
        float m, l;
        const size_t at = (prow0 + h) * a.slots + sg.first;
        merge_stats(a.m_part + at, a.l_part + at, sg.ns, tid % 16, m, l);
        red_m[0][h] = m;
        red_l[0][h] = l;
    }
    __syncthreads();
    merge_rows<D, T>(a, row0, prow0, sg.first, sg.ns, 0, 1, G, red_m[0], red_l[0],
                     reinterpret_cast<f32x4*>(&red_acc[0][0][0]), tid);
}

// After decode_mx_kernel: merges the splits' outputs, and turns the scores into
// weights, TOKENS of a thread (0: no weights).  Workgroup c of a (kv head,
// sequence) has its tokens from c * kThreads * TOKENS on and the heads h with
// h % (workgroups with tokens) == c.  Bound by memory: G + 2 floats a token.
template <int D, class T, int TOKENS>
__global__ void __launch_bounds__(kThreads) decode_mx_finish_kernel(const Params a) {
    constexpr int N = TOKENS > 0 ? TOKENS : 1;
    typedef float scores_t __attribute__((ext_vector_type(N)));
    __shared__ float row_m[kMaxGroup], row_l[kMaxGroup];
    __shared__ f32x4 part[kThreads];
    const int c = blockIdx.x, kvh = blockIdx.y, b = blockIdx.z;
    const int G = a.group, hq = a.hkv * G;
    const int tid = threadIdx.x;
    const int ctx = context(a, b);
    const int active = TOKENS > 0 ? max((ctx + kThreads * N - 1) / (kThreads * N), 1) : gridDim.x;
    if (c >= active) return;
    const int2 cut = a.cuts[b];
    const int first = cut.x, ns = ctx > 0 ? cut.y : 0;
    if (TOKENS == 0 && cut.y == 1) return;  // written by decode_mx_kernel
    const size_t row0 = (size_t)b * hq + (size_t)kvh * G, prow0 = (size_t)kvh * G;
    // The first heads' scores are on their way while the splits are merged.
    constexpr int HEADS = 8;
    const int t = (c * kThreads + tid) * N;
    scores_t s[HEADS];
    auto load = [&](int h0) {
        const float* scores = a.scores + row0 * a.scores_stride + t;
#pragma unroll
        for (int i = 0; i < HEADS; ++i)
            if (h0 + i < G && t < ctx)
                s[i] = *reinterpret_cast<const scores_t*>(scores + (size_t)(h0 + i) * a.scores_stride);
    };
    float* wt = a.weights + b * a.w_stride_b + kvh * a.w_stride_h + t;
    float old[N];
    if constexpr (TOKENS > 0) {
        load(0);
#pragma unroll
        for (int j = 0; j < N; ++j) old[j] = t + j < ctx ? wt[j] : 0.f;
    }
    if (const int h = tid / 16; h < G) {
        float m, l;
        const size_t at = (prow0 + h) * a.slots + first;
        merge_stats(a.m_part + at, a.l_part + at, ns, tid % 16, m, l);
        row_m[h] = m;
        row_l[h] = l;
    }
    __syncthreads();
    if constexpr (TOKENS > 0) {
        float sum[N] = {};
        for (int h0 = 0; h0 < G; h0 += HEADS) {
            if (h0 > 0) load(h0);
#pragma unroll
            for (int i = 0; i < HEADS; ++i)
                if (h0 + i < G && row_l[h0 + i] != 0.f) {
                    const float inv = 1.f / row_l[h0 + i], m = row_m[h0 + i];
#pragma unroll
                    for (int j = 0; j < N; ++j) sum[j] += exp2_fast(s[i][j] - m) * inv;
                }
        }
#pragma unroll
        for (int j = 0; j < N; ++j)
            if (t + j < ctx) wt[j] = old[j] + sum[j];
    }
    if (c < G)
        merge_rows<D, T>(a, row0, prow0, first, ns, c, active, (G - c + active - 1) / active, row_m, row_l, part, tid);
}

template <int D, class T, bool MX, bool WEIGHTS>
hipError_t launch(const DecodeMxArgs& x) {
    Params p{};
    p.q = x.q;
    p.k = x.k;
    p.v = x.v;
    p.k_scales = static_cast<const uint8_t*>(x.k_scales);
    p.v_scales = static_cast<const uint8_t*>(x.v_scales);
    p.block_tables = x.block_tables;
    p.ctx_lens = x.context_lens;
    p.out = x.out;
    p.o_part = x.o_part;
    p.m_part = x.m_part;
    p.l_part = x.l_part;
    p.scores = x.scores;
    p.weights = x.weights;
    p.scores_stride = x.scores_stride;
    p.w_stride_b = x.w_stride_b;
    p.w_stride_h = x.w_stride_h;
    p.hkv = (int)x.hkv;
    p.group = (int)(x.hq / x.hkv);
    p.bs = (int)x.bs;
    p.bs_shift = (x.bs & (x.bs - 1)) == 0 ? __builtin_ctzll((unsigned long long)x.bs) : -1;
    p.max_blocks = (int)x.max_blocks;
    p.num_blocks = (int)x.num_blocks;
    p.max_tok = (int)std::min(x.max_blocks * x.bs, x.max_ctx);
    p.batch = (int)x.batch;
    p.partition = (int)x.partition;
    p.slots = (int)x.slots;
    p.sl2 = x.sl2;
    p.counters = WEIGHTS ? nullptr : x.counters;
    const bool finish = WEIGHTS || (x.slots > x.batch && !x.counters);
    p.cuts = finish ? static_cast<int2*>(x.cuts) : nullptr;
    const int64_t slots = x.slots < kManySlots ? x.slots : (x.slots + kXcds - 1) / kXcds * kXcds;
    hipLaunchKernelGGL((decode_mx_kernel<D, T, MX, WEIGHTS>), dim3((unsigned)(x.hkv * slots)), dim3(kThreads), 0,
                       (hipStream_t)x.stream, p);
    if (!finish) return hipGetLastError();
    auto run = [&](auto* kernel, int64_t workgroups) {
        hipLaunchKernelGGL(kernel, dim3((unsigned)workgroups, (unsigned)x.hkv, (unsigned)x.batch), dim3(kThreads), 0,
                           (hipStream_t)x.stream, p);
    };
    if constexpr (WEIGHTS) {
        // Four tokens of a thread where that leaves eight workgroups a CU.
        const int64_t wide = (p.max_tok + 4 * kThreads - 1) / (4 * kThreads);
        if (wide * x.hkv * x.batch >= 2048) run(decode_mx_finish_kernel<D, T, 4>, wide);
        else run(decode_mx_finish_kernel<D, T, 2>, (p.max_tok + 2 * kThreads - 1) / (2 * kThreads));
    } else {
        run(decode_mx_finish_kernel<D, T, 0>, p.group);
    }
    return hipGetLastError();
}

template <int D, class T>
hipError_t launch_typed(const DecodeMxArgs& x) {
    if (!x.k_scales) return launch<D, T, false, true>(x);  // without weights a full-precision cache is paged_decode's
    return x.weights ? launch<D, T, true, true>(x) : launch<D, T, true, false>(x);
}

}  // namespace

// Splits of a kv head over the whole batch.  Cut evenly: a workgroup for every 272
// KB of K and V at max_ctx, but one to four for each of the 256 CUs; at least a
// quarter more than sequences (that the longest are cut), none of less than
// kMinSplit tokens, and no more than 64 a sequence on average for one workgroup to
// merge.  Measured at 256 / 512 / 768 / 1024 / 1280 workgroups, us: 16 x 8192 tokens,
// Hq=32, Hkv=8, 4 bits 35.2 / 30.5 / 32.3 / 32.7 / -; 4 x 4096 12.3 / 14.9 / 14.8; 8 x
// 32768, 32 heads, D=64, 4 bits with weights - / 172 / 159 / 156 / 173; 16 of 512-8192,
// Hq=64, Hkv=8, fp16 with weights 85.2 / 82.7 / 81.6 / 80.4 / 81.7.
// row_bytes: of a token's K and V for one kv head.
int64_t decode_mx_slots(int64_t batch, int64_t hkv, int64_t max_ctx, int64_t partition, int64_t row_bytes) {
    if (partition > 0) return batch * ((max_ctx + partition - 1) / partition);
    constexpr int64_t kBytes = 272 << 10, kMost = 64;
    const double bytes = (double)batch * (double)hkv * (double)max_ctx * (double)row_bytes;
    const int64_t workgroups = (int64_t)std::min(1024.0, std::max(256.0, bytes / kBytes));
    const int64_t chunks = std::min(kMost, (max_ctx + kMinSplit - 1) / kMinSplit);
    return std::min(batch * chunks, std::max((workgroups + hkv - 1) / hkv, batch + (batch + 3) / 4));
}

hipError_t decode_mx_launch(const DecodeMxArgs& x) {
    if (x.d == 128) return x.bf16 ? launch_typed<128, bf16>(x) : launch_typed<128, f16>(x);
    return x.bf16 ? launch_typed<64, bf16>(x) : launch_typed<64, f16>(x);
}

}  // namespace ak
