// C-ABI entry points (include/attnkernels.h): argument validation, the
// reference's error wording, and dispatch to the HIP launchers.  Validation
// runs before any HIP call, so a rejected call never touches the GPU.
#include <algorithm>
#include <climits>
#include <cmath>
#include <cstdio>
#include <string>

#include "attn_kernels.hpp"
#include "attnkernels.h"

static_assert(AK_PAGED_DECODE_NOALLOC_MAX_BYTES == ak::kDecodeScratchBytes,
              "the header states the static scratch size");

namespace {

thread_local std::string g_last_error;
constexpr double kLog2e = 1.4426950408889634;
constexpr int64_t kChunk = 256;  // partitions are multiples of it (paged_decode.cu:37)

int fail(int code, const std::string& msg) {
    g_last_error = msg;
    return code;
}

int ok() {
    g_last_error.clear();
    return AK_OK;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

int hip_status(hipError_t e, const char* who) {
    if (e == hipSuccess) return ok();
    return fail(AK_ERR_HIP, std::string(who) + ": HIP error: " + hipGetErrorString(e));
}

// Shared by every prefill entry point.  kv_heads divides heads (GQA); cu is
// null for the dense [B, H, N, D] layout, else the packed layout's sequence
// starts with total_rows rows in q/k/v and seq_len the longest sequence.
int prefill(const char* who, const void* q, const void* k, const void* v, void* o, int64_t batch,
            int64_t heads, int64_t kv_heads, int64_t seq_len, int64_t head_dim, int causal, double scale,
            const int32_t* cu, int64_t total_rows, void* stream) {
    if (batch < 0 || heads < 0 || seq_len < 0 || kv_heads < 0 || total_rows < 0)
        return fail(AK_ERR_INVALID_ARGUMENT, std::string(who) + ": negative size");
    if (kv_heads == 0 ? heads != 0 : heads % kv_heads != 0)
        return fail(AK_ERR_INVALID_ARGUMENT, std::string(who) + ": num_heads must be a multiple of num_kv_heads");
    if (batch * heads * seq_len == 0 || (cu && total_rows == 0)) return ok();  // nothing to compute
    if (!q || !k || !v || !o) return fail(AK_ERR_INVALID_ARGUMENT, std::string(who) + ": null pointer");
    if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(o))
        return fail(AK_ERR_INVALID_ARGUMENT, std::string(who) + ": pointers must be 16-byte aligned");
    // Workgroups = query-tile units (128 or 256 rows, causal: pairs) x batch x
    // heads: an int, counted here for the smaller tile.
    const int64_t tiles = (seq_len + 127) / 128, units = causal ? (tiles + 1) / 2 : tiles;
    if (seq_len > INT_MAX / 2 || total_rows > INT_MAX / 2 || batch * heads > INT_MAX / units)
        return fail(AK_ERR_INVALID_ARGUMENT, std::string(who) + ": size out of range");
    ak::PrefillArgs a{};
    a.q = q;
    a.k = k;
    a.v = v;
    a.o = o;
    a.bh = batch * heads;
    a.hq = heads;
    a.hkv = kv_heads;
    a.cu = cu;
    a.total_rows = total_rows;
    a.n = cu ? std::min(seq_len, total_rows) : seq_len;  // packed: no sequence has more rows than there are
    a.d = (int)head_dim;
    a.causal = causal != 0;
    // |scale| * log2(e), kept >= 1e-30 so that masked scores (-inf) still map to
    // 2^-inf = 0; below that every score rounds to the same weight anyway.
    a.sl2 = (float)std::fmax(std::fabs(scale) * kLog2e, 1e-30);
    a.qflip = std::signbit(scale) && scale != 0.0 ? 0x80008000u : 0u;
    a.stream = stream;
    return hip_status(ak::prefill_launch(a), who);
}

// Validation shared by both decode entry points, in the reference's order
// (paged_decode.cu:260-262, 275), and the launch arguments except the split
// partials.  batch == 0 passes validation with nothing to launch.
int decode_args(const void* q, const void* k_cache, const void* v_cache, const int32_t* block_tables,
                const int32_t* context_lens, void* out, int64_t batch, int64_t num_heads, int64_t num_kv_heads,
                int64_t head_dim, int64_t num_blocks, int64_t block_size, int64_t max_blocks_per_seq,
                int64_t max_context_len, double scale, int64_t partition, void* stream, ak::DecodeArgs& a) {
    if (num_kv_heads <= 0 || num_heads <= 0 || num_heads % num_kv_heads != 0)
        return fail(AK_ERR_INVALID_ARGUMENT, "num_heads must be a multiple of num_kv_heads");
    if (partition <= 0 || partition % kChunk != 0)
        return fail(AK_ERR_INVALID_ARGUMENT, "partition size must be a positive multiple of 256");
    const int64_t G = num_heads / num_kv_heads;
    if ((head_dim != 64 && head_dim != 128) || (G != 1 && G != 2 && G != 4 && G != 8))
        return fail(AK_ERR_UNSUPPORTED,
                    "paged_decode: head_dim must be 64/128 and num_heads/num_kv_heads in {1,2,4,8}");
    if (batch < 0 || num_blocks < 0 || block_size <= 0 || max_blocks_per_seq < 0)
        return fail(AK_ERR_INVALID_ARGUMENT, "paged_decode: invalid size");
    if (batch == 0) return ok();
    if (max_context_len < 1)
        return fail(AK_ERR_INVALID_ARGUMENT, "paged_decode: max_context_len must be >= 1");
    if (max_blocks_per_seq < 1 || num_blocks < 1)
        return fail(AK_ERR_INVALID_ARGUMENT, "paged_decode: empty block table or cache");
    if (!q || !k_cache || !v_cache || !block_tables || !context_lens || !out)
        return fail(AK_ERR_INVALID_ARGUMENT, "paged_decode: null pointer");
    if (!aligned16(q) || !aligned16(k_cache) || !aligned16(v_cache) || !aligned16(out))
        return fail(AK_ERR_INVALID_ARGUMENT, "paged_decode: q, caches and out must be 16-byte aligned");
    if ((reinterpret_cast<uintptr_t>(block_tables) & 3u) || (reinterpret_cast<uintptr_t>(context_lens) & 3u))
        return fail(AK_ERR_INVALID_ARGUMENT, "paged_decode: int32 arrays must be 4-byte aligned");
    if (max_context_len > INT_MAX - partition || partition > INT_MAX || num_blocks > INT_MAX ||
        max_blocks_per_seq * block_size > INT_MAX || batch > 65535 || num_kv_heads > 65535)
        return fail(AK_ERR_INVALID_ARGUMENT, "paged_decode: size out of range");
    const int64_t splits = (max_context_len + partition - 1) / partition;
    if (splits > 65535) return fail(AK_ERR_INVALID_ARGUMENT, "paged_decode: more than 65535 splits");
    a.q = q;
    a.k_cache = k_cache;
    a.v_cache = v_cache;
    a.block_tables = block_tables;
    a.context_lens = context_lens;
    a.out = out;
    a.batch = batch;
    a.hq = num_heads;
    a.hkv = num_kv_heads;
    a.d = head_dim;
    a.num_blocks = num_blocks;
    a.bs = block_size;
    a.max_blocks = max_blocks_per_seq;
    a.partition = partition;
    a.num_splits = splits;
    a.sl2 = (float)(scale * kLog2e);
    a.stream = stream;
    return ok();
}

// Bytes of the split partials in one fp32 buffer: o [B, Hq, S, D], m [B, Hq, S], l [B, Hq, S].
size_t partials_bytes(int64_t batch, int64_t num_heads, int64_t splits, int64_t head_dim) {
    return (size_t)batch * (size_t)num_heads * (size_t)splits * (size_t)(head_dim + 2) * sizeof(float);
}

void set_partials(ak::DecodeArgs& a, void* buf, size_t rows) {
    float* ws = static_cast<float*>(buf);
    a.o_part = ws;
    a.m_part = ws + rows * (size_t)a.d;
    a.l_part = a.m_part + rows;
}

// The balanced launch for these sizes; no workers: none (invalid sizes, or
// fixed splits serve).  The most tokens it reads of a sequence are those fixed
// splits of `partition` tokens would read.
ak::BalancedPlan balanced_plan(int64_t batch, int64_t num_heads, int64_t num_kv_heads, int64_t head_dim,
                               int64_t max_context_len, int64_t partition) {
    if (num_kv_heads <= 0 || num_heads <= 0 || num_heads % num_kv_heads != 0 || head_dim <= 0 || partition <= 0 ||
        max_context_len < 1 || max_context_len > INT_MAX - partition)
        return {0, 0};
    const int64_t cap = (max_context_len + partition - 1) / partition * partition;
    return ak::decode_balanced_plan(batch, num_heads, num_kv_heads, head_dim, max_context_len, cap);
}

size_t round16(size_t x) { return (x + 15) / 16 * 16; }

// A row of scores of ak_paged_decode_mx_*: whole tiles of 64 tokens.
int64_t scores_row(int64_t max_context_len) { return (max_context_len + 63) / 64 * 64; }

// Whether a [batch, kv heads, length] array of these strides has no two rows in one place.
int weights_rows(const char* who, int64_t batch, int64_t kv_heads, int64_t stride_b, int64_t stride_h, int64_t length) {
    const bool b = batch > 1, h = kv_heads > 1;
    constexpr int64_t kMost = INT64_MAX >> 17;  // products below fit
    bool fine = (!b || (stride_b >= length && stride_b < kMost)) && (!h || (stride_h >= length && stride_h < kMost));
    if (fine && b && h && length > 0)
        fine = stride_b >= stride_h ? stride_b >= stride_h * (kv_heads - 1) + length
                                    : stride_h >= stride_b * (batch - 1) + length;
    return fine ? AK_OK : fail(AK_ERR_INVALID_ARGUMENT, std::string(who) + ": rows of weights overlap");
}

// Validation shared by the 4-bit cache's writer and reader, and their launch arguments but the rows.
int mx_rows(const char* name, const void* key, const void* value, void* k_cache, void* k_scales, void* v_cache,
            void* v_scales, const int64_t* slots, int64_t num_tokens, int64_t num_kv_heads, int64_t head_dim,
            int64_t num_blocks, int64_t block_size, int bf16, void* stream, ak::CacheMxArgs& a) {
    const std::string who(name);
    if (num_tokens < 0 || num_kv_heads <= 0 || num_blocks < 0 || block_size <= 0)
        return fail(AK_ERR_INVALID_ARGUMENT, who + ": invalid size");
    if (head_dim <= 0 || head_dim % 32 != 0 || head_dim > 512)
        return fail(AK_ERR_UNSUPPORTED, who + ": head_dim must be a multiple of 32 up to 512");
    if (num_tokens > 0 && (!key || !value || !slots || (num_blocks > 0 && (!k_cache || !k_scales || !v_cache || !v_scales))))
        return fail(AK_ERR_INVALID_ARGUMENT, who + ": null pointer");
    if (!aligned16(key) || !aligned16(value) || !aligned16(k_cache) || !aligned16(v_cache) ||
        (reinterpret_cast<uintptr_t>(slots) & 7u))
        return fail(AK_ERR_INVALID_ARGUMENT, who + ": tensors must be 16-byte aligned");
    // Grid: x = token (< 2^31), y = groups of 256 lanes of one token (<= 65535).
    if (num_kv_heads > 65535LL * 256 / (head_dim / 8) || block_size > INT_MAX ||
        num_blocks > INT64_MAX / block_size / (num_kv_heads * head_dim) || num_tokens > INT_MAX)
        return fail(AK_ERR_INVALID_ARGUMENT, who + ": size out of range");
    a.k_codes = k_cache;
    a.k_scales = k_scales;
    a.v_codes = v_cache;
    a.v_scales = v_scales;
    a.slots = slots;
    a.num_tokens = num_tokens;
    a.hkv = num_kv_heads;
    a.head_dim = head_dim;
    a.num_blocks = num_blocks;
    a.bs = block_size;
    a.bf16 = bf16 != 0;
    a.stream = stream;
    return ok();
}

// Decode over MXFP4 caches (k_scales set) or 16-bit ones with weights.
int decode_mx(const char* name, const void* q, const void* k_cache, const void* k_scales, const void* v_cache,
              const void* v_scales, const int32_t* block_tables, const int32_t* context_lens, void* out,
              float* weights, int64_t w_stride_b, int64_t w_stride_h, int64_t w_length, int64_t batch,
              int64_t num_heads, int64_t num_kv_heads, int64_t head_dim, int64_t num_blocks, int64_t block_size,
              int64_t max_blocks_per_seq, int64_t max_context_len, double scale, int64_t partition, int bf16,
              void* workspace, size_t workspace_bytes, int32_t* counters, int64_t counters_len, void* stream) {
    const std::string who(name);
    if (num_kv_heads <= 0 || num_heads <= 0 || num_heads % num_kv_heads != 0)
        return fail(AK_ERR_INVALID_ARGUMENT, who + ": num_heads must be a multiple of num_kv_heads");
    if (partition < 0 || partition % kChunk != 0)
        return fail(AK_ERR_INVALID_ARGUMENT, who + ": partition size must be 0 or a positive multiple of 256");
    if ((head_dim != 64 && head_dim != 128) || num_heads / num_kv_heads > 16)
        return fail(AK_ERR_UNSUPPORTED, who + ": head_dim must be 64 or 128 and num_heads / num_kv_heads at most 16");
    if (batch < 0 || num_blocks < 0 || block_size <= 0 || max_blocks_per_seq < 0)
        return fail(AK_ERR_INVALID_ARGUMENT, who + ": invalid size");
    if (batch == 0) return ok();
    if (max_context_len < 1) return fail(AK_ERR_INVALID_ARGUMENT, who + ": max_context_len must be >= 1");
    if (max_blocks_per_seq < 1 || num_blocks < 1)
        return fail(AK_ERR_INVALID_ARGUMENT, who + ": empty block table or cache");
    if (!q || !k_cache || !v_cache || !block_tables || !context_lens || !out)
        return fail(AK_ERR_INVALID_ARGUMENT, who + ": null pointer");
    if (!aligned16(q) || !aligned16(k_cache) || !aligned16(v_cache) || !aligned16(out))
        return fail(AK_ERR_INVALID_ARGUMENT, who + ": q, caches and out must be 16-byte aligned");
    if (!aligned16(k_scales) || !aligned16(v_scales))
        return fail(AK_ERR_INVALID_ARGUMENT, who + ": scales must be 16-byte aligned");
    for (const void* p : {(const void*)block_tables, (const void*)context_lens, (const void*)weights,
                          (const void*)counters})
        if (reinterpret_cast<uintptr_t>(p) & 3u)
            return fail(AK_ERR_INVALID_ARGUMENT, who + ": int32 and float arrays must be 4-byte aligned");
    if (max_context_len > INT_MAX / 2 || partition > INT_MAX / 2 || num_blocks > INT_MAX ||
        max_blocks_per_seq > INT_MAX / 2 / block_size || batch > 65535 || num_kv_heads > 65535)
        return fail(AK_ERR_INVALID_ARGUMENT, who + ": size out of range");
    const int64_t row_bytes = k_scales ? head_dim * 17 / 16 : 4 * head_dim;
    const int64_t slots = ak::decode_mx_slots(batch, num_kv_heads, max_context_len, partition, row_bytes);
    if (slots > INT_MAX / num_kv_heads - 8) return fail(AK_ERR_INVALID_ARGUMENT, who + ": too many splits");
    if (weights) {
        if (w_length < max_context_len)
            return fail(AK_ERR_INVALID_ARGUMENT, who + ": weights are shorter than max_context_len");
        if (const int rc = weights_rows(name, batch, num_kv_heads, w_stride_b, w_stride_h, w_length)) return rc;
    }
    if (counters && counters_len < batch * num_kv_heads)
        return fail(AK_ERR_INVALID_ARGUMENT, who + ": counters must be an int32 array of at least batch * num_kv_heads "
                                                   "elements");
    const size_t need = ak_paged_decode_mx_workspace_size(batch, num_heads, num_kv_heads, head_dim, max_context_len,
                                                          partition, weights != nullptr);
    if (need > 0 && (!workspace || workspace_bytes < need))
        return fail(AK_ERR_WORKSPACE, who + ": workspace of " + std::to_string(need) + " bytes required, got " +
                                          std::to_string(workspace_bytes));
    if (!aligned16(workspace)) return fail(AK_ERR_INVALID_ARGUMENT, who + ": workspace must be 16-byte aligned");
    ak::DecodeMxArgs a{};
    a.q = q;
    a.k = k_cache;
    a.v = v_cache;
    a.k_scales = k_scales;
    a.v_scales = v_scales;
    a.block_tables = block_tables;
    a.context_lens = context_lens;
    a.out = out;
    a.weights = weights;
    a.counters = counters;
    a.batch = batch;
    a.hq = num_heads;
    a.hkv = num_kv_heads;
    a.d = head_dim;
    a.num_blocks = num_blocks;
    a.bs = block_size;
    a.max_blocks = max_blocks_per_seq;
    a.max_ctx = max_context_len;
    a.partition = partition;
    a.slots = slots;
    a.w_stride_b = w_stride_b;
    a.w_stride_h = w_stride_h;
    a.bf16 = bf16 != 0;
    a.sl2 = (float)(scale * kLog2e);
    a.stream = stream;
    if (need > 0) {
        const size_t rows = (size_t)(num_heads * slots);
        a.o_part = static_cast<float*>(workspace);
        a.m_part = a.o_part + rows * (size_t)head_dim;
        a.l_part = a.m_part + rows;
        size_t at = (partials_bytes(1, num_heads, slots, head_dim) + 7) / 8 * 8;
        a.cuts = static_cast<char*>(workspace) + at;
        if (weights) {
            at = round16(at + (size_t)batch * 2 * sizeof(int32_t));
            a.scores = reinterpret_cast<float*>(static_cast<char*>(workspace) + at);
            a.scores_stride = scores_row(max_context_len);
        }
    }
    return hip_status(ak::decode_mx_launch(a), name);
}

}  // namespace

extern "C" {

const char* ak_last_error(void) { return g_last_error.c_str(); }

int ak_abi_version(void) { return 101; }

int ak_naive_attention(const void* q, const void* k, const void* v, void* o, int64_t batch,
                       int64_t heads, int64_t seq_len, int64_t head_dim, int causal, double scale,
                       void* stream) {
    if (head_dim != 64 && head_dim != 128)
        return fail(AK_ERR_UNSUPPORTED, "naive_attention: head_dim must be 64 or 128");
    return prefill("naive_attention", q, k, v, o, batch, heads, heads, seq_len, head_dim, causal, scale, nullptr, 0,
                   stream);
}

int ak_flash_simt(const void* q, const void* k, const void* v, void* o, int64_t batch, int64_t heads,
                  int64_t seq_len, int64_t head_dim, int causal, double scale, void* stream) {
    if (head_dim != 64 && head_dim != 128)
        return fail(AK_ERR_UNSUPPORTED, "flash_simt: head_dim must be 64 or 128");
    return prefill("flash_simt", q, k, v, o, batch, heads, heads, seq_len, head_dim, causal, scale, nullptr, 0,
                   stream);
}

int ak_flash_wmma(const void* q, const void* k, const void* v, void* o, int64_t batch, int64_t heads,
                  int64_t seq_len, int64_t head_dim, int causal, double scale, int64_t block_n,
                  void* stream) {
    if ((head_dim != 64 && head_dim != 128) || (block_n != 32 && block_n != 64))
        return fail(AK_ERR_UNSUPPORTED, "flash_wmma: head_dim must be 64 or 128 and block_n 32 or 64");
    return prefill("flash_wmma", q, k, v, o, batch, heads, heads, seq_len, head_dim, causal, scale, nullptr, 0,
                   stream);
}

int ak_prefill_gqa(const void* q, const void* k, const void* v, void* o, int64_t batch, int64_t num_heads,
                   int64_t num_kv_heads, int64_t seq_len, int64_t head_dim, int causal, double scale,
                   void* stream) {
    if (head_dim != 64 && head_dim != 128)
        return fail(AK_ERR_UNSUPPORTED, "prefill_gqa: head_dim must be 64 or 128");
    return prefill("prefill_gqa", q, k, v, o, batch, num_heads, num_kv_heads, seq_len, head_dim, causal, scale,
                   nullptr, 0, stream);
}

int ak_prefill_varlen(const void* q, const void* k, const void* v, void* o, const int32_t* cu_seqlens,
                      int64_t batch, int64_t total_rows, int64_t num_heads, int64_t num_kv_heads,
                      int64_t max_seqlen, int64_t head_dim, int causal, double scale, void* stream) {
    if (head_dim != 64 && head_dim != 128)
        return fail(AK_ERR_UNSUPPORTED, "prefill_varlen: head_dim must be 64 or 128");
    if (batch > 0 && (!cu_seqlens || (reinterpret_cast<uintptr_t>(cu_seqlens) & 3u)))
        return fail(AK_ERR_INVALID_ARGUMENT, "prefill_varlen: cu_seqlens must be a 4-byte aligned int32 array");
    return prefill("prefill_varlen", q, k, v, o, batch, num_heads, num_kv_heads, max_seqlen, head_dim, causal,
                   scale, batch > 0 ? cu_seqlens : nullptr, total_rows, stream);
}

size_t ak_paged_decode_workspace_size(int64_t batch, int64_t num_heads, int64_t head_dim,
                                      int64_t max_context_len, int64_t partition) {
    if (batch < 0 || num_heads < 0 || head_dim <= 0 || max_context_len < 1 || partition <= 0) return 0;
    const int64_t splits = (max_context_len + partition - 1) / partition;
    if (splits <= 1) return 0;
    return partials_bytes(batch, num_heads, splits, head_dim);
}

int ak_paged_decode(const void* q, const void* k_cache, const void* v_cache, const int32_t* block_tables,
                    const int32_t* context_lens, void* out, int64_t batch, int64_t num_heads,
                    int64_t num_kv_heads, int64_t head_dim, int64_t num_blocks, int64_t block_size,
                    int64_t max_blocks_per_seq, int64_t max_context_len, double scale, int64_t partition,
                    void* workspace, size_t workspace_bytes, void* stream) {
    return ak_paged_decode_fused(q, k_cache, v_cache, block_tables, context_lens, out, batch, num_heads,
                                 num_kv_heads, head_dim, num_blocks, block_size, max_blocks_per_seq,
                                 max_context_len, scale, partition, workspace, workspace_bytes, nullptr, 0, stream);
}

int ak_paged_decode_fused(const void* q, const void* k_cache, const void* v_cache, const int32_t* block_tables,
                          const int32_t* context_lens, void* out, int64_t batch, int64_t num_heads,
                          int64_t num_kv_heads, int64_t head_dim, int64_t num_blocks, int64_t block_size,
                          int64_t max_blocks_per_seq, int64_t max_context_len, double scale, int64_t partition,
                          void* workspace, size_t workspace_bytes, int32_t* counters, int64_t counters_len,
                          void* stream) {
    ak::DecodeArgs a{};
    const int rc = decode_args(q, k_cache, v_cache, block_tables, context_lens, out, batch, num_heads, num_kv_heads,
                               head_dim, num_blocks, block_size, max_blocks_per_seq, max_context_len, scale,
                               partition, stream, a);
    if (rc != AK_OK || batch == 0) return rc;
    if (counters && (counters_len < batch * num_kv_heads || (reinterpret_cast<uintptr_t>(counters) & 3u)))
        return fail(AK_ERR_INVALID_ARGUMENT, "paged_decode: counters must be a 4-byte aligned int32 array of at least "
                                             "batch * num_kv_heads = " + std::to_string(batch * num_kv_heads) +
                                             " elements");
    if (a.num_splits > 1) {
        const size_t need = ak_paged_decode_workspace_size(batch, num_heads, head_dim, max_context_len, partition);
        if (!workspace || workspace_bytes < need)
            return fail(AK_ERR_WORKSPACE, "paged_decode: workspace of " + std::to_string(need) +
                                              " bytes required, got " + std::to_string(workspace_bytes));
        if (!aligned16(workspace))
            return fail(AK_ERR_INVALID_ARGUMENT, "paged_decode: workspace must be 16-byte aligned");
        set_partials(a, workspace, (size_t)(a.batch * a.hq * a.num_splits));
        a.counters = counters;
    }
    return hip_status(ak::decode_launch(a), "paged_decode");
}

size_t ak_paged_decode_balanced_workspace_size(int64_t batch, int64_t num_heads, int64_t num_kv_heads,
                                               int64_t head_dim, int64_t max_context_len, int64_t partition) {
    const int64_t workers =
        balanced_plan(batch, num_heads, num_kv_heads, head_dim, max_context_len, partition).workers;
    return partials_bytes(1, num_heads, workers, head_dim);
}

int ak_paged_decode_balanced(const void* q, const void* k_cache, const void* v_cache, const int32_t* block_tables,
                             const int32_t* context_lens, void* out, int64_t batch, int64_t num_heads,
                             int64_t num_kv_heads, int64_t head_dim, int64_t num_blocks, int64_t block_size,
                             int64_t max_blocks_per_seq, int64_t max_context_len, double scale, int64_t partition,
                             void* workspace, size_t workspace_bytes, int32_t* counters, int64_t counters_len,
                             void* stream) {
    ak::DecodeArgs a{};
    const int rc = decode_args(q, k_cache, v_cache, block_tables, context_lens, out, batch, num_heads, num_kv_heads,
                               head_dim, num_blocks, block_size, max_blocks_per_seq, max_context_len, scale,
                               partition, stream, a);
    if (rc != AK_OK || batch == 0) return rc;
    const auto [workers, order] =
        balanced_plan(batch, num_heads, num_kv_heads, head_dim, max_context_len, partition);
    if (workers == 0)
        return fail(AK_ERR_UNSUPPORTED, "paged_decode_balanced: fixed splits serve these sizes "
                                        "(ak_paged_decode_balanced_workspace_size is 0)");
    if (!counters || counters_len < batch * num_kv_heads || (reinterpret_cast<uintptr_t>(counters) & 3u))
        return fail(AK_ERR_INVALID_ARGUMENT, "paged_decode_balanced: counters must be a 4-byte aligned int32 array of "
                                             "at least batch * num_kv_heads = " +
                                                 std::to_string(batch * num_kv_heads) + " elements");
    const size_t need = partials_bytes(1, num_heads, workers, head_dim);
    if (!workspace || workspace_bytes < need)
        return fail(AK_ERR_WORKSPACE, "paged_decode_balanced: workspace of " + std::to_string(need) +
                                          " bytes required, got " + std::to_string(workspace_bytes));
    if (!aligned16(workspace))
        return fail(AK_ERR_INVALID_ARGUMENT, "paged_decode_balanced: workspace must be 16-byte aligned");
    a.token_cap = std::min(a.num_splits * a.partition, a.max_blocks * a.bs);
    a.balanced = true;
    a.order = order;
    a.partition = ak::kBalancedMinSplit;
    a.num_splits = workers;
    a.counters = counters;
    set_partials(a, workspace, (size_t)a.hq * (size_t)workers);
    return hip_status(ak::decode_launch(a), "paged_decode_balanced");
}

int ak_paged_decode_noalloc(const void* q, const void* k_cache, const void* v_cache, const int32_t* block_tables,
                            const int32_t* context_lens, void* out, int64_t batch, int64_t num_heads,
                            int64_t num_kv_heads, int64_t head_dim, int64_t num_blocks, int64_t block_size,
                            int64_t max_blocks_per_seq, int64_t max_context_len, double scale, int64_t partition,
                            void* stream) {
    ak::DecodeArgs a{};
    const int rc = decode_args(q, k_cache, v_cache, block_tables, context_lens, out, batch, num_heads, num_kv_heads,
                               head_dim, num_blocks, block_size, max_blocks_per_seq, max_context_len, scale,
                               partition, stream, a);
    if (rc != AK_OK || batch == 0) return rc;
    if (a.num_splits > 1) {
        const size_t need = partials_bytes(batch, num_heads, a.num_splits, head_dim);
        if (need > ak::kDecodeScratchBytes)
            return fail(AK_ERR_WORKSPACE, "paged_decode_noalloc: the split partials need " + std::to_string(need) +
                                              " bytes, more than the static scratch of " +
                                              std::to_string(ak::kDecodeScratchBytes) +
                                              " bytes; use a larger partition or ak_paged_decode with a workspace");
        // The scratch array of the current device: the stream must run there.
        if (stream) {
            int cur = 0;
            hipDevice_t sdev = 0;
            hipError_t e = hipGetDevice(&cur);
            if (e == hipSuccess) e = hipStreamGetDevice((hipStream_t)stream, &sdev);
            if (e != hipSuccess) return hip_status(e, "paged_decode_noalloc");
            if ((int)sdev != cur)
                return fail(AK_ERR_INVALID_ARGUMENT,
                            "paged_decode_noalloc: the stream must belong to the current device");
        }
        void* ws = nullptr;
        int32_t* counters = nullptr;
        const hipError_t e = ak::decode_scratch(&ws, &counters);
        if (e != hipSuccess) return hip_status(e, "paged_decode_noalloc");
        set_partials(a, ws, (size_t)(a.batch * a.hq * a.num_splits));
        // counters for every (sequence, kv head) fit the static array: merged in
        // the decode kernel; otherwise by the reduce kernel
        if ((size_t)batch * (size_t)num_kv_heads <= ak::kDecodeScratchCounters) a.counters = counters;
    }
    return hip_status(ak::decode_launch(a), "paged_decode_noalloc");
}

int ak_reshape_and_cache(const void* key, const void* value, void* k_cache, void* v_cache,
                         const int64_t* slot_mapping, int64_t num_tokens, int64_t num_kv_heads,
                         int64_t head_dim, int64_t num_blocks, int64_t block_size, int64_t key_stride,
                         int64_t value_stride, void* stream) {
    if (num_tokens < 0 || num_kv_heads <= 0 || num_blocks < 0 || block_size <= 0)
        return fail(AK_ERR_INVALID_ARGUMENT, "reshape_and_cache: invalid size");
    if (head_dim <= 0 || head_dim % 8 != 0 || head_dim > 512)
        return fail(AK_ERR_UNSUPPORTED, "reshape_and_cache: head_dim must be a multiple of 8 up to 512");
    const int64_t row = num_kv_heads * head_dim;
    if (key_stride < row || value_stride < row || key_stride % 8 || value_stride % 8)
        return fail(AK_ERR_INVALID_ARGUMENT,
                    "reshape_and_cache: token strides must be multiples of 8 and >= num_kv_heads * head_dim");
    if (num_tokens == 0 || num_blocks == 0) return ok();  // nothing to write, or no slot in range
    if (!key || !value || !k_cache || !v_cache || !slot_mapping)
        return fail(AK_ERR_INVALID_ARGUMENT, "reshape_and_cache: null pointer");
    if (!aligned16(key) || !aligned16(value) || !aligned16(k_cache) || !aligned16(v_cache) ||
        (reinterpret_cast<uintptr_t>(slot_mapping) & 7u))
        return fail(AK_ERR_INVALID_ARGUMENT, "reshape_and_cache: tensors must be 16-byte aligned");
    // Grid: x = token (< 2^31), y = groups of 256 chunks of one token (<= 65535).
    if (num_kv_heads * (head_dim / 8) > 65535LL * 256 || block_size > INT_MAX ||
        num_blocks > INT64_MAX / block_size / row || num_tokens > INT_MAX)
        return fail(AK_ERR_INVALID_ARGUMENT, "reshape_and_cache: size out of range");
    ak::CacheWriteArgs a{};
    a.key = key;
    a.value = value;
    a.k_cache = k_cache;
    a.v_cache = v_cache;
    a.slots = slot_mapping;
    a.num_tokens = num_tokens;
    a.hkv = num_kv_heads;
    a.head_dim = head_dim;
    a.num_blocks = num_blocks;
    a.bs = block_size;
    a.key_stride = key_stride;
    a.value_stride = value_stride;
    a.stream = stream;
    return hip_status(ak::cache_write_launch(a), "reshape_and_cache");
}

int ak_stream_checksum(const void* src, size_t bytes, uint32_t* out, void* stream) {
    if (bytes % 16 != 0) return fail(AK_ERR_INVALID_ARGUMENT, "stream_checksum: bytes must be a multiple of 16");
    if (bytes > 0 && (!src || !aligned16(src)))
        return fail(AK_ERR_INVALID_ARGUMENT, "stream_checksum: src must be a 16-byte aligned device pointer");
    if (!out || (reinterpret_cast<uintptr_t>(out) & 3u))
        return fail(AK_ERR_INVALID_ARGUMENT, "stream_checksum: out must be a 4-byte aligned device pointer");
    return hip_status(ak::stream_checksum_launch(src, bytes, out, stream), "stream_checksum");
}

int ak_reshape_and_cache_mxfp4(const void* key, const void* value, void* k_cache, void* k_scales, void* v_cache,
                               void* v_scales, const int64_t* slot_mapping, int64_t num_tokens, int64_t num_kv_heads,
                               int64_t head_dim, int64_t num_blocks, int64_t block_size, int64_t key_stride,
                               int64_t value_stride, int bf16, void* stream) {
    const char* who = "reshape_and_cache_mxfp4";
    const int64_t row = num_kv_heads * head_dim;
    ak::CacheMxArgs a{};
    const int rc = mx_rows(who, key, value, k_cache, k_scales, v_cache, v_scales, slot_mapping, num_tokens,
                           num_kv_heads, head_dim, num_blocks, block_size, bf16, stream, a);
    if (rc != AK_OK) return rc;
    if (key_stride < row || value_stride < row || key_stride % 8 || value_stride % 8)
        return fail(AK_ERR_INVALID_ARGUMENT, "reshape_and_cache_mxfp4: token strides must be multiples of 8 and >= "
                                             "num_kv_heads * head_dim");
    if (num_tokens == 0 || num_blocks == 0) return ok();  // nothing to write, or no slot in range
    a.key = key;
    a.value = value;
    a.key_stride = key_stride;
    a.value_stride = value_stride;
    return hip_status(ak::cache_write_mxfp4_launch(a), who);
}

int ak_gather_cache_mxfp4(const void* k_cache, const void* k_scales, const void* v_cache, const void* v_scales,
                          const int64_t* slot_mapping, void* key, void* value, int64_t num_tokens,
                          int64_t num_kv_heads, int64_t head_dim, int64_t num_blocks, int64_t block_size, int bf16,
                          void* stream) {
    const char* who = "gather_cache_mxfp4";
    ak::CacheMxArgs a{};
    const int rc = mx_rows(who, key, value, const_cast<void*>(k_cache), const_cast<void*>(k_scales),
                           const_cast<void*>(v_cache), const_cast<void*>(v_scales), slot_mapping, num_tokens,
                           num_kv_heads, head_dim, num_blocks, block_size, bf16, stream, a);
    if (rc != AK_OK || num_tokens == 0) return rc;
    a.key_out = key;
    a.value_out = value;
    return hip_status(ak::cache_read_mxfp4_launch(a), who);
}

size_t ak_paged_decode_mx_workspace_size(int64_t batch, int64_t num_heads, int64_t num_kv_heads, int64_t head_dim,
                                         int64_t max_context_len, int64_t partition, int with_weights) {
    if (batch < 1 || num_heads < 1 || num_kv_heads < 1 || head_dim <= 0 || max_context_len < 1 || partition < 0 ||
        max_context_len > INT_MAX / 2)
        return 0;
    // As for 16-bit caches, which are cut into as many splits as 4-bit ones or more.
    const int64_t slots = ak::decode_mx_slots(batch, num_kv_heads, max_context_len, partition, 4 * head_dim);
    if (slots <= batch && !with_weights) return 0;
    const size_t parts = partials_bytes(1, num_heads, slots, head_dim) + (size_t)batch * 2 * sizeof(int32_t) + 8;
    return with_weights ? round16(parts) + (size_t)batch * (size_t)num_heads * (size_t)scores_row(max_context_len) *
                                               sizeof(float)
                        : parts;
}

int ak_paged_decode_mxfp4(const void* q, const void* k_cache, const void* k_scales, const void* v_cache,
                          const void* v_scales, const int32_t* block_tables, const int32_t* context_lens, void* out,
                          float* weights, int64_t weights_stride_b, int64_t weights_stride_h, int64_t weights_length,
                          int64_t batch, int64_t num_heads, int64_t num_kv_heads, int64_t head_dim,
                          int64_t num_blocks, int64_t block_size, int64_t max_blocks_per_seq, int64_t max_context_len,
                          double scale, int64_t partition, int bf16, void* workspace, size_t workspace_bytes,
                          int32_t* counters, int64_t counters_len, void* stream) {
    const char* who = "paged_decode_mxfp4";
    if (batch > 0 && (!k_scales || !v_scales)) return fail(AK_ERR_INVALID_ARGUMENT, "paged_decode_mxfp4: null pointer");
    return decode_mx(who, q, k_cache, k_scales, v_cache, v_scales, block_tables, context_lens, out, weights,
                     weights_stride_b, weights_stride_h, weights_length, batch, num_heads, num_kv_heads, head_dim,
                     num_blocks, block_size, max_blocks_per_seq, max_context_len, scale, partition, bf16, workspace,
                     workspace_bytes, counters, counters_len, stream);
}

int ak_paged_decode_weights(const void* q, const void* k_cache, const void* v_cache, const int32_t* block_tables,
                            const int32_t* context_lens, void* out, float* weights, int64_t weights_stride_b,
                            int64_t weights_stride_h, int64_t weights_length, int64_t batch, int64_t num_heads,
                            int64_t num_kv_heads, int64_t head_dim, int64_t num_blocks, int64_t block_size,
                            int64_t max_blocks_per_seq, int64_t max_context_len, double scale, int64_t partition,
                            int bf16, void* workspace, size_t workspace_bytes, void* stream) {
    if (batch > 0 && !weights) return fail(AK_ERR_INVALID_ARGUMENT, "paged_decode_weights: null pointer");
    return decode_mx("paged_decode_weights", q, k_cache, nullptr, v_cache, nullptr, block_tables, context_lens, out,
                     weights, weights_stride_b, weights_stride_h, weights_length, batch, num_heads, num_kv_heads,
                     head_dim, num_blocks, block_size, max_blocks_per_seq, max_context_len, scale, partition, bf16,
                     workspace, workspace_bytes, nullptr, 0, stream);
}

size_t ak_prompt_weights_workspace_size(int64_t batch, int64_t total_rows, int64_t num_heads, int64_t num_kv_heads,
                                        int64_t head_dim, int64_t max_seqlen, int64_t last) {
    if (batch <= 0 || total_rows <= 0 || num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads ||
        head_dim <= 0 || max_seqlen <= 0 || last <= 0 || total_rows > INT_MAX / 2)
        return 0;
    const int64_t longest = std::min(max_seqlen, total_rows);
    return ak::prompt_weights_workspace(batch, total_rows, num_heads, num_kv_heads, longest, std::min(last, longest));
}

int ak_prompt_weights(const void* q, const void* k, const int32_t* cu_seqlens, float* weights,
                      int64_t weights_stride_b, int64_t weights_stride_h, int64_t weights_length, int64_t batch,
                      int64_t total_rows, int64_t num_heads, int64_t num_kv_heads, int64_t head_dim, int64_t q_stride,
                      int64_t k_stride, int64_t max_seqlen, int64_t last, double scale, int bf16, void* workspace,
                      size_t workspace_bytes, void* stream) {
    const char* who = "prompt_weights";
    if (num_kv_heads <= 0 || num_heads <= 0 || num_heads % num_kv_heads != 0)
        return fail(AK_ERR_INVALID_ARGUMENT, "prompt_weights: num_heads must be a multiple of num_kv_heads");
    if (head_dim != 64 && head_dim != 128)
        return fail(AK_ERR_UNSUPPORTED, "prompt_weights: head_dim must be 64 or 128");
    if (batch < 0 || total_rows < 0 || max_seqlen < 0 || weights_length < 0 || last < 1)
        return fail(AK_ERR_INVALID_ARGUMENT, "prompt_weights: invalid size");
    const int64_t longest = std::min(max_seqlen, total_rows);
    if (longest > weights_length)
        return fail(AK_ERR_INVALID_ARGUMENT, "prompt_weights: weights are shorter than max_seqlen");
    if (batch == 0 || weights_length == 0) return ok();  // nothing to write
    if (!weights || !cu_seqlens || (total_rows > 0 && (!q || !k)))
        return fail(AK_ERR_INVALID_ARGUMENT, "prompt_weights: null pointer");
    if (!aligned16(q) || !aligned16(k) || (reinterpret_cast<uintptr_t>(weights) & 3u) ||
        (reinterpret_cast<uintptr_t>(cu_seqlens) & 3u))
        return fail(AK_ERR_INVALID_ARGUMENT, "prompt_weights: q and k must be 16-byte, int32 and float arrays 4-byte "
                                             "aligned");
    if (q_stride % 8 || k_stride % 8 || q_stride < num_heads * head_dim || k_stride < num_kv_heads * head_dim)
        return fail(AK_ERR_INVALID_ARGUMENT, "prompt_weights: token strides must be multiples of 8 and hold all heads");
    // Offsets inside a tile of 64 rows are 32 bits wide.
    if (q_stride > 1 << 24 || k_stride > 1 << 24 || total_rows > INT_MAX / 2 || weights_length > INT_MAX / 2 ||
        batch > 65535 || num_heads > 65535)
        return fail(AK_ERR_INVALID_ARGUMENT, "prompt_weights: size out of range");
    if (const int rc = weights_rows(who, batch, num_kv_heads, weights_stride_b, weights_stride_h, weights_length))
        return rc;
    ak::PromptWeightsArgs a{};
    const size_t need = ak_prompt_weights_workspace_size(batch, total_rows, num_heads, num_kv_heads, head_dim,
                                                         max_seqlen, last);
    if (need > 0 && (!workspace || workspace_bytes < need))
        return fail(AK_ERR_WORKSPACE, "prompt_weights: workspace of " + std::to_string(need) +
                                          " bytes required, got " + std::to_string(workspace_bytes));
    if (!aligned16(workspace))
        return fail(AK_ERR_INVALID_ARGUMENT, "prompt_weights: workspace must be 16-byte aligned");
    a.q = q;
    a.k = k;
    a.cu = cu_seqlens;
    a.weights = weights;
    a.workspace = workspace;
    a.batch = batch;
    a.total = total_rows;
    a.hq = num_heads;
    a.hkv = num_kv_heads;
    a.d = head_dim;
    a.max_seqlen = longest;
    a.last = std::min(last, std::max<int64_t>(longest, 1));
    a.length = weights_length;
    a.q_stride = q_stride;
    a.k_stride = k_stride;
    a.w_stride_b = weights_stride_b;
    a.w_stride_h = weights_stride_h;
    a.bf16 = bf16 != 0;
    // |scale| * log2(e) is kept >= 1e-30, so that masked scores (infinite) still get no
    // weight; below that every score weighs the same anyway.
    a.sl2 = (float)std::copysign(std::fmax(std::fabs(scale) * kLog2e, 1e-30), scale);
    a.stream = stream;
    if (!ak::prompt_weights_fits(a)) return fail(AK_ERR_INVALID_ARGUMENT, "prompt_weights: size out of range");
    return hip_status(ak::prompt_weights_launch(a), who);
}

int ak_evict_cache(void* k_cache, void* v_cache, int64_t row_bytes, void* k_scales, void* v_scales,
                   int64_t scale_bytes, const int32_t* block_tables, const int32_t* new_block_tables,
                   const int32_t* context_lens, const float* weights, int64_t weights_stride_b,
                   int64_t weights_stride_h, int64_t weights_length, int32_t* new_lens, float* new_weights,
                   int32_t* kept, int64_t batch, int64_t num_kv_heads, int64_t num_blocks, int64_t block_size,
                   int64_t max_blocks_per_seq, int64_t new_max_blocks, int64_t budget, int64_t recent, void* stream) {
    const char* who = "evict_cache";
    if (batch < 0 || num_kv_heads <= 0 || num_blocks < 0 || block_size <= 0 || max_blocks_per_seq < 0 ||
        weights_length < 0 || (new_block_tables && new_max_blocks < 0))
        return fail(AK_ERR_INVALID_ARGUMENT, "evict_cache: invalid size");
    if (budget < 1 || recent < 0 || recent > budget)
        return fail(AK_ERR_INVALID_ARGUMENT, "evict_cache: budget must be >= 1 and recent from 0 to budget");
    const bool scales = k_scales || v_scales || scale_bytes != 0;
    if (row_bytes < 16 || row_bytes > 1024 || row_bytes % 16 || (scales && (scale_bytes < 1 || scale_bytes > 128)))
        return fail(AK_ERR_UNSUPPORTED, "evict_cache: rows must be a multiple of 16 bytes up to 1024, scales up to 128");
    if (batch == 0) return ok();
    if (!block_tables || !context_lens || !weights || !new_lens || !new_weights || !kept || !k_cache || !v_cache ||
        (scales && (!k_scales || !v_scales)))
        return fail(AK_ERR_INVALID_ARGUMENT, "evict_cache: null pointer");
    if (!aligned16(k_cache) || !aligned16(v_cache) || !aligned16(k_scales) || !aligned16(v_scales))
        return fail(AK_ERR_INVALID_ARGUMENT, "evict_cache: caches and scales must be 16-byte aligned");
    for (const void* p : {(const void*)block_tables, (const void*)new_block_tables, (const void*)context_lens,
                          (const void*)weights, (const void*)new_lens, (const void*)new_weights, (const void*)kept})
        if (reinterpret_cast<uintptr_t>(p) & 3u)
            return fail(AK_ERR_INVALID_ARGUMENT, "evict_cache: int32 and float arrays must be 4-byte aligned");
    if (max_blocks_per_seq > INT_MAX / 2 / block_size || weights_length > INT_MAX / 2 || budget > INT_MAX / 2 ||
        num_blocks > INT_MAX || batch > 65535 || num_kv_heads > 65535)
        return fail(AK_ERR_INVALID_ARGUMENT, "evict_cache: size out of range");
    if (const int rc = weights_rows(who, batch, num_kv_heads, weights_stride_b, weights_stride_h, weights_length))
        return rc;
    const int64_t longest = std::min(weights_length, max_blocks_per_seq * block_size);
    if (new_block_tables && (new_max_blocks > INT_MAX / 2 / block_size ||
                             new_max_blocks * block_size < std::min(budget, longest)))
        return fail(AK_ERR_INVALID_ARGUMENT, "evict_cache: new_block_tables must have pages for budget tokens");
    ak::EvictArgs a{};
    a.rows[0] = k_cache;
    a.rows[1] = v_cache;
    a.rows[2] = k_scales;
    a.rows[3] = v_scales;
    a.row_bytes[0] = a.row_bytes[1] = row_bytes;
    a.row_bytes[2] = a.row_bytes[3] = scale_bytes;
    a.block_tables = block_tables;
    a.new_block_tables = new_block_tables;
    a.context_lens = context_lens;
    a.weights = weights;
    a.new_lens = new_lens;
    a.new_weights = new_weights;
    a.kept = kept;
    a.w_stride_b = weights_stride_b;
    a.w_stride_h = weights_stride_h;
    a.batch = batch;
    a.hkv = num_kv_heads;
    a.num_blocks = num_blocks;
    a.bs = block_size;
    a.max_blocks = max_blocks_per_seq;
    a.new_max_blocks = new_max_blocks;
    a.length = weights_length;
    a.budget = budget;
    a.recent = recent;
    a.stream = stream;
    return hip_status(ak::evict_launch(a), who);
}

}  // extern "C"
