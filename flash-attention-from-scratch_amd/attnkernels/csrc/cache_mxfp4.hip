// The 4-bit paged KV cache's writer and reader (MXFP4, format in mxfp4.hpp).
// Not in the reference, whose cache is fp16 (attnkernels/reference.py:21-44);
// pages, slots and their rules are those of cache_write.hip: token t goes to
// page slot / block_size, row slot % block_size; a negative slot or one past
// the pool is skipped by the writer and read as zeros.
//
// Codes are [num_blocks, num_kv_heads, block_size, D/2] bytes, scales
// [num_blocks, num_kv_heads, block_size, D/32] bytes.  Both kernels are bound by
// memory: a row is 2 D bytes on one side and 17 D / 32 on the other.  One lane
// holds 8 channels (16 bytes, 4 bytes of codes), so four lanes are a scale
// group: its largest magnitude comes from two DPP lane exchanges on the bit
// patterns (magnitudes of one type order as integers), and the codes from the
// hardware's conversions, which round to nearest even.  Rows of the wide side are
// read and written once, 16 bytes a lane.  Measured: 16384 tokens, 8 heads of 128 from
// a fused projection 18.6 us to write (4.6 TB/s) and 17.5 to read back (4.9 TB/s; a
// copy reaches 4.9); 64 tokens 4.5 us each, the launch and two round trips.
#include <hip/hip_runtime.h>

#include "attn_kernels.hpp"
#include "mxfp4.hpp"

namespace ak {

namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ uint32_t max16(uint32_t a, uint32_t b) {  // the larger of each half
    typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a),
                                                                  __builtin_bit_cast(u16x2, b)));
}

template <int CTRL>
__device__ __forceinline__ uint32_t dpp32(uint32_t x) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xF, 0xF, false);
}

// The scale byte of the group that the lane's eight elements belong to.
template <class T>
__device__ __forceinline__ uint32_t group_scale(u32x4 x) {
    uint32_t m = max16(max16(x[0] & 0x7fff7fffu, x[1] & 0x7fff7fffu), max16(x[2] & 0x7fff7fffu, x[3] & 0x7fff7fffu));
    m = max16(m, m >> 16);
    m = max16(m, dpp32<kDppXor1>(m));
    m = max16(m, dpp32<kDppXor2>(m)) & 0xffffu;
    if (m >= Half<T>::kInf) return 255;  // an infinity or a NaN
    const int e = (int)((__builtin_bit_cast(uint32_t, Half<T>::widen(m)) + (1u << 21)) >> 23) - 2;
    return (uint32_t)max(e, 1);
}

template <class T>
__device__ __forceinline__ uint32_t encode8(u32x4 x, uint32_t s) {
    if (s == 255) return 0;
    const float scale = mx_scale(s);
    uint32_t c = Half<T>::template encode<0>(0, x[0], scale);
    c = Half<T>::template encode<1>(c, x[1], scale);
    c = Half<T>::template encode<2>(c, x[2], scale);
    return Half<T>::template encode<3>(c, x[3], scale);
}

template <class T>
__device__ __forceinline__ u32x4 decode8(uint32_t codes, uint32_t s) {
    const u32x4 x = mx_decode8<T>(codes, s == 0 ? __builtin_bit_cast(float, 0x00400000u) : mx_scale(s));
    const uint32_t nan = Half<T>::kInf << 16 | Half<T>::kInf | 0x00400040u;
    return s == 255 ? u32x4{nan, nan, nan, nan} : x;
}

// One workgroup per token and group of up to 256 lanes; lane r holds channels
// 8 r .. 8 r + 7 of the token's Hkv * D.
template <class T>
__global__ void __launch_bounds__(kThreads)
cache_write_mxfp4_kernel(const u32x4* __restrict__ key, const u32x4* __restrict__ value, uint32_t* __restrict__ k_codes,
                         uint8_t* __restrict__ k_scales, uint32_t* __restrict__ v_codes, uint8_t* __restrict__ v_scales,
                         const int64_t* __restrict__ slots, int hkv, int cpr, int64_t key_stride, int64_t value_stride,
                         int64_t num_slots, int bs) {
    const int r = (int)(blockIdx.y * blockDim.x + threadIdx.x);
    if (r >= hkv * cpr) return;
    const int64_t t = blockIdx.x, slot = slots[t];
    if (slot < 0 || slot >= num_slots) return;
    const u32x4 kx = __builtin_nontemporal_load(key + t * key_stride + r);
    const u32x4 vx = __builtin_nontemporal_load(value + t * value_stride + r);
    const int h = r / cpr, c = r - h * cpr;
    const int64_t page = slot / bs, row = (page * hkv + h) * bs + (slot - page * bs);
    const uint32_t ks = group_scale<T>(kx), vs = group_scale<T>(vx);
    k_codes[row * cpr + c] = encode8<T>(kx, ks);
    v_codes[row * cpr + c] = encode8<T>(vx, vs);
    if (c % 4 == 0) {
        k_scales[(row * cpr + c) / 4] = (uint8_t)ks;
        v_scales[(row * cpr + c) / 4] = (uint8_t)vs;
    }
}

template <class T>
__global__ void __launch_bounds__(kThreads)
cache_read_mxfp4_kernel(const uint32_t* __restrict__ k_codes, const uint8_t* __restrict__ k_scales,
                        const uint32_t* __restrict__ v_codes, const uint8_t* __restrict__ v_scales,
                        const int64_t* __restrict__ slots, u32x4* __restrict__ key, u32x4* __restrict__ value, int hkv,
                        int cpr, int64_t num_slots, int bs) {
    const int r = (int)(blockIdx.y * blockDim.x + threadIdx.x);
    if (r >= hkv * cpr) return;
    const int64_t t = blockIdx.x, slot = slots[t], dst = t * hkv * cpr + r;
    u32x4 kx = {0, 0, 0, 0}, vx = {0, 0, 0, 0};
    if (slot >= 0 && slot < num_slots) {
        const int h = r / cpr, c = r - h * cpr;
        const int64_t page = slot / bs, at = ((page * hkv + h) * bs + (slot - page * bs)) * cpr + c;
        kx = decode8<T>(k_codes[at], k_scales[at / 4]);
        vx = decode8<T>(v_codes[at], v_scales[at / 4]);
    }
    key[dst] = kx;
    value[dst] = vx;
}

dim3 rows_grid(const CacheMxArgs& a, int& threads) {
    const int64_t per_token = a.hkv * (a.head_dim / 8);
    threads = per_token >= kThreads ? kThreads : (int)((per_token + 63) / 64 * 64);
    return dim3((unsigned)a.num_tokens, (unsigned)((per_token + threads - 1) / threads));
}

}  // namespace

hipError_t cache_write_mxfp4_launch(const CacheMxArgs& a) {
    int threads;
    const dim3 grid = rows_grid(a, threads);
    auto launch = [&](auto* kernel) {
        hipLaunchKernelGGL(kernel, grid, dim3(threads), 0, (hipStream_t)a.stream, static_cast<const u32x4*>(a.key),
                           static_cast<const u32x4*>(a.value), static_cast<uint32_t*>(a.k_codes),
                           static_cast<uint8_t*>(a.k_scales), static_cast<uint32_t*>(a.v_codes),
                           static_cast<uint8_t*>(a.v_scales), a.slots, (int)a.hkv, (int)(a.head_dim / 8),
                           a.key_stride / 8, a.value_stride / 8, a.num_blocks * a.bs, (int)a.bs);
    };
    a.bf16 ? launch(cache_write_mxfp4_kernel<bf16>) : launch(cache_write_mxfp4_kernel<f16>);
    return hipGetLastError();
}

hipError_t cache_read_mxfp4_launch(const CacheMxArgs& a) {
    int threads;
    const dim3 grid = rows_grid(a, threads);
    auto launch = [&](auto* kernel) {
        hipLaunchKernelGGL(kernel, grid, dim3(threads), 0, (hipStream_t)a.stream,
                           static_cast<const uint32_t*>(a.k_codes), static_cast<const uint8_t*>(a.k_scales),
                           static_cast<const uint32_t*>(a.v_codes), static_cast<const uint8_t*>(a.v_scales), a.slots,
                           static_cast<u32x4*>(a.key_out), static_cast<u32x4*>(a.value_out), (int)a.hkv,
                           (int)(a.head_dim / 8), a.num_blocks * a.bs, (int)a.bs);
    };
    a.bf16 ? launch(cache_read_mxfp4_kernel<bf16>) : launch(cache_read_mxfp4_kernel<f16>);
    return hipGetLastError();
}

}  // namespace ak
