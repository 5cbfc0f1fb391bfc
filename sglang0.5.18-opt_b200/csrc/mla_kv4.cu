// The 4-bit MLA slot: its writer and its paged read.
//
// Slot (432 bytes): 512 e2m1 codes (256 bytes, element 2j in the low half of byte j) | 32 e4m3
// scales, one per 16 elements | one fp32 token scale, a power of two | 12 zero bytes | 64 bf16 rope.
//   t    = 2^(floor(log2(amax)) - 10), amax over the 512 elements (2^-100 at least)
//   sg   = e4m3(amax_g / (6 t))          round to nearest even, saturated: at most 1024 / 3 < 448
//   code = e2m1(x / (sg t))              round to nearest even, saturated to 6; 0 where sg is 0
// With t a power of two, code * sg has at most six significant bits: every value the slot stands
// for is exact in bf16 and, divided by t, in f16, so readers never round.  A second level of scales
// costs 4 bytes and keeps latents of any magnitude in e4m3's normal range.
//
// Both kernels are HBM streams: a warp per token, lane l owning the 16 elements of group l.
#include <cuda_bf16.h>
#include <cuda_fp4.h>
#include <cuda_fp8.h>

#include "common.cuh"
#include "mla_slots.cuh"

HCU_DEFINE_STATUS(status_kv4)

namespace hcu {
namespace {

constexpr int kQThreads = 256;
constexpr int kDqUnroll = 4;  // tokens per warp whose loads are in flight before the first store

__device__ __forceinline__ float bf_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf_hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

// RN(x / s) from rc = RN(1 / s): the remainder of the first guess is exact in one FMA, and adding
// its quotient gives the correctly rounded result (Markstein), so codes on e2m1's midpoints round
// as the division's would.
__device__ __forceinline__ float quotient(float x, float s, float rc) {
  const float q = x * rc;
  return fmaf(fmaf(-q, s, x), rc, q);
}

__global__ __launch_bounds__(kQThreads) void store_kv4_kernel(const uint16_t* __restrict__ kv_c, int64_t kv_tok,
                                                              const uint16_t* __restrict__ k_pe, int64_t k_tok,
                                                              bool pe_aligned, const int64_t* __restrict__ loc,
                                                              int64_t n, uint8_t* __restrict__ kv, int64_t n_slots,
                                                              int64_t slot_stride) {
  const int lane = threadIdx.x & 31;
  const int64_t warp = (static_cast<int64_t>(blockIdx.x) * kQThreads + threadIdx.x) >> 5;
  const int64_t n_warps = (static_cast<int64_t>(gridDim.x) * kQThreads) >> 5;
  for (int64_t t = warp; t < n; t += n_warps) {
    const int64_t slot = __ldg(loc + t);
    const uint4* src = reinterpret_cast<const uint4*>(kv_c + t * kv_tok) + 2 * lane;
    const uint4 a = __ldg(src), b = __ldg(src + 1);
    const uint16_t* pe = k_pe + t * k_tok;
    uint4 rope = make_uint4(0, 0, 0, 0);
    uint32_t rope2 = 0;
    if (pe_aligned) {
      if (lane < 8) rope = __ldg(reinterpret_cast<const uint4*>(pe) + lane);
    } else {
      rope2 = __ldg(pe + 2 * lane) | (static_cast<uint32_t>(__ldg(pe + 2 * lane + 1)) << 16);
    }
    if (slot < 0 || slot >= n_slots) {
      if (lane == 0) atomicOr(&g_hcu_status, HCU_STATUS_BAD_INPUT);
      continue;
    }
    const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    // |x| of bf16 bits orders as an integer
    uint32_t am = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) am = max(am, max((w[i] << 16) & 0x7fff0000u, w[i] & 0x7fff0000u));
    const uint32_t top = __reduce_max_sync(0xffffffffu, am);
    // exponent of t: floor(log2(amax)) - 10, from the bits (a subnormal amax is below the 2^-100 floor)
    const int e = max(static_cast<int>(top >> 23) - 127 - 10, -100);
    const float ts = __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
    const uint8_t sg = static_cast<uint8_t>(
        __nv_cvt_float_to_fp8(__fdiv_rn(__uint_as_float(am), 6.f * ts), __NV_SATFINITE, __NV_E4M3));
    const float s = e4m3_to_float(sg) * ts;
    const float rc = s > 0.f ? __frcp_rn(s) : 0.f;
    uint32_t code[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      // a group whose scale is 0 has rc = 0 and code 0 throughout
      const float2 q = make_float2(quotient(bf_lo(w[i]), s, rc), quotient(bf_hi(w[i]), s, rc));
      code[i >> 2] |= static_cast<uint32_t>(__nv_cvt_float2_to_fp4x2(q, __NV_E2M1, cudaRoundNearest) & 0xff)
                      << (8 * (i & 3));
    }
    uint8_t* dst = kv + slot * slot_stride;
    *reinterpret_cast<uint2*>(dst + 8 * lane) = make_uint2(code[0], code[1]);
    dst[kKv4Scales + lane] = sg;
    if (lane < 4) *reinterpret_cast<uint32_t*>(dst + kKv4Token + 4 * lane) = lane == 0 ? __float_as_uint(ts) : 0u;
    if (pe_aligned) {
      if (lane < 8) *reinterpret_cast<uint4*>(dst + kKv4Rope + 16 * lane) = rope;
    } else {
      *reinterpret_cast<uint32_t*>(dst + kKv4Rope + 4 * lane) = rope2;
    }
  }
}

__global__ __launch_bounds__(kQThreads) void dequant_kv4_kernel(const uint8_t* __restrict__ kv, int64_t n_slots,
                                                                int64_t slot_stride,
                                                                const int32_t* __restrict__ slots, int64_t n,
                                                                uint16_t* __restrict__ out) {
  const int lane = threadIdx.x & 31;
  const int64_t warp = (static_cast<int64_t>(blockIdx.x) * kQThreads + threadIdx.x) >> 5;
  const int64_t n_warps = (static_cast<int64_t>(gridDim.x) * kQThreads) >> 5;
  for (int64_t t0 = warp * kDqUnroll; t0 < n; t0 += n_warps * kDqUnroll) {
    uint2 q[kDqUnroll];
    uint4 rope[kDqUnroll];
    float s[kDqUnroll];
    bool ok[kDqUnroll];
#pragma unroll
    for (int u = 0; u < kDqUnroll; ++u) {
      const int64_t t = t0 + u;
      const int64_t src = t < n ? static_cast<int64_t>(__ldg(slots + t)) : -1;
      ok[u] = src >= 0 && src < n_slots;
      if (t < n && !ok[u] && lane == 0) atomicOr(&g_hcu_status, HCU_STATUS_BAD_INPUT);
      const uint8_t* row = kv + (ok[u] ? src : 0) * slot_stride;
      q[u] = make_uint2(0, 0);
      rope[u] = make_uint4(0, 0, 0, 0);
      s[u] = 0.f;
      if (ok[u]) {
        q[u] = __ldg(reinterpret_cast<const uint2*>(row) + lane);
        s[u] = e4m3_to_float(__ldg(row + kKv4Scales + lane)) * __ldg(reinterpret_cast<const float*>(row + kKv4Token));
        if (lane < 8) rope[u] = __ldg(reinterpret_cast<const uint4*>(row + kKv4Rope) + lane);
      }
    }
#pragma unroll
    for (int u = 0; u < kDqUnroll; ++u) {
      if (!ok[u]) continue;
      uint32_t r[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t two = ((i < 4 ? q[u].x : q[u].y) >> (8 * (i & 3))) & 0xffu;
        const float2 f = __half22float2(e2m1x2_to_half2(two));
        const __nv_bfloat162 o = __floats2bfloat162_rn(f.x * s[u], f.y * s[u]);
        r[i] = *reinterpret_cast<const uint32_t*>(&o);
      }
      uint4* dst = reinterpret_cast<uint4*>(out + (t0 + u) * kQkDim);
      dst[2 * lane] = make_uint4(r[0], r[1], r[2], r[3]);
      dst[2 * lane + 1] = make_uint4(r[4], r[5], r[6], r[7]);
      if (lane < 8) dst[64 + lane] = rope[u];
    }
  }
}

int grid_for_tokens(int64_t warps) {
  const int64_t per = kQThreads / 32, cap = static_cast<int64_t>(sm_count()) * 8;
  const int64_t b = (warps + per - 1) / per;
  return static_cast<int>(b < 1 ? 1 : (b > cap ? cap : b));
}

}  // namespace
}  // namespace hcu

extern "C" int hcu_store_mla_kv4(const uint16_t* kv_c, int64_t kv_tok, const uint16_t* k_pe, int64_t k_tok,
                                 const int64_t* loc, int64_t n_tokens, uint8_t* kv_buffer, int64_t n_slots,
                                 int64_t slot_stride, hcu_stream_t stream) {
  using namespace hcu;
  if (n_tokens < 0 || n_slots < 0 || kv_tok % 8 != 0 || slot_stride < kKv4Slot || slot_stride % 16 != 0)
    return HCU_ERR_ARG;
  if (n_tokens == 0) return HCU_OK;
  if (!kv_c || !k_pe || !loc || !kv_buffer) return HCU_ERR_ARG;
  if ((reinterpret_cast<uintptr_t>(kv_c) | reinterpret_cast<uintptr_t>(kv_buffer)) % 16 != 0) return HCU_ERR_ARG;
  const bool al = reinterpret_cast<uintptr_t>(k_pe) % 16 == 0 && k_tok % 8 == 0;
  store_kv4_kernel<<<grid_for_tokens(n_tokens), kQThreads, 0, reinterpret_cast<cudaStream_t>(stream)>>>(
      kv_c, kv_tok, k_pe, k_tok, al, loc, n_tokens, kv_buffer, n_slots, slot_stride);
  return launch_status();
}

extern "C" int hcu_dequant_mla_kv4_paged(const uint8_t* kv_buffer, int64_t n_slots, int64_t slot_stride,
                                         const int32_t* page_table_1, int64_t n_tokens, uint16_t* out,
                                         hcu_stream_t stream) {
  using namespace hcu;
  if (n_tokens < 0 || n_slots < 0 || slot_stride < kKv4Slot || slot_stride % 16 != 0) return HCU_ERR_ARG;
  if (n_tokens == 0) return HCU_OK;
  if (!kv_buffer || !page_table_1 || !out) return HCU_ERR_ARG;
  if ((reinterpret_cast<uintptr_t>(kv_buffer) | reinterpret_cast<uintptr_t>(out)) % 16 != 0) return HCU_ERR_ARG;
  dequant_kv4_kernel<<<grid_for_tokens((n_tokens + kDqUnroll - 1) / kDqUnroll), kQThreads, 0,
                       reinterpret_cast<cudaStream_t>(stream)>>>(kv_buffer, n_slots, slot_stride, page_table_1,
                                                                 n_tokens, out);
  return launch_status();
}
