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
// Both kernels are HBM streams, a warp per token and the store's lane l owning the 16 elements of
// group l.  Bound: 1584 bytes a token each way.  70001 tokens (111 MB, 17 us at the copy rate of
// 6.45 TB/s) take 28.7 us to store and 26.7 us to read with L2 flushed and events around the call, 22.2 and 21.4 in
// a graph of launches; 400000 tokens (634 MB, 98 us) 125 and 119 us, 116 and 114 in a graph, 5.5 TB/s.  The random
// order of the slots is a smaller part of what keeps them from the copy rate: in order 109 and 107 us.  The
// store's arithmetic goes in pairs (packed fp32, bf16 maxima), two tokens' loads ahead of it: 143 us for
// 400000 with one element an instruction and one token a warp.
#include <cuda_fp4.h>
#include <cuda_fp8.h>

#include "common.cuh"
#include "mla_slots.cuh"

HCU_DEFINE_STATUS(status_kv4)

namespace hcu {
namespace {

constexpr int kQThreads = 256;
constexpr int kStTokens = 2;  // tokens per warp whose loads are in flight before the first is packed

__device__ __forceinline__ float bf_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf_hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

__device__ __forceinline__ __nv_bfloat162 abs2(uint32_t w) { return __habs2(*reinterpret_cast<__nv_bfloat162*>(&w)); }

// RN(x / s) from rc = RN(1 / s): the remainder of the first guess is exact in one FMA, and adding
// its quotient gives the correctly rounded result (Markstein), so codes on e2m1's midpoints round
// as the division's would.  ns is -s.
__device__ __forceinline__ float2 quotients(float2 x, float2 ns, float2 rc) {
  const float2 q = __fmul2_rn(x, rc);
  return __ffma2_rn(__ffma2_rn(q, ns, x), rc, q);
}

__global__ __launch_bounds__(kQThreads, 5) void store_kv4_kernel(const uint16_t* __restrict__ kv_c, int64_t kv_tok,
                                                                 const uint16_t* __restrict__ k_pe, int64_t k_tok,
                                                                 bool pe_aligned, const int64_t* __restrict__ loc,
                                                                 int64_t n, uint8_t* __restrict__ kv, int64_t n_slots,
                                                                 int64_t slot_stride) {
  const int lane = threadIdx.x & 31;
  const int64_t warp = (static_cast<int64_t>(blockIdx.x) * kQThreads + threadIdx.x) >> 5;
  const int64_t n_warps = (static_cast<int64_t>(gridDim.x) * kQThreads) >> 5;
  for (int64_t t0 = warp * kStTokens; t0 < n; t0 += n_warps * kStTokens) {
    uint4 a[kStTokens], b[kStTokens], rope[kStTokens];
    uint32_t rope2[kStTokens];
    int64_t slot[kStTokens];
#pragma unroll
    for (int u = 0; u < kStTokens; ++u) {
      const int64_t t = min(t0 + u, n - 1);
      slot[u] = __ldg(loc + t);
      const uint4* src = reinterpret_cast<const uint4*>(kv_c + t * kv_tok) + 2 * lane;
      a[u] = __ldg(src);
      b[u] = __ldg(src + 1);
      const uint16_t* pe = k_pe + t * k_tok;
      rope[u] = make_uint4(0, 0, 0, 0);
      rope2[u] = 0;
      if (pe_aligned) {
        if (lane < 8) rope[u] = __ldg(reinterpret_cast<const uint4*>(pe) + lane);
      } else {
        rope2[u] = __ldg(pe + 2 * lane) | (static_cast<uint32_t>(__ldg(pe + 2 * lane + 1)) << 16);
      }
    }
#pragma unroll
    for (int u = 0; u < kStTokens; ++u) {
      if (t0 + u >= n) break;
      if (slot[u] < 0 || slot[u] >= n_slots) {
        if (lane == 0) atomicOr(&g_hcu_status, HCU_STATUS_BAD_INPUT);
        continue;
      }
      const uint32_t w[8] = {a[u].x, a[u].y, a[u].z, a[u].w, b[u].x, b[u].y, b[u].z, b[u].w};
      __nv_bfloat162 am2 = abs2(w[0]);
#pragma unroll
      for (int i = 1; i < 8; ++i) am2 = __hmax2(am2, abs2(w[i]));
      const uint32_t am = __float_as_uint(fmaxf(__low2float(am2), __high2float(am2)));
      const uint32_t top = __reduce_max_sync(0xffffffffu, am);
      // exponent of t: floor(log2(amax)) - 10, from the bits (a subnormal amax is below the 2^-100 floor)
      const int e = max(static_cast<int>(top >> 23) - 127 - 10, -100);
      const float ts = __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
      const uint8_t sg = static_cast<uint8_t>(
          __nv_cvt_float_to_fp8(__fdiv_rn(__uint_as_float(am), 6.f * ts), __NV_SATFINITE, __NV_E4M3));
      const float s = e4m3_to_float(sg) * ts;
      const float rc = s > 0.f ? __frcp_rn(s) : 0.f;
      const float2 ns2 = make_float2(-s, -s), rc2 = make_float2(rc, rc);
      uint32_t code[2] = {0, 0};
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        // a group whose scale is 0 has rc = 0 and code 0 throughout
        const float2 q = quotients(make_float2(bf_lo(w[i]), bf_hi(w[i])), ns2, rc2);
        code[i >> 2] |= static_cast<uint32_t>(__nv_cvt_float2_to_fp4x2(q, __NV_E2M1, cudaRoundNearest) & 0xff)
                        << (8 * (i & 3));
      }
      uint8_t* dst = kv + slot[u] * slot_stride;
      *reinterpret_cast<uint2*>(dst + 8 * lane) = make_uint2(code[0], code[1]);
      dst[kKv4Scales + lane] = sg;
      if (lane < 4) *reinterpret_cast<uint32_t*>(dst + kKv4Token + 4 * lane) = lane == 0 ? __float_as_uint(ts) : 0u;
      if (pe_aligned) {
        if (lane < 8) *reinterpret_cast<uint4*>(dst + kKv4Rope + 16 * lane) = rope[u];
      } else {
        *reinterpret_cast<uint32_t*>(dst + kKv4Rope + 4 * lane) = rope2[u];
      }
    }
  }
}

// Lane l writes pieces l and 32 + l of the row's 64 latent pieces of 16 bytes: with whole lines per
// store instruction 26.6 us for 70001 tokens, with a lane's own group of 16 (two stores 32 bytes
// apart) 30.7.
__global__ __launch_bounds__(kQThreads) void dequant_kv4_kernel(const uint8_t* __restrict__ kv, int64_t n_slots,
                                                                int64_t slot_stride,
                                                                const int32_t* __restrict__ slots, int64_t n,
                                                                uint16_t* __restrict__ out) {
  const int lane = threadIdx.x & 31;
  const int64_t warp = (static_cast<int64_t>(blockIdx.x) * kQThreads + threadIdx.x) >> 5;
  const int64_t n_warps = (static_cast<int64_t>(gridDim.x) * kQThreads) >> 5;
  for (int64_t t = warp; t < n; t += n_warps) {
    const int32_t src = __ldg(slots + t);
    if (src < 0 || src >= n_slots) {
      if (lane == 0) atomicOr(&g_hcu_status, HCU_STATUS_BAD_INPUT);
      continue;
    }
    const uint8_t* row = kv + src * slot_stride;
    const float ts = __ldg(reinterpret_cast<const float*>(row + kKv4Token));
    uint32_t q[2];
    float s[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      q[j] = __ldg(reinterpret_cast<const uint32_t*>(row) + 32 * j + lane);
      s[j] = e4m3_to_float(__ldg(row + kKv4Scales + 16 * j + (lane >> 1))) * ts;
    }
    uint4 rope = make_uint4(0, 0, 0, 0);
    if (lane < 8) rope = __ldg(reinterpret_cast<const uint4*>(row + kKv4Rope) + lane);
    uint4* dst = reinterpret_cast<uint4*>(out + t * kQkDim);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      uint32_t r[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(e2m1x2_to_half2((q[j] >> (8 * i)) & 0xffu));
        const __nv_bfloat162 o = __floats2bfloat162_rn(f.x * s[j], f.y * s[j]);
        r[i] = *reinterpret_cast<const uint32_t*>(&o);
      }
      dst[32 * j + lane] = make_uint4(r[0], r[1], r[2], r[3]);
    }
    if (lane < 8) dst[64 + lane] = rope;
  }
}

// Up to 16 CTAs an SM, two or three times what is resident, then warps loop: 400000 tokens take 120 us
// to read, 125 with a CTA for every 8 tokens; at 8 an SM their store takes 133 against 125.
int grid_for_tokens(int64_t warps) {
  const int64_t per = kQThreads / 32, cap = static_cast<int64_t>(sm_count()) * 16;
  const int64_t b = (warps + per - 1) / per;
  return static_cast<int>(b > cap ? cap : b);
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
  store_kv4_kernel<<<grid_for_tokens((n_tokens + kStTokens - 1) / kStTokens), kQThreads, 0, reinterpret_cast<cudaStream_t>(stream)>>>(
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
  dequant_kv4_kernel<<<grid_for_tokens(n_tokens), kQThreads, 0,
                       reinterpret_cast<cudaStream_t>(stream)>>>(kv_buffer, n_slots, slot_stride, page_table_1,
                                                                 n_tokens, out);
  return launch_status();
}
