// Layouts of the two MLA slot formats and the conversions their readers share.
#pragma once

#include <cuda_fp16.h>
#include <cuda_fp4.h>
#include <cuda_fp8.h>
#include <stdint.h>

namespace hcu {

constexpr int kLatentDim = 512;
constexpr int kRopeDim = 64;
constexpr int kQkDim = kLatentDim + kRopeDim;  // 576

// 656 bytes: 512 fp8 e4m3 | 4 fp32 scales of 128 elements | 64 bf16 rope
constexpr int kFp8Slot = 656;
constexpr int kFp8Scales = 512;
constexpr int kFp8Rope = 528;

// 432 bytes: 512 e2m1 | 32 e4m3 scales of 16 elements | fp32 token scale (2^e) | 12 zeros | 64 bf16 rope
constexpr int kKv4Slot = 432;
constexpr int kKv4Scales = 256;
constexpr int kKv4Token = 288;
constexpr int kKv4Rope = 304;

__device__ __forceinline__ float e4m3_to_float(uint8_t b) {
  const __half_raw h = __nv_cvt_fp8_to_halfraw(b, __NV_E4M3);
  return __half2float(*reinterpret_cast<const __half*>(&h));
}

// Two e4m3 (low byte first) / two e2m1 (low half of the byte first) as f16, both exact.
__device__ __forceinline__ __half2 e4m3x2_to_half2(uint32_t two) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(two), __NV_E4M3);
  return *reinterpret_cast<const __half2*>(&h);
}
__device__ __forceinline__ __half2 e2m1x2_to_half2(uint32_t two) {
  const __half2_raw h = __nv_cvt_fp4x2_to_halfraw2(static_cast<__nv_fp4x2_storage_t>(two), __NV_E2M1);
  return *reinterpret_cast<const __half2*>(&h);
}

}  // namespace hcu
