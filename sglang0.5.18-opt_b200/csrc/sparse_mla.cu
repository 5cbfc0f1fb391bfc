// Attention of MLA queries over selected tokens of a paged latent cache.
//
//   s[h, t] = sm_scale * sum_d q[h, d] * k[t, d]     d < 576: 512 latent, 64 rope
//   out[h]  = sum_t softmax(s[h])[t] * k[t, :512],   lse[h] = log sum_t exp(s[h, t])
// over the tokens of the row's list: slots (token form), or the visible tokens of chosen 64-token
// blocks (block form).
//
// One warp per (row, head), one pass over the tokens with a running maximum and sum; lane l holds
// latent elements 16 l .. 16 l + 15 and rope elements 2 l, 2 l + 1 of the query and of the output.
#include <cuda_bf16.h>

#include "common.cuh"
#include "mla_slots.cuh"

HCU_DEFINE_STATUS(status_sparse_mla)

namespace hcu {
namespace {

struct AttnArgs {
  const uint16_t* q;
  int64_t q_row, q_head;
  const uint8_t* kv;
  int64_t n_slots, slot_stride;
  const int32_t* idx;
  int64_t idx_stride;
  int n_idx;
  const int32_t* bt;  // block form: the rows' block tables
  int64_t bt_stride;
  int n_bt;
  const int32_t* lengths;
  float sm_scale;
  int rows, heads;
  uint16_t* out;
  float* lse;
};

// Slot of the row's j-th candidate, -1 where there is none.
template <bool kBlocks>
__device__ __forceinline__ int64_t slot_of(const AttnArgs& a, int64_t row, int j) {
  if (!kBlocks) {
    const int32_t s = __ldg(a.idx + row * a.idx_stride + j);
    if (s >= a.n_slots) atomicOr(&g_hcu_status, HCU_STATUS_BAD_INPUT);
    return s < a.n_slots ? s : -1;
  }
  const int32_t b = __ldg(a.idx + row * a.idx_stride + j / kPage);
  if (b < 0) return -1;
  if (static_cast<int64_t>(b) * kPage + j % kPage >= __ldg(a.lengths + row)) return -1;
  const int64_t s = b < a.n_bt ? static_cast<int64_t>(__ldg(a.bt + row * a.bt_stride + b)) * kPage + j % kPage : -1;
  if (s < 0 || s >= a.n_slots) {
    atomicOr(&g_hcu_status, HCU_STATUS_BAD_INPUT);
    return -1;
  }
  return s;
}

template <bool kFp4, bool kBlocks>
__global__ __launch_bounds__(256) void sparse_mla_kernel(const AttnArgs a) {
  const int lane = threadIdx.x & 31;
  const int64_t w = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) >> 5;
  if (w >= static_cast<int64_t>(a.rows) * a.heads) return;
  const int64_t row = w / a.heads;
  const int head = static_cast<int>(w % a.heads);
  const uint16_t* qp = a.q + row * a.q_row + head * a.q_head;
  float q[18], o[16];
  for (int i = 0; i < 16; ++i) q[i] = __uint_as_float(static_cast<uint32_t>(qp[16 * lane + i]) << 16);
  for (int i = 0; i < 2; ++i) q[16 + i] = __uint_as_float(static_cast<uint32_t>(qp[512 + 2 * lane + i]) << 16);
  for (int i = 0; i < 16; ++i) o[i] = 0.f;
  float m = -INFINITY, l = 0.f;
  const float c = a.sm_scale * 1.4426950408889634f;
  const int n = a.n_idx * (kBlocks ? kPage : 1);
  for (int j = 0; j < n; ++j) {
    const int64_t slot = slot_of<kBlocks>(a, row, j);
    if (slot < 0) continue;
    const uint8_t* p = a.kv + slot * a.slot_stride;
    float v[18];
    if (kFp4) {
      const uint2 x = __ldg(reinterpret_cast<const uint2*>(p) + lane);
      const float s = e4m3_to_float(p[kKv4Scales + lane]) * *reinterpret_cast<const float*>(p + kKv4Token);
      for (int i = 0; i < 8; ++i) {
        const float2 f = __half22float2(e2m1x2_to_half2(((i < 4 ? x.x : x.y) >> (8 * (i & 3))) & 255));
        v[2 * i] = f.x * s;
        v[2 * i + 1] = f.y * s;
      }
    } else {
      const uint4 x = __ldg(reinterpret_cast<const uint4*>(p) + lane);
      const uint32_t xs[4] = {x.x, x.y, x.z, x.w};
      const float s = *reinterpret_cast<const float*>(p + kFp8Scales + 4 * (lane >> 3));
      for (int i = 0; i < 8; ++i) {
        const float2 f = __half22float2(e4m3x2_to_half2((xs[i >> 1] >> (16 * (i & 1))) & 0xffff));
        v[2 * i] = f.x * s;
        v[2 * i + 1] = f.y * s;
      }
    }
    const uint32_t r = __ldg(reinterpret_cast<const uint32_t*>(p + (kFp4 ? kKv4Rope : kFp8Rope)) + lane);
    v[16] = __uint_as_float(r << 16);
    v[17] = __uint_as_float(r & 0xffff0000u);
    float s = 0.f;
    for (int i = 0; i < 18; ++i) s = fmaf(q[i], v[i], s);
    for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
    s *= c;
    const float mn = fmaxf(m, s), f = exp2f(m - mn), e = exp2f(s - mn);
    m = mn;
    l = l * f + e;
    for (int i = 0; i < 16; ++i) o[i] = fmaf(o[i], f, e * v[i]);
  }
  uint16_t* op = a.out + w * kLatentDim + 16 * lane;
  for (int i = 0; i < 16; ++i) op[i] = __bfloat16_as_ushort(__float2bfloat16_rn(l > 0.f ? o[i] / l : 0.f));
  if (lane == 0) a.lse[w] = l > 0.f ? (m + log2f(l)) * 0.6931471805599453f : -INFINITY;
}

}  // namespace
}  // namespace hcu

extern "C" int64_t hcu_sparse_mla_attention_workspace_bytes(int64_t rows, int64_t heads, int64_t n_tokens) {
  if (rows < 0 || heads < 0 || n_tokens < 0) return -1;
  return 0;
}

extern "C" int hcu_sparse_mla_attention(const uint16_t* q, int64_t rows, int64_t heads, int64_t q_row, int64_t q_head,
                                        const uint8_t* kv_cache, int64_t n_slots, int64_t slot_stride,
                                        int32_t kv_format, const int32_t* indices, int64_t n_idx, int64_t idx_stride,
                                        const int32_t* block_table, int64_t bt_stride, int64_t n_bt,
                                        const int32_t* lengths, float sm_scale, void* workspace,
                                        int64_t workspace_bytes, uint16_t* out, float* lse, hcu_stream_t stream) {
  using namespace hcu;
  constexpr int64_t kMaxInt = 0x7fffffff;
  if (kv_format != HCU_KV_FP8_656 && kv_format != HCU_KV_FP4_432) return HCU_ERR_ARG;
  const bool fp4 = kv_format == HCU_KV_FP4_432, blocks = block_table != nullptr;
  if (rows < 0 || heads < 1 || q_row % 8 != 0 || q_head % 8 != 0 || n_slots < 0 ||
      slot_stride < (fp4 ? kKv4Slot : kFp8Slot) || slot_stride % 16 != 0 || n_idx < 0 || idx_stride < 0 ||
      n_idx > kMaxInt / kPage || (blocks && (n_bt < 0 || bt_stride < 0 || !lengths)))
    return HCU_ERR_ARG;
  if (rows == 0) return HCU_OK;
  if (heads > 1024 || rows > kMaxInt / 1024 || n_bt > kMaxInt / kPage) return HCU_ERR_UNSUPPORTED;
  if (!q || !out || !lse || (n_idx > 0 && (!indices || !kv_cache))) return HCU_ERR_ARG;
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(kv_cache) | reinterpret_cast<uintptr_t>(out)) % 16)
    return HCU_ERR_ARG;
  AttnArgs a{q,  q_row, q_head, kv_cache, n_slots, slot_stride, indices, idx_stride, static_cast<int>(n_idx),
             block_table, bt_stride, static_cast<int>(n_bt), lengths, sm_scale, static_cast<int>(rows),
             static_cast<int>(heads), out, lse};
  const unsigned grid = static_cast<unsigned>((rows * heads + 7) / 8);
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (fp4) {
    if (blocks)
      sparse_mla_kernel<true, true><<<grid, 256, 0, st>>>(a);
    else
      sparse_mla_kernel<true, false><<<grid, 256, 0, st>>>(a);
  } else {
    if (blocks)
      sparse_mla_kernel<false, true><<<grid, 256, 0, st>>>(a);
    else
      sparse_mla_kernel<false, false><<<grid, 256, 0, st>>>(a);
  }
  return launch_status();
}
