// The 64-token blocks a row attends to, chosen by the indexer's scores.
//
//   m_b = max over the visible tokens of block b of (mask bit set ? score : +0)
// and the n blocks with the largest m_b, ties to the lower index, the first n_sink and the last
// n_local visible blocks always among them, written in ascending order (-1 pads).
//
// One cluster of S CTAs per row.  Every CTA streams its share of the row's blocks (half a warp per
// block, 16 bytes a lane, 8 blocks in flight per warp), reduces each block to one monotone integer key
// and stores it into rank 0's shared memory; after the cluster barrier rank 0 finds the n-th largest
// key and writes the chosen blocks by one block-wide scan.  The select takes its digits from the top
// bit of the keys' range (2048 bins a pass) and stops as soon as a bin is taken whole, so one or two
// passes serve where fixed 8-bit digits took four, each a few barriers long.  With rows enough to fill
// the SMs S is 1 and the select of one row overlaps the streams of the others on its SM.
//
// Bound: the read of the scores, 4 B + 1 bit per visible token.  4096 rows of 67K tokens (1.14 GB, 177 us
// at the copy rate of 6.45 TB/s) take 208 us in a graph of launches, 5.5 TB/s, and 225 as one call with L2 flushed.
// 128 rows of 4K to 64K tokens (18 MB, 2.9 us) take 12.8 us in a graph: the cluster's two barriers and the
// select's passes, each a few barriers long, stand around the stream; their shares have not been measured apart.
#include <cooperative_groups.h>

#include "common.cuh"

HCU_DEFINE_STATUS(status_blocks)

namespace cg = cooperative_groups;

namespace hcu {
namespace {

constexpr int kSbThreads = 256;
constexpr int kSbWarps = kSbThreads / 32;
constexpr int kLoads = 4;                  // loads of two blocks each that a warp has in flight
constexpr int kUnit = 2 * kLoads;          // blocks per warp step
constexpr int kSbBins = 2048;
constexpr uint32_t kForced = 0xffffffffu;  // key of a block that is always chosen
constexpr int kMaxRowBlocks = 49152;       // keys of a row held in shared memory (192 KB)
constexpr int kMaxSbSplits = 8;            // portable cluster size
constexpr int kSbFill = 4;                 // CTAs per SM up to which a row is split (2, 6 and 8 measure the same)

struct BlocksArgs {
  const float* score;
  int64_t score_stride;
  const int16_t* mask;
  int64_t mask_stride;
  const int32_t* lengths;
  int width;      // tokens
  int n;          // blocks to choose
  int n_sink, n_local;
  int splits;
  int32_t* out;  // [rows, n]
};

struct SbSmem {
  int hist[kSbBins];
  int warp_sum[kSbWarps];
  int warp_above[kSbWarps], warp_tie[kSbWarps];
  uint32_t kmin, kmax;  // of the keys that are not forced
  int bin, above, count;
};

// Monotone signed image of a float: a larger score has a larger image; NaN with a clear sign is
// above +inf.
__device__ __forceinline__ int ordered(uint32_t b) {
  return static_cast<int>(b) ^ (static_cast<int>(static_cast<int>(b) >> 31) & 0x7fffffff);
}

__global__ __launch_bounds__(kSbThreads, 5) void select_blocks_kernel(const BlocksArgs a) {
  extern __shared__ uint32_t keys[];  // rank 0: one key per visible block of the row
  __shared__ SbSmem sm;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = a.splits > 1 ? static_cast<int>(blockIdx.x) % a.splits : 0;
  const int64_t row = a.splits > 1 ? blockIdx.x / a.splits : blockIdx.x;
  const int len = max(0, min(__ldg(a.lengths + row), a.width));
  const int nb = (len + kPage - 1) / kPage;
  int32_t* out = a.out + row * a.n;
  if (tid == 0) {
    sm.kmin = 0xffffffffu;
    sm.kmax = 0;
  }
  uint32_t* dst_keys = keys;
  SbSmem* dst_sm = &sm;
  if (a.splits > 1) {
    cg::this_cluster().sync();  // rank 0 has started: its shared memory may be written
    dst_keys = cg::this_cluster().map_shared_rank(keys, 0);
    dst_sm = cg::this_cluster().map_shared_rank(&sm, 0);
  } else {
    __syncthreads();
  }

  const bool all = nb <= a.n;  // uniform over the cluster
  if (!all) {
    const float* score = a.score + row * a.score_stride;
    const int16_t* mask = a.mask + row * a.mask_stride;
    const int units = (nb + kUnit - 1) / kUnit;
    uint32_t kmin = 0xffffffffu, kmax = 0;
    for (int u = rank * kSbWarps + warp; u < units; u += a.splits * kSbWarps) {
      float4 x[kLoads];
      // mask words of the unit's blocks, one a lane
      const int word = u * (kUnit * kPage / 16) + lane;
      const uint32_t mw = 16 * word < len ? static_cast<uint16_t>(__ldg(mask + word)) : 0u;
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {  // load i: blocks 2i (lanes 0-15) and 2i + 1
        const int tok = (u * kUnit + 2 * i) * kPage + 4 * lane;
        x[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (tok + 3 < len) {
          x[i] = __ldcs(reinterpret_cast<const float4*>(score + tok));
        } else if (tok < len) {
          x[i].x = score[tok];
          if (tok + 1 < len) x[i].y = score[tok + 1];
          if (tok + 2 < len) x[i].z = score[tok + 2];
        }
      }
      int k[kLoads];
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int tok = (u * kUnit + 2 * i) * kPage + 4 * lane;
        const uint32_t m = __shfl_sync(0xffffffffu, mw, 8 * i + (lane >> 2)) >> (4 * (lane & 3));
        // a visible token without its mask bit counts as +0 (image 0); one past the length not at all
        const int lo = static_cast<int>(0x80000000u);
        const int k0 = (m & 1) ? ordered(__float_as_uint(x[i].x)) : 0;
        const int k1 = (m & 2) ? ordered(__float_as_uint(x[i].y)) : 0;
        const int k2 = (m & 4) ? ordered(__float_as_uint(x[i].z)) : 0;
        const int k3 = (m & 8) ? ordered(__float_as_uint(x[i].w)) : 0;
        k[i] = tok < len ? k0 : lo;
        if (tok + 3 < len) {
          k[i] = max(max(k0, k1), max(k2, k3));
        } else {
          if (tok + 1 < len) k[i] = max(k[i], k1);
          if (tok + 2 < len) k[i] = max(k[i], k2);
        }
      }
      // Maxima over the 16 lanes of each half warp, all four loads at once: each step halves the loads a
      // lane carries, so they take 2 + 1 + 1 + 1 shuffles instead of 4 x 4.
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const int half = kLoads / 2 >> s, o = 1 << s;
        const bool hi = lane & o;
#pragma unroll
        for (int i = 0; i < half; ++i) {
          const int send = hi ? k[i] : k[i + half];
          const int keep = hi ? k[i + half] : k[i];
          k[i] = max(keep, __shfl_xor_sync(0xffffffffu, send, o));
        }
      }
      k[0] = max(k[0], __shfl_xor_sync(0xffffffffu, k[0], 4));
      k[0] = max(k[0], __shfl_xor_sync(0xffffffffu, k[0], 8));
      // lane bits 0 and 1 name the load: bit 0 chose the upper two, bit 1 the second of them
      const int b = u * kUnit + 2 * (((lane & 1) << 1) | ((lane >> 1) & 1)) + (lane >> 4);
      if (!(lane & 12) && b < nb) {
        const bool forced = b < a.n_sink || b >= nb - a.n_local;
        const int im = k[0] == -1 ? 0 : k[0];  // -0 ties with +0
        const uint32_t key = max(1u, min(static_cast<uint32_t>(im) ^ 0x80000000u, kForced - 1));
        dst_keys[b] = forced ? kForced : key;
        if (!forced) {
          kmin = min(kmin, key);
          kmax = max(kmax, key);
        }
      }
    }
    kmin = __reduce_min_sync(0xffffffffu, kmin);
    kmax = __reduce_max_sync(0xffffffffu, kmax);
    if (lane == 0 && kmin <= kmax) {
      atomicMin(&dst_sm->kmin, kmin);
      atomicMax(&dst_sm->kmax, kmax);
    }
  }
  if (a.splits > 1)
    cg::this_cluster().sync();  // rank 0 reads below what every rank stored above; no rank touches
                                // another's shared memory after this barrier
  else
    __syncthreads();
  if (rank != 0) return;
  if (all) {
    for (int i = tid; i < a.n; i += kSbThreads) out[i] = i < nb ? i : -1;
    return;
  }

  // The `left` largest of the keys that are not forced (n_sink + n_local <= n < nb are): bins of the range
  // [lo, lo + 2^(shift + 11)) from the top.  Ends with the threshold key `prefix` and the number of keys
  // equal to it that are taken; with none where a whole bin is.
  int left = a.n - a.n_sink - a.n_local;
  uint32_t lo = sm.kmin, prefix = kForced - 1;
  const uint32_t range = sm.kmax - lo;
  int shift = max(0, 32 - __clz(static_cast<int>(range)) - 11);
  uint32_t width_bits = 32 - __clz(static_cast<int>(range));  // keys considered: (k - lo) >> width_bits == 0
  while (left > 0) {
    for (int i = tid; i < kSbBins; i += kSbThreads) sm.hist[i] = 0;
    __syncthreads();
    for (int b = tid; b < nb; b += kSbThreads) {
      const uint32_t d = keys[b] - lo;
      if (keys[b] != kForced && keys[b] >= lo && (width_bits >= 32 || d >> width_bits == 0)) atomicAdd(&sm.hist[d >> shift], 1);
    }
    __syncthreads();
    // thread t: bins 8t .. 8t + 7; suffix sums over threads from the top
    int c[8], sum = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) sum += c[j] = sm.hist[8 * tid + j];
    int suf = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_down_sync(0xffffffffu, suf, o);
      if (lane + o < 32) suf += y;
    }
    if (lane == 0) sm.warp_sum[warp] = suf;
    __syncthreads();
    for (int w = warp + 1; w < kSbWarps; ++w) suf += sm.warp_sum[w];
    int above = suf - sum;
    if (above < left && suf >= left) {
#pragma unroll
      for (int j = 7; j >= 0; --j) {
        if (above < left && above + c[j] >= left) {
          sm.bin = 8 * tid + j;
          sm.above = above;
          sm.count = c[j];
        }
        above += c[j];
      }
    }
    __syncthreads();
    lo += static_cast<uint32_t>(sm.bin) << shift;
    left -= sm.above;
    if (shift == 0) {  // a bin is one key: `left` of those equal to it
      prefix = lo;
      break;
    }
    if (sm.count == left) {  // the whole bin
      prefix = lo - 1;  // keys start at 1
      left = 0;
      break;
    }
    width_bits = shift;
    shift = max(0, shift - 11);
    __syncthreads();
  }

  // blocks above the threshold key, and the `left` lowest of those equal to it
  const int per = (nb + kSbThreads - 1) / kSbThreads;
  const int b0 = min(tid * per, nb), b1 = min(b0 + per, nb);
  int above = 0, tie = 0;
  for (int b = b0; b < b1; ++b) {
    above += keys[b] > prefix;
    tie += keys[b] == prefix;
  }
  int ia = above, it = tie;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int ya = __shfl_up_sync(0xffffffffu, ia, o), yt = __shfl_up_sync(0xffffffffu, it, o);
    if (lane >= o) {
      ia += ya;
      it += yt;
    }
  }
  if (lane == 31) {
    sm.warp_above[warp] = ia;
    sm.warp_tie[warp] = it;
  }
  __syncthreads();
  int na = ia - above, nt = it - tie;
  for (int w = 0; w < warp; ++w) {
    na += sm.warp_above[w];
    nt += sm.warp_tie[w];
  }
  for (int b = b0; b < b1; ++b) {
    const uint32_t k = keys[b];
    if (k > prefix) {
      out[na + min(nt, left)] = b;
      ++na;
    } else if (k == prefix) {
      if (nt < left) out[na + nt] = b;
      ++nt;
    }
  }
}

}  // namespace
}  // namespace hcu

extern "C" int hcu_select_blocks(const float* score, int64_t rows, int64_t width, int64_t score_stride,
                                 const int16_t* mask, int64_t mask_stride, const int32_t* lengths, int64_t n_blocks,
                                 int64_t n_sink, int64_t n_local, int32_t* out, hcu_stream_t stream) {
  using namespace hcu;
  if (rows < 0 || width < 0 || score_stride < width || score_stride % 4 != 0 || mask_stride < (width + 15) / 16 ||
      n_blocks < 1 || n_sink < 0 || n_local < 0 || n_sink + n_local > n_blocks)
    return HCU_ERR_ARG;
  if (rows == 0) return HCU_OK;
  const int64_t row_blocks = (width + kPage - 1) / kPage;
  if (row_blocks > kMaxRowBlocks || n_blocks > 0x7fffffff || rows > 0x7fffffff / kMaxSbSplits)
    return HCU_ERR_UNSUPPORTED;
  if (!lengths || !out || (width > 0 && (!score || !mask))) return HCU_ERR_ARG;
  if (reinterpret_cast<uintptr_t>(score) % 16 != 0) return HCU_ERR_ARG;
  BlocksArgs a{score, score_stride, mask, mask_stride, lengths, static_cast<int>(width), static_cast<int>(n_blocks),
               static_cast<int>(n_sink), static_cast<int>(n_local), 1, out};
  // Splits: as many CTAs as are resident at once, each with 64 blocks (4096 tokens) at least.
  int s = 1;
  while (s < kMaxSbSplits && rows * 2 * s <= kSbFill * sm_count() && row_blocks >= 2 * s * 64) s *= 2;
  a.splits = s;
  static_assert(32 * 1024 + sizeof(SbSmem) <= 48 * 1024, "shared memory without opt-in");
  const size_t smem = static_cast<size_t>(row_blocks) * sizeof(uint32_t);
  if (smem > 32 * 1024) {  // with the kernel's static part (sizeof(SbSmem)) below the 48 KB of a launch that asks for none
    const cudaError_t e = cudaFuncSetAttribute(select_blocks_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               kMaxRowBlocks * static_cast<int>(sizeof(uint32_t)));
    if (e != cudaSuccess) {
      set_last_error(e);
      return HCU_ERR_LAUNCH;
    }
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(rows * s));
  cfg.blockDim = dim3(kSbThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = reinterpret_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(s);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = s > 1 ? 1 : 0;
  cudaLaunchKernelEx(&cfg, select_blocks_kernel, a);
  return launch_status();
}
