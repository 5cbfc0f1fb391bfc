// Attention of MLA queries over selected tokens of a paged latent cache (sm_100a tensor cores).
//
//   s[h, t] = sm_scale * sum_d q[h, d] * k[t, d]     d < 576: 512 latent, 64 rope
//   out[h]  = sum_t softmax(s[h])[t] * k[t, :512],   lse[h] = log sum_t exp(s[h, t])
// over the tokens of the row's list: slots (token form), or the visible tokens of chosen 64-token
// blocks (block form).
//
// Work: a job is (row, group of up to 64 heads), cut into tiles of 64 candidates.  The flat list of
// all tiles is split evenly over one persistent CTA per SM; a CTA's share of one job is a segment.
// A segment that is the whole job writes the result, any other one a partial (out, lse) that
// combine_kernel joins.  Per tile:
//   * 8 loader warps (one 8-token swizzle group each) gather the slots with 16-byte loads into
//     registers, convert them to f16 and store them as the tile's K: 9 chunks of [64 tokens][64
//     values], rows of 128 bytes, 128-byte swizzle.  A chunk is a K-major operand for q k^T and, read
//     the other way, an MN-major one for v^T, so the latent is stored once.  Raw loads of the next
//     tile are issued as the registers of this one are consumed;
//   * the MMA thread issues S = Q K^T (M = 64 heads, N = 64 tokens, K = 576) and, one tile behind,
//     O^T += V^T P^T (M = 128 latent values x 4, N = heads, K = 64 tokens): with the latent as M both
//     products run without padding rows at 64 heads, and O^T takes 4 x 64 TMEM columns;
//   * 4 softmax warps (16 heads each) read S, keep the running maximum and sum in fp32 and write P
//     in f16 over the tile's rope chunk, which S no longer needs.  O^T is rescaled only when a
//     maximum has risen by more than 2^kLazy.
//
// Number format.  f16 operands hold 11 bits where bf16 holds 8, and an fp8 or e2m1 value is exact in
// f16; its range is met by powers of two taken out per token and per query row:
//   * token t: 2^E, E from its largest scale; latent codes are multiplied by scale * 2^-E (rounded to
//     f16, exact for the 4-bit slot's power of two) and the rope by 2^-E 2^-10; E is raised where the
//     rope would leave f16's range (latents 2^-35 below the rope);
//   * query row: 2^e, its largest element just below 2^4 (latent part) or 2^14 (rope part, which
//     takes the 2^10 back), so elements down to 2^-18 of the largest keep all their bits.
// S * 2^(E + e) is the score; P carries 2^E of its token in its exponent (w = s + E, whose maximum is
// the running one), so O needs no correction, and the sum takes 2^-E back per token.
//
// Bound: at 64 heads the shared-memory port.  A 64-token tile moves 72 KB of K in, 147 KB of Q and K
// operands for S and 96 KB of V and P for O out: about 2500 cycles at 128 B per cycle, 39 per token,
// against 24 per token for its products at the dense rate and 15 for its share of HBM.
#include <cuda_bf16.h>

#include "common.cuh"
#include "mla_slots.cuh"

HCU_DEFINE_STATUS(status_sparse_mla)

namespace hcu {
namespace {

constexpr int kTile = 64;        // candidates per tile
constexpr int kHg = 64;          // heads per job
constexpr int kChunks = kQkDim / 64;
constexpr int kChunkBytes = 64 * 128;  // [64 rows][64 f16]
constexpr int kTileBytes = kChunks * kChunkBytes;
constexpr int kSoftWarps = 4;
constexpr int kMmaWarp = kSoftWarps;
constexpr int kLoadWarp = kSoftWarps + 1;
constexpr int kLoadWarps = 8;
constexpr int kAtThreads = (kLoadWarp + kLoadWarps) * 32;
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kTmemO = 0;    // 4 blocks of 128 latent values x 64 heads
constexpr uint32_t kTmemS = 256;  // 2 score buffers of 64 columns
// P is 2^(w - m + kBias): a row's largest weight is 2^11, 2^15 while its maximum has grown by the
// tolerated 2^kLazy, and weights down to 2^-25 of the largest are normal f16 numbers.
constexpr float kLazy = 4.f;
constexpr float kBias = 11.f;
constexpr int kRopeShift = 10;
constexpr int kPartFloats = kHg * kLatentDim + kHg;

struct __align__(1024) AtSmem {
  uint8_t q[kTileBytes];
  uint8_t k[2][kTileBytes];
  float tok_e[2][kTile];    // E of each token (-inf: no token)
  float tok_up[2][kTile];   // 2^E (0: no token)
  float tok_dn[2][kTile];   // 2^-E (0: no token)
  float cq[2][kHg];         // per head: 2^e * sm_scale * log2(e), beside a segment's first tile
  float factor[kHg];        // rescale of O, then 1 / sum
  int empty_tile[2];        // the tile holds no token
  uint64_t full[2], empty[2], sfull[2], pready[2];
  uint64_t qfull, qempty, oempty, done;
  uint32_t tmem;
  int abort;
};
static_assert(sizeof(AtSmem) + 1024 <= 232448, "shared memory");

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
  int heads, n_hg;
  int tiles;      // per job
  int64_t total;  // jobs * tiles
  uint16_t* out;
  float* lse;
  float* part;    // [grid][2][kPartFloats]
};

__device__ __forceinline__ int64_t first_tile(int64_t total, int cta, int grid) { return total * cta / grid; }

// ---------------------------------------------------------------- PTX
__device__ __forceinline__ void mma_f16(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                        uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// f16 x f16 -> f32; a_mn: A is MN-major.
__host__ __device__ constexpr uint32_t idesc_f16(int M, int N, bool a_mn) {
  return (1u << 4) | (a_mn ? 1u << 15 : 0u) | (static_cast<uint32_t>(N >> 3) << 17) |
         (static_cast<uint32_t>(M >> 4) << 24);
}

// MN-major operand in the same swizzled rows: 64 M values per 128-byte row, 8 K rows per 1024 bytes,
// the next 64 M values one chunk further.
__device__ __forceinline__ uint64_t sw128_mnmajor_desc(uint32_t smem_addr) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((smem_addr & 0x3FFFFu) >> 4);
  d |= static_cast<uint64_t>(kChunkBytes >> 4) << 16;  // leading offset: next 64 M values
  d |= static_cast<uint64_t>(1024 >> 4) << 32;         // stride offset: next 8 K rows
  d |= static_cast<uint64_t>(1) << 46;
  d |= static_cast<uint64_t>(2) << 61;
  return d;
}

// 16 lanes x 64 columns, as 8 column groups of an 8x8-pair fragment: thread t holds, for group n,
// rows t / 4 (r[4n], r[4n + 1]) and t / 4 + 8 (r[4n + 2], r[4n + 3]), columns 8n + 2 (t % 4) + {0, 1}.
__device__ __forceinline__ void tmem_ld_16x256_x8(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]),
        "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]),
        "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}

__device__ __forceinline__ void tmem_st_x32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, "
      "%14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};" ::"r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]),
      "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]),
      "r"(r[29]), "r"(r[30]), "r"(r[31]), "r"(taddr)
      : "memory");
}

__device__ __forceinline__ void stmatrix_x4(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c),
               "r"(d)
               : "memory");
}

__device__ __forceinline__ void st_shared_v4(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

__device__ __forceinline__ void fence_async_shared() {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// OR of a predicate over the softmax warps.
__device__ __forceinline__ bool soft_any(bool p) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %1, 0;\n\t"
      "barrier.cta.red.or.pred q, 1, %2, p;\n\t"
      "selp.b32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(static_cast<uint32_t>(p)), "n"(kSoftWarps * 32)
      : "memory");
  return r != 0;
}

__device__ __forceinline__ uint32_t h2_bits(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }

__device__ __forceinline__ uint4 ldg_v4(const uint8_t* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

// ---------------------------------------------------------------- loader
// One lane's view of a tile's candidates.
struct Cand {
  int32_t a, b;  // token form: slots of candidates 2 lane, 2 lane + 1 (-1: none); block form: first slot, count
  bool any;      // the tile holds a token (uniform)
};

template <bool kBlocks>
__device__ __forceinline__ Cand candidates(const AttnArgs& p, int64_t row, int tile, int lane) {
  Cand c;
  if constexpr (kBlocks) {
    c.a = c.b = 0;
    const int32_t b = tile < p.n_idx ? __ldg(p.idx + row * p.idx_stride + tile) : -1;
    if (b >= 0) {
      const int64_t left = static_cast<int64_t>(__ldg(p.lengths + row)) - static_cast<int64_t>(b) * kPage;
      const int n = left <= 0 ? 0 : static_cast<int>(left < kPage ? left : kPage);
      const int32_t page = n > 0 && b < p.n_bt ? __ldg(p.bt + row * p.bt_stride + b) : -1;
      const int64_t s = static_cast<int64_t>(page) * kPage;
      if (page >= 0 && s + n <= p.n_slots) {
        c.a = static_cast<int32_t>(s);
        c.b = n;
      } else if (n > 0 && lane == 0) {
        atomicOr(&g_hcu_status, HCU_STATUS_BAD_INPUT);
      }
    }
    c.any = c.b > 0;
  } else {
    const int j = tile * kTile + 2 * lane;
    const int32_t* p0 = p.idx + row * p.idx_stride;
    c.a = j < p.n_idx ? __ldg(p0 + j) : -1;
    c.b = j + 1 < p.n_idx ? __ldg(p0 + j + 1) : -1;
    const bool bad_a = c.a >= p.n_slots, bad_b = c.b >= p.n_slots;
    if (bad_a || bad_b) atomicOr(&g_hcu_status, HCU_STATUS_BAD_INPUT);
    if (bad_a) c.a = -1;
    if (bad_b) c.b = -1;
    c.any = __any_sync(0xffffffffu, c.a >= 0 || c.b >= 0);
  }
  return c;
}

// Slot of candidate j of the tile (uniform), -1 where there is none.
template <bool kBlocks>
__device__ __forceinline__ int32_t slot_at(const Cand& c, int j) {
  if constexpr (kBlocks) return j < c.b ? c.a + j : -1;
  return __shfl_sync(0xffffffffu, j & 1 ? c.b : c.a, j >> 1);
}

// A lane's raw bytes of its warp's 8 tokens of one tile.
template <bool kFp4>
struct Raw {
  uint4 x[8];       // latent codes 16 lane .. 16 lane + 15 (4-bit: .x, .y)
  uint32_t sc[8];   // fp8: the lane's group scale; 4-bit: its e4m3 scale
  float ts[8];      // 4-bit: the token scale
  uint4 rope[2];    // tokens 4 i + lane / 8, rope elements 8 (lane % 8) ..
};

template <bool kFp4, bool kBlocks>
__device__ __forceinline__ void load_token(const AttnArgs& p, const Cand& c, int lw, int lane, int t, Raw<kFp4>& r) {
  const int32_t s = slot_at<kBlocks>(c, lw * 8 + t);
  r.x[t] = make_uint4(0, 0, 0, 0);
  r.sc[t] = 0;
  if constexpr (kFp4) r.ts[t] = 0.f;
  if (s >= 0) {
    const uint8_t* b = p.kv + s * p.slot_stride;
    if constexpr (kFp4) {
      const uint2 v = __ldg(reinterpret_cast<const uint2*>(b) + lane);
      r.x[t].x = v.x;
      r.x[t].y = v.y;
      r.sc[t] = __ldg(b + kKv4Scales + lane);
      r.ts[t] = __ldg(reinterpret_cast<const float*>(b + kKv4Token));
    } else {
      r.x[t] = ldg_v4(b + 16 * lane);
      r.sc[t] = __ldg(reinterpret_cast<const uint32_t*>(b + kFp8Scales) + (lane >> 3));
    }
  }
}

template <bool kFp4, bool kBlocks>
__device__ __forceinline__ void load_rope(const AttnArgs& p, const Cand& c, int lw, int lane, Raw<kFp4>& r) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int j = lw * 8 + 4 * i + (lane >> 3);
    int32_t s;
    if constexpr (kBlocks) {
      s = j < c.b ? c.a + j : -1;
    } else {
      const int32_t a = __shfl_sync(0xffffffffu, c.a, j >> 1), b = __shfl_sync(0xffffffffu, c.b, j >> 1);
      s = j & 1 ? b : a;
    }
    r.rope[i] = make_uint4(0, 0, 0, 0);
    if (s >= 0) r.rope[i] = ldg_v4(p.kv + s * p.slot_stride + (kFp4 ? kKv4Rope : kFp8Rope) + 16 * (lane & 7));
  }
}

// bf16 pair (packed) * f -> f16 pair.
__device__ __forceinline__ uint32_t bf2_to_h2(uint32_t w, float f) {
  return h2_bits(__floats2half2_rn(__uint_as_float(w << 16) * f, __uint_as_float(w & 0xffff0000u) * f));
}

// The 64 heads of a job into the Q buffer: warp lw takes heads 8 lw .. 8 lw + 7, four lanes each.
// Returns the head's factor from the product to the score in base 2.  Two passes (the second reads
// L1) instead of 72 registers.
__device__ __forceinline__ float load_q(const AttnArgs& p, AtSmem& sm, int64_t row, int h0, int lw, int lane) {
  const int hr = lane >> 2, sub = lane & 3;
  const int h = h0 + lw * 8 + hr;
  const bool on = h < p.heads;
  const uint4* src = reinterpret_cast<const uint4*>(p.q + row * p.q_row + static_cast<int64_t>(h) * p.q_head);
  uint32_t am = 0;
#pragma unroll 6
  for (int i = 0; i < 18; ++i) {
    const uint4 v = on ? __ldg(src + sub + 4 * i) : make_uint4(0, 0, 0, 0);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) am = max(am, max(w[j] & 0x7fffu, (w[j] >> 16) & 0x7fffu));
  }
  am = max(am, __shfl_xor_sync(0xffffffffu, am, 1));
  am = max(am, __shfl_xor_sync(0xffffffffu, am, 2));
  // biased exponent of the largest element, kept where the scales below are normal floats
  const int eb = min(max(static_cast<int>(am >> 7), 20), 240);
  const float f_lat = __uint_as_float(static_cast<uint32_t>(254 - eb + 3) << 23);   // largest into [2^3, 2^4)
  const float f_rope = __uint_as_float(static_cast<uint32_t>(254 - eb + 13) << 23);  // 2^10 more
  const uint32_t base = smem_u32(sm.q) + lw * 1024 + hr * 128;
#pragma unroll 6
  for (int i = 0; i < 18; ++i) {
    const int u = sub + 4 * i;
    const float f = i < 16 ? f_lat : f_rope;
    const uint4 v = on ? __ldg(src + u) : make_uint4(0, 0, 0, 0);
    st_shared_v4(base + (u >> 3) * kChunkBytes + (((u & 7) ^ hr) << 4), bf2_to_h2(v.x, f), bf2_to_h2(v.y, f),
                 bf2_to_h2(v.z, f), bf2_to_h2(v.w, f));
  }
  return p.sm_scale * 1.4426950408889634f * __uint_as_float(static_cast<uint32_t>(eb - 3) << 23);
}

// Converts and stores the warp's 8 tokens of a tile; `next` (the following tile's candidates, null at
// the end) is loaded into the registers as they fall free.
template <bool kFp4, bool kBlocks>
__device__ __forceinline__ void store_tile(const AttnArgs& p, AtSmem& sm, int b, const Cand& c, const Cand* next,
                                           int lw, int lane, Raw<kFp4>& r) {
  // rope exponents: largest biased exponent of each token's rope, at lanes 8 (t % 4) .. of er[t / 4]
  uint32_t er[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t w[4] = {r.rope[i].x, r.rope[i].y, r.rope[i].z, r.rope[i].w};
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) m = max(m, max(w[j] & 0x7fffu, (w[j] >> 16) & 0x7fffu));
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    er[i] = m >> 7;
  }
  uint32_t eb_rope[2] = {0, 0};
  const uint32_t base = smem_u32(sm.k[b]) + lw * 1024;
  const int half = (lane >> 2) & 1;  // odd chunks store their upper 16 bytes first: no bank conflict
#pragma unroll
  for (int t = 0; t < 8; ++t) {
    uint32_t sexp;
    if constexpr (kFp4) {
      sexp = (__float_as_uint(r.ts[t]) & 0x7fffffffu) >> 23;
    } else {
      sexp = (r.sc[t] & 0x7fffffffu) >> 23;
      sexp = max(sexp, __shfl_xor_sync(0xffffffffu, sexp, 8));
      sexp = max(sexp, __shfl_xor_sync(0xffffffffu, sexp, 16));
    }
    const int re = static_cast<int>(__shfl_sync(0xffffffffu, er[t >> 2], 8 * (t & 3)));
    const int eb = min(max(max(static_cast<int>(sexp), re - 13 - kRopeShift), 27), 247);
    if ((lane >> 3) == (t & 3)) eb_rope[t >> 2] = eb;
    const float dn = __uint_as_float(static_cast<uint32_t>(254 - eb) << 23);
    uint32_t y[8];
    if constexpr (kFp4) {
      const __half2 s =
          __float2half2_rn(e4m3_to_float(static_cast<uint8_t>(r.sc[t])) * (r.ts[t] * dn));
      const uint32_t x0 = half ? r.x[t].y : r.x[t].x, x1 = half ? r.x[t].x : r.x[t].y;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        y[i] = h2_bits(__hmul2(e2m1x2_to_half2((x0 >> (8 * i)) & 0xff), s));
        y[4 + i] = h2_bits(__hmul2(e2m1x2_to_half2((x1 >> (8 * i)) & 0xff), s));
      }
    } else {
      const __half2 s = __float2half2_rn(__uint_as_float(r.sc[t]) * dn);
      const uint32_t x[4] = {half ? r.x[t].z : r.x[t].x, half ? r.x[t].w : r.x[t].y, half ? r.x[t].x : r.x[t].z,
                             half ? r.x[t].y : r.x[t].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        y[2 * i] = h2_bits(__hmul2(e4m3x2_to_half2(x[i] & 0xffffu), s));
        y[2 * i + 1] = h2_bits(__hmul2(e4m3x2_to_half2(x[i] >> 16), s));
      }
    }
    const uint32_t a = base + (lane >> 2) * kChunkBytes + t * 128;
    const int u = 2 * (lane & 3) + half;
    st_shared_v4(a + ((u ^ t) << 4), y[0], y[1], y[2], y[3]);
    st_shared_v4(a + (((u ^ 1) ^ t) << 4), y[4], y[5], y[6], y[7]);
    const bool on = slot_at<kBlocks>(c, lw * 8 + t) >= 0;
    if (lane == t) {
      sm.tok_e[b][lw * 8 + t] = on ? static_cast<float>(eb - 127) : -INFINITY;
      sm.tok_up[b][lw * 8 + t] = on ? __uint_as_float(static_cast<uint32_t>(eb) << 23) : 0.f;
      sm.tok_dn[b][lw * 8 + t] = on ? dn : 0.f;
    }
    if (next) load_token<kFp4, kBlocks>(p, *next, lw, lane, t, r);
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int t = 4 * i + (lane >> 3);
    const float f = __uint_as_float(static_cast<uint32_t>(254 - eb_rope[i]) << 23) * (1.f / (1 << kRopeShift));
    st_shared_v4(base + 8 * kChunkBytes + t * 128 + (((lane & 7) ^ t) << 4), bf2_to_h2(r.rope[i].x, f),
                 bf2_to_h2(r.rope[i].y, f), bf2_to_h2(r.rope[i].z, f), bf2_to_h2(r.rope[i].w, f));
  }
  if (next) load_rope<kFp4, kBlocks>(p, *next, lw, lane, r);
}

template <bool kFp4, bool kBlocks>
__global__ __launch_bounds__(kAtThreads, 1) void sparse_mla_kernel(const AttnArgs p) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  AtSmem& sm = smem_aligned_1024<AtSmem>(smem_raw);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t f0 = first_tile(p.total, blockIdx.x, gridDim.x);
  const int n = static_cast<int>(first_tile(p.total, blockIdx.x + 1, gridDim.x) - f0);  // at least 1
  const int64_t job0 = f0 / p.tiles;
  const int tile0 = static_cast<int>(f0 - job0 * p.tiles);

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sm.full[i], kLoadWarps);
      mbar_init(&sm.empty[i], 1);
      mbar_init(&sm.sfull[i], 1);
      mbar_init(&sm.pready[i], kSoftWarps);
    }
    mbar_init(&sm.qfull, kLoadWarps);
    mbar_init(&sm.qempty, 1);
    mbar_init(&sm.oempty, kSoftWarps);
    mbar_init(&sm.done, 1);
    sm.abort = 0;
    fence_barrier_init();
  }
  if (warp == kMmaWarp) {
    tmem_alloc(&sm.tmem, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sm.tmem;
  volatile int* abort = &sm.abort;

  // Every role walks the CTA's n tiles; no role leaves early, so that the named barriers of the
  // softmax warps stay complete: after a wait ran out (abort) the remaining waits return at once and
  // no more MMAs are issued.
  if (warp >= kLoadWarp) {
    // ------------------------------------------------ loaders
    const int lw = warp - kLoadWarp;
    Raw<kFp4> raw;
    int64_t job = job0, njob = job0;
    int tile = tile0, ntile = tile0, seg = 0;
    Cand cur = candidates<kBlocks>(p, job / p.n_hg, tile, lane), nxt = cur;
#pragma unroll
    for (int t = 0; t < 8; ++t) load_token<kFp4, kBlocks>(p, cur, lw, lane, t, raw);
    load_rope<kFp4, kBlocks>(p, cur, lw, lane, raw);
    for (int g = 0; g < n; ++g) {
      const int b = g & 1;
      const bool more = g + 1 < n;
      if (more) {
        if (++ntile == p.tiles) {
          ntile = 0;
          ++njob;
        }
        nxt = candidates<kBlocks>(p, njob / p.n_hg, ntile, lane);
      }
      const bool first = g == 0 || tile == 0;
      float cq = 0.f;
      if (first) {
        if (seg > 0) mbar_wait(&sm.qempty, (seg - 1) & 1, abort, &g_hcu_status);
        ++seg;
        cq = load_q(p, sm, job / p.n_hg, static_cast<int>(job % p.n_hg) * kHg, lw, lane);
        fence_async_shared();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.qfull);
      }
      if (g >= 2) mbar_wait(&sm.empty[b], ((g >> 1) - 1) & 1, abort, &g_hcu_status);
      if (first && (lane & 3) == 0) sm.cq[b][lw * 8 + (lane >> 2)] = cq;
      if (cur.any) {
        store_tile<kFp4, kBlocks>(p, sm, b, cur, more ? &nxt : nullptr, lw, lane, raw);
        fence_async_shared();
      } else if (more) {
#pragma unroll
        for (int t = 0; t < 8; ++t) load_token<kFp4, kBlocks>(p, nxt, lw, lane, t, raw);
        load_rope<kFp4, kBlocks>(p, nxt, lw, lane, raw);
      }
      if (lw == 0 && lane == 0) sm.empty_tile[b] = !cur.any;
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.full[b]);
      cur = nxt;
      job = njob;
      tile = ntile;
    }
  } else if (warp == kMmaWarp) {
    // ------------------------------------------------ MMA issuer
    if (elect_one()) {
      constexpr uint32_t id_s = idesc_f16(64, kTile, false);
      int64_t job = job0;
      int tile = tile0, seg = -1;
      bool prev_empty = true, prev_first = false;  // of the tile whose second product is due
      int prev_seg = 0, prev_n = kHg;
      uint32_t acc = 0;  // the segment's O holds something
      const auto second = [&](int h) {  // O^T += V^T P^T of tile h
        const int b = h & 1;
        if (prev_first) acc = 0;
        bool ok = mbar_wait(&sm.pready[b], (h >> 1) & 1, abort, &g_hcu_status);
        if (prev_empty) {
          mbar_arrive(&sm.empty[b]);
          return;
        }
        if (acc == 0 && prev_seg > 0) ok = mbar_wait(&sm.oempty, (prev_seg - 1) & 1, abort, &g_hcu_status) && ok;
        tc_fence_after();
        if (ok && !*abort) {
          const uint32_t id_o = idesc_f16(128, prev_n, true);
          const uint64_t v = sw128_mnmajor_desc(smem_u32(sm.k[b]));
          const uint64_t pd = sw128_kmajor_desc(smem_u32(sm.k[b]) + 8 * kChunkBytes);
#pragma unroll
          for (int ks = 0; ks < kTile / 16; ++ks)
#pragma unroll
            for (int d = 0; d < 4; ++d)
              mma_f16(tmem + kTmemO + 64 * d, v + ((2 * d * kChunkBytes + ks * 2048) >> 4), pd + 2 * ks, id_o,
                      ks > 0 ? 1u : acc);
        }
        acc = 1;
        tc_commit(&sm.empty[b]);
      };
      for (int g = 0; g < n; ++g) {
        const int b = g & 1;
        const bool first = g == 0 || tile == 0;
        const bool last = tile + 1 == p.tiles;  // of the job; the CTA's last segment needs no release
        if (first) mbar_wait(&sm.qfull, (++seg) & 1, abort, &g_hcu_status);
        const bool ok = mbar_wait(&sm.full[b], (g >> 1) & 1, abort, &g_hcu_status);
        const bool none = !ok || sm.empty_tile[b];
        tc_fence_after();
        if (!none) {
          const uint64_t qd = sw128_kmajor_desc(smem_u32(sm.q)), kd = sw128_kmajor_desc(smem_u32(sm.k[b]));
#pragma unroll
          for (int k = 0; k < kQkDim / 16; ++k) {
            const uint32_t off = ((k >> 2) * kChunkBytes + (k & 3) * 32) >> 4;
            mma_f16(tmem + kTmemS + 64 * b, qd + off, kd + off, id_s, k > 0 ? 1u : 0u);
          }
          tc_commit(&sm.sfull[b]);
        } else {
          mbar_arrive(&sm.sfull[b]);
        }
        if (last) tc_commit(&sm.qempty);
        if (g > 0) second(g - 1);
        prev_empty = none;
        prev_first = first;
        prev_seg = seg;
        prev_n = (min(kHg, p.heads - static_cast<int>(job % p.n_hg) * kHg) + 15) & ~15;
        if (++tile == p.tiles) {
          tile = 0;
          ++job;
        }
      }
      second(n - 1);
      tc_commit(&sm.done);
      mbar_wait_drain(&sm.done, 0, &g_hcu_status);
    }
  } else {
    // ------------------------------------------------ softmax and output
    const int r0 = 16 * warp + (lane >> 2), r1 = r0 + 8;  // the thread's two heads of the job
    const int cl = 2 * (lane & 3);                         // its columns: 8 n + cl, 8 n + cl + 1
    const uint32_t quad = static_cast<uint32_t>(warp * 32) << 16;
    int64_t job = job0;
    int tile = tile0, seg = 0;
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f, cq0 = 0.f, cq1 = 0.f;
    bool started = false;  // O holds something
    for (int g = 0; g < n; ++g) {
      const int b = g & 1;
      mbar_wait(&sm.full[b], (g >> 1) & 1, abort, &g_hcu_status);  // the loaders' factors and exponents
      mbar_wait(&sm.sfull[b], (g >> 1) & 1, abort, &g_hcu_status);
      if (g == 0 || tile == 0) {
        m0 = m1 = -INFINITY;
        l0 = l1 = 0.f;
        cq0 = sm.cq[b][r0];
        cq1 = sm.cq[b][r1];
        started = false;
      }
      const bool none = sm.empty_tile[b] || *abort;
      // a wait that ran out leaves the warps with different views: let all of them see the same one
      if (!soft_any(!none)) {
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.pready[b]);
      } else {
        tc_fence_after();
        uint32_t s[32];
        tmem_ld_16x256_x8(tmem + kTmemS + 64 * b + quad, s);
        float mx0 = -INFINITY, mx1 = -INFINITY;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float2 up = *reinterpret_cast<const float2*>(&sm.tok_up[b][8 * i + cl]);
          const float2 e = *reinterpret_cast<const float2*>(&sm.tok_e[b][8 * i + cl]);
          const float w0 = fmaf(__uint_as_float(s[4 * i]) * up.x, cq0, e.x);
          const float w1 = fmaf(__uint_as_float(s[4 * i + 1]) * up.y, cq0, e.y);
          const float w2 = fmaf(__uint_as_float(s[4 * i + 2]) * up.x, cq1, e.x);
          const float w3 = fmaf(__uint_as_float(s[4 * i + 3]) * up.y, cq1, e.y);
          mx0 = fmaxf(mx0, fmaxf(w0, w1));
          mx1 = fmaxf(mx1, fmaxf(w2, w3));
          s[4 * i] = __float_as_uint(w0);
          s[4 * i + 1] = __float_as_uint(w1);
          s[4 * i + 2] = __float_as_uint(w2);
          s[4 * i + 3] = __float_as_uint(w3);
        }
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) {
          mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, o));
          mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, o));
        }
        if (soft_any(mx0 > m0 + kLazy || mx1 > m1 + kLazy)) {  // m = -inf: any finite maximum
          const float n0 = fmaxf(m0, mx0), n1 = fmaxf(m1, mx1);
          const float x0 = m0 == n0 ? 1.f : ex2(m0 - n0), x1 = m1 == n1 ? 1.f : ex2(m1 - n1);
          l0 *= x0;
          l1 *= x1;
          m0 = n0;
          m1 = n1;
          if (started) {
            if ((lane & 3) == 0) {
              sm.factor[r0] = x0;
              sm.factor[r1] = x1;
            }
            mbar_wait(&sm.empty[(g - 1) & 1], ((g - 1) >> 1) & 1, abort, &g_hcu_status);  // O is complete so far
            named_bar(2, kSoftWarps * 32);
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < 8; ++c) {
              uint32_t o[32];
              tmem_ld_x32_sync(tmem + kTmemO + quad + 32 * c, o);
              const float4* f4 = reinterpret_cast<const float4*>(sm.factor + 32 * (c & 1));
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                const float4 f = f4[j];
                o[4 * j] = __float_as_uint(__uint_as_float(o[4 * j]) * f.x);
                o[4 * j + 1] = __float_as_uint(__uint_as_float(o[4 * j + 1]) * f.y);
                o[4 * j + 2] = __float_as_uint(__uint_as_float(o[4 * j + 2]) * f.z);
                o[4 * j + 3] = __float_as_uint(__uint_as_float(o[4 * j + 3]) * f.w);
              }
              tmem_st_x32(tmem + kTmemO + quad + 32 * c, o);
            }
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            named_bar(2, kSoftWarps * 32);  // factor may be written again
          }
        }
        const float b0 = m0 == -INFINITY ? 0.f : m0 - kBias, b1 = m1 == -INFINITY ? 0.f : m1 - kBias;
        const uint32_t pbase = smem_u32(sm.k[b]) + 8 * kChunkBytes + warp * 2048 + ((lane >> 3) & 1) * 1024 +
                               (lane & 7) * 128;
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
          uint32_t h[4];
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const float2 dn = *reinterpret_cast<const float2*>(&sm.tok_dn[b][8 * (i + k) + cl]);
            const float p0 = ex2(__uint_as_float(s[4 * (i + k)]) - b0), p1 = ex2(__uint_as_float(s[4 * (i + k) + 1]) - b0);
            const float p2 = ex2(__uint_as_float(s[4 * (i + k) + 2]) - b1),
                        p3 = ex2(__uint_as_float(s[4 * (i + k) + 3]) - b1);
            l0 = fmaf(p0, dn.x, l0);
            l0 = fmaf(p1, dn.y, l0);
            l1 = fmaf(p2, dn.x, l1);
            l1 = fmaf(p3, dn.y, l1);
            h[2 * k] = h2_bits(__floats2half2_rn(p0, p1));
            h[2 * k + 1] = h2_bits(__floats2half2_rn(p2, p3));
          }
          // matrices: (tokens 8 i.., heads r0), (.., heads r1), (tokens 8 (i + 1).., heads r0), (.., r1)
          const int unit = i + (lane >> 4);
          stmatrix_x4(pbase + ((unit ^ (lane & 7)) << 4), h[0], h[1], h[2], h[3]);
        }
        started = true;
        fence_async_shared();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.pready[b]);
      }

      const bool job_end = tile + 1 == p.tiles;
      if (job_end || g + 1 == n) {
        // ---- the segment's result
        const int64_t row = job / p.n_hg;
        const int h0 = static_cast<int>(job % p.n_hg) * kHg;
        const int nh = min(kHg, p.heads - h0);
        const bool whole = job_end && (g + 1 >= p.tiles);  // the segment began with the job's first tile
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) {
          l0 += __shfl_xor_sync(0xffffffffu, l0, o);
          l1 += __shfl_xor_sync(0xffffffffu, l1, o);
        }
        float* part = p.part + (static_cast<int64_t>(blockIdx.x) * 2 + (job == job0 ? 0 : 1)) * kPartFloats;
        if ((lane & 3) == 0) {
          sm.factor[r0] = l0 == 0.f ? 0.f : 1.f / l0;
          sm.factor[r1] = l1 == 0.f ? 0.f : 1.f / l1;
          const float z0 = l0 == 0.f ? -INFINITY : m0 - kBias + log2f(l0);
          const float z1 = l1 == 0.f ? -INFINITY : m1 - kBias + log2f(l1);
          if (whole) {
            if (r0 < nh) p.lse[row * p.heads + h0 + r0] = z0 * 0.6931471805599453f;
            if (r1 < nh) p.lse[row * p.heads + h0 + r1] = z1 * 0.6931471805599453f;
          } else {
            part[kHg * kLatentDim + r0] = z0;
            part[kHg * kLatentDim + r1] = z1;
          }
        }
        mbar_wait(&sm.empty[b], (g >> 1) & 1, abort, &g_hcu_status);  // the last product is complete
        named_bar(2, kSoftWarps * 32);
        tc_fence_after();
#pragma unroll 1
        for (int c = 0; c < 8; ++c) {  // 32 heads of 128 latent values
          const int hb = 32 * (c & 1);
          if (hb >= nh) continue;
          const int d = 128 * (c >> 1) + 32 * warp + lane;
          uint32_t o[32];
          if (started) {
            tmem_ld_x32_sync(tmem + kTmemO + quad + 32 * c, o);
          } else {
#pragma unroll
            for (int j = 0; j < 32; ++j) o[j] = 0;
          }
          const float4* f4 = reinterpret_cast<const float4*>(sm.factor + hb);
          if (whole) {
            // neighbouring lanes trade halves: each stores two adjacent values of one head
            uint16_t* dst = p.out + ((row * p.heads + h0 + hb + (lane & 1)) * kLatentDim + (d & ~1));
#pragma unroll
            for (int j = 0; j < 32; j += 4) {
              const float4 f = f4[j / 4];
              const float v0 = __uint_as_float(o[j]) * f.x, v1 = __uint_as_float(o[j + 1]) * f.y;
              const float v2 = __uint_as_float(o[j + 2]) * f.z, v3 = __uint_as_float(o[j + 3]) * f.w;
              const float t0 = __shfl_xor_sync(0xffffffffu, lane & 1 ? v0 : v1, 1);
              const float t1 = __shfl_xor_sync(0xffffffffu, lane & 1 ? v2 : v3, 1);
              const __nv_bfloat162 w0 = lane & 1 ? __floats2bfloat162_rn(t0, v1) : __floats2bfloat162_rn(v0, t0);
              const __nv_bfloat162 w1 = lane & 1 ? __floats2bfloat162_rn(t1, v3) : __floats2bfloat162_rn(v2, t1);
              if (hb + j + (lane & 1) < nh)
                *reinterpret_cast<__nv_bfloat162*>(dst + static_cast<int64_t>(j) * kLatentDim) = w0;
              if (hb + j + 2 + (lane & 1) < nh)
                *reinterpret_cast<__nv_bfloat162*>(dst + static_cast<int64_t>(j + 2) * kLatentDim) = w1;
            }
          } else {
            float* dst = part + hb * kLatentDim + d;
#pragma unroll
            for (int j = 0; j < 32; j += 4) {
              const float4 f = f4[j / 4];
              dst[j * kLatentDim] = __uint_as_float(o[j]) * f.x;
              dst[(j + 1) * kLatentDim] = __uint_as_float(o[j + 1]) * f.y;
              dst[(j + 2) * kLatentDim] = __uint_as_float(o[j + 2]) * f.z;
              dst[(j + 3) * kLatentDim] = __uint_as_float(o[j + 3]) * f.w;
            }
          }
        }
        tc_fence_before();
        named_bar(2, kSoftWarps * 32);  // factor may be written again
        if (lane == 0) mbar_arrive(&sm.oempty);
        ++seg;
      }
      if (++tile == p.tiles) {
        tile = 0;
        ++job;
      }
    }
  }

  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

// Joins the partial results of a job that several CTAs shared: weights 2^(lse_i - max).  Block
// (c - 1, h): the job at the boundary between CTAs c - 1 and c, if that is the job's first boundary.
__global__ __launch_bounds__(128) void combine_kernel(const AttnArgs p, int grid) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int c = blockIdx.x + 1, h = blockIdx.y;
  const int64_t at = first_tile(p.total, c, grid);
  const int64_t job = at / p.tiles;
  const int64_t begin = job * p.tiles, end = begin + p.tiles;
  if (at == begin || first_tile(p.total, c - 1, grid) > begin) return;
  const int64_t row = job / p.n_hg;
  const int head = static_cast<int>(job % p.n_hg) * kHg + h;
  if (head >= p.heads) return;
  const auto part_of = [&](int cta) {
    const int slot = first_tile(p.total, cta, grid) / p.tiles == job ? 0 : 1;
    return p.part + (static_cast<int64_t>(cta) * 2 + slot) * kPartFloats;
  };
  float m = -INFINITY;
  for (int i = c - 1; i < grid && first_tile(p.total, i, grid) < end; ++i)
    m = fmaxf(m, part_of(i)[kHg * kLatentDim + h]);
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  float l = 0.f;
  for (int i = c - 1; m != -INFINITY && i < grid && first_tile(p.total, i, grid) < end; ++i) {
    const float* q = part_of(i);
    const float w = exp2f(q[kHg * kLatentDim + h] - m);
    const float4 v = *reinterpret_cast<const float4*>(q + h * kLatentDim + 4 * threadIdx.x);
    l += w;
    o.x = fmaf(w, v.x, o.x);
    o.y = fmaf(w, v.y, o.y);
    o.z = fmaf(w, v.z, o.z);
    o.w = fmaf(w, v.w, o.w);
  }
  const float f = l == 0.f ? 0.f : 1.f / l;
  const __nv_bfloat162 a = __floats2bfloat162_rn(o.x * f, o.y * f), b = __floats2bfloat162_rn(o.z * f, o.w * f);
  const int64_t rh = row * p.heads + head;
  *reinterpret_cast<uint2*>(p.out + rh * kLatentDim + 4 * threadIdx.x) =
      make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
  if (threadIdx.x == 0) p.lse[rh] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
}

int attn_grid(int64_t total) {
  const int64_t sms = sm_count();
  return static_cast<int>(total < sms ? total : sms);
}

int64_t tiles_of(int64_t n_tokens) { return n_tokens <= 0 ? 1 : (n_tokens + kTile - 1) / kTile; }

template <bool kFp4, bool kBlocks>
int launch_attn(const AttnArgs& a, int grid, cudaStream_t st) {
  constexpr int smem = static_cast<int>(sizeof(AtSmem)) + 1024;
  cudaError_t e = cudaFuncSetAttribute(sparse_mla_kernel<kFp4, kBlocks>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) {
    set_last_error(e);
    return HCU_ERR_LAUNCH;
  }
  sparse_mla_kernel<kFp4, kBlocks><<<grid, kAtThreads, smem, st>>>(a);
  bool split = false;
  for (int c = 1; c < grid && !split; ++c) split = (a.total * c / grid) % a.tiles != 0;
  if (split) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(grid - 1), static_cast<unsigned>(a.heads < kHg ? a.heads : kHg));
    cfg.blockDim = dim3(128);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cudaLaunchKernelEx(&cfg, combine_kernel, a, grid);
  }
  return launch_status();
}

}  // namespace
}  // namespace hcu

extern "C" int64_t hcu_sparse_mla_attention_workspace_bytes(int64_t rows, int64_t heads, int64_t n_tokens) {
  using namespace hcu;
  if (rows < 0 || heads < 0 || n_tokens < 0) return -1;
  const int64_t total = rows * ((heads + kHg - 1) / kHg) * tiles_of(n_tokens);
  return static_cast<int64_t>(attn_grid(total)) * 2 * kPartFloats * static_cast<int64_t>(sizeof(float));
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
  if (heads > 1024 || rows > kMaxInt / 1024 || n_bt > kMaxInt / kPage || n_slots > kMaxInt) return HCU_ERR_UNSUPPORTED;
  if (!q || !out || !lse || !workspace || (n_idx > 0 && (!indices || !kv_cache))) return HCU_ERR_ARG;
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(kv_cache) | reinterpret_cast<uintptr_t>(out) |
       reinterpret_cast<uintptr_t>(workspace)) %
      16)
    return HCU_ERR_ARG;
  const int64_t n_tokens = blocks ? n_idx * kPage : n_idx;
  if (workspace_bytes < hcu_sparse_mla_attention_workspace_bytes(rows, heads, n_tokens)) return HCU_ERR_ARG;
  AttnArgs a{};
  a.q = q;
  a.q_row = q_row;
  a.q_head = q_head;
  a.kv = kv_cache;
  a.n_slots = n_slots;
  a.slot_stride = slot_stride;
  a.idx = indices;
  a.idx_stride = idx_stride;
  a.n_idx = static_cast<int>(n_idx);
  a.bt = block_table;
  a.bt_stride = bt_stride;
  a.n_bt = static_cast<int>(n_bt);
  a.lengths = lengths;
  a.sm_scale = sm_scale;
  a.heads = static_cast<int>(heads);
  a.n_hg = static_cast<int>((heads + kHg - 1) / kHg);
  a.tiles = static_cast<int>(tiles_of(n_tokens));
  a.total = rows * a.n_hg * a.tiles;
  a.out = out;
  a.lse = lse;
  a.part = static_cast<float*>(workspace);
  const int grid = attn_grid(a.total);
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (fp4) return blocks ? launch_attn<true, true>(a, grid, st) : launch_attn<true, false>(a, grid, st);
  return blocks ? launch_attn<false, true>(a, grid, st) : launch_attn<false, false>(a, grid, st);
}
