// Attention of MLA queries over selected tokens of a paged latent cache (sm_100a tensor cores).
//
//   s[h, t] = sm_scale * sum_d q[h, d] * k[t, d]     d < 576: 512 latent, 64 rope
//   out[h]  = sum_t softmax(s[h])[t] * k[t, :512],   lse[h] = log sum_t exp(s[h, t])
// over the tokens of the row's list: slots (token form), or the visible tokens of chosen 64-token
// blocks (block form).
//
// Work: a job is (row, group of up to 64 heads), cut into tiles of 48 candidates.  The flat list of
// all tiles is split evenly over one persistent CTA per SM, or job by job where that costs less; a
// CTA's share of one job is a segment.  A segment that is the whole job writes the result, any other
// one a partial (out, lse) that combine_kernel joins.  Per tile:
//   * the gather warp looks the candidates up three tiles ahead, asks their slots into L2 two tiles
//     ahead, and copies them into the raw buffer, four slots per TMA gather;
//   * 6 loader warps (one 8-token swizzle group each) read the raw slots, convert them to f16 in
//     registers, which frees the raw buffer, and store them as the tile's K once a K buffer is free: 9
//     chunks of [48 tokens][64 values], rows of 128 bytes, 128-byte swizzle; for fp8 slots a tenth, the
//     rope's second operand, whose one buffer is free, and filled, earlier: once the last tile's S is there.
//     A chunk is a K-major operand for q k^T and, read the other way, an MN-major one for v^T, so the
//     latent is stored once;
//   * 4 warps bring each segment's Q in as f16: two chunks to TMEM, seven to shared memory;
//   * the MMA thread issues S = Q K^T (M = 64 heads, N = 48 tokens, K = 576) and, up to two tiles
//     behind, O^T += V^T P^T (M = 128 latent values x 4, N = heads, K = 48 tokens): with the latent as M
//     the second product runs at the full rate, and O^T takes 4 x 64 TMEM columns;
//   * 4 softmax warps (16 heads each) read S, keep the running maximum and sum in fp32 and write P
//     in f16 over the tile's rope chunk, which S no longer needs.  O^T is rescaled only when a
//     maximum has risen by more than 2^kLazy.
// 48 tokens: Q (57 KB), two K tiles (55 KB each), three more P (18 KB, below), a tenth chunk (6 KB) and the raw
// slots (34 KB) fill the 227 KB; with 4-bit slots (one P, 23 KB of raw slots) 32 KB are free.
//
// Number format.  f16 operands hold 11 bits where bf16 holds 8, and an fp8 or e2m1 value is exact in
// f16; its range is met by powers of two taken out per token and per query row:
//   * token t: 2^E, E from its largest scale; latent codes are multiplied by scale * 2^-E and the rope by
//     2^-E 2^-10; E is raised where the rope would leave f16's range (latents 2^-35 below the rope);
//   * query row: 2^e, its largest element just below 2^4 (latent part) or 2^14 (rope part, which
//     takes the 2^10 back), so elements down to 2^-18 of the largest keep all their bits.
// Nothing of a 4-bit slot is rounded: its token scale is a power of two, code * group scale six bits.  An
// fp8 group's scale has 24, and rounded products put lse of 33 tokens 5e-5 of itself off.  So scales are
// rounded to 7 bits, whose products with a value's 4 are exact, and what a scale is of its rounding,
// r = 1 +- 2^-8, is put in where a group's sums are: S has a part per 128-value group, s = sum_g r_g S_g in
// fp32, and block g of O^T takes P r_g, a P of its own.  The rope joins S_3 as two operands that make rope / r_3:
// the rope, exact, and rope * (1 / r_3 - 1), at most 2^-7 of it and rounded (2^-18 of the rope; the quotient
// as one operand, rounded by 2^-12, put lse of 33 tokens 8e-6 off).  lse of 33 tokens is 1.3e-7 of itself off,
// of 2048 tokens 7e-8, as with 4-bit slots.  A scale that is not finite is not rounded: its NaN or infinity goes
// through the products into the row.
//
// S * 2^(E + e) is the score; P carries 2^E of its token in its exponent (w = s + E, whose maximum is
// the running one), so O needs no correction, and the sum takes 2^-E back per token.
//
// Bound.  A 48-token fp8 tile needs 1340 cycles of the tensor pipe (960 for S, whose M of 64 fills half of
// it, 380 for O) and about 2700 of the shared-memory port at 128 B per cycle (34 KB of raw slots in and
// out, 61 KB of K and 24 KB of P in, 124 KB of Q and K operands for S, 72 KB of V and P for O); it takes
// 4100.  What is left is the chain of a tile through its warps (copy 2900, convert 650, store 1000,
// S 960, softmax 1250 with one P, O 380 cycles), with two K tiles and one of raw slots to overlap it.  Both
// were traded, with one P: a third K tile took 7 % longer, a second raw buffer 11 %, copies of 16 bytes from
// the loader warps in place of the raw ring 14 to 19 %.  2048 rows x 64 heads x 2048 fp8 tokens (584 GFLOP)
// take 1.27 ms, 460 TFLOP/s (1.015 ms with rounded scales, one S and one P); 128 rows 103 us; one row 28 us;
// 192 rows of 4-bit slots 136 us.  L2 flushed before each call; in a graph of launches 1.26 ms, 96, 21 and 129 us.
#include <cudaTypedefs.h>
#include <cuda_bf16.h>

#include <mutex>
#include <type_traits>

#include "common.cuh"
#include "mla_slots.cuh"

HCU_DEFINE_STATUS(status_sparse_mla)

namespace hcu {
namespace {

constexpr int kTile = 48;        // candidates per tile
constexpr int kHg = 64;          // heads per job
constexpr int kChunks = kQkDim / 64;
constexpr int kQChunk = kHg * 128;     // [64 heads][64 f16]
constexpr int kChunk = kTile * 128;    // [48 tokens][64 f16]
constexpr int kTileBytes = kChunks * kChunk;
constexpr int kPBytes = kTile * kHg * 2;
constexpr int kQTmem = 2;              // chunks of Q in TMEM, the others in shared memory
constexpr int kRawFp8 = 704, kRawFp4 = 480;  // a slot's row in the raw buffer (see Raw), the slot padded with zeros
constexpr int kSoftWarps = 4;
constexpr int kMmaWarp = kSoftWarps;
constexpr int kGatherWarp = kMmaWarp + 1;
constexpr int kQWarp = kGatherWarp + 1;
constexpr int kQWarps = 4;
constexpr int kLoadWarp = kQWarp + kQWarps;
constexpr int kLoadWarps = kTile / 8;
constexpr int kAtThreads = (kLoadWarp + kLoadWarps) * 32;
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kTmemO = 0;    // 4 blocks of 128 latent values x 64 heads
constexpr uint32_t kTmemS = 256;  // fp8: 4 score parts of 48 columns; 4-bit: 2 score buffers, 64 apart
constexpr uint32_t kTmemQ = 448;  // 32 columns a chunk
// P is 2^(w - m + kBias), m the row's maximum when it was last taken: the largest weight is 2^8 then,
// 2^15 while the maximum has grown by the tolerated 2^kLazy (scores of a row with a spread of 2.2 in
// base 2 hardly ever rise by 7 over their first 48's maximum), and weights down to 2^-22 of the
// largest are normal f16 numbers.
constexpr float kLazy = 7.f;
constexpr float kBias = 8.f;
constexpr int kRopeShift = 10;
constexpr int kPartFloats = kHg * kLatentDim + kHg;

// What the scales of fp8 slots need beside the tile.  Output rows on their way out (kSoftWarps KB) have the first
// bytes, of P where there is one: a segment's last product has read it by then, its writers are the same warps.
template <bool kFp4>
struct Groups {
  uint8_t p[3][kPBytes];   // P of groups 1 to 3 (of group 0, as the only P of 4-bit slots: the tile's rope chunk)
  uint8_t rest[kChunk];    // the rope's second operand
  float4 tok_r[2][kTile];  // what each group's scale is of its 7-bit rounding
};
template <>
struct Groups<true> {
  uint8_t stage[kSoftWarps * 1024];
};

template <bool kFp4>
struct __align__(1024) AtSmem {
  uint8_t q[(kChunks - kQTmem) * kQChunk];
  uint8_t k[2][kTileBytes];
  __align__(1024) Groups<kFp4> grp;
  // slots of the tile to be converted next, as they are in the cache
  __align__(128) uint8_t raw[kTile * (kFp4 ? kRawFp4 : kRawFp8)];
  float tok_e[2][kTile];    // E of each token (-inf: no token)
  float tok_up[2][kTile];   // 2^E (0: no token)
  float tok_dn[2][kTile];   // 2^-E (0: no token)
  float cq[4][kHg];         // per segment and head: 2^e * sm_scale * log2(e)
  float factor[kHg];        // rescale of O, then 1 / sum
  uint32_t mask[2];         // candidates in raw that are tokens
  int empty_tile[2];        // the tile in buffer b holds no token
  uint64_t full[2], empty[2], sfull[2], pready[2];
  uint64_t rfull, rempty, sempty, qfull, qempty, oempty, done;
  uint32_t tmem;
  int abort;
};
static_assert(sizeof(AtSmem<false>) + 1024 <= 232448 && sizeof(AtSmem<true>) + 1024 <= 232448, "shared memory");

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
  int quantum;    // a CTA's share is a multiple of this many tiles: 1, or a job's
  uint16_t* out;
  float* lse;
  float* part;    // [grid][2][kPartFloats]
};

__host__ __device__ __forceinline__ int64_t first_tile(const AttnArgs& p, int cta, int grid) {
  return p.total / p.quantum * cta / grid * p.quantum;
}

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

// The same with A in TMEM.
__device__ __forceinline__ void mma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
                                           uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
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
  d |= static_cast<uint64_t>(kChunk >> 4) << 16;  // leading offset: next 64 M values
  d |= static_cast<uint64_t>(1024 >> 4) << 32;         // stride offset: next 8 K rows
  d |= static_cast<uint64_t>(1) << 46;
  d |= static_cast<uint64_t>(2) << 61;
  return d;
}

// K-major operand in rows of 32 bytes (16 K values) with the 32-byte swizzle, 8 rows per 256 bytes.
__device__ __forceinline__ uint64_t sw32_kmajor_desc(uint32_t smem_addr) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((smem_addr & 0x3FFFFu) >> 4);
  d |= static_cast<uint64_t>(1) << 16;          // leading offset (unused: one 32-byte row of K)
  d |= static_cast<uint64_t>(256 >> 4) << 32;   // stride offset: next 8 rows
  d |= static_cast<uint64_t>(1) << 46;
  d |= static_cast<uint64_t>(6) << 61;
  return d;
}

// 16 lanes x 48 columns, as 6 column groups of an 8x8-pair fragment: thread t holds, for group n, rows
// t / 4 (r[4n], r[4n + 1]) and t / 4 + 8 (r[4n + 2], r[4n + 3]), columns 8n + 2 (t % 4) + {0, 1}.
__device__ __forceinline__ void tmem_ld_scores(uint32_t taddr, uint32_t (&r)[24]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15}, [%24];\n\t"
      "tcgen05.ld.sync.aligned.16x256b.x2.b32 {%16, %17, %18, %19, %20, %21, %22, %23}, [%25];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]),
        "=r"(r[23])
      : "r"(taddr), "r"(taddr + 32)
      : "memory");
}

// The same of 32 columns.
__device__ __forceinline__ void tmem_ld_16x256_x4(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15}, [%16];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
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

__device__ __forceinline__ void tmem_st_16x256_x8(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.16x256b.x8.b32 [%32], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, "
      "%14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};" ::"r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]),
      "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]),
      "r"(r[29]), "r"(r[30]), "r"(r[31]), "r"(taddr)
      : "memory");
}

// The four score parts' columns of 16 tokens: r[g] as tmem_ld_scores' first 8 of part g.
__device__ __forceinline__ void tmem_ld_parts(uint32_t taddr, uint32_t (&r)[4][8]) {
#pragma unroll
  for (int g = 0; g < 4; ++g)
    asm volatile("tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(r[g][0]), "=r"(r[g][1]), "=r"(r[g][2]), "=r"(r[g][3]), "=r"(r[g][4]), "=r"(r[g][5]),
                   "=r"(r[g][6]), "=r"(r[g][7])
                 : "r"(taddr + kTile * g)
                 : "memory");
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0][0]), "+r"(r[0][1]), "+r"(r[0][2]), "+r"(r[0][3]), "+r"(r[0][4]), "+r"(r[0][5]),
                 "+r"(r[0][6]), "+r"(r[0][7]), "+r"(r[1][0]), "+r"(r[1][1]), "+r"(r[1][2]), "+r"(r[1][3]),
                 "+r"(r[1][4]), "+r"(r[1][5]), "+r"(r[1][6]), "+r"(r[1][7])
               :
               : "memory");
  asm volatile(""
               : "+r"(r[2][0]), "+r"(r[2][1]), "+r"(r[2][2]), "+r"(r[2][3]), "+r"(r[2][4]), "+r"(r[2][5]),
                 "+r"(r[2][6]), "+r"(r[2][7]), "+r"(r[3][0]), "+r"(r[3][1]), "+r"(r[3][2]), "+r"(r[3][3]),
                 "+r"(r[3][4]), "+r"(r[3][5]), "+r"(r[3][6]), "+r"(r[3][7])
               :
               : "memory");
}

__device__ __forceinline__ void stmatrix_x4(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c),
               "r"(d)
               : "memory");
}

__device__ __forceinline__ void stmatrix_x4_trans(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b),
               "r"(c), "r"(d)
               : "memory");
}

// 16-byte piece `part` of row h in rows of 32 bytes with the 32-byte swizzle: the pieces of every
// other group of four rows swapped, so that eight rows' pieces fall into different banks.
__device__ __forceinline__ int st_piece(int h, int part) { return h * 32 + ((part ^ ((h >> 2) & 1)) << 4); }

__device__ __forceinline__ uint4 ld_shared_v4(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

template <int kOffset = 0>
__device__ __forceinline__ void st_shared_v4(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0 + %5], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d), "n"(kOffset)
               : "memory");
}

// f(0), .., f(7) with the index as a constant.
template <typename F>
__device__ __forceinline__ void unroll8(F&& f) {
  f(std::integral_constant<int, 0>());
  f(std::integral_constant<int, 1>());
  f(std::integral_constant<int, 2>());
  f(std::integral_constant<int, 3>());
  f(std::integral_constant<int, 4>());
  f(std::integral_constant<int, 5>());
  f(std::integral_constant<int, 6>());
  f(std::integral_constant<int, 7>());
}

__device__ __forceinline__ void fence_async_shared() {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Whether the phase of the given parity has completed (no wait).
__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred P;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 P, [%1], %2;\n\t"
      "selp.b32 %0, 1, 0, P;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}

__device__ __forceinline__ uint32_t pack2(float2 v) {
  const __half2 h = __floats2half2_rn(v.x, v.y);
  return *reinterpret_cast<const uint32_t*>(&h);
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

__device__ __forceinline__ uint2 ld_shared_v2(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t ld_shared_u32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t ldg_u32(const void* p) {
  uint32_t v;
  asm volatile("ld.global.nc.u32 %0, [%1];" : "=r"(v) : "l"(p));
  return v;
}
// The same rows into L2 only.
__device__ __forceinline__ void tma_prefetch4(const CUtensorMap* map, int r0, int r1, int r2, int r3) {
  asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile::gather4 [%0, {%1, %2, %3, %4, %5}];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(0), "r"(r0), "r"(r1), "r"(r2), "r"(r3)
               : "memory");
}
// Asynchronous copy of four slots (rows of the map, one row per box) into consecutive rows of shared
// memory; a row out of range (-1) and the box's bytes past the slot are filled with zeros.
__device__ __forceinline__ void tma_gather4(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int r0, int r1, int r2,
                                            int r3) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes [%0], "
      "[%1, {%3, %4, %5, %6, %7}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(0), "r"(r0), "r"(r1), "r"(r2), "r"(r3)
      : "memory");
}

// ---------------------------------------------------------------- gather
// Lane l < 12 of the gather warp looks up candidates 4 l .. 4 l + 3 of each tile, in stages a tile apart
// so that no load waits for the one that names it: list entries, then (block form) the page and the
// row's length.  What a stage loads is not touched before the next one (a select on it would wait for
// it): places past the list's end or the CTA's range read some entry of it and are marked instead.
constexpr int kGatherLanes = kTile / 4;
struct Entry {
  int32_t v[4];  // list entries: slots, or blocks
  int in;        // bit i: v[i] lies in the list
};
struct Place {
  int32_t v[4];    // token form: slots; block form: pages
  int32_t len;     // block form: the row's length
  int32_t pos[4];  // block form: the candidates' positions in the row
  int in;          // bit i: a candidate; bit 4 + i: its block lies past the table
};

template <bool kBlocks>
__device__ __forceinline__ Entry load_entry(const AttnArgs& p, int64_t row, int tile, int lane, bool on) {
  Entry e;
  const int32_t* p0 = p.idx + (on ? row : 0) * p.idx_stride;
  const int last = on && lane < kGatherLanes ? p.n_idx - 1 : -1;
  e.in = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    int j = tile * kTile + 4 * lane + i;
    if constexpr (kBlocks) j /= kPage;
    e.v[i] = static_cast<int32_t>(ldg_u32(p0 + max(min(j, last), 0)));
    e.in |= j <= last ? 1 << i : 0;
  }
  return e;
}

template <bool kBlocks>
__device__ __forceinline__ Place load_place(const AttnArgs& p, int64_t row, int tile, int lane, const Entry& e) {
  Place c;
  c.in = e.in;
  c.len = kBlocks ? static_cast<int32_t>(ldg_u32(p.lengths + (e.in ? row : 0))) : 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    c.v[i] = e.v[i];
    if constexpr (kBlocks) {
      const bool on = (e.in >> i & 1) && e.v[i] >= 0;
      c.pos[i] = on ? e.v[i] * kPage + (tile * kTile + 4 * lane + i) % kPage : 0;
      c.v[i] = static_cast<int32_t>(
          ldg_u32(p.bt + (on ? row : 0) * p.bt_stride + max(min(on ? e.v[i] : 0, p.n_bt - 1), 0)));
      c.in = (c.in & ~(1 << i)) | (on ? 1 << i : 0) | (on && e.v[i] >= p.n_bt ? 16 << i : 0);
    }
  }
  return c;
}

// Slot of candidate i of the lane, -1: none.
template <bool kBlocks>
__device__ __forceinline__ int32_t resolve(const AttnArgs& p, const Place& c, int i) {
  if (!(c.in >> i & 1)) return -1;
  int64_t s = c.v[i];
  bool bad;
  if constexpr (kBlocks) {
    if (c.pos[i] >= c.len) return -1;
    s = s * kPage + c.pos[i] % kPage;
    bad = (c.in >> (4 + i) & 1) || c.v[i] < 0 || s >= p.n_slots;
  } else {
    if (s < 0) return -1;
    bad = s >= p.n_slots;
  }
  if (bad) atomicOr(&g_hcu_status, HCU_STATUS_BAD_INPUT);
  return bad ? -1 : static_cast<int32_t>(s);
}

// ---------------------------------------------------------------- loader
// Lane l of loader warp lw owns a quarter (sub = l % 4) of token 8 lw + l / 4: latent elements
// 64 i + 16 sub .. + 15 of every chunk i and rope elements 16 sub .. + 15.  A quarter warp's two tokens
// fall into different halves of the swizzle, so the converted 16-byte pieces store without bank
// conflicts, all addresses are one register plus constants, and scales stay in their own lane; the raw
// rows' strides (704 and 480 bytes) put the same lanes' raw pieces into different banks too.
template <bool kFp4>
struct Raw {
  uint4 x[8];   // fp8 codes
  uint2 y[8];   // e2m1 codes
  uint4 gs[2];  // 4-bit: the token's 32 e4m3 scales
  uint4 sc;     // fp8: the token's 4 group scales; 4-bit: .x the token scale
  uint4 rope[2];
};

template <bool kFp4>
__device__ __forceinline__ void read_raw(uint32_t row, int sub, Raw<kFp4>& r) {
  if constexpr (kFp4) {
    r.gs[0] = ld_shared_v4(row + kKv4Scales);
    r.gs[1] = ld_shared_v4(row + kKv4Scales + 16);
    r.sc.x = ld_shared_u32(row + kKv4Token);
  } else {
    r.sc = ld_shared_v4(row + kFp8Scales);
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) r.rope[i] = ld_shared_v4(row + (kFp4 ? kKv4Rope : kFp8Rope) + 32 * sub + 16 * i);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if constexpr (kFp4)
      r.y[i] = ld_shared_v2(row + 32 * i + 8 * sub);
    else
      r.x[i] = ld_shared_v4(row + 64 * i + 16 * sub);
  }
}

// bf16 pair (packed) * f -> f16 pair.
__device__ __forceinline__ uint32_t bf2_to_h2(uint32_t w, float f) {
  return h2_bits(__floats2half2_rn(__uint_as_float(w << 16) * f, __uint_as_float(w & 0xffff0000u) * f));
}

// Largest magnitude among 8 packed bf16 values, per half word.
__device__ __forceinline__ __nv_bfloat162 amax8(const uint4& v) {
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&v);
  return __hmax2(__hmax2(__habs2(h[0]), __habs2(h[1])), __hmax2(__habs2(h[2]), __habs2(h[3])));
}
// Biased exponent of the larger half of a non-negative pair (255: inf or nothing but NaN).
__device__ __forceinline__ int exponent2(__nv_bfloat162 m) {
  const uint32_t w = *reinterpret_cast<const uint32_t*>(&m);
  return static_cast<int>(max(w & 0x7fffu, w >> 16 & 0x7fffu) >> 7);
}

__device__ __forceinline__ float exp2_of(int biased) { return __uint_as_float(static_cast<uint32_t>(biased) << 23); }

// Q of a job, 16 heads a warp: lane l owns a quarter (sub = l % 4) of heads l / 4 and l / 4 + 8 of them.
// The first two chunks go to TMEM as fragments of 8 columns (16 values), values 16 j + 4 sub .. + 3 of both
// heads for step j, from registers (fetch_q); the others straight to their places in the Q buffer as
// bf16, 14 pieces of 16 bytes a head and lane (copy_q), converted in place once they are there.
// cq[h] is the head's factor from the product to the score in base 2.
constexpr int kQPieces = 2 * (kChunks - kQTmem);  // a lane's, per head

__device__ __forceinline__ const uint16_t* q_head(const AttnArgs& p, int64_t row, int h) {
  // a head past the last reads head 0: rows of S and columns of O are independent, and its are not stored
  return p.q + row * p.q_row + (h < p.heads ? h * p.q_head : 0);
}

__device__ __forceinline__ uint32_t q_piece(uint32_t base, int h, int u) {
  return base + h * 128 + (u >> 3) * kQChunk + (((u & 7) ^ (h & 7)) << 4);
}

__device__ __forceinline__ uint2 ldg_v2(const void* p) {
  uint2 v;
  asm volatile("ld.global.nc.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
  return v;
}

__device__ __forceinline__ void fetch_q(const uint16_t* q, int sub, uint2 (&v)[8]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = ldg_v2(q + 16 * j + 4 * sub);
}

__device__ __forceinline__ void copy_q(const uint16_t* q, uint32_t dst, int h, int sub) {
#pragma unroll
  for (int i = 0; i < kQPieces; ++i)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(q_piece(dst, h, sub + 4 * i)),
                 "l"(q + 64 * kQTmem + 8 * (sub + 4 * i))
                 : "memory");
}

// Returns the factor of the head's latent part.
__device__ __forceinline__ float convert_q(const AttnArgs& p, uint32_t q, float* cq, int h, int sub, const uint2 (&t)[8]) {
  uint4 v[kQPieces];
#pragma unroll
  for (int i = 0; i < kQPieces; ++i) v[i] = ld_shared_v4(q_piece(q, h, sub + 4 * i));
  __nv_bfloat162 am = amax8(v[0]);
#pragma unroll
  for (int i = 1; i < kQPieces; ++i) am = __hmax2(am, amax8(v[i]));
#pragma unroll
  for (int j = 0; j < 8; j += 2) am = __hmax2(am, amax8(make_uint4(t[j].x, t[j].y, t[j + 1].x, t[j + 1].y)));
  int eb = exponent2(am);
  eb = max(eb, __shfl_xor_sync(0xffffffffu, eb, 1));
  eb = max(eb, __shfl_xor_sync(0xffffffffu, eb, 2));
  eb = min(max(eb, 20), 240);  // where the factors below are normal floats
  const float f_lat = exp2_of(254 - eb + 3);    // the largest into [2^3, 2^4)
  const float f_rope = exp2_of(254 - eb + 13);  // 2^10 more
#pragma unroll
  for (int i = 0; i < kQPieces; ++i) {
    const float f = i < kQPieces - 2 ? f_lat : f_rope;
    st_shared_v4(q_piece(q, h, sub + 4 * i), bf2_to_h2(v[i].x, f), bf2_to_h2(v[i].y, f), bf2_to_h2(v[i].z, f),
                 bf2_to_h2(v[i].w, f));
  }
  if (sub == 0) cq[h] = p.sm_scale * 1.4426950408889634f * exp2_of(eb - 3);
  return f_lat;
}

// A lane's converted share of a tile, held in registers until the tile's buffer is free.
struct Conv {
  uint32_t y[8][8];  // latent elements 64 i + 16 sub .. + 15, two f16 a word
  uint32_t r[8];     // rope
  uint32_t dr;       // fp8: 1 / r_3 - 1, twice; 0 (no second operand) beside an infinite rope, which it could make a NaN
  int eb;            // biased exponent taken out of the token
  float rest;        // fp8: group sub's scale over its rounding
};

template <bool kFp4>
__device__ __forceinline__ void convert(const Raw<kFp4>& r, int sub, Conv& c) {
  int re = exponent2(__hmax2(amax8(r.rope[0]), amax8(r.rope[1])));
  re = max(re, __shfl_xor_sync(0xffffffffu, re, 1));
  re = max(re, __shfl_xor_sync(0xffffffffu, re, 2));
  uint32_t smax = r.sc.x & 0x7fffffffu;
  if constexpr (!kFp4)
    smax = max(max(smax, r.sc.y & 0x7fffffffu), max(r.sc.z & 0x7fffffffu, r.sc.w & 0x7fffffffu));
  // A token of zeros may take any E: 2^-64, so that its 2^-E counts into the sum of a list of any length (2^-100 with
  // P's 2^kBias overflows it at 2^20 tokens) and its weight is no flushed one beside tokens of large latents.
  bool zero = re == 0;
  if constexpr (kFp4)
    zero = zero && (smax == 0 || ((r.gs[0].x | r.gs[0].y | r.gs[0].z | r.gs[0].w | r.gs[1].x | r.gs[1].y | r.gs[1].z |
                                   r.gs[1].w) & 0x7f7f7f7fu) == 0);
  else
    zero = zero && smax == 0;
  c.eb = min(max(max(static_cast<int>(smax >> 23), re - 13 - kRopeShift), zero ? 63 : 27), 247);
  const float dn = exp2_of(254 - c.eb);
  const float fr = dn * (1.f / (1 << kRopeShift));
  __half2 scale[4];
  if constexpr (!kFp4) {
    // scales to 7 bits, so that their products with an fp8 value's 4 are exact in f16's 11
    const uint32_t w[4] = {r.sc.x, r.sc.y, r.sc.z, r.sc.w};
    float f = 0.f, h = 0.f;  // group sub's scale and its rounding
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const float x = __uint_as_float(w[g]) * dn;
      // the rounding's carry would make a zero of a NaN: what is not finite stays
      const uint32_t xb = __float_as_uint(x), xr = (xb + 0x10000u) & 0xfffe0000u;
      scale[g] = __float2half2_rn(__uint_as_float((~xb & 0x7f800000u) == 0 ? xb : xr));
      f = g == sub ? x : f;
      h = g == sub ? __low2float(scale[g]) : h;
    }
    c.rest = h != 0.f ? __fdividef(f, h) : 1.f;  // h is 0 where the group is 2^-25 of the token's largest
    const float r3 = __shfl_sync(0xffffffffu, c.rest, (threadIdx.x & 31) | 3);
    c.dr = re == 255 ? 0u : h2_bits(__float2half2_rn(__fdividef(1.f - r3, r3)));
  }
  const uint32_t rw[8] = {r.rope[0].x, r.rope[0].y, r.rope[0].z, r.rope[0].w,
                          r.rope[1].x, r.rope[1].y, r.rope[1].z, r.rope[1].w};
#pragma unroll
  for (int i = 0; i < 8; ++i) c.r[i] = bf2_to_h2(rw[i], fr);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if constexpr (kFp4) {
      const uint4 g = r.gs[i >> 2];
      const uint32_t w = (i & 3) == 0 ? g.x : (i & 3) == 1 ? g.y : (i & 3) == 2 ? g.z : g.w;
      const __half2 s =
          __float2half2_rn(e4m3_to_float(static_cast<uint8_t>(w >> (8 * sub))) * (__uint_as_float(r.sc.x) * dn));
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        c.y[i][k] = h2_bits(__hmul2(e2m1x2_to_half2((r.y[i].x >> (8 * k)) & 0xff), s));
        c.y[i][4 + k] = h2_bits(__hmul2(e2m1x2_to_half2((r.y[i].y >> (8 * k)) & 0xff), s));
      }
    } else {
      const __half2 s = scale[i >> 1];
      const uint32_t x[4] = {r.x[i].x, r.x[i].y, r.x[i].z, r.x[i].w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        c.y[i][2 * k] = h2_bits(__hmul2(e4m3x2_to_half2(x[k] & 0xffffu), s));
        c.y[i][2 * k + 1] = h2_bits(__hmul2(e4m3x2_to_half2(x[k] >> 16), s));
      }
    }
  }
}

// Stores the warp's 8 tokens as rows 8 lw .. 8 lw + 7 of tile buffer b; on: the lane's token exists.
template <bool kFp4>
__device__ __forceinline__ void store_tile(AtSmem<kFp4>& sm, int b, int lw, int lane, bool on, const Conv& c) {
  const int tok = lane >> 2, sub = lane & 3;
  if constexpr (!kFp4) reinterpret_cast<float*>(&sm.grp.tok_r[b][lw * 8 + tok])[sub] = c.rest;
  if (sub == 0) {
    const int t = lw * 8 + tok;
    sm.tok_e[b][t] = on ? static_cast<float>(c.eb - 127) : -INFINITY;
    sm.tok_up[b][t] = on ? exp2_of(c.eb) : 0.f;
    sm.tok_dn[b][t] = on ? exp2_of(254 - c.eb) : 0.f;
  }
  // 16-byte pieces 2 sub and 2 sub + 1 of the token's row in every chunk
  const uint32_t p0 = smem_u32(sm.k[b]) + lw * 1024 + tok * 128 + (((2 * sub) ^ tok) << 4), p1 = p0 ^ 16u;
  unroll8([&](auto I) {
    constexpr int i = decltype(I)::value;
    st_shared_v4<i * kChunk>(p0, c.y[i][0], c.y[i][1], c.y[i][2], c.y[i][3]);
    st_shared_v4<i * kChunk>(p1, c.y[i][4], c.y[i][5], c.y[i][6], c.y[i][7]);
  });
  st_shared_v4<8 * kChunk>(p0, c.r[0], c.r[1], c.r[2], c.r[3]);
  st_shared_v4<8 * kChunk>(p1, c.r[4], c.r[5], c.r[6], c.r[7]);
}

// The rope's second operand for the same tokens.
__device__ __forceinline__ void store_rest(uint32_t base, int lw, int lane, const Conv& c) {
  const int tok = lane >> 2, sub = lane & 3;
  const uint32_t p0 = base + lw * 1024 + tok * 128 + (((2 * sub) ^ tok) << 4), p1 = p0 ^ 16u;
  uint32_t h[8];
#pragma unroll
  for (int i = 0; i < 8; ++i)
    h[i] = c.dr == 0 ? 0u
                     : h2_bits(__hmul2(*reinterpret_cast<const __half2*>(&c.r[i]), *reinterpret_cast<const __half2*>(&c.dr)));
  st_shared_v4(p0, h[0], h[1], h[2], h[3]);
  st_shared_v4(p1, h[4], h[5], h[6], h[7]);
}

// Walks the tiles of a CTA's range.
struct Walk {
  int64_t row;
  int hg, tile, seg;  // seg: jobs since the first
  __device__ __forceinline__ Walk(const AttnArgs& p, int64_t job, int t)
      : row(job / p.n_hg), hg(static_cast<int>(job % p.n_hg)), tile(t), seg(0) {}
  __device__ __forceinline__ void next(const AttnArgs& p) {
    if (++tile == p.tiles) {
      tile = 0;
      next_job(p);
    }
  }
  __device__ __forceinline__ void next_job(const AttnArgs& p) {
    ++seg;
    if (++hg == p.n_hg) {
      hg = 0;
      ++row;
    }
  }
};

template <bool kFp4, bool kBlocks>
__global__ __launch_bounds__(kAtThreads, 1) void sparse_mla_kernel(const __grid_constant__ CUtensorMap map,
                                                                    const AttnArgs p) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  AtSmem<kFp4>& sm = smem_aligned_1024<AtSmem<kFp4>>(smem_raw);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t f0 = first_tile(p, blockIdx.x, gridDim.x);
  const int n = static_cast<int>(first_tile(p, blockIdx.x + 1, gridDim.x) - f0);  // at least 1
  const int64_t job0 = f0 / p.tiles;
  const int tile0 = static_cast<int>(f0 - job0 * p.tiles);

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sm.full[i], kLoadWarps);
      mbar_init(&sm.empty[i], 1);
      mbar_init(&sm.sfull[i], 1);
      mbar_init(&sm.pready[i], kSoftWarps);
    }
    mbar_init(&sm.rfull, 1);
    mbar_init(&sm.rempty, kLoadWarps);
    mbar_init(&sm.sempty, kSoftWarps);
    mbar_init(&sm.qfull, kQWarps);
    mbar_init(&sm.qempty, 1);
    mbar_init(&sm.oempty, kSoftWarps);
    mbar_init(&sm.done, 1);
    sm.abort = 0;
    fence_barrier_init();
    tma_prefetch_desc(&map);
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
  const uint64_t limit = wait_limit_ns();

  // Every role walks the CTA's n tiles; no role leaves early, so that the named barriers of the
  // softmax warps stay complete: after a wait ran out (abort) the remaining waits return at once and
  // no more MMAs are issued.
  if (warp >= kLoadWarp) {
    // ------------------------------------------------ loaders
    const int lw = warp - kLoadWarp, tok = lw * 8 + (lane >> 2);
    const uint32_t mine = smem_u32(sm.raw) + tok * (kFp4 ? kRawFp4 : kRawFp8);
    int tile = tile0, seg = 0;
    for (int g = 0; g < n; ++g) {
      const int b = g & 1;
      mbar_wait(&sm.rfull, g & 1, abort, &g_hcu_status);
      const uint32_t m0 = sm.mask[0], m1 = sm.mask[1];
      const bool some = (m0 | m1) != 0;
      const bool on = (tok < 32 ? m0 >> tok : m1 >> (tok - 32)) & 1;
      Conv conv;
      if (some) {
        Raw<kFp4> raw;
        read_raw<kFp4>(mine, lane & 3, raw);
        // The next gather writes these bytes through the async proxy: without the proxy fence it overtook
        // reads that were still under way (about one row of 2048 tokens x 64 heads in 500 came out wrong).
        fence_async_shared();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.rempty);
        convert<kFp4>(raw, lane & 3, conv);
      } else {
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.rempty);
      }
      if constexpr (!kFp4) {
        if (some) {
          // One buffer: the scores of the tiles before have been formed (also when the last tile held no token).
          // Stored here it costs nothing; after the tile, where S waits for it, 7 % (2048 rows: 1273 and 1365 us).
          if (g > 0) mbar_wait(&sm.sfull[(g - 1) & 1], ((g - 1) >> 1) & 1, abort, &g_hcu_status);
          store_rest(smem_u32(sm.grp.rest), lw, lane, conv);
        }
      }
      if (g >= 2) mbar_wait(&sm.empty[b], ((g >> 1) - 1) & 1, abort, &g_hcu_status);
      if (some) {
        store_tile<kFp4>(sm, b, lw, lane, on, conv);
        fence_async_shared();
      }
      if (lw == 0) {
        // the softmax warps read the segment's cq after this tile's `full`: pass the Q warps' writes on
        if (g == 0 || tile == 0) mbar_wait(&sm.qfull, (seg++) & 1, abort, &g_hcu_status);
        if (lane == 0) sm.empty_tile[b] = !some;
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.full[b]);
      if (++tile == p.tiles) tile = 0;
    }
  } else if (warp == kGatherWarp) {
    // ------------------------------------------------ gather: slots into the raw buffer
    constexpr int stride = kFp4 ? kRawFp4 : kRawFp8;
    const uint32_t dst = smem_u32(sm.raw) + 4 * lane * stride;
    int last_copies = -1;  // the last tile that has copies
    // Three tiles ahead of the copy: a tile's entries are fetched, then its places; once these are there
    // its slots are brought into L2, so that the copy into the one raw buffer waits for L2, not HBM.
    Walk ahead(p, job0, tile0), at = ahead;  // `ahead` names the tile whose entries are fetched next, `at` the place's
    Entry entry;
    Place place;
    int32_t s[4], nx[4];  // slots of tile g, of tile g + 1
    uint32_t has, hasn = 0;
    const auto step = [&](int fetch) {  // place -> slots, entry -> place, list -> entry of tile `fetch`
#pragma unroll
      for (int i = 0; i < 4; ++i) nx[i] = resolve<kBlocks>(p, place, i);
      hasn = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) hasn |= nx[i] >= 0 ? 1u << i : 0u;
      place = load_place<kBlocks>(p, at.row, at.tile, lane, entry);
      at.next(p);
      entry = load_entry<kBlocks>(p, ahead.row, ahead.tile, lane, fetch < n);
      ahead.next(p);
    };
    entry = load_entry<kBlocks>(p, ahead.row, ahead.tile, lane, true);
    ahead.next(p);
    place = load_place<kBlocks>(p, at.row, at.tile, lane, entry);
    at.next(p);
    entry = load_entry<kBlocks>(p, ahead.row, ahead.tile, lane, n > 1);
    ahead.next(p);
    step(2);
    for (int g = 0; g < n; ++g) {
#pragma unroll
      for (int i = 0; i < 4; ++i) s[i] = nx[i];
      has = hasn;
      const uint32_t m0 = __reduce_or_sync(0xffffffffu, lane < 8 ? has << (4 * lane) : 0u);
      const uint32_t m1 = __reduce_or_sync(0xffffffffu, lane >= 8 && lane < kGatherLanes ? has << (4 * (lane - 8)) : 0u);
      const bool some = (m0 | m1) != 0;
      // a wait that ran out: no more copies (their barrier phases could no longer be told apart)
      if (g > 0 && !mbar_wait(&sm.rempty, (g - 1) & 1, abort, &g_hcu_status)) break;
      if (lane == 0) {
        sm.mask[0] = m0;
        sm.mask[1] = m1;
        if (some)
          mbar_arrive_expect_tx(&sm.rfull, kTile * stride);
        else
          mbar_arrive(&sm.rfull);
      }
      __syncwarp();
      if (some) {
        if (lane < kGatherLanes) tma_gather4(dst, &map, &sm.rfull, s[0], s[1], s[2], s[3]);
        last_copies = g;
      }
      step(g + 3);
      if (hasn) tma_prefetch4(&map, nx[0], nx[1], nx[2], nx[3]);
      __syncwarp();
    }
    // copies in flight must land before the CTA may exit
    if (last_copies >= 0 && *abort) mbar_wait_drain(&sm.rfull, last_copies & 1, &g_hcu_status);
  } else if (warp == kMmaWarp) {
    // ------------------------------------------------ MMA issuer
    if (elect_one()) {
      // The first product of tile s and the second of tile o, whichever has its operands: the second
      // must not wait for a later tile's slots (its buffer is what they are waiting for), nor the
      // first for the softmax in between.  S has two buffers, so s runs at most two tiles ahead of o.
      constexpr uint32_t id_s = idesc_f16(64, kTile, false);
      int s = 0, o = 0;                                      // tiles of the CTA's range
      int s_tile = tile0, s_seg = 0, o_tile = tile0, o_seg = 0;  // their places in their jobs
      int o_hg = static_cast<int>(job0 % p.n_hg);
      uint32_t s_none = 0;  // bit b: the tile in buffer b holds no token
      uint32_t acc = 0;     // the segment's O holds something
      bool q_ok = false;    // the segment's Q has been waited for
      uint64_t t0 = 0;
      int idle = 0;
      while (o < n) {
        bool moved = false;
        if (s < n && s < o + 2) {
          const int b = s & 1;
          if (!q_ok) q_ok = mbar_test(&sm.qfull, s_seg & 1);
          // the fp8 score parts have one buffer, which the softmax warps empty into registers
          if (q_ok && mbar_test(&sm.full[b], (s >> 1) & 1) && (kFp4 || s == 0 || mbar_test(&sm.sempty, (s - 1) & 1))) {
            moved = true;
            tc_fence_after();
            s_none &= ~(1u << b);
            if (!sm.empty_tile[b]) {
              const uint64_t qd = sw128_kmajor_desc(smem_u32(sm.q)), kd = sw128_kmajor_desc(smem_u32(sm.k[b]));
#pragma unroll
              for (int k = 0; k < kQkDim / 16; ++k) {
                const uint32_t c = k >> 2, off = (k & 3) * 32;
                const uint32_t g = c >> 1 < 3 ? c >> 1 : 3;  // 128 values; the rope is the last one's
                const uint32_t d = tmem + kTmemS + (kFp4 ? 64 * b : kTile * g);
                const uint32_t add = (kFp4 ? k == 0 : k % 8 == 0 && c < 8) ? 0u : 1u;
                if (c < kQTmem)
                  mma_f16_ts(d, tmem + kTmemQ + 8 * k, kd + ((c * kChunk + off) >> 4), id_s, add);
                else
                  mma_f16(d, qd + (((c - kQTmem) * kQChunk + off) >> 4), kd + ((c * kChunk + off) >> 4), id_s, add);
              }
              if constexpr (!kFp4) {
                const uint64_t ld = sw128_kmajor_desc(smem_u32(sm.grp.rest));
#pragma unroll
                for (uint32_t k = 0; k < 4; ++k)
                  mma_f16(tmem + kTmemS + kTile * 3, qd + (((kChunks - 1 - kQTmem) * kQChunk + 32 * k) >> 4),
                          ld + (32 * k >> 4), id_s, 1u);
              }
              tc_commit(&sm.sfull[b]);
            } else {
              s_none |= 1u << b;
              tc_commit(&sm.sfull[b]);  // stands for the scores of the tiles before, like any other tile's
            }
            ++s;
            if (++s_tile == p.tiles) {
              tc_commit(&sm.qempty);  // the job's last product with this Q
              s_tile = 0;
              ++s_seg;
              q_ok = false;
            }
          }
        }
        if (o < s) {
          const int b = o & 1;
          const bool none = s_none >> b & 1;
          if (o == 0 || o_tile == 0) acc = 0;
          // a segment's first product overwrites O: the output of the segment before must be done
          if (mbar_test(&sm.pready[b], (o >> 1) & 1) &&
              (none || acc != 0 || o_seg == 0 || mbar_test(&sm.oempty, (o_seg - 1) & 1))) {
            moved = true;
            if (!none) {
              tc_fence_after();
              const uint32_t id_o = idesc_f16(128, (min(kHg, p.heads - o_hg * kHg) + 15) & ~15, true);
              const uint64_t v = sw128_mnmajor_desc(smem_u32(sm.k[b]));
              const uint64_t pd = sw32_kmajor_desc(smem_u32(sm.k[b]) + 8 * kChunk), px = sw32_kmajor_desc(smem_u32(&sm.grp));
#pragma unroll
              for (int ks = 0; ks < kTile / 16; ++ks)
#pragma unroll
                for (int d = 0; d < 4; ++d)
                  mma_f16(tmem + kTmemO + 64 * d, v + ((2 * d * kChunk + ks * 2048) >> 4),
                          (kFp4 || d == 0 ? pd : px + (((d - 1) * kPBytes) >> 4)) + ((ks * 2048) >> 4), id_o,
                          ks > 0 ? 1u : acc);
              acc = 1;
            }
            // For a tile without tokens too: the output may wait for its barrier alone, which must then stand for
            // the products of the tiles before it.
            tc_commit(&sm.empty[b]);
            ++o;
            if (++o_tile == p.tiles) {
              o_tile = 0;
              ++o_seg;
              if (++o_hg == p.n_hg) o_hg = 0;
            }
          }
        }
        if (moved) {
          idle = 0;
        } else if ((++idle & 63) == 0) {  // the time is looked at every 64 rounds: a round is on the tile's path
          if (idle == 64) t0 = globaltimer();
          if (*abort || globaltimer() - t0 > limit) {  // nothing became ready for too long: give up
            if (!*abort) atomicOr(&g_hcu_status, HCU_STATUS_WAIT_TIMEOUT);
            *abort = 1;
            break;
          }
        }
      }
      tc_commit(&sm.done);
      mbar_wait_drain(&sm.done, 0, &g_hcu_status);
    }
  } else if (warp >= kQWarp) {
    // ------------------------------------------------ queries
    // Q is single-buffered: the next segment's rows are brought into L2 while this one's are in use.
    // Four cq buffers: when a segment's Q is released, its second predecessor's first tile is done with.
    const int qw = warp - kQWarp, quad = warp & 3, sub = lane & 3, h0 = 16 * quad + (lane >> 2);
    Walk at(p, job0, 0);
    const int segs = (tile0 + n + p.tiles - 1) / p.tiles;
    for (int seg = 0; seg < segs; ++seg) {
      uint2 v[2][8];
      float f[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) fetch_q(q_head(p, at.row, at.hg * kHg + h0 + 8 * i), sub, v[i]);
      if (seg > 0) mbar_wait(&sm.qempty, (seg - 1) & 1, abort, &g_hcu_status);
      tc_fence_after();
      const uint32_t q = smem_u32(sm.q);
#pragma unroll
      for (int i = 0; i < 2; ++i) copy_q(q_head(p, at.row, at.hg * kHg + h0 + 8 * i), q, h0 + 8 * i, sub);
      asm volatile("cp.async.wait_all;" ::: "memory");  // each lane converts what it copied
#pragma unroll
      for (int i = 0; i < 2; ++i) f[i] = convert_q(p, q, sm.cq[seg & 3], h0 + 8 * i, sub, v[i]);
      uint32_t r[32];
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          r[4 * j + 2 * i] = bf2_to_h2(v[i][j].x, f[i]);
          r[4 * j + 2 * i + 1] = bf2_to_h2(v[i][j].y, f[i]);
        }
      tmem_st_16x256_x8(tmem + kTmemQ + (static_cast<uint32_t>(quad * 32) << 16), r);
      asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
      tc_fence_before();
      fence_async_shared();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.qfull);
      at.next_job(p);
      if (seg + 1 < segs) {
        for (int h = qw * 32 + lane; h < kHg * 9; h += kQWarps * 32) {  // 9 lines of 128 bytes per head
          const int hd = at.hg * kHg + h / 9;
          if (hd < p.heads)
            asm volatile("prefetch.global.L2 [%0];" ::"l"(p.q + at.row * p.q_row + hd * p.q_head + 64 * (h % 9)));
        }
      }
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
      if (g == 0 || tile == 0) {
        m0 = m1 = -INFINITY;
        l0 = l1 = 0.f;
        cq0 = sm.cq[seg & 3][r0];
        cq1 = sm.cq[seg & 3][r1];
        started = false;
      }
      float2 up[6], e[6];  // of the thread's tokens, read while S is computed
#pragma unroll
      for (int i = 0; i < 6; ++i) {
        up[i] = *reinterpret_cast<const float2*>(&sm.tok_up[b][8 * i + cl]);
        e[i] = *reinterpret_cast<const float2*>(&sm.tok_e[b][8 * i + cl]);
      }
      const bool none = sm.empty_tile[b];
      mbar_wait(&sm.sfull[b], (g >> 1) & 1, abort, &g_hcu_status);
      // Every warp goes through the same barriers whatever it saw (after a wait that ran out the warps'
      // views may differ): one soft_any per tile, and the rescale's two when any warp asks for one.
      float2 w[12];  // scores in base 2 plus the token's exponent: rows r0 (even), r1 (odd)
      float mx0 = -INFINITY, mx1 = -INFINITY;
      if (!none) {
        tc_fence_after();
        const float2 c0 = make_float2(cq0, cq0), c1 = make_float2(cq1, cq1);
        const auto score = [&](int i, float2 a, float2 d) {
          w[2 * i] = __ffma2_rn(__fmul2_rn(a, up[i]), c0, e[i]);
          w[2 * i + 1] = __ffma2_rn(__fmul2_rn(d, up[i]), c1, e[i]);
          mx0 = fmaxf(mx0, fmaxf(w[2 * i].x, w[2 * i].y));
          mx1 = fmaxf(mx1, fmaxf(w[2 * i + 1].x, w[2 * i + 1].y));
        };
        if constexpr (kFp4) {
          uint32_t s[24];
          tmem_ld_scores(tmem + kTmemS + 64 * b + quad, s);
#pragma unroll
          for (int i = 0; i < 6; ++i)
            score(i, make_float2(__uint_as_float(s[4 * i]), __uint_as_float(s[4 * i + 1])),
                  make_float2(__uint_as_float(s[4 * i + 2]), __uint_as_float(s[4 * i + 3])));
        } else {
#pragma unroll
          for (int j = 0; j < 3; ++j) {
            uint32_t s[4][8];
            tmem_ld_parts(tmem + kTmemS + 16 * j + quad, s);
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const float4 x = sm.grp.tok_r[b][16 * j + 8 * k + cl], y = sm.grp.tok_r[b][16 * j + 8 * k + cl + 1];
              const float2 r[4] = {make_float2(x.x, y.x), make_float2(x.y, y.y), make_float2(x.z, y.z), make_float2(x.w, y.w)};
              float2 a = make_float2(0.f, 0.f), d = a;
#pragma unroll
              for (int g = 0; g < 4; ++g) {
                a = __ffma2_rn(make_float2(__uint_as_float(s[g][4 * k]), __uint_as_float(s[g][4 * k + 1])), r[g], a);
                d = __ffma2_rn(make_float2(__uint_as_float(s[g][4 * k + 2]), __uint_as_float(s[g][4 * k + 3])), r[g], d);
              }
              score(2 * j + k, a, d);
            }
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&sm.sempty);
        }
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) {
          mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, o));
          mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, o));
        }
      } else if (!kFp4 && lane == 0) {
        mbar_arrive(&sm.sempty);
      }
      if (soft_any(mx0 > m0 + kLazy || mx1 > m1 + kLazy)) {  // m = -inf: any finite maximum
        const float n0 = fmaxf(m0, mx0), n1 = fmaxf(m1, mx1);
        const float x0 = m0 == n0 ? 1.f : ex2(m0 - n0), x1 = m1 == n1 ? 1.f : ex2(m1 - n1);
        l0 *= x0;
        l1 *= x1;
        m0 = n0;
        m1 = n1;
        if ((lane & 3) == 0) {
          sm.factor[r0] = x0;
          sm.factor[r1] = x1;
        }
        if (started) mbar_wait(&sm.empty[(g - 1) & 1], ((g - 1) >> 1) & 1, abort, &g_hcu_status);  // O is complete so far
        named_bar(2, kSoftWarps * 32);
        if (started) {
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
        }
        named_bar(2, kSoftWarps * 32);  // factor may be written again
      }
      if (!none) {
        const float b0 = m0 == -INFINITY ? 0.f : m0 - kBias, b1 = m1 == -INFINITY ? 0.f : m1 - kBias;
        // P: for every 16 tokens [64 heads][16 tokens], rows of 32 bytes with the 32-byte swizzle
        const int ph = 16 * warp + 8 * ((lane >> 3) & 1) + (lane & 7);
        const uint32_t pdst = smem_u32(sm.k[b]) + 8 * kChunk + st_piece(ph, lane >> 4);
        const uint32_t pxdst = smem_u32(&sm.grp) + st_piece(ph, lane >> 4);  // grp.p
        // groups 1 to 3 have one buffer: the last tile's product has read it (the one before that came before
        // this tile's scores)
        if (!kFp4 && g > 0) mbar_wait(&sm.empty[(g - 1) & 1], ((g - 1) >> 1) & 1, abort, &g_hcu_status);
        const float2 n0 = make_float2(-b0, -b0), n1 = make_float2(-b1, -b1);
        float2 z0 = make_float2(l0, 0.f), z1 = make_float2(l1, 0.f);
#pragma unroll
        for (int i = 0; i < 6; i += 2) {
          float2 p0[2], p1[2];
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const float2 x0 = __fadd2_rn(w[2 * (i + k)], n0), x1 = __fadd2_rn(w[2 * (i + k) + 1], n1);
            p0[k] = make_float2(ex2(x0.x), ex2(x0.y));
            p1[k] = make_float2(ex2(x1.x), ex2(x1.y));
            const float2 dn = *reinterpret_cast<const float2*>(&sm.tok_dn[b][8 * (i + k) + cl]);
            z0 = __ffma2_rn(p0[k], dn, z0);
            z1 = __ffma2_rn(p1[k], dn, z1);
          }
          // matrices: (tokens 8 i.., heads r0), (.., heads r1), (tokens 8 (i + 1).., heads r0), (.., r1)
          if constexpr (kFp4) {
            stmatrix_x4(pdst + i * 1024, pack2(p0[0]), pack2(p1[0]), pack2(p0[1]), pack2(p1[1]));
          } else {
            const float4 x0 = sm.grp.tok_r[b][8 * i + cl], y0 = sm.grp.tok_r[b][8 * i + cl + 1];
            const float4 x1 = sm.grp.tok_r[b][8 * i + 8 + cl], y1 = sm.grp.tok_r[b][8 * i + 8 + cl + 1];
            const auto put = [&](uint32_t dst, float2 ra, float2 rb) {
              stmatrix_x4(dst + i * 1024, pack2(__fmul2_rn(p0[0], ra)), pack2(__fmul2_rn(p1[0], ra)),
                          pack2(__fmul2_rn(p0[1], rb)), pack2(__fmul2_rn(p1[1], rb)));
            };
            put(pdst, make_float2(x0.x, y0.x), make_float2(x1.x, y1.x));
            put(pxdst, make_float2(x0.y, y0.y), make_float2(x1.y, y1.y));
            put(pxdst + kPBytes, make_float2(x0.z, y0.z), make_float2(x1.z, y1.z));
            put(pxdst + 2 * kPBytes, make_float2(x0.w, y0.w), make_float2(x1.w, y1.w));
          }
        }
        l0 = z0.x + z0.y;
        l1 = z1.x + z1.y;
        started = true;
        fence_async_shared();
        tc_fence_before();
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.pready[b]);

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
        if (whole) {
          // 16 latent values x 32 heads at a time: fragments, transposed into the warp's 1 KB as rows of
          // 32 bytes per head, then stored as whole sectors
          const uint32_t st = smem_u32(&sm.grp) + 1024 * warp;
          uint16_t* dst = p.out + (row * p.heads + h0) * kLatentDim + 32 * warp + 8 * (lane & 1);
          const int piece = st_piece(lane >> 1, lane & 1);
#pragma unroll 1
          for (int hb = 0; hb < nh; hb += 32) {
            float2 f[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) f[i] = *reinterpret_cast<const float2*>(&sm.factor[hb + 8 * i + cl]);
#pragma unroll 2
            for (int c = 0; c < 8; ++c) {  // latent values 128 (c / 2) + 32 warp + 16 (c % 2) ..
              uint32_t o[16];
              if (started) {
                tmem_ld_16x256_x4(tmem + kTmemO + 64 * (c >> 1) + hb + quad + (static_cast<uint32_t>(16 * (c & 1)) << 16),
                                  o);
              } else {
#pragma unroll
                for (int j = 0; j < 16; ++j) o[j] = 0;
              }
              uint32_t w[8];
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const __nv_bfloat162 lo = __floats2bfloat162_rn(__uint_as_float(o[4 * i]) * f[i].x,
                                                                __uint_as_float(o[4 * i + 1]) * f[i].y);
                const __nv_bfloat162 hi = __floats2bfloat162_rn(__uint_as_float(o[4 * i + 2]) * f[i].x,
                                                                __uint_as_float(o[4 * i + 3]) * f[i].y);
                w[2 * i] = *reinterpret_cast<const uint32_t*>(&lo);
                w[2 * i + 1] = *reinterpret_cast<const uint32_t*>(&hi);
              }
              // matrices: (values 0-7, heads 8 i ..), (values 8-15, heads 8 i ..), then heads 8 (i + 1) ..
              const int hr = 8 * (lane >> 4) + (lane & 7), part = (lane >> 3) & 1;
              stmatrix_x4_trans(st + st_piece(hr, part), w[0], w[1], w[2], w[3]);
              stmatrix_x4_trans(st + st_piece(hr + 16, part), w[4], w[5], w[6], w[7]);
              __syncwarp();
              const uint4 a0 = ld_shared_v4(st + piece), a1 = ld_shared_v4(st + piece + 16 * 32);
              uint16_t* d0 = dst + 128 * (c >> 1) + 16 * (c & 1) + static_cast<int64_t>(hb + (lane >> 1)) * kLatentDim;
              if (hb + (lane >> 1) < nh) *reinterpret_cast<uint4*>(d0) = a0;
              if (hb + (lane >> 1) + 16 < nh) *reinterpret_cast<uint4*>(d0 + 16 * kLatentDim) = a1;
              __syncwarp();
            }
          }
        } else {
#pragma unroll 1
          for (int c = 0; c < 8; ++c) {  // 32 heads of 128 latent values
            const int hb = 32 * (c & 1);
            if (hb >= nh) continue;
            uint32_t o[32];
            if (started) {
              tmem_ld_x32_sync(tmem + kTmemO + quad + 32 * c, o);
            } else {
#pragma unroll
              for (int j = 0; j < 32; ++j) o[j] = 0;
            }
            const float4* f4 = reinterpret_cast<const float4*>(sm.factor + hb);
            float* dst = part + hb * kLatentDim + 128 * (c >> 1) + 32 * warp + lane;
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
// (c - 1, y): two heads of the job at the boundary between CTAs c - 1 and c, if that is the job's first
// boundary; half a block per head, four latent values a thread.  The partials lie in L2; what the join
// takes is the latency of its loads, so a head's weights are formed by 128 threads at once and its
// partials loaded eight at a time (one row in 43 parts: the whole call 25 us; with serial loads 52).
constexpr int kCombineThreads = 256, kCombineHeads = 2, kMaxParts = 256;

__global__ __launch_bounds__(kCombineThreads) void combine_kernel(const AttnArgs p, int grid) {
  __shared__ float weight[2][kMaxParts], red[2][4];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int c = blockIdx.x + 1;
  const int64_t at = first_tile(p, c, grid);
  const int64_t job = at / p.tiles;
  const int64_t begin = job * p.tiles, end = begin + p.tiles;
  if (at == begin || first_tile(p, c - 1, grid) > begin) return;
  const int64_t row = job / p.n_hg;
  const int h0 = static_cast<int>(job % p.n_hg) * kHg;
  // CTAs c - 1 .. c - 2 + parts share the job: the last one that starts before its end
  const int64_t last = (end / p.quantum * grid - 1) / (p.total / p.quantum);
  const int parts = static_cast<int>(min(last, static_cast<int64_t>(grid - 1))) - c + 2;
  // only the first of them may have started in another job: its part of this one is its second
  const float* const first = p.part + (static_cast<int64_t>(c - 1) * 2 + (first_tile(p, c - 1, grid) < begin ? 1 : 0)) * kPartFloats;
  const float* const rest = p.part + static_cast<int64_t>(c) * 2 * kPartFloats;  // of CTA c; CTA c + i: 2 i further
  const auto part_of = [&](int i) { return i == 0 ? first : rest + static_cast<int64_t>(i - 1) * 2 * kPartFloats; };
  const int sub = threadIdx.x >> 7, t = threadIdx.x & 127, lane = t & 31;
  const int h = blockIdx.y * kCombineHeads + sub;
  const bool on = h0 + h < p.heads && h < kHg;
  float lse[kMaxParts / 128], m = -INFINITY;
#pragma unroll
  for (int k = 0; k < kMaxParts / 128; ++k) {
    const int i = 128 * k + t;
    lse[k] = on && i < parts ? part_of(i)[kHg * kLatentDim + h] : -INFINITY;
    m = fmaxf(m, lse[k]);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (lane == 0) red[sub][t >> 5] = m;
  __syncthreads();
  m = fmaxf(fmaxf(red[sub][0], red[sub][1]), fmaxf(red[sub][2], red[sub][3]));
#pragma unroll
  for (int k = 0; k < kMaxParts / 128; ++k)  // an empty part weighs nothing; a NaN one shows beside empty ones too
    weight[sub][128 * k + t] = lse[k] == -INFINITY ? 0.f : exp2f(lse[k] - m);
  __syncthreads();
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  float l = 0.f;
  if (on) {
#pragma unroll 8
    for (int i = 0; i < parts; ++i) {
      const float w = weight[sub][i];
      const float4 v = *reinterpret_cast<const float4*>(part_of(i) + h * kLatentDim + 4 * t);
      l += w;
      o.x = fmaf(w, v.x, o.x);
      o.y = fmaf(w, v.y, o.y);
      o.z = fmaf(w, v.z, o.z);
      o.w = fmaf(w, v.w, o.w);
    }
    const float f = l == 0.f ? 0.f : 1.f / l;
    const __nv_bfloat162 a = __floats2bfloat162_rn(o.x * f, o.y * f), b = __floats2bfloat162_rn(o.z * f, o.w * f);
    const int64_t rh = row * p.heads + h0 + h;
    *reinterpret_cast<uint2*>(p.out + rh * kLatentDim + 4 * t) =
        make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
    if (t == 0) p.lse[rh] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
  }
}

// CTAs: one per SM at most, no more than the parts the join holds, and two tiles each at least.  One row of 43
// tiles: 25.6 us with 22 CTAs, 27.6 with 43, whose partials are twice as many.  Over one to four rows of 2 to 171
// tiles (16 and 64 heads, both formats) one tile at least would be 2.4 us shorter on average at 5 and 11 tiles and 2 to
// 5 longer from 43 on, three at least 4 us longer at 2 tiles and 1 to 2 shorter from 86 on.
int attn_grid(int64_t total) {
  const int64_t sms = sm_count() < kMaxParts ? sm_count() : kMaxParts, pairs = (total + 1) / 2;
  return static_cast<int>(pairs < sms ? pairs : sms);
}

int64_t tiles_of(int64_t n_tokens) { return n_tokens <= 0 ? 1 : (n_tokens + kTile - 1) / kTile; }

// The cache as rows of 4-byte words (a slot's words; the box is one row, padded to the raw stride).
int slot_map(CUtensorMap* m, const AttnArgs& a, bool fp4) {
  static std::once_flag once;
  static PFN_cuTensorMapEncodeTiled_v12000 encode = nullptr;
  std::call_once(once, [] {
    cudaDriverEntryPointQueryResult q;
    void* ptr = nullptr;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      encode = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr);
  });
  // an empty cache: a map that no copy reads (every candidate is out of range)
  const void* base = a.n_slots > 0 ? static_cast<const void*>(a.kv) : static_cast<const void*>(a.q);
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>((fp4 ? kKv4Slot : kFp8Slot) / 4),
                              static_cast<cuuint64_t>(a.n_slots > 0 ? a.n_slots : 1)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(a.slot_stride)};
  const cuuint32_t box[2] = {static_cast<cuuint32_t>((fp4 ? kRawFp4 : kRawFp8) / 4), 1};
  const cuuint32_t step[2] = {1, 1};
  if (!encode || encode(m, CU_TENSOR_MAP_DATA_TYPE_UINT32, 2, const_cast<void*>(base), dims, strides, box, step,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_NONE,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS) {
    set_last_error_msg("cuTensorMapEncodeTiled rejected the tensor map of ", "the MLA cache");
    return HCU_ERR_LAUNCH;
  }
  return HCU_OK;
}

template <bool kFp4, bool kBlocks>
int launch_attn(const AttnArgs& a, int grid, cudaStream_t st) {
  CUtensorMap map;
  const int rc = slot_map(&map, a, kFp4);
  if (rc != HCU_OK) return rc;
  constexpr int smem = static_cast<int>(sizeof(AtSmem<kFp4>)) + 1024;
  cudaError_t e = cudaFuncSetAttribute(sparse_mla_kernel<kFp4, kBlocks>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) {
    set_last_error(e);
    return HCU_ERR_LAUNCH;
  }
  sparse_mla_kernel<kFp4, kBlocks><<<grid, kAtThreads, smem, st>>>(map, a);
  bool split = false;
  for (int c = 1; c < grid && !split; ++c) split = first_tile(a, c, grid) % a.tiles != 0;
  if (split) {
    cudaLaunchConfig_t cfg = {};
    const int heads = a.heads < kHg ? a.heads : kHg;
    cfg.gridDim = dim3(static_cast<unsigned>(grid - 1), static_cast<unsigned>((heads + kCombineHeads - 1) / kCombineHeads));
    cfg.blockDim = dim3(kCombineThreads);
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
  if (!q || !out || !lse || !workspace || (n_idx > 0 && (!indices || (n_slots > 0 && !kv_cache)))) return HCU_ERR_ARG;
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
  // an empty list or table is read (its entries dropped) at some valid address
  if (n_idx == 0) a.idx = reinterpret_cast<const int32_t*>(q), a.idx_stride = 0;
  if (blocks && n_bt == 0) a.bt = reinterpret_cast<const int32_t*>(q), a.bt_stride = 0;
  // Whole jobs per CTA where that costs less than the join of split ones: sharing a job costs its CTAs
  // about eight tiles' time (a partial written, read and joined: 128 rows of 43 tiles take 15 us longer split).
  // Both ways measured for 8 to 128 heads, 10 to 420 rows of 3 to 86 tiles, both formats (672 shapes).  Per head
  // count and format the rule's choice takes 0.1 to 0.8 % more than the better way on average, 5 to 16 % at
  // worst; with 4 tiles for 8 it would be 0.6 to 3.8 % and 14 to 41 %, with 12 tiles 0.1 to 1.9 % and 3 to 29 %.
  const int64_t jobs = rows * a.n_hg, sms = attn_grid(a.total);
  a.quantum = (jobs + sms - 1) / sms * a.tiles <= (a.total + sms - 1) / sms + 8 ? a.tiles : 1;
  const int grid = static_cast<int>(a.quantum == 1 ? sms : (jobs < sms ? jobs : sms));
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (fp4) return blocks ? launch_attn<true, true>(a, grid, st) : launch_attn<true, false>(a, grid, st);
  return blocks ? launch_attn<false, true>(a, grid, st) : launch_attn<false, false>(a, grid, st);
}
