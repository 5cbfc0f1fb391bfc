// Tables of one decode or prefill step, from the requests' lengths, in one launch.
//
//   need_i   = ceil((seq_i + new_i) / 64) - ceil(seq_i / 64)      pages request i takes
//   before_i = free_head + sum_{j < i} need_j                      its first entry of free_pages
//   page_i(p) = req_pages[req_idx_i, p]          for p <  ceil(seq_i / 64)
//             = free_pages[before_i + p - ...]   for the pages taken in this step
//
// Query rows are the new tokens, request-major: row r of request i is its token at position
// seq_i + j.  One CTA per (row, 128 pages) finds the row's request and its page prefix by a block
// scan over the requests (a few hundred bytes from L2), then writes that part of the row's block
// table and slot table; the last CTA appends the taken pages to req_pages and writes the new head.
// No CTA reads what another writes: rows take their new pages from free_pages, not from req_pages.
//
// Bound: the stores, 4 B per (row, token of width) + 4 B per (row, page).  4096 rows of a prompt chunk at 64K (1.09 GB,
// 169 us at the copy rate of 6.45 TB/s) take 193 us, 5.7 TB/s.  128 rows of 65536 tokens (34 MB, 5.3 us) take
// 9.4 us in a graph of launches, 3.7 TB/s: a CTA stores its 32 KB only after its scan of the requests, three
// barriers long.  One row takes 3.2 us.
#include "common.cuh"

HCU_DEFINE_STATUS(status_tables)

namespace hcu {
namespace {

constexpr int kTbThreads = 256;
constexpr int kTbPages = 128;  // pages of a row per CTA (128 rows of 65536 tokens: 9.4 us; 64 pages 11.6, 256 pages 9.2)

struct TablesArgs {
  int32_t* req_pages;
  int64_t n_req, max_pages, req_stride;
  const int32_t* req_idx;
  const int32_t* seq_lens;
  const int32_t* new_lens;
  int batch;
  const int32_t* free_pages;
  int64_t n_free;
  const int32_t* free_head;
  int n_rows;
  int width_pages;
  int32_t* block_table;
  int32_t* page_table;
  int32_t* lengths;
  int32_t* positions;
  int32_t* token_loc;
  int64_t* loc;
  int32_t* free_head_out;
};

struct Req {
  int64_t have, total;  // pages before / after the step (capped at max_pages)
  int32_t seq, nw;
};

// Request i's lengths (negatives count as 0; a request row out of range takes no pages).
__device__ __forceinline__ Req load_req(const TablesArgs& a, int i, bool& bad) {
  Req r;
  const int32_t s = __ldg(a.seq_lens + i), n = __ldg(a.new_lens + i), row = __ldg(a.req_idx + i);
  r.seq = s < 0 ? 0 : s;
  r.nw = n < 0 ? 0 : n;
  const int64_t t = static_cast<int64_t>(r.seq) + r.nw;
  r.have = min((static_cast<int64_t>(r.seq) + kPage - 1) / kPage, a.max_pages);
  r.total = min((t + kPage - 1) / kPage, a.max_pages);
  bad = s < 0 || n < 0 || t > a.max_pages * kPage;
  if (row < 0 || row >= a.n_req) {
    bad = true;
    r.total = r.have;
  }
  return r;
}

// Inclusive block scan of (new tokens, pages taken), packed high / low.
__device__ __forceinline__ uint64_t block_scan(uint64_t v, uint64_t* warp_sum) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint64_t y = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += y;
  }
  __syncthreads();  // the previous chunk's readers of warp_sum are done
  if (lane == 31) warp_sum[warp] = v;
  __syncthreads();
  for (int w = 0; w < warp; ++w) v += warp_sum[w];
  return v;
}

__device__ __forceinline__ int32_t taken_page(const TablesArgs& a, int64_t k) {
  return k >= 0 && k < a.n_free ? __ldg(a.free_pages + k) : -1;
}

__global__ __launch_bounds__(kTbThreads) void step_tables_kernel(const TablesArgs a) {
  __shared__ uint64_t warp_sum[kTbThreads / 32];
  __shared__ int s_req;  // the row's request, -1 for a row past the last new token
  __shared__ int s_j;    // its index among the request's new tokens
  __shared__ int64_t s_before;
  __shared__ uint64_t s_run;
  __shared__ int32_t s_page[kTbPages];
  const int tid = threadIdx.x;
  const int n_chunk = (a.width_pages + kTbPages - 1) / kTbPages;
  const bool tail = blockIdx.x == static_cast<unsigned>(n_chunk) * a.n_rows;  // the appending CTA
  const int row = tail ? -1 : static_cast<int>(blockIdx.x) / n_chunk;
  const int chunk = tail ? 0 : static_cast<int>(blockIdx.x) % n_chunk;
  const int64_t head = __ldg(a.free_head);
  if (tid == 0) {
    s_req = -1;
    s_run = 0;
  }
  __syncthreads();

  for (int base = 0; base < a.batch; base += kTbThreads) {
    const int i = base + tid;
    Req r{};
    bool bad = false;
    if (i < a.batch) r = load_req(a, i, bad);
    const int64_t need = r.total - r.have;
    const uint64_t mine = (static_cast<uint64_t>(r.nw) << 32) | static_cast<uint64_t>(need);
    const uint64_t inc = s_run + block_scan(mine, warp_sum);
    const uint64_t exc = inc - mine;
    const int64_t first = static_cast<int64_t>(exc >> 32);                        // the request's first row
    const int64_t before = head + static_cast<int64_t>(exc & 0xffffffffull);  // its first free page
    if (tail) {
      if (i < a.batch) {
        const int32_t rr = __ldg(a.req_idx + i);
        for (int64_t k = 0; k < need; ++k)
          a.req_pages[rr * a.req_stride + r.have + k] = taken_page(a, before + k);
        if (bad || before < 0 || before + need > a.n_free || first + r.nw > a.n_rows ||
            static_cast<int64_t>(r.seq) + r.nw > static_cast<int64_t>(a.width_pages) * kPage)
          atomicOr(&g_hcu_status, HCU_STATUS_BAD_INPUT);
      }
    } else if (i < a.batch && row >= first && row < first + r.nw) {
      s_req = i;
      s_j = static_cast<int>(row - first);
      s_before = before;
    }
    __syncthreads();
    if (!tail && s_req >= 0) break;  // uniform: read after the barrier
    if (tid == kTbThreads - 1) s_run = inc;
    __syncthreads();
  }
  if (tail) {
    if (tid == 0) a.free_head_out[0] = static_cast<int32_t>(head + static_cast<int64_t>(s_run & 0xffffffffull));
    return;
  }

  const int i = s_req;
  bool bad = false;
  Req r{};
  int64_t src = 0;
  bool row_ok = false;
  if (i >= 0) {
    r = load_req(a, i, bad);
    const int32_t rr = __ldg(a.req_idx + i);
    row_ok = rr >= 0 && rr < a.n_req;
    src = static_cast<int64_t>(rr) * a.req_stride;
  }
  const auto page_at = [&](int64_t p) -> int32_t {
    if (i < 0 || !row_ok || p >= r.total) return -1;
    return p < r.have ? __ldg(a.req_pages + src + p) : taken_page(a, s_before + p - r.have);
  };
  const int p0 = chunk * kTbPages;
  const int np = min(kTbPages, a.width_pages - p0);
  for (int p = tid; p < np; p += kTbThreads) {
    const int32_t id = page_at(p0 + p);
    s_page[p] = id;
    a.block_table[static_cast<int64_t>(row) * a.width_pages + p0 + p] = id;
  }
  __syncthreads();
  const int64_t total_tok = static_cast<int64_t>(r.seq) + r.nw;  // 0 for a row without a request
  int4* out = reinterpret_cast<int4*>(a.page_table + (static_cast<int64_t>(row) * a.width_pages + p0) * kPage);
  for (int v = tid; v < np * (kPage / 4); v += kTbThreads) {
    const int32_t id = s_page[v / (kPage / 4)];
    const int64_t t = static_cast<int64_t>(p0) * kPage + 4 * v;
    const int32_t s = id * kPage + (4 * v) % kPage;
    out[v] = make_int4(id >= 0 && t < total_tok ? s : -1, id >= 0 && t + 1 < total_tok ? s + 1 : -1,
                       id >= 0 && t + 2 < total_tok ? s + 2 : -1, id >= 0 && t + 3 < total_tok ? s + 3 : -1);
  }
  if (chunk == 0 && tid == 0) {
    const int64_t pos = i >= 0 ? static_cast<int64_t>(r.seq) + s_j : 0;
    const int32_t id = i >= 0 ? page_at(pos / kPage) : -1;
    const int64_t slot = id >= 0 ? static_cast<int64_t>(id) * kPage + pos % kPage : -1;
    a.positions[row] = static_cast<int32_t>(pos);
    a.lengths[row] =
        i >= 0 ? static_cast<int32_t>(min(pos + 1, static_cast<int64_t>(a.width_pages) * kPage)) : 0;
    a.token_loc[row] = static_cast<int32_t>(slot);
    a.loc[row] = slot;
  }
}

}  // namespace
}  // namespace hcu

extern "C" int hcu_step_tables(int32_t* req_pages, int64_t n_req, int64_t max_pages, int64_t req_stride,
                               const int32_t* req_idx, const int32_t* seq_lens, const int32_t* new_lens, int64_t batch,
                               const int32_t* free_pages, int64_t n_free, const int32_t* free_head, int64_t n_rows,
                               int64_t width, int32_t* block_table, int32_t* page_table, int32_t* lengths,
                               int32_t* positions, int32_t* token_loc, int64_t* loc, int32_t* free_head_out,
                               hcu_stream_t stream) {
  using namespace hcu;
  constexpr int64_t kMaxInt = 0x7fffffff;
  if (n_req < 0 || max_pages < 0 || req_stride < max_pages || batch < 0 || batch > kMaxInt - kTbThreads ||
      n_free < 0 || n_rows < 0 || width <= 0 || width % kPage != 0 || width / kPage > kMaxInt / kPage)
    return HCU_ERR_ARG;
  if (!free_head || !free_head_out) return HCU_ERR_ARG;
  if (batch > 0 && (!req_pages || !req_idx || !seq_lens || !new_lens)) return HCU_ERR_ARG;
  if (n_free > 0 && !free_pages) return HCU_ERR_ARG;
  if (n_rows > 0 && (!block_table || !page_table || !lengths || !positions || !token_loc || !loc)) return HCU_ERR_ARG;
  if (reinterpret_cast<uintptr_t>(page_table) % 16 != 0) return HCU_ERR_ARG;
  const int64_t wp = width / kPage;
  const int64_t grid = ((wp + kTbPages - 1) / kTbPages) * n_rows + 1;
  if (grid > kMaxInt) return HCU_ERR_UNSUPPORTED;
  TablesArgs a{req_pages, n_req,  max_pages, req_stride, req_idx,     seq_lens,   new_lens, static_cast<int>(batch),
               free_pages, n_free, free_head, static_cast<int>(n_rows), static_cast<int>(wp), block_table, page_table,
               lengths,    positions, token_loc, loc, free_head_out};
  step_tables_kernel<<<static_cast<unsigned>(grid), kTbThreads, 0, reinterpret_cast<cudaStream_t>(stream)>>>(a);
  return launch_status();
}
