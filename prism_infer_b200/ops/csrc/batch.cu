// Maps of a step, built on the device from the lengths of its requests: block tables, the cache slot, position, request and adapter of
// every new token, running sums of the lengths and the row of every request's last token.
//
// Request i has cached_i tokens in the cache and fresh_i new ones, so kv_i = cached_i + fresh_i tokens live on n_i = ceil(kv_i / page)
// pages, which start at sum_{j<i} n_j of one flat list (or where page_offsets says).  New token t belongs to the request with
// cu_i <= t < cu_{i+1}, cu the running sum of fresh; it is the cache's token p = cached_i + t - cu_i and its slot is
// pages[start_i + p / page] * page + p % page.
//
// A few KB to a few MB move, so a launch is what the step costs: one launch, in which every block adds up all lengths itself (1024
// requests: 8 KB from L2, read twice, for the sums of each thread's requests and, after one exchange between warps, for the sum behind each of
// them) instead of waiting for a block that does, then writes its share of the tables, 128 entries of a row per warp, and of the tokens, which
// find their request by halving the running sum in shared memory.  1 request 3.5 us, 1024 requests of up to 8192 tokens in pages of 16 (4 MB, 0.6 us of copy bandwidth) 9.2 us.
#include "common.cuh"

PRISM_DEFINE_TU_STATUS(batch)

namespace {

constexpr int MAP_THREADS = 256;
constexpr int MAP_WARPS = MAP_THREADS / 32;
constexpr int MAP_MAX_REQUESTS = 8192;   // 12 bytes of shared memory each
constexpr int MAP_MAX_ROWS = 1 << 30;     // tokens, and entries of a table row: strides stay inside 31 bits
constexpr int MAP_SEGMENT = 128;         // entries of a table row that a warp writes at a time

struct MapArgs {
  const int* pages;          // [n_pages] pages of all requests, one after another
  const int* page_offsets;   // [S + 1] (null: every request's pages follow the one's before)
  const int* cached;         // [S]
  const int* fresh;          // [S]
  const int* shift;          // [S] added to the positions (null: zero)
  const int* adapter;        // [S] (null: no adapters)
  int S, T, W, page, n_pages;
  int* tables;               // [S][W]
  long long* slots;          // [T]
  int* positions;            // [3][T]
  int* token_seq;            // [T]
  int* token_adapter;        // [T] (null with adapter)
  int* cu_q;                 // [S + 1]
  int* cu_kv;                // [S + 1]
  int* kv_lens;              // [S]
  long long* sample_rows;    // [S]
};

enum { MAP_LENGTH = 1, MAP_TOKENS = 2, MAP_WIDTH = 3, MAP_PAGES = 4 };   // details of a failed bounds check

__device__ __forceinline__ int lengths_of(const MapArgs& a, int i, int& cached, int& fresh) {
  const int c = __ldcg(a.cached + i), f = __ldcg(a.fresh + i);   // the step before may have written them on this SM
  const bool bad = c < 0 || f < 0 || c > 0x7fffffff - f;
  cached = bad ? 0 : c;
  fresh = bad ? 0 : f;
  if (bad) prism_report(PRISM_ERR_BOUNDS, MAP_LENGTH);
  return cached + fresh;
}
// ceil(n / page); n + page - 1 may pass 31 bits.
__device__ __forceinline__ int pages_of(int n, int page) { return n == 0 ? 0 : (n - 1) / page + 1; }

__global__ void __launch_bounds__(MAP_THREADS) step_maps_kernel(const MapArgs a) {
  extern __shared__ int smem[];
  int* const cu = smem;                    // [S + 1] running sum of the new tokens
  int* const start = cu + a.S + 1;         // [S + 1] and of the pages
  int* const behind = start + a.S + 1;     // [S] tokens in the cache
  __shared__ long long warp_sum[3][MAP_WARPS];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const bool first = blockIdx.x == 0;
  pdl_launch_dependents();
  pdl_wait();

  // Running sums: a run of requests per thread.  64 bits: a sum past 31 bits is reported, not wrapped.
  const int per = (a.S + MAP_THREADS - 1) / MAP_THREADS, i0 = min(a.S, (int)threadIdx.x * per), i1 = min(a.S, i0 + per);
  long long mine[3] = {0, 0, 0}, at[3];
#pragma unroll 4
  for (int i = i0; i < i1; ++i) {
    int cached, fresh;
    const int kv = lengths_of(a, i, cached, fresh);
    mine[0] += fresh;
    mine[1] += kv;
    mine[2] += pages_of(kv, a.page);
  }
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    at[k] = mine[k];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long up = __shfl_up_sync(0xffffffffu, at[k], o);
      if (lane >= o) at[k] += up;
    }
    if (lane == 31) warp_sum[k][warp] = at[k];
    at[k] -= mine[k];
  }
  __syncthreads();
  long long all[3] = {0, 0, 0};
#pragma unroll
  for (int k = 0; k < 3; ++k)
#pragma unroll
    for (int w = 0; w < MAP_WARPS; ++w) {
      if (w < warp) at[k] += warp_sum[k][w];
      all[k] += warp_sum[k][w];
    }
  for (int i = i0; i < i1; ++i) {
    int cached, fresh;
    const int kv = lengths_of(a, i, cached, fresh);
    at[0] += fresh;
    at[1] += kv;
    at[2] += pages_of(kv, a.page);
    // tokens past T have no rows: every sum stops there
    cu[i + 1] = (int)min(at[0], (long long)a.T);
    start[i + 1] = (int)min(at[2], (long long)a.n_pages);
    behind[i] = cached;
    if (first) {
      a.cu_q[i + 1] = cu[i + 1];
      a.cu_kv[i + 1] = (int)min(at[1], 0x7fffffffll);
      a.kv_lens[i] = kv;
      a.sample_rows[i] = fresh > 0 && at[0] <= a.T ? at[0] - 1 : -1;
    }
  }
  if (threadIdx.x == 0) {
    cu[0] = start[0] = 0;
    if (first) {
      a.cu_q[0] = a.cu_kv[0] = 0;
      if (all[0] > a.T || all[1] > 0x7fffffffll) prism_report(PRISM_ERR_BOUNDS, MAP_TOKENS);
      if (a.page_offsets == nullptr && all[2] > a.n_pages) prism_report(PRISM_ERR_BOUNDS, MAP_PAGES);
    }
  }
  __syncthreads();
  // first page of request i in the list, and the end of its pages
  auto span = [&](int i, int& lo, int& hi) {
    if (a.page_offsets != nullptr) {
      lo = a.page_offsets[i];
      hi = a.page_offsets[i + 1];
      if (lo < 0 || hi < lo || hi > a.n_pages) lo = hi = 0;
    } else {
      lo = start[i];
      hi = start[i + 1];
    }
  };

  const int segments = (a.W + MAP_SEGMENT - 1) / MAP_SEGMENT;
  for (long long w = (long long)blockIdx.x * MAP_WARPS + warp; w < (long long)a.S * segments; w += (long long)gridDim.x * MAP_WARPS) {
    const int i = (int)(w / segments), j0 = (int)(w - (long long)i * segments) * MAP_SEGMENT;
    int cached, fresh, lo, hi;
    const int need = pages_of(lengths_of(a, i, cached, fresh), a.page);
    span(i, lo, hi);
    if (lane == 0 && need > a.W) prism_report(PRISM_ERR_BOUNDS, MAP_WIDTH);
    if (lane == 0 && need > hi - lo) prism_report(PRISM_ERR_BOUNDS, MAP_PAGES);
    const int n = min(need, hi - lo);
    int* const row = a.tables + (size_t)i * a.W;
    int id[MAP_SEGMENT / 32];
#pragma unroll
    for (int e = 0; e < MAP_SEGMENT / 32; ++e) id[e] = j0 + e * 32 + lane < n ? a.pages[lo + j0 + e * 32 + lane] : -1;
#pragma unroll
    for (int e = 0; e < MAP_SEGMENT / 32; ++e)
      if (j0 + e * 32 + lane < a.W) row[j0 + e * 32 + lane] = id[e];
  }

  const int total = cu[a.S];
  for (int t = blockIdx.x * MAP_THREADS + threadIdx.x; t < a.T; t += gridDim.x * MAP_THREADS) {
    long long slot = -1;
    int pos = 0, seq = -1, who = -1;
    if (t < total) {
      int lo = 0, hi = a.S;   // cu[lo] <= t < cu[hi]; requests without new tokens are never the answer
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (cu[mid] <= t) lo = mid;
        else hi = mid;
      }
      seq = lo;
      int first_page, end_page;
      span(seq, first_page, end_page);
      const int p = behind[seq] + (t - cu[seq]), q = p / a.page;
      if (q < end_page - first_page) {
        const int id = a.pages[first_page + q];
        if (id >= 0) slot = (long long)id * a.page + (p - q * a.page);
      }
      pos = p + (a.shift ? a.shift[seq] : 0);
      if (a.adapter) who = a.adapter[seq];
    }
    a.slots[t] = slot;
    a.positions[t] = pos;
    a.positions[(size_t)a.T + t] = pos;
    a.positions[2 * (size_t)a.T + t] = pos;
    a.token_seq[t] = seq;
    if (a.token_adapter) a.token_adapter[t] = who;
  }
}

}  // namespace

// Fails with -1 for sizes outside the kernel's range.  Lengths, pages and offsets that contradict one another set the status word
// (negative or overflowing lengths count as zero, tokens without a page get slot -1, entries past the width are cut off).
PRISM_API int prism_step_maps(const void* pages, const void* page_offsets, const void* cached, const void* fresh, const void* shift,
                              const void* adapter, int S, int T, int W, int page, int n_pages, void* tables, void* slots, void* positions,
                              void* token_seq, void* token_adapter, void* cu_q, void* cu_kv, void* kv_lens, void* sample_rows,
                              void* stream, int pdl) {
  if (S < 0 || S > MAP_MAX_REQUESTS || T < 0 || T > MAP_MAX_ROWS || W < 1 || W > MAP_MAX_ROWS || page < 1 || n_pages < 0) return -1;
  MapArgs a;
  a.pages = (const int*)pages;
  a.page_offsets = (const int*)page_offsets;
  a.cached = (const int*)cached;
  a.fresh = (const int*)fresh;
  a.shift = (const int*)shift;
  a.adapter = (const int*)adapter;
  a.S = S;
  a.T = T;
  a.W = W;
  a.page = page;
  a.n_pages = n_pages;
  a.tables = (int*)tables;
  a.slots = (long long*)slots;
  a.positions = (int*)positions;
  a.token_seq = (int*)token_seq;
  a.token_adapter = (int*)token_adapter;
  a.cu_q = (int*)cu_q;
  a.cu_kv = (int*)cu_kv;
  a.kv_lens = (int*)kv_lens;
  a.sample_rows = (long long*)sample_rows;
  // four blocks per SM at most: every one of them adds up the lengths
  const long long warps = (long long)S * ((W + MAP_SEGMENT - 1) / MAP_SEGMENT), tokens = ((long long)T + MAP_THREADS - 1) / MAP_THREADS;
  long long grid = (warps + MAP_WARPS - 1) / MAP_WARPS;
  if (grid < tokens) grid = tokens;
  if (grid > 4 * 148) grid = 4 * 148;
  if (grid < 1) grid = 1;
  const size_t smem = (size_t)(3 * S + 2) * sizeof(int);
  if (smem > 47 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(step_maps_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (3 * MAP_MAX_REQUESTS + 2) * 4);
    if (e != cudaSuccess) return (int)e;
  }
  return (int)prism_launch(step_maps_kernel, dim3((unsigned)grid), dim3(MAP_THREADS), smem, (cudaStream_t)stream, pdl != 0, a);
}
