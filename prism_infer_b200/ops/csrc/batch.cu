// Maps of a step, built on the device from the lengths of its requests: block tables, the cache slot, position, request and adapter of
// every new token, running sums of the lengths and the row of every request's last token.
//
// Request i has cached_i tokens in the cache and fresh_i new ones, so kv_i = cached_i + fresh_i tokens live on n_i = ceil(kv_i / page)
// pages, which start at sum_{j<i} n_j of one flat list (or where page_offsets says).  New token t belongs to the request with
// cu_i <= t < cu_{i+1}, cu the running sum of fresh; it is the cache's token p = cached_i + t - cu_i and its slot is
// pages[start_i + p / page] * page + p % page.
//
// A few KB to a few MB move, so a launch is what the step costs: one launch, in which every block adds up all lengths itself (1024
// requests: 8 KB from L2) instead of waiting for a block that does, then writes its share of the tables, a row per warp, and of the
// tokens, which find their request by halving the running sum in shared memory.
#include "common.cuh"

PRISM_DEFINE_TU_STATUS(batch)

namespace {

constexpr int MAP_THREADS = 256;
constexpr int MAP_WARPS = MAP_THREADS / 32;
constexpr int MAP_MAX_REQUESTS = 8192;   // 8 bytes of shared memory each

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
  const int c = a.cached[i], f = a.fresh[i];
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
  int* const start = smem + a.S + 1;       // [S + 1] and of the pages
  __shared__ long long warp_sum[3][MAP_WARPS];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const bool first = blockIdx.x == 0;
  pdl_launch_dependents();
  pdl_wait();

  // Running sums, MAP_THREADS requests at a time.  64 bits: a sum past 31 bits is reported, not wrapped.
  long long base[3] = {0, 0, 0};
  for (int i0 = 0; i0 < a.S; i0 += MAP_THREADS) {
    const int i = i0 + threadIdx.x;
    int cached = 0, fresh = 0, kv = 0;
    if (i < a.S) kv = lengths_of(a, i, cached, fresh);
    long long v[3] = {fresh, kv, pages_of(kv, a.page)}, incl[3];
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      incl[k] = v[k];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long up = __shfl_up_sync(0xffffffffu, incl[k], o);
        if (lane >= o) incl[k] += up;
      }
      if (lane == 31) warp_sum[k][warp] = incl[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      long long before = base[k];
      for (int w = 0; w < MAP_WARPS; ++w) {
        if (w < warp) before += warp_sum[k][w];
        base[k] += warp_sum[k][w];
      }
      incl[k] += before;
    }
    if (i < a.S) {
      // tokens past T have no rows: every sum stops there
      cu[i + 1] = (int)min(incl[0], (long long)a.T);
      start[i + 1] = (int)min(incl[2], (long long)a.n_pages);
      if (first) {
        a.cu_q[i + 1] = cu[i + 1];
        a.cu_kv[i + 1] = (int)min(incl[1], 0x7fffffffll);
        a.kv_lens[i] = kv;
        a.sample_rows[i] = fresh > 0 && incl[0] <= a.T ? incl[0] - 1 : -1;
      }
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    cu[0] = start[0] = 0;
    if (first) {
      a.cu_q[0] = a.cu_kv[0] = 0;
      if (base[0] > a.T || base[1] > 0x7fffffffll) prism_report(PRISM_ERR_BOUNDS, MAP_TOKENS);
      if (a.page_offsets == nullptr && base[2] > a.n_pages) prism_report(PRISM_ERR_BOUNDS, MAP_PAGES);
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

  for (int i = blockIdx.x * MAP_WARPS + warp; i < a.S; i += gridDim.x * MAP_WARPS) {
    int cached, fresh, lo, hi;
    const int need = pages_of(lengths_of(a, i, cached, fresh), a.page);
    span(i, lo, hi);
    if (lane == 0 && need > a.W) prism_report(PRISM_ERR_BOUNDS, MAP_WIDTH);
    if (lane == 0 && need > hi - lo) prism_report(PRISM_ERR_BOUNDS, MAP_PAGES);
    const int n = min(need, hi - lo);
    int* const row = a.tables + (size_t)i * a.W;
#pragma unroll 4
    for (int j = lane; j < a.W; j += 32) row[j] = j < n ? a.pages[lo + j] : -1;
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
      int cached, fresh, first_page, end_page;
      lengths_of(a, seq, cached, fresh);
      span(seq, first_page, end_page);
      const int p = cached + (t - cu[seq]), q = p / a.page;
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
  if (S < 0 || S > MAP_MAX_REQUESTS || T < 0 || W < 1 || page < 1 || n_pages < 0) return -1;
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
  const long long rows = ((long long)S + MAP_WARPS - 1) / MAP_WARPS, tokens = ((long long)T + MAP_THREADS - 1) / MAP_THREADS;
  long long grid = rows > tokens ? rows : tokens;
  if (grid > 296) grid = 296;
  if (grid < 1) grid = 1;
  const size_t smem = (size_t)(2 * S + 2) * sizeof(int);
  if (smem > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(step_maps_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (2 * MAP_MAX_REQUESTS + 2) * 4);
    if (e != cudaSuccess) return (int)e;
  }
  return (int)prism_launch(step_maps_kernel, dim3((unsigned)grid), dim3(MAP_THREADS), smem, (cudaStream_t)stream, pdl != 0, a);
}
