// Low-rank adapters of many requests beside a shared projection:
//   y_t = W x_t + bias + scale_a B_a (A_a x_t),   a the adapter of token t (negative: none),
// with stacked W: the features of section s have factors A_a^s, B_a^s of their own.
//
// Pools (ops/adapters.py) hold the factors of all loaded adapters with ranks padded to panels of 16: A as rows of K, panel after panel,
// section after section; B as [slot][panel of a section][feature][16], so that the 16 ranks of a run of features are one piece of memory.
#include "common.cuh"

#include <type_traits>

PRISM_DEFINE_TU_STATUS(adapters)

namespace {

typedef __nv_bfloat16 bf16;

constexpr int PLAN_TILE = 256;          // tokens that share a list of adapters
constexpr int PLAN_MAX_SLOTS = 8192;
constexpr int MAX_SECTIONS = 8;

enum { ADAPTER_SLOT = 1 };              // detail of a failed bounds check

// One block per tile: the adapters in use, ascending, and every token's place in that list.  A bit per slot, one word of 32 per thread.
__global__ void __launch_bounds__(PLAN_TILE) adapter_plan_kernel(const int* adapter, int T, int slots, int capacity, int* index, int* lists,
                                                                 int* counts) {
  __shared__ uint32_t bits[PLAN_MAX_SLOTS / 32];
  __shared__ int before[PLAN_MAX_SLOTS / 32];
  __shared__ int warp_sum[PLAN_TILE / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, t = blockIdx.x * PLAN_TILE + threadIdx.x;
  bits[threadIdx.x] = 0;
  pdl_launch_dependents();
  pdl_wait();
  __syncthreads();
  int who = t < T ? adapter[t] : -1;
  if (who >= slots) {
    prism_report(PRISM_ERR_BOUNDS, ADAPTER_SLOT);
    who = -1;
  }
  if (who >= 0) atomicOr(&bits[who >> 5], 1u << (who & 31));
  __syncthreads();
  const uint32_t mine = bits[threadIdx.x];
  int incl = __popc(mine);
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += up;
  }
  if (lane == 31) warp_sum[warp] = incl;
  __syncthreads();
  int total = 0;
  for (int w = 0; w < PLAN_TILE / 32; ++w) {
    if (w < warp) incl += warp_sum[w];
    total += warp_sum[w];
  }
  int at = incl - __popc(mine);
  before[threadIdx.x] = at;
  int* const list = lists + (size_t)blockIdx.x * capacity;
  for (uint32_t left = mine; left != 0; left &= left - 1) list[at++] = threadIdx.x * 32 + __ffs(left) - 1;
  for (int j = total + threadIdx.x; j < capacity; j += PLAN_TILE) list[j] = -1;
  if (threadIdx.x == 0) counts[blockIdx.x] = total;
  __syncthreads();
  if (t < T) index[t] = who < 0 ? -1 : before[who >> 5] + __popc(bits[who >> 5] & ((1u << (who & 31)) - 1));
}

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(bf16 v) { return __bfloat162float(v); }

struct ShrinkArgs {
  const void* x;        // [T][ldx]
  const void* a;        // [slots][low][K]
  const float* scale;   // [slots]
  const int* adapter;   // [T]
  float* h;             // [T][low]
  int T, K, low, slots;
  long long ldx;
};

// h_t = scale A x_t.  One block per token, a warp per row of A.
template <typename T>
__global__ void __launch_bounds__(256) adapter_shrink_kernel(const ShrinkArgs a) {
  const int t = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  pdl_launch_dependents();
  pdl_wait();
  const int who = a.adapter[t];
  if (who < 0 || who >= a.slots) return;
  const T* const x = (const T*)a.x + (size_t)t * a.ldx;
  const float scale = a.scale[who];
  for (int r = warp; r < a.low; r += 8) {
    const T* const row = (const T*)a.a + ((size_t)who * a.low + r) * a.K;
    float sum = 0.0f;
    for (int k = lane; k < a.K; k += 32) sum += to_float(x[k]) * to_float(row[k]);
    sum = warp_sum(sum);
    if (lane == 0) a.h[(size_t)t * a.low + r] = sum * scale;
  }
}

struct ExpandArgs {
  const float* base;    // [T][M] W x
  const float* h;       // [T][low]
  const void* b;        // [slots][panels][M][16]
  const void* bias;     // [M] (null: none)
  const int* adapter;   // [T]
  void* out;            // [T][ldo]
  int T, M, low, panels, slots, sections;
  int end[MAX_SECTIONS];
  int gated;            // silu / gelu of the first half times the second half (PRISM_GLU_*), 0: plain
  long long ldo;
};

template <typename T>
__device__ __forceinline__ float adapted(const ExpandArgs& a, int t, int m, int who) {
  float v = a.base[(size_t)t * a.M + m];
  if (a.bias != nullptr) v += to_float(((const T*)a.bias)[m]);
  if (who < 0) return v;
  int s = 0;
  while (s + 1 < a.sections && m >= a.end[s]) ++s;
  const float* const h = a.h + (size_t)t * a.low + s * a.panels * 16;
  float sum = 0.0f;
  for (int p = 0; p < a.panels; ++p) {
    const T* const b = (const T*)a.b + (((size_t)who * a.panels + p) * a.M + m) * 16;
#pragma unroll
    for (int r = 0; r < 16; ++r) sum += h[p * 16 + r] * to_float(b[r]);
  }
  return v + sum;
}

// y_t = base_t + bias + B h_t, through the gated unit if asked for; a thread per feature.
template <typename T>
__global__ void __launch_bounds__(256) adapter_expand_kernel(const ExpandArgs a) {
  const int m = blockIdx.x * 256 + threadIdx.x, t = blockIdx.y, out_features = a.gated ? a.M / 2 : a.M;
  pdl_launch_dependents();
  pdl_wait();
  if (m >= out_features) return;
  int who = a.adapter[t];
  if (who >= a.slots) who = -1;
  float v = adapted<T>(a, t, m, who);
  if (a.gated) v = glu(v, adapted<T>(a, t, m + a.M / 2, who), a.gated);
  T* const out = (T*)a.out + (size_t)t * a.ldo + m;
  if constexpr (std::is_same<T, float>::value) *out = v;
  else *out = __float2bfloat16_rn(v);
}

}  // namespace

// index [T], lists [tiles][capacity], counts [tiles], for tiles of 256 tokens.
PRISM_API int prism_adapter_plan(const void* adapter, int T, int slots, int capacity, void* index, void* lists, void* counts, void* stream,
                                 int pdl) {
  if (T < 1 || slots < 1 || slots > PLAN_MAX_SLOTS || capacity < (slots < PLAN_TILE ? (slots < T ? slots : T) : (T < PLAN_TILE ? T : PLAN_TILE)))
    return -1;
  return (int)prism_launch(adapter_plan_kernel, dim3((T + PLAN_TILE - 1) / PLAN_TILE), dim3(PLAN_TILE), 0, (cudaStream_t)stream, pdl != 0,
                           (const int*)adapter, T, slots, capacity, (int*)index, (int*)lists, (int*)counts);
}

PRISM_API int prism_adapter_shrink(int f32, const void* x, const void* a, const void* scale, const void* adapter, void* h, int T, int K, int low,
                                   int slots, long long ldx, void* stream, int pdl) {
  if (T < 1 || K < 1 || low < 16 || low % 16 || slots < 1) return -1;
  ShrinkArgs s{x, a, (const float*)scale, (const int*)adapter, (float*)h, T, K, low, slots, ldx};
  return (int)prism_launch(f32 ? adapter_shrink_kernel<float> : adapter_shrink_kernel<bf16>, dim3(T), dim3(256), 0, (cudaStream_t)stream, pdl != 0, s);
}

PRISM_API int prism_adapter_expand(int f32, const void* base, const void* h, const void* b, const void* bias, const void* adapter, void* out,
                                   int T, int M, int panels, int slots, int sections, const void* ends, int gated, long long ldo, void* stream,
                                   int pdl) {
  if (T < 1 || T > 65535 || M < 1 || panels < 1 || sections < 1 || sections > MAX_SECTIONS || slots < 1 || (gated && (M % 2 || sections != 2))) return -1;
  ExpandArgs e{(const float*)base, (const float*)h, b, bias, (const int*)adapter, out, T, M, sections * panels * 16, panels, slots, sections, {}, gated, ldo};
  for (int s = 0; s < sections; ++s) e.end[s] = ((const int*)ends)[s];
  const int features = gated ? M / 2 : M;
  return (int)prism_launch(f32 ? adapter_expand_kernel<float> : adapter_expand_kernel<bf16>, dim3((features + 255) / 256, T), dim3(256), 0,
                           (cudaStream_t)stream, pdl != 0, e);
}
