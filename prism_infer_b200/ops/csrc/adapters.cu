// Low-rank adapters of many requests beside a shared projection:
//   y_t = W x_t + bias + scale_a B_a (A_a x_t),   a the adapter of token t (negative: none),
// with stacked W: the features of section s have factors A_a^s, B_a^s of their own.
//
// Pools (ops/adapters.py) hold the factors of all loaded adapters with ranks padded to panels of 16: A as rows of K, panel after panel,
// section after section; B as [slot][panel of a section][feature][16], every section's features padded to a multiple of 8, in bf16 with the
// 16 ranks of 8 features as [2][8 features][8 ranks], the order in which the matrix instructions read them.
#include "common.cuh"

#include <atomic>

PRISM_DEFINE_TU_STATUS(adapters)

namespace {

typedef __nv_bfloat16 bf16;

constexpr int PLAN_TILE = 256;          // tokens that share a list of adapters
constexpr int PLAN_MAX_SLOTS = 8192;
constexpr int MAX_SECTIONS = 8;
constexpr int MAX_TOKENS = 65535 * 128; // of a call: tiles of 128 along one axis of the grid

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

// ------------------------------------------------------------------------------------------------------------------------------------
// bf16 on the tensor cores: two launches, the low-rank rows (adapter_low_kernel) and the projection with them (adapter_gemm_kernel, or
// gemm_pair.cuh from 129 tokens).
//
// Tokens of different adapters share tiles.  A tile's adapters (AdapterPlan.lists) become panels of 16 ranks: in the first kernel 128
// rows of A of up to eight panels multiply all tokens of the tile, and what is kept is each token's row in its own adapter's panels,
// zeros elsewhere; in the second every panel is one more MMA of 16 columns in the sum of the projection.  Both waste tensor cycles on
// tokens of other adapters, which a weight stream (decode) hides and a sum over K dwarfs (prompts).  A is read once for all tokens of a decode
// step and once for every 128 tokens of a prompt that have the adapter, B once for every tile of tokens; where 129 to 256 tokens run as two
// decode tiles (launch_prompt), both go through the panels of all 256 tokens' adapters, those that only the other has among them.
// The low-rank row is rounded to bf16, as an operand of the matrix instructions has to be; scale and sums are 32-bit.  That rounding, of up to
// 2^-8 of each low-rank value, is what the result has on top of its own: 0.0019 of the outputs' norm where 32-bit rows would leave 0.0017 (median
// over shapes of 4096 outputs and more, low-rank terms as large as the rest).
// ------------------------------------------------------------------------------------------------------------------------------------
constexpr int TC_THREADS = 192;         // TMA warp, MMA warp, four epilogue warps
constexpr int W_BYTES = 128 * 64 * 2;   // 128 rows of a k-block of 64
constexpr int RED_PITCH = 132;          // floats of one token's 128 sums in shared memory

template <int BN>
__host__ __device__ constexpr int stage_bytes() { return W_BYTES + BN * 128; }

__device__ __forceinline__ float4 ld_cluster4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ float4 add4(const float4& a, const float4& b) { return make_float4(a.x + b.x, a.y + b.y, a.z + b.z, a.w + b.w); }
__device__ __forceinline__ uint2 pack4(const float4& v) {
  uint2 o;
  *reinterpret_cast<__nv_bfloat162*>(&o.x) = __floats2bfloat162_rn(v.x, v.y);
  *reinterpret_cast<__nv_bfloat162*>(&o.y) = __floats2bfloat162_rn(v.z, v.w);
  return o;
}
// Share z of a sum over kb k-blocks in CS parts, none of them empty (CS <= kb).
__device__ __forceinline__ int part_begin(int kb, int z, int cs) { return (int)((long long)kb * z / cs); }

// The accumulator's 128 rows (lanes) of every token to shared memory, token after token.
template <int BN, int PITCH>
__device__ __forceinline__ void accumulator_to_smem(uint32_t tmem, float* red, int q, int lane, int tokens) {
  const uint32_t t_lane = tmem + ((uint32_t)(q * 32) << 16);
  for (int c0 = 0; c0 < tokens; c0 += 16) {
    uint32_t r[16];
    tmem_ld16(t_lane + c0, r);
    tmem_ld_wait();
#pragma unroll
    for (int j = 0; j < 16; ++j) red[(c0 + j) * PITCH + q * 32 + lane] = __uint_as_float(r[j]);
  }
}

struct LowArgs {
  const int* lists;      // [tiles][capacity]
  const int* counts;     // [tiles]
  const int* index;      // [T]
  const float* scale;    // [slots]
  const int* ranks;      // [slots][sections] of every slot's own factors; the rest of its panels is padding
  bf16* h;               // [tiles][capacity][all_panels] panels of tile_rows tokens
  int T, kb, capacity, panels, all_panels, tile_rows, stages;   // panels: of one section
  int run;               // panels that one copy moves: a divisor of all_panels, since an adapter's rows of A lie together
};

// The place of every token of a tile in the list of adapters, and the list itself (-1 behind its end), of which no more than MOST are in use.
template <int TOKENS, int MOST>
__device__ __forceinline__ void load_owners(const LowArgs& a, int* who, int* slot, int token0, int tile) {
  for (int c = threadIdx.x; c < TOKENS; c += TC_THREADS) who[c] = token0 + c < a.T ? a.index[token0 + c] : -1;
  for (int j = threadIdx.x; j < min(a.capacity, MOST); j += TC_THREADS) slot[j] = a.lists[(size_t)tile * a.capacity + j];
}
// And the scale and ranks of every token's adapter; by the epilogue warps, while the sums are under way.
template <int TOKENS>
__device__ __forceinline__ void load_scales(const LowArgs& a, const int* who, const int* slot, float* scale, short (*ranks)[MAX_SECTIONS]) {
  const int sections = a.all_panels / a.panels;
  for (int c = threadIdx.x - 64; c < TOKENS; c += TC_THREADS - 64) {
    const int s = who[c] >= 0 ? slot[who[c]] : -1;
    scale[c] = s >= 0 ? a.scale[s] : 0.0f;
#pragma unroll
    for (int k = 0; k < MAX_SECTIONS; ++k)
      if (k < sections) ranks[c][k] = s >= 0 ? (short)a.ranks[s * sections + k] : 0;
  }
}

// Sum over the cluster of four floats that every CTA keeps at the same place.
__device__ __forceinline__ float4 cluster_sum4(const float* mine, int cs) {
  const uint32_t at = smem_u32(mine);
  float4 v[8];
#pragma unroll
  for (int peer = 0; peer < 8; ++peer)
    if (peer < cs) {
      uint32_t remote;
      asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(at), "r"(peer));
      v[peer] = ld_cluster4(remote);
    }
#pragma unroll
  for (int peer = 1; peer < 8; ++peer)
    if (peer < cs) v[0] = add4(v[0], v[peer]);
  return v[0];
}

// Where ranks 8 * half .. + 8 of a panel's row lie.
__device__ __forceinline__ size_t in_panel(int row, int half) { return (size_t)(row >> 3) * 128 + half * 64 + (row & 7) * 8; }

// Panels of h from the sums in `red`, of which every CTA of the cluster holds a part: each CTA adds up and stores its share of the tokens,
// zeros in panels of adapters that are not the token's and in the padding of its own: a row with an infinite value has sums there that are no
// numbers, and these would stay so through the padding's zeros in B.  panel_at(g) is the g-th of the np panels.
template <int PITCH, bool TOKEN_MAJOR, int TOKENS, typename PanelAt>
__device__ __forceinline__ void store_low_rows(const LowArgs& a, const float* red, const int* who, const float* scale, const short (*ranks)[MAX_SECTIONS],
                                               PanelAt panel_at, int np, int token0, int tile) {
  const int cs = gridDim.z, share = TOKENS / cs, first = blockIdx.z * share, shift = __ffs(share) - 1;   // a power of two
  bf16* const h = a.h + (size_t)tile * a.capacity * a.all_panels * a.tile_rows * 16;
  for (int i = threadIdx.x; i < np * share * 2; i += TC_THREADS) {   // items of eight ranks
    const int half = (i >> shift) & 1, c = first + (i & (share - 1)), g = i >> (1 + shift), p = panel_at(g), own = p - who[c] * a.all_panels;
    uint4 o = make_uint4(0, 0, 0, 0);
    int left = 0;   // of these eight ranks, the adapter has so many
    if (who[c] >= 0 && own >= 0 && own < a.all_panels) {
      const int section = own / a.panels;
      left = ranks[c][section] - (own - section * a.panels) * 16 - half * 8;
    }
    if (left > 0) {
      const float* const mine = red + (TOKEN_MAJOR ? c * PITCH + g * 16 : (g * TOKENS + c) * PITCH) + half * 8;
      const float4 v = cluster_sum4(mine, cs), u = cluster_sum4(mine + 4, cs);
      const float f = scale[c];
      const uint2 lo = pack4(make_float4(v.x * f, left > 1 ? v.y * f : 0.0f, left > 2 ? v.z * f : 0.0f, left > 3 ? v.w * f : 0.0f));
      const uint2 hi = pack4(make_float4(left > 4 ? u.x * f : 0.0f, left > 5 ? u.y * f : 0.0f, left > 6 ? u.z * f : 0.0f, left > 7 ? u.w * f : 0.0f));
      o = make_uint4(lo.x, lo.y, hi.x, hi.y);
    }
    *reinterpret_cast<uint4*>(h + (size_t)p * a.tile_rows * 16 + in_panel(token0 - tile * PLAN_TILE + c, half)) = o;
  }
}

// Decode steps, one tile of BN tokens: the panels' rows of A are the MMA's 128 rows (G runs of eight panels at a time), the tokens its
// columns.  Cluster (1, 1, CS) splits K.
template <int BN, int G>
__global__ void __launch_bounds__(TC_THREADS, 1)
adapter_low_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmX, const LowArgs a) {
  constexpr int TMEM_COLS = G * BN < 32 ? 32 : G * BN, X_AT = G * W_BYTES, STAGE = X_AT + BN * 128, PITCH = G * 128 + 4;
  // The projection starts now: what it reads besides h comes from kernels that are done when the last block is here, so it streams its
  // weights meanwhile and waits for this kernel only before its panels.
  pdl_wait();   // tokens and plan come from the previous kernels, and h may still be read by them
  pdl_launch_dependents();
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* const red = reinterpret_cast<float*>(smem);   // the ring's memory, between two passes
  const int stages = a.stages;
  const size_t ring = max((size_t)stages * STAGE, (size_t)BN * PITCH * 4);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + ring);
  uint64_t* empty = full + stages;
  uint64_t* acc_full = empty + stages;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_full + 1);
  const int warp = uniform_warp(), lane = threadIdx.x & 31;
  const int panels = min(a.counts[0], min(a.capacity, BN)) * a.all_panels;
  __shared__ int who[BN], slot[BN];   // no more adapters than tokens
  __shared__ float scale[BN];
  __shared__ short ranks[BN][MAX_SECTIONS];

  const int kb0 = part_begin(a.kb, blockIdx.z, gridDim.z), kb1 = part_begin(a.kb, blockIdx.z + 1, gridDim.z);
  // the first tokens are under way before the list of adapters is read; their bytes are announced with those of the factors
  const int pass = G * 8 / a.run * a.run;   // panels of a pass
  const int pre = (int)blockIdx.x * pass < panels ? min(stages, kb1 - kb0) : 0;
  if (warp == 0 && elect_one()) {
    for (int s = 0; s < stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(acc_full, 1);
    fence_barrier_init();
    for (int i = 0; i < pre; ++i) tma_load_2d(smem + (size_t)i * STAGE + X_AT, &tmX, &full[i], (kb0 + i) * 64, 0);
    tma_prefetch_desc(&tmA);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, TMEM_COLS);
    tmem_relinquish();
  }
  load_owners<BN, BN>(a, who, slot, 0, 0);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  int s = 0, round = 0;   // ring stage; passes done
  uint32_t parity = 0;    // of the full barriers (MMA); the producer waits for the phase before
  bool ok = true;         // this thread's role goes on; after a wait that ran out it only keeps step with the cluster
  for (int p0 = blockIdx.x * pass; p0 < panels; p0 += gridDim.x * pass, ++round) {
    const int np = min(pass, panels - p0);
    if (warp == 0) {
      if (elect_one() && ok) {
        int row[G * 8];
#pragma unroll
        for (int i = 0; i < G * 8; ++i) {
          const int p = p0 + min(i * a.run, np - 1), j = p / a.all_panels;
          row[i] = (slot[j] * a.all_panels + (p - j * a.all_panels)) * 16;
        }
        for (int kb = kb0; kb < kb1; ++kb) {
          ok = mbar_wait(&empty[s], parity ^ 1, 1);
          if (!ok) break;
          uint8_t* const st = smem + (size_t)s * STAGE;
          mbar_expect_tx(&full[s], np * 2048 + BN * 128);
          if (round > 0 || kb - kb0 >= pre) tma_load_2d(st + X_AT, &tmX, &full[s], kb * 64, 0);
#pragma unroll
          for (int i = 0; i < G * 8; ++i)
            if (i * a.run < np) tma_load_2d(st + i * a.run * 2048, &tmA, &full[s], kb * 64, row[i]);
          if (++s == stages) s = 0, parity ^= 1;
        }
        if (!ok) {
          // unwinding: copies already in flight land before shared memory is used for the sums
          for (int j = 0; j < stages; ++j) {
            if (--s < 0) s = stages - 1, parity ^= 1;
            (void)mbar_wait(&full[s], parity, 4);
          }
        }
      }
    } else if (warp == 1) {
      if (elect_one() && ok) {
        constexpr uint32_t idesc = umma_idesc_bf16(128, BN);
        for (int kb = kb0; kb < kb1; ++kb) {
          ok = mbar_wait(&full[s], parity, 2);
          if (!ok) break;
          tc_fence_after();
          const uint32_t st = smem_u32(smem + (size_t)s * STAGE);
          const uint64_t db = umma_desc_sw128(st + X_AT);
#pragma unroll
          for (int g = 0; g < G; ++g)
            if (g * 8 < np) {
              const uint64_t da = umma_desc_sw128(st + g * W_BYTES);
#pragma unroll
              for (int k = 0; k < 4; ++k) tc_mma_f16(tmem + g * BN, da + 2 * k, db + 2 * k, idesc, kb != kb0 || k != 0);
            }
          tc_commit(&empty[s]);
          if (++s == stages) s = 0, parity ^= 1;
        }
        if (ok) tc_commit(acc_full);
      }
    } else {
      if (round == 0) load_scales<BN>(a, who, slot, scale, ranks);
      // rows of unused panels hold what earlier loads left; nothing reads them
      ok = ok && __all_sync(0xffffffffu, mbar_wait(acc_full, round & 1, 3));
      if (ok) {
        tc_fence_after();
        for (int g = 0; g * 8 < np; ++g) accumulator_to_smem<BN, PITCH>(tmem + g * BN, red + g * 128, warp & 3, lane, BN);
      }
    }
    tc_fence_before();
    __syncwarp();
    cluster_sync_all();
    tc_fence_after();
    store_low_rows<PITCH, true, BN>(a, red, who, scale, ranks, [&](int g) { return p0 + g; }, np, 0, 0);
    // the ring is written again by copies once every CTA has read the sums
    fence_proxy_async();
    cluster_sync_all();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, TMEM_COLS);
  }
}

constexpr int LOW_PASS = 16, LOW_STAGES = 12;
constexpr int LOW_PITCH = 20;            // floats of a row of 16 sums, without bank conflicts
constexpr int LOW_RING = 208 * 1024;     // bytes; the sums of a pass (160 KB) take the same place

// Prompts, 128 tokens: the tokens are the MMA's rows and up to 16 panels its columns, those of the adapters that these tokens have, so that a
// k-block moves the tokens once and the factors of these adapters; the panels of the tile's other adapters get zeros.  Cluster (1, 1, CS)
// splits K; where token tiles are few, blocks side by side take 16 panels each (512 tokens of 256 adapters of rank 16, 4096 -> 4096: 223 us a
// call one after another, 120 so).
__global__ void __launch_bounds__(TC_THREADS, 1)
adapter_low_prompt_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmX, const LowArgs a) {
  constexpr int PASS = LOW_PASS, TMEM_COLS = PASS * 16, PITCH = LOW_PITCH;
  pdl_wait();
  pdl_launch_dependents();   // as above
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* const red = reinterpret_cast<float*>(smem);   // [panel of the pass][token][PITCH], in the ring's memory
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + LOW_RING);
  uint64_t* empty = full + LOW_STAGES;
  uint64_t* acc_full = empty + LOW_STAGES;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_full + 1);
  const int warp = uniform_warp(), lane = threadIdx.x & 31;
  const int token0 = blockIdx.y * 128, tile = token0 / PLAN_TILE;
  const int count = min(a.counts[tile], a.capacity), pass = PASS / a.run * a.run, p_first = blockIdx.x * pass;
  if (p_first > 0 && p_first >= count * a.all_panels) return;   // blocks for more adapters than the tile has
  __shared__ int who[128], slot[PLAN_TILE];
  __shared__ float scale[128];
  __shared__ short ranks[128][MAX_SECTIONS];
  __shared__ short place[PLAN_TILE], active[128];   // of the list's adapters: which of the active ones, -1: none; and back
  __shared__ int n_active;
  for (int j = threadIdx.x; j < count; j += TC_THREADS) place[j] = -1;

  const int kb0 = part_begin(a.kb, blockIdx.z, gridDim.z), kb1 = part_begin(a.kb, blockIdx.z + 1, gridDim.z);
  // as many stages as the ring holds for the panels that these tokens may have
  const int stage = W_BYTES + min(pass, count * a.all_panels) * 2048, stages = min(LOW_STAGES, LOW_RING / stage);
  const int pre = count > 0 ? min(stages, kb1 - kb0) : 0;   // as above
  if (warp == 0 && elect_one()) {
    for (int s = 0; s < stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(acc_full, 1);
    fence_barrier_init();
    for (int i = 0; i < pre; ++i) tma_load_2d(smem + (size_t)i * stage, &tmX, &full[i], (kb0 + i) * 64, token0);
    tma_prefetch_desc(&tmA);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, TMEM_COLS);
    tmem_relinquish();
  }
  load_owners<128, PLAN_TILE>(a, who, slot, token0, tile);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  if (threadIdx.x < 128 && who[threadIdx.x] >= 0) place[who[threadIdx.x]] = 0;
  __syncthreads();
  if (warp == 2) {
    int n = 0;
    for (int j0 = 0; j0 < count; j0 += 32) {
      const int j = j0 + lane;
      const bool used = j < count && place[j] >= 0;
      const unsigned votes = __ballot_sync(0xffffffffu, used);
      const int at = n + __popc(votes & ((1u << lane) - 1));
      if (used) {
        place[j] = (short)at;
        active[at] = (short)j;
      }
      n += __popc(votes);
    }
    if (lane == 0) n_active = n;
  }
  __syncthreads();
  const int panels = n_active * a.all_panels;
  if (p_first >= panels && warp == 0 && elect_one()) {   // the tokens loaded ahead are not needed: only let them land
    for (int i = 0; i < pre; ++i) {
      mbar_expect_tx(&full[i], W_BYTES);
      (void)mbar_wait(&full[i], 0, 4);
    }
  }
  if (blockIdx.x == 0 && warp >= 2) {   // zeros for adapters that only the tile's other 128 tokens have
    const int cs = gridDim.z, share = 128 / cs;
    bf16* const h = a.h + (size_t)tile * a.capacity * a.all_panels * a.tile_rows * 16;
    for (int j = 0; j < count; ++j)
      if (place[j] < 0)
        for (int i = threadIdx.x - 64; i < a.all_panels * share * 2; i += 128)
          *reinterpret_cast<uint4*>(h + ((size_t)j * a.all_panels + i / (share * 2)) * a.tile_rows * 16 +
                                    in_panel(token0 - tile * PLAN_TILE + blockIdx.z * share + (i >> 1) % share, i & 1)) = make_uint4(0, 0, 0, 0);
  }

  int s = 0, round = 0;
  uint32_t parity = 0;
  bool ok = true;
  for (int p0 = p_first; p0 < panels; p0 += gridDim.x * pass, ++round) {
    const int np = min(pass, panels - p0);
    if (warp == 0) {
      if (elect_one() && ok) {
        int row[PASS];
#pragma unroll
        for (int i = 0; i < PASS; ++i) {
          const int p = p0 + min(i * a.run, np - 1), j = p / a.all_panels;
          row[i] = (slot[active[j]] * a.all_panels + (p - j * a.all_panels)) * 16;
        }
        for (int kb = kb0; kb < kb1; ++kb) {
          ok = mbar_wait(&empty[s], parity ^ 1, 1);
          if (!ok) break;
          uint8_t* const st = smem + (size_t)s * stage;
          mbar_expect_tx(&full[s], W_BYTES + np * 2048);
          if (round > 0 || kb - kb0 >= pre) tma_load_2d(st, &tmX, &full[s], kb * 64, token0);
#pragma unroll
          for (int i = 0; i < PASS; ++i)
            if (i * a.run < np) tma_load_2d(st + W_BYTES + i * a.run * 2048, &tmA, &full[s], kb * 64, row[i]);
          if (++s == stages) s = 0, parity ^= 1;
        }
        if (!ok) {
          for (int j = 0; j < stages; ++j) {
            if (--s < 0) s = stages - 1, parity ^= 1;
            (void)mbar_wait(&full[s], parity, 4);
          }
        }
      }
    } else if (warp == 1) {
      if (elect_one() && ok) {
        const uint32_t idesc = umma_idesc_bf16(128, np * 16);
        for (int kb = kb0; kb < kb1; ++kb) {
          ok = mbar_wait(&full[s], parity, 2);
          if (!ok) break;
          tc_fence_after();
          const uint32_t st = smem_u32(smem + (size_t)s * stage);
          const uint64_t da = umma_desc_sw128(st), db = umma_desc_sw128(st + W_BYTES);
#pragma unroll
          for (int k = 0; k < 4; ++k) tc_mma_f16(tmem, da + 2 * k, db + 2 * k, idesc, kb != kb0 || k != 0);
          tc_commit(&empty[s]);
          if (++s == stages) s = 0, parity ^= 1;
        }
        if (ok) tc_commit(acc_full);
      }
    } else {
      if (round == 0) load_scales<128>(a, who, slot, scale, ranks);
      const int q = warp & 3, c = q * 32 + lane, first_own = who[c] < 0 ? panels : place[who[c]] * a.all_panels;
      ok = ok && __all_sync(0xffffffffu, mbar_wait(acc_full, round & 1, 3));
      if (ok) {
        tc_fence_after();
        for (int g = 0; g < np; ++g) {
          const bool keep = p0 + g >= first_own && p0 + g < first_own + a.all_panels;
          if (!__any_sync(0xffffffffu, keep)) continue;
          uint32_t r[16];
          tmem_ld16(tmem + ((uint32_t)(q * 32) << 16) + g * 16, r);
          tmem_ld_wait();
          float4* const dst = reinterpret_cast<float4*>(red + (g * 128 + c) * PITCH);
          if (keep)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              dst[e] = make_float4(__uint_as_float(r[4 * e]), __uint_as_float(r[4 * e + 1]), __uint_as_float(r[4 * e + 2]), __uint_as_float(r[4 * e + 3]));
        }
      }
    }
    tc_fence_before();
    __syncwarp();
    cluster_sync_all();
    tc_fence_after();
    auto panel_at = [&](int g) {
      const int k = (p0 + g) / a.all_panels;
      return active[k] * a.all_panels + (p0 + g - k * a.all_panels);
    };
    store_low_rows<PITCH, false, 128>(a, red, who, scale, ranks, panel_at, np, token0, tile);
    fence_proxy_async();
    cluster_sync_all();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, TMEM_COLS);
  }
}

struct TileArgs {
  const int* lists;
  const int* counts;
  const bf16* bias;      // [M] (null: none)
  bf16* out;             // [T][ldo]
  long long ldo;
  int T, M, kb, capacity, panels, all_panels, tile_rows, stages;
  int act;               // DUAL: PRISM_GLU_*
  int b_groups, no_group;   // groups of 8 features in a panel of B; a group behind all of them, which reads as zeros
  int vec;               // four features of a row can be stored at once
  int sections;
  int start[MAX_SECTIONS], end[MAX_SECTIONS], first_tile[MAX_SECTIONS], b_start[MAX_SECTIONS];   // b_start: in groups
};

// 128 features (DUAL: 64 gates and their 64 ups) of BN tokens.  Weights are the A operand and stream once; cluster (1, 1, CS) splits the
// k-blocks and the panels of the tile's adapters, and adds the parts through shared memory.
template <int BN, bool DUAL>
__global__ void __launch_bounds__(TC_THREADS, 1)
adapter_gemm_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmB,
                    const __grid_constant__ CUtensorMap tmH, const TileArgs a) {
  constexpr int TMEM_COLS = BN < 32 ? 32 : BN, STAGE = stage_bytes<BN>(), FEATURES = DUAL ? 64 : 128;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* const red = reinterpret_cast<float*>(smem);   // the ring's memory, once the sums are done
  const int stages = a.stages;
  const size_t ring = max((size_t)stages * STAGE, (size_t)BN * RED_PITCH * 4);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + ring);
  uint64_t* empty = full + stages;
  uint64_t* acc_full = empty + stages;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_full + 1);
  const int warp = uniform_warp(), lane = threadIdx.x & 31;
  const int cs = gridDim.z, z = blockIdx.z, token0 = blockIdx.y * BN, tile = token0 / PLAN_TILE;
  int section = 0;
  if (!DUAL)
    while (section + 1 < a.sections && (int)blockIdx.x >= a.first_tile[section + 1]) ++section;
  const int f0 = DUAL ? blockIdx.x * FEATURES : a.start[section] + ((int)blockIdx.x - a.first_tile[section]) * FEATURES;
  const int f_end = DUAL ? a.M / 2 : a.end[section];

  const int kb0 = part_begin(a.kb, z, cs), kb1 = part_begin(a.kb, z + 1, cs);
  const int pre = min(stages, kb1 - kb0);
  auto load_block = [&](int s, int kb) {
    uint8_t* const st = smem + (size_t)s * STAGE;
    mbar_expect_tx(&full[s], STAGE);
    tma_load_2d(st, &tmW, &full[s], kb * 64, f0);
    if (DUAL) tma_load_2d(st + W_BYTES / 2, &tmW, &full[s], kb * 64, a.M / 2 + f0);
    tma_load_2d(st + W_BYTES, &tmX, &full[s], kb * 64, token0);
  };
  if (warp == 0 && elect_one()) {
    for (int s = 0; s < stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(acc_full, 1);
    fence_barrier_init();
    for (int i = 0; i < pre; ++i) load_block(i, kb0 + i);   // the first ring is under way before anything else is set up
    tma_prefetch_desc(&tmB);
    tma_prefetch_desc(&tmH);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, TMEM_COLS);
    tmem_relinquish();
  }
  // The plan's kernel is done, but this one has not waited for it: list and count come from L2, past what an older kernel left in L1.
  __shared__ int list[PLAN_TILE];
  for (int j = (int)threadIdx.x - 64; j >= 0 && j < a.capacity; j += TC_THREADS - 64) list[j] = __ldcg(a.lists + (size_t)tile * a.capacity + j);
  const int count = min(__ldcg(a.counts + tile), a.capacity);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_launch_dependents();

  const int per = DUAL ? a.all_panels : a.panels, extra = count * per;   // panels of one adapter that reach this tile, and of all its adapters
  if (warp == 0) {
    if (elect_one()) {
      // this CTA's panels: adapter j of the list, panel rp of its section (of: of all sections)
      const int e_begin = part_begin(extra, z, cs), e_end = part_begin(extra, z + 1, cs), of0 = DUAL ? 0 : section * a.panels;
      int j = e_begin / per, of = of0 + (e_begin - j * per), rp = of % a.panels;
      const int b_at = DUAL ? f0 / 8 : a.b_start[section] + (f0 - a.start[section]) / 8;
      int s = 0;
      uint32_t parity = 1;   // a fresh empty barrier counts as free
      bool ok = true;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (kb - kb0 >= pre) {
          ok = mbar_wait(&empty[s], parity, 1);
          if (!ok) break;
          load_block(s, kb);
        }
        if (++s == stages) s = 0, parity ^= 1;
      }
      pdl_wait();   // the low-rank rows
      for (int e0 = e_begin; e0 < e_end && ok; e0 += 4) {
        const int n = min(4, e_end - e0);
        ok = mbar_wait(&empty[s], parity, 1);
        if (!ok) break;
        uint8_t* const st = smem + (size_t)s * STAGE;
        mbar_expect_tx(&full[s], n * (4096 + BN * 32));
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (i < n) {
            const int group = (list[j] * a.panels + rp) * a.b_groups + b_at;
            if (DUAL) {   // a gate's panel adds nothing to the up half, and the other way round
              const bool up = of >= a.panels;
              tma_load_2d(st + i * 4096, &tmB, &full[s], 0, up ? a.no_group : group);
              tma_load_2d(st + i * 4096 + 2048, &tmB, &full[s], 0, up ? group + a.b_start[1] : a.no_group);
            } else {
              tma_load_2d(st + i * 4096, &tmB, &full[s], 0, group);
            }
            tma_load_2d(st + W_BYTES + i * BN * 32, &tmH, &full[s], 0,
                        (((tile * a.capacity + j) * a.all_panels + of) * a.tile_rows + (token0 - tile * PLAN_TILE)) / 8);
            ++of;
            if (++rp == a.panels) {
              rp = 0;
              if (!DUAL || of == a.all_panels) {
                of = of0;
                ++j;
              }
            }
          }
        if (++s == stages) s = 0, parity ^= 1;
      }
      if (!ok) {
        // unwinding after a timed-out wait: copies already in flight land before shared memory is used for the sums
        for (int j = 0; j < stages; ++j) {
          if (--s < 0) s = stages - 1, parity ^= 1;
          (void)mbar_wait(&full[s], parity ^ 1, 4);
        }
      }
    }
  } else if (warp == 1) {
    if (elect_one()) {
      constexpr uint32_t idesc = umma_idesc_bf16(128, BN);
      int s = 0;
      uint32_t parity = 0;
      bool ok = true;
      for (int kb = kb0; kb < kb1; ++kb) {
        ok = mbar_wait(&full[s], parity, 2);
        if (!ok) break;
        tc_fence_after();
        const uint32_t st = smem_u32(smem + (size_t)s * STAGE);
        const uint64_t da = umma_desc_sw128(st), db = umma_desc_sw128(st + W_BYTES);
#pragma unroll
        for (int k = 0; k < 4; ++k) tc_mma_f16(tmem, da + 2 * k, db + 2 * k, idesc, kb != kb0 || k != 0);
        tc_commit(&empty[s]);
        if (++s == stages) s = 0, parity ^= 1;
      }
      const int e_end = part_begin(extra, z + 1, cs);
      for (int e0 = part_begin(extra, z, cs); e0 < e_end && ok; e0 += 4) {
        ok = mbar_wait(&full[s], parity, 2);
        if (!ok) break;
        tc_fence_after();
        const uint32_t st = smem_u32(smem + (size_t)s * STAGE);
        for (int i = 0; i < min(4, e_end - e0); ++i)
          tc_mma_f16(tmem, umma_desc_panel(st + i * 4096), umma_desc_panel(st + W_BYTES + i * BN * 32), idesc, 1);
        tc_commit(&empty[s]);
        if (++s == stages) s = 0, parity ^= 1;
      }
      if (ok) tc_commit(acc_full);
    }
  } else {
    pdl_wait();
    if (__all_sync(0xffffffffu, mbar_wait(acc_full, 0, 3))) {
      tc_fence_after();
      accumulator_to_smem<BN, RED_PITCH>(tmem, red, warp & 3, lane, min(BN, a.T - token0));
    }
  }
  tc_fence_before();
  __syncwarp();
  cluster_sync_all();
  // items of four features of a token, features fastest, shared out among the CTAs of the cluster
  constexpr int QUADS = FEATURES / 4;
  const int items = min(BN, a.T - token0) * QUADS;
  for (int i = part_begin(items, z, cs) + threadIdx.x; i < part_begin(items, z + 1, cs); i += TC_THREADS) {
    const int c = i / QUADS, f = f0 + (i % QUADS) * 4, n = min(4, f_end - f);
    if (n <= 0) continue;
    float4 v = cluster_sum4(red + c * RED_PITCH + (i % QUADS) * 4, cs);
    float* const x = &v.x;
    if (DUAL) {
      const float4 u = cluster_sum4(red + c * RED_PITCH + 64 + (i % QUADS) * 4, cs);
      v = make_float4(glu(v.x, u.x, a.act), glu(v.y, u.y, a.act), glu(v.z, u.z, a.act), glu(v.w, u.w, a.act));
    } else if (a.bias != nullptr) {
      for (int e = 0; e < n; ++e) x[e] += __bfloat162float(a.bias[f + e]);
    }
    bf16* const dst = a.out + (size_t)(token0 + c) * a.ldo + f;
    if (a.vec && n == 4) *reinterpret_cast<uint2*>(dst) = pack4(v);
    else
      for (int e = 0; e < n; ++e) dst[e] = __float2bfloat16_rn(x[e]);
  }
  // nobody leaves while a peer may read its sums
  cluster_sync_all();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, TMEM_COLS);
  }
}

// ------------------------------------------------------------------------------------------------------------------------------------
// fp32: true 32-bit multiply-adds.  The low-rank rows first, a block per token; then the projection in tiles of 64 features, whose epilogue adds
// each token's low-rank term.  Clusters split K where the tiles are few.
// Sums run over 128 products in one accumulator, which is then added to another: a plain chain over K = 7064 was off by five times as much
// (1.1e-6 of the outputs' scale against 2e-7).
// ------------------------------------------------------------------------------------------------------------------------------------
struct LowF32Args {
  const float* x;       // [T][ldx]
  const float* a;       // [slots][low][K]
  const float* scale;   // [slots]
  const int* ranks;     // [slots][sections]
  const int* adapter;   // [T]
  float* h;             // [T][low]; rows of tokens without an adapter are not written
  int K, low, slots, padded;   // padded: ranks of a section
  long long ldx;
};

// Four consecutive values, zeros behind the end.  VEC: rows are whole 16-byte vectors, and the load is a single predicated one; with a branch
// around it loads waited for one another.  From L2: the projection starts before it has waited for the kernels whose results it reads here
// (they are done), so nothing may come from a line that an older kernel left in L1.
template <bool VEC>
__device__ __forceinline__ float4 load4(const float* p, int k, int K) {
  if (VEC) return k < K ? __ldcg(reinterpret_cast<const float4*>(p + k)) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  return make_float4(k < K ? __ldcg(p + k) : 0.0f, k + 1 < K ? __ldcg(p + k + 1) : 0.0f, k + 2 < K ? __ldcg(p + k + 2) : 0.0f,
                     k + 3 < K ? __ldcg(p + k + 3) : 0.0f);
}

// A warp per two rows of A, whose sums it keeps in four parts per lane.
template <bool VEC>
__global__ void __launch_bounds__(256) adapter_low_f32_kernel(const LowF32Args a) {
  const int t = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  pdl_wait();
  pdl_launch_dependents();   // the projection reads h last
  const int who = a.adapter[t];
  if (who < 0 || who >= a.slots) return;
  const float* const x = a.x + (size_t)t * a.ldx;
  const float scale = a.scale[who];
  for (int r = (blockIdx.y * 8 + warp) * 2; r < a.low; r += gridDim.y * 16) {
    const float* const row = a.a + ((size_t)who * a.low + r) * a.K;
    float4 s0 = make_float4(0, 0, 0, 0), s1 = s0;
    for (int k0 = lane * 4; k0 < a.K; k0 += 4 * 128) {   // twelve loads under way at a time
      float4 v[4], p[4], q[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[i] = load4<VEC>(x, k0 + i * 128, a.K);
        p[i] = load4<VEC>(row, k0 + i * 128, a.K);
        q[i] = load4<VEC>(row + a.K, k0 + i * 128, a.K);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s0 = make_float4(fmaf(v[i].x, p[i].x, s0.x), fmaf(v[i].y, p[i].y, s0.y), fmaf(v[i].z, p[i].z, s0.z), fmaf(v[i].w, p[i].w, s0.w));
        s1 = make_float4(fmaf(v[i].x, q[i].x, s1.x), fmaf(v[i].y, q[i].y, s1.y), fmaf(v[i].z, q[i].z, s1.z), fmaf(v[i].w, q[i].w, s1.w));
      }
    }
    const float u = warp_sum((s0.x + s0.y) + (s0.z + s0.w)), w = warp_sum((s1.x + s1.y) + (s1.z + s1.w));
    // zeros in the padding, as in bf16; both rows are of one section
    const int section = r / a.padded, rank = a.ranks[who * (a.low / a.padded) + section];
    if (lane < 2) a.h[(size_t)t * a.low + r + lane] = r + lane - section * a.padded < rank ? (lane ? w : u) * scale : 0.0f;
  }
}

struct TileF32Args {
  const float* x;       // [T][ldx]
  const float* w;       // [M][ldw]
  const float* b;       // [slots][panels][b_rows][16]
  const float* h;       // [T][low]
  const float* bias;    // [M] (null: none)
  const int* adapter;   // [T]
  float* out;           // [T][ldo]
  int T, M, K, low, panels, slots, b_rows, act;
  long long ldx, ldw, ldo;
  int sections;
  int end[MAX_SECTIONS], shift[MAX_SECTIONS];   // shift: of a section's features in b
};

__device__ __forceinline__ float glu_f32(float z, float u, int act) {
  return (act == PRISM_GLU_GELU_TANH ? 0.5f * z * (1.0f + tanhf(0.7978845608028654f * (z + 0.044715f * z * z * z))) : z / (1.0f + expf(-z))) * u;
}

// Low-rank term of feature m for the token whose row of h is given.
__device__ __forceinline__ float low_term(const TileF32Args& a, const float* h, int who, int m) {
  int s = 0;
  while (s + 1 < a.sections && m >= a.end[s]) ++s;
  h += s * a.panels * 16;
  float sum = 0.0f;
  for (int p = 0; p < a.panels; ++p) {
    const float4* const b = reinterpret_cast<const float4*>(a.b + (((size_t)who * a.panels + p) * a.b_rows + m + a.shift[s]) * 16);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float4 v = b[e], g = *reinterpret_cast<const float4*>(h + p * 16 + e * 4);
      sum += (v.x * g.x + v.y * g.y) + (v.z * g.z + v.w * g.w);
    }
  }
  return sum;
}

constexpr int F32_THREADS = 128, F32_SUM = 128;   // F32_SUM products per accumulator
__host__ __device__ constexpr int f32_chunk(int nt) { return nt == 2 ? 64 : 16; }   // columns of a chunk: few tokens are bound by the weights under way

// A thread sums NF of the tile's 64 features for NT tokens.  8 x 8 from 65 tokens: 4 loads of 16 bytes from shared memory feed 64 multiply-adds,
// where 4 x 8 was bound by these loads (300 tokens, 2048 -> 4096: 297 us with 4 x 8, 196 us with 8 x 8 though a quarter of its tokens is
// padding; 700 tokens, 4096 -> 4096: 689 us, 34 TFLOP/s).  Chunks are stored k by k; runs of features or tokens change places with k / 4, which
// keeps stores and loads clear of bank conflicts (1.6 million of them in 0.54 million stores without).
template <int NF, int NT, bool DUAL, bool VEC>
__global__ void __launch_bounds__(F32_THREADS, NF == 8 ? 3 : 4) adapter_gemm_f32_kernel(const TileF32Args a) {
  constexpr int KC = f32_chunk(NT), QUADS_K = KC / 4, ROWS = F32_THREADS / QUADS_K, FOLD = F32_SUM / KC;
  constexpr int FX = 64 / NF, TG = F32_THREADS / FX, TN = TG * NT;   // threads side by side over the features, groups of tokens
  constexpr int WP = 68, XP = TN + 4, W_LOADS = 64 / ROWS, LOADS = (TN + ROWS - 1) / ROWS, QUADS = DUAL ? 8 : 16, RED = 68;
  extern __shared__ float4 smem_f32[];
  float* const smem = reinterpret_cast<float*>(smem_f32);
  float (*const ws)[KC][WP] = reinterpret_cast<float (*)[KC][WP]>(smem);
  float (*const xs)[KC][XP] = reinterpret_cast<float (*)[KC][XP]>(smem + 2 * KC * WP);
  float* const red = smem + 2 * KC * (WP + XP);   // the sums so far: registers hold those of the last chunks only
  const int cs = gridDim.z, z = blockIdx.z, tid = threadIdx.x;
  const int f0 = blockIdx.x * (DUAL ? 32 : 64), t0 = blockIdx.y * TN, half = a.M / 2;
  const int chunks = (a.K + KC - 1) / KC, c0 = part_begin(chunks, z, cs), c1 = part_begin(chunks, z + 1, cs);
  const int quad = tid % QUADS_K, line = tid / QUADS_K;   // the four columns of a chunk and the rows that this thread copies
  auto turn_of = [](int q) { return KC == 16 ? q << 3 : (q & 7) << 2; };
  // row i of the weight tile; a row outside the matrix reads as zeros
  auto w_row = [&](int i) { return DUAL ? (i < 32 ? (f0 + i < half ? f0 + i : -1) : (f0 + i - 32 < half ? half + f0 + i - 32 : -1)) : (f0 + i < a.M ? f0 + i : -1); };
  float4 wr[W_LOADS], xr[LOADS];
  auto fetch = [&](int chunk) {
    const int k = chunk * KC + quad * 4;
#pragma unroll
    for (int i = 0; i < W_LOADS; ++i) {
      const int r = w_row(line + i * ROWS);
      wr[i] = r < 0 ? make_float4(0, 0, 0, 0) : load4<VEC>(a.w + (size_t)r * a.ldw, k, a.K);
    }
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int c = line + i * ROWS;
      xr[i] = c < TN && t0 + c < a.T ? load4<VEC>(a.x + (size_t)(t0 + c) * a.ldx, k, a.K) : make_float4(0, 0, 0, 0);
    }
  };
  auto keep = [&](int buf) {
    const int k = quad * 4;
#pragma unroll
    for (int i = 0; i < W_LOADS; ++i) {
      const int r = (line + i * ROWS) ^ turn_of(quad);
      ws[buf][k][r] = wr[i].x, ws[buf][k + 1][r] = wr[i].y, ws[buf][k + 2][r] = wr[i].z, ws[buf][k + 3][r] = wr[i].w;
    }
#pragma unroll
    for (int i = 0; i < LOADS; ++i)
      if (line + i * ROWS < TN) {
        const int r = (line + i * ROWS) ^ (turn_of(quad) & (TN - 1));
        xs[buf][k][r] = xr[i].x, xs[buf][k + 1][r] = xr[i].y, xs[buf][k + 2][r] = xr[i].z, xs[buf][k + 3][r] = xr[i].w;
      }
  };
  // this thread's features fx .. + 4 (and 32 further on) and tokens tx .. + 4 (and TG * 4 further on; NT 2: tx .. + 2)
  const int fx = (tid % FX) * 4, tx = (tid / FX) * (NT < 4 ? NT : 4);
  float acc[NT][NF] = {};
  pdl_launch_dependents();
  fetch(c0);
  keep(0);
  __syncthreads();
  for (int c = c0; c < c1; ++c) {
    const int buf = (c - c0) & 1;
    if (c + 1 < c1) fetch(c + 1);
#pragma unroll
    for (int k = 0; k < KC; ++k) {
      const int turn = turn_of(k >> 2);
      float w[NF], x[NT];
#pragma unroll
      for (int e = 0; e < NF; e += 4) *reinterpret_cast<float4*>(&w[e]) = *reinterpret_cast<const float4*>(&ws[buf][k][(fx + e * 8) ^ turn]);
      if (NT < 4) {
        *reinterpret_cast<float2*>(x) = *reinterpret_cast<const float2*>(&xs[buf][k][tx ^ (turn & (TN - 1))]);
      } else {
#pragma unroll
        for (int i = 0; i < NT; i += 4) *reinterpret_cast<float4*>(&x[i]) = *reinterpret_cast<const float4*>(&xs[buf][k][(tx + i * TG) ^ turn]);
      }
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int e = 0; e < NF; ++e) acc[i][e] = fmaf(x[i], w[e], acc[i][e]);
    }
    if ((c - c0) % FOLD == FOLD - 1 || c + 1 == c1) {
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int e = 0; e < NF; e += 4) {
          float4* const sum = reinterpret_cast<float4*>(&red[(NT < 4 ? tx + i : tx + (i & 3) + (i >> 2) * 4 * TG) * RED + fx + e * 8]);
          float4 v = make_float4(acc[i][e], acc[i][e + 1], acc[i][e + 2], acc[i][e + 3]);
          if (c - c0 >= FOLD) v = add4(*sum, v);
          *sum = v;
          acc[i][e] = acc[i][e + 1] = acc[i][e + 2] = acc[i][e + 3] = 0.0f;
        }
    }
    if (c + 1 < c1) keep(buf ^ 1);
    __syncthreads();
  }
  pdl_wait();   // the low-rank rows
  cluster_sync_all();
  const int items = min(TN, a.T - t0) * QUADS;
  for (int i = part_begin(items, z, cs) + tid; i < part_begin(items, z + 1, cs); i += F32_THREADS) {
    const int c = i / QUADS, f = f0 + (i % QUADS) * 4, n = min(4, (DUAL ? half : a.M) - f);
    if (n <= 0) continue;
    const int who_raw = a.adapter[t0 + c], who = who_raw < a.slots ? who_raw : -1;
    const float* const h = a.h + (size_t)(t0 + c) * a.low;
    const float4 v = cluster_sum4(red + c * RED + (i % QUADS) * 4, cs);
    float y[4] = {v.x, v.y, v.z, v.w};
    float u[4] = {};
    if (DUAL) {
      const float4 r = cluster_sum4(red + c * RED + 32 + (i % QUADS) * 4, cs);
      u[0] = r.x, u[1] = r.y, u[2] = r.z, u[3] = r.w;
    }
    float* const dst = a.out + (size_t)(t0 + c) * a.ldo + f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (e >= n) break;
      if (a.bias != nullptr) y[e] += a.bias[f + e];
      if (who >= 0) y[e] += low_term(a, h, who, f + e);
      if (DUAL) {
        if (who >= 0) u[e] += low_term(a, h, who, half + f + e);
        y[e] = glu_f32(y[e], u[e], a.act);
      }
      dst[e] = y[e];
    }
  }
  cluster_sync_all();   // nobody leaves while a peer may read its sums
}

constexpr int SMS = 148;
constexpr int SMEM_LIMIT = 232448 - 4096;   // 227 KB, 4 KB of it for static arrays

// Dynamic shared memory above 48 KB has to be allowed once per kernel and device.
template <typename Kernel>
cudaError_t allow_smem(Kernel kernel, std::atomic<unsigned long long>& devices, int bytes = SMEM_LIMIT) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const unsigned long long bit = 1ull << (dev & 63);
  if (devices.load(std::memory_order_acquire) & bit) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) devices.fetch_or(bit, std::memory_order_release);
  return e;
}

// Ring stages of `stage` bytes in `budget` bytes, the sums of `red` bytes in the same memory, and the whole of the dynamic shared memory.
int ring_stages(int budget, int stage, size_t red, size_t& smem) {
  int stages = (budget - 1024 - 256) / stage;
  if (stages > 12) stages = 12;
  if (stages < 2) stages = 2;
  size_t ring = (size_t)stages * stage;
  if (ring < red) ring = red;
  smem = 1024 + ring + (2 * stages + 1) * 8 + 16;
  return stages;
}

struct Call {
  const void *x, *w;
  long long ldx, ldw;
  const void *a, *b;
  const float* scale;
  const int* ranks;
  const int* index;
  PrismAdapterTerms terms;
  const void* bias;
  void* out;
  long long ldo;
  void* h;
  int T, M, K, act, tile_rows;
  int pair_tiles;        // tiles of the projection on pairs of SMs (0: another kernel runs it)
  cudaStream_t stream;
  bool pdl;
};

constexpr int HALF_SM = 111 * 1024;   // two such blocks share an SM: the projection streams weights beside the low-rank rows

// The largest cluster of 8, 4 or 2 blocks along z, at most `most`, of which n fit the device at once; 1 if none does.  More clusters than fit
// take a second round: 16 clusters of 8 blocks with an SM each took 22 us, 13 of them 11.6.  The count is asked for with an empty kernel: for
// kernels that allocate tensor memory the runtime counts one block per SM, but two run there where shared memory and columns allow it (256
// blocks of the projection 12288 -> 4096 38 us, 128 of them 48).
__global__ void __launch_bounds__(TC_THREADS) placeholder_kernel() {}
struct ClusterTable {
  std::atomic<int> known[16][4];   // per device: clusters that fit with one amount of shared memory, plus one
};
int cluster_size(ClusterTable& table, long long n, int most, size_t smem) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 1;
  for (int k = 3; k > 0; --k) {
    const int cs = 1 << k;
    if (cs > most) continue;
    std::atomic<int>* const slot = dev < 16 ? &table.known[dev][k] : nullptr;
    int fit = slot ? slot->load(std::memory_order_relaxed) - 1 : -1;
    if (fit < 0) {
      static std::atomic<unsigned long long> devices{0};
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3(1, 1, cs);
      cfg.blockDim = dim3(TC_THREADS);
      cfg.dynamicSmemBytes = smem;
      cudaLaunchAttribute attr[1];
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim.x = attr[0].val.clusterDim.y = 1;
      attr[0].val.clusterDim.z = cs;
      cfg.attrs = attr;
      cfg.numAttrs = 1;
      if (allow_smem(placeholder_kernel, devices) != cudaSuccess || cudaOccupancyMaxActiveClusters(&fit, placeholder_kernel, &cfg) != cudaSuccess) {
        (void)cudaGetLastError();
        fit = 0;
      }
      if (slot) slot->store(fit + 1, std::memory_order_relaxed);
    }
    if (n <= fit) return cs;
  }
  return 1;
}

// The longest run of panels that leaves at most `unused` of a pass empty.  A copy per panel kept a prompt's issuing thread busy for longer than
// the copies took (13 of them a k-block, 8192 tokens: 48 us; in runs of 6 panels 38).
int panel_run(int all_panels, int pass, int unused) {
  for (int run = all_panels < pass ? all_panels : pass; run > 1; --run)
    if (all_panels % run == 0 && pass % run <= unused) return run;
  return 1;
}

LowArgs low_args(const Call& c, int pass, int unused) {
  return LowArgs{c.terms.lists, c.terms.counts, c.index, c.scale, c.ranks, (bf16*)c.h, c.T, (c.K + 63) / 64, c.terms.capacity, c.terms.panels,
                 c.terms.panels * c.terms.sec.n, c.tile_rows, 0, panel_run(c.terms.panels * c.terms.sec.n, pass, unused)};
}

template <int BN, int G>
int launch_low(const Call& c) {
  static std::atomic<unsigned long long> devices{0};
  static ClusterTable table;
  cudaError_t e = allow_smem(adapter_low_kernel<BN, G>, devices);
  if (e != cudaSuccess) return (int)e;
  LowArgs a = low_args(c, G * 8, 0);
  const int pass = G * 8 / a.run * a.run, most = (a.capacity * a.all_panels + pass - 1) / pass;   // a step may bring as many adapters as tokens
  size_t smem;
  a.stages = ring_stages(G == 1 ? HALF_SM : SMEM_LIMIT, G * W_BYTES + BN * 128, (size_t)BN * (G * 128 + 4) * 4, smem);
  const int cs = most > SMS ? 1 : cluster_size(table, most, a.kb < SMS / most ? a.kb : SMS / most, smem);
  const int gx = SMS / cs < most ? SMS / cs : most;
  CUtensorMap ta, tx;
  int rc = prism_get_tensor_map(c.a, (unsigned long long)c.terms.slots * a.all_panels * 16, (unsigned long long)c.K, (unsigned long long)c.K, 16 * a.run, &ta);
  if (!rc) rc = prism_get_tensor_map(c.x, (unsigned long long)c.T, (unsigned long long)c.K, (unsigned long long)c.ldx, BN, &tx);
  if (rc) return rc;
  return (int)prism_launch_clusters(adapter_low_kernel<BN, G>, dim3(gx, 1, cs), dim3(TC_THREADS), smem, c.stream, c.pdl, cs, ta, tx, a);
}

int launch_low_prompt(const Call& c) {
  static std::atomic<unsigned long long> devices{0};
  static ClusterTable table;
  const size_t smem = 1024 + LOW_RING + (2 * LOW_STAGES + 1) * 8 + 16;
  cudaError_t e = allow_smem(adapter_low_prompt_kernel, devices, (int)smem);
  if (e != cudaSuccess) return (int)e;
  LowArgs a = low_args(c, LOW_PASS, LOW_PASS / 4);
  const int tiles = (c.T + 127) / 128;
  static_assert(LOW_PASS * 128 * LOW_PITCH * 4 <= LOW_RING, "the sums fit the ring");
  // The projection's pairs of SMs that walk one tile more than the others are its first blocks.  Where there are SMs for them beside these
  // blocks they start at once, and the others have as much time for the low-rank rows as a tile takes (8192 tokens, 4096 -> 6144 qkv: 64
  // blocks, 300 us; 128 blocks, whose rows take half the time, 306).  Where most pairs walk one tile more the rows come first, as fast as may be.
  const int more = c.pair_tiles % (SMS / 2), beside = SMS - 2 * (more ? more : SMS / 2);
  const int room = tiles <= beside ? beside : SMS;
  const int cs = tiles > room ? 1 : cluster_size(table, tiles, a.kb < room / tiles ? a.kb : room / tiles, smem);
  CUtensorMap ta, tx;
  int rc = prism_get_tensor_map(c.a, (unsigned long long)c.terms.slots * a.all_panels * 16, (unsigned long long)c.K, (unsigned long long)c.K, 16 * a.run, &ta);
  if (!rc) rc = prism_get_tensor_map(c.x, (unsigned long long)c.T, (unsigned long long)c.K, (unsigned long long)c.ldx, 128, &tx);
  if (rc) return rc;
  const int pass = LOW_PASS / a.run * a.run, passes = (a.capacity * a.all_panels + pass - 1) / pass, places = SMS / (tiles * cs);
  const int gx = places < 1 ? 1 : places < passes ? places : passes;
  return (int)prism_launch_clusters(adapter_low_prompt_kernel, dim3(gx, tiles, cs), dim3(TC_THREADS), smem, c.stream, c.pdl, cs, ta, tx, a);
}

template <int BN, bool DUAL>
int launch_tiles(const Call& c) {
  static std::atomic<unsigned long long> devices{0};
  static ClusterTable table, deep_table;
  cudaError_t e = allow_smem(adapter_gemm_kernel<BN, DUAL>, devices);
  if (e != cudaSuccess) return (int)e;
  constexpr int FEATURES = DUAL ? 64 : 128;
  const PrismAdapterTerms& t = c.terms;
  const int all = t.panels * t.sec.n, token_tiles = (c.T + BN - 1) / BN;
  TileArgs a = {};
  a.lists = t.lists;
  a.counts = t.counts;
  a.bias = (const bf16*)c.bias;
  a.out = (bf16*)c.out;
  a.ldo = c.ldo;
  a.T = c.T;
  a.M = c.M;
  a.kb = (c.K + 63) / 64;
  a.capacity = t.capacity;
  a.panels = t.panels;
  a.all_panels = all;
  a.tile_rows = c.tile_rows;
  a.act = c.act;
  a.b_groups = t.b_rows / 8;
  a.no_group = t.slots * t.panels * a.b_groups;
  a.sections = t.sec.n;
  a.vec = (reinterpret_cast<uintptr_t>(c.out) & 7) == 0 && c.ldo % 4 == 0;
  int m_tiles = 0;
  for (int s = 0; s < t.sec.n; ++s) {
    a.start[s] = s == 0 ? 0 : t.sec.end[s - 1];
    a.end[s] = t.sec.end[s];
    a.b_start[s] = s == 0 ? 0 : a.b_start[s - 1] + (a.end[s - 1] - a.start[s - 1] + 7) / 8;
    a.first_tile[s] = m_tiles;
    m_tiles += (a.end[s] - a.start[s] + FEATURES - 1) / FEATURES;
    if (a.start[s] % 4) a.vec = 0;
  }
  if (DUAL) m_tiles = (c.M / 2 + FEATURES - 1) / FEATURES;
  const long long tiles = (long long)m_tiles * token_tiles;
  // Few tiles of few tokens: one block per SM with a ring as deep as fits (4096 -> 6144, 32 tokens: 96 blocks 17.7 us a call, 192 blocks of half
  // the depth 19.7).  Otherwise two per SM: their rings together are as deep, and one's epilogue hides behind the other (12288 -> 4096, 128
  // tokens: 256 blocks 76, 128 blocks with an SM each 82; 4096 -> 2 x 12288, 32 tokens: 46 and 57).
  const bool deep = BN <= 64 && tiles <= SMS / 2;
  size_t smem;
  a.stages = ring_stages(deep ? SMEM_LIMIT : HALF_SM, stage_bytes<BN>(), (size_t)BN * RED_PITCH * 4, smem);
  const int most = deep && SMS / tiles < a.kb ? (int)(SMS / tiles) : a.kb;
  const int cs = tiles > 2 * SMS ? 1 : cluster_size(deep ? deep_table : table, tiles, most, smem);
  CUtensorMap tw, tx, tb, th;
  int rc = prism_get_tensor_map(c.w, (unsigned long long)c.M, (unsigned long long)c.K, (unsigned long long)c.ldw, FEATURES, &tw);
  if (!rc) rc = prism_get_tensor_map(c.x, (unsigned long long)c.T, (unsigned long long)c.K, (unsigned long long)c.ldx, BN, &tx);
  if (!rc) rc = prism_get_panel_tensor_map(c.b, (unsigned long long)a.no_group, FEATURES / 8, &tb);
  if (!rc) rc = prism_get_panel_tensor_map(c.h, (unsigned long long)t.tiles * t.capacity * all * c.tile_rows / 8, BN / 8, &th);
  if (rc) return rc;
  return (int)prism_launch_clusters(adapter_gemm_kernel<BN, DUAL>, dim3(m_tiles, token_tiles, cs), dim3(TC_THREADS), smem, c.stream, true, cs, tw, tx, tb,
                                    th, a);
}

template <int BN>
int launch_decode(const Call& c) {
  // Many panels: 16 at a time read the tokens half as often and keep twice the bytes in flight (128 adapters of rank 64, 12288 features).
  const bool wide = c.terms.capacity * c.terms.panels * c.terms.sec.n > 8 * SMS / 4;
  const int rc = wide ? launch_low<BN, 2>(c) : launch_low<BN, 1>(c);
  if (rc) return rc;
  return c.act ? launch_tiles<BN, true>(c) : launch_tiles<BN, false>(c);
}

int launch_prompt(Call& c) {
  bool pair = prism_adapter_pair_fits(c.M, c.act != 0, c.terms, c.out, c.ldo, c.bias);
  int bn;
  c.pair_tiles = pair ? prism_adapter_pair_tiles(c.M, c.T, c.act != 0, c.terms, &bn) : 0;
  // A pair of SMs adds all panels of its token tile one after another (0.8 us for four, their copies' issue); the blocks of a decode form's cluster
  // share them out.  Up to 256 tokens that may have many adapters, where the pairs would have no second tile to hide that behind, run as two decode
  // tiles: 4096 -> 4096, 256 tokens, 256 / 16 adapters of rank 16: 66 / 28 us, on pairs 115 / 26; 160 tokens, 40 / 4 adapters: 27 / 21 and 43 / 23.
  // Other widths and gated units were not compared.  The host knows how many adapters there may be, not how many there are.
  if (pair && c.T <= PLAN_TILE && c.pair_tiles <= SMS / 2 && c.terms.capacity * c.terms.panels > 16) pair = false, c.pair_tiles = 0;
  const int rc = launch_low_prompt(c);
  if (rc) return rc;
  if (pair)
    return prism_adapter_pair(c.w, c.x, c.out, c.M, c.T, c.K, c.ldw, c.ldx, c.ldo, c.bias, c.act != 0, c.act, c.terms, c.stream, true);
  return c.act ? launch_tiles<128, true>(c) : launch_tiles<128, false>(c);
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

namespace {

template <int NF, int NT, bool DUAL, bool VEC>
int launch_f32_tiles(const TileF32Args& a, cudaStream_t stream) {
  static std::atomic<unsigned long long> devices{0};
  static ClusterTable table;
  constexpr int TN = F32_THREADS / (64 / NF) * NT;
  constexpr int KC = f32_chunk(NT);
  const size_t smem = (size_t)(2 * KC * (68 + TN + 4) + TN * 68) * sizeof(float);
  const cudaError_t e = allow_smem(adapter_gemm_f32_kernel<NF, NT, DUAL, VEC>, devices);
  if (e != cudaSuccess) return (int)e;
  const int f_tiles = DUAL ? (a.M / 2 + 31) / 32 : (a.M + 63) / 64, t_tiles = (a.T + TN - 1) / TN, most = a.K / F32_SUM;
  // At least 128 products a block.  What counts is the SM with the most blocks, each a share of K; one block alone, four warps, keeps an SM little
  // more than half as busy as three do (300 tokens, 2048 -> 4096, 192 tiles: 376 us, in clusters of two 196).
  const long long tiles = (long long)f_tiles * t_tiles;
  int cs = 1;
  double best = 0.0;
  for (int n = 1; n <= 8 && n <= (most < 1 ? 1 : most); n *= 2) {
    const long long blocks = (tiles * n + SMS - 1) / SMS;
    if (n > 1 && (blocks > 3 || cluster_size(table, tiles, n, 64 * 1024) != n)) break;
    const double cost = (double)blocks / n * (blocks == 1 ? 1.7 : blocks == 2 ? 1.2 : 1.0);
    if (n == 1 || cost <= best) cs = n, best = cost;
  }
  return (int)prism_launch_clusters(adapter_gemm_f32_kernel<NF, NT, DUAL, VEC>, dim3(f_tiles, t_tiles, cs), dim3(F32_THREADS), smem, stream, true, cs, a);
}

template <int NF, int NT>
int launch_f32(const TileF32Args& a, bool vec, cudaStream_t on) {
  if (vec) return a.act ? launch_f32_tiles<NF, NT, true, true>(a, on) : launch_f32_tiles<NF, NT, false, true>(a, on);
  return a.act ? launch_f32_tiles<NF, NT, true, false>(a, on) : launch_f32_tiles<NF, NT, false, false>(a, on);
}

}  // namespace

// The same in 32 bits; b: [slots][panels][rows][16], h: T x low floats of workspace.
PRISM_API int prism_adapter_linear_f32(const void* x, const void* w, const void* a, const void* b, const void* scale, const void* ranks, const void* adapter,
                                       const void* bias, void* out, void* h, int T, int M, int K, int slots, int panels, int sections, const void* ends,
                                       int act, long long ldx, long long ldw, long long ldo, void* stream, int pdl) {
  if (T < 1 || T > MAX_TOKENS || M < 1 || K < 1 || slots < 1 || panels < 1 || sections < 1 || sections > MAX_SECTIONS) return -1;
  if (act && (M % 2 || sections != 2 || bias != nullptr)) return -2;
  const bool vec = (((uintptr_t)x | (uintptr_t)w | (uintptr_t)a) & 15) == 0 && K % 4 == 0 && ldx % 4 == 0 && ldw % 4 == 0;
  const int low = sections * panels * 16;
  LowF32Args l{(const float*)x, (const float*)a, (const float*)scale, (const int*)ranks, (const int*)adapter, (float*)h, K, low, slots, panels * 16, ldx};
  // few tokens: a block per 16 rows
  const cudaError_t e = prism_launch(vec ? adapter_low_f32_kernel<true> : adapter_low_f32_kernel<false>, dim3(T, T < 148 ? (low + 15) / 16 : 1), dim3(256), 0, (cudaStream_t)stream, pdl != 0, l);
  if (e != cudaSuccess) return (int)e;
  TileF32Args t{(const float*)x, (const float*)w, (const float*)b, (const float*)h, (const float*)bias, (const int*)adapter, (float*)out,
                T, M, K, low, panels, slots, 0, act, ldx, ldw, ldo, sections, {}, {}};
  for (int s = 0; s < sections; ++s) {
    const int start = s ? t.end[s - 1] : 0;
    t.end[s] = ((const int*)ends)[s];
    t.shift[s] = t.b_rows - start;
    t.b_rows += (t.end[s] - start + 7) / 8 * 8;
  }
  cudaStream_t on = (cudaStream_t)stream;
  if (T <= 16) return launch_f32<4, 2>(t, vec, on);
  if (T <= 64) return launch_f32<4, 8>(t, vec, on);
  return launch_f32<8, 8>(t, vec, on);
}

// bf16 projection (act 0) or gated unit (PRISM_GLU_*) with the adapters of a plan.  lists, counts: of the call's tiles of 256 tokens;
// b: [slots][panels] panels; ranks: [slots][sections]; h: tiles x capacity x all panels x tile_rows x 16 bf16 of workspace, tile_rows 16, 32, 64, 128 (as many as the tokens need) or 256.
PRISM_API int prism_adapter_linear(const void* x, const void* w, const void* a, const void* b, const void* scale, const void* ranks, const void* index,
                                   const void* lists, const void* counts, const void* bias, void* out, void* h, int T, int M, int K, int slots,
                                   int panels, int sections, const void* ends, int capacity, int tile_rows, int act, long long ldx, long long ldw,
                                   long long ldo, void* stream, int pdl) {
  if (T < 1 || T > MAX_TOKENS || M < 1 || K < 1 || K % 8 || slots < 1 || panels < 1 || sections < 1 || sections > MAX_SECTIONS || capacity < 1 || capacity > PLAN_TILE) return -1;
  if (act && (M % 2 || sections != 2 || bias != nullptr)) return -2;
  const int bn = T <= 16 ? 16 : T <= 32 ? 32 : T <= 64 ? 64 : 128;
  if (tile_rows != (T <= 128 ? bn : PLAN_TILE)) return -3;
  Call c = {};
  c.x = x;
  c.w = w;
  c.ldx = ldx;
  c.ldw = ldw;
  c.a = a;
  c.b = b;
  c.scale = (const float*)scale;
  c.ranks = (const int*)ranks;
  c.index = (const int*)index;
  c.terms.h = h;
  c.terms.b = b;
  c.terms.lists = (const int*)lists;
  c.terms.counts = (const int*)counts;
  c.terms.tiles = (T + PLAN_TILE - 1) / PLAN_TILE;
  c.terms.capacity = capacity;
  c.terms.panels = panels;
  c.terms.slots = slots;
  c.terms.sec.n = sections;
  for (int s = 0; s < sections; ++s) {
    c.terms.sec.end[s] = ((const int*)ends)[s];
    const int width = c.terms.sec.end[s] - (s ? c.terms.sec.end[s - 1] : 0);
    if (width < 1) return -4;
    c.terms.b_rows += (width + 7) / 8 * 8;
  }
  if (c.terms.sec.end[sections - 1] != M) return -4;
  if ((long long)slots * panels * c.terms.b_rows >= 0x7fffffffll || (long long)c.terms.tiles * capacity * panels * sections * tile_rows >= 0x7fffffffll) return -5;
  c.bias = bias;
  c.out = out;
  c.ldo = ldo;
  c.h = h;
  c.T = T;
  c.M = M;
  c.K = K;
  c.act = act;
  c.tile_rows = tile_rows;
  c.stream = (cudaStream_t)stream;
  c.pdl = pdl != 0;
  if (T > 128) return launch_prompt(c);
  switch (bn) {
    case 16: return launch_decode<16>(c);
    case 32: return launch_decode<32>(c);
    case 64: return launch_decode<64>(c);
    default: return launch_decode<128>(c);
  }
}
