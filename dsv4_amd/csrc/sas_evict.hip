// Eviction of cache rows by their weight on MI355X (gfx950): of each sequence with more
// than `budget` rows stay its first ones, its last ones and the heaviest of the others
// (of equal ones those at the lowest positions), moved together in their order.
//
//  evict_select_kernel  one workgroup a sequence finds the weight that divides the
//     candidates by a radix search over order-preserving 64-bit keys, 11 bits a pass
//     (counts in LDS; a pass ends the search once it takes a whole bin), lists the rows
//     that stay, and closes up their weights;
//  evict_move_kernel    a workgroup owns one slice of the rows' bytes of one sequence
//     and walks the list: since row i comes from a row at or behind i, the rows of a
//     chunk are loaded before any of them is written, and later chunks read only rows
//     behind them. Rows that stay where they are are not touched.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>
#include <cstdint>

#include "sas_kern.h"

namespace sas {
namespace {

struct EvictParams {
  uint8_t* cache;
  double* weights;
  const int32_t* bt;
  const int32_t* act_kv;
  int32_t* act_kv_out;
  int32_t* kept;
  int B, bt_stride, bs, nblocks, weight_rows, budget, first, recent;
  int row_bytes;
};

constexpr int kSelThreads = 1024, kSelWaves = kSelThreads / 64;
constexpr int kBins = 2048;

// Keys in the weights' order: NaN below everything, -0 = 0.
__device__ __forceinline__ uint64_t key_of(double w) {
  if (w != w) return 0;
  const uint64_t u = __builtin_bit_cast(uint64_t, w + 0.);
  return u >> 63 ? ~u : u | 1ull << 63;
}

__global__ void __launch_bounds__(kSelThreads) evict_select_kernel(const EvictParams p) {
  __shared__ int hist[kBins];
  __shared__ int wsum[kSelWaves], wtie[kSelWaves];
  __shared__ int found[3];   // bin, candidates above it, candidates in it
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int b = blockIdx.x;
  const int n = max(p.act_kv[b], 0);
  int32_t* kept = p.kept + (size_t)b * p.budget;
  if (n <= p.budget) {
    for (int i = tid; i < p.budget; i += kSelThreads) kept[i] = i < n ? i : -1;
    __syncthreads();   // act_kv_out may be act_kv
    if (tid == 0) p.act_kv_out[b] = n;
    return;
  }
  double* w = p.weights + (size_t)b * p.weight_rows;
  // candidates [lo, hi), of which `need` stay; rows without a weight count as 0
  const int lo = p.first, hi = n - p.recent;
  int need = p.budget - p.first - p.recent;
  auto key_at = [&](int j) { return key_of(j < p.weight_rows ? w[j] : 0.); };

  // the keys that stay: those above `edge`, and the first `need` of those equal to it
  uint64_t edge = ~0ull, mask = 0;   // bits of edge found so far
  bool whole = need == 0;            // edge: nothing equals it (a key is at most that of +inf)
  if (need == hi - lo) { edge = 0; whole = true; }   // (n > budget: never)
  uint64_t prefix = 0;
  for (int shift = 53; !whole && shift > -11; shift -= 11) {
    const int sh = max(shift, 0), bits = shift < 0 ? 11 + shift : 11;
    for (int i = tid; i < kBins; i += kSelThreads) hist[i] = 0;
    __syncthreads();
    for (int j = lo + tid; j < hi; j += kSelThreads) {
      const uint64_t k = key_at(j);
      if ((k & mask) == prefix) atomicAdd(&hist[(int)(k >> sh) & ((1 << bits) - 1)], 1);
    }
    __syncthreads();
    // bins from the top: thread i holds bins 2047 - 2 i and 2046 - 2 i
    const int h0 = hist[kBins - 1 - 2 * tid], h1 = hist[kBins - 2 - 2 * tid];
    int x = h0 + h1;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) { const int v = __shfl_up(x, d); x += lane >= d ? v : 0; }
    if (lane == 63) wsum[wave] = x;
    __syncthreads();
    int above = x - h0 - h1;
    for (int i = 0; i < wave; ++i) above += wsum[i];
    if (above < need && above + h0 + h1 >= need) {   // one thread
      const bool second = above + h0 < need;
      found[0] = kBins - 1 - 2 * tid - second;
      found[1] = above + (second ? h0 : 0);
      found[2] = second ? h1 : h0;
    }
    __syncthreads();
    prefix |= (uint64_t)found[0] << sh;
    mask |= ((1ull << bits) - 1ull) << sh;
    need -= found[1];
    if (need == found[2]) {   // the whole bin stays: every key from its lowest on
      edge = prefix - 1;      // (prefix 0: the search would have taken every candidate)
      whole = true;
    }
  }
  if (!whole) edge = prefix;   // all 64 bits: `need` of its equals stay
  else need = 0;

  // list: each wave takes a run of rows; its place follows from the runs before it
  const int run = ((n + kSelWaves - 1) / kSelWaves + 63) & ~63;
  const int r0 = min(wave * run, n), r1 = min(r0 + run, n);
  int nk = 0, nt = 0;
  for (int j0 = r0; j0 < r1; j0 += 64) {
    const int j = j0 + lane;
    const bool cand = j >= lo && j < hi;
    const uint64_t k = cand ? key_at(j) : 0;
    nk += __popcll(__ballot(j < r1 && (!cand || k > edge)));
    nt += __popcll(__ballot(cand && j < r1 && k == edge));
  }
  if (lane == 0) { wsum[wave] = nk; wtie[wave] = nt; }
  __syncthreads();
  int pk = 0, pt = 0;
  for (int i = 0; i < wave; ++i) { pk += wsum[i]; pt += wtie[i]; }
  for (int j0 = r0; j0 < r1; j0 += 64) {
    const int j = j0 + lane;
    const bool cand = j >= lo && j < hi;
    const uint64_t k = cand ? key_at(j) : 0;
    const uint64_t mk = __ballot(j < r1 && (!cand || k > edge)), mt = __ballot(cand && j < r1 && k == edge);
    const uint64_t below = (1ull << lane) - 1ull;
    const int tie = pt + __popcll(mt & below), at = pk + __popcll(mk & below) + min(tie, need);
    if ((mk >> lane & 1) || ((mt >> lane & 1) && tie < need)) kept[at] = j;
    pk += __popcll(mk);
    pt += __popcll(mt);
  }
  __syncthreads();
  // the weights close up as the rows do; those of the rows that are left behind are 0
  for (int i0 = 0; i0 < p.budget; i0 += kSelThreads) {
    const int i = i0 + tid;
    const int j = i < p.budget ? kept[i] : 0;
    const double v = i < p.budget && j < p.weight_rows ? w[j] : 0.;
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();   // the chunk's weights are read; later ones lie behind it
    if (i < p.budget && i < p.weight_rows) w[i] = v;
  }
  for (int i = p.budget + tid; i < min(n, p.weight_rows); i += kSelThreads) w[i] = 0.;
  if (tid == 0) p.act_kv_out[b] = p.budget;
}

// SB bytes of every row; U rows a thread in flight.
template <int SB, int U>
__global__ void __launch_bounds__(256) evict_move_kernel(const EvictParams p) {
  constexpr int LPR = SB / 16, RPP = 256 / LPR, CHUNK = RPP * U;
  const int tid = threadIdx.x, b = blockIdx.y;
  const int m = p.budget;
  const int32_t* kept = p.kept + (size_t)b * m;
  if (kept[m - 1] <= m - 1) return;   // nothing moves (fewer rows than the budget: -1)
  const int32_t* bt = p.bt + (size_t)b * p.bt_stride;
  const int off = (int)blockIdx.x * SB + (tid % LPR) * 16;
  const bool in = off < p.row_bytes;
  auto addr = [&](int j) -> uint8_t* {
    const int blk = j / p.bs;
    if (blk >= p.bt_stride) return nullptr;
    const int ph = bt[blk];
    if (ph < 0 || ph >= p.nblocks) return nullptr;
    return p.cache + ((size_t)ph * p.bs + (j - blk * p.bs)) * p.row_bytes + off;
  };
  for (int i0 = 0; i0 < m; i0 += CHUNK) {
    uint4 v[U];
    uint8_t* dst[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * RPP + tid / LPR;
      dst[u] = nullptr;
      if (i < m && in) {
        const int j = kept[i];
        if (j > i) {
          const uint8_t* src = addr(j);
          if (src) {
            dst[u] = addr(i);
            v[u] = *reinterpret_cast<const uint4*>(src);
          }
        }
      }
    }
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();   // the chunk's rows are read
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (dst[u]) *reinterpret_cast<uint4*>(dst[u]) = v[u];
    // the next chunk reads rows behind this one's: no barrier between
  }
}

int evict_impl(const SasCacheEvictArgs* a, hipStream_t st) {
  if (a->B < 0 || a->B > 65535) return set_error(SAS_EINVAL, "evict: B must be 0..65535 (got %lld)", (long long)a->B);
  if (a->budget < 1 || a->budget > INT_MAX) return set_error(SAS_EINVAL, "evict: budget must be at least 1 (got %lld)", (long long)a->budget);
  if (a->keep_first < 0 || a->keep_recent < 0 || a->keep_first > a->budget || a->keep_recent > a->budget - a->keep_first)
    return set_error(SAS_EINVAL, "evict: keep_first and keep_recent must not be negative and fit the budget (%lld + %lld, %lld)",
                     (long long)a->keep_first, (long long)a->keep_recent, (long long)a->budget);
  if (a->row_bytes < 16 || a->row_bytes % 16 || a->row_bytes > 1 << 20)
    return set_error(SAS_EINVAL, "evict: rows must be a multiple of 16 bytes, at most 1 MiB (got %lld)", (long long)a->row_bytes);
  if (a->weight_rows < 0 || a->weight_rows > INT_MAX) return set_error(SAS_EINVAL, "evict: weight_rows out of range");
  if (a->bt_stride < 1 || a->bt_stride > INT_MAX || a->block_size < 1 || a->num_blocks < 1 ||
      (double)a->num_blocks * a->block_size > 2147483000.0)
    return set_error(SAS_EINVAL, "evict: bad cache geometry");
  if (a->B == 0) return SAS_OK;
  if (!a->cache || !a->block_table || !a->act_kv || !a->act_kv_out || !a->kept || (a->weight_rows > 0 && !a->weights))
    return set_error(SAS_EINVAL, "evict: null device pointer");
  if (reinterpret_cast<uintptr_t>(a->cache) & 15) return set_error(SAS_EINVAL, "evict: cache must be 16-byte aligned");
  if (reinterpret_cast<uintptr_t>(a->weights) & 7) return set_error(SAS_EINVAL, "evict: weights must be 8-byte aligned");
  EvictParams p{};
  p.cache = (uint8_t*)a->cache;
  p.weights = a->weights;
  p.bt = a->block_table;
  p.act_kv = a->act_kv;
  p.act_kv_out = a->act_kv_out;
  p.kept = a->kept;
  p.B = (int)a->B; p.bt_stride = (int)a->bt_stride; p.bs = (int)a->block_size; p.nblocks = (int)a->num_blocks;
  p.weight_rows = (int)a->weight_rows; p.budget = (int)a->budget; p.first = (int)a->keep_first; p.recent = (int)a->keep_recent;
  p.row_bytes = (int)a->row_bytes;
  hipLaunchKernelGGL(evict_select_kernel, dim3((unsigned)p.B), dim3(kSelThreads), 0, st, p);
  constexpr int SB = 64, U = 4;
  const dim3 grid((unsigned)((p.row_bytes + SB - 1) / SB), (unsigned)p.B);
  hipLaunchKernelGGL((evict_move_kernel<SB, U>), grid, dim3(256), 0, st, p);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return set_error(SAS_ELAUNCH, "evict launch: %s", hipGetErrorString(e));
  return SAS_OK;
}

}  // namespace
}  // namespace sas

extern "C" int sas_cache_evict_v1(const SasCacheEvictArgs* a, void* stream) {
  sas::clear_error();
  if (!a) return sas::set_error(SAS_EINVAL, "evict: null args");
  return sas::evict_impl(a, (hipStream_t)stream);
}
