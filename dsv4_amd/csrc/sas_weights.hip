// Attention weight of cache rows on MI355X (gfx950): for every row j of a sequence
//   w[j] += mean over heads h of sum over tokens t of exp(scale q_th . k_j - lse_th)
// over the forward's keys, what a program that keeps its caches bounded orders rows by.
//
// The weights are fp64 and every addition is a multiple of 2^-36, so sums below 2^17
// are exact: whatever order the adds of workgroups, tokens and calls come in, the bits
// are the same. Products, exponentials and a workgroup's own sums are fp32.
//
// A workgroup (4 waves) owns 64 RT slots of one token, slots being its first rows, its
// window and its compressed rows without gaps. A wave holds the K fragments of its 16 RT
// rows in registers, loaded straight from the cache (16 bytes a lane: the MFMA's B
// operand), and the queries, 16 heads at a time, reach LDS by DMA, four tiles deep, one
// barrier a tile: S[head][row] = Q . K^T (16x16x32 MFMA), P = 2^(S - lse), summed over
// the lane's four heads, over tiles, and last over the four lane groups.

#include "sas_kern.h"

namespace sas {
namespace {

struct WeightParams {
  FwdParams f;
  double* ori_w;    // [B, ori_rows], or null: raw rows are left out
  double* cmp_w;    // [B, cmp_rows], or null
  double units;     // 2^36 / H: grid units of one head's weight
  int ori_rows, cmp_rows;
  int ori_cap, cmp_cap;   // rows that a block table can address
  int chunks;       // workgroups a token
  int spread;       // 1: a token's workgroups lie on one XCD (else on all)
};

constexpr double kGrid = 68719476736.;   // 2^36

// The largest b with q_prefix[b] <= t, as resolve() finds it.
struct Where { int b, spos, aq, akv; };
__device__ __forceinline__ Where batch_of(const FwdParams& p, int t, int lane) {
  const bool cu = p.act_q == nullptr;
  Where w{0, 0, 0, 0};
  int qpb = 0;
  for (int c = 0; c < p.B; c += 64) {
    const int i = c + lane;
    int qpi = INT_MAX, aqi = 0, akvi = 0;
    if (i < p.B) { qpi = p.q_prefix[i]; aqi = cu ? p.q_prefix[i + 1] : p.act_q[i]; akvi = p.act_kv[i]; }
    const uint64_t m = __ballot(qpi <= t);
    const int n = __popcll(m);
    if (n) { w.b = c + n - 1; qpb = __shfl(qpi, n - 1); w.aq = __shfl(aqi, n - 1); w.akv = __shfl(akvi, n - 1); }
    if (n < 64) break;
  }
  if (cu) w.aq -= qpb;
  w.spos = t - qpb;
  w.b = __builtin_amdgcn_readfirstlane(w.b);
  w.spos = __builtin_amdgcn_readfirstlane(w.spos);
  w.aq = __builtin_amdgcn_readfirstlane(w.aq);
  w.akv = __builtin_amdgcn_readfirstlane(w.akv);
  return w;
}

// Adds a row's weight, its heads' sum over their count, rounded to the grid.
__device__ __forceinline__ void add_weight(double* at, float sum, double units) {
  unsafeAtomicAdd(at, rint((double)sum * units) * (1. / kGrid));
}

template <int D, typename QT, bool F8, int RT>
__global__ void __launch_bounds__(256, 2) sas_weights_kernel(const WeightParams wp) {
  constexpr int CH = D / 8, KS = D / 32, SG = kSwzGroup<CH>;
  constexpr int NI = 16 * CH / 64, OPS = (NI + 3) / 4;   // DMA instructions a query tile, and a wave's most
  constexpr int NB = 4;                                  // query tiles in LDS
  constexpr int ROWS = 64 * RT;
  static_assert(NI * 64 == 16 * CH, "whole instructions");
  __shared__ __attribute__((aligned(1024))) uint4 lq[NB][16 * CH];
  __shared__ __attribute__((aligned(16))) float ll[NB][256];   // a tile's 16 lse (written 16 times over)

  const FwdParams& p = wp.f;
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int c16 = lane & 15, g = lane >> 4;
  int t, chunk;
  if (wp.spread) {
    const int nx = p.nxcd, x = (int)(blockIdx.x % (unsigned)nx), l = (int)(blockIdx.x / (unsigned)nx);
    t = (l / wp.chunks) * nx + x;
    chunk = l % wp.chunks;
  } else {
    t = (int)(blockIdx.x / (unsigned)wp.chunks);
    chunk = (int)(blockIdx.x % (unsigned)wp.chunks);
  }
  if (t >= p.T) return;
  const Where at = batch_of(p, t, lane);
  if (at.spos < 0 || at.spos >= at.aq) return;           // padded
  const int sg = at.akv - at.aq + at.spos;
  if (sg < 0) return;
  // the token's slots: [0, nf) first rows, [nf, nr) the window, [nr, ns) compressed rows
  int nf = 0, nr = 0, wlo = 0;
  if (wp.ori_w) {
    wlo = max(sg - p.win_left, 0);
    nf = min(min(p.first, wlo), wp.ori_cap);
    nr = nf + max(min(sg + 1, wp.ori_cap) - wlo, 0);
  }
  int thr = 0, ns = nr;
  if (wp.cmp_w) {
    thr = (sg + 1) / p.cmp_ratio;
    ns = nr + (p.scenario == SAS_SCFA ? p.K : min(min(thr, p.K), wp.cmp_cap));
  }
  const int s0 = chunk * ROWS + wave * 16 * RT;
  if (chunk * ROWS >= ns) return;                        // uniform

  // queries: tile i of the token's H / 16 goes to buffer i % NB
  const int ntile = p.H / 16;
  const uint8_t* qb = p.q + (size_t)t * p.H * D * 2;
  const float* lb = p.lse + (size_t)t * p.H;
  uint32_t qoff[OPS];
#pragma unroll
  for (int o = 0; o < OPS; ++o) {
    const int P = (o * 4 + wave) * 64 + lane, r = P / CH;
    qoff[o] = (uint32_t)(r * CH + ((P - r * CH) ^ swz<CH>(r))) * 16;
  }
  const bool wide = wave == 3 || (NI % 4 != 0 && wave < NI % 4);   // five instructions a tile, else four
  static_assert(NI / 4 == 4 && NI % 4 < 3 && NB == 4, "instructions a tile: four, the left-over ones, wave 3's lse");
  auto issue = [&](int i) {
    const uint32_t dst = lds_addr_of(lq[i % NB]);
#pragma unroll
    for (int o = 0; o < OPS; ++o)
      if (o * 4 + wave < NI)   // uniform
        dma16s(qoff[o], qb + (size_t)i * 16 * D * 2, __builtin_amdgcn_readfirstlane(dst + (o * 4 + wave) * 1024));
    if (wave == 3) dma16s((uint32_t)(lane & 3) * 16, lb + i * 16, __builtin_amdgcn_readfirstlane(lds_addr_of(ll[i % NB])));
  };
#pragma unroll
  for (int i = 0; i < NB - 1; ++i)
    if (i < ntile) issue(i);

  // rows: lane (g, c16) holds slot s0 + 16 rt + c16 (all four g), channels 32 ks + 8 g ..
  bool ok[RT];
  double* dest[RT];
  uint4 k[RT][KS];
  float sc[RT][F8 ? 4 : 1];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int s = s0 + 16 * rt + c16;
    const bool ori = s < nr;
    int pos = s < nf ? s : wlo + s - nf;
    ok[rt] = s < ns;
    if (!ori) {
      pos = s - nr;
      if (p.scenario == SAS_SCFA && ok[rt]) pos = p.cmp_idx[(size_t)t * p.K + pos];
      ok[rt] = ok[rt] && pos >= 0 && pos < thr;
    }
    const int bs = ori ? p.ori_bs : p.cmp_bs, blk = max(pos, 0) / bs;
    const int stride = ori ? p.ori_bt_stride : p.cmp_bt_stride;
    ok[rt] = ok[rt] && blk < stride && pos < (ori ? wp.ori_rows : wp.cmp_rows);
    const int32_t* bt = ori ? p.ori_bt : p.cmp_bt;
    const int phys = ok[rt] ? bt[(size_t)at.b * stride + blk] : -1;
    ok[rt] = ok[rt] && phys >= 0 && phys < (ori ? p.ori_nblocks : p.cmp_nblocks);
    constexpr int ROWB = F8 ? kRow656 : D * 2;
    // (a row that is not there: the query's bytes, masked out)
    const uint64_t row = ok[rt] ? reinterpret_cast<uint64_t>(ori ? p.ori_kv : p.cmp_kv) +
                                      (uint64_t)(uint32_t)(phys * bs + pos - blk * bs) * ROWB
                                : reinterpret_cast<uint64_t>(qb);
    dest[rt] = ok[rt] ? (ori ? wp.ori_w + (size_t)at.b * wp.ori_rows : wp.cmp_w + (size_t)at.b * wp.cmp_rows) + pos
                      : nullptr;
    if constexpr (F8) {
      // 16 latent values of a lane are its channels of two k-steps
      uint4 raw[8];
#pragma unroll
      for (int m = 0; m < 8; ++m) raw[m] = gld16(row + (4 * m + g) * 16);
#pragma unroll
      for (int m = 0; m < 2; ++m) k[rt][16 + m] = gld16(row + 528 + (4 * m + g) * 16);
#pragma unroll
      for (int m = 0; m < 4; ++m) sc[rt][m] = gldf(row + 512 + 4 * m);
#pragma unroll
      for (int m = 0; m < 8; ++m) {
        e4m3x4_to_bf16(raw[m].x, k[rt][2 * m].x, k[rt][2 * m].y);
        e4m3x4_to_bf16(raw[m].y, k[rt][2 * m].z, k[rt][2 * m].w);
        e4m3x4_to_bf16(raw[m].z, k[rt][2 * m + 1].x, k[rt][2 * m + 1].y);
        e4m3x4_to_bf16(raw[m].w, k[rt][2 * m + 1].z, k[rt][2 * m + 1].w);
      }
    } else {
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) k[rt][ks] = gld16(row + (4 * ks + g) * 16);
    }
  }

  float acc[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) acc[rt] = 0.f;
  const int qsw = swz<CH>(c16);
  // the K fragments and the first tiles' DMA: known to the compiler to be done, so none
  // of its waits falls into the loop
  __builtin_amdgcn_s_waitcnt(0);
  for (int i = 0; i < ntile; ++i) {
    // tile i is here once only the tiles behind it, at most NB - 2 of them, are under way
    if (i >= NB - 1) {
      const int m = min(NB - 2, ntile - 1 - i);
      if (wide) m == 2 ? wait_vm<10>() : m == 1 ? wait_vm<5>() : wait_vm<0>();
      else m == 2 ? wait_vm<8>() : m == 1 ? wait_vm<4>() : wait_vm<0>();
    }
    lds_barrier();   // every wave's part of tile i is here, and tile i - 1 is read
    if (i + NB - 1 < ntile) issue(i + NB - 1);
    const uint4* qt = lq[i % NB] + c16 * CH;
    f32x4 s[RT], part[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) s[rt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const int L = F8 && ks < 16 ? 8 * (ks >> 1) + 2 * g + (ks & 1) : 4 * ks + g;
      const uint4 a = qt[(L & -SG) | ((L & (SG - 1)) ^ qsw)];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        if (F8 && ks < 16) {
          part[rt] = mfma32k<QT>(a, k[rt][ks], ks % 4 == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : part[rt]);
          if (ks % 4 == 3) s[rt] += part[rt] * sc[rt][F8 ? ks / 4 : 0];
        } else {
          s[rt] = mfma32k<QT>(a, k[rt][ks], s[rt]);
        }
      }
    }
    // lane (g, c16): heads 4 g + j of the tile, row c16
    const f32x4 l2 = *reinterpret_cast<const f32x4*>(&ll[i % NB][4 * g]) * kLog2e;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[rt] += __builtin_amdgcn_exp2f(s[rt][j] * p.scale_log2 - l2[j]);
  }
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const float w = rows_sum(acc[rt]);
    if (g == 0 && ok[rt]) add_weight(dest[rt], w, wp.units);
  }
}

template <int D, typename QT, bool F8>
int launch_weights(const WeightParams& wp, long long blocks, hipStream_t st) {
  hipLaunchKernelGGL((sas_weights_kernel<D, QT, F8, 2>), dim3((unsigned)blocks), dim3(256), 0, st, wp);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return set_error(SAS_ELAUNCH, "row weights launch: %s", hipGetErrorString(e));
  return SAS_OK;
}

int weights_impl(const SasRowWeightsArgs* ra, hipStream_t st) {
  const SasFwdArgs* a = &ra->fwd;
  if (a->T < 0 || a->B < 1 || a->H < 16 || a->H % 16)
    return set_error(SAS_EINVAL, "row weights: bad T/B/H (H a multiple of 16)");
  if (a->T > INT_MAX || a->B > INT_MAX || a->H > INT_MAX) return set_error(SAS_EINVAL, "row weights: T, B or H beyond 2^31");
  if (a->D != 512 && a->D != 576) return set_error(SAS_EINVAL, "row weights: D must be 512 or 576 (got %lld)", (long long)a->D);
  if (a->scenario < SAS_SWA || a->scenario > SAS_SCFA) return set_error(SAS_EINVAL, "row weights: bad scenario");
  if (a->q_dtype != SAS_DT_BF16 && a->q_dtype != SAS_DT_FP16) return set_error(SAS_EINVAL, "row weights: q dtype");
  const bool fp8 = a->kv_dtype == SAS_DT_FP8_E4M3_ROW656;
  if (fp8 && (a->q_dtype != SAS_DT_BF16 || a->D != 576))
    return set_error(SAS_EINVAL, "row weights: fp8 cache rows need bf16 q and D=576");
  if (!fp8 && a->kv_dtype != a->q_dtype) return set_error(SAS_EINVAL, "row weights: kv dtype must match q dtype");
  if (a->win_left < 0) return set_error(SAS_EINVAL, "row weights: win_left out of range");
  if (ra->ori_first < 0 || ra->ori_first > INT_MAX)
    return set_error(SAS_EINVAL, "row weights: ori_first out of range (got %lld)", (long long)ra->ori_first);
  const bool cmp = ra->cmp_weights != nullptr;
  if (!ra->ori_weights && !cmp) return set_error(SAS_EINVAL, "row weights: neither raw nor compressed rows' weights asked for");
  if (cmp && a->scenario == SAS_SWA) return set_error(SAS_EINVAL, "row weights: compressed rows' weights without compressed rows");
  if (cmp && (a->cmp_ratio < 1 || a->K < 0 || a->K > INT_MAX)) return set_error(SAS_EINVAL, "row weights: bad cmp_ratio/K");
  if (ra->ori_rows < 0 || ra->cmp_rows < 0 || ra->ori_rows > INT_MAX || ra->cmp_rows > INT_MAX)
    return set_error(SAS_EINVAL, "row weights: ori_rows or cmp_rows out of range");
  if (a->T == 0) return SAS_OK;
  if (!a->q || !a->q_prefix || !a->act_kv || !a->lse) return set_error(SAS_EINVAL, "row weights: null device pointer");
  if ((reinterpret_cast<uintptr_t>(a->q) | reinterpret_cast<uintptr_t>(a->lse)) & 15)
    return set_error(SAS_EINVAL, "row weights: q and lse must be 16-byte aligned");
  if ((reinterpret_cast<uintptr_t>(ra->ori_weights) | reinterpret_cast<uintptr_t>(ra->cmp_weights)) & 7)
    return set_error(SAS_EINVAL, "row weights: weights must be 8-byte aligned");
  if (ra->ori_weights) {
    if (!a->ori_kv || !a->ori_block_table || (reinterpret_cast<uintptr_t>(a->ori_kv) & 15))
      return set_error(SAS_EINVAL, "row weights: ori_kv (16-byte aligned) and ori_block_table needed");
    if (a->ori_block_size < 1 || a->ori_bt_stride < 1 || a->ori_num_blocks < 1 ||
        (double)a->ori_num_blocks * a->ori_block_size > 2147483000.0)
      return set_error(SAS_EINVAL, "row weights: bad ori cache geometry");
  }
  if (cmp) {
    if (!a->cmp_kv || !a->cmp_block_table || (reinterpret_cast<uintptr_t>(a->cmp_kv) & 15))
      return set_error(SAS_EINVAL, "row weights: cmp_kv (16-byte aligned) and cmp_block_table needed");
    if (a->scenario == SAS_SCFA && a->K > 0 && !a->cmp_indices) return set_error(SAS_EINVAL, "row weights: SCFA needs cmp_indices");
    if (a->cmp_block_size < 1 || a->cmp_bt_stride < 1 || a->cmp_num_blocks < 1 ||
        (double)a->cmp_num_blocks * a->cmp_block_size > 2147483000.0)
      return set_error(SAS_EINVAL, "row weights: bad cmp cache geometry");
  }

  WeightParams wp{};
  FwdParams& fp = wp.f;
  fp.q = (const uint8_t*)a->q;
  fp.ori_kv = (const uint8_t*)a->ori_kv;
  fp.ori_bt = a->ori_block_table;
  fp.cmp_kv = (const uint8_t*)a->cmp_kv;
  fp.cmp_bt = a->cmp_block_table;
  fp.cmp_idx = a->cmp_indices;
  fp.q_prefix = a->q_prefix;
  fp.act_q = a->act_q;
  fp.act_kv = a->act_kv;
  fp.lse = a->lse;
  fp.T = (int)a->T; fp.B = (int)a->B; fp.H = (int)a->H;
  fp.ori_bs = (int)std::max<int64_t>(a->ori_block_size, 1);
  fp.ori_bt_stride = (int)a->ori_bt_stride; fp.ori_nblocks = (int)a->ori_num_blocks;
  fp.cmp_bs = (int)std::max<int64_t>(a->cmp_block_size, 1);
  fp.cmp_bt_stride = (int)a->cmp_bt_stride; fp.cmp_nblocks = (int)a->cmp_num_blocks;
  fp.K = (int)a->K; fp.scenario = a->scenario;
  fp.cmp_ratio = std::max(1, a->cmp_ratio); fp.win_left = a->win_left; fp.first = (int)ra->ori_first;
  fp.scale_log2 = a->softmax_scale * kLog2e;
  fp.nxcd = device_xcds();
  wp.units = kGrid / (double)a->H;
  wp.ori_w = ra->ori_weights;
  wp.cmp_w = ra->cmp_weights;
  wp.ori_rows = (int)ra->ori_rows;
  wp.cmp_rows = (int)ra->cmp_rows;
  // rows past a table's end are not there
  wp.ori_cap = ra->ori_weights ? (int)std::min<long long>(INT_MAX / 2, (long long)a->ori_bt_stride * a->ori_block_size) : 0;
  wp.cmp_cap = cmp ? (int)std::min<long long>(INT_MAX / 2, (long long)a->cmp_bt_stride * a->cmp_block_size) : 0;
  constexpr int ROWS = 128;
  const long long nori = std::min<long long>(wp.ori_cap, ra->ori_first + a->win_left + 1);
  const long long ncmp = !cmp ? 0 : a->scenario == SAS_SCFA ? a->K : std::min<long long>(wp.cmp_cap, a->K);
  const long long chunks = (nori + ncmp + ROWS - 1) / ROWS;
  if (chunks == 0) return SAS_OK;
  wp.spread = a->T >= 2 * fp.nxcd;
  const long long blocks = (wp.spread ? (a->T + fp.nxcd - 1) / fp.nxcd * fp.nxcd : a->T) * chunks;
  if (blocks > INT_MAX) return set_error(SAS_EINVAL, "row weights: %lld workgroups beyond one launch", blocks);
  wp.chunks = (int)chunks;
  if (fp8) return launch_weights<576, __bf16, true>(wp, blocks, st);
  if (a->q_dtype == SAS_DT_BF16)
    return a->D == 576 ? launch_weights<576, __bf16, false>(wp, blocks, st) : launch_weights<512, __bf16, false>(wp, blocks, st);
  return a->D == 576 ? launch_weights<576, _Float16, false>(wp, blocks, st) : launch_weights<512, _Float16, false>(wp, blocks, st);
}

}  // namespace
}  // namespace sas

extern "C" int sas_row_weights_v1(const SasRowWeightsArgs* a, void* stream) {
  sas::clear_error();
  if (!a) return sas::set_error(SAS_EINVAL, "row weights: null args");
  return sas::weights_impl(a, (hipStream_t)stream);
}
