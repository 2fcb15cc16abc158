// Attention weight of cache rows on MI355X (gfx950): for every row j of a sequence
//   w[j] += mean over heads h of sum over tokens t of exp(scale q_th . k_j - lse_th)
// over the forward's keys, what a program that keeps its caches bounded orders rows by.
//
// The weights are fp64 and every addition is a multiple of 2^-36, so sums below 2^17
// are exact: whatever order the adds of workgroups, tokens and calls come in, the bits
// are the same. Products, exponentials and a workgroup's own sums are fp32.
//
// Rows stay with a wave, as K fragments in registers loaded straight from the cache (16
// bytes a lane: the MFMA's B operand), and queries reach LDS by DMA, 16 heads of one token at
// a time, one barrier a tile: S[head][row] = Q . K^T (16x16x32 MFMA), P = 2^(S - lse), summed
// over the lane's four heads, over tiles, and last over the four lane groups. One kernel
// for the slots of single tokens, one for rows that several tokens attend.

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

// A row's K fragments: lane group g holds channels 32 ks + 8 g .. of k-step ks; of fp8 rows the
// latent values of two k-steps from one 16-byte load (the queries' fragments follow), and
// the row's scales.
template <int D, bool F8>
__device__ __forceinline__ void load_row(uint64_t row, int g, uint4 (&k)[D / 32], float (&sc)[F8 ? 4 : 1]) {
  if constexpr (F8) {
    uint4 raw[8];
#pragma unroll
    for (int m = 0; m < 8; ++m) raw[m] = gld16(row + (4 * m + g) * 16);
#pragma unroll
    for (int m = 0; m < 2; ++m) k[16 + m] = gld16(row + 528 + (4 * m + g) * 16);
#pragma unroll
    for (int m = 0; m < 4; ++m) sc[m] = gldf(row + 512 + 4 * m);
#pragma unroll
    for (int m = 0; m < 8; ++m) {
      e4m3x4_to_bf16(raw[m].x, k[2 * m].x, k[2 * m].y);
      e4m3x4_to_bf16(raw[m].y, k[2 * m].z, k[2 * m].w);
      e4m3x4_to_bf16(raw[m].z, k[2 * m + 1].x, k[2 * m + 1].y);
      e4m3x4_to_bf16(raw[m].w, k[2 * m + 1].z, k[2 * m + 1].w);
    }
  } else {
#pragma unroll
    for (int ks = 0; ks < D / 32; ++ks) k[ks] = gld16(row + (4 * ks + g) * 16);
  }
}

// The queries' way into LDS: tiles of 16 heads of one token, D channels each and their 16
// lse, by DMA of a workgroup's four waves.
template <int D>
struct Queries {
  static constexpr int CH = D / 8, SG = kSwzGroup<CH>;
  static constexpr int NI = 16 * CH / 64, OPS = (NI + 3) / 4;   // instructions a tile, and a wave's most
  static_assert(NI * 64 == 16 * CH && NI / 4 == 4 && NI % 4 < 3, "four instructions a wave; the left-over ones and the lse make five");
  struct Tile {
    uint4 q[16 * CH];      // chunk c of head r at c ^ swz(r), in its swizzle group
    float lse[256];        // 16 of them, 16 times over
  };
  const uint8_t* q;
  const float* lse;
  int wave, lane;
  uint32_t off[OPS];
  bool wide;               // five instructions a tile, else four
  __device__ __forceinline__ Queries(const FwdParams& p, size_t token, int wave_, int lane_)
      : q(p.q + token * p.H * D * 2), lse(p.lse + token * p.H), wave(wave_), lane(lane_),
        wide(wave_ == 3 || wave_ < NI % 4) {
#pragma unroll
    for (int o = 0; o < OPS; ++o) {
      const int P = (o * 4 + wave) * 64 + lane, r = P / CH;
      off[o] = (uint32_t)(r * CH + ((P - r * CH) ^ swz<CH>(r))) * 16;
    }
  }
  // tile i, counted from the first token's first
  __device__ __forceinline__ void issue(Tile& to, int i) const {
    const uint32_t dst = lds_addr_of(to.q);
#pragma unroll
    for (int o = 0; o < OPS; ++o)
      if (o * 4 + wave < NI)   // uniform
        dma16s(off[o], q + (size_t)i * 16 * D * 2, __builtin_amdgcn_readfirstlane(dst + (o * 4 + wave) * 1024));
    if (wave == 3) dma16s((uint32_t)(lane & 3) * 16, lse + (size_t)i * 16, __builtin_amdgcn_readfirstlane(lds_addr_of(to.lse)));
  }
  // all but the `n` newest tiles are here
  __device__ __forceinline__ void wait(int n) const {
    if (wide) n == 2 ? wait_vm<10>() : n == 1 ? wait_vm<5>() : wait_vm<0>();
    else n == 2 ? wait_vm<8>() : n == 1 ? wait_vm<4>() : wait_vm<0>();
  }
  // a tile's fragment of k-step ks for lane group g, head c16; of fp8 rows as load_row() has them
  template <bool F8>
  static __device__ __forceinline__ uint4 frag(const Tile& t, int ks, int g, int c16) {
    const int L = F8 && ks < 16 ? 8 * (ks >> 1) + 2 * g + (ks & 1) : 4 * ks + g;
    return t.q[c16 * CH + ((L & -SG) | ((L & (SG - 1)) ^ swz<CH>(c16)))];
  }
};

// S[head][row] of a tile against RT row tiles. PF fragments are read ahead; work(), VALU
// work of another tile, goes between the MFMAs.
template <int D, typename QT, bool F8, int RT, int PF, typename Work>
__device__ __forceinline__ void tile_scores(const typename Queries<D>::Tile& t, const uint4 (&k)[RT][D / 32],
                                            const float (&sc)[RT][F8 ? 4 : 1], int g, int c16, f32x4 (&s)[RT], Work&& work) {
  constexpr int KS = D / 32;
  f32x4 part[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) s[rt] = f32x4{0.f, 0.f, 0.f, 0.f};
  uint4 a[PF];
#pragma unroll
  for (int ks = 0; ks < PF; ++ks) a[ks] = Queries<D>::template frag<F8>(t, ks, g, c16);
  work();
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) {
    const uint4 q = a[ks % PF];
    if (ks + PF < KS) a[ks % PF] = Queries<D>::template frag<F8>(t, ks + PF, g, c16);
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      if (F8 && ks < 16) {
        // one scale's 128 channels at a time, unscaled e4m3 values (exact in bf16)
        part[rt] = mfma32k<QT>(q, k[rt][ks], ks % 4 == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : part[rt]);
        if (ks % 4 == 3) s[rt] += part[rt] * sc[rt][F8 ? ks / 4 : 0];
      } else {
        s[rt] = mfma32k<QT>(q, k[rt][ks], s[rt]);
      }
    }
  }
  if constexpr (!F8 && RT > 1) {
    __builtin_amdgcn_sched_group_barrier(0x100, PF + 1, 0);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      __builtin_amdgcn_sched_group_barrier(0x008, RT, 0);
      if (ks + PF < KS) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x002, RT, 0);
    }
  }
}

// The sum over the lane's four heads of 2^(scale S - lse).
__device__ __forceinline__ float shares(const f32x4& s, const f32x4& lse2, float scale_log2) {
  float x[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) x[j] = __builtin_amdgcn_exp2f(s[j] * scale_log2 - lse2[j]);
  return (x[0] + x[1]) + (x[2] + x[3]);
}

// ---------------------------------------------------------------------------
// slots of one token
// ---------------------------------------------------------------------------
//
// A workgroup owns 64 slots of one token, slots being its first rows, its window and its
// compressed rows without gaps, 16 to a wave. HBM-bound where the rows are many; short
// workgroups, four to a CU, keep the last round of a grid short (32 tokens of 64 heads over
// 2000 rows, 576 channels: 26.2 us a call with 128 slots, two to a CU, 23.7 with 64; one
// token 13.9 and 10.9).
template <int D, typename QT, bool F8>
__global__ void __launch_bounds__(256, 4) sas_weights_kernel(const WeightParams wp) {
  using Q = Queries<D>;
  constexpr int NB = 2, ROWS = 64;
  __shared__ __attribute__((aligned(1024))) typename Q::Tile tiles[NB];

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
  if (chunk * ROWS >= ns) return;                        // uniform

  const int ntile = p.H / 16;
  const Q queries(p, (size_t)t, wave, lane);
  queries.issue(tiles[0], 0);

  // lane (g, c16) holds slot 16 wave + c16 of the chunk (all four g)
  const int s = chunk * ROWS + wave * 16 + c16;
  const bool ori = s < nr;
  int pos = s < nf ? s : wlo + s - nf;
  bool ok = s < ns;
  if (!ori) {
    pos = s - nr;
    if (p.scenario == SAS_SCFA && ok) pos = p.cmp_idx[(size_t)t * p.K + pos];
    ok = ok && pos >= 0 && pos < thr;
  }
  const int bs = ori ? p.ori_bs : p.cmp_bs, blk = max(pos, 0) / bs;
  const int stride = ori ? p.ori_bt_stride : p.cmp_bt_stride;
  ok = ok && blk < stride && pos < (ori ? wp.ori_rows : wp.cmp_rows);
  const int32_t* bt = ori ? p.ori_bt : p.cmp_bt;
  const int phys = ok ? bt[(size_t)at.b * stride + blk] : -1;
  ok = ok && phys >= 0 && phys < (ori ? p.ori_nblocks : p.cmp_nblocks);
  constexpr int ROWB = F8 ? kRow656 : D * 2;
  // (a row that is not there: the query's bytes, masked out)
  const uint64_t row = ok ? reinterpret_cast<uint64_t>(ori ? p.ori_kv : p.cmp_kv) +
                                (uint64_t)(uint32_t)(phys * bs + pos - blk * bs) * ROWB
                          : reinterpret_cast<uint64_t>(queries.q);
  uint4 k[1][D / 32];
  float sc[1][F8 ? 4 : 1];
  load_row<D, F8>(row, g, k[0], sc[0]);

  float acc = 0.f;
  // the K fragments and the first tile's DMA: known to the compiler to be done, so none
  // of its waits falls into the loop
  __builtin_amdgcn_s_waitcnt(0);
  for (int i = 0; i < ntile; ++i) {
    if (i > 0) queries.wait(0);
    lds_barrier();   // every wave's part of tile i is here, and tile i - 1 is read
    if (i + 1 < ntile) queries.issue(tiles[(i + 1) % NB], i + 1);
    const typename Q::Tile& tile = tiles[i % NB];
    const f32x4 l2 = *reinterpret_cast<const f32x4*>(&tile.lse[4 * g]) * kLog2e;
    f32x4 x[1];
    tile_scores<D, QT, F8, 1, 4>(tile, k, sc, g, c16, x, [] {});
    acc += shares(x[0], l2, p.scale_log2);
  }
  const float w = rows_sum(acc);
  if (g == 0 && ok)
    add_weight((ori ? wp.ori_w + (size_t)at.b * wp.ori_rows : wp.cmp_w + (size_t)at.b * wp.cmp_rows) + pos, w, wp.units);
}

// ---------------------------------------------------------------------------
// rows of several tokens
// ---------------------------------------------------------------------------
//
// A prompt's end, a chunk, drafts: the rows are keys of many tokens, so a workgroup keeps
// 128 consecutive rows of a sequence (raw ones of the windows, first ones that a window
// has left behind, or compressed ones), 32 to a wave, and streams a segment of the tokens
// that attend any of them, a tile of 16 heads at a time; the exponentials of one tile stand
// between the MFMAs of the next. Two workgroups a CU: 64 tokens each of two sequences, 64 heads
// over 57400 rows of 512 channels in all, 208 us, 1.16 PFLOP/s (a large matrix product: 1.20).
// A wave with 64 rows (half the LDS reads, but alone on its SIMD) took 297 us where this took
// 228, with 48 rows 295.
// Tiles of at most 32 rows (a few first rows: keys of every token behind them) are held by
// all four waves, which take four tiles of queries at once.

struct RowParts {
  int seg;                        // tokens a segment
  int win_blocks, first_blocks;   // workgroups of window tiles, then of first rows' tiles; compressed ones follow
};

// Part, sequence, tile and segment of a workgroup: tiles x segments of the part's sequences one
// after the other.
struct RowItem {
  int part;                  // 0 window, 1 first rows, 2 compressed
  int b, p0, rows;           // sequence; the tile's first position and how many
  int a0, a1;                // its tokens, offsets in the sequence
  int qp, sg0;               // packed index of the sequence's first token, its position
};

template <int ROWS>
__device__ __forceinline__ bool find_item(const WeightParams& wp, const RowParts& rp, int blk, int lane, RowItem& o) {
  const FwdParams& p = wp.f;
  o.part = blk < rp.win_blocks ? 0 : blk < rp.win_blocks + rp.first_blocks ? 1 : 2;
  const int at = blk - (o.part == 0 ? 0 : o.part == 1 ? rp.win_blocks : rp.win_blocks + rp.first_blocks);
  const bool cu = p.act_q == nullptr;
  long long base = 0;
  for (int c = 0; c < p.B; c += 64) {
    const int i = c + lane;
    int qp = 0, aq = 0, sg0 = 0, lo = 0, hi = 0, nseg = 0;
    if (i < p.B) {
      qp = p.q_prefix[i];
      const int next = i + 1 < p.B ? p.q_prefix[i + 1] : p.T;
      const int len = cu ? p.q_prefix[i + 1] - qp : p.act_q[i];
      sg0 = p.act_kv[i] - len;
      // tokens up to the next sequence's first, as batch_of() tells them apart
      aq = qp < 0 ? 0 : max(0, min(len, min(next, p.T) - qp));
      const int last = sg0 + aq - 1;                     // last position
      if (aq > 0 && last >= 0) {
        int most = aq;                                   // tokens of a tile
        if (o.part == 0) {
          lo = max(max(sg0, 0) - p.win_left, 0);
          hi = min(last + 1, wp.ori_cap);
          most = (int)min((long long)aq, (long long)p.win_left + ROWS);
        } else if (o.part == 1) {
          hi = min(min(p.first, wp.ori_cap), last - p.win_left);
        } else {
          hi = min(min((last + 1) / p.cmp_ratio, p.K), wp.cmp_cap);
        }
        nseg = (most + rp.seg - 1) / rp.seg;
      }
    }
    const int n = max(hi - lo, 0);
    const long long items = (long long)((n + ROWS - 1) / ROWS) * nseg;
    long long x = items;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) { const long long v = __shfl_up(x, d); x += lane >= d ? v : 0; }
    const uint64_t m = __ballot(base + x > at);
    if (m) {
      const int j = __ffsll((unsigned long long)m) - 1;
      const int k = __builtin_amdgcn_readfirstlane((int)(at - base - (__shfl(x, j) - __shfl(items, j))));
      nseg = __builtin_amdgcn_readfirstlane(__shfl(nseg, j));
      lo = __builtin_amdgcn_readfirstlane(__shfl(lo, j));
      hi = __builtin_amdgcn_readfirstlane(__shfl(hi, j));
      aq = __builtin_amdgcn_readfirstlane(__shfl(aq, j));
      o.b = c + j;
      o.qp = __builtin_amdgcn_readfirstlane(__shfl(qp, j));
      o.sg0 = __builtin_amdgcn_readfirstlane(__shfl(sg0, j));
      o.p0 = lo + k / nseg * ROWS;
      o.rows = min(ROWS, hi - o.p0);
      // tokens [a0, a1) that attend any row of the tile, of which this segment
      long long a0 = max(0, -o.sg0), a1 = aq;
      if (o.part == 0) {
        a0 = max(a0, (long long)o.p0 - o.sg0);
        a1 = min(a1, (long long)o.p0 + o.rows + p.win_left - o.sg0);
      } else if (o.part == 1) {
        a0 = max(a0, (long long)o.p0 + p.win_left + 1 - o.sg0);
      } else {
        a0 = max(a0, ((long long)o.p0 + 1) * p.cmp_ratio - 1 - o.sg0);
      }
      a0 += (long long)(k % nseg) * rp.seg;
      o.a0 = (int)min(a0, a1);
      o.a1 = (int)min(a1, a0 + rp.seg);
      return o.a0 < o.a1;
    }
    base += __shfl(x, 63);
  }
  return false;
}

template <int D, typename QT, bool F8, int RT>
__global__ void __launch_bounds__(256, 2) sas_weights_rows_kernel(const WeightParams wp, const RowParts rp) {
  using Q = Queries<D>;
  constexpr int NB = 4, ROWS = 64 * RT, PF = 5;
  __shared__ __attribute__((aligned(1024))) typename Q::Tile tiles[NB];
  __shared__ float joined[4][16 * RT];

  const FwdParams& p = wp.f;
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int c16 = lane & 15, g = lane >> 4;
  RowItem it;
  if (!find_item<ROWS>(wp, rp, (int)blockIdx.x, lane, it)) return;
  const bool few = it.rows <= 16 * RT;      // every wave holds all rows
  const int ntile = p.H / 16, units = (it.a1 - it.a0) * ntile;
  const Q queries(p, (size_t)it.qp + it.a0, wave, lane);
#pragma unroll
  for (int i = 0; i < NB - 1; ++i)
    if (i < units) queries.issue(tiles[i], i);

  // lane (g, c16) holds rows r0 + 16 rt + c16 of the tile, attended from position `from` to `to`
  const int r0 = few ? 0 : 16 * RT * wave;
  const bool cmp = it.part == 2;
  const int bs = cmp ? p.cmp_bs : p.ori_bs, stride = cmp ? p.cmp_bt_stride : p.ori_bt_stride;
  const int32_t* bt = (cmp ? p.cmp_bt : p.ori_bt) + (size_t)it.b * stride;
  double* const wrow = cmp ? wp.cmp_w + (size_t)it.b * wp.cmp_rows : wp.ori_w + (size_t)it.b * wp.ori_rows;
  bool ok[RT];
  int from[RT], to[RT];
  uint4 k[RT][D / 32];
  float sc[RT][F8 ? 4 : 1];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int r = r0 + 16 * rt + c16, pos = it.p0 + r, blk = pos / bs;
    ok[rt] = r < it.rows && blk < stride && pos < (cmp ? wp.cmp_rows : wp.ori_rows);
    const int phys = ok[rt] ? bt[blk] : -1;
    ok[rt] = ok[rt] && phys >= 0 && phys < (cmp ? p.cmp_nblocks : p.ori_nblocks);
    from[rt] = it.part == 0 ? pos : it.part == 1 ? (int)min((long long)pos + p.win_left + 1, (long long)INT_MAX)
                                                 : (int)min(((long long)pos + 1) * p.cmp_ratio - 1, (long long)INT_MAX);
    to[rt] = it.part == 0 ? (int)min((long long)pos + p.win_left, (long long)INT_MAX) : INT_MAX;
    constexpr int ROWB = F8 ? kRow656 : D * 2;
    // (a row that is not there: the query's bytes, masked out)
    const uint64_t row = ok[rt] ? reinterpret_cast<uint64_t>(cmp ? p.cmp_kv : p.ori_kv) +
                                      (uint64_t)(uint32_t)(phys * bs + pos - blk * bs) * ROWB
                                : reinterpret_cast<uint64_t>(queries.q);
    load_row<D, F8>(row, g, k[rt], sc[rt]);
  }
  const int sg1 = it.sg0 + it.a0;           // position of the first token

  float acc[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) acc[rt] = 0.f;
  __builtin_amdgcn_s_waitcnt(0);
  if (few) {
    for (int i0 = 0; i0 < units; i0 += NB) {
#pragma unroll
      for (int j = 0; j < NB; ++j)          // (of the first four, three are under way)
        if (i0 + j < units && (i0 > 0 || j == NB - 1)) queries.issue(tiles[j], i0 + j);
      queries.wait(0);
      lds_barrier();
      const int i = i0 + wave;
      if (i < units) {
        const typename Q::Tile& tile = tiles[wave];
        const int sg = sg1 + i / ntile;
        const f32x4 l2 = *reinterpret_cast<const f32x4*>(&tile.lse[4 * g]) * kLog2e;
        f32x4 s[RT];
        tile_scores<D, QT, F8, RT, PF>(tile, k, sc, g, c16, s, [] {});
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          const float x = shares(s[rt], l2, p.scale_log2);
          acc[rt] += sg >= from[rt] && sg <= to[rt] ? x : 0.f;
        }
      }
      lds_barrier();                        // the four are read
    }
    // the waves' sums meet in wave 0
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const float w = rows_sum(acc[rt]);
      if (g == 0) joined[wave][16 * rt + c16] = w;
    }
    __syncthreads();
    if (wave == 0 && g == 0) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        const int r = 16 * rt + c16;
        if (ok[rt]) add_weight(wrow + it.p0 + r, (joined[0][r] + joined[1][r]) + (joined[2][r] + joined[3][r]), wp.units);
      }
    }
    return;
  }
  // unit i's scores are computed while unit i - 1's become weights
  f32x4 so[RT], lse2 = f32x4{0.f, 0.f, 0.f, 0.f};
  int tok = 0, head = 0;                    // unit i's token and head tile
  bool use[RT], uso[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) { so[rt] = lse2; uso[rt] = false; use[rt] = false; }
  auto weigh = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const float x = shares(so[rt], lse2, p.scale_log2);
      acc[rt] += uso[rt] ? x : 0.f;
    }
  };
  for (int i = 0; i < units; ++i) {
    // unit i is here once only the units behind it, at most NB - 2 of them, are under way
    if (i >= NB - 1) queries.wait(min(NB - 2, units - 1 - i));
    lds_barrier();   // every wave's part of unit i is here, and unit i - 1 is read
    if (i + NB - 1 < units) queries.issue(tiles[(i + NB - 1) % NB], i + NB - 1);
    if (head == 0) {
      const int sg = sg1 + tok;
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) use[rt] = sg >= from[rt] && sg <= to[rt];
    }
    const typename Q::Tile& tile = tiles[i % NB];
    const f32x4 l2 = *reinterpret_cast<const f32x4*>(&tile.lse[4 * g]) * kLog2e;
    f32x4 s[RT];
    tile_scores<D, QT, F8, RT, PF>(tile, k, sc, g, c16, s, weigh);
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) { so[rt] = s[rt]; uso[rt] = use[rt]; }
    lse2 = l2;
    if (++head == ntile) { head = 0; ++tok; }
  }
  weigh();
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const float w = rows_sum(acc[rt]);
    if (g == 0 && ok[rt]) add_weight(wrow + it.p0 + r0 + 16 * rt + c16, w, wp.units);
  }
}

struct WeightPlan {
  long long slots;       // workgroups of sas_weights_kernel, 0: none
  long long rows;        // workgroups of sas_weights_rows_kernel, 0: none
  RowParts parts;
  WeightParams by_slot;  // what the former covers
};

constexpr int kRowTiles = 2;     // 16-row tiles a wave in sas_weights_rows_kernel
constexpr int kSegMax = 64, kSegMin = 4;   // its tokens a segment

template <int D, typename QT, bool F8>
int launch_weights(const WeightParams& wp, const WeightPlan& pl, hipStream_t st) {
  if (pl.rows)
    hipLaunchKernelGGL((sas_weights_rows_kernel<D, QT, F8, kRowTiles>), dim3((unsigned)pl.rows), dim3(256), 0, st, wp, pl.parts);
  if (pl.slots)
    hipLaunchKernelGGL((sas_weights_kernel<D, QT, F8>), dim3((unsigned)pl.slots), dim3(256), 0, st, pl.by_slot);
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
  WeightPlan pl{};
  pl.by_slot = wp;
  // tokens of a sequence that share its rows: by rows, but for the top-k ones
  const bool by_rows = a->T >= 4 * a->B;
  if (by_rows) {
    constexpr long long R = 64 * kRowTiles;
    // segments: as long as the tiles then still give most CUs their two workgroups
    auto up = [](long long n, long long d) { return (n + d - 1) / d; };
    const long long mean = std::max<long long>(1, a->T / a->B), before = std::min<long long>(a->win_left, wp.ori_cap);
    const long long ncmp = cmp && a->scenario == SAS_CFA ? std::min<long long>(wp.cmp_cap, a->K) : 0;
    const long long all = a->B * ((wp.ori_w ? up(std::min<long long>(wp.ori_cap, mean + before), R) : 0) + up(ncmp, R));
    int& seg = pl.parts.seg;
    seg = kSegMax;
    while (seg > kSegMin && 2 * all * up(std::min<long long>(mean, a->win_left + R), seg) < 3LL * device_cus()) seg /= 2;
    // A grid that holds any lengths. Of one sequence with m tokens: up(m, seg) segments for each
    // of its first or compressed rows' tiles; (before + m) / R + 1 tiles of window rows, each
    // with up(min(m, win_left + R), seg) segments.
    const long long segs = a->T / seg + a->B;
    if (wp.ori_w) {
      const long long w = (before / R + 2) * segs +
                          up(a->T, R) * (std::min<long long>(a->T, a->win_left + R) / seg + 1);
      const long long f = up(std::min<long long>(ra->ori_first, wp.ori_cap), R) * segs;
      if (w + f > INT_MAX) return set_error(SAS_EINVAL, "row weights: %lld workgroups beyond one launch", w + f);
      pl.parts.win_blocks = (int)w;
      pl.parts.first_blocks = (int)f;
      pl.rows = w + f;
      pl.by_slot.ori_w = nullptr;
    }
    if (ncmp) {
      pl.rows += up(ncmp, R) * segs;
      pl.by_slot.cmp_w = nullptr;
    }
    if (pl.rows > INT_MAX) return set_error(SAS_EINVAL, "row weights: %lld workgroups beyond one launch", pl.rows);
  }
  constexpr int ROWS = 64;
  const long long nori = pl.by_slot.ori_w ? std::min<long long>(wp.ori_cap, ra->ori_first + a->win_left + 1) : 0;
  const long long ncmp = !pl.by_slot.cmp_w ? 0 : a->scenario == SAS_SCFA ? a->K : std::min<long long>(wp.cmp_cap, a->K);
  const long long chunks = (nori + ncmp + ROWS - 1) / ROWS;
  pl.by_slot.spread = a->T >= 2 * fp.nxcd;
  pl.slots = (pl.by_slot.spread ? (a->T + fp.nxcd - 1) / fp.nxcd * fp.nxcd : a->T) * chunks;
  if (pl.slots > INT_MAX) return set_error(SAS_EINVAL, "row weights: %lld workgroups beyond one launch", pl.slots);
  pl.by_slot.chunks = (int)chunks;
  if (fp8) return launch_weights<576, __bf16, true>(wp, pl, st);
  if (a->q_dtype == SAS_DT_BF16)
    return a->D == 576 ? launch_weights<576, __bf16, false>(wp, pl, st) : launch_weights<512, __bf16, false>(wp, pl, st);
  return a->D == 576 ? launch_weights<576, _Float16, false>(wp, pl, st) : launch_weights<512, _Float16, false>(wp, pl, st);
}

}  // namespace
}  // namespace sas

extern "C" int sas_row_weights_v1(const SasRowWeightsArgs* a, void* stream) {
  sas::clear_error();
  if (!a) return sas::set_error(SAS_EINVAL, "row weights: null args");
  return sas::weights_impl(a, (hipStream_t)stream);
}
