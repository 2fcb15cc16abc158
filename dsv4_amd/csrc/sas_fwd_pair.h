// Draft trees, and calls with first rows, of more (token, 64 heads) items than compute units,
// and windows of fewer (use_pairs() has the rule): one item a workgroup of 4 waves, two workgroups on a CU,
// MI355X (gfx950). Where heads are no multiple of 64, waves without heads only move rows.
//
// The 8-wave kernel has a CU to itself: its ring fills the LDS, and nothing runs
// beside a token's slot resolution, its first rows and its output (8 of 46 us at 640
// rows of 576 channels). Here a workgroup keeps two 32-row slots (74 KB) and its row
// list as 32-bit indices, so that two share a CU, one's loads and softmax beside the
// other's MFMAs. A wave holds 16 heads over all keys and channels (O 128 registers,
// Q^T 72): scores, online softmax seeded by the sink (O and l rescaled when a row's
// maximum rises by more than 2^8), P.V, in steps of 32 rows whose DMA runs a step ahead.
//
// us against the 8-wave kernel (window-only: the exact-window one), 64 heads, 480 nodes
// / 960: 128-row window, D = 512 18 / 35 against 28 / 55, D = 576 19 / 37 against 29 / 58;
// with 512 top-k rows D = 512 50 / 94 against 63 / 122, D = 576 53 / 101 against 62 / 122;
// over contexts of 8 K to 32 K, read from HBM, 62 / 115 against 71 / 133 and 65 / 123 against
// 73 / 141. With lane offsets that spilled it was no faster at D = 576.
//
// What bounds it (518 nodes, 64 heads, 640 rows of 576 channels): no unit alone. Of a CU's
// time MFMAs take a third, LDS 37%, VALU 35%; a wave's phases hang on each other and only
// two waves share a SIMD. K and V operands read further ahead, wave priorities and rows in
// cache order gave nothing. 512 items take 57 us, the next six 18 more.
#pragma once

#include "sas_kern.h"

#ifndef SAS_FWD_TREE
#define SAS_FWD_TREE 0
#endif
#ifndef SAS_FWD_FIRST
#define SAS_FWD_FIRST 0
#endif

namespace sas {
namespace {

constexpr bool kPairTree = SAS_FWD_TREE, kPairFirst = SAS_FWD_FIRST;
constexpr int kPairPT = 4, kPairSRB = kPairPT * 32 + 16, kPairStage = 16 * kPairSRB;   // output staging of a wave

// 16 heads x 512 channels (lane (g, c16): channels 16 i + 4 g .. + 3 of head c16) scaled
// by inv, kPairPT channel tiles at a time through the wave's own LDS rows, out in
// whole runs of a head's row
template <typename QT>
__device__ __forceinline__ void put_out(const f32x4 (&acc)[kDV / 16], float inv, uint8_t* sb, uint8_t* ob, int lane) {
  constexpr int CPR = kPairPT * 2;
  const int c16 = lane & 15, g = lane >> 4;
#pragma unroll
  for (int c = 0; c < kDV / 16; c += kPairPT) {
#pragma unroll
    for (int i = 0; i < kPairPT; ++i)
      *reinterpret_cast<uint2*>(sb + c16 * kPairSRB + (i * 16 + 4 * g) * 2) =
          make_uint2(pack2<QT>(acc[c + i][0] * inv, acc[c + i][1] * inv), pack2<QT>(acc[c + i][2] * inv, acc[c + i][3] * inv));
#pragma unroll
    for (int i = 0; i < 16 * CPR / 64; ++i) {
      const int e = i * 64 + lane, r = e / CPR, q = e - r * CPR;
      const u32x4g w = *reinterpret_cast<const u32x4g*>(sb + r * kPairSRB + q * 16);
      __builtin_nontemporal_store(w, reinterpret_cast<u32x4g*>(ob + (size_t)r * kDV * 2 + c * 32 + q * 16));
    }
  }
}
// an item without rows: zeros, and the sink (a padded token: 0)
__device__ __forceinline__ void put_none(uint8_t* ob, float* lse, float lse0, int lane) {
  uint4* o = reinterpret_cast<uint4*>(ob);
#pragma unroll
  for (int i = 0; i < 16 * kDV * 2 / 16 / 64; ++i) o[i * 64 + lane] = make_uint4(0, 0, 0, 0);
  if (lane < 16) lse[lane] = lse0;
}

// Online softmax of a step's scores (lane (g, c16): keys 16 mt + 4 g + j of head c16;
// nk of the 32 keys count), in the log2 domain: P in s, the lane's sum in l, and O and l
// rescaled in place where a row's maximum rises by more than 2^8 over the reference m.
// The callers round P (or P x scale) once to 16 bits, which P.V's MFMAs take; l sums
// it in fp32 before that. Half a step a key, independent over the keys: outputs are
// 0.0021-0.0023 of their norm from 64 bits (bf16; fp16 0.00029), with P in 32 bits 0.0017
// (0.00021), which is the output's own rounding.
__device__ __forceinline__ void softmax_step(f32x4 (&s)[2], f32x4 (&acc)[kDV / 16], float& m, float& l, float scale,
                                             int nk, int g) {
  float mx = -INFINITY;
#pragma unroll
  for (int mt = 0; mt < 2; ++mt) s[mt] *= scale;
  if (nk < 32) {
#pragma unroll
    for (int mt = 0; mt < 2; ++mt)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (16 * mt + 4 * g + j >= nk) s[mt][j] = -INFINITY;
  }
#pragma unroll
  for (int mt = 0; mt < 2; ++mt) mx = fmaxf(mx, fmaxf(fmaxf(s[mt][0], s[mt][1]), fmaxf(s[mt][2], s[mt][3])));
  mx = rows_max(mx);
  if (__ballot(mx > m + kLazyLog2)) {
    const float mn = fmaxf(m, mx), al = m == mn ? 1.f : __builtin_amdgcn_exp2f(m - mn);
    l *= al;
    m = mn;
#pragma unroll
    for (int i = 0; i < kDV / 16; ++i)   // in place: written as a product, the accumulators are copied on both paths
      asm volatile("v_mul_f32 %0, %4, %0\n\tv_mul_f32 %1, %4, %1\n\tv_mul_f32 %2, %4, %2\n\tv_mul_f32 %3, %4, %3"
                   : "+v"(acc[i][0]), "+v"(acc[i][1]), "+v"(acc[i][2]), "+v"(acc[i][3]) : "v"(al));
  }
  const float mb = m == -INFINITY ? 0.f : m;             // no sink and no finite score yet: every P is 0
#pragma unroll
  for (int mt = 0; mt < 2; ++mt)
#pragma unroll
    for (int j = 0; j < 4; ++j) { s[mt][j] = __builtin_amdgcn_exp2f(s[mt][j] - mb); l += s[mt][j]; }
}

template <int D, typename QT>
__global__ void __launch_bounds__(256, 2) sas_fwd_pair_kernel(const FwdParams p) {
  // slot: the 32 rows' latent chunks [32][64] (chunk c of row r at c ^ swz<64>(r)), then,
  // D = 576, their rope chunks [32][8] (at c ^ (r >> 1)): a latent row is one DMA
  // instruction, eight rows' rope another
  constexpr int KS = D / 32, NT = kDV / 16, LCH = 64, ROPE = D > kDV, RI = 8 + ROPE;
  constexpr int LAT = 32 * LCH * 16, SLOT = LAT + ROPE * 32 * 128;
  static_assert(4 * kPairStage <= SLOT, "the output is staged in the first slot");
  static_assert(2 * SLOT + kMaxSlots * 4 + 1024 <= 80 * 1024, "two workgroups share a CU's LDS");
  __shared__ __attribute__((aligned(1024))) uint8_t ring[2 * SLOT];
  __shared__ uint32_t rows[kMaxSlots];

  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int c16 = lane & 15, g = lane >> 4;
  const int item = item_index<kPairTree>(p);
  if (item < 0) return;
  Tok k = item_of(p, item);
  // (heads past the last: a wave without heads only moves rows; its addresses stay valid)
  const bool mine = k.hg * 64 + wave * 16 < p.H;
  const int hq = mine ? k.hg * 64 + wave * 16 : p.H - 16;
  uint4 qf[KS];
  resolve<256, D * 2, kPairTree, true, kPairFirst>(p, k, tid, lane, wave, [&] {
    const uint4* q = reinterpret_cast<const uint4*>(p.q + ((size_t)k.t * p.H + hq + c16) * D * 2) + g;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) qf[ks] = q[ks * 4];
  }, rows);
  const int n = __builtin_amdgcn_readfirstlane(k.nvalid), steps = (n + 31) >> 5;
  uint8_t* ob = p.out + ((size_t)k.t * p.H + hq) * kDV * 2;
  float* lse = p.lse + (size_t)k.t * p.H + hq;
  const float sink2 = p.sinks[hq + c16] * kLog2e;
  if (n == 0) {
    if (mine) put_none(ob, lse, k.padded ? 0.f : sink2 * kLn2, lane);
    return;
  }

  // producer: a wave moves rows 8 wave .. + 7 of every step in RI instructions; rows
  // past the last repeat it (masked out of the softmax, and finite for P.V)
  const uint64_t ob_ = reinterpret_cast<uint64_t>(p.ori_kv), cb_ = reinterpret_cast<uint64_t>(p.cmp_kv);
  auto row_addr = [&](int j) {
    const uint32_t e = rows[min(j, n - 1)];
    return (e >> 31 ? cb_ : ob_) + (uint64_t)(e & 0x7fffffffu) * (D * 2);
  };
  int ps = 0;                // producer's step
  uint64_t pl = 0, pp = 0;   // address of row 8 wave + (lane & 7) / + (lane >> 3) of the step
  auto prep = [&](int ln) {
    pl = row_addr(ps * 32 + 8 * wave + (ln & 7));
    if (ROPE) pp = row_addr(ps * 32 + 8 * wave + (ln >> 3));
  };
  // Lane offsets are made anew from the lane index each step (ln: a copy the compiler
  // cannot see through): kept over the loop they spill, and a reload waits for the
  // row DMA in flight.
  auto fire = [&](int m, int ln) {
    const uint32_t ol = (uint32_t)ln * 16, orp = 1024 + (uint32_t)(((ln & 7) ^ (((8 * wave + (ln >> 3)) >> 1) & 7)) * 16);
    const uint32_t slot = lds_addr_of(ring + (ps & 1) * SLOT);
    if (m < 8) {
      const uint64_t a = ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(pl >> 32), m) << 32) |
                         (uint32_t)__builtin_amdgcn_readlane((int)pl, m);
      dma16s(ol ^ (uint32_t)(swz<LCH>(m) * 16), reinterpret_cast<const void*>(a),
             __builtin_amdgcn_readfirstlane(slot + (8 * wave + m) * 1024));
    } else {
      dma16(reinterpret_cast<const void*>(pp + orp), __builtin_amdgcn_readfirstlane(slot + LAT + 8 * wave * 128));
    }
  };
  prep(lane);
#pragma unroll
  for (int m = 0; m < RI; ++m) fire(m, lane);
  ++ps;
  if (!mine) {   // wave-uniform; the same barriers as below
    for (int st = 0; st < steps; ++st, ++ps) {
      wait_vm<0>();
      lds_barrier();
      asm volatile("" ::: "memory");   // (the barrier's builtins alone hold no memory access back)
      prep(lane);
#pragma unroll
      for (int m = 0; m < RI; ++m) fire(m, lane);
    }
    wait_vm<0>();
    lds_barrier();
    return;
  }
  f32x4 acc[NT];
#pragma unroll
  for (int i = 0; i < NT; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = sink2, l = 0.f;                                // l: this lane's keys
  // the query is here before the loop: a load the compiler tracks inside it would
  // make each step wait for every row DMA in flight
  __builtin_amdgcn_s_waitcnt(0);
  for (int st = 0; st < steps; ++st) {
    wait_vm<0>();                                          // my DMA of this step
    lds_barrier();
    asm volatile("" ::: "memory");
    const uint8_t* kt = ring + (st & 1) * SLOT;
    int ln = lane;
    asm volatile("" : "+v"(ln));
    const int lc = ln & 15, lg = ln >> 4;
    prep(ln);
    const uint32_t ka = (uint32_t)(lc * 1024 + ((lg ^ swz<LCH>(lc)) * 16));
    const uint32_t kr = (uint32_t)(LAT + lc * 128 + ((lg ^ (lc >> 1)) * 16));   // rope: rows 16 apart share the xor
    f32x4 s[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
    {
      auto kfrag = [&](int ks, int mt) {
        return *reinterpret_cast<const uint4*>(
            kt + (ks < 16 ? (ka ^ (uint32_t)((ks & 3) * 64)) + (ks >> 2) * 256 + mt * 16 * 1024
                          : (kr ^ (uint32_t)((ks & 1) * 64)) + mt * 16 * 128));
      };
      constexpr int PF = 2;
      uint4 a[PF][2];
#pragma unroll
      for (int i = 0; i < PF; ++i) { a[i][0] = kfrag(i, 0); a[i][1] = kfrag(i, 1); }
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const uint4 a0 = a[ks % PF][0], a1 = a[ks % PF][1];
        if (ks + PF < KS) { a[ks % PF][0] = kfrag(ks + PF, 0); a[ks % PF][1] = kfrag(ks + PF, 1); }
        s[0] = mfma32k<QT>(a0, qf[ks], s[0]);
        s[1] = mfma32k<QT>(a1, qf[ks], s[1]);
        if (ks % 2 == 1 && ks / 2 < RI) fire(ks / 2, ln);  // the next step's rows (past the last: its last again)
      }
      ++ps;
    }
    softmax_step(s, acc, m, l, p.scale_log2, n - st * 32, lg);
    uint32_t pk[4];
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
      pk[2 * mt] = pack2<QT>(s[mt][0], s[mt][1]);
      pk[2 * mt + 1] = pack2<QT>(s[mt][2], s[mt][3]);
    }
    const uint4 pf = make_uint4(pk[0], pk[1], pk[2], pk[3]);
    int vn = lane;
    asm volatile("" : "+v"(vn));
    const int vr = 4 * (vn >> 4) + ((vn & 15) >> 2);
    const uint32_t va = (uint32_t)(vr * 1024 + ((((vn & 3) >> 1) ^ swz<LCH>(vr)) * 16) + (vn & 1) * 8);
    auto vfrag = [&](int ct) {
      const uint8_t* b0 = kt + ((va ^ (uint32_t)((ct & 7) * 32)) + (ct >> 3) * 256);
      const uint2 u0 = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS_AS i16x4*)(b0)));
      const uint2 u1 = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS_AS i16x4*)(b0 + 16 * 1024)));
      return make_uint4(u0.x, u0.y, u1.x, u1.y);
    };
    constexpr int PV = 4;
    uint4 v[PV];
#pragma unroll
    for (int i = 0; i < PV; ++i) v[i] = vfrag(i);
#pragma unroll
    for (int ct = 0; ct < NT; ++ct) {
      const uint4 a = v[ct % PV];
      if (ct + PV < NT) v[ct % PV] = vfrag(ct + PV);
      acc[ct] = mfma32k<QT>(a, pf, acc[ct]);
    }
    __builtin_amdgcn_sched_group_barrier(0x100, 2 * PV, 1);
#pragma unroll
    for (int ct = 0; ct < NT; ++ct) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 1);
      if (ct + PV < NT) __builtin_amdgcn_sched_group_barrier(0x100, 2, 1);
    }
  }
  l = rows_sum(l) + __builtin_amdgcn_exp2f(sink2 - (m == -INFINITY ? 0.f : m));
  const float inv = l == 0.f ? 0.f : 1.f / l;              // (0: no sink, no row)
  wait_vm<0>();                                            // the spare step's DMA
  lds_barrier();                                           // every wave has done with the ring: the output is staged there
  asm volatile("" ::: "memory");
  put_out<QT>(acc, inv, ring + wave * kPairStage, ob, lane);
  if (g == 0) lse[c16] = m * kLn2 + logf(l);
}

// The same over fp8 rows (576 channels): two slots of 21 KB take the rows as they are
// (latent bytes [32 rows][512], rope [32][8 chunks] (chunk c of row r at c ^ (r >> 1)), the
// rows' four scales [32][16 bytes]), and at a step's head each wave turns the latent bytes
// that it loaded into bf16 (exactly, unscaled) in one tile of the other kernel's layout: one
// conversion a value where a fragment converted as it is read has one in each of four
// waves (4 trees of 64 nodes, 128 heads, 1152 rows: 115-117 us against 134, 381 VALU instructions
// a step and wave against 729, 68 of them MFMAs). A scale group's four k-steps are a chain of
// their own, folded into S with the rows' fp32 scales, and P x scale is what is rounded for P.V.
// us against the 32-head kernel, which needs four rounds: 480 nodes, 64 heads, 128-row window
// 24 against 64, with 1024 top-k rows 115 against 162.
constexpr int kPair8Slot = 21 * 1024, kPair8Rope = 16 * 1024, kPair8Scl = 20 * 1024;

__global__ void __launch_bounds__(256, 2) sas_fwd_pair8_kernel(const FwdParams p) {
  constexpr int D = 576, KS = D / 32, NT = kDV / 16, LCH = 64;
  typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
  static_assert(4 * kPairStage <= kPair8Slot && 2 * kPair8Slot + 32 * LCH * 16 + kMaxSlots * 4 + 1024 <= 80 * 1024, "LDS");
  __shared__ __attribute__((aligned(1024))) uint8_t ring[2 * kPair8Slot];
  __shared__ __attribute__((aligned(1024))) uint8_t tile[32 * LCH * 16];
  __shared__ uint32_t rows[kMaxSlots];

  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int c16 = lane & 15, g = lane >> 4;
  const int item = item_index<kPairTree>(p);
  if (item < 0) return;
  Tok k = item_of(p, item);
  // (heads past the last: a wave without heads only moves rows; its addresses stay valid)
  const bool mine = k.hg * 64 + wave * 16 < p.H;
  const int hq = mine ? k.hg * 64 + wave * 16 : p.H - 16;
  uint4 qf[KS];
  resolve<256, kRow656, kPairTree, true, kPairFirst>(p, k, tid, lane, wave, [&] {
    const uint4* q = reinterpret_cast<const uint4*>(p.q + ((size_t)k.t * p.H + hq + c16) * D * 2) + g;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) qf[ks] = q[ks * 4];
  }, rows);
  const int n = __builtin_amdgcn_readfirstlane(k.nvalid), steps = (n + 31) >> 5;
  uint8_t* ob = p.out + ((size_t)k.t * p.H + hq) * kDV * 2;
  float* lse = p.lse + (size_t)k.t * p.H + hq;
  const float sink2 = p.sinks[hq + c16] * kLog2e;
  if (n == 0) {
    if (mine) put_none(ob, lse, k.padded ? 0.f : sink2 * kLn2, lane);
    return;
  }

  // producer: of a step's 21 DMA instructions wave w issues latent ones w + 4 j (rows 2 w + 8 j
  // and the next), rope one w (eight rows) and, wave 0, the scales' (32 rows); rows past the
  // last repeat it
  const uint64_t ob_ = reinterpret_cast<uint64_t>(p.ori_kv), cb_ = reinterpret_cast<uint64_t>(p.cmp_kv);
  auto fire = [&](int step, int j, int ln) {
    const int r = j < 4 ? 2 * (wave + 4 * j) + (ln >> 5) : j == 4 ? 8 * wave + (ln >> 3) : ln & 31;
    const uint32_t col = j < 4 ? (uint32_t)((ln & 31) * 16)
                         : j == 4 ? 528u + (uint32_t)(((ln & 7) ^ ((r >> 1) & 7)) * 16) : 512u;
    const uint32_t e = rows[min(step * 32 + r, n - 1)];
    const uint64_t a = (e >> 31 ? cb_ : ob_) + (uint64_t)(e & 0x7fffffffu) * kRow656 + col;
    const int i = j < 4 ? wave + 4 * j : j == 4 ? 16 + wave : 20;
    dma16(reinterpret_cast<const void*>(a),
          __builtin_amdgcn_readfirstlane(lds_addr_of(ring) + (uint32_t)(step & 1) * kPair8Slot + i * 1024));
  };
  // my rows of the slot at sl, bf16, into the tile
  auto convert = [&](uint32_t sl, int ln) {
    const uint32_t src = sl + (uint32_t)(2 * wave * 512 + ln * 8), dst = lds_addr_of(tile) + (uint32_t)(2 * wave * 1024);
    constexpr int kBatch = 4;
#pragma unroll
    for (int b0 = 0; b0 < 8; b0 += kBatch) {
      u32x2 raw[kBatch];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {   // row 2 wave + 8 (i / 2) + i % 2
        const int e = b0 + i;
        raw[i] = *reinterpret_cast<const LDS_AS u32x2*>((size_t)(src + (uint32_t)((e >> 1) * 8 + (e & 1)) * 512));
      }
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const int e = b0 + i;
        uint4 b;
        e4m3x4_to_bf16(raw[i].x, b.x, b.y);
        e4m3x4_to_bf16(raw[i].y, b.z, b.w);
        *reinterpret_cast<LDS_AS u32x4g*>((size_t)(dst + (uint32_t)((ln ^ swz<LCH>(2 * wave + (e & 1))) * 16) +
                                                   (uint32_t)((e >> 1) * 8 + (e & 1)) * 1024)) = __builtin_bit_cast(u32x4g, b);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
#pragma unroll
  for (int j = 0; j < 5; ++j) fire(0, j, lane);
  if (wave == 0) fire(0, 5, lane);
  if (!mine) {   // wave-uniform; the same barriers as below (wave 0 always has heads)
    for (int st = 0; st < steps; ++st) {
      wait_vm<0>();
      lds_barrier();
      asm volatile("" ::: "memory");
      convert(lds_addr_of(ring) + (uint32_t)(st & 1) * kPair8Slot, lane);
      lds_barrier();
      asm volatile("" ::: "memory");
#pragma unroll
      for (int j = 0; j < 5; ++j) fire(st + 1, j, lane);
    }
    wait_vm<0>();
    lds_barrier();
    return;
  }
  f32x4 acc[NT];
#pragma unroll
  for (int i = 0; i < NT; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = sink2, l = 0.f;                                // l: this lane's keys
  __builtin_amdgcn_s_waitcnt(0);                           // the query is here before the loop, as above
  for (int st = 0; st < steps; ++st) {
    wait_vm<0>();                                          // my DMA of this step
    lds_barrier();                                         // the last step's tile has been read
    asm volatile("" ::: "memory");
    const uint32_t sl = lds_addr_of(ring) + (uint32_t)(st & 1) * kPair8Slot, kt = lds_addr_of(tile);
    // (lane offsets made anew each step: kept, they spill, and a reload waits for the DMA)
    int ln = lane;
    asm volatile("" : "+v"(ln));
    convert(sl, ln);
    lds_barrier();
    asm volatile("" ::: "memory");
    const int lc = ln & 15, lg = ln >> 4;
    const uint32_t ka = kt + (uint32_t)(lc * 1024 + ((lg ^ swz<LCH>(lc)) * 16));
    const uint32_t kr = sl + (uint32_t)(kPair8Rope + lc * 128 + ((lg ^ ((lc >> 1) & 7)) * 16));
    const uint32_t sa = sl + (uint32_t)(kPair8Scl + lg * 64);
    auto kfrag = [&](int ks, int mt) {
      return __builtin_bit_cast(uint4, *reinterpret_cast<const LDS_AS u32x4g*>((size_t)(
          ks < 16 ? (ka ^ (uint32_t)((ks & 3) * 64)) + (uint32_t)((ks >> 2) * 256 + mt * 16 * 1024)
                  : (kr ^ (uint32_t)((ks & 1) * 64)) + (uint32_t)(mt * 16 * 128))));
    };
    auto scales = [&](int G, int mt) {   // of the lane's keys 16 mt + 4 g + j
      const LDS_AS float* f = reinterpret_cast<const LDS_AS float*>((size_t)(sa + (uint32_t)(16 * mt * 16 + 4 * G)));
      return f32x4{f[0], f[4], f[8], f[12]};
    };
    f32x4 s[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
    {
      uint4 a[2] = {kfrag(0, 0), kfrag(0, 1)};   // (two k-steps ahead, a fragment of Q^T spills: 115 -> 122 us)
      f32x4 gacc[2];
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const uint4 a0 = a[0], a1 = a[1];
        if (ks + 1 < KS) { a[0] = kfrag(ks + 1, 0); a[1] = kfrag(ks + 1, 1); }
        if (ks < 16) {
          const bool first = ks % 4 == 0;
          gacc[0] = mfma32k<__bf16>(a0, qf[ks], first ? f32x4{0.f, 0.f, 0.f, 0.f} : gacc[0]);
          gacc[1] = mfma32k<__bf16>(a1, qf[ks], first ? f32x4{0.f, 0.f, 0.f, 0.f} : gacc[1]);
          if (ks % 4 == 3) {
            s[0] += scales(ks / 4, 0) * gacc[0];
            s[1] += scales(ks / 4, 1) * gacc[1];
            __builtin_amdgcn_sched_barrier(0);   // (the next groups' scales at once spill)
          }
        } else {
          s[0] = mfma32k<__bf16>(a0, qf[ks], s[0]);
          s[1] = mfma32k<__bf16>(a1, qf[ks], s[1]);
        }
        if (ks % 3 == 1 && ks / 3 < 5) fire(st + 1, ks / 3, ln);   // (past the last step: its last row again)
      }
      if (wave == 0) fire(st + 1, 5, ln);
    }
    softmax_step(s, acc, m, l, p.scale_log2, n - st * 32, lg);
    int vn = lane;
    asm volatile("" : "+v"(vn));
    const int vr = 4 * (vn >> 4) + ((vn & 15) >> 2);
    const uint32_t va = kt + (uint32_t)(vr * 1024 + ((((vn & 3) >> 1) ^ swz<LCH>(vr)) * 16) + (vn & 1) * 8);
    auto vfrag = [&](int ct) {
      const uint32_t b0 = (va ^ (uint32_t)((ct & 7) * 32)) + (uint32_t)((ct >> 3) * 256);
      const uint2 u0 = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS_AS i16x4*)(size_t)b0));
      const uint2 u1 = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS_AS i16x4*)(size_t)(b0 + 16 * 1024)));
      return make_uint4(u0.x, u0.y, u1.x, u1.y);
    };
    constexpr int PV = 4;
    uint4 v[PV];
#pragma unroll
    for (int i = 0; i < PV; ++i) v[i] = vfrag(i);
#pragma unroll
    for (int G = 0; G < 4; ++G) {
      uint32_t pk[4];
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
        const f32x4 f = scales(G, mt) * s[mt];
        pk[2 * mt] = pack2<__bf16>(f[0], f[1]);
        pk[2 * mt + 1] = pack2<__bf16>(f[2], f[3]);
        __builtin_amdgcn_sched_barrier(0);
      }
      const uint4 pf = make_uint4(pk[0], pk[1], pk[2], pk[3]);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int ct = 8 * G + i;
        const uint4 a = v[ct % PV];
        if (ct + PV < NT) v[ct % PV] = vfrag(ct + PV);
        acc[ct] = mfma32k<__bf16>(a, pf, acc[ct]);
      }
    }
  }
  l = rows_sum(l) + __builtin_amdgcn_exp2f(sink2 - (m == -INFINITY ? 0.f : m));
  const float inv = l == 0.f ? 0.f : 1.f / l;              // (0: no sink, no row)
  wait_vm<0>();                                            // the spare step's DMA
  lds_barrier();                                           // every wave has done with the ring: the output is staged there
  asm volatile("" ::: "memory");
  put_out<__bf16>(acc, inv, ring + wave * kPairStage, ob, lane);
  if (g == 0) lse[c16] = m * kLn2 + logf(l);
}

int pair_launched() {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? SAS_OK : sas::set_error(SAS_ELAUNCH, "sas_fwd_pair launch: %s", hipGetErrorString(e));
}
template <int D, typename QT>
int launch_pair(const FwdParams& fp, int nblocks, hipStream_t st) {
  hipLaunchKernelGGL((sas_fwd_pair_kernel<D, QT>), dim3(nblocks), dim3(256), 0, st, fp);
  return pair_launched();
}
int launch_pair8(const FwdParams& fp, int nblocks, hipStream_t st) {
  hipLaunchKernelGGL(sas_fwd_pair8_kernel, dim3(nblocks), dim3(256), 0, st, fp);
  return pair_launched();
}

}  // namespace
}  // namespace sas
