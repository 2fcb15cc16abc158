// Norms of queries and KV rows for each head with the rotation by position in
// the same pass, its backward, and the cache append that writes the rotated KV
// rows where the forward reads them, MI355X (gfx950).
//
// A row is one head of one token (or one token's KV row), D channels. With n
// normed channels, weights w and the angle pairs (c, s) of the row's position:
//   y = x,  y[:n] = x[:n] r w,  r = (sum x[:n]^2 / n + eps)^(-1/2)
//   (a, b) -> (a c - b s, a s + b c)  on the pairs of the last R channels
// and for an output gradient dy, with u = dy rotated back and g = u w:
//   dx[:n] = r (g - x r^2 (sum g x) / n),  dx[n:] = u,  dw = sum_rows u x r.
//
// All of it is HBM-bound: a row is read once and written once (backward: two
// reads), 2 D bytes each way, against some 5 VALU operations a channel. Eight
// lanes share a row and a wave takes eight rows: channel chunk (8 channels, 16
// bytes) 8 i + l of its row belongs to lane l of the eight, so a load
// instruction covers whole 128-byte lines, 512 and 576 channels come out even (8 or
// 9 loads a lane, all in flight at once; a wave a row leaves 56 of 64 lanes
// idle in the second load of 576), and a row's sums take three DPP steps. The 64
// rotated channels are then the last chunk of every lane. Nothing passes
// through LDS but the backward's weight sums.

#include "sas_kern.h"

namespace sas {
namespace {

constexpr int kRopeThreads = 256, kRopeRows = kRopeThreads / 8;   // rows a workgroup takes at a time
constexpr int kFp8ScaleOff = 512, kFp8RopeOff = 528;
constexpr float kFp8Max = 448.f;

// One input: x [tokens, heads, D] with strides, its weights, and where it goes.
struct RopePart {
  const uint8_t* x;
  uint8_t* y;                  // [rows, D] contiguous
  const uint8_t* w;            // [n] or null
  const uint8_t* dy;           // backward: strided like x
  float* dw;                   // backward: partial sums [blocks][D]
  long long st, sh, dst, dsh;  // byte strides of x and dy
  uint32_t rows, H;
  int n;                       // normed channels
  int blocks;                  // workgroups
};

struct RopeParams {
  RopePart part[2];            // KV rows, queries
  const int32_t* pos;          // [T] or null (append: the cache positions)
  const float* table;          // [table_rows, R / 2, 2]
  int table_rows, D, R, T;
  int wf32;                    // weights are fp32 (else the rows' type)
  float eps, sign;             // sign of the rotation
  // append
  const int32_t* cu;           // [B + 1]
  const int32_t* used;         // [B]
  const int32_t* bt;
  uint8_t* cache;
  int B, bt_stride, bs, nblocks;
};

template <int CTRL>
__device__ __forceinline__ float dpp(float x) {
  return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), CTRL, 0xf, 0xf, true));
}
// over the eight lanes of a row: pairs, quads, then the other quad (half-row mirror)
__device__ __forceinline__ float sum8(float x) {
  x += dpp<0xB1>(x);
  x += dpp<0x4E>(x);
  return x + dpp<0x141>(x);
}
__device__ __forceinline__ float max8(float x) {
  x = fmaxf(x, dpp<0xB1>(x));
  x = fmaxf(x, dpp<0x4E>(x));
  return fmaxf(x, dpp<0x141>(x));
}

template <typename QT>
__device__ __forceinline__ void unpack8(const uint4& v, float (&f)[8]) {
  typedef QT v8 __attribute__((ext_vector_type(8)));
  const v8 a = __builtin_bit_cast(v8, v);
#pragma unroll
  for (int k = 0; k < 8; ++k) f[k] = (float)a[k];
}
template <typename QT>
__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
  return make_uint4(pack2<QT>(f[0], f[1]), pack2<QT>(f[2], f[3]), pack2<QT>(f[4], f[5]), pack2<QT>(f[6], f[7]));
}
// weights of channels 8 c .. 8 c + 7
template <typename QT>
__device__ __forceinline__ void weights8(const RopeParams& p, const uint8_t* w, int c, float (&f)[8]) {
  if (p.wf32) {
    const float4 a = reinterpret_cast<const float4*>(w)[2 * c], b = reinterpret_cast<const float4*>(w)[2 * c + 1];
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
  } else {
    unpack8<QT>(reinterpret_cast<const uint4*>(w)[c], f);
  }
}

// Token -> (sequence, place): the largest b with cu[b] <= t, one ballot per row and 64
// sequences. Every lane of the wave takes part; `t` is the token of the lane's row.
struct Place { int slot, b; bool padded; };
__device__ __forceinline__ Place place_of(const RopeParams& p, int t, int lane) {
  Place o{0, 0, true};
  int len = 0, start = 0;
  for (int c0 = 0; c0 < p.B; c0 += 64) {
    const int i = c0 + lane;
    int q0 = INT_MAX, q1 = 0, kv = 0;
    if (i < p.B) { q0 = p.cu[i]; q1 = p.cu[i + 1]; kv = p.used[i]; }
    int n = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int m = __popcll(__ballot(q0 <= __builtin_amdgcn_readlane(t, 8 * j)));
      n = (lane >> 3) == j ? m : n;
    }
    const int at = max(n - 1, 0);
    const int s = __shfl(q0, at), e = __shfl(q1, at), u = __shfl(kv, at);
    if (n > 0) { o.b = c0 + at; start = s; len = e - s; o.slot = u - len + (t - s); o.padded = false; }
    if (__ballot(n == 64) == 0) break;   // wave-uniform: no row's sequence lies further on
  }
  o.padded = o.padded || t < start || t - start >= len || o.slot < 0;
  return o;
}

// A lane's share of one row. LAST: D = 64 NI and R = 64, so the rotated
// channels are exactly the lanes' last chunks (the branch and its late loads go).
template <typename QT, int NI, bool LAST, bool HALF>
struct Row {
  int sub, nch, nn, rc0, hc;   // lane of eight; chunks: row's, normed, first rotated, half the rotated ones
  uint4 v[NI];

  __device__ Row(const RopeParams& p, int n, int lane)
      : sub(lane & 7), nch(LAST ? 8 * NI : p.D / 8), nn(n / 8), rc0(LAST ? 8 * (NI - 1) : (p.D - p.R) / 8),
        hc(LAST ? 4 : p.R / 16) {}
  __device__ __forceinline__ int chunk(int i) const { return 8 * i + sub; }
  __device__ __forceinline__ bool has(int i) const { return LAST || chunk(i) < nch; }
  // wave-uniform: chunks of iteration i are rotated
  __device__ __forceinline__ bool turns(int i) const { return LAST ? i == NI - 1 : 8 * i + 7 >= rc0 && 8 * i < nch; }
  __device__ __forceinline__ int partner(int c) const { return c - rc0 < hc ? c + hc : c - hc; }

  __device__ __forceinline__ static uint4 ld(const uint8_t* x, int c) {
    return gld16(reinterpret_cast<uint64_t>(x) + 16 * c);
  }
  // every lane loads (a clamped chunk)
  __device__ __forceinline__ void load(const uint8_t* x) {
#pragma unroll
    for (int i = 0; i < NI; ++i) v[i] = ld(x, LAST ? chunk(i) : min(chunk(i), nch - 1));
  }
  // y (channels of chunk c) rotated by the position's angles; `other` holds the
  // partner chunk's channels (HALF)
  __device__ __forceinline__ void rotate(const RopeParams& p, const float* cs, int c, const float (&y)[8],
                                         const float (&other)[8], float sign, float (&o)[8]) const {
    if constexpr (HALF) {
      const int j = c - rc0;
      const bool first = j < hc;
      const float4* e = reinterpret_cast<const float4*>(cs + 16 * (first ? j : j - hc));
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float4 a = e[k];
        // first half: a c - b s; second: b c + a s, `other` being the pair's other channel
        const float s0 = first ? -sign * a.y : sign * a.y, s1 = first ? -sign * a.w : sign * a.w;
        o[2 * k] = fmaf(y[2 * k], a.x, other[2 * k] * s0);
        o[2 * k + 1] = fmaf(y[2 * k + 1], a.z, other[2 * k + 1] * s1);
      }
    } else {
      const float4* e = reinterpret_cast<const float4*>(cs + 8 * (c - rc0));
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const float4 a = e[k];
        o[4 * k] = fmaf(y[4 * k], a.x, -sign * a.y * y[4 * k + 1]);
        o[4 * k + 1] = fmaf(y[4 * k + 1], a.x, sign * a.y * y[4 * k]);
        o[4 * k + 2] = fmaf(y[4 * k + 2], a.z, -sign * a.w * y[4 * k + 3]);
        o[4 * k + 3] = fmaf(y[4 * k + 3], a.z, sign * a.w * y[4 * k + 2]);
      }
    }
  }
};

// Destinations: rows of a contiguous tensor, rows of the paged cache in their own
// type, 656-byte fp8 rows of the paged cache.
enum { kToRows = 0, kToCache = 1, kToFp8 = 2 };

// latent channels of iterations 2 g and 2 g + 1 are one 128-channel scale group
__device__ __forceinline__ void put_fp8_group(uint8_t* dst, int g, int sub, const float (&a)[8], const float (&b)[8],
                                              bool write) {
  float amax = 0.f;
#pragma unroll
  for (int k = 0; k < 8; ++k) amax = fmaxf(amax, fmaxf(fabsf(a[k]), fabsf(b[k])));
  amax = max8(amax);
  const float scale = amax > 0.f ? amax / kFp8Max : 1.f;
  // (at most the largest float: zeros beside channels below 1e-36 stay zeros)
  const float inv = amax > 0.f ? fminf(kFp8Max / amax, 3.402823466e38f) : 1.f;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const float (&x)[8] = h ? b : a;
    uint32_t q[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      auto cl = [&](float f) { return __builtin_amdgcn_fmed3f(f * inv, -kFp8Max, kFp8Max); };
      int t = __builtin_amdgcn_cvt_pk_fp8_f32(cl(x[4 * j]), cl(x[4 * j + 1]), 0, false);
      t = __builtin_amdgcn_cvt_pk_fp8_f32(cl(x[4 * j + 2]), cl(x[4 * j + 3]), t, true);
      q[j] = (uint32_t)t;
    }
    if (write) *reinterpret_cast<uint2*>(dst + 128 * g + 64 * h + 8 * sub) = make_uint2(q[0], q[1]);
  }
  if (write && sub == 0) *reinterpret_cast<float*>(dst + kFp8ScaleOff + 4 * g) = scale;
}

// Rows of one part: workgroup `blk` of its grid.
template <typename QT, int NI, bool LAST, bool HALF, int DST, bool APPEND>
__device__ __forceinline__ void rope_rows(const RopeParams& p, const RopePart& a, uint32_t blk, int tid) {
  const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t r0 = blk * kRopeRows + wave * 8;   // the wave's first row
  if (r0 >= a.rows) return;
  const uint32_t row = r0 + (lane >> 3);
  const bool live = row < a.rows;
  // its token and head: one division for the wave, the rows after it step on
  uint32_t t = r0 / a.H, h = r0 - t * a.H + (lane >> 3);
  if (a.H >= 8) {
    if (h >= a.H) { h -= a.H; ++t; }
  } else {
    const uint32_t k = h / a.H;
    t += k;
    h -= k * a.H;
  }
  if (!live) { t = r0 / a.H; h = r0 - t * a.H; }   // a row to load; nothing of it is stored

  Row<QT, NI, LAST, HALF> r(p, a.n, lane);
  const uint8_t* x = a.x + (long long)t * a.st + (long long)h * a.sh;
  r.load(x);

  Place at{0, 0, false};
  if constexpr (APPEND) at = place_of(p, (int)t, lane);
  int pos = 0;
  if (p.R) pos = APPEND && !p.pos ? at.slot : p.pos[t];
  const bool in = (!p.R || (pos >= 0 && pos < p.table_rows)) && !at.padded;
  const float* cs = p.table + (size_t)(in ? pos : 0) * p.R;
  uint8_t* dst = nullptr;
  if constexpr (DST == kToRows) {
    dst = a.y + (size_t)row * p.D * 2;
  } else {
    const int blkno = in ? at.slot / p.bs : 0;
    const bool okt = in && blkno < p.bt_stride;
    const int phys = p.bt[okt ? (size_t)at.b * p.bt_stride + blkno : 0];
    if (live && okt && phys >= 0 && phys < p.nblocks)
      dst = p.cache + ((size_t)phys * p.bs + (at.slot - blkno * p.bs)) * (DST == kToFp8 ? kRow656 : p.D * 2);
  }
  const bool write = DST == kToRows ? live : dst != nullptr;

  // the norm
  float rinv = 1.f;
  if (a.n) {
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      float f[8], s = 0.f;
      unpack8<QT>(r.v[i], f);
#pragma unroll
      for (int k = 0; k < 8; ++k) s = fmaf(f[k], f[k], s);
      ss += r.chunk(i) < r.nn ? s : 0.f;
    }
    rinv = rsqrtf(sum8(ss) / (float)a.n + p.eps);
  }
  auto normed = [&](const uint4& v, int c, float (&f)[8]) {
    unpack8<QT>(v, f);
    if (c < r.nn) {
      float w[8];
      if (a.w) weights8<QT>(p, a.w, c, w);
#pragma unroll
      for (int k = 0; k < 8; ++k) f[k] *= a.w ? rinv * w[k] : rinv;
    }
  };
  float keep[8];   // fp8: the first chunk of a scale group's two
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int c = r.chunk(i);
    float f[8];
    normed(r.v[i], c, f);
    if (p.R && r.turns(i)) {
      const bool turn = LAST || (c >= r.rc0 && c < r.nch);
      const int ct = turn ? c : r.rc0;
      float other[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, o[8];
      if constexpr (HALF) {
        const int pc = r.partner(ct);
        normed(r.ld(x, pc), pc, other);
      }
      r.rotate(p, cs, ct, f, other, p.sign, o);
#pragma unroll
      for (int k = 0; k < 8; ++k) f[k] = turn ? o[k] : f[k];
    }
    if constexpr (DST == kToFp8) {
      if (i < 8) {
        if (i & 1) put_fp8_group(dst, i >> 1, r.sub, keep, f, write);
        else {
#pragma unroll
          for (int k = 0; k < 8; ++k) keep[k] = f[k];
        }
      } else if (write) {
        *reinterpret_cast<uint4*>(dst + kFp8RopeOff + 16 * r.sub) = pack8<__bf16>(f);
      }
    } else if (write && r.has(i)) {
      uint4 o = pack8<QT>(f);
      if (DST == kToRows && !in) o = make_uint4(0, 0, 0, 0);   // a padded row
      *reinterpret_cast<uint4*>(dst + 16 * c) = o;
    }
  }
}

// Workgroups [0, part[0].blocks) take the KV rows (the longer chain of loads
// starts first), the others the queries.
template <typename QT, int NI, bool LAST, bool HALF, int DST>
__global__ void __launch_bounds__(kRopeThreads) sas_rope_kernel(const RopeParams p) {
  constexpr bool kAppend = DST != kToRows;
  const uint32_t b = blockIdx.x, nkv = (uint32_t)p.part[0].blocks;
  if (b < nkv) rope_rows<QT, NI, LAST, HALF, DST, kAppend>(p, p.part[0], b, threadIdx.x);
  else rope_rows<QT, NI, LAST, HALF, kToRows, kAppend>(p, p.part[1], b - nkv, threadIdx.x);
}

// ---------------------------------------------------------------------------
// backward
// ---------------------------------------------------------------------------

// A workgroup walks its part's rows; with weights every lane sums its channels'
// weight gradients in registers, the workgroup adds them up through LDS once
// at its end and leaves one partial row: no atomics, the same order every time.
template <typename QT, int NI, bool LAST, bool HALF, bool W>
__device__ __forceinline__ void rope_grad_rows(const RopeParams& p, const RopePart& a, uint32_t blk, int tid,
                                               float* lds) {
  const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  float dw[W ? NI : 1][8];
#pragma unroll
  for (int i = 0; i < (W ? NI : 1); ++i)
#pragma unroll
    for (int k = 0; k < 8; ++k) dw[i][k] = 0.f;
  Row<QT, NI, LAST, HALF> r(p, a.n, lane), g(p, a.n, lane);
  for (uint32_t r0 = blk * kRopeRows + wave * 8; r0 < a.rows; r0 += (uint32_t)a.blocks * kRopeRows) {
    const uint32_t row = r0 + (lane >> 3);
    const bool live = row < a.rows;
    uint32_t t = r0 / a.H, h = r0 - t * a.H + (lane >> 3);
    if (a.H >= 8) {
      if (h >= a.H) { h -= a.H; ++t; }
    } else {
      const uint32_t k = h / a.H;
      t += k;
      h -= k * a.H;
    }
    if (!live) { t = r0 / a.H; h = r0 - t * a.H; }
    r.load(a.x + (long long)t * a.st + (long long)h * a.sh);
    const uint8_t* dy = a.dy + (long long)t * a.dst + (long long)h * a.dsh;
    g.load(dy);
    const int pos = p.R ? p.pos[t] : 0;
    const bool in = live && (!p.R || (pos >= 0 && pos < p.table_rows));
    const float* cs = p.table + (size_t)(in ? pos : 0) * p.R;
    // dy rotated back, in place (HALF: partners come from memory again, which is still dy)
    float ut[LAST ? 1 : NI][8];   // rotated chunks, in 32 bits
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      if (!(p.R && r.turns(i))) continue;
      const int c = r.chunk(i);
      const bool turn = LAST || (c >= r.rc0 && c < r.nch);
      const int ct = turn ? c : r.rc0;
      float f[8], other[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, o[8];
      unpack8<QT>(g.v[i], f);
      if constexpr (HALF) unpack8<QT>(r.ld(dy, r.partner(ct)), other);
      r.rotate(p, cs, ct, f, other, -p.sign, o);
#pragma unroll
      for (int k = 0; k < 8; ++k) ut[LAST ? 0 : i][k] = turn ? o[k] : f[k];
    }
    auto grad = [&](int i, float (&u)[8]) {
      if (p.R && r.turns(i)) {
#pragma unroll
        for (int k = 0; k < 8; ++k) u[k] = ut[LAST ? 0 : i][k];
      } else {
        unpack8<QT>(g.v[i], u);
      }
    };
    float rinv = 1.f, m = 0.f;
    if (a.n) {
      float ss = 0.f, sg = 0.f;
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int c = r.chunk(i);
        if (!(c < r.nn)) continue;
        float f[8], u[8], w[8];
        unpack8<QT>(r.v[i], f);
        grad(i, u);
        if (a.w) weights8<QT>(p, a.w, c, w);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          ss = fmaf(f[k], f[k], ss);
          sg = fmaf(a.w ? u[k] * w[k] : u[k], f[k], sg);
        }
      }
      rinv = rsqrtf(sum8(ss) / (float)a.n + p.eps);
      m = sum8(sg) / (float)a.n * rinv * rinv;
    }
    uint8_t* dst = a.y + (size_t)row * p.D * 2;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int c = r.chunk(i);
      float u[8], o[8];
      grad(i, u);
      if (c < r.nn) {
        float f[8], w[8];
        unpack8<QT>(r.v[i], f);
        if (a.w) weights8<QT>(p, a.w, c, w);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          o[k] = rinv * ((a.w ? u[k] * w[k] : u[k]) - f[k] * m);
          if constexpr (W) dw[i][k] += in ? u[k] * (f[k] * rinv) : 0.f;
        }
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) o[k] = u[k];
      }
      if (live && r.has(i)) {
        uint4 v = pack8<QT>(o);
        if (!in) v = make_uint4(0, 0, 0, 0);
        *reinterpret_cast<uint4*>(dst + 16 * c) = v;
      }
    }
  }
  if constexpr (W) {
    if (!a.dw) return;   // workgroup-uniform
    // the wave's eight rows, then its four waves
#pragma unroll
    for (int i = 0; i < NI; ++i) {
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        float s = dw[i][k];
        s += dpp<0x128>(s);   // the other row of the 16 lanes
        s = rows_sum(s);
        if (lane < 8) lds[wave * (NI * 64) + r.chunk(i) * 8 + k] = s;
      }
    }
    __syncthreads();
    for (int j = tid; j < a.n; j += kRopeThreads) {
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < kRopeThreads / 64; ++w) s += lds[w * (NI * 64) + j];
      a.dw[(size_t)blk * p.D + j] = s;
    }
  }
}

template <typename QT, int NI, bool LAST, bool HALF, bool W>
__global__ void __launch_bounds__(kRopeThreads) sas_rope_grad_kernel(const RopeParams p) {
  __shared__ float lds[W ? (kRopeThreads / 64) * NI * 64 : 1];
  const uint32_t b = blockIdx.x, nkv = (uint32_t)p.part[0].blocks;
  if (b < nkv) rope_grad_rows<QT, NI, LAST, HALF, W>(p, p.part[0], b, threadIdx.x, lds);
  else rope_grad_rows<QT, NI, LAST, HALF, W>(p, p.part[1], b - nkv, threadIdx.x, lds);
}

// Weight gradients from the workgroups' partial rows: 16 channels a workgroup, 16
// threads a channel, in a fixed order.
struct RopeSum { const float* part[2]; float* dw[2]; int rows[2], n[2], D; };
__global__ void __launch_bounds__(256) sas_rope_dw_kernel(const RopeSum s) {
  __shared__ float lds[16][17];
  const int w = blockIdx.y, c = threadIdx.x & 15, k = threadIdx.x >> 4, j = blockIdx.x * 16 + c;
  if (!s.dw[w]) return;
  float v = 0.f;
  if (j < s.n[w]) {
#pragma unroll 8
    for (int i = k; i < s.rows[w]; i += 16) v += s.part[w][(size_t)i * s.D + j];
  }
  lds[k][c] = v;
  __syncthreads();
  if (k == 0 && j < s.n[w]) {
    v = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) v += lds[i][c];
    s.dw[w][j] = v;
  }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// dims, types and pointers of a call; `grad` checks nothing of the outputs
int check_rope(const SasNormRopeArgs* a, const char* what) {
  if (a->T < 0 || a->H < 0 || a->D < 8 || a->D % 8 || a->D > 1024)
    return set_error(SAS_EINVAL, "%s: T and H must not be negative, D a multiple of 8 in [8, 1024]", what);
  if (a->dtype != SAS_DT_BF16 && a->dtype != SAS_DT_FP16) return set_error(SAS_EINVAL, "%s: dtype must be bf16 or fp16", what);
  if (a->weight_dtype != SAS_DT_FP32 && a->weight_dtype != a->dtype)
    return set_error(SAS_EINVAL, "%s: weights must be fp32 or of the rows' dtype", what);
  if (a->flags & ~(SAS_ROPE_HALF | SAS_ROPE_INVERSE)) return set_error(SAS_EINVAL, "%s: unknown flags 0x%x", what, a->flags);
  const int unit = a->flags & SAS_ROPE_HALF ? 16 : 8;
  if (a->rope_dim < 0 || a->rope_dim > a->D || a->rope_dim % unit)
    return set_error(SAS_EINVAL, "%s: rope_dim must be a multiple of %d in [0, D] (got %d)", what, unit, a->rope_dim);
  if (a->q_norm_dim < 0 || a->q_norm_dim > a->D || a->q_norm_dim % 8 || a->kv_norm_dim < 0 || a->kv_norm_dim > a->D ||
      a->kv_norm_dim % 8)
    return set_error(SAS_EINVAL, "%s: norm dims must be multiples of 8 in [0, D]", what);
  if (!(a->eps >= 0.f)) return set_error(SAS_EINVAL, "%s: eps must not be negative", what);
  if ((double)a->T * (double)std::max<int64_t>(a->H, 1) > 2147483000.0)
    return set_error(SAS_EINVAL, "%s: more than 2^31 rows", what);
  if (a->T == 0) return SAS_OK;
  if ((a->H > 0) != (a->q != nullptr)) return set_error(SAS_EINVAL, "%s: q and H go together", what);
  if (!a->q && !a->kv) return set_error(SAS_EINVAL, "%s: null device pointer", what);
  if (a->rope_dim && (!a->table || a->table_rows < 1 || a->table_rows > INT32_MAX))
    return set_error(SAS_EINVAL, "%s: a rotation needs its table", what);
  const int64_t st[3] = {a->q ? a->q_stride_t : 0, a->q ? a->q_stride_h : 0, a->kv ? a->kv_stride_t : 0};
  for (int64_t s : st)
    if (s % 8) return set_error(SAS_EINVAL, "%s: strides must be multiples of 8 elements", what);
  if (!aligned16(a->q) || !aligned16(a->kv) || !aligned16(a->q_weight) || !aligned16(a->kv_weight) || !aligned16(a->table) ||
      !aligned16(a->q_out) || !aligned16(a->kv_out))
    return set_error(SAS_EINVAL, "%s: rows, weights and table must be 16-byte aligned", what);
  return SAS_OK;
}

void fill_rope(const SasNormRopeArgs* a, RopeParams* p) {
  p->pos = a->positions;
  p->table = a->table;
  p->table_rows = (int)a->table_rows;
  p->D = (int)a->D; p->R = a->rope_dim; p->T = (int)a->T;
  p->wf32 = a->weight_dtype == SAS_DT_FP32;
  p->eps = a->eps;
  p->sign = a->flags & SAS_ROPE_INVERSE ? -1.f : 1.f;
  RopePart& kv = p->part[0];
  RopePart& q = p->part[1];
  kv.H = 1;
  q.H = (uint32_t)std::max<int64_t>(a->H, 1);
  kv.n = a->kv_norm_dim;
  q.n = a->q_norm_dim;
  if (a->kv) {
    kv.x = (const uint8_t*)a->kv; kv.y = (uint8_t*)a->kv_out; kv.w = (const uint8_t*)a->kv_weight;
    kv.st = a->kv_stride_t * 2; kv.rows = (uint32_t)a->T;
  }
  if (a->q) {
    q.x = (const uint8_t*)a->q; q.y = (uint8_t*)a->q_out; q.w = (const uint8_t*)a->q_weight;
    q.st = a->q_stride_t * 2; q.sh = a->q_stride_h * 2; q.rows = (uint32_t)(a->T * a->H);
  }
  for (RopePart& x : p->part) x.blocks = (int)((x.rows + kRopeRows - 1) / kRopeRows);
}

// The kernel for a row width: 128, 512 or 576 channels with 64 rotated ones (or none) in
// their own builds, any other in one of up to 16 chunks a lane.
template <typename F>
int by_width(const SasNormRopeArgs* a, F&& f) {
  const bool last = a->rope_dim == 64 || a->rope_dim == 0;
  auto half = [&](auto ni, auto l) {
    return a->flags & SAS_ROPE_HALF ? f(ni, l, std::true_type{}) : f(ni, l, std::false_type{});
  };
  if (last && a->D == 576) return half(std::integral_constant<int, 9>{}, std::true_type{});
  if (last && a->D == 512) return half(std::integral_constant<int, 8>{}, std::true_type{});
  if (last && a->D == 128) return half(std::integral_constant<int, 2>{}, std::true_type{});
  return half(std::integral_constant<int, 16>{}, std::false_type{});
}

int launched(const char* what) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? SAS_OK : set_error(SAS_ELAUNCH, "%s launch: %s", what, hipGetErrorString(e));
}

template <int DST>
int launch_rope(const SasNormRopeArgs* a, const RopeParams& p, hipStream_t st, const char* what) {
  const dim3 grid((unsigned)(p.part[0].blocks + p.part[1].blocks));
  return by_width(a, [&](auto ni, auto last, auto half) {
    constexpr int NI = decltype(ni)::value;
    constexpr bool L = decltype(last)::value, HF = decltype(half)::value;
    if (a->dtype == SAS_DT_BF16)
      hipLaunchKernelGGL((sas_rope_kernel<__bf16, NI, L, HF, DST>), grid, dim3(kRopeThreads), 0, st, p);
    else
      hipLaunchKernelGGL((sas_rope_kernel<_Float16, NI, L, HF, DST>), grid, dim3(kRopeThreads), 0, st, p);
    return launched(what);
  });
}

// Workgroups of the backward's two parts: two a CU (a build holds 2 to 3 waves a
// SIMD), shared out by rows, none without rows of its own.
void grad_blocks(RopeParams* p) {
  const double all = (double)p->part[0].rows + p->part[1].rows;
  const long long most = 2LL * device_cus();
  for (RopePart& x : p->part) {
    const long long full = ((long long)x.rows + kRopeRows - 1) / kRopeRows;
    const long long share = std::max<long long>(1, (long long)(most * (double)x.rows / std::max(all, 1.0) + 0.5));
    x.blocks = (int)std::min(full, share);
  }
}

size_t grad_workspace(const SasNormRopeBwdArgs* a, const RopeParams& p) {
  size_t rows = 0;
  if (a->dkv_weight && p.part[0].n) rows += p.part[0].blocks;
  if (a->dq_weight && p.part[1].n) rows += p.part[1].blocks;
  return rows * (size_t)p.D * sizeof(float);
}

int check_grad(const SasNormRopeBwdArgs* a, RopeParams* p) {
  const SasNormRopeArgs* f = &a->fwd;
  const int rc = check_rope(f, "norm_rope_bwd");
  if (rc) return rc;
  if ((a->dq_weight && !f->q_weight) || (a->dkv_weight && !f->kv_weight))
    return set_error(SAS_EINVAL, "norm_rope_bwd: a weight gradient needs its weight");
  fill_rope(f, p);
  grad_blocks(p);
  return SAS_OK;
}

}  // namespace
}  // namespace sas

extern "C" int sas_norm_rope_v1(const SasNormRopeArgs* a, void* stream) {
  using namespace sas;
  clear_error();
  if (!a) return set_error(SAS_EINVAL, "norm_rope: null args");
  const int rc = check_rope(a, "norm_rope");
  if (rc || a->T == 0) return rc;
  if ((a->q && !a->q_out) || (a->kv && !a->kv_out) || (a->rope_dim && !a->positions))
    return set_error(SAS_EINVAL, "norm_rope: null device pointer");
  RopeParams p{};
  fill_rope(a, &p);
  return launch_rope<kToRows>(a, p, (hipStream_t)stream, "norm_rope");
}

extern "C" int sas_norm_rope_bwd_plan(const SasNormRopeBwdArgs* a, size_t* workspace_bytes) {
  using namespace sas;
  clear_error();
  if (!a) return set_error(SAS_EINVAL, "norm_rope_bwd: null args");
  RopeParams p{};
  const int rc = check_grad(a, &p);
  if (rc) return rc;
  if (workspace_bytes) *workspace_bytes = grad_workspace(a, p);
  return SAS_OK;
}

extern "C" int sas_norm_rope_bwd_v1(const SasNormRopeBwdArgs* a, void* stream) {
  using namespace sas;
  clear_error();
  if (!a) return set_error(SAS_EINVAL, "norm_rope_bwd: null args");
  RopeParams p{};
  const int rc = check_grad(a, &p);
  if (rc) return rc;
  const SasNormRopeArgs* f = &a->fwd;
  hipStream_t st = (hipStream_t)stream;
  RopeSum s{};
  s.D = (int)f->D;
  float* dw[2] = {p.part[0].n ? a->dkv_weight : nullptr, p.part[1].n ? a->dq_weight : nullptr};
  const size_t need = grad_workspace(a, p);
  if (f->T > 0) {
    if ((f->q && (!a->dq || !a->dq_out)) || (f->kv && (!a->dkv || !a->dkv_out)) || (f->rope_dim && !f->positions))
      return set_error(SAS_EINVAL, "norm_rope_bwd: null device pointer");
    if ((f->q && (a->dq_out_stride_t % 8 || a->dq_out_stride_h % 8)) || (f->kv && a->dkv_out_stride_t % 8))
      return set_error(SAS_EINVAL, "norm_rope_bwd: strides must be multiples of 8 elements");
    if (!aligned16(a->dq) || !aligned16(a->dq_out) || !aligned16(a->dkv) || !aligned16(a->dkv_out))
      return set_error(SAS_EINVAL, "norm_rope_bwd: rows must be 16-byte aligned");
    if (need && (!a->workspace || a->workspace_bytes < need))
      return set_error(SAS_ENOWS, "workspace of %zu bytes required", need);
  }
  p.part[0].dy = (const uint8_t*)a->dkv_out; p.part[0].y = (uint8_t*)a->dkv;
  p.part[0].dst = a->dkv_out_stride_t * 2;
  p.part[1].dy = (const uint8_t*)a->dq_out; p.part[1].y = (uint8_t*)a->dq;
  p.part[1].dst = a->dq_out_stride_t * 2; p.part[1].dsh = a->dq_out_stride_h * 2;
  float* ws = (float*)a->workspace;
  for (int k = 0; k < 2; ++k) {
    s.n[k] = p.part[k].n;
    s.dw[k] = dw[k];
    if (!dw[k]) continue;
    s.rows[k] = p.part[k].blocks;   // none: zeros
    s.part[k] = p.part[k].dw = ws;
    ws += (size_t)p.part[k].blocks * p.D;
  }
  if (f->T > 0) {
    const dim3 grid((unsigned)(p.part[0].blocks + p.part[1].blocks));
    const bool w = dw[0] || dw[1];
    const int e = by_width(f, [&](auto ni, auto last, auto half) {
      constexpr int NI = decltype(ni)::value;
      constexpr bool L = decltype(last)::value, HF = decltype(half)::value;
      auto go = [&](auto kern) { hipLaunchKernelGGL(kern, grid, dim3(kRopeThreads), 0, st, p); };
      if (f->dtype == SAS_DT_BF16) {
        if (w) go(sas_rope_grad_kernel<__bf16, NI, L, HF, true>);
        else go(sas_rope_grad_kernel<__bf16, NI, L, HF, false>);
      } else {
        if (w) go(sas_rope_grad_kernel<_Float16, NI, L, HF, true>);
        else go(sas_rope_grad_kernel<_Float16, NI, L, HF, false>);
      }
      return launched("norm_rope_bwd");
    });
    if (e) return e;
  }
  if (dw[0] || dw[1]) {
    hipLaunchKernelGGL(sas_rope_dw_kernel, dim3((unsigned)((f->D + 15) / 16), 2), dim3(256), 0, st, s);
    return launched("norm_rope_bwd");
  }
  return SAS_OK;
}

extern "C" int sas_cache_append_v1(const SasCacheAppendArgs* a, void* stream) {
  using namespace sas;
  clear_error();
  if (!a) return set_error(SAS_EINVAL, "cache_append: null args");
  const SasNormRopeArgs* r = &a->rope;
  if (a->B < 1 || a->bt_stride < 1 || a->block_size < 1 || a->num_blocks < 1)
    return set_error(SAS_EINVAL, "cache_append: bad sizes");
  int rc = check_rope(r, "cache_append");
  if (rc) return rc;
  const bool fp8 = a->cache_dtype == SAS_DT_FP8_E4M3_ROW656;
  if (fp8 && (r->dtype != SAS_DT_BF16 || r->D != 576))
    return set_error(SAS_EINVAL, "cache_append: fp8 rows need bf16 kv with D = 576");
  if (!fp8 && a->cache_dtype != r->dtype)
    return set_error(SAS_EINVAL, "cache_append: cache dtype must be the kv dtype or fp8 rows");
  if (a->B > INT32_MAX - 1 || a->bt_stride > INT32_MAX || (double)a->num_blocks * a->block_size > 2147483000.0)
    return set_error(SAS_EINVAL, "cache_append: sizes beyond 32-bit indexing");
  if (r->T == 0) return SAS_OK;
  if (!r->kv || !a->cu_seqlens_q || !a->act_kv || !a->block_table || !a->cache || (r->q && !r->q_out))
    return set_error(SAS_EINVAL, "cache_append: null device pointer");
  if (!aligned16(a->cache)) return set_error(SAS_EINVAL, "cache_append: cache must be 16-byte aligned");
  RopeParams p{};
  fill_rope(r, &p);
  p.cu = a->cu_seqlens_q; p.used = a->act_kv; p.bt = a->block_table; p.cache = (uint8_t*)a->cache;
  p.B = (int)a->B; p.bt_stride = (int)a->bt_stride; p.bs = (int)a->block_size; p.nblocks = (int)a->num_blocks;
  hipStream_t st = (hipStream_t)stream;
  if (!fp8) return launch_rope<kToCache>(r, p, st, "cache_append");
  const dim3 grid((unsigned)(p.part[0].blocks + p.part[1].blocks)), block(kRopeThreads);
  auto go = [&](auto kern) { hipLaunchKernelGGL(kern, grid, block, 0, st, p); };
  const bool half = r->flags & SAS_ROPE_HALF;
  if (r->rope_dim == 64 || r->rope_dim == 0) {
    if (half) go(sas_rope_kernel<__bf16, 9, true, true, kToFp8>);
    else go(sas_rope_kernel<__bf16, 9, true, false, kToFp8>);
  } else {
    if (half) go(sas_rope_kernel<__bf16, 9, false, true, kToFp8>);
    else go(sas_rope_kernel<__bf16, 9, false, false, kToFp8>);
  }
  return launched("cache_append");
}
