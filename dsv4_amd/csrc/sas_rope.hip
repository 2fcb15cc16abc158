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
// reads), 2 D bytes each way, against some 5 (15) VALU operations a channel. Sixteen
// lanes share a row and a wave takes four: channel chunk (8 channels, 16
// bytes) 16 i + l of its row belongs to lane l of the sixteen, so a load
// instruction covers whole 256-byte pieces of four rows, all of a lane's loads are
// in flight at once, and a row's sums are four DPP steps inside the sixteen lanes.
// Nothing passes through LDS but the weights and the backward's sums of theirs.

#include "sas_kern.h"

namespace sas {
namespace {

constexpr int kLanes = 16;                                            // of a row
constexpr int kRopeThreads = 256, kRopeRows = kRopeThreads / kLanes;   // rows a workgroup takes at a time
constexpr int kWaveRows = 64 / kLanes;
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
  const int32_t* pos;          // [T]; any readable address where there are none
  int has_pos;                 // 0: none (append: the cache positions)
  const float* table;          // [table_rows, R / 2, 2]
  int table_rows, D, R;
  int wf32;                    // weights are fp32 (else the rows' type)
  float eps, sign;             // sign of the rotation
  int nt_load, nt_store;       // rows are read / written non-temporally
  // append
  const int32_t* cu;           // [B + 1]
  const int32_t* used;         // [B]
  const int32_t* bt;
  uint8_t* cache;
  int B, bt_stride, bs, nblocks;
  int bs_shift;                // log2 of bs, or -1
};

template <int CTRL>
__device__ __forceinline__ float dpp(float x) {
  return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), CTRL, 0xf, 0xf, true));
}
// over a row's sixteen lanes: pairs, quads, eights (mirrored halves), all (mirrored)
__device__ __forceinline__ float sum16(float x) {
  x += dpp<0xB1>(x);
  x += dpp<0x4E>(x);
  x += dpp<0x141>(x);
  return x + dpp<0x140>(x);
}
// of magnitudes, NaN above all of them: by their bits
__device__ __forceinline__ float max16(float x) {
  uint32_t u = __float_as_uint(x);
  u = max(u, __float_as_uint(dpp<0xB1>(__uint_as_float(u))));
  u = max(u, __float_as_uint(dpp<0x4E>(__uint_as_float(u))));
  u = max(u, __float_as_uint(dpp<0x141>(__uint_as_float(u))));
  return __uint_as_float(max(u, __float_as_uint(dpp<0x140>(__uint_as_float(u)))));
}

// v as a value of its own: what was computed from it before is not kept for later
// (and what it is computed from is not sunk into a branch that alone reads it)
__device__ __forceinline__ void opaque(uint4& v) { asm volatile("" : "+v"(v.x), "+v"(v.y), "+v"(v.z), "+v"(v.w)); }
__device__ __forceinline__ void opaque(float4& v) { asm volatile("" : "+v"(v.x), "+v"(v.y), "+v"(v.z), "+v"(v.w)); }
__device__ __forceinline__ void opaque(float& v) { asm volatile("" : "+v"(v)); }

// 16 bytes of a row, past the caches with NT
template <bool NT>
__device__ __forceinline__ uint4 ld16(uint64_t a) {
  const SAS_GLOBAL u32x4g* p = reinterpret_cast<const SAS_GLOBAL u32x4g*>(a);
  return __builtin_bit_cast(uint4, NT ? __builtin_nontemporal_load(p) : *p);
}
// One of two branches that differ in nothing but NT: the compiler would merge
// them and drop it.
template <typename F, typename G>
__device__ __forceinline__ void either(int nt, F&& yes, G&& no) {
  if (nt) {
    asm volatile("; nt" ::: "memory");
    yes();
    asm volatile("; nt end" ::: "memory");
  } else {
    asm volatile("; cached" ::: "memory");
    no();
    asm volatile("; cached end" ::: "memory");
  }
}
__device__ __forceinline__ void st16(uint8_t* p, const uint4& v, int nt) {
  u32x4g* d = reinterpret_cast<u32x4g*>(p);
  const u32x4g w = __builtin_bit_cast(u32x4g, v);
  either(nt, [&] { __builtin_nontemporal_store(w, d); }, [&] { *d = w; });
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
// The part's weights as fp32 in LDS, ones past them and where there are none: a
// workgroup's rows share them, in global memory each wave would fetch its chunks'
// anew, in two types. `get` issues the loads (whole dwords, whatever the type: a load
// under a branch waits for itself there), `put` writes them behind the caller's own.
template <typename QT, int NI>
struct Weights {
  static constexpr int kAll = NI * kLanes * 8, N = (kAll + kRopeThreads - 1) / kRopeThreads;
  uint32_t w[N];
  __device__ __forceinline__ void get(const RopeParams& p, const RopePart& a, int tid) {
    const uint64_t base = reinterpret_cast<uint64_t>(a.w);
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int j = min(tid + k * kRopeThreads, max(a.n, 1) - 1);
      w[k] = *reinterpret_cast<const SAS_GLOBAL uint32_t*>(base + (p.wf32 ? 4u * (uint32_t)j : 2u * (uint32_t)(j & ~1)));
    }
  }
  __device__ __forceinline__ void put(const RopeParams& p, const RopePart& a, float* lds, int tid) {
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int j = tid + k * kRopeThreads;
      if (a.w) asm volatile("" : "+v"(w[k]));
      const uint16_t h = (uint16_t)(j & 1 ? w[k] >> 16 : w[k]);
      const float f = p.wf32 ? __uint_as_float(w[k]) : (float)__builtin_bit_cast(QT, h);
      if (kAll % kRopeThreads == 0 || j < kAll) lds[j] = a.w && j < a.n ? f : 1.f;
    }
    asm volatile("" ::: "memory");
    lds_barrier();
    asm volatile("" ::: "memory");
  }
};
// weights of channels 8 c .. 8 c + 7
__device__ __forceinline__ void weights8(uint32_t lds, int c, float (&f)[8]) {
  const LDS_AS f32x4* w = reinterpret_cast<const LDS_AS f32x4*>((size_t)(lds + 32 * c));
  const f32x4 a = w[0], b = w[1];
#pragma unroll
  for (int k = 0; k < 4; ++k) { f[k] = a[k]; f[4 + k] = b[k]; }
}

// Token -> (sequence, place): the largest b with cu[b] <= t, one ballot per row and 64
// sequences. Every lane of the wave takes part; `t` is the token of the lane's row.
// `seq` holds the lane's own sequence of the first 64, loaded ahead of the row.
struct Seq { int q0, q1, kv; };
__device__ __forceinline__ Seq seq_of(const RopeParams& p, int i) {
  const int j = min(i, p.B - 1);
  const Seq s{p.cu[j], p.cu[j + 1], p.used[j]};
  return {i < p.B ? s.q0 : INT_MAX, s.q1, s.kv};
}
struct Place { int slot, b; bool padded; };
__device__ __forceinline__ Place place_of(const RopeParams& p, Seq seq, int t, int lane) {
  Place o{0, 0, true};
  int len = 0, start = 0;
  auto among = [&](const Seq& s, int c0) {   // whether a row's sequence may lie past these 64
    int n = 0;
#pragma unroll
    for (int j = 0; j < kWaveRows; ++j) {
      const int m = __popcll(__ballot(s.q0 <= __builtin_amdgcn_readlane(t, kLanes * j)));
      n = lane / kLanes == j ? m : n;
    }
    const int at = max(n - 1, 0);
    const int q0 = __shfl(s.q0, at), q1 = __shfl(s.q1, at), kv = __shfl(s.kv, at);
    if (n > 0) { o.b = c0 + at; start = q0; len = q1 - q0; o.slot = kv - len + (t - q0); o.padded = false; }
    return __ballot(n == 64) != 0;
  };
  // (the first step apart: at the head of a loop the wait for `seq` would be for
  // every load in flight)
  bool more = among(seq, 0);
  for (int c0 = 64; more && c0 < p.B; c0 += 64) more = among(seq_of(p, c0 + lane), c0);
  o.padded = o.padded || t < start || t - start >= len || o.slot < 0;
  return o;
}

// Token and head of the lane's row, the wave's first row being r0: one division for
// the wave, the rows after it step on. A lane without a row takes r0's.
struct Head { uint32_t t, h; };
__device__ __forceinline__ Head head_of(uint32_t r0, uint32_t H, int lane, bool live) {
  const uint32_t t0 = r0 / H, h0 = r0 - t0 * H;
  uint32_t t = t0, h = h0 + lane / kLanes;
  if (H == 1) {
    t += h;
    h = 0;
  } else if (H >= (uint32_t)kWaveRows) {
    if (h >= H) { h -= H; ++t; }
  } else {
    const uint32_t k = h / H;
    t += k;
    h -= k * H;
  }
  return live ? Head{t, h} : Head{t0, h0};
}

// A lane's share of one row of up to 128 NI channels. LAST: more than 128 (NI - 1), and the
// rotated channels are the row's last 64 (or none), which lie in iteration NI - 1.
template <typename QT, int NI, bool LAST, bool HALF>
struct Row {
  int sub, nch, nn, rc0, hc;   // lane of sixteen; chunks: row's, normed, first rotated, half the rotated ones
  uint4 v[NI];

  __device__ Row(const RopeParams& p, int n, int lane)
      : sub(lane & (kLanes - 1)), nch(p.D / 8), nn(n / 8), rc0((p.D - p.R) / 8), hc(p.R / 16) {}
  __device__ __forceinline__ int chunk(int i) const { return kLanes * i + sub; }
  __device__ __forceinline__ bool has(int i) const { return (LAST && i < NI - 1) || chunk(i) < nch; }
  // wave-uniform: iteration i has rotated chunks
  __device__ __forceinline__ bool turns(int i) const {
    return LAST ? i == NI - 1 : kLanes * (i + 1) > rc0 && kLanes * i < nch;
  }
  __device__ __forceinline__ int partner(int c) const { return c - rc0 < hc ? c + hc : c - hc; }

  // every lane loads; chunks past the row's (normed: past its normed ones, whose
  // lines are then not fetched) are clamped to the last of them
  template <bool NT>
  __device__ __forceinline__ void load(const uint8_t* x) {
    const uint64_t b = reinterpret_cast<uint64_t>(x) + 16 * sub;
#pragma unroll
    for (int i = 0; i < NI; ++i)
      v[i] = ld16<NT>(LAST && i < NI - 1 ? b + 16 * kLanes * i
                                         : reinterpret_cast<uint64_t>(x) + 16u * (uint32_t)min(chunk(i), nch - 1));
  }
  template <bool NT>
  __device__ __forceinline__ void load_normed(const uint8_t* x) {
    const int last = max(nn - 1, 0);
#pragma unroll
    for (int i = 0; i < NI; ++i) v[i] = ld16<NT>(reinterpret_cast<uint64_t>(x) + 16u * (uint32_t)min(chunk(i), last));
  }
};

// The rotation of one chunk: the angles of its pairs and, where these lie apart
// (HALF), the pairs' other channels, loaded as early as the position is known.
template <typename QT, bool HALF>
struct Turn {
  static constexpr int NE = HALF ? 4 : 2;   // (cos, sin, cos, sin) of two pairs each
  float4 e[NE];
  uint4 other;
  int j, hc;
  // chunk c of the row x; a chunk that is not rotated loads the first rotated one's
  template <typename R>
  __device__ __forceinline__ void load(const R& r, const float* cs, const uint8_t* x, int c) {
    hc = r.hc;
    const bool turn = c >= r.rc0 && c < r.nch;
    j = turn ? c - r.rc0 : 0;
    const uint64_t at = reinterpret_cast<uint64_t>(cs) + (HALF ? 64 * (j < hc ? j : j - hc) : 32 * j);
#pragma unroll
    for (int k = 0; k < NE; ++k) e[k] = __builtin_bit_cast(float4, gld16(at + 16 * k));
    if constexpr (HALF) other = gld16(reinterpret_cast<uint64_t>(x) + 16u * (uint32_t)r.partner(r.rc0 + j));
  }
  __device__ __forceinline__ void ready() {
#pragma unroll
    for (int k = 0; k < NE; ++k) opaque(e[k]);
  }
  // y rotated, z being its pairs' other channels (HALF)
  __device__ __forceinline__ void turn(const float (&y)[8], const float (&z)[8], float sign, float (&o)[8]) const {
    if constexpr (HALF) {
      const float s = j < hc ? -sign : sign;   // first half: a c - b s; second: b c + a s
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        o[2 * k] = fmaf(y[2 * k], e[k].x, z[2 * k] * (s * e[k].y));
        o[2 * k + 1] = fmaf(y[2 * k + 1], e[k].z, z[2 * k + 1] * (s * e[k].w));
      }
    } else {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const float s0 = sign * e[k].y, s1 = sign * e[k].w;
        o[4 * k] = fmaf(y[4 * k], e[k].x, -s0 * y[4 * k + 1]);
        o[4 * k + 1] = fmaf(y[4 * k + 1], e[k].x, s0 * y[4 * k]);
        o[4 * k + 2] = fmaf(y[4 * k + 2], e[k].z, -s1 * y[4 * k + 3]);
        o[4 * k + 3] = fmaf(y[4 * k + 3], e[k].z, s1 * y[4 * k + 2]);
      }
    }
  }
};

// Destinations: rows of a contiguous tensor, rows of the paged cache in their own
// type, 656-byte fp8 rows of the paged cache.
enum { kToRows = 0, kToCache = 1, kToFp8 = 2 };

// 128 latent channels x m, one iteration of the row's lanes, share a scale. (The
// quotients by reciprocal: within an ulp of the true ones, which move a byte only
// where its value lies that near a tie.) A NaN stays one, with scale 1 for its group; an
// infinity makes its group NaN, with a scale of infinity: as the codec of fp8 rows has it.
__device__ __forceinline__ void put_fp8_group(uint8_t* dst, int g, int sub, const float (&x)[8], float m, bool write) {
  float amax = 0.f;
#pragma unroll
  for (int k = 0; k < 8; ++k) amax = __builtin_elementwise_maximum(amax, fabsf(x[k]));   // (keeps a NaN)
  amax = max16(fabsf(amax * m));
  const float scale = amax > 0.f ? amax * (1.f / kFp8Max) : 1.f;
  const float q = amax > 0.f ? m * (kFp8Max * __builtin_amdgcn_rcpf(amax)) : m;
  uint32_t w[2];
  auto pack = [&](auto&& value) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      auto cl = [&](int k) { return __builtin_amdgcn_fmed3f(value(4 * j + k), -kFp8Max, kFp8Max); };
      const int t = __builtin_amdgcn_cvt_pk_fp8_f32(cl(0), cl(1), 0, false);
      w[j] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(cl(2), cl(3), t, true);
    }
  };
  pack([&](int k) { return x[k] * q; });
  // Not of finite factors: NaN and infinities, channels below 1e-33. These are raised by 2^64
  // ahead of the quotient (q past the largest float made NaN of the zeros beside them).
  if (!(amax < INFINITY && q < INFINITY)) {
    const float s = amax < 1.f ? 0x1p64f : 1.f, inv = amax > 0.f ? kFp8Max * __builtin_amdgcn_rcpf(amax * s) : 1.f;
    auto value = [&](int k) { return x[k] * m * s * inv; };
    pack(value);
#pragma unroll
    for (int k = 0; k < 8; ++k)   // (the clamp makes -448 of a NaN: 0xfe)
      if (value(k) != value(k)) w[k / 4] |= 0x7fu << 8 * (k % 4);
  }
  if (!write) return;
  *reinterpret_cast<uint2*>(dst + 128 * g + 8 * sub) = make_uint2(w[0], w[1]);
  if (sub == 0) *reinterpret_cast<float*>(dst + kFp8ScaleOff + 4 * g) = scale;
}

// Rows of one part: workgroup `blk` of its grid. `cached`: they go to the cache
// (workgroup-uniform; DST says how).
template <typename QT, int NI, bool LAST, bool HALF, int DST, bool APPEND, bool NT>
__device__ __forceinline__ void rope_rows(const RopeParams& p, const RopePart& a, uint32_t blk, int tid, float* lds,
                                          bool cached) {
  const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t w0 = blk * kRopeRows + wave * kWaveRows;   // the wave's first row
  const uint32_t r0 = w0 < a.rows ? w0 : 0;                 // (a wave without rows stays for the barrier)
  const uint32_t row = r0 + lane / kLanes;
  const bool live = row < a.rows && w0 < a.rows;
  const auto [t, h] = head_of(r0, a.H, lane, live);
  Row<QT, NI, LAST, HALF> r(p, a.n, lane);
  const uint8_t* x = a.x + (long long)t * a.st + (long long)h * a.sh;
  // Loads in the order of their chains, straight on (where paths with other loads in
  // flight meet, the compiler waits for all of them): what positions and places
  // hang on, the row, the weights; then the angles and the block, which come back
  // while the weights go to LDS.
  Seq seq{};
  if constexpr (APPEND) seq = seq_of(p, lane);
  int pos = p.pos[p.has_pos ? t : 0];
  r.template load<NT>(x);
  Weights<QT, NI> w;
  if (a.w) w.get(p, a, tid);   // workgroup-uniform
  Place at{0, 0, false};
  if constexpr (APPEND) at = place_of(p, seq, (int)t, lane);
  if (!p.has_pos) pos = at.slot;
  const bool in = (!p.R || (pos >= 0 && pos < p.table_rows)) && !at.padded;
  const float* cs = p.table + (size_t)(in ? pos : 0) * p.R;
  Turn<QT, HALF> last;   // of iteration NI - 1
  if (LAST && p.R) last.load(r, cs, x, r.chunk(NI - 1));
  uint8_t* dst = nullptr;
  if (!cached) {
    if (live) dst = a.y + (size_t)row * p.D * 2;
  } else {
    const int blkno = !in ? 0 : p.bs_shift >= 0 ? at.slot >> p.bs_shift : at.slot / p.bs;
    const bool okt = in && blkno < p.bt_stride;
    const int phys = p.bt[okt ? (size_t)at.b * p.bt_stride + blkno : 0];
    if (live && okt && phys >= 0 && phys < p.nblocks)
      dst = p.cache + ((size_t)phys * p.bs + (at.slot - blkno * p.bs)) * (DST == kToFp8 ? kRow656 : p.D * 2);
  }
  const bool write = dst != nullptr;
  if (a.w) w.put(p, a, lds, tid);
  if (w0 >= a.rows) return;

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
    rinv = rsqrtf(sum16(ss) / (float)a.n + p.eps);
  }
  // x w, and the factor that is left
  auto weighted = [&](const uint4& v, int c, float (&f)[8]) {
    unpack8<QT>(v, f);
    if (a.w) {
      float w[8];
      weights8(lds_addr_of(lds), c, w);
#pragma unroll
      for (int k = 0; k < 8; ++k) f[k] *= w[k];
    }
    return c < r.nn ? rinv : 1.f;
  };
  auto normed = [&](const uint4& v, int c, float (&f)[8]) {
    const float s = weighted(v, c, f);
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] *= s;
  };
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int c = r.chunk(i);
    float f[8];
    if constexpr (DST == kToFp8 && LAST) {
      if (i < 4) {   // latent channels, none of them rotated
        const float s = weighted(r.v[i], c, f);
        put_fp8_group(dst, i, r.sub, f, s, write);
        continue;
      }
    }
    normed(r.v[i], c, f);
    if (p.R && r.turns(i)) {
      Turn<QT, HALF> one;
      if constexpr (!LAST) one.load(r, cs, x, c);
      Turn<QT, HALF>& e = LAST ? last : one;
      e.ready();
      float other[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, o[8];
      if constexpr (HALF) normed(e.other, r.partner(r.rc0 + e.j), other);
      e.turn(f, other, p.sign, o);
#pragma unroll
      for (int k = 0; k < 8; ++k) f[k] = c >= r.rc0 && c < r.nch ? o[k] : f[k];
    }
    if constexpr (DST == kToFp8) {
      if (i < 4) put_fp8_group(dst, i, r.sub, f, 1.f, write);
      else if (write && r.sub < 8) *reinterpret_cast<uint4*>(dst + kFp8RopeOff + 16 * r.sub) = pack8<__bf16>(f);
    } else if (write && r.has(i)) {
      uint4 o = pack8<QT>(f);
      if (!in) o = make_uint4(0, 0, 0, 0);   // a padded row (of the queries: none goes to the cache)
      st16(dst + 16 * c, o, p.nt_store);
    }
  }
}

// Workgroups [0, part[0].blocks) take the KV rows (the longer chain of loads
// starts first), the others the queries.
// NT: the rows are read past the caches
template <typename QT, int NI, bool LAST, bool HALF, int DST, bool NT>
__global__ void __launch_bounds__(kRopeThreads) sas_rope_kernel(const RopeParams p) {
  constexpr bool kAppend = DST != kToRows;
  __shared__ __attribute__((aligned(16))) float lds[Weights<QT, NI>::kAll];
  const uint32_t b = blockIdx.x, nkv = (uint32_t)p.part[0].blocks;
  // one copy of the code where it can be: its first fetch is much of a small call
  const RopePart& a = p.part[b < nkv ? 0 : 1];
  const uint32_t blk = b < nkv ? b : b - nkv;
  if constexpr (DST == kToFp8) {
    if (b < nkv) rope_rows<QT, NI, LAST, HALF, kToFp8, true, NT>(p, a, blk, threadIdx.x, lds, true);
    else rope_rows<QT, NI, LAST, HALF, kToCache, true, NT>(p, a, blk, threadIdx.x, lds, false);
  } else {
    rope_rows<QT, NI, LAST, HALF, DST, kAppend, NT>(p, a, blk, threadIdx.x, lds, kAppend && b < nkv);
  }
}

// ---------------------------------------------------------------------------
// backward
// ---------------------------------------------------------------------------

// A workgroup walks its part's rows; with weights every lane sums its channels'
// weight gradients in registers, the workgroup adds them up through LDS once
// at its end and leaves one partial row: no atomics, the same order every time.
// W: weight gradients are wanted of a part at least (else none has weights in
// need of sums; weights themselves may be there).
template <typename QT, int NI, bool LAST, bool HALF, bool W>
__global__ void __launch_bounds__(kRopeThreads, NI <= 5 ? 3 : 2) sas_rope_grad_kernel(const RopeParams p) {
  constexpr int kWaves = kRopeThreads / 64;
  constexpr int kAll = Weights<QT, NI>::kAll;
  __shared__ __attribute__((aligned(16))) float lds[W ? kWaves * kAll : kAll];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t nkv = (uint32_t)p.part[0].blocks;
  const RopePart& a = p.part[blockIdx.x < nkv ? 0 : 1];
  const uint32_t blk = blockIdx.x < nkv ? blockIdx.x : blockIdx.x - nkv;
  Weights<QT, NI> w;   // ones where there are none
  if (a.w) w.get(p, a, tid);
  float dw[W ? NI : 1][8];
#pragma unroll
  for (int i = 0; i < (W ? NI : 1); ++i)
#pragma unroll
    for (int k = 0; k < 8; ++k) dw[i][k] = 0.f;
  Row<QT, NI, LAST, HALF> r(p, a.n, lane), g(p, a.n, lane);
  w.put(p, a, lds, tid);
  for (uint32_t r0 = blk * kRopeRows + wave * kWaveRows; r0 < a.rows; r0 += (uint32_t)a.blocks * kRopeRows) {
    const uint32_t row = r0 + lane / kLanes;
    const bool live = row < a.rows;
    const auto [t, h] = head_of(r0, a.H, lane, live);
    const int pos = p.pos[p.has_pos ? t : 0];
    // (kept out of registers: hoisted out of the loop the weights cost a wave a SIMD)
    uint32_t wl = lds_addr_of(lds);
    asm volatile("" : "+v"(wl));
    // x of normed channels alone is needed: the others' lines are not fetched
    const uint8_t* x = a.x + (long long)t * a.st + (long long)h * a.sh;
    const uint8_t* dy = a.dy + (long long)t * a.dst + (long long)h * a.dsh;
    either(p.nt_load, [&] { r.template load_normed<true>(x); g.template load<true>(dy); },
           [&] { r.template load_normed<false>(x); g.template load<false>(dy); });
    const bool in = live && (!p.R || (pos >= 0 && pos < p.table_rows));
    const float* cs = p.table + (size_t)(in ? pos : 0) * p.R;
    // u = dy rotated back, of iteration i
    auto grad = [&](int i, float (&u)[8]) {
      unpack8<QT>(g.v[i], u);
      if (p.R && r.turns(i)) {
        const int c = r.chunk(i);
        Turn<QT, HALF> e;
        e.load(r, cs, dy, c);
        e.ready();
        float other[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, o[8];
        if constexpr (HALF) unpack8<QT>(e.other, other);
        e.turn(u, other, -p.sign, o);
#pragma unroll
        for (int k = 0; k < 8; ++k) u[k] = c >= r.rc0 && c < r.nch ? (in ? o[k] : 0.f) : u[k];
      }
    };
    // the rotated channels of the builds with one such iteration are kept, the
    // others' made twice
    float last[8];
    if constexpr (LAST) grad(NI - 1, last);
    auto get = [&](int i, float (&u)[8]) {
      if (LAST && i == NI - 1) {
#pragma unroll
        for (int k = 0; k < 8; ++k) u[k] = last[k];
      } else {
        grad(i, u);
      }
    };
    // x of the other channels, and rows that are padding or past the last one,
    // count as zeros whatever they hold
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      if (!in || r.chunk(i) >= r.nn) r.v[i] = make_uint4(0, 0, 0, 0);
      if (!in) g.v[i] = make_uint4(0, 0, 0, 0);
      opaque(r.v[i]);
      opaque(g.v[i]);
    }
    if constexpr (LAST) {
#pragma unroll
      for (int k = 0; k < 8; ++k) last[k] = in ? last[k] : 0.f;
    }
    float ss = 0.f, sg = 0.f;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int c = r.chunk(i);
      float f[8], u[8], w[8], s2 = 0.f;
      unpack8<QT>(r.v[i], f);
      get(i, u);
      weights8(wl, c, w);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        ss = fmaf(f[k], f[k], ss);
        s2 = fmaf(u[k] * w[k], f[k], s2);
      }
      sg += c < r.nn ? s2 : 0.f;   // (an infinite gradient of the other channels stays out)
      __builtin_amdgcn_sched_barrier(0);   // chunk by chunk: their 32-bit values all at once spill
    }
    const float n = (float)max(a.n, 1);
    float rinv = rsqrtf(sum16(ss) / n + p.eps);
    opaque(rinv);
    rinv = in ? rinv : 0.f;   // (eps 0: no infinity in a padded row)
    const float m = sum16(sg) / n * rinv * rinv * rinv;
    uint8_t* dst = a.y + (size_t)row * p.D * 2 + 16 * r.sub;
    // the second pass unpacks anew: kept from the first, the values in 32 bits spill
    asm volatile("" : "+v"(wl));
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      opaque(r.v[i]);
      opaque(g.v[i]);
    }
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int c = r.chunk(i);
      float f[8], u[8], w[8], o[8];
      unpack8<QT>(r.v[i], f);
      get(i, u);
      weights8(wl, c, w);
      // past the normed channels: u 1 - 0 0
      const float ri = c < r.nn ? rinv : 1.f, mi = c < r.nn ? m : 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        o[k] = fmaf(u[k] * w[k], ri, -(f[k] * mi));
        if constexpr (W) dw[i][k] = fmaf(u[k], f[k] * rinv, dw[i][k]);   // (past n: never read)
      }
      const uint4 v = pack8<QT>(o);
      if (live && r.has(i)) st16(dst + 16 * kLanes * i, v, p.nt_store);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  if constexpr (W) {
    if (!a.dw) return;   // workgroup-uniform
    lds_barrier();       // every wave has done with the weights
    asm volatile("" ::: "memory");
    // the wave's four rows, then its four waves
#pragma unroll
    for (int i = 0; i < NI; ++i) {
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float s = rows_sum(dw[i][k]);
        if (lane < kLanes) lds[wave * kAll + r.chunk(i) * 8 + k] = s;
      }
    }
    __syncthreads();
    for (int j = tid; j < a.n; j += kRopeThreads) {
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) s += lds[w * kAll + j];
      a.dw[(size_t)blk * p.D + j] = s;
    }
  }
}

// Weight gradients from the workgroups' partial rows: 16 channels a workgroup, 64
// threads a channel (16: 4.2 us for 512 rows, a load after the other), in a fixed order.
struct RopeSum { const float* part[2]; float* dw[2]; int rows[2], n[2], D; };
constexpr int kSumThreads = 1024, kSumRows = kSumThreads / 16;
__global__ void __launch_bounds__(kSumThreads) sas_rope_dw_kernel(const RopeSum s) {
  __shared__ float lds[kSumRows][17];
  const int w = blockIdx.y, c = threadIdx.x & 15, k = threadIdx.x >> 4, j = blockIdx.x * 16 + c;
  if (!s.dw[w]) return;   // workgroup-uniform
  float v = 0.f;
  if (j < s.n[w]) {
#pragma unroll 8
    for (int i = k; i < s.rows[w]; i += kSumRows) v += s.part[w][(size_t)i * s.D + j];
  }
  lds[k][c] = v;
  __syncthreads();
  if (k == 0 && j < s.n[w]) {
    v = 0.f;
#pragma unroll
    for (int i = 0; i < kSumRows; ++i) v += lds[i][c];
    s.dw[w][j] = v;
  }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------

constexpr double kInfinityCache = 256e6;
constexpr double kMostRows = (1 << 28) - 2 * kRopeRows;

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
  // (a launch has fewer than 2^32 threads, sixteen of them a row)
  const double rows = (double)a->T * ((double)a->H + (a->kv ? 1 : 0));
  if (rows > kMostRows)
    return set_error(SAS_EINVAL, "%s: %s rows, a call takes at most 2^28 - %d", what,
                     rows >= 2147483648.0 ? "2^31 or more" : "too many", 2 * kRopeRows);
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
  // (no rotation, or an append's own positions: an address that is read and ignored)
  p->has_pos = a->positions && a->rope_dim;
  p->pos = p->has_pos ? a->positions : (const int32_t*)(a->kv ? a->kv : a->q);
  p->table = a->table;
  p->table_rows = (int)a->table_rows;
  p->D = (int)a->D; p->R = a->rope_dim;
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
    kv.x = (const uint8_t*)a->kv; kv.y = (uint8_t*)a->kv_out; kv.w = kv.n ? (const uint8_t*)a->kv_weight : nullptr;
    kv.st = a->kv_stride_t * 2; kv.rows = (uint32_t)a->T;
  }
  if (a->q) {
    q.x = (const uint8_t*)a->q; q.y = (uint8_t*)a->q_out; q.w = q.n ? (const uint8_t*)a->q_weight : nullptr;
    q.st = a->q_stride_t * 2; q.sh = a->q_stride_h * 2; q.rows = (uint32_t)(a->T * a->H);
  }
  for (RopePart& x : p->part) x.blocks = (int)((x.rows + kRopeRows - 1) / kRopeRows);
  // Rows that with the output outgrow the 256 MB Infinity Cache are read past the
  // caches, and an output of twice its size written so. us a call without, with
  // the loads, with both, and of call and attention over its output, 64 heads of 512
  // channels: 2048 tokens 42 / 43 / 45, 103 / 103 / 113; 4096 94 / 80 / 88, 217 / 206 /
  // 215; 8192 187 / 181 / 173, 421 / 414 / 415. Smaller outputs are left for their
  // reader: written past the caches, 43 -> 38 us alone for 5300 tokens of 16 heads, but
  // call and attention of 2048 tokens 103 -> 115. Appends with their queries, loads alone: 64
  // heads of 512, 2000 / 3000 / 4096 tokens 42 -> 42, 71 -> 60, 94 -> 81; fp8 rows 48 -> 48, 82 -> 68, 111 -> 105.
  const double bytes = 2.0 * a->D * ((double)p->part[0].rows + p->part[1].rows);
  p->nt_load = 2 * bytes >= kInfinityCache;
  p->nt_store = bytes >= 2 * kInfinityCache;
}

// The kernel for a row width: 128, 512 or 576 channels with 64 rotated ones (or none) in
// their own builds, any other in one of up to eight chunks a lane. That costs a narrow
// forward its idle chunks (about 270 MB of rows of 64 heads, TB/s read and written: 192
// channels 3.1, 256 3.8, 576 with 96 rotated 4.7, 512 with 32 or 128, 640 and 1024 6.3 to 6.7)
// and the backward its registers: eight chunks of x and dy and (W) 64 sums spill 21 to
// 151 of them. Its us with / without weights: 192 1743 / 622, 256 1342 / 484, 512 with
// 128 rotated 727 / 274, 640 620 / 240, 1024 432 / 167; 512 in its own build 114 / 101.
template <typename F>
int by_width(const SasNormRopeArgs* a, F&& f) {
  const bool last = a->rope_dim == 64 || a->rope_dim == 0;
  auto half = [&](auto ni, auto l) {
    return a->flags & SAS_ROPE_HALF ? f(ni, l, std::true_type{}) : f(ni, l, std::false_type{});
  };
  if (last && a->D == 576) return half(std::integral_constant<int, 5>{}, std::true_type{});
  if (last && a->D == 512) return half(std::integral_constant<int, 4>{}, std::true_type{});
  if (last && a->D == 128) return half(std::integral_constant<int, 1>{}, std::true_type{});
  return half(std::integral_constant<int, 8>{}, std::false_type{});
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
    auto go = [&](auto kern) { hipLaunchKernelGGL(kern, grid, dim3(kRopeThreads), 0, st, p); };
    if (a->dtype == SAS_DT_BF16) {
      if (p.nt_load) go(sas_rope_kernel<__bf16, NI, L, HF, DST, true>);
      else go(sas_rope_kernel<__bf16, NI, L, HF, DST, false>);
    } else {
      if (p.nt_load) go(sas_rope_kernel<_Float16, NI, L, HF, DST, true>);
      else go(sas_rope_kernel<_Float16, NI, L, HF, DST, false>);
    }
    return launched(what);
  });
}

// Workgroups of the backward's two parts: three a CU (what the builds with weights hold, 3 waves a
// SIMD; those without hold four or five), shared out by rows, none without rows of its own.
// A count of rows just above one round makes some walk twice: 736 tokens of 16 heads are
// 782 groups of rows for 768 workgroups, 12-14 us.
void grad_blocks(RopeParams* p) {
  const double all = (double)p->part[0].rows + p->part[1].rows;
  const long long most = 3LL * device_cus();
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
  // us without, with loads, with both, 64 heads of 512 channels: 1024 tokens 37 / 38 /
  // 36; 2048 80 / 68 / 67; 4096 153 / 148 / 129; 8192 304 / 294 / 285
  const double bytes = 2.0 * f->D * ((double)p->part[0].rows + p->part[1].rows);
  p->nt_load = p->nt_store = 3 * bytes >= kInfinityCache;
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
    hipLaunchKernelGGL(sas_rope_dw_kernel, dim3((unsigned)((f->D + 15) / 16), 2), dim3(kSumThreads), 0, st, s);
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
  p.bs_shift = p.bs & (p.bs - 1) ? -1 : __builtin_ctz(p.bs);
  hipStream_t st = (hipStream_t)stream;
  if (!fp8) return launch_rope<kToCache>(r, p, st, "cache_append");
  const dim3 grid((unsigned)(p.part[0].blocks + p.part[1].blocks)), block(kRopeThreads);
  auto go = [&](auto kern) { hipLaunchKernelGGL(kern, grid, block, 0, st, p); };
  const bool half = r->flags & SAS_ROPE_HALF;
  auto by_load = [&](auto last, auto hf) {
    constexpr bool L = decltype(last)::value, HF = decltype(hf)::value;
    if (p.nt_load) go(sas_rope_kernel<__bf16, 5, L, HF, kToFp8, true>);
    else go(sas_rope_kernel<__bf16, 5, L, HF, kToFp8, false>);
  };
  if (r->rope_dim == 64 || r->rope_dim == 0) half ? by_load(std::true_type{}, std::true_type{}) : by_load(std::true_type{}, std::false_type{});
  else half ? by_load(std::false_type{}, std::true_type{}) : by_load(std::false_type{}, std::false_type{});
  return launched("cache_append");
}
