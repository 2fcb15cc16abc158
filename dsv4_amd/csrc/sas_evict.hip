// Eviction of cache rows by their weight on MI355X (gfx950): of each sequence with more
// than `budget` rows stay its first ones, its last ones and the heaviest of the others
// (of equal ones those at the lowest positions), moved together in their order.
//
//  evict_select_kernel  one workgroup a sequence reads its weights once, as
//     order-preserving 64-bit keys (in registers up to 4096 rows, the keys' high words in
//     LDS up to 32768; longer sequences are read anew in each pass), and finds the key that
//     divides the candidates: passes of 2048 counts in LDS over the range of the weights or
//     over 11 bits, until the bin in question holds at most 128 keys, which are ranked
//     against each other, or one key alone. Then every wave lists the rows of its run that
//     stay. 32 sequences of 2100 rows 8.5 us; four of 20000 to 32768 26 us, 6 of them one
//     CU's load of 208 KB. A call on 32768 / 33000 / 131072 rows 38 / 75 / 200 us, and where
//     the cut falls among many rows of weight 0 72 / 134 / 418.
//  evict_move_kernel    a workgroup owns one slice of the rows' bytes of one sequence
//     and walks the list: since row i comes from a row at or behind i, the rows of a
//     chunk are loaded before any of them is written, and later chunks read only rows
//     behind them. Rows that stay where they are are not touched. One more workgroup a
//     sequence closes up the weights. 32 sequences of 2048 rows of 1152 bytes 12.5 us (an
//     eviction of a few rows moves those behind the first that leaves: up to 75 MB read and
//     as much written, most of it in the Infinity Cache), four of 4096 rows of 656 bytes 13.

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
  int bs_log;        // log2(bs), -1: no power of two
  int nxcd, groups, run, slices;   // evict_move_kernel: XCDs, those of a sequence, workgroups on each, slices of a row
};

constexpr int kSelThreads = 1024, kSelWaves = kSelThreads / 64;
constexpr int kBins = 2048, kCopies = 4;   // a pass's counts; lanes with equal lane % 4 share a copy
constexpr int kList = 4096;                // so few candidates go to LDS for the passes that are left
constexpr int kRank = 128;                 // and so few are ranked instead of counted
constexpr int kRegRows = 4, kWordRows = 32768;   // rows a thread in registers, rows a workgroup in LDS

// A weight's key, in the weights' order, as two words (64-bit shifts and compares cost
// several times the 32-bit ones that a word at a time takes): NaN below everything,
// -0 = 0. Keys' high words lie between the two that mark other rows.
struct Key { uint32_t hi, lo; };
constexpr uint32_t kNone = 0, kStays = ~0u;   // no row; a row that stays anyway
constexpr uint32_t kZero = 0x80000000u;       // a weight of 0
__device__ __forceinline__ bool is_key(Key k) { return k.hi - 1u < kStays - 1u; }
__device__ __forceinline__ Key key_of(double w) {
  const uint64_t u = __builtin_bit_cast(uint64_t, w + 0.);
  const uint32_t hi = (uint32_t)(u >> 32), lo = (uint32_t)u, neg = (uint32_t)((int32_t)hi >> 31);
  return w != w ? Key{1u, 0u} : Key{hi ^ (neg | 0x80000000u), lo ^ neg};
}
struct SelShared {
  int hist[kCopies][kBins];
  Key lkey[kList];
  int lpos[kList];
};
struct SelLong {
  int hist[kBins];
  uint32_t word[kWordRows];   // keys' high words
};
struct SelSmall {
  int wsum[kSelWaves], wtie[kSelWaves];
  int found[3];             // bin, candidates above it, candidates in it
  int nlist, nrank;
  Key rkey[kRank];
  int rpos[kRank];
  Key edge;
  uint32_t any[4];          // or, and of the high words, of the low ones
  int need;
};

// Sum of v over the waves before this one.
__device__ __forceinline__ int before(const int* v, int wave, int lane) {
  int x = lane < kSelWaves && lane < wave ? v[lane] : 0;
#pragma unroll
  for (int d = 1; d < kSelWaves; d <<= 1) x += __shfl_xor(x, d);
  return __builtin_amdgcn_readfirstlane(x);
}

// Where the need-th candidate from the top falls: bin, candidates above it and in it, to
// sh.found. Barriers before (the counts are there) and after.
template <typename Count>
__device__ __forceinline__ void find_bin(SelSmall& sh, int need, Count&& count) {
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  __syncthreads();
  // bins from the top: thread i holds bins 2047 - 2 i and 2046 - 2 i
  const int h0 = count(kBins - 1 - 2 * tid), h1 = count(kBins - 2 - 2 * tid);
  int x = h0 + h1;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) { const int v = __shfl_up(x, d); x += lane >= d ? v : 0; }
  if (lane == 63) sh.wsum[wave] = x;
  __syncthreads();
  const int above = x - h0 - h1 + before(sh.wsum, wave, lane);
  if (above < need && above + h0 + h1 >= need) {   // one thread
    const bool second = above + h0 < need;
    sh.found[0] = kBins - 1 - 2 * tid - second;
    sh.found[1] = above + (second ? h0 : 0);
    sh.found[2] = second ? h1 : h0;
  }
  __syncthreads();
}

// The need-th heaviest of the `left` keys in sh.rkey, to sh.edge, and how many of those equal
// to it are wanted, to sh.need. Barriers before and after.
__device__ __forceinline__ void rank_keys(SelSmall& sh, int left, int need) {
  constexpr int TK = kSelThreads / kRank;    // threads a key
  const int i = threadIdx.x / TK, part = threadIdx.x % TK;
  __syncthreads();
  int above = 0, ahead = 0;
  const Key ki = i < left ? sh.rkey[i] : Key{0, 0};
  const int pi = i < left ? sh.rpos[i] : 0;
  for (int j = part; j < left; j += TK) {
    const Key k = sh.rkey[j];
    above += k.hi > ki.hi || (k.hi == ki.hi && k.lo > ki.lo);
    ahead += k.hi == ki.hi && k.lo == ki.lo && sh.rpos[j] < pi;
  }
#pragma unroll
  for (int d = 1; d < TK; d <<= 1) { above += __shfl_xor(above, d); ahead += __shfl_xor(ahead, d); }
  if (part == 0 && i < left && above + ahead == need - 1) { sh.edge = ki; sh.need = need - above; }
  __syncthreads();
}

// Whether the workgroup's words are one: their or and and joined in any[0], any[1] (0 and ~0
// before), of the threads that have some. Barriers between and after.
__device__ __forceinline__ bool one_word(uint32_t* any, uint32_t o, uint32_t a, bool has) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) { o |= __shfl_xor(o, d); a &= __shfl_xor(a, d); }
  if (__ballot(has) && (threadIdx.x & 63) == 0) { atomicOr(&any[0], o); atomicAnd(&any[1], a); }
  __syncthreads();
  return any[0] == any[1];
}

__device__ __forceinline__ int lanes_before(uint64_t m) {
  return (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0));
}

// (Weights that another stream changes meanwhile give any choice of rows, but no access out
// of range: places are held below the lists' ends, and the moves look at what they are given.)

// A sequence of n > budget rows. Wave w has the run of rows from w * run on, lane l its rows
// l, l + 64, ..: E of them in registers, or (E = 0) read where they are needed.
template <int E>
__device__ __forceinline__ void select_rows(const EvictParams& p, SelShared& big, SelSmall& sh, int n, const double* w, int32_t* kept) {
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  // candidates [lo, hi), of which `need` stay; rows without a weight count as 0
  const int lo = p.first, hi = n - p.recent;
  int need = p.budget - p.first - p.recent;
  const int run = ((n - 1) / kSelThreads + 1) * 64, r0 = wave * run;
  const int ne = E ? E : run / 64;
  // (16 runs end at 2^31 at most; what lies past the last row of one is not looked at)
  auto load = [&](int e) {
    const int j = r0 + e * 64 + lane;
    return j < n && j < p.weight_rows ? w[j] : 0.;
  };
  auto mark = [&](int e, double v) {
    const int j = r0 + e * 64 + lane;
    Key k = key_of(v);
    if (j < lo || j >= hi) k.hi = kStays;
    if (e * 64 >= run || j >= n) k.hi = kNone;
    return k;
  };
  Key reg[E ? E : 1];
  if constexpr (E > 0) {
    constexpr int U = E < 8 ? E : 8;   // loads in flight (more take the keys' registers)
#pragma unroll
    for (int e0 = 0; e0 < E; e0 += U) {
      double v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) v[u] = load(e0 + u);
#pragma unroll
      for (int u = 0; u < U; ++u) reg[e0 + u] = mark(e0 + u, v[u]);
      asm volatile("" ::: "memory");
    }
  }
  // f(row, key) for the lane's rows
  auto each = [&](auto&& f) __attribute__((always_inline)) {
    if constexpr (E > 0) {
#pragma unroll
      for (int e = 0; e < E; ++e) f(r0 + e * 64 + lane, reg[e]);
    } else {
      constexpr int U = 8;   // loads in flight
      for (int e0 = 0; e0 < ne; e0 += U) {
        double v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = load(min(e0 + u, ne - 1));
#pragma unroll
        for (int u = 0; u < U; ++u) f(r0 + (e0 + u) * 64 + lane, mark(e0 + u, v[u]));
      }
    }
  };

  // the keys that stay: those above `edge`, and the first `need` of those equal to it
  Key edge{kStays - 1, ~0u};                     // above every key (none is wanted)
  Key prefix{0, 0}, mask{0, 0};
  bool done = need == 0;
  int left = hi - lo;                            // candidates that share the prefix
  int listed = -1;                               // candidates in LDS, -1: none are yet
  auto same = [&](Key k) { return (k.hi & mask.hi) == prefix.hi && (k.lo & mask.lo) == prefix.lo; };
  // f(row, key) for the candidates that share the prefix
  auto scan = [&](auto&& f) __attribute__((always_inline)) {
    if (listed < 0) {
      each([&](int j, Key k) {
        if (is_key(k) && same(k)) f(j, k);
      });
    } else {
      for (int i = tid; i < listed; i += kSelThreads) {
        const Key k = big.lkey[i];
        if (same(k)) f(big.lpos[i], k);
      }
    }
  };
  if (tid == 0) sh.nlist = sh.nrank = 0;
  if constexpr (E > 0) {
    if (!done && left > kRank) {
      // first over the range of the positive weights, in up to 2047 even steps of their high
      // words (bin 0: the others): a bin of few keys, or of one key (0), ends the search
      uint32_t most = 0, least = ~0u;   // the highest word, and the lowest above 0's less that and 1
      each([&](int, Key k) {
        const uint32_t h = is_key(k) ? k.hi : 0u;
        most = max(most, h);
        least = min(least, h - (kZero + 1));
      });
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) { most = max(most, __shfl_xor(most, d)); least = min(least, __shfl_xor(least, d)); }
      for (int i = tid; i < kCopies * kBins; i += kSelThreads) (&big.hist[0][0])[i] = 0;
      if (tid < 4) sh.any[tid] = tid & 1 ? ~0u : 0u;
      __syncthreads();
      if (lane == 0) { atomicMax(&sh.any[0], most); atomicMin(&sh.any[1], least); }
      __syncthreads();
      most = __builtin_amdgcn_readfirstlane(sh.any[0]);
      const uint32_t base = min(kZero + 1 + (uint32_t)__builtin_amdgcn_readfirstlane(sh.any[1]), most);
      const int s = max(0, 32 - __clz((int)((most - base) / (kBins - 1))));
      auto bin_of = [&](Key k) { return k.hi > kZero ? 1 + (int)((k.hi - base) >> s) : 0; };
      int* hist = big.hist[lane % kCopies];
      each([&](int, Key k) {
        if (is_key(k)) atomicAdd(&hist[bin_of(k)], 1);
      });
      find_bin(sh, need, [&](int i) { return big.hist[0][i] + big.hist[1][i] + big.hist[2][i] + big.hist[3][i]; });
      const int bin = __builtin_amdgcn_readfirstlane(sh.found[0]), rest = need - __builtin_amdgcn_readfirstlane(sh.found[1]);
      const int in = __builtin_amdgcn_readfirstlane(sh.found[2]);
      if (in <= kRank) {
        each([&](int j, Key k) {
          if (is_key(k) && bin_of(k) == bin) {
            const int at = atomicAdd(&sh.nrank, 1);
            if (at < kRank) { sh.rkey[at] = k; sh.rpos[at] = j; }
          }
        });
        rank_keys(sh, in, rest);
        edge = sh.edge;
        need = sh.need;
        done = true;
      } else if (bin == 0) {
        if (tid < 4) sh.any[tid] = tid & 1 ? ~0u : 0u;
        __syncthreads();
        uint32_t o[4] = {0, ~0u, 0, ~0u};
        bool has = false;
        each([&](int, Key k) {
          if (is_key(k) && k.hi <= kZero) { o[0] |= k.hi; o[1] &= k.hi; o[2] |= k.lo; o[3] &= k.lo; has = true; }
        });
        const bool hi1 = one_word(sh.any, o[0], o[1], has), lo1 = one_word(sh.any + 2, o[2], o[3], has);
        if (hi1 && lo1) { edge = Key{sh.any[0], sh.any[2]}; need = rest; done = true; }
      }
      __syncthreads();   // found and any are read
    }
  }
  // passes: bits 21.., 10.., 0.. of the high word, then of the low one
  for (int pass = 0; !done && pass < 6; ++pass) {
    if (left <= kRank) {
      // rank them: the need-th heaviest is the edge
      __syncthreads();
      scan([&](int j, Key k) {
        const int at = atomicAdd(&sh.nrank, 1);
        if (at < kRank) { sh.rkey[at] = k; sh.rpos[at] = j; }
      });
      rank_keys(sh, left, need);
      edge = sh.edge;
      need = sh.need;
      done = true;
      break;
    }
    const int third = pass % 3, s = third == 0 ? 21 : third == 1 ? 10 : 0;
    const uint32_t digit = third == 2 ? 1023u : 2047u;
    const bool high = pass < 3;
    for (int i = tid; i < kCopies * kBins; i += kSelThreads) (&big.hist[0][0])[i] = 0;
    if (tid < 4) sh.any[tid] = tid & 1 ? ~0u : 0u;
    __syncthreads();
    int* hist = big.hist[lane % kCopies];
    scan([&](int, Key k) { atomicAdd(&hist[(high ? k.hi : k.lo) >> s & digit], 1); });
    find_bin(sh, need, [&](int i) { return big.hist[0][i] + big.hist[1][i] + big.hist[2][i] + big.hist[3][i]; });
    const uint32_t bin = (uint32_t)__builtin_amdgcn_readfirstlane(sh.found[0]) << s;
    (high ? prefix.hi : prefix.lo) |= bin;
    (high ? mask.hi : mask.lo) |= digit << s;
    need -= __builtin_amdgcn_readfirstlane(sh.found[1]);
    left = __builtin_amdgcn_readfirstlane(sh.found[2]);
    if (need == left) {   // the whole bin stays: every key from its lowest on
      // (prefix 0: the search would have taken every candidate)
      edge = Key{prefix.hi - (prefix.lo == 0), prefix.lo - 1};
      need = 0;
      done = true;
    } else if (left > kRank) {
      if (listed < 0 && left <= kList) {
        // (in any order: their places tell them apart)
        int mine = 0;
        each([&](int, Key k) { mine += is_key(k) && same(k); });
        int y = mine;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) { const int v = __shfl_up(y, d); y += lane >= d ? v : 0; }
        int at = 0;
        if (lane == 63) at = atomicAdd(&sh.nlist, y);
        at = __shfl(at, 63) + y - mine;
        each([&](int j, Key k) {
          if (is_key(k) && same(k) && at < kList) { big.lkey[at] = k; big.lpos[at] = j; ++at; }
        });
        listed = left;
        __syncthreads();
      }
      if (listed >= 0) {
        // one key alone (weights of 0, say) needs no further pass
        uint32_t o[4] = {0, ~0u, 0, ~0u};
        bool has = false;
        scan([&](int, Key k) { o[0] |= k.hi; o[1] &= k.hi; o[2] |= k.lo; o[3] &= k.lo; has = true; });
        const bool hi1 = one_word(sh.any, o[0], o[1], has), lo1 = one_word(sh.any + 2, o[2], o[3], has);
        if (hi1 && lo1) { edge = Key{sh.any[0], sh.any[2]}; done = true; }
        __syncthreads();   // read before the next pass clears them
      }
    }
  }
  if (!done) edge = prefix;   // all 64 bits: `need` of its equals stay

  // list: a wave's places follow from the runs before it
  // (keys that share the edge's high word are rare: their low words are looked at only then)
  auto split = [&](Key k, uint64_t& over, uint64_t& tie) __attribute__((always_inline)) {
    over = __ballot(k.hi > edge.hi);
    tie = __ballot(k.hi == edge.hi);
    if (tie) {
      over |= tie & __ballot(k.lo > edge.lo);
      tie &= __ballot(k.lo == edge.lo);
    }
  };
  int nk = 0, nt = 0;
  each([&](int, Key k) {
    uint64_t over, tie;
    split(k, over, tie);
    nk += __popcll(over);
    nt += __popcll(tie);
  });
  __syncthreads();   // wsum is read
  if (lane == 0) { sh.wsum[wave] = nk; sh.wtie[wave] = nt; }
  __syncthreads();
  int pk = before(sh.wsum, wave, lane), pt = before(sh.wtie, wave, lane);
  each([&](int j, Key k) {
    uint64_t over, tie;
    split(k, over, tie);
    if (over | tie) {
      const int rank = pt + lanes_before(tie), at = pk + lanes_before(over) + min(rank, need);
      if (((over >> lane & 1) || ((tie >> lane & 1) && rank < need)) && (unsigned)at < (unsigned)p.budget) kept[at] = j;
      pk += __popcll(over);
      pt += __popcll(tie);
    }
  });
}

// A sequence of n > budget rows, at most kWordRows, with its keys' high words in LDS: many
// rows a thread in registers are as many unrolled copies of every step, whose instructions
// then have to be fetched (26000 rows: 52 us, 12 of them one pass of counts). Low words are
// read from memory where they matter. One CU works here, and what a pass takes is the
// instructions it issues for a row: so no pass looks where a wave's rows end (the words
// behind are kNone), a weight's word takes two instructions where it is finite and not
// below 0, and ties are counted only in steps that hold some.
__device__ __forceinline__ void select_long(const EvictParams& p, SelLong& big, SelSmall& sh, int n, const double* w, int32_t* kept) {
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int lo = p.first, hi = n - p.recent;
  int need = p.budget - p.first - p.recent, left = hi - lo;
  const int run = ((n - 1) / (2 * kSelThreads) + 1) * 128, r0 = wave * run;   // 16 runs: at most kWordRows
  auto weight = [&](int j) { return (unsigned)j < (unsigned)p.weight_rows ? w[j] : 0.; };
  auto each = [&](auto&& f) __attribute__((always_inline)) {   // f(row, word)
    for (int i = 0; i < run; i += 128) {
      const int j = r0 + i + lane;
      const uint32_t v0 = big.word[j], v1 = big.word[j + 64];
      f(j, v0);
      f(j + 64, v1);
    }
  };
  // the same with the low words of the rows whose word is `word`: f(row, low word), the
  // others' left out
  auto lows = [&](uint32_t word, auto&& f) __attribute__((always_inline)) {
    for (int i = 0; i < run; i += 128) {
      const int j = r0 + i + lane;
      const bool h0 = big.word[j] == word, h1 = big.word[j + 64] == word;
      const double v0 = h0 ? weight(j) : 0., v1 = h1 ? weight(j + 64) : 0.;
      if (h0) f(j, key_of(v0).lo);
      if (h1) f(j + 64, key_of(v1).lo);
    }
  };
  auto is_word = [](uint32_t k) { return k - 1u < kStays - 1u; };
  auto clear = [&] {   // counts and joined words, behind a barrier; one follows
    __syncthreads();
    for (int i = tid; i < kBins; i += kSelThreads) big.hist[i] = 0;
    if (tid < 4) sh.any[tid] = tid & 1 ? ~0u : 0u;
    __syncthreads();
  };
  if (tid == 0) sh.nrank = 0;
  clear();
  uint32_t most = 0, least = ~0u;   // the candidates' highest word, and the lowest above 0's less that and 1
  {
    constexpr int U = 8;   // rows a lane under way (4: 0.5 us more; 16 and 32: no less, a CU's 208 KB take 6 us)
    const uint32_t* wh = reinterpret_cast<const uint32_t*>(w) + 1;
    const int have = min(n, p.weight_rows);
    for (int i = 0; i < run; i += 64 * U) {
      uint32_t h[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int j = r0 + i + 64 * u + lane;
        h[u] = i + 64 * u < run && j < have ? wh[2 * (size_t)j] : 0u;
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (i + 64 * u >= run) break;   // uniform
        const int j = r0 + i + 64 * u + lane;
        uint32_t k = h[u] | 0x80000000u;
        if (h[u] >= 0x7ff00000u) k = key_of(w[j]).hi;   // below 0, -0, infinite or NaN
        const bool cand = (unsigned)(j - lo) < (unsigned)left;
        big.word[j] = cand ? k : j < n ? kStays : kNone;
        k = cand ? k : 0u;
        most = max(most, k);
        least = min(least, k - (kZero + 1));
      }
    }
  }
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) { most = max(most, __shfl_xor(most, d)); least = min(least, __shfl_xor(least, d)); }
  if (lane == 0) { atomicMax(&sh.any[0], most); atomicMin(&sh.any[1], least); }

  Key edge{kStays - 1, ~0u}, prefix{0, 0}, mask{0, 0};
  bool done = need == 0, sorted = false;   // sorted: the rows that share the edge's high word are told apart
  int pass = 0;
  auto take = [&](int j) {
    const int at = atomicAdd(&sh.nrank, 1);
    if (at < kRank) sh.rpos[at] = j;
  };
  // the need-th of the `left` rows in rpos; `all`: no other row has one of their high words
  auto rank_list = [&](bool all) {
    __syncthreads();
    if (tid < left) sh.rkey[tid] = key_of(weight(sh.rpos[tid]));
    rank_keys(sh, left, need);
    edge = sh.edge;
    need = sh.need;
    done = true;
    if (all) {
      if (tid < left && sh.rkey[tid].hi == edge.hi) {
        const uint32_t l = sh.rkey[tid].lo;
        big.word[sh.rpos[tid]] = l > edge.lo ? kStays : l == edge.lo ? edge.hi : kNone;
      }
      sorted = true;
      __syncthreads();
    }
  };
  // whether one low word is all that the rows of high word prefix.hi have (any is clear)
  auto one_low = [&] {
    uint32_t o = 0, a = ~0u;
    bool has = false;
    lows(prefix.hi, [&](int, uint32_t k) { o |= k; a &= k; has = true; });
    if (one_word(sh.any + 2, o, a, has)) { edge = Key{prefix.hi, sh.any[2]}; done = true; }
  };
  if (!done) {
    __syncthreads();
    most = __builtin_amdgcn_readfirstlane(sh.any[0]);
    if (most > kZero) {
      // first over the range of the positive weights, in up to 2047 even steps of their high
      // words (bin 0: the others), then over 2048 steps of the bin that divides them; a bin
      // of few keys ends the search
      uint32_t base = kZero + 1 + (uint32_t)__builtin_amdgcn_readfirstlane(sh.any[1]);
      int s = max(0, 32 - __clz((int)((most - base) / (kBins - 1))));
      each([&](int, uint32_t k) {
        if (is_word(k)) atomicAdd(&big.hist[k > kZero ? 1 + ((k - base) >> s) : 0], 1);
      });
      find_bin(sh, need, [&](int i) { return big.hist[i]; });
      int bin = __builtin_amdgcn_readfirstlane(sh.found[0]) - 1;
      if (bin < 0) {
        // 0 and below: often one key
        const int above = __builtin_amdgcn_readfirstlane(sh.found[1]);
        clear();
        uint32_t o = 0, x = ~0u;
        bool has = false;
        each([&](int, uint32_t k) {
          if (is_word(k) && k <= kZero) { o |= k; x &= k; has = true; }
        });
        if (one_word(sh.any, o, x, has)) {
          prefix.hi = sh.any[0];
          mask.hi = ~0u;
          need -= above;
          pass = 3;
          one_low();
        }
      }
      while (bin >= 0) {
        need -= __builtin_amdgcn_readfirstlane(sh.found[1]);
        left = __builtin_amdgcn_readfirstlane(sh.found[2]);
        base += (uint32_t)bin << s;
        if (left <= kRank) {
          each([&](int j, uint32_t k) {
            if (is_word(k) && (k - base) >> s == 0) take(j);
          });
          rank_list(true);
          break;
        }
        clear();
        if (s == 0) {   // one high word: on to the low ones
          prefix.hi = base;
          mask.hi = ~0u;
          pass = 3;
          one_low();
          break;
        }
        const int t = max(0, s - 11);
        each([&](int, uint32_t k) {
          if (is_word(k) && (k - base) >> s == 0) atomicAdd(&big.hist[(k - base) >> t], 1);
        });
        find_bin(sh, need, [&](int i) { return big.hist[i]; });
        bin = __builtin_amdgcn_readfirstlane(sh.found[0]);
        s = t;
      }
    }
  }
  for (; !done && pass < 6; ++pass) {
    const bool high = pass < 3;
    const int third = pass % 3, s = third == 0 ? 21 : third == 1 ? 10 : 0;
    const uint32_t digit = third == 2 ? 1023u : 2047u;
    clear();
    if (high)
      each([&](int, uint32_t k) {
        if (is_word(k) && (k & mask.hi) == prefix.hi) atomicAdd(&big.hist[k >> s & digit], 1);
      });
    else
      lows(prefix.hi, [&](int, uint32_t k) {
        if ((k & mask.lo) == prefix.lo) atomicAdd(&big.hist[k >> s & digit], 1);
      });
    find_bin(sh, need, [&](int i) { return big.hist[i]; });
    const uint32_t bin = (uint32_t)__builtin_amdgcn_readfirstlane(sh.found[0]) << s;
    (high ? prefix.hi : prefix.lo) |= bin;
    (high ? mask.hi : mask.lo) |= digit << s;
    need -= __builtin_amdgcn_readfirstlane(sh.found[1]);
    left = __builtin_amdgcn_readfirstlane(sh.found[2]);
    if (need == left) {   // the whole bin stays: every key from its lowest on
      edge = Key{prefix.hi - (prefix.lo == 0), prefix.lo - 1};
      need = 0;
      done = true;
    } else if (left <= kRank) {
      if (high)
        each([&](int j, uint32_t k) {
          if (is_word(k) && (k & mask.hi) == prefix.hi) take(j);
        });
      else
        lows(prefix.hi, [&](int j, uint32_t k) {
          if ((k & mask.lo) == prefix.lo) take(j);
        });
      rank_list(high);
    } else if (high) {
      // one high word alone: on to the low ones, if those are not one as well (weights of 0)
      if (pass < 2) {
        uint32_t o = 0, a = ~0u;
        bool has = false;
        each([&](int, uint32_t k) {
          if (is_word(k) && (k & mask.hi) == prefix.hi) { o |= k; a &= k; has = true; }
        });
        if (one_word(sh.any, o, a, has)) { prefix.hi = sh.any[0]; mask.hi = ~0u; }
      }
      if (mask.hi == ~0u) {
        pass = 2;
        one_low();
      }
    }
  }
  if (!done) edge = prefix;

  // among the rows that share the edge's high word: those above it stay, those below are none
  if (!sorted && (need > 0 || edge.lo != ~0u))
    lows(edge.hi, [&](int j, uint32_t k) { big.word[j] = k > edge.lo ? kStays : k == edge.lo ? edge.hi : kNone; });
  // list: a wave's places follow from the runs before it
  int nk = 0, nt = 0;
  each([&](int, uint32_t k) {
    nk += __popcll(__ballot(k > edge.hi));
    nt += __popcll(__ballot(k == edge.hi));
  });
  __syncthreads();   // wsum is read
  if (lane == 0) { sh.wsum[wave] = nk; sh.wtie[wave] = nt; }
  __syncthreads();
  int pk = before(sh.wsum, wave, lane), pt = before(sh.wtie, wave, lane);
  each([&](int j, uint32_t k) {
    const uint64_t over = __ballot(k > edge.hi), tie = __ballot(k == edge.hi);
    bool stays = k > edge.hi;
    int at = pk + min(pt, need) + lanes_before(over);
    if (tie) {   // uniform
      const int rank = pt + lanes_before(tie);
      at += min(rank, need) - min(pt, need);
      stays |= k == edge.hi && rank < need;
      pt += __popcll(tie);
    }
    if (stays && (unsigned)at < (unsigned)p.budget) kept[at] = j;
    pk += __popcll(over);
  });
}

__global__ void __launch_bounds__(kSelThreads) evict_select_kernel(const EvictParams p) {
  __shared__ union { SelShared few; SelLong many; } big;
  __shared__ SelSmall sh;
  const int tid = threadIdx.x, b = blockIdx.x;
  const int n = __builtin_amdgcn_readfirstlane(max(p.act_kv[b], 0));
  int32_t* kept = p.kept + (size_t)b * p.budget;
  if (n <= p.budget) {
    for (int i = tid; i < p.budget; i += kSelThreads) kept[i] = i < n ? i : -1;
    if (tid == 0) p.act_kv_out[b] = n;
    return;
  }
  const double* w = p.weights + (size_t)b * p.weight_rows;
  if (n <= kRegRows * kSelThreads) select_rows<kRegRows>(p, big.few, sh, n, w, kept);
  else if (n <= kWordRows) select_long(p, big.many, sh, n, w, kept);
  else select_rows<0>(p, big.few, sh, n, w, kept);
  if (tid == 0) p.act_kv_out[b] = p.budget;
}

// 16 LPR bytes of every row; U rows a thread in flight, so that sequences of up to 1024
// U / LPR rows are one chunk: read, one barrier, written. The slices of a sequence lie next
// to each other on one XCD, whose L2 joins the lines that they share, or, where there are
// fewer sequences than XCDs, in `groups` runs on as many of them.
constexpr int kMoveThreads = 1024;
template <int LPR, int U>
__global__ void __launch_bounds__(kMoveThreads) evict_move_kernel(const EvictParams p) {
  constexpr int RPP = kMoveThreads / LPR, CHUNK = RPP * U;
  const int tid = threadIdx.x;
  const int x = (int)(blockIdx.x % (unsigned)p.nxcd), q = (int)(blockIdx.x / (unsigned)p.nxcd);
  const int unit = q / p.run * p.nxcd + x, b = unit / p.groups, slice = unit % p.groups * p.run + q % p.run;
  if (b >= p.B || slice > p.slices) return;
  const int m = p.budget, n = p.act_kv[b];
  if (n <= m) return;
  const int32_t* kept = p.kept + (size_t)b * m;
  if (slice == p.slices) {
    // the weights close up as the rows do; those of the rows that are left behind are 0
    double* w = p.weights + (size_t)b * p.weight_rows;
    constexpr int UW = 8;
    for (int i0 = 0; i0 < m; i0 += kMoveThreads * UW) {
      double v[UW];
#pragma unroll
      for (int u = 0; u < UW; ++u) {
        const int i = i0 + u * kMoveThreads + tid, j = i < m ? kept[i] : n;
        v[u] = (unsigned)j < (unsigned)min(n, p.weight_rows) ? w[j] : 0.;
      }
      __builtin_amdgcn_s_waitcnt(0);
      __syncthreads();   // the chunk's weights are read; later ones lie behind it
#pragma unroll
      for (int u = 0; u < UW; ++u) {
        const int i = i0 + u * kMoveThreads + tid;
        if (i < m && i < p.weight_rows) w[i] = v[u];
      }
    }
    for (int i = m + tid; i < min(n, p.weight_rows); i += kMoveThreads) w[i] = 0.;
    return;
  }
  const int32_t* bt = p.bt + (size_t)b * p.bt_stride;
  const int off = (slice * LPR + tid % LPR) * 16;
  const bool in = off < p.row_bytes;
  // the cache row of position j, -1 where it has no block
  auto place = [&](int j, bool want) {
    const int blk = p.bs_log >= 0 ? j >> p.bs_log : j / p.bs;
    const bool ok = want && blk < p.bt_stride;
    const int ph = ok ? bt[blk] : -1;
    return ph >= 0 && ph < p.nblocks ? ph * p.bs + (j - blk * p.bs) : -1;
  };
  for (int i0 = 0; i0 < m; i0 += CHUNK) {
    u32x4g v[U];
    int src[U], dst[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * RPP + tid / LPR;
      src[u] = in && i < m ? kept[i] : 0;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * RPP + tid / LPR, j = src[u];
      src[u] = place(j, j > i);
      dst[u] = place(i, j > i);
      if (src[u] < 0) dst[u] = -1;
    }
#pragma unroll
    for (int u = 0; u < U; ++u)   // (rows that do not move: row 0's bytes, not written)
      v[u] = *reinterpret_cast<const u32x4g*>(p.cache + (size_t)max(src[u], 0) * p.row_bytes + (in ? off : 0));
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();   // the chunk's rows are read
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (dst[u] >= 0) *reinterpret_cast<u32x4g*>(p.cache + (size_t)dst[u] * p.row_bytes + off) = v[u];
    // the next chunk reads rows behind this one's: no barrier between
  }
}

template <int LPR, int U>
int launch_move(EvictParams p, hipStream_t st) {
  p.groups = std::max(1, p.nxcd / p.B);
  p.slices = (p.row_bytes + 16 * LPR - 1) / (16 * LPR);
  p.run = (p.slices + 1 + p.groups - 1) / p.groups;   // the weights are one more
  const long long blocks = ((long long)p.B * p.groups + p.nxcd - 1) / p.nxcd * p.nxcd * p.run;
  if (blocks > INT_MAX) return set_error(SAS_EINVAL, "evict: %lld workgroups beyond one launch", blocks);
  hipLaunchKernelGGL((evict_move_kernel<LPR, U>), dim3((unsigned)blocks), dim3(kMoveThreads), 0, st, p);
  return SAS_OK;
}

int evict_impl(const SasCacheEvictArgs* a, hipStream_t st) {
  if (a->B < 0 || a->B > 65535) return set_error(SAS_EINVAL, "evict: B must be 0..65535 (got %lld)", (long long)a->B);
  if (a->budget < 1 || a->budget > 1 << 30) return set_error(SAS_EINVAL, "evict: budget must be 1..2^30 (got %lld)", (long long)a->budget);
  if (a->keep_first < 0 || a->keep_recent < 0 || a->keep_first > a->budget || a->keep_recent > a->budget - a->keep_first)
    return set_error(SAS_EINVAL, "evict: keep_first and keep_recent must not be negative and fit the budget (%lld + %lld, %lld)",
                     (long long)a->keep_first, (long long)a->keep_recent, (long long)a->budget);
  if (a->row_bytes < 16 || a->row_bytes % 16 || a->row_bytes > 1 << 20)
    return set_error(SAS_EINVAL, "evict: rows must be a multiple of 16 bytes, at most 1 MiB (got %lld)", (long long)a->row_bytes);
  if (a->weight_rows < 0 || a->weight_rows > 1 << 30)
    return set_error(SAS_EINVAL, "evict: weight_rows must be 0..2^30 (got %lld)", (long long)a->weight_rows);
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
  p.nxcd = device_xcds();
  p.bs_log = (p.bs & (p.bs - 1)) ? -1 : __builtin_ctz(p.bs);
  hipLaunchKernelGGL(evict_select_kernel, dim3((unsigned)p.B), dim3(kSelThreads), 0, st, p);
  // Slices of 64 bytes, or narrower where those leave CUs without work: calls with slices of 64
  // / 32 / 16 bytes, 2048 rows of 1152 bytes of 1 / 8 / 16 / 32 sequences 17.2 / 16.5 / 15.5, 16.4
  // / 18.0 / 18.3 (on the wrong side), 18.6 / 20.7 / 21.8 and 22.1 / 27.1 / 31.4 us, 4 of 4096 rows
  // of 656 49.8 / 44.7 / 42.5.
  const long long quarters = (long long)p.B * ((p.row_bytes + 15) / 16);
  const int rc = quarters >= 4LL * device_cus() ? launch_move<4, 8>(p, st)
               : quarters >= 2LL * device_cus() ? launch_move<2, 8>(p, st) : launch_move<1, 4>(p, st);
  if (rc) return rc;
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
