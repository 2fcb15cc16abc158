// The key-major pass's narrow tiles of first rows (sas_bwd_pre.hip, sas_bwd_keys_kernel with
// at most 32 first rows): 16 rows of a sequence against a segment of the tokens whose windows
// have left them behind. In a 64-row tile four first rows cost as much as 64 window rows, a
// quarter of the pass for a 128-row window (819 us for the gradients of 4096 tokens of 64
// heads, 576 wide; 755 with narrow tiles). Units are that kernel's, a token's 32 heads, q and
// dO by DMA into its two buffers from the L2 that the window tiles of the same tokens fill:
//   waves 0, 1: S and dP of 16 heads each against the 16 rows (K in registers), P and dS,
//     masked and rounded to the query dtype, to an LDS table [row][head];
//   every wave: dkv[row][ch] += dS^T . Q + P^T . dO for its V channel tiles w, w + 8, w + 16,
//     w + 24, and waves 0 .. 3 a rope tile (16x16x32 MFMA, q / dO by transposed reads).
#pragma once

// (included inside sas_bwd_pre.hip's namespaces)

template <int D, typename QT, typename LQ, typename LO>
__device__ __forceinline__ void first_rows_tile(const BwdParams& bp, LQ& lds_q, LO& lds_o, uint8_t* lds_t0, uint8_t* lds_t1,
                                                float (&lds_h)[2][2][32], uint64_t* lds_r, int b, int qp, int sg0, int a0,
                                                int a1, int p0, int hg) {
  constexpr int CH = D / 8, OCH = kDV / 8, KS = D / 32, VS = kDV / 32;
  constexpr int SGQ = kSwzGroup<CH>, SGO = kSwzGroup<OCH>, TS = 80;
  constexpr bool ROPE = D > kDV;
  const FwdParams& p = bp.f;
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int c16 = lane & 15, g4 = lane >> 4, nhg = p.H / 32, h0 = hg * 32;
  if (tid < kFirstRows) {
    const int pos = p0 + tid, blk = pos / p.ori_bs;
    uint64_t a = 0;
    if (pos < p.first && blk < p.ori_bt_stride) {
      const int phys = p.ori_bt[(size_t)b * p.ori_bt_stride + blk];
      if (phys >= 0 && phys < p.ori_nblocks)
        a = reinterpret_cast<uint64_t>(p.ori_kv) + (uint64_t)(uint32_t)(phys * p.ori_bs + pos - blk * p.ori_bs) * (D * 2);
    }
    lds_r[tid] = a;
  }
  // (a segment has fewer tokens than the workgroup threads)
  const bool nf = __syncthreads_or(
      tid < a1 - a0 && reinterpret_cast<const uint32_t*>(bp.nonfinite)[((size_t)qp + a0 + tid) * nhg + hg] != 0);
  uint4 kf[KS];
  const uint64_t ra = lds_r[c16];
  const bool rok = ra != 0;
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) kf[ks] = rok ? gld16(ra + (32 * ks + 8 * g4) * 2) : make_uint4(0, 0, 0, 0);

  // a unit's (lse, Delta) two units ahead into registers, one ahead into LDS; its q and dO one
  // unit ahead by DMA, as sas_bwd_keys_kernel splits it
  float hv = 0.f;
  auto load_small = [&](int a) {
    if (wave == 0) hv = (lane < 32 ? p.lse : bp.delta)[((size_t)qp + a) * p.H + h0 + (lane & 31)];
  };
  auto put_small = [&](int buf) {
    if (wave == 0) lds_h[buf][lane >> 5][lane & 31] = lane < 32 ? hv * kLog2e : hv;
  };
  constexpr int RI = CH / 8;
  const int Pq = wave * 64 + lane, rq = Pq / CH, Px = 8 * 64 + lane, rx = Px / CH;
  const uint32_t oq = (uint32_t)(rq * CH + ((Pq - rq * CH) ^ swz<CH>(rq))) * 16;
  const uint32_t ox = (uint32_t)(rx * CH + ((Px - rx * CH) ^ swz<CH>(rx))) * 16;
  const uint32_t oo = (uint32_t)(wave * OCH + (lane ^ swz<OCH>(wave))) * 16;
  auto dma = [&](int a, int buf) {
    const size_t t = (size_t)qp + a;
    const uint8_t* qs = p.q + (t * p.H + h0) * D * 2;
    const uint8_t* os = bp.dout + (t * p.H + h0) * kDV * 2;
    const uint32_t qb = lds_addr_of(lds_q[buf]) + wave * 1024, ob = lds_addr_of(lds_o[buf]) + wave * 1024;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      dma16s(oq, qs + j * 8 * D * 2, __builtin_amdgcn_readfirstlane(qb + j * RI * 1024));
      dma16s(oo, os + j * 8 * kDV * 2, __builtin_amdgcn_readfirstlane(ob + j * 8 * 1024));
    }
    if (RI == 9 && wave < 4)
      dma16s(ox, qs + wave * 8 * D * 2, __builtin_amdgcn_readfirstlane(lds_addr_of(lds_q[buf]) + (8 + 9 * wave) * 1024));
  };

  f32x4 acc[4], accr = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int m = 0; m < 4; ++m) acc[m] = accr;
  const float scale = p.scale_log2 / kLog2e;
  const int qsw = swz<CH>(c16), osw = swz<OCH>(c16);
  const int vr = 4 * g4 + (c16 >> 2), vqs = swz<CH>(vr), vos = swz<OCH>(vr), vb = (c16 & 3) >> 1;
  auto trbase = [&](auto RC, int vsw, int ct0) {
    constexpr int rc = decltype(RC)::value, SG = kSwzGroup<rc>;
    const int L = 2 * ct0 + vb;
    return (vr * rc + ((L & -SG) | ((L & (SG - 1)) ^ vsw))) * 16 + (c16 & 1) * 8;
  };
  auto trfrag = [&](const uint4* base, auto RC, int off) {
    constexpr int rc = decltype(RC)::value;
    const char* b0 = reinterpret_cast<const char*>(base) + off;
    const uint2 u0 = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS_AS i16x4*)(b0)));
    const uint2 u1 = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS_AS i16x4*)(b0 + 16 * rc * 16)));
    return make_uint4(u0.x, u0.y, u1.x, u1.y);
  };
  const std::integral_constant<int, CH> QC;
  const std::integral_constant<int, OCH> OC;
  const int tq0 = trbase(QC, vqs, wave), to0 = trbase(OC, vos, wave), tr0 = trbase(QC, vqs, kDV / 16 + (wave & 3));

  load_small(a0);
  put_small(0);
  load_small(min(a0 + 1, a1 - 1));
  dma(a0, 0);
  for (int a = a0; a < a1; ++a) {
    const int buf = (a - a0) & 1;
    __builtin_amdgcn_s_waitcnt(0);   // the unit's q and dO, and every load the compiler tracks
    __builtin_amdgcn_s_barrier();
    const uint4* tq = lds_q[buf];
    const uint4* to = lds_o[buf];
    put_small(buf ^ 1);
    load_small(min(a + 2, a1 - 1));
    dma(min(a + 1, a1 - 1), buf ^ 1);   // (past the last unit it is staged again, into the spare buffer)
    if (wave < 2) {
      const int ht = wave;
      auto qfrag = [&](int ks) {
        const int L = 4 * ks + g4;
        return tq[(16 * ht + c16) * CH + ((L & -SGQ) | ((L & (SGQ - 1)) ^ qsw))];
      };
      auto ofrag = [&](int ks) {
        const int L = 4 * ks + g4;
        return to[(16 * ht + c16) * OCH + ((L & -SGO) | ((L & (SGO - 1)) ^ osw))];
      };
      const f32x4 l2 = *reinterpret_cast<const f32x4*>(&lds_h[buf][0][16 * ht + 4 * g4]);
      const f32x4 dl = *reinterpret_cast<const f32x4*>(&lds_h[buf][1][16 * ht + 4 * g4]);
      f32x4 sc[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}}, dc[2] = {sc[0], sc[0]};
      constexpr int PF = 4;
      auto kq = [](int i) { return (i & 1) * (KS / 2) + i / 2; };
      auto ko = [](int i) { return (i & 1) * (VS / 2) + i / 2; };
      uint4 qa[PF], oa[PF];
#pragma unroll
      for (int i = 0; i < PF; ++i) { qa[i] = qfrag(kq(i)); oa[i] = ofrag(ko(i)); }
#pragma unroll
      for (int i = 0; i < KS; ++i) {
        const uint4 qv = qa[i % PF];
        if (i + PF < KS) qa[i % PF] = qfrag(kq(i + PF));
        sc[i & 1] = mfma32k<QT>(qv, kf[kq(i)], sc[i & 1]);
        if (i < VS) {
          const uint4 ov = oa[i % PF];
          if (i + PF < VS) oa[i % PF] = ofrag(ko(i + PF));
          dc[i & 1] = mfma32k<QT>(ov, kf[ko(i)], dc[i & 1]);
        }
      }
      const f32x4 s_ = sc[0] + sc[1], d_ = dc[0] + dc[1];
      // lane (g4, c16): heads 16 ht + 4 g4 .. + 3 of row c16
      const bool n = rok && p0 + c16 < sg0 + a - p.win_left;
      float pr[4], ds[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        pr[i] = n ? __builtin_amdgcn_exp2f(s_[i] * p.scale_log2 - l2[i]) : 0.f;
        ds[i] = n ? pr[i] * (d_[i] - dl[i]) * scale : 0.f;
      }
      // table position of head 16 ht + 4 g4 + i: 8 g4 + 4 ht + i, the k order of the
      // transposed q / dO reads
      const int at = c16 * TS + (8 * g4 + 4 * ht) * 2;
      *reinterpret_cast<uint2*>(lds_t0 + at) = make_uint2(pack2<QT>(ds[0], ds[1]), pack2<QT>(ds[2], ds[3]));
      *reinterpret_cast<uint2*>(lds_t1 + at) = make_uint2(pack2<QT>(pr[0], pr[1]), pack2<QT>(pr[2], pr[3]));
    }
    lds_barrier();
    if (nf) {   // as in sas_bwd_keys_kernel: the rows that a token does not attend stay finite
      auto clear = [&](uint4* v, int n) {
#pragma unroll 1
        for (int i = tid; i < n; i += 512) {
          const uint4 w = v[i];
          v[i] = make_uint4(finite2<QT>(w.x), finite2<QT>(w.y), finite2<QT>(w.z), finite2<QT>(w.w));
        }
      };
      clear(lds_q[buf], 32 * CH);
      clear(lds_o[buf], 32 * OCH);
      lds_barrier();
    }
    const uint4 ads = *reinterpret_cast<const uint4*>(lds_t0 + c16 * TS + g4 * 16);
    const uint4 ap = *reinterpret_cast<const uint4*>(lds_t1 + c16 * TS + g4 * 16);
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      acc[m] = mfma32k<QT>(ads, trfrag(tq, QC, tq0 + m * 256), acc[m]);
      acc[m] = mfma32k<QT>(ap, trfrag(to, OC, to0 + m * 256), acc[m]);
    }
    if (ROPE && wave < 4) accr = mfma32k<QT>(ads, trfrag(tq, QC, tr0), accr);
  }
  wait_vm<0>();   // the spare unit's DMA
  // lane (g4, c16): rows 4 g4 + i, channel 16 ct + c16
  const uint64_t lo = reinterpret_cast<uint64_t>(p.ori_kv);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint64_t ad = lds_r[4 * g4 + i];
    if (!ad) continue;
    float* gr = bp.d_ori + (ad - lo) / 2 + c16;
#pragma unroll
    for (int m = 0; m < 4; ++m) atomicAdd(gr + (wave + 8 * m) * 16, acc[m][i]);
    if (ROPE && wave < 4) atomicAdd(gr + kDV + wave * 16, accr[i]);
  }
}
