// Attention over heads, backward. The probabilities are formed again from q, k
// and the forward's logsumexp, never stored:
//   P = 2^(c q.k - lse log2 e),  D = dO . O,  dS = P (dO V^T - D),
//   dV = P^T dO,  dK = scale dS^T Q,  dQ = scale dS K.
//
//   pass 1, a wave per 32 packed rows (heads.hpp), keys streamed through LDS:
//     S^T = K Q^T, dP^T = V dO^T, dQ^T += K^T dS^T; writes -lse and -D.
//   pass 2, a wave per 32 keys of one key head, the queries of its group's heads
//   streamed, head after head:
//     S = Q K^T, dP = dO V^T, dV^T += dO^T P, dK^T += Q^T dS.
// Two products of the seven are formed twice; in exchange no gradient is summed
// by atomics, and each is the same bits on every run. A shared key head's
// gradient is one sum over the queries of its group.
#pragma once

#include "heads.hpp"

namespace tarmac {

namespace mha {

constexpr int kBwdRows = 32;  // keys (pass 1) or queries (pass 2) a tile in LDS

template <typename E, int DP>
constexpr size_t bwd_lds() { return size_t(4) * kBwdRows * Rows<E, DP>::ROWB + 2 * 2 * kBwdRows * 4; }

// Registers of two waves a SIMD hold the operands and accumulators of the
// 16-bit types; fp32 operands are twice as large.
template <typename E, int DP>
constexpr int bwd_waves() { return sizeof(raw_t<E>) == 4 && DP > 32 ? 1 : 2; }

template <typename E, int DP, int NW>
__global__ void __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(bwd_waves<E, DP>())))
mha_bwd_dq_kernel(MhaArgs a, float2* __restrict__ stats, int tiles, int nblocks) {
  using R = Rows<E, DP>;
  using raw = raw_t<E>;
  constexpr int BN = kBwdRows, KS = R::KS, OB = R::OB, TILE = BN * R::ROWB;
  extern __shared__ __align__(1024) unsigned char smem[];

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 31, half = lane >> 5;
  const int blk = __builtin_amdgcn_readfirstlane(xcd_logical_block(blockIdx.x, nblocks));
  const int bh = blk / tiles, tile = tiles - 1 - (blk - bh * tiles);
  const int b = __builtin_amdgcn_readfirstlane(bh / a.Hkv), hk = __builtin_amdgcn_readfirstlane(bh - b * a.Hkv);
  const int G = a.Hq / a.Hkv, rows = a.Nq * G;
  const RowMask mask(a, b);
  const float c = uniform_value(a.scale * kLog2eF);

  auto end_of = [&](int first, int count) {
    const int i0 = first / G, i1 = min(min(first + count, rows) - 1, mask.q_len * G - 1) / G;
    return first < rows && i1 >= i0 && mask.q_len > 0 ? mask.end(i1) : 0;
  };
  const int wg0 = tile * 32 * NW, r0 = wg0 + 32 * wave;
  const int kend = __builtin_amdgcn_readfirstlane(end_of(wg0, 32 * NW));
  const int wend = __builtin_amdgcn_readfirstlane(end_of(r0, 32));

  const int r = min(r0 + col, rows - 1), i = r / G, g = r - i * G, head = hk * G + g;
  const int hi = mask.end(i), self = mask.self_out ? mask.start + i : -1;
  const int64_t stat = (static_cast<int64_t>(b) * a.Hq + head) * a.Nq + i;
  frag_t<E> qf[KS], gf[KS];
  float nl, nd;  // -lse in the log2 domain, -D
  {
    const raw* const qr = static_cast<const raw*>(a.q.p) + b * a.q.sb + i * a.q.sn + head * a.q.sh;
    const raw* const gr = static_cast<const raw*>(a.dout.p) + b * a.dout.sb + i * a.dout.sn + head * a.dout.sh;
    const raw* const orow = static_cast<const raw*>(a.out.p) + b * a.out.sb + i * a.out.sn + head * a.out.sh;
    const bool live = hi > 0;
    float dd = 0.f;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const int ch = 16 * ks + 8 * half;
      qf[ks] = load_frag<E>(qr + ch, live && ch < a.d);
      gf[ks] = load_frag<E>(gr + ch, live && ch < a.d);
      const frag_t<E> of = load_frag<E>(orow + ch, live && ch < a.d);
#pragma unroll
      for (int e = 0; e < 8; ++e) dd = fmaf(static_cast<float>(gf[ks][e]), static_cast<float>(of[e]), dd);
    }
    dd = add_xor32(dd);
    const float lse = a.lse[stat];
    nl = lse == -INFINITY ? -INFINITY : -lse * kLog2eF;  // an empty row: weights 2^-inf
    nd = -dd;
    if (half == 0 && r0 + col < rows) stats[stat] = make_float2(nl, nd);
  }

  const raw* const kb = static_cast<const raw*>(a.k.p) + b * a.k.sb + hk * a.k.sh;
  const raw* const vb = static_cast<const raw*>(a.v.p) + b * a.v.sb + hk * a.v.sh;
  const TileCopy<E, DP, NW, BN> kc(lane, wave, a.k.sn, a.d), vc(lane, wave, a.v.sn, a.d);
  auto issue = [&](int k0, unsigned char* t) {
    kc.issue(t, uniform_ptr(kb + k0 * a.k.sn), kend - k0);
    vc.issue(t + TILE, uniform_ptr(vb + k0 * a.v.sn), kend - k0);
  };

  f32x16 acc[OB];
#pragma unroll
  for (int n = 0; n < OB; ++n) acc[n] = f32x16{};
  const uint32_t lds0 = lds_address(smem), row_at = R::row_at(lane), t_at = R::t_at(lane);
  if (kend > 0) issue(0, smem);
  int buf = 0;
  for (int k0 = 0; k0 < kend; k0 += BN, buf ^= 1) {
    const uint32_t Ks = lds0 + buf * 2 * TILE;
    wait_loads();
    lds_barrier();
    if (k0 + BN < kend) issue(k0 + BN, smem + (buf ^ 1) * 2 * TILE);
    if (k0 < wend) {
      f32x16 s = {}, dp = {};
      const uint32_t ka = fresh(Ks + row_at);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        s = Elem<E>::mma(R::row_frag(ka, 0, ks), qf[ks], s);
        dp = Elem<E>::mma(R::row_frag(ka + TILE, 0, ks), gf[ks], dp);
      }
      const int base = k0 + 4 * half;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int key = base + tile_row(e);
        const float p = fast_exp2(fmaf(s[e], c, nl));
        s[e] = key < hi && key != self ? p * (dp[e] + nd) : 0.f;
      }
      const uint32_t kt = fresh(Ks + t_at);
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const frag_t<E> df = to_frag<E>(s, t);
#pragma unroll
        for (int n = 0; n < OB; ++n) acc[n] = Elem<E>::mma(R::t_frag(kt, 16 * t, n), df, acc[n]);
      }
    }
  }

  if (r0 + col >= rows) return;
  raw* const o = static_cast<raw*>(a.dq.p) + b * a.dq.sb + i * a.dq.sn + head * a.dq.sh;
  store_row<E, OB>(o, acc, a.scale, half, a.d);
}

template <typename E, int DP, int NW>
__global__ void __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(bwd_waves<E, DP>())))
mha_bwd_dkv_kernel(MhaArgs a, const float2* __restrict__ stats, int tiles, int nblocks) {
  using R = Rows<E, DP>;
  using raw = raw_t<E>;
  constexpr int BN = kBwdRows, KS = R::KS, OB = R::OB, TILE = BN * R::ROWB;
  extern __shared__ __align__(1024) unsigned char smem[];
  unsigned char* const sts = smem + 4 * TILE;  // a tile's -lse, then its -D: two buffers

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 31, half = lane >> 5;
  const int blk = __builtin_amdgcn_readfirstlane(xcd_logical_block(blockIdx.x, nblocks));
  const int bh = blk / tiles, tile = blk - bh * tiles;  // causal: the first keys have the most rows
  const int b = __builtin_amdgcn_readfirstlane(bh / a.Hkv), hk = __builtin_amdgcn_readfirstlane(bh - b * a.Hkv);
  const int G = a.Hq / a.Hkv;
  const RowMask mask(a, b);
  const float c = uniform_value(a.scale * kLog2eF);

  // queries this workgroup (and this wave) comes to: from the first whose place
  // is at or behind the first key, to the end; head after head of the group
  const int wg0 = tile * 32 * NW, k0 = wg0 + 32 * wave;
  const int iend = __builtin_amdgcn_readfirstlane(wg0 < mask.kv_len ? mask.q_len : 0);
  const int ibeg = __builtin_amdgcn_readfirstlane(mask.causal ? min(max(wg0 - mask.start, 0), iend) / BN * BN : 0);
  const int wbeg = __builtin_amdgcn_readfirstlane(
      k0 >= mask.kv_len ? iend + BN : mask.causal ? min(max(k0 - mask.start, 0), iend) : 0);
  const int steps = iend > ibeg ? (iend - ibeg + BN - 1) / BN : 0;

  const int key = k0 + col;
  const bool live = key < mask.kv_len;
  frag_t<E> kf[KS], vf[KS];
  {
    const int64_t kr = min(key, a.Nk - 1);
    const raw* const kp = static_cast<const raw*>(a.k.p) + b * a.k.sb + kr * a.k.sn + hk * a.k.sh;
    const raw* const vp = static_cast<const raw*>(a.v.p) + b * a.v.sb + kr * a.v.sn + hk * a.v.sh;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const int ch = 16 * ks + 8 * half;
      kf[ks] = load_frag<E>(kp + ch, live && ch < a.d);
      vf[ks] = load_frag<E>(vp + ch, live && ch < a.d);
    }
  }

  const TileCopy<E, DP, NW, BN> qc(lane, wave, a.q.sn, a.d), gc(lane, wave, a.dout.sn, a.d);
  auto issue = [&](int g, int i0, int bf) {
    using lds_void = __attribute__((address_space(3))) void;
    const int64_t h = hk * G + g;
    unsigned char* const t = smem + bf * 2 * TILE;
    qc.issue(t, uniform_ptr(static_cast<const raw*>(a.q.p) + b * a.q.sb + h * a.q.sh + i0 * a.q.sn), iend - i0);
    gc.issue(t + TILE, uniform_ptr(static_cast<const raw*>(a.dout.p) + b * a.dout.sb + h * a.dout.sh + i0 * a.dout.sn),
             iend - i0);
    if (wave == 0) {  // 32 rows of two floats; behind the end: zeros, beside rows of zeros
      const float2* const s = uniform_ptr(stats + (b * static_cast<int64_t>(a.Hq) + h) * a.Nq + i0);
      const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(
          const_cast<float2*>(s), 0, min(iend - i0, BN) * 8, 0x00027000);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_void*)(sts + bf * BN * 8), 4, col * 8 + half * 4, 0, 0, 0);
    }
  };

  f32x16 ak[OB], av[OB];
#pragma unroll
  for (int n = 0; n < OB; ++n) ak[n] = av[n] = f32x16{};
  int g = 0, i0 = ibeg, buf = 0;
  const uint32_t lds0 = lds_address(smem), row_at = R::row_at(lane), t_at = R::t_at(lane);
  if (steps > 0) issue(0, ibeg, 0);
  for (int t = steps * G; t > 0; --t, buf ^= 1) {
    const uint32_t Qs = lds0 + buf * 2 * TILE, Gs = Qs + TILE;
    const uint32_t st = lds0 + 4 * TILE + buf * BN * 8 + 16 * half;
    const int at = i0;
    i0 += BN;
    if (i0 >= iend) {
      i0 = ibeg;
      ++g;
    }
    wait_loads();
    lds_barrier();
    if (t > 1) issue(g, i0, buf ^ 1);
    if (at + BN > wbeg) {
      // The products of P before those of dS: what is live between them is one
      // tile, and both accumulators fit two waves a SIMD at the widest heads.
      f32x16 s = {};
      const uint32_t qa = fresh(Qs + row_at);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) s = Elem<E>::mma(R::row_frag(qa, 0, ks), kf[ks], s);
      // a lane's rows: tile_row(e) + 4 half
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        const f32x4 nl = lds_read<f32x4>(st + 4 * tile_row(e));
#pragma unroll
        for (int q = 0; q < 4; ++q) s[e + q] = fast_exp2(fmaf(s[e + q], c, nl[q]));
      }
      // pairs to leave out: keys behind the end, or behind (at) a row's place
      const int p0 = mask.start + at;
      const bool masked = k0 + 32 > mask.kv_len || (mask.causal && k0 + 31 > p0) ||
                          (mask.self_out && k0 <= p0 + BN - 1 && k0 + 31 >= p0);
      const int rel = key - p0 - 4 * half;  // the lane's key, in rows of this tile
      auto leave_out = [&](f32x16& x) {
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (!live || (mask.causal && rel > tile_row(e)) || (mask.self_out && rel == tile_row(e))) x[e] = 0.f;
      };
      if (masked) leave_out(s);
      const uint32_t gt = fresh(Gs + t_at);
#pragma unroll
      for (int t2 = 0; t2 < 2; ++t2) {
        const frag_t<E> pf = to_frag<E>(s, t2);
#pragma unroll
        for (int n = 0; n < OB; ++n) av[n] = Elem<E>::mma(R::t_frag(gt, 16 * t2, n), pf, av[n]);
      }
      __builtin_amdgcn_sched_barrier(0);
      f32x16 dp = {};
      const uint32_t ga = fresh(Gs + row_at);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) dp = Elem<E>::mma(R::row_frag(ga, 0, ks), vf[ks], dp);
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        const f32x4 nd = lds_read<f32x4>(st + 4 * BN + 4 * tile_row(e));
#pragma unroll
        for (int q = 0; q < 4; ++q) s[e + q] *= dp[e + q] + nd[q];
      }
      if (masked) leave_out(s);
      const uint32_t qt = fresh(Qs + t_at);
#pragma unroll
      for (int t2 = 0; t2 < 2; ++t2) {
        const frag_t<E> df = to_frag<E>(s, t2);
#pragma unroll
        for (int n = 0; n < OB; ++n) ak[n] = Elem<E>::mma(R::t_frag(qt, 16 * t2, n), df, ak[n]);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  }

  if (key >= a.Nk) return;
  raw* const ok = static_cast<raw*>(a.dk.p) + b * a.dk.sb + key * a.dk.sn + hk * a.dk.sh;
  raw* const ov = static_cast<raw*>(a.dv.p) + b * a.dv.sb + key * a.dv.sn + hk * a.dv.sh;
  store_row<E, OB>(ok, ak, a.scale, half, a.d);
  store_row<E, OB>(ov, av, 1.f, half, a.d);
}

template <typename E, int DP>
hipError_t launch_bwd(const MhaArgs& a) {
  constexpr int NW = 4;
  constexpr size_t lds = bwd_lds<E, DP>();
  hipStream_t st = static_cast<hipStream_t>(a.stream);
  float2* const stats = static_cast<float2*>(a.ws);  // (-lse, -D) of each row
  const int rows = a.Nq * (a.Hq / a.Hkv);
  const int t1 = (rows + 32 * NW - 1) / (32 * NW), n1 = t1 * a.B * a.Hkv;
  hipLaunchKernelGGL((mha_bwd_dq_kernel<E, DP, NW>), dim3(n1), dim3(64 * NW), lds, st, a, stats, t1, n1);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const int t2 = (a.Nk + 32 * NW - 1) / (32 * NW), n2 = t2 * a.B * a.Hkv;
  hipLaunchKernelGGL((mha_bwd_dkv_kernel<E, DP, NW>), dim3(n2), dim3(64 * NW), lds, st, a, stats, t2, n2);
  return hipGetLastError();
}

template <typename E>
hipError_t run_bwd(const MhaArgs& a) {
  if (a.d <= 16) return launch_bwd<E, 16>(a);
  if (a.d <= 32) return launch_bwd<E, 32>(a);
  if (a.d <= 64) return launch_bwd<E, 64>(a);
  if (a.d <= 96) return launch_bwd<E, 96>(a);
  return launch_bwd<E, 128>(a);
}

}  // namespace mha

}  // namespace tarmac
