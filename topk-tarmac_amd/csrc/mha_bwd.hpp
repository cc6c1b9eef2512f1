// Attention over heads, backward. The probabilities are formed again from q, k
// and the forward's logsumexp, never stored:
//   P = 2^(c q.k - lse log2 e),  D = dO . O,  dS = P (dO V^T - D),
//   dV = P^T dO,  dK = scale dS^T Q,  dQ = scale dS K.
//
//   pass 1, a wave per 32 packed rows (heads.hpp), keys streamed through LDS:
//     S^T = K Q^T, dP^T = V dO^T, dQ^T += K^T dS^T; writes D.
//   pass 2, a wave per 32 keys of one key head, its packed rows streamed:
//     S = Q K^T, dP = dO V^T, dV^T += dO^T P, dK^T += Q^T dS.
// Two products of the seven are formed twice; in exchange no gradient is summed
// by atomics, and each is the same bits on every run. A shared key head's
// gradient is one sum over the rows of its group.
#pragma once

#include "heads.hpp"

namespace tarmac {

namespace mha {

constexpr int kBwdRows = 32;  // keys (pass 1) or packed rows (pass 2) a tile in LDS

template <typename E, int DP>
constexpr size_t bwd_lds() { return size_t(4) * kBwdRows * Rows<E, DP>::ROWB + 2 * 3 * kBwdRows * 4; }

// Registers of two waves a SIMD hold the operands and accumulators of the
// 16-bit types; fp32 operands are twice as large.
template <typename E, int DP>
constexpr int bwd_waves() { return sizeof(raw_t<E>) == 4 && DP > 32 ? 1 : 2; }

template <typename E, int DP, int NW>
__global__ void __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(bwd_waves<E, DP>())))
mha_bwd_dq_kernel(MhaArgs a, float* __restrict__ delta, int tiles, int nblocks) {
  using R = Rows<E, DP>;
  using raw = raw_t<E>;
  constexpr int BN = kBwdRows, KS = R::KS, OB = R::OB, NT = 64 * NW, CE = 16 / R::SZ;
  constexpr int U = (BN * R::CH + NT - 1) / NT;
  extern __shared__ __align__(16) unsigned char smem[];

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
    if (half == 0 && r0 + col < rows) delta[stat] = dd;
  }

  f32x4 xk[U], xv[U];
  const raw* const kb = static_cast<const raw*>(a.k.p) + b * a.k.sb + hk * a.k.sh;
  const raw* const vb = static_cast<const raw*>(a.v.p) + b * a.v.sb + hk * a.v.sh;
  auto load_tile = [&](int k0) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int e = threadIdx.x + u * NT, row = e / R::CH, ch = e - row * R::CH;
      xk[u] = xv[u] = f32x4{0.f, 0.f, 0.f, 0.f};
      if (row < BN && k0 + row < kend && ch * CE < a.d) {
        xk[u] = *reinterpret_cast<const f32x4*>(kb + static_cast<int64_t>(k0 + row) * a.k.sn + ch * CE);
        xv[u] = *reinterpret_cast<const f32x4*>(vb + static_cast<int64_t>(k0 + row) * a.v.sn + ch * CE);
      }
    }
  };
  auto store_tile = [&](unsigned char* t) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int e = threadIdx.x + u * NT, row = e / R::CH, ch = e - row * R::CH;
      if (row < BN) {
        *reinterpret_cast<f32x4*>(t + R::off(row, ch)) = xk[u];
        *reinterpret_cast<f32x4*>(t + BN * R::ROWB + R::off(row, ch)) = xv[u];
      }
    }
  };

  f32x16 acc[OB];
#pragma unroll
  for (int n = 0; n < OB; ++n) acc[n] = f32x16{};
  if (kend > 0) {
    load_tile(0);
    store_tile(smem);
  }
  int buf = 0;
  for (int k0 = 0; k0 < kend; k0 += BN, buf ^= 1) {
    const unsigned char* const Ks = smem + buf * 2 * BN * R::ROWB;
    const unsigned char* const Vs = Ks + BN * R::ROWB;
    const bool more = k0 + BN < kend;
    if (more) load_tile(k0 + BN);
    lds_barrier();
    if (k0 < wend) {
      f32x16 s = {}, dp = {};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        s = Elem<E>::mma(R::frag(Ks, 0, ks, lane), qf[ks], s);
        dp = Elem<E>::mma(R::frag(Vs, 0, ks, lane), gf[ks], dp);
      }
      const int base = k0 + 4 * half;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int key = base + tile_row(e);
        const float p = fast_exp2(fmaf(s[e], c, nl));
        s[e] = key < hi && key != self ? p * (dp[e] + nd) : 0.f;
      }
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const frag_t<E> df = to_frag<E>(s, t);
#pragma unroll
        for (int n = 0; n < OB; ++n) acc[n] = Elem<E>::mma(R::frag_t32(Ks, 16 * t, n, lane), df, acc[n]);
      }
    }
    if (more) store_tile(smem + (buf ^ 1) * 2 * BN * R::ROWB);
  }

  if (r0 + col >= rows) return;
  raw* const o = static_cast<raw*>(a.dq.p) + b * a.dq.sb + i * a.dq.sn + head * a.dq.sh;
  store_row<E, OB>(o, acc, a.scale, half, a.d);
}

template <typename E, int DP, int NW>
__global__ void __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(bwd_waves<E, DP>())))
mha_bwd_dkv_kernel(MhaArgs a, const float* __restrict__ delta, int tiles, int nblocks) {
  using R = Rows<E, DP>;
  using raw = raw_t<E>;
  constexpr int BN = kBwdRows, KS = R::KS, OB = R::OB, NT = 64 * NW, CE = 16 / R::SZ;
  constexpr int U = (BN * R::CH + NT - 1) / NT;
  extern __shared__ __align__(16) unsigned char smem[];
  float* const stats = reinterpret_cast<float*>(smem + 4 * BN * R::ROWB);  // -lse, -D, place: two buffers

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 31, half = lane >> 5;
  const int blk = __builtin_amdgcn_readfirstlane(xcd_logical_block(blockIdx.x, nblocks));
  const int bh = blk / tiles, tile = blk - bh * tiles;  // causal: the first keys have the most rows
  const int b = __builtin_amdgcn_readfirstlane(bh / a.Hkv), hk = __builtin_amdgcn_readfirstlane(bh - b * a.Hkv);
  const int G = a.Hq / a.Hkv;
  const RowMask mask(a, b);
  const float c = uniform_value(a.scale * kLog2eF);

  // rows this workgroup (and this wave) comes to: from the first query whose
  // place is at or behind the first key, to the end of the queries
  const int wg0 = tile * 32 * NW, k0 = wg0 + 32 * wave;
  const int rend = wg0 < mask.kv_len ? mask.q_len * G : 0;
  const int rbeg = __builtin_amdgcn_readfirstlane(
      mask.causal ? min(max(wg0 - mask.start, 0), mask.q_len) * G / BN * BN : 0);
  const int wbeg = __builtin_amdgcn_readfirstlane(
      k0 >= mask.kv_len ? rend : mask.causal ? min(max(k0 - mask.start, 0), mask.q_len) * G : 0);

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

  f32x4 xq[U], xg[U];
  float xl = 0.f, xd = 0.f;
  int xp = 0;
  const raw* const qb = static_cast<const raw*>(a.q.p) + b * a.q.sb;
  const raw* const gb = static_cast<const raw*>(a.dout.p) + b * a.dout.sb;
  auto load_tile = [&](int row0) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int e = threadIdx.x + u * NT, row = e / R::CH, ch = e - row * R::CH, r = row0 + row;
      xq[u] = xg[u] = f32x4{0.f, 0.f, 0.f, 0.f};
      if (row < BN && r < rend && ch * CE < a.d) {
        const int i = r / G;
        const int64_t h = hk * G + r - i * G;
        xq[u] = *reinterpret_cast<const f32x4*>(qb + i * a.q.sn + h * a.q.sh + ch * CE);
        xg[u] = *reinterpret_cast<const f32x4*>(gb + i * a.dout.sn + h * a.dout.sh + ch * CE);
      }
    }
    if (threadIdx.x < BN) {
      const int r = row0 + threadIdx.x, i = r / G;
      xl = -INFINITY;
      xd = 0.f;
      xp = mask.start + i;
      if (r < rend) {
        const int64_t stat = (static_cast<int64_t>(b) * a.Hq + hk * G + r - i * G) * a.Nq + i;
        const float lse = a.lse[stat];
        xl = lse == -INFINITY ? -INFINITY : -lse * kLog2eF;
        xd = -delta[stat];
      }
    }
  };
  auto store_tile = [&](int bf) {
    unsigned char* const t = smem + bf * 2 * BN * R::ROWB;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int e = threadIdx.x + u * NT, row = e / R::CH, ch = e - row * R::CH;
      if (row < BN) {
        *reinterpret_cast<f32x4*>(t + R::off(row, ch)) = xq[u];
        *reinterpret_cast<f32x4*>(t + BN * R::ROWB + R::off(row, ch)) = xg[u];
      }
    }
    if (threadIdx.x < BN) {
      float* const st = stats + bf * 3 * BN;
      st[threadIdx.x] = xl;
      st[BN + threadIdx.x] = xd;
      reinterpret_cast<int*>(st)[2 * BN + threadIdx.x] = xp;
    }
  };

  f32x16 ak[OB], av[OB];
#pragma unroll
  for (int n = 0; n < OB; ++n) ak[n] = av[n] = f32x16{};
  if (rbeg < rend) {
    load_tile(rbeg);
    store_tile(0);
  }
  int buf = 0;
  for (int row0 = rbeg; row0 < rend; row0 += BN, buf ^= 1) {
    const unsigned char* const Qs = smem + buf * 2 * BN * R::ROWB;
    const unsigned char* const Gs = Qs + BN * R::ROWB;
    const float* const st = stats + buf * 3 * BN;
    const bool more = row0 + BN < rend;
    if (more) load_tile(row0 + BN);
    lds_barrier();
    if (row0 + BN > wbeg) {
      f32x16 s = {}, dp = {};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        s = Elem<E>::mma(R::frag(Qs, 0, ks, lane), kf[ks], s);
        dp = Elem<E>::mma(R::frag(Gs, 0, ks, lane), vf[ks], dp);
      }
      // a lane's rows: 4 half + 8 q + 0 .. 3
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        const f32x4 nl = *reinterpret_cast<const f32x4*>(st + tile_row(e) + 4 * half);
        const f32x4 nd = *reinterpret_cast<const f32x4*>(st + BN + tile_row(e) + 4 * half);
        const int4 pl = *reinterpret_cast<const int4*>(st + 2 * BN + tile_row(e) + 4 * half);
        const int place[4] = {pl.x, pl.y, pl.z, pl.w};
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const bool in = live && !(mask.causal && key > place[q]) && !(mask.self_out && key == place[q]);
          const float p = in ? fast_exp2(fmaf(s[e + q], c, nl[q])) : 0.f;
          s[e + q] = p;
          dp[e + q] = in ? p * (dp[e + q] + nd[q]) : 0.f;
        }
      }
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const frag_t<E> pf = to_frag<E>(s, t), df = to_frag<E>(dp, t);
#pragma unroll
        for (int n = 0; n < OB; ++n) {
          av[n] = Elem<E>::mma(R::frag_t32(Gs, 16 * t, n, lane), pf, av[n]);
          ak[n] = Elem<E>::mma(R::frag_t32(Qs, 16 * t, n, lane), df, ak[n]);
        }
      }
    }
    if (more) store_tile(buf ^ 1);
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
  float* const delta = static_cast<float*>(a.ws);
  const int rows = a.Nq * (a.Hq / a.Hkv);
  const int t1 = (rows + 32 * NW - 1) / (32 * NW), n1 = t1 * a.B * a.Hkv;
  hipLaunchKernelGGL((mha_bwd_dq_kernel<E, DP, NW>), dim3(n1), dim3(64 * NW), lds, st, a, delta, t1, n1);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const int t2 = (a.Nk + 32 * NW - 1) / (32 * NW), n2 = t2 * a.B * a.Hkv;
  hipLaunchKernelGGL((mha_bwd_dkv_kernel<E, DP, NW>), dim3(n2), dim3(64 * NW), lds, st, a, delta, t2, n2);
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
