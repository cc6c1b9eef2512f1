// Attention over heads, forward: out = softmax(scale q k^T) v over the keys a
// query is allowed, and the logsumexp of its scaled scores.
//
// A wave owns 32 packed rows (heads.hpp), one a lane pair: scores are formed as
// S^T = K Q^T, so a lane's sixteen results of a tile belong to its own row, the
// running maximum and sum need one exchange (lanes l, l + 32) a tile, and the
// weights are the operand of O^T += V^T P^T as they stand. K and V pass through
// two LDS buffers, one barrier a tile: the next tile is copied while the current
// one is computed on.
//
// The running maximum is only moved when a row's scores exceed it by more than
// 2^8 (the weights are then at most 2^8, far inside every type's range): the
// output registers are rescaled a few times a row instead of once a tile.
#pragma once

#include "heads.hpp"

namespace tarmac {

namespace mha {

constexpr float kLn2 = 0.69314718055994530942f;
constexpr float kMaxSlack = 8.f;  // log2 of how far weights may exceed 1

// Keys a tile in LDS: both buffers of K and V stay within 64 KB.
template <typename E, int DP>
constexpr int fwd_keys() { return Rows<E, DP>::ROWB > 256 ? 32 : 64; }

template <typename E, int DP>
constexpr size_t fwd_lds() { return size_t(4) * fwd_keys<E, DP>() * Rows<E, DP>::ROWB; }

template <typename E, int DP, int NW>
__global__ void __launch_bounds__(64 * NW)
    __attribute__((amdgpu_waves_per_eu(sizeof(raw_t<E>) == 4 && DP > 32 ? 1 : 2)))
mha_fwd_kernel(MhaArgs a, int tiles, int nblocks) {
  using R = Rows<E, DP>;
  using raw = raw_t<E>;
  constexpr int BN = fwd_keys<E, DP>(), NB = BN / 32, KS = R::KS, OB = R::OB, TILE = BN * R::ROWB;
  extern __shared__ __align__(1024) unsigned char smem[];

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 31, half = lane >> 5;
  const int blk = __builtin_amdgcn_readfirstlane(xcd_logical_block(blockIdx.x, nblocks));
  const int bh = blk / tiles, tile = tiles - 1 - (blk - bh * tiles);  // causal: long rows first
  const int b = __builtin_amdgcn_readfirstlane(bh / a.Hkv), hk = __builtin_amdgcn_readfirstlane(bh - b * a.Hkv);
  const int G = a.Hq / a.Hkv, rows = a.Nq * G;
  const RowMask mask(a, b);
  const float c = uniform_value(a.scale * kLog2eF);

  // the keys this workgroup, and this wave, come to: its last query within q_len
  auto end_of = [&](int first, int count) {
    const int i0 = first / G, i1 = min(min(first + count, rows) - 1, mask.q_len * G - 1) / G;
    return first < rows && i1 >= i0 && mask.q_len > 0 ? mask.end(i1) : 0;
  };
  const int wg0 = tile * 32 * NW, r0 = wg0 + 32 * wave;
  const int kend = __builtin_amdgcn_readfirstlane(end_of(wg0, 32 * NW));
  const int wend = __builtin_amdgcn_readfirstlane(end_of(r0, 32));
  // keys below wfull are allowed to every row of the wave (its own place apart);
  // rows behind q_len are not stored from their tiles
  const int i_first = min(r0, rows - 1) / G, i_last = min(r0 + 31, rows - 1) / G;
  const int wfull = __builtin_amdgcn_readfirstlane(
      mask.causal ? max(0, min(mask.kv_len, mask.start + i_first + 1)) : mask.kv_len);

  const int r = min(r0 + col, rows - 1), i = r / G, g = r - i * G, head = hk * G + g;
  const int hi = mask.end(i), self = mask.self_out ? mask.start + i : -1;
  frag_t<E> qf[KS];
  {
    const raw* const qr = static_cast<const raw*>(a.q.p) + b * a.q.sb + i * a.q.sn + head * a.q.sh;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) qf[ks] = load_frag<E>(qr + 16 * ks + 8 * half, 16 * ks + 8 * half < a.d);
  }

  const raw* const kb = static_cast<const raw*>(a.k.p) + b * a.k.sb + hk * a.k.sh;
  const raw* const vb = static_cast<const raw*>(a.v.p) + b * a.v.sb + hk * a.v.sh;
  const TileCopy<E, DP, NW, BN> kc(lane, wave, a.k.sn, a.d), vc(lane, wave, a.v.sn, a.d);
  auto issue = [&](int k0, unsigned char* t) {  // rows from kend on: zeros, what they hold is never used
    kc.issue(t, uniform_ptr(kb + k0 * a.k.sn), kend - k0);
    vc.issue(t + TILE, uniform_ptr(vb + k0 * a.v.sn), kend - k0);
  };

  f32x16 acc[OB];
#pragma unroll
  for (int n = 0; n < OB; ++n) acc[n] = f32x16{};
  float m = -INFINITY, sum = 0.f;  // of this lane's half of the keys: added up at the end

  const uint32_t lds0 = lds_address(smem), row_at = R::row_at(lane), t_at = R::t_at(lane);
  if (kend > 0) issue(0, smem);
  int buf = 0;
  for (int k0 = 0; k0 < kend; k0 += BN, buf ^= 1) {
    const uint32_t Ks = lds0 + buf * 2 * TILE, Vs = Ks + TILE;
    wait_loads();
    lds_barrier();
    if (k0 + BN < kend) issue(k0 + BN, smem + (buf ^ 1) * 2 * TILE);
    if (k0 < wend) {
      f32x16 s[NB];
      const uint32_t ka = fresh(Ks + row_at);
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        s[nb] = f32x16{};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) s[nb] = Elem<E>::mma(R::row_frag(ka, 32 * nb, ks), qf[ks], s[nb]);
      }
      const bool own = mask.self_out && mask.start + i_last >= k0 && mask.start + i_first < k0 + BN;
      if (k0 + BN > wfull || own) {
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          const int base = k0 + 32 * nb + 4 * half;
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const int key = base + tile_row(e);
            if (key >= hi || key == self) s[nb][e] = -INFINITY;
          }
        }
      }
      float mx = s[0][0];
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int e = 0; e < 16; ++e) mx = fmaxf(mx, s[nb][e]);
      mx = max_xor32(mx) * c;
      if (__any(mx > m + kMaxSlack)) {  // -inf: the row's first allowed key
        const float mn = fmaxf(m, mx);
        const float f = m == -INFINITY ? 0.f : fast_exp2(m - mn);
        sum *= f;
#pragma unroll
        for (int n = 0; n < OB; ++n) acc[n] *= f;
        m = mn;
      }
      const float off = m == -INFINITY ? 0.f : m;
      frag_t<E> pf[2 * NB];
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          s[nb][e] = fast_exp2(fmaf(s[nb][e], c, -off));
          sum += s[nb][e];
        }
        pf[2 * nb] = to_frag<E>(s[nb], 0);
        pf[2 * nb + 1] = to_frag<E>(s[nb], 1);
      }
      const uint32_t va = fresh(Vs + t_at);
#pragma unroll
      for (int t = 0; t < 2 * NB; ++t)
#pragma unroll
        for (int n = 0; n < OB; ++n) acc[n] = Elem<E>::mma(R::t_frag(va, 16 * t, n), pf[t], acc[n]);
    }
  }

  if (r0 + col >= rows) return;
  sum = add_xor32(sum);
  const bool some = hi > 0 && m > -INFINITY;
  const bool nan = hi > 0 && !(sum > 0.f || m == -INFINITY);  // a score that is not a number
  const float inv = some ? 1.f / sum : 0.f;
  raw* const o = static_cast<raw*>(a.out.p) + b * a.out.sb + i * a.out.sn + head * a.out.sh;
  if (some || nan) {
    store_row<E, OB>(o, acc, nan ? NAN : inv, half, a.d);
  } else {
#pragma unroll
    for (int n = 0; n < OB; ++n) acc[n] = f32x16{};
    store_row<E, OB>(o, acc, 0.f, half, a.d);
  }
  if (half == 0)
    a.lse[(static_cast<int64_t>(b) * a.Hq + head) * a.Nq + i] =
        some || nan ? kLn2 * (m + __builtin_amdgcn_logf(sum)) : -INFINITY;
}

template <typename E, int DP>
hipError_t launch_fwd(const MhaArgs& a) {
  const int rows = a.Nq * (a.Hq / a.Hkv);
  const int waves = (rows + 31) / 32;
  constexpr size_t lds = fwd_lds<E, DP>();
  hipStream_t st = static_cast<hipStream_t>(a.stream);
  const int tiles = (waves + 3) / 4, n = tiles * a.B * a.Hkv;
  hipLaunchKernelGGL((mha_fwd_kernel<E, DP, 4>), dim3(n), dim3(256), lds, st, a, tiles, n);
  return hipGetLastError();
}

template <typename E>
hipError_t run_fwd(const MhaArgs& a) {
  if (a.d <= 16) return launch_fwd<E, 16>(a);
  if (a.d <= 32) return launch_fwd<E, 32>(a);
  if (a.d <= 64) return launch_fwd<E, 64>(a);
  if (a.d <= 96) return launch_fwd<E, 96>(a);
  return launch_fwd<E, 128>(a);
}

}  // namespace mha

}  // namespace tarmac
