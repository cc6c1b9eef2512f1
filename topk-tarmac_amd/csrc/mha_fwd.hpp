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
//
// Bounds. Long sequences: MFMA and VALU issue. bf16, 32 heads of 128 on 8192, causal: 540
// to 565 us, 0.97 to 1.02 PFLOP/s where a large library product reaches 1.18; the
// matrix units are busy 52 % of the time. A token over a cache: HBM. bf16, 32 caches
// of up to 8192, 8 key heads of 128: 144 us, 5.0 TB/s. Teams: a wave's own latency
// and VALU. fp32, 256 x 4 heads of 16 on up to 96: 12 us.
#pragma once

#include "heads.hpp"

namespace tarmac {

namespace mha {

constexpr float kLn2 = 0.69314718055994530942f;
constexpr float kMaxSlack = 8.f;  // log2 of how far weights may exceed 1

// Running state of a lane's row: output channels, and maximum and sum of the
// weights (of the lane's half of the keys: halves are added up at the end).
template <typename E, int DP>
struct FwdState {
  using R = Rows<E, DP>;
  static constexpr int KS = R::KS, OB = R::OB;
  f32x16 acc[OB];
  float m = -INFINITY, sum = 0.f;

  __device__ __forceinline__ FwdState() {
#pragma unroll
    for (int n = 0; n < OB; ++n) acc[n] = f32x16{};
  }

  // 32 NB keys from k0, staged as L: K at ka (row_at), V at va (t_at).
  template <typename L, int NB>
  __device__ __forceinline__ void step(const frag_t<E> (&qf)[KS], uint32_t ka, uint32_t va, int k0, const WaveRows& w,
                                       const RowMask& mask, int half, float c) {
    f32x16 s[NB];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) s[nb] = w.start_of(k0 + 32 * nb, half, mask);
    ka = fresh(ka);
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) s[nb] = score_tile<E, DP, L>(ka, 32 * nb, qf, s[nb]);
    float mx = s[0][0];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int e = 0; e < 16; ++e) mx = fmaxf(mx, s[nb][e]);
    mx = max_xor32(mx) * c;
    if (__any(mx > m + kMaxSlack)) {  // m = -inf: the row's first allowed key
      const float mn = fmaxf(m, mx);
      const float f = m == -INFINITY ? 0.f : fast_exp2(m - mn);
      sum *= f;
#pragma unroll
      for (int n = 0; n < OB; ++n) acc[n] *= f;
      m = mn;
    }
    const float off = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        s[nb][e] = fast_exp2(fmaf(s[nb][e], c, -off));
        sum += s[nb][e];
      }
    va = fresh(va);
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) add_product<E, DP, L>(va, 32 * nb, s[nb], acc);
  }
};

// What a row's sums come to: the factor of its output channels, and its
// logsumexp. A row with no key has an output of 0; a sum that is not a number
// stays one.
__device__ __forceinline__ float out_factor(float m, float sum) { return m == -INFINITY && sum == 0.f ? 0.f : 1.f / sum; }
__device__ __forceinline__ float lse_of(float m, float sum) {
  return m == -INFINITY && sum == 0.f ? -INFINITY : kLn2 * (m + __builtin_amdgcn_logf(sum));
}

// The workspace of a call whose keys are divided: each split's sums of each row's
// output channels, then its maximum and sum of weights.
struct Parts {
  float* const part;
  const int64_t all;  // rows
  float2* const ms;
  __device__ __forceinline__ Parts(const MhaArgs& a, int splits)
      : part(static_cast<float*>(a.ws)), all(static_cast<int64_t>(a.B) * a.Hq * a.Nq),
        ms(reinterpret_cast<float2*>(part + splits * all * a.d)) {}
  __device__ __forceinline__ float* row(int split, int64_t row, int d) const { return part + (split * all + row) * d; }
  __device__ __forceinline__ float2& stats(int split, int64_t row) const { return ms[split * all + row]; }
};

template <typename E, int DP>
__device__ __forceinline__ void load_queries(const MhaArgs& a, int b, const WaveRows& w, int half,
                                             frag_t<E> (&qf)[Rows<E, DP>::KS]) {
  const raw_t<E>* const q = static_cast<const raw_t<E>*>(a.q.p) + b * a.q.sb + w.i * a.q.sn + w.head * a.q.sh;
#pragma unroll
  for (int ks = 0; ks < Rows<E, DP>::KS; ++ks)
    qf[ks] = Eight<E>(q + 16 * ks + 8 * half, w.hi > 0 && 16 * ks + 8 * half < a.d).frag();
}

// -- many rows: a workgroup of four waves shares the tiles of K and V ----------
//
// gridDim.y workgroups divide the keys (`chunk` each); with more than one their
// sums are added by mha_fwd_join_kernel.

// Keys a tile in LDS: both buffers of K and V stay within 64 KB, and the parts of
// fp32 heads in registers.
template <typename E, int DP>
constexpr int fwd_keys() { return sizeof(raw_t<E>) == 4 ? 32 : 64; }
// Waves a SIMD whose registers hold the operands and accumulators: teams of narrow
// heads take a few steps each and want as many as there are.
template <typename E, int DP>
constexpr int fwd_waves_per_simd() { return sizeof(raw_t<E>) == 4 && DP > 64 ? 1 : DP == 16 ? 4 : 2; }

constexpr int kFwdWaves = 4;

template <typename E, int DP>
__global__ void __launch_bounds__(64 * kFwdWaves)
    __attribute__((amdgpu_waves_per_eu(fwd_waves_per_simd<E, DP>())))
mha_fwd_kernel(MhaArgs a, int tiles, int chunk, int nblocks, Order order) {
  using R = Rows<E, DP>;
  using L = Staged<E, DP>;
  using raw = raw_t<E>;
  constexpr int NW = kFwdWaves, BN = fwd_keys<E, DP>(), TILE = staged_bytes<E, DP>(BN);
  constexpr bool PARTS = sizeof(raw) == 4;
  extern __shared__ __align__(1024) unsigned char smem[];

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 31, half = lane >> 5;
  int bh, tile;
  tile_of(blockIdx.x, blockIdx.y, gridDim.y, tiles, nblocks, order, bh, tile);
  const int b = __builtin_amdgcn_readfirstlane(bh / a.Hkv), hk = __builtin_amdgcn_readfirstlane(bh - b * a.Hkv);
  const int G = a.Hq / a.Hkv, rows = a.Nq * G;
  const RowMask mask(a, b);
  const float c = uniform_value(a.scale * kLog2eF);
  const int wg0 = (tiles - 1 - tile) * 32 * NW, r0 = wg0 + 32 * wave;  // causal: long rows first
  const int kbeg = blockIdx.y * chunk;
  const int kend = min(__builtin_amdgcn_readfirstlane(WaveRows::end_of(mask, wg0, 32 * NW, rows, G)), kbeg + chunk);
  const WaveRows w(a, mask, hk, r0, col, rows, G);
  frag_t<E> qf[R::KS];
  load_queries<E, DP>(a, b, w, half, qf);

  const raw* const kb = static_cast<const raw*>(a.k.p) + b * a.k.sb + hk * a.k.sh;
  const raw* const vb = static_cast<const raw*>(a.v.p) + b * a.v.sb + hk * a.v.sh;
  std::conditional_t<PARTS, TileSplit<DP, NW>, TileCopy<E, DP, NW, BN>> kc(lane, wave, a.k.sn, a.d),
      vc(lane, wave, a.v.sn, a.d);
  FwdState<E, DP> st;
  const uint32_t lds0 = lds_address(smem), row_at = L::row_at(lane), t_at = TILE + L::t_at(lane);
  // rows from kend on: zeros, what they hold is never used
  if constexpr (PARTS) {
    auto fetch = [&](int k0) {
      kc.fetch(uniform_ptr(kb + k0 * a.k.sn), kend - k0);
      vc.fetch(uniform_ptr(vb + k0 * a.v.sn), kend - k0);
    };
    auto put = [&](uint32_t t) {
      kc.put(t);
      vc.put(t + TILE);
    };
    if (kbeg < kend) {
      fetch(kbeg);
      put(lds0);
      if (kbeg + BN < kend) fetch(kbeg + BN);
    }
    uint32_t at = lds0, other = lds0 + 2 * TILE;
    for (int k0 = kbeg; k0 < kend; k0 += BN) {
      lds_barrier();
      if (k0 + BN < kend) {
        put(other);
        if (k0 + 2 * BN < kend) fetch(k0 + 2 * BN);
      }
      if (k0 < w.kend) st.template step<L, BN / 32>(qf, at + row_at, at + t_at, k0, w, mask, half, c);
      const uint32_t t = at;
      at = other;
      other = t;
    }
  } else {
    auto issue = [&](int k0, unsigned char* t) {
      kc.issue(t, uniform_ptr(kb + k0 * a.k.sn), kend - k0);
      vc.issue(t + TILE, uniform_ptr(vb + k0 * a.v.sn), kend - k0);
    };
    if (kbeg < kend) issue(kbeg, smem);
    int buf = 0;
    for (int k0 = kbeg; k0 < kend; k0 += BN, buf ^= 1) {
      wait_loads();
      lds_barrier();
      if (k0 + BN < kend) issue(k0 + BN, smem + (buf ^ 1) * 2 * TILE);
      const uint32_t at = lds0 + buf * 2 * TILE;
      if (k0 < w.kend) st.template step<L, BN / 32>(qf, at + row_at, at + t_at, k0, w, mask, half, c);
    }
  }

  if (r0 + col >= rows) return;
  const float sum = add_xor32(st.sum);
  const int64_t row = (static_cast<int64_t>(b) * a.Hq + w.head) * a.Nq + w.i;
  if (gridDim.y > 1) {
    const Parts parts(a, gridDim.y);
    const bool some = w.hi > 0 && !(sum == 0.f);  // else the join does not read the part
    if (some) store_row<float, R::OB>(parts.row(blockIdx.y, row, a.d), st.acc, 1.f, half, a.d);
    if (half == 0) parts.stats(blockIdx.y, row) = some ? make_float2(st.m, sum) : make_float2(-INFINITY, 0.f);
    return;
  }
  raw* const o = static_cast<raw*>(a.out.p) + b * a.out.sb + w.i * a.out.sn + w.head * a.out.sh;
  store_row<E, R::OB>(o, st.acc, w.hi > 0 ? out_factor(st.m, sum) : 0.f, half, a.d);
  if (half == 0) a.lse[row] = w.hi > 0 ? lse_of(st.m, sum) : -INFINITY;
}

// -- few rows: the waves of a workgroup share 32 rows, each takes its own keys --
//
// One new token over a cache (its group's heads fill the 32 rows), or too few
// tiles of 128 rows for the chip. A wave copies its own tiles of 32 keys into its
// own two buffers and never waits for another; at the end the waves' sums are
// added in a fixed order. With `splits` > 1 the keys are also divided among that
// many workgroups, whose partial sums mha_fwd_join_kernel adds.

//
// Four waves, or eight on half as many parts where the keys are divided and LDS
// holds their tiles (rows of up to 128 bytes): the sums are added within the workgroup,
// and a cache of up to 1024 keys takes one launch instead of two (two key heads of 64
// on 700 keys: 15.5 -> 12.0 us; 8 of 64 on 32768: 58 -> 38).
template <typename E, int DP>
constexpr int few_waves(bool more) { return Rows<E, DP>::ROWB > 256 ? 2 : more && Rows<E, DP>::ROWB <= 128 ? 8 : 4; }
template <typename E, int DP>
constexpr size_t few_lds(int nw) { return size_t(nw) * 4 * 32 * Rows<E, DP>::ROWB + nw * 64 * 4; }

template <typename E, int DP, int NW>
__global__ void __launch_bounds__(64 * NW)
    __attribute__((amdgpu_waves_per_eu(fwd_waves_per_simd<E, DP>())))
mha_fwd_few_kernel(MhaArgs a, int tiles, int splits, int chunk, int nblocks) {
  using R = Rows<E, DP>;
  using raw = raw_t<E>;
  constexpr int TILE = 32 * R::ROWB, OB = R::OB;
  extern __shared__ __align__(1024) unsigned char smem[];

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 31, half = lane >> 5;
  const int blk = __builtin_amdgcn_readfirstlane(xcd_logical_block(blockIdx.x, nblocks));
  const int split = blk % splits, rest = blk / splits, tile = rest % tiles, bh = rest / tiles;
  const int b = __builtin_amdgcn_readfirstlane(bh / a.Hkv), hk = __builtin_amdgcn_readfirstlane(bh - b * a.Hkv);
  const int G = a.Hq / a.Hkv, rows = a.Nq * G;
  const RowMask mask(a, b);
  const float c = uniform_value(a.scale * kLog2eF);
  const int r0 = 32 * tile;
  const WaveRows w(a, mask, hk, r0, col, rows, G);
  const int kbeg = split * chunk, kend = min(w.kend, kbeg + chunk);  // splits * chunk < Nk + chunk
  frag_t<E> qf[R::KS];
  load_queries<E, DP>(a, b, w, half, qf);

  const raw* const kb = static_cast<const raw*>(a.k.p) + b * a.k.sb + hk * a.k.sh;
  const raw* const vb = static_cast<const raw*>(a.v.p) + b * a.v.sb + hk * a.v.sh;
  const TileCopy<E, DP, 1, 32> kc(lane, 0, a.k.sn, a.d), vc(lane, 0, a.v.sn, a.d);
  unsigned char* const own = smem + wave * 4 * TILE;
  auto issue = [&](int k0, unsigned char* t) {
    kc.issue(t, uniform_ptr(kb + k0 * a.k.sn), kend - k0);
    vc.issue(t + TILE, uniform_ptr(vb + k0 * a.v.sn), kend - k0);
  };

  FwdState<E, DP> st;
  const uint32_t lds0 = lds_address(own), row_at = R::row_at(lane), t_at = TILE + R::t_at(lane);
  const int first = kbeg + 32 * wave;
  if (first < kend) issue(first, own);
  int buf = 0;
  for (int k0 = first; k0 < kend; k0 += 32 * NW, buf ^= 1) {
    wait_loads();
    lds_fence();  // the last tile's reads are done before its buffer is written again
    if (k0 + 32 * NW < kend) issue(k0 + 32 * NW, own + (buf ^ 1) * 2 * TILE);
    const uint32_t at = lds0 + buf * 2 * TILE;
    st.template step<R, 1>(qf, at + row_at, at + t_at, k0, w, mask, half, c);
  }

  float m = st.m, sum = add_xor32(st.sum);
  if constexpr (NW > 1) {
    // each wave's maximum and sum, then its channels at the common maximum
    float* const ms = reinterpret_cast<float*>(smem + NW * 4 * TILE);
    if (half == 0) {
      ms[wave * 64 + col] = m;
      ms[wave * 64 + 32 + col] = sum;
    }
    __syncthreads();
    float mw[NW], total = 0.f;
#pragma unroll
    for (int x = 0; x < NW; ++x) mw[x] = ms[x * 64 + col];
    float mm = mw[0];
#pragma unroll
    for (int x = 1; x < NW; ++x) mm = fmaxf(mm, mw[x]);
#pragma unroll
    for (int x = 0; x < NW; ++x) {
      const float f = mw[x] == -INFINITY ? 0.f : fast_exp2(mw[x] - mm);
      total += ms[x * 64 + 32 + col] * f;
    }
    const float f = m == -INFINITY ? 0.f : fast_exp2(m - mm);
    m = mm;
    sum = total;
    f32x4* const mine = reinterpret_cast<f32x4*>(own);  // 64 lanes x 4 channels of each of 4 OB groups: own tiles' room
#pragma unroll
    for (int q = 0; q < 4 * OB; ++q) {
      const int n = q / 4, e = 4 * (q % 4);
      mine[q * 64 + lane] = f32x4{st.acc[n][e] * f, st.acc[n][e + 1] * f, st.acc[n][e + 2] * f, st.acc[n][e + 3] * f};
    }
    __syncthreads();
  }
  if (r0 + col >= rows) return;
  const int64_t row = (static_cast<int64_t>(b) * a.Hq + w.head) * a.Nq + w.i;
  const bool some = w.hi > 0;
  const float inv = splits > 1 ? 1.f : some ? out_factor(m, sum) : 0.f;
  raw* const o = static_cast<raw*>(a.out.p) + b * a.out.sb + w.i * a.out.sn + w.head * a.out.sh;
  const Parts parts(a, splits);
  // a wave's share of the channels, four at a time
#pragma unroll
  for (int q = 0; q < 4 * OB; q += NW) {
    const int qq = q + wave;
    if (qq >= 4 * OB) break;
    const int ch = 32 * (qq / 4) + 8 * (qq % 4) + 4 * half;  // 32 n + tile_row(4 (q % 4)) + 4 half
    f32x4 x = {};
    if constexpr (NW > 1) {
#pragma unroll
      for (int y = 0; y < NW; ++y) x += reinterpret_cast<const f32x4*>(smem + y * 4 * TILE)[qq * 64 + lane];
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = st.acc[q / 4][4 * (q % 4) + e];
    }
    if (ch >= a.d) continue;
    if (splits > 1) {  // no key: the join does not read it
      if (!(sum == 0.f)) *reinterpret_cast<f32x4*>(parts.row(split, row, a.d) + ch) = x;
    } else {
      x *= inv;
      if constexpr (sizeof(raw) == 4) *reinterpret_cast<f32x4*>(o + ch) = x;
      else *reinterpret_cast<uint2*>(o + ch) = make_uint2(Elem<E>::down2(x[0], x[1]), Elem<E>::down2(x[2], x[3]));
    }
  }
  if (wave == 0 && half == 0) {
    if (splits > 1) parts.stats(split, row) = some ? make_float2(m, sum) : make_float2(-INFINITY, 0.f);
    else
      a.lse[row] = some ? lse_of(m, sum) : -INFINITY;
  }
}

// Adds the partial sums of a row's splits in their order: a thread per four
// channels. Splits without a key (sum 0) are not read.
template <typename E>
__global__ void __launch_bounds__(256) mha_fwd_join_kernel(MhaArgs a, int splits) {
  const int per = a.d / 4;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int64_t row = t / per;
  const Parts parts(a, splits);
  if (row >= parts.all) return;
  const int ch = static_cast<int>(t - row * per) * 4;
  float m = -INFINITY;
  for (int s = 0; s < splits; ++s) m = fmaxf(m, parts.stats(s, row).x);
  float sum = 0.f;
  f32x4 x = {};
#pragma unroll 4
  for (int s = 0; s < splits; ++s) {
    const float2 p = parts.stats(s, row);
    if (p.y == 0.f) continue;
    const float f = p.x == m ? 1.f : fast_exp2(p.x - m);
    sum += p.y * f;
    x += f * *reinterpret_cast<const f32x4*>(parts.row(s, row, a.d) + ch);
  }
  const int i = static_cast<int>(row % a.Nq);
  const int64_t bh = row / a.Nq;
  const int64_t b = bh / a.Hq, h = bh - b * a.Hq;
  x *= out_factor(m, sum);
  raw_t<E>* const o = static_cast<raw_t<E>*>(a.out.p) + b * a.out.sb + i * a.out.sn + h * a.out.sh + ch;
  if constexpr (sizeof(raw_t<E>) == 4) *reinterpret_cast<f32x4*>(o) = x;
  else *reinterpret_cast<uint2*>(o) = make_uint2(Elem<E>::down2(x[0], x[1]), Elem<E>::down2(x[2], x[3]));
  if (ch == 0) a.lse[row] = lse_of(m, sum);
}

template <typename E, int DP>
hipError_t launch_fwd(const MhaArgs& a) {
  const FwdPlan p = fwd_plan(a);
  hipStream_t st = static_cast<hipStream_t>(a.stream);
  const int n = p.tiles * a.B * a.Hkv;
  if (!p.few) {
    constexpr size_t lds = size_t(4) * staged_bytes<E, DP>(fwd_keys<E, DP>());
    hipLaunchKernelGGL((mha_fwd_kernel<E, DP>), dim3(n, p.splits), dim3(64 * kFwdWaves), lds, st, a, p.tiles, p.chunk, n,
                       order_of(a, p.tiles, p.splits));
  } else if (a.Nk <= 32) {
    hipLaunchKernelGGL((mha_fwd_few_kernel<E, DP, 1>), dim3(n), dim3(64), (few_lds<E, DP>(1)), st, a, p.tiles, 1, a.Nk,
                       n);
  } else {
    auto few = [&](auto kernel, int waves) {
      hipLaunchKernelGGL(kernel, dim3(n * p.splits), dim3(64 * waves), (few_lds<E, DP>(waves)), st, a, p.tiles, p.splits,
                         p.chunk, n * p.splits);
    };
    constexpr int LESS = few_waves<E, DP>(false), MOST = few_waves<E, DP>(true);
    if (p.more_waves) few(mha_fwd_few_kernel<E, DP, MOST>, MOST);
    else few(mha_fwd_few_kernel<E, DP, LESS>, LESS);
  }
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || p.splits == 1) return e;
  const int64_t threads = static_cast<int64_t>(a.B) * a.Hq * a.Nq * (a.d / 4);
  hipLaunchKernelGGL((mha_fwd_join_kernel<E>), dim3(static_cast<uint32_t>((threads + 255) / 256)), dim3(256), 0, st, a,
                     p.splits);
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
