// Attention over heads, backward. The probabilities are formed again from q, k
// and the forward's logsumexp, never stored:
//   P = 2^(c q.k - lse log2 e),  D = dO . O,  dS = P (dO V^T - D),
//   dV = P^T dO,  dK = scale dS^T Q,  dQ = scale dS K.
//
//   dQ, a wave per 32 packed rows (heads.hpp), keys streamed through LDS:
//     S^T = K Q^T, dP^T = V dO^T, dQ^T += K^T dS^T;
//   dK and dV, a wave per 32 keys of one key head, the queries of its group's heads
//   streamed, head after head:
//     S = Q K^T, dP = dO V^T, dV^T += dO^T P, dK^T += Q^T dS.
// Two products of the seven are formed twice; in exchange no gradient is summed
// by atomics, each is the same bits on every run, and the two need nothing of each
// other but (-lse, -D), which a small launch before them writes. A shared key head's
// gradient is one sum over the queries of its group.
//
// Bounds: MFMA issue and the dependent chain of a tile (score, exponent, two products).
// bf16, 32 heads of 128 on 4096, causal: 530 us (and 15 of statistics), 0.91 PFLOP/s of
// what is performed; matrix units busy 47 %. fp32, 64 x 4 heads of 32 on up to 256: 52
// us, 29 %, the rest VALU (splits and exponents) and latency at two waves a SIMD.
#pragma once

#include "heads.hpp"

namespace tarmac {

namespace mha {

constexpr int kBwdRows = 32;   // keys (of dQ) or queries a tile in LDS
constexpr int kBwdWaves = 4;

// Rows of up to this many keys: what the rounding of dS leaves goes into dQ and dK too.
// dS = P (dP - D) has two errors of the type's size, its own rounding and that of O
// in D. Over many keys O is small beside V, and so is the second; over few they come
// to more than the rounding of a gradient itself. bf16, causal, 1111 queries: dQ 1.50
// and dK 1.49 times as far off as rounded once, with this 1.32 and 1.30 (every row of
// dQ so: 1.11, but 9 % more time at N=4096, where this takes 1 %).
constexpr int kFewKeys = 128;

// LDS: two buffers of two tiles and a tile's statistics, for each group of waves
// that shares them.
template <typename E, int DP, bool FEW>
constexpr size_t bwd_lds() {
  return size_t(4) * (FEW ? kBwdRows * Rows<E, DP>::ROWB : staged_bytes<E, DP>(kBwdRows)) + 1024;
}

// Most waves of a workgroup that divide the streamed side among them (see below):
// what LDS holds.
template <typename E, int DP>
constexpr int bwd_few_waves() { return Rows<E, DP>::ROWB > 256 ? 2 : Rows<E, DP>::ROWB > 128 ? 4 : 8; }

// Registers of two waves a SIMD hold the operands and accumulators, but for wide
// fp32 heads; where LDS leaves room for one wave a SIMD, it has them all.
template <typename E, int DP, int FEW>
constexpr int bwd_waves() { return DP > (sizeof(raw_t<E>) == 4 ? 32 : FEW > 0 ? 64 : 128) ? 1 : 2; }

// A tensor of the kernel's first argument, read from the kernel's arguments where it
// is used: the compiler otherwise loads all of them at the start and runs out of
// scalar registers to hold them in.
__device__ __forceinline__ HeadsView late_view(size_t offset) {
  using word = const __attribute__((address_space(4))) int64_t;
  uint64_t at = reinterpret_cast<uint64_t>(__builtin_amdgcn_kernarg_segment_ptr()) + offset;
  asm volatile("" : "+s"(at));
  word* const w = reinterpret_cast<word*>(at);
  return {reinterpret_cast<void*>(w[0]), w[1], w[2], w[3]};
}

// Adds the accumulators of a workgroup's waves in their order, through each
// wave's own LDS (`stride` bytes a wave), and stores the row they belong to, or
// this workgroup's part of it in fp32: a wave stores every NW-th group of four
// channels.
template <typename E, int OB, int NW>
__device__ __forceinline__ void add_and_store(unsigned char* smem, int stride, int wave, int lane,
                                              const f32x16 (&acc)[OB], raw_t<E>* row, float* part, bool in, float m,
                                              int d) {
  f32x4* const mine = reinterpret_cast<f32x4*>(smem + wave * stride);
#pragma unroll
  for (int q = 0; q < 4 * OB; ++q) {
    const int n = q / 4, e = 4 * (q % 4);
    mine[q * 64 + lane] = f32x4{acc[n][e], acc[n][e + 1], acc[n][e + 2], acc[n][e + 3]};
  }
  __syncthreads();
#pragma unroll
  for (int q = 0; q < 4 * OB; q += NW) {
    const int qq = q + wave, ch = 32 * (qq / 4) + 8 * (qq % 4) + 4 * (lane >> 5);
    if (qq >= 4 * OB) break;
    f32x4 x = {};
#pragma unroll
    for (int y = 0; y < NW; ++y) x += reinterpret_cast<const f32x4*>(smem + y * stride)[qq * 64 + lane];
    if (!in || ch >= d) continue;
    x *= m;
    if (part) *reinterpret_cast<f32x4*>(part + ch) = x;
    else if constexpr (sizeof(raw_t<E>) == 4) *reinterpret_cast<f32x4*>(row + ch) = x;
    else *reinterpret_cast<uint2*>(row + ch) = make_uint2(Elem<E>::down2(x[0], x[1]), Elem<E>::down2(x[2], x[3]));
  }
  __syncthreads();
}

// One side of the gradient's launch: dQ (tiles of rows against keys) or dK and dV
// (tiles of keys against rows). `splits` workgroups divide the streamed side; with more
// than one their parts are added by mha_bwd_join_kernel.
struct BwdSide {
  float* part;
  int tiles, blocks, splits;  // blocks: workgroups a split
  Order order;
};

// dQ. FEW > 0: that many waves of a workgroup share 32 rows and each takes its own
// tiles of keys, without waiting for the others; used where workgroups of 32 rows
// a wave would not fill the chip.
template <typename E, int DP, int FEW>
__device__ __forceinline__ void bwd_dq(const MhaArgs& a, const float2* __restrict__ stats, const BwdSide& side, int id) {
  using R = Rows<E, DP>;
  using raw = raw_t<E>;
  constexpr bool PARTS = !FEW && sizeof(raw) == 4;
  using L = std::conditional_t<PARTS, PartRows<DP>, R>;
  constexpr int BN = kBwdRows, KS = R::KS, OB = R::OB, TILE = FEW ? BN * R::ROWB : staged_bytes<E, DP>(BN);
  constexpr int NW = FEW ? FEW : kBwdWaves, STEP = FEW ? BN * NW : BN;
  extern __shared__ __align__(1024) unsigned char smem[];

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 31, half = lane >> 5;
  int bh, tile;
  const int splits = side.splits, split = __builtin_amdgcn_readfirstlane(id / side.blocks), tiles = side.tiles;
  float* const part = splits > 1 ? side.part : nullptr;
  tile_of(id - split * side.blocks, split, splits, tiles, side.blocks, side.order, bh, tile);
  const int b = __builtin_amdgcn_readfirstlane(bh / a.Hkv), hk = __builtin_amdgcn_readfirstlane(bh - b * a.Hkv);
  const int G = a.Hq / a.Hkv, rows = a.Nq * G;
  const RowMask mask(a, b);
  const float c = uniform_value(a.scale * kLog2eF);
  const int wg0 = (tiles - 1 - tile) * 32 * (FEW ? 1 : NW), r0 = wg0 + (FEW ? 0 : 32 * wave);
  const WaveRows w(a, mask, hk, r0, col, rows, G);
  int kbeg, kend = FEW ? w.kend : __builtin_amdgcn_readfirstlane(WaveRows::end_of(mask, wg0, 32 * NW, rows, G));
  const int share = ((kend + BN - 1) / BN + splits - 1) / splits * BN;
  kbeg = split * share;
  kend = min(kend, kbeg + share);

  frag_t<E> qf[KS], gf[KS];
  const float2 st = stats[(static_cast<int64_t>(b) * a.Hq + w.head) * a.Nq + w.i];
  const float nl = st.x, nd = st.y;
  {
    const raw* const qr = static_cast<const raw*>(a.q.p) + b * a.q.sb + w.i * a.q.sn + w.head * a.q.sh;
    const raw* const gr = static_cast<const raw*>(a.dout.p) + b * a.dout.sb + w.i * a.dout.sn + w.head * a.dout.sh;
    const bool live = w.hi > 0;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const int ch = 16 * ks + 8 * half;
      qf[ks] = Eight<E>(qr + ch, live && ch < a.d).frag();
      gf[ks] = Eight<E>(gr + ch, live && ch < a.d).frag();
    }
  }

  const raw* const kb = static_cast<const raw*>(a.k.p) + b * a.k.sb + hk * a.k.sh;
  const raw* const vb = static_cast<const raw*>(a.v.p) + b * a.v.sb + hk * a.v.sh;
  std::conditional_t<PARTS, TileSplit<DP, NW>, TileCopy<E, DP, FEW ? 1 : NW, BN>> kc(lane, FEW ? 0 : wave, a.k.sn, a.d),
      vc(lane, FEW ? 0 : wave, a.v.sn, a.d);
  unsigned char* const own = smem + (FEW ? wave * 4 * TILE : 0);
  f32x16 acc[OB];
#pragma unroll
  for (int n = 0; n < OB; ++n) acc[n] = f32x16{};
  const uint32_t lds0 = lds_address(own), row_at = L::row_at(lane), t_at = L::t_at(lane);
  const int first = kbeg + (FEW ? BN * wave : 0);
  auto step = [&](uint32_t Ks, int k0) {
    const f32x16 s0 = w.start_of(k0, half, mask);
    const uint32_t ka = fresh(Ks + row_at);
    f32x16 s = score_tile<E, DP, L>(ka, 0, qf, s0);
    const f32x16 dp = score_tile<E, DP, L>(ka + TILE, 0, gf, f32x16{});
#pragma unroll
    for (int e = 0; e < 16; ++e) s[e] = fast_exp2(fmaf(s[e], c, nl)) * (dp[e] + nd);
    if (sizeof(raw) == 2 && w.kend <= kFewKeys) add_product<E, DP, L>(fresh(Ks + t_at), 0, rounding_of<E>(s), acc);
    add_product<E, DP, L>(fresh(Ks + t_at), 0, s, acc);
  };
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
      if (k0 < w.kend) step(at, k0);
      const uint32_t t = at;
      at = other;
      other = t;
    }
  } else {
    auto issue = [&](int k0, unsigned char* t) {
      kc.issue(t, uniform_ptr(kb + k0 * a.k.sn), kend - k0);
      vc.issue(t + TILE, uniform_ptr(vb + k0 * a.v.sn), kend - k0);
    };
    if (first < kend) issue(first, own);
    int buf = 0;
    for (int k0 = first; k0 < kend; k0 += STEP, buf ^= 1) {
      wait_loads();
      if constexpr (FEW > 0) lds_fence();  // the last tile's reads are done before its buffer is written again
      else lds_barrier();
      if (k0 + STEP < kend) issue(k0 + STEP, own + (buf ^ 1) * 2 * TILE);
      if (FEW || k0 < w.kend) step(lds0 + buf * 2 * TILE, k0);
    }
  }

  const bool in = r0 + col < rows;
  const HeadsView dq = late_view(offsetof(MhaArgs, dq));
  raw* const o = static_cast<raw*>(dq.p) + b * dq.sb + w.i * dq.sn + w.head * dq.sh;
  const float m = w.hi > 0 ? a.scale : 0.f;
  float* p = nullptr;
  if (part) {
    const int64_t row = (static_cast<int64_t>(b) * a.Nq + w.i) * a.Hq + w.head;
    p = part + (static_cast<int64_t>(split) * a.B * a.Nq * a.Hq + row) * a.d;
  }
  if constexpr (FEW > 0) {
    __syncthreads();
    add_and_store<E, OB, NW>(smem, 4 * TILE, wave, lane, acc, o, p, in, m, a.d);
  } else if (in) {
    if (p) store_row<float, OB>(p, acc, m, half, a.d);
    else store_row<E, OB>(o, acc, m, half, a.d);
  }
}

// dK and dV. FEW > 0: that many waves of a workgroup share 32 keys and each takes its own
// tiles of queries.
template <typename E, int DP, int FEW>
__device__ __forceinline__ void bwd_dkv(const MhaArgs& a, const float2* __restrict__ stats, const BwdSide& side, int id) {
  using R = Rows<E, DP>;
  using raw = raw_t<E>;
  constexpr bool PARTS = !FEW && sizeof(raw) == 4;
  using L = std::conditional_t<PARTS, PartRows<DP>, R>;
  constexpr int BN = kBwdRows, KS = R::KS, OB = R::OB, TILE = FEW ? BN * R::ROWB : staged_bytes<E, DP>(BN);
  constexpr int NW = FEW ? FEW : kBwdWaves, STEP = FEW ? NW : 1;
  extern __shared__ __align__(1024) unsigned char smem[];

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 31, half = lane >> 5;
  int bh, tile;
  const int splits = side.splits, split = __builtin_amdgcn_readfirstlane(id / side.blocks), tiles = side.tiles;
  float* const part = splits > 1 ? side.part : nullptr;
  tile_of(id - split * side.blocks, split, splits, tiles, side.blocks, side.order, bh, tile);  // causal: the first keys have the most queries
  const int b = __builtin_amdgcn_readfirstlane(bh / a.Hkv), hk = __builtin_amdgcn_readfirstlane(bh - b * a.Hkv);
  const int G = a.Hq / a.Hkv;
  const RowMask mask(a, b);
  const float c = uniform_value(a.scale * kLog2eF);

  // queries this workgroup (and this wave) comes to: from the first whose place
  // is at or behind the first key, to the end; head after head of the group
  const int wg0 = tile * 32 * (FEW ? 1 : NW), k0 = wg0 + (FEW ? 0 : 32 * wave);
  const int iend = __builtin_amdgcn_readfirstlane(wg0 < mask.kv_len ? mask.q_len : 0);
  const int ibeg = __builtin_amdgcn_readfirstlane(mask.causal ? min(max(wg0 - mask.start, 0), iend) / BN * BN : 0);
  const int wbeg = __builtin_amdgcn_readfirstlane(
      k0 >= mask.kv_len ? iend + BN : mask.causal ? min(max(k0 - mask.start, 0), iend) : 0);
  const int per = iend > ibeg ? (iend - ibeg + BN - 1) / BN : 0;  // tiles a head

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
      kf[ks] = Eight<E>(kp + ch, live && ch < a.d).frag();
      vf[ks] = Eight<E>(vp + ch, live && ch < a.d).frag();
    }
  }

  std::conditional_t<PARTS, TileSplit<DP, NW>, TileCopy<E, DP, FEW ? 1 : NW, BN>> qc(lane, FEW ? 0 : wave, a.q.sn, a.d),
      gc(lane, FEW ? 0 : wave, a.dout.sn, a.d);
  unsigned char* const own = smem + (FEW ? wave * 4 * TILE : 0);
  unsigned char* const sts = smem + (FEW ? NW * 4 * TILE + wave * 1024 : 4 * TILE);  // -lse, -D of a tile: two buffers
  const raw* const qb = static_cast<const raw*>(a.q.p) + b * a.q.sb;
  const raw* const gb = static_cast<const raw*>(a.dout.p) + b * a.dout.sb;
  auto issue_stats = [&](int g, int i0, int bf) {
    using lds_void = __attribute__((address_space(3))) void;
    if (FEW || wave == 0) {  // 32 rows of two floats; behind the end: zeros, beside rows of zeros
      const float2* const s = uniform_ptr(stats + (b * static_cast<int64_t>(a.Hq) + hk * G + g) * a.Nq + i0);
      const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(
          const_cast<float2*>(s), 0, min(iend - i0, BN) * 8, 0x00027000);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_void*)(sts + bf * BN * 8), 4, col * 8 + half * 4, 0, 0, 0);
    }
  };

  f32x16 ak[OB], av[OB];
#pragma unroll
  for (int n = 0; n < OB; ++n) ak[n] = av[n] = f32x16{};
  const int share = (per * G + splits - 1) / splits, first = split * share + (FEW ? wave : 0);
  const int all = min(per * G, (split + 1) * share);
  int g = 0, i0 = ibeg, buf = 0;
  auto advance = [&](int n) {  // by n tiles
    i0 += n * BN;
    while (i0 >= iend) {
      i0 -= per * BN;
      ++g;
    }
  };
  const uint32_t lds0 = lds_address(own), sts0 = lds_address(sts) + 16 * half, row_at = L::row_at(lane),
                 t_at = L::t_at(lane);
  auto step = [&](int buf, int at) {  // the tile of queries from `at`
    const uint32_t Qs = lds0 + buf * 2 * TILE, Gs = Qs + TILE;
    const uint32_t st = sts0 + buf * BN * 8;
    // pairs to leave out: keys behind the end, or behind (at) a row's place
    const int p0 = mask.start + at;
    f32x16 s = {};
    if (k0 + 32 > mask.kv_len || (mask.causal && k0 + 31 > p0) ||
        (mask.self_out && k0 <= p0 + BN - 1 && k0 + 31 >= p0)) {
      asm volatile("");  // a branch: most tiles have nothing to leave out
      const int rel = key - p0 - 4 * half;  // the lane's key, in rows of this tile
      const int low = !live ? 64 : mask.causal ? rel : -64, self = mask.self_out ? rel : -64;
#pragma unroll
      for (int e = 0; e < 16; ++e) s[e] = tile_row(e) < low || tile_row(e) == self ? -INFINITY : 0.f;
    }
    // The products of P before those of dS: what is live between them is one
    // tile, and both accumulators fit two waves a SIMD at the widest heads.
    s = score_tile<E, DP, L>(fresh(Qs + row_at), 0, kf, s);
    // a lane's rows: tile_row(e) + 4 half
#pragma unroll
    for (int e = 0; e < 16; e += 4) {
      const f32x4 nl = lds_read<f32x4>(st + 4 * tile_row(e));
#pragma unroll
      for (int q = 0; q < 4; ++q) s[e + q] = fast_exp2(fmaf(s[e + q], c, nl[q]));
    }
    add_product<E, DP, L>(fresh(Gs + t_at), 0, s, av);
    if constexpr (DP > 64) __builtin_amdgcn_sched_barrier(0);
    const f32x16 dp = score_tile<E, DP, L>(fresh(Gs + row_at), 0, vf, f32x16{});
#pragma unroll
    for (int e = 0; e < 16; e += 4) {
      const f32x4 nd = lds_read<f32x4>(st + 4 * BN + 4 * tile_row(e));
#pragma unroll
      for (int q = 0; q < 4; ++q) s[e + q] *= dp[e + q] + nd[q];
    }
    const bool few_keys = sizeof(raw) == 2 && (mask.causal ? min(p0 + BN, mask.kv_len) : mask.kv_len) <= kFewKeys;
    auto add_rounding = [&] { add_product<E, DP, L>(fresh(Qs + t_at), 0, rounding_of<E>(s), ak); };
    if constexpr (DP > 64) {  // in this order for its registers; up to 64 the other is faster (64 x 8 heads on 256: 72 us, 80)
      __builtin_amdgcn_sched_barrier(0);
      add_product<E, DP, L>(fresh(Qs + t_at), 0, s, ak);
      if (few_keys) add_rounding();
    } else {
      if (few_keys) add_rounding();
      add_product<E, DP, L>(fresh(Qs + t_at), 0, s, ak);
    }
  };
  if constexpr (PARTS) {
    auto fetch = [&] {
      const int64_t h = hk * G + g;
      qc.fetch(uniform_ptr(qb + h * a.q.sh + i0 * a.q.sn), iend - i0);
      gc.fetch(uniform_ptr(gb + h * a.dout.sh + i0 * a.dout.sn), iend - i0);
    };
    auto put = [&](int bf) {
      qc.put(lds0 + bf * 2 * TILE);
      gc.put(lds0 + bf * 2 * TILE + TILE);
    };
    int at = 0;
    if (first < all) {
      advance(first);
      fetch();
      issue_stats(g, i0, 0);
      put(0);
      at = i0;
      if (first + 1 < all) {
        advance(1);
        fetch();
      }
    }
    for (int t = first; t < all; ++t, buf ^= 1) {
      wait_loads();
      lds_barrier();
      const int now = at;
      if (t + 1 < all) {
        put(buf ^ 1);
        issue_stats(g, i0, buf ^ 1);
        at = i0;
        if (t + 2 < all) {
          advance(1);
          fetch();
        }
      }
      if (now + BN > wbeg) step(buf, now);
    }
  } else {
    auto issue = [&](int bf) {
      const int64_t h = hk * G + g;
      unsigned char* const t = own + bf * 2 * TILE;
      qc.issue(t, uniform_ptr(qb + h * a.q.sh + i0 * a.q.sn), iend - i0);
      gc.issue(t + TILE, uniform_ptr(gb + h * a.dout.sh + i0 * a.dout.sn), iend - i0);
      issue_stats(g, i0, bf);
    };
    if (first < all) {
      advance(first);
      issue(0);
    }
    for (int t = first; t < all; t += STEP, buf ^= 1) {
      const int at = i0;
      wait_loads();
      if constexpr (FEW > 0) lds_fence();  // the last tile's reads are done before its buffer is written again
      else lds_barrier();
      if (t + STEP < all) {
        advance(STEP);
        issue(buf ^ 1);
      }
      if (FEW || at + BN > wbeg) step(buf, at);
    }
  }

  const bool in = key < a.Nk;
  const int64_t kr = min(key, a.Nk - 1);
  const HeadsView dk = late_view(offsetof(MhaArgs, dk)), dv = late_view(offsetof(MhaArgs, dv));
  raw* const ok = static_cast<raw*>(dk.p) + b * dk.sb + kr * dk.sn + hk * dk.sh;
  raw* const ov = static_cast<raw*>(dv.p) + b * dv.sb + kr * dv.sn + hk * dv.sh;
  float *pk = nullptr, *pv = nullptr;
  if (part) {
    const int64_t all_rows = static_cast<int64_t>(a.B) * a.Nk * a.Hkv;
    const int64_t row = (static_cast<int64_t>(b) * a.Nk + kr) * a.Hkv + hk;
    pk = part + (2 * split * all_rows + row) * a.d;
    pv = pk + all_rows * a.d;
  }
  if constexpr (FEW > 0) {
    __syncthreads();
    add_and_store<E, OB, NW>(smem, 4 * TILE, wave, lane, ak, ok, pk, in, a.scale, a.d);
    add_and_store<E, OB, NW>(smem, 4 * TILE, wave, lane, av, ov, pv, in, 1.f, a.d);
  } else if (in && part) {
    store_row<float, OB>(pk, ak, a.scale, half, a.d);
    store_row<float, OB>(pv, av, 1.f, half, a.d);
  } else if (in) {
    store_row<E, OB>(ok, ak, a.scale, half, a.d);
    store_row<E, OB>(ov, av, 1.f, half, a.d);
  }
}

// Both in one launch: where teams or causal rows are of several lengths, one fills what
// the other leaves idle. The longer, dK and dV, comes first. (bf16, in two launches
// and in one, with the forward: 8 x 8 heads of 128 on 1024 144 and 122 us, 2 x 4 of 64
// on 2048 62 and 51; 32 of 128 on 4096 679 and 668.)
template <typename E, int DP, int FEW>
__global__ void __launch_bounds__(64 * (FEW ? FEW : kBwdWaves))
    __attribute__((amdgpu_waves_per_eu(bwd_waves<E, DP, FEW>())))
mha_bwd_kernel(MhaArgs a, const float2* __restrict__ stats, BwdSide k, BwdSide q) {
  const int id = blockIdx.x, first = k.blocks * k.splits;
  if (id < first) bwd_dkv<E, DP, FEW>(a, stats, k, id);
  else bwd_dq<E, DP, FEW>(a, stats, q, id - first);
}

// (-lse log2 e, -D) of each row, D = dO . O; (-inf, 0) of rows without a key, whose dO
// and O are not read. A lane takes eight channels, rows in memory's order.
template <typename E, int DP>
__global__ void __launch_bounds__(256) mha_bwd_stats_kernel(MhaArgs a, float2* __restrict__ stats) {
  constexpr int LP = DP <= 16 ? 2 : DP <= 32 ? 4 : DP <= 64 ? 8 : 16;
  using raw = raw_t<E>;
  const int64_t row = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) / LP;
  const int ch = threadIdx.x % LP * 8;
  if (row >= static_cast<int64_t>(a.B) * a.Nq * a.Hq) return;
  const int64_t bn = row / a.Hq;
  const int h = static_cast<int>(row - bn * a.Hq), b = static_cast<int>(bn / a.Nq);
  const int i = static_cast<int>(bn - b * static_cast<int64_t>(a.Nq));
  const bool some = RowMask(a, b).end(i) > 0, in = some && ch < a.d;
  const Eight<E> g(static_cast<const raw*>(a.dout.p) + b * a.dout.sb + i * a.dout.sn + h * a.dout.sh + ch, in);
  const Eight<E> o(static_cast<const raw*>(a.out.p) + b * a.out.sb + i * a.out.sn + h * a.out.sh + ch, in);
  float dd = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) dd = fmaf(g[e], o[e], dd);
  dd = group_sum<LP>(dd);
  const int64_t at = (static_cast<int64_t>(b) * a.Hq + h) * a.Nq + i;
  const float lse = some ? a.lse[at] : -INFINITY;
  if (ch == 0) stats[at] = make_float2(lse == -INFINITY ? -INFINITY : -lse * kLog2eF, -dd);
}

// Adds the parts of one or two gradients' rows in their order: a thread per four
// channels. part: [splits][gridDim.y][rows][d] floats, rows [B, N, H].
template <typename E>
__global__ void __launch_bounds__(256) mha_bwd_join_kernel(HeadsView out0, HeadsView out1, const float* __restrict__ part,
                                                           int splits, int64_t rows, int N, int H, int d) {
  const int per = d / 4;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x, row = t / per;
  if (row >= rows) return;
  const HeadsView& out = blockIdx.y ? out1 : out0;
  const int ch = static_cast<int>(t - row * per) * 4;
  const int64_t stride = gridDim.y * rows * d;
  const float* const p = part + (blockIdx.y * rows + row) * d + ch;
  f32x4 x = *reinterpret_cast<const f32x4*>(p);
#pragma unroll 4
  for (int s = 1; s < splits; ++s) x += *reinterpret_cast<const f32x4*>(p + s * stride);
  const int64_t bn = row / H, b = bn / N;
  raw_t<E>* const o =
      static_cast<raw_t<E>*>(out.p) + b * out.sb + (bn - b * N) * out.sn + (row - bn * H) * out.sh + ch;
  if constexpr (sizeof(raw_t<E>) == 4) *reinterpret_cast<f32x4*>(o) = x;
  else *reinterpret_cast<uint2*>(o) = make_uint2(Elem<E>::down2(x[0], x[1]), Elem<E>::down2(x[2], x[3]));
}

template <typename E, int DP>
hipError_t launch_bwd(const MhaArgs& a) {
  constexpr int MOST = bwd_few_waves<E, DP>(), LESS = MOST > 4 ? 4 : MOST;
  constexpr size_t few_lds = bwd_lds<E, DP, true>(), wide_lds = bwd_lds<E, DP, false>();
  hipStream_t st = static_cast<hipStream_t>(a.stream);
  float2* const stats = static_cast<float2*>(a.ws);
  float* const parts = static_cast<float*>(a.ws) + mha_bwd_stats_floats(a);
  const int heads = a.B * a.Hkv;
  const BwdPlan p = bwd_plan(a);
  auto side = [&](const BwdPass& x, float* part) {
    return BwdSide{part, x.tiles, x.tiles * heads, x.splits, order_of(a, x.tiles, x.splits)};
  };
  const BwdSide q = side(p.dq, parts + p.dkv_floats), k = side(p.dkv, parts), none = {nullptr, 1, 0, 1, kByHead};
  auto waves_of = [&](const BwdPass& x) { return !x.few ? 0 : x.more_waves ? MOST : LESS; };
  auto launch = [&](int few, const BwdSide& kk, const BwdSide& qq) {
    const int waves = few ? few : kBwdWaves;
    const auto wide = mha_bwd_kernel<E, DP, 0>;
    const auto less = mha_bwd_kernel<E, DP, LESS>;
    const auto most = mha_bwd_kernel<E, DP, MOST>;
    hipLaunchKernelGGL(!few ? wide : few == MOST ? most : less,
                       dim3(kk.blocks * kk.splits + qq.blocks * qq.splits), dim3(64 * waves),
                       few ? waves * few_lds : wide_lds, st, a, static_cast<const float2*>(stats), kk, qq);
    return hipGetLastError();
  };
  auto join = [&](const HeadsView& out0, const HeadsView& out1, const float* part, int n, int splits, int N, int H) {
    const int64_t rows = static_cast<int64_t>(a.B) * N * H, threads = rows * (a.d / 4);
    hipLaunchKernelGGL((mha_bwd_join_kernel<E>), dim3(static_cast<uint32_t>((threads + 255) / 256), n), dim3(256), 0, st,
                       out0, out1, part, splits, rows, N, H, a.d);
    return hipGetLastError();
  };
  constexpr int LP = DP <= 16 ? 2 : DP <= 32 ? 4 : DP <= 64 ? 8 : 16;
  const int64_t threads = static_cast<int64_t>(a.B) * a.Nq * a.Hq * LP;
  hipLaunchKernelGGL((mha_bwd_stats_kernel<E, DP>), dim3(static_cast<uint32_t>((threads + 255) / 256)), dim3(256), 0, st, a,
                     stats);
  hipError_t e = hipGetLastError();
  const int wq = waves_of(p.dq), wk = waves_of(p.dkv);
  const int64_t blocks = static_cast<int64_t>(k.blocks) * k.splits + static_cast<int64_t>(q.blocks) * q.splits;
  if (e == hipSuccess && wq == wk && blocks * 64 * (wq ? wq : kBwdWaves) >> 32 == 0) {
    e = launch(wq, k, q);
  } else if (e == hipSuccess) {
    e = launch(wk, k, none);
    if (e == hipSuccess) e = launch(wq, none, q);
  }
  if (e == hipSuccess && p.dq.splits > 1) e = join(a.dq, a.dq, q.part, 1, p.dq.splits, a.Nq, a.Hq);
  if (e == hipSuccess && p.dkv.splits > 1) e = join(a.dk, a.dv, k.part, 2, p.dkv.splits, a.Nk, a.Hkv);
  return e;
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
