// Attention over heads ([B, N, H, d] tensors of any strides): element types,
// tiles in LDS, row and mask arithmetic shared by the forward and backward
// kernels.
//
// Rows. The G = Hq / Hkv query heads that share a key head are packed into one
// list of Nq * G rows, row r being head r % G of query r / G: a tile of rows
// reads each key once for the whole group, one new token of a group of heads
// fills a tile's rows, and a key head's gradient is one sum over its rows, with
// no atomics.
//
// Products run on the 32x32x16 matrix instructions of 16-bit types (fp32: on three
// bf16 parts, Elem<float>). Lane l of an
// operand holds column (or row) l % 32 and slots 8 (l / 32) .. + 7. Which element
// of the contraction a slot stands for is free as long as both operands agree: a
// result tile (lane l: column l % 32, rows tile_row(i) + 4 (l / 32)) is, rounded
// to the element type, the second operand of the next product as it stands.
#pragma once

#include <type_traits>

#include "parts.hpp"
#include "tarmac_internal.hpp"

namespace tarmac {

struct F16 {};   // element tags: storage is 16 bits
struct BF16 {};

template <typename E>
struct Elem;

template <>
struct Elem<BF16> {
  using raw = uint16_t;
  using Fr = bf16x8;
  static __device__ __forceinline__ f32x16 mma(Fr a, Fr b, f32x16 c) { return mfma_bf16_32(a, b, c); }
  static __device__ __forceinline__ float up(raw x) { return bf16_to_f32(x); }
  static __device__ __forceinline__ raw down(float x) { return __builtin_bit_cast(raw, static_cast<__bf16>(x)); }
  static __device__ __forceinline__ uint32_t down2(float a, float b) {
    typedef __bf16 pair_t __attribute__((ext_vector_type(2)));
    const pair_t p = {static_cast<__bf16>(a), static_cast<__bf16>(b)};
    return __builtin_bit_cast(uint32_t, p);
  }
};

template <>
struct Elem<F16> {
  using raw = uint16_t;
  using Fr = f16x8;
  static __device__ __forceinline__ f32x16 mma(Fr a, Fr b, f32x16 c) { return mfma_f16_32(a, b, c); }
  static __device__ __forceinline__ float up(raw x) { return static_cast<float>(__builtin_bit_cast(_Float16, x)); }
  static __device__ __forceinline__ raw down(float x) { return __builtin_bit_cast(raw, static_cast<_Float16>(x)); }
  static __device__ __forceinline__ uint32_t down2(float a, float b) {
    const f16x2 p = {static_cast<_Float16>(a), static_cast<_Float16>(b)};
    return __builtin_bit_cast(uint32_t, p);
  }
};

// fp32 operands are three bf16 parts (24 significand bits, fp32's exponent
// range; a value below 2^-110 is held to 2^-133), six of whose nine products are
// formed: what is left out is 2^-24 of the whole, as an fp32 product's rounding.
// Six 16-bit instructions take 192 cycles where eight fp32 ones take 512, and the
// VALU works beside them. The matrix unit cuts what it adds at the accumulator's
// last place, so products go in from the smallest up and long sums are formed in
// tiles of their own, added with rounding (score_tile, add_product).
template <>
struct Elem<float> {
  using raw = float;
  struct Fr {
    bf16x8 hi, mid, lo;
  };
  static __device__ __forceinline__ float up(raw x) { return x; }
  static __device__ __forceinline__ Fr split(const float (&x)[8]) {
    uint32_t h[4], m[4], l[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) split3_dot(x[2 * e], x[2 * e + 1], h[e], m[e], l[e]);
    return {__builtin_bit_cast(bf16x8, h), __builtin_bit_cast(bf16x8, m), __builtin_bit_cast(bf16x8, l)};
  }
  static __device__ __forceinline__ f32x16 low(const Fr& a, const Fr& b, f32x16 c) {
    c = mfma_bf16_32(a.lo, b.hi, c);
    c = mfma_bf16_32(a.hi, b.lo, c);
    c = mfma_bf16_32(a.mid, b.mid, c);
    c = mfma_bf16_32(a.mid, b.hi, c);
    return mfma_bf16_32(a.hi, b.mid, c);
  }
  static __device__ __forceinline__ f32x16 high(const bf16x8& a, const Fr& b, f32x16 c) {
    return mfma_bf16_32(a, b.hi, c);
  }
};

template <typename E>
using raw_t = typename Elem<E>::raw;
template <typename E>
using frag_t = typename Elem<E>::Fr;

// Elements 8 t .. 8 t + 7 of a result tile as an operand. 16-bit types round the
// weights (and score gradients) here, to nearest: a relative error of at most
// half a step a term, as their inputs have; sums and statistics stay in fp32.
template <typename E>
__device__ __forceinline__ frag_t<E> to_frag(const f32x16& w, int t) {
  if constexpr (sizeof(raw_t<E>) == 4) {
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = w[8 * t + e];
    return Elem<E>::split(x);
  } else {
    uint32_t h[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) h[e] = Elem<E>::down2(w[8 * t + 2 * e], w[8 * t + 2 * e + 1]);
    return __builtin_bit_cast(frag_t<E>, h);
  }
}

// Eight elements of a row in global memory; zeros where !in.
template <typename E>
struct Eight {
  typedef raw_t<E> vec __attribute__((ext_vector_type(8)));
  vec v;
  __device__ __forceinline__ Eight(const raw_t<E>* p, bool in) : v{} {
    if (in) v = *reinterpret_cast<const vec*>(p);
  }
  __device__ __forceinline__ float operator[](int e) const { return Elem<E>::up(v[e]); }
  __device__ __forceinline__ frag_t<E> frag() const {
    if constexpr (sizeof(raw_t<E>) == 4) {
      const float x[8] = {v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7]};
      return Elem<E>::split(x);
    } else {
      return __builtin_bit_cast(frag_t<E>, v);
    }
  }
};

// LDS by byte address.
__device__ __forceinline__ uint32_t lds_address(const unsigned char* p) {
  return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((const __attribute__((address_space(3))) unsigned char*)p));
}
template <typename T>
__device__ __forceinline__ T lds_read(uint32_t at) {
  return *(const __attribute__((address_space(3))) T*)(at);
}
// A copy of x that the compiler knows nothing of.
__device__ __forceinline__ uint32_t fresh(uint32_t x) {
  asm volatile("" : "+v"(x));
  return x;
}

// Rows of DP elements in LDS, in 16-byte chunks. Chunk c of row r is stored at
// chunk c ^ swz(r): sixteen rows read at one chunk (the operand read of a row
// per lane) and the 8 rows x 64 bytes of a transposing read both touch each of
// the 64 banks equally often.
template <typename E, int DP>
struct Rows {
  static constexpr int SZ = sizeof(raw_t<E>);
  static constexpr int CH = DP * SZ / 16;                                              // chunks with data
  static constexpr int CHP = CH <= 2 ? 2 : CH <= 4 ? 4 : CH <= 8 ? 8 : CH <= 16 ? 16 : 32;  // stored
  static constexpr int ROWB = CHP * 16;
  static constexpr int KS = DP / 16;                   // contraction steps over the channels
  static constexpr int OB = DP > 32 ? DP / 32 : 1;     // 32-channel blocks of a result

  static __device__ constexpr int swz(int r) {  // exclusive-or of bits of r: swz(r ^ s) = swz(r) ^ swz(s)
    return CHP >= 16  ? ((r & 3) << 2) | ((r >> 2) & 3)
           : CHP == 8 ? (((r >> 1) & 1) << 2) | ((r >> 2) & 3)
           : CHP == 4 ? (r >> 2) & 3
                      : (r >> 3) & 1;
  }
  static __device__ __forceinline__ int off(int r, int c) { return r * ROWB + ((c ^ swz(r)) << 4); }

  // Operand reads. A lane's address within a tile is formed once (row_at, t_at); as
  // tiles start on multiples of 1 KB, a step of the contraction and a block of
  // channels are an exclusive-or of it, rows a constant offset. Kernels pass an
  // opaque copy of the address (fresh) to each use: the compiler otherwise keeps
  // every step's address in a register across the loop.
  //
  // Step ks of the 32 rows from r0: lane l has row l % 32.
  static __device__ __forceinline__ uint32_t row_at(int lane) {
    return off(lane & 31, (SZ == 2 ? 1 : 2) * (lane >> 5));
  }
  static __device__ __forceinline__ frag_t<E> row_frag(uint32_t at, int r0, int ks) {
    if constexpr (SZ == 2) {
      return lds_read<frag_t<E>>((at ^ (ks << 5)) + r0 * ROWB);
    } else {
      const f32x4 a = lds_read<f32x4>((at ^ (ks << 6)) + r0 * ROWB);
      const f32x4 b = lds_read<f32x4>((at ^ (ks << 6) ^ 16) + r0 * ROWB);
      const float x[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
      return Elem<E>::split(x);
    }
  }

  // Operand of the transpose: channels 32 n + l % 32 of the sixteen rows from r0
  // (a multiple of 16), in the row order of a result tile's half: slot 8 (l / 32)
  // + e is row 4 (l / 32) + e, or 8 + 4 (l / 32) + e - 4 from e = 4 on. At DP = 16
  // the upper sixteen lanes repeat the lower ones' channels. 16-bit types: the
  // transposing read, a lane's piece being 8 bytes of row 4 (l / 32) + (l % 16) / 4.
  static __device__ __forceinline__ uint32_t t_at(int lane) {
    const int half = lane >> 5;
    if constexpr (SZ == 2) {
      const int c = (CH > 2 ? 2 * ((lane >> 4) & 1) : 0) + ((lane & 3) >> 1);
      return off(4 * half + ((lane & 15) >> 2), c) + 8 * (lane & 1);
    } else {
      const int ch = DP == 16 ? (lane & 15) : (lane & 31);
      return off(4 * half, ch >> 2) + 4 * (ch & 3);
    }
  }
  static __device__ __forceinline__ frag_t<E> t_frag(uint32_t at, int r0, int n) {
    if constexpr (SZ == 2) {
      using lds_t = __attribute__((address_space(3))) i16x4_t;
      const uint32_t x = at ^ (n << 6), y = x ^ (swz(8) << 4);
      i16x4_t w[2] = {__builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_t*)(x + r0 * ROWB)),
                      __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_t*)(y + (r0 + 8) * ROWB))};
      return __builtin_bit_cast(frag_t<E>, w);
    } else {
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int r = e < 4 ? e : 4 + e;  // from the lane's first row
        x[e] = lds_read<float>((at ^ (n << 7) ^ (swz(r) << 4)) + (r0 + r) * ROWB);
      }
      return Elem<E>::split(x);
    }
  }
};

// A tile of fp32 rows staged as its parts: BN = 32 rows of hi, 32 of mid, 32 of lo,
// each as rows of bf16. Where several waves read a tile, each element is split
// once (TileSplit) instead of in every wave's operand reads, and the operand of
// the transpose comes from transposing reads (gradient of 64 x 4 heads of 32 on
// 256: 90 -> 76 us; attention of 256 x 4 heads of 16 on 96: 16.2 -> 14.3).
template <int DP>
struct PartRows {
  using R = Rows<BF16, DP>;
  static constexpr int KS = R::KS, OB = R::OB, TILE = 3 * 32 * R::ROWB;
  static __device__ __forceinline__ uint32_t row_at(int lane) { return R::row_at(lane); }
  static __device__ __forceinline__ uint32_t t_at(int lane) { return R::t_at(lane); }
  static __device__ __forceinline__ Elem<float>::Fr row_frag(uint32_t at, int r0, int ks) {
    return {R::row_frag(at, r0, ks), R::row_frag(at, r0 + 32, ks), R::row_frag(at, r0 + 64, ks)};
  }
  static __device__ __forceinline__ Elem<float>::Fr t_frag(uint32_t at, int r0, int n) {
    return {R::t_frag(at, r0, n), R::t_frag(at, r0 + 32, n), R::t_frag(at, r0 + 64, n)};
  }
};
// How tiles that a whole workgroup reads are staged.
template <typename E, int DP>
using Staged = std::conditional_t<sizeof(raw_t<E>) == 4, PartRows<DP>, Rows<E, DP>>;
template <typename E, int DP>
constexpr int staged_bytes(int rows) { return sizeof(raw_t<E>) == 4 ? PartRows<DP>::TILE : rows * Rows<E, DP>::ROWB; }

// s + (32 staged rows from r0) . (the lanes' rows q). Pairs to leave out start at
// -inf: the products then stand in one straight line with what reads them. (A
// branch between the two keeps the compiler from moving loads and products past
// each other; and where one stood, it did not add the wait that the read needs.)
template <typename E, int DP, typename R = Rows<E, DP>>
__device__ __forceinline__ f32x16 score_tile(uint32_t at, int r0, const frag_t<E> (&q)[Rows<E, DP>::KS], f32x16 s) {
  if constexpr (sizeof(raw_t<E>) == 4) {
    f32x16 high = {};  // the largest products apart from the others
#pragma unroll
    for (int ks = 0; ks < R::KS; ++ks) {
      const frag_t<E> a = R::row_frag(at, r0, ks);
      s = Elem<E>::low(a, q[ks], s);
      high = Elem<E>::high(a.hi, q[ks], high);
    }
    s += high;
  } else {
#pragma unroll
    for (int ks = 0; ks < R::KS; ++ks) s = Elem<E>::mma(R::row_frag(at, r0, ks), q[ks], s);
  }
  return s;
}

// acc += (32 staged rows from r0)^T . w.
template <typename E, int DP, typename R = Rows<E, DP>>
__device__ __forceinline__ void add_product(uint32_t at, int r0, const f32x16& w, f32x16 (&acc)[Rows<E, DP>::OB]) {
  if constexpr (sizeof(raw_t<E>) == 4 && DP == 16) {  // half by half: registers of four waves a SIMD
    const frag_t<E> w0 = to_frag<E>(w, 0), a0 = R::t_frag(at, r0, 0);
    f32x16 x = Elem<E>::low(a0, w0, f32x16{});
    __builtin_amdgcn_sched_barrier(0);
    const frag_t<E> w1 = to_frag<E>(w, 1), a1 = R::t_frag(at, r0 + 16, 0);
    x = Elem<E>::low(a1, w1, x);
    acc[0] += Elem<E>::high(a1.hi, w1, Elem<E>::high(a0.hi, w0, x));
    return;
  }
  const frag_t<E> w0 = to_frag<E>(w, 0), w1 = to_frag<E>(w, 1);
#pragma unroll
  for (int n = 0; n < R::OB; ++n) {
    if constexpr (sizeof(raw_t<E>) == 4) {
      const frag_t<E> a0 = R::t_frag(at, r0, n), a1 = R::t_frag(at, r0 + 16, n);
      f32x16 x = Elem<E>::low(a1, w1, Elem<E>::low(a0, w0, f32x16{}));
      acc[n] += Elem<E>::high(a1.hi, w1, Elem<E>::high(a0.hi, w0, x));
    } else {
      acc[n] = Elem<E>::mma(R::t_frag(at, r0, n), w0, acc[n]);
    }
  }
  if constexpr (sizeof(raw_t<E>) == 2)
#pragma unroll
    for (int n = 0; n < R::OB; ++n) acc[n] = Elem<E>::mma(R::t_frag(at, r0 + 16, n), w1, acc[n]);
}

// What the rounding of a 16-bit w to an operand leaves of it (nothing of fp32).
template <typename E>
__device__ __forceinline__ f32x16 rounding_of(const f32x16& w) {
  f32x16 left = {};
  if constexpr (sizeof(raw_t<E>) == 2) {
    typedef raw_t<E> raw8 __attribute__((ext_vector_type(8)));
    const raw8 h0 = __builtin_bit_cast(raw8, to_frag<E>(w, 0)), h1 = __builtin_bit_cast(raw8, to_frag<E>(w, 1));
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      left[e] = w[e] - Elem<E>::up(h0[e]);
      left[8 + e] = w[8 + e] - Elem<E>::up(h1[e]);
    }
  }
  return left;
}

// A tile of BN rows copied into LDS without passing through registers: each wave
// moves pieces of 1 KB (64 lanes of 16 bytes), a lane fetching the chunk that
// belongs at its place (Rows::off). Loads go through a buffer descriptor: a lane
// with nothing to fetch (a row from `valid` on, a channel from d on) is given an
// offset behind the descriptor's end, for which the hardware stores zeros. The
// data is there once the issuing waves have waited (wait_loads) and met at a
// barrier.
template <typename E, int DP, int NW, int BN>
struct TileCopy {
  using R = Rows<E, DP>;
  static constexpr int RPP = 1024 / R::ROWB, PIECES = BN / RPP, U = (PIECES + NW - 1) / NW;
  static constexpr uint32_t kSpan = 0x7fffffffu, kNone = 0x80000000u;
  static_assert(BN % RPP == 0, "whole pieces");
  int wave, d, row, chunk;  // the lane's row within a piece, and its chunk at row 0 of a tile
  uint32_t bytes, at;       // of a row's stride; of the lane's row

  // sn: row stride in elements (below 2^31 / 64 bytes: the host checks)
  __device__ __forceinline__ TileCopy(int lane, int wave_, int64_t sn, int d_)
      : wave(wave_), d(d_), row(lane / R::CHP), chunk((lane % R::CHP) ^ R::swz(lane / R::CHP)),
        bytes(static_cast<uint32_t>(sn) * R::SZ), at(row * bytes) {}
  // Offset of the lane's chunk in a piece, whose first row the scalar offset adds.
  __device__ __forceinline__ uint32_t offset(int piece) const {
    return at + ((chunk ^ R::swz(piece * RPP)) << 4);
  }
  __device__ __forceinline__ bool fetched(int piece, int valid) const {
    return piece * RPP + row < valid && (chunk ^ R::swz(piece * RPP)) * (16 / R::SZ) < d;
  }
  __device__ __forceinline__ void issue(unsigned char* tile, const raw_t<E>* base, int valid) const {
    using lds_void = __attribute__((address_space(3))) void;
    const __amdgpu_buffer_rsrc_t rsrc =
        __builtin_amdgcn_make_buffer_rsrc(const_cast<raw_t<E>*>(base), 0, kSpan, 0x00027000);
    auto copy = [&](int piece, uint32_t o) {
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_void*)(tile + piece * 1024), 16, o, piece * RPP * bytes, 0, 0);
    };
    if (valid >= BN && d == DP && R::CH == R::CHP) {
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (PIECES % NW == 0 || u * NW + wave < PIECES) copy(u * NW + wave, offset(u * NW + wave));
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (PIECES % NW == 0 || u * NW + wave < PIECES)
          copy(u * NW + wave, fetched(u * NW + wave, valid) ? offset(u * NW + wave) : kNone);
    }
  }
};

// The same for fp32 rows staged as parts: fetched into registers, and a tile later
// split and stored (PartRows).
template <int DP, int NW>
struct TileSplit {
  using R = Rows<BF16, DP>;
  static constexpr int PER = Rows<float, DP>::CHP, RPP = 64 / PER, PIECES = 32 / RPP, U = (PIECES + NW - 1) / NW;
  static constexpr uint32_t kSpan = 0x7fffffffu, kNone = 0x80000000u;
  int wave, d, row, chunk;  // four channels
  uint32_t bytes, from, to;
  f32x4 x[U];

  __device__ __forceinline__ TileSplit(int lane, int wave_, int64_t sn, int d_)
      : wave(wave_), d(d_), row(lane / PER), chunk(lane % PER), bytes(static_cast<uint32_t>(sn) * 4),
        from(row * bytes + (chunk << 4)), to(R::off(row, chunk >> 1) + 8 * (chunk & 1)) {}
  __device__ __forceinline__ bool there(int piece) const { return PIECES % NW == 0 || piece < PIECES; }
  __device__ __forceinline__ void fetch(const float* base, int valid) {
    const __amdgpu_buffer_rsrc_t rsrc =
        __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(base), 0, kSpan, 0x00027000);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int piece = u * NW + wave;
      if (!there(piece)) continue;
      const uint32_t o = piece * RPP + row < valid && 4 * chunk < d ? from : kNone;
      x[u] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rsrc, o, piece * RPP * bytes, 0));
    }
  }
  __device__ __forceinline__ void put(uint32_t tile) const {
    typedef uint32_t pair_t __attribute__((ext_vector_type(2)));
    using lds_t = __attribute__((address_space(3))) pair_t;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int piece = u * NW + wave;
      if (!there(piece)) continue;
      uint32_t hi[2], mid[2], lo[2];
      split3_dot(x[u][0], x[u][1], hi[0], mid[0], lo[0]);
      split3_dot(x[u][2], x[u][3], hi[1], mid[1], lo[1]);
      const uint32_t p = tile + (to ^ (R::swz(piece * RPP) << 4)) + piece * RPP * R::ROWB;
      *(lds_t*)(p) = pair_t{hi[0], hi[1]};
      *(lds_t*)(p + 32 * R::ROWB) = pair_t{mid[0], mid[1]};
      *(lds_t*)(p + 64 * R::ROWB) = pair_t{lo[0], lo[1]};
    }
  }
};

// Orders this wave's LDS reads before what follows.
__device__ __forceinline__ void lds_fence() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup", "local"); }

// This wave's loads have arrived.
__device__ __forceinline__ void wait_loads() { __builtin_amdgcn_s_waitcnt(0x0f70); }  // vmcnt(0)

// A wave-uniform pointer in scalar registers.
template <typename T>
__device__ __forceinline__ T* uniform_ptr(T* p) {
  return reinterpret_cast<T*>(uniform_offset(reinterpret_cast<size_t>(p)));
}

// A row's elements 32 n + tile_row(i) + 4 half of acc, times m, to p (a row of d
// elements, four at a time).
template <typename E, int OB>
__device__ __forceinline__ void store_row(raw_t<E>* p, const f32x16 (&acc)[OB], float m, int half, int d) {
#pragma unroll
  for (int n = 0; n < OB; ++n)
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      const int c = 32 * n + tile_row(i) + 4 * half;
      if (c >= d) continue;
      if constexpr (sizeof(raw_t<E>) == 4) {
        *reinterpret_cast<f32x4*>(p + c) =
            f32x4{acc[n][i] * m, acc[n][i + 1] * m, acc[n][i + 2] * m, acc[n][i + 3] * m};
      } else {
        *reinterpret_cast<uint2*>(p + c) = make_uint2(Elem<E>::down2(acc[n][i] * m, acc[n][i + 1] * m),
                                                      Elem<E>::down2(acc[n][i + 2] * m, acc[n][i + 3] * m));
      }
    }
}

// Which key head and tile this workgroup takes. By tile (every key head's first
// tile, then every second one) the longest tiles of a causal call start first and
// a padded batch's short rows spread over the chip; by key head, in runs of
// consecutive ones on one XCD, the tiles at work on an XCD share its L2's copy of
// K and V. Where `splits` workgroups divide the streamed side and all are at work at
// once, two a CU, the later half of them takes the tiles from the other end: a CU
// then has a long and a short one (bf16 of 2048 tokens, 16 heads of 64 on 4, causal:
// 34.2 -> 31.0 us forward; with too few workgroups for that it costs 12 %).
enum Order { kByHead, kByTile, kByTileBothEnds };
__device__ __forceinline__ void tile_of(int id, int split, int splits, int tiles, int nblocks, Order order, int& bh,
                                        int& tile) {
  if (order != kByHead) {
    const int heads = nblocks / tiles;
    tile = __builtin_amdgcn_readfirstlane(id / heads);
    bh = __builtin_amdgcn_readfirstlane(id - tile * heads);
    if (order == kByTileBothEnds && 2 * split >= splits) tile = tiles - 1 - tile;
  } else {
    const int blk = __builtin_amdgcn_readfirstlane(xcd_logical_block(id, nblocks));
    bh = blk / tiles;
    tile = blk - bh * tiles;
  }
}
// By tile as long as the K and V (or Q and dO) that an XCD's share of the heads
// reads stay within twice its 4 MB of L2. Either side of it, bf16 heads of 128 in
// causal order, by key head against by tile: 32 of N=4096 with their gradient (twice
// the L2) 811 and 650 us, 32 of N=8192 forward (four times) 549 and 564.
inline Order order_of(const MhaArgs& a, int tiles, int splits) {
  const int64_t heads = static_cast<int64_t>(a.B) * a.Hkv, n = a.Nk > a.Nq ? a.Nk : a.Nq;
  const int64_t bytes = 2 * n * a.d * (a.dtype == kF32 ? 4 : 2);
  if (tiles == 1 || (heads + 7) / 8 * bytes > int64_t(8) << 20) return kByHead;
  return splits > 1 && heads * tiles * splits >= 512 ? kByTileBothEnds : kByTile;
}

// What a batch row's mask allows, in scalars.
struct RowMask {
  int kv_len, q_len, start;
  bool causal, self_out;

  __device__ __forceinline__ RowMask(const MhaArgs& a, int b) {
    kv_len = a.lengths ? min(max(a.lengths[b], 0), a.Nk) : a.Nk;
    q_len = a.q_lengths ? min(max(a.q_lengths[b], 0), a.Nq) : a.Nq;
    start = a.q_start ? min(max(a.q_start[b], -kFar), kFar) : 0;
    causal = a.causal != 0;
    self_out = a.exclude_self != 0;
  }
  // keys 0 .. end(i) - 1 are before query i's end, its own place apart
  __device__ __forceinline__ int end(int i) const {
    if (i >= q_len) return 0;
    return causal ? max(0, min(kv_len, start + i + 1)) : kv_len;
  }
  static constexpr int kFar = 1 << 30;  // positions are clamped to +- 2^30: sums stay in 32 bits
};

// A wave's 32 rows: which keys they come to.
struct WaveRows {
  int kend;     // of the wave: keys from here on are no row's
  int full;     // keys below are allowed to every row, its own place apart
  int p0, p1;   // places of the first and last row's query
  // the lane's row
  int i, head;
  int hi, self;  // its allowed keys are below hi and are not self

  // rows from r0 on, of a list of `rows`; keys a workgroup of `count` rows comes to
  static __device__ __forceinline__ int end_of(const RowMask& m, int r0, int count, int rows, int G) {
    const int i1 = min(min(r0 + count, rows) - 1, m.q_len * G - 1) / G;
    return r0 < rows && m.q_len > 0 && i1 >= r0 / G ? m.end(i1) : 0;
  }
  __device__ __forceinline__ WaveRows(const MhaArgs& a, const RowMask& m, int hk, int r0, int col, int rows, int G) {
    kend = __builtin_amdgcn_readfirstlane(end_of(m, r0, 32, rows, G));
    const int i0 = min(r0, rows - 1) / G;
    p0 = m.start + i0;
    p1 = m.start + min(r0 + 31, rows - 1) / G;
    full = __builtin_amdgcn_readfirstlane(m.causal ? max(0, min(m.kv_len, p0 + 1)) : m.kv_len);
    const int r = min(r0 + col, rows - 1);
    i = r / G;
    head = hk * G + r - i * G;
    hi = m.end(i);
    self = m.self_out ? m.start + i : -1;
  }
  // Where the scores of 32 keys from k0 start: 0, or -inf for those that the
  // lane's row is not allowed.
  __device__ __forceinline__ f32x16 start_of(int k0, int half, const RowMask& m) const {
    f32x16 s = {};
    if (k0 + 32 > full || (m.self_out && p1 >= k0 && p0 < k0 + 32)) {
      asm volatile("");  // a branch: most tiles have nothing to leave out
      const int below = hi - (k0 + 4 * half), own = self - (k0 + 4 * half);
#pragma unroll
      for (int e = 0; e < 16; ++e) s[e] = tile_row(e) >= below || tile_row(e) == own ? -INFINITY : 0.f;
    }
    return s;
  }
};

}  // namespace tarmac
