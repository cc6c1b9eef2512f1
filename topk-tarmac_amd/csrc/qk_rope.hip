// Norm and position rotation of queries and keys per head, and its gradient.
//
//   y = x * rsqrt(mean(x^2) + eps) * w                       (where w is given)
//   z_j = y_j cos_j - y_{j+h} sin_j,  z_{j+h} = y_{j+h} cos_j + y_j sin_j,
//   j < h = rot / 2; channels from rot on pass as they are   (where a table is)
// and, with dy the rotation of dz by the opposite angle, g = dy w, n = x rstd,
//   dx = rstd (g - n mean(g n)),  dw = sum dy n over tokens and heads.
// Everything between the inputs and the one rounding of an output is fp32.
//
// HBM bound: 2 (forward) or 3 (backward) bytes moved a byte of q and k, a few
// VALU each. A head is spread over LP lanes, 2 V channels each: V of the
// rotation's lower half and the V they turn with, so a rotation needs no other
// lane, and the norm one sum over the lanes. V = 8 (16-byte accesses of 16-bit
// types) where widths allow, else 4. A wave takes a token's queries or its keys
// (several tokens', where there are fewer heads than the wave has room for): the
// token's angles are read once for them. One launch does both, workgroups of
// queries first. bf16, 4 x 4096 tokens of 32 + 8 heads of 128: 69 us forward (4.9 TB/s),
// 105 with gradient of everything (4.8 TB/s), where a large copy reaches 5.16.
#include "heads.hpp"

namespace tarmac {

namespace {

constexpr int kThreads = 256;
constexpr int kBwdBlocks = 1024;  // most workgroups of the gradient a side: each leaves one partial sum of the weight's

// One side, queries or keys, and how its heads lie on lanes: a wave takes gp
// (a power of two) heads at once of each of `per` tokens.
struct Side {
  HeadsView x, z, dx;  // input, output (or its gradient), gradient
  const void* w;
  int heads, gp, per, blocks;
};

// Where a lane stands: channels o1 .. + V - 1 and o2 .. + V - 1 of every gp-th
// head, from head h0 on, of one of the wave's tokens.
template <int V, int LP>
struct Lane {
  int c, o1, o2, h0, tok;
  bool chan, turns;
  __device__ __forceinline__ Lane(const RopeArgs& a, int lane, int gp) {
    c = lane % LP;
    const int grp = lane / LP;
    h0 = grp & (gp - 1);
    tok = grp / gp;
    chan = 2 * V * c < a.d;
    turns = a.table != nullptr && 2 * V * c < a.rot;
    o1 = turns ? V * c : 2 * V * c;
    o2 = turns ? a.rot / 2 + V * c : 2 * V * c + V;
  }
};

template <int V>
struct Floats {
  f32x4 x[V / 4];
};

template <typename E, int V>
struct Chunk {  // V channels as they are stored
  static constexpr int W = V * sizeof(raw_t<E>) / 4;
  uint32_t w[W];
  __device__ __forceinline__ void load(const raw_t<E>* p) {
    if constexpr (W == 2) {
      const uint2 u = *reinterpret_cast<const uint2*>(p);
      w[0] = u.x, w[1] = u.y;
    } else {
#pragma unroll
      for (int q = 0; q < W; q += 4) {
        const uint4 u = reinterpret_cast<const uint4*>(p)[q / 4];
        w[q] = u.x, w[q + 1] = u.y, w[q + 2] = u.z, w[q + 3] = u.w;
      }
    }
  }
  __device__ __forceinline__ void store(raw_t<E>* p) const {
    if constexpr (W == 2) {
      *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    } else {
#pragma unroll
      for (int q = 0; q < W; q += 4)
        reinterpret_cast<uint4*>(p)[q / 4] = make_uint4(w[q], w[q + 1], w[q + 2], w[q + 3]);
    }
  }
  __device__ __forceinline__ Floats<V> up() const {
    Floats<V> f;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      if constexpr (sizeof(raw_t<E>) == 4) f.x[e / 4][e % 4] = __uint_as_float(w[e]);
      else f.x[e / 4][e % 4] = Elem<E>::up(static_cast<uint16_t>(w[e / 2] >> 16 * (e & 1)));
    }
    return f;
  }
  __device__ __forceinline__ void down(const Floats<V>& f) {
    if constexpr (sizeof(raw_t<E>) == 4) {
#pragma unroll
      for (int e = 0; e < V; ++e) w[e] = __float_as_uint(f.x[e / 4][e % 4]);
    } else {
#pragma unroll
      for (int e = 0; e < V; e += 2) w[e / 2] = Elem<E>::down2(f.x[e / 4][e % 4], f.x[e / 4][e % 4 + 1]);
    }
  }
};

template <int V>
__device__ __forceinline__ float dot(const Floats<V>& a, const Floats<V>& b) {
  f32x4 s = a.x[0] * b.x[0];
#pragma unroll
  for (int q = 1; q < V / 4; ++q) s += a.x[q] * b.x[q];
  return (s[0] + s[1]) + (s[2] + s[3]);
}

template <int V>
__device__ __forceinline__ Floats<V> all_of(float v) {
  Floats<V> f;
#pragma unroll
  for (int q = 0; q < V / 4; ++q) f.x[q] = f32x4{v, v, v, v};
  return f;
}
template <int V>
__device__ __forceinline__ Floats<V> load_f32(const float* p) {
  Floats<V> f;
#pragma unroll
  for (int q = 0; q < V / 4; ++q) f.x[q] = reinterpret_cast<const f32x4*>(p)[q];
  return f;
}

// Weights of channels c ..: fp32, or the heads' type; 1 where there are none.
template <typename E, int V>
__device__ __forceinline__ Floats<V> weights(const void* w, int w_f32, int c, bool in) {
  if (!w || !in) return all_of<V>(1.f);
  if (w_f32) return load_f32<V>(static_cast<const float*>(w) + c);
  Chunk<E, V> t;
  t.load(static_cast<const raw_t<E>*>(w) + c);
  return t.up();
}

// A token's angles: cosines and sines of the lane's V pairs. A position outside
// the table is never read: its rows come out NaN.
template <int V>
__device__ __forceinline__ void angles(const RopeArgs& a, int token, int n, int cv, bool turns, Floats<V>& co,
                                       Floats<V>& si) {
  int64_t at = n;
  if (a.table && a.positions)
    at = a.pos_i64 ? static_cast<const int64_t*>(a.positions)[token] : static_cast<const int32_t*>(a.positions)[token];
  const bool off = a.table && (at < 0 || at >= a.table_rows);
  if (!off && turns) {
    const float* const t = a.table + at * a.rot;
    co = load_f32<V>(t + cv);
    si = load_f32<V>(t + a.rot / 2 + cv);
  } else {
    co = all_of<V>(off ? NAN : 1.f);
    si = all_of<V>(off ? NAN : 0.f);
  }
}

template <typename E>
__device__ __forceinline__ raw_t<E>* row_of(const HeadsView& v, int b, int n) {
  return static_cast<raw_t<E>*>(v.p) + b * v.sb + n * v.sn;
}

// U: heads a lane has in flight.
template <typename E, int V, int LP, int U>
__global__ void __launch_bounds__(kThreads) qk_rope_kernel(RopeArgs a, Side sq, Side sk) {
  const bool key = static_cast<int>(blockIdx.x) >= sq.blocks;
  const Side& s = key ? sk : sq;
  const int blk = blockIdx.x - (key ? sq.blocks : 0), gp = s.gp, H = s.heads;
  const Lane<V, LP> l(a, threadIdx.x & 63, gp);
  const int64_t token = static_cast<int64_t>(blk * (kThreads / 64) + (threadIdx.x >> 6)) * s.per + l.tok;
  if (token >= a.B * a.N) return;
  const int b = static_cast<int>(token) / a.N, n = static_cast<int>(token) - b * a.N;
  const raw_t<E>* const x = row_of<E>(s.x, b, n);
  raw_t<E>* const z = row_of<E>(s.z, b, n);
  const int64_t xh = s.x.sh, zh = s.z.sh;
  Floats<V> co, si;
  angles<V>(a, static_cast<int>(token), n, V * l.c, l.turns, co, si);
  const bool normed = s.w != nullptr;
  const Floats<V> w1 = weights<E, V>(s.w, a.w_f32, l.o1, l.chan), w2 = weights<E, V>(s.w, a.w_f32, l.o2, l.chan);
  const float inv_d = 1.f / a.d;
  for (int h0 = l.h0; h0 < H; h0 += U * gp) {
    Chunk<E, V> x1[U] = {}, x2[U] = {};
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int h = h0 + u * gp;
      if (h < H && l.chan) {
        x1[u].load(x + h * xh + l.o1);
        x2[u].load(x + h * xh + l.o2);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int h = h0 + u * gp;
      Floats<V> f1 = x1[u].up(), f2 = x2[u].up(), g1, g2;
      if (normed) {
        const float ss = group_sum<LP>(dot<V>(f1, f1) + dot<V>(f2, f2));
        const float r = 1.f / sqrtf(fmaf(ss, inv_d, a.eps));
#pragma unroll
        for (int q = 0; q < V / 4; ++q) {
          f1.x[q] *= r * w1.x[q];
          f2.x[q] *= r * w2.x[q];
        }
      }
#pragma unroll
      for (int q = 0; q < V / 4; ++q) {
        g1.x[q] = f1.x[q] * co.x[q];
        g2.x[q] = f2.x[q] * co.x[q];
        if (l.turns) {  // else co is 1, or NaN
          g1.x[q] -= f2.x[q] * si.x[q];
          g2.x[q] += f1.x[q] * si.x[q];
        }
      }
      if (h < H && l.chan) {
        Chunk<E, V> o;
        o.down(g1);
        o.store(z + h * zh + l.o1);
        o.down(g2);
        o.store(z + h * zh + l.o2);
      }
    }
  }
}

// The gradient. part: [blocks of both sides][d], each workgroup's sums for its
// side's weight.
template <typename E, int V, int LP, int U>
__global__ void __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(3)))
qk_rope_bwd_kernel(RopeArgs a, Side sq, Side sk, float* __restrict__ part) {
  constexpr int Q = V / 4;
  __shared__ f32x4 red[2 * Q][kThreads];
  const bool key = static_cast<int>(blockIdx.x) >= sq.blocks;
  const Side& s = key ? sk : sq;
  const int blk = blockIdx.x - (key ? sq.blocks : 0), gp = s.gp, H = s.heads, per = s.per;
  const Lane<V, LP> l(a, threadIdx.x & 63, gp);
  const int tokens = a.B * a.N;
  const bool normed = s.w != nullptr;
  const Floats<V> w1 = weights<E, V>(s.w, a.w_f32, l.o1, l.chan), w2 = weights<E, V>(s.w, a.w_f32, l.o2, l.chan);
  const float inv_d = 1.f / a.d;
  f32x4 dw[2 * Q] = {};  // lower chunk, upper chunk
  for (int64_t t0 = static_cast<int64_t>(blk * (kThreads / 64) + (threadIdx.x >> 6)) * per; t0 < tokens;
       t0 += static_cast<int64_t>(s.blocks) * (kThreads / 64) * per) {
    const int token = static_cast<int>(min(t0 + l.tok, static_cast<int64_t>(tokens - 1)));
    const bool live = t0 + l.tok < tokens && l.chan;  // tokens behind the last: a copy, neither added nor stored
    const int b = token / a.N, n = token - b * a.N;
    const raw_t<E>* const x = row_of<E>(s.x, b, n);
    const raw_t<E>* const z = row_of<E>(s.z, b, n);
    raw_t<E>* const o = row_of<E>(s.dx, b, n);
    Floats<V> co, si;
    angles<V>(a, token, n, V * l.c, l.turns, co, si);
    for (int h0 = l.h0; h0 < H; h0 += U * gp) {
      Chunk<E, V> x1[U] = {}, x2[U] = {}, z1[U] = {}, z2[U] = {};
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int h = h0 + u * gp;
        if (h < H && live) {
          x1[u].load(x + h * s.x.sh + l.o1);
          x2[u].load(x + h * s.x.sh + l.o2);
          z1[u].load(z + h * s.z.sh + l.o1);
          z2[u].load(z + h * s.z.sh + l.o2);
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int h = h0 + u * gp;
        const bool in = h < H && live;
        const Floats<V> g1 = z1[u].up(), g2 = z2[u].up();
        Floats<V> y1, y2;  // dy, then dx
#pragma unroll
        for (int q = 0; q < Q; ++q) {
          y1.x[q] = g1.x[q] * co.x[q];
          y2.x[q] = g2.x[q] * co.x[q];
          if (l.turns) {
            y1.x[q] += g2.x[q] * si.x[q];
            y2.x[q] -= g1.x[q] * si.x[q];
          }
        }
        if (normed) {
          Floats<V> n1 = x1[u].up(), n2 = x2[u].up();
          const float ss = group_sum<LP>(dot<V>(n1, n1) + dot<V>(n2, n2));
          const float r = 1.f / sqrtf(fmaf(ss, inv_d, a.eps));
#pragma unroll
          for (int q = 0; q < Q; ++q) {
            n1.x[q] *= r;
            n2.x[q] *= r;
            if (in) {
              dw[q] += y1.x[q] * n1.x[q];
              dw[Q + q] += y2.x[q] * n2.x[q];
            }
            y1.x[q] *= w1.x[q];
            y2.x[q] *= w2.x[q];
          }
          const float m = group_sum<LP>(dot<V>(y1, n1) + dot<V>(y2, n2)) * inv_d;
#pragma unroll
          for (int q = 0; q < Q; ++q) {
            y1.x[q] = r * (y1.x[q] - n1.x[q] * m);
            y2.x[q] = r * (y2.x[q] - n2.x[q] * m);
          }
        }
        if (in) {
          Chunk<E, V> d;
          d.down(y1);
          d.store(o + h * s.dx.sh + l.o1);
          d.down(y2);
          d.store(o + h * s.dx.sh + l.o2);
        }
      }
    }
  }
  if (!normed) return;
#pragma unroll
  for (int e = 0; e < 2 * Q; ++e) red[e][threadIdx.x] = dw[e];
  __syncthreads();
  // sums over the workgroup's lanes of the same channels
  for (int t = threadIdx.x; t < 2 * Q * LP; t += kThreads) {
    const int e = t / LP, cc = t % LP;
    if (2 * V * cc >= a.d) continue;
    f32x4 sum = {};
#pragma unroll 4
    for (int gg = 0; gg < kThreads / LP; ++gg) sum += red[e][gg * LP + cc];
    const bool turns = a.table && 2 * V * cc < a.rot;
    const int o = (e < Q ? (turns ? V * cc : 2 * V * cc) : (turns ? a.rot / 2 + V * cc : 2 * V * cc + V)) + 4 * (e % Q);
    *reinterpret_cast<f32x4*>(part + static_cast<int64_t>(blockIdx.x) * a.d + o) = sum;
  }
}

// The partial sums of nq (queries) and nk (keys) workgroups, added in a fixed
// order: a workgroup per 8 columns of one of the weights, 128 threads a column.
__global__ void __launch_bounds__(1024) qk_rope_weights_kernel(const float* __restrict__ part, int nq, int nk, int d,
                                                               float* __restrict__ dwq, float* __restrict__ dwk) {
  __shared__ float red[128][9];
  const bool key = static_cast<int>(blockIdx.x) >= d / 8;
  float* const out = key ? dwk : dwq;
  if (!out) return;
  const int x = threadIdx.x & 7, col = (blockIdx.x - (key ? d / 8 : 0)) * 8 + x, by = threadIdx.x >> 3;
  const float* const p = part + (key ? static_cast<int64_t>(nq) * d : 0);
  const int nb = key ? nk : nq;
  float s = 0.f;
#pragma unroll 8
  for (int r = by; r < nb; r += 128) s += p[static_cast<int64_t>(r) * d + col];
  red[by][x] = s;
  __syncthreads();
  for (int n = 64; n > 0; n >>= 1) {
    if (by < n) red[by][x] += red[by + n][x];
    __syncthreads();
  }
  if (by == 0) out[col] = red[0][x];
}

int chunk_of(const RopeArgs& a) { return a.d % 16 == 0 && a.rot % 16 == 0 ? 8 : 4; }
int lanes_of(const RopeArgs& a) {
  int lp = 1;
  while (2 * chunk_of(a) * lp < a.d) lp <<= 1;
  return lp;
}
Side side_of(const RopeArgs& a, bool key, int most) {
  Side s = key ? Side{a.k, a.k_out, a.dk, a.wk, a.Hkv} : Side{a.q, a.q_out, a.dq, a.wq, a.Hq};
  const int groups = 64 / lanes_of(a);
  for (s.gp = 1; s.gp < s.heads && s.gp < groups;) s.gp <<= 1;
  s.per = groups / s.gp;
  const int64_t per = 4 * s.per, n = (static_cast<int64_t>(a.B) * a.N + per - 1) / per;
  s.blocks = static_cast<int>(n < most ? n : most);
  return s;
}

template <typename E, int V, int LP>
hipError_t launch(const RopeArgs& a, bool back) {
  hipStream_t st = static_cast<hipStream_t>(a.stream);
  const int most = back ? kBwdBlocks : 0x7fffffff;
  const Side q = side_of(a, false, most), k = side_of(a, true, most);
  const dim3 grid(static_cast<uint32_t>(q.blocks) + static_cast<uint32_t>(k.blocks));
  if (!back) {
    hipLaunchKernelGGL((qk_rope_kernel<E, V, LP, 4>), grid, dim3(kThreads), 0, st, a, q, k);
    return hipGetLastError();
  }
  float* const part = static_cast<float*>(a.ws);
  hipLaunchKernelGGL((qk_rope_bwd_kernel<E, V, LP, (V * sizeof(raw_t<E>) > 16 ? 1 : 2)>), grid, dim3(kThreads), 0, st, a,
                     q, k, part);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || !(a.dwq || a.dwk)) return e;
  hipLaunchKernelGGL(qk_rope_weights_kernel, dim3(2 * a.d / 8), dim3(1024), 0, st, part, q.blocks, k.blocks, a.d, a.dwq,
                     a.dwk);
  return hipGetLastError();
}

template <typename E>
hipError_t run(const RopeArgs& a, bool back) {
  const int lp = lanes_of(a);
  if (chunk_of(a) == 8) switch (lp) {
      case 1: return launch<E, 8, 1>(a, back);
      case 2: return launch<E, 8, 2>(a, back);
      case 4: return launch<E, 8, 4>(a, back);
      case 8: return launch<E, 8, 8>(a, back);
    }
  switch (lp) {
    case 1: return launch<E, 4, 1>(a, back);
    case 2: return launch<E, 4, 2>(a, back);
    case 4: return launch<E, 4, 4>(a, back);
    case 8: return launch<E, 4, 8>(a, back);
    case 16: return launch<E, 4, 16>(a, back);
  }
  return hipErrorInvalidValue;
}

}  // namespace

int64_t qk_rope_bwd_workspace(const RopeArgs& a) {
  return (static_cast<int64_t>(side_of(a, false, kBwdBlocks).blocks) + side_of(a, true, kBwdBlocks).blocks) * a.d * 4;
}

int64_t qk_rope_threads(const RopeArgs& a) {
  return (static_cast<int64_t>(side_of(a, false, 0x7fffffff).blocks) + side_of(a, true, 0x7fffffff).blocks) * kThreads;
}

hipError_t run_qk_rope(const RopeArgs& a, bool back) {
  if (a.dtype == kF32) return run<float>(a, back);
  if (a.dtype == kBf16) return run<BF16>(a, back);
  return run<F16>(a, back);
}

}  // namespace tarmac
