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
// VALU each. A head is spread over LP lanes (the power of two from d / 8 up),
// eight channels each: four of the rotation's lower half and the four they turn
// with, so a rotation needs no other lane, and the norm one sum over the group.
// Queries and keys are one list of rows (token, head): one launch does both.
#include "heads.hpp"

namespace tarmac {

namespace {

constexpr int kThreads = 256;
constexpr int kFwdRows = 4;      // rows a group has in flight
constexpr int kBwdRowsAhead = 2;
constexpr int kBwdBlocks = 1024; // workgroups of the gradient: each leaves one partial sum of the weights'

struct Place {  // a row of the list
  bool in, key;
  int b, n, head, token;
};

__device__ __forceinline__ Place place_of(const RopeArgs& a, int64_t row, int64_t rows) {
  Place p;
  p.in = row < rows;
  const uint32_t H = a.Hq + a.Hkv;
  const uint32_t r = static_cast<uint32_t>(p.in ? row : 0);  // rows < 2^31
  p.token = static_cast<int>(r / H);
  const int h = static_cast<int>(r - p.token * H);
  p.key = h >= a.Hq;
  p.head = p.key ? h - a.Hq : h;
  p.b = p.token / a.N;
  p.n = p.token - p.b * a.N;
  return p;
}

template <typename E>
__device__ __forceinline__ raw_t<E>* row_of(const HeadsView& v, const Place& p) {
  return static_cast<raw_t<E>*>(v.p) + p.b * v.sb + p.n * v.sn + p.head * v.sh;
}
__device__ __forceinline__ HeadsView pick(const HeadsView& q, const HeadsView& k, bool key) {
  return HeadsView{key ? k.p : q.p, key ? k.sb : q.sb, key ? k.sn : q.sn, key ? k.sh : q.sh};
}

template <typename E>
struct Packed4;
template <>
struct Packed4<float> { using type = f32x4; };
template <>
struct Packed4<BF16> { using type = uint2; };
template <>
struct Packed4<F16> { using type = uint2; };
template <typename E>
using packed4_t = typename Packed4<E>::type;

template <typename E>
__device__ __forceinline__ f32x4 up4(packed4_t<E> x) {
  if constexpr (sizeof(raw_t<E>) == 4) {
    return x;
  } else {
    const uint32_t w[2] = {x.x, x.y};
    f32x4 f;
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] = Elem<E>::up(static_cast<uint16_t>(w[e / 2] >> 16 * (e & 1)));
    return f;
  }
}
template <typename E>
__device__ __forceinline__ packed4_t<E> down4(f32x4 f) {
  if constexpr (sizeof(raw_t<E>) == 4) return f;
  else return make_uint2(Elem<E>::down2(f[0], f[1]), Elem<E>::down2(f[2], f[3]));
}
template <typename E>
__device__ __forceinline__ packed4_t<E> ld4(const raw_t<E>* p) {
  return *reinterpret_cast<const packed4_t<E>*>(p);
}
template <typename E>
__device__ __forceinline__ void st4(raw_t<E>* p, f32x4 f) {
  *reinterpret_cast<packed4_t<E>*>(p) = down4<E>(f);
}

// Four weights from channel c: fp32, or the heads' type.
template <typename E>
__device__ __forceinline__ f32x4 weights(const void* w, int w_f32, int c) {
  if (w_f32) return *reinterpret_cast<const f32x4*>(static_cast<const float*>(w) + c);
  return up4<E>(ld4<E>(static_cast<const raw_t<E>*>(w) + c));
}

__device__ __forceinline__ float sum4(f32x4 a) { return (a[0] + a[1]) + (a[2] + a[3]); }

// A row's angles: cosines and sines of the lane's four pairs. A position
// outside the table is never read: its row comes out NaN.
__device__ __forceinline__ void angles(const RopeArgs& a, const Place& p, int c4, bool turns, f32x4& co,
                                       f32x4& si) {
  co = f32x4{1.f, 1.f, 1.f, 1.f};
  si = f32x4{0.f, 0.f, 0.f, 0.f};
  if (!a.table || !p.in) return;
  int64_t at = p.n;
  if (a.positions)
    at = a.pos_i64 ? static_cast<const int64_t*>(a.positions)[p.token]
                   : static_cast<const int32_t*>(a.positions)[p.token];
  if (at < 0 || at >= a.table_rows) {
    co = si = f32x4{NAN, NAN, NAN, NAN};
    return;
  }
  if (!turns) return;
  const float* const t = a.table + at * a.rot;
  co = *reinterpret_cast<const f32x4*>(t + c4);
  si = *reinterpret_cast<const f32x4*>(t + a.rot / 2 + c4);
}

template <typename E, int LP>
__global__ void __launch_bounds__(kThreads) qk_rope_kernel(RopeArgs a, int64_t rows) {
  constexpr int RPB = kThreads / LP;
  const int c = threadIdx.x % LP, grp = threadIdx.x / LP;
  const bool chan = 8 * c < a.d, turns = a.table && 8 * c < a.rot;
  const int o1 = turns ? 4 * c : 8 * c, o2 = turns ? a.rot / 2 + 4 * c : 8 * c + 4;
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * RPB * kFwdRows + grp;

  Place p[kFwdRows];
  packed4_t<E> x1[kFwdRows] = {}, x2[kFwdRows] = {};
#pragma unroll
  for (int u = 0; u < kFwdRows; ++u) {
    p[u] = place_of(a, row0 + u * RPB, rows);
    if (p[u].in && chan) {
      const raw_t<E>* const x = row_of<E>(pick(a.q, a.k, p[u].key), p[u]);
      x1[u] = ld4<E>(x + o1);
      x2[u] = ld4<E>(x + o2);
    }
  }
  const f32x4 one = {1.f, 1.f, 1.f, 1.f};
  f32x4 wq1 = one, wq2 = one, wk1 = one, wk2 = one;
  if (chan && a.wq) {
    wq1 = weights<E>(a.wq, a.w_f32, o1);
    wq2 = weights<E>(a.wq, a.w_f32, o2);
  }
  if (chan && a.wk) {
    wk1 = weights<E>(a.wk, a.w_f32, o1);
    wk2 = weights<E>(a.wk, a.w_f32, o2);
  }
  const float inv_d = 1.f / a.d;
#pragma unroll
  for (int u = 0; u < kFwdRows; ++u) {
    f32x4 co, si;
    angles(a, p[u], 4 * c, turns, co, si);
    f32x4 f1 = up4<E>(x1[u]), f2 = up4<E>(x2[u]);
    const float ss = group_sum<LP>(sum4(f1 * f1) + sum4(f2 * f2));
    if (p[u].key ? a.wk != nullptr : a.wq != nullptr) {
      const float r = 1.f / sqrtf(fmaf(ss, inv_d, a.eps));
      f1 *= r * (p[u].key ? wk1 : wq1);
      f2 *= r * (p[u].key ? wk2 : wq2);
    }
    if (p[u].in && chan) {
      raw_t<E>* const o = row_of<E>(pick(a.q_out, a.k_out, p[u].key), p[u]);
      if (turns) {
        st4<E>(o + o1, f1 * co - f2 * si);
        st4<E>(o + o2, f2 * co + f1 * si);
      } else {  // co: 1, or NaN
        st4<E>(o + o1, f1 * co);
        st4<E>(o + o2, f2 * co);
      }
    }
  }
}

// The gradient. part: [gridDim.x][2][d], each workgroup's sums for the weights.
template <typename E, int LP>
__global__ void __launch_bounds__(kThreads) qk_rope_bwd_kernel(RopeArgs a, int64_t rows, float* __restrict__ part) {
  constexpr int RPB = kThreads / LP, U = kBwdRowsAhead;
  __shared__ f32x4 red[4][kThreads];
  const int c = threadIdx.x % LP, grp = threadIdx.x / LP;
  const bool chan = 8 * c < a.d, turns = a.table && 8 * c < a.rot;
  const int o1 = turns ? 4 * c : 8 * c, o2 = turns ? a.rot / 2 + 4 * c : 8 * c + 4;
  const f32x4 one = {1.f, 1.f, 1.f, 1.f};
  f32x4 w[2][2] = {{one, one}, {one, one}};
  if (chan && a.wq) {
    w[0][0] = weights<E>(a.wq, a.w_f32, o1);
    w[0][1] = weights<E>(a.wq, a.w_f32, o2);
  }
  if (chan && a.wk) {
    w[1][0] = weights<E>(a.wk, a.w_f32, o1);
    w[1][1] = weights<E>(a.wk, a.w_f32, o2);
  }
  const float inv_d = 1.f / a.d;
  f32x4 dw[2][2] = {};
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * RPB * U; base < rows;
       base += static_cast<int64_t>(gridDim.x) * RPB * U) {
    Place p[U];
    packed4_t<E> x1[U] = {}, x2[U] = {}, z1[U] = {}, z2[U] = {};
    f32x4 co[U], si[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      p[u] = place_of(a, base + u * RPB + grp, rows);
      if (p[u].in && chan) {
        const raw_t<E>* const x = row_of<E>(pick(a.q, a.k, p[u].key), p[u]);
        const raw_t<E>* const z = row_of<E>(pick(a.q_out, a.k_out, p[u].key), p[u]);
        x1[u] = ld4<E>(x + o1);
        x2[u] = ld4<E>(x + o2);
        z1[u] = ld4<E>(z + o1);
        z2[u] = ld4<E>(z + o2);
      }
      angles(a, p[u], 4 * c, turns, co[u], si[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int key = p[u].key;
      const f32x4 f1 = up4<E>(x1[u]), f2 = up4<E>(x2[u]);
      const f32x4 g1 = up4<E>(z1[u]), g2 = up4<E>(z2[u]);
      f32x4 dy1 = g1 * co[u], dy2 = g2 * co[u];
      if (turns) {
        dy1 += g2 * si[u];
        dy2 -= g1 * si[u];
      }
      f32x4 dx1 = dy1, dx2 = dy2;
      if (key ? a.wk != nullptr : a.wq != nullptr) {
        const float ss = group_sum<LP>(sum4(f1 * f1) + sum4(f2 * f2));
        const float r = 1.f / sqrtf(fmaf(ss, inv_d, a.eps));
        const f32x4 n1 = f1 * r, n2 = f2 * r;
        const f32x4 a1 = dy1 * n1, a2 = dy2 * n2;
        const f32x4 w1 = key ? w[1][0] : w[0][0], w2 = key ? w[1][1] : w[0][1];
        const float m = group_sum<LP>(sum4(a1 * w1) + sum4(a2 * w2)) * inv_d;
        dx1 = r * (dy1 * w1 - n1 * m);
        dx2 = r * (dy2 * w2 - n2 * m);
        const f32x4 zero = {};
        dw[0][0] += key ? zero : a1;
        dw[0][1] += key ? zero : a2;
        dw[1][0] += key ? a1 : zero;
        dw[1][1] += key ? a2 : zero;
      }
      if (p[u].in && chan) {
        raw_t<E>* const o = row_of<E>(pick(a.dq, a.dk, key), p[u]);
        st4<E>(o + o1, dx1);
        st4<E>(o + o2, dx2);
      }
    }
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) red[e][threadIdx.x] = dw[e / 2][e % 2];
  __syncthreads();
  // 2 x 2 x LP four-channel sums over the workgroup's groups
  for (int t = threadIdx.x; t < 4 * LP; t += kThreads) {
    const int e = t / LP, cc = t % LP;
    if (8 * cc >= a.d) continue;
    f32x4 s = {};
#pragma unroll 4
    for (int gg = 0; gg < RPB; ++gg) s += red[e][gg * LP + cc];
    const bool tt = a.table && 8 * cc < a.rot;
    const int o = (e & 1) ? (tt ? a.rot / 2 + 4 * cc : 8 * cc + 4) : (tt ? 4 * cc : 8 * cc);
    *reinterpret_cast<f32x4*>(part + (static_cast<int64_t>(blockIdx.x) * 2 + e / 2) * a.d + o) = s;
  }
}

// The partial sums of nb workgroups, added in a fixed order: a workgroup per 32
// of the 2 d columns, 32 threads a column.
__global__ void __launch_bounds__(1024) qk_rope_weights_kernel(const float* __restrict__ part, int nb, int d,
                                                               float* __restrict__ dwq, float* __restrict__ dwk) {
  __shared__ float red[32][33];
  const int col = blockIdx.x * 32 + (threadIdx.x & 31), by = threadIdx.x >> 5;
  float s = 0.f;
  if (col < 2 * d)
    for (int r = by; r < nb; r += 32) s += part[static_cast<int64_t>(r) * 2 * d + col];
  red[by][threadIdx.x & 31] = s;
  __syncthreads();
  if (by == 0 && col < 2 * d) {
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) t += red[i][threadIdx.x];
    if (col < d) {
      if (dwq) dwq[col] = t;
    } else if (dwk) {
      dwk[col - d] = t;
    }
  }
}

int lanes_per_head(int d) {
  int lp = 1;
  while (8 * lp < d) lp <<= 1;
  return lp;
}
int64_t rows_of(const RopeArgs& a) { return static_cast<int64_t>(a.B) * a.N * (a.Hq + a.Hkv); }
int bwd_blocks(const RopeArgs& a) {
  const int64_t per = static_cast<int64_t>(kThreads / lanes_per_head(a.d)) * kBwdRowsAhead;
  const int64_t n = (rows_of(a) + per - 1) / per;
  return static_cast<int>(n < kBwdBlocks ? n : kBwdBlocks);
}

template <typename E, int LP>
hipError_t launch(const RopeArgs& a, bool back) {
  hipStream_t st = static_cast<hipStream_t>(a.stream);
  const int64_t rows = rows_of(a);
  if (!back) {
    const int64_t per = static_cast<int64_t>(kThreads / LP) * kFwdRows;
    hipLaunchKernelGGL((qk_rope_kernel<E, LP>), dim3(static_cast<uint32_t>((rows + per - 1) / per)), dim3(kThreads), 0,
                       st, a, rows);
    return hipGetLastError();
  }
  const int nb = bwd_blocks(a);
  float* const part = static_cast<float*>(a.ws);
  hipLaunchKernelGGL((qk_rope_bwd_kernel<E, LP>), dim3(nb), dim3(kThreads), 0, st, a, rows, part);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || !(a.dwq || a.dwk)) return e;
  hipLaunchKernelGGL(qk_rope_weights_kernel, dim3((2 * a.d + 31) / 32), dim3(1024), 0, st, part, nb, a.d, a.dwq, a.dwk);
  return hipGetLastError();
}

template <typename E>
hipError_t run(const RopeArgs& a, bool back) {
  switch (lanes_per_head(a.d)) {
    case 1: return launch<E, 1>(a, back);
    case 2: return launch<E, 2>(a, back);
    case 4: return launch<E, 4>(a, back);
    case 8: return launch<E, 8>(a, back);
    case 16: return launch<E, 16>(a, back);
  }
  return hipErrorInvalidValue;
}

}  // namespace

int64_t qk_rope_bwd_workspace(const RopeArgs& a) { return static_cast<int64_t>(bwd_blocks(a)) * 2 * a.d * 4; }

hipError_t run_qk_rope(const RopeArgs& a, bool back) {
  if (a.dtype == kF32) return run<float>(a, back);
  if (a.dtype == kBf16) return run<BF16>(a, back);
  return run<F16>(a, back);
}

}  // namespace tarmac
