// Attention over heads: how a call is divided over the chip (host code).
#include <algorithm>

#include "tarmac_internal.hpp"

namespace tarmac {

namespace {
constexpr int64_t kCUs = 256;
}

FwdPlan fwd_plan(const MhaArgs& a) {
  const int64_t rows = static_cast<int64_t>(a.Nq) * (a.Hq / a.Hkv), heads = static_cast<int64_t>(a.B) * a.Hkv;
  const int wide = static_cast<int>((rows + 127) / 128);
  if (rows > 64 && heads * wide >= 2 * kCUs) return {false, wide, 1, a.Nk};
  const int tiles = static_cast<int>((rows + 31) / 32);
  // a workgroup per CU twice over, but no fewer than 256 keys each
  const int64_t blocks = heads * tiles;
  const int64_t want = std::max<int64_t>(1, (2 * kCUs + blocks - 1) / blocks);
  const int64_t most = std::max(1, a.Nk / 256);
  int splits = static_cast<int>(std::min(want, most));
  const int chunk = ((a.Nk + splits - 1) / splits + 127) / 128 * 128;
  splits = (a.Nk + chunk - 1) / chunk;
  return {true, tiles, splits, chunk};
}

int64_t mha_fwd_workspace(const MhaArgs& a) {
  const FwdPlan p = fwd_plan(a);
  if (p.splits == 1) return 0;
  const int64_t all = static_cast<int64_t>(a.B) * a.Hq * a.Nq;
  return p.splits * all * (a.d + 2) * 4;
}

// n rows (or keys) a key head against `steps` streamed tiles.
static BwdPass bwd_pass(int64_t heads, int64_t n, int64_t steps) {
  const int64_t wide = (n + 127) / 128, tiles = (n + 31) / 32;
  if (heads * wide >= 2 * kCUs && n > 64) return {false, false, static_cast<int>(wide), 1};
  // workgroups of more waves where there is about one a CU; parts of the streamed
  // side where there is less than one, of no fewer than sixteen tiles each
  const int64_t blocks = heads * tiles, most = std::max<int64_t>(1, steps / 16);
  const int splits = static_cast<int>(std::max<int64_t>(1, std::min(kCUs / blocks, most)));
  return {true, blocks * splits < kCUs * 3 / 2, static_cast<int>(tiles), splits};
}

BwdPlan bwd_plan(const MhaArgs& a) {
  const int64_t heads = static_cast<int64_t>(a.B) * a.Hkv, G = a.Hq / a.Hkv;
  return {bwd_pass(heads, a.Nq * G, (a.Nk + 31) / 32), bwd_pass(heads, a.Nk, (a.Nq + 31) / 32 * G)};
}

int64_t mha_bwd_stats_floats(const MhaArgs& a) {
  return (2 * static_cast<int64_t>(a.B) * a.Hq * a.Nq + 3) / 4 * 4;
}

int64_t mha_bwd_workspace(const MhaArgs& a) {
  const BwdPlan p = bwd_plan(a);
  const int64_t dq = p.dq.splits > 1 ? p.dq.splits * static_cast<int64_t>(a.B) * a.Nq * a.Hq * a.d : 0;
  const int64_t dkv = p.dkv.splits > 1 ? 2 * p.dkv.splits * static_cast<int64_t>(a.B) * a.Nk * a.Hkv * a.d : 0;
  return (mha_bwd_stats_floats(a) + std::max(dq, dkv)) * 4;
}

int64_t mha_threads(const MhaArgs& a) {
  const int64_t heads = static_cast<int64_t>(a.B) * a.Hkv;
  const FwdPlan f = fwd_plan(a);
  const BwdPlan b = bwd_plan(a);
  // few rows: up to eight waves share a tile, fewer where there are many (one key
  // tile, or the backward above 384 workgroups)
  const int64_t fwd = heads * f.tiles * f.splits * (!f.few ? 256 : a.Nk <= 32 ? 64 : 512);
  const auto pass = [&](const BwdPass& p) { return heads * p.tiles * (p.more_waves ? 512 : 256); };
  return std::max(fwd, std::max(pass(b.dq), pass(b.dkv)));
}

}  // namespace tarmac
