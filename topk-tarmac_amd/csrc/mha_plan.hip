// Attention over heads: how a call is divided over the chip (host code).
#include <algorithm>

#include "tarmac_internal.hpp"

namespace tarmac {

namespace {
constexpr int kCUs = 256;
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

}  // namespace tarmac
