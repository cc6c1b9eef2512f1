// Attention over heads: how a call is divided over the chip (host code).
#include <algorithm>

#include "tarmac_internal.hpp"

namespace tarmac {

namespace {

constexpr int64_t kCUs = 256;

// In how many parts workgroups of 128 rows divide the streamed side so that there
// are two a CU; 0: not even parts of `least` steps make `enough` workgroups.
int wide_splits(int64_t blocks, int64_t steps, int64_t least, int64_t enough) {
  const int64_t s = std::min((2 * kCUs + blocks - 1) / blocks, std::max<int64_t>(1, steps / least));
  return blocks * s >= enough ? static_cast<int>(s) : 0;
}

int row_bytes(const MhaArgs& a) { return a.d * (a.dtype == kF32 ? 4 : 2); }

}  // namespace

// Workgroups of 128 rows, whose four waves share what is streamed, where they come to
// two a CU, if need be by dividing the streamed side among them; else workgroups
// of 32 rows whose waves divide it: these read it four times as often, but need
// no join (bf16, 8 heads of 64 on 1024 tokens: 11.3 us; in two parts of 512
// keys 17.4).
FwdPlan fwd_plan(const MhaArgs& a) {
  const int64_t rows = static_cast<int64_t>(a.Nq) * (a.Hq / a.Hkv), heads = static_cast<int64_t>(a.B) * a.Hkv;
  const int wide = static_cast<int>((rows + 127) / 128);
  // In parts of 512 keys at least, one workgroup a CU at least; where 32 rows keep up
  // (16-bit heads up to 64, fp32 up to 32) of 1024, two a CU. Causal, in parts and by 32
  // rows: bf16, 4 heads of 128 on 4096 tokens 45 and 82 us, 16 heads of 64 on 4 of
  // 2048 31 and 37, but 2 x 4 heads of 64 in two parts 27 and 21; fp32, 4 heads of 128
  // on 2048 71 and 138.
  const bool narrow = row_bytes(a) <= 128;
  int splits = rows > 64 ? wide_splits(heads * wide, a.Nk, narrow ? 1024 : 512, narrow ? 2 * kCUs : kCUs) : 0;
  if (splits) {
    const int chunk = ((a.Nk + splits - 1) / splits + 63) / 64 * 64;
    if (splits > 1) splits = (a.Nk + chunk - 1) / chunk;
    if (splits > 1 || heads * wide >= 2 * kCUs) return {false, false, wide, splits, splits > 1 ? chunk : a.Nk};
  }
  const int tiles = static_cast<int>((rows + 31) / 32);
  // a workgroup of four waves per CU twice over, but no fewer than 256 keys each; of
  // eight, once over and 512
  const int64_t blocks = heads * tiles;
  int64_t each = 256;
  const auto parts = [&](int64_t cus) {
    return static_cast<int>(std::min(std::max<int64_t>(1, (cus + blocks - 1) / blocks), std::max<int64_t>(1, a.Nk / each)));
  };
  splits = parts(2 * kCUs);
  const bool more = splits > 1 && narrow;
  if (more) each = 512, splits = parts(kCUs);
  const int chunk = ((a.Nk + splits - 1) / splits + 127) / 128 * 128;
  splits = (a.Nk + chunk - 1) / chunk;
  return {true, more, tiles, splits, chunk};
}

int64_t mha_fwd_workspace(const MhaArgs& a) {
  const FwdPlan p = fwd_plan(a);
  if (p.splits == 1) return 0;
  const int64_t all = static_cast<int64_t>(a.B) * a.Hq * a.Nq;
  return p.splits * all * (a.d + 2) * 4;
}

// n rows (or keys) a key head against `steps` streamed tiles.
static BwdPass bwd_pass(const MhaArgs& a, int64_t n, int64_t steps) {
  const int64_t heads = static_cast<int64_t>(a.B) * a.Hkv, wide = (n + 127) / 128, tiles = (n + 31) / 32;
  if (heads * wide >= 2 * kCUs && n > 64) return {false, false, static_cast<int>(wide), 1};
  // In parts of 128 rows where LDS holds the tiles of four waves of 32 rows (bf16 above
  // 64 channels, fp32 above 32) or of two (fp32 above 64), not of eight, a CU: bf16,
  // 4 heads of 128 on 4096 tokens 209 and 263 us, 8 on 2 of 1024, 4 teams 124 and 146;
  // fp32, 4 heads of 128 on 2048 316 and 474. Eight waves of 32 rows win: bf16, 2 x 4
  // heads of 64 on 2048 72 us, in parts 88.
  const int row = row_bytes(a);
  if (n > 64 && row > 128)
    if (const int s = wide_splits(heads * wide, steps, 8, row > 256 ? kCUs : 2 * kCUs); s > 1)
      return {false, false, static_cast<int>(wide), s};
  // workgroups of more waves where there is about one a CU; parts of the streamed
  // side where there is less than one, of no fewer than sixteen tiles each
  const int64_t blocks = heads * tiles, most = std::max<int64_t>(1, steps / 16);
  const int splits = static_cast<int>(std::max<int64_t>(1, std::min(kCUs / blocks, most)));
  return {true, blocks * splits < kCUs * 3 / 2, static_cast<int>(tiles), splits};
}

BwdPlan bwd_plan(const MhaArgs& a) {
  const int64_t G = a.Hq / a.Hkv;
  BwdPlan p = {bwd_pass(a, a.Nq * G, (a.Nk + 31) / 32), bwd_pass(a, a.Nk, (a.Nq + 31) / 32 * G), 0, 0};
  // one launch holds both if their workgroups are alike: eight waves are the better of
  // two (bf16, 3 x 8 heads of 64 on 2 of 1111, causal, with the forward: in two launches
  // 65 us, of four waves 71, of eight 56)
  if (p.dq.few && p.dkv.few) p.dq.more_waves = p.dkv.more_waves = p.dq.more_waves || p.dkv.more_waves;
  if (p.dq.splits > 1) p.dq_floats = p.dq.splits * static_cast<int64_t>(a.B) * a.Nq * a.Hq * a.d;
  if (p.dkv.splits > 1) p.dkv_floats = 2 * p.dkv.splits * static_cast<int64_t>(a.B) * a.Nk * a.Hkv * a.d;
  return p;
}

int64_t mha_bwd_stats_floats(const MhaArgs& a) {
  return (2 * static_cast<int64_t>(a.B) * a.Hq * a.Nq + 3) / 4 * 4;
}

int64_t mha_bwd_workspace(const MhaArgs& a) {
  const BwdPlan p = bwd_plan(a);
  return (mha_bwd_stats_floats(a) + p.dq_floats + p.dkv_floats) * 4;
}

int64_t mha_threads(const MhaArgs& a) {
  const int64_t heads = static_cast<int64_t>(a.B) * a.Hkv;
  const FwdPlan f = fwd_plan(a);
  const BwdPlan b = bwd_plan(a);
  // few rows: up to eight waves share a tile, fewer where there are many (one key
  // tile, or the backward above 384 workgroups)
  const int64_t fwd = heads * f.tiles * f.splits * (!f.few ? 256 : a.Nk <= 32 ? 64 : 512);
  const auto pass = [&](const BwdPass& p) { return heads * p.tiles * p.splits * (p.few && p.more_waves ? 512 : 256); };
  const int64_t rows = static_cast<int64_t>(a.B) * a.Hq * a.Nq;
  const int64_t lanes = rows * (a.d <= 16 ? 2 : a.d <= 32 ? 4 : a.d <= 64 ? 8 : 16);  // mha_bwd_stats_kernel
  return std::max(std::max(fwd, lanes), std::max(pass(b.dq), pass(b.dkv)));
}

}  // namespace tarmac
