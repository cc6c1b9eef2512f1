// Attention over heads, backward: the bf16 kernels of mha_bwd.hpp.
#include "mha_bwd.hpp"

namespace tarmac {

hipError_t run_mha_bwd_bf16(const MhaArgs& a) { return mha::run_bwd<BF16>(a); }

}  // namespace tarmac
