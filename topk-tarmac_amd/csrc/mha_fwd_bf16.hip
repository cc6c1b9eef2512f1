// Attention over heads, forward: the bf16 kernels of mha_fwd.hpp.
#include "mha_fwd.hpp"

namespace tarmac {

hipError_t run_mha_fwd_bf16(const MhaArgs& a) { return mha::run_fwd<BF16>(a); }

}  // namespace tarmac
