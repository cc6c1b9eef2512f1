// Attention over heads, forward: the f16 kernels of mha_fwd.hpp.
#include "mha_fwd.hpp"

namespace tarmac {

hipError_t run_mha_fwd_f16(const MhaArgs& a) { return mha::run_fwd<F16>(a); }

}  // namespace tarmac
