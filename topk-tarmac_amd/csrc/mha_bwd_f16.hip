// Attention over heads, backward: the f16 kernels of mha_bwd.hpp.
#include "mha_bwd.hpp"

namespace tarmac {

hipError_t run_mha_bwd_f16(const MhaArgs& a) { return mha::run_bwd<F16>(a); }

}  // namespace tarmac
