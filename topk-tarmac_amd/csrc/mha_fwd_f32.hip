// Attention over heads, forward: the f32 kernels of mha_fwd.hpp.
#include "mha_fwd.hpp"

namespace tarmac {

hipError_t run_mha_fwd_f32(const MhaArgs& a) { return mha::run_fwd<float>(a); }

}  // namespace tarmac
