// Attention over heads, backward: the f32 kernels of mha_bwd.hpp.
#include "mha_bwd.hpp"

namespace tarmac {

hipError_t run_mha_bwd_f32(const MhaArgs& a) { return mha::run_bwd<float>(a); }

}  // namespace tarmac
