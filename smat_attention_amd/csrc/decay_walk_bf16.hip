// The walks of linear attention with a decay for each head, for bf16 inputs.
#include "decay_walk.hpp"

namespace smat {
namespace hd {
template int launch_walk<bf16>(const Walks&, bool, int, hipStream_t);
}  // namespace hd
}  // namespace smat
