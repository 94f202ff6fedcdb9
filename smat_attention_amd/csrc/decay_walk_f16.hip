// The walks of linear attention with a decay for each head, for f16 inputs.
#include "decay_walk.hpp"

namespace smat {
namespace hd {
template int launch_walk<f16>(const Walks&, bool, int, hipStream_t);
}  // namespace hd
}  // namespace smat
