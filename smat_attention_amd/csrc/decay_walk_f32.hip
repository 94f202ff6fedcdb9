// The walks of linear attention with a decay for each head, for f32 inputs.
#include "decay_walk.hpp"

namespace smat {
namespace hd {
template int launch_walk<float>(const Walks&, bool, int, hipStream_t);
}  // namespace hd
}  // namespace smat
