// The tree attention kernels over heads of 256 elements.
#include "fvs_kv_tree.cuh"

namespace fvs {
namespace kv {
namespace tree {
template int launch_types<256>(fvs_stream_t, Args, int);
}
}  // namespace kv
}  // namespace fvs
