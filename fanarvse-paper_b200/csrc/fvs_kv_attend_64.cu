// The attention kernels over heads of 64 elements.
#include "fvs_kv_attend.cuh"

namespace fvs {
namespace kv {
template int launch_types<64>(fvs_stream_t, const AttendArgs&, int);
}
}  // namespace fvs
