// gpx_attend_f32.hip -- the attention kernels of gpx_attend_kernel.hpp and gpx_attend_grad.hpp for float elements.
#include "gpx_attend_grad.hpp"
#include "gpx_attend_kernel.hpp"

namespace gpx {
template void attend_launch_fwd<float>(const AttendFwd &, hipStream_t);
template void attend_launch_pair<float>(const AttendPair &, hipStream_t);
template void attend_launch_join<float>(const AttendJoin &, hipStream_t);
template void attend_launch_bwd<float>(const AttendBwd &, hipStream_t);
}  // namespace gpx
