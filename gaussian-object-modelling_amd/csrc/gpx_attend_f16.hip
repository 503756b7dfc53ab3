// gpx_attend_f16.hip -- the attention kernels of gpx_attend_kernel.hpp and gpx_attend_grad.hpp for _Float16 elements.
#include "gpx_attend_grad.hpp"
#include "gpx_attend_kernel.hpp"

namespace gpx {
template void attend_launch_fwd<_Float16>(const AttendFwd &, hipStream_t);
template void attend_launch_pair<_Float16>(const AttendPair &, hipStream_t);
template void attend_launch_join<_Float16>(const AttendJoin &, hipStream_t);
template void attend_launch_bwd<_Float16>(const AttendBwd &, hipStream_t);
}  // namespace gpx
