// gpx_attend_bf16.hip -- the attention kernels of gpx_attend_kernel.hpp and gpx_attend_grad.hpp for __bf16 elements.
#include "gpx_attend_grad.hpp"
#include "gpx_attend_kernel.hpp"

namespace gpx {
template void attend_launch_fwd<__bf16>(const AttendFwd &, hipStream_t);
template void attend_launch_pair<__bf16>(const AttendPair &, hipStream_t);
template void attend_launch_join<__bf16>(const AttendJoin &, hipStream_t);
template void attend_launch_bwd<__bf16>(const AttendBwd &, hipStream_t);
}  // namespace gpx
