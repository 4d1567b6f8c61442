// Instantiates the bounds-checked kernels of ragged products.
#include "ragged_checked.h"

namespace catcoc {

template <uint32_t DT>
static void launch16(const RaggedArgs &a, bool kn, bool dw, uint32_t wgs, hipStream_t stream)
{
    if (dw) hipLaunchKernelGGL((ragged_checked_kernel<DT, false, true>), grid_of(wgs, 256), dim3(256), 0, stream, a);
    else if (kn) hipLaunchKernelGGL((ragged_checked_kernel<DT, true, false>), grid_of(wgs, 256), dim3(256), 0, stream, a);
    else hipLaunchKernelGGL((ragged_checked_kernel<DT, false, false>), grid_of(wgs, 256), dim3(256), 0, stream, a);
}

int launch_ragged_checked(uint32_t dtype, const RaggedArgs &a, bool kn, bool dw, uint32_t wgs, void *stream)
{
    if (dtype == DT_F8) hipLaunchKernelGGL((ragged_checked_kernel<DT_F8, false, false>), grid_of(wgs, 256), dim3(256), 0, (hipStream_t)stream, a);
    else if (dtype == DT_F16) launch16<DT_F16>(a, kn, dw, wgs, (hipStream_t)stream);
    else launch16<DT_BF16>(a, kn, dw, wgs, (hipStream_t)stream);
    return (int)hipGetLastError();
}

}  // namespace catcoc
