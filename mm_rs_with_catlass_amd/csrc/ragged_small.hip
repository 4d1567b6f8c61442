// Instantiates the small tiles of ragged products.
#include "ragged_small.h"

namespace catcoc {

// Ring depths: two workgroups a CU, one with more than 16 rows of a matrix as [k, n].
template <uint32_t DT>
static void launch_nk(const RaggedArgs &a, uint32_t rows, uint32_t wgs, hipStream_t stream)
{
    const dim3 grid(wgs), block(256);
    if (rows == 16u) hipLaunchKernelGGL((ragged_small_kernel<DT, false, 1, 2, 3>), grid, block, 0, stream, a);
    else hipLaunchKernelGGL((ragged_small_kernel<DT, false, 2, 2, 2>), grid, block, 0, stream, a);
}

template <uint32_t DT>
static void launch_kn(const RaggedArgs &a, uint32_t rows, uint32_t wgs, hipStream_t stream)
{
    const dim3 grid(wgs), block(256);
    if (rows == 16u) hipLaunchKernelGGL((ragged_small_kernel<DT, true, 1, 4, 2>), grid, block, 0, stream, a);
    else if (rows == 32u) hipLaunchKernelGGL((ragged_small_kernel<DT, true, 2, 4, 3>), grid, block, 0, stream, a);
    else hipLaunchKernelGGL((ragged_small_kernel<DT, true, 4, 4, 2>), grid, block, 0, stream, a);
}

int launch_ragged_small(uint32_t dtype, const RaggedArgs &a, bool kn, uint32_t rows, uint32_t wgs, void *stream)
{
    if (dtype == DT_F8) launch_nk<DT_F8>(a, rows, wgs, (hipStream_t)stream);
    else if (dtype == DT_F16 && kn) launch_kn<DT_F16>(a, rows, wgs, (hipStream_t)stream);
    else if (dtype == DT_F16) launch_nk<DT_F16>(a, rows, wgs, (hipStream_t)stream);
    else if (kn) launch_kn<DT_BF16>(a, rows, wgs, (hipStream_t)stream);
    else launch_nk<DT_BF16>(a, rows, wgs, (hipStream_t)stream);
    return (int)hipGetLastError();
}

}  // namespace catcoc
