// Instantiates the large tiles of ragged products.
#include "ragged_tile.h"

namespace catcoc {

template <uint32_t DT, bool KN, bool DW>
static void launch_cols(const RaggedArgs &a, uint32_t cols, uint32_t teams, uint32_t wgs, hipStream_t stream)
{
    if (cols == 256u) hipLaunchKernelGGL((ragged_tile_kernel<DT, KN, DW, 4, 8, 1>), dim3(wgs), dim3(512), 0, stream, a);
    else if (!DW && teams == 2u) hipLaunchKernelGGL((ragged_tile_kernel<DT, KN, DW, 2, 4, DW ? 1 : 2>), dim3(wgs), dim3(512), 0, stream, a);
    else hipLaunchKernelGGL((ragged_tile_kernel<DT, KN, DW, 2, 4, 1>), dim3(wgs), dim3(256), 0, stream, a);
}

template <uint32_t DT>
static void launch16(const RaggedArgs &a, bool kn, bool dw, uint32_t cols, uint32_t teams, uint32_t wgs, hipStream_t stream)
{
    if (dw) launch_cols<DT, false, true>(a, cols, teams, wgs, stream);
    else if (kn) launch_cols<DT, true, false>(a, cols, teams, wgs, stream);
    else launch_cols<DT, false, false>(a, cols, teams, wgs, stream);
}

int launch_ragged_tile(uint32_t dtype, const RaggedArgs &a, bool kn, bool dw, uint32_t cols, uint32_t teams, uint32_t wgs, void *stream)
{
    if (dtype == DT_F8) launch_cols<DT_F8, false, false>(a, cols, teams, wgs, (hipStream_t)stream);
    else if (dtype == DT_F16) launch16<DT_F16>(a, kn, dw, cols, teams, wgs, (hipStream_t)stream);
    else launch16<DT_BF16>(a, kn, dw, cols, teams, wgs, (hipStream_t)stream);
    return (int)hipGetLastError();
}

}  // namespace catcoc
