#include "ehip_linear_tile.hpp"

namespace ehip {

hipError_t launch_linear_tile_bf16(const LinearArgs &a, int form, long long blocks_m, hipStream_t s)
{
  return run_linear_tile<EHIP_BF16>(a, form, blocks_m, s);
}

}  // namespace ehip
