#pragma once
#include "ehip_layers.hpp"

namespace ehip {
// many rows: tiles of 128 x 128 (form 0) or 256 x 256 (form 1) results staged through LDS
hipError_t launch_linear_tile(const LinearArgs &a, int type, int form, long long blocks_m, hipStream_t s);
}
