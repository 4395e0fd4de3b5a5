#pragma once
#include "ehip_layers.hpp"

namespace ehip {
// many rows: tiles of 128 x 128 (form 0; form 1: four steps in LDS) or 256 x 256 (form 2) results staged through LDS
hipError_t launch_linear_tile(const LinearArgs &a, int type, int form, long long blocks_m, hipStream_t s);
}
