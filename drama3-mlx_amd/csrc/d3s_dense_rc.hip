/* k_tile for one order of the operands: w stored [k, n]. */
#include "d3s_dense_tile.h"

namespace d3s {
template void launch_tiles<false, true>(const Operands &, const Out &, const TilePlan &, hipStream_t);
}
