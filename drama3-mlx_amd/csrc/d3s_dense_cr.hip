/* k_tile for one order of the operands: x stored [k, m]. */
#include "d3s_dense_tile.h"

namespace d3s {
template void launch_tiles<true, false>(const Operands &, const Out &, const TilePlan &, hipStream_t);
}
