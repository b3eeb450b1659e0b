/* k_tile for one order of the operands: both by rows. */
#include "d3s_dense_tile.h"

namespace d3s {
template void launch_tiles<false, false>(const Operands &, const Out &, const TilePlan &, hipStream_t);
}
