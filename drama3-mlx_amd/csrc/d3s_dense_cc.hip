/* k_tile for one order of the operands: both stored by the inner index. */
#include "d3s_dense_tile.h"

namespace d3s {
template void launch_tiles<true, true>(const Operands &, const Out &, const TilePlan &, hipStream_t);
}
