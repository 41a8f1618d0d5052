// The grouped products' tiles for fp32 elements.

#include "grouped_tiles.hpp"

namespace gx::layer {

template void launch_rows_tiles<float>(const GroupedArgs&, bool, bool, hipStream_t);
template void launch_dw_tiles<float>(const GroupedArgs&, bool, bool, int, hipStream_t);

}  // namespace gx::layer
