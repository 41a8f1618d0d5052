// The grouped products' tiles for fp16 elements.

#include "grouped_tiles.hpp"

namespace gx::layer {

template void launch_rows_tiles<_Float16>(const GroupedArgs&, bool, bool, hipStream_t);
template void launch_dw_tiles<_Float16>(const GroupedArgs&, bool, bool, int, hipStream_t);

}  // namespace gx::layer
