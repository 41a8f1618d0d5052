// The grouped products' tiles for bf16 elements.

#include "grouped_tiles.hpp"

namespace gx::layer {

template void launch_rows_tiles<bf16_t>(const GroupedArgs&, bool, bool, hipStream_t);
template void launch_dw_tiles<bf16_t>(const GroupedArgs&, bool, bool, int, hipStream_t);

}  // namespace gx::layer
