// hk_rows_bin.hip -- the row products of hk_rows_kernel.h for HK_BIN organs.
#include "hk_rows_kernel.h"

namespace hk {
hipError_t launch_rows_bin(const RowsShape& sh, const RowsArgs& a, hipStream_t s) {
    return launch_rows_kind<HK_BIN>(sh, a, s);
}
}  // namespace hk
