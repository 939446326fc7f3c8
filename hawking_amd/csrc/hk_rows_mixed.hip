// hk_rows_mixed.hip -- the row products of hk_rows_kernel.h for HK_MIXED organs.
#include "hk_rows_kernel.h"

namespace hk {
hipError_t launch_rows_mixed(const RowsShape& sh, const RowsArgs& a, hipStream_t s) {
    return launch_rows_kind<HK_MIXED>(sh, a, s);
}
}  // namespace hk
