// hk_rows_u3.hip -- the row products of hk_rows_kernel.h for HK_U3 organs.
#include "hk_rows_kernel.h"

namespace hk {
hipError_t launch_rows_u3(const RowsShape& sh, const RowsArgs& a, hipStream_t s) {
    return launch_rows_kind<HK_U3>(sh, a, s);
}
}  // namespace hk
