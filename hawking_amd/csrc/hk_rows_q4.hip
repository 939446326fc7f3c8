// hk_rows_q4.hip -- the row products of hk_rows_kernel.h for HK_Q4 organs.
#include "hk_rows_kernel.h"

namespace hk {
hipError_t launch_rows_q4(const RowsShape& sh, const RowsArgs& a, hipStream_t s) {
    return launch_rows_kind<HK_Q4>(sh, a, s);
}
}  // namespace hk
