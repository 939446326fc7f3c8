// hk_rows_q8.hip -- the row products of hk_rows_kernel.h for HK_Q8 organs.
#include "hk_rows_kernel.h"

namespace hk {
hipError_t launch_rows_q8(const RowsShape& sh, const RowsArgs& a, hipStream_t s) {
    return launch_rows_kind<HK_Q8>(sh, a, s);
}
}  // namespace hk
