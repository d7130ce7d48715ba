// scan.h and scan_short.h for __hip_bfloat16 rows.
#include "scan_short.h"

namespace vrwkv {
namespace scan {
template int launch_forward<__hip_bfloat16>(const Params&, hipStream_t);
template int launch_short<__hip_bfloat16>(const Params&, int, hipStream_t);
}
}  // namespace vrwkv
