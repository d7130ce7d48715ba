// scan_bwd.h for __hip_bfloat16 rows.
#include "scan_bwd.h"

namespace vrwkv {
namespace scan {
template int launch_backward<__hip_bfloat16>(const BackParams&, int, hipStream_t);
}
}  // namespace vrwkv
