// scan.h for __hip_bfloat16 rows.
#include "scan.h"

namespace vrwkv {
namespace scan {
template int launch_forward<__hip_bfloat16>(const Params&, hipStream_t);
}
}  // namespace vrwkv
