// scan.h and scan_short.h for float rows.
#include "scan_short.h"

namespace vrwkv {
namespace scan {
template int launch_forward<float>(const Params&, hipStream_t);
template int launch_short<float>(const Params&, int, hipStream_t);
}
}  // namespace vrwkv
