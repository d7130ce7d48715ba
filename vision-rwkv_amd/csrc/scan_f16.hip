// scan.h and scan_short.h for __half rows.
#include "scan_short.h"

namespace vrwkv {
namespace scan {
template int launch_forward<__half>(const Params&, hipStream_t);
template int launch_short<__half>(const Params&, int, hipStream_t);
}
}  // namespace vrwkv
