// scan_bwd.h for __half rows.
#include "scan_bwd.h"

namespace vrwkv {
namespace scan {
template int launch_backward<__half>(const BackParams&, int, hipStream_t);
}
}  // namespace vrwkv
