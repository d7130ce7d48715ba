// scan_bwd.h for float rows.
#include "scan_bwd.h"

namespace vrwkv {
namespace scan {
template int launch_backward<float>(const BackParams&, int, hipStream_t);
}
}  // namespace vrwkv
