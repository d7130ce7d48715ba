// scan.h for float rows.
#include "scan.h"

namespace vrwkv {
namespace scan {
template int launch_forward<float>(const Params&, hipStream_t);
}
}  // namespace vrwkv
