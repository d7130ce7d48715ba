// scan.h for __half rows.
#include "scan.h"

namespace vrwkv {
namespace scan {
template int launch_forward<__half>(const Params&, hipStream_t);
}
}  // namespace vrwkv
