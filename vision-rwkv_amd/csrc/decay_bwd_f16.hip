// decay_bwd.h for __half rows.
#include "decay_bwd.h"

namespace vrwkv {
namespace decay {
template int launch_decay_bwd<__half>(const BwdParams&, bool, hipStream_t);
}
}
