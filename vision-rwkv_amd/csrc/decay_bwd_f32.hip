// decay_bwd.h for float rows.
#include "decay_bwd.h"

namespace vrwkv {
namespace decay {
template int launch_decay_bwd<float>(const BwdParams&, bool, hipStream_t);
}
}
