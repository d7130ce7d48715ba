// decay_bwd.h for __hip_bfloat16 rows.
#include "decay_bwd.h"

namespace vrwkv {
namespace decay {
template int launch_decay_bwd<__hip_bfloat16>(const BwdParams&, bool, hipStream_t);
}
}
