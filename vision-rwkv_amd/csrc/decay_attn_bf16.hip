// decay_attn.h for __hip_bfloat16 rows.
#include "decay_attn.h"

namespace vrwkv {
namespace decay {
template int launch_decay<__hip_bfloat16>(const Params&, int, int, bool, hipStream_t);
}
}
