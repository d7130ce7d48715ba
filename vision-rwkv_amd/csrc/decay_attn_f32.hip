// decay_attn.h for float rows.
#include "decay_attn.h"

namespace vrwkv {
namespace decay {
template int launch_decay<float>(const Params&, int, int, bool, hipStream_t);
}
}
