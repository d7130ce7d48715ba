// decay_attn.h for __half rows.
#include "decay_attn.h"

namespace vrwkv {
namespace decay {
template int launch_decay<__half>(const Params&, int, int, bool, hipStream_t);
}
}
