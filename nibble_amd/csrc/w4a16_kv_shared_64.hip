// Attention behind shared prefixes: the kernels of head_dim 64.
#include "w4a16_kv_shared.h"

namespace w4a16 {

template void launch_shared<64>(const SharedCall&, int, int);

}  // namespace w4a16
