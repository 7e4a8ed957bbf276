// Attention behind shared prefixes: the kernels of head_dim 256.
#include "w4a16_kv_shared.h"

namespace w4a16 {

template void launch_shared<256>(const SharedCall&, int, int);

}  // namespace w4a16
