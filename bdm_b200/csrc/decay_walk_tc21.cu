// Tensor-core walk: 65 to 128 key columns, up to 64 value columns.
#include "decay_walk_tc.cuh"

namespace bdm {
namespace walk {
BDM_TC_DEFINE(2, 1)
}
}
