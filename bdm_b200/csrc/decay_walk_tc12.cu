// Tensor-core walk: up to 64 key columns, 65 to 128 value columns.
#include "decay_walk_tc.cuh"

namespace bdm {
namespace walk {
BDM_TC_DEFINE(1, 2)
}
}
