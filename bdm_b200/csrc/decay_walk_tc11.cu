// Tensor-core walk: up to 64 key columns, up to 64 value columns.
#include "decay_walk_tc.cuh"

namespace bdm {
namespace walk {
BDM_TC_DEFINE(1, 1)
}
}
