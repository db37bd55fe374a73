// Tiled products of the learned projections for bf16 rows and weights.
#include "project_tile.h"

namespace vdb {
PJ_DEFINE(bf16, VDB_BF16)
}  // namespace vdb
