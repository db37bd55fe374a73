// Tiled products of the learned projections for f16 rows and weights.
#include "project_tile.h"

namespace vdb {
PJ_DEFINE(f16, VDB_F16)
}  // namespace vdb
