// Tiled products of the learned projections for f32 rows and weights.
#include "project_tile.h"

namespace vdb {
PJ_DEFINE(f32, VDB_F32)
}  // namespace vdb
