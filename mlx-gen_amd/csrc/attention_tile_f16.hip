// attention_tile_f16.hip — the f16 instances of the tiled attention kernel.
#include "attention_tile.h"

namespace mlxq {
int run_attn_tile_f16(const AttnArgs& a, const AttnPlan& plan, hipStream_t st) { return tile_of<_Float16>(a, plan, st); }
}  // namespace mlxq
