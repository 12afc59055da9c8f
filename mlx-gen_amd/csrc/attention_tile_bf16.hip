// attention_tile_bf16.hip — the bf16 instances of the tiled attention kernel.
#include "attention_tile.h"

namespace mlxq {
int run_attn_tile_bf16(const AttnArgs& a, const AttnPlan& plan, hipStream_t st) { return tile_of<uint16_t>(a, plan, st); }
}  // namespace mlxq
