// attention_stream_bf16.hip — the bf16 instances of the streaming attention kernel.
#include "attention_stream.h"

namespace mlxq {
int run_attn_stream_bf16(const AttnArgs& a, const AttnPlan& plan, hipStream_t st) { return stream_of<uint16_t>(a, plan, st); }
}  // namespace mlxq
