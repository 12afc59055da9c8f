// attention_stream_f32.hip — the f32 instances of the streaming attention kernel.
#include "attention_stream.h"

namespace mlxq {
int run_attn_stream_f32(const AttnArgs& a, const AttnPlan& plan, hipStream_t st) { return stream_of<float>(a, plan, st); }
}  // namespace mlxq
