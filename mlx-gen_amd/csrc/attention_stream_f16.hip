// attention_stream_f16.hip — the f16 instances of the streaming attention kernel.
#include "attention_stream.h"

namespace mlxq {
int run_attn_stream_f16(const AttnArgs& a, const AttnPlan& plan, hipStream_t st) { return stream_of<_Float16>(a, plan, st); }
}  // namespace mlxq
