// mx_matmul_e4m3_f32.hip — products with 8-bit activations, f32 and fp16 results (mx_matmul.h).
#include "mx_matmul.h"

namespace mlxq {
int run_mx_product_e4m3_f32(const MxProduct& p, hipStream_t st) { return mx_product<kE4M3, true>(p, st); }
}  // namespace mlxq
