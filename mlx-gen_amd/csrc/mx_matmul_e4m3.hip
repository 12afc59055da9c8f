// mx_matmul_e4m3.hip — products with 8-bit activations, bf16 results (mx_matmul.h).
#include "mx_matmul.h"

namespace mlxq {
int run_mx_product_e4m3(const MxProduct& p, hipStream_t st) { return mx_product<kE4M3, false>(p, st); }
}  // namespace mlxq
