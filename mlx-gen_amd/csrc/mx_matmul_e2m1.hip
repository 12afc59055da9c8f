// mx_matmul_e2m1.hip — products with 4-bit activations (mx_matmul.h).
#include "mx_matmul.h"

namespace mlxq {
int run_mx_product_e2m1(const MxProduct& p, hipStream_t st) { return mx_product<kE2M1, false>(p, st); }
}  // namespace mlxq
