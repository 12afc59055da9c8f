// mx.h — microscaled types: their conversions, and declarations shared by the operators of a decoder block.
#pragma once

#include "mlxq_common.h"
#include "paged.h"

namespace mlxq {

typedef int i32x8 __attribute__((ext_vector_type(8)));

enum MxFormat : int { kE2M1 = MLXQ_MX_E2M1, kE4M3 = MLXQ_MX_E4M3 };

// The scale's exponent of a block whose largest magnitude has these f32 bits: the smallest e >= -127 with
// top / 2^e <= 6 = 1.5 * 2^2 (e2m1) or 448 = 1.75 * 2^8 (e4m3).
template <int FMT>
__device__ __forceinline__ int mx_exponent(uint32_t top) {
  const int e = (int)(top >> 23) - (FMT == kE2M1 ? 129 : 135) + ((top & 0x7fffffu) > (FMT == kE2M1 ? 0x400000u : 0x600000u));
  return max(e, -127);
}

// Two values, already divided by the scale, to codes (round to nearest even; nothing saturates).
__device__ __forceinline__ uint32_t mx_pack_e4m3(float a, float b, float c, float d) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
}
template <int BYTE>
__device__ __forceinline__ uint32_t mx_pack_e2m1(uint32_t w, float a, float b) {
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, a, b, 1.0f, BYTE);
}

// 2^(b - 127) as f32; 255 is NaN.
__device__ __forceinline__ float mx_scale(uint32_t b) {
  return b == 255 ? __uint_as_float(0x7fc00000u) : b == 0 ? __uint_as_float(0x00400000u) : __uint_as_float(b << 23);
}

// v of another lane by a data-parallel move within the vector unit (a shuffle goes through LDS and takes ten times as long).
template <int CTRL, typename V>
__device__ __forceinline__ V dpp_move(V v) {
  if constexpr (sizeof(V) == 4) {
    const int i = __builtin_bit_cast(int, v);
    return __builtin_bit_cast(V, __builtin_amdgcn_update_dpp(i, i, CTRL, 15, 15, false));
  } else {
    const u32x2 w = __builtin_bit_cast(u32x2, v);
    const int a = (int)w[0], b = (int)w[1];
    return __builtin_bit_cast(V, u32x2{(uint32_t)__builtin_amdgcn_update_dpp(a, a, CTRL, 15, 15, false),
                                       (uint32_t)__builtin_amdgcn_update_dpp(b, b, CTRL, 15, 15, false)});
  }
}
template <typename V>
__device__ __forceinline__ V lane_value(V v, int lane) {
  if constexpr (sizeof(V) == 4) {
    return __builtin_bit_cast(V, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
  } else {
    const u32x2 w = __builtin_bit_cast(u32x2, v);
    return __builtin_bit_cast(V, u32x2{(uint32_t)__builtin_amdgcn_readlane((int)w[0], lane),
                                       (uint32_t)__builtin_amdgcn_readlane((int)w[1], lane)});
  }
}
// v of all lanes of a group of LANES (2 to 64, aligned) combined by f, in each of them.
template <int LANES = 64, typename V, typename F>
__device__ __forceinline__ V lanes_reduce(V v, F&& f) {
  v = f(v, dpp_move<0xb1>(v));                            // quad_perm 1, 0, 3, 2
  if constexpr (LANES > 2) v = f(v, dpp_move<0x4e>(v));   // quad_perm 2, 3, 0, 1
  if constexpr (LANES > 4) v = f(v, dpp_move<0x141>(v));  // row_half_mirror
  if constexpr (LANES > 8) v = f(v, dpp_move<0x140>(v));  // row_mirror
  if constexpr (LANES == 32) {
    const V a = lane_value(v, 0), b = lane_value(v, 16), c = lane_value(v, 32), d = lane_value(v, 48);
    return (threadIdx.x & 32) ? f(c, d) : f(a, b);
  }
  if constexpr (LANES == 64) return f(f(lane_value(v, 0), lane_value(v, 16)), f(lane_value(v, 32), lane_value(v, 48)));
  return v;
}

// A microscaled matrix as kernels see it.
struct MxView {
  unsigned char* codes;
  unsigned char* scales;
  int64_t scale_stride;
};

// [token][head][feature] rows with an element stride each; p null: absent.
struct RowsView {
  unsigned char* p;
  int64_t ts, hs;
};

struct NormArgs {
  RowsView x, res, sum, y;
  MxView mx;
  const void* w;
  int w_dtype;  // -1: ones
  float eps;
  int64_t rows, first;  // first: this launch's first row
  int heads, D;
  Divisor by_heads;
};
int run_rms_norm(const NormArgs& a, int dtype, hipStream_t st);

struct NormGradArgs {
  RowsView dy, x, dsum, dx;
  const void* w;
  int w_dtype;
  void* dw;
  float* part;  // [parts, D]
  float eps;
  int64_t rows;
  int heads, D, parts;
  Divisor by_heads;
};
int64_t norm_grad_parts(int64_t rows, int64_t D, int dtype);
int run_rms_norm_backward(const NormGradArgs& a, int dtype, hipStream_t st);

int run_mx_quantize(const void* x, int dtype, int64_t rows, int64_t K, int64_t row_stride, const MxView& out, int format,
                    hipStream_t st);
int run_mx_dequantize(const MxView& x, int format, int64_t rows, int64_t K, void* out, int dtype, hipStream_t st);

struct RouteArgs {
  const void* logits;
  int64_t row_stride;
  int T, E, k;
  int scoring, groups, kept, best, normalize;
  float scale;
  const float* bias;
  const uint8_t* active;
  int32_t* ids;
  float* weights;
};
int run_route(const RouteArgs& a, int dtype, hipStream_t st);
size_t route_plan_workspace(int64_t choices, int64_t E);
int run_route_plan(const int32_t* ids, int64_t choices, int64_t E, int32_t* starts, int32_t* rows, void* ws, hipStream_t st);
int run_route_backward(const RouteArgs& a, int dtype, const float* dweights, void* dlogits, hipStream_t st);

// A product of microscaled operands, dense or of routed experts.
struct MxProduct {
  MxView x, w;
  int64_t M, N, K;       // M: rows of y (dense) or choices
  const void* bias;      // [E, N] or null
  int bias_dtype;
  void* y;               // [M, N]
  int y_dtype;
  // routed: E experts' runs of `rows`; E = 0: dense
  int E;
  const int32_t *starts, *rows;
  bool skip_none;        // rows of choices without an expert are not written
  Divisor by_choices;    // x row of a choice: choice / by_choices (1: a row for each choice)
};
int run_mx_product(const MxProduct& p, int format, hipStream_t st);
int run_mx_combine(const void* y, int dtype, const int32_t* ids, const float* weights, int64_t T, int64_t k, int64_t E,
                   int64_t N, void* out, hipStream_t st);

}  // namespace mlxq
