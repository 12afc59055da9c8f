// mx_quantize.hip — quantisation to microscaled codes, and back.
//
// A lane holds 8 values (e2m1: 4 bytes of codes, e4m3: 8), four neighbouring lanes a block of 32: its largest
// magnitude takes two exchanges, its exponent is read off the bits of that maximum, and the values are divided
// exactly (ldexp) and rounded by the conversion instructions.  Both directions move every byte once and are bound
// by HBM; units of 8 values are numbered over the whole matrix, so that rows need not fill a workgroup.  Four units a thread
// have their loads in flight together: 5119 x 13824 f32 to e2m1 65 us, 4.9 TB/s, and back to bf16 27 us, 6.6 TB/s, most of it
// writes (a large copy 5.2, a fill 6.9).
#include <algorithm>

#include "mx.h"

namespace mlxq {

constexpr int kUnits = 4;  // of 8 values a thread, their loads in flight together

template <typename T>
struct Eight {
  u32x4 v[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) v[i] = load_chunk(p + i * Elem<T>::C);
  }
  __device__ __forceinline__ float get(int e) const { return Elem<T>::get(v[e / Elem<T>::C], e % Elem<T>::C); }
};

// Units [first, first + n) of rows of K / 8: n below 2^30.
template <typename T, int FMT>
__global__ __launch_bounds__(256) void mx_quantize_kernel(const T* __restrict__ x, int64_t row_stride, MxView out, int n,
                                                          int row_units, Divisor by_row, int K) {
  const int base = blockIdx.x * (256 * kUnits) + threadIdx.x;
  Eight<T> in[kUnits];
  int row[kUnits], at[kUnits];
#pragma unroll
  for (int k = 0; k < kUnits; ++k) {
    const int u = min(base + k * 256, n - 1);
    row[k] = by_row.div(u);
    at[k] = u - row[k] * row_units;
    in[k].load(x + row[k] * row_stride + at[k] * 8);
  }
#pragma unroll
  for (int k = 0; k < kUnits; ++k) {
    if (base + k * 256 >= n) break;  // whole blocks: n is a multiple of 4
    uint32_t top = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(in[k].get(e)) & 0x7fffffffu);
    top = lanes_reduce<4>(top, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
    const bool bad = top >= 0x7f800000u;
    const int ex = mx_exponent<FMT>(top);
    float f[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = bad ? 0.0f : __builtin_amdgcn_ldexpf(in[k].get(e), -ex);
    unsigned char* codes = out.codes + (int64_t)row[k] * (FMT == kE2M1 ? K / 2 : K);
    if constexpr (FMT == kE2M1) {
      uint32_t w = mx_pack_e2m1<0>(0, f[0], f[1]);
      w = mx_pack_e2m1<1>(w, f[2], f[3]);
      w = mx_pack_e2m1<2>(w, f[4], f[5]);
      w = mx_pack_e2m1<3>(w, f[6], f[7]);
      *reinterpret_cast<uint32_t*>(codes + at[k] * 4) = w;
    } else {
      *reinterpret_cast<u32x2*>(codes + at[k] * 8) =
          u32x2{mx_pack_e4m3(f[0], f[1], f[2], f[3]), mx_pack_e4m3(f[4], f[5], f[6], f[7])};
    }
    if ((at[k] & 3) == 0) {
      unsigned char* s = out.scales + row[k] * out.scale_stride;
      const int block = at[k] >> 2;
      s[block] = bad ? 255 : (unsigned char)(ex + 127);
      if (block == (K >> 5) - 1)  // up to the next multiple of 4
        for (int i = block + 1; i < ((K >> 5) + 3 & ~3); ++i) s[i] = 0;
    }
  }
}

template <typename T, int FMT>
__global__ __launch_bounds__(256) void mx_dequantize_kernel(MxView x, T* __restrict__ out, int n, int row_units,
                                                            Divisor by_row, int K) {
  const int base = blockIdx.x * (256 * kUnits) + threadIdx.x;
  u32x2 code[kUnits];
  uint32_t scale[kUnits];
  int64_t to[kUnits];
#pragma unroll
  for (int k = 0; k < kUnits; ++k) {
    const int u = min(base + k * 256, n - 1), row = by_row.div(u), at = u - row * row_units;
    const unsigned char* c = x.codes + (int64_t)row * (FMT == kE2M1 ? K / 2 : K);
    if constexpr (FMT == kE2M1) code[k][0] = *reinterpret_cast<const uint32_t*>(c + at * 4);
    else code[k] = *reinterpret_cast<const u32x2*>(c + at * 8);
    scale[k] = x.scales[row * x.scale_stride + (at >> 2)];
    to[k] = (int64_t)row * K + at * 8;
  }
#pragma unroll
  for (int k = 0; k < kUnits; ++k) {
    if (base + k * 256 >= n) break;
    f32x2 p[4];
    if constexpr (FMT == kE2M1) {
      p[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code[k][0], 1.0f, 0);
      p[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code[k][0], 1.0f, 1);
      p[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code[k][0], 1.0f, 2);
      p[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code[k][0], 1.0f, 3);
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        p[2 * i] = __builtin_amdgcn_cvt_pk_f32_fp8((int)code[k][i], false);
        p[2 * i + 1] = __builtin_amdgcn_cvt_pk_f32_fp8((int)code[k][i], true);
      }
    }
    float f[8];
#pragma unroll
    for (int e = 0; e < 8; ++e)
      f[e] = scale[k] == 255 ? __uint_as_float(0x7fc00000u) : __builtin_amdgcn_ldexpf(p[e / 2][e % 2], (int)scale[k] - 127);
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) store_chunk(out + to[k] + i * Elem<T>::C, pack_chunk<T>(f + i * Elem<T>::C));
  }
}

namespace {

// Calls launch(first row, rows) on slices whose units are counted in 30 bits.
template <typename F>
int in_slices(const char* what, int64_t rows, int64_t K, F&& launch) {
  const int64_t most = std::max<int64_t>(1, (1 << 30) / (K / 8) - 1);
  for (int64_t r = 0; r < rows; r += most) {
    const int64_t m = std::min(most, rows - r);
    launch(r, (int)(m * (K / 8)));
    if (int rc = check_launch(what)) return rc;
  }
  return MLXQ_OK;
}

template <typename T>
int quantize(const T* x, int64_t rows, int64_t K, int64_t row_stride, const MxView& out, int format, hipStream_t st) {
  return in_slices("mx_quantize", rows, K, [&](int64_t r, int n) {
    MxView o = out;
    o.codes += r * (format == kE2M1 ? K / 2 : K);
    o.scales += r * out.scale_stride;
    const unsigned grid = (unsigned)((n + 256 * kUnits - 1) / (256 * kUnits));
    if (format == kE2M1)
      mx_quantize_kernel<T, kE2M1><<<grid, 256, 0, st>>>(x + r * row_stride, row_stride, o, n, (int)(K / 8), Divisor(K / 8), (int)K);
    else
      mx_quantize_kernel<T, kE4M3><<<grid, 256, 0, st>>>(x + r * row_stride, row_stride, o, n, (int)(K / 8), Divisor(K / 8), (int)K);
  });
}

template <typename T>
int dequantize(const MxView& x, int format, int64_t rows, int64_t K, T* out, hipStream_t st) {
  return in_slices("mx_dequantize", rows, K, [&](int64_t r, int n) {
    MxView v = x;
    v.codes += r * (format == kE2M1 ? K / 2 : K);
    v.scales += r * x.scale_stride;
    const unsigned grid = (unsigned)((n + 256 * kUnits - 1) / (256 * kUnits));
    if (format == kE2M1)
      mx_dequantize_kernel<T, kE2M1><<<grid, 256, 0, st>>>(v, out + r * K, n, (int)(K / 8), Divisor(K / 8), (int)K);
    else
      mx_dequantize_kernel<T, kE4M3><<<grid, 256, 0, st>>>(v, out + r * K, n, (int)(K / 8), Divisor(K / 8), (int)K);
  });
}

}  // namespace

int run_mx_quantize(const void* x, int dtype, int64_t rows, int64_t K, int64_t row_stride, const MxView& out, int format,
                    hipStream_t st) {
  if (dtype == MLXQ_BFLOAT16) return quantize((const uint16_t*)x, rows, K, row_stride, out, format, st);
  if (dtype == MLXQ_FLOAT16) return quantize((const _Float16*)x, rows, K, row_stride, out, format, st);
  return quantize((const float*)x, rows, K, row_stride, out, format, st);
}

int run_mx_dequantize(const MxView& x, int format, int64_t rows, int64_t K, void* out, int dtype, hipStream_t st) {
  if (dtype == MLXQ_BFLOAT16) return dequantize(x, format, rows, K, (uint16_t*)out, st);
  if (dtype == MLXQ_FLOAT16) return dequantize(x, format, rows, K, (_Float16*)out, st);
  return dequantize(x, format, rows, K, (float*)out, st);
}

}  // namespace mlxq
