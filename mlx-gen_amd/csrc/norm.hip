// norm.hip — root-mean-square norms with the residual's addition, their 8-bit results, and their gradient.
//
//   y = h (mean(h^2) + eps)^(-1/2) w,  h = x + residual
//   dx = r (g - n mean(g n)) + dsum,  n = x r,  g = dy w;   dw = sum of dy n over the rows
//
// The gradient is multiplied in this order, mean(g n) being mean(g x) r: r^3 is subnormal from rows of 5e12 on, and infinite below
// 1e-13 with eps 0, where r, the sums and the result are ordinary numbers.
//
// A row is held in registers by 8 to 64 lanes of a wave (short rows: several to a wave), by a workgroup of 256 or by
// one of 512, in 16-byte pieces, and is read once; the sums take exchanges within a wave and one step through LDS
// between waves.  Both directions are bound by HBM: 8190 x 5120 bf16 29 us, 5.8 TB/s; with a residual 60, 5.6; with that to
// 8 bits 55, 5.3 (without one 36: the rounding's vector instructions then take as long as the memory).  Pieces are loaded at the element's alignment, so that rows of odd
// length or stride take the same path; only a row's last, partial piece goes element by element.
//
// The gradient of the weight is a sum over all rows: each workgroup walks many rows and holds its features' sums in
// registers; they go to the workspace once and a second launch adds them up in a fixed order.  Two workgroups of 256 a CU
// hide each other's reductions, and a row's loads go out once the sums of the row before are there: 8190 x 5120 bf16
// with dsum 71 us with the second launch, 4.7 TB/s, a large copy's rate (loads at the row's own start 75, a whole row
// ahead in registers 71, three workgroups a CU 85).
#include <algorithm>

#include "mx.h"

namespace mlxq {

namespace {

template <typename T>
constexpr int kC = Elem<T>::C;

// A row's pieces of 16 bytes, the i-th of a lane at element (i LANES + lane) C.  Every load is made, so that all of them are
// in flight together: a piece that reaches past the row's end is read from further to the left, and set_right once it is
// used; one that begins past it holds anything.  Rows shorter than a piece go element by element.
template <typename T, int LANES, int CH>
__device__ __forceinline__ void load_row(u32x4 (&v)[CH], const T* row, int lane, int D) {
  if (D >= kC<T>) {
#pragma unroll
    for (int i = 0; i < CH; ++i) __builtin_memcpy(&v[i], row + min((i * LANES + lane) * kC<T>, D - kC<T>), 16);
  } else {
    v[0] = u32x4{0, 0, 0, 0};
    for (int i = 0; i < D; ++i) {
      if constexpr (sizeof(T) == 4) v[0][i] = __float_as_uint(row[i]);
      else v[0][i / 2] |= (uint32_t)__builtin_bit_cast(uint16_t, row[i]) << 16 * (i % 2);
    }
  }
}
template <typename T>
__device__ __forceinline__ void set_right(u32x4& v, int e, int D) {
  if (D >= kC<T> && e < D && e + kC<T> > D)
    for (int k = e + kC<T> - D; k > 0; --k) {
      if constexpr (sizeof(T) == 4) v = u32x4{v[1], v[2], v[3], 0};
      else v = u32x4{v[0] >> 16 | v[1] << 16, v[1] >> 16 | v[2] << 16, v[2] >> 16 | v[3] << 16, v[3] >> 16};
    }
}
template <typename T>
__device__ __forceinline__ void store_piece(T* row, int e, int D, const u32x4& v) {
  if (e + kC<T> <= D) {
    __builtin_memcpy(row + e, &v, 16);
  } else if (e < D) {
#pragma unroll
    for (int i = 0; i < kC<T>; ++i)
      if (e + i < D) {
        if constexpr (sizeof(T) == 4) row[e + i] = __uint_as_float(v[i]);
        else row[e + i] = __builtin_bit_cast(T, (uint16_t)(v[i / 2] >> 16 * (i % 2)));
      }
  }
}

template <typename W, int C>
__device__ __forceinline__ void load_weights_of(const W* w, int e, int D, float (&f)[C]) {
  if (D >= C) {
    const int at = min(e, D - C);
    constexpr int N = C > kC<W> ? C / kC<W> : 1, B = C < kC<W> ? C * (int)sizeof(W) : 16;
    u32x4 v[N];
#pragma unroll
    for (int k = 0; k < N; ++k) __builtin_memcpy(&v[k], w + at + k * kC<W>, B);
#pragma unroll
    for (int i = 0; i < C; ++i) f[i] = Elem<W>::get(v[i / kC<W>], i % kC<W>);
    if (e < D)
      for (int k = e - at; k > 0; --k) {
#pragma unroll
        for (int i = 0; i + 1 < C; ++i) f[i] = f[i + 1];
        f[C - 1] = 0.0f;
      }
  } else {
#pragma unroll
    for (int i = 0; i < C; ++i) f[i] = e + i < D ? Act<W>::ld(w, e + i) : 0.0f;
  }
}
// C weights from feature e on; ones without a weight.
template <int C>
__device__ __forceinline__ void load_weights(const void* w, int dtype, int e, int D, float (&f)[C]) {
  if (dtype < 0) {
#pragma unroll
    for (int i = 0; i < C; ++i) f[i] = 1.0f;
  } else if (dtype == MLXQ_BFLOAT16) {
    load_weights_of((const uint16_t*)w, e, D, f);
  } else if (dtype == MLXQ_FLOAT16) {
    load_weights_of((const _Float16*)w, e, D, f);
  } else {
    load_weights_of((const float*)w, e, D, f);
  }
}

// The sums of v over a row's LANES lanes, in every lane.  Rows of several waves go through `slot`, which nothing
// may still be reading: callers take turns between two.
template <int LANES, int N, typename V>
__device__ __forceinline__ void row_sum(V (&v)[N], V* slot) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = lanes_reduce<(LANES < 64 ? LANES : 64)>(v[i], [](V a, V b) { return a + b; });
  if constexpr (LANES > 64) {
    const int w = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0)
#pragma unroll
      for (int i = 0; i < N; ++i) slot[w * N + i] = v[i];
    // Of LDS alone: a barrier for all memory would wait for the last row's stores too.
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = slot[i];
#pragma unroll
    for (int k = 1; k < LANES / 64; ++k)
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] += slot[k * N + i];
  }
}

// The f32 that has y's leading bits and, where any were lost, an odd last one: rounding it to fewer bits is
// rounding y.
__device__ __forceinline__ float round_to_odd(double y) {
  const float f = (float)y;
  const double back = (double)f;
  uint32_t b = __float_as_uint(f);
  b -= fabs(back) > fabs(y);
  return __uint_as_float(back != y ? b | 1u : b);
}

__device__ __forceinline__ double ldexp_f64(double v, int e) { return __builtin_amdgcn_ldexp(v, e); }

template <typename T>
__device__ __forceinline__ T* row_of(const RowsView& v, int t, int h) {
  return reinterpret_cast<T*>(v.p) + t * v.ts + h * v.hs;
}

template <typename T, int LANES, int CH, bool MX>
__global__ __launch_bounds__(LANES > 256 ? LANES : 256) void rms_norm_kernel(NormArgs a) {
  constexpr int C = kC<T>, R = LANES > 256 ? 1 : 256 / LANES, TW = LANES / 64 > 0 ? LANES / 64 : 1;
  using Sum = typename std::conditional<MX, double, float>::type;
  __shared__ Sum slot[TW];
  const int lane = threadIdx.x % LANES, D = a.D;
  const int64_t at = a.first + (int64_t)blockIdx.x * R + threadIdx.x / LANES;
  const bool live = at < a.rows;
  const int row = (int)(live ? at : a.rows - 1);
  const int t = a.by_heads.div(row), h = row - t * a.heads;
  const T* x = row_of<const T>(a.x, t, h);
  u32x4 v[CH];
  load_row<T, LANES>(v, x, lane, D);
  if (a.res.p) {
    u32x4 r[CH];
    load_row<T, LANES>(r, row_of<const T>(a.res, t, h), lane, D);
    T* sum = row_of<T>(a.sum, t, h);
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int e0 = (i * LANES + lane) * C;
      if (e0 >= D) continue;
      float f[C];
#pragma unroll
      for (int e = 0; e < C; ++e) f[e] = Elem<T>::get(v[i], e) + Elem<T>::get(r[i], e);
      v[i] = pack_chunk<T>(f);
      set_right<T>(v[i], e0, D);
      if (live) store_piece(sum, e0, D, v[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < CH; ++i) set_right<T>(v[i], (i * LANES + lane) * C, D);
  }
  // The weights of short rows are under way while the sum is taken.
  constexpr bool EARLY = CH <= 2;
  float w[EARLY ? CH : 1][C];
  if constexpr (EARLY)
#pragma unroll
    for (int i = 0; i < CH; ++i) load_weights(a.w, a.w_dtype, (i * LANES + lane) * C, D, w[i]);
  Sum s[1] = {0};
#pragma unroll
  for (int i = 0; i < CH; ++i)
    if ((i * LANES + lane) * C < D)
#pragma unroll
      for (int e = 0; e < C; ++e) {
        const Sum f = Elem<T>::get(v[i], e);
        s[0] += f * f;
      }
  row_sum<LANES>(s, slot);
  if constexpr (!MX) {
    const float r = 1.0f / sqrtf(s[0] / (float)D + a.eps);
    if (!live) return;
    T* y = row_of<T>(a.y, t, h);
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int e0 = (i * LANES + lane) * C;
      if (e0 >= D) break;
      if constexpr (!EARLY) load_weights(a.w, a.w_dtype, e0, D, w[0]);
      float f[C];
#pragma unroll
      for (int e = 0; e < C; ++e) f[e] = Elem<T>::get(v[i], e) * r * w[EARLY ? i : 0][e];
      store_piece(y, e0, D, pack_chunk<T>(f));
    }
  } else {
    // As in 64 bits up to the rounding to 8: which code a value next to a border gets, and a block its scale, is then
    // not a matter of the order of the sum.  In 32 bits a value is off by less than 2^-22 of it (its two products, r's rounding),
    // so where codes and scale are the same 2^-21 to either side they are right; one piece of a wave in a hundred has
    // another, and takes the 64 bits (8190 x 5120 bf16: all pieces in 64 bits 43 us).
    const double r = 1.0 / sqrt(s[0] / (double)D + (double)a.eps);
    const float r32 = (float)r;
    if (!live) return;
    unsigned char* codes = a.mx.codes + (int64_t)row * D;
    unsigned char* scales = a.mx.scales + row * a.mx.scale_stride;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int e0 = (i * LANES + lane) * C;
      if (e0 >= D) break;  // D is a multiple of 32: whole blocks of lanes
      if constexpr (!EARLY) load_weights(a.w, a.w_dtype, e0, D, w[0]);
      uint32_t code[C / 4];
      int ex;
      bool bad = false, sure = r32 >= 0x1p-60f && r32 <= 0x1p60f;
      {
        float y[C];
        uint32_t top = 0;
#pragma unroll
        for (int e = 0; e < C; ++e) {
          const float x = Elem<T>::get(v[i], e), n = x * r32, weight = w[EARLY ? i : 0][e];
          y[e] = n * weight;
          // a product next to f32's smallest numbers is off by more; NaN is never sure
          sure &= (fabsf(n) >= 0x1p-100f && fabsf(y[e]) >= 0x1p-100f) || (x == 0.0f && fabsf(weight) < INFINITY);
          top = max(top, __float_as_uint(y[e]) & 0x7fffffffu);
        }
        top = lanes_reduce<32 / C>(top, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
        ex = mx_exponent<kE4M3>(top + 16);
        sure &= top + 16 < 0x7f800000u && ex == mx_exponent<kE4M3>(max(top, 16u) - 16);
        float lo[C], hi[C];
#pragma unroll
        for (int e = 0; e < C; ++e) {
          const float f = __builtin_amdgcn_ldexpf(y[e], -ex);
          lo[e] = f * (1.0f - 0x1p-21f);
          hi[e] = f * (1.0f + 0x1p-21f);
        }
#pragma unroll
        for (int k = 0; k < C; k += 4) {
          code[k / 4] = mx_pack_e4m3(lo[k], lo[k + 1], lo[k + 2], lo[k + 3]);
          sure &= code[k / 4] == mx_pack_e4m3(hi[k], hi[k + 1], hi[k + 2], hi[k + 3]);
        }
      }
      if (__any(!sure)) {
        double y[C];
        unsigned long long top = 0;
#pragma unroll
        for (int e = 0; e < C; ++e) {
          y[e] = (double)Elem<T>::get(v[i], e) * r * (double)w[EARLY ? i : 0][e];
          top = max(top, (unsigned long long)__double_as_longlong(y[e]) & 0x7fffffffffffffffull);
        }
        top = lanes_reduce<32 / C>(top, [](unsigned long long a, unsigned long long b) { return a > b ? a : b; });
        // 448 = 1.75 * 2^8; magnitudes past f32 are as infinite as f32's infinity
        ex = max((int)(top >> 52) - 1023 - 8 + ((top & 0xfffffffffffffull) > 0xc000000000000ull), -127);
        bad = top >= 0x47f0000000000000ull;
        float f[C];
#pragma unroll
        for (int e = 0; e < C; ++e) f[e] = bad ? 0.0f : round_to_odd(ldexp_f64(y[e], -ex));
#pragma unroll
        for (int k = 0; k < C; k += 4) code[k / 4] = mx_pack_e4m3(f[k], f[k + 1], f[k + 2], f[k + 3]);
      }
      __builtin_memcpy(codes + e0, code, C);
      if (e0 % 32 == 0) {
        scales[e0 / 32] = bad ? 255 : (unsigned char)(ex + 127);
        if (e0 + 32 == D)
          for (int b = D / 32; b < (D / 32 + 3 & ~3); ++b) scales[b] = 0;
      }
    }
  }
}

template <typename T, int LANES, int CH>
__global__ __launch_bounds__(LANES > 256 ? LANES : 256) void rms_norm_grad_kernel(NormGradArgs a) {
  constexpr int C = kC<T>, R = LANES > 256 ? 1 : 256 / LANES, TW = LANES / 64 > 0 ? LANES / 64 : 1;
  __shared__ float slot[2][2 * TW];
  const int lane = threadIdx.x % LANES, D = a.D;
  const bool has_w = a.w_dtype >= 0;
  float w[CH][C], dw[CH][C];
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    load_weights(a.w, a.w_dtype, (i * LANES + lane) * C, D, w[i]);
#pragma unroll
    for (int e = 0; e < C; ++e) dw[i][e] = 0.0f;
  }
  u32x4 x[CH], dy[CH], ds[CH];
  auto load = [&](int64_t at) {
    const int row = (int)min(at, a.rows - 1), t = a.by_heads.div(row), h = row - t * a.heads;
    load_row<T, LANES>(x, row_of<const T>(a.x, t, h), lane, D);
    load_row<T, LANES>(dy, row_of<const T>(a.dy, t, h), lane, D);
    if (a.dsum.p) load_row<T, LANES>(ds, row_of<const T>(a.dsum, t, h), lane, D);
  };
  const int64_t step = (int64_t)gridDim.x * R;
  int64_t first = (int64_t)blockIdx.x * R;
  int turn = 0;
  load(first + threadIdx.x / LANES);
  for (; first < a.rows; first += step, turn ^= 1) {  // the same count for every lane
    const int64_t at = first + threadIdx.x / LANES;
    const bool live = at < a.rows;
    float s[2] = {0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int e0 = (i * LANES + lane) * C;
      if (e0 >= D) continue;
      set_right<T>(x[i], e0, D);
      set_right<T>(dy[i], e0, D);
#pragma unroll
      for (int e = 0; e < C; ++e) {
        const float xv = Elem<T>::get(x[i], e);
        s[0] = fmaf(xv, xv, s[0]);
        s[1] = fmaf(Elem<T>::get(dy[i], e) * w[i][e], xv, s[1]);
      }
    }
    row_sum<LANES>(s, slot[turn]);
    // The next row's loads go out beside this one's results.
    u32x4 x0[CH], dy0[CH], ds0[CH];
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      x0[i] = x[i];
      dy0[i] = dy[i];
      ds0[i] = ds[i];
    }
    if (first + step < a.rows) load(at + step);
    const float r = 1.0f / sqrtf(s[0] / (float)D + a.eps), mean = s[1] / (float)D * r;
    if (!live) continue;
    const int row = (int)at, t = a.by_heads.div(row), h = row - t * a.heads;
    T* dx = row_of<T>(a.dx, t, h);
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int e0 = (i * LANES + lane) * C;
      if (e0 >= D) continue;
      float f[C];
#pragma unroll
      for (int e = 0; e < C; ++e) {
        const float n = Elem<T>::get(x0[i], e) * r, g = Elem<T>::get(dy0[i], e);
        f[e] = r * fmaf(-n, mean, g * w[i][e]);
        dw[i][e] = fmaf(g, n, dw[i][e]);
      }
      if (a.dsum.p) {
        set_right<T>(ds0[i], e0, D);
#pragma unroll
        for (int e = 0; e < C; ++e) f[e] += Elem<T>::get(ds0[i], e);
      }
      store_piece(dx, e0, D, pack_chunk<T>(f));
    }
  }
  if (!has_w) return;
  // The workgroup's rows are added up, then its sums are one row of the workspace.
  float* part = a.part + (int64_t)blockIdx.x * D;
  if constexpr (R > 1) {
    __shared__ float all[R][LANES * CH * C];
#pragma unroll
    for (int i = 0; i < CH; ++i)
#pragma unroll
      for (int e = 0; e < C; ++e) all[threadIdx.x / LANES][(i * LANES + lane) * C + e] = dw[i][e];
    __syncthreads();
    for (int e = threadIdx.x; e < D; e += 256) {
      float s = 0.0f;
      for (int k = 0; k < R; ++k) s += all[k][e];
      part[e] = s;
    }
  } else {
#pragma unroll
    for (int i = 0; i < CH; ++i)
#pragma unroll
      for (int e = 0; e < C; ++e) {
        const int at = (i * LANES + lane) * C + e;
        if (at < D) part[at] = dw[i][e];
      }
  }
}

// Rows of more than 2048 pieces leave no registers for themselves: a workgroup of sixteen waves reads them twice, the second time
// from the cache, and the weight's sums are in LDS, each lane's its own.
template <typename T>
__global__ __launch_bounds__(1024) void rms_norm_grad_long_kernel(NormGradArgs a) {
  constexpr int C = kC<T>, LANES = 1024;
  __shared__ float slot[2][2 * LANES / 64];
  __shared__ __align__(16) float dw[32768];
  const int D = a.D, e_first = threadIdx.x * C;
  for (int e0 = e_first; e0 < D; e0 += LANES * C)
#pragma unroll
    for (int e = 0; e < C; ++e) dw[e0 + e] = 0.0f;
  int turn = 0;
  for (int row = blockIdx.x; row < a.rows; row += gridDim.x, turn ^= 1) {
    const int t = a.by_heads.div(row), h = row - t * a.heads;
    const T *x = row_of<const T>(a.x, t, h), *dy = row_of<const T>(a.dy, t, h);
    const T* ds = a.dsum.p ? row_of<const T>(a.dsum, t, h) : nullptr;
    T* dx = row_of<T>(a.dx, t, h);
    float s[2] = {0.0f, 0.0f};
#pragma unroll 2
    for (int e0 = e_first; e0 < D; e0 += LANES * C) {
      u32x4 xv[1], g[1];
      float w[C];
      load_row<T, 1>(xv, x, e0 / C, D);
      load_row<T, 1>(g, dy, e0 / C, D);
      load_weights(a.w, a.w_dtype, e0, D, w);
      set_right<T>(xv[0], e0, D);
      set_right<T>(g[0], e0, D);
#pragma unroll
      for (int e = 0; e < C; ++e) {
        const float v = Elem<T>::get(xv[0], e);
        s[0] = fmaf(v, v, s[0]);
        s[1] = fmaf(Elem<T>::get(g[0], e) * w[e], v, s[1]);
      }
    }
    row_sum<LANES>(s, slot[turn]);
    const float r = 1.0f / sqrtf(s[0] / (float)D + a.eps), mean = s[1] / (float)D * r;
#pragma unroll 2
    for (int e0 = e_first; e0 < D; e0 += LANES * C) {
      u32x4 xv[1], g[1], d[1] = {u32x4{0, 0, 0, 0}};
      float w[C], f[C];
      load_row<T, 1>(xv, x, e0 / C, D);
      load_row<T, 1>(g, dy, e0 / C, D);
      if (ds) load_row<T, 1>(d, ds, e0 / C, D);
      load_weights(a.w, a.w_dtype, e0, D, w);
      set_right<T>(xv[0], e0, D);
      set_right<T>(g[0], e0, D);
      if (ds) set_right<T>(d[0], e0, D);
#pragma unroll
      for (int e = 0; e < C; ++e) {
        const float n = Elem<T>::get(xv[0], e) * r, gv = Elem<T>::get(g[0], e);
        f[e] = r * fmaf(-n, mean, gv * w[e]);
        dw[e0 + e] = fmaf(gv, n, dw[e0 + e]);
        if (ds) f[e] += Elem<T>::get(d[0], e);
      }
      store_piece(dx, e0, D, pack_chunk<T>(f));
    }
  }
  if (a.w_dtype < 0) return;
  float* part = a.part + (int64_t)blockIdx.x * D;
  for (int e0 = e_first; e0 < D; e0 += LANES * C)
#pragma unroll
    for (int e = 0; e < C; ++e)
      if (e0 + e < D) part[e0 + e] = dw[e0 + e];
}

// 64 features a workgroup, its sixteen waves a sixteenth of the parts each.
template <typename W>
__global__ __launch_bounds__(1024) void rms_norm_weight_kernel(const float* __restrict__ part, W* __restrict__ dw, int D, int parts) {
  __shared__ float s[16][64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, e = blockIdx.x * 64 + lane;
  float sum = 0.0f;
  if (e < D) {
#pragma unroll 8
    for (int k = w; k < parts; k += 16) sum += part[(int64_t)k * D + e];
  }
  s[w][lane] = sum;
  __syncthreads();
  if (w == 0 && e < D) {
#pragma unroll
    for (int k = 1; k < 16; ++k) sum += s[k][lane];
    Act<W>::st(dw, e, sum);
  }
}

// Lanes of a row and pieces of a lane, by the pieces of a row.
template <typename F>
int by_pieces(int64_t pieces, F&& f) {
#define MLXQ_ROW(MOST, LANES, CH) \
  if (pieces <= MOST) return f(std::integral_constant<int, LANES>{}, std::integral_constant<int, CH>{})
  MLXQ_ROW(8, 8, 1);
  MLXQ_ROW(16, 16, 1);
  MLXQ_ROW(32, 32, 1);
  MLXQ_ROW(64, 64, 1);
  MLXQ_ROW(128, 64, 2);
  MLXQ_ROW(256, 256, 1);
  MLXQ_ROW(512, 256, 2);
  MLXQ_ROW(1024, 256, 4);
  MLXQ_ROW(2048, 512, 4);
  MLXQ_ROW(4096, 512, 8);
  return f(std::integral_constant<int, 512>{}, std::integral_constant<int, 16>{});
#undef MLXQ_ROW
}

template <typename T>
int norm(const NormArgs& a, hipStream_t st) {
  return by_pieces((a.D + kC<T> - 1) / kC<T>, [&](auto lanes, auto ch) {
    constexpr int LANES = decltype(lanes)::value, CH = decltype(ch)::value, R = LANES > 256 ? 1 : 256 / LANES;
    int rc = MLXQ_OK;
    if constexpr (LANES * CH * kC<T> <= 32768) {
      constexpr int threads = LANES > 256 ? LANES : 256;
      NormArgs part = a;
      rc = in_launches("rms_norm", (a.rows + R - 1) / R, threads, [&](int64_t group, unsigned grid) {
        part.first = group * R;
        if (a.mx.codes) rms_norm_kernel<T, LANES, CH, true><<<grid, threads, 0, st>>>(part);
        else rms_norm_kernel<T, LANES, CH, false><<<grid, threads, 0, st>>>(part);
      });
    }
    return rc;
  });
}

template <typename T>
int norm_grad(const NormGradArgs& a, hipStream_t st) {
  const int64_t pieces = (a.D + kC<T> - 1) / kC<T>;
  if (pieces > 2048) {
    rms_norm_grad_long_kernel<T><<<(unsigned)a.parts, 1024, 0, st>>>(a);
    return check_launch("rms_norm_backward");
  }
  return by_pieces(pieces, [&](auto lanes, auto ch) {
    constexpr int LANES = decltype(lanes)::value, CH = decltype(ch)::value;
    if constexpr (LANES * CH <= 2048)
      rms_norm_grad_kernel<T, LANES, CH><<<(unsigned)a.parts, LANES > 256 ? LANES : 256, 0, st>>>(a);
    return check_launch("rms_norm_backward");
  });
}

}  // namespace

int run_rms_norm(const NormArgs& a, int dtype, hipStream_t st) {
  if (dtype == MLXQ_BFLOAT16) return norm<uint16_t>(a, st);
  if (dtype == MLXQ_FLOAT16) return norm<_Float16>(a, st);
  return norm<float>(a, st);
}

// Workgroups of the gradient: four to a CU of the MI355X's 256 where a row is a wave's or less, two where it is 256 lanes', one
// above; fewer where there are no rows for them.  By sizes alone, so that sums are the same everywhere.
int64_t norm_grad_parts(int64_t rows, int64_t D, int dtype) {
  const int64_t C = dtype == MLXQ_FLOAT32 ? 4 : 8, pieces = (D + C - 1) / C;
  const int64_t lanes = pieces <= 8 ? 8 : pieces <= 16 ? 16 : pieces <= 32 ? 32 : pieces <= 128 ? 64 : 256;
  const int64_t groups = (rows + 256 / lanes - 1) / (256 / lanes);
  return std::min<int64_t>(groups, pieces <= 128 ? 1024 : pieces <= 1024 ? 512 : 256);
}

int run_rms_norm_backward(const NormGradArgs& a, int dtype, hipStream_t st) {
  int rc = MLXQ_OK;
  if (a.parts == 0) {}  // no rows: the weight's gradient is 0
  else if (dtype == MLXQ_BFLOAT16) rc = norm_grad<uint16_t>(a, st);
  else if (dtype == MLXQ_FLOAT16) rc = norm_grad<_Float16>(a, st);
  else rc = norm_grad<float>(a, st);
  if (rc != MLXQ_OK || a.w_dtype < 0) return rc;
  const unsigned grid = (unsigned)((a.D + 63) / 64);
  if (a.w_dtype == MLXQ_BFLOAT16) rms_norm_weight_kernel<<<grid, 1024, 0, st>>>(a.part, (uint16_t*)a.dw, a.D, a.parts);
  else if (a.w_dtype == MLXQ_FLOAT16) rms_norm_weight_kernel<<<grid, 1024, 0, st>>>(a.part, (_Float16*)a.dw, a.D, a.parts);
  else rms_norm_weight_kernel<<<grid, 1024, 0, st>>>(a.part, (float*)a.dw, a.D, a.parts);
  return check_launch("rms_norm_backward");
}

}  // namespace mlxq
