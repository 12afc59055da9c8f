// rotary.hip — rotary positions, and the write of a step's keys and values into the paged cache.
//
// Pair (a, b) of a head turned by the angle of its token's position: (a c - b s, b c + a s), with
// (c, s) read from a table [position, pair] of f32 (mlxq_rotary_table).  Both kernels move every
// value once in 16-byte pieces and are bound by HBM; the table's rows (4 rotary_dim bytes a token, shared
// by all heads of the token) come from L2.  A thread keeps the (c, s) of its pairs in registers over
// several heads.  Products and sums are f32, rounded once to the dtype.
//
// Rotation of 8190 tokens, 40 f32 heads of 128: 71 us, 4.7 TB/s, the rate of a large copy.  4 tokens of 24 heads: 2.5 us.
#include <algorithm>

#include "paged.h"

namespace mlxq {

// What a unit of a token's head is: a pair of chunks (half layout), a chunk (interleaved), a chunk
// past the rotated features, or, where rotary_dim does not divide into chunks, a single pair or
// feature.
enum RotMode : int { kHalf = 0, kInter = 1, kScalar = 2 };

template <int C>
__host__ __device__ inline int rot_mode(int R, int interleaved) {
  if (R == 0) return kInter;
  return interleaved ? (R % C == 0 ? kInter : kScalar) : (R / 2 % C == 0 ? kHalf : kScalar);
}
template <int C>
__host__ __device__ inline int rot_units(int mode, int R, int D) {
  return mode == kHalf ? R / 2 / C + (D - R) / C : mode == kInter ? D / C : R / 2 + (D - R);
}

// A unit's pairs: their (c, s), NaN for a position outside the table.
template <typename T, int MODE>
struct Turn {
  static constexpr int C = Elem<T>::C;
  static constexpr int N = MODE == kHalf ? C : MODE == kInter ? C / 2 : 1;
  float c[N], s[N];
  bool turned;  // else the unit is copied
  int lo, hi;   // element offsets within the head; hi: the partner's (half layout and single pairs)

  __device__ __forceinline__ void load(const RotaryArgs& r, int pos, int unit) {
    int first;
    if constexpr (MODE == kHalf) {
      const int h = r.R / 2 / C;
      turned = unit < h;
      first = unit * C;
      lo = turned ? first : r.R + (unit - h) * C;
      hi = lo + r.R / 2;
    } else if constexpr (MODE == kInter) {
      lo = unit * C;
      turned = lo < r.R;
      first = lo / 2;
      hi = lo;
    } else {
      turned = unit < r.R / 2;
      first = unit;
      lo = !turned ? r.R / 2 + unit : r.interleaved ? 2 * unit : unit;
      hi = r.interleaved ? lo + 1 : lo + r.R / 2;
    }
    if (!turned) return;
    const bool in = (unsigned)pos < (unsigned)r.rows;
    const f32x2* t = reinterpret_cast<const f32x2*>(r.table) + (int64_t)(in ? pos : 0) * (r.R / 2) + first;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const f32x2 cs = t[i];
      c[i] = in ? cs[0] : __builtin_nanf("");
      s[i] = in ? (r.inverse ? -cs[1] : cs[1]) : __builtin_nanf("");
    }
  }

  // y and x: the head's first element.  kcache != null: the result goes to K's blocks instead, where
  // chunk i of a token lies 16 * C * i elements from the token's first.
  __device__ __forceinline__ void apply(const T* x, T* y, bool blocked) const {
    if constexpr (MODE == kScalar) {
      auto at = [&](int e) { return blocked ? e / C * 16 * C + e % C : e; };
      if (!turned) {
        y[at(lo)] = x[lo];
        return;
      }
      const float a = Act<T>::ld(x, lo), b = Act<T>::ld(x, hi);
      Act<T>::st(y, at(lo), a * c[0] - b * s[0]);
      Act<T>::st(y, at(hi), b * c[0] + a * s[0]);
    } else {
      auto at = [&](int e) { return blocked ? e * 16 : e; };  // e is a multiple of C
      const u32x4 u = load_chunk(x + lo);
      if (!turned) {
        store_chunk(y + at(lo), u);
        return;
      }
      float a[C];
      if constexpr (MODE == kHalf) {
        const u32x4 w = load_chunk(x + hi);
        float b[C];
#pragma unroll
        for (int i = 0; i < C; ++i) {
          const float p = Elem<T>::get(u, i), q = Elem<T>::get(w, i);
          a[i] = p * c[i] - q * s[i];
          b[i] = q * c[i] + p * s[i];
        }
        store_chunk(y + at(hi), pack_chunk<T>(b));
      } else {
#pragma unroll
        for (int i = 0; i < C / 2; ++i) {
          const float p = Elem<T>::get(u, 2 * i), q = Elem<T>::get(u, 2 * i + 1);
          a[2 * i] = p * c[i] - q * s[i];
          a[2 * i + 1] = q * c[i] + p * s[i];
        }
      }
      store_chunk(y + at(lo), pack_chunk<T>(a));
    }
  }
};

// Thread: one unit of one token in up to HPT consecutive heads.
template <typename T, int MODE>
__global__ __launch_bounds__(256) void rotary_kernel(Heads x, Heads y, RotaryArgs r, int64_t total, int units, int groups,
                                                     int hpt, int H) {
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (id >= total) return;
  const int64_t rest = id / units;
  const int unit = (int)(id - rest * units);
  const int64_t t = rest / groups;
  const int h0 = (int)(rest - t * groups) * hpt, h1 = min(h0 + hpt, H);
  Turn<T, MODE> turn;
  turn.load(r, r.table ? r.positions[t] : 0, unit);
  const T* xp = (const T*)x.p + t * x.ts;
  T* yp = (T*)y.p + t * y.ts;
  for (int h = h0; h < h1; ++h) turn.apply(xp + h * x.hs, yp + h * y.hs, false);
}

template <typename T, int MODE>
static int launch_rotary(const Heads& x, int64_t T_, int64_t H, int64_t D, const RotaryArgs& r, const Heads& y,
                         hipStream_t st) {
  const int units = rot_units<Elem<T>::C>(MODE, r.R, (int)D);
  // As many heads a thread as leave the chip 512 threads a CU, at most 8: the (c, s) of a unit are then
  // read once for them.
  const int64_t one = T_ * units * H;
  const int hpt = (int)std::min<int64_t>(std::max<int64_t>(one / (device_cu_count() * 512), 1), 8);
  const int groups = (int)((H + hpt - 1) / hpt);
  const int64_t total = T_ * units * groups, blocks = (total + 255) / 256;
  if (blocks > 0x7fffffff) return set_error(MLXQ_EINVAL, "rotary: problem too large");
  hipLaunchKernelGGL((rotary_kernel<T, MODE>), dim3((unsigned)blocks), dim3(256), 0, st, x, y, r, total, units, groups, hpt,
                     (int)H);
  return check_launch("rotary");
}

template <typename T>
static int rotary_of(const Heads& x, int64_t T_, int64_t H, int64_t D, const RotaryArgs& r, const Heads& y, hipStream_t st) {
  switch (rot_mode<Elem<T>::C>(r.R, r.interleaved)) {
    case kHalf: return launch_rotary<T, kHalf>(x, T_, H, D, r, y, st);
    case kInter: return launch_rotary<T, kInter>(x, T_, H, D, r, y, st);
    default: return launch_rotary<T, kScalar>(x, T_, H, D, r, y, st);
  }
}

int run_rotary(const Heads& x, int dtype, int64_t T, int64_t H, int64_t D, const RotaryArgs& r, const Heads& y,
               hipStream_t st) {
  if (dtype == MLXQ_BFLOAT16) return rotary_of<uint16_t>(x, T, H, D, r, y, st);
  if (dtype == MLXQ_FLOAT16) return rotary_of<_Float16>(x, T, H, D, r, y, st);
  return rotary_of<float>(x, T, H, D, r, y, st);
}

struct Frequencies {
  double f[128];
};

// A thread a pair, in double precision: an angle of 2^20 radians is right to 2^-33, where f32 would be off by
// 2^-4.  Bound by double arithmetic and the sincos of large arguments; made once for a model (131072 positions of 64 pairs,
// 67 MB: 31 us).
__global__ __launch_bounds__(256) void rotary_table_kernel(Frequencies fr, int half, double magnitude, int64_t total,
                                                           f32x2* __restrict__ table) {
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (id >= total) return;
  const int64_t pos = id / half;
  double s, c;
  sincos((double)pos * fr.f[id - pos * half], &s, &c);
  table[id] = f32x2{(float)(magnitude * c), (float)(magnitude * s)};
}

int run_rotary_table(const double* inv_freq, int64_t half, double magnitude, int64_t positions, float* table,
                     hipStream_t st) {
  Frequencies fr = {};
  for (int64_t i = 0; i < half; ++i) fr.f[i] = inv_freq[i];
  const int64_t total = positions * half, blocks = (total + 255) / 256;
  if (blocks > 0x7fffffff) return set_error(MLXQ_EINVAL, "rotary_table: %lld positions are too many", (long long)positions);
  hipLaunchKernelGGL(rotary_table_kernel, dim3((unsigned)blocks), dim3(256), 0, st, fr, (int)half, magnitude, total,
                     (f32x2*)table);
  return check_launch("rotary_table");
}

// ---- cache_append --------------------------------------------------------------------------------
//
// Workgroup: the new tokens of one sequence that fall into one block of 16 places, for one key head
// and its query heads.  Keys: a token's chunks lie 16 chunks apart in the block, so the 16 tokens'
// stores of a chunk make up 256 contiguous bytes (in L2).  Values: C tokens of a feature lie side by
// side, which the workgroup turns around in LDS, storing whole chunks where all C tokens are new.
//
// One token of 24 sequences, 32 + 8 heads of 128: 5 us, a launch and three dependent reads (the sequence's bounds,
// its page, the tokens).  Five prompts, 47 MB in fp16: 14 us, 3.4 TB/s: the same chain of reads in 1276 workgroups
// that all fit the chip at once, so that nothing hides it.  More heads a thread at once, 14 -> 18 us, or two units
// side by side, 15 us, lose workgroups a CU to registers.
template <typename T, int MODE>
__global__ __launch_bounds__(256) void append_kernel(AppendArgs a) {
  constexpr int C = Elem<T>::C;
  // [16 tokens][D] of the values, rows 4 bytes longer: the reads below go down the columns.
  __shared__ __align__(16) T vt[16 * (256 + 4 / sizeof(T))];
  const int unit = blockIdx.x / a.Hkv, h = blockIdx.x - unit * a.Hkv, tid = threadIdx.x, D = a.D, row = D + 4 / (int)sizeof(T);
  const Batch& bt = a.batch;
  auto blocks_of = [](const Seq& s) { return s.n == 0 ? 0 : ((s.L - 1) >> 4) - ((s.L - s.n) >> 4) + 1; };
  int b = unit, first = 0;
  if (!a.direct && !Finder(bt, blocks_of).find(unit, b, first)) return;
  const Seq s = load_seq(bt, b);
  const int G = a.q.p ? a.Hq / a.Hkv : 0;
  const int units = rot_units<C>(MODE, a.rot.R, D);
  const int last = a.direct ? blocks_of(s) : first + 1;
  for (int at = first; at < last; ++at) {
    // An arithmetic shift: places below 0 (more new tokens than kv_lens) are blocks of their own.
    const int blk = ((s.L - s.n) >> 4) + at;
    const int p0 = max(blk * 16, s.L - s.n), p1 = min(blk * 16 + 16, s.L), nt = p1 - p0;
    const int64_t t0 = s.q0 + (p0 - (s.L - s.n));
    int page = -1;
    if (blk >= 0 && blk < bt.capacity >> 4) page = bt.tables[b * bt.table_stride + (blk >> (bt.page_log2 - 4))];
    const bool write = (unsigned)page < (unsigned)bt.pages;
    const int64_t in_page = ((int64_t)h << bt.page_log2) * D + (int64_t)(blk & ((1 << (bt.page_log2 - 4)) - 1)) * 16 * D;
    T* kb = (T*)a.k_cache + page * a.k_page + in_page;
    T* vb = (T*)a.v_cache + page * a.v_page + in_page;
    // Values into LDS first: their stores come last.
    if (write) {
      const T* vp = (const T*)a.v.p + h * a.v.hs;
      for (int i = tid; i < nt * (D / C); i += 256) {
        const int tok = i / (D / C), c = i - tok * (D / C);
        const u32x4 u = load_chunk(vp + (t0 + tok) * a.v.ts + c * C);
        uint32_t* d = reinterpret_cast<uint32_t*>(vt + (p0 + tok - blk * 16) * row + c * C);
#pragma unroll
        for (int w = 0; w < 4; ++w) d[w] = u[w];
      }
    }
    // Keys and queries: (token, unit) shared by `share` threads, each with its own heads; head 0 is the key's.
    const int tu = nt * units, share = max(1, 256 / max(tu, 1));
    for (int i = tid; i < tu * share; i += 256) {
      const int sh = i / tu, k = i - sh * tu, tok = k / units, un = k - tok * units;
      const int64_t t = t0 + tok;
      Turn<T, MODE> turn;
      turn.load(a.rot, a.rot.positions ? a.rot.positions[t] : p0 + tok, un);
      for (int j = sh; j <= G; j += share) {
        if (j == 0) {
          if (write) turn.apply((const T*)a.k.p + t * a.k.ts + h * a.k.hs, kb + (p0 + tok - blk * 16) * C, true);
        } else {
          const int qh = h * G + j - 1;
          turn.apply((const T*)a.q.p + t * a.q.ts + qh * a.q.hs, (T*)a.q_out.p + t * a.q_out.ts + qh * a.q_out.hs, false);
        }
      }
    }
    __syncthreads();
    if (write) {
      for (int i = tid; i < 16 / C * D; i += 256) {
        const int grp = i / D, d = i - grp * D, lo = blk * 16 + grp * C;
        T* dst = vb + (grp * (int64_t)D + d) * C;
        const T* src = vt + grp * C * row + d;
        if (lo >= p0 && lo + C <= p1) {
          T e[C];
#pragma unroll
          for (int k = 0; k < C; ++k) e[k] = src[k * row];
          u32x4 o;
          __builtin_memcpy(&o, e, 16);
          store_chunk(dst, o);
        } else {
          for (int k = max(p0 - lo, 0); k < min(p1 - lo, C); ++k) dst[k] = src[k * row];
        }
      }
    }
    if (at + 1 < last) __syncthreads();
  }
}

template <typename T>
static int append_of(const AppendArgs& a, int64_t units, hipStream_t st) {
  const dim3 grid((unsigned)(a.Hkv * units));
  switch (rot_mode<Elem<T>::C>(a.rot.R, a.rot.interleaved)) {
    case kHalf: hipLaunchKernelGGL((append_kernel<T, kHalf>), grid, dim3(256), 0, st, a); break;
    case kInter: hipLaunchKernelGGL((append_kernel<T, kInter>), grid, dim3(256), 0, st, a); break;
    default: hipLaunchKernelGGL((append_kernel<T, kScalar>), grid, dim3(256), 0, st, a); break;
  }
  return check_launch("cache_append");
}

int run_cache_append(const AppendArgs& a, int dtype, int64_t units, hipStream_t st) {
  if (dtype == MLXQ_BFLOAT16) return append_of<uint16_t>(a, units, st);
  if (dtype == MLXQ_FLOAT16) return append_of<_Float16>(a, units, st);
  return append_of<float>(a, units, st);
}

}  // namespace mlxq
