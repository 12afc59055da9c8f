// mx_matmul.h — products of microscaled operands: y[m, n] = sum_k x[m, k] w[n, k], dense or of routed experts.
//
// The matrix cores multiply 16 weight rows by 16 rows of x over 128 values of K and apply the blocks' scales
// themselves, so codes go from memory to the operands as they lie: nothing is converted.  The weights are the A operand
// and x the B operand, so that a lane's results are four neighbouring features of one row.  With lane = 16 g + c, a
// lane holds of row c: e2m1 the values 32 g .. 32 g + 31 of the 128; e4m3 16 g .. 16 g + 15 and those 64 further on;
// and the scale of values 32 g .. 32 g + 31 in either.
//
// The 8-bit instruction adds eight neighbouring products at a time and cuts each of them below 2^-13 of the largest one's power of
// two: up to 7 2^-13 of the largest of eight is lost, always towards 0, and so less than 2^-10 of the magnitudes' sum (measured: 256
// and seven values of 2^-13.1 of it lose 8.0e-4 of their sum; ordinary activations, whose neighbours are of one size, 1e-7 to
// 7e-6).  A rounding to bf16 is 2^-9 to 2^-8 of a result, so bf16 results take this instruction.  One to fp16 is 2^-12 to 2^-11,
// less than the loss: f32 and fp16 results of e4m3 take bf16 instructions instead (EXACT): codes times scales are bf16 numbers
// (past bf16's range infinite, below 2^-126 with the bits that its subnormals have), and their sums are as f32's.  8190 rows, K
// 4096, 14336 features then take 900 us for 387, one row of 6144 features 7.4 for 5.9.  Lane group g holds the values 32 g .. 32 g + 31 of
// either operand, eight to each of four instructions.  e2m1 by e2m1 is exact as it is: its products are 2^-2 to 36.
//
// Routed products go by a plan: runs of choices of one expert, cut into tiles.  Every workgroup finds its tile by a
// scan over the runs' lengths; the last run, of choices without an expert, is written as zeros.
#pragma once

#include <math.h>

#include "mx.h"

namespace mlxq {

// Zeros that lanes past the end of K read.
static __device__ const u32x4 mx_zeros = {0, 0, 0, 0};

// A tile of rows: positions [first, first + count) of y's rows (dense) or of the plan; expert e (E: none).
struct MxTile {
  int first, count, e;
  bool found;
};

// Tile `at` of `tiles`, cut TM rows at a time; `total` gives all tiles of all runs.  Starts that are no plan's may make runs that
// overlap, and more tiles than there are integers: sums stop at kMost, which no plan reaches.
struct MxTiles {
  static constexpr int kMost = (1 << 30) - 1;
  const MxProduct& p;
  int TM;
  __device__ __forceinline__ int bound(int i) const {  // the start of run i; the last ends with the choices
    const int M = (int)p.M;
    return i > p.E ? M : min(max(p.starts[i], 0), M);
  }
  __device__ __forceinline__ int tiles_of(int i) const { return (max(bound(i + 1) - bound(i), 0) + TM - 1) / TM; }
  __device__ __forceinline__ int scan(int i, int& own) const {
    const int lane = threadIdx.x & 63;
    own = i <= p.E ? tiles_of(i) : 0;
    int s = own;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int o = __shfl_up(s, d);
      if (lane >= d) s = min(s + o, kMost);
    }
    return s;
  }
  __device__ __forceinline__ int total() const {
    if (p.E == 0) return ((int)p.M + TM - 1) / TM;
    int n = 0, own;
    for (int i0 = 0; i0 <= p.E; i0 += 64) n = min(n + __builtin_amdgcn_readlane(scan(i0 + (threadIdx.x & 63), own), 63), kMost);
    return n;
  }
  __device__ __forceinline__ MxTile find(int at) const {
    const int M = (int)p.M;
    if (p.E == 0) return {at * TM, min(TM, M - at * TM), 0, at * TM < M};
    for (int i0 = 0; i0 <= p.E; i0 += 64) {
      int own;
      const int s = scan(i0 + (threadIdx.x & 63), own), all = __builtin_amdgcn_readlane(s, 63);
      if (at < all) {
        const int l = __builtin_ctzll(__ballot(s > at)), i = i0 + l;
        const int k = at - (__builtin_amdgcn_readlane(s, l) - __builtin_amdgcn_readlane(own, l));
        if (k >= __builtin_amdgcn_readlane(own, l)) return {0, 0, 0, false};
        const int first = bound(i) + k * TM;
        return {first, min(TM, bound(i + 1) - first), i, true};
      }
      at -= all;
    }
    return {0, 0, 0, false};
  }
  // The row of y at a position; -1 where the plan names none.
  __device__ __forceinline__ int row(int position) const {
    if (p.E == 0) return position;
    const int r = p.rows[position];
    return (unsigned)r < (unsigned)p.M ? r : -1;
  }
  __device__ __forceinline__ int64_t x_row(int row) const {
    if (p.E == 0) return row;
    return p.by_choices.div(max(row, 0));
  }
};

// The bias of four neighbouring features of expert e; 0 past the last.
__device__ __forceinline__ f32x4 mx_bias(const MxProduct& p, int e, int n) {
  f32x4 v = {0, 0, 0, 0};
  if (!p.bias || e >= max(p.E, 1)) return v;
  const int64_t at = (int64_t)e * p.N;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t k = at + min(n + i, (int)p.N - 1);
    v[i] = p.bias_dtype == MLXQ_BFLOAT16 ? Act<uint16_t>::ld((const uint16_t*)p.bias, k)
           : p.bias_dtype == MLXQ_FLOAT16 ? Act<_Float16>::ld((const _Float16*)p.bias, k) : ((const float*)p.bias)[k];
  }
  return v;
}
// Four neighbouring features in a type of 16 bits.
__device__ __forceinline__ u32x2 mx_round(const MxProduct& p, const f32x4& v) {
  return p.y_dtype == MLXQ_BFLOAT16 ? u32x2{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])}
                                    : u32x2{Elem<_Float16>::pack2(v[0], v[1]), Elem<_Float16>::pack2(v[2], v[3])};
}
// Four neighbouring features of a row, rounded to y's type.  Rows of any N start at any element.
__device__ __forceinline__ void mx_store(const MxProduct& p, int row, int n, const f32x4& v) {
  const int N = (int)p.N;
  if (n >= N) return;
  const int64_t at = (int64_t)row * N + n;
  const bool four = n + 4 <= N;
  if (p.y_dtype == MLXQ_FLOAT32) {
    float* y = (float*)p.y + at;
    if (four) {
      __builtin_memcpy(y, &v, 16);
    } else {
      for (int i = 0; i < 4; ++i)
        if (n + i < N) y[i] = v[i];
    }
    return;
  }
  const u32x2 h = mx_round(p, v);
  uint16_t* y = (uint16_t*)p.y + at;
  if (four) {
    __builtin_memcpy(y, &h, 8);
  } else {
    for (int i = 0; i < 4; ++i)
      if (n + i < N) y[i] = (uint16_t)(h[i / 2] >> 16 * (i % 2));
  }
}

// Eight neighbouring features of a row, past the caches or not.
__device__ __forceinline__ void mx_store8(const MxProduct& p, int row, int n, const u32x4& v, bool past) {
  typedef u32x4 __attribute__((aligned(2))) any_u32x4;
  const int N = (int)p.N;
  uint16_t* y = (uint16_t*)p.y + (int64_t)row * N + n;
  if (n + 8 <= N) {
    if (past) {
      // between two statements that keep the compiler from making one ordinary store of both
      asm volatile("");
      __builtin_nontemporal_store(v, reinterpret_cast<any_u32x4*>(y));
      asm volatile("");
    } else {
      *reinterpret_cast<any_u32x4*>(y) = v;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (n + i < N) y[i] = (uint16_t)(v[i / 2] >> 16 * (i % 2));
  }
}

// What a lane holds of 16 rows over 128 values of K, ready for the matrix cores.
template <int XF, bool EXACT>
struct MxFrag {
  static constexpr int N = XF == kE4M3 ? 2 : 1;  // 16-byte pieces
  i32x8 v;
  int scale;
  __device__ __forceinline__ void set(const u32x4 (&p)[N], int s) {
    scale = s;
    v = i32x8{(int)p[0][0], (int)p[0][1], (int)p[0][2], (int)p[0][3], 0, 0, 0, 0};
    if constexpr (N == 2)
#pragma unroll
      for (int i = 0; i < 4; ++i) v[4 + i] = (int)p[1][i];
  }
};
typedef __bf16 bf16x2v __attribute__((ext_vector_type(2)));
template <int XF>
struct MxFrag<XF, true> {
  static constexpr int N = XF == kE4M3 ? 2 : 1;
  bf16x8 v[4];
  __device__ __forceinline__ void set(const u32x4 (&p)[N], int s) {
    const float f = mx_scale((uint32_t)s);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      bf16x2v h[4];
      if constexpr (XF == kE4M3) {
        const uint32_t lo = p[i / 2][2 * (i % 2)], hi = p[i / 2][2 * (i % 2) + 1];
        h[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, f, false);
        h[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, f, true);
        h[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, f, false);
        h[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, f, true);
      } else {
        const uint32_t w = p[0][i];
        h[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, f, 0);
        h[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, f, 1);
        h[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, f, 2);
        h[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, f, 3);
      }
      __builtin_memcpy(&v[i], h, 16);
    }
  }
};
template <int XF, bool EXACT>
__device__ __forceinline__ f32x4 mx_mma(const MxFrag<kE2M1, EXACT>& w, const MxFrag<XF, EXACT>& x, f32x4 c) {
  if constexpr (EXACT) {
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w.v[i], x.v[i], c, 0, 0, 0);
    return c;
  } else {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w.v, x.v, c, 4, XF == kE4M3 ? 0 : 4, 0, w.scale, 0, x.scale);
  }
}

// 16 or 4 bytes a lane from memory to LDS, lane i's to lds + 16 i (4 i).  As inline asm without a result, so that the
// compiler adds no wait of its own before later LDS reads; callers wait for vmcnt themselves.  M0 holds the LDS address
// and is restored.
#define MLXQ_DMA(LOAD, FROM, LDS)                                                                                       \
  {                                                                                                                    \
    uint32_t saved;                                                                                                    \
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\t" LOAD " %2, off\n\ts_mov_b32 m0, %0\n\ts_nop 0" \
                 : "=&s"(saved)                                                                                        \
                 : "s"(LDS), "v"(FROM)                                                                                 \
                 : "memory");                                                                                          \
  }
__device__ __forceinline__ void mx_dma16(const unsigned char* from, uint32_t lds) MLXQ_DMA("global_load_lds_dwordx4", from, lds)
__device__ __forceinline__ void mx_dma4(const unsigned char* from, uint32_t lds) MLXQ_DMA("global_load_lds_dword", from, lds)
#undef MLXQ_DMA

// What bounds it: few rows, the weights' bytes (1 row, K 8192, 28672 features: 30 us, 4.1 TB/s); many, the matrix cores and the way to
// them: 8190 rows, K 4096, 14336 features of e4m3 380 us, 2.53 PFLOP/s (e2m1 277 us, 3.5; a large library product of 8-bit operands 2.8
// to 3.2).  The large tile without its matrix instructions takes 265 us, without its loads 346, with both 415 before its results were
// written as whole lines: neither side hides the other in full, at two waves a SIMD.  Matrix cores 52 % busy, L2 hits 90 %.  Loads
// spread between the matrix instructions took 5 % more, leaving out the loads of rows that a short tile lacks 4 % (the waits then
// branch); deeper rings do not fit LDS, smaller tiles read more.
//
// A workgroup of WM x WN waves takes TM rows by TN features; steps of 128 values of K go through a ring of STAGES
// buffers in LDS by DMA, one barrier a step.  The scales of four steps go together, 16 bytes of 16 rows a load: a row's
// scales of one step are 4 bytes of a cache line of their own, and fetched step by step they were half of all requests.
//
// KG groups of WM x WN waves share a tile, a run of K with buffers of its own each, and join their sums in LDS: a few rows
// make few tiles, whose steps are a chain of latencies.
template <int XF, bool EXACT, int TM, int TN, int WM, int WN, int STAGES, int KG>
__global__ __launch_bounds__(64 * WM * WN * KG) void mx_tile_kernel(MxProduct p, int n_tiles) {
  constexpr int NW = WM * WN, XB = XF == kE4M3 ? 128 : 64, XN = XF == kE4M3 ? 2 : 1;
  constexpr int FM = TM / WM / 16, FN = TN / WN / 16;
  // DMA loads of 1 KB a step, and those of a wave: every wave makes as many, some of them twice where there are fewer than waves.
  constexpr int XL = TM * XB / 1024, WL = TN * 64 / 1024, XI = XL > NW ? XL / NW : 1, WI = WL > NW ? WL / NW : 1, PER = XI + WI;
  constexpr int W0 = TM * XB, STAGE = W0 + TN * 64;
  // A group of scales: loads of 16 rows each, in up to four parts of a load a wave.
  constexpr int SP = (TM + TN) / 16, GROUP = (TM + TN) * 16, GROUPS = STAGES == 3 ? 2 : 3, S0 = STAGE * STAGES;
  constexpr int RING = S0 + GROUP * GROUPS;
  static_assert(XL >= 1 && WL >= 1 && (XL % NW == 0 || NW % XL == 0) && (WL % NW == 0 || NW % WL == 0) && RING * KG <= 163840 && (KG == 1 || TM * TN * 4 <= RING) && SP <= 4 * NW, "a step is whole loads of each wave");
  __shared__ __align__(1024) unsigned char all_lds[RING * KG];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kg = KG > 1 ? wave / NW : 0, w = KG > 1 ? wave % NW : wave;
  unsigned char* lds = all_lds + kg * RING;
  const int c = lane & 15, g = lane >> 4;

  // Neighbouring workgroups go to different dies: each die takes a run of tiles of its own, in bands of 4 tiles of
  // rows by all of the features, so that what its workgroups read at a time shares its cache (8192 rows, 14336 features,
  // K 4096: bands of 4, 8 and 16 tiles 416, 422 and 431 us).
  constexpr int BAND = 4;
  MxTiles tiles{p, TM};
  // A launch has workgroups for every tile of a plan.
  const int m_tiles = min(tiles.total(), (int)(gridDim.x / (unsigned)n_tiles)), all = m_tiles * n_tiles, chunk = (all + 7) / 8;
  const int l = (blockIdx.x & 7) * chunk + (blockIdx.x >> 3);
  if ((int)(blockIdx.x >> 3) >= chunk || l >= all) return;
  const int band = l / (BAND * n_tiles), in = l - band * BAND * n_tiles, high = min(BAND, m_tiles - BAND * band);
  const int nt = in / high, mt = BAND * band + in - nt * high;
  const MxTile tile = tiles.find(mt);
  if (!tile.found || (p.skip_none && tile.e == p.E)) return;
  const int n0 = nt * TN, N = (int)p.N, K = (int)p.K;
  const int steps = (K + 127) / 128;
  // This group's steps, k0 of all its first, a multiple of 4; the first group has the most.
  const int most = KG > 1 ? min(steps, ((steps + KG - 1) / KG + 3) & ~3) : steps;
  const int k0 = kg * most, cnt = max(0, min(steps - k0, most));
  // Waves of one SIMD (w and w + 4) hold different rows: where a run's last tile has half its rows or fewer, a wave of
  // each SIMD has none and leaves the matrix cores to the other.
  const int wm = w / WN, wn = w % WN;
  const bool idle = wm * (TM / WM) >= tile.count;

  f32x4 acc[FN][FM];
#pragma unroll
  for (int i = 0; i < FN; ++i)
#pragma unroll
    for (int j = 0; j < FM; ++j) acc[i][j] = f32x4{0, 0, 0, 0};

  if (tile.e < max(p.E, 1)) {
    const unsigned char *xp[XI], *wp[WI], *sp[4];
    int xk[XI], wk;  // the first value of K of a lane's piece
    const int64_t x_pitch = XF == kE4M3 ? K : K / 2, w_pitch = K / 2;
    auto x_row = [&](int r) { return tiles.x_row(tiles.row(tile.first + min(r, tile.count - 1))); };
#pragma unroll
    for (int i = 0; i < XI; ++i) {
      const int j = (w * XI + i) % XL, r = XF == kE4M3 ? 8 * j + (lane >> 3) : 16 * j + (lane >> 2);
      const int piece = XF == kE4M3 ? (lane & 7) ^ (r & 7) : (lane & 3) ^ (r >> 1 & 3);
      xk[i] = piece * (XF == kE4M3 ? 16 : 32);
      xp[i] = p.x.codes + x_row(r) * x_pitch + piece * 16;
    }
    const int64_t w_row0 = (int64_t)tile.e * N;
#pragma unroll
    for (int i = 0; i < WI; ++i) {
      const int r = 16 * ((w * WI + i) % WL) + (lane >> 2), piece = (lane & 3) ^ (r >> 1 & 3);
      wk = piece * 32;
      wp[i] = p.w.codes + (w_row0 + min(n0 + r, N - 1)) * w_pitch + piece * 16;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = 16 * (i * NW + w) + (lane >> 2);
      if (i * NW + w < SP)
        sp[i] = r < TM ? p.x.scales + x_row(r) * p.x.scale_stride : p.w.scales + (w_row0 + min(n0 + r - TM, N - 1)) * p.w.scale_stride;
    }
    const uint32_t base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)lds;
    const unsigned char* zeros = reinterpret_cast<const unsigned char*>(&mx_zeros);
    const bool ragged = K % 128 != 0;
    const int last_dword = (K / 32 - 1) & ~3;  // of a row's scales

    auto load_scales = [&](int group, int part) {
      if (group * 4 >= cnt || part * NW + w >= SP) return;
      mx_dma4(sp[part] + min(k0 * 4 + group * 16 + 4 * (lane & 3), last_dword), base + S0 + (uint32_t)(group % GROUPS) * GROUP + (part * NW + w) * 256);
    };
    auto load = [&](int s) {  // the group's step s
      // The parts of a group of scales are spread over the steps before it so that two are held at a time (STAGES 3).  They
      // come before the step's codes: a wait for these is one for all scales before them.
      if (s == 0) {
#pragma unroll
        for (int i = 0; i < 4; ++i) load_scales(0, i);
      } else if ((s & 3) == 2) {
        load_scales((s >> 2) + 1, 0);
        load_scales((s >> 2) + 1, 1);
      } else if ((s & 3) == 3) {
        load_scales((s >> 2) + 1, 2);
      } else if ((s & 3) == 0) {
        load_scales(s >> 2, 3);
      }
      const uint32_t to = base + (uint32_t)(s % STAGES) * STAGE;
      const int left = ragged && k0 + s == steps - 1 ? K - (k0 + s) * 128 : 128;
#pragma unroll
      for (int i = 0; i < XI; ++i)
        mx_dma16(xk[i] < left ? xp[i] + (int64_t)(k0 + s) * XB : zeros, to + (w * XI + i) % XL * 1024);
#pragma unroll
      for (int i = 0; i < WI; ++i) mx_dma16(wk < left ? wp[i] + (int64_t)(k0 + s) * 64 : zeros, to + W0 + (w * WI + i) % WL * 1024);
    };
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i)
      if (i < cnt) load(i);

    const int xr = wm * (TM / WM) + c, wr = wn * (TN / WN) + c;  // this lane's rows of the first fragments
    // Of an e4m3 row a lane reads pieces g and g + 4 (EXACT: 2 g and 2 g + 1); piece i of row r lies at i ^ (r % 8).
    constexpr int SECOND = EXACT ? 16 : 64;
    const int x_at = XF == kE4M3 ? xr * 128 + (((EXACT ? 2 * g : g) ^ (c & 7)) * 16) : xr * 64 + ((g ^ (c >> 1 & 3)) * 16);
    const int w_at = W0 + wr * 64 + ((g ^ (c >> 1 & 3)) * 16);
    const int xs_at = xr * 16 + g, ws_at = (TM + wr) * 16 + g;

    // One step.  Fragments are read a few at a time, those of a square that grows by one of x and Q of the weights, and
    // multiplied as soon as a square is there: after a barrier all waves read at once, and the matrix cores would wait
    // until the last had everything.
    constexpr int Q = FN / FM;
    static_assert(FN % FM == 0, "squares of fragments");
    auto meet = [&](int s) {  // the group's step s is there for all of its waves
      if (s + STAGES - 2 < cnt) mlxq_vmcnt<(STAGES - 2) * PER>();
      else mlxq_vmcnt<0>();
      if constexpr (NW > 1) __builtin_amdgcn_s_barrier();  // a group of one wave has its buffers to itself
      asm volatile("" ::: "memory");
    };
    auto step = [&](int s, bool ahead, auto LAST) {
      meet(s);
      const unsigned char *b = lds + (s % STAGES) * STAGE, *sb = lds + S0 + ((s >> 2) % GROUPS) * GROUP + (s & 3) * 4;
      const bool past = decltype(LAST)::value && g * 32 >= K - (k0 + s) * 128;  // this lane's block is past K
      MxFrag<XF, EXACT> x[FM];
      MxFrag<kE2M1, EXACT> a[FN];
      auto read = [&](int j) {
        u32x4 v[XN];
        v[0] = *reinterpret_cast<const u32x4*>(b + x_at + j * 16 * XB);
        if constexpr (XN == 2) v[1] = *reinterpret_cast<const u32x4*>(b + (x_at ^ SECOND) + j * 16 * XB);
        const int xs = sb[xs_at + j * 256];
        x[j].set(v, past ? 0 : xs);
#pragma unroll
        for (int i = j * Q; i < (j + 1) * Q; ++i) {
          const u32x4 u[1] = {*reinterpret_cast<const u32x4*>(b + w_at + i * 1024)};
          const int ws = sb[ws_at + i * 256];
          a[i].set(u, past ? 0 : ws);
        }
      };
      read(0);
      if constexpr (FM > 1) read(1);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int j = 0; j < FM; ++j) {
        if (j > 0 && j + 1 < FM) read(j + 1);
        __builtin_amdgcn_sched_barrier(0);
        if (j == 0 && ahead) load(s + STAGES - 1);
#pragma unroll
        for (int i = 0; i < (j + 1) * Q; ++i)
#pragma unroll
          for (int k = 0; k <= j; ++k)
            if (k == j || i >= j * Q) acc[i][k] = mx_mma<XF, EXACT>(a[i], x[k], acc[i][k]);
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    if (idle) {
      for (int s = 0; s < most; ++s) {
        meet(s);
        if (s + STAGES - 1 < cnt) load(s + STAGES - 1);
      }
      if constexpr (KG == 1) return;
    } else {
      for (int s = 0; s + 1 < cnt; ++s) step(s, s + STAGES - 1 < cnt, std::false_type{});
      if (cnt > 0) step(cnt - 1, false, std::true_type{});
      if constexpr (NW > 1)
        for (int s = cnt; s < most; ++s) meet(s);
    }
    if constexpr (KG > 1) {
      __syncthreads();
      f32x4* sums = reinterpret_cast<f32x4*>(lds);
      if (kg > 0 && !idle)
#pragma unroll
        for (int i = 0; i < FN; ++i)
#pragma unroll
          for (int j = 0; j < FM; ++j) sums[(i * FM + j) * 64 * NW + w * 64 + lane] = acc[i][j];
      __syncthreads();
      if (kg > 0) return;
#pragma unroll
      for (int k = 1; k < KG; ++k)
#pragma unroll
        for (int i = 0; i < FN; ++i)
#pragma unroll
          for (int j = 0; j < FM; ++j)
            acc[i][j] += reinterpret_cast<const f32x4*>(all_lds + k * RING)[(i * FM + j) * 64 * NW + w * 64 + lane];
    }
  } else if (KG > 1 && kg > 0) {
    return;
  }
  if (idle) return;
  constexpr int WT = TN / WN;  // a wave's features
  const int n_wave = n0 + wn * WT;
  f32x4 bias[FN];
#pragma unroll
  for (int i = 0; i < FN; ++i) bias[i] = mx_bias(p, tile.e, n_wave + i * 16 + 4 * g);
  // A lane's four features are 8 bytes of a row, and stores of such pieces touch 16 rows each.  The large tiles' results of 16
  // bits are turned around in LDS, 16 rows of the wave at a time, and written as whole lines (8192 rows, 14336 features, K 4096:
  // 415 -> 393 us).  The buffer of the step that is not there any more is free: its last readers have passed the last step's
  // barrier.  Piece i of row r lies at i ^ r.  A result of more than half of the 256 MB that all dies share goes past the
  // caches, where it would take the operands' place (235 MB: 394 -> 379 us); a smaller one is left there for its reader (94 MB of
  // experts' products, then their sum: 215 + 24 us; past the caches 207 + 32).
  if constexpr (KG == 1 && WT >= 64) {
    if (p.y_dtype != MLXQ_FLOAT32) {
      constexpr int PIECES = WT / 8;
      static_assert(NW * 16 * WT * 2 <= STAGE && 16 * PIECES % 64 == 0);
      const bool past = p.M * p.N > (int64_t)64 << 20;
      unsigned char* own = lds + cnt % STAGES * STAGE + w * (16 * WT * 2);
#pragma unroll
      for (int j = 0; j < FM; ++j) {
#pragma unroll
        for (int i = 0; i < FN; ++i)
          *reinterpret_cast<u32x2*>(own + c * WT * 2 + ((2 * i + (g >> 1)) ^ (c % PIECES)) * 16 + (g & 1) * 8) =
              mx_round(p, acc[i][j] + bias[i]);
        asm volatile("" ::: "memory");
#pragma unroll
        for (int t = 0; t < 16 * PIECES / 64; ++t) {
          const int r = t * (64 / PIECES) + lane / PIECES, piece = lane % PIECES;
          const u32x4 v = *reinterpret_cast<const u32x4*>(own + r * WT * 2 + (piece ^ (r % PIECES)) * 16);
          const int at = wm * (TM / WM) + j * 16 + r, row = at < tile.count ? tiles.row(tile.first + at) : -1;
          const int n = n_wave + piece * 8;
          if (row >= 0 && n < N) mx_store8(p, row, n, v, past);
        }
        asm volatile("" ::: "memory");
      }
      return;
    }
  }
#pragma unroll
  for (int j = 0; j < FM; ++j) {
    const int r = wm * (TM / WM) + j * 16 + c, row = r < tile.count ? tiles.row(tile.first + r) : -1;
    if (row < 0) continue;
#pragma unroll
    for (int i = 0; i < FN; ++i) mx_store(p, row, n_wave + i * 16 + 4 * g, acc[i][j] + bias[i]);
  }
}

namespace {

// Tiles of TM rows that a launch is made for: as many as there can be, by sizes alone.
inline int64_t mx_most_tiles(const MxProduct& p, int64_t TM) {
  if (p.E == 0) return (p.M + TM - 1) / TM;
  return p.M / TM + (p.M < p.E + 1 ? p.M : p.E + 1);
}

template <int XF, bool EXACT, int TM, int TN, int WM, int WN, int STAGES, int KG>
int mx_launch_tile(const MxProduct& p, hipStream_t st) {
  const int64_t n_tiles = (p.N + TN - 1) / TN, grid = (mx_most_tiles(p, TM) * n_tiles + 7) / 8 * 8;
  constexpr int threads = 64 * WM * WN * KG;
  if (grid > most_groups(threads))
    return set_error(MLXQ_EUNSUPPORTED, "mx product: %lld tiles of %d threads are too many for one launch", (long long)grid, threads);
  mx_tile_kernel<XF, EXACT, TM, TN, WM, WN, STAGES, KG><<<(unsigned)grid, threads, 0, st>>>(p, (int)n_tiles);
  return check_launch("mx product");
}

// About as many tiles as there will be: every expert's rows, as many as the mean, end in a part of one.
inline double mx_tiles(const MxProduct& p, int64_t TM, int64_t TN) {
  const double n = (double)((p.N + TN - 1) / TN);
  if (p.E == 0) return n * (double)((p.M + TM - 1) / TM);
  const double m = p.E * ((double)p.M / p.E / TM + 0.5), most = (double)mx_most_tiles(p, TM);
  return n * (m < most ? m : most);
}

// The instance for a product, by its rows (of an expert, the mean) and by how many workgroups there are for 256 CUs.  Few: small
// tiles, K split over groups of waves; many: tiles that read less for each product.  Measured in us with e4m3:
//   1 row, K 14336, 4096 features      16 x 16, 16 groups 8.6; 8 groups 9.4; 16 x 32, 8 groups 10.9; 32 x 32, 8 groups 14.3
//   1 row, K 4096, 14336 features      16 x 32, 4 groups 7.4; 16 x 64, 4 groups 7.9; 32 x 64, 4 groups 8.2; 16 x 32, 8 groups 9.3
//   3 tokens, 4 of 32 experts of 5760 x 2880       32 x 128 17.5; 64 x 128 18.1; 32 x 64 18.3; 16 x 32, 4 groups 27
//   32 rows, K 4096, 14336 features    32 x 64, 4 groups 9.1; 2 groups 9.8; 64 x 64, 2 groups 10.8
//   120 / 500 tokens, 4 of 32 experts of 2880 x 2880   64 x 128 44 / 73 (three stages 46 / 74); 128 x 128 53 / 71; 32 x 128 50 / 80; 64 x 64 67 / 112
//   64 / 128 rows, K 4096, 2000 features           16 x 32, 8 groups 6.5 / 9.2; 4 groups 6.8 / 7.5; 32 x 64 8.9 / 9.0; 64 x 64 11.4 / 11.5
//   256 / 512 rows, K 4096, 1000 features          16 x 32, 4 groups 7.5 / 12.1; 32 x 64 9.0 / 9.2; 64 x 64 11.4 / 11.5
//   256 rows, K 4096, 4096 features    64 x 64, 2 groups 11.8; 1 group 15.1; 64 x 128, 2 groups 16.1; 32 x 64 16.7
//   512 rows, K 4096, 4096 features    64 x 128, 2 groups 17.8; 1 group 19.7; 64 x 64 19.9; 128 x 128 28
//   256 rows, K 4096, 14336 features   64 x 128 27.9; 128 x 128 28.8; 64 x 128, 2 groups 32.8
//   2048 rows, K 4096, 4096 / 14336 features       128 x 128 37 / 118; 256 x 256 52 / 105
//   4090 tokens, 4 of 32 experts of 2880 x 2880    256 x 256 173; 128 x 128 183
template <int XF, bool EXACT>
int mx_product(const MxProduct& p, hipStream_t st) {
  const int64_t rows = p.E ? (p.M + p.E - 1) / p.E : p.M;
  const double t = mx_tiles(p, 16, 16);
  if (t <= 256) return mx_launch_tile<XF, EXACT, 16, 16, 1, 1, 3, 16>(p, st);
  if (t <= 512) return mx_launch_tile<XF, EXACT, 16, 32, 1, 1, 4, 8>(p, st);
  if (t <= 1024) return mx_launch_tile<XF, EXACT, 16, 32, 1, 1, 4, 4>(p, st);
  if (rows <= 16) return mx_launch_tile<XF, EXACT, 32, 128, 2, 4, 4, 1>(p, st);
  if (mx_tiles(p, 32, 64) <= 256) return mx_launch_tile<XF, EXACT, 32, 64, 2, 2, 4, 4>(p, st);
  if (mx_tiles(p, 64, 64) <= 256) return mx_launch_tile<XF, EXACT, 64, 64, 2, 2, 4, 2>(p, st);
  if (mx_tiles(p, 64, 128) <= 256) return mx_launch_tile<XF, EXACT, 64, 128, 2, 4, 3, 2>(p, st);
  const double mid = mx_tiles(p, 128, 128);
  if (mid <= 256 || rows <= 64) return mx_launch_tile<XF, EXACT, 64, 128, 2, 4, 4, 1>(p, st);
  // One round of the largest tiles takes a little less than the mid ones' second of 512 (2048 rows, 6000 features: 54 for 56 us);
  // several take as long as three quarters of 1024 of them each (4096 rows, 6000 features: 105 for 99).  Their operands as bf16 do
  // not fit the registers (8190 rows, K 4096, 14336 features in f32: 3.5 ms; the mid ones 0.91).
  const double rounds = ceil(mx_tiles(p, 256, 256) / 256);
  if (!EXACT && mid >= (rounds > 1 ? 768 * rounds : 513)) return mx_launch_tile<XF, false, 256, 256, 4, 2, 3, 1>(p, st);
  return mx_launch_tile<XF, EXACT, 128, 128, 2, 2, 3, 1>(p, st);
}

}  // namespace

}  // namespace mlxq
