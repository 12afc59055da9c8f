// attention_tile.h — paged attention for many rows a key head (chunks of prompts) in 16-bit types.
//
// A workgroup holds 4 waves of 32 * RW rows, (token, query head) pairs of one sequence and key head, and
// walks the sequence's keys in tiles of KT.  Keys and values go from the pages to LDS by DMA, one tile
// ahead: a block of 16 keys is contiguous in a page, so a copy is linear and a wave moves whole blocks.
// As in the streaming kernel the products are S^T = K Q^T and O^T = V^T P^T, here with 32x32x16: a lane
// holds one row's scores, the maximum needs one exchange between the halves of a wave, and the exponentials
// are the second product's B operand without moving.  With lane = 32 h + c, D rows are 8 (r / 4) + 4 h +
// r % 4 and the B operand wants keys 8 h + e: row 8 a + 4 h + i of a block's 16 is therefore key
// 8 h + 4 a + i, and register 8 j + e of a score tile is key 16 j + 8 h + e.
//
// Bound by the matrix cores and, nearly as much, by the exponentials (a quarter-rate instruction each).
#pragma once

#include "attention_stream.h"

namespace mlxq {

template <typename T>
__device__ __forceinline__ f32x16 mma32(const u32x4& a, const u32x4& b, f32x16 acc) {
  if constexpr (__is_same(T, _Float16))
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), acc, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), acc, 0, 0, 0);
}

// 16 bytes a lane from memory to LDS: lane i's land at lds + 16 i.  As inline asm without a result, so that the
// compiler adds no wait of its own before later LDS reads; callers wait for vmcnt themselves.  M0 holds the
// LDS address and is restored.  COUNT loads of 1 KB follow each other on both sides.
template <int COUNT>
__device__ __forceinline__ void dma_to_lds(const void* base, uint32_t voffset, uint32_t lds) {
  static_assert(COUNT >= 1 && COUNT <= 4, "offsets reach 4095 bytes");
  const uint64_t b = (uint64_t)(uintptr_t)base;
  uint32_t saved;
#define MLXQ_DMA(LOADS)                                                                       \
  asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\t" LOADS "s_mov_b32 m0, %0\n\ts_nop 0" \
               : "=&s"(saved)                                                                 \
               : "s"(lds), "v"(voffset), "s"(b)                                               \
               : "memory")
  if constexpr (COUNT == 1) MLXQ_DMA("global_load_lds_dwordx4 %2, %3\n\t");
  if constexpr (COUNT == 2) MLXQ_DMA("global_load_lds_dwordx4 %2, %3\n\tglobal_load_lds_dwordx4 %2, %3 offset:1024\n\t");
  if constexpr (COUNT == 3)
    MLXQ_DMA("global_load_lds_dwordx4 %2, %3\n\tglobal_load_lds_dwordx4 %2, %3 offset:1024\n\t"
             "global_load_lds_dwordx4 %2, %3 offset:2048\n\t");
  if constexpr (COUNT == 4)
    MLXQ_DMA("global_load_lds_dwordx4 %2, %3\n\tglobal_load_lds_dwordx4 %2, %3 offset:1024\n\t"
             "global_load_lds_dwordx4 %2, %3 offset:2048\n\tglobal_load_lds_dwordx4 %2, %3 offset:3072\n\t");
#undef MLXQ_DMA
}

__device__ __forceinline__ float half_max(float v) {
  const uint32_t u = __float_as_uint(v);
  auto b = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float half_sum(float v) {
  const uint32_t u = __float_as_uint(v);
  auto b = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// Tells the scheduler to keep READ_AHEAD LDS reads in flight before the matrix products that use them, one more read
// for each read used.  By itself it reads into one register quad and waits for each where registers are short.
#ifndef READ_AHEAD
#define READ_AHEAD 4
#endif
template <int READS, int PER>
__device__ __forceinline__ void reads_ahead() {
  constexpr int kMfma = 0x008, kDsRead = 0x100, AHEAD = READ_AHEAD < READS ? READ_AHEAD : READS;
  __builtin_amdgcn_sched_group_barrier(kDsRead, AHEAD, 0);
#pragma unroll
  for (int i = 0; i < READS - AHEAD; ++i) {
    __builtin_amdgcn_sched_group_barrier(kMfma, PER, 0);
    __builtin_amdgcn_sched_group_barrier(kDsRead, 1, 0);
  }
  __builtin_amdgcn_sched_group_barrier(kMfma, AHEAD * PER, 0);
}

template <bool B>
struct BoolConstant {
  static constexpr bool value = B;
};

template <typename T, int DT, int RW, int BEND>
__global__ __launch_bounds__(256, RW == 1 ? 2 : 1) void attn_tile_kernel(AttnArgs a) {
  constexpr int C = 8, KT = DT <= 128 ? 64 : 32, NB = KT / 16, NK = KT / 32, NS = DT / 16, ND = DT / 32, TM = 128 * RW;
  constexpr int BLOCK = 16 * DT * 2;   // bytes of a block's keys (or values) in LDS, at most
  constexpr int BUF = 2 * NB * BLOCK;  // a tile: the blocks' keys, then their values
  __shared__ __align__(1024) unsigned char lds[2 * BUF];  // the only LDS, from its start: M0 addresses 64 KB
  static_assert(sizeof(lds) <= 65536, "M0");
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int half = lane >> 5, c = lane & 31, unit = a.by_hkv.div(blockIdx.x), h = blockIdx.x - unit * a.Hkv, z = blockIdx.y;
  const Batch& bt = a.batch;
  int b, at;
  if (!Finder(bt, [&](const Seq& s) { return (s.n * a.G + TM - 1) / TM; }).find(unit, b, at)) return;
  const Seq s = load_seq(bt, b);
  const int rows = s.n * a.G, prefix = a.prefix ? a.prefix[b] : 0;
  const int row0 = ((rows + TM - 1) / TM - 1 - at) * TM;  // the longest first
  const int row1 = min(rows, row0 + TM) - 1;
  const KeyRange kr = key_range(a, s, row0, row1, prefix);
  const int tb = kr.lo / KT, te = kr.hi > kr.lo ? (kr.hi + KT - 1) / KT : tb;
  const int ct = (1 << a.chunk_log2) / KT, ns = max(1, min(a.S, (te - tb + ct - 1) >> (a.chunk_log2 - (KT == 64 ? 6 : 5))));
  if (z >= ns) return;
  const int t0 = tb + z * ct, t1 = z == a.S - 1 ? te : min(te, t0 + ct);
  const int blo = kr.lo >> 4, bhi = (kr.hi - 1) >> 4;  // blocks with keys that are seen
  const int32_t* table = bt.tables + b * bt.table_stride;
  const int blog = bt.page_log2 - 4, bmask = (1 << blog) - 1, D = a.D;

  // One tile's DMA.  Item i of a tile: the keys of block i, or from NB on the values; wave w moves items w, w + 4,
  // ...  Blocks that no row sees are never looked up: their entries may name nothing.
  constexpr int ITEMS = 2 * NB / 4, RUN = ND < 4 ? ND : 4;
  static_assert(ND % RUN == 0, "a block is whole runs");
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)lds;
  const int64_t head = ((int64_t)h << bt.page_log2) * D;
  int pg[ITEMS];
  bool bad = false;
  auto pages = [&](int t) {
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) pg[i] = table[min(max(t * NB + (w + 4 * i) % NB, blo), bhi) >> blog];
  };
  auto dma = [&](int t) {
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int item = w + 4 * i, blk = min(max(t * NB + item % NB, blo), bhi);
      const bool in = (unsigned)pg[i] < (unsigned)bt.pages;
      bad |= !in;
      const T* src = (item < NB ? (const T*)a.k : (const T*)a.v) + head + (int64_t)(blk & bmask) * 16 * D +
                     (int64_t)(in ? pg[i] : 0) * (item < NB ? a.k_page : a.v_page);
      const uint32_t dst = lds0 + (t & 1) * BUF + item * BLOCK;
      if (D == DT) {
#pragma unroll
        for (int k = 0; k < ND; k += RUN) dma_to_lds<RUN>((const unsigned char*)src + k * 1024, lane * 16, dst + k * 1024);
      } else {
        for (int k = 0; k * 64 < 2 * D; ++k)
          if (k * 64 + lane < 2 * D) dma_to_lds<1>((const unsigned char*)src + k * 1024, lane * 16, dst + k * 1024);
      }
    }
  };
  if (D < DT) {
    // The features from D to DT of the keys, which no DMA writes: zeros, as the queries' are.
    for (int i = tid; i < 2 * BUF / 16; i += 256) reinterpret_cast<u32x4*>(lds)[i] = u32x4{0, 0, 0, 0};
    __syncthreads();
  }
  if (t0 < t1) {
    pages(t0);
    dma(t0);
    pages(min(t0 + 1, t1 - 1));
  }

  // Rows of this wave, their queries, and what the wave's rows see.
  const int wr0 = row0 + w * 32 * RW, wr1 = min(row1, wr0 + 32 * RW - 1);
  const KeyRange wk = wr0 > row1 ? KeyRange{0, 0, 0, 0} : key_range(a, s, wr0, wr1, prefix);
  int place[RW], lo[RW], span[RW];
  float slope[RW];
  u32x4 qf[RW][NS];
#pragma unroll
  for (int m = 0; m < RW; ++m) {
    const int r = min(wr0 + m * 32 + c, row1), i = a.by_g.div(r), qh = h * a.G + (r - i * a.G);
    const int p = s.L - s.n + i;
    const RowRange rr = row_range(a, s, p, prefix);
    place[m] = p;
    lo[m] = rr.lo;
    span[m] = max(rr.hi - rr.lo, 0);
    slope[m] = BEND == kBias ? a.slopes[qh] * kLog2e : 0.0f;
    const T* q = (const T*)a.q.p + (s.q0 + i) * a.q.ts + qh * a.q.hs;
#pragma unroll
    for (int k = 0; k < NS; ++k) qf[m][k] = 16 * k < D ? load_chunk(q + (2 * k + half) * C) : u32x4{0, 0, 0, 0};
  }
  // The queries have to be there before the loop: a wait for them inside it would be one for the next tile's DMA too.
#pragma unroll
  for (int m = 0; m < RW; ++m)
#pragma unroll
    for (int k = 0; k < NS; ++k) asm volatile("" : "+v"(qf[m][k]));
  f32x16 o[RW][ND];
  float ref[RW], sum[RW];
#pragma unroll
  for (int m = 0; m < RW; ++m) {
    ref[m] = -INFINITY;
    sum[m] = 0.0f;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[m][d][i] = 0.0f;
  }
  const float cs = BEND != kPlain ? 1.0f : a.scale;

  // One tile against this wave's rows.  PART: some row does not see some key of it.
  auto step = [&](int t, auto PARTIAL) {
    constexpr bool PART = decltype(PARTIAL)::value;
    const unsigned char* kl = lds + (t & 1) * BUF;
    const unsigned char* vl = kl + NB * BLOCK;
    f32x16 st[RW][NK];
#pragma unroll
    for (int m = 0; m < RW; ++m)
#pragma unroll
      for (int k = 0; k < NK; ++k)
#pragma unroll
        for (int i = 0; i < 16; ++i) st[m][k][i] = 0.0f;
    {
      // Row c of a score tile is key 8 (c / 4 % 2) + 4 (c / 8 % 2) + c % 4 of block c / 16.
      const int key = (c & 3) | (c & 4) << 1 | (c & 8) >> 1;
      const unsigned char* base = kl + (c >> 4) * BLOCK + half * 256 + key * 16;
#pragma unroll
      for (int ss = 0; ss < NS; ++ss)
#pragma unroll
        for (int k = 0; k < NK; ++k) {
          const u32x4 kf = *reinterpret_cast<const u32x4*>(base + k * 2 * BLOCK + ss * 512);
#pragma unroll
          for (int m = 0; m < RW; ++m) st[m][k] = mma32<T>(kf, qf[m][ss], st[m][k]);
        }
      reads_ahead<NS * NK, RW>();
    }
    if constexpr (BEND != kPlain || PART) {
#pragma unroll
      for (int m = 0; m < RW; ++m) {
        const float away = (float)(t * KT + 8 * half - place[m]);
#pragma unroll
        for (int k = 0; k < NK; ++k)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int i = 32 * k + 16 * (r >> 3) + (r & 7), j = t * KT + 8 * half + i;
            float v = st[m][k][r];
            if constexpr (BEND != kPlain) v = bent_score<T, BEND>(a, v, slope[m], away + (float)i);
            if constexpr (PART) v = (unsigned)(j - lo[m]) < (unsigned)span[m] ? v : -INFINITY;
            st[m][k][r] = v;
          }
      }
    }
    u32x4 pf[RW][NB];
#pragma unroll
    for (int m = 0; m < RW; ++m) {
      float v = st[m][0][0];
#pragma unroll
      for (int k = 0; k < NK; ++k)
#pragma unroll
        for (int r = 0; r < 16; ++r) v = fmaxf(v, st[m][k][r]);
      v = half_max(v) * cs;
      const bool up = v > ref[m] + kSlack;
      if (__any(up)) {
        const float now = up ? v : ref[m];
        const float alpha = up ? __builtin_amdgcn_exp2f(ref[m] - now) : 1.0f;
        ref[m] = now;
        sum[m] *= alpha;
#pragma unroll
        for (int d = 0; d < ND; ++d) o[m][d] *= alpha;
      }
      const float neg = ref[m] == -INFINITY ? 0.0f : -ref[m];  // nothing seen yet: all weights are exp2(-inf)
      float add = 0.0f;
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        float e[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          e[i] = __builtin_amdgcn_exp2f(fmaf(st[m][j / 2][8 * (j % 2) + i], cs, neg));
          add += e[i];
        }
        // The weights are rounded to the type for the product with the values, as the values are.
        pf[m][j] = pack_chunk<T>(e);
      }
      sum[m] += add;
    }
    auto value = [&](int j, int d) { return *reinterpret_cast<const u32x4*>(vl + j * BLOCK + (half * D + 32 * d + c) * 16); };
    if constexpr (!PART) {
#pragma unroll
      for (int j = 0; j < NB; ++j)
#pragma unroll
        for (int d = 0; d < ND; ++d) {
          const u32x4 vf = value(j, d);
#pragma unroll
          for (int m = 0; m < RW; ++m) o[m][d] = mma32<T>(vf, pf[m][j], o[m][d]);
        }
      reads_ahead<NB * ND, RW>();
    } else {
      // Values of keys that no row of the workgroup sees are cleared; of the others, those that are not finite are
      // left to the second product.
      auto seen_of = [&](int j) {
        const int j0 = t * KT + 16 * j + 8 * half - kr.lo;
        u32x4 seen;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          seen[i] = ((unsigned)(j0 + 2 * i) < (unsigned)(kr.hi - kr.lo) ? 0xffffu : 0u) |
                    ((unsigned)(j0 + 2 * i + 1) < (unsigned)(kr.hi - kr.lo) ? 0xffff0000u : 0u);
        return seen;
      };
      uint32_t nf = 0;
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        const u32x4 seen = seen_of(j);
#pragma unroll
        for (int d = 0; d < ND; ++d) {
          u32x4 vf = value(j, d) & seen;
          const u32x4 fin = each<T>(vf, finite_mask<T>);
          nf |= 32 * d + c < D ? ~(fin[0] & fin[1] & fin[2] & fin[3]) : 0u;
          vf &= fin;
#pragma unroll
          for (int m = 0; m < RW; ++m) o[m][d] = mma32<T>(vf, pf[m][j], o[m][d]);
        }
      }
      if (__any(nf != 0)) {
#pragma unroll 1
        for (int j = 0; j < NB; ++j) {
          const u32x4 seen = seen_of(j);
#pragma unroll
          for (int m = 0; m < RW; ++m) {
            u32x4 ch = pf[m][0];
#pragma unroll
            for (int i = 1; i < NB; ++i) ch = j == i ? pf[m][i] : ch;
            ch = each<T>(ch, weight_code<T>);
#pragma unroll
            for (int d = 0; d < ND; ++d) {
              f32x16 x;
#pragma unroll
              for (int i = 0; i < 16; ++i) x[i] = 0.0f;
              x = mma32<T>(each<T>(value(j, d) & seen, value_code<T>), ch, x);
#pragma unroll
              for (int i = 0; i < 16; ++i) o[m][d][i] += decoded(x[i]);
            }
          }
        }
      }
    }
  };

  // Tiles [ta, tb) are seen whole by every row; those before (a window's start) and after (the diagonal) are not.
  // One loop each, run twice, so that the long one has no branch but the rescaling.
  int ta = min(max((kr.lo_all + KT - 1) / KT, t0), t1);
  const int tz = max(min(kr.hi_all / KT, t1), ta);
  auto arrive = [&](int t) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (t + 1 < t1) {
      dma(t + 1);
      pages(min(t + 2, t1 - 1));
    }
  };
#pragma unroll 1
  for (int t = t0; t < t1;) {
#pragma unroll 1
    for (; t < ta; ++t) {
      arrive(t);
      if (t * KT < wk.hi && (t + 1) * KT > wk.lo) step(t, BoolConstant<true>{});
    }
    ta = t1;
#pragma unroll 1
    for (; t < tz; ++t) {
      arrive(t);
      if (wr0 <= row1) step(t, BoolConstant<false>{});
    }
  }

  __syncthreads();
  if (any_wave<4>(bad, reinterpret_cast<int*>(lds))) poison(bt, table, max(t0 * KT, kr.lo), min(t1 * KT, kr.hi), lo, span, sum);
#pragma unroll
  for (int m = 0; m < RW; ++m) {
    const int r = wr0 + m * 32 + c;
    float l = half_sum(sum[m]);
    if (r > row1) continue;
    const int tok = a.by_g.div(r), qh = h * a.G + (r - tok * a.G);
    const int64_t orow = (int64_t)(s.q0 + tok) * a.Hkv * a.G + qh;
    if (ns > 1) {
      float* y = a.part + (orow * a.S + z) * D;
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int f = 32 * d + 8 * i + 4 * half;
          if (f < D) *reinterpret_cast<f32x4*>(y + f) = f32x4{o[m][d][4 * i], o[m][d][4 * i + 1], o[m][d][4 * i + 2], o[m][d][4 * i + 3]};
        }
      if (half == 0) {
        *reinterpret_cast<f32x2*>(a.ml + (orow * a.S + z) * 2) = f32x2{ref[m], l};
        if (z == 0) a.splits[orow] = ns;
      }
    } else {
      if (a.S > 1 && half == 0) a.splits[orow] = 1;
      if (a.sinks) l += __builtin_amdgcn_exp2f(a.sinks[qh] * kLog2e - (ref[m] == -INFINITY ? 0.0f : ref[m]));
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
      T* y = (T*)a.out.p + (s.q0 + tok) * a.out.ts + qh * a.out.hs;
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int f = 32 * d + 8 * i + 4 * half;
          if (f < D)
            *reinterpret_cast<u32x2*>(y + f) = u32x2{Elem<T>::pack2(o[m][d][4 * i] * inv, o[m][d][4 * i + 1] * inv),
                                                     Elem<T>::pack2(o[m][d][4 * i + 2] * inv, o[m][d][4 * i + 3] * inv)};
        }
    }
  }
}

template <typename T, int DT, int RW>
static int launch_tile(const AttnArgs& a, const AttnPlan& plan, hipStream_t st) {
  const dim3 grid((unsigned)plan.blocks, (unsigned)a.S);
  if (a.slopes) hipLaunchKernelGGL((attn_tile_kernel<T, DT, RW, kBias>), grid, dim3(256), 0, st, a);
  else if (a.softcap > 0.0f) hipLaunchKernelGGL((attn_tile_kernel<T, DT, RW, kCap>), grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((attn_tile_kernel<T, DT, RW, kPlain>), grid, dim3(256), 0, st, a);
  return check_launch("paged_attention");
}

template <typename T>
static int tile_of(const AttnArgs& a, const AttnPlan& plan, hipStream_t st) {
  if (a.D <= 64) return launch_tile<T, 64, 1>(a, plan, st);
  if (a.D <= 96) return launch_tile<T, 96, 1>(a, plan, st);
  if (a.D <= 128) return launch_tile<T, 128, 1>(a, plan, st);
  return launch_tile<T, 256, 1>(a, plan, st);
}

}  // namespace mlxq
