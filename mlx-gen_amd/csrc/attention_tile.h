// attention_tile.h — paged attention for many rows a key head (chunks of prompts) in 16-bit types.
//
// A workgroup holds 4 waves of 32 rows, (token, query head) pairs of one sequence and key head, and
// walks the sequence's keys in tiles of 64.  Keys and values go from the pages to LDS by DMA, one to three tiles
// ahead: a block of 16 keys is contiguous in a page, so a copy is linear and a wave moves whole blocks.
// As in the streaming kernel the products are S^T = K Q^T and O^T = V^T P^T, here with 32x32x16: a lane
// holds one row's scores, the maximum needs one exchange between the halves of a wave, and the exponentials
// are the second product's B operand without moving.  With lane = 32 h + c, D rows are 8 (r / 4) + 4 h +
// r % 4 and the B operand wants keys 8 h + e: row 8 a + 4 h + i of a block's 16 is therefore key
// 8 h + 4 a + i, and register 8 j + e of a score tile is key 16 j + 8 h + e.
//
// Bound by the matrix cores and, nearly as much, by the exponentials (a quarter-rate instruction each) and the LDS
// reads, one for every product.  7001 tokens, 32 + 8 bf16 heads of 128: 385-395 us, 1020-1045 TFLOP/s, 90 % of what a
// large bf16 product reaches.  Heads past 128 have one wave a SIMD and wait for their own chain of products and
// exponentials: 500 tokens, 16 + 8 heads of 256 over a window of 4096, capped, in four splits: 64-73 us, 8 of them the join.
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

// N matrix products, each with an LDS read of its own: read(i) gives the operand, use(i, v) multiplies.  kAhead reads are
// in flight, one more for each used.  Left to itself the compiler reads into one register quad and waits for each
// read where registers are short, so neither reads nor products may pass the points between the steps; other
// instructions may.
constexpr int kAhead = 4;
template <int N, typename R, typename U>
__device__ __forceinline__ void read_and_multiply(R read, U use) {
  constexpr int kOthers = 0x002 | 0x004 | 0x010 | 0x400;  // VALU, SALU, memory, transcendentals
  u32x4 v[kAhead];
#pragma unroll
  for (int i = 0; i < kAhead; ++i) v[i] = read(i);
  __builtin_amdgcn_sched_barrier(kOthers);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    use(i, v[i % kAhead]);
    if (i + kAhead < N) v[i % kAhead] = read(i + kAhead);
    __builtin_amdgcn_sched_barrier(kOthers);
  }
}

// The largest sum of weights that a lane takes from a tile: fp16's weights end at 2^16.
constexpr float kMost = 32768.0f;

template <bool B>
struct BoolConstant {
  static constexpr bool value = B;
};

template <typename T, int DT, int BEND>
__global__ __launch_bounds__(256, DT <= 128 ? 2 : 1) void attn_tile_kernel(AttnArgs a) {
  constexpr bool ACC = DT > 128;  // 500 tokens, 16 heads of 256, a window of 4096: 75 us instead of 83
  constexpr int C = 8, KT = 64, NB = KT / 16, NK = KT / 32, NS = DT / 16, ND = DT / 32, TM = 128;
  constexpr int BLOCK = 16 * DT * 2;   // bytes of a block's keys (or values) in LDS, at most
  constexpr int BUF = 2 * NB * BLOCK;  // a tile: the blocks' keys, then their values
  // Tiles in LDS, one in use and the others on their way: as many as leave room for a second workgroup on the CU.  Heads
  // past 128, whose accumulators leave a SIMD one wave, take its LDS too (500 tokens, 16 heads of 256, a window of
  // 4096: 71 us; four tiles of 32 keys instead of two of 64: 75).
  constexpr int BUFS = DT == 64 ? 4 : 2;
  constexpr int PER = 2 * ND;  // DMA loads of a wave a tile
  __shared__ __align__(1024) unsigned char lds[BUFS * BUF];
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
  const int ct = a.chunk / KT, ns = max(1, min(a.S, a.by_chunk.div((te - tb) * KT + a.chunk - 1)));
  if (z >= ns) return;
  const int t0 = tb + z * ct, t1 = z == a.S - 1 ? te : min(te, t0 + ct);
  const int blo = kr.lo >> 4, bhi = (kr.hi - 1) >> 4;  // blocks with keys that are seen
  const int32_t* table = bt.tables + b * bt.table_stride;
  // Looked up by scalar loads: a vector load in the loop would have to be waited for, and with it every DMA before it.
  const auto* pages = (const __attribute__((address_space(4))) int32_t*)(uintptr_t)table;
  const int blog = bt.page_log2 - 4, bmask = (1 << blog) - 1, D = a.D;

  // DMA of a tile's keys and of its values: a wave moves one block of 16 of each.  Blocks that no row sees are never
  // looked up: their entries may name nothing.
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)lds;
  const int64_t head = ((int64_t)h << bt.page_log2) * D;
  bool bad = false;
  auto block_of = [&](int t) { return min(max(t * NB + w, blo), bhi); };
  auto page_of = [&](int t) { return pages[block_of(min(t, t1 - 1)) >> blog]; };
  auto dma = [&](int t, int page, const void* pool, int64_t stride, uint32_t to) {
    const bool in = (unsigned)page < (unsigned)bt.pages;
    bad |= !in;
    const T* src = (const T*)pool + head + (int64_t)(block_of(t) & bmask) * 16 * D + (int64_t)(in ? page : 0) * stride;
    const uint32_t dst = lds0 + (t & (BUFS - 1)) * BUF + to + w * BLOCK;
    constexpr int RUN = ND < 4 ? ND : 4;
    static_assert(ND % RUN == 0, "a block is whole runs");
    if (D == DT) {
#pragma unroll
      for (int k = 0; k < ND; k += RUN) dma_to_lds<RUN>((const unsigned char*)src + k * 1024, lane * 16, dst + k * 1024);
    } else {
      for (int k = 0; k * 64 < 2 * D; ++k)
        if (k * 64 + lane < 2 * D) dma_to_lds<1>((const unsigned char*)src + k * 1024, lane * 16, dst + k * 1024);
    }
  };
  int page = 0;  // of the next tile's block
  auto load = [&](int t) {
    dma(t, page, a.k, a.k_page, 0);
    dma(t, page, a.v, a.v_page, NB * BLOCK);
    page = page_of(t + 1);
  };
  if (D < DT) {
    // The features from D to DT of the keys, which no DMA writes: zeros, as the queries' are.
    for (int i = tid; i < BUFS * BUF / 16; i += 256) reinterpret_cast<u32x4*>(lds)[i] = u32x4{0, 0, 0, 0};
    __syncthreads();
  }
  if (t0 < t1) {
    page = page_of(t0);
#pragma unroll
    for (int i = 0; i < BUFS - 1; ++i)
      if (t0 + i < t1) load(t0 + i);
  }

  // This lane's row, its query, and what the wave's rows see.
  const int wr0 = row0 + w * 32, wr1 = min(row1, wr0 + 31);
  const bool idle = wr0 > row1;
  const KeyRange wk = idle ? KeyRange{0, 0, 0, 0} : key_range(a, s, wr0, wr1, prefix);
  const int r = min(wr0 + c, row1), tok = a.by_g.div(r), qh = h * a.G + (r - tok * a.G), place = s.L - s.n + tok;
  const RowRange rr = row_range(a, s, place, prefix);
  const int lo[1] = {rr.lo}, span[1] = {max(rr.hi - rr.lo, 0)};
  const float slope = slope_of<BEND>(a, qh);
  u32x4 qf[NS];
  const T* q = (const T*)a.q.p + (s.q0 + tok) * a.q.ts + qh * a.q.hs;
#pragma unroll
  for (int k = 0; k < NS; ++k) qf[k] = 16 * k < D ? load_chunk(q + (2 * k + half) * C) : u32x4{0, 0, 0, 0};
  // The queries have to be there before the loop: a wait for them inside it would be one for the next tile's DMA too.
#pragma unroll
  for (int k = 0; k < NS; ++k) {
    if constexpr (ACC) pin<true>(qf[k]);
    else asm volatile("" : "+v"(qf[k]));
  }
  f32x16 o[ND];
  float ref = -INFINITY, sum[1] = {first_sum(a, s, place, prefix)};
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[d][i] = 0.0f;
  const float cs = BEND != kPlain ? 1.0f : a.scale;

  // The scores of tile t.
  auto products = [&](int t, f32x16 (&st)[NK]) {
    // Row c of a score tile is key 8 (c / 4 % 2) + 4 (c / 8 % 2) + c % 4 of block c / 16.
    const int key = (c & 3) | (c & 4) << 1 | (c & 8) >> 1;
    const unsigned char* base = lds + (t & (BUFS - 1)) * BUF + (c >> 4) * BLOCK + half * 256 + key * 16;
#pragma unroll
    for (int k = 0; k < NK; ++k)
#pragma unroll
      for (int i = 0; i < 16; ++i) st[k][i] = 0.0f;
    read_and_multiply<NS * NK>([&](int i) { return *reinterpret_cast<const u32x4*>(base + i % NK * 2 * BLOCK + i / NK * 512); },
                               [&](int i, u32x4 v) { st[i % NK] = mma32<T>(v, qf[i / NK], st[i % NK]); });
  };

  // Tile t.  PART: some row does not see some key of it.
  auto step = [&](int t, auto PARTIAL) {
    f32x16 st[NK];
    constexpr bool PART = decltype(PARTIAL)::value;
    const unsigned char* vl = lds + (t & (BUFS - 1)) * BUF + NB * BLOCK;
    if (PART && (t * KT >= wk.hi || (t + 1) * KT <= wk.lo)) return;
    products(t, st);
    if constexpr (BEND != kPlain || PART) {
      const float away = (float)(t * KT + 8 * half - place);
#pragma unroll
      for (int k = 0; k < NK; ++k)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int i = 32 * k + 16 * (r >> 3) + (r & 7), j = t * KT + 8 * half + i;
          float v = st[k][r];
          if constexpr (BEND != kPlain) v = bent_score<T, BEND>(a, v, slope, away + (float)i);
          if constexpr (PART) v = (unsigned)(j - lo[0]) < (unsigned)span[0] ? v : -INFINITY;
          st[k][r] = v;
        }
    }
    // Weights against the reference that the row has.  The maximum is looked for only where that gives a sum of
    // weights past kMost (or no key was seen before): far from overflow in the types, and as exact.
    u32x4 pf[NB];
    float add = 0.0f;
    auto weights = [&] {
      const float neg = ref == -INFINITY ? 0.0f : -ref;  // nothing seen yet: all weights are exp2(-inf)
      add = 0.0f;
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        float e[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = __builtin_amdgcn_exp2f(fmaf(st[j / 2][8 * (j % 2) + i], cs, neg));
        // The weights are rounded to the type for the product with the values, as the values are, and their sum
        // is that of the rounded ones.
        pf[j] = pack_chunk<T>(e);
#pragma unroll
        for (int i = 0; i < 4; ++i) add = pair_sum<T>(pf[j][i], add);
      }
    };
    weights();
    if (__builtin_expect(__any(add > kMost || ref == -INFINITY), 0)) {
      float v = st[0][0];
#pragma unroll
      for (int k = 0; k < NK; ++k)
#pragma unroll
        for (int r = 0; r < 16; ++r) v = fmaxf(v, st[k][r]);
      const float now = fmaxf(ref, half_max(v) * cs);
      const float alpha = now == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(ref - now);
      ref = now;
      sum[0] *= alpha;
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        pin<ACC>(o[d]);
        o[d] *= alpha;
        pin<ACC>(o[d]);
      }
      weights();
    }
    sum[0] += add;
    auto value = [&](int j, int d) { return *reinterpret_cast<const u32x4*>(vl + j * BLOCK + (half * D + 32 * d + c) * 16); };
    if constexpr (!PART) {
      read_and_multiply<NB * ND>([&](int i) { return value(i / ND, i % ND); },
                                 [&](int i, u32x4 v) { o[i % ND] = mma32<T>(v, pf[i / ND], o[i % ND]); });
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
          o[d] = mma32<T>(vf, pf[j], o[d]);
        }
      }
      if (__any(nf != 0)) {
#pragma unroll 1
        for (int j = 0; j < NB; ++j) {
          const u32x4 seen = seen_of(j);
          u32x4 ch = pf[0];
#pragma unroll
          for (int i = 1; i < NB; ++i) ch = j == i ? pf[i] : ch;
          ch = each<T>(ch, weight_code<T>);
#pragma unroll
          for (int d = 0; d < ND; ++d) {
            f32x16 x;
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] = 0.0f;
            x = mma32<T>(each<T>(value(j, d) & seen, value_code<T>), ch, x);
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] = decoded(x[i]);
            pin<ACC>(o[d]);
            o[d] += x;
            pin<ACC>(o[d]);
          }
        }
      }
    }
  };

  // Tile t has arrived, and everyone is done with the one before it: the next to load takes its place.  The tiles after t
  // may be on their way still; a narrower head's loads are fewer, and then all are waited for.
  auto arrive = [&](int t) {
    if (BUFS > 2 && D == DT && t + BUFS - 2 < t1) mlxq_vmcnt<(BUFS - 2) * PER>();
    else mlxq_vmcnt<0>();
    asm volatile("" ::: "memory");
    __syncthreads();
    if (t + BUFS - 1 < t1) load(t + BUFS - 1);
  };
  // Tiles [ta, tb) are seen whole by every row; those before (a window's start) and after (the diagonal) are not.
  // One loop each, run twice, so that the long one has no branch but the rescaling.
  int ta = min(max((kr.lo_all + KT - 1) / KT, t0), t1);
  const int tz = max(min(kr.hi_all / KT, t1), ta);
#pragma unroll 1
  for (int t = t0; t < t1;) {
#pragma unroll 1
    for (; t < ta; ++t) {
      arrive(t);
      if (idle) continue;
      step(t, BoolConstant<true>{});
    }
    ta = t1;
#pragma unroll 1
    for (; t < tz; ++t) {
      arrive(t);
      if (idle) continue;
      step(t, BoolConstant<false>{});
    }
  }

#pragma unroll
  for (int d = 0; d < ND; ++d) pin<ACC>(o[d]);
  __syncthreads();
  if (any_wave<4>(bad, reinterpret_cast<int*>(lds))) poison(bt, table, max(t0 * KT, kr.lo), min(t1 * KT, kr.hi), lo, span, sum);
  float l = half_sum(sum[0]);
  if (wr0 + c > row1) return;
  const int64_t orow = (int64_t)(s.q0 + tok) * a.Hkv * a.G + qh;
  if (ns > 1) {
    float* y = a.part + (orow * a.S + z) * D;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int f = 32 * d + 8 * i + 4 * half;
        if (f < D) *reinterpret_cast<f32x4*>(y + f) = f32x4{o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]};
      }
    if (half == 0) {
      *reinterpret_cast<f32x2*>(a.ml + (orow * a.S + z) * 2) = f32x2{ref, l};
      if (z == 0) a.splits[orow] = ns;
    }
  } else {
    if (a.S > 1 && half == 0) a.splits[orow] = 1;
    if (a.sinks) l += __builtin_amdgcn_exp2f(a.sinks[qh] * kLog2e - (ref == -INFINITY ? 0.0f : ref));
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    T* y = (T*)a.out.p + (s.q0 + tok) * a.out.ts + qh * a.out.hs;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int f = 32 * d + 8 * i + 4 * half;
        if (f < D)
          *reinterpret_cast<u32x2*>(y + f) = u32x2{Elem<T>::pack2(o[d][4 * i] * inv, o[d][4 * i + 1] * inv),
                                                   Elem<T>::pack2(o[d][4 * i + 2] * inv, o[d][4 * i + 3] * inv)};
      }
  }
}

template <typename T, int DT>
static int launch_tile(const AttnArgs& a, const AttnPlan& plan, hipStream_t st) {
  const dim3 grid((unsigned)plan.blocks, (unsigned)a.S);
  if (a.softcap > kNearCap) hipLaunchKernelGGL((attn_tile_kernel<T, DT, kFar>), grid, dim3(256), 0, st, a);
  else if (a.slopes) hipLaunchKernelGGL((attn_tile_kernel<T, DT, kBias>), grid, dim3(256), 0, st, a);
  else if (a.softcap > 0.0f) hipLaunchKernelGGL((attn_tile_kernel<T, DT, kCap>), grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((attn_tile_kernel<T, DT, kPlain>), grid, dim3(256), 0, st, a);
  return check_launch("paged_attention");
}

template <typename T>
static int tile_of(const AttnArgs& a, const AttnPlan& plan, hipStream_t st) {
  if (a.D <= 64) return launch_tile<T, 64>(a, plan, st);
  if (a.D <= 96) return launch_tile<T, 96>(a, plan, st);
  if (a.D <= 128) return launch_tile<T, 128>(a, plan, st);
  return launch_tile<T, 256>(a, plan, st);
}

}  // namespace mlxq
