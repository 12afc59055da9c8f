// pages.hip — copies of cache pages, and the block tables that follow them.
//
// Bound by HBM: each page is read and written once, in 16-byte pieces, four in flight a thread (600 pages in 32
// planes, 1.26 GB moved: 258 us, 4.9 TB/s, the rate of a large copy; 8 pages in 48 planes: 5.2 us).  The
// pages of all planes (the keys and values of every layer) are one launch, so that forking a
// sequence's last page in every layer is not a launch a layer.  The table entries are redirected by
// further workgroups of the same launch: each holds 1024 entries and runs through the list of moves,
// staged in LDS; rows * width * count comparisons, a few microseconds against the milliseconds that
// moving as many pages takes.
#include "paged.h"

namespace mlxq {

constexpr int kPiece = 16384;  // bytes of a page that a workgroup copies

__global__ __launch_bounds__(256) void copy_pages_kernel(unsigned char* cache, int64_t plane_stride, int64_t page_stride,
                                                         int64_t page_bytes, int pages, const int32_t* __restrict__ src,
                                                         const int32_t* __restrict__ dst, int64_t count, int pieces,
                                                         int64_t copies, int32_t* tables, int64_t entries, int64_t width,
                                                         int64_t table_stride) {
  __shared__ int32_t ls[1024], ld[1024];
  const int tid = threadIdx.x;
  if ((int64_t)blockIdx.x >= copies) {
    const int64_t base = ((int64_t)blockIdx.x - copies) * 1024 + tid;
    int32_t *at[4], old[4], now[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int64_t e = base + k * 256, r = e / width;
      at[k] = e < entries ? tables + r * table_stride + (e - r * width) : nullptr;
      old[k] = now[k] = at[k] ? *at[k] : -1;
    }
    for (int64_t m = 0; m < count; m += 1024) {
      const int n = (int)(count - m < 1024 ? count - m : 1024);
      for (int i = tid; i < n; i += 256) {
        const int32_t s = src[m + i], d = dst[m + i];
        ls[i] = s;
        // A move that the copy leaves out leaves its entries alone too.
        ld[i] = (unsigned)s < (unsigned)pages && (unsigned)d < (unsigned)pages ? d : s;
      }
      __syncthreads();
      for (int i = 0; i < n; ++i) {
        const int32_t s = ls[i], d = ld[i];
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (old[k] == s) now[k] = d;
      }
      __syncthreads();
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (at[k] && now[k] != old[k]) *at[k] = now[k];
    return;
  }
  const int64_t item = (int64_t)blockIdx.x / pieces;
  const int piece = (int)((int64_t)blockIdx.x - item * pieces);
  const int64_t plane = item / count, move = item - plane * count;
  const int32_t s = src[move], d = dst[move];
  if ((unsigned)s >= (unsigned)pages || (unsigned)d >= (unsigned)pages || s == d) return;
  const unsigned char* from = cache + plane * plane_stride + s * page_stride;
  unsigned char* to = cache + plane * plane_stride + d * page_stride;
  const int64_t end = page_bytes < (int64_t)(piece + 1) * kPiece ? page_bytes : (int64_t)(piece + 1) * kPiece;
  int64_t i = (int64_t)piece * kPiece + tid * 16;
  for (; i + 3 * 4096 < end; i += 4 * 4096) {
    u32x4 v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = *reinterpret_cast<const u32x4*>(from + i + k * 4096);
#pragma unroll
    for (int k = 0; k < 4; ++k) *reinterpret_cast<u32x4*>(to + i + k * 4096) = v[k];
  }
  for (; i < end; i += 4096) *reinterpret_cast<u32x4*>(to + i) = *reinterpret_cast<const u32x4*>(from + i);
}

int run_copy_pages(void* cache, int64_t planes, int64_t plane_stride, int64_t pages, int64_t page_bytes,
                   int64_t page_stride, const int32_t* src, const int32_t* dst, int64_t count, int32_t* tables,
                   int64_t rows, int64_t width, int64_t table_stride, hipStream_t st) {
  const int64_t pieces = (page_bytes + kPiece - 1) / kPiece, copies = planes * count * pieces;
  const int64_t entries = tables ? rows * width : 0, blocks = copies + (entries + 1023) / 1024;
  if (blocks > 0x7fffffff) return set_error(MLXQ_EINVAL, "copy_pages: problem too large");
  if (blocks == 0) return MLXQ_OK;
  hipLaunchKernelGGL(copy_pages_kernel, dim3((unsigned)blocks), dim3(256), 0, st, (unsigned char*)cache, plane_stride,
                     page_stride, page_bytes, (int)pages, src, dst, count, (int)pieces, copies, tables, entries, width,
                     table_stride);
  return check_launch("copy_pages");
}

}  // namespace mlxq
