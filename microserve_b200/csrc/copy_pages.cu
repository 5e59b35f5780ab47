// Page copies inside a paged KV cache: for every pair i and every plane (K or V of every
// layer), tokens [0, n_i) of page src[i] -> page dst[i], codes and scales in one launch.
// A page is `outer` runs of block_size rows (one run of [tokens][kv_heads * head_dim]
// in the FP8 cache, one per kv head in the 4-bit cache), so the first n tokens are a
// prefix of every run.
//
// Bound by memory: every byte is read and written once. One CTA copies one piece of up
// to kPiece bytes of a run (16-byte vectors, all loads of a thread issued before its
// stores); the pieces of all pairs, planes and runs form one flat grid-stride index.
#include "common.cuh"
#include "kernels.h"

namespace ms {
namespace {

constexpr int kThreads = 256;
constexpr int kUnroll = 4;
constexpr int kPiece = kThreads * kUnroll * 16;  // bytes of a piece

struct CopyArr {
  unsigned char* base;
  int64_t plane_stride;  // bytes between planes
  int64_t page_bytes;    // outer * block_size * row
  int64_t run_bytes;     // block_size * row
  int row;               // bytes of one token in a run
  int pieces;            // pieces of a full run
};

struct CopyArgs {
  CopyArr arr[2];  // codes, scales
  const int32_t* src;
  const int32_t* dst;
  const int32_t* tokens;  // null: whole pages
  int n, planes, outer, block_size;
  int64_t num_pages;
  int64_t work[2];  // pieces in all of arr[0], arr[1]
};

__global__ void __launch_bounds__(kThreads) copy_pages_kernel(const __grid_constant__ CopyArgs a) {
  pdl_wait();
  pdl_trigger();
  for (int64_t w = blockIdx.x; w < a.work[0] + a.work[1]; w += gridDim.x) {
    const CopyArr& c = a.arr[w < a.work[0] ? 0 : 1];
    int64_t i = w < a.work[0] ? w : w - a.work[0];
    const int piece = (int)(i % c.pieces);
    i /= c.pieces;
    const int run = (int)(i % a.outer);
    i /= a.outer;
    const int plane = (int)(i % a.planes);
    const int pair = (int)(i / a.planes);
    const int32_t s = a.src[pair], d = a.dst[pair];
    const int tok = a.tokens != nullptr ? min(max(a.tokens[pair], 0), a.block_size) : a.block_size;
    if (s < 0 || d < 0 || s >= a.num_pages || d >= a.num_pages) {
      if (threadIdx.x == 0) set_device_status(kStatusBadPage);
      continue;
    }
    const int64_t bytes = (int64_t)tok * c.row - (int64_t)piece * kPiece;  // left in this run from this piece on
    if (bytes <= 0 || s == d) continue;
    const int64_t at = plane * c.plane_stride + run * c.run_bytes + (int64_t)piece * kPiece;
    const unsigned char* sp = c.base + at + s * c.page_bytes;
    unsigned char* dp = c.base + at + d * c.page_bytes;
    uint4 v[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int o = (u * kThreads + (int)threadIdx.x) * 16;
      if (o + 16 <= bytes) v[u] = *reinterpret_cast<const uint4*>(sp + o);
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int o = (u * kThreads + (int)threadIdx.x) * 16;
      if (o + 16 <= bytes) *reinterpret_cast<uint4*>(dp + o) = v[u];
    }
    // rows are multiples of 4 bytes: up to 3 words behind the last vector of the run
    if (bytes < kPiece) {
      const int o = ((int)bytes & ~15) + (int)threadIdx.x * 4;
      if (threadIdx.x < 4 && o + 4 <= bytes)
        *reinterpret_cast<uint32_t*>(dp + o) = *reinterpret_cast<const uint32_t*>(sp + o);
    }
  }
}

}  // namespace

cudaError_t launch_copy_pages(void* cache, int64_t cache_plane_stride, int row_bytes, void* scale,
                              int64_t scale_plane_stride, int scale_row_bytes, int planes, int outer, int block_size,
                              int64_t num_pages, const int32_t* src, const int32_t* dst, const int32_t* tokens, int n,
                              int num_sms, cudaStream_t stream) {
  if (n == 0 || planes == 0) return cudaSuccess;
  if (tokens == nullptr) {  // whole pages: one run each (64 pages x 36 layers, 4-bit: 212 us, in runs 247)
    block_size *= outer;
    outer = 1;
  }
  CopyArgs a = {};
  a.src = src;
  a.dst = dst;
  a.tokens = tokens;
  a.n = n;
  a.planes = planes;
  a.outer = outer;
  a.block_size = block_size;
  a.num_pages = num_pages;
  const int rows[2] = {row_bytes, scale_row_bytes};
  void* base[2] = {cache, scale};
  const int64_t ps[2] = {cache_plane_stride, scale_plane_stride};
  for (int k = 0; k < 2; ++k) {
    CopyArr& c = a.arr[k];
    c.base = (unsigned char*)base[k];
    c.plane_stride = ps[k];
    c.row = rows[k];
    c.run_bytes = (int64_t)block_size * rows[k];
    c.page_bytes = c.run_bytes * outer;
    c.pieces = (int)((c.run_bytes + kPiece - 1) / kPiece);
    a.work[k] = (int64_t)n * planes * outer * c.pieces;
  }
  const int64_t all = a.work[0] + a.work[1];
  const int64_t ctas = all < (int64_t)num_sms * 32 ? all : (int64_t)num_sms * 32;
  return launch_kernel(copy_pages_kernel, dim3((unsigned)ctas), dim3(kThreads), 0, stream, a);
}

}  // namespace ms
