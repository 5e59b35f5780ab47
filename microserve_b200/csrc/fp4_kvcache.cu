// Writer and reader of the paged 4-bit KV cache (format: fp4_kv.cuh).
//
//  * store_kv_fp4: fp16 key / value rows -> codes and scales, scattered to `slots`
//    (slot = block * block_size + offset; negative = skipped).
//  * load_kv_fp4: the tokens at `slots` as fp16 rows (negative slot: zeros).
//
// Both are bound by memory (a row is 256 bytes of fp16 and 72 bytes of cache) and, for
// the few hundred rows of a decode step, by latency. 16 lanes share a row: a lane moves
// one 16-byte vector of fp16 (8 elements) and 4 bytes of codes, two lanes share a scale
// group (one shuffle for its maximum), so a warp reads 512 and writes 128 contiguous
// bytes for two rows; K and V of a row are in flight together.
#include "fp4_kv.cuh"
#include "kernels.h"

namespace ms {
namespace {

constexpr int kThreads = 256;
constexpr int kRowsPerCta = kThreads / 16;

struct KvFp4Args {
  const __half* k;  // store: inputs [T, Hkv, 128]; load: outputs
  const __half* v;
  int64_t k_ts, k_hs, v_ts, v_hs;  // strides of k and v in elements: token, head
  int64_t rows;                    // T * Hkv
  int kv_heads, block_size, bs_log2;
  int64_t num_slots;  // num_blocks * block_size
  const int64_t* slots;
  uint8_t* kc;
  uint8_t* vc;
  uint8_t* ks;
  uint8_t* vs;
};

// Row of (slot, head) in the cache (codes at row * 64, scales at row * 8); -1 if the slot
// is negative or outside the cache (recorded in the device status word).
__device__ __forceinline__ int64_t cache_row(const KvFp4Args& a, int64_t slot, int head) {
  if (slot < 0) return -1;
  if (slot >= a.num_slots) {
    set_device_status(kStatusBadPage);
    return -1;
  }
  const uint32_t s = (uint32_t)slot;  // num_slots < 2^31
  const uint32_t blk = a.bs_log2 >= 0 ? s >> a.bs_log2 : s / (uint32_t)a.block_size;
  const uint32_t off = s - blk * (uint32_t)a.block_size;
  return ((int64_t)blk * a.kv_heads + head) * a.block_size + off;
}

__device__ __forceinline__ void store_row(const uint4& x, int64_t row, uint8_t* __restrict__ codes,
                                          uint8_t* __restrict__ scales) {
  const int l = threadIdx.x & 15;
  const uint32_t h[4] = {x.x, x.y, x.z, x.w};
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t b = h[i] & 0x7FFF7FFFu;
    m = max(m, max(b & 0xFFFFu, b >> 16));
  }
  m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
  const uint32_t sc = fp4_scale_code(m);
  const uint32_t w = fp4_encode8(h, sc);
  if (row < 0) return;
  reinterpret_cast<uint32_t*>(codes + row * kFp4RowBytes)[l] = w;
  if ((l & 1) == 0) scales[row * kFp4ScaleBytes + (l >> 1)] = (uint8_t)sc;
}

__global__ void __launch_bounds__(kThreads) store_kv_fp4_kernel(KvFp4Args a) {
  pdl_wait();
  pdl_trigger();
  const int64_t r = (int64_t)blockIdx.x * kRowsPerCta + (threadIdx.x >> 4);
  const int l = threadIdx.x & 15;
  const bool in = r < a.rows;  // lanes past the end stay for the shuffles
  const int64_t t = in ? r / a.kv_heads : 0;
  const int head = in ? (int)(r - t * a.kv_heads) : 0;
  const uint4 kx = reinterpret_cast<const uint4*>(a.k + t * a.k_ts + head * a.k_hs)[l];
  const uint4 vx = reinterpret_cast<const uint4*>(a.v + t * a.v_ts + head * a.v_hs)[l];
  const int64_t row = in ? cache_row(a, a.slots[t], head) : -1;
  store_row(kx, row, a.kc, a.ks);
  store_row(vx, row, a.vc, a.vs);
}

__device__ __forceinline__ uint4 load_row(int64_t row, const uint8_t* __restrict__ codes,
                                          const uint8_t* __restrict__ scales) {
  if (row < 0) return make_uint4(0, 0, 0, 0);
  const int l = threadIdx.x & 15;
  const uint32_t w = reinterpret_cast<const uint32_t*>(codes + row * kFp4RowBytes)[l];
  const uint32_t s = fp4_scale_h2(scales[row * kFp4ScaleBytes + (l >> 1)]);
  uint32_t o[4];
  fp4x8_to_f16x2(w, o);
  return make_uint4(h2_mul(o[0], s), h2_mul(o[1], s), h2_mul(o[2], s), h2_mul(o[3], s));
}

__global__ void __launch_bounds__(kThreads) load_kv_fp4_kernel(KvFp4Args a) {
  pdl_wait();
  pdl_trigger();
  const int64_t r = (int64_t)blockIdx.x * kRowsPerCta + (threadIdx.x >> 4);
  if (r >= a.rows) return;
  const int64_t t = r / a.kv_heads;
  const int head = (int)(r - t * a.kv_heads);
  const int64_t row = cache_row(a, a.slots[t], head);
  const uint4 kx = load_row(row, a.kc, a.ks), vx = load_row(row, a.vc, a.vs);
  const int l = threadIdx.x & 15;
  reinterpret_cast<uint4*>(const_cast<__half*>(a.k) + r * kFp4Dim)[l] = kx;
  reinterpret_cast<uint4*>(const_cast<__half*>(a.v) + r * kFp4Dim)[l] = vx;
}

KvFp4Args kv_args(const void* k, const void* v, int64_t T, int kv_heads, const int64_t* slots, void* k_cache,
                  void* v_cache, void* k_scale, void* v_scale, int64_t num_blocks, int block_size) {
  KvFp4Args a = {};
  a.k = (const __half*)k;
  a.v = (const __half*)v;
  a.rows = T * kv_heads;
  a.kv_heads = kv_heads;
  a.block_size = block_size;
  a.bs_log2 = (block_size & (block_size - 1)) == 0 ? __builtin_ctz((unsigned)block_size) : -1;
  a.num_slots = num_blocks * block_size;
  a.slots = slots;
  a.kc = (uint8_t*)k_cache;
  a.vc = (uint8_t*)v_cache;
  a.ks = (uint8_t*)k_scale;
  a.vs = (uint8_t*)v_scale;
  return a;
}

}  // namespace

cudaError_t launch_store_kv_fp4(const void* k, const void* v, int64_t k_ts, int64_t k_hs, int64_t v_ts, int64_t v_hs,
                                int64_t T, int kv_heads, const int64_t* slots, void* k_cache, void* v_cache,
                                void* k_scale, void* v_scale, int64_t num_blocks, int block_size,
                                cudaStream_t stream) {
  if (T == 0) return cudaSuccess;
  KvFp4Args a = kv_args(k, v, T, kv_heads, slots, k_cache, v_cache, k_scale, v_scale, num_blocks, block_size);
  a.k_ts = k_ts;
  a.k_hs = k_hs;
  a.v_ts = v_ts;
  a.v_hs = v_hs;
  const int64_t ctas = (a.rows + kRowsPerCta - 1) / kRowsPerCta;
  return launch_kernel(store_kv_fp4_kernel, dim3((unsigned)ctas), dim3(kThreads), 0, stream, a);
}

cudaError_t launch_load_kv_fp4(const void* k_cache, const void* v_cache, const void* k_scale, const void* v_scale,
                               int64_t num_blocks, int block_size, int64_t T, int kv_heads, const int64_t* slots,
                               void* k, void* v, cudaStream_t stream) {
  if (T == 0) return cudaSuccess;
  const KvFp4Args a = kv_args(k, v, T, kv_heads, slots, const_cast<void*>(k_cache), const_cast<void*>(v_cache),
                              const_cast<void*>(k_scale), const_cast<void*>(v_scale), num_blocks, block_size);
  const int64_t ctas = (a.rows + kRowsPerCta - 1) / kRowsPerCta;
  return launch_kernel(load_kv_fp4_kernel, dim3((unsigned)ctas), dim3(kThreads), 0, stream, a);
}

}  // namespace ms
