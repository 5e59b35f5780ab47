// Writer and reader of the paged 4-bit KV cache (format: fp4_kv.cuh).
//
//  * store_kv_fp4: fp16 key / value rows -> codes and scales, scattered to `slots`
//    (slot = block * block_size + offset; negative = skipped).
//  * load_kv_fp4: the tokens at `slots` as fp16 rows (negative slot: zeros).
//
// Both are bound by memory (a row is 256 bytes of fp16 and 72 bytes of cache) and, for
// the few hundred rows of a decode step, by latency. A CTA handles tokens of one head, because
// the cache keeps a head's tokens together: consecutive slots give contiguous codes and
// scales.
//  * store: a lane has one group of 16 elements (32 bytes), 8 lanes a row, 4 tokens a warp, so
//    a warp's scale bytes fill a 32-byte sector and nothing is exchanged between lanes
//    (16 lanes a row, two a group: 13.4 us for 8192 tokens x 8 heads, now 10.6).
//  * load: 16 lanes a row, so a lane's 8 values are one 16-byte store; R tokens a lane, all
//    loads first.
#include "fp4_kv.cuh"
#include "kernels.h"

namespace ms {
namespace {

constexpr int kThreads = 256;
constexpr int kGroups = kThreads / 16;     // tokens of a load CTA (times R)
constexpr int kStoreThreads = 128;
constexpr int kStoreTokens = kStoreThreads / 8;

struct KvFp4Args {
  const __half* k;  // store: inputs [T, Hkv, 128]; load: outputs
  const __half* v;
  int64_t k_ts, k_hs, v_ts, v_hs;  // strides of k and v in elements: token, head
  int tokens, kv_heads, block_size, bs_log2;
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

__device__ __forceinline__ void store_group(const uint4& x0, const uint4& x1, int64_t row,
                                            uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
  const int l = threadIdx.x & 7;
  const uint32_t h0[4] = {x0.x, x0.y, x0.z, x0.w}, h1[4] = {x1.x, x1.y, x1.z, x1.w};
  // the largest |x| of the group as fp16 bits, which order as numbers do (NaN above all)
  uint32_t m2 = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) m2 = __vmaxu2(m2, __vmaxu2(h0[i] & 0x7FFF7FFFu, h1[i] & 0x7FFF7FFFu));
  const uint32_t m = max(m2 & 0xFFFFu, m2 >> 16);
  const uint32_t sc = fp4_scale_code(m);
  const uint2 w = make_uint2(fp4_encode8(h0, sc, m), fp4_encode8(h1, sc, m));
  if (row < 0) return;
  reinterpret_cast<uint2*>(codes + row * kFp4RowBytes)[l] = w;
  scales[row * kFp4ScaleBytes + l] = (uint8_t)sc;
}

__global__ void __launch_bounds__(kStoreThreads) store_kv_fp4_kernel(const __grid_constant__ KvFp4Args a) {
  pdl_wait();
  pdl_trigger();
  const int l = threadIdx.x & 7, head = blockIdx.y;
  const int64_t t = (int64_t)blockIdx.x * kStoreTokens + (threadIdx.x >> 3);
  if (t >= a.tokens) return;
  const uint4* kp = reinterpret_cast<const uint4*>(a.k + t * a.k_ts + head * a.k_hs) + 2 * l;
  const uint4* vp = reinterpret_cast<const uint4*>(a.v + t * a.v_ts + head * a.v_hs) + 2 * l;
  const uint4 k0 = kp[0], k1 = kp[1], v0 = vp[0], v1 = vp[1];
  const int64_t row = cache_row(a, a.slots[t], head);
  store_group(k0, k1, row, a.kc, a.ks);
  store_group(v0, v1, row, a.vc, a.vs);
}

// Token i of this lane's group of 16 in the CTA.
template <int R>
__device__ __forceinline__ int64_t token_of(int i) {
  return ((int64_t)blockIdx.x * R + i) * kGroups + (threadIdx.x >> 4);
}

template <int R>
__global__ void __launch_bounds__(kThreads) load_kv_fp4_kernel(const __grid_constant__ KvFp4Args a) {
  pdl_wait();
  pdl_trigger();
  const int l = threadIdx.x & 15, head = blockIdx.y;
  int64_t row[R];
#pragma unroll
  for (int i = 0; i < R; ++i) row[i] = cache_row(a, a.slots[min(token_of<R>(i), (int64_t)a.tokens - 1)], head);
  uint32_t kw[R], vw[R], ks[R], vs[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int64_t at = max(row[i], (int64_t)0);
    kw[i] = reinterpret_cast<const uint32_t*>(a.kc + at * kFp4RowBytes)[l];
    vw[i] = reinterpret_cast<const uint32_t*>(a.vc + at * kFp4RowBytes)[l];
    ks[i] = a.ks[at * kFp4ScaleBytes + (l >> 1)];
    vs[i] = a.vs[at * kFp4ScaleBytes + (l >> 1)];
  }
  auto values = [](uint32_t w, uint32_t sc) {
    uint32_t o[4];
    fp4x8_to_f16x2(w, o);
    const uint32_t s = fp4_scale_h2(sc);
    return make_uint4(h2_mul(o[0], s), h2_mul(o[1], s), h2_mul(o[2], s), h2_mul(o[3], s));
  };
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int64_t t = token_of<R>(i);
    if (t >= a.tokens) break;
    const int64_t at = (t * a.kv_heads + head) * kFp4Dim;
    const uint4 zero = make_uint4(0, 0, 0, 0);
    reinterpret_cast<uint4*>(const_cast<__half*>(a.k) + at)[l] = row[i] < 0 ? zero : values(kw[i], ks[i]);
    reinterpret_cast<uint4*>(const_cast<__half*>(a.v) + at)[l] = row[i] < 0 ? zero : values(vw[i], vs[i]);
  }
}

// Two tokens a lane where that still gives every SM several CTAs, else one. Reading 32768 tokens x 8
// heads: 34.3 us with one, 31.8 with two, 36.0 with four.
bool many_rows(int64_t T, int kv_heads, int num_sms) { return T * kv_heads >= (int64_t)num_sms * 8 * kGroups; }
template <int R>
dim3 grid_for(int64_t T, int kv_heads) {
  return dim3((unsigned)((T + kGroups * R - 1) / (kGroups * R)), (unsigned)kv_heads);
}

KvFp4Args kv_args(const void* k, const void* v, int64_t T, int kv_heads, const int64_t* slots, void* k_cache,
                  void* v_cache, void* k_scale, void* v_scale, int64_t num_blocks, int block_size) {
  KvFp4Args a = {};
  a.k = (const __half*)k;
  a.v = (const __half*)v;
  a.tokens = (int)T;
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
  const dim3 grid((unsigned)((T + kStoreTokens - 1) / kStoreTokens), (unsigned)kv_heads);
  return launch_kernel(store_kv_fp4_kernel, grid, dim3(kStoreThreads), 0, stream, a);
}

cudaError_t launch_load_kv_fp4(const void* k_cache, const void* v_cache, const void* k_scale, const void* v_scale,
                               int64_t num_blocks, int block_size, int64_t T, int kv_heads, const int64_t* slots,
                               void* k, void* v, int num_sms, cudaStream_t stream) {
  if (T == 0) return cudaSuccess;
  const KvFp4Args a = kv_args(k, v, T, kv_heads, slots, const_cast<void*>(k_cache), const_cast<void*>(v_cache),
                              const_cast<void*>(k_scale), const_cast<void*>(v_scale), num_blocks, block_size);
  if (many_rows(T, kv_heads, num_sms))
    return launch_kernel(load_kv_fp4_kernel<2>, grid_for<2>(T, kv_heads), dim3(kThreads), 0, stream, a);
  return launch_kernel(load_kv_fp4_kernel<1>, grid_for<1>(T, kv_heads), dim3(kThreads), 0, stream, a);
}

}  // namespace ms
