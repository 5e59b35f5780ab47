// Attention over the paged 4-bit KV cache (format: fp4_kv.cuh), one warp per (query
// token, query head): lanes take a key each for the scores, then 8 head_dim elements
// of every other key for the weighted sum of the values; online softmax in fp32.
#include "fp4_kv.cuh"
#include "kernels.h"

namespace ms {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float2 h2f(uint32_t x) {
  __half2 h;
  memcpy(&h, &x, 4);
  return __half22float2(h);
}

struct AttnArgs {
  const __half* q;
  int64_t q_ts;
  const uint8_t *kc, *vc, *ks, *vs;
  int64_t num_blocks;
  const int32_t* tables;
  const int32_t* cu_q;  // null: decode
  const int32_t* kv_lens;
  __half* out;
  int num_seqs, total_q, Hq, Hkv, block_size, max_blocks;
  float scale_log2;
};

__global__ void __launch_bounds__(128) attn_kernel(AttnArgs a) {
  pdl_wait();
  pdl_trigger();
  __shared__ float sq[4][kFp4Dim];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t item = (int64_t)blockIdx.x * 4 + warp;
  if (item >= (int64_t)a.total_q * a.Hq) return;
  const int tok = (int)(item / a.Hq), hq = (int)(item % a.Hq), kvh = hq / (a.Hq / a.Hkv);
  int seq = tok, L;
  const int cap = (int)min((int64_t)a.max_blocks * a.block_size, (int64_t)INT32_MAX);
  if (a.cu_q != nullptr) {
    seq = -1;
    for (int s = 0; s < a.num_seqs; ++s)
      if (tok >= a.cu_q[s] && tok < a.cu_q[s + 1]) {
        seq = s;
        break;
      }
    if (seq < 0) return;
    L = a.kv_lens[seq] - (a.cu_q[seq + 1] - tok) + 1;
  } else {
    L = a.kv_lens[tok];
  }
  if (L > cap) {
    set_device_status(kStatusBadPage);
    L = cap;
  }
  const __half* qp = a.q + tok * a.q_ts + hq * kFp4Dim;
  for (int i = 0; i < 4; ++i) sq[warp][lane * 4 + i] = __half2float(qp[lane * 4 + i]);
  __syncwarp();
  float m = -INFINITY, l = 0.f, o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  for (int k0 = 0; k0 < L; k0 += 32) {
    const int pg = k0 / a.block_size;
    const int64_t blk = a.tables[(int64_t)seq * a.max_blocks + pg];
    if (blk < 0 || blk >= a.num_blocks) {
      set_device_status(kStatusBadPage);
      continue;
    }
    const int64_t row0 = (blk * a.Hkv + kvh) * a.block_size + (k0 - pg * a.block_size);
    float s = -INFINITY;
    if (k0 + lane < L) {
      const uint32_t* cp = reinterpret_cast<const uint32_t*>(a.kc + (row0 + lane) * kFp4RowBytes);
      const uint8_t* sp = a.ks + (row0 + lane) * kFp4ScaleBytes;
      s = 0.f;
      for (int w = 0; w < 16; ++w) {
        uint32_t h[4];
        fp4x8_to_f16x2(cp[w], h);
        const uint32_t sc = fp4_scale_h2(sp[w >> 1]);
        for (int i = 0; i < 4; ++i) {
          const float2 f = h2f(h2_mul(h[i], sc));
          s += f.x * sq[warp][w * 8 + 2 * i] + f.y * sq[warp][w * 8 + 2 * i + 1];
        }
      }
      s *= a.scale_log2;
    }
    const float mn = fmaxf(m, warp_max(s));
    const float mu = mn == -INFINITY ? 0.f : mn;
    const float al = exp2f(m - mu);
    const float p = exp2f(s - mu);
    m = mn;
    l = l * al + warp_sum(p);
    for (int i = 0; i < 8; ++i) o[i] *= al;
    const int n = min(32, L - k0);
    for (int j0 = 0; j0 < n; j0 += 2) {  // lanes 0-15: key j0, lanes 16-31: key j0 + 1; 8 elements each
      const int j = j0 + (lane >> 4), e = lane & 15;
      const float pj = __shfl_sync(0xffffffffu, p, j);
      if (j >= n) continue;
      uint32_t h[4];
      fp4x8_to_f16x2(reinterpret_cast<const uint32_t*>(a.vc + (row0 + j) * kFp4RowBytes)[e], h);
      const uint32_t sc = fp4_scale_h2(a.vs[(row0 + j) * kFp4ScaleBytes + (e >> 1)]);
      for (int i = 0; i < 4; ++i) {
        const float2 f = h2f(h2_mul(h[i], sc));
        o[2 * i] += pj * f.x;
        o[2 * i + 1] += pj * f.y;
      }
    }
  }
  for (int i = 0; i < 8; ++i) o[i] += __shfl_xor_sync(0xffffffffu, o[i], 16);
  const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
  __half* op = a.out + ((int64_t)tok * a.Hq + hq) * kFp4Dim;
  if (lane < 16)
    for (int i = 0; i < 8; ++i) op[lane * 8 + i] = __float2half_rn(o[i] * inv);
}

}  // namespace

cudaError_t launch_fp4_attention(const void* q, int64_t q_ts, const void* k_cache, const void* v_cache,
                                 const void* k_scale, const void* v_scale, int64_t num_blocks,
                                 const int32_t* block_tables, const int32_t* cu_q, const int32_t* kv_lens, void* out,
                                 int num_seqs, int total_q, int Hq, int Hkv, int block_size, int max_blocks,
                                 float softmax_scale, cudaStream_t stream) {
  AttnArgs a;
  a.q = (const __half*)q;
  a.q_ts = q_ts;
  a.kc = (const uint8_t*)k_cache;
  a.vc = (const uint8_t*)v_cache;
  a.ks = (const uint8_t*)k_scale;
  a.vs = (const uint8_t*)v_scale;
  a.num_blocks = num_blocks;
  a.tables = block_tables;
  a.cu_q = cu_q;
  a.kv_lens = kv_lens;
  a.out = (__half*)out;
  a.num_seqs = num_seqs;
  a.total_q = total_q;
  a.Hq = Hq;
  a.Hkv = Hkv;
  a.block_size = block_size;
  a.max_blocks = max_blocks;
  a.scale_log2 = softmax_scale * kLog2e;
  const int64_t items = (int64_t)total_q * Hq;
  return launch_kernel(attn_kernel, dim3((unsigned)((items + 3) / 4)), dim3(128), 0, stream, a);
}

}  // namespace ms
