// Causal chunk-prefill attention over the paged 4-bit KV cache (format: fp4_kv.cuh), any
// number of sequences: sequence s has queries q[cu_q[s] .. cu_q[s + 1]) at positions
// kv_lens[s] - q_len + i, each attending to the cached keys up to its own position.
//
// Tensor bound (4 * 128 * Hq operations per visible pair), so both products run on tcgen05
// with fp32 accumulators in TMEM. One CTA handles two tiles of 128 query rows, a row being
// a (token, query head) pair of the G = Hq / Hkv heads that share a kv head, over steps of
// 64 keys that both read:
//   warps 0-3, 4-7   softmax of tile 0 / 1: a thread owns a row. It reads its 64 scores of a
//                    step from TMEM, writes the weights over them as f16, and keeps the row's
//                    maximum and sum (fp32).
//   warps 8-13       decode K and V codes to f16 in shared memory (128-byte swizzle), a
//                    ring of kSlots 16 KB slots in the order K0 V0 K1 V1 ..., a warp a slot:
//                    the fence between its stores and the tensor core's reads and the
//                    barriers cost as much as 16 keys' work (16 keys a turn: 1.34 ms).
//   warps 14, 15     each issues one tile's S = Q K^T (both in shared memory, K-major) and
//                    O += P V (P from TMEM, V as it lies in the cache: MN-major). One warp for
//                    both tiles spends 1.6 thousand cycles a step on waits and issue, the
//                    tensor core needs 1.24. Warp 15 allocates TMEM.
// The scores are double-buffered (TMEM: two tiles x two S of 64 columns, two O of 128), so S of
// the next step is there when a softmax ends and the chain S -> softmax -> P V of a tile never
// stalls its softmax warps: with one S a tile (128 keys a step, or 64 and Q in TMEM) the
// chain's latencies showed, 1.11 and 1.25 ms for 2048 queries on 30720 tokens.
// Softmax in the exp2 domain against a lazy reference: weights are 2^(s - m) for a reference
// m that moves, with a rescale of O in TMEM, only when a row's maximum exceeds it by 8 or
// more. Weights are rounded to f16 for the second product (2^-11 relative; the first
// rounding below fp32 in the kernel, K and V are exact), the row sums take them unrounded.
//
// V rows behind the sequence's end and rows of bad pages are written as zeros, and a NaN group
// of V as zeros too, because a zero weight does not hide a NaN from the product: the first
// key with a NaN is kept per 16 elements, and the rows that see it get NaN at the end.
#define MS_WHOLE_PROGRAM  // setmaxnreg below
#include <mutex>

#include "fp4_kv.cuh"
#include "kernels.h"

namespace ms {
namespace {

constexpr int kD = kFp4Dim;
constexpr int kRows = 128;                    // query rows of a tile (MMA M)
constexpr int kKeys = 64;                     // keys of a step
constexpr int kHalf = kKeys * 128;            // 64 keys x 64 elements of f16, 128-byte swizzled
constexpr int kSlotBytes = 2 * kHalf;         // K or V of a step
constexpr int kSlots = 10;
constexpr int kDecodeWarps = 6;
constexpr int kThreads = (8 + kDecodeWarps + 2) * 32;
constexpr int kMmaWarp = 8 + kDecodeWarps;     // of tile 0; the next one is tile 1's

constexpr int kQHalf = kRows * 128;             // 128 rows x 64 elements of Q, 128-byte swizzled
constexpr int kQBytes = 2 * 2 * kQHalf;        // two tiles
constexpr int kSmemBytes = kQBytes + kSlots * kSlotBytes + 1024 /* alignment */;
constexpr int kTmemCols = 512;
constexpr int kColO = 256;                    // first column of O0; S of tile t, step j: t * 128 + (j & 1) * 64
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kPScaleLog2 = 6.f;            // weights up to 2^(6 + 8)
constexpr float kMove = 8.f;                  // the reference moves when a maximum exceeds it by this

// tcgen05 instruction descriptors: D f32, A and B f16, M = 128, N = 64 keys / 128 elements; V is
// MN-major (bit 16)
constexpr uint32_t kIdescQK = (1u << 4) | ((uint32_t)(kKeys >> 3) << 17) | ((uint32_t)(kRows >> 4) << 24);
constexpr uint32_t kIdescPV =
    (1u << 4) | (1u << 16) | ((uint32_t)(kD >> 3) << 17) | ((uint32_t)(kRows >> 4) << 24);

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ uint32_t pack_h2(float lo, float hi) {
  __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&h);
}

// Shared-memory descriptors of 128-byte swizzled f16 tiles (rows of 128 bytes, 8-row groups
// 1024 bytes apart). K-major (Q, K): a row is 64 elements of the contracted axis. MN-major
// (V): a row is 64 output elements of one key, the next 64 lie kHalf bytes further.
__device__ __forceinline__ uint64_t desc_base(uint32_t addr, uint32_t lbo) {
  return (uint64_t)((addr & 0x3FFFF) >> 4) | ((uint64_t)(lbo >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
         ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}

__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t accum,
                                       uint32_t lead) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(da), "l"(db), "r"(idesc), "r"(accum), "r"(lead));
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t db, uint32_t idesc, uint32_t accum, uint32_t lead) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(db), "r"(idesc), "r"(accum), "r"(lead));
}
__device__ __forceinline__ void mma_commit(uint64_t* bar, uint32_t lead) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar)),
      "r"(lead)
      : "memory");
}
// One lane of the (converged) warp.
__device__ __forceinline__ uint32_t elect_one() {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(r));
  return r;
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// 32 columns of this thread's TMEM lane
__device__ __forceinline__ void tmem_ld32(uint32_t addr, float (&v)[32]) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr));
}
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(
          addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
// Scores of keys that the row does not see (bits of `seen` not set).
__device__ __forceinline__ void hide(float (&x)[32], uint32_t seen) {
#pragma unroll
  for (int i = 0; i < 32; ++i)
    if (!((seen >> i) & 1u)) x[i] = -INFINITY;
}
__device__ __forceinline__ float max32(const float (&x)[32], float m) {
  float t[4] = {m, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
  for (int i = 0; i < 32; i += 8)
#pragma unroll
    for (int u = 0; u < 4; ++u) t[u] = fmaxf(fmaxf(t[u], x[i + 2 * u]), x[i + 2 * u + 1]);
  return fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3]));
}

// Every thread of the CTA, from the ends of the roles.
__device__ __forceinline__ void role_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kThreads) : "memory"); }

__device__ __forceinline__ void tmem_ld16(uint32_t addr, float (&v)[16]) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(addr));
}

struct PrefillArgs {
  const __half* q;  // [T, Hq, D], token stride q_ts elements
  int64_t q_ts;
  const uint8_t *kc, *vc, *ks, *vs;
  int64_t num_blocks;
  const int32_t* tables;  // [S, max_blocks]
  const int32_t* cu_q;    // [S + 1]
  const int32_t* kv_lens;
  __half* out;  // [T, Hq, D]
  int num_seqs, total_q, Hkv, G, block_size, bs_log2, max_blocks;
  int cap;  // tokens that a table row can hold
  float scale_log2;
};

struct Item {
  int seq, tok0;  // first query token of the CTA within its sequence
};

__global__ void __launch_bounds__(kThreads, 1) prefill_fp4_kernel(const __grid_constant__ PrefillArgs a) {
  extern __shared__ __align__(16) unsigned char smem_raw[];
  __shared__ uint64_t q_full[2], full[kSlots], empty[kSlots], s_full[2][2], p_ready[2][2], pv_done[2];
  __shared__ uint32_t s_tmem;
  __shared__ Item s_item;
  __shared__ int s_nan[8];  // first key whose V group is NaN, per 16 elements
  __shared__ int s_bad;     // the sequence has a page outside the cache
  unsigned char* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  unsigned char* s_q = smem;
  unsigned char* s_kv = smem + kQBytes;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_wait();
  pdl_trigger();
  const int G = a.G, tpt = kRows / G;  // tokens per tile
  const int kvh = blockIdx.y;

  if (warp == kMmaWarp + 1) {
    // this CTA's sequence and first token: a scan of the sequences' numbers of CTAs
    int left = blockIdx.x, found = -1, tok0 = 0;
    for (int s0 = 0; s0 < a.num_seqs && found < 0; s0 += 32) {
      const int s = s0 + lane;
      const int ql = s < a.num_seqs ? max(a.cu_q[s + 1] - a.cu_q[s], 0) : 0;
      const int nb = (ql + 2 * tpt - 1) / (2 * tpt);
      int inc = nb;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += up;
      }
      const uint32_t hit = __ballot_sync(0xffffffffu, left < inc);
      if (hit != 0) {
        const int l = __ffs(hit) - 1;
        const int before = __shfl_sync(0xffffffffu, inc - nb, l), mine = __shfl_sync(0xffffffffu, nb, l);
        found = s0 + l;
        tok0 = (mine - 1 - (left - before)) * 2 * tpt;  // the longest prefixes first
      } else {
        left -= __shfl_sync(0xffffffffu, inc, 31);
      }
    }
    if (lane == 0) {
      s_item = Item{found, tok0};
      s_bad = 0;
      const int ql = found < 0 ? 0 : a.cu_q[found + 1] - a.cu_q[found];
      for (int i = 0; i < kSlots; ++i) {
        mbar_init(&full[i], 1);
        mbar_init(&empty[i], ql - tok0 > tpt ? 2 : 1);  // the products of every tile have read the slot
      }
      for (int i = 0; i < 2; ++i) {
        mbar_init(&q_full[i], 128);
        for (int h = 0; h < 2; ++h) {  // the steps' parities
          mbar_init(&s_full[i][h], 1);
          mbar_init(&p_ready[i][h], 128);
        }
        mbar_init(&pv_done[i], 1);
      }
      fence_barrier_init();
    }
    if (lane < 8) s_nan[lane] = INT32_MAX;
    __syncwarp();
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)),
                 "r"(kTmemCols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;
  const Item item = s_item;
  const int q_start = item.seq < 0 ? 0 : a.cu_q[item.seq];
  const int q_len = item.seq < 0 ? 0 : a.cu_q[item.seq + 1] - q_start;
  int kv_len = item.seq < 0 ? 0 : a.kv_lens[item.seq];
  const int prefix = kv_len - q_len;  // position of the first query
  if (kv_len > a.cap) {
    if (threadIdx.x == 0) set_device_status(kStatusBadPage);
    kv_len = a.cap;
  }
  const int n_tok = min(2 * tpt, q_len - item.tok0);  // query tokens of this CTA
  const int tiles = n_tok > tpt ? 2 : 1;
  const int last_pos = prefix + item.tok0 + n_tok - 1;  // of the CTA's last query
  const int n_keys = item.seq < 0 ? 0 : max(0, min(kv_len, last_pos + 1));
  const int n_kv = (n_keys + kKeys - 1) / kKeys;
  const int32_t* table = a.tables + (int64_t)max(item.seq, 0) * a.max_blocks;

  if (item.seq >= 0 && warp < 8) {
    // ------------------------------------------------------------------ softmax
    const int t = warp >> 2;                                  // tile
    const int row = (warp & 3) * 32 + lane;                   // TMEM lane
    const int tt = t * tpt + row / G, h = row % G;            // token of the CTA, head of the group
    const bool valid = row < tpt * G && tt < n_tok;
    const int lim = valid ? min(prefix + item.tok0 + tt, kv_len - 1) : -1;  // last visible key
    if (t < tiles) {
      const uint32_t lane_base = tmem + ((uint32_t)((warp & 3) * 32) << 16);
      const uint32_t o_addr = lane_base + kColO + t * kD;
      // Q: 16 lanes a row
      const int tw = threadIdx.x & 127;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int r = (tw >> 4) + 8 * i, ch = tw & 15;
        const int rt = t * tpt + r / G;
        uint4 x = make_uint4(0, 0, 0, 0);
        if (r < tpt * G && rt < n_tok)
          x = *reinterpret_cast<const uint4*>(a.q + (int64_t)(q_start + item.tok0 + rt) * a.q_ts +
                                              (kvh * G + r % G) * kD + ch * 8);
        *reinterpret_cast<uint4*>(s_q + (t * 2 + (ch >> 3)) * kQHalf + r * 128 + (((ch & 7) ^ (r & 7)) << 4)) = x;
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      mbar_arrive(&q_full[t]);
      int low = lim;  // smallest limit of the warp: tiles below it need no mask
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) low = min(low, __shfl_xor_sync(0xffffffffu, low, o));
      float m = -INFINITY, l = 0.f;  // reference (log2 units, less kPScaleLog2) and sum
      bool ok = true;
      for (int j = 0; j < n_kv; ++j) {
        if (!mbar_wait(&s_full[t][j & 1], (j >> 1) & 1)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const int kbase = j * kKeys;
        const uint32_t s_addr = lane_base + t * 128 + (j & 1) * kKeys;
        const bool masked = kbase + kKeys - 1 > low || *reinterpret_cast<volatile int*>(&s_bad) != 0;
        // ---- the row's 64 scores, and their maximum ---------------------------------------------
        float v[2][32];
#pragma unroll
        for (int c = 0; c < 2; ++c) tmem_ld32(s_addr + 32 * c, v[c]);
        tmem_ld_wait();
        if (masked) {
          const bool bad = *reinterpret_cast<volatile int*>(&s_bad) != 0;
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const int k0 = kbase + 32 * c, n = lim - k0 + 1;  // keys of these 32 that the row sees
            uint32_t seen = n >= 32 ? 0xffffffffu : (n <= 0 ? 0u : (1u << n) - 1u);
            if (bad) {  // rare: leave out the keys of bad pages
              const int pg = k0 / a.block_size;
              const int64_t blk = pg < a.max_blocks ? table[pg] : -1;
              if (blk < 0 || blk >= a.num_blocks) seen = 0;
            }
            hide(v[c], seen);
          }
        }
        const float mx = max32(v[1], max32(v[0], -INFINITY)) * a.scale_log2;
        // ---- the reference moves when some row's maximum is far above it ---------------------
        const bool far = mx - kPScaleLog2 > m + kMove || (m == -INFINITY && mx > -INFINITY);
        if (__any_sync(0xffffffffu, far)) {
          const float mn = far ? mx - kPScaleLog2 : m;
          const float al = m == -INFINITY ? 1.f : ex2(m - mn);
          m = mn;
          l *= al;
          if (j > 0) {
            if (!mbar_wait(&pv_done[t], (j - 1) & 1)) {
              ok = false;
              break;
            }
            tc_fence_after();
#pragma unroll
            for (int c = 0; c < 8; ++c) {
              float o[16];
              tmem_ld16(o_addr + 16 * c, o);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] *= al;
              tmem_st16(o_addr + 16 * c, *reinterpret_cast<uint32_t(*)[16]>(o));
            }
            tmem_st_wait();
          }
        }
        // ---- weights, f16, over the scores ----------------------------------------------------
        const float neg = m == -INFINITY ? 0.f : -m;
        const uint64_t sc2 = f32x2(a.scale_log2, a.scale_log2), neg2 = f32x2(neg, neg);
        uint64_t sum[2] = {0, 0};
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t p[16];
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            float x0, x1;
            unpack2(fma2(f32x2(v[c][i], v[c][i + 1]), sc2, neg2), x0, x1);
            x0 = ex2(x0);
            x1 = ex2(x1);
            sum[(i >> 1) & 1] = add2(sum[(i >> 1) & 1], f32x2(x0, x1));
            p[i >> 1] = pack_h2(x0, x1);
          }
          tmem_st16(s_addr + 16 * c, p);
        }
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(&p_ready[t][j & 1]);
        {
          float x0, x1;
          unpack2(add2(sum[0], sum[1]), x0, x1);
          l += x0 + x1;
        }
      }
      // ---- O / l ----------------------------------------------------------------------------------
      if (ok && n_kv > 0) {
        ok = mbar_wait(&pv_done[t], (n_kv - 1) & 1);
        tc_fence_after();
      }
      role_sync();  // every V tile has been decoded: s_nan is complete
      const float inv = l == 0.f ? 0.f : 1.f / l;
      __half* dst = a.out + ((int64_t)(q_start + item.tok0 + tt) * a.Hkv * G + kvh * G + h) * kD;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        float v[32];
        if (n_kv > 0) {
          tmem_ld32(o_addr + 32 * c, v);
          tmem_ld_wait();
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = 0.f;
        }
        if (ok && valid) {
#pragma unroll
          for (int g2 = 0; g2 < 2; ++g2) {
            const float f = s_nan[2 * c + g2] <= lim ? __int_as_float(0x7fffffff) : inv;
#pragma unroll
            for (int i = 0; i < 16; i += 8) {
              const float* x = v + 16 * g2 + i;
              *reinterpret_cast<uint4*>(dst + 32 * c + 16 * g2 + i) =
                  make_uint4(pack_h2(x[0] * f, x[1] * f), pack_h2(x[2] * f, x[3] * f), pack_h2(x[4] * f, x[5] * f),
                             pack_h2(x[6] * f, x[7] * f));
            }
          }
        }
      }
    } else {
      role_sync();
    }
  } else if (item.seq >= 0) {
    if (warp < kMmaWarp) {
    // ------------------------------------------------------------------ decode of K and V
    // a lane's part of a slot: rows lr + 8 i, elements 64 half + 32 c2 .. + 32 of each
    const int lr = (lane >> 1) & 7, c2 = lane & 1, half = lane >> 4;
    // 16-byte chunks 4 c2 + k of a row, swizzled; 8 lanes (4 rows, both c2) hit 8 chunk positions
    uint32_t chunk[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) chunk[k] = (uint32_t)(half * kHalf + lr * 128 + (((4 * c2 + k) ^ lr) << 4));
    // Consecutive uses of a slot belong to different warps. A warp waits for its use by parity all the
    // same: its own slot before lay kDecodeWarps back and waited for the release of the one kSlots
    // before that, which (releases keep the order, but for neighbours) came after the release
    // of the use before the last of this slot.
    static_assert(kSlots > kDecodeWarps, "parity of the slots' uses");
    for (int n = warp - 8; n < 2 * n_kv; n += kDecodeWarps) {  // K (n even) or V (odd) of step n / 2
      const int k0 = (n >> 1) * kKeys;
      const int page = a.bs_log2 >= 0 ? k0 >> a.bs_log2 : k0 / a.block_size;
      const int64_t blk = page < a.max_blocks ? __ldg(table + page) : -1;
      const bool live = blk >= 0 && blk < a.num_blocks;
      uint4 codes[kKeys / 8];
      uint32_t sc[kKeys / 8];  // two scale bytes; 0: zeros, whatever the codes
      if (live) {
        const int64_t r0 = (blk * a.Hkv + kvh) * a.block_size + (k0 - page * a.block_size) + lr;
        const uint8_t* cp = ((n & 1) ? a.vc : a.kc) + r0 * kFp4RowBytes + half * 32 + c2 * 16;
        const uint8_t* sp = ((n & 1) ? a.vs : a.ks) + r0 * kFp4ScaleBytes + half * 4 + c2 * 2;
#pragma unroll
        for (int i = 0; i < kKeys / 8; ++i) {
          codes[i] = __ldg(reinterpret_cast<const uint4*>(cp + i * 8 * kFp4RowBytes));
          sc[i] = __ldg(reinterpret_cast<const uint16_t*>(sp + i * 8 * kFp4ScaleBytes));
        }
        if (k0 + kKeys > n_keys) {
#pragma unroll
          for (int i = 0; i < kKeys / 8; ++i)
            if (k0 + lr + 8 * i >= n_keys) sc[i] = 0;
        }
      } else {
        set_device_status(kStatusBadPage);
        s_bad = 1;
#pragma unroll
        for (int i = 0; i < kKeys / 8; ++i) {
          codes[i] = make_uint4(0, 0, 0, 0);
          sc[i] = 0;
        }
      }
      const int slot = n % kSlots;
      if (!mbar_wait(&empty[slot], ((n / kSlots) & 1) ^ 1)) break;
      unsigned char* dst = s_kv + slot * kSlotBytes;
#pragma unroll
      for (int i = 0; i < kKeys / 8; ++i) {
        uint32_t s = sc[i];
        if ((n & 1) && ((s & 0xF8u) == 0xF8u || (s & 0xF800u) == 0xF800u)) {
          // V: no NaN (or infinity) reaches the product
          const int key = k0 + lr + 8 * i;
          if ((s & 0xF8u) == 0xF8u) {
            atomicMin(&s_nan[4 * half + 2 * c2], key);
            s &= 0xFF00u;
          }
          if ((s & 0xF800u) == 0xF800u) {
            atomicMin(&s_nan[4 * half + 2 * c2 + 1], key);
            s &= 0xFFu;
          }
        }
        const uint32_t f[2] = {fp4_scale_h2(s & 0xFFu), fp4_scale_h2(s >> 8)};
        const uint32_t cw[4] = {codes[i].x, codes[i].y, codes[i].z, codes[i].w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          uint32_t e[4];
          fp4x8_to_f16x2(cw[k], e);
          *reinterpret_cast<uint4*>(dst + chunk[k] + i * 1024) =
              make_uint4(h2_mul(e[0], f[k >> 1]), h2_mul(e[1], f[k >> 1]), h2_mul(e[2], f[k >> 1]), h2_mul(e[3], f[k >> 1]));
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // plain stores -> the tensor core's reads
      __syncwarp();
      if (lane == 0) mbar_arrive(&full[slot]);
    }
    __syncwarp();
    role_sync();
    } else {
    // ------------------------------------------------------------------ MMA issue
    // The whole warp walks the loop, so that descriptors and addresses stay in uniform registers, and
    // one lane's products and commits count: issued by one thread in a divergent branch, a product took
    // some 70 cycles to issue, more than to run.
    const int t = warp - kMmaWarp;  // tile
    if (t < tiles && n_kv > 0) {
      const uint32_t lead = elect_one();
      const uint32_t kv0 = smem_u32(s_kv);
      const uint64_t dq = desc_base(smem_u32(s_q) + t * 2 * kQHalf, 16);
      // slot number n is stage n % kSlots in its use n / kSlots
      auto wait_full = [&](int stage, int use) { return mbar_wait(&full[stage], use & 1); };
      auto scores = [&](int stage, int j) {  // S = Q K_j^T
        const uint64_t dk = desc_base(kv0 + stage * kSlotBytes, 16);
        const uint32_t d = tmem + t * 128 + (j & 1) * kKeys;
#pragma unroll
        for (int k = 0; k < 8; ++k)  // 16 elements each
          mma_ss(d, dq + (uint64_t)(((k >> 2) * kQHalf + (k & 3) * 32) >> 4),
                 dk + (uint64_t)(((k >> 2) * kHalf + (k & 3) * 32) >> 4), kIdescQK, k > 0, lead);
        mma_commit(&s_full[t][j & 1], lead);
      };
      // nobody waits for the last slots: no arrival may outlive the CTA
      const int last_release = 2 * n_kv - kSlots;
      bool ok = mbar_wait(&q_full[t], 0) && wait_full(0, 0);
      if (ok) {
        tc_fence_after();
        scores(0, 0);
        if (0 < last_release) mma_commit(&empty[0], lead);
      }
      int kst = 2 % kSlots, kuse = 0, vst = 1, vuse = 0;  // stages and uses of K_{j+1} and V_j
      static_assert(kSlots % 2 == 0 && kSlots > 2, "K and V keep their parity of stages");
      for (int j = 0; ok && j < n_kv; ++j) {
        if (j + 1 < n_kv) {
          // S of the next step: its buffer held the weights of step j - 1, whose product was issued before
          ok = wait_full(kst, kuse);
          if (!ok) break;
          tc_fence_after();
          scores(kst, j + 1);
          if (2 * j + 2 < last_release) mma_commit(&empty[kst], lead);
          kst += 2;
          if (kst >= kSlots) {
            kst -= kSlots;
            ++kuse;
          }
        }
        ok = wait_full(vst, vuse) && mbar_wait(&p_ready[t][j & 1], (j >> 1) & 1);
        if (!ok) break;
        tc_fence_after();
        const uint64_t dv = desc_base(kv0 + vst * kSlotBytes, kHalf);
        const uint32_t p = tmem + t * 128 + (j & 1) * kKeys;
#pragma unroll
        for (int k = 0; k < kKeys / 16; ++k)  // 16 keys each
          mma_ts(tmem + kColO + t * kD, p + 8 * k, dv + (uint64_t)((k * 2048) >> 4), kIdescPV, j > 0 || k > 0, lead);
        mma_commit(&pv_done[t], lead);
        if (2 * j + 1 < last_release) mma_commit(&empty[vst], lead);
        vst += 2;
        if (vst >= kSlots) {
          vst -= kSlots;
          ++vuse;
        }
      }
    }
    __syncwarp();
    role_sync();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp + 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols));
  }
}

}  // namespace

cudaError_t prefill_fp4_take_status(int* host, cudaStream_t stream) {
  static const int zero = 0;
  cudaError_t e = cudaMemcpyFromSymbolAsync(host, g_device_status, sizeof(int), 0, cudaMemcpyDeviceToHost, stream);
  if (e == cudaSuccess)
    e = cudaMemcpyToSymbolAsync(g_device_status, &zero, sizeof(int), 0, cudaMemcpyHostToDevice, stream);
  return e;
}

cudaError_t prefill_fp4_set_wait_limit(unsigned long long ns) {
  return cudaMemcpyToSymbol(g_wait_limit_ns, &ns, sizeof(ns));
}

cudaError_t launch_prefill_fp4(const void* q, int64_t q_ts, const void* k_cache, const void* v_cache,
                               const void* k_scale, const void* v_scale, int64_t num_blocks,
                               const int32_t* block_tables, const int32_t* cu_q, const int32_t* kv_lens, void* out,
                               int num_seqs, int total_q, int Hq, int Hkv, int block_size, int max_blocks,
                               float softmax_scale, cudaStream_t stream) {
  PrefillArgs a = {};
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
  a.Hkv = Hkv;
  a.G = Hq / Hkv;
  a.block_size = block_size;
  a.bs_log2 = (block_size & (block_size - 1)) == 0 ? __builtin_ctz((unsigned)block_size) : -1;
  a.max_blocks = max_blocks;
  const int64_t cap = (int64_t)max_blocks * block_size;
  a.cap = (int)(cap < (1 << 30) ? cap : (1 << 30));
  a.scale_log2 = softmax_scale * kLog2e;
  const int tpc = 2 * (kRows / a.G);
  // CTAs over all sequences: sum ceil(len / tpc) <= total / tpc + sequences
  const int64_t blocks = (int64_t)total_q / tpc + num_seqs;
  static std::once_flag once;
  static cudaError_t attr = cudaSuccess;
  std::call_once(once, [] {
    attr = cudaFuncSetAttribute(prefill_fp4_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes);
  });
  if (attr != cudaSuccess) return attr;
  return launch_kernel(prefill_fp4_kernel, dim3((unsigned)blocks, (unsigned)Hkv), dim3(kThreads), kSmemBytes, stream, a);
}

}  // namespace ms
