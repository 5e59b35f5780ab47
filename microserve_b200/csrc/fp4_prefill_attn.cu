// Causal chunk-prefill attention over the paged 4-bit KV cache (format: fp4_kv.cuh), any
// number of sequences: sequence s has queries q[cu_q[s] .. cu_q[s + 1]) at positions
// kv_lens[s] - q_len + i, each attending to the cached keys up to its own position.
//
// Tensor bound (4 * 128 * Hq operations per visible pair), so both products run on tcgen05
// with fp32 accumulators in TMEM. One CTA handles two tiles of 128 query rows, a row being
// a (token, query head) pair of the G = Hq / Hkv heads that share a kv head, over tiles of
// 128 keys that both read:
//   warps 0-3, 4-7   softmax of tile 0 / 1: a thread owns a row. It reads its 128 scores from
//                    TMEM, writes the weights over them as f16, and keeps the
//                    row's maximum and sum (fp32). While one tile's softmax runs, the
//                    tensor core works for the other.
//   warps 8-14       decode K and V codes to f16 in shared memory (128-byte swizzle), a
//                    ring of kSlots 32 KB slots in the order K0 V0 K1 V1 ..., 32 keys a
//                    warp at a time (three warps, with the next codes prefetched, could not
//                    keep up: 1.76 ms against 1.01 ms without decoding, 2048 queries on
//                    30720 tokens).
//   warp 15          allocates TMEM; one thread issues S = Q K^T (both operands K-major in
//                    shared memory) and O += P V (P from TMEM, V as it lies in the cache:
//                    MN-major).
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
constexpr int kKeys = 128;                    // keys of a tile
constexpr int kHalf = 128 * 128;              // 128 rows x 64 elements of f16, 128-byte swizzled
constexpr int kSlotBytes = 2 * kHalf;         // a K or V tile
constexpr int kSlots = 5;
constexpr int kQBytes = 2 * 2 * kHalf;        // two tiles
constexpr int kDecodeWarps = 7;
constexpr int kThreads = (8 + kDecodeWarps + 1) * 32;
constexpr int kMmaWarp = 8 + kDecodeWarps;
// Registers: 512 threads start with 128 each; the decode and MMA warps hand some to softmax.
constexpr int kSoftmaxRegs = 184, kDecodeRegs = 72;
static_assert(256 * (kSoftmaxRegs + kDecodeRegs) <= 65536, "register shares");
constexpr int kSmemBytes = kQBytes + kSlots * kSlotBytes + 1024 /* alignment */;
constexpr int kTmemCols = 512;                // S0 S1 O0 O1, 128 columns each
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kPScaleLog2 = 6.f;            // weights up to 2^(6 + 8)
constexpr float kMove = 8.f;                  // the reference moves when a maximum exceeds it by this

// tcgen05 instruction descriptor: D f32, A and B f16, M = N = 128; V is MN-major (bit 16)
constexpr uint32_t kIdescQK = (1u << 4) | ((uint32_t)(kKeys >> 3) << 17) | ((uint32_t)(kRows >> 4) << 24);
constexpr uint32_t kIdescPV = kIdescQK | (1u << 16);

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

__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t accum) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(da), "l"(db), "r"(idesc), "r"(accum));
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t db, uint32_t idesc, uint32_t accum) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(db), "r"(idesc), "r"(accum));
}
__device__ __forceinline__ void mma_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
               : "memory");
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

// Pairs of floats in one 64-bit register: one instruction for two.
__device__ __forceinline__ uint64_t f32x2(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ void unpack2(uint64_t v, float& x, float& y) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
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

// The codes of one thread's part of a K or V tile: rows lane / 4 + 8 i of its warp's 32 keys,
// elements 32 (lane % 4) .. + 32 of each.
struct Codes {
  uint4 c[4];
  uint32_t s[4];  // two scale bytes
};

__global__ void __launch_bounds__(kThreads, 1) prefill_fp4_kernel(const __grid_constant__ PrefillArgs a) {
  extern __shared__ __align__(16) unsigned char smem_raw[];
  __shared__ uint64_t q_full[2], full[kSlots], empty[kSlots], s_full[2], p_ready[2], pv_done[2];
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

  if (warp == kMmaWarp) {
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
      for (int i = 0; i < kSlots; ++i) {
        mbar_init(&full[i], 4);
        mbar_init(&empty[i], 1);
      }
      for (int i = 0; i < 2; ++i) {
        mbar_init(&q_full[i], 128);
        mbar_init(&s_full[i], 1);
        mbar_init(&p_ready[i], 128);
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
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
    const int t = warp >> 2;                                  // tile
    const int row = (warp & 3) * 32 + lane;                   // TMEM lane
    const int tt = t * tpt + row / G, h = row % G;            // token of the CTA, head of the group
    const bool valid = row < tpt * G && tt < n_tok;
    const int lim = valid ? min(prefix + item.tok0 + tt, kv_len - 1) : -1;  // last visible key
    if (t < tiles) {
      // Q: 16 lanes a row
      const int tw = threadIdx.x & 127;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int r = (tw >> 4) + 8 * i, ch = tw & 15;
        const int rt = t * tpt + r / G;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (r < tpt * G && rt < n_tok)
          v = *reinterpret_cast<const uint4*>(a.q + (int64_t)(q_start + item.tok0 + rt) * a.q_ts +
                                              (kvh * G + r % G) * kD + ch * 8);
        *reinterpret_cast<uint4*>(s_q + (t * 2 + (ch >> 3)) * kHalf + r * 128 + (((ch & 7) ^ (r & 7)) << 4)) = v;
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      mbar_arrive(&q_full[t]);

      const uint32_t lane_base = tmem + ((uint32_t)((warp & 3) * 32) << 16);
      const uint32_t s_addr = lane_base + t * 128, o_addr = lane_base + 256 + t * 128;
      int low = lim;  // smallest limit of the warp: tiles below it need no mask
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) low = min(low, __shfl_xor_sync(0xffffffffu, low, o));
      float m = -INFINITY, l = 0.f;  // reference (log2 units, less kPScaleLog2) and sum
      bool ok = true;
      for (int j = 0; j < n_kv; ++j) {
        if (!mbar_wait(&s_full[t], j & 1)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const int kbase = j * kKeys;
        uint32_t seen[4];  // visible keys of the tile, a bit each
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int k0 = kbase + 32 * c, n = lim - k0 + 1;
          seen[c] = n >= 32 ? 0xffffffffu : (n <= 0 ? 0u : (1u << n) - 1u);
        }
        bool masked = kbase + kKeys - 1 > low;
        if (*reinterpret_cast<volatile int*>(&s_bad) != 0) {  // rare: leave out the keys of bad pages
          for (int c = 0; c < 4; ++c) {
            const int pg = (kbase + 32 * c) / a.block_size;
            const int64_t blk = pg < a.max_blocks ? table[pg] : -1;
            if (blk < 0 || blk >= a.num_blocks) seen[c] = 0;
          }
          masked = true;
        }
        // ---- the row's 128 scores, and their maximum --------------------------------------------
        float v[4][32];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld32(s_addr + 32 * c, v[c]);
        tmem_ld_wait();
        if (masked) {
#pragma unroll
          for (int c = 0; c < 4; ++c) hide(v[c], seen[c]);
        }
        const float mx = max32(v[3], max32(v[2], max32(v[1], max32(v[0], -INFINITY)))) * a.scale_log2;
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
        for (int c = 0; c < 4; ++c) {
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
        {
          float x0, x1;
          unpack2(add2(sum[0], sum[1]), x0, x1);
          l += x0 + x1;
        }
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(&p_ready[t]);
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
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kDecodeRegs));
    if (warp < kMmaWarp) {
    // ------------------------------------------------------------------ decode of K and V
    const int lr = lane >> 2, lc = lane & 3;
    // unit u: 32 keys (u % 4) of slot number n = u / 4, which is K (n even) or V (odd) of tile n / 2
    auto fetch = [&](int u, Codes& x, bool& live) {
      const int n = u >> 2, k0 = (n >> 1) * kKeys + (u & 3) * 32;
      const int page = a.bs_log2 >= 0 ? k0 >> a.bs_log2 : k0 / a.block_size;
      const int64_t blk = k0 < n_keys && page < a.max_blocks ? __ldg(table + page) : -1;
      live = blk >= 0 && blk < a.num_blocks;
      if (!live) {
        if (k0 < n_keys) {
          set_device_status(kStatusBadPage);
          s_bad = 1;
        }
        return;
      }
      const int64_t r0 = (blk * a.Hkv + kvh) * a.block_size + (k0 - page * a.block_size) + lr;
      const uint8_t* codes = ((n & 1) ? a.vc : a.kc) + r0 * kFp4RowBytes + lc * 16;
      const uint8_t* scales = ((n & 1) ? a.vs : a.ks) + r0 * kFp4ScaleBytes + lc * 2;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x.c[i] = __ldg(reinterpret_cast<const uint4*>(codes + i * 8 * kFp4RowBytes));
        x.s[i] = __ldg(reinterpret_cast<const uint16_t*>(scales + i * 8 * kFp4ScaleBytes));
      }
    };
    Codes cur;
    bool cur_live = false;
    const int total = 8 * n_kv;
    // A warp does not write every slot, so it may skip a use of one: it waits by parity all the
    // same, because its previous unit lay at most two slots back and waited for a release that
    // comes after the one before last of this slot.
    static_assert(kDecodeWarps <= 8 && kSlots > 2, "a warp's units are at most two slots apart");
    for (int u = warp - 8; u < total; u += kDecodeWarps) {
      fetch(u, cur, cur_live);
      const int n = u >> 2, slot = n % kSlots;
      if (!mbar_wait(&empty[slot], ((n / kSlots) & 1) ^ 1)) break;
      unsigned char* dst = s_kv + slot * kSlotBytes + (lc >> 1) * kHalf;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = (u & 3) * 32 + lr + 8 * i;  // key of the tile
        const int key = (n >> 1) * kKeys + r;
        uint32_t s = cur.s[i];
        bool zero = !cur_live || key >= n_keys;
        if ((n & 1) && !zero) {  // V: no NaN (or infinity) reaches the product
          if ((s & 0xFFu) >= 248u) {
            atomicMin(&s_nan[2 * lc], key);
            s &= 0xFF00u;
          }
          if ((s >> 8) >= 248u) {
            atomicMin(&s_nan[2 * lc + 1], key);
            s &= 0xFFu;
          }
        }
        const uint32_t f[2] = {fp4_scale_h2(s & 0xFFu), fp4_scale_h2(s >> 8)};
        const uint32_t cw[4] = {cur.c[i].x, cur.c[i].y, cur.c[i].z, cur.c[i].w};
        uint4 o[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          uint32_t e[4];
          fp4x8_to_f16x2(cw[k], e);
          o[k] = make_uint4(h2_mul(e[0], f[k >> 1]), h2_mul(e[1], f[k >> 1]), h2_mul(e[2], f[k >> 1]),
                            h2_mul(e[3], f[k >> 1]));
          if (zero) o[k] = make_uint4(0, 0, 0, 0);
        }
        // 16-byte chunk 4 (lc % 2) + k of the row, swizzled; lanes of the second half take the
        // chunks in the order 2 3 0 1, so that 8 lanes always hit 8 different chunk positions
        const bool second = lc >= 2;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint4 val = second ? o[k ^ 2] : o[k];
          const int ch = (lc & 1) * 4 + (second ? k ^ 2 : k);
          *reinterpret_cast<uint4*>(dst + r * 128 + ((ch ^ (r & 7)) << 4)) = val;
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
    if (lane == 0 && n_kv > 0) {
      const uint32_t kv0 = smem_u32(s_kv), q0 = smem_u32(s_q);
      bool ok = true;
      auto scores = [&](int t, int n) {  // S_t = Q_t K^T, K in slot number n
        const uint64_t dq = desc_base(q0 + t * 2 * kHalf, 16), dk = desc_base(kv0 + (n % kSlots) * kSlotBytes, 16);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const uint64_t off = (uint64_t)(((k >> 2) * kHalf + (k & 3) * 32) >> 4);
          mma_ss(tmem + t * 128, dq + off, dk + off, kIdescQK, k > 0);
        }
        mma_commit(&s_full[t]);
      };
      auto release = [&](int n) {  // nobody waits for the last slots: no arrival may outlive the CTA
        if (n + kSlots < 2 * n_kv) mma_commit(&empty[n % kSlots]);
      };
      auto wait_full = [&](int n) { return mbar_wait(&full[n % kSlots], (n / kSlots) & 1); };
      for (int t = 0; t < tiles && ok; ++t) ok = mbar_wait(&q_full[t], 0);
      ok = ok && wait_full(0);
      if (ok) {
        tc_fence_after();
        for (int t = 0; t < tiles; ++t) scores(t, 0);
        release(0);
      }
      for (int j = 0; ok && j < n_kv; ++j) {
        const int nv = 2 * j + 1, nk = 2 * j + 2;
        const bool more = j + 1 < n_kv;
        ok = wait_full(nv) && (!more || wait_full(nk));
        for (int t = 0; ok && t < tiles; ++t) {
          ok = mbar_wait(&p_ready[t], j & 1);
          if (!ok) break;
          tc_fence_after();
          const uint64_t dv = desc_base(kv0 + (nv % kSlots) * kSlotBytes, kHalf);
#pragma unroll
          for (int k = 0; k < 8; ++k)  // 16 keys each
            mma_ts(tmem + 256 + t * 128, tmem + t * 128 + 8 * k, dv + (uint64_t)((k * 2048) >> 4), kIdescPV,
                   j > 0 || k > 0);
          mma_commit(&pv_done[t]);
          if (more) scores(t, nk);
        }
        if (ok) {
          release(nv);
          if (more) release(nk);
        }
      }
    }
    __syncwarp();
    role_sync();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
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
