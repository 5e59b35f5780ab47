// Causal chunk-prefill attention over the paged 4-bit KV cache (format: fp4_kv.cuh), any
// number of sequences: sequence s has queries q[cu_q[s] .. cu_q[s + 1]) at positions
// kv_lens[s] - q_len + i, each attending to the cached keys up to its own position.
//
// Tensor bound (4 * 128 * Hq operations per visible pair), so both products run on tcgen05
// with fp32 accumulators in TMEM. An item is two tiles of 128 query rows of one kv head, a row
// being a (token, query head) pair of the G = Hq / Hkv heads that share it, over steps of 64
// keys that both tiles read. The steps of all items (sequence, block of tokens, kv head) form
// one list that is dealt evenly to one CTA per SM, whatever the lengths are; an item that
// crosses CTAs leaves fp32 partials (O, reference, sum) in the workspace, joined by a second kernel.
// 2048 queries behind 30720 tokens (32 / 8 heads) take 1001 us, 1064 TFLOP/s of visible pairs.
// The roles below walk a CTA's items on their own, so decoding runs ahead into the next one.
//   warps 0-3, 4-7   softmax of tile 0 / 1: a thread owns a row. It reads its 64 scores of a
//                    step from TMEM, writes the weights over them as f16, and keeps the row's
//                    maximum and sum (fp32). Its registers are full, so an item's numbers come
//                    from shared memory where they are needed (kept in registers: 1141 us).
//   warps 8-13       decode K and V codes to f16 in shared memory (128-byte swizzle), a
//                    ring of kSlots 16 KB slots in the order K0 V0 K1 V1 ..., a warp a slot:
//                    the fence between its stores and the tensor core's reads and the
//                    barriers cost as much as 16 keys' work.
//   warps 14, 15     each walks the items of one tile, fetches Q by TMA, and issues S = Q K^T (both
//                    in shared memory, K-major) and O += P V (P from TMEM, V as it lies in the cache:
//                    MN-major). One warp for both tiles spends 1.6 thousand cycles a step on waits and
//                    issue, the tensor core needs 1.24. The next item's Q and first scores are made
//                    under the last product and the output of the one at hand. Warp 15 allocates TMEM.
// The scores are double-buffered (TMEM: two tiles x two S of 64 columns, two O of 128), so S of
// the next step is there when a softmax ends and the chain S -> softmax -> P V of a tile never
// stalls its softmax warps: with one S a tile (128 keys a step, or 64 and Q in TMEM) the
// chain's latencies show, 4 and 16 % more time.
// Softmax in the exp2 domain against a lazy reference: weights are 2^(s - m) for a reference
// m that moves, with a rescale of O in TMEM, only when a row's maximum exceeds it by 8 or
// more. Weights are rounded to f16 for the second product (2^-11 relative, 2^-31 of the largest
// where they are subnormal; the first rounding below fp32 in the kernel, K and V are exact), the
// row sums take them unrounded. Rows whose scores are too far from zero for that form (4 million and more) are done once
// more at the end, from differences of scores (far_rows).
//
// V rows behind an item's last key and rows of bad pages are written as zeros, and a NaN group
// of V as zeros too, because a zero weight does not hide a NaN from the product; where one was
// met, the first key with a NaN is looked up per 16 elements at the end of the item, and the rows
// that see it get NaN.
#include "fp4_kv.cuh"
#include "kernels.h"
#include "tensor_map.h"

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

__device__ __forceinline__ void tmem_ld16(uint32_t addr, float (&v)[16]) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(addr));
}

__device__ __forceinline__ void tma_load_3d(const CUtensorMap* map, uint32_t dst, uint64_t* bar, int c0, int c1,
                                            int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::
          "r"(dst),
      "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(smem_u32(bar))
      : "memory");
}
// Lanes 4 i .. 4 i + 3 hold a row each, as four pieces of 16 bytes: afterwards lane 4 i + k has piece k of all four.
__device__ __forceinline__ void transpose4(uint32_t (&p)[16]) {
#pragma unroll
  for (int b = 1; b <= 2; b <<= 1) {
    const bool up = threadIdx.x & b;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (j & b) continue;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        uint32_t &lo = p[4 * j + w], &hi = p[4 * (j ^ b) + w];
        const uint32_t got = __shfl_xor_sync(0xffffffffu, up ? lo : hi, b);
        lo = up ? got : lo;
        hi = up ? hi : got;
      }
    }
  }
}

// mbar_wait by a whole warp, with one answer (lanes may run out of time at different moments).
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t phase) {
  return __all_sync(0xffffffffu, mbar_wait(bar, phase)) != 0;
}

struct PrefillArgs {
  const __half* q;  // [T, Hq, D], token stride q_ts elements (read by TMA but for far scores)
  int64_t q_ts;
  const uint8_t *kc, *vc, *ks, *vs;
  int64_t num_blocks;
  const int32_t* tables;  // [S, max_blocks]
  const int32_t* cu_q;    // [S + 1]
  const int32_t* kv_lens;
  __half* out;       // [T, Hq, D]
  int4* open_items;  // workspace: per CTA, the item that it leaves open: CTAs it goes on in, seq, block, kv head
  float* ws;         // workspace: [CTAs][2] partials of kPartFloats: O, and the reference (a score) and sum of each row
  int num_seqs, total_q, Hkv, G, tok, block_size, bs_log2, max_blocks;  // tok: query tokens of an item, 2 (128 / G)
  int inv_g;  // r / G = r * inv_g >> 16 for rows r of a tile
  int cap;  // tokens that a table row can hold
  float scale_log2;
};

// The list is dealt in units of a step's time; an item's output or partial and its first softmax, in which the
// tensor core idles, count as kItemUnits more in front of its steps. (Without them the CTAs with the shortest items end
// last: half as much time again for a ragged batch.)
constexpr int kItemUnits = 4;
// Units of a CTA at least: the join costs less than a step or two. Two tails of 8 queries on 500 tokens take 13.3 us
// with 3, 13.9 with 4, 12.8 with 2; one on 2400 takes 15.8 with 3 and 4, 16.6 with 2.
constexpr int kMinShare = 3;
constexpr int kPartRows = 2 * kRows;
constexpr int kPartFloats = kPartRows * (kD + 2);  // O as [32 x 4 elements][row][4], then (reference, sum) per row

struct Seq {
  int q_start, q_len, kv_len, prefix, blocks;  // prefix: position of the first query
};
__device__ __forceinline__ Seq seq_of(const PrefillArgs& a, int s) {
  Seq q;
  q.q_start = min(max(a.cu_q[s], 0), a.total_q);
  q.q_len = max(min(a.cu_q[s + 1], a.total_q) - q.q_start, 0);
  const int kv = a.kv_lens[s];
  q.prefix = kv - q.q_len;
  q.kv_len = min(kv, a.cap);
  q.blocks = (q.q_len + a.tok - 1) / a.tok;
  return q;
}
// Keys that block b of a sequence sees, and its steps (one even without keys: its rows become zeros).
__device__ __forceinline__ int keys_of(const PrefillArgs& a, const Seq& q, int b) {
  return max(0, min(q.kv_len, q.prefix + min((b + 1) * a.tok, q.q_len)));
}
__device__ __forceinline__ int steps_of(int keys) { return max(1, (keys + kKeys - 1) / kKeys); }

// Place in the CTA's list: item (s, b, h) of `steps` steps begins at unit `start` of the CTA's `count` (negative: in an
// earlier CTA). [j0, j1): its steps of this CTA, none if only units in front of them are; j0 is the CTA's step `first`.
struct Cursor {
  int s, b, h, steps, keys, start, j0, j1, first;
  Seq q;
  __device__ __forceinline__ void own_steps(int count) {
    j0 = max(0, -start - kItemUnits);
    j1 = max(j0, min(steps, count - start - kItemUnits));
  }
  __device__ __forceinline__ int end() const { return start + kItemUnits + steps; }
  // to the next item with steps of this CTA; false: there is none
  __device__ __forceinline__ bool next_item(const PrefillArgs& a, int count) {
    start = end();
    first += j1 - j0;
    if (start + kItemUnits >= count) return false;
    if (++h == a.Hkv) {
      h = 0;
      ++b;
      while (b >= q.blocks) {
        b = 0;
        if (++s >= a.num_seqs) return false;  // only if the lengths changed meanwhile
        q = seq_of(a, s);
      }
      keys = keys_of(a, q, b);
      steps = steps_of(keys);
    }
    own_steps(count);
    return true;
  }
};

// What a tile's softmax warps need to know of an item; written by the warp that issues the tile's products.
struct Item {
  int seq, kvh, q0, n_tok;         // q0: row of q of the item's first token, n_tok: its tokens
  int pos, kv_len, key_end;        // pos: position of the first token, key_end: end of the keys of this CTA's steps
  int j0, j1, whole;               // this CTA's steps, and whether they are all of them
};

// The 16-element groups in which V has a NaN among keys [k0, k1) up to `lim` of the calling lane's row, a
// bit each. A warp; rare, so it simply reads the scales again.
__device__ __noinline__ uint32_t nan_groups(const PrefillArgs& a, int seq, int kvh, int k0, int k1, int lim) {
  int first[8];
#pragma unroll
  for (int g = 0; g < 8; ++g) first[g] = INT32_MAX;
  for (int k = k0 + (int)(threadIdx.x & 31); k < k1; k += 32) {
    const int pg = k / a.block_size;
    const int64_t blk = pg < a.max_blocks ? a.tables[(int64_t)seq * a.max_blocks + pg] : -1;
    if (blk < 0 || blk >= a.num_blocks) continue;
    const uint8_t* sp = a.vs + ((blk * a.Hkv + kvh) * a.block_size + (k - pg * a.block_size)) * kFp4ScaleBytes;
#pragma unroll
    for (int g = 0; g < 8; ++g)
      if (sp[g] >= 248) first[g] = min(first[g], k);
  }
  __syncwarp();
  uint32_t bits = 0;
#pragma unroll
  for (int g = 0; g < 8; ++g) bits |= __reduce_min_sync(0xffffffffu, first[g]) <= lim ? 1u << g : 0u;
  return bits;
}

__device__ __forceinline__ int warp_scan(int v) {  // inclusive
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += up;
  }
  return v;
}

// Units of one kv head in sequence s0 + lane (a whole warp: long sequences are shared by its lanes).
__device__ __forceinline__ int seq_units(const PrefillArgs& a, int s0) {
  const int lane = threadIdx.x & 31;
  const bool in = s0 + lane < a.num_seqs;
  const Seq q = in ? seq_of(a, s0 + lane) : Seq{0, 0, 0, 0, 0};
  if (in && q.kv_len < a.kv_lens[s0 + lane]) set_device_status(kStatusBadPage);
  int mine = 0;
  constexpr int kOwn = 4;
  if (q.blocks <= kOwn)
    for (int b = 0; b < q.blocks; ++b) mine += kItemUnits + steps_of(keys_of(a, q, b));
  uint32_t longer = __ballot_sync(0xffffffffu, q.blocks > kOwn);
  while (longer != 0) {
    const int l = __ffs(longer) - 1;
    longer &= longer - 1;
    const Seq o{0, __shfl_sync(0xffffffffu, q.q_len, l), __shfl_sync(0xffffffffu, q.kv_len, l),
                __shfl_sync(0xffffffffu, q.prefix, l), __shfl_sync(0xffffffffu, q.blocks, l)};
    int part = 0;
    for (int b = lane; b < o.blocks; b += 32) part += kItemUnits + steps_of(keys_of(a, o, b));
    part = __shfl_sync(0xffffffffu, warp_scan(part), 31);
    if (lane == l) mine = part;
  }
  return mine;
}

// This CTA's share of the list: its units (0: no steps), its first item, and the share of every CTA. A warp.
__device__ __forceinline__ int find_share(const PrefillArgs& a, Cursor& c, int64_t& share) {
  const int lane = threadIdx.x & 31;
  int64_t total = 0;
  int last = 0;  // this lane's sequence of the last 32
  for (int s0 = 0; s0 < a.num_seqs; s0 += 32) {
    last = seq_units(a, s0);
    total += (int64_t)__shfl_sync(0xffffffffu, warp_scan(last), 31) * a.Hkv;
  }
  const int64_t even = (total + gridDim.x - 1) / gridDim.x;
  share = even > kMinShare ? even : kMinShare;
  const int64_t begin = (int64_t)blockIdx.x * share;
  if (begin >= total) return 0;
  int64_t at = 0;  // units before sequence s0
  int s0 = 0;
  for (;; s0 += 32) {
    if (s0 >= a.num_seqs) return 0;  // only if the lengths changed meanwhile
    const int mine = a.num_seqs <= 32 ? last : seq_units(a, s0);
    const int inc = warp_scan(mine);
    const int64_t end = at + (int64_t)inc * a.Hkv;
    const uint32_t hit = __ballot_sync(0xffffffffu, begin < end);
    if (hit == 0) {
      at = __shfl_sync(0xffffffffu, end, 31);
      continue;
    }
    const int l = __ffs(hit) - 1;
    at += (int64_t)__shfl_sync(0xffffffffu, inc - mine, l) * a.Hkv;
    c.s = s0 + l;
    break;
  }
  if (c.s >= a.num_seqs) return 0;
  c.q = seq_of(a, c.s);
  for (int b0 = 0;; b0 += 32) {
    const int keys = b0 + lane < c.q.blocks ? keys_of(a, c.q, b0 + lane) : 0;
    const int mine = b0 + lane < c.q.blocks ? kItemUnits + steps_of(keys) : 0;
    const int inc = warp_scan(mine);
    const uint32_t hit = __ballot_sync(0xffffffffu, begin < at + (int64_t)inc * a.Hkv);
    if (hit == 0) {
      if (b0 + 32 >= c.q.blocks) return 0;  // as above
      at += (int64_t)__shfl_sync(0xffffffffu, inc, 31) * a.Hkv;
      continue;
    }
    const int l = __ffs(hit) - 1;
    at += (int64_t)__shfl_sync(0xffffffffu, inc - mine, l) * a.Hkv;
    c.b = b0 + l;
    c.steps = max(__shfl_sync(0xffffffffu, mine, l) - kItemUnits, 1);
    c.keys = __shfl_sync(0xffffffffu, keys, l);
    break;
  }
  const int off = (int)(begin - at), units = kItemUnits + c.steps;
  c.h = off / units;
  c.start = -(off - c.h * units);
  const int count = (int)(total - begin < share ? total - begin : share);
  c.own_steps(count);
  return c.j0 < c.j1 || c.next_item(a, count) ? count : 0;
}

// Outputs and partials once more where scores are so far from zero that the rounding of s c - (r c - b) would decide their
// weights (far_score; from 2^27 on in the log2 domain weights would leave f16's range): the rows of the softmax warps that
// met such a reference, in all items of the CTA, from differences of scores and in fp32. All warps, when the roles have
// ended: a call inside the softmax loop cost 2 % there (and the cursor passed by value 1.5 % of a ragged batch). A warp has
// a row, four keys at a time. Rare, so simple: 2048 queries on 32768 keys (32 / 8 heads), every row far, take 290 ms.
__device__ __noinline__ void far_rows(const PrefillArgs& a, const Cursor* first, int count, const int* far) {
  Cursor c = *first;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, tpt = kRows / a.G;
  auto values = [&](const uint8_t* codes, const uint8_t* scales, int64_t r, float (&x)[4]) {  // elements 4 lane ..
    uint32_t o[4];
    fp4x8_to_f16x2(*reinterpret_cast<const uint32_t*>(codes + r * kFp4RowBytes + (lane >> 1) * 4), o);
    const uint32_t f = fp4_scale_h2(scales[r * kFp4ScaleBytes + (lane >> 2)]);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t w = h2_mul(lane & 1 ? o[2 + i] : o[i], f);
      __half2 h;
      memcpy(&h, &w, 4);
      const float2 p = __half22float2(h);
      x[2 * i] = p.x;
      x[2 * i + 1] = p.y;
    }
  };
  for (bool more = count > 0; more; more = c.next_item(a, count)) {
    const int tok0 = c.b * a.tok, n_tok = min(a.tok, c.q.q_len - tok0), key_end = min(c.j1 * kKeys, c.keys);
    for (int pr = warp; pr < kPartRows; pr += kThreads / 32) {
      const int t = pr / kRows, row = pr % kRows, rt = row / a.G, tt = t * tpt + rt;
      if (far[pr / 32] == 0 || rt >= tpt || tt >= n_tok) continue;
      const int head = c.h * a.G + row - rt * a.G, tok = c.q.q_start + tok0 + tt;
      const int end = min(min(c.q.prefix + tok0 + tt, c.q.kv_len - 1) + 1, key_end);
      float q[4], m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int e = 0; e < 4; ++e) q[e] = __half2float(a.q[tok * a.q_ts + head * kD + 4 * lane + e]);
      for (int k = c.j0 * kKeys; k < end; k += 4) {  // four keys lie in one page
        const int pg = k / a.block_size;
        const int64_t blk = pg < a.max_blocks ? a.tables[(int64_t)c.s * a.max_blocks + pg] : -1;
        if (blk < 0 || blk >= a.num_blocks) continue;
        const int64_t r = (blk * a.Hkv + c.h) * a.block_size + (k - pg * a.block_size);
        float s[4], v[4][4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          float x[4];
          values(a.kc, a.ks, r + u, x);
          values(a.vc, a.vs, r + u, v[u]);
          s[u] = q[0] * x[0] + q[1] * x[1] + q[2] * x[2] + q[3] * x[3];
        }
#pragma unroll
        for (int d = 16; d > 0; d >>= 1)
#pragma unroll
          for (int u = 0; u < 4; ++u) s[u] += __shfl_xor_sync(0xffffffffu, s[u], d);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          if (k + u >= end) break;
          const float mn = fmaxf(m, s[u]);
          const float w0 = m == -INFINITY ? 1.f : ex2((m - mn) * a.scale_log2);
          // (a reference that is not far: as everywhere else, so that partials with the same one fit together)
          const float w = ex2(far_score(mn, a.scale_log2)
                                  ? fmaf(s[u] - mn, a.scale_log2, kPScaleLog2)
                                  : fmaf(s[u], a.scale_log2, fmaf(-mn, a.scale_log2, kPScaleLog2)));
          m = mn;
          l = l * w0 + w;
#pragma unroll
          for (int e = 0; e < 4; ++e) o[e] = o[e] * w0 + w * v[u][e];
        }
      }
      if (c.j0 == 0 && c.j1 == c.steps) {
        const float f = l == 0.f ? 0.f : 1.f / l;
        *reinterpret_cast<uint2*>(a.out + ((int64_t)tok * a.Hkv * a.G + head) * kD + 4 * lane) =
            make_uint2(pack_h2(o[0] * f, o[1] * f), pack_h2(o[2] * f, o[3] * f));
      } else {
        float* part = a.ws + ((int64_t)blockIdx.x * 2 + (c.j0 > 0 ? 0 : 1)) * kPartFloats;
        *reinterpret_cast<float4*>(part + (lane * kPartRows + pr) * 4) = make_float4(o[0], o[1], o[2], o[3]);
        if (lane == 0) *reinterpret_cast<float2*>(part + kPartRows * kD + pr * 2) = make_float2(m, l);
      }
    }
  }
}

__global__ void __launch_bounds__(kThreads, 1)
    prefill_fp4_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ PrefillArgs a) {
  extern __shared__ __align__(16) unsigned char smem_raw[];
  __shared__ uint64_t q_full[2], full[kSlots], empty[kSlots], s_full[2][2], p_ready[2][2], pv_done[2][2], item_full[2];
  __shared__ Item s_item[2][2];  // per tile, the item at hand and the one behind it
  __shared__ uint32_t s_tmem;
  __shared__ Cursor s_first;
  __shared__ int s_count;
  __shared__ int64_t s_share;
  __shared__ int s_seen_nan;  // a V group with a NaN was decoded
  __shared__ int s_bad;       // a page outside the cache was met
  __shared__ int s_far[8];    // per softmax warp: a row had a far score as its reference
  unsigned char* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  unsigned char* s_q = smem;
  unsigned char* s_kv = smem + kQBytes;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_wait();
  pdl_trigger();
  const int G = a.G, tpt = kRows / G;  // tokens per tile

  if (threadIdx.x == 0) a.open_items[blockIdx.x] = make_int4(0, 0, 0, 0);  // rewritten below where one is left
  if (warp == kMmaWarp) {
    Cursor c = {};
    int64_t share;
    const int count = find_share(a, c, share);
    if (lane == 0) {
      s_first = c;
      s_count = count;
      s_share = share;
      s_bad = 0;
      s_seen_nan = 0;
    }
    if (lane < 8) s_far[lane] = 0;
  }
  if (warp == kMmaWarp + 1) {
    if (lane == 0) {
      for (int i = 0; i < kSlots; ++i) {
        mbar_init(&full[i], 1);
        mbar_init(&empty[i], 2);  // both tiles' warps are done with the slot
      }
      for (int i = 0; i < 2; ++i) {
        mbar_init(&q_full[i], 1);
        mbar_init(&item_full[i], 1);
        for (int h = 0; h < 2; ++h) {  // the steps' parities
          mbar_init(&s_full[i][h], 1);
          mbar_init(&p_ready[i][h], 128);
          mbar_init(&pv_done[i][h], 1);
        }
      }
      fence_barrier_init();
    }
    __syncwarp();
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)),
                 "r"(kTmemCols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;
  const int count = s_count;
  Cursor cu = s_first;

  if (warp < 8) {
    // ------------------------------------------------------------------ softmax
    const int t = warp >> 2;                        // tile
    const int row = (warp & 3) * 32 + lane;         // TMEM lane
    const int tt = t * tpt + ((row * a.inv_g) >> 16);  // token of the item
    const uint32_t lane_base = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t o_addr = lane_base + kColO + t * kD;
    int js = 0;  // steps of this tile so far: the barriers' phases
    for (int it = 0; warp_wait(&item_full[t], it & 1); ++it) {
      // read where it is needed: the loop over the steps has no registers to spare
      const volatile Item& item = s_item[t][it & 1];
      const int j0 = item.j0, j1 = item.j1;
      if (j0 == j1) break;  // behind the last item
      const int lim = row < tpt * G && tt < item.n_tok ? min(item.pos + tt, item.kv_len - 1) : -1;  // last visible key
      int low = lim;  // smallest limit of the warp: steps below it need no mask
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) low = min(low, __shfl_xor_sync(0xffffffffu, low, o));
      float m = -INFINITY, l = 0.f;  // reference (a score) and sum
      bool ok = true;
      for (int j = j0; j < j1; ++j, ++js) {
        ok = warp_wait(&s_full[t][js & 1], (js >> 1) & 1);
        if (!ok) break;
        tc_fence_after();
        const int kbase = j * kKeys;
        const uint32_t s_addr = lane_base + t * 128 + (js & 1) * kKeys;
        const bool bad = *reinterpret_cast<volatile int*>(&s_bad) != 0;
        // ---- the row's 64 scores, and their maximum ---------------------------------------------
        float v[2][32];
#pragma unroll
        for (int c = 0; c < 2; ++c) tmem_ld32(s_addr + 32 * c, v[c]);
        tmem_ld_wait();
        if (kbase + kKeys - 1 > low || bad) {
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const int k0 = kbase + 32 * c, n = lim - k0 + 1;  // keys of these 32 that the row sees
            uint32_t seen = n >= 32 ? 0xffffffffu : (n <= 0 ? 0u : (1u << n) - 1u);
            if (bad) {  // rare: leave out the keys of bad pages
              const int pg = k0 / a.block_size;
              const int64_t blk = pg < a.max_blocks ? a.tables[(int64_t)item.seq * a.max_blocks + pg] : -1;
              if (blk < 0 || blk >= a.num_blocks) seen = 0;
            }
            hide(v[c], seen);
          }
        }
        const float mx = max32(v[1], max32(v[0], -INFINITY));
        // ---- the reference moves when some row's maximum is far above it (or the first one) --------
        const bool far = (mx - m) * a.scale_log2 > kMove;
        if (__any_sync(0xffffffffu, far)) {
          const float mn = far ? mx : m;
          const float al = m == -INFINITY ? 1.f : ex2((m - mn) * a.scale_log2);
          m = mn;
          l *= al;
          if (far_score(m, a.scale_log2)) s_far[warp] = 1;
          if (j > j0) {
            // S of this step was issued behind the product of step js - 2, so the phase of this barrier before
            // the awaited one is over
            ok = warp_wait(&pv_done[t][(js - 1) & 1], ((js - 1) >> 1) & 1);
            if (!ok) break;
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
        const float neg = m == -INFINITY ? 0.f : fmaf(-m, a.scale_log2, kPScaleLog2);
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
        mbar_arrive(&p_ready[t][js & 1]);
        float x0, x1;
        unpack2(add2(sum[0], sum[1]), x0, x1);
        l += x0 + x1;
      }
      if (!ok) break;
      // The last product. S of its step was issued before the product of step js - 2, which may still run,
      // hence a barrier per parity of steps: one for both could not tell the two by its phase.
      ok = warp_wait(&pv_done[t][(js - 1) & 1], ((js - 1) >> 1) & 1);
      if (!ok) break;
      tc_fence_after();
      // ---- the item's steps of this CTA are done: O / l, or a partial ------------------------------
      uint32_t nan = 0;  // 16-element groups in which this row sees a NaN of V
      if (__any_sync(0xffffffffu, *reinterpret_cast<volatile int*>(&s_seen_nan) != 0))
        nan = nan_groups(a, item.seq, item.kvh, item.j0 * kKeys, item.key_end, lim);
      const float qnan = __int_as_float(0x7fffffff);
      if (item.whole) {
        const float inv = l == 0.f ? 0.f : 1.f / l;
        // four lanes store 64 bytes of a row: 8 lines an instruction, where a row a lane would take 32
        const int n_tok = item.n_tok, q0 = item.q0, kvh = item.kvh;
        __half* dst[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = (row & ~3) + i, rt = (r * a.inv_g) >> 16, tok = t * tpt + rt;
          dst[i] = rt < tpt && tok < n_tok
                       ? a.out + ((((int64_t)(q0 + tok) * a.Hkv + kvh) * G + (r - rt * G)) * kD + (lane & 3) * 8)
                       : nullptr;
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          float o[32];
          uint32_t p[16];
          tmem_ld32(o_addr + 32 * c, o);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            const float f = (nan >> (2 * c + (i >> 4))) & 1u ? qnan : inv;
            p[i >> 1] = pack_h2(o[i] * f, o[i + 1] * f);
          }
          transpose4(p);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (dst[i] != nullptr)
              *reinterpret_cast<uint4*>(dst[i] + 32 * c) = make_uint4(p[4 * i], p[4 * i + 1], p[4 * i + 2], p[4 * i + 3]);
        }
      } else {  // slot 0: the item began in an earlier CTA; slot 1: it begins here and goes on
        float* part = a.ws + ((int64_t)blockIdx.x * 2 + (item.j0 > 0 ? 0 : 1)) * kPartFloats;
        const int pr = t * kRows + row;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          float o[32];
          tmem_ld32(o_addr + 32 * c, o);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            const float f = (nan >> (2 * c + (i >> 4))) & 1u ? qnan : 1.f;
            *reinterpret_cast<float4*>(part + ((8 * c + (i >> 2)) * kPartRows + pr) * 4) =
                make_float4(o[i] * f, o[i + 1] * f, o[i + 2] * f, o[i + 3] * f);
          }
        }
        *reinterpret_cast<float2*>(part + kPartRows * kD + pr * 2) = make_float2(m, l);
      }
      tc_fence_before();  // O is read before the next item's first product, which waits for p_ready
    }
  } else if (warp < kMmaWarp) {
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
    bool more = count > 0;
    for (int n = warp - 8;; n += kDecodeWarps) {  // K (n even) or V (odd) of the CTA's step n / 2
      while (more && (n >> 1) >= cu.first + cu.j1 - cu.j0) more = cu.next_item(a, count);
      if (!more) break;
      const int k0 = ((n >> 1) - cu.first + cu.j0) * kKeys;
      const int page = a.bs_log2 >= 0 ? k0 >> a.bs_log2 : k0 / a.block_size;
      const int64_t blk =
          k0 < cu.keys && page < a.max_blocks ? __ldg(a.tables + (int64_t)cu.s * a.max_blocks + page) : -1;
      const bool live = blk >= 0 && blk < a.num_blocks;
      uint4 codes[kKeys / 8];
      uint32_t sc[kKeys / 8];  // two scale bytes; 0: zeros, whatever the codes
      if (live) {
        const int64_t r0 = (blk * a.Hkv + cu.h) * a.block_size + (k0 - page * a.block_size) + lr;
        const uint8_t* cp = ((n & 1) ? a.vc : a.kc) + r0 * kFp4RowBytes + half * 32 + c2 * 16;
        const uint8_t* sp = ((n & 1) ? a.vs : a.ks) + r0 * kFp4ScaleBytes + half * 4 + c2 * 2;
#pragma unroll
        for (int i = 0; i < kKeys / 8; ++i) {
          codes[i] = __ldg(reinterpret_cast<const uint4*>(cp + i * 8 * kFp4RowBytes));
          sc[i] = __ldg(reinterpret_cast<const uint16_t*>(sp + i * 8 * kFp4ScaleBytes));
        }
        if (k0 + kKeys > cu.keys) {
#pragma unroll
          for (int i = 0; i < kKeys / 8; ++i)
            if (k0 + lr + 8 * i >= cu.keys) sc[i] = 0;
        }
      } else {
        if (k0 < cu.keys) {
          set_device_status(kStatusBadPage);
          s_bad = 1;
        }
#pragma unroll
        for (int i = 0; i < kKeys / 8; ++i) {
          codes[i] = make_uint4(0, 0, 0, 0);
          sc[i] = 0;
        }
      }
      const int slot = n % kSlots;
      if (!warp_wait(&empty[slot], ((n / kSlots) & 1) ^ 1)) break;
      unsigned char* dst = s_kv + slot * kSlotBytes;
#pragma unroll
      for (int i = 0; i < kKeys / 8; ++i) {
        uint32_t s = sc[i];
        if ((n & 1) && ((s & 0xF8u) == 0xF8u || (s & 0xF800u) == 0xF800u)) {
          // V: no NaN (or infinity) reaches the product
          s_seen_nan = 1;
          if ((s & 0xF8u) == 0xF8u) s &= 0xFF00u;
          if ((s & 0xF800u) == 0xF800u) s &= 0xFFu;
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
  } else {
    // ------------------------------------------------------------------ MMA issue
    // The whole warp walks the loop, so that descriptors and addresses stay in uniform registers, and
    // one lane's products and commits count: issued by one thread in a divergent branch, a product took
    // some 70 cycles to issue, more than to run.
    const int t = warp - kMmaWarp;  // tile
    const uint32_t lead = elect_one();
    const uint32_t kv0 = smem_u32(s_kv);
    const uint64_t dq = desc_base(smem_u32(s_q) + t * 2 * kQHalf, 16);
    auto scores = [&](int stage, int js) {  // S = Q K^T
      const uint64_t dk = desc_base(kv0 + stage * kSlotBytes, 16);
      const uint32_t d = tmem + t * 128 + (js & 1) * kKeys;
#pragma unroll
      for (int k = 0; k < 8; ++k)  // 16 elements each
        mma_ss(d, dq + (uint64_t)(((k >> 2) * kQHalf + (k & 3) * 32) >> 4),
               dk + (uint64_t)(((k >> 2) * kHalf + (k & 3) * 32) >> 4), kIdescQK, k > 0, lead);
      mma_commit(&s_full[t][js & 1], lead);
    };
    // the next K and the next V: slot of the ring, parity of its use
    struct Place {
      int stage, par;
    } k = {0, 0}, v = {1, 0};
    static_assert(kSlots % 2 == 0 && kSlots > 2, "K and V keep their parity of stages");
    auto release = [&](Place& p) {  // by a commit even without products: the warp's releases keep their order
      mma_commit(&empty[p.stage], lead);
      p.stage += 2;
      if (p.stage >= kSlots) {
        p.stage -= kSlots;
        p.par ^= 1;
      }
    };
    int js = 0, items = 0;
    bool ok = true;
    bool more = count > 0;
    while (more) {
      const int j0 = cu.j0, j1 = cu.j1, tok0 = cu.b * a.tok;
      const bool rows = t * tpt < cu.q.q_len - tok0;
      if (rows && lead) {
        if (t == 0 && j0 == 0 && j1 < cu.steps)
          a.open_items[blockIdx.x] = make_int4((int)((cu.end() - count + s_share - 1) / s_share), cu.s, cu.b, cu.h);
        // the buffer's last item was the one before the last: its softmax is over, since the last one's steps are
        s_item[t][items & 1] = Item{cu.s, cu.h, cu.q.q_start + tok0, min(a.tok, cu.q.q_len - tok0),
                                    cu.q.prefix + tok0, cu.q.kv_len, min(j1 * kKeys, cu.keys),
                                    j0, j1, j0 == 0 && j1 == cu.steps};
        mbar_arrive(&item_full[t]);
        // Q was last read for the scores whose weights have been waited for. The box has rows (token, head), also of
        // tokens behind the item's
        mbar_arrive_expect_tx(&q_full[t], 2 * tpt * G * 128);
        for (int i = 0; i < 2; ++i)
          tma_load_3d(&tmap_q, smem_u32(s_q) + (t * 2 + i) * kQHalf, &q_full[t], i * 64, cu.h * G,
                      cu.q.q_start + tok0 + t * tpt);
      }
      __syncwarp();
      more = cu.next_item(a, count);  // from here on `cu` is the next item
      if (!rows) {  // pass the slots on
        for (int j = j0; ok && j < j1; ++j) {
          ok = warp_wait(&full[k.stage], k.par);
          if (ok) release(k);
          ok = ok && warp_wait(&full[v.stage], v.par);
          if (ok) release(v);
        }
        if (!ok) break;
        continue;
      }
      ok = warp_wait(&q_full[t], items & 1) && warp_wait(&full[k.stage], k.par);
      if (!ok) break;
      ++items;
      tc_fence_after();
      scores(k.stage, js);
      release(k);
      for (int j = j0; j < j1; ++j, ++js) {
        if (j + 1 < j1) {
          // S of the next step: its buffer held the weights of step js - 1, whose product was issued before
          ok = warp_wait(&full[k.stage], k.par);
          if (!ok) break;
          tc_fence_after();
          scores(k.stage, js + 1);
          release(k);
        }
        ok = warp_wait(&full[v.stage], v.par) && warp_wait(&p_ready[t][js & 1], (js >> 1) & 1);
        if (!ok) break;
        tc_fence_after();
        const uint64_t dv = desc_base(kv0 + v.stage * kSlotBytes, kHalf);
        const uint32_t p = tmem + t * 128 + (js & 1) * kKeys;
#pragma unroll
        for (int i = 0; i < kKeys / 16; ++i)  // 16 keys each
          mma_ts(tmem + kColO + t * kD, p + 8 * i, dv + (uint64_t)((i * 2048) >> 4), kIdescPV, j > j0 || i > 0, lead);
        mma_commit(&pv_done[t][js & 1], lead);
        release(v);
      }
      if (!ok) break;
    }
    if (lead) {
      s_item[t][items & 1].j0 = s_item[t][items & 1].j1 = 0;
      mbar_arrive(&item_full[t]);
    }
    __syncwarp();
    // no arrival may outlive the CTA: wait for the release of each slot's last use (the places point behind it)
    for (int i = 0; ok && i < kSlots; ++i) {
      const Place& p = (i & 1) ? v : k;
      ok = warp_wait(&empty[i], i < p.stage ? p.par : p.par ^ 1);
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp + 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols));
  }
  int far = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) far |= s_far[i];
  if (far != 0) far_rows(a, &s_first, s_count, s_far);
}

// Items that cross CTAs: block (i, y) joins 32 rows of the one that CTA i leaves open, if any, from its
// partial there (slot 1) and those of the CTAs behind it (slot 0). A lane has a row, a warp 16 elements.
constexpr int kMergeThreads = 256;
__global__ void __launch_bounds__(kMergeThreads) merge_prefill_fp4_kernel(const __grid_constant__ PrefillArgs a) {
  pdl_wait();
  pdl_trigger();
  const int4 item = a.open_items[blockIdx.x];
  const int n = min(item.x, (int)(gridDim.x - blockIdx.x));  // partials behind the first
  if (n <= 0) return;
  const int row = blockIdx.y * 32 + (threadIdx.x & 31), e0 = (threadIdx.x >> 5) * 16;
  const int tpt = kRows / a.G, r = row % kRows, tt = row / kRows * tpt + r / a.G;
  const Seq q = seq_of(a, item.y);
  const int tok = item.z * a.tok + tt;
  if (r >= tpt * a.G || tok >= q.q_len) return;
  float M = -INFINITY, L = 0.f, o[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) o[i] = 0.f;
#pragma unroll 2
  for (int j = 0; j <= n; ++j) {
    const float* part = a.ws + ((int64_t)(blockIdx.x + j) * 2 + (j == 0 ? 1 : 0)) * kPartFloats;
    const float2 ml = *reinterpret_cast<const float2*>(part + kPartRows * kD + row * 2);
    float4 u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      u[i] = *reinterpret_cast<const float4*>(part + ((e0 / 4 + i) * kPartRows + row) * 4);
    const float mn = fmaxf(M, ml.x);
    const float w0 = M == -INFINITY ? 1.f : ex2((M - mn) * a.scale_log2);
    const float w1 = ml.x == -INFINITY ? 1.f : ex2((ml.x - mn) * a.scale_log2);
    M = mn;
    L = L * w0 + ml.y * w1;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      o[4 * i] = o[4 * i] * w0 + u[i].x * w1;
      o[4 * i + 1] = o[4 * i + 1] * w0 + u[i].y * w1;
      o[4 * i + 2] = o[4 * i + 2] * w0 + u[i].z * w1;
      o[4 * i + 3] = o[4 * i + 3] * w0 + u[i].w * w1;
    }
  }
  const float f = L == 0.f ? 0.f : 1.f / L;
  __half* dst = a.out + ((int64_t)(q.q_start + tok) * a.Hkv * a.G + item.w * a.G + r % a.G) * kD + e0;
#pragma unroll
  for (int i = 0; i < 16; i += 8)
    *reinterpret_cast<uint4*>(dst + i) =
        make_uint4(pack_h2(o[i] * f, o[i + 1] * f), pack_h2(o[i + 2] * f, o[i + 3] * f),
                   pack_h2(o[i + 4] * f, o[i + 5] * f), pack_h2(o[i + 6] * f, o[i + 7] * f));
}

// One CTA per SM; fewer when even full tables would not give every CTA kMinShare units.
int prefill_fp4_ctas(int num_seqs, int total_q, int Hkv, int G, int max_blocks, int block_size, int num_sms) {
  const int64_t items = ((int64_t)total_q / (2 * (kRows / G)) + num_seqs) * Hkv;
  const int64_t units = items * ((int64_t)max_blocks * (block_size / kKeys) + kItemUnits);
  const int64_t need = (units + kMinShare - 1) / kMinShare;
  return (int)(need < num_sms ? (need > 0 ? need : 1) : num_sms);
}

}  // namespace

size_t prefill_fp4_workspace_bytes(int num_seqs, int total_q, int Hq, int Hkv, int max_blocks, int block_size,
                                   int num_sms) {
  const int ctas = prefill_fp4_ctas(num_seqs, total_q, Hkv, Hq / Hkv, max_blocks, block_size, num_sms);
  return (size_t)ctas * (sizeof(int4) + 2 * kPartFloats * sizeof(float));
}

cudaError_t launch_prefill_fp4(const void* q, int64_t q_ts, const void* k_cache, const void* v_cache,
                               const void* k_scale, const void* v_scale, int64_t num_blocks,
                               const int32_t* block_tables, const int32_t* cu_q, const int32_t* kv_lens, void* out,
                               int num_seqs, int total_q, int Hq, int Hkv, int block_size, int max_blocks,
                               float softmax_scale, void* workspace, int num_sms, cudaStream_t stream) {
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
  a.inv_g = (65536 + a.G - 1) / a.G;
  a.tok = 2 * (kRows / a.G);
  a.block_size = block_size;
  a.bs_log2 = (block_size & (block_size - 1)) == 0 ? __builtin_ctz((unsigned)block_size) : -1;
  a.max_blocks = max_blocks;
  const int64_t cap = (int64_t)max_blocks * block_size;
  a.cap = (int)(cap < (1 << 30) ? cap : (1 << 30));
  a.scale_log2 = softmax_scale * kLog2e;
  // sums of units fit 32 bits in the kernel
  if (((int64_t)total_q / a.tok + num_seqs) * (a.cap / kKeys + 1 + kItemUnits) >= ((int64_t)1 << 31) / Hkv)
    return cudaErrorInvalidValue;
  const int ctas = prefill_fp4_ctas(num_seqs, total_q, Hkv, a.G, max_blocks, block_size, num_sms);
  a.open_items = (int4*)workspace;
  a.ws = (float*)((int4*)workspace + ctas);
  static std::atomic<uint64_t> allowed{0};
  cudaError_t e = allow_smem(prefill_fp4_kernel, kSmemBytes, allowed);
  if (e != cudaSuccess) return e;
  // Q as (element, head, token); a box is 64 elements of a tile's rows
  const EncodeTiledFn encode = get_encode_fn();
  if (encode == nullptr) return cudaErrorNotSupported;
  CUtensorMap map;
  const cuuint64_t dims[3] = {(cuuint64_t)kD, (cuuint64_t)Hq, (cuuint64_t)total_q};
  const cuuint64_t strides[2] = {(cuuint64_t)kD * 2, (cuuint64_t)q_ts * 2};
  const cuuint32_t box[3] = {64, (cuuint32_t)a.G, (cuuint32_t)(kRows / a.G)}, step[3] = {1, 1, 1};
  if (encode(&map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(q), dims, strides, box, step,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
    return cudaErrorInvalidValue;
  e = launch_kernel(prefill_fp4_kernel, dim3(ctas), dim3(kThreads), kSmemBytes, stream, map, a);
  if (e != cudaSuccess || ctas == 1) return e;
  return launch_kernel(merge_prefill_fp4_kernel, dim3(ctas - 1, kPartRows / 32), dim3(kMergeThreads), 0, stream, a);
}

}  // namespace ms
