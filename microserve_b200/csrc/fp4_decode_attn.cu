// Decode attention over the paged 4-bit KV cache (format: fp4_kv.cuh), one query token
// per sequence:
//   o[b, hq] = softmax_t(q[b, hq] . k[t] * scale) . v[t],  t < seqlens[b];  0 for no token.
//
// Its floor is the cache's bytes (144 per token and kv head); what binds it now is waiting inside a warp's one chain per
// tile (decode K, scores, softmax, decode V, product), nothing of the next tile being mixed in.
// 241 MB of cache (256 sequences of 128 to 1536 tokens, 32 / 8 heads) take 58.7 us, 0.63 of the copy bandwidth:
// 4.5 us to the first tile (scan, page look-up, copy: three memory latencies), 46 to 50 for an SM's tiles (its
// copies alone 44, its arithmetic alone 54 with the overheads, where the issue of 640 instructions a tile and warp would
// take 30: a scheduler issues 0.54 of the time), 3 for the join, 2.5 for the second kernel.
//  * The work is one flat list of 32-token tiles over (sequence, kv head, tile). The grid
//    fills the SMs once; every CTA takes an equal contiguous share of the list, an item's own
//    cost counted like a tile (found by a scan of seqlens), and every warp a quarter of that,
//    whatever the lengths are. A warp keeps kStages tiles (codes and scales of K and V) in flight through its own ring
//    of shared memory (cp.async), across the borders of items (sequence, kv head). An item
//    inside one warp's share is finished by that warp alone; the pieces of one that
//    crosses warps are joined in shared memory at the end of the CTA, of one that crosses
//    CTAs through fp32 partials (o, m, l) in the workspace by a second kernel. A CTA leaves
//    at most two such partials.
//  * The G = Hq / Hkv <= 8 query heads of a kv head are the N side of mma.m16n8k16, so K
//    and V are read and decoded once for all of them:
//        S^T[tok, head] = K[tok, d] . Q^T[d, head],   O^T[d, head] += V^T[d, tok] . P^T[tok, head]
//    Codes become f16 in registers (cvt e2m1x2, times the scale: exact). head_dim is
//    permuted in the first product so that a thread's fragment is the 16 contiguous bytes
//    it reads (Q is loaded in the same order), and the tokens of a tile are permuted so that the
//    8 tokens a thread needs of V are consecutive; neither changes a result.
//  * Softmax in the exp2 domain, fp32 sums, with a lazy reference: weights are 2^(s - m)
//    for a reference m that moves (and the sums are rescaled) only when a score exceeds it by
//    5 or more, which after an item's first tile is rare (or is too far from zero for one rounding of
//    its product with the scale: fp4_kv.cuh). A weight enters the second
//    product as two f16 parts (hi + lo, scaled by 2^10: at most 2^15), so outputs keep
//    fp32-level accuracy; with G <= 4 both parts share one MMA (columns 0-3 hi, 4-7 lo),
//    with more heads it takes two.
#include "fp4_kv.cuh"
#include "kernels.h"

namespace ms {
namespace {

constexpr int kD = kFp4Dim;
constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kStages = 2;                 // tiles in flight per warp
constexpr int kTile = 32;                  // tokens of a tile
constexpr int kCodeBytes = kTile * kFp4RowBytes;
constexpr int kScBytes = kTile * kFp4ScaleBytes;
constexpr int kStageBytes = 2 * kCodeBytes + 2 * kScBytes;
constexpr int kRingBytes = kWarps * kStages * kStageBytes;
constexpr int kRowFloats = kD + 4;         // a partial of one head in shared memory: o[128], m, l, padding
constexpr int kCtasPerSm = 3;
// The list is dealt in units of a tile's time: an item's first load of Q, sums over lanes and output count as
// kItemUnits behind its tiles (256 sequences of 128 to 1536 tokens: 60.5 us without, 58.0 with 1, 58.4 with 2).
constexpr int kItemUnits = 1;
constexpr int kMinShare = 4;               // units of a CTA at least: one a warp (one sequence of 300: 7.9 us, 8.8 with two)
constexpr int kPartFloats = kD + 2;        // a partial of one head: o[128], m, l
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kPScaleLog2 = 10.f;        // weights are scaled by 2^10: lo stays a normal f16 where it matters,
constexpr float kPMaxLog2 = 15.f;          // and hi finite up to a score 5 above the reference

constexpr int smem_bytes(int heads) { return kRingBytes + kWarps * heads * kRowFloats * 4; }
static_assert(kStages * kStageBytes >= 8 * kRowFloats * 4, "a warp's last partial fits its ring");

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

__device__ __forceinline__ uint32_t pack_h2(float lo, float hi) {
  __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&h);
}

__device__ __forceinline__ float2 h2_to_f2(uint32_t x) {
  __half2 h;
  memcpy(&h, &x, 4);
  return __half22float2(h);
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

struct DecodeArgs {
  const __half* q;  // [B, Hq, D], token stride q_ts elements
  int64_t q_ts;
  const uint8_t *kc, *vc, *ks, *vs;
  int64_t num_blocks;
  const int32_t* seqlens;
  const int32_t* tables;  // [B, max_blocks]
  __half* out;            // [B, Hq, D]
  int4* open_items;       // workspace: per CTA, the item that it leaves open: CTAs it goes on in, b, kv head
  float* ws;              // workspace: [CTAs][2][G][kPartFloats]
  int B, Hkv, G, block_size, bs_log2, max_blocks;
  int cap;                // tokens that a table row can hold
  float scale_log2;
};

// Tokens of sequence b (0 where negative, cut at the table's end) and its tiles.
__device__ __forceinline__ int seq_len(const DecodeArgs& a, int b) { return min(max(a.seqlens[b], 0), a.cap); }
__device__ __forceinline__ int tiles_of(int len) { return (len + kTile - 1) / kTile; }
__device__ __forceinline__ int units_of(int nt) { return nt > 0 ? nt + kItemUnits : 0; }  // of an item of nt tiles

// The flat tile list: the units of a kv head in all sequences before the calling thread's own,
// [b0, b1), and in all of them. Whole block.
struct Scan {
  int64_t before, total;  // in units of one kv head
  int b0, b1;
};
__device__ __forceinline__ Scan scan_lens(const DecodeArgs& a, int64_t* red) {
  Scan s;
  const int per = (a.B + kThreads - 1) / kThreads;
  s.b0 = min((int)threadIdx.x * per, a.B);
  s.b1 = min(s.b0 + per, a.B);
  int64_t mine = 0;
  for (int b = s.b0; b < s.b1; ++b) mine += units_of(tiles_of(seq_len(a, b)));
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int64_t inc = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t up = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += up;
  }
  if (lane == 31) red[warp] = inc;
  __syncthreads();
  s.before = inc - mine;
  s.total = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) s.before += red[w];
    s.total += red[w];
  }
  return s;
}
// Units a CTA takes.
__device__ __forceinline__ int64_t share_of(int64_t total, int ctas) {
  const int64_t even = (total + ctas - 1) / ctas;
  return even > kMinShare ? even : kMinShare;
}

// Position in a warp's units: item (b, h) of nt tiles and len tokens starts at relative
// unit `start` (negative: in an earlier warp).
struct Cursor {
  int b, h, nt, len, start;
  __device__ __forceinline__ void next_item(const DecodeArgs& a) {
    start += nt + kItemUnits;
    if (++h == a.Hkv) {
      h = 0;
      do {
        ++b;
        len = b < a.B ? seq_len(a, b) : 0;
        nt = b < a.B ? tiles_of(len) : 1 << 30;  // behind the last sequence: only if seqlens changed meanwhile
      } while (nt == 0);
    }
  }
};

// The pieces of items that a warp leaves for the CTA's join: of its first item if that began
// before the warp's share, and of its last one if that goes on behind it.
struct Pieces {
  int head, head_goes_on, tail;  // flags
  int hb, hh, tb, th;            // their items
  int over;                      // tiles of the last one behind the CTA's share (0 or less: none)
};

template <bool kTwoParts>  // false: G <= 4, hi and lo weights share an MMA; true: G = 5..8
__global__ void __launch_bounds__(kThreads, kCtasPerSm) decode_fp4_kernel(const __grid_constant__ DecodeArgs a) {
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ int64_t s_red[kWarps];
  __shared__ Cursor s_first[kWarps];
  __shared__ Pieces s_pieces[kWarps];
  constexpr int kHeads = kTwoParts ? 8 : 4;  // head columns of a partial
  pdl_wait();
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, c = lane & 3;
  const int G = a.G;

  // ---- this CTA's share, and this warp's quarter of it ------------------------------
  const Scan sc = scan_lens(a, s_red);
  const int64_t total = sc.total * a.Hkv;
  const int64_t share = share_of(total, gridDim.x);
  const int64_t begin = (int64_t)blockIdx.x * share;
  // sequences without tokens: zero rows, dealt to the CTAs
  for (int b = blockIdx.x; b < a.B; b += gridDim.x) {
    const int n = a.seqlens[b];
    if (n > a.cap && threadIdx.x == 0) set_device_status(kStatusBadPage);
    if (n <= 0)
      for (int i = threadIdx.x; i < a.Hkv * G * (kD / 8); i += kThreads)
        reinterpret_cast<uint4*>(a.out + (int64_t)b * a.Hkv * G * kD)[i] = make_uint4(0, 0, 0, 0);
  }
  if (begin >= total) {
    if (threadIdx.x == 0) a.open_items[blockIdx.x] = make_int4(0, 0, 0, 0);
    return;
  }
  const int cta_units = (int)(total - begin < share ? total - begin : share);
  auto warp_begin = [&](int w) { return (int)((int64_t)cta_units * w / kWarps); };
  {  // the threads whose sequences hold the warps' first tiles leave their items
    int64_t at = sc.before * a.Hkv;
    for (int b = sc.b0; b < sc.b1; ++b) {
      const int len = seq_len(a, b), nt = tiles_of(len), nu = units_of(nt);
      const int64_t end = at + (int64_t)nu * a.Hkv;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const int64_t x = begin + warp_begin(w);
        if (x >= at && x < end) {
          const int h = (int)((x - at) / nu);
          s_first[w] = Cursor{b, h, nt, len, -(int)(x - at - (int64_t)h * nu)};
        }
      }
      at = end;
    }
  }
  __syncthreads();
  const int count = warp_begin(warp + 1) - warp_begin(warp);  // units of this warp

  // ---- this warp's ring --------------------------------------------------------------
  unsigned char* ring = smem + warp * (kStages * kStageBytes);
  const uint32_t ring_u32 = smem_u32(ring);
  // V rows of 64 bytes are placed so that the 8-byte reads below are conflict free: rows
  // 2k, 2k + 1 swapped in the upper half of the tile, 32-byte halves of a row swapped in
  // every other 8 rows.
  uint32_t v_dst[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int q = lane + 32 * i, tok = q >> 2, j = q & 3;
    v_dst[i] = (uint32_t)(kCodeBytes + ((tok ^ ((tok >> 4) & 1)) * kFp4RowBytes) + ((j ^ (((tok >> 3) & 1) << 1)) << 4));
  }
  Cursor cu = s_first[warp];
  if (count > 0 && cu.start + cu.nt <= 0) cu.next_item(a);  // the share begins behind the item's tiles
  Cursor is = cu;  // issue side: the item of tile is_r
  int is_r = max(is.start, 0);
  uint32_t bad = 0;     // stages whose tile has no valid page
  int64_t is_row = 0;   // first cache row of tile is_r, -1: none
  int page_left = 0;    // tiles left in its page, this one included
  auto look_up = [&] {  // the page of tile is_r
    if (is_r == is.start + is.nt) {
      is.next_item(a);
      is_r = is.start;
      if (is_r >= count) return;
    }
    const int p0 = (is_r - is.start) * kTile;
    const int page = a.bs_log2 >= 0 ? p0 >> a.bs_log2 : p0 / a.block_size;
    const int off = p0 - page * a.block_size;
    const int64_t blk = is.b < a.B && page < a.max_blocks ? __ldg(a.tables + (int64_t)is.b * a.max_blocks + page) : -1;
    is_row = (blk < 0 || blk >= a.num_blocks) ? -1 : (blk * a.Hkv + is.h) * a.block_size + off;
    page_left = min((a.block_size - off) / kTile, is.start + is.nt - is_r);
  };
  auto issue = [&](int slot) {
    if (is_r < count) {
      if (is_row >= 0) {
        const uint32_t st = ring_u32 + (uint32_t)(slot * kStageBytes);
        const uint8_t* kp = a.kc + is_row * kFp4RowBytes + lane * 16;
        const uint8_t* vp = a.vc + is_row * kFp4RowBytes + lane * 16;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          cp_async16(st + lane * 16 + i * 512, kp + i * 512);
          cp_async16(st + v_dst[i], vp + i * 512);
        }
        cp_async16(st + 2 * kCodeBytes + lane * 16,
                   (lane < 16 ? a.ks : a.vs) + is_row * kFp4ScaleBytes + (lane & 15) * 16);
        bad &= ~(1u << slot);
        is_row += kTile;
      } else {
        if (lane == 0) set_device_status(kStatusBadPage);
        bad |= 1u << slot;
      }
      ++is_r;
      if (--page_left == 0 && is_r < count) look_up();
    }
    cp_async_commit();  // one group per slot, empty or not
  };
  if (is_r < count) look_up();
#pragma unroll
  for (int k = 0; k < kStages; ++k) issue(k);

  float* head_part = reinterpret_cast<float*>(smem + kRingBytes) + warp * kHeads * kRowFloats;
  const uint32_t v_even = (uint32_t)((8 * c + (c >> 1)) * kFp4RowBytes + (((g >> 1) ^ ((c & 1) << 1)) << 4) + (g & 1) * 8);
  const uint32_t v_odd = (uint32_t)((8 * c + 1 - (c >> 1)) * kFp4RowBytes + (((g >> 1) ^ ((c & 1) << 1)) << 4) + (g & 1) * 8);
  const int tok_a = 8 * (g >> 1) + (g & 1);  // token of MMA row g: tok_a + 4 tile + 2 (row >= 8)

  Pieces pieces = {0, 0, 0, 0, 0, 0, 0, 0};
  int r = max(cu.start, 0), slot = 0;
  while (r < count && cu.b < a.B) {  // (behind the last sequence: only if seqlens changed meanwhile)
    const int seg_end = min(cu.start + cu.nt, count);
    // Q fragment: column g = head g (G <= 4: columns 4-7 repeat 0-3), d = 32 c + [0, 32)
    uint32_t qf[16];
    {
      const int hq = kTwoParts ? g : (g & 3);
      const bool valid = hq < G;
      const uint4* qp = reinterpret_cast<const uint4*>(a.q + cu.b * a.q_ts + (cu.h * G + (valid ? hq : 0)) * kD + 32 * c);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint4 u = valid ? qp[i] : make_uint4(0, 0, 0, 0);
        qf[4 * i] = u.x;
        qf[4 * i + 1] = u.y;
        qf[4 * i + 2] = u.z;
        qf[4 * i + 3] = u.w;
      }
    }
    float acc[8][4];
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
    float m_ref[2] = {-INFINITY, -INFINITY};  // columns 2c, 2c + 1: the reference, a score
    // 10 - m_ref scale_log2; infinite where the reference is a far score (fp4_kv.cuh), so that tiles with keys take the
    // branch below, which forms differences
    float neg[2] = {INFINITY, INFINITY};
    float l_run[2] = {0.f, 0.f};

    for (; r < seg_end; ++r) {
      cp_async_wait<kStages - 1>();
      __syncwarp();
      const unsigned char* st = ring + slot * kStageBytes;
      const int left = (bad >> slot) & 1u ? 0 : cu.len - (r - cu.start) * kTile;  // valid tokens from here on
      // ---- scores: rows of MMA tile t are tokens tok_a + 4 t (+ 2 for rows 8-15) ----
      float s[2][4];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        s[t][0] = s[t][1] = s[t][2] = s[t][3] = 0.f;
        const unsigned char* k0 = st + (tok_a + 4 * t) * kFp4RowBytes + c * 16;
        const unsigned char* sp = st + 2 * kCodeBytes + (tok_a + 4 * t) * kFp4ScaleBytes + c * 2;
        const uint4 x0 = *reinterpret_cast<const uint4*>(k0);
        const uint4 x1 = *reinterpret_cast<const uint4*>(k0 + 2 * kFp4RowBytes);
        const uint32_t f0[2] = {fp4_scale_h2(sp[0]), fp4_scale_h2(sp[1])};
        const uint32_t f1[2] = {fp4_scale_h2(sp[2 * kFp4ScaleBytes]), fp4_scale_h2(sp[2 * kFp4ScaleBytes + 1])};
        const uint32_t w0[4] = {x0.x, x0.y, x0.z, x0.w}, w1[4] = {x1.x, x1.y, x1.z, x1.w};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          uint32_t h0[4], h1[4];
          fp4x8_to_f16x2(w0[w], h0);
          fp4x8_to_f16x2(w1[w], h1);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            h0[i] = h2_mul(h0[i], f0[w >> 1]);
            h1[i] = h2_mul(h1[i], f1[w >> 1]);
          }
          mma16816(s[t], h0[0], h1[0], h0[1], h1[1], qf[4 * w], qf[4 * w + 1]);
          mma16816(s[t], h0[2], h1[2], h0[3], h1[3], qf[4 * w + 2], qf[4 * w + 3]);
        }
      }
      // ---- softmax: exponents against the reference ------------------------------------
      float e[2][4];
      auto exponents = [&](bool differences) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            e[t][j] = fmaf(s[t][j], a.scale_log2, neg[j & 1]);
            if (differences && neg[j & 1] == INFINITY)
              e[t][j] = fmaf(s[t][j] - m_ref[j & 1], a.scale_log2, kPScaleLog2);
          }
          if (left < kTile) {
            if (tok_a + 4 * t >= left) e[t][0] = e[t][1] = -INFINITY;
            if (tok_a + 4 * t + 2 >= left) e[t][2] = e[t][3] = -INFINITY;
          }
        }
      };
      exponents(false);
      const float top = fmaxf(fmaxf(fmaxf(e[0][0], e[0][1]), fmaxf(e[0][2], e[0][3])),
                              fmaxf(fmaxf(e[1][0], e[1][1]), fmaxf(e[1][2], e[1][3])));
      if (__any_sync(0xffffffffu, top > kPMaxLog2)) {  // move the reference to this tile's maximum
        float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          if (tok_a + 4 * t < left) {
            mx[0] = fmaxf(mx[0], s[t][0]);
            mx[1] = fmaxf(mx[1], s[t][1]);
          }
          if (tok_a + 4 * t + 2 < left) {
            mx[0] = fmaxf(mx[0], s[t][2]);
            mx[1] = fmaxf(mx[1], s[t][3]);
          }
        }
        float al[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) mx[j] = fmaxf(mx[j], __shfl_xor_sync(0xffffffffu, mx[j], o));
          const float mn = fmaxf(m_ref[j], mx[j]);
          al[j] = m_ref[j] == -INFINITY ? 1.f : ex2((m_ref[j] - mn) * a.scale_log2);  // nothing summed yet: nothing to rescale
          m_ref[j] = mn;
          neg[j] = far_score(mn, a.scale_log2) ? INFINITY : fmaf(-mn, a.scale_log2, kPScaleLog2);
          l_run[j] *= al[j];
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          acc[i][0] *= al[0];
          acc[i][1] *= al[1];
          acc[i][2] *= al[0];
          acc[i][3] *= al[1];
        }
        exponents(true);
      }
      uint32_t hi[2][2], lo[2][2];  // [MMA tile][rows 0-7, 8-15]
#pragma unroll
      for (int t = 0; t < 2; ++t) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const float p0 = ex2(e[t][2 * u]), p1 = ex2(e[t][2 * u + 1]);
          l_run[0] += p0;
          l_run[1] += p1;
          const uint32_t h = pack_h2(p0, p1);
          const float2 hf = h2_to_f2(h);
          const uint32_t l = pack_h2(p0 - hf.x, p1 - hf.y);
          if (kTwoParts) {
            hi[t][u] = movmatrix_trans(h);
            lo[t][u] = movmatrix_trans(l);
          } else {
            hi[t][u] = movmatrix_trans(c < 2 ? h : l);  // columns 4-7: the same heads' lo parts
          }
        }
      }
      // ---- O^T += V^T P^T: k index 2c + w + 8u of step t is token 8c + 4t + 2u + w ----
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        uint32_t x[4][2], f[2];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint2 v = *reinterpret_cast<const uint2*>(st + kCodeBytes + ((i & 1) ? v_odd : v_even) +
                                                          (4 * t + (i & 2)) * kFp4RowBytes);
          x[i][0] = v.x;
          x[i][1] = v.y;
        }
        const unsigned char* sp = st + 2 * kCodeBytes + kScBytes + (8 * c + 4 * t) * kFp4ScaleBytes + g;
        uint32_t b[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) b[i] = sp[i * kFp4ScaleBytes];
        if (left < kTile) {  // what lies behind the end may be anything
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (8 * c + 4 * t + i >= left) x[i][0] = x[i][1] = b[i] = 0;
        }
        f[0] = b[0] * 0x80u + b[1] * 0x800000u;
        f[1] = b[2] * 0x80u + b[3] * 0x800000u;
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          // bytes of (token 0, token 1) pairs: even elements, then odd ones
          uint32_t e0[4], o0[4], e1[4], o1[4];
          constexpr uint32_t kLow = 0x0F0F0F0Fu;
          fp4x8_to_f16x2((x[0][w] & kLow) | ((x[1][w] << 4) & ~kLow), e0);
          fp4x8_to_f16x2(((x[0][w] >> 4) & kLow) | (x[1][w] & ~kLow), o0);
          fp4x8_to_f16x2((x[2][w] & kLow) | ((x[3][w] << 4) & ~kLow), e1);
          fp4x8_to_f16x2(((x[2][w] >> 4) & kLow) | (x[3][w] & ~kLow), o1);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t a0 = h2_mul(e0[i], f[0]), a1 = h2_mul(o0[i], f[0]);
            const uint32_t a2 = h2_mul(e1[i], f[1]), a3 = h2_mul(o1[i], f[1]);
            mma16816(acc[4 * w + i], a0, a1, a2, a3, hi[t][0], hi[t][1]);
            if (kTwoParts) mma16816(acc[4 * w + i], a0, a1, a2, a3, lo[t][0], lo[t][1]);
          }
        }
      }
      __syncwarp();  // every lane is done with the slot
      issue(slot);
      slot = slot + 1 == kStages ? 0 : slot + 1;
    }

    // ---- the item's tiles of this warp are done -------------------------------------------
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) {
      l_run[0] += __shfl_xor_sync(0xffffffffu, l_run[0], o);
      l_run[1] += __shfl_xor_sync(0xffffffffu, l_run[1], o);
    }
    if (!kTwoParts) {  // hi + lo
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] += __shfl_xor_sync(0xffffffffu, acc[i][j], 2);
    }
    // acc[i][j], acc[i][2 + j]: d = 16 g + 2 i, + 1 of head 2 c + j
    const bool began = cu.start >= 0, goes_on = cu.start + cu.nt > count;
    if (began && !goes_on) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        if ((kTwoParts || c < 2) && 2 * c + j < G) {
          const float inv = l_run[j] == 0.f ? 0.f : 1.f / l_run[j];
          uint4* dst = reinterpret_cast<uint4*>(a.out + (((int64_t)cu.b * a.Hkv + cu.h) * G + 2 * c + j) * kD + 16 * g);
#pragma unroll
          for (int i = 0; i < 8; i += 4)
            dst[i >> 2] = make_uint4(
                pack_h2(acc[i][j] * inv, acc[i][2 + j] * inv), pack_h2(acc[i + 1][j] * inv, acc[i + 1][2 + j] * inv),
                pack_h2(acc[i + 2][j] * inv, acc[i + 2][2 + j] * inv), pack_h2(acc[i + 3][j] * inv, acc[i + 3][2 + j] * inv));
        }
      }
    } else {
      // the last piece may take the ring: every copy into it has landed and been read
      float* part = began ? reinterpret_cast<float*>(ring) : head_part;
      if (began) {
        cp_async_wait<0>();
        __syncwarp();
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        if (kTwoParts || c < 2) {
          float* row = part + (2 * c + j) * kRowFloats;
#pragma unroll
          for (int i = 0; i < 8; i += 2)
            *reinterpret_cast<float4*>(row + 16 * g + 2 * i) =
                make_float4(acc[i][j], acc[i][2 + j], acc[i + 1][j], acc[i + 1][2 + j]);
          if (g == 0) {
            row[kD] = m_ref[j];
            row[kD + 1] = l_run[j];
          }
        }
      }
      if (began) {
        pieces.tail = 1;
        pieces.tb = cu.b;
        pieces.th = cu.h;
        pieces.over = warp_begin(warp) + cu.start + cu.nt - cta_units;
      } else {
        pieces.head = 1;
        pieces.head_goes_on = goes_on;
        pieces.hb = cu.b;
        pieces.hh = cu.h;
      }
    }
    if (seg_end == count) break;
    cu.next_item(a);
    r = cu.start;
  }
  cp_async_wait<0>();
  if (lane == 0) s_pieces[warp] = pieces;
  __syncthreads();

  // ---- join the pieces of items that cross warps, in the order of the list; a thread has
  // 8 elements of one head ------------------------------------------------------------------
  const int h = threadIdx.x >> 4, d0 = (threadIdx.x & 15) * 8;
  if (h >= G) return;
  float M = -INFINITY, L = 0.f, o[8];
  bool before = true, open = false;  // the item at hand began in an earlier CTA; has pieces
  int ib = 0, ih = 0, over = 0;
  auto take = [&](const float* part) {
    const float* row = part + h * kRowFloats;
    const float m = row[kD], mn = fmaxf(M, m);
    const float w0 = M == -INFINITY ? 1.f : ex2((M - mn) * a.scale_log2);  // a sum without valid tokens is 0 (or NaN)
    const float w1 = m == -INFINITY ? 1.f : ex2((m - mn) * a.scale_log2);
    M = mn;
    L = L * w0 + row[kD + 1] * w1;
    const float4 u0 = *reinterpret_cast<const float4*>(row + d0), u1 = *reinterpret_cast<const float4*>(row + d0 + 4);
    const float u[8] = {u0.x, u0.y, u0.z, u0.w, u1.x, u1.y, u1.z, u1.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = o[i] * w0 + u[i] * w1;
  };
  auto start = [&](bool from_before, int b, int hh) {
    M = -INFINITY;
    L = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = 0.f;
    before = from_before;
    open = true;
    ib = b;
    ih = hh;
  };
  auto leave = [&](int which) {  // partial for the merge kernel
    float* dst = a.ws + (((int64_t)blockIdx.x * 2 + which) * G + h) * kPartFloats;
#pragma unroll
    for (int i = 0; i < 8; i += 2) *reinterpret_cast<float2*>(dst + d0 + i) = make_float2(o[i], o[i + 1]);
    if (d0 == 0) *reinterpret_cast<float2*>(dst + kD) = make_float2(M, L);
  };
#pragma unroll 1
  for (int w = 0; w < kWarps; ++w) {
    const Pieces p = s_pieces[w];
    if (p.head) {
      if (!open) start(true, p.hb, p.hh);
      take(reinterpret_cast<const float*>(smem + kRingBytes) + w * kHeads * kRowFloats);
      if (!p.head_goes_on) {
        if (before) {
          leave(0);
        } else {
          const float inv = L == 0.f ? 0.f : 1.f / L;
          *reinterpret_cast<uint4*>(a.out + (((int64_t)ib * a.Hkv + ih) * G + h) * kD + d0) =
              make_uint4(pack_h2(o[0] * inv, o[1] * inv), pack_h2(o[2] * inv, o[3] * inv),
                         pack_h2(o[4] * inv, o[5] * inv), pack_h2(o[6] * inv, o[7] * inv));
        }
        open = false;
      }
    }
    if (p.tail) {
      start(false, p.tb, p.th);
      over = p.over;
      take(reinterpret_cast<const float*>(smem + w * (kStages * kStageBytes)));
    }
  }
  if (open) leave(before ? 0 : 1);  // goes on in the next CTA
  if (threadIdx.x == 0)
    a.open_items[blockIdx.x] = make_int4(open && !before ? (int)((over + share - 1) / share) : 0, ib, ih, 0);
}

// Items that cross CTAs: block i joins the one that CTA i leaves open, if any, from its piece
// there (slot 1) and those of the CTAs behind it (slot 0). 16 lanes cover head_dim with 8
// elements each; the rows of 16 lanes are (head, stream) and the streams take the pieces in
// turn, four loads in flight each.
constexpr int kMergeThreads = 256;
__global__ void __launch_bounds__(kMergeThreads) merge_fp4_kernel(const __grid_constant__ DecodeArgs a) {
  __shared__ float s_part[kMergeThreads / 16][kD + 4];
  pdl_wait();
  pdl_trigger();
  const int4 item = a.open_items[blockIdx.x];
  const int n = item.x;  // pieces behind the first
  if (n <= 0) return;
  const int streams = kMergeThreads / 16 / a.G;
  const int row = threadIdx.x >> 4, d0 = (threadIdx.x & 15) * 8;
  const int h = row % a.G, stream = row / a.G;
  float M = -INFINITY, L = 0.f, o[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) o[i] = 0.f;
  auto take = [&](float m, float l, const float (&u)[8]) {
    const float mn = fmaxf(M, m);
    const float w0 = M == -INFINITY ? 1.f : ex2((M - mn) * a.scale_log2);
    const float w1 = m == -INFINITY ? 1.f : ex2((m - mn) * a.scale_log2);
    M = mn;
    L = L * w0 + l * w1;
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = o[i] * w0 + u[i] * w1;
  };
  if (stream < streams) {
    for (int j0 = stream; j0 <= n; j0 += 4 * streams) {
      float2 ml[4];
      float u[4][8];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int j = j0 + k * streams;
        if (j > n) continue;
        const float* p = a.ws + (((int64_t)(blockIdx.x + j) * 2 + (j == 0 ? 1 : 0)) * a.G + h) * kPartFloats;
        ml[k] = *reinterpret_cast<const float2*>(p + kD);
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
          const float2 v = *reinterpret_cast<const float2*>(p + d0 + i);
          u[k][i] = v.x;
          u[k][i + 1] = v.y;
        }
      }
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (j0 + k * streams <= n) take(ml[k].x, ml[k].y, u[k]);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) s_part[row][d0 + i] = o[i];
    if (d0 == 0) {
      s_part[row][kD] = M;
      s_part[row][kD + 1] = L;
    }
  }
  __syncthreads();
  if (row >= a.G) return;  // stream 0 of each head joins the others
  for (int k = 1; k < streams; ++k) {
    const float* p = s_part[row + k * a.G];
    float u[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) u[i] = p[d0 + i];
    take(p[kD], p[kD + 1], u);
  }
  const float inv = L == 0.f ? 0.f : 1.f / L;
  *reinterpret_cast<uint4*>(a.out + (((int64_t)item.y * a.Hkv + item.z) * a.G + h) * kD + d0) =
      make_uint4(pack_h2(o[0] * inv, o[1] * inv), pack_h2(o[2] * inv, o[3] * inv), pack_h2(o[4] * inv, o[5] * inv),
                 pack_h2(o[6] * inv, o[7] * inv));
}

// CTAs of the main kernel: what the SMs hold at once, fewer when even tables full of tokens would not
// give every CTA kMinShare units.
int decode_fp4_ctas(int B, int Hkv, int max_blocks, int block_size, int num_sms) {
  const int64_t most = (int64_t)B * Hkv * ((int64_t)max_blocks * (block_size / kTile) + kItemUnits);
  const int64_t fill = (int64_t)num_sms * kCtasPerSm, need = (most + kMinShare - 1) / kMinShare;
  return (int)(need < fill ? (need > 0 ? need : 1) : fill);
}

}  // namespace

size_t decode_fp4_workspace_bytes(int B, int Hq, int Hkv, int max_blocks, int block_size, int num_sms) {
  return (size_t)decode_fp4_ctas(B, Hkv, max_blocks, block_size, num_sms) *
         (sizeof(int4) + 2 * (Hq / Hkv) * kPartFloats * sizeof(float));
}

cudaError_t launch_decode_fp4(const void* q, int64_t q_ts, const void* k_cache, const void* v_cache,
                              const void* k_scale, const void* v_scale, int64_t num_blocks, const int32_t* seqlens,
                              const int32_t* block_tables, void* out, int B, int Hq, int Hkv, int block_size,
                              int max_blocks, float softmax_scale, void* workspace, int num_sms,
                              cudaStream_t stream) {
  DecodeArgs a = {};
  a.q = (const __half*)q;
  a.q_ts = q_ts;
  a.kc = (const uint8_t*)k_cache;
  a.vc = (const uint8_t*)v_cache;
  a.ks = (const uint8_t*)k_scale;
  a.vs = (const uint8_t*)v_scale;
  a.num_blocks = num_blocks;
  a.seqlens = seqlens;
  a.tables = block_tables;
  a.out = (__half*)out;
  a.B = B;
  a.Hkv = Hkv;
  a.G = Hq / Hkv;
  a.block_size = block_size;
  a.bs_log2 = (block_size & (block_size - 1)) == 0 ? __builtin_ctz((unsigned)block_size) : -1;
  a.max_blocks = max_blocks;
  const int64_t cap = (int64_t)max_blocks * block_size;
  a.cap = (int)(cap < (1 << 30) ? cap : (1 << 30));
  a.scale_log2 = softmax_scale * kLog2e;
  // a CTA counts its units in 32 bits, with room for one item more (2^30 on every SM's three CTAs: hours of work)
  if ((double)B * Hkv * (a.cap / kTile + kItemUnits + 1) >= (double)num_sms * kCtasPerSm * (1 << 30))
    return cudaErrorInvalidValue;
  const int ctas = decode_fp4_ctas(B, Hkv, max_blocks, block_size, num_sms);
  a.open_items = (int4*)workspace;
  a.ws = (float*)((int4*)workspace + ctas);
  const bool two = a.G > 4;
  static std::atomic<uint64_t> allowed[2];
  cudaError_t e = two ? allow_smem(decode_fp4_kernel<true>, smem_bytes(8), allowed[1])
                      : allow_smem(decode_fp4_kernel<false>, smem_bytes(4), allowed[0]);
  if (e != cudaSuccess) return e;
  e = two ? launch_kernel(decode_fp4_kernel<true>, dim3(ctas), dim3(kThreads), smem_bytes(8), stream, a)
          : launch_kernel(decode_fp4_kernel<false>, dim3(ctas), dim3(kThreads), smem_bytes(4), stream, a);
  if (e != cudaSuccess || ctas == 1) return e;
  return launch_kernel(merge_fp4_kernel, dim3(ctas - 1), dim3(kMergeThreads), 0, stream, a);
}

}  // namespace ms
