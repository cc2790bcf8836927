// attention_paged.cu — attention of single new tokens over the paged KV cache
// (fp16 or int8 rows), split over the cache's length and joined.
//
// For token t, kv head g and its G query heads:
//     o_h = sum_j p_hj v_j / sum_j p_hj,  p_hj = exp(q_h . k_j / sqrt(D) - m_h)
// over positions j = 0..positions[t]. The kernel reads each cached row once:
// 2 (positions[t] + 1) rows of D fp16 values, or of D codes and a scale, per
// (token, kv head), and is bound by HBM.
//
// The positions of a (token, kv head) are dealt to the CTAs of a cluster (and,
// for few tokens over a long cache, to several clusters). A CTA's four warps (one,
// where there are many short items)
// stream 32-position tiles of K and V through a per-warp cp.async ring, the
// rows' addresses taken from the page table one tile ahead; pages hold eight
// positions at least, so eight rows share one address. Both products run on
// mma.sync m16n8k16 with the cached rows as the M side: S^T = K Q^T (16
// positions x 8 heads) and O^T += V^T P^T (16 dims x 8 heads), so a group of up
// to eight query heads fills the N side; with heads as the M side half or more
// of every fragment, exponential and accumulator would be padding.
//
// int8 rows. K: the codes go into integer products as they are (mma m16n8k32),
// with the query head as three int8 digits, q = qmax / (127 2^14) (2^14 h + 2^7 m
// + l): exact sums of codes with a query that is off by at most 2^-21 of its
// head's largest value (half a unit, and the fp32 product that makes it). The
// key's scale multiplies its scores. V: a code c
// becomes the fp16 1024 + (c + 128) by placing its byte, top bit flipped, under
// the exponent byte 0x64 (one logic operation for two codes), and one packed
// subtraction of 1152 leaves c exactly; the value's scale multiplies its
// probabilities. (K through the same conversion was 2 to 3% slower at 2048
// sequences of up to 4095 positions, where instruction issue is the bound.)
//
// Softmax: each warp keeps a reference r per head and takes the powers
// 2^(s - r). Only a tile with a power above kMost (in practice the first one)
// pays for a new reference, a rescale of the sums and its powers again. r lies
// kLift below the largest score met, which places the largest probabilities
// near the top of fp16's range, so that those down to 2^-25 of the largest keep
// 11 bits as operands of the second product; for int8 rows, whose probabilities
// carry the scale of the value, that scale is taken relative to a power of two
// at or above the largest the warp has met. Scores, sums and accumulators are
// fp32.
//
// fp16 rows take the probabilities in two fp16 parts, 21 bits: with one, outputs
// are off by 1.1 to 1.4 times what rounding the exact result to fp16 leaves (1.6
// for single tokens), with two by 1.0. HBM hides the second part (2048 sequences
// of up to 4095 positions, 312 / 315 us with one / two; short ones 1 to 4% slower,
// with more than eight query heads a kv head 5 to 8%). int8 rows take one part:
// half a step of the cached values themselves is up to 2^-8 of a row's largest,
// eight times the rounding of the probabilities, and issue bounds this form (184
// us, with two parts 199).
//
// Rescales and joins go by r itself: past 2^24 kLift no longer comes off
// the maximum exactly. While the largest score is below kFar, an exponent is one
// FMA: the dot product times its factor, exact, minus r. Past that the product
// is rounded first, as it is for the maximum: what that rounding leaves out
// (half a step, 16 at 2^28) would take the largest power out of fp16's range.
//
// Batches of more items than run at once are taken longest first.
//
// Join: the warps of a CTA through shared memory, the CTAs of a cluster through
// distributed shared memory (each takes a slice of the output), clusters
// through the caller's workspace and a second kernel.
//
// Measured (several B200s, of the 6540 GB/s copy rate; all of a read-only
// stream), 14 heads over 2 kv heads of 64, pages of 16, kernel alone at full
// clock: 2048 sequences of 1 to 4095 positions fp16 309 to 315 us (1.05 to 1.07),
// int8 183 to 206 us (0.85 to 0.96); a call, repeated until the power cap acts,
// 312 to 321 and 203 to 219 us (0.80 to 0.87). 29 sequences of 77 to 4093, 32
// heads of 128, int8: 79 to 80 us (0.98), a call 84 to 91. One token over 131072
// positions, fp16: 17.1 to 17.6 us (0.59: about 6 us of dependent first loads and
// joins); over 1001: 5.5 to 6.0.
#include <math.h>

#include "mma.cuh"
#include "paged.cuh"
#include "tcgen05.cuh"  // smem_u32, cluster_sync

namespace kb {
namespace {

constexpr int kWarps = 4;        // of a CTA; 1 in the narrow form
constexpr int kTile = 32;        // positions per warp tile
constexpr int kStages = 2;       // tiles of the cp.async ring (3: fewer resident CTAs, 2 to 3% slower)
constexpr int kMaxGroups = 16;   // query heads per kv head
constexpr int kMaxCluster = 8;   // CTAs that join over distributed shared memory
constexpr int kMaxSplits = 16;   // clusters of one (token, kv head)
constexpr int kCombineWarps = 4;
constexpr int kOrderThreads = 1024, kOrderPer = 8;  // tokens that one CTA puts in order: 8192
constexpr int kOrderWaves = 8;    // a batch of more waves of CTAs is not put in order,
constexpr int kLong = 2048;       // nor one without a sequence of this many positions
constexpr int kPartWaves = 4;     // waves of CTAs up to which long sequences are split,
constexpr int64_t kPart = 4096;   // positions of capacity that a CTA keeps at least then,
constexpr int kPartLeast = 1024;  // and of a sequence
constexpr int64_t kNarrow = 128;  // positions of capacity per wave of CTAs up to which a CTA is one warp
constexpr float kLift = 11.f;      // log2 of the power of the score that sets the reference
constexpr float kMost = 32768.f;   // a larger power moves the reference (fp16 ends at 65504)
constexpr float kFar = 0x1p20f;    // scores (log2 units) from which products are rounded before the reference is taken
constexpr float kUnset = -3.4028235e38f;  // reference of a head that has met no score: every power is infinite

struct PagedAttnArgs {
  const __half* q;
  int64_t q_stride;
  __half* out;
  int64_t out_stride;
  const void* k_pages;
  const void* v_pages;
  const float* k_scales;
  const float* v_scales;
  PagedView view;
  const int32_t* positions;
  const int32_t* seqs;
  int64_t n_tokens;
  int n_heads, groups;
  int cluster;     // CTAs per cluster
  int splits;      // clusters per (token, kv head)
  int parts_shift;  // log2(cluster * splits)
  int min_tiles;   // tiles of a CTA below which a sequence takes fewer clusters
  float* part_o;   // [T, Hq, splits, D], sums of p v against the part's own reference
  float* part_ml;  // [T, Hq, splits, 2] (reference, sum); sum -1: the part met a bad page
  int4* order;     // [T] (token, position, sequence, -), longest first, or NULL
  int32_t* err_flags;
  float scale_log2;  // log2(e) / sqrt(D)
};

// Tiles of each CTA of a sequence of all_tiles: the clusters that have
// min_tiles for each of their CTAs (one at least) share them.
__device__ __forceinline__ int tiles_per_part(const PagedAttnArgs& a, int all_tiles) {
  const int least = a.cluster * a.min_tiles;
  const int clusters = max(1, min(a.splits, (all_tiles + least - 1) / least));
  return (all_tiles + clusters * a.cluster - 1) / (clusters * a.cluster);
}

__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, int src_bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;\n" ::"r"(dst), "l"(src), "r"(src_bytes) : "memory");
}
// Two floats as an fp16 pair, rounded towards zero.
__device__ __forceinline__ uint32_t f2_to_h2_down(float lo, float hi) {
  uint32_t r;
  asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// Transpose of an 8 x 8 fp16 matrix held two elements of a row per lane.
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(r) : "r"(v));
  return r;
}
// c = a * b for one m16n8k16 tile (no registers to clear first).
__device__ __forceinline__ void mma16816_new(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%10,%10,%10,%10};\n"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
// The same of int8, m16n8k32.
__device__ __forceinline__ void mma16832_new(int (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%10,%10,%10,%10};\n"
      : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "r"(0));
}
__device__ __forceinline__ void mma16832(int (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};\n"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The digits h, m, l of four values x = 2^14 h + 2^7 m + l (|x| <= 127 2^14), a
// byte of each digit's register per value.
__device__ __forceinline__ void digits(const float (&x)[4], uint32_t (&w)[3]) {
  w[0] = w[1] = w[2] = 0u;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float h = rintf(x[i] * 0x1p-14f), r = fmaf(h, -0x1p14f, x[i]);
    const float m = rintf(r * 0x1p-7f), l = rintf(fmaf(m, -0x1p7f, r));
    w[0] |= (static_cast<uint32_t>(static_cast<int>(h)) & 0xffu) << (8 * i);
    w[1] |= (static_cast<uint32_t>(static_cast<int>(m)) & 0xffu) << (8 * i);
    w[2] |= (static_cast<uint32_t>(static_cast<int>(l)) & 0xffu) << (8 * i);
  }
}

// Codes of bytes 0 and 2 of `w` as an fp16 pair (bytes 1 and 3: shift by 8).
__device__ __forceinline__ uint32_t codes_h2(uint32_t w) {
  const uint32_t bias = 0x64806480u;  // 1152, 1152
  const uint32_t x = (w & 0x00ff00ffu) ^ bias;
  const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&x), *reinterpret_cast<const __half2*>(&bias));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// Four floats in the shared memory of CTA `rank` of the cluster, at this CTA's
// `local` (16-byte aligned).
__device__ __forceinline__ float4 ld_peer(const float* local, uint32_t rank) {
  uint32_t at;
  float4 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(local)), "r"(rank));
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(at)
               : "memory");
  return v;
}
__device__ __forceinline__ void fma4(float4& acc, float w, float4 x) {
  acc.x = fmaf(w, x.x, acc.x);
  acc.y = fmaf(w, x.y, acc.y);
  acc.z = fmaf(w, x.z, acc.z);
  acc.w = fmaf(w, x.w, acc.w);
}

// Byte offset of 16-byte chunk `ch` of row `r` in a tile of ROW-byte rows; the
// chunk is XOR-ed so that the eight rows of one ldmatrix phase fall in eight
// different bank groups (64-byte rows: two rows share 128 bytes).
template <int ROW>
__device__ __forceinline__ uint32_t swz(int r, int ch) {
  return static_cast<uint32_t>(r * ROW + ((ROW == 64 ? ch ^ ((r >> 1) & 3) : ch ^ (r & 7)) << 4));
}

template <int D, bool I8, int W>
struct Ring {
  static constexpr int kRow = I8 ? D : 2 * D;  // bytes of a cached row
  static constexpr int kTileBytes = kTile * kRow;
  static constexpr int kStageBytes = 2 * kTileBytes + (I8 ? 2 * kTile * 4 : 0);  // K, V, their scales
  static constexpr int kBytes = W * kStages * kStageBytes;
};

// Shared memory of the join, over the idle rings.
template <int D, int NH, int W>
struct Join {
  static constexpr int kHeads = 8 * NH;
  static constexpr int kRedRow = D + 4;  // padded: eight heads' rows spread over the banks
  static constexpr int kBytes = (W * kHeads * (kRedRow + 2) + kHeads * (D + 4)) * 4;
};

// Reference for a largest score x: kLift below it where fp32 has such a number
// to a unit, else the nearest below that it has, or x itself (steps of 16 and
// more; an infinity). The power of x is then at most 2^(kLift + 1).
__device__ __forceinline__ float reference_of(float x) {
  const float r = x - kLift;
  return x - r <= kLift + 1.f ? r : x;
}
// One row's (or part's) share of the joined output: exp2 of its reference against
// the joint one; a part that saw nothing (kUnset) has weight 0 beside any other.
__device__ __forceinline__ float join_weight(float r, float top) { return exp2_approx(r - top); }

// Resident CTAs that the registers are held to: int8 rows of 64 codes have the
// shared memory for five, and want their warps (2048 sequences of up to 4095
// positions, on one GPU: 204 us, with four 215, with six and their spills 230).
constexpr int min_ctas(int head_dim, bool i8, int n_heads_8, int warps) {
  return warps == kWarps && i8 && head_dim == 64 && n_heads_8 == 1 ? 5 : 1;
}

template <int D, bool I8, int NH, int W>
constexpr size_t smem_bytes() {
  return Ring<D, I8, W>::kBytes > Join<D, NH, W>::kBytes ? Ring<D, I8, W>::kBytes : Join<D, NH, W>::kBytes;
}

template <int D, bool I8, int NH, int W>
__global__ void __launch_bounds__(W * 32, min_ctas(D, I8, NH, W))
attn_paged_kernel(const __grid_constant__ PagedAttnArgs a) {
  using R = Ring<D, I8, W>;
  constexpr int kThreads = W * 32;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ int s_bad;
  constexpr int kRow = R::kRow;
  constexpr int kChunks = kRow / 16;
  constexpr int kStep = 32 / kChunks;  // rows the warp's lanes copy at once; divides 8
  constexpr int kM = D / 16;           // m16 tiles of O^T over head_dim, k16 steps of K Q^T
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int gid = lane >> 2, tig = lane & 3;
  const int parts = 1 << a.parts_shift;  // clusters and splits are powers of two
  const unsigned item = blockIdx.x >> a.parts_shift, hkv = a.view.n_kv_heads;
  const int part = blockIdx.x & (parts - 1);
  // a token's heads side by side, neighbours in its pages (90 against 94 us at 29 x 32 heads)
  const unsigned place = item / hkv;
  const int g = static_cast<int>(item - place * hkv);
  const int G = a.groups;
  if (threadIdx.x == 0) s_bad = 0;

  grid_dep_wait();
  grid_dep_launch();
  int64_t t = place;
  int pos, seq;
  if (a.order != nullptr) {
    const int4 e = a.order[place];
    t = e.x;
    pos = e.y;
    seq = e.z;
  } else {
    pos = a.positions[t];
    seq = a.seqs[t];
  }
  const __half* q_t = a.q + t * a.q_stride + static_cast<int64_t>(g) * G * D;
  // int8: four query values a thread and step, on their way while the page
  // table is read
  constexpr int kQuads = 8 * NH * D / 4 / kThreads;
  uint2 raw[I8 ? kQuads : 1];
  if constexpr (I8) {
#pragma unroll
    for (int i = 0; i < kQuads; ++i) {
      const int at = 4 * (threadIdx.x + i * kThreads);
      raw[i] = at < G * D ? *reinterpret_cast<const uint2*>(q_t + at) : make_uint2(0u, 0u);
    }
  }
  __half* out_t = a.out + t * a.out_stride + static_cast<int64_t>(g) * G * D;
  int flag;
  if (token_state(a.view, pos, seq, flag) != kTokenOk) {  // alike in every CTA of the cluster
    if (part == 0) {
      if (threadIdx.x == 0 && g == 0 && flag != 0) set_flag(a.err_flags, flag);
      for (int i = threadIdx.x; i < G * D / 8; i += kThreads) st_plain(out_t + i * 8, make_uint4(0u, 0u, 0u, 0u));
    }
    return;
  }
  const int n = pos + 1;
  const int all_tiles = (n + kTile - 1) / kTile;
  const int per_part = tiles_per_part(a, all_tiles);
  const int cluster_part = part / a.cluster;
  if (cluster_part * a.cluster * per_part >= all_tiles) return;  // nothing left for this cluster
  const int tile0 = min(part * per_part, all_tiles);
  const int n_tiles = min(per_part, all_tiles - tile0);
  const int my_tiles = n_tiles > warp ? (n_tiles - warp + W - 1) / W : 0;

  const int shift = a.view.page_shift, mask = (1 << shift) - 1;
  const int32_t* table = a.view.table + seq * a.view.max_pages;
  unsigned char* ring = smem + warp * (kStages * R::kStageBytes);
  bool bad = false;

  // The page of this lane's position of warp tile i (-1 past the end).
  auto page_of = [&](int i) {
    const int j = (tile0 + warp + i * W) * kTile + lane;
    return i < my_tiles && j < n ? __ldg(table + (j >> shift)) : -1;
  };
  const int lane_row = lane / kChunks, lane_ch = lane % kChunks;
  const char* const k_bytes = static_cast<const char*>(a.k_pages) + lane_row * kRow + lane_ch * 16;
  const char* const v_bytes = static_cast<const char*>(a.v_pages) + lane_row * kRow + lane_ch * 16;
  // Copies warp tile i into stage `st`; rows past the last position are
  // zero-filled, so no stale bits reach the products.
  auto issue = [&](int i, int page, int st) {
    if (i < my_tiles) {
      const int j0 = (tile0 + warp + i * W) * kTile;
      unsigned char* sk = ring + st * R::kStageBytes;
      unsigned char* sv = sk + R::kTileBytes;
      const bool in = j0 + lane < n, fine = page_ok(a.view, page);
      bad |= in && !fine;
      const bool ok = in && fine;
      // row index of this lane's position in K and V (row 0 where there is none)
      const int64_t row =
          ok ? (((static_cast<int64_t>(page) * a.view.n_kv_heads + g) << shift) + ((j0 + lane) & mask)) : 0;
      const unsigned live = __ballot_sync(0xffffffffu, ok);
      if (I8) {
        float* ss = reinterpret_cast<float*>(sv + R::kTileBytes);
        cp_async4(smem_u32(ss + lane), a.k_scales + row, ok ? 4 : 0);
        cp_async4(smem_u32(ss + kTile + lane), a.v_scales + row, ok ? 4 : 0);
      }
      const int64_t row_bytes = row * kRow;
      auto copy = [&](bool all) {
#pragma unroll
        for (int o = 0; o < kTile / 8; ++o) {
          // rows 8 o .. 8 o + 7 follow one another in one page (page 0's first rows where there are none)
          const int64_t off = __shfl_sync(0xffffffffu, row_bytes, 8 * o);
#pragma unroll
          for (int it = 0; it < 8 / kStep; ++it) {
            const int r = 8 * o + it * kStep + lane_row;
            const int bytes = all || (live >> r) & 1 ? 16 : 0;
            cp_async16(smem_u32(sk + swz<kRow>(r, lane_ch)), k_bytes + off + it * kStep * kRow, bytes);
            cp_async16(smem_u32(sv + swz<kRow>(r, lane_ch)), v_bytes + off + it * kStep * kRow, bytes);
          }
        }
      };
      if (live == 0xffffffffu) copy(true); else copy(false);
    }
    cp_async_commit();  // empty groups keep the count uniform
  };

  {
    int first[kStages - 1];
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) first[i] = page_of(i);
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) issue(i, first[i], i);
  }
  int next_page = page_of(kStages - 1);

  // B fragments of Q^T: fp16 pairs, or (int8) the three digits of four dims
  // each, with what takes a head's integer sums back to its scale. The digits
  // are made once per CTA (each warp for itself: 3 us of a CTA's life).
  constexpr int kQ = I8 ? D / 32 : kM;  // k steps of K Q^T
  uint32_t qb[NH][kQ][2][I8 ? 3 : 1];
  float unit[NH][2];
  if constexpr (!I8) {
#pragma unroll
    for (int h = 0; h < NH; ++h) {
      const int head = h * 8 + gid;
      const __half* qh = q_t + (head < G ? head : 0) * D;
#pragma unroll
      for (int ks = 0; ks < kQ; ++ks) {
        qb[h][ks][0][0] = head < G ? *reinterpret_cast<const uint32_t*>(qh + ks * 16 + 2 * tig) : 0u;
        qb[h][ks][1][0] = head < G ? *reinterpret_cast<const uint32_t*>(qh + ks * 16 + 2 * tig + 8) : 0u;
      }
    }
  } else {
    __shared__ uint32_t s_digits[3][8 * NH * D / 4];
    __shared__ float s_unit[8 * NH];
#pragma unroll
    for (int i = 0; i < kQuads; ++i) {
      const int quad = threadIdx.x + i * kThreads;  // D / 4 lanes of a warp hold a head
      if (4 * (warp * 32 + i * kThreads) >= G * D) {  // no head in this warp's: one head per kv head leaves 7 of 8 out
        for (int d = 0; d < 3; ++d) s_digits[d][quad] = 0u;
        if (quad % (D / 4) == 0) s_unit[quad / (D / 4)] = 0.f;
        continue;
      }
      const float2 x = h2_to_f2(raw[i].x), y = h2_to_f2(raw[i].y);
      float qmax = max_nan(max_nan(fabsf(x.x), fabsf(x.y)), max_nan(fabsf(y.x), fabsf(y.y)));
#pragma unroll
      for (int d = D / 8; d > 0; d >>= 1) qmax = max_nan(qmax, __shfl_xor_sync(0xffffffffu, qmax, d));
      const float inv = qmax > 0.f ? 2080768.f / qmax : 0.f;  // 127 * 2^14
      const float v[4] = {x.x * inv, x.y * inv, y.x * inv, y.y * inv};
      uint32_t w[3];
      digits(v, w);
#pragma unroll
      for (int d = 0; d < 3; ++d) s_digits[d][quad] = w[d];
      // an infinite or NaN query makes the unit, and with it every score, NaN
      if (quad % (D / 4) == 0) {
        s_unit[quad / (D / 4)] =
            qmax * (a.scale_log2 / 2080768.f) * (qmax <= 65504.f ? 1.f : __int_as_float(0x7fffffff));
      }
    }
    __syncthreads();
#pragma unroll
    for (int h = 0; h < NH; ++h) {
#pragma unroll
      for (int ks = 0; ks < kQ; ++ks) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
          for (int d = 0; d < 3; ++d) qb[h][ks][e][d] = s_digits[d][(h * 8 + gid) * (D / 4) + ks * 8 + 4 * e + tig];
        }
      }
      // the heads of this lane's scores are 2 tig and 2 tig + 1
      unit[h][0] = s_unit[h * 8 + 2 * tig];
      unit[h][1] = s_unit[h * 8 + 2 * tig + 1];
    }
  }

  float o[NH][kM][4];
  // ref: the heads' references. Before the first tile every power is infinite,
  // which makes that tile set them.
  float ref[NH][2], l[NH][2];
  bool far = false;  // some head of the warp has met a score of kFar
#pragma unroll
  for (int h = 0; h < NH; ++h) {
    ref[h][0] = ref[h][1] = kUnset;
    l[h][0] = l[h][1] = 0.f;
#pragma unroll
    for (int i = 0; i < kM; ++i) o[h][i][0] = o[h][i][1] = o[h][i][2] = o[h][i][3] = 0.f;
  }
  float vref = 0.f, inv_vref = 0.f;  // int8: power of two at or above the value scales met
  const float sl2 = a.scale_log2;

  int st = 0, st_in = kStages - 1;  // stage of tile i, and of the tile issued beside it
  for (int i = 0; i < my_tiles; ++i) {
    issue(i + kStages - 1, next_page, st_in);
    next_page = page_of(i + kStages);
    cp_async_wait<kStages - 1>();
    __syncwarp();
    const int j0 = (tile0 + warp + i * W) * kTile;
    const unsigned char* sk = ring + st * R::kStageBytes;
    const unsigned char* sv = sk + R::kTileBytes;
    const float* ss = reinterpret_cast<const float*>(sv + R::kTileBytes);
    st_in = st;
    st = st + 1 == kStages ? 0 : st + 1;

    // S^T: two m16 tiles of positions x NH n8 tiles of heads; element e belongs
    // to position gid + 8 (e >> 1), head 2 tig + (e & 1)
    float s[2][NH][4];
    float f[2][2];  // what takes a position's scores to log2 units
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
      if constexpr (!I8) {
#pragma unroll
        for (int ks = 0; ks < kQ; ++ks) {
          uint32_t b[4];
          ldsm_x4(b, smem_u32(sk + swz<kRow>(mt * 16 + (lane & 15), 2 * ks + (lane >> 4))));
#pragma unroll
          for (int h = 0; h < NH; ++h) {
            if (ks == 0) mma16816_new(s[mt][h], b, qb[h][ks][0][0], qb[h][ks][1][0]);
            else mma16816(s[mt][h], b, qb[h][ks][0][0], qb[h][ks][1][0]);
          }
        }
        f[mt][0] = f[mt][1] = sl2;
      } else {
        int c[NH][3][4];
#pragma unroll
        for (int ks = 0; ks < kQ; ++ks) {
          uint32_t b[4];
          ldsm_x4(b, smem_u32(sk + swz<kRow>(mt * 16 + (lane & 15), 2 * ks + (lane >> 4))));
#pragma unroll
          for (int h = 0; h < NH; ++h) {
#pragma unroll
            for (int d = 0; d < 3; ++d) {
              if (ks == 0) mma16832_new(c[h][d], b, qb[h][ks][0][d], qb[h][ks][1][d]);
              else mma16832(c[h][d], b, qb[h][ks][0][d], qb[h][ks][1][d]);
            }
          }
        }
#pragma unroll
        for (int h = 0; h < NH; ++h) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            // the first digit's sum stays below 2^21, the others' together below 2^28
            const float low = static_cast<float>(c[h][1][e] * 128 + c[h][2][e]);
            s[mt][h][e] = fmaf(static_cast<float>(c[h][0][e]), 0x1p14f, low) * unit[h][e & 1];
          }
        }
        f[mt][0] = ss[mt * 16 + gid];
        f[mt][1] = ss[mt * 16 + gid + 8];
      }
    }
    float p[2][NH][4];
    const bool last = j0 + kTile > n;
    // the scores as rounded products
    auto round_scores = [&]() {
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
        for (int h = 0; h < NH; ++h) {
#pragma unroll
          for (int e = 0; e < 4; ++e) s[mt][h][e] = __fmul_rn(s[mt][h][e], f[mt][e >> 1]);
        }
        f[mt][0] = f[mt][1] = 1.f;
      }
    };
    if (far) round_scores();
    auto powers = [&]() {
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
        for (int h = 0; h < NH; ++h) {
#pragma unroll
          for (int e = 0; e < 4; ++e) p[mt][h][e] = exp2_approx(fmaf(s[mt][h][e], f[mt][e >> 1], -ref[h][e & 1]));
        }
      }
      if (last) {
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if (j0 + mt * 16 + gid + 8 * (e >> 1) >= n) {
#pragma unroll
              for (int h = 0; h < NH; ++h) p[mt][h][e] = 0.f;
            }
          }
        }
      }
    };
    powers();
    float most = 0.f;
#pragma unroll
    for (int h = 0; h < NH; ++h) {
#pragma unroll
      for (int e = 0; e < 4; ++e) most = fmaxf(most, fmaxf(p[0][h][e], p[1][h][e]));
    }
    float vs = 0.f;
    bool over = most > kMost;
    if (I8) {
      vs = fabsf(ss[kTile + lane]);
      over |= vs > vref;
    }
    if (__any_sync(0xffffffffu, over)) {
      float ratio = 1.f;
      if (I8) {
        // the power of two above the largest scale of the tile (a NaN scale
        // never compares and poisons the probabilities by itself)
        const unsigned bits = __reduce_max_sync(0xffffffffu, vs <= 3.4028235e38f ? __float_as_uint(vs) : 0u);
        const float up = __uint_as_float(min((bits >> 23) + 1u, 0xfeu) << 23);
        if (bits != 0u && up > vref) {
          ratio = vref / up;
          vref = up;
          inv_vref = 1.f / up;
        }
      }
      float top[NH][2];
      bool high = false;
#pragma unroll
      for (int h = 0; h < NH; ++h) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float x = -INFINITY;
#pragma unroll
          for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              if (j0 + mt * 16 + gid + 8 * half < n) x = fmaxf(x, __fmul_rn(s[mt][h][2 * half + e], f[mt][half]));
            }
          }
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
          top[h][e] = x;
          high |= fabsf(x) >= kFar && x != -INFINITY;
        }
      }
      if (!far && __any_sync(0xffffffffu, high)) {
        far = true;
        round_scores();
      }
#pragma unroll
      for (int h = 0; h < NH; ++h) {
        float cr[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float r = fmaxf(ref[h][e], reference_of(top[h][e]));  // all scores -inf so far: still unset
          cr[e] = exp2_approx(ref[h][e] - r);
          ref[h][e] = r;
          l[h][e] *= cr[e];
          cr[e] *= ratio;
        }
#pragma unroll
        for (int k = 0; k < kM; ++k) {
          o[h][k][0] *= cr[0];
          o[h][k][1] *= cr[1];
          o[h][k][2] *= cr[0];
          o[h][k][3] *= cr[1];
        }
      }
      powers();
    }
    // O^T += V^T P^T, for 16 positions at a time. P^T as B fragments is the
    // transpose of each 8 x 8 block: for int8 rows the powers rounded to fp16; for
    // fp16 rows [h][0..1] the powers rounded towards zero and [h][2..3] what that
    // left, 2^-24 (fp16's smallest, 2^-35 of the largest power) at least: neither
    // negative nor zero, so that an infinite value stays that infinity. fp16: m tile
    // k holds dims 16 k + gid, + 8; int8: dims 16 k + 2 gid, 2 gid + 1 (the two codes
    // of the 16-bit units transposed)
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
      uint32_t pb[NH][I8 ? 2 : 4];
      float v0 = 1.f, v1 = 1.f;
      if (I8) {
        v0 = ss[kTile + mt * 16 + gid] * inv_vref;
        v1 = ss[kTile + mt * 16 + gid + 8] * inv_vref;
      }
#pragma unroll
      for (int h = 0; h < NH; ++h) {
        l[h][0] += p[mt][h][0] + p[mt][h][2];
        l[h][1] += p[mt][h][1] + p[mt][h][3];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const float v = half == 0 ? v0 : v1;
          const float x = p[mt][h][2 * half] * v, y = p[mt][h][2 * half + 1] * v;
          if constexpr (I8) {
            pb[h][half] = transpose8x8(f2_to_h2(x, y));
          } else {
            const uint32_t most_of = f2_to_h2_down(x, y);
            const float2 kept = h2_to_f2(most_of);
            pb[h][half] = transpose8x8(most_of);
            pb[h][2 + half] = transpose8x8(f2_to_h2(fmaxf(x - kept.x, 0x1p-24f), fmaxf(y - kept.y, 0x1p-24f)));
          }
        }
      }
      const int mtx = lane >> 3;
#pragma unroll
      for (int kp = 0; kp < (I8 ? kM / 2 : kM); ++kp) {
        uint32_t b[4];
        if constexpr (!I8) {
          ldsm_x4_trans(b, smem_u32(sv + swz<kRow>(mt * 16 + 8 * (mtx >> 1) + (lane & 7), 2 * kp + (mtx & 1))));
#pragma unroll
          for (int h = 0; h < NH; ++h) {
            mma16816(o[h][kp], b, pb[h][0], pb[h][1]);
            mma16816(o[h][kp], b, pb[h][2], pb[h][3]);
          }
        } else {
          ldsm_x4_trans(b, smem_u32(sv + swz<kRow>(mt * 16 + 8 * (mtx & 1) + (lane & 7), 2 * kp + (mtx >> 1))));
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const uint32_t codes[4] = {codes_h2(b[2 * e]), codes_h2(b[2 * e] >> 8), codes_h2(b[2 * e + 1]),
                                       codes_h2(b[2 * e + 1] >> 8)};
#pragma unroll
            for (int h = 0; h < NH; ++h) mma16816(o[h][2 * kp + e], codes, pb[h][0], pb[h][1]);
          }
        }
      }
    }
    __syncwarp();  // the stage is refilled by the next iteration's issue
  }
  cp_async_wait<0>();

  // join the warps; a head's sum is spread over the eight lanes of its column
#pragma unroll
  for (int h = 0; h < NH; ++h) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) l[h][e] += __shfl_xor_sync(0xffffffffu, l[h][e], x);
    }
  }
  __syncthreads();  // s_bad is initialised and every ring is idle: the rings hold the join
  if (__any_sync(0xffffffffu, bad) && lane == 0) s_bad = 1;
  using J = Join<D, NH, W>;
  float* red_o = reinterpret_cast<float*>(smem);
  float* red_ml = red_o + W * J::kHeads * J::kRedRow;
  float* cta_o = red_ml + W * J::kHeads * 2;  // [heads][D]
  float* cta_ml = cta_o + J::kHeads * D;           // [heads][4]: reference, sum, the bad mark
  const float back = I8 ? vref : 1.f;
#pragma unroll
  for (int h = 0; h < NH; ++h) {
#pragma unroll
    for (int k = 0; k < kM; ++k) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int head = h * 8 + 2 * tig + (e & 1);
        const int d = 16 * k + (I8 ? 2 * gid + (e >> 1) : gid + 8 * (e >> 1));
        red_o[(warp * J::kHeads + head) * J::kRedRow + d] = o[h][k][e] * back;
      }
    }
    if (gid == 0) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        red_ml[(warp * J::kHeads + h * 8 + 2 * tig + e) * 2] = ref[h][e];
        red_ml[(warp * J::kHeads + h * 8 + 2 * tig + e) * 2 + 1] = l[h][e];
      }
    }
  }
  __syncthreads();
  bool any_bad = s_bad != 0;
  if (any_bad && threadIdx.x == 0 && g == 0) set_flag(a.err_flags, KLLM_B200_FLAG_BAD_PAGE);
  // Four dims of head `head` over this cluster's positions: of the output itself, or its share of it.
  const bool whole = per_part * a.cluster >= all_tiles;
  auto finish = [&](int head, int d, float4 acc, float top, float sum) {
    if (whole) {
      uint2 v;
      v.x = f2_to_h2(any_bad ? 0.f : acc.x / sum, any_bad ? 0.f : acc.y / sum);
      v.y = f2_to_h2(any_bad ? 0.f : acc.z / sum, any_bad ? 0.f : acc.w / sum);
      *reinterpret_cast<uint2*>(out_t + head * D + d) = v;
    } else {
      const int64_t prow = (t * a.n_heads + static_cast<int64_t>(g) * G + head) * a.splits + cluster_part;
      *reinterpret_cast<float4*>(a.part_o + prow * D + d) = acc;
      if (d == 0) {
        a.part_ml[prow * 2] = top;
        a.part_ml[prow * 2 + 1] = any_bad ? -1.f : sum;
      }
    }
  };
  for (int quad = threadIdx.x; quad < G * D / 4; quad += kThreads) {
    const int head = quad / (D / 4), d = quad % (D / 4) * 4;
    float2 ml[W];
    float4 x[W];
    float M = kUnset;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      ml[w] = *reinterpret_cast<const float2*>(red_ml + (w * J::kHeads + head) * 2);
      x[w] = *reinterpret_cast<const float4*>(red_o + (w * J::kHeads + head) * J::kRedRow + d);
      M = fmaxf(M, ml[w].x);
    }
    float L = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float f = join_weight(ml[w].x, M);  // a warp without tiles holds zeros and weight 0
      L = fmaf(f, ml[w].y, L);
      fma4(acc, f, x[w]);
    }
    if (a.cluster == 1) {
      finish(head, d, acc, M, L);
    } else {
      *reinterpret_cast<float4*>(cta_o + head * D + d) = acc;
      if (d == 0) *reinterpret_cast<float4*>(cta_ml + 4 * head) = make_float4(M, L, any_bad ? 1.f : 0.f, 0.f);
    }
  }
  if (a.cluster == 1) return;
  cluster_sync();
  const int rank = part & (a.cluster - 1);
  for (int quad = threadIdx.x * a.cluster + rank; quad < G * D / 4; quad += a.cluster * kThreads) {
    const int head = quad / (D / 4), d = quad % (D / 4) * 4;
    float4 ml[kMaxCluster], x[kMaxCluster];
#pragma unroll
    for (int c = 0; c < kMaxCluster; ++c) {
      ml[c] = c < a.cluster ? ld_peer(cta_ml + 4 * head, c) : make_float4(kUnset, 0.f, 0.f, 0.f);
      x[c] = c < a.cluster ? ld_peer(cta_o + head * D + d, c) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    float M = kUnset, L = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int c = 0; c < kMaxCluster; ++c) {
      M = fmaxf(M, ml[c].x);
      any_bad |= ml[c].z != 0.f;
    }
#pragma unroll
    for (int c = 0; c < kMaxCluster; ++c) {
      const float f = join_weight(ml[c].x, M);
      L = fmaf(f, ml[c].y, L);
      fma4(acc, f, x[c]);
    }
    finish(head, d, acc, M, L);
  }
  cluster_sync();  // no CTA leaves while its shared memory may be read
}

// One warp per (token, query head) that has several parts. Always launched with
// programmatic dependent launch: positions and sequences are read before the
// wait (the attention kernel lets dependents start only after its own wait, so
// whatever wrote them is done), the parts after it, all at once.
template <int D>
__global__ void __launch_bounds__(kCombineWarps * 32) attn_paged_combine_kernel(const __grid_constant__ PagedAttnArgs a) {
  constexpr int kPer = D / 32;
  const int lane = threadIdx.x & 31;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kCombineWarps + (threadIdx.x >> 5);
  int used = 0;
  if (row < a.n_tokens * a.n_heads) {
    const int64_t t = row / a.n_heads;
    const int pos = a.positions[t], seq = a.seqs[t];
    int flag;
    if (token_state(a.view, pos, seq, flag) == kTokenOk) {
      const int all_tiles = (pos + kTile) / kTile;
      const int per_cluster = tiles_per_part(a, all_tiles) * a.cluster;
      used = (all_tiles + per_cluster - 1) / per_cluster;
    }
  }
  grid_dep_wait();
  grid_dep_launch();
  if (used <= 1) return;  // written by the attention kernel
  // lane c holds part c's reference and sum; its weight goes to all by shuffles
  const float* ml = a.part_ml + row * a.splits * 2;
  const float* po = a.part_o + row * a.splits * D + lane * kPer;
  float pm = kUnset, pl = 0.f;
  if (lane < used) {
    pm = ml[2 * lane];
    pl = ml[2 * lane + 1];
  }
  float x[kMaxSplits][kPer];
#pragma unroll
  for (int c = 0; c < kMaxSplits; ++c) {
#pragma unroll
    for (int k = 0; k < kPer; ++k) x[c][k] = c < used ? po[c * D + k] : 0.f;
  }
  const bool bad = __any_sync(0xffffffffu, pl == -1.f);
  float M = pm;
#pragma unroll
  for (int i = 16; i > 0; i >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, i));
  const float weight = join_weight(pm, M);
  const float L = group_sum<32>(weight * pl);
  float acc[kPer];
#pragma unroll
  for (int k = 0; k < kPer; ++k) acc[k] = 0.f;
#pragma unroll
  for (int c = 0; c < kMaxSplits; ++c) {
    const float w = __shfl_sync(0xffffffffu, weight, c);
#pragma unroll
    for (int k = 0; k < kPer; ++k) acc[k] += w * x[c][k];
  }
  const int64_t t = row / a.n_heads;
  __half* dst = a.out + t * a.out_stride + (row - t * a.n_heads) * D + lane * kPer;
#pragma unroll
  for (int k = 0; k < kPer; ++k) dst[k] = __float2half_rn(bad ? 0.f : acc[k] / L);
}

// Class of a length >= 1, longest first: eighths of octaves, by the top bits of
// its float (exponent and three bits, 1016 for 1).
__host__ __device__ constexpr int length_class(uint32_t float_bits) {
  return 255 - (static_cast<int>(float_bits >> 20) - 1016);
}

// Tokens, longest first, for grids of more CTAs than run at once: CTAs start in
// the order of their index, so the last ones to start are the shortest and the
// device stays full to the end. A counting sort by one CTA; the order within a
// class is the atomics', which no output depends on. Costs 2 to 3 us (one more
// with a match of the warp's classes before each atomic). Without / with, us,
// lengths of 1 to 4095: 29 sequences of 32 kv heads of 128, int8 90 / 79; 14
// over 2 heads of 64, 600 sequences fp16 99 / 95, int8 72 / 61; 2048 int8
// 201-215 / 182-186 (6 waves), fp16 312 / 310 (9 waves, not put in order); 4096
// (11 waves) int8 411 / 409. Lengths below kLong keep their order: 2048
// sequences of up to 1023, fp16, 86 without this kernel, 90 with it, 96 sorted,
// when the short ones, which latency bounds, come together at the end.
__global__ void __launch_bounds__(kOrderThreads) attn_paged_order_kernel(const __grid_constant__ PagedAttnArgs a) {
  __shared__ int s_first[256];
  const int lane = threadIdx.x & 31;
  if (threadIdx.x < 256) s_first[threadIdx.x] = 0;
  grid_dep_wait();
  grid_dep_launch();
  int pos[kOrderPer], seq[kOrderPer], cls[kOrderPer], at[kOrderPer];
  const int n = static_cast<int>(a.n_tokens);
#pragma unroll
  for (int u = 0; u < kOrderPer; ++u) {
    const int t = threadIdx.x + u * kOrderThreads;
    cls[u] = -1;
    if (t < n) {
      pos[u] = a.positions[t];
      seq[u] = a.seqs[t];
      const bool real = pos[u] >= 0 && pos[u] < a.view.capacity;  // others are done at once
      cls[u] = real ? length_class(__float_as_uint(static_cast<float>(pos[u] + 1))) : 255;
    }
  }
  __syncthreads();
#pragma unroll
  for (int u = 0; u < kOrderPer; ++u) {
    if (u * kOrderThreads >= n) break;
    const int front = __shfl_sync(0xffffffffu, cls[u], 0);  // by all lanes, before any condition on their class
    if (__all_sync(0xffffffffu, front >= 0 && cls[u] == front)) {
      const int base = lane == 0 ? atomicAdd(&s_first[cls[u]], 32) : 0;  // equal lengths: one atomic, not 32 in turn
      at[u] = __shfl_sync(0xffffffffu, base, 0) + lane;
    } else if (cls[u] >= 0) {
      at[u] = atomicAdd(&s_first[cls[u]], 1);
    }
  }
  __syncthreads();
  if (threadIdx.x < 32) {  // counts to first places
    int c[8], sum = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      c[i] = sum;
      sum += s_first[8 * lane + i];
    }
    int before = sum;
#pragma unroll
    for (int m = 1; m < 32; m *= 2) {
      const int x = __shfl_up_sync(0xffffffffu, before, m);
      if (lane >= m) before += x;
    }
    before -= sum;
#pragma unroll
    for (int i = 0; i < 8; ++i) s_first[8 * lane + i] = before + c[i];
  }
  __syncthreads();
  constexpr int kLongClass = length_class(0x45000000u);  // of 2048.f
  static_assert(kLong == 2048, "its float is written above");
  const bool sort = s_first[kLongClass + 1] > 0;  // tokens of kLong positions or more
#pragma unroll
  for (int u = 0; u < kOrderPer; ++u) {
    const int t = threadIdx.x + u * kOrderThreads;
    if (t < n) a.order[sort ? s_first[cls[u]] + at[u] : t] = make_int4(t, pos[u], seq[u], 0);
  }
}

int check_heads(const char* what, int64_t n_tokens, int64_t n_heads, int64_t hkv) {
  if (n_tokens < 0 || n_heads < 0) return fail(KLLM_B200_ERR_INVALID_ARG, "%s: negative size", what);
  if (n_heads == 0 || n_heads % hkv != 0) {
    return fail(KLLM_B200_ERR_SHAPE, "%s: %lld query heads not a positive multiple of %lld kv heads", what,
                (long long)n_heads, (long long)hkv);
  }
  if (n_heads / hkv > kMaxGroups) {
    return fail(KLLM_B200_ERR_SHAPE, "%s: more than %d query heads per kv head", what, kMaxGroups);
  }
  // a CTA per (token, kv head) at least, all parts of few
  if (n_tokens > 0x7fffffffLL / (kMaxSplits * kMaxCluster) || n_tokens * hkv > 0x7fffffffLL) {
    return fail(KLLM_B200_ERR_SHAPE, "%s: too many tokens", what);
  }
  return KLLM_B200_OK;
}

// Batches of one wave at most over long caches are split further than fits at
// once, while a CTA keeps kPart positions of the capacity: padded rows and short
// sequences then leave no slot idle, and the longest ones are shared. A sequence
// takes the clusters that have kPartLeast positions for each of their CTAs.
// Measured, us, without / with: int8, 40/8 x 128, 2 sequences of 51 and 91
// thousand and 5 padded rows 147 / 61; 6/6 x 64, 4 of 63 to 100 thousand and 5
// padded rows 79 / 55; 16/1 x 64, 94 of 51 to 67 thousand 245 / 190; 14/2 x 64,
// 64 of 100 to 32768 79 / 70; fp16, 14/2 x 64, 64 of 32768 each 158 / 163.
//
// Narrow: many short items are bound by a CTA's fixed 3 to 5 us (dependent first
// loads, the join), so there a CTA is one warp, with a quarter of the shared
// memory and more than twice to seven times the CTAs per SM. By waves of the
// four-warp form: the longer the sequences may be, the more waves it takes
// until the device stays full to the end without several warps per item. The
// rule (items * kNarrow >= capacity * CTAs of a wave) goes by these sizes; at its
// edge one warp is the slower by up to 3% (2000 items of 512, 16000 of 2048), and
// past a capacity of 2048 it stands unmeasured.
// Measured, us, four warps / one, lengths of a quarter to all of the capacity:
//                          capacity 32      128         512         1024        2048
//   fp16 14/2 x 64    2000 items 14 / 8     17 / 11     32 / 33     55 / 59     100 / 109
//                    16000      109 / 39   121 / 61    215 / 198   383 / 383    741 / 750
//   fp16 32/32 x 128  1984       35 / 9     42 / 18     70 / 52    111 / 100    192 / 192
//                    16000      298 / 58   314 / 102   535 / 361   832 / 715   1514 / 1421
//   int8 32/32 x 128  1984       25 / 17    27 / 22     44 / 41     64 / 73     107 / 128
//                    16000      163 / 91   186 / 128   304 / 235   440 / 398    766 / 779
//
// How the positions of a (token, kv head) are dealt out, by sizes the host
// knows: the largest cluster of which the device holds one for every item at
// once, and, where the largest leaves room, several clusters per item while a
// CTA's share of the capacity stays at 256 positions or more. A CTA costs about 6 us
// of one slot beside its rows (positions, page table and first rows are read
// one after another, and its parts are joined), so items that fill the device
// by themselves are not split. Measured, us, clusters of 1 / 2 / 4 / 8 for
// sequences of up to 4095 positions, 14 heads over 2 kv heads of 64:
//   int8   8 sequences  23.4 / 16.2 / 10.9 /  9.4;   64: 27.8 / 20.8 / 17.9 / 22.8
//   fp16 128 sequences  31.1 / 30.6 / 31.5 / 46.0;  512: 87.4 / 88.0 / 100  / 166
struct Split {
  int cluster, splits;
  bool order, narrow;
  int min_tiles;
};

template <int D, bool I8, int NH>
Split split_of(int64_t n_tokens, int64_t hkv, int64_t capacity) {
  const int64_t items = n_tokens * hkv;
  const void* kernel = reinterpret_cast<const void*>(attn_paged_kernel<D, I8, NH, kWarps>);
  constexpr int kThreads = kWarps * 32;
  constexpr size_t smem = smem_bytes<D, I8, NH, kWarps>();
  Split x = {1, 1, false, false, 1};
  (void)allow_smem(kernel, smem);  // occupancy is asked for with the opt-in in place
  for (int c = kMaxCluster; c > 1; c /= 2) {
    if (capacity < c * kWarps * kTile) continue;
    const int fit = active_clusters_raw(kernel, kThreads, smem, c);
    if (fit < items) continue;
    x.cluster = c;
    while (c == kMaxCluster && x.splits < kMaxSplits && items * x.splits * 2 <= fit &&
           capacity >= int64_t{KLLM_B200_PAGED_SPLIT_MIN} * x.splits) {  // 512 positions of each of 8 CTAs
      x.splits *= 2;
    }
    break;
  }
  // more than one wave, few enough that its last one counts
  const int64_t slots = static_cast<int64_t>(sm_count()) * resident_ctas_raw(kernel, kThreads, smem);
  while (items <= slots && x.splits < kMaxSplits && items * x.cluster * x.splits * 2 <= kPartWaves * slots &&
         capacity >= 2 * kPart * x.cluster * x.splits) {
    x.splits *= 2;
    x.min_tiles = kPartLeast / kTile;
  }
  x.order = x.cluster == 1 && x.splits == 1 && items > slots && items <= kOrderWaves * slots && n_tokens > 1 &&
            n_tokens <= kOrderThreads * kOrderPer && capacity >= KLLM_B200_PAGED_SPLIT_MIN;
  x.narrow = x.cluster == 1 && x.splits == 1 && items > slots && items * kNarrow >= capacity * slots;
  return x;
}

Split preferred_split(int64_t n_tokens, int64_t n_heads, const PagedView& view, int64_t head_dim, bool i8) {
  const auto pick = [&](auto narrow, auto wide) {
    return (n_heads / view.n_kv_heads <= 8 ? narrow : wide)(n_tokens, view.n_kv_heads, view.capacity);
  };
  if (head_dim == 64) {
    return i8 ? pick(split_of<64, true, 1>, split_of<64, true, 2>) : pick(split_of<64, false, 1>, split_of<64, false, 2>);
  }
  return i8 ? pick(split_of<128, true, 1>, split_of<128, true, 2>)
            : pick(split_of<128, false, 1>, split_of<128, false, 2>);
}

// The workspace: parts to join, or the order of the tokens; never both.
int64_t workspace_for(int64_t n_tokens, int64_t n_heads, int64_t head_dim, const Split& split) {
  if (split.order) return n_tokens * static_cast<int64_t>(sizeof(int4));
  return split.splits <= 1 ? 0 : n_tokens * n_heads * split.splits * (head_dim + 2) * static_cast<int64_t>(sizeof(float));
}

template <int D, bool I8, int NH, int W>
int launch_attention(const PagedAttnArgs& a, const LaunchOpts& o) {
  const char* what = "attention_paged";
  constexpr int kThreads = W * 32;
  constexpr size_t smem = smem_bytes<D, I8, NH, W>();
  auto kernel = attn_paged_kernel<D, I8, NH, W>;
  cudaError_t err = allow_smem(reinterpret_cast<const void*>(kernel), smem);
  if (err != cudaSuccess) return launch_status(err, "attention_paged: shared memory opt-in");
  const dim3 grid(static_cast<unsigned>(a.n_tokens * a.view.n_kv_heads * a.splits * a.cluster));
  if (a.order != nullptr) {
    err = launch(attn_paged_order_kernel, dim3(1), dim3(kOrderThreads), 0, o.stream, o.pdl, a);
    if (err != cudaSuccess) return launch_status(err, what);
  }
  err = a.cluster == 1 ? launch(kernel, grid, dim3(kThreads), smem, o.stream, o.pdl || a.order != nullptr, a)
                       : launch_clustered(kernel, grid, dim3(kThreads), smem, o.stream, o.pdl, a.cluster, a);
  const int rc = launch_status(err, what);
  if (rc != KLLM_B200_OK || a.splits == 1) return rc;
  const int64_t rows = a.n_tokens * a.n_heads;
  const dim3 cgrid(static_cast<unsigned>((rows + kCombineWarps - 1) / kCombineWarps));
  return launch_status(launch(attn_paged_combine_kernel<D>, cgrid, dim3(kCombineWarps * 32), 0, o.stream, true, a), what);
}

template <int D, bool I8>
int launch_groups(const PagedAttnArgs& a, bool narrow, const LaunchOpts& o) {
  if (narrow) return a.groups <= 8 ? launch_attention<D, I8, 1, 1>(a, o) : launch_attention<D, I8, 2, 1>(a, o);
  return a.groups <= 8 ? launch_attention<D, I8, 1, kWarps>(a, o) : launch_attention<D, I8, 2, kWarps>(a, o);
}

}  // namespace

int attention_paged_workspace_bytes(int64_t n_tokens, int64_t n_heads, const kllm_b200_paged_cache* cache,
                                    int64_t* bytes) {
  const char* what = "attention_paged_workspace_bytes";
  if (!bytes) return fail(KLLM_B200_ERR_INVALID_ARG, "%s: null pointer", what);
  *bytes = 0;
  PagedView view;
  int rc = paged_view(cache, what, &view);
  if (rc == KLLM_B200_OK) rc = check_heads(what, n_tokens, n_heads, view.n_kv_heads);
  if (rc != KLLM_B200_OK || n_tokens == 0) return rc;
  *bytes = workspace_for(n_tokens, n_heads, cache->head_dim,
                         preferred_split(n_tokens, n_heads, view, cache->head_dim, cache->cache_dtype == KLLM_B200_I8));
  return KLLM_B200_OK;
}

int attention_paged(const void* q, int64_t q_stride, const kllm_b200_paged_cache* cache, const int32_t* positions,
                    const int32_t* seqs, int64_t n_tokens, int64_t n_heads, void* out, int64_t out_stride,
                    void* workspace, int64_t workspace_bytes, int32_t* err_flags, const LaunchOpts& o) {
  const char* what = "attention_paged";
  PagedAttnArgs a = {};
  int rc = paged_view(cache, what, &a.view);
  if (rc == KLLM_B200_OK) rc = check_heads(what, n_tokens, n_heads, a.view.n_kv_heads);
  if (rc != KLLM_B200_OK || n_tokens == 0) return rc;
  if (!q || !out || !positions || !seqs) return fail(KLLM_B200_ERR_INVALID_ARG, "%s: null pointer", what);
  const int64_t D = cache->head_dim;
  if (q_stride < n_heads * D || out_stride < n_heads * D) {
    return fail(KLLM_B200_ERR_SHAPE, "%s: a token stride is shorter than the token's row", what);
  }
  if ((q_stride | out_stride) % 8 != 0 || !aligned16(q) || !aligned16(out)) {
    return fail(KLLM_B200_ERR_ALIGN, "%s: q and out must be 16-byte aligned, their strides multiples of 8 elements",
                what);
  }
  if (workspace_bytes < 0) return fail(KLLM_B200_ERR_INVALID_ARG, "%s: negative workspace size", what);
  if (workspace_bytes > 0 && (!workspace || !aligned16(workspace))) {
    return fail(KLLM_B200_ERR_ALIGN, "%s: workspace must be non-null and 16-byte aligned", what);
  }
  if (q == out) return fail(KLLM_B200_ERR_INVALID_ARG, "%s: out must not overlap q", what);
  Split split = preferred_split(n_tokens, n_heads, a.view, D, cache->cache_dtype == KLLM_B200_I8);
  const auto fits = [&] { return workspace_for(n_tokens, n_heads, D, split) <= (workspace ? workspace_bytes : 0); };
  if (split.order && !fits()) split.order = false;
  while (!fits()) split.splits /= 2;
  a.q = static_cast<const __half*>(q);
  a.q_stride = q_stride;
  a.out = static_cast<__half*>(out);
  a.out_stride = out_stride;
  a.k_pages = cache->k_pages;
  a.v_pages = cache->v_pages;
  a.k_scales = cache->k_scales;
  a.v_scales = cache->v_scales;
  a.positions = positions;
  a.seqs = seqs;
  a.n_tokens = n_tokens;
  a.n_heads = static_cast<int>(n_heads);
  a.groups = static_cast<int>(n_heads / a.view.n_kv_heads);
  a.cluster = split.cluster;
  a.splits = split.splits;
  a.min_tiles = split.min_tiles;
  while ((1 << a.parts_shift) < a.cluster * a.splits) ++a.parts_shift;
  a.err_flags = err_flags;
  a.scale_log2 = 1.4426950408889634f / sqrtf(static_cast<float>(D));
  if (split.order) a.order = static_cast<int4*>(workspace);
  if (split.splits > 1) {
    a.part_o = static_cast<float*>(workspace);
    a.part_ml = a.part_o + n_tokens * n_heads * split.splits * D;
  }
  if (cache->cache_dtype == KLLM_B200_I8) {
    return D == 64 ? launch_groups<64, true>(a, split.narrow, o) : launch_groups<128, true>(a, split.narrow, o);
  }
  return D == 64 ? launch_groups<64, false>(a, split.narrow, o) : launch_groups<128, false>(a, split.narrow, o);
}

}  // namespace kb

extern "C" int kllm_b200_attention_paged_workspace_bytes(int64_t n_tokens, int64_t n_heads,
                                                         const kllm_b200_paged_cache* cache, int64_t* bytes) {
  return kb::attention_paged_workspace_bytes(n_tokens, n_heads, cache, bytes);
}

extern "C" int kllm_b200_attention_paged(const void* q, int64_t q_stride, const kllm_b200_paged_cache* cache,
                                         const int32_t* positions, const int32_t* seqs, int64_t n_tokens,
                                         int64_t n_heads, void* out, int64_t out_stride, void* workspace,
                                         int64_t workspace_bytes, int32_t* err_flags, void* stream) {
  kb::LaunchOpts o;
  o.stream = static_cast<cudaStream_t>(stream);
  return kb::attention_paged(q, q_stride, cache, positions, seqs, n_tokens, n_heads, out, out_stride, workspace,
                             workspace_bytes, err_flags, o);
}
