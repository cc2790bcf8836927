// attention_paged.cu — attention of single new tokens over the paged KV cache
// (fp16 or int8 rows), split over the cache's length and joined.
//
// For token t, kv head g and its G query heads:
//     o_h = sum_j p_hj v_j / sum_j p_hj,  p_hj = exp(q_h . k_j / sqrt(D) - m_h)
// over positions j = 0..positions[t]. The kernel reads each cached row once:
// 2 (positions[t] + 1) rows of D fp16 values, or of D codes and a scale, per
// (token, kv head), and is bound by HBM.
//
// A CTA takes one part of the positions of a (token, kv head); its four warps
// stream 32-position tiles of K and V through a per-warp cp.async ring, the
// rows' addresses taken from the page table one tile ahead. Both products run
// on mma.sync m16n8k16 with the cached rows as the M side: S^T = K Q^T (16
// positions x 8 heads) and O^T += V^T P^T (16 dims x 8 heads), so a group of up
// to eight query heads fills the N side; with heads as the M side half or more
// of every fragment, exponential and accumulator would be padding.
//
// int8 rows: a code c becomes the fp16 1024 + (c + 128) by placing its biased
// byte under the exponent byte 0x64, and one packed subtraction of 1152 leaves
// c exactly; the scale of a key multiplies its scores, that of a value its
// probabilities. Codes enter the products exactly.
//
// Softmax: each warp keeps a reference m per head that bounds its scores up to
// kLag (log2) and the powers 2^(s - m + kLift). Only a tile that exceeds the
// bound (in practice the first ones) pays for a new maximum and a rescale of
// the sums. kLift places the largest probabilities near the top of fp16's
// range, so that those down to 2^-25 of the largest keep 11 bits as operands
// of the second product; for int8 rows, whose probabilities carry the scale of
// the value, that scale is taken relative to a power of two at or above the
// largest the warp has met. Scores, sums and accumulators are fp32.
#include <math.h>

#include "paged.cuh"
#include "tcgen05.cuh"  // smem_u32

namespace kb {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kTile = 32;        // positions per warp tile
constexpr int kStages = 3;       // tiles of the cp.async ring
constexpr int kMaxGroups = 16;   // query heads per kv head
constexpr int kMaxSplits = 64;   // parts of one (token, kv head)
constexpr int kCombineWarps = 4;
constexpr float kLag = 4.f;      // log2 by which a score may exceed the reference
constexpr float kLift = 11.f;    // 2^(kLift + kLag) < 65504

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
  int splits;
  float* part_o;   // [T, Hq, splits, D], sums of p v against the part's own max
  float* part_ml;  // [T, Hq, splits, 2] (max, sum); sum -1: the part met a bad page
  int32_t* err_flags;
  float scale_log2;  // log2(e) / sqrt(D)
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, int src_bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(src_bytes) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, int src_bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;\n" ::"r"(dst), "l"(src), "r"(src_bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;\n" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;\n" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldsm_x4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldsm_x4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
// Transpose of an 8 x 8 fp16 matrix held two elements of a row per lane.
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};\n"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Codes of bytes (i, j) of `w` (bytes already biased by 128) as an fp16 pair.
template <int SEL>
__device__ __forceinline__ uint32_t codes_h2(uint32_t w) {
  const uint32_t x = __byte_perm(w, 0x64646464u, SEL);
  const uint32_t bias = 0x64806480u;  // 1152, 1152
  const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&x), *reinterpret_cast<const __half2*>(&bias));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// Byte offset of 16-byte chunk `ch` of row `r` in a tile of ROW-byte rows; the
// chunk is XOR-ed so that the eight rows of one ldmatrix phase fall in eight
// different bank groups (64-byte rows: two rows share 128 bytes).
template <int ROW>
__device__ __forceinline__ uint32_t swz(int r, int ch) {
  return static_cast<uint32_t>(r * ROW + ((ROW == 64 ? ch ^ ((r >> 1) & 3) : ch ^ (r & 7)) << 4));
}

template <int D, bool I8>
struct Ring {
  static constexpr int kRow = I8 ? D : 2 * D;  // bytes of a cached row
  static constexpr int kTileBytes = kTile * kRow;
  static constexpr int kStageBytes = 2 * kTileBytes + (I8 ? 2 * kTile * 4 : 0);  // K, V, their scales
  static constexpr int kBytes = kWarps * kStages * kStageBytes;
};

// One row's (or part's) share of the joined output: exp2 of its max against the
// joint max; a part that saw nothing has max -inf and weight 0.
__device__ __forceinline__ float join_weight(float m, float top) { return m == -INFINITY ? 0.f : exp2f(m - top); }

template <int D, bool I8, int NH>
__global__ void __launch_bounds__(kThreads) attn_paged_kernel(const __grid_constant__ PagedAttnArgs a) {
  using R = Ring<D, I8>;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ int s_bad;
  constexpr int kRow = R::kRow;
  constexpr int kChunks = kRow / 16;
  constexpr int kM = D / 16;  // m16 tiles of O^T over head_dim, k16 steps of K Q^T
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int gid = lane >> 2, tig = lane & 3;
  const int64_t t = blockIdx.x / a.splits;
  const int part = static_cast<int>(blockIdx.x - t * a.splits);
  const int g = blockIdx.y;
  const int G = a.groups;
  if (threadIdx.x == 0) s_bad = 0;

  grid_dep_wait();
  grid_dep_launch();
  const int pos = a.positions[t], seq = a.seqs[t];
  __half* out_t = a.out + t * a.out_stride + static_cast<int64_t>(g) * G * D;
  int flag;
  if (token_state(a.view, pos, seq, flag) != kTokenOk) {
    if (part == 0) {
      if (threadIdx.x == 0 && g == 0 && flag != 0) set_flag(a.err_flags, flag);
      for (int i = threadIdx.x; i < G * D / 8; i += kThreads) st_plain(out_t + i * 8, make_uint4(0u, 0u, 0u, 0u));
    }
    return;
  }
  const int n = pos + 1;
  const int all_tiles = (n + kTile - 1) / kTile;
  const int per_part = (all_tiles + a.splits - 1) / a.splits;
  const int tile0 = part * per_part;
  if (tile0 >= all_tiles) return;
  const int n_tiles = min(per_part, all_tiles - tile0);
  const int my_tiles = n_tiles > warp ? (n_tiles - warp + kWarps - 1) / kWarps : 0;

  const int shift = a.view.page_shift, mask = (1 << shift) - 1;
  const int32_t* table = a.view.table + seq * a.view.max_pages;
  unsigned char* ring = smem + warp * (kStages * R::kStageBytes);
  bool bad = false;

  // The page of this lane's position of warp tile i (-1 past the end).
  auto page_of = [&](int i) {
    const int j = (tile0 + warp + i * kWarps) * kTile + lane;
    return i < my_tiles && j < n ? __ldg(table + (j >> shift)) : -1;
  };
  // Copies warp tile i into its stage; rows past the last position are
  // zero-filled, so no stale bits reach the products.
  auto issue = [&](int i, int page) {
    if (i < my_tiles) {
      const int j0 = (tile0 + warp + i * kWarps) * kTile;
      unsigned char* sk = ring + (i % kStages) * R::kStageBytes;
      unsigned char* sv = sk + R::kTileBytes;
      const bool in = j0 + lane < n;
      if (in && !page_ok(a.view, page)) bad = true;
      const bool ok = in && page_ok(a.view, page);
      // row index of this lane's position in K and V (row 0 where there is none)
      const int64_t row =
          ok ? (((static_cast<int64_t>(page) * a.view.n_kv_heads + g) << shift) + ((j0 + lane) & mask)) : 0;
      const unsigned live = __ballot_sync(0xffffffffu, ok);
      if (I8) {
        float* ss = reinterpret_cast<float*>(sv + R::kTileBytes);
        cp_async4(smem_u32(ss + lane), a.k_scales + row, ok ? 4 : 0);
        cp_async4(smem_u32(ss + kTile + lane), a.v_scales + row, ok ? 4 : 0);
      }
#pragma unroll
      for (int it = 0; it < kTile * kChunks / 32; ++it) {
        const int r = (lane + it * 32) / kChunks, ch = (lane + it * 32) % kChunks;
        const int64_t off = __shfl_sync(0xffffffffu, row, r) * kRow + ch * 16;
        const int bytes = (live >> r) & 1 ? 16 : 0;
        cp_async16(smem_u32(sk + swz<kRow>(r, ch)), static_cast<const char*>(a.k_pages) + off, bytes);
        cp_async16(smem_u32(sv + swz<kRow>(r, ch)), static_cast<const char*>(a.v_pages) + off, bytes);
      }
    }
    cp_async_commit();  // empty groups keep the count uniform
  };

  {
    int first[kStages - 1];
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) first[i] = page_of(i);
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) issue(i, first[i]);
  }
  int next_page = page_of(kStages - 1);

  // B fragments of Q^T. int8: lane tig holds dims 4 tig .. 4 tig + 3 of each 16
  // (the bytes ldmatrix hands it), so the k index is permuted alike on both sides.
  uint32_t qb[NH][kM][2];
#pragma unroll
  for (int h = 0; h < NH; ++h) {
    const int head = h * 8 + gid;
    const __half* qh = a.q + t * a.q_stride + (static_cast<int64_t>(g) * G + (head < G ? head : 0)) * D;
#pragma unroll
    for (int ks = 0; ks < kM; ++ks) {
      const int d0 = ks * 16 + (I8 ? 4 : 2) * tig;
      qb[h][ks][0] = head < G ? *reinterpret_cast<const uint32_t*>(qh + d0) : 0u;
      qb[h][ks][1] = head < G ? *reinterpret_cast<const uint32_t*>(qh + d0 + (I8 ? 2 : 8)) : 0u;
    }
  }

  float o[NH][kM][4];
  float m[NH][2], l[NH][2];
#pragma unroll
  for (int h = 0; h < NH; ++h) {
    m[h][0] = m[h][1] = -INFINITY;
    l[h][0] = l[h][1] = 0.f;
#pragma unroll
    for (int i = 0; i < kM; ++i) o[h][i][0] = o[h][i][1] = o[h][i][2] = o[h][i][3] = 0.f;
  }
  float vref = 0.f, inv_vref = 0.f;  // int8: power of two at or above the value scales met
  const float sl2 = a.scale_log2;

  for (int i = 0; i < my_tiles; ++i) {
    issue(i + kStages - 1, next_page);
    next_page = page_of(i + kStages);
    cp_async_wait<kStages - 1>();
    __syncwarp();
    const int j0 = (tile0 + warp + i * kWarps) * kTile;
    const unsigned char* sk = ring + (i % kStages) * R::kStageBytes;
    const unsigned char* sv = sk + R::kTileBytes;
    const float* ss = reinterpret_cast<const float*>(sv + R::kTileBytes);

    // S^T: two m16 tiles of positions x NH n8 tiles of heads
    float s[2][NH][4];
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
      for (int h = 0; h < NH; ++h) s[mt][h][0] = s[mt][h][1] = s[mt][h][2] = s[mt][h][3] = 0.f;
      if (!I8) {
#pragma unroll
        for (int ks = 0; ks < kM; ++ks) {
          uint32_t b[4];
          ldsm_x4(b, smem_u32(sk + swz<kRow>(mt * 16 + (lane & 15), 2 * ks + (lane >> 4))));
#pragma unroll
          for (int h = 0; h < NH; ++h) mma16816(s[mt][h], b[0], b[1], b[2], b[3], qb[h][ks][0], qb[h][ks][1]);
        }
      } else {
#pragma unroll
        for (int kp = 0; kp < kM / 2; ++kp) {
          uint32_t b[4];
          ldsm_x4(b, smem_u32(sk + swz<kRow>(mt * 16 + (lane & 15), 2 * kp + (lane >> 4))));
#pragma unroll
          for (int e = 0; e < 4; ++e) b[e] ^= 0x80808080u;
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const uint32_t a0 = codes_h2<0x4140>(b[2 * e]), a2 = codes_h2<0x4342>(b[2 * e]);
            const uint32_t a1 = codes_h2<0x4140>(b[2 * e + 1]), a3 = codes_h2<0x4342>(b[2 * e + 1]);
#pragma unroll
            for (int h = 0; h < NH; ++h) {
              mma16816(s[mt][h], a0, a1, a2, a3, qb[h][2 * kp + e][0], qb[h][2 * kp + e][1]);
            }
          }
        }
      }
      // log2 units; element e belongs to position gid + 8 (e >> 1), head 2 tig + (e & 1)
      float f0 = sl2, f1 = sl2;
      if (I8) {
        f0 *= ss[mt * 16 + gid];
        f1 *= ss[mt * 16 + gid + 8];
      }
#pragma unroll
      for (int h = 0; h < NH; ++h) {
        s[mt][h][0] *= f0;
        s[mt][h][1] *= f0;
        s[mt][h][2] *= f1;
        s[mt][h][3] *= f1;
      }
    }
    if (j0 + kTile > n) {
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (j0 + mt * 16 + gid + 8 * (e >> 1) >= n) {
#pragma unroll
            for (int h = 0; h < NH; ++h) s[mt][h][e] = -INFINITY;
          }
        }
      }
    }
    float top[NH][2];
    bool over = false;
#pragma unroll
    for (int h = 0; h < NH; ++h) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        top[h][e] = fmaxf(fmaxf(s[0][h][e], s[0][h][e + 2]), fmaxf(s[1][h][e], s[1][h][e + 2]));
        over |= top[h][e] > m[h][e] + kLag;
      }
    }
    float vs = 0.f;
    if (I8) {
      vs = fabsf(ss[kTile + lane]);
      over |= vs > vref;
    }
    if (__any_sync(0xffffffffu, over)) {
      float new_ref = vref, ratio = 1.f;
      if (I8) {
        // the power of two above the largest scale of the tile (a NaN scale
        // never compares and poisons the probabilities by itself)
        const unsigned bits = __reduce_max_sync(0xffffffffu, vs <= 3.4028235e38f ? __float_as_uint(vs) : 0u);
        const float up = __uint_as_float(min((bits >> 23) + 1u, 0xfeu) << 23);
        if (bits != 0u && up > vref) new_ref = up;
        ratio = new_ref > 0.f ? vref / new_ref : 1.f;
        vref = new_ref;
        inv_vref = vref > 0.f ? 1.f / vref : 0.f;
      }
#pragma unroll
      for (int h = 0; h < NH; ++h) {
        float cr[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float x = fmaxf(top[h][e], m[h][e]);
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
          cr[e] = m[h][e] == -INFINITY ? 0.f : exp2f(m[h][e] - x);
          m[h][e] = x;
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
    }
    // probabilities, and P^T as B fragments: the transpose of each 8 x 8 block
    uint32_t pb[2][NH][2];
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
      float v0 = 1.f, v1 = 1.f;
      if (I8) {
        v0 = ss[kTile + mt * 16 + gid] * inv_vref;
        v1 = ss[kTile + mt * 16 + gid + 8] * inv_vref;
      }
#pragma unroll
      for (int h = 0; h < NH; ++h) {
        // a head whose every score so far is -inf keeps base 0
        const float b0 = kLift - (m[h][0] == -INFINITY ? 0.f : m[h][0]);
        const float b1 = kLift - (m[h][1] == -INFINITY ? 0.f : m[h][1]);
        const float p0 = exp2f(s[mt][h][0] + b0), p1 = exp2f(s[mt][h][1] + b1);
        const float p2 = exp2f(s[mt][h][2] + b0), p3 = exp2f(s[mt][h][3] + b1);
        l[h][0] += p0 + p2;
        l[h][1] += p1 + p3;
        pb[mt][h][0] = transpose8x8(f2_to_h2(p0 * v0, p1 * v0));
        pb[mt][h][1] = transpose8x8(f2_to_h2(p2 * v1, p3 * v1));
      }
    }
    // O^T += V^T P^T. fp16: m tile k holds dims 16 k + gid, + 8; int8: dims
    // 16 k + 2 gid, 2 gid + 1 (the two codes of the 16-bit units transposed)
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
      const int mtx = lane >> 3;
      if (!I8) {
#pragma unroll
        for (int k = 0; k < kM; ++k) {
          uint32_t b[4];
          ldsm_x4_trans(b, smem_u32(sv + swz<kRow>(mt * 16 + 8 * (mtx >> 1) + (lane & 7), 2 * k + (mtx & 1))));
#pragma unroll
          for (int h = 0; h < NH; ++h) mma16816(o[h][k], b[0], b[1], b[2], b[3], pb[mt][h][0], pb[mt][h][1]);
        }
      } else {
#pragma unroll
        for (int kp = 0; kp < kM / 2; ++kp) {
          uint32_t b[4];
          ldsm_x4_trans(b, smem_u32(sv + swz<kRow>(mt * 16 + 8 * (mtx & 1) + (lane & 7), 2 * kp + (mtx >> 1))));
#pragma unroll
          for (int e = 0; e < 4; ++e) b[e] ^= 0x80808080u;
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const uint32_t a0 = codes_h2<0x4240>(b[2 * e]), a1 = codes_h2<0x4341>(b[2 * e]);
            const uint32_t a2 = codes_h2<0x4240>(b[2 * e + 1]), a3 = codes_h2<0x4341>(b[2 * e + 1]);
#pragma unroll
            for (int h = 0; h < NH; ++h) mma16816(o[h][2 * kp + e], a0, a1, a2, a3, pb[mt][h][0], pb[mt][h][1]);
          }
        }
      }
    }
    __syncwarp();  // the stage is refilled by the next iteration's issue
  }
  cp_async_wait<0>();

  // join the four warps; a head's sum is spread over the eight lanes of its column
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
  constexpr int kHeads = 8 * NH;
  constexpr int kRedRow = D + 4;
  float* red_o = reinterpret_cast<float*>(smem);          // [warps][heads][kRedRow]
  float* red_ml = red_o + kWarps * kHeads * kRedRow;      // [warps][heads][2]
  const float back = I8 ? vref : 1.f;
#pragma unroll
  for (int h = 0; h < NH; ++h) {
#pragma unroll
    for (int k = 0; k < kM; ++k) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int head = h * 8 + 2 * tig + (e & 1);
        const int d = 16 * k + (I8 ? 2 * gid + (e >> 1) : gid + 8 * (e >> 1));
        red_o[(warp * kHeads + head) * kRedRow + d] = o[h][k][e] * back;
      }
    }
    if (gid == 0) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        red_ml[(warp * kHeads + h * 8 + 2 * tig + e) * 2] = m[h][e];
        red_ml[(warp * kHeads + h * 8 + 2 * tig + e) * 2 + 1] = l[h][e];
      }
    }
  }
  __syncthreads();
  const bool any_bad = s_bad != 0;
  if (any_bad && threadIdx.x == 0 && g == 0) set_flag(a.err_flags, KLLM_B200_FLAG_BAD_PAGE);
  const bool whole = per_part >= all_tiles;  // this part is all there is
  for (int idx = threadIdx.x; idx < G * D; idx += kThreads) {
    const int head = idx / D, d = idx - head * D;
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) M = fmaxf(M, red_ml[(w * kHeads + head) * 2]);
    float L = 0.f, acc = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      // a warp without tiles holds zeros and weight 0
      const float f = join_weight(red_ml[(w * kHeads + head) * 2], M);
      L += red_ml[(w * kHeads + head) * 2 + 1] * f;
      acc += red_o[(w * kHeads + head) * kRedRow + d] * f;
    }
    if (whole) {
      out_t[idx] = __float2half_rn(any_bad ? 0.f : acc / L);
    } else {
      const int64_t prow = (t * a.n_heads + static_cast<int64_t>(g) * G + head) * a.splits + part;
      a.part_o[prow * D + d] = acc;
      if (d == 0) {
        a.part_ml[prow * 2] = M;
        a.part_ml[prow * 2 + 1] = any_bad ? -1.f : L;
      }
    }
  }
}

// One warp per (token, query head) that has several parts.
template <int D>
__global__ void __launch_bounds__(kCombineWarps * 32) attn_paged_combine_kernel(const __grid_constant__ PagedAttnArgs a) {
  constexpr int kPer = D / 32;
  const int lane = threadIdx.x & 31;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kCombineWarps + (threadIdx.x >> 5);
  grid_dep_wait();
  grid_dep_launch();
  if (row >= a.n_tokens * a.n_heads) return;
  const int64_t t = row / a.n_heads;
  const int pos = a.positions[t], seq = a.seqs[t];
  int flag;
  if (token_state(a.view, pos, seq, flag) != kTokenOk) return;
  const int all_tiles = (pos + kTile) / kTile;
  const int per_part = (all_tiles + a.splits - 1) / a.splits;
  const int used = (all_tiles + per_part - 1) / per_part;
  if (used <= 1) return;
  const float* ml = a.part_ml + row * a.splits * 2;
  const float* po = a.part_o + row * a.splits * D;
  float M = -INFINITY;
  bool bad = false;
  for (int c = lane; c < used; c += 32) {
    M = fmaxf(M, ml[2 * c]);
    bad |= ml[2 * c + 1] == -1.f;
  }
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, x));
  bad = __any_sync(0xffffffffu, bad);
  float L = 0.f, acc[kPer];
#pragma unroll
  for (int k = 0; k < kPer; ++k) acc[k] = 0.f;
  for (int c = 0; c < used; ++c) {
    const float w = join_weight(ml[2 * c], M);
    L += w * ml[2 * c + 1];
#pragma unroll
    for (int k = 0; k < kPer; ++k) acc[k] += w * po[c * D + lane * kPer + k];
  }
  __half* dst = a.out + t * a.out_stride + (row - t * a.n_heads) * D + lane * kPer;
#pragma unroll
  for (int k = 0; k < kPer; ++k) dst[k] = __float2half_rn(bad ? 0.f : acc[k] / L);
}

// Parts per (token, kv head): enough CTAs for several waves of the device.
int64_t preferred_splits(int64_t items, int64_t capacity) {
  const int64_t want = 8LL * sm_count();
  int64_t s = (want + items - 1) / items;
  const int64_t most = (capacity + kWarps * kTile - 1) / (kWarps * kTile);
  if (s > most) s = most;
  if (s > kMaxSplits) s = kMaxSplits;
  return s < 1 ? 1 : s;
}

int64_t workspace_for(int64_t n_tokens, int64_t n_heads, int64_t head_dim, int64_t splits) {
  return splits <= 1 ? 0 : n_tokens * n_heads * splits * (head_dim + 2) * static_cast<int64_t>(sizeof(float));
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
  if (n_tokens * kMaxSplits > 0x7fffffffLL) return fail(KLLM_B200_ERR_SHAPE, "%s: too many tokens", what);
  return KLLM_B200_OK;
}

template <int D, bool I8, int NH>
int launch_attention(const PagedAttnArgs& a, const LaunchOpts& o) {
  const char* what = "attention_paged";
  const size_t smem = Ring<D, I8>::kBytes;
  static_assert(Ring<D, I8>::kBytes >= kWarps * 8 * NH * (D + 4 + 2) * 4, "the join fits the rings");
  auto kernel = attn_paged_kernel<D, I8, NH>;
  cudaError_t err = allow_smem(reinterpret_cast<const void*>(kernel), smem);
  if (err != cudaSuccess) return launch_status(err, "attention_paged: shared memory opt-in");
  const dim3 grid(static_cast<unsigned>(a.n_tokens * a.splits), static_cast<unsigned>(a.view.n_kv_heads));
  const int rc = launch_status(launch(kernel, grid, dim3(kThreads), smem, o.stream, o.pdl, a), what);
  if (rc != KLLM_B200_OK || a.splits == 1) return rc;
  const int64_t rows = a.n_tokens * a.n_heads;
  const dim3 cgrid(static_cast<unsigned>((rows + kCombineWarps - 1) / kCombineWarps));
  return launch_status(launch(attn_paged_combine_kernel<D>, cgrid, dim3(kCombineWarps * 32), 0, o.stream, true, a), what);
}

template <int D, bool I8>
int launch_groups(const PagedAttnArgs& a, const LaunchOpts& o) {
  return a.groups <= 8 ? launch_attention<D, I8, 1>(a, o) : launch_attention<D, I8, 2>(a, o);
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
  *bytes = workspace_for(n_tokens, n_heads, cache->head_dim, preferred_splits(n_tokens * view.n_kv_heads, view.capacity));
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
  int64_t splits = preferred_splits(n_tokens * a.view.n_kv_heads, a.view.capacity);
  while (workspace_for(n_tokens, n_heads, D, splits) > (workspace ? workspace_bytes : 0)) splits = (splits + 1) / 2;
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
  a.splits = static_cast<int>(splits);
  a.err_flags = err_flags;
  a.scale_log2 = 1.4426950408889634f / sqrtf(static_cast<float>(D));
  if (splits > 1) {
    a.part_o = static_cast<float*>(workspace);
    a.part_ml = a.part_o + n_tokens * n_heads * splits * D;
  }
  if (cache->cache_dtype == KLLM_B200_I8) return D == 64 ? launch_groups<64, true>(a, o) : launch_groups<128, true>(a, o);
  return D == 64 ? launch_groups<64, false>(a, o) : launch_groups<128, false>(a, o);
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
