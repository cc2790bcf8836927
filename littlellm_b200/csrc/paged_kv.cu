// paged_kv.cu — writing and reading the paged KV cache (one layer): bias +
// per-head RMSNorm of q and k + rotate-half RoPE + append in fp16 or int8,
// and the read back to fp16 rows.
//
// Append. Per head x of D values, in fp32 with one rounding at the end:
//     x += b;  q, k: x *= w / sqrt(mean(x^2) + eps);  q, k: rotate;
//     q -> fp16;  k, v -> fp16, or scale = max|x| / 127 and
//     code = rint(x / scale).
// D / 16 lanes own a head, lane c the elements 8c..8c+7 and D/2 + 8c..+7:
// both members of its rotation pairs, two 16-byte loads and stores, so the
// norm's sum and the row's maximum are two or three shuffles and nothing goes
// through shared memory but the token's cos/sin. A warp covers 32 / (D / 16)
// heads at a time and U such sets of one token; the inputs of all U are
// loaded before anything else runs.
//
// The angle pos * theta^(-2d/D) is formed in 64 bits and in turns: its
// fraction is exact to 2^-53 * pos, while an fp32 product would be off by
// 0.06 rad at position 10^6. The reduced fraction goes to sincospif, which has
// no slow path.
//
// Both kernels are bound by HBM: the append reads T (Hq + 2 Hkv) D fp16 values
// and writes T Hq D fp16 and 2 T Hkv rows; the read back moves each row once.
#include <cmath>

#include "paged.cuh"

namespace kb {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kMaxPairs = 64;  // head_dim <= 128

struct AppendArgs {
  const __half* q;
  const __half* k;
  const __half* v;
  int64_t q_stride, k_stride, v_stride, q_out_stride;
  const void* bq;
  const void* bk;
  const void* bv;
  const void* q_norm;
  const void* k_norm;
  int bias_f32, norm_f32;
  float eps;
  const int32_t* positions;
  const int32_t* seqs;
  int64_t n_tokens;
  int n_heads;
  int warps_per_token;
  PagedView view;
  void* k_pages;
  void* v_pages;
  float* k_scales;
  float* v_scales;
  __half* q_out;
  int32_t* err_flags;
  double turns[kMaxPairs];  // theta^(-2d/D) / (2 pi)
};

// Eight values of a bias or weight vector (fp16 or fp32, 16-byte aligned) from element `at`.
__device__ __forceinline__ void load8(const void* p, int f32, int at, float (&f)[8]) {
  if (f32) {
    const float4 x = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(p) + at));
    const float4 y = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(p) + at + 4));
    f[0] = x.x; f[1] = x.y; f[2] = x.z; f[3] = x.w; f[4] = y.x; f[5] = y.y; f[6] = y.z; f[7] = y.w;
  } else {
    unpack8(ld_keep(static_cast<const __half*>(p) + at), f);
  }
}

// 1 / x to an ulp (normal x).
__device__ __forceinline__ float rcp_approx(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// rint(x / scale) of eight values as codes, the quotient by Markstein's residual
// correction (P. Markstein, Computation of elementary functions on the IBM RISC
// System/6000 processor, 1990). inv is 1 / scale to an ulp or two, so q = x inv
// is off by some 2^-22; r = x - q scale is exact as an FMA but for a rounding,
// and q + r inv is off by that error's square, 2^-45, before it is rounded. So a
// value half way between two codes is seen as such and goes to the even one, and
// codes are those of the fp32 quotient (all pairs of fp16 significands, and three
// million fp32 values within two steps of half way, agree bit for bit). Adding
// 1.5 * 2^23 rounds to a whole number, ties to even, and leaves the code in the
// low byte.
__device__ __forceinline__ uint2 codes8(const float (&x)[8], float scale, float inv) {
  const unsigned long long i2 = f32x2_pack(inv, inv), n2 = f32x2_pack(-scale, -scale);
  const unsigned long long magic = f32x2_pack(12582912.f, 12582912.f);
  uint32_t w[8];
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    const unsigned long long v = f32x2_pack(x[i], x[i + 1]);
    const unsigned long long q = f32x2_mul(v, i2);
    const unsigned long long c = f32x2_add(f32x2_fma(f32x2_fma(q, n2, v), i2, q), magic);
    float lo, hi;
    f32x2_unpack(c, lo, hi);
    w[i] = __float_as_uint(lo);
    w[i + 1] = __float_as_uint(hi);
  }
  return make_uint2(__byte_perm(__byte_perm(w[0], w[1], 0x0040), __byte_perm(w[2], w[3], 0x0040), 0x5410),
                    __byte_perm(__byte_perm(w[4], w[5], 0x0040), __byte_perm(w[6], w[7], 0x0040), 0x5410));
}

// x *= r * w for eight values, two per packed multiply.
__device__ __forceinline__ void scale8(float (&x)[8], float r, const float (&w)[8]) {
  const unsigned long long r2 = f32x2_pack(r, r);
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    f32x2_unpack(f32x2_mul(f32x2_pack(x[i], x[i + 1]), f32x2_mul(r2, f32x2_pack(w[i], w[i + 1]))), x[i], x[i + 1]);
  }
}

// Eight floats of shared memory (32-byte aligned).
__device__ __forceinline__ void lds8(const float* p, float (&f)[8]) {
  const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
  f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
}

// U sets of heads per warp. SHARED: every warp of the CTA works on the same
// token, which computes its cos/sin once; else each warp computes its own
// token's. Many tokens want warps more than registers: 16384 tokens of 96
// heads of 128, int8, 148 us held to 9 CTAs per SM (8 bytes spilled), 164 at the
// 7 that fit unheld (103 us of HBM time; the rest is issue, about 290
// instructions for four heads, and the wait for a warp's first loads: CTAs that
// stay and load their next token beside the present one took 188 us).
template <int D, bool I8, int U, bool SHARED>
__global__ void __launch_bounds__(kThreads, SHARED && U > 1 ? (I8 ? 9 : 8) : 1) qkv_norm_rope_append_paged_kernel(const __grid_constant__ AppendArgs a) {
  constexpr int L = D / 16;    // lanes of one head
  constexpr int kSet = 32 / L;  // heads a warp takes at once
  constexpr int kTables = SHARED ? 1 : kWarps;
  __shared__ __align__(32) float s_cos[kTables][D / 2], s_sin[kTables][D / 2], s_neg[kTables][D / 2];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // SHARED: CTA (x, y) takes part y of token x; else consecutive warps
  const unsigned w0 = blockIdx.x * kWarps + warp, wpt = a.warps_per_token;
  const int64_t t = SHARED ? blockIdx.x : w0 / wpt;
  const int part = SHARED ? blockIdx.y * kWarps + warp : static_cast<int>(w0 - static_cast<unsigned>(t) * wpt);
  grid_dep_wait();
  grid_dep_launch();
  if (t >= a.n_tokens) return;  // uniform per warp; with SHARED per CTA

  const int hkv = a.view.n_kv_heads;
  const int n_rows = a.n_heads + 2 * hkv;
  const int c = lane % L;
  const int pos = __ldg(a.positions + t), seq = __ldg(a.seqs + t);
  uint4 lo[U], hi[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int h = (part * U + u) * kSet + lane / L;
    lo[u] = hi[u] = make_uint4(0u, 0u, 0u, 0u);
    if (h < n_rows) {
      const __half* src = h < a.n_heads         ? a.q + t * a.q_stride + h * D
                          : h < a.n_heads + hkv ? a.k + t * a.k_stride + (h - a.n_heads) * D
                                                : a.v + t * a.v_stride + (h - a.n_heads - hkv) * D;
      // coherent loads: with q_out == q this kernel writes what it reads
      lo[u] = ld_cg(src + 8 * c);
      hi[u] = ld_cg(src + D / 2 + 8 * c);
    }
  }
  int flag;
  const TokenState state = token_state(a.view, pos, seq, flag);
  int page = -1;
  if (state == kTokenOk) {
    page = __ldg(a.view.table + seq * a.view.max_pages + (pos >> a.view.page_shift));
    if (!page_ok(a.view, page)) flag = KLLM_B200_FLAG_BAD_PAGE;
  }
  if (state != kTokenOk || flag != 0) {
    if (flag != 0 && part == 0 && lane == 0) set_flag(a.err_flags, flag);
    return;
  }
  const int table = SHARED ? 0 : warp;
  for (int i = SHARED ? threadIdx.x : lane; i < D / 2; i += SHARED ? kThreads : 32) {
    const double w = static_cast<double>(pos) * a.turns[i];
    const float f = static_cast<float>(w - rint(w));
    float sn, cs;
    sincospif(2.f * f, &sn, &cs);
    s_cos[table][i] = cs;
    s_sin[table][i] = sn;
    s_neg[table][i] = -sn;
  }
  if (SHARED) __syncthreads(); else __syncwarp();
  const int64_t row0 = ((static_cast<int64_t>(page) * hkv) << a.view.page_shift) + (pos & ((1 << a.view.page_shift) - 1));

#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int h0 = (part * U + u) * kSet;  // the set's first head: what follows is uniform per warp where it can be
    if (h0 >= n_rows) break;
    const int h = h0 + lane / L;
    const bool live = h < n_rows, is_q = h < a.n_heads, is_v = h >= a.n_heads + hkv;
    const int hh = is_q ? h : is_v ? h - a.n_heads - hkv : h - a.n_heads;  // within its tensor
    float x[8], y[8], p[8];
    unpack8(lo[u], x);
    unpack8(hi[u], y);
    const void* bias = is_q ? a.bq : is_v ? a.bv : a.bk;
    if (live && bias != nullptr) {
      load8(bias, a.bias_f32, hh * D + 8 * c, p);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] += p[i];
      load8(bias, a.bias_f32, hh * D + D / 2 + 8 * c, p);
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] += p[i];
    }
    if (h0 < a.n_heads + hkv) {  // some q or k head
      if (a.q_norm != nullptr || a.k_norm != nullptr) {
        unsigned long long s2 = 0ull;
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
          const unsigned long long v = f32x2_pack(x[i], x[i + 1]), w = f32x2_pack(y[i], y[i + 1]);
          s2 = f32x2_fma(v, v, f32x2_fma(w, w, s2));
        }
        float ss, s1;
        f32x2_unpack(s2, ss, s1);
        ss += s1;
#pragma unroll
        for (int m = L / 2; m > 0; m >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, m);
        const void* weight = is_v ? nullptr : is_q ? a.q_norm : a.k_norm;
        if (weight != nullptr) {
          const float r = rsqrtf(ss * (1.f / D) + a.eps);
          load8(weight, a.norm_f32, 8 * c, p);
          scale8(x, r, p);
          load8(weight, a.norm_f32, D / 2 + 8 * c, p);
          scale8(y, r, p);
        }
      }
      if (!is_v) {
        float cs[8], sn[8], ns[8], rx[8], ry[8];
        lds8(&s_cos[table][8 * c], cs);
        lds8(&s_sin[table][8 * c], sn);
        lds8(&s_neg[table][8 * c], ns);
        rope_rotate8_x2(x, y, cs, sn, ns, rx, ry);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          x[i] = rx[i];
          y[i] = ry[i];
        }
      }
      if (live && is_q) {
        __half* dst = a.q_out + t * a.q_out_stride + hh * D + 8 * c;
        st_plain(dst, pack8(x));
        st_plain(dst + D / 2, pack8(y));
      }
    }
    if (h0 + kSet <= a.n_heads) continue;  // no k or v head in the set
    const int64_t row = row0 + (static_cast<int64_t>(hh) << a.view.page_shift);
    if (!I8) {
      if (live && !is_q) {
        __half* dst = static_cast<__half*>(is_v ? a.v_pages : a.k_pages) + row * D + 8 * c;
        st_plain(dst, pack8(x));
        st_plain(dst + D / 2, pack8(y));
      }
    } else {
      float mx = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) mx = max_nan(mx, max_nan(fabsf(x[i]), fabsf(y[i])));
#pragma unroll
      for (int m = L / 2; m > 0; m >>= 1) mx = max_nan(mx, __shfl_xor_sync(0xffffffffu, mx, m));
      if (live && !is_q) {
        // below 2^-60 a row is zero in every use (fp16 ends at 2^-24) and its
        // reciprocal would leave fp32; an infinity or NaN marks the whole row
        const bool tiny = mx < 0x1p-60f, sound = mx <= 3.4028235e38f;
        // mx / 127 correctly rounded: the rounded reciprocal's product and its residual (Markstein, as above)
        const float s0 = mx * (1.f / 127.f), s1 = fmaf(fmaf(-127.f, s0, mx), 1.f / 127.f, s0);
        const bool coded = sound && !tiny;
        const float scale = coded ? s1 : 0.f, inv = coded ? rcp_approx(s1) : 0.f;
        if (!sound) {
#pragma unroll
          for (int i = 0; i < 8; ++i) x[i] = y[i] = 0.f;
        }
        int8_t* dst = static_cast<int8_t*>(is_v ? a.v_pages : a.k_pages) + row * D + 8 * c;
        *reinterpret_cast<uint2*>(dst) = codes8(x, scale, inv);
        *reinterpret_cast<uint2*>(dst + D / 2) = codes8(y, scale, inv);
        if (c == 0) (is_v ? a.v_scales : a.k_scales)[row] = sound ? scale : __int_as_float(0x7fffffff);
      }
    }
  }
}

// How a token's sets of heads go to warps: u sets a warp, `warps` warps, whole
// CTAs per token (shared) or not.
struct Deal {
  int u, warps;
  bool shared;
};

template <int D, bool I8>
void (*pick_append(Deal d))(AppendArgs) {
  if (!d.shared) return qkv_norm_rope_append_paged_kernel<D, I8, 3, false>;
  return d.u == 1   ? qkv_norm_rope_append_paged_kernel<D, I8, 1, true>
         : d.u == 2 ? qkv_norm_rope_append_paged_kernel<D, I8, 2, true>
                    : qkv_norm_rope_append_paged_kernel<D, I8, 3, true>;
}

// Few tokens: one set a warp, which is the shortest path through a token. Many:
// two or three sets a warp, which computes cos/sin for more heads at a time;
// heads that do not fill a CTA then share one with other tokens. 14 + 2 * 2
// heads of 64, int8, us (one set / three sets): 1 token 3.3 / 5.0, 1024 4.1 /
// 5.5, 4096 9.6 / 10.8, 16384 33.7 / 29.9, 65536 123 / 98.9.
Deal deal_sets(int64_t sets, int64_t n_tokens) {
  auto warps = [&](int u) { return static_cast<int>((sets + u - 1) / u); };
  auto whole = [&](int u) { return (warps(u) + kWarps - 1) / kWarps * kWarps; };  // in whole CTAs
  if (n_tokens * whole(1) <= 16384) return {1, whole(1), true};
  if (warps(3) < kWarps) return {3, warps(3), false};
  const int u = 2 * whole(2) < 3 * whole(3) ? 2 : 3;  // the one that leaves fewer idle sets
  return {u, whole(u), true};
}

// ---------------------------------------------------------------------------
// Read back
// ---------------------------------------------------------------------------

constexpr int kReadThreads = 256;

struct ReadArgs {
  const void* k_pages;
  const void* v_pages;
  const float* k_scales;
  const float* v_scales;
  PagedView view;
  const int32_t* positions;
  const int32_t* seqs;
  int64_t n_tokens;
  const int32_t* out_slots;
  int64_t n_out_slots, out_max_seq;
  __half* k_out;
  __half* v_out;
  bool wide;  // outputs 32-byte aligned
  int32_t* err_flags;
};

// Sixteen codes times the row's scale, as fp16. The byte c + 128 under the
// exponent of 2^23 is the fp32 2^23 + c + 128; the difference is c exactly, the
// product rounds to fp32 and then to fp16.
__device__ __forceinline__ void dequant16(uint4 w, float scale, uint4& lo, uint4& hi) {
  const uint32_t r[4] = {w.x, w.y, w.z, w.w};
  const unsigned long long s2 = f32x2_pack(scale, scale), off = f32x2_pack(-8388736.f, -8388736.f);
  uint32_t h[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t b = r[i] ^ 0x80808080u;
    const uint32_t e = 0x4b000000u;
    const unsigned long long x =
        f32x2_pack(__uint_as_float(__byte_perm(b, e, 0x7440)), __uint_as_float(__byte_perm(b, e, 0x7441)));
    const unsigned long long y =
        f32x2_pack(__uint_as_float(__byte_perm(b, e, 0x7442)), __uint_as_float(__byte_perm(b, e, 0x7443)));
    float p, q;
    f32x2_unpack(f32x2_mul(f32x2_add(x, off), s2), p, q);
    h[2 * i] = f2_to_h2(p, q);
    f32x2_unpack(f32x2_mul(f32x2_add(y, off), s2), p, q);
    h[2 * i + 1] = f2_to_h2(p, q);
  }
  lo = make_uint4(h[0], h[1], h[2], h[3]);
  hi = make_uint4(h[4], h[5], h[6], h[7]);
}

// 32 bytes of an output row whose base is 16-byte aligned only.
__device__ __forceinline__ void store32(__half* p, bool aligned, uint4 lo, uint4 hi) {
  if (aligned) {
    st_plain32(p, lo, hi);
  } else {
    st_plain(p, lo);
    st_plain(p + 8, hi);
  }
}

// A CTA reads one kv head of a block of consecutive tokens, so consecutive
// positions are consecutive rows of a page and of a head-major output. A lane
// takes 16 bytes of a cached row of K and the same of V. 32 x 2048 positions of
// 32 heads of 128: int8 258 us (0.96 of the copy rate), fp16 337 us (0.97); two
// tokens a lane took 269 us, heads before tokens 306 us.
template <int D, bool I8>
__global__ void __launch_bounds__(kReadThreads) kv_read_paged_kernel(const __grid_constant__ ReadArgs a) {
  constexpr int L = I8 ? D / 16 : D / 8;  // lanes of one row
  grid_dep_wait();
  grid_dep_launch();
  const int h = blockIdx.y, hkv = a.view.n_kv_heads;
  const int c = threadIdx.x % L;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * (kReadThreads / L) + threadIdx.x / L;
  if (t >= a.n_tokens) return;
  const int pos = __ldg(a.positions + t), seq = __ldg(a.seqs + t);
  int flag;
  const TokenState state = token_state(a.view, pos, seq, flag);
  if (state == kTokenPadding) return;
  int64_t to = t * hkv + h;
  if (a.out_slots != nullptr) {
    const int slot = __ldg(a.out_slots + t);
    if (pos >= a.out_max_seq) flag |= KLLM_B200_FLAG_BAD_POSITION;
    if (slot < 0 || slot >= a.n_out_slots) flag |= KLLM_B200_FLAG_BAD_SLOT;
    to = (static_cast<int64_t>(slot) * hkv + h) * a.out_max_seq + pos;
  }
  int page = 0;
  if (state == kTokenOk) {
    page = __ldg(a.view.table + seq * a.view.max_pages + (pos >> a.view.page_shift));
    if (!page_ok(a.view, page)) flag |= KLLM_B200_FLAG_BAD_PAGE;
  }
  if (flag != 0) {
    if (h == 0 && c == 0) set_flag(a.err_flags, flag);
    return;
  }
  const int64_t from =
      ((static_cast<int64_t>(page) * hkv + h) << a.view.page_shift) + (pos & ((1 << a.view.page_shift) - 1));
  const int64_t at = from * (I8 ? D : 2 * D) + 16 * c;
  const uint4 k = ld_stream(static_cast<const char*>(a.k_pages) + at);
  const uint4 v = ld_stream(static_cast<const char*>(a.v_pages) + at);
  if (I8) {
    const float ks = __ldg(a.k_scales + from), vs = __ldg(a.v_scales + from);
    uint4 lo, hi;
    dequant16(k, ks, lo, hi);
    store32(a.k_out + to * D + 16 * c, a.wide, lo, hi);
    dequant16(v, vs, lo, hi);
    store32(a.v_out + to * D + 16 * c, a.wide, lo, hi);
  } else {
    st_plain(a.k_out + to * D + 8 * c, k);
    st_plain(a.v_out + to * D + 8 * c, v);
  }
}

template <int D, bool I8>
int launch_read(const ReadArgs& a, const LaunchOpts& o) {
  constexpr int kTokens = kReadThreads / (I8 ? D / 16 : D / 8);
  const int64_t blocks = (a.n_tokens + kTokens - 1) / kTokens;
  const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>(a.view.n_kv_heads));
  return launch_status(launch(kv_read_paged_kernel<D, I8>, grid, dim3(kReadThreads), 0, o.stream, o.pdl, a),
                       "kv_read_paged");
}

}  // namespace

int paged_view(const kllm_b200_paged_cache* c, const char* what, PagedView* v) {
  if (!c) return fail(KLLM_B200_ERR_INVALID_ARG, "%s: null cache", what);
  if (c->cache_dtype != KLLM_B200_F16 && c->cache_dtype != KLLM_B200_I8) {
    return fail(KLLM_B200_ERR_DTYPE, "%s: cache dtype %d not supported (F16, I8)", what, c->cache_dtype);
  }
  if (c->n_pages < 0 || c->n_kv_heads < 0 || c->n_seqs < 0 || c->max_pages < 0) {
    return fail(KLLM_B200_ERR_INVALID_ARG, "%s: negative size", what);
  }
  if (c->head_dim != 64 && c->head_dim != 128) {
    return fail(KLLM_B200_ERR_SHAPE, "%s: head_dim %lld not supported (64, 128)", what, (long long)c->head_dim);
  }
  if (c->page_size < 8 || c->page_size > (1LL << 20) || (c->page_size & (c->page_size - 1)) != 0) {
    return fail(KLLM_B200_ERR_SHAPE, "%s: page_size %lld must be a power of two from 8 to 2^20", what,
                (long long)c->page_size);
  }
  if (c->n_pages == 0 || c->n_kv_heads == 0 || c->n_seqs == 0 || c->max_pages == 0) {
    return fail(KLLM_B200_ERR_SHAPE, "%s: empty cache", what);
  }
  if (c->n_pages > 0x7fffffffLL || c->n_kv_heads > 65535 || c->max_pages > (1LL << 30) / c->page_size ||
      c->n_seqs > 0x7fffffffLL) {
    return fail(KLLM_B200_ERR_SHAPE, "%s: cache too large", what);
  }
  if (!c->k_pages || !c->v_pages || !c->page_table) return fail(KLLM_B200_ERR_INVALID_ARG, "%s: null pointer", what);
  if (c->cache_dtype == KLLM_B200_I8 && (!c->k_scales || !c->v_scales)) {
    return fail(KLLM_B200_ERR_INVALID_ARG, "%s: an I8 cache needs k_scales and v_scales", what);
  }
  if (!aligned16(c->k_pages) || !aligned16(c->v_pages)) {
    return fail(KLLM_B200_ERR_ALIGN, "%s: pages must be 16-byte aligned", what);
  }
  v->table = c->page_table;
  v->max_pages = c->max_pages;
  v->n_seqs = c->n_seqs;
  v->n_pages = static_cast<int>(c->n_pages);
  v->n_kv_heads = static_cast<int>(c->n_kv_heads);
  v->page_shift = 0;
  while ((1LL << v->page_shift) < c->page_size) ++v->page_shift;
  v->capacity = static_cast<int>(c->max_pages * c->page_size);
  return KLLM_B200_OK;
}

int qkv_norm_rope_kv_append_paged(const void* q, int64_t q_stride, const void* k, int64_t k_stride, const void* v,
                                  int64_t v_stride, const void* bq, const void* bk, const void* bv, int bias_dtype,
                                  const void* q_norm, const void* k_norm, int norm_dtype, float eps, float theta,
                                  const int32_t* positions, const int32_t* seqs, int64_t n_tokens, int64_t n_heads,
                                  const kllm_b200_paged_cache* cache, void* q_out, int64_t q_out_stride,
                                  int32_t* err_flags, const LaunchOpts& o) {
  const char* what = "qkv_norm_rope_kv_append_paged";
  if (n_tokens < 0 || n_heads < 0) return fail(KLLM_B200_ERR_INVALID_ARG, "%s: negative size", what);
  AppendArgs a = {};
  const int rc = paged_view(cache, what, &a.view);
  if (rc != KLLM_B200_OK) return rc;
  if (n_tokens == 0) return KLLM_B200_OK;
  if (n_tokens > 0x7fffffffLL) return fail(KLLM_B200_ERR_SHAPE, "%s: too many tokens", what);
  const int64_t D = cache->head_dim, hkv = cache->n_kv_heads;
  if (n_heads == 0 || n_heads > 65535) return fail(KLLM_B200_ERR_SHAPE, "%s: 1 to 65535 query heads", what);
  if ((bq || bk || bv) && !is_float_dtype(bias_dtype)) {
    return fail(KLLM_B200_ERR_DTYPE, "%s: bias dtype %d not supported", what, bias_dtype);
  }
  if ((q_norm || k_norm) && !is_float_dtype(norm_dtype)) {
    return fail(KLLM_B200_ERR_DTYPE, "%s: norm weight dtype %d not supported", what, norm_dtype);
  }
  if (!q || !k || !v || !q_out || !positions || !seqs) return fail(KLLM_B200_ERR_INVALID_ARG, "%s: null pointer", what);
  if (!(theta > 0.f) || !std::isfinite(theta)) return fail(KLLM_B200_ERR_INVALID_ARG, "%s: theta must be positive", what);
  if (!(eps >= 0.f) || !std::isfinite(eps)) return fail(KLLM_B200_ERR_INVALID_ARG, "%s: eps must not be negative", what);
  if (q_stride < n_heads * D || q_out_stride < n_heads * D || k_stride < hkv * D || v_stride < hkv * D) {
    return fail(KLLM_B200_ERR_SHAPE, "%s: a token stride is shorter than the token's row", what);
  }
  if (q_out == q && q_out_stride != q_stride) {
    return fail(KLLM_B200_ERR_SHAPE, "%s: in place, q_out_stride must equal q_stride", what);
  }
  if ((q_stride | k_stride | v_stride | q_out_stride) % 8 != 0) {
    return fail(KLLM_B200_ERR_ALIGN, "%s: token strides must be multiples of 8 elements", what);
  }
  for (const void* p : {q, k, v, static_cast<const void*>(q_out), bq, bk, bv, q_norm, k_norm}) {
    if (!aligned16(p)) return fail(KLLM_B200_ERR_ALIGN, "%s: pointers must be 16-byte aligned", what);
  }
  a.q = static_cast<const __half*>(q);
  a.k = static_cast<const __half*>(k);
  a.v = static_cast<const __half*>(v);
  a.q_stride = q_stride;
  a.k_stride = k_stride;
  a.v_stride = v_stride;
  a.q_out_stride = q_out_stride;
  a.bq = bq;
  a.bk = bk;
  a.bv = bv;
  a.q_norm = q_norm;
  a.k_norm = k_norm;
  a.bias_f32 = bias_dtype == KLLM_B200_F32;
  a.norm_f32 = norm_dtype == KLLM_B200_F32;
  a.eps = eps;
  a.positions = positions;
  a.seqs = seqs;
  a.n_tokens = n_tokens;
  a.n_heads = static_cast<int>(n_heads);
  a.k_pages = cache->k_pages;
  a.v_pages = cache->v_pages;
  a.k_scales = cache->k_scales;
  a.v_scales = cache->v_scales;
  a.q_out = static_cast<__half*>(q_out);
  a.err_flags = err_flags;
  // powers by repeated products: 63 roundings of 2^-53 are 10^-8 of a turn at position 10^6
  const double step = std::pow(static_cast<double>(theta), -2.0 / static_cast<double>(D));
  a.turns[0] = 1.0 / 6.283185307179586476925;
  for (int d = 1; d < D / 2; ++d) a.turns[d] = a.turns[d - 1] * step;
  const int set = static_cast<int>(32 / (D / 16));
  const int64_t sets = (n_heads + 2 * hkv + set - 1) / set;
  const Deal deal = deal_sets(sets, n_tokens);
  a.warps_per_token = deal.warps;
  if (n_tokens * deal.warps >= (int64_t{1} << 31)) return fail(KLLM_B200_ERR_SHAPE, "%s: too many tokens", what);
  const dim3 grid = deal.shared ? dim3(static_cast<unsigned>(n_tokens), static_cast<unsigned>(deal.warps / kWarps))
                                : dim3(static_cast<unsigned>((n_tokens * deal.warps + kWarps - 1) / kWarps));
  const bool i8 = cache->cache_dtype == KLLM_B200_I8;
  void (*kernel)(AppendArgs) = D == 64 ? (i8 ? pick_append<64, true>(deal) : pick_append<64, false>(deal))
                                       : (i8 ? pick_append<128, true>(deal) : pick_append<128, false>(deal));
  return launch_status(launch(kernel, grid, dim3(kThreads), 0, o.stream, o.pdl, a), what);
}

int kv_read_paged(const kllm_b200_paged_cache* cache, const int32_t* positions, const int32_t* seqs, int64_t n_tokens,
                  const int32_t* out_slots, int64_t n_out_slots, int64_t out_max_seq, void* k_out, void* v_out,
                  int32_t* err_flags, const LaunchOpts& o) {
  const char* what = "kv_read_paged";
  if (n_tokens < 0 || n_out_slots < 0 || out_max_seq < 0) {
    return fail(KLLM_B200_ERR_INVALID_ARG, "%s: negative size", what);
  }
  ReadArgs a = {};
  const int rc = paged_view(cache, what, &a.view);
  if (rc != KLLM_B200_OK) return rc;
  if (n_tokens == 0) return KLLM_B200_OK;
  if (n_tokens > 0x7fffffffLL) return fail(KLLM_B200_ERR_SHAPE, "%s: too many tokens", what);
  if (!positions || !seqs || !k_out || !v_out) return fail(KLLM_B200_ERR_INVALID_ARG, "%s: null pointer", what);
  if (out_slots && (n_out_slots == 0 || out_max_seq == 0)) return fail(KLLM_B200_ERR_SHAPE, "%s: empty output cache", what);
  if (!aligned16(k_out) || !aligned16(v_out)) {
    return fail(KLLM_B200_ERR_ALIGN, "%s: outputs must be 16-byte aligned", what);
  }
  a.k_pages = cache->k_pages;
  a.v_pages = cache->v_pages;
  a.k_scales = cache->k_scales;
  a.v_scales = cache->v_scales;
  a.positions = positions;
  a.seqs = seqs;
  a.n_tokens = n_tokens;
  a.out_slots = out_slots;
  a.n_out_slots = n_out_slots;
  a.out_max_seq = out_max_seq;
  a.k_out = static_cast<__half*>(k_out);
  a.v_out = static_cast<__half*>(v_out);
  a.wide = aligned32(k_out) && aligned32(v_out);
  a.err_flags = err_flags;
  if (cache->cache_dtype == KLLM_B200_I8) {
    return cache->head_dim == 64 ? launch_read<64, true>(a, o) : launch_read<128, true>(a, o);
  }
  return cache->head_dim == 64 ? launch_read<64, false>(a, o) : launch_read<128, false>(a, o);
}

}  // namespace kb

extern "C" int kllm_b200_qkv_norm_rope_kv_append_paged(
    const void* q, int64_t q_stride, const void* k, int64_t k_stride, const void* v, int64_t v_stride, const void* bq,
    const void* bk, const void* bv, int bias_dtype, const void* q_norm, const void* k_norm, int norm_dtype, float eps,
    float theta, const int32_t* positions, const int32_t* seqs, int64_t n_tokens, int64_t n_heads,
    const kllm_b200_paged_cache* cache, void* q_out, int64_t q_out_stride, int32_t* err_flags, void* stream) {
  kb::LaunchOpts o;
  o.stream = static_cast<cudaStream_t>(stream);
  return kb::qkv_norm_rope_kv_append_paged(q, q_stride, k, k_stride, v, v_stride, bq, bk, bv, bias_dtype, q_norm, k_norm,
                                           norm_dtype, eps, theta, positions, seqs, n_tokens, n_heads, cache, q_out,
                                           q_out_stride, err_flags, o);
}

extern "C" int kllm_b200_kv_read_paged(const kllm_b200_paged_cache* cache, const int32_t* positions,
                                       const int32_t* seqs, int64_t n_tokens, const int32_t* out_slots,
                                       int64_t n_out_slots, int64_t out_max_seq, void* k_out, void* v_out,
                                       int32_t* err_flags, void* stream) {
  kb::LaunchOpts o;
  o.stream = static_cast<cudaStream_t>(stream);
  return kb::kv_read_paged(cache, positions, seqs, n_tokens, out_slots, n_out_slots, out_max_seq, k_out, v_out, err_flags,
                           o);
}
