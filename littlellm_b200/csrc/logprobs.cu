// logprobs.cu — log probability and rank of a given token, entropy and the
// largest entries of each row of logits, from one read of the row.
//
// With m the maximum, t_i = (x_i - m) log2 e, s = sum 2^t and w = sum 2^t t:
//     log p_i = (x_i - m) - ln s,   entropy = (log2 s - w / s) ln 2.
// All in fp32. Each thread keeps s and w against its warp's maximum m, rescaling
// them where a batch of values brings the warp a new one (three or four times a
// row, where a maximum per thread moves in some lane of nearly every batch);
// warps and CTAs join the same way: for m' = m + dm (dm in log2 units),
// s' = s 2^-dm and w' = 2^-dm (w - dm s). With m the true maximum no term of the
// results cancels another, and the largest term is 1 (for fp16, whose exponent
// is one FMA, once the rounding common to all terms is taken out at the end of
// the row): a row with one possible token has log probability and entropy 0.
//
// Largest entries: every thread also keeps the maximum of what it read, and the
// CTA keeps values in shared memory: all of them where they fit (kKeep vectors),
// else each thread's batch with its maximum. The k-th largest of 64 groups'
// maxima bounds the row's k-th largest value from below, and little more than k
// values reach it; they are listed from what was kept. Only where more of a
// thread than its kept batch reaches the bound are its values read again, by the
// whole CTA. (Reading them again in every case waits for HBM once more, behind
// the streams of the other rows, since the rows under way do not stay in L2:
// 2048 x 151936 fp16 with 5 / 20 entries took 120 / 137 us when the same sums took
// 116 / 119 this way.)
// A list that overflows (many equal values) is replaced by an exact scan with a
// sorted list per warp. Entries are ordered by (value, lower id first) as one
// 64-bit number, so equal values have one order whatever the schedule.
//
// A row is read by a cluster of 1 to 8 CTAs whose parts are pushed to the
// first one's shared memory: one launch, no workspace. Per value there are its
// bytes from HBM, one exponential and 8.6 instructions (0.9 of them for five
// entries: keeping batches, the bound, the list). For 2048 x 151936 fp16 that is
// 95 us at the copy rate, 69 us of the special-function unit and 75 us of issue
// at 1.9 GHz, 82 and 89 us at the 1.6 GHz that the power cap leaves a loop of
// calls; the three do not overlap fully. Kernel alone at full clock 116 to 120 us
// with 5 entries (0.79 to 0.82 of the copy rate), 106 without; a call, repeated,
// 131 to 133 (0.72). One row with 20: 8 to 10 us. Whole batches are loaded without
// predicates into two sets in turn (a copy of 16 registers and as many defaults
// per batch less: 4%). CTAs that stay and load their next row's first batch while
// they finish one took 131 us where these took 118 (spills).
#include <math.h>

#include "ops.cuh"
#include "tcgen05.cuh"  // smem_u32, cluster_rank

namespace kb {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxTop = 32;
constexpr int kMaxCluster = 8;
constexpr int kListed = 512;   // values at or above the bound that fit
constexpr int kKeep = 2560;    // vectors of a CTA that are all kept (40 KB)
constexpr int kBatch = 4;      // 16-byte vectors a thread loads at once
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct LogprobArgs {
  const void* logits;
  int64_t rows, vocab, row_stride;
  const int32_t* tokens;
  float* logprobs;
  int32_t* ranks;
  float* entropies;
  int top_k;
  int32_t* top_ids;
  float* top_logprobs;
  int32_t* err_flags;
};

// Order of the values as unsigned numbers: NaN lowest, then -inf ... +inf; the
// two zeros are one value.
__device__ __forceinline__ uint32_t order_of(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  return x != x ? 0u : b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t o) {
  return o == 0u ? __int_as_float(0x7fffffff) : __uint_as_float(o & 0x80000000u ? o ^ 0x80000000u : ~o);
}
constexpr uint32_t kOrderNegInf = 0x007fffffu;  // order_of(-inf)

__device__ __forceinline__ unsigned long long entry_of(uint32_t order, uint32_t id) {
  return (static_cast<unsigned long long>(order) << 32) | (0xffffffffu - id);
}

// Terms below 2^kFloor are 0 as fp32; t ends there, so that the 0 of a -inf
// logit never meets an infinite t.
constexpr float kFloor = -300.f;

// Sums of a set of values against their maximum. A term is 2^t, t = x log2 e -
// c, c the reference of the maximum m in log2 units. fp16 logits: c = m log2 e
// rounded and t one FMA, off by its own rounding and, alike in every term, by
// that of c; fp32 logits, whose product could leave the range: t = (x - m)
// log2 e, and c stands for m itself.
template <typename T>
struct Sums {
  static constexpr bool kFma = sizeof(T) == 2;
  float m, s, w;  // {-inf, 0, 0}: nothing yet
  static __device__ __forceinline__ float term(float x, float at) {
    return kFma ? fmaf(x, kLog2e, -__fmul_rn(at, kLog2e)) : (x - at) * kLog2e;
  }
  __device__ __forceinline__ void rebase(float to) {  // to >= m
    if (m != to) {
      if (m != -INFINITY) {
        const float step = kFma ? __fsub_rn(__fmul_rn(m, kLog2e), __fmul_rn(to, kLog2e)) : (m - to) * kLog2e;
        const float d = fmaxf(step, kFloor), f = exp2_approx(d);
        w = f * fmaf(d, s, w);
        s *= f;
      }
      m = to;
    }
  }
  // the maximum in use: 0 while everything met is -inf
  __device__ __forceinline__ float base() const { return m == -INFINITY ? 0.f : m; }
  // Before adding values up to `top`, which differs from lane to lane; m does not.
  __device__ __forceinline__ void admit(float top) {
    if (__any_sync(0xffffffffu, top > m)) {
#pragma unroll
      for (int x = 16; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
      rebase(top);
    }
  }
  __device__ __forceinline__ void add(float x) {
    const float t = max_nan(term(x, base()), kFloor), e = exp2_approx(t);
    s += e;
    w = fmaf(e, t, w);
  }
  // Takes the reference's rounding out: every term of a value m is 2^t0 as
  // computed, and is 1 afterwards.
  __device__ __forceinline__ void settle() {
    if (kFma && m != -INFINITY) {
      const float t0 = term(m, m), unit = exp2_approx(t0);
      w = __fsub_rn(w, __fmul_rn(t0, s)) / unit;
      s = s / unit;
    }
  }
};

template <typename T>
struct Vec {
  static constexpr int kN = 16 / sizeof(T);
};
__device__ __forceinline__ void unpack(uint4 v, float (&f)[8]) { unpack8(v, f); }
__device__ __forceinline__ void unpack(uint4 v, float (&f)[4]) {
  f[0] = __uint_as_float(v.x); f[1] = __uint_as_float(v.y); f[2] = __uint_as_float(v.z); f[3] = __uint_as_float(v.w);
}

__device__ __forceinline__ __half2 as_h2(uint32_t v) { return *reinterpret_cast<const __half2*>(&v); }

// kBatch 16-byte vectors of a thread. Vectors past the row's part are -inf,
// which changes no sum, maximum or count.
template <typename T>
struct Batch;

template <>
struct Batch<__half> {
  uint4 v[kBatch];
  static __device__ __forceinline__ uint4 none() { return make_uint4(0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u); }
  // NaN is passed over, as in every maximum here: it reaches the sums by itself
  __device__ __forceinline__ float top() const {
    __half2 m = as_h2(0xfc00fc00u);
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      m = __hmax2(m, __hmax2(__hmax2(as_h2(v[b].x), as_h2(v[b].y)), __hmax2(as_h2(v[b].z), as_h2(v[b].w))));
    }
    return fmaxf(__low2float(m), __high2float(m));
  }
  __device__ __forceinline__ int above(float given) const {
    const __half2 g = __float2half2_rn(given);  // a logit: exact
    __half2 n = as_h2(0u);
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      n = __hadd2(n, __hadd2(__hadd2(__hgt2(as_h2(v[b].x), g), __hgt2(as_h2(v[b].y), g)),
                             __hadd2(__hgt2(as_h2(v[b].z), g), __hgt2(as_h2(v[b].w), g))));
    }
    return static_cast<int>(__low2float(n) + __high2float(n));
  }
  // Two values per packed fp32 instruction; s2, w2 are pairs of partial sums. A
  // -inf is taken as the type's lowest value, whose power is 0 too: one packed
  // maximum instead of a clamp of each t. Only a maximum near the lowest value
  // itself needs the clamps.
  __device__ __forceinline__ void add(float at, unsigned long long& s2, unsigned long long& w2) const {
    if (at > -65000.f) add_all<false>(at, s2, w2); else add_all<true>(at, s2, w2);
  }
  template <bool CLAMP>
  __device__ __forceinline__ void add_all(float at, unsigned long long& s2, unsigned long long& w2) const {
    const float c = -__fmul_rn(at, kLog2e);
    const unsigned long long scale = f32x2_pack(kLog2e, kLog2e), less = f32x2_pack(c, c);
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const uint32_t r[4] = {v[b].x, v[b].y, v[b].z, v[b].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 x = __half22float2(CLAMP ? as_h2(r[i]) : __hmax2_nan(as_h2(r[i]), as_h2(0xfbfffbffu)));
        add_terms<CLAMP>(f32x2_fma(f32x2_pack(x.x, x.y), scale, less), s2, w2);
      }
    }
  }
  template <bool CLAMP>
  static __device__ __forceinline__ void add_terms(unsigned long long t2, unsigned long long& s2, unsigned long long& w2) {
    float lo, hi;
    f32x2_unpack(t2, lo, hi);
    if (CLAMP) {
      lo = max_nan(lo, kFloor);
      hi = max_nan(hi, kFloor);
    }
    const unsigned long long e2 = f32x2_pack(exp2_approx(lo), exp2_approx(hi));
    s2 = f32x2_add(s2, e2);
    w2 = f32x2_fma(e2, f32x2_pack(lo, hi), w2);
  }
};

template <>
struct Batch<float> {
  uint4 v[kBatch];
  static __device__ __forceinline__ uint4 none() { return make_uint4(0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u); }
  __device__ __forceinline__ float top() const {
    float m = -INFINITY;
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      float f[4];
      unpack(v[b], f);
      m = fmaxf(m, fmaxf(fmaxf(f[0], f[1]), fmaxf(f[2], f[3])));
    }
    return m;
  }
  __device__ __forceinline__ int above(float given) const {
    int n = 0;
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      float f[4];
      unpack(v[b], f);
      n += (f[0] > given) + (f[1] > given) + (f[2] > given) + (f[3] > given);
    }
    return n;
  }
  __device__ __forceinline__ void add(float at, unsigned long long& s2, unsigned long long& w2) const {
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      float f[4];
      unpack(v[b], f);
#pragma unroll
      for (int i = 0; i < 4; i += 2) {
        Batch<__half>::add_terms<true>(f32x2_pack(Sums<float>::term(f[i], at), Sums<float>::term(f[i + 1], at)), s2, w2);
      }
    }
  }
};

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.aligned;\n" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.aligned;\n" ::: "memory"); }
// Stores to the same shared variable of the cluster's first CTA.
__device__ __forceinline__ uint32_t first_cta(const void* local) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(smem_u32(local)));
  return r;
}
__device__ __forceinline__ void push32(const void* local, uint32_t v) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(first_cta(local)), "r"(v) : "memory");
}
__device__ __forceinline__ void push64(const void* local, unsigned long long v) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(first_cta(local)), "l"(v) : "memory");
}

struct Shared {
  unsigned long long listed[kListed];              // unsorted candidates
  unsigned long long joined[kMaxCluster * kMaxTop];  // first CTA: every CTA's largest entries
  uint32_t maxima[kThreads];
  float m[kWarps], s[kWarps], w[kWarps];
  int above[kWarps];
  float all_m[kMaxCluster], all_s[kMaxCluster], all_w[kMaxCluster];  // first CTA: every CTA's sums
  int all_above[kMaxCluster];
  uint32_t group[64];      // maxima of 64 groups of threads
  int readers[kThreads];   // threads whose kept batch reaches the bound, from the front,
  int reader_at[kThreads];  // its first vector; from the back, threads to read again
  int n_readers, n_again;
  int n_listed;
  uint32_t bound;
};

// The part of a row one CTA reads: n_vec 16-byte vectors of the aligned body,
// and (first and last CTA) the single values before and after it.
template <typename T>
struct Part {
  const T* row;
  const uint4* body;
  int n_vec;
  int head, tail;    // single values before the body / after it that this CTA reads
  int body0, tail0;  // ids of the first value of this CTA's vectors and of the first tail value
};

template <typename T>
__device__ __forceinline__ Part<T> part_of(const LogprobArgs& a, int64_t r, int rank, int cta_shift) {
  constexpr int N = Vec<T>::kN;
  Part<T> p;
  p.row = static_cast<const T*>(a.logits) + r * a.row_stride;
  const int vocab = static_cast<int>(a.vocab);  // <= 2^30
  const int lead = static_cast<int>(((16 - (reinterpret_cast<uintptr_t>(p.row) & 15)) & 15) / sizeof(T));
  const int head = min(lead, vocab);
  const int n_vec = (vocab - head) / N;
  const int per = (n_vec + (1 << cta_shift) - 1) >> cta_shift;
  const int v0 = min(per * rank, n_vec);
  p.n_vec = min(per, n_vec - v0);
  p.body = reinterpret_cast<const uint4*>(p.row + head) + v0;
  p.body0 = head + v0 * N;
  p.tail0 = head + n_vec * N;
  p.head = rank == 0 ? head : 0;
  p.tail = rank == (1 << cta_shift) - 1 ? vocab - p.tail0 : 0;
  return p;
}

// Joins the sums and counts of `n` (a power of two) lanes' worth of sets; every lane gets all.
template <typename T>
__device__ __forceinline__ void join_lanes(Sums<T>& a, int& count, int n) {
  float top = a.m;
  for (int x = n / 2; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
  a.rebase(top);
  for (int x = n / 2; x > 0; x >>= 1) {
    a.s += __shfl_xor_sync(0xffffffffu, a.s, x);
    a.w += __shfl_xor_sync(0xffffffffu, a.w, x);
    count += __shfl_xor_sync(0xffffffffu, count, x);
  }
}

// The 32 largest of two lists sorted over the lanes, largest first: of each
// pair of opposite places the larger (a bitonic sequence), then its merge.
__device__ __forceinline__ unsigned long long merge_lists(unsigned long long a, unsigned long long b, int lane) {
  b = __shfl_sync(0xffffffffu, b, 31 - lane);
  unsigned long long x = a > b ? a : b;
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) {
    const unsigned long long y = __shfl_xor_sync(0xffffffffu, x, d);
    x = ((lane & d) != 0) == (x > y) ? y : x;
  }
  return x;
}

// Inserts the lanes' entries above the list's k-th into the warp's sorted list
// (lane i holds the i-th largest).
__device__ __forceinline__ void insert_all(unsigned long long& list, unsigned long long mine, int k, int lane) {
  unsigned long long least = __shfl_sync(0xffffffffu, list, k - 1);
  unsigned todo = __ballot_sync(0xffffffffu, mine > least);
  while (todo != 0u) {
    const unsigned long long x = __shfl_sync(0xffffffffu, mine, __ffs(todo) - 1);
    const int at = __popc(__ballot_sync(0xffffffffu, list > x));
    const unsigned long long up = __shfl_up_sync(0xffffffffu, list, 1);
    list = lane < at ? list : lane == at ? x : up;
    least = __shfl_sync(0xffffffffu, list, k - 1);
    todo &= todo - 1;
    todo &= __ballot_sync(0xffffffffu, mine > least);
  }
}

template <typename T, bool KEEP_ALL>
__global__ void __launch_bounds__(kThreads, 4) token_logprobs_kernel(const __grid_constant__ LogprobArgs a,
                                                                     int cta_shift) {
  constexpr int N = Vec<T>::kN;
  // the CTA's vectors, or vector b of thread t's largest batch at b * kThreads + t
  extern __shared__ uint4 kept_all[];
  __shared__ uint4 kept_best[KEEP_ALL ? 1 : kBatch * kThreads];
  uint4* const kept = KEEP_ALL ? kept_all : kept_best;
  __shared__ Shared sh;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int n_cta = 1 << cta_shift;
  const int rank = n_cta > 1 ? static_cast<int>(cluster_rank()) : 0;
  const int64_t r = blockIdx.x >> cta_shift;
  const int k = a.top_k;
  if (rank == 0) {
    for (int i = tid; i < n_cta * k; i += kThreads) sh.joined[i] = 0ull;
  }
  if (n_cta > 1) cluster_arrive();  // waited for before the first store to a peer: by then it has cleared `joined`
  grid_dep_wait();
  grid_dep_launch();
  const int token = a.tokens != nullptr ? a.tokens[r] : -1;
  const Part<T> p = part_of<T>(a, r, rank, cta_shift);
  const int n_vec = p.n_vec;
  // Batch i of the thread, from vector `at`; whole ones load without predicates
  constexpr int kSpan = kThreads * kBatch;
  const int whole = n_vec / kSpan, n_batches = (n_vec + kSpan - 1) / kSpan;
  auto load = [&](Batch<T>& x, int i, int at) {
    if (i < whole) {
#pragma unroll
      for (int b = 0; b < kBatch; ++b) x.v[b] = ld_stream(p.body + at + b * kThreads);
    } else {
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        const int v = at + b * kThreads;
        x.v[b] = v < n_vec ? ld_stream(p.body + v) : Batch<T>::none();
      }
    }
  };
  Batch<T> even, odd;
  load(even, 0, tid);
  const bool asked = token >= 0 && token < a.vocab;
  const float given = asked ? to_f(p.row[token]) : INFINITY;

  // ---- one read: sums, count above the given token, the thread's largest batch
  Sums<T> acc = {-INFINITY, 0.f, 0.f};
  int above = 0;
  int best_at = tid;  // first vector of the kept batch
  float best = -INFINITY, second = -INFINITY, single = -INFINITY;
  const float first = tid < p.head ? to_f(p.row[tid]) : -INFINITY;
  const float last = tid < p.tail ? to_f(p.row[p.tail0 + tid]) : -INFINITY;
  single = fmaxf(first, last);  // -inf, which adds nothing, where there is none
  acc.admit(single);
  acc.add(first);
  acc.add(last);
  above += (first > given) + (last > given);
  auto take = [&](const Batch<T>& x, int at) {
    const float top = x.top();
    second = fmaxf(second, fminf(best, top));
    acc.admit(top);
    if (top > given) above += x.above(given);
    if constexpr (KEEP_ALL) {
      best = fmaxf(best, top);
      if (k > 0) {
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
          if (at + b * kThreads < n_vec) kept[at + b * kThreads] = x.v[b];
        }
      }
    } else if (top > best) {
      best = top;
      if (k > 0) {
#pragma unroll
        for (int b = 0; b < kBatch; ++b) kept[b * kThreads + tid] = x.v[b];
        best_at = at;
      }
    }
    unsigned long long s2 = f32x2_pack(acc.s, 0.f), w2 = f32x2_pack(acc.w, 0.f);
    x.add(acc.base(), s2, w2);
    float lo, hi;
    f32x2_unpack(s2, lo, hi);
    acc.s = lo + hi;
    f32x2_unpack(w2, lo, hi);
    acc.w = lo + hi;
  };
  for (int i = 0, at = tid; i < n_batches; i += 2, at += 2 * kSpan) {
    load(odd, i + 1, at + kSpan);
    take(even, at);
    if (i + 1 == n_batches) break;
    load(even, i + 2, at + 2 * kSpan);
    take(odd, at + kSpan);
  }

  // ---- the CTA's sums
  join_lanes(acc, above, 32);
  if (lane == 0) {
    sh.m[warp] = acc.m;
    sh.s[warp] = acc.s;
    sh.w[warp] = acc.w;
    sh.above[warp] = above;
  }
  sh.maxima[tid] = order_of(fmaxf(best, single));
  if (tid == 0) sh.n_listed = sh.n_readers = sh.n_again = 0;
  if (n_cta > 1) cluster_wait();
  __syncthreads();
  if (warp == kWarps - 1) {
    Sums<T> all = {sh.m[lane % kWarps], sh.s[lane % kWarps], sh.w[lane % kWarps]};
    int n = sh.above[lane % kWarps];
    join_lanes(all, n, kWarps);
    if (lane == 0) {
      if (rank == 0) {
        sh.all_m[0] = all.m;
        sh.all_s[0] = all.s;
        sh.all_w[0] = all.w;
        sh.all_above[0] = n;
      } else {
        push32(&sh.all_m[rank], __float_as_uint(all.m));
        push32(&sh.all_s[rank], __float_as_uint(all.s));
        push32(&sh.all_w[rank], __float_as_uint(all.w));
        push32(&sh.all_above[rank], static_cast<uint32_t>(n));
      }
    }
  }

  if (k > 0) {
    // ---- bound: the k-th largest of 64 maxima, each over the same lane of
    // every other warp, by the numbers above and at each; four lanes a group
    const int g = tid >> 2, sub = tid & 3;
    uint32_t mine = sh.maxima[(2 * sub + (g >> 5)) * 32 + (g & 31)];
    mine = max(mine, __shfl_xor_sync(0xffffffffu, mine, 1));
    mine = max(mine, __shfl_xor_sync(0xffffffffu, mine, 2));
    if (sub == 0) sh.group[g] = mine;
    __syncthreads();
    int counts = 0;  // those above, and 2^16 times those at or above
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      const uint4 o = *reinterpret_cast<const uint4*>(&sh.group[16 * sub + i]);
      counts += (o.x > mine) + (o.y > mine) + (o.z > mine) + (o.w > mine);
      counts += ((o.x >= mine) + (o.y >= mine) + (o.z >= mine) + (o.w >= mine)) << 16;
    }
    counts += __shfl_xor_sync(0xffffffffu, counts, 1);
    counts += __shfl_xor_sync(0xffffffffu, counts, 2);
    // threads without a value carry -inf as well: such a bound says nothing
    if ((counts & 0xffff) < k && counts >> 16 >= k) sh.bound = mine <= kOrderNegInf ? 0u : mine;
    __syncthreads();
    const uint32_t bound = sh.bound;
    const float least = value_of(bound);  // NaN where everything counts
    // the values of a vector that reach the bound
    auto list_vector = [&](uint4 raw, int v) {
      float x[N];
      unpack(raw, x);
      unsigned hits = 0u;
#pragma unroll
      for (int j = 0; j < N; ++j) hits |= x[j] >= least ? 1u << j : 0u;
      if (bound == 0u) hits = (1u << N) - 1u;
      if (hits != 0u) {
        int at = atomicAdd(&sh.n_listed, __popc(hits));
#pragma unroll
        for (int j = 0; j < N; ++j) {
          if (hits >> j & 1u) {
            if (at < kListed) sh.listed[at] = entry_of(order_of(x[j]), p.body0 + v * N + j);
            ++at;
          }
        }
      }
    };
    auto list_single = [&](float x, int id) {
      if (bound == 0u || x >= least) {
        const int at = atomicAdd(&sh.n_listed, 1);
        if (at < kListed) sh.listed[at] = entry_of(order_of(x), id);
      }
    };
    if (tid < p.head) list_single(first, tid);
    if (tid < p.tail) list_single(last, p.tail0 + tid);
    if (!KEEP_ALL && (bound == 0u || second >= least)) {
      sh.readers[kThreads - 1 - atomicAdd(&sh.n_again, 1)] = tid;
    } else if (bound == 0u || best >= least) {
      const int at = atomicAdd(&sh.n_readers, 1);
      sh.readers[at] = tid;
      sh.reader_at[at] = KEEP_ALL ? tid : best_at;
    }
    __syncthreads();
    // the kept vectors of the listed threads, dealt to all
    const unsigned per_reader = (n_vec + kThreads - 1) / kThreads;  // vectors of a thread
    const unsigned per_kept = KEEP_ALL ? per_reader : kBatch, n_kept = sh.n_readers * per_kept;
    for (unsigned i = tid; i < n_kept; i += kThreads) {
      if (*static_cast<volatile int*>(&sh.n_listed) > kListed) break;  // the list is full already
      const unsigned q = i / per_kept, b = i - q * per_kept;
      const int at = sh.reader_at[q] + b * kThreads;
      if (at < n_vec) list_vector(kept[KEEP_ALL ? at : b * kThreads + sh.readers[q]], at);
    }
    // the vectors of the threads to read again
    const unsigned n_items = sh.n_again * per_reader;
    for (unsigned i0 = tid; i0 < n_items; i0 += kThreads * kBatch) {
      if (*static_cast<volatile int*>(&sh.n_listed) > kListed) break;  // the list is full already
      Batch<T> again;
      int at[kBatch];
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        const unsigned i = i0 + b * kThreads, q = i / per_reader;
        at[b] = i < n_items ? sh.readers[kThreads - 1 - q] + static_cast<int>(i - q * per_reader) * kThreads : n_vec;
        again.v[b] = at[b] < n_vec ? __ldg(p.body + at[b]) : Batch<T>::none();
      }
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        if (at[b] < n_vec) list_vector(again.v[b], at[b]);
      }
    }
    __syncthreads();
    int n = sh.n_listed;
    if (n > kListed) {
      // ---- too many: a sorted list per warp over everything
      unsigned long long list = 0ull;
      insert_all(list, tid < p.head ? entry_of(order_of(first), tid) : 0ull, k, lane);
      insert_all(list, tid < p.tail ? entry_of(order_of(last), p.tail0 + tid) : 0ull, k, lane);
      for (int v = warp * 32; v < n_vec; v += kThreads) {
        float x[N];
        const bool in = v + lane < n_vec;
        unpack(in ? __ldg(p.body + v + lane) : make_uint4(0u, 0u, 0u, 0u), x);
#pragma unroll
        for (int i = 0; i < N; ++i) {
          insert_all(list, in ? entry_of(order_of(x[i]), p.body0 + (v + lane) * N + i) : 0ull, k, lane);
        }
      }
      __syncthreads();
      if (lane < k) sh.listed[warp * k + lane] = list;
      n = kWarps * k;
      __syncthreads();
    }
    // ---- the CTA's k largest: an entry's place is the number above it, counted by eight lanes
    for (int i0 = 0; i0 < n; i0 += kThreads / 8) {
      const int i = i0 + tid / 8;
      const unsigned long long e = i < n ? sh.listed[i] : 0ull;
      int place = 0;
      for (int j = tid % 8; j < n; j += 8) place += sh.listed[j] > e;
#pragma unroll
      for (int x = 1; x < 8; x <<= 1) place += __shfl_xor_sync(0xffffffffu, place, x);
      if (tid % 8 == 0 && place < k && e != 0ull) {
        if (rank == 0) sh.joined[place] = e; else push64(&sh.joined[rank * k + place], e);
      }
    }
  }

  // ---- the row: the first CTA joins and writes
  if (n_cta > 1) {
    cluster_arrive();
    cluster_wait();
  } else {
    __syncthreads();
  }
  if (rank != 0) return;
  if (warp == kWarps - 1) {
    Sums<T> all = {sh.all_m[lane % n_cta], sh.all_s[lane % n_cta], sh.all_w[lane % n_cta]};
    int count = sh.all_above[lane % n_cta];
    join_lanes(all, count, n_cta);
    all.settle();
    const bool nothing = all.s == 0.f;  // every logit is -inf
    const float logs = nothing ? INFINITY : log2f(all.s);  // then every log probability is -inf
    const float lns = logs * kLn2;
    if (lane == 0) {
      sh.m[0] = nothing ? 0.f : all.m;
      sh.s[0] = lns;
      if (a.tokens != nullptr) {
        if (!asked && token != -1) set_flag(a.err_flags, KLLM_B200_FLAG_BAD_TOKEN);
        a.logprobs[r] = !asked ? 0.f : nothing ? -INFINITY : (given - all.m) - lns;
        a.ranks[r] = asked ? 1 + count : 0;
      }
      if (a.entropies != nullptr) {
        const float h = (logs - all.w / all.s) * kLn2;
        a.entropies[r] = nothing || h < 0.f ? 0.f : h;
      }
    }
  }
  if (k == 0) return;
  // the cluster's lists, two by two
  for (int m = n_cta / 2; m > 0; m /= 2) {
    if (warp < m) {
      const unsigned long long x = merge_lists(lane < k ? sh.joined[warp * k + lane] : 0ull,
                                               lane < k ? sh.joined[(warp + m) * k + lane] : 0ull, lane);
      if (lane < k) sh.joined[warp * k + lane] = x;
    }
    if (m > 1) __syncthreads();
  }
  __syncthreads();
  if (tid < k) {
    const unsigned long long e = sh.joined[tid];
    const float x = value_of(static_cast<uint32_t>(e >> 32));
    a.top_ids[r * k + tid] = static_cast<int32_t>(0xffffffffu - static_cast<uint32_t>(e));
    a.top_logprobs[r * k + tid] = sh.s[0] == INFINITY ? -INFINITY : (x - sh.m[0]) - sh.s[0];
  }
}

// log2 of the CTAs per row: rows are split while their CTAs stay within two per
// SM and each keeps at least 4096 values. Measured, us, rows of 151936 fp16 with
// 5 entries, 1 / 2 / 4 / 8 CTAs a row: 8 rows 14.0 / 10.6 / 8.6 / 7.3, 64 rows
// 15.2 / 11.6 / 11.5 / 12.5, 256 rows 23.3 / 24.7 / 28.0 / 39.0.
int cluster_shift_for(int64_t rows, int64_t vocab) {
  int c = 0;
  while ((1 << c) < kMaxCluster && (rows << (c + 1)) <= 2LL * sm_count() && (vocab >> (c + 1)) >= 4096) ++c;
  return c;
}

// KEEP_ALL: the CTA's `vectors` all fit in shared memory.
template <typename T, bool KEEP_ALL>
int launch_logprobs(const LogprobArgs& a, int cta_shift, int64_t vectors, const LaunchOpts& o) {
  auto kernel = token_logprobs_kernel<T, KEEP_ALL>;
  size_t smem = 0;
  if constexpr (KEEP_ALL) {
    // opted in to the most any call keeps: with the static part it passes the default 48 KB
    const cudaError_t err = allow_smem(reinterpret_cast<const void*>(kernel), kKeep * 16 + sizeof(Shared));
    if (err != cudaSuccess) return launch_status(err, "token_logprobs: shared memory opt-in");
    if (a.top_k > 0) smem = static_cast<size_t>(vectors) * 16;
  }
  const dim3 grid(static_cast<unsigned>(a.rows << cta_shift));
  const cudaError_t err =
      cta_shift == 0 ? launch(kernel, grid, dim3(kThreads), smem, o.stream, o.pdl, a, 0)
                     : launch_clustered(kernel, grid, dim3(kThreads), smem, o.stream, o.pdl, 1 << cta_shift, a,
                                        cta_shift);
  return launch_status(err, "token_logprobs");
}

template <typename T>
int run_logprobs(const LogprobArgs& a, const LaunchOpts& o) {
  const int c = cluster_shift_for(a.rows, a.vocab);
  const int64_t vectors = ((a.vocab / Vec<T>::kN) >> c) + 1;  // of a CTA, at most
  return vectors <= kKeep ? launch_logprobs<T, true>(a, c, vectors, o) : launch_logprobs<T, false>(a, c, vectors, o);
}

}  // namespace

int token_logprobs(const void* logits, int dtype, int64_t rows, int64_t vocab, int64_t row_stride,
                   const int32_t* tokens, float* logprobs, int32_t* ranks, float* entropies, int top_k,
                   int32_t* top_ids, float* top_logprobs, int32_t* err_flags, const LaunchOpts& o) {
  const char* what = "token_logprobs";
  if (rows < 0 || vocab < 0 || top_k < 0) return fail(KLLM_B200_ERR_INVALID_ARG, "%s: negative size", what);
  if (!is_float_dtype(dtype)) return fail(KLLM_B200_ERR_DTYPE, "%s: dtype %d not supported (F16, F32)", what, dtype);
  if (vocab == 0 || vocab > (1LL << 30)) return fail(KLLM_B200_ERR_SHAPE, "%s: vocab must be 1 to 2^30", what);
  if (rows > 0x7fffffffLL / kMaxCluster) return fail(KLLM_B200_ERR_SHAPE, "%s: too many rows", what);
  if (row_stride < vocab) return fail(KLLM_B200_ERR_SHAPE, "%s: row_stride is shorter than a row", what);
  if (top_k > kMaxTop || top_k > vocab) {
    return fail(KLLM_B200_ERR_SHAPE, "%s: top_k %d must be at most %d and at most vocab", what, top_k, kMaxTop);
  }
  if (rows == 0) return KLLM_B200_OK;
  if (!logits) return fail(KLLM_B200_ERR_INVALID_ARG, "%s: null pointer", what);
  if ((tokens != nullptr) != (logprobs != nullptr) || (tokens != nullptr) != (ranks != nullptr)) {
    return fail(KLLM_B200_ERR_INVALID_ARG, "%s: tokens, logprobs and ranks go together", what);
  }
  if (top_k > 0 && (!top_ids || !top_logprobs)) {
    return fail(KLLM_B200_ERR_INVALID_ARG, "%s: top_k needs top_ids and top_logprobs", what);
  }
  if (reinterpret_cast<uintptr_t>(logits) % dtype_size(dtype) != 0) {
    return fail(KLLM_B200_ERR_ALIGN, "%s: logits are not aligned to their element type", what);
  }
  LogprobArgs a = {logits,    rows,  vocab,   row_stride,   tokens,   logprobs, ranks,
                   entropies, top_k, top_ids, top_logprobs, err_flags};
  return dtype == KLLM_B200_F16 ? run_logprobs<__half>(a, o) : run_logprobs<float>(a, o);
}

}  // namespace kb

extern "C" int kllm_b200_token_logprobs(const void* logits, int dtype, int64_t rows, int64_t vocab, int64_t row_stride,
                                        const int32_t* tokens, float* logprobs, int32_t* ranks, float* entropies,
                                        int top_k, int32_t* top_ids, float* top_logprobs, int32_t* err_flags,
                                        void* stream) {
  kb::LaunchOpts o;
  o.stream = static_cast<cudaStream_t>(stream);
  return kb::token_logprobs(logits, dtype, rows, vocab, row_stride, tokens, logprobs, ranks, entropies, top_k, top_ids,
                            top_logprobs, err_flags, o);
}
