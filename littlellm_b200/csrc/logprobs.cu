// logprobs.cu — log probability and rank of a given token, entropy and the
// largest entries of each row of logits, from one read of the row.
//
// With c a reference near the row's maximum, t_i = (x_i - c) log2 e,
// s = sum 2^t and w = sum 2^t t:
//     log2 p_i = t_i - log2 s,   entropy = (log2 s - w / s) ln 2.
// Each thread keeps its own (c, s, w) in fp32, moving c only when a batch of
// values exceeds it by more than kLag (sums stay far from overflow, and what
// the entropy's two terms cancel is bounded); threads and CTAs join by the same
// rescaling: for c' = c + dc, s' = s 2^-dc and w' = 2^-dc (w - dc s).
//
// fp16 logits take t as one FMA, x log2 e - c', with the reference c' kept in
// log2 units: the rounding of c' moves all t alike and cancels. fp32 logits
// subtract first (x log2 e would overflow at the type's end).
//
// Largest entries: every thread also keeps the maximum of what it read. The
// k-th largest of these maxima bounds the row's k-th largest value from below,
// and about k values reach it. The threads whose maximum does are listed, and
// the CTA reads their values again together (from L2), listing those at or
// above the bound. A list that overflows (many equal values) is replaced by an
// exact scan with a sorted list per warp. Entries are ordered by (value, lower
// id first) as one 64-bit number, so equal values have one order whatever the
// schedule.
//
// A row is read by a cluster of 1 to 8 CTAs whose parts are pushed to the
// first one's shared memory: one launch, no workspace. Bound: rows * vocab
// values from HBM; one exponential per value (the special-function unit needs
// three quarters of the time that fp16 values need from HBM), about five
// issue slots per value.
#include <math.h>

#include "ops.cuh"
#include "tcgen05.cuh"  // smem_u32

namespace kb {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxTop = 32;
constexpr int kMaxCluster = 8;
constexpr int kListed = 512;   // values at or above the bound that fit
constexpr int kBatch = 4;      // 16-byte vectors a thread loads at once
constexpr float kLag = 8.f;
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

// 2^x in one instruction (2 ulp; results below the normal range are 0).
__device__ __forceinline__ float exp2_approx(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// The larger of two values, NaN when either is.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Terms below 2^kFloor are 0 as fp32; t ends there, so that the 0 of a -inf
// logit never meets an infinite t.
constexpr float kFloor = -300.f;

// How a type's values relate to the reference (fp16: in log2 units, fp32: the
// value itself).
template <typename T>
struct Scale;
template <>
struct Scale<__half> {
  static constexpr float kUnit = kLog2e;  // reference units per logit
  static __device__ __forceinline__ float t_of(float x, float ref) { return __fmaf_rn(x, kLog2e, -ref); }
  static __device__ __forceinline__ float between(float from, float to) { return from - to; }
  // log p of x, given log2 of the sum
  static __device__ __forceinline__ float log_of(float x, float ref, float logs) { return (t_of(x, ref) - logs) * kLn2; }
};
template <>
struct Scale<float> {
  static constexpr float kUnit = 1.f;
  static __device__ __forceinline__ float t_of(float x, float ref) { return (x - ref) * kLog2e; }
  static __device__ __forceinline__ float between(float from, float to) { return (from - to) * kLog2e; }
  static __device__ __forceinline__ float log_of(float x, float ref, float logs) { return (x - ref) - logs * kLn2; }
};

// Sums of a set of values against a reference.
template <typename T>
struct Sums {
  float ref, s, w;  // {-inf, 0, 0}: nothing yet
  __device__ __forceinline__ void rebase(float to) {  // to >= ref
    if (ref != to) {
      if (ref != -INFINITY) {
        const float d = fmaxf(Scale<T>::between(ref, to), kFloor), f = exp2_approx(d);
        w = f * fmaf(d, s, w);
        s *= f;
      }
      ref = to;
    }
  }
  __device__ __forceinline__ void join(Sums b) {
    const float top = fmaxf(ref, b.ref);
    rebase(top);
    b.rebase(top);
    s += b.s;
    w += b.w;
  }
  // the reference in use: 0 while everything met is -inf
  __device__ __forceinline__ float base() const { return ref == -INFINITY ? 0.f : ref; }
  __device__ __forceinline__ void admit(float top) {  // before adding values up to `top`
    if (top * Scale<T>::kUnit > ref + kLag || ref == -INFINITY) rebase(fmaxf(top * Scale<T>::kUnit, ref));
  }
  __device__ __forceinline__ void add(float x, float at) {
    const float t = max_nan(Scale<T>::t_of(x, at), kFloor), e = exp2_approx(t);
    s += e;
    w = fmaf(e, t, w);
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
  // Two values per packed fp32 instruction; s2, w2 are pairs of partial sums.
  __device__ __forceinline__ void add(float at, unsigned long long& s2, unsigned long long& w2) const {
    const unsigned long long scale = f32x2_pack(kLog2e, kLog2e), shift = f32x2_pack(-at, -at);
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const uint32_t r[4] = {v[b].x, v[b].y, v[b].z, v[b].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 x = h2_to_f2(r[i]);
        unsigned long long t2;
        asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(t2) : "l"(f32x2_pack(x.x, x.y)), "l"(scale), "l"(shift));
        add_terms(t2, s2, w2);
      }
    }
  }
  static __device__ __forceinline__ void add_terms(unsigned long long t2, unsigned long long& s2, unsigned long long& w2) {
    float lo, hi;
    f32x2_unpack(t2, lo, hi);
    lo = max_nan(lo, kFloor);
    hi = max_nan(hi, kFloor);
    const unsigned long long e2 = f32x2_pack(exp2_approx(lo), exp2_approx(hi));
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(s2) : "l"(s2), "l"(e2));
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(w2) : "l"(e2), "l"(f32x2_pack(lo, hi)), "l"(w2));
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
        Batch<__half>::add_terms(f32x2_pack(Scale<float>::t_of(f[i], at), Scale<float>::t_of(f[i + 1], at)), s2, w2);
      }
    }
  }
};

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.aligned;\n" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.aligned;\n" ::: "memory"); }
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
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
  float ref[kWarps], s[kWarps], w[kWarps];
  int above[kWarps];
  float all_ref[kMaxCluster], all_s[kMaxCluster], all_w[kMaxCluster];  // first CTA: every CTA's sums
  int all_above[kMaxCluster];
  int readers[kThreads];  // threads whose maximum reaches the bound
  int n_readers;
  int n_listed;
  uint32_t bound;
};

// The part of a row one CTA reads: 16-byte vectors [v0, v1) of the aligned
// body, and (first and last CTA) the single values before and after it.
template <typename T>
struct Part {
  const T* row;
  const uint4* body;
  int64_t v0, v1;
  int head, tail;       // single values before the body / after it that this CTA reads
  int64_t body0, tail0;  // ids of the first body value and of the first tail value
};

template <typename T>
__device__ __forceinline__ Part<T> part_of(const LogprobArgs& a, int64_t r, uint32_t rank, uint32_t n_cta) {
  constexpr int N = Vec<T>::kN;
  Part<T> p;
  p.row = static_cast<const T*>(a.logits) + r * a.row_stride;
  const int64_t lead =
      static_cast<int64_t>(((16 - (reinterpret_cast<uintptr_t>(p.row) & 15)) & 15) / sizeof(T));
  const int64_t head = lead < a.vocab ? lead : a.vocab;
  const int64_t n_vec = (a.vocab - head) / N;
  const int64_t per = (n_vec + n_cta - 1) / n_cta;
  p.body = reinterpret_cast<const uint4*>(p.row + head);
  p.v0 = min(per * rank, n_vec);
  p.v1 = min(p.v0 + per, n_vec);
  p.body0 = head;
  p.tail0 = head + n_vec * N;
  p.head = rank == 0 ? static_cast<int>(head) : 0;
  p.tail = rank == n_cta - 1 ? static_cast<int>(a.vocab - p.tail0) : 0;
  return p;
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

template <typename T>
__global__ void __launch_bounds__(kThreads, 4) token_logprobs_kernel(const __grid_constant__ LogprobArgs a, int n_cta) {
  constexpr int N = Vec<T>::kN;
  __shared__ Shared sh;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t rank = n_cta > 1 ? cluster_rank() : 0;
  const int64_t r = blockIdx.x / n_cta;
  const int k = a.top_k;
  if (rank == 0) {
    for (int i = tid; i < n_cta * k; i += kThreads) sh.joined[i] = 0ull;
  }
  if (n_cta > 1) cluster_arrive();  // waited for before the first store to a peer: by then it has cleared `joined`
  grid_dep_wait();
  grid_dep_launch();
  const Part<T> p = part_of<T>(a, r, rank, n_cta);
  const int n_vec = static_cast<int>(p.v1 - p.v0);  // of the CTA; vocab <= 2^30
  const uint4* body = p.body + p.v0;
  auto load = [&](Batch<T>& x, int at) {
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int v = at + b * kThreads;
      x.v[b] = v < n_vec ? __ldg(body + v) : Batch<T>::none();
    }
  };
  Batch<T> next;
  load(next, tid);
  const int token = a.tokens != nullptr ? a.tokens[r] : -1;
  const bool asked = token >= 0 && token < a.vocab;
  const float given = asked ? to_f(p.row[token]) : INFINITY;

  // ---- one read: sums, count above the given token, the thread's maximum
  Sums<T> acc = {-INFINITY, 0.f, 0.f};
  int above = 0;
  float most = -INFINITY;
  auto take = [&](float x) {
    most = fmaxf(most, x);
    acc.admit(x);
    acc.add(x, acc.base());
    above += x > given;
  };
  if (tid < p.head) take(to_f(p.row[tid]));
  if (tid < p.tail) take(to_f(p.row[p.tail0 + tid]));
  for (int at = tid; at < n_vec; at += kThreads * kBatch) {
    const Batch<T> x = next;
    load(next, at + kThreads * kBatch);
    const float top = x.top();
    most = fmaxf(most, top);
    acc.admit(top);
    if (top > given) above += x.above(given);
    unsigned long long s2 = f32x2_pack(acc.s, 0.f), w2 = f32x2_pack(acc.w, 0.f);
    x.add(acc.base(), s2, w2);
    float lo, hi;
    f32x2_unpack(s2, lo, hi);
    acc.s = lo + hi;
    f32x2_unpack(w2, lo, hi);
    acc.w = lo + hi;
  }

  // ---- the CTA's sums
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) {
    Sums<T> b;
    b.ref = __shfl_xor_sync(0xffffffffu, acc.ref, x);
    b.s = __shfl_xor_sync(0xffffffffu, acc.s, x);
    b.w = __shfl_xor_sync(0xffffffffu, acc.w, x);
    acc.join(b);
  }
  above = __reduce_add_sync(0xffffffffu, above);
  if (lane == 0) {
    sh.ref[warp] = acc.ref;
    sh.s[warp] = acc.s;
    sh.w[warp] = acc.w;
    sh.above[warp] = above;
  }
  const uint32_t my_most = order_of(most);
  sh.maxima[tid] = my_most;
  if (tid == 0) sh.n_listed = sh.n_readers = 0;
  if (n_cta > 1) cluster_wait();
  __syncthreads();
  if (tid == kThreads - 1) {
    Sums<T> all = {-INFINITY, 0.f, 0.f};
    int n = 0;
    for (int w = 0; w < kWarps; ++w) {
      all.join({sh.ref[w], sh.s[w], sh.w[w]});
      n += sh.above[w];
    }
    if (rank == 0) {
      sh.all_ref[0] = all.ref;
      sh.all_s[0] = all.s;
      sh.all_w[0] = all.w;
      sh.all_above[0] = n;
    } else {
      push32(&sh.all_ref[rank], __float_as_uint(all.ref));
      push32(&sh.all_s[rank], __float_as_uint(all.s));
      push32(&sh.all_w[rank], __float_as_uint(all.w));
      push32(&sh.all_above[rank], static_cast<uint32_t>(n));
    }
  }

  if (k > 0) {
    // ---- bound: the k-th largest of the threads' maxima, bit by bit from the
    // first one in which they differ (fp16 values end at bit 13)
    if (warp == 0) {
      uint32_t mine[kThreads / 32], least = 0xffffffffu, largest = 0u;
#pragma unroll
      for (int i = 0; i < kThreads / 32; ++i) {
        mine[i] = sh.maxima[i * 32 + lane];
        least = min(least, mine[i]);
        largest = max(largest, mine[i]);
      }
      least = __reduce_min_sync(0xffffffffu, least);
      largest = __reduce_max_sync(0xffffffffu, largest);
      constexpr int kLowBit = sizeof(T) == 2 ? 13 : 0;
      const int first = 31 - __clz(least ^ largest);  // -1: all equal
      uint32_t bound = first < 0 ? least : largest >> first >> 1 << first << 1;
      for (int bit = first; bit >= kLowBit; --bit) {
        const uint32_t trial = bound | (1u << bit);
        int n = 0;
#pragma unroll
        for (int i = 0; i < kThreads / 32; ++i) n += mine[i] >= trial;
        if (static_cast<int>(__reduce_add_sync(0xffffffffu, n)) >= k) bound = trial;
      }
      // threads without a value carry -inf as well: such a bound says nothing
      if (lane == 0) sh.bound = bound <= kOrderNegInf ? 0u : bound;
    }
    __syncthreads();
    const uint32_t bound = sh.bound;
    if (my_most >= bound) sh.readers[atomicAdd(&sh.n_readers, 1)] = tid;
    auto list_it = [&](float x, int64_t id) {
      const uint32_t o = order_of(x);
      if (o >= bound) {
        const int at = atomicAdd(&sh.n_listed, 1);
        if (at < kListed) sh.listed[at] = entry_of(o, static_cast<uint32_t>(id));
      }
    };
    if (tid < p.head) list_it(to_f(p.row[tid]), tid);
    if (tid < p.tail) list_it(to_f(p.row[p.tail0 + tid]), p.tail0 + tid);
    __syncthreads();
    const int n_readers = sh.n_readers;
    for (int i = warp; i < n_readers; i += kWarps) {
      const int from = sh.readers[i];
      for (int v = from + lane * kThreads; v < n_vec; v += 32 * kThreads) {
        float x[N];
        unpack(__ldg(body + v), x);
        float top = x[0];
#pragma unroll
        for (int j = 1; j < N; ++j) top = fmaxf(top, x[j]);
        if (bound == 0u || order_of(top) >= bound) {
#pragma unroll
          for (int j = 0; j < N; ++j) list_it(x[j], p.body0 + (p.v0 + v) * N + j);
        }
      }
    }
    __syncthreads();
    int n = sh.n_listed;
    if (n > kListed) {
      // ---- too many: a sorted list per warp over everything
      unsigned long long list = 0ull;
      insert_all(list, tid < p.head ? entry_of(order_of(to_f(p.row[tid])), tid) : 0ull, k, lane);
      insert_all(list,
                 tid < p.tail ? entry_of(order_of(to_f(p.row[p.tail0 + tid])), static_cast<uint32_t>(p.tail0 + tid))
                              : 0ull,
                 k, lane);
      for (int v = warp * 32; v < n_vec; v += kThreads) {
        float x[N];
        const bool in = v + lane < n_vec;
        unpack(in ? __ldg(body + v + lane) : make_uint4(0u, 0u, 0u, 0u), x);
#pragma unroll
        for (int i = 0; i < N; ++i) {
          insert_all(list,
                     in ? entry_of(order_of(x[i]), static_cast<uint32_t>(p.body0 + (p.v0 + v + lane) * N + i)) : 0ull, k,
                     lane);
        }
      }
      __syncthreads();
      if (lane < k) sh.listed[warp * k + lane] = list;
      n = kWarps * k;
      __syncthreads();
    }
    // ---- the CTA's k largest: an entry's place is the number above it
    for (int i = tid; i < n; i += kThreads) {
      const unsigned long long e = sh.listed[i];
      int place = 0;
      for (int j = 0; j < n; ++j) place += sh.listed[j] > e;
      if (place < k && e != 0ull) {
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
  Sums<T> all = {sh.all_ref[0], sh.all_s[0], sh.all_w[0]};
  int count = sh.all_above[0];
  for (int c = 1; c < n_cta; ++c) {
    all.join({sh.all_ref[c], sh.all_s[c], sh.all_w[c]});
    count += sh.all_above[c];
  }
  const bool nothing = all.s == 0.f;  // every logit is -inf
  const float logs = log2f(all.s);
  auto logprob = [&](float x) { return nothing ? -INFINITY : Scale<T>::log_of(x, all.ref, logs); };
  if (tid == 0) {
    if (a.tokens != nullptr) {
      if (!asked && token != -1) set_flag(a.err_flags, KLLM_B200_FLAG_BAD_TOKEN);
      a.logprobs[r] = asked ? logprob(given) : 0.f;
      a.ranks[r] = asked ? 1 + count : 0;
    }
    if (a.entropies != nullptr) {
      const float h = (logs - all.w / all.s) * kLn2;
      a.entropies[r] = nothing || h < 0.f ? 0.f : h;
    }
  }
  const int n = n_cta * k;  // <= kThreads
  if (tid < n) {
    const unsigned long long e = sh.joined[tid];
    int place = tid;
    if (n_cta > 1) {
      place = 0;
      for (int j = 0; j < n; ++j) place += sh.joined[j] > e;
    }
    if (place < k && e != 0ull) {
      a.top_ids[r * k + place] = static_cast<int32_t>(0xffffffffu - static_cast<uint32_t>(e));
      a.top_logprobs[r * k + place] = logprob(value_of(static_cast<uint32_t>(e >> 32)));
    }
  }
}

// CTAs per row: rows are split while the device has CTA slots to spare and a
// CTA keeps at least 4096 values.
int cluster_for(int64_t rows, int64_t vocab) {
  int c = 1;
  while (c < kMaxCluster && rows * c * 2 <= 2LL * sm_count() && vocab / (2 * c) >= 4096) c *= 2;
  return c;
}

template <typename T>
int launch_logprobs(const LogprobArgs& a, const LaunchOpts& o) {
  const char* what = "token_logprobs";
  const int c = cluster_for(a.rows, a.vocab);
  const dim3 grid(static_cast<unsigned>(a.rows * c));
  if (c == 1) {
    return launch_status(launch(token_logprobs_kernel<T>, grid, dim3(kThreads), 0, o.stream, o.pdl, a, c), what);
  }
  return launch_status(launch_clustered(token_logprobs_kernel<T>, grid, dim3(kThreads), 0, o.stream, o.pdl, c, a, c),
                       what);
}

}  // namespace

int token_logprobs(const void* logits, int dtype, int64_t rows, int64_t vocab, int64_t row_stride,
                   const int32_t* tokens, float* logprobs, int32_t* ranks, float* entropies, int top_k,
                   int32_t* top_ids, float* top_logprobs, int32_t* err_flags, const LaunchOpts& o) {
  const char* what = "token_logprobs";
  if (rows < 0 || vocab < 0 || top_k < 0) return fail(KLLM_B200_ERR_INVALID_ARG, "%s: negative size", what);
  if (!is_float_dtype(dtype)) return fail(KLLM_B200_ERR_DTYPE, "%s: dtype %d not supported (F16, F32)", what, dtype);
  if (vocab == 0 || vocab > (1LL << 30)) return fail(KLLM_B200_ERR_SHAPE, "%s: vocab must be 1 to 2^30", what);
  if (rows * kMaxCluster > 0x7fffffffLL) return fail(KLLM_B200_ERR_SHAPE, "%s: too many rows", what);
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
  return dtype == KLLM_B200_F16 ? launch_logprobs<__half>(a, o) : launch_logprobs<float>(a, o);
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
