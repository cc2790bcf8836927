// logprobs.cu — log probability and rank of a given token, entropy and the
// largest entries of each row of logits, from one read of the row.
//
// With m a reference near the row's maximum, s = sum exp(x - m) and
// w = sum exp(x - m) (x - m):
//     log p_i = (x_i - m) - log s,   entropy = log s - w / s.
// Each thread keeps its own (m, s, w) in fp32, moving m only when a batch of
// values exceeds it by more than kLag (sums stay far from overflow, and the
// cancellation in the entropy is bounded by kLag); threads, CTAs of a cluster
// and rows join by the same rescaling: for m' = m + dm, s' = s e^-dm and
// w' = e^-dm (w - dm s).
//
// Largest entries: every thread also keeps the maximum of what it read. The
// k-th largest of these maxima bounds the row's k-th largest value from below,
// and few values reach it, so only the threads whose maximum does look at their
// values again (from L2) and list those at or above the bound. A list that
// overflows (many equal values) is replaced by an exact scan with a sorted list
// per warp. Entries are ordered by (value, lower id first) as one 64-bit
// number, so equal values have one order whatever the schedule.
//
// A row is read by a cluster of 1 to 8 CTAs that join over distributed shared
// memory: one launch, no workspace. Bound: rows * vocab values from HBM, one
// exponential per value.
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

// Sums of a set of values against a reference.
struct Sums {
  float m, s, w;  // {-inf, 0, 0}: nothing yet
  __device__ __forceinline__ void rebase(float to) {  // to >= m
    if (m != to) {
      if (m != -INFINITY) {
        const float dm = fmaxf(m - to, -200.f), f = exp2_approx(dm * kLog2e);  // 0 below e^-200, never 0 * inf
        w = f * fmaf(dm, s, w);
        s *= f;
      }
      m = to;
    }
  }
  __device__ __forceinline__ void join(Sums b) {
    const float top = fmaxf(m, b.m);
    rebase(top);
    b.rebase(top);
    s += b.s;
    w += b.w;
  }
  __device__ __forceinline__ void add(float x, float base) {
    const float d = x - base, e = exp2_approx(d * kLog2e);
    s += e;
    w = fmaf(e, fmaxf(d, -200.f), w);  // e is 0 below e^-200; -inf must not meet it as 0 * inf
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

__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.aligned;\nbarrier.cluster.wait.aligned;\n" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t peer_addr(const void* local, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(local)), "r"(rank));
  return r;
}
__device__ __forceinline__ uint32_t ld_peer32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ unsigned long long ld_peer64(uint32_t addr) {
  unsigned long long v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(addr) : "memory");
  return v;
}

struct Shared {
  unsigned long long top[kMaxTop];             // this CTA's largest entries, sorted
  unsigned long long listed[kListed];          // unsorted candidates
  uint32_t maxima[kThreads];
  float m[kWarps], s[kWarps], w[kWarps];
  int above[kWarps];
  Sums sums;
  int n_above;
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
__global__ void __launch_bounds__(kThreads) token_logprobs_kernel(const __grid_constant__ LogprobArgs a, int n_cta) {
  constexpr int N = Vec<T>::kN;
  __shared__ Shared sh;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t rank = n_cta > 1 ? cluster_rank() : 0;
  const int64_t r = blockIdx.x / n_cta;
  const int k = a.top_k;
  grid_dep_wait();
  grid_dep_launch();
  const Part<T> p = part_of<T>(a, r, rank, n_cta);
  const int token = a.tokens != nullptr ? a.tokens[r] : -1;
  const bool asked = token >= 0 && token < a.vocab;
  const float given = asked ? to_f(p.row[token]) : INFINITY;

  // ---- one read: sums, count above the given token, the thread's maximum
  Sums acc = {-INFINITY, 0.f, 0.f};
  int above = 0;
  float most = -INFINITY;
  auto take = [&](float x) {
    most = fmaxf(most, x);
    if (x > acc.m + kLag || acc.m == -INFINITY) acc.rebase(fmaxf(x, acc.m));
    acc.add(x, acc.m == -INFINITY ? 0.f : acc.m);
    above += x > given;
  };
  if (tid < p.head) take(to_f(p.row[tid]));
  if (tid < p.tail) take(to_f(p.row[p.tail0 + tid]));
  for (int64_t v = p.v0 + tid; v < p.v1; v += kThreads * kBatch) {
    uint4 raw[kBatch];
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      if (v + b * kThreads < p.v1) raw[b] = __ldg(p.body + v + b * kThreads);
    }
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      if (v + b * kThreads < p.v1) {
        float x[N];
        unpack(raw[b], x);
        float top = x[0];
#pragma unroll
        for (int i = 1; i < N; ++i) top = fmaxf(top, x[i]);
        most = fmaxf(most, top);
        if (top > acc.m + kLag || acc.m == -INFINITY) acc.rebase(fmaxf(top, acc.m));
        const float base = acc.m == -INFINITY ? 0.f : acc.m;
#pragma unroll
        for (int i = 0; i < N; ++i) acc.add(x[i], base);
        if (top > given) {
#pragma unroll
          for (int i = 0; i < N; ++i) above += x[i] > given;
        }
      }
    }
  }

  // ---- the CTA's sums
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) {
    Sums b;
    b.m = __shfl_xor_sync(0xffffffffu, acc.m, x);
    b.s = __shfl_xor_sync(0xffffffffu, acc.s, x);
    b.w = __shfl_xor_sync(0xffffffffu, acc.w, x);
    acc.join(b);
  }
  above = __reduce_add_sync(0xffffffffu, above);
  if (lane == 0) {
    sh.m[warp] = acc.m;
    sh.s[warp] = acc.s;
    sh.w[warp] = acc.w;
    sh.above[warp] = above;
  }
  const uint32_t my_most = order_of(most);
  sh.maxima[tid] = my_most;
  if (tid == 0) sh.n_listed = 0;
  if (tid < kMaxTop) sh.top[tid] = 0ull;
  __syncthreads();
  if (tid == 0) {
    Sums all = {-INFINITY, 0.f, 0.f};
    int n = 0;
    for (int w = 0; w < kWarps; ++w) {
      Sums b;
      b.m = sh.m[w];
      b.s = sh.s[w];
      b.w = sh.w[w];
      all.join(b);
      n += sh.above[w];
    }
    sh.sums = all;
    sh.n_above = n;
  }

  if (k > 0) {
    // ---- bound: the k-th largest of the threads' maxima (bit by bit, in warp 0)
    if (warp == 0) {
      uint32_t mine[kThreads / 32];
#pragma unroll
      for (int i = 0; i < kThreads / 32; ++i) mine[i] = sh.maxima[i * 32 + lane];
      uint32_t bound = 0u;
      for (int bit = 31; bit >= 0; --bit) {
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
    auto list_it = [&](float x, int64_t id) {
      const uint32_t o = order_of(x);
      if (o >= bound) {
        const int at = atomicAdd(&sh.n_listed, 1);
        if (at < kListed) sh.listed[at] = entry_of(o, static_cast<uint32_t>(id));
      }
    };
    if (my_most >= bound) {
      if (tid < p.head) list_it(to_f(p.row[tid]), tid);
      if (tid < p.tail) list_it(to_f(p.row[p.tail0 + tid]), p.tail0 + tid);
      for (int64_t v = p.v0 + tid; v < p.v1; v += kThreads) {
        float x[N];
        unpack(__ldg(p.body + v), x);
#pragma unroll
        for (int i = 0; i < N; ++i) list_it(x[i], p.body0 + v * N + i);
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
      for (int64_t v = p.v0 + warp * 32; v < p.v1; v += kThreads) {
        float x[N];
        const bool in = v + lane < p.v1;
        unpack(in ? __ldg(p.body + v + lane) : make_uint4(0u, 0u, 0u, 0u), x);
#pragma unroll
        for (int i = 0; i < N; ++i) {
          insert_all(list, in ? entry_of(order_of(x[i]), static_cast<uint32_t>(p.body0 + (v + lane) * N + i)) : 0ull, k,
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
      if (place < k && e != 0ull) sh.top[place] = e;
    }
  }

  // ---- the row: CTA 0 of the cluster joins and writes
  if (n_cta > 1) cluster_barrier(); else __syncthreads();
  if (rank == 0) {
    Sums all = sh.sums;
    int count = sh.n_above;
    if (n_cta > 1) {
      for (int c = 1; c < n_cta; ++c) {
        Sums b;
        b.m = __uint_as_float(ld_peer32(peer_addr(&sh.sums.m, c)));
        b.s = __uint_as_float(ld_peer32(peer_addr(&sh.sums.s, c)));
        b.w = __uint_as_float(ld_peer32(peer_addr(&sh.sums.w, c)));
        all.join(b);
        count += static_cast<int>(ld_peer32(peer_addr(&sh.n_above, c)));
      }
    }
    const bool nothing = all.s == 0.f;  // every logit is -inf
    const float logs = logf(all.s);
    auto logprob = [&](float x) { return nothing ? -INFINITY : (x - all.m) - logs; };
    if (tid == 0) {
      if (a.tokens != nullptr) {
        if (!asked && token != -1) set_flag(a.err_flags, KLLM_B200_FLAG_BAD_TOKEN);
        a.logprobs[r] = asked ? logprob(given) : 0.f;
        a.ranks[r] = asked ? 1 + count : 0;
      }
      if (a.entropies != nullptr) {
        const float h = logs - all.w / all.s;
        a.entropies[r] = nothing || h < 0.f ? 0.f : h;
      }
    }
    if (k > 0) {
      const int n = n_cta * k;  // <= 256
      for (int i = tid; i < n; i += kThreads) {
        sh.listed[i] = i < k ? sh.top[i] : ld_peer64(peer_addr(&sh.top[i % k], i / k));
      }
      __syncthreads();
      for (int i = tid; i < n; i += kThreads) {
        const unsigned long long e = sh.listed[i];
        int place = 0;
        for (int j = 0; j < n; ++j) place += sh.listed[j] > e;
        if (place < k && e != 0ull) {
          a.top_ids[r * k + place] = static_cast<int32_t>(0xffffffffu - static_cast<uint32_t>(e));
          a.top_logprobs[r * k + place] = logprob(value_of(static_cast<uint32_t>(e >> 32)));
        }
      }
    }
  }
  if (n_cta > 1) cluster_barrier();  // no CTA leaves while its shared memory may be read
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
