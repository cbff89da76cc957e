// Load-balance loss of a router, per-expert counts and the gradient to the logits.
//
// With p[t, .] = softmax(l[t, .]) or sigmoid(l[t, .]) / sum_e sigmoid(l[t, e]), C[s, e] the
// selections of expert e by the counted tokens of sequence s, n[s] their number, S' the number of
// sequences that have any, N = sum_s n[s]:
//   balance = 1/S' sum_s sum_e (E C[s,e] / (k n[s])) (1/n[s]) sum_{t in s} p[t, e]
//           = sum_t a_s sum_e C[s,e] p[t,e],       a_s = E / (k n[s]^2 S')
//   z       = 1/N sum_t logsumexp(l[t, .])^2
// The second form needs no sum of p over the tokens: once the counts (integers, so any order of
// the atomics gives the same ones) are known, each token's term is a dot product with its
// sequence's counts.  With D_t = sum_e C[s,e] p[t,e] the gradients are
//   d balance / d l[t,j] = a_s p[t,j] (C[s,j] - D_t)                  (softmax)
//                        = a_s p[t,j] (1 - sigmoid(l[t,j])) (C[s,j] - D_t)   (sigmoid)
//   d z / d l[t,j]       = (2/N) logsumexp(l[t, .]) softmax(l[t, .])[j]
// Three passes: counts (reads the selections), the losses (reads the logits), the gradient (reads
// the logits again rather than keeping p: the same bytes as reading a kept p, and none written).
//
// With e = exp(-|l|) both sigmoid(l) and 1 - sigmoid(l) are 1 or e over 1 + e: one exponential and one
// reciprocal.  Where every logit of a row is below -40 the sigmoids are taken relative to the
// largest, so that a row whose sigmoids all underflow still has its probabilities.  A row of -inf
// alone has p = 0, adds nothing to either sum and gets a zero gradient; rows that are masked or
// belong to no sequence are not read.
//
// A token is spread over G lanes (the power of two that E fills, at most a warp), V logits a lane,
// and the next token's logits are on their way while one is worked on.  Per-token terms are fp32;
// sums over tokens are kept in double and joined in a fixed order.
#include "dmoe_common.cuh"

namespace dmoe {
namespace {

constexpr int kBalThreads = 256;
constexpr int kMaxGrid = 1184;  // 148 SMs x 8

struct BalArgs {
  const void* logits;
  int T, E, k;
  const int32_t* seq_end;  // NULL: one sequence of T tokens
  int n_seq;
  const uint8_t* mask;  // NULL: every token counts
  int32_t* counts;      // [n_seq][E], then n [n_seq], then a ticket
};

// Ends of the sequences in shared memory where they fit: a search through global memory is a chain
// of loads, 2 us for 37 sequences.
constexpr int kSharedEnds = 1024;
struct Ends {
  const int32_t* at;  // shared or global
  int n, T;
  __device__ __forceinline__ int operator[](int s) const { return at ? min(at[s], T) : T; }
  // First sequence that ends behind token t (n if none does).
  __device__ __forceinline__ int of(int t) const {
    int lo = 0, hi = n;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if ((*this)[mid] > t) hi = mid; else lo = mid + 1;
    }
    return lo;
  }
};

// `sh`: kSharedEnds int32 of shared memory; the caller synchronises the CTA before the first use.
__device__ __forceinline__ Ends fetch_ends(const BalArgs& a, int32_t* sh) {
  if (a.seq_end == nullptr || a.n_seq > kSharedEnds) return Ends{a.seq_end, a.n_seq, a.T};
  for (int s = threadIdx.x; s < a.n_seq; s += kBalThreads) sh[s] = a.seq_end[s];
  return Ends{sh, a.n_seq, a.T};
}

// Selections and counted tokens.  A CTA takes a run of tokens; a sequence that lies in it has its
// histogram built in shared memory and added once.
__global__ void __launch_bounds__(kBalThreads)
    balance_count_kernel(BalArgs a, const int64_t* __restrict__ idx, int run, int32_t* __restrict__ status) {
  extern __shared__ int32_t hist[];  // [E], then the number of tokens
  __shared__ int32_t sh_ends[kSharedEnds];
  const Ends ends = fetch_ends(a, sh_ends);
  if (blockIdx.x == 0 && a.seq_end != nullptr) {
    int bad = 0;
    for (int s = threadIdx.x; s < a.n_seq; s += kBalThreads) {
      const int en = a.seq_end[s], before = s > 0 ? a.seq_end[s - 1] : 0;
      bad |= en < before || en > a.T;
    }
    if (bad) atomicOr(status, DMOE_DEVERR_BAD_SEGMENT);
  }
  for (int e = threadIdx.x; e <= a.E; e += kBalThreads) hist[e] = 0;
  __syncthreads();
  int t0 = (int)min((int64_t)blockIdx.x * run, (int64_t)a.T);
  const int t_end = (int)min((int64_t)t0 + run, (int64_t)a.T);
  int s = ends.of(t0);
  while (t0 < t_end && s < a.n_seq) {  // block-uniform
    const int t1 = min(t_end, ends[s]);
    if (t1 > t0) {
      const unsigned i1 = (unsigned)t1 * a.k;  // T * k < 2^31
      for (unsigned i = (unsigned)t0 * a.k + threadIdx.x; i < i1; i += kBalThreads) {
        const int64_t e = idx[i];
        if (a.mask != nullptr && !a.mask[i / (unsigned)a.k]) continue;
        if (e >= 0 && e < a.E) atomicAdd(&hist[e], 1);
      }
      int mine = 0;
      if (a.mask != nullptr) {
        // unsigned, as i above: a step past t1 may pass 2^31
        for (unsigned t = (unsigned)t0 + threadIdx.x; t < (unsigned)t1; t += kBalThreads) mine += a.mask[t] != 0;
      } else if (threadIdx.x == 0) {
        mine = t1 - t0;
      }
      if (mine) atomicAdd(&hist[a.E], mine);
      __syncthreads();
      int32_t* row = a.counts + (int64_t)s * a.E;
      for (int e = threadIdx.x; e <= a.E; e += kBalThreads) {
        if (hist[e]) atomicAdd(e < a.E ? &row[e] : &a.counts[(int64_t)a.n_seq * a.E + s], hist[e]);
        hist[e] = 0;
      }
      __syncthreads();
      t0 = t1;
    }
    ++s;
  }
}

// Sequences that have tokens and tokens in all, by every thread of the CTA.
__device__ __forceinline__ void totals(const BalArgs& a, int& full, int& tokens) {
  __shared__ int sh[2];
  if (threadIdx.x == 0) sh[0] = sh[1] = 0;
  __syncthreads();
  const int32_t* n = a.counts + (int64_t)a.n_seq * a.E;
  int f = 0, c = 0;
  for (int s = threadIdx.x; s < a.n_seq; s += kBalThreads) {
    f += n[s] > 0;
    c += n[s];
  }
  if (c) {
    atomicAdd(&sh[0], f);
    atomicAdd(&sh[1], c);
  }
  __syncthreads();
  full = sh[0];
  tokens = sh[1];
}

template <int G>
__device__ __forceinline__ float group_max(float v) {
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
template <int G>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

__device__ __forceinline__ float exp_ftz(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x * 1.442695041f));
  return r;
}

// Expert of value i of a lane: runs of four neighbours where a lane has four or more.
template <int G, int V>
__device__ __forceinline__ int expert_of(int i, int lane) {
  return V >= 4 ? (i >> 2) * (4 * G) + lane * 4 + (i & 3) : i * G + lane;
}

// One token's row, -inf where it has no expert or is not read.
template <int G, int V, int DT>
__device__ __forceinline__ void load_row(const void* logits, int64_t row, int E, int lane, bool live, bool vec, float* l) {
  const int64_t base = row * E;
  if (V >= 4 && vec) {
#pragma unroll
    for (int i = 0; i < V; i += 4) {
      const int e = expert_of<G, V>(i, lane);
      float v[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
      if (live && e < E) {
        if constexpr (DT == DMOE_F32) {
          const float4 f = __ldg(reinterpret_cast<const float4*>(reinterpret_cast<const float*>(logits) + base + e));
          v[0] = f.x, v[1] = f.y, v[2] = f.z, v[3] = f.w;
        } else {
          const uint2 w = __ldg(reinterpret_cast<const uint2*>(reinterpret_cast<const char*>(logits) + (base + e) * 2));
          float f[8];
          unpack8<DT>(make_uint4(w.x, w.y, 0, 0), f);
          v[0] = f[0], v[1] = f[1], v[2] = f[2], v[3] = f[3];
        }
      }
#pragma unroll
      for (int j = 0; j < 4 && i + j < V; ++j) l[i + j] = v[j];
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int e = expert_of<G, V>(i, lane);
      l[i] = live && e < E ? load_as_float(logits, base + e, DT) : -INFINITY;
    }
  }
}

// One token's probabilities (not yet divided by their sum) and what its loss terms need.
template <int G, int V, bool SIGMOID>
struct Row {
  float p[V];                         // numerators of p
  float soft[SIGMOID ? V : 1];        // numerators of softmax(l) where p is another thing
  float away[SIGMOID ? V : 1];        // 1 - sigmoid(l)
  float total, soft_total, lse;
  bool any;                           // some logit is above -inf (or is NaN)

  __device__ __forceinline__ void compute(const float* l) {
    float m = l[0];
#pragma unroll
    for (int i = 1; i < V; ++i) m = fmaxf(m, l[i]);  // prefers a number to NaN
    m = group_max<G>(m);
    const float base = m > -INFINITY ? m : 0.f;
    float sum = 0.f, ssum = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float ex = exp_ftz(l[i] - base);
      ssum += ex;
      if constexpr (SIGMOID) {
        soft[i] = ex;
        const float e = exp_ftz(-fabsf(l[i]));
        const float r = __fdividef(1.f, 1.f + e);
        p[i] = (l[i] >= 0.f ? 1.f : e) * r;
        away[i] = (l[i] >= 0.f ? e : 1.f) * r;
        sum += p[i];
      } else {
        p[i] = ex;
      }
    }
    if constexpr (SIGMOID) {
      if (base < -40.f) {  // sigmoid(l) / exp(base), 1 + e is 1
        sum = 0.f;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          p[i] = soft[i];
          sum += p[i];
        }
      }
    }
    soft_total = group_sum<G>(ssum);
    any = !(soft_total == 0.f);  // with a number or NaN in the row the largest term is 1 or NaN
    total = SIGMOID ? group_sum<G>(sum) : soft_total;
    lse = __logf(soft_total) + base;
  }
};

// The tokens [t0, t1) of a group in turn: their sequences, which of them count, and their rows, one
// token ahead.
template <int G, int V, int DT>
struct Walk {
  const BalArgs& a;
  const Ends& ends;
  int t, t1, s, s_end, lane;
  bool vec;
  // the token that comes next
  bool live;
  int seq;
  float l[V];
  __device__ __forceinline__ Walk(const BalArgs& args, const Ends& en, int first, int end, int ln)
      : a(args), ends(en), t(first), t1(end), lane(ln) {
    s = t < t1 ? ends.of(t) : a.n_seq;
    s_end = s < a.n_seq ? ends[s] : a.T;
    vec = a.E % 4 == 0 && (reinterpret_cast<uintptr_t>(a.logits) & 15u) == 0;
    fetch();
  }
  __device__ __forceinline__ void next() {
    if (t < t1) ++t;  // no further: behind the last token t + run may pass 2^31
    fetch();
  }
  __device__ __forceinline__ void fetch() {
    while (t < t1 && s < a.n_seq && t >= s_end) {
      ++s;
      if (s < a.n_seq) s_end = ends[s];
    }
    live = t < t1 && s < a.n_seq && (a.mask == nullptr || a.mask[t]);
    seq = s;
    load_row<G, V, DT>(a.logits, t, a.E, lane, live, vec, l);
  }
};

// The loss terms of a group's tokens [t0, t1), in lane 0 of the group; every group of a warp makes
// `run` steps, since the shuffles span the warp.
template <int G, int V, bool SIGMOID, int DT>
__device__ __forceinline__ void token_losses(const BalArgs& a, const Ends& ends, int full, int t0, int t1, int run,
                                             double& bal, double& zz) {
  const int lane = threadIdx.x & (G - 1);
  const int32_t* n_of = a.counts + (int64_t)a.n_seq * a.E;
  Walk<G, V, DT> w(a, ends, t0, t1, lane);
  int loaded = -1;
  float c[V], coef = 0.f;
  bal = zz = 0.0;
  for (int i = 0; i < run; ++i) {
    const bool live = w.live;
    const int s = w.seq;
    float l[V];
#pragma unroll
    for (int v = 0; v < V; ++v) l[v] = w.l[v];
    if (i + 1 < run) w.next();
    if (live && loaded != s) {
      loaded = s;
      const float n = (float)n_of[s];
      coef = __fdividef((float)a.E, (float)a.k * n) / (n * (float)full);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const int e = expert_of<G, V>(v, lane);
        c[v] = e < a.E ? (float)a.counts[(int64_t)s * a.E + e] : 0.f;
      }
    }
    Row<G, V, SIGMOID> r;
    r.compute(l);
    float dot = 0.f;
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (live) dot += c[v] * r.p[v];
    dot = group_sum<G>(dot);
    if (live && r.any && lane == 0) {
      bal += (double)(coef * __fdiv_rn(dot, r.total));
      zz += (double)r.lse * (double)r.lse;
    }
  }
}

// Sums of two values over the CTA, in a fixed order, by thread 0; `sums` is used again by the next
// call only after a synchronisation.
__device__ __forceinline__ void cta_sums(double& b, double& z, double (*sums)[kBalThreads / 32]) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    b += __shfl_xor_sync(0xffffffffu, b, o);
    z += __shfl_xor_sync(0xffffffffu, z, o);
  }
  if ((threadIdx.x & 31) == 0) {
    sums[0][threadIdx.x >> 5] = b;
    sums[1][threadIdx.x >> 5] = z;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    b = z = 0.0;
    for (int i = 0; i < kBalThreads / 32; ++i) {
      b += sums[0][i];
      z += sums[1][i];
    }
  }
}

template <int G, int V, bool SIGMOID, int DT>
__global__ void __launch_bounds__(kBalThreads)
    balance_loss_kernel(BalArgs a, int run, float* __restrict__ loss, double* __restrict__ part,
                        int32_t* __restrict__ counts_out) {
  __shared__ double sums[2][kBalThreads / 32];
  __shared__ int last;
  __shared__ int32_t sh_ends[kSharedEnds];
  const Ends ends = fetch_ends(a, sh_ends);
  int full, tokens;
  totals(a, full, tokens);  // synchronises
  if (counts_out != nullptr)
    for (int64_t i = (int64_t)blockIdx.x * kBalThreads + threadIdx.x; i < (int64_t)a.n_seq * a.E;
         i += (int64_t)gridDim.x * kBalThreads)
      counts_out[i] = a.counts[i];
  const int group = blockIdx.x * (kBalThreads / G) + threadIdx.x / G;
  const int t0 = (int)min((int64_t)group * run, (int64_t)a.T), t1 = (int)min((int64_t)t0 + run, (int64_t)a.T);
  double b, z;
  token_losses<G, V, SIGMOID, DT>(a, ends, full, t0, t1, run, b, z);
  cta_sums(b, z, sums);
  if (threadIdx.x == 0) {
    part[2 * blockIdx.x] = b;
    part[2 * blockIdx.x + 1] = z;
    __threadfence();
    last = atomicAdd(&a.counts[(int64_t)a.n_seq * (a.E + 1)], 1) == (int)gridDim.x - 1;
  }
  __syncthreads();
  if (!last) return;
  __threadfence();
  // The last CTA joins the parts, each thread its strided run of them in order, then the warps.
  b = z = 0.0;
  for (int i = threadIdx.x; i < (int)gridDim.x; i += kBalThreads) {
    b += __ldcg(&part[2 * i]);
    z += __ldcg(&part[2 * i + 1]);
  }
  cta_sums(b, z, sums);
  if (threadIdx.x == 0) {
    loss[0] = (float)b;
    loss[1] = tokens > 0 ? (float)(z / (double)tokens) : 0.f;
  }
}

// The whole forward pass in one launch, for problems whose three launches cost more than their work:
// a cluster of eight CTAs counts its tokens' selections in shared memory, adds the ranks' counts through
// distributed shared memory and goes on to the losses.
constexpr int kSmallRanks = 8;
constexpr int kSmallCounts = 1024;        // n_seq * (E + 1) at most
// T * E at most.  One launch saves the host 4 us (24.5 against 28.5 a call at every size here), and the GPU
// 3-6 us where tokens are few: 64 x 64 takes 4.3 us against 10.4 in three launches, 512 x 64 7.4 against
// 11.0, 256 x 128 6.1 against 11.3.  The more tokens, the less: 4096 x 8 10.7 against 10.4, and past the limit
// 8192 x 8 17.6 against 10.4 (16384 x 8 then also costs the call: 32.9 against 28.5).
constexpr int64_t kSmallLogits = 1 << 15;

__device__ __forceinline__ uint32_t in_rank(const void* p, int rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_addr(p)), "r"(rank));
  return r;
}
__device__ __forceinline__ void meet_cluster() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

template <int G, int V, bool SIGMOID, int DT>
__global__ void __launch_bounds__(kBalThreads)
    balance_small_kernel(BalArgs a, const int64_t* __restrict__ idx, int run, float* __restrict__ loss,
                         int32_t* __restrict__ counts_out, int32_t* __restrict__ status) {
  __shared__ double sums[2][kBalThreads / 32];
  __shared__ double parts[2][kSmallRanks];
  __shared__ int32_t sh_ends[kSharedEnds];
  __shared__ int32_t mine[kSmallCounts], all[kSmallCounts];
  const int rank = blockIdx.x;  // one cluster
  const Ends ends = fetch_ends(a, sh_ends);
  const int n = a.n_seq * (a.E + 1);
  for (int i = threadIdx.x; i < n; i += kBalThreads) mine[i] = 0;
  __syncthreads();
  if (rank == 0 && a.seq_end != nullptr) {
    int bad = 0;
    for (int s = threadIdx.x; s < a.n_seq; s += kBalThreads) {
      const int en = a.seq_end[s], before = s > 0 ? a.seq_end[s - 1] : 0;
      bad |= en < before || en > a.T;
    }
    if (bad) atomicOr(status, DMOE_DEVERR_BAD_SEGMENT);
  }
  constexpr int kGroups = kBalThreads / G;
  const int first = min(rank * kGroups * run, a.T), end = min(first + kGroups * run, a.T);
  for (int i = first * a.k + threadIdx.x; i < end * a.k; i += kBalThreads) {
    const int t = i / a.k;
    const int64_t e = idx[i];
    if (a.mask != nullptr && !a.mask[t]) continue;
    const int s = ends.of(t);
    if (s >= a.n_seq) continue;
    if (e >= 0 && e < a.E) atomicAdd(&mine[s * a.E + (int)e], 1);
    if (i == t * a.k) atomicAdd(&mine[a.n_seq * a.E + s], 1);  // the token itself, once
  }
  meet_cluster();
  for (int i = threadIdx.x; i < n; i += kBalThreads) {
    int v[kSmallRanks], sum = 0;
#pragma unroll
    for (int r = 0; r < kSmallRanks; ++r)
      asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v[r]) : "r"(in_rank(&mine[i], r)) : "memory");
#pragma unroll
    for (int r = 0; r < kSmallRanks; ++r) sum += v[r];
    all[i] = sum;
    if (rank == 0) {
      a.counts[i] = sum;
      if (counts_out != nullptr && i < a.n_seq * a.E) counts_out[i] = sum;
    }
  }
  BalArgs here = a;
  here.counts = all;
  __syncthreads();
  int full, tokens;
  totals(here, full, tokens);
  const int t0 = min(first + (int)(threadIdx.x / G) * run, a.T), t1 = min(t0 + run, end);
  double b, z;
  token_losses<G, V, SIGMOID, DT>(here, ends, full, t0, t1, run, b, z);
  cta_sums(b, z, sums);
  if (threadIdx.x == 0) {
    asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(in_rank(&parts[0][rank], 0)), "d"(b) : "memory");
    asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(in_rank(&parts[1][rank], 0)), "d"(z) : "memory");
  }
  __syncwarp();
  meet_cluster();
  if (rank == 0 && threadIdx.x == 0) {
    b = z = 0.0;
    for (int r = 0; r < kSmallRanks; ++r) {
      b += parts[0][r];
      z += parts[1][r];
    }
    loss[0] = (float)b;
    loss[1] = tokens > 0 ? (float)(z / (double)tokens) : 0.f;
  }
}

template <int G, int V, bool SIGMOID, int DT>
__global__ void __launch_bounds__(kBalThreads)
    balance_grad_kernel(BalArgs a, int run, const float* __restrict__ g_bal, const float* __restrict__ g_z,
                        void* __restrict__ grad) {
  __shared__ int32_t sh_ends[kSharedEnds];
  const Ends ends = fetch_ends(a, sh_ends);
  int full, tokens;
  totals(a, full, tokens);  // synchronises
  const int lane = threadIdx.x & (G - 1);
  const int group = blockIdx.x * (kBalThreads / G) + threadIdx.x / G;
  const int t0 = (int)min((int64_t)group * run, (int64_t)a.T), t1 = (int)min((int64_t)t0 + run, (int64_t)a.T);
  const int32_t* n_of = a.counts + (int64_t)a.n_seq * a.E;
  const float gb = g_bal ? *g_bal : 0.f;
  const float gz = g_z && tokens > 0 ? *g_z * 2.f / (float)tokens : 0.f;
  const bool vec_out = V >= 4 && a.E % 4 == 0 && (reinterpret_cast<uintptr_t>(grad) & 15u) == 0;
  Walk<G, V, DT> w(a, ends, t0, t1, lane);
  int loaded = -1;
  float c[V], coef = 0.f;
  for (int i = 0; i < run; ++i) {
    const bool live = w.live;
    const int s = w.seq, t = w.t;
    float l[V];
#pragma unroll
    for (int v = 0; v < V; ++v) l[v] = w.l[v];
    if (i + 1 < run) w.next();
    if (live && loaded != s) {
      loaded = s;
      const float n = (float)n_of[s];
      coef = gb * (__fdividef((float)a.E, (float)a.k * n) / (n * (float)full));
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const int e = expert_of<G, V>(v, lane);
        c[v] = e < a.E ? (float)a.counts[(int64_t)s * a.E + e] : 0.f;
      }
    }
    Row<G, V, SIGMOID> r;
    r.compute(l);
    float dot = 0.f;
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (live) dot += c[v] * r.p[v];
    const float inv = 1.f / r.total;
    dot = group_sum<G>(dot) * inv;
    if (t < t1) {
      const bool on = live && r.any;
      const float zc = on && gz != 0.f ? gz * r.lse / r.soft_total : 0.f;
      float d[V];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        d[v] = 0.f;
        if (on) {
          d[v] = coef * (r.p[v] * inv) * (c[v] - dot);
          if constexpr (SIGMOID) d[v] *= r.away[v];
          // left out without a gradient of z: lse may be infinite where the balance is not
          if (gz != 0.f) d[v] += zc * (SIGMOID ? r.soft[SIGMOID ? v : 0] : r.p[v]);
        }
      }
      const int64_t base = (int64_t)t * a.E;
      if (vec_out) {
#pragma unroll
        for (int v = 0; v + 3 < V; v += 4) {
          const int e = expert_of<G, V>(v, lane);
          if (e >= a.E) continue;
          if constexpr (DT == DMOE_F32)
            *reinterpret_cast<float4*>(reinterpret_cast<float*>(grad) + base + e) = make_float4(d[v], d[v + 1], d[v + 2], d[v + 3]);
          else
            *reinterpret_cast<uint2*>(reinterpret_cast<char*>(grad) + (base + e) * 2) =
                make_uint2(pack2<DT>(d[v], d[v + 1]), pack2<DT>(d[v + 2], d[v + 3]));
        }
      } else {
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const int e = expert_of<G, V>(v, lane);
          if (e < a.E) store_from_float(grad, base + e, d[v], DT);
        }
      }
    }
  }
}

// Tokens a group takes and CTAs: about eight CTAs an SM, runs no longer than that needs.
void shape(int T, int per_cta, int* run, int* grid) {
  const int64_t groups = (int64_t)kMaxGrid * per_cta;
  *run = (int)((T + groups - 1) / groups);
  if (*run < 1) *run = 1;
  const int64_t g = ((int64_t)T + (int64_t)per_cta * *run - 1) / ((int64_t)per_cta * *run);
  *grid = (int)(g < 1 ? 1 : g);
}

// Where the forward (grad NULL) and the backward pass write.
struct BalOut {
  const int64_t* small;  // the selections, where one launch does the whole forward pass
  int32_t* status;
  float* loss;
  double* part;
  int32_t* counts_out;
  const float* gb;
  const float* gz;
  void* grad;
  bool backward;
};

template <int G, int V, bool SIGMOID, int DT>
int run_balance(const BalArgs& a, const BalOut& o, cudaStream_t st) {
  int run, grid;
  if (o.small != nullptr) {
    const int per_step = kSmallRanks * (kBalThreads / G);
    run = (a.T + per_step - 1) / per_step;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = kSmallRanks;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.gridDim = dim3(kSmallRanks);
    cfg.blockDim = dim3(kBalThreads);
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    DMOE_CUDA(cudaLaunchKernelEx(&cfg, balance_small_kernel<G, V, SIGMOID, DT>, a, o.small, run, o.loss, o.counts_out,
                                 o.status));
    DMOE_LAUNCH_CHECK();
    return DMOE_OK;
  }
  shape(a.T, kBalThreads / G, &run, &grid);
  if (o.backward)
    balance_grad_kernel<G, V, SIGMOID, DT><<<grid, kBalThreads, 0, st>>>(a, run, o.gb, o.gz, o.grad);
  else
    balance_loss_kernel<G, V, SIGMOID, DT><<<grid, kBalThreads, 0, st>>>(a, run, o.loss, o.part, o.counts_out);
  DMOE_LAUNCH_CHECK();
  return DMOE_OK;
}

template <bool SIGMOID, int DT>
int by_experts(const BalArgs& a, const BalOut& o, cudaStream_t st) {
  if (a.E <= 8) return run_balance<8, 1, SIGMOID, DT>(a, o, st);
  if (a.E <= 16) return run_balance<16, 1, SIGMOID, DT>(a, o, st);
  if (a.E <= 32) return run_balance<32, 1, SIGMOID, DT>(a, o, st);
  if (a.E <= 64) return run_balance<32, 2, SIGMOID, DT>(a, o, st);
  if (a.E <= 128) return run_balance<32, 4, SIGMOID, DT>(a, o, st);
  if (a.E <= 256) return run_balance<32, 8, SIGMOID, DT>(a, o, st);
  if (a.E <= 512) return run_balance<32, 16, SIGMOID, DT>(a, o, st);
  return run_balance<32, 32, SIGMOID, DT>(a, o, st);
}

template <bool SIGMOID>
int by_type(const BalArgs& a, int dt, const BalOut& o, cudaStream_t st) {
  if (dt == DMOE_F32) return by_experts<SIGMOID, DMOE_F32>(a, o, st);
  if (dt == DMOE_BF16) return by_experts<SIGMOID, DMOE_BF16>(a, o, st);
  return by_experts<SIGMOID, DMOE_F16>(a, o, st);
}

int launch_balance(const BalArgs& a, int dt, int mode, const BalOut& o, cudaStream_t st) {
  return mode == DMOE_ROUTER_SOFTMAX ? by_type<false>(a, dt, o, st) : by_type<true>(a, dt, o, st);
}

uintptr_t value_size(int dtype) { return dtype == DMOE_F32 ? 4 : 2; }

int check_balance(const char* name, const void* logits, int dtype, int T, int E, int k, int mode,
                  const int32_t* seq_end, int n_seq, const void* counts) {
  DMOE_REQUIRE(dtype_ok(dtype), "%s: logits must be f32, f16 or bf16", name);
  DMOE_REQUIRE(mode == DMOE_ROUTER_SOFTMAX || mode == DMOE_ROUTER_SIGMOID_GROUP, "%s: bad mode %d", name, mode);
  DMOE_REQUIRE(T >= 0 && E >= 1 && E <= 1024 && k >= 1 && k <= E, "%s: T=%d, E=%d (1..1024), k=%d (1..E)", name, T, E, k);
  DMOE_REQUIRE(n_seq >= 0 && n_seq <= (1 << 20) && (seq_end != nullptr || n_seq <= 1),
               "%s: n_seq=%d (0..2^20; at most 1 without seq_end)", name, n_seq);
  DMOE_REQUIRE((int64_t)T * k < INT32_MAX && (int64_t)n_seq * (E + 1) < INT32_MAX, "%s: too many tokens or sequences",
               name);
  DMOE_REQUIRE(counts != nullptr && (T == 0 || logits != nullptr), "%s: null pointer", name);
  DMOE_REQUIRE((reinterpret_cast<uintptr_t>(logits) & (value_size(dtype) - 1)) == 0 &&
                   (reinterpret_cast<uintptr_t>(counts) & 3u) == 0,
               "%s: logits must be aligned to their type, counts 4-byte aligned", name);
  return DMOE_OK;
}

}  // namespace
}  // namespace dmoe

using namespace dmoe;

extern "C" size_t dmoe_balance_loss_workspace_size(void) { return kMaxGrid * 2 * sizeof(double); }

extern "C" int dmoe_balance_loss(const void* logits, int dtype, const int64_t* idx, int T, int E, int k, int mode,
                                 const int32_t* seq_end, int n_seq, const uint8_t* mask, int32_t* counts,
                                 int32_t* counts_out, float* loss, void* workspace, size_t workspace_bytes, int32_t* dev_status, void* stream) {
  clear_error();
  const char* name = "dmoe_balance_loss";
  if (int r = check_balance(name, logits, dtype, T, E, k, mode, seq_end, n_seq, counts)) return r;
  DMOE_REQUIRE((T == 0 || idx) && loss && workspace && dev_status, "%s: null pointer", name);
  DMOE_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 7u) == 0 && workspace_bytes >= dmoe_balance_loss_workspace_size(),
               "%s: workspace %zu < %zu bytes or not 8-byte aligned", name, workspace_bytes,
               dmoe_balance_loss_workspace_size());
  cudaStream_t st = as_stream(stream);
  const BalArgs a{logits, T, E, k, seq_end, n_seq, mask, counts};
  if (T > 0 && n_seq > 0 && (int64_t)T * E <= kSmallLogits && (int64_t)n_seq * (E + 1) <= kSmallCounts &&
      n_seq <= kSharedEnds) {
    const BalOut o{idx, dev_status, loss, nullptr, counts_out, nullptr, nullptr, nullptr, false};
    return launch_balance(a, dtype, mode, o, st);
  }
  DMOE_CUDA(cudaMemsetAsync(counts, 0, ((size_t)n_seq * (E + 1) + 1) * 4, st));
  if (T == 0 || n_seq == 0) {
    DMOE_CUDA(cudaMemsetAsync(loss, 0, 8, st));
    if (counts_out != nullptr && n_seq > 0) DMOE_CUDA(cudaMemsetAsync(counts_out, 0, (size_t)n_seq * E * 4, st));
    return DMOE_OK;
  }
  // Runs of at least 1024 selections a CTA: shorter ones spend their time on the histogram.
  int run = (1024 + k - 1) / k;
  const int64_t least = ((int64_t)T + kMaxGrid - 1) / kMaxGrid;
  if (run < least) run = (int)least;
  balance_count_kernel<<<(unsigned)(((int64_t)T + run - 1) / run), kBalThreads, (E + 1) * 4, st>>>(a, idx, run, dev_status);
  DMOE_LAUNCH_CHECK();
  const BalOut o{nullptr, nullptr, loss, reinterpret_cast<double*>(workspace), counts_out, nullptr, nullptr, nullptr, false};
  return launch_balance(a, dtype, mode, o, st);
}

extern "C" int dmoe_balance_loss_backward(const void* logits, int dtype, int T, int E, int k, int mode,
                                          const int32_t* seq_end, int n_seq, const uint8_t* mask,
                                          const int32_t* counts, const float* g_balance, const float* g_z,
                                          void* grad, void* stream) {
  clear_error();
  const char* name = "dmoe_balance_loss_backward";
  if (int r = check_balance(name, logits, dtype, T, E, k, mode, seq_end, n_seq, counts)) return r;
  if (T == 0) return DMOE_OK;
  DMOE_REQUIRE(grad != nullptr && (reinterpret_cast<uintptr_t>(grad) & (value_size(dtype) - 1)) == 0,
               "%s: bad gradient pointer", name);
  const BalArgs a{logits, T, E, k, seq_end, n_seq, mask, const_cast<int32_t*>(counts)};
  const BalOut o{nullptr, nullptr, nullptr, nullptr, nullptr, g_balance, g_z, grad, true};
  return launch_balance(a, dtype, mode, o, as_stream(stream));
}
