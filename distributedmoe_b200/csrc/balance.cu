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
// p of the sigmoid form is taken relative to the row's largest logit, so that a row whose sigmoids
// all underflow still has its probabilities.  A row of -inf alone has p = 0, adds nothing to
// either sum and gets a zero gradient; rows that are masked or belong to no sequence are not read.
//
// A token is spread over G lanes (the power of two that E fills, at most a warp), V logits a lane.
// Per-token terms are fp32; sums over tokens are kept in double and joined in a fixed order.
#include "dmoe_common.cuh"

namespace dmoe {
namespace {

constexpr int kBalThreads = 256;
constexpr int kMaxGrid = 1024;

struct BalArgs {
  const void* logits;
  int T, E, k;
  const int32_t* seq_end;  // NULL: one sequence of T tokens
  int n_seq;
  const uint8_t* mask;  // NULL: every token counts
  int32_t* counts;      // [n_seq][E], then n [n_seq], then a ticket
};

__device__ __forceinline__ int seq_end_of(const BalArgs& a, int s) { return a.seq_end ? min(a.seq_end[s], a.T) : a.T; }

// First sequence that ends behind token t (n_seq if none does).
__device__ __forceinline__ int seq_of(const BalArgs& a, int t) {
  int lo = 0, hi = a.n_seq;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (seq_end_of(a, mid) > t) hi = mid; else lo = mid + 1;
  }
  return lo;
}

// Selections and counted tokens.  A CTA takes a run of tokens; a sequence that lies in it has its
// histogram built in shared memory and added once.
__global__ void __launch_bounds__(kBalThreads)
    balance_count_kernel(BalArgs a, const int64_t* __restrict__ idx, int run, int32_t* __restrict__ status) {
  extern __shared__ int32_t hist[];  // [E], then the number of tokens
  if (blockIdx.x == 0 && a.seq_end != nullptr) {
    int bad = 0;
    for (int s = threadIdx.x; s < a.n_seq; s += kBalThreads) {
      const int en = a.seq_end[s], before = s > 0 ? a.seq_end[s - 1] : 0;
      bad |= en < before || en > a.T;
    }
    if (bad) atomicOr(status, DMOE_DEVERR_BAD_SEGMENT);
  }
  int t0 = min((int64_t)blockIdx.x * run, (int64_t)a.T);
  const int t_end = min((int64_t)t0 + run, (int64_t)a.T);
  int s = seq_of(a, t0);
  while (t0 < t_end && s < a.n_seq) {  // block-uniform
    const int t1 = min(t_end, seq_end_of(a, s));
    if (t1 > t0) {
      for (int e = threadIdx.x; e <= a.E; e += kBalThreads) hist[e] = 0;
      __syncthreads();
      const int64_t i1 = (int64_t)t1 * a.k;
      for (int64_t i = (int64_t)t0 * a.k + threadIdx.x; i < i1; i += kBalThreads) {
        if (a.mask != nullptr && !a.mask[i / a.k]) continue;
        const int64_t e = idx[i];
        if (e >= 0 && e < a.E) atomicAdd(&hist[e], 1);
      }
      int mine = 0;
      if (a.mask != nullptr) {
        for (int t = t0 + threadIdx.x; t < t1; t += kBalThreads) mine += a.mask[t] != 0;
      } else if (threadIdx.x == 0) {
        mine = t1 - t0;
      }
      if (mine) atomicAdd(&hist[a.E], mine);
      __syncthreads();
      int32_t* row = a.counts + (int64_t)s * a.E;
      for (int e = threadIdx.x; e < a.E; e += kBalThreads)
        if (hist[e]) atomicAdd(&row[e], hist[e]);
      if (threadIdx.x == 0 && hist[a.E]) atomicAdd(&a.counts[(int64_t)a.n_seq * a.E + s], hist[a.E]);
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

// One token's probabilities (not yet divided by their sum) and what its loss terms need.
template <int G, int V, bool SIGMOID>
struct Row {
  float p[V];     // numerators of p
  float soft[SIGMOID ? V : 1];  // numerators of softmax(l) where p is another thing
  float total, soft_total, lse;
  bool any;       // some logit is above -inf (or is NaN)

  __device__ __forceinline__ void load(const void* logits, int dt, int64_t row, int E, int lane, bool live, float* l) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int e = i * G + lane;
      l[i] = live && e < E ? load_as_float(logits, row * E + e, dt) : -INFINITY;
    }
  }

  __device__ __forceinline__ void compute(const float* l) {
    float m = l[0];
#pragma unroll
    for (int i = 1; i < V; ++i) m = fmaxf(m, l[i]);  // prefers a number to NaN
    m = group_max<G>(m);
    const float base = m > -INFINITY ? m : 0.f;
    float sum = 0.f, ssum = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float ex = __expf(l[i] - base);
      ssum += ex;
      if constexpr (SIGMOID) {
        soft[i] = ex;
        // sigmoid(l) = exp(min(l, 0)) / (1 + exp(-|l|)), over its largest exp(min(base, 0))
        p[i] = __fdividef(__expf(fminf(l[i], 0.f) - fminf(base, 0.f)), 1.f + __expf(-fabsf(l[i])));
        sum += p[i];
        if (l[i] != l[i]) sum = l[i];  // the minimum above prefers a number, too
      } else {
        p[i] = ex;
      }
    }
    soft_total = group_sum<G>(ssum);
    any = !(soft_total == 0.f);  // with a number or NaN in the row the largest term is 1 or NaN
    total = SIGMOID ? group_sum<G>(sum) : soft_total;
    lse = __logf(soft_total) + base;
  }
};

template <int G, int V, bool SIGMOID>
__global__ void __launch_bounds__(kBalThreads)
    balance_loss_kernel(BalArgs a, int dt, int run, float* __restrict__ loss, double* __restrict__ part) {
  __shared__ double sums[2][kBalThreads / 32];
  __shared__ int last;
  int full, tokens;
  totals(a, full, tokens);
  const int lane = threadIdx.x & (G - 1);
  const int group = blockIdx.x * (kBalThreads / G) + threadIdx.x / G;  // takes tokens [t0, t1)
  const int t0 = (int)min((int64_t)group * run, (int64_t)a.T), t1 = (int)min((int64_t)t0 + run, (int64_t)a.T);
  const int32_t* n_of = a.counts + (int64_t)a.n_seq * a.E;
  int s = t0 < t1 ? seq_of(a, t0) : a.n_seq, loaded = -1;
  int s_end = s < a.n_seq ? seq_end_of(a, s) : a.T;
  float c[V], coef = 0.f;
  double bal = 0.0, zz = 0.0;
  for (int i = 0; i < run; ++i) {  // every group makes `run` steps: the shuffles span the warp
    const int t = t0 + i;
    while (t < t1 && s < a.n_seq && t >= s_end) {
      ++s;
      if (s < a.n_seq) s_end = seq_end_of(a, s);
    }
    const bool live = t < t1 && s < a.n_seq && (a.mask == nullptr || a.mask[t]);
    if (live && loaded != s) {
      loaded = s;
      const float n = (float)n_of[s];
      coef = __fdividef((float)a.E, (float)a.k * n) / (n * (float)full);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const int e = v * G + lane;
        c[v] = e < a.E ? (float)a.counts[(int64_t)s * a.E + e] : 0.f;
      }
    }
    Row<G, V, SIGMOID> r;
    float l[V];
    r.load(a.logits, dt, t, a.E, lane, live, l);
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
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    bal += __shfl_xor_sync(0xffffffffu, bal, o);
    zz += __shfl_xor_sync(0xffffffffu, zz, o);
  }
  if ((threadIdx.x & 31) == 0) {
    sums[0][threadIdx.x >> 5] = bal;
    sums[1][threadIdx.x >> 5] = zz;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    double b = 0.0, z = 0.0;
    for (int w = 0; w < kBalThreads / 32; ++w) {
      b += sums[0][w];
      z += sums[1][w];
    }
    part[2 * blockIdx.x] = b;
    part[2 * blockIdx.x + 1] = z;
    __threadfence();
    last = atomicAdd(&a.counts[(int64_t)a.n_seq * (a.E + 1)], 1) == (int)gridDim.x - 1;
  }
  __syncthreads();
  if (!last) return;
  __threadfence();
  // The last CTA joins the parts, each warp-strided run of them in order, then the warps.
  double b = 0.0, z = 0.0;
  for (int i = threadIdx.x; i < (int)gridDim.x; i += kBalThreads) {
    b += __ldcg(&part[2 * i]);
    z += __ldcg(&part[2 * i + 1]);
  }
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
    for (int w = 0; w < kBalThreads / 32; ++w) {
      b += sums[0][w];
      z += sums[1][w];
    }
    loss[0] = (float)b;
    loss[1] = tokens > 0 ? (float)(z / (double)tokens) : 0.f;
  }
}

template <int G, int V, bool SIGMOID>
__global__ void __launch_bounds__(kBalThreads)
    balance_grad_kernel(BalArgs a, int dt, int run, const float* __restrict__ g_bal, const float* __restrict__ g_z,
                        void* __restrict__ grad) {
  int full, tokens;
  totals(a, full, tokens);
  const int lane = threadIdx.x & (G - 1);
  const int group = blockIdx.x * (kBalThreads / G) + threadIdx.x / G;
  const int t0 = (int)min((int64_t)group * run, (int64_t)a.T), t1 = (int)min((int64_t)t0 + run, (int64_t)a.T);
  const int32_t* n_of = a.counts + (int64_t)a.n_seq * a.E;
  const float gb = g_bal ? *g_bal : 0.f;
  const float gz = g_z && tokens > 0 ? *g_z * 2.f / (float)tokens : 0.f;
  int s = t0 < t1 ? seq_of(a, t0) : a.n_seq, loaded = -1;
  int s_end = s < a.n_seq ? seq_end_of(a, s) : a.T;
  float c[V], coef = 0.f;
  for (int i = 0; i < run; ++i) {
    const int t = t0 + i;
    while (t < t1 && s < a.n_seq && t >= s_end) {
      ++s;
      if (s < a.n_seq) s_end = seq_end_of(a, s);
    }
    const bool live = t < t1 && s < a.n_seq && (a.mask == nullptr || a.mask[t]);
    if (live && loaded != s) {
      loaded = s;
      const float n = (float)n_of[s];
      coef = gb * (__fdividef((float)a.E, (float)a.k * n) / (n * (float)full));
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const int e = v * G + lane;
        c[v] = e < a.E ? (float)a.counts[(int64_t)s * a.E + e] : 0.f;
      }
    }
    Row<G, V, SIGMOID> r;
    float l[V];
    r.load(a.logits, dt, t, a.E, lane, live, l);
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
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const int e = v * G + lane;
        if (e < a.E) {
          float d = 0.f;
          if (on) {
            d = coef * (r.p[v] * inv) * (c[v] - dot);
            if constexpr (SIGMOID) {
              const float x = __expf(-fabsf(l[v]));
              d *= __fdividef(l[v] >= 0.f ? x : 1.f, 1.f + x);  // 1 - sigmoid(l)
            }
            // left out without a gradient of z: lse may be infinite where the balance is not
            if (gz != 0.f) d += zc * (SIGMOID ? r.soft[SIGMOID ? v : 0] : r.p[v]);
          }
          store_from_float(grad, (int64_t)t * a.E + e, d, dt);
        }
      }
    }
  }
}

// Tokens a group takes and CTAs: up to four CTAs an SM, runs no longer than that needs.
void shape(int T, int per_cta, int* run, int* grid) {
  const int64_t groups = (int64_t)kMaxGrid / 2 * per_cta;
  *run = (int)((T + groups - 1) / groups);
  if (*run < 1) *run = 1;
  const int64_t g = ((int64_t)T + (int64_t)per_cta * *run - 1) / ((int64_t)per_cta * *run);
  *grid = (int)(g < 1 ? 1 : g);
}

template <int G, int V, bool SIGMOID>
int run_balance(const BalArgs& a, int dt, float* loss, double* part, const float* gb, const float* gz, void* grad,
                cudaStream_t st) {
  int run, grid;
  shape(a.T, kBalThreads / G, &run, &grid);
  if (grad == nullptr)
    balance_loss_kernel<G, V, SIGMOID><<<grid, kBalThreads, 0, st>>>(a, dt, run, loss, part);
  else
    balance_grad_kernel<G, V, SIGMOID><<<grid, kBalThreads, 0, st>>>(a, dt, run, gb, gz, grad);
  DMOE_LAUNCH_CHECK();
  return DMOE_OK;
}

template <bool SIGMOID>
int dispatch_balance(const BalArgs& a, int dt, float* loss, double* part, const float* gb, const float* gz, void* grad,
                     cudaStream_t st) {
#define DMOE_BAL(G, V) return run_balance<G, V, SIGMOID>(a, dt, loss, part, gb, gz, grad, st)
  if (a.E <= 8) DMOE_BAL(8, 1);
  if (a.E <= 16) DMOE_BAL(16, 1);
  if (a.E <= 32) DMOE_BAL(32, 1);
  if (a.E <= 64) DMOE_BAL(32, 2);
  if (a.E <= 128) DMOE_BAL(32, 4);
  if (a.E <= 256) DMOE_BAL(32, 8);
  if (a.E <= 512) DMOE_BAL(32, 16);
  DMOE_BAL(32, 32);
#undef DMOE_BAL
}

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
  DMOE_REQUIRE((reinterpret_cast<uintptr_t>(logits) & 3u) == 0 && (reinterpret_cast<uintptr_t>(counts) & 3u) == 0,
               "%s: logits and counts must be 4-byte aligned", name);
  return DMOE_OK;
}

}  // namespace
}  // namespace dmoe

using namespace dmoe;

extern "C" size_t dmoe_balance_loss_workspace_size(void) { return kMaxGrid * 2 * sizeof(double); }

extern "C" int dmoe_balance_loss(const void* logits, int dtype, const int64_t* idx, int T, int E, int k, int mode,
                                 const int32_t* seq_end, int n_seq, const uint8_t* mask, int32_t* counts, float* loss,
                                 void* workspace, size_t workspace_bytes, int32_t* dev_status, void* stream) {
  clear_error();
  const char* name = "dmoe_balance_loss";
  if (int r = check_balance(name, logits, dtype, T, E, k, mode, seq_end, n_seq, counts)) return r;
  DMOE_REQUIRE((T == 0 || idx) && loss && workspace && dev_status, "%s: null pointer", name);
  DMOE_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 7u) == 0 && workspace_bytes >= dmoe_balance_loss_workspace_size(),
               "%s: workspace %zu < %zu bytes or not 8-byte aligned", name, workspace_bytes,
               dmoe_balance_loss_workspace_size());
  cudaStream_t st = as_stream(stream);
  DMOE_CUDA(cudaMemsetAsync(counts, 0, ((size_t)n_seq * (E + 1) + 1) * 4, st));
  if (T == 0 || n_seq == 0) {
    DMOE_CUDA(cudaMemsetAsync(loss, 0, 8, st));
    return DMOE_OK;
  }
  const BalArgs a{logits, T, E, k, seq_end, n_seq, mask, counts};
  // Runs of at least 1024 selections a CTA: shorter ones spend their time on the histogram.
  int run = (1024 + k - 1) / k;
  const int64_t least = ((int64_t)T + kMaxGrid - 1) / kMaxGrid;
  if (run < least) run = (int)least;
  balance_count_kernel<<<(T + run - 1) / run, kBalThreads, (E + 1) * 4, st>>>(a, idx, run, dev_status);
  DMOE_LAUNCH_CHECK();
  double* part = reinterpret_cast<double*>(workspace);
  return mode == DMOE_ROUTER_SOFTMAX ? dispatch_balance<false>(a, dtype, loss, part, nullptr, nullptr, nullptr, st)
                                     : dispatch_balance<true>(a, dtype, loss, part, nullptr, nullptr, nullptr, st);
}

extern "C" int dmoe_balance_loss_backward(const void* logits, int dtype, int T, int E, int k, int mode,
                                          const int32_t* seq_end, int n_seq, const uint8_t* mask,
                                          const int32_t* counts, const float* g_balance, const float* g_z,
                                          void* grad, void* stream) {
  clear_error();
  const char* name = "dmoe_balance_loss_backward";
  if (int r = check_balance(name, logits, dtype, T, E, k, mode, seq_end, n_seq, counts)) return r;
  if (T == 0) return DMOE_OK;
  DMOE_REQUIRE(grad != nullptr && (reinterpret_cast<uintptr_t>(grad) & 3u) == 0, "%s: bad gradient pointer", name);
  const BalArgs a{logits, T, E, k, seq_end, n_seq, mask, const_cast<int32_t*>(counts)};
  cudaStream_t st = as_stream(stream);
  return mode == DMOE_ROUTER_SOFTMAX ? dispatch_balance<false>(a, dtype, nullptr, nullptr, g_balance, g_z, grad, st)
                                     : dispatch_balance<true>(a, dtype, nullptr, nullptr, g_balance, g_z, grad, st);
}
