// Objectives on a model's own answers: log-probabilities of chosen tokens with their entropy and the gradient of both, the clipped policy
// loss with a KL term on logits, the paired preference loss on log-probabilities.  Every call is asynchronous, keeps no scratch of its own
// (what is carried from one kernel to the next lies in the caller's outputs) and sums in a fixed order.
#include <math.h>

#include <algorithm>

#include "objectives.cuh"

namespace {
// Bit 8: offsets that do not ascend inside the rows (the answer counts as empty).  Part of the library image, so that no call allocates;
// femto_status_word(NULL, ..) reads and clears it.
__device__ unsigned int g_objectives_status = 0;

// One value for the whole block of 1024 threads: fixed tree.
template <typename S> __device__ S block_total(S v) {
  __shared__ S red[32];
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = red[threadIdx.x & 31];
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

__global__ void __launch_bounds__(1024) k_count_targets(const int* __restrict__ tgt0, int N, int V, int* __restrict__ out) {
  pdl_trigger();
  int n = 0;
  for (unsigned i0 = threadIdx.x; i0 < (unsigned)N; i0 += 8 * 1024) {      // eight in flight: the first rows' slopes wait for this
    int t[8];
#pragma unroll
    for (int k = 0; k < 8; k++) t[k] = i0 + k * 1024 < (unsigned)N ? tgt0[i0 + k * 1024] : -1;
#pragma unroll
    for (int k = 0; k < 8; k++) n += t[k] >= 0 && t[k] < V;
  }
  n = block_total(n);
  if (threadIdx.x == 0) *out = n;
}

// Sum (or mean over the rows with a target) of the token losses, and how many tokens the clipping held.  One block, or a cluster for many
// rows (60000 rows: 40 us with one block, 8 with eight).
__global__ void __launch_bounds__(1024) k_policy_sum(const RowsArgs p, int mean, float* loss_out, int* n_valid_out, int* n_clipped_out) {
  pdl_trigger();
  __shared__ double sums[MOST_CLUSTER];      // token losses have both signs: their sum is held in 64 bits
  __shared__ int counts[2][MOST_CLUSTER];
  const int C = (int)cluster_size(), rank = (int)cluster_rank();
  if (C > 1) asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory");
  pdl_wait();
  double sum = 0.0;
  int n = 0, clipped = 0;
  const unsigned N = p.N, step = C * 1024;
  for (unsigned i0 = rank * 1024 + threadIdx.x; i0 < N; i0 += 4 * step) {
    int t[4];
    float loss[4], lp[4], old[4], A[4];
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const unsigned i = min(i0 + k * step, N - 1);
      t[k] = p.tgt0[i];
      loss[k] = __ldcg(p.token_losses + i);      // 0 without a target
      lp[k] = __ldcg(p.logp + i);
      old[k] = p.old[i];
      A[k] = p.adv[i];
    }
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const bool has = t[k] >= 0 && t[k] < p.V && i0 + k * step < N;
      n += has;
      sum += has ? (double)loss[k] : 0.0;
      clipped += has && policy_clipped(p.term, policy_ratio(lp[k], old[k]), A[k]);
    }
  }
  sum = block_total(sum);
  n = block_total(n);
  clipped = block_total(clipped);
  if (C > 1) asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
  if (threadIdx.x == 0) {
    store_remote(&sums[rank], 0, sum);
    store_remote(&counts[0][rank], 0, n);
    store_remote(&counts[1][rank], 0, clipped);
  }
  if (C > 1) asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;" ::: "memory");
  if (rank == 0 && threadIdx.x == 0) {
    for (int i = 1; i < C; i++) { sum += sums[i]; n += counts[0][i]; clipped += counts[1][i]; }
    *loss_out = (float)(mean && n > 0 ? sum / n : sum);
    *n_valid_out = n;
    if (n_clipped_out) *n_clipped_out = clipped;
  }
}

// ---- paired preference loss ---------------------------------------------------------------------------------------------------------------
typedef PreferenceArgs Preference;

// The rows of one answer, and whether they count: none of an answer does whose offsets leave the rows or descend.  Its rows still get a gradient
// of 0: a row from offsets[0] on that no good answer holds lies between the offsets of a bad one.
__device__ __forceinline__ int3 answer_rows(const Preference& p, int answer, bool flag) {
  const int a = p.offsets[answer], b = p.offsets[answer + 1];
  if (a >= 0 && a <= b && b <= p.N) return make_int3(a, b, 1);
  if (flag) atomicOr(&g_objectives_status, ST_BAD_RANGE);
  const int first = min(max(a, 0), p.N);
  return make_int3(first, max(first, min(b, p.N)), 0);
}

// One block per pair, or a cluster of blocks for long answers; half of a block on each answer.  Sums of log ratios of two long answers nearly
// cancel: they are held in 64 bits.  Bound by latency (two dependent loads, a reduction, one thread's logarithm) until there are some
// thousands of pairs, by HBM behind that.
__global__ void __launch_bounds__(1024) k_preference_pairs(const Preference p) {
  pdl_trigger();
  __shared__ double sums[32], all_sums[2][MOST_CLUSTER];
  __shared__ int counts[32], all_counts[2][MOST_CLUSTER];
  __shared__ float slope_s[2];
  const int C = (int)cluster_size(), rank = (int)cluster_rank();
  if (C > 1) asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory");      // this block runs: its shared memory may be written
  const int pair = blockIdx.x / C, half = blockDim.x >> 1, side = threadIdx.x >= half, tid = threadIdx.x - side * half, warps = half >> 5;
  const int3 rows = answer_rows(p, 2 * pair + side, rank == 0 && tid == 0);
  const unsigned first = rows.x + rank * half + tid, end = rows.y, step = C * half;
  double sum = 0.0;
  int n = 0;
  uint32_t seen = 0;      // which of the thread's first 32 rows count
  int q = 0;
  for (unsigned i0 = first, counted_end = rows.z ? end : 0; i0 < counted_end; i0 += 4 * step, q += 4) {      // four rows a thread in flight
    int t[4];
    float lp[4], ref[4];
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const unsigned i = min(i0 + k * step, end - 1);
      t[k] = p.tgt0 ? p.tgt0[i] : 0;
      lp[k] = p.logp[i];
      ref[k] = p.ref ? p.ref[i] : 0.f;
    }
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const bool counted = t[k] >= 0 && i0 + k * step < end;
      n += counted;
      if (q < 32) seen |= (uint32_t)counted << (q + k);
      sum += counted ? (double)(lp[k] - ref[k]) : 0.0;      // rows that do not count may hold anything
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) { sum += __shfl_xor_sync(0xffffffffu, sum, o); n += __shfl_xor_sync(0xffffffffu, n, o); }
  if ((threadIdx.x & 31) == 0) { sums[threadIdx.x >> 5] = sum; counts[threadIdx.x >> 5] = n; }
  __syncthreads();
  if (C > 1) asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
  if (threadIdx.x < 2) {      // each answer's sum over the block, to every block
    const int k = threadIdx.x;
    double total = 0.0;
    int count = 0;
    for (int i = 0; i < warps; i++) { total += sums[k * warps + i]; count += counts[k * warps + i]; }
    for (int to = 0; to < C; to++) {
      store_remote(&all_sums[k][rank], to, total);
      store_remote(&all_counts[k][rank], to, count);
    }
  }
  if (C > 1) asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;" ::: "memory"); else __syncthreads();
  if (threadIdx.x == 0) {
    double rho[2], per[2];
    for (int k = 0; k < 2; k++) {
      int count = 0;
      rho[k] = 0.0;
      for (int i = 0; i < C; i++) { rho[k] += all_sums[k][i]; count += all_counts[k][i]; }
      per[k] = p.normalised ? 1.0 / max(count, 1) : 1.0;
      rho[k] *= per[k];
      if (rank == 0) p.ratios[2 * pair + k] = (float)rho[k];
    }
    const double delta = rho[0] - rho[1], beta = p.beta;
    double loss, slope;      // slope: by delta
    if (p.kind == FEMTO_PREFERENCE_SIGMOID) {
      // -(1 - e) log sigma(h) - e log sigma(-h), with log(1 + e^-|h|) once
      const double h = beta * delta - (double)p.margin, e = p.smoothing, q = exp(-fabs(h)), s = log1p(q);
      loss = s + (e < 1.0 ? (1.0 - e) * fmax(-h, 0.0) : 0.0) + (e > 0.0 ? e * fmax(h, 0.0) : 0.0);      // h may be infinite
      slope = beta * ((h >= 0.0 ? 1.0 / (1.0 + q) : q / (1.0 + q)) - (1.0 - e));
    } else {
      const double u = delta - 0.5 / beta;
      loss = u * u;
      slope = 2.0 * u;
    }
    if (rank == 0) p.pair_losses[pair] = (float)loss;
    slope *= (double)p.scale / (p.mean ? p.P : 1);
    slope_s[0] = (float)(slope * per[0]);
    slope_s[1] = (float)(-slope * per[1]);
  }
  if (!p.dlogp) return;
  __syncthreads();
  const float d = rows.z ? slope_s[side] : 0.f;
  q = 0;
#pragma unroll 4
  for (unsigned i = first; i < end; i += step, q++) p.dlogp[i] = (q < 32 ? seen >> q & 1u : !p.tgt0 || p.tgt0[i] >= 0) ? d : 0.f;
}

// Sum or mean over the pairs, and zeros as the gradient of rows that belong to no answer.
__global__ void __launch_bounds__(1024) k_preference_sum(const Preference p, float* loss_out) {
  pdl_trigger();
  pdl_wait();
  if (blockIdx.x == 0) {
    double sum = 0.0;
#pragma unroll 4
    for (int i = threadIdx.x; i < p.P; i += 1024) sum += (double)__ldcg(p.pair_losses + i);
    sum = block_total(sum);
    if (threadIdx.x == 0) *loss_out = (float)(p.mean && p.P > 0 ? sum / p.P : sum);
  }
  if (!p.dlogp) return;
  const int first = p.P > 0 ? min(max(p.offsets[0], 0), p.N) : p.N, last = p.P > 0 ? min(max(p.offsets[2 * p.P], 0), p.N) : p.N;
  const long long step = (long long)gridDim.x * 1024;
  for (long long i = blockIdx.x * 1024ll + threadIdx.x; i < first; i += step) p.dlogp[i] = 0.f;
  for (long long i = last + blockIdx.x * 1024ll + threadIdx.x; i < p.N; i += step) p.dlogp[i] = 0.f;
}
}  // namespace

// Status word of these entry points on the current device; reading clears it.
unsigned int objectives_status_word() {
  unsigned int w = 0, zero = 0;
  if (cudaMemcpyFromSymbol(&w, g_objectives_status, sizeof(w)) != cudaSuccess) return 0;
  if (w) cudaMemcpyToSymbol(g_objectives_status, &zero, sizeof(zero));
  return w | objective_rows_status_word();
}

int policy_sum(const RowsArgs& p, bool mean, float* loss_out, int* n_valid_out, int* n_clipped_out, cudaStream_t s) {
  const int C = p.N > 2048 ? MOST_CLUSTER : 1;
  CUDA_TRY(launch_dependent_clusters(k_policy_sum, C, dim3(C), dim3(1024), 0, s, p, (int)mean, loss_out, n_valid_out, n_clipped_out));
  KERNEL_CHECK();
  return 0;
}

PreferenceArgs preference_args(const femto_preference_config& c, int N, int P) {
  PreferenceArgs p = {};
  p.N = N; p.P = P;
  p.kind = c.kind; p.normalised = c.length_normalised != 0; p.mean = c.reduction == FEMTO_REDUCTION_MEAN;
  p.beta = c.beta; p.margin = c.margin; p.smoothing = c.label_smoothing;
  p.scale = 1.f;
  return p;
}
int preference(const PreferenceArgs& p, float* loss_out, cudaStream_t s) {
  if (p.P > 0) {
    // A thread has some eight rows of an answer of average length; where pairs are few and long, a cluster shares one (one pair of 70000 rows
    // each: 87 -> 10 us), and where they are many, small blocks let one's reduction pass behind others' loads (1024 pairs of 1536 rows each, 24 rows a
    // thread: 13.4 us with 128 threads, half on each answer, 15.9 with 256, 21.2 with 512).
    int threads = 64, C = 1;
    while (threads < (p.P < 4 * device_sm_count() ? 1024 : 128) && (long long)threads * p.P * 8 < p.N) threads *= 2;
    while (C < MOST_CLUSTER && (long long)C * p.P < device_sm_count() && (long long)C * 1024 * p.P * 8 < p.N) C *= 2;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = C; at.val.clusterDim.y = 1; at.val.clusterDim.z = 1;
    cfg.gridDim = dim3((unsigned)(p.P * C)); cfg.blockDim = dim3(threads); cfg.stream = s; cfg.attrs = &at; cfg.numAttrs = C > 1;
    CUDA_TRY(cudaLaunchKernelEx(&cfg, k_preference_pairs, p));
    KERNEL_CHECK();
  }
  CUDA_TRY(launch_dependent(k_preference_sum, dim3(p.dlogp ? std::min(cdiv(p.N, 4096) + 1, 148) : 1), dim3(1024), 0, s, p, loss_out));
  KERNEL_CHECK();
  return 0;
}

// ---- behind the lm_head tail -------------------------------------------------------------------------------------------------------------------
namespace {
__global__ void __launch_bounds__(256) k_objective_rows(const RowsArgs p, const float* __restrict__ nll, float* __restrict__ logp, float* __restrict__ slopes,
                                                        int row0, int n, const float* __restrict__ scale_dev, bool policy) {
  pdl_trigger();
  const int i = blockIdx.x * 256 + threadIdx.x, row = row0 + i;
  if (i >= n) return;
  const float lp = 0.f - nll[row];
  logp[row] = lp;
  if (!policy) { slopes[row] = 0.f; return; }
  if (p.tgt0[row] < 0) { p.token_losses[row] = slopes[row] = 0.f; return; }
  float loss, slope;
  policy_token(p.term, lp, p.old[row], p.adv[row], p.term.kl != 0.f ? p.ref[row] : 0.f, p.w ? p.w[row] : 1.f, &loss, &slope);
  p.token_losses[row] = loss;
  slopes[row] = -slope * (scale_dev ? scale_dev[0] : 1.f) * p.inv_t;
}
__global__ void __launch_bounds__(256) k_negate(float* x, long long n) {
  pdl_trigger();
  const long long i = blockIdx.x * 256ll + threadIdx.x;
  if (i < n) x[i] = 0.f - x[i];
}
}  // namespace
int objective_negate(float* x, long long n, cudaStream_t s) {
  k_negate<<<cdiv(n, 256), 256, 0, s>>>(x, n);
  KERNEL_CHECK();
  return 0;
}
int objective_slopes(const TokenObjective& o, const float* nll, int row0, int n, const float* scale_dev, float* loss_out, cudaStream_t s) {
  k_objective_rows<<<cdiv(n, 256), 256, 0, s>>>(o.policy, nll, o.logp, o.slopes, row0, n, scale_dev, !o.pairs);
  KERNEL_CHECK();
  return o.pairs ? preference(o.preference, loss_out, s) : 0;
}

int check_temperature(float t) {
  return t >= 1e-6f && t <= 1e6f ? 0 : femto_fail(FEMTO_ERR_ARG, "temperature must lie in 1e-6 .. 1e6");
}
PolicyTerm policy_term(const femto_policy_config& c) { return {1.f - c.clip_low, 1.f + c.clip_high, c.kl_coef}; }

// ---- checks of arguments ------------------------------------------------------------------------------------------------------------------
namespace {
int check_dtype(int dtype) {
  return dtype == FEMTO_F32 || dtype == FEMTO_BF16 ? 0 : femto_fail(FEMTO_ERR_ARG, "dtype must be FEMTO_F32 or FEMTO_BF16");
}
int check_rows(int dtype, const void* logits, long long ldl, const int* tgt0, int N, int V) {
  FEMTO_TRY(check_dtype(dtype));
  if (N < 0 || V <= 0) return femto_fail(FEMTO_ERR_SHAPE, "N = %d rows of V = %d logits", N, V);
  if (ldl < V) return femto_fail(FEMTO_ERR_SHAPE, "ldl = %lld is less than V = %d", ldl, V);
  if (N > 0 && (!logits || !tgt0)) return femto_fail(FEMTO_ERR_ARG, "NULL argument");
  const uintptr_t size = dtype == FEMTO_BF16 ? 2 : 4;
  if (reinterpret_cast<uintptr_t>(logits) % size) return femto_fail(FEMTO_ERR_ALIGN, "logits are not aligned to their type");
  return 0;
}
// The gradient lies apart from the logits, or in their place.  With one pitch the rows of both may also lie in turn, in one wide buffer: the distance of
// their first rows, modulo the pitch, leaves room for a row on either side.
int check_gradient(int dtype, const void* dlogits, long long ldd, const void* logits, long long ldl, int N, int V) {
  if (ldd < V) return femto_fail(FEMTO_ERR_SHAPE, "ldd = %lld is less than V = %d", ldd, V);
  const uintptr_t size = dtype == FEMTO_BF16 ? 2 : 4, a = reinterpret_cast<uintptr_t>(dlogits), b = reinterpret_cast<uintptr_t>(logits);
  if (a % size) return femto_fail(FEMTO_ERR_ALIGN, "dlogits are not aligned to their type");
  if (N == 0 || (a == b && ldd == ldl)) return 0;
  const uintptr_t row = size * V, pitch = size * ldl, a_end = a + size * ((uintptr_t)(N - 1) * ldd + V), b_end = b + size * ((uintptr_t)(N - 1) * ldl + V);
  if (a >= b_end || b >= a_end) return 0;
  if (ldd == ldl) {
    const uintptr_t apart = (a > b ? a - b : b - a) % pitch;
    if (apart >= row && pitch - apart >= row) return 0;
  }
  return femto_fail(FEMTO_ERR_ARG, "dlogits overlap the logits: give the same rows and pitch, or memory of their own");
}
float log2e_over(float temperature) { return (float)(1.4426950408889634074 / (double)temperature); }

RowsArgs rows_args(const void* logits, long long ldl, const int* tgt0, int N, int V, float temperature) {
  RowsArgs p = {};
  p.logits = logits; p.ldl = ldl; p.tgt0 = tgt0; p.N = N; p.V = V;
  p.c = log2e_over(temperature); p.inv_t = 1.f / temperature; p.inv_t64 = 1.0 / (double)temperature;
  return p;
}
}  // namespace

extern "C" int32_t femto_token_logprobs(int32_t dtype, const void* logits, int64_t ldl, const int32_t* targets0, int32_t N, int32_t V, float temperature,
                                        float* logp, float* entropy_out, void* stream) {
  FEMTO_TRY(check_rows(dtype, logits, ldl, targets0, N, V));
  FEMTO_TRY(check_temperature(temperature));
  if (N == 0) return 0;
  if (!logp) return femto_fail(FEMTO_ERR_ARG, "NULL argument");
  RowsArgs p = rows_args(logits, ldl, targets0, N, V, temperature);
  p.logp = logp; p.ent = entropy_out;
  return objective_rows(dtype, LOGPROBS, p, (cudaStream_t)stream);
}

extern "C" int32_t femto_token_logprobs_gradient(int32_t dtype, void* dlogits, int64_t ldd, const void* logits, int64_t ldl, const int32_t* targets0, int32_t N,
                                                 int32_t V, float temperature, const float* dlogp, const float* dentropy, void* stream) {
  FEMTO_TRY(check_rows(dtype, logits, ldl, targets0, N, V));
  FEMTO_TRY(check_temperature(temperature));
  FEMTO_TRY(check_gradient(dtype, dlogits, ldd, logits, ldl, N, V));
  if (N == 0) return 0;
  if (!dlogits || !dlogp) return femto_fail(FEMTO_ERR_ARG, "NULL argument");
  RowsArgs p = rows_args(logits, ldl, targets0, N, V, temperature);
  p.dlogits = dlogits; p.ldd = ldd; p.dlogp = dlogp; p.dent = dentropy;
  return objective_rows(dtype, GRADIENT, p, (cudaStream_t)stream);
}

int check_policy(const femto_policy_config* c, const float* ref_logp) {
  if (!c) return femto_fail(FEMTO_ERR_ARG, "NULL configuration");
  FEMTO_TRY(check_temperature(c->temperature));
  if (!(c->clip_low >= 0.f && c->clip_low <= 1.f) || !(c->clip_high >= 0.f))
    return femto_fail(FEMTO_ERR_ARG, "clip_low must lie in 0..1 and clip_high be 0 or more");
  if (!(c->kl_coef >= 0.f) || !isfinite(c->kl_coef)) return femto_fail(FEMTO_ERR_ARG, "kl_coef must be 0 or more, and finite");
  if (c->kl_coef > 0.f && !ref_logp) return femto_fail(FEMTO_ERR_ARG, "kl_coef needs ref_logp");
  if (c->reduction != FEMTO_REDUCTION_SUM && c->reduction != FEMTO_REDUCTION_MEAN)
    return femto_fail(FEMTO_ERR_ARG, "reduction must be FEMTO_REDUCTION_SUM or FEMTO_REDUCTION_MEAN");
  return 0;
}

extern "C" int32_t femto_policy_loss(int32_t dtype, const void* logits, int64_t ldl, const int32_t* targets0, int32_t N, int32_t V, const float* old_logp,
                                     const float* advantages, const float* ref_logp, const float* weights, const femto_policy_config* h_cfg, void* dlogits,
                                     int64_t ldd, float* token_losses, float* logp, float* loss_out, int32_t* n_valid_out, int32_t* n_clipped_out,
                                     void* stream) {
  FEMTO_TRY(check_rows(dtype, logits, ldl, targets0, N, V));
  FEMTO_TRY(check_policy(h_cfg, N > 0 ? ref_logp : h_cfg ? &h_cfg->kl_coef : nullptr));
  if (dlogits) FEMTO_TRY(check_gradient(dtype, dlogits, ldd, logits, ldl, N, V));
  if (!loss_out || !n_valid_out || (N > 0 && (!old_logp || !advantages || !token_losses || !logp))) return femto_fail(FEMTO_ERR_ARG, "NULL argument");
  cudaStream_t s = (cudaStream_t)stream;
  const bool mean = h_cfg->reduction == FEMTO_REDUCTION_MEAN;
  RowsArgs p = rows_args(logits, ldl, targets0, N, V, h_cfg->temperature);
  p.dlogits = dlogits; p.ldd = ldd; p.logp = logp; p.token_losses = token_losses;
  p.old = old_logp; p.ref = ref_logp; p.adv = advantages; p.w = weights;
  p.term = policy_term(*h_cfg);
  if (N > 0) {
    if (mean && dlogits) {
      k_count_targets<<<1, 1024, 0, s>>>(targets0, N, V, n_valid_out);
      KERNEL_CHECK();
      p.n_valid = n_valid_out;
    }
    FEMTO_TRY(objective_rows(dtype, POLICY, p, s));
  }
  return policy_sum(p, mean, loss_out, n_valid_out, n_clipped_out, s);
}

int check_preference(const femto_preference_config* c) {
  if (!c) return femto_fail(FEMTO_ERR_ARG, "NULL configuration");
  if (c->kind != FEMTO_PREFERENCE_SIGMOID && c->kind != FEMTO_PREFERENCE_SQUARED)
    return femto_fail(FEMTO_ERR_ARG, "kind must be FEMTO_PREFERENCE_SIGMOID or FEMTO_PREFERENCE_SQUARED");
  if (!(c->beta > 0.f) || !isfinite(c->beta)) return femto_fail(FEMTO_ERR_ARG, "beta must be positive and finite");
  if (!isfinite(c->margin) || !(c->label_smoothing >= 0.f && c->label_smoothing <= 1.f))
    return femto_fail(FEMTO_ERR_ARG, "the margin must be finite and label_smoothing lie in 0..1");
  if (c->kind == FEMTO_PREFERENCE_SQUARED && (c->margin != 0.f || c->label_smoothing != 0.f))
    return femto_fail(FEMTO_ERR_ARG, "the squared loss has no margin and no label smoothing");
  if (c->reduction != FEMTO_REDUCTION_SUM && c->reduction != FEMTO_REDUCTION_MEAN)
    return femto_fail(FEMTO_ERR_ARG, "reduction must be FEMTO_REDUCTION_SUM or FEMTO_REDUCTION_MEAN");
  return 0;
}

extern "C" int32_t femto_preference_loss(const float* logp, const float* ref_logp, const int32_t* targets0, int32_t N, const int32_t* offsets, int32_t P,
                                         const femto_preference_config* h_cfg, float* loss_out, float* pair_losses, float* ratios, float* dlogp,
                                         void* stream) {
  FEMTO_TRY(check_preference(h_cfg));
  if (N < 0 || P < 0 || P > (1 << 29)) return femto_fail(FEMTO_ERR_SHAPE, "P = %d pairs of answers in N = %d rows", P, N);
  if (!loss_out || (N > 0 && !logp) || (P > 0 && (!offsets || !pair_losses || !ratios))) return femto_fail(FEMTO_ERR_ARG, "NULL argument");
  cudaStream_t s = (cudaStream_t)stream;
  PreferenceArgs p = preference_args(*h_cfg, N, P);
  p.logp = logp; p.ref = ref_logp; p.tgt0 = targets0; p.offsets = offsets;
  p.pair_losses = pair_losses; p.ratios = ratios; p.dlogp = dlogp;
  return preference(p, loss_out, s);
}
