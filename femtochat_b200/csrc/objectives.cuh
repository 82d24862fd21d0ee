// Arithmetic that the objectives on a model's own answers share: the softmax statistics of a row of logits, the clipped policy term of a
// token, the paired preference term (objectives.cu), also used behind the lm_head tail of a training step (xent.cu).
#pragma once
#include "common.cuh"

// Softmax statistics of a row.  With c = log2(e) / temperature, m = max(z) and u_j = c (z_j - m) <= 0:
//   l = sum 2^u_j,  a = sum 2^u_j u_j,  log p_j = ln2 u_j - ln l,  H = ln l - ln2 a / l.
// The difference comes before the product.  (As one fused product, c z_j - c m, the rounding of c m would stand in every exponent: logits of the
// type's lowest value, or of some millions, came out as 0 / 0.  It is no faster.)
struct RowStats {
  float m = -INFINITY, l = 0.f, a = 0.f;
};

struct PolicyTerm {
  float lo, hi, kl;
};

#ifdef __CUDACC__
constexpr double LN2 = 0.69314718055994530942;
constexpr float LOG2E = 1.4426950408889634f;
constexpr float LEAST_U = -200.f;      // 2^u is 0 there, and u stays finite beside it

__device__ __forceinline__ float exp2_fast(float x) {   // relative error 2^-22, 0 for -inf
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// What a maximum of -inf (nothing seen, or a row without any logit above -inf) is taken as: -inf - 0 gives 2^-inf = 0, where -inf + inf is NaN.
__device__ __forceinline__ float finite_or_zero(float m) { return m == -INFINITY ? 0.f : m; }

// Moves statistics to a maximum that is no lower: with d = c (m_old - m_new) every 2^u scales by 2^d and every u moves by d.
template <bool ENTROPY> __device__ __forceinline__ void rebase(RowStats& s, float m, float c) {
  if (s.l != 0.f) {
    const float d = fmaxf((s.m - m) * c, LEAST_U), f = exp2_fast(d);
    if (ENTROPY) s.a = f * fmaf(s.l, d, s.a);
    s.l *= f;
  }
  s.m = m;
}
template <bool ENTROPY> __device__ __forceinline__ RowStats merged(RowStats x, RowStats y, float c) {
  const float m = fmaxf(x.m, y.m);
  rebase<ENTROPY>(x, m, c);
  rebase<ENTROPY>(y, m, c);
  x.l += y.l;
  if (ENTROPY) x.a += y.a;
  return x;
}
// l = 2^k f with f in [0.7, 1.4]: log l is k ln2 + log f, a small number.  A log-probability is put together in 64 bits, a few instructions of one
// warp a row: log(l) in one piece is 5e-7 off at l = 65536, and so would every ratio of two log-probabilities be.
__device__ __forceinline__ double log_sum(float l) {
  if (!(l < INFINITY)) return (double)logf(l);
  const int bits = __float_as_int(l), k = (bits - 0x3f3504f3) >> 23;      // sqrt(1/2)
  return LN2 * k + (double)logf(__int_as_float(bits - (k << 23)));
}
// The statistics of a row's other tokens, with its own token's logit z added.  The others' part of l is kept beside the sum: of a token that the
// model is all but sure of, 1 - p = others / l and -log p = log(1 + others) are small numbers, of which the rounding of l = 1 + others leaves little
// (1 - p = 1e-6: 6 %).
struct TokenStats {
  RowStats all;
  float others, z;
};
template <bool ENTROPY> __device__ __forceinline__ TokenStats with_token(const RowStats& others, float z, float c) {
  TokenStats s;
  const float d = fminf(fabsf(z - others.m) * c, -LEAST_U), f = exp2_fast(-d);
  float own = z == -INFINITY ? 0.f : 1.f + (z - z), own_a = 0.f;      // NaN and +inf give NaN
  s.z = z; s.others = others.l; s.all.a = others.a;
  if (z >= others.m) {
    s.others = others.l * f;
    if (ENTROPY) s.all.a = f * fmaf(-others.l, d, others.a);
  } else {
    own *= f;
    own_a = -own * d;
  }
  s.all.m = fmaxf(others.m, z);
  s.all.l = s.others + own;
  if (ENTROPY) s.all.a += own_a;
  return s;
}
// log l, where the token is the row's maximum and its others are few from what they are
__device__ __forceinline__ double log_total(const TokenStats& s) {
  return s.z == s.all.m && s.others < 0.5f ? (double)log1pf(s.others) : log_sum(s.all.l);
}
// log p of the token; a row without any logit above -inf (l = 0) has no distribution: -inf.
__device__ __forceinline__ double log_prob(const TokenStats& s, double inv_t) {
  return s.all.l == 0.f ? -(double)INFINITY : ((double)s.z - (double)s.all.m) * inv_t - log_total(s);
}
__device__ __forceinline__ float entropy(const TokenStats& s) {
  return s.all.l == 0.f ? 0.f : (float)(log_total(s) - LN2 * (double)s.all.a / (double)s.all.l);
}

// ---- clusters ----------------------------------------------------------------------------------------------------------------------------------
constexpr int MOST_CLUSTER = 8;
__device__ __forceinline__ uint32_t cluster_size() { uint32_t n; asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(n)); return n; }
__device__ __forceinline__ uint32_t cluster_rank() { uint32_t r; asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ uint32_t remote_address(const void* local, uint32_t rank) {
  uint32_t there;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"((uint32_t)__cvta_generic_to_shared(local)), "r"(rank));
  return there;
}
// `v` to where `local` lies in another block's shared memory
__device__ __forceinline__ void store_remote(const float* local, uint32_t rank, float v) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(remote_address(local, rank)), "f"(v) : "memory");
}
__device__ __forceinline__ void store_remote(const double* local, uint32_t rank, double v) {
  asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(remote_address(local, rank)), "d"(v) : "memory");
}
__device__ __forceinline__ void store_remote(const int* local, uint32_t rank, int v) {
  asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(remote_address(local, rank)), "r"(v) : "memory");
}

// ---- clipped policy term of one token ---------------------------------------------------------------------------------------------------
// loss = w (-min(r A, clamp(r, lo, hi) A) + beta (e^g - g - 1)),  r = e^(lp - old),  g = ref - lp, and its derivative by lp.  The minimum is
// the bounded product, which does not depend on lp, where A > 0 and r > hi or A < 0 and r < lo.  A weight of 0 counts nothing, whatever
// the other numbers are.
__device__ __forceinline__ bool policy_clipped(const PolicyTerm& t, float r, float A) { return (A > 0.f && r > t.hi) || (A < 0.f && r < t.lo); }
__device__ __forceinline__ float policy_ratio(double lp, float old) { return expf((float)(lp - (double)old)); }
__device__ __forceinline__ void policy_token(const PolicyTerm& t, double lp, float old, float A, float ref, float w, float* loss, float* slope) {
  if (w == 0.f) { *loss = *slope = 0.f; return; }
  const float r = policy_ratio(lp, old);
  const float gain = A == 0.f ? 0.f : r * A;      // r may be inf
  const bool clipped = policy_clipped(t, policy_ratio((float)lp, old), A);      // of the number that goes out: the count of clipped tokens is taken from it
  float l = clipped ? -(A > 0.f ? t.hi : t.lo) * A : -gain, d = clipped ? 0.f : -gain;
  if (t.kl != 0.f) {
    const float g = (float)((double)ref - lp), e = expm1f(g);
    l += t.kl * (e == INFINITY ? e : e - g);      // of a token that the model rules out infinite, and not inf - inf
    d -= t.kl * e;
  }
  *loss = w * l;
  *slope = w * d;
}
#endif

// ---- passes over rows of logits (objective_rows.cu) ------------------------------------------------------------------------------------------
enum RowsMode { LOGPROBS, GRADIENT, POLICY };

struct RowsArgs {
  const void* logits;
  void* dlogits;                 // GRADIENT, POLICY (NULL there: the numbers only)
  long long ldl, ldd;
  const int* tgt0;
  int V, N;
  float c, inv_t;                // log2(e) / temperature, 1 / temperature
  double inv_t64;
  float *logp, *ent;             // LOGPROBS (ent may be NULL), POLICY: logp
  const float *dlogp, *dent;     // GRADIENT (dent may be NULL)
  const float *old, *ref, *adv, *w;      // POLICY
  float* token_losses;
  const int* n_valid;            // POLICY, mean: the slopes are divided by it
  PolicyTerm term;
  uint32_t wait_limit = 1u << 22;      // polls of a wait, as sm100::WAIT_LIMIT
};
int objective_rows(int dtype, RowsMode mode, const RowsArgs& p, cudaStream_t s);
unsigned int objective_rows_status_word();
int check_policy(const femto_policy_config* c, const float* ref_logp);
int check_preference(const femto_preference_config* c);
int check_temperature(float t);
PolicyTerm policy_term(const femto_policy_config& c);
int objective_negate(float* x, long long n, cudaStream_t s);      // x = -x
// The reduced loss, the rows with a target and those that the clipping held, from token_losses and logp.
int policy_sum(const RowsArgs& p, bool mean, float* loss_out, int* n_valid_out, int* n_clipped_out, cudaStream_t s);

// ---- paired preference loss on log-probabilities -------------------------------------------------------------------------------------------------
struct PreferenceArgs {
  const float *logp, *ref;
  const int *tgt0, *offsets;
  int N, P, kind, normalised, mean;
  float beta, margin, smoothing;
  float scale;                   // of the slopes, beside the mean's 1 / P
  float *pair_losses, *ratios, *dlogp;
};
PreferenceArgs preference_args(const femto_preference_config& c, int N, int P);
int preference(const PreferenceArgs& p, float* loss_out, cudaStream_t s);

// ---- behind the lm_head tail of a training step ---------------------------------------------------------------------------------------------------
// The tail gives the cross-entropy of each row, -log p; the objective gives back the factors of its gradient, d loss / d (-log p) / temperature.
struct TokenObjective {
  bool pairs = false;            // preference (needs all rows at once), or policy (row by row)
  RowsArgs policy = {};          // tgt0, N, V, old, ref, adv, w, token_losses, logp, term, inv_t
  PreferenceArgs preference = {};      // logp and dlogp: the workspace below
  float* logp = nullptr;         // [N]
  float* slopes = nullptr;       // [N]
};
int objective_slopes(const TokenObjective& o, const float* nll, int row0, int n, const float* scale_dev, float* loss_out, cudaStream_t s);
