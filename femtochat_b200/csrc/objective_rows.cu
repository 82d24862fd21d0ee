// Passes over rows of logits for the objectives on a model's own answers: softmax statistics, what they give for the row's token (its
// log-probability, the entropy, the policy term), and the gradient by the logits, from one reading of the row.
//
// Three kernels that differ in where a row lies between its reading and the writing of its gradient: in the registers of a cluster (k_rows_few),
// in a buffer of the group of warps that works on it (k_rows_near), in a ring that a block's groups share (k_rows_ring); launch() says
// which takes what.  A thread's exponentials are relative to a maximum of its own, the (m, l, a) of threads and warps are added in a fixed order.
// They are those of the tokens other than the row's own, which is added at the end (with_token).
//
// The floor is HBM: every logit is read once and its gradient written once.  Beside it stand an exponential an element for the numbers, another one for the
// gradient (16 a cycle and multiprocessor: both together half of the time that bf16 takes to come and go), and with the gradient some 17 instructions;
// one block's chain of load, statistics, exchange, slopes and stores is ten times as long as a row's share of the bandwidth, so rows have to
// overlap.  Measured (time, share of the measured copy rate; bytes of the floor):
//   log-probabilities    gradient          policy loss and gradient
//     70 us  0.88         171 us  0.84      175 us  0.82    4096 x 65536 bf16, a quarter of the rows without target   ring, a row to two blocks (*)
//     89     0.93         170     0.96      178     0.92    2048 x 65536 fp32                                         ring, the same
//     51     0.79         103     0.77      112     0.71    1000 x 131000 bf16                                        ring, the same
//     31     0.60          48     0.76       55     0.67    2000 x 30000 bf16                                         ring
//     30     0.68          44     0.93       49     0.83    8192 x 4096 fp32                                          near
//     22     0.47          32     0.64       40     0.52    8192 x 4096 bf16                                          near
//     29     0.51          45     0.66       54     0.54    20000 x 2400 bf16                                         near
//      3.8   0.17           5.2   0.25        7.6   0.17    16 x 65536 fp32                                           few
// (* log-probabilities: to one.)
// The exponential pipe is busy 64 % (gradient) to 68 % with 65536 logits in bf16.  Arithmetic in f32x2 pairs or in single floats takes the same time.
#include <limits.h>

#include <algorithm>
#include <type_traits>

#include "objectives.cuh"
#include "sm100_ptx.cuh"

namespace {
using namespace sm100;

// Bit 1: a target outside the vocabulary (its row counts as one without a target); bit 2: a bounded wait ran out.  Part of the library
// image, so that no call allocates; femto_status_word(NULL, ..) reads and clears it.
__device__ unsigned int g_rows_status = 0;

// The row's target, or -1 where it has none.
__device__ __forceinline__ int checked_target(const RowsArgs& p, int t, bool flag) {
  if (t >= p.V) { if (flag) atomicOr(&g_rows_status, ST_BAD_TOKEN); return -1; }
  return t < 0 ? -1 : t;
}

// The targets of the rows that a block (or group) walks, every `step`-th from its first: a warp holds 32 of them, so that one load serves 32
// rows.  (One row ahead at a time, a run of 14 rows without target cost a block 7 us.)  Called by whole warps.
struct Targets {
  const int* tgt0;
  long long first, step;
  int N, held;
  __device__ __forceinline__ Targets(const RowsArgs& p, long long first, long long step) : tgt0(p.tgt0), first(first), step(step), N(p.N) { load(0); }
  __device__ __forceinline__ void load(int k) {
    const long long row = first + (long long)(k + (threadIdx.x & 31)) * step;
    held = row < N ? tgt0[row] : -1;
  }
  // of the k-th row; asked for in order
  __device__ __forceinline__ int operator()(int k) {
    if (k > 0 && (k & 31) == 0) load(k);
    return __shfl_sync(0xffffffffu, held, k & 31);
  }
};

__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) { uint64_t v; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b)); return v; }

// A word that is there, or `none`.  One instruction each, volatile: with a branch around a plain load the compiler put every word's arithmetic
// between its load and the next one's, and a thread waited for its words one after the other (8192 x 4096 in fp32: 44 -> 58 us).
__device__ __forceinline__ uint4 load_word(const uint4* p, bool there, uint32_t none) {
  uint4 q = make_uint4(none, none, none, none);
  asm volatile("{\n.reg .pred there;\nsetp.ne.u32 there, %5, 0;\n@there ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];\n}"
               : "+r"(q.x), "+r"(q.y), "+r"(q.z), "+r"(q.w) : "l"(p), "r"((uint32_t)there) : "memory");
  return q;
}

// A 16-byte word of logits: its pairs in fp32, its largest element, and back.
template <typename T> struct Word {
  static constexpr int n = VecN<T>::n;
  static constexpr uint32_t LEAST = sizeof(T) == 4 ? 0xff800000u : 0xff80ff80u;      // -inf
  static __device__ __forceinline__ uint64_t get(const uint4& q, int i) {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
    if constexpr (sizeof(T) == 4) return pack2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
    else return pack2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
  }
  static __device__ __forceinline__ void put(uint4& q, int i, uint64_t v) {
    float lo, hi;
    unpack2(v, lo, hi);
    uint32_t* w = reinterpret_cast<uint32_t*>(&q);
    if constexpr (sizeof(T) == 4) { w[2 * i] = __float_as_uint(lo); w[2 * i + 1] = __float_as_uint(hi); }
    else {
      const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
  }
  static __device__ __forceinline__ float most(const uint4& q) {
    if constexpr (sizeof(T) == 4)
      return fmaxf(fmaxf(__uint_as_float(q.x), __uint_as_float(q.y)), fmaxf(__uint_as_float(q.z), __uint_as_float(q.w)));
    else {
      const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&q);
      const __nv_bfloat162 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
      return fmaxf(__low2float(m), __high2float(m));
    }
  }
};

// Where a row's 16-byte words lie.  The elements before the first and behind the last whole word belong to threads of the row's own.
struct RowShape {
  int head, nvec, tail;
};
template <typename T> __device__ __forceinline__ RowShape row_shape(const T* p, int V) {
  RowShape r;
  const uintptr_t a = reinterpret_cast<uintptr_t>(p);
  r.head = min(V, (int)(((16u - (a & 15u)) & 15u) / sizeof(T)));
  r.nvec = (V - r.head) / VecN<T>::n;
  r.tail = V - r.head - r.nvec * VecN<T>::n;
  return r;
}
// The element outside the words that thread i of the row takes, or -1.
template <typename T> __device__ __forceinline__ int edge_of(const RowShape& r, int i) {
  return i < r.head ? i : i >= 16 && i < 16 + r.tail ? r.head + r.nvec * VecN<T>::n + i - 16 : -1;
}

// u = c (z - m) of a pair of logits.
struct Exponent {
  uint64_t c2, m2;
  __device__ __forceinline__ Exponent(float m, float c) : c2(pack2(c, c)), m2(pack2(-finite_or_zero(m), -finite_or_zero(m))) {}
  __device__ __forceinline__ void of(uint64_t z2, float& u0, float& u1) const { unpack2(mul2(add2(z2, m2), c2), u0, u1); }
};
// The word that holds the target, or -1 where it lies outside the words.
template <typename T> __device__ __forceinline__ int word_of_target(const RowShape& r, int t) {
  const int v = (t - r.head) / VecN<T>::n;
  return t >= r.head && v < r.nvec ? v : -1;
}
// Takes the target's element out of its word in shared memory, by the thread that reads the word, ahead of its reading.  (In registers, a selection for every
// word in flight: 8000 x 16000 in bf16, gradient, 97 us for 87.)  The next copy to this memory is another proxy's.
template <typename T> __device__ __forceinline__ void take_out(uint4* word, int e) {
  reinterpret_cast<T*>(word)[e] = from_f<T>(-INFINITY);
  fence_proxy_async();
}

// Adds pairs of logits to a thread's sums.
template <bool ENTROPY> struct Adder {
  uint64_t l2 = 0, a2 = 0;
  __device__ __forceinline__ void add(const Exponent& x, uint64_t z2) {
    float u0, u1;
    x.of(z2, u0, u1);
    const uint64_t e2 = pack2(exp2_fast(u0), exp2_fast(u1));
    l2 = add2(l2, e2);
    if (ENTROPY) a2 = fma2(e2, pack2(fmaxf(u0, LEAST_U), fmaxf(u1, LEAST_U)), a2);
  }
  // The sums so far join the statistics, whose maximum they are relative to.
  __device__ __forceinline__ void join(RowStats& s) {
    float v0, v1;
    unpack2(l2, v0, v1);
    s.l += v0 + v1;
    if (ENTROPY) { unpack2(a2, v0, v1); s.a += v0 + v1; }
    l2 = a2 = 0;
  }
};

// A thread's statistics, relative to a maximum of its own that grows a few times in a row.  They are those of the row without its target, which
// with_token() adds.
template <typename T, bool ENTROPY> struct Running {
  RowStats s;
  Exponent x;
  Adder<ENTROPY> sum;
  __device__ __forceinline__ Running(bool there, float edge, float c) : x(edge, c) {
    s.m = edge;
    if (there) sum.add(x, pack2(edge, -INFINITY));
  }
  template <int K> __device__ __forceinline__ void add(const uint4 (&q)[K], float c) {
    float m = Word<T>::most(q[0]);
#pragma unroll
    for (int h = 1; h < K; h++) m = fmaxf(m, Word<T>::most(q[h]));
    if (m > s.m) {
      sum.join(s);
      rebase<ENTROPY>(s, m, c);
      x = Exponent(m, c);
    }
#pragma unroll
    for (int h = 0; h < K; h++)
#pragma unroll
      for (int i = 0; i < VecN<T>::n / 2; i++) sum.add(x, Word<T>::get(q[h], i));
  }
  // The words that are left of a row, fewer than K for each of `threads`: `rest`, and counted from this thread on `mine`.  Where few are left, no
  // exponentials of what is not there (16000 x 3200 in bf16, gradient: 47 -> 43 us).  `loaded` is called when the words have been read.
  template <int K, class F> __device__ __forceinline__ void add_rest(const uint4* words, int threads, int mine, int rest, float c, const F& loaded) {
    if (rest > K / 2 * threads) {
      uint4 q[K];
#pragma unroll
      for (int h = 0; h < K; h++) q[h] = word_or_none(words + h * threads, h * threads < mine);
      loaded();
      add(q, c);
    } else {
      for (; rest > 0; rest -= threads, mine -= threads, words += threads) {
        uint4 q[1] = {word_or_none(words, mine > 0)};
        add(q, c);
      }
      loaded();
    }
  }
  static __device__ __forceinline__ uint4 word_or_none(const uint4* word, bool there) {
    uint4 q = make_uint4(Word<T>::LEAST, Word<T>::LEAST, Word<T>::LEAST, Word<T>::LEAST);
    if (there) q = *word;
    return q;
  }
  // The warp's statistics, in every lane.
  __device__ __forceinline__ RowStats of_warp(float c) {
    sum.join(s);
    rebase<ENTROPY>(s, warp_max(s.m), c);
    s.l = warp_sum(s.l);
    if (ENTROPY) s.a = warp_sum(s.a);
    return s;
  }
};

// The statistics of `slots` warps (m, l, a in three runs of `pitch`), by every warp that calls it: fixed order, the same bits in all.
template <bool ENTROPY> __device__ __forceinline__ RowStats merged_parts(const float* part, int pitch, int slots, float c) {
  const int lane = threadIdx.x & 31;
  RowStats r;
  for (int i = lane; i < slots; i += 32) r.m = fmaxf(r.m, part[i]);
  r.m = warp_max(r.m);
  for (int i = lane; i < slots; i += 32) {
    RowStats y;
    y.m = part[i]; y.l = part[pitch + i]; y.a = ENTROPY ? part[2 * pitch + i] : 0.f;
    rebase<ENTROPY>(y, r.m, c);
    r.l += y.l;
    if (ENTROPY) r.a += y.a;
  }
  r.l = warp_sum(r.l);
  if (ENTROPY) r.a = warp_sum(r.a);
  return r;
}

// What a row's token needs beside the statistics, asked for before the row is read.
struct RowNumbers {
  float z = 0.f, x[4] = {0.f, 0.f, 0.f, 1.f};
};
template <typename T, RowsMode MODE, bool ENTROPY> __device__ __forceinline__ RowNumbers row_numbers(const RowsArgs& p, long long row, const T* z, int t) {
  RowNumbers r;
  r.z = to_f<T>(z[t]);
  if (MODE == GRADIENT) { r.x[0] = p.dlogp[row]; if (ENTROPY) r.x[1] = p.dent[row]; }
  if (MODE == POLICY) {
    r.x[0] = p.old[row]; r.x[1] = p.adv[row];
    if (p.term.kl != 0.f) r.x[2] = p.ref[row];
    if (p.w) r.x[3] = p.w[row];
  }
  return r;
}
// The same in one register while the row is read: a number for each of a warp's first lanes, from one load.  (With four more registers the
// narrow rows' policy kernel spaced its loads out: 8000 x 4600 in fp32 66 us for 57.)  By whole warps.
struct LaneNumbers {
  float z = 0.f, v = 1.f;
  __device__ __forceinline__ RowNumbers all() const {
    RowNumbers r;
    r.z = z;
#pragma unroll
    for (int i = 0; i < 4; i++) r.x[i] = __shfl_sync(0xffffffffu, v, i);
    return r;
  }
};
template <typename T, RowsMode MODE, bool ENTROPY> __device__ __forceinline__ LaneNumbers lane_numbers(const RowsArgs& p, long long row, const T* z, int t) {
  LaneNumbers r;
  r.z = to_f<T>(z[t]);
  const int lane = threadIdx.x & 31;
  const float* from = nullptr;
  if (MODE == GRADIENT) from = lane == 0 ? p.dlogp : ENTROPY && lane == 1 ? p.dent : nullptr;
  if (MODE == POLICY) from = lane == 0 ? p.old : lane == 1 ? p.adv : lane == 2 && p.term.kl != 0.f ? p.ref : lane == 3 ? p.w : nullptr;
  if (from) r.v = from[row];
  return r;
}
// A kernel that started beside the one that counts the targets does not end before it, even if no row of its has asked for the count: what follows
// in the stream waits for this kernel alone.
template <RowsMode MODE> __device__ __forceinline__ void end_behind_the_count(const RowsArgs& p) {
  if (MODE == POLICY && p.n_valid) pdl_wait();
}

// What the gradient of a row needs: dz_j = 2^u_j (k + h u_j) for j other than the target, u_j = c (z_j - m), and the target's.
struct RowSlope {
  float m = 0.f, k = 0.f, h = 0.f, target = 0.f;
};
// dz_j = g (1[j = t] - p_j) - y p_j (u_j - a / l), where log p + H = ln2 (u - a / l) and y has the factor ln2.  At the target 1 - p comes from the
// other tokens' part of l.  A row without a distribution has no gradient.
template <bool ENTROPY> __device__ __forceinline__ RowSlope row_slope(const TokenStats& s, float g, float y, float c) {
  RowSlope r;
  if (s.all.l == 0.f) return r;
  const float inv_l = 1.f / s.all.l, mean = ENTROPY ? s.all.a / s.all.l : 0.f;
  r.m = s.all.m;
  r.k = -(ENTROPY ? g - y * mean : g) * inv_l;
  r.h = ENTROPY ? -y * inv_l : 0.f;
  r.target = g * (s.others * inv_l);
  if (ENTROPY) {
    const float u = fmaxf((s.z - s.all.m) * c, LEAST_U);
    r.target += exp2_fast(u) * inv_l * (y * (mean - u));
  }
  return r;
}
// The row's numbers go out (where `write`), and what its gradient needs comes back, from the statistics of the tokens other than its target.
// scale: 0 until the rows with a target have been counted.
template <RowsMode MODE, bool ENTROPY>
__device__ __forceinline__ RowSlope row_result(const RowsArgs& p, long long row, const RowStats& others, const RowNumbers& k, float& scale, bool write) {
  const TokenStats s = with_token<ENTROPY>(others, k.z, p.c);
  if (MODE == LOGPROBS) {
    if (write) {
      p.logp[row] = (float)log_prob(s, p.inv_t64);
      if (ENTROPY) p.ent[row] = entropy(s);
    }
    return RowSlope();
  }
  if (MODE == GRADIENT) return row_slope<ENTROPY>(s, k.x[0] * p.inv_t, ENTROPY ? k.x[1] * p.inv_t * (float)LN2 : 0.f, p.c);
  const double lp = log_prob(s, p.inv_t64);
  float loss, slope;
  policy_token(p.term, lp, k.x[0], k.x[1], k.x[2], k.x[3], &loss, &slope);
  if (write) { p.token_losses[row] = loss; p.logp[row] = (float)lp; }
  if (p.n_valid && scale == 0.f) {      // a kernel of the same call counts the targets beside the first rows
    pdl_wait();
    scale = 1.f / (float)*reinterpret_cast<const volatile int*>(p.n_valid);
  }
  if (k.x[3] == 0.f) return RowSlope();      // whatever the logits are.  Behind the wait: a kernel of few rows ends behind the count by it
  return row_slope<false>(s, (p.n_valid ? slope * scale : slope) * p.inv_t, 0.f, p.c);
}
template <RowsMode MODE, bool ENTROPY> __device__ __forceinline__ void row_without_target(const RowsArgs& p, long long row) {
  if (MODE == LOGPROBS) { p.logp[row] = 0.f; if (ENTROPY) p.ent[row] = 0.f; }
  if (MODE == POLICY) p.logp[row] = p.token_losses[row] = 0.f;
}

// POLICY: rows with k = 0 (clipped, or of weight 0) have zeros, whatever their logits are.  Where k is infinite (the KL term of a token that the model
// rules out, or all but) tokens of p = 0 still have no gradient: such rows are written element by element.
template <typename T, bool ENTROPY, bool POLICY> struct Slope {
  static constexpr int n = VecN<T>::n;
  Exponent x;
  uint64_t k2, h2;
  float at_target;
  int t;
  bool zero, unbounded;
  __device__ __forceinline__ Slope(const RowSlope& s, float c, int target)
      : x(s.m, c), k2(pack2(s.k, s.k)), h2(pack2(s.h, s.h)), at_target(s.target), t(target), zero(POLICY && s.k == 0.f),
        unbounded(POLICY && fabsf(s.k) == INFINITY) {}
  __device__ __forceinline__ uint64_t of(uint64_t z2) const {
    float u0, u1;
    x.of(z2, u0, u1);
    const uint64_t e2 = pack2(exp2_fast(u0), exp2_fast(u1));
    return mul2(e2, ENTROPY ? fma2(h2, pack2(fmaxf(u0, LEAST_U), fmaxf(u1, LEAST_U)), k2) : k2);
  }
  __device__ __forceinline__ void elements(uint64_t z2, float& lo, float& hi) const {
    float k, unused;
    unpack2(of(z2), lo, hi);
    if (zero) lo = hi = 0.f;
    if (unbounded) {
      x.of(z2, lo, hi);
      unpack2(k2, k, unused);
      lo = exp2_fast(lo) == 0.f ? 0.f : exp2_fast(lo) * k;
      hi = exp2_fast(hi) == 0.f ? 0.f : exp2_fast(hi) * k;
    }
  }
  // (Rows of zeros take a loop of their own: with the question at every word the policy's kernel for medium rows took 56 us for 53.)
  __device__ __forceinline__ uint4 word(const uint4& q) const {
    uint4 o;
#pragma unroll
    for (int i = 0; i < n / 2; i++) Word<T>::put(o, i, of(Word<T>::get(q, i)));
    return o;
  }
  __device__ __forceinline__ uint4 word_or_zeros(const uint4& q) const { return zero ? make_uint4(0, 0, 0, 0) : word(q); }
  // a word that does not lie in the gradient as it does in the logits
  __device__ __forceinline__ void scatter(T* d, const uint4& q) const {
#pragma unroll
    for (int i = 0; i < n / 2; i++) {
      float lo, hi;
      elements(Word<T>::get(q, i), lo, hi);
      d[2 * i] = from_f<T>(lo);
      d[2 * i + 1] = from_f<T>(hi);
    }
  }
  // The target's element, over what stands there of its word, by the thread that stored the word.  (A comparison with the target at every word was
  // a third of the instructions.)
  __device__ __forceinline__ void store_target(T* d) const { d[t] = from_f<T>(at_target); }
  __device__ __forceinline__ void store_edge(T* d, int at, float z) const {
    float lo, hi;
    elements(pack2(z, z), lo, hi);
    d[at] = from_f<T>(at == t ? at_target : lo);
  }
};
// Words of the gradient may be stored whole where they lie as the logits' do.
template <typename T> __device__ __forceinline__ bool same_phase(const T* z, const T* d) {
  return ((reinterpret_cast<uintptr_t>(z) ^ reinterpret_cast<uintptr_t>(d)) & 15) == 0;
}

__device__ __forceinline__ void group_barrier(int id, int threads) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory"); }

// ---- few rows -----------------------------------------------------------------------------------------------------------------------------------
// A cluster of blocks holds a row in registers, NV words a thread; the statistics of all its warps go to every block's shared memory.  There is
// little to overlap: what counts is that a row is brought by many multiprocessors at once (1 x 65536 in fp32: 3.1 us, of which a launch with
// nothing to do is 2).  Four blocks a multiprocessor in fp32: left to the compiler, 220 rows of 50021 take 32 us for 24 (gradient, three blocks), 150 of 8000
// 4.2 for 3.7 (numbers only, fewer words on their way).
constexpr int FEW_WARPS = 8, FEW_WORDS = 8;

template <typename T, RowsMode MODE, bool STORE, bool ENTROPY, int NV>
__global__ void __launch_bounds__(32 * FEW_WARPS, sizeof(T) == 4 && NV == FEW_WORDS ? 4 : 0) k_rows_few(const RowsArgs p) {
  pdl_trigger();
  constexpr int threads = 32 * FEW_WARPS, pitch = MOST_CLUSTER * FEW_WARPS;
  __shared__ float part[3 * pitch];
  __shared__ RowSlope slope_s;
  const int C = (int)cluster_size(), rank = (int)cluster_rank(), tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory");      // this block runs: its shared memory may be written
  const long long row = blockIdx.x / C;
  const int t = checked_target(p, p.tgt0[row], rank == 0 && tid == 0);
  const T* z = reinterpret_cast<const T*>(p.logits) + row * p.ldl;
  T* d = reinterpret_cast<T*>(p.dlogits) + row * p.ldd;
  const RowShape r = row_shape<T>(STORE && t < 0 ? d : z, p.V);      // the logits', or, where they are not read, the gradient's
  const int per = (r.nvec + C - 1) / C, first = min(r.nvec, rank * per), last = min(r.nvec, first + per);
  // the word that holds the target goes with the elements outside the words, one to a thread
  const int vt = t >= 0 ? word_of_target<T>(r, t) : -1;
  const int at = rank != 0 ? -1 : vt >= 0 && tid >= 8 && tid < 8 + VecN<T>::n ? r.head + vt * VecN<T>::n + tid - 8 : edge_of<T>(r, tid);
  if (t < 0) {
    asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
    if (rank == 0 && tid == 0) row_without_target<MODE, ENTROPY>(p, row);
    if (STORE) {
      for (int v = first + tid; v < last; v += threads) reinterpret_cast<uint4*>(d + r.head)[v] = make_uint4(0, 0, 0, 0);
      if (at >= 0) d[at] = from_f<T>(0.f);
    }
    end_behind_the_count<MODE>(p);
    return;
  }
  const uint4* words = reinterpret_cast<const uint4*>(z + r.head);
  uint4 q[NV];
#pragma unroll
  for (int k = 0; k < NV; k++) {
    const int v = first + k * threads + tid;
    q[k] = load_word(words + v, v < last && v != vt, Word<T>::LEAST);
  }
  RowNumbers numbers;
  if (warp == 0) numbers = row_numbers<T, MODE, ENTROPY>(p, row, z, t);      // in every block: each works the slopes out for itself
  const bool there = at >= 0 && at != t;
  const float edge = there ? to_f<T>(z[at]) : -INFINITY;
  Running<T, ENTROPY> run(there, edge, p.c);
  run.add(q, p.c);
  const RowStats s = run.of_warp(p.c);
  asm volatile("barrier.cluster.wait.acquire;" ::: "memory");      // all blocks run
  const int slot = rank * FEW_WARPS + warp;
  if (lane < C) {
    store_remote(part + slot, lane, s.m); store_remote(part + pitch + slot, lane, s.l);
    if (ENTROPY) store_remote(part + 2 * pitch + slot, lane, s.a);
  }
  asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;" ::: "memory");
  if (!STORE && (rank != 0 || warp != 0)) return;
  if (warp == 0) {
    float scale = 0.f;
    const RowSlope given = row_result<MODE, ENTROPY>(p, row, merged_parts<ENTROPY>(part, pitch, FEW_WARPS * C, p.c), numbers, scale, rank == 0 && lane == 0);
    if (lane == 0) slope_s = given;
  }
  if (!STORE) return;
  __syncthreads();
  const Slope<T, ENTROPY, MODE == POLICY> slope(slope_s, p.c, t);
  const bool same = same_phase(z, d) && !slope.unbounded;
#pragma unroll
  for (int k = 0; k < NV; k++) {
    const int v = first + k * threads + tid;
    if (v >= last || v == vt) continue;
    if (same) reinterpret_cast<uint4*>(d + r.head)[v] = slope.word_or_zeros(q[k]);
    else slope.scatter(d + r.head + v * VecN<T>::n, q[k]);
  }
  if (at >= 0) slope.store_edge(d, at, edge);
}

// ---- narrow rows --------------------------------------------------------------------------------------------------------------------------------
// Groups of W warps walk the rows in turn.  A group has two buffers in shared memory: while it works on a row, a bulk copy brings its next one,
// and three blocks a multiprocessor keep up to 24 rows going.  Rows in registers, one group of warps each, took 56 us where this takes 45
// (8192 x 4096 in fp32, gradient): a row's loads could not start before the row ahead was written.
constexpr int NEAR_WARPS = 8, NEAR_WORDS = 4;

template <typename T, RowsMode MODE, bool STORE, bool ENTROPY>
__global__ void __launch_bounds__(32 * NEAR_WARPS, 3) k_rows_near(const RowsArgs p, const int W, const int pitch) {
  pdl_trigger();
  extern __shared__ __align__(128) uint4 ring[];
  __shared__ uint64_t full[NEAR_WARPS][2];
  __shared__ float part[2][3][NEAR_WARPS];
  __shared__ RowSlope slope_s[NEAR_WARPS];
  __shared__ int abort_flag;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, group = warp / W, groups = blockDim.x / (32 * W);
  const int threads = W * 32, tid = threadIdx.x - group * threads, first_warp = group * W;
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2 * NEAR_WARPS; i++) mbar_init(&full[i / 2][i % 2], 1);
    abort_flag = 0;
    fence_barrier_init();
  }
  __syncthreads();
  uint4* buffer = ring + (size_t)group * 2 * pitch;
  // one thread of the group asks for a row's words
  auto ask = [&](long long row, int which) {
    const T* z = reinterpret_cast<const T*>(p.logits) + row * p.ldl;
    const RowShape r = row_shape<T>(z, p.V);
    if (r.nvec > 0) {
      mbar_expect_tx(&full[group][which], (uint32_t)r.nvec * 16u);
      bulk_load_1d(buffer + (size_t)which * pitch, z + r.head, (uint32_t)r.nvec * 16u, &full[group][which]);
    } else mbar_arrive(&full[group][which]);
  };
  const long long step = (long long)gridDim.x * groups;
  long long row = (long long)blockIdx.x * groups + group;
  Targets targets(p, row, step);
  int t_next = targets(0), k = 0, n_asked = 0;      // k: rows with a target so far
  bool alive = true, asked = false;
  float scale = 0.f;
  for (int nth = 1; row < p.N; row += step, nth++) {
    const int t = checked_target(p, t_next, tid == 0);
    t_next = targets(nth);
    const T* z = reinterpret_cast<const T*>(p.logits) + row * p.ldl;
    T* d = reinterpret_cast<T*>(p.dlogits) + row * p.ldd;
    const RowShape r = row_shape<T>(STORE && t < 0 ? d : z, p.V);      // the logits', or, where they are not read, the gradient's
    const int at = edge_of<T>(r, tid);
    if (t < 0) {
      if (tid == 0) row_without_target<MODE, ENTROPY>(p, row);
      if (STORE) {
        for (int v = tid; v < r.nvec; v += threads) reinterpret_cast<uint4*>(d + r.head)[v] = make_uint4(0, 0, 0, 0);
        if (at >= 0) d[at] = from_f<T>(0.f);
      }
      continue;
    }
    const int which = k & 1;
    const uint32_t parity = (uint32_t)(k >> 1) & 1u;
    k++;
    if (!asked && tid == 0 && alive) { ask(row, which); n_asked = k; }      // the row before the last but one, which this buffer held, is done: a barrier lies between
    LaneNumbers numbers;
    if (warp == first_warp) numbers = lane_numbers<T, MODE, ENTROPY>(p, row, z, t);
    const bool there = at >= 0 && at != t;
    const float edge = there ? to_f<T>(z[at]) : -INFINITY;
    Running<T, ENTROPY> run(there, edge, p.c);
    const int vt = word_of_target<T>(r, t);
    const bool own = vt >= 0 && (vt & (threads - 1)) == tid;      // the target's word is this thread's (W is a power of two)
    uint4* words = buffer + (size_t)which * pitch;
    alive = alive && mbar_wait_limit(&full[group][which], parity, &abort_flag, &g_rows_status, p.wait_limit);
    if (own) take_out<T>(words + vt, (t - r.head) % VecN<T>::n);
    int v0 = 0;
    for (; v0 + NEAR_WORDS * threads <= r.nvec; v0 += NEAR_WORDS * threads) {
      uint4 q[NEAR_WORDS];
#pragma unroll
      for (int h = 0; h < NEAR_WORDS; h++) q[h] = words[v0 + h * threads + tid];
      run.add(q, p.c);
    }
    run.template add_rest<NEAR_WORDS>(words + v0 + tid, threads, r.nvec - v0 - tid, r.nvec - v0, p.c, [] {});
    RowStats s = run.of_warp(p.c);
    if (W > 1) {
      float* mine = part[which][0];
      if (lane == 0) { mine[warp] = s.m; mine[NEAR_WARPS + warp] = s.l; if (ENTROPY) mine[2 * NEAR_WARPS + warp] = s.a; }
      group_barrier(1 + group, threads);
      if (warp == first_warp) s = merged_parts<ENTROPY>(mine + first_warp, NEAR_WARPS, W, p.c);
    } else __syncwarp();
    // all of the group are done with the row before this one: its buffer is free
    asked = t_next >= 0 && t_next < p.V;
    if (asked && tid == 0 && alive) { ask(row + step, which ^ 1); n_asked = k + 1; }
    RowSlope given;
    if (warp == first_warp) given = row_result<MODE, ENTROPY>(p, row, s, numbers.all(), scale, lane == 0);
    if (!STORE) continue;
    if (W > 1) {
      if (warp == first_warp && lane == 0) slope_s[group] = given;
      group_barrier(1 + group, threads);
      given = slope_s[group];
    }
    const Slope<T, ENTROPY, MODE == POLICY> slope(given, p.c, t);
    const bool same = same_phase(z, d) && !slope.unbounded;
    if (same) {
      uint4* out = reinterpret_cast<uint4*>(d + r.head);
      // Four words at a time while every thread has as many, and one by one from there: unrolled with a remainder for each thread, the code of
      // 24 warps that are at different places of it took more time than its instructions (30000 x 1000 in bf16: 38 -> 32 us).
      int v = 0;
      for (; !slope.zero && v + 4 * threads <= r.nvec; v += 4 * threads) {
        uint4 q[4];
#pragma unroll
        for (int h = 0; h < 4; h++) q[h] = words[v + h * threads + tid];
#pragma unroll
        for (int h = 0; h < 4; h++) out[v + h * threads + tid] = slope.word(q[h]);
      }
#pragma unroll 1
      for (v += tid; v < r.nvec; v += threads) out[v] = slope.word_or_zeros(words[v]);
    } else {
      for (int v = tid; v < r.nvec; v += threads) slope.scatter(d + r.head + v * VecN<T>::n, words[v]);
    }
    if (own) slope.store_target(d);
    if (at >= 0) slope.store_edge(d, at, edge);
  }
  end_behind_the_count<MODE>(p);
  if (!alive && tid == 0)      // nothing may still be on its way to this block's memory when it ends: the last row asked for in either buffer
    for (int b = 0; b < 2; b++)
      for (uint32_t polls = 0; n_asked > b && polls < WAIT_LIMIT && !mbar_try_wait(&full[group][b], (uint32_t)((n_asked - b - 1) >> 1) & 1u); polls++) {}
}

// ---- rows through a ring in shared memory -----------------------------------------------------------------------------------------------------
// One block a multiprocessor: a warp brings the words of its rows in chunks (bulk copies, an mbarrier each), and groups of warps take the rows
// in turn, so that one's pass over a row goes on while another works out its slopes or writes its gradient.  Chunks stay where they are until
// their gradient is written.  Of a row that the ring does not hold the first chunks are given back at once and brought `again`, behind the
// row's last: two passes over the ring's length later they are still in L2.  Wide rows are shared by the two blocks of a cluster, half a row each, so
// that a ring holds more of the rows that follow; their groups exchange statistics.  The warp that brings rows also writes the zeros of those without
// target, by bulk copies, one such row behind each that it brings: all at once in their turn they took the reads' place (4096 x 65536 in bf16, the
// first half of the rows without target, gradient: 157 -> 145 us).
template <int BLOCKS_, int GROUPS_, int WARPS_, int PER_, int SLOTS_> struct Ring {
  static constexpr int BLOCKS = BLOCKS_, GROUPS = GROUPS_, WARPS = WARPS_, THREADS = 32 * WARPS_, PER = PER_, CHUNK = PER_ * THREADS, SLOTS = SLOTS_;
  static constexpr int SPARE = 2;      // slots that a row wider than the ring leaves to what follows
  static constexpr int BLOCK = GROUPS * THREADS + 32;
  static constexpr int ZEROS = 512;      // words of zeros behind the ring, the source of the gradient of rows without target
  static constexpr size_t BYTES = ((size_t)SLOTS * CHUNK + ZEROS) * 16;
};
// Four numbers to where `local` lies in another block of the cluster, 16 bytes that its barrier counts.
__device__ __forceinline__ void send_remote(const float4* local, const uint64_t* barrier, uint32_t rank, float4 v) {
  asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v4.f32 [%0], {%1, %2, %3, %4}, [%5];"
               ::"r"(remote_address(local, rank)), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w), "r"(remote_address(barrier, rank)) : "memory");
}
// As mbar_wait_limit, for what another block of the cluster sends.
__device__ __forceinline__ bool mbar_try_wait_cluster(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile("{\n.reg .pred p;\nmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}"
               : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity) : "memory");
  return ok != 0;
}
__device__ __forceinline__ bool mbar_wait_cluster(uint64_t* bar, uint32_t parity, volatile int* abort_flag, uint32_t limit) {
  for (uint32_t polls = 0; polls < limit; polls++) {
    if (mbar_try_wait_cluster(bar, parity)) return true;
    if ((polls & 255u) == 255u && *abort_flag) return false;
  }
  *abort_flag = 1;
  atomicOr(&g_rows_status, ST_WAIT_TIMEOUT);
  return false;
}
__device__ __forceinline__ void bulk_store_1d(void* gdst, const void* smem_src, uint32_t bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(gdst), "r"(smem_u32(smem_src)), "r"(bytes) : "memory");
}
template <typename T, RowsMode MODE, bool STORE, bool ENTROPY, class R>
__global__ void __launch_bounds__(R::BLOCK) k_rows_ring(const RowsArgs p, const int chunks, const int again) {
  constexpr int C = R::BLOCKS, GROUPS = R::GROUPS, GROUP_WARPS = R::WARPS, GROUP_THREADS = R::THREADS, PER_CHUNK = R::PER, CHUNK = R::CHUNK, SLOTS = R::SLOTS;
  auto next_slot = [](int slot) { return slot + 1 == SLOTS ? 0 : slot + 1; };
  pdl_trigger();
  extern __shared__ __align__(128) uint4 ring[];
  __shared__ uint64_t full[GROUPS][SLOTS], empty[SLOTS];
  __shared__ float part[GROUPS][3][GROUP_WARPS];
  __shared__ RowSlope slope_s[GROUPS];
  __shared__ uint64_t met[GROUPS][2];      // a group's statistics of a row from the other block of the cluster, two rows in turn
  __shared__ __align__(16) float4 theirs[GROUPS][2];
  __shared__ int their_sent[GROUPS];      // how many rows' statistics the other block has sent in all
  __shared__ int abort_flag;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, rank = C > 1 ? (int)cluster_rank() : 0;
  const long long first_row = blockIdx.x / C, step = gridDim.x / C;
  if (threadIdx.x == 0) {
    for (int i = 0; i < SLOTS; i++) {
      for (int g = 0; g < GROUPS; g++) mbar_init(&full[g][i], 1);
      mbar_init(&empty[i], GROUP_WARPS);
    }
    for (int g = 0; g < GROUPS; g++) { mbar_init(&met[g][0], 1); mbar_init(&met[g][1], 1); }
    abort_flag = 0;
    fence_barrier_init();
  }
  uint4* zeros = ring + (size_t)SLOTS * CHUNK;
  if (STORE) {
    for (int i = threadIdx.x; i < R::ZEROS; i += R::BLOCK) zeros[i] = make_uint4(0, 0, 0, 0);
    fence_proxy_async();
  }
  __syncthreads();
  if (C > 1) asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;" ::: "memory");      // the other block's barriers are there
  // the words of a row that are this block's
  auto mine_of = [&](const RowShape& r, int& from) {
    const int per = (r.nvec + C - 1) / C;
    from = min(r.nvec, rank * per);
    return min(r.nvec, from + per) - from;
  };
  if (warp == GROUPS * GROUP_WARPS) {      // the warp that brings the rows
    int slot = 0, k = 0, nth = 0;
    uint32_t round = 0, used[GROUPS] = {}, parity[GROUPS] = {};      // bits: slots that a group's barriers have been used for, and how often, modulo 2
    bool alive = true;
    auto bring = [&](const uint4* words, int nvec, int n_chunks, int group) {      // by one lane
      for (int c = 0; c < n_chunks; c++) {
        if (round > 0) alive = mbar_wait_limit(&empty[slot], (round - 1) & 1u, &abort_flag, &g_rows_status, p.wait_limit);
        if (!alive) return;
        const int n = min(CHUNK, nvec - c * CHUNK);
        if (n > 0) {
          mbar_expect_tx(&full[group][slot], (uint32_t)n * 16u);
          bulk_load_1d(ring + (size_t)slot * CHUNK, words + (size_t)c * CHUNK, (uint32_t)n * 16u, &full[group][slot]);
        } else mbar_arrive(&full[group][slot]);
        used[group] |= 1u << slot;
        parity[group] ^= 1u << slot;
        slot = next_slot(slot);
        if (slot == 0) round++;
      }
    };
    // the next row without target among the block's first `end`, behind those that have been dealt with
    Targets masked(p, first_row, step);
    int masked_nth = 0;
    auto clear_next = [&](int end) -> bool {
      for (long long row; masked_nth < end && (row = first_row + (long long)masked_nth * step) < p.N;) {
        const int t = masked(masked_nth++);
        if (t >= 0 && t < p.V) continue;
        if (rank == 0 && lane == 0) row_without_target<MODE, ENTROPY>(p, row);
        if (STORE) {
          T* d = reinterpret_cast<T*>(p.dlogits) + row * p.ldd;
          const RowShape r = row_shape<T>(d, p.V);
          if (lane == 0) {
            int from;
            const int n = mine_of(r, from);
            uint4* words = reinterpret_cast<uint4*>(d + r.head) + from;
            for (int v = 0; v < n; v += R::ZEROS) bulk_store_1d(words + v, zeros, (uint32_t)min(R::ZEROS, n - v) * 16u);
            bulk_commit();
          }
          const int at = rank == 0 ? edge_of<T>(r, lane) : -1;
          if (at >= 0) d[at] = from_f<T>(0.f);
        }
        return true;
      }
      return false;
    };
    Targets targets(p, first_row, step);
    for (long long row = first_row; row < p.N; row += step) {
      const int t = targets(nth++);
      if (t < 0 || t >= p.V) continue;
      const T* z = reinterpret_cast<const T*>(p.logits) + row * p.ldl;
      const RowShape r = row_shape<T>(z, p.V);
      int from;
      const int n = mine_of(r, from);
      const uint4* words = reinterpret_cast<const uint4*>(z + r.head) + from;
      if (lane == 0) {
        if (alive) bring(words, n, chunks, k % GROUPS);
        if (STORE && alive) bring(words, n, again, k % GROUPS);
      }
      __syncwarp();
      clear_next(nth);
      k++;
    }
    while (clear_next(INT_MAX)) {}
    if (STORE && lane == 0) bulk_wait_all();
    group_barrier(0, R::BLOCK);                                 // every group has dealt with its rows, or given up,
    if (lane == 0 && *(const volatile int*)&abort_flag)      // and nothing may still be on its way to this block's memory when it ends
      for (int i = 0; i < GROUPS * SLOTS; i++)
        if (used[i / SLOTS] >> (i % SLOTS) & 1u)
          for (uint32_t polls = 0; polls < WAIT_LIMIT && !mbar_try_wait(&full[i / SLOTS][i % SLOTS], (parity[i / SLOTS] >> (i % SLOTS) & 1u) ^ 1u); polls++) {}
    __syncwarp();
    if (C > 1) asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;" ::: "memory");
    return;
  }

  const int group = warp / GROUP_WARPS, tid = threadIdx.x - group * GROUP_THREADS, gwarp = warp - group * GROUP_WARPS;
  // After a wait that ran out nothing is waited for any more (barriers of the group are), and no slot is handed back: the copy into it may not have come,
  // and a barrier is not armed for another one before.  (The bringing warp asking for the flag ahead of each copy: 8000 x 16000 in bf16, numbers only, 71 us for 53.)
  bool alive = true;
  // How often the group has waited for each slot, modulo 2.  A group's barriers are its own: of a barrier for both, a group that waits while the
  // other's row passes through the slot could not tell the phase it waits for from the one before the other's.
  uint32_t parity = 0;
  auto wait_full = [&](int slot) {
    alive = alive && mbar_wait_limit(&full[group][slot], parity >> slot & 1u, &abort_flag, &g_rows_status, p.wait_limit);
    parity ^= 1u << slot;
  };
  int k = 0, nth = 0;
  uint32_t rows = 0, sent = 0;      // that the group has worked on; whose statistics have gone to the other block
  float scale = 0.f;
  Targets targets(p, first_row, step);
  for (long long row = first_row; row < p.N; row += step) {
    const int t = checked_target(p, targets(nth++), rank == 0 && threadIdx.x == 0);
    if (t < 0) continue;
    const int mine = k++;
    if (mine % GROUPS != group) continue;
    const T* z = reinterpret_cast<const T*>(p.logits) + row * p.ldl;
    T* d = reinterpret_cast<T*>(p.dlogits) + row * p.ldd;
    const RowShape r = row_shape<T>(z, p.V);
    int from_word;
    const int nvec = mine_of(r, from_word);
    const int at = rank == 0 ? edge_of<T>(r, tid) : -1;
    RowNumbers numbers;
    if (gwarp == 0) numbers = row_numbers<T, MODE, ENTROPY>(p, row, z, t);
    const bool there = at >= 0 && at != t;
    const float edge = there ? to_f<T>(z[at]) : -INFINITY;

    Running<T, ENTROPY> run(there, edge, p.c);
    const int vt = word_of_target<T>(r, t) - from_word;
    const bool own = vt >= 0 && vt < nvec && vt % CHUNK % GROUP_THREADS == tid;      // the target's word is this thread's
    const int target_chunk = own ? vt / CHUNK : -1;
    const int first_slot = (int)((long long)mine * (chunks + (STORE ? again : 0)) % SLOTS);
    int slot = first_slot;
    for (int c = 0; c < chunks; c++, slot = next_slot(slot)) {
      wait_full(slot);
      if (c == target_chunk) take_out<T>(ring + slot * CHUNK + vt % CHUNK, (t - r.head) % VecN<T>::n);
      const uint4* from = ring + slot * CHUNK + tid;
      auto done = [&]() {
        if (STORE && c >= again) return;
        __syncwarp();
        if (lane == 0 && alive) mbar_arrive(&empty[slot]);
      };
      if ((c + 1) * CHUNK <= nvec) {
        uint4 q[PER_CHUNK];
#pragma unroll
        for (int h = 0; h < PER_CHUNK; h++) q[h] = from[h * GROUP_THREADS];
        done();
        run.add(q, p.c);
      } else {      // a row's last
        run.template add_rest<PER_CHUNK>(from, GROUP_THREADS, nvec - c * CHUNK - tid, nvec - c * CHUNK, p.c, done);
      }
    }
    RowStats s = run.of_warp(p.c);
    float* parts = part[group][0];
    if (lane == 0) { parts[gwarp] = s.m; parts[GROUP_WARPS + gwarp] = s.l; if (ENTROPY) parts[2 * GROUP_WARPS + gwarp] = s.a; }
    group_barrier(1 + group, GROUP_THREADS);
    if (gwarp == 0) {
      s = merged_parts<ENTROPY>(parts, GROUP_WARPS, GROUP_WARPS, p.c);
      if (C > 1) {
        // Two rows in turn: the other block sends a row's statistics when it has this block's of the row before, and those go out ahead of the wait.
        const int turn = rows & 1u;
        if (lane == 0 && alive) {
          sent++;
          mbar_expect_tx(&met[group][turn], 16);
          // the target's logit goes along: it has been read then, and the other block may write over it
          send_remote(&theirs[group][turn], &met[group][turn], rank ^ 1, make_float4(s.m, s.l, s.a, numbers.z));
        }
        alive = alive && mbar_wait_cluster(&met[group][turn], rows >> 1 & 1u, &abort_flag, p.wait_limit);
        __syncwarp();
        const float4 o = theirs[group][turn];
        RowStats other;
        other.m = o.x; other.l = o.y; other.a = o.z;
        s = rank == 0 ? merged<ENTROPY>(s, other, p.c) : merged<ENTROPY>(other, s, p.c);      // the same order, the same bits, in both
      }
      const RowSlope given = row_result<MODE, ENTROPY>(p, row, s, numbers, scale, rank == 0 && lane == 0);
      if (STORE && lane == 0) slope_s[group] = given;
    }
    rows++;
    group_barrier(1 + group, GROUP_THREADS);      // the parts are read, the slopes are there
    if (!STORE) continue;
    const Slope<T, ENTROPY, MODE == POLICY> slope(slope_s[group], p.c, t);
    const bool same = same_phase(z, d) && !slope.unbounded;
    slot = (first_slot + again) % SLOTS;
    for (int i = 0; i < chunks; i++, slot = next_slot(slot)) {
      const int c = i + again < chunks ? i + again : i + again - chunks;      // those that are still here first
      if (i + again >= chunks) wait_full(slot);
      const uint4* from = ring + slot * CHUNK + tid;
      if (same && !slope.zero && (c + 1) * CHUNK <= nvec) {
        uint4* out = reinterpret_cast<uint4*>(d + r.head) + from_word + c * CHUNK + tid;
#pragma unroll
        for (int h = 0; h < PER_CHUNK; h++) out[h * GROUP_THREADS] = slope.word(from[h * GROUP_THREADS]);
      } else {
        for (int h = 0, v = c * CHUNK + tid; v < nvec && h < PER_CHUNK; h++, v += GROUP_THREADS) {
          if (same) reinterpret_cast<uint4*>(d + r.head)[from_word + v] = slope.word_or_zeros(from[h * GROUP_THREADS]);
          else slope.scatter(d + r.head + (from_word + v) * VecN<T>::n, from[h * GROUP_THREADS]);
        }
      }
      __syncwarp();
      if (lane == 0 && alive) mbar_arrive(&empty[slot]);
    }
    if (own) slope.store_target(d);
    if (at >= 0) slope.store_edge(d, at, edge);
  }
  end_behind_the_count<MODE>(p);
  const bool leader = gwarp == 0 && lane == 0;
  if (C > 1 && leader) store_remote(&their_sent[group], rank ^ 1, (int)sent);
  group_barrier(0, R::BLOCK);
  if (C > 1) {
    asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;" ::: "memory");      // the other block sends nothing more
    // Where every wait came to its end, all that was sent has come.  Behind one that ran out the last of either turn may be on its way to this block's
    // memory: waited for as well, after arming the barrier for one that this block did not wait for.  (The other block sends a row's when it
    // has this block's of the row before: one more at the most.)
    if (leader && *(const volatile int*)&abort_flag)
      for (int turn = 0; turn < 2; turn++) {
        const int here = ((int)sent + 1 - turn) / 2, came = (*(const volatile int*)&their_sent[group] + 1 - turn) / 2;
        auto settle = [&](int n) { for (uint32_t polls = 0; n > 0 && polls < WAIT_LIMIT && !mbar_try_wait_cluster(&met[group][turn], (uint32_t)(n - 1) & 1u); polls++) {} };
        settle(min(here, came));
        if (came > here) { mbar_expect_tx(&met[group][turn], 16); settle(came); }
      }
  }
}

// ---- launch -----------------------------------------------------------------------------------------------------------------------------------
// Where the kernels meet (gradient, us; the chosen one first).  few / others: 220 rows, where a block each leaves multiprocessors idle in the
// second turn, 65536 fp32 27.0 / 30.7, 8000 fp32 5.7 / 7.6; 296 rows, 65536 bf16 27.3 / 22.6, so not there.  near / a ring: 1024 words (8192 x 4096
// fp32) 45 / 62, 1500 (4000 x 6000 fp32) 35 / 42, (4000 x 12000 bf16) 44 / 46, 1700 (4000 x 13600 bf16, a quarter masked) 43 / 42.  Medium / Wide:
// 2500 words (3000 x 20000 bf16, masked alike) 41 / 48, 5000 (1000 x 40000 bf16) 36 / 39, 6250 (1500 x 25000 fp32) 53 / 59.  Wide / Medium: 8192 words
// (1000 x 32768 fp32) 46 / 48, (2048 x 65536 bf16) 93 / 105, 12505 (999 x 50021 fp32) 62 / 71.
// Medium and writing: 20 warps that may have 80 registers; with 24, as for numbers only, the policy's kernels spill (8000 x 16000 bf16 94 / 105,
// 2000 x 30000 52 / 56, 1500 x 25000 fp32 57 / 61; numbers only, 2000 x 16000 fp32, 29 to the 26 of 24).  Wide and writing: a row to two blocks;
// two groups of twelve warps 112 at 2048 x 65536 bf16, four of six 108, a row to each block (two groups of twelve) 103.  Numbers only: nothing waits for
// its gradient, so a row to a block, in fewer and larger groups, 2048 x 65536 bf16 46 / 53 with Medium, 1500 x 25000 fp32 the same 28.  Eight words a
// thread and wait where a thread took four before: numbers only, 2048 x 65536 bf16, 51 -> 47; the gradient of Wide rows keeps four, eight spill.
constexpr int MOST_NEAR = 1700, MOST_MEDIUM = 7168;      // words of a row
typedef Ring<1, 4, 6, 8, 9> MediumReading;
typedef Ring<1, 4, 5, 8, 10> MediumWriting;
typedef Ring<1, 3, 8, 8, 6> WideReading;
typedef Ring<2, 3, 8, 4, 13> WideWriting;

// Behind the kernel that counts the targets (n_valid) the rows may start at once: nothing else of theirs depends on it, and it started
// itself when everything before the call was done.  Otherwise the launch is an ordinary one.
template <typename... P, typename... A>
int launch_kernel(const RowsArgs& p, void (*kernel)(P...), int C, dim3 grid, int threads, size_t smem, cudaStream_t s, const A&... args) {
  if (p.n_valid) {
    CUDA_TRY(launch_dependent_clusters(kernel, C, grid, dim3(threads), smem, s, args...));
  } else {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = C; at.val.clusterDim.y = 1; at.val.clusterDim.z = 1;
    cfg.gridDim = grid; cfg.blockDim = dim3(threads); cfg.dynamicSmemBytes = smem; cfg.stream = s;
    cfg.attrs = &at; cfg.numAttrs = C > 1;
    CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...));
  }
  KERNEL_CHECK();
  return 0;
}
template <typename T, RowsMode MODE, bool STORE, bool ENTROPY, class R> int launch_ring(const RowsArgs& p, int words, cudaStream_t s) {
  constexpr auto kernel = k_rows_ring<T, MODE, STORE, ENTROPY, R>;
  const int chunks = cdiv(cdiv(words, R::BLOCKS), R::CHUNK), again = chunks <= R::SLOTS ? 0 : chunks - (R::SLOTS - R::SPARE);
  FEMTO_TRY(allow_smem<kernel>(R::BYTES));
  return launch_kernel(p, kernel, R::BLOCKS, dim3((unsigned)(std::min(p.N, device_sm_count() / R::BLOCKS) * R::BLOCKS)), R::BLOCK, R::BYTES, s, p, chunks, again);
}
template <typename T, RowsMode MODE, bool STORE, bool ENTROPY> int launch(const RowsArgs& p, cudaStream_t s) {
  const int words = std::max(1, p.V / VecN<T>::n), sms = device_sm_count(), block = 32 * FEW_WARPS;
  if (2ll * p.N < 3 * sms && words <= MOST_CLUSTER * block * FEW_WORDS) {
    // as many blocks for a row as there is room for, while a thread keeps a word; and no fewer than hold it
    int C = 1;
    while (C < MOST_CLUSTER && (words > C * block * FEW_WORDS || ((long long)p.N * C < sms && words > C * block))) C *= 2;
    const dim3 grid((unsigned)(p.N * C));
    if (words <= C * block * 2) return launch_kernel(p, k_rows_few<T, MODE, STORE, ENTROPY, 2>, C, grid, block, 0, s, p);
    return launch_kernel(p, k_rows_few<T, MODE, STORE, ENTROPY, FEW_WORDS>, C, grid, block, 0, s, p);
  }
  if (words <= MOST_NEAR) {
    // W warps a row, `groups` of them a block: most rows in flight on a multiprocessor, if 16 warps work on them.  (Gradient, us, each pair at one size: 300 words
    // of bf16 21 rows of a warp 48, 12 of two warps 62; 450 words 15 of one 54, 12 of two 60; 1150 words of fp32 6 of two 50, 3 of eight 67; but 1280
    // words of bf16 5 of one 98, 4 of four 78.)
    auto smem_of = [&](int n) { return (size_t)n * 2 * words * 16; };
    auto blocks_of = [&](int n) { return std::min(3, (int)((220 << 10) / (smem_of(n) + 2048))); };
    int W = 1, groups = 1, best = 0;
    for (int w = 1; w <= NEAR_WARPS; w *= 2)
      for (int n = 1; n <= NEAR_WARPS / w; n++) {
        const int rows = n * blocks_of(n), score = rows * std::min(16, w * rows);
        if (score >= best) { W = w; groups = n; best = score; }
      }
    const int blocks = blocks_of(groups);
    const size_t smem = smem_of(groups);
    constexpr auto kernel = k_rows_near<T, MODE, STORE, ENTROPY>;
    FEMTO_TRY(allow_smem<kernel>(smem));
    return launch_kernel(p, kernel, 1, dim3((unsigned)std::min(cdiv(p.N, groups), sms * blocks)), 32 * W * groups, smem, s, p, W, words);
  }
  typedef typename std::conditional<STORE, MediumWriting, MediumReading>::type Medium;
  typedef typename std::conditional<STORE, WideWriting, WideReading>::type Wide;
  return words <= MOST_MEDIUM ? launch_ring<T, MODE, STORE, ENTROPY, Medium>(p, words, s) : launch_ring<T, MODE, STORE, ENTROPY, Wide>(p, words, s);
}
template <RowsMode MODE, bool STORE, bool ENTROPY> int typed(int dtype, const RowsArgs& p, cudaStream_t s) {
  return dtype == FEMTO_BF16 ? launch<bf16, MODE, STORE, ENTROPY>(p, s) : launch<float, MODE, STORE, ENTROPY>(p, s);
}
}  // namespace

int objective_rows(int dtype, RowsMode mode, const RowsArgs& p, cudaStream_t s) {
  switch (mode) {
    case LOGPROBS: return p.ent ? typed<LOGPROBS, false, true>(dtype, p, s) : typed<LOGPROBS, false, false>(dtype, p, s);
    case GRADIENT: return p.dent ? typed<GRADIENT, true, true>(dtype, p, s) : typed<GRADIENT, true, false>(dtype, p, s);
    default: return p.dlogits ? typed<POLICY, true, false>(dtype, p, s) : typed<POLICY, false, false>(dtype, p, s);
  }
}

// Status word of these kernels on the current device; reading clears it.
unsigned int objective_rows_status_word() {
  unsigned int w = 0, zero = 0;
  if (cudaMemcpyFromSymbol(&w, g_rows_status, sizeof(w)) != cudaSuccess) return 0;
  if (w) cudaMemcpyToSymbol(g_rows_status, &zero, sizeof(zero));
  return w;
}

// The gradient, or with dlogits = NULL the log-probabilities, by kernels whose waits give up after `polls` polls: right away with 0, while the
// copies that they wait for are on their way.
extern "C" int32_t femto_selftest_rows_wait(int32_t dtype, void* dlogits, const void* logits, int64_t ldl, const int32_t* targets0, int32_t N, int32_t V,
                                            const float* dlogp, float* logp, int32_t polls, int32_t* h_status, void* stream) {
  if (!logits || !targets0 || (dlogits ? !dlogp : !logp) || !h_status || (dtype != FEMTO_F32 && dtype != FEMTO_BF16)) return femto_fail(FEMTO_ERR_ARG, "bad argument");
  if (N <= 0 || V <= 0 || ldl < V || polls < 0) return femto_fail(FEMTO_ERR_SHAPE, "bad shape");
  cudaStream_t s = (cudaStream_t)stream;
  RowsArgs p = {};
  p.logits = logits; p.ldl = p.ldd = ldl; p.dlogits = dlogits; p.tgt0 = targets0; p.N = N; p.V = V;
  p.c = LOG2E; p.inv_t = 1.f; p.inv_t64 = 1.0; p.dlogp = dlogp; p.logp = logp;
  p.wait_limit = (uint32_t)polls;
  objective_rows_status_word();
  FEMTO_TRY(objective_rows(dtype, dlogits ? GRADIENT : LOGPROBS, p, s));
  CUDA_TRY(cudaStreamSynchronize(s));
  *h_status = (int32_t)objective_rows_status_word();
  return 0;
}
