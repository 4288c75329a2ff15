// Log-probabilities of given tokens, the clipped policy loss over packed sequences, and the gradient of both with respect
// to the logits.  One decode engine's samples are scored and trained on with these: logits are the largest tensors of a
// policy step, so everything here is arranged around reading them once per direction.
#include "lfm2_common.h"

namespace {

constexpr float kLn2 = 0.6931471805599453f;
constexpr float kInf = __builtin_huge_valf();

#define DISPATCH_LOGITS(dtype, ...)                                                        \
  switch (dtype) {   /* check_scoring has seen it */                                       \
    case LFM2_DTYPE_BF16: { typedef __bf16 T; __VA_ARGS__; } break;                        \
    case LFM2_DTYPE_F16: { typedef _Float16 T; __VA_ARGS__; } break;                       \
    case LFM2_DTYPE_F32: { typedef float T; __VA_ARGS__; } break;                          \
  }

// Sixteen bytes of a row.  A row of an odd vocabulary, or one inside a padded matrix, starts at any multiple of the
// element size; the vector type says so and the hardware takes such addresses as they are.
template <typename T> struct RowVec {
  static constexpr int N = 16 / sizeof(T);
  typedef T type __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T))));
};

// The same in every thread of the workgroup.
template <int THREADS> __device__ __forceinline__ float group_max(float v, float* scratch) { return block_max<THREADS / 64>(v, scratch); }
template <int THREADS> __device__ __forceinline__ float group_sum(float v, float* scratch) { return block_sum<THREADS / 64>(v, scratch); }

// ===================================================================================== one row of logits
// Softmax statistics of a row z at temperature T in one pass: m = max z, s = sum e^{(z-m)/T}, u = sum e^{d} d with
// d = (z-m)/T in units of ln 2 (k = log2(e) / T turns differences of logits into base-2 exponents).  A new maximum m'
// moves d by c = (m - m') k: s' = s 2^c and u' = (u + c s) 2^c.
// Limits: -inf logits add nothing; a row of nothing else ends with m = -inf, s = 0.  A NaN or +inf makes s NaN.
struct RowStats { float m, s, u; };
template <bool ENTROPY> __device__ __forceinline__ void merge_stats(RowStats& a, float m, float s, float u, float k) {
  const float mm = fmaxf(a.m, m);
  if (mm == -kInf) { a.s += s; return; }   // both empty (s is 0, or NaN from a NaN row, which has to survive)
  const float ca = (a.m - mm) * k, cb = (m - mm) * k;
  const float fa = __builtin_amdgcn_exp2f(ca), fb = __builtin_amdgcn_exp2f(cb);
  if (ENTROPY) {
    const float ua = a.m == -kInf ? 0.f : (a.u + fmaxf(ca, -1.0e30f) * a.s) * fa;
    const float ub = m == -kInf ? 0.f : (u + fmaxf(cb, -1.0e30f) * s) * fb;
    a.u = ua + ub;
  }
  a.s = a.s * fa + s * fb;
  a.m = mm;
}
template <bool ENTROPY, int N> __device__ __forceinline__ void add_values(RowStats& a, const float* z, float k) {
  float mx = z[0];
#pragma unroll
  for (int i = 1; i < N; ++i) mx = fmaxf(mx, z[i]);
  const float base = mx == -kInf ? 0.f : mx;   // nothing but -inf (or NaN): the exponentials are 0 (or NaN)
  float s = 0.f, u = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float d = (z[i] - base) * k, e = __builtin_amdgcn_exp2f(d);
    s += e;
    if (ENTROPY) u = fmaf(e, fmaxf(d, -1.0e30f), u);   // 0 * -inf has no place in the sum
  }
  merge_stats<ENTROPY>(a, mx, s, u, k);
}

// Statistics of a whole row, the same in every thread: threads keep their own maximum and sums (four 16-byte loads in
// flight each), which are joined once at the end.
template <bool STREAM, typename V> __device__ __forceinline__ V load_row(const V* p) {
  if constexpr (STREAM) return __builtin_nontemporal_load(p);
  else return *p;
}
template <typename T, int THREADS, bool ENTROPY, bool STREAM>
__device__ __forceinline__ RowStats row_stats(const T* __restrict__ row, int64_t V, float k, float* scratch) {
  constexpr int VE = RowVec<T>::N;
  typedef typename RowVec<T>::type vec;
  const int64_t nvec = V / VE;
  RowStats a{-kInf, 0.f, 0.f};
  int64_t i = threadIdx.x;
  for (; i + 3 * THREADS < nvec; i += 4 * THREADS) {
    vec v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = load_row<STREAM>(reinterpret_cast<const vec*>(row + (i + j * THREADS) * VE));
    float z[4 * VE];
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int e = 0; e < VE; ++e) z[j * VE + e] = (float)v[j][e];
    add_values<ENTROPY, 4 * VE>(a, z, k);
  }
  for (; i < nvec; i += THREADS) {
    const vec v = load_row<STREAM>(reinterpret_cast<const vec*>(row + i * VE));
    float z[VE];
#pragma unroll
    for (int e = 0; e < VE; ++e) z[e] = (float)v[e];
    add_values<ENTROPY, VE>(a, z, k);
  }
  if (threadIdx.x < V - nvec * VE) {
    const float z = (float)row[nvec * VE + threadIdx.x];
    add_values<ENTROPY, 1>(a, &z, k);
  }
  // joined: the row's maximum first, then the sums moved to it
  const float m = group_max<THREADS>(a.m, scratch);
  const float c = a.m == -kInf ? 0.f : (a.m - m) * k, f = __builtin_amdgcn_exp2f(c);
  RowStats out{m, 0.f, 0.f};
  if (ENTROPY) out.u = group_sum<THREADS>((a.u + fmaxf(c, -1.0e30f) * a.s) * f, scratch);
  out.s = group_sum<THREADS>(a.s * f, scratch);
  return out;
}

// What the rest of a row's work needs: the log-probability of the target, the entropy, log s and log2 s.
struct RowResult { float logprob, entropy, log_s; };
__device__ __forceinline__ RowResult finish_row(const RowStats& a, float z_target, bool in_range, float temperature) {
  RowResult r;
  r.log_s = logf(a.s);
  if (a.s == 0.f) { r.logprob = -kInf; r.entropy = 0.f; return r; }   // no finite logit: nothing can be drawn
  r.logprob = in_range ? (z_target - a.m) / temperature - r.log_s : __builtin_nanf("");
  r.entropy = r.log_s - (a.u / a.s) * kLn2;
  return r;
}
__device__ __forceinline__ float row_temperature(const float* temperatures, float temperature, int64_t row) {
  const float t = temperatures ? temperatures[row] : temperature;
  return t <= 0.f ? 1.f : t;   // greedy rows are scored by the raw softmax, as the sampler scores them
}

struct LogprobArgs {
  float *logprobs, *entropy, *stats;
  const void* logits;
  const int64_t* targets;
  const float* temperatures;
  int64_t stride, V;
  float temperature;
};

// One workgroup per row; reads the row once.  stats[row] = (max, log s, entropy, 0) for the gradient.  Bound by reading:
// 4096 rows of 65536 bf16 values (537 MB) take 82 us, 6.6 TB/s (a loads-only kernel: 7.0); with entropies the vector unit is
// about as busy as the memory (483 MB: 89 us, 5.4 TB/s).  A call of a few rows is the latency of one (6.5 us).
template <typename T, int THREADS, bool ENTROPY, bool STREAM>
__global__ void __launch_bounds__(THREADS) token_logprobs_kernel(LogprobArgs a) {
  __shared__ float scratch[THREADS / 64];
  const int64_t row = blockIdx.x, target = a.targets[row];
  float* stats = a.stats + 4 * row;
  if (target < 0) {
    if (threadIdx.x == 0) {
      a.logprobs[row] = 0.f;
      if (a.entropy) a.entropy[row] = 0.f;
      stats[0] = stats[1] = stats[2] = stats[3] = 0.f;
    }
    return;
  }
  const T* z = (const T*)a.logits + row * a.stride;
  const float t = row_temperature(a.temperatures, a.temperature, row);
  const bool in_range = target < a.V;
  const float zt = (float)z[in_range ? target : 0];
  const RowStats st = row_stats<T, THREADS, ENTROPY, STREAM>(z, a.V, LFM2_LOG2E / t, scratch);
  if (threadIdx.x == 0) {
    const RowResult r = finish_row(st, zt, in_range, t);
    a.logprobs[row] = r.logprob;
    if (ENTROPY) a.entropy[row] = r.entropy;
    stats[0] = st.m;
    stats[1] = r.log_s;
    stats[2] = ENTROPY ? r.entropy : __builtin_nanf("");
    stats[3] = 0.f;
  }
}

// d/dz_v of g logp(target) + h H = (g ([v = target] - p_v) - h p_v (log p_v + H)) / T for N consecutive elements, the
// first of which is `first`; c holds what is the same along the row.
struct GradRow { float m, k, log2_s, g, h, entropy, inv_t, scale; int64_t target; };   // scale = -g / T
template <typename T, int N, bool ENTROPY>
__device__ __forceinline__ void grad_values(const GradRow& c, const float* z, int64_t first, T* out) {
  const int64_t hot = c.target - first;
  float v[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float d = fmaf(z[i] - c.m, c.k, -c.log2_s);   // log2 p
    const float p = __builtin_amdgcn_exp2f(d);
    if constexpr (ENTROPY) {
      v[i] = -p * fmaf(c.h, fmaf(fmaxf(d, -1.0e30f), kLn2, c.entropy), c.g) * c.inv_t;   // 0 * -inf has no place in the sum
    } else {
      v[i] = p * c.scale;
    }
  }
  if (hot >= 0 && hot < N) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = fmaf(i == hot ? c.g : 0.f, c.inv_t, v[i]);
  }
#pragma unroll
  for (int i = 0; i < N; ++i) out[i] = Elem<T>::store(v[i]);
}
__device__ __forceinline__ GradRow grad_row(float m, float log_s, float entropy, float g, float h, float temperature,
                                            int64_t target, int64_t V) {
  GradRow c;
  c.inv_t = 1.0f / temperature;
  c.k = LFM2_LOG2E / temperature;
  c.m = m;
  c.log2_s = log_s * LFM2_LOG2E;
  c.entropy = entropy;
  c.h = h;
  // a row with a NaN, or a target outside the vocabulary, has no gradient: NaN everywhere (the clamp above would
  // otherwise turn a NaN into a probability of 0)
  c.g = log_s == log_s && target < V ? g : __builtin_nanf("");
  c.target = target;
  if (m == -kInf && log_s == -kInf) { c.g = 0.f; c.h = 0.f; c.m = 0.f; c.log2_s = 0.f; c.entropy = 0.f; }   // no finite logit: no gradient
  c.scale = -c.g * c.inv_t;
  return c;
}

struct BackwardArgs {
  void* grad;
  const void* logits;
  const int64_t* targets;
  const float *stats, *grad_logprobs, *grad_entropy, *temperatures;
  int64_t grad_stride, stride, V;
  float temperature;
};
constexpr int kBackwardVecs = 4;   // 16-byte pieces per thread

// Elementwise given the row's statistics: workgroup (x, row) covers 256 * kBackwardVecs pieces of a row.  Bound by reading
// and writing: 4096 rows of 65536 bf16 values, a tenth of which does not count (1.02 GB), take 189 us, 5.4 TB/s (a copy on
// this card: 4.7).
template <typename T, bool ENTROPY>
__global__ void __launch_bounds__(256) token_logprobs_backward_kernel(BackwardArgs a) {
  constexpr int VE = RowVec<T>::N;
  typedef typename RowVec<T>::type vec;
  const int64_t row = blockIdx.y, target = a.targets[row];
  const int64_t nvec = a.V / VE, first = (int64_t)blockIdx.x * (256 * kBackwardVecs) + threadIdx.x;
  T* out = (T*)a.grad + row * a.grad_stride;
  const bool has_tail = blockIdx.x == 0 && threadIdx.x < a.V - nvec * VE;
  const int64_t tail = nvec * VE + threadIdx.x;
  if (target < 0) {
    vec zero = {};
#pragma unroll
    for (int j = 0; j < kBackwardVecs; ++j)
      if (first + 256 * j < nvec) *reinterpret_cast<vec*>(out + (first + 256 * j) * VE) = zero;
    if (has_tail) out[tail] = Elem<T>::store(0.f);
    return;
  }
  const T* z = (const T*)a.logits + row * a.stride;
  vec v[kBackwardVecs];
#pragma unroll
  for (int j = 0; j < kBackwardVecs; ++j)
    if (first + 256 * j < nvec) v[j] = *reinterpret_cast<const vec*>(z + (first + 256 * j) * VE);
  const float* st = a.stats + 4 * row;
  const GradRow c = grad_row(st[0], st[1], ENTROPY ? st[2] : 0.f, a.grad_logprobs[row], ENTROPY ? a.grad_entropy[row] : 0.f,
                             row_temperature(a.temperatures, a.temperature, row), target, a.V);
#pragma unroll
  for (int j = 0; j < kBackwardVecs; ++j) {
    const int64_t i = first + 256 * j;
    if (i >= nvec) continue;
    float x[VE];
    T y[VE];
#pragma unroll
    for (int e = 0; e < VE; ++e) x[e] = (float)v[j][e];
    grad_values<T, VE, ENTROPY>(c, x, i * VE, y);
    vec w;
#pragma unroll
    for (int e = 0; e < VE; ++e) w[e] = y[e];
    *reinterpret_cast<vec*>(out + i * VE) = w;
  }
  if (has_tail) {
    const float x = (float)z[tail];
    grad_values<T, 1, ENTROPY>(c, &x, tail, out + tail);
  }
}

// ===================================================================================== the loss of a token
struct LossArgs {
  const float *logprobs, *old, *advantages, *ref, *entropy;
  const uint8_t* mask;
  const int64_t* targets;     // or null; a negative target takes its token out, like the mask
  const int32_t* cu;          // int32[S + 1], or null: one sequence of all N tokens
  const int32_t* counts;      // tokens that count, per sequence (per block of kCountBlock tokens without cu); null: all of them
  const int32_t* totals;      // the batch's (tokens, sequences), or null: every workgroup sums the counts
  int64_t N, S, ncounts;
  int per_sequence, aggregate, kl;
  float clip_low, clip_high, dual_clip, kl_coef, entropy_coef;
  double log_low, log_high, log_dual;   // where the ratio is cut, as bounds of the log ratio
};
constexpr int kCountBlock = 4096;

// e^x - 1 - x without the cancellation: the Taylor series up to x^12 / 12! for |x| < 1 (what is left out is below
// 2e-10 there, against a value of at least x^2 / 2 (1 - |x| / 3)), the difference itself beyond (at least 0.36).
__device__ __forceinline__ float exp_excess(float x) {
  if (fabsf(x) < 1.f) {
    float r = 1.f / 479001600.f;
    r = fmaf(r, x, 1.f / 39916800.f);
    r = fmaf(r, x, 1.f / 3628800.f);
    r = fmaf(r, x, 1.f / 362880.f);
    r = fmaf(r, x, 1.f / 40320.f);
    r = fmaf(r, x, 1.f / 5040.f);
    r = fmaf(r, x, 1.f / 720.f);
    r = fmaf(r, x, 1.f / 120.f);
    r = fmaf(r, x, 1.f / 24.f);
    r = fmaf(r, x, 1.f / 6.f);
    r = fmaf(r, x, 0.5f);
    return r * x * x;
  }
  return (expf(x) - 1.f) - x;
}

// One token that counts: the terms of the loss and its derivative with respect to the log-probability, before the weight.
struct TokenTerms { float policy, kl, slope, ratio, excess; bool cut; };
__device__ __forceinline__ TokenTerms token_terms(const LossArgs& a, float logp, float old, float ref, float advantage) {
  TokenTerms t;
  // the log ratio in 64 bits: whether it is beyond the border decides between two values of the gradient
  const double delta = (double)logp - (double)old;
  const float d = (float)delta;
  t.ratio = expf(d);
  t.excess = exp_excess(d);
  t.cut = (advantage > 0.f && delta > a.log_high) || (advantage < 0.f && delta < a.log_low);
  float gain = t.cut ? (advantage > 0.f ? 1.f + a.clip_high : 1.f - a.clip_low) * advantage : t.ratio * advantage;
  if (a.dual_clip > 0.f && advantage < 0.f && delta > a.log_dual) { gain = a.dual_clip * advantage; t.cut = true; }
  t.policy = -gain;
  t.slope = t.cut ? 0.f : -t.ratio * advantage;
  t.kl = 0.f;
  if (a.ref) {
    const float x = (float)((double)ref - (double)logp);
    float derivative;
    if (a.kl == LFM2_KL_K1) { t.kl = -x; derivative = 1.f; }
    else if (a.kl == LFM2_KL_K2) { t.kl = 0.5f * x * x; derivative = -x; }
    else { t.kl = exp_excess(x); derivative = -(t.kl + x); }   // 1 - e^x
    t.slope = fmaf(a.kl_coef, derivative, t.slope);
  }
  return t;
}

__device__ __forceinline__ int64_t clamp_token(int64_t v, int64_t n) { return v < 0 ? 0 : v > n ? n : v; }
// Sequence of token t among the sequences [lo, hi): the last one that starts at or before t.
__device__ __forceinline__ int64_t sequence_of(const int32_t* cu, int64_t lo, int64_t hi, int64_t t) {
  while (hi - lo > 1) {
    const int64_t mid = (lo + hi) >> 1;
    if (cu[mid] <= t) lo = mid; else hi = mid;
  }
  return lo;
}
__device__ __forceinline__ bool token_counts(const LossArgs& a, int64_t t) {
  if (a.cu && (t < a.cu[0] || t >= a.cu[a.S])) return false;   // behind the last sequence
  if (a.mask && !a.mask[t]) return false;
  return !a.targets || a.targets[t] >= 0;
}
// Tokens that count in sequence s.
__device__ __forceinline__ int sequence_count(const LossArgs& a, int64_t s) {
  if (a.counts) return a.counts[s];
  if (!a.cu) return (int)a.N;
  const int64_t n = clamp_token(a.cu[s + 1], a.N) - clamp_token(a.cu[s], a.N);
  return n > 0 ? (int)n : 0;
}
__device__ __forceinline__ int wave_sum_int(int v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
__device__ __forceinline__ double wave_sum_double(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
template <int WAVES> __device__ __forceinline__ int block_sum_int(int v, int* scratch) {
  v = wave_sum_int(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = v;
  __syncthreads();
  int t = 0;
#pragma unroll
  for (int i = 0; i < WAVES; ++i) t += scratch[i];
  return t;
}

// What every weight of the batch is divided by besides its sequence's count: all tokens that count, or the sequences that
// have any.  `first` .. in steps of `step`: one thread's share of the sequences.
struct Totals { int tokens, sequences; };
__device__ __forceinline__ Totals partial_totals(const LossArgs& a, int first, int step) {
  Totals t{0, 0};
  for (int64_t s = first; s < a.ncounts; s += step) {
    const int n = sequence_count(a, s);
    t.tokens += n;
    t.sequences += n > 0;
  }
  return t;
}
template <int WAVES> __device__ __forceinline__ Totals batch_totals(const LossArgs& a, int* scratch) {
  if (a.totals) return Totals{a.totals[0], a.totals[1]};
  Totals t = partial_totals(a, threadIdx.x, 64 * WAVES);
  t.tokens = block_sum_int<WAVES>(t.tokens, scratch);
  t.sequences = block_sum_int<WAVES>(t.sequences, scratch);
  return t;
}
__device__ __forceinline__ float token_weight(const LossArgs& a, const Totals& total, int sequence_tokens) {
  if (a.aggregate == LFM2_MEAN_SUM) return 1.f;
  if (a.aggregate == LFM2_MEAN_SEQUENCES && a.cu) return (float)(1.0 / ((double)sequence_tokens * (double)total.sequences));
  return (float)(1.0 / (double)total.tokens);
}

// Tokens that count, per sequence (per block of kCountBlock tokens without sequences): one workgroup each.  This and the two
// kernels after the next are chains of dependent loads, not of bytes: 16384 tokens of 64 sequences take 5, 11 and 4 us.
__global__ void __launch_bounds__(256) policy_count_kernel(int32_t* counts, LossArgs a) {
  __shared__ int scratch[4];
  const int64_t s = blockIdx.x;
  const int64_t begin = a.cu ? clamp_token(a.cu[s], a.N) : s * kCountBlock;
  const int64_t end = a.cu ? clamp_token(a.cu[s + 1], a.N) : clamp_token((s + 1) * kCountBlock, a.N);
  int n = 0;
  for (int64_t t = begin + threadIdx.x; t < end; t += 256) n += (!a.mask || a.mask[t]) && (!a.targets || a.targets[t] >= 0);
  n = block_sum_int<4>(n, scratch);
  if (threadIdx.x == 0) counts[s] = n;
}

// Their totals, where there are too many counts for every workgroup to sum.
__global__ void __launch_bounds__(1024) policy_totals_kernel(int32_t* totals, LossArgs a) {
  __shared__ int scratch[16];
  const Totals t = batch_totals<16>(a, scratch);
  if (threadIdx.x == 0) { totals[0] = t.tokens; totals[1] = t.sequences; }
}

// The per-token part: gradients out, sums of the terms per workgroup.  Sums are kept in 64 bits and joined in a fixed
// order, so the result does not depend on how workgroups are scheduled.
constexpr int kLossTerms = 6;          // policy, kl, entropy, cut, ratio, excess
// Tokens per workgroup of 256 threads, each of which sweeps all sequences.  With 512 a loss of 16384 tokens (64 sequences)
// takes 12 us instead of 14, and one of 2^20 tokens (1024 sequences) 28 instead of 21.
constexpr int kLossTokens = 1024;
// What a token brings, read before anything is known about its weight (a token that does not count is read and not used).
struct TokenInputs {
  float logprob, old, ref, entropy, advantage;
  bool counts;
  __device__ __forceinline__ void read(const LossArgs& a, int64_t t, int64_t end) {
    counts = t < end;
    if (!counts) return;
    logprob = a.logprobs[t];
    old = a.old[t];
    if (a.ref) ref = a.ref[t];
    if (a.entropy) entropy = a.entropy[t];
    if (!a.per_sequence) advantage = a.advantages[t];
    counts = (!a.mask || a.mask[t]) && (!a.targets || a.targets[t] >= 0);
  }
};
struct TermSums {
  double v[kLossTerms] = {};
  // a token of sequence s with weight w: returns its gradient
  __device__ __forceinline__ float add(const LossArgs& a, const TokenInputs& x, int64_t s, float w) {
    const TokenTerms term = token_terms(a, x.logprob, x.old, x.ref, a.per_sequence ? a.advantages[s] : x.advantage);
    v[0] += (double)w * term.policy;
    v[1] += (double)w * term.kl;
    if (a.entropy) v[2] += (double)w * x.entropy;
    v[3] += term.cut;
    v[4] += term.ratio;
    v[5] += term.excess;
    return w * term.slope;
  }
  // over the workgroup, to out[kLossTerms] (valid after the next barrier)
  template <int WAVES> __device__ __forceinline__ void join(double (*scratch)[kLossTerms], double* out) const {
#pragma unroll
    for (int i = 0; i < kLossTerms; ++i) {
      const double x = wave_sum_double(v[i]);
      if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6][i] = x;
    }
    __syncthreads();
    if (threadIdx.x < kLossTerms) {
      double x = 0.0;
#pragma unroll
      for (int i = 0; i < WAVES; ++i) x += scratch[i][threadIdx.x];
      out[threadIdx.x] = x;
    }
  }
};
// loss, then (policy, kl, entropy, share cut, mean ratio, mean of r - 1 - log r, tokens) from the summed terms.
__device__ __forceinline__ void store_loss(const LossArgs& a, const double* sum, int tokens, float* loss, float* stats) {
  const double n = tokens > 0 ? tokens : 1;
  *loss = (float)(sum[0] + (double)a.kl_coef * sum[1] - (double)a.entropy_coef * sum[2]);
  stats[0] = (float)sum[0];
  stats[1] = (float)sum[1];
  stats[2] = (float)sum[2];
  stats[3] = (float)(sum[3] / n);
  stats[4] = (float)(sum[4] / n);
  stats[5] = (float)(sum[5] / n);
  stats[6] = (float)tokens;
}

__global__ void __launch_bounds__(256)
policy_tokens_kernel(LossArgs a, float* grad, float* grad_entropy, double* partials, int* tokens) {
  __shared__ i32x4 counts[4];
  __shared__ double scratch[4][kLossTerms], out[kLossTerms];
  constexpr int PER = kLossTokens / 256;
  const int64_t begin = (int64_t)blockIdx.x * kLossTokens, end = clamp_token(begin + kLossTokens, a.N);
  TokenInputs inputs[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) inputs[i].read(a, begin + threadIdx.x + 256 * i, end);
  const int64_t cu_first = a.cu ? a.cu[0] : 0, cu_last = a.cu ? a.cu[a.S] : a.N;
  Totals total;
  int64_t s_first = 0, s_last = a.S - 1;   // sequences that this range's tokens may belong to
  if (a.totals) {
    total = Totals{a.totals[0], a.totals[1]};
  } else {
    // one sweep over the sequences: the totals, and how many start at or before this range's first and last token
    i32x4 n = {0, 0, 0, 0};
    for (int64_t s = threadIdx.x; s < a.ncounts; s += 256) {
      const int here = sequence_count(a, s);
      n[0] += here;
      n[1] += here > 0;
      if (a.cu) {
        n[2] += a.cu[s] <= begin;
        n[3] += a.cu[s] < end;
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) n[i] = wave_sum_int(n[i]);
    if ((threadIdx.x & 63) == 0) counts[threadIdx.x >> 6] = n;
    __syncthreads();
    n = (counts[0] + counts[1]) + (counts[2] + counts[3]);
    total = Totals{n[0], n[1]};
    if (a.cu) {
      s_first = n[2] > 0 ? n[2] - 1 : 0;
      s_last = n[3] > 0 ? n[3] - 1 : 0;
    }
  }
  TermSums sums;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int64_t t = begin + threadIdx.x + 256 * i;
    if (t >= end) continue;
    float g = 0.f, gh = 0.f;
    if (inputs[i].counts && t >= cu_first && t < cu_last) {   // not behind the last sequence
      const int64_t s = a.cu ? sequence_of(a.cu, s_first, s_last + 1, t) : 0;
      const float w = token_weight(a, total, a.aggregate == LFM2_MEAN_SEQUENCES && a.cu ? sequence_count(a, s) : 0);
      g = sums.add(a, inputs[i], s, w);
      gh = -a.entropy_coef * w;
    }
    if (grad) grad[t] = g;
    if (grad_entropy) grad_entropy[t] = gh;
  }
  sums.join<4>(scratch, out);
  __syncthreads();
  if (threadIdx.x < kLossTerms) partials[(int64_t)blockIdx.x * kLossTerms + threadIdx.x] = out[threadIdx.x];
  if (!a.totals && blockIdx.x == 0 && threadIdx.x == 0) *tokens = total.tokens;   // (the totals are there already)
}
__global__ void __launch_bounds__(256)
policy_finish_kernel(LossArgs a, const double* partials, const int* tokens, int64_t blocks, float* loss, float* stats) {
  __shared__ double sums[4][kLossTerms], out[kLossTerms];
#pragma unroll
  for (int i = 0; i < kLossTerms; ++i) {
    double v = 0.0;
    for (int64_t b = threadIdx.x; b < blocks; b += 256) v += partials[b * kLossTerms + i];
    v = wave_sum_double(v);
    if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6][i] = v;
  }
  __syncthreads();
  if (threadIdx.x < kLossTerms) out[threadIdx.x] = (sums[0][threadIdx.x] + sums[1][threadIdx.x]) + (sums[2][threadIdx.x] + sums[3][threadIdx.x]);
  __syncthreads();
  if (threadIdx.x == 0) store_loss(a, out, *tokens, loss, stats);
}
// Few tokens and sequences: one workgroup counts, weighs and sums everything; the bounds and counts are in LDS.  One launch
// instead of three: 1024 tokens of 16 sequences 8.6 us against 14.2, 4096 tokens 13.1 against 13.8 (of 2048 sequences 13.2
// against 20.5); beyond that the one workgroup is the longer way.
constexpr int kSingleTokens = 4096, kSingleSequences = 2048;
__global__ void __launch_bounds__(1024) policy_single_kernel(LossArgs a, float* grad, float* grad_entropy, float* loss, float* stats) {
  constexpr int PER = kSingleTokens / 1024;
  __shared__ int bounds[kSingleSequences + 1], counts[kSingleSequences], iscratch[16];
  __shared__ double scratch[16][kLossTerms], out[kLossTerms];
  const int tid = threadIdx.x, S = a.cu ? (int)a.S : 1;
  for (int s = tid; s <= S; s += 1024) {
    bounds[s] = a.cu ? (int)clamp_token(a.cu[s], a.N) : s ? (int)a.N : 0;
    if (s < S) counts[s] = 0;
  }
  TokenInputs inputs[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) inputs[i].read(a, tid + 1024 * i, a.N);
  __syncthreads();
  int sequence[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int t = tid + 1024 * i;
    sequence[i] = 0;
    if (!inputs[i].counts) continue;
    if (t < bounds[0] || t >= bounds[S]) { inputs[i].counts = false; continue; }   // behind the last sequence
    int lo = 0, hi = S;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (bounds[mid] <= t) lo = mid; else hi = mid;
    }
    sequence[i] = lo;
    atomicAdd(&counts[lo], 1);
  }
  __syncthreads();
  Totals total{0, 0};
  for (int s = tid; s < S; s += 1024) { total.tokens += counts[s]; total.sequences += counts[s] > 0; }
  total.tokens = block_sum_int<16>(total.tokens, iscratch);
  total.sequences = block_sum_int<16>(total.sequences, iscratch);
  TermSums sums;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int64_t t = tid + 1024 * i;
    if (t >= a.N) continue;
    float g = 0.f, gh = 0.f;
    if (inputs[i].counts) {
      const float w = token_weight(a, total, counts[sequence[i]]);
      g = sums.add(a, inputs[i], sequence[i], w);
      gh = -a.entropy_coef * w;
    }
    if (grad) grad[t] = g;
    if (grad_entropy) grad_entropy[t] = gh;
  }
  sums.join<16>(scratch, out);
  __syncthreads();
  if (tid == 0) store_loss(a, out, total.tokens, loss, stats);
}

// ===================================================================================== loss and gradient from the logits
struct GradientArgs {
  LossArgs loss;              // loss.logprobs and loss.entropy are written here, row by row
  float *logprobs, *entropy;
  void* grad;
  const void* logits;
  const float* temperatures;
  int64_t grad_stride, stride, V;
  float temperature, grad_scale;
};

// Keeps the compiler from holding a row's values unpacked (twice the registers of 16-bit ones) from one sweep to the next.
template <typename V, int N> __device__ __forceinline__ void forget_unpacked(V (&held)[N]) {
#pragma unroll
  for (int j = 0; j < N; ++j) {
    i32x4 raw = __builtin_bit_cast(i32x4, held[j]);
    asm volatile("" : "+v"(raw));
    held[j] = __builtin_bit_cast(V, raw);
  }
}

// One workgroup per row: statistics, the token's loss slope, and the row's gradient.  VECS > 0: the row is read once and
// waits in registers (16 bytes each) while its statistics are joined; 0: a row too long for that is read twice.  Bound by
// reading and writing: 8958 rows of 65536 bf16 values, three tenths of which do not count (2.0 GB), take 381 us, 5.2 TB/s.
// Whole calls (three to four launches), 4096 rows of 8192 / 32768 / 65536 values: 46 / 107 / 219 us, read twice 54 / 145 /
// 270.  256 threads hold rows of up to 16 KiB: with 512, 4096 rows of 8192 values take 57.  1024 threads for the longest
// rows that are held leave room for one row per CU at a time: 489 us for the 8958 rows, 406 with 512.
template <typename T, int THREADS, int VECS, bool ENTROPY>
__global__ void __launch_bounds__(THREADS) policy_gradient_kernel(GradientArgs a) {
  constexpr int VE = RowVec<T>::N;
  typedef typename RowVec<T>::type vec;
  __shared__ float scratch[THREADS / 64];
  __shared__ int iscratch[THREADS / 64];
  const int64_t row = blockIdx.x, nvec = a.V / VE, tail = nvec * VE + threadIdx.x;
  const bool has_tail = tail < a.V;
  T* out = (T*)a.grad + row * a.grad_stride;
  if (!token_counts(a.loss, row)) {
    const vec zero = {};
    for (int64_t i = threadIdx.x; i < nvec; i += THREADS) *reinterpret_cast<vec*>(out + i * VE) = zero;
    if (has_tail) out[tail] = Elem<T>::store(0.f);
    if (threadIdx.x == 0) {
      a.logprobs[row] = 0.f;
      if (a.entropy) a.entropy[row] = 0.f;
    }
    return;
  }
  const int64_t target = a.loss.targets[row];
  const T* z = (const T*)a.logits + row * a.stride;
  vec held[VECS > 0 ? VECS : 1];
  if constexpr (VECS > 0) {
#pragma unroll
    for (int j = 0; j < VECS; ++j) {
      const int64_t i = threadIdx.x + (int64_t)j * THREADS;
      if (i < nvec) held[j] = __builtin_nontemporal_load(reinterpret_cast<const vec*>(z + i * VE));
    }
  }
  const float t = row_temperature(a.temperatures, a.temperature, row), k = LFM2_LOG2E / t;
  const bool in_range = target < a.V;
  const float zt = (float)z[in_range ? target : 0];
  const float zl = has_tail ? (float)z[tail] : -kInf;
  // while the row is on its way: the token's weight
  const Totals total = batch_totals<THREADS / 64>(a.loss, iscratch);
  const int64_t s = a.loss.cu ? sequence_of(a.loss.cu, 0, a.loss.S, row) : 0;
  const float w = token_weight(a.loss, total, a.loss.aggregate == LFM2_MEAN_SEQUENCES && a.loss.cu ? sequence_count(a.loss, s) : 0);
  const float old = a.loss.old[row], ref = a.loss.ref ? a.loss.ref[row] : 0.f, advantage = a.loss.advantages[a.loss.per_sequence ? s : row];
  RowStats st;
  if constexpr (VECS > 0) {
    float mx = zl;
#pragma unroll
    for (int j = 0; j < VECS; ++j)
      if (threadIdx.x + (int64_t)j * THREADS < nvec) {
#pragma unroll
        for (int e = 0; e < VE; ++e) mx = fmaxf(mx, (float)held[j][e]);
      }
    forget_unpacked(held);
    st.m = group_max<THREADS>(mx, scratch);
    const float base = st.m == -kInf ? 0.f : st.m;   // nothing but -inf (or NaN): the exponentials are 0 (or NaN)
    float sum = 0.f, u = 0.f;
    auto add = [&](float x) {
      const float d = (x - base) * k, e = __builtin_amdgcn_exp2f(d);
      sum += e;
      if (ENTROPY) u = fmaf(e, fmaxf(d, -1.0e30f), u);
    };
#pragma unroll
    for (int j = 0; j < VECS; ++j)
      if (threadIdx.x + (int64_t)j * THREADS < nvec) {
#pragma unroll
        for (int e = 0; e < VE; ++e) add((float)held[j][e]);
      }
    if (has_tail) add(zl);
    st.u = ENTROPY ? group_sum<THREADS>(u, scratch) : 0.f;
    st.s = group_sum<THREADS>(sum, scratch);
  } else {
    st = row_stats<T, THREADS, ENTROPY, false>(z, a.V, k, scratch);
  }
  const RowResult r = finish_row(st, zt, in_range, t);
  const TokenTerms term = token_terms(a.loss, r.logprob, old, ref, advantage);
  if (threadIdx.x == 0) {
    a.logprobs[row] = r.logprob;
    if (ENTROPY) a.entropy[row] = r.entropy;
  }
  const GradRow c = grad_row(st.m, r.log_s, ENTROPY ? r.entropy : 0.f, a.grad_scale * w * term.slope,
                             ENTROPY ? -a.grad_scale * a.loss.entropy_coef * w : 0.f, t, target, a.V);
  auto store = [&](int64_t i, const vec v) {
    float x[VE];
    T y[VE];
#pragma unroll
    for (int e = 0; e < VE; ++e) x[e] = (float)v[e];
    grad_values<T, VE, ENTROPY>(c, x, i * VE, y);
    vec o;
#pragma unroll
    for (int e = 0; e < VE; ++e) o[e] = y[e];
    *reinterpret_cast<vec*>(out + i * VE) = o;
  };
  if constexpr (VECS > 0) {
    forget_unpacked(held);
#pragma unroll
    for (int j = 0; j < VECS; ++j) {
      const int64_t i = threadIdx.x + (int64_t)j * THREADS;
      if (i < nvec) store(i, held[j]);
    }
  } else {
    for (int64_t i = threadIdx.x; i < nvec; i += THREADS) store(i, *reinterpret_cast<const vec*>(z + i * VE));
  }
  if (has_tail) grad_values<T, 1, ENTROPY>(c, &zl, tail, out + tail);
}

// ===================================================================================== host side
// The type, and the number that divides the logits: log2(e) / temperature has to be a finite float.
int check_scoring(const char* name, const float* temperatures, float temperature, int dtype) {
  LFM2_REQUIRE(temperatures || (temperature >= __FLT_MIN__ && temperature <= __FLT_MAX__), "%s: temperature must be a positive normal number", name);
  if (dtype != LFM2_DTYPE_BF16 && dtype != LFM2_DTYPE_F16 && dtype != LFM2_DTYPE_F32)
    LFM2_FAIL(LFM2_ERR_UNSUPPORTED, "%s: dtype %d is not bf16/f16/f32", name, dtype);
  return LFM2_OK;
}
bool finite(float v) { return v >= -__FLT_MAX__ && v <= __FLT_MAX__; }
constexpr int64_t kMostGroups = 1 << 22;   // workgroups of a launch: the threads of a grid are counted in 32 bits
int check_logits(const char* name, int64_t N, int64_t V, int64_t stride) {
  LFM2_REQUIRE(N > 0 && V > 0, "%s: empty logits", name);
  LFM2_REQUIRE(N <= 0x7fffffff && V <= 0x7fffffff, "%s: at most 2^31 - 1 rows and columns", name);
  LFM2_REQUIRE(N <= kMostGroups, "%s: more than 2^22 rows", name);
  LFM2_REQUIRE(stride >= V, "%s: rows overlap", name);
  return LFM2_OK;
}

int fill_loss(const char* name, LossArgs* a, const float* logprobs, const float* old, const float* advantages, const float* ref,
              const float* entropy, const uint8_t* mask, const int64_t* targets, const int32_t* cu, int64_t N, int64_t S,
              int per_sequence, int aggregate, int kl, float clip_low, float clip_high, float dual_clip, float kl_coef,
              float entropy_coef) {
  LFM2_REQUIRE(N > 0 && N <= 0x7fffffff, "%s: 1 to 2^31 - 1 tokens", name);
  LFM2_REQUIRE(!cu || (S > 0 && S <= 0x7fffffff), "%s: cu_seqlens needs at least one sequence", name);
  LFM2_REQUIRE(!cu || S <= kMostGroups, "%s: more than 2^22 sequences", name);
  LFM2_REQUIRE(old && advantages, "%s: old log-probabilities and advantages are required", name);
  LFM2_REQUIRE(aggregate >= LFM2_MEAN_TOKENS && aggregate <= LFM2_MEAN_SUM, "%s: unknown aggregate %d", name, aggregate);
  LFM2_REQUIRE(kl >= LFM2_KL_K1 && kl <= LFM2_KL_K3, "%s: unknown KL estimator %d", name, kl);
  LFM2_REQUIRE(clip_low >= 0.f && clip_low < 1.f && clip_high >= 0.f && clip_high <= 3.0e38f, "%s: clip range outside [0, 1) x [0, inf)", name);
  LFM2_REQUIRE(dual_clip == 0.f || (dual_clip > 1.f && finite(dual_clip)), "%s: dual_clip is 0 (off) or above 1", name);
  LFM2_REQUIRE(finite(kl_coef) && finite(entropy_coef), "%s: coefficients must be finite", name);
  *a = LossArgs{logprobs, old, advantages, ref, entropy, mask, targets, cu, nullptr, nullptr, N, cu ? S : 1, cu ? S : 1, per_sequence, aggregate, kl,
                clip_low, clip_high, dual_clip, kl_coef, entropy_coef, __builtin_log1p(-(double)clip_low),
                __builtin_log1p((double)clip_high), dual_clip > 0.f ? __builtin_log((double)dual_clip) : 0.0};
  return LFM2_OK;
}

// Logits of this size or more leave the last-level cache (256 MB) before anybody reads them again: the scoring pass then
// loads them with the non-temporal hint; smaller ones stay there for the gradient.  Scoring and gradient of 134 / 210 MB: 68 /
// 117 us with the hint, 66 / 109 without; of 288 / 537 MB: 158 / 276 with it, 171 / 300 without.
constexpr int64_t kStreamBytes = 224ll << 20;

int64_t count_slots(int64_t N, int64_t S, bool cu) { return cu ? S : (N + kCountBlock - 1) / kCountBlock; }
int64_t loss_blocks(int64_t N) { return (N + kLossTokens - 1) / kLossTokens; }
// Workspace: the partial sums (64 bits, first for their alignment), the token count, the per-sequence counts.
int64_t workspace_words(int64_t N, int64_t S, bool cu) { return 2 * loss_blocks(N) * kLossTerms + 2 + count_slots(N, S, cu); }
struct LossWorkspace { double* partials; int *tokens, *counts; };   // tokens: two of them where they are the totals
LossWorkspace split_workspace(float* ws, int64_t N) {
  double* partials = reinterpret_cast<double*>(ws);
  int* tokens = reinterpret_cast<int*>(partials + loss_blocks(N) * kLossTerms);
  return LossWorkspace{partials, tokens, tokens + 2};
}
// Up to so many counts every workgroup sums them itself; more are summed once, in a launch of their own (and a token's sequence
// is looked for among all of them).  A workgroup of the loss has 1024 tokens, one of policy_gradient a row.  A loss of 2^18
// masked tokens in 2048 / 4096 / 8192 sequences takes 18.7 / 22.9 / 31 us without that launch and 21.6 / 23.6 / 27 with it, of
// 2^20 in 65536 146 and 78; policy_gradient of 8192 rows of 2048 values in 512 / 1024 / 4096 sequences 51 / 55 / 73 and 49 / 50 /
// 57, of 32768 rows of 512 in 32768 505 and 153.
constexpr int64_t kLossSweep = 4096, kRowSweep = 512;
void launch_counts(LossArgs* a, int64_t sweep, const LossWorkspace& ws, hipStream_t s) {
  if (a->mask || a->targets) {   // otherwise every token counts: the bounds say how many
    a->ncounts = count_slots(a->N, a->S, a->cu != nullptr);
    hipLaunchKernelGGL(policy_count_kernel, dim3((unsigned)a->ncounts), dim3(256), 0, s, ws.counts, *a);
    a->counts = ws.counts;
  }
  if (a->ncounts > sweep) {
    hipLaunchKernelGGL(policy_totals_kernel, dim3(1), dim3(1024), 0, s, ws.tokens, *a);
    a->totals = ws.tokens;
  }
}
bool single_workgroup(const LossArgs& a) { return a.N <= kSingleTokens && a.S <= kSingleSequences; }
void launch_loss(const LossArgs& a, float* grad, float* grad_entropy, const LossWorkspace& ws, float* loss, float* stats, hipStream_t s) {
  if (single_workgroup(a)) {
    hipLaunchKernelGGL(policy_single_kernel, dim3(1), dim3(1024), 0, s, a, grad, grad_entropy, loss, stats);
    return;
  }
  const int64_t blocks = loss_blocks(a.N);
  hipLaunchKernelGGL(policy_tokens_kernel, dim3((unsigned)blocks), dim3(256), 0, s, a, grad, grad_entropy, ws.partials, ws.tokens);
  hipLaunchKernelGGL(policy_finish_kernel, dim3(1), dim3(256), 0, s, a, (const double*)ws.partials, (const int*)ws.tokens, blocks, loss, stats);
}

}  // namespace

extern "C" {

int lfm2_token_logprobs(float* logprobs, float* entropy, float* stats, const void* logits, int64_t row_stride,
                        const int64_t* targets, const float* temperatures, float temperature, int64_t N, int64_t V, int dtype,
                        void* stream) {
  const int bad = check_logits("token_logprobs", N, V, row_stride);
  if (bad) return bad;
  LFM2_REQUIRE(logprobs && stats && logits && targets, "token_logprobs: null argument");
  if (int e = check_scoring("token_logprobs", temperatures, temperature, dtype)) return e;
  const LogprobArgs a{logprobs, entropy, stats, logits, targets, temperatures, row_stride, V, temperature};
  hipStream_t s = (hipStream_t)stream;
#define LOGPROBS_(THREADS, ENTROPY, STREAM) \
  hipLaunchKernelGGL((token_logprobs_kernel<T, THREADS, ENTROPY, STREAM>), dim3((unsigned)N), dim3(THREADS), 0, s, a)
  DISPATCH_LOGITS(dtype,
    // 4096 rows of 4096 / 8192 values: 7.7 / 14.5 us with 128 threads, 11.7 / 16.2 with 512; of 65536: 85 and 83; 64 rows of
    // 16384: 5.2 and 4.2
    const bool stream_once = N * V * (int64_t)sizeof(T) >= kStreamBytes;   // what is read, however far apart the rows are
    if (V <= 8192) {
      if (stream_once) { if (entropy) LOGPROBS_(128, true, true); else LOGPROBS_(128, false, true); }
      else { if (entropy) LOGPROBS_(128, true, false); else LOGPROBS_(128, false, false); }
    } else {
      if (stream_once) { if (entropy) LOGPROBS_(512, true, true); else LOGPROBS_(512, false, true); }
      else { if (entropy) LOGPROBS_(512, true, false); else LOGPROBS_(512, false, false); }
    })
#undef LOGPROBS_
  LFM2_LAUNCH_CHECK();
}

int lfm2_token_logprobs_backward(void* grad, int64_t grad_stride, const void* logits, int64_t row_stride, const int64_t* targets,
                                 const float* stats, const float* grad_logprobs, const float* grad_entropy,
                                 const float* temperatures, float temperature, int64_t N, int64_t V, int dtype, void* stream) {
  int bad = check_logits("token_logprobs_backward", N, V, row_stride);
  if (!bad) bad = check_logits("token_logprobs_backward", N, V, grad_stride);
  if (bad) return bad;
  LFM2_REQUIRE(grad && stats && logits && targets && grad_logprobs, "token_logprobs_backward: null argument");
  if (int e = check_scoring("token_logprobs_backward", temperatures, temperature, dtype)) return e;
  const BackwardArgs a{grad, logits, targets, stats, grad_logprobs, grad_entropy, temperatures, grad_stride, row_stride, V, temperature};
  hipStream_t s = (hipStream_t)stream;
  // a grid's y holds 65535 rows
  DISPATCH_LOGITS(dtype,
    const int64_t pieces = V / RowVec<T>::N;
    const unsigned x = (unsigned)(pieces ? (pieces + 256 * kBackwardVecs - 1) / (256 * kBackwardVecs) : 1);
    for (int64_t row = 0; row < N; row += 65535) {
      BackwardArgs part = a;
      const int64_t rows = N - row < 65535 ? N - row : 65535;
      part.grad = (T*)a.grad + row * grad_stride;
      part.logits = (const T*)a.logits + row * row_stride;
      part.targets = targets + row; part.stats = stats + 4 * row; part.grad_logprobs = grad_logprobs + row;
      part.grad_entropy = grad_entropy ? grad_entropy + row : nullptr;
      part.temperatures = temperatures ? temperatures + row : nullptr;
      if (grad_entropy) hipLaunchKernelGGL((token_logprobs_backward_kernel<T, true>), dim3(x, (unsigned)rows), dim3(256), 0, s, part);
      else hipLaunchKernelGGL((token_logprobs_backward_kernel<T, false>), dim3(x, (unsigned)rows), dim3(256), 0, s, part);
    })
  LFM2_LAUNCH_CHECK();
}

int64_t lfm2_policy_workspace(int64_t N, int64_t S, int has_cu) {
  return N <= 0 ? 0 : workspace_words(N, S, has_cu != 0);
}

int lfm2_policy_loss(float* loss, float* stats, float* grad_logprobs, float* grad_entropy, const float* logprobs, const float* old_logprobs,
                     const float* advantages, const float* ref_logprobs, const float* entropy, const uint8_t* mask,
                     const int32_t* cu_seqlens, float* workspace, int64_t N, int64_t S, int per_sequence, int aggregate, int kl,
                     float clip_low, float clip_high, float dual_clip, float kl_coef, float entropy_coef, void* stream) {
  LossArgs a;
  const int bad = fill_loss("policy_loss", &a, logprobs, old_logprobs, advantages, ref_logprobs, entropy, mask, nullptr, cu_seqlens, N, S,
                            per_sequence, aggregate, kl, clip_low, clip_high, dual_clip, kl_coef, entropy_coef);
  if (bad) return bad;
  LFM2_REQUIRE(loss && stats && logprobs && workspace, "policy_loss: null argument");
  hipStream_t s = (hipStream_t)stream;
  const LossWorkspace ws = split_workspace(workspace, N);
  if (!single_workgroup(a)) launch_counts(&a, kLossSweep, ws, s);
  launch_loss(a, grad_logprobs, grad_entropy, ws, loss, stats, s);
  LFM2_LAUNCH_CHECK();
}

int lfm2_policy_gradient(float* loss, float* stats, float* logprobs, float* entropy, void* grad, int64_t grad_stride, const void* logits,
                         int64_t row_stride, const int64_t* targets, const float* old_logprobs, const float* advantages,
                         const float* ref_logprobs, const uint8_t* mask, const int32_t* cu_seqlens, const float* temperatures,
                         float temperature, float* workspace, int64_t N, int64_t V, int64_t S, int per_sequence, int aggregate,
                         int kl, float clip_low, float clip_high, float dual_clip, float kl_coef, float entropy_coef,
                         float grad_scale, int dtype, void* stream) {
  int bad = check_logits("policy_gradient", N, V, row_stride);
  if (!bad) bad = check_logits("policy_gradient", N, V, grad_stride);
  if (bad) return bad;
  GradientArgs g;
  bad = fill_loss("policy_gradient", &g.loss, logprobs, old_logprobs, advantages, ref_logprobs, entropy, mask, targets, cu_seqlens, N, S,
                  per_sequence, aggregate, kl, clip_low, clip_high, dual_clip, kl_coef, entropy_coef);
  if (bad) return bad;
  LFM2_REQUIRE(loss && stats && logprobs && grad && logits && targets && workspace, "policy_gradient: null argument");
  LFM2_REQUIRE(entropy_coef == 0.f || entropy, "policy_gradient: an entropy term needs the entropy output");
  LFM2_REQUIRE(finite(grad_scale), "policy_gradient: grad_scale must be finite");
  if (int e = check_scoring("policy_gradient", temperatures, temperature, dtype)) return e;
  g.logprobs = logprobs; g.entropy = entropy; g.grad = grad; g.logits = logits; g.temperatures = temperatures;
  g.grad_stride = grad_stride; g.stride = row_stride; g.V = V; g.temperature = temperature; g.grad_scale = grad_scale;
  hipStream_t s = (hipStream_t)stream;
  const LossWorkspace ws = split_workspace(workspace, N);
  launch_counts(&g.loss, kRowSweep, ws, s);
#define GRADIENT_(THREADS, VECS)                                                                                                  \
  do {                                                                                                                            \
    if (entropy) hipLaunchKernelGGL((policy_gradient_kernel<T, THREADS, VECS, true>), dim3((unsigned)N), dim3(THREADS), 0, s, g);  \
    else hipLaunchKernelGGL((policy_gradient_kernel<T, THREADS, VECS, false>), dim3((unsigned)N), dim3(THREADS), 0, s, g);         \
  } while (0)
  DISPATCH_LOGITS(dtype,
    const int64_t pieces = V / RowVec<T>::N;
    if (pieces <= 256 * 4) GRADIENT_(256, 4);
    else if (pieces <= 512 * 8) GRADIENT_(512, 8);
    else if (pieces <= 512 * 16) GRADIENT_(512, 16);
    else GRADIENT_(512, 0);)
#undef GRADIENT_
  launch_loss(g.loss, nullptr, nullptr, ws, loss, stats, s);
  LFM2_LAUNCH_CHECK();
}

}  // extern "C"
