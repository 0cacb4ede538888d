// Operators on token probabilities for sm_100a: what follows the head's logits in scoring, policy-gradient training and
// distillation.  A row of logits z (bf16, fp16 or fp32, V of them) is a token's:
//
//   u = cap * tanh(z / cap) (or z),   x = u / tau,   p = softmax(x),   log p_j = x_j - lse,   lse = log sum exp x
//
//   scores    log p_t of the given token t, H = -sum p log p, and the K largest z (ties: the lowest index) with their log p
//   policy    L = -min(r A, clip(r) A) + beta (e^d - d - 1) - c H,   r = exp(log p_t - old),  d = ref - log p_t  (without old: -A log p_t)
//             dL/dx_j = g (1[j = t] - p_j) + c p_j (log p_j + H),    g = dL/dlog p_t
//   distill   q over K tokens, from a teacher:  L = (1 - w) tau^2 KL + w CE,  CE at tau = 1,  KL = sum_k q_k (log q_k - log p_k)
//             dKL/dx_j = p_j - q_j;  with all other tokens as one more outcome, q_r = 1 - sum q and p_r = sum of their p,
//             KL += q_r (log q_r - log p_r)  and  dKL/dx_j = p_j (1 - q_r / p_r) for each of them
//
// Sums are in fp32, in base 2 relative to a row's largest logit m: e_j = 2^((u_j - m) log2(e) / tau), so that no difference of two
// large numbers is rounded; the exponential is the hardware's (2^-22).  Rows that are left out (a target outside the vocabulary, a
// mask of zero) are not read: their outputs and gradients are zero.  A row without a finite logit has no distribution and reads as
// NaN, as does one with a NaN or with +inf (which under a cap is a token at the cap).  Compiled without fast math: logarithms and divisions
// of a row are the rounded ones.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>
#include <type_traits>

#include "ptx.cuh"

// Arguments of the entry points, 8 bytes each; strides in elements, rows contiguous; type 0 bf16, 1 fp16, 2 fp32.
struct RowArgs {
  const void* z;
  void* out;                              // gradient; null: none
  const int64_t* targets;                 // null: none
  const float* mask;                      // rows count where it is above zero; null: all
  float *loss, *logprob, *entropy, *lse;
  int64_t* top_ids;
  float* top_logprob;
  const float *adv, *old, *ref;
  const int64_t* ids;
  const float* teacher;
  int64_t type, ldz, ldo, T, V, K, ignore, bucket;
  double tau, cap, scale, clip_low, clip_high, kl, bonus, ce;
  cudaStream_t stream;
};

struct GradArgs {
  const void* z;
  void* out;
  const int64_t* targets;
  const float *mask, *lse, *entropy, *dlogprob, *dentropy, *dtop;
  const int64_t* top_ids;
  int64_t type, ldz, ldo, T, V, K, ignore;
  double tau, cap, scale;
  cudaStream_t stream;
};

namespace {

typedef __nv_bfloat16 bf16;
constexpr int MOST_TOP = 128;            // tokens of a teacher, alternatives of a row
constexpr float LN2 = 0.6931471805599453f, LOG2E = 1.4426950408889634f;

enum Op { SCORES, POLICY, DISTILL };

struct Row {
  const void* z;
  void* out;
  const int64_t* targets;
  const float* mask;
  float *loss, *logprob, *entropy, *lse;
  int64_t* top_ids;
  float* top_logprob;
  const float *adv, *old, *ref;
  const int64_t* ids;
  const float* teacher;
  long ldz, ldo, ignore;
  int T, V, K, bucket;
  float inv_tau, tau, c, cap, inv_cap, scale, clip_low, clip_high, kl, bonus, ce;
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max_nan(float a, float b) {      // a NaN stays one
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
__device__ __forceinline__ float to_float(bf16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(float v) { return v; }
template <typename E>
__device__ __forceinline__ E from_float(float v);
template <>
__device__ __forceinline__ bf16 from_float<bf16>(float v) { return __float2bfloat16(v); }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half(v); }
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }

// tanh y and 1 - tanh^2 y.  Near zero y (1 + s P(s)), s = y^2, P fitted to (tanh(y) / y - 1) / s on |y| <= 3/4 for the smallest largest
// relative error (8e-9 with the coefficients in fp32, some 2^-23.5 with the steps' roundings); beyond it 1 - 2 / (1 + e^2y), whose slope is
// formed without 1 - t^2.
constexpr float TANH_NEAR = 0.75f;
__device__ __forceinline__ float tanh_far(float y, float& slope) {
  const float r = __fdividef(2.f, 1.f + ex2(fminf(fabsf(y) * (2.f * LOG2E), 100.f)));
  slope = r * (2.f - r);
  return y != y ? y : copysignf(1.f - r, y);
}
__device__ __forceinline__ float tanh_of(float y, float& slope) {
  const float s = y * y;
  float p = 0.001736928359605372f;
  p = fmaf(p, s, -0.007657244335860014f);
  p = fmaf(p, s, 0.021452028304338455f);
  p = fmaf(p, s, -0.053892724215984344f);
  p = fmaf(p, s, 0.1333269476890564f);
  p = fmaf(p, s, -0.33333316445350647f);
  const float near = fmaf(y, s * p, y);
  float far_slope;
  const float far = tanh_far(y, far_slope);
  const bool is_near = fabsf(y) <= TANH_NEAR;
  slope = is_near ? 1.f - near * near : far_slope;
  return is_near ? near : far;
}

// the cap and its slope
template <bool CAP>
__device__ __forceinline__ float capped(const Row& a, float z, float& slope) {
  if (!CAP) {
    slope = 1.f;
    return z;
  }
  const float t = tanh_of(z * a.inv_cap, slope);
  return z == -INFINITY ? z : a.cap * t;                       // (a token without probability stays one)
}
template <bool CAP>
__device__ __forceinline__ float capped(const Row& a, float z) {
  float slope;
  return capped<CAP>(a, z, slope);
}

constexpr uint32_t NAN_ORDER = 0xFFFFFFFEu;
// whole numbers in the order of the floats: -0 is +0, a NaN is above all
__device__ __forceinline__ uint32_t order_of(float f) {
  if (f != f) return NAN_ORDER;
  const uint32_t b = __float_as_uint(f + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

template <int NT>
__device__ __forceinline__ float block_sum(float v, float* sh) {
  __syncthreads();
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.f;
#pragma unroll
  for (int i = 0; i < NT / 32; ++i) v += sh[i];
  return v;
}

// What a policy row is given besides its logits, asked for long before it is used.
struct Given {
  float adv, old, ref;
};
__device__ __forceinline__ Given given_of(const Row& a, int row) {
  return {a.adv ? a.adv[row] : 1.f, a.old ? a.old[row] : 0.f, a.ref ? a.ref[row] : 0.f};
}
// Loss of a policy-gradient row and its derivative by log p of the taken token.  The unclipped side counts where both are equal, so
// a ratio inside the borders, and on them, has a gradient.
__device__ __forceinline__ float policy_row(const Row& a, const Given& v, float lp, float H, float& g) {
  float L = -v.adv * lp;
  g = -v.adv;
  if (a.old) {
    const float r = expf(lp - v.old);
    const float free = r * v.adv, held = fminf(fmaxf(r, 1.f - a.clip_low), 1.f + a.clip_high) * v.adv;
    L = -fminf(free, held);
    g = free <= held ? -free : 0.f;
    if (r != r || v.adv != v.adv) L = g = r * v.adv;         // (minima and maxima leave NaN out)
  }
  if (a.ref && a.kl != 0.f) {
    const float d = v.ref - lp, e = expm1f(d);
    L += a.kl * (e - d);
    g -= a.kl * e;
  }
  return a.bonus != 0.f ? L - a.bonus * H : L;
}

// ------------------------------------------------------------------------------------------------- a row's totals
// What a part of a row (one block's) adds to them.  ``m``: largest u of the tokens that are not named (the given token of scores and
// policy rows, the teacher's of distillation are, and are added by themselves), S and A sums of e and of e log2 e relative to it, S1 of
// e at a temperature of one.
struct __align__(16) Part {
  float m, S, A, S1;
  float B, En, En1, kl, Q;                // distillation: the named tokens of this part relative to their largest u, B
  float ut, has_t;                        // the given token's u, in the part that holds it
  uint32_t low;                           // scores: as many tokens of the part as is its share of K are not below it
};
// what follows from all parts
struct Totals {
  float M, lS, lp, H, miss, g;            // largest u, log2 of the sum, log p_t, entropy, 1 - p_t, dL/dlog p_t
  float base, k0, ka, kb;                 // gradient of a token that is not named: 2^((u - base) c + k0) (ka + kb log p) ...
  float share, h0;                        // ... + ce 2^((u - M) log2 e - h0); distillation: the sum of q
  uint32_t low;                           // scores: at least K tokens are not below it
};
constexpr int MOST_PARTS = 8;               // blocks of a cluster
typedef unsigned long long u64;
constexpr int PART_PIECES = sizeof(Part) / 16;

__device__ __forceinline__ Part no_part() { return {-INFINITY, 0.f, 0.f, 0.f, -INFINITY, 0.f, 0.f, 0.f, 0.f, -INFINITY, 0.f, 0xFFFFFFFFu}; }
// By one warp, every lane the same over all parts (those that there are not: no_part).  ``first``: of the row's blocks this one writes
// its results.
template <Op OP, bool HARD>
__device__ __forceinline__ void total(const Row& a, int row, const Part* rec, float qr, const Given& given, bool first, Totals* fin) {
  const bool writes = first && (threadIdx.x & 31) == 0;
  Totals t = {};
  float rest = -INFINITY, ut = -INFINITY, B = -INFINITY;      // largest of the tokens that are not named, the given token's, of the named
  bool has = false;
#pragma unroll
  for (int r = 0; r < MOST_PARTS; ++r) {
    rest = fmaxf(rest, rec[r].m);
    if (rec[r].has_t > 0.f) has = true, ut = rec[r].ut;
    if (OP == DISTILL) B = fmaxf(B, rec[r].B);
  }
  if (OP != DISTILL) {
    t.M = fmaxf(rest, ut);
    float O = 0.f, A = 0.f;
#pragma unroll
    for (int r = 0; r < MOST_PARTS; ++r) {
        const float d = (rec[r].m - t.M) * a.c;
      const bool none = rec[r].m == -INFINITY;
      const float down = none ? 0.f : ex2(d);
      O += down * rec[r].S;
      A += down == 0.f ? 0.f : down * (rec[r].A + rec[r].S * d);
      if (OP == SCORES) t.low = r == 0 ? rec[r].low : min(t.low, rec[r].low);
    }
    const float yt = (ut - t.M) * a.c, et = has ? ex2(yt) : 0.f, S = O + et;
    if (has) A += et * max_nan(yt, -256.f);
    t.lS = S > 0.f ? log2f(S) : NAN;                          // no finite logit (or a NaN): all that follows is NaN
    // a token that has most of the row: the others' sum by itself, so that a small log p keeps its digits
    const bool most = has && ut >= rest && S > 0.f;
    const float ln_S = most ? log1pf(O) : t.lS * LN2;
    t.lp = most ? -ln_S : (ut - t.M) * a.inv_tau - ln_S;      // (not from yt: a mask's lowest value is beyond fp32 in base 2)
    t.H = ln_S - A / S * LN2;
    t.miss = O / S;
    t.base = t.M;
    t.k0 = -t.lS;
    if (OP == SCORES) {
      if (writes) {
        if (a.logprob) a.logprob[row] = t.lp;
        a.entropy[row] = t.H;
        a.lse[row] = t.M * a.inv_tau + ln_S;
      }
    } else {
      const float L = policy_row(a, given, t.lp, t.H, t.g);
      t.ka = a.bonus * t.H - t.g;
      t.kb = a.bonus;
      if (writes) {
        a.loss[row] = L;
        a.logprob[row] = t.lp;
        a.entropy[row] = t.H;
      }
    }
  } else {
    t.M = fmaxf(rest, B);
    const float base = rest == -INFINITY ? 0.f : rest;
    float others = 0.f, named = 0.f, S1 = 0.f, Q = 0.f, kl = 0.f;
#pragma unroll
    for (int r = 0; r < MOST_PARTS; ++r) {
        const Part& p = rec[r];
      const bool none = p.m == -INFINITY, no_names = p.B == -INFINITY;        // (a sum of nothing may still be NaN: it is kept)
      others += p.S * (none ? 0.f : ex2((p.m - base) * a.c));
      if (HARD) S1 += p.S1 * (none ? 0.f : ex2((p.m - t.M) * LOG2E));
      named += p.En * (no_names ? 0.f : ex2((p.B - t.M) * a.c));
      if (HARD) S1 += p.En1 * (no_names ? 0.f : ex2((p.B - t.M) * LOG2E));
      kl += no_names || p.Q == 0.f ? 0.f : p.Q * (t.M - p.B) * a.inv_tau;
      kl += p.kl;
      Q += p.Q;
    }
    const float S = others * (rest == -INFINITY ? 0.f : ex2((base - t.M) * a.c)) + named;
    t.lS = S > 0.f ? log2f(S) : NAN;
    // q (log q - log p), where log p = (u - M) / tau - ln S and a part has (u - B) / tau
    if (Q != 0.f || t.lS != t.lS) kl += Q * t.lS * LN2;        // (a row without a distribution is NaN without a teacher's tokens as well)
    t.base = base;
    t.k0 = (base - t.M) * a.c - t.lS;
    t.share = a.bucket ? Q + qr : (Q != 0.f ? 1.f : 0.f);
    t.ka = t.share;
    if (a.bucket) {
      if (rest != -INFINITY && qr > 0.f) {
        const float l2 = (base - t.M) * a.c + log2f(others) - t.lS;       // log2 of the student's share of the others
        kl += qr * (logf(qr) - l2 * LN2);
        if (l2 <= -60.f) {                                    // (p itself is nothing beside the teacher's share there)
          t.k0 = -log2f(others);
          t.ka = -qr;
        } else {                                              // (NaN too, which the gradients keep)
          t.ka = t.share - qr / ex2(l2);
        }
      } else {                                                // nothing is left beside the named tokens
        t.share = t.ka = Q;
      }
    }
    const bool alone = HARD && a.ce >= 1.f;                   // cross entropy and nothing else: no share of an infinite divergence
    if (alone) t.share = t.ka = 0.f;
    float L = alone ? 0.f : (1.f - a.ce) * a.tau * a.tau * kl;
    if (HARD) {
      t.h0 = S1 > 0.f ? log2f(S1) : NAN;
      L -= a.ce * ((ut - t.M) - t.h0 * LN2);
    }
    if (writes) a.loss[row] = L;
  }
  if ((threadIdx.x & 31) == 0) *fin = t;
}

// gradients, before the slope of the cap and the scale
template <Op OP, bool HARD>
__device__ __forceinline__ float grad_rest(const Row& a, const Totals& t, float u) {
  const float y = (u - t.base) * a.c + t.k0;
  if (OP == POLICY) return t.kb != 0.f ? ex2(y) * (t.ka + t.kb * LN2 * max_nan(y, -256.f)) : ex2(y) * t.ka;
  const float v = (1.f - a.ce) * a.tau * (ex2(y) * t.ka);
  return HARD ? v + a.ce * ex2((u - t.M) * LOG2E - t.h0) : v;
}
__device__ __forceinline__ float grad_taken(const Totals& t, float bonus) {        // policy: p (g' ...) + g (1 - p)
  return bonus != 0.f ? t.g * t.miss + bonus * expf(t.lp) * (max_nan(t.lp, -200.f) + t.H) : t.g * t.miss;
}
template <bool HARD>
__device__ __forceinline__ float grad_named(const Row& a, const Totals& t, float u, float q, bool is_t) {
  const float v = HARD && a.ce >= 1.f ? 0.f : (1.f - a.ce) * a.tau * (ex2((u - t.M) * a.c - t.lS) * t.share - q);
  return HARD ? v + a.ce * (ex2((u - t.M) * LOG2E - t.h0) - (is_t ? 1.f : 0.f)) : v;
}

__device__ __forceinline__ bool row_on(const Row& a, int row, long t) {
  return (!a.targets || (t != a.ignore && t >= 0 && t < a.V)) && (!a.mask || a.mask[row] > 0.f);
}
template <Op OP>
__device__ __forceinline__ void row_off(const Row& a, int row) {                  // by a block
  if (threadIdx.x == 0) {
    if (OP != SCORES) a.loss[row] = 0.f;
    if (OP != DISTILL && a.logprob) a.logprob[row] = 0.f;
    if (OP != DISTILL) a.entropy[row] = 0.f;
    if (OP == SCORES) a.lse[row] = 0.f;
  }
  if (OP == SCORES)
    for (int k = threadIdx.x; k < a.K; k += blockDim.x) {
      a.top_ids[(size_t)row * a.K + k] = -1;
      a.top_logprob[(size_t)row * a.K + k] = -INFINITY;
    }
}

// The teacher's entries k = lane, lane + 32, ... by one warp: token (-1: none), q and log q; in the part that holds it the token's logit,
// and of entries of the same token one that stands for all.
constexpr int ENTRIES = MOST_TOP / 32;
struct Named {
  int id[ENTRIES];
  float q[ENTRIES], log_q[ENTRIES], z[ENTRIES];
  bool here[ENTRIES], first[ENTRIES];
};
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(~0u, v, o));
  return v;
}
// Returns what the teacher leaves to all others (0 without the bucket); ``id`` and ``q`` are of MOST_TOP, ``named_t``: t is among them.
__device__ __forceinline__ float teacher_of(const Row& a, int row, long t, int* id, float* q, Named& n, bool& named_t) {
  const int lane = threadIdx.x & 31;
  float top = -INFINITY, sum = 0.f, said[ENTRIES];
  bool has_t = false;
  long named[ENTRIES];
#pragma unroll
  for (int j = 0; j < ENTRIES; ++j) {                         // (all asked for before the first is looked at)
    const bool in = lane + 32 * j < a.K;
    named[j] = in ? a.ids[(size_t)row * a.K + lane + 32 * j] : -1;
    said[j] = in ? a.teacher[(size_t)row * a.K + lane + 32 * j] : 0.f;
  }
#pragma unroll
  for (int j = 0; j < ENTRIES; ++j) {
    const int k = lane + 32 * j;
    n.id[j] = -1;
    n.log_q[j] = -INFINITY;
    n.here[j] = n.first[j] = false;
    n.z[j] = 0.f;
    const long i = named[j];
    if (i >= 0 && i < a.V) {
      n.id[j] = static_cast<int>(i);
      n.log_q[j] = said[j];
      has_t |= i == t;
    }
    if (k < a.K) id[k] = n.id[j];
    top = fmaxf(top, n.log_q[j]);
  }
  named_t = __any_sync(~0u, has_t);
  top = warp_max(top);
  if (a.bucket || top == -INFINITY) top = 0.f;
#pragma unroll
  for (int j = 0; j < ENTRIES; ++j) {
    n.log_q[j] -= top;
    n.q[j] = n.id[j] >= 0 ? expf(n.log_q[j]) : 0.f;
    sum += n.q[j];
  }
  sum = warp_sum(sum);
  if (!a.bucket && sum != 0.f) {
    const float l = logf(sum);
#pragma unroll
    for (int j = 0; j < ENTRIES; ++j) {
      n.log_q[j] -= l;
      n.q[j] = n.id[j] >= 0 ? expf(n.log_q[j]) : 0.f;
    }
  }
#pragma unroll
  for (int j = 0; j < ENTRIES; ++j)
    if (lane + 32 * j < a.K) q[lane + 32 * j] = n.q[j];
  return a.bucket && sum < 1.f ? 1.f - sum : 0.f;
}
// B, En, En1, kl and Q of a part
template <bool CAP, bool HARD>
__device__ __forceinline__ void named_part(const Row& a, const Named& n, Part& p) {
  float u[ENTRIES], B = -INFINITY, En = 0.f, En1 = 0.f, kl = 0.f, Q = 0.f;
#pragma unroll
  for (int j = 0; j < ENTRIES; ++j) {
    u[j] = n.here[j] ? capped<CAP>(a, n.z[j]) : -INFINITY;
    B = fmaxf(B, u[j]);
  }
  B = warp_max(B);
#pragma unroll
  for (int j = 0; j < ENTRIES; ++j) {
    const float d = u[j] - (B == -INFINITY ? 0.f : B);
    if (n.first[j]) En += ex2(d * a.c);
    if (HARD && n.first[j]) En1 += ex2(d * LOG2E);
    if (n.here[j] && n.q[j] != 0.f) kl += n.q[j] * (n.log_q[j] - d * a.inv_tau);
    if (n.here[j]) Q += n.q[j];
  }
  p.B = B;
  p.En = warp_sum(En);
  if (HARD) p.En1 = warp_sum(En1);
  p.kl = warp_sum(kl);
  p.Q = warp_sum(Q);
}
__device__ __forceinline__ float q_of(const int* id, const float* q, int K, int mine) {
  float s = 0.f;
  for (int k = 0; k < K; ++k) s += id[k] == mine ? q[k] : 0.f;
  return s;
}
// the gradients of the named tokens, by the same warp
template <typename E, bool CAP, bool HARD>
__device__ __forceinline__ void write_named(const Row& a, const Totals& t, const Named& n, const int* id, const float* q, long target, float scale, E* out) {
  bool more = false;
#pragma unroll
  for (int j = 0; j < ENTRIES; ++j) more |= n.here[j] && !n.first[j];
  more = __any_sync(~0u, more);
#pragma unroll
  for (int j = 0; j < ENTRIES; ++j)
    if (n.first[j]) {
      float slope;
      const float u = capped<CAP>(a, n.z[j], slope), qs = more ? q_of(id, q, a.K, n.id[j]) : n.q[j];
      out[n.id[j]] = from_float<E>(grad_named<HARD>(a, t, u, qs, n.id[j] == target) * slope * scale);
    }
}


// ---------------------------------------------------------------------------------------------- clusters and pieces
// (Times of this file: B200, us of a call back to back with others on two inputs beyond the second level of cache; 16-bit logits, a quarter
// of the rows left out where there are 4,096 of them.  In turn with other work the longest ones take up to a seventh more.)
// Pieces of 16 bytes that a thread asks for at once: 8 for the totals (4096 x 151936 scores 153, 173 with 4), 4 under a soft-cap, whose code
// is long (1001 x 256000 policy gradient 321, 314 with 8), and for the gradient (4096 x 151936 417, 427 with 8, 455 with 2).
constexpr int BATCH = 8, GRAD_BATCH = 4;
// Bytes of a row's slice from which a block has 512 threads and not 256, for some operators.  Alternatives: more threads give a closer bound.
// Policy gradients, and soft-caps: half as many rows at a time, which the second level of cache then still has when the gradient reads them
// again.  With 256 / 512 threads, 64 alternatives at 2048 x 32000 80 / 98, x 57600 (just above the border) 115 / 117, x 80000 157 / 150, 1024 x
// 128256 123 / 98; policy gradients 60 / 67, 100 / 100, 142 / 133 and 121 / 107.  Under a cap the sides meet later: policy gradients at 1500 x
// 57600 138 / 146, 1001 x 100000 154 / 155, x 256000 375 / 366; scores 64 / 71, 71 / 73, 166 / 165; alternatives 115 / 120, 134 / 118, 301 / 249.
// Scores and distillation without a cap: 256 threads, four blocks whose steps lie beside one another (4096 x 151936 scores 153, 167 with 512;
// held-out distillation 2048 x 151936 114 and 136; with gradient 4096 x 128256 450 and 477).
constexpr int LONG_ROW = 114688;
// Rows are cut over a cluster where there are fewer blocks than two for each SM.  In 1 / 2 / 4 parts: 148 x 50257 scores 10.1 / 8.7 / 10.4,
// distillation 21 / 19 / 25; 295 x 50257 scores 11.8 / 11.3 / 15, 20 alternatives 19 / 19 / 30, policy gradient 18.4 / 17.4 / 24; 297 rows 12.6 /
// 13.1 / 15, 20 / 24 / 31, 20.6 / 21.9 / 25.  Longer rows: 295 x 151936 scores 24 / 21 / 25, alternatives 32 / 39 / 45, distillation 64 / 59 / 70;
// 400 rows 29 / 29 / 31, 50 / 54 / 54, 84 / 82 / 88.
constexpr int FEW_BLOCKS = 2 * 148;
__device__ __forceinline__ uint32_t in_cluster(const void* p, int rank) {          // the same place in another block's shared memory
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(ftb::smem_u32(p)), "r"(rank));
  return r;
}
__device__ __forceinline__ void put32(uint32_t at, uint32_t v) { asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(at), "r"(v) : "memory"); }
__device__ __forceinline__ void put64(uint32_t at, u64 v) { asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(at), "l"(v) : "memory"); }
// 16 bytes to another block, counted on a barrier there
__device__ __forceinline__ void send16(uint32_t at, const uint4& v, uint32_t barrier) {
  asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v4.b32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z),
               "r"(v.w), "r"(barrier)
               : "memory");
}
__device__ __forceinline__ void cluster_arrive() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_arrive_relaxed() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// what other blocks sent; bounded as ftb::mbar_wait, and once more as long after it was reported
__device__ __forceinline__ void sent_wait(uint64_t* bar, int where) {
  for (int again = 0; again < 2; ++again) {
    for (uint32_t it = 0; it < FTB_WAIT_LIMIT; ++it) {
      uint32_t ok;
      asm volatile(
          "{\n.reg .pred p;\n"
          "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], 0;\n"
          "selp.u32 %0, 1, 0, p;\n}\n"
          : "=r"(ok)
          : "r"(ftb::smem_u32(bar))
          : "memory");
      if (ok) return;
    }
    ftb::set_error(1, where);
  }
}

// two floats to an instruction
typedef u64 f32x2;
__device__ __forceinline__ f32x2 pair(float a, float b) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void split(f32x2 v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ f32x2 exp2_2(f32x2 x) {
  float a, b;
  split(x, a, b);
  return pair(ex2(a), ex2(b));
}

// 16 bytes of a row as pairs of floats, their largest, and back
template <typename E>
struct Vec;
template <>
struct Vec<bf16> {
  static constexpr int N = 8;
  static constexpr float LOW = -0x1p100f;                     // a finite number below all logits that are not a mask's
  __device__ static uint32_t max2(uint32_t a, uint32_t b) {
    const __nv_bfloat162 r = __hmax2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  __device__ static f32x2 one(uint32_t w) { return pair(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u)); }
  __device__ static float top(uint32_t m) { return fmaxf(__uint_as_float(m << 16), __uint_as_float(m & 0xFFFF0000u)); }
  __device__ static uint32_t word(f32x2 v) {
    float a, b;
    split(v, a, b);
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static constexpr uint32_t NONE = 0xFF80FF80u, FLOOR = 0xF180F180u;      // -inf, LOW
};
template <>
struct Vec<__half> {
  static constexpr int N = 8;
  static constexpr float LOW = -65504.f;
  __device__ static uint32_t max2(uint32_t a, uint32_t b) {
    const __half2 r = __hmax2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  __device__ static f32x2 one(uint32_t w) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
    return pair(f.x, f.y);
  }
  __device__ static float top(uint32_t m) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&m));
    return fmaxf(f.x, f.y);
  }
  __device__ static uint32_t word(f32x2 v) {
    float a, b;
    split(v, a, b);
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static constexpr uint32_t NONE = 0xFC00FC00u, FLOOR = 0xFBFFFBFFu;
};
template <>
struct Vec<float> {
  static constexpr int N = 4;
  static constexpr float LOW = -0x1p100f;
  __device__ static uint32_t max2(uint32_t a, uint32_t b) { return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b))); }
  __device__ static float top(uint32_t m) { return __uint_as_float(m); }
  static constexpr uint32_t NONE = 0xFF800000u, FLOOR = 0xF1800000u;
};
template <typename E>
__device__ __forceinline__ uint32_t vec_max(const uint4& v) {
  return Vec<E>::max2(Vec<E>::max2(v.x, v.y), Vec<E>::max2(v.z, v.w));
}
template <typename E>
__device__ __forceinline__ uint4 vec_floor(const uint4& v) {  // -inf and all below LOW to LOW
  constexpr uint32_t f = Vec<E>::FLOOR;
  return make_uint4(Vec<E>::max2(v.x, f), Vec<E>::max2(v.y, f), Vec<E>::max2(v.z, f), Vec<E>::max2(v.w, f));
}
template <typename E>
__device__ __forceinline__ void pairs_of(const uint4& v, f32x2 (&x)[Vec<E>::N / 2]) {
  if constexpr (sizeof(E) == 4) {
    x[0] = pair(__uint_as_float(v.x), __uint_as_float(v.y));
    x[1] = pair(__uint_as_float(v.z), __uint_as_float(v.w));
  } else {
    x[0] = Vec<E>::one(v.x); x[1] = Vec<E>::one(v.y); x[2] = Vec<E>::one(v.z); x[3] = Vec<E>::one(v.w);
  }
}
template <typename E>
__device__ __forceinline__ uint4 vec_of(const f32x2 (&x)[Vec<E>::N / 2]) {
  if constexpr (sizeof(E) == 4) {
    float a, b, c, d;
    split(x[0], a, b);
    split(x[1], c, d);
    return make_uint4(__float_as_uint(a), __float_as_uint(b), __float_as_uint(c), __float_as_uint(d));
  } else {
    return make_uint4(Vec<E>::word(x[0]), Vec<E>::word(x[1]), Vec<E>::word(x[2]), Vec<E>::word(x[3]));
  }
}
template <typename E>
__device__ __forceinline__ void floats_of(const uint4& v, float (&f)[Vec<E>::N]) {
  f32x2 x[Vec<E>::N / 2];
  pairs_of<E>(v, x);
#pragma unroll
  for (int i = 0; i < Vec<E>::N / 2; ++i) split(x[i], f[2 * i], f[2 * i + 1]);
}
// What few pieces need lies outside the loops, whose instructions are read from a cache as well.
__device__ __noinline__ f32x2 cap_far(float inv_cap, float cap, f32x2 z, f32x2& slope) {
  float c, d, sc, sd;
  split(z, c, d);
  const float tc = tanh_of(c * inv_cap, sc), td = tanh_of(d * inv_cap, sd);
  slope = pair(sc, sd);
  return pair(c == -INFINITY ? c : cap * tc, d == -INFINITY ? d : cap * td);        // (as capped)
}
// sum of e log2 e of a pair, nothing where e is nothing
__device__ __noinline__ float careful_part(f32x2 y) {
  float b, c;
  split(y, b, c);
  return ex2(b) * max_nan(b, -256.f) + ex2(c) * max_nan(c, -256.f);
}
// z to u in place, and the slopes; the tanh of all pairs near zero by its polynomial, of any beyond it one by one
template <typename E, bool SLOPE>
__device__ __forceinline__ void cap_pairs(const Row& a, f32x2 (&x)[Vec<E>::N / 2], f32x2 (&slope)[Vec<E>::N / 2]) {
  constexpr int P = Vec<E>::N / 2;
  f32x2 y[P];
  float most = 0.f;
#pragma unroll
  for (int i = 0; i < P; ++i) {
    y[i] = mul2(x[i], pair(a.inv_cap, a.inv_cap));
    float c, d;
    split(y[i], c, d);
    most = fmaxf(most, fmaxf(fabsf(c), fabsf(d)));
  }
  if (most <= TANH_NEAR) {
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const f32x2 s = mul2(y[i], y[i]);
      f32x2 p = pair(0.001736928359605372f, 0.001736928359605372f);
      p = fma2(p, s, pair(-0.007657244335860014f, -0.007657244335860014f));
      p = fma2(p, s, pair(0.021452028304338455f, 0.021452028304338455f));
      p = fma2(p, s, pair(-0.053892724215984344f, -0.053892724215984344f));
      p = fma2(p, s, pair(0.1333269476890564f, 0.1333269476890564f));
      p = fma2(p, s, pair(-0.33333316445350647f, -0.33333316445350647f));
      const f32x2 t = fma2(y[i], mul2(s, p), y[i]);
      if (SLOPE) slope[i] = fma2(mul2(t, pair(-1.f, -1.f)), t, pair(1.f, 1.f));
      x[i] = mul2(t, pair(a.cap, a.cap));
    }
  } else {
#pragma unroll
    for (int i = 0; i < P; ++i) {
      f32x2 far;
      x[i] = cap_far(a.inv_cap, a.cap, x[i], far);
      if (SLOPE) slope[i] = far;
    }
  }
}

__device__ __forceinline__ u64 key_of(float z, int token) { return static_cast<u64>(order_of(z)) << 32 | static_cast<uint32_t>(~token); }
__device__ __forceinline__ float logit_of(uint32_t order) {
  return order == NAN_ORDER ? NAN : __uint_as_float(order & 0x80000000u ? order & 0x7FFFFFFFu : ~order);
}

// --------------------------------------------------------------------------------------------------- a row's passes
// A block takes a row, or a cluster of up to eight blocks where there are few rows, a piece of it each (pieces of 16 bytes; the ones that
// a row begins and ends in by single threads).  Memory is read once for the totals: each thread keeps the largest logit that it has seen
// and its sums relative to it.  The blocks of a cluster send one another their parts of the totals.  The gradient reads the row a second
// time, from the second level of cache, and is the only other traffic; alternatives read a few threads' pieces again.
//
// Alternatives: a bound that at least K tokens are not below, from the largest ones by thread (found by halving an interval of whole
// numbers that are in the order of the floats); every block gives the tokens from the lowest of the blocks' bounds on to all, and ranks
// its own among them.  Where these are too many because the blocks' tokens differ, the bound is the highest of bounds by K threads of a
// block; where thousands of logits are equal, the cluster halves the interval of (logit, index) of all tokens until exactly K are left.
//
// What bounds it: scores by memory, 153 us for 142 at 4096 x 151936 (6.1 of 6.55 TB/s); with the gradient by the second reading, whose rows
// the cache has lost in part (policy gradients 412 for 332; the pass goes through the row from its end, 4 % more from its beginning), and
// with cross entropy at another temperature beside it by the exponentials, four an element (distillation 4096 x 128256 450 for 281).  64
// alternatives 2048 x 128256 184 for 80: rows by two blocks of 512 threads an SM, whose steps follow one another, and 44 to 76 bytes of
// spilled registers.  64 registers a thread, so that four blocks of 256 or two of 512 fit: with registers
// for three and one of them scores take 166, distillation 5 % and policy gradients a fifth more; for five and two 165, 1 % and 2 %.  The price
// are spills in distillation with cross entropy (52 bytes) and under a soft-cap (up to 68).
// Earlier builds: rows in the shared memory of clusters of eight, each block a piece that stays for the gradient, with clusters that take
// over rows of others (policy gradients 427, but scores 206 and distillation 631: the blocks of a row wait for the slowest of them at every
// row); pieces kept in shared memory, up to 208 KB an SM (a sixth slower: what the first level of cache loses was in use for loads on their
// way), up to 96 KB (1 % faster).
template <typename E, Op OP, bool TOP, bool CAP, bool HARD, int NT>
__global__ void __launch_bounds__(NT, 1024 / NT) row_kernel(Row a, int slice, int room) {
  constexpr int VE = Vec<E>::N, P = VE / 2, W = NT / 32, U = CAP ? BATCH / 2 : BATCH, GU = GRAD_BATCH;
  extern __shared__ __align__(16) unsigned char buf[];        // DISTILL: for each piece which of its tokens are named; TOP: tokens given
  __shared__ __align__(8) uint64_t sent;
  __shared__ int found;
  __shared__ float sh[32], most[W], least[W], sums[3][W];
  __shared__ Part rec[MOST_PARTS], own;
  __shared__ Totals fin;
  __shared__ int count[2][MOST_PARTS];
  __shared__ uint32_t bounds[MOST_PARTS];
  __shared__ int id[OP == DISTILL ? MOST_TOP : 1];
  __shared__ float q[OP == DISTILL ? MOST_TOP : 1];
  __shared__ Named names[OP == DISTILL ? 32 : 1];

  int rank, parts;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(parts));
  const int row = blockIdx.x / parts, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, V = a.V, K = a.K;
  const E* z = static_cast<const E*>(a.z) + row * a.ldz;
  E* out = static_cast<E*>(a.out) + row * a.ldo;
  // the row from the 16-byte piece that it begins in: ``lead`` elements before it, this block's from ``lo`` on, n of them in nv pieces,
  // those from full to end_full with no others in them
  const int lead = static_cast<int>((reinterpret_cast<uintptr_t>(z) & 15) / sizeof(E));
  const int lo = rank * slice, n = max(0, min(lead + V - lo, slice)), nv = (n + VE - 1) / VE, first_token = lo - lead;
  const int full = first_token < 0 ? 1 : 0, end_full = n / VE;
  const uint4* zv = reinterpret_cast<const uint4*>(z - lead + lo);
  const bool whole = OP != SCORES && (reinterpret_cast<uintptr_t>(out) & 15) / sizeof(E) == lead;       // the gradient's pieces lie as the logits' do
  const long t = a.targets ? a.targets[row] : -1;
  if (!row_on(a, row, t)) {
    if (OP != SCORES && a.out)
      for (int v = tid; v < nv; v += NT) {
        const int token = first_token + v * VE;
        if (whole && token >= 0 && token + VE <= V) {
          *reinterpret_cast<uint4*>(out + token) = make_uint4(0, 0, 0, 0);
        } else {
          for (int e = 0; e < VE; ++e)
            if (token + e >= 0 && token + e < V) out[token + e] = from_float<E>(0.f);
        }
      }
    if (rank == 0) row_off<OP>(a, row);
    return;
  }
  if (tid == 0) {
    found = 0;
    ftb::mbar_init(&sent, 1);
    ftb::fence_barrier_init();
    ftb::mbar_expect_tx(&sent, parts * sizeof(Part));
  }
  if (parts > 1) cluster_arrive_relaxed();                    // (the others may be sent to once all have begun)
  if (tid < MOST_PARTS && tid >= parts) rec[tid] = no_part();
  const int at_t = static_cast<int>(t) - first_token;         // where the given token lies
  const bool mine_t = a.targets && at_t >= 0 && at_t < n;
  const int piece_t = OP != DISTILL && mine_t ? at_t / VE : -1;
  float zt = 0.f;
  Given policy = {};
  if (warp == 0) {
    if (mine_t) zt = to_float(z[t]);
    if (OP == POLICY) policy = given_of(a, row);
  }
  float qr = 0.f;
  bool named_t = false;
  if (OP == DISTILL) {
    Named mine;
    for (int i = tid; i < (nv + 15) / 16; i += NT) reinterpret_cast<uint4*>(buf)[i] = make_uint4(0, 0, 0, 0);
    if (warp == 0) qr = teacher_of(a, row, t, id, q, mine, named_t);
    __syncthreads();
    if (warp == 0) {
#pragma unroll
      for (int j = 0; j < ENTRIES; ++j) {
        const int at = mine.id[j] - first_token;
        mine.here[j] = mine.id[j] >= 0 && at >= 0 && at < n;
        if (!mine.here[j]) continue;
        mine.z[j] = to_float(z[mine.id[j]]);
        const int v = at / VE;
        const uint32_t bit = 1u << ((v & 3) * 8 + at % VE);
        mine.first[j] = !(atomicOr(reinterpret_cast<uint32_t*>(buf) + (v >> 2), bit) & bit);      // (of entries of one token, one stands for all)
      }
      names[lane] = mine;
    }
    __syncthreads();
  }

  // The totals' parts.  struck: tokens of a piece that are not summed here, a bit each.
  float top = -INFINITY, base = 0.f, A = 0.f;                 // largest logit, u that the sums are relative to
  f32x2 S = 0, S1 = 0;
  const f32x2 cc = pair(a.c, a.c), l2 = pair(LOG2E, LOG2E);
  auto strike = [&](uint4& w, uint32_t struck) {
    uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (sizeof(E) == 4) {
        if (struck >> i & 1) x[i] = Vec<E>::NONE;
      } else {
        if (struck >> (2 * i) & 1) x[i] = (x[i] & 0xFFFF0000u) | (Vec<E>::NONE & 0xFFFFu);
        if (struck >> (2 * i + 1) & 1) x[i] = (x[i] & 0xFFFFu) | (Vec<E>::NONE & 0xFFFF0000u);
      }
    }
    w = make_uint4(x[0], x[1], x[2], x[3]);
  };
  auto struck_in = [&](int v) -> uint32_t {
    if (OP == DISTILL) return buf[v];
    return v == piece_t ? 1u << (at_t % VE) : 0u;
  };
  auto raise = [&](float m) {                                 // to logits of up to m
    if (!(m > top)) return;
    top = m;
    const float b = capped<CAP>(a, m), d = base - b, down = ex2(d * a.c);
    float s0, s1;
    split(S, s0, s1);
    if (s0 + s1 != 0.f) {
      A = down != 0.f ? down * (A + d * a.c * (s0 + s1)) : 0.f;               // (the difference may be minus infinity)
      S = mul2(S, pair(down, down));
      if (HARD) {
        const float down1 = ex2(d * LOG2E);
        S1 = mul2(S1, pair(down1, down1));
      }
    }
    base = b;
  };
  auto add = [&](const uint4& w) {
    const f32x2 minus = pair(-base, -base);
    f32x2 x[P], slope[P], part = 0;
    pairs_of<E>(w, x);
    if (CAP) cap_pairs<E, false>(a, x, slope);
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const f32x2 d = add2(x[i], minus), y = mul2(d, cc), e = exp2_2(y);
      S = add2(S, e);
      if (OP != DISTILL) part = fma2(e, y, part);
      if (HARD) S1 = add2(S1, exp2_2(mul2(d, l2)));
    }
    if (OP != DISTILL) {
      float b, c;
      split(part, b, c);
      b += c;
      if (b != b) {                                           // (a logit of -inf: nothing times minus infinity)
        b = 0.f;
#pragma unroll
        for (int i = 0; i < P; ++i) b += careful_part(mul2(add2(x[i], minus), cc));
      }
      A += b;
    }
  };
  // (piece_t is looked for once in U pieces, by the thread that has it)
  const int piece_mine = piece_t >= full && (piece_t - full) % NT == tid ? piece_t : -1;
  auto batch = [&](int v0, int most_v) {                      // pieces v0, v0 + NT, ... up to U of them, below most_v
    const uint4* at = zv + v0;
    uint4 w[U];
#pragma unroll
    for (int i = 0; i < U; ++i) w[i] = i == 0 || v0 + i * NT < most_v ? at[i * NT] : make_uint4(Vec<E>::NONE, Vec<E>::NONE, Vec<E>::NONE, Vec<E>::NONE);
    if (OP == DISTILL) {
#pragma unroll
      for (int i = 0; i < U; ++i)
        if (i == 0 || v0 + i * NT < most_v) {
          const uint32_t struck = buf[v0 + i * NT];
          if (struck) strike(w[i], struck);
        }
    } else if (static_cast<unsigned>(piece_mine - v0) < static_cast<unsigned>(U * NT)) {
#pragma unroll
      for (int i = 0; i < U; ++i)
        if (v0 + i * NT == piece_mine) strike(w[i], 1u << (at_t % VE));
    }
    uint32_t m2 = vec_max<E>(w[0]);
#pragma unroll
    for (int i = 1; i < U; ++i) m2 = Vec<E>::max2(m2, vec_max<E>(w[i]));
    raise(Vec<E>::top(m2));
#pragma unroll
    for (int i = 0; i < U; ++i)
      if (i == 0 || v0 + i * NT < most_v) add(w[i]);
  };
  {
    int v0 = full + tid;
    for (; v0 + (U - 1) * NT < end_full; v0 += U * NT) batch(v0, 0x7FFFFFFF);
    if (v0 < end_full) batch(v0, end_full);
  }
  // the pieces with others in them: the first by thread 0, the last by the last thread
  auto edge = [&](int v) {
    uint4 w = zv[v];
    uint32_t struck = struck_in(v);
    for (int e = 0; e < VE; ++e) {
      const int token = first_token + v * VE + e;
      if (token < 0 || token >= V) struck |= 1u << e;
    }
    strike(w, struck);
    raise(Vec<E>::top(vec_max<E>(w)));
    add(w);
  };
  if (tid == 0 && full == 1 && nv > 0) edge(0);
  if (tid == NT - 1 && end_full < nv && end_full >= full) edge(end_full);

  // of the block
  {
    const float w = warp_max(top);
    if (lane == 0) most[warp] = w;
    if (TOP) {
      float l = full + tid < end_full ? top : INFINITY;
#pragma unroll
      for (int o = 16; o; o >>= 1) l = fminf(l, __shfl_xor_sync(~0u, l, o));
      if (lane == 0) least[warp] = l;
    }
  }
  __syncthreads();
  float mz = most[0];
#pragma unroll
  for (int w = 1; w < W; ++w) mz = fmaxf(mz, most[w]);
  const float um = mz == -INFINITY ? mz : capped<CAP>(a, mz);
  {
    float b, c;
    split(S, b, c);
    b += c;
    const float d = base - (mz == -INFINITY ? 0.f : um), down = b != 0.f ? ex2(d * a.c) : 0.f;      // (nothing where there is nothing)
    const float s = warp_sum(b * down);
    if (lane == 0) sums[0][warp] = s;
    if (OP != DISTILL) {
      A = warp_sum(down != 0.f ? down * (A + d * a.c * b) : 0.f);
      if (lane == 0) sums[1][warp] = A;
    }
    if (HARD) {
      split(S1, b, c);
      b = warp_sum(b + c != 0.f ? (b + c) * ex2(d * LOG2E) : 0.f);
      if (lane == 0) sums[2][warp] = b;
    }
  }
  // the largest of at least ``want`` threads are not below it, and of not many more
  const int busy = min(end_full - full, NT);                  // threads with pieces of their own
  auto bound_of = [&](int want) {
    float l = least[0];
#pragma unroll
    for (int w = 1; w < W; ++w) l = fminf(l, least[w]);
    uint32_t low = order_of(l), high = order_of(mz) + 1;
    const uint32_t key = tid < busy ? order_of(top) : 0;
    for (int it = 0; it < 32 && high - low > 1; ++it) {
      const uint32_t mid = low + (high - low) / 2;
      const int c = __syncthreads_count(key >= mid);
      if (c >= want) low = mid;
      else high = mid;
      if (c >= want && c <= want + want / 4 + 4) break;
    }
    return low;
  };
  uint32_t low = 0;
  if (TOP) {
    const int filled = (lead + V + slice - 1) / slice, share = (K + filled - 1) / filled;      // (blocks without tokens have no share)
    if (nv == 0) low = 0xFFFFFFFFu;
    else if (busy >= share) low = bound_of(share);
  }
  __syncthreads();
  float slope_t = 1.f;
  if (parts > 1) cluster_wait();
  if (warp == 0) {
    Part p = {};
    p.B = -INFINITY;
    if (OP == DISTILL) named_part<CAP, HARD>(a, names[lane], p);
    p.m = um;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      p.S += sums[0][w];
      if (OP != DISTILL) p.A += sums[1][w];
      if (HARD) p.S1 += sums[2][w];
    }
    p.has_t = mine_t ? 1.f : 0.f;
    p.ut = mine_t ? capped<CAP>(a, zt, slope_t) : 0.f;
    p.low = low;
    if (parts > 1) {                                          // to every block of the cluster, this one among them
      if (lane == 0) own = p;
      __syncwarp();
      if (lane < parts * PART_PIECES) {
        const int to = lane / PART_PIECES, piece = lane - to * PART_PIECES;
        send16(in_cluster(reinterpret_cast<const uint4*>(&rec[rank]) + piece, to), reinterpret_cast<const uint4*>(&own)[piece], in_cluster(&sent, to));
      }
      sent_wait(&sent, 3);
    } else {
      if (lane == 0) rec[0] = p;
      __syncwarp();
    }
    total<OP, HARD>(a, row, rec, qr, policy, rank == 0, &fin);
  }
  if (OP == SCORES ? !TOP : a.out == nullptr) return;
  __syncthreads();
  const Totals T = fin;

  if (OP == SCORES) {
    u64* taken = reinterpret_cast<u64*>(buf);
    const bool broken = T.lS != T.lS;                         // (a thread's largest leaves NaN out)
    u64* ours = taken + rank * room;
    auto give = [&](float f, int token, u64 bound) {
      const u64 key = key_of(f, token);
      if (key < bound || token < 0 || token >= V) return;
      const int i = atomicAdd(&found, 1);
      if (i < room) ours[i] = key;
    };
    auto met = [&] {                                          // of the cluster; what was written to others' shared memory is there
      if (parts > 1) {
        cluster_arrive();
        cluster_wait();
      } else {
        __syncthreads();
      }
    };
    // A warp takes the threads with such tokens one by one, half a piece a lane; the pieces at the row's ends by themselves.
    auto collect = [&](u64 bound, bool all) {
      typedef typename std::conditional<sizeof(E) == 2, uint2, float2>::type Half;
      const uint32_t order = static_cast<uint32_t>(bound >> 32);
      if (warp == 0) {
        const int edge = full == 1 && nv > 0 && lane < VE ? first_token + lane : end_full < nv && end_full >= full && lane >= 8 && lane < 8 + VE ? first_token + end_full * VE + lane - 8 : -1;
        if (edge >= 0 && edge < V) give(to_float(z[edge]), edge, bound);
      }
      uint32_t those = __ballot_sync(~0u, tid < busy && (all || order_of(top) >= order));
      while (those) {
        const int first = full + (warp << 5) + __ffs(those) - 1;
        those &= those - 1;
        for (int h = lane; h < 2 * ((end_full - first + NT - 1) / NT); h += 32) {
          const int at = (first + (h >> 1) * NT) * VE + (h & 1) * (VE / 2);
          const Half w = *reinterpret_cast<const Half*>(reinterpret_cast<const E*>(zv) + at);
          float f[VE / 2];
          if constexpr (sizeof(E) == 4) {
            f[0] = w.x, f[1] = w.y;
          } else {
            split(Vec<E>::one(w.x), f[0], f[1]);
            split(Vec<E>::one(w.y), f[2], f[3]);
          }
#pragma unroll
          for (int e = 0; e < VE / 2; ++e) {
            const int token = first_token + at + e;
            if (order_of(f[e]) >= order && token != t) give(f[e], token, bound);
          }
        }
      }
      // (the given token is not among the threads' largest)
      if (tid == 0 && mine_t && piece_t >= full && piece_t < end_full) give(zt, static_cast<int>(t), bound);
      __syncthreads();
      if (parts > 1) {
        const int have = min(found, room);
        for (int i = tid; i < have * parts; i += NT) {
          const int to = i % parts, c = i / parts;
          if (to != rank) put64(in_cluster(ours + c, to), ours[c]);
        }
      }
      if (tid < parts) put32(in_cluster(&count[0][rank], tid), found);
      met();
      bool over = false;
      for (int r = 0; r < parts; ++r) over |= count[0][r] > room;
      return over;
    };
    u64 bound = static_cast<u64>(T.low) << 32;
    bool over = collect(bound, T.low == 0 || broken);
    if (over && parts > 1) {
      // the blocks' tokens differ: the highest of bounds that K threads of a block each are not below
      const uint32_t mine_low = busy >= K ? bound_of(K) : 0;
      if (tid < parts) put32(in_cluster(&bounds[rank], tid), mine_low);
      if (tid == 0) found = 0;
      met();                                                  // (all have read the last counts)
      uint32_t highest = T.low;
      for (int r = 0; r < parts; ++r) highest = max(highest, bounds[r]);
      bound = static_cast<u64>(highest) << 32;
      over = collect(bound, highest == 0 || broken);
    }
    if (over) {
      u64 below = 0, above = ~0ull;                           // at least K keys are not below the one, fewer not below the other
      for (int it = 0; above - below > 1; ++it) {
        const u64 mid = below + (above - below) / 2;
        int c = 0;
        for (int i = tid; i < n; i += NT) {
          const int token = first_token + i;
          c += token >= 0 && key_of(to_float(reinterpret_cast<const E*>(zv)[i]), token) >= mid;
        }
        c = static_cast<int>(block_sum<NT>(static_cast<float>(c), sh));           // (whole numbers below 2^24)
        if (tid < parts) put32(in_cluster(&count[1 - (it & 1)][rank], tid), c);
        met();
        int sum = 0;
        for (int r = 0; r < parts; ++r) sum += count[1 - (it & 1)][r];
        if (sum >= K) below = mid;
        else above = mid;
        if (sum == K) break;
      }
      if (tid == 0) found = 0;
      met();                                                  // (all have read the last counts)
      bound = below;
      collect(bound, true);
    }
    // eight threads to a token, one for each block's (an eighth of them where there is one block)
    const int mine_found = count[0][rank];
    for (int i = tid / MOST_PARTS; i < (mine_found + NT / MOST_PARTS - 1) / (NT / MOST_PARTS) * (NT / MOST_PARTS); i += NT / MOST_PARTS) {
      const int r = tid % MOST_PARTS;
      const bool valid = i < mine_found;
      const u64 key = valid ? ours[i] : ~0ull;
      int above = 0;
      if (parts > 1) {
        const int others = r < parts ? count[0][r] : 0;
#pragma unroll 4
        for (int j = 0; j < others; ++j) above += taken[r * room + j] > key;
      } else {
#pragma unroll 4
        for (int j = r; j < mine_found; j += MOST_PARTS) above += ours[j] > key;
      }
#pragma unroll
      for (int o = MOST_PARTS / 2; o; o >>= 1) above += __shfl_xor_sync(~0u, above, o);
      if (valid && r == 0 && above < K) {
        const int token = static_cast<int>(~static_cast<uint32_t>(key));
        a.top_ids[(size_t)row * K + above] = token;
        a.top_logprob[(size_t)row * K + above] =
            token == t ? T.lp : (capped<CAP>(a, logit_of(static_cast<uint32_t>(key >> 32))) - T.M) * a.inv_tau - T.lS * LN2;
      }
    }
    return;
  }

  const float scale = OP == DISTILL ? a.scale : a.scale * a.inv_tau;
  const bool bonus = OP == POLICY && T.kb != 0.f;
  // One by one: entropy's gradient where a cap leaves -inf (elsewhere it is brought to a number that has no p log p, unless all of the row
  // are such).
  const bool careful = bonus && (CAP || !(T.M > Vec<E>::LOW * 0.9f) || a.inv_tau < 0.05f);
  const f32x2 minus = pair(-T.base, -T.base), k0 = pair(T.k0, T.k0);
  const float fa = OP == POLICY ? T.ka * scale : (1.f - a.ce) * a.tau * T.ka * scale, fb = T.kb * LN2 * scale;
  const f32x2 ka = pair(fa, fa), kb = pair(fb, fb);
  const float f1 = (T.base - T.M) * LOG2E - T.h0;
  const f32x2 h1 = pair(f1, f1), ce = pair(a.ce * scale, a.ce * scale);
  // The exponents: from the difference of logits, which is exact or nearly so; or, one instruction a pair less, as a product and a constant
  // of its size, whose roundings are 2^-25 of both each: 3e-6 of a probability up to 64, so for rows of 16 bits below that (4096 x 128256
  // distillation 450 us, 458 with the difference; 4096 x 151936 policy gradient 412 and 415; gradients at logits of 1,000 would be off by 4e-5).
  const bool near = !CAP && sizeof(E) == 2 && fmaxf(fabsf(T.base), fabsf(T.M)) * fmaxf(a.c, LOG2E) < 64.f;
  const float f2 = fmaf(-T.base, a.c, T.k0), f3 = fmaf(-T.M, LOG2E, -T.h0);
  const f32x2 k2 = pair(f2, f2), h2 = pair(f3, f3);
  auto pass = [&](auto with_bonus, auto with_care, auto with_near) {
    constexpr bool BONUS = decltype(with_bonus)::value, CARE = decltype(with_care)::value, NEAR = decltype(with_near)::value;
    auto grad = [&](uint4 w) {
      f32x2 x[P], slope[P];
      pairs_of<E>(BONUS && !CARE ? vec_floor<E>(w) : w, x);
      if (CAP) cap_pairs<E, true>(a, x, slope);
#pragma unroll
      for (int i = 0; i < P; ++i) {
        f32x2 r;
        if (CARE) {
          float b, c;
          split(x[i], b, c);
          r = pair(grad_rest<OP, HARD>(a, T, b) * scale, grad_rest<OP, HARD>(a, T, c) * scale);
        } else {
          const f32x2 d = NEAR ? x[i] : add2(x[i], minus), y = fma2(d, cc, NEAR ? k2 : k0);
          r = mul2(exp2_2(y), BONUS ? fma2(kb, y, ka) : ka);
          if (HARD) r = fma2(exp2_2(fma2(d, l2, NEAR ? h2 : h1)), ce, r);
        }
        x[i] = CAP ? mul2(r, slope[i]) : r;
      }
      return vec_of<E>(x);
    };
    auto store = [&](int v, const uint4& w) {
      const int token = first_token + v * VE;
      if (whole && v >= full && v < end_full) {
        __stcs(reinterpret_cast<uint4*>(out + token), w);
      } else {
        float f[VE];
        floats_of<E>(w, f);
#pragma unroll
        for (int e = 0; e < VE; ++e)
          if (token + e >= 0 && token + e < V) out[token + e] = from_float<E>(f[e]);
      }
    };
    auto batch = [&](int v0, int most_v) {
      const uint4* at = zv + v0;
      uint4 w[GU];
#pragma unroll
      for (int i = 0; i < GU; ++i)
        if (i == 0 || v0 + i * NT < most_v) w[i] = __ldcs(at + i * NT);
#pragma unroll
      for (int i = 0; i < GU; ++i)
        if (i == 0 || v0 + i * NT < most_v) store(v0 + i * NT, grad(w[i]));
    };
    // (from the row's end: what was read last is still in the cache)
    const int whole_batches = max(0, (end_full - full - tid + NT - 1) / NT) / GU;
    int v0 = full + tid + whole_batches * GU * NT;
    if (v0 < end_full) batch(v0, end_full);
    for (v0 -= GU * NT; v0 >= full; v0 -= GU * NT) batch(v0, 0x7FFFFFFF);
    if (tid == 0 && full == 1 && nv > 0) store(0, grad(zv[0]));
    if (tid == NT - 1 && end_full < nv && end_full >= full) store(end_full, grad(zv[end_full]));
  };
  // (the row's named tokens have been read)
  constexpr std::true_type yes;
  constexpr std::false_type no;
  if (careful) pass(no, yes, no);
  else if (OP == POLICY && !CAP && bonus && near) pass(yes, no, yes);
  else if (OP == POLICY && !CAP && bonus) pass(yes, no, no);
  else if (near) pass(no, no, yes);
  else pass(no, no, no);
  __syncthreads();
  if (OP == POLICY && mine_t && tid == 0) out[t] = from_float<E>(grad_taken(T, a.bonus) * slope_t * scale);
  if (OP == DISTILL && warp == 0) {
    write_named<E, CAP, HARD>(a, T, names[lane], id, q, t, scale, out);
    if (HARD && mine_t && lane == 0 && !named_t) {
      const float u = capped<CAP>(a, zt, slope_t);
      out[t] = from_float<E>((grad_rest<OP, HARD>(a, T, u) - a.ce) * slope_t * scale);
    }
  }
}

// -------------------------------------------------------------------------------------------------------- launching
constexpr int MOST_SMEM = 200 * 1024;      // a block's dynamic shared memory

// the kernel may ask for as much shared memory as there is; once for each device
template <typename K>
bool allow(K kernel, std::atomic<unsigned long long>& done) {
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess) return false;
  const unsigned long long bit = 1ull << (device & 63);
  if (device < 64 && (done.load(std::memory_order_relaxed) & bit)) return true;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, MOST_SMEM) != cudaSuccess) return false;
  done.fetch_or(bit, std::memory_order_relaxed);
  return true;
}

template <typename E, Op OP, bool TOP, bool CAP, bool HARD, int NT>
int launch_block(const Row& a, int parts, int slice, int room, int smem, cudaStream_t stream) {
  static std::atomic<unsigned long long> done{0};
  auto kernel = row_kernel<E, OP, TOP, CAP, HARD, NT>;
  if (smem > 40 * 1024 && !allow(kernel, done)) return -400;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(static_cast<unsigned>(a.T) * parts);
  config.blockDim = dim3(NT);
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  cudaLaunchAttribute cluster;
  cluster.id = cudaLaunchAttributeClusterDimension;
  cluster.val.clusterDim.x = parts;
  cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
  config.attrs = &cluster;
  config.numAttrs = parts > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&config, kernel, a, slice, room) == cudaSuccess ? 0 : -400;
}

template <typename E, Op OP, bool TOP, bool CAP, bool HARD>
int launch_rows(const Row& a, cudaStream_t stream) {
  constexpr int VE = 16 / sizeof(E);
  const long bytes = static_cast<long>(a.V + VE - 1) * sizeof(E);
  // few rows: more blocks to each, down to 4 KB a block
  int parts = 1;
  while (parts < MOST_PARTS && ((static_cast<long>(a.T) * parts < FEW_BLOCKS && bytes > 4096l * parts) ||
                                (OP == DISTILL && bytes / 16 > static_cast<long>(MOST_SMEM - 64) * parts)))
    parts *= 2;
  if (static_cast<long>(a.T) * parts > 0x7FFFFFFFl) return -3;
  const long slice = ((a.V + VE - 1 + parts - 1) / parts + VE - 1) / VE * VE;
  // (where fewer threads than K have tokens, there are fewer than 2,048 of them and there is room for all)
  const int room = TOP ? (a.V < 2048 ? a.V : 32 + 3 * a.K / 2) : 0;
  const long smem = TOP ? static_cast<long>(room) * parts * 8 : OP == DISTILL ? (slice / VE + 15) / 16 * 16 : 0;
  if (smem > MOST_SMEM) return -5;
  const int s = static_cast<int>(slice), m = static_cast<int>(smem);
  if constexpr (TOP || CAP || OP == POLICY) {
    if ((TOP || CAP || a.out != nullptr) && slice * static_cast<long>(sizeof(E)) > LONG_ROW)
      return launch_block<E, OP, TOP, CAP, HARD, 512>(a, parts, s, room, m, stream);
  }
  return launch_block<E, OP, TOP, CAP, HARD, 256>(a, parts, s, room, m, stream);
}

template <typename E, bool CAP>
int launch_op(Op op, const Row& a, cudaStream_t stream) {
  if (op == SCORES) return a.K > 0 ? launch_rows<E, SCORES, true, CAP, false>(a, stream) : launch_rows<E, SCORES, false, CAP, false>(a, stream);
  if (op == POLICY) return launch_rows<E, POLICY, false, CAP, false>(a, stream);
  return a.ce != 0.f ? launch_rows<E, DISTILL, false, CAP, true>(a, stream) : launch_rows<E, DISTILL, false, CAP, false>(a, stream);
}

int run_rows(Op op, const RowArgs* r) {
  if (r->T <= 0 || r->V <= 0) return 0;
  if (r->T > 0x7FFFFFFFll || r->V > 0x7FFF0000ll || r->K < 0 || r->K > MOST_TOP || r->type < 0 || r->type > 2) return -3;
  if (!(r->tau > 0.0)) return -2;
  Row a;
  a.z = r->z; a.out = r->out; a.targets = r->targets; a.mask = r->mask;
  a.loss = r->loss; a.logprob = r->logprob; a.entropy = r->entropy; a.lse = r->lse;
  a.top_ids = r->top_ids; a.top_logprob = r->top_logprob;
  a.adv = r->adv; a.old = r->old; a.ref = r->ref; a.ids = r->ids; a.teacher = r->teacher;
  a.ldz = r->ldz; a.ldo = r->ldo; a.ignore = r->ignore;
  a.T = static_cast<int>(r->T); a.V = static_cast<int>(r->V); a.K = static_cast<int>(r->K); a.bucket = r->bucket != 0;
  a.tau = static_cast<float>(r->tau); a.inv_tau = static_cast<float>(1.0 / r->tau);
  a.c = static_cast<float>(1.4426950408889634 / r->tau);
  a.cap = static_cast<float>(r->cap); a.inv_cap = r->cap > 0.0 ? static_cast<float>(1.0 / r->cap) : 0.f;
  a.scale = static_cast<float>(r->scale);
  a.clip_low = static_cast<float>(r->clip_low); a.clip_high = static_cast<float>(r->clip_high);
  a.kl = static_cast<float>(r->kl); a.bonus = static_cast<float>(r->bonus); a.ce = static_cast<float>(r->ce);
  auto go = [&](auto e) {
    using E = decltype(e);
    return a.cap > 0.f ? launch_op<E, true>(op, a, r->stream) : launch_op<E, false>(op, a, r->stream);
  };
  return r->type == 0 ? go(bf16()) : r->type == 1 ? go(__half()) : go(float());
}

// ---------------------------------------------------------------------------------------- gradient of the scores
//   dz_j = (scale / tau) u'(z_j) [ -p_j (sum of the gradients of log p_t and of the alternatives + dH (log p_j + H)) + the gradients of j's own ]
//
// One pass, nothing between the tokens of a row: blocks of 256 threads take 1,024 pieces of 16 bytes, four a thread that are all asked for
// before the first is used.  The tokens with gradients of their own are written again behind the others of their block.  Bound by memory:
// 2048 x 128256 bf16 with a quarter of the rows left out 164 us (5.6 of 6.55 TB/s).
constexpr int GRAD_NT = 256, GRAD_EACH = 4;
template <typename E, bool CAP>
__global__ void __launch_bounds__(GRAD_NT) grad_kernel(Row a, const float* lse, const float* dlogprob, const float* dentropy, const float* dtop, int blocks) {
  constexpr int VE = Vec<E>::N, P = VE / 2;
  __shared__ float part[GRAD_NT / 32];
  __shared__ int id[MOST_TOP];
  __shared__ float gk[MOST_TOP];
  const int row = blockIdx.x / blocks, tid = threadIdx.x, V = a.V, K = a.K;
  const E* z = static_cast<const E*>(a.z) + row * a.ldz;
  E* out = static_cast<E*>(a.out) + row * a.ldo;
  const int lead = static_cast<int>((reinterpret_cast<uintptr_t>(z) & 15) / sizeof(E)), nv = (lead + V + VE - 1) / VE;
  const bool whole = (reinterpret_cast<uintptr_t>(out) & 15) / sizeof(E) == lead;
  const int v0 = (blockIdx.x - row * blocks) * (GRAD_NT * GRAD_EACH), from = v0 * VE - lead, to = from + GRAD_NT * GRAD_EACH * VE;
  const long t = a.targets ? a.targets[row] : -1;
  const bool on = row_on(a, row, t);
  uint4 w[GRAD_EACH];
  if (on) {
    const uint4* zv = reinterpret_cast<const uint4*>(z - lead);
#pragma unroll
    for (int i = 0; i < GRAD_EACH; ++i) {
      const int v = v0 + i * GRAD_NT + tid;
      if (v < nv) w[i] = zv[v];
    }
  }
  auto store = [&](int i, const uint4& u) {
    const int v = v0 + i * GRAD_NT + tid, token = v * VE - lead;
    if (v >= nv) return;
    if (whole && token >= 0 && token + VE <= V) {
      *reinterpret_cast<uint4*>(out + token) = u;
    } else {
      float f[VE];
      floats_of<E>(u, f);
#pragma unroll
      for (int e = 0; e < VE; ++e)
        if (token + e >= 0 && token + e < V) out[token + e] = from_float<E>(f[e]);
    }
  };
  if (!on) {
#pragma unroll
    for (int i = 0; i < GRAD_EACH; ++i) store(i, make_uint4(0, 0, 0, 0));
    return;
  }
  // thread k < K: the alternatives; thread K: the given token
  int mine = -1;
  float g = 0.f;
  const float gt = dlogprob ? dlogprob[row] : 0.f;
  if (tid < K) {
    const long k = a.top_ids[(size_t)row * K + tid];
    if (k >= 0 && k < V) {
      mine = static_cast<int>(k);
      g = dtop[(size_t)row * K + tid];
    }
    id[tid] = mine;
    gk[tid] = g;
  }
  if (tid == K && dlogprob) {
    mine = static_cast<int>(t);
    g = gt;
  }
  const bool here = mine >= from && mine < to && mine >= 0;
  const float zm = here ? to_float(z[mine]) : 0.f;
  if (K > 0) {
    const float s = warp_sum(g);
    if ((tid & 31) == 0) part[tid >> 5] = s;
  }
  const bool some = __syncthreads_or(here);                   // (and what is read by index has been read)
  float sum = gt;
  if (K > 0) {
    sum = part[0];
#pragma unroll
    for (int i = 1; i < GRAD_NT / 32; ++i) sum += part[i];
  }
  const float dh = dentropy ? dentropy[row] : 0.f, l = lse[row], scale = a.scale * a.inv_tau;
  const float ka = -sum - (dentropy ? dh * a.entropy[row] : 0.f);
  auto at = [&](float u, float slope, float own) {
    const float y = fmaf(u, a.inv_tau, -l) * LOG2E, p = ex2(y);               // (one rounding of the difference)
    return ((dentropy ? p * (ka - dh * LN2 * max_nan(y, -256.f)) : p * ka) + own) * slope * scale;
  };
  const bool careful = dentropy && (CAP || !(l > Vec<E>::LOW * 0.9f * a.inv_tau) || a.inv_tau < 0.05f);
  const f32x2 it = pair(a.inv_tau, a.inv_tau), ml = pair(-l, -l), l2 = pair(LOG2E, LOG2E), fa = pair(ka * scale, ka * scale);
  const f32x2 fb = pair(-dh * LN2 * scale, -dh * LN2 * scale);
#pragma unroll
  for (int i = 0; i < GRAD_EACH; ++i) {
    if (v0 + i * GRAD_NT + tid >= nv) break;
    f32x2 x[P], slope[P];
    pairs_of<E>(dentropy && !careful ? vec_floor<E>(w[i]) : w[i], x);
    if (CAP) cap_pairs<E, true>(a, x, slope);
#pragma unroll
    for (int j = 0; j < P; ++j) {
      f32x2 r;
      if (careful) {
        float b, c;
        split(x[j], b, c);
        r = pair(at(b, 1.f, 0.f), at(c, 1.f, 0.f));
      } else {
        const f32x2 y = mul2(fma2(x[j], it, ml), l2);
        r = mul2(exp2_2(y), dentropy ? fma2(fb, y, fa) : fa);
      }
      x[j] = CAP ? mul2(r, slope[j]) : r;
    }
    store(i, vec_of<E>(x));
  }
  if (!some) return;
  __syncthreads();
  if (here) {                                                 // (of a token twice both write the same)
    float own = 0.f, slope;
    for (int k = 0; k < K; ++k) own += id[k] == mine ? gk[k] : 0.f;
    if (dlogprob && mine == t) own += gt;
    const float u = capped<CAP>(a, zm, slope);
    out[mine] = from_float<E>(at(u, slope, own));
  }
}

template <typename E>
int launch_grad(const Row& a, const GradArgs* r) {
  constexpr int each = GRAD_NT * GRAD_EACH * Vec<E>::N;
  const int blocks = (a.V + Vec<E>::N - 1 + each - 1) / each;
  if (static_cast<long>(a.T) * blocks > 0x7FFFFFFFl) return -3;
  auto kernel = a.cap > 0.f ? grad_kernel<E, true> : grad_kernel<E, false>;
  kernel<<<a.T * blocks, GRAD_NT, 0, r->stream>>>(a, r->lse, r->dlogprob, r->dentropy, r->dtop, blocks);
  return cudaGetLastError() == cudaSuccess ? 0 : -400;
}

}  // namespace

extern "C" {

int ftb_token_loss_error(void) {
  int h[2] = {0, 0};
  cudaMemcpyFromSymbol(&h[0], ftb::g_error_word, sizeof(int));
  cudaMemcpyFromSymbol(&h[1], ftb::g_error_where, sizeof(int));
  if (h[0] != 0) {
    const int z = 0;
    cudaMemcpyToSymbol(ftb::g_error_word, &z, sizeof(int));
    cudaMemcpyToSymbol(ftb::g_error_where, &z, sizeof(int));
  }
  return h[0] * 1000 + h[1];
}

int ftb_token_scores(const RowArgs* a) { return run_rows(SCORES, a); }
int ftb_policy_loss(const RowArgs* a) { return run_rows(POLICY, a); }
int ftb_distill_loss(const RowArgs* a) { return run_rows(DISTILL, a); }

int ftb_token_scores_bwd(const GradArgs* r) {
  if (r->T <= 0 || r->V <= 0) return 0;
  if (r->T > 0x7FFFFFFFll || r->V > 0x7FFF0000ll || r->K < 0 || r->K > MOST_TOP || r->type < 0 || r->type > 2) return -3;
  if (!(r->tau > 0.0)) return -2;
  Row a = {};
  a.z = r->z; a.out = r->out; a.targets = r->targets; a.mask = r->mask;
  a.entropy = const_cast<float*>(r->entropy); a.top_ids = const_cast<int64_t*>(r->top_ids);
  a.ldz = r->ldz; a.ldo = r->ldo; a.ignore = r->ignore;
  a.T = static_cast<int>(r->T); a.V = static_cast<int>(r->V); a.K = static_cast<int>(r->K);
  a.inv_tau = static_cast<float>(1.0 / r->tau);
  a.c = static_cast<float>(1.4426950408889634 / r->tau);
  a.cap = static_cast<float>(r->cap); a.inv_cap = r->cap > 0.0 ? static_cast<float>(1.0 / r->cap) : 0.f;
  a.scale = static_cast<float>(r->scale);
  return r->type == 0 ? launch_grad<bf16>(a, r) : r->type == 1 ? launch_grad<__half>(a, r) : launch_grad<float>(a, r);
}

}  // extern "C"
