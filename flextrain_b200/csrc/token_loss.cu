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
// NaN, as does one with a NaN or +inf.  Compiled without fast math: tanh, log2 and divisions are the rounded ones.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
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
// relative error (2e-9; with the roundings of fp32 it is some 2^-23.5); beyond it 1 - 2 / (1 + e^2y), whose slope is formed without 1 - t^2.
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
template <int NT>
__device__ __forceinline__ float block_max(float v, float* sh) {
  __syncthreads();
#pragma unroll
  for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(~0u, v, o));
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  v = sh[0];
#pragma unroll
  for (int i = 1; i < NT / 32; ++i) v = fmaxf(v, sh[i]);
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
      A += none ? 0.f : down * (rec[r].A + rec[r].S * d);
      if (OP == SCORES) t.low = r == 0 ? rec[r].low : min(t.low, rec[r].low);
    }
    const float yt = (ut - t.M) * a.c, et = has ? ex2(yt) : 0.f, S = O + et;
    if (has) A += et * max_nan(yt, -256.f);
    t.lS = S > 0.f ? log2f(S) : NAN;                          // no finite logit (or a NaN): all that follows is NaN
    // a token that has most of the row: the others' sum by itself, so that a small log p keeps its digits
    const bool most = has && ut >= rest && S > 0.f;
    const float ln_S = most ? log1pf(O) : t.lS * LN2;
    t.lp = most ? -ln_S : (yt - t.lS) * LN2;
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
      const bool none = p.m == -INFINITY, no_names = p.B == -INFINITY;
      others += none ? 0.f : p.S * ex2((p.m - base) * a.c);
      if (HARD) S1 += none ? 0.f : p.S1 * ex2((p.m - t.M) * LOG2E);
      named += no_names ? 0.f : p.En * ex2((p.B - t.M) * a.c);
      if (HARD) S1 += no_names ? 0.f : p.En1 * ex2((p.B - t.M) * LOG2E);
      kl += no_names || p.Q == 0.f ? 0.f : p.Q * (t.M - p.B) * a.inv_tau;
      kl += p.kl;
      Q += p.Q;
    }
    const float S = others * (rest == -INFINITY ? 0.f : ex2((base - t.M) * a.c)) + named;
    t.lS = S > 0.f ? log2f(S) : NAN;
    // q (log q - log p), where log p = (u - M) / tau - ln S and a part has (u - B) / tau
    if (Q != 0.f) kl += Q * t.lS * LN2;
    t.base = base;
    t.k0 = (base - t.M) * a.c - t.lS;
    t.share = a.bucket ? Q + qr : (Q != 0.f ? 1.f : 0.f);
    t.ka = t.share;
    if (a.bucket) {
      if (rest != -INFINITY && qr > 0.f) {
        const float l2 = (base - t.M) * a.c + log2f(others) - t.lS;       // log2 of the student's share of the others
        kl += qr * (logf(qr) - l2 * LN2);
        if (l2 > -60.f) {
          t.ka = t.share - qr / ex2(l2);
        } else {                                              // (p itself is nothing beside the teacher's share there)
          t.k0 = -log2f(others);
          t.ka = -qr;
        }
      } else {                                                // nothing is left beside the named tokens
        t.share = t.ka = Q;
      }
    }
    float L = (1.f - a.ce) * a.tau * a.tau * kl;
    if (HARD) {
      t.h0 = S1 > 0.f ? log2f(S1) : NAN;
      L -= a.ce * ((ut - t.M) * LOG2E - t.h0) * LN2;
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
  const float v = (1.f - a.ce) * a.tau * (ex2((u - t.M) * a.c - t.lS) * t.share - q);
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


// ------------------------------------------------------------------------------------------- rows in shared memory
// A cluster of up to eight blocks takes a row and keeps it in their shared memory, so that memory is read once and the gradient is the
// only other traffic: a piece of 16 bytes on for each block, by one bulk copy, rows off the 16-byte grid with the pieces that they
// begin and end in.  The blocks exchange their parts of the totals through one another's shared memory, at one meeting of the cluster
// (one more for alternatives).  Several blocks an SM: while one waits for its piece others compute.
//
// Alternatives: a bound that at least K tokens are not below, from each block's largest ones by thread (found by halving an interval of
// whole numbers that are in the order of the floats); tokens from the highest of the blocks' bounds on go to one block, which ranks
// them.  Where they are too many (thousands of equal logits) the cluster halves the interval of (logit, index) of all tokens until
// exactly K are left.

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
__device__ __forceinline__ bool sent_wait(uint64_t* bar, uint32_t parity, int where) {
  for (int again = 0; again < 2; ++again) {
    for (uint32_t it = 0; it < FTB_WAIT_LIMIT; ++it) {
      uint32_t ok;
      asm volatile(
          "{\n.reg .pred p;\n"
          "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n"
          "selp.u32 %0, 1, 0, p;\n}\n"
          : "=r"(ok)
          : "r"(ftb::smem_u32(bar)), "r"(parity)
          : "memory");
      if (ok) return true;
    }
    ftb::set_error(1, where);
  }
  return false;
}
// A cluster that has not begun is taken over by this one, or none is: the answer's 16 bytes are counted on a barrier.  first: the index
// of its first block, -1 where there was none (after which there is none any more).
__device__ __forceinline__ void take_over(void* answer, uint64_t* bar) {
  ftb::fence_proxy_async();
  ftb::mbar_expect_tx(bar, 16);
  asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(ftb::smem_u32(answer)),
               "r"(ftb::smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ int taken_over(const void* answer) {
  uint32_t got, first;
  asm volatile(
      "{\n.reg .b128 h;\n.reg .pred p;\n"
      "ld.shared.b128 h, [%2];\n"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, h;\n"
      "selp.u32 %0, 1, 0, p;\n"
      "mov.u32 %1, 0;\n"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, h;\n}\n"
      : "=r"(got), "=r"(first)
      : "r"(ftb::smem_u32(answer))
      : "memory");
  return got ? static_cast<int>(first) : -1;
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
      float c, d, sc, sd;
      split(x[i], c, d);
      c = capped<true>(a, c, sc);
      d = capped<true>(a, d, sd);
      x[i] = pair(c, d);
      if (SLOPE) slope[i] = pair(sc, sd);
    }
  }
}

__device__ __forceinline__ u64 key_of(float z, int token) { return static_cast<u64>(order_of(z)) << 32 | static_cast<uint32_t>(~token); }
__device__ __forceinline__ float logit_of(uint32_t order) {
  return order == NAN_ORDER ? NAN : __uint_as_float(order & 0x80000000u ? order & 0x7FFFFFFFu : ~order);
}

// NW threads work on the tokens; one warp more begins copies, takes the named tokens out and exchanges the parts, so that what it does
// for a row lies beside the others' passes.  A cluster that is done with a row takes over the row of one that has not begun (``more``:
// there are some), since beginning blocks costs as long as their work on a row: its first block asks for it while the others are at
// work and tells them; a copy begins as soon as the last row's tokens are no longer read.
template <int NW>
__host__ __device__ constexpr int slice_blocks() { return NW == 128 ? 6 : NW == 256 ? 3 : 1; }      // of an SM
template <typename E, Op OP, bool TOP, bool CAP, bool HARD, int NW>
__global__ void __launch_bounds__(NW + 32, slice_blocks<NW>()) slice_kernel(Row a, int slice, int room, int more) {
  constexpr int VE = Vec<E>::N, P = VE / 2, W = NW / 32, NT = NW + 32;
  extern __shared__ __align__(128) unsigned char buf[];
  const bool early = OP == SCORES ? !TOP : a.out == nullptr;  // nothing reads a row's tokens after its sums
  __shared__ __align__(8) uint64_t bar, sent[2], told[2], answered;
  __shared__ __align__(16) int4 next[2];                      // a row to come (-1: none), whether it counts, its given token
  __shared__ __align__(16) int4 answer;
  __shared__ int gave_up, found;
  __shared__ float sh[32], most[W], least[W], sums[3][W];
  __shared__ Part rec[2][MOST_PARTS], own;
  __shared__ Totals fin;
  __shared__ int count[2][MOST_PARTS];
  __shared__ uint32_t bounds[MOST_PARTS];
  __shared__ int id[OP == DISTILL ? MOST_TOP : 1];
  __shared__ float q[OP == DISTILL ? MOST_TOP : 1];
  E* zs = reinterpret_cast<E*>(buf);
  const uint4* zv = reinterpret_cast<const uint4*>(buf);

  int rank, parts;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(parts));
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, V = a.V, K = a.K;
  const bool works = warp < W, takes = more && rank == 0;
  if (tid == NW) {
    gave_up = found = 0;
    ftb::mbar_init(&bar, 1);
    ftb::mbar_init(&answered, 1);
    for (int i = 0; i < 2; ++i) {
      ftb::mbar_init(&sent[i], 1);
      ftb::mbar_init(&told[i], 1);
    }
    ftb::fence_barrier_init();
  }
  cluster_arrive_relaxed();                                   // (the others may be sent to once all have begun)
  if (tid < 2 * MOST_PARTS && tid % MOST_PARTS >= parts) rec[tid / MOST_PARTS][tid % MOST_PARTS] = no_part();
  int row = blockIdx.x / parts, answers = 0, loads = 0;
  long t = a.targets ? a.targets[row] : -1;
  bool on = row_on(a, row, t);
  // the row from the 16-byte piece that it begins in: ``lead`` elements before it, this block's from ``lo`` on, in pieces
  auto lead_of = [&](int r) { return static_cast<int>((reinterpret_cast<uintptr_t>(static_cast<const E*>(a.z) + r * a.ldz) & 15) / sizeof(E)); };
  auto count_of = [&](int lead) { return max(0, min(lead + V - rank * slice, slice)); };
  auto load = [&](int r) {                                    // by one thread
    const int lead = lead_of(r), nv = (count_of(lead) + VE - 1) / VE;
    if (nv > 0) {
      ftb::fence_proxy_async();
      ftb::mbar_expect_tx(&bar, nv * 16);
      ftb::bulk_load_g2s(buf, static_cast<const E*>(a.z) + r * a.ldz - lead + rank * slice, nv * 16, &bar);
    }
  };
  if (tid == NW && on) load(row);
  __syncthreads();
  cluster_wait();
  // Where nothing waits for a row's totals its last part is left for the next row's passes (by the warp that exchanges).
  int last = -1, last_it = 0;
  float last_qr = 0.f;
  Given last_given = {};
  auto finish = [&] {
    if (last < 0) return;
    sent_wait(&sent[last_it & 1], (last_it >> 1) & 1, 3);
    total<OP, HARD>(a, last, rec[last_it & 1], last_qr, last_given, rank == 0, &fin);
    last = -1;
  };

  for (int it = 0; row >= 0; ++it) {
    const E* z = static_cast<const E*>(a.z) + row * a.ldz;
    E* out = static_cast<E*>(a.out) + row * a.ldo;
    const int lo = rank * slice, lead = lead_of(row), n = count_of(lead), nv = (n + VE - 1) / VE, first_token = lo - lead;
    const bool whole = OP != SCORES && (reinterpret_cast<uintptr_t>(out) & 15) / sizeof(E) == lead;       // the gradient's pieces lie as the logits' do
    const int now = it & 1, then = now ^ 1;
    const uint32_t told_parity = (it >> 1) & 1;
    if (tid == NW) {
      ftb::mbar_expect_tx(&sent[now], parts * sizeof(Part));
      if (more) ftb::mbar_expect_tx(&told[then], 16);
    }
    // The next row: asked for when this row's tokens are here (by then all blocks that find room have begun), told to the cluster.
    auto ask = [&] {
      if (takes && tid == NW) take_over(&answer, &answered);
    };
    auto tell = [&] {
      if (!takes || works) return;
      int4 v = make_int4(-1, 0, 0, 0);
      if (lane == 0) {
        const int first = sent_wait(&answered, answers & 1, 5) ? taken_over(&answer) : -1;
        if (first >= 0) {
          v.x = first / parts;
          const long given = a.targets ? a.targets[v.x] : -1;
          v.y = row_on(a, v.x, given);
          v.z = static_cast<int>(given);                      // (a token where the row counts)
        }
      }
      ++answers;
      v = make_int4(__shfl_sync(~0u, v.x, 0), __shfl_sync(~0u, v.y, 0), __shfl_sync(~0u, v.z, 0), 0);
      if (lane < parts)
        send16(in_cluster(&next[then], lane), make_uint4(v.x, v.y, v.z, 0), in_cluster(&told[then], lane));
    };
    auto load_next = [&] {                                    // by the warp
      if (!more) return;
      if (sent_wait(&told[then], told_parity, 6) && lane == 0 && next[then].x >= 0 && next[then].y) load(next[then].x);
    };
    auto send_part = [&](const Part& p) {                     // to every block of the cluster, this one among them
      if (lane == 0) own = p;
      __syncwarp();
      if (lane < parts * PART_PIECES) {
        const int to = lane / PART_PIECES, piece = lane - to * PART_PIECES;
        send16(in_cluster(reinterpret_cast<const uint4*>(&rec[now][rank]) + piece, to), reinterpret_cast<const uint4*>(&own)[piece],
               in_cluster(&sent[now], to));
      }
    };
    auto step = [&] {                                         // by all
      const bool known = more && sent_wait(&told[then], told_parity, 6);
      row = known ? next[then].x : -1;
      on = known && next[then].y;
      t = on && a.targets ? next[then].z : -1;
    };
    if (!on) {
      // (nothing is exchanged, but no block may be two rows ahead of another, nor of a thread of its own that has not read where to go)
      __syncthreads();
      ask();
      if (works && OP != SCORES && a.out)
        for (int v = tid; v < nv; v += NW) {
          const int token = first_token + v * VE;
          if (whole && token >= 0 && token + VE <= V) {
            *reinterpret_cast<uint4*>(out + token) = make_uint4(0, 0, 0, 0);
          } else {
            for (int e = 0; e < VE; ++e)
              if (token + e >= 0 && token + e < V) out[token + e] = from_float<E>(0.f);
          }
        }
      if (rank == 0) row_off<OP>(a, row);
      if (!works) {
        finish();
        tell();
        send_part(Part{});
        load_next();
        sent_wait(&sent[now], (it >> 1) & 1, 3);
      }
      step();
      continue;
    }
    const long given = t;
    float qr = 0.f;
    bool named_t = false;
    Named mine;
    Given policy = {};
    if (OP == POLICY && !works) policy = given_of(a, row);
    if (OP == DISTILL && !works) qr = teacher_of(a, row, t, id, q, mine, named_t);
    if (nv > 0) {
      if (!ftb::mbar_wait(&bar, loads & 1, &gave_up, 1)) {    // (reported; the copy gets as long again before the block goes on)
        int again = 0;
        ftb::mbar_wait(&bar, loads & 1, &again, 2);
      }
      ++loads;
    }

    // what lies around the row is no token; named tokens by themselves
    const int at_t = static_cast<int>(t) - first_token;         // where the given token lies
    const bool mine_t = a.targets && at_t >= 0 && at_t < n;
    float zt = 0.f;
    if (!works) {
      if (lane < VE) {
        if (lo + lane < lead && lane < nv * VE) zs[lane] = from_float<E>(-INFINITY);
        if (n + lane < nv * VE) zs[n + lane] = from_float<E>(-INFINITY);
      }
      if (mine_t) zt = to_float(zs[at_t]);
      __syncwarp();
      if (OP != DISTILL && mine_t && lane == 0) zs[at_t] = from_float<E>(-INFINITY);
      if (OP == DISTILL) {
        typedef typename std::conditional<sizeof(E) == 2, uint16_t, uint32_t>::type Bits;
        Bits* tag = reinterpret_cast<Bits*>(buf);
#pragma unroll
        for (int j = 0; j < ENTRIES; ++j) {
          mine.here[j] = mine.id[j] >= first_token && mine.id[j] < first_token + n && mine.id[j] >= 0;
          if (mine.here[j]) mine.z[j] = to_float(zs[mine.id[j] - first_token]);
        }
        __syncwarp();
#pragma unroll
        for (int j = 0; j < ENTRIES; ++j)                       // of entries of one token, the one whose number stays in its place
          if (mine.here[j]) tag[mine.id[j] - first_token] = static_cast<Bits>(lane + 32 * j);
        __syncwarp();
#pragma unroll
        for (int j = 0; j < ENTRIES; ++j) mine.first[j] = mine.here[j] && tag[mine.id[j] - first_token] == static_cast<Bits>(lane + 32 * j);
        __syncwarp();
#pragma unroll
        for (int j = 0; j < ENTRIES; ++j)
          if (mine.here[j]) zs[mine.id[j] - first_token] = from_float<E>(-INFINITY);
      }
      ftb::fence_proxy_async();                                 // (the next copy comes after these)
      ask();
    }
    __syncthreads();

    // largest of each thread, of the block
    float mt = -INFINITY;
    Part p = {};
    p.B = -INFINITY;
    if (works) {
      uint32_t m2 = Vec<E>::NONE;
#pragma unroll 4
      for (int v = tid; v < nv; v += NW) m2 = Vec<E>::max2(m2, vec_max<E>(zv[v]));
      mt = Vec<E>::top(m2);
      const float w = warp_max(mt);
      if (lane == 0) most[warp] = w;
      if (TOP) {
        float l = tid < nv ? mt : INFINITY;
#pragma unroll
        for (int o = 16; o; o >>= 1) l = fminf(l, __shfl_xor_sync(~0u, l, o));
        if (lane == 0) least[warp] = l;
      }
    } else if (OP == DISTILL) {
      named_part<CAP, HARD>(a, mine, p);
    }
    __syncthreads();
    if (!works) finish();                                     // (before the cluster is told: all have read what they were told last)
    tell();
    float mz = most[0];
#pragma unroll
    for (int w = 1; w < W; ++w) mz = fmaxf(mz, most[w]);
    const float um = mz == -INFINITY ? mz : capped<CAP>(a, mz), base = mz == -INFINITY ? 0.f : um;

    // sums relative to it.  16-bit logits: the exponent's argument by one fused operation, relative to the rounded product of base and c; what
    // the rounding is goes into the sums at the end.  (Bases whose product leaves no digits: as fp32 logits.)
    float off = 0.f, off1 = 0.f;                                // base c and base log2 e less what the sums are relative to
    if (works) {
      f32x2 S = 0, S1 = 0;
      float A = 0.f;
      const float kb = base * a.c, kb1 = base * LOG2E;
      const bool fused = sizeof(E) == 2 && fabsf(kb) < 0x1p24f && fabsf(kb1) < 0x1p24f;
      const f32x2 minus = pair(-base, -base), cc = pair(a.c, a.c), l2 = pair(LOG2E, LOG2E), mk = pair(-kb, -kb), mk1 = pair(-kb1, -kb1);
      auto pass = [&](auto f) {
        constexpr bool FUSED = decltype(f)::value;
#pragma unroll 2
        for (int v = tid; v < nv; v += NW) {
          const uint4 w = zv[v];
          f32x2 x[P], slope[P], part = 0;
          pairs_of<E>(w, x);
          if (CAP) cap_pairs<E, false>(a, x, slope);
#pragma unroll
          for (int i = 0; i < P; ++i) {
            f32x2 y, y1;
            if (FUSED) {
              y = fma2(x[i], cc, mk);
              if (HARD) y1 = fma2(x[i], l2, mk1);
            } else {
              const f32x2 d = add2(x[i], minus);
              y = mul2(d, cc);
              if (HARD) y1 = mul2(d, l2);
            }
            const f32x2 e = exp2_2(y);
            S = add2(S, e);
            if (OP != DISTILL) part = fma2(e, y, part);
            if (HARD) S1 = add2(S1, exp2_2(y1));
          }
          if (OP != DISTILL) {
            float b, c;
            split(part, b, c);
            b += c;
            if (b != b) {                                       // (a logit of -inf: nothing times minus infinity)
              float g[VE];
              floats_of<E>(w, g);
              b = 0.f;
#pragma unroll
              for (int e = 0; e < VE; ++e) {
                const float u = capped<CAP>(a, g[e]), y = FUSED ? fmaf(u, a.c, -kb) : (u - base) * a.c;
                b += ex2(y) * max_nan(y, -256.f);
              }
            }
            A += b;
          }
        }
      };
      if (fused) {
        pass(std::true_type());
        off = fmaf(base, a.c, -kb);
        off1 = fmaf(base, LOG2E, -kb1);
      } else {
        pass(std::false_type());
      }
      auto back = [](float o) { return fabsf(o) < 1e-4f ? fmaf(-o, LN2, 1.f) : ex2(-o); };      // 2^-off
      float b, c;
      split(S, b, c);
      b += c;
      const float down = back(off);
      const float s = warp_sum(b * down);
      if (lane == 0) sums[0][warp] = s;
      if (OP != DISTILL) {
        A = warp_sum(down * (A - off * b));
        if (lane == 0) sums[1][warp] = A;
      }
      if (HARD) {
        split(S1, b, c);
        b = warp_sum((b + c) * back(off1));
        if (lane == 0) sums[2][warp] = b;
      }
    }
    // the largest of at least ``want`` threads are not below it, and of not many more
    auto bound_of = [&](int want) {
      float l = least[0];
#pragma unroll
      for (int w = 1; w < W; ++w) l = fminf(l, least[w]);
      uint32_t low = order_of(l), high = order_of(mz) + 1;
      const uint32_t key = works && tid < nv ? order_of(mt) : 0;
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
      else if (min(nv, NW) >= share) low = bound_of(share);
    }
    __syncthreads();
    float slope_t = 1.f;
    if (!works) {
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
      send_part(p);
      last = row, last_it = it, last_qr = qr, last_given = policy;
      if (early) load_next();
      else finish();
    }
    if (early) {
      step();
      continue;
    }
    __syncthreads();
    const Totals T = fin;

    if (OP == SCORES) {
      // tokens from the bound on to every block, which then ranks its own among them
      u64* taken = reinterpret_cast<u64*>(buf + slice * static_cast<int>(sizeof(E)));
      const bool broken = T.lS != T.lS;                         // (a thread's largest leaves NaN out)
      u64* ours = taken + rank * room;
      // A warp takes the threads with such tokens one by one, half a piece a lane.
      auto collect = [&](u64 bound, bool all) {
        typedef typename std::conditional<sizeof(E) == 2, uint2, float2>::type Half;
        const uint32_t order = static_cast<uint32_t>(bound >> 32);
        auto give = [&](float f, int token) {
          const u64 key = key_of(f, token);
          if (key < bound) return;
          const int i = atomicAdd(&found, 1);
          if (i < room) ours[i] = key;
        };
        if (tid == NW && mine_t) give(zt, static_cast<int>(t));
        uint32_t those = __ballot_sync(~0u, works && tid < nv && (all || order_of(mt) >= order));
        while (those) {
          const int first = (warp << 5) + __ffs(those) - 1;
          those &= those - 1;
          for (int h = lane; h < 2 * ((nv - first + NW - 1) / NW); h += 32) {
            const int at = (first + (h >> 1) * NW) * VE + (h & 1) * (VE / 2);
            const Half w = *reinterpret_cast<const Half*>(zs + at);
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
              if (order_of(f[e]) >= order && token >= 0 && token < V && token != t) give(f[e], token);
            }
          }
        }
        __syncthreads();
        const int have = min(found, room);
        for (int i = tid; i < have * parts; i += NT) {
          const int to = i % parts, c = i / parts;
          if (to != rank) put64(in_cluster(ours + c, to), ours[c]);
        }
        if (tid < parts) put32(in_cluster(&count[0][rank], tid), found);
        cluster_arrive();
        cluster_wait();
        bool over = false;
        for (int r = 0; r < parts; ++r) over |= count[0][r] > room;
        return over;
      };
      u64 bound = static_cast<u64>(T.low) << 32;
      bool over = collect(bound, T.low == 0 || broken);
      if (over) {
        // the blocks' tokens differ: the highest of bounds that K threads of a block each are not below
        const uint32_t mine_low = min(nv, NW) >= K ? bound_of(K) : 0;
        if (tid < parts) put32(in_cluster(&bounds[rank], tid), mine_low);
        if (tid == 0) found = 0;
        cluster_arrive();                                       // (all have read the last counts)
        cluster_wait();
        uint32_t highest = T.low;
        for (int r = 0; r < parts; ++r) highest = max(highest, bounds[r]);
        bound = static_cast<u64>(highest) << 32;
        over = collect(bound, highest == 0 || broken);
      }
      if (over) {
        u64 below = 0, above = ~0ull;                           // at least K keys are not below the one, fewer not below the other
        for (int it = 0; above - below > 1; ++it) {
          const u64 mid = below + (above - below) / 2;
          int c = tid == NW && mine_t && key_of(zt, static_cast<int>(t)) >= mid;
          if (works)
            for (int v = tid; v < nv; v += NW) {
              float f[VE];
              floats_of<E>(zv[v], f);
#pragma unroll
              for (int e = 0; e < VE; ++e) {
                const int token = first_token + v * VE + e;
                c += token >= 0 && token < V && token != t && key_of(f[e], token) >= mid;
              }
            }
          c = static_cast<int>(block_sum<NT>(static_cast<float>(c), sh));           // (whole numbers below 2^24)
          if (tid < parts) put32(in_cluster(&count[1 - (it & 1)][rank], tid), c);
          cluster_arrive();
          cluster_wait();
          int sum = 0;
          for (int r = 0; r < parts; ++r) sum += count[1 - (it & 1)][r];
          if (sum >= K) below = mid;
          else above = mid;
          if (sum == K) break;
        }
        if (tid == 0) found = 0;
        cluster_arrive();                                       // (all have read the last counts)
        cluster_wait();
        bound = below;
        collect(bound, true);
      }
      if (!works) load_next();                                // (the row was read when the counts were exchanged)
      // eight threads to a token, one for each block's
      for (int i = tid / MOST_PARTS; i < (count[0][rank] + NT / MOST_PARTS - 1) / (NT / MOST_PARTS) * (NT / MOST_PARTS); i += NT / MOST_PARTS) {
        const int r = tid % MOST_PARTS, others = r < parts ? count[0][r] : 0;
        const bool valid = i < count[0][rank];
        const u64 key = valid ? taken[rank * room + i] : ~0ull;
        int above = 0;
#pragma unroll 4
        for (int j = 0; j < others; ++j) above += taken[r * room + j] > key;
#pragma unroll
        for (int o = MOST_PARTS / 2; o; o >>= 1) above += __shfl_xor_sync(~0u, above, o);
        if (valid && r == 0 && above < K) {
          const int token = static_cast<int>(~static_cast<uint32_t>(key));
          a.top_ids[(size_t)row * K + above] = token;
          a.top_logprob[(size_t)row * K + above] =
              token == t ? T.lp : ((capped<CAP>(a, logit_of(static_cast<uint32_t>(key >> 32))) - T.M) * a.c - T.lS) * LN2;
        }
      }
      if (tid == 0) found = 0;
      step();
      continue;
    }

    const float scale = OP == DISTILL ? a.scale : a.scale * a.inv_tau;
    if (works) {
      const bool bonus = OP == POLICY && T.kb != 0.f;
      // One by one: entropy's gradient where a cap leaves -inf (elsewhere it is brought to a number that has no p log p, unless all of the row
      // are such), and logits so large that their differences have to be formed first.
      const bool careful = (bonus && (CAP || !(T.M > Vec<E>::LOW * 0.9f) || a.inv_tau < 0.05f)) ||
                           (sizeof(E) == 2 && !(fabsf(T.base) * fmaxf(a.c, LOG2E) < 4096.f && fabsf(T.M) * LOG2E < 4096.f));
      const f32x2 minus = pair(-T.base, -T.base), cc = pair(a.c, a.c), k0 = pair(T.k0, T.k0);
      const float fa = OP == POLICY ? T.ka * scale : (1.f - a.ce) * a.tau * T.ka * scale, fb = T.kb * LN2 * scale;
      const float f0 = fmaf(-T.base, a.c, T.k0), f1 = fmaf(-T.M, LOG2E, -T.h0);
      const f32x2 ka = pair(fa, fa), kb = pair(fb, fb), kc = pair(f0, f0), kh = pair(f1, f1);
      const f32x2 minus_m = pair(-T.M, -T.M), l2 = pair(LOG2E, LOG2E), h0 = pair(-T.h0, -T.h0), ce = pair(a.ce * scale, a.ce * scale);
      auto pass = [&](auto with_bonus, auto with_care) {
        constexpr bool BONUS = decltype(with_bonus)::value, CARE = decltype(with_care)::value;
#pragma unroll 2
        for (int v = tid; v < nv; v += NW) {
          f32x2 x[P], slope[P];
          pairs_of<E>(BONUS && !CARE ? vec_floor<E>(zv[v]) : zv[v], x);
          if (CAP) cap_pairs<E, true>(a, x, slope);
#pragma unroll
          for (int i = 0; i < P; ++i) {
            f32x2 r;
            if (CARE) {
              float b, c;
              split(x[i], b, c);
              r = pair(grad_rest<OP, HARD>(a, T, b) * scale, grad_rest<OP, HARD>(a, T, c) * scale);
            } else {
              const f32x2 y = sizeof(E) == 2 ? fma2(x[i], cc, kc) : fma2(add2(x[i], minus), cc, k0);
              r = mul2(exp2_2(y), BONUS ? fma2(kb, y, ka) : ka);
              if (HARD) r = fma2(exp2_2(sizeof(E) == 2 ? fma2(x[i], l2, kh) : fma2(add2(x[i], minus_m), l2, h0)), ce, r);
            }
            x[i] = CAP ? mul2(r, slope[i]) : r;
          }
          const uint4 w = vec_of<E>(x);
          const int token = first_token + v * VE;
          if (whole && token >= 0 && token + VE <= V) {
            *reinterpret_cast<uint4*>(out + token) = w;
          } else {
            float f[VE];
            floats_of<E>(w, f);
#pragma unroll
            for (int e = 0; e < VE; ++e)
              if (token + e >= 0 && token + e < V) out[token + e] = from_float<E>(f[e]);
          }
        }
      };
      if (careful) pass(std::false_type(), std::true_type());
      else if (OP == POLICY && !CAP && bonus) pass(std::true_type(), std::false_type());
      else pass(std::false_type(), std::false_type());
    }
    __syncthreads();
    step();
    if (works) continue;
    load_next();
    if (OP == POLICY && mine_t && lane == 0) out[given] = from_float<E>(grad_taken(T, a.bonus) * slope_t * scale);
    if (OP == DISTILL) {
      write_named<E, CAP, HARD>(a, T, mine, id, q, given, scale, out);
      if (HARD && mine_t && lane == 0 && !named_t) {
        const float u = capped<CAP>(a, zt, slope_t);
        out[given] = from_float<E>((grad_rest<OP, HARD>(a, T, u) - a.ce) * slope_t * scale);
      }
    }
  }
  if (!works) finish();
}

// ---------------------------------------------------------------------------------- rows that shared memory does not hold
// A block for a row, which is read from memory in every pass (the alternatives: one pass for each).
constexpr int LONG_NT = 512;
template <typename E, Op OP, bool CAP, bool HARD>
__global__ void __launch_bounds__(LONG_NT) long_kernel(Row a) {
  constexpr int NT = LONG_NT;
  __shared__ float sh[32];
  __shared__ u64 best[32];
  __shared__ int id[MOST_TOP];
  __shared__ float q[MOST_TOP];
  __shared__ Part rec[MOST_PARTS];
  __shared__ Totals fin;
  extern __shared__ uint32_t bits[];                          // DISTILL: which tokens the teacher names
  const int row = blockIdx.x, tid = threadIdx.x, V = a.V, K = a.K;
  const E* z = static_cast<const E*>(a.z) + row * a.ldz;
  E* out = static_cast<E*>(a.out) + row * a.ldo;
  const long t = a.targets ? a.targets[row] : -1;
  if (!row_on(a, row, t)) {
    if (OP != SCORES && a.out)
      for (int i = tid; i < V; i += NT) out[i] = from_float<E>(0.f);
    row_off<OP>(a, row);
    return;
  }
  float qr = 0.f;
  bool named_t = false;
  Named mine;
  if (OP == DISTILL) {
    for (int i = tid; i < (V + 31) / 32; i += NT) bits[i] = 0;
    __syncthreads();
    if (tid < 32) {
      qr = teacher_of(a, row, t, id, q, mine, named_t);
#pragma unroll
      for (int j = 0; j < ENTRIES; ++j) {
        const int i = mine.id[j];
        if (i < 0) continue;
        mine.here[j] = true;
        mine.z[j] = to_float(z[i]);
        const uint32_t bit = 1u << (i & 31);
        mine.first[j] = !(atomicOr(&bits[i >> 5], bit) & bit);
      }
    }
    __syncthreads();
  }
  auto named = [&](int i) { return OP == DISTILL ? (bits[i >> 5] >> (i & 31) & 1) != 0 : i == t; };
  float m = -INFINITY;
  for (int i = tid; i < V; i += NT)
    if (!named(i)) m = fmaxf(m, to_float(z[i]));
  m = block_max<NT>(m, sh);
  Part p = {};
  p.m = m == -INFINITY ? m : capped<CAP>(a, m);
  const float base = m == -INFINITY ? 0.f : p.m;
  float S = 0.f, A = 0.f, S1 = 0.f;
  for (int i = tid; i < V; i += NT) {
    if (named(i)) continue;
    const float d = capped<CAP>(a, to_float(z[i])) - base, x = d * a.c, e = ex2(x);
    S += e;
    if (OP != DISTILL) A += e * max_nan(x, -256.f);
    if (HARD) S1 += ex2(d * LOG2E);
  }
  p.S = block_sum<NT>(S, sh);
  if (OP != DISTILL) p.A = block_sum<NT>(A, sh);
  if (HARD) p.S1 = block_sum<NT>(S1, sh);
  p.B = -INFINITY;
  if (OP == DISTILL && tid < 32) named_part<CAP, HARD>(a, mine, p);
  float slope_t = 1.f, ut = 0.f;
  if (a.targets) ut = capped<CAP>(a, to_float(z[t]), slope_t);
  p.has_t = a.targets ? 1.f : 0.f;
  p.ut = ut;
  p.low = 0;
  if (tid < MOST_PARTS) rec[tid] = tid == 0 ? p : no_part();
  __syncthreads();                                            // the logits that are read by index have been read
  if (tid < 32) total<OP, HARD>(a, row, rec, qr, given_of(a, row), true, &fin);
  __syncthreads();
  const Totals T = fin;
  if (OP == SCORES) {
    u64 below = ~0ull;
    for (int k = 0; k < K; ++k) {
      u64 key = 0;
      for (int i = tid; i < V; i += NT) {
        const u64 v = key_of(to_float(z[i]), i);
        if (v < below && v > key) key = v;
      }
      for (int o = 16; o; o >>= 1) {
        const u64 other = __shfl_xor_sync(~0u, key, o);
        key = other > key ? other : key;
      }
      __syncthreads();
      if ((tid & 31) == 0) best[tid >> 5] = key;
      __syncthreads();
      for (int w = 0; w < NT / 32; ++w) key = best[w] > key ? best[w] : key;
      below = key;
      if (tid == 0) {
        const int i = static_cast<int>(~static_cast<uint32_t>(key));
        a.top_ids[(size_t)row * K + k] = i;
        a.top_logprob[(size_t)row * K + k] = i == t ? T.lp : ((capped<CAP>(a, to_float(z[i])) - T.M) * a.c - T.lS) * LN2;
      }
    }
    return;
  }
  if (!a.out) return;
  const float scale = OP == DISTILL ? a.scale : a.scale * a.inv_tau;
  for (int i = tid; i < V; i += NT) {
    if (named(i)) continue;
    float slope;
    const float u = capped<CAP>(a, to_float(z[i]), slope);
    float v = grad_rest<OP, HARD>(a, T, u);
    if (HARD && i == t) v -= a.ce;
    out[i] = from_float<E>(v * slope * scale);
  }
  if (OP == POLICY && tid == 0) out[t] = from_float<E>(grad_taken(T, a.bonus) * slope_t * scale);
  if (OP == DISTILL && tid < 32) write_named<E, CAP, HARD>(a, T, mine, id, q, t, scale, out);
}

// -------------------------------------------------------------------------------------------------------- launching
constexpr int MOST_SMEM = 220 * 1024;      // a block's dynamic shared memory
constexpr int SLICE = 33 * 1024;           // bytes of a row a block, where eight blocks are enough for that

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

template <typename E, Op OP, bool TOP, bool CAP, bool HARD, int NW>
int launch_slices(const Row& a, int parts, int slice, int room, int smem, cudaStream_t stream) {
  static std::atomic<unsigned long long> done{0};
  auto kernel = slice_kernel<E, OP, TOP, CAP, HARD, NW>;
  if (!allow(kernel, done)) return -400;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(static_cast<unsigned>(a.T) * parts);
  config.blockDim = dim3(NW + 32);
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  cudaLaunchAttribute cluster;
  cluster.id = cudaLaunchAttributeClusterDimension;
  cluster.val.clusterDim.x = parts;
  cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
  config.attrs = &cluster;
  config.numAttrs = 1;
  // (blocks that an SM holds by their shared memory; where all begin at once there is nothing to take over)
  const int most = 148 * std::max(1, std::min(slice_blocks<NW>(), (227 * 1024) / (smem + 4096)));
  const int more = static_cast<long>(a.T) * parts > most;
  return cudaLaunchKernelEx(&config, kernel, a, slice, room, more) == cudaSuccess ? 0 : -400;
}

template <typename E, Op OP, bool TOP, bool CAP, bool HARD>
int launch_rows(const Row& a, cudaStream_t stream) {
  constexpr int VE = 16 / sizeof(E);
  const long bytes = static_cast<long>(a.V + VE - 1) * sizeof(E);
  int parts = 1;
  while (parts < MOST_PARTS && (bytes > static_cast<long>(SLICE) * parts || (static_cast<long>(a.T) * parts < 2 * 148 && bytes > 4096l * parts))) parts *= 2;
  const long slice = ((a.V + VE - 1 + parts - 1) / parts + VE - 1) / VE * VE, size = slice * static_cast<long>(sizeof(E));
  // (where fewer threads than K have tokens, there are fewer than 1,024 of them and there is room for all)
  const int room = TOP ? (a.V < 1024 ? a.V : 32 + 3 * a.K / 2) : 0;
  const long listed = static_cast<long>(room) * parts * 8, smem = size + listed;
  if (smem <= MOST_SMEM && static_cast<long>(a.T) * parts <= 0x7FFFFFFFl) {
    const int s = static_cast<int>(slice), m = static_cast<int>(smem);
    if (size <= 48 * 1024) return launch_slices<E, OP, TOP, CAP, HARD, 128>(a, parts, s, room, m, stream);
    if (size <= 96 * 1024) return launch_slices<E, OP, TOP, CAP, HARD, 256>(a, parts, s, room, m, stream);
    return launch_slices<E, OP, TOP, CAP, HARD, 512>(a, parts, s, room, m, stream);
  }
  static std::atomic<unsigned long long> done{0};
  auto kernel = long_kernel<E, OP, CAP, HARD>;
  const int bits = OP == DISTILL ? (a.V + 31) / 32 * 4 : 0;
  if (bits > MOST_SMEM) return -5;
  if (!allow(kernel, done)) return -400;
  kernel<<<a.T, LONG_NT, bits, stream>>>(a);
  return cudaGetLastError() == cudaSuccess ? 0 : -400;
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
// before the first is used.  The tokens with gradients of their own are written again behind the others of their block.
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
