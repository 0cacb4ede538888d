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

#include <atomic>

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

// the cap and its slope
template <bool CAP>
__device__ __forceinline__ float capped(const Row& a, float z, float& slope) {
  if (!CAP) {
    slope = 1.f;
    return z;
  }
  const float t = tanhf(z * a.inv_cap);
  slope = 1.f - t * t;
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

// Loss of a policy-gradient row and its derivative by log p of the taken token.  The unclipped side counts where both are equal, so
// a ratio inside the borders, and on them, has a gradient.
__device__ __forceinline__ float policy_row(const Row& a, int row, float lp, float H, float& g) {
  const float adv = a.adv ? a.adv[row] : 1.f;
  float L = -adv * lp;
  g = -adv;
  if (a.old) {
    const float r = expf(lp - a.old[row]);
    const float free = r * adv, held = fminf(fmaxf(r, 1.f - a.clip_low), 1.f + a.clip_high) * adv;
    L = -fminf(free, held);
    g = free <= held ? -free : 0.f;
    if (r != r || adv != adv) L = g = r * adv;             // (minima and maxima leave NaN out)
  }
  if (a.ref && a.kl != 0.f) {
    const float d = a.ref[row] - lp;
    L += a.kl * (expm1f(d) - d);
    g -= a.kl * expm1f(d);
  }
  return a.bonus != 0.f ? L - a.bonus * H : L;
}

// ------------------------------------------------------------------------------------------------- a row's totals
// What a part of a row (one block's) adds to them.  ``m``: largest u of the tokens that are not named (the given token of scores and
// policy rows, the teacher's of distillation are, and are added by themselves), S and A sums of e and of e log2 e relative to it, S1 of
// e at a temperature of one.
struct Part {
  float m, S, A, S1;
  float B, En, En1, kl, Q;                // distillation: the named tokens of this part relative to their largest u, B
  float ut, has_t;                        // the given token's u, in the part that holds it
  uint32_t tau;                           // scores: at least K tokens of the part are not below it
};
// what follows from all parts
struct Totals {
  float M, lS, lp, H, miss, g;            // largest u, log2 of the sum, log p_t, entropy, 1 - p_t, dL/dlog p_t
  float base, k0, ka, kb;                 // gradient of a token that is not named: 2^((u - base) c + k0) (ka + kb log p) ...
  float share, h0;                        // ... + ce 2^((u - M) log2 e - h0); distillation: the sum of q
  uint32_t tau;
};
constexpr int PART_WORDS = sizeof(Part) / 4;

template <typename F>
__device__ __forceinline__ float over8(float v, F f) {        // over the eight lanes that hold the parts
#pragma unroll
  for (int o = 4; o; o >>= 1) v = f(v, __shfl_xor_sync(~0u, v, o));
  return v;
}
__device__ __forceinline__ float sum8(float v) { return over8(v, [](float a, float b) { return a + b; }); }
__device__ __forceinline__ float max8(float v) { return over8(v, [](float a, float b) { return fmaxf(a, b); }); }

// By one warp: lane r of each eight holds part r (those from ``parts`` on hold none), so that all four eights go the same ways.  ``first``: of the row's blocks this one writes its results.
template <Op OP, bool HARD>
__device__ __forceinline__ void total(const Row& a, int row, int parts, const Part* rec, float qr, bool first, Totals* fin) {
  const int lane = threadIdx.x & 31;
  Part p = {-INFINITY, 0.f, 0.f, 0.f, -INFINITY, 0.f, 0.f, 0.f, 0.f, -INFINITY, 0.f, 0u};
  if ((lane & 7) < parts) p = rec[lane & 7];
  Totals t = {};
  const float rest = max8(p.m);                               // of the tokens that are not named
  const bool none = p.m == -INFINITY;
  if (OP != DISTILL) {
    const float has = max8(p.has_t);
    const float given = sum8(p.has_t > 0.f ? p.ut : 0.f), ut = has > 0.f ? given : -INFINITY;
    t.M = fmaxf(rest, ut);
    const float down = none ? 0.f : ex2((p.m - t.M) * a.c);
    const float O = sum8(down * p.S);
    float A = sum8(none ? 0.f : down * (p.A + p.S * ((p.m - t.M) * a.c)));
    const float yt = (ut - t.M) * a.c, et = has > 0.f ? ex2(yt) : 0.f, S = O + et;
    if (has > 0.f) A += et * max_nan(yt, -256.f);
    t.lS = S > 0.f ? log2f(S) : NAN;                          // no finite logit (or a NaN): all that follows is NaN
    // a token that has most of the row: the others' sum by itself, so that a small log p keeps its digits
    const bool most = has > 0.f && ut >= rest && S > 0.f;
    t.lp = most ? -log1pf(O) : (yt - t.lS) * LN2;
    t.H = (most ? log1pf(O) : t.lS * LN2) - A / S * LN2;
    t.miss = O / S;
    t.base = t.M;
    t.k0 = -t.lS;
    if (OP == SCORES) {
      uint32_t tau = p.tau;
#pragma unroll
      for (int o = 4; o; o >>= 1) tau = max(tau, __shfl_xor_sync(~0u, tau, o));
      t.tau = tau;
      if (first && lane == 0) {
        if (a.logprob) a.logprob[row] = t.lp;
        a.entropy[row] = t.H;
        a.lse[row] = t.M * a.inv_tau + (most ? log1pf(O) : t.lS * LN2);
      }
    } else {
      const float L = policy_row(a, row, t.lp, t.H, t.g);
      t.ka = a.bonus * t.H - t.g;
      t.kb = a.bonus;
      if (first && lane == 0) {
        a.loss[row] = L;
        a.logprob[row] = t.lp;
        a.entropy[row] = t.H;
      }
    }
  } else {
    t.M = fmaxf(rest, max8(p.B));
    const float base = rest == -INFINITY ? 0.f : rest;
    const bool no_names = p.B == -INFINITY;
    const float others = sum8(none ? 0.f : p.S * ex2((p.m - base) * a.c));
    const float S = others * (rest == -INFINITY ? 0.f : ex2((base - t.M) * a.c)) + sum8(no_names ? 0.f : p.En * ex2((p.B - t.M) * a.c));
    t.lS = S > 0.f ? log2f(S) : NAN;
    const float Q = sum8(p.Q);
    // q (log q - log p), where log p = (u - M) / tau - ln S and a part has (u - B) / tau
    float kl = sum8(p.kl + (p.Q != 0.f && !no_names ? p.Q * (t.M - p.B) * a.inv_tau : 0.f)) + (Q != 0.f ? Q * t.lS * LN2 : 0.f);
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
      const float S1 = sum8(none ? 0.f : p.S1 * ex2((p.m - t.M) * LOG2E)) + sum8(no_names ? 0.f : p.En1 * ex2((p.B - t.M) * LOG2E));
      const float ut = sum8(p.has_t > 0.f ? p.ut : 0.f);
      t.h0 = S1 > 0.f ? log2f(S1) : NAN;
      L -= a.ce * ((ut - t.M) * LOG2E - t.h0) * LN2;
    }
    if (first && lane == 0) a.loss[row] = L;
  }
  if (lane == 0) *fin = t;
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

// The teacher's entry of thread k: its token (-1: none), q and log q; which entries name a token for the first time.
struct Named {
  int id;
  float q, log_q;
  bool first;
};
// By a block; ``id`` and ``q`` are of MOST_TOP.  Returns what the teacher leaves to all others (0 without the bucket).
template <int NT>
__device__ __forceinline__ float teacher_of(const Row& a, int row, int* id, float* q, float* sh, Named& n) {
  const int tid = threadIdx.x;
  n = {-1, 0.f, -INFINITY, false};
  if (tid < a.K) {
    const long k = a.ids[(size_t)row * a.K + tid];
    if (k >= 0 && k < a.V) {
      n.id = static_cast<int>(k);
      n.log_q = a.teacher[(size_t)row * a.K + tid];
    }
    id[tid] = n.id;
  }
  if (!a.bucket) {
    const float top = block_max<NT>(n.log_q, sh);
    if (top != -INFINITY) n.log_q -= top;
    const float s = block_sum<NT>(n.id >= 0 ? expf(n.log_q) : 0.f, sh);
    if (top != -INFINITY) n.log_q -= logf(s);
  }
  n.q = n.id >= 0 ? expf(n.log_q) : 0.f;
  const float sum = block_sum<NT>(n.q, sh);
  if (tid < a.K) q[tid] = n.q;
  n.first = n.id >= 0;
  for (int k = 0; n.first && k < tid; ++k) n.first = id[k] != n.id;
  __syncthreads();
  return a.bucket && sum < 1.f ? 1.f - sum : 0.f;
}
// its share of the part: B, En, En1, kl, Q in thread 0 (``u`` -inf and ``here`` false where another part holds it)
template <bool HARD, int NT>
__device__ __forceinline__ void named_part(const Row& a, const Named& n, bool here, float u, float* sh, Part& p) {
  p.B = block_max<NT>(here ? u : -INFINITY, sh);
  const float d = u - (p.B == -INFINITY ? 0.f : p.B);
  p.En = block_sum<NT>(here && n.first ? ex2(d * a.c) : 0.f, sh);
  if (HARD) p.En1 = block_sum<NT>(here && n.first ? ex2(d * LOG2E) : 0.f, sh);
  p.kl = block_sum<NT>(here && n.q != 0.f ? n.q * (n.log_q - d * a.inv_tau) : 0.f, sh);
  p.Q = block_sum<NT>(here ? n.q : 0.f, sh);
}
__device__ __forceinline__ float q_of(const int* id, const float* q, int K, int mine) {
  float s = 0.f;
  for (int k = 0; k < K; ++k) s += id[k] == mine ? q[k] : 0.f;
  return s;
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
constexpr int MOST_PARTS = 8;
typedef unsigned long long u64;

__device__ __forceinline__ uint32_t in_cluster(const void* p, int rank) {          // the same place in another block's shared memory
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(ftb::smem_u32(p)), "r"(rank));
  return r;
}
__device__ __forceinline__ void put32(uint32_t at, uint32_t v) { asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(at), "r"(v) : "memory"); }
__device__ __forceinline__ void put64(uint32_t at, u64 v) { asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(at), "l"(v) : "memory"); }
__device__ __forceinline__ void cluster_arrive() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

template <typename E>
struct Vec {
  static constexpr int N = 16 / sizeof(E);
};
__device__ __forceinline__ void unpack(const uint4& v, float (&f)[8], bf16) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __uint_as_float(w[i] << 16);
    f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
}
__device__ __forceinline__ void unpack(const uint4& v, float (&f)[8], __half) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 g = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    f[2 * i] = g.x;
    f[2 * i + 1] = g.y;
  }
}
__device__ __forceinline__ void unpack(const uint4& v, float (&f)[4], float) {
  f[0] = __uint_as_float(v.x); f[1] = __uint_as_float(v.y); f[2] = __uint_as_float(v.z); f[3] = __uint_as_float(v.w);
}
__device__ __forceinline__ uint4 pack(const float (&f)[8], bf16) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ uint4 pack(const float (&f)[8], __half) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 h = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ uint4 pack(const float (&f)[4], float) {
  return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
}

__device__ __forceinline__ u64 key_of(float z, int token) { return static_cast<u64>(order_of(z)) << 32 | static_cast<uint32_t>(~token); }
__device__ __forceinline__ float logit_of(uint32_t order) {
  return order == NAN_ORDER ? NAN : __uint_as_float(order & 0x80000000u ? order & 0x7FFFFFFFu : ~order);
}

template <typename E, Op OP, bool TOP, bool CAP, bool HARD, int NT>
__global__ void __launch_bounds__(NT, NT == 256 ? 5 : 2) slice_kernel(Row a, int slice, int room) {
  constexpr int VE = Vec<E>::N;
  extern __shared__ __align__(128) unsigned char buf[];
  __shared__ __align__(8) uint64_t bar;
  __shared__ int gave_up, found;
  __shared__ float sh[32];
  __shared__ Part rec[MOST_PARTS];
  __shared__ Totals fin;
  __shared__ int count[2][MOST_PARTS];
  __shared__ int id[OP == DISTILL ? MOST_TOP : 1];
  __shared__ float q[OP == DISTILL ? MOST_TOP : 1];
  E* zs = reinterpret_cast<E*>(buf);
  const uint4* zv = reinterpret_cast<const uint4*>(buf);

  int rank, parts;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(parts));
  const int row = blockIdx.x / parts, tid = threadIdx.x, V = a.V;
  const E* z = static_cast<const E*>(a.z) + row * a.ldz;
  E* out = static_cast<E*>(a.out) + row * a.ldo;
  // the row from the 16-byte piece that it begins in: ``lead`` elements before it, this block's from ``lo`` on, n of them in pieces
  const int lead = static_cast<int>((reinterpret_cast<uintptr_t>(z) & 15) / sizeof(E));
  const int lo = rank * slice, n = max(0, min(lead + V - lo, slice)), nv = (n + VE - 1) / VE, first_token = lo - lead;
  const long t = a.targets ? a.targets[row] : -1;
  if (!row_on(a, row, t)) {
    if (OP != SCORES && a.out) {
      const int from = max(first_token, 0), to = min(first_token + n, V);
      for (int j = from + tid; j < to; j += NT) out[j] = from_float<E>(0.f);
    }
    if (rank == 0) row_off<OP>(a, row);
    return;
  }
  if (tid == 0) {
    gave_up = 0;
    ftb::mbar_init(&bar, 1);
    ftb::fence_barrier_init();
    if (nv > 0) {
      ftb::mbar_expect_tx(&bar, nv * 16);
      ftb::bulk_load_g2s(buf, z - lead + lo, nv * 16, &bar);
    }
  }
  cluster_arrive();                                           // (the others' shared memory may be written once all have begun)
  float qr = 0.f;
  Named mine = {-1, 0.f, -INFINITY, false};
  if (OP == DISTILL) qr = teacher_of<NT>(a, row, id, q, sh, mine);
  else __syncthreads();
  if (nv > 0 && !ftb::mbar_wait(&bar, 0, &gave_up, 1)) {      // (reported; the copy gets as long again before the block goes on)
    int again = 0;
    ftb::mbar_wait(&bar, 0, &again, 2);
  }

  // what lies around the row is no token; named tokens by themselves
  if (tid < VE) {
    if (lo + tid < lead && tid < nv * VE) zs[tid] = from_float<E>(-INFINITY);
    if (n + tid < nv * VE) zs[n + tid] = from_float<E>(-INFINITY);
  }
  const int at_t = static_cast<int>(t) - first_token;         // where the given token lies
  const bool mine_t = a.targets && at_t >= 0 && at_t < n;
  const bool here = OP == DISTILL && mine.id >= first_token && mine.id < first_token + n && mine.id >= 0;
  float zt = 0.f, zk = 0.f;
  if (mine_t && tid == 0) zt = to_float(zs[at_t]);
  if (here) zk = to_float(zs[mine.id - first_token]);
  if (OP == DISTILL) __syncthreads();                         // (an entry twice: both have read)
  if (here) zs[mine.id - first_token] = from_float<E>(-INFINITY);
  if (OP != DISTILL && mine_t && tid == 0) zs[at_t] = from_float<E>(-INFINITY);
  __syncthreads();

  // largest of each thread, of the block
  float mt = -INFINITY;
  for (int v = tid; v < nv; v += NT) {
    float f[VE];
    unpack(zv[v], f, E());
#pragma unroll
    for (int e = 0; e < VE; ++e) mt = fmaxf(mt, f[e]);
  }
  const float mz = block_max<NT>(mt, sh);
  Part p = {};
  p.m = mz == -INFINITY ? mz : capped<CAP>(a, mz);
  const float base = mz == -INFINITY ? 0.f : p.m;
  float S = 0.f, A = 0.f, S1 = 0.f;
  for (int v = tid; v < nv; v += NT) {
    float f[VE];
    unpack(zv[v], f, E());
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      const float d = capped<CAP>(a, f[e]) - base, x = d * a.c, w = ex2(x);
      S += w;
      if (OP != DISTILL) A += w * max_nan(x, -256.f);
      if (HARD) S1 += ex2(d * LOG2E);
    }
  }
  p.S = block_sum<NT>(S, sh);
  if (OP != DISTILL) p.A = block_sum<NT>(A, sh);
  if (HARD) p.S1 = block_sum<NT>(S1, sh);
  p.B = -INFINITY;
  if (OP == DISTILL) named_part<HARD, NT>(a, mine, here, here ? capped<CAP>(a, zk) : -INFINITY, sh, p);
  const int K = a.K;
  if (TOP) {
    // the largest of some K to K + K / 8 + 8 threads are not below tau (all tokens where fewer threads have any)
    uint32_t low = 0, high = order_of(mz) + 1;
    const uint32_t key = tid < nv ? order_of(mt) : 0;
    if (min(nv, NT) >= K) {
      for (int it = 0; it < 32 && high - low > 1; ++it) {
        const uint32_t mid = low + (high - low) / 2;
        const int c = __syncthreads_count(tid < nv && key >= mid);
        if (c >= K) low = mid;
        else high = mid;
        if (c >= K && c <= K + K / 8 + 8) break;
      }
    }
    p.tau = low;
  }
  float slope_t = 1.f;
  if (tid == 0) {
    p.has_t = mine_t ? 1.f : 0.f;
    p.ut = mine_t ? capped<CAP>(a, zt, slope_t) : 0.f;
    rec[rank] = p;
    found = 0;
  }
  __syncthreads();
  cluster_wait();
  // word w of this block's part to every other block
  for (int i = tid; i < parts * PART_WORDS; i += NT) {
    const int to = i / PART_WORDS, w = i - to * PART_WORDS;
    if (to != rank) put32(in_cluster(reinterpret_cast<uint32_t*>(&rec[rank]) + w, to), reinterpret_cast<const uint32_t*>(&rec[rank])[w]);
  }
  cluster_arrive();
  cluster_wait();
  if (tid < 32) total<OP, HARD>(a, row, parts, rec, qr, rank == 0, &fin);
  __syncthreads();
  const Totals T = fin;

  if (OP == SCORES) {
    if (!TOP) return;
    // tokens from the bound on to one block
    u64* taken = reinterpret_cast<u64*>(buf + max(slice * static_cast<int>(sizeof(E)), room * parts * 8));
    const int keeper = row & (parts - 1);
    const uint32_t theirs = in_cluster(taken + rank * room, keeper);
    auto collect = [&](u64 bound, bool all) {
      auto give = [&](u64 key) {
        const int i = atomicAdd(&found, 1);
        if (i < room) put64(theirs + i * 8, key);
      };
      if (tid == 0 && mine_t && key_of(zt, static_cast<int>(t)) >= bound) give(key_of(zt, static_cast<int>(t)));
      if (all || (tid < nv && order_of(mt) >= static_cast<uint32_t>(bound >> 32)))
        for (int v = tid; v < nv; v += NT) {
          float f[VE];
          unpack(zv[v], f, E());
#pragma unroll
          for (int e = 0; e < VE; ++e) {
            const int token = first_token + v * VE + e;
            if (token >= 0 && token < V && token != t && key_of(f[e], token) >= bound) give(key_of(f[e], token));
          }
        }
      __syncthreads();
      if (tid < parts) put32(in_cluster(&count[0][rank], tid), found);
      cluster_arrive();
      cluster_wait();
    };
    collect(static_cast<u64>(T.tau) << 32, T.lS != T.lS);     // (a thread's largest leaves NaN out)
    bool over = false;
    for (int r = 0; r < parts; ++r) over |= count[0][r] > room;
    if (over) {
      u64 low = 0, high = ~0ull;                              // at least K keys are not below low, fewer not below high
      for (int it = 0; high - low > 1; ++it) {
        const u64 mid = low + (high - low) / 2;
        int c = tid == 0 && mine_t && key_of(zt, static_cast<int>(t)) >= mid;
        for (int v = tid; v < nv; v += NT) {
          float f[VE];
          unpack(zv[v], f, E());
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
        if (sum >= K) low = mid;
        else high = mid;
        if (sum == K) break;
      }
      if (tid == 0) found = 0;
      cluster_arrive();                                       // (all have read the last counts)
      cluster_wait();
      collect(low, true);
    }
    if (rank != keeper) return;
    // ranks among what was collected, fewer of them first where they are many
    u64* list = reinterpret_cast<u64*>(buf);
    int total_found = 0;
    for (int r = 0; r < parts; ++r) total_found += count[0][r];
    uint32_t low = 0, high = 0xFFFFFFFFu;
    int kept = total_found;
    for (int it = 0; it < 32 && kept > K + K / 2 + 16 && high - low > 1; ++it) {
      const uint32_t mid = low + (high - low) / 2;
      int c = 0;
      for (int r = 0; r < parts; ++r)
        for (int i = tid; i < count[0][r]; i += NT) c += static_cast<uint32_t>(taken[r * room + i] >> 32) >= mid;
      c = static_cast<int>(block_sum<NT>(static_cast<float>(c), sh));
      if (c >= K) low = mid, kept = c;
      else high = mid;
    }
    __syncthreads();
    if (tid == 0) found = 0;
    __syncthreads();
    for (int r = 0; r < parts; ++r)
      for (int i = tid; i < count[0][r]; i += NT) {
        const u64 key = taken[r * room + i];
        if (static_cast<uint32_t>(key >> 32) >= low) list[atomicAdd(&found, 1)] = key;
      }
    __syncthreads();
    for (int i = tid; i < kept; i += NT) {
      const u64 key = list[i];
      int above = 0;
      for (int j = 0; j < kept; ++j) above += list[j] > key;
      if (above < K) {
        const int token = static_cast<int>(~static_cast<uint32_t>(key));
        a.top_ids[(size_t)row * K + above] = token;
        a.top_logprob[(size_t)row * K + above] =
            token == t ? T.lp : ((capped<CAP>(a, logit_of(static_cast<uint32_t>(key >> 32))) - T.M) * a.c - T.lS) * LN2;
      }
    }
    return;
  }

  if (!a.out) return;
  const float scale = OP == DISTILL ? a.scale : a.scale * a.inv_tau;
  const bool whole = (reinterpret_cast<uintptr_t>(out) & 15) / sizeof(E) == lead;       // pieces of the gradient lie as the logits' do
  for (int v = tid; v < nv; v += NT) {
    float f[VE];
    unpack(zv[v], f, E());
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      float slope;
      const float u = capped<CAP>(a, f[e], slope);
      f[e] = grad_rest<OP, HARD>(a, T, u) * slope * scale;
    }
    const int token = first_token + v * VE;
    if (whole && token >= 0 && token + VE <= V) {
      *reinterpret_cast<uint4*>(out + token) = pack(f, E());
    } else {
#pragma unroll
      for (int e = 0; e < VE; ++e)
        if (token + e >= 0 && token + e < V) out[token + e] = from_float<E>(f[e]);
    }
  }
  __syncthreads();
  if (OP == POLICY && mine_t && tid == 0) out[t] = from_float<E>(grad_taken(T, a.bonus) * slope_t * scale);
  if (OP == DISTILL) {
    if (here && mine.first) {
      float slope;
      const float u = capped<CAP>(a, zk, slope);
      out[mine.id] = from_float<E>(grad_named<HARD>(a, T, u, q_of(id, q, K, mine.id), mine.id == t) * slope * scale);
    }
    if (HARD && mine_t && tid == 0) {
      bool named = false;
      for (int k = 0; k < K; ++k) named |= id[k] == t;
      const float u = capped<CAP>(a, zt, slope_t);
      if (!named) out[t] = from_float<E>((grad_rest<OP, HARD>(a, T, u) - a.ce) * slope_t * scale);
    }
  }
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
  __shared__ Part rec;
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
  float qr = 0.f, zk = 0.f;
  Named mine = {-1, 0.f, -INFINITY, false};
  if (OP == DISTILL) {
    for (int i = tid; i < (V + 31) / 32; i += NT) bits[i] = 0;
    qr = teacher_of<NT>(a, row, id, q, sh, mine);
    if (mine.id >= 0) {
      zk = to_float(z[mine.id]);
      atomicOr(&bits[mine.id >> 5], 1u << (mine.id & 31));
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
  if (OP == DISTILL) named_part<HARD, NT>(a, mine, mine.id >= 0, mine.id >= 0 ? capped<CAP>(a, zk) : -INFINITY, sh, p);
  float slope_t = 1.f, ut = 0.f;
  if (a.targets) ut = capped<CAP>(a, to_float(z[t]), slope_t);
  p.has_t = a.targets ? 1.f : 0.f;
  p.ut = ut;
  if (tid == 0) rec = p;
  __syncthreads();                                            // the logits that are read by index have been read
  if (tid < 32) total<OP, HARD>(a, row, 1, &rec, qr, true, &fin);
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
  if (OP == DISTILL && mine.first) {
    float slope;
    const float u = capped<CAP>(a, zk, slope);
    out[mine.id] = from_float<E>(grad_named<HARD>(a, T, u, q_of(id, q, K, mine.id), mine.id == t) * slope * scale);
  }
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

template <typename E, Op OP, bool TOP, bool CAP, bool HARD, int NT>
int launch_slices(const Row& a, int parts, int slice, int room, int smem, cudaStream_t stream) {
  static std::atomic<unsigned long long> done{0};
  auto kernel = slice_kernel<E, OP, TOP, CAP, HARD, NT>;
  if (!allow(kernel, done)) return -400;
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
  config.numAttrs = 1;
  return cudaLaunchKernelEx(&config, kernel, a, slice, room) == cudaSuccess ? 0 : -400;
}

template <typename E, Op OP, bool TOP, bool CAP, bool HARD>
int launch_rows(const Row& a, cudaStream_t stream) {
  constexpr int VE = 16 / sizeof(E);
  const long bytes = static_cast<long>(a.V + VE - 1) * sizeof(E);
  int parts = 1;
  while (parts < MOST_PARTS && (bytes > static_cast<long>(SLICE) * parts || (static_cast<long>(a.T) * parts < 2 * 148 && bytes > 4096l * parts))) parts *= 2;
  const long slice = ((a.V + VE - 1 + parts - 1) / parts + VE - 1) / VE * VE;
  // (where fewer threads than K have tokens, there are fewer than 1,024 of them and there is room for all)
  const int room = TOP ? (a.V < 1024 ? a.V : 64 + 5 * a.K / 2) : 0;
  const long listed = static_cast<long>(room) * parts * 8, smem = (slice * static_cast<long>(sizeof(E)) > listed ? slice * static_cast<long>(sizeof(E)) : listed) + listed;
  if (smem <= MOST_SMEM && static_cast<long>(a.T) * parts <= 0x7FFFFFFFl) {
    const int s = static_cast<int>(slice);
    return smem > 2 * SLICE ? launch_slices<E, OP, TOP, CAP, HARD, 512>(a, parts, s, room, static_cast<int>(smem), stream)
                            : launch_slices<E, OP, TOP, CAP, HARD, 256>(a, parts, s, room, static_cast<int>(smem), stream);
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
constexpr int NT = 512;
template <typename E, bool CAP>
__global__ void __launch_bounds__(NT) grad_kernel(Row a, const float* lse, const float* dlogprob, const float* dentropy, const float* dtop) {
  __shared__ float sh[32];
  __shared__ int id[MOST_TOP];
  __shared__ float gk[MOST_TOP];
  const int row = blockIdx.x, tid = threadIdx.x, V = a.V, K = a.K;
  const E* z = static_cast<const E*>(a.z) + row * a.ldz;
  E* out = static_cast<E*>(a.out) + row * a.ldo;
  const long t = a.targets ? a.targets[row] : 0;
  const bool on = (!a.targets || (t != a.ignore && t >= 0 && t < V)) && (!a.mask || a.mask[row] > 0.f);
  if (!on) {
    for (int i = tid; i < V; i += NT) out[i] = from_float<E>(0.f);
    return;
  }
  // entry 0..K-1: the alternatives; entry K: the given token
  int mine = -1;
  float g = 0.f;
  if (tid < K) {
    const long k = a.top_ids[(size_t)row * K + tid];
    if (k >= 0 && k < V) {
      mine = static_cast<int>(k);
      g = dtop[(size_t)row * K + tid];
    }
    id[tid] = mine;
    gk[tid] = g;
  }
  const float gt = dlogprob ? dlogprob[row] : 0.f;
  if (tid == K && dlogprob) {
    mine = static_cast<int>(t);
    g = gt;
  }
  const float sum = block_sum<NT>(g, sh);
  float zm = 0.f;
  bool first = mine >= 0;
  if (first) {
    zm = to_float(z[mine]);
    for (int k = 0; k < (tid < K ? tid : K); ++k) first = first && id[k] != mine;
  }
  const float dh = dentropy ? dentropy[row] : 0.f, ka = -sum - (dentropy ? dh * a.entropy[row] : 0.f), l = lse[row];
  const float scale = a.scale * a.inv_tau;
  __syncthreads();
  auto at = [&](float zi, float own) {
    float slope;
    const float y = fmaf(capped<CAP>(a, zi, slope), a.inv_tau, -l) * LOG2E, p = ex2(y);      // (one rounding of the difference)
    return from_float<E>(((dentropy ? p * (ka - dh * LN2 * max_nan(y, -256.f)) : p * ka) + own) * slope * scale);
  };
  for (int i = tid; i < V; i += NT) out[i] = at(to_float(z[i]), 0.f);
  __syncthreads();
  if (first) {
    float own = 0.f;
    for (int k = 0; k < K; ++k) own += id[k] == mine ? gk[k] : 0.f;
    if (dlogprob && mine == t) own += gt;
    out[mine] = at(zm, own);
  }
}

template <typename E>
int launch_grad(const Row& a, const GradArgs* r) {
  auto kernel = a.cap > 0.f ? grad_kernel<E, true> : grad_kernel<E, false>;
  kernel<<<a.T, NT, 0, r->stream>>>(a, r->lse, r->dlogprob, r->dentropy, r->dtop);
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
