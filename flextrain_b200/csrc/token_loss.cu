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
__device__ __forceinline__ float capped(const Row& a, float z) { return CAP ? a.cap * tanhf(z * a.inv_cap) : z; }
template <bool CAP>
__device__ __forceinline__ float capped(const Row& a, float z, float& slope) {
  if (!CAP) {
    slope = 1.f;
    return z;
  }
  const float t = tanhf(z * a.inv_cap);
  slope = 1.f - t * t;
  return a.cap * t;
}

// whole numbers in the order of the floats: -0 is +0, a NaN is above all
__device__ __forceinline__ uint32_t order_of(float f) {
  if (f != f) return 0xFFFFFFFFu;
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

// ------------------------------------------------------------------------------------------------ a block for a row
// The row is read from memory in every pass.
constexpr int NT = 512;
template <typename E, Op OP, bool CAP>
__global__ void __launch_bounds__(NT) row_kernel(Row a) {
  __shared__ float sh[32];
  __shared__ unsigned long long best[32];
  __shared__ int id[MOST_TOP];
  __shared__ float q[MOST_TOP], zk[MOST_TOP];
  __shared__ float target[2];
  extern __shared__ uint32_t bits[];                         // DISTILL: which tokens the teacher names
  const int row = blockIdx.x, tid = threadIdx.x, V = a.V, K = a.K;
  const E* z = static_cast<const E*>(a.z) + row * a.ldz;
  E* out = static_cast<E*>(a.out) + row * a.ldo;
  const long t = a.targets ? a.targets[row] : 0;
  const bool on = (!a.targets || (t != a.ignore && t >= 0 && t < V)) && (!a.mask || a.mask[row] > 0.f);
  if (!on) {
    if (a.out)
      for (int i = tid; i < V; i += NT) out[i] = from_float<E>(0.f);
    if (tid == 0) {
      if (a.loss) a.loss[row] = 0.f;
      if (a.logprob) a.logprob[row] = 0.f;
      if (a.entropy) a.entropy[row] = 0.f;
      if (a.lse) a.lse[row] = 0.f;
    }
    if (OP == SCORES)
      for (int k = tid; k < K; k += NT) {
        a.top_ids[(size_t)row * K + k] = -1;
        a.top_logprob[(size_t)row * K + k] = -INFINITY;
      }
    return;
  }
  // the teacher's tokens: q, its sum, which entries name a token for the first time
  float log_q = -INFINITY, my_q = 0.f, share = 1.f, qr = 0.f, mk = -INFINITY;
  bool first = false;
  int mine = -1;
  if (OP == DISTILL) {
    for (int i = tid; i < (V + 31) / 32; i += NT) bits[i] = 0;
    float sum_max = -INFINITY;
    if (tid < K) {
      const long k = a.ids[(size_t)row * K + tid];
      mine = k >= 0 && k < V ? static_cast<int>(k) : -1;
      if (mine >= 0) log_q = a.teacher[(size_t)row * K + tid];
      id[tid] = mine;
    }
    if (!a.bucket) {
      sum_max = block_max<NT>(log_q, sh);
      const float s = block_sum<NT>(mine >= 0 ? expf(log_q - (sum_max == -INFINITY ? 0.f : sum_max)) : 0.f, sh);
      log_q = log_q - (sum_max == -INFINITY ? 0.f : sum_max) - logf(s);
      if (sum_max == -INFINITY) log_q = -INFINITY;
    }
    my_q = mine >= 0 && log_q != -INFINITY ? expf(log_q) : 0.f;
    const float sum = block_sum<NT>(my_q, sh);
    if (a.bucket) qr = sum < 1.f ? 1.f - sum : 0.f;
    share = a.bucket ? sum + qr : (sum > 0.f ? 1.f : sum);
    if (tid < K) q[tid] = my_q;
    if (mine >= 0) {
      zk[tid] = to_float(z[mine]);
      mk = capped<CAP>(a, zk[tid]);
      first = true;
      for (int k = 0; k < tid; ++k) first = first && id[k] != mine;
      if (first) atomicOr(&bits[mine >> 5], 1u << (mine & 31));
    }
    __syncthreads();
  }
  auto named = [&](int i) { return OP == DISTILL && (bits[i >> 5] >> (i & 31) & 1); };
  float m = -INFINITY;
  for (int i = tid; i < V; i += NT)
    if (!named(i)) m = fmaxf(m, to_float(z[i]));
  m = block_max<NT>(m, sh);
  m = m == -INFINITY ? m : capped<CAP>(a, m);               // of the tokens that are not named
  const float base = m == -INFINITY ? 0.f : m;
  const bool hard = OP == DISTILL && a.ce != 0.f;
  float S = 0.f, A = 0.f, S1 = 0.f;
  for (int i = tid; i < V; i += NT) {
    if (named(i)) continue;
    const float d = capped<CAP>(a, to_float(z[i])) - base, e = ex2(d * a.c);
    S += e;
    if (OP != DISTILL) A += e * max_nan(d * a.c, -256.f);
    if (hard) S1 += ex2(d * LOG2E);
  }
  S = block_sum<NT>(S, sh);
  if (OP != DISTILL) A = block_sum<NT>(A, sh);
  const float rest = S;
  float M = base, lS1 = 0.f;
  if (OP == DISTILL) {
    M = fmaxf(m, block_max<NT>(mk, sh));
    M = M == -INFINITY ? 0.f : M;
    const float down = ex2((base - M) * a.c);
    S = (m == -INFINITY ? 0.f : rest * down) + block_sum<NT>(first ? ex2((mk - M) * a.c) : 0.f, sh);
    if (hard) {
      S1 = block_sum<NT>(S1, sh);
      S1 = (m == -INFINITY ? 0.f : S1 * ex2((base - M) * LOG2E)) + block_sum<NT>(first ? ex2((mk - M) * LOG2E) : 0.f, sh);
      lS1 = log2f(S1);
    }
  }
  const float lS = S != 0.f ? log2f(S) : NAN;                // no finite logit: all that follows is NaN
  float slope_t = 1.f, ut = 0.f, zt = 0.f;
  if (a.targets) {
    zt = to_float(z[t]);
    ut = capped<CAP>(a, zt, slope_t);
  }
  const float lp = ((ut - M) * a.c - lS) * LN2, H = OP == DISTILL ? 0.f : (lS - A / S) * LN2;
  float g = 0.f, ka = 0.f, kb = 0.f, k0 = 0.f, kr = 0.f;     // gradient of an unnamed token: 2^(t + k0) (ka + kb log p) + hard part
  if (OP == SCORES) {
    if (tid == 0) {
      if (a.logprob) a.logprob[row] = lp;
      a.entropy[row] = H;
      a.lse[row] = M * a.inv_tau + lS * LN2;
    }
    unsigned long long below = ~0ull;
    for (int k = 0; k < K; ++k) {
      unsigned long long key = 0;
      for (int i = tid; i < V; i += NT) {
        const unsigned long long v = static_cast<unsigned long long>(order_of(to_float(z[i]))) << 32 | static_cast<uint32_t>(~i);
        if (v < below && v > key) key = v;
      }
      for (int o = 16; o; o >>= 1) {
        const unsigned long long other = __shfl_xor_sync(~0u, key, o);
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
        a.top_logprob[(size_t)row * K + k] = ((capped<CAP>(a, to_float(z[i])) - M) * a.c - lS) * LN2;
      }
    }
    return;
  }
  if (OP == POLICY) {
    const float L = policy_row(a, row, lp, H, g);
    if (tid == 0) {
      a.loss[row] = L;
      a.logprob[row] = lp;
      a.entropy[row] = H;
    }
    ka = a.bonus * H - g;
    kb = a.bonus;
    k0 = -lS;
  }
  float pr = 1.f;
  if (OP == DISTILL) {
    const float lpk = ((mk - M) * a.c - lS) * LN2;
    float kl = block_sum<NT>(my_q > 0.f ? my_q * (log_q - lpk) : 0.f, sh);
    k0 = (base - M) * a.c - lS;
    ka = share;
    if (a.bucket && m != -INFINITY && qr > 0.f) {
      const float l2 = (base - M) * a.c + log2f(rest) - lS;  // log2 of the student's share of the others
      kl += qr * (logf(qr) - l2 * LN2);
      if (l2 > -60.f) {
        ka = share - qr / ex2(l2);
      } else {                                               // (p itself is nothing beside the teacher's share there)
        k0 = -log2f(rest);
        ka = -qr;
      }
    } else if (a.bucket) {
      share -= qr;                                           // nothing is left beside the named tokens
      ka = share;
    }
    kr = 1.f - a.ce;
    float L = kr * a.tau * a.tau * kl;
    if (hard) L -= a.ce * ((ut - M) * LOG2E - lS1) * LN2;
    if (tid == 0) a.loss[row] = L;
  }
  if (!a.out) return;
  const float scale = OP == DISTILL ? a.scale : a.scale * a.inv_tau;
  __syncthreads();                                           // the logits that are read by index have been read
  for (int i = tid; i < V; i += NT) {
    if (named(i)) continue;
    float slope;
    const float d = capped<CAP>(a, to_float(z[i]), slope) - base, y = d * a.c + k0;
    float v;
    if (OP == POLICY) v = kb != 0.f ? ex2(y) * (ka + kb * LN2 * max_nan(y, -256.f)) : ex2(y) * ka;
    else v = kr * a.tau * (ex2(y) * ka) + (hard ? a.ce * ex2(d * LOG2E + (base - M) * LOG2E - lS1) : 0.f);
    out[i] = from_float<E>(v * slope * scale);
  }
  __syncthreads();
  if (OP == POLICY && tid == 0) out[t] = from_float<E>((ex2(lp * LOG2E) * (ka + kb * lp) + g) * slope_t * scale);
  if (OP == DISTILL) {
    if (first) {
      float slope, qs = 0.f;
      const float d = capped<CAP>(a, zk[tid], slope) - M;
      for (int k = 0; k < K; ++k) qs += id[k] == mine ? q[k] : 0.f;
      float v = kr * a.tau * (ex2(d * a.c - lS) * share - qs);
      if (hard) v += a.ce * (ex2(d * LOG2E - lS1) - (mine == t ? 1.f : 0.f));
      out[mine] = from_float<E>(v * slope * scale);
    }
    if (hard && tid == 0 && !named(static_cast<int>(t))) {
      const float d = ut - M;
      const float v = kr * a.tau * (ex2((ut - base) * a.c + k0) * ka) + a.ce * (ex2(d * LOG2E - lS1) - 1.f);
      out[t] = from_float<E>(v * slope_t * scale);
    }
  }
}

template <typename E, Op OP>
int launch_rows(const Row& a, cudaStream_t stream) {
  auto kernel = a.cap > 0.f ? row_kernel<E, OP, true> : row_kernel<E, OP, false>;
  const int smem = OP == DISTILL ? (a.V + 31) / 32 * 4 : 0;
  if (smem > 200 * 1024) return -5;
  if (smem > 40 * 1024 && cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) return -400;
  kernel<<<a.T, NT, smem, stream>>>(a);
  return cudaGetLastError() == cudaSuccess ? 0 : -400;
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
    if (op == SCORES) return launch_rows<E, SCORES>(a, r->stream);
    if (op == POLICY) return launch_rows<E, POLICY>(a, r->stream);
    return launch_rows<E, DISTILL>(a, r->stream);
  };
  return r->type == 0 ? go(bf16()) : r->type == 1 ? go(__half()) : go(float());
}

// ---------------------------------------------------------------------------------------- gradient of the scores
//   dz_j = (scale / tau) u'(z_j) [ -p_j (sum of the gradients of log p_t and of the alternatives + dH (log p_j + H)) + the gradients of j's own ]
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
