// Quantisers to 8 bits for sm_100a: e4m3 values with one fp32 scale for each group of 128 elements along a row, down a column
// or of each square of 128 x 128, and RMSNorm (with the residual's addition) writing its output in that form.
//
//   s = max(max |x| / 448, 2^-126),   q = e4m3(x * (1 / s)) to nearest even,   the value held is q * s
//
// 448 is the largest e4m3 value.  The floor keeps 1 / s finite, for groups of zeros too.  Maxima are taken of the magnitudes'
// bit patterns as integers, whose order puts NaN above infinity above numbers, so that a group with a NaN or an infinity gets a
// scale that is one, and all of its values read as NaN.  Compiled without fast math: the two divisions of a group are IEEE's,
// and denormal inputs count.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace {

typedef __nv_bfloat16 bf16;
constexpr int G = 128;             // elements of a group along its axis

__device__ __forceinline__ uint32_t magnitude(float f) { return __float_as_uint(f) & 0x7FFFFFFFu; }

// four values to e4m3, the first in the lowest byte
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
  return static_cast<uint32_t>(hi) << 16 | lo;
}
__device__ __forceinline__ uint2 e4m3x8(const float (&f)[8], float inv) {
  return make_uint2(e4m3x4(f[0] * inv, f[1] * inv, f[2] * inv, f[3] * inv), e4m3x4(f[4] * inv, f[5] * inv, f[6] * inv, f[7] * inv));
}

// the scale of a group from the bits of its largest magnitude (NaN stays NaN: the comparison is false for it)
__device__ __forceinline__ float scale_of(uint32_t top) {
  const float s = __uint_as_float(top) / 448.f;
  return s < 1.17549435e-38f ? 1.17549435e-38f : s;
}

__device__ __forceinline__ void unpack8(const uint4& u, float (&f)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __uint_as_float(w[i] << 16);
    f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
}
__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
  uint4 u;
  __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&u);
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
  return u;
}

// Eight elements from column c of a row of n: 16-byte loads where the row allows them, zeros behind its end.
__device__ __forceinline__ void load8(const bf16* row, int c, int n, bool vec, float (&f)[8]) {
  if (vec && c + 8 <= n) {
    unpack8(*reinterpret_cast<const uint4*>(row + c), f);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = c + j < n ? __bfloat162float(row[c + j]) : 0.f;
  }
}
__device__ __forceinline__ void load8(const float* row, int c, int n, bool vec, float (&f)[8]) {
  if (vec && c + 8 <= n) {
    const float4 a = *reinterpret_cast<const float4*>(row + c), b = *reinterpret_cast<const float4*>(row + c + 4);
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
    f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = c + j < n ? row[c + j] : 0.f;
  }
}

__device__ __forceinline__ uint32_t top8(const float (&f)[8]) {
  uint32_t t = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) t = max(t, magnitude(f[j]));
  return t;
}
// over the 16 lanes that hold one group of a row
__device__ __forceinline__ uint32_t top16(uint32_t t) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) t = max(t, __shfl_xor_sync(0xffffffffu, t, o));
  return t;
}

struct QuantParams {
  const void* x;
  long ldx, batch_x;                 // elements
  uint8_t* q;
  long ldq, batch_q;                 // bytes, multiples of 16
  float* scale;
  long scale_m, scale_n, batch_s;    // strides of the scale in groups down and along
  int M, N;
  int tiles_m, tiles_n;
  int vec;
};

// One block per tile of 128 x 128: a thread holds 8 columns of 8 rows that lie 16 apart, so that a warp reads 256 bytes of two
// rows at a time and the tile's groups are inside the block.
template <int GROUP, typename T>
__global__ void __launch_bounds__(256) quant_kernel(const QuantParams p) {
  __shared__ uint32_t sh[GROUP == 1 ? 16 * G : 8];
  const long tile = blockIdx.x;
  const int tn = static_cast<int>(tile % p.tiles_n);
  const long rest = tile / p.tiles_n;
  const int tm = static_cast<int>(rest % p.tiles_m);
  const long b = rest / p.tiles_m;
  const int l16 = threadIdx.x & 15, r0 = threadIdx.x >> 4;
  const int c = tn * G + l16 * 8;
  const T* x = static_cast<const T*>(p.x) + b * p.batch_x;
  float* scale = p.scale + b * p.batch_s;
  float f[8][8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int row = tm * G + r0 + 16 * i;
    if (row < p.M) {
      load8(x + row * p.ldx, c, p.N, p.vec, f[i]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) f[i][j] = 0.f;
    }
  }
  float inv[8];                      // of the rows (row groups) or of the columns (column groups)
  if constexpr (GROUP == 0) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int row = tm * G + r0 + 16 * i;
      const float s = scale_of(top16(top8(f[i])));
      inv[i] = 1.f / s;
      if (l16 == 0 && row < p.M) scale[row * p.scale_m + tn * p.scale_n] = s;
    }
  } else if constexpr (GROUP == 1) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      uint32_t t = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) t = max(t, magnitude(f[i][j]));
      sh[r0 * G + l16 * 8 + j] = t;
    }
    __syncthreads();
    if (threadIdx.x < G) {
      uint32_t t = 0;
#pragma unroll
      for (int i = 0; i < 16; ++i) t = max(t, sh[i * G + threadIdx.x]);
      const float s = scale_of(t);
      if (tn * G + threadIdx.x < p.N) scale[tm * p.scale_m + (tn * G + threadIdx.x) * p.scale_n] = s;
      sh[threadIdx.x] = __float_as_uint(1.f / s);     // (row 0 of the column's maxima: read by this thread only)
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 8; ++j) inv[j] = __uint_as_float(sh[l16 * 8 + j]);
  } else {
    uint32_t t = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) t = max(t, top8(f[i]));
    t = __reduce_max_sync(0xffffffffu, t);
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = t;
    __syncthreads();
    t = sh[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) t = max(t, sh[i]);
    const float s = scale_of(t);
    inv[0] = 1.f / s;
    if (threadIdx.x == 0) scale[tm * p.scale_m + tn * p.scale_n] = s;
  }
  if (c >= p.ldq) return;            // (a row of q has room up to a multiple of 16)
  uint8_t* q = p.q + b * p.batch_q;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int row = tm * G + r0 + 16 * i;
    if (row >= p.M) break;
    uint2 o;
    if constexpr (GROUP == 1)
      o = make_uint2(e4m3x4(f[i][0] * inv[0], f[i][1] * inv[1], f[i][2] * inv[2], f[i][3] * inv[3]),
                     e4m3x4(f[i][4] * inv[4], f[i][5] * inv[5], f[i][6] * inv[6], f[i][7] * inv[7]));
    else
      o = e4m3x8(f[i], inv[GROUP == 0 ? i : 0]);
    *reinterpret_cast<uint2*>(q + row * p.ldq + c) = o;
  }
}

// ------------------------------------------------------------------------------------------------ RMSNorm
//   h = bf16(x + residual),   r = 1 / sqrt(mean h^2 + eps),   y = h r w,   y in row groups of 8 bits
// The norm is of the rounded h, which is what the backward pass reads.
struct NormParams {
  const bf16* x;
  long ldx;
  const bf16* res;
  long ldr;
  const float* w;
  uint8_t* q;
  long ldq;
  float* scale;
  long scale_n;                      // stride between the scales of neighbouring groups; rows lie next to one another
  float* rstd;
  bf16* h;                           // contiguous; written when a residual is given
  int T, D;
  float eps;
  int vec;                           // x, res and h in 16-byte pieces
  int vec_w;
};

__device__ __forceinline__ void norm_input(const NormParams& p, long row, int c, float (&f)[8]) {
  load8(p.x + row * p.ldx, c, p.D, p.vec, f);
  if (p.res == nullptr) return;
  float r[8];
  load8(p.res + row * p.ldr, c, p.D, p.vec, r);
#pragma unroll
  for (int j = 0; j < 8; ++j) f[j] += r[j];
  const uint4 u = pack8(f);
  unpack8(u, f);
  bf16* h = p.h + row * p.D + c;
  if (p.vec && c + 8 <= p.D) {
    *reinterpret_cast<uint4*>(h) = u;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (c + j < p.D) h[j] = __float2bfloat16_rn(f[j]);
  }
}
// (y of eight elements, its group's scale, and their 8 bits)
__device__ __forceinline__ void norm_output(const NormParams& p, long row, int c, float (&f)[8], float r) {
  if (p.w != nullptr) {
    float w[8];
    load8(p.w, c, p.D, p.vec_w, w);
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = f[j] * r * w[j];
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] *= r;
  }
  const float s = scale_of(top16(top8(f)));
  if ((threadIdx.x & 15) == 0 && c < p.D) p.scale[row + (c >> 7) * p.scale_n] = s;
  if (c < p.ldq) *reinterpret_cast<uint2*>(p.q + row * p.ldq + c) = e4m3x8(f, 1.f / s);
}

template <int NT>
__device__ __forceinline__ float block_sum(float v, float* sh) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.f;
#pragma unroll
  for (int i = 0; i < NT / 32; ++i) v += sh[i];
  __syncthreads();
  return v;
}

// V > 0: a block of NT threads holds a row of up to 8 NT V elements in registers.  V = 0: longer rows are read twice (the
// second time h comes from what the first pass wrote, by the same thread).
template <int NT, int V>
__global__ void __launch_bounds__(NT) rmsnorm_fp8_kernel(const NormParams p) {
  __shared__ float sh[NT / 32];
  const long row = blockIdx.x;
  float ss = 0.f;
  const float rD = 1.f / static_cast<float>(p.D);
  if constexpr (V > 0) {
    float f[V][8];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      norm_input(p, row, (threadIdx.x + i * NT) * 8, f[i]);
#pragma unroll
      for (int j = 0; j < 8; ++j) ss += f[i][j] * f[i][j];
    }
    const float r = rsqrtf(block_sum<NT>(ss, sh) * rD + p.eps);
    if (threadIdx.x == 0) p.rstd[row] = r;
#pragma unroll
    for (int i = 0; i < V; ++i) norm_output(p, row, (threadIdx.x + i * NT) * 8, f[i], r);
  } else {
    float f[8];
    for (int c0 = 0; c0 < p.D; c0 += 8 * NT) {
      norm_input(p, row, c0 + threadIdx.x * 8, f);
#pragma unroll
      for (int j = 0; j < 8; ++j) ss += f[j] * f[j];
    }
    const float r = rsqrtf(block_sum<NT>(ss, sh) * rD + p.eps);
    if (threadIdx.x == 0) p.rstd[row] = r;
    for (int c0 = 0; c0 < p.D; c0 += 8 * NT) {
      const int c = c0 + threadIdx.x * 8;
      if (p.res != nullptr) load8(p.h + row * p.D, c, p.D, p.vec, f);
      else load8(p.x + row * p.ldx, c, p.D, p.vec, f);
      norm_output(p, row, c, f, r);
    }
  }
}

template <typename T>
int launch_quant(int group, const QuantParams& p, long blocks, cudaStream_t stream) {
  const unsigned grid = static_cast<unsigned>(blocks);
  if (group == 0) quant_kernel<0, T><<<grid, 256, 0, stream>>>(p);
  else if (group == 1) quant_kernel<1, T><<<grid, 256, 0, stream>>>(p);
  else quant_kernel<2, T><<<grid, 256, 0, stream>>>(p);
  return cudaGetLastError() == cudaSuccess ? 0 : -400;
}

}  // namespace

extern "C" {

// Arguments in 8 bytes each.  x (batch, M, N) fp32 or bf16 with strides in elements, rows contiguous -> q (rows ldq bytes apart, a
// multiple of 16 that holds N) and the scales of group 0 (1 x 128), 1 (128 x 1) or 2 (128 x 128), at scale + gm * scale_m + gn *
// scale_n.
struct QuantArgs {
  const void* x;
  void* q;
  float* scale;
  int64_t x_fp32, ldx, batch_x, ldq, batch_q, scale_m, scale_n, batch_s, batch, M, N, group;
  cudaStream_t stream;
};

int ftb_quant_fp8(const QuantArgs* a) {
  if (a->batch <= 0 || a->M <= 0 || a->N <= 0) return 0;
  if (a->group < 0 || a->group > 2 || a->ldq < a->N || ((a->ldq | a->batch_q) & 15) || (reinterpret_cast<uintptr_t>(a->q) & 15)) return -2;
  const int64_t tiles_m = (a->M + G - 1) / G, tiles_n = (a->N + G - 1) / G;
  // (sizes and tiles in 31 bits; each factor is checked before the products are formed)
  if (a->M > 0x7FFFFF00ll || a->N > 0x7FFFFF00ll || a->batch > 0x7FFFFFFFll || tiles_m * tiles_n > 0x7FFFFFFFll / a->batch) return -3;
  QuantParams p;
  p.x = a->x; p.ldx = a->ldx; p.batch_x = a->batch_x;
  p.q = static_cast<uint8_t*>(a->q); p.ldq = a->ldq; p.batch_q = a->batch_q;
  p.scale = a->scale; p.scale_m = a->scale_m; p.scale_n = a->scale_n; p.batch_s = a->batch_s;
  p.M = static_cast<int>(a->M); p.N = static_cast<int>(a->N);
  p.tiles_m = static_cast<int>(tiles_m);
  p.tiles_n = static_cast<int>(tiles_n);
  const long es = a->x_fp32 ? 4 : 2, blocks = a->batch * tiles_m * tiles_n;
  const int group = static_cast<int>(a->group);
  p.vec = (reinterpret_cast<uintptr_t>(a->x) & 15) == 0 && (a->M == 1 || (a->ldx * es & 15) == 0) && (a->batch == 1 || (a->batch_x * es & 15) == 0);
  return a->x_fp32 ? launch_quant<float>(group, p, blocks, a->stream) : launch_quant<bf16>(group, p, blocks, a->stream);
}

// See NormParams.  res and h may be null together; w may be null.  The scale of row t and group g lies at scale + t + g * scale_n.
struct NormArgs {
  const void *x, *res;
  const float* w;
  void* q;
  float *scale, *rstd;
  void* h;
  int64_t ldx, ldr, ldq, scale_n, T, D;
  double eps;
  cudaStream_t stream;
};

int ftb_rmsnorm_fp8_fwd(const NormArgs* a) {
  if (a->T <= 0 || a->D <= 0) return 0;
  if (a->T > 0x7FFFFFFFll || a->D > 0x7FFF0000ll) return -3;
  if (a->ldq < a->D || (a->ldq & 15) || (reinterpret_cast<uintptr_t>(a->q) & 15) || (a->res == nullptr) != (a->h == nullptr)) return -2;
  NormParams p;
  p.x = static_cast<const bf16*>(a->x); p.ldx = a->ldx;
  p.res = static_cast<const bf16*>(a->res); p.ldr = a->ldr;
  p.w = a->w; p.q = static_cast<uint8_t*>(a->q); p.ldq = a->ldq; p.scale = a->scale; p.scale_n = a->scale_n;
  p.rstd = a->rstd; p.h = static_cast<bf16*>(a->h);
  p.T = static_cast<int>(a->T); p.D = static_cast<int>(a->D); p.eps = static_cast<float>(a->eps);
  auto rows16 = [&](const void* t, long ld) { return (reinterpret_cast<uintptr_t>(t) & 15) == 0 && (a->T == 1 || (ld & 7) == 0); };
  p.vec = rows16(a->x, a->ldx) && (a->res == nullptr || (rows16(a->res, a->ldr) && rows16(a->h, a->D)));
  p.vec_w = (reinterpret_cast<uintptr_t>(a->w) & 15) == 0;
  const unsigned grid = static_cast<unsigned>(a->T);
  const int D = p.D;
  cudaStream_t stream = a->stream;
  if (D <= 1024) rmsnorm_fp8_kernel<128, 1><<<grid, 128, 0, stream>>>(p);
  else if (D <= 2048) rmsnorm_fp8_kernel<128, 2><<<grid, 128, 0, stream>>>(p);
  else if (D <= 4096) rmsnorm_fp8_kernel<256, 2><<<grid, 256, 0, stream>>>(p);
  else if (D <= 8192) rmsnorm_fp8_kernel<256, 4><<<grid, 256, 0, stream>>>(p);
  else rmsnorm_fp8_kernel<256, 0><<<grid, 256, 0, stream>>>(p);
  return cudaGetLastError() == cudaSuccess ? 0 : -400;
}

}  // extern "C"
