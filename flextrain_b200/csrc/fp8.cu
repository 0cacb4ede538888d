// Quantisers to 8 bits for sm_100a: e4m3 values with one fp32 scale for each group of 128 elements along a row, down a column
// or of each square of 128 x 128, and RMSNorm (with the residual's addition) writing its output in that form.
//
//   s = max(max |x| / 448, 2^-126),   q = e4m3(x * (1 / s)) to nearest even,   the value held is q * s
//
// 448 is the largest e4m3 value.  The floor keeps 1 / s finite, for groups of zeros too.  Maxima are taken of the magnitudes'
// bit patterns as integers, whose order puts NaN above infinity above numbers, so that a group with a NaN or an infinity gets a
// scale that is one, and all of its values read as NaN.  Compiled without fast math: the quantisers' two divisions of a group are
// IEEE's (the norm's are not, see there), and denormal inputs count.
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
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pack2(float a, float b) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpack2(f32x2 v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ f32x2 widen(uint32_t w) { return pack2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u)); }
__device__ __forceinline__ uint32_t e4m3x4(f32x2 lo, f32x2 hi) {
  float a, b, c, d;
  unpack2(lo, a, b);
  unpack2(hi, c, d);
  return e4m3x4(a, b, c, d);
}

// the scale of a group from the bits of its largest magnitude (NaN stays NaN: the comparison is false for it)
__device__ __forceinline__ float scale_of(uint32_t top) {
  const float s = __uint_as_float(top) / 448.f;
  return s < 1.17549435e-38f ? 1.17549435e-38f : s;
}

// Eight bf16 elements from wherever they start, in the largest pieces that may be read there.
__device__ __forceinline__ uint4 load8_any(const uint16_t* x) {
  const uintptr_t at = reinterpret_cast<uintptr_t>(x);
  const uint32_t* w = reinterpret_cast<const uint32_t*>(x);
  if ((at & 7) == 0) {
    const uint2 a = *reinterpret_cast<const uint2*>(x), b = *reinterpret_cast<const uint2*>(x + 4);
    return make_uint4(a.x, a.y, b.x, b.y);
  }
  if ((at & 3) == 0) return make_uint4(w[0], w[1], w[2], w[3]);
  const uint32_t first = x[0], last = x[7];
  w = reinterpret_cast<const uint32_t*>(x + 1);
  const uint32_t a = w[0], b = w[1], c = w[2];
  return make_uint4(first | a << 16, a >> 16 | b << 16, b >> 16 | c << 16, c >> 16 | last << 16);
}
__device__ __forceinline__ void store8_any(uint16_t* x, const uint4& u) {
  const uintptr_t at = reinterpret_cast<uintptr_t>(x);
  uint32_t* w = reinterpret_cast<uint32_t*>(x);
  if ((at & 7) == 0) {
    *reinterpret_cast<uint2*>(x) = make_uint2(u.x, u.y);
    *reinterpret_cast<uint2*>(x + 4) = make_uint2(u.z, u.w);
  } else if ((at & 3) == 0) {
    w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w;
  } else {
    x[0] = static_cast<uint16_t>(u.x);
    w = reinterpret_cast<uint32_t*>(x + 1);
    w[0] = u.x >> 16 | u.y << 16;
    w[1] = u.y >> 16 | u.z << 16;
    w[2] = u.z >> 16 | u.w << 16;
    x[7] = static_cast<uint16_t>(u.w >> 16);
  }
}

// Eight elements from column c of a row of n: 16-byte loads where the row allows them, zeros behind its end.
__device__ __forceinline__ void load8(const float* row, int c, int n, bool vec, float (&f)[8]) {
  if (vec && c + 8 <= n) {
    const float4 a = *reinterpret_cast<const float4*>(row + c), b = *reinterpret_cast<const float4*>(row + c + 4);
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
    f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
  } else if (c + 8 <= n && (reinterpret_cast<uintptr_t>(row) & 7) == 0) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 a = *reinterpret_cast<const float2*>(row + c + 2 * j);
      f[2 * j] = a.x;
      f[2 * j + 1] = a.y;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = c + j < n ? row[c + j] : 0.f;
  }
}

// Eight elements of a row as they came: magnitudes' maxima are taken of the bits, bf16 by pairs.
__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.u16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
template <typename T>
struct Raw;
template <>
struct Raw<bf16> {
  uint4 u;
  static constexpr int TOPS = 4;                 // words of magnitudes: two columns each
  __device__ __forceinline__ void load(const bf16* row, int c, int n, bool vec) {
    if (vec && c + 8 <= n) {
      u = *reinterpret_cast<const uint4*>(row + c);
    } else if (c + 8 <= n) {
      u = load8_any(reinterpret_cast<const uint16_t*>(row + c));
    } else {
      uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (c + j < n) w[j / 2] |= static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(row + c + j)) << (16 * (j & 1));
      u = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
  __device__ __forceinline__ void clear() { u = make_uint4(0, 0, 0, 0); }
  __device__ __forceinline__ uint32_t top(int i) const { return (i == 0 ? u.x : i == 1 ? u.y : i == 2 ? u.z : u.w) & 0x7FFF7FFFu; }
  __device__ static __forceinline__ uint32_t larger(uint32_t a, uint32_t b) { return max_u16x2(a, b); }
  __device__ __forceinline__ uint32_t top() const { return max_u16x2(max_u16x2(top(0), top(1)), max_u16x2(top(2), top(3))); }
  // the larger of a word's two, as the bits of an fp32 number
  __device__ static __forceinline__ uint32_t single(uint32_t t) { return max(t << 16, t & 0xFFFF0000u); }
  __device__ static __forceinline__ uint32_t column(uint32_t t, int j) { return j & 1 ? t & 0xFFFF0000u : t << 16; }
  __device__ __forceinline__ f32x2 pair(int i) const { return widen(i == 0 ? u.x : i == 1 ? u.y : i == 2 ? u.z : u.w); }
};
template <>
struct Raw<float> {
  float f[8];
  static constexpr int TOPS = 8;
  __device__ __forceinline__ void load(const float* row, int c, int n, bool vec) { load8(row, c, n, vec, f); }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = 0.f;
  }
  __device__ __forceinline__ uint32_t top(int i) const { return magnitude(f[i]); }
  __device__ static __forceinline__ uint32_t larger(uint32_t a, uint32_t b) { return max(a, b); }
  __device__ __forceinline__ uint32_t top() const {
    uint32_t t = top(0);
#pragma unroll
    for (int j = 1; j < 8; ++j) t = max(t, top(j));
    return t;
  }
  __device__ static __forceinline__ uint32_t single(uint32_t t) { return t; }
  __device__ static __forceinline__ uint32_t column(uint32_t t, int) { return t; }
  __device__ __forceinline__ f32x2 pair(int i) const { return pack2(f[2 * i], f[2 * i + 1]); }
};

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

// Bound by memory: 16384 x 4096 bf16, 203 MB, 37 us (5.5 TB/s; back to back 35; the measured copy 6.5) in rows and columns, 36 in
// squares; fp32 of half the rows 33 us (5.1 TB/s).  One block per tile of 128 x 128: a thread holds 8 columns of 8 rows that lie 16
// apart, so that a warp reads 256 bytes of two rows at a time and the tile's groups are inside the block.  The elements stay packed as
// they came until they are converted, so that four blocks fit an SM (two for fp32): unpacked in registers two fit, with each row's
// divisions in all of its lanes, and the rows took 123 us.  Five blocks 35 to 37, six, with spills, 40 to 52; two or three that walk
// over tiles, the next one's elements asked for before the current one's are converted, 34 to 41.
template <int GROUP, typename T>
__global__ void __launch_bounds__(256, sizeof(T) == 2 ? 4 : 2) quant_kernel(const QuantParams p) {
  using R = Raw<T>;
  __shared__ uint32_t sh[GROUP == 1 ? 8 * 16 * R::TOPS : 8];
  __shared__ float sh_inv[GROUP == 1 ? G : 1];
  const long tile = blockIdx.x;
  const int tn = static_cast<int>(tile % p.tiles_n);
  const long rest = tile / p.tiles_n;
  const int tm = static_cast<int>(rest % p.tiles_m);
  const long b = rest / p.tiles_m;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, l16 = threadIdx.x & 15, r0 = threadIdx.x >> 4;
  const int c = tn * G + l16 * 8;
  const T* x = static_cast<const T*>(p.x) + b * p.batch_x;
  float* scale = p.scale + b * p.batch_s;
  R raw[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int row = tm * G + r0 + 16 * i;
    if (row < p.M) raw[i].load(x + row * p.ldx, c, p.N, p.vec);
    else raw[i].clear();
  }
  float inv[8];                      // of the rows (row groups) or of the columns (column groups)
  if constexpr (GROUP == 0) {
    // The maxima of eight rows over 16 lanes: in each of three steps a lane hands over half of its rows and keeps the larger of
    // the others, so that it ends with one row's, whose two divisions it makes for all.
    uint32_t t[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = R::single(raw[i].top());
#pragma unroll
    for (int h = 4; h > 0; h >>= 1) {
      const bool up = lane & h;      // keeps the rows from h on
#pragma unroll
      for (int i = 0; i < h; ++i) {
        const uint32_t mine = up ? t[i + h] : t[i], theirs = up ? t[i] : t[i + h];
        t[i] = max(mine, __shfl_xor_sync(0xffffffffu, theirs, h));
      }
    }
    const uint32_t top = max(t[0], __shfl_xor_sync(0xffffffffu, t[0], 8));
    const float s = scale_of(top), r = 1.f / s;
    const int row = tm * G + r0 + 16 * (lane & 7);
    if ((lane & 8) == 0 && row < p.M) scale[row * p.scale_m + tn * p.scale_n] = s;
#pragma unroll
    for (int i = 0; i < 8; ++i) inv[i] = __shfl_sync(0xffffffffu, r, i, 16);
  } else if constexpr (GROUP == 1) {
#pragma unroll
    for (int j = 0; j < R::TOPS; ++j) {
      uint32_t t = raw[0].top(j);
#pragma unroll
      for (int i = 1; i < 8; ++i) t = R::larger(t, raw[i].top(j));
      t = R::larger(t, __shfl_xor_sync(0xffffffffu, t, 16));
      if (lane < 16) sh[warp * (16 * R::TOPS) + l16 * R::TOPS + j] = t;
    }
    __syncthreads();
    if (threadIdx.x < G) {
      const int word = threadIdx.x * R::TOPS / 8;
      uint32_t t = sh[word];
#pragma unroll
      for (int i = 1; i < 8; ++i) t = R::larger(t, sh[i * (16 * R::TOPS) + word]);
      const float s = scale_of(R::column(t, threadIdx.x));
      if (tn * G + threadIdx.x < p.N) scale[tm * p.scale_m + (tn * G + threadIdx.x) * p.scale_n] = s;
      sh_inv[threadIdx.x] = 1.f / s;
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 8; ++j) inv[j] = sh_inv[l16 * 8 + j];
  } else {
    uint32_t t = raw[0].top();
#pragma unroll
    for (int i = 1; i < 8; ++i) t = R::larger(t, raw[i].top());
    t = __reduce_max_sync(0xffffffffu, R::single(t));
    if (lane == 0) sh[warp] = t;
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
    f32x2 v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const f32x2 k = GROUP == 1 ? pack2(inv[2 * j], inv[2 * j + 1]) : pack2(inv[GROUP == 0 ? i : 0], inv[GROUP == 0 ? i : 0]);
      v[j] = mul2(raw[i].pair(j), k);
    }
    const uint2 o = make_uint2(e4m3x4(v[0], v[1]), e4m3x4(v[2], v[3]));
    *reinterpret_cast<uint2*>(q + row * p.ldq + c) = o;
  }
}

// ------------------------------------------------------------------------------------------------ RMSNorm
//   h = bf16(x + residual),   r = 1 / sqrt(mean h^2 + eps),   y = h r w,   y in row groups of 8 bits
// The norm is of the rounded h, which is what the backward pass reads.  r is common to a row, so it goes into the factor that a
// group is converted with: q = e4m3((h w) (r / s)), s = max(r max |h w| / 448, 2^-126).
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

// the largest magnitude; NaN if one is
__device__ __forceinline__ float max_abs(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(fabsf(b)));
  return r;
}

__device__ __forceinline__ float reciprocal(float x) {
  float r;
  asm("rcp.approx.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// Eight elements of x, and of the residual where there is one, as they came
template <bool RES>
struct NormIn {
  Raw<bf16> x[RES ? 2 : 1];
  __device__ __forceinline__ void load(const NormParams& p, long row, int c) {
    x[0].load(p.x + row * p.ldx, c, p.D, p.vec);
    if constexpr (RES) x[1].load(p.res + row * p.ldr, c, p.D, p.vec);
  }
};
// h of them, written where there is a residual; adds the squares
template <bool RES>
__device__ __forceinline__ uint4 norm_h(const NormParams& p, const NormIn<RES>& in, long row, int c, f32x2& ss) {
  uint4 h = in.x[0].u;
  if constexpr (RES) {
    const uint4 r = in.x[1].u;
    const uint32_t xs[4] = {h.x, h.y, h.z, h.w}, rs[4] = {r.x, r.y, r.z, r.w};
    uint32_t hs[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float a, b;
      unpack2(add2(widen(xs[i]), widen(rs[i])), a, b);
      const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
      hs[i] = *reinterpret_cast<const uint32_t*>(&v);
    }
    h = make_uint4(hs[0], hs[1], hs[2], hs[3]);
    uint16_t* to = reinterpret_cast<uint16_t*>(p.h) + row * p.D + c;
    if (p.vec && c + 8 <= p.D) {
      *reinterpret_cast<uint4*>(to) = h;
    } else if (c + 8 <= p.D) {
      store8_any(to, h);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (c + j < p.D) to[j] = static_cast<uint16_t>(hs[j / 2] >> (16 * (j & 1)));
    }
  }
  const uint32_t hs[4] = {h.x, h.y, h.z, h.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const f32x2 v = widen(hs[i]);
    ss = fma2(v, v, ss);
  }
  return h;
}
// 8 bits of eight elements, and their group's scale.  y / s is 448 (h w) / max |h w|: r and the rounding of s have no part in it, and
// the factor is one reciprocal (approximate, then one step of Newton's, which leaves little more than a rounding).  q and s fit
// together to a few 2^-24.  A value that near to the middle of two e4m3 numbers falls to either side: of 4e8 normal ones 257 are a step off
// the nearest, 309 with the same formula in fp32 operations, which of them differing from one input to another.  Settling those exactly
// costs 41 -> 49 us at 16384 x 4096 (finding them 2 of it), and is left out.
__device__ __forceinline__ void norm_q(const NormParams& p, const uint4& h, const f32x2 (&w)[4], long row, int c, float r) {
  const uint32_t hs[4] = {h.x, h.y, h.z, h.w};
  f32x2 t[4];
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    t[i] = mul2(widen(hs[i]), w[i]);
    float a, b;
    unpack2(t[i], a, b);
    top = max_abs(max_abs(top, a), b);
  }
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) top = max_abs(top, __shfl_xor_sync(0xffffffffu, top, o));     // the 16 lanes of a group
  float s = top * r * (1.f / 448.f);
  s = s < 1.17549435e-38f ? 1.17549435e-38f : s;
  if ((threadIdx.x & 15) == 0 && c < p.D) p.scale[row + (c >> 7) * p.scale_n] = s;
  const float inv = reciprocal(top);
  float factor = s == 1.17549435e-38f ? r * 0x1p126f : 448.f * fmaf(inv, fmaf(-top, inv, 1.f), inv);
  if (!(factor <= 3.402823466e38f)) {                // (groups of next to nothing, and rows that are not numbers)
#pragma unroll
    for (int i = 0; i < 4; ++i) t[i] = mul2(t[i], pack2(r, r));
    factor = reciprocal(s);
  }
  const f32x2 k = pack2(factor, factor);
  float f[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) unpack2(mul2(t[i], k), f[2 * i], f[2 * i + 1]);
  if (c < p.ldq) *reinterpret_cast<uint2*>(p.q + row * p.ldq + c) = make_uint2(e4m3x4(f[0], f[1], f[2], f[3]), e4m3x4(f[4], f[5], f[6], f[7]));
}
__device__ __forceinline__ void norm_gain(const NormParams& p, int c, f32x2 (&w)[4]) {
  float f[8] = {1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f};
  if (p.w != nullptr) load8(p.w, c, p.D, p.vec_w, f);
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = pack2(f[2 * i], f[2 * i + 1]);
}

// (sh: a piece that the last call did not use)
template <int NT>
__device__ __forceinline__ float block_sum(float v, float* sh) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.f;
#pragma unroll
  for (int i = 0; i < NT / 32; ++i) v += sh[i];
  return v;
}

// Threads of an SM, in blocks of NT: what fits with a row's pieces and the gain's in registers.  16384 x 2048 with a residual and
// without: 43 and 27 us with 1024, 47 and 32 with 768; x 4096 84 / 43 and 75 / 43; x 8192 (half the rows) 77 / 41 with 512 in blocks
// of 256, 82 / 45 with 1024 in blocks of 512.
constexpr int norm_threads(int V) { return V > 2 ? 512 : V == 2 ? 768 : 1024; }

// Bound by memory with a residual: 16384 x 4096, 472 MB, 75 us (6.3 TB/s; 72 back to back in a graph); without one, 201 MB, 45 us (4.5 TB/s;
// 41 in a graph), half by the chain of a row's sum, scale and conversion.  A block for each row, which read the gain again and waited
// for its loads, took 99 and 67 us; blocks of 128 threads 99 and 70, of 512 82 and 56.
//
// V > 0: a block of NT threads walks over rows of up to 8 NT V elements, its part of the gain in registers, the next row's
// elements asked for before the current row's sum is known (two rows ahead gained nothing).  V = 0: longer rows are read twice (the
// second time h comes from what the first pass wrote, by the same thread): 8192 x 16384 198 us with a residual, 144 for a floor of 61 without.
template <int NT, int V, bool RES>
__global__ void __launch_bounds__(NT, norm_threads(V) / NT) rmsnorm_fp8_kernel(const NormParams p) {
  __shared__ float sh[2][NT / 32];
  const float rD = 1.f / static_cast<float>(p.D);
  int turn = 0;
  auto rstd_of = [&](f32x2 ss, long row) {
    float a, b;
    unpack2(ss, a, b);
    const float r = rsqrtf(block_sum<NT>(a + b, sh[turn]) * rD + p.eps);
    turn ^= 1;
    if (threadIdx.x == 0) p.rstd[row] = r;
    return r;
  };
  if constexpr (V > 0) {
    f32x2 w[V][4];
    NormIn<RES> in[V];
    long row = blockIdx.x;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      in[i].load(p, row, (threadIdx.x + i * NT) * 8);
      norm_gain(p, (threadIdx.x + i * NT) * 8, w[i]);
    }
    while (true) {
      uint4 h[V];
      f32x2 ss = 0;
#pragma unroll
      for (int i = 0; i < V; ++i) h[i] = norm_h(p, in[i], row, (threadIdx.x + i * NT) * 8, ss);
      const long next = row + gridDim.x;
      if (next < p.T) {
#pragma unroll
        for (int i = 0; i < V; ++i) in[i].load(p, next, (threadIdx.x + i * NT) * 8);
      }
      const float r = rstd_of(ss, row);
#pragma unroll
      for (int i = 0; i < V; ++i) norm_q(p, h[i], w[i], row, (threadIdx.x + i * NT) * 8, r);
      if (next >= p.T) break;
      row = next;
    }
  } else {
    NormIn<RES> in;
    for (long row = blockIdx.x; row < p.T; row += gridDim.x) {
      f32x2 ss = 0, w[4];
      for (int c0 = 0; c0 < p.D; c0 += 8 * NT) {
        in.load(p, row, c0 + threadIdx.x * 8);
        norm_h(p, in, row, c0 + threadIdx.x * 8, ss);
      }
      const float r = rstd_of(ss, row);
      for (int c0 = 0; c0 < p.D; c0 += 8 * NT) {
        const int c = c0 + threadIdx.x * 8;
        Raw<bf16> h;
        if constexpr (RES) h.load(p.h + row * p.D, c, p.D, p.vec);
        else h.load(p.x + row * p.ldx, c, p.D, p.vec);
        norm_gain(p, c, w);
        norm_q(p, h.u, w, row, c, r);
      }
    }
  }
}

template <int NT, int V>
int launch_norm(const NormParams& p, cudaStream_t stream) {
  const int most = 148 * (norm_threads(V) / NT);
  const int grid = p.T < most ? p.T : most;
  if (p.res != nullptr) rmsnorm_fp8_kernel<NT, V, true><<<grid, NT, 0, stream>>>(p);
  else rmsnorm_fp8_kernel<NT, V, false><<<grid, NT, 0, stream>>>(p);
  return cudaGetLastError() == cudaSuccess ? 0 : -400;
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
  if (p.D <= 1024) return launch_norm<128, 1>(p, a->stream);
  if (p.D <= 2048) return launch_norm<256, 1>(p, a->stream);
  if (p.D <= 4096) return launch_norm<256, 2>(p, a->stream);
  if (p.D <= 6144) return launch_norm<256, 3>(p, a->stream);
  if (p.D <= 8192) return launch_norm<256, 4>(p, a->stream);
  return launch_norm<256, 0>(p, a->stream);
}

}  // extern "C"
