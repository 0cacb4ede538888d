// Matrix products of e4m3 operands with a scale for each block of 128, for sm_100a.
//
//   D[m,n] = alpha * sum_kb sa[m,kb] * sb[n,kb] * ( sum_{k in kb} op(A)[m,k] * op(B)[k,n] )  + beta * C[m,n] (+ bias[n])
//
// kb runs over blocks of 128 of the reduction.  sa has one value for a row of op(A) or for 128 of them, sb for a column of
// op(B) or for 128.  The tensor cores (tcgen05.mma kind::f8f6f4) form the inner sum in tensor memory, 128 deep, from zero; then
// eight warps read it out, multiply it by its scales and add it to fp32 sums that they keep in registers for the whole
// reduction.  So a scale costs one multiplication for each output and block, and the long sum is rounded to nearest in fp32
// whatever the tensor core's adder does.
//
//   warp 0     TMA producer (128-byte swizzle; operands K-major or MN-major, as they lie in memory)
//   warp 1     tcgen05.mma, one thread
//   warps 4-11 read out, scale and add; at the end of a tile turn it over in shared memory and store whole pieces of rows
//              (a thread's 128 sums, and 32 values on the way, need more than the 168 registers of 384 threads: the first four
//              warps give theirs up)
//
// CG = 2: a pair of SMs works on 256 x BN (each CTA 128 rows, half of B).  Grouped forms take their row or reduction ranges
// from device offsets.  Every wait is bounded.
#include <mutex>

#include "ptx.cuh"

namespace ftb {
namespace {

constexpr int BM = 128, BK = 128, MMA_K = 32;
constexpr int EPI_WARPS = 8, EPI_FIRST = 4, THREADS = 32 * (EPI_FIRST + EPI_WARPS);
constexpr int WARP_BYTES = 32 * 128;                     // a warp's piece of shared memory: 32 rows x 128 bytes
constexpr int BOX_BYTES = 128 * 128;

typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pack2(float a, float b) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ f32x2 pack2u(uint32_t a, uint32_t b) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ void unpack2(f32x2 v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// e4m3 x e4m3 -> fp32
template <int CG>
__device__ __forceinline__ void umma_f8(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  if constexpr (CG == 1)
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n}\n" ::"r"(tmem_d),
                 "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
                 : "memory");
  else
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n}\n" ::"r"(tmem_d),
                 "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
                 : "memory");
}

struct Params {
  int M, N, K;
  void* D;
  const void* C;
  const float* bias;
  long ldd, ldc;                     // elements
  float alpha, beta;
  int d_fp32, vec;                   // vec: rows of D and C in pieces of 16 bytes
  const float* sa;                   // scale of row m and block kb at sa[(m >> sa_shift) * sa_m + kb * sa_k]
  long sa_m, sa_k;
  int sa_shift;
  const float* sb;                   // scale of column n at sb[(n >> 7, or n) * sb_n + kb * sb_k]
  long sb_n, sb_k, sb_g;
  int a_mn, b_mn;
  // mode 0 one product; 1 row segments, each with a B of its own; 2 segments of the reduction, each with a D of its own
  int mode, groups;
  const int* offsets;
  long d_g;                          // mode 2: elements between the groups' results
  int total;                         // rows that the offsets run over
  int tiles_m, tiles_n, num_tiles, k_blocks;
};

struct Tile {
  int row0, left, tn, g, kb0, kbs;
};

// Where a tile lies.  Tiles come in ascending order, and the walk over the groups goes on where the last tile left it.
// Offsets are held inside the rows that there are.
template <int TM, int GM>
struct Walk {
  int e = 0, acc = 0;
  __device__ __forceinline__ bool at(const Params& p, int tile, Tile& t) {
    if (p.mode == 1) {
      for (; e < p.groups; ++e) {
        const int a = min(max(p.offsets[e], 0), p.total), b = min(max(p.offsets[e + 1], a), p.total);
        const int tm_e = (b - a + TM - 1) / TM;
        if (tile < acc + tm_e * p.tiles_n) {
          const int r = tile - acc;
          t.g = e;
          t.tn = r / tm_e;
          t.row0 = a + (r - t.tn * tm_e) * TM;
          t.left = b - t.row0;
          t.kb0 = 0;
          t.kbs = p.k_blocks;
          return true;
        }
        acc += tm_e * p.tiles_n;
      }
      return false;
    }
    t.g = 0;
    t.kb0 = 0;
    t.kbs = p.k_blocks;
    if (p.mode == 2) {
      t.g = tile / (p.tiles_m * p.tiles_n);
      tile -= t.g * p.tiles_m * p.tiles_n;
      const int a = min(max(p.offsets[t.g], 0), p.total), b = min(max(p.offsets[t.g + 1], a), p.total);
      t.kb0 = a / BK;
      t.kbs = (b - a + BK - 1) / BK;
    }
    const int per_group = GM * p.tiles_n, grp = tile / per_group;
    const int gm = min(GM, p.tiles_m - grp * GM), r = tile - grp * per_group;
    t.row0 = (grp * GM + r % gm) * TM;
    t.tn = r / gm;
    t.left = p.M - t.row0;
    return true;
  }
};

template <int CG, int BN, bool BVEC>
struct Ring {
  static constexpr int B_BYTES = BN / CG * BK;
  static constexpr int STAGE = BM * BK + B_BYTES;
  static constexpr int EXTRA = EPI_WARPS * (WARP_BYTES + (BVEC ? 2 * BN / 2 * 4 : 0));
  static constexpr int STAGES = (227 * 1024 - 1024 - 256 - EXTRA) / STAGE;
  static constexpr int TOTAL = STAGES * STAGE + EXTRA + 256 + 1024;
  static constexpr int NACC = 512 / BN;
  static_assert(STAGES >= 3 && STAGES <= 8 && NACC <= 4, "barriers in 256 bytes");
};

// 32 rows x 128 bytes of a warp in 16-byte pieces, free of bank conflicts row-wise and piece-wise
__device__ __forceinline__ uint4* piece_at(uint8_t* buf, int row, int piece) {
  return reinterpret_cast<uint4*>(buf + row * 128 + ((piece ^ (row & 7)) << 4));
}
template <typename T>
__device__ __forceinline__ T* element_at(uint8_t* buf, int row, int e) {
  const int byte = e * static_cast<int>(sizeof(T));
  return reinterpret_cast<T*>(buf + row * 128 + (((byte >> 4) ^ (row & 7)) << 4) + (byte & 15));
}

// `cols` columns of `rows` rows between global memory (row r at g + r * ld) and a warp's piece of shared memory
template <typename T>
__device__ __forceinline__ void rows_in(uint8_t* buf, const T* g, long ld, int rows, int cols, int vec, int lane) {
  if (vec) {
    const int pieces = min(8, cols * static_cast<int>(sizeof(T)) >> 4), lr = lane >> 3, lp = lane & 7;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i * 4 + lr < rows && lp < pieces)
        *piece_at(buf, i * 4 + lr, lp) = *reinterpret_cast<const uint4*>(reinterpret_cast<const char*>(g + (i * 4 + lr) * ld) + lp * 16);
  } else {
    for (int r = 0; r < rows; ++r)
      for (int e = lane; e < min(cols, static_cast<int>(128 / sizeof(T))); e += 32) *element_at<T>(buf, r, e) = g[r * ld + e];
  }
}
template <typename T>
__device__ __forceinline__ void rows_out(uint8_t* buf, T* g, long ld, int rows, int cols, int vec, int lane) {
  if (vec) {
    const int pieces = min(8, cols * static_cast<int>(sizeof(T)) >> 4), lr = lane >> 3, lp = lane & 7;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i * 4 + lr < rows && lp < pieces)
        *reinterpret_cast<uint4*>(reinterpret_cast<char*>(g + (i * 4 + lr) * ld) + lp * 16) = *piece_at(buf, i * 4 + lr, lp);
  } else {
    for (int r = 0; r < rows; ++r)
      for (int e = lane; e < min(cols, static_cast<int>(128 / sizeof(T))); e += 32) g[r * ld + e] = *element_at<T>(buf, r, e);
  }
}

// A thread's row of NP pairs of sums, from column col0 of D on: alpha, bias, C, rounding once, and out in 128-byte pieces.
template <int NP>
__device__ __forceinline__ void store_tile(const Params& p, const f32x2 (&acc)[NP], uint8_t* buf, long row, long skip, int rows,
                                           int col0, int lane) {
  if (rows <= 0) return;                               // (the whole warp)
  const bool add = p.beta != 0.f;
  if (p.d_fp32) {
    float* D = static_cast<float*>(p.D) + skip + row * p.ldd;
    const float* C = static_cast<const float*>(p.C) + skip + row * p.ldc;
#pragma unroll
    for (int c = 0; c < 2 * NP; c += 32) {
      const int col = col0 + c, cols = p.N - col;
      if (cols <= 0) break;
      if (add) {
        rows_in(buf, C + col, p.ldc, rows, cols, p.vec, lane);
        __syncwarp();
      }
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        float v[4];
        unpack2(acc[c / 2 + 2 * q], v[0], v[1]);
        unpack2(acc[c / 2 + 2 * q + 1], v[2], v[3]);
        uint4* at = piece_at(buf, lane, q);
        const uint4 cu = *at;
        const float cc[4] = {__uint_as_float(cu.x), __uint_as_float(cu.y), __uint_as_float(cu.z), __uint_as_float(cu.w)};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          v[j] *= p.alpha;
          if (p.bias != nullptr && 4 * q + j < cols) v[j] += p.bias[col + 4 * q + j];
          if (add) v[j] += p.beta * cc[j];
        }
        *at = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
      }
      __syncwarp();
      rows_out(buf, D + col, p.ldd, rows, cols, p.vec, lane);
      __syncwarp();
    }
  } else {
    __nv_bfloat16* D = static_cast<__nv_bfloat16*>(p.D) + skip + row * p.ldd;
    const __nv_bfloat16* C = static_cast<const __nv_bfloat16*>(p.C) + skip + row * p.ldc;
#pragma unroll
    for (int c = 0; c < 2 * NP; c += 64) {
      const int col = col0 + c, cols = p.N - col;
      if (cols <= 0) break;
      if (add) {
        rows_in(buf, C + col, p.ldc, rows, cols, p.vec, lane);
        __syncwarp();
      }
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        uint4* at = piece_at(buf, lane, q);
        const uint4 cu = *at;
        const uint32_t cw[4] = {cu.x, cu.y, cu.z, cu.w};
        uint32_t ow[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float a, b;
          unpack2(acc[c / 2 + 4 * q + j], a, b);
          a *= p.alpha;
          b *= p.alpha;
          if (p.bias != nullptr) {
            if (8 * q + 2 * j < cols) a += p.bias[col + 8 * q + 2 * j];
            if (8 * q + 2 * j + 1 < cols) b += p.bias[col + 8 * q + 2 * j + 1];
          }
          if (add) {
            a += p.beta * __uint_as_float(cw[j] << 16);
            b += p.beta * __uint_as_float(cw[j] & 0xFFFF0000u);
          }
          const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
          ow[j] = *reinterpret_cast<const uint32_t*>(&h);
        }
        *at = make_uint4(ow[0], ow[1], ow[2], ow[3]);
      }
      __syncwarp();
      rows_out(buf, D + col, p.ldd, rows, cols, p.vec, lane);
      __syncwarp();
    }
  }
}

template <int CG, int BN, bool BVEC>
__global__ void __launch_bounds__(THREADS, 1)
gemm_fp8_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const Params p) {
  using R = Ring<CG, BN, BVEC>;
  using W = Walk<BM * CG, 16 / CG>;
  constexpr int ST = R::STAGES, NACC = R::NACC;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* smem_epi = smem + ST * R::STAGE;
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem_epi + R::EXTRA);
  uint64_t* empty_bar = full_bar + ST;
  uint64_t* tfull_bar = empty_bar + ST;
  uint64_t* tempty_bar = tfull_bar + NACC;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty_bar + NACC);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int cta = CG == 2 ? static_cast<int>(cluster_ctarank()) : 0;
  const int first = blockIdx.x / CG, step = gridDim.x / CG;

  if (threadIdx.x == 0) {
    *abort_flag = 0;
    for (int s = 0; s < ST; ++s) { mbar_init(&full_bar[s], 1); mbar_init(&empty_bar[s], 1); }
    for (int a = 0; a < NACC; ++a) { mbar_init(&tfull_bar[a], 1); mbar_init(&tempty_bar[a], CG * EPI_WARPS); }
    fence_barrier_init();
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
  }
  if (warp == 1) {
    if constexpr (CG == 2) { tmem_alloc_2cta(tmem_slot, 512); tmem_relinquish_2cta(); }
    else { tmem_alloc(tmem_slot, 512); tmem_relinquish(); }
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (CG == 2) cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  // registers a thread: 384 x 168 at launch = 128 x 40 + 256 x 232
  if (warp < EPI_FIRST) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 40;\n");
    if (warp == 0 && lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      W walk;
      Tile t;
      for (int tile = first; tile < p.num_tiles && ok; tile += step) {
        if (!walk.at(p, tile, t)) break;
        const int row0 = t.row0 + cta * BM;
        const int col0 = t.tn * BN + cta * (BN / CG);
        const int z = p.mode == 1 ? t.g : 0;
        for (int kb = 0; kb < t.kbs; ++kb) {
          if (!(ok = mbar_wait(&empty_bar[stage], phase ^ 1, abort_flag, 10))) break;
          uint8_t* sa = smem + stage * R::STAGE;
          uint8_t* sb = sa + BM * BK;
          if (cta == 0) mbar_expect_tx(&full_bar[stage], CG * R::STAGE);
          const int k0 = (t.kb0 + kb) * BK;
          if constexpr (CG == 2) tma_load_2d_2cta(sa, &tmA, &full_bar[stage], p.a_mn ? row0 : k0, p.a_mn ? k0 : row0);
          else tma_load_2d(sa, &tmA, &full_bar[stage], p.a_mn ? row0 : k0, p.a_mn ? k0 : row0);
          if (p.b_mn) {
#pragma unroll
            for (int j = 0; j < BN / CG / 128; ++j) {
              if constexpr (CG == 2) tma_load_3d_2cta(sb + j * BOX_BYTES, &tmB, &full_bar[stage], col0 + j * 128, k0, z);
              else tma_load_3d(sb + j * BOX_BYTES, &tmB, &full_bar[stage], col0 + j * 128, k0, z);
            }
          } else {
            if constexpr (CG == 2) tma_load_3d_2cta(sb, &tmB, &full_bar[stage], k0, col0, z);
            else tma_load_3d(sb, &tmB, &full_bar[stage], k0, col0, z);
          }
          if (++stage == ST) { stage = 0; phase ^= 1; }
        }
      }
      // a block that unwinds leaves no copy in flight
      if (!ok && cta == 0)
        for (int s = 0; s < ST; ++s)
          for (uint32_t it = 0; it < (1u << 16); ++it)
            if (mbar_try_wait(&full_bar[s], 0) || mbar_try_wait(&full_bar[s], 1)) break;
    }
    if (warp == 1 && lane == 0 && cta == 0) {
      // e4m3 operands (format 0), fp32 sums
      const uint32_t idesc = (1u << 4) | static_cast<uint32_t>(p.a_mn) << 15 | static_cast<uint32_t>(p.b_mn) << 16 |
                             static_cast<uint32_t>(BN >> 3) << 17 | static_cast<uint32_t>(BM * CG >> 4) << 24;
      // K-major: 32 bytes along the swizzled row of 128; MN-major: 32 rows of 128 bytes, blocks of 128 wide behind one another
      const uint32_t a_step = p.a_mn ? MMA_K * 128 : MMA_K, b_step = p.b_mn ? MMA_K * 128 : MMA_K;
      const uint32_t a_lbo = p.a_mn ? BOX_BYTES : 16, b_lbo = p.b_mn ? BOX_BYTES : 16;
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true;
      W walk;
      Tile t;
      for (int tile = first; tile < p.num_tiles && ok; tile += step) {
        if (!walk.at(p, tile, t)) break;
        for (int kb = 0; kb < t.kbs; ++kb) {
          if (!(ok = mbar_wait(&tempty_bar[acc], acc_phase ^ 1, abort_flag, 20))) break;
          if (!(ok = mbar_wait(&full_bar[stage], phase, abort_flag, 21))) break;
          tc_fence_after();
          const uint32_t sa = smem_u32(smem + stage * R::STAGE), sb = sa + BM * BK;
#pragma unroll
          for (int kk = 0; kk < BK / MMA_K; ++kk)
            umma_f8<CG>(tmem_base + acc * BN, make_smem_desc(sa + kk * a_step, a_lbo, 1024), make_smem_desc(sb + kk * b_step, b_lbo, 1024),
                        idesc, kk != 0);
          if constexpr (CG == 2) { umma_commit_2cta(&empty_bar[stage], 3); umma_commit_2cta(&tfull_bar[acc], 3); }
          else { umma_commit(&empty_bar[stage]); umma_commit(&tfull_bar[acc]); }
          if (++stage == ST) { stage = 0; phase ^= 1; }
          if (++acc == NACC) { acc = 0; acc_phase ^= 1; }
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 232;\n");
    constexpr int HALF = BN / 2, NP = HALF / 2;
    const int quad = warp & 3, part = (warp - EPI_FIRST) >> 2;
    uint8_t* buf = smem_epi + (warp - EPI_FIRST) * (R::EXTRA / EPI_WARPS);
    [[maybe_unused]] float* sbuf = reinterpret_cast<float*>(buf + WARP_BYTES);
    int acc = 0;
    uint32_t acc_phase = 0;
    bool ok = true;
    W walk;
    Tile t;
    for (int tile = first; tile < p.num_tiles && ok; tile += step) {
      if (!walk.at(p, tile, t)) break;
      if (t.kbs == 0 && p.mode == 2) continue;           // a group without rows leaves its result as it is
      const int in_tile = cta * BM + quad * 32;
      const int rows = max(0, min(32, t.left - in_tile));
      const int col0 = t.tn * BN + part * HALF;
      // (rows and columns outside read a scale that exists; what they compute is not stored)
      const float* sa = p.sa + (min(t.row0 + in_tile + lane, p.M - 1) >> p.sa_shift) * p.sa_m + t.kb0 * p.sa_k;
      const float* sb = p.sb + t.kb0 * p.sb_k + (p.mode == 1 ? t.g * p.sb_g : 0);
      if constexpr (!BVEC) sb += (min(col0, p.N - 1) >> 7) * p.sb_n;
      f32x2 sum[NP];
#pragma unroll
      for (int i = 0; i < NP; ++i) sum[i] = 0;
      for (int kb = 0; kb < t.kbs; ++kb) {
        const float a = sa[kb * p.sa_k];
        [[maybe_unused]] float s = 0.f;
        if constexpr (BVEC) {
#pragma unroll
          for (int j = 0; j < HALF / 32; ++j) {
            const int n = col0 + lane + 32 * j;
            sbuf[(kb & 1) * HALF + lane + 32 * j] = n < p.N ? sb[n * p.sb_n + kb * p.sb_k] : 0.f;
          }
          __syncwarp();
        } else {
          s = a * sb[kb * p.sb_k];
        }
        if (!(ok = mbar_wait(&tfull_bar[acc], acc_phase, abort_flag, 30))) break;
        tc_fence_after();
        const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quad * 32) << 16) + acc * BN + part * HALF;
        const f32x2 s2 = BVEC ? pack2(a, a) : pack2(s, s);
#pragma unroll
        for (int c = 0; c < HALF; c += 32) {
          uint32_t r[32];
          tmem_ld_32x32(taddr + c, r);
          tmem_ld_wait();
          if (c + 32 == HALF) {                          // the last of this block's values are in registers
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
              if constexpr (CG == 2) mbar_arrive_leader(&tempty_bar[acc]);
              else mbar_arrive(&tempty_bar[acc]);
            }
          }
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            f32x2 v = pack2u(r[2 * i], r[2 * i + 1]);
            if constexpr (BVEC) v = mul2(v, *reinterpret_cast<const f32x2*>(&sbuf[(kb & 1) * HALF + c + 2 * i]));
            sum[c / 2 + i] = fma2(v, s2, sum[c / 2 + i]);
          }
        }
        if (++acc == NACC) { acc = 0; acc_phase ^= 1; }
      }
      if (!ok) break;
      store_tile(p, sum, buf, static_cast<long>(t.row0) + in_tile, p.mode == 2 ? t.g * p.d_g : 0, rows, col0, lane);
    }
  }

  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if constexpr (CG == 2) cluster_sync_all();             // the leader's MMAs also write the peer's tensor memory
  if (warp == 1) {
    tc_fence_after();
    if constexpr (CG == 2) tmem_dealloc_2cta(tmem_base, 512);
    else tmem_dealloc(tmem_base, 512);
  }
}

// ------------------------------------------------------------------------------------------------ host side
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                  const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_fn() {
  static const EncodeTiledFn fn = [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess)
      ptr = nullptr;
    return reinterpret_cast<EncodeTiledFn>(ptr);
  }();
  return fn;
}

// Map of `depth` stacked row-major byte matrices (rows x inner), boxes of box_rows x 128 bytes.
int make_map(CUtensorMap* out, const void* base, int rank, uint64_t inner, uint64_t rows, uint64_t depth, uint64_t ld, uint64_t stack,
             uint32_t box_rows) {
  EncodeTiledFn enc = encode_fn();
  if (enc == nullptr) return -100;
  const cuuint64_t dims[3] = {inner, rows, depth}, strides[2] = {ld, stack};
  const cuuint32_t box[3] = {128, box_rows, 1}, es[3] = {1, 1, 1};
  const CUresult r = enc(out, CU_TENSOR_MAP_DATA_TYPE_UINT8, rank, const_cast<void*>(base), dims, strides, box, es,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : -200 - static_cast<int>(r);
}

constexpr int MAX_DEVICES = 64;

int sm_count(int dev) {
  static int counts[MAX_DEVICES];
  if (counts[dev] == 0) {
    int n = 0;
    cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    counts[dev] = n;
  }
  return counts[dev];
}

template <int CG, int BN, bool BVEC>
int launch(const CUtensorMap& ta, const CUtensorMap& tb, const Params& p, int dev, int most, cudaStream_t stream) {
  using R = Ring<CG, BN, BVEC>;
  auto kern = gemm_fp8_kernel<CG, BN, BVEC>;
  static bool configured[MAX_DEVICES];
  if (!configured[dev]) {
    // the warps that ask for registers get them out of the 168 that the others were launched with
    cudaFuncAttributes fa;
    if (cudaFuncGetAttributes(&fa, kern) != cudaSuccess || fa.numRegs != 168) return -301;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, R::TOTAL) != cudaSuccess) return -300;
    configured[dev] = true;
  }
  const int sms = most < CG ? CG : most / CG * CG;
  const long want = static_cast<long>(p.num_tiles) * CG;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(want < sms ? want : sms));
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = R::TOTAL;
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = CG;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, ta, tb, p) == cudaSuccess && cudaGetLastError() == cudaSuccess ? 0 : -400;
}

}  // namespace
}  // namespace ftb

using namespace ftb;

extern "C" {

// The arguments of ftb_gemm_fp8 in 8 bytes each.
struct Fp8GemmArgs {
  const void *A, *B;                  // e4m3; rows start on 16 bytes
  void* D;
  const void* C;                      // or null
  const float *bias, *sa, *sb;
  const int* offsets;                 // of the grouped forms
  // a_mn = 0: A is (M, K), 1: (K, M); b_mn = 0: B is (N, K), 1: (K, N); leading dimensions in bytes (A, B) and elements (D, C)
  int64_t M, N, K, a_mn, b_mn, lda, ldb, ldd, ldc;
  int64_t sa_m, sa_k, sa_shift, sb_n, sb_k, sb_shift, sb_g;
  double alpha, beta;
  int64_t d_fp32;
  int64_t mode, groups, b_g, d_g;     // see Params; b_g: bytes between the groups' B
  int64_t variant, max_ctas;          // 0: by size
  cudaStream_t stream;
};

int ftb_gemm_fp8(const Fp8GemmArgs* a) {
  if (a->M <= 0 || a->N <= 0 || (a->mode != 0 && a->groups <= 0)) return 0;
  if (a->K <= 0) return -1;
  if (((a->lda | a->ldb | a->b_g) & 15) || ((reinterpret_cast<uintptr_t>(a->A) | reinterpret_cast<uintptr_t>(a->B)) & 15)) return -2;
  if (a->M >= 1ll << 31 || a->N >= 1ll << 31 || a->K >= 1ll << 31) return -3;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= MAX_DEVICES) return -4;
  Params p;
  p.M = static_cast<int>(a->M); p.N = static_cast<int>(a->N); p.K = static_cast<int>(a->K);
  p.D = a->D; p.C = a->C != nullptr ? a->C : a->D; p.bias = a->bias;
  p.ldd = a->ldd; p.ldc = a->C != nullptr ? a->ldc : a->ldd;
  p.alpha = static_cast<float>(a->alpha); p.beta = static_cast<float>(a->beta);
  p.d_fp32 = static_cast<int>(a->d_fp32);
  const int64_t es = p.d_fp32 ? 4 : 2;
  p.vec = ((reinterpret_cast<uintptr_t>(p.D) | reinterpret_cast<uintptr_t>(p.C) | static_cast<uintptr_t>(p.N * es) |
            static_cast<uintptr_t>(p.ldd * es) | static_cast<uintptr_t>(p.ldc * es) | static_cast<uintptr_t>(a->mode == 2 ? a->d_g * es : 0)) & 15) == 0;
  p.sa = a->sa; p.sa_m = a->sa_m; p.sa_k = a->sa_k; p.sa_shift = static_cast<int>(a->sa_shift);
  p.sb = a->sb; p.sb_n = a->sb_n; p.sb_k = a->sb_k; p.sb_g = a->sb_g;
  p.a_mn = a->a_mn != 0; p.b_mn = a->b_mn != 0;
  p.mode = static_cast<int>(a->mode); p.groups = static_cast<int>(a->groups); p.offsets = a->offsets; p.d_g = a->d_g;
  p.total = p.mode == 1 ? p.M : p.K;
  p.k_blocks = (p.K + BK - 1) / BK;

  const int variant = a->variant ? static_cast<int>(a->variant) : (p.M >= 512 && p.N >= 512 ? 3 : p.N > 128 && p.M > 128 ? 2 : 1);
  const int cg = variant == 3 ? 2 : 1, bn = variant == 1 ? 128 : 256;
  const int tile_m = BM * cg;
  p.tiles_m = (p.M + tile_m - 1) / tile_m;
  p.tiles_n = (p.N + bn - 1) / bn;
  const int64_t tiles = (p.mode == 2 ? static_cast<int64_t>(p.groups) * p.tiles_m
                                     : p.tiles_m + (p.mode == 1 ? p.groups : 0)) * static_cast<int64_t>(p.tiles_n);
  if (tiles >= 1ll << 30) return -3;
  p.num_tiles = static_cast<int>(tiles);

  CUtensorMap ta, tb;
  const uint64_t z = p.mode == 1 ? p.groups : 1;
  int rc = p.a_mn ? make_map(&ta, a->A, 2, p.M, p.K, 1, a->lda, 0, 128) : make_map(&ta, a->A, 2, p.K, p.M, 1, a->lda, 0, 128);
  if (rc) return rc;
  // (a stack of one has no stride of its own)
  const uint64_t stack = z > 1 ? a->b_g : (p.b_mn ? p.K : p.N) * static_cast<uint64_t>(a->ldb);
  rc = p.b_mn ? make_map(&tb, a->B, 3, p.N, p.K, z, a->ldb, stack, 128) : make_map(&tb, a->B, 3, p.K, p.N, z, a->ldb, stack, bn / cg);
  if (rc) return rc;
  const int sms = sm_count(dev), most = a->max_ctas > 0 && a->max_ctas < sms ? static_cast<int>(a->max_ctas) : sms;
  const bool bvec = a->sb_shift == 0;
  if (variant == 1) return bvec ? launch<1, 128, true>(ta, tb, p, dev, most, a->stream) : launch<1, 128, false>(ta, tb, p, dev, most, a->stream);
  if (variant == 2) return bvec ? launch<1, 256, true>(ta, tb, p, dev, most, a->stream) : launch<1, 256, false>(ta, tb, p, dev, most, a->stream);
  return bvec ? launch<2, 256, true>(ta, tb, p, dev, most, a->stream) : launch<2, 256, false>(ta, tb, p, dev, most, a->stream);
}

// (and clears it) code * 1000 + where of a wait that ran out, 0 if none did
int ftb_gemm_fp8_error(void) {
  int h[2] = {0, 0};
  cudaMemcpyFromSymbol(&h[0], g_error_word, sizeof(int));
  cudaMemcpyFromSymbol(&h[1], g_error_where, sizeof(int));
  if (h[0] != 0) {
    const int z = 0;
    cudaMemcpyToSymbol(g_error_word, &z, sizeof(int));
    cudaMemcpyToSymbol(g_error_where, &z, sizeof(int));
  }
  return h[0] * 1000 + h[1];
}

}  // extern "C"
