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
//   warps 1, 2 tcgen05.mma, one thread each: one half of the tile's 256 columns each (128 columns: warp 1, all of them)
//   warps 4-11 four for each half: read out, scale and add; at the end of a tile turn it over in shared memory and store whole pieces of rows
//              (a thread's 128 sums, and 32 values on the way, need more than the 168 registers of 384 threads: the first four
//              warps give theirs up)
//
// SPLIT: products with few tiles.  A cluster of up to four CTAs takes one tile, a range of the reduction each; the parts are added
// through the cluster's shared memory, in the order of the ranges, so that results do not depend on who comes first.
//
// CG = 2: a pair of SMs works on 256 x BN (each CTA 128 rows, half of B).  Grouped forms take their row or reduction ranges
// from device offsets.  Every wait is bounded.
//
// What bounds it.  A block of 256 x 256 x 128 takes a pair of SMs some 1035 cycles of the 512 that the tensor cores would need: an
// accumulator is multiplied (400 cycles for a half, 400 behind the other half), seen to be complete (250), read out (490), released
// across the pair and multiplied into again (530), 2070 in all, and each half has two of them in tensor memory.  Sustained, power
// does: 16384 x 28672 x 4096 runs at 1.56 GHz (without additions and without reading tensor memory, 1890 us at 1.52 GHz; the library's
// product with one scale for everything, which accumulates in tensor memory throughout, 1535).  Measured beside 2390 us of that
// product: one thread and one product for all 256 columns 2540, which reads A once but lets both halves wait for one another; tiles of
// 256 x 128 with four accumulators 3070; sixteen warps of 64 columns each 3050; additions on pairs of fp32 2360; chunks of 32 columns
// 2480 (registers spilled).  What brought it to 2290: four products in one piece of code, C on its way before the loop over the blocks
// and not within it, and warps without rows in a loop of their own.  Back to back for a second:
//   16384 x 28672 x 4096      2.29 ms  1680 TFLOP/s      8192 x 4096 x 14336, B across     560 us  1718 TFLOP/s
//   3001 x 4096 x 14336 + C    233 us  1510 TFLOP/s      4096 x 2048 x 9377, both across   134 us  1178 TFLOP/s (column scales)
//   14336 x 4096 x 16384      1.18 ms  1626 TFLOP/s (weight gradient, B in blocks; in columns 1.51 ms)
// 16384 x 28672 x 4096 takes 1.95 ms, 1974 TFLOP/s, where the power limit is not reached.  Few rows, in a graph, the weight in the second
// level of cache: 16 x 4096 x 4096 8.2 us, 1 x 14336 x 4096 15.9, 1 x 4096 x 14336 15.0; from memory 10 and 18.5 for the first two, of which
// some 8 are the launch, the start and the end (twice the stages in flight: the same).
#include <type_traits>

#include "ptx.cuh"

namespace ftb {
namespace {

constexpr int BM = 128, BK = 128, MMA_K = 32;
constexpr int EPI_WARPS = 8, EPI_FIRST = 4, THREADS = 32 * (EPI_FIRST + EPI_WARPS);
constexpr int PIECE_BYTES = 32 * 128;                    // a warp's piece of shared memory: 32 rows x 128 bytes
constexpr int BOX_BYTES = 128 * 128;

// The four products of a stage (e4m3 x e4m3, fp32 sums from zero on), as one piece: a thread that puts descriptors together
// between them takes longer than the tensor core.  Descriptors come in halves, of which the lower one holds the address in units
// of 16 bytes; a_step and b_step are those units from one product to the next.
#define FTB_MMA4(CG_)                                                                                                          \
  asm volatile(                                                                                                                \
      "{\n.reg .pred z, a;\n.reg .b32 x, y;\n.reg .b64 da, db;\n"                                                             \
      "setp.ne.b32 z, 0, 0;\nsetp.eq.b32 a, 0, 0;\n"                                                                           \
      "mov.b64 da, {%1, %2};\nmov.b64 db, {%3, %4};\n"                                                                         \
      "tcgen05.mma.cta_group::" CG_ ".kind::f8f6f4 [%0], da, db, %7, z;\n"                                                     \
      "add.u32 x, %1, %5;\nadd.u32 y, %3, %6;\nmov.b64 da, {x, %2};\nmov.b64 db, {y, %4};\n"                                  \
      "tcgen05.mma.cta_group::" CG_ ".kind::f8f6f4 [%0], da, db, %7, a;\n"                                                     \
      "add.u32 x, x, %5;\nadd.u32 y, y, %6;\nmov.b64 da, {x, %2};\nmov.b64 db, {y, %4};\n"                                    \
      "tcgen05.mma.cta_group::" CG_ ".kind::f8f6f4 [%0], da, db, %7, a;\n"                                                     \
      "add.u32 x, x, %5;\nadd.u32 y, y, %6;\nmov.b64 da, {x, %2};\nmov.b64 db, {y, %4};\n"                                    \
      "tcgen05.mma.cta_group::" CG_ ".kind::f8f6f4 [%0], da, db, %7, a;\n}\n" ::"r"(tmem_d),                                   \
      "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(a_step), "r"(b_step), "r"(idesc)                                         \
      : "memory")
template <int CG>
__device__ __forceinline__ void umma4_f8(uint32_t tmem_d, uint32_t a_lo, uint32_t a_hi, uint32_t b_lo, uint32_t b_hi, uint32_t a_step,
                                         uint32_t b_step, uint32_t idesc) {
  static_assert(BK / MMA_K == 4, "four products of a stage");
  if constexpr (CG == 1) FTB_MMA4("1");
  else FTB_MMA4("2");
}

// whether a phase is complete, without waiting for it
__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile("{\n.reg .pred p;\nmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}\n"
               : "=r"(ok)
               : "r"(smem_u32(bar)), "r"(parity)
               : "memory");
  return ok != 0;
}

#define FTB_R16 "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}"
#define FTB_OUT16(r)                                                                                                           \
  "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),       \
      "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
// 16 lanes x 32 columns: r[4 j + 2 e + i] is lane 8 e + (thread >> 2), column 8 j + 2 (thread & 3) + i
__device__ __forceinline__ void tmem_ld_16x32(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile("tcgen05.ld.sync.aligned.16x256b.x4.b32 " FTB_R16 ", [%16];" : FTB_OUT16(r) : "r"(taddr) : "memory");
}
// sum += v * f * a on pairs of fp32 in two instructions
__device__ __forceinline__ void mul_add2(float* sum, const uint32_t* v, float2 f, float a) {
  unsigned long long x, y, z, w;
  asm("mov.b64 %0, {%1, %2};" : "=l"(x) : "r"(v[0]), "r"(v[1]));
  asm("mov.b64 %0, {%1, %2};" : "=l"(y) : "f"(f.x), "f"(f.y));
  asm("mov.b64 %0, {%1, %1};" : "=l"(w) : "f"(a));
  asm("mov.b64 %0, {%1, %2};" : "=l"(z) : "f"(sum[0]), "f"(sum[1]));
  asm("mul.rn.f32x2 %0, %0, %1;" : "+l"(x) : "l"(y));
  asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(z) : "l"(x), "l"(w));
  asm("mov.b64 {%0, %1}, %2;" : "=f"(sum[0]), "=f"(sum[1]) : "l"(z));
}
// a row of 16 columns for each thread
__device__ __forceinline__ void tmem_ld_row16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 " FTB_R16 ", [%16];" : FTB_OUT16(r) : "r"(taddr) : "memory");
}

// Tiled stores of a box of shared memory, and its addition to fp32 values where they lie.
__device__ __forceinline__ void tma_store_3d(const CUtensorMap* m, const void* src, int x, int y, int z) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%1, %2, %3}], [%4];" ::"l"(reinterpret_cast<uint64_t>(m)),
               "r"(x), "r"(y), "r"(z), "r"(smem_u32(src))
               : "memory");
}
__device__ __forceinline__ void tma_add_3d(const CUtensorMap* m, const void* src, int x, int y, int z) {
  asm volatile("cp.reduce.async.bulk.tensor.3d.global.shared::cta.add.tile.bulk_group [%0, {%1, %2, %3}], [%4];" ::"l"(reinterpret_cast<uint64_t>(m)),
               "r"(x), "r"(y), "r"(z), "r"(smem_u32(src))
               : "memory");
}
template <int N>
__device__ __forceinline__ void bulk_wait_read() { asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory"); }

struct Params {
  int M, N, K;
  void* D;
  const void* C;
  const float* bias;
  long ldd, ldc;                     // elements
  float alpha, beta;
  int d_fp32, vec;                   // vec: rows of D and C in pieces of 16 bytes
  int add_in_place;                  // C is D, in fp32 with beta = 1: the sums are added to it where it lies, and C is not read
  const float* sa;                   // scale of row m and block kb at sa[(m >> sa_shift) * sa_m + kb * sa_k]
  long sa_m, sa_k;
  int sa_shift;
  const float* sb;                   // scale of column n at sb[(n >> 7, or n) * sb_n + kb * sb_k]
  long sb_n, sb_k, sb_g;
  int a_mn, b_mn;
  int stage_bytes;                   // that a CTA's copies of a stage bring
  // mode 0 one product; 1 row segments, each with a B of its own; 2 segments of the reduction, each with a D of its own
  int mode, groups;
  const int* offsets;
  long d_g;                          // mode 2: elements between the groups' results
  int total;                         // rows that the offsets run over
  int tiles_m, tiles_n, num_tiles, k_blocks;
  int split_blocks;                  // SPLIT: blocks of a CTA's range (the last one's may be shorter)
};

struct Tile {
  int row0, left, tn, g, kb0, kbs;    // kbs: blocks of the reduction; -1 for a segment that is left out
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
      // A segment that starts or ends inside a group of 128 would take its neighbour's rows along, whose scales are the same: it is left
      // out, and reported.
      if (t.kbs > 0 && (p.offsets[t.g] % BK != 0 || (p.offsets[t.g + 1] % BK != 0 && p.offsets[t.g + 1] < p.total))) t.kbs = -1;
    }
    const int per_group = GM * p.tiles_n, grp = tile / per_group;
    const int gm = min(GM, p.tiles_m - grp * GM), r = tile - grp * per_group;
    t.row0 = (grp * GM + r % gm) * TM;
    t.tn = r / gm;
    t.left = p.M - t.row0;
    return true;
  }
};

constexpr int C_BUFS = 2;                                // pieces of C under way for a warp
constexpr int SLOTS = 3;                                 // blocks of scales under way for a warp (BVEC)

template <int CG, int BN, bool BVEC>
struct Ring {
  static constexpr int B_BYTES = BN / CG * BK;
  static constexpr int STAGE = BM * BK + B_BYTES;
  static constexpr int SLOT = BN / 2 + 32;                // column scales of a half, then row scales of a warp
  static constexpr int WARP = C_BUFS * PIECE_BYTES + (BVEC ? SLOTS * SLOT * 4 : 0);
  static constexpr int STAGES = (227 * 1024 - 1024 - 512 - EPI_WARPS * WARP) / STAGE;
  static constexpr int TOTAL = STAGES * STAGE + EPI_WARPS * WARP + 512 + 1024;
  static constexpr int NACC = 512 / BN;              // accumulators of each issuer
  // (128 columns have four accumulators as they are, and A is read once: 1024 x 2048 x 2048 14.3 -> 13.4 us, 4096 x 4096 x 4096 in
  // such tiles 108 -> 105, where the second level of cache brings 10 TB/s)
  static constexpr int ISSUERS = BN == 128 ? 1 : 2;
  static_assert(STAGES >= 3 && 2 * STAGES + 4 * NACC + 1 <= 64, "barriers in 512 bytes");
};

__device__ __forceinline__ void cp_async16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
// four bytes, or zeros in their place
__device__ __forceinline__ void cp_async4(void* dst, const void* src, bool there) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(there ? 4 : 0) : "memory");
}
// two bytes, or zeros in their place without looking there
__device__ __forceinline__ uint16_t load_u16(const uint16_t* x, bool there) {
  uint16_t v;
  asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %2, 0;\nmov.b16 %0, 0;\n@p ld.global.u16 %0, [%1];\n}\n" : "=h"(v) : "l"(x), "r"(static_cast<int>(there)) : "memory");
  return v;
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// all of the thread's copies, committed or not
__device__ __forceinline__ void cp_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// 32 rows x 128 bytes of a warp in 16-byte pieces, free of bank conflicts row-wise and piece-wise
__device__ __forceinline__ uint4* piece_at(uint8_t* buf, int row, int piece) {
  return reinterpret_cast<uint4*>(buf + row * 128 + ((piece ^ (row & 7)) << 4));
}
__device__ __forceinline__ uint8_t* byte_at(uint8_t* buf, int row, int byte) {
  return buf + row * 128 + (((byte >> 4) ^ (row & 7)) << 4) + (byte & 15);
}

// Where a warp's part of a tile lies in D and C: 32 rows (so many of them real) from column col0 on.  A step is 128 bytes of a row.
struct Patch {
  uint8_t* d;
  const uint8_t* c;
  long ldd, ldc;                     // bytes
  int rows, cols;                    // cols: from col0 to the end of a row of D
};
// First column, from col0 on, of a thread's columns c, c + 1, ...: a pair of SMs has 64 of each 128 in a half of its tile.
template <int CG>
__device__ __forceinline__ constexpr int column(int c) { return CG == 1 ? c : (c >> 6) * 128 + (c & 63); }

// the step of C from column col on its way into a piece of shared memory (complete after a wait for the thread's copies and a __syncwarp)
__device__ __forceinline__ void fetch_c(const Patch& w, int es, int vec, int col, uint8_t* buf, int lane) {
  const int bytes = min(128, (w.cols - col) * es);
  const uint8_t* c = w.c + col * es;
  if (vec) {
    const int lr = lane >> 3, lp = lane & 7;
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k * 4 + lr < w.rows && lp * 16 < bytes) cp_async16(piece_at(buf, k * 4 + lr, lp), c + (k * 4 + lr) * w.ldc + lp * 16);
  } else if (es == 4) {
    c += lane * 4;
    if (lane * 4 < bytes)
      for (int r0 = 0; r0 < w.rows; r0 += 8) {
#pragma unroll
        for (int i = 0; i < 8; ++i, c += w.ldc)            // (eight rows: their places in the piece are the lane's and constants)
          if (r0 + i < w.rows) cp_async4(byte_at(buf + r0 * 128, i, lane * 4), c, true);
      }
  } else {
    // Two elements of a row for each lane: as one copy where they lie on four bytes, else loads for eight rows before their stores.
    const int at = lane * 4, n = min(2, (bytes - at) >> 1);
    const uint16_t* from = reinterpret_cast<const uint16_t*>(c + at);
    const long ld = w.ldc >> 1;
    if (n > 0)
      for (int r0 = 0; r0 < w.rows; r0 += 8, from += 8 * ld) {
        uint16_t lo[8], hi[8];
        bool apart[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint16_t* x = from + i * ld;
          apart[i] = r0 + i < w.rows && (n != 2 || (reinterpret_cast<uintptr_t>(x) & 3) != 0);
          if (r0 + i < w.rows && !apart[i]) cp_async4(byte_at(buf + r0 * 128, i, at), x, true);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {                      // (predicates, no branches: a branch would wait for its own load)
          lo[i] = load_u16(from + i * ld, apart[i]);
          hi[i] = load_u16(from + i * ld + 1, apart[i] && n == 2);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (apart[i]) *reinterpret_cast<uint32_t*>(byte_at(buf + r0 * 128, i, at)) = lo[i] | static_cast<uint32_t>(hi[i]) << 16;
      }
  }
}
// (add: to what lies there, in fp32)
__device__ __forceinline__ void store_d(const Patch& w, int es, int vec, bool add, int col, uint8_t* buf, int lane) {
  const int bytes = min(128, (w.cols - col) * es);
  uint8_t* d = w.d + col * es;
  if (es == 4 && (add || !vec)) {
    d += lane * 4;
    if (lane * 4 < bytes)
      for (int r0 = 0; r0 < w.rows; r0 += 8) {
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = *reinterpret_cast<const float*>(byte_at(buf + r0 * 128, i, lane * 4));
#pragma unroll
        for (int i = 0; i < 8; ++i, d += w.ldd) {
          if (r0 + i >= w.rows) break;
          // (each element is added to once: the order of the additions is that of the launches)
          if (add) asm volatile("red.global.add.f32 [%0], %1;" ::"l"(d), "f"(v[i]) : "memory");
          else *reinterpret_cast<float*>(d) = v[i];
        }
      }
  } else if (vec) {
    const int lr = lane >> 3, lp = lane & 7;
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k * 4 + lr < w.rows && lp * 16 < bytes) *reinterpret_cast<uint4*>(d + (k * 4 + lr) * w.ldd + lp * 16) = *piece_at(buf, k * 4 + lr, lp);
  } else {
    const int at = lane * 4, n = min(2, (bytes - at) >> 1);
    uint16_t* to = reinterpret_cast<uint16_t*>(d + at);
    const long ld = w.ldd >> 1;
    if (n > 0)
      for (int r0 = 0; r0 < w.rows; r0 += 8) {
        uint32_t v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = *reinterpret_cast<const uint32_t*>(byte_at(buf + r0 * 128, i, at));
#pragma unroll
        for (int i = 0; i < 8; ++i, to += ld) {
          if (r0 + i >= w.rows) break;
          if (n == 2 && (reinterpret_cast<uintptr_t>(to) & 3) == 0) {
            *reinterpret_cast<uint32_t*>(to) = v[i];
          } else {
            to[0] = static_cast<uint16_t>(v[i]);
            if (n == 2) to[1] = static_cast<uint16_t>(v[i] >> 16);
          }
        }
      }
  }
}

// A warp's 32 rows of NC sums: alpha, bias, C, rounding once, and out step by step.  ROWS: a thread has a row of them, else the
// fragments of tmem_ld_16x32, 32 columns after 32 columns.  The first C_BUFS steps of C are under way already, in the pieces of
// buf.  Whole patches leave as tiled copies, of which the thread does not see the end; `map` is null for patches whose last rows
// are another group's, and for rows off the 16-byte grid.
template <bool FP32, bool ROWS, int CG, int NC>
__device__ __forceinline__ void store_tile(const Params& p, const float (&sum)[NC], const Patch& w, const float* bias, uint8_t* buf,
                                           const CUtensorMap* map, int x, int y, int z, bool add, int lane) {
  constexpr int ES = FP32 ? 4 : 2, STEP = 128 / ES, STEPS = NC / STEP, TURN = STEPS < C_BUFS ? STEPS : C_BUFS;
#pragma unroll
  for (int turn = 0; turn < STEPS; turn += TURN) {         // as many steps at a time as there are pieces
    if (w.cols <= column<CG>(turn * STEP)) break;
    if (add) {
      cp_wait_all();
      __syncwarp();
    } else if (turn > 0) {
      if (lane == 0) bulk_wait_read<0>();                  // the stores of the last turn have read the pieces
      __syncwarp();
    }
#pragma unroll
    for (int i = turn; i < turn + TURN; ++i) {
      const int col = column<CG>(i * STEP), cols = w.cols - col;
      if (cols <= 0) break;
      uint8_t* at = buf + (i % C_BUFS) * PIECE_BYTES;
      // (PLAIN: neither C nor bias; the tests for them, element by element, took four times as long as the rest)
      auto write = [&](auto plain) {
        constexpr bool PLAIN = decltype(plain)::value;
        if constexpr (ROWS) {
#pragma unroll
          for (int q = 0; q < 8; ++q) {
            uint4* pc = piece_at(at, lane, q);
            constexpr int E = 16 / ES;                     // elements of a piece
            float v[E];
#pragma unroll
            for (int j = 0; j < E; ++j) v[j] = sum[i * STEP + q * E + j] * p.alpha;
            if constexpr (!PLAIN) {
              if (bias != nullptr) {
#pragma unroll
                for (int j = 0; j < E; ++j)
                  if (q * E + j < cols) v[j] += bias[col + q * E + j];
              }
              if (add) {
                const uint4 cu = *pc;
                const uint32_t cw[4] = {cu.x, cu.y, cu.z, cu.w};
#pragma unroll
                for (int j = 0; j < E; ++j)
                  v[j] += p.beta * __uint_as_float(FP32 ? cw[j % 4] : j & 1 ? cw[j / 2] & 0xFFFF0000u : cw[j / 2] << 16);
              }
            }
            uint32_t ow[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              if constexpr (FP32) {
                ow[j] = __float_as_uint(v[j]);
              } else {
                const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
                ow[j] = *reinterpret_cast<const uint32_t*>(&h);
              }
            }
            *pc = make_uint4(ow[0], ow[1], ow[2], ow[3]);
          }
        } else {
#pragma unroll
          for (int c = 0; c < STEP; c += 32)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int e0 = c + 8 * j + 2 * (lane & 3);     // in the step
              float b0 = 0.f, b1 = 0.f;
              if constexpr (!PLAIN) {
                if (bias != nullptr && e0 < cols) b0 = bias[col + e0];
                if (bias != nullptr && e0 + 1 < cols) b1 = bias[col + e0 + 1];
              }
#pragma unroll
              for (int k = 0; k < 4; ++k) {                  // rows 8 k + (lane >> 2)
                const float* f = &sum[((i * STEP + c) / 32 * 2 + (k >> 1)) * 16 + 4 * j + 2 * (k & 1)];
                float v0 = f[0] * p.alpha + b0, v1 = f[1] * p.alpha + b1;
                uint8_t* to = byte_at(at, 8 * k + (lane >> 2), e0 * ES);
                if constexpr (!PLAIN) {
                  if (add) {
                    const float2 cc = FP32 ? *reinterpret_cast<const float2*>(to) : __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(to));
                    v0 += p.beta * cc.x;
                    v1 += p.beta * cc.y;
                  }
                }
                if constexpr (FP32) *reinterpret_cast<float2*>(to) = make_float2(v0, v1);
                else *reinterpret_cast<__nv_bfloat162*>(to) = __floats2bfloat162_rn(v0, v1);
              }
            }
        }
      };
      if (bias == nullptr && !add) write(std::true_type());
      else write(std::false_type());
    }
    if (map != nullptr) fence_proxy_async();
    __syncwarp();
#pragma unroll
    for (int i = turn; i < turn + TURN; ++i) {
      const int col = column<CG>(i * STEP);
      if (w.cols <= col) break;
      uint8_t* at = buf + (i % C_BUFS) * PIECE_BYTES;
      if (map == nullptr) store_d(w, ES, p.vec, FP32 && p.add_in_place, col, at, lane);
      else if (lane == 0 && FP32 && p.add_in_place) tma_add_3d(map, at, x + col, y, z);
      else if (lane == 0) tma_store_3d(map, at, x + col, y, z);
    }
    if (map == nullptr) __syncwarp();
    else if (lane == 0) bulk_commit();
    if (add && turn + TURN < STEPS) {
      if (lane == 0) bulk_wait_read<0>();
      __syncwarp();
#pragma unroll
      for (int i = turn + TURN; i < turn + 2 * TURN; ++i)
        if (w.cols > column<CG>(i * STEP)) fetch_c(w, ES, p.vec, column<CG>(i * STEP), buf + (i % C_BUFS) * PIECE_BYTES, lane);
    }
  }
}

// A CTA's part of a tile of 128 x 128 fp32 sums in its shared memory: 16-byte pieces turned over by the row's number.
__device__ __forceinline__ uint32_t part_offset(int row, int piece) { return row * 512 + ((piece ^ (row & 31)) << 4); }
__device__ __forceinline__ float4 ld_cluster(uint32_t local, int rank) {
  uint32_t at;
  float4 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(local), "r"(rank));
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at) : "memory");
  return v;
}

template <int CG, int BN, bool BVEC, bool SPLIT>
__global__ void __launch_bounds__(THREADS, 1)
gemm_fp8_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const __grid_constant__ CUtensorMap tmD,
                const Params p) {
  using R = Ring<CG, BN, BVEC>;
  using W = Walk<BM * CG, 16 / CG>;
  constexpr int ST = R::STAGES, NACC = R::NACC, HALF = BN / 2;
  static_assert(!SPLIT || (CG == 1 && BN == 128 && ST * R::STAGE >= 128 * 512), "the parts lie where the stages were");
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* smem_epi = smem + ST * R::STAGE;
  uint8_t* smem_slots = smem_epi + EPI_WARPS * C_BUFS * PIECE_BYTES;
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem_epi + EPI_WARPS * R::WARP);
  uint64_t* empty_bar = full_bar + ST;
  uint64_t* tfull_bar = empty_bar + ST;
  uint64_t* tempty_bar = tfull_bar + 2 * NACC;            // (of the first issuer, then of the second)
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty_bar + 2 * NACC);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int cta = CG == 2 ? static_cast<int>(cluster_ctarank()) : 0;
  uint32_t ranges = 1;
  if constexpr (SPLIT) asm volatile("mov.u32 %0, %cluster_nctaid.x;" : "=r"(ranges));
  const int range = SPLIT ? static_cast<int>(cluster_ctarank()) : 0;
  const int first = SPLIT ? blockIdx.x / ranges : blockIdx.x / CG, step = SPLIT ? p.num_tiles : gridDim.x / CG;
  auto locate = [&](W& walk, int tile, Tile& t) {
    if (!walk.at(p, tile, t)) return false;
    if constexpr (SPLIT) {
      t.kb0 = range * p.split_blocks;
      t.kbs = min(p.split_blocks, p.k_blocks - t.kb0);
    }
    return true;
  };

  if (threadIdx.x == 0) {
    *abort_flag = 0;
    for (int s = 0; s < ST; ++s) { mbar_init(&full_bar[s], 1); mbar_init(&empty_bar[s], R::ISSUERS); }
    for (int a = 0; a < 2 * NACC; ++a) { mbar_init(&tfull_bar[a], 1); mbar_init(&tempty_bar[a], CG * EPI_WARPS / R::ISSUERS); }
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
        if (!locate(walk, tile, t)) break;
        const int row0 = t.row0 + cta * BM;
        const int col0 = t.tn * BN + cta * (BN / CG);
        const int z = p.mode == 1 ? t.g : 0;
        if (t.kbs < 0) set_error(3, 40);
        for (int kb = 0; kb < t.kbs; ++kb) {
          if (!(ok = mbar_wait(&empty_bar[stage], phase ^ 1, abort_flag, 10))) break;
          uint8_t* sa = smem + stage * R::STAGE;
          uint8_t* sb = sa + BM * BK;
          if (cta == 0) mbar_expect_tx(&full_bar[stage], CG * p.stage_bytes);
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
    if ((warp == 1 || (warp == 2 && R::ISSUERS == 2)) && lane == 0 && cta == 0) {
      // A barrier's word is some 250 cycles away while the tensor core reads shared memory, a block's products take 512.  So a
      // thread asks for both of its barriers at once, and each half of the columns has a thread and accumulators of its own: a
      // half is multiplied while the other one's are read out.
      const int half = warp - 1;
      uint64_t *tfull = tfull_bar + half * NACC, *tempty = tempty_bar + half * NACC;
      const uint32_t tmem_half = tmem_base + half * NACC * HALF;
      constexpr int WIDE = BN / R::ISSUERS;
      // e4m3 operands (format 0), fp32 sums
      const uint32_t idesc = (1u << 4) | static_cast<uint32_t>(p.a_mn) << 15 | static_cast<uint32_t>(p.b_mn) << 16 |
                             static_cast<uint32_t>(WIDE >> 3) << 17 | static_cast<uint32_t>(BM * CG >> 4) << 24;
      // K-major: 32 bytes along the swizzled row of 128; MN-major: 32 rows of 128 bytes, blocks of 128 wide behind one another
      const uint32_t a_step = (p.a_mn ? MMA_K * 128 : MMA_K) >> 4, b_step = (p.b_mn ? MMA_K * 128 : MMA_K) >> 4;
      // the half's columns of this CTA's part of B: rows of it, or bytes of its rows, or its second box
      constexpr int OWN = WIDE / CG;
      const uint32_t b_off = half * (p.b_mn ? (OWN == 128 ? BOX_BYTES : OWN) : OWN * 128);
      const uint64_t a_desc = make_smem_desc(smem_u32(smem), p.a_mn ? BOX_BYTES : 16, 1024);
      const uint64_t b_desc = make_smem_desc(smem_u32(smem) + BM * BK + b_off, p.b_mn ? BOX_BYTES : 16, 1024);
      const uint32_t a_lo = static_cast<uint32_t>(a_desc), a_hi = static_cast<uint32_t>(a_desc >> 32);
      const uint32_t b_lo = static_cast<uint32_t>(b_desc), b_hi = static_cast<uint32_t>(b_desc >> 32);
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true;
      W walk;
      Tile t;
      for (int tile = first; tile < p.num_tiles && ok; tile += step) {
        if (!locate(walk, tile, t)) break;
        for (int kb = 0; kb < t.kbs; ++kb) {
          const bool e = mbar_try_wait(&tempty[acc], acc_phase ^ 1), f = mbar_try_wait(&full_bar[stage], phase);
          if (!e && !(ok = mbar_wait(&tempty[acc], acc_phase ^ 1, abort_flag, 20))) break;
          if (!f && !(ok = mbar_wait(&full_bar[stage], phase, abort_flag, 21))) break;
          tc_fence_after();
          const uint32_t at = stage * (R::STAGE >> 4);
          umma4_f8<CG>(tmem_half + acc * WIDE, a_lo + at, a_hi, b_lo + at, b_hi, a_step, b_step, idesc);
          if constexpr (CG == 2) { umma_commit_2cta(&tfull[acc], 3); umma_commit_2cta(&empty_bar[stage], 3); }
          else { umma_commit(&tfull[acc]); umma_commit(&empty_bar[stage]); }
          if (++stage == ST) { stage = 0; phase ^= 1; }
          if (++acc == NACC) { acc = 0; acc_phase ^= 1; }
        }
      }
    }
    if constexpr (SPLIT) {                               // (the others' two barriers, see there)
      __syncwarp();
      cluster_sync_all();
      cluster_sync_all();
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 232;\n");
    constexpr int SEG = CG, SEG_COLS = HALF / SEG;         // (a half of a pair's tile has columns of two blocks of 128)
    constexpr int AHEAD = 2;
    static_assert(AHEAD < SLOTS, "a slot is written when all lanes have read it");
    const int quad = warp & 3, part = (warp - EPI_FIRST) >> 2;
    uint8_t* buf = smem_epi + (warp - EPI_FIRST) * (C_BUFS * PIECE_BYTES);
    [[maybe_unused]] float* slots = reinterpret_cast<float*>(smem_slots) + (warp - EPI_FIRST) * (SLOTS * R::SLOT);
    const int in_tile = cta * BM + quad * 32, es = p.d_fp32 ? 4 : 2;
    const bool add = !SPLIT && p.beta != 0.f && !p.add_in_place;
    uint64_t *tfull = tfull_bar + (R::ISSUERS == 2 ? part * NACC : 0), *tempty = tempty_bar + (R::ISSUERS == 2 ? part * NACC : 0);
    const uint32_t tmem_part = tmem_base + (static_cast<uint32_t>(quad * 32) << 16) + part * (R::ISSUERS == 2 ? NACC * HALF : HALF);
    constexpr int ACC_STEP = BN / R::ISSUERS;
    int acc = 0;
    uint32_t acc_phase = 0;
    [[maybe_unused]] int slot = 0;                  // of the next block of scales to be asked for
    W walk;
    Tile t = {};
    const float *sa = nullptr, *sb = nullptr;            // of the next block to be asked for
    [[maybe_unused]] long sb_seg = 0;
    int asked = 0;
    [[maybe_unused]] int sb_left = 0;
    // scales of the next blocks, asked for that much before they are needed: in registers (a row's, and those of its blocks of
    // columns), or, of columns, in shared memory
    [[maybe_unused]] float a_next[AHEAD], b_next[SEG][AHEAD];
    auto ask = [&](int to) {
      const bool there = asked++ < t.kbs;
      if constexpr (BVEC) {
        float* at = slots + slot * R::SLOT + lane;
        slot = slot + 1 == SLOTS ? 0 : slot + 1;
        if (there) {
#pragma unroll
          for (int j = 0; j < HALF / 32; ++j) {
            const bool in = column<CG>(32 * j) < sb_left;
            cp_async4(at + 32 * j, sb + (in ? column<CG>(32 * j) * p.sb_n : 0), in);
          }
          cp_async4(at + HALF, sa, true);
        }
        cp_commit();
      } else if (there) {
        a_next[to] = *sa;
#pragma unroll
        for (int g = 0; g < SEG; ++g) b_next[g][to] = sb[g * sb_seg];
      }
      sa += p.sa_k;
      sb += p.sb_k;
    };
    // the tile's place and the scales of its first blocks; -1 behind the last tile
    auto begin = [&](int tile) {
      do {
        if (tile >= p.num_tiles || !locate(walk, tile, t)) return -1;
        if (t.kbs > 0) break;                            // (a group without rows, or left out, leaves its result as it is)
        tile += step;
      } while (true);
      // (rows and columns outside read a scale that exists; what they compute is not stored)
      sa = p.sa + (min(t.row0 + in_tile + lane, p.M - 1) >> p.sa_shift) * p.sa_m + t.kb0 * p.sa_k;
      sb = p.sb + t.kb0 * p.sb_k + (p.mode == 1 ? t.g * p.sb_g : 0);
      if constexpr (BVEC) {
        const int n = t.tn * BN + part * SEG_COLS + lane;
        sb_left = p.N - n;
        if (sb_left > 0) sb += n * p.sb_n;
      }
      if constexpr (!BVEC) {
        const int n0 = t.tn * BN + part * SEG_COLS;
        sb += (min(n0, p.N - 1) >> 7) * p.sb_n;
        sb_seg = SEG == 2 && n0 + 128 < p.N ? p.sb_n : 0;
      }
      asked = 0;
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) ask(i);
      return tile;
    };
    bool ok = true, ready = false;
    for (int tile = begin(first); tile >= 0;) {
      const int row = t.row0 + in_tile, rows = max(0, min(32, t.left - in_tile)), col0 = t.tn * BN + part * SEG_COLS, kbs = t.kbs, g = t.g;
      auto patch = [&] {
        Patch w;
        w.rows = rows;
        w.cols = rows > 0 ? max(0, min(SEG * 128 - (SEG - 1) * 64, p.N - col0)) : 0;
        const long skip = p.mode == 2 ? g * p.d_g : 0;
        w.ldd = p.ldd * es;
        w.ldc = p.ldc * es;
        w.d = static_cast<uint8_t*>(p.D) + (skip + row * p.ldd + col0) * es;
        w.c = static_cast<const uint8_t*>(p.C) + (skip + row * p.ldc + col0) * es;
        return w;
      };
      // The first steps of C are on their way during the whole reduction.  (Asked for from inside the loop over the blocks, the
      // code for it slows the loop, C or no C: 581 us for 745 of 8192 x 4096 x 14336.)
      if (add) {
        if (lane == 0) bulk_wait_read<0>();                // the last tile's stores have read the pieces
        __syncwarp();
        const Patch w = patch();
        const int first_steps = min(C_BUFS, HALF * es / 128);
        for (int i = 0; i < first_steps; ++i) {
          const int col = column<CG>(i * (128 / es));
          if (w.cols > col) fetch_c(w, es, p.vec, col, buf + i * PIECE_BYTES, lane);
        }
      }
      float sum[HALF];
#pragma unroll
      for (int i = 0; i < HALF; ++i) sum[i] = 0.f;
      auto release = [&] {                               // the last of a block's values are in registers
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if constexpr (CG == 2) mbar_arrive_leader(&tempty[acc]);
          else mbar_arrive(&tempty[acc]);
        }
      };
      // Whether the block's values are there.  Lanes see a barrier's phase end each for itself, early (`ready`) or in the wait; what reads
      // tensor memory is one instruction of the whole warp, so all lanes meet here and go one way.
      auto complete = [&](bool early) { return __all_sync(0xffffffffu, early || mbar_wait(&tfull[acc], acc_phase, abort_flag, 30)) != 0; };
      // Warps of which nothing is stored leave their values where they are.
#pragma unroll 1
      for (int kb = rows == 0 ? 0 : kbs; kb < kbs; ++kb) {
        if (!(ok = complete(ready))) break;
        ready = false;
        if constexpr (BVEC) {
          cp_wait<AHEAD - 1>();
          __syncwarp();
        }
        ask(AHEAD - 1);
        release();
        if (++acc == NACC) { acc = 0; acc_phase ^= 1; }
      }
#pragma unroll 1
      for (int kb = rows == 0 ? kbs : 0; kb < kbs; ++kb) {
        if (!(ok = complete(ready))) break;
        tc_fence_after();
        const uint32_t taddr = tmem_part + acc * ACC_STEP;
        const bool wrap = acc + 1 == NACC;
        if constexpr (BVEC) {
          uint32_t r[2][16];
          tmem_ld_16x32(taddr, r[0]);
          cp_wait<AHEAD - 1>();
          __syncwarp();
          const float* s = slots + (slot >= AHEAD ? slot - AHEAD : slot + SLOTS - AHEAD) * R::SLOT;
          ask(0);
          float a[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) a[k] = s[HALF + 8 * k + (lane >> 2)];
          tmem_ld_wait();
          constexpr int CHUNKS = HALF / 16;
          float2 f[2][4];
          auto columns = [&](int g) {
#pragma unroll
            for (int j = 0; j < 4; ++j) f[g & 1][j] = *reinterpret_cast<const float2*>(s + g * 32 + 8 * j + 2 * (lane & 3));
          };
          columns(0);
#pragma unroll
          for (int q = 0; q < CHUNKS; ++q) {             // 32 columns of lanes 0 to 15, of lanes 16 to 31
            if (q + 1 < CHUNKS) tmem_ld_16x32(taddr + (q + 1) / 2 * 32 + (((q + 1) & 1) << 20), r[(q + 1) & 1]);
            if (q + 1 == CHUNKS) ready = mbar_test(&tfull[wrap ? 0 : acc + 1], acc_phase ^ wrap);
            if (q % 2 == 1 && q + 1 < CHUNKS) columns(q / 2 + 1);
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
              for (int e = 0; e < 2; ++e) mul_add2(&sum[q * 16 + 4 * j + 2 * e], &r[q & 1][4 * j + 2 * e], f[q / 2 & 1][j], a[2 * (q & 1) + e]);
            if (q + 1 < CHUNKS) tmem_ld_wait();
            if (q + 2 == CHUNKS) release();
          }
        } else {
          float s[SEG];
#pragma unroll
          for (int g = 0; g < SEG; ++g) s[g] = a_next[0] * b_next[g][0];
          auto scales = [&] {
#pragma unroll
            for (int i = 0; i + 1 < AHEAD; ++i) {
              a_next[i] = a_next[i + 1];
#pragma unroll
              for (int g = 0; g < SEG; ++g) b_next[g][i] = b_next[g][i + 1];
            }
            ask(AHEAD - 1);
          };
          if constexpr (HALF == 64) {                    // there are registers for all of them at once
            uint32_t r[2][32];
            tmem_ld_32x32(taddr, r[0]);
            tmem_ld_32x32(taddr + 32, r[1]);
            scales();
            tmem_ld_wait();
            release();
            ready = mbar_test(&tfull[wrap ? 0 : acc + 1], acc_phase ^ wrap);
#pragma unroll
            for (int i = 0; i < HALF; ++i) sum[i] = fmaf(__uint_as_float(r[i / 32][i % 32]), s[0], sum[i]);
          } else {
            constexpr int CH = 16;
            uint32_t r[2][CH];
            tmem_ld_row16(taddr, r[0]);
            scales();
            tmem_ld_wait();
#pragma unroll
            for (int c = 0; c < HALF; c += CH) {
              if (c + CH < HALF) tmem_ld_row16(taddr + c + CH, r[(c / CH + 1) & 1]);
              else ready = mbar_test(&tfull[wrap ? 0 : acc + 1], acc_phase ^ wrap);
#pragma unroll
              for (int i = 0; i < CH; ++i) sum[c + i] = fmaf(__uint_as_float(r[c / CH & 1][i]), s[c / SEG_COLS % SEG], sum[c + i]);
              if (c + CH < HALF) tmem_ld_wait();
              if (c + 2 * CH == HALF) release();
            }
          }
        }
        if (wrap) { acc = 0; acc_phase ^= 1; }
        else ++acc;
      }
      // SPLIT: the parts go where the stages were, once both halves' products have read them (a CTA has one tile)
      if constexpr (SPLIT) asm volatile("bar.sync 1, %0;" ::"n"(32 * EPI_WARPS) : "memory");
      if (!ok) break;
      __syncwarp();                                      // (all lanes have read the last slot)
      const Patch w = patch();
      tile = begin(tile + step);
      if constexpr (SPLIT) {
#pragma unroll
        for (int i = 0; i < HALF; i += BVEC ? 2 : 4) {
          const int c = BVEC ? i / 32 * 32 + i % 16 / 4 * 8 + 2 * (lane & 3) : i;       // of the half
          const int r = quad * 32 + (BVEC ? i / 16 % 2 * 16 + i / 2 % 2 * 8 + (lane >> 2) : lane), col = part * HALF + c;
          if (r - quad * 32 >= w.rows) continue;
          uint8_t* to = smem + part_offset(r, col / 4) + col % 4 * 4;
          if constexpr (BVEC) *reinterpret_cast<float2*>(to) = make_float2(sum[i], sum[i + 1]);
          else *reinterpret_cast<float4*>(to) = make_float4(sum[i], sum[i + 1], sum[i + 2], sum[i + 3]);
        }
      } else if (w.cols > 0) {
        const float* bias = p.bias == nullptr ? nullptr : p.bias + col0;
        // a patch whose last rows are not its own, but another group's, is stored row by row
        const CUtensorMap* map = p.vec && (rows == 32 || p.mode != 1) ? &tmD : nullptr;
        const int z = p.mode == 2 ? g : 0;
        if (!add) {
          if (lane == 0) bulk_wait_read<0>();
          __syncwarp();
        }
        if (p.d_fp32) store_tile<true, !BVEC, CG>(p, sum, w, bias, buf, map, col0, row, z, add, lane);
        else store_tile<false, !BVEC, CG>(p, sum, w, bias, buf, map, col0, row, z, add, lane);
      }
    }
    cp_wait_all();                                       // no copy outlives the block
    if (lane == 0) bulk_wait_all();
    if constexpr (SPLIT) {
      __syncwarp();
      cluster_sync_all();                                // the ranges' parts lie there
      W again;
      again.at(p, first, t);
      // this CTA's share of the columns: pieces of four, the ranges' parts added in their order
      const int share = 32 / ranges, rows = min(BM, t.left);
      for (int i = threadIdx.x - 32 * EPI_FIRST; i < rows * share; i += 32 * EPI_WARPS) {
        const int r = i / share, piece = range * share + i % share, col = t.tn * BN + 4 * piece;
        if (col >= p.N) continue;
        const uint32_t at = smem_u32(smem) + part_offset(r, piece);
        float4 u[4];
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (k < static_cast<int>(ranges)) u[k] = ld_cluster(at, k);
        float4 v = u[0];
#pragma unroll
        for (int k = 1; k < 4; ++k)
          if (k < static_cast<int>(ranges)) { v.x += u[k].x; v.y += u[k].y; v.z += u[k].z; v.w += u[k].w; }
        float f[4] = {v.x * p.alpha, v.y * p.alpha, v.z * p.alpha, v.w * p.alpha};
        const long row = t.row0 + r;
        float* d32 = static_cast<float*>(p.D) + row * p.ldd + col;
        __nv_bfloat16* d16 = static_cast<__nv_bfloat16*>(p.D) + row * p.ldd + col;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (col + j >= p.N) break;
          if (p.bias != nullptr) f[j] += p.bias[col + j];
          if (p.beta != 0.f)
            f[j] += p.beta * (p.d_fp32 ? static_cast<const float*>(p.C)[row * p.ldc + col + j]
                                       : __bfloat162float(static_cast<const __nv_bfloat16*>(p.C)[row * p.ldc + col + j]));
        }
        if (p.vec) {                                     // (N is a multiple of four then)
          if (p.d_fp32) {
            *reinterpret_cast<float4*>(d32) = make_float4(f[0], f[1], f[2], f[3]);
          } else {
            const __nv_bfloat162 lo = __floats2bfloat162_rn(f[0], f[1]), hi = __floats2bfloat162_rn(f[2], f[3]);
            *reinterpret_cast<uint2*>(d16) = make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
          }
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (col + j >= p.N) break;
            if (p.d_fp32) d32[j] = f[j];
            else d16[j] = __float2bfloat16_rn(f[j]);
          }
        }
      }
      __syncwarp();
      cluster_sync_all();                                // nobody leaves while its part is read
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

// Map of `depth` stacked row-major matrices (rows x inner elements of es bytes, 1: e4m3), strides in bytes, boxes of box_rows x 128
// bytes.
int make_map(CUtensorMap* out, const void* base, int rank, int es, uint64_t inner, uint64_t rows, uint64_t depth, uint64_t ld, uint64_t stack,
             uint32_t box_rows) {
  EncodeTiledFn enc = encode_fn();
  if (enc == nullptr) return -100;
  const cuuint64_t dims[3] = {inner, rows, depth}, strides[2] = {ld, stack};
  const cuuint32_t box[3] = {128u / es, box_rows, 1}, steps[3] = {1, 1, 1};
  const CUtensorMapDataType type = es == 1 ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                           : es == 2 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32;
  const CUresult r = enc(out, type, rank, const_cast<void*>(base), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
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

// Ranges of the reduction for tiles of 128 x 128: a power of two up to four, as there are SMs for, each of two blocks at least and
// none empty.  (Clusters of eight start later: 1 x 2048 x 2048 15.3 to 17.2 us, 14.3 with four.)
int split_ranges(int64_t tiles, int k_blocks, int sms) {
  int ranges = 4;
  while (ranges > 1 && (tiles * ranges > sms || k_blocks < 2 * ranges || (ranges - 1) * ((k_blocks + ranges - 1) / ranges) >= k_blocks)) ranges /= 2;
  return ranges;
}

// The tile of a product: 1 128 x 128 (cut along the reduction where that fills the GPU), 2 128 x 256, 3 256 x 256 on two SMs.  By
// the waves and the blocks of each: a block takes some 0.5, 0.7 and 0.66 us, with column scales 0.51, 0.86 and 0.84, joined ranges 2 us
// and a pair's start 1.5 (a pair loads less for the same work, and is bound by power later).  us on the device with 1 / 2 / 3, back to back
// in a graph, x W^T:
//   16 x 4096 x 4096    8.2 / 20 / 21     256 x 4096 x 4096    15 / 23 / 23     200 x 14336 x 4096   32 / 24 / 24
//   768 x 4096 x 4096    32 / 23 / 23     1024 x 2048 x 2048   12 / 15 / 15     512 x 4096 x 14336   52 / 66 / 63
//   column scales: 768 x 4096 x 4096   37 / 31 / 33     1536 x 4096 x 4096   52 / 59 / 60
int pick_variant(int64_t M, int64_t N, int k_blocks, int sms, bool columns) {
  auto up = [](int64_t a, int64_t b) { return (a + b - 1) / b; };
  const int64_t t1 = up(M, 128) * up(N, 128), t2 = up(M, 128) * up(N, 256), t3 = up(M, 256) * up(N, 256);
  const int r = split_ranges(t1, k_blocks, sms);
  const double c1 = up(t1 * r, sms) * up(k_blocks, r) * (columns ? 0.51 : 0.5) + (r > 1 ? 2.0 : 0.0),
               c2 = up(t2, sms) * k_blocks * (columns ? 0.86 : 0.7),
               c3 = up(t3, sms / 2 > 0 ? sms / 2 : 1) * k_blocks * (columns ? 0.84 : 0.66) + 1.5;
  return c3 <= c1 && c3 <= c2 ? 3 : c2 <= c1 ? 2 : 1;
}

template <int CG, int BN, bool BVEC, bool SPLIT = false>
int launch(const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& td, const Params& p, int dev, int most, cudaStream_t stream, int ranges = 1) {
  using R = Ring<CG, BN, BVEC>;
  auto kern = gemm_fp8_kernel<CG, BN, BVEC, SPLIT>;
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
  cfg.gridDim = dim3(static_cast<unsigned>(SPLIT ? want * ranges : want < sms ? want : sms));
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = R::TOTAL;
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = SPLIT ? ranges : CG;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, ta, tb, td, p) == cudaSuccess && cudaGetLastError() == cudaSuccess ? 0 : -400;
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
  constexpr int64_t MOST = 0x7FFFFC00ll;          // rows, columns and depth, a tile behind the last one included, in 31 bits
  if (a->M > MOST || a->N > MOST || a->K > MOST) return -3;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= MAX_DEVICES) return -4;
  Params p;
  p.M = static_cast<int>(a->M); p.N = static_cast<int>(a->N); p.K = static_cast<int>(a->K);
  p.D = a->D; p.C = a->C != nullptr ? a->C : a->D; p.bias = a->bias;
  p.ldd = a->ldd; p.ldc = a->C != nullptr ? a->ldc : a->ldd;
  p.alpha = static_cast<float>(a->alpha); p.beta = static_cast<float>(a->beta);
  p.d_fp32 = static_cast<int>(a->d_fp32);
  const int64_t es = p.d_fp32 ? 4 : 2;
  if (p.M == 1 && a->mode != 2) p.ldd = p.ldc = (p.N * es + 15) / 16 * 16 / es;      // (a single row has no stride of its own)
  p.vec = ((reinterpret_cast<uintptr_t>(p.D) | reinterpret_cast<uintptr_t>(p.C) | static_cast<uintptr_t>(p.N * es) |
            static_cast<uintptr_t>(p.ldd * es) | static_cast<uintptr_t>(p.ldc * es) | static_cast<uintptr_t>(a->mode == 2 ? a->d_g * es : 0)) & 15) == 0;
  p.sa = a->sa; p.sa_m = a->sa_m; p.sa_k = a->sa_k; p.sa_shift = static_cast<int>(a->sa_shift);
  p.sb = a->sb; p.sb_n = a->sb_n; p.sb_k = a->sb_k; p.sb_g = a->sb_g;
  p.a_mn = a->a_mn != 0; p.b_mn = a->b_mn != 0;
  p.mode = static_cast<int>(a->mode); p.groups = static_cast<int>(a->groups); p.offsets = a->offsets; p.d_g = a->d_g;
  p.total = p.mode == 1 ? p.M : p.K;
  p.k_blocks = (p.K + BK - 1) / BK;

  const int sms = sm_count(dev), most = a->max_ctas > 0 && a->max_ctas < sms ? static_cast<int>(a->max_ctas) : sms;
  const int variant = a->variant ? static_cast<int>(a->variant)
                      : p.mode == 0 ? pick_variant(p.M, p.N, p.k_blocks, most, a->sb_shift == 0)
                      : p.N <= 128  ? 1
                      : p.mode == 1 ? 2
                      : p.M > 128   ? 3
                                    : 2;
  const int cg = variant == 3 ? 2 : 1, bn = variant == 1 ? 128 : 256;
  const int tile_m = BM * cg;
  p.tiles_m = (p.M + tile_m - 1) / tile_m;
  p.tiles_n = (p.N + bn - 1) / bn;
  const int64_t tiles = (p.mode == 2 ? static_cast<int64_t>(p.groups) * p.tiles_m
                                     : p.tiles_m + (p.mode == 1 ? p.groups : 0)) * static_cast<int64_t>(p.tiles_n);
  if (tiles >= 1ll << 30) return -3;
  p.num_tiles = static_cast<int>(tiles);

  p.add_in_place = p.d_fp32 && p.beta == 1.f && p.C == p.D && p.ldc == p.ldd;

  CUtensorMap ta, tb, td;
  const uint64_t z = p.mode == 1 ? p.groups : 1;
  // Few rows are copied as they are, without zeros behind them: a copy takes its time by rows, and the products of what the stage held
  // there are rows of their own, which nothing reads (1 x 14336 x 4096 24.5 -> 18.5 us).
  const int a_rows = !p.a_mn && p.M < BM ? (p.M + 7) / 8 * 8 : BM;
  p.stage_bytes = a_rows * BK + bn / cg * BK;
  int rc = p.a_mn ? make_map(&ta, a->A, 2, 1, p.M, p.K, 1, a->lda, 0, 128) : make_map(&ta, a->A, 2, 1, p.K, p.M, 1, a->lda, 0, a_rows);
  if (rc) return rc;
  // (a stack of one has no stride of its own)
  const uint64_t stack = z > 1 ? a->b_g : (p.b_mn ? p.K : p.N) * static_cast<uint64_t>(a->ldb);
  rc = p.b_mn ? make_map(&tb, a->B, 3, 1, p.N, p.K, z, a->ldb, stack, 128) : make_map(&tb, a->B, 3, 1, p.K, p.N, z, a->ldb, stack, bn / cg);
  if (rc) return rc;
  const bool bvec = a->sb_shift == 0;
  if (variant == 1 && p.mode == 0) {
    const int ranges = split_ranges(tiles, p.k_blocks, most);
    p.split_blocks = (p.k_blocks + ranges - 1) / ranges;
    if (ranges > 1)
      return bvec ? launch<1, 128, true, true>(ta, tb, ta, p, dev, most, a->stream, ranges)
                  : launch<1, 128, false, true>(ta, tb, ta, p, dev, most, a->stream, ranges);
  }
  if (p.vec) {
    const uint64_t depth = p.mode == 2 ? p.groups : 1;
    rc = make_map(&td, p.D, 3, static_cast<int>(es), p.N, p.M, depth, p.ldd * es, depth > 1 ? p.d_g * es : p.M * static_cast<uint64_t>(p.ldd * es), 32);
    if (rc) return rc;
  } else {
    td = ta;                            // (not used)
  }
  if (variant == 1) return bvec ? launch<1, 128, true>(ta, tb, td, p, dev, most, a->stream) : launch<1, 128, false>(ta, tb, td, p, dev, most, a->stream);
  if (variant == 2) return bvec ? launch<1, 256, true>(ta, tb, td, p, dev, most, a->stream) : launch<1, 256, false>(ta, tb, td, p, dev, most, a->stream);
  return bvec ? launch<2, 256, true>(ta, tb, td, p, dev, most, a->stream) : launch<2, 256, false>(ta, tb, td, p, dev, most, a->stream);
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
