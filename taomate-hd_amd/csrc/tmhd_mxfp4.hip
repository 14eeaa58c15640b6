// MXFP4 projections for gfx950: row quantization to e2m1 codes with a
// power-of-two scale for each 32 values, its inverse, and the product of two
// such matrices on the block-scaled MFMA (formats: include/tmhd_lowbit.h).
#include <type_traits>

#include <algorithm>

#include "tmhd_gemm.h"
#include "tmhd_internal.h"
#include "tmhd_lowbit.h"

namespace tmhd {
namespace {

using i32x8 = int __attribute__((ext_vector_type(8)));
using u16x2 = unsigned short __attribute__((ext_vector_type(2)));

constexpr int kSuper = 512;  // columns that a scale word spans

// Scale word of (512-column block s, column group g, row): R4 rows, a multiple of 4.
__device__ __forceinline__ int64_t scale_word(int s, int g, int row, int32_t r4) {
  return ((int64_t)s * 4 + g) * r4 + row;
}

// ---------------------------------------------------------------------------
// Row quantization: bound by HBM.  A wave takes one 512-column block of RQ
// consecutive rows: per row a 16-byte load of 8 values per lane (1 KiB in all),
// four lanes to a block of 32.  The maximum is taken on the magnitudes' bits
// (packed 16-bit integers), so a block's exponent is that maximum's exponent
// field and an infinity or NaN shows as a maximum of 0x7f80 and more.  The
// conversion instruction divides by the scale, rounds to nearest even and
// saturates.
constexpr int RQ = 4;

// max of the magnitudes of 8 bf16, in both halves of the result
__device__ __forceinline__ uint32_t amax8(const i32x4 &v) {
  u16x2 m = {0, 0};
#pragma unroll
  for (int e = 0; e < 4; ++e)
    m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, (uint32_t)v[e] & 0x7fff7fffu));
  return max((uint32_t)m[0], (uint32_t)m[1]);
}

// scale byte of a block whose largest magnitude has the bf16 bits amax
__device__ __forceinline__ uint32_t scale_byte(uint32_t amax) {
  const uint32_t e = amax >> 7;  // exponent field
  return e == 255u ? 255u : (uint32_t)max((int)e - 2, 2);
}

// 8 bf16 -> 8 codes; a block without finite values (byte 255) gives codes 0
__device__ __forceinline__ uint32_t codes8(const i32x4 &v, uint32_t byte) {
  const float scale = __uint_as_float(byte << 23);
  uint32_t c = 0;
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2, (uint32_t)v[0]), scale, 0);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2, (uint32_t)v[1]), scale, 1);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2, (uint32_t)v[2]), scale, 2);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2, (uint32_t)v[3]), scale, 3);
  return byte == 255u ? 0u : c;
}

__global__ void __launch_bounds__(256) mxfp4_quant_kernel(uint8_t *__restrict__ q, uint32_t *__restrict__ scale,
                                                          const uint16_t *__restrict__ x, int32_t rows, int32_t r4,
                                                          int32_t cols, int64_t xs, int32_t blocks) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int s = blockIdx.x % blocks, row0 = (blockIdx.x / blocks * 4 + w) * RQ;
  if (row0 >= r4) return;
  const int col = s * kSuper + lane * 8;
  const bool live = col < cols;
  i32x4 v[RQ];
#pragma unroll
  for (int i = 0; i < RQ; ++i)
    v[i] = live && row0 + i < rows ? *(const i32x4 *)(x + (int64_t)(row0 + i) * xs + col) : i32x4{0, 0, 0, 0};
  uint32_t word = 0;
#pragma unroll
  for (int i = 0; i < RQ; ++i) {
    uint32_t m = amax8(v[i]);
    m = max(m, (uint32_t)__shfl_xor((int)m, 1));
    m = max(m, (uint32_t)__shfl_xor((int)m, 2));
    const bool there = live && row0 + i < rows;
    uint32_t byte = scale_byte(m);
    if (there) *(uint32_t *)(q + (int64_t)(row0 + i) * (cols >> 1) + (col >> 1)) = codes8(v[i], byte);
    byte = there ? byte : 0u;
    // block 4 b + g of the 512 columns sits in lanes 16 b + 4 g ..: word g of
    // the row gathers lanes 4 g + 16 b
    uint32_t gathered = byte | (uint32_t)__shfl_xor((int)byte, 16) << 8;
    gathered |= (uint32_t)__shfl_xor((int)gathered, 32) << 16;
    if ((lane & 3) == i) word = gathered;  // lanes 4 g + i of the first 16 keep row i's word g
  }
  if (lane < 16) scale[scale_word(s, lane >> 2, row0 + (lane & 3), r4)] = word;
}

// The inverse: a lane reads 8 codes and their scale byte, writes 16 bytes.
__global__ void __launch_bounds__(256) mxfp4_dequant_kernel(uint16_t *__restrict__ x, const uint8_t *__restrict__ q,
                                                            const uint32_t *__restrict__ scale, int32_t rows,
                                                            int32_t r4, int32_t cols, int32_t blocks) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int s = blockIdx.x % blocks, row0 = (blockIdx.x / blocks * 4 + w) * RQ;
  const int col = s * kSuper + lane * 8;
  if (col >= cols) return;
  uint32_t c[RQ], sw[RQ];
#pragma unroll
  for (int i = 0; i < RQ; ++i) {
    const int row = min(row0 + i, rows - 1);
    c[i] = *(const uint32_t *)(q + (int64_t)row * (cols >> 1) + (col >> 1));
    sw[i] = scale[scale_word(s, (lane >> 2) & 3, row, r4)];
  }
#pragma unroll
  for (int i = 0; i < RQ; ++i) {
    if (row0 + i >= rows) break;
    const uint32_t byte = (sw[i] >> (8 * (lane >> 4))) & 255u;
    const float f = __uint_as_float(byte << 23);
    i32x4 o;
    o[0] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c[i], f, 0));
    o[1] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c[i], f, 1));
    o[2] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c[i], f, 2));
    o[3] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c[i], f, 3));
    if (byte == 255u) o = i32x4{0x7fc07fc0, 0x7fc07fc0, 0x7fc07fc0, 0x7fc07fc0};
    *(i32x4 *)(x + (int64_t)(row0 + i) * cols + col) = o;
  }
}

// ---------------------------------------------------------------------------
// Products.  D[n][m] = B rows x A rows on v_mfma_scale_f32_16x16x128_f8f6f4: a
// lane (i, g) = (lane % 16, lane / 16) holds the 16 bytes of columns 32 g .. of
// row i for each 128 columns, so a 32-column block and its scale belong to one
// lane, and word g of a row's scales serves four MFMAs (byte b for columns 128 b
// .. of 512).  It gets four consecutive n of one m.
struct XArgs {
  const uint8_t *a;
  const uint8_t *b;
  const uint32_t *as;
  const uint32_t *bs;
  uint16_t *out;
  const uint16_t *bias;
  int32_t m, n, k;
  int32_t am4, bn4;  // rows of the scale arrays
  int64_t lda, ldb, ldo;
  int32_t st_ok;     // 8-byte stores of 4 columns
  int32_t st16_ok;   // 16-byte stores of 8
  int32_t full;      // tiles of the big kernel
};

template <int B>
__device__ __forceinline__ f32x4 mfma_fp4(const i32x4 &b, const i32x4 &a, const f32x4 &c, int sb, int sa) {
  const i32x8 bb = {b[0], b[1], b[2], b[3]}, aa = {a[0], a[1], a[2], a[3]};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(bb, aa, c, 4, 4, B, sb, B, sa);
}

// The same with the accumulators pinned to AGPRs (IN_AGPR) or VGPRs: left to the
// builtin, the compiler moves the tiles' accumulators between the two around
// their MFMAs.  FIRST: c = b a.  mfma_settle() goes before other code reads them.
template <int B, bool IN_AGPR, bool FIRST = false>
__device__ __forceinline__ void mfma_fp4_into(f32x4 &c, const i32x4 &b, const i32x4 &a, int sb, int sa) {
#define TMHD_MFMA(reg, sel)                                                                                      \
  if constexpr (FIRST)                                                                                           \
    asm("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, 0, %3, %4 " sel " cbsz:4 blgp:4"                          \
        : "=&" reg(c) : "v"(b), "v"(a), "v"(sb), "v"(sa));                                                        \
  else                                                                                                           \
    asm("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 " sel " cbsz:4 blgp:4"                         \
        : "+" reg(c) : "v"(b), "v"(a), "v"(sb), "v"(sa))
#define TMHD_MFMA_BYTE(reg)                                       \
  if constexpr (B == 0) {                                         \
    TMHD_MFMA(reg, "op_sel:[0,0,0] op_sel_hi:[0,0,0]");           \
  } else if constexpr (B == 1) {                                  \
    TMHD_MFMA(reg, "op_sel:[1,1,0] op_sel_hi:[0,0,0]");           \
  } else if constexpr (B == 2) {                                  \
    TMHD_MFMA(reg, "op_sel:[0,0,0] op_sel_hi:[1,1,0]");           \
  } else {                                                        \
    TMHD_MFMA(reg, "op_sel:[1,1,0] op_sel_hi:[1,1,0]");           \
  }
  if constexpr (IN_AGPR) {
    TMHD_MFMA_BYTE("a")
  } else {
    TMHD_MFMA_BYTE("v")
  }
#undef TMHD_MFMA_BYTE
#undef TMHD_MFMA
}

// The wait states between the last MFMAs and code that reads their results.
template <bool IN_AGPR, int NB, int MB>
__device__ __forceinline__ void mfma_settle(f32x4 (&acc)[NB][MB]) {
  asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");
#pragma unroll
  for (int i = 0; i < NB; ++i)
#pragma unroll
    for (int j = 0; j < MB; ++j) {
      if constexpr (IN_AGPR)
        asm volatile("" : "+a"(acc[i][j]));
      else
        asm volatile("" : "+v"(acc[i][j]));
    }
}

// Four columns n .. n + 3 of row m, bias added, rounded once.
__device__ __forceinline__ void store_quad(const XArgs &xa, const f32x4 &v, int m, int n) {
  if (m >= xa.m || n >= xa.n) return;
  float t[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) t[e] = v[e] + (xa.bias ? bf16_bits_to_f32(xa.bias[min(n + e, xa.n - 1)]) : 0.0f);
  const i32x2 o = {(int)pack_bf16_rne(t[0], t[1]), (int)pack_bf16_rne(t[2], t[3])};
  uint16_t *op = xa.out + (int64_t)m * xa.ldo + n;
  if (xa.st_ok && n + 3 < xa.n)
    *(i32x2 *)op = o;
  else
    for (int e = 0; e < 4 && n + e < xa.n; ++e) op[e] = (uint16_t)((uint32_t)o[e >> 1] >> (16 * (e & 1)));
}

// 32 bf16 (a lane's block) -> 16 bytes of codes; returns the scale byte
__device__ __forceinline__ uint32_t quant32(const i32x4 (&x)[4], i32x4 &codes) {
  const uint32_t byte = scale_byte(max(max(amax8(x[0]), amax8(x[1])), max(amax8(x[2]), amax8(x[3]))));
#pragma unroll
  for (int i = 0; i < 4; ++i) codes[i] = (int)codes8(x[i], byte);
  return byte;
}

// Few rows: 16 columns of n and 16 MB rows of m a workgroup, its W waves take
// the 512-column blocks of k in turn, straight from global memory to the MFMA
// (each code is used once or by MB MFMAs), and add their sums through LDS in
// wave order.  QUANT: the rows are bf16 (xa.a, lda in elements); a lane's
// operand is a whole 32-column block, so it finds the block's scale and codes
// by itself.
template <int MB, int W, bool QUANT>
__global__ void __launch_bounds__(64 * W) mxfp4_rows_kernel(const XArgs xa) {
  __shared__ f32x4 part[W][MB][64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, li = lane & 15, lg = lane >> 4;
  const int n0 = blockIdx.x * 16, m0 = blockIdx.y * 16 * MB;
  const int chunks = xa.k >> 5, blocks = (xa.k + kSuper - 1) / kSuper;
  const int brow = min(n0 + li, xa.n - 1);
  const uint8_t *bp = xa.b + (int64_t)brow * xa.ldb + lg * 16;
  const uint8_t *ap[MB];
  int arow[MB];
#pragma unroll
  for (int j = 0; j < MB; ++j) {
    arow[j] = min(m0 + j * 16 + li, xa.m - 1);
    ap[j] = xa.a + (int64_t)arow[j] * xa.lda * (QUANT ? 2 : 1) + lg * (QUANT ? 64 : 16);
  }
  f32x4 acc[MB];
#pragma unroll
  for (int j = 0; j < MB; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int s = w; s < blocks; s += W) {
    // chunk 16 s + 4 t + lg; behind the last column: zero codes (their scale bytes are zero too)
    const int64_t at = (int64_t)s * (kSuper / 2);
    i32x4 bv[4], av[MB][4];
    int sa[MB];
    const int sb = (int)xa.bs[scale_word(s, lg, brow, xa.bn4)];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const bool in = 16 * s + 4 * t + lg < chunks;
      bv[t] = in ? *(const i32x4 *)(bp + at + 64 * t) : i32x4{0, 0, 0, 0};
    }
    if constexpr (QUANT) {
#pragma unroll
      for (int j = 0; j < MB; ++j) {
        sa[j] = 0;
        i32x4 x[4][4];
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            x[t][e] = 16 * s + 4 * t + lg < chunks ? *(const i32x4 *)(ap[j] + 4 * (at + 64 * t) + 16 * e) : i32x4{0, 0, 0, 0};
#pragma unroll
        for (int t = 0; t < 4; ++t) sa[j] |= (int)(quant32(x[t], av[j][t]) << (8 * t));
      }
    } else {
#pragma unroll
      for (int j = 0; j < MB; ++j) {
#pragma unroll
        for (int t = 0; t < 4; ++t)
          av[j][t] = 16 * s + 4 * t + lg < chunks ? *(const i32x4 *)(ap[j] + at + 64 * t) : i32x4{0, 0, 0, 0};
        sa[j] = (int)xa.as[scale_word(s, lg, arow[j], xa.am4)];
      }
    }
#pragma unroll
    for (int j = 0; j < MB; ++j) {
      acc[j] = mfma_fp4<0>(bv[0], av[j][0], acc[j], sb, sa[j]);
      acc[j] = mfma_fp4<1>(bv[1], av[j][1], acc[j], sb, sa[j]);
      acc[j] = mfma_fp4<2>(bv[2], av[j][2], acc[j], sb, sa[j]);
      acc[j] = mfma_fp4<3>(bv[3], av[j][3], acc[j], sb, sa[j]);
    }
  }
#pragma unroll
  for (int j = 0; j < MB; ++j) part[w][j][lane] = acc[j];
  __syncthreads();
  for (int j = w; j < MB; j += W) {
    f32x4 sum = part[0][j][lane];
#pragma unroll
    for (int i = 1; i < W; ++i) sum += part[i][j][lane];
    store_quad(xa, sum, m0 + j * 16 + li, n0 + 4 * lg);
  }
}

// ---------------------------------------------------------------------------
// Tiles of 2 MH rows x 2 NH columns, 4 waves as 2 x 2 of MH x NH (blocks of
// 16 x 16).  k moves in blocks of 128 bytes (256 columns, two MFMA steps), NBUF
// blocks deep in LDS: rows of 128 bytes (whole cache lines) with chunk c of row
// r at c ^ ((r >> 1) & 7), which keeps the 16-byte operand reads free of bank
// conflicts, and each row's scale words for the block's 512 columns, entry g of
// row r at (r + 16 g) mod rows.  Block d: step 0 multiplies operands that are
// in registers and reads step 1's; behind the wait for block d + 1 and the
// barrier nobody reads block d any more, so step 1 loads block d + NBUF in its
// place and reads block d + 1's first operands and scale words.
// Columns past k: the loads repeat the row's last chunk, and its scale bytes
// there are zero, 2^-127 on both sides: the products underflow to 0.
constexpr int KB = 128;  // bytes of a row in a block

// hload_lds16 with the wait states that a vector-memory instruction needs after
// the vector instruction that wrote its scalar base (five: v_readlane of a
// spilled register, v_readfirstlane) and after the write of m0 (one).  The
// compiler keeps those for its own instructions, not for inline asm, and the
// product kernels hold enough scalars for it to spill some to vector lanes.  The
// copy of the base is a scalar instruction: it waits for the vector write by
// itself, and a scalar write needs no wait states before the load.
__device__ __forceinline__ void load_lds16_any(const void *base, uint32_t off, uint32_t lds_addr) {
  const void *copy;
  asm volatile("s_mov_b64 %0, %2\n\tglobal_load_lds_dwordx4 %1, %0" : "=&s"(copy) : "v"(off), "s"(base), "{m0}"(lds_addr) : "memory");
}

// A wave's sums, rounded to bf16 and stored from registers: rows m0 .., columns n0 ...  A
// pair of 16-column blocks trades halves between neighbouring lane groups, so that a
// lane holds 8 consecutive columns of one block (16 bytes).
template <int NB, int MB>
__device__ __forceinline__ void store_tile(const XArgs &xa, const f32x4 (&acc)[NB][MB], int m0, int n0, int li, int lg) {
#pragma unroll
  for (int i = 0; i < NB; i += 2) {
    const int n = n0 + i * 16 + 4 * lg;  // of the lane's own columns, in block i
    float bf[2][4];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int e = 0; e < 4; ++e) bf[h][e] = xa.bias ? bf16_bits_to_f32(xa.bias[min(n + 16 * h + e, xa.n - 1)]) : 0.0f;
    const int nn = n0 + (i + (lg & 1)) * 16 + 8 * (lg >> 1);  // of what it stores
#pragma unroll
    for (int j = 0; j < MB; ++j) {
      uint32_t p[2][2];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          p[h][e] = pack_bf16_rne(acc[i + h][j][2 * e] + bf[h][2 * e], acc[i + h][j][2 * e + 1] + bf[h][2 * e + 1]);
      const auto lo = __builtin_amdgcn_permlane16_swap(p[0][0], p[1][0], false, false);
      const auto hi = __builtin_amdgcn_permlane16_swap(p[0][1], p[1][1], false, false);
      const i32x4 v = {(int)lo[0], (int)hi[0], (int)lo[1], (int)hi[1]};
      const int m = m0 + j * 16 + li;
      if (m < xa.m && nn < xa.n) {
        uint16_t *op = xa.out + (int64_t)m * xa.ldo + nn;
        if (xa.st16_ok && nn + 7 < xa.n)
          *(i32x4 *)op = v;
        else
          for (int e = 0; e < 8 && nn + e < xa.n; ++e) op[e] = (uint16_t)((uint32_t)v[e >> 1] >> (16 * (e & 1)));
      }
    }
  }
}

// The k loop of one tile: DATA / SCALE bytes of a buffer, a wave's loads and the
// operands of its MFMAs.
template <int MH, int NH, int NBUF>
struct TileLoop {
  static constexpr int BM = 2 * MH, BN = 2 * NH, MB = MH / 16, NB = NH / 16, NR = MB + NB, NM = MB * NB;
  static constexpr int DATA = (BM + BN) * KB, SCALE = (BM + BN) * 16, BUF = DATA + SCALE;
  static constexpr int AL = BM / 32, DL = (BM + BN) / 32;  // 1 KiB data loads of a wave: of A, in all
  static constexpr int SN = (BM + BN) / 64;                // 1 KiB scale loads of the workgroup
  static constexpr int SL = (SN + 3) / 4;                  // of a wave (where 4 does not divide them, waves repeat some)
  static constexpr int LPB = DL + SL;
  static constexpr bool AG = NM > 32;
  static_assert(NBUF >= 2 && NBUF * BUF <= 160 * 1024 && (NBUF - 1) * LPB < 64, "buffers fit the LDS and vmcnt");

  const XArgs &xa;
  char *smem;
  uint32_t lds0;
  int w, wm, wn, lane, li, lg, lch, chunks, nd;
  uint32_t doff[DL], soff[SL], sdst[SL], rdq[2], rds[NR];
  f32x4 acc[NB][MB];  // D[n][m]: lane (j, g4) holds n = 16 nb + 4 g4 + (0..3), m = 16 mb + j
  i32x4 cur[NR], nxt[NR];
  int sc[NR], nsc[NR];

  __device__ __forceinline__ TileLoop(const XArgs &args, char *lds) : xa(args), smem(lds) {
    lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)lds;
    lane = threadIdx.x & 63, li = lane & 15, lg = lane >> 4;
    w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = w >> 1, wn = w & 1;
    chunks = xa.k >> 5, nd = (xa.k + 255) >> 8;
    lch = (lane & 7) ^ ((4 * (w & 1) + (lane >> 4)) & 7);
    // operand reads: row i of a 16-row block, logical chunk 4 q + lg
#pragma unroll
    for (int q = 0; q < 2; ++q) rdq[q] = (uint32_t)(li * KB + (((4 * q + lg) ^ ((li >> 1) & 7)) * 16));
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      const int rows = r < MB ? BM : BN, row = (r < MB ? wm * MH + r * 16 : wn * NH + (r - MB) * 16) + li;
      rds[r] = (uint32_t)(DATA + (r < MB ? 0 : BM * 16) + (lg * rows + (row + 16 * lg) % rows) * 4);
    }
  }
  // Where the tile's rows and scale words lie.  Data loads: 8 rows of 128 bytes
  // each; lane: row lane / 8, physical chunk lane % 8.  Scale loads: 64 lanes of 4
  // words; word q of the area is entry g = q / rows of row (q - 16 g) mod rows.
  __device__ __forceinline__ void at(int m0, int n0) {
#pragma unroll
    for (int i = 0; i < DL; ++i) {
      const int r = (w + 4 * (i < AL ? i : i - AL)) * 8 + (lane >> 3);
      doff[i] = i < AL ? (uint32_t)((int64_t)min(m0 + r, xa.m - 1) * xa.lda) : (uint32_t)((int64_t)min(n0 + r, xa.n - 1) * xa.ldb);
    }
#pragma unroll
    for (int i = 0; i < SL; ++i) {
      const int load = (w + 4 * i) % SN;  // of the workgroup's scale loads, A's first
      const bool is_a = scale_of_a(i);
      const int rows = is_a ? BM : BN, q = (is_a ? load : load - BM / 64) * 256 + lane * 4;
      const int g = q / rows, r = (q % rows - 16 * g + 4 * rows) % rows;
      const int r4 = is_a ? xa.am4 : xa.bn4;
      soff[i] = (uint32_t)(((int64_t)g * r4 + min((is_a ? m0 : n0) + r, r4 - 4)) * 4);
      sdst[i] = (uint32_t)(DATA + load * 1024);
    }
  }
  // whether scale load i of the wave is one of A's (known at compile time for 256 x 256)
  __device__ __forceinline__ bool scale_of_a(int i) const { return BM == 256 && BN == 256 ? i == 0 : (w + 4 * i) % SN < BM / 64; }
  // load n of block d (blocks past the last repeat it, into a buffer nobody reads)
  __device__ __forceinline__ void load_one(int d, uint32_t koff, int buf, int n) {
    const uint32_t to = lds0 + (uint32_t)(buf * BUF);
    if (n < DL) {
      const uint32_t dst = to + (n < AL ? (w + 4 * n) * 1024 : BM * KB + (w + 4 * (n - AL)) * 1024);
      load_lds16_any(n < AL ? xa.a : xa.b, doff[n] + koff, dst);
    } else {
      const int i = n - DL;
      const uint32_t *base = scale_of_a(i) ? xa.as + (int64_t)(d >> 1) * 4 * xa.am4 : xa.bs + (int64_t)(d >> 1) * 4 * xa.bn4;
      load_lds16_any(base, soff[i], to + sdst[i]);
    }
  }
  __device__ __forceinline__ uint32_t koff_of(int d) const { return (uint32_t)(min(8 * d + lch, chunks - 1) * 16); }
  __device__ __forceinline__ i32x4 read_op(int buf, int q, int r) const {
    const uint32_t from = (uint32_t)(buf * BUF) + rdq[q];
    return *(const i32x4 *)(smem + from + (r < MB ? (wm * MH + r * 16) * KB : (BM + wn * NH + (r - MB) * 16) * KB));
  }
  __device__ __forceinline__ int read_scale(int buf, int r) const { return *(const int *)(smem + (uint32_t)(buf * BUF) + rds[r]); }

  // the loads of the tile's first NBUF blocks
  __device__ __forceinline__ void first_loads() {
#pragma unroll
    for (int u = 0; u < NBUF; ++u) {
      const int d = min(u, nd - 1);
      const uint32_t ko = koff_of(d);
#pragma unroll
      for (int n = 0; n < LPB; ++n) load_one(d, ko, u, n);
    }
  }
  // block d in buffer `buf`; ODD: the second of its 512 columns' blocks; returns the next buffer
  template <int ODD>
  __device__ __forceinline__ int block(int d, int buf) {
    const int nbuf = buf + 1 == NBUF ? 0 : buf + 1;
#pragma unroll
    for (int idx = 0; idx < NM; ++idx) {
#pragma unroll
      for (int r = idx * NR / NM; r < (idx + 1) * NR / NM; ++r) nxt[r] = read_op(buf, 1, r);
      mfma_fp4_into<2 * ODD, AG>(acc[idx / MB][idx % MB], cur[MB + idx / MB], cur[idx % MB], sc[MB + idx / MB], sc[idx % MB]);
      __builtin_amdgcn_sched_barrier(0);
    }
    __builtin_amdgcn_s_waitcnt(vmcnt_imm((NBUF - 2) * LPB));
    __syncthreads();
    const int dl = min(d + NBUF, nd - 1);
    const uint32_t ko = koff_of(dl);
#pragma unroll
    for (int idx = 0; idx < NM; ++idx) {
#pragma unroll
      for (int r = idx * NR / NM; r < (idx + 1) * NR / NM; ++r) {
        cur[r] = read_op(nbuf, 0, r);
        nsc[r] = read_scale(nbuf, r);
      }
      // loads in the step's first half: they have until the next block's barrier
#pragma unroll
      for (int n = 2 * idx * LPB / NM; n < 2 * (idx + 1) * LPB / NM; ++n)
        if (n < LPB) load_one(dl, ko, buf, n);
      mfma_fp4_into<2 * ODD + 1, AG>(acc[idx / MB][idx % MB], nxt[MB + idx / MB], nxt[idx % MB], sc[MB + idx / MB], sc[idx % MB]);
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int r = 0; r < NR; ++r) sc[r] = nsc[r];
    // a register that vector code wrote (a copy above) may be an MFMA's operand two wait states later
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_nop 1");
    __builtin_amdgcn_sched_barrier(0);
    return nbuf;
  }
  // The sums of the tile whose first block has landed for every wave.  Leaves the
  // buffers free for every wave and no load in flight.
  __device__ __forceinline__ void run() {
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
      for (int j = 0; j < MB; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      cur[r] = read_op(0, 0, r);
      sc[r] = read_scale(0, r);
    }
    int buf = 0, d = 0;
    for (; d + 1 < nd; d += 2) {
      buf = block<0>(d, buf);
      buf = block<1>(d + 1, buf);
    }
    if (d < nd) block<0>(d, buf);
    __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
    mfma_settle<AG>(acc);
    __syncthreads();
  }
  __device__ __forceinline__ void store(int m0, int n0) {
    store_tile<NB, MB>(xa, acc, m0 + wm * MH, n0 + wn * NH, li, lg);
  }
};

// Tiles of a launch of its own (few workgroups): one tile each.
template <int MH, int NH, int NBUF, int WPE>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(WPE, WPE))) mxfp4_tile_kernel(const XArgs xa) {
  using T = TileLoop<MH, NH, NBUF>;
  __shared__ __attribute__((aligned(1024))) char smem[NBUF * T::BUF];
  T t(xa, smem);
  int tm, tn;
  grouped_tile(xcd_logical_id(blockIdx.x, gridDim.x), (xa.m + T::BM - 1) / T::BM, (xa.n + T::BN - 1) / T::BN, tm, tn);
  t.at(tm * T::BM, tn * T::BN);
  t.first_loads();
  __builtin_amdgcn_s_waitcnt(vmcnt_imm((NBUF - 1) * T::LPB));
  __syncthreads();
  t.run();
  t.store(tm * T::BM, tn * T::BN);
}

// 256 x 256 tiles [0, xa.full), 4 waves as 2 x 2 of 128 x 128 (256 sums a lane, in
// AGPRs), by a grid that is resident at once: a workgroup takes one tile after the
// other and its loads never pause, for the next tile's first blocks are loaded
// under the last MFMAs of a tile and land while it is stored.
// k moves in blocks of 128 bytes.  A block's operands are four units of 128 rows
// (A rows 0 .., B rows 0 .., A rows 128 .., B rows 128 ..; rows and swizzle as in
// TileLoop) in a ring of nine; its scale words, 8 KiB, in one of two buffers: all
// of the LDS.  Block d: step 0 multiplies operands that are in registers, reads
// step 1's and loads the first unit of block d + 2 (the ninth slot); behind the
// wait for block d + 1 and the barrier, step 1 reads block d + 1's first operands
// and scale words and loads the other three units and the scale words of block
// d + 2.  With whole blocks in two buffers instead, all loads in half a step, the
// loads came in bursts that the L1 took 1,150 cycles and more to deliver, and the
// matrix units were busy 41% of the time.
template <int UNITS>
struct BigLoop {
  static constexpr int UNIT = 128 * KB, RING = UNITS * UNIT, SBUF = 512 * 16;
  static_assert(RING + 2 * SBUF <= 160 * 1024, "the ring fits the LDS");

  const XArgs &xa;
  char *smem;
  uint32_t lds0;
  int w, wm, wn, lane, li, lg, lch, chunks, nd, tmc, tnc;
  int L, end, wgs;           // the tile whose blocks are loaded, and the workgroup's others
  int lb;                    // its next block
  int tm, tn;                // its place
  int slot, sbuf;            // ring slot of the current block's first unit, its scale buffer
  uint32_t doff[4][4], soff[2], rdq[2], rds[16];
  f32x4 acc[8][8];           // D[n][m]: lane (j, g4) holds n = 16 nb + 4 g4 + (0..3), m = 16 mb + j
  i32x4 cur[16], nxt[16];    // operands: A blocks 0 .. 7, B blocks 0 .. 7
  int sc[16], nsc[16];

  __device__ __forceinline__ BigLoop(const XArgs &args, char *lds) : xa(args), smem(lds) {
    lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)lds;
    lane = threadIdx.x & 63, li = lane & 15, lg = lane >> 4;
    w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = w >> 1, wn = w & 1;
    chunks = xa.k >> 5, nd = (xa.k + 255) >> 8;
    lch = (lane & 7) ^ ((4 * (w & 1) + (lane >> 4)) & 7);
#pragma unroll
    for (int q = 0; q < 2; ++q) rdq[q] = (uint32_t)(li * KB + (((4 * q + lg) ^ ((li >> 1) & 7)) * 16));
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int row = (r < 8 ? wm * 128 + r * 16 : wn * 128 + (r - 8) * 16) + li;
      rds[r] = (uint32_t)(RING + (r < 8 ? 0 : 4096) + (lg * 256 + (row + 16 * lg) % 256) * 4);
    }
    tmc = (xa.m + 255) / 256, tnc = (xa.n + 255) / 256;
  }
  // Where tile L's rows and scale words lie (see TileLoop::at)
  __device__ __forceinline__ void at() {
    grouped_tile(L, tmc, tnc, tm, tn);
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = (j >> 1) * 128 + (w + 4 * i) * 8 + (lane >> 3);
        doff[j][i] = j & 1 ? (uint32_t)((int64_t)min(tn * 256 + r, xa.n - 1) * xa.ldb)
                           : (uint32_t)((int64_t)min(tm * 256 + r, xa.m - 1) * xa.lda);
      }
    const int r = (lane * 4 - 16 * w + 256) % 256;  // entry g = w of A's words, then of B's
    soff[0] = (uint32_t)(((int64_t)w * xa.am4 + min(tm * 256 + r, xa.am4 - 4)) * 4);
    soff[1] = (uint32_t)(((int64_t)w * xa.bn4 + min(tn * 256 + r, xa.bn4 - 4)) * 4);
  }
  // load i of unit j of the block at the load cursor, into ring slot s
  __device__ __forceinline__ void load_data(int s, int j, int i, uint32_t koff) {
    load_lds16_any(j & 1 ? xa.b : xa.a, doff[j][i] + koff, lds0 + (uint32_t)(s * UNIT + (w + 4 * i) * 1024));
  }
  __device__ __forceinline__ void load_scale(int buf, int i) {
    const uint32_t *base = i ? xa.bs + (int64_t)(lb >> 1) * 4 * xa.bn4 : xa.as + (int64_t)(lb >> 1) * 4 * xa.am4;
    load_lds16_any(base, soff[i], lds0 + (uint32_t)(RING + buf * SBUF + i * 4096 + w * 1024));
  }
  __device__ __forceinline__ uint32_t koff() const { return (uint32_t)(min(8 * lb + lch, chunks - 1) * 16); }
  // the load cursor's next block: of this tile, of the workgroup's next one, or
  // (none left) the same again, into slots that nobody reads
  __device__ __forceinline__ void advance() {
    if (lb + 1 < nd) {
      ++lb;
    } else if (L + wgs < end) {
      L += wgs;
      lb = 0;
      at();
    }
  }
  static __device__ __forceinline__ int wrap(int s) { return s >= UNITS ? s - UNITS : s; }
  __device__ __forceinline__ i32x4 read_op(int s, int q, int r) const {  // s: slot of the block's first unit
    const int unit = r < 8 ? 2 * wm : 2 * wn + 1;
    return *(const i32x4 *)(smem + (uint32_t)(wrap(s + unit) * UNIT) + rdq[q] + (r & 7) * 16 * KB);
  }
  __device__ __forceinline__ int read_scale(int buf, int r) const { return *(const int *)(smem + (uint32_t)(buf * SBUF) + rds[r]); }

  // the first tile's first two blocks on their way, the first in registers
  __device__ __forceinline__ void begin() {
    slot = 0, sbuf = 0, lb = 0;
    at();
#pragma unroll
    for (int d = 0; d < 2; ++d) {
      const uint32_t ko = koff();
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) load_data(4 * d + j, j, i, ko);
      load_scale(d, 0);
      load_scale(d, 1);
      advance();
    }
    __builtin_amdgcn_s_waitcnt(vmcnt_imm(18));
    __syncthreads();
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      cur[r] = read_op(0, 0, r);
      sc[r] = read_scale(0, r);
    }
  }
  template <int ODD, bool FIRST>
  __device__ __forceinline__ void block() {
    const int next = wrap(slot + 4), over = wrap(next + 4);  // over: block d + 2's first unit
    uint32_t ko = koff();
#pragma unroll
    for (int idx = 0; idx < 64; ++idx) {
      if (idx % 4 == 0) nxt[idx / 4] = read_op(slot, 1, idx / 4);
      if (idx % 16 == 2) load_data(over, 0, idx / 16, ko);
      mfma_fp4_into<2 * ODD, true, FIRST>(acc[idx >> 3][idx & 7], cur[8 + (idx >> 3)], cur[idx & 7], sc[8 + (idx >> 3)], sc[idx & 7]);
      __builtin_amdgcn_sched_barrier(0);
    }
    __builtin_amdgcn_s_waitcnt(vmcnt_imm(4));
    __syncthreads();
#pragma unroll
    for (int idx = 0; idx < 64; ++idx) {
      if (idx % 4 == 0) {
        cur[idx / 4] = read_op(next, 0, idx / 4);
        nsc[idx / 4] = read_scale(sbuf ^ 1, idx / 4);
      }
      if (idx % 4 == 2 && idx / 4 < 12) load_data(wrap(over + 1 + idx / 16), 1 + idx / 16, idx / 4 % 4, ko);
      if (idx % 4 == 2 && idx / 4 >= 12 && idx / 4 < 14) load_scale(sbuf, idx / 4 - 12);
      mfma_fp4_into<2 * ODD + 1, true>(acc[idx >> 3][idx & 7], nxt[8 + (idx >> 3)], nxt[idx & 7], sc[8 + (idx >> 3)], sc[idx & 7]);
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) sc[r] = nsc[r];
    slot = next, sbuf ^= 1;
    // a register that vector code wrote (a copy above) may be an MFMA's operand two wait states later
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_nop 1");
    __builtin_amdgcn_sched_barrier(0);
  }
  __device__ __forceinline__ void store(int m0, int n0) {
    store_tile<8, 8>(xa, acc, m0 + wm * 128, n0 + wn * 128, li, lg);
  }
};

__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(1, 1))) mxfp4_big_kernel(const XArgs xa) {
  using T = BigLoop<9>;
  __shared__ __attribute__((aligned(1024))) char smem[T::RING + 2 * T::SBUF];
  T t(xa, smem);
  // XCD x = b % 8 takes a contiguous share of the tiles, its workgroups in turn
  const int xcd = blockIdx.x & 7, per = xa.full >> 3, rem = xa.full & 7;
  const int first = xcd * per + min(xcd, rem);
  t.wgs = ((int)gridDim.x - xcd + 7) >> 3;
  t.end = first + per + (xcd < rem);
  t.L = first + (int)(blockIdx.x >> 3);
  if (t.L >= t.end) return;
  int L = t.L;  // the tile that is multiplied
  t.begin();
  for (;;) {
    int d = 1;
    t.template block<0, true>();
    t.advance();
    for (; d + 1 < t.nd; d += 2) {
      t.template block<1, false>();
      t.advance();
      t.template block<0, false>();
      t.advance();
    }
    if (d < t.nd) {
      t.template block<1, false>();
      t.advance();
    }
    mfma_settle<true>(t.acc);
    int tm, tn;
    grouped_tile(L, t.tmc, t.tnc, tm, tn);
    t.store(tm * 256, tn * 256);
    L += t.wgs;
    if (L >= t.end) break;
  }
  // every wave drains its loads before the workgroup ends
  __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
}

int round4(int32_t rows) { return (int)(((int64_t)rows + 3) / 4 * 4); }

int check_matrix(const char *what, int32_t rows, int32_t cols) {
  if (rows < 0 || rows > INT32_MAX - 64) return set_error(TMHD_ERR_INVALID, "%s: rows %d", what, rows);
  if (cols <= 0 || cols % 32) return set_error(TMHD_ERR_UNSUPPORTED, "%s: columns %d must be a positive multiple of 32", what, cols);
  return TMHD_OK;
}

// Workgroups of 4 RQ rows x 512 columns; 0: more than a launch holds.
unsigned quant_grid(int32_t rows, int32_t cols) {
  const int64_t g = (((int64_t)rows + 4 * RQ - 1) / (4 * RQ)) * ((cols + kSuper - 1) / kSuper);
  return g <= INT32_MAX ? (unsigned)g : 0u;
}

// rows that mxfp4_rows_kernel quantizes itself
constexpr int kFusedRows = 16;

int64_t codes_bytes(int32_t rows, int32_t k) { return ((int64_t)rows * (k / 2) + 255) / 256 * 256; }
int64_t scale_bytes(int32_t rows, int32_t k) { return ((int64_t)k + kSuper - 1) / kSuper * 16 * round4(rows); }

int check_product(const char *what, const void *out, const uint8_t *b, const uint8_t *b_scale, const void *bias, int32_t m,
                  int32_t n, int32_t k, int64_t ldb, int64_t ldo) {
  if (int st = check_matrix(what, m, k)) return st;
  if (n <= 0 || n > INT32_MAX - 64) return set_error(TMHD_ERR_INVALID, "%s: n %d", what, n);
  if (m == 0) return TMHD_OK;
  if (!out || !b || !b_scale || (uintptr_t)b % 16 || (uintptr_t)b_scale % 16 || (uintptr_t)out % 2 || (uintptr_t)bias % 2)
    return set_error(TMHD_ERR_INVALID, "%s: null or misaligned pointer", what);
  if (ldb % 16 || ldb < k / 2 || ldo < n)
    return set_error(TMHD_ERR_INVALID, "%s: row strides %lld, %lld", what, (long long)ldb, (long long)ldo);
  if ((m + 63) / 64 > 65535) return set_error(TMHD_ERR_UNSUPPORTED, "%s: m %d is too large", what, m);
  return TMHD_OK;
}

XArgs product_args(void *out, const uint8_t *a, const uint8_t *a_scale, const uint8_t *b, const uint8_t *b_scale,
                   const void *bias, int32_t m, int32_t n, int32_t k, int64_t lda, int64_t ldb, int64_t ldo) {
  return XArgs{a, b, (const uint32_t *)a_scale, (const uint32_t *)b_scale, (uint16_t *)out, (const uint16_t *)bias,
               m, n, k, round4(m), round4(n), lda, ldb, ldo,
               (int32_t)((uintptr_t)out % 8 == 0 && ldo % 4 == 0), (int32_t)((uintptr_t)out % 16 == 0 && ldo % 8 == 0), 0};
}

// The product of checked arguments.
int launch_product(const char *what, void *out, const uint8_t *a, const uint8_t *a_scale, const uint8_t *b,
                   const uint8_t *b_scale, const void *bias, int32_t m, int32_t n, int32_t k, int64_t lda, int64_t ldb,
                   int64_t ldo, hipStream_t s) {
  XArgs xa = product_args(out, a, a_scale, b, b_scale, bias, m, n, k, lda, ldb, ldo);
  const unsigned nt = (unsigned)((n + 15) / 16);
  // the tiles take 32-bit row and scale offsets
  const bool wide = (int64_t)(m - 1) * lda + k < (int64_t)1 << 32 && (int64_t)(n - 1) * ldb + k < (int64_t)1 << 32;
  if (wide && m > 64) {
    const int64_t big = ((int64_t)(m + 255) / 256) * ((n + 255) / 256);
    if (big >= 128) {
      xa.full = (int32_t)big;
      hipLaunchKernelGGL(mxfp4_big_kernel, dim3((unsigned)std::min<int64_t>(big, std::max(device_cus(), 8))), dim3(256), 0, s, xa);
    }
    else
      hipLaunchKernelGGL((mxfp4_tile_kernel<64, 64, 4, 1>), dim3((unsigned)(((int64_t)(m + 127) / 128) * ((n + 127) / 128))),
                         dim3(256), 0, s, xa);
  } else if (m <= 16)
    hipLaunchKernelGGL((mxfp4_rows_kernel<1, 4, false>), dim3(nt, 1), dim3(256), 0, s, xa);
  else
    hipLaunchKernelGGL((mxfp4_rows_kernel<4, 4, false>), dim3(nt, (unsigned)((m + 63) / 64)), dim3(256), 0, s, xa);
  return check_launch(what);
}

}  // namespace
}  // namespace tmhd

extern "C" int tmhd_mxfp4_quant(uint8_t *q, uint8_t *scale, const void *x, int32_t rows, int32_t cols,
                                int64_t x_stride, void *stream) {
  using namespace tmhd;
  const char *what = "tmhd_mxfp4_quant";
  if (int st = check_matrix(what, rows, cols)) return st;
  if (rows == 0) return TMHD_OK;
  if (!q || !scale || !x || (uintptr_t)x % 16 || (uintptr_t)q % 16 || (uintptr_t)scale % 16)
    return set_error(TMHD_ERR_INVALID, "%s: null or misaligned pointer", what);
  if (x_stride < cols || x_stride % 8) return set_error(TMHD_ERR_INVALID, "%s: row stride %lld", what, (long long)x_stride);
  const unsigned grid = quant_grid(rows, cols);
  if (!grid) return set_error(TMHD_ERR_UNSUPPORTED, "%s: %d x %d is too large", what, rows, cols);
  hipLaunchKernelGGL(mxfp4_quant_kernel, dim3(grid), dim3(256), 0, (hipStream_t)stream, q, (uint32_t *)scale,
                     (const uint16_t *)x, rows, round4(rows), cols, x_stride, (cols + kSuper - 1) / kSuper);
  return check_launch(what);
}

extern "C" int tmhd_mxfp4_dequant(void *x, const uint8_t *q, const uint8_t *scale, int32_t rows, int32_t cols,
                                  void *stream) {
  using namespace tmhd;
  const char *what = "tmhd_mxfp4_dequant";
  if (int st = check_matrix(what, rows, cols)) return st;
  if (rows == 0) return TMHD_OK;
  if (!q || !scale || !x || (uintptr_t)x % 16 || (uintptr_t)q % 16 || (uintptr_t)scale % 16)
    return set_error(TMHD_ERR_INVALID, "%s: null or misaligned pointer", what);
  const unsigned grid = quant_grid(rows, cols);
  if (!grid) return set_error(TMHD_ERR_UNSUPPORTED, "%s: %d x %d is too large", what, rows, cols);
  hipLaunchKernelGGL(mxfp4_dequant_kernel, dim3(grid), dim3(256), 0, (hipStream_t)stream, (uint16_t *)x, q,
                     (const uint32_t *)scale, rows, round4(rows), cols, (cols + kSuper - 1) / kSuper);
  return check_launch(what);
}

extern "C" int tmhd_gemm_mxfp4(void *out, const uint8_t *a, const uint8_t *b, const uint8_t *a_scale,
                               const uint8_t *b_scale, const void *bias, int32_t m, int32_t n, int32_t k, int64_t lda,
                               int64_t ldb, int64_t ldo, void *stream) {
  using namespace tmhd;
  const char *what = "tmhd_gemm_mxfp4";
  if (int st = check_product(what, out, b, b_scale, bias, m, n, k, ldb, ldo)) return st;
  if (m == 0) return TMHD_OK;
  if (!a || !a_scale || (uintptr_t)a % 16 || (uintptr_t)a_scale % 16)
    return set_error(TMHD_ERR_INVALID, "%s: null or misaligned pointer", what);
  if (lda % 16 || lda < k / 2) return set_error(TMHD_ERR_INVALID, "%s: row stride %lld", what, (long long)lda);
  return launch_product(what, out, a, a_scale, b, b_scale, bias, m, n, k, lda, ldb, ldo, (hipStream_t)stream);
}

extern "C" int64_t tmhd_linear_mxfp4_workspace_bytes(int32_t m, int32_t n, int32_t k) {
  (void)n;
  if (m <= tmhd::kFusedRows || k <= 0 || k % 32) return 0;
  return tmhd::codes_bytes(m, k) + tmhd::scale_bytes(m, k);
}

extern "C" int tmhd_linear_mxfp4(void *out, const void *x, const uint8_t *b, const uint8_t *b_scale, const void *bias,
                                 int32_t m, int32_t n, int32_t k, int64_t ldx, int64_t ldb, int64_t ldo,
                                 void *workspace, int64_t workspace_bytes, void *stream) {
  using namespace tmhd;
  const char *what = "tmhd_linear_mxfp4";
  if (int st = check_product(what, out, b, b_scale, bias, m, n, k, ldb, ldo)) return st;
  if (m == 0) return TMHD_OK;
  if (!x || (uintptr_t)x % 16) return set_error(TMHD_ERR_INVALID, "%s: null or misaligned pointer", what);
  if (ldx % 8 || ldx < k) return set_error(TMHD_ERR_INVALID, "%s: row stride %lld", what, (long long)ldx);
  hipStream_t s = (hipStream_t)stream;
  if (m <= kFusedRows) {
    const XArgs xa = product_args(out, (const uint8_t *)x, nullptr, b, b_scale, bias, m, n, k, ldx, ldb, ldo);
    hipLaunchKernelGGL((mxfp4_rows_kernel<1, 4, true>), dim3((unsigned)((n + 15) / 16)), dim3(256), 0, s, xa);
    return check_launch(what);
  }
  if (!workspace || (uintptr_t)workspace % 16 || workspace_bytes < codes_bytes(m, k) + scale_bytes(m, k))
    return set_error(TMHD_ERR_INVALID, "%s: workspace of %lld bytes", what, (long long)workspace_bytes);
  uint8_t *q = (uint8_t *)workspace, *scale = q + codes_bytes(m, k);
  if (int st = tmhd_mxfp4_quant(q, scale, x, m, k, ldx, stream)) return st;
  return launch_product(what, out, q, scale, b, b_scale, bias, m, n, k, k / 2, ldb, ldo, s);
}
