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
// saturates.  12,252 x 5,376: 32 us (5.2 TB/s); the inverse 26 (6.4, its codes partly
// from the Infinity Cache).
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

// The wait states between the last MFMAs and code that reads their results (the
// sums named on both sides, so that neither may move across).
template <bool IN_AGPR, int NB, int MB>
__device__ __forceinline__ void mfma_settle(f32x4 (&acc)[NB][MB]) {
  auto hold = [&]() {
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
      for (int j = 0; j < MB; ++j) {
        if constexpr (IN_AGPR)
          asm volatile("" : "+a"(acc[i][j]));
        else
          asm volatile("" : "+v"(acc[i][j]));
      }
  };
  hold();
  asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");
  hold();
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

// Few rows: 16 columns of n and 16 rows of m a workgroup, its four waves take the
// 512-column blocks of k in turn, straight from global memory to the MFMA (each
// code is used once), and add their sums through LDS in wave order.  Bound by the
// weight's bytes and the latency of its loads; 1 x 5,376 x 5,376 5.6 us (2.7 TB/s).  (Also
// the form of matrices beyond 32-bit offsets.)  QUANT: the rows are bf16 (xa.a, lda in
// elements); a lane's operand is a whole 32-column block, so it finds the block's
// scale and codes by itself.
template <bool QUANT>
__global__ void __launch_bounds__(256) mxfp4_rows_kernel(const XArgs xa) {
  constexpr int W = 4;
  __shared__ f32x4 part[W][64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, li = lane & 15, lg = lane >> 4;
  const int tiles_n = (xa.n + 15) / 16;
  const int n0 = (int)(blockIdx.x % tiles_n) * 16, m0 = (int)(blockIdx.x / tiles_n) * 16;
  const int chunks = xa.k >> 5, blocks = (xa.k + kSuper - 1) / kSuper;
  const int brow = min(n0 + li, xa.n - 1), arow = min(m0 + li, xa.m - 1);
  const uint8_t *bp = xa.b + (int64_t)brow * xa.ldb + lg * 16;
  const uint8_t *ap = xa.a + (int64_t)arow * xa.lda * (QUANT ? 2 : 1) + lg * (QUANT ? 64 : 16);
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  for (int s = w; s < blocks; s += W) {
    // chunk 16 s + 4 t + lg; behind the last column: zero codes (their scale bytes are zero too)
    const int64_t at = (int64_t)s * (kSuper / 2);
    i32x4 bv[4], av[4];
    const int sb = (int)xa.bs[scale_word(s, lg, brow, xa.bn4)];
    int sa;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const bool in = 16 * s + 4 * t + lg < chunks;
      bv[t] = in ? *(const i32x4 *)(bp + at + 64 * t) : i32x4{0, 0, 0, 0};
    }
    if constexpr (QUANT) {
      sa = 0;
      i32x4 x[4][4];
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          x[t][e] = 16 * s + 4 * t + lg < chunks ? *(const i32x4 *)(ap + 4 * (at + 64 * t) + 16 * e) : i32x4{0, 0, 0, 0};
#pragma unroll
      for (int t = 0; t < 4; ++t) sa |= (int)(quant32(x[t], av[t]) << (8 * t));
    } else {
#pragma unroll
      for (int t = 0; t < 4; ++t)
        av[t] = 16 * s + 4 * t + lg < chunks ? *(const i32x4 *)(ap + at + 64 * t) : i32x4{0, 0, 0, 0};
      sa = (int)xa.as[scale_word(s, lg, arow, xa.am4)];
    }
    acc = mfma_fp4<0>(bv[0], av[0], acc, sb, sa);
    acc = mfma_fp4<1>(bv[1], av[1], acc, sb, sa);
    acc = mfma_fp4<2>(bv[2], av[2], acc, sb, sa);
    acc = mfma_fp4<3>(bv[3], av[3], acc, sb, sa);
  }
  part[w][lane] = acc;
  __syncthreads();
  if (w) return;
#pragma unroll
  for (int i = 1; i < W; ++i) acc += part[i][lane];
  store_quad(xa, acc, m0 + li, n0 + 4 * lg);
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

// A wave's sums, rounded to bf16 and stored from registers: rows m0 .., columns n0 ...  A
// pair of 16-column blocks trades halves between neighbouring lane groups, so that a
// lane holds 8 consecutive columns of one block (16 bytes).  WHOLE: every row and
// column is inside the matrix and rows are 16-byte aligned: one address a row.  Rows of
// another alignment (a width that is not a multiple of 8) are stored two bytes at a
// time: 12,252 x 9,001 x 832 271 us, 9,008 columns 83; 4,836 x 10,751 x 5,376 222, 10,752
// columns 132; 331 x 10,751 x 5,376 22 and 15.
template <int NB, int MB, bool BIAS, bool WHOLE>
__device__ __forceinline__ void store_blocks(const XArgs &xa, const f32x4 (&acc)[NB][MB], int m0, int n0, int li, int lg) {
  const int n1 = n0 + (lg & 1) * 16 + 8 * (lg >> 1);  // first of the lane's stored columns
  float bf[NB][4];
  if constexpr (BIAS) {
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int n = n0 + i * 16 + 4 * lg + e;
        bf[i][e] = bf16_bits_to_f32(xa.bias[WHOLE ? n : min(n, xa.n - 1)]);
      }
  }
#pragma unroll
  for (int j = 0; j < MB; ++j) {
    const int m = m0 + j * 16 + li;
    uint16_t *row = xa.out + (int64_t)m * xa.ldo + n1;
#pragma unroll
    for (int i = 0; i < NB; i += 2) {
      uint32_t p[2][2];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          p[h][e] = BIAS ? pack_bf16_rne(acc[i + h][j][2 * e] + bf[i + h][2 * e], acc[i + h][j][2 * e + 1] + bf[i + h][2 * e + 1])
                         : pack_bf16_rne(acc[i + h][j][2 * e], acc[i + h][j][2 * e + 1]);
      const auto lo = __builtin_amdgcn_permlane16_swap(p[0][0], p[1][0], false, false);
      const auto hi = __builtin_amdgcn_permlane16_swap(p[0][1], p[1][1], false, false);
      const i32x4 v = {(int)lo[0], (int)hi[0], (int)lo[1], (int)hi[1]};
      if constexpr (WHOLE) {
        *(i32x4 *)(row + i * 16) = v;
      } else {
        const int nn = n1 + i * 16;
        if (m >= xa.m || nn >= xa.n) continue;
        if (xa.st16_ok && nn + 7 < xa.n)
          *(i32x4 *)(row + i * 16) = v;
        else
          for (int e = 0; e < 8 && nn + e < xa.n; ++e) row[i * 16 + e] = (uint16_t)((uint32_t)v[e >> 1] >> (16 * (e & 1)));
      }
    }
  }
}

template <int NB, int MB>
__device__ __forceinline__ void store_tile(const XArgs &xa, const f32x4 (&acc)[NB][MB], int m0, int n0, int li, int lg) {
  if (xa.st16_ok && m0 + MB * 16 <= xa.m && n0 + NB * 16 <= xa.n) {
    if (xa.bias)
      store_blocks<NB, MB, true, true>(xa, acc, m0, n0, li, lg);
    else
      store_blocks<NB, MB, false, true>(xa, acc, m0, n0, li, lg);
  } else if (xa.bias) {
    store_blocks<NB, MB, true, false>(xa, acc, m0, n0, li, lg);
  } else {
    store_blocks<NB, MB, false, false>(xa, acc, m0, n0, li, lg);
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
      load_lds16_base(n < AL ? xa.a : xa.b, doff[n] + koff, dst);
    } else {
      const int i = n - DL;
      const uint32_t *base = scale_of_a(i) ? xa.as + (int64_t)(d >> 1) * 4 * xa.am4 : xa.bs + (int64_t)(d >> 1) * 4 * xa.bn4;
      load_lds16_base(base, soff[i], to + sdst[i]);
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
};

// Tiles smaller than 256 x 256, one a workgroup: all of the matrix (xa.full < 0), or
// the parts of the 256 x 256 tiles from xa.full on.
template <int MH, int NH, int NBUF, int WPE>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(WPE, WPE))) mxfp4_tile_kernel(const XArgs xa) {
  using T = TileLoop<MH, NH, NBUF>;
  __shared__ __attribute__((aligned(1024))) char smem[NBUF * T::BUF];
  T t(xa, smem);
  const int L = xcd_logical_id(blockIdx.x, gridDim.x);
  int m0, n0;
  if (xa.full >= 0) {
    // consecutive ids, which run on one XCD, are parts of one tile
    constexpr int PM = 256 / T::BM, PN = 256 / T::BN;
    int tm, tn;
    grouped_tile(xa.full + L / (PM * PN), (xa.m + 255) / 256, (xa.n + 255) / 256, tm, tn);
    m0 = tm * 256 + L % (PM * PN) / PN * T::BM, n0 = tn * 256 + L % PN * T::BN;
    if (m0 >= xa.m || n0 >= xa.n) return;  // the whole workgroup: no barrier is left waiting
  } else {
    // the row tiles that share a weight panel run next to each other
    const int tmc = (xa.m + T::BM - 1) / T::BM;
    m0 = L % tmc * T::BM, n0 = L / tmc * T::BN;
  }
  t.at(m0, n0);
  t.first_loads();
  __builtin_amdgcn_s_waitcnt(vmcnt_imm((NBUF - 1) * T::LPB));
  __syncthreads();
  t.run();
  store_tile<T::NB, T::MB>(xa, t.acc, m0 + t.wm * MH, n0 + t.wn * NH, t.li, t.lg);
}

// 256 x 256 tiles [0, xa.full), 8 waves as 2 x 4 of 128 x 64 (128 sums a lane, in
// AGPRs), two on a SIMD, by a grid that is resident at once: a workgroup takes one tile
// after the other and its loads never pause, for the next tile's first blocks are loaded
// under the last MFMAs of a tile and land while it is stored.
// k moves in blocks of 128 bytes.  A block's operands are four units of 128 rows
// (A rows 0 .., B rows 0 .., A rows 128 .., B rows 128 ..; rows and swizzle as in
// TileLoop) in a ring of nine; the scale words of two blocks, 8 KiB, in one of two
// buffers: all of the LDS.  An operand's register is read anew behind its last MFMA of
// the step: in step 0 of block d for step 1, in step 1 for block d + 1 (with its scale
// bytes), behind the wait for that block and the barrier, which come when step 1's
// operands have long arrived.  Step 0 loads the first unit of block d + 2 (the ninth
// slot), step 1 the other three and their scale words.
// 12,252 x 13,824 x 5,120 397 to 425 us by card (404: 4,290 TFLOPS), 4,836 x 10,752 x
// 5,376 132 us (4,220), the last round in smaller tiles in both; under a profiler, ten
// calls with pauses, 430 to 453.  Four waves of 128 x 128, each step's operands read
// a step ahead into a second set of registers, took 411 and 137 us, 2,717 x 5,376 x
// 5,376 47 against 43.  Without stores it takes 352 us, without loads and stores 294, and
// the MFMAs alone take 243 at the clock that the power limit leaves them: what the tile
// moves costs time by its energy more than by its latency (the barrier, earlier or
// later in the step, and wave priorities change nothing).
template <int UNITS>
struct BigLoop {
  static constexpr int UNIT = 128 * KB, RING = UNITS * UNIT, SBUF = 512 * 16;
  static_assert(RING + 2 * SBUF <= 160 * 1024, "the ring fits the LDS");

  const XArgs &xa;
  char *smem;
  uint32_t lds0;
  int w, wm, wn, lane, li, lg, lch, chunks, nd, tmc, tnc;
  int L, end, wgs;             // the tile whose blocks are loaded, and the workgroup's others
  int lb;                      // its next block
  const uint8_t *abase, *bbase;  // the codes from that block on
  int slot;                    // ring slot of the current block's first unit
  int sload;                   // buffer of the next scale words
  int sread, rb;               // where the next block's scale bytes are read, and its number in its tile
  uint32_t doff[4][2], soff, rdq[2], rds[2][4];
  f32x4 acc[4][8];             // D[n][m]: lane (j, g4) holds n = 16 nb + 4 g4 + (0..3), m = 16 mb + j
  i32x4 cur[12];               // operands: A blocks 0 .. 7, B blocks 0 .. 3
  int sc[12];                  // their scale words

  __device__ __forceinline__ BigLoop(const XArgs &args, char *lds) : xa(args), smem(lds) {
    lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)lds;
    lane = threadIdx.x & 63, li = lane & 15, lg = lane >> 4;
    w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = w >> 2, wn = w & 3;
    chunks = xa.k >> 5, nd = (xa.k + 255) >> 8;
    lch = (lane & 7) ^ ((4 * (w & 1) + (lane >> 4)) & 7);
#pragma unroll
    for (int q = 0; q < 2; ++q) rdq[q] = (uint32_t)(li * KB + (((4 * q + lg) ^ ((li >> 1) & 7)) * 16));
    // scale word of entry g, row r: word r ^ 16 g of the entry's 256 (a read of 16
    // rows and 4 entries meets 64 banks); rds: by r / 16 mod 4
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const uint32_t word = (uint32_t)(RING + lg * 1024 + ((c ^ lg) * 16 + li) * 4);
      rds[0][c] = word + wm * 512, rds[1][c] = word + 4096 + wn * 256;
    }
    tmc = (xa.m + 255) / 256, tnc = (xa.n + 255) / 256;
  }
  // Where tile L's rows and scale words lie (see TileLoop::at), from its first block
  __device__ __forceinline__ void at() {
    int tm, tn;
    grouped_tile(L, tmc, tnc, tm, tn);
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = (j >> 1) * 128 + (w + 8 * i) * 8 + (lane >> 3);
        doff[j][i] = (j & 1 ? (uint32_t)((int64_t)min(tn * 256 + r, xa.n - 1) * xa.ldb)
                            : (uint32_t)((int64_t)min(tm * 256 + r, xa.m - 1) * xa.lda)) + lch * 16;
      }
    const int e = w & 3, r = (lane * 4) ^ (16 * e);  // entry e of A's words (waves 0 .. 3) or of B's
    soff = (uint32_t)(w < 4 ? ((int64_t)e * xa.am4 + min(tm * 256 + r, xa.am4 - 4)) * 4 : ((int64_t)e * xa.bn4 + min(tn * 256 + r, xa.bn4 - 4)) * 4);
    lb = 0, abase = xa.a, bbase = xa.b;
    if (nd == 1) last_block();
  }
  // the load cursor is at the row's last block: chunks past the row's end repeat its last
  __device__ __forceinline__ void last_block() {
    const uint32_t back = (uint32_t)max(8 * (nd - 1) + lch - (chunks - 1), 0) * 16;
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < 2; ++i) doff[j][i] -= back;
  }
  // load i of unit j of the block at the load cursor, into ring slot s
  __device__ __forceinline__ void load_data(int s, int j, int i) {
    load_lds16_base(j & 1 ? bbase : abase, doff[j][i], lds0 + (uint32_t)(s * UNIT + (w + 8 * i) * 1024));
  }
  __device__ __forceinline__ void load_scales() {
    const uint32_t to = lds0 + (uint32_t)(RING + sload * SBUF + w * 1024);
    load_lds16_base(w < 4 ? xa.as + (int64_t)(lb >> 1) * 4 * xa.am4 : xa.bs + (int64_t)(lb >> 1) * 4 * xa.bn4, soff, to);
    sload ^= 1;
  }
  // the load cursor's next block: of this tile, of the workgroup's next one, or
  // (none left) the same again, into slots that nobody reads
  __device__ __forceinline__ void advance() {
    if (lb + 1 < nd) {
      ++lb;
      abase += KB, bbase += KB;
      if (lb + 1 == nd && (chunks & 7)) last_block();
    } else if (L + wgs < end) {
      L += wgs;
      at();
    }
  }
  static __device__ __forceinline__ int wrap(int s) { return s >= UNITS ? s - UNITS : s; }
  // operand r (A blocks 0 .. 7, then B's) of step q of the block whose units start at ring slot s
  __device__ __forceinline__ uint32_t op_base(int s, int q, bool b) const {
    return (uint32_t)(wrap(s + (b ? (wn & 2) + 1 : 2 * wm)) * UNIT + (b ? (wn & 1) * 64 * KB : 0)) + rdq[q];
  }
  __device__ __forceinline__ i32x4 read_op(uint32_t base, int r) const { return *(const i32x4 *)(smem + base + (r & 7) * 16 * KB); }
  // scale bytes of operand r for the block whose bytes start at `from` of the buffers: step 0's, then step 1's
  __device__ __forceinline__ int read_scale(const uint32_t (&at)[2][4], int r) const {
    return *(const uint16_t *)(smem + at[r >> 3][r & 3] + ((r & 7) >> 2) * 256);
  }
  // where the next block's scale bytes are read: the other two bytes of the words, or the other buffer's first two
  __device__ __forceinline__ void next_scales() { sread = rb & 1 ? (sread ^ SBUF) & ~2 : rb + 1 == nd ? sread ^ SBUF : sread | 2, rb = rb + 1 == nd ? 0 : rb + 1; }

  // the first tile's first two blocks on their way, the first in registers
  __device__ __forceinline__ void begin() {
    slot = 0, sload = 0;
    at();
#pragma unroll
    for (int d = 0; d < 2; ++d) {
      if ((lb & 1) == 0) load_scales();
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int i = 0; i < 2; ++i) load_data(4 * d + j, j, i);
      advance();
    }
    __builtin_amdgcn_s_waitcnt(vmcnt_imm(8));
    __syncthreads();
    const uint32_t a = op_base(0, 0, false), b = op_base(0, 0, true);
#pragma unroll
    for (int r = 0; r < 12; ++r) {
      cur[r] = read_op(r < 8 ? a : b, r);
      sc[r] = read_scale(rds, r);
    }
    sread = 0, rb = 0;
    next_scales();
    clear();
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  __device__ __forceinline__ void block() {
    const int next = wrap(slot + 4), over = wrap(next + 4);  // over: block d + 2's first unit
    {
      const uint32_t a = op_base(slot, 1, false), b = op_base(slot, 1, true);
#pragma unroll
      for (int idx = 0; idx < 32; ++idx) {
        const int nb = idx >> 3, mb = idx & 7;
        if (idx % 16 == 2) load_data(over, 0, idx / 16);
        mfma_fp4_into<0, true>(acc[nb][mb], cur[8 + nb], cur[mb], sc[8 + nb], sc[mb]);
        __builtin_amdgcn_sched_barrier(0);
        if (nb == 3) cur[mb] = read_op(a, mb);
        if (mb == 7) cur[8 + nb] = read_op(b, 8 + nb);
      }
    }
    uint32_t at[2][4];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int c = 0; c < 4; ++c) at[h][c] = rds[h][c] + sread;
    {
      const uint32_t a = op_base(next, 0, false), b = op_base(next, 0, true);
#pragma unroll
      for (int idx = 0; idx < 32; ++idx) {
        const int nb = idx >> 3, mb = idx & 7;
        if (idx == 6) {
          __builtin_amdgcn_s_waitcnt(vmcnt_imm(2));
          __syncthreads();
          if ((lb & 1) == 0) load_scales();
        }
        if (idx >= 8 && idx % 4 == 0) load_data(wrap(over + 1 + (idx - 8) / 8), 1 + (idx - 8) / 8, (idx - 8) / 4 % 2);
        mfma_fp4_into<1, true>(acc[nb][mb], cur[8 + nb], cur[mb], sc[8 + nb], sc[mb]);
        __builtin_amdgcn_sched_barrier(0);
        if (nb == 3) cur[mb] = read_op(a, mb), sc[mb] = read_scale(at, mb);
        if (mb == 7) cur[8 + nb] = read_op(b, 8 + nb), sc[8 + nb] = read_scale(at, 8 + nb);
      }
    }
    next_scales();
    slot = next;
    advance();
    // a register that vector code wrote may be an MFMA's operand two wait states later
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_nop 1");
    __builtin_amdgcn_sched_barrier(0);
  }
};

__global__ void __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2, 2))) mxfp4_big_kernel(const XArgs xa) {
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
    for (int d = 0; d < t.nd; ++d) t.block();
    mfma_settle<true>(t.acc);
    int tm, tn;
    grouped_tile(L, t.tmc, t.tnc, tm, tn);
    store_tile<4, 8>(xa, t.acc, tm * 256 + t.wm * 128, tn * 256 + t.wn * 64, t.li, t.lg);
    L += t.wgs;
    if (L >= t.end) break;
    t.clear();
  }
  // every wave drains its loads before the workgroup ends
  __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
}

int round4(int32_t rows) { return (int)(((int64_t)rows + 3) / 4 * 4); }

int check_matrix(const char *what, int32_t rows, int32_t cols) {
  if (rows < 0 || rows > INT32_MAX - 256) return set_error(TMHD_ERR_INVALID, "%s: rows %d", what, rows);
  if (cols <= 0 || cols % 32) return set_error(TMHD_ERR_UNSUPPORTED, "%s: columns %d must be a positive multiple of 32", what, cols);
  return TMHD_OK;
}

constexpr int64_t kMaxGrid = (1 << 24) - 1;  // workgroups of 256 threads that a launch holds

// Workgroups of 4 RQ rows x 512 columns; 0: more than a launch holds.
unsigned quant_grid(int32_t rows, int32_t cols) {
  const int64_t g = (((int64_t)rows + 4 * RQ - 1) / (4 * RQ)) * ((cols + kSuper - 1) / kSuper);
  return g <= kMaxGrid ? (unsigned)g : 0u;
}

int64_t codes_bytes(int32_t rows, int32_t k) { return ((int64_t)rows * (k / 2) + 255) / 256 * 256; }
int64_t scale_bytes(int32_t rows, int32_t k) { return ((int64_t)k + kSuper - 1) / kSuper * 16 * round4(rows); }

int check_product(const char *what, const void *out, const uint8_t *b, const uint8_t *b_scale, const void *bias, int32_t m,
                  int32_t n, int32_t k, int64_t ldb, int64_t ldo) {
  if (int st = check_matrix(what, m, k)) return st;
  if (n <= 0 || n > INT32_MAX - 256) return set_error(TMHD_ERR_INVALID, "%s: n %d", what, n);
  if (m == 0) return TMHD_OK;
  if (!out || !b || !b_scale || (uintptr_t)b % 16 || (uintptr_t)b_scale % 16 || (uintptr_t)out % 2 || (uintptr_t)bias % 2)
    return set_error(TMHD_ERR_INVALID, "%s: null or misaligned pointer", what);
  if (ldb % 16 || ldb < k / 2 || ldo < n)
    return set_error(TMHD_ERR_INVALID, "%s: row strides %lld, %lld", what, (long long)ldb, (long long)ldo);
  return TMHD_OK;
}

XArgs product_args(void *out, const uint8_t *a, const uint8_t *a_scale, const uint8_t *b, const uint8_t *b_scale,
                   const void *bias, int32_t m, int32_t n, int32_t k, int64_t lda, int64_t ldb, int64_t ldo) {
  return XArgs{a, b, (const uint32_t *)a_scale, (const uint32_t *)b_scale, (uint16_t *)out, (const uint16_t *)bias,
               m, n, k, round4(m), round4(n), lda, ldb, ldo,
               (int32_t)((uintptr_t)out % 8 == 0 && ldo % 4 == 0), (int32_t)((uintptr_t)out % 16 == 0 && ldo % 8 == 0), 0};
}

// Tiles of 2 MH x 2 NH: the parts of the last `tiles` 256 x 256 tiles, or (0) all of the matrix.
template <int MH, int NH, int NBUF, int WPE>
void launch_tiles(XArgs xa, int64_t tiles, hipStream_t s) {
  const int64_t wgs = tiles ? tiles * (256 / (2 * MH)) * (256 / (2 * NH))
                            : (int64_t)((xa.m + 2 * MH - 1) / (2 * MH)) * ((xa.n + 2 * NH - 1) / (2 * NH));
  if (!tiles) xa.full = -1;
  hipLaunchKernelGGL((mxfp4_tile_kernel<MH, NH, NBUF, WPE>), dim3((unsigned)wgs), dim3(256), 0, s, xa);
}

// The tiled forms and, per 256 columns of k, the microseconds of a round of them:
// `one` + `fill` * (share of the CUs in use), or `two` with a second workgroup on
// each CU.  Fitted to every form forced on products of 1 to 12,252 rows and weights
// of 640 x 2,048 to 13,824 x 5,120 that were not read shortly before; us, rows on
// 13,824 x 5,120 (and on 5,376 x 5,376):
//   rows          1            64           200          331          1,024        2,048
//   64 x 64       7.8  (7.2)   8.7  (7.7)   21.6 (11.7)  30.7 (12.4)  70   (30.7)  177  (71)
//   128 x 64      10.3 (9.9)   11.0 (10.3)  21.0 (11.0)  30.6 (11.5)  67   (29.9)  144  (63)
//   128 x 128     13.1 (12.9)  13.8 (13.3)  15.9 (14.3)  27.5 (14.4)  57.6 (28.2)  105  (46)
//   128 x 128, 2  14.7 (14.2)  15.4 (14.5)  16.6 (15.2)  22.8 (15.3)  44.2 (21.8)  86   (41)
//   256 x 256     32.3 (31.7)  31.6 (31.9)  34.3 (34.2)  36.5 (35.6)  44.7 (38.4)  81   (42)
struct TileCost {
  int form, bm, bn, per_cu;
  double one, fill, two;
};
constexpr TileCost kTiles[] = {
    {TMHD_MXFP4_64X64, 64, 64, 2, 0.20, 0.03, 0.46},
    {TMHD_MXFP4_128X64, 128, 64, 1, 0.37, 0.02, 0.0},
    {TMHD_MXFP4_128X128, 128, 128, 1, 0.52, 0.10, 0.0},
    {TMHD_MXFP4_128X128X2, 128, 128, 2, 0.58, 0.08, 1.12},
    {TMHD_MXFP4_256X256, 256, 256, 1, 1.32, 0.74, 0.0},
};
constexpr double kLaunchUs = 3.5;  // first loads, stores and the launch itself

double tiles_us(const TileCost &c, int64_t wgs, double blocks, int cus) {
  const int64_t slots = (int64_t)cus * c.per_cu, rest = wgs % slots;
  const double full = c.per_cu == 2 ? c.two : c.one + c.fill;
  const double last = rest == 0 ? 0.0 : rest <= cus ? c.one + c.fill * (double)rest / cus : c.two;
  return kLaunchUs + blocks * ((double)(wgs / slots) * full + last);
}

// The cheapest form of an m x n x k product: `rows` or tiles of one kind, or 256 x
// 256 tiles in whole rounds and `tail` tiles of another kind behind them.
struct Form {
  int form;
  int64_t tail;  // 256 x 256 tiles that `form` runs in parts; 0: `form` runs all
};
Form pick_form(int32_t m, int32_t n, int32_t k, int cus) {
  // 16 x 16 tiles straight from memory: up to 16 rows and about a workgroup and a
  // half per CU (1 row on 5,376 x 5,376: 5.6 us, 64 x 64 tiles 7.2; on 13,824 x
  // 5,120 8.7 and 7.8; on 640 x 2,048 4.0 and 4.5)
  if (m <= 16 && (n + 15) / 16 <= cus * 3 / 2) return {TMHD_MXFP4_ROWS, 0};
  const double blocks = (double)((k + 255) / 256);
  const int64_t big = (int64_t)((m + 255) / 256) * ((n + 255) / 256);
  Form best{TMHD_MXFP4_256X256, 0};
  double us = 1e30;
  for (const TileCost &c : kTiles) {
    const double t = tiles_us(c, (int64_t)((m + c.bm - 1) / c.bm) * ((n + c.bn - 1) / c.bn), blocks, cus);
    if (t < us) us = t, best = {c.form, 0};
  }
  const int64_t tail = big % cus;
  if (big > cus && tail) {
    const double whole = blocks * (double)(big / cus) * 2.06;
    for (const TileCost &c : kTiles) {
      if (c.form != TMHD_MXFP4_64X64 && c.form != TMHD_MXFP4_128X64 && c.form != TMHD_MXFP4_128X128) continue;
      const double t = kLaunchUs + whole + tiles_us(c, tail * (256 / c.bm) * (256 / c.bn), blocks, cus);
      if (t < us) us = t, best = {c.form, tail};
    }
  }
  return best;
}

// Whether mxfp4_rows_kernel quantizes the rows itself: it takes the product, and its
// waves have one block of k each.  A launch less (1 row on 640 x 2,048: 3.6 us
// against 4.8, 16 rows 4.9 and 5.5), but every workgroup quantizes all of k: with
// more of it a wave's blocks wait for each other (1 row on 5,376 x 5,376: 9.2 against
// 8.1, 16 rows 15.8 and 10.3).
bool fused_quant(int32_t m, int32_t n, int32_t k) {
  return m <= 16 && k <= 4 * kSuper && pick_form(m, n, k, std::max(device_cus(), 8)).form == TMHD_MXFP4_ROWS;
}

// The product of checked arguments.
int launch_product(const char *what, void *out, const uint8_t *a, const uint8_t *a_scale, const uint8_t *b,
                   const uint8_t *b_scale, const void *bias, int32_t m, int32_t n, int32_t k, int64_t lda, int64_t ldb,
                   int64_t ldo, hipStream_t s) {
  XArgs xa = product_args(out, a, a_scale, b, b_scale, bias, m, n, k, lda, ldb, ldo);
  const int cus = std::max(device_cus(), 8);
  // the tiles take 32-bit row and scale offsets
  const bool narrow = (int64_t)(m - 1) * lda + k < (int64_t)1 << 32 && (int64_t)(n - 1) * ldb + k < (int64_t)1 << 32;
  const Form f = narrow ? pick_form(m, n, k, cus) : Form{TMHD_MXFP4_ROWS, 0};
  const int64_t big = (int64_t)((m + 255) / 256) * ((n + 255) / 256);
  const int64_t rows_grid = (int64_t)((m + 15) / 16) * ((n + 15) / 16);
  if (f.form == TMHD_MXFP4_ROWS ? rows_grid > kMaxGrid : big > kMaxGrid / 16)
    return set_error(TMHD_ERR_UNSUPPORTED, "%s: %d x %d is too large", what, m, n);
  if (f.tail || f.form == TMHD_MXFP4_256X256) {
    xa.full = (int32_t)(big - f.tail);
    hipLaunchKernelGGL(mxfp4_big_kernel, dim3((unsigned)std::min<int64_t>(xa.full, cus)), dim3(512), 0, s, xa);
  }
  switch (f.form) {
    case TMHD_MXFP4_ROWS:
      hipLaunchKernelGGL(mxfp4_rows_kernel<false>, dim3((unsigned)rows_grid), dim3(256), 0, s, xa);
      break;
    case TMHD_MXFP4_64X64:
      launch_tiles<32, 32, 4, 2>(xa, f.tail, s);
      break;
    case TMHD_MXFP4_128X64:
      launch_tiles<64, 32, 5, 1>(xa, f.tail, s);
      break;
    case TMHD_MXFP4_128X128:
      launch_tiles<64, 64, 4, 1>(xa, f.tail, s);
      break;
    case TMHD_MXFP4_128X128X2:
      launch_tiles<64, 64, 2, 2>(xa, f.tail, s);
  }
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
  if (m <= 0 || n <= 0 || k <= 0 || k % 32 || tmhd::fused_quant(m, n, k)) return 0;
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
  if (fused_quant(m, n, k)) {
    const XArgs xa = product_args(out, (const uint8_t *)x, nullptr, b, b_scale, bias, m, n, k, ldx, ldb, ldo);
    hipLaunchKernelGGL(mxfp4_rows_kernel<true>, dim3((unsigned)((n + 15) / 16)), dim3(256), 0, s, xa);
    return check_launch(what);
  }
  if (!workspace || (uintptr_t)workspace % 16 || workspace_bytes < codes_bytes(m, k) + scale_bytes(m, k))
    return set_error(TMHD_ERR_INVALID, "%s: workspace of %lld bytes", what, (long long)workspace_bytes);
  uint8_t *q = (uint8_t *)workspace, *scale = q + codes_bytes(m, k);
  if (int st = tmhd_mxfp4_quant(q, scale, x, m, k, ldx, stream)) return st;
  return launch_product(what, out, q, scale, b, b_scale, bias, m, n, k, k / 2, ldb, ldo, s);
}

extern "C" int tmhd_gemm_mxfp4_form(int32_t m, int32_t n, int32_t k, int32_t cus) {
  using namespace tmhd;
  if (m <= 0 || n <= 0 || k <= 0 || k % 32) return -1;
  return pick_form(m, n, k, cus > 0 ? cus : std::max(device_cus(), 8)).form;
}
