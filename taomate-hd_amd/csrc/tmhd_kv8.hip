// K/V slots held in 8 bits (e4m3 or int8 codes, a power-of-two scale for each 64
// tokens of a head; formats: include/tmhd_lowbit.h): the quantizing pack, the
// exact expansion to bf16 and attention that reads the codes.
#include <math.h>

#include <type_traits>

#include <algorithm>

#include "tmhd_internal.h"
#include "tmhd_lowbit.h"

namespace tmhd {
namespace {

using u16x2 = unsigned short __attribute__((ext_vector_type(2)));
using i16x2 = short __attribute__((ext_vector_type(2)));

constexpr int kBlock = 64;  // tokens of a scale
constexpr int kMaxRanges = 32, kMaxCalls = 16, kMaxSegs = 24;
constexpr int kMinByte = 10;  // 2^-117: the least code times it is a normal number

// ---- codes

// 2^(byte - 127); NaN for 255 (byte >= kMinByte)
__device__ __forceinline__ float scale_of(uint32_t byte) {
  return byte == 255u ? __uint_as_float(0x7fc00000u) : __uint_as_float(byte << 23);
}

// scale byte of a block whose largest magnitude has the bf16 bits amax: the
// least power of two with amax <= 448 (1.75 * 2^8) or 127 (1.984375 * 2^6) times it
template <bool E4M3>
__device__ __forceinline__ uint32_t scale_byte(uint32_t amax) {
  if (amax >= 0x7f80u) return 255u;
  const int e = (int)(amax >> 7), m = (int)(amax & 0x7fu);
  return (uint32_t)max(E4M3 ? e - 8 + (m > 0x60) : e - 6 + (m > 0x7e), kMinByte);
}

// Largest scale byte of finite values, and the largest magnitude (bf16 bits) that is
// encoded under it: codes from the next one on (248 and more halfway to 256 in e4m3,
// 63.5 halfway to 64 in int8) would stand for 2^128, which bf16 does not hold.
template <bool E4M3>
constexpr uint32_t kTopByte = E4M3 ? 247 : 249;
template <bool E4M3>
constexpr uint32_t kTopMagnitude = E4M3 ? 0x7f77 : 0x7f7d;

// The magnitudes of 2 bf16 brought down to kTopMagnitude
template <bool E4M3>
__device__ __forceinline__ int below_top(int w) {
  constexpr uint16_t top = kTopMagnitude<E4M3>;
  const u16x2 m = __builtin_elementwise_min(__builtin_bit_cast(u16x2, (uint32_t)w & 0x7fff7fffu), u16x2{top, top});
  return (int)(__builtin_bit_cast(uint32_t, m) | ((uint32_t)w & 0x80008000u));
}

// 8 bf16 -> 8 codes (2 words)
template <bool E4M3>
__device__ __forceinline__ i32x2 encode8(const i32x4 &v, uint32_t byte) {
  i32x2 c;
  if (byte == 255u) return i32x2{0, 0};
  if constexpr (E4M3) {
    const float s = __uint_as_float(byte << 23);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      i16x2 p = {0, 0};
      const uint32_t lo = (uint32_t)v[2 * h], hi = (uint32_t)v[2 * h + 1];
      p = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(p, __builtin_bit_cast(bf16x2, lo), s, false);
      p = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(p, __builtin_bit_cast(bf16x2, hi), s, true);
      c[h] = __builtin_bit_cast(int, p);
    }
  } else {
    const float inv = __uint_as_float((254u - byte) << 23);  // exact: the byte is 10 .. 249
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t p = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t w = (uint32_t)v[2 * h + (e >> 1)];
        const float x = bf16_bits_to_f32((e & 1) ? w >> 16 : w & 0xffffu);
        p |= ((uint32_t)(int)__builtin_rintf(x * inv) & 255u) << (8 * e);
      }
      c[h] = (int)p;
    }
  }
  return c;
}

// 4 codes -> 4 bf16 (2 words), times `scale` (a power of two or NaN)
template <bool E4M3>
__device__ __forceinline__ i32x2 decode4(uint32_t c, float scale, bool nan) {
  if constexpr (E4M3) {
    i32x2 o;
    o[0] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c, scale, false));
    o[1] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c, scale, true));
    return nan ? i32x2{0x7fc07fc0, 0x7fc07fc0} : o;
  } else {
    const float a = (float)(int8_t)c, b = (float)(int8_t)(c >> 8), d = (float)(int8_t)(c >> 16), e = (float)(int8_t)(c >> 24);
    return i32x2{(int)pack_bf16_rne(a * scale, b * scale), (int)pack_bf16_rne(d * scale, e * scale)};
  }
}

// ---- pack

struct PackArgs {
  const uint16_t *k, *v;
  int64_t ts, hs;
  uint8_t *ko, *vo, *kso, *vso;
  int32_t cap, n_ranges;
  struct {
    const int32_t *rows;
    int32_t row0, n, dst, first;  // first: of the launch's 64-token blocks
  } r[kMaxRanges];
};

// bytes of a word -> word i holds byte i of the four words
__device__ __forceinline__ void transpose4(uint32_t (&w)[4]) {
  const uint32_t a = __builtin_amdgcn_perm(w[1], w[0], 0x05010400u), b = __builtin_amdgcn_perm(w[1], w[0], 0x07030602u);
  const uint32_t c = __builtin_amdgcn_perm(w[3], w[2], 0x05010400u), d = __builtin_amdgcn_perm(w[3], w[2], 0x07030602u);
  w[0] = __builtin_amdgcn_perm(c, a, 0x05040100u);
  w[1] = __builtin_amdgcn_perm(c, a, 0x07060302u);
  w[2] = __builtin_amdgcn_perm(d, b, 0x05040100u);
  w[3] = __builtin_amdgcn_perm(d, b, 0x07060302u);
}

// Quantizing pack of one 64-token block of K or of V of one head; bound by HBM.
// 2 D threads: thread (tg, dl) holds channels 8 dl .. of tokens 4 tg .. (four
// 16-byte loads, whole rows of a head per wave), the workgroup's maximum gives
// the scale, and the codes go through LDS into the slot's chunk order, so that
// the block leaves as 64 D contiguous bytes.  4,836 tokens of 14 heads 16.5 us (3.2 TB/s
// in two short rounds), 11,232 rows picked from a sequence of 40 heads 73 to 89 (4.7 to
// 3.9 TB/s: rows of 256 bytes, 10 KiB apart).
template <int D, bool E4M3>
__global__ void __launch_bounds__(2 * D) kv8_pack_kernel(const PackArgs pa) {
  constexpr int T = 2 * D, L = D / 8;  // threads; lanes of a token row
  __shared__ uint32_t img[16 * D];
  __shared__ uint32_t part[T / 64];
  const int tid = threadIdx.x, dl = tid % L, tg = tid / L;
  const bool is_v = blockIdx.y & 1;
  const int h = blockIdx.y >> 1;
  int ri = 0;
  while (ri + 1 < pa.n_ranges && (int)blockIdx.x >= pa.r[ri + 1].first) ++ri;
  const int b = (int)blockIdx.x - pa.r[ri].first, n = pa.r[ri].n;  // block of the range; n > 64 b
  const int32_t *rows = pa.r[ri].rows;
  const uint16_t *src = (is_v ? pa.v : pa.k) + (int64_t)h * pa.hs + dl * 8;
  i32x4 v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int t = 64 * b + 4 * tg + i, tc = min(t, n - 1);
    const int64_t row = rows ? rows[tc] : pa.r[ri].row0 + tc;
    v[i] = *(const i32x4 *)(src + row * pa.ts);
    if (t >= n) v[i] = i32x4{0, 0, 0, 0};
  }
  u16x2 mx = {0, 0};
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) mx = __builtin_elementwise_max(mx, __builtin_bit_cast(u16x2, (uint32_t)v[i][e] & 0x7fff7fffu));
  int m = max((int)mx[0], (int)mx[1]);
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) m = max(m, __shfl_xor(m, off));
  if ((tid & 63) == 0) part[tid >> 6] = (uint32_t)m;
  __syncthreads();
  uint32_t amax = part[0];
#pragma unroll
  for (int i = 1; i < T / 64; ++i) amax = max(amax, part[i]);
  const uint32_t byte = scale_byte<E4M3>(amax);
  if (byte >= kTopByte<E4M3>) {  // (the same for the whole workgroup)
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) v[i][e] = below_top<E4M3>(v[i][e]);
  }
  const int64_t blk = pa.r[ri].dst / kBlock + b;  // of the slot
  if (tid == 0) (is_v ? pa.vso : pa.kso)[(int64_t)h * (pa.cap / kBlock) + blk] = (uint8_t)byte;
  i32x2 c[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) c[i] = encode8<E4M3>(v[i], byte);
  if (is_v) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      uint32_t w[4] = {(uint32_t)c[0][half], (uint32_t)c[1][half], (uint32_t)c[2][half], (uint32_t)c[3][half]};
      transpose4(w);  // word e: channel 8 dl + 4 half + e of the four tokens
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int d = 8 * dl + 4 * half + e;
        img[(tg >> 3) * (8 * D) + (d >> 5) * 256 + (tg & 1) * 128 + (d & 31) * 4 + ((tg >> 1) & 3)] = w[e];
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int t = 4 * tg + i;
      *(i32x2 *)&img[(t >> 5) * (8 * D) + (dl >> 1) * 128 + (t & 31) * 4 + (dl & 1) * 2] = c[i];
    }
  }
  __syncthreads();
  uint8_t *out = (is_v ? pa.vo : pa.ko) + ((int64_t)h * pa.cap + blk * kBlock) * D;
#pragma unroll
  for (int i = 0; i < 2; ++i) *(i32x4 *)(out + (i * T + tid) * 16) = *(const i32x4 *)&img[(i * T + tid) * 4];
}

// ---- expansion

struct View {
  const uint8_t *k, *v, *ks, *vs;  // at the view's first row
  int32_t cap, tokens, dst, first;
};
struct ExpandArgs {
  uint16_t *k, *vt;
  int64_t khs, vhs;
  int32_t vrs, n_views;
  View view[kMaxSegs];
};

// The first n of four bf16 (2 words), the others zero
__device__ __forceinline__ i32x2 first_of4(const i32x2 &v, int n) {
  auto word = [](int w, int k) { return k >= 2 ? w : k == 1 ? w & 0xffff : 0; };
  return i32x2{word(v[0], n), word(v[1], n - 2)};
}

// One 64-token block of K or V of one head into the bf16 slot format; bound by
// HBM.  K: lanes run along a token row, so that rows are written whole.  V: the
// 16 codes of a chunk are two runs of 8 consecutive positions of a transposed row.
// Rows behind the view become zero, whatever the slot holds there.  40,788 tokens of
// 14 heads of 128 89 us (4.9 TB/s).
template <int D, bool E4M3>
__global__ void __launch_bounds__(2 * D) kv8_expand_kernel(const ExpandArgs ea) {
  constexpr int T = 2 * D, C = D / 16;
  const int tid = threadIdx.x, h = blockIdx.y >> 1;
  const bool is_v = blockIdx.y & 1;
  int vi = 0;
  while (vi + 1 < ea.n_views && (int)blockIdx.x >= ea.view[vi + 1].first) ++vi;
  const View &vw = ea.view[vi];
  const int b = (int)blockIdx.x - vw.first;
  const int64_t in_at = ((int64_t)h * vw.cap + b * kBlock) * D;
  const uint32_t byte = (is_v ? vw.vs : vw.ks)[(int64_t)h * (vw.cap / kBlock) + b];
  const float s = scale_of(byte);
  const bool nan = byte == 255u;
  const int left = vw.tokens - b * kBlock;  // valid rows of the block, 64 and more for a whole one
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int c = i * T + tid;
    if (is_v) {
      const int g = c & 1, tile = (c >> 1) & 1, d = c >> 2;
      const i32x4 w = *(const i32x4 *)(vw.v + in_at + tile * (32 * D) + (d >> 5) * 1024 + g * 512 + (d & 31) * 16);
      uint16_t *o = ea.vt + (int64_t)h * ea.vhs + (int64_t)d * ea.vrs + vw.dst + b * kBlock + tile * 32 + g * 8;
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        i32x2 lo = decode4<E4M3>((uint32_t)w[2 * m], s, nan), hi = decode4<E4M3>((uint32_t)w[2 * m + 1], s, nan);
        if (left < kBlock) {  // word j of the chunk: tokens 8 j + 4 g ..
          const int keep = left - tile * 32 - 4 * g - 16 * m;
          lo = first_of4(lo, keep), hi = first_of4(hi, keep - 8);
        }
        *(i32x4 *)(o + 16 * m) = i32x4{lo[0], lo[1], hi[0], hi[1]};
      }
    } else {
      const int dc = c % C, t = c / C;
      const i32x4 w = *(const i32x4 *)(vw.k + in_at + (t >> 5) * (32 * D) + dc * 512 + (t & 31) * 16);
      uint16_t *o = ea.k + (int64_t)h * ea.khs + (int64_t)(vw.dst + b * kBlock + t) * D + dc * 16;
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        const i32x2 lo = decode4<E4M3>((uint32_t)w[2 * m], s, nan), hi = decode4<E4M3>((uint32_t)w[2 * m + 1], s, nan);
        *(i32x4 *)(o + 8 * m) = t < left ? i32x4{lo[0], lo[1], hi[0], hi[1]} : i32x4{0, 0, 0, 0};
      }
    }
  }
}

// One 64-token block of K or V of one head as token-major rows: the pack's
// thread layout run backwards; bound by HBM.  11,232 tokens of 40 heads 65 us (5.3 TB/s).
template <int D, bool E4M3>
__global__ void __launch_bounds__(2 * D) kv8_token_major_kernel(const View vw, uint16_t *__restrict__ ko,
                                                                uint16_t *__restrict__ vo, int32_t heads) {
  constexpr int L = D / 8;
  const int tid = threadIdx.x, dl = tid % L, tg = tid / L, h = blockIdx.y >> 1, b = blockIdx.x;
  const bool is_v = blockIdx.y & 1;
  const uint8_t *in = (is_v ? vw.v : vw.k) + ((int64_t)h * vw.cap + b * kBlock) * D;
  const uint32_t byte = (is_v ? vw.vs : vw.ks)[(int64_t)h * (vw.cap / kBlock) + b];
  const float s = scale_of(byte);
  uint32_t c[4][2];
  if (is_v) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      uint32_t w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int d = 8 * dl + 4 * half + e;
        w[e] = *(const uint32_t *)(in + (tg >> 3) * (32 * D) + (d >> 5) * 1024 + (tg & 1) * 512 + (d & 31) * 16 + ((tg >> 1) & 3) * 4);
      }
      transpose4(w);
#pragma unroll
      for (int i = 0; i < 4; ++i) c[i][half] = w[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int t = 4 * tg + i;
      const i32x2 w = *(const i32x2 *)(in + (t >> 5) * (32 * D) + (dl >> 1) * 512 + (t & 31) * 16 + (dl & 1) * 8);
      c[i][0] = (uint32_t)w[0], c[i][1] = (uint32_t)w[1];
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int t = b * kBlock + 4 * tg + i;
    if (t >= vw.tokens) break;
    const i32x2 lo = decode4<E4M3>(c[i][0], s, byte == 255u), hi = decode4<E4M3>(c[i][1], s, byte == 255u);
    *(i32x4 *)((is_v ? vo : ko) + ((int64_t)t * heads + h) * D + dl * 8) = i32x4{lo[0], lo[1], hi[0], hi[1]};
  }
}

// ---- attention
//
// Scores, maxima and sums are fp32.  Weights go into the second product rounded to bf16,
// the MFMA's operand type (each off by at most 2^-8; the values are bf16 numbers already),
// while their sum takes them unrounded.  Results are off by 0.0023 in the 2-norm on N(0, 1)
// keys, the rounding of the result alone by 0.0017; a second bf16 term of each weight would
// double that product's MFMAs.

struct Seg8 {
  const uint8_t *k, *v, *ks, *vs;
  int32_t cap, tokens;
};
struct Call8 {
  const uint16_t *q;
  uint16_t *o;
  int64_t qts, qhs, ots, ohs;
  const int32_t *q_rows, *o_rows;
  int32_t q_row0, o_row0, lq;
  int32_t seg0, blocks;     // its first segment, and its segments' 64-token blocks in all
  int32_t row_tiles, first;  // first: of the launch's units of work (item, block)
};
struct Args8 {
  Call8 call[kMaxCalls];
  Seg8 seg[kMaxSegs];
  int32_t n_calls, heads;
  int32_t units, wgs;  // the launch's units of work, and the workgroups they are dealt to
  int32_t whole;       // an item to a workgroup
  float scale2;        // |softmax scale| times log2 e
  int32_t flip;        // sign bits to change in Q: a negative scale's
  float *ws;
};

// The work is one item per (call, head, tile of query rows), of its call's 64-token
// blocks each; the items' blocks in a row are dealt evenly to the workgroups,
// which so all end at about the same time (short items of 32 rows go whole to one each:
// kWholeBlocks).  An item that lies in one workgroup's
// range is written out; the parts of a cut one go to ws, two slots a workgroup
// (its range may begin and end inside an item), and are merged afterwards.
__device__ __forceinline__ int range_begin(const Args8 &aa, int wg) { return (int)((int64_t)aa.units * wg / aa.wgs); }
// First unit of item `item` of the launch, all of its units for the item behind the last
__device__ __forceinline__ int item_begin(const Args8 &aa, int item) {
  int ci = 0;
  while (ci < aa.n_calls && item >= aa.heads * aa.call[ci].row_tiles) item -= aa.heads * aa.call[ci++].row_tiles;
  return ci < aa.n_calls ? aa.call[ci].first + item * aa.call[ci].blocks : aa.units;
}

// The range of a workgroup where neighbouring ranges share keys: runs on one XCD
__device__ __forceinline__ int xcd_wg(int wgs) {
  const int b = (int)blockIdx.x, xcd = b & 7, per = wgs >> 3, rem = wgs & 7;
  return (b >> 3) + xcd * per + min(xcd, rem);
}

struct Piece {
  int call, head, tile, b_begin, b_end;  // blocks of the item
  bool whole;
};
// The piece of work that starts at unit x of a range that ends at `end`
__device__ __forceinline__ Piece piece_at(const Args8 &aa, int x, int end) {
  Piece p;
  p.call = 0;
  while (p.call + 1 < aa.n_calls && x >= aa.call[p.call + 1].first) ++p.call;
  const Call8 &cl = aa.call[p.call];
  const int rel = x - cl.first, item = rel / cl.blocks;
  p.b_begin = rel - item * cl.blocks;
  p.b_end = min(cl.blocks, p.b_begin + end - x);
  p.head = item / cl.row_tiles, p.tile = item - p.head * cl.row_tiles;
  p.whole = p.b_begin == 0 && p.b_end == cl.blocks;
  return p;
}

// The segment that holds block b of a call, going on from segment si, whose first block is `first`
__device__ __forceinline__ void find_segment(const Args8 &aa, int b, int &si, int &first) {
  for (;;) {
    const int n = (aa.seg[si].tokens + kBlock - 1) / kBlock;
    if (b - first < n) return;
    first += n;
    ++si;
  }
}

// A walk over a call's blocks of one head's K or V: the block's codes, its scale byte
// and the valid tokens from its first on.  The segment's own numbers are read where a
// segment begins: read for every block, their latency is the loop's.
template <int D, bool V>
struct Walk {
  const uint8_t *p, *s;
  int left, b, si;
  __device__ __forceinline__ void enter(const Args8 &aa, int h, int at) {  // block `at` of segment si
    const Seg8 &sg = aa.seg[si];
    p = (V ? sg.v : sg.k) + ((int64_t)h * sg.cap + (int64_t)at * kBlock) * D;
    s = (V ? sg.vs : sg.ks) + (int64_t)h * (sg.cap / kBlock) + at;
    left = sg.tokens - at * kBlock;
  }
  __device__ __forceinline__ Walk(const Args8 &aa, const Call8 &cl, int h, int first) : b(first), si(cl.seg0) {
    int seg_first = 0;
    find_segment(aa, b, si, seg_first);
    enter(aa, h, b - seg_first);
  }
  __device__ __forceinline__ void next(const Args8 &aa, int h, int b_end) {  // (stays on the last one)
    if (b + 1 >= b_end) return;
    ++b;
    if (left > kBlock) {
      p += kBlock * D, ++s, left -= kBlock;
    } else {
      ++si;
      enter(aa, h, 0);
    }
  }
};

// floats of a partial result: ROWS of D sums, then the references and the weights' sums
template <int D, int ROWS>
constexpr int part_floats() { return ROWS * (D + 2); }

// Q operands of 32 rows from row r0 on, PERM: in the channel order of the K chunks
template <int D, bool PERM>
__device__ __forceinline__ void load_q(const Args8 &aa, const Call8 &cl, int head, int r0, int lr, int g, bf16x8 (&qf)[D / 16]) {
  const int r = min(r0 + lr, cl.lq - 1);
  const int64_t row = cl.q_rows ? cl.q_rows[r] : cl.q_row0 + r;
  const uint16_t *qp = cl.q + row * cl.qts + (int64_t)head * cl.qhs;
#pragma unroll
  for (int t = 0; t < D / 16; ++t) {
    i32x4 v = *(const i32x4 *)(qp + (PERM ? 32 * (t >> 1) + 16 * g + 8 * (t & 1) : 16 * t + 8 * g));
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] ^= aa.flip;
    qf[t] = __builtin_bit_cast(bf16x8, v);
  }
}

__device__ __forceinline__ i32x2 pack4(const f32x4 &v, float f) {
  return i32x2{(int)pack_bf16_rne(v[0] * f, v[1] * f), (int)pack_bf16_rne(v[2] * f, v[3] * f)};
}

// The number of valid keys, as only a branch that few tiles take sees it: the
// compiler may not run the branch's instructions (two per score) for every tile.
__device__ __forceinline__ int in_branch(int keys) {
  asm volatile("" : "+s"(keys));
  return keys;
}

// A row's reference before its first score: a number, so that scores of -inf (sums that
// overflowed) weigh 2^(-inf - kLeast) = 0 and not NaN
constexpr float kLeast = -3.402823466e38f;

// A score times the scale, rounded, less the reference, which is the largest such
// product: what one rounding less (a fused multiply-add) leaves of the largest itself
// is up to 2^-24 of it, and of products beyond 2^31 its power of two is infinite.
__device__ __forceinline__ float below(float s, float scale, float reference) {
#pragma clang fp contract(off)
  return s * scale - reference;
}
// References up to which the fused form does (2^28: off by at most 2^4)
constexpr float kFused = 268435456.f;

// 32 query rows an item.  The W waves of a workgroup take an item's blocks in
// turn and merge through LDS.  Per 32 keys a lane loads the 16-byte
// chunks that are its MFMA operands (no LDS on the way: each code is used once)
// and turns them into bf16, exactly; S^T = K Q^T leaves 16 keys of one query in a
// lane, in the order in which the V chunks hold them, so P feeds the second
// product from registers.  A block's K scale joins the softmax scale, its V scale
// the conversion (e4m3) or P (int8).  Bound by HBM over a long cache: two waves a SIMD
// keep two tiles each in flight.  One row of 14 heads of 128 over 40,788 tokens, e4m3: 26
// to 28 us (5.2 to 5.6 TB/s), 36 with the merge and the launches.
template <int D, int W, bool E4M3>
__global__ void __launch_bounds__(W * 64) __attribute__((amdgpu_waves_per_eu(2, 2))) kv8_rows_kernel(const Args8 aa) {
  constexpr int KC = D / 32;  // 16-byte K chunks of a lane per 32 keys, and V chunks (32-channel blocks)
  constexpr int RS = D + 4;   // floats of a staged row
  __shared__ __attribute__((aligned(16))) float stage[W * 32 * RS];
  __shared__ float stat[2][W][32];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lr = lane & 31, g = lane >> 5;
  const int x0 = aa.whole ? item_begin(aa, blockIdx.x) : range_begin(aa, blockIdx.x);
  const int end = aa.whole ? item_begin(aa, blockIdx.x + 1) : range_begin(aa, blockIdx.x + 1);
  for (int x = x0; x < end;) {
    const Piece pc = piece_at(aa, x, end);
    const Call8 &cl = aa.call[pc.call];
    const int h = pc.head, r0 = pc.tile * 32;
    if (x != x0) __syncthreads();  // the staging area is read out
    bf16x8 qf[2 * KC];
    load_q<D, true>(aa, cl, h, r0, lr, g, qf);
    f32x16 acc[KC];
    float mx = kLeast, sum = 0.f;
#pragma unroll
    for (int d = 0; d < KC; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[d][i] = 0.f;

    // The wave's tiles of 32 keys, in order: where the next one's chunks lie, the
    // scale bytes of its block, its valid keys.  The next tile's K and V chunks are
    // loaded as soon as the current ones are operands.
    int si = cl.seg0, s_first = 0, b = pc.b_begin + w, t = 0;
    const uint8_t *kp = nullptr, *vp = nullptr;
    // (scale bytes as loaded: turning them into factors here would wait for every load in flight)
    uint32_t kb = 0, vb = 0;
    int left = 0;
    auto locate = [&]() {  // block b of the call, tile 0
      find_segment(aa, b, si, s_first);
      const Seg8 &sg = aa.seg[si];
      const int sb = b - s_first;
      const int64_t off = ((int64_t)h * sg.cap + (int64_t)sb * kBlock) * D, s_at = (int64_t)h * (sg.cap / kBlock) + sb;
      kp = sg.k + off + lane * 16, vp = sg.v + off + lane * 16;
      left = sg.tokens - sb * kBlock;  // 1 or more
      kb = sg.ks[s_at], vb = sg.vs[s_at];
      t = 0;
    };
    i32x4 kr[KC], vr[KC];
    if (b < pc.b_end) {
      locate();
#pragma unroll
      for (int j = 0; j < KC; ++j) kr[j] = *(const i32x4 *)(kp + j * 1024);
#pragma unroll
      for (int j = 0; j < KC; ++j) vr[j] = *(const i32x4 *)(vp + j * 1024);
    }
    while (b < pc.b_end) {
      const int here = left;  // valid keys from the tile's first
      const uint32_t kb_now = kb, vb_now = vb;
      // the next tile: the block's second, or the first of the wave's next block
      if (t == 0 && left > 32) {
        t = 1, left -= 32, kp += 32 * D, vp += 32 * D;
      } else {
        b += W;
        if (b < pc.b_end) locate();
      }
      f32x16 s;
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] = 0.f;
      auto operand = [](const i32x4 &raw, int half, float scale) {
        const i32x2 lo = decode4<E4M3>((uint32_t)raw[2 * half], scale, false);
        const i32x2 hi = decode4<E4M3>((uint32_t)raw[2 * half + 1], scale, false);
        return __builtin_bit_cast(bf16x8, i32x4{lo[0], lo[1], hi[0], hi[1]});
      };
#pragma unroll
      for (int j = 0; j < 2 * KC; ++j)
        s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(operand(kr[j >> 1], j & 1, 1.0f), qf[j], s, 0, 0, 0);
      const float kc = scale_of(kb_now) * aa.scale2, vc = scale_of(vb_now);
      // (after the last tile: its own chunks again)
#pragma unroll
      for (int j = 0; j < KC; ++j) kr[j] = *(const i32x4 *)(kp + j * 1024);
      if (here < 32) {
        const int keys = in_branch(here) - 4 * g;  // keys past the last: out of the maximum, weight 0 below
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (8 * (i >> 2) + (i & 3) >= keys) s[i] = -3.4e38f;
      }
      float top = fmaxf(s[0], s[1]);
#pragma unroll
      for (int i = 2; i < 16; i += 2) top = fmaxf(fmaxf(top, s[i]), s[i + 1]);
      top *= kc;
      // the reference moves only where a score passes it by 8 (weights up to 2^8); a row's
      // two lanes have half of its scores each
      if (__any(top > mx + 8.0f)) {
        const float m = fmaxf(mx, fmaxf(top, __shfl_xor(top, 32)));
        const float f = m == mx ? 1.0f : __builtin_amdgcn_exp2f(mx - m);
        mx = m;
        sum *= f;
#pragma unroll
        for (int d = 0; d < KC; ++d)
#pragma unroll
          for (int i = 0; i < 16; ++i) acc[d][i] *= f;
      }
      float p[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) p[i] = __builtin_amdgcn_exp2f(below(s[i], kc, mx));
      if (here < 32) {
        const int keys = in_branch(here) - 4 * g;
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (8 * (i >> 2) + (i & 3) >= keys) p[i] = 0.f;
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) sum += p[i];
      bf16x8 pf[2];
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        i32x4 pk;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          pk[e] = E4M3 ? (int)pack_bf16_rne(p[8 * m + 2 * e], p[8 * m + 2 * e + 1])
                       : (int)pack_bf16_rne(p[8 * m + 2 * e] * vc, p[8 * m + 2 * e + 1] * vc);
        pf[m] = __builtin_bit_cast(bf16x8, pk);
      }
#pragma unroll
      for (int d = 0; d < KC; ++d)
#pragma unroll
        for (int m = 0; m < 2; ++m)
          acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(operand(vr[d], m, E4M3 ? vc : 1.0f), pf[m], acc[d], 0, 0, 0);
      if (E4M3 && vc != vc) sum = vc;  // (the conversion's scale operand has no NaN)
#pragma unroll
      for (int j = 0; j < KC; ++j) vr[j] = *(const i32x4 *)(vp + j * 1024);
    }

    // merge of the waves, in their order
    const float l = sum + __shfl_xor(sum, 32);
    if (g == 0) stat[0][w][lr] = mx, stat[1][w][lr] = l;
#pragma unroll
    for (int d = 0; d < KC; ++d)
#pragma unroll
      for (int u = 0; u < 4; ++u)
        *(f32x4 *)&stage[(w * 32 + lr) * RS + d * 32 + 8 * u + 4 * g] =
            f32x4{acc[d][4 * u], acc[d][4 * u + 1], acc[d][4 * u + 2], acc[d][4 * u + 3]};
    __syncthreads();
    // thread: row tid / 2 W, channels 4 (tid % 2 W) + 8 W j ..
    const int r = threadIdx.x / (2 * W), dq = threadIdx.x % (2 * W), row = r0 + r;
    if (row < cl.lq) {
      float m = stat[0][0][r], f[W], ls = 0.f;
#pragma unroll
      for (int i = 1; i < W; ++i) m = fmaxf(m, stat[0][i][r]);
#pragma unroll
      for (int i = 0; i < W; ++i) {
        // a wave without blocks has the reference kLeast and sums 0
        f[i] = stat[0][i][r] == m ? 1.0f : __builtin_amdgcn_exp2f(stat[0][i][r] - m);
        ls += f[i] * stat[1][i][r];
      }
      float *ws = aa.ws + (int64_t)(2 * blockIdx.x + (x != x0)) * part_floats<D, 32>();
      const float inv = 1.0f / ls;
      uint16_t *op = nullptr;
      if (pc.whole) {
        const int64_t orow = cl.o_rows ? cl.o_rows[row] : cl.o_row0 + row;
        op = cl.o + orow * cl.ots + (int64_t)h * cl.ohs;
      } else if (dq == 0) {
        ws[32 * D + r] = m;
        ws[32 * (D + 1) + r] = ls;
      }
#pragma unroll
      for (int j = 0; j < D / (8 * W); ++j) {
        const int d = 8 * W * j + 4 * dq;
        f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < W; ++i) v += f[i] * *(const f32x4 *)&stage[(i * 32 + r) * RS + d];
        if (op)
          *(i32x2 *)(op + d) = pack4(v, inv);
        else
          *(f32x4 *)&ws[r * D + d] = v;
      }
    }
    x += pc.b_end - pc.b_begin;
  }
}

// 128 query rows an item: four waves of 32 rows, two workgroups a CU.  A block of 64
// tokens is turned into bf16 once, its scales included (exact), by all threads,
// into MFMA operand order in LDS (chunks of 16 bytes, a wave's read 1 KiB in a row);
// then every wave multiplies its rows with it.  Two buffers: while block b is
// multiplied, block b + 1 (in registers since the block before) is converted and
// block b + 2 loaded; one barrier a block.  14 heads of 128 over 40,788 tokens, e4m3: 64
// rows 53 to 57 us (2.6 TB/s), 128 rows 66 to 76 (490 TFLOPS); 40 heads, 91 rows over
// 11,232 tokens, int8: 52 to 57 (the lower figures of a faster card).  Bound by a block's
// steps that follow each other, which the CU's other workgroup only half fills: of the
// last 57 us, 20 go without the products and the softmax, 10 without the conversion, 7
// without the loads, 4 without the barrier.
template <int D, bool E4M3>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2))) kv8_tile_kernel(const Args8 aa) {
  constexpr int KC = D / 32, T = 256, ROWS = 128;
  constexpr int HALF = kBlock * D * 2;             // bytes of a block's K (or V) in bf16
  constexpr int CH = kBlock * D / 8 / T;           // 16-byte chunks of codes a thread converts, of K then of V
  constexpr int KCH = kBlock * D / 16;             // chunks of K
  static_assert(CH >= 1 && CH * T * 8 == kBlock * D, "the threads share a block's chunks");
  __shared__ __attribute__((aligned(1024))) char smem[2 * 2 * HALF];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), lr = lane & 31, g = lane >> 5;
  const int x0 = range_begin(aa, xcd_wg(aa.wgs)), end = range_begin(aa, xcd_wg(aa.wgs) + 1);
  for (int x = x0; x < end;) {
    const Piece pc = piece_at(aa, x, end);
    const Call8 &cl = aa.call[pc.call];
    const int h = pc.head, r0 = pc.tile * ROWS + 32 * w;
    const bool live = r0 < cl.lq;  // a wave without rows only converts
    bf16x8 qf[2 * KC];
    load_q<D, false>(aa, cl, h, r0, lr, g, qf);
    f32x16 acc[KC];
    float mx = kLeast, sum = 0.f;
    bool large = false;  // references beyond kFused: the scores are brought below them one by one
#pragma unroll
    for (int d = 0; d < KC; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[d][i] = 0.f;

    // the block that is loaded next (the last one again behind it)
    Walk<D, false> kw(aa, cl, h, pc.b_begin);
    Walk<D, true> vw(aa, cl, h, pc.b_begin);
    i32x4 raw[CH];
    uint32_t kb = 0, vb = 0;
    int raw_left = 0;  // valid keys from its first on
    auto load = [&]() {
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        const int c = i * T + tid;
        raw[i] = *(const i32x4 *)((c < KCH ? kw.p : vw.p - KCH * 16) + c * 16);
      }
      kb = *kw.s, vb = *vw.s;
      raw_left = kw.left;
      kw.next(aa, h, pc.b_end);
      vw.next(aa, h, pc.b_end);
    };
    // K chunk (tile, 16 channels, key): two chunks of 8 channels, 512 bytes apart; V
    // chunk (tile, 32 channels, key group, channel): two of 8 keys, 1 KiB apart
    // A block without finite values makes every output NaN: by way of `poison`, not of its values.
    float poison = 0.f;
    auto convert = [&](int buf) {
      const float fk = scale_of(kb), fv = scale_of(vb);
      poison += fk + fv == fk + fv ? 0.f : fk + fv;
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        const int c = i * T + tid;
        const bool is_v = c >= KCH;
        asm volatile("" : "+v"(raw[i]));  // (converted here, not where it was loaded: four times the registers)
        const float f = is_v ? fv : fk;
        i32x4 o[2];
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          const i32x2 lo = decode4<E4M3>((uint32_t)raw[i][2 * m], f, false), hi = decode4<E4M3>((uint32_t)raw[i][2 * m + 1], f, false);
          o[m] = i32x4{lo[0], lo[1], hi[0], hi[1]};
        }
        const int cc = is_v ? c - KCH : c;
        // K: [tile][D / 8][32 keys]; V: [tile][D / 32][2][2 groups][32 channels]
        const int at = is_v ? HALF + (cc >> 6) * 2048 + (cc & 63) * 16 : (cc >> 5) * 1024 + (cc & 31) * 16;
        char *to = smem + buf * 2 * HALF + at;
        *(i32x4 *)to = o[0];
        *(i32x4 *)(to + (is_v ? 1024 : 512)) = o[1];
        __builtin_amdgcn_sched_barrier(0);  // (a chunk's registers at a time)
      }
    };
    if (x != x0) __syncthreads();  // the last piece's buffers are read out
    load();
    int left = raw_left;  // valid keys from block b's first on
    convert(0);
    load();
    const int blocks = pc.b_end - pc.b_begin;
    for (int b = 0; b < blocks; ++b) {
      const int buf = b & 1, next_left = raw_left;
      __syncthreads();
      if (live) {
        // operands half a block ahead of their MFMAs: K's first half behind the
        // barrier, V's behind the scores, so that it lands under the softmax
        const char *kt = smem + buf * 2 * HALF + lane * 16, *vt = kt + HALF;
        bf16x8 op[2 * KC];
        auto k_op = [&](int i) { return *(const bf16x8 *)(kt + (i & 1) * (HALF / 2) + (i >> 1) * 1024); };
        auto v_op = [&](int i) { return *(const bf16x8 *)(vt + i / (2 * KC) * (HALF / 2) + i / KC % 2 * 1024 + i % KC * 2048); };
#pragma unroll
        for (int i = 0; i < 2 * KC; ++i) op[i] = k_op(i);
        __builtin_amdgcn_sched_barrier(0);
        const f32x16 zero = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        f32x16 s[2];
#pragma unroll
        for (int i = 0; i < 4 * KC; ++i) {
          s[i & 1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(op[i % (2 * KC)], qf[i >> 1], i < 2 ? zero : s[i & 1], 0, 0, 0);
          op[i % (2 * KC)] = i < 2 * KC ? k_op(i + 2 * KC) : v_op(i - 2 * KC);
          __builtin_amdgcn_sched_barrier(0);
        }
        if (left < kBlock) {
          const int keys = in_branch(left) - 4 * g;
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i)
              if (32 * t + 8 * (i >> 2) + (i & 3) >= keys) s[t][i] = -3.4e38f;
        }
        float top = fmaxf(s[0][0], s[1][0]);
#pragma unroll
        for (int i = 1; i < 16; ++i) top = fmaxf(fmaxf(top, s[0][i]), s[1][i]);
        top *= aa.scale2;
        // (as in kv8_rows_kernel)
        if (__any(top > mx + 8.0f)) {
          const float m = fmaxf(mx, fmaxf(top, __shfl_xor(top, 32)));
          const float f = m == mx ? 1.0f : __builtin_amdgcn_exp2f(mx - m);
          mx = m;
          sum *= f;
#pragma unroll
          for (int d = 0; d < KC; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[d][i] *= f;
          large = __any(fabsf(mx) > kFused);
        }
        float mul = aa.scale2, ref = mx;
        if (large) {
          mul = 1.0f, ref = 0.f;
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) s[t][i] = below(s[t][i], aa.scale2, mx);
        }
        bf16x8 pf[2][2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          float p[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) p[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][i], mul, -ref));
          if (left < kBlock) {
            const int keys = in_branch(left) - 4 * g;
#pragma unroll
            for (int i = 0; i < 16; ++i)
              if (32 * t + 8 * (i >> 2) + (i & 3) >= keys) p[i] = 0.f;
          }
#pragma unroll
          for (int i = 0; i < 16; ++i) sum += p[i];
#pragma unroll
          for (int m = 0; m < 2; ++m) {
            i32x4 pk;
#pragma unroll
            for (int e = 0; e < 4; ++e) pk[e] = (int)pack_bf16_rne(p[8 * m + 2 * e], p[8 * m + 2 * e + 1]);
            pf[t][m] = __builtin_bit_cast(bf16x8, pk);
          }
        }
#pragma unroll
        for (int i = 0; i < 4 * KC; ++i) {
          acc[i % KC] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(op[i % (2 * KC)], pf[i / (2 * KC)][i / KC % 2], acc[i % KC], 0, 0, 0);
          if (i < 2 * KC) op[i % (2 * KC)] = v_op(i + 2 * KC);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      // (the last MFMAs run meanwhile, and the scores' registers are free)
      if (b + 1 < blocks) {
        convert(buf ^ 1);
        load();
      }
      left = next_left;
    }

    const float l = sum + __shfl_xor(sum, 32) + poison;
    const int row = r0 + lr;
    if (row < cl.lq) {
      if (pc.whole) {
        const int64_t orow = cl.o_rows ? cl.o_rows[row] : cl.o_row0 + row;
        uint16_t *op = cl.o + orow * cl.ots + (int64_t)h * cl.ohs + 4 * g;
        const float inv = 1.0f / l;
#pragma unroll
        for (int d = 0; d < KC; ++d)
#pragma unroll
          for (int u = 0; u < 4; ++u)
            *(i32x2 *)(op + 32 * d + 8 * u) = pack4(f32x4{acc[d][4 * u], acc[d][4 * u + 1], acc[d][4 * u + 2], acc[d][4 * u + 3]}, inv);
      } else {
        const int r = 32 * w + lr;
        float *ws = aa.ws + (int64_t)(2 * xcd_wg(aa.wgs) + (x != x0)) * part_floats<D, ROWS>();
        if (g == 0) ws[ROWS * D + r] = mx, ws[ROWS * (D + 1) + r] = l;
#pragma unroll
        for (int d = 0; d < KC; ++d)
#pragma unroll
          for (int u = 0; u < 4; ++u)
            *(f32x4 *)&ws[r * D + 32 * d + 8 * u + 4 * g] =
                f32x4{acc[d][4 * u], acc[d][4 * u + 1], acc[d][4 * u + 2], acc[d][4 * u + 3]};
      }
    }
    x += blocks;
  }
}

// MFMAs of kv8_wide_kernel: volatile asm, so that they stay where the source has them
// (the compiler gathers the vector work between builtins into one place) and the sums
// and Q stay in AGPRs.  The compiler does not see the hazards: a weight that a vector
// instruction wrote goes through two wait states (FRESH), results through settle().
template <bool FIRST>
__device__ __forceinline__ void mfma_scores(f32x16 &s, const bf16x8 &k, const bf16x8 &q) {
  if constexpr (FIRST)
    asm volatile("v_mfma_f32_32x32x16_bf16 %0, %1, %2, 0" : "=&v"(s) : "v"(k), "a"(q));
  else
    asm volatile("v_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+v"(s) : "v"(k), "a"(q));
}
template <bool FRESH>
__device__ __forceinline__ void mfma_output(f32x16 &o, const bf16x8 &v, const bf16x8 &p) {
  if constexpr (FRESH)
    asm volatile("s_nop 1\n\tv_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+a"(o) : "v"(v), "v"(p));
  else
    asm volatile("v_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+a"(o) : "v"(v), "v"(p));
}
// An MFMA of 8 passes wrote the scores: 11 wait states and more before they are read
__device__ __forceinline__ void settle(f32x16 (&s)[2]) { asm volatile("s_nop 15" : "+v"(s[0]), "+v"(s[1])); }
template <int KC>
__device__ __forceinline__ void settle(f32x16 (&o)[2][KC]) {  // (and after vector writes to them)
#pragma unroll
  for (int d = 0; d < KC; ++d) asm volatile("s_nop 7" : "+a"(o[0][d]), "+a"(o[1][d]));
}

// 256 query rows an item, two blocks of 32 rows for each of four waves, one wave a
// SIMD: an operand read from LDS serves two MFMAs.  Codes become bf16 in LDS as in
// kv8_tile_kernel.  A wave goes through tiles of 32 keys: while the scores of the next
// tile are multiplied, the weights of this one are computed, a pair in front of two MFMAs
// of three; then this tile's outputs, with the last weights, the next tile's maximum
// and the conversion of block b + 2's K or block b + 1's V (loaded an iteration before)
// in front of the MFMAs.  K in three buffers, V in two, one barrier for 64 keys.
// 14 heads of 128 over 40,788 tokens, e4m3 (int8): 256 rows 97 to 102 us (104 to 108),
// 1,024 rows 284 to 305 (308 to 332; 983 TFLOPS), 4,836 rows 1,283 to 1,383 (1,380 to
// 1,479), the lower figures of a faster card.  Bound by issue: MFMAs busy 48% of the
// time, instructions issuing 59%; without the conversion (16 cycles for two values) 13%
// less time, without the exponentials 9%, without the barrier 3%.  Eight waves of 32 rows
// took 104, 339 and 1,356 us (int8 108, 353, 1,459) and read LDS for as long as they
// multiplied; with segment numbers read for every block this one took 1,467 us.
template <int D, bool E4M3>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(1, 1))) kv8_wide_kernel(const Args8 aa) {
  constexpr int KC = D / 32, T = 256, ROWS = 256;
  constexpr int HALF = kBlock * D * 2;    // bytes of a block's K (or V) in bf16
  constexpr int CH = kBlock * D / 8 / T;  // 16-byte chunks of codes a thread converts: the first half K, then V
  constexpr int NQ = 2 * KC, NS = 4 * KC, LA = 4;  // slots of a 32-key tile: scores, then outputs; operands read ahead
  __shared__ __attribute__((aligned(1024))) char smem[5 * HALF];  // three of K, two of V
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), lr = lane & 31, g = lane >> 5;
  const int x0 = range_begin(aa, xcd_wg(aa.wgs)), end = range_begin(aa, xcd_wg(aa.wgs) + 1);
  // (-inf, a masked score, times it stays -inf)
  const float scale2 = aa.scale2 == 0.f ? __uint_as_float(1u) : aa.scale2;
  for (int x = x0; x < end;) {
    const Piece pc = piece_at(aa, x, end);
    const Call8 &cl = aa.call[pc.call];
    const int h = pc.head, r0 = pc.tile * ROWS + 64 * w, blocks = pc.b_end - pc.b_begin;
    bf16x8 qf[2][NQ];
    load_q<D, false>(aa, cl, h, r0, lr, g, qf[0]);
    load_q<D, false>(aa, cl, h, r0 + 32, lr, g, qf[1]);
#pragma unroll
    for (int i = 0; i < NQ; ++i) asm volatile("" : "+a"(qf[0][i]), "+a"(qf[1][i]));
    f32x16 acc[2][KC];
    float mx[2] = {kLeast, kLeast}, sum[2] = {0.f, 0.f};
    float mul = scale2, ref[2] = {kLeast, kLeast};  // (as in kv8_tile_kernel)
    bool large = false;
#pragma unroll
    for (int d = 0; d < KC; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[0][d][i] = acc[1][d][i] = 0.f;

    // the blocks whose K and whose V codes are loaded next (the last one again behind it)
    Walk<D, false> kw(aa, cl, h, pc.b_begin);
    Walk<D, true> vw(aa, cl, h, pc.b_begin);
    i32x4 raw[CH];
    uint32_t byte[2];
    int raw_left = 0;  // valid keys from the first of the K block in raw on
    auto load_k = [&]() {
#pragma unroll
      for (int i = 0; i < CH / 2; ++i) raw[i] = *(const i32x4 *)(kw.p + (i * T + tid) * 16);
      byte[0] = *kw.s;
      raw_left = kw.left;
      kw.next(aa, h, pc.b_end);
    };
    auto load_v = [&]() {
#pragma unroll
      for (int i = 0; i < CH / 2; ++i) raw[CH / 2 + i] = *(const i32x4 *)(vw.p + (i * T + tid) * 16);
      byte[1] = *vw.s;
      vw.next(aa, h, pc.b_end);
    };
    // Half m of chunk i.  A block without finite values makes every output NaN: by way of
    // `poison`, not of its values.
    float poison = 0.f;
    auto convert = [&](int i, int m, char *to) {
      const bool v = i >= CH / 2;
      int w0 = raw[i][2 * m], w1 = raw[i][2 * m + 1];
      asm volatile("" : "+v"(w0), "+v"(w1));  // (converted here, not where it was loaded: four times the registers)
      const float f = scale_of(byte[v]);
      if (m == 0) poison += f == f ? 0.f : f;
      const int c = (v ? i - CH / 2 : i) * T + tid;
      const i32x2 lo = decode4<E4M3>((uint32_t)w0, f, false), hi = decode4<E4M3>((uint32_t)w1, f, false);
      *(i32x4 *)(to + (v ? (c >> 6) * 2048 + (c & 63) * 16 + m * 1024 : (c >> 5) * 1024 + (c & 31) * 16 + m * 512)) =
          i32x4{lo[0], lo[1], hi[0], hi[1]};
    };
    auto mask = [&](f32x16 (&sc)[2], int left) {  // keys of a 32-key tile from `left` on
      const int keys = in_branch(left) - 4 * g;
#pragma unroll
      for (int rb = 0; rb < 2; ++rb)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (8 * (i >> 2) + (i & 3) >= keys) sc[rb][i] = -__builtin_inff();
    };
    auto largest = [&](const f32x16 &sc) {
      float m = sc[0];
#pragma unroll
      for (int i = 1; i < 16; ++i) m = fmaxf(m, sc[i]);
      return m;
    };
    auto move = [&](float (&top)[2], f32x16 (&sc)[2]) {  // (as in kv8_rows_kernel; sc: the scores)
      top[0] *= scale2, top[1] *= scale2;
      if (__any(top[0] > mx[0] + 8.0f || top[1] > mx[1] + 8.0f)) {
        settle<KC>(acc);
#pragma unroll
        for (int rb = 0; rb < 2; ++rb) {
          const float m = fmaxf(mx[rb], fmaxf(top[rb], __shfl_xor(top[rb], 32)));
          const float f = m == mx[rb] ? 1.0f : __builtin_amdgcn_exp2f(mx[rb] - m);
          mx[rb] = m;
          sum[rb] *= f;
#pragma unroll
          for (int d = 0; d < KC; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[rb][d][i] *= f;
        }
        settle<KC>(acc);
        large = __any(fabsf(mx[0]) > kFused || fabsf(mx[1]) > kFused);
        mul = large ? 1.0f : scale2;
        ref[0] = large ? 0.f : mx[0], ref[1] = large ? 0.f : mx[1];
      }
      if (large) {
#pragma unroll
        for (int rb = 0; rb < 2; ++rb)
#pragma unroll
          for (int i = 0; i < 16; ++i) sc[rb][i] = below(sc[rb][i], scale2, mx[rb]);
      }
    };

    bf16x8 op[NS + LA];
    // Slot i of a 32-key tile: operand op[i] times both row blocks.  i < NQ: the scores
    // of the next tile (kt: its keys), else this tile's weights times V (vt)
    auto read_op = [&](int i, const char *kt, const char *vt) {
      return i < NQ ? *(const bf16x8 *)(kt + i * 1024) : *(const bf16x8 *)(vt + (i - NQ) / KC * 1024 + (i - NQ) % KC * 2048);
    };
    // One tile: sc its scores, nx the next tile's (left: its valid keys); chunks c0 .. of
    // the codes in raw are converted
    auto tile = [&](f32x16 (&sc)[2], f32x16 (&nx)[2], const char *kt, const char *vt, const char *kt_next, int left, int c0,
                    char *k_to, char *v_to) {
      i32x4 pf[2][2];  // weights: [row block][16 keys]
      float pe[16][2], top[2];
      // Where the pairs of weights are computed (in the order in which the outputs' MFMAs
      // need them): the exponentials, and one MFMA later the rest
      auto pair_at = [](int u) { return u < 11 ? u * 2 * NQ / 11 : 2 * NQ + (u - 11) * 2 * KC / 5; };
#pragma clang loop unroll(full)
      for (int r = 0; r < 2 * NS; ++r) {  // what goes in front of MFMA r
        const int i = r >> 1, rb = r & 1;
        if (rb == 1) op[i + LA] = i + LA < NS ? read_op(i + LA, kt, vt) : read_op(i + LA - NS, kt_next, vt);
#pragma unroll
        for (int u = 0; u < 16; ++u) {
          const int st = u >> 3, b = (u >> 2) & 1, q = u & 3;
          if (pair_at(u) == r) {
            pe[u][0] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[b][8 * st + 2 * q], mul, -ref[b]));
            pe[u][1] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[b][8 * st + 2 * q + 1], mul, -ref[b]));
            asm volatile("" : "+v"(pe[u][0]), "+v"(pe[u][1]));
          }
          if (pair_at(u) + 1 == r) {
            int pk = (int)pack_bf16_rne(pe[u][0], pe[u][1]);
            sum[b] += pe[u][0];
            sum[b] += pe[u][1];
            asm volatile("" : "+v"(pk), "+v"(sum[b]));
            pf[b][st][q] = pk;
          }
        }
        if (r == 2 * NQ + 2) settle(nx);
#pragma unroll
        for (int u = 0; u < 8; ++u)
          if (r == 2 * NQ + 2 + u * (2 * NQ - 2) / 8) {
#pragma unroll
            for (int b = 0; b < 2; ++b) {
              const float m = fmaxf(nx[b][2 * u], nx[b][2 * u + 1]);
              top[b] = u ? fmaxf(top[b], m) : m;
              asm volatile("" : "+v"(top[b]));
            }
          }
#pragma unroll
        for (int c = 0; c < CH; ++c)
          if (r == 2 * NQ + 2 * KC + c * 2 * KC / CH) convert(c0 + (c >> 1), c & 1, c0 ? v_to : k_to);
        __builtin_amdgcn_sched_barrier(0);
        if (i == 0)
          mfma_scores<true>(nx[rb], op[i], qf[rb][i]);
        else if (i < NQ)
          mfma_scores<false>(nx[rb], op[i], qf[rb][i]);
        else if (i == NQ || i == NQ + KC)
          mfma_output<true>(acc[rb][0], op[i], __builtin_bit_cast(bf16x8, pf[rb][(i - NQ) / KC]));
        else
          mfma_output<false>(acc[rb][(i - NQ) % KC], op[i], __builtin_bit_cast(bf16x8, pf[rb][(i - NQ) / KC]));
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int i = 0; i < LA; ++i) op[i] = op[NS + i];
      if (left < 32) {
        mask(nx, left);
        top[0] = largest(nx[0]), top[1] = largest(nx[1]);
      }
      move(top, nx);
    };

    // K of blocks 0 and 1, V of block 0; the codes of block 2's K and block 1's V
    if (x != x0) __syncthreads();  // the last piece's buffers are read out
    char *const vb0 = smem + 3 * HALF;
    load_k();
    load_v();
    int left0 = raw_left;  // valid keys from block b's first on, and from block b + 1's
#pragma unroll
    for (int i = 0; i < 2 * CH; ++i) convert(i >> 1, i & 1, i < CH ? smem : vb0);
    load_k();
    int left1 = raw_left;
#pragma unroll
    for (int i = 0; i < CH; ++i) convert(i >> 1, i & 1, smem + HALF);
    load_k();
    load_v();
    __syncthreads();
    f32x16 sa[2], sb[2];
    const char *const mine = smem + lane * 16;
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
      const bf16x8 o = read_op(i, mine, mine);
#pragma unroll
      for (int rb = 0; rb < 2; ++rb) {
        if (i)
          mfma_scores<false>(sa[rb], o, qf[rb][i]);
        else
          mfma_scores<true>(sa[rb], o, qf[rb][i]);
      }
    }
    settle(sa);
    if (left0 < 32) mask(sa, left0);
    {
      float top[2] = {largest(sa[0]), largest(sa[1])};
      move(top, sa);
    }
    int k0 = 0, k1 = HALF, k2 = 2 * HALF;  // the K buffers of blocks b, b + 1, b + 2
#pragma unroll
    for (int i = 0; i < LA; ++i) op[i] = read_op(i, mine + HALF / 2, mine);
    for (int b = 0; b < blocks; ++b) {
      const char *vt = mine + (3 + (b & 1)) * HALF;
      char *v_to = vb0 + ((b & 1) ^ 1) * HALF;
      if (b) __syncthreads();
      tile(sa, sb, mine + k0 + HALF / 2, vt, mine + k1, left0 - 32, 0, smem + k2, v_to);
      const int left2 = raw_left;
      load_k();  // (a whole iteration ahead of its conversion, as V's)
      tile(sb, sa, mine + k1, vt + HALF / 2, mine + k1 + HALF / 2, left1, CH / 2, smem + k2, v_to);
      load_v();
      left0 = left1, left1 = left2;
      const int t = k0;
      k0 = k1, k1 = k2, k2 = t;
    }

    settle<KC>(acc);
#pragma unroll
    for (int rb = 0; rb < 2; ++rb) {
      const float l = sum[rb] + __shfl_xor(sum[rb], 32) + poison;
      const int row = r0 + 32 * rb + lr;
      if (row < cl.lq) {
        if (pc.whole) {
          const int64_t orow = cl.o_rows ? cl.o_rows[row] : cl.o_row0 + row;
          uint16_t *o = cl.o + orow * cl.ots + (int64_t)h * cl.ohs + 4 * g;
          const float inv = 1.0f / l;
#pragma unroll
          for (int d = 0; d < KC; ++d)
#pragma unroll
            for (int u = 0; u < 4; ++u)
              *(i32x2 *)(o + 32 * d + 8 * u) =
                  pack4(f32x4{acc[rb][d][4 * u], acc[rb][d][4 * u + 1], acc[rb][d][4 * u + 2], acc[rb][d][4 * u + 3]}, inv);
        } else {
          const int r = 64 * w + 32 * rb + lr;
          float *ws = aa.ws + (int64_t)(2 * xcd_wg(aa.wgs) + (x != x0)) * part_floats<D, ROWS>();
          if (g == 0) ws[ROWS * D + r] = mx[rb], ws[ROWS * (D + 1) + r] = l;
#pragma unroll
          for (int d = 0; d < KC; ++d)
#pragma unroll
            for (int u = 0; u < 4; ++u)
              *(f32x4 *)&ws[r * D + 32 * d + 8 * u + 4 * g] =
                  f32x4{acc[rb][d][4 * u], acc[rb][d][4 * u + 1], acc[rb][d][4 * u + 2], acc[rb][d][4 * u + 3]};
        }
      }
    }
    x += blocks;
  }
}

// Merge of the cut items, RPW rows of an item a workgroup: 256 threads as RPW x PG x
// D / 4, where PG threads share a row's parts and add through LDS, in order.  Bound by
// its launch and two reads one after the other: 7 us for 14 rows of 37 parts, 10 for
// 3,640 of 13.
template <int D, int ROWS, int RPW>
__global__ void __launch_bounds__(256) kv8_merge_kernel(const Args8 aa, int32_t groups_of_rows) {
  constexpr int PF = part_floats<D, ROWS>(), Q4 = D / 4, PG = 256 / Q4 / RPW;
  static_assert(PG * Q4 * RPW == 256, "the threads share the rows");
  __shared__ f32x4 part[RPW][PG][Q4];
  __shared__ float lsum[RPW][PG], rtop[RPW][PG];
  int item = (int)blockIdx.x / groups_of_rows, rg = (int)blockIdx.x % groups_of_rows, ci = 0;
  while (item >= aa.heads * aa.call[ci].row_tiles) item -= aa.heads * aa.call[ci++].row_tiles;
  const Call8 &cl = aa.call[ci];
  const int head = item / cl.row_tiles, tile = item - head * cl.row_tiles;
  if (tile * ROWS + rg * RPW >= cl.lq) return;
  const int begin = cl.first + item * cl.blocks, end = begin + cl.blocks;  // the item's units
  // parts: from the range that holds its first unit to that of its last
  int first_wg = (int)((int64_t)begin * aa.wgs / aa.units);
  while (range_begin(aa, first_wg + 1) <= begin) ++first_wg;
  while (range_begin(aa, first_wg) > begin) --first_wg;
  if (range_begin(aa, first_wg + 1) >= end) return;  // whole
  int last_wg = first_wg + 1;
  while (range_begin(aa, last_wg + 1) < end) ++last_wg;
  const int late = range_begin(aa, first_wg) < begin;  // not the first piece of that range
  auto slot = [&](int wg) { return aa.ws + (int64_t)(2 * wg + (wg == first_wg ? late : 0)) * PF; };
  const int d4 = threadIdx.x % Q4, pg = threadIdx.x / Q4 % PG, rr = threadIdx.x / Q4 / PG;
  const int r = rg * RPW + rr, row = tile * ROWS + r;
  // a thread's first parts are read whole before the row's reference is known
  constexpr int AHEAD = 4;
  float top[AHEAD], sums[AHEAD];
  f32x4 vals[AHEAD];
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) {
    const float *p = slot(min(first_wg + pg + i * PG, last_wg));
    top[i] = p[ROWS * D + r], sums[i] = p[ROWS * (D + 1) + r], vals[i] = *(const f32x4 *)&p[r * D + 4 * d4];
  }
  float m = -__builtin_inff();
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) m = fmaxf(m, top[i]);  // (the last part's again behind it)
  for (int wg = first_wg + pg + AHEAD * PG; wg <= last_wg; wg += PG) m = fmaxf(m, slot(wg)[ROWS * D + r]);
  if (PG > 1) {
    if (d4 == 0) rtop[rr][pg] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PG; ++i) m = fmaxf(m, rtop[rr][i]);
  }
  float l = 0.f;
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
  auto add = [&](float t, float s, const f32x4 &x) {
    const float f = t == m ? 1.0f : __builtin_amdgcn_exp2f(t - m);
    l += f * s;
    v += f * x;
  };
#pragma unroll
  for (int i = 0; i < AHEAD; ++i)
    if (first_wg + pg + i * PG <= last_wg) add(top[i], sums[i], vals[i]);
#pragma unroll 4
  for (int wg = first_wg + pg + AHEAD * PG; wg <= last_wg; wg += PG) {
    const float *p = slot(wg);
    add(p[ROWS * D + r], p[ROWS * (D + 1) + r], *(const f32x4 *)&p[r * D + 4 * d4]);
  }
  if (PG > 1) {
    part[rr][pg][d4] = v;
    if (d4 == 0) lsum[rr][pg] = l;
    __syncthreads();
    if (pg) return;
#pragma unroll
    for (int i = 1; i < PG; ++i) {
      v += part[rr][i][d4];
      l += lsum[rr][i];
    }
  }
  if (row >= cl.lq) return;
  const int64_t orow = cl.o_rows ? cl.o_rows[row] : cl.o_row0 + row;
  *(i32x2 *)(cl.o + orow * cl.ots + (int64_t)head * cl.ohs + 4 * d4) = pack4(v, 1.0f / l);
}

// ---- host side

int check_heads(const char *what, int32_t heads, int32_t head_dim) {
  if (heads <= 0 || heads > 32767) return set_error(TMHD_ERR_INVALID, "%s: heads %d", what, heads);
  if (head_dim != 64 && head_dim != 128) return set_error(TMHD_ERR_UNSUPPORTED, "%s: head_dim %d (64 or 128)", what, head_dim);
  return TMHD_OK;
}

int check_slot(const char *what, const tmhd_kv8_segment &s) {
  if (!s.k || !s.v || !s.ks || !s.vs || (uintptr_t)s.k % 16 || (uintptr_t)s.v % 16)
    return set_error(TMHD_ERR_INVALID, "%s: null or misaligned slot", what);
  if (s.cap <= 0 || s.cap % kBlock || s.cap >= 1 << 23) return set_error(TMHD_ERR_INVALID, "%s: slot capacity %d", what, s.cap);
  if (s.format != TMHD_KV8_E4M3 && s.format != TMHD_KV8_INT8)
    return set_error(TMHD_ERR_UNSUPPORTED, "%s: format %d", what, s.format);
  return TMHD_OK;
}

int check_view(const char *what, const tmhd_kv8_segment &s) {
  if (int st = check_slot(what, s)) return st;
  if (s.row0 < 0 || s.row0 % kBlock || s.tokens <= 0 || (int64_t)s.row0 + s.tokens > s.cap)
    return set_error(TMHD_ERR_INVALID, "%s: rows [%d, %d + %d) of a slot of %d", what, s.row0, s.row0, s.tokens, s.cap);
  return TMHD_OK;
}

View view_of(const tmhd_kv8_segment &s, int D) {
  return View{(const uint8_t *)s.k + (int64_t)s.row0 * D, (const uint8_t *)s.v + (int64_t)s.row0 * D,
              s.ks + s.row0 / kBlock, s.vs + s.row0 / kBlock, s.cap, s.tokens, 0, 0};
}

template <typename F>
void dispatch(int D, int format, F &&f) {
  using std::integral_constant;
  if (D == 128)
    format == TMHD_KV8_E4M3 ? f(integral_constant<int, 128>{}, std::true_type{}) : f(integral_constant<int, 128>{}, std::false_type{});
  else
    format == TMHD_KV8_E4M3 ? f(integral_constant<int, 64>{}, std::true_type{}) : f(integral_constant<int, 64>{}, std::false_type{});
}

int blocks_of(const tmhd_kv8_call &c) {
  int64_t b = 0;
  for (int i = 0; i < c.n_segments; ++i) b += (c.seg[i].tokens + kBlock - 1) / kBlock;
  return (int)std::min<int64_t>(b, INT32_MAX);
}

// Items of 32 rows of up to so many blocks go to a workgroup whole: nothing to merge, a
// launch and a workspace less.  us, whole against dealt evenly: 14 heads of 128, 1 row
// over 700 tokens (11 blocks) 17.7/22.4, 2,717 (43) 19.7/22.5, 5,000 (79) 29.6/21.7; 40
// heads, 3 calls of 20 rows over 2,717 32.5/37.7.  Of eight waves where there are no more
// of them than CUs (against four: 14 heads, 200 rows over 2,717 18.2/21.9, 40 heads, 1
// row 21.0/24.9; but 400 items 44.3/37.5).
constexpr int kWholeBlocks = 48;

// Rows of an item, the units of work (item, block) and the workgroups they are dealt to.
struct Plan8 {
  int rows;
  int64_t items, units;
  int wgs;
  int most;    // query rows of the longest call
  bool whole;  // an item to a workgroup, nothing to merge
  bool eight;  // of eight waves
};

// The calls of one launch: items of 32 rows (two workgroups a CU) for up to 32 rows, or
// where they are up to 28 * 128 / D units a workgroup; else of 128 rows (two a CU) or,
// beyond 128 rows, of 256 (one).  A workgroup of 32 rows turns the codes into bf16 for
// them alone, but has no barriers and small parts to merge.  us, items of 32 against
// wider ones, e4m3: 14 heads of 128, 200 rows over 400 tokens (1.3 units) 23/31, 400 rows
// over 1,500 (8.5) 24/41, 256 over 6,000 (21) 36/49; 40 heads, 400 rows over 1,500 (24)
// 36/46, 128 over 6,000 (29) 47/46, 91 over 12,000 (44) 65/53; 14 heads of 64, 256 rows
// over 12,000 (41) 34/44, 400 over 12,000 (67) 48/52.
// A workgroup takes at least 8 blocks (two for each wave that loads blocks of its
// own) or 4.
Plan8 plan(const tmhd_kv8_call *calls, int n, int heads, int D, int64_t cus, Call8 *out) {
  Plan8 p{32, 0, 0, 0, 0, false, false};
  int longest = 0;  // blocks of an item
  int64_t units32 = 0;
  for (int i = 0; i < n; ++i) {
    p.most = std::max(p.most, calls[i].lq);
    longest = std::max(longest, calls[i].lq > 0 ? blocks_of(calls[i]) : 0);
    units32 += (int64_t)heads * (((int64_t)calls[i].lq + 31) / 32) * blocks_of(calls[i]);
  }
  p.rows = p.most <= 32 || units32 <= 2 * cus * 28 * 128 / D ? 32 : p.most <= 128 ? 128 : 256;
  for (int i = 0; i < n; ++i) {
    Call8 c{};
    c.lq = calls[i].lq;
    c.blocks = blocks_of(calls[i]);
    c.row_tiles = (int32_t)(((int64_t)c.lq + p.rows - 1) / p.rows);
    c.first = (int32_t)std::min<int64_t>(p.units, INT32_MAX);
    p.items += (int64_t)heads * c.row_tiles;
    p.units += (int64_t)heads * c.row_tiles * c.blocks;
    if (out) out[i] = c;
  }
  p.whole = p.rows == 32 && longest <= kWholeBlocks;
  const int64_t room = cus * (p.rows == 256 ? 1 : 2), least = p.rows == 32 ? 8 : 4;
  p.wgs = (int)std::min<int64_t>(room, (p.units + least - 1) / least);
  if (p.whole) p.wgs = (int)std::min<int64_t>(p.items, INT32_MAX), p.eight = p.items <= cus;
  return p;
}

// Calls of the launch that starts at calls[i]
int group_end(const tmhd_kv8_call *calls, int n, int i) {
  int segs = 0, e = i;
  while (e < n && e - i < kMaxCalls && segs + calls[e].n_segments <= kMaxSegs) segs += calls[e++].n_segments;
  return e;
}

int check_calls(const char *what, const tmhd_kv8_call *calls, int n) {
  for (int i = 0; i < n; ++i) {
    const tmhd_kv8_call &c = calls[i];
    if (c.lq < 0) return set_error(TMHD_ERR_INVALID, "%s: %d query rows", what, c.lq);
    if (c.n_segments <= 0 || c.n_segments > TMHD_MAX_SEGMENTS)
      return set_error(TMHD_ERR_INVALID, "%s: %d segments (1 .. %d)", what, c.n_segments, TMHD_MAX_SEGMENTS);
    for (int j = 0; j < c.n_segments; ++j) {
      if (int st = check_view(what, c.seg[j])) return st;
      if (c.seg[j].format != calls[0].seg[0].format)
        return set_error(TMHD_ERR_UNSUPPORTED, "%s: segments of both formats in one call", what);
    }
    if (c.lq == 0) continue;
    if (!c.q || !c.o || (uintptr_t)c.q % 16 || (uintptr_t)c.o % 8 || c.q_token_stride % 8 || c.q_head_stride % 8 ||
        c.o_token_stride % 4 || c.o_head_stride % 4)
      return set_error(TMHD_ERR_INVALID, "%s: queries need 16-byte and outputs 8-byte aligned rows", what);
    if ((!c.q_rows && c.q_row0 < 0) || (!c.o_rows && c.o_row0 < 0))
      return set_error(TMHD_ERR_INVALID, "%s: first row %d, %d", what, c.q_row0, c.o_row0);
  }
  return TMHD_OK;
}

template <int D, int ROWS>
void launch_merge(const Args8 &aa, const Plan8 &p, hipStream_t s) {
  if (p.wgs <= 1 || p.whole) return;
  const int rows = std::min(p.most, ROWS);
  // Items of many parts: a row to a workgroup, its parts shared by 1024 / D threads; else
  // 1024 / D rows to a workgroup.  Whole call of 14 heads of 128 over 40,788 tokens (36
  // parts), us: 1 row 34 against 46, 64 rows 57 against 64; 256 rows (18 parts) 105
  // against 99; 40 heads, 91 rows over 11,232 tokens (13 parts) 62 against 54.
  constexpr int RPW = 1024 / D;
  const bool many = p.wgs > 24 * p.items;
  const int groups = many ? rows : (rows + RPW - 1) / RPW;
  if (many)
    hipLaunchKernelGGL((kv8_merge_kernel<D, ROWS, 1>), dim3((unsigned)(p.items * groups)), dim3(256), 0, s, aa, groups);
  else
    hipLaunchKernelGGL((kv8_merge_kernel<D, ROWS, RPW>), dim3((unsigned)(p.items * groups)), dim3(256), 0, s, aa, groups);
}

template <int D, bool E4M3>
void launch_attn(const Args8 &aa, const Plan8 &p, hipStream_t s) {
  if (p.rows == 32) {
    if (p.eight)
      hipLaunchKernelGGL((kv8_rows_kernel<D, 8, E4M3>), dim3((unsigned)p.wgs), dim3(512), 0, s, aa);
    else
      hipLaunchKernelGGL((kv8_rows_kernel<D, 4, E4M3>), dim3((unsigned)p.wgs), dim3(256), 0, s, aa);
    launch_merge<D, 32>(aa, p, s);
  } else if (p.rows == 128) {
    hipLaunchKernelGGL((kv8_tile_kernel<D, E4M3>), dim3((unsigned)p.wgs), dim3(256), 0, s, aa);
    launch_merge<D, 128>(aa, p, s);
  } else {
    hipLaunchKernelGGL((kv8_wide_kernel<D, E4M3>), dim3((unsigned)p.wgs), dim3(256), 0, s, aa);
    launch_merge<D, 256>(aa, p, s);
  }
}

// two slots for each workgroup (none if one takes all)
int64_t parts_bytes(const Plan8 &p, int D) { return p.wgs > 1 && !p.whole ? (int64_t)p.wgs * 2 * p.rows * (D + 2) * 4 : 0; }

}  // namespace
}  // namespace tmhd

extern "C" int tmhd_kv8_pack_ranges(const void *k, const void *v, int64_t token_stride, int64_t head_stride,
                                    const tmhd_pack_range *ranges, int32_t n_ranges, const tmhd_kv8_segment *slot,
                                    int32_t heads, int32_t head_dim, void *stream) {
  using namespace tmhd;
  const char *what = "tmhd_kv8_pack";
  if (int st = check_heads(what, heads, head_dim)) return st;
  if (n_ranges < 0 || (n_ranges > 0 && !ranges) || !slot) return set_error(TMHD_ERR_INVALID, "%s: %d ranges", what, n_ranges);
  if (int st = check_slot(what, *slot)) return st;
  bool any = false;
  for (int i = 0; i < n_ranges; ++i) {
    const tmhd_pack_range &r = ranges[i];
    if (r.n < 0 || r.dst < 0 || r.dst % kBlock || (int64_t)r.dst + r.n > slot->cap || (!r.rows && r.row0 < 0))
      return set_error(TMHD_ERR_INVALID, "%s: %d rows to slot row %d of %d", what, r.n, r.dst, slot->cap);
    for (int j = 0; j < i; ++j)
      if (r.n > 0 && ranges[j].n > 0 && r.dst < (ranges[j].dst + ranges[j].n + kBlock - 1) / kBlock * kBlock &&
          ranges[j].dst < (r.dst + r.n + kBlock - 1) / kBlock * kBlock)
        return set_error(TMHD_ERR_INVALID, "%s: ranges %d and %d share a 64-row block of the slot", what, j, i);
    any = any || r.n > 0;
  }
  if (!any) return TMHD_OK;
  if (!k || !v || (uintptr_t)k % 16 || (uintptr_t)v % 16 || token_stride % 8 || head_stride % 8)
    return set_error(TMHD_ERR_INVALID, "%s: K/V rows must be 16-byte aligned", what);
  PackArgs pa{(const uint16_t *)k, (const uint16_t *)v, token_stride, head_stride, (uint8_t *)slot->k, (uint8_t *)slot->v,
              (uint8_t *)slot->ks, (uint8_t *)slot->vs, slot->cap, 0, {}};
  for (int i = 0; i < n_ranges;) {
    int32_t blocks = 0;
    pa.n_ranges = 0;
    for (; i < n_ranges && pa.n_ranges < kMaxRanges; ++i) {
      if (ranges[i].n == 0) continue;
      auto &r = pa.r[pa.n_ranges++];
      r.rows = ranges[i].rows, r.row0 = ranges[i].row0, r.n = ranges[i].n, r.dst = ranges[i].dst, r.first = blocks;
      blocks += (ranges[i].n + kBlock - 1) / kBlock;
    }
    if (blocks == 0) break;
    dispatch(head_dim, slot->format, [&](auto d, auto e4m3) {
      hipLaunchKernelGGL((kv8_pack_kernel<d.value, e4m3.value>), dim3((unsigned)blocks, (unsigned)heads * 2),
                         dim3(2 * d.value), 0, (hipStream_t)stream, pa);
    });
    if (int st = check_launch(what)) return st;
  }
  return TMHD_OK;
}

extern "C" int tmhd_kv8_expand(const tmhd_kv8_segment *views, const int32_t *dst, int32_t n, void *k_slot,
                               void *vt_slot, int64_t k_head_stride, int64_t vt_head_stride, int32_t vt_row_stride,
                               int32_t heads, int32_t head_dim, void *stream) {
  using namespace tmhd;
  const char *what = "tmhd_kv8_expand";
  if (int st = check_heads(what, heads, head_dim)) return st;
  if (n < 0 || (n > 0 && (!views || !dst))) return set_error(TMHD_ERR_INVALID, "%s: %d views", what, n);
  if (n == 0) return TMHD_OK;
  if (!k_slot || !vt_slot || (uintptr_t)k_slot % 16 || (uintptr_t)vt_slot % 16 || k_head_stride % 8 || vt_head_stride % 8 ||
      vt_row_stride % 8 || vt_head_stride < (int64_t)head_dim * vt_row_stride)
    return set_error(TMHD_ERR_INVALID, "%s: null or misaligned slot", what);
  auto end_of = [&](int i) { return (int64_t)dst[i] + (views[i].tokens + kBlock - 1) / kBlock * kBlock; };
  for (int i = 0; i < n; ++i) {
    if (int st = check_view(what, views[i])) return st;
    const int64_t end = end_of(i);
    if (dst[i] < 0 || dst[i] % kBlock || end > vt_row_stride || end * head_dim > k_head_stride)
      return set_error(TMHD_ERR_INVALID, "%s: view %d of %d rows at slot row %d", what, i, views[i].tokens, dst[i]);
    for (int j = 0; j < i; ++j)
      if (dst[j] < end && dst[i] < end_of(j))
        return set_error(TMHD_ERR_INVALID, "%s: views %d and %d share rows of the slot", what, j, i);
  }
  for (int i = 0; i < n;) {
    ExpandArgs ea{(uint16_t *)k_slot, (uint16_t *)vt_slot, k_head_stride, vt_head_stride, vt_row_stride, 0, {}};
    const int format = views[i].format;  // a launch expands views of one format
    int32_t blocks = 0;
    for (; i < n && ea.n_views < kMaxSegs && views[i].format == format; ++i) {
      View &vw = ea.view[ea.n_views++];
      vw = view_of(views[i], head_dim);
      vw.dst = dst[i], vw.first = blocks;
      blocks += (views[i].tokens + kBlock - 1) / kBlock;
    }
    dispatch(head_dim, format, [&](auto d, auto e4m3) {
      hipLaunchKernelGGL((kv8_expand_kernel<d.value, e4m3.value>), dim3((unsigned)blocks, (unsigned)heads * 2),
                         dim3(2 * d.value), 0, (hipStream_t)stream, ea);
    });
    if (int st = check_launch(what)) return st;
  }
  return TMHD_OK;
}

extern "C" int tmhd_kv8_token_major(const tmhd_kv8_segment *view, void *k, void *v, int32_t heads, int32_t head_dim,
                                    void *stream) {
  using namespace tmhd;
  const char *what = "tmhd_kv8_token_major";
  if (int st = check_heads(what, heads, head_dim)) return st;
  if (!view) return set_error(TMHD_ERR_INVALID, "%s: null view", what);
  if (int st = check_view(what, *view)) return st;
  if (!k || !v || (uintptr_t)k % 16 || (uintptr_t)v % 16) return set_error(TMHD_ERR_INVALID, "%s: null or misaligned output", what);
  const View vw = view_of(*view, head_dim);
  dispatch(head_dim, view->format, [&](auto d, auto e4m3) {
    hipLaunchKernelGGL((kv8_token_major_kernel<d.value, e4m3.value>),
                       dim3((unsigned)((view->tokens + kBlock - 1) / kBlock), (unsigned)heads * 2), dim3(2 * d.value), 0,
                       (hipStream_t)stream, vw, (uint16_t *)k, (uint16_t *)v, heads);
  });
  return check_launch(what);
}

extern "C" int tmhd_attn_kv8_item_rows(const tmhd_kv8_call *calls, int32_t n, int32_t heads, int32_t head_dim, int32_t cus) {
  using namespace tmhd;
  const char *what = "tmhd_attn_kv8_item_rows";
  if (n <= 0 || !calls || check_heads(what, heads, head_dim) || check_calls(what, calls, n)) return -1;
  return plan(calls, group_end(calls, n, 0), heads, head_dim, cus > 0 ? cus : std::max(device_cus(), 8), nullptr).rows;
}

extern "C" int64_t tmhd_attn_kv8_workspace_bytes(const tmhd_kv8_call *calls, int32_t n, int32_t heads, int32_t head_dim) {
  using namespace tmhd;
  if (n <= 0 || !calls || check_heads("tmhd_attn_kv8_workspace_bytes", heads, head_dim) ||
      check_calls("tmhd_attn_kv8_workspace_bytes", calls, n))
    return 0;
  int64_t most = 0;
  for (int i = 0; i < n;) {
    const int e = group_end(calls, n, i);
    most = std::max(most, parts_bytes(plan(calls + i, e - i, heads, head_dim, std::max(device_cus(), 8), nullptr), head_dim));
    i = e;
  }
  return most;
}

extern "C" int tmhd_attn_fwd_kv8(const tmhd_kv8_call *calls, int32_t n, int32_t heads, int32_t head_dim, float scale,
                                 void *workspace, int64_t workspace_bytes, void *stream) {
  using namespace tmhd;
  const char *what = "tmhd_attn_fwd_kv8";
  if (int st = check_heads(what, heads, head_dim)) return st;
  if (n < 0 || (n > 0 && !calls)) return set_error(TMHD_ERR_INVALID, "%s: %d calls", what, n);
  if (int st = check_calls(what, calls, n)) return st;
  if (workspace && (uintptr_t)workspace % 16) return set_error(TMHD_ERR_INVALID, "%s: misaligned workspace", what);
  for (int i = 0; i < n;) {
    const int e = group_end(calls, n, i);
    Args8 aa{};
    const Plan8 p = plan(calls + i, e - i, heads, head_dim, std::max(device_cus(), 8), aa.call);
    // (the merge's workgroups, 1024 / head_dim rows each, within what a launch holds)
    if (p.units > INT32_MAX || p.items * (p.rows * head_dim / 1024) >= 1 << 24)
      return set_error(TMHD_ERR_UNSUPPORTED, "%s: too many query rows and keys", what);
    if (parts_bytes(p, head_dim) > (workspace ? workspace_bytes : 0))
      return set_error(TMHD_ERR_INVALID, "%s: workspace of %lld bytes, %lld needed", what, (long long)workspace_bytes,
                       (long long)parts_bytes(p, head_dim));
    aa.n_calls = e - i;
    aa.heads = heads;
    aa.units = (int32_t)p.units, aa.wgs = p.wgs, aa.whole = p.whole;
    aa.scale2 = fabsf(scale) * 1.4426950408889634f;
    aa.flip = scale < 0.f ? (int32_t)0x80008000u : 0;
    aa.ws = (float *)workspace;
    int segs = 0;
    for (int c = 0; c < aa.n_calls; ++c) {
      const tmhd_kv8_call &in = calls[i + c];
      Call8 &o = aa.call[c];
      o.q = (const uint16_t *)in.q, o.o = (uint16_t *)in.o;
      o.qts = in.q_token_stride, o.qhs = in.q_head_stride, o.ots = in.o_token_stride, o.ohs = in.o_head_stride;
      o.q_rows = in.q_rows, o.o_rows = in.o_rows, o.q_row0 = in.q_row0, o.o_row0 = in.o_row0;
      o.seg0 = segs;
      for (int j = 0; j < in.n_segments; ++j) {
        const View vw = view_of(in.seg[j], head_dim);
        aa.seg[segs++] = Seg8{vw.k, vw.v, vw.ks, vw.vs, vw.cap, vw.tokens};
      }
    }
    if (p.wgs > 0) {
      const int format = calls[i].seg[0].format;
      dispatch(head_dim, format, [&](auto d, auto e4m3) { launch_attn<d.value, e4m3.value>(aa, p, (hipStream_t)stream); });
      if (int st = check_launch(what)) return st;
    }
    i = e;
  }
  return TMHD_OK;
}
