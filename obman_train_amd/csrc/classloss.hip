// K17: softmax cross entropy of features against a table of classes, without keeping the logits.
//
//   z[r, v] = x[r] . w[v] + b[v]          lse[r] = log sum_v exp z[r, v]          loss[r] = lse[r] - z[r, t[r]]
//   g[r, v] = (exp(z[r, v] - lse[r]) - [v = t[r]]) c[r]                           c[r] = d(total) / d(loss[r])
//   dx = g w,   dw = g^T x,   db = sum_r g[r, :]
//
// Forward: one matrix product whose epilogue keeps, per row and tile of 256 classes, the maximum and the sum of exponentials; a join
// over the tiles.  Backward, in pieces of the class axis: the product again, its epilogue writes g of the piece in 16 bits, two
// products read it.  8 rows * classes * width multiply-adds' flops instead of 6 buys that only a piece of g exists at a time.
//
// All products run on 16-bit matrix instructions with fp32 accumulators.  bf16 and fp16 operands go in as they are.  An fp32 operand
// is written as hi + lo, two fp16 numbers (22 bits) after a power-of-two scaling of the whole tensor to 2^13 .. 2^14, and a product is
// lo*hi + hi*lo + hi*hi: 2^-22 relative, and three fp16 products are 5 times the rate of the fp32 matrix instruction.  One scale for the
// whole tensor ends at 2^-39 of its largest element, so this holds while every row's largest element (all zeros aside) is within
// SPREAD = 2^16 of it: 2^-22 of the row's own.  The pass that finds the largest element finds that out too, on the device; if a row of x or
// a class of w lies further off, the same kernels take the operands as fp32 and the fp32 instruction (FULL below; 19 200 x 16 050 x 512 forward and
// backward: 9.6 ms against 3.7).  g has |g| <= max |c|: in fp16 it is scaled to 2^14.  Rounding g to the inputs' 16 bits (its own
// size, before sums of many rows or classes) adds a quarter to the error that rounding the result makes: 2-norms of dx and dw 2.05e-3 off for 1.66e-3 in
// bf16, 2.56e-4 for 2.07e-4 in fp16; a second plane would cost two products more of four.  With fp32 operands g is hi + lo too, and its lo
// is kept 2^12 times as large (the factor comes out of the other operand's hi): g is mostly probabilities, whose small ones are what a class
// that is never a label learns from, and so its bits end at 2^-51 of max |c| instead of 2^-39.
//
// Rows that are ignored take no part: their x (which may be garbage) is packed as zeros, their g is zero.
#include "common.h"
#include "../../include/obman_hip.h"

namespace cl {

typedef unsigned short u16;
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4* lds_s16x4;
typedef u16 u16x8u __attribute__((ext_vector_type(8), aligned(2)));
typedef u16 u16x4u __attribute__((ext_vector_type(4), aligned(2)));
typedef unsigned u32x4u __attribute__((ext_vector_type(4), aligned(2)));
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));

enum { F32 = 0, BF16 = 1, F16 = 2 };

// Operands are kept in blocks of columns, [blocks][rows][64 bytes]: 32 columns of a 16-bit operand, or 16 of a split one, hi beside lo.
// Whatever a step of the contraction needs of one - a block of 256 rows, or some rows of all blocks - is read in runs of 1 KB or more.
// (Row-major, a step reads 64 of each row's bytes, half cache lines, and the path from L2 to LDS is what holds the products back:
// without those reads they run at 1170 - 1270 Tflop/s.)  A split step of 16 has its two planes loaded once for three products.  Rows
// are padded with zeros to whole tiles, so no address leaves an operand.
// Tile 256 x 128, four waves of 128 x 64.  72 KB of LDS, so two blocks share a CU and one's epilogue and waits run under the other's
// products.  (256 x 256 with eight waves, four steps deep, one block on a CU, fetches a third less; at 19 200 x 64 050 x 512 it
// measured 1 474 us for the forward product against 1 330, 328 against 304 for g, 290 against 300 and 250 against 253 for the other two;
// with four waves of 128 x 128, the next half step's reads under the products, the other two together took 499 against 478.)
constexpr int BI = 256, BJ = 128, WAVES = 4, STAGES = 3;
constexpr int A_BYTES = BI * 64, STAGE_BYTES = A_BYTES + BJ * 64;
constexpr int BIAS_AT = STAGES * STAGE_BYTES, LDS_BYTES = BIAS_AT + BI * 4;
constexpr long MOST_ROWS = 1L << 22;  // of an operand: sixteen blocks of its columns stay within 32-bit offsets
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr float G_SCALE = 16384.f;  // |g| / max|c| <= 1 in fp16
constexpr float SPREAD = 65536.f;
constexpr float G_LO = 4096.f;      // factor on g's lo: at 2^14 it is at most 2^2, and fp16 ends at 2^16

template <bool SPLIT>
constexpr int Step = SPLIT ? 16 : 32;  // columns of a block, and the contraction of a step
// FULL: the block's 64 bytes are 16 fp32 numbers instead of 16 hi beside 16 lo.  Places, tiles and loads are the same.

struct Side {  // [blocks][rows][32]
  const u16* p;
  long rows;   // of a block
};
struct Gemm {
  Side a, b;
  long ni, nj;      // extents of the result
  long k;           // contraction, a multiple of the step
  long k_part;      // of it per part
  int ti, tj, parts; // tiles, and parts of the contraction
  int na, nb;       // column blocks of a / b (an operand whose rows are contracted: tiles that run over its columns repeat the last block)
  const float* full; // fp32 operands: not 0 where they are kept in full
};

__device__ __forceinline__ void dma16(__amdgpu_buffer_rsrc_t r, unsigned lds, unsigned voff) {
  // lane l writes 16 bytes at lds + 16 l; a load to LDS must not be the instruction behind the write of m0: one wait state, which the
  // compiler inserts for its own loads but not inside an asm statement
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds), "v"(voff), "s"(r) : "memory", "m0");
}

// One operand's tile for a step of Step<SPLIT> k, R (i or j) wide, in 64-byte rows of LDS.  KC: the rows are i or j and their columns
// are k; 16-byte chunks are placed at chunk ^ (row >> 2 & 3), so that the wide reads do not meet in a bank (the DMA writes LDS
// linearly: the source address carries the swizzle).  KR: the rows are k, a step of them for each column block, read by the
// transposing LDS reads, which take four whole rows at a time; with split operands they take half of each, and every other block
// has its halves exchanged.
template <bool KR, int R, bool SPLIT>
struct Operand {
  static constexpr int N = R * 64 / 1024 / WAVES;  // wave-wide loads of 1 KB per wave and step
  const u16* base;  // at the next step's k
  long step;
  unsigned voff[N];
  __device__ __forceinline__ void init(const Side& s, int first_block, int blocks, int wave, int lane) {
    step = KR ? Step<SPLIT> * 32 : s.rows * 32;
    const int last = blocks - 1 - first_block;
#pragma unroll
    for (int q = 0; q < N; ++q) {
      const int at = wave * N + q;
      if constexpr (!KR) {
        voff[q] = at * 1024 + (lane >> 2) * 64 + ((lane & 3) ^ ((lane >> 4) & 3)) * 16;
      } else if constexpr (!SPLIT) {
        const int b = at >> 1;
        voff[q] = (unsigned)((b < last ? b : last) * s.rows * 64) + (at & 1) * 1024 + lane * 16;
      } else {
        voff[q] = (unsigned)((at < last ? at : last) * s.rows * 64) + (lane >> 2) * 64 + ((lane & 3) ^ ((at & 1) << 1)) * 16;
      }
    }
  }
  // row0: first row (KC: of the tile; KR: of the contraction), col0: first column of the contraction (KC) or of the tile (KR)
  __device__ __forceinline__ void start(const Side& s, long row0, long col0) { base = s.p + (col0 / Step<SPLIT> * s.rows + row0) * 32; }
  __device__ __forceinline__ void issue(unsigned lds, int wave) {
    const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(const_cast<u16*>(base), 0, (int)0xfffffff0u, 0x00020000);
#pragma unroll
    for (int q = 0; q < N; ++q) dma16(r, lds + wave * (N * 1024) + q * 1024, voff[q]);
    base += step;
  }
};

// fragment of 32 rows x 16 k: lane -> row lane % 32, k = 8 (lane / 32) .. + 7; of the step's two halves, or of hi and lo.  FULL: of 8 k,
// lane -> k = 4 (lane / 32) .. + 3
template <bool KR, bool SPLIT, bool FULL>
struct Frag {
  unsigned off[2];
  __device__ __forceinline__ void init(int first_row, int lane) {  // first_row: a multiple of 32
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      // the transposing read: in a group of 16 lanes, lane c receives element c of the four rows that lanes 4 r .. 4 r + 3 point at
      const int k = 8 * (lane >> 5) + ((lane & 15) >> 2), right = (lane >> 4) & 1;
      if constexpr (!KR) off[h] = (first_row + (lane & 31)) * 64 + ((2 * h + (lane >> 5)) ^ ((lane >> 2) & 3)) * 16;
      else if constexpr (FULL) off[h] = first_row * 64 + right * 1024 + (8 * h + 4 * (lane >> 5)) * 64 + (((lane & 15) >> 2) ^ (right << 1)) * 16 + (lane & 3) * 4;
      else if constexpr (!SPLIT) off[h] = first_row * 64 + (h * 16 + k) * 64 + right * 32 + (lane & 3) * 8;
      else off[h] = first_row * 64 + right * 1024 + k * 64 + (h ^ right) * 32 + (lane & 3) * 8;
    }
  }
  __device__ __forceinline__ u32x4 read(const char* tile, int f, int h) const {
    const char* p = tile + off[h] + f * 2048;
    if constexpr (!KR) return *reinterpret_cast<const u32x4*>(p);
    if constexpr (KR && FULL) {  // (two lanes a bank: this path is for the rare tensor)
      u32x4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = *reinterpret_cast<const unsigned*>(p + e * 64);
      return v;
    }
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(p));
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(p + 4 * 64));
    return __builtin_bit_cast(u32x4, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  }
};

template <int T>
__device__ __forceinline__ f32x16 mfma(u32x4 a, u32x4 b, f32x16 c) {
  if constexpr (T == BF16) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

__device__ __forceinline__ f32x16 mfma_f32(u32x4 a, u32x4 b, f32x16 c) {
#pragma unroll
  for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a[e]), __uint_as_float(b[e]), c, 0, 0, 0);
  return c;
}

template <int T>
__device__ __forceinline__ u16 narrow(float x) {
  if constexpr (T == BF16) return __builtin_bit_cast(u16, (__bf16)x);
  else return __builtin_bit_cast(u16, (_Float16)x);
}
template <int T>
__device__ __forceinline__ float widen(u16 u) {
  if constexpr (T == BF16) return __uint_as_float((unsigned)u << 16);
  else return (float)__builtin_bit_cast(_Float16, u);
}
__device__ __forceinline__ float load_one(const void* p, int type, long i) {
  if (type == F32) return static_cast<const float*>(p)[i];
  const u16 u = static_cast<const u16*>(p)[i];
  return type == BF16 ? widen<BF16>(u) : widen<F16>(u);
}
__device__ __forceinline__ void store_one(void* p, int type, long i, float x) {
  if (type == F32) static_cast<float*>(p)[i] = x;
  else static_cast<u16*>(p)[i] = type == BF16 ? narrow<BF16>(x) : narrow<F16>(x);
}
__device__ __forceinline__ long target_of(const void* t, int wide, long r) {
  return wide ? static_cast<const long*>(t)[r] : (long)static_cast<const int*>(t)[r];
}

// Consecutive ids of one XCD (ids go round the eight) take consecutive tiles of one part of the contraction; tiles run 8 j wide, so
// that what an XCD's CUs work on at a time (8 x 8 tiles: 3 MB of operands at width 512) stays in its 4 MB L2.
__device__ __forceinline__ void tile_of(const Gemm& g, int id, int& i, int& j, int& part) {
  const int tiles = g.ti * g.tj, n = tiles * g.parts, x = id & 7, q = n >> 3, rem = n & 7;
  int v = x * q + (x < rem ? x : rem) + (id >> 3);
  part = v / tiles;
  v -= part * tiles;
  const int per = 8 * g.ti, group = v / per, in = v - group * per;
  const int w = g.tj - group * 8 < 8 ? g.tj - group * 8 : 8;
  i = in / w;
  j = group * 8 + in % w;
}

// what the epilogues need to know about the scaling of split operands: exponents on the device
struct Scale {
  const float* a;  // NULL = 1; else the power of two that operand was multiplied by
  const float* b;
  // at most 2^127: two tensors near the end of fp32 would give an infinite factor, and 0 times that for a row of zeros
  __device__ __forceinline__ float inverse() const { return fminf((a ? 1.f / *a : 1.f) * (b ? 1.f / *b : 1.f), 0x1p127f); }
};

struct Ctx {
  long i0, j0;
  int wi, wj, lane, tid, ti_index, tj_index, split;
  char *smem, *bias;
};

__device__ __forceinline__ void clear(f32x16 (&acc)[4][2]) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
}

// The bias of the tile's classes, -inf behind the last one, goes into LDS.  Without scales the accumulators start from it; a scaled
// product adds it afterwards.
template <bool SPLIT>
struct Bias {
  Scale scale;
  const void* bias;
  int type;
  long class0, classes;
  __device__ __forceinline__ static const float* mine(const Ctx& c) {  // of this lane's classes: 8 q + 0 .. 3 from here on
    return reinterpret_cast<const float*>(c.bias) + c.wi * 128 + 4 * (c.lane >> 5);
  }
  __device__ __forceinline__ void before(const Ctx& c, f32x16 (&acc)[4][2]) const {
    const long v0 = class0 + c.i0;
    const bool plain = !bias && v0 + BI <= classes;
    if (SPLIT || !plain) {
      const long v = v0 + c.tid;
      reinterpret_cast<float*>(c.bias)[c.tid] = v >= classes ? -INFINITY : bias ? load_one(bias, type, v) : 0.f;
    }
    if (SPLIT || plain) {
      clear(acc);
      return;
    }
    __syncthreads();
    const float* bl = mine(c);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const f32x4 b = *reinterpret_cast<const f32x4*>(bl + i * 32 + q * 8);
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[i][j][q * 4 + e] = b[e];
      }
  }
  // the logits in place of the sums; factor: what they come out multiplied by
  __device__ __forceinline__ void finish(const Ctx& c, f32x16 (&acc)[4][2]) const {
    if constexpr (SPLIT) {
      const float s = scale.inverse();
      const float* bl = mine(c);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const f32x4 b = *reinterpret_cast<const f32x4*>(bl + i * 32 + q * 8);
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[i][j][q * 4 + e] = __builtin_fmaf(acc[i][j][q * 4 + e], s, b[e]);
        }
    }
  }
};

// where a row's target is among this lane's 64 classes of a 128-wide half tile, or -1
__device__ __forceinline__ int target_at(long target, long first_class, int lane) {
  const long t = target - first_class - 4 * (lane >> 5);
  return t >= 0 && t < 128 && !(t & 4) ? (int)t : -1;
}

// Statistics of a set of logits are (m, s): the maximum, and the sum of exp(z - m).  exp is 2^(z log2 e - m log2 e) in one multiply-add, and
// what rounding m log2 e put into every term is taken out of the sum.  That holds while the rounding is small: for |m| beyond FAR (classes
// masked with a large negative number leave such maxima; past 2.4e38 m log2 e would not even be finite) the difference comes first.
constexpr float FAR = 1048576.f;
__device__ __forceinline__ bool is_far(float m) { return fabsf(m) > FAR; }
// sum of exp(z(i) - m), i < N; m: the largest of them, 0 where that is -inf
template <int N, class Z>
__device__ __forceinline__ float sum_exp(const Z& z, float m) {
  float part[4] = {0.f, 0.f, 0.f, 0.f};
  if (__any(is_far(m))) {
#pragma unroll
    for (int i = 0; i < N; ++i) part[i & 3] += __builtin_amdgcn_exp2f((z(i) - m) * LOG2E);
    return (part[0] + part[1]) + (part[2] + part[3]);
  }
  const float ref = m * LOG2E;
#pragma unroll
  for (int i = 0; i < N; ++i) part[i & 3] += __builtin_amdgcn_exp2f(__builtin_fmaf(z(i), LOG2E, -ref));
  return ((part[0] + part[1]) + (part[2] + part[3])) * __builtin_amdgcn_exp2f(-__builtin_fmaf(m, LOG2E, -ref));
}
// (m, s) <- (m, s) with (m2, s2)
__device__ __forceinline__ void join_stats(float& m, float& s, float m2, float s2) {
  const float top = fmaxf(m, m2), ref = top == -INFINITY ? 0.f : top;
  s = s * __builtin_amdgcn_exp2f((m - ref) * LOG2E) + s2 * __builtin_amdgcn_exp2f((m2 - ref) * LOG2E);
  m = top;
}

// forward: per row (j) and tile of classes (i) the maximum and the sum of exponentials
template <bool SPLIT>
struct Stats {
  Bias<SPLIT> bias;
  const void* target;
  int target_wide;
  float2* part;  // [ti][rows]
  float* picked; // [rows]
  __device__ __forceinline__ void before(const Gemm&, const Ctx& c, f32x16 (&acc)[4][2]) const { bias.before(c, acc); }
  template <bool FULL>
  __device__ __forceinline__ void after(const Gemm& g, const Ctx& c, f32x16 (&acc)[4][2]) const {
    float2* red = reinterpret_cast<float2*>(c.smem);
    bias.finish(c, acc);
    float m[2], sum[2];
#pragma unroll
    for (int fj = 0; fj < 2; ++fj) {
      const long r = c.j0 + c.wj * 64 + fj * 32 + (c.lane & 31);
      const int t = target_at(r < g.nj ? target_of(target, target_wide, r) : -1, bias.class0 + c.i0 + c.wi * 128, c.lane);
      if (__any(t >= 0)) {
        float z = 0.f;
#pragma unroll
        for (int fi = 0; fi < 4; ++fi)
#pragma unroll
          for (int q = 0; q < 16; ++q) z = t == fi * 32 + (q >> 2) * 8 + (q & 3) ? acc[fi][fj][q] : z;
        if (t >= 0) picked[r] = z;
      }
      float top = -INFINITY;
#pragma unroll
      for (int fi = 0; fi < 4; ++fi)
#pragma unroll
        for (int q = 0; q < 16; q += 2) top = fmaxf(top, fmaxf(acc[fi][fj][q], acc[fi][fj][q + 1]));
      top = fmaxf(top, __shfl_xor(top, 32, 64));
      float total = sum_exp<64>([&](int i) { return acc[i >> 4][fj][i & 15]; }, top == -INFINITY ? 0.f : top);
      total += __shfl_xor(total, 32, 64);
      m[fj] = top;
      sum[fj] = total;
      if (c.wi == 1 && c.lane < 32) red[c.wj * 64 + fj * 32 + c.lane] = make_float2(top, total);
    }
    __syncthreads();
    if (c.wi == 0 && c.lane < 32) {
#pragma unroll
      for (int fj = 0; fj < 2; ++fj) {
        const long r = c.j0 + c.wj * 64 + fj * 32 + c.lane;
        const float2 o = red[c.wj * 64 + fj * 32 + c.lane];
        join_stats(m[fj], sum[fj], o.x, o.y);
        if (r < g.nj) part[(long)c.ti_index * g.nj + r] = make_float2(m[fj], sum[fj]);
      }
    }
  }
};

struct RowConst {  // per row of the backward pass
  float lse2;      // (lse - shift - log |c|) in units of log 2, +inf for a row without a gradient: g = exp2(z - shift - lse2) is p |c| in one step
  float c;
  int target;      // -1: none
  float shift;     // the row's maximum where that is far from 0, else 0
};
// of a row whose statistics are m and log2 s
__device__ __forceinline__ RowConst row_const(float m, float log_s, float c, int target) {
  return is_far(m) ? RowConst{log_s - log2f(fabsf(c)), c, target, m} : RowConst{__builtin_fmaf(m, LOG2E, log_s) - log2f(fabsf(c)), c, target, 0.f};
}
constexpr RowConst NO_ROW = {INFINITY, 0.f, -1, 0.f};

// backward: g of a piece of the classes, blocks of 32 classes like every operand; its column sums over the tile's rows on request
template <int T, bool SPLIT>
struct Grad {
  Bias<SPLIT> bias;
  const RowConst* rows;
  long n_rows, rows_padded;
  u16* out;
  int columns;      // of out
  float* sums;      // [tj][columns]: the bias gradient's parts, summed before g is rounded
  __device__ __forceinline__ void before(const Gemm&, const Ctx& c, f32x16 (&acc)[4][2]) const { bias.before(c, acc); }
  template <bool FULL>
  __device__ __forceinline__ void after(const Gemm& g, const Ctx& c, f32x16 (&acc)[4][2]) const {
    bias.finish(c, acc);
#pragma unroll
    for (int fj = 0; fj < 2; ++fj) {
      const long r = c.j0 + c.wj * 64 + fj * 32 + (c.lane & 31);
      RowConst k = NO_ROW;
      if (r < n_rows) k = rows[r];
      const int t = target_at(k.target, bias.class0 + c.i0 + c.wi * 128, c.lane);
      if (__any(k.shift != 0.f)) {
#pragma unroll
        for (int fi = 0; fi < 4; ++fi)
#pragma unroll
          for (int q = 0; q < 16; ++q) acc[fi][fj][q] -= k.shift;
      }
#pragma unroll
      for (int fi = 0; fi < 4; ++fi)
#pragma unroll
        for (int q = 0; q < 16; ++q) acc[fi][fj][q] = __builtin_amdgcn_exp2f(__builtin_fmaf(acc[fi][fj][q], LOG2E, -k.lse2));
      if (__any(t >= 0)) {
#pragma unroll
        for (int fi = 0; fi < 4; ++fi)
#pragma unroll
          for (int q = 0; q < 16; ++q) acc[fi][fj][q] -= t == fi * 32 + (q >> 2) * 8 + (q & 3) ? fabsf(k.c) : 0.f;
      }
      if (__any(k.c < 0.f)) {
        const float sign = k.c < 0.f ? -1.f : 1.f;
#pragma unroll
        for (int fi = 0; fi < 4; ++fi)
#pragma unroll
          for (int q = 0; q < 16; ++q) acc[fi][fj][q] *= sign;
      }
      // lanes l and l + 32 hold classes 0 .. 3 and 4 .. 7 of each 8: an exchange gives each 8 in a row, 16 bytes
      u16* o = out + ((c.i0 + c.wi * 128) / Step<SPLIT> * rows_padded + r) * 32 + 8 * (c.lane >> 5);
#pragma unroll
      for (int fi = 0; fi < 4; ++fi) {
        if (c.i0 + c.wi * 128 + fi * 32 >= columns) continue;
        if constexpr (FULL) {  // four classes a lane, 16 bytes as they are
          float* f = reinterpret_cast<float*>(out) + ((c.i0 + c.wi * 128 + fi * 32) / Step<SPLIT> * rows_padded + r) * 16 + 4 * (c.lane >> 5);
#pragma unroll
          for (int q = 0; q < 4; ++q)
            *reinterpret_cast<f32x4*>(f + (q >> 1) * rows_padded * 16 + (q & 1) * 8) = f32x4{acc[fi][fj][q * 4], acc[fi][fj][q * 4 + 1], acc[fi][fj][q * 4 + 2], acc[fi][fj][q * 4 + 3]};
          continue;
        }
#pragma unroll
        for (int q = 0; q < 4; q += 2) {
          unsigned hi[2][2], lo[2][2];
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float x = acc[fi][fj][(q + u) * 4 + e * 2], y = acc[fi][fj][(q + u) * 4 + e * 2 + 1];
              const u16 hx = narrow<T>(x), hy = narrow<T>(y);
              hi[u][e] = hx | (unsigned)hy << 16;
              if constexpr (SPLIT) lo[u][e] = narrow<T>((x - widen<T>(hx)) * G_LO) | (unsigned)narrow<T>((y - widen<T>(hy)) * G_LO) << 16;
            }
          u16* to = o + (SPLIT ? (fi * 2 + q / 2) * rows_padded * 32 : fi * rows_padded * 32 + q * 8);
          {
            const u32x2 s0 = __builtin_amdgcn_permlane32_swap(hi[0][0], hi[1][0], false, false);
            const u32x2 s1 = __builtin_amdgcn_permlane32_swap(hi[0][1], hi[1][1], false, false);
            *reinterpret_cast<u32x4*>(to) = u32x4{s0[0], s1[0], s0[1], s1[1]};
          }
          if constexpr (SPLIT) {
            const u32x2 s0 = __builtin_amdgcn_permlane32_swap(lo[0][0], lo[1][0], false, false);
            const u32x2 s1 = __builtin_amdgcn_permlane32_swap(lo[0][1], lo[1][1], false, false);
            *reinterpret_cast<u32x4*>(to + 16) = u32x4{s0[0], s1[0], s0[1], s1[1]};
          }
        }
      }
    }
    if (!sums) return;
    // over the 16 lanes of a row of lanes in registers, then [wj][half][class] in LDS
    float* red = reinterpret_cast<float*>(c.smem);
    const int l16 = c.lane & 15;
#pragma unroll
    for (int fi = 0; fi < 4; ++fi) {
      float mine = 0.f;
#pragma unroll
      for (int q = 0; q < 16; ++q) {
        float v = acc[fi][0][q] + acc[fi][1][q];
        v += obman_dpp<0xB1>(v);
        v += obman_dpp<0x4E>(v);
        v += obman_dpp<0x141>(v);
        v += obman_dpp<0x140>(v);
        mine = l16 == q ? v : mine;
      }
      red[(c.wj * 2 + ((c.lane >> 4) & 1)) * 256 + c.wi * 128 + fi * 32 + (l16 >> 2) * 8 + 4 * (c.lane >> 5) + (l16 & 3)] = mine;
    }
    __syncthreads();
    if (c.i0 + c.tid < columns) sums[(long)c.tj_index * columns + c.i0 + c.tid] = (red[c.tid] + red[256 + c.tid]) + (red[512 + c.tid] + red[768 + c.tid]);
  }
};

// a product's result: fp32 slabs [split][nj][ld] (WIDE: the columns are i) or [split][ni][ld] (they are j), added to what is there or not
struct Slab {
  float* out;
  long slab;
  int ld, add;
};
template <bool WIDE>
struct SlabStore {
  Slab s;
  __device__ __forceinline__ void before(const Gemm&, const Ctx&, f32x16 (&acc)[4][2]) const { clear(acc); }
  template <bool FULL>
  __device__ __forceinline__ void after(const Gemm& g, const Ctx& c, f32x16 (&acc)[4][2]) const {
    float* o = s.out + c.split * s.slab;
    const int ld = s.ld;
    if constexpr (!WIDE) {
#pragma unroll
      for (int fj = 0; fj < 2; ++fj) {
        const long j = c.j0 + c.wj * 64 + fj * 32 + (c.lane & 31);
        if (j >= ld) continue;
#pragma unroll
        for (int fi = 0; fi < 4; ++fi)
#pragma unroll
          for (int q = 0; q < 16; ++q) {
            const long i = c.i0 + c.wi * 128 + fi * 32 + (q >> 2) * 8 + 4 * (c.lane >> 5) + (q & 3);
            if (i >= g.ni) continue;
            float* p = o + i * ld + j;
            *p = s.add ? acc[fi][fj][q] + *p : acc[fi][fj][q];
          }
      }
      return;
    }
#pragma unroll
    for (int fj = 0; fj < 2; ++fj) {
      const long j = c.j0 + c.wj * 64 + fj * 32 + (c.lane & 31);
      if (j >= g.nj) continue;
#pragma unroll
      for (int fi = 0; fi < 4; ++fi)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const long i = c.i0 + c.wi * 128 + fi * 32 + q * 8 + 4 * (c.lane >> 5);
          if (i >= ld) continue;
          f32x4* p = reinterpret_cast<f32x4*>(o + j * ld + i);
          f32x4 v = {acc[fi][fj][q * 4], acc[fi][fj][q * 4 + 1], acc[fi][fj][q * 4 + 2], acc[fi][fj][q * 4 + 3]};
          if (s.add) v += *p;
          *p = v;
        }
    }
  }
};

// C[i, j] = sum_k A(i, k) B(j, k)
// Bound: the matrix pipe waits.  At 19 200 x 64 050 x 512 in bf16 the forward product takes 1.21 - 1.37 ms (920 - 1040 Tflop/s) with the pipe busy 55 % of
// cycles at 1.81 GHz, dx and dw of a piece 0.46 ms, 55 % at 1.89; a library's 8192^3 product on the same card has it busy 87 % at 1.59 GHz (1460 Tflop/s under
// the profiler).  The clock falls as the pipe fills: busy share times clock is 1.00 here and 1.39 there.  LDS is read in 14 - 22 % of cycles, without
// conflicts; a step's twelve fragment reads stand before its first product, with one other wave on the SIMD to cover them.  fp32 at 19 200 x 16 050 x 512:
// 70 % at 1.68 GHz.  (Counters: profiles/training_tail_kernel_stats.md.)
// G: which operand is g (its lo is G_LO times as large)
enum { G_NONE, G_A, G_B };
__device__ __forceinline__ u32x4 lowered(u32x4 hi) { return __builtin_bit_cast(u32x4, __builtin_bit_cast(f16x8, hi) * (_Float16)(1.f / G_LO)); }
template <bool A_KR, bool B_KR, int T, bool SPLIT, bool FULL, int G, class Epi>
__device__ __forceinline__ void gemm_as(const Gemm& g, const Epi& epi, int id, char* smem) {
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int bi, bj, part;
  tile_of(g, id, bi, bj, part);
  bi = __builtin_amdgcn_readfirstlane(bi);
  bj = __builtin_amdgcn_readfirstlane(bj);
  part = __builtin_amdgcn_readfirstlane(part);
  const Ctx ctx{(long)bi * BI, (long)bj * BJ, wave & 1, wave >> 1, lane, tid, bi, bj, part, smem, smem + BIAS_AT};
  constexpr int K = Step<SPLIT>;
  Operand<A_KR, BI, SPLIT> oa;
  Operand<B_KR, BJ, SPLIT> ob;
  oa.init(g.a, bi * (BI / K), g.na, wave, lane);
  ob.init(g.b, bj * (BJ / K), g.nb, wave, lane);
  Frag<A_KR, SPLIT, FULL> fa;
  Frag<B_KR, SPLIT, FULL> fb;
  fa.init(ctx.wi * 128, lane);
  fb.init(ctx.wj * 64, lane);
  const long kb = part * g.k_part, ke = kb + g.k_part < g.k ? kb + g.k_part : g.k;
  const int steps = ke > kb ? (int)((ke - kb) / K) : 0;
  const unsigned lds0 = (unsigned)(size_t)(__attribute__((address_space(3))) char*)smem;

  f32x16 acc[4][2];
  epi.before(g, ctx, acc);
  oa.start(g.a, A_KR ? kb : ctx.i0, A_KR ? ctx.i0 : kb);
  ob.start(g.b, B_KR ? kb : ctx.j0, B_KR ? ctx.j0 : kb);
  unsigned to = lds0;
  const auto issue = [&]() {
    oa.issue(to, wave);
    ob.issue(to + A_BYTES, wave);
    to = to == lds0 + (STAGES - 1) * STAGE_BYTES ? lds0 : to + STAGE_BYTES;
  };
  const char* from = smem;
  const auto products = [&](const u32x4 (&a)[4], const u32x4 (&b)[2]) {
    __builtin_amdgcn_sched_barrier(0);  // the reads before go out first
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int f = 0; f < 4; ++f)
#pragma unroll
      for (int h = 0; h < 2; ++h) acc[f][h] = FULL ? mfma_f32(a[f], b[h], acc[f][h]) : mfma<T>(a[f], b[h], acc[f][h]);
    __builtin_amdgcn_s_setprio(0);
    __builtin_amdgcn_sched_barrier(0);
  };
  static_assert(Operand<A_KR, BI, SPLIT>::N + Operand<B_KR, BJ, SPLIT>::N == 6, "the counted wait below");
  if (steps > 0) issue();
  if (steps > 1) issue();
  for (int s = 0; s < steps; ++s) {
    // step s has arrived for every wave (only step s + 1 may still be under way), and every wave has read step s - 1, whose slot is next
    if (s + 1 < steps) asm volatile("s_waitcnt vmcnt(6) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    u32x4 a[2][4], b[2][2];  // the step's two halves of 16, or hi and lo
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int f = 0; f < 2; ++f) b[h][f] = fb.read(from + A_BYTES, f, h);
#pragma unroll
      for (int f = 0; f < 4; ++f) a[h][f] = fa.read(from, f, h);
    }
    from = from == smem + (STAGES - 1) * STAGE_BYTES ? smem : from + STAGE_BYTES;
    products(a[0], b[0]);
    if (s + 2 < steps) issue();  // (here rather than before the reads: 2 - 5 % of the logits products)
    if constexpr (SPLIT && !FULL) {
      if constexpr (G == G_B) {
#pragma unroll
        for (int f = 0; f < 4; ++f) a[0][f] = lowered(a[0][f]);
      }
      products(a[0], b[1]);
      if constexpr (G == G_A) {
#pragma unroll
        for (int f = 0; f < 2; ++f) b[0][f] = lowered(b[0][f]);
      }
      products(a[1], b[0]);
    } else {
      products(a[1], b[1]);
    }
  }
  __syncthreads();
  epi.template after<FULL>(g, ctx, acc);
}
template <bool A_KR, bool B_KR, int T, bool SPLIT, int G, class Epi>
__device__ __forceinline__ void gemm(const Gemm& g, const Epi& epi, int id, char* smem) {
  if constexpr (SPLIT) {
    if (*g.full != 0.f) {
      gemm_as<A_KR, B_KR, T, SPLIT, true, G>(g, epi, id, smem);
      return;
    }
  }
  gemm_as<A_KR, B_KR, T, SPLIT, false, G>(g, epi, id, smem);
}

template <int T, bool SPLIT, class Epi>
__global__ __launch_bounds__(WAVES * 64, 2) void logits_kernel(Gemm g, Epi epi) {
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  gemm<false, false, T, SPLIT, G_NONE>(g, epi, blockIdx.x, smem);
}

// dx and dw of a piece of the classes in one launch (each may have no blocks): both read the same g, and their blocks fill each
// other's last round.  The longer ones come first; first: how many blocks that is, rounded up to whole rounds of the XCDs.
// WIDE: the width is on the tile's 256 side; else on its 128 side, where 256 would leave half a tile empty (wide_of).
template <int T, bool SPLIT, bool WIDE>
__global__ __launch_bounds__(WAVES * 64, 2) void grads_kernel(Gemm gx, Slab ex, int nx, Gemm gw, Slab ew, int nw, int x_first) {
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  const int first = ((x_first ? nx : nw) + 7) & ~7;
  const bool is_x = ((int)blockIdx.x < first) == (x_first != 0);
  const int id = (int)blockIdx.x < first ? blockIdx.x : blockIdx.x - first;
  if (id >= (is_x ? nx : nw)) return;
  if (is_x) gemm<WIDE, !WIDE, T, SPLIT, WIDE ? G_B : G_A>(gx, SlabStore<WIDE>{ex}, id, smem);
  else gemm<true, true, T, SPLIT, WIDE ? G_B : G_A>(gw, SlabStore<WIDE>{ew}, id, smem);
}

// ------------------------------------------------------------------------------------------------------- operands and rows

// of the kept rows of x (grid row 0) and of w (1): the largest finite |element|, and the least of the rows' largest (rows of zeros
// aside).  MAX_PARTS block values each: [largest of x, of w, least of x, of w]
constexpr int MAX_PARTS = 512;
__device__ __forceinline__ float wave_max(float m) {  // within 16 lanes, then of the four 16s, all in registers
  m = fmaxf(m, obman_dpp<0xB1>(m));
  m = fmaxf(m, obman_dpp<0x4E>(m));
  m = fmaxf(m, obman_dpp<0x141>(m));
  m = fmaxf(m, obman_dpp<0x140>(m));
  u32x2 s = __builtin_amdgcn_permlane16_swap(__float_as_uint(m), __float_as_uint(m), false, false);
  m = fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
  s = __builtin_amdgcn_permlane32_swap(__float_as_uint(m), __float_as_uint(m), false, false);
  return fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
}
__global__ __launch_bounds__(256) void absmax_kernel(const float* __restrict__ x, long rows, const float* __restrict__ w, long classes, int width, const void* target, int wide,
                                                    long ignore, float* __restrict__ part) {
  const bool first = blockIdx.y == 0;
  const float* p = first ? x : w;
  const long n = first ? rows : classes;
  const int lane = threadIdx.x & 63, full = width & ~3;
  float top = 0.f, least = INFINITY;
  for (long r = (long)blockIdx.x * 4 + (threadIdx.x >> 6); r < n; r += MAX_PARTS * 4) {  // a wave takes a row
    if (first && target_of(target, wide, r) == ignore) continue;
    const float* q = p + r * width;
    float m = 0.f;
    for (int i = lane * 4; i < full; i += 256) {
      const f32x4u v = *reinterpret_cast<const f32x4u*>(q + i);
#pragma unroll
      for (int e = 0; e < 4; ++e) { const float a = fabsf(v[e]); m = a > m && a < INFINITY ? a : m; }
    }
    if (full + lane < width) { const float a = fabsf(q[full + lane]); m = a > m && a < INFINITY ? a : m; }
    m = wave_max(m);
    top = fmaxf(top, m);
    if (m > 0.f) least = fminf(least, m);
  }
  __shared__ float red[2][4];
  if (lane == 0) { red[0][threadIdx.x >> 6] = top; red[1][threadIdx.x >> 6] = least; }
  __syncthreads();
  if (threadIdx.x == 0) {
    part[blockIdx.y * MAX_PARTS + blockIdx.x] = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
    part[(2 + blockIdx.y) * MAX_PARTS + blockIdx.x] = fminf(fminf(red[1][0], red[1][1]), fminf(red[1][2], red[1][3]));
  }
}

// Every thread of the block: whether fp32 operands are kept in full, and the powers of two that bring the largest elements to 2^13 .. 2^14
// (1 for an all-zero tensor, and in full)
struct Scales { float x, w; bool full; };
__device__ __forceinline__ float scale_to(float m) {
  int e = 0;
  if (m > 0.f) (void)frexpf(m, &e);  // m = f 2^e, f in [0.5, 1)
  e = 14 - e;
  e = e > 120 ? 120 : e < -112 ? -112 : e;  // a power of two and its inverse are normal numbers
  return m > 0.f ? ldexpf(1.f, e) : 1.f;
}
__device__ Scales scales_of(const float* __restrict__ part) {
  __shared__ float red[4][4];
  float v[4][2];
#pragma unroll
  for (int k = 0; k < 4; ++k) { v[k][0] = part[k * MAX_PARTS + threadIdx.x]; v[k][1] = part[k * MAX_PARTS + threadIdx.x + 256]; }
#pragma unroll
  for (int k = 0; k < 4; ++k) red[k][threadIdx.x >> 6] = k < 2 ? wave_max(fmaxf(v[k][0], v[k][1])) : -wave_max(-fminf(v[k][0], v[k][1]));  // (64 lanes, one value)
  __syncthreads();
  const auto top = [&](int k) { return fmaxf(fmaxf(red[k][0], red[k][1]), fmaxf(red[k][2], red[k][3])); };
  const auto least = [&](int k) { return fminf(fminf(red[k][0], red[k][1]), fminf(red[k][2], red[k][3])); };
  const float x = top(0), w = top(1);
  const bool full = (x > 0.f && x * (1.f / SPREAD) > least(2)) || (w > 0.f && w * (1.f / SPREAD) > least(3));
  return full ? Scales{1.f, 1.f, true} : Scales{scale_to(x), scale_to(w), false};
}

// x (grid row 0) and w (1) into blocks of columns, [blocks][padded rows][32]: zeros behind the width, behind the last row and for
// ignored rows
struct Pack { const void* src; u16* dst; long rows, padded; };
constexpr int FULL_AT = 3;  // where the scales say whether the operands are kept in full
template <int TYPE>
__global__ __launch_bounds__(256) void pack_kernel(Pack px, Pack pw, int width, int chunks, const void* target, int wide, long ignore, const float* __restrict__ part,
                                                  float* __restrict__ scale) {
  const bool first = blockIdx.y == 0;
  const Pack p = first ? px : pw;
  float sc = 1.f;
  bool full = false;
  if constexpr (TYPE == F32) {
    const Scales s = scales_of(part);
    sc = first ? s.x : s.w;
    full = s.full;
    if (blockIdx.x == 0 && threadIdx.x == 0) {
      scale[blockIdx.y] = sc;
      if (first) scale[FULL_AT] = full ? 1.f : 0.f;
    }
  }
  const long n = p.padded * chunks;  // of 8 columns
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long)gridDim.x * 256) {
    const long r = i / chunks;
    const int c = (int)(i - r * chunks) * 8;
    u32x4 one = {0, 0, 0, 0}, two = {0, 0, 0, 0};  // fp32: hi and lo, or in full the first four and the others
    if (r < p.rows && (!first || target_of(target, wide, r) != ignore)) {
      const long at = r * width + c;
      if constexpr (TYPE == F32) {
        const float* q = static_cast<const float*>(p.src) + at;
        float v[8];
        if (c + 8 <= width) {
          const f32x4u a = *reinterpret_cast<const f32x4u*>(q), b = *reinterpret_cast<const f32x4u*>(q + 4);
#pragma unroll
          for (int e = 0; e < 4; ++e) { v[e] = a[e]; v[e + 4] = b[e]; }
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = c + e < width ? q[e] : 0.f;
        }
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
          const float y0 = v[e] * sc, y1 = v[e + 1] * sc;
          const u16 h0 = narrow<F16>(y0), h1 = narrow<F16>(y1);
          const u16 l0 = fabsf(y0) < INFINITY ? narrow<F16>(y0 - widen<F16>(h0)) : (u16)0, l1 = fabsf(y1) < INFINITY ? narrow<F16>(y1 - widen<F16>(h1)) : (u16)0;
          one[e / 2] = h0 | (unsigned)h1 << 16;
          two[e / 2] = l0 | (unsigned)l1 << 16;
        }
        if (full) {
#pragma unroll
          for (int e = 0; e < 4; ++e) { one[e] = __float_as_uint(v[e]); two[e] = __float_as_uint(v[e + 4]); }
        }
      } else {
        const u16* q = static_cast<const u16*>(p.src) + at;
        if (c + 8 <= width) {
          const u16x8u a = *reinterpret_cast<const u16x8u*>(q);
#pragma unroll
          for (int e = 0; e < 8; ++e) one[e / 2] |= (unsigned)a[e] << (16 * (e & 1));
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) one[e / 2] |= (c + e < width ? (unsigned)q[e] : 0u) << (16 * (e & 1));
        }
      }
    }
    constexpr int K = Step<TYPE == F32>;
    u16* o = p.dst + ((long)(c / K) * p.padded + r) * 32 + (full ? 2 : 1) * (c % K);
    *reinterpret_cast<u32x4*>(o) = one;
    if constexpr (TYPE == F32) *reinterpret_cast<u32x4*>(o + (full ? 8 : 16)) = two;
  }
}

// Few rows (scoring single features): the table is read once, as it is, and that read is the time.  A wave holds 32 classes x 32 G rows:
// its lanes load 16 bytes of each of the 32 class rows straight into matrix operands (a lane's element order along the width is free
// as long as x, staged in LDS, has the same), fp32 on the fp32 instruction.  Blocks run over the table with running statistics; a
// second launch joins them (one block for everything is 3 us quicker up to 2^17 elements of the table and loses soon behind: left out).
// One row against 64 050 x 512 in bf16: 17 us under the profiler, 3.9 TB/s, the 66 MB partly from the 256 MB cache (a large copy: 4.8).
constexpr int FEW = 64;  // most rows: at 64 050 classes x 512 in bf16, 64 take 36 us here and 60 packed, 128 would take 70 and 62
template <int TYPE> struct FewT { static constexpr int E = 8; };  // elements of a 16-byte piece
template <> struct FewT<F32> { static constexpr int E = 4; };
template <int TYPE, int G>
__global__ __launch_bounds__(256) void few_kernel(const void* __restrict__ xs, const void* __restrict__ ws, const void* __restrict__ bias, const void* target, int wide, int rows,
                                                 long classes, int width, float2* __restrict__ part, float* __restrict__ picked) {
  constexpr int E = FewT<TYPE>::E, SIZE = 16 / E, AHEAD = 8, R = 32 * G;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  __shared__ float2 red[4][R];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, half = lane >> 5;
  const int pieces = (width + 2 * E - 1) / (2 * E);  // of 2 E columns, one 16-byte half for each half of the wave
  const int safe = width / (2 * E);                  // pieces that lie inside the row
  long v0 = ((long)blockIdx.x * 4 + wave) * 32;
  const auto row_of = [&](long v) { return static_cast<const char*>(ws) + (v < classes ? v : classes - 1) * width * SIZE + half * 16; };
  const char* row = row_of(v0 + (lane & 31));
  u32x4 a[AHEAD];
  const auto load = [&](int p) {
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) a[u] = *reinterpret_cast<const u32x4u*>(row + (p + u) * 32);
  };
  if (safe >= AHEAD) load(0);  // under way while x is staged
  // x in LDS: [piece][half][row] 16 bytes, zeros behind the width and the last row
  for (int i = tid; i < pieces * 2 * R; i += 256) {
    const int r = i % R, c = i / R * E;
    u32x4 v = {0, 0, 0, 0};
    if (r < rows) {
      const char* p = static_cast<const char*>(xs) + ((long)r * width + c) * SIZE;
      if (c + E <= width) v = *reinterpret_cast<const u32x4u*>(p);
      else
#pragma unroll
        for (int e = 0; e < E; ++e) {
          if (c + e >= width) continue;
          if constexpr (TYPE == F32) v[e] = reinterpret_cast<const unsigned*>(p)[e];
          else v[e >> 1] |= (unsigned)reinterpret_cast<const u16*>(p)[e] << (16 * (e & 1));
        }
    }
    reinterpret_cast<u32x4*>(smem)[i] = v;
  }
  __syncthreads();
  const char* xl = smem + (half * R + (lane & 31)) * 16;
  long t[G];
  float m[G], s[G];
#pragma unroll
  for (int g = 0; g < G; ++g) {
    const int r = g * 32 + (lane & 31);
    t[g] = r < rows ? target_of(target, wide, r) : -1;
    m[g] = -INFINITY;
    s[g] = 0.f;
  }
  for (bool first = true; v0 < classes; v0 += (long)gridDim.x * 128, first = false) {
    if (!first) {
      row = row_of(v0 + (lane & 31));
      if (safe >= AHEAD) load(0);
    }
    f32x16 acc[G];
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int q = 0; q < 16; ++q) acc[g][q] = 0.f;
    const auto step = [&](u32x4 w, int p) {
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const u32x4 b = *reinterpret_cast<const u32x4*>(xl + (p * 2 * R + g * 32) * 16);
        if constexpr (TYPE == F32) acc[g] = mfma_f32(w, b, acc[g]);
        else acc[g] = mfma<TYPE>(w, b, acc[g]);
      }
    };
    int p = 0;
    for (; p + AHEAD <= safe; p += AHEAD) {
      if (p) load(p);
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) step(a[u], p + u);
    }
    for (; p < safe; ++p) step(*reinterpret_cast<const u32x4u*>(row + p * 32), p);
    if (p < pieces) {
      u32x4 w = {0, 0, 0, 0};
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int c = p * 2 * E + half * E + e;
        if (c >= width) continue;
        if constexpr (TYPE == F32) w[e] = reinterpret_cast<const unsigned*>(row + p * 32)[e];
        else w[e >> 1] |= (unsigned)reinterpret_cast<const u16*>(row + p * 32)[e] << (16 * (e & 1));
      }
      step(w, p);
    }
    // lane: row 32 g + lane % 32, classes v0 + 8 (q / 4) + 4 half + q % 4
#pragma unroll
    for (int g = 0; g < G; ++g) {
      float top = m[g];
#pragma unroll
      for (int q = 0; q < 16; ++q) {
        const long c = v0 + 8 * (q >> 2) + 4 * half + (q & 3);
        acc[g][q] = c < classes ? acc[g][q] + (bias ? load_one(bias, TYPE, c) : 0.f) : -INFINITY;
        if (c == t[g]) picked[g * 32 + (lane & 31)] = acc[g][q];
        top = fmaxf(top, acc[g][q]);
      }
      const float ref = top == -INFINITY ? 0.f : top;
      s[g] = s[g] * __builtin_amdgcn_exp2f((m[g] - ref) * LOG2E) + sum_exp<16>([&](int q) { return acc[g][q]; }, ref);
      m[g] = top;
    }
  }
#pragma unroll
  for (int g = 0; g < G; ++g) {
    join_stats(m[g], s[g], __shfl_xor(m[g], 32, 64), __shfl_xor(s[g], 32, 64));
    if (half == 0) red[wave][g * 32 + lane] = make_float2(m[g], s[g]);
  }
  __syncthreads();
  if (tid < rows && tid < R) {
    float2 k = red[0][tid];
#pragma unroll
    for (int w = 1; w < 4; ++w) join_stats(k.x, k.y, red[w][tid].x, red[w][tid].y);
    part[(long)tid * gridDim.x + blockIdx.x] = k;
  }
}

// a row's loss from its statistics: the label's distance from the maximum first, log s may be lost beside either.  A label outside the
// table poisons the loss instead of being read
__device__ __forceinline__ float row_loss(float m, float log_s, long t, long classes, long ignore, const float* picked, long r) {
  return t == ignore ? 0.f : t >= 0 && t < classes ? (m - picked[r]) + LN2 * log_s : NAN;
}
// loss = sum or mean over the kept rows (no row kept: 0); norm = what a row's gradient is multiplied by
__device__ __forceinline__ void total_loss(double l, double k, int mean, float* loss, float* norm) {
  if (k < 1.0) k = 1.0;
  *loss = (float)(mean ? l / k : l);
  *norm = (float)(mean ? 1.0 / k : 1.0);
}

// the end of few_kernel: a wave joins a row's block statistics, one block everything
__global__ __launch_bounds__(1024) void few_join_kernel(const float2* __restrict__ part, int n, int rows, long classes, const float* __restrict__ picked, const void* target, int wide,
                                                       long ignore, int reduction, float* __restrict__ loss, float* __restrict__ norm) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  __shared__ double2 red[FEW];
  for (int r = wave; r < rows; r += 16) {
    float m = -INFINITY, s = 0.f;
    for (int i = lane; i < n; i += 64) { const float2 p = part[(long)r * n + i]; join_stats(m, s, p.x, p.y); }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) join_stats(m, s, __shfl_xor(m, off, 64), __shfl_xor(s, off, 64));
    const long t = target_of(target, wide, r);
    const float l = row_loss(m, __builtin_amdgcn_logf(s), t, classes, ignore, picked, r);  // v_log_f32: log2
    if (lane == 0) {
      if (reduction == 0) loss[r] = l;
      red[r] = make_double2(l, t != ignore);
    }
  }
  if (reduction == 0) return;
  __syncthreads();
  if (threadIdx.x) return;
  double l = 0.0, k = 0.0;
  for (int r = 0; r < rows; ++r) { l += red[r].x; k += red[r].y; }
  total_loss(l, k, reduction == 2, loss, norm);
}

// what g is scaled by: to use fp16's range, and not at all where it is kept in fp32
struct GScale {
  float value;
  const float* full;
  __device__ __forceinline__ float get() const { return full && *full != 0.f ? 1.f : value; }
};

// Per row: join over the tiles of classes; loss per row, what the backward pass needs of the row if every row weighs the same, and per
// block of 64 rows the sum of losses and the number of kept rows.  WHOLE: one block does all rows and the reduction.
template <bool WHOLE>
__global__ __launch_bounds__(WHOLE ? 1024 : 256) void join_rows_kernel(const float2* __restrict__ part, int tiles, long rows, long classes, const float* __restrict__ picked,
                                                                      const void* target, int wide, long ignore, int reduction, GScale g_scale, float2* __restrict__ lse,
                                                                      float* __restrict__ loss, RowConst* __restrict__ consts, double2* __restrict__ sums, float* __restrict__ norm) {
  constexpr int GROUPS = WHOLE ? 4 : 1;  // of 64 rows x 4 threads
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, w = wave & 3, group = wave >> 2;
  __shared__ float2 red[GROUPS][4][64];
  double l = 0.0, kept = 0.0;
  for (long r0 = (long)blockIdx.x * 64; r0 < rows; r0 += WHOLE ? 256 : rows) {  // (not WHOLE: once)
    const long r = r0 + group * 64 + lane;
    float m = -INFINITY, s = 0.f;
    const auto join = [&](float2 p) { join_stats(m, s, p.x, p.y); };
    if (r < rows)
      for (int t = w; t < tiles; t += 4) join(part[(long)t * rows + r]);
    red[group][w][lane] = make_float2(m, s);
    __syncthreads();
    if (w == 0 && r < rows) {
#pragma unroll
      for (int k = 1; k < 4; ++k) join(red[group][k][lane]);
      const long t = target_of(target, wide, r);
      const bool none = t == ignore, outside = t < 0 || t >= classes;
      const float log_s = !none && outside ? NAN : __builtin_amdgcn_logf(s);  // v_log_f32: log2
      lse[r] = make_float2(m, log_s);
      const float row = row_loss(m, log_s, t, classes, ignore, picked, r);
      if (reduction == 0) loss[r] = row;
      if (consts) consts[r] = none ? NO_ROW : row_const(m, log_s, g_scale.get(), outside ? -1 : (int)t);
      l += row;
      kept += t != ignore;
    }
    __syncthreads();
  }
  if (reduction == 0) return;
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) { l += __shfl_xor(l, off, 64); kept += __shfl_xor(kept, off, 64); }
  if constexpr (!WHOLE) {
    if (threadIdx.x == 0) sums[blockIdx.x] = make_double2(l, kept);
  } else {
    __shared__ double2 total[GROUPS];
    if (w == 0 && lane == 0) total[group] = make_double2(l, kept);
    __syncthreads();
    if (threadIdx.x == 0)
      total_loss((total[0].x + total[1].x) + (total[2].x + total[3].x), (total[0].y + total[1].y) + (total[2].y + total[3].y), reduction == 2, loss, norm);
  }
}

__global__ __launch_bounds__(256) void reduce_kernel(const double2* __restrict__ sums, int n, int mean, float* __restrict__ loss, float* __restrict__ norm) {
  double l = 0.0, k = 0.0;
  for (int i = threadIdx.x; i < n; i += 256) { const double2 p = sums[i]; l += p.x; k += p.y; }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) { l += __shfl_xor(l, off, 64); k += __shfl_xor(k, off, 64); }
  __shared__ double red[2][4];
  if ((threadIdx.x & 63) == 0) { red[0][threadIdx.x >> 6] = l; red[1][threadIdx.x >> 6] = k; }
  __syncthreads();
  if (threadIdx.x) return;
  l = (red[0][0] + red[0][1]) + (red[0][2] + red[0][3]);
  k = (red[1][0] + red[1][1]) + (red[1][2] + red[1][3]);
  total_loss(l, k, mean, loss, norm);
}

// the largest finite |weight| of the kept rows from `first` on, `step` blocks of 1024 apart; every thread of the block has it
__device__ float weight_max(const void* target, int wide, long ignore, long rows, const float* __restrict__ g_loss, long first, long step) {
  float top = 0.f;
  __shared__ float red[16];
  for (long r = first * 1024 + threadIdx.x; r < rows; r += step * 1024) {
    const float a = fabsf(g_loss[r]);
    if (a > top && a < INFINITY && target_of(target, wide, r) != ignore) top = a;
  }
  top = obman_wave_max(top);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = top;
  __syncthreads();
  top = red[0];
#pragma unroll
  for (int w = 1; w < 16; ++w) top = fmaxf(top, red[w]);
  return top;
}
constexpr int ROW_MAX_BLOCKS = 64;
__global__ __launch_bounds__(1024) void row_max_kernel(const void* target, int wide, long ignore, long rows, const float* __restrict__ g_loss, float* __restrict__ part) {
  const float top = weight_max(target, wide, ignore, rows, g_loss, blockIdx.x, ROW_MAX_BLOCKS);
  if (threadIdx.x == 0) part[blockIdx.x] = top;
}

// A gradient for every row: RowConst with its weight, scaled to at most 1 in magnitude by a power of two; alpha takes it back.  part: the
// ROW_MAX_BLOCKS maxima of row_max_kernel, or NULL: every block looks through all rows.
__global__ __launch_bounds__(1024) void rows_kernel(const float2* __restrict__ lse, const void* target, int wide, long ignore, long rows, const float* __restrict__ g_loss,
                                                   const float* __restrict__ part, GScale g_scale, RowConst* __restrict__ out, float* __restrict__ alpha) {
  const float top = part ? obman_wave_max(part[threadIdx.x & (ROW_MAX_BLOCKS - 1)]) : weight_max(target, wide, ignore, rows, g_loss, 0, 1);
  int e = 0;
  if (top > 0.f) (void)frexpf(top, &e);
  e = e > 120 ? 120 : e < -120 ? -120 : e;
  const float up = ldexpf(1.f, e), down = ldexpf(1.f, -e);
  if (blockIdx.x == 0 && threadIdx.x == 0) *alpha = up;
  const long r = (long)blockIdx.x * 1024 + threadIdx.x;
  if (r >= rows) return;
  const long t = target_of(target, wide, r);
  const float w = t == ignore ? 0.f : g_loss[r] * down * g_scale.get();
  out[r] = w == 0.f ? NO_ROW : row_const(lse[r].x, lse[r].y, w, t < 0 || t > 0x7fffffffL ? -1 : (int)t);
}

// The end of a piece: the slabs' sums times alpha in the gradient's own type (x: grid row 0, w: 1), and the bias gradient from the
// column sums of the tiles of rows, in order (2).  rows = 0: nothing to do.  alpha = *a * *b / g_scale.
struct Finish { const float* slabs; int n; long slab, rows; const float* scale; void* out; };
struct FinishBias { const float* sums; int n, columns; long classes; void* out; };
struct Alpha {
  const float *a, *b;
  GScale g_scale;  // a power of two
  __device__ __forceinline__ float value() const { return *a * (b ? *b : 1.f) / g_scale.get(); }
};
__global__ __launch_bounds__(256) void finish_kernel(Finish fx, Finish fw, FinishBias fb, int ld, int width, Alpha alpha, int type) {
  if (blockIdx.y == 2) {
    const float k = alpha.value();
    for (long v = (long)blockIdx.x * 256 + threadIdx.x; v < fb.classes; v += (long)gridDim.x * 256) {
      double s = 0.0;
      for (int t = 0; t < fb.n; ++t) s += fb.sums[(long)t * fb.columns + v];
      store_one(fb.out, type, v, (float)(s * k));
    }
    return;
  }
  const Finish f = blockIdx.y == 0 ? fx : fw;
  const int per = (width + 3) >> 2;
  const long total = f.rows * per;
  if ((long)blockIdx.x * 256 >= total) return;
  const float k = alpha.value(), k2 = f.scale ? 1.f / *f.scale : 1.f;  // (in turn: their product may end below the normal numbers, with few bits)
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long)gridDim.x * 256) {
    const long r = i / per;
    const int c = (int)(i - r * per) * 4;
    const float* p = f.slabs + r * ld + c;
    f32x4 v = *reinterpret_cast<const f32x4*>(p);
    for (int s = 1; s < f.n; ++s) v += *reinterpret_cast<const f32x4*>(p + s * f.slab);
    v = v * k * k2;
    const long at = r * width + c;
    if (c + 4 <= width) {
      if (type == F32) *reinterpret_cast<f32x4u*>(static_cast<float*>(f.out) + at) = f32x4u{v[0], v[1], v[2], v[3]};
      else {
        u16x4u o;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = type == BF16 ? narrow<BF16>(v[e]) : narrow<F16>(v[e]);
        *reinterpret_cast<u16x4u*>(static_cast<u16*>(f.out) + at) = o;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (c + e < width) store_one(f.out, type, at + e, v[e]);
    }
  }
}

// --------------------------------------------------------------------------------------------------------------- the calls

static inline long up(long x, long m) { return (x + m - 1) / m * m; }

struct Carve {  // scratch: offsets first, pointers once a base is there
  char* base;
  size_t at = 0;
  template <class P>
  P* take(size_t n) {
    P* p = base ? reinterpret_cast<P*>(base + at) : nullptr;
    at = (at + n * sizeof(P) + 255) & ~(size_t)255;
    return p;
  }
};

constexpr long PIECE_BYTES = 512L << 20;  // of g at a time

// what the forward pass leaves for the backward pass: both operands in blocks, their scales and whether they are kept in full, and per row the statistics (maximum, log2 of
// the sum) and, if all rows weigh the same, the constants
struct Keep {
  Side x, w;
  u16 *xp, *wp;
  float *scales, *norm;
  float2* lse;
  RowConst* rows;
  int ld;  // the width, up to whole blocks
  size_t bytes;
};
// Which side of the tiles of dx and dw the width goes to: the 128 wide one where that leaves out 15 % of what is multiplied, whole tiles
// counted, and the tiles are many.  Rows of g then come in 256s, each further one costing its logits and, like 512 columns, their
// exponentials.  Forward and backward at 19 200 x 16 050: width 64 in bf16 622 -> 530 us, in fp32 1 384 -> 1 050; width 515 in fp32
// 4 032 -> 3 820.  (At 8 000 x 4 000 x 640, 14 %: 517 -> 527; at 1 344 x 778 x 100, few tiles: 65 -> 72.)
static bool wide_of(const obman_class_loss_params& p) {
  const double ld = (double)up(p.width, 32), r1 = (double)up(p.rows, BJ), r2 = (double)up(p.rows, BI), v = (double)p.classes, v1 = (double)up(p.classes, BJ);
  const double wide = up(p.width, BI) * (r1 * v + v1 * r1), tall = up(p.width, BJ) * (r2 * v + up(p.classes, BI) * r2) + (r2 - r1) * v * (ld + 512);
  return tall > 0.85 * wide || (r1 + v1) / BJ * obman_cdiv(p.width, BI) < 128;
}
static Keep keep_of(const obman_class_loss_params& p, void* mem) {
  Carve c{static_cast<char*>(mem)};
  Keep k;
  const int planes = p.type == F32 ? 2 : 1;
  k.ld = (int)up(p.width, 32);
  const long xr = up(p.rows, wide_of(p) ? BJ : BI), wr = up(p.classes, BI);  // (x has the rows of g)
  k.scales = c.take<float>(4);
  k.norm = k.scales + 2;
  k.lse = c.take<float2>(p.rows);
  k.rows = c.take<RowConst>(p.reduction ? p.rows : 0);
  k.xp = c.take<u16>(xr * k.ld * planes);
  k.wp = c.take<u16>(wr * k.ld * planes);
  k.x = {k.xp, xr};
  k.w = {k.wp, wr};
  k.bytes = c.at;
  return k;
}

// dynamic LDS of a kernel, allowed once per device
template <auto KERNEL, int BYTES>
static hipError_t allow_lds() {
  static std::atomic<unsigned> done{0};
  const int dev = current_device();
  if (done.load(std::memory_order_relaxed) >> dev & 1) return hipSuccess;
  const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(KERNEL), hipFuncAttributeMaxDynamicSharedMemorySize, BYTES);
  if (e == hipSuccess) done.fetch_or(1u << dev, std::memory_order_relaxed);
  return e;
}

// scoring of few rows: the table is read as it is
constexpr int FEW_BLOCKS = 512;
constexpr size_t FEW_LDS = 128 * 1024;  // of x: 32 rows of 4 KB, 64 of 2 KB
struct Few {
  float2* part;
  float *picked, *norm;
  int blocks, groups;
  size_t bytes, lds;
};
static bool few_of(const obman_class_loss_params& p, void* mem, Few* o) {
  Carve c{static_cast<char*>(mem)};
  const long tiles = (p.classes + 127) / 128;
  o->groups = p.rows <= 32 ? 1 : 2;
  o->blocks = (int)(tiles < FEW_BLOCKS ? tiles : FEW_BLOCKS);
  o->part = c.take<float2>((size_t)o->blocks * FEW);
  o->picked = c.take<float>(FEW);
  o->norm = c.take<float>(1);
  o->bytes = c.at;
  const int e = p.type == F32 ? 4 : 8;
  o->lds = (size_t)up(p.width, 2 * e) / e * (32 * o->groups) * 16;
  return p.rows <= FEW && o->lds <= FEW_LDS;
}
template <int TYPE, int G>
static int launch_few(const obman_class_loss_params& p, const Few& o, hipStream_t st) {
  const hipError_t a = allow_lds<few_kernel<TYPE, G>, (int)FEW_LDS>();
  if (a != hipSuccess) return (int)a;
  few_kernel<TYPE, G><<<o.blocks, 256, o.lds, st>>>(p.x, p.w, p.bias, p.target, p.target_wide, (int)p.rows, p.classes, p.width, o.part, o.picked);
  OBMAN_LAUNCH_CHECK();
  return 0;
}
template <int TYPE>
static int few(const obman_class_loss_params& p, const Few& o, float* loss, hipStream_t st) {
  const int e = o.groups == 1 ? launch_few<TYPE, 1>(p, o, st) : launch_few<TYPE, 2>(p, o, st);
  if (e) return e;
  few_join_kernel<<<1, 1024, 0, st>>>(o.part, o.blocks, (int)p.rows, p.classes, o.picked, p.target, p.target_wide, p.ignore_index, p.reduction, loss, o.norm);
  OBMAN_LAUNCH_CHECK();
  return 0;
}

struct Forward {
  float* max_part;
  float2* part;
  float* picked;
  double2* sums;
  int ti, row_blocks;
  size_t bytes;
};
static Forward forward_of(const obman_class_loss_params& p, void* mem) {
  Carve c{static_cast<char*>(mem)};
  Forward o;
  o.ti = obman_cdiv(p.classes, BI);
  o.row_blocks = obman_cdiv(p.rows, 64);
  o.max_part = c.take<float>(4 * MAX_PARTS);
  o.part = c.take<float2>((size_t)o.ti * p.rows);
  o.picked = c.take<float>(p.rows);
  o.sums = c.take<double2>(o.row_blocks);
  o.bytes = c.at;
  return o;
}

// Into how many parts the contractions of dx and dw are cut: the least time of their common launch in steps of 32, a part costing
// START steps more (its pipeline's start and its slab).  A CU does the steps of its two blocks at one rate, a single block at
// 1 / ALONE of it.  Up to two blocks a CU: the largest sum of the two; beyond: the work of all spread over the CUs, and half of a short
// block of unevenness.  (At 19 200 x 12 800 x 512 the measured times of ten cuts are 0.43 - 0.45 us per such step.)
constexpr double START = 15.0, ALONE = 1.2;
constexpr int CUS = 256;
struct Parts { int x, w; bool x_first; double steps; };
static double launch_steps(double n_long, double l_long, double n_short, double l_short) {
  const double n = n_long + n_short;
  if (n > 2 * CUS) {
    const double spread = (n_long * l_long + n_short * l_short) / CUS + 0.5 * (n_short > 0 ? l_short : l_long);
    return spread > 2.0 * l_long ? spread : 2.0 * l_long;  // a block beside another runs at half the CU's rate
  }
  const double first = n_long > 0 ? l_long : l_short;                                       // the CU of the first block
  if (n <= CUS) return first * ALONE;
  const double paired = n_long > CUS ? l_long : n_short > 0 ? l_short : l_long;            // its second block is block CUS
  return first + paired;
}
static Parts parts_of(long tiles_x, long k_x, long tiles_w, long k_w) {
  Parts best{1, 1, true, 0.0};
  double least = 0.0;
  for (int x = 1; x <= (tiles_x ? 32 : 1); ++x) {
    if (x > 1 && k_x / x < 256) break;
    for (int w = 1; w <= (tiles_w ? 32 : 1); ++w) {
      if (w > 1 && k_w / w < 256) break;
      const double lx = k_x / 32 / x + START, lw = k_w / 32 / w + START, nx = (double)tiles_x * x, nw = (double)tiles_w * w;
      const bool first = !tiles_w || (tiles_x && lx >= lw);
      const double t = first ? launch_steps(nx, lx, nw, lw) : launch_steps(nw, lw, nx, lx);
      if (least == 0.0 || t < least) { least = t; best = {x, w, first, t}; }
    }
  }
  return best;
}

struct Backward {
  RowConst* rows;
  float *alpha, *row_max;
  u16* g;
  long piece;
  float *dx_slabs, *dw_slabs, *sums;
  Parts parts;
  size_t bytes;
};
static Backward backward_of(const obman_class_loss_params& p, const Keep& k, void* mem, bool need_x, bool need_w, bool need_b) {
  Carve c{static_cast<char*>(mem)};
  Backward o;
  const int planes = p.type == F32 ? 2 : 1, terms = p.type == F32 ? 3 : 1, ld = k.ld;
  const long xr = k.x.rows, all = up(p.classes, 32);
  o.rows = c.take<RowConst>(p.reduction ? 0 : p.rows);
  o.alpha = c.take<float>(1);
  o.row_max = c.take<float>(p.reduction ? 0 : ROW_MAX_BLOCKS);
  const int of_width = wide_of(p) ? BI : BJ, of_rows = BI + BJ - of_width;
  const long tiles_d = obman_cdiv(ld, of_width), tiles_x = need_x ? tiles_d * obman_cdiv(p.rows, of_rows) : 0;
  const auto cut = [&](long piece) { return parts_of(tiles_x, piece * terms, need_w ? tiles_d * obman_cdiv(piece, of_rows) : 0, xr * terms); };
  long most = PIECE_BYTES / (xr * 2 * planes) / BI * BI;
  if (most < 2 * BI) most = 2 * BI;
  o.piece = all;
  if (most < all) {  // equal pieces; of a few numbers of them the one whose launches fill the CUs best
    const long least = (all + most - 1) / most;
    double best = 0.0;
    for (long n = least; n < least + 6; ++n) {
      const long piece = up(all / n + 1, BI);
      if (piece > most && n > least) continue;
      const double t = cut(piece).steps * ((all + piece - 1) / piece);
      if (best == 0.0 || t < best) { best = t; o.piece = piece; }
    }
  }
  if (o.piece > all) o.piece = all;
  o.parts = cut(o.piece);
  o.g = c.take<u16>((size_t)planes * xr * o.piece);
  o.dx_slabs = c.take<float>(need_x ? (size_t)o.parts.x * p.rows * ld : 0);
  o.dw_slabs = c.take<float>(need_w ? (size_t)o.parts.w * o.piece * ld : 0);
  o.sums = c.take<float>(need_b ? (size_t)(xr / BJ) * o.piece : 0);
  o.bytes = c.at;
  return o;
}

static int blocks_for(long items) {
  const long b = (items + 255) / 256;
  return (int)(b < 1 ? 1 : b > 8192 ? 8192 : b);
}

static Gemm gemm_of(const Keep& keep, const Side& a, const Side& b, long ni, long nj, long k, int parts, int na, int nb) {
  return Gemm{a, b, ni, nj, k, up((k + parts - 1) / parts, 32), obman_cdiv(ni, BI), obman_cdiv(nj, BJ), parts, na, nb, keep.scales + FULL_AT};
}
template <int T, bool SPLIT, class Epi>
static int launch_logits(const Gemm& g, const Epi& epi, hipStream_t st) {
  const hipError_t a = allow_lds<logits_kernel<T, SPLIT, Epi>, LDS_BYTES>();
  if (a != hipSuccess) return (int)a;
  logits_kernel<T, SPLIT, Epi><<<g.ti * g.tj, WAVES * 64, LDS_BYTES, st>>>(g, epi);
  OBMAN_LAUNCH_CHECK();
  return 0;
}

static int operands(const obman_class_loss_params& p, const Keep& k, float* max_part, hipStream_t st) {
  if (p.type == F32) {
    absmax_kernel<<<dim3(MAX_PARTS, 2), 256, 0, st>>>(static_cast<const float*>(p.x), p.rows, static_cast<const float*>(p.w), p.classes, p.width, p.target, p.target_wide,
                                                      p.ignore_index, max_part);
    OBMAN_LAUNCH_CHECK();
  }
  const Pack px{p.x, k.xp, p.rows, k.x.rows}, pw{p.w, k.wp, p.classes, k.w.rows};
  const long rows = px.padded > pw.padded ? px.padded : pw.padded;
  const dim3 grid(blocks_for(rows * k.ld / 8), 2);
  if (p.type == F32) pack_kernel<F32><<<grid, 256, 0, st>>>(px, pw, p.width, k.ld / 8, p.target, p.target_wide, p.ignore_index, max_part, k.scales);
  else if (p.type == BF16) pack_kernel<BF16><<<grid, 256, 0, st>>>(px, pw, p.width, k.ld / 8, p.target, p.target_wide, p.ignore_index, max_part, k.scales);
  else pack_kernel<F16><<<grid, 256, 0, st>>>(px, pw, p.width, k.ld / 8, p.target, p.target_wide, p.ignore_index, max_part, k.scales);
  OBMAN_LAUNCH_CHECK();
  return 0;
}

static int check(const obman_class_loss_params* p) {
  if (!p || !p->target) return -1;
  if (p->rows <= 0 || p->classes <= 0 || p->width <= 0 || p->width > 16384) return -2;
  if (p->rows > MOST_ROWS || p->classes > MOST_ROWS) return -2;
  if (p->type < 0 || p->type > 2 || p->reduction < 0 || p->reduction > 2) return -3;
  return 0;
}

// |g| in 16 bits: scaled in fp16
static GScale g_scale_of(int type, const Keep& k) { return GScale{type == BF16 ? 1.f : G_SCALE, type == F32 ? k.scales + FULL_AT : nullptr}; }

// Pieces of the classes again, but only for the launch: it may have fewer than 2^32 threads.
constexpr long MOST_BLOCKS = 1L << 23;
template <int T, bool SPLIT>
static int forward(const obman_class_loss_params& p, const Keep& k, const Forward& o, hipStream_t st) {
  const long per = MOST_BLOCKS / obman_cdiv(p.rows, BJ);  // tiles of classes a launch: 256 for the most rows
  for (long t0 = 0; t0 < o.ti; t0 += per) {
    const long v0 = t0 * BI, nv = p.classes - v0 < per * BI ? p.classes - v0 : per * BI;
    const Side w{k.wp + v0 * 32, k.w.rows};
    const Stats<SPLIT> epi{{Scale{SPLIT ? k.scales : nullptr, SPLIT ? k.scales + 1 : nullptr}, p.bias, p.type, v0, p.classes}, p.target, p.target_wide, o.part + t0 * p.rows, o.picked};
    if (const int e = launch_logits<T, SPLIT>(gemm_of(k, w, k.x, nv, p.rows, k.ld, 1, 0, 0), epi, st)) return e;
  }
  return 0;
}

template <int T, bool SPLIT, bool WIDE>
static int backward(const obman_class_loss_params& p, const Keep& k, const Backward& o, const RowConst* rows, const Alpha& alpha, void* dx, void* dw, void* db, hipStream_t st) {
  const float *sx = SPLIT ? k.scales : nullptr, *sw = SPLIT ? k.scales + 1 : nullptr;
  const long xr = k.x.rows;
  const int ld = k.ld, size = p.type == F32 ? 4 : 2;
  const hipError_t a = allow_lds<grads_kernel<T, SPLIT, WIDE>, LDS_BYTES>();
  if (a != hipSuccess) return (int)a;
  for (long v0 = 0; v0 < p.classes; v0 += o.piece) {
    const long nv = p.classes - v0 < o.piece ? p.classes - v0 : o.piece, kv = up(nv, 32);
    const bool last = v0 + nv == p.classes;
    const Side w{k.wp + v0 * 32, k.w.rows}, gs{o.g, xr};
    const Grad<T, SPLIT> ge{{Scale{sx, sw}, p.bias, p.type, v0, v0 + nv}, rows, p.rows, xr, o.g, (int)kv, db ? o.sums : nullptr};
    if (const int e = launch_logits<T, SPLIT>(gemm_of(k, w, k.x, kv, xr, ld, 1, 0, 0), ge, st)) return e;
    const int d = ld / Step<SPLIT>, v = (int)(kv / Step<SPLIT>);  // column blocks of the operands and of g
    const Gemm gx = WIDE ? gemm_of(k, w, gs, ld, p.rows, kv, o.parts.x, d, 0) : gemm_of(k, gs, w, p.rows, ld, kv, o.parts.x, 0, d);
    const Gemm gw = WIDE ? gemm_of(k, k.x, gs, ld, nv, xr, o.parts.w, d, v) : gemm_of(k, gs, k.x, nv, ld, xr, o.parts.w, v, d);
    const int nx = dx ? gx.ti * gx.tj * gx.parts : 0, nw = dw ? gw.ti * gw.tj * gw.parts : 0;
    if (nx + nw) {
      const int second = o.parts.x_first ? nw : nx, first = nx + nw - second;
      grads_kernel<T, SPLIT, WIDE><<<((first + 7) & ~7) + second, WAVES * 64, LDS_BYTES, st>>>(gx, Slab{o.dx_slabs, p.rows * ld, ld, v0 > 0}, nx, gw,
                                                                                               Slab{o.dw_slabs, o.piece * ld, ld, 0}, nw, o.parts.x_first);
      OBMAN_LAUNCH_CHECK();
    }
    const Finish fx{o.dx_slabs, o.parts.x, p.rows * ld, dx && last ? p.rows : 0, sw, dx};
    const Finish fw{o.dw_slabs, o.parts.w, o.piece * ld, dw ? nv : 0, sx, static_cast<char*>(dw) + (size_t)v0 * p.width * size};
    const FinishBias fb{o.sums, (int)(xr / BJ), (int)kv, db ? nv : 0, static_cast<char*>(db) + (size_t)v0 * size};
    const long most = (fx.rows > fw.rows ? fx.rows : fw.rows) * ((p.width + 3) / 4);
    if (most || db) {
      finish_kernel<<<dim3(blocks_for(most > fb.classes ? most : fb.classes), db ? 3 : 2), 256, 0, st>>>(fx, fw, fb, ld, p.width, alpha, p.type);
      OBMAN_LAUNCH_CHECK();
    }
  }
  return 0;
}

// Up to here every block of rows_kernel looks for the largest weight itself: 8 192 rows take 5.6 us, against 2.8 + 3.5 and a launch more;
// 65 536 would take about 36 against 3.0 + 3.5.
constexpr long SCAN_ROWS = 8192;
constexpr long WHOLE_ROWS = 512, WHOLE_PARTS = 16384;  // what one block joins: a second launch costs more than the idle CUs

}  // namespace cl

extern "C" {

int obman_class_loss_sizes(const obman_class_loss_params* p, int keeps, int need_x, int need_w, int need_b, long* keep_bytes, long* fwd_bytes, long* bwd_bytes) {
  const int e = cl::check(p);
  if (e) return e;
  if (!keep_bytes || !fwd_bytes || !bwd_bytes) return -1;
  const cl::Keep k = cl::keep_of(*p, nullptr);
  cl::Few few;
  *keep_bytes = (long)k.bytes;
  *fwd_bytes = !keeps && cl::few_of(*p, nullptr, &few) ? (long)few.bytes : (long)(cl::forward_of(*p, nullptr).bytes + (keeps ? 0 : k.bytes));
  *bwd_bytes = (long)cl::backward_of(*p, k, nullptr, need_x, need_w, need_b).bytes;
  return 0;
}

int obman_class_loss_fwd(const obman_class_loss_params* p, void* keep, void* ws, float* loss, obman_stream_t stream) {
  int e = cl::check(p);
  if (e) return e;
  if (!p->x || !p->w || !ws || !loss) return -1;
  hipStream_t st = (hipStream_t)stream;
  cl::Few few;
  if (!keep && cl::few_of(*p, ws, &few))
    return p->type == cl::F32    ? cl::few<cl::F32>(*p, few, loss, st)
           : p->type == cl::BF16 ? cl::few<cl::BF16>(*p, few, loss, st)
                                 : cl::few<cl::F16>(*p, few, loss, st);
  const cl::Keep k = cl::keep_of(*p, keep ? keep : static_cast<char*>(ws) + cl::forward_of(*p, nullptr).bytes);
  const cl::Forward o = cl::forward_of(*p, ws);
  if ((e = cl::operands(*p, k, o.max_part, st))) return e;
  e = p->type == cl::F32    ? cl::forward<cl::F16, true>(*p, k, o, st)
      : p->type == cl::BF16 ? cl::forward<cl::BF16, false>(*p, k, o, st)
                            : cl::forward<cl::F16, false>(*p, k, o, st);
  if (e) return e;
  cl::RowConst* consts = keep && p->reduction ? k.rows : nullptr;
  const cl::GScale gs = cl::g_scale_of(p->type, k);
  if (p->rows <= cl::WHOLE_ROWS && p->rows * o.ti <= cl::WHOLE_PARTS) {
    cl::join_rows_kernel<true><<<1, 1024, 0, st>>>(o.part, o.ti, p->rows, p->classes, o.picked, p->target, p->target_wide, p->ignore_index, p->reduction, gs, k.lse, loss,
                                                   consts, nullptr, k.norm);
    OBMAN_LAUNCH_CHECK();
    return 0;
  }
  cl::join_rows_kernel<false><<<o.row_blocks, 256, 0, st>>>(o.part, o.ti, p->rows, p->classes, o.picked, p->target, p->target_wide, p->ignore_index, p->reduction, gs, k.lse,
                                                            loss, consts, o.sums, nullptr);
  OBMAN_LAUNCH_CHECK();
  if (p->reduction) {
    cl::reduce_kernel<<<1, 256, 0, st>>>(o.sums, o.row_blocks, p->reduction == 2, loss, k.norm);
    OBMAN_LAUNCH_CHECK();
  }
  return 0;
}

int obman_class_loss_bwd(const obman_class_loss_params* p, const void* keep, const float* g_loss, void* ws, void* dx, void* dw, void* db, obman_stream_t stream) {
  const int e = cl::check(p);
  if (e) return e;
  if (!keep || !ws || !g_loss) return -1;
  if (!dx && !dw && !db) return 0;
  hipStream_t st = (hipStream_t)stream;
  const cl::Keep k = cl::keep_of(*p, const_cast<void*>(keep));
  const cl::Backward o = cl::backward_of(*p, k, ws, dx != nullptr, dw != nullptr, db != nullptr);
  const cl::GScale gs = cl::g_scale_of(p->type, k);
  cl::Alpha alpha{g_loss, k.norm, gs};
  if (!p->reduction) {
    const bool split = p->rows > cl::SCAN_ROWS;
    if (split) {
      cl::row_max_kernel<<<cl::ROW_MAX_BLOCKS, 1024, 0, st>>>(p->target, p->target_wide, p->ignore_index, p->rows, g_loss, o.row_max);
      OBMAN_LAUNCH_CHECK();
    }
    cl::rows_kernel<<<obman_cdiv(p->rows, 1024), 1024, 0, st>>>(k.lse, p->target, p->target_wide, p->ignore_index, p->rows, g_loss, split ? o.row_max : nullptr, gs, o.rows,
                                                                o.alpha);
    OBMAN_LAUNCH_CHECK();
    alpha = cl::Alpha{o.alpha, nullptr, gs};
  }
  const cl::RowConst* rows = p->reduction ? k.rows : o.rows;
  if (cl::wide_of(*p))
    return p->type == cl::F32    ? cl::backward<cl::F16, true, true>(*p, k, o, rows, alpha, dx, dw, db, st)
           : p->type == cl::BF16 ? cl::backward<cl::BF16, false, true>(*p, k, o, rows, alpha, dx, dw, db, st)
                                 : cl::backward<cl::F16, false, true>(*p, k, o, rows, alpha, dx, dw, db, st);
  return p->type == cl::F32    ? cl::backward<cl::F16, true, false>(*p, k, o, rows, alpha, dx, dw, db, st)
         : p->type == cl::BF16 ? cl::backward<cl::BF16, false, false>(*p, k, o, rows, alpha, dx, dw, db, st)
                               : cl::backward<cl::F16, false, false>(*p, k, o, rows, alpha, dx, dw, db, st);
}

}  // extern "C"
