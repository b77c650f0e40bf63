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
// lo*hi + hi*lo + hi*hi: 2^-22 relative, an element 2^27 below the tensor's largest still has 11 bits, and three fp16 products are
// 5 times the rate of the fp32 matrix instruction.  g has |g| <= max |c|: in fp16 it is scaled to 2^14.  Rounding g to 16 bits (its own
// size, before sums of many rows or classes) costs as much again as rounding the result.
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
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));

enum { F32 = 0, BF16 = 1, F16 = 2 };

constexpr int BI = 256, BJ = 128, BK = 32;  // tile: 256 x 128, four waves of 128 x 64; 72 KB of LDS, so two blocks share a CU and one's
constexpr int STAGES = 3;                    // epilogue runs beside the other's products
constexpr int A_BYTES = BI * BK * 2, B_BYTES = BJ * BK * 2, STAGE_BYTES = A_BYTES + B_BYTES;
constexpr int LDS_BYTES = STAGES * STAGE_BYTES + BI * 4;
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr float G_SCALE = 16384.f;  // |g| / max|c| <= 1 in fp16

struct Gemm {
  const u16 *a, *b;          // [planes][rows][ld]
  long a_plane, b_plane;     // elements from the hi to the lo plane
  long a_rows, b_rows;       // rows of memory (a contiguous-k operand: its i or j extent; else: its k extent)
  int lda, ldb;
  long ni, nj;               // extents of the result
  long k;                    // contraction, a multiple of 32
  long k_split;              // of it per block row of the grid's second axis
  int ti, tj;                // tiles
  int k_tail;                // 0, or how many k rows of a are there in the last step (A_KR)
};

__device__ __forceinline__ void dma16(__amdgpu_buffer_rsrc_t r, unsigned lds, unsigned voff) {
  // lane l writes 16 bytes at lds + 16 l
  asm volatile("s_mov_b32 m0, %0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds), "v"(voff), "s"(r) : "memory", "m0");
}

// One operand's tile: R rows (i or j) x 32 k.  KC: k contiguous in memory, LDS [row][64 bytes]; KR: a memory row is one k, LDS
// [k][2 R bytes].  16-byte chunks are placed at (chunk ^ f(row)) so that neither the wide reads of KC (f = row >> 2 & 3) nor the
// transposing reads of KR (f = 4 (k & 3)) meet in a bank; the DMA writes LDS linearly, so the source address carries the swizzle.
// Every address is inside the operand: rows (KC) or columns (KR) behind the extent repeat the last ones and their results are not kept.
template <bool KR, int R>
struct Operand {
  static constexpr int N = R * BK * 2 / 1024 / 4;  // wave-wide loads per wave and step
  static constexpr int C = R / 8;                  // chunks of a k row (KR)
  const u16* base;  // at the next step's k
  long plane, rows, row0;
  int ld;
  unsigned voff[N];
  __device__ __forceinline__ void init(const u16* p, long plane_, long rows_, int ld_, long row0_, int wave, int lane) {
    base = p; plane = plane_; rows = rows_; ld = ld_; row0 = row0_;
#pragma unroll
    for (int q = 0; q < N; ++q) {
      const int at = wave * N + q;
      if constexpr (!KR) {
        const int row = at * 16 + (lane >> 2), c = (lane & 3) ^ ((lane >> 4) & 3);
        const long left = rows - 1 - row0;
        voff[q] = (unsigned)((row < left ? row : left) * ld * 2 + c * 16);
      } else {
        const int k = at * (64 / C) + lane / C, c = (lane % C) ^ ((k & 3) << 2);
        const int last = (int)(ld - row0) / 8 - 1;
        voff[q] = (unsigned)(k * ld * 2 + (c < last ? c : last) * 16);
      }
    }
  }
  __device__ __forceinline__ const u16* at(const u16* p, int pl, long k) const {
    return p + (pl ? plane : 0) + (KR ? k * ld + row0 : row0 * ld + k);
  }
  __device__ __forceinline__ void issue(unsigned lds, int wave, int lane, bool tail, int k_left) {
    const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(const_cast<u16*>(base), 0, 0x7ffffff0, 0x00020000);
    const unsigned to = lds + wave * (N * 1024);
    if (KR && tail) {  // the table's last rows: the last one again, where the other operand is zero
#pragma unroll
      for (int q = 0; q < N; ++q) {
        const int k = (wave * N + q) * (64 / C) + lane / C;
        dma16(r, to + q * 1024, voff[q] - (unsigned)((k >= k_left ? k - k_left + 1 : 0) * ld * 2));
      }
    } else {
#pragma unroll
      for (int q = 0; q < N; ++q) dma16(r, to + q * 1024, voff[q]);
    }
    base += KR ? (long)BK * ld : BK;
  }
};

// fragment of 32 rows x 16 k: lane -> row lane % 32, k = 8 (lane / 32) .. + 7
template <bool KR, int R>
struct Frag {
  unsigned off[KR ? 4 : 2];
  __device__ __forceinline__ void init(int first_row, int lane) {  // first_row: a multiple of 64 (of 128 where four fragments are read)
    if constexpr (!KR) {
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) off[ks] = (first_row + (lane & 31)) * 64 + ((2 * ks + (lane >> 5)) ^ ((lane >> 2) & 3)) * 16;
    } else {
      const int k = 8 * (lane >> 5) + ((lane & 15) >> 2), kk = k & 3;
#pragma unroll
      for (int f = 0; f < 4; ++f) {
        const int chunk = ((first_row / 8 + f * 4) ^ (kk << 2)) + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
        off[f] = k * (R * 2) + chunk * 16 + (lane & 1) * 8;
      }
    }
  }
  __device__ __forceinline__ u32x4 read(const char* tile, int f, int ks, int lane) const {
    if constexpr (!KR) {
      return *reinterpret_cast<const u32x4*>(tile + off[ks] + f * 2048);
    } else {
      const char* p = tile + off[f] + ks * 16 * (R * 2);
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(p));
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(p + 4 * (R * 2)));
      return __builtin_bit_cast(u32x4, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    }
  }
};

template <int T>
__device__ __forceinline__ f32x16 mfma(u32x4 a, u32x4 b, f32x16 c) {
  if constexpr (T == BF16) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
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

// Consecutive ids of one XCD (ids go round the eight) take consecutive tiles; tiles run 8 j wide, so that what an XCD's CUs work on
// at a time (8 x 8 tiles: 3 MB of operands at width 512) stays in its 4 MB L2.
__device__ __forceinline__ void tile_of(const Gemm& g, int& i, int& j) {
  const int n = g.ti * g.tj, id = blockIdx.x, x = id & 7, q = n >> 3, rem = n & 7;
  const int v = x * q + (x < rem ? x : rem) + (id >> 3);
  const int per = 8 * g.ti, group = v / per, in = v - group * per;
  const int w = g.tj - group * 8 < 8 ? g.tj - group * 8 : 8;
  i = in / w;
  j = group * 8 + in % w;
}

// what the epilogues need to know about the scaling of split operands: exponents on the device
struct Scale {
  const float* a;  // NULL = 1; else the power of two that operand was multiplied by
  const float* b;
  __device__ __forceinline__ float inverse() const { return (a ? 1.f / *a : 1.f) * (b ? 1.f / *b : 1.f); }
};

struct Ctx {
  long i0, j0;
  int wi, wj, lane, wave, tid, ti_index, split;
  char* smem;
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
    return reinterpret_cast<const float*>(c.smem + STAGES * STAGE_BYTES) + c.wi * 128 + 4 * (c.lane >> 5);
  }
  __device__ __forceinline__ void before(const Ctx& c, f32x16 (&acc)[4][2]) const {
    const long v0 = class0 + c.i0;
    const bool plain = !bias && v0 + BI <= classes;
    if (SPLIT || !plain) {
      const long v = v0 + c.tid;
      reinterpret_cast<float*>(c.smem + STAGES * STAGE_BYTES)[c.tid] = v >= classes ? -INFINITY : bias ? load_one(bias, type, v) : 0.f;
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

// forward: per row (j) and tile of classes (i) the maximum and the sum of exponentials
template <bool SPLIT>
struct Stats {
  Bias<SPLIT> bias;
  const void* target;
  int target_wide;
  float2* part;  // [ti][rows]
  float* picked; // [rows]
  __device__ __forceinline__ void before(const Gemm&, const Ctx& c, f32x16 (&acc)[4][2]) const { bias.before(c, acc); }
  __device__ __forceinline__ void after(const Gemm& g, const Ctx& c, f32x16 (&acc)[4][2]) const {
    float2* red = reinterpret_cast<float2*>(c.smem);
    bias.finish(c, acc);
    float m[2], sum[2];
#pragma unroll
    for (int fj = 0; fj < 2; ++fj) {
      const long r = c.j0 + c.wj * 64 + fj * 32 + (c.lane & 31);
      const int t = target_at(r < g.nj ? target_of(target, target_wide, r) : -1, c.i0 + c.wi * 128, c.lane);
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
      const float ref = top == -INFINITY ? 0.f : top * LOG2E;
      float part4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int fi = 0; fi < 4; ++fi)
#pragma unroll
        for (int q = 0; q < 16; ++q) part4[q & 3] += __builtin_amdgcn_exp2f(__builtin_fmaf(acc[fi][fj][q], LOG2E, -ref));
      float total = (part4[0] + part4[1]) + (part4[2] + part4[3]);
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
        const float top = fmaxf(m[fj], o.x), ref = top == -INFINITY ? 0.f : top * LOG2E;
        const float total = sum[fj] * __builtin_amdgcn_exp2f(m[fj] * LOG2E - ref) + o.y * __builtin_amdgcn_exp2f(o.x * LOG2E - ref);
        if (r < g.nj) part[(long)c.ti_index * g.nj + r] = make_float2(top, total);
      }
    }
  }
};

struct RowConst {  // per row of the backward pass
  float lse2;      // (lse - log |c|) in units of log 2, +inf for a row without a gradient: g = exp2(z - lse2) is p |c| in one step
  float c;         // |c|
  int target;      // -1: none
  unsigned sign;   // 0x80008000 where c < 0: the sign of two 16-bit values
};

// backward: g of a piece of the classes, [rows_padded][ld] in 16 bits
template <int T, bool SPLIT>
struct Grad {
  Bias<SPLIT> bias;
  const RowConst* rows;
  long rows_padded;
  u16* out;
  long plane;
  int ld;
  __device__ __forceinline__ void before(const Gemm&, const Ctx& c, f32x16 (&acc)[4][2]) const { bias.before(c, acc); }
  __device__ __forceinline__ void after(const Gemm& g, const Ctx& c, f32x16 (&acc)[4][2]) const {
    bias.finish(c, acc);
#pragma unroll
    for (int fj = 0; fj < 2; ++fj) {
      const long r = c.j0 + c.wj * 64 + fj * 32 + (c.lane & 31);
      RowConst k = {INFINITY, 0.f, -1, 0};
      if (r < g.nj) k = rows[r];
      const int t = target_at(k.target, bias.class0 + c.i0 + c.wi * 128, c.lane);
#pragma unroll
      for (int fi = 0; fi < 4; ++fi)
#pragma unroll
        for (int q = 0; q < 16; ++q) acc[fi][fj][q] = __builtin_amdgcn_exp2f(__builtin_fmaf(acc[fi][fj][q], LOG2E, -k.lse2));
      if (__any(t >= 0)) {
#pragma unroll
        for (int fi = 0; fi < 4; ++fi)
#pragma unroll
          for (int q = 0; q < 16; ++q) acc[fi][fj][q] -= t == fi * 32 + (q >> 2) * 8 + (q & 3) ? k.c : 0.f;
      }
      // lanes l and l + 32 hold classes 0 .. 3 and 4 .. 7 of each 8: an exchange gives each 8 in a row, 16 bytes
      u16* o = out + r * ld + (c.i0 + c.wi * 128 + 8 * (c.lane >> 5));
#pragma unroll
      for (int fi = 0; fi < 4; ++fi)
#pragma unroll
        for (int q = 0; q < 4; q += 2) {
          const int at = fi * 32 + q * 8;
          unsigned hi[2][2], lo[2][2];
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float x = acc[fi][fj][(q + u) * 4 + e * 2], y = acc[fi][fj][(q + u) * 4 + e * 2 + 1];
              const u16 hx = narrow<T>(x), hy = narrow<T>(y);
              hi[u][e] = (hx | (unsigned)hy << 16) ^ k.sign;
              if constexpr (SPLIT) lo[u][e] = (narrow<T>(x - widen<T>(hx)) | (unsigned)narrow<T>(y - widen<T>(hy)) << 16) ^ k.sign;
            }
          const bool keep = r < rows_padded && c.i0 + c.wi * 128 + at + 8 * (c.lane >> 5) < ld;
          {
            const u32x2 s0 = __builtin_amdgcn_permlane32_swap(hi[0][0], hi[1][0], false, false);
            const u32x2 s1 = __builtin_amdgcn_permlane32_swap(hi[0][1], hi[1][1], false, false);
            if (keep) *reinterpret_cast<u32x4*>(o + at) = u32x4{s0[0], s1[0], s0[1], s1[1]};
          }
          if constexpr (SPLIT) {
            const u32x2 s0 = __builtin_amdgcn_permlane32_swap(lo[0][0], lo[1][0], false, false);
            const u32x2 s1 = __builtin_amdgcn_permlane32_swap(lo[0][1], lo[1][1], false, false);
            if (keep) *reinterpret_cast<u32x4*>(o + plane + at) = u32x4{s0[0], s1[0], s0[1], s1[1]};
          }
        }
    }
  }
};

// a product's result: fp32 slabs [split][nj][ld], added to what is there or not
struct Slab {
  float* out;
  long slab;
  int ld, add;
  __device__ __forceinline__ void before(const Gemm&, const Ctx&, f32x16 (&acc)[4][2]) const { clear(acc); }
  __device__ __forceinline__ void after(const Gemm& g, const Ctx& c, f32x16 (&acc)[4][2]) const {
    float* o = out + c.split * slab;
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
          if (add) v += *p;
          *p = v;
        }
    }
  }
};

// C[i, j] = sum_k A(i, k) B(j, k); TERMS = 3: both operands in two planes
template <bool A_KR, bool B_KR, int T, int TERMS, class Epi>
__global__ __launch_bounds__(256, 2) void gemm_kernel(Gemm g, Epi epi) {
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int bi, bj;
  tile_of(g, bi, bj);
  bi = __builtin_amdgcn_readfirstlane(bi);
  bj = __builtin_amdgcn_readfirstlane(bj);
  const Ctx ctx{(long)bi * BI, (long)bj * BJ, wave & 1, wave >> 1, lane, wave, tid, bi, (int)blockIdx.y, smem};
  Operand<A_KR, BI> oa;
  Operand<B_KR, BJ> ob;
  oa.init(g.a, g.a_plane, g.a_rows, g.lda, ctx.i0, wave, lane);
  ob.init(g.b, g.b_plane, g.b_rows, g.ldb, ctx.j0, wave, lane);
  Frag<A_KR, BI> fa;
  Frag<B_KR, BJ> fb;
  fa.init(ctx.wi * 128, lane);
  fb.init(ctx.wj * 64, lane);
  const long kb = (long)blockIdx.y * g.k_split, ke = kb + g.k_split < g.k ? kb + g.k_split : g.k;
  const int steps = ke > kb ? (int)((ke - kb) / BK) * TERMS : 0;
  const unsigned lds0 = (unsigned)(size_t)(__attribute__((address_space(3))) char*)smem;

  f32x16 acc[4][2];
  epi.before(g, ctx, acc);
  int term = TERMS == 3 ? 0 : 2, left = (int)((ke - kb) / BK);  // terms: lo hi, hi lo, hi hi
  const int per_term = left;
  oa.base = oa.at(g.a, term == 0, kb);
  ob.base = ob.at(g.b, term == 1, kb);
  const bool tail = g.k_tail && ke == g.k;  // the last step runs over the end of the table
  unsigned to = lds0;
  const auto issue = [&]() {
    oa.issue(to, wave, lane, A_KR && tail && left == 1, g.k_tail);
    ob.issue(to + A_BYTES, wave, lane, false, 0);
    to = to == lds0 + (STAGES - 1) * STAGE_BYTES ? lds0 : to + STAGE_BYTES;
    --left;
    if (TERMS == 3 && left == 0) {
      left = per_term;
      ++term;
      oa.base = oa.at(g.a, 0, kb);
      ob.base = ob.at(g.b, term == 1, kb);
    }
  };
  constexpr int PER = Operand<A_KR, BI>::N + Operand<B_KR, BJ>::N;
  static_assert(PER == 6, "the counted wait below");
  if (steps > 0) issue();
  if (steps > 1) issue();
  const char* from = smem;
  for (int s = 0; s < steps; ++s) {
    // step s has arrived for every wave (only step s + 1 may still be under way), and every wave has read step s - 1, whose slot is next
    if (s + 1 < steps) asm volatile("s_waitcnt vmcnt(6) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    u32x4 a[2][4], b[2][2];
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
#pragma unroll
      for (int f = 0; f < 2; ++f) b[ks][f] = fb.read(from + A_BYTES, f, ks, lane);
#pragma unroll
      for (int f = 0; f < 4; ++f) a[ks][f] = fa.read(from, f, ks, lane);
    }
    if (s + 2 < steps) issue();
    from = from == smem + (STAGES - 1) * STAGE_BYTES ? smem : from + STAGE_BYTES;
    __builtin_amdgcn_sched_barrier(0);  // all reads go out before the first product waits for one
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
#pragma unroll
      for (int f = 0; f < 4; ++f)
#pragma unroll
        for (int h = 0; h < 2; ++h) acc[f][h] = mfma<T>(a[ks][f], b[ks][h], acc[f][h]);
    __builtin_amdgcn_s_setprio(0);
    __builtin_amdgcn_sched_barrier(0);
  }
  __syncthreads();
  epi.after(g, ctx, acc);
}

// ------------------------------------------------------------------------------------------------------- operands and rows

// largest finite |x| of the kept rows: 256 block maxima
__global__ __launch_bounds__(256) void absmax_kernel(const float* __restrict__ x, long rows, int width, const void* target, int wide, long ignore, float* __restrict__ part) {
  float m = 0.f;
  const long n = rows * width;
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < n; i += 256L * 256) {
    const float a = fabsf(x[i]);
    if (a > m && a < INFINITY && (!target || target_of(target, wide, i / width) != ignore)) m = a;
  }
  m = obman_wave_max(m);
  __shared__ float red[4];
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
  __syncthreads();
  if (threadIdx.x == 0) part[blockIdx.x] = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
}

// the power of two that brings the largest element to 2^13 .. 2^14 (1 for an all-zero tensor)
__global__ __launch_bounds__(256) void scale_kernel(const float* __restrict__ part, float* __restrict__ scale) {
  float m = obman_wave_max(part[(size_t)blockIdx.x * 256 + threadIdx.x]);
  __shared__ float red[4];
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
  __syncthreads();
  if (threadIdx.x == 0) {
    m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    int e = 0;
    if (m > 0.f) (void)frexpf(m, &e);  // m = f 2^e, f in [0.5, 1)
    e = 14 - e;
    e = e > 126 ? 126 : e < -126 ? -126 : e;
    scale[blockIdx.x] = m > 0.f ? ldexpf(1.f, e) : 1.f;
  }
}

// rows of an operand into 16-bit planes [planes][rows_padded][ld]: zeros behind the width, for ignored rows and behind the last row;
// `ones`: column `width` is 1 (its product with g is the gradient of the bias)
template <int TYPE>
__global__ __launch_bounds__(256) void pack_kernel(const void* __restrict__ src, long rows, long rows_padded, int width, int ld, const void* target, int wide, long ignore,
                                                  int ones, const float* __restrict__ scale, u16* __restrict__ dst, long plane) {
  const int per = ld >> 3;
  const long n = rows_padded * per;
  const float sc = TYPE == F32 ? *scale : 1.f;
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long)gridDim.x * 256) {
    const long r = i / per;
    const int c = (int)(i - r * per) * 8;
    const bool keep = r < rows && (!target || target_of(target, wide, r) != ignore);
    u16 hi[8], lo[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) hi[e] = lo[e] = 0;
    if (keep) {
      const long at = r * width + c;
      if constexpr (TYPE == F32) {
        const float* p = static_cast<const float*>(src) + at;
        float v[8];
        if (c + 8 <= width) {
          const f32x4u a = *reinterpret_cast<const f32x4u*>(p), b = *reinterpret_cast<const f32x4u*>(p + 4);
#pragma unroll
          for (int e = 0; e < 4; ++e) { v[e] = a[e]; v[e + 4] = b[e]; }
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = c + e < width ? p[e] : 0.f;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float y = v[e] * sc;
          hi[e] = narrow<F16>(y);
          const float rest = y - widen<F16>(hi[e]);
          lo[e] = fabsf(y) < INFINITY ? narrow<F16>(rest) : (u16)0;
        }
      } else {
        const u16* p = static_cast<const u16*>(src) + at;
        if (c + 8 <= width) {
          const u16x8u a = *reinterpret_cast<const u16x8u*>(p);
#pragma unroll
          for (int e = 0; e < 8; ++e) hi[e] = a[e];
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) hi[e] = c + e < width ? p[e] : (u16)0;
        }
      }
      if (ones && width >= c && width < c + 8) hi[width - c] = TYPE == F32 ? narrow<F16>(1.f) : TYPE == BF16 ? narrow<BF16>(1.f) : narrow<F16>(1.f);
    }
    *reinterpret_cast<u32x4*>(dst + r * ld + c) = *reinterpret_cast<u32x4*>(hi);
    if constexpr (TYPE == F32) *reinterpret_cast<u32x4*>(dst + plane + r * ld + c) = *reinterpret_cast<u32x4*>(lo);
  }
}

// per row: join over the tiles of classes; loss per row, and per block of rows the sum of losses and the number of kept rows
__global__ __launch_bounds__(256) void join_rows_kernel(const float2* __restrict__ part, int tiles, long rows, long classes, const float* __restrict__ picked,
                                                       const void* target, int wide, long ignore, float* __restrict__ lse, float* __restrict__ loss,
                                                       double2* __restrict__ sums) {
  // 64 rows a block, four threads a row
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const long r = (long)blockIdx.x * 64 + lane;
  __shared__ float2 red[4][64];
  float m = -INFINITY, s = 0.f;
  if (r < rows)
    for (int t = w; t < tiles; t += 4) {
      const float2 p = part[(long)t * rows + r];
      const float top = fmaxf(m, p.x), ref = top == -INFINITY ? 0.f : top * LOG2E;
      s = s * __builtin_amdgcn_exp2f(m * LOG2E - ref) + p.y * __builtin_amdgcn_exp2f(p.x * LOG2E - ref);
      m = top;
    }
  red[w][lane] = make_float2(m, s);
  __syncthreads();
  if (w) return;
  double l = 0.0, kept = 0.0;
  if (r < rows) {
#pragma unroll
    for (int k = 1; k < 4; ++k) {
      const float2 p = red[k][lane];
      const float top = fmaxf(m, p.x), ref = top == -INFINITY ? 0.f : top * LOG2E;
      s = s * __builtin_amdgcn_exp2f(m * LOG2E - ref) + p.y * __builtin_amdgcn_exp2f(p.x * LOG2E - ref);
      m = top;
    }
    const long t = target_of(target, wide, r);
    float z = m + LN2 * __builtin_amdgcn_logf(s);  // v_log_f32: log2
    if (t != ignore && (t < 0 || t >= classes)) z = NAN;  // a label outside the table poisons the loss instead of being read
    lse[r] = z;
    const float row = t == ignore ? 0.f : z - (t >= 0 && t < classes ? picked[r] : 0.f);
    if (loss) loss[r] = row;
    l = row;
    kept = t != ignore;
  }
  if (sums) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) { l += __shfl_xor(l, off, 64); kept += __shfl_xor(kept, off, 64); }
    if (lane == 0) sums[blockIdx.x] = make_double2(l, kept);
  }
}

// loss = sum or mean over the kept rows (no row kept: 0); norm = what a row's gradient is multiplied by
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
  if (k < 1.0) k = 1.0;
  *loss = (float)(mean ? l / k : l);
  *norm = (float)(mean ? 1.0 / k : 1.0);
}

// backward constants: RowConst per row and alpha, the factor of every result.  g_loss: one value (sum, mean) or one per row, scaled
// here to at most 1 in magnitude by a power of two that alpha takes back
__global__ __launch_bounds__(1024) void rows_kernel(const float* __restrict__ lse, const void* target, int wide, long ignore, long rows, const float* __restrict__ g_loss,
                                                   int per_row, const float* __restrict__ norm, float g_scale, RowConst* __restrict__ out, float* __restrict__ alpha) {
  float top = 0.f;
  __shared__ float red[16];
  if (per_row) {  // every block finds the same maximum
    for (long r = threadIdx.x; r < rows; r += 1024) {
      const float a = fabsf(g_loss[r]);
      if (a > top && a < INFINITY && target_of(target, wide, r) != ignore) top = a;
    }
    top = obman_wave_max(top);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = top;
    __syncthreads();
    top = red[0];
#pragma unroll
    for (int w = 1; w < 16; ++w) top = fmaxf(top, red[w]);
  }
  int e = 0;
  if (top > 0.f) (void)frexpf(top, &e);
  e = e > 120 ? 120 : e < -120 ? -120 : e;
  const float up = ldexpf(1.f, e), down = ldexpf(1.f, -e);
  if (blockIdx.x == 0 && threadIdx.x == 0) *alpha = per_row ? up / g_scale : *g_loss * *norm / g_scale;
  const long r = (long)blockIdx.x * 1024 + threadIdx.x;
  if (r >= rows) return;
  const long t = target_of(target, wide, r);
  RowConst k;
  const float w = t == ignore ? 0.f : (per_row ? g_loss[r] * down : 1.f) * g_scale;
  k.c = fabsf(w);
  k.lse2 = w == 0.f ? INFINITY : lse[r] * LOG2E - log2f(k.c);
  k.target = w == 0.f || t < 0 || t > 0x7fffffffL ? -1 : (int)t;
  k.sign = w < 0.f ? 0x80008000u : 0u;
  out[r] = k;
}

// sum of the slabs times alpha into the gradient's own type; column `width` is the bias gradient
__global__ __launch_bounds__(256) void finish_kernel(const float* __restrict__ slabs, int n, long slab, long rows, int ld, int width, const float* __restrict__ alpha, Scale scale,
                                                    void* __restrict__ out, int type, void* __restrict__ bias_out) {
  const float k = *alpha * scale.inverse();
  const int per = ld >> 2;
  const long total = rows * per;
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long)gridDim.x * 256) {
    const long r = i / per;
    const int c = (int)(i - r * per) * 4;
    if (c > width || (c == width && !bias_out)) continue;
    const float* p = slabs + r * ld + c;
    f32x4 v = *reinterpret_cast<const f32x4*>(p);
    for (int s = 1; s < n; ++s) v += *reinterpret_cast<const f32x4*>(p + s * slab);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (c + e < width) { if (out) store_one(out, type, r * width + c + e, v[e] * k); }
      else if (c + e == width && bias_out) store_one(bias_out, type, r, v[e] * (*alpha));
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
constexpr int SLOTS = 512;                // blocks that run at a time: two per CU

struct Packed { u16* p; long plane; int ld; long rows; };

struct Work {
  // both directions
  float *max_part, *scales;
  Packed x, w;
  // forward
  float2* part;
  float* picked;
  double2* sums;
  int ti, row_blocks;
  // backward
  RowConst* rows;
  float* alpha;
  u16* g;
  long g_plane, piece;
  float *dx_slabs, *dw_slabs;
  int dx_split, dw_split;
  size_t bytes;
};

static bool in_place(const obman_class_loss_params& p, const void* q) {
  return p.type != F32 && p.width % BK == 0 && ((size_t)q & 15) == 0;
}

// Into how many parts the contraction is cut: the fewest step times of 32 over all rounds of the slots, a part costing START steps
// more (its pipeline's start and its slab)
constexpr long START = 40;
static int split_of(long tiles, long k) {
  long best = 0;
  int n = 1;
  for (int c = 1; c <= 64; ++c) {
    if (c > 1 && k / c < 256) break;
    const long t = (tiles * c + SLOTS - 1) / SLOTS * (k / BK / c + START);
    if (c == 1 || t < best) { best = t; n = c; }
  }
  return n;
}
static long split_len(long k, int n) { return up((k + n - 1) / n, BK); }

static Work plan(const obman_class_loss_params& p, void* ws, bool back, bool need_x, bool need_w, bool need_b) {
  Work o;
  Carve c{static_cast<char*>(ws)};
  const bool split = p.type == F32;
  const int planes = split ? 2 : 1;
  o.max_part = c.take<float>(split ? 512 : 0);
  o.scales = c.take<float>(4);
  const bool bias_col = back && need_b;
  const int ld = (int)up(p.width + (bias_col ? 1 : 0), BK);
  const bool wrap = !in_place(p, p.w) || ld != p.width, xpack = back || !in_place(p, p.x);
  const long xr = back ? up(p.rows, BK) : p.rows;
  o.x = {xpack ? c.take<u16>((size_t)planes * xr * ld) : nullptr, xr * ld, ld, xr};
  o.w = {wrap ? c.take<u16>((size_t)planes * p.classes * ld) : nullptr, p.classes * ld, ld, p.classes};
  if (!xpack) o.x = {static_cast<u16*>(const_cast<void*>(p.x)), 0, p.width, p.rows};
  if (!wrap) o.w = {static_cast<u16*>(const_cast<void*>(p.w)), 0, p.width, p.classes};
  if (!back) {
    o.ti = obman_cdiv(p.classes, BI);
    o.row_blocks = obman_cdiv(p.rows, 64);
    o.part = c.take<float2>((size_t)o.ti * p.rows);
    o.picked = c.take<float>(p.rows);
    o.sums = c.take<double2>(o.row_blocks);
  } else {
    o.rows = c.take<RowConst>(p.rows);
    o.alpha = c.take<float>(1);
    long piece = PIECE_BYTES / (xr * 2 * planes) / BI * BI;
    if (piece < 2 * BI) piece = 2 * BI;
    const long all = up(p.classes, BK);
    if (piece >= all) piece = all;
    else piece = up(up(p.classes, BK) / ((p.classes + piece - 1) / piece) + BI, BI);  // equal pieces
    o.piece = piece > all ? all : piece;
    o.g_plane = xr * o.piece;
    o.g = c.take<u16>((size_t)planes * xr * o.piece);
    const long dx_tiles = (long)obman_cdiv(ld, BI) * obman_cdiv(p.rows, BJ), dw_tiles = (long)obman_cdiv(ld, BI) * obman_cdiv(o.piece, BJ);
    o.dx_split = split_of(dx_tiles, o.piece);
    o.dw_split = split_of(dw_tiles, xr);
    o.dx_slabs = c.take<float>(need_x ? (size_t)o.dx_split * p.rows * ld : 0);
    o.dw_slabs = c.take<float>(need_w || need_b ? (size_t)o.dw_split * o.piece * ld : 0);
  }
  o.bytes = c.at;
  return o;
}

static int blocks_for(long items) {
  const long b = (items + 255) / 256;
  return (int)(b < 1 ? 1 : b > 8192 ? 8192 : b);
}

template <bool A_KR, bool B_KR, class Epi, int T, int TERMS>
static int launch_gemm(const Gemm& g, int splits, const Epi& epi, hipStream_t st) {
  static std::atomic<unsigned> done{0};
  const int dev = current_device();
  if (!(done.load(std::memory_order_relaxed) >> dev & 1)) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(gemm_kernel<A_KR, B_KR, T, TERMS, Epi>), hipFuncAttributeMaxDynamicSharedMemorySize, LDS_BYTES);
    if (e != hipSuccess) return (int)e;
    done.fetch_or(1u << dev, std::memory_order_relaxed);
  }
  gemm_kernel<A_KR, B_KR, T, TERMS, Epi><<<dim3(g.ti * g.tj, splits), 256, LDS_BYTES, st>>>(g, epi);
  OBMAN_LAUNCH_CHECK();
  return 0;
}

static int pack(const obman_class_loss_params& p, const void* src, long rows, const Packed& d, bool masked, bool ones, const float* scale, hipStream_t st) {
  const void* t = masked ? p.target : nullptr;
  const int blocks = blocks_for(d.rows * (d.ld / 8));
  if (p.type == F32) pack_kernel<F32><<<blocks, 256, 0, st>>>(src, rows, d.rows, p.width, d.ld, t, p.target_wide, p.ignore_index, ones, scale, d.p, d.plane);
  else if (p.type == BF16) pack_kernel<BF16><<<blocks, 256, 0, st>>>(src, rows, d.rows, p.width, d.ld, t, p.target_wide, p.ignore_index, ones, scale, d.p, d.plane);
  else pack_kernel<F16><<<blocks, 256, 0, st>>>(src, rows, d.rows, p.width, d.ld, t, p.target_wide, p.ignore_index, ones, scale, d.p, d.plane);
  OBMAN_LAUNCH_CHECK();
  return 0;
}

static int operands(const obman_class_loss_params& p, const Work& o, bool ones, hipStream_t st) {
  if (p.type == F32) {
    absmax_kernel<<<256, 256, 0, st>>>(static_cast<const float*>(p.x), p.rows, p.width, p.target, p.target_wide, p.ignore_index, o.max_part);
    OBMAN_LAUNCH_CHECK();
    absmax_kernel<<<256, 256, 0, st>>>(static_cast<const float*>(p.w), p.classes, p.width, nullptr, 0, 0, o.max_part + 256);
    OBMAN_LAUNCH_CHECK();
    scale_kernel<<<2, 256, 0, st>>>(o.max_part, o.scales);
    OBMAN_LAUNCH_CHECK();
  }
  int e = 0;
  if (o.x.p != p.x) e = pack(p, p.x, p.rows, o.x, true, ones, o.scales, st);
  if (!e && o.w.p != p.w) e = pack(p, p.w, p.classes, o.w, false, false, o.scales + 1, st);
  return e;
}

static int check(const obman_class_loss_params* p) {
  if (!p || !p->x || !p->w || !p->target) return -1;
  if (p->rows <= 0 || p->classes <= 0 || p->width <= 0 || p->width > 16384) return -2;
  if (p->rows > 0x7fffffffL || p->classes > 0x7fffff00L) return -2;
  if (p->type < 0 || p->type > 2 || p->reduction < 0 || p->reduction > 2) return -3;
  if ((long)obman_cdiv(p->classes, BI) * obman_cdiv(p->rows, BJ) > 0x7fffffffL) return -4;
  return 0;
}

template <int T, int TERMS>
static int forward(const obman_class_loss_params& p, const Work& o, hipStream_t st) {
  constexpr bool split = TERMS == 3;
  const Gemm g{o.w.p, o.x.p, o.w.plane, o.x.plane, p.classes, p.rows, o.w.ld, o.x.ld, p.classes, p.rows, o.w.ld, o.w.ld, o.ti, obman_cdiv(p.rows, BJ), 0};
  const Stats<split> epi{{Scale{split ? o.scales : nullptr, split ? o.scales + 1 : nullptr}, p.bias, p.type, 0, p.classes}, p.target, p.target_wide, o.part, o.picked};
  return launch_gemm<false, false, Stats<split>, T, TERMS>(g, 1, epi, st);
}

template <int T, int TERMS>
static int backward(const obman_class_loss_params& p, const Work& o, void* dx, void* dw, void* db, hipStream_t st) {
  constexpr bool split = TERMS == 3;
  const float *sx = split ? o.scales : nullptr, *sw = split ? o.scales + 1 : nullptr;
  const long xr = o.x.rows;
  const int ld = o.w.ld, size = p.type == F32 ? 4 : 2;
  int e;
  for (long v0 = 0; v0 < p.classes; v0 += o.piece) {
    const long nv = p.classes - v0 < o.piece ? p.classes - v0 : o.piece, kv = up(nv, BK);
    const u16* wp = o.w.p + v0 * ld;
    const Gemm gg{wp, o.x.p, o.w.plane, o.x.plane, p.classes - v0, xr, ld, ld, kv, p.rows, ld, ld, obman_cdiv(kv, BI), obman_cdiv(xr, BJ), 0};
    const Grad<T, split> ge{{Scale{sx, sw}, p.bias, p.type, v0, v0 + nv}, o.rows, xr, o.g, o.g_plane, (int)kv};
    if ((e = launch_gemm<false, false, Grad<T, split>, T, TERMS>(gg, 1, ge, st))) return e;
    if (dx) {
      const Gemm gx{wp, o.g, o.w.plane, o.g_plane, p.classes - v0, xr, ld, (int)kv, ld, p.rows, kv, split_len(kv, o.dx_split), obman_cdiv(ld, BI), obman_cdiv(p.rows, BJ), nv == kv ? 0 : (int)(nv - (kv - BK))};
      const Slab ex{o.dx_slabs, p.rows * ld, ld, v0 > 0};
      if ((e = launch_gemm<true, false, Slab, T, TERMS>(gx, o.dx_split, ex, st))) return e;
    }
    if (dw || db) {
      const Gemm gw{o.x.p, o.g, o.x.plane, o.g_plane, xr, xr, ld, (int)kv, ld, nv, xr, split_len(xr, o.dw_split), obman_cdiv(ld, BI), obman_cdiv(nv, BJ), 0};
      const Slab ew{o.dw_slabs, o.piece * ld, ld, 0};
      if ((e = launch_gemm<true, true, Slab, T, TERMS>(gw, o.dw_split, ew, st))) return e;
      finish_kernel<<<blocks_for(nv * (ld / 4)), 256, 0, st>>>(o.dw_slabs, o.dw_split, o.piece * ld, nv, ld, p.width, o.alpha, Scale{sx, nullptr},
                                                               dw ? static_cast<char*>(dw) + (size_t)v0 * p.width * size : nullptr, p.type,
                                                               db ? static_cast<char*>(db) + (size_t)v0 * size : nullptr);
      OBMAN_LAUNCH_CHECK();
    }
  }
  if (dx) {
    finish_kernel<<<blocks_for(p.rows * (ld / 4)), 256, 0, st>>>(o.dx_slabs, o.dx_split, p.rows * ld, p.rows, ld, p.width, o.alpha, Scale{sw, nullptr}, dx, p.type, nullptr);
    OBMAN_LAUNCH_CHECK();
  }
  return 0;
}

}  // namespace cl

extern "C" {

long obman_class_loss_fwd_ws_bytes(const obman_class_loss_params* p) {
  const int e = cl::check(p);
  return e ? e : (long)cl::plan(*p, nullptr, false, false, false, false).bytes;
}

int obman_class_loss_fwd(const obman_class_loss_params* p, void* ws, float* loss, float* lse, float* norm, obman_stream_t stream) {
  int e = cl::check(p);
  if (e) return e;
  if (!ws || !loss || !lse || !norm) return -1;
  hipStream_t st = (hipStream_t)stream;
  const cl::Work o = cl::plan(*p, ws, false, false, false, false);
  if ((e = cl::operands(*p, o, false, st))) return e;
  e = p->type == cl::F32 ? cl::forward<cl::F16, 3>(*p, o, st) : p->type == cl::BF16 ? cl::forward<cl::BF16, 1>(*p, o, st) : cl::forward<cl::F16, 1>(*p, o, st);
  if (e) return e;
  cl::join_rows_kernel<<<o.row_blocks, 256, 0, st>>>(o.part, o.ti, p->rows, p->classes, o.picked, p->target, p->target_wide, p->ignore_index, lse,
                                                     p->reduction ? nullptr : loss, p->reduction ? o.sums : nullptr);
  OBMAN_LAUNCH_CHECK();
  if (p->reduction) {
    cl::reduce_kernel<<<1, 256, 0, st>>>(o.sums, o.row_blocks, p->reduction == 2, loss, norm);
    OBMAN_LAUNCH_CHECK();
  }
  return 0;
}

long obman_class_loss_bwd_ws_bytes(const obman_class_loss_params* p, int need_x, int need_w, int need_b) {
  const int e = cl::check(p);
  return e ? e : (long)cl::plan(*p, nullptr, true, need_x, need_w, need_b).bytes;
}

int obman_class_loss_bwd(const obman_class_loss_params* p, const float* lse, const float* norm, const float* g_loss, void* ws, void* dx, void* dw, void* db,
                         obman_stream_t stream) {
  int e = cl::check(p);
  if (e) return e;
  if (!ws || !lse || !g_loss || (p->reduction && !norm)) return -1;
  if (!dx && !dw && !db) return 0;
  hipStream_t st = (hipStream_t)stream;
  const cl::Work o = cl::plan(*p, ws, true, dx != nullptr, dw != nullptr, db != nullptr);
  if ((e = cl::operands(*p, o, db != nullptr, st))) return e;
  cl::rows_kernel<<<obman_cdiv(p->rows, 1024), 1024, 0, st>>>(lse, p->target, p->target_wide, p->ignore_index, p->rows, g_loss, p->reduction == 0, norm,
                                                              p->type == cl::BF16 ? 1.f : cl::G_SCALE, o.rows, o.alpha);
  OBMAN_LAUNCH_CHECK();
  return p->type == cl::F32    ? cl::backward<cl::F16, 3>(*p, o, dx, dw, db, st)
         : p->type == cl::BF16 ? cl::backward<cl::BF16, 1>(*p, o, dx, dw, db, st)
                               : cl::backward<cl::F16, 1>(*p, o, dx, dw, db, st);
}

}  // extern "C"
