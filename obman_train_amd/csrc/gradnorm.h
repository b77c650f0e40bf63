// Device parts of the gradient norm shared by gradnorm.hip (norm, clipping) and stepops.hip (the clipped optimizer step).
#pragma once
#include "common.h"

namespace gn {

enum { NORM_INF = 0, NORM_1 = 1, NORM_2 = 2 };
enum { F32 = 0, BF16 = 1, F16 = 2 };

constexpr int MAX_TENSORS = 192;  // per launch: 192 x 20 bytes of kernel arguments (limit 4 KB)
constexpr int CHUNK_BYTES = 16384;  // four 16-byte loads in flight per thread of a 256-thread block
__host__ __device__ constexpr int chunk_of(int type) { return type == 0 ? CHUNK_BYTES / 4 : CHUNK_BYTES / 2; }
constexpr int GN_BLOCKS = 2048;   // eight blocks per CU; also what the join reads
constexpr int GN_SMALL_CHUNKS = 8;

struct Batch {
  void* p[MAX_TENSORS];
  unsigned long n_type[MAX_TENSORS];    // elements | type << 60
  int first_chunk[MAX_TENSORS + 1];     // prefix of the per-tensor chunk counts
  int count;
};
static_assert(sizeof(Batch) <= 4096 - 64, "kernel argument block");

__device__ __forceinline__ long count_of(const Batch& b, int t) { return (long)(b.n_type[t] & ((1UL << 60) - 1)); }
__device__ __forceinline__ int type_of(const Batch& b, int t) { return (int)(b.n_type[t] >> 60); }

__device__ __forceinline__ int find(const Batch& b, long c) {
  int lo = 0, hi = b.count;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (c >= b.first_chunk[mid]) lo = mid; else hi = mid;
  }
  return lo;
}

// 16-byte vectors at element alignment: gradients packed back to back start anywhere, and the memory pipe takes such addresses
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned short u16x8u __attribute__((ext_vector_type(8), aligned(2)));

template <int TYPE>
__device__ __forceinline__ float widen(unsigned short u) {
  if constexpr (TYPE == BF16) return __uint_as_float((unsigned)u << 16);
  else return (float)__builtin_bit_cast(_Float16, u);
}
template <int TYPE>
__device__ __forceinline__ unsigned short narrow(float x) {  // round to nearest even
  if constexpr (TYPE == BF16) return __builtin_bit_cast(unsigned short, (__bf16)x);
  else return __builtin_bit_cast(unsigned short, (_Float16)x);
}

__device__ __forceinline__ void add(float x, int norm, double& acc, unsigned& top) {
  if (norm == NORM_2) {
    const double d = (double)x;
    acc = __builtin_fma(d, d, acc);
  } else if (norm == NORM_1) {
    acc += (double)fabsf(x);
  } else {
    const unsigned u = __float_as_uint(x) & 0x7fffffffu;  // ordered like |x|, with NaN above infinity: a NaN stays
    top = u > top ? u : top;
  }
}

template <int TYPE>
__device__ __forceinline__ void chunk_sum16(const unsigned short* __restrict__ g, int n, int norm, int tid, int threads, double& acc, unsigned& top) {
  const int full = n & ~7;
  for (int i = tid * 8; i < full; i += threads * 32) {
    u16x8u v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int j = i + k * threads * 8;
      v[k] = u16x8u{0, 0, 0, 0, 0, 0, 0, 0};
      if (j < full) v[k] = *reinterpret_cast<const u16x8u*>(g + j);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int e = 0; e < 8; ++e) add(widen<TYPE>(v[k][e]), norm, acc, top);
  }
  for (int i = full + tid; i < n; i += threads) add(widen<TYPE>(g[i]), norm, acc, top);
}

// elements [at, at + n) of one tensor into the thread's running sum / maximum
__device__ __forceinline__ void chunk_sum(const void* p, int type, long at, int n, int norm, int tid, int threads, double& acc, unsigned& top) {
  if (type == F32) {
    const float* __restrict__ g = static_cast<const float*>(p) + at;
    const int full = n & ~3;
    for (int i = tid * 4; i < full; i += threads * 16) {
      f32x4u v[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int j = i + k * threads * 4;
        v[k] = f32x4u{0.f, 0.f, 0.f, 0.f};
        if (j < full) v[k] = *reinterpret_cast<const f32x4u*>(g + j);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) add(v[k][e], norm, acc, top);
    }
    for (int i = full + tid; i < n; i += threads) add(g[i], norm, acc, top);
  } else if (type == BF16) {
    chunk_sum16<BF16>(static_cast<const unsigned short*>(p) + at, n, norm, tid, threads, acc, top);
  } else {
    chunk_sum16<F16>(static_cast<const unsigned short*>(p) + at, n, norm, tid, threads, acc, top);
  }
}

template <int TYPE>
__device__ __forceinline__ void chunk_scale16(unsigned short* __restrict__ g, int n, float k, int tid, int threads) {
  const int full = n & ~7;
  for (int i = tid * 8; i < full; i += threads * 32) {
    u16x8u v[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int j = i + q * threads * 8;
      if (j < full) v[q] = *reinterpret_cast<u16x8u*>(g + j);
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int j = i + q * threads * 8;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[q][e] = narrow<TYPE>(widen<TYPE>(v[q][e]) * k);  // one rounding, to the gradient's own type
      if (j < full) *reinterpret_cast<u16x8u*>(g + j) = v[q];
    }
  }
  for (int i = full + tid; i < n; i += threads) g[i] = narrow<TYPE>(widen<TYPE>(g[i]) * k);
}

__device__ __forceinline__ void chunk_scale(void* p, int type, long at, int n, float k, int tid, int threads) {
  if (type == F32) {
    float* __restrict__ g = static_cast<float*>(p) + at;
    const int full = n & ~3;
    for (int i = tid * 4; i < full; i += threads * 16) {
      f32x4u v[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int j = i + q * threads * 4;
        if (j < full) v[q] = *reinterpret_cast<f32x4u*>(g + j);
      }
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int j = i + q * threads * 4;
        if (j < full) *reinterpret_cast<f32x4u*>(g + j) = v[q] * k;
      }
    }
    for (int i = full + tid; i < n; i += threads) g[i] *= k;
  } else if (type == BF16) {
    chunk_scale16<BF16>(static_cast<unsigned short*>(p) + at, n, k, tid, threads);
  } else {
    chunk_scale16<F16>(static_cast<unsigned short*>(p) + at, n, k, tid, threads);
  }
}

// block-wide sum / maximum, the same bits in every thread; fixed order
template <int THREADS>
__device__ __forceinline__ double block_sum(double v) {
  __shared__ double red[THREADS / 64];
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  double s = red[0];
#pragma unroll
  for (int w = 1; w < THREADS / 64; ++w) s += red[w];
  __syncthreads();
  return s;
}
template <int THREADS>
__device__ __forceinline__ unsigned block_max(unsigned v) {
  __shared__ unsigned red[THREADS / 64];
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    const unsigned o = __shfl_xor(v, off, 64);
    v = o > v ? o : v;
  }
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  unsigned s = red[0];
#pragma unroll
  for (int w = 1; w < THREADS / 64; ++w) s = red[w] > s ? red[w] : s;
  __syncthreads();
  return s;
}

// the norm from the block sums; every thread of the block has it
template <int THREADS>
__device__ __forceinline__ double join(const double* __restrict__ part, int count, int norm) {
  if (norm == NORM_INF) {
    unsigned top = 0;
    for (int i = threadIdx.x; i < count; i += THREADS) {
      const unsigned u = __float_as_uint((float)part[i]);
      top = u > top ? u : top;
    }
    return (double)__uint_as_float(block_max<THREADS>(top));
  }
  double acc = 0.0;
  for (int i = threadIdx.x; i < count; i += THREADS) acc += part[i];
  acc = block_sum<THREADS>(acc);
  return norm == NORM_2 ? sqrt(acc) : acc;
}

// min(1, max_norm / (norm + 1e-6)) in fp32, as torch forms it; a NaN norm gives NaN, an infinite one 0
__device__ __forceinline__ float clip_factor(float norm, float max_norm) {
  const float k = max_norm / (norm + 1e-6f);
  return k > 1.f ? 1.f : k;
}

// what a list says about its i-th tensor
struct Item { void* p; long n; int type; };

// the next table of a list of `count` tensors from i on; skips empty tensors; -> 0 or a negative error
template <class Get>
static inline int fill(Batch& b, const Get& get, int count, int& i) {
  b.count = 0;
  b.first_chunk[0] = 0;
  for (; i < count && b.count < MAX_TENSORS; ++i) {
    const Item t = get(i);
    if (t.n < 0 || t.type < 0 || t.type > 2) return -2;
    if (t.n == 0) continue;
    const int chunk = chunk_of(t.type);
    if (!t.p || t.n > (long)chunk * 0x7fffffffL) return -2;
    const long c = b.first_chunk[b.count] + (t.n + chunk - 1) / chunk;
    if (c > 0x7fffffffL) {
      if (!b.count) return -3;
      break;  // the chunk index would leave 32 bits: this tensor opens the next table
    }
    b.p[b.count] = t.p;
    b.n_type[b.count] = (unsigned long)t.n | ((unsigned long)t.type << 60);
    b.first_chunk[++b.count] = (int)c;
  }
  return 0;
}
static inline int blocks_of(const Batch& b) {
  const int c = b.first_chunk[b.count];
  return c < GN_BLOCKS ? c : GN_BLOCKS;
}
// doubles of scratch for the block sums of a list; a table may end early where its chunk index ends, hence the second term
static inline long ws_doubles(int count) { return ((long)(count + MAX_TENSORS - 1) / MAX_TENSORS + 16) * GN_BLOCKS; }

int launch_partials(const Batch& b, int norm, double* ws, int* parts, long cap, hipStream_t st);

// launches the block sums of a list; *parts = how many doubles of ws they fill
template <class Get>
static inline int partials(const Get& get, int count, int norm, double* ws, int* parts, hipStream_t st) {
  *parts = 0;
  for (int i = 0; i < count;) {
    Batch b;
    int e = fill(b, get, count, i);
    if (e) return e;
    if (!b.count) break;
    e = launch_partials(b, norm, ws, parts, ws_doubles(count), st);
    if (e) return e;
  }
  return 0;
}

}  // namespace gn
