// K16: the norm of all gradients together and clipping by it, over a list of tensors of any sizes and of mixed types.
//
//   norm = (sum over tensors, elements |g|^p)^(1/p), p = 1 or 2, or max |g| (p = inf)
//   g   <- g * min(1, max_norm / (norm + 1e-6))
//
// Bound: memory.  The norm reads every gradient once; clipping has to read it again (no value can be scaled before the last one is
// summed) and write it.  Sums are held in 64 bits from the first element on: one fp64 multiply-add per element is a few per cent of
// the vector rate at the rate memory delivers elements, no square of an fp32 value leaves the range of a double, and the result does
// not depend on how the elements are split (1e-16 relative), so the tile size is free.  Order: each block sums a fixed run of
// chunks, the block sums are added in index order - no atomics, the same bits every call.
//
// Measured: 268 M bf16 in 114 us, 4.7 TB/s (a large copy reaches 4.8; with half the loads in flight it was 3.4); clipping 120 M
// values of two types, packed at odd offsets, 243 us, 4.5 TB/s of its three passes; 13.2 M fp32 in 92 tensors: 15 + 21 us.
// Two launches: block sums, then their join - by one block for the norm alone, by every block of the scaling pass for clipping
// (<= GN_BLOCKS doubles out of L2, cheaper than a third launch).  Up to GN_SMALL_CHUNKS chunks, one block does everything in one launch.
#include "gradnorm.h"
#include "../../include/obman_hip.h"

namespace gn {

__global__ __launch_bounds__(256) void partial_kernel(Batch b, int norm, double* __restrict__ part) {
  // contiguous run of chunks per block: one search, then the table is walked
  const long total = b.first_chunk[b.count];
  long c = total * blockIdx.x / gridDim.x;
  const long c1 = total * (blockIdx.x + 1) / gridDim.x;
  int t = find(b, c);
  double acc = 0.0;
  unsigned top = 0;
  for (; c < c1; ++c) {
    while (c >= b.first_chunk[t + 1]) ++t;
    const int type = type_of(b, t), chunk = chunk_of(type);
    const long at = (c - b.first_chunk[t]) * chunk;
    const long n = count_of(b, t) - at;
    chunk_sum(b.p[t], type, at, n < chunk ? (int)n : chunk, norm, threadIdx.x, 256, acc, top);
  }
  const double s = norm == NORM_INF ? (double)__uint_as_float(block_max<256>(top)) : block_sum<256>(acc);
  if (threadIdx.x == 0) part[blockIdx.x] = s;
}

__global__ __launch_bounds__(256) void join_kernel(const double* __restrict__ part, int count, int norm, float* __restrict__ out) {
  const double s = join<256>(part, count, norm);
  if (threadIdx.x == 0) *out = (float)s;
}

__global__ __launch_bounds__(256) void scale_kernel(Batch b, int norm, const double* __restrict__ part, int parts, float max_norm, float* __restrict__ out) {
  const float n32 = (float)join<256>(part, parts, norm);
  const float k = clip_factor(n32, max_norm);
  if (blockIdx.x == 0 && threadIdx.x == 0) *out = n32;
  const long total = b.first_chunk[b.count];
  // from the end backwards: what the norm's pass read last is what the 256 MB cache still holds
  const int r = gridDim.x - 1 - blockIdx.x;
  const long c0 = total * r / gridDim.x;
  long c = total * (r + 1) / gridDim.x - 1;
  int t = find(b, c);
  for (; c >= c0; --c) {
    while (c < b.first_chunk[t]) --t;
    const int type = type_of(b, t), chunk = chunk_of(type);
    const long at = (c - b.first_chunk[t]) * chunk;
    const long n = count_of(b, t) - at;
    chunk_scale(b.p[t], type, at, n < chunk ? (int)n : chunk, k, threadIdx.x, 256);
  }
}

// everything in one block of 1024 threads: below GN_SMALL_CHUNKS chunks a second launch costs more than the idle CUs
__global__ __launch_bounds__(1024) void small_kernel(Batch b, int norm, int scale, float max_norm, float* __restrict__ out) {
  double acc = 0.0;
  unsigned top = 0;
  for (int t = 0; t < b.count; ++t) chunk_sum(b.p[t], type_of(b, t), 0, (int)count_of(b, t), norm, threadIdx.x, 1024, acc, top);
  double s = norm == NORM_INF ? (double)__uint_as_float(block_max<1024>(top)) : block_sum<1024>(acc);
  if (norm == NORM_2) s = sqrt(s);
  const float n32 = (float)s;
  if (threadIdx.x == 0) *out = n32;
  if (!scale) return;
  const float k = clip_factor(n32, max_norm);
  for (int t = 0; t < b.count; ++t) chunk_scale(b.p[t], type_of(b, t), 0, (int)count_of(b, t), k, threadIdx.x, 1024);
}

int launch_partials(const Batch& b, int norm, double* ws, int* parts, long cap, hipStream_t st) {
  const int g = blocks_of(b);
  if (*parts + (long)g > cap) return -4;
  partial_kernel<<<g, 256, 0, st>>>(b, norm, ws + *parts);
  OBMAN_LAUNCH_CHECK();
  *parts += g;
  return 0;
}

static int run(void* const* p, const long* n, const int* type, int count, int norm, bool scale, float max_norm, double* ws, float* out, hipStream_t st) {
  if (count < 0 || (count && (!p || !n || !type)) || !ws || !out || norm < 0 || norm > 2 || !(max_norm >= 0.f)) return -1;
  const auto get = [&](int i) { return Item{p[i], n[i], type[i]}; };
  Batch b;
  int i = 0, parts = 0, e = fill(b, get, count, i);
  if (e) return e;
  if (i == count && b.first_chunk[b.count] <= GN_SMALL_CHUNKS) {
    small_kernel<<<1, 1024, 0, st>>>(b, norm, scale, max_norm, out);
    OBMAN_LAUNCH_CHECK();
    return 0;
  }
  e = partials(get, count, norm, ws, &parts, st);
  if (e) return e;
  if (!scale) {
    join_kernel<<<1, 256, 0, st>>>(ws, parts, norm, out);
    OBMAN_LAUNCH_CHECK();
    return 0;
  }
  for (i = 0; i < count;) {
    e = fill(b, get, count, i);
    if (e) return e;
    if (!b.count) break;
    scale_kernel<<<blocks_of(b), 256, 0, st>>>(b, norm, ws, parts, max_norm, out);
    OBMAN_LAUNCH_CHECK();
  }
  return 0;
}

}  // namespace gn

extern "C" {

long obman_grad_norm_ws_doubles(int count) { return count < 0 ? -1 : gn::ws_doubles(count); }

int obman_grad_norm(void* const* g, const long* n, const int* type, int count, int norm, double* ws, float* out, obman_stream_t stream) {
  return gn::run(g, n, type, count, norm, false, 0.f, ws, out, (hipStream_t)stream);
}

int obman_grad_clip(void* const* g, const long* n, const int* type, int count, int norm, float max_norm, double* ws, float* out, obman_stream_t stream) {
  return gn::run(g, n, type, count, norm, true, max_norm, ws, out, (hipStream_t)stream);
}

}  // extern "C"
