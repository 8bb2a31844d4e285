// Global gradient norm over many tensors and the scaling that bounds it.
//   norm = sqrt(sum over all elements of g^2);  g' = g * bound / max(norm, bound)
// (tf.clip_by_global_norm: a norm that is not finite makes every g' NaN).
// Memory bound: the norm reads every element once, the scaling reads it again and writes it once; nothing else moves.
// The tensors travel by value in the kernel arguments (address, size, type), so a call needs no table on the device and
// a captured graph owns its list.  Squares are summed in fp64: no element of any of the three types overflows or
// vanishes there, and the fp64 pipe (half the fp32 rate) is far from the bound.  One partial per block, added in block
// order by every block of the second launch: results are the same bits on every run, and there is no third launch.
// Measured (60 tensors of fp32 and bf16, 815 MB in all, into other tensors; averages of a kernel trace over calls in a
// row): the squares 167 us, 4.9 TB/s, the scaling 293 us, 5.6 TB/s; a large copy reaches 4.9.  24 small tensors: 4.5 us and
// 1.7 for the norm, launches.
#include "types.h"
#include <math.h>

namespace ctr {

constexpr int CLIP_TENSORS = 96;                     // per launch: 96 * (8 + 8 + 8 + 4) bytes of kernel arguments
// Partials per launch at most; the scaling takes twice as many blocks.  815 MB of squares: 165 us (171 with 512 or 2048).
constexpr int CLIP_BLOCKS = 1024;
// Bytes of one tensor that a block takes at a time, eight packets per thread: 165 and 290 us (171 and 291 with twice as
// much, 165 and 295 with half).
constexpr int CLIP_CHUNK = 32768;

struct ClipList {
  const void* src[CLIP_TENSORS];
  void* dst[CLIP_TENSORS];
  int64_t count[CLIP_TENSORS];
  int first[CLIP_TENSORS + 1];                       // chunks before tensor i
  unsigned char type[CLIP_TENSORS];
  int n;
};

__host__ __device__ static inline int64_t clip_chunk_elems(int type) { return type == CTR_F32 ? CLIP_CHUNK / 4 : CLIP_CHUNK / 2; }

// the tensor that chunk c belongs to (uniform over the block)
__device__ static inline int clip_find(const ClipList& a, int c) {
  int lo = 0, hi = a.n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (a.first[mid] <= c) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

__device__ static inline double wave_sum64(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}
// sum over the 256 threads, in every thread, in a fixed order
__device__ static inline double block_sum64(double v, double* red) {
  v = wave_sum64(v);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  const double s = (red[0] + red[1]) + (red[2] + red[3]);
  __syncthreads();
  return s;
}

// sum of squares of elements [at, end) of a tensor: 256 threads, 8 packets in flight per thread
template <class T>
__device__ static inline double chunk_squares(const T* p, int64_t at, int64_t end) {
  constexpr int V = Packet<T>::V;
  double s0 = 0., s1 = 0.;
  const int n = (int)(end - at), full = n / V;
  p += at;
  constexpr int PER = CLIP_CHUNK / 16 / 256;
  if (full == PER * 256) {
    uint4 r[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) r[i] = packet_load(p + (int64_t)(threadIdx.x + i * 256) * V);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      float f[V];
      Packet<T>::unpack(r[i], f);
#pragma unroll
      for (int j = 0; j < V; j += 2) {
        s0 = fma((double)f[j], (double)f[j], s0);
        s1 = fma((double)f[j + 1], (double)f[j + 1], s1);
      }
    }
    return s0 + s1;
  }
  for (int k = threadIdx.x; k < full; k += 256) {
    float f[V];
    Packet<T>::unpack(packet_load(p + (int64_t)k * V), f);
#pragma unroll
    for (int j = 0; j < V; j += 2) {
      s0 = fma((double)f[j], (double)f[j], s0);
      s1 = fma((double)f[j + 1], (double)f[j + 1], s1);
    }
  }
  if (threadIdx.x < n - full * V) {
    const double f = (double)(float)p[full * V + threadIdx.x];
    s0 = fma(f, f, s0);
  }
  return s0 + s1;
}

__global__ __launch_bounds__(256) void clip_squares_kernel(ClipList a, double* __restrict__ part) {
  __shared__ double red[4];
  double s = 0.;
  const int chunks = a.first[a.n];
  for (int c = blockIdx.x; c < chunks; c += gridDim.x) {
    const int t = clip_find(a, c);
    const int64_t per = clip_chunk_elems(a.type[t]), at = (int64_t)(c - a.first[t]) * per;
    const int64_t end = min(a.count[t], at + per);
    if (a.type[t] == CTR_F32) s += chunk_squares((const float*)a.src[t], at, end);
    else if (a.type[t] == CTR_BF16) s += chunk_squares((const bf16_t*)a.src[t], at, end);
    else s += chunk_squares((const f16_t*)a.src[t], at, end);
  }
  s = block_sum64(s, red);
  if (threadIdx.x == 0) part[blockIdx.x] = s;
}

__device__ static inline double clip_norm(const double* __restrict__ part, int parts, double* red) {
  double s = 0.;
  for (int i = threadIdx.x; i < parts; i += 256) s += part[i];
  return sqrt(block_sum64(s, red));
}

__global__ __launch_bounds__(256) void clip_norm_kernel(const double* __restrict__ part, int parts,
                                                        float* __restrict__ norm_out) {
  __shared__ double red[4];
  const double norm = clip_norm(part, parts, red);
  if (threadIdx.x == 0) norm_out[0] = (float)norm;
}

// The factor as m 2^e, m in [0.5, 1]: beside gradients near the end of fp32 it is below fp32's normal range.
struct Factor { float m; int e; };
__device__ static inline float scaled(float f, const Factor& by) { return ldexpf(f * by.m, by.e); }

template <class T>
__device__ static inline void chunk_scale(const T* p, T* o, int64_t at, int64_t end, Factor by) {
  constexpr int V = Packet<T>::V;
  const int n = (int)(end - at), full = n / V;
  p += at;
  o += at;
  constexpr int PER = CLIP_CHUNK / 16 / 256;
  if (full == PER * 256) {
    uint4 r[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) r[i] = packet_load(p + (int64_t)(threadIdx.x + i * 256) * V);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      float f[V];
      Packet<T>::unpack(r[i], f);
#pragma unroll
      for (int j = 0; j < V; ++j) f[j] = scaled(f[j], by);
      packet_store(o + (int64_t)(threadIdx.x + i * 256) * V, Packet<T>::pack(f));
    }
    return;
  }
  for (int k = threadIdx.x; k < full; k += 256) {
    float f[V];
    Packet<T>::unpack(packet_load(p + (int64_t)k * V), f);
#pragma unroll
    for (int j = 0; j < V; ++j) f[j] = scaled(f[j], by);
    packet_store(o + (int64_t)k * V, Packet<T>::pack(f));
  }
  if (threadIdx.x < n - full * V) o[full * V + threadIdx.x] = (T)scaled((float)p[full * V + threadIdx.x], by);
}

// in_place: every tensor is its own destination, and a factor of one leaves it unread
__global__ __launch_bounds__(256) void clip_scale_kernel(ClipList a, const double* __restrict__ part, int parts,
                                                         float bound, int in_place, float* __restrict__ norm_out) {
  __shared__ double red[4];
  const double norm = clip_norm(part, parts, red);
  if (blockIdx.x == 0 && threadIdx.x == 0 && norm_out) norm_out[0] = (float)norm;
  Factor by = {1.f, 0};
  if (norm > (double)bound) by.m = (float)frexp((double)bound / norm, &by.e);
  if (!(norm <= 1.7976931348623157e308)) by = {__builtin_nanf(""), 0};
  else if (in_place && !(norm > (double)bound)) return;
  const int chunks = a.first[a.n];
  for (int c = blockIdx.x; c < chunks; c += gridDim.x) {
    const int t = clip_find(a, c);
    const int64_t per = clip_chunk_elems(a.type[t]), at = (int64_t)(c - a.first[t]) * per;
    const int64_t end = min(a.count[t], at + per);
    if (a.type[t] == CTR_F32) chunk_scale((const float*)a.src[t], (float*)a.dst[t], at, end, by);
    else if (a.type[t] == CTR_BF16) chunk_scale((const bf16_t*)a.src[t], (bf16_t*)a.dst[t], at, end, by);
    else chunk_scale((const f16_t*)a.src[t], (f16_t*)a.dst[t], at, end, by);
  }
}

// The next launch's list: tensors from `at` on; returns the first one it does not hold.  (clip_check keeps the bytes of
// all tensors below 2^44, so the chunk counts stay far inside an int.)
static int clip_fill(const void* const* src, void* const* dst, const int64_t* counts, const int* types, int n, int at,
                     ClipList* a) {
  a->n = 0;
  a->first[0] = 0;
  int64_t chunks = 0;
  for (; at < n && a->n < CLIP_TENSORS; ++at) {
    if (counts[at] == 0) continue;
    chunks += cdiv(counts[at], clip_chunk_elems(types[at]));
    a->src[a->n] = src[at];
    a->dst[a->n] = dst ? dst[at] : nullptr;
    a->count[a->n] = counts[at];
    a->type[a->n] = (unsigned char)types[at];
    a->first[++a->n] = (int)chunks;
  }
  return at;
}

static int clip_check(const char* what, const void* const* src, const int64_t* counts, const int* types, int n) {
  CTR_REQUIRE(n >= 0 && (n == 0 || (src && counts && types)), "%s: %d tensors without their lists", what, n);
  int64_t room = (int64_t)1 << 44;
  for (int i = 0; i < n; ++i) {
    CTR_REQUIRE(type_bytes(types[i]) != 0, "%s: tensor %d has unknown dtype %d", what, i, types[i]);
    CTR_REQUIRE(counts[i] >= 0 && counts[i] <= room / type_bytes(types[i]), "%s: tensor %d has %lld elements", what, i,
                (long long)counts[i]);
    CTR_REQUIRE(counts[i] == 0 || src[i], "%s: tensor %d is NULL", what, i);
    room -= counts[i] * type_bytes(types[i]);
  }
  return CTR_OK;
}

static size_t clip_ws(int n) { return (size_t)cdiv(n < 1 ? 1 : n, CLIP_TENSORS) * CLIP_BLOCKS * sizeof(double); }

// squares of all tensors into ws; *parts = partials written, or <0 / >0 on error
static int clip_squares(const void* const* src, const int64_t* counts, const int* types, int n, double* ws, int* parts,
                        hipStream_t st) {
  *parts = 0;
  for (int at = 0; at < n;) {
    ClipList a;
    at = clip_fill(src, nullptr, counts, types, n, at, &a);
    const int blocks = a.first[a.n] < CLIP_BLOCKS ? a.first[a.n] : CLIP_BLOCKS;
    if (!blocks) continue;
    clip_squares_kernel<<<blocks, 256, 0, st>>>(a, ws + *parts);
    CTR_LAUNCH_CHECK();
    *parts += blocks;
  }
  return CTR_OK;
}

}  // namespace ctr

using namespace ctr;

extern "C" size_t ctr_grad_norm_workspace_bytes(int n_tensors) { return clip_ws(n_tensors); }

extern "C" int ctr_grad_norm(const void* const* grads_host, const int64_t* counts_host, const int* dtypes_host,
                             int n_tensors, float* norm_out, void* workspace, size_t workspace_bytes, void* stream) {
  const int rc = clip_check("grad_norm", grads_host, counts_host, dtypes_host, n_tensors);
  if (rc) return rc;
  CTR_REQUIRE(norm_out, "grad_norm: norm_out is NULL");
  if (!workspace || workspace_bytes < clip_ws(n_tensors)) {
    set_error("grad_norm: workspace %zu < %zu", workspace_bytes, clip_ws(n_tensors));
    return CTR_EWORKSPACE;
  }
  hipStream_t st = (hipStream_t)stream;
  int parts = 0;
  const int r2 = clip_squares(grads_host, counts_host, dtypes_host, n_tensors, (double*)workspace, &parts, st);
  if (r2) return r2;
  clip_norm_kernel<<<1, 256, 0, st>>>((const double*)workspace, parts, norm_out);
  CTR_LAUNCH_CHECK();
  return CTR_OK;
}

extern "C" int ctr_clip_grads(const void* const* grads_host, void* const* out_host, const int64_t* counts_host,
                              const int* dtypes_host, int n_tensors, float max_norm, float* norm_out, void* workspace,
                              size_t workspace_bytes, void* stream) {
  const int rc = clip_check("clip_grads", grads_host, counts_host, dtypes_host, n_tensors);
  if (rc) return rc;
  CTR_REQUIRE(max_norm > 0.f && max_norm <= 3.402823466e38f, "clip_grads: max_norm must be positive and finite");
  CTR_REQUIRE(n_tensors == 0 || out_host, "clip_grads: out_host is NULL");
  int in_place = 1;
  for (int i = 0; i < n_tensors; ++i) {
    CTR_REQUIRE(counts_host[i] == 0 || out_host[i], "clip_grads: output %d is NULL", i);
    if (counts_host[i] && out_host[i] != grads_host[i]) in_place = 0;
  }
  if (!workspace || workspace_bytes < clip_ws(n_tensors)) {
    set_error("clip_grads: workspace %zu < %zu", workspace_bytes, clip_ws(n_tensors));
    return CTR_EWORKSPACE;
  }
  hipStream_t st = (hipStream_t)stream;
  int parts = 0;
  const int r2 = clip_squares(grads_host, counts_host, dtypes_host, n_tensors, (double*)workspace, &parts, st);
  if (r2) return r2;
  int launched = 0;
  for (int at = 0; at < n_tensors;) {
    ClipList a;
    at = clip_fill(grads_host, out_host, counts_host, dtypes_host, n_tensors, at, &a);
    const int chunks = a.first[a.n], blocks = chunks < 2 * CLIP_BLOCKS ? chunks : 2 * CLIP_BLOCKS;
    if (!blocks) continue;
    clip_scale_kernel<<<blocks, 256, 0, st>>>(a, (const double*)workspace, parts, max_norm, in_place,
                                              launched++ ? nullptr : norm_out);
    CTR_LAUNCH_CHECK();
  }
  if (!launched && norm_out) {                       // no elements at all: the norm is zero
    clip_norm_kernel<<<1, 256, 0, st>>>((const double*)workspace, 0, norm_out);
    CTR_LAUNCH_CHECK();
  }
  return CTR_OK;
}
