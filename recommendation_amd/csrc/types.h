// Element types of the operators that take fp32, bf16 and fp16 tensors: 16-byte packets of T and their conversion to
// and from fp32 registers.
#pragma once
#include "common.h"

namespace ctr {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;
typedef bf16_t bf16x2 __attribute__((ext_vector_type(2)));
typedef f16_t f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

__host__ static inline int type_bytes(int t) { return t == CTR_F32 ? 4 : (t == CTR_BF16 || t == CTR_F16) ? 2 : 0; }

// Packet<T>: V elements in 16 bytes.  load / store take any element-aligned address (the compiler emits one 16-byte
// access: global memory needs no more than element alignment here); the *_part forms touch the first n elements only.
template <class T>
struct Packet;

template <>
struct Packet<float> {
  static constexpr int V = 4;
  __device__ static inline void unpack(const uint4& r, float* f) {
    f[0] = __uint_as_float(r.x); f[1] = __uint_as_float(r.y); f[2] = __uint_as_float(r.z); f[3] = __uint_as_float(r.w);
  }
  __device__ static inline uint4 pack(const float* f) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
};

template <>
struct Packet<bf16_t> {
  static constexpr int V = 8;
  __device__ static inline void unpack(const uint4& r, float* f) {
    const unsigned w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  __device__ static inline uint4 pack(const float* f) {
    unsigned w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f32x2 v = {f[2 * i], f[2 * i + 1]};
      w[i] = __builtin_bit_cast(unsigned, __builtin_convertvector(v, bf16x2));   // round to nearest even
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};

template <>
struct Packet<f16_t> {
  static constexpr int V = 8;
  __device__ static inline void unpack(const uint4& r, float* f) {
    const unsigned w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f16x2 h = __builtin_bit_cast(f16x2, w[i]);
      f[2 * i] = (float)h[0];
      f[2 * i + 1] = (float)h[1];
    }
  }
  __device__ static inline uint4 pack(const float* f) {
    unsigned w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f16x2 h = {(f16_t)f[2 * i], (f16_t)f[2 * i + 1]};
      w[i] = __builtin_bit_cast(unsigned, h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};

template <class T>
__device__ static inline uint4 packet_load(const T* p) {
  uint4 r;
  __builtin_memcpy(&r, p, 16);
  return r;
}
template <class T>
__device__ static inline void packet_store(T* p, const uint4& r) {
  __builtin_memcpy(p, &r, 16);
}
// n in [0, V]: elements n.. read as `fill`
template <class T>
__device__ static inline void load_part(const T* p, int n, float fill, float* f) {
#pragma unroll
  for (int j = 0; j < Packet<T>::V; ++j) f[j] = j < n ? (float)p[j] : fill;
}
template <class T>
__device__ static inline void store_part(T* p, int n, const float* f) {
#pragma unroll
  for (int j = 0; j < Packet<T>::V; ++j)
    if (j < n) p[j] = (T)f[j];
}

// Sum over the G lanes (a power of two, aligned) a lane belongs to, the same bits in every one of them.
template <int G>
__device__ static inline float group_sum(float v) {
  if (G >= 2) v = dpp_add<DPP_XOR1>(v);
  if (G >= 4) v = dpp_add<DPP_XOR2>(v);
  if (G >= 8) v = dpp_add<0x141>(v);        // mirror inside 8 lanes: the quads hold one value each by now
  if (G >= 16) v = dpp_add<DPP_ROR + 8>(v);
  if (G >= 32) v = row_swap_sum(v, v);
  if (G >= 64) v = half_swap_sum(v, v);
  return v;
}

}  // namespace ctr
