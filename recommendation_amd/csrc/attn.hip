// Multi-head cross attention, forward and backward: Tq query rows attend to the Tk states of another sequence.
//   s = scale q k^T over the keys t < sl[b] that mask[b] leaves;  p = softmax(s);  out = p v;  lse = log sum exp s
//   delta = sum_d dout out;  ds = p (dout v^T - delta);  dq = scale ds k;  dk = scale ds^T q;  dv = p^T dout
// H query heads share Hkv key heads in groups of G = H / Hkv.  The Tq * G query rows of one (sample, key head) form one
// list (row r = query r / G, head r % G of the group), so a key tile is fetched once for the whole group and the sums
// of dk / dv over the group fall out of the row loop.
//
// All products run on 32x32x16 matrix instructions.  The forward and the dq pass keep scores transposed (keys down,
// query rows across): a lane owns one query row, so the running maximum, the sum and the rescaling are per-lane
// scalars, and its 16 scores of a 32-key strip are already the second operand of the product with V (or K) once that
// operand's rows are taken in the same order (Tile::cols), which the transposing LDS read delivers.  The dk / dv pass
// is the mirror image: a lane owns one key, the strip runs over query rows.
// fp32 tensors are split into three bf16 terms (24 significant bits) and every product is the six largest of the nine
// term products; the sums are fp32 in all types.  For 16-bit tensors p and ds are rounded to the tensors' type before
// the second product (half a step each, independent over the keys that are summed, like the rounding of v and k
// themselves); fp16's narrow exponent is met by a power of two on p (2^14) and a running one per row on ds.
// A key behind sl[b] or off in the mask is staged as zeros and its p is set to zero, so nothing that its memory holds
// reaches a result.  A row without keys gives zeros, lse = -inf and no gradient.  No float atomics: same bits every run.
// Bound: matrix and vector instructions, which overlap by about half, and waiting.  A loop of 4 products, 32 fma and 8 exp
// takes a wave, two to a SIMD, 63 ns, 38 and 31 one by one; fma and exp together 80, products and exp 71, products and fma
// 90, all three 107 (no overlap of products and the rest would be 143, a full one 80).  At head size 128 (4 x 16 heads of
// 1025 x 2047 on 4, bf16) the waves wait for half of their cycles besides; for what, the counters taken do not say.
// 16 heads of 2048 x 4096 of 64, batch 8, bf16: forward 336 us, 820 TFLOP/s counting its two products; dq 574 us, dk / dv
// 600 us, 720 and 920 TFLOP/s counting three and four (a large bf16 matrix product reaches 1390 on the same card).
// Times without a second one beside them are averages of a kernel trace over whole passes in a row on the same inputs;
// times that are compared come from one sweep each and are to be read against each other only.
#include "types.h"

namespace ctr {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef bf16_t bf16x8 __attribute__((ext_vector_type(8)));
typedef f16_t f16x8 __attribute__((ext_vector_type(8)));

// T: the tensors' type; NP: 16-bit terms per value; BIAS: log2 of the factor on p
template <class T> struct Terms;
template <> struct Terms<bf16_t> { static constexpr int NP = 1; static constexpr float BIAS = 0.f; };
template <> struct Terms<f16_t> { static constexpr int NP = 1; static constexpr float BIAS = 14.f; };
template <> struct Terms<float> { static constexpr int NP = 3; static constexpr float BIAS = 0.f; };

// eight 16-bit values per term: one operand of a matrix instruction
template <class T> struct Frag { s16x8 t[Terms<T>::NP]; };

template <class T>
__device__ static inline f32x16 mfma1(s16x8 a, s16x8 b, f32x16 c) {
  if constexpr (__is_same(T, f16_t))
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
template <class T>
__device__ static inline f32x16 mfma(const Frag<T>& a, const Frag<T>& b, f32x16 c) {
  if constexpr (Terms<T>::NP == 1) {
    return mfma1<T>(a.t[0], b.t[0], c);
  } else {                                              // smallest products first
    c = mfma1<T>(a.t[2], b.t[0], c);
    c = mfma1<T>(a.t[0], b.t[2], c);
    c = mfma1<T>(a.t[1], b.t[1], c);
    c = mfma1<T>(a.t[1], b.t[0], c);
    c = mfma1<T>(a.t[0], b.t[1], c);
    return mfma1<T>(a.t[0], b.t[0], c);
  }
}

__device__ static inline unsigned pack_bf16(float a, float b) {
  const f32x2 v = {a, b};
  return __builtin_bit_cast(unsigned, __builtin_convertvector(v, bf16x2));
}
// eight fp32 values -> operand (fp32: x = hi + mid + lo, each the bf16 nearest to what is left)
template <class T>
__device__ static inline Frag<T> make_frag(const float* f) {
  Frag<T> r;
  if constexpr (Terms<T>::NP == 1) {
    r.t[0] = __builtin_bit_cast(s16x8, Packet<T>::pack(f));
  } else {
    unsigned w[3][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float a = f[2 * i], b = f[2 * i + 1];
#pragma unroll
      for (int t = 0; t < 3; ++t) {
        const unsigned h = pack_bf16(a, b);
        w[t][i] = h;
        a -= __uint_as_float(h << 16);
        b -= __uint_as_float(h & 0xffff0000u);
      }
    }
#pragma unroll
    for (int t = 0; t < 3; ++t) r.t[t] = __builtin_bit_cast(s16x8, make_uint4(w[t][0], w[t][1], w[t][2], w[t][3]));
  }
  return r;
}

// Eight consecutive elements as they lie in memory (16 bytes of a 16-bit type, 32 of fp32).
template <class T> struct Raw { uint4 w[sizeof(T) / 2]; };
template <class T>
__device__ static inline Raw<T> raw_load(const T* p) {
  Raw<T> r;
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i) r.w[i] = reinterpret_cast<const uint4*>(p)[i];
  return r;
}
template <class T>
__device__ static inline Raw<T> raw_zero() {
  Raw<T> r;
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i) r.w[i] = make_uint4(0, 0, 0, 0);
  return r;
}
template <class T>
__device__ static inline void raw_floats(const Raw<T>& r, float* f) {
  if constexpr (sizeof(T) == 2) {
    Packet<T>::unpack(r.w[0], f);
  } else {
    Packet<float>::unpack(r.w[0], f);
    Packet<float>::unpack(r.w[1], f + 4);
  }
}
template <class T>
__device__ static inline Frag<T> raw_frag(const Raw<T>& r) {
  Frag<T> o;
  if constexpr (sizeof(T) == 2) {
    o.t[0] = __builtin_bit_cast(s16x8, r.w[0]);
  } else {
    float f[8];
    raw_floats<T>(r, f);
    o = make_frag<T>(f);
  }
  return o;
}

// A tile of ROWS x DP values in LDS, one plane per term.  PAD (16-bit values) spreads the rows over the 32 banks: 8 for
// rows() - eight lanes read 16 bytes of eight rows per cycle -, 16 where only cols() reads - four rows of 32 bytes.
template <class T, int ROWS, int DP, int PAD = 8>
struct Tile {
  static constexpr int LD = DP + PAD, NP = Terms<T>::NP, PLANE = ROWS * LD;
  short v[NP * PLANE];
  __device__ inline void put(int row, int col, const Frag<T>& f) {
#pragma unroll
    for (int t = 0; t < NP; ++t) *reinterpret_cast<s16x8*>(&v[t * PLANE + row * LD + col]) = f.t[t];
  }
  // first operand, rows r0 .. r0+31 down, columns col .. col+15 along the sum
  __device__ inline Frag<T> rows(int r0, int col) const {
    const int lane = threadIdx.x & 63;
    Frag<T> f;
#pragma unroll
    for (int t = 0; t < NP; ++t)
      f.t[t] = *reinterpret_cast<const s16x8*>(&v[t * PLANE + (r0 + (lane & 31)) * LD + col + (lane >> 5) * 8]);
    return f;
  }
  // first operand, columns col .. col+31 down, rows r0 .. r0+15 along the sum in the order in which a lane holds the
  // scores of 16 rows: element j of half h is row r0 + 4h + j (j < 4), r0 + 8 + 4h + j - 4 (j >= 4).  The transposing
  // read takes, per 16 lanes, four rows of sixteen 16-bit values (four to a lane) and returns a column to each lane.
  __device__ inline Frag<T> cols(int r0, int col) const {
    const int lane = threadIdx.x & 63, i = lane & 15;
    const int at = (r0 + 4 * (lane >> 5) + (i >> 2)) * LD + col + ((lane >> 4) & 1) * 16 + (i & 3) * 4;
    Frag<T> f;
#pragma unroll
    for (int t = 0; t < NP; ++t) {
      typedef __attribute__((address_space(3))) s16x4 lds4;
      const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(&v[t * PLANE + at]));
      const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(&v[t * PLANE + at + 8 * LD]));
      f.t[t] = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    }
    return f;
  }
};
// row of register r of a 32x32 product, before the 4 * (lane >> 5)
__device__ static constexpr int acc_row(int r) { return (r & 3) + 8 * (r >> 2); }

struct View4 {                                         // [B, T, heads, D]; strides in elements, the last is 1
  const void* p;
  int64_t b, t, h;
};

struct Attn {
  View4 q, k, v, out, dout, dq, dk, dv;
  float* lse;                                          // [B, H, Tq]
  float* delta;                                        // [B, H, Tq]
  const int32_t* sl;
  const uint8_t* mask;
  int64_t mask_ld;
  int B, Tq, Tk, Hkv, G, D;
  float scale, scale2;                                 // scale2 = scale * log2(e)
  int rows, row_tiles, key_tiles, splits, per_split;
  int row_waves, key_waves, row_splits, rows_per;      // waves per block; splits of the row list in the dk / dv pass
  float *part, *part_lse;                              // forward: [splits][B H Tq][D], [splits][B H Tq]; dq: attn_dq_kernel
  float* kept;                                         // few rows: p, then dp, [B Hkv][Tk][R]
  bool near;                                           // a tile's rows lie within 2^31 bytes of its first
  int few, waves, lanes;                               // rows padded to 1, 2 or 4 (0: the tiled kernels); waves per
                                                       // block, lanes per key
};

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

__device__ static inline float minus_inf() { return -__builtin_inff(); }

// Where block `id` of a launch with `per` blocks per pair (sample, key head) works.  The hardware deals consecutive blocks
// to the eight dies in turn; a pair's blocks read the same keys (or rows), so they are kept on one die, whose L2 then
// holds them once.  Die x takes the pairs x, x + 8, ...: the samples of a ragged batch, neighbours in this order, go to
// different dies (500 candidates against up to 1000 events: 42.5 us; 46.5 with blocks of a pair dealt to all dies, 49.6
// with four neighbouring pairs to a die).  Where the pairs would leave some dies a turn short, every die takes blocks of
// all pairs.
struct BlockAt { int pair, part; };
__host__ __device__ static inline bool by_dies(int64_t pairs) { return pairs >= 64 || (pairs & 7) == 0; }
__device__ static inline BlockAt block_at(const Attn& a, int per) {
  const int id = blockIdx.x;
  if (!by_dies((int64_t)a.B * a.Hkv)) return {id / per, id % per};
  const int turn = id >> 3;
  return {turn / per * 8 + (id & 7), turn % per};
}
static int64_t pair_blocks(const Attn& a, int64_t per) {               // blocks of pairs beyond the last one leave at once
  const int64_t pairs = (int64_t)a.B * a.Hkv;
  return (by_dies(pairs) ? (pairs + 7) / 8 * 8 : pairs) * per;
}

__device__ static inline int key_count(const Attn& a, int b) {
  if (!a.sl) return a.Tk;
  return min(max(a.sl[b], 0), a.Tk);
}

// Fewer than two keys left: p is 1 whatever the score, so dq and dk are zero - exactly, not up to the rounding of p.
__device__ static inline bool lone_key(const Attn& a, int b) {
  const int len = key_count(a, b), lane = threadIdx.x & 63;
  if (len < 2) return true;
  if (!a.mask) return false;
  const uint8_t* mask = a.mask + (int64_t)b * a.mask_ld;
  int n = 0;
  for (int base = 0; base < len && n < 2; base += 512) {               // eight loads in flight: the first keys may all be off
    bool on[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) on[i] = mask[min(base + i * 64 + lane, len - 1)] != 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) n += __popcll(__ballot(on[i] && base + i * 64 + lane < len));
  }
  return n < 2;
}

struct RowAt { int t, h; };
// A lane's row again after a loop: without this the compiler keeps the row's addresses in registers all along.
__device__ static inline int row_again(int r0) {
  int lane = threadIdx.x & 31;
  asm volatile("" : "+v"(lane));
  return r0 + lane;
}
__device__ static inline RowAt row_at(const Attn& a, int r, int hk) {
  if (a.G == 1) return {r, hk};
  const int t = r / a.G;
  return {t, hk * a.G + (r - t * a.G)};
}
template <class T>
__device__ static inline const T* row_ptr(const View4& w, int b, const RowAt& ra) {
  return (const T*)w.p + (int64_t)b * w.b + (int64_t)ra.t * w.t + (int64_t)ra.h * w.h;
}
__device__ static inline int64_t row_id(const Attn& a, int b, const RowAt& ra) {
  return ((int64_t)b * (a.Hkv * a.G) + ra.h) * a.Tq + ra.t;
}

// max over a lane and its partner 32 lanes away
__device__ static inline float half_max(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, v), __builtin_bit_cast(unsigned, v), false, false);
  return fmaxf(__builtin_bit_cast(float, (unsigned)r[0]), __builtin_bit_cast(float, (unsigned)r[1]));
}

// The 32 rows from r0 of a row list as second operands: lane holds row r0 + (lane & 31)
template <class T, int DP>
__device__ static inline void load_row_frags(const T* p, bool ok, int D, Frag<T>* f) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int s = 0; s < DP / 16; ++s) {
    const int d = s * 16 + (lane >> 5) * 8;
    f[s] = raw_frag<T>(ok && d < D ? raw_load(p + d) : raw_zero<T>());
  }
}

// A lane's 16 values of one 32-column strip (columns acc_row(r) + 4 * half) to its row, four at a time
template <class T>
__device__ static inline void store_strip(T* row, int col0, int D, const f32x16& acc, float by) {
  const int h4 = 4 * ((threadIdx.x & 63) >> 5);
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const int d = col0 + 8 * g + h4;
    if (d < D) {
      const float a0 = acc[4 * g] * by, a1 = acc[4 * g + 1] * by, a2 = acc[4 * g + 2] * by, a3 = acc[4 * g + 3] * by;
      if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float4*>(row + d) = make_float4(a0, a1, a2, a3);
      } else if constexpr (__is_same(T, bf16_t)) {
        *reinterpret_cast<uint2*>(row + d) = make_uint2(pack_bf16(a0, a1), pack_bf16(a2, a3));
      } else {
        const f16x2 x = {(f16_t)a0, (f16_t)a1}, y = {(f16_t)a2, (f16_t)a3};
        *reinterpret_cast<uint2*>(row + d) = make_uint2(__builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, y));
      }
    }
  }
}

// Registers of a thread on the way from memory to a tile: ROWS rows of DP values, dealt to THREADS.  Loads are
// unconditional: a row behind the end reads the last one, a column behind D the first, both stay in bounds and are
// zeroed (rows) or never stored (columns) by put().  As long as whole tiles lie inside, a thread's offsets from the
// tile's first row are the same for every tile, so the loop adds nothing per lane.
template <class T, int ROWS, int DP, int THREADS>
struct Stage {
  static constexpr int PER = DP / 8, N = (ROWS * PER + THREADS - 1) / THREADS;
  static constexpr bool EVEN = THREADS % PER == 0;     // a thread's packets lie in one column, THREADS / PER rows apart
  Raw<T> a[N];
  unsigned off[EVEN ? 1 : N];                          // byte offsets of its packets (EVEN: of the first) in a whole tile
  __device__ static inline int row(int i) { return (int)(threadIdx.x + i * THREADS) / PER; }
  __device__ static inline int col(int i) { return (int)(threadIdx.x + i * THREADS) % PER * 8; }
  __device__ inline void load(const T* first, int64_t step) {           // step: elements between a thread's packets (EVEN)
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const char* p = reinterpret_cast<const char*>(EVEN ? first + i * step : first);
      a[i] = raw_load(reinterpret_cast<const T*>(p + off[EVEN ? 0 : i]));
    }
  }
  __device__ inline void keys_init(const Attn& p, const View4& w) {
#pragma unroll
    for (int i = 0; i < (EVEN ? 1 : N); ++i)
      off[i] = (unsigned)((min(row(i), ROWS - 1) * w.t + (col(i) < p.D ? col(i) : 0)) * sizeof(T));
  }
  // keys k0 .. of one (sample, head), k0 < k1
  __device__ inline void keys(const Attn& p, const View4& w, const T* base, int k0, int k1) {
    if (k0 + ROWS <= k1 && p.near) return load(base + (int64_t)k0 * w.t, THREADS / PER * w.t);
#pragma unroll
    for (int i = 0; i < N; ++i)
      a[i] = raw_load(base + (int64_t)min(k0 + row(i), k1 - 1) * w.t + (col(i) < p.D ? col(i) : 0));
  }
  // bit i: the mask leaves the key of packet i
  __device__ static inline unsigned mask_bits(const uint8_t* mask, int k0, int k1) {
    unsigned on = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) on |= (mask[min(k0 + row(i), k1 - 1)] != 0 ? 1u : 0u) << i;
    return on;
  }
  __device__ inline void list_init(const Attn& p, const View4& w) {
#pragma unroll
    for (int i = 0; i < (EVEN ? 1 : N); ++i) {
      const int r = min(row(i), ROWS - 1), t = r / p.G, h = r - t * p.G;
      off[i] = (unsigned)((t * w.t + h * w.h + (col(i) < p.D ? col(i) : 0)) * sizeof(T));
    }
  }
  // rows r0 .. of the row list, r0 < rows
  __device__ inline void list(const Attn& p, const View4& w, int b, int hk, int r0) {
    // whole groups between a thread's packets: G divides ROWS and their distance
    constexpr int APART = EVEN && N > 1 ? THREADS / PER : ROWS;
    if (r0 + ROWS <= p.rows && APART % p.G == 0 && p.near)
      return load(row_ptr<T>(w, b, {r0 / p.G, hk * p.G}), APART / p.G * w.t);
#pragma unroll
    for (int i = 0; i < N; ++i)
      a[i] = raw_load(row_ptr<T>(w, b, row_at(p, min(r0 + row(i), p.rows - 1), hk)) + (col(i) < p.D ? col(i) : 0));
  }
  // the tile holds rows first .. of `end`; rows behind the end and masked ones (bit i of on: kept) become zeros
  template <class TILE>
  __device__ inline void put(TILE& t, int D, int first, int end, bool masked = false, unsigned on = 0) const {
    if (first + ROWS <= end && !masked) {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (row(i) < ROWS && col(i) < D) t.put(row(i), col(i), raw_frag<T>(a[i]));
      return;
    }
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (row(i) < ROWS && col(i) < D) {
        const bool in = first + row(i) < end && (!masked || (on >> i & 1));
        t.put(row(i), col(i), raw_frag<T>(in ? a[i] : raw_zero<T>()));
      }
  }
};

// LDS starts as zeros where the head size leaves columns of a tile unwritten (0 * NaN in the products over d otherwise)
template <class TILE>
__device__ static inline void clear_tile(TILE& t) {
  constexpr int N = sizeof(t.v) / 16;
  static_assert(sizeof(t.v) % 16 == 0, "16-byte rows");
  for (int i = threadIdx.x; i < N; i += blockDim.x) reinterpret_cast<uint4*>(t.v)[i] = make_uint4(0, 0, 0, 0);
}

// Bit i: key k0 + i may be attended to
__device__ static inline uint64_t key_bits(const uint8_t* mask, int k0, int k1, int n) {
  const int lane = threadIdx.x & 63, key = k0 + lane;
  return __ballot(lane < n && key < k1 && (!mask || mask[key]));
}
// -infinity for the scores of the keys that strip i of a tile leaves out: a bit as a word of ones or zeros, and a select
// by it, two instructions per score.
__device__ static inline void leave_out(f32x16& s, uint64_t bits, int i) {
  const unsigned off = ~(unsigned)(bits >> (32 * i)) >> (4 * ((threadIdx.x & 63) >> 5));
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const unsigned all = (unsigned)__builtin_amdgcn_sbfe((int)off, acc_row(e), 1);
    s[e] = __uint_as_float((all & 0xff800000u) | (~all & __float_as_uint(s[e])));
  }
}

// Waves per SIMD the tiled kernels are built for.  Two keep a wave within 256 registers, and only then does the compiler
// leave the accumulators where the vector units reach them: at one (512 registers) it keeps them in the other half of
// the register file and moves every value over and back (a third of the instructions of the forward's loop).  Three spill
// in the backward (head size 64: 940 and 1000 us for 600 and 710).  At two some blocks of one and two waves spill as well,
// by the compiler's report (registers per lane, bf16 / fp16): dq of one wave 66 / 70 at head size 96 and 81 / 88 at 128, of
// two waves 4 / 0 and 21 / 32; dk / dv of two waves 50 / 67 at 128; fp32 dk / dv 77 by one wave and 8 by four at 64, 64 by
// four at 128.  Those are many samples of short sequences (4096 pairs of 20 rows and 500 keys of 128, bf16: dq 356 us).
template <class T, int DP>
constexpr int WAVES = Terms<T>::NP == 3 && DP > 64 ? 1 : 2;
// The forward of 16-bit tensors needs fewer registers: at head sizes up to 64, blocks of four waves run four to a SIMD
// (16 heads of 2048 x 4096 of 64, batch 8, bf16: 369 us; 410 with three).  Above that, and for fp32, more change nothing.
template <class T, int DP, int NW>
constexpr int FWD_WAVES = NW == 4 && Terms<T>::NP == 1 && DP <= 64 ? 4 : WAVES<T, DP>;

// A wave of the backward has two operands of its own (rows of q and dout, or keys of k and v).  16-bit types above head
// size 64: the second stays in LDS, in registers it spills (4 x 16 heads of 1024 x 1024 of 128, bf16: dq 89 us and dk / dv
// 97 for 123 and 137) - but not with single waves on keys of 128, which LDS then limits (4096 pairs of 500 rows and 30
// keys: 304 us for 358).  Head size 64, dk / dv: with that operand in LDS and tiles of 32 rows three waves fit a SIMD (660 us
// for the shape above, 710 with two), and in blocks of two waves fp16 spills no more (4096 pairs of 500 rows and 60 keys:
// 199 us for 244; bf16 192 for 178).  dq gains nothing from it.
template <class T, int DP, int NW>
constexpr int DKV_WAVES = NW == 4 && Terms<T>::NP == 1 && DP == 64 ? 3 : WAVES<T, DP>;
template <class T, int DP, int NW>
constexpr bool DKV_ASIDE = Terms<T>::NP == 1 && (NW == 1 ? DP == 96 : DP >= 64);
template <class T, int DP>
constexpr bool DQ_ASIDE = Terms<T>::NP == 1 && DP > 64;

// ---- forward -------------------------------------------------------------------------------------------------------
// A wave owns 32 query rows; the NW waves of a block share each tile of KT keys.  Two tiles of LDS and one barrier per
// tile: behind it tile i + 1 goes from registers to the buffer that tile i - 1 has left, tile i + 2 is requested, and
// tile i is computed.  One wave alone needs neither.
// The running maximum is a reference, not the maximum itself: accumulators and sum are rescaled only when a score passes
// it by more than LIMIT (a power of two), so p stays below 2^(BIAS + LIMIT) and after the first tiles that is rare.
// (fp16: 2^15, the largest power it holds.)  Tiles of 64 keys where two buffers of them leave room for the waves: 16-bit
// types up to head size 64 (369 us for the shape above; 416 with 32), 32 keys otherwise (head size 128, 4 x 16 heads of
// 1025 x 2047: 121 us; 206 with 64; fp32, head size 32, 2048 pairs of 100 x 200: 41 us; 50 with 64).
template <class T, int DP, int NW, int KT>
__global__ __launch_bounds__(NW * 64, (FWD_WAVES<T, DP, NW>)) void attn_fwd_kernel(Attn a) {
  constexpr int NS = KT / 32, NK = DP / 16, ND = DP / 32, NBUF = NW > 1 ? 2 : 1;
  constexpr float BIAS = __is_same(T, f16_t) ? 8.f : 0.f, LIMIT = 7.f;
  __shared__ Tile<T, KT, DP> kt[NBUF];
  __shared__ Tile<T, KT, DP, 16> vt[NBUF];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const BlockAt ba = block_at(a, a.row_tiles * a.splits);
  if (ba.pair >= a.B * a.Hkv) return;
  const int split = ba.part % a.splits, tile = ba.part / a.splits, b = ba.pair / a.Hkv, hk = ba.pair - b * a.Hkv;
  const int k0 = split * a.per_split, k1 = min(key_count(a, b), k0 + a.per_split);
  const int r0 = (tile * NW + wave) * 32;
  const bool busy = r0 < a.rows;
  const T* kp = (const T*)a.k.p + (int64_t)b * a.k.b + (int64_t)hk * a.k.h;
  const T* vp = (const T*)a.v.p + (int64_t)b * a.v.b + (int64_t)hk * a.v.h;
  const uint8_t* mask = a.mask ? a.mask + (int64_t)b * a.mask_ld : nullptr;

  Stage<T, KT, DP, NW * 64> nk, nv;
  nk.keys_init(a, a.k);
  nv.keys_init(a, a.v);
  unsigned left = 0;
  auto load = [&](int kb) {
    if (kb >= k1) return;
    nk.keys(a, a.k, kp, kb, k1);
    nv.keys(a, a.v, vp, kb, k1);
    if (mask) left = nk.mask_bits(mask, kb, k1);
  };
  auto put = [&](int buf, int kb) {
    if (kb >= k1) return;
    nk.put(kt[buf], a.D, kb, k1, mask, left);
    nv.put(vt[buf], a.D, kb, k1, mask, left);
  };
  load(k0);
  Frag<T> qf[NK];
  {
    const int r = r0 + (lane & 31);
    load_row_frags<T, DP>(row_ptr<T>(a.q, b, row_at(a, r < a.rows ? r : 0, hk)), r < a.rows, a.D, qf);
  }
  f32x16 o[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d) o[d] = f32x16{};
  float m = minus_inf(), l = 0.f;
  if (a.D < DP) {
#pragma unroll
    for (int i = 0; i < NBUF; ++i) clear_tile(kt[i]);
    __syncthreads();
  }
  if constexpr (NBUF == 2) {
    put(0, k0);
    load(k0 + KT);
  }
  int at = 0;
  for (int kb = k0; kb < k1; kb += KT) {
    __syncthreads();
    if constexpr (NBUF == 2) {
      put(at ^ 1, kb + KT);
      load(kb + 2 * KT);
    } else {
      put(0, kb);
      load(kb + KT);
      __syncthreads();
    }
    const auto& ks = kt[at];
    const auto& vs = vt[at];
    if constexpr (NBUF == 2) at ^= 1;
    if (!busy) continue;
    const bool whole = !mask && kb + KT <= k1;
    const uint64_t bits = whole ? 0 : key_bits(mask, kb, k1, KT);
    if (!whole && !bits) continue;                     // the mask leaves nothing of this tile
    f32x16 s[NS];
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      s[i] = f32x16{};
#pragma unroll
      for (int c = 0; c < NK; ++c) s[i] = mfma<T>(ks.rows(i * 32, c * 16), qf[c], s[i]);
    }
    if (!whole) {
#pragma unroll
      for (int i = 0; i < NS; ++i) leave_out(s[i], bits, i);
    }
    float top = s[0][0];
#pragma unroll
    for (int i = 0; i < NS; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) top = fmaxf(top, s[i][e]);
    top = half_max(top);
    if (__any((top - m) * a.scale2 > LIMIT)) {         // a row's first score is infinitely far from m
      const float to = fmaxf(m, top);
      const float fade = to == minus_inf() ? 1.f : __builtin_amdgcn_exp2f((m - to) * a.scale2);
      m = to;
      l *= fade;
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[d][e] *= fade;
    }
    const float shift = BIAS - (m == minus_inf() ? 0.f : m) * a.scale2;      // nothing seen yet: p = 2^-inf
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < NS; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        s[i][e] = __builtin_amdgcn_exp2f(fmaf(s[i][e], a.scale2, shift));
        sum += s[i][e];
      }
    l += sum;
#pragma unroll
    for (int i = 0; i < NS; ++i)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float f[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = s[i][c * 8 + j];
        const Frag<T> pf = make_frag<T>(f);
#pragma unroll
        for (int d = 0; d < ND; ++d) o[d] = mfma<T>(vs.cols(i * 32 + c * 16, d * 32), pf, o[d]);
      }
  }
  const float sum = half_swap_sum(l, l);
  const int r = row_again(r0);
  if (r >= a.rows) return;
  const RowAt ra = row_at(a, r, hk);
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  const int64_t rid = row_id(a, b, ra);
  const float lse = sum == 0.f ? minus_inf() : m * a.scale + (logf(sum) - BIAS * LN2);
  if (a.splits == 1) {
    T* dst = const_cast<T*>(row_ptr<T>(a.out, b, ra));
#pragma unroll
    for (int d = 0; d < ND; ++d) store_strip<T>(dst, d * 32, a.D, o[d], inv);
    if (a.lse && lane < 32) a.lse[rid] = lse;
  } else {
    const int64_t to = (int64_t)split * ((int64_t)a.B * a.Hkv * a.rows) + rid;
    float* dst = a.part + to * a.D;
#pragma unroll
    for (int d = 0; d < ND; ++d) store_strip<float>(dst, d * 32, a.D, o[d], inv);
    if (lane < 32) a.part_lse[to] = lse;
  }
}

// A row's place in a [B, T, heads, D] view from its number
template <class T>
__device__ static inline T* row_of(const Attn& a, const View4& w, int64_t rid) {
  const int H = a.Hkv * a.G;
  const int64_t bhead = rid / a.Tq;
  const RowAt ra = {(int)(rid - bhead * a.Tq), (int)(bhead % H)};
  return const_cast<T*>(row_ptr<T>(w, (int)(bhead / H), ra));
}

// Joins the splits of a row: sum over i of weight(i) * part[i], in split order.  Few splits: a thread per four columns of
// a row walks them all; from JOIN_WIDE on, a block per row, eight groups of 32 threads take every eighth split and are
// added in group order (one thread over 128 splits took 33 us where the forward before it took 48).
constexpr int JOIN_WIDE = 8;
template <class T, bool WIDE>
__global__ __launch_bounds__(256) void attn_join_kernel(Attn a, int64_t n_rows) {
  const int quads = a.D / 4;
  int64_t rid;
  int quad, first = 0, every = 1;
  if constexpr (WIDE) {
    rid = blockIdx.x;
    quad = threadIdx.x & 31;
    first = threadIdx.x >> 5;
    every = 8;
  } else {
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (id >= n_rows * quads) return;
    rid = id / quads;
    quad = (int)(id - rid * quads);
  }
  const int d = quad * 4;
  float top = minus_inf();
  if constexpr (WIDE) {
    for (int i = threadIdx.x & 63; i < a.splits; i += 64) top = fmaxf(top, a.part_lse[i * n_rows + rid]);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
  } else {
    for (int i = 0; i < a.splits; ++i) top = fmaxf(top, a.part_lse[i * n_rows + rid]);
  }
  const float base = top == minus_inf() ? 0.f : top;
  float sum = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int i = first; i < a.splits; i += every) {
    const float w = expf(a.part_lse[i * n_rows + rid] - base);
    sum += w;
    if (quad < quads) {
      const float4 v = *reinterpret_cast<const float4*>(a.part + (i * n_rows + rid) * a.D + d);
      acc[0] = fmaf(w, v.x, acc[0]);
      acc[1] = fmaf(w, v.y, acc[1]);
      acc[2] = fmaf(w, v.z, acc[2]);
      acc[3] = fmaf(w, v.w, acc[3]);
    }
  }
  if constexpr (WIDE) {
    __shared__ float red[8][32][5];
    float* mine = red[first][quad];
    mine[0] = acc[0]; mine[1] = acc[1]; mine[2] = acc[2]; mine[3] = acc[3]; mine[4] = sum;
    __syncthreads();
    if (first) return;
    for (int g = 1; g < 8; ++g) {
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[j] += red[g][quad][j];
      sum += red[g][quad][4];
    }
    if (quad >= quads) return;
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  T* dst = row_of<T>(a, a.out, rid) + d;
#pragma unroll
  for (int j = 0; j < 4; ++j) dst[j] = (T)(acc[j] * inv);
  if (a.lse && d == 0) a.lse[rid] = sum == 0.f ? minus_inf() : base + logf(sum);
}

// ---- backward ------------------------------------------------------------------------------------------------------
// fp16: keeps ds * factor below 2^15 with a power of two per lane that only ever shrinks; the accumulators and the sum
// follow it
template <int ND>
__device__ static inline float fit_f16(const f32x16& ds, float factor, f32x16* acc, float& sum) {
  float top = 0.f;
#pragma unroll
  for (int r = 0; r < 16; ++r) top = fmaxf(top, fabsf(ds[r]));
  top = half_max(top);
  const bool over = top * factor > 16384.f;
  if (__any(over)) {
    const float next = over ? ldexpf(1.f, 13 - ilogbf(fminf(top, 3.0e38f))) : factor;
    const float by = next / factor;
    factor = next;
    sum *= by;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[d][r] *= by;
  }
  return factor;
}
// sum + the eight 16-bit values of an operand, in fp32
template <class T>
__device__ static inline float add_frag(const Frag<T>& f, float sum) {
  const uint4 w = __builtin_bit_cast(uint4, f.t[0]);
  const unsigned u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (__is_same(T, f16_t)) {
      const f16x2 one = {(f16_t)1.f, (f16_t)1.f};
      sum = __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, u[i]), one, sum, false);
    } else {
      const bf16x2 one = {(bf16_t)1.f, (bf16_t)1.f};
      sum = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, u[i]), one, sum, false);
    }
  }
  return sum;
}
constexpr float F16_FACTOR0 = 1.2676506e30f;           // 2^100: the first strip with a gradient sets the factor

// dq, and delta for the dk / dv pass.  A wave owns 32 query rows; buffers and barrier as in the forward, both tiles at
// the same distance.
// For 16-bit tensors delta = sum_d dout out carries the rounding of out, the same error e for every key of a row: dq
// would be off by e times the row's mean key, dk alike.  The sum of ds over all keys is exactly that error (it is zero
// otherwise), so it is summed in fp32, put into delta for the dk / dv pass, and taken out of dq with the row's mean key
// (KEYS: sum p k, a second product per strip over operands that are there already).  For dq it is the sum of the rounded
// ds that is taken out: what their roundings have in common over the keys goes with it (8 rows against 14000 keys, bf16:
// dq 0.26 % off instead of 0.27; 40 against 3: 0.21 instead of 0.25; 0.17 to 0.2 are the last rounding's; 635 us for
// the shape above, 600 without).
template <class T, int DP, int NW, int KT>
__global__ __launch_bounds__(NW * 64, (WAVES<T, DP>)) void attn_dq_kernel(Attn a) {
  constexpr int NS = KT / 32, NK = DP / 16, ND = DP / 32, NBUF = NW > 1 ? 2 : 1;
  constexpr bool F16 = __is_same(T, f16_t), KEYS = Terms<T>::NP == 1;
  constexpr bool ASIDE = DQ_ASIDE<T, DP>;
  __shared__ Tile<T, KT, DP> kt[NBUF], vt[NBUF];
  __shared__ Tile<T, ASIDE ? 32 : 1, DP> mine[ASIDE ? NW : 1];         // a wave's own rows of dout
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const BlockAt ba = block_at(a, a.row_tiles * a.splits);
  if (ba.pair >= a.B * a.Hkv) return;
  const int split = ba.part % a.splits, tile = ba.part / a.splits, b = ba.pair / a.Hkv, hk = ba.pair - b * a.Hkv;
  const int k0 = split * a.per_split, k1 = min(key_count(a, b), k0 + a.per_split);
  const int r0 = (tile * NW + wave) * 32;
  const bool busy = r0 < a.rows;
  const T* kp = (const T*)a.k.p + (int64_t)b * a.k.b + (int64_t)hk * a.k.h;
  const T* vp = (const T*)a.v.p + (int64_t)b * a.v.b + (int64_t)hk * a.v.h;
  const uint8_t* mask = a.mask ? a.mask + (int64_t)b * a.mask_ld : nullptr;

  Stage<T, KT, DP, NW * 64> nk, nv;
  nk.keys_init(a, a.k);
  nv.keys_init(a, a.v);
  unsigned left = 0;
  auto is_whole = [&](int kb) { return !mask && kb + KT <= k1; };
  auto load = [&](int kb) {
    if (kb >= k1) return;
    nk.keys(a, a.k, kp, kb, k1);
    nv.keys(a, a.v, vp, kb, k1);
    if (mask) left = nk.mask_bits(mask, kb, k1);
  };
  auto put = [&](int buf, int kb) {
    if (kb >= k1) return;
    nk.put(kt[buf], a.D, kb, k1, mask, left);
    nv.put(vt[buf], a.D, kb, k1, mask, left);
  };
  load(k0);
  Frag<T> qf[NK], gf[ASIDE ? 1 : NK];
  float delta = 0.f, shift = minus_inf();              // a row without keys: p = 2^-inf
  {
    const int r = r0 + (lane & 31);
    const bool in = r < a.rows;
    const RowAt ra = row_at(a, in ? r : 0, hk);
    load_row_frags<T, DP>(row_ptr<T>(a.q, b, ra), in, a.D, qf);
    const T* gp = row_ptr<T>(a.dout, b, ra);
    const T* op = row_ptr<T>(a.out, b, ra);
#pragma unroll
    for (int s = 0; s < NK; ++s) {
      const int d = s * 16 + (lane >> 5) * 8;
      const bool ok = in && d < a.D;
      const Raw<T> g = ok ? raw_load(gp + d) : raw_zero<T>(), w = ok ? raw_load(op + d) : raw_zero<T>();
      float gv[8], wv[8];
      raw_floats<T>(g, gv);
      raw_floats<T>(w, wv);
#pragma unroll
      for (int j = 0; j < 8; ++j) delta = fmaf(gv[j], wv[j], delta);
      if constexpr (ASIDE) mine[wave].put(lane & 31, d, raw_frag<T>(g));
      else gf[s] = raw_frag<T>(g);
    }
    delta = half_swap_sum(delta, delta);
    if (in) {
      const float lse = a.lse[row_id(a, b, ra)];
      shift = lse == minus_inf() ? minus_inf() : Terms<T>::BIAS - lse * LOG2E;
    }
  }
  f32x16 acc[ND], keys[KEYS ? ND : 1];
#pragma unroll
  for (int d = 0; d < ND; ++d) acc[d] = f32x16{};
#pragma unroll
  for (int d = 0; d < (KEYS ? ND : 1); ++d) keys[d] = f32x16{};
  float factor = F16 ? F16_FACTOR0 : 1.f, rest = 0.f, drop = 0.f;    // sums of ds and of the rounded ds * factor

  auto tile_work = [&](int buf, bool whole, int kb) {
    const uint64_t bits = whole ? 0 : key_bits(mask, kb, k1, KT);
    if (!whole && !bits) return;                       // the mask leaves nothing of this tile
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      f32x16 s = f32x16{}, dp = f32x16{};
#pragma unroll
      for (int c = 0; c < NK; ++c) {
        s = mfma<T>(kt[buf].rows(i * 32, c * 16), qf[c], s);
        if constexpr (ASIDE) dp = mfma<T>(vt[buf].rows(i * 32, c * 16), mine[wave].rows(0, c * 16), dp);
        else dp = mfma<T>(vt[buf].rows(i * 32, c * 16), gf[c], dp);
      }
      if (!whole) leave_out(s, bits, i);
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        s[e] = __builtin_amdgcn_exp2f(fmaf(s[e], a.scale2, shift));
        dp[e] = s[e] * (dp[e] - delta);
        if (KEYS) rest += dp[e];
      }
      if constexpr (F16) factor = fit_f16<ND>(dp, factor, acc, drop);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float f[8], e[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          f[j] = F16 ? dp[c * 8 + j] * factor : dp[c * 8 + j];
          e[j] = s[c * 8 + j];
        }
        const Frag<T> df = make_frag<T>(f);
        Frag<T> pf;
        if constexpr (KEYS) {
          pf = make_frag<T>(e);
          drop = add_frag<T>(df, drop);
        }
#pragma unroll
        for (int d = 0; d < ND; ++d) {
          const Frag<T> kf = kt[buf].cols(i * 32 + c * 16, d * 32);
          acc[d] = mfma<T>(kf, df, acc[d]);
          if constexpr (KEYS) keys[d] = mfma<T>(kf, pf, keys[d]);
        }
      }
    }
  };
  if (a.D < DP) {
#pragma unroll
    for (int i = 0; i < NBUF; ++i) {
      clear_tile(kt[i]);
      clear_tile(vt[i]);
    }
    __syncthreads();
  }
  if constexpr (NBUF == 2) {
    put(0, k0);
    load(k0 + KT);
  }
  int at = 0;
  for (int kb = k0; kb < k1; kb += KT) {
    __syncthreads();
    if constexpr (NBUF == 2) {
      put(at ^ 1, kb + KT);
      load(kb + 2 * KT);
    } else {
      put(0, kb);
      load(kb + KT);
      __syncthreads();
    }
    if (busy) tile_work(at, is_whole(kb), kb);
    if constexpr (NBUF == 2) at ^= 1;
  }
  constexpr float unbias = 1.f / (1 << (int)Terms<T>::BIAS);
  rest = half_swap_sum(rest, rest) * unbias;
  drop = half_swap_sum(drop, drop) * (unbias / factor);
  if (lone_key(a, b)) {
    rest = drop = 0.f;
#pragma unroll
    for (int d = 0; d < ND; ++d) acc[d] = f32x16{};
  }
  const int r = row_again(r0);
  if (r >= a.rows) return;
  const RowAt ra = row_at(a, r, hk);
  const int64_t rid = row_id(a, b, ra);
  if (a.splits == 1) {
    if (lane < 32) a.delta[rid] = delta + rest;
    T* dst = const_cast<T*>(row_ptr<T>(a.dq, b, ra));
#pragma unroll
    for (int d = 0; d < ND; ++d) {
      if constexpr (KEYS)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[d][e] = acc[d][e] * (unbias / factor) - drop * (keys[d][e] * unbias);
      store_strip<T>(dst, d * 32, a.D, acc[d], a.scale);
    }
  } else {                                             // sum ds k, then sum p k; both sums of ds; the join follows
    const int64_t n_rows = (int64_t)a.B * a.Hkv * a.rows;
    float* dst = a.part + ((int64_t)split * n_rows + rid) * (KEYS ? 2 * a.D : a.D);
#pragma unroll
    for (int d = 0; d < ND; ++d) {
      store_strip<float>(dst, d * 32, a.D, acc[d], unbias / factor);
      if constexpr (KEYS) store_strip<float>(dst + a.D, d * 32, a.D, keys[d], unbias);
    }
    if (lane < 32) {
      if constexpr (KEYS)
        *reinterpret_cast<float2*>(a.part_lse + 2 * ((int64_t)split * n_rows + rid)) = make_float2(rest, drop);
      if (split == 0) a.delta[rid] = delta;
    }
  }
}

// dk and dv.  A wave owns 32 keys and walks the query rows in tiles of QB: 64 where registers allow (head size 32: fp32
// 100 us for 2048 pairs of 100 x 200, 113 with 32; bf16 209 us for 8 x 16 heads of 2048 x 2048, 225 with 32), else 32.
// Single waves of fp32 do with one buffer, for two leave LDS for two waves per CU (2048 pairs of 200 rows and 30 keys of 96:
// 302 us for 453); for 16-bit types the registers bound that number.
template <class T, int DP, int NW, int QB>
__global__ __launch_bounds__(NW * 64, (DKV_WAVES<T, DP, NW>)) void attn_dkv_kernel(Attn a) {
  constexpr int NS = QB / 32, NK = DP / 16, ND = DP / 32, NBUF = NW > 1 || Terms<T>::NP == 1 ? 2 : 1;
  constexpr bool F16 = __is_same(T, f16_t);
  constexpr bool ASIDE = DKV_ASIDE<T, DP, NW>;
  __shared__ Tile<T, QB, DP> qt[NBUF], gt[NBUF];
  __shared__ Tile<T, ASIDE ? 32 : 1, DP> mine[ASIDE ? NW : 1];         // a wave's own rows of v
  __shared__ float4 shift_s[NBUF][QB / 4], delta_s[NBUF][QB / 4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const BlockAt ba = block_at(a, a.key_tiles * a.row_splits);
  if (ba.pair >= a.B * a.Hkv) return;
  const int split = ba.part % a.row_splits, tile = ba.part / a.row_splits, b = ba.pair / a.Hkv, hk = ba.pair - b * a.Hkv;
  const int len = key_count(a, b);
  const int row0 = split * a.rows_per, row1 = min(a.rows, row0 + a.rows_per);
  const int key0 = tile * NW * 32, key = key0 + wave * 32 + (lane & 31);
  const bool on = key < len && (!a.mask || a.mask[(int64_t)b * a.mask_ld + key]);
  const bool busy = __any(on);
  f32x16 dk[ND], dv[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d) dk[d] = dv[d] = f32x16{};
  float factor = F16 ? F16_FACTOR0 : 1.f, none = 0.f;
  if (key0 < len && row0 < row1) {
    Stage<T, QB, DP, NW * 64> nq, ng;
    nq.list_init(a, a.q);
    ng.list_init(a, a.dout);
    float lse_n = 0.f, delta_n = 0.f;
    auto load = [&](int r0) {
      if (r0 >= row1) return;
      nq.list(a, a.q, b, hk, r0);
      ng.list(a, a.dout, b, hk, r0);
      if (threadIdx.x < QB) {
        const int r = r0 + threadIdx.x;
        lse_n = minus_inf();
        delta_n = 0.f;
        if (r < a.rows) {
          const int64_t rid = row_id(a, b, row_at(a, r, hk));
          lse_n = a.lse[rid];
          delta_n = a.delta[rid];
        }
      }
    };
    auto put = [&](int buf, int r0) {
      if (r0 >= row1) return;
      nq.put(qt[buf], a.D, 0, QB);                      // rows behind the list repeat its last one: their p is 2^-inf
      ng.put(gt[buf], a.D, 0, QB);
      if (threadIdx.x < QB) {
        reinterpret_cast<float*>(shift_s[buf])[threadIdx.x] = lse_n == minus_inf() ? minus_inf() : Terms<T>::BIAS - lse_n * LOG2E;
        reinterpret_cast<float*>(delta_s[buf])[threadIdx.x] = delta_n;
      }
    };
    load(row0);
    Frag<T> kf[NK], vf[ASIDE ? 1 : NK];
    load_row_frags<T, DP>((const T*)a.k.p + (int64_t)b * a.k.b + (int64_t)hk * a.k.h + (int64_t)(on ? key : 0) * a.k.t, on, a.D, kf);
    const T* vp = (const T*)a.v.p + (int64_t)b * a.v.b + (int64_t)hk * a.v.h + (int64_t)(on ? key : 0) * a.v.t;
    if constexpr (ASIDE) {
#pragma unroll
      for (int s = 0; s < NK; ++s) {
        const int d = s * 16 + (lane >> 5) * 8;
        mine[wave].put(lane & 31, d, raw_frag<T>(on && d < a.D ? raw_load(vp + d) : raw_zero<T>()));
      }
    } else {
      load_row_frags<T, DP>(vp, on, a.D, vf);
    }
    if (a.D < DP) {
#pragma unroll
      for (int i = 0; i < NBUF; ++i) {
        clear_tile(qt[i]);
        clear_tile(gt[i]);
      }
      __syncthreads();
    }
    auto tile_work = [&](int buf) {
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        f32x16 s = f32x16{}, dp = f32x16{};
#pragma unroll
        for (int c = 0; c < NK; ++c) {
          s = mfma<T>(qt[buf].rows(i * 32, c * 16), kf[c], s);
          if constexpr (ASIDE) dp = mfma<T>(gt[buf].rows(i * 32, c * 16), mine[wave].rows(0, c * 16), dp);
          else dp = mfma<T>(gt[buf].rows(i * 32, c * 16), vf[c], dp);
        }
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int g4 = i * 8 + 2 * g + (lane >> 5);   // rows i * 32 + 8 g + 4 half .. + 3
          const float4 sh = shift_s[buf][g4], de = delta_s[buf][g4];
          const float shv[4] = {sh.x, sh.y, sh.z, sh.w}, dev[4] = {de.x, de.y, de.z, de.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float p = __builtin_amdgcn_exp2f(fmaf(s[4 * g + j], a.scale2, shv[j]));
            const float ds = p * (dp[4 * g + j] - dev[j]);
            s[4 * g + j] = p;
            dp[4 * g + j] = ds;
          }
        }
        if constexpr (F16) factor = fit_f16<ND>(dp, factor, dk, none);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float f[8], e[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            f[j] = s[c * 8 + j];
            e[j] = F16 ? dp[c * 8 + j] * factor : dp[c * 8 + j];
          }
          const Frag<T> pf = make_frag<T>(f), df = make_frag<T>(e);
#pragma unroll
          for (int d = 0; d < ND; ++d) {
            dv[d] = mfma<T>(gt[buf].cols(i * 32 + c * 16, d * 32), pf, dv[d]);
            dk[d] = mfma<T>(qt[buf].cols(i * 32 + c * 16, d * 32), df, dk[d]);
          }
        }
      }
    };
    if constexpr (NBUF == 2) {
      put(0, row0);
      load(row0 + QB);
    }
    int at = 0;
    for (int r0 = row0; r0 < row1; r0 += QB) {
      __syncthreads();
      if constexpr (NBUF == 2) {
        put(at ^ 1, r0 + QB);
        load(r0 + 2 * QB);
      } else {
        put(0, r0);
        load(r0 + QB);
        __syncthreads();
      }
      if (busy) tile_work(at);
      if constexpr (NBUF == 2) at ^= 1;
    }
  }
  const bool lone = lone_key(a, b);
  if (key >= a.Tk) return;
  if (!on) factor = 1.f;
  constexpr float one = 1.f / (1 << (int)Terms<T>::BIAS);   // ds carries p's factor too
  if (a.row_splits > 1) {                              // fp32, both of a key side by side; attn_key_sum_kernel follows
    float* to = a.part + ((int64_t)(split * a.B + b) * a.Hkv + hk) * a.Tk * 2 * a.D + (int64_t)key * 2 * a.D;
#pragma unroll
    for (int d = 0; d < ND; ++d) {
      if (lone) dk[d] = f32x16{};
      if (!on) dk[d] = dv[d] = f32x16{};
      store_strip<float>(to, d * 32, a.D, dk[d], a.scale * one / factor);
      store_strip<float>(to + a.D, d * 32, a.D, dv[d], one);
    }
    return;
  }
  T* kd = (T*)a.dk.p + (int64_t)b * a.dk.b + (int64_t)key * a.dk.t + (int64_t)hk * a.dk.h;
  T* vd = (T*)a.dv.p + (int64_t)b * a.dv.b + (int64_t)key * a.dv.t + (int64_t)hk * a.dv.h;
#pragma unroll
  for (int d = 0; d < ND; ++d) {
    if (lone) dk[d] = f32x16{};
    if (!on) dk[d] = dv[d] = f32x16{};                  // a key that is left out: its lane computed with zeros for k, v
    store_strip<T>(kd, d * 32, a.D, dk[d], a.scale * one / factor);
    store_strip<T>(vd, d * 32, a.D, dv[d], one);
  }
}

// dk and dv from the row splits, in split order: a thread per four columns of a key
template <class T>
__global__ __launch_bounds__(256) void attn_key_sum_kernel(Attn a) {
  const int quads = a.D / 4;
  const int64_t n_keys = (int64_t)a.B * a.Hkv * a.Tk, id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (id >= n_keys * 2 * quads) return;
  const int64_t at = id / (2 * quads);                 // (b, hk, key)
  const int w = (int)(id - at * 2 * quads), d = w % quads * 4;
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
  for (int i = 0; i < a.row_splits; ++i) {
    const float4 v = *reinterpret_cast<const float4*>(a.part + ((int64_t)i * n_keys + at) * 2 * a.D + w * 4);
    acc[0] += v.x;
    acc[1] += v.y;
    acc[2] += v.z;
    acc[3] += v.w;
  }
  const int64_t pair = at / a.Tk;
  const RowAt ra = {(int)(at - pair * a.Tk), (int)(pair % a.Hkv)};
  T* dst = const_cast<T*>(row_ptr<T>(w < quads ? a.dk : a.dv, (int)(pair / a.Hkv), ra)) + d;
#pragma unroll
  for (int j = 0; j < 4; ++j) dst[j] = (T)acc[j];
}

// Joins the splits of dq as attn_join_kernel does the forward's; KEYS: also what delta was off by (attn_dq_kernel)
template <class T, bool WIDE>
__global__ __launch_bounds__(256) void attn_sum_kernel(Attn a, int64_t n_rows) {
  constexpr bool KEYS = Terms<T>::NP == 1;
  constexpr int N = KEYS ? 10 : 4;                     // four columns of sum ds k, of sum p k, sum ds, sum of the rounded
  const int quads = a.D / 4, width = KEYS ? 2 * a.D : a.D;
  int64_t rid;
  int quad, first = 0, every = 1;
  if constexpr (WIDE) {
    rid = blockIdx.x;
    quad = threadIdx.x & 31;
    first = threadIdx.x >> 5;
    every = 8;
  } else {
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (id >= n_rows * quads) return;
    rid = id / quads;
    quad = (int)(id - rid * quads);
  }
  const int d = quad * 4;
  float acc[N];
#pragma unroll
  for (int j = 0; j < N; ++j) acc[j] = 0.f;
  if (quad < quads)
#pragma unroll 4
    for (int i = first; i < a.splits; i += every) {
      const float* from = a.part + (i * n_rows + rid) * width + d;
      const float4 v = *reinterpret_cast<const float4*>(from);
      acc[0] += v.x;
      acc[1] += v.y;
      acc[2] += v.z;
      acc[3] += v.w;
      if constexpr (KEYS) {
        const float4 k = *reinterpret_cast<const float4*>(from + a.D);
        acc[4] += k.x;
        acc[5] += k.y;
        acc[6] += k.z;
        acc[7] += k.w;
        const float2 both = *reinterpret_cast<const float2*>(a.part_lse + 2 * (i * n_rows + rid));
        acc[8] += both.x;
        acc[9] += both.y;
      }
    }
  if constexpr (WIDE) {
    __shared__ float red[8][32][N];
#pragma unroll
    for (int j = 0; j < N; ++j) red[first][quad][j] = acc[j];
    __syncthreads();
    if (first || quad >= quads) return;
    for (int g = 1; g < 8; ++g)
#pragma unroll
      for (int j = 0; j < N; ++j) acc[j] += red[g][quad][j];
  }
  if (KEYS && d == 0) a.delta[rid] += acc[N - 2];
  T* dst = row_of<T>(a, a.dq, rid) + d;
#pragma unroll
  for (int j = 0; j < 4; ++j) dst[j] = (T)(a.scale * (KEYS ? acc[j] - acc[N - 1] * acc[KEYS ? 4 + j : 0] : acc[j]));
}

// ---- few query rows --------------------------------------------------------------------------------------------------
// One to four rows per (sample, key head): a candidate per user, a decoded token.  Nothing to tile, the keys and values
// are read once and that is the time: LPK lanes hold a key (16 bytes each), a wave 64 / LPK keys per step and ROW_STEP
// steps in flight; products on the vector units, in fp32 throughout (p and ds are not rounded).  Every group of LPK lanes
// keeps a running softmax of its own; they are joined at the end, over lanes, waves (LDS) and splits (a second launch).
// The backward needs no `out`: pass one reads k and v, keeps p and dp = dout v^T per key and sums
//   delta = sum p dp,  A = sum p dp k,  S = sum p k   (dq = scale (A - delta S)),
// pass two writes dk = scale p (dp - delta) q and dv = p dout from the kept numbers: k and v are read once, delta is
// the exact row sum.  While p and dp fit the LDS of one block the two passes are one launch.
// Measured: 8192 pairs of one row and up to 200 keys of 32, fp32: 38 us forward by itself (5.5 TB/s), 75 behind a backward,
// whose writes are still on their way to memory; 109 backward (5.8 TB/s).  128 pairs of one row and 32768 keys of 64, bf16,
// 1.07 GB of keys and values: 205 us forward by itself (5.2 TB/s), 263 behind a backward; 258 + 285 backward.
constexpr int ROW_STEP = 4;                            // 2: 3 % slower on those shapes; 8: within 3 % either way
constexpr int ROWS_LDS = 4096;                         // (key, row) pairs whose p and dp a block keeps in LDS: backward of the
                                                       // first shape 104 us in one launch, 132 in two

template <int LPK>
__device__ static inline float slot_sum(float v) {
#pragma unroll
  for (int o = LPK; o < 64; o <<= 1) v += __shfl_xor(v, o);
  return v;
}
template <int LPK>
__device__ static inline float slot_max(float v) {
#pragma unroll
  for (int o = LPK; o < 64; o <<= 1) v = fmaxf(v, __shfl_xor(v, o));
  return v;
}
template <class T>
__device__ static inline void packet_floats(const T* p, bool ok, float* f) {
  Packet<T>::unpack(ok ? *reinterpret_cast<const uint4*>(p) : make_uint4(0, 0, 0, 0), f);
}

// NW waves work on one pair.  A wave alone on its pair shares a block with the three next ones: they are the neighbouring
// heads of the same sample, whose rows lie side by side in memory, and are read at the same time.
struct PairAt { int split, b, hk, k0, k1; bool live; };
template <int NW>
__device__ static inline PairAt pair_at(const Attn& a) {
  PairAt p;
  int pair;
  if constexpr (NW == 1) {
    pair = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    p.split = 0;
  } else {
    const BlockAt ba = block_at(a, a.splits);
    pair = ba.pair;
    p.split = ba.part;
  }
  p.live = pair < a.B * a.Hkv;
  if (!p.live) pair = 0;
  p.b = pair / a.Hkv;
  p.hk = pair - p.b * a.Hkv;
  p.k0 = p.split * a.per_split;
  p.k1 = min(key_count(a, p.b), p.k0 + a.per_split);
  return p;
}
// LDS written by a wave's lanes before, read by its other lanes after
__device__ static inline void wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

template <class T, int R, int LPK, int NW>
__global__ __launch_bounds__(256) void attn_rows_fwd_kernel(Attn a) {
  constexpr int V = Packet<T>::V, KPW = 64 / LPK, U = ROW_STEP;
  __shared__ float sm[NW > 1 ? NW * R * (LPK * V + 2) : 1];
  const int lane = threadIdx.x & 63, wave = NW == 1 ? 0 : threadIdx.x >> 6, sub = lane % LPK, slot = lane / LPK, d = sub * V;
  const PairAt pa = pair_at<NW>(a);
  if (!pa.live) return;
  const bool in_d = d < a.D;
  const T* kp = (const T*)a.k.p + (int64_t)pa.b * a.k.b + (int64_t)pa.hk * a.k.h + d;
  const T* vp = (const T*)a.v.p + (int64_t)pa.b * a.v.b + (int64_t)pa.hk * a.v.h + d;
  const uint8_t* mask = a.mask ? a.mask + (int64_t)pa.b * a.mask_ld : nullptr;
  float q[R][V], o[R][V], m[R], l[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    packet_floats(row_ptr<T>(a.q, pa.b, row_at(a, r < a.rows ? r : 0, pa.hk)) + d, in_d && r < a.rows, q[r]);
    m[r] = minus_inf();
    l[r] = 0.f;
#pragma unroll
    for (int j = 0; j < V; ++j) { q[r][j] *= a.scale2; o[r][j] = 0.f; }
  }
  for (int base = pa.k0 + wave * KPW * U; base < pa.k1; base += NW * KPW * U) {
    uint4 kr[U], vr[U];
    bool ok[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int key = base + u * KPW + slot;
      ok[u] = key < pa.k1;
      const bool in = ok[u] && in_d;
      kr[u] = in ? *reinterpret_cast<const uint4*>(kp + (int64_t)key * a.k.t) : make_uint4(0, 0, 0, 0);
      vr[u] = in ? *reinterpret_cast<const uint4*>(vp + (int64_t)key * a.v.t) : make_uint4(0, 0, 0, 0);
      if (mask && ok[u]) ok[u] = mask[key] != 0;
    }
    float s[U][R];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float f[V];
      Packet<T>::unpack(kr[u], f);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        float t = 0.f;
#pragma unroll
        for (int j = 0; j < V; ++j) t = fmaf(q[r][j], f[j], t);
        s[u][r] = t;
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float t = group_sum<LPK>(s[u][r]);
        s[u][r] = ok[u] ? t : minus_inf();
      }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float top = m[r];
#pragma unroll
      for (int u = 0; u < U; ++u) top = fmaxf(top, s[u][r]);
      const float at = top == minus_inf() ? 0.f : top;
      const float fade = __builtin_amdgcn_exp2f(m[r] - at);
      m[r] = top;
      l[r] *= fade;
#pragma unroll
      for (int j = 0; j < V; ++j) o[r][j] *= fade;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        s[u][r] = __builtin_amdgcn_exp2f(s[u][r] - at);
        l[r] += s[u][r];
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float f[V];
      Packet<T>::unpack(ok[u] ? vr[u] : make_uint4(0, 0, 0, 0), f);
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int j = 0; j < V; ++j) o[r][j] = fmaf(s[u][r], f[j], o[r][j]);
    }
  }
  // join the lane groups, then the waves
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const float top = slot_max<LPK>(m[r]);
    const float fade = top == minus_inf() ? 0.f : __builtin_amdgcn_exp2f(m[r] - top);
    m[r] = top;
    l[r] = slot_sum<LPK>(l[r] * fade);
#pragma unroll
    for (int j = 0; j < V; ++j) o[r][j] = slot_sum<LPK>(o[r][j] * fade);
  }
  if constexpr (NW > 1) {
    constexpr int W = LPK * V + 2;
    if (slot == 0)
#pragma unroll
      for (int r = 0; r < R; ++r) {
        float* w = sm + (wave * R + r) * W;
#pragma unroll
        for (int j = 0; j < V; ++j) w[d + j] = o[r][j];
        if (sub == 0) { w[LPK * V] = m[r]; w[LPK * V + 1] = l[r]; }
      }
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float top = minus_inf();
      for (int w = 0; w < NW; ++w) top = fmaxf(top, sm[(w * R + r) * W + LPK * V]);
      const float at = top == minus_inf() ? 0.f : top;
      m[r] = top;
      l[r] = 0.f;
#pragma unroll
      for (int j = 0; j < V; ++j) o[r][j] = 0.f;
      for (int w = 0; w < NW; ++w) {
        const float* from = sm + (w * R + r) * W;
        const float fade = __builtin_amdgcn_exp2f(from[LPK * V] - at);
        l[r] = fmaf(from[LPK * V + 1], fade, l[r]);
#pragma unroll
        for (int j = 0; j < V; ++j) o[r][j] = fmaf(from[d + j], fade, o[r][j]);
      }
    }
  }
  if (slot) return;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    if (r >= a.rows) break;
    const RowAt ra = row_at(a, r, pa.hk);
    const int64_t rid = row_id(a, pa.b, ra);
    const float inv = l[r] == 0.f ? 0.f : 1.f / l[r];
    const float lse = l[r] == 0.f ? minus_inf() : m[r] * LN2 + logf(l[r]);
#pragma unroll
    for (int j = 0; j < V; ++j) o[r][j] *= inv;
    if (a.splits == 1) {
      if (in_d) *reinterpret_cast<uint4*>(const_cast<T*>(row_ptr<T>(a.out, pa.b, ra)) + d) = Packet<T>::pack(o[r]);
      if (a.lse && sub == 0) a.lse[rid] = lse;
    } else {
      const int64_t at = (int64_t)pa.split * ((int64_t)a.B * a.Hkv * a.rows) + rid;
      if (in_d)
#pragma unroll
        for (int j = 0; j < V; j += 4)
          *reinterpret_cast<float4*>(a.part + at * a.D + d + j) = make_float4(o[r][j], o[r][j + 1], o[r][j + 2], o[r][j + 3]);
      if (sub == 0) a.part_lse[at] = lse;
    }
  }
}

// dk and dv of the keys [k0, k1) of a pair, KPW keys per wave and step; kept: p and dp of key k, row r at
// kept[(k - from) * R + r] and `apart` floats behind.  A key that is left out carries p = -1: its zeros do not depend on
// what q and dout hold (0 * infinity).
template <class T, int R, int LPK>
__device__ static inline void rows_write_kv(const Attn& a, int b, int hk, int k0, int k1, int live, int from,
                                            const float* kept, int64_t apart, const float (&q)[R][Packet<T>::V],
                                            const float (&g)[R][Packet<T>::V], const float (&delta)[R], bool lone,
                                            int wave, int waves) {
  constexpr int V = Packet<T>::V, KPW = 64 / LPK;
  const int lane = threadIdx.x & 63, sub = lane % LPK, slot = lane / LPK, d = sub * V;
  T* kp = (T*)a.dk.p + (int64_t)b * a.dk.b + (int64_t)hk * a.dk.h + d;
  T* vp = (T*)a.dv.p + (int64_t)b * a.dv.b + (int64_t)hk * a.dv.h + d;
  for (int key = k0 + wave * KPW + slot; key < k1; key += waves * KPW) {
    float dk[V], dv[V];
#pragma unroll
    for (int j = 0; j < V; ++j) dk[j] = dv[j] = 0.f;
    if (key < live) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float p = kept[(int64_t)(key - from) * R + r], dp = kept[apart + (int64_t)(key - from) * R + r];
        if (p < 0.f) continue;
        const float ds = p == 0.f || lone ? 0.f : p * (dp - delta[r]) * a.scale;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          dk[j] = fmaf(ds, q[r][j], dk[j]);
          dv[j] = fmaf(p, g[r][j], dv[j]);
        }
      }
    }
    if (d < a.D) {
      *reinterpret_cast<uint4*>(kp + (int64_t)key * a.dk.t) = Packet<T>::pack(dk);
      *reinterpret_cast<uint4*>(vp + (int64_t)key * a.dv.t) = Packet<T>::pack(dv);
    }
  }
}

// FUSED: one block holds all keys of its pair in LDS; else p and dp go to a.kept and the sums to a.part
template <class T, int R, int LPK, int NW, bool FUSED>
__global__ __launch_bounds__(256) void attn_rows_bwd_kernel(Attn a) {
  constexpr int V = Packet<T>::V, KPW = 64 / LPK, U = ROW_STEP, W = 2 * LPK * V + 1;
  extern __shared__ float lds[];                       // joins [NW][R][W], then (FUSED) p, dp [per_split * R] each
  float* dyn = lds;
  if (NW == 1) dyn += (threadIdx.x >> 6) * a.per_split * R * 2;          // one per pair, nothing to join
  const int lane = threadIdx.x & 63, wave = NW == 1 ? 0 : threadIdx.x >> 6, sub = lane % LPK, slot = lane / LPK, d = sub * V;
  const PairAt pa = pair_at<NW>(a);
  if (!pa.live) return;
  const bool in_d = d < a.D;
  const T* kp = (const T*)a.k.p + (int64_t)pa.b * a.k.b + (int64_t)pa.hk * a.k.h + d;
  const T* vp = (const T*)a.v.p + (int64_t)pa.b * a.v.b + (int64_t)pa.hk * a.v.h + d;
  const uint8_t* mask = a.mask ? a.mask + (int64_t)pa.b * a.mask_ld : nullptr;
  float* kept;
  int64_t apart;
  if constexpr (FUSED) {
    kept = dyn + (NW == 1 ? 0 : NW * R * W);
    apart = (int64_t)a.per_split * R;
  } else {
    kept = a.kept + ((int64_t)(pa.b * a.Hkv + pa.hk) * a.Tk + pa.k0) * R;
    apart = (int64_t)a.B * a.Hkv * a.Tk * R;
  }
  float q[R][V], g[R][V], A[R][V], S[R][V], delta[R], shift[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const bool in = r < a.rows;
    const RowAt ra = row_at(a, in ? r : 0, pa.hk);
    packet_floats(row_ptr<T>(a.q, pa.b, ra) + d, in_d && in, q[r]);
    packet_floats(row_ptr<T>(a.dout, pa.b, ra) + d, in_d && in, g[r]);
    const float lse = in ? a.lse[row_id(a, pa.b, ra)] : minus_inf();
    shift[r] = lse == minus_inf() ? minus_inf() : -lse * LOG2E;
    delta[r] = 0.f;
#pragma unroll
    for (int j = 0; j < V; ++j) A[r][j] = S[r][j] = 0.f;
  }
  for (int base = pa.k0 + wave * KPW * U; base < pa.k1; base += NW * KPW * U) {
    uint4 kr[U], vr[U];
    bool ok[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int key = base + u * KPW + slot;
      ok[u] = key < pa.k1;
      const bool in = ok[u] && in_d;
      kr[u] = in ? *reinterpret_cast<const uint4*>(kp + (int64_t)key * a.k.t) : make_uint4(0, 0, 0, 0);
      vr[u] = in ? *reinterpret_cast<const uint4*>(vp + (int64_t)key * a.v.t) : make_uint4(0, 0, 0, 0);
      if (mask && ok[u]) ok[u] = mask[key] != 0;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int key = base + u * KPW + slot;
      float f[V], h[V];
      Packet<T>::unpack(ok[u] ? kr[u] : make_uint4(0, 0, 0, 0), f);
      Packet<T>::unpack(ok[u] ? vr[u] : make_uint4(0, 0, 0, 0), h);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        float s = 0.f, dp = 0.f;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          s = fmaf(q[r][j], f[j], s);
          dp = fmaf(g[r][j], h[j], dp);
        }
        s = group_sum<LPK>(s);
        dp = group_sum<LPK>(dp);
        const float p = ok[u] ? __builtin_amdgcn_exp2f(fmaf(s, a.scale2, shift[r])) : 0.f;
        const float pd = p == 0.f ? 0.f : p * dp;
        delta[r] += pd;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          A[r][j] = fmaf(pd, f[j], A[r][j]);
          S[r][j] = fmaf(p, f[j], S[r][j]);
        }
        if (sub == 0 && key < pa.k1) {
          kept[(int64_t)(key - pa.k0) * R + r] = ok[u] ? p : -1.f;
          kept[apart + (int64_t)(key - pa.k0) * R + r] = dp;
        }
      }
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    delta[r] = slot_sum<LPK>(delta[r]);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      A[r][j] = slot_sum<LPK>(A[r][j]);
      S[r][j] = slot_sum<LPK>(S[r][j]);
    }
  }
  if constexpr (NW > 1) {
    if (slot == 0)
#pragma unroll
      for (int r = 0; r < R; ++r) {
        float* w = dyn + (wave * R + r) * W;
#pragma unroll
        for (int j = 0; j < V; ++j) { w[d + j] = A[r][j]; w[LPK * V + d + j] = S[r][j]; }
        if (sub == 0) w[2 * LPK * V] = delta[r];
      }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < R; ++r) {
      delta[r] = 0.f;
      for (int w = 0; w < NW; ++w) delta[r] += dyn[(w * R + r) * W + 2 * LPK * V];
    }
    if (wave == 0)                                     // only this one writes dq
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          float x = 0.f, y = 0.f;
          for (int w = 0; w < NW; ++w) {
            x += dyn[(w * R + r) * W + d + j];
            y += dyn[(w * R + r) * W + LPK * V + d + j];
          }
          A[r][j] = x;
          S[r][j] = y;
        }
  } else if constexpr (FUSED) {
    wave_fence();                                      // p and dp of this wave's other lanes
  }
  const bool lone = FUSED && lone_key(a, pa.b);
  if (wave == 0 && slot == 0)
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (r >= a.rows) break;
      const RowAt ra = row_at(a, r, pa.hk);
      const int64_t rid = row_id(a, pa.b, ra);
      if constexpr (FUSED) {
        float dq[V];
#pragma unroll
        for (int j = 0; j < V; ++j) dq[j] = lone ? 0.f : a.scale * (A[r][j] - delta[r] * S[r][j]);
        if (in_d) *reinterpret_cast<uint4*>((T*)a.dq.p + (int64_t)pa.b * a.dq.b + (int64_t)ra.t * a.dq.t + (int64_t)ra.h * a.dq.h + d) = Packet<T>::pack(dq);
      } else {
        float* part = a.part + ((int64_t)pa.split * ((int64_t)a.B * a.Hkv * a.rows) + rid) * (2 * a.D + 1);
        if (in_d)
#pragma unroll
          for (int j = 0; j < V; ++j) { part[d + j] = A[r][j]; part[a.D + d + j] = S[r][j]; }
        if (sub == 0) part[2 * a.D] = delta[r];
      }
    }
  if constexpr (FUSED)
    rows_write_kv<T, R, LPK>(a, pa.b, pa.hk, 0, a.Tk, pa.k1, 0, kept, apart, q, g, delta, lone, wave, NW);
}

// Pass two over kept p and dp: block `chunk` of a pair writes its keys; chunk 0 also dq
template <class T, int R, int LPK>
__global__ __launch_bounds__(256) void attn_rows_kv_kernel(Attn a, int chunks, int per_chunk) {
  constexpr int V = Packet<T>::V;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, sub = lane % LPK, d = sub * V;
  const int chunk = blockIdx.x % chunks, pair = blockIdx.x / chunks, b = pair / a.Hkv, hk = pair - b * a.Hkv;
  const bool in_d = d < a.D;
  const bool lone = lone_key(a, b);
  float q[R][V], g[R][V], delta[R];
  const int64_t n_rows = (int64_t)a.B * a.Hkv * a.rows;
  const int width = 2 * a.D + 1;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const bool in = r < a.rows;
    const RowAt ra = row_at(a, in ? r : 0, hk);
    packet_floats(row_ptr<T>(a.q, b, ra) + d, in_d && in, q[r]);
    packet_floats(row_ptr<T>(a.dout, b, ra) + d, in_d && in, g[r]);
    delta[r] = 0.f;
    if (in) {
      const int64_t rid = row_id(a, b, ra);
      for (int i = lane; i < a.splits; i += 64) delta[r] += a.part[(i * n_rows + rid) * width + 2 * a.D];
    }
    delta[r] = wave_sum(delta[r]);
  }
  if (chunk == 0) {                                    // a thread per element of dq
    __shared__ float delta_s[R];
    if (threadIdx.x == 0)
#pragma unroll
      for (int r = 0; r < R; ++r) delta_s[r] = delta[r];
    __syncthreads();
    for (int i = threadIdx.x; i < a.rows * a.D; i += 256) {
      const int r = i / a.D, at = i - r * a.D;
      const RowAt ra = row_at(a, r, hk);
      const float* part = a.part + row_id(a, b, ra) * width + at;
      float A = 0.f, S = 0.f;
#pragma unroll 4
      for (int k = 0; k < a.splits; ++k) {
        A += part[k * n_rows * width];
        S += part[k * n_rows * width + a.D];
      }
      const_cast<T*>(row_ptr<T>(a.dq, b, ra))[at] = (T)(lone ? 0.f : a.scale * (A - delta_s[r] * S));
    }
  }
  const int k0 = chunk * per_chunk, k1 = min(a.Tk, k0 + per_chunk);
  rows_write_kv<T, R, LPK>(a, b, hk, k0, k1, key_count(a, b), 0, a.kept + (int64_t)pair * a.Tk * R,
                           (int64_t)a.B * a.Hkv * a.Tk * R, q, g, delta, lone, wave, 4);
}

// ---- host ----------------------------------------------------------------------------------------------------------
// keys that a wave of the few-row kernels holds at once
static int rows_lanes(int D, int dtype) {
  const int packets = D / (16 / type_bytes(dtype));
  return packets <= 2 ? 2 : packets <= 4 ? 4 : packets <= 8 ? 8 : packets <= 16 ? 16 : 32;
}
static int rows_step_keys(int D, int dtype) { return 64 / rows_lanes(D, dtype); }
static int padded_dim(int D) { return D <= 32 ? 32 : D <= 64 ? 64 : D <= 96 ? 96 : 128; }
// Waves of a block: as many as there are strips of 32 rows (or keys), one, two or four.  Where even walks of 64 along the
// other axis would not give every CU eight blocks, four in any case: the idle ones help to stage the tiles (6 rows of 22
// keys, fp32, D 104, the three passes: 39 us for 60; 16 rows against 32768 keys, in walks enough: 48 us alone, 58 by four).
// fp32 above 96: four, since one wave's tiles alone fill a third of the LDS (2048 pairs of 20 rows and 200 keys of 128,
// forward 225 us, dq 309; 284 and 466 by single waves; at 96 single waves still win, 43 and 60 us for 53 and 73).
static int strip_waves(int n, int64_t pairs, int other, int dtype, int D) {
  if (dtype == CTR_F32 && D > 96) return 4;
  if (pairs * cdiv(other, 64) < 2048) return 4;
  return n <= 32 ? 1 : n <= 64 ? 2 : 4;
}

// Splits of the key axis: only where the row tiles alone leave part of the chip without waves (every split writes its
// share of the result as fp32, which is read again), and never below 64 keys each.  One block of four waves per CU is
// enough for tiles that are computed; single waves want four per CU (16 rows against 32768 keys of 128: 48 us with 1024,
// 56 with 2048, 70 with 512).
static int key_splits(int64_t blocks, int waves, int Tk) {
  const int64_t want = (waves == 1 ? 1024 : 512) / (blocks < 1 ? 1 : blocks), most = Tk / 64;
  const int64_t n = want < most ? want : most;
  return (int)(n < 1 ? 1 : n);
}
// Splits of the row list for dk / dv, on the same grounds: at least 64 rows each.  fp32: at most 1024, since one
// accumulator that takes every row of a long list rounds after each 16 of them (4592 rows: 1.1e-6 off, in five splits
// 0.5e-6) - as far as the splits stay small beside the rows themselves.
static int list_splits(int64_t blocks, int rows, int keys, int dtype) {
  const int64_t want = 512 / (blocks < 1 ? 1 : blocks), most = rows / 64;
  int64_t n = want < most ? want : most;
  if (dtype == CTR_F32) {
    const int64_t fine = cdiv(rows, 1024), small = rows / (4 * (int64_t)(keys < 1 ? 1 : keys));
    n = n > fine ? n : fine < small ? fine : n > small ? n : small;
  }
  return (int)(n < 1 ? 1 : n);
}

// Few rows: waves for about eight per SIMD (four or sixteen: within 3 %), each with at least ROW_STEP steps of keys; four to
// a block, more as splits.  A wave alone where there are pairs enough: nothing to join (32768 pairs of 50 keys, fp32: 78 and
// 141 us, 85 and 148 by four; of four rows 100 and 176, 183 and 378).
static void rows_plan(Attn* a, int dtype) {
  a->lanes = rows_lanes(a->D, dtype);
  a->few = a->rows <= 1 ? 1 : a->rows <= 2 ? 2 : 4;
  const int64_t pairs = (int64_t)a->B * a->Hkv, step = rows_step_keys(a->D, dtype) * ROW_STEP;
  const int64_t most = cdiv(a->Tk < 1 ? 1 : a->Tk, step), want = pairs < 1 ? 1 : 8192 / pairs;
  const int64_t waves = want < 1 ? 1 : want < most ? want : most;
  a->waves = waves >= 4 ? 4 : 1;
  int64_t splits = waves / 8;                          // below eight waves one block holds the pair
  a->splits = (int)(splits < 1 ? 1 : splits > 128 ? 128 : splits);
  a->per_split = (int)align_up(cdiv(a->Tk, a->splits), step);
  a->splits = a->Tk > 0 ? (int)cdiv(a->Tk, a->per_split) : 1;
}

static void attn_plan(Attn* a, int dtype) {
  a->rows = a->Tq * a->G;
  // Up to four rows the vector units keep up with memory.  Eight were tried in the backward and lost (8 rows against 8757
  // keys of 128: 430 us for the two passes, 280 for the tiles').
  if (a->rows >= 1 && a->rows <= 4) {
    rows_plan(a, dtype);
    return;
  }
  a->few = 0;
  a->row_waves = strip_waves(a->rows, (int64_t)a->B * a->Hkv, a->Tk, dtype, a->D);
  a->row_tiles = (int)cdiv(a->rows, 32 * a->row_waves);
  a->splits = key_splits((int64_t)a->row_tiles * a->B * a->Hkv, a->row_waves, a->Tk);
  a->per_split = (int)align_up(cdiv(a->Tk, a->splits), 64);
  a->splits = a->Tk > 0 ? (int)cdiv(a->Tk, a->per_split) : 1;
  a->key_waves = strip_waves(a->Tk, (int64_t)a->B * a->Hkv, a->rows, dtype, a->D);
  a->key_tiles = (int)cdiv(a->Tk, 32 * a->key_waves);
  a->row_splits = list_splits((int64_t)a->key_tiles * a->B * a->Hkv, a->rows, a->Tk, dtype);
  a->rows_per = (int)align_up(cdiv(a->rows, a->row_splits), 64);
  a->row_splits = a->rows > 0 ? (int)cdiv(a->rows, a->rows_per) : 1;
}
static int64_t total_rows(const Attn& a) { return (int64_t)a.B * a.Hkv * a.rows; }
static bool rows_fused(const Attn& a) {
  return a.splits == 1 && (int64_t)a.per_split * a.few <= (a.waves == 1 ? ROWS_LDS / 4 : ROWS_LDS);
}
static size_t fwd_ws(const Attn& a) { return a.splits > 1 ? (size_t)a.splits * total_rows(a) * (a.D + 1) * 4 + 256 : 0; }
// tiled: delta, then the splits' dq; few rows: the splits' sums, then p and dp of every key
static size_t bwd_ws_first(const Attn& a) {
  if (a.few) return rows_fused(a) ? 0 : align_up((size_t)a.splits * total_rows(a) * (2 * a.D + 1) * 4, 256);
  return align_up((size_t)total_rows(a) * 4, 256);
}
static size_t bwd_ws(const Attn& a) {
  if (a.few) return rows_fused(a) ? 256 : bwd_ws_first(a) + (size_t)a.B * a.Hkv * a.Tk * a.few * 8 + 256;
  const size_t rows = a.splits > 1 ? (size_t)a.splits * total_rows(a) * (2 * a.D + 2) * 4 : 0;
  const size_t keys = a.row_splits > 1 ? (size_t)a.row_splits * a.B * a.Hkv * a.Tk * 2 * a.D * 4 : 0;
  return bwd_ws_first(a) + (rows > keys ? rows : keys) + 256;           // one after the other
}

// Blocks of attn_rows_kv_kernel per pair, and keys for each
static int kv_chunk_keys(const Attn& a) {
  const int64_t want = cdiv(2048, (int64_t)a.B * a.Hkv), most = cdiv(a.Tk, 64);
  return (int)cdiv(a.Tk, want < most ? want : most);
}
static int kv_chunks(const Attn& a) { return (int)cdiv(a.Tk, kv_chunk_keys(a)); }

// Whether every launch of a call has fewer than 2^32 threads: the hardware counts them in 32 bits
static bool launches_fit(const Attn& a, bool backward) {
  auto fits = [](int64_t blocks, int threads) { return blocks < (1ll << 32) / threads; };
  const int64_t pairs = (int64_t)a.B * a.Hkv;
  if (a.few) {
    const bool alone = a.waves == 1 && (!backward || rows_fused(a));
    if (!fits(alone ? cdiv(pairs, 4) : pair_blocks(a, a.splits), 256)) return false;
    return !backward || rows_fused(a) || pairs == 0 || fits(pairs * kv_chunks(a), 256);
  }
  if (!fits(pair_blocks(a, (int64_t)a.row_tiles * a.splits), 64 * a.row_waves)) return false;
  if (a.splits > 1 && !fits(a.splits >= JOIN_WIDE ? total_rows(a) : cdiv(total_rows(a) * (a.D / 4), 256), 256)) return false;
  if (!backward) return true;
  return fits(pair_blocks(a, (int64_t)a.key_tiles * a.row_splits), 64 * a.key_waves) &&
         (a.row_splits == 1 || fits(cdiv(pairs * a.Tk * (a.D / 2), 256), 256));
}

static int attn_shape(const char* what, const ctr_attn_t* s, bool backward, Attn* a) {
  CTR_REQUIRE(s, "%s: no shape", what);
  CTR_REQUIRE(type_bytes(s->dtype) != 0, "%s: unknown dtype %d", what, s->dtype);
  CTR_REQUIRE(s->B >= 0 && s->Tq >= 0 && s->Tk >= 0 && s->H >= 1 && s->Hkv >= 1 && s->H % s->Hkv == 0,
              "%s: B %d Tq %d Tk %d H %d Hkv %d (Hkv must divide H)", what, s->B, s->Tq, s->Tk, s->H, s->Hkv);
  CTR_REQUIRE(s->D >= 8 && s->D <= 128 && s->D % 8 == 0, "%s: head size %d is not a multiple of 8 up to 128", what, s->D);
  CTR_REQUIRE(s->scale >= 1e-30f && s->scale <= 1e30f, "%s: scale must lie between 1e-30 and 1e30", what);
  CTR_REQUIRE((int64_t)s->Tq * (s->H / s->Hkv) < (1 << 30) && s->Tk < (1 << 30) && (int64_t)s->B * s->H < (1 << 30),
              "%s: more than 2^30 rows, keys or heads", what);
  CTR_REQUIRE(!s->mask || s->mask_ld >= 0, "%s: the mask has a negative stride", what);
  *a = Attn{};
  a->B = s->B; a->Tq = s->Tq; a->Tk = s->Tk; a->Hkv = s->Hkv; a->G = s->H / s->Hkv; a->D = s->D;
  a->scale = s->scale;
  a->scale2 = s->scale * LOG2E;
  a->sl = s->sl; a->mask = s->mask; a->mask_ld = s->mask_ld;
  attn_plan(a, s->dtype);
  CTR_REQUIRE(launches_fit(*a, backward), "%s: a launch of 2^32 threads or more", what);
  return CTR_OK;
}

// strides of a [B, T, heads, D] view: 16-byte rows; an output may not name an element twice
static int attn_view(const char* what, const char* name, const ctr_heads_t* v, int B, int T, int heads, int D, int dtype,
                     bool output, View4* w) {
  CTR_REQUIRE(v, "%s: %s is missing", what, name);
  *w = View4{v->p, v->stride_b, v->stride_t, v->stride_h};
  if ((int64_t)B * T * heads == 0) return CTR_OK;
  const int per = 16 / type_bytes(dtype);
  CTR_REQUIRE(v->p, "%s: %s is NULL", what, name);
  CTR_REQUIRE(((uintptr_t)v->p & 15) == 0 && v->stride_b % per == 0 && v->stride_t % per == 0 && v->stride_h % per == 0,
              "%s: %s and its rows must lie on 16-byte boundaries", what, name);
  CTR_REQUIRE(v->stride_b >= 0 && v->stride_t >= 0 && v->stride_h >= 0, "%s: %s has a negative stride", what, name);
  if (output) {
    int64_t st[3] = {v->stride_b, v->stride_t, v->stride_h}, n[3] = {B, T, heads}, span = D;
    for (int i = 0; i < 3; ++i)
      for (int j = i + 1; j < 3; ++j)
        if (st[j] < st[i]) { const int64_t x = st[i], y = n[i]; st[i] = st[j]; n[i] = n[j]; st[j] = x; n[j] = y; }
    for (int i = 0; i < 3; ++i) {
      if (n[i] == 1) continue;
      CTR_REQUIRE(st[i] >= span, "%s: %s holds an element twice", what, name);
      span = st[i] * (n[i] - 1) + span;
    }
  }
  return CTR_OK;
}

// Whether strip_waves gives blocks of one or two waves
template <class T, int DP>
constexpr bool SMALL_BLOCKS = sizeof(T) == 2 || DP <= 96;

#define ATTN_DIM(T, D, CALL)                    \
  do {                                          \
    switch (padded_dim(D)) {                    \
      case 32: { CALL(T, 32); } break;          \
      case 64: { CALL(T, 64); } break;          \
      case 96: { CALL(T, 96); } break;          \
      default: { CALL(T, 128); } break;         \
    }                                           \
  } while (0)

// LPK is at most 16 for 16-bit types
#define ROWS_LANES(T, LPK, CALL)                                                     \
  do {                                                                               \
    switch (LPK) {                                                                   \
      case 2: { CALL(T, 2); } break;                                                 \
      case 4: { CALL(T, 4); } break;                                                 \
      case 8: { CALL(T, 8); } break;                                                 \
      case 16: { CALL(T, 16); } break;                                               \
      default: if constexpr (sizeof(T) == 4) { CALL(T, 32); } break;                 \
    }                                                                                \
  } while (0)

template <class T, int R>
static void rows_fwd_launch(const Attn& a, hipStream_t st) {
  const unsigned blocks = a.waves == 1 ? (unsigned)cdiv((int64_t)a.B * a.Hkv, 4) : pair_blocks(a, a.splits);
#define ROWS_FWD(T_, LPK_)                                                           \
  if (a.waves == 1) attn_rows_fwd_kernel<T_, R, LPK_, 1><<<blocks, 256, 0, st>>>(a); \
  else attn_rows_fwd_kernel<T_, R, LPK_, 4><<<blocks, 256, 0, st>>>(a)
  ROWS_LANES(T, a.lanes, ROWS_FWD);
#undef ROWS_FWD
}

template <class T, int R>
static void rows_bwd_launch(const Attn& a, hipStream_t st) {
  const bool fused = rows_fused(a), alone = a.waves == 1 && fused;
  const unsigned blocks = alone ? (unsigned)cdiv((int64_t)a.B * a.Hkv, 4) : pair_blocks(a, a.splits);
  const size_t joins = (size_t)4 * R * (2 * a.lanes * Packet<T>::V + 1) * 4, keep = (size_t)a.per_split * R * 8;
  if (fused) {
    const size_t lds = alone ? 4 * keep : joins + keep;
#define ROWS_BWD(T_, LPK_)                                                                        \
  if (alone) attn_rows_bwd_kernel<T_, R, LPK_, 1, true><<<blocks, 256, lds, st>>>(a);      \
  else attn_rows_bwd_kernel<T_, R, LPK_, 4, true><<<blocks, 256, lds, st>>>(a)
    ROWS_LANES(T, a.lanes, ROWS_BWD);
#undef ROWS_BWD
    return;
  }
  const int64_t pairs = (int64_t)a.B * a.Hkv;
  const int per = kv_chunk_keys(a), chunks = kv_chunks(a);
#define ROWS_BWD(T_, LPK_)                                                                        \
  attn_rows_bwd_kernel<T_, R, LPK_, 4, false><<<blocks, 256, joins, st>>>(a);                     \
  attn_rows_kv_kernel<T_, R, LPK_><<<(unsigned)(pairs * chunks), 256, 0, st>>>(a, chunks, per)
  ROWS_LANES(T, a.lanes, ROWS_BWD);
#undef ROWS_BWD
}

static bool tile_is_near(const View4& w, int64_t rows, int bytes) {
  return rows * (w.t + w.h) * bytes < ((int64_t)1 << 31);
}

template <class T>
static void join_launch(const Attn& a, hipStream_t st) {
  if (a.splits == 1) return;
  const int64_t n = total_rows(a);
  if (a.splits >= JOIN_WIDE) attn_join_kernel<T, true><<<(unsigned)n, 256, 0, st>>>(a, n);
  else attn_join_kernel<T, false><<<(unsigned)cdiv(n * (a.D / 4), 256), 256, 0, st>>>(a, n);
}

template <class T>
static void attn_fwd_launch(const Attn& a, hipStream_t st) {
  if (a.few) {
    if (a.few == 1) rows_fwd_launch<T, 1>(a, st);
    else if (a.few == 2) rows_fwd_launch<T, 2>(a, st);
    else rows_fwd_launch<T, 4>(a, st);
    join_launch<T>(a, st);
    return;
  }
  const unsigned blocks = pair_blocks(a, (int64_t)a.row_tiles * a.splits);
#define ATTN_FWD(T_, DP_)                                                                                        \
  constexpr int KT = sizeof(T_) == 4 || DP_ > 64 ? 32 : 64;                                                      \
  if (a.row_waves == 4) attn_fwd_kernel<T_, DP_, 4, KT><<<blocks, 256, 0, st>>>(a);                              \
  else if constexpr (SMALL_BLOCKS<T_, DP_>) {                                                                    \
    if (a.row_waves == 1) attn_fwd_kernel<T_, DP_, 1, 32><<<blocks, 64, 0, st>>>(a);                             \
    else attn_fwd_kernel<T_, DP_, 2, KT><<<blocks, 128, 0, st>>>(a);                                             \
  }
  ATTN_DIM(T, a.D, ATTN_FWD);
#undef ATTN_FWD
  join_launch<T>(a, st);
}

template <class T>
static void attn_bwd_launch(const Attn& a, hipStream_t st) {
  if (a.few) {
    if (a.few == 1) rows_bwd_launch<T, 1>(a, st);
    else if (a.few == 2) rows_bwd_launch<T, 2>(a, st);
    else rows_bwd_launch<T, 4>(a, st);
    return;
  }
  const unsigned blocks = pair_blocks(a, (int64_t)a.row_tiles * a.splits);
  if (blocks) {
#define ATTN_DQ(T_, DP_)                                                                                         \
  constexpr int KT = sizeof(T_) == 4 || DP_ > 64 ? 32 : 64;                                                      \
  if (a.row_waves == 4) attn_dq_kernel<T_, DP_, 4, KT><<<blocks, 256, 0, st>>>(a);                               \
  else if constexpr (SMALL_BLOCKS<T_, DP_>) {                                                                    \
    if (a.row_waves == 1) attn_dq_kernel<T_, DP_, 1, 32><<<blocks, 64, 0, st>>>(a);                              \
    else attn_dq_kernel<T_, DP_, 2, KT><<<blocks, 128, 0, st>>>(a);                                              \
  }
    ATTN_DIM(T, a.D, ATTN_DQ);
#undef ATTN_DQ
    if (a.splits > 1) {
      const int64_t n = total_rows(a);
      if (a.splits >= JOIN_WIDE) attn_sum_kernel<T, true><<<(unsigned)n, 256, 0, st>>>(a, n);
      else attn_sum_kernel<T, false><<<(unsigned)cdiv(n * (a.D / 4), 256), 256, 0, st>>>(a, n);
    }
  }
  const unsigned kblocks = pair_blocks(a, (int64_t)a.key_tiles * a.row_splits);
  if (kblocks) {
#define ATTN_DKV(T_, DP_)                                                                                        \
  constexpr int QB = sizeof(T_) == 2 && DP_ <= 32 ? 64 : 32, QB4 = DP_ <= 32 ? 64 : 32;                          \
  if (a.key_waves == 4) attn_dkv_kernel<T_, DP_, 4, QB4><<<kblocks, 256, 0, st>>>(a);                            \
  else if constexpr (SMALL_BLOCKS<T_, DP_>) {                                                                    \
    if (a.key_waves == 1) attn_dkv_kernel<T_, DP_, 1, 32><<<kblocks, 64, 0, st>>>(a);                            \
    else attn_dkv_kernel<T_, DP_, 2, QB><<<kblocks, 128, 0, st>>>(a);                                            \
  }
    ATTN_DIM(T, a.D, ATTN_DKV);
#undef ATTN_DKV
    if (a.row_splits > 1)
      attn_key_sum_kernel<T><<<(unsigned)cdiv((int64_t)a.B * a.Hkv * a.Tk * (a.D / 2), 256), 256, 0, st>>>(a);
  }
}

}  // namespace ctr

using namespace ctr;

extern "C" size_t ctr_cross_attn_fwd_workspace_bytes(const ctr_attn_t* shape) {
  Attn a;
  return attn_shape("cross_attn_fwd", shape, false, &a) ? 0 : fwd_ws(a);
}
extern "C" size_t ctr_cross_attn_bwd_workspace_bytes(const ctr_attn_t* shape) {
  Attn a;
  return attn_shape("cross_attn_bwd", shape, true, &a) ? 0 : bwd_ws(a);
}

extern "C" int ctr_cross_attn_fwd(const ctr_attn_t* s, const ctr_heads_t* q, const ctr_heads_t* k, const ctr_heads_t* v,
                                  const ctr_heads_t* out, float* lse_out, void* workspace, size_t workspace_bytes,
                                  void* stream) {
  const char* what = "cross_attn_fwd";
  Attn a;
  int rc = attn_shape(what, s, false, &a);
  if (rc) return rc;
  if ((rc = attn_view(what, "q", q, s->B, s->Tq, s->H, s->D, s->dtype, false, &a.q))) return rc;
  if ((rc = attn_view(what, "k", k, s->B, s->Tk, s->Hkv, s->D, s->dtype, false, &a.k))) return rc;
  if ((rc = attn_view(what, "v", v, s->B, s->Tk, s->Hkv, s->D, s->dtype, false, &a.v))) return rc;
  if ((rc = attn_view(what, "out", out, s->B, s->Tq, s->H, s->D, s->dtype, true, &a.out))) return rc;
  a.lse = lse_out;
  if (total_rows(a) == 0) return CTR_OK;
  if (workspace_bytes < fwd_ws(a) || (!workspace && fwd_ws(a))) {
    set_error("%s: workspace %zu < %zu", what, workspace_bytes, fwd_ws(a));
    return CTR_EWORKSPACE;
  }
  a.near = tile_is_near(a.k, 128, type_bytes(s->dtype)) && tile_is_near(a.v, 128, type_bytes(s->dtype));
  if (a.splits > 1) {
    a.part = (float*)align_up((size_t)workspace, 256);
    a.part_lse = a.part + (size_t)a.splits * total_rows(a) * a.D;
  }
  hipStream_t st = (hipStream_t)stream;
  if (s->dtype == CTR_F32) attn_fwd_launch<float>(a, st);
  else if (s->dtype == CTR_BF16) attn_fwd_launch<bf16_t>(a, st);
  else attn_fwd_launch<f16_t>(a, st);
  CTR_LAUNCH_CHECK();
  return CTR_OK;
}

extern "C" int ctr_cross_attn_bwd(const ctr_attn_t* s, const ctr_heads_t* dout, const ctr_heads_t* q,
                                  const ctr_heads_t* k, const ctr_heads_t* v, const ctr_heads_t* out, const float* lse,
                                  const ctr_heads_t* dq, const ctr_heads_t* dk, const ctr_heads_t* dv, void* workspace,
                                  size_t workspace_bytes, void* stream) {
  const char* what = "cross_attn_bwd";
  Attn a;
  int rc = attn_shape(what, s, true, &a);
  if (rc) return rc;
  if ((rc = attn_view(what, "dout", dout, s->B, s->Tq, s->H, s->D, s->dtype, false, &a.dout))) return rc;
  if ((rc = attn_view(what, "q", q, s->B, s->Tq, s->H, s->D, s->dtype, false, &a.q))) return rc;
  if ((rc = attn_view(what, "k", k, s->B, s->Tk, s->Hkv, s->D, s->dtype, false, &a.k))) return rc;
  if ((rc = attn_view(what, "v", v, s->B, s->Tk, s->Hkv, s->D, s->dtype, false, &a.v))) return rc;
  if ((rc = attn_view(what, "out", out, s->B, s->Tq, s->H, s->D, s->dtype, false, &a.out))) return rc;
  if ((rc = attn_view(what, "dq", dq, s->B, s->Tq, s->H, s->D, s->dtype, true, &a.dq))) return rc;
  if ((rc = attn_view(what, "dk", dk, s->B, s->Tk, s->Hkv, s->D, s->dtype, true, &a.dk))) return rc;
  if ((rc = attn_view(what, "dv", dv, s->B, s->Tk, s->Hkv, s->D, s->dtype, true, &a.dv))) return rc;
  CTR_REQUIRE(lse || total_rows(a) == 0, "%s: lse is NULL", what);
  if (s->B == 0) return CTR_OK;
  if (!workspace || workspace_bytes < bwd_ws(a)) {
    set_error("%s: workspace %zu < %zu", what, workspace_bytes, bwd_ws(a));
    return CTR_EWORKSPACE;
  }
  a.lse = const_cast<float*>(lse);
  a.near = true;
  for (const View4* w : {&a.k, &a.v, &a.q, &a.dout}) a.near = a.near && tile_is_near(*w, 128, type_bytes(s->dtype));
  float* ws = (float*)align_up((size_t)workspace, 256);
  if (a.few) {
    a.part = ws;
    a.kept = ws + bwd_ws_first(a) / 4;
  } else {
    a.delta = ws;
    a.part = ws + bwd_ws_first(a) / 4;
    a.part_lse = a.part + (size_t)a.splits * total_rows(a) * 2 * a.D;
  }
  hipStream_t st = (hipStream_t)stream;
  if (s->dtype == CTR_F32) attn_bwd_launch<float>(a, st);
  else if (s->dtype == CTR_BF16) attn_bwd_launch<bf16_t>(a, st);
  else attn_bwd_launch<f16_t>(a, st);
  CTR_LAUNCH_CHECK();
  return CTR_OK;
}
