// Layer norm over the last axis of a [rows, cols] view, forward and backward.
//   mean = sum x / n,  var = sum (x - mean)^2 / n,  rstd = 1 / sqrt(var + eps),  xh = (x - mean) rstd
// The mean's own rounding would be a common offset of its row, large beside a spread that is small against the mean, so
// the second pass sums the residuals d = x - mean too: c = sum d / n is what the mean is off by, and is taken out of
// it, of d and of the variance (sum d^2 / n - c^2).
//   y = xh gamma + beta
//   g = dy gamma;  dx = rstd (g - sum g / n - xh sum(g xh) / n);  dgamma = sum_rows dy xh;  dbeta = sum_rows dy
// Memory bound: the forward reads x and writes y once, the backward reads x and dy and writes dx once.  A row lives in
// the registers of LPR lanes (16 elements per lane at most), so the two-pass variance costs no second read, and the
// backward accumulates dgamma / dbeta of its lane's columns over all rows of its block before it writes one partial row
// per block; a second launch adds those in block order.  Sums are fp32, in a fixed order: results are the same bits on
// every run.  Rows above 16384 columns are walked in several passes instead.
// Measured (32 Mi elements, forward and backward in turn on the same inputs, averages of a kernel trace; a large copy
// reaches 4.9 TB/s).  bf16, 64 to 4096 columns: forward 22 - 23 us, 5.8 - 6.0 TB/s; backward 32 - 35 us, 5.7 - 6.3 TB/s, and
// 4.7 us for the partial rows.  24 columns: 29 and 55 (three of four lanes of a row at work, and a row's arithmetic on so
// few elements).  8192 columns: 24 and 49 + 7.5, 16384: 27 and 56 + 13 (one row to a block, two barriers in sight each).
// fp32, 64 to 8192 columns: 43 - 48 and 76 - 80; 16384: 50 and 91 + 13; 128 columns, 50 Mi elements: 74 and 124 us, 5.7 and
// 5.1 TB/s.  Walked rows are five times as far from memory's time: 1600 x 20000, bf16: forward 134, backward 161 + 27 + 7.
#include "types.h"

// Fused multiply-adds where the code says so and nowhere else: left to itself the compiler fuses a row's mean (sum / n)
// or gamma into the arithmetic of some of its entries and not of others, and equal entries of a row get different results.
#pragma clang fp contract(off)

namespace ctr {

constexpr int LN_LANE_ELEMS = 16;
constexpr int LN_MAX_COLS = 1024 * LN_LANE_ELEMS;     // a block of 1024 lanes holds the row
constexpr int LN_STRIP = 64;                          // rows per block of the column sums of wider rows

// Sum of v over the LPR lanes of a row; LPR > 64: over the row's waves through LDS, one barrier.  red holds one float per
// wave; the next sum of the block must use another array (it may come back to this one after that).
template <int LPR>
__device__ static inline float row_sum(float v, float* red) {
  if constexpr (LPR <= 64) {
    return group_sum<LPR>(v);
  } else {
    constexpr int W = LPR / 64;
    v = wave_sum(v);
    const int wave = threadIdx.x >> 6, first = wave / W * W;
    if ((threadIdx.x & 63) == 0) red[wave] = v;
    __syncthreads();
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < W; ++i) s += red[first + i];
    return s;
  }
}
// two sums behind one barrier; red: one array for each
template <int LPR>
__device__ static inline float2 row_sum2(float v, float w, float (*red)[16]) {
  if constexpr (LPR <= 64) {
    return make_float2(group_sum<LPR>(v), group_sum<LPR>(w));
  } else {
    constexpr int W = LPR / 64;
    v = wave_sum(v);
    w = wave_sum(w);
    const int wave = threadIdx.x >> 6, first = wave / W * W;
    if ((threadIdx.x & 63) == 0) {
      red[0][wave] = v;
      red[1][wave] = w;
    }
    __syncthreads();
    float2 s = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < W; ++i) {
      s.x += red[0][first + i];
      s.y += red[1][first + i];
    }
    return s;
  }
}
// What the residuals d of a row around `mean` say: the mean corrected, and rstd and shift with xh = d rstd + shift
struct RowStat { float mean, rstd, shift; };
__device__ static inline RowStat row_stat(float mean, float sum_d, float sum_d2, float inv_n, float eps) {
  const float c = sum_d * inv_n;
  const float var = fmaf(sum_d2, inv_n, -c * c);       // below zero by its rounding at most; NaN stays NaN
  const float rstd = 1.f / sqrtf((var < 0.f ? 0.f : var) + eps);
  return {mean + c, rstd, -c * rstd};
}
// a packet on its way: whole ones as they lie, the one at the end of a row element by element
template <class T>
__device__ static inline uint4 fetch_packet(const T* p, int have) {
  if (have == Packet<T>::V) return packet_load(p);
  float f[Packet<T>::V];
  load_part(p, have, 0.f, f);
  return Packet<T>::pack(f);
}

// V entries of a parameter vector from column c on, n of them inside the row (16 bytes at a time where all are)
template <int V>
__device__ static inline void load_param(const float* __restrict__ w, int c, int n, float fill, float* f) {
  if (w && n == V) {
#pragma unroll
    for (int j = 0; j < V; j += 4) {
      float4 v;
      __builtin_memcpy(&v, w + c + j, 16);
      f[j] = v.x; f[j + 1] = v.y; f[j + 2] = v.z; f[j + 3] = v.w;
    }
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) f[j] = w && j < n ? w[c + j] : fill;
  }
}

// Row in registers: lane `l` of LPR holds the packets l, l + LPR, ... (NV of them).
template <class T, int LPR, int NV, int THREADS>
__global__ __launch_bounds__(THREADS) void ln_fwd_kernel(const T* x, int64_t x_ld, int64_t rows, int cols,
                                                         const float* __restrict__ gamma,
                                                         const float* __restrict__ beta, float eps, T* y, int64_t y_ld,
                                                         float* __restrict__ mean_out, float* __restrict__ rstd_out) {
  constexpr int V = Packet<T>::V, GPB = THREADS / LPR;
  __shared__ float red[3][16];
  const int l = threadIdx.x % LPR, group = threadIdx.x / LPR;
  const float inv_n = 1.f / (float)cols;
  float ga[NV][V], be[NV][V];
  int have[NV];                                        // elements of packet i inside the row
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (l + i * LPR) * V;
    have[i] = min(max(cols - c, 0), V);
    load_param<V>(gamma, c, have[i], 1.f, ga[i]);
    load_param<V>(beta, c, have[i], 0.f, be[i]);
  }
  const int64_t step = (int64_t)gridDim.x * GPB;
  uint4 next[NV];                                      // the next row travels while this one is reduced
  auto fetch = [&](int64_t row) {
    const T* xr = x + min(row, rows - 1) * x_ld;
#pragma unroll
    for (int i = 0; i < NV; ++i) next[i] = fetch_packet(xr + (l + i * LPR) * V, have[i]);
  };
  fetch((int64_t)blockIdx.x * GPB + group);
  for (int64_t base = (int64_t)blockIdx.x * GPB; base < rows; base += step) {
    const int64_t row = base + group;
    const bool active = row < rows;
    float v[NV][V];
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      Packet<T>::unpack(next[i], v[i]);
#pragma unroll
      for (int j = 0; j < V; ++j) s += v[i][j];
    }
    if (base + step < rows) fetch(row + step);
    const float mean = row_sum<LPR>(s, red[0]) * inv_n;
    float q = 0.f, r = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (have[i] == V) {
#pragma unroll
        for (int j = 0; j < V; ++j) { v[i][j] -= mean; r += v[i][j]; q = fmaf(v[i][j], v[i][j], q); }
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j)
          if (j < have[i]) { v[i][j] -= mean; r += v[i][j]; q = fmaf(v[i][j], v[i][j], q); }
      }
    }
    const float2 sums = row_sum2<LPR>(r, q, red + 1);
    const RowStat st = row_stat(mean, sums.x, sums.y, inv_n, eps);
    if (active) {
      T* yr = y + row * y_ld;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (l + i * LPR) * V;
        float o[V];
#pragma unroll
        for (int j = 0; j < V; ++j) o[j] = fmaf(fmaf(v[i][j], st.rstd, st.shift), ga[i][j], be[i][j]);
        if (have[i] == V) packet_store(yr + c, Packet<T>::pack(o));
        else store_part(yr + c, have[i], o);
      }
      if (l == 0) {
        if (mean_out) mean_out[row] = st.mean;
        if (rstd_out) rstd_out[row] = st.rstd;
      }
    }
  }
}

// part: [gridDim.x][2][cols], dgamma and dbeta of the block's rows (NULL: not wanted)
template <class T, int LPR, int NV, int THREADS>
__global__ __launch_bounds__(THREADS) void ln_bwd_kernel(const T* dy, int64_t dy_ld, const T* x, int64_t x_ld,
                                                         const float* __restrict__ mean_in,
                                                         const float* __restrict__ rstd_in, int64_t rows, int cols,
                                                         const float* __restrict__ gamma, T* dx, int64_t dx_ld, int acc,
                                                         float* __restrict__ part) {
  constexpr int V = Packet<T>::V, GPB = THREADS / LPR;
  __shared__ float red[2][2][THREADS / 64];
  __shared__ float fold[GPB > 1 ? THREADS * NV * V : 1];
  const int l = threadIdx.x % LPR, group = threadIdx.x / LPR;
  const float inv_n = 1.f / (float)cols;
  float ga[NV][V], dg[NV][V], db[NV][V];
  int have[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (l + i * LPR) * V;
    have[i] = min(max(cols - c, 0), V);
    load_param<V>(gamma, c, have[i], 1.f, ga[i]);
#pragma unroll
    for (int j = 0; j < V; ++j) dg[i][j] = db[i][j] = 0.f;
  }
  const int64_t step = (int64_t)gridDim.x * GPB;
  uint4 next_x[NV], next_g[NV];
  float next_mean, next_rstd;
  auto fetch = [&](int64_t row) {
    row = min(row, rows - 1);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      next_x[i] = fetch_packet(x + row * x_ld + (l + i * LPR) * V, have[i]);
      next_g[i] = fetch_packet(dy + row * dy_ld + (l + i * LPR) * V, have[i]);
    }
    next_mean = mean_in[row];
    next_rstd = rstd_in[row];
  };
  constexpr bool AHEAD = THREADS == 256;               // 1024 threads have 128 registers each, and the row needs them
  if (AHEAD) fetch((int64_t)blockIdx.x * GPB + group);
  int turn = 0;
  for (int64_t base = (int64_t)blockIdx.x * GPB; base < rows; base += step, turn ^= 1) {
    const int64_t row = base + group;
    const bool active = row < rows;
    if (!AHEAD) fetch(row);
    const float mean = next_mean, rstd = next_rstd;
    float xh[NV][V], g[NV][V];
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      Packet<T>::unpack(next_x[i], xh[i]);
      Packet<T>::unpack(next_g[i], g[i]);
    }
    if (AHEAD && base + step < rows) fetch(row + step);
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        xh[i][j] = (xh[i][j] - mean) * rstd;
        if (active) {
          dg[i][j] = fmaf(g[i][j], xh[i][j], dg[i][j]);
          db[i][j] += g[i][j];
        }
        g[i][j] *= ga[i][j];
        s1 += g[i][j];
        s2 = fmaf(g[i][j], xh[i][j], s2);
      }
    s1 = row_sum<LPR>(s1, red[turn][0]) * inv_n;
    s2 = row_sum<LPR>(s2, red[turn][1]) * inv_n;
    if (active) {
      T* dr = dx + row * dx_ld;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (l + i * LPR) * V;
        float o[V];
#pragma unroll
        for (int j = 0; j < V; ++j) o[j] = rstd * fmaf(-xh[i][j], s2, g[i][j] - s1);
        if (acc) {
          float old[V];
          if (have[i] == V) Packet<T>::unpack(packet_load(dr + c), old);
          else load_part(dr + c, have[i], 0.f, old);
#pragma unroll
          for (int j = 0; j < V; ++j) o[j] += old[j];
        }
        if (have[i] == V) packet_store(dr + c, Packet<T>::pack(o));
        else store_part(dr + c, have[i], o);
      }
    }
  }
  if (!part) return;
  float* out = part + (int64_t)blockIdx.x * 2 * cols;
  if constexpr (GPB == 1) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (j < have[i]) {
          out[(l + i * LPR) * V + j] = dg[i][j];
          out[cols + (l + i * LPR) * V + j] = db[i][j];
        }
  } else {
    constexpr int W = LPR * NV * V;                    // padded row of one group
#pragma unroll
    for (int which = 0; which < 2; ++which) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) fold[group * W + (l + i * LPR) * V + j] = which ? db[i][j] : dg[i][j];
      __syncthreads();
      for (int c = threadIdx.x; c < cols; c += THREADS) {
        float s = 0.f;
        for (int k = 0; k < GPB; ++k) s += fold[k * W + c];
        out[which * cols + c] = s;
      }
      __syncthreads();
    }
  }
}

// out[c] = sum_b part[b * stride + c]: 16 columns per block, 64 threads per column, folded through LDS in a fixed order
__global__ __launch_bounds__(1024) void ln_fold_kernel(const float* __restrict__ part, int blocks, int cols,
                                                       float* __restrict__ dgamma, float* __restrict__ dbeta) {
  __shared__ float red[64][17];
  const int c16 = threadIdx.x & 15, r = threadIdx.x >> 4;
  const int c = blockIdx.x * 16 + c16;
  float* out = blockIdx.y ? dbeta : dgamma;
  const float* p = part + (blockIdx.y ? cols : 0) + c;
  float s = 0.f;
  if (c < cols)
    for (int b = r; b < blocks; b += 64) s += p[(int64_t)b * 2 * cols];
  red[r][c16] = s;
  __syncthreads();
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    if (r < o) red[r][c16] += red[r + o][c16];
    __syncthreads();
  }
  if (r == 0 && c < cols && out) out[c] = red[0][c16];
}

// ---- rows wider than LN_MAX_COLS: a block walks its row once per sum (the re-reads come from the caches) -----------
template <class T>
__device__ static inline void wide_load(const T* p, int c, int cols, float fill, float* f) {
  if (c + Packet<T>::V <= cols) Packet<T>::unpack(packet_load(p + c), f);
  else load_part(p + c, cols - c, fill, f);
}

template <class T>
__global__ __launch_bounds__(1024) void ln_fwd_wide_kernel(const T* x, int64_t x_ld, int64_t rows, int cols,
                                                           const float* __restrict__ gamma,
                                                           const float* __restrict__ beta, float eps, T* y,
                                                           int64_t y_ld, float* __restrict__ mean_out,
                                                           float* __restrict__ rstd_out) {
  constexpr int V = Packet<T>::V, STEP = 1024 * V;
  __shared__ float red[3][16];
  const float inv_n = 1.f / (float)cols;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const T* xr = x + row * x_ld;
    T* yr = y + row * y_ld;
    float f[V], s = 0.f, q = 0.f, r = 0.f;
    for (int c = threadIdx.x * V; c < cols; c += STEP) {
      wide_load(xr, c, cols, 0.f, f);
#pragma unroll
      for (int j = 0; j < V; ++j) s += f[j];
    }
    const float mean = row_sum<1024>(s, red[0]) * inv_n;
    for (int c = threadIdx.x * V; c < cols; c += STEP) {
      wide_load(xr, c, cols, mean, f);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        r += f[j] - mean;
        q = fmaf(f[j] - mean, f[j] - mean, q);
      }
    }
    const float2 sums = row_sum2<1024>(r, q, red + 1);
    const RowStat st = row_stat(mean, sums.x, sums.y, inv_n, eps);
    for (int c = threadIdx.x * V; c < cols; c += STEP) {
      wide_load(xr, c, cols, 0.f, f);
      const int n = min(V, cols - c);
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (j < n) f[j] = fmaf(fmaf(f[j] - mean, st.rstd, st.shift), gamma ? gamma[c + j] : 1.f, beta ? beta[c + j] : 0.f);
      if (n == V) packet_store(yr + c, Packet<T>::pack(f));
      else store_part(yr + c, n, f);
    }
    if (threadIdx.x == 0) {
      if (mean_out) mean_out[row] = st.mean;
      if (rstd_out) rstd_out[row] = st.rstd;
    }
  }
}

template <class T>
__global__ __launch_bounds__(1024) void ln_dx_wide_kernel(const T* dy, int64_t dy_ld, const T* x, int64_t x_ld,
                                                          const float* __restrict__ mean_in,
                                                          const float* __restrict__ rstd_in, int64_t rows, int cols,
                                                          const float* __restrict__ gamma, T* dx, int64_t dx_ld,
                                                          int acc) {
  constexpr int V = Packet<T>::V, STEP = 1024 * V;
  __shared__ float red[2][16];
  const float inv_n = 1.f / (float)cols;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const T* xr = x + row * x_ld;
    const T* gr = dy + row * dy_ld;
    T* dr = dx + row * dx_ld;
    const float mean = mean_in[row], rstd = rstd_in[row];
    float f[V], g[V], old[V], s1 = 0.f, s2 = 0.f;
    for (int c = threadIdx.x * V; c < cols; c += STEP) {
      wide_load(xr, c, cols, 0.f, f);
      wide_load(gr, c, cols, 0.f, g);
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (c + j < cols) {
          const float h = g[j] * (gamma ? gamma[c + j] : 1.f);
          s1 += h;
          s2 = fmaf(h, (f[j] - mean) * rstd, s2);
        }
    }
    s1 = row_sum<1024>(s1, red[0]) * inv_n;
    s2 = row_sum<1024>(s2, red[1]) * inv_n;
    for (int c = threadIdx.x * V; c < cols; c += STEP) {
      const int n = min(V, cols - c);
      wide_load(xr, c, cols, 0.f, f);
      wide_load(gr, c, cols, 0.f, g);
      if (acc) wide_load(dr, c, cols, 0.f, old);
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (j < n) {
          const float h = g[j] * (gamma ? gamma[c + j] : 1.f);
          f[j] = fmaf(rstd, fmaf(-(f[j] - mean) * rstd, s2, h - s1), acc ? old[j] : 0.f);
        }
      if (n == V) packet_store(dr + c, Packet<T>::pack(f));
      else store_part(dr + c, n, f);
    }
  }
}

// dgamma / dbeta of LN_STRIP rows x 256 columns per block
template <class T>
__global__ __launch_bounds__(256) void ln_cols_wide_kernel(const T* dy, int64_t dy_ld, const T* x, int64_t x_ld,
                                                           const float* __restrict__ mean_in,
                                                           const float* __restrict__ rstd_in, int64_t rows, int cols,
                                                           int strip, float* __restrict__ part) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= cols) return;
  float dg = 0.f, db = 0.f;
  const int64_t r0 = (int64_t)blockIdx.y * strip, r1 = min(rows, r0 + strip);
  for (int64_t r = r0; r < r1; ++r) {
    const float g = (float)dy[r * dy_ld + c];
    dg = fmaf(g, ((float)x[r * x_ld + c] - mean_in[r]) * rstd_in[r], dg);
    db += g;
  }
  float* out = part + (int64_t)blockIdx.y * 2 * cols;
  out[c] = dg;
  out[cols + c] = db;
}

// ---- host ----------------------------------------------------------------------------------------------------------
// Blocks of the backward: every block ends with one partial row of 2 cols floats.  Two blocks of 256 threads per CU (1024
// columns of bf16: 32 + 4.7 us for the sums; 38 + 6.8 with four), one of 1024 (4096 columns: 36 us; 45 with half as many,
// 39 with twice).
static int ln_bwd_blocks(int64_t rows, int gpb, int threads) {
  const int64_t need = cdiv(rows, gpb);
  const int64_t cap = threads == 256 ? 512 : 256;
  return (int)(need < cap ? (need < 1 ? 1 : need) : cap);
}
// Column sums of wider rows: strips of LN_STRIP rows, longer ones when that would make more than 256 (rows >= 1).
static int ln_wide_strip(int64_t rows) { return (int)(rows <= 256 * LN_STRIP ? LN_STRIP : cdiv(rows, 256)); }
static int ln_wide_strips(int64_t rows) { return (int)cdiv(rows, ln_wide_strip(rows)); }

struct LnShape { int lpr, nv, threads; };
// The fewest lanes that hold the row at one packet per lane; from a whole wave on, up to 16 elements per lane, then
// four waves to a row (forward and backward of 32 Mi fp32 elements, 1024 columns: 45 and 76 us by one wave, 71 and 94 by
// four; 512 columns of bf16: 24 and 34 at one packet per lane, 31 and 51 at two), then a block of 1024 lanes.  A row that
// half the elements per lane would hold gets the kernel for half (bf16, 2048 columns: 24 and 35 us for 33 and 44).
template <class T>
static LnShape ln_shape(int cols) {
  constexpr int V = Packet<T>::V, NVMAX = LN_LANE_ELEMS / V;
  for (int lpr = 2; lpr <= 64; lpr *= 2)
    if (cols <= lpr * V) return {lpr, 1, 256};
  if (cols <= 64 * 2 * V) return {64, 2, 256};
  if (cols <= 64 * NVMAX * V) return {64, NVMAX, 256};
  if (cols <= 256 * NVMAX * V) return {256, cols <= 256 * NVMAX / 2 * V ? NVMAX / 2 : NVMAX, 1024};
  return {1024, cols <= 1024 * NVMAX / 2 * V ? NVMAX / 2 : NVMAX, 1024};
}

#define LN_DISPATCH(T, CALL)                                          \
  do {                                                                \
    constexpr int NVMAX = LN_LANE_ELEMS / Packet<T>::V;               \
    const LnShape sh = ln_shape<T>(cols);                             \
    if (sh.lpr == 2) { CALL(T, 2, 1, 256); }                          \
    else if (sh.lpr == 4) { CALL(T, 4, 1, 256); }                     \
    else if (sh.lpr == 8) { CALL(T, 8, 1, 256); }                     \
    else if (sh.lpr == 16) { CALL(T, 16, 1, 256); }                   \
    else if (sh.lpr == 32) { CALL(T, 32, 1, 256); }                   \
    else if (sh.lpr == 64 && sh.nv == 1) { CALL(T, 64, 1, 256); }     \
    else if (sh.lpr == 64 && sh.nv == 2) { CALL(T, 64, 2, 256); }     \
    else if (sh.lpr == 64) { CALL(T, 64, NVMAX, 256); }               \
    else if (sh.lpr == 256 && sh.nv < NVMAX) { CALL(T, 256, NVMAX / 2, 1024); } \
    else if (sh.lpr == 256) { CALL(T, 256, NVMAX, 1024); }            \
    else if (sh.nv < NVMAX) { CALL(T, 1024, NVMAX / 2, 1024); }       \
    else { CALL(T, 1024, NVMAX, 1024); }                              \
  } while (0)

template <class T>
static void ln_fwd_launch(const T* x, int64_t x_ld, int64_t rows, int cols, const float* gamma, const float* beta,
                          float eps, T* y, int64_t y_ld, float* mean, float* rstd, hipStream_t st) {
  if (cols > LN_MAX_COLS) {
    ln_fwd_wide_kernel<T><<<(int)(rows < 2048 ? rows : 2048), 1024, 0, st>>>(x, x_ld, rows, cols, gamma, beta, eps, y,
                                                                            y_ld, mean, rstd);
    return;
  }
#define LN_FWD(T_, LPR_, NV_, TH_)                                                                               \
  do {                                                                                                           \
    constexpr int TH2 = LPR_ == 256 ? 256 : TH_;                                                                 \
    const int64_t need = cdiv(rows, TH2 / LPR_), cap = TH2 == 256 ? 2048 : 512;                                  \
    ln_fwd_kernel<T_, LPR_, NV_, TH2><<<(int)(need < cap ? need : cap), TH2, 0, st>>>(x, x_ld, rows, cols, gamma, \
                                                                                     beta, eps, y, y_ld, mean, rstd); \
  } while (0)
  LN_DISPATCH(T, LN_FWD);
#undef LN_FWD
}

template <class T>
static void ln_bwd_launch(const T* dy, int64_t dy_ld, const T* x, int64_t x_ld, const float* mean, const float* rstd,
                          int64_t rows, int cols, const float* gamma, T* dx, int64_t dx_ld, int acc, float* dgamma,
                          float* dbeta, float* ws, hipStream_t st) {
  const bool sums = dgamma || dbeta;
  float* part = sums ? ws : nullptr;
  int blocks = 0;
  if (rows > 0 && cols > LN_MAX_COLS) {
    if (part) {
      blocks = ln_wide_strips(rows);
      ln_cols_wide_kernel<T><<<dim3((unsigned)cdiv(cols, 256), blocks), 256, 0, st>>>(dy, dy_ld, x, x_ld, mean, rstd,
                                                                                     rows, cols, ln_wide_strip(rows), part);
    }
    ln_dx_wide_kernel<T><<<(int)(rows < 2048 ? rows : 2048), 1024, 0, st>>>(dy, dy_ld, x, x_ld, mean, rstd, rows, cols,
                                                                           gamma, dx, dx_ld, acc);
  } else if (rows > 0) {
#define LN_BWD(T_, LPR_, NV_, TH_)                                                                                   \
  do {                                                                                                               \
    blocks = ln_bwd_blocks(rows, TH_ / LPR_, TH_);                                                             \
    ln_bwd_kernel<T_, LPR_, NV_, TH_><<<blocks, TH_, 0, st>>>(dy, dy_ld, x, x_ld, mean, rstd, rows, cols, gamma, dx, \
                                                             dx_ld, acc, part);                                      \
  } while (0)
    LN_DISPATCH(T, LN_BWD);
#undef LN_BWD
  }
  if (sums)                                            // without rows: zeros
    ln_fold_kernel<<<dim3((unsigned)cdiv(cols, 16), 2), 1024, 0, st>>>(part, blocks, cols, dgamma, dbeta);
}

static size_t ln_bwd_ws(int64_t rows, int cols) {
  if (rows < 1 || cols < 1) return 0;
  int64_t b = cols > LN_MAX_COLS ? ln_wide_strips(rows) : (rows < 512 ? rows : 512);
  return (size_t)b * 2 * cols * sizeof(float);
}

}  // namespace ctr

using namespace ctr;

extern "C" int ctr_layer_norm_fwd(const void* x, int64_t x_ld, int64_t rows, int cols, int dtype, const float* gamma,
                                  const float* beta, float eps, void* y, int64_t y_ld, float* mean_out, float* rstd_out,
                                  void* stream) {
  CTR_REQUIRE(rows >= 0 && cols >= 1 && cols < (1 << 30), "layer_norm_fwd: rows %lld cols %d (1 to 2^30 - 1)",
              (long long)rows, cols);
  CTR_REQUIRE(type_bytes(dtype) != 0, "layer_norm_fwd: unknown dtype %d", dtype);
  CTR_REQUIRE(eps >= 0.f, "layer_norm_fwd: eps must not be negative");
  if (rows == 0) return CTR_OK;
  CTR_REQUIRE(x && y && x_ld >= cols && y_ld >= cols, "layer_norm_fwd: missing x / y or a leading dimension below cols");
  hipStream_t st = (hipStream_t)stream;
  if (dtype == CTR_F32) ln_fwd_launch((const float*)x, x_ld, rows, cols, gamma, beta, eps, (float*)y, y_ld, mean_out, rstd_out, st);
  else if (dtype == CTR_BF16) ln_fwd_launch((const bf16_t*)x, x_ld, rows, cols, gamma, beta, eps, (bf16_t*)y, y_ld, mean_out, rstd_out, st);
  else ln_fwd_launch((const f16_t*)x, x_ld, rows, cols, gamma, beta, eps, (f16_t*)y, y_ld, mean_out, rstd_out, st);
  CTR_LAUNCH_CHECK();
  return CTR_OK;
}

extern "C" size_t ctr_layer_norm_bwd_workspace_bytes(int64_t rows, int cols) { return ln_bwd_ws(rows, cols); }

extern "C" int ctr_layer_norm_bwd(const void* dy, int64_t dy_ld, const void* x, int64_t x_ld, const float* mean,
                                  const float* rstd, int64_t rows, int cols, int dtype, const float* gamma, void* dx,
                                  int64_t dx_ld, int accumulate_dx, float* dgamma, float* dbeta, void* workspace,
                                  size_t workspace_bytes, void* stream) {
  CTR_REQUIRE(rows >= 0 && cols >= 1 && cols < (1 << 30), "layer_norm_bwd: rows %lld cols %d (1 to 2^30 - 1)",
              (long long)rows, cols);
  CTR_REQUIRE(type_bytes(dtype) != 0, "layer_norm_bwd: unknown dtype %d", dtype);
  CTR_REQUIRE(rows == 0 || (dy && x && mean && rstd && dx && dy_ld >= cols && x_ld >= cols && dx_ld >= cols),
              "layer_norm_bwd: missing tensor or a leading dimension below cols");
  if ((dgamma || dbeta) && (workspace_bytes < ln_bwd_ws(rows, cols) || (!workspace && rows > 0))) {
    set_error("layer_norm_bwd: workspace %zu < %zu", workspace_bytes, ln_bwd_ws(rows, cols));
    return CTR_EWORKSPACE;
  }
  if (rows == 0 && !dgamma && !dbeta) return CTR_OK;
  hipStream_t st = (hipStream_t)stream;
  float* ws = (float*)workspace;
  if (dtype == CTR_F32)
    ln_bwd_launch((const float*)dy, dy_ld, (const float*)x, x_ld, mean, rstd, rows, cols, gamma, (float*)dx, dx_ld,
                  accumulate_dx, dgamma, dbeta, ws, st);
  else if (dtype == CTR_BF16)
    ln_bwd_launch((const bf16_t*)dy, dy_ld, (const bf16_t*)x, x_ld, mean, rstd, rows, cols, gamma, (bf16_t*)dx, dx_ld,
                  accumulate_dx, dgamma, dbeta, ws, st);
  else
    ln_bwd_launch((const f16_t*)dy, dy_ld, (const f16_t*)x, x_ld, mean, rstd, rows, cols, gamma, (f16_t*)dx, dx_ld,
                  accumulate_dx, dgamma, dbeta, ws, st);
  CTR_LAUNCH_CHECK();
  return CTR_OK;
}
