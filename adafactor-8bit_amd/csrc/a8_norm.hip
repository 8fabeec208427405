// Root-mean-square norm with the residual's addition, its output in the input's type or in
// MX blocks, and its backward pass.
//   h = x + r;  s = (mean(h^2) + eps)^(-1/2);  y = h s w
//   g = dy w;   dx = s (g - h s mean(g h s)) + dh;   dw = sum over rows of dy h s
#include "a8_abi_impl.h"
#include "a8_mx.cuh"

namespace a8 {
namespace {

// Sum over the TPR threads of a row (all of the workgroup's when TPR >= 256, else one wave's), the same
// value in each of them.  `lds`: TPR / 64 floats of this call's own.
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* lds) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) v += __shfl_xor(v, o);
  if constexpr (TPR > 64) {
    constexpr int N = TPR / 64;
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    float t[N];
#pragma unroll
    for (int i = 0; i < N; ++i) t[i] = lds[i];
#pragma unroll
    for (int o = N / 2; o > 0; o >>= 1)
#pragma unroll
      for (int i = 0; i < o; ++i) t[i] += t[i + o];
    v = t[0];
  }
  return v;
}

template <typename T>
__device__ __forceinline__ void load8(const T* p, int64_t col, int64_t cols, float* v) {
  if (col + 8 <= cols) {
    mx_loadn<8>(p + col, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = col + i < cols ? mx_f(p[col + i]) : 0.0f;
  }
}

template <typename T>
__device__ __forceinline__ void store8(T* p, int64_t col, int64_t cols, const float* v) {
  if (col + 8 <= cols) {
    mx_storen<8>(p + col, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (col + i < cols) p[col + i] = mx_to<T>(v[i]);
  }
}

// Eight columns as they lie in memory (zeros past the row's end), and as fp32.
template <typename T>
struct Raw8 {
  static constexpr int N = (int)sizeof(T) / 2;
  u32x4 w[N];
  __device__ __forceinline__ void load(const T* p, int64_t col, int64_t cols) {
    if (col + 8 <= cols) {
#pragma unroll
      for (int i = 0; i < N; ++i) w[i] = *(const A8_G u32x4_a2*)gp(reinterpret_cast<const u32x4*>(p + col + i * (8 / N)));
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) w[i] = u32x4{0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (col + i < cols) {
          if constexpr (N == 2) w[i / 4][i % 4] = *gp(reinterpret_cast<const uint32_t*>(p + col + i));
          else w[0][i / 2] |= (uint32_t)*gp(reinterpret_cast<const uint16_t*>(p + col + i)) << (16 * (i & 1));
        }
    }
  }
  __device__ __forceinline__ void get(float* v) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (N == 2) {
        v[i] = __uint_as_float(w[i / 4][i % 4]);
      } else {
        const uint16_t u = (uint16_t)(w[0][i / 2] >> (16 * (i & 1)));
        v[i] = mx_f(__builtin_bit_cast(T, u));
      }
    }
  }
};

// What lies below h's 16-bit value: the next four bits of the fp32 mantissa, rounded, for eight columns in a
// word.  With them the backward pass has h to a sixteenth of its type's unit; from the rounded h alone, dw of
// 16384 rows is off by as much again as its own rounding to bf16 (2.5e-3 in all, 1.7e-3 with the bits), for half a
// byte an element written and read once.  Zero where h is exact, infinite or NaN.
template <typename R>
constexpr bool kLow = sizeof(R) == 2;
template <typename R>
constexpr int kLowShift = std::is_same<R, __half>::value ? 9 : 12;   // fp32's bits below those four

template <typename R>
__device__ __forceinline__ void put_low(uint32_t* low, int64_t row, int64_t col, int64_t cols, const float* v) {
  if (col >= cols) return;
  constexpr int S = kLowShift<R>;
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t b = __float_as_uint(v[i]), n = __float_as_uint(mx_f(mx_to<R>(v[i])));
    int e = (int)((b + (1u << (S - 1))) >> S) - (int)(n >> S);
    e = e < -8 ? -8 : e > 7 ? 7 : e;   // half a unit up is 8: there, and among fp16's subnormals, a quantum short
    if ((n & 0x7f800000u) == 0x7f800000u) e = 0;
    w |= ((uint32_t)e & 15) << (4 * i);
  }
  low[row * ((cols + 7) / 8) + col / 8] = w;
}

__device__ __forceinline__ uint32_t get_low(const uint32_t* low, int64_t row, int64_t col, int64_t cols) {
  return low && col < cols ? *gp(low + row * ((cols + 7) / 8) + col / 8) : 0;
}

template <typename R>
__device__ __forceinline__ void add_low(uint32_t w, float* v) {
#pragma unroll
  for (int i = 0; i < 8; ++i)
    v[i] = __uint_as_float(__float_as_uint(v[i]) + (uint32_t)(((int32_t)(w << (28 - 4 * i)) >> 28) * (1 << kLowShift<R>)));
}

// y = v w s of eight columns; OUT: 0 the input's type, 1 + format an MX tensor
template <int OUT, typename T>
__device__ __forceinline__ void put8(T* y, uint8_t* codes, uint8_t* scales, int64_t row, int64_t col, int64_t cols,
                                     int64_t pitch, const float* v, int ceil) {
  if constexpr (OUT == 0) {
    store8(y + row * cols, col, cols, v);
  } else {
    constexpr int FMT = OUT - 1;
    const int64_t e = row * pitch + col;
    mx_put8<FMT, false>(v, ceil != 0, 0, 0, codes + (FMT == kFp8 ? e : e / 2), scales + e / 32);
  }
}

// A row by TPR threads, eight columns and NC times that a thread, read once: x, r and the weight are
// asked for together, and h stays in registers between the sum and the output.  Bound by memory: 16384 x 4096
// bf16 with a residual 100 us (5.3 TB/s), into 8 bits 90 us; one row of 4096 4.3 us, its loads' and the sum's latency.
template <typename T, typename R, typename W, int OUT, int TPR, int NC>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void k_rms(const T* x, int64_t xs, const R* r, int64_t rs, const W* w,
                                                               T* y, uint8_t* codes, uint8_t* scales, R* h,
                                                               uint32_t* low, float* rstd, int64_t rows, int64_t cols, float eps,
                                                               int ceil) {
  __shared__ float lds[TPR / 64];
  constexpr int kRows = TPR < 256 ? 256 / TPR : 1;
  const int t = threadIdx.x % TPR;
  const int64_t row = (int64_t)blockIdx.x * kRows + threadIdx.x / TPR;
  if (row >= rows) return;   // whole waves, and only where a row is one wave's
  const int64_t pitch = mx_pitch(cols), end = OUT ? pitch : cols;
  float v[NC][8], u[NC][8];
  float sum = 0.0f;
#pragma unroll
  for (int i = 0; i < NC; ++i) load8(x + row * xs, (i * TPR + t) * 8, cols, v[i]);
  if (r) {
#pragma unroll
    for (int i = 0; i < NC; ++i) load8(r + row * rs, (i * TPR + t) * 8, cols, u[i]);
#pragma unroll
    for (int i = 0; i < NC; ++i) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] += u[i][j];
      store8(h + row * cols, (i * TPR + t) * 8, cols, v[i]);
      if (kLow<R> && low) put_low<R>(low, row, (i * TPR + t) * 8, cols, v[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < NC; ++i) load8(w, (i * TPR + t) * 8, cols, u[i]);
#pragma unroll
  for (int i = 0; i < NC; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) sum += v[i][j] * v[i][j];
  sum = row_sum<TPR>(sum, lds);
  const float s = 1.0f / __builtin_sqrtf(sum / (float)cols + eps);
  if (rstd && t == 0) rstd[row] = s;
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const int64_t c = (i * TPR + t) * 8;
#pragma unroll
    for (int j = 0; j < 8; ++j) v[i][j] = (v[i][j] * s) * u[i][j];
    if (c < end) put8<OUT>(y, codes, scales, row, c, cols, pitch, v[i], ceil);
  }
}

// Rows longer than the registers hold: a second reading, mostly from the caches.
template <typename T, typename R, typename W, int OUT>
__global__ __launch_bounds__(1024) void k_rms_long(const T* x, int64_t xs, const R* r, int64_t rs, const W* w, T* y,
                                                   uint8_t* codes, uint8_t* scales, R* h, uint32_t* low, float* rstd,
                                                   int64_t cols, float eps, int ceil) {
  __shared__ float lds[16];
  const int64_t row = blockIdx.x, pitch = mx_pitch(cols), end = OUT ? pitch : cols;
  x += row * xs;
  auto load = [&](int64_t c, float* v, bool first) {
    load8(x, c, cols, v);
    if (r) {
      float u[8];
      load8(r + row * rs, c, cols, u);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] += u[i];
      if (first) store8(h + row * cols, c, cols, v);
      if (kLow<R> && first && low) put_low<R>(low, row, c, cols, v);
    }
  };
  float sum = 0.0f;
  for (int64_t c = (int64_t)threadIdx.x * 8; c < cols; c += 8192) {
    float v[8], part = 0.0f;
    load(c, v, true);
#pragma unroll
    for (int i = 0; i < 8; ++i) part += v[i] * v[i];
    sum += part;
  }
  sum = row_sum<1024>(sum, lds);
  const float s = 1.0f / __builtin_sqrtf(sum / (float)cols + eps);
  if (rstd && threadIdx.x == 0) rstd[row] = s;
  for (int64_t c = (int64_t)threadIdx.x * 8; c < end; c += 8192) {
    float v[8], u[8];
    load(c, v, false);
    load8(w, c, cols, u);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (v[i] * s) * u[i];
    put8<OUT>(y, codes, scales, row, c, cols, pitch, v, ceil);
  }
}

// A workgroup takes every grid-th row (every grid-th four, one a wave, where a row is one wave's); a thread
// keeps its columns of the weight and of dw's sum in registers, and asks for its next row before this one's sum
// is known: without that 16384 x 4096 bf16 with a residual takes 165 us, with it 117 (4.6 TB/s), bound by memory;
// 124 with the bits below h.
// parts [grid, cols]: each workgroup's dw (NULL: none).
template <typename T, typename R, typename W, int TPR, int NC>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void k_rms_bwd(const T* dy, const R* dh, const R* h, const uint32_t* low,
                                                 const W* w, const float* rstd, T* dx, R* dr, float* parts,
                                                 int64_t rows, int64_t cols) {
  __shared__ float lds[2][TPR / 64];
  constexpr int K = TPR < 256 ? 256 / TPR : 1;
  const int t = threadIdx.x % TPR, slot = threadIdx.x / TPR;
  // sixteen waves have 128 registers each: too few for the weight and for the next row's dh (4096 x 16384
  // bf16 with a residual: 145 us, 264 with them)
  constexpr bool kRoom = TPR < 1024;
  float wv[NC][8], dw[NC][8];
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    if (kRoom) load8(w, (i * TPR + t) * 8, cols, wv[i]);
#pragma unroll
    for (int j = 0; j < 8; ++j) dw[i][j] = 0.0f;
  }
  const float inv = 1.0f / (float)cols;
  Raw8<T> gr[NC];
  Raw8<R> vr[NC], ur[NC];
  uint32_t lr[NC];
  float sr = 0.0f;
  auto load = [&](int64_t row) {
    sr = rstd[row];
#pragma unroll
    for (int i = 0; i < NC; ++i) gr[i].load(dy + row * cols, (i * TPR + t) * 8, cols);
#pragma unroll
    for (int i = 0; i < NC; ++i) vr[i].load(h + row * cols, (i * TPR + t) * 8, cols);
    if constexpr (kLow<R>)
#pragma unroll
      for (int i = 0; i < NC; ++i) lr[i] = get_low(low, row, (i * TPR + t) * 8, cols);
    if (kRoom && dh)
#pragma unroll
      for (int i = 0; i < NC; ++i) ur[i].load(dh + row * cols, (i * TPR + t) * 8, cols);
  };
  int64_t row = (int64_t)blockIdx.x * K + slot;
  const int64_t step = (int64_t)gridDim.x * K;
  if (row < rows) load(row);
  for (int turn = 0; row < rows; row += step, turn ^= 1) {
    float g[NC][8], v[NC][8], u[NC][8];
    const float s = sr;
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      gr[i].get(g[i]);
      vr[i].get(v[i]);
      if constexpr (kLow<R>) add_low<R>(lr[i], v[i]);
      if (kRoom && dh) ur[i].get(u[i]);
      if (!kRoom) load8(w, (i * TPR + t) * 8, cols, wv[i]);
    }
    if (row + step < rows) load(row + step);   // in flight while this row's sum and output are formed
#pragma unroll
    for (int i = 0; i < NC; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        v[i][j] *= s;
        dw[i][j] += g[i][j] * v[i][j];
        g[i][j] *= wv[i][j];
        sum += g[i][j] * v[i][j];
      }
    sum = row_sum<TPR>(sum, lds[turn]) * inv;
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int64_t c = (i * TPR + t) * 8;
      if (!kRoom && dh) load8(dh + row * cols, c, cols, u[i]);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        v[i][j] = s * (g[i][j] - v[i][j] * sum);
        if (dh) v[i][j] += u[i][j];
      }
      if (c < cols) {
        store8(dx + row * cols, c, cols, v[i]);
        if (dr) store8(dr + row * cols, c, cols, v[i]);
      }
    }
  }
  if (!parts) return;      // the weight's gradient is not wanted
  if constexpr (K > 1) {   // the waves' sums, in their order
    __shared__ __align__(16) float all[K][8 * TPR];
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      if (i) __syncthreads();
#pragma unroll
      for (int j = 0; j < 8; j += 4)
        *reinterpret_cast<f32x4*>(&all[slot][8 * t + j]) = f32x4{dw[i][j], dw[i][j + 1], dw[i][j + 2], dw[i][j + 3]};
      __syncthreads();
      if (slot == 0)
#pragma unroll
        for (int k = 1; k < K; ++k)
#pragma unroll
          for (int j = 0; j < 8; ++j) dw[i][j] += all[k][8 * t + j];
    }
    if (slot) return;
  }
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const int64_t c = (i * TPR + t) * 8;
    if (c < cols) store8(parts + (int64_t)blockIdx.x * cols, c, cols, dw[i]);
  }
}

template <typename T, typename R, typename W>
__global__ __launch_bounds__(1024) void k_rms_bwd_long(const T* dy, const R* dh, const R* h, const uint32_t* low,
                                                       const W* w, const float* rstd, T* dx, R* dr, float* parts, int64_t rows,
                                                       int64_t cols) {
  __shared__ float lds[2][16];
  int turn = 0;
  const bool sums = parts != nullptr;
  if (sums) parts += (int64_t)blockIdx.x * cols;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x, turn ^= 1) {
    const float s = rstd[row];
    float sum = 0.0f;
    for (int64_t c = (int64_t)threadIdx.x * 8; c < cols; c += 8192) {
      float g[8], v[8], u[8], d[8], part = 0.0f;
      load8(dy + row * cols, c, cols, g);
      load8(h + row * cols, c, cols, v);
      if constexpr (kLow<R>) add_low<R>(get_low(low, row, c, cols), v);
      load8(w, c, cols, u);
      if (sums && row != blockIdx.x) load8(parts, c, cols, d);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float xn = v[i] * s;
        part += (g[i] * u[i]) * xn;
        d[i] = row == blockIdx.x ? g[i] * xn : d[i] + g[i] * xn;
      }
      sum += part;
      if (sums) store8(parts, c, cols, d);
    }
    sum = row_sum<1024>(sum, lds[turn]) / (float)cols;
    for (int64_t c = (int64_t)threadIdx.x * 8; c < cols; c += 8192) {
      float g[8], v[8], u[8];
      load8(dy + row * cols, c, cols, g);
      load8(h + row * cols, c, cols, v);
      if constexpr (kLow<R>) add_low<R>(get_low(low, row, c, cols), v);
      load8(w, c, cols, u);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = s * (g[i] * u[i] - (v[i] * s) * sum);
      if (dh) {
        load8(dh + row * cols, c, cols, u);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] += u[i];
      }
      store8(dx + row * cols, c, cols, v);
      if (dr) store8(dr + row * cols, c, cols, v);
    }
  }
}

// dw from the workgroups' sums: 32 columns a workgroup, 32 half waves each a run of the n rows of parts (1024 x
// 4096: 5 us), in a fixed order.
template <typename W>
__global__ __launch_bounds__(1024) void k_rms_dw(const float* parts, W* dw, int64_t cols, int n) {
  __shared__ float lds[32][32];
  const int part = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t c = (int64_t)blockIdx.x * 32 + lane;
  float s = 0.0f;
  if (c < cols) {
    const int i1 = n * (part + 1) / 32;
    int i = n * part / 32;
    for (; i + 8 <= i1; i += 8) {
      float t[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) t[j] = parts[(int64_t)(i + j) * cols + c];
      s += ((t[0] + t[1]) + (t[2] + t[3])) + ((t[4] + t[5]) + (t[6] + t[7]));
    }
    for (; i < i1; ++i) s += parts[(int64_t)i * cols + c];
  }
  lds[part][lane] = s;
  __syncthreads();
  if (part == 0 && c < cols) {
#pragma unroll
    for (int j = 1; j < 32; ++j) s += lds[j][lane];
    dw[c] = mx_to<W>(s);
  }
}

// Workgroups of the backward pass: about sixteen waves a CU, fewer where that leaves each the same number
// of rows.
int bwd_groups(int64_t rows, int64_t cols) {
  const int64_t at_once = cols <= 1024 ? 4 : 1, most = cols <= 4096 ? 1024 : cols <= 8192 ? 512 : 256;
  const int64_t turns = (rows + at_once - 1) / at_once, each = (turns + most - 1) / most;
  return (int)(each ? (turns + each - 1) / each : 0);
}

// Threads a row, and times eight columns a thread (eight keep every access 16 bytes wide).  A row goes to
// the fewest threads that hold it: two such pieces a thread leave the backward pass three waves a SIMD
// (777 x 5003 fp32: 17.4 us with 512 threads, 26.2 with 256 and four pieces); four are for the longest rows of
// the forward pass alone.
template <bool kForward, typename F>
int with_shape(int64_t cols, F&& f) {
  if (cols <= 512) return f(std::integral_constant<int, 64>{}, std::integral_constant<int, 1>{});
  if (cols <= 1024) return f(std::integral_constant<int, 64>{}, std::integral_constant<int, 2>{});
  if (cols <= 2048) return f(std::integral_constant<int, 256>{}, std::integral_constant<int, 1>{});
  if (cols <= 4096) return f(std::integral_constant<int, 256>{}, std::integral_constant<int, 2>{});
  if (cols <= 8192) return f(std::integral_constant<int, 512>{}, std::integral_constant<int, 2>{});
  if constexpr (kForward)
    if (cols > 16384) return f(std::integral_constant<int, 1024>{}, std::integral_constant<int, 4>{});
  return f(std::integral_constant<int, 1024>{}, std::integral_constant<int, 2>{});
}
constexpr int64_t kLong = 32768, kLongBwd = 16384;

template <typename T, typename R, typename W, int OUT>
int rms_out(const T* x, int64_t xs, const R* r, int64_t rs, const W* w, T* y, uint8_t* codes, uint8_t* scales, R* h,
            uint32_t* low, float* rstd, int64_t rows, int64_t cols, float eps, int ceil, hipStream_t st) {
  const int64_t pitch = mx_pitch(cols), wide = OUT ? pitch : cols;
  // `most` rows a launch: f(first row, rows, the arrays from the first row on)
  auto go = [&](int64_t most, auto&& f) {
    return in_runs(rows, most, [&](int64_t first, int64_t count) {
      const int64_t e = first * pitch;
      return f(count, x + first * xs, r ? r + first * rs : nullptr, y ? y + first * cols : nullptr,
               codes ? codes + (OUT == 1 + kFp8 ? e : e / 2) : nullptr, scales ? scales + e / 32 : nullptr,
               h ? h + first * cols : nullptr, low ? low + first * ((cols + 7) / 8) : nullptr,
               rstd ? rstd + first : nullptr);
    });
  };
  if (wide > kLong)
    return go(most_groups(1024), [&](int64_t n, auto x, auto r, auto y, auto codes, auto scales, auto h, auto low, auto rstd) {
      k_rms_long<T, R, W, OUT><<<(uint32_t)n, 1024, 0, st>>>(x, xs, r, rs, w, y, codes, scales, h, low, rstd, cols, eps, ceil);
      return check_launch("k_rms_long");
    });
  return with_shape<true>(wide, [&](auto tpr, auto nc) {
    constexpr int TPR = decltype(tpr)::value, NC = decltype(nc)::value, B = TPR < 256 ? 256 : TPR, K = B / TPR;
    return go(most_groups(B) * K, [&](int64_t n, auto x, auto r, auto y, auto codes, auto scales, auto h, auto low, auto rstd) {
      k_rms<T, R, W, OUT, TPR, NC><<<(uint32_t)((n + K - 1) / K), B, 0, st>>>(x, xs, r, rs, w, y, codes, scales, h, low, rstd,
                                                                              n, cols, eps, ceil);
      return check_launch("k_rms");
    });
  });
}

template <typename T, typename R, typename W>
int rms(int out, const void* x, int64_t xs, const void* r, int64_t rs, const void* w, void* y, uint8_t* codes,
        uint8_t* scales, void* h, uint32_t* low, float* rstd, int64_t rows, int64_t cols, float eps, int ceil,
        hipStream_t st) {
  auto go = [&](auto o) {
    return rms_out<T, R, W, decltype(o)::value>(static_cast<const T*>(x), xs, static_cast<const R*>(r), rs,
                                                static_cast<const W*>(w), static_cast<T*>(y), codes, scales,
                                                static_cast<R*>(h), low, rstd, rows, cols, eps, ceil, st);
  };
  if (out == 0) return go(std::integral_constant<int, 0>{});
  if (out == 1 + kFp4) return go(std::integral_constant<int, 1 + kFp4>{});
  return go(std::integral_constant<int, 1 + kFp8>{});
}

template <typename T, typename R, typename W>
int rms_bwd(const void* dy_, const void* dh_, const void* h_, const uint32_t* low, const void* w_, const float* rstd,
            void* dx_, void* dr_, void* dw, float* parts, int64_t rows, int64_t cols, hipStream_t st) {
  const int n = bwd_groups(rows, cols);
  if (!dw) parts = nullptr;
  const T* dy = static_cast<const T*>(dy_);
  const R *dh = static_cast<const R*>(dh_), *h = static_cast<const R*>(h_);
  const W* w = static_cast<const W*>(w_);
  T* dx = static_cast<T*>(dx_);
  R* dr = static_cast<R*>(dr_);
  int e = A8_OK;
  if (n > 0 && cols > kLongBwd) {
    k_rms_bwd_long<T, R, W><<<n, 1024, 0, st>>>(dy, dh, h, low, w, rstd, dx, dr, parts, rows, cols);
    e = check_launch("k_rms_bwd_long");
  } else if (n > 0) {
    e = with_shape<false>(cols, [&](auto tpr, auto nc) {
      constexpr int TPR = decltype(tpr)::value, NC = decltype(nc)::value;
      k_rms_bwd<T, R, W, TPR, NC><<<n, TPR < 256 ? 256 : TPR, 0, st>>>(dy, dh, h, low, w, rstd, dx, dr, parts, rows, cols);
      return check_launch("k_rms_bwd");
    });
  }
  if (e || !dw) return e;
  k_rms_dw<W><<<(uint32_t)((cols + 31) / 32), 1024, 0, st>>>(parts, static_cast<W*>(dw), cols, n);
  return check_launch("k_rms_dw");
}

// The types a call may have: x, y, dx and dy in `dtype`; the residual stream and the weight in
// that type or in fp32.
template <typename F>
int with_types(int dtype, int rdtype, int wdtype, F&& f) {
  auto rest = [&](auto t) {
    typedef decltype(t) T;
    if (rdtype == dtype) return wdtype == dtype ? f(T{}, T{}, T{}) : f(T{}, T{}, float{});
    return wdtype == dtype ? f(T{}, float{}, T{}) : f(T{}, float{}, float{});
  };
  if (dtype == A8_F32) return f(float{}, float{}, float{});
  if (dtype == A8_BF16) return rest(__hip_bfloat16{});
  return rest(__half{});
}

int check_types(int dtype, int rdtype, int wdtype, const char* msg) {
  if (dtype != A8_F32 && dtype != A8_BF16 && dtype != A8_F16) return set_error(A8_ERR_DTYPE, msg);
  if ((rdtype != dtype && rdtype != A8_F32) || (wdtype != dtype && wdtype != A8_F32)) return set_error(A8_ERR_DTYPE, msg);
  return A8_OK;
}

constexpr int64_t kLim = (int64_t)1 << 31;

}  // namespace
}  // namespace a8

using namespace a8;

extern "C" int a8_rms_norm(int dtype, int res_dtype, int w_dtype, int out_fmt, const void* x, int64_t x_stride,
                           const void* residual, int64_t r_stride, const void* weight, void* y, uint8_t* codes,
                           uint8_t* scales, void* h, uint32_t* h_low, float* rstd, int64_t rows, int64_t cols,
                           float eps, void* stream) {
  if (int e = check_types(dtype, res_dtype, w_dtype, "rms_norm: x must be fp32, bf16 or fp16, the residual and the "
                                                     "weight of that type or fp32")) return e;
  const int ceil = out_fmt >= 0 && (out_fmt & A8_MX_CEIL) != 0;
  if (ceil) out_fmt &= ~A8_MX_CEIL;
  if (out_fmt != A8_MX_NONE && out_fmt != A8_MXFP4 && out_fmt != A8_MXFP8)
    return set_error(A8_ERR_ARG, "rms_norm: unknown output format");
  if (rows < 0 || rows >= kLim || cols < 1 || cols >= kLim) return set_error(A8_ERR_SIZE, "rms_norm: rows or cols out of range");
  if (rows == 0) return A8_OK;
  if (x_stride < 0 || r_stride < 0) return set_error(A8_ERR_ARG, "rms_norm: negative row stride");
  if (!x || !weight || (residual && !h) || (out_fmt == A8_MX_NONE ? !y : (!codes || !scales)))
    return set_error(A8_ERR_ARG, "rms_norm: null pointer");
  if (out_fmt != A8_MX_NONE && !aligned16(codes)) return set_error(A8_ERR_ALIGN, "rms_norm: codes must be 16-byte aligned");
  return with_types(dtype, res_dtype, w_dtype, [&](auto t, auto r, auto w) {
    return rms<decltype(t), decltype(r), decltype(w)>(out_fmt + 1, x, x_stride, residual, r_stride, weight, y, codes, scales,
                                                      h, h_low, rstd, rows, cols, eps, ceil, static_cast<hipStream_t>(stream));
  });
}

extern "C" int64_t a8_rms_norm_workspace_floats(int64_t rows, int64_t cols) {
  return rows < 0 || cols < 0 ? -1 : (int64_t)bwd_groups(rows, cols) * cols;
}

extern "C" int a8_rms_norm_backward(int dtype, int res_dtype, int w_dtype, const void* dy, const void* dh, const void* h,
                                    const uint32_t* h_low, const void* weight, const float* rstd, void* dx, void* dr, void* dw,
                                    float* workspace, int64_t rows, int64_t cols, void* stream) {
  if (int e = check_types(dtype, res_dtype, w_dtype, "rms_norm_backward: dy must be fp32, bf16 or fp16, the residual and "
                                                     "the weight of that type or fp32")) return e;
  if (rows < 0 || rows >= kLim || cols < 1 || (cols + 31) / 32 > most_groups(1024))   // k_rms_dw's workgroups
    return set_error(A8_ERR_SIZE, "rms_norm_backward: rows or cols out of range");
  if (rows > 0 && (!dy || !h || !weight || !rstd || !dx || (dw && !workspace)))
    return set_error(A8_ERR_ARG, "rms_norm_backward: null pointer");
  return with_types(dtype, res_dtype, w_dtype, [&](auto t, auto r, auto w) {
    return rms_bwd<decltype(t), decltype(r), decltype(w)>(dy, dh, h, h_low, weight, rstd, dx, dr, dw, workspace, rows, cols,
                                                          static_cast<hipStream_t>(stream));
  });
}
