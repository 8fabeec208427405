// Microscaled (MX) blocks: 32 elements along a row share a power-of-two scale in
// 8 bits (E8M0: byte b stands for 2^(b - 127), 255 for NaN) and are held as E2M1
// (two a byte, the even element in the low half) or E4M3 codes.
//
//   scale    e = floor(log2 amax) - emax (emax 2 / 8); "ceil" adds one where amax
//            would saturate, so that amax <= top * 2^e (top 6 / 448); e >= -127
//   code     v * 2^-e (exact), saturated to +-top, to the grid: ties to even, or
//            stochastically floor(t / step + (u + 1/2) / 2^16) * step
//   special  a NaN or infinity in a block: scale 255, codes 0 (it reads as NaN)
//
// Rows are padded to a multiple of 256 elements with codes 0 (and scale 2^-127),
// so the products need no mask along the contraction.
#pragma once
#include "a8_common.cuh"
#include "a8_mcodec.cuh"

namespace a8 {

constexpr int kFp4 = A8_MXFP4, kFp8 = A8_MXFP8;
constexpr int64_t kMxPad = 256;

__host__ __device__ inline int64_t mx_pitch(int64_t cols) { return (cols + kMxPad - 1) / kMxPad * kMxPad; }

typedef short s16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
// loads and stores at any element alignment
typedef u32x4 u32x4_a2 __attribute__((aligned(2)));
typedef u32x2 u32x2_a2 __attribute__((aligned(2)));

template <typename T>
__device__ __forceinline__ float mx_f(T v) {
  if constexpr (std::is_same<T, __hip_bfloat16>::value) return __uint_as_float((uint32_t)__bfloat16_as_ushort(v) << 16);
  else if constexpr (std::is_same<T, __half>::value) return __half2float(v);
  else return v;
}

// fp32 -> T, round to nearest even (NaN stays NaN)
template <typename T>
__device__ __forceinline__ T mx_to(float v) {
  if constexpr (std::is_same<T, __hip_bfloat16>::value) {
    typedef __bf16 b;
    const b r = (b)v;
    return __ushort_as_bfloat16(__builtin_bit_cast(uint16_t, r));
  } else if constexpr (std::is_same<T, __half>::value) {
    return __float2half_rn(v);
  } else {
    return v;
  }
}

// N consecutive elements from an address aligned to the element only, in 16-byte
// accesses (gfx950 takes them at any element alignment).
template <int N, typename T>
__device__ __forceinline__ void mx_loadn(const T* p, float* v) {
  constexpr int W = 16 / (int)sizeof(T);
  static_assert(N % W == 0, "");
#pragma unroll
  for (int i = 0; i < N; i += W) {
    const u32x4 w = *(const A8_G u32x4_a2*)gp(reinterpret_cast<const u32x4*>(p + i));
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (sizeof(T) == 4) {
        v[i + j] = __uint_as_float(w[j]);
      } else {
        const uint16_t lo = (uint16_t)w[j], hi = (uint16_t)(w[j] >> 16);
        v[i + 2 * j] = mx_f(__builtin_bit_cast(T, lo));
        v[i + 2 * j + 1] = mx_f(__builtin_bit_cast(T, hi));
      }
    }
  }
}

template <typename T>
__device__ __forceinline__ void mx_load4(const T* p, float* v) {
  if constexpr (sizeof(T) == 4) {
    const u32x4 w = *(const A8_G u32x4_a2*)gp(reinterpret_cast<const u32x4*>(p));
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = __uint_as_float(w[j]);
  } else {
    const u32x2 w = *(const A8_G u32x2_a2*)gp(reinterpret_cast<const u32x2*>(p));
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint16_t lo = (uint16_t)w[j], hi = (uint16_t)(w[j] >> 16);
      v[2 * j] = mx_f(__builtin_bit_cast(T, lo));
      v[2 * j + 1] = mx_f(__builtin_bit_cast(T, hi));
    }
  }
}

template <typename T>
__device__ __forceinline__ uint32_t mx_pack2(float a, float b) {
  static_assert(sizeof(T) == 2, "");
  const T x = mx_to<T>(a), y = mx_to<T>(b);
  return (uint32_t)__builtin_bit_cast(uint16_t, x) | ((uint32_t)__builtin_bit_cast(uint16_t, y) << 16);
}

template <int N, typename T>
__device__ __forceinline__ void mx_storen(T* p, const float* v) {
  constexpr int W = sizeof(T) == 4 ? 4 : 8;
  static_assert(N % W == 0, "");
#pragma unroll
  for (int i = 0; i < N; i += W) {
    u32x4 w;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (sizeof(T) == 4) w[j] = __float_as_uint(v[i + j]);
      else w[j] = mx_pack2<T>(v[i + 2 * j], v[i + 2 * j + 1]);
    }
    *(A8_G u32x4_a2*)gp(reinterpret_cast<u32x4*>(p + i)) = w;
  }
}

__device__ __forceinline__ uint32_t mx_absbits(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }
__device__ __forceinline__ uint32_t mx_umax(uint32_t a, uint32_t b) { return a > b ? a : b; }

// A block's scale from the largest magnitude's bits: the E8M0 byte (255 when the
// block holds a NaN or an infinity) and 2^-e.
struct MxScale {
  uint32_t byte;
  float inv;
  __device__ __forceinline__ bool bad() const { return byte == 255u; }
};
template <int FMT>
__device__ __forceinline__ MxScale mx_scale(uint32_t amax, bool ceil) {
  constexpr int emax = FMT == kFp4 ? 2 : 8;
  constexpr uint32_t topm = FMT == kFp4 ? 0x400000u : 0x600000u;
  int b = (int)(amax >> 23) - emax + (int)(ceil && (amax & 0x7FFFFFu) > topm);   // e + 127
  b = b < 0 ? 0 : b;
  MxScale s;
  s.byte = amax >= 0x7F800000u ? 255u : (uint32_t)b;
  s.inv = __uint_as_float((uint32_t)(254 - b) << 23);
  return s;
}

// E8M0 byte -> fp32
__device__ __forceinline__ float mx_scale_value(uint32_t b) {
  const uint32_t u = b == 0u ? 0x00400000u : (b == 255u ? 0x7FC00000u : b << 23);
  return __uint_as_float(u);
}

// Four scaled values to the grid, up with the probability of the distance: value j by the j-th 16 bits u of
// r, floor(t / step + (u + 1/2) / 2^16) * step in fp32.  In the bits of a normal value the grid's digits end
// mb below the point, so (u + 1/2) / 2^16 added to the rest of the mantissa carries into them exactly where
// that floor is one more; below the grid's normal values the step is the same for all.
template <int FMT>
__device__ __forceinline__ void mx_sr4(float* t, uint64_t r) {
  constexpr int mb = FMT == kFp4 ? 1 : 3, cut = 23 - mb;
  constexpr float low = FMT == kFp4 ? 1.0f : 0.015625f, top = FMT == kFp4 ? 6.0f : 448.0f;
  constexpr float step = low / (1 << mb);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t word = (uint32_t)(r >> (32 * (j / 2))), u = j & 1 ? word >> 16 : word & 0xFFFFu;
    uint32_t b = (__float_as_uint(t[j]) + (u << (cut - 16)) + (1u << (cut - 17))) & ~((1u << cut) - 1u);
    const float up = __builtin_fmaf((float)u, 1.0f / 65536.0f, 0.5f / 65536.0f);
    float s = floorf(__builtin_fmaf(fabsf(t[j]), 1.0f / step, up)) * step;
    asm("" : "+v"(b), "+v"(s));   // both are formed: a branch for each element costs more
    const float q = fabsf(t[j]) < low ? s : fabsf(__uint_as_float(b));
    t[j] = __builtin_copysignf(__builtin_amdgcn_fmed3f(q, 0.0f, top), t[j]);
  }
}

// Four consecutive elements' 16 random bits each: one output of SplitMix64, whose counter is base +
// (element index / 4), base = seed * 0x9E3779B97F4A7C15, for the transpose + 0xD1B54A32D192ED03.
__device__ __forceinline__ uint64_t mx_random(uint64_t base, uint64_t word) {
  uint64_t z = base + word + 0x9E3779B97F4A7C15ULL;
  z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ULL;
  z = (z ^ (z >> 27)) * 0x94D049BB133111EBULL;
  return z ^ (z >> 31);
}

// N scaled values (a multiple of 4, or of 8 for E2M1) to codes: N bytes (E4M3) or N / 2 (E2M1).  SAT: they
// may lie beyond the format's largest value.
template <int FMT, int N, bool SAT>
__device__ __forceinline__ void mx_encode(const float* t, uint32_t* out) {
  if constexpr (FMT == kFp8) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      float c[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) c[j] = SAT ? __builtin_amdgcn_fmed3f(t[i + j], -448.0f, 448.0f) : t[i + j];
      int w = __builtin_amdgcn_cvt_pk_fp8_f32(c[0], c[1], 0, false);
      out[i / 4] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c[2], c[3], w, true);
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 8) {   // the conversion saturates
      uint32_t w = 0;
      w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, t[i], t[i + 1], 1.0f, 0);
      w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, t[i + 2], t[i + 3], 1.0f, 1);
      w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, t[i + 4], t[i + 5], 1.0f, 2);
      out[i / 8] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, t[i + 6], t[i + 7], 1.0f, 3);
    }
  }
}

// Four scaled values as four bytes (E4M3) or the low two (E2M1).
template <int FMT, bool SAT>
__device__ __forceinline__ uint32_t mx_encode4(const float* t) {
  if constexpr (FMT == kFp8) {
    uint32_t w;
    mx_encode<FMT, 4, SAT>(t, &w);
    return w;
  } else {
    const uint32_t w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, t[0], t[1], 1.0f, 0);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, t[2], t[3], 1.0f, 1);
  }
}

// Eight elements of a lane as a quarter of a block (lanes 4b .. 4b+3 hold block b,
// all of them active): scale them, write the codes at `codes` (8 or 4 bytes) and,
// from the first lane of the four, the scale byte.
template <int FMT, bool SR>
__device__ __forceinline__ void mx_put8(const float* v, bool ceil, uint64_t base, uint64_t elem, uint8_t* codes,
                                        uint8_t* scale) {
  uint32_t a = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) a = mx_umax(a, mx_absbits(v[i]));
  a = mx_umax(a, (uint32_t)__builtin_amdgcn_mov_dpp((int)a, 0xB1, 0xF, 0xF, true));   // lane ^ 1
  a = mx_umax(a, (uint32_t)__builtin_amdgcn_mov_dpp((int)a, 0x4E, 0xF, 0xF, true));   // lane ^ 2
  const MxScale s = mx_scale<FMT>(a, ceil);
  float t[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) t[i] = v[i] * s.inv;
  if constexpr (SR) {
#pragma unroll
    for (int i = 0; i < 8; i += 4) mx_sr4<FMT>(t + i, mx_random(base, (elem + i) >> 2));
  }
  uint32_t w[2] = {0, 0};
  mx_encode<FMT, 8, !SR>(t, w);
  if (s.bad()) w[0] = w[1] = 0;
  if constexpr (FMT == kFp8) *(A8_G u32x2*)gp(reinterpret_cast<u32x2*>(codes)) = u32x2{w[0], w[1]};
  else *(A8_G uint32_t*)gp(reinterpret_cast<uint32_t*>(codes)) = w[0];
  if ((threadIdx.x & 3) == 0) *gp(scale) = (uint8_t)s.byte;
}

}  // namespace a8
