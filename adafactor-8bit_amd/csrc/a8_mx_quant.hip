// Microscaled quantisation and reading back (the format: a8_mx.cuh).
#include "a8_abi_impl.h"
#include "a8_mx.cuh"

namespace a8 {
namespace {

// Along the rows: a lane takes eight elements (16 bytes of a 16-bit input), four lanes a block, whose
// maximum takes two cross-lane steps.  A workgroup owns 256 consecutive lanes' worth of the padded matrix.
// Bound by memory: 14336 x 4096 fp32 into 4 bits 38 us (6.9 TB/s, part of it from the last-level cache),
// 8192 x 14336 bf16 into 8 bits 67 us (5.4 TB/s).
template <typename T, int FMT, bool SR>
__global__ __launch_bounds__(256) void k_mx_rows(const T* x, int64_t stride, int64_t rows, int64_t cols,
                                                 uint8_t* codes, uint8_t* scales, int ceil, uint64_t seed) {
  const int64_t pitch = mx_pitch(cols);
  const uint32_t per = (uint32_t)(pitch / 8);
  const int64_t c0 = (int64_t)blockIdx.x * 256;
  const int64_t r0 = c0 / per;
  const uint64_t at = (uint64_t)(c0 - r0 * per) + threadIdx.x;
  const int64_t row = r0 + (int64_t)(at / per);
  const int64_t col = (int64_t)(at % per) * 8;
  if (row >= rows) return;   // whole groups of 32 lanes
  const T* p = x + row * stride + col;
  float v[8];
  if (col + 8 <= cols) {
    mx_loadn<8>(p, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = col + i < cols ? mx_f(p[i]) : 0.0f;
  }
  const int64_t e = row * pitch + col;
  mx_put8<FMT, SR>(v, ceil != 0, seed, (uint64_t)e, codes + (FMT == kFp8 ? e : e / 2), scales + e / 32);
}

// Down the columns (the transposed matrix [cols, rows] in blocks along its rows), and along the
// rows from the same reading.  A wave owns 32 rows x 128 columns, lane (q, h) columns 4 q .. 4 q + 3 of
// rows 16 h .. 16 h + 15: eight lanes a block along the rows, two lanes a block down the columns, so both
// maxima take a few cross-lane steps.  Four waves make 128 x 128, CW times that a workgroup 128 x 256 where
// there are tiles enough to fill the CUs evenly; codes and scales are gathered in LDS,
// so that memory gets whole lines (half ones of a column's 4-bit codes), four of a column's scales and
// eight of a row's at a time.  A run of tiles down the same columns goes to one XCD, whose L2 joins the
// parts of lines that are left.  Four waves a SIMD: more registers cost more in waves than they save
// (8192 x 14336 bf16 into 4 bits: 81 us, 4.4 TB/s; three waves 95; stochastic, bound by its arithmetic,
// 139).
template <typename T, int FMT, bool SR, bool ALONG, int CW>
__global__ __launch_bounds__(256 * CW, 4) void k_mx_both(const T* x, int64_t stride, int64_t rows, int64_t cols, uint8_t* codes,
                                                 uint8_t* scales, uint8_t* codes_t, uint8_t* scales_t, int ceil,
                                                 uint64_t seed, uint64_t seed_t, uint32_t down) {
  constexpr int kCol = FMT == kFp8 ? 128 : 64, kPitch = kCol + 16;   // bytes of a column's codes
  __shared__ __align__(16) uint8_t col_codes[128 * CW * kPitch];
  constexpr int kRow = (FMT == kFp8 ? 128 : 64) * CW, kPitchR = kRow + 16;   // bytes of a row's codes
  __shared__ __align__(16) uint8_t row_codes[ALONG ? 128 * kPitchR : 16];
  __shared__ __align__(16) uint8_t col_scales[128 * CW * 4], row_scales[128 * 4 * CW];
  const uint32_t xcd = blockIdx.x & 7, n8 = gridDim.x >> 3, rem = gridDim.x & 7;
  const uint32_t id = xcd * n8 + (xcd < rem ? xcd : rem) + (blockIdx.x >> 3);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int wr = (wave & 3) * 32, wc = (wave >> 2) * 128;   // the wave's place in the tile
  const int q = lane & 31, h = lane >> 5;
  const int64_t tile_row = (int64_t)(id % down) * 128, tile_col = (int64_t)(id / down) * (128 * CW);
  const int64_t row = tile_row + wr + 16 * h, col = tile_col + wc + 4 * q;
  const int64_t pitch = mx_pitch(cols), pitch_t = mx_pitch(rows);
  float v[16][4];
  if (tile_row + wr + 32 <= rows && tile_col + wc + 128 <= cols) {
    const T* p = x + row * stride + col;
#pragma unroll
    for (int i = 0; i < 16; ++i) mx_load4(p + i * stride, v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        v[i][j] = row + i < rows && col + j < cols ? mx_f(x[(row + i) * stride + col + j]) : 0.0f;
  }
  uint32_t down_max[4] = {0, 0, 0, 0};
  uint32_t keep[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    uint32_t a[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      a[j] = mx_absbits(v[i][j]);
      down_max[j] = mx_umax(down_max[j], a[j]);
    }
    if constexpr (ALONG) {
      uint32_t m = mx_umax(mx_umax(a[0], a[1]), mx_umax(a[2], a[3]));
      m = mx_umax(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0xB1, 0xF, 0xF, true));    // lane ^ 1
      m = mx_umax(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0x4E, 0xF, 0xF, true));    // lane ^ 2
      m = mx_umax(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0x141, 0xF, 0xF, true));   // 7 - lane of eight
      const MxScale s = mx_scale<FMT>(m, ceil != 0);
      if ((lane & 7) == (i & 7)) keep[i >> 3] = s.byte;
      float t[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) t[j] = v[i][j] * s.inv;
      if constexpr (SR) mx_sr4<FMT>(t, mx_random(seed, (uint64_t)((row + i) * pitch + col) >> 2));
      const uint32_t w = mx_encode4<FMT, !SR>(t);
      uint8_t* o = row_codes + (wr + 16 * h + i) * kPitchR;
      if constexpr (FMT == kFp8) *reinterpret_cast<uint32_t*>(o + wc + 4 * q) = s.bad() ? 0u : w;
      else *reinterpret_cast<uint16_t*>(o + wc / 2 + 2 * q) = (uint16_t)(s.bad() ? 0u : w);
    }
  }
  if constexpr (ALONG) {
#pragma unroll
    for (int j = 0; j < 2; ++j) row_scales[(wr + 16 * h + 8 * j + (lane & 7)) * 4 * CW + (wc >> 5) + (q >> 3)] = (uint8_t)keep[j];
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t m = mx_umax(down_max[j], (uint32_t)__shfl_xor((int)down_max[j], 32));
    const MxScale s = mx_scale<FMT>(m, ceil != 0);
    float t[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) t[i] = v[i][j] * s.inv;
    if constexpr (SR) {
      const uint64_t word = (uint64_t)((col + j) * pitch_t + row) >> 2;
#pragma unroll
      for (int i = 0; i < 16; i += 4) mx_sr4<FMT>(t + i, mx_random(seed_t, word + i / 4));
    }
    uint32_t w[4];
    mx_encode<FMT, 16, !SR>(t, w);
    const int c = wc + 4 * q + j;
    if constexpr (FMT == kFp8)
      *reinterpret_cast<u32x4*>(col_codes + c * kPitch + wr + 16 * h) = s.bad() ? u32x4{0, 0, 0, 0} : u32x4{w[0], w[1], w[2], w[3]};
    else
      *reinterpret_cast<u32x2*>(col_codes + c * kPitch + (wr + 16 * h) / 2) = s.bad() ? u32x2{0, 0} : u32x2{w[0], w[1]};
    if (h == 0) col_scales[c * 4 + (wr >> 5)] = (uint8_t)s.byte;
  }
  __syncthreads();
  constexpr int kChunks = kCol / 16;   // lanes a column
#pragma unroll
  for (int i = 0; i < kChunks / 2; ++i) {
    const int k = i * 256 * CW + threadIdx.x, c = k / kChunks, at = k % kChunks * 16;
    if (tile_col + c < cols) {
      const int64_t e = (tile_col + c) * pitch_t + tile_row;
      *(A8_G u32x4*)gp(reinterpret_cast<u32x4*>(codes_t + (FMT == kFp8 ? e : e / 2) + at)) =
          *reinterpret_cast<const u32x4*>(col_codes + c * kPitch + at);
    }
  }
  if constexpr (ALONG) {
    constexpr int kParts = kRow / 16;   // lanes a row
#pragma unroll
    for (int i = 0; i < 128 * kParts / (256 * CW); ++i) {
      const int k = i * 256 * CW + threadIdx.x, r = k / kParts, at = k % kParts * 16;
      if (tile_row + r < rows) {
        const int64_t e = (tile_row + r) * pitch + tile_col;
        *(A8_G u32x4*)gp(reinterpret_cast<u32x4*>(codes + (FMT == kFp8 ? e : e / 2) + at)) =
            *reinterpret_cast<const u32x4*>(row_codes + r * kPitchR + at);
      }
    }
  }
  if (threadIdx.x < 128 * CW) {
    const int c = threadIdx.x;
    if (tile_col + c < cols)
      *gp(reinterpret_cast<uint32_t*>(scales_t + (tile_col + c) * (pitch_t / 32) + tile_row / 32)) =
          *reinterpret_cast<const uint32_t*>(col_scales + 4 * c);
  } else if (ALONG && threadIdx.x < 128 * CW + 128) {
    typedef typename std::conditional<CW == 2, u32x2, uint32_t>::type scales_t4;
    const int r = threadIdx.x - 128 * CW;
    if (tile_row + r < rows)
      *(A8_G scales_t4*)gp(reinterpret_cast<scales_t4*>(scales + (tile_row + r) * (pitch / 32) + tile_col / 32)) =
          *reinterpret_cast<const scales_t4*>(row_scales + 4 * CW * r);
  }
}

// Reading back: eight elements a lane.  Bound by memory: 8192 x 14336 from 8 bits to bf16 65 us (5.5 TB/s).
template <typename T, int FMT>
__global__ __launch_bounds__(256) void k_mx_read(T* out, const uint8_t* codes, const uint8_t* scales, int64_t rows,
                                                 int64_t cols) {
  const int64_t pitch = mx_pitch(cols);
  const uint32_t per = (uint32_t)((cols + 7) / 8);
  const int64_t c0 = (int64_t)blockIdx.x * 256;
  const int64_t r0 = c0 / per;
  const uint64_t at = (uint64_t)(c0 - r0 * per) + threadIdx.x;
  const int64_t row = r0 + (int64_t)(at / per), col = (int64_t)(at % per) * 8;
  if (row >= rows) return;
  const int64_t e = row * pitch + col;
  const float s = mx_scale_value(*gp(scales + e / 32));
  float v[8];
  if constexpr (FMT == kFp8) {
    const u32x2 w = *(const A8_G u32x2*)gp(reinterpret_cast<const u32x2*>(codes + e));
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i], false);
      const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i], true);
      v[4 * i] = lo[0], v[4 * i + 1] = lo[1], v[4 * i + 2] = hi[0], v[4 * i + 3] = hi[1];
    }
  } else {
    const uint32_t w = *(const A8_G uint32_t*)gp(reinterpret_cast<const uint32_t*>(codes + e / 2));
    const auto a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 0);
    const auto b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 1);
    const auto c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 2);
    const auto d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 3);
    v[0] = a[0], v[1] = a[1], v[2] = b[0], v[3] = b[1], v[4] = c[0], v[5] = c[1], v[6] = d[0], v[7] = d[1];
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] *= s;
  T* o = out + row * cols + col;
  if (col + 8 <= cols) {
    mx_storen<8>(o, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (col + i < cols) o[i] = mx_to<T>(v[i]);
  }
}

template <typename T, int FMT, bool SR>
int quantize(const T* x, int64_t rows, int64_t cols, int64_t stride, uint8_t* codes, uint8_t* scales, uint8_t* codes_t,
             uint8_t* scales_t, int ceil, uint64_t seed, hipStream_t st) {
  const uint64_t base = seed * 0x9E3779B97F4A7C15ULL, base_t = base + 0xD1B54A32D192ED03ULL;
  if (codes_t) {
    const int64_t down = mx_pitch(rows) / 128;
    auto go = [&](auto along, auto cw) {
      constexpr int CW = decltype(cw)::value;
      const int64_t g = down * (mx_pitch(cols) / (128 * CW));
      if (g > most_groups(256 * CW)) return set_error(A8_ERR_SIZE, "mx_quantize: more tiles than one launch takes");
      k_mx_both<T, FMT, SR, decltype(along)::value, CW><<<(uint32_t)g, 256 * CW, 0, st>>>(
          x, stride, rows, cols, codes, scales, codes_t, scales_t, ceil, base, base_t, (uint32_t)down);
      return check_launch("k_mx_both");
    };
    // 128 x 256 tiles make whole lines of a row's 4-bit codes and pay where memory is the bound and there are
    // tiles enough (14336 x 4096 fp32 into 4 bits: 52.7 us against 57.8); elsewhere smaller ones spread better
    // (5632 x 2048 bf16 into 8 bits: 11.8 us against 13.1, stochastic 21 against 25).
    auto way = [&](auto along) {
      if constexpr (!SR)
        if (down * (mx_pitch(cols) / 256) >= 1024) return go(along, std::integral_constant<int, 2>{});
      return go(along, std::integral_constant<int, 1>{});
    };
    return codes ? way(std::true_type{}) : way(std::false_type{});
  }
  const int64_t pitch = mx_pitch(cols);
  return in_runs(rows, most_groups(256) * 256 / (pitch / 8), [&](int64_t first, int64_t count) {
    const int64_t e = first * pitch;
    k_mx_rows<T, FMT, SR><<<(uint32_t)((count * (pitch / 8) + 255) / 256), 256, 0, st>>>(
        x + first * stride, stride, count, cols, codes + (FMT == kFp8 ? e : e / 2), scales + e / 32, ceil,
        base + (uint64_t)e / 4);
    return check_launch("k_mx_rows");
  });
}

template <typename T>
int quantize_t(int fmt, int sr, const void* x, int64_t rows, int64_t cols, int64_t stride, uint8_t* codes,
               uint8_t* scales, uint8_t* codes_t, uint8_t* scales_t, int ceil, uint64_t seed, hipStream_t st) {
  const T* p = static_cast<const T*>(x);
  if (fmt == kFp4)
    return sr ? quantize<T, kFp4, true>(p, rows, cols, stride, codes, scales, codes_t, scales_t, ceil, seed, st)
              : quantize<T, kFp4, false>(p, rows, cols, stride, codes, scales, codes_t, scales_t, ceil, seed, st);
  return sr ? quantize<T, kFp8, true>(p, rows, cols, stride, codes, scales, codes_t, scales_t, ceil, seed, st)
            : quantize<T, kFp8, false>(p, rows, cols, stride, codes, scales, codes_t, scales_t, ceil, seed, st);
}

constexpr int64_t kMaxSide = (int64_t)1 << 31;

bool fits(int64_t rows, int64_t cols) {
  return rows < kMaxSide && cols < kMaxSide && mx_pitch(rows) / 128 * (mx_pitch(cols) / 16) < kMaxSide;
}

}  // namespace
}  // namespace a8

using namespace a8;

extern "C" int64_t a8_mx_pitch(int64_t cols) { return cols < 0 ? -1 : mx_pitch(cols); }

extern "C" int a8_mx_quantize(int dtype, int fmt, int scale_rule, int stochastic, const void* x, int64_t rows,
                              int64_t cols, int64_t row_stride, uint8_t* codes, uint8_t* scales, uint8_t* codes_t,
                              uint8_t* scales_t, uint64_t seed, void* stream) {
  if (dtype != A8_F32 && dtype != A8_BF16 && dtype != A8_F16)
    return set_error(A8_ERR_DTYPE, "mx_quantize: dtype must be fp32, bf16 or fp16");
  if (fmt != A8_MXFP4 && fmt != A8_MXFP8) return set_error(A8_ERR_ARG, "mx_quantize: unknown format");
  if (scale_rule != 0 && scale_rule != 1) return set_error(A8_ERR_ARG, "mx_quantize: unknown scale rule");
  if (rows < 0 || cols < 0 || !fits(rows, cols)) return set_error(A8_ERR_SIZE, "mx_quantize: rows or cols out of range");
  if (rows == 0 || cols == 0) return A8_OK;
  if (row_stride < cols && rows > 1) return set_error(A8_ERR_ARG, "mx_quantize: row_stride below cols");
  if (!x || (!codes && !codes_t) || (codes && !scales) || (codes_t && !scales_t))
    return set_error(A8_ERR_ARG, "mx_quantize: null pointer");
  if ((codes && !aligned16(codes)) || (codes_t && !aligned16(codes_t)) || (reinterpret_cast<uintptr_t>(scales) & 7) ||
      (reinterpret_cast<uintptr_t>(scales_t) & 7))
    return set_error(A8_ERR_ALIGN, "mx_quantize: codes must be 16-byte aligned, scales 8-byte");
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == A8_F32)
    return quantize_t<float>(fmt, stochastic, x, rows, cols, row_stride, codes, scales, codes_t, scales_t, scale_rule, seed, st);
  if (dtype == A8_BF16)
    return quantize_t<__hip_bfloat16>(fmt, stochastic, x, rows, cols, row_stride, codes, scales, codes_t, scales_t, scale_rule, seed, st);
  return quantize_t<__half>(fmt, stochastic, x, rows, cols, row_stride, codes, scales, codes_t, scales_t, scale_rule, seed, st);
}

extern "C" int a8_mx_dequantize(int dtype, int fmt, void* out, const uint8_t* codes, const uint8_t* scales,
                                int64_t rows, int64_t cols, void* stream) {
  if (dtype != A8_F32 && dtype != A8_BF16 && dtype != A8_F16)
    return set_error(A8_ERR_DTYPE, "mx_dequantize: dtype must be fp32, bf16 or fp16");
  if (fmt != A8_MXFP4 && fmt != A8_MXFP8) return set_error(A8_ERR_ARG, "mx_dequantize: unknown format");
  if (rows < 0 || cols < 0 || !fits(rows, cols)) return set_error(A8_ERR_SIZE, "mx_dequantize: rows or cols out of range");
  if (rows == 0 || cols == 0) return A8_OK;
  if (!out || !codes || !scales) return set_error(A8_ERR_ARG, "mx_dequantize: null pointer");
  if (!aligned16(codes)) return set_error(A8_ERR_ALIGN, "mx_dequantize: codes must be 16-byte aligned");
  hipStream_t st = static_cast<hipStream_t>(stream);
  auto go = [&](auto* o) {
    typedef std::remove_pointer_t<decltype(o)> T;
    const int64_t pitch = mx_pitch(cols), per = (cols + 7) / 8;
    return in_runs(rows, most_groups(256) * 256 / per, [&](int64_t first, int64_t count) {
      const uint32_t g = (uint32_t)((count * per + 255) / 256);
      const int64_t e = first * pitch;
      if (fmt == A8_MXFP4)
        k_mx_read<T, kFp4><<<g, 256, 0, st>>>(o + first * cols, codes + e / 2, scales + e / 32, count, cols);
      else
        k_mx_read<T, kFp8><<<g, 256, 0, st>>>(o + first * cols, codes + e, scales + e / 32, count, cols);
      return check_launch("k_mx_read");
    });
  };
  if (dtype == A8_F32) return go(static_cast<float*>(out));
  if (dtype == A8_BF16) return go(static_cast<__hip_bfloat16*>(out));
  return go(static_cast<__half*>(out));
}
