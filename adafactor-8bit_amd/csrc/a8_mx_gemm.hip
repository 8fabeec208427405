// Products of microscaled matrices: C[m, n] = sum over blocks of 2^(ea + eb) * sum a b,
// a [m, k] and b [n, k] as MX tensors (a8_mx.cuh), fp32 accumulation in the matrix cores.
#include "a8_abi_impl.h"
#include "a8_mx.cuh"
#include "a8_mx_lds.h"
#include "a8_once.h"

namespace a8 {
namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

// The matrix instruction takes 64 elements (two blocks) of 32 rows of either side.  Lane (r, h)
// holds of row r: in 4 bits the 32 elements of block h, in 8 bits elements 16 h .. 16 h + 15 of both
// blocks; its scale byte is block h's.  The result's lane (r, h) holds row r of the second operand and
// rows 8 q + 4 h + (0..3) of the first.
//
// ---------------------------------------------------------------- few rows
// a of at most 32 rows: 32 rows of b a workgroup, whose W waves share the contraction out among
// them, operands straight from memory (b is read once: nothing to keep in LDS), and add up through LDS
// in a fixed order.  Step s of 256 elements takes blocks 2 s and 2 s + 1, so that a row's two lanes
// read 32 adjacent bytes.
template <int FMT>
__device__ __forceinline__ i32x8 mx_operand(const uint8_t* p, int h, int s) {
  i32x8 o = {};
  if constexpr (FMT == kFp4) {
    const i32x4 a = *(const A8_G i32x4*)gp(reinterpret_cast<const i32x4*>(p + s * 32 + h * 16));
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = a[i];
  } else {
    const i32x4 a = *(const A8_G i32x4*)gp(reinterpret_cast<const i32x4*>(p + s * 64 + h * 16));
    const i32x4 b = *(const A8_G i32x4*)gp(reinterpret_cast<const i32x4*>(p + s * 64 + 32 + h * 16));
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = a[i], o[4 + i] = b[i];
  }
  return o;
}

// Operands and scales of one row for 256 elements (step s: byte 2 (s % 2) of scale word s / 2).
template <int FMT>
struct MxRow {
  i32x8 v[4];
  int x[2];
  __device__ __forceinline__ void load(const uint8_t* codes, const uint8_t* scales, int64_t kb, int h) {
    const u32x2 w = *(const A8_G u32x2*)gp(reinterpret_cast<const u32x2*>(scales + kb / 32));
    const uint8_t* p = codes + (FMT == kFp4 ? kb / 2 : kb);
#pragma unroll
    for (int s = 0; s < 4; ++s) v[s] = mx_operand<FMT>(p, h, s);
    x[0] = (int)(w[0] >> (8 * h)), x[1] = (int)(w[1] >> (8 * h));
  }
};

template <int FA, int FB, int W, bool STREAM, typename T>
__global__ __launch_bounds__(64 * W, 2) void k_mx_few(const uint8_t* a, const uint8_t* sa, const uint8_t* b,
                                                   const uint8_t* sb, T* c, int64_t m, int64_t n, int64_t k) {
  constexpr int TA = FA == kFp4 ? 4 : 0, TB = FB == kFp4 ? 4 : 0;
  constexpr int kPad = 36;   // floats a row of the partial sums: 16-byte writes of 8 rows meet all banks
  __shared__ __align__(16) float part[W * 32 * kPad];
  const int64_t pitch = mx_pitch(k), ps = pitch / 32;
  const int64_t pa = FA == kFp4 ? pitch / 2 : pitch, pb = FB == kFp4 ? pitch / 2 : pitch;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int r = lane & 31, h = lane >> 5;
  const int64_t n0 = (int64_t)blockIdx.x * 32;
  const int64_t rb = n0 + r < n ? n0 + r : n - 1;
  const uint8_t *qb = b + rb * pb, *xb = sb + rb * ps;
  const int64_t ra = r < m ? r : m - 1;
  const uint8_t *qa = a + ra * pa, *xa = sa + ra * ps;
  f32x16 acc = {};
  const int64_t blocks = pitch / 256;
  const int64_t i0 = blocks * wave / W, i1 = blocks * (wave + 1) / W;
  struct Blocks {   // 256 elements of both sides
    MxRow<FB> b;
    MxRow<FA> a;
  };
  auto load = [&](Blocks& x, int64_t i) {
    x.b.load(qb, xb, i * 256, h);
    x.a.load(qa, xa, i * 256, h);
  };
  auto multiply = [&](const Blocks& x) {
    const MxRow<FB>& y = x.b;
    const MxRow<FA>& z = x.a;
    acc = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(y.v[0], z.v[0], acc, TB, TA, 0, y.x[0], 0, z.x[0]);
    acc = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(y.v[1], z.v[1], acc, TB, TA, 2, y.x[0], 2, z.x[0]);
    acc = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(y.v[2], z.v[2], acc, TB, TA, 0, y.x[1], 0, z.x[1]);
    acc = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(y.v[3], z.v[3], acc, TB, TA, 2, y.x[1], 2, z.x[1]);
  };
  if constexpr (STREAM) {   // the next block on its way during the products of one
    if (i0 < i1) {
      Blocks x, y;
      load(x, i0);
      for (int64_t i = i0;;) {
        if (i + 1 < i1) load(y, i + 1);
        multiply(x);
        if (++i >= i1) break;
        if (i + 1 < i1) load(x, i + 1);
        multiply(y);
        if (++i >= i1) break;
      }
    }
  } else {                  // four blocks asked for before the first product waits
    auto some = [&](int64_t i, auto count) {
      constexpr int N = decltype(count)::value;
      Blocks x[N];
#pragma unroll
      for (int u = 0; u < N; ++u) load(x[u], i + u);
#pragma unroll
      for (int u = 0; u < N; ++u) multiply(x[u]);
    };
    int64_t i = i0;
    for (; i + 4 <= i1; i += 4) some(i, std::integral_constant<int, 4>{});
    if (i + 2 <= i1) {
      some(i, std::integral_constant<int, 2>{});
      i += 2;
    }
    if (i < i1) some(i, std::integral_constant<int, 1>{});
  }
  float* p = part + (wave * 32 + r) * kPad + 4 * h;
#pragma unroll
  for (int e = 0; e < 16; e += 4)
    *reinterpret_cast<f32x4*>(p + 2 * e) = f32x4{acc[e], acc[e + 1], acc[e + 2], acc[e + 3]};
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 16 / W; ++i) {
    const int j = threadIdx.x + i * 64 * W;
    const int64_t row = j / 32, col = n0 + j % 32;
    float t = 0.0f;
#pragma unroll
    for (int w = 0; w < W; ++w) t += part[(w * 32 + j / 32) * kPad + j % 32];
    if (row < m && col < n) c[row * n + col] = mx_to<T>(t);
  }
}

// ---------------------------------------------------------------- tiles through LDS
// Raw buffer resource over `bytes` from p: accesses beyond them read 0 (per 4 bytes), so tiles
// that hang over the last row need no masks.
__device__ __forceinline__ i32x4 mx_buffer(const uint8_t* p, int64_t bytes) {
  const uint64_t a = (uint64_t)p;
  const uint32_t n = bytes > 0xFFFFFFFFll ? 0xFFFFFFFFu : (uint32_t)(bytes < 0 ? 0 : bytes);
  i32x4 r;
  r[0] = __builtin_amdgcn_readfirstlane((int)(uint32_t)a);
  r[1] = __builtin_amdgcn_readfirstlane((int)((uint32_t)(a >> 32) & 0xFFFFu));
  r[2] = __builtin_amdgcn_readfirstlane((int)n);
  r[3] = 0x00020000;
  return r;
}

// 16 bytes a lane from buffer + off to LDS at lds + 16 * lane.  No register is written but m0, and
// the caller waits (vmcnt) before it reads the LDS.  The compiler sets m0 before a use of its own and may join
// such settings; m0 is named so that it joins none across the block (the warning: nothing saves m0 here).
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void mx_to_lds(i32x4 buf, uint32_t off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
               :
               : "s"(lds), "v"(off), "s"(buf)
               : "m0", "memory");
}
#pragma clang diagnostic pop

template <int N>
__device__ __forceinline__ void mx_wait_barrier() {   // own loads to LDS but the last N, own LDS reads; then everyone's
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" : : "n"(N) : "memory");
}

typedef __attribute__((address_space(3))) uint8_t lds_u8;
constexpr uint32_t kBeyond = 0x80000000u;   // an offset past every buffer (the caller keeps them below 2^31 bytes)

// One side of a product in LDS: ROWS rows in NB places of KS elements, 64 or 128 bytes a row in chunks of
// 16.  Chunk c of row r lies at place c ^ (r / 4 % 4) (64 bytes) or c ^ (r / 2 % 8) (128): 16 rows of one
// chunk then fall on all 64 banks.
template <int FMT, int ROWS, int KS, int NB>
struct MxSide {
  static constexpr int kRow = FMT == kFp4 ? KS / 2 : KS;
  static_assert(kRow == 64 || kRow == 128, "");
  static constexpr int kBytes = ROWS * kRow;              // a place
  static constexpr int kLoads = ROWS / 4 * kRow / 1024;   // 1 KB instructions a wave and stage
  static constexpr int kStep = 1024 / kRow;               // rows an instruction
  i32x4 buf;
  uint32_t off[2];
  uint32_t step;
  __device__ __forceinline__ void init(const uint8_t* p, int64_t row0, int64_t rows, int64_t pitch, int wave, int lane) {
    buf = mx_buffer(p + row0 * pitch, (rows - row0 < ROWS ? rows - row0 : ROWS) * pitch);
    step = (uint32_t)(kStep * pitch);
    const int r = kRow == 64 ? lane >> 2 : lane >> 3;
    const uint32_t base = (uint32_t)(wave * (ROWS / 4) + r) * (uint32_t)pitch;
    if constexpr (kRow == 64) {
      off[0] = off[1] = base + (uint32_t)(((lane & 3) ^ (r >> 2)) * 16);
    } else {   // rows 8 t + r: (row / 2) % 8 = 4 (t % 2) + r / 2
      off[0] = base + (uint32_t)(((lane & 7) ^ (r >> 1)) * 16);
      off[1] = base + (uint32_t)(((lane & 7) ^ (r >> 1) ^ 4) * 16);
    }
  }
  // The t-th load of stage i of the `stages` from `first` on; past the end it reads zeros, from nowhere.
  __device__ __forceinline__ void load(uint32_t lds, int i, int first, int stages, int wave, int t) const {
    const uint32_t at = i < stages ? (uint32_t)(first + i) * kRow : kBeyond;
    mx_to_lds(buf, off[t & 1] + at + (uint32_t)t * step, lds + (uint32_t)(i % NB) * kBytes + wave * (kBytes / 4) + t * 1024);
  }
  // The operand of row `row` (row % 32 = r) in step s of stage i.  A stage has S = KS / 64 steps; step s takes
  // blocks s and S + s, so that a lane's scale bytes are neighbours.
  __device__ __forceinline__ static i32x8 frag(const lds_u8* side, int i, int row, int r, int h, int s) {
    typedef const __attribute__((address_space(3))) i32x4 lds_i32x4;
    constexpr int S = KS / 64;
    const int x = kRow == 64 ? r >> 2 & 3 : r >> 1 & 7;
    const lds_u8* p = side + (uint32_t)(i % NB) * kBytes + row * kRow;
    i32x8 o = {};
    if constexpr (FMT == kFp4) {
      const i32x4 a = *(lds_i32x4*)(p + (((S * h + s) ^ x) * 16));
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] = a[j];
    } else {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const i32x4 a = *(lds_i32x4*)(p + (((2 * (S * j + s) + h) ^ x) * 16));
#pragma unroll
        for (int l = 0; l < 4; ++l) o[4 * j + l] = a[l];
      }
    }
    return o;
  }
};

// How a tile is fed.  Memory gives lines of 128 bytes whether half of one is wanted or not, so two 4-bit
// sides go in stages of 256 elements (8192 x 14336 x 4096: 252 us against 310 in 128); beside 8 bits a 4-bit
// side's half lines cost 2 % and stay.  Large tiles have two stages in LDS; small ones, which wait for memory
// rather than for its rate, what fits 64 KB, two workgroups a CU, or a quarter of a CU's LDS.
template <int FA, int FB, int MI, int NI, int KG>
struct MxStage {
  static constexpr int kElems = FA == kFp4 && FB == kFp4 ? 256 : 128;
  static constexpr int kStage = 64 * kElems * ((FA == kFp4 ? MI : 2 * MI) + (FB == kFp4 ? NI : 2 * NI)) / 2;
  static constexpr int kRing = KG > 1 ? (FA != FB ? 3 : 2) : MI * NI == 1 ? 65536 / kStage : 2;
  typedef MxSide<FA, 64 * MI, kElems, kRing> A;
  typedef MxSide<FB, 64 * NI, kElems, kRing> B;
  static constexpr int kSpanK = KG > 1 ? 512 : 1024;      // elements whose scales are asked for together
  static constexpr int kScales = kSpanK / 32 * 64 * (MI + NI);
  // Groups of stages whose scales are on their way: a wait leaves the last kRing - 2 stages' loads open,
  // so a group is asked for at least kRing - 1 stages before its first use.
  static constexpr int kGroup = kSpanK / kElems;
  static constexpr int kAhead = (kRing - 1 + kGroup - 1) / kGroup;
  static constexpr int kCodes = kRing * (A::kBytes + B::kBytes);
  static constexpr int kPart = kCodes + (kAhead + 1) * kScales;   // a group of waves'
  static constexpr int kLds = KG * kPart;
  static_assert(kLds <= 160 * 1024, "");
};

// Bound: on operands as quantisation gives them the matrix cores alone, fed from registers, reach 5.7 - 6.7
// PFLOP/s in 4 bits and 3.9 - 4.2 in 8 (the card lowers its clock; 9.6 and 5.0 on zeros).  8192 x 4096 x 14336 takes
// 203 us in 4 bits (4.7 PFLOP/s, cores busy 63 % of the cycles), 314 us in 8 by 4 bits (3.1, 75 %), 330 us in 8 bits
// (2.9, 73 %).  Left out by themselves, its operand reads (LDS busy 26 - 29 % of the cycles, a quarter of that on
// conflicts) and its L2 misses (16 - 18 % of requests) cost nothing, the loads to LDS about a sixth.  Outputs leave when a tile is done, unhidden:
// 8192 x 14336 x 4096, with 3.5 times as many, takes 234, 346 and 361 us.
//
// 64 MI x 64 NI outputs a workgroup: four waves of 32 MI x 32 NI, stages of KS elements in a
// ring of NB.  KG such groups of waves share the contraction out among them, each in its own part of
// LDS, and add up at the end in their order.
template <int FA, int FB, int MI, int NI, int KG, typename T>
__global__ __launch_bounds__(256 * KG, MI * NI == 16 || KG > 1 ? 1 : 2) void k_mx_tile(
    const uint8_t* a, const uint8_t* sa, const uint8_t* b, const uint8_t* sb, T* c, int64_t m, int64_t n, int64_t k) {
  constexpr int TA = FA == kFp4 ? 4 : 0, TB = FB == kFp4 ? 4 : 0;
  typedef MxStage<FA, FB, MI, NI, KG> Stage;
  constexpr int BM = 64 * MI, BN = 64 * NI, KS = Stage::kElems, NB = Stage::kRing, S = KS / 64;
  constexpr int GS = Stage::kGroup, kAhead = Stage::kAhead;   // scales come 16 bytes a row, for GS stages
  typedef typename Stage::A SA;
  typedef typename Stage::B SB;
  constexpr int kScale = Stage::kScales, kLoads = SA::kLoads + SB::kLoads;
  extern __shared__ __align__(1024) uint8_t smem[];
  const int group = KG > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 8) : 0;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6 & 3), lane = threadIdx.x & 63;
  lds_u8* lds = (lds_u8*)smem + group * Stage::kPart;
  const uint32_t lds0 = (uint32_t)(uintptr_t)lds;

  // A group's stages are [first, first + stages), whole groups of scales; every group turns `turns` times.
  const int64_t pitch = mx_pitch(k);
  const int total = (int)(pitch / KS);
  const int turns = KG > 1 ? ((total + GS - 1) / GS + KG - 1) / KG * GS : total;
  const int first = group * turns;
  const int stages = total - first < turns ? (total > first ? total - first : 0) : turns;
  const int r = lane & 31, h = lane >> 5;

  // workgroups go to the eight XCDs in turn: each takes a run of tiles that share rows in its L2
  const uint32_t tm = (uint32_t)((m + BM - 1) / BM), tn = (uint32_t)((n + BN - 1) / BN), tiles = tm * tn;
  const uint32_t x = blockIdx.x & 7, q = tiles >> 3, rem = tiles & 7;
  const uint32_t id = x * q + (x < rem ? x : rem) + (blockIdx.x >> 3);
  constexpr uint32_t G = 8;
  const uint32_t grp = id / (G * tn), in = id - grp * G * tn;
  const uint32_t gm = tm - grp * G < G ? tm - grp * G : G;
  const int64_t m0 = (int64_t)(grp * G + in % gm) * BM, n0 = (int64_t)(in / gm) * BN;

  SA la;
  SB lb;
  la.init(a, m0, m, FA == kFp4 ? pitch / 2 : pitch, wave, lane);
  lb.init(b, n0, n, FB == kFp4 ? pitch / 2 : pitch, wave, lane);
  const int64_t ps = pitch / 32;
  const i32x4 qa = mx_buffer(sa + m0 * ps, (m - m0) * ps), qb = mx_buffer(sb + n0 * ps, (n - n0) * ps);
  auto load_one = [&](int i, int t) {
    if (t < SA::kLoads) la.load(lds0, i, first, stages, wave, t);
    else lb.load(lds0 + NB * SA::kBytes, i, first, stages, wave, t - SA::kLoads);
  };
  // A row's scales of 512 elements are 16 bytes, one lane's; those of 1024 go as two halves of 32 rows each
  // an instruction, so that the second finds the line that the first brought.
  constexpr int kHalves = Stage::kSpanK / 512, kRowsIn = 64 / kHalves;
  auto load_scales = [&](int g) {
    const uint32_t at = lds0 + Stage::kCodes + (uint32_t)(g % (kAhead + 1)) * kScale;
    const uint32_t from = (uint32_t)((first / GS + g) * kHalves + lane / kRowsIn) * 16;
    constexpr int kA = BM / kRowsIn, kAll = (BM + BN) / kRowsIn;
#pragma unroll
    for (int t = 0; t < (kAll + 3) / 4; ++t) {
      const int j = 4 * t + wave;
      if (j < kA) mx_to_lds(qa, (uint32_t)(kRowsIn * j + lane % kRowsIn) * (uint32_t)ps + from, at + j * 1024);
      else if (j < kAll) mx_to_lds(qb, (uint32_t)(kRowsIn * (j - kA) + lane % kRowsIn) * (uint32_t)ps + from, at + j * 1024);
    }
  };
  const int wm = (wave & 1) * 32 * MI, wn = (wave >> 1) * 32 * NI;
  typedef typename std::conditional<S == 4, int, uint16_t>::type scales_t;   // a lane's scales of a stage
  typedef const __attribute__((address_space(3))) scales_t lds_scales;
  i32x8 fa[2][MI], fb[2][NI];
  int xa[MI], xb[NI], ya[MI], yb[NI];
  // the j-th operand of step s of stage i, then the scales of its rows in the same order
  auto read_one = [&](int i, int s, int j) {
    if (j < MI) fa[s & 1][j] = SA::frag(lds, i, wm + 32 * j + r, r, h, s);
    else fb[s & 1][j - MI] = SB::frag(lds + NB * SA::kBytes, i, wn + 32 * (j - MI) + r, r, h, s);
  };
  auto read_scale = [&](int i, int j) {
    const int in = i % GS * KS / 32;   // the stage's first byte of a row's
    const lds_u8* p = lds + Stage::kCodes + (uint32_t)(i / GS % (kAhead + 1)) * kScale + in / 16 * 512 + in % 16 + h * S;
    const int row = j < MI ? wm + 32 * j : BM + wn + 32 * (j - MI);
    const int v = *(lds_scales*)(p + row * 16 * kHalves + r * 16);
    if (j < MI) ya[j] = v;
    else yb[j - MI] = v;
  };
  auto take_scales = [&] {
#pragma unroll
    for (int f = 0; f < MI; ++f) xa[f] = ya[f];
#pragma unroll
    for (int f = 0; f < NI; ++f) xb[f] = yb[f];
  };

  f32x16 acc[MI][NI];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NI; ++j) acc[i][j] = f32x16{};

  // A stage is S runs of products, one for each step.  The place of stage i is free after the wait
  // before its last run; the loads of stage i + NB are issued from there on, a few at a time over
  // kSpan products: a run's time alone is too short for them, and a wave that cannot issue a load
  // issues no products either.
  constexpr int kMul = MI * NI, kOps = MI + NI;
  constexpr int kSpan = S == 4 ? 3 * kMul : NB == 2 ? 3 * kMul / 2 : 2 * kMul;
  constexpr int kFirst = kLoads * kMul / kSpan;   // loads in the last run; the others follow in the next stage
#pragma unroll
  for (int g = 0; g < kAhead; ++g) load_scales(g);
#pragma unroll
  for (int i = 0; i < NB; ++i)
#pragma unroll
    for (int t = 0; t < (i < NB - 1 ? kLoads : kFirst); ++t) load_one(i, t);
  mx_wait_barrier<(NB - 2) * kLoads + kFirst>();
#pragma unroll
  for (int j = 0; j < kOps; ++j) read_one(0, 0, j);
#pragma unroll
  for (int j = 0; j < kOps; ++j) read_scale(0, j);
  take_scales();
  auto multiply = [&](auto step, int t) {
    constexpr int s = decltype(step)::value;
    const int f = t / NI, g = t % NI;
    acc[f][g] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(fb[s & 1][g], fa[s & 1][f], acc[f][g], TB, TA, s, xb[g], s, xa[f]);
  };
  // a step before the last: its products, the next step's operands from the same stage, loads; the order
  // is kept as written
  auto run = [&](auto step, int i) {
#pragma unroll
    for (int t = 0; t < kMul; ++t) {
#pragma unroll
      for (int j = t * 2 * kOps / kMul; j < kOps && j < (t + 1) * 2 * kOps / kMul; ++j) read_one(i, step + 1, j);
      const int q = (step + 1) * kMul + t;
#pragma unroll
      for (int j = q * kLoads / kSpan; j < kLoads && j < (q + 1) * kLoads / kSpan; ++j) load_one(i - 1 + NB, j);
      multiply(step, t);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  for (int i = 0; i < turns; ++i) {
    if (KG > 1 && i >= stages) {   // the other groups' stages go on
      mx_wait_barrier<0>();
      continue;
    }
    __builtin_amdgcn_sched_barrier(0);
    run(std::integral_constant<int, 0>{}, i);
    if constexpr (S == 4) {
      run(std::integral_constant<int, 1>{}, i);
      run(std::integral_constant<int, 2>{}, i);
    }
    // stage i + 1 has arrived and everyone has read stage i: its place takes stage i + NB
    mx_wait_barrier<(NB - 2) * kLoads>();
    if (i % GS == 0 && i + kAhead * GS < stages) load_scales(i / GS + kAhead);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int t = 0; t < kMul; ++t) {
      // past the last stage the reads find whatever lies there, unused
#pragma unroll
      for (int j = t * 4 * kOps / kMul; j < 2 * kOps && j < (t + 1) * 4 * kOps / kMul; ++j) {
        if (j < kOps) read_scale(i + 1, j);
        else read_one(i + 1, 0, j - kOps);
      }
#pragma unroll
      for (int j = t * kLoads / kSpan; j < (t + 1) * kLoads / kSpan; ++j) load_one(i + NB, j);
      multiply(std::integral_constant<int, S - 1>{}, t);
      __builtin_amdgcn_sched_barrier(0);
    }
    take_scales();
  }

  // A lane (r, h) holds of a 32 x 32 tile row r, columns 8 q + 4 h + (0..3).  Through LDS (a part of
  // it for each wave) 32 rows become runs of 16 bytes a lane, whole rows of the wave's columns.
  mx_wait_barrier<0>();
  typedef MxEnd<NI, KG, (int)sizeof(T)> End;
  static_assert(End::kBytes <= Stage::kLds, "");
  if constexpr (KG > 1) {
    static_assert(MI == 1 && NI == 1, "");
    typedef __attribute__((address_space(3))) f32x4 lds_f32x4;
    lds_u8* sums = (lds_u8*)smem + lane * 16;   // of a wave: a quarter of its sums for each lane, then the next
    if (group)
#pragma unroll
      for (int e = 0; e < 16; e += 4)
        *(lds_f32x4*)(sums + End::sums(group, wave) + e * 256) =
            f32x4{acc[0][0][e], acc[0][0][e + 1], acc[0][0][e + 2], acc[0][0][e + 3]};
    mx_wait_barrier<0>();
    if (group) return;
#pragma unroll
    for (int g = 1; g < KG; ++g)
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        const f32x4 t = *(lds_f32x4*)(sums + End::sums(g, wave) + e * 256);
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[0][0][e + j] += t[j];
      }
  }
  constexpr int kCols = 32 * NI, kOut = End::kRow;
  constexpr int V = 16 / (int)sizeof(T), kLanes = kCols / V;   // elements a lane, lanes a row
  lds_u8* mine = lds + End::staged(wave);   // group 0's part of the LDS starts where all of it does
#pragma unroll
  for (int f = 0; f < MI; ++f) {
#pragma unroll
    for (int g = 0; g < NI; ++g)
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        lds_u8* p = mine + r * kOut + (32 * g + 2 * e + 4 * h) * (int)sizeof(T);
        if constexpr (sizeof(T) == 4)
          *(__attribute__((address_space(3))) f32x4*)p = f32x4{acc[f][g][e], acc[f][g][e + 1], acc[f][g][e + 2], acc[f][g][e + 3]};
        else
          *(__attribute__((address_space(3))) u32x2*)p =
              u32x2{mx_pack2<T>(acc[f][g][e], acc[f][g][e + 1]), mx_pack2<T>(acc[f][g][e + 2], acc[f][g][e + 3])};
      }
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int t = 0; t < 32 * kLanes / 64; ++t) {
      const int rr = t * (64 / kLanes) + lane / kLanes, cc = lane % kLanes * V;
      const u32x4 w = *(__attribute__((address_space(3))) u32x4*)(mine + rr * kOut + cc * (int)sizeof(T));
      const int64_t row = m0 + wm + 32 * f + rr, col = n0 + wn + cc;
      if (row < m && col + V <= n) {
        A8_G u32x4_a2* o = (A8_G u32x4_a2*)gp(reinterpret_cast<u32x4*>(c + row * n + col));
        // large outputs pass the L2 by, which holds the operands (8192 x 14336 x 4096 in 8 bits: 361 us, 374 else)
        if constexpr (MI * NI == 16) __builtin_nontemporal_store(w, o);
        else *o = w;
      } else if (row < m) {
#pragma unroll
        for (int j = 0; j < V; ++j)
          if (col + j < n) {
            if constexpr (sizeof(T) == 4) *gp(reinterpret_cast<uint32_t*>(c + row * n + col + j)) = w[j];
            else *gp(reinterpret_cast<uint16_t*>(c + row * n + col + j)) = (uint16_t)(w[j / 2] >> (16 * (j & 1)));
          }
      }
    }
    __builtin_amdgcn_wave_barrier();
  }
}

template <typename T>
__global__ __launch_bounds__(256) void k_mx_zero(T* c, int64_t n) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i < n) c[i] = mx_to<T>(0.0f);
}

template <int FA, int FB, int MI, int NI, int KG, typename T>
int tiles(const uint8_t* a, const uint8_t* sa, const uint8_t* b, const uint8_t* sb, T* c, int64_t m, int64_t n,
          int64_t k, hipStream_t st) {
  constexpr int lds = MxStage<FA, FB, MI, NI, KG>::kLds;
  static OncePerDevice once;
  int device = 0;
  if (hipGetDevice(&device) != hipSuccess) return set_error(A8_ERR_HIP, "mx_matmul: no current device");
  const int e = once(device, [] {
    return (int)hipFuncSetAttribute(reinterpret_cast<const void*>(&k_mx_tile<FA, FB, MI, NI, KG, T>),
                                    hipFuncAttributeMaxDynamicSharedMemorySize, MxStage<FA, FB, MI, NI, KG>::kLds);
  });
  if (e != 0) return set_error(A8_ERR_HIP, "mx_matmul: no LDS for the tile kernel");
  const int64_t t = ((m + 64 * MI - 1) / (64 * MI)) * ((n + 64 * NI - 1) / (64 * NI));
  if (t > most_groups(256 * KG)) return set_error(A8_ERR_SIZE, "mx_matmul: more tiles than one launch takes");
  k_mx_tile<FA, FB, MI, NI, KG, T><<<(uint32_t)t, 256 * KG, lds, st>>>(a, sa, b, sb, c, m, n, k);
  return check_launch("k_mx_tile");
}

template <int FA, int FB, typename T>
int few(const uint8_t* a, const uint8_t* sa, const uint8_t* b, const uint8_t* sb, T* c, int64_t m, int64_t n,
        int64_t k, hipStream_t st) {
  const int64_t g = (n + 31) / 32;
  if (g > most_groups(256)) return set_error(A8_ERR_SIZE, "mx_matmul: more rows of b than one launch takes");
  // Fewer tiles than CUs take eight waves each.  Where every CU has several in turn memory's rate is the
  // bound, and a steady stream reads faster than bursts (1 x 128256 x 4096, 8 by 4 bits: 55 us against 65;
  // 1 x 14336 x 4096 the other way, 8.6 against 8.0).
  if (g > 1024) k_mx_few<FA, FB, 4, true, T><<<(uint32_t)g, 256, 0, st>>>(a, sa, b, sb, c, m, n, k);
  else if (g >= 256) k_mx_few<FA, FB, 4, false, T><<<(uint32_t)g, 256, 0, st>>>(a, sa, b, sb, c, m, n, k);
  else k_mx_few<FA, FB, 8, false, T><<<(uint32_t)g, 512, 0, st>>>(a, sa, b, sb, c, m, n, k);
  return check_launch("k_mx_few");
}

template <int FA, int FB, typename T>
int matmul(const uint8_t* a, const uint8_t* sa, const uint8_t* b, const uint8_t* sb, void* c, int64_t m, int64_t n,
           int64_t k, hipStream_t st) {
  T* o = static_cast<T*>(c);
  if (k == 0) {
    return in_runs(m * n, most_groups(256) * 256, [&](int64_t first, int64_t count) {
      k_mx_zero<T><<<(uint32_t)((count + 255) / 256), 256, 0, st>>>(o + first, count);
      return check_launch("k_mx_zero");
    });
  }
  // Few rows: a workgroup reads all of a from the L2 beside its rows of b, so the more rows a has, the more
  // the tiles save that read it once for 64 of them, if there are tiles enough (24 x 32000 x 2048, 8 by 4 bits: 9.1
  // us against 12.2; 8 rows 8.8 against 9.2, one row 8.7 against 7.9; 24 x 4096 x 4096 9.3 against 7.1).  With both
  // sides alike the few rows pay only for the largest weights (1 x 14336 x 4096 in 8 bits 10.9 against 12.5,
  // 1 x 128256 x 4096 125 against 94).
  if (m <= 32 && (n < 12288 || (m <= 8 && (FA != FB || n > 65536)))) return few<FA, FB, T>(a, sa, b, sb, o, m, n, k, st);
  // The largest tile that keeps the CUs busy.  64 x 64 while there are at most two a CU (517 x 2081 x 1283 in
  // 4 bits: 6.0 us against 8.5 with 128 x 128; 512 x 5632 x 2048, three a CU: 10.0 against 9.0).  Beyond, rounds
  // over the CUs decide: one of 128 x 128, two a CU, takes about 0.62 of one of 256 x 256 (4096 x 4096 x 4096 in 4
  // bits: two rounds 45 us, one 36; 2048 x 4096 x 4096: 24 against 28).
  auto tiles_of = [&](int64_t e) { return ((m + e - 1) / e) * ((n + e - 1) / e); };
  const int64_t small = tiles_of(64);
  if (small <= 512) {
    // 8 by 4 bits have the smallest stages: over a long contraction four groups of waves keep more of them on
    // their way (256 x 2048 x 5632: 11.5 us against 14.4; two 8-bit sides 12.5 against 13.7, two of 4 bits 8.7
    // against 9.1, but 16.6 against 14.7 and 9.7 against 9.7 at 512 x 2048 x 5632).
    if constexpr (FA != FB)
      if (k >= 4096 && small <= 256) return tiles<FA, FB, 1, 1, 4, T>(a, sa, b, sb, o, m, n, k, st);
    return tiles<FA, FB, 1, 1, 1, T>(a, sa, b, sb, o, m, n, k, st);
  }
  const int64_t rounds = (tiles_of(256) + 255) / 256, rounds2 = (tiles_of(128) + 511) / 512;
  if (62 * rounds2 < 100 * rounds) return tiles<FA, FB, 2, 2, 1, T>(a, sa, b, sb, o, m, n, k, st);
  return tiles<FA, FB, 4, 4, 1, T>(a, sa, b, sb, o, m, n, k, st);
}

template <int FA, int FB>
int matmul_o(int out, const uint8_t* a, const uint8_t* sa, const uint8_t* b, const uint8_t* sb, void* c, int64_t m,
             int64_t n, int64_t k, hipStream_t st) {
  if (out == A8_F32) return matmul<FA, FB, float>(a, sa, b, sb, c, m, n, k, st);
  if (out == A8_BF16) return matmul<FA, FB, __hip_bfloat16>(a, sa, b, sb, c, m, n, k, st);
  return matmul<FA, FB, __half>(a, sa, b, sb, c, m, n, k, st);
}

}  // namespace
}  // namespace a8

using namespace a8;

extern "C" int a8_mx_matmul(int fmt_a, int fmt_b, int out_dtype, const uint8_t* a_codes, const uint8_t* a_scales,
                            const uint8_t* b_codes, const uint8_t* b_scales, void* c, int64_t m, int64_t n, int64_t k,
                            void* stream) {
  if (out_dtype != A8_F32 && out_dtype != A8_BF16 && out_dtype != A8_F16)
    return set_error(A8_ERR_DTYPE, "mx_matmul: out dtype must be fp32, bf16 or fp16");
  if ((fmt_a != A8_MXFP4 && fmt_a != A8_MXFP8) || (fmt_b != A8_MXFP4 && fmt_b != A8_MXFP8))
    return set_error(A8_ERR_ARG, "mx_matmul: unknown format");
  constexpr int64_t lim = (int64_t)1 << 31;
  // k: a tile's 256 rows of codes stay below 2^31 bytes
  if (m < 0 || n < 0 || k < 0 || m >= lim || n >= lim || k >= lim / 256 || ((m + 31) / 32) * ((n + 31) / 32) >= lim)
    return set_error(A8_ERR_SIZE, "mx_matmul: sizes out of range");
  if (m == 0 || n == 0) return A8_OK;
  if (!c || (k > 0 && (!a_codes || !a_scales || !b_codes || !b_scales)))
    return set_error(A8_ERR_ARG, "mx_matmul: null pointer");
  if (!aligned16(a_codes) || !aligned16(b_codes) || !aligned16(a_scales) || !aligned16(b_scales) || !aligned16(c))
    return set_error(A8_ERR_ALIGN, "mx_matmul: operands must be 16-byte aligned");
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (fmt_a == A8_MXFP4)
    return fmt_b == A8_MXFP4 ? matmul_o<kFp4, kFp4>(out_dtype, a_codes, a_scales, b_codes, b_scales, c, m, n, k, st)
                             : matmul_o<kFp4, kFp8>(out_dtype, a_codes, a_scales, b_codes, b_scales, c, m, n, k, st);
  return fmt_b == A8_MXFP4 ? matmul_o<kFp8, kFp4>(out_dtype, a_codes, a_scales, b_codes, b_scales, c, m, n, k, st)
                           : matmul_o<kFp8, kFp8>(out_dtype, a_codes, a_scales, b_codes, b_scales, c, m, n, k, st);
}
