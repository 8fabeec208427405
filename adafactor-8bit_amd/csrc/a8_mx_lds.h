// Where the end of a product's tile lies in LDS.  No device code, so that a host compiler can check it.
//
// A wave of group 0 stages its outputs, 32 rows at a time, in a part of its own.  With KG groups of waves
// the others leave their sums in LDS first: a wave reads those of its own place and stages its outputs
// with no barrier in between, so the sums lie behind all four waves' staging.
#pragma once

namespace a8 {

template <int NI, int KG, int BYTES>   // 32 NI columns a wave, BYTES an output
struct MxEnd {
  static constexpr int kRow = 32 * NI * BYTES + 16;   // of a staged row
  static constexpr int kPart = 32 * kRow;             // a wave's staging
  static constexpr int kStaging = 4 * kPart;
  static constexpr int kWaveSums = 64 * 16 * 4;       // 16 fp32 sums a lane
  static constexpr int kGroupSums = 4 * kWaveSums;
  static constexpr int staged(int wave) { return wave * kPart; }
  static constexpr int sums(int group, int wave) {    // of group 1, 2 ..
    return kStaging + (group - 1) * kGroupSums + wave * kWaveSums;
  }
  static constexpr int kBytes = kStaging + (KG - 1) * kGroupSums;
};

}  // namespace a8
