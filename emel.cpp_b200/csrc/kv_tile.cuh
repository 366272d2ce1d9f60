// Where the bytes of a 16-token tile of a key / value head stand (include/emelb_paged.h says what they mean).
//
// Scores and mixes run on mma.sync.m16n8k16 with the cache as the A operand, so a tile keeps the quants in the order of that
// operand's fragments: lane (g, t) = (lane / 4, lane % 4) reads whole words, neighbouring lanes neighbouring vectors, and
// a word's nibbles spread to f16 pairs by a mask each.
//   keys    rows are tokens, k is the head's dims.  The word of (token, group of 32 dims j, t) holds dims 8t .. 8t+7 of
//           the group: nibble p = dim 8t + 2p, nibble p + 4 = dim 8t + 2p + 1.
//   values  rows are dims, k is the tokens.  The word of (16 dims i, lane) holds for row pair g (dims 2g and 2g + 1, low
//           and high nibble) the tokens 2t, 2t + 8, 2t + 1, 2t + 9, a byte each.
//   scales  keys [token][group], values [t][group][2t, 2t + 1, 2t + 8, 2t + 9].
// Vectors are the widest loads that divide a lane's words: 16 bytes of keys at head_dim 128, 8 at 64.
#pragma once

#include <stdint.h>

namespace emelb {
namespace kv {

constexpr int kTile = 16;   // tokens
constexpr int kGroup = 32;  // values that share a scale

template <int D>
struct Tile {
  static_assert(D % kGroup == 0 && D <= 128, "head_dim");
  static constexpr int kGroups = D / kGroup;
  static constexpr int kVecK = kGroups == 3 ? 1 : kGroups;          // words a load
  static constexpr int kVecV = kGroups % 2 == 0 ? 4 : 2;
  static constexpr int kQuants = kTile * D / 2;
  static constexpr int kV = kQuants, kScaleK = 2 * kQuants, kScaleV = kScaleK + kTile * kGroups * 2;
  static constexpr int kBytes = kScaleV + kTile * kGroups * 2;

  // byte of the word of keys (token, group j, t)
  __host__ __device__ static constexpr int key_word(int token, int j, int t) {
    const int lane = (token & 7) * 4 + t;
    return ((((token >> 3) * (kGroups / kVecK) + j / kVecK) * 32 + lane) * kVecK + j % kVecK) * 4;
  }
  // byte of values (token, dims d and d + 1), d even
  __host__ __device__ static constexpr int value_byte(int token, int d) {
    const int i = d >> 4, g = (d & 15) >> 1, lane = g * 4 + ((token & 7) >> 1);
    return kV + ((i / kVecV * 32 + lane) * kVecV + i % kVecV) * 4 + (token & 1) * 2 + (token >> 3);
  }
  __host__ __device__ static constexpr int key_scale(int token, int j) { return kScaleK + (token * kGroups + j) * 2; }
  __host__ __device__ static constexpr int value_scale(int token, int j) {
    return kScaleV + ((((token & 7) >> 1) * kGroups + j) * 4 + (token & 1) + 2 * (token >> 3)) * 2;
  }
};

}  // namespace kv
}  // namespace emelb
