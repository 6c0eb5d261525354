// rope_axes.cuh — position gather with one position per axis and token, shared
// by the multi-axis rotary kernels and the rotating KV-cache append.
//
// Pair i (lanes 192 + i and 224 + i of a head, i < 32) belongs to one of up to
// four axes and is rotated by the cos/sin of that axis' position:
//     c = cache[positions[axis(i)][t]][i]     s = cache[positions[axis(i)][t]][32 + i]
// One axis with all 32 pairs is the ordinary rotary embedding.

#ifndef WELM_ROPE_AXES_CUH_
#define WELM_ROPE_AXES_CUH_

#include "rope_host.cuh"

namespace {

constexpr int kMaxAxes = WELM_ROPE_MAX_AXES;
constexpr int kQuads = kHalf / 4;  // groups of four neighbouring pairs

// The axis of every pair, built on the host (make_axis_map).
struct AxisMap {
  uint64_t axis;   // two bits a pair
  uint32_t quads;  // bit g: pairs 4g .. 4g + 3 share one axis, so one 16-byte load serves them
  uint32_t used;   // bit a: axis a rotates some pair; an axis of no pairs is not read
};

struct AxisArgs {
  const int64_t* positions;  // [axes][n_tokens], rows pos_stride apart
  int64_t pos_stride;
  const float* cache;  // [max_position, 64]
  int64_t max_position;
  AxisMap map;
};

// Cache rows of one token.  load() starts the position loads, ready() turns
// them into rows: false when a used axis' position lies outside the cache (then
// nothing may be read).  Every thread of a token comes to the same answer,
// whichever pairs it rotates.
struct AxisRows {
  int64_t pos[kMaxAxes];
  const float* row[kMaxAxes];
  __device__ __forceinline__ void load(const AxisArgs& a, int64_t tok) {
#pragma unroll
    for (int x = 0; x < kMaxAxes; ++x)
      pos[x] = a.map.used >> x & 1u ? __ldg(a.positions + x * a.pos_stride + tok) : 0;
  }
  __device__ __forceinline__ bool ready(const AxisArgs& a) {
    bool ok = true;
#pragma unroll
    for (int x = 0; x < kMaxAxes; ++x) {
      if (a.map.used >> x & 1u) ok = ok && pos[x] >= 0 && pos[x] < a.max_position;
      row[x] = a.cache + pos[x] * kRopeDim;
    }
    return ok;
  }
  __device__ __forceinline__ const float* of(uint64_t axis, int pair) const {
    const uint32_t x = uint32_t(axis >> (2 * pair)) & 3u;
    const float* p = row[0];
    if (x == 1) p = row[1];
    if (x == 2) p = row[2];
    if (x == 3) p = row[3];
    return p;
  }
  // cos and sin of the eight pairs of `part`.
  __device__ __forceinline__ void gather(const AxisMap& m, int part, CosSin& cs) const {
#pragma unroll
    for (int g = 0; g < kLanes / 4; ++g) {
      const int pair = part * kLanes + 4 * g;
      if (m.quads >> (pair / 4) & 1u) {
        const float* p = of(m.axis, pair) + pair;
        const float4 c = __ldg(reinterpret_cast<const float4*>(p));
        const float4 s = __ldg(reinterpret_cast<const float4*>(p + kHalf));
        cs.c[4 * g] = c.x; cs.c[4 * g + 1] = c.y; cs.c[4 * g + 2] = c.z; cs.c[4 * g + 3] = c.w;
        cs.s[4 * g] = s.x; cs.s[4 * g + 1] = s.y; cs.s[4 * g + 2] = s.z; cs.s[4 * g + 3] = s.w;
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float* p = of(m.axis, pair + i) + pair + i;
          cs.c[4 * g + i] = __ldg(p);
          cs.s[4 * g + i] = __ldg(p + kHalf);
        }
      }
    }
  }
};

// All 256 lanes of a head, the part of them that one of its four threads
// holds: six 16-byte chunks of lanes 0..191 and its eight x1 and x2 lanes.
constexpr int kHeadNopeChunks = kRopeLane0 / kParts / 8;

struct WholeHead {
  uint4 nope[kHeadNopeChunks];
  uint4 x1, x2;
  __device__ __forceinline__ void load(const uint16_t* head, int part) {
#pragma unroll
    for (int c = 0; c < kHeadNopeChunks; ++c)
      nope[c] = *reinterpret_cast<const uint4*>(head + part * 8 + 8 * kParts * c);
    x1 = *reinterpret_cast<const uint4*>(head + kRopeLane0 + part * kLanes);
    x2 = *reinterpret_cast<const uint4*>(head + kRopeLane0 + kHalf + part * kLanes);
  }
  __device__ __forceinline__ void store(uint16_t* head, int part) const {
#pragma unroll
    for (int c = 0; c < kHeadNopeChunks; ++c)
      *reinterpret_cast<uint4*>(head + part * 8 + 8 * kParts * c) = nope[c];
    *reinterpret_cast<uint4*>(head + kRopeLane0 + part * kLanes) = x1;
    *reinterpret_cast<uint4*>(head + kRopeLane0 + kHalf + part * kLanes) = x2;
  }
};

// ---------------------------------------------------------------------------
// Host side.
// ---------------------------------------------------------------------------
// In-place rotations of at most this many (token, head) rows take one head a
// thread, so that a small launch spreads over more threads; larger ones take up
// to four, so that more loads share a position and are in flight at once.
constexpr int64_t kOneHeadRows = 8192;

// Sections: the pairs of each axis, 32 in all.  In runs (axis 0's pairs
// first), or dealt out in turn over the axes that still have pairs left.
bool make_axis_map(const int32_t* sections, int64_t axes, int64_t interleaved, AxisMap& m) {
  int left[kMaxAxes] = {0, 0, 0, 0};
  int sum = 0;
  for (int x = 0; x < axes; ++x) {
    if (sections[x] < 0 || sections[x] > kHalf) return false;
    left[x] = sections[x];
    sum += sections[x];
  }
  if (sum != kHalf) return false;
  m = AxisMap{0, 0, 0};
  int of[kHalf];
  int pair = 0;
  while (pair < kHalf) {
    for (int x = 0; x < axes; ++x) {
      for (int n = interleaved ? (left[x] > 0 ? 1 : 0) : left[x]; n > 0; --n) {
        of[pair] = x;
        --left[x];
        m.axis |= uint64_t(x) << (2 * pair);
        m.used |= 1u << x;
        ++pair;
      }
    }
  }
  for (int g = 0; g < kQuads; ++g)
    if (of[4 * g] == of[4 * g + 1] && of[4 * g] == of[4 * g + 2] && of[4 * g] == of[4 * g + 3]) m.quads |= 1u << g;
  return true;
}

}  // namespace

#endif  // WELM_ROPE_AXES_CUH_
