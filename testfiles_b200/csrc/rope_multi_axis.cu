// rope_multi_axis.cu — rotary embedding with a position per axis (time,
// height, width, ...), in place or into new tensors, forward or inverse, and
// its C entry welm_rope_multi_axis.
//
// The rotation of a pair is orthogonal, so the gradient of the inputs is the
// inverse rotation (sin negated) of the gradient of the outputs: the backward
// pass is the same kernel again.  Memory-bound: six FP32 operations a pair.
// Four threads ("parts") share a head's rotated lanes as in the other kernels;
// the Q heads of a token come first, then its K heads.

#include "rope_axes.cuh"

namespace {

struct MultiAxisArgs {
  const uint16_t* src[2];  // Q and K
  uint16_t* dst[2];        // src in place, or the copies
  int64_t src_token[2], src_head[2], dst_token[2], dst_head[2];
  AxisArgs axes;
  int32_t* status;
  int32_t items, heads, q_heads;
  float sign;  // +1 forward, -1 inverse
};

// In place: only the rotated lanes move.  A thread rotates up to kHeads heads of
// its token with the cos/sin it gathered once, their loads all in flight.
template <int kHeads>
__global__ void __launch_bounds__(kBlock) rope_multi_axis_kernel(const MultiAxisArgs a) {
  const int item = blockIdx.x * blockDim.x + threadIdx.x;
  const int part = item & (kParts - 1);
  const int row = item >> kPartShift;
  const int chunks = (a.heads + kHeads - 1) / kHeads;
  const int tok = row / chunks;
  const int first = row - tok * chunks;  // heads first, first + chunks, ...
  uint16_t* head[kHeads];
#pragma unroll
  for (int i = 0; i < kHeads; ++i) {
    const int h = first + i * chunks;
    const int x = h >= a.q_heads;
    head[i] = h < a.heads ? a.dst[x] + tok * a.dst_token[x] + (x ? h - a.q_heads : h) * a.dst_head[x] + kRopeLane0 +
                                part * kLanes
                          : nullptr;
  }
  if (kHeads > 1 && item < a.items) {
#pragma unroll
    for (int i = 0; i < kHeads; ++i)
      if ((i & 3) == part && head[i] != nullptr) prefetch_line(head[i]);
  }
  pdl_enter();
  if (item >= a.items) return;
  AxisRows rows;
  rows.load(a.axes, tok);
  uint4 x1[kHeads], x2[kHeads];
#pragma unroll
  for (int i = 0; i < kHeads; ++i) {
    if (head[i] == nullptr) continue;
    x1[i] = *reinterpret_cast<const uint4*>(head[i]);
    x2[i] = *reinterpret_cast<const uint4*>(head[i] + kHalf);
  }
  if (!rows.ready(a.axes)) {  // the token stays as it is
    if (part == 0 && first == 0) raise_status(a.status, WELM_ROPE_DEV_BAD_POSITION);
    return;
  }
  CosSin cs;
  rows.gather(a.axes.map, part, cs);
#pragma unroll
  for (int i = 0; i < kLanes; ++i) cs.s[i] *= a.sign;
#pragma unroll
  for (int i = 0; i < kHeads; ++i) {
    if (head[i] == nullptr) continue;
    rotate8(x1[i], x2[i], cs);
    *reinterpret_cast<uint4*>(head[i]) = x1[i];
    *reinterpret_cast<uint4*>(head[i] + kHalf) = x2[i];
  }
}

// Into new tensors: whole heads are read and written, one a thread group of
// four (eight 16-byte loads in flight a thread).  A token whose position is out
// of range is copied as it is.
__global__ void __launch_bounds__(kBlock) rope_multi_axis_copy_kernel(const MultiAxisArgs a) {
  const int item = blockIdx.x * blockDim.x + threadIdx.x;
  const int part = item & (kParts - 1);
  const int row = item >> kPartShift;
  const int tok = row / a.heads;
  const int head = row - tok * a.heads;
  const int x = head >= a.q_heads;
  const int h = x ? head - a.q_heads : head;
  const uint16_t* src = a.src[x] + tok * a.src_token[x] + h * a.src_head[x];
  if (item < a.items) prefetch_line(src + part * 64);
  pdl_enter();
  if (item >= a.items) return;
  AxisRows rows;
  rows.load(a.axes, tok);
  WholeHead piece;
  piece.load(src, part);
  if (rows.ready(a.axes)) {
    CosSin cs;
    rows.gather(a.axes.map, part, cs);
#pragma unroll
    for (int i = 0; i < kLanes; ++i) cs.s[i] *= a.sign;
    rotate8(piece.x1, piece.x2, cs);
  } else if (part == 0 && head == 0) {
    raise_status(a.status, WELM_ROPE_DEV_BAD_POSITION);
  }
  piece.store(a.dst[x] + tok * a.dst_token[x] + h * a.dst_head[x], part);
}

}  // namespace

extern "C" {

int welm_rope_multi_axis(const void* q, void* q_out, const void* k, void* k_out, const int64_t* positions,
                         const float* cos_sin_cache, const int32_t* sections, int64_t num_axes, int64_t interleaved,
                         int64_t inverse, int64_t n_tokens, int64_t num_q_heads, int64_t num_k_heads,
                         int64_t q_token_stride, int64_t q_head_stride, int64_t q_out_token_stride,
                         int64_t q_out_head_stride, int64_t k_token_stride, int64_t k_head_stride,
                         int64_t k_out_token_stride, int64_t k_out_head_stride, int64_t position_stride,
                         int64_t max_position, int32_t* device_status, void* stream) {
  if (num_axes < 1 || num_axes > kMaxAxes || (interleaved != 0 && interleaved != 1) || (inverse != 0 && inverse != 1))
    return WELM_ROPE_ERR_BAD_MODE;
  if (!sections) return WELM_ROPE_ERR_NULL_POINTER;
  MultiAxisArgs a{};
  if (!make_axis_map(sections, num_axes, interleaved, a.axes.map)) return WELM_ROPE_ERR_BAD_MODE;
  if (n_tokens < 0 || num_q_heads < 0 || num_k_heads < 0 || max_position < 0) return WELM_ROPE_ERR_BAD_SIZE;
  if (num_q_heads > kMaxItems || num_k_heads > kMaxItems) return WELM_ROPE_ERR_BAD_SIZE;
  const int64_t heads = num_q_heads + num_k_heads;
  if (n_tokens == 0 || heads == 0) return WELM_ROPE_OK;
  if (n_tokens > kMaxItems / kParts / heads) return WELM_ROPE_ERR_BAD_SIZE;
  if ((num_q_heads > 0 && (!q || !q_out)) || (num_k_heads > 0 && (!k || !k_out)) || !positions || !cos_sin_cache)
    return WELM_ROPE_ERR_NULL_POINTER;
  const void* src[2] = {q, k};
  void* dst[2] = {q_out, k_out};
  const int64_t count[2] = {num_q_heads, num_k_heads};
  const int64_t strides[2][4] = {{q_token_stride, q_head_stride, q_out_token_stride, q_out_head_stride},
                                 {k_token_stride, k_head_stride, k_out_token_stride, k_out_head_stride}};
  bool in_place = true;
  for (int x = 0; x < 2; ++x) {
    if (count[x] == 0) continue;
    const int64_t* s = strides[x];
    // sources may repeat a row (stride 0); destinations may not
    if (s[0] < 0 || s[1] < 0 || !rows_apart<2>({n_tokens, count[x]}, {s[2], s[3]})) return WELM_ROPE_ERR_BAD_STRIDE;
    if (!aligned16(src[x]) || !aligned16(dst[x]) || ((s[0] | s[1] | s[2] | s[3]) & 7)) return WELM_ROPE_ERR_BAD_STRIDE;
    if (src[x] != dst[x]) in_place = false;
    else if (s[0] != s[2] || s[1] != s[3]) return WELM_ROPE_ERR_BAD_STRIDE;
    a.src[x] = static_cast<const uint16_t*>(src[x]);
    a.dst[x] = static_cast<uint16_t*>(dst[x]);
    a.src_token[x] = s[0];
    a.src_head[x] = s[1];
    a.dst_token[x] = s[2];
    a.dst_head[x] = s[3];
  }
  if (!aligned16(cos_sin_cache) || (num_axes > 1 && position_stride < 0)) return WELM_ROPE_ERR_BAD_STRIDE;
  // No thread may write what another reads or writes.
  auto rows = [&](const void* at, int x, int first) {
    return RowSet{reinterpret_cast<uintptr_t>(at), {n_tokens, count[x], 1}, {strides[x][first], strides[x][first + 1], 0}};
  };
  if (rows_meet(rows(dst[0], 0, 2), rows(dst[1], 1, 2))) return WELM_ROPE_ERR_BAD_STRIDE;
  for (int x = 0; x < 2; ++x) {
    if (src[x] == dst[x]) continue;  // in place: its own rows
    for (int to = 0; to < 2; ++to)
      if (rows_meet(rows(src[x], x, 0), rows(dst[to], to, 2))) return WELM_ROPE_ERR_BAD_STRIDE;
  }
  a.axes.positions = positions;
  a.axes.pos_stride = position_stride;
  a.axes.cache = cos_sin_cache;
  a.axes.max_position = max_position;
  a.status = device_status;
  a.heads = int32_t(heads);
  a.q_heads = int32_t(num_q_heads);
  a.sign = inverse ? -1.0f : 1.0f;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  auto grid = [&](int64_t rows) {
    a.items = int32_t(rows * kParts);
    return unsigned((rows * kParts + kBlock - 1) / kBlock);
  };
  if (!in_place) {
    const unsigned ctas = grid(n_tokens * heads);
    return launch(rope_multi_axis_copy_kernel, ctas, kBlock, 0, s, a);
  }
  if (n_tokens * heads <= kOneHeadRows) {
    const unsigned ctas = grid(n_tokens * heads);
    return launch(rope_multi_axis_kernel<1>, ctas, kBlock, 0, s, a);
  }
  const unsigned ctas = grid(n_tokens * ((heads + 3) / 4));
  return launch(rope_multi_axis_kernel<4>, ctas, kBlock, 0, s, a);
}

}  // extern "C"
