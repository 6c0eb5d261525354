// rope_kv_append.cu — rotary embedding fused with the append to a paged KV
// cache (ordinary prefill and decode), and its C entry welm_rope_kv_append.
//
// Q is rotated in place; the rotated K and the V of every token are written to
// the token's cache slot, so K is read once and never written back.
// Memory-bound.  Work items: one per (token, K head, part), whose thread moves a
// quarter of a K head and of its V head with all sixteen 16-byte loads in
// flight at once, then one per (token, chunk of Q heads, part).

#include "rope_axes.cuh"

namespace {

struct AppendArgs {
  uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  uint16_t* key_cache;
  uint16_t* value_cache;
  const int64_t* slots;
  int64_t q_token, q_head, k_token, k_head, v_token, v_head;
  int64_t key_block, key_slot, key_head, value_block, value_slot, value_head;
  int64_t num_slots;
  AxisArgs axes;
  int32_t* status;
  int32_t q_items, kv_items, q_heads, q_chunks, k_heads, block_size;
};

constexpr int kValueChunks = kHeadDim / kParts / 8;  // 16-byte chunks of V a thread moves

// Whether the token is written; otherwise it is padding or flagged.  `tell`:
// this thread reports.
__device__ __forceinline__ bool append_token(const AppendArgs& a, int64_t slot, AxisRows& rows, bool tell) {
  if (slot < 0) return false;
  const bool ok = rows.ready(a.axes);
  if (tell && !ok) raise_status(a.status, WELM_ROPE_DEV_BAD_POSITION);
  if (slot < a.num_slots) return ok;
  if (tell) raise_status(a.status, WELM_ROPE_DEV_BAD_SLOT);
  return false;
}

// kHeads: Q heads a thread rotates with the cos/sin that it gathered once.
template <int kHeads>
__global__ void __launch_bounds__(kBlock) rope_kv_append_kernel(const AppendArgs a) {
  const int item = blockIdx.x * blockDim.x + threadIdx.x;
  const int part = item & (kParts - 1);
  const bool is_q = item >= a.kv_items;
  const int row = (is_q ? item - a.kv_items : item) >> kPartShift;
  const int per_token = is_q ? max(a.q_chunks, 1) : a.k_heads;
  const int tok = row / per_token;
  const int h = row - tok * per_token;
  const bool live = item < a.kv_items + a.q_items;
  const uint16_t* k = a.k + tok * a.k_token + h * a.k_head;
  const uint16_t* v = a.v + tok * a.v_token + h * a.v_head;
  uint16_t* q = a.q + tok * a.q_token + h * a.q_head + kRopeLane0 + part * kLanes;
  const int64_t q_step = a.q_chunks * a.q_head;
  const int heads = (a.q_heads - h + a.q_chunks - 1) / per_token;  // h, h + chunks, ...
  if (live) {
    if (!is_q) {
      prefetch_line(k + part * 64);
      prefetch_line(v + part * 64);
    } else if (kHeads > 1 && part < heads) {
      prefetch_line(q + part * q_step);
    }
  }
  pdl_enter();
  if (!live) return;
  const int64_t slot = __ldg(a.slots + tok);
  AxisRows rows;
  rows.load(a.axes, tok);
  CosSin cs;
  if (is_q) {
    uint4 x1[kHeads], x2[kHeads];
#pragma unroll
    for (int i = 0; i < kHeads; ++i) {
      if (i >= heads) continue;
      x1[i] = *reinterpret_cast<const uint4*>(q + i * q_step);
      x2[i] = *reinterpret_cast<const uint4*>(q + i * q_step + kHalf);
    }
    if (!append_token(a, slot, rows, false)) return;
    rows.gather(a.axes.map, part, cs);
#pragma unroll
    for (int i = 0; i < kHeads; ++i) {
      if (i >= heads) continue;
      rotate8(x1[i], x2[i], cs);
      *reinterpret_cast<uint4*>(q + i * q_step) = x1[i];
      *reinterpret_cast<uint4*>(q + i * q_step + kHalf) = x2[i];
    }
  } else {
    WholeHead piece;
    piece.load(k, part);
    uint4 vv[kValueChunks];
#pragma unroll
    for (int c = 0; c < kValueChunks; ++c)
      vv[c] = *reinterpret_cast<const uint4*>(v + part * 8 + 8 * kParts * c);
    if (!append_token(a, slot, rows, part == 0 && h == 0)) return;
    rows.gather(a.axes.map, part, cs);
    rotate8(piece.x1, piece.x2, cs);
    const int64_t block = slot / a.block_size;
    const int64_t place = slot - block * a.block_size;
    piece.store(a.key_cache + block * a.key_block + place * a.key_slot + h * a.key_head, part);
    uint16_t* to = a.value_cache + block * a.value_block + place * a.value_slot + h * a.value_head + part * 8;
#pragma unroll
    for (int c = 0; c < kValueChunks; ++c) *reinterpret_cast<uint4*>(to + 8 * kParts * c) = vv[c];
  }
}

}  // namespace

extern "C" {

int welm_rope_kv_append(void* q, const void* k, const void* v, const int64_t* positions, const float* cos_sin_cache,
                        const int32_t* sections, int64_t num_axes, int64_t interleaved, const int64_t* slot_mapping,
                        void* key_cache, void* value_cache, int64_t n_tokens, int64_t num_q_heads,
                        int64_t num_k_heads, int64_t q_token_stride, int64_t q_head_stride, int64_t k_token_stride,
                        int64_t k_head_stride, int64_t v_token_stride, int64_t v_head_stride, int64_t num_blocks,
                        int64_t block_size, const int64_t* key_cache_strides, const int64_t* value_cache_strides,
                        int64_t position_stride, int64_t max_position, int32_t* device_status, void* stream) {
  if (num_axes < 1 || num_axes > kMaxAxes || (interleaved != 0 && interleaved != 1)) return WELM_ROPE_ERR_BAD_MODE;
  if (!sections || !key_cache_strides || !value_cache_strides) return WELM_ROPE_ERR_NULL_POINTER;
  AppendArgs a{};
  if (!make_axis_map(sections, num_axes, interleaved, a.axes.map)) return WELM_ROPE_ERR_BAD_MODE;
  if (n_tokens < 0 || num_q_heads < 0 || num_k_heads < 1 || num_blocks < 0 || block_size < 1 || max_position < 0)
    return WELM_ROPE_ERR_BAD_SIZE;
  if (num_q_heads > kMaxItems || num_k_heads > kMaxItems || block_size > kMaxItems ||
      num_blocks > INT64_MAX / block_size)
    return WELM_ROPE_ERR_BAD_SIZE;
  if (n_tokens == 0) return WELM_ROPE_OK;
  if (n_tokens > kMaxItems / kParts / (num_q_heads + num_k_heads)) return WELM_ROPE_ERR_BAD_SIZE;
  if ((num_q_heads > 0 && !q) || !k || !v || !positions || !cos_sin_cache || !slot_mapping || !key_cache ||
      !value_cache)
    return WELM_ROPE_ERR_NULL_POINTER;
  if (num_q_heads > 0 && !rows_apart<2>({n_tokens, num_q_heads}, {q_token_stride, q_head_stride}))
    return WELM_ROPE_ERR_BAD_STRIDE;
  for (const int64_t* s : {key_cache_strides, value_cache_strides})
    if (!rows_apart<3>({num_blocks, block_size, num_k_heads}, {s[0], s[1], s[2]})) return WELM_ROPE_ERR_BAD_STRIDE;
  int64_t low = 0, bits = num_q_heads > 0 ? q_token_stride | q_head_stride : 0;
  for (const int64_t s : {k_token_stride, k_head_stride, v_token_stride, v_head_stride}) {
    low = s < low ? s : low;
    bits |= s;
  }
  for (int i = 0; i < 3; ++i) {
    for (const int64_t s : {key_cache_strides[i], value_cache_strides[i]}) {
      low = s < low ? s : low;
      bits |= s;
    }
  }
  if (low < 0 || (bits & 7) || (num_axes > 1 && position_stride < 0)) return WELM_ROPE_ERR_BAD_STRIDE;
  for (const void* p : {static_cast<const void*>(q), k, v, static_cast<const void*>(cos_sin_cache),
                        static_cast<const void*>(key_cache), static_cast<const void*>(value_cache)})
    if (!aligned16(p)) return WELM_ROPE_ERR_BAD_STRIDE;
  // No thread may write what another reads or writes.  K and V may lie in the
  // caches: which of those rows are written depends on the slots.
  auto rows = [&](const void* at, int64_t heads, int64_t token, int64_t head) {
    return RowSet{reinterpret_cast<uintptr_t>(at), {n_tokens, heads, 1}, {token, head, 0}};
  };
  auto pages = [&](const void* at, const int64_t* s) {
    return RowSet{reinterpret_cast<uintptr_t>(at), {num_blocks, block_size, num_k_heads}, {s[0], s[1], s[2]}};
  };
  const RowSet q_rows = rows(q, num_q_heads, q_token_stride, q_head_stride);
  const RowSet keys = pages(key_cache, key_cache_strides), values = pages(value_cache, value_cache_strides);
  if (rows_meet(q_rows, rows(k, num_k_heads, k_token_stride, k_head_stride)) ||
      rows_meet(q_rows, rows(v, num_k_heads, v_token_stride, v_head_stride)) || rows_meet(q_rows, keys) ||
      rows_meet(q_rows, values) || rows_meet(keys, values))
    return WELM_ROPE_ERR_BAD_STRIDE;
  a.q = static_cast<uint16_t*>(q);
  a.k = static_cast<const uint16_t*>(k);
  a.v = static_cast<const uint16_t*>(v);
  a.key_cache = static_cast<uint16_t*>(key_cache);
  a.value_cache = static_cast<uint16_t*>(value_cache);
  a.slots = slot_mapping;
  a.q_token = q_token_stride;
  a.q_head = q_head_stride;
  a.k_token = k_token_stride;
  a.k_head = k_head_stride;
  a.v_token = v_token_stride;
  a.v_head = v_head_stride;
  a.key_block = key_cache_strides[0];
  a.key_slot = key_cache_strides[1];
  a.key_head = key_cache_strides[2];
  a.value_block = value_cache_strides[0];
  a.value_slot = value_cache_strides[1];
  a.value_head = value_cache_strides[2];
  a.num_slots = num_blocks * block_size;
  a.axes.positions = positions;
  a.axes.pos_stride = position_stride;
  a.axes.cache = cos_sin_cache;
  a.axes.max_position = max_position;
  a.status = device_status;
  a.q_heads = int32_t(num_q_heads);
  a.k_heads = int32_t(num_k_heads);
  a.block_size = int32_t(block_size);
  const bool one = n_tokens * num_q_heads <= kOneHeadRows;
  a.q_chunks = int32_t(one ? num_q_heads : (num_q_heads + 3) / 4);
  a.q_items = int32_t(n_tokens * a.q_chunks * kParts);
  a.kv_items = int32_t(n_tokens * num_k_heads * kParts);
  const unsigned grid = unsigned((int64_t(a.q_items) + a.kv_items + kBlock - 1) / kBlock);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  return one ? launch(rope_kv_append_kernel<1>, grid, kBlock, 0, s, a)
             : launch(rope_kv_append_kernel<4>, grid, kBlock, 0, s, a);
}

}  // extern "C"
