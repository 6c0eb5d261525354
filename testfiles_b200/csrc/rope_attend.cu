// rope_attend.cu — attention of a batch over a paged KV cache whose requests
// share a prefix, and its C entries welm_rope_attend and
// welm_rope_attend_workspace.
//
// Query row (token t, head): o = sum_j p_j v_j / sum_j p_j with p_j =
// exp(scale q.k_j - max) over the prefix's keys and the request's own keys up
// to the token's position.  Both parts are exact softmax partial results (m,
// l, O) with m the maximum, l = sum p and O = sum p v; two of them join as
//     m = max(m1, m2), l = l1 2^(m1 - m) + l2 2^(m2 - m), O likewise.
//
// Work.  An item is 128 query rows (tokens x the query heads of one KV head)
// against a run of keys.  The prefix's items take their rows from all requests
// together, so a prefix key is read once for every 128 rows instead of once
// for every request; a request's own items hold its own rows.  Where requests
// fill their row tiles by themselves that gains nothing, and an item is a
// request's rows against the prefix and its own keys in one.  All items'
// 128-key tiles form one line, cut into equal runs, one for each CTA; a CTA
// walks the pieces of items in its run.  An item that is cut, or whose rows
// also have the other part, leaves FP32 partial results in the workspace, and
// a second kernel joins them row by row in the order of the keys, so results
// do not depend on timing.  Lengths stay on the device: every CTA adds the
// requests' tiles up for itself, and a captured launch follows new lengths.
//
// One CTA on an SM, twelve warps:
//   0      TMA producer: K and V, half a tile (32 KB) at a time, into rings of
//          three and two
//   1, 2   issue tcgen05.mma: S = Q K^T (128 x 128), and O += P V (128 x 256)
//   3      adds up the line, lists the CTA's pieces and brings their Q rows into
//          shared memory (64 KB)
//   4..11  softmax: two threads a row, 64 keys each; rescaling of O; results.
//          At first they help to add up the line and bring the first Q rows
// S and O live in TMEM, S twice, so that the softmax of one tile runs beside
// the products of its neighbours; P (BF16) takes columns of S.  P is rounded
// to BF16 because the product with the BF16 values takes both operands in one
// type; l sums the unrounded p, and S, m, l and O are FP32.

#include <cmath>

#include "rope_tma.cuh"

namespace {

constexpr int kRows = 128;             // query rows of an item
constexpr int kKeys = 128;             // keys of a tile
constexpr int kHalfLanes = kHeadDim / 2;   // lanes of half a K or V tile
// Halves of K and V tiles in shared memory.  Each ring has one warp that fills it
// and one that empties it, each in order, so nobody looks at a stage before its
// last contents have landed.
constexpr int kStagesK = 3, kStagesV = 2;
constexpr int kHalfKeys = kKeys / 2;  // keys of half a V tile
constexpr int kChunkBytes = kKeys * 128;   // 64 lanes of 128 keys
constexpr int kStageBytes = 2 * kChunkBytes;
constexpr int kQChunkBytes = kRows * 128;  // 64 lanes of 128 rows
constexpr int kQBytes = kRows * kHeadDim * 2;
// What an item costs beside its tiles (its Q rows, its results), in tiles.
// Measured with 1, 2 and 3 on one B200 (graph replay, us): 128 requests over a
// prefix 31.2, 29.6, 30.6; 48 requests 24.7, 24.6, 25.3; 24 requests' verification
// 20.7, 22.0, 21.6; 256 requests over 32768 shared keys 84 to 89 with each.
constexpr int kItemCost = 2;
constexpr int kPieces = 4;             // ring of piece descriptors
constexpr int kThreads = 384;
constexpr int kSoftmaxWarp0 = 4, kSoftmaxWarps = 8;
constexpr int kPieceReaders = 3 + kSoftmaxWarps;  // producer, two issuers, softmax warps
// TMEM columns.  S (128 columns) and P (64) of three tiles in turn share the first
// 256, in quarters: S(t) in 0 and 1, P(t) in 0; S(t + 1) in 2 and 3, P(t + 1) in 3;
// S(t + 2) in 1 and 2, P(t + 2) in 2.  Then the scores of two tiles in three need
// not wait for the products before them, only for S to have been read: 2560 query
// tokens 119.2 us with S and P of a tile in the same half, 116.4 so.
constexpr uint32_t kColO = 256;
__host__ __device__ constexpr uint32_t col_s(uint32_t third) { return third == 0 ? 0 : third == 1 ? 128 : 64; }
__host__ __device__ constexpr uint32_t col_p(uint32_t third) { return third == 0 ? 0 : third == 1 ? 192 : 128; }
constexpr long long kWaitClocks = 1ll << 32;  // about two seconds
constexpr float kLog2E = 1.4426950408889634f;
constexpr float kRescaleStep = 8.0f;   // O is rescaled when the maximum grows by more than 2^8

// Division by a number that the host knows: x / d for 0 <= x < 2^31 as one
// multiplication and a shift.  mul = ceil(2^(31 + L) / d) with L = ceil(log2 d)
// is less than d <= 2^L over 2^(31 + L) / d, too little to reach the next quotient.
struct Divisor {
  uint32_t mul = 0;
  int32_t shift = 0, d = 1;
  Divisor() = default;
  __host__ __device__ explicit Divisor(int64_t by) : d(int32_t(by)) {
    int log = 0;
    while ((int64_t(1) << log) < by) ++log;
    shift = 31 + log;
    mul = uint32_t(((uint64_t(1) << shift) + uint64_t(by) - 1) / uint64_t(by));
  }
  __device__ __forceinline__ int of(int x) const { return int((uint64_t(uint32_t(x)) * mul) >> shift); }
};

struct AttendArgs {
  const uint16_t* q;
  uint16_t* out;
  float* lse;  // may be null
  int64_t q_token, q_head, out_token, out_head;
  const int32_t* prefix_table;
  const int32_t* block_table;
  int64_t table_stride;
  const int64_t* seq_lens;
  const int64_t* query_starts;  // may be null: one token a request
  int32_t tokens, batch, q_heads, k_heads, group;
  Divisor by_group, by_block, by_q_heads;
  int32_t prefix_len, max_len;  // max_len: keys that a row of block_table can name
  int32_t block_size, num_blocks;
  int32_t box_k, box_v;         // keys of one TMA box: powers of two that divide block_size, up to 128 and 64
  int32_t slot_rows;            // rows of a workspace slot
  int32_t grid;
  int32_t fill;                 // 1: rows of no request become zeros; their lse is minus infinity either way
  float scale;                  // times log2(e)
  int32_t give_up;              // 1: at the first wait that is not over
  struct LineNote* note;        // what the join needs of the line
  int32_t* gave_up;             // [grid] 1: a wait of the CTA did not end
  int32_t* units_before;        // [batch] units of the own items before each request
  // Partial results.  O is laid out [32][rows][8 lanes]: the threads of a warp,
  // a row each, then write (and a row's reader reads) whole 32-byte sectors.
  float* slot_ml;               // [2 grid][slot_rows][2]
  float* slot_o;                // [2 grid][32][slot_rows][8]
  float* part_ml;               // [2][k_heads * tokens * group][2]: whole items' rows, prefix and own
  float* part_o;                // [2][32][k_heads * tokens * group][8]
  int32_t* status;
};

__device__ __forceinline__ int div_up(int a, int b) { return (a + b - 1) / b; }
__device__ __forceinline__ int64_t clamp64(int64_t v, int64_t lo, int64_t hi) {
  return v < lo ? lo : v > hi ? hi : v;
}

// One request's own part: `count` query tokens from token `first`, the last of
// them at the last of `len` keys.  `joint` is the number of the prefix's key tiles
// where its items hold the prefix too, and -1 where they do not.
struct Request {
  int first, count, len;
  __device__ __forceinline__ int row_tiles(const AttendArgs& a) const { return div_up(count * a.group, kRows); }
  // Keys that the last row of row tile rt sees: every row of it sees at most these.
  __device__ __forceinline__ int seen(const AttendArgs& a, int rt) const {
    const int last = min(a.by_group.of(rt * kRows + kRows - 1), count - 1);
    return max(len - count + last + 1, 0);
  }
  __device__ __forceinline__ int tiles(const AttendArgs& a, int rt) const { return div_up(seen(a, rt), kKeys); }
  // Key tiles of one head's row tiles before rt, rt below row_tiles.  Row tile x
  // (not the last) has ceil((b + floor((128 x + 127) / G)) / 128) of them, b =
  // len - count + 1; nested floors make that floor((x + c) / G) with c = floor((127
  // + G (b + 127)) / 128), or none if negative, and sums of floor(i / G) are
  // triangular numbers.
  __device__ __forceinline__ int tiles_before(const AttendArgs& a, int rt) const {
    if (rt == 0) return 0;
    const int c = int((127 + int64_t(a.group) * (len - count + 128)) >> 7);
    auto sum = [&](int x) {  // of floor(i / G) over 0 <= i < x
      if (x <= 0) return 0;
      const int q = a.by_group.of(x);
      return int(int64_t(a.group) * q * (q - 1) / 2) + q * (x - q * a.group);
    };
    return sum(rt + c) - sum(c);
  }
  // Row tiles before rt that see own keys (tile x does not while x + c < G).
  __device__ __forceinline__ int seeing_before(const AttendArgs& a, int rt) const {
    if (rt == 0) return 0;
    const int c = int((127 + int64_t(a.group) * (len - count + 128)) >> 7);
    return rt - min(max(a.group - c, 0), rt);
  }
  // Units of the line that one head's row tiles before rt take: their tiles,
  // and kItemCost for each that has any.
  __device__ __forceinline__ int units_before(const AttendArgs& a, int rt, int joint) const {
    return tiles_before(a, rt) + (joint >= 0 ? rt * (joint + kItemCost) : seeing_before(a, rt) * kItemCost);
  }
  __device__ __forceinline__ int all_units(const AttendArgs& a, int joint) const {
    const int n = row_tiles(a);
    return n == 0 ? 0 : units_before(a, n - 1, joint) + units(len > 0 ? div_up(len, kKeys) : 0, joint);
  }
  // Units of an item with `tiles` own tiles.
  static __device__ __forceinline__ int units(int tiles, int joint) {
    return joint >= 0 ? joint + tiles + kItemCost : tiles > 0 ? tiles + kItemCost : 0;
  }
};

// A request as the device arrays have it, and checked.
struct RawRequest {
  int64_t start, end, len;
  __device__ __forceinline__ void load(const AttendArgs& a, int b, bool hint = false) {
    start = end = b;
    if (a.query_starts != nullptr) {
      start = hint ? hint_load(a.query_starts + b) : __ldg(a.query_starts + b);
      end = hint ? hint_load(a.query_starts + b + 1) : __ldg(a.query_starts + b + 1);
    } else {
      ++end;
    }
    len = hint ? hint_load(a.seq_lens + b) : __ldg(a.seq_lens + b);
  }
  __device__ __forceinline__ Request checked(const AttendArgs& a, bool tell) const {
    const int64_t lo = clamp64(start, 0, a.tokens), hi = clamp64(end, lo, a.tokens), n = clamp64(len, 0, a.max_len);
    if (tell && !(lo == start && hi == end && n == len)) raise_status(a.status, WELM_ROPE_DEV_BAD_LENGTH);
    return Request{int(lo), int(hi - lo), int(n)};
  }
};

// Query tokens in use: those behind the last request are left alone.
__device__ __forceinline__ int used_tokens(const AttendArgs& a) {
  return a.query_starts != nullptr ? int(clamp64(__ldg(a.query_starts + a.batch), 0, a.tokens)) : a.tokens;
}

// The line of all items' units, cut into `grid` runs: CTA c has [begin(c),
// begin(c + 1)).  An item's first kItemCost units stand for its own cost (its
// rows, its results) and hold no tile; a run that ends among them does nothing
// for the item.  No run is empty: a line of fewer units than CTAs keeps only as
// many busy.  Runs that are longer by a unit come first (with them last, 48
// requests 25.4 -> 26.3 us, 128 over a prefix 29.9 -> 30.7).
struct Line {
  int units, grid, each, more;  // the first `more` runs have each + 1 tiles
  __device__ __forceinline__ Line(int n, int ctas) : units(max(n, 0)), grid(min(units, ctas)) {
    each = grid > 0 ? units / grid : 0;
    more = units - each * grid;
  }
  __device__ __forceinline__ int begin(int c) const { return each * c + (c < more ? c : more); }
};

// The line as the join kernel reads it; divisions are by each and each + 1.
struct LineNote {
  int32_t pre, joint, each, more;
  int32_t nothing;  // 1: no row belongs to a request
  Divisor by_each, by_longer;
  __device__ __forceinline__ int cta_of(int u) const {
    const int longer = more * (each + 1);
    return u < longer ? by_longer.of(u) : more + by_each.of(u - longer);
  }
};

__device__ __forceinline__ int prefix_units(const AttendArgs& a, int used) {
  return a.prefix_len == 0 ? 0 : div_up(used * a.group, kRows) * a.k_heads * (div_up(a.prefix_len, kKeys) + kItemCost);
}

enum Destination { kToOutput, kToSlot, kToPart };

// A piece of an item, as the warps of a CTA read it.
struct Piece {
  int32_t tiles;       // 0: no more pieces
  int32_t first_tile;
  int32_t keys;        // keys that some row of the item sees
  int32_t head;        // KV head
  int32_t row0;        // first row, as (token - first) * group + query head in the group
  int32_t rows;
  int32_t first;       // token that rows are counted from
  int32_t seen0;       // keys that token `first` sees; a later token sees one more each, or `keys` in the prefix
  int32_t own;         // 1: a request's own keys, behind the prefix's if the item has them; 0: the prefix
  int32_t shared_tiles;  // the item's tiles of the prefix, which come first
  int32_t table_row;   // row of block_table
  int32_t once;        // 1: no other item reads the own keys
  int32_t to;          // Destination
  int32_t slot;
};

// What the line is made of, of one head of some requests.
struct LineSums {
  int units, row_tiles, seeing;  // own items' units; row tiles, and those that see own keys
  int decreasing;                // requests that end before they start
};

struct Control {
  uint64_t full_k[kStagesK], empty_k[kStagesK], full_v[kStagesV], empty_v[kStagesV];
  uint64_t s_full[2], s_read[2], p_full[4], pv_done[4];
  uint64_t q_first, q_full, q_empty, o_free, drained[2];
  uint64_t swap[4];  // the two warps of 32 rows
  uint64_t piece_full[kPieces], piece_empty[kPieces];
  uint64_t added, checked;
  Piece piece[kPieces];
  LineSums sums[kSoftmaxWarps];
  uint32_t tmem;
  int32_t failed;
  int32_t changed;  // 1: some of the requests were not as hinted
};

// The two halves of a row's keys swap their maxima (even and odd tiles apart)
// and at last their sums through shared memory.
struct Swap {
  float value[2][2][kRows];  // [tile parity][half]
};

constexpr int kSmemBytes = kQBytes + (kStagesK + kStagesV) * kStageBytes + sizeof(Swap) + 896;
static_assert(sizeof(Control) <= 896, "control block");
static_assert(kSmemBytes <= 227 * 1024, "shared memory of one CTA");

// Waits for a phase of `bar`; false once any warp of the CTA has given up.
__device__ __forceinline__ bool mbar_wait(Control& ctl, uint64_t* bar, uint32_t parity) {
  if (mbar_poll(bar, parity)) return true;
  const long long t0 = clock64();
  while (!mbar_poll(bar, parity)) {
    if (*reinterpret_cast<volatile int32_t*>(&ctl.failed)) return false;
    if (clock64() - t0 > kWaitClocks) {
      *reinterpret_cast<volatile int32_t*>(&ctl.failed) = 1;
      return false;
    }
  }
  return true;
}

__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// ---------------------------------------------------------------------------
// tcgen05: descriptors, products, TMEM reads and writes.
// ---------------------------------------------------------------------------
// Shared-memory operand descriptor, 128-byte swizzle.  K-major (Q and K: lanes
// are the contraction): `stride` is the step between groups of eight rows.
// MN-major (V: keys are the contraction): `lead` steps between 64-lane chunks
// and `stride` between groups of eight keys.
__device__ __forceinline__ uint64_t operand_desc(uint32_t addr, uint32_t lead, uint32_t stride) {
  return uint64_t((addr & 0x3ffffu) >> 4) | uint64_t(lead >> 4) << 16 | uint64_t(stride >> 4) << 32 |
         uint64_t(1) << 46 | uint64_t(2) << 61;
}

// Instruction descriptor: FP32 accumulator, BF16 operands, M = 128.
__host__ __device__ constexpr uint32_t instr_desc(int n, bool b_mn_major) {
  return 1u << 4 | 1u << 7 | 1u << 10 | uint32_t(b_mn_major) << 16 | uint32_t(n / 8) << 17 | uint32_t(kRows / 16) << 24;
}

__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d), "l"(a), "l"(b), "r"(idesc),
      "r"(uint32_t(add))
      : "memory");
}

__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d), "r"(a), "l"(b), "r"(idesc),
      "r"(uint32_t(add))
      : "memory");
}

// Arrives on `bar` when every product issued so far is done.
__device__ __forceinline__ void mma_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
               : "memory");
}

// One lane of a whole warp.  What the lane's products take is computed by the
// warp, alike in every lane, so that it can stay in uniform registers.
__device__ __forceinline__ bool elect_one() {
  uint32_t one;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(one));
  return one != 0;
}
__device__ __forceinline__ uint32_t uniform(uint32_t x) { return __shfl_sync(0xffffffffu, x, 0); }

__device__ __forceinline__ void tmem_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// 32 columns of the thread's TMEM lane.
__device__ __forceinline__ void tmem_load32(uint32_t addr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
      "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr));
}
__device__ __forceinline__ void tmem_store32(uint32_t addr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,"
      "%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};" ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]),
      "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]),
      "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]),
      "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]),
      "r"(r[31]), "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tmem_load_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_store_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Eight FP32 values to 32 aligned bytes.
__device__ __forceinline__ void store8f(float* p, const float* v) {
  asm volatile("st.global.v8.f32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]),
               "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7])
               : "memory");
}

// ---------------------------------------------------------------------------
// The roles.
// ---------------------------------------------------------------------------
// Every warp that walks the pieces: next piece, or false at the end (or when
// the CTA has given up).
struct PieceReader {
  int n = 0;
  __device__ __forceinline__ bool next(Control& ctl, Piece& p) {
    const int s = n % kPieces;
    if (!__all_sync(0xffffffffu, mbar_wait(ctl, &ctl.piece_full[s], (n / kPieces) & 1))) return false;
    p = ctl.piece[s];
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(&ctl.piece_empty[s]);
    ++n;
    return p.tiles > 0;
  }
};

// Q rows of a piece: one row of 512 bytes a warp instruction, into the 128-byte
// swizzle that the products read.  The softmax warps, which have nothing to do
// yet, bring the first piece's rows, a share each; the listing warp brings those
// of the pieces after it, with the addresses of four rows worked out by each lane
// beforehand.  Rows past the item's stay as they are: a row of S and O depends
// on its own Q row alone.
__device__ __forceinline__ void load_first_queries(const AttendArgs& a, Control& ctl, const Piece& p, int warp,
                                                   uint32_t q) {
  const int lane = threadIdx.x & 31;
  const uint32_t to = q + (lane >> 3) * kQChunkBytes;
  const uint16_t* rows_at = a.q + p.first * a.q_token + p.head * a.group * a.q_head + lane * 8;
#pragma unroll 4
  for (int r = warp; r < p.rows; r += kSoftmaxWarps) {
    const int in_item = p.row0 + r, tok = a.by_group.of(in_item);
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + r * 128 + (((lane & 7) ^ (r & 7)) << 4)),
                 "l"(rows_at + tok * a.q_token + (in_item - tok * a.group) * a.q_head)
                 : "memory");
  }
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&ctl.q_first)) : "memory");
}

__device__ __forceinline__ bool load_queries(const AttendArgs& a, Control& ctl, const Piece& p, uint32_t np,
                                             uint32_t q) {
  const int lane = threadIdx.x & 31;
  const uint16_t* mine[kRows / 32];
#pragma unroll
  for (int i = 0; i < kRows / 32; ++i) {
    const int in_item = p.row0 + min(i * 32 + lane, p.rows - 1);
    const int tok = a.by_group.of(in_item);
    mine[i] = a.q + (p.first + tok) * a.q_token + (p.head * a.group + in_item - tok * a.group) * a.q_head;
  }
  if (!__all_sync(0xffffffffu, mbar_wait(ctl, &ctl.q_empty, (np & 1) ^ 1))) return false;
  const uint32_t to = q + (lane >> 3) * kQChunkBytes;
#pragma unroll
  for (int i = 0; i < kRows / 32; ++i) {
    const int rows = min(p.rows - i * 32, 32);
#pragma unroll 8
    for (int r = 0; r < rows; ++r) {
      const uint64_t src = __shfl_sync(0xffffffffu, reinterpret_cast<uint64_t>(mine[i]), r) + lane * 16;
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + (i * 32 + r) * 128 +
                                                                     (((lane & 7) ^ (r & 7)) << 4)),
                   "l"(src)
                   : "memory");
    }
  }
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&ctl.q_full)) : "memory");
  return true;
}

// Units of the requests from `first` on, a request a lane and then every `step`th
// after it, one copy of the code, which nobody has run yet, for all of them.
// `kept` becomes the lane's first request.  With `hint` the arrays may not be
// written yet.
__device__ __forceinline__ LineSums add_up(const AttendArgs& a, int first, int step, bool hint, RawRequest& kept) {
  const int lane = threadIdx.x & 31;
  LineSums sums{0, 0, 0, 0};
  RawRequest next;
  if (first + lane < a.batch) next.load(a, first + lane, hint);
#pragma unroll 1
  for (int b = first + lane; b < a.batch; b += step) {
    const RawRequest raw = next;
    if (b + step < a.batch) next.load(a, b + step, hint);
    const Request r = raw.checked(a, !hint && blockIdx.x == 0);
    const int n = r.row_tiles(a);
    sums.units += r.all_units(a, -1);
    sums.row_tiles += n;
    sums.seeing += n == 0 ? 0 : r.seeing_before(a, n - 1) + (r.len > 0);
    sums.decreasing += raw.end < raw.start;
    if (b == first + lane) kept = raw;
  }
  sums.units = __reduce_add_sync(0xffffffffu, sums.units);
  sums.row_tiles = __reduce_add_sync(0xffffffffu, sums.row_tiles);
  sums.seeing = __reduce_add_sync(0xffffffffu, sums.seeing);
  sums.decreasing = __reduce_add_sync(0xffffffffu, sums.decreasing);
  return sums;
}

// Whether what was read of request `b` before the dependency wait still holds, in
// every lane; CTA 0 reports what is out of range.
__device__ __forceinline__ bool still_so(const AttendArgs& a, int b, const RawRequest& hint) {
  bool same = true;
  if (b < a.batch) {
    RawRequest now;
    now.load(a, b);
    now.checked(a, blockIdx.x == 0);
    same = now.start == hint.start && now.end == hint.end && now.len == hint.len;
  }
  return __all_sync(0xffffffffu, same);
}

// While the previous kernel may still run, a batch of a request a lane is added up
// and the CTA's first piece found from lengths and starts as they are then.  After
// the dependency wait every warp reads its requests again: if one has changed, all
// is done again from what it says now.  128 requests over a prefix, in a row of
// calls 30.4 -> 29.5 us; behind an append, which is too short to hide it, a layer's
// step 41.6 -> 42.4.
__device__ __forceinline__ bool hints(const AttendArgs& a) { return a.batch <= 32 * (1 + kSoftmaxWarps); }

// Adds up the requests' units, finds where this CTA's run begins and lists the
// run's pieces; CTA 0 also notes the line for the join.  The softmax warps, which
// have nothing to do yet, add up what is past the first 32 requests: 128 requests
// over a prefix 33.0 us with one warp for all, eight requests a lane at once, and
// 32.0 so; one request 11.1 and 10.5.
// Returns true if all has to be done again, without hints.
__device__ __forceinline__ bool list_once(const AttendArgs& a, Control& ctl, uint32_t q, bool hint) {
  const int lane = threadIdx.x & 31, cta = blockIdx.x;
  const int key_tiles = div_up(a.prefix_len, kKeys);
  bool entered = !hint, again = false;
  RawRequest first_raw{0, 0, 0};
  const int64_t end_of_last = a.query_starts == nullptr ? a.tokens
                              : hint                    ? hint_load(a.query_starts + a.batch)
                                                        : __ldg(a.query_starts + a.batch);
  LineSums sums = add_up(a, 0, 32 * (1 + kSoftmaxWarps), hint, first_raw);
  // Ends the time of hints; false if they do not hold (any more).
  auto enter = [&] {
    if (entered) return true;
    entered = true;
    pdl_enter();
    bool same = still_so(a, lane, first_raw);
    if (a.query_starts != nullptr) same = same && __ldg(a.query_starts + a.batch) == end_of_last;
    if (a.batch > 32) {
      same = __all_sync(0xffffffffu, mbar_wait(ctl, &ctl.checked, 0)) && same;
      same = same && *reinterpret_cast<volatile int32_t*>(&ctl.changed) == 0;
    }
    again = !same;
    return same;
  };
  // The 32 requests from `held` on, one a lane: its units, and with those before it in the 32.
  Request mine{0, 0, 0};
  if (lane < a.batch) mine = first_raw.checked(a, false);
  int held = 0, my_units = 0, my_sum = 0, joint = -1;
  auto hold = [&](int b0) {
    if (b0 != held) {
      held = b0;
      mine = Request{0, 0, 0};
      if (!enter()) return;
      if (b0 + lane < a.batch) {
        RawRequest raw;
        raw.load(a, b0 + lane);
        mine = raw.checked(a, false);
      }
    }
    my_units = my_sum = mine.all_units(a, joint) * a.k_heads;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, my_sum, d);
      if (lane >= d) my_sum += x;
    }
  };
  if (a.batch > 32) {
    if (!__all_sync(0xffffffffu, mbar_wait(ctl, &ctl.added, 0))) return false;
#pragma unroll
    for (int w = 0; w < kSoftmaxWarps; ++w) {
      sums.units += ctl.sums[w].units;
      sums.row_tiles += ctl.sums[w].row_tiles;
      sums.seeing += ctl.sums[w].seeing;
      sums.decreasing += ctl.sums[w].decreasing;
    }
  }
  // Starts that decrease would let many requests claim the same tokens, more work
  // than any batch of this size has: nothing is done then.
  const int used = sums.decreasing ? 0 : int(clamp64(end_of_last, 0, a.tokens));
  const int row_tiles = div_up(used * a.group, kRows);
  int total = sums.decreasing ? 0 : sums.units;
  int pre = prefix_units(a, used);
  if (pre > 0) {
    // The shorter line: row tiles of all requests together against the prefix and of
    // each against its own keys, or of each against both.  2560 query tokens of four
    // requests over 8192 shared keys: 136 us apart, 119 in one, with no partial results
    // but of cut items.
    const int64_t both = int64_t(sums.row_tiles) * (key_tiles + kItemCost) - int64_t(sums.seeing) * kItemCost;
    if (both * a.k_heads <= pre) {
      joint = key_tiles;
      total += int(both);
      pre = 0;
    }
  }
  const Line line(pre + total * a.k_heads, a.grid);
  int n = 0;
  // every lane holds the piece; lane 0 writes it
  auto emit = [&](const Piece& p) {
    if (!enter()) return false;
    const int s = n % kPieces;
    const bool ok = __all_sync(0xffffffffu, mbar_wait(ctl, &ctl.piece_empty[s], ((n / kPieces) & 1) ^ 1));
    if (!ok) return false;
    if (lane == 0) {
      ctl.piece[s] = p;
      mbar_arrive(&ctl.piece_full[s]);
    }
    // this waits for the piece before: the other warps know one piece ahead
    const bool loaded = n == 0 || p.tiles == 0 || load_queries(a, ctl, p, n, q);
    ++n;
    return loaded;
  };
  const bool works = cta < line.grid;
  bool ok = true;
  int u = works ? line.begin(cta) : 0;
  const int end = works ? line.begin(cta + 1) : 0;
  while (ok && u < end && u < pre) {
    const int item = u / (key_tiles + kItemCost);
    const int at = u - item * (key_tiles + kItemCost), step = min(end - u, key_tiles + kItemCost - at);
    u += step;
    Piece p;
    p.first_tile = max(at - kItemCost, 0);
    p.tiles = at + step - kItemCost - p.first_tile;
    if (p.tiles <= 0) continue;
    p.keys = a.prefix_len;
    p.head = item / row_tiles;
    p.row0 = (item - p.head * row_tiles) * kRows;
    p.rows = min(used * a.group - p.row0, kRows);
    p.first = 0;
    p.seen0 = a.prefix_len;
    p.own = 0;
    p.shared_tiles = key_tiles;
    p.table_row = 0;
    p.once = 0;
    p.to = p.tiles == key_tiles ? kToPart : kToSlot;
    p.slot = 2 * cta + (p.first_tile > 0 ? 0 : 1);
    ok = emit(p);
  }
  int held_base = pre;  // units before the 32 requests in hand
  if (u < end) hold(0);
  while (ok && u < end) {
    const uint32_t past = __ballot_sync(0xffffffffu, u < held_base + my_sum);
    if (past == 0) {  // none of these 32
      held_base += __shfl_sync(0xffffffffu, my_sum, 31);
      if (held + 32 >= a.batch) break;
      hold(held + 32);
      if (again) break;
      continue;
    }
    const int i = __ffs(past) - 1, b = held + i;
    int base = held_base + __shfl_sync(0xffffffffu, my_sum - my_units, i);  // of request b
    const Request r{__shfl_sync(0xffffffffu, mine.first, i), __shfl_sync(0xffffffffu, mine.count, i),
                    __shfl_sync(0xffffffffu, mine.len, i)};
    const int rts = r.row_tiles(a);
    int rt = 0;
    if (rts > 1 && u > base) {  // the last row tile that begins at or before u
      int hi = rts;
      while (hi - rt > 1) {
        const int mid = (rt + hi) >> 1;
        if (base + a.k_heads * r.units_before(a, mid, joint) <= u) rt = mid; else hi = mid;
      }
      base += a.k_heads * r.units_before(a, rt, joint);
    }
    for (; ok && rt < rts && u < end; ++rt) {
      const int cost = Request::units(r.tiles(a, rt), joint);
      for (int h = 0; ok && h < a.k_heads && u < end; ++h, base += cost) {
        if (u >= base + cost) continue;
        const int at = u - base, step = min(end - u, cost - at);
        u += step;
        Piece p;
        p.first_tile = max(at - kItemCost, 0);
        p.tiles = at + step - kItemCost - p.first_tile;
        if (p.tiles <= 0) continue;
        p.keys = r.seen(a, rt);
        p.head = h;
        p.row0 = rt * kRows;
        p.rows = min(r.count * a.group - p.row0, kRows);
        p.first = r.first;
        p.seen0 = r.len - r.count + 1;
        p.own = 1;
        p.shared_tiles = max(joint, 0);
        p.table_row = b;
        p.once = rts == 1;
        p.to = p.tiles < cost - kItemCost ? kToSlot : pre > 0 ? kToPart : kToOutput;
        p.slot = 2 * cta + (p.first_tile > 0 ? 0 : 1);
        ok = emit(p);
      }
    }
  }
  if (ok && !again) emit(Piece{});
  if (again) return true;
  asm volatile("cp.async.wait_all;" ::: "memory");
  if (lane == 0) a.gave_up[cta] = 0;  // now, so that the kernel's end does not wait for it
  if (cta != 0) return false;
  // for the join: every request's place on the line
  int before = 0;
  for (int b0 = 0; b0 < a.batch; b0 += 32) {
    hold(b0);
    if (b0 + lane < a.batch) a.units_before[b0 + lane] = before + my_sum - my_units;
    before += __shfl_sync(0xffffffffu, my_sum, 31);
  }
  if (lane == 0) {
    LineNote note;
    note.pre = pre;
    note.joint = joint;
    note.nothing = sums.decreasing > 0;
    note.each = line.each;
    note.more = line.more;
    note.by_each = Divisor(max(line.each, 1));
    note.by_longer = Divisor(line.each + 1);
    *a.note = note;
  }
  return false;
}

__device__ void list_pieces(const AttendArgs& a, Control& ctl, uint32_t q) {
  bool hint = hints(a);
  if (!hint) pdl_enter();
  while (list_once(a, ctl, q, hint)) hint = false;
}

// Where a box of keys is in the cache.  The block is looked at when its copies
// are issued, a tile after it was asked for, and not as soon as it is there.
struct BoxPlace {
  int block = 0, place = 0;
  bool keys = false;  // some row sees keys of the box
  __device__ __forceinline__ void ask(const AttendArgs& a, const Piece& p, const int32_t* own, int j, int box_keys) {
    const int tile = p.first_tile + j, at = (threadIdx.x & 31) * box_keys;
    const bool shared = tile < p.shared_tiles;
    const int key = (shared ? tile : tile - p.shared_tiles) * kKeys + at;
    keys = j < p.tiles && at < kKeys && key < (shared ? a.prefix_len : p.keys);
    if (!keys) return;
    const int page = a.by_block.of(key);
    place = key - page * a.block_size;
    block = __ldg((shared ? a.prefix_table : own) + page);
  }
  // The block past the cache, whose box is filled with zeros, for boxes behind the keys and blocks that do not exist.
  __device__ __forceinline__ int checked(const AttendArgs& a) const {
    const bool there = uint32_t(block) < uint32_t(a.num_blocks);
    if (keys && !there) raise_status(a.status, WELM_ROPE_DEV_BAD_PAGE);
    return keys && there ? block : a.num_blocks;
  }
};

// After a failed wait, the copies in flight still have to land.
template <int kStages>
__device__ __forceinline__ void await_copies(Control& ctl, uint64_t* full, uint32_t n) {
  if (*reinterpret_cast<volatile int32_t*>(&ctl.failed) == 0) return;
  for (uint32_t i = n > kStages ? n - kStages : 0; i < n; ++i) {
    const long long t0 = clock64();
    while (!mbar_poll(&full[i % kStages], (i / kStages) & 1) && clock64() - t0 < kWaitClocks) {
    }
  }
}

// The producer warp.  Half a K tile is [2 chunks of 64 lanes][128 keys][128
// bytes]: its products take all keys at once.  Half a V tile is 64 keys,
// [boxes][4 chunks of 64 lanes][box_v keys][128 bytes]: one copy brings all
// lanes of a box.  Lane g of the warp looks up the block of the tile's g-th box
// of K, and of V, one tile ahead, and issues that box's copies.
__device__ void produce(const AttendArgs& a, Control& ctl, const CUtensorMap* kmap, const CUtensorMap* vmap,
                        uint32_t k_at, uint32_t v_at) {
  const int lane = threadIdx.x & 31;
  const int boxes_k = kKeys / a.box_k, boxes_v = kHalfKeys / a.box_v;
  const int v_half = lane < boxes_v ? 0 : lane < 2 * boxes_v ? 1 : 2;  // the half of V that the lane's box is in
  const uint32_t my_k = k_at + lane * a.box_k * 128;
  const uint32_t my_v = v_at + (lane - v_half * boxes_v) * a.box_v * (kHeadDim * 2);
  // Keys that one item alone reads leave L2 first, so that the prefix's, which many
  // CTAs read from there, stay: with L2 cold, 48 requests' own 95 MB 39.9 -> 33.8 us,
  // 256 requests over 32768 shared keys 91.1 -> 87.0.
  uint64_t first_out, as_usual;
  asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(first_out));
  asm("createpolicy.fractional.L2::evict_normal.b64 %0, 1.0;" : "=l"(as_usual));
  PieceReader pieces;
  Piece p;
  uint32_t nk = 0, nv = 0;  // halves so far
  bool ok = true;
  while (ok && pieces.next(ctl, p)) {
    const int32_t* own = a.block_table + p.table_row * a.table_stride;
    BoxPlace at_k, at_v, next_k, next_v;
    at_k.ask(a, p, own, 0, a.box_k);
    for (int j = 0; j <= p.tiles && ok; ++j) {
      const uint64_t policy_k = p.once && p.first_tile + j >= p.shared_tiles ? first_out : as_usual;
      const uint64_t policy_v = p.once && p.first_tile + j > p.shared_tiles ? first_out : as_usual;
      if (j < p.tiles) {
        const int block = at_k.checked(a);
#pragma unroll 1
        for (int half = 0; half < 2; ++half, ++nk) {
          const uint32_t s = nk % kStagesK;
          ok = ok && __all_sync(0xffffffffu, mbar_wait(ctl, &ctl.empty_k[s], ((nk / kStagesK) & 1) ^ 1));
          if (!ok) break;
          if (lane == 0) mbar_arm(&ctl.full_k[s], kStageBytes);
          __syncwarp();
          if (lane < boxes_k) {
#pragma unroll
            for (int c = 0; c < 2; ++c)
              asm volatile(
                  "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint "
                  "[%0], [%1, {%2, %3, %4, %5}], [%6], %7;" ::"r"(my_k + s * kStageBytes + c * kChunkBytes),
                  "l"(kmap), "r"(half * kHalfLanes + c * 64), "r"(at_k.place), "r"(p.head), "r"(block),
                  "r"(smem_u32(&ctl.full_k[s])), "l"(policy_k)
                  : "memory");
          }
        }
      }
      next_k.ask(a, p, own, j + 1, a.box_k);
      next_v.ask(a, p, own, j, a.box_v);
      if (j > 0) {
        const int block = at_v.checked(a);
#pragma unroll 1
        for (int half = 0; half < 2; ++half, ++nv) {
          const uint32_t s = nv % kStagesV;
          ok = ok && __all_sync(0xffffffffu, mbar_wait(ctl, &ctl.empty_v[s], ((nv / kStagesV) & 1) ^ 1));
          if (!ok) break;
          if (lane == 0) mbar_arm(&ctl.full_v[s], kStageBytes);
          __syncwarp();
          if (v_half == half)
            asm volatile(
                "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint "
                "[%0], [%1, {%2, %3, %2, %4, %5}], [%6], %7;" ::"r"(my_v + s * kStageBytes),
                "l"(vmap), "r"(0), "r"(at_v.place), "r"(p.head), "r"(block), "r"(smem_u32(&ctl.full_v[s])),
                "l"(policy_v)
                : "memory");
        }
      }
      at_k = next_k;
      at_v = next_v;
    }
  }
  await_copies<kStagesK>(ctl, ctl.full_k, nk);
  await_copies<kStagesV>(ctl, ctl.full_v, nv);
}

// No product may outlive the TMEM or the shared memory it works on.
__device__ __forceinline__ void drain(uint64_t* bar) {
  if (elect_one()) mma_commit(bar);
  __syncwarp();
  const long long t0 = clock64();
  while (!mbar_poll(bar, 0) && clock64() - t0 < kWaitClocks) {
  }
}

// Two warps issue the products, so that what one waits for does not hold up the
// other's (both waits take some 300 clocks even when they are over).
//
// The products of a tile take 2050 clocks by themselves.  Beside the copies they
// take 2600 to 2800: those of the scores read Q and K from shared memory at 128
// bytes a clock, all that it has, so that a tile's 128 KB (Q, K), 64 KB (V) and
// 128 KB of copies written make 2500.
//
// S(t) = Q K(t)^T, once what its columns held before has been used: S(t - 1)
// read, but for the second of three tiles, and the products with P(t - 3) done, or
// for the second with P(t - 2); the third's wait for S(t - 1) says so too.
__device__ void issue_scores(Control& ctl, uint32_t q, uint32_t ring, uint32_t tmem) {
  constexpr uint32_t kIdesc = instr_desc(kKeys, false);
  const uint64_t q_desc = operand_desc(q, 16, 1024);
  PieceReader pieces;
  Piece p;
  uint32_t t = 0, n = 0, third = 0;  // tiles and halves of K so far; t % 3
  bool ok = true;
  for (uint32_t np = 0; ok && pieces.next(ctl, p); ++np) {
    const int tiles = int(uniform(p.tiles));
    for (int j = 0; ok && j < tiles; ++j, ++t, third = third == 2 ? 0 : third + 1) {
      const uint32_t buf = t & 1;
      const uint32_t d = uniform(tmem + col_s(third));
      if (j == 0) {
        ok = np == 0 ? mbar_wait(ctl, &ctl.q_first, 0) : mbar_wait(ctl, &ctl.q_full, (np & 1) ^ 1);
        // the Q rows came by ordinary asynchronous copies
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      }
#pragma unroll
      for (int half = 0; half < 2; ++half, ++n) {
        const uint32_t s = uniform(n % kStagesK);
        const uint64_t k_desc = operand_desc(ring + s * kStageBytes, 16, 1024);
        ok = ok && mbar_wait(ctl, &ctl.full_k[s], (n / kStagesK) & 1);
        if (half == 0) {
          const uint32_t used = t - (third == 1 ? 2 : 3), read = t - 1;
          if (third < 2 && t >= 3) ok = ok && mbar_wait(ctl, &ctl.pv_done[used & 3], (used >> 2) & 1);
          if (third != 1 && t >= 2) ok = ok && mbar_wait(ctl, &ctl.s_read[read & 1], (read >> 1) & 1);
        }
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tmem_fence_after();
        if (elect_one()) {
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              mma_ss(d, q_desc + (((2 * half + c) * kQChunkBytes + kk * 32) >> 4),
                     k_desc + ((c * kChunkBytes + kk * 32) >> 4), kIdesc, half + c + kk > 0);
          if (half == 1) mma_commit(&ctl.s_full[buf]);
          mma_commit(&ctl.empty_k[s]);
          if (half == 1 && j == tiles - 1) mma_commit(&ctl.q_empty);
        }
        __syncwarp();
      }
    }
  }
  if (t > 0) drain(&ctl.drained[0]);
}

// O += P(t) V(t).
__device__ void issue_values(const AttendArgs& a, Control& ctl, uint32_t ring, uint32_t tmem) {
  constexpr uint32_t kIdesc = instr_desc(kHeadDim, true);
  // 16 keys, a product's, lie in one box, or in two boxes of eight
  const uint32_t box = uniform(a.box_v);
  const uint32_t lead = box * 128, stride = box > 8 ? 1024 : 4096;
  const uint32_t per = box > 8 ? box / 16 : 1;  // products of a box
  uint32_t at[kHalfKeys / 16];
#pragma unroll
  for (uint32_t ks = 0; ks < kHalfKeys / 16; ++ks) at[ks] = (ks / per * per * 16 * 512 + ks % per * 16 * 128) >> 4;
  PieceReader pieces;
  Piece p;
  uint32_t t = 0, n = 0, third = 0;
  bool ok = true;
  for (uint32_t np = 0; ok && pieces.next(ctl, p); ++np) {
    const int tiles = int(uniform(p.tiles));
    for (int j = 0; ok && j < tiles; ++j, ++t, third = third == 2 ? 0 : third + 1) {
      const uint32_t buf = t & 3;
      const uint32_t p_at = uniform(tmem + col_p(third));
#pragma unroll
      for (int half = 0; half < 2; ++half, ++n) {
        const uint32_t s = uniform(n % kStagesV);
        const uint64_t v_desc = operand_desc(ring + s * kStageBytes, lead, stride);
        ok = ok && mbar_wait(ctl, &ctl.full_v[s], (n / kStagesV) & 1);
        if (half == 0)
          ok = ok && (j > 0 || mbar_wait(ctl, &ctl.o_free, (np & 1) ^ 1)) &&
               mbar_wait(ctl, &ctl.p_full[buf], (t >> 2) & 1);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tmem_fence_after();
        if (elect_one()) {
#pragma unroll
          for (int ks = 0; ks < kHalfKeys / 16; ++ks)
            mma_ts(tmem + kColO, p_at + half * 32 + ks * 8, v_desc + at[ks], kIdesc, j + half + ks > 0);
          if (half == 1) mma_commit(&ctl.pv_done[buf]);
          mma_commit(&ctl.empty_v[s]);
        }
        __syncwarp();
      }
    }
  }
  if (t > 0) drain(&ctl.drained[1]);
}

// Softmax of the tiles, rescaling of O, and the results.  Two threads hold a
// row: the first four warps its keys 0..63 of a tile and lanes 0..127 of O,
// the others the rest; they swap maxima, so both come to the same ones.
__device__ void softmax_rows(const AttendArgs& a, Control& ctl, Swap& swap, uint32_t q, uint8_t* ring,
                             uint32_t tmem) {
  const int lane = threadIdx.x & 31;
  const int warp = ((threadIdx.x >> 5) - kSoftmaxWarp0) & 3;
  const int half = (threadIdx.x >> 5) >= kSoftmaxWarp0 + 4;
  const int row = warp * 32 + lane;
  const uint32_t mine = tmem + (uint32_t(warp * 32) << 16);
  const uint32_t my_o = mine + kColO + half * kHalfLanes;
  const float c = a.scale;
  if (a.batch <= 32) {
    pdl_enter();
  } else {
    const int w = (threadIdx.x >> 5) - kSoftmaxWarp0;
    bool hint = hints(a);
    if (!hint) pdl_enter();
    for (int pass = 0;; ++pass) {
      RawRequest first{0, 0, 0};
      const LineSums sums = add_up(a, 32 * (1 + w), 32 * (1 + kSoftmaxWarps), hint, first);
      if (lane == 0) {
        ctl.sums[w] = sums;
        if (pass == 0) mbar_arrive(&ctl.added);
      }
      bool same = true;
      if (hint) {
        pdl_enter();
        same = still_so(a, 32 * (1 + w) + lane, first);
        hint = false;
        if (!same && lane == 0) *reinterpret_cast<volatile int32_t*>(&ctl.changed) = 1;
      }
      if (same) break;
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(&ctl.checked);
  }
  PieceReader pieces;
  Piece p;
  uint32_t tile = 0, third = 0, swaps = 0;
  // hands `value` to the row's other thread and returns that thread's
  auto trade = [&](float value, float& other) {
    const uint32_t parity = swaps & 1;
    swap.value[parity][half][row] = value;
    __syncwarp();
    if (lane == 0) mbar_arrive(&ctl.swap[warp]);
    if (!__all_sync(0xffffffffu, mbar_wait(ctl, &ctl.swap[warp], parity))) return false;
    other = swap.value[parity][half ^ 1][row];
    ++swaps;
    return true;
  };
  for (; pieces.next(ctl, p); tile += p.tiles) {
    if (tile == 0) load_first_queries(a, ctl, p, (threadIdx.x >> 5) - kSoftmaxWarp0, q);
    const bool busy = warp * 32 < p.rows;  // some lane of the warp has a row
    const int in_item = p.row0 + row;
    const int tok = a.by_group.of(in_item);
    int seen = p.own ? p.seen0 + tok : p.seen0;
    if (seen > p.keys) seen = p.keys;
    // keys from the piece's first tile on, counted from this thread's half of a tile:
    // the prefix's, the request's that the row sees, the request's that any row sees
    const int in_shared = p.shared_tiles - p.first_tile, behind = p.first_tile * kKeys + half * kHalfKeys;
    const int shared_left = a.prefix_len - behind;
    const int own_left = seen - behind + p.shared_tiles * kKeys, all_left = own_left - seen + p.keys;
    float m = -INFINITY, l = 0.0f;
    for (int j = 0; j < p.tiles; ++j) {
      const uint32_t t = tile + j, buf = t & 1;
      const uint32_t my_s = mine + col_s(third) + half * 64, my_p = mine + col_p(third) + half * 32;
      third = third == 2 ? 0 : third + 1;
      if (!__all_sync(0xffffffffu, mbar_wait(ctl, &ctl.s_full[buf], (t >> 1) & 1))) return;
      tmem_fence_after();
      if (!busy && lane == 0) mbar_arrive(&ctl.s_read[buf]);
      if (busy) {
        uint32_t s[2][32];
        tmem_load32(my_s, s[0]);
        tmem_load32(my_s + 32, s[1]);
        tmem_load_wait();
        tmem_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&ctl.s_read[buf]);
        // of these 64 keys, those that the row sees
        const int left = (j < in_shared ? shared_left : own_left) - j * kKeys;
        if (left < 64) {
#pragma unroll
          for (int i = 0; i < 64; ++i)
            if (i >= left) s[i >> 5][i & 31] = 0xff800000u;
        }
        float tops[4] = {m, m, m, m};
#pragma unroll
        for (int i = 0; i < 64; ++i) tops[i & 3] = fmaxf(tops[i & 3], __uint_as_float(s[i >> 5][i & 31]));
        float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])), other;
        if (!trade(top, other)) return;
        top = fmaxf(top, other);
        // The maximum in use only moves when it has grown enough to matter:
        // until then p stays at or below 2^8, well inside BF16 and FP32.
        // Rows past the item's, whose scores may be anything, do not ask for it.
        const bool grown = row < p.rows && (top - m) * c > kRescaleStep;
        if (j > 0 && __any_sync(0xffffffffu, grown)) {
          const uint32_t tp = t - 1;
          if (!__all_sync(0xffffffffu, mbar_wait(ctl, &ctl.pv_done[tp & 3], (tp >> 2) & 1))) return;
          tmem_fence_after();
          const float f = grown ? exp2_approx((m - top) * c) : 1.0f;
          l *= f;
#pragma unroll 1
          for (int g = 0; g < kHalfLanes / 32; ++g) {
            uint32_t o[32];
            tmem_load32(my_o + g * 32, o);
            tmem_load_wait();
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
            tmem_store32(my_o + g * 32, o);
          }
          tmem_store_wait();
          if (grown) m = top;
        } else if (j == 0) {
          m = top;
        }
        const float mc = m == -INFINITY ? 0.0f : m * c;  // nothing seen yet: every p is 0
        uint32_t pk[32];
        float sums[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < 64; i += 2) {
          const float p0 = exp2_approx(fmaf(__uint_as_float(s[i >> 5][i & 31]), c, -mc));
          const float p1 = exp2_approx(fmaf(__uint_as_float(s[i >> 5][(i & 31) + 1]), c, -mc));
          sums[i & 2] += p0;
          sums[(i & 2) + 1] += p1;
          pk[i / 2] = pack_bf16x2(p0, p1);
        }
        l += (sums[0] + sums[1]) + (sums[2] + sums[3]);
        // of columns that the row's other thread may have had in S: it had read them when it gave its maximum
        __syncwarp();
        tmem_store32(my_p, pk);
        tmem_store_wait();
      }
      // V rows past the keys weigh nothing, but what their page holds may be
      // no number, and 0 times that is none either: they are cleared.  Boxes
      // that begin behind the keys were filled with zeros.
      const int whole = (j < in_shared ? shared_left : all_left) - j * kKeys;
      if (whole < kHalfKeys) {
        // V(t - 1), the stage's last contents, has landed if it has been used
        if (t > 0 && !__all_sync(0xffffffffu, mbar_wait(ctl, &ctl.pv_done[(t - 1) & 3], ((t - 1) >> 2) & 1))) return;
        const uint32_t n = 2 * t + half, st = n % kStagesV;
        if (!__all_sync(0xffffffffu, mbar_wait(ctl, &ctl.full_v[st], (n / kStagesV) & 1))) return;
        uint8_t* v = ring + (kStagesK + st) * kStageBytes;
        const int begin = max(whole, 0), end = div_up(begin, a.box_v) * a.box_v;
        for (int i = begin * 32 + row; i < end * 32; i += kRows) {
          const int key = i >> 5, box = key & ~(a.box_v - 1);
          *reinterpret_cast<uint4*>(v + box * 512 + ((i >> 3) & 3) * a.box_v * 128 + (key - box) * 128 + (i & 7) * 16) =
              make_uint4(0, 0, 0, 0);
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      }
      tmem_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&ctl.p_full[t & 3]);
    }
    // O of the piece
    const uint32_t tl = tile + p.tiles - 1;
    if (!__all_sync(0xffffffffu, mbar_wait(ctl, &ctl.pv_done[tl & 3], (tl >> 2) & 1))) return;
    tmem_fence_after();
    if (busy) {
      float other;
      if (!trade(l, other)) return;
      l = half ? other + l : l + other;
      const bool live = row < p.rows;
      const int64_t token = p.first + tok;
      const int head = p.head * a.group + (in_item - tok * a.group);
      if (p.to == kToOutput) {
        uint16_t* out = a.out + token * a.out_token + head * a.out_head + half * kHalfLanes;
        const float scale_out = l == 0.0f ? 0.0f : 1.0f / l;
        if (live && half == 0 && a.lse != nullptr)
          a.lse[token * a.q_heads + head] = l == 0.0f ? -INFINITY : (m * c + log2f(l)) * 0.6931471805599453f;
#pragma unroll 1
        for (int g = 0; g < kHalfLanes / 32; ++g) {
          uint32_t o[32];
          __syncwarp();
          tmem_load32(my_o + g * 32, o);
          tmem_load_wait();
          if (!live) continue;
          uint4* dst = reinterpret_cast<uint4*>(out + g * 32);
#pragma unroll
          for (int i = 0; i < 32; i += 8) {
            float f[8];
#pragma unroll
            for (int x = 0; x < 8; ++x) f[x] = l == 0.0f ? 0.0f : __uint_as_float(o[i + x]) * scale_out;
            dst[i / 8] = make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]),
                                    pack_bf16x2(f[6], f[7]));
          }
        }
      } else {
        const int64_t all = int64_t(a.tokens) * a.q_heads;
        const int64_t at = p.to == kToSlot ? int64_t(p.slot) * a.slot_rows + row
                                           : (p.own * a.k_heads + p.head) * (int64_t(a.tokens) * a.group) +
                                                 p.first * int64_t(a.group) + in_item;
        const int64_t rows = p.to == kToSlot ? a.slot_rows : all;  // from one group of eight lanes to the next
        float* to = p.to == kToSlot ? a.slot_o + (int64_t(p.slot) * 32 * a.slot_rows + row) * 8
                                    : a.part_o + (p.own * 32 * all + at - p.own * all) * 8;
        to += half * 16 * rows * 8;
        if (live && half == 0)
          *reinterpret_cast<float2*>((p.to == kToSlot ? a.slot_ml : a.part_ml) + at * 2) =
              make_float2(m == -INFINITY ? m : m * c, l);
#pragma unroll 1
        for (int g = 0; g < kHalfLanes / 32; ++g) {
          uint32_t o[32];
          __syncwarp();
          tmem_load32(my_o + g * 32, o);
          tmem_load_wait();
          if (!live) continue;
#pragma unroll
          for (int i = 0; i < 32; i += 8) {
            float f[8];
#pragma unroll
            for (int x = 0; x < 8; ++x) f[x] = __uint_as_float(o[i + x]);
            store8f(to + (g * 4 + i / 8) * rows * 8, f);
          }
        }
      }
      __syncwarp();
    }
    tmem_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(&ctl.o_free);
  }
}

__global__ void __launch_bounds__(kThreads, 1)
    rope_attend_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                       const __grid_constant__ AttendArgs a) {
  extern __shared__ __align__(1024) uint8_t smem[];  // the 128-byte swizzle repeats every 1024 bytes
  uint8_t* ring = smem + kQBytes;
  Swap& swap = *reinterpret_cast<Swap*>(ring + (kStagesK + kStagesV) * kStageBytes);
  Control& ctl = *reinterpret_cast<Control*>(&swap + 1);
  const int tid = threadIdx.x, warp = tid >> 5;
  if (tid == 0) {
    for (int s = 0; s < kStagesK; ++s) {
      mbar_init(&ctl.full_k[s], 1);
      mbar_init(&ctl.empty_k[s], 1);
    }
    for (int s = 0; s < kStagesV; ++s) {
      mbar_init(&ctl.full_v[s], 1);
      mbar_init(&ctl.empty_v[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&ctl.s_full[i], 1);
      mbar_init(&ctl.s_read[i], kSoftmaxWarps);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(&ctl.p_full[i], kSoftmaxWarps);
      mbar_init(&ctl.pv_done[i], 1);
    }
    mbar_init(&ctl.q_first, 32 * kSoftmaxWarps);
    mbar_init(&ctl.added, kSoftmaxWarps);
    mbar_init(&ctl.checked, kSoftmaxWarps);
    mbar_init(&ctl.q_full, 32);
    mbar_init(&ctl.q_empty, 1);
    mbar_init(&ctl.o_free, kSoftmaxWarps);
    for (int i = 0; i < 2; ++i) mbar_init(&ctl.drained[i], 1);
    for (int i = 0; i < 4; ++i) mbar_init(&ctl.swap[i], 2);
    for (int i = 0; i < kPieces; ++i) {
      mbar_init(&ctl.piece_full[i], 1);
      mbar_init(&ctl.piece_empty[i], kPieceReaders);
    }
    ctl.failed = a.give_up;
    ctl.changed = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 0 && elect_one()) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(&kmap) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&vmap) : "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&ctl.tmem))
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tmem_fence_before();
  __syncthreads();
  tmem_fence_after();
  const uint32_t tmem = ctl.tmem;
  const uint32_t q_at = smem_u32(smem), k_at = smem_u32(ring), v_at = k_at + kStagesK * kStageBytes;
  if (warp < 3) pdl_enter();  // the others first look at hints
  if (warp == 0) {
    produce(a, ctl, &kmap, &vmap, k_at, v_at);
  } else if (warp == 1) {
    issue_scores(ctl, q_at, k_at, uniform(tmem));
  } else if (warp == 2) {
    issue_values(a, ctl, v_at, uniform(tmem));
  } else if (warp == 3) {
    list_pieces(a, ctl, q_at);
  } else {
    softmax_rows(a, ctl, swap, q_at, ring, tmem);
    asm volatile("cp.async.wait_all;" ::: "memory");
  }
  tmem_fence_before();
  __syncthreads();
  if (tid == 0 && ctl.failed) {
    a.gave_up[blockIdx.x] = 1;
    raise_status(a.status, WELM_ROPE_DEV_WAIT_TIMEOUT);
  }
  if (warp == 1) {
    tmem_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  }
}

// ---------------------------------------------------------------------------
// Joining the partial results of a row, eight lanes of the head a thread.  128
// threads hold four neighbouring rows, four of them a 128-byte line of the
// partial results' layout.  With kGroups > 1 a CTA joins four rows and its
// groups of 128 threads take the rows' partial results in turn (few rows, which
// may have many); with kGroups == 1 a CTA of two such groups joins 32 rows.
// The first threads work out where the parts of the CTA's rows are, a row each.
// ---------------------------------------------------------------------------
struct RowParts {
  int cta[2], count[2], in_tile[2];  // prefix and own item: first CTA, CTAs, row of the item
  int live;                          // 1: this kernel writes the row
  int unused;                        // 1: a row of no request
  int token, head;
};

// The last request that starts at or before `token`, found by the whole CTA before
// the dependency wait: a hint.
__device__ __forceinline__ int find_request(const AttendArgs& a, int token, int& shared) {
  if (a.query_starts == nullptr) return token;
  if (threadIdx.x == 0) shared = 0;
  __syncthreads();
  int last = -1;
  for (int b = threadIdx.x; b < a.batch; b += blockDim.x)
    if (hint_load(a.query_starts + b) <= token) last = b;
  last = __reduce_max_sync(0xffffffffu, last);
  if ((threadIdx.x & 31) == 0 && last > 0) atomicMax(&shared, last);
  __syncthreads();
  return shared;
}

// The last request from `b` on that starts at or before `token`.
__device__ __forceinline__ int request_from(const AttendArgs& a, int token, int b, bool hint) {
  if (a.query_starts == nullptr) return token;
  while (b + 1 < a.batch &&
         (hint ? hint_load(a.query_starts + b + 1) : __ldg(a.query_starts + b + 1)) <= token)
    ++b;
  return b;
}

// `b`: the row's request, as far as was known before the dependency wait.
__device__ __forceinline__ RowParts find_parts(const AttendArgs& a, const LineNote& note, int used, int flat, int b) {
  RowParts r{};
  if (flat >= a.tokens * a.q_heads) return r;
  const int token = a.by_q_heads.of(flat), hq = flat - token * a.q_heads;
  const int h = a.by_group.of(hq), g = hq - h * a.group;
  r.token = token;
  r.head = hq;
  // all that has to be read at once, before any of it is looked at
  RawRequest raw;
  raw.load(a, b);
  int units_before = a.units_before[b];
  Request q = raw.checked(a, false);
  if (!note.nothing && token < used && (token < q.first || token >= q.first + q.count)) {
    b = request_from(a, token, 0, false);
    raw.load(a, b);
    units_before = a.units_before[b];
    q = raw.checked(a, false);
  }
  if (note.nothing || token >= used || token < q.first || token >= q.first + q.count) {  // a row of no request
    r.live = a.fill;
    r.unused = 1;
    return r;
  }
  const int pre = note.pre;
  auto place = [&](int x, int first, int tiles, int in_tile) {
    r.in_tile[x] = in_tile;
    if (tiles == 0) return;
    // Within the line whatever is read here: lengths that another stream changes
    // between the two kernels give wrong rows, but no address outside the workspace.
    auto cta = [&](int u) { return min(max(note.cta_of(u), 0), a.grid - 1); };
    r.cta[x] = cta(first + kItemCost);
    r.count[x] = max(cta(first + kItemCost + tiles - 1) - r.cta[x] + 1, 0);
  };
  if (pre > 0) {
    const int packed = token * a.group + g, key_tiles = div_up(a.prefix_len, kKeys);
    place(0, (h * div_up(used * a.group, kRows) + packed / kRows) * (key_tiles + kItemCost), key_tiles, packed % kRows);
  }
  const int packed = (token - q.first) * a.group + g, rt = packed / kRows;
  const int units = Request::units(q.tiles(a, rt), note.joint);
  place(1, pre + units_before + q.units_before(a, rt, note.joint) * a.k_heads + h * units,
        max(units - kItemCost, 0), packed % kRows);
  r.live = pre > 0 || r.count[1] != 1;  // otherwise the first kernel wrote the row
  return r;
}

// Where a CTA of the first kernel gave up, the note and the partial results may be
// whatever the workspace held before, and rows may not have been written: none of
// it is read, and every row of a request becomes no number.  Apart from the join, so
// that it costs that no registers.
__device__ __noinline__ void no_numbers(const AttendArgs& a, int first_row, int rows) {
  const int used = used_tokens(a);
  for (int i = threadIdx.x; i < rows * 32; i += blockDim.x) {
    const int flat = first_row + (i >> 5), lanes8 = i & 31;
    if (flat >= a.tokens * a.q_heads) continue;
    const int token = a.by_q_heads.of(flat), head = flat - token * a.q_heads;
    RawRequest raw;
    raw.load(a, request_from(a, token, 0, false));
    const Request q = raw.checked(a, false);
    const bool asked = token < used && token >= q.first && token < q.first + q.count;
    if (a.lse != nullptr && lanes8 == 0) a.lse[flat] = __int_as_float(asked ? 0x7fc00000 : 0xff800000);
    if (!asked && !a.fill) continue;
    const uint32_t v = asked ? 0x7fc07fc0u : 0u;
    *reinterpret_cast<uint4*>(a.out + token * a.out_token + head * a.out_head + lanes8 * 8) = make_uint4(v, v, v, v);
  }
}

// Running join of partial results (m, l, eight lanes of O).
struct Joined {
  float m = -INFINITY, l = 0.0f;
  float o[8] = {};
  __device__ __forceinline__ void add(float m1, float l1, const float (&v)[8]) {
    if (m1 == -INFINITY && l1 == 0.0f) return;  // saw no key
    const float top = fmaxf(m, m1);
    const float base = top == -INFINITY ? 0.0f : top;
    const float f0 = exp2_approx(m - base), f1 = exp2_approx(m1 - base);
    l = l * f0 + l1 * f1;
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = o[i] * f0 + v[i] * f1;
    m = top;
  }
};

__device__ __forceinline__ void load8f(const float* p, float (&v)[8]) {
  asm volatile("ld.global.v8.f32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7])
               : "l"(p)
               : "memory");
}

template <int kGroups, int kUnroll, int kResident>
__global__ void __launch_bounds__(kGroups == 1 ? 256 : 128 * kGroups, kResident)
    rope_attend_join_kernel(const __grid_constant__ AttendArgs a) {
  constexpr int kRowsPerCta = kGroups == 1 ? 32 : 4;
  __shared__ RowParts parts[kRowsPerCta];
  __shared__ int s_request;
  __shared__ float s_o[kGroups == 1 ? 1 : kGroups - 1][kGroups == 1 ? 1 : 10][128];
  const int grp = threadIdx.x >> 7, in_grp = threadIdx.x & 127;
  const int lanes8 = in_grp >> 2;  // eight lanes of the head
  // The next kernel may already take the SMs that the first one has left: one
  // request 10.3 -> 9.7 us in a row of calls, 24 requests' verification 21.5 -> 22.0;
  // between an append and a projection no difference.
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int flat = min(int(blockIdx.x * kRowsPerCta + threadIdx.x), a.tokens * a.q_heads - 1);
  int request = find_request(a, a.by_q_heads.of(blockIdx.x * kRowsPerCta), s_request);
  if (threadIdx.x < kRowsPerCta) request = request_from(a, a.by_q_heads.of(flat), request, true);
  pdl_enter();
  const LineNote note = *a.note;
  const int used = used_tokens(a);
  if (threadIdx.x < kRowsPerCta)
    parts[threadIdx.x] = find_parts(a, note, used, blockIdx.x * kRowsPerCta + threadIdx.x, request);
  int lost = 0;  // read by the last threads, as the first are busy
#pragma unroll 1
  for (int c = blockDim.x - 1 - threadIdx.x; c < a.grid; c += blockDim.x) lost |= a.gave_up[c];
  if (__syncthreads_or(lost)) {
    no_numbers(a, blockIdx.x * kRowsPerCta, kRowsPerCta);
    return;
  }
  const int64_t all = int64_t(a.tokens) * a.q_heads;
  for (int row = (kGroups == 1 ? 4 * grp : 0) + (in_grp & 3); row < kRowsPerCta; row += 8) {
    const RowParts r = parts[row];
    const int count = r.live ? r.count[0] + r.count[1] : 0;
    const int h = a.by_group.of(r.head);
    // the row among the whole items' rows
    const int64_t packed = int64_t(h) * a.tokens * a.group + int64_t(r.token) * a.group + (r.head - h * a.group);
    Joined sum;
    for (int i0 = kGroups == 1 ? 0 : grp; i0 < count; i0 += kGroups * kUnroll) {
      float2 ml[kUnroll];
      float v[kUnroll][8];
#pragma unroll
      for (int x = 0; x < kUnroll; ++x) {
        const int i = i0 + x * kGroups;
        ml[x] = make_float2(-INFINITY, 0.0f);
        if (i < count) {
          const bool own = i >= r.count[0];
          if ((own ? r.count[1] : r.count[0]) == 1) {
            ml[x] = *reinterpret_cast<const float2*>(a.part_ml + ((own ? all : 0) + packed) * 2);
            load8f(a.part_o + ((own ? 32 * all : 0) + lanes8 * all + packed) * 8, v[x]);
          } else {  // a CTA's first piece where the item began earlier, else its last
            const int at = own ? i - r.count[0] : i;
            const int64_t slot = 2 * ((own ? r.cta[1] : r.cta[0]) + at) + (at == 0);
            const int in_tile = own ? r.in_tile[1] : r.in_tile[0];
            ml[x] = *reinterpret_cast<const float2*>(a.slot_ml + (slot * a.slot_rows + in_tile) * 2);
            load8f(a.slot_o + ((slot * 32 + lanes8) * a.slot_rows + in_tile) * 8, v[x]);
          }
        } else {
#pragma unroll
          for (int k = 0; k < 8; ++k) v[x][k] = 0.0f;
        }
      }
#pragma unroll
      for (int x = 0; x < kUnroll; ++x) sum.add(ml[x].x, ml[x].y, v[x]);
    }
    if (kGroups > 1) {
      if (grp > 0) {
        float(&to)[kGroups == 1 ? 1 : 10][128] = s_o[grp - 1];
#pragma unroll
        for (int k = 0; k < 8; ++k) to[k][in_grp] = sum.o[k];
        to[8][in_grp] = sum.m;
        to[9][in_grp] = sum.l;
      }
      __syncthreads();
      if (grp > 0) return;
#pragma unroll 1
      for (int w = 0; w < kGroups - 1; ++w) {
        float v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = s_o[w][k][in_grp];
        sum.add(s_o[w][8][in_grp], s_o[w][9][in_grp], v);
      }
    }
    const bool none = sum.l == 0.0f;
    if ((r.live || r.unused) && a.lse != nullptr && lanes8 == 0)
      a.lse[int64_t(r.token) * a.q_heads + r.head] =
          none ? -INFINITY : (sum.m + log2f(sum.l)) * 0.6931471805599453f;
    if (!r.live) continue;
    const float inv = none ? 0.0f : 1.0f / sum.l;
    uint4 packed_out = make_uint4(0, 0, 0, 0);
    if (!none)
      packed_out = make_uint4(pack_bf16x2(sum.o[0] * inv, sum.o[1] * inv), pack_bf16x2(sum.o[2] * inv, sum.o[3] * inv),
                              pack_bf16x2(sum.o[4] * inv, sum.o[5] * inv), pack_bf16x2(sum.o[6] * inv, sum.o[7] * inv));
    *reinterpret_cast<uint4*>(a.out + r.token * a.out_token + r.head * a.out_head + lanes8 * 8) = packed_out;
  }
}

// No request: every row is one of none.  Eight lanes of a row a thread.
__global__ void __launch_bounds__(256) rope_attend_none_kernel(const __grid_constant__ AttendArgs a) {
  pdl_enter();
  const int64_t item = int64_t(blockIdx.x) * blockDim.x + threadIdx.x;
  const int row = int(item >> 5), lanes8 = int(item & 31);
  if (row >= a.tokens * a.q_heads) return;
  const int token = a.by_q_heads.of(row), head = row - token * a.q_heads;
  if (a.fill)
    *reinterpret_cast<uint4*>(a.out + token * a.out_token + head * a.out_head + lanes8 * 8) = make_uint4(0, 0, 0, 0);
  if (a.lse != nullptr && lanes8 == 0) a.lse[row] = -INFINITY;
}

// ---------------------------------------------------------------------------
// Host side.
// ---------------------------------------------------------------------------
// Layout of the workspace, in bytes from its base.
struct Workspace {
  int64_t note, gave_up, units, slot_ml, slot_o, part_ml, part_o, bytes;
};

Workspace attend_workspace(int64_t tokens, int64_t batch, int64_t q_heads, int64_t group, int64_t prefix_len,
                           int64_t grid) {
  auto up = [](int64_t v) { return (v + 255) / 256 * 256; };
  const int64_t rows = tokens * group < kRows ? tokens * group : kRows;
  const int64_t slots = 2 * grid * rows;
  const int64_t parts = prefix_len > 0 ? 2 * tokens * q_heads : 0;
  Workspace w;
  w.note = 0;
  w.gave_up = 256;
  w.units = w.gave_up + up(grid * 4);
  static_assert(sizeof(LineNote) <= 256, "line note");
  w.slot_ml = w.units + up(batch * 4);
  w.slot_o = w.slot_ml + up(slots * 8);
  w.part_ml = w.slot_o + up(slots * kHeadDim * 4);
  w.part_o = w.part_ml + up(parts * 8);
  w.bytes = w.part_o + up(parts * kHeadDim * 4);
  return w;
}

// Tensor map of a cache.  K: {256 lanes, slot, head, block}, boxes of 64 lanes
// and `box_keys` slots.  V: {64 lanes, slot, chunk of 64 lanes, head, block},
// boxes of all lanes and `box_keys` slots.
bool encode_cache_map(CUtensorMap& map, const void* base, int64_t blocks, int64_t block_size, int64_t heads,
                      const int64_t* strides, int box_keys, bool chunks) {
  const PFN_cuTensorMapEncodeTiled_v12000 encode = tensor_map_encoder();
  if (encode == nullptr) return false;
  // the stride of a dimension of one is not used, but has to be one
  auto step = [](int64_t extent, int64_t stride) { return cuuint64_t(extent > 1 ? stride : kHeadDim) * 2; };
  const cuuint64_t slot = step(block_size, strides[1]), head = step(heads, strides[2]);
  const cuuint64_t block = step(blocks, strides[0]);
  const cuuint64_t n = cuuint64_t(block_size), h = cuuint64_t(heads), b = cuuint64_t(blocks);
  const cuuint64_t dim_k[4] = {kHeadDim, n, h, b}, dim_v[5] = {64, n, kHeadDim / 64, h, b};
  const cuuint64_t stride_k[3] = {slot, head, block}, stride_v[4] = {slot, 128, head, block};
  const cuuint32_t box_k[4] = {64, cuuint32_t(box_keys), 1, 1};
  const cuuint32_t box_v[5] = {64, cuuint32_t(box_keys), kHeadDim / 64, 1, 1};
  const cuuint32_t unit[5] = {1, 1, 1, 1, 1};
  return encode(&map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, chunks ? 5 : 4, const_cast<void*>(base),
                chunks ? dim_v : dim_k, chunks ? stride_v : stride_k, chunks ? box_v : box_k, unit,
                CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

bool attend_sizes_ok(int64_t tokens, int64_t batch, int64_t q_heads, int64_t k_heads, int64_t prefix_len) {
  if (tokens < 0 || batch < 0 || q_heads < 1 || k_heads < 1 || prefix_len < 0) return false;
  if (q_heads % k_heads != 0 || batch > kMaxItems || prefix_len > kMaxItems) return false;
  return q_heads <= kMaxItems && tokens <= kMaxItems / q_heads;
}

// WELM_ROPE_GIVE_UP=1 in the environment makes every call behave as one of whose
// waits has not ended, for tests of what becomes of it.
bool give_up() {
  static const bool at_once = [] {
    const char* v = std::getenv("WELM_ROPE_GIVE_UP");
    return v != nullptr && v[0] == '1';
  }();
  return at_once;
}

int launch_attend(const CUtensorMap& kmap, const CUtensorMap& vmap, const AttendArgs& a, cudaStream_t stream) {
  if (cudaFuncSetAttribute(rope_attend_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes) !=
      cudaSuccess) {
    cudaGetLastError();
    return WELM_ROPE_ERR_CUDA;
  }
  int rc = launch(rope_attend_kernel, unsigned(a.grid), kThreads, kSmemBytes, stream, kmap, vmap, a);
  if (rc != WELM_ROPE_OK) return rc;
  const int64_t rows = int64_t(a.tokens) * a.q_heads;
  // Few rows may have many partial results each: four groups of threads to a row's,
  // with as many loads in flight as registers allow for one CTA or two on an SM.
  // 768 rows of some 20 partial results: 34.7 us for both kernels with two groups,
  // 33.0 with four; 288 rows of three: 27.0 with four loads in flight, 27.7 with three.
  if (rows <= 4 * a.grid) return launch(rope_attend_join_kernel<4, 4, 1>, unsigned((rows + 3) / 4), 512, 0, stream, a);
  if (rows <= 8 * a.grid) return launch(rope_attend_join_kernel<4, 3, 2>, unsigned((rows + 3) / 4), 512, 0, stream, a);
  // More rows keep the SMs busy with one group to a row.  Both kernels' us with two
  // groups and with one: decode over a prefix, 4200 rows 57.0 and 61.2, 6000 79.3 and
  // 81.2, 7200 94.8 and 96.4, 8400 110.3 and 107.5; a prompt's chunk, 4200 rows 28.2
  // and 31.0, 6000 34.6 and 34.5, 7200 38.0 and 35.7, 9000 45.0 and 38.7.
  if (rows <= 40 * a.grid) return launch(rope_attend_join_kernel<2, 3, 1>, unsigned((rows + 3) / 4), 256, 0, stream, a);
  return launch(rope_attend_join_kernel<1, 2, 1>, unsigned((rows + 31) / 32), 256, 0, stream, a);
}

}  // namespace

extern "C" {

int welm_rope_attend_workspace(int64_t n_tokens, int64_t batch_size, int64_t num_q_heads, int64_t num_k_heads,
                               int64_t prefix_len, int64_t* bytes) {
  if (!bytes) return WELM_ROPE_ERR_NULL_POINTER;
  if (!attend_sizes_ok(n_tokens, batch_size, num_q_heads, num_k_heads, prefix_len)) return WELM_ROPE_ERR_BAD_SIZE;
  const int sms = current_sm_count();
  if (sms <= 0) {
    cudaGetLastError();
    return WELM_ROPE_ERR_CUDA;
  }
  *bytes = attend_workspace(n_tokens, batch_size, num_q_heads, num_q_heads / num_k_heads, prefix_len, sms).bytes;
  return WELM_ROPE_OK;
}

int welm_rope_attend(const void* q, void* out, float* lse, const void* key_cache, const void* value_cache,
                     const int32_t* block_table, const int64_t* seq_lens, const int64_t* query_starts,
                     const int32_t* prefix_table, int64_t prefix_len, int64_t n_tokens, int64_t batch_size,
                     int64_t num_q_heads, int64_t num_k_heads, int64_t q_token_stride, int64_t q_head_stride,
                     int64_t out_token_stride, int64_t out_head_stride, int64_t table_width, int64_t table_stride,
                     int64_t num_blocks, int64_t block_size, const int64_t* key_cache_strides,
                     const int64_t* value_cache_strides, float scale, int64_t fill_unused, void* workspace,
                     int64_t workspace_bytes, int32_t* device_status, void* stream) {
  if (!attend_sizes_ok(n_tokens, batch_size, num_q_heads, num_k_heads, prefix_len)) return WELM_ROPE_ERR_BAD_SIZE;
  if (num_blocks < 0 || block_size < 1 || table_width < 0 || num_blocks > kMaxItems || block_size > kMaxItems ||
      table_width > kMaxItems / block_size)
    return WELM_ROPE_ERR_BAD_SIZE;
  if (!query_starts && n_tokens != batch_size) return WELM_ROPE_ERR_BAD_SIZE;
  // units are counted in 32 bits, and a request's rows against its keys too
  if (num_q_heads / num_k_heads > (int64_t(1) << 36) / (table_width * block_size + n_tokens + 256))
    return WELM_ROPE_ERR_BAD_SIZE;
  const __int128 row_tiles = (n_tokens * (num_q_heads / num_k_heads) + kRows - 1) / kRows;
  if ((row_tiles * ((prefix_len + kKeys - 1) / kKeys + kItemCost) +
       (row_tiles + batch_size) * ((table_width * block_size + kKeys - 1) / kKeys + kItemCost)) * num_k_heads >=
      INT32_MAX)
    return WELM_ROPE_ERR_BAD_SIZE;
  // in FP32, as the kernels multiply by it
  if (!(scale > 0.0f) || !std::isfinite(scale * kLog2E) || (fill_unused != 0 && fill_unused != 1)) return WELM_ROPE_ERR_BAD_MODE;
  if (n_tokens == 0 || (batch_size == 0 && fill_unused == 0 && lse == nullptr)) return WELM_ROPE_OK;
  if (batch_size == 0) {
    if (fill_unused && !out) return WELM_ROPE_ERR_NULL_POINTER;
    if (fill_unused && (!rows_apart<2>({n_tokens, num_q_heads}, {out_token_stride, out_head_stride}) ||
                        ((out_token_stride | out_head_stride) & 7) || !aligned16(out)))
      return WELM_ROPE_ERR_BAD_STRIDE;
    AttendArgs none{};
    none.out = static_cast<uint16_t*>(out);
    none.lse = lse;
    none.out_token = out_token_stride;
    none.out_head = out_head_stride;
    none.tokens = int32_t(n_tokens);
    none.q_heads = int32_t(num_q_heads);
    none.by_q_heads = Divisor(num_q_heads);
    none.fill = int32_t(fill_unused);
    return launch(rope_attend_none_kernel, unsigned((n_tokens * num_q_heads + 7) / 8), 256, 0,
                  static_cast<cudaStream_t>(stream), none);
  }
  if (block_size % 8 != 0 || num_blocks == 0) return WELM_ROPE_ERR_BAD_SIZE;
  if (!q || !out || !key_cache || !value_cache || !seq_lens || !workspace || !key_cache_strides ||
      !value_cache_strides || (table_width > 0 && !block_table) || (prefix_len > 0 && !prefix_table))
    return WELM_ROPE_ERR_NULL_POINTER;
  if (q_token_stride < 0 || q_head_stride < 0 || table_stride < 0 ||
      !rows_apart<2>({n_tokens, num_q_heads}, {out_token_stride, out_head_stride}))
    return WELM_ROPE_ERR_BAD_STRIDE;
  int64_t bits = q_token_stride | q_head_stride | out_token_stride | out_head_stride;
  const int64_t extent[3] = {num_blocks, block_size, num_k_heads};
  for (const int64_t* s : {key_cache_strides, value_cache_strides}) {
    for (int i = 0; i < 3; ++i) {
      // tensor maps: steps of 16 bytes, below 2^40
      if (extent[i] > 1 && (s[i] < kHeadDim || s[i] >= (int64_t(1) << 39))) return WELM_ROPE_ERR_BAD_STRIDE;
      if (extent[i] > 1) bits |= s[i];
    }
  }
  if (bits & 7) return WELM_ROPE_ERR_BAD_STRIDE;
  for (const void* p : {q, static_cast<const void*>(out), key_cache, value_cache})
    if (!aligned16(p)) return WELM_ROPE_ERR_BAD_STRIDE;
  if (reinterpret_cast<uintptr_t>(workspace) & 31u) return WELM_ROPE_ERR_BAD_STRIDE;
  // Rows of out are written while others are still computed from q and the caches.
  const RowSet out_rows{reinterpret_cast<uintptr_t>(out), {n_tokens, num_q_heads, 1}, {out_token_stride, out_head_stride, 0}};
  if (rows_meet(out_rows, {reinterpret_cast<uintptr_t>(q), {n_tokens, num_q_heads, 1}, {q_token_stride, q_head_stride, 0}}))
    return WELM_ROPE_ERR_BAD_STRIDE;
  for (const auto& [cache, s] : {std::pair(key_cache, key_cache_strides), std::pair(value_cache, value_cache_strides)})
    if (rows_meet(out_rows, {reinterpret_cast<uintptr_t>(cache), {num_blocks, block_size, num_k_heads}, {s[0], s[1], s[2]}}))
      return WELM_ROPE_ERR_BAD_STRIDE;
  const int sms = current_sm_count();
  if (sms <= 0) {
    cudaGetLastError();
    return WELM_ROPE_ERR_CUDA;
  }
  const int64_t group = num_q_heads / num_k_heads;
  const Workspace w = attend_workspace(n_tokens, batch_size, num_q_heads, group, prefix_len, sms);
  if (workspace_bytes < w.bytes) return WELM_ROPE_ERR_CAPACITY;
  int box = 8;
  while (box < kKeys && block_size % (2 * box) == 0) box *= 2;
  CUtensorMap kmap, vmap;
  if (!encode_cache_map(kmap, key_cache, num_blocks, block_size, num_k_heads, key_cache_strides, box, false) ||
      !encode_cache_map(vmap, value_cache, num_blocks, block_size, num_k_heads, value_cache_strides,
                        box < kHalfKeys ? box : kHalfKeys, true))
    return WELM_ROPE_ERR_CUDA;
  AttendArgs a{};
  a.q = static_cast<const uint16_t*>(q);
  a.out = static_cast<uint16_t*>(out);
  a.lse = lse;
  a.q_token = q_token_stride;
  a.q_head = q_head_stride;
  a.out_token = out_token_stride;
  a.out_head = out_head_stride;
  a.prefix_table = prefix_table;
  a.block_table = block_table;
  a.table_stride = table_stride;
  a.seq_lens = seq_lens;
  a.query_starts = query_starts;
  a.tokens = int32_t(n_tokens);
  a.batch = int32_t(batch_size);
  a.q_heads = int32_t(num_q_heads);
  a.k_heads = int32_t(num_k_heads);
  a.group = int32_t(group);
  a.by_group = Divisor(group);
  a.by_block = Divisor(block_size);
  a.by_q_heads = Divisor(num_q_heads);
  a.prefix_len = int32_t(prefix_len);
  a.max_len = int32_t(table_width * block_size);
  a.block_size = int32_t(block_size);
  a.num_blocks = int32_t(num_blocks);
  a.box_k = box;
  a.box_v = box < kHalfKeys ? box : kHalfKeys;
  a.slot_rows = int32_t(n_tokens * group < kRows ? n_tokens * group : kRows);
  a.grid = sms;
  a.fill = int32_t(fill_unused);
  a.scale = scale * kLog2E;
  char* base = static_cast<char*>(workspace);
  a.note = reinterpret_cast<LineNote*>(base + w.note);
  a.gave_up = reinterpret_cast<int32_t*>(base + w.gave_up);
  a.give_up = give_up();
  a.units_before = reinterpret_cast<int32_t*>(base + w.units);
  a.slot_ml = reinterpret_cast<float*>(base + w.slot_ml);
  a.slot_o = reinterpret_cast<float*>(base + w.slot_o);
  a.part_ml = reinterpret_cast<float*>(base + w.part_ml);
  a.part_o = reinterpret_cast<float*>(base + w.part_o);
  a.status = device_status;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  return launch_attend(kmap, vmap, a, s);
}

}  // extern "C"
