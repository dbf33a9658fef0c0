// Attention of the newest tokens of each sequence over a paged cache of e4m3 keys and values with
// one scale per page and head, a sliding window and first tokens that stay visible:
//   s_rj = scale * ks(page of j) * q_r . k_j          for the tokens j that row r sees
//   o_r  = sum_j e^(s_rj) vs(page of j) v_j / sum_j e^(s_rj)
// A row is one query head of one query token; the rows that share a key / value head (heads per
// key head x query tokens) are worked on together, so the cache is read once for all of them.
//
// HBM-bound: a token costs 2 * head_dim bytes per key head.  Both products run on the tensor cores
// straight from the bytes that the tensor memory accelerator put into shared memory; nothing is
// converted on the way.  The tokens are the M side:
//   S^T [128 tokens x N] = K tile (K-major)             x Q parts  [N x head_dim]
//   O^T [head_dim  x N]  = V tile (MN-major, as it lies) x P parts [N x 128 tokens]
// and the other operand, which is small, is split into sums of e4m3 numbers that fill N columns:
// a bf16 has 8 significant bits and is exactly hi + lo / 16 of two e4m3 (4 bits each, and what the
// first rounding leaves over fits the second), an fp16 takes three.  A row of queries has one exponent,
// so that much is true of elements down to 2^-14 of the row's largest (bf16; fp16 2^-15); of smaller
// ones e4m3's smallest step leaves an error of 2^-22 of the largest (fp16 2^-26).  Probabilities
// keep 9 bits (two parts) or 14 (three): one more than a bf16 output has, three more than an fp16 one
// (11 with the first part taken from fp16 too: 32 sequences with a window of 2048 in fp16 26.1 us, with 14 26.4;
// bf16 with three parts of 14 bits: the same in bf16 25.0 -> 26.3, 28 rows 84.4 -> 89.5, for an output of 8 bits).
// The sums of a row take them unrounded: a token whose value scale is far below its tile's
// largest rounds to nothing in the product, but weighs no less.  N = parts * rows, at least 16, was idle
// anyway.
//
// Per tile of 256 tokens each of 256 threads owns one token: it reads its N scores from tensor memory,
// applies both scales and the masks, and takes part in the rows' maxima over the tile (warp reductions
// and one exchange through shared memory, on a barrier of its own).  Probabilities are relative to the
// tile's own maximum (of s + log2 vs, so that they fit e4m3 whatever the scales).  While the maxima of
// one tile get together, the product of the tile before is read back -- now a thread owns one of the
// head's columns and half of the rows -- and joins the running sums in registers with the usual
// rescaling, in fp32.  P is laid out so that a thread writes its token's N bytes in one piece.
//
// Value rows that no query sees are cleared in shared memory before the product: their weight is
// zero, but zero times a NaN that was left in a page would not be.  Of rows that some queries of the
// call see and others do not, NaN bytes are cleared and noted for the rows that see them
// (set_nan_aside): nothing reaches a query that it must not see.
//
// Work: all (sequence, row tile, key head) items in order, each a run of visible tiles (those of
// the first tokens, then those of the window), cut into equal shares for a grid that fills the
// chip.  A share may start and end inside an item; such parts leave their sums in the workspace and
// a second kernel joins them, in token order.  Lengths are read on the device, so a captured call
// follows them.
//
// What bounds it: HBM where there is enough of it to do (64 sequences of 4 to 8 thousand tokens, 8 key
// heads of 128 in bf16: 132 us, 6.1 TB/s; the sums of 16 rows a key head in fp16 keep the softmax
// threads busier than HBM: 31 sequences of 11 to 22 thousand tokens, 28 rows, 90 us, a quarter of HBM's
// rate, with issue slots half used and the rest spent on the exchange of the maxima); below some 20 us
// the chain length -> page -> tile -> scores -> probabilities -> sums, 6.5 us for one sequence of 100 tokens.
// Some 1.5 of them pass until a block knows its share, 1.5 until its first page is asked for and 1 to 2
// until that is there, which is why the first copies leave before anything else is looked up.
// Two CTAs per SM hide one's exchange behind the other's arithmetic.  Measured on the way, the first of
// these cases: a thread per score without tensor cores 9463 us, tiles of 128 tokens with four softmax
// warps 191, pages and scales looked up two steps ahead and products joined a tile later 140, tiles of
// 256 tokens with eight warps 134, a shorter start 132.

#include "elem.cuh"
#include "kv_cache.cuh"
#include "sm100.cuh"

namespace nb200 {
namespace {

using namespace sm100;

constexpr int kHalf = 128;               // tokens of one product: tensor-memory lanes
constexpr int kTile = 256;               // tokens of a step: a thread's each
constexpr int kTileShift = 8;
constexpr int kSmemPerCta = 106 * 1024;
constexpr int kThreads = 320;            // producer, issuer, eight softmax warps
constexpr int kSoftmaxWarp = 2;
constexpr int kJoinThreads = 256;
constexpr int kWholeTiles = 3, kJoinTiles = 2;   // see whole_items
constexpr int kMaxShares = 320;          // two CTAs on each of 148 SMs
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLeastScale = 8.67361738e-19f;   // 2^-60
constexpr float kProbLog2 = 8.0f;        // a tile's largest probability is 2^8 as an operand: e4m3 ends at 448

enum : unsigned int {
  ST_KV_Q = 32, ST_KV_K, ST_KV_V, ST_KV_EMPTY, ST_KV_SCALES, ST_KV_S, ST_KV_P, ST_KV_O, ST_KV_ZERO, ST_KV_MOST, ST_KV_SUM
};

// Division of 0 <= n < 2^31 by a d that the host knows: with 2^(s-1) < d <= 2^s and m = floor(2^(31+s) / d) + 1,
// m d is 2^(31+s) and up to d more, which adds less than 1 / d to n m / 2^(31+s): it is n / d rounded
// down.  A division by a number in a register is some thirty instructions, and a block begins with
// half a dozen of them one behind the other.
struct Divisor {
  uint32_t m, shift;
  Divisor() = default;
  explicit Divisor(int d) {
    int s = 0;
    while ((1ll << s) < d) ++s;
    m = (uint32_t)((1ull << (31 + s)) / (uint32_t)d + 1);
    shift = 31 + s;
  }
  __device__ int divide(int n) const { return (int)(((unsigned long long)(uint32_t)n * m) >> shift); }
};

struct KvAttnParams {
  const void* q;
  void* out;
  const float *k_scales, *v_scales;
  const int32_t* table;
  const int32_t* lengths;
  float* parts;                          // [2 * shares][RP][head_dim]: sums of the parts of cut items
  float2* marks;                         // [2 * shares][RP]: their reference and weight
  int64_t q_batch_stride, q_token_stride, q_head_stride;
  int64_t o_batch_stride, o_token_stride, o_head_stride;
  int64_t table_stride, k_scale_stride, v_scale_stride;
  int batch, nq, kv_heads, group;        // group: query heads per key head
  int rows, row_tiles;                   // nq * group, and how many pieces of RP rows
  int pages, page, page_shift, max_pages, window, sinks;
  int shares, q_aligned;
  int per_seq, stretch;                  // items of a sequence; sequences that a lane of a work list counts
  int share_items, longer_shares;        // whole items: how many a share has, and how many shares have one more
  Divisor by_shares, by_per_seq, by_row_tiles, by_stretch;
  float scale;
  unsigned long long wait_limit_ns;
  unsigned int* status;
};

// The visible tiles of one sequence: [0, first) and [from, ...), `count` together.
struct Seq {
  int len, limit, low, sink_end;   // tokens: in the cache, with a table entry, first of the window, sinks
  int first, from, count;
};

__device__ __forceinline__ Seq make_seq(const KvAttnParams& p, int len) {
  Seq s;
  len = max(len, 0);
  s.len = len;
  s.limit = min(len, p.max_pages << p.page_shift);
  s.low = p.window ? max(max(len, p.nq) - p.nq + 1 - p.window, 0) : 0;   // of the first query there is
  s.sink_end = min(p.sinks, s.limit);
  const int shift = kTileShift, round = (1 << shift) - 1;
  const int tiles = (s.limit + round) >> shift;
  s.first = s.from = 0;
  s.count = tiles;
  if (s.low > 0) {
    const int sink_tiles = (s.sink_end + round) >> shift;
    if ((s.low >> shift) > sink_tiles) {
      s.first = sink_tiles;
      s.from = s.low >> shift;
      s.count = sink_tiles + max(tiles - s.from, 0);
    }
  }
  s.count = max(s.count, 1);       // a sequence without tokens has its zeros to write
  return s;
}
__device__ __forceinline__ int tile_start(const KvAttnParams& p, const Seq& s, int t) {
  return (t < s.first ? t : t - s.first + s.from) << kTileShift;
}
// Does any query of the call see this token, as far as positions go?
__device__ __forceinline__ bool seen_by_any(const Seq& s, int token) {
  return token < s.limit && (token >= s.low || token < s.sink_end);
}

// Where in the work list a tile is: sequence, item of the sequence (key head, row tile), tile.
struct Place {
  int b, head, row_tile, tile;
};

// The work list as one warp sees it: lane i knows how many tiles a stretch of the sequences has and
// how many come before it.  All lanes take part in every call.
struct WorkList {
  int before, sum;            // of this lane's stretch, for one (key head, row tile)
  int total, largest;         // of all: tiles of one (key head, row tile), most of one sequence

  __device__ WorkList(const KvAttnParams& p) {
    const int lane = threadIdx.x & 31, stretch = p.stretch;
    sum = largest = 0;
#pragma unroll 1
    for (int i = 0; i < stretch; ++i) {
      const int b = lane * stretch + i;
      if (b < p.batch) {
        const int count = make_seq(p, __ldg(p.lengths + b)).count;
        sum += count;
        largest = max(largest, count);
      }
    }
    int run = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int other = __shfl_up_sync(0xffffffffu, run, o);
      if (lane >= o) run += other;
    }
    before = run - sum;
    total = __shfl_sync(0xffffffffu, run, 31);
    largest = __reduce_max_sync(0xffffffffu, largest);
  }
  __device__ int tiles(const KvAttnParams& p) const { return total * p.per_seq; }

  // Shares of whole items, or of tiles?  Joining the parts of cut items costs about as much as
  // kJoinTiles tiles: whole items where the longest share of them is no longer than that (1 sequence of
  // 1000 tokens, 8 key heads of 4 tiles: cut 9.6 us, whole 11.1; 16 of them: whole 14.4, cut 15.5).
  // Always whole where every item has up to kWholeTiles: the host then leaves out the joining launch
  // (can_be_cut; 4 sequences of 700 tokens: whole 9.7 us, cut 10.9).
  __device__ int tile_share(const KvAttnParams& p) const { return p.by_shares.divide(tiles(p) + p.shares - 1); }
  __device__ bool whole_items(const KvAttnParams& p) const {
    const long long items = p.share_items + (p.longer_shares > 0);
    return largest <= kWholeTiles || items * largest <= tile_share(p) + kJoinTiles;
  }

  // tiles of the sequences before b and of b, of one (key head, row tile); the same b in all lanes
  __device__ int before_sequence(const KvAttnParams& p, int b, int* count) const {
    const int owner = p.by_stretch.divide(b);
    int at = __shfl_sync(0xffffffffu, before, owner);
    if (p.stretch == 1) {
      *count = __shfl_sync(0xffffffffu, sum, owner);
      return at;
    }
#pragma unroll 1
    for (int k = owner * p.stretch; k < b; ++k) at += make_seq(p, __ldg(p.lengths + k)).count;
    *count = make_seq(p, __ldg(p.lengths + b)).count;
    return at;
  }

  // first tile of share c, from 0 to tiles(); the same c in all lanes
  __device__ int share_start(const KvAttnParams& p, int c) const {
    if (!whole_items(p)) return (int)min((long long)c * tile_share(p), (long long)tiles(p));
    const int i = c * p.share_items + min(c, p.longer_shares), b = p.by_per_seq.divide(i);
    if (b >= p.batch) return tiles(p);
    int count;
    const int at = before_sequence(p, b, &count);
    return at * p.per_seq + (i - b * p.per_seq) * count;
  }

  // The place of a tile, 0 <= flat < tiles(), a tile of its own for every lane if need be.
  __device__ Place locate(const KvAttnParams& p, int flat) const {
    const int q = p.by_per_seq.divide(flat);   // at * per_seq <= flat  <=>  at <= flat / per_seq
    int owner = 0;
#pragma unroll
    for (int step = 16; step > 0; step >>= 1)
      if (__shfl_sync(0xffffffffu, before, owner + step) <= q) owner += step;
    int at = __shfl_sync(0xffffffffu, before, owner);
    int b = owner * p.stretch;
    int count = __shfl_sync(0xffffffffu, sum, owner);
    if (p.stretch > 1) {
      count = make_seq(p, __ldg(p.lengths + b)).count;
#pragma unroll 1
      while (q >= at + count) {
        at += count;
        ++b;
        count = make_seq(p, __ldg(p.lengths + b)).count;
      }
    }
    flat -= at * p.per_seq;
    const int item = flat / count, head = p.by_row_tiles.divide(item);
    return Place{b, head, item - head * p.row_tiles, flat - item * count};
  }
};

// A walk over a share of the work list.
struct Cursor {
  Place at;
  Seq seq;
  int left;      // tiles, this one among them
  __device__ void start(const KvAttnParams& p, const Place& w, int tiles) {
    left = tiles;
    at = Place{0, 0, 0, 0};            // an empty share has no place
    if (left <= 0) return;
    at = w;
    seq = make_seq(p, __ldg(p.lengths + at.b));
  }
  __device__ bool last_tile() const { return at.tile == seq.count - 1; }
  __device__ void next_item(const KvAttnParams& p) {
    if (++at.row_tile < p.row_tiles) return;
    at.row_tile = 0;
    if (++at.head < p.kv_heads) return;
    at.head = 0;
    ++at.b;
    seq = make_seq(p, __ldg(p.lengths + at.b));
  }
  __device__ void advance(const KvAttnParams& p, int tiles) {
    left -= tiles;
    at.tile += tiles;
#pragma unroll 1
    while (left > 0 && at.tile >= seq.count) {
      at.tile -= seq.count;
      next_item(p);
    }
  }
};

template <int D, int RP, int PARTS>
struct Shape {
  static constexpr int kN = (RP * PARTS + 15) / 16 * 16;
  static constexpr int kSlotBytes = kHalf * D;                    // 128 tokens of K or of V
  static constexpr int kQBytes = kN * D;
  static constexpr int kPBytes = kN * kHalf;
  // ring of a tile's K halves, its V halves, the next tile's ...: what two CTAs per SM, and the
  // joining kernel beside them, leave room for
  static constexpr int kRoom = (kSmemPerCta - 3 * 1024 - 320 * RP - 2 * kPBytes - 2 * kQBytes) / kSlotBytes;
  static constexpr int kSlots = kRoom < 12 ? kRoom : 12;
  static constexpr int kTmemO = 4 * kN;                           // behind the scores of two tiles
  static constexpr int kTmemCols = 5 * kN <= 128 ? 128 : 256;
};

template <int D, int RP, int PARTS>
struct Shared {
  using S = Shape<D, RP, PARTS>;
  uint8_t ring[S::kSlots][S::kSlotBytes];      // first: the swizzle counts from 1024-byte boundaries
  uint8_t p[2][S::kPBytes];                    // of a tile's halves
  uint8_t q[2][S::kQBytes];
  float4 scale[4][32];                         // of a step's pages: ks, log2 vs, 1 / vs, 1 if it is there
  float q_factor[2][RP];                       // what takes a row's product to log2 units
  int q_at[2][RP];                             // position of the row's query; -1: no such row
  // where its output is in its sequence and head; -1: no such row.  Four turns: an item's are read
  // by the end of the next one's first maxima, when a warp ahead may be staging two items further.
  int64_t q_out[4][RP];
  float most[2][8][RP];                        // the warps' maxima, alternating by tile
  float sum[2][8][RP];                         // the warps' row sums, alternating by item
  float step[8][3][RP];                        // a warp's own: a row's reference, negative, and what the sums and the tile are scaled by
  uint32_t nan[2][RP][D / 32];                 // columns in which a row has seen NaN set aside, alternating by item
  uint64_t full[S::kSlots], empty[S::kSlots], scale_full[4];
  uint64_t q_full[2], s_full[2], most_full[2], p_full, o_full, sum_full;
  uint32_t tmem_slot, abort_flag;
};

// Two values as e4m3 (low and high byte), and what is left of them, times 16.
__device__ __forceinline__ uint32_t split2(float& a, float& b) {
  const uint32_t q = e4m3x2(a, b);
  const float2 f = e4m3x2_values(q);
  a = (a - f.x) * 16.0f;
  b = (b - f.y) * 16.0f;
  return q;
}
// The same for a pair of fp16.
__device__ __forceinline__ uint32_t split2(__half2& h) {
  uint16_t q;
  uint32_t back;
  asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(q) : "r"(*reinterpret_cast<const uint32_t*>(&h)));
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(back) : "h"(q));
  h = __hmul2(__hsub2(h, *reinterpret_cast<const __half2*>(&back)), __float2half2_rn(16.0f));
  return q;
}

// Queries of one item on their way from global memory to their e4m3 parts: 8 columns of a row per
// softmax thread, as many threads as that takes.
template <typename T, int D, int RP, int PARTS>
struct Queries {
  static constexpr int kPerRow = D / 8;
  static_assert(RP * kPerRow <= 256, "a vector per thread");
  Vec<T> raw;
  int64_t offset;                  // of the row and column; -1: no such row
  int row_tile = -1;               // that the offset is for

  __device__ void load(const KvAttnParams& p, const Cursor& c, int tid) {
    if (row_tile != c.at.row_tile) {
      row_tile = c.at.row_tile;
      const int r = row_tile * RP + tid / kPerRow;
      offset = tid / kPerRow < RP && r < p.rows
                   ? r / p.group * p.q_token_stride + r % p.group * p.q_head_stride + tid % kPerRow * 8
                   : -1;
    }
    raw.raw = make_uint4(0, 0, 0, 0);
    if (offset < 0) return;
    const T* src = static_cast<const T*>(p.q) + c.at.b * p.q_batch_stride +
                   (int64_t)c.at.head * p.group * p.q_head_stride + offset;
    if (p.q_aligned) {
      raw.raw = __ldg(reinterpret_cast<const uint4*>(src));
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) raw.e[j] = src[j];
    }
  }
};

// Row r times 2^-e fits e4m3's range; 2^e goes into the row's factor.  Parts of row r are rows r,
// RP + r, ... of the operand, K-major under the swizzle of its row length.  Out of line: it runs once
// an item, and the tiles' loop has to fit the instruction cache.
template <typename T, int D, int RP, int PARTS>
__device__ __noinline__ void stage_queries(const KvAttnParams& p, Vec<T> raw, int first_at, int row_tile, int tid,
                                           uint8_t* q, float* factor, int* at, int64_t* out) {
  constexpr int kPerRow = D / 8;
  const int r = tid / kPerRow, col8 = tid % kPerRow;
  float f[8], most = 0.0f;
  bool bad = false;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    f[j] = Elem<T>::to_f32(raw.e[j]);
    most = fmaxf(most, fabsf(f[j]));
    bad |= !(fabsf(f[j]) < INFINITY);
  }
#pragma unroll
  for (int o = kPerRow / 2; o > 0; o >>= 1) {
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
    bad |= (bool)__shfl_xor_sync(0xffffffffu, (int)bad, o);
  }
  if (r >= RP) return;
  const int e = max(e4m3_exponent(most), -100);    // most <= 448 * 2^e
  const float down = power_of_two(-e);
  if (col8 == 0) {
    const int row = row_tile * RP + r;
    const bool is = row < p.rows;
    factor[r] = bad ? NAN : power_of_two(e) * (p.scale * kLog2e);
    at[r] = is ? first_at + row / p.group : -1;
    out[r] = is ? row / p.group * p.o_token_stride + row % p.group * p.o_head_stride : -1;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) f[j] *= down;
#pragma unroll
  for (int part = 0; part < PARTS; ++part) {
    const uint32_t w0 = split2(f[0], f[1]), w1 = split2(f[2], f[3]);
    const uint32_t w2 = split2(f[4], f[5]), w3 = split2(f[6], f[7]);
    const int n = part * RP + r;
    const int chunk = (col8 >> 1) ^ (D == 128 ? (n & 7) : ((n >> 1) & 3));
    *reinterpret_cast<uint2*>(q + n * D + chunk * 16 + (col8 & 1) * 8) = make_uint2(w0 | (w1 << 16), w2 | (w3 << 16));
  }
}

// A token that some rows of the item see and others do not: NaN in its value row, `row` of the tile in
// shared memory, becomes 0, as zero times NaN would reach the rows that do not see it; `noted` keeps the
// columns for those that do.  The rows' positions are worked out anew: another warp may be staging the
// item after the next one where this one's stood.  Out of line: it runs at the ends of a window, for
// several query tokens (32 sequences with a window of 2048 and four of them: 26.1 us, without 25.6).
template <int D, int RP>
__device__ __noinline__ void set_nan_aside(const KvAttnParams& p, uint8_t* tile, int row, int token, int first_at,
                                           int row_tile, uint32_t (*noted)[D / 32]) {
  auto nan_bytes = [](uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; };   // 0x7f and 0xff
  uint32_t any = 0;
#pragma unroll
  for (int i = 0; i < D; i += 16) {                // neighbours start at different banks
    const uint4 v = *reinterpret_cast<const uint4*>(tile + row * D + ((i + row * 16) & (D - 1)));
    any |= nan_bytes(v.x) | nan_bytes(v.y) | nan_bytes(v.z) | nan_bytes(v.w);
  }
  if (any == 0) return;
#pragma unroll 1
  for (int i = 0; i < D; i += 16) {
    // where the swizzle of its row length has put these 16 columns
    const int chunk = (i / 16) ^ (D == 128 ? (row & 7) : ((row >> 1) & 3));
    uint32_t* words = reinterpret_cast<uint32_t*>(tile + row * D + chunk * 16);
#pragma unroll 1
    for (int k = 0; k < 4; ++k) {
      const uint32_t w = words[k];
      const uint32_t nan = nan_bytes(w);
      if (nan == 0) continue;
      words[k] = w & ~((nan >> 7) * 0xffu);
      uint32_t columns = 0;
#pragma unroll
      for (int b = 0; b < 4; ++b) columns |= (nan >> (8 * b + 7) & 1u) << b;
      const int first = i + 4 * k;
#pragma unroll 1
      for (int r = 0; r < RP; ++r) {
        const int at = first_at + (row_tile * RP + r) / p.group;
        if (token <= at && (!p.window || token > at - p.window || token < p.sinks))
          atomicOr(&noted[r][first / 32], columns << (first % 32));
      }
    }
  }
}

template <typename T, int D, int RP, int PARTS>
__global__ void __launch_bounds__(kThreads, 2)
    kv_attn_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                   const __grid_constant__ KvAttnParams p) {
  using S = Shape<D, RP, PARTS>;
  constexpr int N = S::kN, SLOTS = S::kSlots, H = 2;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  Shared<D, RP, PARTS>& sh = *reinterpret_cast<Shared<D, RP, PARTS>*>(smem_raw);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const WaitCtx ctx{&sh.abort_flag, p.status, p.wait_limit_ns};

  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");   // the joining kernel may get ready
  for (int i = threadIdx.x; i < 2 * RP * (D / 32); i += kThreads) (&sh.nan[0][0][0])[i] = 0;
  if (threadIdx.x == 0) {
    sh.abort_flag = 0;
    for (int x = 0; x < SLOTS; ++x) {
      mbar_init(smem_u32(&sh.full[x]), 1);
      mbar_init(smem_u32(&sh.empty[x]), 1);
    }
    for (int x = 0; x < 4; ++x) mbar_init(smem_u32(&sh.scale_full[x]), 1);
    for (int x = 0; x < 2; ++x) {
      mbar_init(smem_u32(&sh.q_full[x]), 8);   // one arrival per softmax warp
      mbar_init(smem_u32(&sh.s_full[x]), 1);
      mbar_init(smem_u32(&sh.most_full[x]), 8);
    }
    mbar_init(smem_u32(&sh.p_full), 8);
    mbar_init(smem_u32(&sh.o_full), 1);
    mbar_init(smem_u32(&sh.sum_full), 8);
    mbar_init_fence();
    prefetch_tensormap(&map_k);
    prefetch_tensormap(&map_v);
  }
  __syncwarp();
  if (warp == 1) tmem_alloc(smem_u32(&sh.tmem_slot), S::kTmemCols);
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = sh.tmem_slot;
  // every warp finds the share's place for itself
  const WorkList list(p);
  const int from = list.share_start(p, blockIdx.x), to = list.share_start(p, blockIdx.x + 1);
  Cursor c;
  c.start(p, to > from ? list.locate(p, from) : Place{0, 0, 0, 0}, to - from);

  if (warp == 0) {
    // ---- producer ----
    // It works in steps of 32 pages, a lane per page: pages are looked up two steps ahead and their
    // scales fetched one step ahead, so that neither latency is met per tile.  The scales go to the
    // softmax warps through four turns of shared memory: a step begins when the ring has room for
    // it, that is when all but the ring's tiles before it are done with, and the ring has fewer
    // tiles than the three steps that are in the other turns.
    static_assert(SLOTS <= 3 * 2 * H * (4 / H), "a turn of the scales would be overwritten too early");
    const int per_half = kHalf >> p.page_shift, step_tiles = 32 / (per_half * H);
    const uint32_t page_bytes = (uint32_t)p.page * D;
    const int my_tile = lane / (per_half * H), my_half = lane / per_half % H, my_page = lane % per_half;
    Cursor mine = c;
    auto page_of = [&](Cursor& at) {             // this lane's page, -1: not to be read
      if (at.left <= 0) return -1;
      const int token = tile_start(p, at.seq, at.at.tile) + my_half * kHalf + (my_page << p.page_shift);
      if (!(token < at.seq.limit && (token + p.page > at.seq.low || token < at.seq.sink_end))) return -1;
      const int id = __ldg(p.table + at.at.b * p.table_stride + (token >> p.page_shift));
      return id >= 0 && id < p.pages ? id : -1;
    };
    // of this step, the next one and the one after
    float ks[2], vs[2];
    int id[3], head[3];
    auto fetch_scales = [&](int page, int of_head, float& k_scale, float& v_scale) {
      k_scale = page >= 0 ? __ldg(p.k_scales + page * p.k_scale_stride + of_head) : 0.0f;
      v_scale = page >= 0 ? __ldg(p.v_scales + page * p.v_scale_stride + of_head) : 1.0f;
    };
    auto next_step = [&](int& page, int& of_head) {
      if (mine.left > 0) mine.advance(p, step_tiles);
      page = page_of(mine);
      of_head = mine.at.head;
    };
    if (c.left > 0 && my_tile > 0) mine.advance(p, my_tile);
    id[0] = page_of(mine);
    head[0] = mine.at.head;
    fetch_scales(id[0], head[0], ks[0], vs[0]);
    bool ok = true;
    int left = c.left;
    for (int step = 0; left > 0 && ok; ++step) {
      bool handed = false;
#pragma unroll 1
      for (int k = 0; k < step_tiles && left > 0 && ok; ++k, --left) {
        const int j = step * step_tiles + k;
#pragma unroll
        for (int i = 0; i < 2 * H; ++i) {        // the halves of K, then those of V
          const int g = 2 * H * j + i, x = g % SLOTS;
          const bool in_slot = my_tile == k && my_half == i % H && id[0] >= 0;
          const uint32_t bytes = __popc(__ballot_sync(0xffffffffu, in_slot)) * page_bytes;
          ok = ok && mbar_wait(smem_u32(&sh.empty[x]), ((g / SLOTS) & 1) ^ 1, ctx, ST_KV_EMPTY, g);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          const uint32_t bar = smem_u32(&sh.full[x]);
          if (lane == 0) {
            if (bytes) mbar_arrive_expect_tx(bar, bytes); else mbar_arrive(bar);
          }
          __syncwarp();
          if (in_slot)
            tma_load_4d(smem_u32(&sh.ring[x][my_page * page_bytes]), i < H ? &map_k : &map_v, 0, 0, head[0], id[0], bar);
        }
        if (!handed) {                           // behind the first tile's copies
          if (vs[0] < kLeastScale) vs[0] = kLeastScale;   // its logarithm is used; NaN stays
          sh.scale[step & 3][lane] = make_float4(ks[0], __log2f(vs[0]), 1.0f / vs[0], id[0] >= 0 ? 1.0f : 0.0f);
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&sh.scale_full[step & 3]));
          handed = true;
          // the next step's scales and the one after's pages are under way while this one is issued
          if (step == 0) next_step(id[1], head[1]);
          fetch_scales(id[1], head[1], ks[1], vs[1]);
          next_step(id[2], head[2]);
        }
      }
      id[0] = id[1];
      head[0] = head[1];
      ks[0] = ks[1];
      vs[0] = vs[1];
      id[1] = id[2];
      head[1] = head[2];
    }
  } else if (warp == 1) {
    // ---- issuer ----
    const bool elected = elect_one();
    constexpr uint32_t kIdescQk = instr_desc_e4m3(kHalf, N, false, false);
    constexpr uint32_t kIdescPv = instr_desc_e4m3(kHalf, N, true, true);
    constexpr uint64_t kKMajor = D == 128 ? smem_desc_sw128(16, 1024) : smem_desc_sw64(16, 512);
    // head_dim 64 fills half of the 128 rows: the second slab of 64 is the first one again
    constexpr uint64_t kVDesc = D == 128 ? smem_desc_sw128(16, 1024) : smem_desc_sw64(0, 512);
    constexpr uint64_t kPDesc = smem_desc_plain(128, kHalf * 16);
    auto wait_all = [&](uint64_t* bar, uint32_t parity, unsigned int code, int detail) -> bool {
      return __all_sync(0xffffffffu, mbar_wait(smem_u32(bar), parity, ctx, code, detail));
    };
    bool ok = true;
    int item = 0;                    // items begun
    auto begin = [&](int j, bool new_item) {       // S(j) = K(j) Q of the item
      if (new_item) ok = wait_all(&sh.q_full[item & 1], (item >> 1) & 1, ST_KV_Q, item);
      const uint32_t qb = smem_u32(sh.q[item & 1]);
#pragma unroll
      for (int h = 0; h < H; ++h) {
        const int g = 2 * H * j + h, x = g % SLOTS;
        ok = ok && wait_all(&sh.full[x], (g / SLOTS) & 1, ST_KV_K, j);
        if (!ok) return;
        tc_fence_after_sync();
        const uint32_t kb = smem_u32(sh.ring[x]);
#pragma unroll
        for (int kk = 0; kk < D / 32; ++kk)
          if (elected)
            mma_f8_ss(tmem + ((j & 1) * H + h) * N, with_address(kKMajor, kb + kk * 32),
                      with_address(kKMajor, qb + kk * 32), kIdescQk, kk != 0);
        if (elected) mma_commit(smem_u32(&sh.empty[x]));
      }
      if (elected) mma_commit(smem_u32(&sh.s_full[j & 1]));
      __syncwarp();
    };
    if (c.left > 0) begin(0, true);
#pragma unroll 1
    for (int j = 0; c.left > 0 && ok; ++j) {
      const bool ends = c.last_tile();
      c.advance(p, 1);
      if (c.left > 0) {
        if (ends) ++item;
        begin(j + 1, ends);
      }
      ok = ok && wait_all(&sh.p_full, j & 1, ST_KV_P, j);
#pragma unroll
      for (int h = 0; h < H; ++h) {
        const int g = 2 * H * j + H + h, x = g % SLOTS;
        ok = ok && wait_all(&sh.full[x], (g / SLOTS) & 1, ST_KV_V, j);
        if (!ok) break;
        tc_fence_after_sync();
        const uint32_t vb = smem_u32(sh.ring[x]), pb = smem_u32(sh.p[h]);
#pragma unroll
        for (int kk = 0; kk < kHalf / 32; ++kk)    // 32 tokens: four groups of eight rows
          if (elected)
            mma_f8_ss(tmem + S::kTmemO, with_address(kVDesc, vb + kk * 32 * D),
                      with_address(kPDesc, pb + kk * 4 * 128), kIdescPv, h != 0 || kk != 0);
        if (elected) mma_commit(smem_u32(&sh.empty[x]));
      }
      if (!ok) break;
      if (elected) mma_commit(smem_u32(&sh.o_full));
      __syncwarp();
    }
  } else {
    // ---- softmax and sums: a token of the tile, then a column of the head and half of the rows ----
    constexpr int RH = RP / 2;
    const int quarter = warp & 3;                 // the tensor-memory lanes this warp may touch
    const int half = (warp - kSoftmaxWarp) >> 2;  // of the tile's tokens, later of the rows
    const int me = quarter * 32 + lane, tid = half * 128 + me;
    const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
    const int step_shift = p.page_shift - 3;      // 32 pages are 2^step_shift tiles
    bool ok = true;

    Queries<T, D, RP, PARTS> queries;
    auto stage = [&](const Cursor& at, int of) {
      stage_queries<T, D, RP, PARTS>(p, queries.raw, at.seq.len - p.nq, at.at.row_tile, tid, sh.q[of & 1],
                                     sh.q_factor[of & 1], sh.q_at[of & 1], sh.q_out[of & 3]);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&sh.q_full[of & 1]));
    };
    auto load_behind = [&](const Cursor& at) {     // the queries of the item behind this one, if it is ours
      if (at.left <= at.seq.count - at.at.tile) return;
      Cursor behind = at;
      behind.advance(p, at.seq.count - at.at.tile);
      queries.load(p, behind, tid);
    };
    if (c.left > 0) {
      queries.load(p, c, tid);
      stage(c, 0);
      named_barrier_sync(1, 256);    // the rows' factors and positions are written
      load_behind(c);
    }

    // An item is finished behind the first maxima of the next one, where its last product has long
    // been there and so have the other warps' row sums.
    T* last_out = nullptr;
    int last_part = 0;
    bool last_direct = false;
    using Pair = unsigned long long;  // of two rows' numbers
    Pair acc[RH / 2];                // of this half's rows and this thread's column
    Pair l[RP / 2];                  // of this thread's tokens
    float m = -INFINITY;             // the reference of row lane % RP, log2 units
#pragma unroll
    for (int r = 0; r < RP / 2; ++r) l[r] = 0;
#pragma unroll
    for (int i = 0; i < RH / 2; ++i) acc[i] = 0;
    const Pair sixteenth = pack2(0.0625f, 0.0625f);
    // pairs of RP or RH numbers in shared memory
    auto pairs_of = [](const float* from, auto& to) {
      constexpr int n = sizeof(to) / sizeof(to[0]);
      if constexpr (n % 2 == 0) {
#pragma unroll
        for (int i = 0; i < n; i += 2) {
          const ulonglong2 two = *reinterpret_cast<const ulonglong2*>(from + 2 * i);
          to[i] = two.x;
          to[i + 1] = two.y;
        }
      } else {
        to[0] = *reinterpret_cast<const Pair*>(from);
      }
    };

    for (int item = 0, j = 0; ok; ++item) {
      // one item, as much of it as the share has; or none any more, and the last one's end
      const bool more = c.left > 0;
      if (!more && item == 0) break;
      const int to_end = more ? c.seq.count - c.at.tile : 0;
      const int n = more ? min(to_end, c.left) : 1;
      // The next item's queries are staged before this one's first tile, so that its products follow this
      // one's without a pause, and the ones behind it are loaded.  Where they go, the item before has
      // been read from: all warps' maxima of its last tile were there.
      const bool stage_next = more && c.left > to_end;
      if (stage_next) {
        Cursor next = c;                 // worked out again at the item's end: it is not worth its registers
        next.advance(p, to_end);
        stage(next, item + 1);
        load_behind(next);
      }
#pragma unroll 1
      for (int k = 0; k < n && ok; ++k) {
        const int x = j & 1;
        const int t0 = tile_start(p, c.seq, c.at.tile + k), token = t0 + tid;
        Pair s[RP / 2];
        float inv_vs = 0.0f;
        bool plain = true;                         // seen by every row of the item, as far as is known without looking closer
        if (more) {
          const int step = j >> step_shift;
          ok = mbar_wait(smem_u32(&sh.scale_full[step & 3]), (step >> 2) & 1, ctx, ST_KV_SCALES, j) &&
               mbar_wait(smem_u32(&sh.s_full[x]), (j >> 1) & 1, ctx, ST_KV_S, j);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          tc_fence_after_sync();
          // eight rows' products at a time: more do not fit the registers
          constexpr int ROWS = RP < 8 ? RP : 8;
          uint32_t raw[PARTS][ROWS];
          auto fetch = [&](int first) {
#pragma unroll
            for (int part = 0; part < PARTS; ++part)
              tmem_ld_few(tmem + lane_base + (x * H + half) * N + part * RP + first, raw[part]);
          };
          fetch(0);
          // every query sees the whole tile: no masks but whether the page is there
          const bool clean = t0 + kTile <= c.seq.limit && t0 + kTile - 1 <= c.seq.len - p.nq &&
                             (!p.window || t0 > c.seq.len - 1 - p.window || t0 + kTile <= p.sinks);
          const float4 scale = sh.scale[step & 3][((j << (8 - p.page_shift)) + (tid >> p.page_shift)) & 31];
          inv_vs = scale.z;
          // seen by some query, and its page is there
          const bool there = scale.w != 0.0f && (clean || seen_by_any(c.seq, token));
          plain = there;
          Pair factor[RP / 2];
          pairs_of(sh.q_factor[item & 1], factor);
          const Pair ks = pack2(scale.x, scale.x), log_vs = pack2(scale.y, scale.y);
#pragma unroll
          for (int first = 0; first < RP; first += ROWS) {
            if (first > 0) fetch(first);
            tmem_ld_wait();
#pragma unroll
            for (int part = 0; part < PARTS; ++part) keep_behind(raw[part]);
            auto product = [&](int part, int r) { return pack2(__uint_as_float(raw[part][2 * r]), __uint_as_float(raw[part][2 * r + 1])); };
#pragma unroll
            for (int r = 0; r < ROWS / 2; ++r) {
              Pair v = product(PARTS - 1, r);
#pragma unroll
              for (int part = PARTS - 2; part >= 0; --part) v = fma2(v, sixteenth, product(part, r));
              // a row that only pads has a product of zero and is as good as any: nobody reads it
              s[first / 2 + r] = fma2(v, mul2(factor[first / 2 + r], ks), log_vs);
            }
          }
          if (!there) {
#pragma unroll
            for (int r = 0; r < RP / 2; ++r) s[r] = pack2(-INFINITY, -INFINITY);
          }
          if (!clean) {                          // tokens that some rows do not see
            const int* at = sh.q_at[item & 1];
            auto seen = [&](int r) { return token <= at[r] && (!p.window || token > at[r] - p.window || token < p.sinks); };
#pragma unroll
            for (int r = 0; r < RP / 2; ++r) {
              float a, b;
              unpack2(s[r], a, b);
              s[r] = pack2(seen(2 * r) ? a : -INFINITY, seen(2 * r + 1) ? b : -INFINITY);
            }
            // the item's rows are those of neighbouring positions, the first row's the lowest; one query
            // token's rows see the same
            const int low = at[0], high = c.seq.len - 1;
            if (p.nq > 1) plain = there && token <= low && (!p.window || token > high - p.window || token < p.sinks);
          }
#pragma unroll
          for (int r = 0; r < RP; r += 4) {
            float a, b, c0, d;
            unpack2(s[r / 2], a, b);
            unpack2(s[r / 2 + 1], c0, d);
            const float4 w = make_float4(warp_max(a), warp_max(b), warp_max(c0), warp_max(d));
            if (lane == 0) *reinterpret_cast<float4*>(&sh.most[x][warp - kSoftmaxWarp][r]) = w;
          }
          if (lane == 0) mbar_arrive(smem_u32(&sh.most_full[x]));
        }
        // while the warps' maxima get together, the product of the tile before joins the sums with
        // the factors of its own step
        if (k + item > 0) {
          ok = mbar_wait(smem_u32(&sh.o_full), (j - 1) & 1, ctx, ST_KV_O, j);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          tc_fence_after_sync();
          uint32_t raw[PARTS][RH];
#pragma unroll
          for (int part = 0; part < PARTS; ++part)
            tmem_ld_few(tmem + lane_base + S::kTmemO + part * RP + half * RH, raw[part]);
          tmem_ld_wait();
#pragma unroll
          for (int part = 0; part < PARTS; ++part) keep_behind(raw[part]);
          Pair old[RH / 2], fresh[RH / 2];
          pairs_of(&sh.step[warp - kSoftmaxWarp][1][half * RH], old);
          pairs_of(&sh.step[warp - kSoftmaxWarp][2][half * RH], fresh);
#pragma unroll
          for (int i = 0; i < RH / 2; ++i) {
            auto product = [&](int part) { return pack2(__uint_as_float(raw[part][2 * i]), __uint_as_float(raw[part][2 * i + 1])); };
            Pair v = product(PARTS - 1);
#pragma unroll
            for (int part = PARTS - 2; part >= 0; --part) v = fma2(v, sixteenth, product(part));
            acc[i] = fma2(v, fresh[i], mul2(acc[i], old[i]));
          }
          if (k == 0) {                          // of the item before: its end
            const int of = item - 1;
            ok = mbar_wait(smem_u32(&sh.sum_full), of & 1, ctx, ST_KV_SUM, of);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
#pragma unroll
            for (int i = 0; i < RH; ++i) {
              const int r = half * RH + i;
              float even, odd;
              unpack2(acc[i / 2], even, odd);
              float total = i % 2 ? odd : even;
              if (quarter * 32 < D) {            // this warp's own word
                const uint32_t nan = sh.nan[of & 1][r][quarter];
                if (nan) {
                  if (nan >> lane & 1) total = NAN;
                  __syncwarp();
                  if (lane == 0) sh.nan[of & 1][r][quarter] = 0;   // for the item after the next one
                }
              }
              float sum = 0.0f;
#pragma unroll
              for (int w = 0; w < 8; ++w) sum += sh.sum[of & 1][w][r];
              if (last_direct) {
                const int64_t at = sh.q_out[of & 3][r];
                if (me < D && at >= 0)
                  last_out[at] = Elem<T>::from_f32(sum > 0.0f ? __fdividef(total, sum) : total * 0.0f);   // nothing seen: 0
              } else {
                if (me < D) p.parts[(last_part + r) * D + me] = total;
                if (quarter == 0 && lane == r) p.marks[last_part + r] = make_float2(m, sum);
              }
            }
#pragma unroll
            for (int i = 0; i < RH / 2; ++i) acc[i] = 0;
#pragma unroll
            for (int r = 0; r < RP / 2; ++r) l[r] = 0;
            m = -INFINITY;
          }
        }
        if (!more) break;
        ok = mbar_wait(smem_u32(&sh.most_full[x]), (j >> 1) & 1, ctx, ST_KV_MOST, j);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        // Lane by lane a row each: the reference its probabilities in this tile are relative to, and
        // what brings the sums so far and the tile to the larger of that and the one before.
        {
          const int r = lane % RP;
          float top = sh.most[x][lane / RP][r];
#pragma unroll
          for (int i = 32 / RP; i < 8; i += 32 / RP) top = fmaxf(top, sh.most[x][lane / RP + i][r]);
#pragma unroll
          for (int o = RP; o < 32; o *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
          const float mt = top - kProbLog2, both = fmaxf(m, mt), ref = both == -INFINITY ? 0.0f : both;
          __syncwarp();                            // everyone has read the last tile's
          if (lane < RP) {
            auto& mine = sh.step[warp - kSoftmaxWarp];
            mine[0][r] = mt == -INFINITY ? 0.0f : -mt;
            mine[1][r] = exp2_approx(m - ref);
            mine[2][r] = exp2_approx(mt - ref);
          }
          m = both;
          __syncwarp();
        }
        const auto& row_step = sh.step[warp - kSoftmaxWarp];
        // probabilities (0 where the row sees nothing of the tile) in parts
        uint32_t bytes[PARTS][RP / 4];
        Pair less[RP / 2], old[RP / 2], fresh[RP / 2];
        pairs_of(row_step[0], less);
        pairs_of(row_step[1], old);
        pairs_of(row_step[2], fresh);
        const Pair inv = pack2(inv_vs, inv_vs);
#pragma unroll
        for (int r = 0; r < RP / 2; ++r) {
          float a, b;
          unpack2(add2(s[r], less[r]), a, b);
          a = exp2_approx(a);
          b = exp2_approx(b);
          l[r] = fma2(mul2(pack2(a, b), inv), fresh[r], mul2(l[r], old[r]));
          uint32_t first = 0;
          if (PARTS > 2) first = split2(a, b);     // what is left of it has 11 bits of its own in fp16
          __half2 pair = __floats2half2_rn(a, b);
#pragma unroll
          for (int part = 0; part < PARTS; ++part) {
            const uint32_t q = PARTS > 2 && part == 0 ? first : split2(pair);
            if (r % 2 == 0) bytes[part][r / 2] = q; else bytes[part][r / 2] |= q << 16;
          }
        }
        // the token's row of P: N bytes, 16 at a time
#pragma unroll
        for (int i = 0; i < N; i += 16) {
          uint32_t w[4];
#pragma unroll
          for (int b = 0; b < 4; ++b) {
            const int at = (i + 4 * b) / RP, r = (i + 4 * b) % RP;
            w[b] = at < PARTS ? bytes[at < PARTS ? at : 0][r / 4] : 0u;
          }
          st_shared_v4(smem_u32(sh.p[half]) + (i / 16) * (kHalf * 16) + me * 16, w[0], w[1], w[2], w[3]);
        }
        if (__any_sync(0xffffffffu, !plain)) {
          const int g = 2 * H * j + H + half;
          ok = mbar_wait(smem_u32(&sh.full[g % SLOTS]), (g / SLOTS) & 1, ctx, ST_KV_ZERO, j);
          ok = __all_sync(0xffffffffu, ok);
          const bool there = sh.scale[(j >> step_shift) & 3][((j << (8 - p.page_shift)) + (tid >> p.page_shift)) & 31].w != 0.0f &&
                             seen_by_any(c.seq, token);
          if (!there) {
#pragma unroll 1
            for (int i = 0; i < D; i += 16)     // neighbours start at different banks
              st_shared_v4(smem_u32(&sh.ring[g % SLOTS][me * D + ((i + me * 16) & (D - 1))]), 0, 0, 0, 0);
          } else if (!plain && ok) {
            set_nan_aside<D, RP>(p, sh.ring[g % SLOTS], me, token, c.seq.len - p.nq, c.at.row_tile, sh.nan[item & 1]);
          }
        }
        fence_proxy_async_smem();
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&sh.p_full));

        ++j;
      }
      if (!ok || !more) break;
      // the row sums over the tokens' threads, on their way
      float sums[RP];
#pragma unroll
      for (int r = 0; r < RP; r += 2) {
        unpack2(l[r / 2], sums[r], sums[r + 1]);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
          sums[r] += __shfl_xor_sync(0xffffffffu, sums[r], o);
          sums[r + 1] += __shfl_xor_sync(0xffffffffu, sums[r + 1], o);
        }
      }
      if (lane == 0) {
#pragma unroll
        for (int r = 0; r < RP; r += 4)
          *reinterpret_cast<float4*>(&sh.sum[item & 1][warp - kSoftmaxWarp][r]) = make_float4(sums[r], sums[r + 1], sums[r + 2], sums[r + 3]);
        mbar_arrive(smem_u32(&sh.sum_full));
      }
      last_out = static_cast<T*>(p.out) + c.at.b * p.o_batch_stride + (int64_t)c.at.head * p.group * p.o_head_stride + me;
      last_direct = c.at.tile == 0 && n == to_end;
      last_part = (2 * blockIdx.x + (item == 0 ? 0 : 1)) * RP;    // the share's first or second part
      if (stage_next) c.advance(p, to_end);
      else c.left = 0;
    }
  }

  tc_fence_before_sync();
  __syncthreads();
  if (*(volatile uint32_t*)&sh.abort_flag) {
    for (int i = 0; i < 64; ++i) __nanosleep(2000);   // let copies in flight land
  }
  if (warp == 1) {
    __syncwarp();
    tc_fence_after_sync();
    tmem_dealloc(tmem, S::kTmemCols);
  }
}

// Joins the parts of the items that were cut, in token order.  An item is found by the first
// boundary between two shares inside it; a thread looks at a boundary.  A row of an item is
// one warp's work, or one block's where there are too few rows to fill the chip (then the items
// have many parts).
template <typename T, int D, int RP>
__global__ void __launch_bounds__(kJoinThreads) kv_join_kernel(const KvAttnParams p) {
  constexpr int kWarps = kJoinThreads / 32, kCols = D / 32;     // columns per lane
  __shared__ Place places[kMaxShares];     // of the boundaries that are the first inside their item
  __shared__ short found[kMaxShares];      // which boundaries those are
  __shared__ int in_warps[kWarps];
  __shared__ float column[kWarps][D];
  __shared__ float2 marks[kWarps][kMaxShares];   // a warp's own: its item's parts
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const WorkList list(p);
  const int share = list.share_start(p, 1);            // all but the last are as long as the first
  int count = 0;
  if (!list.whole_items(p)) {
    // in the order of the boundaries, so that every block has the same list
    for (int c0 = 0; c0 < p.shares - 1; c0 += kJoinThreads) {
      const int c = c0 + tid;
      const int flat = (int)min((c + 1ll) * share, (long long)list.tiles(p) - 1);
      const Place w = list.locate(p, flat);
      const bool mine = c < p.shares - 1 && flat == (c + 1ll) * share && w.tile > 0 && (flat - w.tile) / share == c;
      const uint32_t in_warp = __ballot_sync(0xffffffffu, mine);
      if (lane == 0) in_warps[warp] = __popc(in_warp);
      __syncthreads();
      int index = count + __popc(in_warp & ((1u << lane) - 1));
      for (int i = 0; i < kWarps; ++i) {
        if (i < warp) index += in_warps[i];
        count += in_warps[i];
      }
      if (mine) {
        places[index] = w;
        found[index] = (short)c;
      }
      __syncthreads();
    }
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int units = count * RP;
  const bool by_block = units <= (int)gridDim.x;       // the same everywhere
  const int team = by_block ? kWarps : 1, mine = by_block ? warp : 0;
  for (int u = by_block ? blockIdx.x : blockIdx.x * kWarps + warp; u < units;
       u += by_block ? gridDim.x : gridDim.x * kWarps) {
    const int r = u % RP, first = found[u / RP];
    const Place at = places[u / RP];
    const int begin = (first + 1) * share - at.tile;
    const int end = begin + make_seq(p, __ldg(p.lengths + at.b)).count;
    const int skip = begin != first * share;           // the item is its first share's second part
    const int row = at.row_tile * RP + r;
    if (row >= p.rows) continue;                       // by block: the same in every thread
    const int n = (end - 1) / share - first + 1;
    // part i: the first share's first or second part, the first parts of the shares behind it
    auto part = [&](int i) { return (2 * (first + i) + (i == 0 ? skip : 0)) * RP + r; };
    // the first parts' columns are on their way before any weight is known
    constexpr int kBatch = 8;
    float q[kBatch][kCols];
    auto fetch = [&](int base) {
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        const int i = base + b * team;
#pragma unroll
        for (int k = 0; k < kCols; ++k) q[b][k] = i < n ? p.parts[part(i) * D + lane + k * 32] : 0.0f;
      }
    };
    fetch(mine);
    // weights: every warp works out all of them for itself
    float top = -INFINITY;
    for (int i = lane; i < n; i += 32) {
      const float2 mark = p.marks[part(i)];
      marks[warp][i] = mark;
      top = fmaxf(top, mark.x);
    }
    top = warp_max(top);
    const float ref = top == -INFINITY ? 0.0f : top;
    float sum = 0.0f;
    for (int i = lane; i < n; i += 32) {               // this lane's own
      const float w = exp2_approx(marks[warp][i].x - ref);
      sum = fmaf(marks[warp][i].y, w, sum);
      marks[warp][i].x = w;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    __syncwarp();
    float acc[kCols];
#pragma unroll
    for (int k = 0; k < kCols; ++k) acc[k] = 0.0f;
    for (int base = mine; base < n; base += kBatch * team) {
      if (base != mine) fetch(base);
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        const int i = base + b * team;
        const float w = i < n ? marks[warp][i].x : 0.0f;
#pragma unroll
        for (int k = 0; k < kCols; ++k) acc[k] = fmaf(q[b][k], w, acc[k]);
      }
    }
    __syncwarp();                                      // before marks are written again
    if (by_block) {
      __syncthreads();                                 // the row before has been read
#pragma unroll
      for (int k = 0; k < kCols; ++k) column[warp][k * 32 + lane] = acc[k];
      __syncthreads();
      if (warp != 0) continue;
#pragma unroll
      for (int k = 0; k < kCols; ++k) {
        acc[k] = 0.0f;
#pragma unroll
        for (int i = 0; i < kWarps; ++i) acc[k] += column[i][k * 32 + lane];
      }
    }
    T* dst = static_cast<T*>(p.out) + at.b * p.o_batch_stride + row / p.group * p.o_token_stride +
             (at.head * p.group + row % p.group) * p.o_head_stride + lane;
#pragma unroll
    for (int k = 0; k < kCols; ++k)
      dst[k * 32] = Elem<T>::from_f32(sum > 0.0f ? acc[k] / sum : acc[k] * 0.0f);
  }
}

// ---- host ------------------------------------------------------------------------------------------

// Can a sequence of this many pages be long enough for its items to be cut?
bool can_be_cut(int64_t pages, int64_t page) { return cdiv64(pages * page, kTile) > kWholeTiles; }

int row_tile_of(int64_t rows) {
  int rp = 4;
  while (rp < rows && rp < 16) rp *= 2;
  return rp;
}
int shares_of() {
  const int shares = 2 * device_info().sm_count;
  return shares < kMaxShares ? shares : kMaxShares;
}

template <typename T, int D, int RP, int PARTS>
int launch_kv(KvAttnParams p, const CUtensorMap& mk, const CUtensorMap& mv, cudaStream_t stream) {
  auto kern = kv_attn_kernel<T, D, RP, PARTS>;
  const int smem = (int)sizeof(Shared<D, RP, PARTS>);
  static_assert(sizeof(Shared<D, RP, PARTS>) <= kSmemPerCta, "two CTAs per SM, and room for the joining kernel");
  if (int rc = prepare_kernel((const void*)kern, smem)) return rc;
  kern<<<p.shares, kThreads, smem, stream>>>(mk, mv, p);
  if (int rc = cuda_check(cudaGetLastError(), "kv attention launch")) return rc;
  if (!can_be_cut(p.max_pages, p.page)) return 0;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(4u * (unsigned)device_info().sm_count);
  config.blockDim = dim3(kJoinThreads);
  config.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &attr;
  config.numAttrs = 1;
  return cuda_check(cudaLaunchKernelEx(&config, kv_join_kernel<T, D, RP>, p), "kv attention join launch");
}

template <int D>
int dispatch_kv(const KvAttnParams& p, const CUtensorMap& mk, const CUtensorMap& mv, bool bf16, int rp,
                cudaStream_t stream) {
  if (bf16) {
    if (rp == 4) return launch_kv<__nv_bfloat16, D, 4, 2>(p, mk, mv, stream);
    if (rp == 8) return launch_kv<__nv_bfloat16, D, 8, 2>(p, mk, mv, stream);
    return launch_kv<__nv_bfloat16, D, 16, 2>(p, mk, mv, stream);
  }
  if (rp == 4) return launch_kv<__half, D, 4, 3>(p, mk, mv, stream);
  if (rp == 8) return launch_kv<__half, D, 8, 3>(p, mk, mv, stream);
  return launch_kv<__half, D, 16, 3>(p, mk, mv, stream);
}

int encode_pages(CUtensorMap* map, const void* base, const nb200_kv_cache& c, int64_t page_stride,
                 int64_t head_stride, int64_t token_stride) {
  const uint64_t dims[4] = {(uint64_t)c.head_dim, (uint64_t)c.page_size, (uint64_t)c.heads, (uint64_t)c.pages};
  const uint64_t strides[3] = {(uint64_t)token_stride, (uint64_t)head_stride, (uint64_t)page_stride};
  const uint32_t box[4] = {(uint32_t)c.head_dim, (uint32_t)c.page_size, 1u, 1u};
  return encode_tensor_map(map, base, 1, 4, dims, strides, box);
}

}  // namespace
}  // namespace nb200

using namespace nb200;

extern "C" int64_t nb200_kv_attention_workspace_bytes(const nb200_kv_cache* cache, int64_t batch,
                                                      int64_t queries, int64_t heads,
                                                      int64_t max_pages, int dtype) {
  if (!cache || cache->heads <= 0 || batch <= 0 || queries <= 0 || heads <= 0) return 0;
  if ((dtype != NB200_F16 && dtype != NB200_BF16) || !can_be_cut(max_pages, cache->page_size)) return 0;
  const int rp = row_tile_of(queries * (heads / cache->heads));
  return 2ll * shares_of() * rp * (cache->head_dim * (int64_t)sizeof(float) + (int64_t)sizeof(float2));
}

extern "C" int nb200_kv_attention(const void* q, const nb200_kv_cache* cache, void* out,
                                  int64_t batch, int64_t queries, int64_t heads,
                                  int64_t q_batch_stride, int64_t q_token_stride,
                                  int64_t q_head_stride, int64_t o_batch_stride,
                                  int64_t o_token_stride, int64_t o_head_stride,
                                  const int32_t* page_table, int64_t table_stride,
                                  int64_t max_pages, const int32_t* lengths, float scale,
                                  int64_t window, int64_t sinks, int dtype, void* workspace,
                                  int64_t workspace_bytes, void* stream_) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (int rc = check_kv_cache("kv attention", cache)) return rc;
  if (dtype != NB200_F16 && dtype != NB200_BF16)
    return fail(NB200_E_UNSUPPORTED, "kv attention: dtype code %d (fp16 and bf16 only)", dtype);
  if (batch < 0 || queries < 0 || heads < 0 || max_pages < 0 || batch > (1 << 20) || queries > (1 << 20) ||
      heads > 65535 || max_pages > (1 << 30) / cache->page_size)
    return fail(NB200_E_INVALID, "kv attention: bad extent (batch=%lld queries=%lld heads=%lld max_pages=%lld)",
                (long long)batch, (long long)queries, (long long)heads, (long long)max_pages);
  if (batch == 0 || queries == 0 || heads == 0) return 0;
  if (heads % cache->heads)
    return fail(NB200_E_INVALID, "kv attention: %lld query heads over %lld heads of the cache",
                (long long)heads, (long long)cache->heads);
  if (window < 0 || sinks < 0 || window > INT32_MAX || sinks > INT32_MAX)
    return fail(NB200_E_INVALID, "kv attention: window %lld, sinks %lld", (long long)window, (long long)sinks);
  if (!(scale > 0.0f) || scale > 1e30f)
    return fail(NB200_E_INVALID, "kv attention: scale must be positive and finite");
  if (!q || !out || !lengths || (max_pages > 0 && !page_table))
    return fail(NB200_E_INVALID, "kv attention: null tensor pointer");
  if (!aligned_to(2, q, out) || !aligned_to(4, page_table, lengths))
    return fail(NB200_E_INVALID, "kv attention: a tensor does not start on a multiple of its element");
  if (q == out) return fail(NB200_E_INVALID, "kv attention: out must not be q, which other blocks still read");
  if (cache->pages == 0) return fail(NB200_E_INVALID, "kv attention: the cache has no pages");
  const int64_t need = nb200_kv_attention_workspace_bytes(cache, batch, queries, heads, max_pages, dtype);
  if (need > 0 && (!workspace || workspace_bytes < need || !at16(workspace)))
    return fail(NB200_E_INVALID, "kv attention: a 16-byte aligned workspace of %lld bytes is needed (given %lld)",
                (long long)need, (long long)workspace_bytes);
  const bool bf16 = dtype == NB200_BF16;
  KvAttnParams p;
  p.q = q;
  p.out = out;
  p.k_scales = cache->k_scales;
  p.v_scales = cache->v_scales;
  p.table = page_table;
  p.lengths = lengths;
  p.parts = static_cast<float*>(workspace);
  p.q_batch_stride = q_batch_stride;
  p.q_token_stride = q_token_stride;
  p.q_head_stride = q_head_stride;
  p.o_batch_stride = o_batch_stride;
  p.o_token_stride = o_token_stride;
  p.o_head_stride = o_head_stride;
  p.table_stride = table_stride;
  p.k_scale_stride = cache->k_scale_stride;
  p.v_scale_stride = cache->v_scale_stride;
  p.batch = (int)batch;
  p.nq = (int)queries;
  p.kv_heads = (int)cache->heads;
  p.group = (int)(heads / cache->heads);
  if (queries * p.group > INT32_MAX / 64) return fail(NB200_E_INVALID, "kv attention: too many rows per key head");
  p.rows = (int)queries * p.group;
  const int rp = row_tile_of(p.rows);
  p.row_tiles = (p.rows + rp - 1) / rp;
  p.per_seq = p.row_tiles * p.kv_heads;
  p.stretch = (p.batch + 31) / 32;
  // the work list is counted in 32 bits
  const int64_t most_tiles = cdiv64(max_pages * cache->page_size, kHalf) + 1;
  if ((double)most_tiles * batch * p.row_tiles * p.kv_heads > 2e9)
    return fail(NB200_E_UNSUPPORTED, "kv attention: %lld sequences of up to %lld tokens, %lld query tokens: split the batch",
                (long long)batch, (long long)(max_pages * cache->page_size), (long long)queries);
  p.pages = (int)cache->pages;
  p.page = (int)cache->page_size;
  p.page_shift = p.page == 16 ? 4 : p.page == 32 ? 5 : p.page == 64 ? 6 : 7;
  p.max_pages = (int)max_pages;
  p.window = (int)window;
  p.sinks = (int)sinks;
  p.shares = shares_of();
  p.share_items = p.batch * p.per_seq / p.shares;
  p.longer_shares = p.batch * p.per_seq % p.shares;
  p.by_shares = Divisor(p.shares);
  p.by_per_seq = Divisor(p.per_seq);
  p.by_row_tiles = Divisor(p.row_tiles);
  p.by_stretch = Divisor(p.stretch);
  p.marks = need > 0 ? reinterpret_cast<float2*>(p.parts + 2ll * p.shares * rp * cache->head_dim) : nullptr;
  p.q_aligned = at16(q) && q_batch_stride % 8 == 0 && q_token_stride % 8 == 0 && q_head_stride % 8 == 0;
  p.scale = scale;
  p.wait_limit_ns = wait_limit_ns();
  p.status = device_status_ptr();
  if (!p.status) return fail(NB200_E_CUDA, "kv attention: device status word is not addressable");
  CUtensorMap mk, mv;
  if (int rc = encode_pages(&mk, cache->k, *cache, cache->k_page_stride, cache->k_head_stride, cache->k_token_stride))
    return rc;
  if (int rc = encode_pages(&mv, cache->v, *cache, cache->v_page_stride, cache->v_head_stride, cache->v_token_stride))
    return rc;
  return cache->head_dim == 128 ? dispatch_kv<128>(p, mk, mv, bf16, rp, stream)
                                : dispatch_kv<64>(p, mk, mv, bf16, rp, stream);
}
