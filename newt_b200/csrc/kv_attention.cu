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
// first rounding leaves over fits the second), an fp16 takes three.  So the queries lose nothing,
// and the probabilities keep 9 or 14 bits.  N = parts * rows, at least 16, was idle anyway.
//
// Per tile of 128 tokens a thread owns one token: it reads its N scores from tensor memory, applies
// both scales and the masks, and takes part in the rows' maxima over the tile (warp reductions and
// one exchange through shared memory).  Probabilities are relative to the tile's own maximum
// (of s + log2 vs, so that they fit e4m3 whatever the scales); the tile's product is read back --
// now a thread owns one of the head's columns -- and joins the running sums in registers with the
// usual rescaling, in fp32.  P is laid out so that a thread writes its token's N bytes in one piece.
//
// Value rows that no query sees are cleared in shared memory before the product: their weight is
// zero, but zero times a NaN that was left in a page would not be.
//
// Work: all (sequence, row tile, key head) items in order, each a run of visible tiles (those of
// the first tokens, then those of the window), cut into equal shares for a grid that fills the
// chip.  A share may start and end inside an item; such parts leave their sums in the workspace and
// a second kernel joins them, in token order.  Lengths are read on the device, so a captured call
// follows them.

#include <type_traits>

#include "elem.cuh"
#include "kv_cache.cuh"
#include "sm100.cuh"

namespace nb200 {
namespace {

using namespace sm100;

constexpr int kTile = 128;               // tokens
constexpr int kThreads = 192;            // producer, issuer, four softmax warps
constexpr int kSoftmaxWarp = 2;
constexpr int kJoinThreads = 512;
constexpr int kMinShare = 2;             // tiles
constexpr int kWholeItems = 4;           // tiles
constexpr int kMaxShares = kJoinThreads;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLeastScale = 8.67361738e-19f;   // 2^-60
constexpr float kProbScale = 256.0f;     // probabilities of a tile are at most 1

enum : unsigned int {
  ST_KV_Q = 32, ST_KV_K, ST_KV_V, ST_KV_EMPTY, ST_KV_SCALES, ST_KV_S, ST_KV_P, ST_KV_O, ST_KV_ZERO
};

struct KvAttnParams {
  const void* q;
  void* out;
  const float *k_scales, *v_scales;
  const int32_t* table;
  const int32_t* lengths;
  float* parts;                          // [2 * shares][rows padded][head_dim + 2]
  int64_t q_batch_stride, q_token_stride, q_head_stride;
  int64_t o_batch_stride, o_token_stride, o_head_stride;
  int64_t table_stride, k_scale_stride, v_scale_stride;
  int batch, nq, kv_heads, group;        // group: query heads per key head
  int rows, row_tiles;                   // nq * group, and how many pieces of RP rows
  int pages, page, page_shift, max_pages, window, sinks;
  int shares, q_aligned;
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
  const int tiles = (s.limit + kTile - 1) / kTile;
  s.first = s.from = 0;
  s.count = tiles;
  if (s.low > 0) {
    const int sink_tiles = (s.sink_end + kTile - 1) / kTile;
    if (s.low / kTile > sink_tiles) {
      s.first = sink_tiles;
      s.from = s.low / kTile;
      s.count = sink_tiles + max(tiles - s.from, 0);
    }
  }
  s.count = max(s.count, 1);       // a sequence without tokens has its zeros to write
  return s;
}
__device__ __forceinline__ int tile_start(const Seq& s, int t) {
  return (t < s.first ? t : t - s.first + s.from) * kTile;
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
  int stretch, before, sum;   // of this lane's stretch, for one (key head, row tile)
  int total, largest;         // of all: tiles of one (key head, row tile), most of one sequence
  int per_seq;

  __device__ WorkList(const KvAttnParams& p) {
    const int lane = threadIdx.x & 31;
    per_seq = p.row_tiles * p.kv_heads;
    stretch = (p.batch + 31) / 32;
    sum = largest = 0;
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
  __device__ int tiles() const { return total * per_seq; }

  // Shares of whole items where all are short (a cut would cost more than it evens out: below),
  // of tiles otherwise.
  __device__ bool whole_items() const { return largest <= kWholeItems; }

  // first tile of share c, from 0 to tiles(); the same c in all lanes
  __device__ int share_start(const KvAttnParams& p, int c) const {
    if (!whole_items()) {
      const int share = max((tiles() + p.shares - 1) / p.shares, kMinShare);
      return (int)min((long long)c * share, (long long)tiles());
    }
    const int items = p.batch * per_seq;
    const int i = (int)((long long)items * c / p.shares);
    if (i >= items) return tiles();
    const int b = i / per_seq, owner = b / stretch;
    int at = __shfl_sync(0xffffffffu, before, owner);
    for (int k = owner * stretch; k < b; ++k) at += make_seq(p, __ldg(p.lengths + k)).count;
    return at * per_seq + (i - b * per_seq) * make_seq(p, __ldg(p.lengths + b)).count;
  }

  // The place of a tile, 0 <= flat < tiles(), a tile of its own for every lane if need be.
  __device__ Place locate(const KvAttnParams& p, int flat) const {
    const int q = flat / per_seq;            // at * per_seq <= flat  <=>  at <= flat / per_seq
    int owner = 0;
#pragma unroll
    for (int step = 16; step > 0; step >>= 1)
      if (__shfl_sync(0xffffffffu, before, owner + step) <= q) owner += step;
    int at = __shfl_sync(0xffffffffu, before, owner);
    int b = owner * stretch;
    int count = make_seq(p, __ldg(p.lengths + b)).count;
    while (q >= at + count) {
      at += count;
      ++b;
      count = make_seq(p, __ldg(p.lengths + b)).count;
    }
    flat -= at * per_seq;
    const int item = flat / count;
    return Place{b, item / p.row_tiles, item % p.row_tiles, flat % count};
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
    while (left > 0 && at.tile >= seq.count) {
      at.tile -= seq.count;
      next_item(p);
    }
  }
};

template <int D, int RP, int PARTS>
struct Shape {
  static constexpr int kN = (RP * PARTS + 15) / 16 * 16;
  static constexpr int kTileBytes = kTile * D;                    // one K or V tile
  // ring of K0 V0 K1 V1 ...: what two CTAs per SM leave room for
  static constexpr int kSlots = D == 128 ? (kN >= 32 ? 4 : 6) : (kN >= 48 ? 10 : 12);
  static constexpr int kQBytes = kN * D;
  static constexpr int kPBytes = kN * kTile;
  static constexpr int kTmemCols = 4 * kN <= 64 ? 64 : 4 * kN <= 128 ? 128 : 256;
};

template <int D, int RP, int PARTS>
struct Shared {
  using S = Shape<D, RP, PARTS>;
  uint8_t ring[S::kSlots][S::kTileBytes];      // first: the swizzle counts from 1024-byte boundaries
  uint8_t p[2][S::kPBytes];
  uint8_t q[2][S::kQBytes];
  float4 scale[4][32];                         // of a step's pages: ks, log2 vs, 1 / vs, 1 if it is there
  float q_factor[2][RP];                       // what takes a row's product to log2 units
  int q_at[2][RP];                             // position of the row's query; -1: no such row
  float most[2][4][RP];                        // the warps' maxima, alternating by tile
  float sum[4][RP];
  uint64_t full[S::kSlots], empty[S::kSlots], scale_full[4];
  uint64_t q_full[2], s_full[2], p_full[2], o_full[2];
  uint32_t tmem_slot, abort_flag;
};

// Two values as e4m3 (low and high byte), and what is left of them, times 16.
__device__ __forceinline__ uint32_t split2(float& a, float& b) {
  const uint32_t q = e4m3x2(a, b);
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)q, __NV_E4M3);
  const float2 f = __half22float2(__half2(h));
  a = (a - f.x) * 16.0f;
  b = (b - f.y) * 16.0f;
  return q;
}

// Softmax threads: 0..127 here.  `ok` of all of them, behind a barrier.
__device__ __forceinline__ bool all_of_group(bool ok) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %1, 0;\n\t"
      "barrier.cta.red.and.pred q, 1, 128, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"((uint32_t)ok)
      : "memory");
  return r != 0;
}

// Queries of one item on their way from global memory to their e4m3 parts: 8 columns of a row per
// vector, kVectors per thread.
template <typename T, int D, int RP, int PARTS>
struct Queries {
  static constexpr int kPerRow = D / 8;
  static constexpr int kVectors = RP * kPerRow / 128 > 0 ? RP * kPerRow / 128 : 1;
  Vec<T> raw[kVectors];

  __device__ void load(const KvAttnParams& p, const Cursor& c, int tid) {
#pragma unroll
    for (int i = 0; i < kVectors; ++i) {
      const int v = i * 128 + tid;
      const int r = c.at.row_tile * RP + v / kPerRow;
      raw[i].raw = make_uint4(0, 0, 0, 0);
      if (v / kPerRow >= RP || r >= p.rows) continue;
      const T* src = static_cast<const T*>(p.q) + c.at.b * p.q_batch_stride +
                     r / p.group * p.q_token_stride +
                     (c.at.head * p.group + r % p.group) * p.q_head_stride + v % kPerRow * 8;
      if (p.q_aligned) {
        raw[i].raw = __ldg(reinterpret_cast<const uint4*>(src));
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) raw[i].e[j] = src[j];
      }
    }
  }

  // Row r times 2^-e fits e4m3's range; 2^e goes into the row's factor.  Parts of row r are rows r,
  // RP + r, ... of the operand, K-major under the swizzle of its row length.
  __device__ void stage(const KvAttnParams& p, const Cursor& c, int tid, uint8_t* q, float* factor, int* at) {
#pragma unroll
    for (int i = 0; i < kVectors; ++i) {
      const int v = i * 128 + tid;
      const int r = v / kPerRow, col8 = v % kPerRow;
      float f[8], most = 0.0f;
      bool bad = false;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        f[j] = Elem<T>::to_f32(raw[i].e[j]);
        most = fmaxf(most, fabsf(f[j]));
        bad |= !(fabsf(f[j]) < INFINITY);
      }
#pragma unroll
      for (int o = kPerRow / 2; o > 0; o >>= 1) {
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
        bad |= (bool)__shfl_xor_sync(0xffffffffu, (int)bad, o);
      }
      // most <= 448 * 2^e: 448 = 1.75 * 2^8
      const uint32_t bits = __float_as_uint(most);
      int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
      e = max(e, -100);
      const float down = __uint_as_float((uint32_t)(127 - e) << 23);
      if (r < RP) {
        if (col8 == 0) {
          const int row = c.at.row_tile * RP + r;
          factor[r] = bad ? NAN : __uint_as_float((uint32_t)(127 + e) << 23) * (p.scale * kLog2e);
          at[r] = row < p.rows ? c.seq.len - p.nq + row / p.group : -1;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] *= down;
#pragma unroll
        for (int part = 0; part < PARTS; ++part) {
          const uint32_t w0 = split2(f[0], f[1]), w1 = split2(f[2], f[3]);
          const uint32_t w2 = split2(f[4], f[5]), w3 = split2(f[6], f[7]);
          const int n = part * RP + r;
          const int chunk = (col8 >> 1) ^ (D == 128 ? (n & 7) : ((n >> 1) & 3));
          *reinterpret_cast<uint2*>(q + n * D + chunk * 16 + (col8 & 1) * 8) =
              make_uint2(w0 | (w1 << 16), w2 | (w3 << 16));
        }
      }
    }
  }
};

template <typename T, int D, int RP, int PARTS>
__global__ void __launch_bounds__(kThreads, 2)
    kv_attn_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                   const KvAttnParams p) {
  using S = Shape<D, RP, PARTS>;
  constexpr int N = S::kN, SLOTS = S::kSlots;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  Shared<D, RP, PARTS>& sh = *reinterpret_cast<Shared<D, RP, PARTS>*>(smem_raw);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const WaitCtx ctx{&sh.abort_flag, p.status, p.wait_limit_ns};

  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");   // the joining kernel may get ready
  if (threadIdx.x == 0) {
    sh.abort_flag = 0;
    for (int x = 0; x < SLOTS; ++x) {
      mbar_init(smem_u32(&sh.full[x]), 1);
      mbar_init(smem_u32(&sh.empty[x]), 1);
    }
    for (int x = 0; x < 4; ++x) mbar_init(smem_u32(&sh.scale_full[x]), 1);
    for (int x = 0; x < 2; ++x) {
      mbar_init(smem_u32(&sh.q_full[x]), 4);   // one arrival per softmax warp
      mbar_init(smem_u32(&sh.s_full[x]), 1);
      mbar_init(smem_u32(&sh.p_full[x]), 4);
      mbar_init(smem_u32(&sh.o_full[x]), 1);
    }
    mbar_init_fence();
    prefetch_tensormap(&map_k);
    prefetch_tensormap(&map_v);
  }
  __syncwarp();
  if (warp == 1) tmem_alloc(smem_u32(&sh.tmem_slot), S::kTmemCols);
  // every warp finds the share's place for itself
  const WorkList list(p);
  const int from = list.share_start(p, blockIdx.x), to = list.share_start(p, blockIdx.x + 1);
  Cursor c;
  c.start(p, to > from ? list.locate(p, from) : Place{0, 0, 0, 0}, to - from);
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = sh.tmem_slot;

  if (warp == 0) {
    // ---- producer ----
    // It works in steps of 32 pages, a lane per page: pages are looked up two steps ahead and their
    // scales fetched one step ahead, so that neither latency is met per tile.  The scales go to the
    // softmax warps through four turns of shared memory: a step begins when the ring has room for
    // it, that is when all but the ring's tiles before it are done with, and the ring has at most
    // 6 tiles where three steps have at least 12.
    static_assert(SLOTS / 2 <= 12, "a turn of the scales would be overwritten too early");
    const int per_tile = kTile >> p.page_shift, step_tiles = 32 / per_tile;
    const uint32_t page_bytes = (uint32_t)p.page * D;
    const int my_tile = lane / per_tile, my_page = lane % per_tile;
    Cursor mine = c;
    auto page_of = [&](Cursor& at) {             // this lane's page, -1: not to be read
      if (at.left <= 0) return -1;
      const int token = tile_start(at.seq, at.at.tile) + (my_page << p.page_shift);
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
    if (c.left > 0) mine.advance(p, my_tile);
    id[0] = page_of(mine);
    head[0] = mine.at.head;
    if (mine.left > 0) mine.advance(p, step_tiles);
    id[1] = page_of(mine);
    head[1] = mine.at.head;
    fetch_scales(id[0], head[0], ks[0], vs[0]);
    bool ok = true;
    int left = c.left;
    for (int step = 0; left > 0 && ok; ++step) {
      // the next step's scales and the one after's pages are under way while this one is issued
      fetch_scales(id[1], head[1], ks[1], vs[1]);
      if (mine.left > 0) mine.advance(p, step_tiles);
      id[2] = page_of(mine);
      head[2] = mine.at.head;
      bool handed = false;
      for (int k = 0; k < step_tiles && left > 0 && ok; ++k, --left) {
        const int j = step * step_tiles + k;
        const bool in_tile = my_tile == k && id[0] >= 0;
        const uint32_t bytes = __popc(__ballot_sync(0xffffffffu, in_tile)) * page_bytes;
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
          const int g = 2 * j + kv, x = g % SLOTS;
          ok = ok && mbar_wait_nocall(smem_u32(&sh.empty[x]), ((g / SLOTS) & 1) ^ 1, ctx, ST_KV_EMPTY, g);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          const uint32_t bar = smem_u32(&sh.full[x]);
          if (lane == 0) {
            if (bytes) mbar_arrive_expect_tx(bar, bytes); else mbar_arrive(bar);
          }
          __syncwarp();
          if (in_tile)
            tma_load_4d(smem_u32(&sh.ring[x][my_page * page_bytes]), kv ? &map_v : &map_k, 0, 0, head[0], id[0], bar);
        }
        if (!handed) {                           // behind the first tile's copies
          if (vs[0] < kLeastScale) vs[0] = kLeastScale;   // its logarithm is used; NaN stays
          sh.scale[step & 3][lane] = make_float4(ks[0], __log2f(vs[0]), 1.0f / vs[0], id[0] >= 0 ? 1.0f : 0.0f);
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&sh.scale_full[step & 3]));
          handed = true;
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
    constexpr uint32_t kIdescQk = instr_desc_e4m3(kTile, N, false, false);
    constexpr uint32_t kIdescPv = instr_desc_e4m3(kTile, N, true, true);
    constexpr uint64_t kKMajor = D == 128 ? smem_desc_sw128(16, 1024) : smem_desc_sw64(16, 512);
    // head_dim 64 fills half of the 128 rows: the second slab of 64 is the first one again
    constexpr uint64_t kVDesc = D == 128 ? smem_desc_sw128(16, 1024) : smem_desc_sw64(0, 512);
    constexpr uint64_t kPDesc = smem_desc_plain(128, kTile * 16);
    auto wait_all = [&](uint64_t* bar, uint32_t parity, unsigned int code, int detail) -> bool {
      return __all_sync(0xffffffffu, mbar_wait_nocall(smem_u32(bar), parity, ctx, code, detail));
    };
    auto scores = [&](int j, int item) {           // S(j) = K(j) Q of the item
      const uint32_t kb = smem_u32(sh.ring[2 * j % SLOTS]), qb = smem_u32(sh.q[item & 1]);
#pragma unroll
      for (int kk = 0; kk < D / 32; ++kk)
        if (elected)
          mma_f8_ss(tmem + (j & 1) * N, with_address(kKMajor, kb + kk * 32),
                    with_address(kKMajor, qb + kk * 32), kIdescQk, kk != 0);
      if (elected) {
        mma_commit(smem_u32(&sh.s_full[j & 1]));
        mma_commit(smem_u32(&sh.empty[2 * j % SLOTS]));
      }
    };
    bool ok = true;
    int item = 0;                    // items begun
    auto begin = [&](int j, bool new_item) {
      if (new_item) ok = wait_all(&sh.q_full[item & 1], (item >> 1) & 1, ST_KV_Q, item);
      ok = ok && wait_all(&sh.full[2 * j % SLOTS], (2 * j / SLOTS) & 1, ST_KV_K, j);
      if (!ok) return;
      tc_fence_after_sync();
      scores(j, item);
      __syncwarp();
    };
    if (c.left > 0) begin(0, true);
    for (int j = 0; c.left > 0 && ok; ++j) {
      const bool ends = c.last_tile();
      c.advance(p, 1);
      if (c.left > 0) {
        if (ends) ++item;
        begin(j + 1, ends);
      }
      const int x = (2 * j + 1) % SLOTS;
      ok = ok && wait_all(&sh.full[x], ((2 * j + 1) / SLOTS) & 1, ST_KV_V, j);
      ok = ok && wait_all(&sh.p_full[j & 1], (j >> 1) & 1, ST_KV_P, j);
      if (!ok) break;
      tc_fence_after_sync();
      const uint32_t vb = smem_u32(sh.ring[x]), pb = smem_u32(sh.p[j & 1]);
#pragma unroll
      for (int kk = 0; kk < kTile / 32; ++kk)      // 32 tokens: four groups of eight rows
        if (elected)
          mma_f8_ss(tmem + (2 + (j & 1)) * N, with_address(kVDesc, vb + kk * 32 * D),
                    with_address(kPDesc, pb + kk * 4 * 128), kIdescPv, kk != 0);
      if (elected) {
        mma_commit(smem_u32(&sh.o_full[j & 1]));
        mma_commit(smem_u32(&sh.empty[x]));
      }
      __syncwarp();
    }
  } else {
    // ---- softmax and sums: a token of the tile, then a column of the head ----
    const int quarter = warp & 3;                 // the tensor-memory lanes this warp may touch
    const int me = quarter * 32 + lane;
    const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
    bool ok = true;

    Queries<T, D, RP, PARTS> queries;
    if (c.left > 0) {
      queries.load(p, c, me);
      queries.stage(p, c, me, sh.q[0], sh.q_factor[0], sh.q_at[0]);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&sh.q_full[0]));
      all_of_group(true);            // the rows' factors and positions are written
    }

    int item = 0;
    bool whole = c.at.tile == 0;                   // has the item's first tile
    bool first_part = true;                        // the item that the share begins with
    float acc[RP], l[RP], m[RP], now[RP];          // m: log2 units
#pragma unroll
    for (int r = 0; r < RP; ++r) {
      acc[r] = l[r] = now[r] = 0.0f;
      m[r] = -INFINITY;
    }
    // the product of tile j joins the sums with the factors that its own step left in `now`
    auto add_product = [&](int j) {
      ok = ok && mbar_wait_nocall(smem_u32(&sh.o_full[j & 1]), (j >> 1) & 1, ctx, ST_KV_O, j);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) return;
      tc_fence_after_sync();
      uint32_t raw[N];
#pragma unroll
      for (int n = 0; n < N; n += 16)
        tmem_ld_32x32(tmem + lane_base + (2 + (j & 1)) * N + n, *reinterpret_cast<uint32_t (*)[16]>(&raw[n]));
      tmem_ld_wait(raw);
#pragma unroll
      for (int r = 0; r < RP; ++r) {
        float v = __uint_as_float(raw[(PARTS - 1) * RP + r]);
#pragma unroll
        for (int part = PARTS - 2; part >= 0; --part)
          v = fmaf(v, 0.0625f, __uint_as_float(raw[part * RP + r]));
        acc[r] = fmaf(v, now[r], acc[r]);
      }
    };
    bool pending = false;                          // a product of this item has not joined yet
    for (int j = 0; c.left > 0; ++j) {
      // the next item's queries: loaded at the start of an item, staged behind its first tile
      const int skip = c.seq.count - c.at.tile;    // tiles to the next item
      const bool stage_next = (j == 0 || c.at.tile == 0) && c.left > skip;
      Cursor next_item = c;
      if (stage_next) {
        next_item.advance(p, skip);
        queries.load(p, next_item, me);
      }

      const int x = j & 1;
      const int t0 = tile_start(c.seq, c.at.tile);
      const int token = t0 + me;
      // every query sees the whole tile: no masks but whether the page is there
      const bool clean = t0 + kTile <= c.seq.limit && t0 + kTile - 1 <= c.seq.len - p.nq &&
                         (!p.window || t0 > c.seq.len - 1 - p.window || t0 + kTile <= p.sinks);
      const int step = (unsigned)j >> (p.page_shift - 2);    // 32 pages: 2^(shift - 2) tiles
      ok = ok && mbar_wait_nocall(smem_u32(&sh.scale_full[step & 3]), (step >> 2) & 1, ctx, ST_KV_SCALES, j);
      ok = ok && mbar_wait_nocall(smem_u32(&sh.s_full[x]), (j >> 1) & 1, ctx, ST_KV_S, j);
      ok = __all_sync(0xffffffffu, ok);
      const float4 scale = sh.scale[step & 3][((j << (7 - p.page_shift)) + (me >> p.page_shift)) & 31];
      const float lv = scale.y, inv_vs = scale.z;
      // seen by some query, and its page is there
      const bool there = scale.w != 0.0f && (clean || seen_by_any(c.seq, token));
      float s[RP];
      if (ok) {
        tc_fence_after_sync();
        uint32_t raw[N];
#pragma unroll
        for (int n = 0; n < N; n += 16)
          tmem_ld_32x32(tmem + lane_base + x * N + n, *reinterpret_cast<uint32_t (*)[16]>(&raw[n]));
        tmem_ld_wait(raw);
        float w[RP];
#pragma unroll
        for (int r = 0; r < RP; ++r) {
          float v = __uint_as_float(raw[(PARTS - 1) * RP + r]);
#pragma unroll
          for (int part = PARTS - 2; part >= 0; --part)
            v = fmaf(v, 0.0625f, __uint_as_float(raw[part * RP + r]));
          s[r] = there ? fmaf(v, sh.q_factor[item & 1][r] * scale.x, lv) : -INFINITY;
        }
        if (!clean || p.rows < RP * p.row_tiles) {   // tokens that some rows do not see, rows that only pad
          const int* at = sh.q_at[item & 1];
#pragma unroll
          for (int r = 0; r < RP; ++r) {
            const bool seen = token <= at[r] && (!p.window || token > at[r] - p.window || token < p.sinks);
            if (!seen) s[r] = -INFINITY;
          }
        }
#pragma unroll
        for (int r = 0; r < RP; ++r) w[r] = warp_max(s[r]);
        if (lane == 0) {
#pragma unroll
          for (int r = 0; r < RP; r += 4)
            *reinterpret_cast<float4*>(&sh.most[x][quarter][r]) = make_float4(w[r], w[r + 1], w[r + 2], w[r + 3]);
        }
      }
      if (!all_of_group(ok)) break;
      float mt[RP];
#pragma unroll
      for (int r = 0; r < RP; r += 4) {
        float4 w = *reinterpret_cast<const float4*>(&sh.most[x][0][r]);
#pragma unroll
        for (int i = 1; i < 4; ++i) {
          const float4 o = *reinterpret_cast<const float4*>(&sh.most[x][i][r]);
          w = make_float4(fmaxf(w.x, o.x), fmaxf(w.y, o.y), fmaxf(w.z, o.z), fmaxf(w.w, o.w));
        }
        mt[r] = w.x;
        mt[r + 1] = w.y;
        mt[r + 2] = w.z;
        mt[r + 3] = w.w;
      }
      // probabilities relative to the tile's maximum (0 where the row sees nothing of it), in parts
      uint32_t bytes[PARTS][RP / 4];
      float pr[RP];
#pragma unroll
      for (int r = 0; r < RP; ++r) pr[r] = exp2_approx(s[r] - (mt[r] == -INFINITY ? 0.0f : mt[r]));
#pragma unroll
      for (int r = 0; r < RP; r += 2) {
        float a = pr[r] * kProbScale, b = pr[r + 1] * kProbScale;
#pragma unroll
        for (int part = 0; part < PARTS; ++part) {
          const uint32_t q = split2(a, b);
          if (r % 4 == 0) bytes[part][r / 4] = q; else bytes[part][r / 4] |= q << 16;
        }
      }
      // the token's row of P: N bytes, 16 at a time
#pragma unroll
      for (int n = 0; n < N; n += 16) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int at = (n + 4 * i) / RP, r = (n + 4 * i) % RP;
          w[i] = at < PARTS ? bytes[at < PARTS ? at : 0][r / 4] : 0u;
        }
        st_shared_v4(smem_u32(sh.p[x]) + (n / 16) * (kTile * 16) + me * 16, w[0], w[1], w[2], w[3]);
      }
      if (__any_sync(0xffffffffu, !there)) {
        const int g = 2 * j + 1;
        ok = mbar_wait_nocall(smem_u32(&sh.full[g % SLOTS]), (g / SLOTS) & 1, ctx, ST_KV_ZERO, j);
        ok = __all_sync(0xffffffffu, ok);
        if (!there) {
#pragma unroll
          for (int i = 0; i < D; i += 16) st_shared_v4(smem_u32(&sh.ring[g % SLOTS][me * D + i]), 0, 0, 0, 0);
        }
      }
      fence_proxy_async_smem();
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&sh.p_full[x]));

      if (stage_next) {
        const int y = (item + 1) & 1;
        queries.stage(p, next_item, me, sh.q[y], sh.q_factor[y], sh.q_at[y]);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&sh.q_full[y]));
      }

      // the tile before joins the sums while the tensor core works on this one; then they move to
      // the larger of the two references
      if (pending) add_product(j - 1);
#pragma unroll
      for (int r = 0; r < RP; ++r) {
        const float top = fmaxf(m[r], mt[r]);
        const float ref = top == -INFINITY ? 0.0f : top;
        const float old = exp2_approx(m[r] - ref), to = exp2_approx(mt[r] - ref);
        m[r] = top;
        l[r] = fmaf(pr[r] * inv_vs, to, l[r] * old);
        acc[r] *= old;
        now[r] = to * (1.0f / kProbScale);
      }
      pending = true;

      const bool last = c.last_tile();
      if (last || c.left == 1) {
        add_product(j);
        pending = false;
        // the row sums over the 128 tokens' threads
#pragma unroll
        for (int r = 0; r < RP; ++r) {
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) l[r] += __shfl_xor_sync(0xffffffffu, l[r], o);
          if (lane == 0) sh.sum[quarter][r] = l[r];
        }
        if (!all_of_group(ok)) break;
        const int row0 = c.at.row_tile * RP;
        const bool direct = whole && last;
        float* part = p.parts + (2ll * blockIdx.x + (first_part ? 0 : 1)) * RP * (D + 2);
#pragma unroll
        for (int r = 0; r < RP; ++r) {
          const float sum = (sh.sum[0][r] + sh.sum[1][r]) + (sh.sum[2][r] + sh.sum[3][r]);
          const int row = row0 + r;
          if (direct) {
            if (me < D && row < p.rows) {
              T* dst = static_cast<T*>(p.out) + c.at.b * p.o_batch_stride + row / p.group * p.o_token_stride +
                       (c.at.head * p.group + row % p.group) * p.o_head_stride + me;
              *dst = Elem<T>::from_f32(sum > 0.0f ? acc[r] / sum : acc[r] * 0.0f);   // nothing seen: 0
            }
          } else {
            if (me < D) part[r * (D + 2) + me] = acc[r];
            if (me == 0) {
              part[r * (D + 2) + D] = m[r];
              part[r * (D + 2) + D + 1] = sum;
            }
          }
          acc[r] = l[r] = 0.0f;
          m[r] = -INFINITY;
        }
        whole = true;
        first_part = false;
        if (last) ++item;
      }
      c.advance(p, 1);
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
// boundary between two shares inside it; thread i looks at boundary i + 1.
template <typename T, int D, int RP>
__global__ void __launch_bounds__(kJoinThreads) kv_join_kernel(const KvAttnParams p) {
  constexpr int kWarps = kJoinThreads / 32;
  struct Cut { Place place; int first, last, skip; };
  __shared__ Cut cuts[kMaxShares];
  __shared__ int found[kMaxShares];
  __shared__ float column[kJoinThreads / 128][128], best[kWarps], weight[kJoinThreads / 128];
  const int tid = threadIdx.x;
  const WorkList list(p);
  int count = 0;
  if (!list.whole_items()) {
    const int share = list.share_start(p, 1);          // all but the last are as long as the first
    const int flat = (int)min((tid + 1ll) * share, (long long)list.tiles() - 1);
    const Place w = list.locate(p, flat);
    const int begin = flat - w.tile;
    const bool mine = tid < p.shares - 1 && flat == (tid + 1ll) * share && w.tile > 0 && begin / share == tid;
    if (mine) {
      const int end = begin + make_seq(p, __ldg(p.lengths + w.b)).count;
      cuts[tid] = Cut{w, tid, (end - 1) / share, begin != tid * share};
    }
    // in the order of the boundaries, so that every block has the same list
    const uint32_t in_warp = __ballot_sync(0xffffffffu, mine);
    if ((tid & 31) == 0) best[tid >> 5] = (float)__popc(in_warp);
    __syncthreads();
    int index = __popc(in_warp & ((1u << (tid & 31)) - 1));
    for (int i = 0; i < kWarps; ++i) {
      if (i < (tid >> 5)) index += (int)best[i];
      count += (int)best[i];
    }
    if (mine) found[index] = tid;
    __syncthreads();
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int group = tid / 128, lane = tid % 128;
  for (int u = blockIdx.x; u < count * RP; u += gridDim.x) {
    const Cut& f = cuts[found[u / RP]];
    const int r = u % RP;
    const int row = f.place.row_tile * RP + r;
    if (row >= p.rows) continue;                   // the same in every thread
    const int n = f.last - f.first + 1;
    auto part = [&](int i) {
      return p.parts + ((2ll * (f.first + i) + (i == 0 ? f.skip : 0)) * RP + r) * (D + 2);
    };
    float m = -INFINITY;
    for (int i = tid; i < n; i += kJoinThreads) m = fmaxf(m, part(i)[D]);
    m = warp_max(m);
    if ((tid & 31) == 0) best[tid >> 5] = m;
    __syncthreads();
    for (int i = 0; i < kWarps; ++i) m = fmaxf(m, best[i]);
    float acc = 0.0f, sum = 0.0f;
    for (int i = group; i < n; i += kJoinThreads / 128) {
      const float* q = part(i);
      const float w = q[D] == -INFINITY ? 0.0f : exp2_approx(q[D] - m);
      if (lane < D) acc = fmaf(q[lane], w, acc);
      sum = fmaf(q[D + 1], w, sum);
    }
    column[group][lane] = acc;
    if (lane == 0) weight[group] = sum;
    __syncthreads();
    if (tid < D) {
      acc = sum = 0.0f;
#pragma unroll
      for (int i = 0; i < kJoinThreads / 128; ++i) {
        acc += column[i][tid];
        sum += weight[i];
      }
      T* dst = static_cast<T*>(p.out) + f.place.b * p.o_batch_stride + row / p.group * p.o_token_stride +
               (f.place.head * p.group + row % p.group) * p.o_head_stride + tid;
      *dst = Elem<T>::from_f32(sum > 0.0f ? acc / sum : acc * 0.0f);
    }
    __syncthreads();
  }
}

// ---- host ------------------------------------------------------------------------------------------

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
  static_assert(sizeof(Shared<D, RP, PARTS>) <= 113 * 1024, "two CTAs per SM");
  if (int rc = prepare_kernel((const void*)kern, smem)) return rc;
  kern<<<p.shares, kThreads, smem, stream>>>(mk, mv, p);
  if (int rc = cuda_check(cudaGetLastError(), "kv attention launch")) return rc;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3((unsigned)device_info().sm_count);
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
                                                      int64_t queries, int64_t heads, int dtype) {
  if (!cache || cache->heads <= 0 || batch <= 0 || queries <= 0 || heads <= 0) return 0;
  const int rp = row_tile_of(queries * (heads / cache->heads));
  return 2ll * shares_of() * rp * (cache->head_dim + 2) * (int64_t)sizeof(float);
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
  if (cache->pages == 0) return fail(NB200_E_INVALID, "kv attention: the cache has no pages");
  const int64_t need = nb200_kv_attention_workspace_bytes(cache, batch, queries, heads, dtype);
  if (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 15))
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
  // the work list is counted in 32 bits
  const int64_t most_tiles = cdiv64(max_pages * cache->page_size, kTile) + 1;
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
