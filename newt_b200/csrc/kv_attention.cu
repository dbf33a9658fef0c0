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
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kProbScale = 256.0f;     // probabilities of a tile are at most 1

enum : unsigned int {
  ST_KV_Q = 32, ST_KV_K, ST_KV_V, ST_KV_EMPTY, ST_KV_S, ST_KV_P, ST_KV_O, ST_KV_ZERO
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
  int pages, page, max_pages, window, sinks;
  int shares, min_share, q_aligned;
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
  s.limit = max(min(len, p.max_pages * p.page), 0);
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

// Running totals of the sequences' tiles, by stretches of sequences: thread i sums one stretch.
// Leaves the totals before each stretch in `before` [threads + 1]; everyone gets the sum.
// `warp_sum`: one number per warp.
__device__ __forceinline__ long long scan_sequences(const KvAttnParams& p, long long* before,
                                                    long long* warp_sum, int threads) {
  const int stretch = (p.batch + threads - 1) / threads;
  const int tid = threadIdx.x, lane = tid & 31;
  long long sum = 0;
  for (int i = 0; i < stretch; ++i) {
    const int b = tid * stretch + i;
    if (b < p.batch) sum += make_seq(p, p.lengths[b]).count;
  }
  long long run = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long other = __shfl_up_sync(0xffffffffu, run, o);
    if (lane >= o) run += other;
  }
  if (lane == 31) warp_sum[tid >> 5] = run;
  __syncthreads();
  for (int w = 0; w < (tid >> 5); ++w) run += warp_sum[w];
  before[tid + 1] = run;
  if (tid == 0) before[0] = 0;
  __syncthreads();
  return before[threads] * p.row_tiles * p.kv_heads;
}

// Where in the work list a tile is: sequence, item of the sequence (key head, row tile), tile.
struct Place {
  int b, item, tile;
};
__device__ __forceinline__ Place locate(const KvAttnParams& p, const long long* before, int threads,
                                        long long flat) {
  const int per_seq = p.row_tiles * p.kv_heads;
  const int stretch = (p.batch + threads - 1) / threads;
  int lo = 0, hi = threads;                        // before[lo] * per_seq <= flat < before[hi] * per_seq
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (before[mid] * per_seq <= flat) lo = mid; else hi = mid;
  }
  long long at = before[lo] * per_seq;
  int b = lo * stretch;
  int count = make_seq(p, p.lengths[b]).count;
  while (flat >= at + (long long)count * per_seq) {
    at += (long long)count * per_seq;
    ++b;
    count = make_seq(p, p.lengths[b]).count;
  }
  Place w;
  w.b = b;
  w.item = (int)((flat - at) / count);
  w.tile = (int)((flat - at) % count);
  return w;
}
__device__ __forceinline__ long long share_of(const KvAttnParams& p, long long total) {
  const long long share = (total + p.shares - 1) / p.shares;
  return share > p.min_share ? share : p.min_share;
}

// A walk over a share of the work list.
struct Cursor {
  Place at;
  Seq seq;
  long long left;      // tiles, this one among them
  __device__ void start(const KvAttnParams& p, const Place& w, long long tiles) {
    left = tiles;
    at = Place{0, 0, 0};               // an empty share has no place
    if (left <= 0) return;
    at = w;
    seq = make_seq(p, __ldg(p.lengths + at.b));
  }
  __device__ int head(const KvAttnParams& p) const { return at.item / p.row_tiles; }
  __device__ int row_tile(const KvAttnParams& p) const { return at.item % p.row_tiles; }
  __device__ bool last_tile() const { return at.tile == seq.count - 1; }
  __device__ void next(const KvAttnParams& p) {
    --left;
    if (++at.tile < seq.count) return;
    at.tile = 0;
    if (++at.item < p.row_tiles * p.kv_heads) return;
    at.item = 0;
    ++at.b;
    if (left > 0) seq = make_seq(p, __ldg(p.lengths + at.b));
  }
};

template <int D, int RP, int PARTS>
struct Shape {
  static constexpr int kN = (RP * PARTS + 15) / 16 * 16;
  static constexpr int kTileBytes = kTile * D;                    // one K or V tile
  // ring of K0 V0 K1 V1 ...: what two CTAs per SM leave room for
  static constexpr int kSlots = D == 128 ? (kN >= 48 ? 4 : 6) : (kN >= 64 ? 8 : 12);
  static constexpr int kQBytes = kN * D;
  static constexpr int kPBytes = kN * kTile;
  static constexpr int kTmemCols = 3 * kN <= 64 ? 64 : 3 * kN <= 128 ? 128 : 256;
};

template <int D, int RP, int PARTS>
struct Shared {
  using S = Shape<D, RP, PARTS>;
  uint8_t ring[S::kSlots][S::kTileBytes];      // first: the swizzle counts from 1024-byte boundaries
  uint8_t p[S::kPBytes];
  uint8_t q[2][S::kQBytes];
  float q_factor[2][RP];                       // what takes a row's product to log2 units
  int q_at[2][RP];                             // position of the row's query; -1: no such row
  float most[2][RP][4];                        // the warps' maxima, alternating by tile
  float sum[RP][4];
  uint64_t full[S::kSlots], empty[S::kSlots], q_full[2], s_full[2], p_full, o_full;
  long long before[kThreads + 1], warp_sum[kThreads / 32];
  Place start;
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
      const int r = c.row_tile(p) * RP + v / kPerRow;
      raw[i].raw = make_uint4(0, 0, 0, 0);
      if (v / kPerRow >= RP || r >= p.rows) continue;
      const T* src = static_cast<const T*>(p.q) + c.at.b * p.q_batch_stride +
                     r / p.group * p.q_token_stride +
                     (c.head(p) * p.group + r % p.group) * p.q_head_stride + v % kPerRow * 8;
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
          const int row = c.row_tile(p) * RP + r;
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
    for (int x = 0; x < 2; ++x) {
      mbar_init(smem_u32(&sh.q_full[x]), 4);   // one arrival per softmax warp
      mbar_init(smem_u32(&sh.s_full[x]), 1);
    }
    mbar_init(smem_u32(&sh.p_full), 4);
    mbar_init(smem_u32(&sh.o_full), 1);
    mbar_init_fence();
    prefetch_tensormap(&map_k);
    prefetch_tensormap(&map_v);
  }
  if (warp == 1) {
    __syncwarp();
    tmem_alloc(smem_u32(&sh.tmem_slot), S::kTmemCols);
  }
  const long long total = scan_sequences(p, sh.before, sh.warp_sum, kThreads);
  const long long share = share_of(p, total);
  const long long from = blockIdx.x * share;
  const long long tiles = min(share, max(total - from, 0ll));
  if (threadIdx.x == 0 && tiles > 0) sh.start = locate(p, sh.before, kThreads, from);
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = sh.tmem_slot;

  Cursor c;
  c.start(p, sh.start, tiles);

  if (warp == 0) {
    // ---- producer: each lane fetches one page of the tile ----
    const int per_tile = kTile / p.page;
    const uint32_t page_bytes = (uint32_t)p.page * D;
    bool ok = true;
    int g = 0;                        // tiles of K and V so far: ring position
    auto page_of = [&](const Cursor& at) {       // this lane's page of a tile, -1: not to be read
      if (at.left <= 0 || lane >= per_tile) return -1;
      const int token = tile_start(at.seq, at.at.tile) + lane * p.page;
      if (!(token < at.seq.limit && (token + p.page > at.seq.low || token < at.seq.sink_end))) return -1;
      const int id = __ldg(p.table + at.at.b * p.table_stride + token / p.page);
      return id >= 0 && id < p.pages ? id : -1;
    };
    int id = page_of(c);
    while (c.left > 0 && ok) {
      const int head = c.head(p);
      c.next(p);
      const int ahead = page_of(c);   // the next tile's, under way while this one is issued
      const uint32_t bytes = __popc(__ballot_sync(0xffffffffu, id >= 0)) * page_bytes;
#pragma unroll
      for (int kv = 0; kv < 2; ++kv, ++g) {
        const int x = g % SLOTS;
        ok = ok && mbar_wait_nocall(smem_u32(&sh.empty[x]), ((g / SLOTS) & 1) ^ 1, ctx, ST_KV_EMPTY, g);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        const uint32_t bar = smem_u32(&sh.full[x]);
        if (lane == 0) {
          if (bytes) mbar_arrive_expect_tx(bar, bytes); else mbar_arrive(bar);
        }
        __syncwarp();
        if (id >= 0) tma_load_4d(smem_u32(&sh.ring[x][lane * page_bytes]), kv ? &map_v : &map_k, 0, 0, head, id, bar);
      }
      id = ahead;
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
      c.next(p);
      if (c.left > 0) {
        if (ends) ++item;
        begin(j + 1, ends);
      }
      const int x = (2 * j + 1) % SLOTS;
      ok = ok && wait_all(&sh.full[x], ((2 * j + 1) / SLOTS) & 1, ST_KV_V, j);
      ok = ok && wait_all(&sh.p_full, j & 1, ST_KV_P, j);
      if (!ok) break;
      tc_fence_after_sync();
      const uint32_t vb = smem_u32(sh.ring[x]), pb = smem_u32(sh.p);
#pragma unroll
      for (int kk = 0; kk < kTile / 32; ++kk)      // 32 tokens: four groups of eight rows
        if (elected)
          mma_f8_ss(tmem + 2 * N, with_address(kVDesc, vb + kk * 32 * D),
                    with_address(kPDesc, pb + kk * 4 * 128), kIdescPv, kk != 0);
      if (elected) {
        mma_commit(smem_u32(&sh.o_full));
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
    if (c.left > 0) queries.load(p, c, me);
    // the scales of a token's page: two steps ahead the page, one step ahead its scales
    auto page_id = [&](const Cursor& at) {
      if (at.left <= 0) return -1;
      const int token = tile_start(at.seq, at.at.tile) + me;
      if (!seen_by_any(at.seq, token)) return -1;
      const int id = __ldg(p.table + at.at.b * p.table_stride + token / p.page);
      return id >= 0 && id < p.pages ? id : -1;
    };
    float ks = 0.0f, vs = 1.0f;
    auto fetch_scales = [&](int id, int head, float& k_scale, float& v_scale) {
      k_scale = id >= 0 ? __ldg(p.k_scales + id * p.k_scale_stride + head) : 0.0f;
      v_scale = id >= 0 ? __ldg(p.v_scales + id * p.v_scale_stride + head) : 1.0f;
    };
    Cursor ahead = c;
    int id = page_id(c);
    int ahead_id = -1, ahead_head = 0;
    if (c.left > 0) {
      ahead.next(p);
      ahead_id = page_id(ahead);
      if (ahead.left > 0) ahead_head = ahead.head(p);
      queries.stage(p, c, me, sh.q[0], sh.q_factor[0], sh.q_at[0]);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&sh.q_full[0]));
      all_of_group(true);            // the rows' factors and positions are written
    }
    fetch_scales(id, c.left > 0 ? c.head(p) : 0, ks, vs);

    int item = 0;
    bool whole = c.left > 0 && c.at.tile == 0;     // has the item's first tile
    bool first_part = true;                        // the item that the share begins with
    float acc[RP], l[RP], m[RP];                   // m: log2 units
#pragma unroll
    for (int r = 0; r < RP; ++r) {
      acc[r] = l[r] = 0.0f;
      m[r] = -INFINITY;
    }
    for (int j = 0; c.left > 0; ++j) {
      // what the next tile needs, on its way
      const int next_id = ahead_id, next_head = ahead_head;
      float next_ks, next_vs;
      fetch_scales(next_id, next_head, next_ks, next_vs);
      if (ahead.left > 0) {
        ahead.next(p);
        ahead_id = page_id(ahead);
        if (ahead.left > 0) ahead_head = ahead.head(p);
      }
      // the next item's queries, too: loaded at the start of an item, staged behind its first tile
      const bool item_begins = j == 0 || c.at.tile == 0;
      Cursor next_item = c;
      bool stage_next = false;
      if (item_begins) {
        const int skip = c.seq.count - c.at.tile;  // tiles to the next item
        if (c.left > skip) {
          next_item.at.tile = c.seq.count - 1;
          next_item.left = c.left - skip + 1;
          next_item.next(p);
          stage_next = true;
          queries.load(p, next_item, me);
        }
      }

      const int x = j & 1;
      const int t0 = tile_start(c.seq, c.at.tile);
      const int token = t0 + me;
      const bool there = id >= 0;                  // seen by some query, and its page is there
      // every query sees the whole tile: no masks but `there`
      const int first_at = c.seq.len - p.nq;
      const bool clean = t0 + kTile - 1 <= first_at &&
                         (!p.window || t0 > c.seq.len - 1 - p.window || t0 + kTile <= p.sinks);
      float s[RP];
      ok = ok && mbar_wait_nocall(smem_u32(&sh.s_full[x]), (j >> 1) & 1, ctx, ST_KV_S, j);
      ok = __all_sync(0xffffffffu, ok);
      const float lv = log2f(vs);
      if (ok) {
        tc_fence_after_sync();
        uint32_t raw[N];
#pragma unroll
        for (int n = 0; n < N; n += 16)
          tmem_ld_32x32(tmem + lane_base + x * N + n, *reinterpret_cast<uint32_t (*)[16]>(&raw[n]));
        tmem_ld_wait(raw);
        const float* factor = sh.q_factor[item & 1];
#pragma unroll
        for (int r = 0; r < RP; ++r) {
          float v = __uint_as_float(raw[(PARTS - 1) * RP + r]);
#pragma unroll
          for (int part = PARTS - 2; part >= 0; --part)
            v = fmaf(v, 0.0625f, __uint_as_float(raw[part * RP + r]));
          s[r] = there ? v * (factor[r] * ks) : -INFINITY;
        }
        if (!clean) {
          const int* at = sh.q_at[item & 1];
#pragma unroll
          for (int r = 0; r < RP; ++r) {
            const bool seen = token <= at[r] && (!p.window || token > at[r] - p.window || token < p.sinks);
            if (!seen) s[r] = -INFINITY;
          }
        } else if (p.rows < RP * p.row_tiles) {    // rows that only pad
#pragma unroll
          for (int r = 0; r < RP; ++r)
            if (sh.q_at[item & 1][r] < 0) s[r] = -INFINITY;
        }
#pragma unroll
        for (int r = 0; r < RP; ++r) {
          const float w = warp_max(s[r] + lv);
          if (lane == 0) sh.most[x][r][quarter] = w;
        }
      }
      if (!all_of_group(ok)) break;
      float mt[RP];
      uint32_t bytes[PARTS][RP / 4];
      const float inv_vs = 1.0f / vs;
#pragma unroll
      for (int r = 0; r < RP; ++r) {
        const float4 w = *reinterpret_cast<const float4*>(sh.most[x][r]);
        mt[r] = fmaxf(fmaxf(w.x, w.y), fmaxf(w.z, w.w));
      }
#pragma unroll
      for (int r = 0; r < RP; r += 2) {
        float pr[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float ref = mt[r + h] == -INFINITY ? 0.0f : mt[r + h];
          pr[h] = exp2_approx(s[r + h] + lv - ref);
          // the running sums move to the larger of the two references
          const float top = fmaxf(m[r + h], ref);
          const float old = m[r + h] == -INFINITY ? 0.0f : exp2_approx(m[r + h] - top);
          const float now = mt[r + h] == -INFINITY ? 0.0f : exp2_approx(ref - top);
          if (mt[r + h] != -INFINITY) m[r + h] = top;
          l[r + h] = mt[r + h] == -INFINITY ? l[r + h] : fmaf(pr[h] * inv_vs, now, l[r + h] * old);
          acc[r + h] = mt[r + h] == -INFINITY ? acc[r + h] : acc[r + h] * old;
          mt[r + h] = now * (1.0f / kProbScale);   // from here on: the tile's factor
          pr[h] *= kProbScale;
        }
#pragma unroll
        for (int part = 0; part < PARTS; ++part) {
          const uint32_t q = split2(pr[0], pr[1]);
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
        st_shared_v4(smem_u32(sh.p) + (n / 16) * (kTile * 16) + me * 16, w[0], w[1], w[2], w[3]);
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
      if (lane == 0) mbar_arrive(smem_u32(&sh.p_full));

      if (stage_next) {
        queries.stage(p, next_item, me, sh.q[(item + 1) & 1], sh.q_factor[(item + 1) & 1], sh.q_at[(item + 1) & 1]);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&sh.q_full[(item + 1) & 1]));
      }

      ok = ok && mbar_wait_nocall(smem_u32(&sh.o_full), j & 1, ctx, ST_KV_O, j);
      ok = __all_sync(0xffffffffu, ok);
      if (ok) {
        tc_fence_after_sync();
        uint32_t raw[N];
#pragma unroll
        for (int n = 0; n < N; n += 16)
          tmem_ld_32x32(tmem + lane_base + 2 * N + n, *reinterpret_cast<uint32_t (*)[16]>(&raw[n]));
        tmem_ld_wait(raw);
#pragma unroll
        for (int r = 0; r < RP; ++r) {
          float v = __uint_as_float(raw[(PARTS - 1) * RP + r]);
#pragma unroll
          for (int part = PARTS - 2; part >= 0; --part)
            v = fmaf(v, 0.0625f, __uint_as_float(raw[part * RP + r]));
          acc[r] = fmaf(v, mt[r], acc[r]);
        }
      }

      const bool last = c.last_tile();
      if (last || c.left == 1) {
        // the row sums over the 128 tokens' threads
#pragma unroll
        for (int r = 0; r < RP; ++r) {
          float v = l[r];
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
          if (lane == 0) sh.sum[r][quarter] = v;
        }
        if (!all_of_group(ok)) break;
        const int row0 = c.row_tile(p) * RP;
        const bool direct = whole && last;
        float* part = p.parts + (2ll * blockIdx.x + (first_part ? 0 : 1)) * RP * (D + 2);
#pragma unroll
        for (int r = 0; r < RP; ++r) {
          const float4 w = *reinterpret_cast<const float4*>(sh.sum[r]);
          const float sum = (w.x + w.y) + (w.z + w.w);
          const int row = row0 + r;
          if (direct) {
            if (me < D && row < p.rows) {
              T* dst = static_cast<T*>(p.out) + c.at.b * p.o_batch_stride + row / p.group * p.o_token_stride +
                       (c.head(p) * p.group + row % p.group) * p.o_head_stride + me;
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
      c.next(p);
      id = next_id;
      ks = next_ks;
      vs = next_vs;
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
  __shared__ long long before[kJoinThreads + 1], warp_sum[kJoinThreads / 32];
  __shared__ struct { Place place; int first, last, skip; } found[kJoinThreads];
  __shared__ int warp_found[kJoinThreads / 32];
  __shared__ float column[kJoinThreads / 128][128], best[kJoinThreads / 32], weight[kJoinThreads / 128];
  const int tid = threadIdx.x;
  const long long total = scan_sequences(p, before, warp_sum, kJoinThreads);
  const long long share = share_of(p, total);
  const long long flat = (tid + 1) * share;
  bool mine = false;
  Place w;
  long long begin = 0, end = 0;
  if (tid + 1 < p.shares && flat < total) {
    w = locate(p, before, kJoinThreads, flat);
    begin = flat - w.tile;
    end = begin + make_seq(p, p.lengths[w.b]).count;
    mine = w.tile > 0 && begin / share == tid;
  }
  // every block lists the items in the same order, so that they divide the work
  const uint32_t in_warp = __ballot_sync(0xffffffffu, mine);
  if ((tid & 31) == 0) warp_found[tid >> 5] = __popc(in_warp);
  __syncthreads();
  int index = __popc(in_warp & ((1u << (tid & 31)) - 1)), count = 0;
  for (int i = 0; i < kJoinThreads / 32; ++i) {
    if (i < (tid >> 5)) index += warp_found[i];
    count += warp_found[i];
  }
  if (mine) {
    found[index].place = w;
    found[index].first = (int)(begin / share);
    found[index].last = (int)((end - 1) / share);
    found[index].skip = begin != found[index].first * share;   // the item is its first share's second part
  }
  __syncthreads();
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int group = tid / 128, lane = tid % 128;
  for (int u = blockIdx.x; u < count * RP; u += gridDim.x) {
    const auto& f = found[u / RP];
    const int r = u % RP;
    const int row = (f.place.item % p.row_tiles) * RP + r;
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
    for (int i = 0; i < kJoinThreads / 32; ++i) m = fmaxf(m, best[i]);
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
               (f.place.item / p.row_tiles * p.group + row % p.group) * p.o_head_stride + tid;
      *dst = Elem<T>::from_f32(sum > 0.0f ? acc / sum : acc * 0.0f);
    }
    __syncthreads();
  }
}

// ---- host ------------------------------------------------------------------------------------------

constexpr int kMaxShares = kJoinThreads;

int row_tile_of(int64_t rows, bool bf16) {
  const int most = bf16 ? 32 : 16;       // more columns than 64 would need more tensor memory than half an SM's
  int rp = 8;
  while (rp < rows && rp < most) rp *= 2;
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
    if (rp == 8) return launch_kv<__nv_bfloat16, D, 8, 2>(p, mk, mv, stream);
    if (rp == 16) return launch_kv<__nv_bfloat16, D, 16, 2>(p, mk, mv, stream);
    return launch_kv<__nv_bfloat16, D, 32, 2>(p, mk, mv, stream);
  }
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
  const int rp = row_tile_of(queries * (heads / cache->heads), dtype == NB200_BF16);
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
  const int rp = row_tile_of(p.rows, bf16);
  p.row_tiles = (p.rows + rp - 1) / rp;
  if ((int64_t)p.row_tiles * p.kv_heads > INT32_MAX) return fail(NB200_E_INVALID, "kv attention: too many rows");
  p.pages = (int)cache->pages;
  p.page = (int)cache->page_size;
  p.max_pages = (int)max_pages;
  p.window = (int)window;
  p.sinks = (int)sinks;
  p.shares = shares_of();
  p.min_share = 2;
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
