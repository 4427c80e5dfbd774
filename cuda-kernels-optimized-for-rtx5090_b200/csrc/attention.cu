// Attention of a few new tokens per sequence over a paged key/value cache, with a prefix that the whole batch shares.
//
// For query row (b, t, head h of its kv head's group), the positions j < L = lens[b] - T + t + 1, x_j = scale q.k_j:
//   out = sum_j exp(x_j - m) v_j / sum_j exp(x_j - m),  m = max_j x_j
// computed piece by piece: a piece of positions gives (m, l = sum exp(x - m), o = sum exp(x - m) v), and pieces join by
//   M = max m_i,  out = sum_i exp(m_i - M) o_i / sum_i exp(m_i - M) l_i.
// x, m, l and o are fp32; the weights exp(x - m) are rounded to the cache's dtype for the product with v (half a step of
// that dtype on each, as the output's own rounding), q, k and v enter the products as they are. fp16 has no half step of a
// small value: below 2^-14 its steps stay 2^-24, and a weight below 2^-25 would be lost, of which a long context has many.
// So its weights are exp(x - m) 2^15 (weights_from); any m will do for a piece, as long as l, o and the join take the same.
//
// Two kinds of work:
//   own     the positions behind the prefix: a unit is (sequence, kv head, up to 64 of its T * group rows), its tiles are 64
//           of the sequence's own positions. Bound by the bytes of the cache: every key and value is read once, by one CTA
//           (attend_stream; attend_tiles for block sizes that a TMA box does not fit, 0.6 of its rate: 48 ragged sequences
//           422 us in pages of 24, 254 us in pages of 16);
//   shared  the prefix's positions: a unit is (kv head, rows of ALL sequences), so each key and value of the prefix is
//           read once for many rows, not once for every sequence (attend_prefix on tcgen05; attend_tiles for heads of
//           more than 128 columns and those block sizes: 64 behind 4096 tokens 42 us, 83 us with 256 columns and half the heads,
//           105 us in pages of 24). Sequences that end before the prefix does take no part: all their
//           positions are own ones.
// The tiles of all units are laid end to end and cut into runs, one for each CTA (the own lengths are only known on the
// device: every CTA adds them up itself). So unequal lengths and few sequences fill the GPU alike. A run's part of a unit is
// a piece; pieces go to the workspace at slot (unit + CTA), which is different for each, and join_rows joins them. A whole
// unit of a sequence that shares no prefix is written out at once.
#include "ckb200_attention.h"
#include "common.cuh"

#include <algorithm>
#include <climits>
#include <type_traits>

namespace ckb {
namespace {

constexpr int kTile = 64;      // positions of a tile
constexpr int kThreads = 128;  // four warps
constexpr int kMaxShared = 232448;  // bytes of shared memory that a CTA can have
constexpr int kSmShared = 233472;   // and an SM has
// The shared work takes at most 7 of 8 SMs, so that own tokens are read from its first moment on (256 sequences behind 16384
// tokens 128 us, with 6 of 8 SMs 131 us, with all 135 us), and runs of at least 4 tiles, as a CTA spends 5 us before its
// first tile and 3 us on its piece (64 sequences behind 4096 tokens with up to 1023, up to 32 own tokens: 42 and 21 us; runs of 3
// tiles 45 and 25 us, of 8 tiles 41 and 27 us). Where units are shorter than that and many, a run has several of them: 256
// sequences of 5 tokens with 20 rows a key head behind 128 tokens took 138 us with a CTA for each of the 160 units, 126 us with two
// units a CTA; 512 of 4 tokens with 256 units 154 us and 159 us.
constexpr int kPrefixShare = 7;
constexpr int kPrefixRun = 4;
// What the shared work's CTAs are expected to take: 9 us and 1.9 us a tile (half where its groups share the tiles). The own
// work's CTAs that start beside them get so many more tiles, of 2 us, than those that come after (64 behind 4096: 42 us, without
// 50 us; tiles of 1.5 or 2.6 us 44 us). All of these were set at 128 columns with up to 16 rows a key head and are used for every
// other shape as they are: they only balance the load, no result depends on them (64 behind 4096 at 64 columns 31 us).
constexpr int kPrefixCtaNs = 9000, kPrefixTileNs = 1900, kOwnTileNs = 2000;
constexpr int kMaxBatch = 4096;  // lengths and tile counts of all sequences stay in shared memory
constexpr float kLog2e = 1.4426950408889634f;
// The power of 2 by which fp16 weights are lifted: at most 2^15 then, and half a step of the smallest is 2^-40 of the largest.
constexpr float kLift = 15.0f;

struct View3 {
  long long batch, token, head;
};

struct Args {
  const void *q, *key, *value;
  const long long *tables, *lens;
  void* out;
  float* part;     // [slots][rows of a tile][D] of this launch's pieces
  float2* ml;      // [slots][rows of a tile]: (m in powers of 2, l)
  int* plan;       // own work only: [batch + 1] running tile counts, then the runs
  View3 vq;
  long long num_blocks;
  int batch, tokens, q_heads, kv_heads, group, head_dim, block_size, table_width;
  int block_log;   // log2 of block_size, or -1
  int prefix;      // positions of the shared prefix
  int rows;        // tokens * group: query rows of a sequence and kv head
  int row_tiles;   // row tiles of a unit's rows
  float scale_log2;
  bool beside;     // own work launched beside the shared work: see start_all
  // CTAs of the own work that start with the shared work, tiles that they are expected to do before the others start.
  int early, ahead;
};

// ---------------------------------------------------------------------------------------------------------------
// Tensor-core fragments (m16n8k16) and asynchronous copies.
// ---------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ void ldsm4(unsigned (&r)[4], unsigned at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at));
}
__device__ __forceinline__ void ldsm4_trans(unsigned (&r)[4], unsigned at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at));
}
__device__ __forceinline__ void mma(float (&c)[4], const unsigned (&a)[4], unsigned b0, unsigned b1, __nv_bfloat16) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
               "{%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma(float (&c)[4], const unsigned (&a)[4], unsigned b0, unsigned b1, __half) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
               "{%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ unsigned pack2(float lo, float hi, __nv_bfloat16) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const unsigned*>(&v);
}
__device__ __forceinline__ unsigned pack2(float lo, float hi, __half) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const unsigned*>(&v);
}
// 16 bytes global -> shared; without `fill` the bytes are zeros and nothing is read.
__device__ __forceinline__ void copy16(unsigned dst, const void* src, bool fill) {
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(fill ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// What is taken off a row's scores (in powers of 2) whose maximum is m, -inf where it has seen nothing: m, and for fp16
// weights `lift` less. Beyond 2^20, where the rounding of m itself would show in the weights, they are not lifted.
template <typename T>
__device__ __forceinline__ float weights_from(float m, float lift) {
  return std::is_same<T, __half>::value && fabsf(m) < 0x1p20f ? m - lift : m;
}

// Byte offset of 16-byte chunk c of row r in a tile of rows of DT 16-bit values: chunks are exchanged within a row so that
// the 8 rows an ldmatrix reads lie in different banks.
template <int DT>
__device__ __forceinline__ unsigned at_chunk(int r, int c) {
  return r * (DT * 2) + ((c ^ (r & 7)) << 4);
}

// Two neighbouring values of shared memory.
__device__ __forceinline__ unsigned load_word(unsigned at) {
  unsigned w;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w) : "r"(at));
  return w;
}
__device__ __forceinline__ float2 load2(unsigned at, __nv_bfloat16) {
  const unsigned w = load_word(at);
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
__device__ __forceinline__ float2 load2(unsigned at, __half) {
  const unsigned w = load_word(at);
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
// Whether any value of rows row0 .. row0 + kCount - 1 of a tile is infinite or NaN (the whole warp asks).
template <typename T, int DT, int kCount>
__device__ __forceinline__ bool not_finite(unsigned tile, int row0, int lane) {
  bool bad = false;
#pragma unroll 4
  for (int i = lane; i < kCount * (DT / 2); i += 32) {
    const float2 v = load2(tile + row0 * (DT * 2) + i * 4, T{});
    bad |= !(fabsf(v.x) < INFINITY) || !(fabsf(v.y) < INFINITY);
  }
  return __any_sync(0xffffffffu, bad);
}

// The rows of a unit: row r of the tile is query (b, t, head), or nothing.
struct Row {
  int b, t, head;  // head: of the q heads
  bool real;
};
template <bool kShared>
__device__ __forceinline__ Row row_of(const Args& a, int b, int kv_head, int r) {
  Row x;
  x.real = r < (kShared ? a.batch * a.rows : a.rows);
  x.b = kShared ? r / a.rows : b;
  const int in = kShared ? r - x.b * a.rows : r;
  x.t = in / a.group;
  x.head = kv_head * a.group + (in - x.t * a.group);
  return x;
}
// The lengths and tables. The own work beside a prefix starts without a wait of its own (start_all): what came before on the
// stream has ended, as the shared work's CTAs waited for it before they let it start, but only a grid's own wait is said to
// make it visible to that grid. So all its inputs are read in L2, past an SM's L1, where an older copy could lie: these two
// lists here, the queries by cp.async.cg, the cache by TMA or cp.async.cg.
__device__ __forceinline__ long long load_list(const long long* p) { return __ldcg(p); }
__device__ __forceinline__ long long length_of(const Args& a, int b) {
  const long long most = (long long)a.table_width * a.block_size, n = load_list(a.lens + b);
  return n < 0 ? 0 : n < most ? n : most;
}
// Where a sequence's own positions begin: behind the prefix, or, for one that does not see all of it, at 0: such a sequence
// (shorter than the prefix, or none) takes no part in the shared work, whose rows all see every position.
__device__ __forceinline__ int own_begin(int prefix, int tokens, int len) {
  return len - tokens + 1 >= prefix ? prefix : 0;
}
// The first sequence that sees all of the prefix (0 where none does): its table names the shared blocks, as those of padded
// rows and of shorter sequences may hold anything there. The whole warp asks.
__device__ __forceinline__ int first_sharing(const Args& a) {
  for (int base = 0; base < a.batch; base += 32) {
    const int b = base + (threadIdx.x & 31);
    const bool sees = b < a.batch && own_begin(a.prefix, a.tokens, (int)length_of(a, b)) > 0;
    const unsigned some = __ballot_sync(0xffffffffu, sees);
    if (some != 0u) return base + __ffs(some) - 1;
  }
  return 0;
}

// A place on the axis of tiles.
struct Cursor {
  int b, unit, tile, tiles;  // sequence (0 in shared work), unit within it, tile within the unit, the unit's tiles
};

// The own work's axis: cum[b] tiles lie before sequence b, cum[batch] in all; lens[b] the clamped lengths. The whole block of
// kCount threads takes part; `scratch` holds kCount / 32 ints.
template <int kCount>
__device__ __forceinline__ void own_axis(const Args& a, int units, int* cum, int* lens, int* scratch) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  int before = 0;
  for (int base = 0; base < a.batch; base += kCount) {
    const int b = base + tid;
    int mine = 0;
    if (b < a.batch) {
      const int len = (int)length_of(a, b);
      lens[b] = len;
      mine = (len - own_begin(a.prefix, a.tokens, len) + kTile - 1) / kTile * units;
    }
    int upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    if (lane == 31) scratch[warp] = upto;
    __syncthreads();
    for (int k = 0; k < warp; ++k) upto += scratch[k];
    if (b < a.batch) cum[b] = before + upto - mine;
    for (int k = 0; k < kCount / 32; ++k) before += scratch[k];
    __syncthreads();
  }
  if (tid == 0) cum[a.batch] = before;
  __syncthreads();
}
// How the axis of `all` tiles is cut for `ctas` CTAs: the first `early` have runs of `longer` tiles, the others of `run`.
struct Runs {
  int early, longer, run;
  __device__ __forceinline__ int begin(int cta, int all) const {
    const long long w = cta < early ? (long long)cta * longer : (long long)early * longer + (long long)(cta - early) * run;
    return (int)min(w, (long long)all);
  }
  __device__ __forceinline__ int cta_of(int w) const {
    return w < early * longer ? w / longer : early + (w - early * longer) / run;
  }
};
__device__ __forceinline__ Runs runs_of(const Args& a, int all, int ctas) {
  Runs r;
  r.early = a.early;
  const int rest = all - (int)min((long long)a.early * a.ahead, (long long)all);
  if (rest > 0 || a.early == 0) {
    r.run = max(1, (rest + ctas - 1) / ctas);
    r.longer = r.run + a.ahead;
  } else {  // the early ones do it all
    r.run = 1;
    r.longer = max(1, (all + a.early - 1) / a.early);
  }
  return r;
}
// Tile w of the axis of `seqs` sequences (w < cum[seqs]).
__device__ __forceinline__ Cursor axis_start(const int* cum, int seqs, int units, int w) {
  int lo = 0, hi = seqs;  // the last b with cum[b] <= w
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cum[mid] <= w) lo = mid;
    else hi = mid;
  }
  Cursor c;
  c.b = lo;
  c.tiles = (cum[lo + 1] - cum[lo]) / units;
  c.unit = (w - cum[lo]) / c.tiles;
  c.tile = w - cum[lo] - c.unit * c.tiles;
  return c;
}
// The next tile. Past the axis' end the cursor names no tile (callers stop there).
__device__ __forceinline__ void axis_next(const int* cum, int seqs, int units, Cursor& c) {
  if (++c.tile < c.tiles) return;
  c.tile = 0;
  if (++c.unit < units) return;
  c.unit = 0;
  do {
    ++c.b;
    c.tiles = c.b < seqs ? (cum[c.b + 1] - cum[c.b]) / units : 1;
  } while (c.b < seqs && c.tiles == 0);
}

// What the join needs to know of the own work's cuts.
template <int kCount>
__device__ __forceinline__ void write_plan(const Args& a, const int* cum, const Runs& r) {
  for (int b = threadIdx.x; b <= a.batch; b += kCount) a.plan[b] = cum[b];
  if (threadIdx.x == 0) {
    a.plan[a.batch + 1] = r.early;
    a.plan[a.batch + 2] = r.longer;
    a.plan[a.batch + 3] = r.run;
  }
}

// Writes a lane's part of row half i of an accumulator o: the output itself where the piece is the whole unit, else the
// piece at workspace row `at`.
template <typename T, int DT>
__device__ __forceinline__ void write_row(const Args& a, const Row& x, bool whole, bool some, long long at, int lane,
                                          const float (&o)[DT / 8][4], int i, float m, float l) {
  if (!x.real) return;
  if (whole) {
    const float inv = 1.0f / l;
    T* dst = (T*)a.out + (((long long)x.b * a.tokens + x.t) * a.q_heads + x.head) * a.head_dim;
#pragma unroll
    for (int n = 0; n < DT / 8; ++n) {
      const int c = n * 8 + (lane & 3) * 2;
      if (c < a.head_dim)
        *reinterpret_cast<unsigned*>(dst + c) = some ? pack2(o[n][2 * i] * inv, o[n][2 * i + 1] * inv, T{}) : 0u;
    }
  } else {
    float* dst = a.part + at * a.head_dim;
#pragma unroll
    for (int n = 0; n < DT / 8; ++n) {
      const int c = n * 8 + (lane & 3) * 2;
      if (c < a.head_dim) *reinterpret_cast<float2*>(dst + c) = make_float2(o[n][2 * i], o[n][2 * i + 1]);
    }
    if ((lane & 3) == 0) a.ml[at] = make_float2(m, l);
  }
}

template <typename T, int DT, int WR, bool kShared>
struct Shape {
  static constexpr int kRows = 16 * WR;        // query rows of a tile
  static constexpr int kKeyWarps = 4 / WR;     // warps that share a tile's positions
  static constexpr int kKeys = kTile / kKeyWarps;
  static constexpr int kStages = WR == 1 && DT <= 128 ? 3 : 2;  // what leaves room for per_sm() CTAs
  static constexpr int kTileBytes = kTile * DT * 2;
  static constexpr int kQBytes = kRows * DT * 2;
  static constexpr int kOffQ = kStages * 2 * kTileBytes;
  static constexpr int kOffRows = kOffQ + kStages * kQBytes;  // units may be one tile long: a q buffer for each stage
  static constexpr int kOffMl = kOffRows + 2 * kTile * 8;
  static constexpr int kOffLimits = kOffMl + kKeyWarps * kRows * 8;
  static constexpr int kOffCum = kOffLimits + kRows * 4;
  static int bytes(int batch) { return kOffCum + (kShared ? 2 : 2 * batch + 1) * 4; }
};

template <typename T, int DT, int WR, bool kShared>
__global__ void __launch_bounds__(kThreads) attend_tiles(const Args a) {
  using S = Shape<T, DT, WR, kShared>;
  constexpr int kRows = S::kRows, kKeys = S::kKeys, kStages = S::kStages;
  constexpr int kChunks = DT / 8;                // 16-byte chunks of a row
  constexpr int kRowsPerPass = kThreads / kChunks;
  extern __shared__ __align__(128) unsigned char smem[];
  long long* row_at = reinterpret_cast<long long*>(smem + S::kOffRows);  // [2][kTile] cache rows, -1: zeros
  float2* ml_sh = reinterpret_cast<float2*>(smem + S::kOffMl);           // [key warps][rows]
  int* limits = reinterpret_cast<int*>(smem + S::kOffLimits);
  int* cum = reinterpret_cast<int*>(smem + S::kOffCum);
  const unsigned smem_at = smem_u32(smem);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int wr = warp % WR, wk = warp / WR;
  if (kShared || !a.beside) pdl_wait();
  pdl_trigger();

  // The axis of tiles.
  const int units = a.kv_heads * a.row_tiles;  // of a sequence
  const int seqs = kShared ? 1 : a.batch;
  if (kShared) {
    if (tid == 0) {
      cum[0] = 0;
      cum[1] = units * ((a.prefix + kTile - 1) / kTile);
    }
  } else {
    own_axis<kThreads>(a, units, cum, cum + a.batch + 1, reinterpret_cast<int*>(ml_sh));
  }
  __syncthreads();
  const int all = cum[seqs];
  // The join knows the shared work's runs from the host, which cuts them the same way.
  const Runs runs = kShared ? Runs{0, 1, (all + (int)gridDim.x - 1) / (int)gridDim.x} : runs_of(a, all, gridDim.x);
  if (!kShared && blockIdx.x == 0) write_plan<kThreads>(a, cum, runs);
  const int first = runs.begin(blockIdx.x, all), last = runs.begin(blockIdx.x + 1, all);
  if (!kShared && a.beside && blockIdx.x == 0 && first >= last) pdl_wait();
  if (first >= last) return;

  const long long* shared_table = kShared ? a.tables + (long long)first_sharing(a) * a.table_width : nullptr;
  // The cache row of position (tile, lane of the tile), or -1.
  const auto lookup = [&](const Cursor& c, int i) -> long long {
    const int end = kShared ? a.prefix : cum[a.batch + 1 + c.b];
    const int pos = (kShared ? 0 : own_begin(a.prefix, a.tokens, end)) + c.tile * kTile + i;
    if (pos >= end) return -1;
    const int page = pos / a.block_size;
    const long long block = load_list((kShared ? shared_table : a.tables + (long long)c.b * a.table_width) + page);
    if (block < 0 || block >= a.num_blocks) return -1;
    return block * a.block_size + (pos - page * a.block_size);
  };
  const auto issue = [&](const Cursor& c, int stage, int slot, int q_buffer, bool with_q) {
    const int kv_head = c.unit / a.row_tiles, chunk = tid % kChunks;
    const bool inside = chunk * 8 < a.head_dim;
    const unsigned k_at = smem_at + stage * 2 * S::kTileBytes, v_at = k_at + S::kTileBytes;
#pragma unroll
    for (int p = 0; p < kTile / kRowsPerPass; ++p) {
      const int r = p * kRowsPerPass + tid / kChunks;
      const long long row = row_at[slot * kTile + r];
      const bool fill = inside && row >= 0;
      const long long off = fill ? (row * a.kv_heads + kv_head) * a.head_dim + chunk * 8 : 0;
      copy16(k_at + at_chunk<DT>(r, chunk), (const T*)a.key + off, fill);
      copy16(v_at + at_chunk<DT>(r, chunk), (const T*)a.value + off, fill);
    }
    if (with_q) {
      const int row0 = (c.unit - kv_head * a.row_tiles) * kRows;
      for (int r = tid / kChunks; r < kRows; r += kRowsPerPass) {
        const Row x = row_of<kShared>(a, c.b, kv_head, row0 + r);
        const bool fill = inside && x.real;
        const long long off = fill ? x.b * a.vq.batch + x.t * a.vq.token + x.head * a.vq.head + chunk * 8 : 0;
        copy16(smem_at + S::kOffQ + q_buffer * S::kQBytes + at_chunk<DT>(r, chunk), (const T*)a.q + off, fill);
      }
    }
  };

  // Three cursors run along the axis: page look-ups kStages tiles ahead, copies kStages - 1 ahead, the products.
  Cursor look = axis_start(cum, seqs, units, first), load = look, at = look;
  int looked = first, loaded = first, q_loads = 0;
  const auto look_and_store = [&]() {
    if (looked >= last) return;
    if (tid < kTile) row_at[(looked & 1) * kTile + tid] = lookup(look, tid);
    axis_next(cum, seqs, units, look);
    ++looked;
  };
  const auto load_one = [&]() {
    if (loaded < last) {
      const bool with_q = loaded == first || load.tile == 0;
      if (with_q) ++q_loads;
      issue(load, (loaded - first) % kStages, loaded & 1, q_loads % kStages, with_q);
      axis_next(cum, seqs, units, load);
      ++loaded;
    }
    copy_commit();
  };
  look_and_store();
  for (int i = 0; i < kStages - 1; ++i) {
    __syncthreads();
    load_one();
    look_and_store();
  }

  constexpr int kNt = kKeys / 8;   // score tiles of 8 positions
  constexpr int kDt = DT / 8;      // output tiles of 8 columns
  float o[kDt][4], m[2], l[2];
  int min_limit = 0, lim[2] = {0, 0}, q_now = 0, piece_begin = 0, begin = 0;
  const int quad_row = lane >> 2;
  for (int w = first; w < last; ++w) {
    copy_wait<kStages - 2>();
    __syncthreads();  // tile w is there for all, tile w - 1's stage is free
    load_one();
    long long next_row = -1;
    const bool looking = looked < last;
    if (looking && tid < kTile) next_row = lookup(look, tid);

    const int kv_head = at.unit / a.row_tiles, row0 = (at.unit - kv_head * a.row_tiles) * kRows;
    if (w == first || at.tile == 0) {  // a new piece
      ++q_now;
      piece_begin = at.tile;
      begin = kShared ? 0 : own_begin(a.prefix, a.tokens, cum[a.batch + 1 + at.b]);
      if (tid < kRows) {
        const Row x = row_of<kShared>(a, at.b, kv_head, row0 + tid);
        // A row of padding: any finite result.
        limits[tid] = kShared ? a.prefix : x.real ? max(0, cum[a.batch + 1 + at.b] - a.tokens + x.t + 1) : INT_MAX;
      }
      __syncthreads();
      min_limit = INT_MAX;
#pragma unroll
      for (int r = 0; r < 16; ++r) min_limit = min(min_limit, limits[wr * 16 + r]);
      lim[0] = limits[wr * 16 + quad_row];
      lim[1] = limits[wr * 16 + quad_row + 8];
#pragma unroll
      for (int n = 0; n < kDt; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[n][e] = 0.0f;
      m[0] = m[1] = -INFINITY;
      l[0] = l[1] = 0.0f;
    }

    const unsigned k_at = smem_at + ((w - first) % kStages) * 2 * S::kTileBytes, v_at = k_at + S::kTileBytes;
    const unsigned q_at = smem_at + S::kOffQ + (q_now % kStages) * S::kQBytes;
    const int pos0 = begin + at.tile * kTile + wk * kKeys;
    float s[kNt][4];
#pragma unroll
    for (int n = 0; n < kNt; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[n][e] = 0.0f;
#pragma unroll
    for (int k = 0; k < DT / 16; ++k) {
      unsigned qa[4];
      ldsm4(qa, q_at + at_chunk<DT>(wr * 16 + (lane & 15), 2 * k + (lane >> 4)));
#pragma unroll
      for (int n = 0; n < kNt; n += 2) {
        unsigned kb[4];
        ldsm4(kb, k_at + at_chunk<DT>(wk * kKeys + n * 8 + (lane >> 4) * 8 + (lane & 7), 2 * k + ((lane >> 3) & 1)));
        mma(s[n], qa, kb[0], kb[1], T{});
        mma(s[n + 1], qa, kb[2], kb[3], T{});
      }
    }
    const bool masked = pos0 + kKeys > min_limit;
    if (masked) {
#pragma unroll
      for (int n = 0; n < kNt; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (pos0 + n * 8 + (lane & 3) * 2 + (e & 1) >= lim[e >> 1]) s[n][e] = -INFINITY;
    }
    float scale_o[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float top = m[i];
#pragma unroll
      for (int n = 0; n < kNt; ++n) top = fmaxf(top, fmaxf(s[n][2 * i], s[n][2 * i + 1]) * a.scale_log2);
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const float from = weights_from<T>(top, kLift);
      const float ref = from == -INFINITY ? 0.0f : from;  // a row that has seen nothing yet: exp2(-inf - 0) = 0
      scale_o[i] = exp2_fast(weights_from<T>(m[i], kLift) - ref);
      m[i] = top;
      float sum = 0.0f;
#pragma unroll
      for (int n = 0; n < kNt; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float p = exp2_fast(fmaf(s[n][2 * i + e], a.scale_log2, -ref));
          s[n][2 * i + e] = p;
          sum += p;
        }
      l[i] = l[i] * scale_o[i] + sum;
    }
#pragma unroll
    for (int n = 0; n < kDt; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[n][e] *= scale_o[e >> 1];
    if (masked && not_finite<T, DT, kKeys>(v_at, wk * kKeys, lane)) {
      // A value that some row must not see is not finite: 0 * v would carry it over. One position after the other.
#pragma unroll
      for (int n = 0; n < kNt; ++n)
        for (int j = 0; j < 8; ++j) {
          const int key = n * 8 + j, from = (lane & ~3) | (j >> 1);
          const float p0 = round_through<T>(__shfl_sync(0xffffffffu, j & 1 ? s[n][1] : s[n][0], from));
          const float p1 = round_through<T>(__shfl_sync(0xffffffffu, j & 1 ? s[n][3] : s[n][2], from));
          const bool see0 = pos0 + key < lim[0], see1 = pos0 + key < lim[1];
#pragma unroll
          for (int c = 0; c < kDt; ++c) {
            const float2 v = load2(v_at + at_chunk<DT>(wk * kKeys + key, c) + (lane & 3) * 4, T{});
            if (see0) {
              o[c][0] = fmaf(p0, v.x, o[c][0]);
              o[c][1] = fmaf(p0, v.y, o[c][1]);
            }
            if (see1) {
              o[c][2] = fmaf(p1, v.x, o[c][2]);
              o[c][3] = fmaf(p1, v.y, o[c][3]);
            }
          }
        }
    } else
#pragma unroll
    for (int k = 0; k < kKeys / 16; ++k) {
      unsigned pa[4];
      pa[0] = pack2(s[2 * k][0], s[2 * k][1], T{});
      pa[1] = pack2(s[2 * k][2], s[2 * k][3], T{});
      pa[2] = pack2(s[2 * k + 1][0], s[2 * k + 1][1], T{});
      pa[3] = pack2(s[2 * k + 1][2], s[2 * k + 1][3], T{});
#pragma unroll
      for (int n = 0; n < kDt; n += 2) {
        unsigned vb[4];
        ldsm4_trans(vb, v_at + at_chunk<DT>(wk * kKeys + k * 16 + (lane & 15), n + (lane >> 4)));
        mma(o[n], pa, vb[0], vb[1], T{});
        mma(o[n + 1], pa, vb[2], vb[3], T{});
      }
    }

    if (at.tile + 1 == at.tiles || w + 1 == last) {  // the end of a piece
      const bool whole = !kShared && begin == 0 && piece_begin == 0 && at.tile + 1 == at.tiles;
      const long long slot = (long long)at.b * units + at.unit + blockIdx.x;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
        m[i] = weights_from<T>(m[i], kLift);
      }
      if (S::kKeyWarps > 1) {  // join the warps that shared the positions, in the tile's own stage
        if ((lane & 3) == 0) {
          ml_sh[wk * kRows + wr * 16 + quad_row] = make_float2(m[0], l[0]);
          ml_sh[wk * kRows + wr * 16 + quad_row + 8] = make_float2(m[1], l[1]);
        }
        __syncthreads();  // and nobody reads the tile any more
        float* sum_o = reinterpret_cast<float*>(smem + ((w - first) % kStages) * 2 * S::kTileBytes);
        float weight[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int r = wr * 16 + quad_row + 8 * i;
          const float mine = m[i];
          float top = -INFINITY, sum = 0.0f;
#pragma unroll
          for (int k = 0; k < S::kKeyWarps; ++k) top = fmaxf(top, ml_sh[k * kRows + r].x);
          const float ref = top == -INFINITY ? 0.0f : top;
#pragma unroll
          for (int k = 0; k < S::kKeyWarps; ++k) sum += ml_sh[k * kRows + r].y * exp2_fast(ml_sh[k * kRows + r].x - ref);
          weight[i] = exp2_fast(mine - ref);
          m[i] = top;
          l[i] = sum;
        }
        for (int k = 0; k < S::kKeyWarps; ++k) {
          if (wk == k) {
#pragma unroll
            for (int n = 0; n < kDt; ++n)
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                float2* dst = reinterpret_cast<float2*>(sum_o + (wr * 16 + quad_row + 8 * i) * DT + n * 8 + (lane & 3) * 2);
                float2 v = make_float2(o[n][2 * i] * weight[i], o[n][2 * i + 1] * weight[i]);
                if (k > 0) {
                  const float2 u = *dst;
                  v.x += u.x;
                  v.y += u.y;
                }
                *dst = v;
                o[n][2 * i] = v.x;
                o[n][2 * i + 1] = v.y;
              }
          }
          __syncthreads();
        }
      }
      if (wk == S::kKeyWarps - 1) {  // the last to add holds the sums
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int r = wr * 16 + quad_row + 8 * i;
          write_row<T, DT>(a, row_of<kShared>(a, at.b, kv_head, row0 + r), whole, lim[i] > 0, slot * kRows + r, lane, o, i,
                           m[i], l[i]);
        }
      }
    }
    axis_next(cum, seqs, units, at);
    if (looking) {
      if (tid < kTile) row_at[(looked & 1) * kTile + tid] = next_row;
      axis_next(cum, seqs, units, look);
      ++looked;
    }
  }
  copy_wait<0>();
  if (!kShared && a.beside && blockIdx.x == 0) pdl_wait();  // this grid ends after the shared work's
}

}  // namespace
}  // namespace ckb

#include "attention_stream.cuh"
#include "attention_prefix.cuh"

namespace ckb {
namespace {

// Joins the pieces of each output row (b, t, head).
struct JoinArgs {
  void* out;
  const long long* lens;
  const float *own_part, *shared_part;
  const float2 *own_ml, *shared_ml;
  const int* plan;
  int batch, tokens, q_heads, kv_heads, group, head_dim, prefix, rows, table_positions;
  int own_rows, own_row_tiles;        // rows of an own slot, row tiles of an own unit
  int shared_rows, shared_unit_rows;  // rows of a slot and of a unit of the shared work
  int shared_row_tiles;               // 0: none
  int shared_tiles, shared_run;       // tiles of a shared unit, tiles of a run
  int shared_slots, shared_split;     // slots of a piece; whether they are parts of the positions, not of the rows
};

// kWarps warps take a row's pieces in turn: 1 where there are rows enough to fill the GPU, 8 where a few rows have many pieces.
template <typename T, int kWarps>
__global__ void __launch_bounds__(256) join_rows(const JoinArgs a) {
  constexpr int kAhead = 8;  // pieces whose loads are in flight together
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, part = warp % kWarps;
  const int b = blockIdx.y, row = blockIdx.x * (8 / kWarps) + warp / kWarps;  // row of the sequence
  if (row >= a.tokens * a.q_heads) return;
  const int t = row / a.q_heads, head = row - t * a.q_heads;
  const int kv_head = head / a.group, in = t * a.group + (head - kv_head * a.group);

  // Own pieces: slots own_slot, own_slot + 1, ...; shared ones the same.
  const int units = a.kv_heads * a.own_row_tiles, unit = kv_head * a.own_row_tiles + in / a.own_rows;
  const int begin = a.plan[b], tiles = (a.plan[b + 1] - begin) / units;
  const Runs runs{a.plan[a.batch + 1], a.plan[a.batch + 2], a.plan[a.batch + 3]};
  const long long n = a.lens[b];
  const int len = (int)(n < 0 ? 0 : n < a.table_positions ? n : a.table_positions);
  const bool sharing = a.shared_row_tiles > 0 && own_begin(a.prefix, a.tokens, len) > 0;
  int own = 0;
  long long own_at = 0;  // workspace row of the first own piece
  if (tiles > 0) {
    const int w0 = begin + unit * tiles, c0 = runs.cta_of(w0);
    own = runs.cta_of(w0 + tiles - 1) - c0 + 1;
    own_at = ((long long)b * units + unit + c0) * a.own_rows + in % a.own_rows;
    if (own == 1 && !sharing) return;  // written out by its CTA (the same for all warps of the row)
  }
  int shared = 0, shared_step = 0;
  long long shared_at = 0;
  if (sharing) {
    const int all_row = b * a.rows + in, in_unit = all_row % a.shared_unit_rows;
    const int u = kv_head * a.shared_row_tiles + all_row / a.shared_unit_rows, w0 = u * a.shared_tiles, c0 = w0 / a.shared_run;
    shared = (w0 + a.shared_tiles - 1) / a.shared_run - c0 + 1;
    shared_step = a.shared_slots * a.shared_rows;
    shared_at = (u + (long long)c0) * shared_step + in_unit;  // slots of the unit's row tiles lie one after the other
    if (a.shared_split) {
      shared *= a.shared_slots;
      shared_step = a.shared_rows;
    }
  }
  const int pieces = own + shared;
  const bool some = len - a.tokens + t + 1 > 0;
  T* out = (T*)a.out + ((long long)b * a.tokens * a.q_heads + row) * a.head_dim;
  __shared__ float4 partial[kWarps > 1 ? 8 : 1][32];
  __shared__ float2 partial_ml[8];
  for (int c0 = 0; c0 < a.head_dim; c0 += 128) {
    const int c = c0 + lane * 4;
    const bool inside = some && c < a.head_dim;
    float m = -INFINITY, l = 0.0f;
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int i0 = part; i0 < pieces; i0 += kAhead * kWarps) {
      float4 v[kAhead];
      float2 ml[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {  // statistics and sums together
        const int i = i0 + k * kWarps;
        v[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        ml[k] = make_float2(-INFINITY, 0.0f);
        if (i < pieces) {
          const long long w = i < own ? own_at + (long long)i * a.own_rows : shared_at + (long long)(i - own) * shared_step;
          ml[k] = (i < own ? a.own_ml : a.shared_ml)[w];
          if (inside) v[k] = *reinterpret_cast<const float4*>((i < own ? a.own_part : a.shared_part) + w * a.head_dim + c);
        }
      }
      float top = m;
#pragma unroll
      for (int k = 0; k < kAhead; ++k) top = fmaxf(top, ml[k].x);
      const float ref = top == -INFINITY ? 0.0f : top, down = exp2_fast(m - ref);
      m = top;
      l *= down;
      acc = make_float4(acc.x * down, acc.y * down, acc.z * down, acc.w * down);
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const float x = exp2_fast(ml[k].x - ref);
        l = fmaf(x, ml[k].y, l);
        acc.x = fmaf(x, v[k].x, acc.x);
        acc.y = fmaf(x, v[k].y, acc.y);
        acc.z = fmaf(x, v[k].z, acc.z);
        acc.w = fmaf(x, v[k].w, acc.w);
      }
    }
    if (kWarps > 1) {
      partial[warp][lane] = acc;
      if (lane == 0) partial_ml[warp] = make_float2(m, l);
      __syncthreads();  // a block has one row then
      if (part == 0) {
        float top = m;
#pragma unroll
        for (int k = 1; k < kWarps; ++k) top = fmaxf(top, partial_ml[k].x);
        const float ref = top == -INFINITY ? 0.0f : top;
        l = 0.0f;
        acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int k = 0; k < kWarps; ++k) {
          const float4 v = partial[k][lane];
          const float x = exp2_fast(partial_ml[k].x - ref);
          l = fmaf(x, partial_ml[k].y, l);
          acc = make_float4(fmaf(x, v.x, acc.x), fmaf(x, v.y, acc.y), fmaf(x, v.z, acc.z), fmaf(x, v.w, acc.w));
        }
      }
      __syncthreads();
    }
    if (part == 0 && c < a.head_dim) {
      const float inv = 1.0f / l;
      const uint2 v = make_uint2(pack2(acc.x * inv, acc.y * inv, T{}), pack2(acc.z * inv, acc.w * inv, T{}));
      *reinterpret_cast<uint2*>(out + c) = some ? v : make_uint2(0u, 0u);
    }
  }
}

// ---------------------------------------------------------------------------------------------------------------
// Host side.
// ---------------------------------------------------------------------------------------------------------------
struct Sizes {
  int rows, own_warps, own_rows, own_row_tiles, own_per_sm, own_ctas;
  // The shared work on the tensor cores of the fifth generation (0), or by attend_tiles (1).
  struct { int unit_rows, row_tiles, tiles, ctas, run, rows, slots; } shared[2];
  long long own_slots, off_plan, off_own_ml, off_own, off_shared_ml, off_shared, bytes;
};

// CTAs of the own work that an SM holds (attend_stream).
template <int DT>
int per_sm_of(int warps, int batch) {
  return warps == 1 ? Ring<DT, 1>::per_sm(batch) : warps == 2 ? Ring<DT, 2>::per_sm(batch) : Ring<DT, 4>::per_sm(batch);
}
int per_sm(int head_dim, int warps, int batch) {
  return head_dim <= 64    ? per_sm_of<64>(warps, batch)
         : head_dim <= 128 ? per_sm_of<128>(warps, batch)
                           : per_sm_of<256>(warps, batch);
}

bool sizes_of(long long batch, int tokens, int q_heads, int kv_heads, int head_dim, int block_size, long long table_width,
              long long prefix, Sizes& z) {
  if (batch < 1 || batch > kMaxBatch || tokens < 1 || tokens > 65536 || q_heads < 1 || kv_heads < 1 ||
      q_heads > 65536 || q_heads % kv_heads || head_dim < 8 || head_dim > 256 || head_dim % 8 || block_size < 1 ||
      table_width < 1 || prefix < 0 || prefix % block_size || table_width > INT_MAX / block_size - kTile ||
      prefix > table_width * block_size)
    return false;
  const long long rows = (long long)tokens * (q_heads / kv_heads);
  if (rows * batch * kv_heads > (1 << 26)) return false;
  if (batch == 1) prefix = 0;  // nobody to share it with
  z = Sizes{};
  z.rows = (int)rows;
  z.own_warps = rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
  z.own_rows = 16 * z.own_warps;
  z.own_row_tiles = (int)((rows + z.own_rows - 1) / z.own_rows);
  const long long tiles = (table_width * block_size + kTile - 1) / kTile;
  if (tiles * batch * kv_heads * z.own_row_tiles > INT_MAX / 2) return false;
  z.own_per_sm = per_sm(head_dim, z.own_warps, (int)batch);
  const int most = device_sm_count() * z.own_per_sm;
  z.own_ctas = most;
  z.own_slots = batch * kv_heads * z.own_row_tiles + z.own_ctas;
  long long shared_rows = 0;  // of the workspace
  for (int i = 0; i < 2 && prefix > 0; ++i) {
    auto& h = z.shared[i];
    h.rows = i == 0 ? kGroupRows : 64;
    h.unit_rows = i == 0 && rows * batch > kGroupRows ? 2 * kGroupRows : h.rows;
    h.slots = i == 0 ? 2 : 1;
    h.row_tiles = (int)((rows * batch + h.unit_rows - 1) / h.unit_rows);
    const int tile = i == 0 ? kPrefixTile : kTile, at_once = i == 0 ? device_sm_count() * kPrefixShare / 8 : most;
    h.tiles = (int)((prefix + tile - 1) / tile);
    const long long all = (long long)h.tiles * kv_heads * h.row_tiles;
    if (all > INT_MAX / 2) return false;
    h.run = (int)((all + at_once - 1) / at_once);
    if (i == 0) h.run = std::max(h.run, std::min(kPrefixRun, h.tiles));  // longer than a short unit where units are many
    h.ctas = (int)((all + h.run - 1) / h.run);
    const long long need = ((long long)kv_heads * h.row_tiles + h.ctas) * h.slots * h.rows;
    if (need > shared_rows) shared_rows = need;
  }
  const auto up = [](long long n) { return (n + 255) / 256 * 256; };
  z.off_plan = 0;
  z.off_own_ml = up((batch + 4) * 4);
  z.off_own = z.off_own_ml + up(z.own_slots * z.own_rows * 8);
  z.off_shared_ml = z.off_own + up(z.own_slots * z.own_rows * head_dim * 4);
  z.off_shared = z.off_shared_ml + up(shared_rows * 8);
  z.bytes = z.off_shared + up(shared_rows * head_dim * 4);
  return true;
}

// Lets a kernel have all of an SM's shared memory, once for each device (up to 64; a call takes a microsecond).
template <typename K>
cudaError_t open_shared_memory(K* kernel, std::atomic<unsigned long long>& done) {
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err != cudaSuccess) return err;
  const unsigned long long bit = 1ull << (dev & 63);
  if (dev < 64 && (done.load(std::memory_order_acquire) & bit)) return cudaSuccess;
  err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxShared);
  if (err == cudaSuccess && dev < 64) done.fetch_or(bit, std::memory_order_release);
  return err;
}

template <typename T, int DT, int WR, bool kShared>
cudaError_t start(const Args& a, int ctas, cudaStream_t stream) {
  using S = Shape<T, DT, WR, kShared>;
  const int bytes = S::bytes(a.batch);
  static std::atomic<unsigned long long> done{0};
  const cudaError_t err = open_shared_memory(attend_tiles<T, DT, WR, kShared>, done);
  if (err != cudaSuccess) return err;
  return launch_pdl(attend_tiles<T, DT, WR, kShared>, dim3(ctas), dim3(kThreads), bytes, stream, a);
}

// Whether a head has the columns of a tile, so that a box brings whole rows; else the tile's last columns are filled up.
bool whole_rows(const Args& a) { return a.head_dim == 64 || a.head_dim == 128 || a.head_dim == 256; }
// The cache as a TMA reads it: [kv_heads][blocks of 64 columns][rows][64], boxes of box_rows rows of one head (where they
// are not 64, 128 or 256 columns: [kv_heads][1][rows][head_dim], boxes of 64 columns).
using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                 const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiled encode_tiled() {
  static const EncodeTiled fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &found) != cudaSuccess ||
        found != cudaDriverEntryPointSuccess) {
      cudaGetLastError();
      p = nullptr;
    }
    return reinterpret_cast<EncodeTiled>(p);
  }();
  return fn;
}
template <typename T>
bool cache_map(const Args& a, const void* cache, int box_rows, CUtensorMap& map) {
  const EncodeTiled encode = encode_tiled();
  if (encode == nullptr) return false;
  const cuuint64_t rows = (cuuint64_t)a.num_blocks * a.block_size, row_bytes = (cuuint64_t)a.head_dim * a.kv_heads * 2;
  const bool whole = whole_rows(a);
  const cuuint64_t dims[4] = {whole ? 64 : (cuuint64_t)a.head_dim, rows, whole ? (cuuint64_t)a.head_dim / 64 : 1,
                              (cuuint64_t)a.kv_heads};
  const cuuint64_t strides[3] = {row_bytes, 128, (cuuint64_t)a.head_dim * 2};
  const cuuint32_t box[4] = {64, (cuuint32_t)box_rows, (cuuint32_t)dims[2], 1}, step[4] = {1, 1, 1, 1};
  const CUtensorMapDataType type =
      sizeof(T) == 2 && std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  return encode(&map, type, 4, const_cast<void*>(cache), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// Whether boxes of whole pages, or of 64 rows of a page, make up a tile (see attention_stream.cuh).
bool boxes_fit(const Args& a) {
  return a.block_size % 8 == 0 && (kTile % a.block_size == 0 || a.block_size % kTile == 0) && a.num_blocks > 0 &&
         a.num_blocks * a.block_size < INT_MAX;
}

struct Maps {
  bool fit;
  int rows_log;  // rows of a box
  CUtensorMap keys, values;
};

template <typename T>
Maps maps_of(const Args& a, int rows_log) {
  Maps m;
  m.rows_log = rows_log;
  m.fit = boxes_fit(a) && cache_map<T>(a, a.key, 1 << rows_log, m.keys) && cache_map<T>(a, a.value, 1 << rows_log, m.values);
  return m;
}

template <typename T, int DT, int WR>
cudaError_t start_stream(const Args& a, int ctas, const Maps& maps, cudaStream_t stream) {
  const int bytes = Ring<DT, WR>::bytes(a.batch);
  static std::atomic<unsigned long long> done{0};
  const cudaError_t err = open_shared_memory(attend_stream<T, DT, WR>, done);
  if (err != cudaSuccess) return err;
  return launch_pdl(attend_stream<T, DT, WR>, dim3(ctas), dim3(32 * (kConsumers + 1)), bytes, stream, a, maps.rows_log,
                    maps.keys, maps.values);
}

template <typename T, int DT>
cudaError_t start_own(const Args& a, int warps, int ctas, const Maps& maps, cudaStream_t stream) {
  if (maps.fit) {
    if (warps == 1) return start_stream<T, DT, 1>(a, ctas, maps, stream);
    if (warps == 2) return start_stream<T, DT, 2>(a, ctas, maps, stream);
    return start_stream<T, DT, 4>(a, ctas, maps, stream);
  }
  if (warps == 1) return start<T, DT, 1, false>(a, ctas, stream);
  if (warps == 2) return start<T, DT, 2, false>(a, ctas, stream);
  return start<T, DT, 4, false>(a, ctas, stream);
}

template <typename T, int DT>
cudaError_t start_prefix(const Args& a, const Sizes& z, const Maps& own_maps, cudaStream_t stream) {
  const int rows_log = a.block_size == 8 ? 3 : 4;
  const Maps maps = own_maps.rows_log == rows_log ? own_maps : maps_of<T>(a, rows_log);
  if (!maps.fit) return cudaErrorInvalidValue;
  const auto& h = z.shared[0];
  const int bytes = PrefixShape<DT>::kBytes;
  static std::atomic<unsigned long long> done{0};
  const cudaError_t err = open_shared_memory(attend_prefix<T, DT>, done);
  if (err != cudaSuccess) return err;
  const PrefixArgs p{a, h.tiles, h.run, h.unit_rows, maps.rows_log};
  return launch_pdl(attend_prefix<T, DT>, dim3(h.ctas), dim3(kPrefixThreads), bytes, stream, p, maps.keys, maps.values);
}

template <typename T>
int start_all(Args a, const Sizes& z, unsigned char* work, cudaStream_t stream) {
  const int dt = a.head_dim <= 64 ? 64 : a.head_dim <= 128 ? 128 : 256;
  int rows_log = 3;  // a page, at most a tile's rows
  while (rows_log < 6 && 2 << rows_log <= a.block_size) ++rows_log;
  const Maps maps = maps_of<T>(a, rows_log);
  // Two groups' O and S of 256 columns each do not fit TMEM: heads of more than 128 columns take attend_tiles.
  const bool tensor = maps.fit && dt <= 128;
  const auto& h = z.shared[tensor ? 0 : 1];
  // The own work does not need the shared work's results, only the join does. So where both are there, it does not wait for
  // it: the shared work's CTAs wait for what came before on the stream and then let the own work's start, on the SMs that
  // they leave free and on theirs as they end; the own work's first CTA waits for the shared work before it ends, so that the
  // join, which waits for the own work, follows both.
  cudaError_t err = cudaSuccess;
  Args s = a;
  a.beside = a.prefix > 0;
  if (a.beside && tensor && h.ctas < device_sm_count()) {
    a.early = (device_sm_count() - h.ctas) * z.own_per_sm;
    a.ahead = (kPrefixCtaNs + h.run * (h.unit_rows == h.rows ? kPrefixTileNs / 2 : kPrefixTileNs)) / kOwnTileNs;
  }
  a.row_tiles = z.own_row_tiles;
  a.part = reinterpret_cast<float*>(work + z.off_own);
  a.ml = reinterpret_cast<float2*>(work + z.off_own_ml);
  s.row_tiles = h.row_tiles;
  s.part = reinterpret_cast<float*>(work + z.off_shared);
  s.ml = reinterpret_cast<float2*>(work + z.off_shared_ml);
  if (a.prefix > 0) {
    if (tensor)
      err = dt == 64 ? start_prefix<T, 64>(s, z, maps, stream) : start_prefix<T, 128>(s, z, maps, stream);
    else
      err = dt == 64 ? start<T, 64, 4, true>(s, h.ctas, stream)
            : dt == 128 ? start<T, 128, 4, true>(s, h.ctas, stream)
                        : start<T, 256, 4, true>(s, h.ctas, stream);
  }
  int ctas = z.own_ctas;
  if (!maps.fit) {  // what attend_tiles' larger stages leave room for
    const int fit = device_sm_count() * (dt == 64 ? 4 : dt == 128 ? 2 : 1);
    ctas = fit < ctas ? fit : ctas;
  }
  if (err == cudaSuccess)
    err = dt == 64 ? start_own<T, 64>(a, z.own_warps, ctas, maps, stream)
          : dt == 128 ? start_own<T, 128>(a, z.own_warps, ctas, maps, stream)
                      : start_own<T, 256>(a, z.own_warps, ctas, maps, stream);
  if (err == cudaSuccess) {
    const JoinArgs j{a.out, a.lens, a.part, s.part, a.ml, s.ml, a.plan, a.batch, a.tokens, a.q_heads, a.kv_heads, a.group,
                     a.head_dim, a.prefix, a.rows, a.table_width * a.block_size, z.own_rows, z.own_row_tiles, h.rows,
                     h.unit_rows, h.row_tiles, h.tiles, h.run, h.slots, h.unit_rows == h.rows && h.slots > 1};
    const int rows = a.tokens * a.q_heads;
    err = (long long)rows * a.batch < 8LL * device_sm_count()
              ? launch_pdl(join_rows<T, 8>, dim3(rows, a.batch), dim3(256), 0, stream, j)
              : launch_pdl(join_rows<T, 1>, dim3((rows + 7) / 8, a.batch), dim3(256), 0, stream, j);
  }
  if (err != cudaSuccess) {
    cudaGetLastError();
    return (int)err;
  }
  return (int)cudaGetLastError();
}

}  // namespace
}  // namespace ckb

using namespace ckb;

CKB_EXPORT long long ckb_attention_workspace(long long batch, int tokens, int q_heads, int kv_heads, int head_dim,
                                             int block_size, long long table_width, long long shared_prefix) {
  Sizes z;
  return sizes_of(batch, tokens, q_heads, kv_heads, head_dim, block_size, table_width, shared_prefix, z) ? z.bytes : -1;
}

CKB_EXPORT int ckb_attention_paged_launch(const void* q, const void* key_cache, const void* value_cache,
                                          const void* tables, const void* lens, void* out, void* work,
                                          long long work_bytes, const long long* q_strides, long long batch, int tokens,
                                          int q_heads, int kv_heads, int head_dim, long long num_blocks, int block_size,
                                          long long table_width, long long shared_prefix, float scale, int dtype,
                                          cudaStream_t stream) {
  if (batch <= 0) return 0;
  Sizes z;
  if (!sizes_of(batch, tokens, q_heads, kv_heads, head_dim, block_size, table_width, shared_prefix, z)) return -1;
  if (q == nullptr || tables == nullptr || lens == nullptr || out == nullptr || work == nullptr || q_strides == nullptr ||
      num_blocks < 0 || (num_blocks > 0 && (key_cache == nullptr || value_cache == nullptr)) || work_bytes < z.bytes ||
      !aligned16(q) || !aligned16(key_cache) || !aligned16(value_cache) || !aligned16(out) || !aligned16(work) ||
      q_strides[0] % 8 || q_strides[1] % 8 || q_strides[2] % 8 || !(scale > 0.0f) || scale > 1e30f)
    return -1;
  unsigned char* w = static_cast<unsigned char*>(work);
  Args a{};
  a.q = q;
  a.key = key_cache;
  a.value = value_cache;
  a.tables = static_cast<const long long*>(tables);
  a.lens = static_cast<const long long*>(lens);
  a.out = out;
  a.plan = reinterpret_cast<int*>(w + z.off_plan);
  a.vq = View3{q_strides[0], q_strides[1], q_strides[2]};
  a.num_blocks = num_blocks;
  a.batch = (int)batch;
  a.tokens = tokens;
  a.q_heads = q_heads;
  a.kv_heads = kv_heads;
  a.group = q_heads / kv_heads;
  a.head_dim = head_dim;
  a.block_size = block_size;
  a.block_log = block_size & (block_size - 1) ? -1 : __builtin_ctz(block_size);
  a.table_width = (int)table_width;
  a.prefix = batch == 1 ? 0 : (int)shared_prefix;
  a.rows = z.rows;
  a.scale_log2 = scale * kLog2e;
  if (dtype == kBF16) return start_all<__nv_bfloat16>(a, z, w, stream);
  if (dtype == kF16) return start_all<__half>(a, z, w, stream);
  return -1;
}

// Status of the bounded waits since the last reset: 0, or 1 when a wait gave up (that launch's output is void).
CKB_EXPORT int ckb_attention_status(int reset) {
  unsigned int v = 0;
  cudaError_t e = cudaDeviceSynchronize();  // the copy alone does not wait for streams that are non-blocking
  if (e == cudaSuccess) e = cudaMemcpyFromSymbol(&v, g_attention_status, sizeof(v));
  if (e != cudaSuccess) return -(int)e;
  if (reset && v != 0u) {
    const unsigned int zero = 0u;
    e = cudaMemcpyToSymbol(g_attention_status, &zero, sizeof(zero));
    if (e != cudaSuccess) return -(int)e;
  }
  return (int)v;
}
