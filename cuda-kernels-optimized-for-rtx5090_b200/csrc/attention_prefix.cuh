// The shared prefix on the fifth-generation tensor cores (included by attention.cu, whose parts it uses).
//
// A unit is a kv head and 256 (or, where the batch has no more, 128) of the query rows that share it, those of all
// sequences one after the other; its tiles are 128 positions of the prefix. Every row sees every position, so nothing is
// masked but the last tile's overhang. For 128 rows and 128 positions a tile takes 2 x 2 x 128 x 128 x D operations: at
// D = 128 about 1024 clocks of an SM's tensor cores, and 128 x 128 exponentials, 1024 clocks of its MUFUs, while its keys and
// values take about 2800 clocks of an SM's share of HBM, shared by the two row tiles of a unit and, through L2, by the
// other units of the head. So the products and the exponentials have to run at the same time, and do:
//   warps 0-3, 4-7  a softmax group each, a thread a row: scores S from TMEM, running maximum, exp, the weights P back to
//                   TMEM in 16 bits over S, the sum of the unrounded weights in fp32;
//   warps 8, 11     look the pages up and load keys and values by TMA, one each (rings of two tiles);
//   warps 9, 10     issue S = Q K^T and O += P V (P from TMEM), one for each group.
// A step is half a tile, 64 positions, so that each group has two S buffers: while it works on one, the tensor cores fill
// the other. (With one buffer of 128 positions a group waited 1.6 us for its next scores after 1.0 us of work on them: P,
// which lies over S, had to be used up first.)
// Two softmax groups that take turns on the tensor cores, and an O that is scaled down only when it has to be, are published
// techniques (Shah et al. 2024, arXiv 2407.08608; the second T. Dao, Hot Chips 2025).
// The two groups have a row tile of 128 each of a 256-row unit, or every other tile of positions of a 128-row unit (then
// they are two pieces). O stays in TMEM. It is scaled down only when a row's maximum has risen by more than 8 (powers of
// 2) over the one in use; until then weights may reach 2^8, which fp32 sums and 16-bit weights hold as well as 1. (fp16
// weights are lifted by 7 then, and reach 2^15.)
// 1024 rows x 8 heads x 16384 positions at D = 128 take 79 us, 870 TFLOP/s or 0.51 of the measured matrix rate, the tensor
// cores busy 43 % of the time. A step of the two groups takes 1500 clocks: products of 64 columns take 55 clocks instead of
// the 32 of their operations (both operands come from shared memory), 1420 in all for a step of the two; 128 columns have no
// room in TMEM beside two groups' O and a second buffer. The rest, 10 us, is a CTA's start (queries, first tile) and piece.
#pragma once

namespace ckb {
namespace {

constexpr int kPrefixTile = 128;  // positions of a tile
constexpr int kGroupRows = 128;   // query rows of a softmax group
constexpr int kPrefixThreads = 384;
constexpr int kStep = 64;         // positions of a step
constexpr float kSlack = 8.0f;    // by how much a maximum may fall behind
constexpr float kPrefixLift = kLift - kSlack;

// ---------------------------------------------------------------------------------------------------------------
// tcgen05 and TMEM, against the PTX ISA for sm_100a.
// ---------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ void tmem_alloc(unsigned* at, unsigned columns) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(at)), "r"(columns) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_free(unsigned at, unsigned columns) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(at), "r"(columns) : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// D (+)= A B, A and B in shared memory.
__device__ __forceinline__ void tc_mma(unsigned d, uint64_t a, uint64_t b, unsigned kind, bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(kind), "r"((unsigned)add)
      : "memory");
}
// The same with A in TMEM.
__device__ __forceinline__ void tc_mma_tmem(unsigned d, unsigned a, uint64_t b, unsigned kind, bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(kind), "r"((unsigned)add)
      : "memory");
}
// 32 columns of this thread's lane.
__device__ __forceinline__ void tmem_load32(unsigned at, unsigned (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, "
      "%18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]),
        "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]),
        "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]),
        "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(at));
}
__device__ __forceinline__ void tmem_store32(unsigned at, const unsigned (&v)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(at),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]),
      "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]),
      "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]),
      "r"(v[31])
      : "memory");
}
// Waits for this thread's loads. The values pass through it, so that no use of them is moved before it.
__device__ __forceinline__ void tmem_wait_load(unsigned (&v)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]),
                 "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]),
                 "+r"(v[15]), "+r"(v[16]), "+r"(v[17]), "+r"(v[18]), "+r"(v[19]), "+r"(v[20]), "+r"(v[21]),
                 "+r"(v[22]), "+r"(v[23]), "+r"(v[24]), "+r"(v[25]), "+r"(v[26]), "+r"(v[27]), "+r"(v[28]),
                 "+r"(v[29]), "+r"(v[30]), "+r"(v[31])
               :
               : "memory");
}
__device__ __forceinline__ void tmem_wait_store() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Shared-memory operand with the 128-byte swizzle: groups of 8 rows of 128 bytes are `stride` apart; `lead` is the distance
// of the next 64 columns of an operand whose rows run along the sum (values), unused for one whose columns do (queries, keys).
__device__ __forceinline__ uint64_t operand(unsigned at, unsigned lead, unsigned stride) {
  return (uint64_t)((at >> 4) & 0x3fffu) | (uint64_t)((lead >> 4) & 0x3fffu) << 16 | (uint64_t)((stride >> 4) & 0x3fffu) << 32 |
         1ull << 46 | 2ull << 61;
}
// Instruction descriptor: fp32 sums, A and B of T, 128 rows, `columns` columns, B's rows along the sum where `b_rows`.
template <typename T>
__device__ __forceinline__ unsigned mma_kind(int columns, bool b_rows) {
  const unsigned type = std::is_same<T, __half>::value ? 0u : 1u;
  return 1u << 4 | type << 7 | type << 10 | (b_rows ? 1u << 16 : 0u) | (unsigned)(columns >> 3) << 17 | (128u >> 4) << 24;
}

// wait_or_give_up for a wait that decides the tensor cores' pace: it polls instead of sleeping.
__device__ __forceinline__ void wait_quick(uint64_t* bar, unsigned parity, bool& dead) {
#pragma unroll 1
  for (int i = 0; i < 256; ++i)
    if (mbar_try_wait(bar, parity)) return;
  wait_or_give_up(bar, parity, dead);
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

struct PrefixArgs {
  Args a;
  int tiles, run;  // tiles of a unit, tiles of a CTA's run
  int unit_rows;   // 256: the groups have 128 rows each; 128: they have every other tile each
  int rows_log;    // rows of a box: 8 or 16
};

template <int DT>
struct PrefixShape {
  static constexpr int kTileBytes = kPrefixTile * DT * 2;
  static constexpr int kOffK = 2 * kGroupRows * DT * 2;
  static constexpr int kOffV = kOffK + 2 * kTileBytes;
  static constexpr int kOffBars = kOffV + 2 * kTileBytes;
  static constexpr int kOffRows = kOffBars + 22 * 8 + 16;
  static constexpr int kBytes = kOffRows + 2 * kGroupRows * 8 + 1024;
  static constexpr int kHalf = kPrefixTile * 128;  // bytes of 64 columns of a tile
};

template <typename T, int DT>
__global__ void __launch_bounds__(kPrefixThreads, 1)
    attend_prefix(const PrefixArgs p, const __grid_constant__ CUtensorMap key_map, const __grid_constant__ CUtensorMap value_map) {
  using S = PrefixShape<DT>;
  const Args& a = p.a;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const unsigned smem_at = smem_u32(smem);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::kOffBars);
  uint64_t *k_full = bars, *k_empty = bars + 2, *v_full = bars + 4, *v_empty = bars + 6;  // by stage
  uint64_t* q_full = bars + 8;  // by group
  uint64_t *s_full = bars + 10, *p_full = bars + 14, *o_full = bars + 18;  // by group and buffer
  unsigned* tmem_sh = reinterpret_cast<unsigned*>(bars + 22);
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  const bool alternate = p.unit_rows == kGroupRows;
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], alternate ? 1 : 2);  // a tile is read by one group, or by both
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], alternate ? 1 : 2);
      mbar_init(&q_full[i], kGroupRows);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], kGroupRows);
      mbar_init(&o_full[i], 1);
    }
    mbar_fence_init();
    tma_prefetch(&key_map);
    tma_prefetch(&value_map);
  }
  if (warp == 9) tmem_alloc(tmem_sh, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const unsigned tmem = __shfl_sync(0xffffffffu, *tmem_sh, 0);  // columns: S of group 0 (two buffers of 64, P over S), of group 1, then O_0, O_1
  pdl_wait();
  pdl_trigger();

  const int units = a.kv_heads * a.row_tiles;
  const int first = blockIdx.x * p.run, last = min(first + p.run, units * p.tiles);
  bool dead = false;
  if (warp == 8 || warp == 11) {
    const bool is_v = warp == 11;
    uint64_t *full = is_v ? v_full : k_full, *empty = is_v ? v_empty : k_empty;
    const CUtensorMap* map = is_v ? &value_map : &key_map;
    const unsigned ring = smem_at + (is_v ? S::kOffV : S::kOffK);
    const int box_rows = 1 << p.rows_log, pages = kPrefixTile >> p.rows_log, blocks = a.head_dim == DT ? 1 : DT / 64;
    const int page_bytes = box_rows * 128 * (DT / 64);
    const int outside = (int)(a.num_blocks * a.block_size);  // rows of zeros, which a weight of zero must meet
    const bool leader = elect_one();
    // Lane p looks up page p of a tile a tile ahead, as in attend_stream.
    const long long* table = a.tables;
    long long block_next = -1;
    int inside_next = 0;
    const auto look_up = [&](int tile) {
      const int pos = tile * kPrefixTile + lane * box_rows;
      block_next = -1;
      if (lane >= pages || pos >= a.prefix) return;
      const int page = a.block_log >= 0 ? pos >> a.block_log : pos / a.block_size;
      inside_next = pos - page * a.block_size;
      block_next = load_list(table + page);
    };
    int unit = first / p.tiles, tile = first - unit * p.tiles;
    int in_piece = 0, uses0 = 0, uses1 = 0;
    look_up(tile);  // through the first row, on its way while the lengths say whether that is the one to use
    const int row = first_sharing(a);
    if (row != 0) {
      table += (long long)row * a.table_width;
      look_up(tile);
    }
    for (int w = first; w < last; ++w) {
      // Alternate tiles of a piece have a stage each, that of their group, so that every group meets its stage's phases
      // one after the other.
      const int stage = (alternate ? in_piece : w - first) & 1, use = stage == 0 ? uses0++ : uses1++;
      const int kv_head = a.row_tiles == 1 ? unit : unit / a.row_tiles;
      ++in_piece;
      if (++tile == p.tiles) {
        tile = in_piece = 0;
        ++unit;
      }
      const int row_now =
          (int)(block_next < 0 || block_next >= a.num_blocks ? outside : block_next * a.block_size + inside_next);
      look_up(tile);
      wait_or_give_up(&empty[stage], (use & 1) ^ 1, dead);
      if (dead) break;
      if (leader) mbar_arrive_expect_tx(&full[stage], S::kTileBytes);
      const unsigned at = ring + stage * S::kTileBytes;
#pragma unroll 4
      for (int page = 0; page < pages; ++page) {
        const int row = __shfl_sync(0xffffffffu, row_now, page);
        if (leader)
          for (int block = 0; block < blocks; ++block)
            tma_load4(at + page * page_bytes + block * (box_rows * 128), map, block * 64, row, kv_head, &full[stage]);
      }
    }
  } else if (warp >= 9) {
    // The whole warp goes through this, so that addresses and descriptors stay in uniform registers; one lane issues.
    // Its group's step u takes half u & 1 of the group's (u >> 1)-th tile. Scores run two steps ahead of the weights'
    // products; those of step u + 2 go into the buffer that step u's weights lie in, so they wait for its product. A warp for
    // each group: one for both spent 2300 clocks on a step of the two, mostly on waits that were over (130 clocks each).
    const int g = warp - 9;
    const bool leader = elect_one();
    const unsigned score_kind = mma_kind<T>(kStep, false), value_kind = mma_kind<T>(DT, true);
    // Keys and values lie box by box: [box][64 columns][rows of the box][128 bytes]. A step of 64 positions is 8 groups of 8
    // rows at one distance: the first (second) 8 rows of each of the 8 boxes of 16, or the first (second) 8 boxes of 8. The
    // order of the positions within a tile does not matter, as keys and values have the same.
    const unsigned block = 128u << p.rows_log, box = block * (DT / 64), step = p.rows_log == 4 ? 1024u : 8u * box;
    const uint64_t q_operand = operand(smem_at + g * (kGroupRows * DT * 2), 16, 1024);
    const uint64_t k_operand = operand(smem_at + S::kOffK, 16, box), v_operand = operand(smem_at + S::kOffV, block, box);
    const unsigned s_at = tmem + g * 2 * kStep, o_at = tmem + 4 * kStep + g * DT;
    int phase = 0, pieces = 0;  // tiles of the pieces before, pieces
    for (int w = first; w < last;) {
      const int count = min(p.tiles - w % p.tiles, last - w), n0 = w - first;
      const int tiles = !alternate ? count : (count + 1 - g) / 2;  // of this group
      const auto scores = [&](auto half, int j) {
        constexpr int h = decltype(half)::value;
        const int stage = alternate ? g : (n0 + j) & 1, use = alternate ? phase + j : (n0 + j) >> 1;
        if (h == 0 && j == 0) wait_quick(&q_full[g], pieces & 1, dead);
        if (j > 0) wait_quick(&o_full[g * 2 + h], (phase + j - 1) & 1, dead);  // the buffer's last weights are used
        if (h == 0) wait_quick(&k_full[stage], use & 1, dead);
        tc_fence_after();
        const uint64_t k = k_operand + ((stage * S::kTileBytes + h * step) >> 4);
        if (leader) {
#pragma unroll
          for (int i = 0; i < DT / 16; ++i)
            tc_mma(s_at + h * kStep, q_operand + (((i >> 2) * S::kHalf + (i & 3) * 32) >> 4),
                   k + (((i >> 2) * block + (i & 3) * 32) >> 4), score_kind, i > 0);
          tc_commit(&s_full[g * 2 + h]);
          if (h == 1) tc_commit(&k_empty[stage]);
        }
        __syncwarp();
      };
      const auto values = [&](auto half, int j) {
        constexpr int h = decltype(half)::value;
        const int stage = alternate ? g : (n0 + j) & 1, use = alternate ? phase + j : (n0 + j) >> 1;
        if (h == 0) wait_quick(&v_full[stage], use & 1, dead);
        wait_quick(&p_full[g * 2 + h], (phase + j) & 1, dead);
        tc_fence_after();
        const uint64_t v = v_operand + ((stage * S::kTileBytes + h * step) >> 4);
        if (leader) {
#pragma unroll
          for (int i = 0; i < kStep / 16; ++i)
            tc_mma_tmem(o_at, s_at + h * kStep + i * 8, v + ((i * 2 * box) >> 4), value_kind, h > 0 || i > 0 || j > 0);
          tc_commit(&o_full[g * 2 + h]);
          if (h == 1) tc_commit(&v_empty[stage]);
        }
        __syncwarp();
      };
      constexpr std::integral_constant<int, 0> zero{};
      constexpr std::integral_constant<int, 1> one{};
      if (tiles > 0) {
        scores(zero, 0);
        scores(one, 0);
        for (int j = 0; j < tiles; ++j) {
          values(zero, j);
          if (j + 1 < tiles) scores(zero, j + 1);
          values(one, j);
          if (j + 1 < tiles) scores(one, j + 1);
        }
        ++pieces;
      }
      phase += tiles;
      w += count;
    }
  } else {
    const int g = warp >> 2, row = tid & (kGroupRows - 1);
    const unsigned lane_at = (unsigned)((warp & 3) * 32) << 16;
    const unsigned s_at = tmem + lane_at + g * 2 * kStep, o_at = tmem + lane_at + 4 * kStep + g * DT;
    long long* row_offset = reinterpret_cast<long long*>(smem + S::kOffRows) + g * kGroupRows;
    int step = 0;  // this group's steps so far
    for (int w = first; w < last;) {
      const int unit = w / p.tiles, tile0 = w - unit * p.tiles, count = min(p.tiles - tile0, last - w);
      const int kv_head = unit / a.row_tiles;
      const int row0 = (unit - kv_head * a.row_tiles) * p.unit_rows + (alternate ? 0 : g * kGroupRows);
      const bool any = !alternate || g < count;  // a piece of one tile has nothing for the second group
      // The piece's queries, in the products' layout. The copies of all rows are under way together. (Loops here and below
      // stay rolled up: each line of code that runs once costs its fetch, 14000 clocks in all for an unrolled form.)
      if (any) {
        const Row mine = row_of<true>(a, 0, kv_head, row0 + row);
        sync_warps(1 + g, kGroupRows);  // the last piece's rows have left these bytes, and their offsets are read
        row_offset[row] = mine.real ? mine.b * a.vq.batch + mine.t * a.vq.token + mine.head * a.vq.head : -1;
        sync_warps(1 + g, kGroupRows);
        constexpr int kChunks = DT / 8;
        const int chunk = row % kChunks;
        const unsigned q_to = smem_at + g * (kGroupRows * DT * 2) + (chunk >> 3) * S::kHalf;
#pragma unroll 2
        for (int r = row / kChunks; r < kGroupRows; r += kGroupRows / kChunks) {
          const long long off = row_offset[r];
          const bool fill = off >= 0 && chunk * 8 < a.head_dim;
          copy16(q_to + r * 128 + (((chunk ^ r) & 7) << 4), (const T*)a.q + (fill ? off + chunk * 8 : 0), fill);
        }
        copy_commit();
        copy_wait<0>();
        fence_proxy_async();
        mbar_arrive(&q_full[g]);
      }

      constexpr float kHighest = std::is_same<T, __half>::value ? kLift : kSlack;  // of a score over m
      float m = -INFINITY, l = 0.0f;  // m: what is taken off the scores
      const int steps = !alternate ? 2 * count : g == 0 ? (count + 1) / 2 * 2 : count / 2 * 2;
      for (int u = 0; u < steps; ++u, ++step) {
        const int buffer = step & 1, tile = tile0 + (alternate ? (u & ~1) + g : u >> 1);
        const unsigned at = s_at + buffer * kStep;
        wait_quick(&s_full[g * 2 + buffer], (step >> 1) & 1, dead);
        tc_fence_after();
        unsigned s[2][32];
        tmem_load32(at, s[0]);
        tmem_load32(at + 32, s[1]);
        tmem_wait_load(s[0]);
        tmem_wait_load(s[1]);
        const int seen = a.prefix - tile * kPrefixTile;  // positions of the tile: whole boxes
        if (seen < kPrefixTile) {
#pragma unroll
          for (int e = 0; e < kStep; e += 8) {
            const int pos = p.rows_log == 4 ? 2 * e : (u & 1) * kStep + e;  // of the group's box
#pragma unroll
            for (int k = e; k < e + 8; ++k)
              if (pos >= seen) s[k >> 5][k & 31] = __float_as_uint(-INFINITY);
          }
        }
        float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int e = 0; e < kStep; e += 2)
          top[(e >> 1) & 3] = max3(top[(e >> 1) & 3], __uint_as_float(s[e >> 5][e & 31]), __uint_as_float(s[e >> 5][(e & 31) + 1]));
        const float most = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * a.scale_log2;
        if (u == 0) {
          m = weights_from<T>(most, kPrefixLift);
        } else if (__any_sync(0xffffffffu, most > m + kHighest)) {
          const float rise = fmaxf(m, weights_from<T>(most, kPrefixLift)), down = exp2_fast(m - (rise == -INFINITY ? 0.0f : rise));
          m = rise;
          l *= down;
          // The last step's product has reached O (the one before it had, or these scores would not be there).
          wait_or_give_up(&o_full[g * 2 + (buffer ^ 1)], (step - 1) >> 1 & 1, dead);
          tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < DT; c += 32) {
            unsigned o[32];
            tmem_load32(o_at + c, o);
            tmem_wait_load(o);
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * down);
            tmem_store32(o_at + c, o);
          }
        }
        const float ref = m == -INFINITY ? 0.0f : m;
        const float2 scale2 = make_float2(a.scale_log2, a.scale_log2), ref2 = make_float2(-ref, -ref);
        float2 sum[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
        unsigned w16[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          const float2 pair = make_float2(__uint_as_float(s[e >> 4][2 * (e & 15)]), __uint_as_float(s[e >> 4][2 * (e & 15) + 1]));
          float2 x = __ffma2_rn(pair, scale2, ref2);
          x.x = exp2_fast(x.x);
          x.y = exp2_fast(x.y);
          sum[e & 1] = __fadd2_rn(sum[e & 1], x);
          w16[e] = pack2(x.x, x.y, T{});
        }
        tmem_store32(at, w16);
        sum[0] = __fadd2_rn(sum[0], sum[1]);
        l += sum[0].x + sum[0].y;
        tmem_wait_store();
        tc_fence_before();
        mbar_arrive(&p_full[g * 2 + buffer]);
      }

      // The piece: this thread's row of it.
      if (any) {
        wait_or_give_up(&o_full[g * 2 + ((step - 1) & 1)], (step - 1) >> 1 & 1, dead);
        tc_fence_after();
      }
      const long long slot = ((long long)unit + blockIdx.x) * 2 + g;
      // The queries are used up: a quarter of their bytes takes a warp's 32 rows, half of the columns at a time, so that
      // whole rows go out.
      constexpr int kCols = DT / 2, kParts = kCols / 4;  // columns at a time, 16-byte chunks of them
      const unsigned stage = smem_at + g * (kGroupRows * DT * 2) + (warp & 3) * (32 * kCols * 4);
      const int row_first = (warp & 3) * 32, rows = a.batch * a.rows - (row0 + row_first);
#pragma unroll 1
      for (int c0 = 0; c0 < DT; c0 += kCols) {
#pragma unroll 1
        for (int c = 0; c < kCols; c += 32) {
          unsigned o[32];
          tmem_load32(o_at + c0 + c, o);
          tmem_wait_load(o);
#pragma unroll
          for (int e = 0; e < 32; e += 4)
            asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(
                             stage + lane * (kCols * 4) + ((((c + e) >> 2) ^ (lane & (kParts - 1))) << 4)),
                         "r"(any ? o[e] : 0u), "r"(any ? o[e + 1] : 0u), "r"(any ? o[e + 2] : 0u), "r"(any ? o[e + 3] : 0u)
                         : "memory");
        }
        __syncwarp();
        float* dst = a.part + (slot * kGroupRows + row_first) * a.head_dim;
        const int chunk = lane & (kParts - 1), c = c0 + chunk * 4;
#pragma unroll 4
        for (int r = lane / kParts; r < 32; r += 32 / kParts) {
          uint4 v;
          asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                       : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                       : "r"(stage + r * (kCols * 4) + ((chunk ^ (r & (kParts - 1))) << 4)));
          if (r < rows && c < a.head_dim) *reinterpret_cast<uint4*>(dst + (long long)r * a.head_dim + c) = v;
        }
        __syncwarp();
      }
      if (lane < rows) a.ml[slot * kGroupRows + row] = make_float2(m, l);
      tc_fence_before();  // the next piece's products may overwrite O_g once its queries are announced
      w += count;
    }
  }
  settle(dead);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 9) tmem_free(tmem, 512);
}

}  // namespace
}  // namespace ckb
