// Own tokens, with the cache's tiles brought by TMA (included by attention.cu, whose parts it uses).
//
// The same axis of tiles, pieces and joins as attend_tiles. What bounds this work is the cache's bytes, and what kept
// attend_tiles from their rate was instructions: 128 threads spent two thirds of them on addresses and copies of 16 bytes,
// and a block barrier per tile held the warps in step (48 sequences of up to 16001 tokens: 389 us, 4.1 TB/s). Here one
// warp looks the pages up and issues a TMA box for each page and 64 columns, and the four others only multiply; each
// goes on as soon as a tile has arrived (mbarriers), whatever the others do: 254 us, 6.2 TB/s or 0.96 of the measured copy
// bandwidth. With short sequences the 2.5 us before a CTA's first tile, the 0.7 us at the end of each piece and half-filled
// last tiles show (256 sequences of 256 tokens on average: 4.3 TB/s).
//
// A box is one page (or a 64-row part of one) with all columns of a head, as blocks of 64 columns one after the other. Few
// large boxes matter: the TMA took about 70 clocks for each box of 16 rows and 64 columns, 2 KB, which held this kernel to
// 5.2 TB/s and the prefix's to 4 TB/s of L2. Heads of other than 64, 128 or 256 columns take a box for each block
// (the columns that they lack are filled up with zeros). The block size has to divide 64 or be a multiple of it, in steps of 8 rows (the
// swizzle's period); other block sizes, and caches of 2^31 rows, go through attend_tiles.
#pragma once

#include <cuda.h>

namespace ckb {
namespace {

__device__ unsigned int g_attention_status = 0u;

__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// Arrives on bar when this thread's earlier cp.async copies are done (one of the expected arrivals).
__device__ __forceinline__ void mbar_arrive_copies(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tma_load4(unsigned dst, const CUtensorMap* map, int x, int row, int head, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(
          dst),
      "l"(map), "r"(smem_u32(bar)), "r"(x), "r"(row), "r"(0), "r"(head)
      : "memory");
}
__device__ __forceinline__ bool elect_one() {
  unsigned is;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(is));
  return is != 0u;
}
__device__ __forceinline__ void tma_prefetch(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}
// Waits for a phase unless an earlier wait of this thread ran out: then the kernel runs on to its end without waiting
// (its results are void, the status says so).
__device__ __forceinline__ void wait_or_give_up(uint64_t* bar, unsigned parity, bool& dead) {
  if (dead) return;
  if (!mbar_wait(bar, parity)) {
    dead = true;
    atomicOr(&g_attention_status, CKB_STATUS_TIMEOUT);
  }
}
// Before a CTA that gave up ends: 10 ms for the copies and products that it may have in flight.
__device__ __forceinline__ void settle(bool dead) {
  if (!dead) return;
#pragma unroll 1
  for (int i = 0; i < 100; ++i) __nanosleep(100000);
}
__device__ __forceinline__ void sync_warps(int id, int threads) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory"); }

// A tile in shared memory: boxes of R = 2^rows_log rows, each DT / 64 blocks of [R][128 bytes], 16-byte chunks exchanged
// within 128 bytes as the TMA's 128-byte swizzle does. Byte offset of chunk c (of the whole row) of row r: row_part + chunk_part.
template <int DT>
__device__ __forceinline__ unsigned row_part(int r, int rows_log) {
  return (((r >> rows_log) * (DT / 64) << rows_log) + (r & ((1 << rows_log) - 1))) * 128;
}
__device__ __forceinline__ unsigned chunk_part(int r, int c, int rows_log) {
  return ((c >> 3) << rows_log) * 128 + (((c ^ r) & 7) << 4);
}
template <int DT>
__device__ __forceinline__ unsigned at_box(int r, int c, int rows_log) {
  return row_part<DT>(r, rows_log) + chunk_part(r, c, rows_log);
}
// Whether any value of rows row0 .. row0 + kCount - 1 of such a tile is infinite or NaN (the whole warp asks).
template <typename T, int DT, int kCount>
__device__ __forceinline__ bool not_finite_box(unsigned tile, int row0, int lane, int rows_log) {
  bool bad = false;
  for (int i = lane; i < kCount * (DT / 2); i += 32) {
    const int r = i / (DT / 2), w = i % (DT / 2);
    const float2 v = load2(tile + at_box<DT>(row0 + r, w >> 2, rows_log) + (w & 3) * 4, T{});
    bad |= !(fabsf(v.x) < INFINITY) || !(fabsf(v.y) < INFINITY);
  }
  return __any_sync(0xffffffffu, bad);
}

constexpr int kConsumers = 4;  // warps that multiply; one more loads

template <int DT, int WR>
struct Ring {
  static constexpr int kRows = 16 * WR;
  static constexpr int kKeyWarps = 4 / WR;
  static constexpr int kKeys = kTile / kKeyWarps;
  static constexpr int kStages = WR == 1 && DT <= 64 ? 3 : 2;
  static constexpr int kTileBytes = kTile * DT * 2;
  static constexpr int kQBytes = kRows * DT * 2;
  static constexpr int kOffQ = kStages * 2 * kTileBytes;
  static constexpr int kOffMl = kOffQ + kStages * kQBytes;
  static constexpr int kOffBars = kOffMl + kKeyWarps * kRows * 8;
  static constexpr int kOffCum = kOffBars + 2 * kStages * 8;
  static constexpr int bytes(int batch) { return kOffCum + (2 * batch + 1) * 4; }
  // CTAs of an SM by registers (with two stages of 32 KB each three CTAs keep as many bytes in flight as two with three
  // stages, and 12 warps multiply instead of 8: 64 sequences behind 4096 tokens 45.6 -> 42.0 us, 48 ragged ones 259 -> 252;
  // one of 8192 tokens, whose CTAs have an SM for themselves, 11.9 -> 13.1). Of heads of 64 columns four, with up to 32 rows; 64
  // rows spill at the 96 registers of four (32 sequences of 16 tokens, 4 heads a key head, behind 1024 tokens 93 us, with three 69 us; 48
  // ragged ones without a prefix 158 and 151 us).
  static constexpr int kPerSm = DT <= 64 ? (WR == 4 ? 3 : 4) : DT <= 128 ? (WR == 1 ? 3 : 2) : 1;
  // ... and by shared memory, of which the system takes 1 KB for each.
  static int per_sm(int batch) {
    const int fit = kSmShared / (bytes(batch) + 1024);
    return fit < 1 ? 1 : fit < kPerSm ? fit : kPerSm;
  }
};

// The bound matters: at the compiler's own 127 registers for heads of 64 columns three CTAs fitted an SM and the fourth came
// after them (18 x 5 tokens behind 1536 took 21.9 us instead of 17.8 us).
template <typename T, int DT, int WR>
__global__ void __launch_bounds__(32 * (kConsumers + 1), Ring<DT, WR>::kPerSm)
    attend_stream(const Args a, int rows_log, const __grid_constant__ CUtensorMap key_map, const __grid_constant__ CUtensorMap value_map) {
  using S = Ring<DT, WR>;
  constexpr int kRows = S::kRows, kKeys = S::kKeys, kStages = S::kStages;
  constexpr int kAll = 32 * (kConsumers + 1);
  extern __shared__ __align__(1024) unsigned char tiles[];  // 1024: the swizzle's period
  unsigned char* smem = tiles;
  float2* ml_sh = reinterpret_cast<float2*>(smem + S::kOffMl);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + S::kOffBars);
  uint64_t* empty = full + kStages;
  int* cum = reinterpret_cast<int*>(smem + S::kOffCum);
  int* lens = cum + a.batch + 1;
  const unsigned smem_at = smem_u32(smem);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&full[i], 33);  // every lane of the loading warp, and its announcement of the bytes
      mbar_init(&empty[i], kConsumers);
    }
    mbar_fence_init();
    tma_prefetch(&key_map);
    tma_prefetch(&value_map);
  }
  if (!a.beside) pdl_wait();
  pdl_trigger();
  const int units = a.kv_heads * a.row_tiles;
  own_axis<kAll>(a, units, cum, lens, reinterpret_cast<int*>(ml_sh));  // its barriers order the mbarriers' set-up too
  const int all = cum[a.batch];
  const Runs runs = runs_of(a, all, gridDim.x);
  if (blockIdx.x == 0) write_plan<kAll>(a, cum, runs);
  const int first = runs.begin(blockIdx.x, all), last = runs.begin(blockIdx.x + 1, all);
  // The first CTA, which always has a loading warp, ends after the shared work.
  if (first >= last) {
    if (a.beside && blockIdx.x == 0) pdl_wait();
    return;
  }
  Cursor at = axis_start(cum, a.batch, units, first);
  bool dead = false;

  if (warp == kConsumers) {
    // Pages of a tile: box_rows rows each, in `blocks` boxes.
    const int box_rows = 1 << rows_log, pages = kTile >> rows_log, blocks = a.head_dim == DT ? 1 : DT / 64;
    const int page_bytes = box_rows * 128 * (DT / 64);
    const bool leader = elect_one();
    // Lane p looks up page p of a tile a tile ahead: the block's id is on its way while the tile before is copied, and only
    // then becomes the cache row where the page begins.
    long long block_next = -1;
    int inside_next = 0;
    bool there_next = false;
    const auto look_up = [&](const Cursor& c) {
      const int len = lens[c.b], pos = own_begin(a.prefix, a.tokens, len) + c.tile * kTile + lane * box_rows;
      there_next = lane < pages && pos < len;
      if (!there_next) return;
      const int page = a.block_log >= 0 ? pos >> a.block_log : pos / a.block_size;
      inside_next = pos - page * a.block_size;
      block_next = load_list(a.tables + (long long)c.b * a.table_width + page);
    };
    int q_loads = 0, stage = 0, parity = 1;
    look_up(at);
    for (int w = first; w < last; ++w) {
      const int kv_head = a.row_tiles == 1 ? at.unit : at.unit / a.row_tiles;
      Cursor ahead = at;
      axis_next(cum, a.batch, units, ahead);
      // A block outside the cache lies outside the map: zeros.
      const int row_now = (int)(block_next < 0 || block_next >= a.num_blocks ? a.num_blocks * a.block_size
                                                                             : block_next * a.block_size + inside_next);
      const int there = __popc(__ballot_sync(0xffffffffu, there_next));  // the first pages
      if (w + 1 < last) look_up(ahead);
      wait_or_give_up(&empty[stage], parity, dead);
      if (dead) break;
      if (leader) mbar_arrive_expect_tx(&full[stage], there * 2 * page_bytes);
      const unsigned to = smem_at + stage * 2 * S::kTileBytes;
#pragma unroll 4
      for (int page = 0; page < there; ++page) {
        const int row = __shfl_sync(0xffffffffu, row_now, page);
        if (leader) {
          for (int block = 0; block < blocks; ++block) {
            const unsigned dst = to + page * page_bytes + block * (box_rows * 128);
            tma_load4(dst, &key_map, block * 64, row, kv_head, &full[stage]);
            tma_load4(dst + S::kTileBytes, &value_map, block * 64, row, kv_head, &full[stage]);
          }
        }
      }
      if (w == first || at.tile == 0) {  // a piece begins: its queries come with its first tile
        const int row0 = (at.unit - kv_head * a.row_tiles) * kRows;
        for (int i = lane; i < kRows * (DT / 8); i += 32) {
          const int r = i / (DT / 8), chunk = i % (DT / 8);
          const Row x = row_of<false>(a, at.b, kv_head, row0 + r);
          const bool fill = x.real && chunk * 8 < a.head_dim;
          const long long off = fill ? x.b * a.vq.batch + x.t * a.vq.token + x.head * a.vq.head + chunk * 8 : 0;
          copy16(smem_at + S::kOffQ + q_loads * S::kQBytes + at_chunk<DT>(r, chunk), (const T*)a.q + off, fill);
        }
        q_loads = q_loads + 1 == kStages ? 0 : q_loads + 1;
        mbar_arrive_copies(&full[stage]);
      } else {
        mbar_arrive(&full[stage]);
      }
      at = ahead;
      if (++stage == kStages) {
        stage = 0;
        parity ^= 1;
      }
    }
    copy_commit();
    copy_wait<0>();
    settle(dead);
    if (a.beside && blockIdx.x == 0) pdl_wait();
    return;
  }

  const int wr = warp % WR, wk = warp / WR, quad_row = lane >> 2;
  unsigned k_row[kKeys / 16], v_row[kKeys / 16];  // this lane's rows of the fragments
#pragma unroll
  for (int n = 0; n < kKeys / 16; ++n) {
    k_row[n] = row_part<DT>(wk * kKeys + n * 16 + (lane >> 4) * 8 + (lane & 7), rows_log);
    v_row[n] = row_part<DT>(wk * kKeys + n * 16 + (lane & 15), rows_log);
  }
  constexpr int kNt = kKeys / 8, kDt = DT / 8;
  constexpr bool kLifted = std::is_same<T, __half>::value;
  float o[kDt][4], m[2], l[2], from[2];  // from: weights_from of m, where that is another
  int len = 0, begin = 0, min_limit = 0, lim[2] = {0, 0}, q_now = -1, piece_begin = 0, stage = 0, parity = 0;
  for (int w = first; w < last; ++w) {
    const int kv_head = a.row_tiles == 1 ? at.unit : at.unit / a.row_tiles, row0 = (at.unit - kv_head * a.row_tiles) * kRows;
    if (w == first || at.tile == 0) {  // a new piece
      q_now = q_now + 1 == kStages ? 0 : q_now + 1;
      piece_begin = at.tile;
      len = lens[at.b];
      begin = own_begin(a.prefix, a.tokens, len);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int in = row0 + wr * 16 + quad_row + 8 * i;
        lim[i] = in < a.rows ? max(0, len - a.tokens + in / a.group + 1) : INT_MAX;  // padding: any finite result
        m[i] = -INFINITY;
        if constexpr (kLifted) from[i] = -INFINITY;
        l[i] = 0.0f;
      }
      min_limit = __reduce_min_sync(0xffffffffu, min(lim[0], lim[1]));
#pragma unroll
      for (int n = 0; n < kDt; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[n][e] = 0.0f;
    }
    wait_or_give_up(&full[stage], parity, dead);

    const unsigned k_at = smem_at + stage * 2 * S::kTileBytes, v_at = k_at + S::kTileBytes;
    const unsigned q_at = smem_at + S::kOffQ + q_now * S::kQBytes;
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
        ldsm4(kb, k_at + k_row[n / 2] + chunk_part(lane & 7, 2 * k + ((lane >> 3) & 1), rows_log));
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
    float top[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      top[i] = m[i];
#pragma unroll
      for (int n = 0; n < kNt; ++n) top[i] = fmaxf(top[i], fmaxf(s[n][2 * i], s[n][2 * i + 1]) * a.scale_log2);
      top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 1));
      top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 2));
    }
    if (__any_sync(0xffffffffu, top[0] > m[0] || top[1] > m[1])) {  // a new maximum: rarer and rarer along the tiles
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float next = weights_from<T>(top[i], kLift);
        const float scale = exp2_fast((kLifted ? from[i] : m[i]) - (next == -INFINITY ? 0.0f : next));
        m[i] = top[i];
        if constexpr (kLifted) from[i] = next;
        l[i] *= scale;
#pragma unroll
        for (int n = 0; n < kDt; ++n) {
          o[n][2 * i] *= scale;
          o[n][2 * i + 1] *= scale;
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float ref = m[i] == -INFINITY ? 0.0f : kLifted ? from[i] : m[i];  // a row that has seen nothing yet: exp2(-inf - 0) = 0
      float sum = 0.0f;
#pragma unroll
      for (int n = 0; n < kNt; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float p = exp2_fast(fmaf(s[n][2 * i + e], a.scale_log2, -ref));
          s[n][2 * i + e] = p;
          sum += p;
        }
      l[i] += sum;
    }
    if (pos0 + kKeys > len) {  // what lies behind the sequence in its last page is anything: 0 * v must be 0
      for (int i = lane; i < kKeys * (DT / 8); i += 32) {
        const int r = i / (DT / 8);
        if (pos0 + r >= len)
          asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(v_at + at_box<DT>(wk * kKeys + r, i % (DT / 8), rows_log)), "r"(0u)
                       : "memory");
      }
      __syncwarp();
      fence_proxy_async();  // before the ring's next copy into these bytes
    }
    if (masked && a.tokens > 1 && not_finite_box<T, DT, kKeys>(v_at, wk * kKeys, lane, rows_log)) {
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
            const float2 v = load2(v_at + at_box<DT>(wk * kKeys + key, c, rows_log) + (lane & 3) * 4, T{});
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
    } else {
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
          ldsm4_trans(vb, v_at + v_row[k] + chunk_part(lane & 7, n + (lane >> 4), rows_log));
          mma(o[n], pa, vb[0], vb[1], T{});
          mma(o[n + 1], pa, vb[2], vb[3], T{});
        }
      }
    }

    if (at.tile + 1 == at.tiles || w + 1 == last) {  // the end of a piece
      const bool whole = begin == 0 && piece_begin == 0 && at.tile + 1 == at.tiles;
      const long long slot = (long long)at.b * units + at.unit + blockIdx.x;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
        if constexpr (kLifted) m[i] = from[i];
      }
      if (S::kKeyWarps == 1) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
          write_row<T, DT>(a, row_of<false>(a, at.b, kv_head, row0 + wr * 16 + quad_row + 8 * i), whole, lim[i] > 0,
                           slot * kRows + wr * 16 + quad_row + 8 * i, lane, o, i, m[i], l[i]);
      } else {
        // The warps that shared the positions leave their sums in the tile's own stage, and all 128 threads join them,
        // 4 columns each: two barriers (adding up one warp after the other took 2.6 us a piece, this takes 0.5).
        sync_warps(1, 32 * kConsumers);  // nobody reads the tile any more
        float* sums = reinterpret_cast<float*>(smem + stage * 2 * S::kTileBytes);  // [key warps][rows][DT]
        const int real = min(kRows, a.rows - row0);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int r = wr * 16 + quad_row + 8 * i;
          if (r < real) {
            float* dst = sums + (wk * kRows + r) * DT + (lane & 3) * 2;
#pragma unroll
            for (int n = 0; n < kDt; ++n)  // pairs exchanged among the rows' tiles of 8 columns: no bank twice
              *reinterpret_cast<float2*>(dst + ((n ^ (r & 7)) * 8)) = make_float2(o[n][2 * i], o[n][2 * i + 1]);
            if ((lane & 3) == 0) ml_sh[wk * kRows + r] = make_float2(m[i], l[i]);
          }
        }
        sync_warps(1, 32 * kConsumers);
        for (int e = tid; e < real * (DT / 4); e += 32 * kConsumers) {
          const int r = e / (DT / 4), c = (e - r * (DT / 4)) * 4;
          float most = -INFINITY, sum = 0.0f;
#pragma unroll
          for (int k = 0; k < S::kKeyWarps; ++k) most = fmaxf(most, ml_sh[k * kRows + r].x);
          const float ref = most == -INFINITY ? 0.0f : most;
          float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
          for (int k = 0; k < S::kKeyWarps; ++k) {
            const float2 v = ml_sh[k * kRows + r];
            const float weight = exp2_fast(v.x - ref);
            sum = fmaf(v.y, weight, sum);
            const float4 u = *reinterpret_cast<const float4*>(sums + (k * kRows + r) * DT + (((c >> 3) ^ (r & 7)) << 3) + (c & 7));
            acc.x = fmaf(weight, u.x, acc.x);
            acc.y = fmaf(weight, u.y, acc.y);
            acc.z = fmaf(weight, u.z, acc.z);
            acc.w = fmaf(weight, u.w, acc.w);
          }
          if (c >= a.head_dim) continue;
          if (whole) {
            const Row x = row_of<false>(a, at.b, kv_head, row0 + r);
            const bool some = len - a.tokens + x.t + 1 > 0;
            const float inv = 1.0f / sum;
            T* dst = (T*)a.out + (((long long)x.b * a.tokens + x.t) * a.q_heads + x.head) * a.head_dim + c;
            *reinterpret_cast<uint2*>(dst) = some ? make_uint2(pack2(acc.x * inv, acc.y * inv, T{}), pack2(acc.z * inv, acc.w * inv, T{}))
                                                  : make_uint2(0u, 0u);
          } else {
            *reinterpret_cast<float4*>(a.part + (slot * kRows + r) * a.head_dim + c) = acc;
            if (c == 0) a.ml[slot * kRows + r] = make_float2(most, sum);
          }
        }
        fence_proxy_async();
      }
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(&empty[stage]);
    axis_next(cum, a.batch, units, at);
    if (++stage == kStages) {
      stage = 0;
      parity ^= 1;
    }
  }
  settle(dead);
}

}  // namespace
}  // namespace ckb
