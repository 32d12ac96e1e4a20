// What the attention kernels of the paged episode cache share: which stretch of the work a block takes,
// which keys its rows see, and the exchange between blocks that share a tile.
#pragma once
#include <stdint.h>
#include <cuda_runtime.h>

#include "mkx_cache.h"
#include "mkx_device.cuh"
#include "mkx_half.cuh"
#include "mkx_join.h"
#include "mkx_tma.cuh"

namespace mkxa {
using namespace mkx;

struct AttendParams {
  const void* q;
  void* out;
  const int *table, *length, *start;
  unsigned* tickets;  // [MKX_ATTEND_TICKETS], zero between calls
  float* parts;       // [2 slots][tile rows x (HD + 2)]: unnormalised sums, then (maximum, total) of each row
  int* error;
  long long q_row, q_head, o_row, o_head;
  int rows, B, heads, kv_heads, group, group_shift, pages, shift, table_width, max_rows;  // group_shift: log2, or -1
  int causal, window, sinks;
  float scale_log2;       // |scale| * log2(e): scores are kept in powers of two
  uint32_t q_and, q_xor;  // q's words as they enter: the sign of a negative scale, nothing for scale 0
  int slots;      // blocks of the grid
  int min_shift;  // log2 of the key blocks that one block takes at least
  int snap;       // units by which a cut may move to a tile's end
  unsigned long long timeout_ns;
};

__device__ __forceinline__ int ceil_div(int a, int b) { return (a + b - 1) / b; }
__device__ __forceinline__ int by_group(const AttendParams& p, int r) {
  return p.group_shift >= 0 ? r >> p.group_shift : r / p.group;
}
// Quotients of what is nearly always below 2^32: a 64-bit division is a few hundred clocks, at every block's start.
__device__ __forceinline__ long long quotient(long long a, int b) {
  return (unsigned long long)a >> 32 ? a / b : (long long)((unsigned)a / (unsigned)b);
}

// An episode's new rows, its row tiles (MT rows of (new row, head of the group)) and the most key blocks
// (KT keys) that one of its tiles sees.
struct Episode {
  int first_row, fresh, length, past, tiles, units;
};

template <int MT, int KT>
__device__ __forceinline__ Episode episode_from(const AttendParams& p, int first_row, int next, int length) {
  Episode e;
  e.first_row = first_row;
  e.length = max(length, 0);
  e.past = e.length - max(next - first_row, 0);
  e.fresh = (first_row < 0 || next > p.rows) ? 0 : min(max(next - first_row, 0), p.max_rows);
  e.tiles = (int)(((long long)e.fresh * p.group + MT - 1) / MT);
  const long long keys = min((long long)e.length, (long long)p.table_width << p.shift);
  long long blocks = (keys + KT - 1) / KT;
  if (p.window) {
    const long long span = (long long)p.window + min(e.fresh, MT / p.group + 2);
    blocks = min(blocks, (span + KT - 1) / KT + 1 + ((long long)p.sinks + KT - 1) / KT);
  }
  e.units = (int)max(blocks, 1ll);
  return e;
}
template <int MT, int KT>
__device__ __forceinline__ Episode episode_of(const AttendParams& p, int b) {
  return episode_from<MT, KT>(p, p.start[b], p.start[b + 1], p.length[b]);
}

// The work of a call is a line of units, one for each key block of each row tile, K/V head and episode.
// Block c of the grid takes the units from cut c to cut c + 1; the cuts divide the line evenly, but one
// within `snap` units of a tile's end moves there, because a tile in two parts has to be joined, which
// costs about as much as that many units. So tiles of any lengths fill the GPU evenly, short ones stay
// whole, and a long one alone is spread over all blocks. The last block of a tile to finish joins its
// parts. Each role of a block walks the line by itself: no exchange, and the copies run ahead of the
// arithmetic across tiles.
struct Segment {
  int b, kvh, tile;
  int first_row, fresh, length, past;  // of the episode
  int v0, v1, units;                   // units of the tile taken here
  int lead, parts;                     // first block of the tile, number of blocks (parts > 1: to be joined)
};

struct Line {
  long long total, at, begin, end;  // units; first unit of the episode that the stretch begins in; the stretch
  int blocks, b;                    // blocks that the line is cut for; that episode
  Episode e;
};

__device__ __forceinline__ long long snapped(long long u, long long at, int units, int snap) {
  const int v = (int)(u - at - quotient(u - at, units) * units);
  return v <= snap ? u - v : units - v <= snap ? u + (units - v) : u;
}

// All threads of the block call this; false if the block has nothing to do. The scratch is free again after the next
// block barrier.
struct LineScratch {
  long long sums[2][32];
  Line line;
};

// What the thread of episode b (units at .. at + mine - 1) knows of the block's stretch.
__device__ __forceinline__ void cut_line(const AttendParams& p, Line& line, const Episode& e, int b, long long at,
                                         long long mine, long long all, int blocks) {
  const long long u0 = quotient(all * blockIdx.x, blocks), u1 = quotient(all * (blockIdx.x + 1), blocks);
  if (u0 >= at && u0 < at + mine) {
    line.total = all;
    line.at = at;
    line.begin = snapped(u0, at, e.units, p.snap);
    line.blocks = blocks;
    line.b = b;
    line.e = e;
  }
  if (u1 >= at && u1 < at + mine) line.end = snapped(u1, at, e.units, p.snap);
}

template <int MT, int KT, int NTH>
__device__ __forceinline__ bool find_line(const AttendParams& p, LineScratch& scratch, Line& out) {
  constexpr int W = NTH / 32;
  auto& sums = scratch.sums;
  Line& line = scratch.line;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  auto prefix = [&](long long mine) {  // inclusive, over the warp
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const long long o = __shfl_up_sync(0xffffffffu, mine, d);
      if (lane >= d) mine += o;
    }
    return mine;
  };
  auto blocks_of = [&](long long all) { return (int)min((long long)p.slots, (all >> p.min_shift) + 1); };
  if (p.B <= 32) {  // one warp does it, between one pair of barriers less
    if (warp == 0) {
      Episode e;
      long long mine = 0;
      if (lane < p.B) {
        e = episode_of<MT, KT>(p, lane);
        mine = (long long)e.tiles * p.kv_heads * e.units;
      }
      const long long inc = prefix(mine), all = __shfl_sync(0xffffffffu, inc, 31);
      const int blocks = blocks_of(all);
      if (lane == 0) line.begin = line.end = (int)blockIdx.x < blocks ? all : 0;
      __syncwarp();
      if ((int)blockIdx.x < blocks) cut_line(p, line, e, lane, inc - mine, mine, all, blocks);
    }
    __syncthreads();
    out = line;
    return out.begin < out.end;
  }
  Episode e;
  long long all = 0, mine = 0;
  for (int b = threadIdx.x; b < p.B; b += NTH) {
    const Episode x = episode_of<MT, KT>(p, b);
    const long long units = (long long)x.tiles * p.kv_heads * x.units;
    all += units;
    if (b == (int)threadIdx.x) {
      e = x;
      mine = units;
    }
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) all += __shfl_xor_sync(0xffffffffu, all, d);
  if (lane == 0) sums[0][warp] = all;
  __syncthreads();
  all = 0;
#pragma unroll
  for (int w = 0; w < W; ++w) all += sums[0][w];
  const int blocks = blocks_of(all);
  if (all == 0 || (int)blockIdx.x >= blocks) return false;
  const long long u1 = quotient(all * (blockIdx.x + 1), blocks);
  if (threadIdx.x == 0) line.end = all;
  long long before = 0;
  for (int b0 = 0;; b0 += NTH) {
    const int b = b0 + threadIdx.x;
    if (b0 > 0) {
      mine = 0;
      if (b < p.B) {
        e = episode_of<MT, KT>(p, b);
        mine = (long long)e.tiles * p.kv_heads * e.units;
      }
    }
    const long long inc = prefix(mine);
    if (b0 > 0) __syncthreads();  // the sums have been read
    if (lane == 31) sums[1][warp] = inc;
    __syncthreads();
    long long at = before + inc - mine;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      if (w < warp) at += sums[1][w];
      before += sums[1][w];
    }
    cut_line(p, line, e, b, at, mine, all, blocks);
    if (before > u1 || before >= all) break;
  }
  __syncthreads();
  out = line;
  return out.begin < out.end;
}

template <int MT, int KT>
struct Walk {
  const AttendParams& p;
  long long total, left, tile_at;  // units of the line; units left of the stretch; first unit of the tile
  int blocks, b, kvh, tile, v;     // place: unit v of the tile
  Episode e;
  int n_first, n_next, n_length;   // of episode b + 1, asked for ahead

  __device__ __forceinline__ Walk(const AttendParams& params, const Line& l)
      : p(params), total(l.total), left(l.end - l.begin), blocks(l.blocks), b(l.b) {
    e = l.e;
    ask();
    // the stretch may begin behind the episode's last unit: then the first next() goes on
    const long long local = l.begin - l.at, t = quotient(local, e.units);
    v = (int)(local - t * e.units);
    tile_at = l.begin - v;
    kvh = (int)quotient(t, e.tiles);
    tile = e.tiles - 1 - (int)(t - (long long)kvh * e.tiles);
  }
  __device__ __forceinline__ void ask() {
    const int n = min(b + 1, p.B - 1);
    n_first = p.start[n];
    n_next = p.start[n + 1];
    n_length = p.length[n];
  }
  // The last block whose cut lies at or before `unit`.
  __device__ __forceinline__ int block_at(long long unit) const { 
    const long long a = (unit + 1) * blocks - 1;
    return (unsigned long long)(a | total) >> 32 ? (int)(a / total) : (int)((unsigned)a / (unsigned)total);
  }
  __device__ __forceinline__ bool next(Segment& s) {
    if (left <= 0) return false;
    while (kvh >= p.kv_heads || e.tiles == 0) {
      if (++b >= p.B) return false;
      e = episode_from<MT, KT>(p, n_first, n_next, n_length);
      ask();
      kvh = 0;
      tile = e.tiles - 1;
    }
    s.b = b;
    s.kvh = kvh;
    s.tile = tile;
    s.first_row = e.first_row;
    s.fresh = e.fresh;
    s.length = e.length;
    s.past = e.past;
    s.units = e.units;
    s.v0 = v;
    s.v1 = (int)min((long long)e.units, v + left);
    s.lead = blockIdx.x;
    s.parts = 1;
    if (s.v0 > 0 || s.v1 < s.units) {
      s.lead = block_at(tile_at + min(p.snap, s.units - 1));
      s.parts = block_at(tile_at + s.units - p.snap - 1) - s.lead + 1;
    }
    left -= s.v1 - s.v0;
    tile_at += s.units;
    v = 0;
    if (--tile < 0) {
      tile = e.tiles - 1;
      ++kvh;
    }
    return true;
  }
};

// A block keeps at most two parts: of the tile its stretch begins inside of, and of the one it ends inside of.
__device__ __forceinline__ int part_place(const Segment& s, int k) { return 2 * (s.lead + k) + (k == 0); }

// What the teams of both kernels share (see mkx_join.h).
struct TicketTeam {
  bool ok = true;
  __device__ __forceinline__ bool leads() const { return threadIdx.x == 0; }
  __device__ __forceinline__ bool read(const int* word) const { return *word != 0; }
  __device__ __forceinline__ void write(int* word, bool v) const { *word = v; }
  __device__ __forceinline__ unsigned held(const unsigned* ticket) const {
    return (unsigned)ld_acquire_i32(reinterpret_cast<const int*>(ticket));
  }
  __device__ __forceinline__ unsigned take(unsigned* ticket) const {
    unsigned before;
    asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;" : "=r"(before) : "l"(ticket) : "memory");
    return before;
  }
  __device__ __forceinline__ void clear(unsigned* ticket) const { *ticket = 0; }
};
// NTH threads that all walk the same line to its end, whatever runs out on the way: named barrier 1.
template <int NTH>
struct BarrierTeam : TicketTeam {
  __device__ __forceinline__ bool meet() const {
    asm volatile("bar.sync 1, %0;" ::"n"(NTH) : "memory");
    return true;
  }
};

// The key blocks of a segment, of `blocks` that its tile really has (its units are those of the episode's longest tile).
__device__ __forceinline__ int first_block(const Segment& s, int blocks) {
  return s.v0 == 0 ? 0 : (int)quotient((long long)blocks * s.v0, s.units);
}
__device__ __forceinline__ int end_block(const Segment& s, int blocks) {
  return s.v1 == s.units ? blocks : (int)quotient((long long)blocks * s.v1, s.units);
}

// The keys that the rows of a tile see: blocks of KT keys, first those of the sinks, then from the
// window's edge on. Positions are those of rows r0 .. r1 (inclusive) of the tile.
struct Keys {
  int lo, hi;         // keys lo .. hi - 1 are seen by some row, apart from sinks
  int lo_block;       // lo rounded down to a block
  int sink_blocks;    // blocks before lo_block that hold sinks
  int blocks;
  int p_first, p_last;
};

template <int KT>
__device__ __forceinline__ Keys keys_of(const AttendParams& p, const Segment& s, int r0, int r1) {
  Keys k;
  k.p_first = s.past + by_group(p, r0);
  k.p_last = s.past + by_group(p, r1);
  const int held = (int)min((long long)s.length, (long long)p.table_width << p.shift);
  k.hi = p.causal ? max(min(held, k.p_last + 1), 0) : held;
  k.lo = p.window ? min(max(k.p_first - p.window + 1, 0), k.hi) : 0;
  k.lo_block = k.lo / KT * KT;
  k.sink_blocks = p.window ? ceil_div(min(p.sinks, k.lo_block), KT) : 0;
  k.blocks = k.sink_blocks + ceil_div(k.hi - k.lo_block, KT);
  return k;
}
template <int KT>
__device__ __forceinline__ int block_key(const Keys& k, int i) {
  return i < k.sink_blocks ? i * KT : k.lo_block + (i - k.sink_blocks) * KT;
}
// Whether every row of the tile sees every key of the block.
template <int KT>
__device__ __forceinline__ bool whole_block(const AttendParams& p, const Keys& k, int key0) {
  if (key0 + KT > k.hi || (p.causal && key0 + KT - 1 > k.p_first)) return false;
  return !p.window || key0 > k.p_last - p.window || key0 + KT <= p.sinks;
}
// Bit d: whether a row at `position` sees key0 + d, d < 32.
__device__ __forceinline__ uint32_t below(int n) { return n >= 32 ? ~0u : n <= 0 ? 0u : (1u << n) - 1; }
__device__ __forceinline__ uint32_t seen_mask(const AttendParams& p, const Keys& k, int position, int key0) {
  uint32_t m = below((p.causal ? min(k.hi, position + 1) : k.hi) - key0);
  if (p.window) m &= ~below(position - p.window + 1 - key0) | below(p.sinks - key0);
  return m;
}
// Whether new row `row` of the call sees any key.
__device__ __noinline__ bool sees_any(const AttendParams& p, int row) {
  int b = 0, end = p.B;  // its episode: the last one that starts at or before it
  while (end - b > 1) {
    const int mid = (b + end) >> 1;
    if (p.start[mid] <= row) b = mid;
    else end = mid;
  }
  const int length = max(p.length[b], 0), position = length - p.start[b + 1] + row;
  const int held = (int)min((long long)length, (long long)p.table_width << p.shift);
  const int hi = p.causal ? min(held, position + 1) : held;
  return hi > 0 && (!p.window || hi > position - p.window + 1 || p.sinks > 0);
}
// What a row's sums are multiplied by, for the total `l` of its weights: zero where nothing is seen. No total although
// keys are seen means that all their scores are -inf: softmax has no value there, as for NaN or an infinite score. That
// is rare, so the row's episode and position are looked up again instead of being kept.
__device__ __forceinline__ float over_total(const AttendParams& p, int row, float l) {
  return l > 0.f ? 1.f / l : l == 0.f && !sees_any(p, row) ? 0.f : __int_as_float(0x7fffffff);
}
// The page that holds keys [page << shift, ..), or -1 (its rows read as zero) where no row sees any.
__device__ __forceinline__ int page_of(const AttendParams& p, const Keys& k, int b, int page) {
  const int first = page << p.shift;
  if (page >= p.table_width || first >= k.hi) return -1;
  if (first + (1 << p.shift) <= k.lo && first >= p.sinks) return -1;
  const int id = p.table[(size_t)b * p.table_width + page];
  return id >= 0 && id < p.pages ? id : -1;
}

__device__ __forceinline__ uint32_t signed_q(const AttendParams& p, uint32_t v) { return (v & p.q_and) ^ p.q_xor; }

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The maximum, NaN if one of them is.
__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
__device__ __forceinline__ float max_nan(float a, float b, float c) {
  float y;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}

// 4D tiled load (dims, rows, heads, pages); a page of -1 reads as zero. x a multiple of 8.
__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* map, int x, int row, int head, int page,
                                            uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::
          "r"(smem_u32(dst)),
      "l"(map), "r"(x), "r"(row), "r"(head), "r"(page), "r"(smem_u32(bar))
      : "memory");
}

__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ bool wait_bounded(uint64_t* bar, uint32_t parity, unsigned long long limit) {
  if (mbar_try_wait(bar, parity)) return true;
  const uint64_t t0 = globaltimer();
  while (!mbar_try_wait(bar, parity))
    if (globaltimer() - t0 > limit) return false;
  return true;
}

// Warps of which one may leave early, after a wait that ran out: an mbarrier that counts them, waited for with a limit.
// `met` says at which of its phases the warp is; none is ahead by more than one, since a phase needs them all.
struct BoundedTeam : TicketTeam {
  uint64_t* bar;
  unsigned long long limit;
  uint32_t met = 0;
  __device__ __forceinline__ BoundedTeam(uint64_t* barrier, unsigned long long timeout) : bar(barrier), limit(timeout) {}
  __device__ __forceinline__ bool meet() {
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
    ok = __all_sync(0xffffffffu, wait_bounded(bar, met & 1, limit)) != 0;
    ++met;
    return ok;
  }
};

}  // namespace mkxa
