// What the attention kernels of the paged episode cache share: which share of the work a block takes,
// which keys its rows see, the tensor maps of the pages, and the join of the parts of a split tile.
#pragma once
#include <stdint.h>
#include <cuda_runtime.h>

#include "mkx_cache.h"
#include "mkx_device.cuh"
#include "mkx_half.cuh"
#include "mkx_tma.cuh"

namespace mkxa {
using namespace mkx;

struct AttendParams {
  const void* q;
  void* out;
  const int *table, *length, *start;
  unsigned* tickets;  // [MKX_ATTEND_TICKETS], zero between calls
  float* parts;       // [max_parts][tile rows][HD + 2]: unnormalised sums, then (maximum, total)
  int* error;
  long long q_row, q_head, o_row, o_head;
  int rows, B, heads, kv_heads, group, pages, shift, table_width, max_rows;
  int causal, window, sinks;
  float scale_log2;       // |scale| * log2(e): scores are kept in powers of two
  uint32_t q_and, q_xor;  // q's words as they enter: the sign of a negative scale, nothing for scale 0
  int slots;         // blocks that the call's work is meant to be spread over
  int min_blocks;    // key blocks that a part has at least
  int max_parts;
  unsigned long long timeout_ns;
};

// One block's share: part `split` of `splits` of the key blocks of row tile `tile` of (episode, head).
struct Share {
  int b, kvh, tile, split, splits;
  int first_row, fresh, length, past;  // of the episode: row of q, new rows, rows held, position of row 0
  int part, ticket;                    // of the tile (splits > 1)
};

__device__ __forceinline__ int ceil_div(int a, int b) { return (a + b - 1) / b; }

struct Episode {
  int first_row, fresh, length, past, tiles, blocks;
};

// An episode's new rows, row tiles (MT rows of (new row, head of the group)) and the most key blocks
// (KT keys) that one of its tiles sees.
template <int MT, int KT>
__device__ __forceinline__ Episode episode_of(const AttendParams& p, int b) {
  Episode e;
  e.first_row = p.start[b];
  const int next = p.start[b + 1];
  e.length = max(p.length[b], 0);
  e.past = e.length - max(next - e.first_row, 0);
  e.fresh = (e.first_row < 0 || next > p.rows) ? 0 : min(max(next - e.first_row, 0), p.max_rows);
  e.tiles = (int)(((long long)e.fresh * p.group + MT - 1) / MT);
  const long long keys = min((long long)e.length, (long long)p.table_width << p.shift);
  long long blocks = (keys + KT - 1) / KT;
  if (p.window) {
    const long long span = (long long)p.window + min(e.fresh, MT / p.group + 2);
    blocks = min(blocks, (span + KT - 1) / KT + 1 + ((long long)p.sinks + KT - 1) / KT);
  }
  e.blocks = (int)max(blocks, 1ll);
  return e;
}

// Every block works out its share by itself from the B lengths. The work is cut into parts of at most
// `cut` key blocks, cut = all key blocks of all tiles / slots, so that a call with few tiles (single rows,
// few heads) still fills the GPU, and one with many is not split at all. Splits are the same for all
// tiles of an episode: a part is found by a prefix over the episodes.
// NTH threads, all call. Returns false if there is no share left for this block.
template <int MT, int KT, int NTH>
__device__ __forceinline__ bool find_share(const AttendParams& p, long long item, Share& out) {
  constexpr int W = NTH / 32;
  __shared__ long long sums[W];
  __shared__ int3 warp_sums[W];
  __shared__ Share found;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  long long all = 0;
  for (int b = threadIdx.x; b < p.B; b += NTH) {
    const Episode e = episode_of<MT, KT>(p, b);
    all += (long long)e.tiles * p.kv_heads * e.blocks;
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) all += __shfl_xor_sync(0xffffffffu, all, d);
  if (lane == 0) sums[warp] = all;
  if (threadIdx.x == 0) found.b = -1;
  __syncthreads();
  all = 0;
#pragma unroll
  for (int w = 0; w < W; ++w) all += sums[w];
  const int cut = (int)max((long long)p.min_blocks, (all + p.slots - 1) / p.slots);
  int3 before = make_int3(0, 0, 0);  // items, parts of split tiles, split tiles of earlier episodes
  for (int b0 = 0; b0 < p.B; b0 += NTH) {
    const int b = b0 + threadIdx.x;
    Episode e;
    e.tiles = 0;
    int splits = 1;
    int3 v = make_int3(0, 0, 0);
    if (b < p.B) {
      e = episode_of<MT, KT>(p, b);
      splits = ceil_div(e.blocks, cut);
      v.x = e.tiles * p.kv_heads * splits;
      if (splits > 1) {
        v.y = v.x;
        v.z = e.tiles * p.kv_heads;
      }
    }
    int3 inc = v;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, inc.x, d), y = __shfl_up_sync(0xffffffffu, inc.y, d),
                z = __shfl_up_sync(0xffffffffu, inc.z, d);
      if (lane >= d) {
        inc.x += x;
        inc.y += y;
        inc.z += z;
      }
    }
    if (lane == 31) warp_sums[warp] = inc;
    __syncthreads();
    int3 base = before;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const int3 s = warp_sums[w];
      if (w < warp) {
        base.x += s.x;
        base.y += s.y;
        base.z += s.z;
      }
      before.x += s.x;
      before.y += s.y;
      before.z += s.z;
    }
    const int mine = base.x + inc.x - v.x;
    if (item >= mine && item < mine + v.x) {
      const int local = (int)(item - mine);
      Share s;
      s.b = b;
      s.kvh = local % p.kv_heads;
      const int rest = local / p.kv_heads;
      s.split = rest % splits;
      s.tile = rest / splits;
      s.splits = splits;
      s.first_row = e.first_row;
      s.fresh = e.fresh;
      s.length = e.length;
      s.past = e.past;
      const int t = s.tile * p.kv_heads + s.kvh;
      s.part = base.y + inc.y - v.y + t * splits;
      s.ticket = base.z + inc.z - v.z + t;
      found = s;
    }
    __syncthreads();
    if (before.x > item) break;
  }
  out = found;
  // (a `start` that is no prefix could ask for more parts than there are: those tiles stay unwritten)
  return out.b >= 0 && (out.splits == 1 || ((unsigned)(out.part + out.splits) <= (unsigned)p.max_parts &&
                                            (unsigned)out.ticket < MKX_ATTEND_TICKETS));
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
__device__ __forceinline__ Keys keys_of(const AttendParams& p, const Share& s, int r0, int r1) {
  Keys k;
  k.p_first = s.past + r0 / p.group;
  k.p_last = s.past + r1 / p.group;
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

// 4D tiled load (dims, rows, heads, pages); a page of -1 reads as zero. x a multiple of 8.
__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* map, int x, int row, int head, int page,
                                            uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::
          "r"(smem_u32(dst)),
      "l"(map), "r"(x), "r"(row), "r"(head), "r"(page), "r"(smem_u32(bar))
      : "memory");
}

__device__ __forceinline__ bool wait_bounded(uint64_t* bar, uint32_t parity, unsigned long long limit) {
  if (mbar_try_wait(bar, parity)) return true;
  const uint64_t t0 = globaltimer();
  while (!mbar_try_wait(bar, parity))
    if (globaltimer() - t0 > limit) return false;
  return true;
}

}  // namespace mkxa
