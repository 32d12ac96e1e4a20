// Attention of new rows over the paged episode cache (include/mkx_cache.h), in one pass over the keys:
// with m the running maximum of a row's scores (in powers of two), l the sum of 2^(s - m) and o the sum
// of 2^(s - m) v, a larger maximum m' scales l and o by 2^(m - m'), and the row is o / l at the end; the
// same rule joins the parts of a row that different warps or blocks took. m, l, o are fp32 throughout.
// Two kernels, chosen by chunk_is_faster; the work of a call is one line of key blocks that the blocks of
// the grid share evenly, however many episodes of whatever lengths there are (find_line, Walk).
//
// rows_kernel: tiles of 16 rows (new row x head of the group that shares a K/V head). With few rows a
// call is bound by reading the pages: one producer warp keeps a ring of K/V blocks in flight by TMA (one
// box per page, 128-byte swizzle, pages that no row sees read as zero without touching memory), four
// warps each take a quarter of a block's keys with mma.sync m16n8k16 (tcgen05 needs 128 rows to a tile,
// of which a single row of 4 heads would fill 4) and keep their own running maximum and sum, joined once
// at the end; long caches are split over blocks, the last part to finish joins the tile in the order of
// the parts. The probabilities enter the second product as the sum of two 16-bit words, so that a weight
// is off by 2^-16 (bf16; fp16 2^-22) where one word has 2^-8 (2^-11); the tensor pipe is idle enough for that here.
// Two blocks per SM with three stages each. 96 single rows after 4,170 rows each, 32/8 heads x 128
// (1641 MB): 268 us, 6.1 TB/s; 10 rows of 128 episodes of 470, 12 heads x 64, not causal (192 MB): 43 us, 4.5 TB/s
// -- 3 us to the first bytes, and stretches end up to 10 % apart, since the SMs get unequal shares of HBM.
#include <cmath>
#include <cstdint>
#include <cstring>
#include <cuda.h>
#include <cuda_runtime.h>

#include "mkx_attend.cuh"
#include "mkx_cache_host.h"
#include "mkx_pdl.cuh"

namespace mkxa {
namespace {

constexpr int MT = 16;
using mkxc::MAX_DEVICES;
constexpr int MAX_KEYS = 1 << 30;  // rows of an episode: keys and positions are 32-bit
constexpr int ROW_WARPS = 4;
constexpr int ROW_THREADS = 32 * (ROW_WARPS + 1);
constexpr int ROW_STAGES = 3;
constexpr int JOIN_AT_ONCE = 12;      // parts that one block joins; more in two levels
constexpr int ROWS_JOIN_AT_ONCE = 26;  // the same where a part has 16 rows: below it the second level costs more than it saves
                                      // (17 to 26 parts: 13.3 against 14.5 us; 37: 20.8 against 18.4 us)

template <int HD>
struct RowShape {
  static constexpr int KT = 8192 / HD;               // keys per block: 16 KB of K, 16 KB of V
  static constexpr int KW = KT / ROW_WARPS;          // keys of a warp
  static constexpr int HALF = KT * 128;              // bytes of a 64-dim half of K or V
  static constexpr int STAGE = 2 * KT * HD * 2;
  static constexpr int JOIN = HD / 4 + 2;            // floats of a row in the join of the warps
  static constexpr int QROW = HD * 2 + 16;           // bytes of a row of Q: fragments without bank conflicts
  static constexpr int SMEM = ROW_STAGES * STAGE + ROW_WARPS * MT * (JOIN * 4 + 8) + MT * QROW + 1024 + 128;
};

// log2 of what fp16 probabilities are multiplied by (sums and totals alike, so it drops out at the end): below 2^-24 fp16
// ends, and many keys that far under one high one (a first row that everything looks at) weigh something together. 2^15,
// the most that fits, where the largest is 1; in chunks it may be 2^8. What is lost of a key is then below 2^-32 of the
// largest weight, without a cost. bf16 has the exponents of fp32.
template <int DT>
constexpr float ROWS_LIFT = DT == MKX_FP16 ? 15.f : 0.f;
template <int DT>
constexpr float CHUNK_LIFT = DT == MKX_FP16 ? 7.f : 0.f;
// What is taken off the scores whose largest is `top`: top - LIFT, rounded up, since from 2^24 on it is a whole number of
// units of a float, which the lift may not be; rounded down the largest weight would be 2^16, which fp16 does not have. A
// row's maximum is kept in this form, so that sums of different blocks are lifted alike whatever the rounding.
template <int DT>
__device__ __forceinline__ float rows_base(float top) {
  if constexpr (ROWS_LIFT<DT> == 0.f) return top;
  return __fsub_ru(top, ROWS_LIFT<DT>);
}
template <int DT>
__device__ __forceinline__ float chunk_base(float top) {
  if constexpr (CHUNK_LIFT<DT> == 0.f) return top;
  return __fsub_ru(top, CHUNK_LIFT<DT>);
}

template <int DT>
__device__ __forceinline__ void mma16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (DT == MKX_BF16)
    mma_bf16(d, a[0], a[1], a[2], a[3], b0, b1);
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
        "{%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldsm4(uint32_t (&v)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&v)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void row_barrier() { asm volatile("bar.sync 1, %0;" ::"n"(32 * ROW_WARPS) : "memory"); }

extern __shared__ __align__(1024) char asmem[];

template <int DT, int HD>
__global__ void __launch_bounds__(ROW_THREADS, 2)
    rows_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
                const __grid_constant__ AttendParams p) {
  using S = RowShape<HD>;
  constexpr int KT = S::KT, KW = S::KW, PART = MT * (HD + 2);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  char* ring = asmem + ((1024u - (smem_u32(asmem) & 1023u)) & 1023u);
  float* os = reinterpret_cast<float*>(ring + ROW_STAGES * S::STAGE);  // [4 warps][16 rows][S::JOIN]
  float2* ml = reinterpret_cast<float2*>(os + ROW_WARPS * MT * S::JOIN);  // [4][16]
  uint64_t* full = reinterpret_cast<uint64_t*>(ml + ROW_WARPS * MT);
  uint64_t* empty = full + ROW_STAGES;
  uint64_t* qfull = empty + ROW_STAGES;  // the next tile's rows of Q, copied ahead
  uint64_t* qempty = qfull + 1;
  char* qs = reinterpret_cast<char*>(qempty + 1);  // [16 rows][S::QROW]
  if (threadIdx.x == 0) {
    for (int s = 0; s < ROW_STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], ROW_WARPS);
    }
    mbar_init(qfull, 1);
    mbar_init(qempty, ROW_WARPS);
    fence_mbar_init();
  }
  __shared__ LineScratch scratch;
  __shared__ JoinWords words;
  BarrierTeam<32 * ROW_WARPS> team;
  Line line;
  pdl_begin();
  if (!find_line<MT, KT, ROW_THREADS>(p, scratch, line)) return;  // its barriers publish the mbarriers too
  Walk<MT, KT> walk(p, line);
  Segment sg;
  int n = 0, tiles = 0;  // blocks of keys and tiles since the start: n % ROW_STAGES is a block's stage

  if (warp == ROW_WARPS) {
    // producer: lane j fetches the j-th page of each block
    const int rows_box = min(1 << p.shift, KT), boxes = KT / rows_box;
    bool ok = true;
    while (ok && walk.next(sg)) {
      const int r0 = sg.tile * MT, r1 = min(r0 + MT, sg.fresh * p.group) - 1;
      const Keys ks = keys_of<KT>(p, sg, r0, r1);
      const int i0 = first_block(sg, ks.blocks), i1 = end_block(sg, ks.blocks);
      auto page_at = [&](int i) {
        return lane < boxes ? page_of(p, ks, sg.b, (block_key<KT>(ks, i) >> p.shift) + lane) : -1;
      };
      if (i0 >= i1) continue;
      int id = page_at(i0);
      if (tiles >= 1) ok = wait_bounded(qempty, (tiles & 1) ^ 1, p.timeout_ns);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      if (lane == 0) mbar_expect_tx(qfull, (uint32_t)((r1 - r0 + 1) * HD * 2));
      __syncwarp();
      if (lane <= r1 - r0) {
        const int r = r0 + lane, t = by_group(p, r);
        bulk_g2s(qs + lane * S::QROW,
                 (const char*)p.q + 2 * ((long long)(sg.first_row + t) * p.q_row +
                                         (long long)(sg.kvh * p.group + r - t * p.group) * p.q_head),
                 HD * 2, qfull);
      }
      ++tiles;
      for (int i = i0; i < i1; ++i, ++n) {
        const int s = n % ROW_STAGES;
        const int next = i + 1 < i1 ? page_at(i + 1) : -1;
        if (n >= ROW_STAGES) ok = wait_bounded(&empty[s], ((n / ROW_STAGES) & 1) ^ 1, p.timeout_ns);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        if (lane == 0) mbar_expect_tx(&full[s], (uint32_t)S::STAGE);
        __syncwarp();
        if (lane < boxes) {
          const int row = boxes > 1 ? 0 : block_key<KT>(ks, i) & ((1 << p.shift) - 1);
          char* at = ring + s * S::STAGE + lane * rows_box * 128;
#pragma unroll
          for (int h = 0; h < HD / 64; ++h) {
            tma_load_4d(at + h * S::HALF, &tk, 64 * h, row, sg.kvh, id, &full[s]);
            tma_load_4d(at + KT * HD * 2 + h * S::HALF, &tv, 64 * h, row, sg.kvh, id, &full[s]);
          }
        }
        id = next;
      }
    }
    if (!ok && lane == 0) {  // a wait ran out: let what is in flight land before the block ends
      atomicCAS(p.error, 0, 0x201);
      for (int k = max(0, n - ROW_STAGES); k < n; ++k)
        wait_bounded(&full[k % ROW_STAGES], (k / ROW_STAGES) & 1, p.timeout_ns);
      if (tiles > 0) wait_bounded(qfull, (tiles - 1) & 1, p.timeout_ns);
    }
    return;
  }

  const int g = lane >> 2, c = lane & 3;
  // ldmatrix: lane's row and 16-byte chunk of the four 8x8 parts
  const int krow = (lane & 7) + ((lane >> 4) << 3), kchunk = (lane >> 3) & 1;   // keys 0-7, 0-7, 8-15, 8-15
  const int vrow = (lane & 7) + (((lane >> 3) & 1) << 3), vchunk = lane >> 4;   // keys 0-7, 8-15, 0-7, 8-15
  bool ok = true;
  while (walk.next(sg)) {
    const int r0 = sg.tile * MT, r1 = min(r0 + MT, sg.fresh * p.group) - 1;
    const Keys ks = keys_of<KT>(p, sg, r0, r1);
    const int i0 = first_block(sg, ks.blocks), i1 = end_block(sg, ks.blocks);
    // queries: A fragments of the 16 rows (rows that are not there hold anything: no row touches another)
    uint32_t qf[HD / 16][4];
    int pos[2];
    if (i0 < i1) {
      ok = ok && __all_sync(0xffffffffu, wait_bounded(qfull, tiles & 1, p.timeout_ns));
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        pos[x] = sg.past + by_group(p, r0 + g + 8 * x);
        const char* q = qs + (g + 8 * x) * S::QROW + 4 * c;
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk) {
          qf[kk][x] = signed_q(p, *reinterpret_cast<const uint32_t*>(q + 32 * kk));
          qf[kk][x + 2] = signed_q(p, *reinterpret_cast<const uint32_t*>(q + 32 * kk + 16));
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(qempty);
      ++tiles;
    }
    float o[HD / 8][4];
#pragma unroll
    for (int j = 0; j < HD / 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    for (int i = i0; i < i1 && ok; ++i, ++n) {
      const int s = n % ROW_STAGES;
      ok = __all_sync(0xffffffffu, wait_bounded(&full[s], (n / ROW_STAGES) & 1, p.timeout_ns));
      if (!ok) break;
      const int key0 = block_key<KT>(ks, i) + warp * KW;
      char* kt = ring + s * S::STAGE;
      char* vt = kt + KT * HD * 2;
      const bool ragged = key0 + KW > ks.hi;
      if (ragged) {  // rows behind the last key may hold anything, and 0 * NaN is not 0
        for (int e = lane; e < KW * (HD / 8); e += 32) {
          const int row = e / (HD / 8), ch = e % (HD / 8);
          if (key0 + row >= ks.hi)
            *reinterpret_cast<uint4*>(vt + (ch >> 3) * S::HALF + (warp * KW + row) * 128 + (ch & 7) * 16) =
                make_uint4(0, 0, 0, 0);
        }
        __syncwarp();
      }
      const uint32_t ka = smem_u32(kt), va = smem_u32(vt);
      float sc[KW / 8][4];
#pragma unroll
      for (int j = 0; j < KW / 8; ++j) sc[j][0] = sc[j][1] = sc[j][2] = sc[j][3] = 0.f;
#pragma unroll
      for (int kk = 0; kk < HD / 16; ++kk)
#pragma unroll
        for (int j = 0; j < KW / 16; ++j) {
          const int row = warp * KW + 16 * j + krow, ch = 2 * (kk & 3) + kchunk;
          uint32_t b[4];
          ldsm4(b, ka + (kk >> 2) * S::HALF + row * 128 + ((ch ^ (row & 7)) << 4));
          mma16<DT>(sc[2 * j], qf[kk], b[0], b[1]);
          mma16<DT>(sc[2 * j + 1], qf[kk], b[2], b[3]);
        }
      float top[2] = {-INFINITY, -INFINITY};
      uint32_t seen[2] = {~0u, ~0u};  // of this thread's columns 8 j + 2 c + (0, 1)
      if (!whole_block<KT>(p, ks, block_key<KT>(ks, i)))
#pragma unroll
        for (int x = 0; x < 2; ++x) seen[x] = seen_mask(p, ks, pos[x], key0) >> (2 * c);
#pragma unroll
      for (int j = 0; j < KW / 8; ++j)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          float v = sc[j][x] * p.scale_log2;
          if (!((seen[x >> 1] >> (8 * j + (x & 1))) & 1u)) v = -INFINITY;
          sc[j][x] = v;
          top[x >> 1] = fmaxf(top[x >> 1], v);
        }
      float fix[2];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        top[x] = fmaxf(top[x], __shfl_xor_sync(0xffffffffu, top[x], 1));
        top[x] = fmaxf(top[x], __shfl_xor_sync(0xffffffffu, top[x], 2));
        const float now = fmaxf(m[x], rows_base<DT>(top[x]));
        top[x] = now == -INFINITY ? 0.f : now;
        fix[x] = ex2(m[x] - top[x]);
        m[x] = now;
        l[x] *= fix[x];
      }
#pragma unroll
      for (int j = 0; j < HD / 8; ++j) {
        o[j][0] *= fix[0];
        o[j][1] *= fix[0];
        o[j][2] *= fix[1];
        o[j][3] *= fix[1];
      }
#pragma unroll
      for (int j = 0; j < KW / 16; ++j) {
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int y = 0; y < 4; ++y) {  // A fragment words: (row g, keys 0-7), (g + 8, 0-7), (g, 8-15), (g + 8, 8-15)
          const int t = 2 * j + (y >> 1), x = y & 1;
          const float a = ex2(sc[t][2 * x] - top[x]), b = ex2(sc[t][2 * x + 1] - top[x]);
          l[x] += a + b;
          hi[y] = Half16<DT>::pack(a, b);
          const float2 h = Half16<DT>::unpack(hi[y]);
          lo[y] = Half16<DT>::pack(a - h.x, b - h.y);
        }
#pragma unroll
        for (int n16 = 0; n16 < HD / 16; ++n16) {
          const int row = warp * KW + 16 * j + vrow, ch = 2 * (n16 & 3) + vchunk;
          uint32_t b[4];
          ldsm4_t(b, va + (n16 >> 2) * S::HALF + row * 128 + ((ch ^ (row & 7)) << 4));
          mma16<DT>(o[2 * n16], hi, b[0], b[1]);
          mma16<DT>(o[2 * n16 + 1], hi, b[2], b[3]);
          mma16<DT>(o[2 * n16], lo, b[0], b[1]);
          mma16<DT>(o[2 * n16 + 1], lo, b[2], b[3]);
        }
      }
      if (ragged) fence_proxy_async();  // the zeros above, before the next copy into this stage
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[s]);
    }

    // join the four warps, a quarter of the dims at a time (the copies of the next tile own the ring):
    // 8 threads per row, HD / 32 neighbouring dims each
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      l[x] += __shfl_xor_sync(0xffffffffu, l[x], 1);
      l[x] += __shfl_xor_sync(0xffffffffu, l[x], 2);
    }
    if (c == 0) {
      ml[warp * MT + g] = make_float2(m[0], l[0]);
      ml[warp * MT + g + 8] = make_float2(m[1], l[1]);
    }
    constexpr int D = HD / 32;
    const int row = threadIdx.x >> 3, q = threadIdx.x & 7;
    float acc[4][D], mx = -INFINITY, ls = 0.f, f[ROW_WARPS];
#pragma unroll
    for (int quarter = 0; quarter < 4; ++quarter) {
#pragma unroll
      for (int j = 0; j < D; ++j) {
        *reinterpret_cast<float2*>(os + (warp * MT + g) * S::JOIN + 8 * j + 2 * c) =
            make_float2(o[quarter * D + j][0], o[quarter * D + j][1]);
        *reinterpret_cast<float2*>(os + (warp * MT + g + 8) * S::JOIN + 8 * j + 2 * c) =
            make_float2(o[quarter * D + j][2], o[quarter * D + j][3]);
      }
      row_barrier();
      if (quarter == 0) {
#pragma unroll
        for (int w = 0; w < ROW_WARPS; ++w) mx = fmaxf(mx, ml[w * MT + row].x);
        const float safe = mx == -INFINITY ? 0.f : mx;
#pragma unroll
        for (int w = 0; w < ROW_WARPS; ++w) {
          const float2 t = ml[w * MT + row];
          f[w] = ex2(t.x - safe);
          ls += f[w] * t.y;
        }
      }
#pragma unroll
      for (int d = 0; d < D; ++d) {
        acc[quarter][d] = 0.f;
#pragma unroll
        for (int w = 0; w < ROW_WARPS; ++w) acc[quarter][d] += f[w] * os[(w * MT + row) * S::JOIN + q * D + d];
      }
      row_barrier();
    }
    const int r = r0 + row;
    if (sg.parts > 1) {
      auto keep = [&](int k) {  // dims of a thread: quarter * HD / 4 + q * D + d
        if (r > r1) return;
        float* part = p.parts + (size_t)part_place(sg, k) * PART;
#pragma unroll
        for (int quarter = 0; quarter < 4; ++quarter)
#pragma unroll
          for (int d = 0; d < D; d += 2)
            __stcg(reinterpret_cast<float2*>(part + row * HD + quarter * (HD / 4) + q * D + d),
                   make_float2(acc[quarter][d], acc[quarter][d + 1]));
        if (q == 0) __stcg(reinterpret_cast<float2*>(part + MT * HD) + row, make_float2(mx, ls));
      };
      keep(blockIdx.x - sg.lead);
      // sums of parts first, first + step, ..., `count` of them, into acc, mx, ls
      auto add_up = [&](int first, int step, int count) {
        if (r > r1) return;
        mx = -INFINITY;
        ls = 0.f;
#pragma unroll
        for (int quarter = 0; quarter < 4; ++quarter)
#pragma unroll
          for (int d = 0; d < D; ++d) acc[quarter][d] = 0.f;
#pragma unroll 4
        for (int k = 0; k < count; ++k) {
          const float* at = p.parts + (size_t)part_place(sg, first + k * step) * PART;
          const float2 t = __ldcg(reinterpret_cast<const float2*>(at + MT * HD) + row);
          const float top = fmaxf(mx, t.x), safe = top == -INFINITY ? 0.f : top, fix = ex2(mx - safe), w = ex2(t.x - safe);
          mx = top;
          ls = ls * fix + w * t.y;
#pragma unroll
          for (int quarter = 0; quarter < 4; ++quarter)
#pragma unroll
            for (int d = 0; d < D; d += 2) {
              const float2 v = __ldcg(reinterpret_cast<const float2*>(at + row * HD + quarter * (HD / 4) + q * D + d));
              acc[quarter][d] = acc[quarter][d] * fix + w * v.x;
              acc[quarter][d + 1] = acc[quarter][d + 1] * fix + w * v.y;
            }
        }
      };
      // many parts are joined in two levels, so that no block reads more than a few
      int step = 1, groups = sg.parts;
      if (sg.parts > ROWS_JOIN_AT_ONCE) {
        step = JOIN_AT_ONCE;
        groups = ceil_div(sg.parts, step);
        const int first = (int)(blockIdx.x - sg.lead) / step * step, count = min(step, sg.parts - first);
        if (!last_of(team, p.tickets + p.slots + part_place(sg, first), count, words)) continue;
        add_up(first, 1, count);
        row_barrier();  // the group's first part has been read: the group's sums take its place
        keep(first);
      }
      if (!last_of(team, p.tickets + sg.lead, groups, words)) continue;
      add_up(0, step, groups);
    }
    if (r <= r1) {
      const int t = by_group(p, r);
      char* out = (char*)p.out + 2 * ((long long)(sg.first_row + t) * p.o_row +
                                      (long long)(sg.kvh * p.group + r - t * p.group) * p.o_head + q * D);
      const float inv = over_total(p, sg.first_row + t, ls);
#pragma unroll
      for (int quarter = 0; quarter < 4; ++quarter)
#pragma unroll
        for (int d = 0; d < D; d += 2)
          *reinterpret_cast<uint32_t*>(out + 2 * (quarter * (HD / 4) + d)) =
              Half16<DT>::pack(acc[quarter][d] * inv, acc[quarter][d + 1] * inv);
    }
  }
  if (!ok && lane == 0) atomicCAS(p.error, 0, 0x202);
}

// ---- chunks ----------------------------------------------------------------------------------------
// chunk_kernel: tiles of 256 rows as two tiles A, B of 128, one CTA per SM. Both products run on
// tcgen05 (128-key blocks): S = Q K^T from shared memory into TMEM, O += P V with P read from TMEM and V
// as TMA left it (dims contiguous). Four warps per tile, one thread per row: no shuffles, the row's
// maximum and sum stay in registers. O is rescaled only when a maximum has grown by more than 2^8 since the
// last time, which is rare after the first blocks: P stays below 2^8 (2^15 as lifted), inside both types. P is rounded
// to 16 bits once, as the second product takes no wider weights on tcgen05; the sum l is of the unrounded.
// At head_dim 128 TMEM is full with two tiles of S and O, and P overwrites the scores it came from: a
// tile's products wait for its softmax and the other way round, and the two tiles alternate. At head_dim
// 64 P has columns of its own, and the next scores are there before the last ones are done.
// Bound by the exponentials at head_dim 64 (16 a clock per SM: 2048 clocks for two 128 x 128 tiles, whose
// products take 1024), by both alike at 128; a quarter of them is taken off that unit (exp2_pair). What is
// reached is 3850 clocks for the two tiles at 128 (2011 rows after 3007 to 12,007 keys: 1.96 us for each
// further 128 keys of 256 rows at 1965 MHz, 2.24 at 1720), where the softmax between two products of a
// tile (load, maximum, exponentials, store) is a chain that the other tile's covers in part. The start, Q, O,
// parts and joins take some 60,000 clocks of a call beside it.
// 2011 rows after 6007, 32/8 heads x 128 (231 GFLOP): 227 us in short runs, 246 to 253 us in a long one under
// the power cap (0.92 PFLOP/s, 1.75 GHz); six chunks of 1,000 rows, window 1024 and 70 sinks, 12 heads x 64 (20
// GFLOP): 64.6 us.
constexpr int CT = 256;
constexpr int CK = 128;
constexpr int TILE_THREADS = 256;                   // warps 0-3 tile A, 4-7 tile B
constexpr int CHUNK_THREADS = TILE_THREADS + 128;   // 8 TMA, 9 and 11 MMA, 10 walks the line
// Registers per thread: 384 x 168 at launch; the warps of the tiles, a row of scores each, take 216, the others 72
// (256 x 216 + 128 x 72 = 384 x 168).
constexpr int TILE_REGS = 216, OTHER_REGS = 72;
constexpr float LAZY = 8.f;  // log2 of the growth that is let pass
constexpr int JOBS = 4;

template <int HD>
struct ChunkShape {
  static constexpr bool EARLY = HD == 64;               // P beside S in TMEM
  static constexpr int TILE = CK * HD * 2;              // one K or V block
  static constexpr int HALF = CK * 128;                 // its 64-dim half
  static constexpr int SLOTS = HD == 128 ? 5 : 8;
  static constexpr int POLY_EACH = 4;                   // every so many pairs of exponentials is a polynomial
  static constexpr int QHALF = CT * 128;
  // TMEM columns of a tile: S, O, P
  static __device__ __forceinline__ uint32_t s_at(int x) { return 128 * x; }
  static __device__ __forceinline__ uint32_t o_at(int x) { return 256 + HD * x; }
  static __device__ __forceinline__ uint32_t p_at(int x) { return EARLY ? 384 + 64 * x : 128 * x; }
};

// Shared-memory matrix descriptors in two words: the low one (address and leading offset, both / 16) changes from
// product to product by additions, the high one (stride offset 1024 between 8-row groups, version 1, 128-byte
// swizzle) is one constant. Q and K are K-major (leading offset unused). A 64-dim half of V is 128 keys x 128 bytes with
// the dims contiguous ("MN-major" B operand): 8-key groups are a stride offset apart, the halves a leading offset.
constexpr uint32_t DESC_HIGH = 64u | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_low(uint32_t addr, uint32_t leading) {
  return ((addr >> 4) & 0x3FFFu) | ((leading >> 4) << 16);
}
// An MMA warp stays converged, so that descriptors live in uniform registers (one thread by itself moves six
// registers per product, 100 clocks for a product of 64): the instruction is predicated on its one elected lane.
// D[tmem] (+)= A[smem] * B[smem]^T, K = 16.
__device__ __forceinline__ void umma_ss(uint32_t lead, uint32_t d, uint32_t a_low, uint32_t b_low, uint32_t idesc,
                                        uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 a, b;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "mov.b64 a, {%1, %6};\n\tmov.b64 b, {%2, %6};\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t}\n" ::"r"(d),
      "r"(a_low), "r"(b_low), "r"(idesc), "r"(accumulate), "r"(lead), "n"(DESC_HIGH));
}
// D[tmem] (+)= A[tmem] * B[smem]: A is 128 lanes x 16 16-bit values in 8 columns.
__device__ __forceinline__ void umma_ts(uint32_t lead, uint32_t d, uint32_t a, uint32_t b_low, uint32_t idesc,
                                        uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 b;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "mov.b64 b, {%2, %6};\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t}\n" ::"r"(d),
      "r"(a), "r"(b_low), "r"(idesc), "r"(accumulate), "r"(lead), "n"(DESC_HIGH));
}
__device__ __forceinline__ void commit_by(uint32_t lead, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}\n" ::"r"(smem_u32(bar)),
      "r"(lead)
      : "memory");
}
__device__ __forceinline__ uint32_t elect_one() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}\n" : "=r"(r));
  return r;
}
__device__ __forceinline__ int uniform(int v) { return __shfl_sync(0xffffffffu, v, 0); }
// Lanes 32 (warp % 4) .. + 31, 64 columns.
__device__ __forceinline__ void tmem_ld64(uint32_t taddr, uint32_t (&v)[64]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x64.b32 {"
      "%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, "
      "%20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32, %33, %34, %35, %36, %37, "
      "%38, %39, %40, %41, %42, %43, %44, %45, %46, %47, %48, %49, %50, %51, %52, %53, %54, %55, "
      "%56, %57, %58, %59, %60, %61, %62, %63 "
      "}, [%64];\n\ttcgen05.wait::ld.sync.aligned;"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
        "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]),
        "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]),
        "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]),
        "=r"(v[29]), "=r"(v[30]), "=r"(v[31]), "=r"(v[32]), "=r"(v[33]), "=r"(v[34]), "=r"(v[35]),
        "=r"(v[36]), "=r"(v[37]), "=r"(v[38]), "=r"(v[39]), "=r"(v[40]), "=r"(v[41]), "=r"(v[42]),
        "=r"(v[43]), "=r"(v[44]), "=r"(v[45]), "=r"(v[46]), "=r"(v[47]), "=r"(v[48]), "=r"(v[49]),
        "=r"(v[50]), "=r"(v[51]), "=r"(v[52]), "=r"(v[53]), "=r"(v[54]), "=r"(v[55]), "=r"(v[56]),
        "=r"(v[57]), "=r"(v[58]), "=r"(v[59]), "=r"(v[60]), "=r"(v[61]), "=r"(v[62]), "=r"(v[63])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]),
      "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]),
      "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Two floats at a time on the fp32 pipe.
__device__ __forceinline__ uint64_t f2(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ float2 unf2(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// 2^x of two floats without the exponential unit, for x <= 126: 2^x = 2^n 2^f with n the nearest integer (adding
// 1.5 * 2^23 leaves it in the low bits), |f| <= 1/2, and 2^f by a polynomial whose relative error is the smallest
// possible with constant term 1 (so that x = -inf, taken as -127, gives 0): 1.0e-4 in degree 3, a fortieth of half a
// bf16 step, 2.8e-6 in degree 4, for fp16.
template <int DT>
__device__ __forceinline__ float2 exp2_pair(uint64_t x2) {
  const float2 x = unf2(x2);
  x2 = f2(fmaxf(x.x, -127.f), fmaxf(x.y, -127.f));
  const uint64_t magic = f2(12582912.f, 12582912.f);
  const uint64_t r2 = add2(x2, magic);
  const uint64_t f = fma2(add2(r2, f2(-12582912.f, -12582912.f)), f2(-1.f, -1.f), x2);
  uint64_t y;
  if constexpr (DT == MKX_BF16) {
    y = fma2(f2(0.05500893294811249f, 0.05500893294811249f), f, f2(0.24221095442771912f, 0.24221095442771912f));
    y = fma2(y, f, f2(0.6932829022407532f, 0.6932829022407532f));
  } else {
    y = fma2(f2(0.009582852944731712f, 0.009582852944731712f), f, f2(0.055906426161527634f, 0.055906426161527634f));
    y = fma2(y, f, f2(0.24024099111557007f, 0.24024099111557007f));
    y = fma2(y, f, f2(0.6931241750717163f, 0.6931241750717163f));
  }
  const float2 v = unf2(fma2(y, f, f2(1.f, 1.f))), r = unf2(r2);
  return make_float2(__int_as_float(__float_as_int(v.x) + (__float_as_int(r.x) << 23)),
                     __int_as_float(__float_as_int(v.y) + (__float_as_int(r.y) << 23)));
}

// What every role needs to know of a segment, worked out once by a warp of its own and handed on in shared memory.
// Tile x computes the blocks i < to with i < sinks or i >= from; those of whole_from .. whole_to - 1 need no mask.
struct Tile {
  int sinks, from, to, whole_from, whole_to;
  __device__ __forceinline__ bool uses(int i) const { return i < to && (i < sinks || i >= from); }
};
struct Job {
  Segment sg;
  int r0, r1, i0, i1;  // rows (inclusive), key blocks taken here; i0 < 0: no more jobs
  Keys keys;           // of both tiles together
  Tile tile[2];
};
__device__ __forceinline__ void fill(const AttendParams& p, Job& job, const Segment& sg) {
  const int r0 = sg.tile * CT, r1 = min(r0 + CT, sg.fresh * p.group) - 1;
  const Keys all = keys_of<CK>(p, sg, r0, r1);
  job.sg = sg;
  job.r0 = r0;
  job.r1 = r1;
  job.i0 = first_block(sg, all.blocks);
  job.i1 = end_block(sg, all.blocks);
  job.keys = all;
  for (int x = 0; x < 2; ++x) {
    Tile t{0, 0, 0, 0, 0};
    const int a = r0 + 128 * x;
    if (a <= r1) {
      const Keys k = keys_of<CK>(p, sg, a, min(a + 127, r1));
      const int skip = all.sink_blocks - all.lo_block / CK;  // block i of the main range holds keys (i - skip) * CK ..
      t.from = skip + k.lo / CK;
      t.to = k.hi > 0 ? skip + ceil_div(k.hi, CK) : 0;
      t.sinks = p.window ? max(all.sink_blocks, skip + ceil_div(p.sinks, CK)) : 0;
      t.whole_from = p.window ? skip + max(k.p_last - p.window + CK, 0) / CK : 0;
      t.whole_to = skip + max(p.causal ? min(k.hi, k.p_first + 1) : k.hi, 0) / CK;
    }
    job.tile[x] = t;
  }
}

template <int HD>
struct ChunkShared {
  char ring[ChunkShape<HD>::SLOTS * ChunkShape<HD>::TILE];  // K and V blocks
  char q[CT * HD * 2];                                      // [HD / 64][256 rows][128 bytes], 128-byte swizzle
  LineScratch line;
  uint64_t full[ChunkShape<HD>::SLOTS], empty[ChunkShape<HD>::SLOTS], raw;
  uint64_t qfull[2];     // a tile's rows of Q are in shared memory
  uint64_t sfull[2];     // its scores are in TMEM
  uint64_t sfree[2];     // its scores are in registers (EARLY)
  uint64_t pfull[2][2];  // the first, the second half of its probabilities are
  uint64_t ofull[2];     // its sums include them
  uint64_t done;
  uint64_t turns[2];     // the MMA warps' turns
  uint64_t joins;        // the tiles' warps meet to join
  uint64_t jfull[JOBS], jempty[JOBS];
  uint32_t tmem;
  JoinWords words;
  Job jobs[JOBS];
};
static_assert(sizeof(ChunkShared<128>) <= 227 * 1024, "one block's shared memory");

template <int DT, int HD>
__global__ void __launch_bounds__(CHUNK_THREADS, 1)
    chunk_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
                 const __grid_constant__ AttendParams p) {
  using S = ChunkShape<HD>;
  constexpr int SLOTS = S::SLOTS;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  auto& sm = *reinterpret_cast<ChunkShared<HD>*>(asmem);
  char* ring = sm.ring;
  char* qs = sm.q;
  if (smem_u32(asmem) & 1023u) {  // (nothing else is in shared memory)
    if (threadIdx.x == 0) atomicCAS(p.error, 0, 0x210);
    return;
  }
  if (threadIdx.x == 0) {
    for (int s = 0; s < SLOTS; ++s) {
      mbar_init(&sm.full[s], 1);
      mbar_init(&sm.empty[s], 2);  // both tiles' products have read it
    }
    mbar_init(&sm.raw, 1);
    for (int x = 0; x < 2; ++x) {
      mbar_init(&sm.qfull[x], 4);
      mbar_init(&sm.sfull[x], 1);
      mbar_init(&sm.sfree[x], 4);
      mbar_init(&sm.pfull[x][0], 4);
      mbar_init(&sm.pfull[x][1], 4);
      mbar_init(&sm.ofull[x], 1);
      mbar_init(&sm.turns[x], 1);
    }
    mbar_init(&sm.done, 2);
    mbar_init(&sm.joins, TILE_THREADS / 32);
    for (int j = 0; j < JOBS; ++j) {
      mbar_init(&sm.jfull[j], 1);
      mbar_init(&sm.jempty[j], 11);  // the producer, the two MMA warps, the eight warps of the tiles
    }
    fence_mbar_init();
  }
  Line line;
  pdl_begin();
  if (!find_line<CT, CK, CHUNK_THREADS>(p, sm.line, line)) return;
  if (warp == 9) tmem_alloc(&sm.tmem, 512);
  __syncthreads();
  tmem_fence_after();
  const uint32_t tmem = sm.tmem;

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(OTHER_REGS));
    if (warp == 8) {
      // producer: slots hold K, V, K, V, ... of the blocks in order; lane j fetches the j-th page
      const int rows_box = min(1 << p.shift, CK), boxes = CK / rows_box;
      bool ok = true;
      int n = 0, raws = 0;
      for (int jn = 0; ok; ++jn) {
        ok = __all_sync(0xffffffffu, wait_bounded(&sm.jfull[jn % JOBS], (jn / JOBS) & 1, p.timeout_ns));
        if (!ok) break;
        const Job& job = sm.jobs[jn % JOBS];
        const int i0 = job.i0, i1 = job.i1, b = job.sg.b, kvh = job.sg.kvh;
        const Keys ks = job.keys;
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.jempty[jn % JOBS]);
        if (i0 < 0) break;
        auto page_at = [&](int i) {
          return lane < boxes ? page_of(p, ks, b, (block_key<CK>(ks, i) >> p.shift) + lane) : -1;
        };
        int id = i0 < i1 ? page_at(i0) : -1;
        for (int i = i0; i < i1 && ok; ++i) {
          const int next = i + 1 < i1 ? page_at(i + 1) : -1;
          const int key0 = block_key<CK>(ks, i), row = boxes > 1 ? 0 : key0 & ((1 << p.shift) - 1);
#pragma unroll
          for (int kv = 0; kv < 2; ++kv, ++n) {
            const int s = n % SLOTS;
            if (n >= SLOTS) ok = wait_bounded(&sm.empty[s], ((n / SLOTS) & 1) ^ 1, p.timeout_ns);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            // rows of V behind the last key may hold anything, and 0 * NaN is not 0: they are zeroed here
            const bool ragged = kv == 1 && key0 + CK > ks.hi;
            uint64_t* bar = ragged ? &sm.raw : &sm.full[s];
            if (lane == 0) mbar_expect_tx(bar, (uint32_t)S::TILE);
            __syncwarp();
            char* at = ring + s * S::TILE;
            if (lane < boxes)
#pragma unroll
              for (int h = 0; h < HD / 64; ++h)
                tma_load_4d(at + h * S::HALF + lane * rows_box * 128, kv ? &tv : &tk, 64 * h, row, kvh, id, bar);
            if (ragged) {  // a tile's last block
              ok = __all_sync(0xffffffffu, wait_bounded(&sm.raw, raws & 1, p.timeout_ns));
              ++raws;
              for (int e = lane + (ks.hi - key0) * (HD / 8); e < CK * (HD / 8); e += 32) {
                const int r = e / (HD / 8), ch = e % (HD / 8);
                *reinterpret_cast<uint4*>(at + (ch >> 3) * S::HALF + r * 128 + (ch & 7) * 16) = make_uint4(0, 0, 0, 0);
              }
              fence_proxy_async();
              __syncwarp();
              if (lane == 0) mbar_arrive(&sm.full[s]);
            }
          }
          id = next;
        }
      }
      if (!ok && lane == 0) {  // a wait ran out: let what is in flight land before the block ends
        atomicCAS(p.error, 0, 0x211);
        for (int k = max(0, n - SLOTS); k < n; ++k) wait_bounded(&sm.full[k % SLOTS], (k / SLOTS) & 1, p.timeout_ns);
      }
    } else if (warp != 10) {
      // the products of tile A (warp 9) and tile B (warp 11): two warps, because what one does around a block's
      // products, a few hundred clocks, then hides behind the other's. Without columns for P beside S they take turns,
      // so that one tile's products run under the other's softmax (otherwise both do the same at the same time: 281
      // instead of 239 us for 2011 rows after 6007, 32/8 heads x 128)
      constexpr uint32_t fmt = DT == MKX_BF16 ? 1u : 0u;
      constexpr uint32_t base = (1u << 4) | (fmt << 7) | (fmt << 10) | ((uint32_t)(128 >> 4) << 24);
      constexpr uint32_t id_qk = base | ((uint32_t)(CK >> 3) << 17);
      constexpr uint32_t id_pv = base | ((uint32_t)(HD >> 3) << 17) | (1u << 16);  // V: dims contiguous
      const int x = uniform(warp == 11);
      const uint32_t lead = elect_one(), tm = (uint32_t)uniform((int)tmem);
      const uint32_t st = tm + S::s_at(x), ot = tm + S::o_at(x), pt = tm + S::p_at(x);
      const uint32_t q = desc_low(smem_u32(qs), 0) + x * (128 * 128 >> 4), k_low = desc_low(smem_u32(ring), 0),
                     v_low = desc_low(smem_u32(ring), S::HALF);
      auto wait = [&](uint64_t* bar, int parity) {
        return __all_sync(0xffffffffu, wait_bounded(bar, (uint32_t)parity, p.timeout_ns)) != 0;
      };
      int n = 0, segments = 0, steps = 0;  // blocks and segments of this tile; turns taken
      int slot = 0, turn = 0;              // of K(i): slot and its phase
      bool ok = true;
      for (int jn = 0; ok; ++jn) {
        ok = wait(&sm.jfull[jn % JOBS], (jn / JOBS) & 1);
        if (!ok) break;
        const Job& job = sm.jobs[jn % JOBS];
        const int i0 = uniform(job.i0), i1 = uniform(job.i1);
        Tile tile;
        tile.sinks = uniform(job.tile[x].sinks);
        tile.from = uniform(job.tile[x].from);
        tile.to = uniform(job.tile[x].to);
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.jempty[jn % JOBS]);
        if (i0 < 0) break;
        const int n0 = n;
        bool mine = S::EARLY;
        auto my_turn = [&]() {
          const bool got = mine || wait(&sm.turns[x], (steps & 1) ^ (1 - x));
          mine = true;
          return got;
        };
        int done = n0;       // blocks whose V product has been issued
        auto add_pv = [&](int v_slot, int v_turn, bool has) {  // V(i - 1)
          if (!wait(&sm.full[v_slot], v_turn)) return false;
          if (!has) {
            if (lane == 0) mbar_arrive(&sm.empty[v_slot]);
            return true;
          }
          const uint32_t v = v_low + v_slot * (S::TILE >> 4);
#pragma unroll
          for (int part = 0; part < 2; ++part) {
            if (!wait(&sm.pfull[x][part], done & 1)) return false;
            if (part == 0 && !my_turn()) return false;
            tmem_fence_after();
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int kk = 4 * part + k;
              umma_ts(lead, ot, pt + 8 * kk, v + kk * (2048 >> 4), id_pv, (part > 0 || k > 0) ? 1u : (done > n0 ? 1u : 0u));
            }
          }
          commit_by(lead, &sm.ofull[x]);
          commit_by(lead, &sm.empty[v_slot]);
          ++done;
          return true;
        };
        int v_slot = 0, v_turn = 0;
        bool last_used = false;
        for (int i = i0; i <= i1; ++i) {
          const bool used = i < i1 && tile.uses(i);
          if (!S::EARLY && i > i0) ok = add_pv(v_slot, v_turn, last_used);
          if (!ok) break;
          if (i < i1) {
            ok = wait(&sm.full[slot], turn);
            if (used) {
              if (n == n0) ok = ok && wait(&sm.qfull[x], segments++ & 1);
              if (S::EARLY && n > 0) ok = ok && wait(&sm.sfree[x], (n - 1) & 1);
              ok = ok && my_turn();
              if (!ok) break;
              tmem_fence_after();
              const uint32_t k = k_low + slot * (S::TILE >> 4);
#pragma unroll
              for (int kk = 0; kk < HD / 16; ++kk)
                umma_ss(lead, st, q + (kk >> 2) * (S::QHALF >> 4) + 2 * (kk & 3), k + (kk >> 2) * (S::HALF >> 4) + 2 * (kk & 3),
                        id_qk, kk > 0 ? 1u : 0u);
              commit_by(lead, &sm.sfull[x]);
              commit_by(lead, &sm.empty[slot]);
              ++n;
            } else {
              if (!ok) break;
              if (lane == 0) mbar_arrive(&sm.empty[slot]);
            }
          }
          if (S::EARLY && i > i0) ok = add_pv(v_slot, v_turn, last_used);
          if (!ok) break;
          if (i < i1) {
            if (++slot == SLOTS) slot = 0, turn ^= 1;
            v_slot = slot;
            v_turn = turn;
            if (++slot == SLOTS) slot = 0, turn ^= 1;
          }
          last_used = used;
          if (!S::EARLY) {
            ok = my_turn();  // a step without products still takes its turn
            if (!ok) break;
            if (lane == 0) mbar_arrive(&sm.turns[1 - x]);
            ++steps;
            mine = false;
          }
        }
      }
      if (!ok && lane == 0) atomicCAS(p.error, 0, 0x213);
      commit_by(lead, &sm.done);
    } else if (lane == 0) {
      // walks the line
      Walk<CT, CK> walk(p, line);
      Segment sg;
      for (int jn = 0;; ++jn) {
        const bool more = walk.next(sg);
        if (jn >= JOBS && !wait_bounded(&sm.jempty[jn % JOBS], ((jn / JOBS) & 1) ^ 1, p.timeout_ns)) {
          atomicCAS(p.error, 0, 0x215);
          break;
        }
        if (more) fill(p, sm.jobs[jn % JOBS], sg);
        else sm.jobs[jn % JOBS].i0 = -1;
        mbar_arrive(&sm.jfull[jn % JOBS]);
        if (!more) break;
      }
    }
    __syncwarp();
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(TILE_REGS));
    const int x = warp >> 2, row = threadIdx.x;  // one row per thread
    const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
    const uint32_t st = tmem + lanes + S::s_at(x), ot = tmem + lanes + S::o_at(x), pt = tmem + lanes + S::p_at(x);
    const uint64_t scale2 = f2(p.scale_log2, p.scale_log2);
    BoundedTeam team(&sm.joins, p.timeout_ns);
    int n = 0;  // blocks of this tile since the start
    // After a wait that ran out the warp goes on without waiting: others of its barriers still count on it. Where it cannot
    // go on (no job, nobody to join with), it leaves, and those who count on it run into their own limits.
    bool ok = true;
    auto wait = [&](uint64_t* bar, int parity) {
      ok = ok && __all_sync(0xffffffffu, wait_bounded(bar, (uint32_t)parity, p.timeout_ns)) != 0;
    };
    for (int jn = 0;; ++jn) {
      if (!__all_sync(0xffffffffu, wait_bounded(&sm.jfull[jn % JOBS], (jn / JOBS) & 1, p.timeout_ns))) {
        ok = false;
        break;
      }
      const Job& job = sm.jobs[jn % JOBS];
      const int i0 = job.i0, i1 = job.i1;
      if (i0 < 0) break;
      const Tile tile = job.tile[x];
      float m = -INFINITY, l = 0.f;
      const int n0 = n;
      for (int i = i0; i < i1; ++i) {
        if (!tile.uses(i)) continue;
        if (n == n0) {
          // the tile's Q into shared memory, coalesced: 16-byte chunks of a row by neighbouring threads. Only for a
          // tile with work in this segment: warps without any run ahead, by more phases than a barrier tells apart
          const int first = job.r0 + 128 * x, last = job.r1, head = job.sg.kvh * p.group, th = threadIdx.x & 127;
          const char* rows = (const char*)p.q + 2 * (long long)job.sg.first_row * p.q_row;
          uint4 v[HD / 8];
#pragma unroll
          for (int k = 0; k < HD / 8; ++k) {  // all loads in flight at once
            const int e = th + 128 * k, r = first + e / (HD / 8), ch = e % (HD / 8);
            v[k] = make_uint4(0, 0, 0, 0);
            if (r <= last) {
              const int t = by_group(p, r);
              v[k] = __ldg(reinterpret_cast<const uint4*>(
                  rows + 2 * ((long long)t * p.q_row + (long long)(head + r - t * p.group) * p.q_head + 8 * ch)));
            }
          }
#pragma unroll
          for (int k = 0; k < HD / 8; ++k) {
            const int e = th + 128 * k, qr = 128 * x + e / (HD / 8), ch = e % (HD / 8);
            *reinterpret_cast<uint4*>(qs + (ch >> 3) * S::QHALF + qr * 128 + (((ch & 7) ^ (qr & 7)) << 4)) =
                make_uint4(signed_q(p, v[k].x), signed_q(p, v[k].y), signed_q(p, v[k].z), signed_q(p, v[k].w));
          }
          fence_proxy_async();
          __syncwarp();
          if (lane == 0) mbar_arrive(&sm.qfull[x]);
        }
        wait(&sm.sfull[x], n & 1);
        tmem_fence_after();
        uint32_t s[2][64];
        tmem_ld64(st, s[0]);
        tmem_ld64(st + 64, s[1]);
        if (S::EARLY) {  // the next scores may come
          tmem_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&sm.sfree[x]);
        }
        if (i < tile.whole_from || i >= tile.whole_to) {
          const int key0 = block_key<CK>(job.keys, i), position = job.sg.past + by_group(p, job.r0 + row);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t seen = seen_mask(p, job.keys, position, key0 + 32 * j);
            if (__all_sync(0xffffffffu, seen == ~0u)) continue;
#pragma unroll
            for (int d = 0; d < 32; ++d)
              if (!((seen >> d) & 1u)) s[j >> 1][32 * (j & 1) + d] = 0xff800000u;
          }
        }
        float tops[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) tops[k] = max_nan(__uint_as_float(s[0][k]), __uint_as_float(s[0][k + 8]));
#pragma unroll
        for (int j = 16; j < 128; j += 16)
#pragma unroll
          for (int k = 0; k < 8; ++k)
            tops[k] = max_nan(tops[k], __uint_as_float(s[j >> 6][(j & 63) + k]), __uint_as_float(s[j >> 6][(j & 63) + k + 8]));
        // half of a block's probabilities, as words of P; their sum is added to `sums`
        auto half_of = [&](const uint32_t (&sh)[64], uint64_t by, float base, uint32_t (&w)[32], uint64_t (&sums)[4]) {
          const uint64_t base2 = f2(-base, -base);
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            const uint64_t y = fma2(f2(__uint_as_float(sh[2 * j]), __uint_as_float(sh[2 * j + 1])), by, base2);
            float2 v;
            if (j % S::POLY_EACH == S::POLY_EACH - 1) {
              v = exp2_pair<DT>(y);
            } else {
              v = unf2(y);
              v = make_float2(ex2(v.x), ex2(v.y));
            }
            sums[j & 3] = add2(sums[j & 3], f2(v.x, v.y));
            w[j] = Half16<DT>::pack(v.x, v.y);
          }
        };
        uint32_t w[32];
        uint64_t sums[4] = {0, 0, 0, 0};
        const float top = p.scale_log2 *  // > 0: -inf stays
                          max_nan(max_nan(tops[0], tops[1], tops[2]), max_nan(tops[3], tops[4], tops[5]), max_nan(tops[6], tops[7]));
        const float lifted = chunk_base<DT>(top);
        const bool grow = lifted > __fadd_rd(m, LAZY);  // (rounded down: P stays below 2^8 as lifted)
        const bool any_grow = __any_sync(0xffffffffu, grow);
        if ((S::EARLY || any_grow) && n > n0) {  // the last V product: read P (EARLY) and wrote O
          wait(&sm.ofull[x], (n - 1) & 1);
          tmem_fence_after();
        }
        if (any_grow) {
          const float now = grow ? lifted : m, fix = grow ? ex2(m - now) : 1.f;
          if (n > n0)
#pragma unroll
            for (int j = 0; j < HD / 32; ++j) {
              uint32_t o[32];
              tmem_ld32(ot + 32 * j, o);
#pragma unroll
              for (int d = 0; d < 32; ++d) o[d] = __float_as_uint(__uint_as_float(o[d]) * fix);
              tmem_st32(ot + 32 * j, o);
            }
          l *= fix;
          m = now;
        }
        // a score that is NaN or infinite makes the row NaN (exp2_pair would take it for a weight of zero)
        if (!(top < INFINITY)) l = __int_as_float(0x7fffffff);
        const float base = m == -INFINITY ? 0.f : m;
        // Beyond 2^21 the fma's exact product is as much as a weight's exponent away from the rounded one that the maximum
        // is: the scores are rounded first, as it was (finite weights for finite scores of any size)
        uint64_t by = scale2;
        if (__any_sync(0xffffffffu, fabsf(base) > 2097152.f)) {
          by = f2(1.f, 1.f);
#pragma unroll
          for (int j = 0; j < 128; ++j) s[j >> 6][j & 63] = __float_as_uint(__uint_as_float(s[j >> 6][j & 63]) * p.scale_log2);
        }
        half_of(s[0], by, base, w, sums);
#pragma unroll
        for (int part = 0; part < 2; ++part) {
          if (part == 1) half_of(s[1], by, base, w, sums);
          tmem_st32(pt + 32 * part, w);
          tmem_wait_st();
          tmem_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&sm.pfull[x][part]);
        }
        const float2 total = unf2(add2(add2(sums[0], sums[1]), add2(sums[2], sums[3])));
        l += total.x + total.y;
        ++n;
      }
      // the tile's sums: out, or into this block's part
      const bool any = n > n0;
      if (any) {
        wait(&sm.ofull[x], (n - 1) & 1);
        tmem_fence_after();
      }
      const Segment sg = job.sg;
      const int r1 = job.r1, r = job.r0 + row, t = by_group(p, r);
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.jempty[jn % JOBS]);
      char* out = (char*)p.out + 2 * ((long long)(sg.first_row + t) * p.o_row +
                                      (long long)(sg.kvh * p.group + r - t * p.group) * p.o_head);
      auto scale_of = [&](float ls) { return over_total(p, sg.first_row + t, ls); };
      auto write = [&](const float (&o)[32], int j, float inv) {
#pragma unroll
        for (int d = 0; d < 32; d += 8)
          *reinterpret_cast<uint4*>(out + 2 * (32 * j + d)) =
              make_uint4(Half16<DT>::pack(o[d] * inv, o[d + 1] * inv), Half16<DT>::pack(o[d + 2] * inv, o[d + 3] * inv),
                         Half16<DT>::pack(o[d + 4] * inv, o[d + 5] * inv), Half16<DT>::pack(o[d + 6] * inv, o[d + 7] * inv));
      };
      constexpr int PART = CT * (HD + 2);  // [HD / 4][256 rows] float4, then (maximum, total) of each row
      auto sums_of = [&](int j, float (&o)[32]) {
        uint32_t u[32];
#pragma unroll
        for (int d = 0; d < 32; ++d) u[d] = 0u;
        if (any && ok) tmem_ld32(ot + 32 * j, u);  // warp-uniform
#pragma unroll
        for (int d = 0; d < 32; ++d) o[d] = __uint_as_float(u[d]);
      };
      if (sg.parts == 1) {
        const float inv = r <= r1 ? scale_of(l) : 0.f;
#pragma unroll
        for (int j = 0; j < HD / 32; ++j) {
          float o[32];
          sums_of(j, o);
          if (r <= r1) write(o, j, inv);
        }
        tmem_fence_before();
        continue;
      }
      const int own = blockIdx.x - sg.lead;
      auto ml_at = [&](int k) { return reinterpret_cast<float2*>(p.parts + (size_t)part_place(sg, k) * PART + CT * HD) + row; };
      auto sums_at = [&](int k, int j) {
        return reinterpret_cast<float4*>(p.parts + (size_t)part_place(sg, k) * PART) + row + 8 * j * CT;
      };
      // Adds up the parts first, first + step, ..., `count` of them, in their order, whoever is last: the same sums every
      // time. Part `mine` is still in TMEM (-1: none). emit(32 sums, j) for each 32 dims.
      auto join = [&](int first, int step, int count, int mine, float& top, float& ls, auto emit) {
        auto ml_of = [&](int k) { return k == mine ? make_float2(m, l) : __ldcg(ml_at(k)); };
        top = -INFINITY;
        ls = 0.f;
#pragma unroll 4
        for (int i = 0; i < count; ++i) top = fmaxf(top, ml_of(first + i * step).x);
        const float base = top == -INFINITY ? 0.f : top;
#pragma unroll 4
        for (int i = 0; i < count; ++i) {
          const float2 ml = ml_of(first + i * step);
          ls += ex2(ml.x - base) * ml.y;
        }
#pragma unroll 1
        for (int j = 0; j < HD / 32; ++j) {
          float acc[32];
#pragma unroll
          for (int d = 0; d < 32; ++d) acc[d] = 0.f;
#pragma unroll 2
          for (int i = 0; i < count; ++i) {
            const int k = first + i * step;
            float o[32];
            if (k == mine) {
              sums_of(j, o);
            } else {
#pragma unroll
              for (int d = 0; d < 32; d += 4) {
                const float4 v = __ldcg(sums_at(k, j) + (d / 4) * CT);
                o[d] = v.x;
                o[d + 1] = v.y;
                o[d + 2] = v.z;
                o[d + 3] = v.w;
              }
            }
            const float f = ex2(ml_of(k).x - base);
#pragma unroll
            for (int d = 0; d < 32; ++d) acc[d] += f * o[d];
          }
          emit(acc, j);
        }
      };
      auto keep = [&](int k, const float (&o)[32], int j) {
        if (r <= r1)
#pragma unroll
          for (int d = 0; d < 32; d += 4)
            __stcg(sums_at(k, j) + (d / 4) * CT, make_float4(o[d], o[d + 1], o[d + 2], o[d + 3]));
      };
      // many parts are joined in two levels, so that no block reads more than a few
      int step = 1, groups = sg.parts, mine = -1;
      if (sg.parts > JOIN_AT_ONCE)
        while (step * step < sg.parts) ++step;
      if (step == 1 && others_done(team, p.tickets + sg.lead, sg.parts, sm.words)) {
        mine = own;
      } else {
        if (!team.ok) break;
#pragma unroll
        for (int j = 0; j < HD / 32; ++j) {
          float o[32];
          sums_of(j, o);
          keep(own, o, j);
        }
        if (r <= r1) __stcg(ml_at(own), make_float2(m, l));
        if (step > 1) {
          const int first = own / step * step, count = min(step, sg.parts - first);
          if (!last_of(team, p.tickets + p.slots + part_place(sg, first), count, sm.words)) {
            tmem_fence_before();
            if (!team.ok) break;
            continue;
          }
          if (__any_sync(0xffffffffu, r <= r1)) {
            // the sums take the place of the group's first part, each thread's behind its own reads of it
            float top, ls;
            join(first, 1, count, -1, top, ls, [&](const float (&o)[32], int j) { keep(first, o, j); });
            if (r <= r1) __stcg(ml_at(first), make_float2(top, ls));
          }
          groups = ceil_div(sg.parts, step);
        }
        if (!last_of(team, p.tickets + sg.lead, groups, sm.words)) {
          tmem_fence_before();
          if (!team.ok) break;
          continue;
        }
      }
      if (__any_sync(0xffffffffu, r <= r1)) {
        float top, ls;
        join(0, step, groups, mine, top, ls, [&](const float (&o)[32], int j) {
          if (r <= r1) write(o, j, scale_of(ls));
        });
      }
      tmem_fence_before();
    }
    if (!(ok && team.ok) && lane == 0) atomicCAS(p.error, 0, 0x214);
    tmem_fence_before();
  }
  __syncthreads();
  if (warp == 9) {
    wait_bounded(&sm.done, 0, p.timeout_ns);  // no MMA may still write
    tmem_fence_after();
    tmem_free(tmem, 512);
  }
}

// ---- host ----------------------------------------------------------------------------------------
// L2 takes in the bytes that a row of one head has, no more: at head_dim 64 with 256 bytes the neighbouring head's
// row comes along, and may be gone before its block gets there (10 rows of 128 episodes 45.5 instead of 42.8 us, 32
// single rows after 2000 44.4 instead of 42.3); at 128 with 128 bytes the two halves come apart (16 single rows after
// 12,500 140.2 instead of 134.7 us).
bool encode_pages(CUtensorMap* m, const void* base, int dtype, int head_dim, int page_rows, int kv_heads, int pages,
                  long long row, long long head, long long page, int box_rows) {
  EncodeTiledFn fn = tensor_map_encoder();
  if (!fn) return false;
  const cuuint64_t dims[4] = {(cuuint64_t)head_dim, (cuuint64_t)page_rows, (cuuint64_t)kv_heads, (cuuint64_t)pages};
  // a dim of size one has no stride of its own
  const cuuint64_t strides[3] = {(cuuint64_t)row * 2, (cuuint64_t)(kv_heads > 1 ? head : head_dim) * 2,
                                 (cuuint64_t)(pages > 1 ? page : head_dim) * 2};
  const cuuint32_t box[4] = {64, (cuuint32_t)box_rows, 1, 1};
  const cuuint32_t estr[4] = {1, 1, 1, 1};
  return fn(m, dtype == MKX_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
            const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            head_dim == 64 ? CU_TENSOR_MAP_L2_PROMOTION_L2_128B : CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

struct Plan {
  bool chunk;
  int kt;     // key blocks
  int slots;  // blocks of the grid
  size_t bytes;
};

// rows_kernel's time goes with the (16 rows) x keys of all tiles, chunk_kernel's with the (256 rows) x (128 keys), and it
// has more to do around a tile; measured in us (head_dim 64 / 128): a block 1.43 / 1.7 on one of the SMs and 4.5 around a
// tile against 59 / 79 a million keys of a 16-row tile on the whole GPU, 25 against 8 for the launch, and 20 more where so
// few tiles share the SMs that parts are joined twice. How long the caches are is not known here: what the tables can hold
// stands for it. Beyond one 16-row tile, rows_kernel against chunk_kernel (us; episodes x rows per K/V head after keys, K/V
// heads, head_dim): 1 x 32 after 4000, 12, 64: 13.8, 23.0; 1 x 64 after 4000: 14.3, 23.3; after 40000: 57.2, 54.1; 128 x 20
// after 500: 71, 107; 64 x 32 after 4000: 291, 226; 8 x 32 after 8000, 8, 128: 97, 76; 1 x 32 after 100000, 1: 30, 61.
bool chunk_is_faster(const mkx_attend_inputs& a, long long rows) {
  double keys = (double)a.table_width * a.page_rows;
  if (a.window > 0 && (double)a.window + a.sinks + a.max_rows < keys) keys = (double)a.window + a.sinks + a.max_rows;
  const double heads = (double)a.B * a.kv_heads, tiles = heads * ((rows + CT - 1) / CT), sms = 148;
  const double by_rows = 8 + heads * ((rows + MT - 1) / MT) * keys * (a.head_dim == 64 ? 59e-6 : 79e-6);
  const double by_chunk = 25 + tiles / sms * (keys / CK * (a.head_dim == 64 ? 1.43 : 1.7) + 4.5) +
                          (tiles * JOIN_AT_ONCE < sms ? 20 : 0);
  return by_chunk < by_rows;
}

// The launch of a call, from sizes alone; false for sizes that are refused.
bool plan_of(const mkx_attend_inputs& a, int sms, Plan& pl) {
  if (a.rows < 0 || a.B < 1 || a.B > MKX_MAX_EPISODES || a.heads < 1 || a.kv_heads < 1 || a.heads % a.kv_heads != 0 ||
      a.pages < 1 || mkxc::page_shift(a.page_rows) < 0 || a.table_width < 1 || a.max_rows < 0 ||
      (long long)a.table_width * a.page_rows > MAX_KEYS)
    return false;
  if (a.head_dim != 64 && a.head_dim != 128) return false;
  const long long group = a.heads / a.kv_heads;
  const long long most = a.max_rows < a.rows ? a.max_rows : a.rows;
  pl.chunk = most * group > MT && chunk_is_faster(a, most * group);
  pl.kt = pl.chunk ? CK : 8192 / a.head_dim;
  pl.slots = pl.chunk ? sms : 2 * sms;
  pl.bytes = MKX_ATTEND_TICKETS * 4 + (size_t)2 * pl.slots * (pl.chunk ? CT : MT) * (a.head_dim + 2) * 4;
  return 3 * pl.slots <= MKX_ATTEND_TICKETS && (long long)a.rows * group < MAX_KEYS;
}

template <typename Kernel>
bool launch(Kernel kernel, bool (&sized)[MAX_DEVICES], int threads, int smem, const CUtensorMap& tk, const CUtensorMap& tv,
            const AttendParams& p, int device, cudaStream_t stream) {
  if (!sized[device]) {  // the attribute of a kernel is set once per device
    if (!mkxc::cuda_ok(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem))) return false;
    sized[device] = true;
  }
  return pdl_launch(kernel, p.slots, threads, smem, stream, tk, tv, p);
}
template <int DT, int HD>
bool launch_typed(bool chunk, const CUtensorMap& tk, const CUtensorMap& tv, const AttendParams& p, int device,
                  cudaStream_t stream) {
  static bool rows_sized[MAX_DEVICES] = {}, chunk_sized[MAX_DEVICES] = {};
  return chunk ? launch(chunk_kernel<DT, HD>, chunk_sized, CHUNK_THREADS, (int)sizeof(ChunkShared<HD>), tk, tv, p, device, stream)
               : launch(rows_kernel<DT, HD>, rows_sized, ROW_THREADS, RowShape<HD>::SMEM, tk, tv, p, device, stream);
}

}  // namespace
}  // namespace mkxa

using namespace mkxa;

extern "C" size_t mkx_attend_workspace(const mkx_attend_inputs* in, int device) {
  Plan pl;
  const int sms = mkxc::sm_count(device);
  return in && sms > 0 && plan_of(*in, sms, pl) ? pl.bytes : 0;
}

extern "C" mkx_status mkx_cache_attend(const mkx_attend_inputs* in, size_t workspace_bytes, int device,
                                       cudaStream_t stream) {
  if (!in) return MKX_ERR_INVALID_ARG;
  const mkx_attend_inputs a = *in;
  if (a.head_dim != 64 && a.head_dim != 128) return MKX_ERR_UNSUPPORTED;
  if (a.dtype != MKX_BF16 && a.dtype != MKX_FP16) return MKX_ERR_UNSUPPORTED;
  if (a.window < 0 || a.sinks < 0 || (a.window > 0 && !a.causal) || (a.sinks > 0 && a.window == 0) ||
      !std::isfinite(a.scale))
    return MKX_ERR_INVALID_ARG;
  if (!a.q || !a.out || !a.k_pages || !a.v_pages || !a.table || !a.length || !a.start || !a.workspace || !a.error)
    return a.rows == 0 ? MKX_OK : MKX_ERR_INVALID_ARG;
  const long long strides[] = {a.q_row, a.q_head, a.o_row, a.o_head, a.kp_page, a.kp_row, a.kp_head,
                               a.vp_page, a.vp_row, a.vp_head};
  for (long long s : strides)
    if (s < 0 || s % 8 != 0 || s >= (1ll << 38)) return MKX_ERR_INVALID_ARG;
  // a tensor map's strides are not zero
  if ((a.pages > 1 && (a.kp_page == 0 || a.vp_page == 0)) || a.kp_row == 0 || a.vp_row == 0 ||
      (a.kv_heads > 1 && (a.kp_head == 0 || a.vp_head == 0)))
    return MKX_ERR_INVALID_ARG;
  const void* pointers[] = {a.q, a.out, a.k_pages, a.v_pages, a.workspace};
  for (const void* q : pointers)
    if ((reinterpret_cast<uintptr_t>(q) & 15) != 0) return MKX_ERR_INVALID_ARG;
  DeviceScope scope(device);
  if (!mkxc::cuda_ok(scope.err)) return MKX_ERR_CUDA;
  const int sms = mkxc::sm_count(device);
  if (sms == 0) return MKX_ERR_CUDA;
  Plan pl;
  if (!plan_of(a, sms, pl) || workspace_bytes < pl.bytes) return MKX_ERR_INVALID_ARG;
  if (a.rows == 0 || a.max_rows == 0) return MKX_OK;
  const int box = a.page_rows < pl.kt ? a.page_rows : pl.kt;
  CUtensorMap tk, tv;
  if (!encode_pages(&tk, a.k_pages, a.dtype, a.head_dim, a.page_rows, a.kv_heads, a.pages, a.kp_row, a.kp_head,
                    a.kp_page, box) ||
      !encode_pages(&tv, a.v_pages, a.dtype, a.head_dim, a.page_rows, a.kv_heads, a.pages, a.vp_row, a.vp_head,
                    a.vp_page, box)) {
    mkxc::last_error = "cuTensorMapEncodeTiled failed";
    return MKX_ERR_CUDA;
  }
  AttendParams p;
  memset(&p, 0, sizeof(p));
  p.q = a.q;
  p.out = a.out;
  p.table = a.table;
  p.length = a.length;
  p.start = a.start;
  p.tickets = static_cast<unsigned*>(a.workspace);
  p.parts = reinterpret_cast<float*>(static_cast<char*>(a.workspace) + MKX_ATTEND_TICKETS * 4);
  p.error = a.error;
  p.q_row = a.q_row;
  p.q_head = a.q_head;
  p.o_row = a.o_row;
  p.o_head = a.o_head;
  p.rows = a.rows;
  p.B = a.B;
  p.heads = a.heads;
  p.kv_heads = a.kv_heads;
  p.group = a.heads / a.kv_heads;
  p.group_shift = (p.group & (p.group - 1)) == 0 ? __builtin_ctz(p.group) : -1;
  p.pages = a.pages;
  p.shift = mkxc::page_shift(a.page_rows);
  p.table_width = a.table_width;
  p.max_rows = a.max_rows;
  p.causal = a.causal != 0;
  p.window = a.window < MAX_KEYS ? a.window : MAX_KEYS;
  p.sinks = a.sinks < MAX_KEYS ? a.sinks : MAX_KEYS;
  p.scale_log2 = a.scale == 0.f ? 1.f : (float)(std::fabs((double)a.scale) * 1.4426950408889634);
  p.q_and = a.scale == 0.f ? 0u : ~0u;
  p.q_xor = a.scale < 0.f ? 0x80008000u : 0u;
  p.slots = pl.slots;
  p.min_shift = 1;
  p.snap = 2;
  p.timeout_ns = 2000000000ull;
  const bool ok =
      a.head_dim == 64
          ? (a.dtype == MKX_BF16 ? launch_typed<MKX_BF16, 64>(pl.chunk, tk, tv, p, device, stream)
                                 : launch_typed<MKX_FP16, 64>(pl.chunk, tk, tv, p, device, stream))
          : (a.dtype == MKX_BF16 ? launch_typed<MKX_BF16, 128>(pl.chunk, tk, tv, p, device, stream)
                                 : launch_typed<MKX_FP16, 128>(pl.chunk, tk, tv, p, device, stream));
  return ok ? MKX_OK : MKX_ERR_CUDA;
}
