// Attention of new rows over the paged episode cache (include/mkx_cache.h).
//
// rows_kernel: tiles of 16 rows (new row x head of the group that shares a K/V head). With few rows a
// call is bound by reading the pages: one producer warp keeps a ring of K/V blocks in flight by TMA (one
// box per page, 128-byte swizzle, pages that no row sees read as zero without touching memory), four
// warps each take a quarter of a block's keys with mma.sync m16n8k16 and keep their own running
// maximum and sum, joined once at the end; long caches are split over blocks (find_share), the last
// part to finish joins the tile in the order of the parts. The probabilities enter the second product
// as the sum of two 16-bit words, so that it is as exact as fp32 weights; the tensor pipe is idle
// enough for that here.
#include <cmath>
#include <cstdint>
#include <cstring>
#include <cuda.h>
#include <cuda_runtime.h>

#include "mkx_attend.cuh"
#include "mkx_cache_host.h"

namespace mkxa {
namespace {

constexpr int MT = 16;
using mkxc::MAX_DEVICES;
constexpr int MAX_KEYS = 1 << 30;  // rows of an episode: keys and positions are 32-bit
constexpr int ROW_WARPS = 4;
constexpr int ROW_THREADS = 32 * (ROW_WARPS + 1);
constexpr int ROW_STAGES = 3;

template <int HD>
struct RowShape {
  static constexpr int KT = 8192 / HD;               // keys per block: 16 KB of K, 16 KB of V
  static constexpr int KW = KT / ROW_WARPS;          // keys of a warp
  static constexpr int HALF = KT * 128;              // bytes of a 64-dim half of K or V
  static constexpr int STAGE = 2 * KT * HD * 2;
  static constexpr int SMEM = ROW_STAGES * STAGE + 1024 + 256;
};

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
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void row_barrier() { asm volatile("bar.sync 1, %0;" ::"n"(32 * ROW_WARPS) : "memory"); }

extern __shared__ __align__(1024) char asmem[];

template <int DT, int HD>
__global__ void __launch_bounds__(ROW_THREADS)
    rows_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
                const __grid_constant__ AttendParams p) {
  using S = RowShape<HD>;
  constexpr int KT = S::KT, KW = S::KW;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  char* ring = asmem + ((1024u - (smem_u32(asmem) & 1023u)) & 1023u);
  uint64_t* full = reinterpret_cast<uint64_t*>(ring + ROW_STAGES * S::STAGE);
  uint64_t* empty = full + ROW_STAGES;
  if (threadIdx.x == 0) {
    for (int s = 0; s < ROW_STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], ROW_WARPS);
    }
    fence_mbar_init();
  }
  Share sh;
  if (!find_share<MT, KT, ROW_THREADS>(p, blockIdx.x, sh)) return;  // its barriers publish the mbarriers too
  const int total = sh.fresh * p.group, r0 = sh.tile * MT, r1 = min(r0 + MT, total) - 1;
  const Keys ks = keys_of<KT>(p, sh, r0, r1);
  const int i0 = (int)((long long)ks.blocks * sh.split / sh.splits);
  const int i1 = (int)((long long)ks.blocks * (sh.split + 1) / sh.splits);

  if (warp == ROW_WARPS) {
    // producer: lane j fetches the j-th page of each block
    const int rows_box = min(1 << p.shift, KT), boxes = KT / rows_box;
    int id = -1;
    auto page_at = [&](int i) {
      return lane < boxes ? page_of(p, ks, sh.b, (block_key<KT>(ks, i) >> p.shift) + lane) : -1;
    };
    if (i0 < i1) id = page_at(i0);
    bool ok = true;
    int issued = i0;
    for (int i = i0; i < i1; ++i) {
      const int n = i - i0, s = n % ROW_STAGES;
      const int next = i + 1 < i1 ? page_at(i + 1) : -1;
      if (n >= ROW_STAGES && !wait_bounded(&empty[s], ((n / ROW_STAGES) & 1) ^ 1, p.timeout_ns)) {
        atomicCAS(p.error, 0, 0x201);
        ok = false;
      }
      if (!__all_sync(0xffffffffu, ok)) break;
      if (lane == 0) mbar_expect_tx(&full[s], (uint32_t)S::STAGE);
      __syncwarp();
      if (lane < boxes) {
        const int row = block_key<KT>(ks, i) & ((1 << p.shift) - 1);
        char* at = ring + s * S::STAGE + lane * rows_box * 128;
#pragma unroll
        for (int h = 0; h < HD / 64; ++h) {
          tma_load_4d(at + h * S::HALF, &tk, 64 * h, boxes > 1 ? 0 : row, sh.kvh, id, &full[s]);
          tma_load_4d(at + KT * HD * 2 + h * S::HALF, &tv, 64 * h, boxes > 1 ? 0 : row, sh.kvh, id, &full[s]);
        }
      }
      issued = i + 1;
      id = next;
    }
    if (lane == 0 && issued < i1)  // a wait ran out: let what is in flight land before the block ends
      for (int i = max(i0, issued - ROW_STAGES); i < issued; ++i)
        wait_bounded(&full[(i - i0) % ROW_STAGES], ((i - i0) / ROW_STAGES) & 1, p.timeout_ns);
    return;
  }

  // queries: A fragments of the 16 rows, read once
  const int g = lane >> 2, c = lane & 3;
  uint32_t qf[HD / 16][4];
  int pos[2];
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const int r = r0 + g + 8 * x;
    const bool live = r <= r1;
    const int t = r / p.group;
    pos[x] = sh.past + t;
    const char* q = (const char*)p.q + 2 * ((long long)(sh.first_row + t) * p.q_row +
                                            (long long)(sh.kvh * p.group + r - t * p.group) * p.q_head);
#pragma unroll
    for (int kk = 0; kk < HD / 16; ++kk) {
      qf[kk][x] = live ? __ldg(reinterpret_cast<const uint32_t*>(q + 32 * kk + 4 * c)) : 0u;
      qf[kk][x + 2] = live ? __ldg(reinterpret_cast<const uint32_t*>(q + 32 * kk + 16 + 4 * c)) : 0u;
    }
  }
  float o[HD / 8][4];
#pragma unroll
  for (int n = 0; n < HD / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  // ldmatrix: lane's row and 16-byte chunk of the four 8x8 parts
  const int krow = (lane & 7) + ((lane >> 4) << 3), kchunk = (lane >> 3) & 1;   // keys 0-7, 0-7, 8-15, 8-15
  const int vrow = (lane & 7) + (((lane >> 3) & 1) << 3), vchunk = lane >> 4;   // keys 0-7, 8-15, 0-7, 8-15
  bool ok = true;
  for (int i = i0; i < i1; ++i) {
    const int n = i - i0, s = n % ROW_STAGES;
    if (!__all_sync(0xffffffffu, wait_bounded(&full[s], (n / ROW_STAGES) & 1, p.timeout_ns))) {
      if (lane == 0) atomicCAS(p.error, 0, 0x202);
      ok = false;
      break;
    }
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
    const bool whole = whole_block<KT>(p, ks, block_key<KT>(ks, i));
    float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int j = 0; j < KW / 8; ++j)
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        float v = sc[j][x] * p.scale_log2;
        if (!whole && !sees(p, ks, pos[x >> 1], key0 + 8 * j + 2 * c + (x & 1))) v = -INFINITY;
        sc[j][x] = v;
        top[x >> 1] = fmaxf(top[x >> 1], v);
      }
    float fix[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      top[x] = fmaxf(top[x], __shfl_xor_sync(0xffffffffu, top[x], 1));
      top[x] = fmaxf(top[x], __shfl_xor_sync(0xffffffffu, top[x], 2));
      const float now = fmaxf(m[x], top[x]), safe = now == -INFINITY ? 0.f : now;
      fix[x] = ex2(m[x] - safe);
      m[x] = now;
      top[x] = safe;
      l[x] *= fix[x];
    }
#pragma unroll
    for (int n8 = 0; n8 < HD / 8; ++n8) {
      o[n8][0] *= fix[0];
      o[n8][1] *= fix[0];
      o[n8][2] *= fix[1];
      o[n8][3] *= fix[1];
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
  (void)ok;

  // join the four warps: every stage has been read, the ring is free for their sums
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    l[x] += __shfl_xor_sync(0xffffffffu, l[x], 1);
    l[x] += __shfl_xor_sync(0xffffffffu, l[x], 2);
  }
  row_barrier();
  constexpr int LD = HD + 4;
  float* os = reinterpret_cast<float*>(ring);        // [4][16][LD]
  float2* ml = reinterpret_cast<float2*>(os + ROW_WARPS * MT * LD);  // [4][16]
#pragma unroll
  for (int n8 = 0; n8 < HD / 8; ++n8) {
    *reinterpret_cast<float2*>(os + (warp * MT + g) * LD + 8 * n8 + 2 * c) = make_float2(o[n8][0], o[n8][1]);
    *reinterpret_cast<float2*>(os + (warp * MT + g + 8) * LD + 8 * n8 + 2 * c) = make_float2(o[n8][2], o[n8][3]);
  }
  if (c == 0) {
    ml[warp * MT + g] = make_float2(m[0], l[0]);
    ml[warp * MT + g + 8] = make_float2(m[1], l[1]);
  }
  row_barrier();
  // 8 threads per row, HD / 8 dims each, as float4 q, q + 8, ...
  const int row = threadIdx.x >> 3, q = threadIdx.x & 7;
  float4 acc[HD / 32];
  float mx = -INFINITY, ls = 0.f;
#pragma unroll
  for (int w = 0; w < ROW_WARPS; ++w) mx = fmaxf(mx, ml[w * MT + row].x);
  const float safe = mx == -INFINITY ? 0.f : mx;
#pragma unroll
  for (int d = 0; d < HD / 32; ++d) acc[d] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int w = 0; w < ROW_WARPS; ++w) {
    const float2 t = ml[w * MT + row];
    const float f = ex2(t.x - safe);
    ls += f * t.y;
#pragma unroll
    for (int d = 0; d < HD / 32; ++d) {
      const float4 v = *reinterpret_cast<const float4*>(os + (w * MT + row) * LD + 4 * (q + 8 * d));
      acc[d].x += f * v.x;
      acc[d].y += f * v.y;
      acc[d].z += f * v.z;
      acc[d].w += f * v.w;
    }
  }
  if (sh.splits > 1) {
    float* part = p.parts + (size_t)(sh.part + sh.split) * MT * (HD + 2);
#pragma unroll
    for (int d = 0; d < HD / 32; ++d) __stcg(reinterpret_cast<float4*>(part + row * HD + 4 * (q + 8 * d)), acc[d]);
    if (q == 0) __stcg(reinterpret_cast<float2*>(part + MT * HD) + row, make_float2(mx, ls));
    __threadfence();
    row_barrier();
    __shared__ int last;
    if (threadIdx.x == 0) {
      last = atomicAdd(p.tickets + sh.ticket, 1u) == (unsigned)sh.splits - 1;
      if (last) p.tickets[sh.ticket] = 0;
      __threadfence();
    }
    row_barrier();
    if (!last) return;
    const float* parts = p.parts + (size_t)sh.part * MT * (HD + 2);
    mx = -INFINITY;
    for (int k = 0; k < sh.splits; ++k)
      mx = fmaxf(mx, __ldcg(reinterpret_cast<const float2*>(parts + (size_t)k * MT * (HD + 2) + MT * HD) + row).x);
    const float top = mx == -INFINITY ? 0.f : mx;
    ls = 0.f;
#pragma unroll
    for (int d = 0; d < HD / 32; ++d) acc[d] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int k = 0; k < sh.splits; ++k) {
      const float* at = parts + (size_t)k * MT * (HD + 2);
      const float2 t = __ldcg(reinterpret_cast<const float2*>(at + MT * HD) + row);
      const float f = ex2(t.x - top);
      ls += f * t.y;
#pragma unroll
      for (int d = 0; d < HD / 32; ++d) {
        const float4 v = __ldcg(reinterpret_cast<const float4*>(at + row * HD + 4 * (q + 8 * d)));
        acc[d].x += f * v.x;
        acc[d].y += f * v.y;
        acc[d].z += f * v.z;
        acc[d].w += f * v.w;
      }
    }
  }
  const int r = r0 + row;
  if (r <= r1) {
    const int t = r / p.group;
    char* out = (char*)p.out + 2 * ((long long)(sh.first_row + t) * p.o_row +
                                    (long long)(sh.kvh * p.group + r - t * p.group) * p.o_head);
    const float inv = ls > 0.f ? 1.f / ls : (ls == 0.f ? 0.f : ls);  // nothing seen: zero; NaN stays
#pragma unroll
    for (int d = 0; d < HD / 32; ++d)
      *reinterpret_cast<uint2*>(out + 8 * (q + 8 * d)) =
          make_uint2(Half16<DT>::pack(acc[d].x * inv, acc[d].y * inv), Half16<DT>::pack(acc[d].z * inv, acc[d].w * inv));
  }
}

// ---- host ----------------------------------------------------------------------------------------
bool encode_pages(CUtensorMap* m, const void* base, int dtype, int head_dim, int page_rows, int kv_heads, int pages,
                  long long row, long long head, long long page, int box_rows) {
  EncodeTiledFn fn = tensor_map_encoder();
  if (!fn) return false;
  const cuuint64_t dims[4] = {(cuuint64_t)head_dim, (cuuint64_t)page_rows, (cuuint64_t)kv_heads, (cuuint64_t)pages};
  const cuuint64_t strides[3] = {(cuuint64_t)row * 2, (cuuint64_t)head * 2, (cuuint64_t)page * 2};
  const cuuint32_t box[4] = {64, (cuuint32_t)box_rows, 1, 1};
  const cuuint32_t estr[4] = {1, 1, 1, 1};
  return fn(m, dtype == MKX_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
            const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

struct Plan {
  int mt, kt, slots, max_parts;
  long long grid;
  size_t bytes;
};

// The launch of a call, from sizes alone; false for sizes that are refused.
bool plan_of(const mkx_attend_inputs& a, int sms, Plan& pl) {
  if (a.rows < 0 || a.B < 1 || a.B > MKX_MAX_EPISODES || a.heads < 1 || a.kv_heads < 1 || a.heads % a.kv_heads != 0 ||
      a.pages < 1 || mkxc::page_shift(a.page_rows) < 0 || a.table_width < 1 || a.max_rows < 0 ||
      (long long)a.table_width * a.page_rows > MAX_KEYS)
    return false;
  if (a.head_dim != 64 && a.head_dim != 128) return false;
  const long long group = a.heads / a.kv_heads;
  const long long most = a.max_rows < a.rows ? a.max_rows : a.rows;
  pl.mt = MT;
  pl.kt = 8192 / a.head_dim;
  pl.slots = 2 * sms;
  // tiles <= the rows' tiles plus one per episode, and <= episodes x the tiles of the largest
  long long tiles = (a.rows * group) / pl.mt + a.B;
  const long long by_most = a.B * ((most * group + pl.mt - 1) / pl.mt);
  if (by_most < tiles) tiles = by_most;
  pl.grid = tiles * a.kv_heads + pl.slots;
  pl.max_parts = 2 * pl.slots + 2;
  pl.bytes = MKX_ATTEND_TICKETS * 4 + (size_t)pl.max_parts * pl.mt * (a.head_dim + 2) * 4;
  return pl.grid < (1ll << 31);
}

template <int DT, int HD>
bool launch_rows(const CUtensorMap& tk, const CUtensorMap& tv, const AttendParams& p, long long grid, int device,
                 cudaStream_t stream) {
  static bool sized[MAX_DEVICES] = {};  // the attribute of this kernel is set once per device
  if (!sized[device]) {
    if (!mkxc::cuda_ok(cudaFuncSetAttribute(rows_kernel<DT, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                            RowShape<HD>::SMEM)))
      return false;
    sized[device] = true;
  }
  rows_kernel<DT, HD><<<(unsigned)grid, ROW_THREADS, RowShape<HD>::SMEM, stream>>>(tk, tv, p);
  return mkxc::cuda_ok(cudaGetLastError());
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
  p.pages = a.pages;
  p.shift = mkxc::page_shift(a.page_rows);
  p.table_width = a.table_width;
  p.max_rows = a.max_rows;
  p.causal = a.causal != 0;
  p.window = a.window < MAX_KEYS ? a.window : MAX_KEYS;
  p.sinks = a.sinks < MAX_KEYS ? a.sinks : MAX_KEYS;
  p.scale_log2 = (float)((double)a.scale * 1.4426950408889634);
  p.slots = pl.slots;
  p.min_blocks = 2;
  p.max_parts = pl.max_parts;
  p.timeout_ns = 2000000000ull;
  const bool ok = a.head_dim == 64 ? (a.dtype == MKX_BF16 ? launch_rows<MKX_BF16, 64>(tk, tv, p, pl.grid, device, stream)
                                                          : launch_rows<MKX_FP16, 64>(tk, tv, p, pl.grid, device, stream))
                                   : (a.dtype == MKX_BF16 ? launch_rows<MKX_BF16, 128>(tk, tv, p, pl.grid, device, stream)
                                                          : launch_rows<MKX_FP16, 128>(tk, tv, p, pl.grid, device, stream));
  return ok ? MKX_OK : MKX_ERR_CUDA;
}
