// Paged episode cache (include/mkx_cache.h): placing new rows, returning pages, and storing rows with
// rotary positions of several axes.
#include <cmath>
#include <cstdint>
#include <cstring>
#include <cuda_runtime.h>

#include "mkx_cache.h"
#include "mkx_cache_host.h"
#include "mkx_device.cuh"
#include "mkx_half.cuh"
#include "mkx_pdl.cuh"

namespace mkxc {
using namespace mkx;

thread_local const char* last_error = "";

bool cuda_ok(cudaError_t e) {
  if (e == cudaSuccess) return true;
  last_error = cudaGetErrorString(e);
  return false;
}

namespace {

constexpr int NT = 256;        // threads of the placing kernels
constexpr int ROWS_PER_THREAD = 4;

// Exclusive prefix of v over the block (every thread calls); `total` receives the block's sum.
__device__ __forceinline__ long long block_exclusive(long long v, long long* warp_sums, long long& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  long long inc = v;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const long long o = __shfl_up_sync(0xffffffffu, inc, d);
    if (lane >= d) inc += o;
  }
  __syncthreads();  // the previous use of warp_sums is over
  if (lane == 31) warp_sums[warp] = inc;
  __syncthreads();
  long long before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < NT / 32; ++w) {
    const long long s = warp_sums[w];
    if (w < warp) before += s;
    total += s;
  }
  return before + inc - v;
}

// ---- placing -------------------------------------------------------------------------------------
// Every block forms the two prefixes over the episodes (new rows, new pages) by itself from the B
// lengths -- a few KB out of L2 -- and then maps its own share of the rows, so one launch without any
// exchange between blocks does it all; a row's episode comes from a binary search in shared memory. The
// state (lengths, marks) is written by the last block that has read it. Latency bound: 160 rows of 16
// episodes take 6.4 us, 100,003 rows of 700 episodes (1.6 MB of output) 7.1 us, both what a call costs
// (host and launch).
constexpr int MOST_ROWS = 1 << 30;  // that a table row can stand for
struct PlanShared {
  int start;  // first row
  int past;   // rows held before
  int page0;  // first new page of the episode = ceil(past / page_rows)
  int grant;  // pages granted
};

__global__ void __launch_bounds__(NT) plan_kernel(const __grid_constant__ mkx_plan_inputs p, int shift) {
  extern __shared__ __align__(16) char raw[];
  long long* warp_sums = reinterpret_cast<long long*>(raw);
  long long* ring_at = warp_sums + 8;                       // [B] ring place of the episode's first page, mod ring
  PlanShared* ep = reinterpret_cast<PlanShared*>(ring_at + p.B);  // [B]
  __shared__ int is_last;
  pdl_begin();
  // whatever the state holds, no index leaves the ring or a table row
  const long long taken = max(p.marks[0], 0ll), returned = p.marks[1];
  const long long avail = returned > taken ? min(returned - taken, (long long)p.ring_pages) : 0;
  long long rows = 0, pages = 0, lost = 0;
  for (int b0 = 0; b0 < p.B; b0 += NT) {
    const int b = b0 + threadIdx.x;
    int past = 0, fresh = 0;
    if (b < p.B) {
      past = min(max(p.length[b], 0), MOST_ROWS);
      fresh = max(p.new_rows[b], 0);
    }
    long long total;
    const long long at = rows + block_exclusive(fresh, warp_sums, total);
    rows += total;
    const int start = (int)min(at, (long long)p.rows);
    const int fit = (int)min((long long)fresh, (long long)p.rows - start);  // rows beyond `rows` are dropped
    const long long end = (long long)past + fit;
    const int page0 = (int)(((long long)past + (1 << shift) - 1) >> shift);
    const int want = (int)min((end + (1 << shift) - 1) >> shift, (long long)p.table_width);
    const int need = max(want - page0, 0);
    const long long off = pages + block_exclusive(need, warp_sums, total);
    pages += total;
    const int grant = (int)min(max(avail - off, 0ll), (long long)need);
    const long long held = max(min(end, ((long long)page0 + grant) << shift), (long long)past);
    block_exclusive((long long)past + fresh - held, warp_sums, total);
    lost += total;
    if (b < p.B) {
      ring_at[b] = (taken + off) % p.ring_pages;
      ep[b] = PlanShared{start, past, page0, grant};
    }
  }
  __syncthreads();
  // every input of the state has been read: the last block to get here may overwrite it
  if (threadIdx.x == 0) {
    is_last = blockIdx.x == 0;  // without a ticket the state goes elsewhere, and any block may write it
    if (p.ticket) {
      __threadfence();
      is_last = atomicAdd(p.ticket, 1) == (int)gridDim.x - 1;
      if (is_last) *p.ticket = 0;
    }
  }
  __syncthreads();
  if (is_last) {
    for (int b = threadIdx.x; b < p.B; b += NT) {
      const PlanShared e = ep[b];
      const long long next = b + 1 < p.B ? ep[b + 1].start : min(rows, (long long)p.rows);
      const long long end = (long long)e.past + (next - e.start);
      p.length_out[b] = (int)max(min(end, ((long long)e.page0 + e.grant) << shift), (long long)e.past);
      p.start[b] = e.start;
    }
    if (threadIdx.x == 0) {
      p.start[p.B] = (int)min(rows, (long long)p.rows);
      p.marks_out[0] = taken + min(pages, avail);
      p.marks_out[1] = returned;
      p.marks_out[2] = lost;
    }
  }
  const int total_rows = (int)min(rows, (long long)p.rows);
  for (long long r0 = ((long long)blockIdx.x * NT + threadIdx.x) * ROWS_PER_THREAD; r0 < p.rows;
       r0 += (long long)gridDim.x * NT * ROWS_PER_THREAD) {
    long long slot[ROWS_PER_THREAD];
    int epi[ROWS_PER_THREAD], pos[ROWS_PER_THREAD];
    int b = -1;
    if (r0 < total_rows) {  // the last episode that starts at or before r0 (empty ones start there too)
      int lo = 0, hi = p.B - 1;
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (ep[mid].start <= r0) lo = mid;
        else hi = mid - 1;
      }
      b = lo;
    }
#pragma unroll
    for (int i = 0; i < ROWS_PER_THREAD; ++i) {
      const long long r = r0 + i;
      slot[i] = -1;
      epi[i] = -1;
      pos[i] = 0;
      if (r >= total_rows) continue;
      while (b + 1 < p.B && ep[b + 1].start <= r) ++b;
      const PlanShared e = ep[b];
      const unsigned at = (unsigned)e.past + (unsigned)(r - e.start);  // below 2^30 + 2^31
      const int page = (int)(at >> shift);
      int id = -1;
      if (page < e.page0) {
        if (page < p.table_width) id = p.table[(size_t)b * p.table_width + page];
      } else if (page < e.page0 + e.grant) {
        long long k = ring_at[b] + (page - e.page0);
        if (k >= p.ring_pages) k -= p.ring_pages;
        id = p.ring[k];
        if ((at & ((1 << shift) - 1)) == 0) p.table[(size_t)b * p.table_width + page] = id;
      }
      slot[i] = id < 0 ? -1 : ((long long)id << shift) + (at & ((1 << shift) - 1));
      epi[i] = b;
      pos[i] = (int)at;
    }
    if (r0 + ROWS_PER_THREAD <= p.rows) {
      *reinterpret_cast<longlong2*>(p.slot + r0) = make_longlong2(slot[0], slot[1]);
      *reinterpret_cast<longlong2*>(p.slot + r0 + 2) = make_longlong2(slot[2], slot[3]);
      *reinterpret_cast<int4*>(p.episode + r0) = make_int4(epi[0], epi[1], epi[2], epi[3]);
      *reinterpret_cast<int4*>(p.position + r0) = make_int4(pos[0], pos[1], pos[2], pos[3]);
    } else {
      for (int i = 0; i < ROWS_PER_THREAD && r0 + i < p.rows; ++i) {
        p.slot[r0 + i] = slot[i];
        p.episode[r0 + i] = epi[i];
        p.position[r0 + i] = pos[i];
      }
    }
  }
}

// ---- returning pages -----------------------------------------------------------------------------
// The same prefix over the episodes that ended; block x takes episodes x, x + grid, ...
__global__ void __launch_bounds__(NT) release_kernel(const __grid_constant__ mkx_release_inputs p, int shift) {
  extern __shared__ __align__(16) char raw[];
  long long* warp_sums = reinterpret_cast<long long*>(raw);
  int* first = reinterpret_cast<int*>(warp_sums + 8);  // [B] place among the returned pages
  int* count = first + p.B;                            // [B]
  __shared__ int is_last;
  pdl_begin();
  const long long returned = max(p.marks[1], 0ll);
  long long pages = 0;
  for (int b0 = 0; b0 < p.B; b0 += NT) {
    const int b = b0 + threadIdx.x;
    int n = 0;
    if (b < p.B && p.ended[b])
      n = (int)min(((long long)max(p.length[b], 0) + (1 << shift) - 1) >> shift, (long long)p.table_width);
    long long total;
    const long long at = pages + block_exclusive(n, warp_sums, total);
    pages += total;
    if (b < p.B) {
      first[b] = (int)(at % p.ring_pages);
      count[b] = n;
    }
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    __threadfence();
    const int n = atomicAdd(p.ticket, 1);
    is_last = n == (int)gridDim.x - 1;
    if (is_last) *p.ticket = 0;
  }
  __syncthreads();
  const long long base = returned % p.ring_pages;
  for (int b = blockIdx.x; b < p.B; b += gridDim.x) {
    if (!p.ended[b]) continue;
    int* row = p.table + (size_t)b * p.table_width;
    for (int j = threadIdx.x; j < p.table_width; j += NT) {
      if (j < count[b]) p.ring[(base + first[b] + j) % p.ring_pages] = row[j];
      row[j] = -1;
    }
  }
  if (is_last) {
    for (int b = threadIdx.x; b < p.B; b += NT)
      if (p.ended[b]) p.length[b] = 0;
    if (threadIdx.x == 0) p.marks[1] = returned + pages;
  }
}

// ---- rotary positions ----------------------------------------------------------------------------
// An angle in turns is positions * rate with the rate of one frequency split into two floats: the
// leading product is exact with its fma remainder, whole turns drop out by rint, and what is left is
// within half a turn, so cos and sin are as exact for a position of a million as for a small one
// (fp32 angles would be off by 0.03 rad there).
struct Rates {
  float hi[128], lo[128];  // rate = base^(-i / half) / (2 pi), at most half a turn
  unsigned char axis[128];
  int half;
};

__device__ __forceinline__ float turns_of(int position, float hi, float lo) {
  // a position beyond 2^24 is not a float: its low byte is turned apart
  const float a = (float)(position & ~0xff), b = (float)(position & 0xff);
  const float t = a * hi, u = b * hi;
  float r = (t - rintf(t)) + fmaf(a, hi, -t) + a * lo;
  r += (u - rintf(u)) + fmaf(b, hi, -u) + b * lo;
  return r - rintf(r);
}

__global__ void __launch_bounds__(256) tables_kernel(const __grid_constant__ Rates rates, const int* positions,
                                                     long long pos_stride, int rows, int head_dim, float* cos, float* sin) {
  // one (row, frequency or passing pair) per thread: two entries of each table
  pdl_begin();
  const int pairs = head_dim / 2;
  const long long n = (long long)rows * pairs;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) {
    const long long row = i / pairs;
    const int f = (int)(i - row * pairs);
    float2 cs = make_float2(1.f, 0.f);
    int d0 = 2 * f, d1 = 2 * f + 1;  // passing dims 2 half ..
    if (f < rates.half) {
      sincospif(2.f * turns_of(positions[rates.axis[f] * pos_stride + row], rates.hi[f], rates.lo[f]), &cs.y, &cs.x);
      d0 = f;
      d1 = f + rates.half;
    }
    cos[row * head_dim + d0] = cs.x;
    sin[row * head_dim + d0] = cs.y;
    cos[row * head_dim + d1] = cs.x;
    sin[row * head_dim + d1] = cs.y;
  }
}

// ---- storing -------------------------------------------------------------------------------------
// A thread takes 8 dims and their 8 partners (16-byte accesses) of a row for up to HG heads of one of
// q, k, v, and forms the 8 angles once for those heads. Bound by HBM: every row is read and written
// once. The angles are reduced as above, and within half a turn __cosf and __sinf are off by 2^-21 at
// most: x cos - y sin is off by 2^-21 (|x| + |y|), 2^10 times finer than half a step of fp16 at that size (a result in
// which the two nearly cancel is smaller, and off by as much); with sincospif, 20 more instructions an angle and 74
// registers, the same calls take 128 instead of 118 us (30,011 rows of 32 + 8 + 8 heads x 128, 738 MB: 6.2
// TB/s) and 10.0 instead of 8.2 (4096 rows of 3 x 12 heads x 64). With 8 heads (132 registers) they take 162 and
// 14.1 us; 2 heads and sincospif, 174 and 11.3.
constexpr int HG = 4;

template <int DT>
__global__ void __launch_bounds__(256) store_kernel(const __grid_constant__ mkx_store_inputs p,
                                                    const __grid_constant__ Rates rates, int shift, int groups_q,
                                                    int groups_k) {
  const int lanes = p.head_dim / 16;
  const int per_row = (groups_q + 2 * groups_k) * lanes;
  const long long n = (long long)p.rows * per_row;
  const long long cells = (long long)p.pages << shift;
  pdl_begin();
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) {
    const long long row = i / per_row;
    const int u = (int)(i - row * per_row);
    int group = u / lanes;
    const int c = u - group * lanes;
    const int what = group < groups_q ? 0 : group < groups_q + groups_k ? 1 : 2;
    group -= what == 0 ? 0 : what == 1 ? groups_q : groups_q + groups_k;
    const char* src;
    char* dst;
    long long src_head, dst_head;
    if (what == 0) {
      src = (const char*)p.q + 2 * row * p.q_row;
      src_head = p.q_head;
      dst = (char*)p.q_out + 2 * row * p.qo_row;
      dst_head = p.qo_head;
    } else {
      const long long slot = p.slot[row];
      if (slot < 0 || slot >= cells) continue;
      const long long page = slot >> shift, r = slot & ((1 << shift) - 1);
      src = (const char*)(what == 1 ? p.k : p.v) + 2 * row * (what == 1 ? p.k_row : p.v_row);
      src_head = what == 1 ? p.k_head : p.v_head;
      dst = what == 1 ? (char*)p.k_pages + 2 * (page * p.kp_page + r * p.kp_row)
                      : (char*)p.v_pages + 2 * (page * p.vp_page + r * p.vp_row);
      dst_head = what == 1 ? p.kp_head : p.vp_head;
    }
    const int heads = what == 0 ? p.heads : p.kv_heads;
    const int h0 = group * HG, nh = min(HG, heads - h0);
    const bool turns = what != 2 && p.positions && 8 * c < rates.half;
    // dims of this lane: 8 c and their partners, or 16 dims side by side where nothing turns
    // (the condition of `turns` in full: by that name it costs 13 registers, 125 instead of 118 us)
    int d0 = 16 * c, d1 = 16 * c + 8;
    if (what != 2 && p.positions && 8 * c < rates.half) {
      d0 = 8 * c;
      d1 = 8 * c + rates.half;
    }
    uint4 x[HG], y[HG];
#pragma unroll
    for (int h = 0; h < HG; ++h)
      if (h < nh) {
        const char* s = src + 2 * (h0 + h) * src_head;
        x[h] = __ldcs(reinterpret_cast<const uint4*>(s + 2 * d0));
        y[h] = __ldcs(reinterpret_cast<const uint4*>(s + 2 * d1));
      }
    if (turns) {
      float cs[8], sn[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int f = 8 * c + j;
        const float angle =
            6.283185307f * turns_of(p.positions[rates.axis[f] * p.pos_stride + row], rates.hi[f], rates.lo[f]);
        cs[j] = __cosf(angle);
        sn[j] = __sinf(angle);
      }
#pragma unroll
      for (int h = 0; h < HG; ++h)
        if (h < nh) {
          uint32_t* xs = reinterpret_cast<uint32_t*>(&x[h]);
          uint32_t* ys = reinterpret_cast<uint32_t*>(&y[h]);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float2 a = Half16<DT>::unpack(xs[j]), b = Half16<DT>::unpack(ys[j]);
            xs[j] = Half16<DT>::pack(fmaf(a.x, cs[2 * j], -(b.x * sn[2 * j])),
                                     fmaf(a.y, cs[2 * j + 1], -(b.y * sn[2 * j + 1])));
            ys[j] = Half16<DT>::pack(fmaf(b.x, cs[2 * j], a.x * sn[2 * j]), fmaf(b.y, cs[2 * j + 1], a.y * sn[2 * j + 1]));
          }
        }
    }
#pragma unroll
    for (int h = 0; h < HG; ++h)
      if (h < nh) {
        char* d = dst + 2 * (h0 + h) * dst_head;
        *reinterpret_cast<uint4*>(d + 2 * d0) = x[h];
        *reinterpret_cast<uint4*>(d + 2 * d1) = y[h];
      }
  }
}

// ---- host ----------------------------------------------------------------------------------------
bool same_rotary(const mkx_rotary& a, const mkx_rotary& b) {
  if (a.base != b.base || a.axes != b.axes || (a.interleaved != 0) != (b.interleaved != 0)) return false;
  for (int i = 0; i < a.axes; ++i)
    if (a.sections[i] != b.sections[i]) return false;
  return true;
}

bool rotary_fits(const mkx_rotary& r, int head_dim) {
  if (!(r.base > 0.0) || !std::isfinite(r.base) || !std::isfinite(1.0 / r.base) || r.axes < 1 || r.axes > MKX_MAX_AXES) return false;
  int half = 0;
  for (int i = 0; i < r.axes; ++i) {
    if (r.sections[i] < 0 || r.sections[i] > 128) return false;
    half += r.sections[i];
  }
  return half >= 8 && half % 8 == 0 && 2 * half <= head_dim;
}

// The frequencies of a rotary geometry (the last one is kept per thread: 64 powers per call otherwise).
const Rates& rates_of(const mkx_rotary& r) {
  static thread_local mkx_rotary known = {};
  static thread_local Rates rates = {};
  if (known.axes > 0 && same_rotary(known, r)) return rates;
  int half = 0, left[MKX_MAX_AXES] = {0, 0, 0, 0};
  for (int i = 0; i < r.axes; ++i) half += left[i] = r.sections[i];
  rates.half = half;
  int axis = 0;
  for (int i = 0; i < half; ++i) {
    if (r.interleaved) {
      while (left[axis] == 0) axis = (axis + 1) % r.axes;
    } else {
      while (left[axis] == 0) ++axis;
    }
    rates.axis[i] = (unsigned char)axis;
    --left[axis];
    if (r.interleaved) axis = (axis + 1) % r.axes;
    double rate = std::pow(r.base, -(double)i / half) / (2.0 * 3.14159265358979323846);
    rate -= std::nearbyint(rate);  // positions are whole, and so are these turns (a base below 1 has such rates)
    rates.hi[i] = (float)rate;
    rates.lo[i] = (float)(rate - (double)rates.hi[i]);
  }
  known = r;
  return rates;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace

int page_shift(int page_rows) {
  for (int s = 4; s <= 8; ++s)
    if (page_rows == 1 << s) return s;
  return -1;
}

int sm_count(int device) {
  static int known[MAX_DEVICES] = {};
  if (device < 0 || device >= MAX_DEVICES) return 0;
  if (known[device] == 0) {
    int n = 0;
    if (!cuda_ok(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device))) return 0;
    known[device] = n;
  }
  return known[device];
}

}  // namespace mkxc

using namespace mkxc;

extern "C" const char* mkx_cache_last_cuda_error(void) { return last_error; }
extern "C" unsigned long long mkx_cache_key(void) { return MKX_CACHE_KEY; }

extern "C" mkx_status mkx_cache_plan(const mkx_plan_inputs* in, int device, cudaStream_t stream) {
  if (!in) return MKX_ERR_INVALID_ARG;
  const mkx_plan_inputs p = *in;
  const int shift = page_shift(p.page_rows);
  if (!p.length || !p.new_rows || !p.table || !p.ring || !p.marks || !p.start || !p.length_out || !p.marks_out ||
      (!p.ticket && (p.length_out == p.length || p.marks_out == p.marks)) || (p.rows > 0 && (!p.slot || !p.episode || !p.position)))
    return MKX_ERR_INVALID_ARG;
  if (p.B < 1 || p.B > MKX_MAX_EPISODES || p.table_width < 1 || p.ring_pages < 1 || shift < 0 || p.rows < 0)
    return MKX_ERR_INVALID_ARG;
  if (!aligned16(p.slot) || !aligned16(p.episode) || !aligned16(p.position)) return MKX_ERR_INVALID_ARG;
  DeviceScope scope(device);
  if (!cuda_ok(scope.err)) return MKX_ERR_CUDA;
  const int sms = sm_count(device);
  if (sms == 0) return MKX_ERR_CUDA;
  const auto smem_of = [](int episodes) { return 64 + episodes * (int)(sizeof(long long) + sizeof(PlanShared)); };
  const int smem = smem_of(p.B);
  // always the largest size there is: a call's own size might fall below what another thread is about to launch with
  if (smem > 48 * 1024 && !cuda_ok(cudaFuncSetAttribute(plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                        smem_of(MKX_MAX_EPISODES))))
    return MKX_ERR_CUDA;
  long long grid = ((long long)p.rows + NT * ROWS_PER_THREAD - 1) / (NT * ROWS_PER_THREAD);
  grid = grid < 1 ? 1 : grid > sms ? sms : grid;
  return pdl_launch(plan_kernel, (int)grid, NT, smem, stream, p, shift) ? MKX_OK : MKX_ERR_CUDA;
}

extern "C" mkx_status mkx_cache_release(const mkx_release_inputs* in, int device, cudaStream_t stream) {
  if (!in) return MKX_ERR_INVALID_ARG;
  const mkx_release_inputs p = *in;
  const int shift = page_shift(p.page_rows);
  if (!p.ended || !p.length || !p.table || !p.ring || !p.marks || !p.ticket) return MKX_ERR_INVALID_ARG;
  if (p.B < 1 || p.B > MKX_MAX_EPISODES || p.table_width < 1 || p.ring_pages < 1 || shift < 0) return MKX_ERR_INVALID_ARG;
  DeviceScope scope(device);
  if (!cuda_ok(scope.err)) return MKX_ERR_CUDA;
  const int sms = sm_count(device);
  if (sms == 0) return MKX_ERR_CUDA;
  return pdl_launch(release_kernel, p.B < sms ? p.B : sms, NT, 64 + p.B * 8, stream, p, shift) ? MKX_OK : MKX_ERR_CUDA;
}

extern "C" mkx_status mkx_rope_tables(const mkx_rotary* rot, const int* positions, long long pos_stride, int rows,
                                      int head_dim, float* cos, float* sin, int device, cudaStream_t stream) {
  if (!rot || rows < 0 || (rows > 0 && (!positions || !cos || !sin))) return MKX_ERR_INVALID_ARG;
  if (head_dim < 16 || head_dim > 256 || head_dim % 16 != 0 || !rotary_fits(*rot, head_dim)) return MKX_ERR_INVALID_ARG;
  if (rows == 0) return MKX_OK;
  DeviceScope scope(device);
  if (!cuda_ok(scope.err)) return MKX_ERR_CUDA;
  const int sms = sm_count(device);
  if (sms == 0) return MKX_ERR_CUDA;
  long long grid = ((long long)rows * (head_dim / 2) + 255) / 256;
  if (grid > 8ll * sms) grid = 8ll * sms;
  return pdl_launch(tables_kernel, (int)grid, 256, 0, stream, rates_of(*rot), positions, pos_stride, rows, head_dim, cos, sin)
             ? MKX_OK
             : MKX_ERR_CUDA;
}

extern "C" mkx_status mkx_cache_store(const mkx_store_inputs* in, int device, cudaStream_t stream) {
  if (!in) return MKX_ERR_INVALID_ARG;
  const mkx_store_inputs p = *in;
  const int shift = page_shift(p.page_rows);
  if (p.rows < 0 || p.heads < 0 || p.kv_heads < 1 || p.pages < 1 || shift < 0) return MKX_ERR_INVALID_ARG;
  if (p.dtype != MKX_BF16 && p.dtype != MKX_FP16) return MKX_ERR_UNSUPPORTED;
  if (p.head_dim < 16 || p.head_dim > 256 || p.head_dim % 16 != 0) return MKX_ERR_UNSUPPORTED;
  if (p.positions && !rotary_fits(p.rot, p.head_dim)) return MKX_ERR_INVALID_ARG;
  const bool with_q = p.q != nullptr;
  if (with_q && (!p.positions || !p.q_out || p.heads < 1)) return MKX_ERR_INVALID_ARG;
  if (p.rows == 0) return MKX_OK;
  if (!p.k || !p.v || !p.k_pages || !p.v_pages || !p.slot) return MKX_ERR_INVALID_ARG;
  const long long strides[] = {p.k_row, p.k_head, p.v_row, p.v_head, p.kp_page, p.kp_row, p.kp_head,
                               p.vp_page, p.vp_row, p.vp_head, with_q ? p.q_row : 0, with_q ? p.q_head : 0,
                               with_q ? p.qo_row : 0, with_q ? p.qo_head : 0};
  for (long long s : strides)
    if (s < 0 || s % 8 != 0) return MKX_ERR_INVALID_ARG;
  const void* pointers[] = {p.k, p.v, p.k_pages, p.v_pages, with_q ? p.q : nullptr, with_q ? p.q_out : nullptr};
  for (const void* q : pointers)
    if (!aligned16(q)) return MKX_ERR_INVALID_ARG;
  DeviceScope scope(device);
  if (!cuda_ok(scope.err)) return MKX_ERR_CUDA;
  const int sms = sm_count(device);
  if (sms == 0) return MKX_ERR_CUDA;
  static const Rates none = {};
  const Rates& rates = p.positions ? rates_of(p.rot) : none;
  const int gq = with_q ? (p.heads + HG - 1) / HG : 0, gk = (p.kv_heads + HG - 1) / HG;
  long long grid = ((long long)p.rows * (gq + 2 * gk) * (p.head_dim / 16) + 255) / 256;
  if (grid > 64ll * sms) grid = 64ll * sms;
  const bool ok = pdl_launch(p.dtype == MKX_BF16 ? store_kernel<MKX_BF16> : store_kernel<MKX_FP16>, (int)grid, 256, 0, stream, p,
                             rates, shift, gq, gk);
  return ok ? MKX_OK : MKX_ERR_CUDA;
}
