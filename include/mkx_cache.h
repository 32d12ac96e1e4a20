/* C ABI of the paged episode cache on sm_100a: placing the new rows of many episodes (block tables and
 * slot maps), storing their K and V rows (with rotary positions of several axes), and attention of new
 * rows over the pages. No counterpart in the reference, whose K/V are dense per episode
 * (src/mk_expert.py:486-495).
 *
 * A cache is a pool of `pages` pages of `page_rows` rows (a power of two, 16 .. 256), each row one
 * [kv_heads][head_dim] vector of K and one of V. Slot s is row s % page_rows of page s / page_rows. An
 * episode's row j lies in page table[episode][j / page_rows]. All pointers are device pointers of
 * `device`; 16-bit arrays are bf16 or fp16 bit patterns. Strides are in elements. Every call is
 * asynchronous on `stream` (a stream of `device`), can be captured, makes `device` current for the call
 * and restores the caller's device. Status codes are those of mkx.h. */
#ifndef MKX_CACHE_H
#define MKX_CACHE_H

#include <stddef.h>
#include <stdint.h>
#include <cuda_runtime_api.h>
#include "mkx.h"

#ifdef __cplusplus
extern "C" {
#endif

#define MKX_BF16 0
#define MKX_FP16 1
#define MKX_MAX_EPISODES 4096
#define MKX_MAX_AXES 4

/* Places new_rows[b] rows behind the length[b] rows that episode b holds. Episodes take the pages they
 * need from the ring of free pages, in order; pages are granted while the ring holds some, and up to
 * table_width per episode.
 *   marks[0], marks[1]  pages ever taken from / ever returned to the ring (marks[1] - marks[0] are free,
 *                       the next at ring[marks[0] % ring_pages]);
 *   marks[2]            out only: new rows that got no slot (no page left, table too narrow, or `rows`
 *                       too small).
 * Out: start[B + 1] (exclusive prefix of the new rows), and for each row its slot (-1: none), episode
 * and position in the episode; rows behind the last one get -1, -1, 0. table entries of granted pages
 * are written, all others stay. length_out and marks_out may be length and marks: then `ticket` (else it
 * may be null), a word that is zero before the first call and after each, orders reads before writes. Negative lengths
 * and marks count as 0, lengths above 2^30 as 2^30, more free pages than the ring has places as those. */
typedef struct {
  const int* length;         /* [B] */
  const int* new_rows;       /* [B] */
  int* table;                /* [B][table_width] */
  const int* ring;           /* [ring_pages] page ids */
  const long long* marks;    /* [3] */
  int* start;                /* [B + 1] */
  long long* slot;           /* [rows], 16-byte aligned, as episode and position */
  int* episode;              /* [rows] */
  int* position;             /* [rows] */
  int* length_out;           /* [B] */
  long long* marks_out;      /* [3] */
  int* ticket;
  int B, table_width, ring_pages, page_rows, rows;
} mkx_plan_inputs;

mkx_status mkx_cache_plan(const mkx_plan_inputs* in, int device, cudaStream_t stream);

/* Returns all pages of the episodes with ended[b] != 0 to the ring (behind those returned before),
 * sets their length to 0 and their table entries to -1. */
typedef struct {
  const unsigned char* ended; /* [B] */
  int* length;                /* [B] */
  int* table;                 /* [B][table_width] */
  int* ring;                  /* [ring_pages] */
  long long* marks;           /* [3] */
  int* ticket;                /* as above */
  int B, table_width, ring_pages, page_rows;
} mkx_release_inputs;

mkx_status mkx_cache_release(const mkx_release_inputs* in, int device, cudaStream_t stream);

/* Rotary positions with one to four axes. Frequency i of `half` = sum(sections) turns dims i and
 * i + half of a head by positions[axis(i)] * base^(-i / half); dims from 2 * half on pass through.
 * axis(i): runs of sections[a] frequencies per axis, or (interleaved) the axes in turn while each has
 * some left. `half` is a multiple of 8, 2 * half <= head_dim. */
typedef struct {
  double base;
  int axes;
  int sections[MKX_MAX_AXES];
  int interleaved;
} mkx_rotary;

/* cos, sin [rows][head_dim] fp32 of positions [axes][rows] int32 (axis stride pos_stride); dims that pass
 * through get 1 and 0. head_dim a multiple of 16, <= 256. mkx_prep_run and mkx_run read this layout, but turn
 * dims i and i + head_dim / 2 together: tables for them have half = head_dim / 2. */
mkx_status mkx_rope_tables(const mkx_rotary* rot, const int* positions, long long pos_stride, int rows, int head_dim,
                           float* cos, float* sin, int device, cudaStream_t stream);

/* Stores rows k, v [rows][kv_heads][head_dim] at slot[row] (outside 0 .. pages * page_rows - 1: not
 * stored). With `positions`, k is rotated first, and q [rows][heads][head_dim] (may be null) is rotated
 * into q_out. One rounding at the end, the rotation in fp32. Rows, heads and pages have the given
 * strides (multiples of 8), dims are contiguous, pointers 16-byte aligned. Two rows with the same slot:
 * one of them is stored, possibly mixed. */
typedef struct {
  const void *q, *k, *v;
  void *q_out, *k_pages, *v_pages;
  const long long* slot;
  const int* positions;     /* [axes][rows], or null: nothing is rotated */
  long long pos_stride;
  long long q_row, q_head, k_row, k_head, v_row, v_head, qo_row, qo_head;
  long long kp_page, kp_row, kp_head, vp_page, vp_row, vp_head;
  int rows, heads, kv_heads, head_dim, dtype, pages, page_rows;
  mkx_rotary rot;           /* read when positions is not null */
} mkx_store_inputs;

mkx_status mkx_cache_store(const mkx_store_inputs* in, int device, cudaStream_t stream);

/* Attention of the new rows over the pages. Rows start[b] .. start[b + 1] - 1 of q are the last ones of
 * the length[b] rows of episode b: row t has position p = length[b] - (start[b + 1] - start[b]) + t and
 * sees the rows j < length[b] with (not causal, or j <= p) and (window == 0, or j > p - window, or
 * j < sinks):
 *   out[row, h] = sum_j softmax_j(scale * q[row, h] . k[j, h / group]) v[j, h / group],  group = heads / kv_heads
 * and zero where a row sees nothing. Scores, maxima and sums are held in fp32, outputs rounded once; the
 * probabilities exp(score - maximum) enter the second product as two 16-bit words (2^-16 of each in bf16, 2^-22 in
 * fp16) or, in the kernel of long chunks, as one (2^-8, 2^-11; the sum that they are divided by is of the unrounded
 * ones). Which of the two a call of more than 16 rows of a K/V head takes goes by max_rows and table_width, so the same
 * row may differ in its last bits between calls that differ in those; the same call repeats itself. What a
 * K/V page holds beyond an episode's length, and pages that no row sees, do not matter, whatever they
 * hold; K and V rows below the length are finite. Table entries outside 0 .. pages - 1 read as zero rows.
 * A row of a head that sees a score of NaN or +inf, or only scores of -inf, is NaN there.
 * Rows behind start[B] are left as they were. head_dim 64 or 128; window > 0 only with causal.
 * max_rows: no episode has more new rows in this call (more: those behind are left as they were).
 *
 * workspace: mkx_attend_workspace() bytes, of which the first MKX_ATTEND_TICKETS * 4 are zero before
 * the first call (each call leaves them zero); one call at a time per workspace. error: one word, zero
 * at first, set when a bounded wait ran out (outputs are then not to be used); calls may share it. */
#define MKX_ATTEND_TICKETS 4096
typedef struct {
  const void *q, *k_pages, *v_pages;
  void* out;
  const int *table, *length, *start;
  void* workspace;
  int* error;
  long long q_row, q_head, o_row, o_head;
  long long kp_page, kp_row, kp_head, vp_page, vp_row, vp_head;
  int rows, B, heads, kv_heads, head_dim, dtype, pages, page_rows, table_width, max_rows;
  int causal, window, sinks;
  float scale;
} mkx_attend_inputs;

mkx_status mkx_cache_attend(const mkx_attend_inputs* in, size_t workspace_bytes, int device, cudaStream_t stream);

/* Bytes of workspace that a call with these sizes needs (0 for sizes that are refused). */
size_t mkx_attend_workspace(const mkx_attend_inputs* in, int device);

/* MKX_CACHE_KEY as the library was built with: a number that the build derives from this header. A caller that was built
 * apart and hands structs over compares it with its own (0: built without). */
#ifndef MKX_CACHE_KEY
#define MKX_CACHE_KEY 0ull
#endif
unsigned long long mkx_cache_key(void);

/* Last CUDA error string seen by the cache entry points (thread-local, static storage). */
const char* mkx_cache_last_cuda_error(void);

#ifdef __cplusplus
}
#endif
#endif
