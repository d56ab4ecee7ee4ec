// Attention of ragged batches of query rows over a paged (or contiguous) KV cache: what the kernels of
// this family share.  Request r brings n_r new tokens that stand at positions seq_r - n_r ... seq_r - 1
// of its sequence; the query at position p sees the keys
//     j <= p   and   (no window,  j > p - window,  or  j < sinks)   and   j's page is present,
// o = softmax(scale * q k^T) v over the seen keys, zeros if there is none.
//
// Work is cut twice.  An ITEM is a tile of packed query rows (tile_tokens consecutive tokens x the query
// heads that share a KV head, row = token * chunk_heads + head) of one request and one KV head; its cost is the
// number of UNITS (unit_keys consecutive keys) that any of its rows sees.  All units of all items form
// one line, which is cut into equal pieces, one per CTA: a CTA runs through the end of one item, whole
// items, and the start of another.  Whole items are written to the output, the two broken ones leave
// their partial (max, sum, unnormalised output) behind and a second kernel joins them.  The load is even
// whatever the lengths are, nothing about them is needed on the host, and the scratch is two tiles per CTA.
#pragma once

#include <cuda_fp16.h>

#include "spf_internal.cuh"

namespace spf {

struct RaggedParams {
  const void* q; int64_t q_sn, q_sh;
  const void* k; int64_t k_sp, k_st, k_sh;   // strides of a page, a token of a page, a KV head
  const void* v; int64_t v_sp, v_st, v_sh;
  void* out;                                 // [n_rows][H][D]
  const int32_t* table; int64_t table_stride;  // [R][table_width]; nullptr: contiguous keys (one request)
  int table_width, n_pages, page_shift;
  const int32_t* cu; const int32_t* seq;     // [R + 1], [R]; nullptr: one request of n_rows tokens, seq_one keys
  int n_requests, n_rows, seq_one;
  int n_q_heads, n_kv_heads, group;
  int window, sinks;                         // window 0: none
  float scale_log2;
  int fp16;
  // how the work is cut
  int head_chunks, chunk_heads;              // a KV head's group as head_chunks pieces of at most chunk_heads heads
  int stream_rows, stream_tokens;            // an item's rows come in streams (one MMA tile each) of stream_tokens tokens
  int tile_rows, tile_tokens, unit_keys, n_ctas;   // tile_rows / stream_rows streams an item
  char* scratch;
};

// where a CTA starts (written by the schedule kernel; tile: in the line's order); units: what it runs through, 0 if it has no work
// taken: units of its first item that the CTA runs through in which the item starts
struct RaggedStart { int req, head, tile, first, units, item_units, taken, pad; };

// units of one item: [0, sink_units) and then [win_first, win_first + total - sink_units)
struct RaggedSpan { int total, sink_units, win_first, keys; };   // keys: exclusive end of the keys in view

// scratch: where the CTAs start, a stride per request, two partial tiles per CTA
__host__ __device__ inline int ragged_starts_bytes(int n_ctas) { return (n_ctas * int(sizeof(RaggedStart)) + 255) & ~255; }
__host__ __device__ inline int ragged_head_bytes(int n_ctas) { return ragged_starts_bytes(n_ctas) + SPF_MAX_REQUESTS * 4; }
__host__ __device__ inline int64_t ragged_partial_floats(int tile_rows, int head_dim) { return int64_t(tile_rows) * (head_dim + 2); }
inline int64_t ragged_scratch_bytes(int n_ctas, int tile_rows, int head_dim) {
  return ragged_head_bytes(n_ctas) + 2 * n_ctas * ragged_partial_floats(tile_rows, head_dim) * 4;
}

#ifdef __CUDACC__
// first packed row, new tokens, sequence length (whatever the arrays hold, rows stay in the batch); stride of its tiles
struct RaggedReq { int row0, n, seq, stride; };

// `strides`: the schedule has been made
__device__ __forceinline__ RaggedReq ragged_req(const RaggedParams& p, int r, bool strides = true) {
  RaggedReq q;
  q.stride = strides && p.window > 0 ? reinterpret_cast<const int32_t*>(p.scratch + ragged_starts_bytes(p.n_ctas))[r] : 1;
  if (p.cu == nullptr) {
    q.row0 = 0; q.n = p.n_rows; q.seq = p.seq_one;
  } else {
    const int a = min(max(__ldg(p.cu + r), 0), p.n_rows), b = min(max(__ldg(p.cu + r + 1), a), p.n_rows);
    q.row0 = a; q.n = b - a; q.seq = min(max(__ldg(p.seq + r), 0), SPF_MAX_KEYS);
  }
  return q;
}

__device__ __forceinline__ int ragged_tiles(const RaggedParams& p, int n) { return (n + p.tile_tokens - 1) / p.tile_tokens; }

// Tile `at` of a request's part of the line.  With a window a tile's keys are near its tokens only, and CTAs that run at
// the same time should be at neighbouring tiles: `stride`, the tiles that a CTA runs through, makes the line go
// through the tiles by columns of a table of that many columns, so that the CTAs' n-th tiles lie side by side.
// (Without it a 32K prompt of 32 heads with a 2K window read its 134 MB of K and V 27 times from HBM: 3.6 GB.)
__device__ __forceinline__ int ragged_place(const RaggedParams& p, const RaggedReq& q, int at) {
  if (q.stride <= 1) return at;
  const int tiles = ragged_tiles(p, q.n), rows = (tiles + q.stride - 1) / q.stride, full = tiles - (rows - 1) * q.stride;
  const int row = at / q.stride, col = at - row * q.stride;       // columns up to `full` have `rows` tiles, the others one less
  return col * rows - max(col - full, 0) + row;
}

__device__ __forceinline__ RaggedSpan ragged_span(const RaggedParams& p, const RaggedReq& q, int at) {
  const int tile = ragged_place(p, q, at);
  const int t0 = tile * p.tile_tokens, t1 = min(t0 + p.tile_tokens, q.n);
  const int first_pos = q.seq - q.n + t0;
  int64_t end = q.seq - q.n + t1;
  if (p.table != nullptr) end = min(end, int64_t(p.table_width) << p.page_shift);
  RaggedSpan s;
  s.keys = int(max(end, int64_t(0)));
  const int low = p.window > 0 ? max(first_pos - p.window + 1, 0) : 0;
  const int end_unit = (s.keys + p.unit_keys - 1) / p.unit_keys;
  s.win_first = min(low / p.unit_keys, end_unit);
  s.sink_units = min(p.sinks / p.unit_keys + (p.sinks % p.unit_keys != 0), s.win_first);
  s.total = max(s.sink_units + end_unit - s.win_first, 1);   // an item that sees nothing still has zeros to write
  return s;
}

// the item after (req, head, tile); false behind the last one
__device__ __forceinline__ bool ragged_next(const RaggedParams& p, int& req, int& head, int& tile, RaggedReq& q) {
  if (++tile < ragged_tiles(p, q.n)) return true;
  tile = 0;
  if (++head < p.n_kv_heads * p.head_chunks) return true;
  head = 0;
  while (++req < p.n_requests) {
    q = ragged_req(p, req);
    if (q.n > 0) return true;
  }
  return false;
}

// an item's place in the tensors
struct RaggedItem { int kvh, h0, heads, tok0, n_tok, pos0; };   // first head of the chunk (in its group), heads and tokens there are
__device__ __forceinline__ RaggedItem ragged_item(const RaggedParams& p, const RaggedReq& q, int head, int at) {
  RaggedItem t;
  t.kvh = head / p.head_chunks;
  t.h0 = (head - t.kvh * p.head_chunks) * p.chunk_heads;
  t.heads = min(p.chunk_heads, p.group - t.h0);
  t.tok0 = ragged_place(p, q, at) * p.tile_tokens;
  t.n_tok = min(p.tile_tokens, q.n - t.tok0);
  t.pos0 = q.seq - q.n + t.tok0;
  return t;
}
// offset of (token of the item, head of the chunk) in `out`, in elements
__device__ __forceinline__ int64_t ragged_out(const RaggedParams& p, const RaggedReq& q, const RaggedItem& t, int tok, int h, int d) {
  return ((int64_t(q.row0) + t.tok0 + tok) * p.n_q_heads + t.kvh * p.group + t.h0 + h) * d;
}
__device__ __forceinline__ float* ragged_part(const RaggedParams& p, int cta, int which, int d) {
  return reinterpret_cast<float*>(p.scratch + ragged_head_bytes(p.n_ctas)) +
         (2 * int64_t(cta) + which) * ragged_partial_floats(p.tile_rows, d);
}

template <bool FP16>
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  if (FP16) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
#endif  // __CUDACC__

int ragged_schedule(const RaggedParams& p, cudaStream_t st);
int ragged_merge(const RaggedParams& p, int head_dim, cudaStream_t st);
// up to 16 packed rows an item: bandwidth bound (single tokens); also what TMA cannot describe
void ragged_rows_config(RaggedParams& p);
int ragged_rows_attention(const RaggedParams& p, int head_dim, cudaStream_t st);
// items of two 128-row MMA tiles on tcgen05 (spf_ragged_tc5.cu); SPF_ERR_SHAPE where TMA cannot describe the tensors
void ragged_tc5_config(RaggedParams& p);
bool ragged_tc5_describable(const RaggedParams& p);
int ragged_tc5_attention(const RaggedParams& p, int head_dim, cudaStream_t st);
unsigned int ragged_tc5_timeout_count();
bool ragged_tc5_reset_timeouts();
bool ragged_tc5_set_wait_limit(unsigned long long ns);

}  // namespace spf
