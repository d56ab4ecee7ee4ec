// Attention of ragged batches of query rows over a paged (or contiguous) KV cache: what the kernels of
// this family share.  Request r brings n_r new tokens that stand at positions seq_r - n_r ... seq_r - 1
// of its sequence; the query at position p sees the keys
//     j <= p   and   (no window,  j > p - window,  or  j < sinks)   and   j's page is present,
// o = softmax(scale * q k^T) v over the seen keys, zeros if there is none.
//
// Work is cut twice.  An ITEM is a tile of packed query rows (tile_tokens consecutive tokens x the query
// heads that share a KV head, row = token * chunk_heads + head) of one request and one KV head; its cost is the
// number of UNITS (runs of 64 or 128 keys) that any of its rows sees.  All units of all items form
// one line, which is cut into equal pieces, one per CTA: a CTA runs through the end of one item, whole
// items, and the start of another.  Whole items are written to the output, the two broken ones leave
// their partial (max, sum, unnormalised output) behind and a second kernel joins them.  The load is even
// whatever the lengths are, nothing about them is needed on the host, and the scratch is two tiles per CTA.
#pragma once

#include <cuda_fp16.h>

#include "spf_internal.cuh"

namespace spf {

constexpr int RAGGED_FEW_ROWS = 16;          // tokens x heads of a KV head that the bandwidth-bound kernel takes

struct RaggedParams {
  const void* q; int64_t q_sn, q_sh;
  const void* k; int64_t k_sp, k_st, k_sh;   // strides of a page, a token of a page, a KV head
  const void* v; int64_t v_sp, v_st, v_sh;
  void* out;                                 // [n_rows][H][D]
  const int32_t* table; int64_t table_stride;  // [R][table_width]; nullptr: contiguous keys (one request)
  int table_width, n_pages, page_shift;
  const int32_t* cu; const int32_t* seq;     // [R + 1], [R]; nullptr: one request of n_rows tokens, seq_one keys
  int n_requests, n_rows, seq_one;
  int n_q_heads, n_kv_heads, group, head_dim;
  int window, sinks;                         // window 0: none
  float scale_log2;
  int fp16;
  // how the work is cut
  int head_chunks, chunk_heads;              // a KV head's group as head_chunks pieces of at most chunk_heads heads
  int stream_rows, stream_tokens;            // an item's rows come in streams (one MMA tile each) of stream_tokens tokens
  int tile_rows, tile_tokens, unit_shift, n_ctas;  // tile_rows / stream_rows streams an item; log2 of the keys of a unit
  int only;                                  // requests of this launch: 0 all, 1 those of up to 16 rows per KV head, 2 the others
  int granule;                               // keys (a power of two) at whose multiples a window's units may begin
  int copy_rows;                             // keys of one TMA copy
  int solo;                                  // bandwidth-bound kernel: a worker (of n_ctas) per warp
  int few;                                   // every CTA finds its start itself (no schedule kernel): 1 few requests and tiles,
                                             // 2 requests of one tile (what max_new says)
  char* scratch;
};

// Where a CTA starts (tile: in the line's order).  units: what it runs through, 0 if it has no work; taken: units of its
// first item that the CTA runs through in which the item starts; n_tok, heads, out: that item's tokens, heads and
// offset in the output, for the join.
struct alignas(16) RaggedStart { int req, head, tile, first, units, item_units, taken, n_tok, heads, pad; long long out; };

// Units of one item: [0, sink_units) are the keys from 0 on, of which those below sink_keys count; the others are the keys
// from win_key on, up to `keys`.  Where the last units leave room, the window begins `embed` keys earlier and the first
// `embed` columns hold the keys from 0 on instead (those below sink_keys count): four sinks cost no unit of their own.
struct RaggedSpan { int total, sink_units, win_key, keys, sink_keys, embed; };

// scratch: where the CTAs start, a stride per request, two partial tiles per CTA
__host__ __device__ inline int ragged_starts_bytes(int n_ctas) { return (n_ctas * int(sizeof(RaggedStart)) + 255) & ~255; }
__host__ __device__ inline int ragged_head_bytes(int n_ctas) { return ragged_starts_bytes(n_ctas) + SPF_MAX_REQUESTS * 4; }
__host__ __device__ inline int64_t ragged_partial_floats(int tile_rows, int head_dim) { return int64_t(tile_rows) * (head_dim + 2); }
inline int64_t ragged_scratch_bytes(int n_ctas, int tile_rows, int head_dim) {
  return ragged_head_bytes(n_ctas) + 2 * n_ctas * ragged_partial_floats(tile_rows, head_dim) * 4;
}

#ifdef __CUDACC__
// Launch behind `st`'s last kernel so that the blocks may start while that one ends; they call ragged_wait_before()
// before they read what it wrote (or return).
template <typename... A, typename... B>
inline int ragged_launch_after(void (*kernel)(A...), dim3 grid, int threads, int smem, cudaStream_t st, B... args) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr = {};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = grid; cfg.blockDim = dim3(threads); cfg.dynamicSmemBytes = size_t(smem); cfg.stream = st;
  cfg.attrs = &attr; cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
  if (e != cudaSuccess) { note_cuda_error(e); return SPF_ERR_LAUNCH; }
  return check_launch();
}
__device__ __forceinline__ void ragged_wait_before() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// Lengths, offsets, strides, queries and the block table may be what the kernel before writes while this one is already there,
// so none of them is read through the read-only path, which is for what stays the same as long as a kernel lives.  Queries and
// the table are read by plain loads, whose addresses are known behind the wait only; the others like this, so that they are not
// moved above the wait (nor past any copy: windowed 32K prompt 1158 -> 1173 us).
__device__ __forceinline__ int32_t ragged_load(const int32_t* x) {
  int32_t y;
  asm volatile("ld.global.b32 %0, [%1];" : "=r"(y) : "l"(x));
  return y;
}

// first packed row, new tokens, sequence length (whatever the arrays hold, rows stay in the batch); stride of its tiles
struct RaggedReq { int row0, n, seq, stride; };

__device__ __forceinline__ int32_t* ragged_strides(const RaggedParams& p) {
  return reinterpret_cast<int32_t*>(p.scratch + ragged_starts_bytes(p.n_ctas));
}

// request r as if its tiles were in order
__device__ __forceinline__ RaggedReq ragged_req_plain(const RaggedParams& p, int r) {
  RaggedReq q;
  q.stride = 1;
  if (p.cu == nullptr) {
    q.row0 = 0; q.n = p.n_rows; q.seq = p.seq_one;
  } else {
    const int a = min(max(ragged_load(p.cu + r), 0), p.n_rows), b = min(max(ragged_load(p.cu + r + 1), a), p.n_rows);
    q.row0 = a; q.n = b - a; q.seq = min(max(ragged_load(p.seq + r), 0), SPF_MAX_KEYS);
    if (p.only != 0 && (q.n <= RAGGED_FEW_ROWS / p.group) != (p.only == 1)) q.n = 0;
  }
  return q;
}
// `own`: the strides that this CTA found itself (shared memory), where p.few.  (A pointer to either memory instead of
// the branch made a mixed batch of 16 requests 40% slower.)
__device__ __forceinline__ RaggedReq ragged_req(const RaggedParams& p, int r, const int32_t* own) {
  RaggedReq q = ragged_req_plain(p, r);
  if (p.window > 0) {
    if (p.few == 1) q.stride = own[r]; else if (p.few == 0) q.stride = ragged_load(ragged_strides(p) + r);
  }
  return q;
}

__device__ __forceinline__ int ragged_tiles(const RaggedParams& p, int n) {
  return p.few == 2 ? n > 0 : (n + p.tile_tokens - 1) / p.tile_tokens;
}

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
  const int rest = (1 << p.unit_shift) - 1, grain = p.granule - 1;
  s.win_key = min(low, s.keys) & ~grain;
  s.sink_keys = min(p.sinks, s.win_key);
  const int win_units = (s.keys - s.win_key + rest) >> p.unit_shift;
  const int pad = (s.sink_keys + grain) & ~grain;
  s.embed = pad <= (win_units << p.unit_shift) - (s.keys - s.win_key) ? pad : 0;
  s.win_key -= s.embed;
  s.sink_units = s.embed ? 0 : (s.sink_keys + rest) >> p.unit_shift;
  s.total = max(s.sink_units + win_units, 1);   // an item that sees nothing still has zeros to write
  return s;
}

// the item after (req, head, tile); false behind the last one
__device__ __forceinline__ bool ragged_next(const RaggedParams& p, int& req, int& head, int& tile, RaggedReq& q, const int32_t* own) {
  if (++tile < ragged_tiles(p, q.n)) return true;
  tile = 0;
  if (++head < p.n_kv_heads * p.head_chunks) return true;
  head = 0;
  while (++req < p.n_requests) {
    q = ragged_req(p, req, own);
    if (q.n > 0) return true;
  }
  return false;
}

// an item's place in the tensors
struct RaggedItem { int kvh, h0, heads, tok0, n_tok, pos0; };   // first head of the chunk (in its group), heads and tokens there are
__device__ __forceinline__ RaggedItem ragged_item(const RaggedParams& p, const RaggedReq& q, int head, int at) {
  RaggedItem t;
  t.kvh = p.head_chunks == 1 ? head : head / p.head_chunks;
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

__device__ __forceinline__ long long warp_sum_ll(long long v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ long long warp_scan_ll(long long v, int lane) {   // inclusive
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  return v;
}

// 64-bit division takes some hundred instructions, and few lines need it
__device__ __forceinline__ long long div_ll(long long a, long long b) {
  if (((a | b) >> 31) == 0) return (long long)(unsigned(a) / unsigned(b));
  return a / b;
}

// Tiles of a request that a CTA runs through, rounded: `units` of one head's `tiles` tiles, `per` units per CTA.
__device__ __forceinline__ int ragged_stride(long long per, int tiles, long long units) {
  return units > 0 ? int(min(max(div_ll(2 * per * tiles + units, 2 * units), 1ll), (long long)tiles)) : 1;
}

// Where the line is cut for CTA c: `u` units into it, which lies in request `req` (q) whose units begin at `before` and
// are `a_head` per head.  One warp; the result is in every lane.
__device__ __forceinline__ RaggedStart ragged_cut(const RaggedParams& p, int req, const RaggedReq& q, long long before, long long a_head,
                                                  long long u, long long per, long long all, int lane) {
  RaggedStart s = {};
  const int tiles = ragged_tiles(p, q.n);
  s.req = req;
  s.head = int(div_ll(u - before, a_head));
  long long rem = (u - before) - a_head * s.head;
  for (int t0 = 0; t0 < tiles; t0 += 128) {          // four tiles a lane: their spans are independent, the scan is not
    const int mine = t0 + 4 * lane;
    int cost[4], sum = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      cost[i] = mine + i < tiles ? ragged_span(p, q, mine + i).total : 0;
      sum += cost[i];
    }
    int upto = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    const unsigned above = __ballot_sync(0xffffffffu, upto > rem);
    if (above) {
      const int at = __ffs(above) - 1;
      rem -= __shfl_sync(0xffffffffu, upto - sum, at);
      s.tile = t0 + 4 * at;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int c = __shfl_sync(0xffffffffu, cost[i], at);
        if (s.item_units == 0) {
          if (rem < c) { s.item_units = c; s.first = int(rem); }
          else { rem -= c; ++s.tile; }
        }
      }
      break;
    }
    rem -= __shfl_sync(0xffffffffu, upto, 31);
  }
  s.units = int(min(per, all - u));
  s.taken = s.first > 0 ? s.first - int(div_ll(s.first - 1, per) * per) : 0;
  const RaggedItem item = ragged_item(p, q, s.head, s.tile);
  s.n_tok = item.n_tok; s.heads = item.heads;
  s.out = ragged_out(p, q, item, 0, 0, p.head_dim);
  return s;
}

// The schedule of a short line (up to 32 requests, few tiles), found by one warp of every CTA for itself: a kernel less.
// Leaves the strides in `strides` [32] and, for the join, the start in the scratch.
__device__ __forceinline__ RaggedStart ragged_start_few(const RaggedParams& p, int c, int lane, int32_t* strides) {
  const int heads = p.n_kv_heads * p.head_chunks;
  RaggedReq q = {};
  q.stride = 1;
  if (lane < p.n_requests) q = ragged_req_plain(p, lane);
  const int tiles = ragged_tiles(p, q.n);
  long long sum = tiles == 1 ? ragged_span(p, q, 0).total : 0;
  for (unsigned many = __ballot_sync(0xffffffffu, tiles > 1); many; many &= many - 1) {     // the warp adds up a request's tiles
    const int r = __ffs(many) - 1;
    RaggedReq o;
    o.row0 = 0; o.stride = 1;
    o.n = __shfl_sync(0xffffffffu, q.n, r); o.seq = __shfl_sync(0xffffffffu, q.seq, r);
    const int n_tiles = ragged_tiles(p, o.n);
    int part = 0;
#pragma unroll 4
    for (int t = lane; t < n_tiles; t += 32) part += ragged_span(p, o, t).total;
    const long long all = warp_sum_ll(part);
    if (lane == r) sum = all;
  }
  const long long upto = warp_scan_ll(sum * heads, lane), all = __shfl_sync(0xffffffffu, upto, 31);
  const long long per = max(div_ll(all + p.n_ctas - 1, p.n_ctas), 1ll), u = per * c;
  if (p.window > 0) {
    q.stride = ragged_stride(per, tiles, sum);
    strides[lane] = q.stride;
  }
  RaggedStart s = {};
  if (u < all) {
    const int at = __ffs(__ballot_sync(0xffffffffu, upto > u)) - 1;
    RaggedReq o;
    o.row0 = __shfl_sync(0xffffffffu, q.row0, at);
    o.n = __shfl_sync(0xffffffffu, q.n, at); o.seq = __shfl_sync(0xffffffffu, q.seq, at); o.stride = __shfl_sync(0xffffffffu, q.stride, at);
    const long long a_head = __shfl_sync(0xffffffffu, sum, at), end = __shfl_sync(0xffffffffu, upto, at);
    s = ragged_cut(p, at, o, end - a_head * heads, a_head, u, per, all, lane);
  }
  if (lane == 0) reinterpret_cast<RaggedStart*>(p.scratch)[c] = s;
  return s;
}

// The same for requests of one tile each (single tokens; a decode batch of 64 requests up to 8K: 226 us with the schedule
// kernel, 218 without): a lane adds up the units of its run of requests, and those of the run in
// which the CTA starts are looked at again, one a lane.
__device__ __forceinline__ RaggedStart ragged_start_singles(const RaggedParams& p, int c, int lane) {
  const int heads = p.n_kv_heads * p.head_chunks, run = (p.n_requests + 31) / 32;
  auto units_of = [&](int r, RaggedReq& q) {
    q = ragged_req_plain(p, r);
    return q.n > 0 ? ragged_span(p, q, 0).total : 0;
  };
  long long sum = 0;
  RaggedReq q;
#pragma unroll 4
  for (int i = 0; i < run; ++i)
    if (lane * run + i < p.n_requests) sum += units_of(lane * run + i, q);
  long long upto = warp_scan_ll(sum * heads, lane);
  const long long all = __shfl_sync(0xffffffffu, upto, 31), per = max(div_ll(all + p.n_ctas - 1, p.n_ctas), 1ll), u = per * c;
  RaggedStart s = {};
  if (u < all) {
    const int at = __ffs(__ballot_sync(0xffffffffu, upto > u)) - 1;
    const long long before = __shfl_sync(0xffffffffu, upto - sum * heads, at);
    const int r = at * run + lane, mine = lane < run && r < p.n_requests ? units_of(r, q) : 0;
    upto = before + warp_scan_ll((long long)mine * heads, lane);
    const int own = __ffs(__ballot_sync(0xffffffffu, upto > u)) - 1;
    RaggedReq o;
    o.row0 = __shfl_sync(0xffffffffu, q.row0, own);
    o.n = __shfl_sync(0xffffffffu, q.n, own); o.seq = __shfl_sync(0xffffffffu, q.seq, own); o.stride = 1;
    const long long a_head = __shfl_sync(0xffffffffu, mine, own), end = __shfl_sync(0xffffffffu, upto, own);
    s = ragged_cut(p, at * run + own, o, end - a_head * heads, a_head, u, per, all, lane);
  }
  if (lane == 0) reinterpret_cast<RaggedStart*>(p.scratch)[c] = s;
  return s;
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

// decides whether the CTAs find their starts themselves, launches the schedule kernel if not
int ragged_schedule(RaggedParams& p, int max_new, cudaStream_t st);
int ragged_merge(const RaggedParams& p, int max_new, int head_dim, cudaStream_t st);
// up to 16 packed rows an item: bandwidth bound (single tokens); also what TMA cannot describe
// solo: a worker per warp instead of one per CTA (n_ctas counts the workers)
void ragged_rows_config(RaggedParams& p, bool solo);
int ragged_rows_attention(const RaggedParams& p, int head_dim, cudaStream_t st);
// items of two 128-row MMA tiles on tcgen05 (spf_ragged_tc5.cu); SPF_ERR_SHAPE where TMA cannot describe the tensors
void ragged_tc5_config(RaggedParams& p);
bool ragged_tc5_describable(const RaggedParams& p);
int ragged_tc5_attention(const RaggedParams& p, int head_dim, cudaStream_t st);
unsigned int ragged_tc5_timeout_count();
bool ragged_tc5_reset_timeouts();
bool ragged_tc5_set_wait_limit(unsigned long long ns);

}  // namespace spf
