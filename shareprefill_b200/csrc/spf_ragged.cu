// Ragged attention over a paged or contiguous KV cache (see spf_ragged.cuh): the schedule, the kernel for
// items of up to 16 rows, and the kernel that joins broken items.
#include "spf_mma.cuh"
#include "spf_ragged.cuh"

namespace spf {

// ---------------------------------------------------------------- schedule
// Every block sums the units of every request (a thread per request of one tile, a warp, its lanes over the tiles, per
// larger one), scans the sums, and each of its warps finds the start of one CTA: request by binary search, head by division, tile
// by a scan over the tiles.
// (blocks of 1024 threads, so of 32 starts, put the whole work on a few SMs: 15 us for 512 windowed tiles)
constexpr int SCH_NT = 256, SCH_WARPS = SCH_NT / 32;
constexpr int FEW_REQUESTS = 32, FEW_TILES = 512, FEW_SINGLES = 256;

__global__ void __launch_bounds__(SCH_NT) ragged_schedule_kernel(const RaggedParams p) {
  __shared__ long long upto[SPF_MAX_REQUESTS];   // inclusive sums over the requests
  __shared__ long long wsum[SCH_WARPS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int heads = p.n_kv_heads * p.head_chunks;
  int more = 0;
  for (int r = threadIdx.x; r < p.n_requests; r += SCH_NT) {
    const RaggedReq q = ragged_req_plain(p, r);
    const int tiles = ragged_tiles(p, q.n);
    upto[r] = tiles > 1 ? -1 : tiles == 1 ? (long long)ragged_span(p, q, 0).total * heads : 0;
    more |= tiles > 1;
  }
  if (__syncthreads_or(more)) {
    for (int r = warp; r < p.n_requests; r += SCH_WARPS) {
      if (upto[r] >= 0) continue;
      const RaggedReq q = ragged_req_plain(p, r);
      const int tiles = ragged_tiles(p, q.n);
      long long s = 0;
#pragma unroll 4
      for (int t = lane; t < tiles; t += 32) s += ragged_span(p, q, t).total;
      s = warp_sum_ll(s);
      if (lane == 0) upto[r] = s * heads;
    }
    __syncthreads();
  }
  long long carry = 0;
  for (int r0 = 0; r0 < p.n_requests; r0 += SCH_NT) {
    const int r = r0 + threadIdx.x;
    long long v = warp_scan_ll(r < p.n_requests ? upto[r] : 0, lane);
    if (lane == 31) wsum[warp] = v;
    __syncthreads();
    if (warp == 0) {
      const long long t = warp_scan_ll(lane < SCH_WARPS ? wsum[lane] : 0, lane);
      if (lane < SCH_WARPS) wsum[lane] = t;
    }
    __syncthreads();
    if (warp > 0) v += wsum[warp - 1];
    if (r < p.n_requests) upto[r] = v + carry;
    carry += wsum[SCH_WARPS - 1];
    __syncthreads();
  }
  const long long all = carry, per = max(div_ll(all + p.n_ctas - 1, p.n_ctas), 1ll);
  auto head_units = [&](int r) { return div_ll(upto[r] - (r > 0 ? upto[r - 1] : 0), heads); };
  if (blockIdx.x == 0 && p.window > 0)
    for (int r = threadIdx.x; r < p.n_requests; r += SCH_NT)
      ragged_strides(p)[r] = ragged_stride(per, ragged_tiles(p, ragged_req_plain(p, r).n), head_units(r));
  const int c = blockIdx.x * SCH_WARPS + warp;
  if (c >= p.n_ctas) return;
  const long long u = per * c;
  RaggedStart s = {};
  if (u < all) {
    int lo = 0, hi = p.n_requests - 1;   // first request whose inclusive sum is above u
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (upto[mid] > u) hi = mid; else lo = mid + 1;
    }
    RaggedReq q = ragged_req_plain(p, lo);
    if (p.window > 0) q.stride = ragged_stride(per, ragged_tiles(p, q.n), head_units(lo));
    s = ragged_cut(p, lo, q, lo > 0 ? upto[lo - 1] : 0, head_units(lo), u, per, all, lane);
  }
  if (lane == 0) reinterpret_cast<RaggedStart*>(p.scratch)[c] = s;
}

int ragged_schedule(RaggedParams& p, int max_new, cudaStream_t st) {
  p.few = 0;
  if (p.n_requests <= FEW_REQUESTS && p.n_rows / p.tile_tokens + p.n_requests <= FEW_TILES) p.few = 1;
  else if (p.n_requests <= FEW_SINGLES && max_new <= p.tile_tokens && p.tile_rows <= RAGGED_FEW_ROWS) p.few = 2;
  if (p.few) return SPF_OK;
  ragged_schedule_kernel<<<ceil_div(p.n_ctas, SCH_WARPS), SCH_NT, 0, st>>>(p);
  return check_launch();
}

// ---------------------------------------------------------------- join of broken items
// Block (c, y): CTA c's start lies inside an item; if c is the first such CTA of that item, the item's parts are
// CTA c - 1's second slot and the first slots of c, c + 1, ...  The time is the latency of a few dependent loads, so
// what is known to be needed is requested at once and the place of the output comes with the start record.
//   large tiles (a chunk, cut once or twice): D / 16 lanes take a row, 16 columns each, two parts at a time
//   single tokens (28 heads over 128K keys: cut into 74): a block takes a row, whose parts the warps share, four at a
//   time, and add up through shared memory
// (With a warp per row and one part at a time in both cases the join took 43 us after such a token, 25 us after a 2K chunk.)
constexpr int MRG_NT = 256, MRG_WARPS = MRG_NT / 32, MRG_FEW = 4;

// running maximum, sum and output of parts whose m, l and (16-byte pieces of) o are given; m = -inf: no part
template <int N, int V>
__device__ __forceinline__ void merge_in(const float (&m)[N], const float (&l)[N], const float (&o)[N][V], float& top, float& sum, float (&acc)[V]) {
  float t = top;
#pragma unroll
  for (int i = 0; i < N; ++i) t = fmaxf(t, m[i]);
  const float ref = t == -INFINITY ? 0.f : t, a = exp2f(top - ref);
  top = t;
  sum *= a;
#pragma unroll
  for (int e = 0; e < V; ++e) acc[e] *= a;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float w = exp2f(m[i] - ref);
    sum += l[i] * w;
#pragma unroll
    for (int e = 0; e < V; ++e) acc[e] += o[i][e] * w;
  }
}

template <int D, bool FP16>
__global__ void __launch_bounds__(MRG_NT) ragged_merge_kernel(const RaggedParams p, bool large) {
  __shared__ float acc_of[MRG_WARPS][D], sum_of[MRG_WARPS], top_of[MRG_WARPS];
  ragged_wait_before();
  const RaggedStart* starts = reinterpret_cast<const RaggedStart*>(p.scratch);
  const int c = blockIdx.x + 1;
  const RaggedStart s = starts[c];
  const int per = starts[0].units;             // every CTA but the last runs through equally many
  if (s.units == 0 || s.first == 0 || s.first > per) return;   // the last: an earlier CTA starts inside this item too
  const int n = (s.item_units - s.first + per - 1) / per + 1;   // parts
  const int64_t tile = ragged_partial_floats(p.tile_rows, D);
  const float* base = ragged_part(p, c - 1, 1, D);
  auto part = [&](int i) { return i == 0 ? base : base + (2 * i - 1) * tile; };   // (c - 1, 1), (c, 0), (c + 1, 0), ...
  // offset of the row in the output, in elements; -1: not a row of the item
  auto place = [&](int row) -> int64_t {
    const int in_stream = row % p.stream_rows, t = in_stream / p.chunk_heads, h = in_stream - t * p.chunk_heads;
    const int tok = row / p.stream_rows * p.stream_tokens + t;
    if (t >= p.stream_tokens || tok >= s.n_tok || h >= s.heads) return -1;
    return s.out + (int64_t(tok) * p.n_q_heads + h) * D;
  };
  if (large) {
    constexpr int LANES = D / 16, N = 2;       // lane x has columns 4 x + 4 LANES j .. + 3, j < 4
    const int row = blockIdx.y * (MRG_NT / LANES) + threadIdx.x / LANES, x4 = (threadIdx.x % LANES) * 4;
    float top = -INFINITY, sum = 0.f, acc[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[e] = 0.f;
    for (int i0 = 0; i0 < n; i0 += N) {
      float m[N], l[N], o[N][16];
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float* x = part(min(i0 + i, n - 1));
        m[i] = i0 + i < n ? x[row] : -INFINITY;
        l[i] = x[p.tile_rows + row];
#pragma unroll
        for (int j = 0; j < 4; ++j)
          *reinterpret_cast<float4*>(&o[i][4 * j]) = *reinterpret_cast<const float4*>(x + 2 * p.tile_rows + row * D + x4 + j * 4 * LANES);
      }
      merge_in(m, l, o, top, sum, acc);
    }
    const int64_t at = place(row);
    if (at < 0) return;                        // what was read of such a row was never written, and is not used
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + at + x4 + j * 4 * LANES) =
          make_uint2(pack_half2<FP16>(acc[4 * j] * inv, acc[4 * j + 1] * inv), pack_half2<FP16>(acc[4 * j + 2] * inv, acc[4 * j + 3] * inv));
    return;
  }
  constexpr int PER = D / 32;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, row = blockIdx.y;
  const int64_t at = place(row);
  if (at < 0) return;
  float top = -INFINITY, sum = 0.f, acc[PER];
#pragma unroll
  for (int e = 0; e < PER; ++e) acc[e] = 0.f;
  for (int i0 = warp; i0 < n; i0 += MRG_FEW * MRG_WARPS) {
    float m[MRG_FEW], l[MRG_FEW], o[MRG_FEW][PER];
#pragma unroll
    for (int i = 0; i < MRG_FEW; ++i) {
      const bool there = i0 + i * MRG_WARPS < n;
      const float* x = part(there ? i0 + i * MRG_WARPS : i0);
      m[i] = there ? x[row] : -INFINITY;
      l[i] = x[p.tile_rows + row];
#pragma unroll
      for (int e = 0; e < PER; e += 2)
        *reinterpret_cast<float2*>(&o[i][e]) = *reinterpret_cast<const float2*>(x + 2 * p.tile_rows + row * D + lane * PER + e);
    }
    merge_in(m, l, o, top, sum, acc);
  }
#pragma unroll
  for (int e = 0; e < PER; ++e) acc_of[warp][lane * PER + e] = acc[e];
  if (lane == 0) { sum_of[warp] = sum; top_of[warp] = top; }
  __syncthreads();
  if (threadIdx.x < D / 2) {
    float all_top = -INFINITY;
#pragma unroll
    for (int w = 0; w < MRG_WARPS; ++w) all_top = fmaxf(all_top, top_of[w]);
    const float ref = all_top == -INFINITY ? 0.f : all_top;
    float total = 0.f, x = 0.f, y = 0.f;
#pragma unroll
    for (int w = 0; w < MRG_WARPS; ++w) {
      const float a = exp2f(top_of[w] - ref);
      total += sum_of[w] * a;
      x += acc_of[w][2 * threadIdx.x] * a; y += acc_of[w][2 * threadIdx.x + 1] * a;
    }
    const float inv = total == 0.f ? 0.f : 1.f / total;
    reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(p.out) + at)[threadIdx.x] = pack_half2<FP16>(x * inv, y * inv);
  }
}

// Rows that an item can have follow from max_new.
template <int D, bool FP16>
static int launch_merge(const RaggedParams& p, int max_new, cudaStream_t st) {
  const int rows = max_new <= p.stream_tokens ? max_new * p.chunk_heads : p.tile_rows;
  const bool large = rows > RAGGED_FEW_ROWS;
  const int blocks = large ? ceil_div(rows, MRG_NT / (D / 16)) : rows;
  return ragged_launch_after(ragged_merge_kernel<D, FP16>, dim3(p.n_ctas - 1, blocks), MRG_NT, 0, st, p, large);
}

int ragged_merge(const RaggedParams& p, int max_new, int head_dim, cudaStream_t st) {
  if (head_dim == 128) return p.fp16 ? launch_merge<128, true>(p, max_new, st) : launch_merge<128, false>(p, max_new, st);
  return p.fp16 ? launch_merge<64, true>(p, max_new, st) : launch_merge<64, false>(p, max_new, st);
}

// ---------------------------------------------------------------- items of up to 16 rows
// The rows of an item are the 16 rows of mma.sync m16n8k16 tiles.  A unit is 64 keys, 16 per warp; every
// warp streams its tiles through a private ring of cp.async stages and keeps its own running maximum, sum
// and output; the warps meet when the CTA's part of the item ends.  Bound by HBM: 64 tokens of 32 heads over 8 KV heads
// and up to 8K keys (1.33 GB) take 216 - 228 us with the join, 5.8 - 6.1 TB/s; one token of 28 heads over 128K keys 49 us, 5.5 TB/s, of which
// 4 us are launch and start and 3 the end.  Three stages of 16 keys per warp and two CTAs per SM keep 128 KiB of an SM in flight.
constexpr int RR_NT = 128, RR_NW = RR_NT / 32, RR_TT = 16, RR_STAGES = 3, RR_ROWS = 16;

template <int D>
constexpr int rr_smem_bytes() { return RR_NW * RR_STAGES * 2 * RR_TT * D * 2; }

template <bool FP16>
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (FP16) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};\n"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  } else {
    mma_bf16_16816(d, a, b0, b1);
  }
}

__device__ __forceinline__ void cp_async16_all(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(dst), "l"(src));
}
__device__ __forceinline__ float ex2(float x) {      // 2^x; results below 2^-126 are 0
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// SOLO: every warp is a worker with a part of the line of its own (in units of 16 keys) and no one to join with; for
// batches with so many items that a CTA would run through several, one chain of loads after the other.
template <int D, bool FP16, bool SOLO>
__global__ void __launch_bounds__(RR_NT, D == 64 ? 3 : 2) ragged_rows_kernel(const RaggedParams p) {
  constexpr int CH = D / 8, TILE_B = RR_TT * D * 2, UNIT = SOLO ? RR_TT : RR_TT * RR_NW;
  extern __shared__ __align__(128) uint8_t rsm[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t ring = smem_u32(rsm) + warp * (RR_STAGES * 2 * TILE_B);
  const int r0 = lane >> 2, r1 = r0 + 8, cq = (lane & 3) * 2;
  constexpr int ROWS_AT_ONCE = 32 / CH;         // a warp copies this many rows of a tile at a time
  const int lane_row = lane / CH, lane_ch = lane % CH;
  const uint32_t lane_off = tile_off<D>(lane_row, lane_ch);
  __shared__ RaggedStart sh_start;
  __shared__ int32_t sh_strides[SOLO ? RR_NW : 1][FEW_REQUESTS];
  const int worker = SOLO ? blockIdx.x * RR_NW + warp : blockIdx.x, part_col = SOLO ? 0 : warp * RR_TT;
  int32_t* strides = sh_strides[SOLO ? warp : 0];
  ragged_wait_before();
  RaggedStart start;
  if (!p.few) {
    start = reinterpret_cast<const RaggedStart*>(p.scratch)[worker];
  } else {
    if (SOLO || warp == 0) {
      start = p.few == 1 ? ragged_start_few(p, worker, lane, strides) : ragged_start_singles(p, worker, lane);
      if (!SOLO && lane == 0) sh_start = start;
    }
    if (SOLO) {
      __syncwarp();
    } else {
      __syncthreads();
      start = sh_start;
    }
  }
  int left = start.units, req = start.req, head = start.head, tile = start.tile, first = start.first;
  if (left == 0) return;
  RaggedReq q = ragged_req(p, req, strides);

  while (true) {
    const RaggedSpan span = ragged_span(p, q, tile);
    const int units = min(left, span.total - first);
    const RaggedItem item = ragged_item(p, q, head, tile);
    const int kvh = item.kvh, h0 = item.h0, tok0 = item.tok0, pos0 = item.pos0;
    const uint16_t* kb = static_cast<const uint16_t*>(p.k) + kvh * p.k_sh;
    const uint16_t* vb = static_cast<const uint16_t*>(p.v) + kvh * p.v_sh;
    const int32_t* table = p.table ? p.table + req * p.table_stride : nullptr;

    // the item's query rows as A fragments (rows past its end are zero)
    uint32_t qa[D / 16][4];
    const int t_r0 = r0 / p.chunk_heads, t_r1 = r1 / p.chunk_heads;
    const int h_r0 = r0 - t_r0 * p.chunk_heads, h_r1 = r1 - t_r1 * p.chunk_heads;
    const bool in0 = t_r0 < item.n_tok && h_r0 < item.heads, in1 = t_r1 < item.n_tok && h_r1 < item.heads;
    {
      const uint16_t* qb = static_cast<const uint16_t*>(p.q) + (int64_t(q.row0) + tok0) * p.q_sn +
                           int64_t(kvh * p.group + h0) * p.q_sh + cq;
      const uint16_t* q0 = qb + t_r0 * p.q_sn + h_r0 * p.q_sh;
      const uint16_t* q1 = qb + t_r1 * p.q_sn + h_r1 * p.q_sh;
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        qa[ks][0] = in0 ? *reinterpret_cast<const uint32_t*>(q0 + ks * 16) : 0u;
        qa[ks][1] = in1 ? *reinterpret_cast<const uint32_t*>(q1 + ks * 16) : 0u;
        qa[ks][2] = in0 ? *reinterpret_cast<const uint32_t*>(q0 + ks * 16 + 8) : 0u;
        qa[ks][3] = in1 ? *reinterpret_cast<const uint32_t*>(q1 + ks * 16 + 8) : 0u;
      }
    }
    // row r sees keys <= hi that are >= lo or < sinks (rows past the item's end: none)
    const int hi0 = in0 ? pos0 + t_r0 : -1, hi1 = in1 ? pos0 + t_r1 : -1;
    const int lo0 = p.window > 0 ? hi0 - p.window + 1 : 0, lo1 = p.window > 0 ? hi1 - p.window + 1 : 0;
    // keys in [all_lo, all_hi] are seen by every row of the item
    const int all_hi = pos0, all_lo = p.window > 0 ? pos0 + p.tile_tokens - p.window : 0;
    const int any_lo = p.window > 0 ? pos0 - p.window + 1 : 0;   // keys below it that are no sinks are seen by no row

    // step u of this warp: 16 keys from `k0` that count up to `end`; `first_keys`: of the sinks
    struct Step { int k0, end; bool first_keys; };
    const bool plain = span.sink_units == 0 && span.embed == 0;
    const int plain_k0 = span.win_key + first * UNIT + part_col;
    auto step_of = [&](int u) {
      if (plain) return Step{plain_k0 + u * UNIT, span.keys, false};
      const int s = first + u, col = (s < span.sink_units ? s : s - span.sink_units) * UNIT + part_col;
      if (s < span.sink_units || col < span.embed) return Step{col, span.sink_keys, true};
      return Step{span.win_key + col, span.keys, false};
    };
    // its page, -1 if absent
    auto page_of = [&](int u) -> int {
      if (u >= units) return -1;
      const Step x = step_of(u);
      if (x.k0 >= x.end) return -1;
      if (!table) return 0;
      const int pg = table[x.k0 >> p.page_shift];
      return pg >= 0 && pg < p.n_pages ? pg : -1;
    };
    auto issue = [&](int u, int page, int stage) {
      if (u < units) {
        const Step x = step_of(u);
        const int k0 = x.k0, valid = page >= 0 ? x.end - k0 : 0;
        const int in_page = table ? k0 & ((1 << p.page_shift) - 1) : k0;
        const uint32_t ks = ring + stage * (2 * TILE_B), vs = ks + TILE_B;
        const uint16_t* kp = kb + (valid > 0 ? page * p.k_sp + in_page * p.k_st : 0);
        const uint16_t* vp = vb + (valid > 0 ? page * p.v_sp + in_page * p.v_st : 0);
        // A tile of keys that all count is copied without a question per row (rows eight apart lie alike in the swizzled tile).
        // With that and the rescaling left out where no maximum moved, a tile takes 334 instructions of a warp instead of
        // 597: 64 requests up to 8K 233 -> 224 us in a long run, where the power limit counts
        if (valid >= RR_TT && (x.first_keys || k0 >= any_lo)) {
          kp += lane_row * p.k_st + lane_ch * 8;
          vp += lane_row * p.v_st + lane_ch * 8;
#pragma unroll
          for (int r = 0; r < RR_TT; r += ROWS_AT_ONCE) {
            const uint32_t at = (lane_off ^ (uint32_t(r & 7) << 4)) + r * (D * 2);
            cp_async16_all(ks + at, kp);
            cp_async16_all(vs + at, vp);
            kp += ROWS_AT_ONCE * p.k_st; vp += ROWS_AT_ONCE * p.v_st;
          }
        } else {
#pragma unroll 1
          for (int row = lane_row; row < RR_TT; row += ROWS_AT_ONCE) {
            // keys that no row of the item sees are not read: whatever they hold, 0 times it must stay 0
            const bool ok = row < valid && (x.first_keys || k0 + row >= any_lo || k0 + row < p.sinks);
            cp_async16(ks + tile_off<D>(row, lane_ch), kp + (ok ? row * p.k_st + lane_ch * 8 : 0), ok);
            cp_async16(vs + tile_off<D>(row, lane_ch), vp + (ok ? row * p.v_st + lane_ch * 8 : 0), ok);
          }
        }
      }
      cp_async_commit();
    };

    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
    float o[D / 8][4];
#pragma unroll
    for (int j = 0; j < D / 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;

    // page ids run one step ahead of the copies that need them
    int pg_a = page_of(0), pg_b = page_of(1), pg_c = page_of(2);
    issue(0, pg_a, 0);
    issue(1, pg_b, 1);
    int stage = 0;
    for (int u = 0; u < units; ++u) {
      const int page = pg_a, pg_next = page_of(u + 3);
      int pre = stage + 2; if (pre >= RR_STAGES) pre -= RR_STAGES;
      issue(u + 2, pg_c, pre);
      pg_a = pg_b; pg_b = pg_c; pg_c = pg_next;
      cp_async_wait<2>();
      __syncwarp();
      if (page >= 0) {
        const Step x = step_of(u);
        const int k0 = x.k0;
        const uint32_t ks_base = ring + stage * (2 * TILE_B), vs_base = ks_base + TILE_B;
        float s[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
          uint32_t b[4];
          ldmatrix_x4(b, ks_base + tile_off<D>((lane & 7) + ((lane >> 4) << 3), ks * 2 + ((lane >> 3) & 1)));
          mma_16816<FP16>(s[0], qa[ks], b[0], b[1]);
          mma_16816<FP16>(s[1], qa[ks], b[2], b[3]);
        }
        if (x.first_keys || k0 < all_lo || k0 + RR_TT - 1 > all_hi) {
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int key = k0 + j * 8 + cq + (e & 1);
              const int hi = e < 2 ? hi0 : hi1, lo = e < 2 ? lo0 : lo1;
              s[j][e] = key <= hi && (key >= lo || key < p.sinks) && key < x.end ? s[j][e] : -INFINITY;
            }
        }
        float y0 = fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[1][0], s[1][1]));
        float y1 = fmaxf(fmaxf(s[0][2], s[0][3]), fmaxf(s[1][2], s[1][3]));
        y0 = fmaxf(y0, __shfl_xor_sync(0xffffffffu, y0, 1)); y0 = fmaxf(y0, __shfl_xor_sync(0xffffffffu, y0, 2));
        y1 = fmaxf(y1, __shfl_xor_sync(0xffffffffu, y1, 1)); y1 = fmaxf(y1, __shfl_xor_sync(0xffffffffu, y1, 2));
        const float n0 = fmaxf(m0, y0 * p.scale_log2), n1 = fmaxf(m1, y1 * p.scale_log2);
        const float f0 = n0 == -INFINITY ? 0.f : n0, f1 = n1 == -INFINITY ? 0.f : n1;   // nothing seen yet: all weights are 0
        // The largest weight is 2^LIFT; the factor cancels in o / l.  fp16: multiples of 2^-24 lose 2^-40 of it per key; bf16: o
        // does not overflow with values up to 3.4e38
        constexpr float LIFT = FP16 ? 15.f : -32.f;
        const float g0 = f0 - LIFT, g1 = f1 - LIFT;
        if (__any_sync(0xffffffffu, n0 != m0 || n1 != m1)) {      // rare once a few tiles have been seen
          const float a0 = ex2(m0 - f0), a1 = ex2(m1 - f1);
          l0 *= a0; l1 *= a1;
#pragma unroll
          for (int j = 0; j < D / 8; ++j) { o[j][0] *= a0; o[j][1] *= a0; o[j][2] *= a1; o[j][3] *= a1; }
          m0 = n0; m1 = n1;
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          s[j][0] = ex2(fmaf(s[j][0], p.scale_log2, -g0)); s[j][1] = ex2(fmaf(s[j][1], p.scale_log2, -g0));
          s[j][2] = ex2(fmaf(s[j][2], p.scale_log2, -g1)); s[j][3] = ex2(fmaf(s[j][3], p.scale_log2, -g1));
        }
        l0 += (s[0][0] + s[0][1]) + (s[1][0] + s[1][1]);
        l1 += (s[0][2] + s[0][3]) + (s[1][2] + s[1][3]);
        // the weights are rounded to the inputs' type for the product, their sum is taken before that
        const uint32_t pa[4] = {pack_half2<FP16>(s[0][0], s[0][1]), pack_half2<FP16>(s[0][2], s[0][3]),
                                pack_half2<FP16>(s[1][0], s[1][1]), pack_half2<FP16>(s[1][2], s[1][3])};
#pragma unroll
        for (int jj = 0; jj < D / 16; ++jj) {
          uint32_t b[4];
          ldmatrix_x4_trans(b, vs_base + tile_off<D>((lane & 7) + (((lane >> 3) & 1) << 3), jj * 2 + (lane >> 4)));
          mma_16816<FP16>(o[jj * 2], pa, b[0], b[1]);
          mma_16816<FP16>(o[jj * 2 + 1], pa, b[2], b[3]);
        }
      }
      __syncwarp();
      if (++stage == RR_STAGES) stage = 0;
    }
    cp_async_wait<0>();
    l0 += __shfl_xor_sync(0xffffffffu, l0, 1); l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
    l1 += __shfl_xor_sync(0xffffffffu, l1, 1); l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
    const bool whole = units == span.total;
    float* part = ragged_part(p, worker, first == 0 ? 1 : 0, D);
    if (SOLO) {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        if (!(half ? in1 : in0)) continue;
        const int r = half ? r1 : r0;
        const float l = half ? l1 : l0, inv = l == 0.f ? 0.f : 1.f / l;
        uint16_t* dst = static_cast<uint16_t*>(p.out) + ragged_out(p, q, item, half ? t_r1 : t_r0, half ? h_r1 : h_r0, D) + cq;
        if (!whole && (lane & 3) == 0) { part[r] = half ? m1 : m0; part[RR_ROWS + r] = l; }
#pragma unroll
        for (int j = 0; j < D / 8; ++j) {
          const float x = o[j][2 * half], y = o[j][2 * half + 1];
          if (whole) *reinterpret_cast<uint32_t*>(dst + j * 8) = pack_half2<FP16>(x * inv, y * inv);
          else *reinterpret_cast<float2*>(part + 2 * RR_ROWS + r * D + j * 8 + cq) = make_float2(x, y);
        }
      }
      left -= units;
      if (left == 0) return;
      first = 0;
      if (!ragged_next(p, req, head, tile, q, strides)) return;
      continue;
    }
    __syncthreads();

    // join the warps through shared memory (the rings are drained)
    constexpr int DS = D + 8, WSTRIDE = 16 * DS + 32;   // rows 8 banks apart; only rows that there are
    float* wbuf = reinterpret_cast<float*>(rsm) + warp * WSTRIDE;
    if (in0) {
#pragma unroll
      for (int j = 0; j < D / 8; ++j) *reinterpret_cast<float2*>(wbuf + r0 * DS + j * 8 + cq) = make_float2(o[j][0], o[j][1]);
    }
    if (in1) {
#pragma unroll
      for (int j = 0; j < D / 8; ++j) *reinterpret_cast<float2*>(wbuf + r1 * DS + j * 8 + cq) = make_float2(o[j][2], o[j][3]);
    }
    if ((lane & 3) == 0) {
      wbuf[16 * DS + r0] = m0; wbuf[16 * DS + r1] = m1;
      wbuf[16 * DS + 16 + r0] = l0; wbuf[16 * DS + 16 + r1] = l1;
    }
    __syncthreads();
    const float* all = reinterpret_cast<const float*>(rsm);
    for (int idx = threadIdx.x; idx < item.n_tok * p.chunk_heads * (D / 2); idx += RR_NT) {
      const int r = idx / (D / 2), d = (idx % (D / 2)) * 2, t = r / p.chunk_heads, h = r - t * p.chunk_heads;
      if (h >= item.heads) continue;
      float top = -INFINITY;
#pragma unroll
      for (int w = 0; w < RR_NW; ++w) top = fmaxf(top, all[w * WSTRIDE + 16 * DS + r]);
      const float ref = top == -INFINITY ? 0.f : top;
      float sum = 0.f, x = 0.f, y = 0.f;
#pragma unroll
      for (int w = 0; w < RR_NW; ++w) {
        const float sc = exp2f(all[w * WSTRIDE + 16 * DS + r] - ref);
        sum += all[w * WSTRIDE + 16 * DS + 16 + r] * sc;
        const float2 t = *reinterpret_cast<const float2*>(all + w * WSTRIDE + r * DS + d);
        x += t.x * sc; y += t.y * sc;
      }
      if (whole) {
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        *reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(p.out) + ragged_out(p, q, item, t, h, D) + d) =
            pack_half2<FP16>(x * inv, y * inv);
      } else {
        *reinterpret_cast<float2*>(part + 2 * RR_ROWS + r * D + d) = make_float2(x, y);
        if (d == 0) { part[r] = top; part[RR_ROWS + r] = sum; }
      }
    }
    left -= units;
    if (left == 0) return;
    first = 0;
    if (!ragged_next(p, req, head, tile, q, strides)) return;
    __syncthreads();   // the buffers become rings again
  }
}

// As many CTAs as fit: at D = 128 two per SM (96 KiB of rings, 250 registers), at D = 64 three (157 registers).  A decode
// batch of 64 requests up to 8K with D = 64 takes 145 / 129 / 173 us with 2 / 3 / 4 per SM, 133 with four of 128 registers.
void ragged_rows_config(RaggedParams& p, bool solo) {
  p.tile_rows = RR_ROWS;
  p.head_chunks = ceil_div(p.group, RR_ROWS);
  p.chunk_heads = ceil_div(p.group, p.head_chunks);
  p.stream_rows = RR_ROWS;
  p.tile_tokens = p.stream_tokens = RR_ROWS / p.chunk_heads;
  p.solo = solo;
  p.unit_shift = solo ? 4 : 6;
  static_assert(RR_TT == 16 && RR_NW == 4, "keys of a unit");
  p.granule = RR_TT;      // a warp's step lies in one page
  p.n_ctas = (p.head_dim == 64 ? 3 : 2) * 148 * (solo ? RR_NW : 1);
}

template <int D, bool FP16, bool SOLO>
static int launch_rows(const RaggedParams& p, cudaStream_t st) {
  constexpr int SMEM = rr_smem_bytes<D>();
  static_assert(SMEM >= RR_NW * (16 * (D + 8) + 32) * 4, "the join of the warps must fit in the rings");
  const cudaError_t e = cudaFuncSetAttribute(ragged_rows_kernel<D, FP16, SOLO>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
  if (e != cudaSuccess) { note_cuda_error(e); return SPF_ERR_LAUNCH; }
  return ragged_launch_after(ragged_rows_kernel<D, FP16, SOLO>, dim3(SOLO ? p.n_ctas / RR_NW : p.n_ctas), RR_NT, SMEM, st, p);
}

int ragged_rows_attention(const RaggedParams& p, int head_dim, cudaStream_t st) {
  if (head_dim == 128) {
    if (p.solo) return p.fp16 ? launch_rows<128, true, true>(p, st) : launch_rows<128, false, true>(p, st);
    return p.fp16 ? launch_rows<128, true, false>(p, st) : launch_rows<128, false, false>(p, st);
  }
  return p.fp16 ? launch_rows<64, true, false>(p, st) : launch_rows<64, false, false>(p, st);
}

}  // namespace spf
