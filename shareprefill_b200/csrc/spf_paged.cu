// The bookkeeping of a paged KV cache: the plan of a step (pages, offsets, slots) from the requests'
// lengths, and the write of new K/V rows into their slots.
#include <cooperative_groups.h>

#include "spf_internal.cuh"
#include "spf_paged.cuh"

namespace cg = cooperative_groups;

namespace spf {

// ---------------------------------------------------------------- plan
// With c cached and n new tokens of a request and pages of P tokens: it holds ceil(c / P) pages, needs
// ceil((c + n) / P), and the ids it lacks come from the free ring in the order of the requests.  One
// cluster: every CTA scans all requests (a few numbers each) into shared memory, then the CTAs share the
// rows and the table's new entries.  Between the two lies a cluster barrier, so an output may be the
// array that an input was.  Bound by latency: 6.4 us for 8 requests, 13 us for 512 requests and 37K rows (0.3 MB), of
// which the scan and the rows' binary searches in shared memory are most; a single CTA would write the rows at
// an eighth of the rate, and a grid of more needs a second launch for the scan.
constexpr int PLAN_CTAS = 8, PLAN_NT = 512, PLAN_WARPS = PLAN_NT / 32;

__device__ __forceinline__ long long warp_scan_long(long long v, int lane) {   // inclusive
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  return v;
}

__global__ void __cluster_dims__(PLAN_CTAS, 1, 1) __launch_bounds__(PLAN_NT) paged_plan_kernel(const PlanParams p) {
  extern __shared__ int32_t psm[];
  int32_t* cu = psm;                        // [R + 1], rows of the batch
  int32_t* cached = cu + p.n_requests + 1;  // [R]
  int32_t* base = cached + p.n_requests;    // [R] ring offset of the first new page, -1 for a refused request
  __shared__ long long wsum[2][PLAN_WARPS];
  __shared__ int taken_max;
  cg::cluster_group cluster = cg::this_cluster();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = int(cluster.block_rank());
  const int cap = p.ring_capacity, ps = 1 << p.page_shift;
  const int turn = p.ring_state[0] % cap, head = turn < 0 ? turn + cap : turn;
  const int count = min(max(p.ring_state[1], 0), cap);
  if (tid == 0) { cu[0] = 0; taken_max = 0; }
  long long carry_rows = 0, carry_pages = 0;
  for (int r0 = 0; r0 < p.n_requests; r0 += PLAN_NT) {
    const int r = r0 + tid;
    const bool in = r < p.n_requests;
    const long long c = in ? max(p.cached_len[r], 0) : 0, n = in ? max(p.new_len[r], 0) : 0;
    const long long held = (c + ps - 1) >> p.page_shift, total = (c + n + ps - 1) >> p.page_shift;
    long long rows = warp_scan_long(n, lane);
    if (lane == 31) wsum[0][warp] = rows;
    __syncthreads();
    if (warp == 0) {
      const long long t = warp_scan_long(lane < PLAN_WARPS ? wsum[0][lane] : 0, lane);
      if (lane < PLAN_WARPS) wsum[0][lane] = t;
    }
    __syncthreads();
    if (warp > 0) rows += wsum[0][warp - 1];
    rows += carry_rows;
    const bool fits = in && total <= p.table_width && rows <= p.n_rows && c + n <= SPF_MAX_KEYS;
    const long long need = fits ? total - held : 0;
    long long upto = warp_scan_long(need, lane);
    if (lane == 31) wsum[1][warp] = upto;
    __syncthreads();
    if (warp == 0) {
      const long long t = warp_scan_long(lane < PLAN_WARPS ? wsum[1][lane] : 0, lane);
      if (lane < PLAN_WARPS) wsum[1][lane] = t;
    }
    __syncthreads();
    if (warp > 0) upto += wsum[1][warp - 1];
    upto += carry_pages;
    const bool ok = fits && (need == 0 || upto <= count);
    if (in) {
      cu[r + 1] = int(min(rows, (long long)p.n_rows));
      cached[r] = int(c);
      base[r] = ok ? int(upto - need) : -1;
      if (ok && need > 0) atomicMax(&taken_max, int(upto));
    }
    carry_rows += wsum[0][PLAN_WARPS - 1];
    carry_pages += wsum[1][PLAN_WARPS - 1];
    __syncthreads();
  }
  cluster.sync();   // all reads of lengths and state are done

  if (rank == 0) {
    for (int r = tid; r < p.n_requests; r += PLAN_NT) {
      const int n = cu[r + 1] - cu[r];
      p.cu_new[r + 1] = cu[r + 1];
      p.seq_len[r] = base[r] >= 0 ? cached[r] + n : 0;
      p.refused[r] = base[r] >= 0 ? 0 : 1;
    }
    if (tid == 0) {
      p.cu_new[0] = 0;
      p.ring_state_out[0] = int((int64_t(head) + taken_max) % cap);
      p.ring_state_out[1] = count - taken_max;
    }
  }
  // new entries of the table: a warp per request
  for (int r = rank * PLAN_WARPS + warp; r < p.n_requests; r += PLAN_CTAS * PLAN_WARPS) {
    if (base[r] < 0) continue;
    const int c = cached[r], n = cu[r + 1] - cu[r];
    const int held = (c + ps - 1) >> p.page_shift, need = ((c + n + ps - 1) >> p.page_shift) - held;
    for (int i = lane; i < need; i += 32)
      p.table[r * p.table_stride + held + i] = p.ring[(int64_t(head) + base[r] + i) % cap];
  }
  // slots and positions of the rows
  for (int t = rank * PLAN_NT + tid; t < p.n_rows; t += PLAN_CTAS * PLAN_NT) {
    int64_t slot = -1;
    int pos = 0;
    if (t < cu[p.n_requests]) {
      int lo = 0, hi = p.n_requests - 1;     // the request whose rows end first behind t
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (cu[mid + 1] > t) hi = mid; else lo = mid + 1;
      }
      pos = int(min((long long)cached[lo] + (t - cu[lo]), 0x7fffffffll));   // (past the limit for refused requests only)
      if (base[lo] >= 0) {
        const int pg = pos >> p.page_shift, held = (cached[lo] + ps - 1) >> p.page_shift;
        const int id = pg < held ? p.table[lo * p.table_stride + pg] : p.ring[(int64_t(head) + base[lo] + pg - held) % cap];
        if (id >= 0) slot = (int64_t(id) << p.page_shift) + (pos & (ps - 1));
      }
    }
    p.slot_map[t] = slot;
    p.positions[t] = pos;
  }
}

int launch_paged_plan(const PlanParams& p, cudaStream_t st) {
  const int smem = (3 * p.n_requests + 1) * 4;
  // 48 KiB are granted without asking, to this and the kernel's static shared memory together.  (Always the same limit: with the
  // call's own size, a call from another thread could lower it between this and the launch.)
  if (smem > 32 * 1024) {
    const cudaError_t e =
        cudaFuncSetAttribute(paged_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (3 * SPF_MAX_REQUESTS + 1) * 4);
    if (e != cudaSuccess) { note_cuda_error(e); return SPF_ERR_LAUNCH; }
  }
  paged_plan_kernel<<<PLAN_CTAS, PLAN_NT, smem, st>>>(p);
  return check_launch();
}

// ---------------------------------------------------------------- write
// k_cache[slot] = k[row], v_cache[slot] = v[row]: a copy in 16-byte chunks, bound by HBM.  A block takes four rows; the
// slots, then all loads of a thread are requested before its first store: 32K rows of 8 heads x 128 take 43.3 us (6.2
// TB/s, 0.95 of the measured copy bandwidth) where a row per block took 53.6 and two rows 44.1.  Stores that
// bypass L2 would save another microsecond and cost the attention that follows its hits.
constexpr int WR_NT = 256, WR_ROWS = 4;

__global__ void __launch_bounds__(WR_NT) paged_write_kernel(const WriteParams p) {
  const int row0 = blockIdx.x * WR_ROWS;
  int64_t page[WR_ROWS];
  int in_page[WR_ROWS];
  bool ok[WR_ROWS];
#pragma unroll
  for (int r = 0; r < WR_ROWS; ++r) {
    const int64_t slot = row0 + r < p.n_rows ? __ldg(p.slot_map + row0 + r) : -1;
    ok[r] = slot >= 0 && slot < p.n_slots;
    page[r] = slot >> p.page_shift;
    in_page[r] = int(slot) & ((1 << p.page_shift) - 1);
  }
  const int half = p.n_kv_heads << p.chunk_shift;       // chunks of K; as many of V
  for (int i = threadIdx.x; i < 2 * half; i += WR_NT) {
    const bool is_v = i >= half;
    const int j = is_v ? i - half : i, h = j >> p.chunk_shift, ch = j & ((1 << p.chunk_shift) - 1);
    const WriteTensor& t = is_v ? p.v : p.k;
    uint4 x[WR_ROWS];
#pragma unroll
    for (int r = 0; r < WR_ROWS; ++r)
      if (ok[r]) x[r] = __ldcs(reinterpret_cast<const uint4*>(t.src + int64_t(row0 + r) * t.sn + h * t.sh) + ch);
#pragma unroll
    for (int r = 0; r < WR_ROWS; ++r)
      if (ok[r]) *(reinterpret_cast<uint4*>(t.dst + page[r] * t.dp + in_page[r] * t.dt + h * t.dh) + ch) = x[r];
  }
}

int launch_paged_write(const WriteParams& p, cudaStream_t st) {
  if (p.n_rows == 0) return SPF_OK;
  paged_write_kernel<<<ceil_div(p.n_rows, WR_ROWS), WR_NT, 0, st>>>(p);
  return check_launch();
}

}  // namespace spf
