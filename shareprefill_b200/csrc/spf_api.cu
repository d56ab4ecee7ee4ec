// C ABI of libspf_b200.so: argument validation and dispatch.  See include/spf_b200.h.
#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdlib>
#include <cstring>

#include "spf_internal.cuh"
#include "spf_paged.cuh"
#include "spf_ragged.cuh"

namespace spf {
static thread_local cudaError_t g_last_error = cudaSuccess;
// the value spf_device_timeouts() last returned: lets a launcher refuse work without a synchronisation
static std::atomic<unsigned int> g_known_timeouts{0};
static inline bool timeouts_tripped() { return g_known_timeouts.load(std::memory_order_relaxed) > 16u; }
// test hooks (spf_force_generic_kernels): run the mma.sync kernels where the tcgen05 ones would
static std::atomic<int> g_force_generic_attention{0}, g_force_generic_profile{0};
bool force_generic_profile() { return g_force_generic_profile.load(std::memory_order_relaxed) != 0; }
void note_cuda_error(cudaError_t e) { g_last_error = e; }

static inline bool strides_ok(int64_t sn, int64_t sh) { return (sn % 8 == 0) && (sh % 8 == 0); }
static inline bool aligned32(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 31u) == 0; }
static inline int log2_ceil(int x) { int b = 0; while ((1 << b) < x) ++b; return b; }
}  // namespace spf

using namespace spf;

extern "C" {

const char* spf_status_string(int status) {
  switch (status) {
    case SPF_OK: return "ok";
    case SPF_ERR_NULL: return "a required pointer is NULL";
    case SPF_ERR_SHAPE: return "unsupported shape (head_dim in {64,128}, block_size in {16,32,64,128}, n_tokens >= block_size, q heads a multiple of kv heads)";
    case SPF_ERR_ALIGN: return "pointer or stride is not 16-byte aligned";
    case SPF_ERR_RANGE: return "argument out of range";
    case SPF_ERR_LAUNCH: return "CUDA launch error (see spf_last_cuda_error)";
    case SPF_ERR_TOO_LARGE: return "size beyond a compiled-in maximum";
    case SPF_ERR_TIMEOUT: return "bounded device-side waits gave up earlier (spf_device_timeouts); reset with spf_reset_device_timeouts";
    default: return "unknown status";
  }
}

const char* spf_last_cuda_error(void) { return cudaGetErrorString(g_last_error); }
int spf_version(void) { return 100; }

static int check_shape(int n_tokens, int n_q_heads, int n_kv_heads, int head_dim, int block_size) {
  if (!supported_head_dim(head_dim) || !supported_block_size(block_size)) return SPF_ERR_SHAPE;
  if (n_tokens < block_size || n_q_heads <= 0 || n_kv_heads <= 0 || n_q_heads % n_kv_heads) return SPF_ERR_SHAPE;
  if (n_q_heads > SPF_MAX_HEADS) return SPF_ERR_TOO_LARGE;
  if (ceil_div(n_tokens, block_size) > SPF_MAX_BLOCKS) return SPF_ERR_TOO_LARGE;
  return SPF_OK;
}

int spf_pool_qk(const void* q, int64_t q_stride_n, int64_t q_stride_h, const void* k, int64_t k_stride_n,
                int64_t k_stride_h, int n_tokens, int n_q_heads, int n_kv_heads, int head_dim,
                int block_size, void* avg_q, void* avg_k, void* stream) {
  if ((q == nullptr) != (avg_q == nullptr) || (k == nullptr) != (avg_k == nullptr)) return SPF_ERR_NULL;
  if (!q && !k) return SPF_ERR_NULL;
  if (!supported_head_dim(head_dim) || n_tokens <= 0 || block_size <= 0 || block_size > 512) return SPF_ERR_SHAPE;
  if (ceil_div(n_tokens, block_size) > 65535 * 16) return SPF_ERR_TOO_LARGE;
  PoolParams p;
  std::memset(&p, 0, sizeof(p));
  p.n_tokens = n_tokens; p.head_dim = head_dim; p.block_size = block_size;
  const int cph = head_dim / 8;
  if (q) {
    if (!aligned16(q) || !aligned16(avg_q) || !strides_ok(q_stride_n, q_stride_h)) return SPF_ERR_ALIGN;
    if (n_q_heads <= 0) return SPF_ERR_SHAPE;
    p.t[0] = PoolTensor{static_cast<const __nv_bfloat16*>(q), q_stride_n, q_stride_h,
                        static_cast<__nv_bfloat16*>(avg_q), n_q_heads, ceil_div(n_q_heads * cph, 128), 1};
  }
  if (k) {
    if (!aligned16(k) || !aligned16(avg_k) || !strides_ok(k_stride_n, k_stride_h)) return SPF_ERR_ALIGN;
    if (n_kv_heads <= 0) return SPF_ERR_SHAPE;
    p.t[1] = PoolTensor{static_cast<const __nv_bfloat16*>(k), k_stride_n, k_stride_h,
                        static_cast<__nv_bfloat16*>(avg_k), n_kv_heads, ceil_div(n_kv_heads * cph, 128), 0};
  }
  return pool_blocks(p, ceil_div(n_tokens, block_size), static_cast<cudaStream_t>(stream));
}

int64_t spf_lastblock_scratch_bytes(int n_tokens, int n_q_heads, int block_size) {
  (void)block_size;
  if (n_tokens <= 0 || n_q_heads <= 0) return 0;
  const int64_t ntiles = ceil_div(n_tokens, 128);
  return align256(int64_t(n_q_heads) * ntiles * 128 * 4) * 2 + align256(int64_t(n_q_heads) * 128 * 4) * 2;
}

int spf_lastblock_profile(const void* q, int64_t q_stride_n, int64_t q_stride_h, const void* k,
                          int64_t k_stride_n, int64_t k_stride_h, int n_tokens, int n_q_heads,
                          int n_kv_heads, int head_dim, int block_size, float* vertical, float* slash,
                          void* scratch, int64_t scratch_bytes, void* stream) {
  if (!q || !k || !vertical || !slash || !scratch) return SPF_ERR_NULL;
  if (timeouts_tripped()) return SPF_ERR_TIMEOUT;
  int rc = check_shape(n_tokens, n_q_heads, n_kv_heads, head_dim, block_size);
  if (rc) return rc;
  if (!aligned16(q) || !aligned16(k) || !aligned16(scratch) || !strides_ok(q_stride_n, q_stride_h) ||
      !strides_ok(k_stride_n, k_stride_h))
    return SPF_ERR_ALIGN;
  if (scratch_bytes < spf_lastblock_scratch_bytes(n_tokens, n_q_heads, block_size)) return SPF_ERR_RANGE;
  EstParams p;
  p.q = static_cast<const __nv_bfloat16*>(q); p.q_sn = q_stride_n; p.q_sh = q_stride_h;
  p.k = static_cast<const __nv_bfloat16*>(k); p.k_sn = k_stride_n; p.k_sh = k_stride_h;
  p.n_tokens = n_tokens; p.n_q_heads = n_q_heads; p.group = n_q_heads / n_kv_heads;
  p.rq = block_size; p.ntiles = ceil_div(n_tokens, 128); p.n_parts = p.ntiles;
  int tpc = (p.ntiles * n_q_heads) / (148 * 8);
  p.tiles_per_cta = tpc < 1 ? 1 : (tpc > 8 ? 8 : tpc);
  p.sqrt_d = static_cast<float>(std::sqrt(static_cast<double>(head_dim)));
  char* s = static_cast<char*>(scratch);
  const int64_t part = align256(int64_t(n_q_heads) * p.ntiles * 128 * 4);
  const int64_t rows = align256(int64_t(n_q_heads) * 128 * 4);
  p.part_m = reinterpret_cast<float*>(s);
  p.part_l = reinterpret_cast<float*>(s + part);
  p.row_m = reinterpret_cast<float*>(s + 2 * part);
  p.row_z = reinterpret_cast<float*>(s + 2 * part + rows);
  p.vertical = vertical; p.slash = slash;
  return lastblock_profile(p, head_dim, static_cast<cudaStream_t>(stream));
}

int spf_profile_budgets(const float* vertical, const float* slash, int n_heads, int n_tokens, int block_size,
                        double pattern_threshold, int min_blocks, int max_blocks, int32_t* nv, int32_t* ns,
                        float* vpool, float* spool, void* stream) {
  if (!vertical || !slash || !nv || !ns || !vpool || !spool) return SPF_ERR_NULL;
  if (n_heads <= 0 || n_tokens <= 0 || block_size <= 0) return SPF_ERR_SHAPE;
  if (n_heads > SPF_MAX_HEADS || ceil_div(n_tokens, block_size) > SPF_MAX_BLOCKS) return SPF_ERR_TOO_LARGE;
  BudgetParams p;
  p.vertical = vertical; p.slash = slash; p.n_heads = n_heads; p.n_tokens = n_tokens;
  p.block_size = block_size; p.nb = ceil_div(n_tokens, block_size);
  p.thr = static_cast<float>(pattern_threshold);
  p.min_blocks = min_blocks; p.max_blocks = max_blocks < p.nb ? max_blocks : p.nb;
  p.nv = nv; p.ns = ns; p.vpool = vpool; p.spool = spool;
  return launch_budgets(p, static_cast<cudaStream_t>(stream));
}

int spf_pooled_last_row(const void* q, int64_t q_stride_n, int64_t q_stride_h, const void* avg_k, int n_tokens,
                        int n_q_heads, int n_kv_heads, int head_dim, int block_size, float* avg_qk,
                        void* stream) {
  if (!q || !avg_k || !avg_qk) return SPF_ERR_NULL;
  int rc = check_shape(n_tokens, n_q_heads, n_kv_heads, head_dim, block_size);
  if (rc) return rc;
  if (!aligned16(avg_k)) return SPF_ERR_ALIGN;   // pooled key rows are read 16 bytes at a time
  LastRowParams p;
  p.q = static_cast<const __nv_bfloat16*>(q); p.q_sn = q_stride_n; p.q_sh = q_stride_h;
  p.avg_k = static_cast<const __nv_bfloat16*>(avg_k);
  p.n_tokens = n_tokens; p.n_q_heads = n_q_heads; p.n_kv_heads = n_kv_heads; p.head_dim = head_dim;
  p.block_size = block_size; p.nb = ceil_div(n_tokens, block_size);
  p.sqrt_d = static_cast<float>(std::sqrt(static_cast<double>(head_dim)));
  p.avg_qk = avg_qk;
  return launch_last_row(p, static_cast<cudaStream_t>(stream));
}

int64_t spf_sharing_state_bytes(int n_slots, int nb) {
  if (n_slots < 0 || nb <= 0 || nb > SPF_MAX_BLOCKS) return 0;
  int64_t off[13];
  state_offsets(n_slots > 0 ? n_slots : 1, nb, off);
  return off[12];
}

int spf_sharing_state_layout(int n_slots, int nb, int64_t* offsets) {
  if (!offsets) return SPF_ERR_NULL;
  if (n_slots < 0 || nb <= 0 || nb > SPF_MAX_BLOCKS) return SPF_ERR_RANGE;
  int64_t off[13];
  state_offsets(n_slots > 0 ? n_slots : 1, nb, off);
  for (int i = 0; i < 12; ++i) offsets[i] = off[i];
  return SPF_OK;
}

int spf_sharing_state_reset(void* state, int n_slots, int nb, void* stream) {
  if (!state) return SPF_ERR_NULL;
  if (n_slots < 0 || nb <= 0 || nb > SPF_MAX_BLOCKS) return SPF_ERR_RANGE;
  return launch_state_reset(state, n_slots > 0 ? n_slots : 1, nb, static_cast<cudaStream_t>(stream));
}

int spf_classify_heads(const float* avg_qk, const float* vpool, const float* spool, const int32_t* slot_of_head,
                       const void* state, int n_slots, int n_heads, int nb, float* jsd_qa, float* jsd_v,
                       float* jsd_s, void* stream) {
  if (!avg_qk || !vpool || !spool || !slot_of_head || !state || !jsd_qa || !jsd_v || !jsd_s) return SPF_ERR_NULL;
  if (n_heads <= 0 || n_heads > SPF_MAX_HEADS || nb <= 0 || nb > SPF_MAX_BLOCKS || n_slots < 0) return SPF_ERR_RANGE;
  ClassifyParams p;
  p.avg_qk = avg_qk; p.vpool = vpool; p.spool = spool; p.slot_of_head = slot_of_head;
  p.st = state_view(const_cast<void*>(state), n_slots > 0 ? n_slots : 1, nb);
  p.n_slots = n_slots; p.nb = nb; p.jsd_qa = jsd_qa; p.jsd_v = jsd_v; p.jsd_s = jsd_s;
  return launch_classify(p, n_heads, static_cast<cudaStream_t>(stream));
}

int spf_pairwise_sqrt_jsd(const float* x, int n_vec, int len, float* out, void* stream) {
  if (!x || !out) return SPF_ERR_NULL;
  if (n_vec <= 0 || n_vec > 65535 || len <= 0 || len > 2 * SPF_MAX_BLOCKS) return SPF_ERR_RANGE;
  return launch_pairwise_jsd(x, n_vec, len, out, static_cast<cudaStream_t>(stream));
}

int spf_elect_and_share(const float* jsd_qa_all, const int32_t* slot_of_head_all, int n_heads_total,
                        int head_offset, int n_heads, const float* jsd_v, const float* jsd_s,
                        const float* vpool, const float* spool, void* state, int n_slots, int nb, int layer,
                        double queryaware_threshold, double similarity_threshold, double fallback_threshold,
                        int min_blocks, int32_t* nv, int32_t* ns, int32_t* head_flags, void* stream) {
  if (!jsd_qa_all || !slot_of_head_all || !jsd_v || !jsd_s || !vpool || !spool || !state || !nv || !ns || !head_flags)
    return SPF_ERR_NULL;
  if (n_heads <= 0 || n_heads_total < n_heads || head_offset < 0 || head_offset + n_heads > n_heads_total ||
      n_heads_total > SPF_MAX_HEADS || nb <= 0 || nb > SPF_MAX_BLOCKS || n_slots < 0)
    return SPF_ERR_RANGE;
  ElectParams p;
  p.jsd_qa_all = jsd_qa_all; p.slot_of_head_all = slot_of_head_all; p.jsd_v = jsd_v; p.jsd_s = jsd_s;
  p.vpool = vpool; p.spool = spool;
  p.st = state_view(state, n_slots > 0 ? n_slots : 1, nb);
  p.n_slots = n_slots; p.nb = nb; p.layer = layer;
  p.n_heads_total = n_heads_total; p.head_offset = head_offset; p.n_heads = n_heads;
  p.qa_thr = static_cast<float>(queryaware_threshold);
  p.sim_thr = static_cast<float>(similarity_threshold);
  p.fb_thr = static_cast<float>(fallback_threshold);
  p.min_blocks = min_blocks; p.nv = nv; p.ns = ns; p.head_flags = head_flags;
  return launch_elect(p, static_cast<cudaStream_t>(stream));
}

int spf_build_vs_bitmap(const float* vpool, const float* spool, const int32_t* nv, const int32_t* ns,
                        const int32_t* head_flags, const int32_t* slot_of_head, void* state, int n_slots,
                        int n_heads, int nb, uint32_t* bitmap, void* stream) {
  if (!vpool || !spool || !nv || !ns || !head_flags || !slot_of_head || !state || !bitmap) return SPF_ERR_NULL;
  if (n_heads <= 0 || n_heads > SPF_MAX_HEADS || nb <= 0 || nb > SPF_MAX_BLOCKS || n_slots < 0) return SPF_ERR_RANGE;
  VsParams p;
  p.vpool = vpool; p.spool = spool; p.nv = nv; p.ns = ns; p.head_flags = head_flags;
  p.slot_of_head = slot_of_head; p.st = state_view(state, n_slots > 0 ? n_slots : 1, nb);
  p.n_slots = n_slots; p.nb = nb; p.nbw = (nb + 31) / 32; p.bitmap = bitmap;
  return launch_vs_bitmap(p, n_heads, static_cast<cudaStream_t>(stream));
}

int spf_query_aware_scores(const void* avg_q, const void* avg_k, const int32_t* head_flags, int n_q_heads,
                           int n_kv_heads, int head_dim, int nb, float* scores, void* stream) {
  if (!avg_q || !avg_k || !scores) return SPF_ERR_NULL;
  if (!supported_head_dim(head_dim) || n_q_heads <= 0 || n_kv_heads <= 0 || n_q_heads % n_kv_heads) return SPF_ERR_SHAPE;
  if (n_q_heads > SPF_MAX_HEADS || nb <= 0 || nb > SPF_MAX_BLOCKS) return SPF_ERR_TOO_LARGE;
  if (!aligned16(avg_k)) return SPF_ERR_ALIGN;   // pooled key rows are read 16 bytes at a time
  QaScoreParams p;
  p.avg_q = static_cast<const __nv_bfloat16*>(avg_q); p.avg_k = static_cast<const __nv_bfloat16*>(avg_k);
  p.head_flags = head_flags; p.n_q_heads = n_q_heads; p.n_kv_heads = n_kv_heads; p.head_dim = head_dim;
  p.nb = nb; p.sqrt_d = static_cast<float>(std::sqrt(static_cast<double>(head_dim))); p.scores = scores;
  return launch_qa_scores(p, static_cast<cudaStream_t>(stream));
}

int spf_query_aware_select(const float* scores, const int32_t* head_flags, int n_heads, int nb,
                           double pattern_threshold, uint32_t* bitmap, void* stream) {
  if (!scores || !bitmap) return SPF_ERR_NULL;
  if (n_heads <= 0 || n_heads > SPF_MAX_HEADS || nb <= 0 || nb > SPF_MAX_BLOCKS) return SPF_ERR_RANGE;
  QaSelectParams p;
  p.scores = scores; p.head_flags = head_flags; p.nb = nb; p.nbw = (nb + 31) / 32;
  p.thr = static_cast<float>(pattern_threshold * static_cast<double>(nb));
  p.scale_bits = 60 - log2_ceil(nb) - 1;
  p.bitmap = bitmap;
  return launch_qa_select(p, n_heads, static_cast<cudaStream_t>(stream));
}

int spf_bitmap_row_counts(const uint32_t* bitmap, int n_heads, int nb, int32_t* row_counts, int64_t* head_totals,
                          void* stream) {
  if (!bitmap || !row_counts) return SPF_ERR_NULL;
  if (n_heads <= 0 || nb <= 0 || nb > SPF_MAX_BLOCKS) return SPF_ERR_RANGE;
  return launch_row_counts(bitmap, n_heads, nb, row_counts, head_totals, static_cast<cudaStream_t>(stream));
}

int spf_sparse_attention(const void* q, int64_t q_stride_n, int64_t q_stride_h, const void* k, int64_t k_stride_n,
                         int64_t k_stride_h, const void* v, int64_t v_stride_n, int64_t v_stride_h, int n_tokens,
                         int n_q_heads, int n_kv_heads, int head_dim, int block_size, double softmax_scale,
                         const uint32_t* bitmap, const int32_t* head_flags, const int32_t* slot_of_head,
                         void* state, int n_slots, void* out, void* stream) {
  if (!q || !k || !v || !bitmap || !out) return SPF_ERR_NULL;
  if (timeouts_tripped()) return SPF_ERR_TIMEOUT;
  int rc = check_shape(n_tokens, n_q_heads, n_kv_heads, head_dim, block_size);
  if (rc) return rc;
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(out) || !strides_ok(q_stride_n, q_stride_h) ||
      !strides_ok(k_stride_n, k_stride_h) || !strides_ok(v_stride_n, v_stride_h))
    return SPF_ERR_ALIGN;
  AttnParams p;
  p.q = static_cast<const __nv_bfloat16*>(q); p.q_sn = q_stride_n; p.q_sh = q_stride_h;
  p.k = static_cast<const __nv_bfloat16*>(k); p.k_sn = k_stride_n; p.k_sh = k_stride_h;
  p.v = static_cast<const __nv_bfloat16*>(v); p.v_sn = v_stride_n; p.v_sh = v_stride_h;
  p.out = static_cast<__nv_bfloat16*>(out); p.bitmap = bitmap;
  const bool with_state = head_flags && slot_of_head && state && n_slots > 0;
  p.head_flags = with_state ? head_flags : nullptr;
  p.slot_of_head = with_state ? slot_of_head : nullptr;
  p.pivot_attn = with_state ? state_view(state, n_slots, ceil_div(n_tokens, block_size)).pivot_attn : nullptr;
  p.n_tokens = n_tokens; p.n_q_heads = n_q_heads; p.group = n_q_heads / n_kv_heads;
  p.nb = ceil_div(n_tokens, block_size); p.nbw = (p.nb + 31) / 32;
  p.scale_log2 = static_cast<float>(softmax_scale * 1.4426950408889634);
  p.pivot_only = 0;
  p.n_slots = with_state ? n_slots : 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  // block_size = head_dim = 128 runs on the tcgen05 kernel; spf_force_generic_kernels (a test hook)
  // keeps the mma.sync kernel, which also serves every other supported shape
  const bool want_tc5 = block_size == 128 && head_dim == 128 &&
                        g_force_generic_attention.load(std::memory_order_relaxed) == 0;
  if (want_tc5) {
    rc = sparse_attention_tc5(p, n_kv_heads, st);
    if (rc == SPF_OK) {
      if (!with_state) return SPF_OK;
      p.pivot_only = 1;   // pivot heads: the block-mass matrix comes from the two-sweep kernel
      return sparse_attention_generic(p, block_size, head_dim, st);
    }
    if (rc != SPF_ERR_SHAPE) return rc;
  }
  return sparse_attention_generic(p, block_size, head_dim, st);
}

// Token splits of the decode pass: about two CTAs per SM over (splits x CTA rows), at least four
// 16-token tiles per split, every split non-empty.
static int decode_splits(int n_keys, int n_q_heads, int n_kv_heads) {
  const int rows = (n_q_heads / n_kv_heads <= 16) ? n_kv_heads : n_q_heads;   // CTA rows of the grid
  const int tiles = (n_keys + 15) / 16;
  int s = (2 * 148 + rows - 1) / rows;
  if (s > (tiles + 3) / 4) s = (tiles + 3) / 4;
  if (s > 256) s = 256;
  if (s < 1) s = 1;
  const int per = (tiles + s - 1) / s;
  return (tiles + per - 1) / per;
}

int64_t spf_decode_scratch_bytes(int n_keys, int n_q_heads, int n_kv_heads, int head_dim) {
  if (n_keys <= 0 || n_q_heads <= 0 || n_kv_heads <= 0 || n_q_heads % n_kv_heads || !supported_head_dim(head_dim))
    return 0;
  return align256(int64_t(n_q_heads) * decode_splits(n_keys, n_q_heads, n_kv_heads) * (head_dim + 2) * 4);
}

int spf_decode_attention(const void* q, int64_t q_stride_h, const void* k, int64_t k_stride_n, int64_t k_stride_h,
                         const void* v, int64_t v_stride_n, int64_t v_stride_h, int n_keys, int n_q_heads,
                         int n_kv_heads, int head_dim, double softmax_scale, void* out, void* scratch,
                         int64_t scratch_bytes, void* stream) {
  if (!q || !k || !v || !out || !scratch) return SPF_ERR_NULL;
  if (!supported_head_dim(head_dim) || n_keys <= 0 || n_q_heads <= 0 || n_kv_heads <= 0 || n_q_heads % n_kv_heads)
    return SPF_ERR_SHAPE;
  if (n_q_heads > SPF_MAX_HEADS) return SPF_ERR_TOO_LARGE;
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(out) || !aligned16(scratch) ||
      q_stride_h % 8 || !strides_ok(k_stride_n, k_stride_h) || !strides_ok(v_stride_n, v_stride_h))
    return SPF_ERR_ALIGN;
  if (scratch_bytes < spf_decode_scratch_bytes(n_keys, n_q_heads, n_kv_heads, head_dim)) return SPF_ERR_RANGE;
  DecodeParams p;
  p.q = static_cast<const __nv_bfloat16*>(q); p.q_sh = q_stride_h;
  p.k = static_cast<const __nv_bfloat16*>(k); p.k_sn = k_stride_n; p.k_sh = k_stride_h;
  p.v = static_cast<const __nv_bfloat16*>(v); p.v_sn = v_stride_n; p.v_sh = v_stride_h;
  p.out = static_cast<__nv_bfloat16*>(out); p.scratch = static_cast<float*>(scratch);
  p.n_keys = n_keys; p.n_q_heads = n_q_heads; p.group = n_q_heads / n_kv_heads;
  p.splits = decode_splits(n_keys, n_q_heads, n_kv_heads);
  p.scale_log2 = static_cast<float>(softmax_scale * 1.4426950408889634);
  return decode_attention(p, head_dim, static_cast<cudaStream_t>(stream));
}

// log2 of a supported page size, or -1
static int page_shift_of(int page_size) {
  for (int s = 4; s <= 8; ++s)
    if (page_size == 1 << s) return s;
  return -1;
}

int spf_paged_plan(const int32_t* cached_len, const int32_t* new_len, int n_requests, int page_size,
                   int32_t* block_table, int64_t table_stride, int table_width, const int32_t* free_ring,
                   int ring_capacity, const int32_t* ring_state, int32_t* ring_state_out, int32_t* cu_new,
                   int32_t* seq_len, int64_t* slot_map, int32_t* positions, int32_t* refused, int n_rows, void* stream) {
  if (!cached_len || !new_len || !block_table || !free_ring || !ring_state || !ring_state_out || !cu_new || !seq_len ||
      !refused || (n_rows > 0 && (!slot_map || !positions)))
    return SPF_ERR_NULL;
  if (page_shift_of(page_size) < 0) return SPF_ERR_SHAPE;
  if (n_requests <= 0 || n_rows < 0 || table_width <= 0 || table_stride < table_width || ring_capacity <= 0)
    return SPF_ERR_RANGE;
  if (n_requests > SPF_MAX_REQUESTS || n_rows > SPF_MAX_KEYS) return SPF_ERR_TOO_LARGE;
  PlanParams p;
  p.cached_len = cached_len; p.new_len = new_len; p.n_requests = n_requests; p.page_shift = page_shift_of(page_size);
  p.table = block_table; p.table_stride = table_stride; p.table_width = table_width;
  p.ring = free_ring; p.ring_capacity = ring_capacity; p.ring_state = ring_state; p.ring_state_out = ring_state_out;
  p.cu_new = cu_new; p.seq_len = seq_len; p.slot_map = slot_map; p.positions = positions; p.refused = refused;
  p.n_rows = n_rows;
  return launch_paged_plan(p, static_cast<cudaStream_t>(stream));
}

int spf_paged_write(const void* k, int64_t k_stride_n, int64_t k_stride_h, const void* v, int64_t v_stride_n,
                    int64_t v_stride_h, const int64_t* slot_map, int n_rows, int n_kv_heads, int head_dim,
                    void* k_cache, int64_t k_stride_page, int64_t k_stride_token, int64_t k_stride_head,
                    void* v_cache, int64_t v_stride_page, int64_t v_stride_token, int64_t v_stride_head, int n_pages,
                    int page_size, void* stream) {
  if (n_rows == 0) return SPF_OK;
  if (!k || !v || !slot_map || !k_cache || !v_cache) return SPF_ERR_NULL;
  const int shift = page_shift_of(page_size);
  if (!supported_head_dim(head_dim) || n_kv_heads <= 0 || shift < 0) return SPF_ERR_SHAPE;
  if (n_rows < 0 || n_pages <= 0) return SPF_ERR_RANGE;
  if (n_kv_heads > SPF_MAX_HEADS) return SPF_ERR_TOO_LARGE;
  if (!aligned16(k) || !aligned16(v) || !aligned16(k_cache) || !aligned16(v_cache) || !strides_ok(k_stride_n, k_stride_h) ||
      !strides_ok(v_stride_n, v_stride_h) || !strides_ok(k_stride_page, k_stride_token) || k_stride_head % 8 ||
      !strides_ok(v_stride_page, v_stride_token) || v_stride_head % 8)
    return SPF_ERR_ALIGN;
  // several elements in one place (an expanded view) would be written in no order
  const bool heads = n_kv_heads > 1, pages = n_pages > 1;
  if (k_stride_token == 0 || v_stride_token == 0 || (heads && (k_stride_head == 0 || v_stride_head == 0)) ||
      (pages && (k_stride_page == 0 || v_stride_page == 0)))
    return SPF_ERR_RANGE;
  WriteParams p;
  p.k = WriteTensor{static_cast<const uint16_t*>(k), k_stride_n, k_stride_h, static_cast<uint16_t*>(k_cache),
                    k_stride_page, k_stride_token, k_stride_head};
  p.v = WriteTensor{static_cast<const uint16_t*>(v), v_stride_n, v_stride_h, static_cast<uint16_t*>(v_cache),
                    v_stride_page, v_stride_token, v_stride_head};
  p.slot_map = slot_map; p.n_slots = int64_t(n_pages) << shift;
  p.n_rows = n_rows; p.n_kv_heads = n_kv_heads; p.chunk_shift = head_dim == 128 ? 4 : 3; p.page_shift = shift;
  return launch_paged_write(p, static_cast<cudaStream_t>(stream));
}

// what the two attention entry points check alike
static int check_ragged(int n_q_heads, int n_kv_heads, int head_dim, int dtype, double softmax_scale, int window, int sinks) {
  if (!supported_head_dim(head_dim) || n_q_heads <= 0 || n_kv_heads <= 0 || n_q_heads % n_kv_heads) return SPF_ERR_SHAPE;
  if (n_q_heads > SPF_MAX_HEADS) return SPF_ERR_TOO_LARGE;
  const float scale_log2 = static_cast<float>(softmax_scale * 1.4426950408889634);
  if ((dtype != SPF_BF16 && dtype != SPF_FP16) || !std::isfinite(scale_log2) || !(scale_log2 > 0.f) || window < 0 || sinks < 0)
    return SPF_ERR_RANGE;
  return SPF_OK;
}

// Batches whose requests all bring up to 16 rows per KV head (single tokens) go to the bandwidth-bound kernel, others to the
// tcgen05 one.  Tensors that TMA cannot describe (strides of 0 in expanded views) go to the first kernel whole.
static bool few_rows(int group, int max_new) { return int64_t(group) * max_new <= RAGGED_FEW_ROWS; }

// Chunks and single tokens in one batch: a pass of each kernel over its own requests, or all of them through the tcgen05
// kernel, whose 128-row tiles single tokens leave nearly empty.  The second pass costs 10 - 30 us, a token in the wrong kernel
// 0.04 us per 1000 keys of a KV head.  The host knows neither lengths nor which requests are which: of n_rows what passes one token
// a request is taken for as few chunks as can hold it, and a token for half of the table or its window, and 512 keys for its
// tile.  us in two passes
// / one, two chunks of 509 behind up to 16K keys and 4, 16, 20, 24 and 28 tokens with a window of 4096, 32q/8kv, D = 128:
// 120.3 / 89.5, 152.4 / 135.5, 162.1 / 154.7, 173.3 / 173.0, 183.4 / 185.7; D = 64: 92.4 / 75.6, 119.2 / 112.9, 125.8 / 122.8, 131.1
// / 136.2, 136.5 / 148.5.  Without a window, D = 128: 4 tokens 238 / 220, 12 300 / 296, 20 343 / 369; 64 of them 594 / 745; 64 with
// 2K keys 155 / 148 (D = 64 113 / 133); 254 with 500 keys 169 / 211.
constexpr int64_t MIXED_KEYS_128 = 920 * 1024, MIXED_KEYS_64 = 700 * 1024, TILE_KEYS = 512;

static bool two_passes(const RaggedParams& p, int max_new, int head_dim) {
  if (p.n_requests < 2 || p.group > RAGGED_FEW_ROWS || p.n_rows >= int64_t(p.n_requests) * max_new) return false;
  // (max_new >= 2: one token of at most 16 heads is a matter of the first kernel)
  const int64_t over = std::max(p.n_rows - p.n_requests, 0), chunks = (over + max_new - 2) / (max_new - 1);
  int64_t keys = (int64_t(p.table_width) << p.page_shift) / 2;
  if (p.window > 0) keys = std::min(keys, int64_t(p.window) + p.sinks);
  return (p.n_requests - chunks) * p.n_kv_heads * (keys + TILE_KEYS) > (head_dim == 128 ? MIXED_KEYS_128 : MIXED_KEYS_64);
}

// Single tokens with a worker per warp instead of one per CTA: from this many items on, at D = 128.  us with a worker per CTA /
// per warp, 32q/8kv: 64 requests up to 32 keys 18.6 / 16.9, 500 keys 39.6 / 32.1, 3000 91.1 / 90.3, 8192 215.9 / 215.9; 96
// requests up to 500 keys 56.2 / 42.4; 32 requests up to 500 keys 27.5 / 23.0, but 3000 keys 50.1 / 52.4 and 8192 keys 112.5 /
// 114.0.  At D = 64 (96 requests): 500 keys 34.5 / 33.6, 8192 keys 184.6 / 192.2.
constexpr int SOLO_ITEMS = 512;

// A CTA counts the units that it runs through in 32 bits, and so does the search for its start over 128 tiles at a time.
// (The bound takes every request for as long as its table; what it refuses would run for minutes to hours.)
static int64_t line_keys(const RaggedParams& p) { return p.table ? int64_t(p.table_width) << p.page_shift : p.seq_one; }
static bool line_fits(const RaggedParams& p) {
  int64_t keys = line_keys(p);
  if (p.window > 0) keys = std::min(keys, int64_t(p.window) + p.sinks + p.tile_tokens);
  const int64_t units = (keys >> p.unit_shift) + 3, items = (int64_t(p.n_rows / p.tile_tokens) + p.n_requests) * p.n_kv_heads * p.head_chunks;
  return units < (int64_t(1) << 24) && double(units) * double(items) < 2147483647.0 * p.n_ctas;
}

static int run_pass(RaggedParams p, bool tc5, int only, int max_new, int head_dim, cudaStream_t st) {
  p.only = only; p.head_dim = head_dim;
  const bool solo = head_dim == 128 && few_rows(p.group, max_new) && p.n_requests * p.n_kv_heads >= SOLO_ITEMS &&
                    line_keys(p) <= SPF_MAX_KEYS / 2;       // (units of 16 keys)
  if (tc5) ragged_tc5_config(p); else ragged_rows_config(p, solo);
  if (!line_fits(p)) return SPF_ERR_TOO_LARGE;
  int rc = ragged_schedule(p, max_new, st);
  if (rc == SPF_OK) rc = tc5 ? ragged_tc5_attention(p, head_dim, st) : ragged_rows_attention(p, head_dim, st);
  if (rc == SPF_OK) rc = ragged_merge(p, max_new, head_dim, st);
  return rc;
}

static int run_ragged(RaggedParams& p, int max_new, int head_dim, int64_t scratch_bytes, cudaStream_t st) {
  if (scratch_bytes < spf_paged_scratch_bytes(max_new, p.n_q_heads, p.n_kv_heads, head_dim)) return SPF_ERR_RANGE;
  if (few_rows(p.group, max_new) || !ragged_tc5_describable(p)) return run_pass(p, false, 0, max_new, head_dim, st);
  if (timeouts_tripped()) return SPF_ERR_TIMEOUT;
  if (!two_passes(p, max_new, head_dim)) return run_pass(p, true, 0, max_new, head_dim, st);
  const int rc = run_pass(p, false, 1, RAGGED_FEW_ROWS / p.group, head_dim, st);
  return rc == SPF_OK ? run_pass(p, true, 2, max_new, head_dim, st) : rc;
}

int64_t spf_paged_scratch_bytes(int max_new, int n_q_heads, int n_kv_heads, int head_dim) {
  if (max_new <= 0 || check_ragged(n_q_heads, n_kv_heads, head_dim, SPF_BF16, 1.0, 0, 0) != SPF_OK) return 0;
  RaggedParams p;
  std::memset(&p, 0, sizeof(p));
  p.group = n_q_heads / n_kv_heads; p.head_dim = head_dim;
  ragged_rows_config(p, head_dim == 128);
  const int64_t rows = ragged_scratch_bytes(p.n_ctas, p.tile_rows, head_dim);
  if (few_rows(p.group, max_new)) return rows;
  ragged_tc5_config(p);
  const int64_t tc5 = ragged_scratch_bytes(p.n_ctas, p.tile_rows, head_dim);
  return tc5 > rows ? tc5 : rows;
}

int spf_paged_attention(const void* q, int64_t q_stride_n, int64_t q_stride_h, int n_rows, int n_q_heads,
                        const void* k_cache, int64_t k_stride_page, int64_t k_stride_token, int64_t k_stride_head,
                        const void* v_cache, int64_t v_stride_page, int64_t v_stride_token, int64_t v_stride_head,
                        int n_pages, int page_size, int n_kv_heads, int head_dim, int dtype, const int32_t* block_table,
                        int64_t table_stride, int table_width, const int32_t* cu_new, const int32_t* seq_len,
                        int n_requests, int max_new, double softmax_scale, int window, int sinks, void* out,
                        void* scratch, int64_t scratch_bytes, void* stream) {
  if (n_rows == 0) return SPF_OK;
  if (!q || !k_cache || !v_cache || !block_table || !cu_new || !seq_len || !out || !scratch) return SPF_ERR_NULL;
  const int rc = check_ragged(n_q_heads, n_kv_heads, head_dim, dtype, softmax_scale, window, sinks);
  if (rc) return rc;
  const int shift = page_shift_of(page_size);
  if (shift < 0) return SPF_ERR_SHAPE;
  if (n_rows < 0 || n_pages <= 0 || n_requests <= 0 || max_new <= 0 || table_width <= 0 || table_stride < table_width)
    return SPF_ERR_RANGE;
  if (n_requests > SPF_MAX_REQUESTS || (int64_t(table_width) << shift) > SPF_MAX_KEYS || n_rows > SPF_MAX_KEYS)
    return SPF_ERR_TOO_LARGE;
  if (!aligned16(q) || !aligned16(k_cache) || !aligned16(v_cache) || !aligned32(out) || !aligned32(scratch) ||
      !strides_ok(q_stride_n, q_stride_h) || !strides_ok(k_stride_page, k_stride_token) || k_stride_head % 8 ||
      !strides_ok(v_stride_page, v_stride_token) || v_stride_head % 8)
    return SPF_ERR_ALIGN;
  RaggedParams p;
  std::memset(&p, 0, sizeof(p));
  p.q = q; p.q_sn = q_stride_n; p.q_sh = q_stride_h;
  p.k = k_cache; p.k_sp = k_stride_page; p.k_st = k_stride_token; p.k_sh = k_stride_head;
  p.v = v_cache; p.v_sp = v_stride_page; p.v_st = v_stride_token; p.v_sh = v_stride_head;
  p.out = out; p.table = block_table; p.table_stride = table_stride; p.table_width = table_width;
  p.n_pages = n_pages; p.page_shift = shift;
  p.cu = cu_new; p.seq = seq_len; p.n_requests = n_requests; p.n_rows = n_rows;
  p.n_q_heads = n_q_heads; p.n_kv_heads = n_kv_heads; p.group = n_q_heads / n_kv_heads;
  p.window = window < SPF_MAX_KEYS ? window : 0; p.sinks = sinks < SPF_MAX_KEYS ? sinks : SPF_MAX_KEYS;
  p.scale_log2 = static_cast<float>(softmax_scale * 1.4426950408889634);
  p.fp16 = dtype == SPF_FP16; p.scratch = static_cast<char*>(scratch);
  return run_ragged(p, max_new, head_dim, scratch_bytes, static_cast<cudaStream_t>(stream));
}

int spf_window_attention(const void* q, int64_t q_stride_n, int64_t q_stride_h, const void* k, int64_t k_stride_n,
                         int64_t k_stride_h, const void* v, int64_t v_stride_n, int64_t v_stride_h, int n_new,
                         int n_keys, int n_q_heads, int n_kv_heads, int head_dim, int dtype, double softmax_scale,
                         int window, int sinks, void* out, void* scratch, int64_t scratch_bytes, void* stream) {
  if (n_new == 0) return SPF_OK;
  if (!q || !k || !v || !out || !scratch) return SPF_ERR_NULL;
  const int rc = check_ragged(n_q_heads, n_kv_heads, head_dim, dtype, softmax_scale, window, sinks);
  if (rc) return rc;
  if (n_new < 0 || n_keys < n_new) return SPF_ERR_RANGE;
  if (n_keys > SPF_MAX_KEYS) return SPF_ERR_TOO_LARGE;
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned32(out) || !aligned32(scratch) ||
      !strides_ok(q_stride_n, q_stride_h) || !strides_ok(k_stride_n, k_stride_h) || !strides_ok(v_stride_n, v_stride_h))
    return SPF_ERR_ALIGN;
  RaggedParams p;
  std::memset(&p, 0, sizeof(p));
  p.q = q; p.q_sn = q_stride_n; p.q_sh = q_stride_h;
  p.k = k; p.k_st = k_stride_n; p.k_sh = k_stride_h;
  p.v = v; p.v_st = v_stride_n; p.v_sh = v_stride_h;
  p.out = out; p.n_pages = 1;
  p.n_requests = 1; p.n_rows = n_new; p.seq_one = n_keys;
  p.n_q_heads = n_q_heads; p.n_kv_heads = n_kv_heads; p.group = n_q_heads / n_kv_heads;
  p.window = window < SPF_MAX_KEYS ? window : 0; p.sinks = sinks < SPF_MAX_KEYS ? sinks : SPF_MAX_KEYS;
  p.scale_log2 = static_cast<float>(softmax_scale * 1.4426950408889634);
  p.fp16 = dtype == SPF_FP16; p.scratch = static_cast<char*>(scratch);
  return run_ragged(p, n_new, head_dim, scratch_bytes, static_cast<cudaStream_t>(stream));
}

int spf_packed_call(int function, const void* words) {
  // kinds of the parameters: p pointer, l 64-bit integer, d double, i int
  static const char* const kinds[4] = {"ppiiplipipppppppip", "pllpllpiiiplllpllliip", "plliiplllplll" "iiiii" "plippii" "diipplp",
                                       "pllpllplliiiiiidiipplp"};
  if (!words) return SPF_ERR_NULL;
  if (function < 0 || function > 3) return SPF_ERR_RANGE;
  int64_t w[32];
  const int n = int(std::strlen(kinds[function]));
  std::memcpy(w, words, size_t(n) * 8);
  for (int i = 0; i < n; ++i)
    if (kinds[function][i] == 'i' && w[i] != int64_t(int(w[i]))) return SPF_ERR_RANGE;
  auto p = [&](int i) { return reinterpret_cast<void*>(w[i]); };
  auto i32 = [&](int i) { return static_cast<int32_t*>(p(i)); };
  auto i = [&](int k) { return int(w[k]); };
  double d;
  switch (function) {
    case SPF_PACKED_PAGED_PLAN:
      return spf_paged_plan(i32(0), i32(1), i(2), i(3), i32(4), w[5], i(6), i32(7), i(8), i32(9), i32(10), i32(11), i32(12),
                            static_cast<int64_t*>(p(13)), i32(14), i32(15), i(16), p(17));
    case SPF_PACKED_PAGED_WRITE:
      return spf_paged_write(p(0), w[1], w[2], p(3), w[4], w[5], static_cast<int64_t*>(p(6)), i(7), i(8), i(9), p(10), w[11], w[12],
                             w[13], p(14), w[15], w[16], w[17], i(18), i(19), p(20));
    case SPF_PACKED_PAGED_ATTENTION:
      std::memcpy(&d, &w[25], 8);
      return spf_paged_attention(p(0), w[1], w[2], i(3), i(4), p(5), w[6], w[7], w[8], p(9), w[10], w[11], w[12], i(13), i(14), i(15),
                                 i(16), i(17), i32(18), w[19], i(20), i32(21), i32(22), i(23), i(24), d, i(26), i(27), p(28), p(29),
                                 w[30], p(31));
    default:
      std::memcpy(&d, &w[15], 8);
      return spf_window_attention(p(0), w[1], w[2], p(3), w[4], w[5], p(6), w[7], w[8], i(9), i(10), i(11), i(12), i(13), i(14), d,
                                  i(16), i(17), p(18), p(19), w[20], p(21));
  }
}

int spf_device_timeouts(void) {
  const unsigned int n = tc5_timeout_count() + est_tc5_timeout_count() + ragged_tc5_timeout_count();
  g_known_timeouts.store(n, std::memory_order_relaxed);
  return static_cast<int>(n);
}

int spf_reset_device_timeouts(void) {
  if (!tc5_reset_timeouts() || !est_tc5_reset_timeouts() || !ragged_tc5_reset_timeouts()) return SPF_ERR_LAUNCH;
  g_known_timeouts.store(0, std::memory_order_relaxed);
  return SPF_OK;
}

int spf_set_device_wait_limit_ns(uint64_t ns) {
  if (ns == 0) return SPF_ERR_RANGE;
  return (tc5_set_wait_limit(ns) && est_tc5_set_wait_limit(ns) && ragged_tc5_set_wait_limit(ns)) ? SPF_OK : SPF_ERR_LAUNCH;
}

int spf_force_generic_kernels(int attention, int profile) {
  g_force_generic_attention.store(attention ? 1 : 0, std::memory_order_relaxed);
  g_force_generic_profile.store(profile ? 1 : 0, std::memory_order_relaxed);
  return SPF_OK;
}

int spf_wait_limit_selftest(void* stream) { return tc5_wait_limit_selftest(static_cast<cudaStream_t>(stream)); }

int spf_update_pivots(const int32_t* head_flags, const int32_t* slot_of_head, void* state, int n_slots, int n_heads,
                      int nb, double pattern_threshold, void* stream) {
  if (!head_flags || !slot_of_head || !state) return SPF_ERR_NULL;
  if (n_heads <= 0 || n_heads > SPF_MAX_HEADS || nb <= 0 || nb > SPF_MAX_BLOCKS || n_slots < 0) return SPF_ERR_RANGE;
  if (n_slots == 0) return SPF_OK;
  PivotParams p;
  p.head_flags = head_flags; p.slot_of_head = slot_of_head; p.st = state_view(state, n_slots, nb);
  p.n_slots = n_slots; p.nb = nb; p.nbw = (nb + 31) / 32; p.thr = static_cast<float>(pattern_threshold);
  return launch_update_pivots(p, n_heads, static_cast<cudaStream_t>(stream));
}

int64_t spf_pivot_summary_width(int nb) {
  if (nb <= 0 || nb > SPF_MAX_BLOCKS) return 0;
  return 2 + 2 * int64_t(nb) + int64_t(nb) * ((nb + 31) / 32);
}

int spf_pack_pivot_summaries(void* state, int n_slots, int nb, int layer, int head_begin, int head_end,
                             int32_t* packed, void* stream) {
  if (!state || !packed) return SPF_ERR_NULL;
  if (nb <= 0 || nb > SPF_MAX_BLOCKS || n_slots < 0 || head_begin < 0 || head_end < head_begin) return SPF_ERR_RANGE;
  if (n_slots == 0) return SPF_OK;
  return launch_pack_summaries(state, n_slots, nb, layer, head_begin, head_end, packed,
                               static_cast<cudaStream_t>(stream));
}

int spf_merge_pivot_summaries(void* state, int n_slots, int nb, const int32_t* gathered, int n_ranks,
                              void* stream) {
  if (!state || !gathered) return SPF_ERR_NULL;
  if (nb <= 0 || nb > SPF_MAX_BLOCKS || n_slots < 0 || n_ranks <= 0) return SPF_ERR_RANGE;
  if (n_slots == 0) return SPF_OK;
  return launch_merge_summaries(state, n_slots, nb, gathered, n_ranks, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
