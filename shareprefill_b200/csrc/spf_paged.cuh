// Parameter blocks of the paged cache's bookkeeping kernels (spf_paged.cu).
#pragma once

#include "spf_common.cuh"

namespace spf {

struct PlanParams {
  const int32_t* cached_len; const int32_t* new_len; int n_requests, page_shift;
  int32_t* table; int64_t table_stride; int table_width;
  const int32_t* ring; int ring_capacity; const int32_t* ring_state; int32_t* ring_state_out;
  int32_t* cu_new; int32_t* seq_len; int64_t* slot_map; int32_t* positions; int32_t* refused;
  int n_rows;
};

struct WriteTensor {
  const uint16_t* src; int64_t sn, sh;       // token and head strides
  uint16_t* dst; int64_t dp, dt, dh;         // page, token-in-page and head strides
};

struct WriteParams {
  WriteTensor k, v;
  const int64_t* slot_map; int64_t n_slots;
  int n_rows, n_kv_heads, chunk_shift, page_shift;   // chunk_shift: log2 of the 16-byte chunks per head
};

int launch_paged_plan(const PlanParams& p, cudaStream_t st);
int launch_paged_write(const WriteParams& p, cudaStream_t st);

}  // namespace spf
