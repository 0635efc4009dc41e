// The attention kernels' parameters and launchers (attention_rows.cu), and those of the cache kernels (cache_ops.cu). Host and device.
#pragma once

#include "attention_plan.cuh"

namespace qmm {

struct RowsParams {
  AttentionWork work;
  CacheView cache;             // pages
  const uint8_t* q;
  const uint8_t* k;            // rows
  const uint8_t* v;
  uint8_t* out;
  JoinNote* notes;
  float* partial;
  int64_t q_row, q_head, k_row, k_head, v_row, v_head;       // elements
  float scale_log2;
};

struct JoinParams {
  AttentionWork work;
  uint8_t* out;
  const JoinNote* notes;
  const float* partial;
};

int attend_rows_ctas();             // at most
int64_t attend_rows_workspace(int head_dim, int ctas);
// `source`: 0 rows, 1 pages of 16-bit values, 2 pages of e4m3 codes; `rows`: query rows that a sequence and key head have on average, which tiles of 16, 32 or 64 rows are
// chosen by (more of them are more tiles).
// CTAs of a cluster that takes a sequence's tiles of a key head, or 0: shares by weight.
int attend_cluster_ctas(const RowsParams& p, int source, int rows);
int launch_attend_rows(const RowsParams& p, int elem, int head_dim, int source, int rows, cudaStream_t stream);

// 128-row halves on tcgen05. A cache's rows have to be fewer than 2^31.
int attend_tc_ctas();
int64_t attend_tc_workspace(int head_dim, int ctas);
int launch_attend_tc(const RowsParams& p, int elem, int head_dim, int source, int ctas, cudaStream_t stream);

int launch_append(const CacheView& c, const qmm_append_args& a, int head_dim, bool e4m3, int* status, cudaStream_t stream);
int launch_cache_read(const CacheView& c, int64_t seqs, const int32_t* cu_kv, int64_t total, int head_dim, int elem, bool e4m3, void* k_out,
                      void* v_out, int* status, cudaStream_t stream);

}  // namespace qmm
