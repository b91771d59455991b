// Parameters and launchers of the shared-prefix attention (fwd_prefix.cu).
#pragma once

#include "dsa_common.cuh"

namespace dsa {

struct PrefixParams {
  const __nv_bfloat16* q;       // [rows, 512]
  const __nv_bfloat16* q_rope;  // [rows, 64]
  const int32_t* length;        // keys in use, or null (all)
  __nv_bfloat16* out;           // without partials: [rows, 512], [rows], [rows]
  float* out_max;
  float* out_sum;
  float* part_num;              // [row tiles, split, 512 / 8, 128, 8] (groups of 8 columns), or null: write the output
  float* part_max;              // [row tiles, split, 128]
  float* part_sum;
  int32_t* status;
  long long rows;               // queries x heads, even
  int keys, split;
  int group;                    // row tiles of an item and CTAs of an MMA pair: 1 or 2
  float scale_div, scale_log2;
};

struct JoinParams {
  const float* part_num;        // as above
  const float* part_max;
  const float* part_sum;
  const float* own_num;         // [tokens, own_split, heads, 512]
  const float* own_max;         // [tokens, own_split, heads]
  const float* own_sum;
  __nv_bfloat16* out;
  float* out_max;
  float* out_sum;
  long long rows;
  int heads, split, own_split;
};

// Clusters of the prefix kernel with `group` row tiles that are resident at
// once (-1 on error).
int prefix_max_clusters(int group);
cudaError_t launch_fwd_prefix(const PrefixParams& p, const void* kv, const void* k_rope, cudaStream_t stream);
cudaError_t launch_prefix_join(const JoinParams& p, cudaStream_t stream);

}  // namespace dsa
