// Attention over packed prompts and over a paged K/V cache: what the kernel files and the launcher share.
#ifndef HALO_B200_ATTENTION_CUH_
#define HALO_B200_ATTENTION_CUH_

#include <cuda.h>

#include <cstdint>

#include "kernels.h"

namespace halo_b200 {

// One call as the kernels see it. Packed prompts are the case table == NULL: key j of sequence b is row cu[b] + j of
// one long page.
struct AttnCall {
  const uint32_t* cu;      // [batch + 1] first query row of each sequence
  const uint32_t* kv_len;  // [batch] keys of each sequence; NULL: as many as it has query rows
  const int32_t* table;    // [batch][table_stride] page of each block of keys; NULL: packed
  uint64_t table_stride;
  uint32_t table_cols, page_shift;
  uint32_t batch, tokens, kv_heads, group, dim;
  uint32_t box_shift;      // key rows of one copy: min(page size, 64), as a power of two
  int causal;
  float scale_log2;        // softmax scale * log2(e)
  void* out;
  uint64_t out_row, out_head;
  float* lse;              // [tokens][q heads] or NULL
  float* part;             // pieces of split jobs: see attention.cu
  uint32_t* meta;
};

// What one piece of a split job takes: 128 rows of fp32 sums, their maxima and denominators.
constexpr uint32_t kAttnRows = 128;
inline __host__ __device__ uint64_t AttnPieceFloats(uint32_t dim_pad) { return uint64_t{kAttnRows} * (dim_pad + 2); }

}  // namespace halo_b200

#endif  // HALO_B200_ATTENTION_CUH_
