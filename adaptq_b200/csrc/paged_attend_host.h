// What the host side of the paged cache and the translation units of its attention kernels share.
#pragma once
#include "host_common.h"
#include "paged.cuh"

namespace aq {

struct AttendLaunch {
  PagedView c;
  RotaryView r;
  TableView table;
  const int *lengths;
  const void *q;
  void *out;
  long long q_seq, q_head, out_seq, out_head;
  int n_seqs, group, passes, type;
  float scale;
  int out_vec;
  // workspace: the queries as operands and their scales, a header per block, the blocks' partial results, the warps', the
  // warps' sums under way
  uint32_t *operands; // [item][P / 8][32]
  float *query_scales; // [item][8]
  int4 *block_headers;
  float *block_slots, *warp_slots, *warp_sums;
  const void *workspace_end; // for the checked build
  int slot_cols; // columns of a partial result
};

// MODE of the kernel: eight queries a pass, four in two parts, four in two parts with the codebook in two.
enum { ATTEND_EIGHT = 0, ATTEND_SPLIT = 1, ATTEND_EXACT = 2 };

// One call: of AttendLaunch the unit fills in what depends on its kernels (passes, slot_cols and the workspace).
struct AttendCall {
  const char *fn;
  AttendLaunch *launch;
  int padded, mode, device;
  void *workspace;
  cudaStream_t stream;
  size_t *bytes; // if set: only tell the size of the workspace
};

} // namespace aq

#define AQ_ATTEND_UNIT(k, v) AQ_HIDDEN bool aq_attend_##k##_##v(const aq::AttendCall &);
AQ_ATTEND_UNIT(2, 2) AQ_ATTEND_UNIT(2, 3) AQ_ATTEND_UNIT(2, 4)
AQ_ATTEND_UNIT(3, 2) AQ_ATTEND_UNIT(3, 3) AQ_ATTEND_UNIT(3, 4)
AQ_ATTEND_UNIT(4, 2) AQ_ATTEND_UNIT(4, 3) AQ_ATTEND_UNIT(4, 4)
#undef AQ_ATTEND_UNIT
