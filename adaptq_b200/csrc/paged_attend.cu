// Attention over the pages for one pair of bit widths (AQ_KB for keys, AQ_VB for values): the build compiles this file
// once for each.
#include "paged_attend.cuh"

#include <algorithm>
#include <atomic>

using namespace aq;

// The names below are the same in every unit: what differs between units carries the bit widths in its type.
struct AttendRoom { size_t query_scales, block_headers, block_slots, warp_slots, warp_sums, total; }; // offsets in the workspace

template <typename S> static AttendRoom attend_room(int blocks, int cols, size_t items) {
  const size_t slot = (size_t)cols * (S::DIM + 4) * sizeof(float);
  AttendRoom r;
  r.query_scales = items * (S::DIM / 8) * 128;
  r.block_headers = r.query_scales + items * 32;
  r.block_slots = r.block_headers + (size_t)blocks * sizeof(int4);
  r.warp_slots = r.block_slots + blocks * 2 * slot;
  r.warp_sums = r.warp_slots + (size_t)blocks * S::WARPS * 2 * slot;
  r.total = r.warp_sums + (size_t)blocks * S::WARPS * S::SUMS * sizeof(float);
  return r;
}

template <typename S> static bool launch_attend(const AttendCall &call) {
  AttendLaunch &a = *call.launch;
  const char *fn = call.fn;
  const int device = call.device, sms = aq_sm_count(device);
  a.passes = (a.group + S::COLS - 1) / S::COLS;
  a.slot_cols = std::min(S::COLS, a.group);
  const long long items = (long long)a.n_seqs * a.c.heads * a.passes;
  const AttendRoom room = attend_room<S>(sms, a.slot_cols, items);
  if (call.bytes) { *call.bytes = room.total; return true; }
  auto kernel = paged_attend_kernel<S::KEY_BITS, S::VALUE_BITS, S::DIM, S::KIND>;
  static std::atomic<unsigned long long> ready{0}; // devices on which the kernel may use its shared memory
  if (device >= 64 || !(ready.load() >> device & 1)) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM);
    if (e != cudaSuccess) { cudaGetLastError(); aq_set_error("%s: CUDA error: %s", fn, cudaGetErrorString(e)); return false; }
    if (device < 64) ready.fetch_or(1ull << device);
  }
  // no more blocks than the tables have room for units
  const long long most = items * ((((long long)a.table.width << a.c.page_shift) + S::U - 1) / S::U);
  if (most > 0x7fffffff || ((long long)a.table.width << a.c.page_shift) > 0x3fffffff) { aq_set_error("%s: the block tables have room for too many tokens for one call", fn); return false; }
  const int blocks = (int)std::max<long long>(1, std::min<long long>(sms, most));
  uint8_t *base = static_cast<uint8_t *>(call.workspace);
  a.operands = reinterpret_cast<uint32_t *>(base);
  a.query_scales = reinterpret_cast<float *>(base + room.query_scales);
  a.block_headers = reinterpret_cast<int4 *>(base + room.block_headers);
  a.block_slots = reinterpret_cast<float *>(base + room.block_slots);
  a.warp_slots = reinterpret_cast<float *>(base + room.warp_slots);
  a.warp_sums = reinterpret_cast<float *>(base + room.warp_sums);
  a.workspace_end = base + room.total;
  paged_query_kernel<S::DIM><<<(unsigned)items, QUERY_WARPS * 32, 0, call.stream>>>(
      a, S::COLS, 1.4426950408889634f / (S::DIM * table_scale(S::KEY_BITS)));
  if (!aq_launched(fn)) return false;
  // the other two start beside their predecessor and wait for it where they need its results
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.stream = call.stream;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  cfg.gridDim = dim3(blocks);
  cfg.blockDim = dim3(S::THREADS);
  cfg.dynamicSmemBytes = S::SMEM;
  cudaLaunchKernelEx(&cfg, kernel, a);
  if (!aq_launched(fn)) return false;
  cfg.gridDim = dim3(blocks, a.slot_cols);
  cfg.blockDim = dim3(JOIN_WARPS * 32);
  cfg.dynamicSmemBytes = 0;
  cudaLaunchKernelEx(&cfg, paged_join_kernel<S::DIM>, a, blocks, (int)S::COLS);
  return aq_launched(fn);
}

template <int KB, int VB, int P> static bool attend_p(const AttendCall &call) {
  if (call.mode == ATTEND_EIGHT) return launch_attend<AttendShape<KB, VB, P, ATTEND_EIGHT>>(call);
  if (call.mode == ATTEND_SPLIT) return launch_attend<AttendShape<KB, VB, P, ATTEND_SPLIT>>(call);
  return launch_attend<AttendShape<KB, VB, P, ATTEND_EXACT>>(call);
}

#define AQ_NAME_(k, v) aq_attend_##k##_##v
#define AQ_NAME(k, v) AQ_NAME_(k, v)
bool AQ_NAME(AQ_KB, AQ_VB)(const AttendCall &call) {
  return call.padded == 64 ? attend_p<AQ_KB, AQ_VB, 64>(call) : call.padded == 128 ? attend_p<AQ_KB, AQ_VB, 128>(call) : attend_p<AQ_KB, AQ_VB, 256>(call);
}
