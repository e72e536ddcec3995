// Host-side checks shared by the entry points of the paged caches.
#pragma once

#include "paged.cuh"

namespace tq {

int paged_status_ptr(int** out);                       // the current device's status word
int check_paged_params(const tq_paged_params* p);      // sizes, table, lengths
int fill_page_view(const tq_paged_params* p, PageView* v);
// encode: rows are inserted (boundaries needed, `thresholds` filled); otherwise they are read (centroids needed)
int fill_paged_half(const tq_paged_half* h, int dim, const char* what, bool encode, bool need_signs, PagedHalf* out,
                    Table16* thresholds);

// Launches a kernel that may start while the kernel in front of it on the stream drains: it calls griddepcontrol.wait
// before it touches what that kernel may have written or still reads.
template <typename... P, typename... A>
int launch_dependent(const char* what, void (*kernel)(P...), dim3 grid, unsigned threads, unsigned smem, cudaStream_t st,
                     const A&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
  if (e != cudaSuccess) return set_error(TQ_ERR_LAUNCH, "%s: %s", what, cudaGetErrorString(e));
  return check_launch(what);
}

}  // namespace tq
