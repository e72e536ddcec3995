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

}  // namespace tq
