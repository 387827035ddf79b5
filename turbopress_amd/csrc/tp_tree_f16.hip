// Attention of trees of drafted tokens over a paged cache, f16.
#include "tp_paged.h"

int tp::dispatch_tree_f16(const PagedArgs& a, hipStream_t s) { return dispatch_tree<f16_t>(a, s); }
