// Attention of trees of drafted tokens over a paged cache, bf16.
#include "tp_paged.h"

int tp::dispatch_tree_bf16(const PagedArgs& a, hipStream_t s) { return dispatch_tree<bf16_t>(a, s); }
