#include "span_attn.h"
size_t k_span_attn_bwd_workspace_bytes(const mm_span_attn*) { return 0; }
int k_span_attn_bwd(hipStream_t, const mm_span_attn*, void*) { return mm_set_error(MM_ERR_UNSUPPORTED, "span attention: no backward yet"); }
