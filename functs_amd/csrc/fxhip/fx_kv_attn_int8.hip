// Attention over int8 caches.
#include "fx_kv_attn.h"

const void* fx_kv_rows_kernel_int8(int type, int depth) { return fxkv::rows_kernel<1>(type, depth); }
