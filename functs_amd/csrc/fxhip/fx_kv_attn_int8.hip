// Attention over int8 caches.
#include "fx_kv_attn.h"

fxkv::Kernels fx_kv_kernels_int8(int type, int depth, bool wide) { return fxkv::kernels_of<1>(type, depth, wide); }
