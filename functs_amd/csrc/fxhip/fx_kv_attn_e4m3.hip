// Attention over e4m3 caches.
#include "fx_kv_attn.h"

fxkv::Kernels fx_kv_kernels_e4m3(int type, int depth, bool wide) { return fxkv::kernels_of<0>(type, depth, wide); }
