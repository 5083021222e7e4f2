// The attention kernels of rt_attention_tile.h for bf16
#include "rt_attention_tile.h"

int rt_attention_tile_bf16(rt_device* dev, AttnArgs& a, bool paged, bool* done) { return at_dispatch_tile<bf16_t>(dev, a, paged, done); }
