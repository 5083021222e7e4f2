// The attention kernels of rt_attention_tile.h for f32
#include "rt_attention_tile.h"

int rt_attention_tile_f32(rt_device* dev, AttnArgs& a, bool paged, bool* done) { return at_dispatch_tile<float>(dev, a, paged, done); }
