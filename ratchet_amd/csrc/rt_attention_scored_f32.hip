// The attention kernels of rt_attention_tile.h and rt_attention_few.h for f32, for calls that change or mask their scores
#include "rt_attention_few.h"

int rt_attention_scored_f32(rt_device* dev, AttnArgs& a, bool paged, bool* done) { return at_dispatch_tile<float, true>(dev, a, paged, done); }
