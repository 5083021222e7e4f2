// The attention kernels of rt_attention_tile.h and rt_attention_few.h for bf16, for calls that change or mask their scores
#include "rt_attention_few.h"

int rt_attention_scored_bf16(rt_device* dev, AttnArgs& a, bool paged, bool* done) { return at_dispatch_tile<bf16_t, true>(dev, a, paged, done); }
