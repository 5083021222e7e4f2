// The attention kernels of rt_attention_tile.h and rt_attention_weights.h for bf16
#include "rt_attention_weights.h"

int rt_attention_tile_bf16(rt_device* dev, AttnArgs& a, bool paged, bool* done) { return at_dispatch_tile<bf16_t>(dev, a, paged, done); }
int rt_attention_weights_bf16(rt_device* dev, const AttnArgs& a, const float* weights, float* out) { return aw_dispatch<bf16_t>(dev, a, weights, out); }
