// The attention kernels of rt_attention_tile.h and rt_attention_weights.h for f32
#include "rt_attention_weights.h"

int rt_attention_tile_f32(rt_device* dev, AttnArgs& a, bool paged, bool* done) { return at_dispatch_tile<float, false>(dev, a, paged, done); }
int rt_attention_weights_f32(rt_device* dev, const AttnArgs& a, const float* weights, float* out) { return aw_dispatch<float>(dev, a, weights, out); }
