// The order in which a launch of attention starts its row tiles.  Host code only.
#ifndef RT_ATTENTION_ORDER_H
#define RT_ATTENTION_ORDER_H

#include <cstdint>

// Row tiles (of each of `per` sequences and KV heads) to a round of a causal call whose `tiles` row tiles are walked whole, every other round backwards; 0: the longest first.
// held: blocks that a CU's registers and LDS hold.  Where they are two or three, turned rounds pair a long walk with a short one in a launch of up to three blocks to a CU,
// also where it holds two: us turned | longest first, 32 heads, f32: 96 columns, 2176 tokens 270 | 326, 2304 302 | 350, 2560 368 | 397, 2944 467 | 468; 80 columns 251 | 303,
// 282 | 325, 343 | 369, 434 | 434; 128 columns 347 | 423, 391 | 454, 478 | 516, 610 | 609; bf16, 128 columns, 61 | 61, 64 | 64, 73 | 73, 87 | 87.
// Where a CU holds one, the next block is the longest that is left: 256 columns, f16, 2048 tokens 154 | 126.
static inline uint32_t at_round(uint64_t tiles, uint64_t per, uint64_t cus, uint64_t held) {
    return held > 1 && tiles > cus && tiles <= 3 * cus ? (uint32_t)(cus / per) : 0;
}

#endif
