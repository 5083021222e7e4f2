// Prints at_round(tiles, per, cus, held) of the numbers it is given
#include <cstdio>
#include <cstdlib>

#include "rt_attention_order.h"

int main(int argc, char** argv) {
    if (argc != 5) return 1;
    std::printf("%u\n", at_round(std::strtoull(argv[1], nullptr, 10), std::strtoull(argv[2], nullptr, 10), std::strtoull(argv[3], nullptr, 10), std::strtoull(argv[4], nullptr, 10)));
    return 0;
}
