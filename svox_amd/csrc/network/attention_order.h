// attention_order.h -- the launch that puts the tiles of an attention in order.
#pragma once
#include "attention_tile.h"

namespace svox_network {

struct OrderArgs {
    Sequences seq;
    struct Axis {
        int* to;      // tiles
        int tiles, count, rows, group;
        int keys;     // the tiles are of queries' rows, what they see are keys
    } axis[2];
};
void launch_order(const OrderArgs& p, int axes, hipStream_t stream);

}  // namespace svox_network
