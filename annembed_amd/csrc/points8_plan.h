// points8_plan.h -- which form of a kernel a size takes, and how many workgroups: the rules of the 8-bit store's calls, on the host and without HIP.
#pragma once
#include <cstdint>

#include "../../include/annembed_hip.h"

namespace ae {

constexpr int kBlock = 128;   // coordinates that share a scale

inline uint64_t points8_row_bytes(uint64_t dim) { return (dim + 15) / 16 * 16; }
inline uint32_t points8_blocks(uint64_t dim) { return (uint32_t)((dim + kBlock - 1) / kBlock); }

// ---- writes and reads: a group of 16 lanes a block

constexpr int kGroups = 16;    // blocks per workgroup and trip
constexpr int kTrips = 4;      // blocks a group has in flight: 64 to 128 bytes of loads per lane
// Up to this many slots a workgroup looks for later occurrences of its rows' slots itself, in one launch, rows of one block up to 4096: 4096 rows of 128 take 6.9
// us against 7.1 of the two launches otherwise, 8191 of 128 10.1 against 7.1; 5000 of 784 7.3 against 11.1 of three, 8000 of 1500 18.4 against 16.0.
constexpr uint32_t kScan = 6000;
inline bool write_looks(uint64_t n, uint64_t dim) { return n <= (points8_blocks(dim) == 1 ? 4096 : kScan); }

// Whether a group of lanes takes one block instead of kTrips: fewer loads in flight, more waves.  f32 (32 bytes of loads a lane and block) always, 16 bits up
// to a million blocks (write 60 000 x 784 of bf16 26 against 30 us, 262 144 x 1024 145 against 148, but read 200 000 x 784 by ids 139 against 116; f32 read
// 200 000 x 784 137 against 200, write 8191 x 128 scattered 6.8 against 8.1).  Workgroups that look at all slots of the call: while they are few (4096
// rows of 128 6.9 against 20 us, 4096 rows of 4096 18.5 against 16.2).
inline bool spread(uint64_t units, uint32_t type, bool look) { return units <= (look ? 65536 : type == AE_TYPE_F32 ? 1 << 27 : 1 << 20); }

struct BlocksPlan {
    int trips;       // blocks a group of lanes takes
    unsigned grid;   // workgroups; 0: 2^32 threads or more, which no launch has
};
inline BlocksPlan blocks_plan(uint64_t n, uint64_t dim, uint32_t type, bool look) {
    const uint64_t units = n * points8_blocks(dim);
    BlocksPlan p;
    p.trips = spread(units, type, look) ? 1 : kTrips;
    const uint64_t grid = (units + kGroups * p.trips - 1) / (kGroups * p.trips);
    p.grid = grid * 256 > 0xFFFFFFFFull ? 0 : (unsigned)grid;
    return p;
}

// ---- the gradient of the product

// bytes of dc from a tile's first value to its last one in a slice of the points, and not one more: what a 16-byte piece has behind them is not fetched
constexpr uint32_t grad_range(uint32_t rows, uint32_t row_bytes, uint32_t points, uint32_t size) { return (rows - 1) * row_bytes + points * size; }

}  // namespace ae
