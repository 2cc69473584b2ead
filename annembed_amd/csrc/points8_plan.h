// points8_plan.h -- which form of a kernel a size takes, and how many workgroups: the rules of the 8-bit store's calls, on the host and without HIP.
#pragma once
#include <algorithm>
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

// ---- the product

// 256 x 256 tiles read every operand least often but leave one workgroup on a CU: taken where a tile has 8 blocks or more, whole rounds of tiles fill the chip to 7 / 8 and
// edges waste little.  To bf16, against 128 x 128: 8192 x 16 384 x 4096 779 and 915 us, 4096 x 8192 x 4096 203 and 233, 4096 x 4096 x 4096 99 and 117, 8192 x 8192 x 1024 121 and
// 134, 3840 x 4096 x 2048, 240 tiles, 53 and 60 (to f32 62 and 64); but 8192 x 8192 x 512 77 and 81 (to f32 107 and 100), 8192 x 16 384 x 128 87 and 72, 6144 x 6144 x
// 4096, 576 tiles, 282 and 259, 300 x 60 000 x 784, two rows of tiles for 300, 56 and 44.  (Few blocks and very many tiles can go either way: 8192 x 30 000 x 64 159 and 178, 16 384 x
// 16 384 x 128 154 and 138.)
// Workgroups of 64 x 64 that split the coordinates, while each has a CU of its own, or nearly (170 x 258 x 1986 to bf16 9.4 against 19.4 us with 128 x 128 tiles; 1000 x
// 1000 x 1000, 256 of them, 7.6 against 11.8; 128 x 12 000 x 784, 376, 11.4 against 11.8 and to f32 12.4 against 13.2; 512 x 4096 x 512, 512, 9.0 against 8.3
// and 10.9 against 9.7).
struct ProductPlan {
    int tile;   // 64, 128 or 256 rows and points a workgroup
    uint64_t tiles_m, tiles_n;
};
inline ProductPlan product_plan(uint64_t m, uint64_t n, uint64_t dim) {
    auto tiles = [&](int tile) { return ProductPlan{tile, (m + tile - 1) / tile, (n + tile - 1) / tile}; };
    const ProductPlan small = tiles(64), large = tiles(256);
    if (small.tiles_m * small.tiles_n <= 384) return small;
    const uint64_t count = large.tiles_m * large.tiles_n, rounds = (count + 255) / 256;
    if (points8_blocks(dim) >= 8 && count * 8 >= rounds * 256 * 7 && large.tiles_m * 256 * 4 <= m * 5 && large.tiles_n * 256 * 4 <= n * 5) return large;
    return tiles(128);
}

// Few rows: every workgroup quantises them itself, as the bf16 values they stand for in LDS.
constexpr int kFew = 64;
inline uint64_t few_lds_row(uint64_t dim) { return ((dim + kBlock - 1) / kBlock * kBlock) * 2 + 16; }   // (16 bytes more: neighbours start 4 banks apart)
// 16 points a wave leave half of the chip's waves without work below 32 768 points: four waves share them then
inline uint64_t few_points(uint64_t n, uint64_t dim) { return n >= 32768 || points8_blocks(dim) < 4 ? 64 : 16; }
// One launch while the quantising that every workgroup does for itself, and the exact products, cost less than a launch does (one row against 5000 x 4000
// 7.0 against 15.7 us, 16 against 3000 x 1400 9.1 against 10.3, but against 30 000 x 1400 33 against 18; 17 against 2000 x 300 6.1 against 8.2, 32
// against 30 000 x 128 7.0 against 8.5, against 20 000 x 300 9.4 against 8.3; 48 against 20 000 x 28 9.1 against 8.2).
inline bool few_rows(uint64_t m, uint64_t n, uint64_t dim) {
    if (m > kFew || m * few_lds_row(dim) > 48 * 1024 || n >= 1ull << 30) return false;   // (64 points, 256 threads: fewer than 2^32)
    const uint64_t tiles = m <= 16 ? 1 : m <= 32 ? 2 : 4, quantised = (n + few_points(n, dim) - 1) / few_points(n, dim) * m * dim;
    return m <= 16 ? quantised <= 10000000 : tiles * 16 * n <= 1 << 20 && m * dim <= 10000 && quantised <= 2000000;
}

// ---- the gradient of the product

constexpr int kStep = 64;    // points per step: 128 bytes of bf16

struct GradPlan {
    uint32_t fr;   // 64 rows of dc a tile, or 128
    uint64_t tiles_m, tiles_k, slices, per_slice, ldp, bytes;
};
inline GradPlan grad_plan(uint64_t m, uint64_t n, uint64_t dim, uint32_t dctype) {
    GradPlan best{};
    const uint64_t steps = std::max<uint64_t>((n + kStep - 1) / kStep, 1), tiles_k = (dim + kBlock - 1) / kBlock, ldp = (dim + 3) / 4 * 4;
    const uint64_t most = 0x3FFF0000ull / points8_row_bytes(dim) / kStep, least_slices = (steps + most - 1) / most;   // a slice's codes: less than 1 GiB
    // What a choice costs, in us: a workgroup's beginning and end; its steps, with so many workgroups on a CU (measured at 300 x 60 000 x 784, between operands
    // in cache and operands from memory; more workgroups do not fit or do not pay); the slices' sums, written and read again at 5 TB/s; the launch that
    // joins them.  bf16, from memory: 300 x 60 000 x 784 56 us with 128 rows and two workgroups on a CU, 58 to 65 otherwise; 64 rows of it 22.4 with 64
    // and one, 24 to 27 otherwise; 1000 x 1000 x 1000 in one slice 12.6 against 16 to 21 in several.
    struct Choice { uint32_t fr, wgs; float step; };
    static constexpr Choice bf16[] = {{1, 1, 0.43f}, {1, 2, 0.66f}, {2, 1, 0.55f}, {2, 2, 0.86f}};
    static constexpr Choice f16[] = {{1, 1, 0.84f}, {1, 2, 1.1f}, {2, 1, 1.25f}, {2, 2, 1.76f}};
    static constexpr Choice f32[] = {{1, 1, 1.07f}, {1, 2, 1.46f}};
    const Choice* const choices = dctype == AE_TYPE_BF16 ? bf16 : dctype == AE_TYPE_F16 ? f16 : f32;
    const int count = dctype == AE_TYPE_F32 ? 2 : 4;
    double least = 0.;
    for (int q = 0; q < count; q++) {
        const Choice& c = choices[q];
        const uint64_t tiles_m = (m + 64 * c.fr - 1) / (64 * c.fr), tiles = tiles_m * tiles_k, slots = 256 * c.wgs;
        for (const uint64_t want : {(uint64_t)1, slots / tiles}) {
            const uint64_t slices = std::max<uint64_t>({1, least_slices, std::min(want, (steps + 3) / 4)}), per = (steps + slices - 1) / slices, used = (steps + per - 1) / per;
            const double rounds = (double)((tiles * used + slots - 1) / slots);
            const double cost = rounds * ((c.fr == 1 ? 2 : 5) + per * c.step) + (used > 1 ? 4. + used * (0.005 + m * ldp * 8 / 5.1e6) : 0.);
            if (best.fr && cost >= least) continue;
            least = cost;
            best = GradPlan{c.fr, tiles_m, tiles_k, used, per * kStep, ldp, used > 1 ? used * m * ldp * 4 : 0};
        }
    }
    return best;
}

// groups of threads that share a run of the slices' sums when they are joined
inline unsigned join_groups(uint64_t slices) { return slices >= 192 ? 64 : slices >= 48 ? 16 : slices >= 8 ? 4 : 1; }

// bytes of dc from a tile's first value to its last one in a slice of the points, and not one more: what a 16-byte piece has behind them is not fetched
constexpr uint32_t grad_range(uint32_t rows, uint32_t row_bytes, uint32_t points, uint32_t size) { return (rows - 1) * row_bytes + points * size; }

}  // namespace ae
