// points8.hip -- the store of points in 8 bits: rows quantised as they are written, read back as the values they stand for.
//
// Both directions move n dim (1 + size of x) bytes and compute next to nothing: they are bound by HBM, the smallest calls by the launch.
// A group of 16 lanes owns a block of 128 coordinates (8 a lane: 16 or 32 bytes of x, 8 bytes of codes, whatever the type), so the block's
// largest magnitude is four DPP rotations within a row of the wave, no LDS and no barrier; a wave covers 4 blocks = 1 or 2 KB of
// consecutive x.  Blocks are numbered through the whole call (block u = row u / blocks), so rows of any length fill the waves alike.
#include "points8.h"

using namespace ae;

namespace {

struct Blocks {   // the call's blocks
    uint64_t units, n;
    uint32_t nb;
};
// row and block of unit `u0 + t`; u0 is the workgroup's first unit
struct Cursor {
    uint64_t row0;
    uint32_t rem0;
    __device__ Cursor(uint64_t u0, uint32_t nb) {
        if (u0 >> 32) { row0 = u0 / nb; rem0 = (uint32_t)(u0 - row0 * nb); }
        else { row0 = (uint32_t)u0 / nb; rem0 = (uint32_t)u0 - (uint32_t)row0 * nb; }
    }
    __device__ __forceinline__ void at(uint32_t t, uint32_t nb, uint64_t& row, uint32_t& b) const {
        const uint32_t x = rem0 + t, q = x / nb;
        row = row0 + q;
        b = x - q * nb;
    }
};

// the later of two rows with the same slot is the one that is held: every row of the call claims its slot, the largest row wins
__global__ void __launch_bounds__(256) points8_claim_kernel(const uint32_t* __restrict__ slots, uint32_t n, uint64_t capacity, uint32_t* __restrict__ owner) {
    const uint32_t i = blockIdx.x * 256u + threadIdx.x;
    if (i >= n) return;
    const uint32_t s = slots[i];
    if (s < capacity) atomicMax(&owner[s], i + 1);
}
__global__ void __launch_bounds__(256) points8_release_kernel(const uint32_t* __restrict__ slots, uint32_t n, uint64_t capacity, uint32_t* __restrict__ owner) {
    const uint32_t i = blockIdx.x * 256u + threadIdx.x;
    if (i >= n) return;
    const uint32_t s = slots[i];
    if (s < capacity) owner[s] = 0;
}

// SLOTS 0: row i to first + i.  1: to slots[i], unless a later row has the same slot.  2: to slots[i] where owner says so.  3: the same
// for rows of one block, which give their slot back themselves (another row of that slot finds the owner or nobody: not itself).
template <int TYPE, int SLOTS, int TRIPS>
__global__ void __launch_bounds__(256) points8_write_kernel(const typename Elem<TYPE>::T* __restrict__ x, uint64_t ldx, uint64_t dim, Blocks bl, uint64_t first,
                                                            const uint32_t* __restrict__ slots, uint32_t* __restrict__ owner, uint64_t capacity,
                                                            uint8_t* __restrict__ codes, uint64_t row_bytes, uint8_t* __restrict__ scales, uint64_t scale_stride) {
    const uint64_t u0 = blockIdx.x * (uint64_t)(kGroups * TRIPS);
    const Cursor cur(u0, bl.nb);
    const int lane = threadIdx.x & 15, group = threadIdx.x >> 4;
    float v[TRIPS][8];
    uint64_t row[TRIPS];
    uint32_t b[TRIPS];
    bool live[TRIPS];
#pragma unroll
    for (int t = 0; t < TRIPS; t++) {
        const uint32_t off = t * kGroups + group;
        cur.at(off, bl.nb, row[t], b[t]);
        live[t] = u0 + off < bl.units;
        const uint64_t k = b[t] * (uint64_t)kBlock + lane * 8;
        const int count = !live[t] || k >= dim ? 0 : (int)min((uint64_t)8, dim - k);
        load8<TYPE>(x + (count ? row[t] * ldx + k : 0), count, v[t]);
    }
    __shared__ uint8_t later[kGroups * TRIPS];   // rows of this workgroup whose slot comes again
    if constexpr (SLOTS == 1) {   // all slots pass by once, four a thread, and are compared with those of the workgroup's rows
        const uint32_t n = (uint32_t)bl.n, first_row = (uint32_t)cur.row0, rows = min(n - first_row, (cur.rem0 + kGroups * TRIPS - 1) / bl.nb + 1);
        __shared__ __attribute__((aligned(16))) uint32_t mine[kGroups * TRIPS];
        if (threadIdx.x < kGroups * TRIPS) {
            later[threadIdx.x] = 0;
            mine[threadIdx.x] = threadIdx.x < rows ? slots[first_row + threadIdx.x] : 0xFFFFFFFFu;
        }
        __syncthreads();
        for (uint32_t c = (first_row + 1) & ~1023u; c < n; c += 1024) {
            const uint32_t j = c + threadIdx.x * 4;
            uint32_t s[4];
            if (j + 4 <= n) {
                const Piece four = *reinterpret_cast<const Piece*>(slots + j);
#pragma unroll
                for (int e = 0; e < 4; e++) s[e] = four[e];
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++) s[e] = j + e < n ? slots[j + e] : 0xFFFFFFFFu;   // (no row's that is written)
            }
            for (uint32_t r = 0; r < rows; r += 4) {
                const u32x4 to = *reinterpret_cast<const u32x4*>(mine + r);
                uint32_t again = 0;   // bit q: row r + q
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    uint32_t last = 0;
#pragma unroll
                    for (int e = 0; e < 4; e++) last = s[e] == to[q] ? j + e : last;
                    again |= last > first_row + r + q ? 1u << q : 0u;
                }
                if (again) {   // (rarely)
#pragma unroll
                    for (int q = 0; q < 4; q++)
                        if (again >> q & 1) later[r + q] = 1;
                }
            }
        }
        __syncthreads();
    }
#pragma unroll
    for (int t = 0; t < TRIPS; t++) {
        const uint32_t byte = scale_byte(max16(amax8(v[t])));
        uint64_t to = first + row[t];
        if constexpr (SLOTS != 0) {
            if (live[t]) {
                const uint32_t s = slots[row[t]];
                to = s;
                live[t] = s < capacity;
                if constexpr (SLOTS >= 2) live[t] = live[t] && owner[s] == (uint32_t)row[t] + 1;
                if constexpr (SLOTS == 3) { if (live[t] && lane == 0) owner[s] = 0; }
            }
            if constexpr (SLOTS == 1) live[t] = live[t] && !later[row[t] - cur.row0];
        }
        const uint64_t k = b[t] * (uint64_t)kBlock + lane * 8;
        if (live[t] && k < row_bytes) *reinterpret_cast<uint2*>(codes + to * row_bytes + k) = encode8(v[t], byte);
        if (live[t] && lane == 0) scales[b[t] * scale_stride + to] = (uint8_t)byte;
    }
}

template <int TYPE, bool SLOTS, int TRIPS>
__global__ void __launch_bounds__(256) points8_read_kernel(const uint8_t* __restrict__ codes, uint64_t row_bytes, const uint8_t* __restrict__ scales, uint64_t scale_stride,
                                                           uint64_t capacity, uint64_t first, const uint32_t* __restrict__ slots, Blocks bl,
                                                           typename Elem<TYPE>::T* __restrict__ x, uint64_t ldx, uint64_t dim) {
    const uint64_t u0 = blockIdx.x * (uint64_t)(kGroups * TRIPS);
    const Cursor cur(u0, bl.nb);
    const int lane = threadIdx.x & 15, group = threadIdx.x >> 4;
    uint2 c[TRIPS];
    uint32_t byte[TRIPS];
    uint64_t row[TRIPS];
    uint32_t b[TRIPS];
    int count[TRIPS];
    bool bad[TRIPS];
#pragma unroll
    for (int t = 0; t < TRIPS; t++) {
        const uint32_t off = t * kGroups + group;
        cur.at(off, bl.nb, row[t], b[t]);
        const uint64_t k = b[t] * (uint64_t)kBlock + lane * 8;
        count[t] = u0 + off >= bl.units || k >= dim ? 0 : (int)min((uint64_t)8, dim - k);
        c[t] = make_uint2(0, 0);
        byte[t] = 0;
        bad[t] = false;
        if (count[t]) {
            uint64_t from = first + row[t];
            if constexpr (SLOTS) {
                from = slots[row[t]];
                bad[t] = from >= capacity && from != 0xFFFFFFFFull;
            }
            if (from < capacity) {
                c[t] = *reinterpret_cast<const uint2*>(codes + from * row_bytes + k);
                byte[t] = scales[b[t] * scale_stride + from];
            }
        }
    }
#pragma unroll
    for (int t = 0; t < TRIPS; t++) {
        float v[8];
        decode8(c[t], byte[t], v);
        if (SLOTS && bad[t]) {
#pragma unroll
            for (int q = 0; q < 8; q++) v[q] = __uint_as_float(0x7FC00000u);
        }
        const uint64_t k = b[t] * (uint64_t)kBlock + lane * 8;
        if (count[t]) store8<TYPE>(x + row[t] * ldx + k, count[t], v);
    }
}

Blocks blocks_of(uint64_t n, uint64_t dim) {
    Blocks bl;
    bl.n = n;
    bl.nb = points8_blocks(dim);
    bl.units = n * bl.nb;
    return bl;
}
BlocksPlan plan_of(uint64_t n, uint64_t dim, uint32_t type, bool look) {
    const BlocksPlan p = blocks_plan(n, dim, type, look);
    if (!p.grid) fail(AE_ERR_INVALID_ARG, "%llu rows of %u blocks are more than one call takes", (unsigned long long)n, points8_blocks(dim));
    return p;
}

template <int SLOTS>
void launch_write(const void* d_x, uint32_t type, uint64_t n, uint64_t ldx, uint64_t dim, uint64_t first, const uint32_t* slots, uint32_t* owner, uint64_t capacity,
                  uint8_t* codes, uint8_t* scales, uint64_t scale_stride, hipStream_t s) {
    const Blocks bl = blocks_of(n, dim);
    const BlocksPlan plan = plan_of(n, dim, type, SLOTS == 1);
    by_type(type, [&](auto ty) {
        constexpr int TYPE = decltype(ty)::value;
        const auto* x = static_cast<const typename Elem<TYPE>::T*>(d_x);
        auto go = [&](auto kernel) {
            hipLaunchKernelGGL(kernel, dim3(plan.grid), dim3(256), 0, s, x, ldx, dim, bl, first, slots, owner, capacity, codes, points8_row_bytes(dim), scales, scale_stride);
        };
        if (plan.trips == 1) go(points8_write_kernel<TYPE, SLOTS, 1>);
        else go(points8_write_kernel<TYPE, SLOTS, kTrips>);
    });
    check_launch("points8_write");
}

void read_rows(const ae_points8* p, uint64_t first, const uint32_t* slots, uint64_t n, void* d_x, uint32_t type, uint64_t ldx, hipStream_t s) {
    const Blocks bl = blocks_of(n, p->dim);
    const BlocksPlan plan = plan_of(n, p->dim, type, false);
    by_type(type, [&](auto ty) {
        constexpr int TYPE = decltype(ty)::value;
        auto* x = static_cast<typename Elem<TYPE>::T*>(d_x);
        auto go = [&](auto kernel) {
            hipLaunchKernelGGL(kernel, dim3(plan.grid), dim3(256), 0, s, (const uint8_t*)p->codes.p, p->row_bytes, (const uint8_t*)p->scales.p, p->scale_stride, p->capacity, first,
                               slots, bl, x, ldx, p->dim);
        };
        const bool one = plan.trips == 1;
        if (slots) one ? go(points8_read_kernel<TYPE, true, 1>) : go(points8_read_kernel<TYPE, true, kTrips>);
        else one ? go(points8_read_kernel<TYPE, false, 1>) : go(points8_read_kernel<TYPE, false, kTrips>);
    });
    check_launch("points8_read");
}

}  // namespace

namespace ae {

void check_points8(const ae_points8* p, uint64_t first, uint64_t n, const char* what) {
    if (!p) fail(AE_ERR_INVALID_ARG, "%s: the store is NULL", what);
    int dev = 0;
    AE_HIP(hipGetDevice(&dev));
    if (dev != p->device) fail(AE_ERR_INVALID_ARG, "%s: the store lives on device %d, the current device is %d", what, p->device, dev);
    if (first > p->capacity || n > p->capacity - first)
        fail(AE_ERR_INVALID_ARG, "%s: rows %llu ... + %llu are outside a store of %llu", what, (unsigned long long)first, (unsigned long long)n, (unsigned long long)p->capacity);
}

void points8_quantise(const void* d_x, uint32_t type, uint64_t n, uint64_t ldx, uint64_t dim, uint8_t* codes, uint8_t* scales, uint64_t scale_stride, hipStream_t s) {
    launch_write<0>(d_x, type, n, ldx, dim, 0, nullptr, nullptr, n, codes, scales, scale_stride, s);
}

}  // namespace ae

extern "C" {

int32_t ae_points8_create(uint64_t capacity, uint64_t dim, ae_points8** out) {
    return guard([&] {
        require_device();
        if (!out) fail(AE_ERR_INVALID_ARG, "ae_points8_create: out is NULL");
        if (capacity == 0 || capacity >= 0xFFFFFFFFull) fail(AE_ERR_INVALID_ARG, "ae_points8_create: a capacity of %llu rows is out of range", (unsigned long long)capacity);
        if (dim == 0 || dim > (1u << 20)) fail(AE_ERR_INVALID_ARG, "ae_points8_create: dim %llu is not in [1, 2^20]", (unsigned long long)dim);
        std::unique_ptr<ae_points8> p(new ae_points8);
        p->capacity = capacity;
        p->dim = dim;
        p->row_bytes = points8_row_bytes(dim);
        p->blocks = points8_blocks(dim);
        p->scale_stride = points8_scale_stride(capacity);
        AE_HIP(hipGetDevice(&p->device));
        p->codes.alloc(capacity * p->row_bytes);
        p->scales.alloc(p->blocks * p->scale_stride + kScaleSlack);
        p->owner.alloc(capacity);
        p->codes.zero();
        p->scales.zero();
        p->owner.zero();
        sync();
        *out = p.release();
    });
}
int32_t ae_points8_destroy(ae_points8* p) {
    return guard([&] { delete p; });
}
int32_t ae_points8_info(const ae_points8* p, uint64_t* capacity, uint64_t* dim, uint64_t* row_bytes, uint64_t* scale_stride) {
    return guard([&] {
        if (!p) fail(AE_ERR_INVALID_ARG, "ae_points8_info: the store is NULL");
        if (capacity) *capacity = p->capacity;
        if (dim) *dim = p->dim;
        if (row_bytes) *row_bytes = p->row_bytes;
        if (scale_stride) *scale_stride = p->scale_stride;
    });
}
int32_t ae_points8_device(const ae_points8* p, void** d_codes, void** d_scales) {
    return guard([&] {
        if (!p || !d_codes || !d_scales) fail(AE_ERR_INVALID_ARG, "ae_points8_device: null argument");
        *d_codes = p->codes.p;
        *d_scales = p->scales.p;
    });
}

int32_t ae_points8_write(ae_points8* p, const void* d_x, uint32_t type, uint64_t n, uint64_t ldx, uint64_t first, const uint32_t* d_slots, void* stream) {
    return guard([&] {
        require_device();
        check_points8(p, d_slots ? 0 : first, d_slots ? 0 : n, "ae_points8_write");
        check_type(type, "ae_points8_write");
        if (n == 0) return;
        check_rows(d_x, type, n, p->dim, ldx, "ae_points8_write: x");
        hipStream_t s = (hipStream_t)stream;
        if (!d_slots) {
            launch_write<0>(d_x, type, n, ldx, p->dim, first, nullptr, nullptr, p->capacity, p->codes.p, p->scales.p, p->scale_stride, s);
            return;
        }
        check_aligned(d_slots, 4, "ae_points8_write: slots");
        if (n > 0x7FFFFFFFull) fail(AE_ERR_INVALID_ARG, "ae_points8_write: %llu slots are more than one call takes", (unsigned long long)n);
        // The last row of a repeated slot is held.  Few rows: every workgroup looks at the slots behind its own, one launch.  More: the rows claim
        // their slots first and give them back as they are written, or, rows of several blocks, in a launch of their own.
        if (write_looks(n, p->dim)) {
            launch_write<1>(d_x, type, n, ldx, p->dim, 0, d_slots, nullptr, p->capacity, p->codes.p, p->scales.p, p->scale_stride, s);
            return;
        }
        plan_of(n, p->dim, type, false);   // (a call that is refused claims nothing: what stays claimed would keep later rows out)
        const unsigned grid = blocks_for(n, 256);
        hipLaunchKernelGGL(points8_claim_kernel, dim3(grid), dim3(256), 0, s, d_slots, (uint32_t)n, p->capacity, p->owner.p);
        check_launch("points8_claim");
        auto release = [&] { hipLaunchKernelGGL(points8_release_kernel, dim3(grid), dim3(256), 0, s, d_slots, (uint32_t)n, p->capacity, p->owner.p); };
        try {
            if (p->blocks == 1) launch_write<3>(d_x, type, n, ldx, p->dim, 0, d_slots, p->owner.p, p->capacity, p->codes.p, p->scales.p, p->scale_stride, s);
            else launch_write<2>(d_x, type, n, ldx, p->dim, 0, d_slots, p->owner.p, p->capacity, p->codes.p, p->scales.p, p->scale_stride, s);
        } catch (...) {
            release();
            throw;
        }
        if (p->blocks == 1) return;
        release();
        check_launch("points8_release");
    });
}

int32_t ae_points8_read(const ae_points8* p, uint64_t first, const uint32_t* d_slots, uint64_t n, void* d_x, uint32_t type, uint64_t ldx, void* stream) {
    return guard([&] {
        require_device();
        check_points8(p, d_slots ? 0 : first, d_slots ? 0 : n, "ae_points8_read");
        check_type(type, "ae_points8_read");
        if (n == 0) return;
        check_rows(d_x, type, n, p->dim, ldx, "ae_points8_read: x");
        if (d_slots) check_aligned(d_slots, 4, "ae_points8_read: slots");
        read_rows(p, first, d_slots, n, d_x, type, ldx, (hipStream_t)stream);
    });
}

int32_t ae_kgraph_bruteforce_l2_points8(const ae_points8* p, uint64_t first, uint64_t n, uint32_t nbng, void* stream, ae_kgraph** out) {
    return guard([&] {
        require_device();
        check_points8(p, first, n, "ae_kgraph_bruteforce_l2_points8");
        if (!out || n < 2 || nbng == 0 || nbng >= n) fail(AE_ERR_INVALID_ARG, "ae_kgraph_bruteforce_l2_points8: bad arguments");
        DevBuf<float> dx;
        dx.alloc(n * p->dim);
        AE_HIP(hipStreamSynchronize((hipStream_t)stream));
        read_rows(p, first, nullptr, n, dx.p, AE_TYPE_F32, p->dim, ae::stream());
        *out = kgraph_bruteforce_device(dx.p, n, p->dim, nbng);
    });
}

}  // extern "C"
