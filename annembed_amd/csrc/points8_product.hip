// points8_product.hip -- rows times the points held in 8 bits: c[i][j] = <x_i, p_j>, exact products with f32 sums.
//
// Codes travel as 8 bits through memory and LDS and are widened, with their block's power of two, in the registers they are multiplied from: every
// value held is exact in bf16, so are the products, and the bf16 matrix cores add them in f32.  The scaled 8-bit cores would do the products at twice
// the rate, but they add eight of them at a time and cut 13 bits below the largest of the eight (measured on this chip: 2^12 + 2^-1 is kept,
// 2^12 + 2^-2 is 2^12): where two large products cancel, the small ones beside them are lost.  Sums are held in 32 bits here, whatever the result's
// type and however many rows there are.
#include "points8.h"

using namespace ae;

namespace {

// the scale byte of row i of the FM (FN) that a lane holds, four of them in a dword
__device__ __forceinline__ uint32_t byte_of(const uint32_t* dwords, int i) { return (dwords[i >> 2] >> ((i & 3) * 8)) & 255u; }

// lanes 32 ... 63 of a and lanes 0 ... 31 of b change places
__device__ __forceinline__ void swap32(u32x4& a, u32x4& b) {
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const auto r = __builtin_amdgcn_permlane32_swap(a[e], b[e], false, false);
        a[e] = r[0];
        b[e] = r[1];
    }
}
// the odd groups of 16 lanes of a and the even ones of b
__device__ __forceinline__ void swap16(u32x4& a, u32x4& b) {
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const auto r = __builtin_amdgcn_permlane16_swap(a[e], b[e], false, false);
        a[e] = r[0];
        b[e] = r[1];
    }
}

struct ProductArgs {
    Rows8 x, p;       // m rows, n rows
    uint32_t blocks;
    void* c;
    uint64_t ldc;
    uint32_t tiles_m, tiles_n;
    uint32_t near;    // a tile's rows of c span less than 2 GiB
};

// The tiles of a workgroup.  Workgroups go to the 8 XCDs in turn, each with an L2 of its own: an XCD owns a run of the tiles, kPanel rows of
// tiles at a time, and its workgroups walk it side by side, so that the points one of them fetched serve the panel's other rows.
constexpr uint32_t kPanel = 4;
struct Walk {
    uint32_t first, count, at, step, tiles_m, tiles_n;
    __device__ Walk(uint32_t m, uint32_t n) : tiles_m(m), tiles_n(n) {
        const uint32_t total = m * n, each = total / 8, more = total % 8, xcd = blockIdx.x % 8;
        first = xcd * each + min(xcd, more);
        count = each + (xcd < more ? 1 : 0);
        at = blockIdx.x / 8;
        step = gridDim.x / 8;
    }
    __device__ __forceinline__ bool here() const { return at < count; }
    __device__ __forceinline__ void tile(uint32_t& tm, uint32_t& tn) const {
        const uint32_t id = first + at, panel = id / (kPanel * tiles_n), in = id - panel * kPanel * tiles_n;
        const uint32_t rows = max(1u, min(kPanel, tiles_m - panel * kPanel));   // (past the last tile there is no panel: nobody uses what comes out, but 0 does not divide)
        tn = in / rows;
        tm = panel * kPanel + in - tn * rows;
    }
};

// BM x BN tiles of c, waves of WM x 64, a block of 128 coordinates per step, two stages of LDS in turn.
//
// Rows: fragment i of a wave's WM rows is rows i, i + FM, i + 2 FM ... of them (FM = WM / 16): the FM rows of a lane are neighbours, their
// scale bytes one or two dwords.  The same for the points, so a lane ends up with 16 consecutive
// columns of each of its rows and writes them itself.
// LDS: fragment by fragment, a row's 128 codes as 8 chunks of 16 bytes, chunk c of LDS row r at place c ^ ((r >> 1) & 7).  The lanes of group g read
// chunks g and g + 4: the 16 lanes that LDS serves at a time (0-3, 12-15 and 20-27 of a half wave, then the others) touch all 64 banks once.  (With chunks
// 2 g and 2 g + 1 two of them meet in every bank.)  The copies to LDS write lane after lane, so the lanes permute what they fetch.
// Rows beyond the operands and bytes beyond a row lie outside the buffers' range and read as 0.
//
// The blocks of all tiles of a workgroup form one stream: the copy runs two blocks ahead of the products, across the end of a tile, and the
// stores of a tile drain under the next one.  A step's fragment is read two steps ahead.  Two steps before its end a block's stage has been read by
// everybody and the next one has to be there: one barrier a block.  The loop's body has no branch (copies beyond the last tile fetch nothing).
// 8192 x 16 384 x 4096 to bf16 779 us in 256 x 256 tiles, 1411 TF, what a large bf16 product of the library reaches (their sums fill the registers: 20 of 256 spill, to
// f32 42); 300 x 60 000 x 784 44 us in 128 x 128, where the matrix cores are busy for 31 % of the time: 28 % of the rows are padding, a tile has 7 blocks.
template <int TYPE, int BM, int BN, int WM>
__global__ void __launch_bounds__((BM / WM) * (BN / 64) * 64, (BM + BN) * kBlock * 2 > 80 * 1024 ? (BM / WM) * (BN / 64) / 4 : (BM / WM) * (BN / 64) / 2)
product_tile_kernel(ProductArgs a) {
    constexpr int WN = 64, WAVES = (BM / WM) * (BN / WN), FM = WM / 16, FN = WN / 16;
    constexpr int STAGE = (BM + BN) * kBlock;
    constexpr int STEPS = 2 * FM;   // a step: FM-th part of the rows, a half of the block
    using T = typename Elem<TYPE>::T;
    constexpr int STORES = FM * (int)sizeof(T);
    extern __shared__ __attribute__((aligned(128))) uint8_t lds[];
    Walk walk(a.tiles_m, a.tiles_n);
    if (!walk.here()) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wi = (wave / (BN / WN)) * WM, wj = (wave % (BN / WN)) * WN;
    const uint32_t stride = (uint32_t)a.x.row_bytes;

    // ---- the copies
    static_assert(WAVES % 2 == 0 && BM / 8 % WAVES == 0 && BN / 8 % WAVES == 0 && FM % 4 == 0 && FN == 4, "");
    const uint32_t chunk = (lane & 7) ^ (((wave & 1) << 2) + (lane >> 4));   // (r >> 1) & 7 of LDS row r = 8 (q WAVES + wave) + (lane >> 3)
    const uint32_t row16 = (wave & 1) * 8 + (lane >> 3);                     // r % 16
    Walk ahead = walk;
    uint32_t ahead_kb = 0, off_k, off_x, off_p;
    __amdgpu_buffer_rsrc_t rx, rp;
    auto aim = [&]() {   // the copies turn to the tile `ahead`; past the last one to nothing
        uint32_t tm = 0, tn = 0;
        ahead.tile(tm, tn);
        const bool on = ahead.here();
        const uint64_t i0 = on ? (uint64_t)tm * BM : 0, j0 = on ? (uint64_t)tn * BN : 0;
        const uint32_t mi = on ? (uint32_t)min((uint64_t)BM, a.x.rows - i0) : 0, nj = on ? (uint32_t)min((uint64_t)BN, a.p.rows - j0) : 0;
        rx = __builtin_amdgcn_make_buffer_rsrc((void*)(a.x.codes + i0 * stride), (short)0, (int)(mi * stride), 0x00027000);
        rp = __builtin_amdgcn_make_buffer_rsrc((void*)(a.p.codes + j0 * stride), (short)0, (int)(nj * stride), 0x00027000);
        off_k = chunk * 16;
        off_x = row16 * FM * stride + off_k;
        off_p = row16 * FN * stride + off_k;
    };
    auto copy = [&](uint32_t stage) {   // the next block of the stream
        const bool in = off_k < stride;
#pragma unroll
        for (int q = 0; q < (BM + BN) / 8 / WAVES; q++) {
            const bool of_x = q < BM / 8 / WAVES;
            const uint32_t r0 = ((of_x ? q : q - BM / 8 / WAVES) * WAVES + wave) * 8;
            const uint32_t first = of_x ? r0 / WM * WM + r0 % WM / 16 : r0 / WN * WN + r0 % WN / 16;
            const uint32_t off = (of_x ? off_x : off_p) + first * stride;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(of_x ? rx : rp, (__attribute__((address_space(3))) void*)(lds + stage * STAGE + (q * WAVES + wave) * 8 * kBlock), 16,
                                                     (int)(in ? off : 0x7FFFFFFFu), 0, 0, 0);
        }
        off_k += kBlock;
        off_x += kBlock;
        off_p += kBlock;
    };
    auto advance = [&]() {
        if (++ahead_kb == a.blocks) {
            ahead_kb = 0;
            ahead.at += ahead.step;
            aim();
        }
    };

    // ---- the tile's scales: one block ahead
    uint32_t tm, tn;
    walk.tile(tm, tn);
    const uint8_t* sx = a.x.scales + (uint64_t)tm * BM + wi;
    const uint8_t* sp = a.p.scales + (uint64_t)tn * BN + wj;
    const uint32_t at_x = (lane & 15) * FM, at_p = (lane & 15) * FN;
    uint32_t nx[FM / 4], np[1], bx[FM / 4], bp[1];
    auto scales = [&]() {
        __builtin_memcpy(nx, sx + at_x, FM);
        __builtin_memcpy(np, sp + at_p, FN);
    };

    // ---- fragments
    f32x4 acc[FM][FN];
    auto clear = [&]() {
#pragma unroll
        for (int i = 0; i < FM; i++)
#pragma unroll
            for (int j = 0; j < FN; j++) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    };
    u32x4 fx[4], fp[FN];        // codes
    bf16x8 wp[FN][2];           // the points' values of half a block
    const int r_x = wi + (lane & 15), r_p = BM + wj + (lane & 15), c0 = lane >> 4;
    uint32_t in_x = r_x * kBlock + ((c0 ^ ((r_x >> 1) & 7)) << 4), in_p = r_p * kBlock + ((c0 ^ ((r_p >> 1) & 7)) << 4);
    auto chunk_at = [&](uint32_t at) { return *reinterpret_cast<const u32x4*>(lds + at); };
    auto read_x = [&](int s) { fx[s & 3] = chunk_at((in_x ^ (s / FM * 64)) + s % FM * 16 * kBlock); };
    auto read_p = [&](int j, int h) { fp[j] = chunk_at((in_p ^ (h * 64)) + j * 16 * kBlock); };
    auto block = [&](uint32_t stage, auto first) {
#pragma unroll
        for (int q = 0; q < FM / 4; q++) bx[q] = nx[q];
        bp[0] = np[0];
        scales();
#pragma unroll
        for (int s = 0; s < STEPS; s++) {
            if (s == STEPS - 2) {
                // this wave's copies are in LDS; at a tile's first block the stores of the last one, issued after them, may go on
                if constexpr (decltype(first)::value) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(STORES) : "memory");
                else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                __builtin_amdgcn_s_waitcnt(0xC07F);   // lgkmcnt(0): this wave's reads of the stage are done
                __builtin_amdgcn_s_barrier();
                asm volatile("" ::: "memory");
                copy(stage);
                const uint32_t other = stage ? 0u - STAGE : STAGE;
                in_x += other;
                in_p += other;
            }
            read_x((s + 2) % STEPS);
            __builtin_amdgcn_sched_barrier(0);
            const int h = s / FM, i = s % FM;
            if (i == 0) {
#pragma unroll
                for (int j = 0; j < FN; j++) {
#pragma unroll
                    for (int e = 0; e < 2; e++) wp[j][e] = widen8(fp[j][2 * e], fp[j][2 * e + 1], byte_of(bp, j));
                    if (h == 0) read_p(j, 1);
                }
            }
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const bf16x8 wx = widen8(fx[s & 3][2 * e], fx[s & 3][2 * e + 1], byte_of(bx, i));
#pragma unroll
                for (int j = 0; j < FN; j++) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wp[j][e], wx, acc[i][j], 0, 0, 0);
            }
            if (s == STEPS - 1) {
#pragma unroll
                for (int j = 0; j < FN; j++) read_p(j, 0);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        // (the sums are taken note of here, or the compiler moves the products past what follows)
#pragma unroll
        for (int i = 0; i < FM; i++)
#pragma unroll
            for (int j = 0; j < FN; j++) asm volatile("" : "+v"(acc[i][j]));
    };

    aim();
    copy(0);
    advance();
    copy(1);
    advance();
    scales();
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
#pragma unroll
    for (int j = 0; j < FN; j++) read_p(j, 0);
    read_x(0);
    read_x(1);
    uint32_t stage = 0;
    for (;;) {
        const uint64_t i0 = (uint64_t)tm * BM, j0 = (uint64_t)tn * BN;
        clear();
        walk.at += walk.step;
        const bool more = walk.here();
        if (more) walk.tile(tm, tn);
        auto scales_turn = [&](uint32_t kb) {   // the scales' pointers go to the block after kb
            sx += a.x.scale_stride;
            sp += a.p.scale_stride;
            if (kb + 1 == a.blocks) {   // (the last tile's last block takes scales nobody uses)
                sx = a.x.scales + (uint64_t)tm * BM + wi;
                sp = a.p.scales + (uint64_t)tn * BN + wj;
            }
        };
        scales_turn(0);
        block(stage, std::true_type{});
        stage ^= 1;
        advance();
        for (uint32_t kb = 1; kb < a.blocks; kb++) {
            scales_turn(kb);
            block(stage, std::false_type{});
            stage ^= 1;
            advance();
        }
        // c: lane (i, g) holds columns 16 g ... 16 g + 15 of rows i FM ... i FM + FM - 1 of the wave's part, column 4 q + j in acc[.][j][q]
        T* c = static_cast<T*>(a.c) + i0 * a.ldc + j0;
        const int mi = (int)min((uint64_t)BM, a.x.rows - i0), nj = (int)min((uint64_t)BN, a.p.rows - j0);
        constexpr int W = 16 / sizeof(T);
        const int row = wi + (lane & 15) * FM, col = wj + (lane >> 4) * 16;
        if (a.near && (nj == BN || nj % W == 0)) {
            __amdgpu_buffer_rsrc_t rc = __builtin_amdgcn_make_buffer_rsrc((void*)c, (short)0, (int)(((uint32_t)(mi - 1) * (uint32_t)a.ldc + (uint32_t)nj) * (uint32_t)sizeof(T)), 0x00027000);
            // the four lanes of a row change 16-byte pieces among them, so that a store writes 64 consecutive bytes of 16 rows
            const int piece = wj + (lane >> 4) * W;
#pragma unroll
            for (int i = 0; i < FM; i++) {
                u32x4 v[16 / W];
#pragma unroll
                for (int q = 0; q < 16 / W; q++) {
                    using V = __attribute__((ext_vector_type(W))) T;
                    V one;
#pragma unroll
                    for (int e = 0; e < W; e++) one[e] = (T)acc[i][(q * W + e) & 3][(q * W + e) >> 2];
                    v[q] = __builtin_bit_cast(u32x4, one);
                }
                if constexpr (W == 4) { swap32(v[0], v[2]); swap32(v[1], v[3]); swap16(v[0], v[1]); swap16(v[2], v[3]); }
                else { swap16(v[0], v[1]); swap32(v[0], v[1]); }
#pragma unroll
                for (int q = 0; q < 16 / W; q++) {
                    const int at = piece + q * 4 * W;
                    const uint32_t off = ((uint32_t)(row + i) * (uint32_t)a.ldc + (uint32_t)at) * (uint32_t)sizeof(T);
                    __builtin_amdgcn_raw_buffer_store_b128(v[q], rc, (int)(at < nj ? off : 0x7FFFFFFFu), 0, 0);
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < FM; i++)
#pragma unroll
                for (int q = 0; q < 16; q++)
                    if (row + i < mi && col + q < nj) c[(uint64_t)(row + i) * a.ldc + col + q] = (T)acc[i][q & 3][q >> 2];
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // (an unknown number of stores: none may be in flight where STORES of them are allowed for)
        }
        if (!more) break;
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // the copies of nothing have ended before the LDS is given back
}

// Few tiles of long rows: a workgroup owns 64 x 64, its four waves take every fourth block of 128 coordinates of it and their sums are added last, in order.
// Operands go from memory to the lanes that multiply them (32 bytes of 16 rows an access: the caches take 64 lanes one by one, which a chip with
// little to do has time for), the next block's while this one's are multiplied.  Rows of a lane as above: four neighbours, their scales a dword.
template <int TYPE>
__global__ void __launch_bounds__(256, 2) product_deep_kernel(ProductArgs a) {
    using T = typename Elem<TYPE>::T;
    extern __shared__ __attribute__((aligned(128))) uint8_t lds[];
    const uint32_t tn = blockIdx.x / a.tiles_m, tm = blockIdx.x - tn * a.tiles_m;
    const uint64_t i0 = (uint64_t)tm * 64, j0 = (uint64_t)tn * 64;
    const uint32_t mi = (uint32_t)min((uint64_t)64, a.x.rows - i0), nj = (uint32_t)min((uint64_t)64, a.p.rows - j0), stride = (uint32_t)a.x.row_bytes;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4;
    __amdgpu_buffer_rsrc_t rx = __builtin_amdgcn_make_buffer_rsrc((void*)(a.x.codes + i0 * stride), (short)0, (int)(mi * stride), 0x00027000);
    __amdgpu_buffer_rsrc_t rp = __builtin_amdgcn_make_buffer_rsrc((void*)(a.p.codes + j0 * stride), (short)0, (int)(nj * stride), 0x00027000);
    const uint8_t *sx = a.x.scales + i0 + (lane & 15) * 4, *sp = a.p.scales + j0 + (lane & 15) * 4;
    const uint32_t row_at = (lane & 15) * 4 * stride + g * 32;
    struct Block { u32x4 x[4][2], p[4][2]; uint32_t bx, bp; } now, next;
    auto load = [&](uint32_t kb, Block& b) {   // (past the last block or a row's last byte: zeros)
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const uint32_t at = kb * kBlock + g * 32 + h * 16 < stride ? 0u : 0x40000000u;
#pragma unroll
            for (int f = 0; f < 4; f++) {
                const int off = (int)((row_at + f * stride + kb * kBlock + h * 16) | at);
                b.x[f][h] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rx, off, 0, 0));
                b.p[f][h] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rp, off, 0, 0));
            }
        }
        const uint64_t last = min(kb, a.blocks - 1);
        __builtin_memcpy(&b.bx, sx + last * a.x.scale_stride, 4);
        __builtin_memcpy(&b.bp, sp + last * a.p.scale_stride, 4);
    };
    f32x4 acc[4][4];
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    load(wave, now);
    for (uint32_t kb = wave; kb < a.blocks; kb += 4) {
        load(kb + 4, next);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int e = 0; e < 4; e++) {
            bf16x8 wp[4];
#pragma unroll
            for (int j = 0; j < 4; j++) wp[j] = widen8(now.p[j][e >> 1][(e & 1) * 2], now.p[j][e >> 1][(e & 1) * 2 + 1], now.bp >> (j * 8) & 255u);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const bf16x8 wx = widen8(now.x[i][e >> 1][(e & 1) * 2], now.x[i][e >> 1][(e & 1) * 2 + 1], now.bx >> (i * 8) & 255u);
#pragma unroll
                for (int j = 0; j < 4; j++) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wp[j], wx, acc[i][j], 0, 0, 0);
            }
        }
        now = next;
    }
    f32x4* part = reinterpret_cast<f32x4*>(lds);
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) part[(wave * 16 + i * 4 + j) * 64 + lane] = acc[i][j];
    __syncthreads();
    // wave i adds the rows i of the lanes: columns 16 g + 4 e + j
    f32x4 sum[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        sum[j] = part[(wave * 4 + j) * 64 + lane];
#pragma unroll
        for (int w = 1; w < 4; w++) sum[j] += part[(w * 16 + wave * 4 + j) * 64 + lane];
    }
    const uint32_t row = (lane & 15) * 4 + wave, col = g * 16;
    if (row >= mi) return;
    T* c = static_cast<T*>(a.c) + (i0 + row) * a.ldc + j0 + col;
#pragma unroll
    for (int h = 0; h < 2; h++) {
        float v[8];
#pragma unroll
        for (int q = 0; q < 8; q++) v[q] = sum[q & 3][h * 2 + (q >> 2)];
        const int count = (int)nj - (int)col - h * 8;
        if (count > 0) store8<TYPE>(c + h * 8, min(count, 8), v);
    }
}

template <int BM, int BN, int WM>
void launch_tiles(const Rows8& x, const Rows8& p, const ProductPlan& plan, uint64_t dim, void* d_c, uint32_t ctype, uint64_t ldc, hipStream_t s) {
    const uint64_t tiles = plan.tiles_m * plan.tiles_n;
    if (tiles > 0x3FFFFFFFull) fail(AE_ERR_INVALID_ARG, "ae_points8_product: %llu x %llu are more products than one call takes", (unsigned long long)x.rows, (unsigned long long)p.rows);
    constexpr unsigned threads = (BM / WM) * (BN / 64) * 64, bytes = 2 * (BM + BN) * kBlock, resident = 256 * (bytes > 80 * 1024 ? 1 : 2);
    const bool near = ldc * type_size(ctype) < 0x7FFF0000ull / BM;
    const ProductArgs a{x, p, points8_blocks(dim), d_c, ldc, (uint32_t)plan.tiles_m, (uint32_t)plan.tiles_n, near ? 1u : 0u};
    const unsigned grid = tiles < resident ? (unsigned)((tiles + 7) / 8 * 8) : resident;
    by_type(ctype, [&](auto ty) {
        constexpr int TYPE = decltype(ty)::value;
        hipLaunchKernelGGL((product_tile_kernel<TYPE, BM, BN, WM>), dim3(grid), dim3(threads), bytes, s, a);
    });
    check_launch("points8_product");
}

void product(const Rows8& x, const Rows8& p, uint64_t dim, void* d_c, uint32_t ctype, uint64_t ldc, hipStream_t s) {
    const ProductPlan plan = product_plan(x.rows, p.rows, dim);
    if (plan.tile == 64) {
        const ProductArgs a{x, p, points8_blocks(dim), d_c, ldc, (uint32_t)plan.tiles_m, (uint32_t)plan.tiles_n, 0};
        by_type(ctype, [&](auto ty) {
            constexpr int TYPE = decltype(ty)::value;
            hipLaunchKernelGGL((product_deep_kernel<TYPE>), dim3((unsigned)(plan.tiles_m * plan.tiles_n)), dim3(256), 4 * 16 * 64 * 16, s, a);
        });
        check_launch("points8_product_deep");
        return;
    }
    if (plan.tile == 256) launch_tiles<256, 256, 128>(x, p, plan, dim, d_c, ctype, ldc, s);
    else launch_tiles<128, 128, 64>(x, p, plan, dim, d_c, ctype, ldc, s);
}

// Few rows: bound by the points' bytes, which go from memory straight to the matrix cores (16 points a wave, 32 coordinates of a block
// a lane).  Every workgroup quantises the rows itself, into LDS as the bf16 values they stand for, while its first points are on their way: one
// launch.  SPLIT waves share the blocks of a group of points where there are few points.
template <int XTYPE, int SPLIT, int TILES>   // TILES of 16 rows
__global__ void __launch_bounds__(256) product_few_kernel(const typename Elem<XTYPE>::T* __restrict__ x, uint32_t m, uint64_t ldx, uint32_t dim, Rows8 p, void* c_, uint32_t ctype, uint64_t ldc) {
    constexpr int GROUPS = 4 / SPLIT, AHEAD = 4;   // groups of 16 points a workgroup; blocks whose codes are fetched together
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4;
    const uint32_t blocks = (dim + kBlock - 1) / kBlock, stride = (uint32_t)p.row_bytes, lds_row = blocks * (kBlock * 2) + 16;
    const uint64_t j0 = (blockIdx.x * (uint64_t)GROUPS + wave / SPLIT) * 16;
    const uint32_t nj = j0 < p.rows ? (uint32_t)min((uint64_t)16, p.rows - j0) : 0;
    const uint64_t jb = nj ? j0 : 0;
    __amdgpu_buffer_rsrc_t rp = __builtin_amdgcn_make_buffer_rsrc((void*)(p.codes + jb * stride), (short)0, (int)(nj * stride), 0x00027000);
    const uint8_t* sp = p.scales + jb + (lane & 15);
    const uint32_t row_at = (uint32_t)(lane & 15) * stride + g * 32;
    u32x4 code[AHEAD][2];
    uint32_t byte[AHEAD];
    auto load = [&](uint32_t kb, int q) {   // (past the last block or a row's last byte: zeros)
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const uint32_t outside = kb * kBlock + g * 32 + h * 16 < stride ? 0u : 0x40000000u;
            code[q][h] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rp, (int)((row_at + kb * kBlock + h * 16) | outside), 0, 0));
        }
        byte[q] = sp[min(kb, blocks - 1) * p.scale_stride];
    };
    const uint32_t kb0 = SPLIT == 1 ? 0 : wave % SPLIT;
#pragma unroll
    for (int q = 0; q < AHEAD; q++) load(kb0 + q * SPLIT, q);
    // the rows: as ae_points8_write holds them, 16 lanes a block
    for (uint32_t u = tid >> 4; u < m * blocks; u += 16) {
        const uint32_t i = u / blocks, b = u - i * blocks, k = b * kBlock + (lane & 15) * 8;
        float v[8];
        load8<XTYPE>(x + i * ldx + (k < dim ? k : 0), k < dim ? (int)min(8u, dim - k) : 0, v);
        const uint32_t scale = scale_byte(max16(amax8(v)));
        const uint2 e = encode8(v, scale);
        *reinterpret_cast<bf16x8*>(lds + i * lds_row + k * 2) = widen8(e.x, e.y, scale);
    }
    __syncthreads();
    uint32_t mine[TILES];   // (rows that do not exist repeat the last one, for nobody)
    f32x4 acc[TILES][2];
#pragma unroll
    for (int i = 0; i < TILES; i++) {
        mine[i] = min((uint32_t)(lane & 15) + i * 16, m - 1) * lds_row + g * 64;
        acc[i][0] = acc[i][1] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    for (uint32_t kb = kb0; kb < blocks; kb += AHEAD * SPLIT) {
#pragma unroll
        for (int q = 0; q < AHEAD; q++) {
            const uint32_t at = min(kb + q * SPLIT, blocks - 1);   // (past the last block the codes are zeros)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const bf16x8 wp = widen8(code[q][e >> 1][(e & 1) * 2], code[q][e >> 1][(e & 1) * 2 + 1], byte[q]);
#pragma unroll
                for (int i = 0; i < TILES; i++) {
                    const bf16x8 wx = *reinterpret_cast<const bf16x8*>(lds + mine[i] + at * (kBlock * 2) + e * 16);
                    acc[i][e & 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wp, wx, acc[i][e & 1], 0, 0, 0);
                }
            }
            load(kb + (q + AHEAD) * SPLIT, q);
        }
    }
    f32x4 sum[TILES];
#pragma unroll
    for (int i = 0; i < TILES; i++) sum[i] = acc[i][0] + acc[i][1];
    if constexpr (SPLIT > 1) {   // the waves' shares in order
        __syncthreads();
        f32x4* part = reinterpret_cast<f32x4*>(lds);
#pragma unroll
        for (int i = 0; i < TILES; i++) part[i * 256 + tid] = sum[i];
        __syncthreads();
        if (wave % SPLIT) return;
#pragma unroll
        for (int i = 0; i < TILES; i++)
#pragma unroll
            for (int q = 1; q < SPLIT; q++) sum[i] += part[i * 256 + tid + q * 64];
    }
    // a lane holds 4 consecutive points of rows lane & 15
#pragma unroll
    for (int i = 0; i < TILES; i++) {
        const uint32_t r = i * 16 + (lane & 15);
        if (r >= m) continue;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const uint32_t j = g * 4 + e;
            if (j >= nj) continue;
            const uint64_t at = r * ldc + j0 + j;
            if (ctype == AE_TYPE_F32) static_cast<float*>(c_)[at] = sum[i][e];
            else if (ctype == AE_TYPE_BF16) static_cast<__bf16*>(c_)[at] = (__bf16)sum[i][e];
            else static_cast<_Float16*>(c_)[at] = (_Float16)sum[i][e];
        }
    }
}

void product_few(const void* d_x, uint32_t xtype, uint64_t m, uint64_t ldx, uint64_t dim, const Rows8& p, void* d_c, uint32_t ctype, uint64_t ldc, hipStream_t s) {
    const unsigned tiles = m <= 16 ? 1 : m <= 32 ? 2 : 4, bytes = (unsigned)std::max<uint64_t>(m * few_lds_row(dim), 4096 * tiles);
    by_type(xtype, [&](auto ty) {
        constexpr int TYPE = decltype(ty)::value;
        auto go = [&](auto kernel, unsigned points) {
            hipLaunchKernelGGL(kernel, dim3((unsigned)((p.rows + points - 1) / points)), dim3(256), bytes, s, static_cast<const typename Elem<TYPE>::T*>(d_x), (uint32_t)m, ldx,
                               (uint32_t)dim, p, d_c, ctype, ldc);
        };
        const bool whole = few_points(p.rows, dim) == 64;
        if (tiles == 1) whole ? go(product_few_kernel<TYPE, 1, 1>, 64) : go(product_few_kernel<TYPE, 4, 1>, 16);
        else if (tiles == 2) whole ? go(product_few_kernel<TYPE, 1, 2>, 64) : go(product_few_kernel<TYPE, 4, 2>, 16);
        else go(product_few_kernel<TYPE, 1, 4>, 64);   // (33 rows or more have at most 303 coordinates)
    });
    check_launch("points8_product_few");
}

uint64_t product_work(uint64_t m, uint64_t dim) { return m * points8_row_bytes(dim) + points8_blocks(dim) * points8_scale_stride(m) + kScaleSlack; }

}  // namespace

extern "C" {

int32_t ae_points8_product_work(const ae_points8* p, uint64_t n, uint64_t m, uint64_t* bytes) {
    return guard([&] {
        if (!p || !bytes) fail(AE_ERR_INVALID_ARG, "ae_points8_product_work: null argument");
        if (m > (1ull << 32)) fail(AE_ERR_INVALID_ARG, "ae_points8_product_work: %llu rows are out of range", (unsigned long long)m);
        *bytes = m && n && !few_rows(m, n, p->dim) ? product_work(m, p->dim) : 0;
    });
}

int32_t ae_points8_product(const ae_points8* p, uint64_t first, uint64_t n, const void* d_x, uint32_t xtype, uint64_t m, uint64_t ldx, void* d_c, uint32_t ctype, uint64_t ldc,
                           void* d_work, uint64_t work_bytes, void* stream) {
    return guard([&] {
        require_device();
        check_points8(p, first, n, "ae_points8_product");
        check_type(xtype, "ae_points8_product: x");
        check_type(ctype, "ae_points8_product: c");
        if (n == 0 || m == 0) return;
        check_rows(d_x, xtype, m, p->dim, ldx, "ae_points8_product: x");
        check_rows(d_c, ctype, m, n, ldc, "ae_points8_product: c");
        if (few_rows(m, n, p->dim)) return product_few(d_x, xtype, m, ldx, p->dim, points8_rows(p, first, n), d_c, ctype, ldc, (hipStream_t)stream);
        const uint64_t need = product_work(m, p->dim);
        if (!d_work || work_bytes < need) fail(AE_ERR_INVALID_ARG, "ae_points8_product: %llu bytes of scratch are needed, %llu given", (unsigned long long)need, (unsigned long long)work_bytes);
        check_aligned(d_work, 16, "ae_points8_product: work");
        uint8_t* codes = static_cast<uint8_t*>(d_work);
        uint8_t* scales = codes + m * p->row_bytes;
        points8_quantise(d_x, xtype, m, ldx, p->dim, codes, scales, points8_scale_stride(m), (hipStream_t)stream);
        product(Rows8{codes, scales, p->row_bytes, points8_scale_stride(m), m}, points8_rows(p, first, n), p->dim, d_c, ctype, ldc, (hipStream_t)stream);
    });
}

int32_t ae_points8_product_points(const ae_points8* p, uint64_t first, uint64_t n, const ae_points8* q, uint64_t q_first, uint64_t m, void* d_c, uint32_t ctype, uint64_t ldc,
                                  void* stream) {
    return guard([&] {
        require_device();
        check_points8(p, first, n, "ae_points8_product_points");
        check_points8(q, q_first, m, "ae_points8_product_points");
        if (p->dim != q->dim) fail(AE_ERR_INVALID_ARG, "ae_points8_product_points: stores of %llu and %llu coordinates", (unsigned long long)p->dim, (unsigned long long)q->dim);
        check_type(ctype, "ae_points8_product_points: c");
        if (n == 0 || m == 0) return;
        check_rows(d_c, ctype, m, n, ldc, "ae_points8_product_points: c");
        product(points8_rows(q, q_first, m), points8_rows(p, first, n), p->dim, d_c, ctype, ldc, (hipStream_t)stream);
    });
}

}  // extern "C"
