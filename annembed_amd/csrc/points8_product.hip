// points8_product.hip -- rows times the points held in 8 bits: c[i][j] = <x_i, p_j> on the scaled 8-bit matrix cores.
//
// v_mfma_scale_f32_32x32x64_f8f6f4 takes 32 + 32 rows of 64 e4m3 codes and one power-of-two scale per row and 32 coordinates: two of them
// cover a block of 128 with the block's own scale bytes, so the scales cost no arithmetic at all.  Which of the 64 coordinates a lane holds
// does not matter as long as both operands agree (the scale is one for the block).
//
// The 8-bit cores add eight products of consecutive codes at a time, cut 13 bits below the largest of the eight (measured on this chip:
// 2^12 + 2^-1 is kept, 2^12 + 2^-2 is 2^12).  That is at most 7 * 2^-13 of the sum of the products' magnitudes, 1e-5 of it in the
// root mean square over encoder-like rows: below a 16-bit result's own rounding, not below an f32 result's.  So c of 16 bits takes the 8-bit
// cores, and c of f32 takes the bf16 cores at half their rate: every value held is exact in bf16, the products too, the sums are f32.
#include "points8.h"

using namespace ae;

namespace {

// Tiles in LDS: a row's block of 128 codes is 8 chunks of 16 bytes; chunk c of row r lies at place c ^ ((r >> 1) & 7), so 16 lanes that read
// the same chunk of consecutive rows touch all 64 banks once.  The copy to LDS writes lane after lane, so the lanes permute what they fetch.
__device__ __forceinline__ int swizzled(int row, int chunk) { return row * kBlock + ((chunk ^ ((row >> 1) & 7)) << 4); }


__device__ __forceinline__ i32x8 join(u32x4 a, u32x4 b) {
    return i32x8{(int)a[0], (int)a[1], (int)a[2], (int)a[3], (int)b[0], (int)b[1], (int)b[2], (int)b[3]};
}

struct ProductArgs {
    Rows8 x, p;       // m rows, n rows
    uint32_t blocks;
    void* c;
    uint64_t ldc;
    uint32_t tiles_m, tiles_n;
    uint32_t vec;     // rows of c can be written 16 bytes at a time
};

// Which tile a workgroup owns.  Workgroups go to the 8 XCDs in turn, each with an L2 of its own: the tiles are handed out so that an XCD
// walks a run of them, kPanel rows of tiles at a time, and the points it fetched serve all rows of the panel.
constexpr uint32_t kPanel = 4;
__device__ __forceinline__ void tile_of(uint32_t tiles_m, uint32_t tiles_n, uint32_t& tm, uint32_t& tn) {
    const uint32_t total = tiles_m * tiles_n, each = total / 8, more = total % 8, xcd = blockIdx.x % 8, at = blockIdx.x / 8;
    const uint32_t id = xcd * each + min(xcd, more) + at;
    const uint32_t panel = id / (kPanel * tiles_n), in = id - panel * kPanel * tiles_n;
    const uint32_t rows = min(kPanel, tiles_m - panel * kPanel);
    tn = in / rows;
    tm = panel * kPanel + in - tn * rows;
}

// A BM x BN tile of c, waves of WM x 64, one block of 128 coordinates per step, two stages of LDS in turn: the copies of the next block are
// in flight while the matrix cores work on this one.
template <int TYPE, int BM, int BN, int WM>
__global__ void __launch_bounds__((BM / WM) * (BN / 64) * 64, (BM + BN) * kBlock * 2 > 80 * 1024 ? (BM / WM) * (BN / 64) / 4 : (BM / WM) * (BN / 64) / 2)
product_tile_kernel(ProductArgs a) {
    constexpr int WN = 64, WAVES = (BM / WM) * (BN / WN), FM = WM / 32, FN = WN / 32;
    constexpr int STAGE = (BM + BN) * kBlock;
    extern __shared__ __attribute__((aligned(128))) uint8_t lds[];
    using T = typename Elem<TYPE>::T;
    uint32_t tm, tn;
    tile_of(a.tiles_m, a.tiles_n, tm, tn);
    const uint64_t i0 = (uint64_t)tm * BM, j0 = (uint64_t)tn * BN;
    const int mi = (int)min((uint64_t)BM, a.x.rows - i0), nj = (int)min((uint64_t)BN, a.p.rows - j0);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wi = (wave / (BN / WN)) * WM, wj = (wave % (BN / WN)) * WN;
    // rows beyond the tile and bytes beyond a row are outside the buffers' range: they read as 0
    const uint32_t stride = (uint32_t)a.x.row_bytes;
    __amdgpu_buffer_rsrc_t rx = __builtin_amdgcn_make_buffer_rsrc((void*)(a.x.codes + i0 * stride), (short)0, (int)((uint32_t)mi * stride), 0x00027000);
    __amdgpu_buffer_rsrc_t rp = __builtin_amdgcn_make_buffer_rsrc((void*)(a.p.codes + j0 * stride), (short)0, (int)((uint32_t)nj * stride), 0x00027000);
    static_assert(WAVES % 2 == 0 && BM / 8 % WAVES == 0 && BN / 8 % WAVES == 0, "a wave copies whole groups of 8 rows of one operand");
    const uint32_t chunk = (lane & 7) ^ (((wave & 1) << 2) + (lane >> 4));   // (row >> 1) & 7 of row = 8 (q WAVES + wave) + (lane >> 3)
    const uint32_t lane_off = (uint32_t)(wave * 8 + (lane >> 3)) * stride + chunk * 16;
    auto fetch = [&](uint32_t kb, uint8_t* to) {
        const bool in = kb * kBlock + chunk * 16 < stride;
#pragma unroll
        for (int q = 0; q < (BM + BN) / 8 / WAVES; q++) {
            const bool of_x = q < BM / 8 / WAVES;
            const uint32_t off = lane_off + (uint32_t)((of_x ? q : q - BM / 8 / WAVES) * WAVES * 8) * stride + kb * kBlock;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(of_x ? rx : rp, (__attribute__((address_space(3))) void*)(to + (q * WAVES + wave) * 8 * kBlock), 16, (int)(in ? off : 0x7FFFFFFFu), 0, 0, 0);
        }
    };
    f32x16 acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; i++)
#pragma unroll
        for (int j = 0; j < FN; j++)
#pragma unroll
            for (int t = 0; t < 16; t++) acc[i][j][t] = 0.f;
    // scale bytes: a dword holds four blocks of a row; the next four are on their way while four are used
    const uint32_t* sx[FM];
    const uint32_t* sp[FN];
    uint32_t nx[FM], np[FN], bx[FM], bp[FN];
#pragma unroll
    for (int i = 0; i < FM; i++) {
        sx[i] = reinterpret_cast<const uint32_t*>(a.x.scales + (i0 + min(wi + i * 32 + (lane & 31), mi - 1)) * a.x.scale_stride);
        nx[i] = sx[i][0];
    }
#pragma unroll
    for (int j = 0; j < FN; j++) {
        sp[j] = reinterpret_cast<const uint32_t*>(a.p.scales + (j0 + min(wj + j * 32 + (lane & 31), nj - 1)) * a.p.scale_stride);
        np[j] = sp[j][0];
    }
    fetch(0, lds);
    for (uint32_t kb = 0; kb < a.blocks; kb++) {
        __syncthreads();   // this stage has arrived, everybody has left the other one
        if ((kb & 3) == 0) {
            const uint32_t next = min(kb / 4 + 1, (a.blocks - 1) / 4);
#pragma unroll
            for (int i = 0; i < FM; i++) { bx[i] = nx[i]; nx[i] = sx[i][next]; }
#pragma unroll
            for (int j = 0; j < FN; j++) { bp[j] = np[j]; np[j] = sp[j][next]; }
        } else {
#pragma unroll
            for (int i = 0; i < FM; i++) bx[i] >>= 8;
#pragma unroll
            for (int j = 0; j < FN; j++) bp[j] >>= 8;
        }
        const uint8_t* t = lds + (kb & 1) * STAGE;
        if (kb + 1 < a.blocks) fetch(kb + 1, lds + ((kb + 1) & 1) * STAGE);
#pragma unroll
        for (int h = 0; h < 2; h++) {
            u32x4 fx[FM][2], fp[FN][2];
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const int c = h * 4 + (lane >> 5) * 2 + e;
#pragma unroll
                for (int j = 0; j < FN; j++) fp[j][e] = *reinterpret_cast<const u32x4*>(t + swizzled(BM + wj + j * 32 + (lane & 31), c));
#pragma unroll
                for (int i = 0; i < FM; i++) fx[i][e] = *reinterpret_cast<const u32x4*>(t + swizzled(wi + i * 32 + (lane & 31), c));
            }
            if constexpr (TYPE == AE_TYPE_F32) {
#pragma unroll
                for (int e = 0; e < 4; e++) {   // 8 codes of each operand
                    bf16x8 wx[FM], wp[FN];
#pragma unroll
                    for (int j = 0; j < FN; j++) wp[j] = widen8(fp[j][e >> 1][(e & 1) * 2], fp[j][e >> 1][(e & 1) * 2 + 1], bp[j] & 255u);
#pragma unroll
                    for (int i = 0; i < FM; i++) wx[i] = widen8(fx[i][e >> 1][(e & 1) * 2], fx[i][e >> 1][(e & 1) * 2 + 1], bx[i] & 255u);
#pragma unroll
                    for (int i = 0; i < FM; i++)
#pragma unroll
                        for (int j = 0; j < FN; j++) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(wp[j], wx[i], acc[i][j], 0, 0, 0);
                }
            } else {
#pragma unroll
                for (int i = 0; i < FM; i++)
#pragma unroll
                    for (int j = 0; j < FN; j++)
                        acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(join(fp[j][0], fp[j][1]), join(fx[i][0], fx[i][1]), acc[i][j], 0, 0, 0, (int)bp[j], 0, (int)bx[i]);
            }
        }
    }
    // The points are the matrix cores' rows: a lane holds runs of 4 consecutive j of one row i.  A wave turns its part in a share of the
    // stages and writes rows of 64 j, 16 bytes a lane.
    __syncthreads();
    constexpr int ROW = WN * sizeof(T), CH = ROW / 16;                      // bytes and 16-byte chunks of a row
    constexpr int FIT = 2 * STAGE / WAVES / (32 * ROW);                      // fragments of 32 rows that a wave has room for
    constexpr int STEP = FIT >= FM ? FM : FIT >= FM / 2 ? FM / 2 : 1;
    static_assert(WAVES * STEP * 32 * ROW <= 2 * STAGE, "the turned tiles fit in the stages");
    uint8_t* mine = lds + wave * (STEP * 32 * ROW);
    T* c = static_cast<T*>(a.c);
    auto place = [&](int r, int ch) { return r * ROW + ((ch ^ (ROW == 128 ? (r >> 1) & 7 : r & 15)) << 4); };
#pragma unroll
    for (int i = 0; i < FM; i += STEP) {
#pragma unroll
        for (int f = 0; f < STEP; f++)
#pragma unroll
            for (int j = 0; j < FN; j++)
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    using V = __attribute__((ext_vector_type(4))) T;
                    V v;
#pragma unroll
                    for (int e = 0; e < 4; e++) v[e] = (T)acc[i + f][j][q * 4 + e];
                    const int byte = (j * 32 + q * 8 + (lane >> 5) * 4) * (int)sizeof(T);
                    *reinterpret_cast<V*>(mine + place(f * 32 + (lane & 31), byte >> 4) + (byte & 15)) = v;
                }
        // (within a wave LDS operations are in order)
#pragma unroll
        for (int q = 0; q < STEP * 32 * CH / 64; q++) {
            const int at = q * 64 + lane, r = at / CH, ch = at % CH;
            const int row = wi + i * 32 + r, col = wj + ch * (16 / (int)sizeof(T));
            const u32x4 v = *reinterpret_cast<const u32x4*>(mine + place(r, ch));
            if (row >= mi || col >= nj) continue;
            T* to = c + (i0 + row) * a.ldc + j0 + col;
            if (a.vec && col + 16 / (int)sizeof(T) <= nj) *reinterpret_cast<u32x4*>(to) = v;
            else {
                const T* one = reinterpret_cast<const T*>(&v);
#pragma unroll
                for (int e = 0; e < 16 / (int)sizeof(T); e++)
                    if (col + e < nj) to[e] = one[e];
            }
        }
    }
}

template <int BM, int BN, int WM>
void launch_tiles(const Rows8& x, const Rows8& p, uint64_t dim, void* d_c, uint32_t ctype, uint64_t ldc, hipStream_t s) {
    const uint64_t tiles_m = (x.rows + BM - 1) / BM, tiles_n = (p.rows + BN - 1) / BN;
    if (tiles_m * tiles_n > 0x3FFFFFull) fail(AE_ERR_INVALID_ARG, "ae_points8_product: %llu x %llu are more products than one call takes", (unsigned long long)x.rows, (unsigned long long)p.rows);
    const ProductArgs a{x, p, points8_blocks(dim), d_c, ldc, (uint32_t)tiles_m, (uint32_t)tiles_n, vector_rows(d_c, ctype, ldc) ? 1u : 0u};
    constexpr unsigned threads = (BM / WM) * (BN / 64) * 64, bytes = 2 * (BM + BN) * kBlock;
    by_type(ctype, [&](auto ty) {
        constexpr int TYPE = decltype(ty)::value;
        hipLaunchKernelGGL((product_tile_kernel<TYPE, BM, BN, WM>), dim3((unsigned)(tiles_m * tiles_n)), dim3(threads), bytes, s, a);
    });
    check_launch("points8_product");
}

void product(const Rows8& x, const Rows8& p, uint64_t dim, void* d_c, uint32_t ctype, uint64_t ldc, hipStream_t s) {
    const char* v = debug_knob("AE_P8");
    const int w = v ? atoi(v) : 1;
    if (w == 2) launch_tiles<256, 256, 128>(x, p, dim, d_c, ctype, ldc, s);
    else if (w == 3) launch_tiles<64, 256, 64>(x, p, dim, d_c, ctype, ldc, s);
    else if (w == 4) launch_tiles<128, 256, 64>(x, p, dim, d_c, ctype, ldc, s);
    else launch_tiles<128, 128, 64>(x, p, dim, d_c, ctype, ldc, s);
}

uint64_t product_work(uint64_t m, uint64_t dim) { return m * (points8_row_bytes(dim) + points8_scale_stride(dim)); }

}  // namespace

extern "C" {

int32_t ae_points8_product_work(const ae_points8* p, uint64_t n, uint64_t m, uint64_t* bytes) {
    return guard([&] {
        if (!p || !bytes) fail(AE_ERR_INVALID_ARG, "ae_points8_product_work: null argument");
        if (m > (1ull << 32)) fail(AE_ERR_INVALID_ARG, "ae_points8_product_work: %llu rows are out of range", (unsigned long long)m);
        *bytes = product_work(m, p->dim);
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
        const uint64_t need = product_work(m, p->dim);
        if (!d_work || work_bytes < need) fail(AE_ERR_INVALID_ARG, "ae_points8_product: %llu bytes of scratch are needed, %llu given", (unsigned long long)need, (unsigned long long)work_bytes);
        check_aligned(d_work, 16, "ae_points8_product: work");
        uint8_t* codes = static_cast<uint8_t*>(d_work);
        uint8_t* scales = codes + m * p->row_bytes;
        points8_quantise(d_x, xtype, m, ldx, p->dim, codes, scales, (hipStream_t)stream);
        product(Rows8{codes, scales, p->row_bytes, p->scale_stride, m}, points8_rows(p, first, n), p->dim, d_c, ctype, ldc, (hipStream_t)stream);
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
