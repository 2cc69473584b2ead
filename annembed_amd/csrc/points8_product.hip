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
};

// 128 x 128 tile of c, 4 waves of 64 x 64, one block of 128 coordinates per step, two tiles of LDS in turn
template <int TYPE>
__global__ void __launch_bounds__(256, 2) product_tile_kernel(ProductArgs a, uint32_t tiles_n) {
    constexpr int BM = 128, BN = 128;
    __shared__ __attribute__((aligned(128))) uint8_t lds[2][(BM + BN) * kBlock];
    const uint32_t tm = blockIdx.x / tiles_n, tn = blockIdx.x - tm * tiles_n;
    const uint64_t i0 = (uint64_t)tm * BM, j0 = (uint64_t)tn * BN;
    const int mi = (int)min((uint64_t)BM, a.x.rows - i0), nj = (int)min((uint64_t)BN, a.p.rows - j0);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int wi = (wave >> 1) * 64, wj = (wave & 1) * 64;
    // rows beyond the tile and bytes beyond a row are outside the buffers' range: they read as 0
    const uint32_t stride = (uint32_t)a.x.row_bytes;
    __amdgpu_buffer_rsrc_t rx = __builtin_amdgcn_make_buffer_rsrc((void*)(a.x.codes + i0 * stride), (short)0, (int)((uint32_t)mi * stride), 0x00027000);
    __amdgpu_buffer_rsrc_t rp = __builtin_amdgcn_make_buffer_rsrc((void*)(a.p.codes + j0 * stride), (short)0, (int)((uint32_t)nj * stride), 0x00027000);
    auto fetch = [&](uint32_t kb, uint8_t* to) {
#pragma unroll
        for (int q = 0; q < (BM + BN) / 32; q++) {   // 8 rows a wave and turn
            const int r = (q * 4 + wave) * 8 + (lane >> 3);   // row of the tile: x first, then p
            const int rr = q < BM / 32 ? r : r - BM;
            const int chunk = (lane & 7) ^ ((r >> 1) & 7);
            const uint32_t k = kb * kBlock + chunk * 16;
            const uint32_t off = k < stride ? (uint32_t)rr * stride + k : 0x7FFFFFFFu;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(q < BM / 32 ? rx : rp, (__attribute__((address_space(3))) void*)(to + (q * 4 + wave) * 8 * kBlock), 16, (int)off, 0, 0, 0);
        }
    };
    f32x16 acc[2][2];
#pragma unroll
    for (int q = 0; q < 4; q++)
#pragma unroll
        for (int t = 0; t < 16; t++) acc[q >> 1][q & 1][t] = 0.f;
    const uint8_t* sx[2];
    const uint8_t* sp[2];
#pragma unroll
    for (int q = 0; q < 2; q++) {
        sx[q] = a.x.scales + (i0 + min(wi + q * 32 + (lane & 31), mi - 1)) * a.x.scale_stride;
        sp[q] = a.p.scales + (j0 + min(wj + q * 32 + (lane & 31), nj - 1)) * a.p.scale_stride;
    }
    fetch(0, lds[0]);
    for (uint32_t kb = 0; kb < a.blocks; kb++) {
        __syncthreads();   // (waits for the loads to LDS)
        if (kb + 1 < a.blocks) fetch(kb + 1, lds[(kb + 1) & 1]);
        const uint8_t* t = lds[kb & 1];
        int bx[2], bp[2];
#pragma unroll
        for (int q = 0; q < 2; q++) { bx[q] = sx[q][kb]; bp[q] = sp[q][kb]; }
#pragma unroll
        for (int h = 0; h < 2; h++) {
            u32x4 fx[2][2], fp[2][2];
#pragma unroll
            for (int q = 0; q < 2; q++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const int chunk = h * 4 + (lane >> 5) * 2 + e;
                    fx[q][e] = *reinterpret_cast<const u32x4*>(t + swizzled(wi + q * 32 + (lane & 31), chunk));
                    fp[q][e] = *reinterpret_cast<const u32x4*>(t + swizzled(BM + wj + q * 32 + (lane & 31), chunk));
                }
            if constexpr (TYPE == AE_TYPE_F32) {
#pragma unroll
                for (int e = 0; e < 4; e++) {   // 8 codes of each operand
                    bf16x8 wx[2], wp[2];
#pragma unroll
                    for (int q = 0; q < 2; q++) {
                        wx[q] = widen8(fx[q][e >> 1][(e & 1) * 2], fx[q][e >> 1][(e & 1) * 2 + 1], bx[q]);
                        wp[q] = widen8(fp[q][e >> 1][(e & 1) * 2], fp[q][e >> 1][(e & 1) * 2 + 1], bp[q]);
                    }
#pragma unroll
                    for (int i = 0; i < 2; i++)
#pragma unroll
                        for (int j = 0; j < 2; j++) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(wp[j], wx[i], acc[i][j], 0, 0, 0);
                }
            } else {
#pragma unroll
                for (int i = 0; i < 2; i++)
#pragma unroll
                    for (int j = 0; j < 2; j++)
                        acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(join(fp[j][0], fp[j][1]), join(fx[i][0], fx[i][1]), acc[i][j], 0, 0, 0, bp[j], 0, bx[i]);
            }
        }
    }
    // the points are the matrix cores' rows: a lane holds runs of 4 consecutive j of one i
    using T = typename Elem<TYPE>::T;
    T* c = static_cast<T*>(a.c);
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const int r = wi + i * 32 + (lane & 31);
        if (r >= mi) continue;
        T* to = c + (i0 + r) * a.ldc + j0;
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
            for (int q = 0; q < 4; q++) {
                const int col = wj + j * 32 + q * 8 + (lane >> 5) * 4;
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (col + e < nj) to[col + e] = (T)acc[i][j][q * 4 + e];
            }
    }
}

void product(const Rows8& x, const Rows8& p, uint64_t dim, void* d_c, uint32_t ctype, uint64_t ldc, hipStream_t s) {
    const uint64_t tiles_m = (x.rows + 127) / 128, tiles_n = (p.rows + 127) / 128;
    if (tiles_m * tiles_n > 0xFFFFFFull) fail(AE_ERR_INVALID_ARG, "ae_points8_product: %llu x %llu are more products than one call takes", (unsigned long long)x.rows, (unsigned long long)p.rows);
    by_type(ctype, [&](auto ty) {
        constexpr int TYPE = decltype(ty)::value;
        hipLaunchKernelGGL((product_tile_kernel<TYPE>), dim3((unsigned)(tiles_m * tiles_n)), dim3(256), 0, s, ProductArgs{x, p, points8_blocks(dim), d_c, ldc}, (uint32_t)tiles_n);
    });
    check_launch("points8_product");
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
