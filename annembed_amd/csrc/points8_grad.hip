// points8_grad.hip -- the gradient of the 8-bit product to its rows: dx[i][k] = sum_j dc[i][j] * p_j[k].
//
// The sum runs over the points, and a point's scales change with j: they cannot go into the matrix cores' scale operand, which belongs to a
// run of the summed axis.  But code * 2^e is exact in bf16, and dc of f32 (f16) is the sum of three (two) bf16 numbers, so bf16 matrix cores
// compute the product of the values themselves with f32 sums: nothing is rounded before the result.
//
// A workgroup owns 128 rows x 128 coordinates (one block: one scale byte per point) and walks a slice of the points 64 at a time.  The
// points' codes are turned on the way to LDS: a thread takes 4 coordinates of 8 points, widens them and writes 8 points of one coordinate
// as 16 bytes, the matrix cores' operand.  Few rows leave few tiles: the points are split into slices whose sums are joined in order.
#include "points8.h"

using namespace ae;

namespace {

constexpr int kTile = 128;   // rows and coordinates of a workgroup
constexpr int kStep = 64;    // points per step: 128 bytes of bf16

template <int TYPE> constexpr int terms_of() { return TYPE == AE_TYPE_F32 ? 3 : TYPE == AE_TYPE_F16 ? 2 : 1; }

__device__ __forceinline__ int at_rows(int r, int chunk) { return r * 128 + ((chunk ^ ((r >> 1) & 7)) << 4); }
// coordinates: written four rows apart, read row after row -- both without bank conflicts
__device__ __forceinline__ int at_coords(int k, int chunk) { return k * 128 + ((chunk ^ ((k >> 2) & 7) ^ ((k & 2) << 1)) << 4); }

// v as the sum of TERMS bf16 numbers, the first ones cut off (never past the largest bf16), exact apart from what lies below bf16's range
template <int TERMS>
__device__ __forceinline__ void split(float v, __bf16 (&t)[TERMS]) {
    if constexpr (TERMS == 1) { t[0] = (__bf16)v; return; }
    const bool finite = (__float_as_uint(v) & 0x7FFFFFFFu) < 0x7F800000u;
#pragma unroll
    for (int q = 0; q + 1 < TERMS; q++) {
        const float cut = __uint_as_float(__float_as_uint(v) & 0xFFFF0000u);
        t[q] = finite ? (__bf16)cut : (__bf16)v;
        v = finite ? v - cut : 0.f;
    }
    t[TERMS - 1] = (__bf16)v;
}

struct GradArgs {
    const void* dc;
    uint64_t lddc;
    uint64_t m, n, dim;
    Rows8 p;
    uint64_t per_slice;   // points per slice, a multiple of kStep
    float* part;          // [slices][m][ldp]
    uint64_t ldp;
};

template <int TYPE>
__global__ void __launch_bounds__(256) grad_tile_kernel(GradArgs a, uint32_t tiles_k, bool vec) {
    using T = typename Elem<TYPE>::T;
    constexpr int TERMS = terms_of<TYPE>();
    __shared__ __attribute__((aligned(128))) uint8_t ldc_[TERMS][kTile * 128];
    __shared__ __attribute__((aligned(128))) uint8_t ldp_[kTile * 128];
    const uint32_t ti = blockIdx.x / tiles_k, tk = blockIdx.x - ti * tiles_k;
    const uint64_t i0 = (uint64_t)ti * kTile, k0 = (uint64_t)tk * kTile;
    const uint64_t jb = blockIdx.y * a.per_slice, je = min(a.n, jb + a.per_slice);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int wi = (wave >> 1) * 64, wk = (wave & 1) * 64;
    const int kg = tid & 31, jg = tid >> 5;   // this thread's 4 coordinates and 8 points
    const T* dc = static_cast<const T*>(a.dc);
    float va[4][8];
    uint32_t code[8];
    uint32_t byte[8];
    auto load = [&](uint64_t j0) {
#pragma unroll
        for (int q = 0; q < 4; q++) {
            const int idx = tid + q * 256, r = idx >> 3;
            const uint64_t j = j0 + (idx & 7) * 8;
            const int count = i0 + r < a.m && j < je ? (int)min((uint64_t)8, je - j) : 0;
            load8<TYPE>(dc + (count ? (i0 + r) * a.lddc + j : 0), vec && count == 8, count, va[q]);
        }
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const uint64_t j = j0 + jg * 8 + e, k = k0 + kg * 4;
            const bool in = j < je && k < a.p.row_bytes;
            code[e] = in ? *reinterpret_cast<const uint32_t*>(a.p.codes + j * a.p.row_bytes + k) : 0;
            byte[e] = in ? a.p.scales[tk * a.p.scale_stride + j] : 0;
        }
    };
    f32x16 acc[2][2];
#pragma unroll
    for (int q = 0; q < 4; q++)
#pragma unroll
        for (int t = 0; t < 16; t++) acc[q >> 1][q & 1][t] = 0.f;
    load(jb);
    for (uint64_t j0 = jb; j0 < je; j0 += kStep) {
#pragma unroll
        for (int q = 0; q < 4; q++) {
            const int idx = tid + q * 256;
            bf16x8 t[TERMS];
#pragma unroll
            for (int e = 0; e < 8; e++) {
                __bf16 one[TERMS];
                split<TERMS>(va[q][e], one);
#pragma unroll
                for (int u = 0; u < TERMS; u++) t[u][e] = one[u];
            }
#pragma unroll
            for (int u = 0; u < TERMS; u++) *reinterpret_cast<bf16x8*>(ldc_[u] + at_rows(idx >> 3, idx & 7)) = t[u];
        }
        uint32_t wide[8][2];   // [point][coordinates 0, 1 | 2, 3] as pairs of bf16
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const float scale = __uint_as_float(byte[e] << 23);
            const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)code[e], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)code[e], true);
            const float v0 = lo[0] * scale, v1 = lo[1] * scale, v2 = hi[0] * scale, v3 = hi[1] * scale;   // exact, and bf16 numbers: the upper halves
            wide[e][0] = __builtin_amdgcn_perm(__float_as_uint(v1), __float_as_uint(v0), 0x07060302u);
            wide[e][1] = __builtin_amdgcn_perm(__float_as_uint(v3), __float_as_uint(v2), 0x07060302u);
        }
#pragma unroll
        for (int t = 0; t < 4; t++) {
            u32x4 w;
#pragma unroll
            for (int e = 0; e < 4; e++)
                w[e] = __builtin_amdgcn_perm(wide[2 * e + 1][t >> 1], wide[2 * e][t >> 1], t & 1 ? 0x07060302u : 0x05040100u);
            *reinterpret_cast<u32x4*>(ldp_ + at_coords(kg * 4 + t, jg)) = w;
        }
        __syncthreads();
        if (j0 + kStep < je) load(j0 + kStep);
#pragma unroll
        for (int h = 0; h < kStep / 16; h++) {
            const int chunk = h * 2 + (lane >> 5);
            bf16x8 fp[2];
#pragma unroll
            for (int q = 0; q < 2; q++) fp[q] = *reinterpret_cast<const bf16x8*>(ldp_ + at_coords(wk + q * 32 + (lane & 31), chunk));
#pragma unroll
            for (int u = TERMS - 1; u >= 0; u--)
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const bf16x8 fc = *reinterpret_cast<const bf16x8*>(ldc_[u] + at_rows(wi + i * 32 + (lane & 31), chunk));
#pragma unroll
                    for (int q = 0; q < 2; q++) acc[i][q] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fp[q], fc, acc[i][q], 0, 0, 0);
                }
        }
        __syncthreads();
    }
    // coordinates are the matrix cores' rows: a lane holds runs of 4 consecutive k of one row i
    float* part = a.part + blockIdx.y * (a.m * a.ldp);
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const uint64_t r = i0 + wi + i * 32 + (lane & 31);
        if (r >= a.m) continue;
#pragma unroll
        for (int q = 0; q < 2; q++)
#pragma unroll
            for (int g = 0; g < 4; g++) {
                const uint64_t k = k0 + wk + q * 32 + g * 8 + (lane >> 5) * 4;
                if (k < a.ldp) *reinterpret_cast<f32x4*>(part + r * a.ldp + k) = f32x4{acc[i][q][g * 4], acc[i][q][g * 4 + 1], acc[i][q][g * 4 + 2], acc[i][q][g * 4 + 3]};
            }
    }
}

// the slices' sums in order
template <int TYPE>
__global__ void __launch_bounds__(256) grad_join_kernel(const float* __restrict__ part, uint32_t slices, uint64_t m, uint64_t dim, uint64_t ldp, typename Elem<TYPE>::T* __restrict__ dx,
                                                        uint64_t lddx) {
    const uint64_t quads = ldp / 4;
    for (uint64_t u = blockIdx.x * 256ull + threadIdx.x; u < m * quads; u += gridDim.x * 256ull) {
        const uint64_t i = u / quads, k = (u - i * quads) * 4;
        f32x4 s = {0.f, 0.f, 0.f, 0.f};
        for (uint32_t q = 0; q < slices; q++) s += *reinterpret_cast<const f32x4*>(part + (q * m + i) * ldp + k);
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (k + e < dim) dx[i * lddx + k + e] = (typename Elem<TYPE>::T)s[e];
    }
}

struct GradPlan {
    uint64_t tiles_m, tiles_k, slices, per_slice, ldp, bytes;
};
// 512 workgroups fill 256 CUs twice; a slice has at least 4 steps
GradPlan grad_plan(uint64_t m, uint64_t n, uint64_t dim) {
    GradPlan g;
    g.tiles_m = (m + kTile - 1) / kTile;
    g.tiles_k = (dim + kTile - 1) / kTile;
    const uint64_t steps = (n + kStep - 1) / kStep, tiles = g.tiles_m * g.tiles_k;
    uint64_t want = tiles >= 512 ? 1 : 512 / tiles;
    if (want > (steps + 3) / 4) want = (steps + 3) / 4;
    if (want < 1) want = 1;
    const uint64_t per = (steps + want - 1) / want;
    g.per_slice = per * kStep;
    g.slices = steps ? (steps + per - 1) / per : 1;
    g.ldp = (dim + 3) / 4 * 4;
    g.bytes = g.slices * m * g.ldp * 4;
    return g;
}

}  // namespace

extern "C" {

int32_t ae_points8_product_grad_work(const ae_points8* p, uint64_t n, uint64_t m, uint32_t dctype, uint64_t* bytes) {
    return guard([&] {
        if (!p || !bytes) fail(AE_ERR_INVALID_ARG, "ae_points8_product_grad_work: null argument");
        check_type(dctype, "ae_points8_product_grad_work");
        if (m > (1ull << 32)) fail(AE_ERR_INVALID_ARG, "ae_points8_product_grad_work: %llu rows are out of range", (unsigned long long)m);
        *bytes = m && n ? grad_plan(m, n, p->dim).bytes : 0;
    });
}

int32_t ae_points8_product_grad(const ae_points8* p, uint64_t first, uint64_t n, const void* d_dc, uint32_t dctype, uint64_t m, uint64_t lddc, void* d_dx, uint32_t xtype, uint64_t lddx,
                                void* d_work, uint64_t work_bytes, void* stream) {
    return guard([&] {
        require_device();
        check_points8(p, first, n, "ae_points8_product_grad");
        check_type(dctype, "ae_points8_product_grad: dc");
        check_type(xtype, "ae_points8_product_grad: dx");
        if (m == 0) return;
        check_rows(d_dx, xtype, m, p->dim, lddx, "ae_points8_product_grad: dx");
        hipStream_t s = (hipStream_t)stream;
        GradPlan g = grad_plan(m, n, p->dim);
        if (n == 0) g.slices = 0, g.bytes = 0;   // the sum over no points
        else check_rows(d_dc, dctype, m, n, lddc, "ae_points8_product_grad: dc");
        if (g.bytes && (!d_work || work_bytes < g.bytes))
            fail(AE_ERR_INVALID_ARG, "ae_points8_product_grad: %llu bytes of scratch are needed, %llu given", (unsigned long long)g.bytes, (unsigned long long)work_bytes);
        check_aligned(d_work, 16, "ae_points8_product_grad: work");
        if (g.tiles_m * g.tiles_k > 0xFFFFFFull) fail(AE_ERR_INVALID_ARG, "ae_points8_product_grad: %llu rows are more than one call takes", (unsigned long long)m);
        if (n) {
            GradArgs a{d_dc, lddc, m, n, p->dim, points8_rows(p, first, n), g.per_slice, (float*)d_work, g.ldp};
            by_type(dctype, [&](auto ty) {
                hipLaunchKernelGGL((grad_tile_kernel<decltype(ty)::value>), dim3((unsigned)(g.tiles_m * g.tiles_k), (unsigned)g.slices), dim3(256), 0, s, a, (uint32_t)g.tiles_k,
                                   vector_rows(d_dc, dctype, lddc));
            });
            check_launch("points8_product_grad");
        }
        by_type(xtype, [&](auto ty) {
            constexpr int TYPE = decltype(ty)::value;
            hipLaunchKernelGGL((grad_join_kernel<TYPE>), dim3(grid_cap(m * g.ldp / 4, 256)), dim3(256), 0, s, (const float*)d_work, (uint32_t)g.slices, m, p->dim, g.ldp,
                               static_cast<typename Elem<TYPE>::T*>(d_dx), lddx);
        });
        check_launch("points8_grad_join");
    });
}

}  // extern "C"
