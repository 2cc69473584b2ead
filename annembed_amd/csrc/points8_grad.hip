// points8_grad.hip -- the gradient of the 8-bit product to its rows: dx[i][k] = sum_j dc[i][j] * p_j[k].
//
// The sum runs over the points, and a point's scales change with j: they cannot go into the matrix cores' scale operand, which belongs to a
// run of the summed axis.  But code * 2^e is exact in bf16, and dc of f32 (f16) is the sum of three (two) bf16 numbers, so bf16 matrix cores
// compute the product of the values themselves with f32 sums: nothing is rounded before the result.
//
// A workgroup owns 64 FR rows x 128 coordinates (one block: one scale byte per point) and walks a slice of the points 64 at a time; a wave owns
// 16 FR of the rows and all coordinates.  dc never touches LDS: a lane's 8 consecutive points of a row are the matrix cores' operand as they
// lie in memory.  The codes are turned on the way to LDS: a thread takes 4 coordinates of 8 points, widens them and writes 8 points of one
// coordinate as 16 bytes.  Both are fetched two steps ahead into the registers that the step frees.  Few rows leave few tiles: the points are
// split into slices whose sums are joined in order.
#include "points8.h"

#include <algorithm>

using namespace ae;

namespace {

constexpr int kStep = 64;    // points per step: 128 bytes of bf16
constexpr uint32_t kOutside = 0x80000000u;   // or-ed into an offset: outside every buffer's range (they span less than 2 GiB)

template <int TYPE> constexpr int terms_of() { return TYPE == AE_TYPE_F32 ? 3 : TYPE == AE_TYPE_F16 ? 2 : 1; }

// a coordinate's 64 points as 8 chunks of 16 bytes; written four coordinates apart, read coordinate after coordinate, both without bank conflicts
__device__ __forceinline__ int at_coords(int k, int chunk) { return k * 128 + ((chunk ^ ((k >> 2) & 7) ^ ((k & 2) << 1)) << 4); }

// eight values as the sum of TERMS bf16 numbers, the first ones cut off (never past the largest bf16): exact apart from what lies below bf16's range
template <int TYPE>
__device__ __forceinline__ void split8(const typename Elem<TYPE>::T (&v)[8], bf16x8 (&t)[terms_of<TYPE>()]) {
    constexpr int TERMS = terms_of<TYPE>();
#pragma unroll
    for (int e = 0; e < 8; e++) {
        if constexpr (TERMS == 1) t[0][e] = (__bf16)v[e];
        else {
            float r = (float)v[e];
            const bool finite = (__float_as_uint(r) & 0x7FFFFFFFu) < 0x7F800000u;
#pragma unroll
            for (int q = 0; q + 1 < TERMS; q++) {
                const float cut = __uint_as_float(__float_as_uint(r) & 0xFFFF0000u);
                t[q][e] = finite ? (__bf16)cut : (__bf16)r;
                r = finite ? r - cut : 0.f;
            }
            t[TERMS - 1][e] = (__bf16)r;
        }
    }
}

struct GradArgs {
    const void* dc;
    uint64_t lddc;
    uint64_t m, n, dim;
    Rows8 p;
    uint64_t per_slice;   // points per slice, a multiple of kStep
    float* part;          // [slices][m][ldp]
    uint64_t ldp;
    uint32_t tiles_k, tiles, slices;
};

template <int TYPE, int FR, bool VEC>   // VEC: rows of dc lie on 16 bytes, 64 FR of them and a slice's codes span less than 2 GiB
__global__ void __launch_bounds__(256, FR <= 2 ? 2 : 1) grad_tile_kernel(GradArgs a) {
    using T = typename Elem<TYPE>::T;
    constexpr int TERMS = terms_of<TYPE>(), PIECES = (int)sizeof(T) / 2;   // 16-byte pieces of 8 values
    __shared__ __attribute__((aligned(128))) uint8_t lds[2][kBlock * 128];
    // Workgroups go to the 8 XCDs in turn, each with an L2 of its own: an XCD owns a run of slices, all tiles of a slice one after the other, so
    // that dc and the points are fetched from memory once and shared there.
    const uint32_t total = a.tiles * a.slices, each = total / 8, more = total % 8, xcd = blockIdx.x % 8, at = blockIdx.x / 8;
    if (at >= each + (xcd < more ? 1 : 0)) return;
    const uint32_t id = xcd * each + min(xcd, more) + at, slice = id / a.tiles, tile = id - slice * a.tiles, ti = tile / a.tiles_k, tk = tile - ti * a.tiles_k;
    const uint64_t i0 = (uint64_t)ti * (64 * FR), k0 = (uint64_t)tk * kBlock;
    const uint64_t jb = slice * a.per_slice, je = min(a.n, jb + a.per_slice);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int kg = tid & 31, jg = tid >> 5;   // this thread's 4 coordinates and 8 points
    const uint32_t mi = (uint32_t)min((uint64_t)(64 * FR), a.m - i0), points = (uint32_t)(je - jb), steps = (points + kStep - 1) / kStep;
    const int r0 = wave * 16 * FR + (lane & 15);   // this lane's first row of the tile; the others 16 apart
    const T* dc = static_cast<const T*>(a.dc) + i0 * a.lddc + jb;
    // Rows beyond m and pieces behind the last point lie outside the buffer's range, or are put there.  The piece with the last point is fetched
    // whole -- it lies on 16 bytes, so in one page -- and cut.
    const uint32_t row_bytes = (uint32_t)a.lddc * (uint32_t)sizeof(T);
    __amdgpu_buffer_rsrc_t rd = __builtin_amdgcn_make_buffer_rsrc((void*)dc, (short)0, VEC ? (int)((mi - 1) * row_bytes + (points * (uint32_t)sizeof(T) + 15) / 16 * 16) : 0, 0x00027000);
    __amdgpu_buffer_rsrc_t rc = __builtin_amdgcn_make_buffer_rsrc((void*)(a.p.codes + jb * a.p.row_bytes), (short)0, (int)(points * (uint32_t)a.p.row_bytes), 0x00027000);
    const uint32_t code_at = (uint32_t)k0 + kg * 4;
    const uint8_t* sc = a.p.scales + tk * a.p.scale_stride + jb + jg * 8;
    const uint32_t k_out = code_at < a.p.row_bytes ? 0u : kOutside;
    struct Fragment { u32x4 piece[2][PIECES]; };   // 8 points of a row in each half of the step
    struct Codes { uint32_t code[8]; uint2 bytes; };
    Fragment fa[2][FR];
    Codes fc[2];
    auto load_row = [&](uint32_t step, int i, Fragment& f) {
        const uint32_t r = r0 + i * 16;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const uint32_t j = step * kStep + h * 32 + (lane >> 4) * 8;
            if constexpr (VEC) {
#pragma unroll
                for (int q = 0; q < PIECES; q++) {
                    const uint32_t jq = j + q * (8 / PIECES);
                    f.piece[h][q] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rd, (int)((r * row_bytes + jq * (uint32_t)sizeof(T)) | (jq < points ? 0u : kOutside)), 0, 0));
                }
            } else {
                T v[8];
#pragma unroll
                for (int e = 0; e < 8; e++) v[e] = r < mi && j + e < points ? dc[r * a.lddc + j + e] : (T)0.f;
                __builtin_memcpy(f.piece[h], v, sizeof(v));
            }
        }
    };
    auto load_codes = [&](uint32_t step, Codes& c) {
        const uint32_t j = step * kStep + jg * 8;
#pragma unroll
        for (int e = 0; e < 8; e++) c.code[e] = (uint32_t)__builtin_amdgcn_raw_buffer_load_b32(rc, (int)(((j + e) * (uint32_t)a.p.row_bytes + code_at) | k_out), 0, 0);
        __builtin_memcpy(&c.bytes, sc + min(step, steps) * kStep, 8);   // (bytes of points that do not exist multiply zeros; kScaleSlack)
    };
    auto widen = [&](const Codes& c, uint8_t* to) {
        using bf16x2 = __attribute__((ext_vector_type(2))) __bf16;
        uint32_t wide[8][2];   // [point][coordinates 0, 1 | 2, 3]
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const float scale = __uint_as_float(((e < 4 ? c.bytes.x >> (e * 8) : c.bytes.y >> (e * 8 - 32)) & 255u) << 23);
            wide[e][0] = __builtin_bit_cast(uint32_t, (bf16x2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c.code[e], scale, false));
            wide[e][1] = __builtin_bit_cast(uint32_t, (bf16x2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c.code[e], scale, true));
        }
#pragma unroll
        for (int t = 0; t < 4; t++) {
            u32x4 w;
#pragma unroll
            for (int e = 0; e < 4; e++) w[e] = __builtin_amdgcn_perm(wide[2 * e + 1][t >> 1], wide[2 * e][t >> 1], t & 1 ? 0x07060302u : 0x05040100u);
            *reinterpret_cast<u32x4*>(to + at_coords(kg * 4 + t, jg)) = w;
        }
    };
    f32x4 acc[FR][8];
#pragma unroll
    for (int i = 0; i < FR; i++)
#pragma unroll
        for (int q = 0; q < 8; q++) acc[i][q] = f32x4{0.f, 0.f, 0.f, 0.f};
    auto step = [&](uint32_t t, auto which, auto last) {
        constexpr int S = decltype(which)::value;
        widen(fc[S], lds[S]);
        load_codes(t + 2, fc[S]);
        __syncthreads();   // (the other buffer's readers have passed it too: one barrier a step)
        bf16x8 terms[FR][2][TERMS];
#pragma unroll
        for (int i = 0; i < FR; i++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                T v[8];
                __builtin_memcpy(v, fa[S][i].piece[h], sizeof(v));
                if constexpr (VEC && decltype(last)::value) {   // cut what lies behind the last point
#pragma unroll
                    for (int e = 0; e < 8; e++) v[e] = t * kStep + h * 32 + (lane >> 4) * 8 + e < points ? v[e] : (T)0.f;
                }
                split8<TYPE>(v, terms[i][h]);
            }
        bf16x8 fp[4];   // 16 coordinates x 32 points, read two ahead
        auto read = [&](int x) { fp[x & 3] = *reinterpret_cast<const bf16x8*>(lds[S] + at_coords((x & 7) * 16 + (lane & 15), (x >> 3) * 4 + (lane >> 4))); };
        read(0);
        read(1);
#pragma unroll
        for (int x = 0; x < 16; x++) {
            if (x + 2 < 16) read(x + 2);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < FR; i++)
#pragma unroll
                for (int u = TERMS - 1; u >= 0; u--) acc[i][x & 7] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fp[x & 3], terms[i][x >> 3][u], acc[i][x & 7], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int i = 0; i < FR; i++) load_row(t + 2, i, fa[S][i]);
    };
#pragma unroll
    for (int s = 0; s < 2; s++) {
        load_codes(s, fc[s]);
#pragma unroll
        for (int i = 0; i < FR; i++) load_row(s, i, fa[s][i]);
    }
    constexpr std::integral_constant<int, 0> even;
    constexpr std::integral_constant<int, 1> odd;
    uint32_t t = 0;
    for (; t + 2 < steps; t += 2) {
        step(t, even, std::false_type{});
        step(t + 1, odd, std::false_type{});
    }
    if (t + 1 < steps) {
        step(t, even, std::false_type{});
        step(t + 1, odd, std::true_type{});
    } else step(t, even, std::true_type{});
    // coordinates are the matrix cores' rows: a lane holds runs of 4 consecutive k of its rows
    float* part = a.part + slice * (a.m * a.ldp);
#pragma unroll
    for (int i = 0; i < FR; i++) {
        const uint64_t r = i0 + r0 + i * 16;
        if (r >= a.m) continue;
#pragma unroll
        for (int q = 0; q < 8; q++) {
            const uint64_t k = k0 + q * 16 + (lane >> 4) * 4;
            if (k < a.ldp) *reinterpret_cast<f32x4*>(part + r * a.ldp + k) = acc[i][q];
        }
    }
}

// The slices' sums in order: 256 / GROUPS runs of 4 coordinates a workgroup, GROUPS threads for each, whose shares of the slices are added last.
template <int TYPE, int GROUPS>
__global__ void __launch_bounds__(256) grad_join_kernel(const float* __restrict__ part, uint32_t slices, uint64_t m, uint64_t dim, uint64_t ldp, typename Elem<TYPE>::T* __restrict__ dx,
                                                        uint64_t lddx) {
    constexpr int RUNS = 256 / GROUPS;
    __shared__ f32x4 sum[256];
    const uint64_t quads = ldp / 4, u = blockIdx.x * (uint64_t)RUNS + threadIdx.x % RUNS;
    const uint32_t group = threadIdx.x / RUNS, per = (slices + GROUPS - 1) / GROUPS, b = group * per, e = min(slices, b + per);
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
    if (u < m * quads) {
        const float* from = part + u * 4;
        for (uint32_t q = b; q < e; q++) s += *reinterpret_cast<const f32x4*>(from + q * (m * ldp));
    }
    if constexpr (GROUPS > 1) {
        sum[threadIdx.x] = s;
        __syncthreads();
        if (group) return;
#pragma unroll
        for (int g = 1; g < GROUPS; g++) s += sum[g * RUNS + threadIdx.x];
    }
    if (u >= m * quads) return;
    const uint64_t i = u / quads, k = (u - i * quads) * 4;
#pragma unroll
    for (int t = 0; t < 4; t++)
        if (k + t < dim) dx[i * lddx + k + t] = (typename Elem<TYPE>::T)s[t];
}

constexpr uint32_t kMostRows[3] = {3, 5, 4};   // f32, bf16, f16: what a lane's registers hold

struct GradPlan {
    uint32_t fr;
    uint64_t tiles_m, tiles_k, slices, per_slice, ldp, bytes;
};
GradPlan grad_plan(uint64_t m, uint64_t n, uint64_t dim, uint32_t dctype) {
    GradPlan g;
    const char* v = debug_knob("AE_P8G");
    uint32_t best = 1;
    uint64_t least = ~0ull;
    for (uint32_t fr = 1; fr <= kMostRows[dctype]; fr++) {
        const uint64_t padded = (m + 64 * fr - 1) / (64 * fr) * (64 * fr);
        if (padded <= least) { least = padded; best = fr; }
    }
    g.fr = v ? std::min<uint32_t>(atoi(v), kMostRows[dctype]) : best;
    g.tiles_m = (m + 64 * g.fr - 1) / (64 * g.fr);
    g.tiles_k = (dim + kBlock - 1) / kBlock;
    const uint64_t resident = g.fr <= 2 ? 512 : 256;
    const uint64_t steps = (n + kStep - 1) / kStep, tiles = g.tiles_m * g.tiles_k;
    uint64_t want = tiles >= resident ? 1 : resident / tiles;
    if (want > (steps + 3) / 4) want = (steps + 3) / 4;
    if (want < 1) want = 1;
    const uint64_t per = (steps + want - 1) / want;
    g.per_slice = per * kStep;
    g.slices = steps ? (steps + per - 1) / per : 1;
    g.ldp = (dim + 3) / 4 * 4;
    g.bytes = g.slices * m * g.ldp * 4;
    return g;
}

template <int TYPE, int FR>
void launch_grad(const GradArgs& a, bool vec, unsigned grid, hipStream_t s) {
    if (vec) hipLaunchKernelGGL((grad_tile_kernel<TYPE, FR, true>), dim3(grid), dim3(256), 0, s, a);
    else hipLaunchKernelGGL((grad_tile_kernel<TYPE, FR, false>), dim3(grid), dim3(256), 0, s, a);
}

}  // namespace

extern "C" {

int32_t ae_points8_product_grad_work(const ae_points8* p, uint64_t n, uint64_t m, uint32_t dctype, uint64_t* bytes) {
    return guard([&] {
        if (!p || !bytes) fail(AE_ERR_INVALID_ARG, "ae_points8_product_grad_work: null argument");
        check_type(dctype, "ae_points8_product_grad_work");
        if (m > (1ull << 32)) fail(AE_ERR_INVALID_ARG, "ae_points8_product_grad_work: %llu rows are out of range", (unsigned long long)m);
        *bytes = m && n ? grad_plan(m, n, p->dim, dctype).bytes : 0;
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
        GradPlan g = grad_plan(m, n, p->dim, dctype);
        if (n == 0) g.slices = 0, g.bytes = 0;   // the sum over no points
        else check_rows(d_dc, dctype, m, n, lddc, "ae_points8_product_grad: dc");
        if (g.bytes && (!d_work || work_bytes < g.bytes))
            fail(AE_ERR_INVALID_ARG, "ae_points8_product_grad: %llu bytes of scratch are needed, %llu given", (unsigned long long)g.bytes, (unsigned long long)work_bytes);
        check_aligned(d_work, 16, "ae_points8_product_grad: work");
        if (g.tiles_m * g.tiles_k * g.slices > 0x3FFFFFull) fail(AE_ERR_INVALID_ARG, "ae_points8_product_grad: %llu rows are more than one call takes", (unsigned long long)m);
        if (n) {
            const uint64_t tiles = g.tiles_m * g.tiles_k;
            GradArgs a{d_dc, lddc, m, n, p->dim, points8_rows(p, first, n), g.per_slice, (float*)d_work, g.ldp, (uint32_t)g.tiles_k, (uint32_t)tiles, (uint32_t)g.slices};
            const unsigned grid = (unsigned)((tiles * g.slices + 7) / 8 * 8);
            const bool vec = vector_rows(d_dc, dctype, lddc) && lddc * type_size(dctype) < 0x7FFF0000ull / (64 * g.fr);
            by_type(dctype, [&](auto ty) {
                constexpr int TYPE = decltype(ty)::value;
                switch (g.fr) {
                    case 1: launch_grad<TYPE, 1>(a, vec, grid, s); break;
                    case 2: launch_grad<TYPE, 2>(a, vec, grid, s); break;
                    case 3: launch_grad<TYPE, 3>(a, vec, grid, s); break;
                    case 4: if constexpr (TYPE != AE_TYPE_F32) launch_grad<TYPE, 4>(a, vec, grid, s); break;
                    default: if constexpr (TYPE == AE_TYPE_BF16) launch_grad<TYPE, 5>(a, vec, grid, s); break;
                }
            });
            check_launch("points8_product_grad");
        }
        by_type(xtype, [&](auto ty) {
            constexpr int TYPE = decltype(ty)::value;
            const uint64_t runs = m * (g.ldp / 4);
            auto go = [&](auto kernel, unsigned groups) {
                hipLaunchKernelGGL(kernel, dim3(blocks_for(runs * groups, 256)), dim3(256), 0, s, (const float*)d_work, (uint32_t)g.slices, m, p->dim, g.ldp,
                                   static_cast<typename Elem<TYPE>::T*>(d_dx), lddx);
            };
            if (g.slices >= 64) go(grad_join_kernel<TYPE, 16>, 16);
            else if (g.slices >= 8) go(grad_join_kernel<TYPE, 4>, 4);
            else go(grad_join_kernel<TYPE, 1>, 1);
        });
        check_launch("points8_grad_join");
    });
}

}  // extern "C"
