// points8_grad.hip -- the gradient of the 8-bit product to its rows: dx[i][k] = sum_j dc[i][j] * p_j[k].
//
// The sum runs over the points, and a point's scales change with j: they cannot go into the matrix cores' scale operand, which belongs to a
// run of the summed axis.  But code * 2^e is exact in bf16, and dc of f32 (f16) is the sum of three (two) bf16 numbers, so bf16 matrix cores
// compute the product of the values themselves with f32 sums: nothing is rounded before the result.
//
// A workgroup owns 64 FR rows x 128 coordinates (one block: one scale byte per point) and walks a slice of the points 64 at a time; a wave owns
// 16 FR of the rows and all coordinates.  dc goes to LDS as it is, three steps deep.  (Straight to the lanes that multiply it, 16 bytes of 16
// rows each, every lane would be an access of its own to the cache: 57 us where this takes 4x fewer.)  The codes are turned on the way to LDS:
// a thread takes 4 coordinates of 8 points, widens them under the products of the step before and writes 8 points of one coordinate as 16
// bytes.  One barrier a step.  Few rows leave few tiles: the points are split into slices whose sums are joined in order.
#include "points8.h"

using namespace ae;

namespace {

constexpr int kStep = 64;    // points per step: 128 bytes of bf16
constexpr uint32_t kOutside = 0x40000000u;   // an offset outside every buffer's range (dc's rows of a tile, a slice's codes: less than 1 GiB)

template <int TYPE> constexpr int terms_of() { return TYPE == AE_TYPE_F32 ? 3 : TYPE == AE_TYPE_F16 ? 2 : 1; }

// The 64 points of a step are 8 chunks of 8.  Lane group g takes chunk part(h, g) of half h, of dc and of the coordinates alike: with these and
// the places below the 16 lanes that LDS serves at a time (0-3, 12-15 and 20-27 of a half wave, then the others) touch all 64 banks once.
__device__ __forceinline__ int part(int h, int g) { return ((h ? 0x4352 : 0x6170) >> (g * 4)) & 7; }
// a coordinate's chunks of 16 bytes: written four coordinates apart, read coordinate after coordinate
__device__ __forceinline__ int at_coords(int k, int chunk) { return k * 128 + ((chunk ^ ((k >> 2) & 7) ^ ((k & 2) << 1)) << 4); }
// a row of dc: 8 (f32: 16) pieces of 16 bytes
template <int PIECES> __device__ __forceinline__ int turn(int r) { return PIECES == 8 ? (r >> 1) & 7 : r & 15; }

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

template <int TYPE, int FR> constexpr int grad_lds() { return 3 * 64 * FR * kStep * (TYPE == AE_TYPE_F32 ? 4 : 2) + 2 * kBlock * 128; }   // 56 or 80 KB: two workgroups a CU

template <int TYPE, int FR, bool VEC>   // VEC: the copies' 32-bit offsets and whole pieces do for dc
__global__ void __launch_bounds__(256, 2) grad_tile_kernel(GradArgs a) {
    using T = typename Elem<TYPE>::T;
    constexpr int TERMS = terms_of<TYPE>(), ROW = kStep * (int)sizeof(T), PIECES = ROW / 16, STAGE = 64 * FR * ROW, COPIES = STAGE / 4096;
    extern __shared__ __attribute__((aligned(128))) uint8_t lds[];   // three stages of dc, two of coordinates
    // Workgroups go to the 8 XCDs in turn, each with an L2 of its own: an XCD owns a run of slices, all tiles of a slice one after the other, so
    // that dc and the points are fetched from memory once and shared there.
    const uint32_t total = a.tiles * a.slices, each = total / 8, more = total % 8, xcd = blockIdx.x % 8, at = blockIdx.x / 8;
    if (at >= each + (xcd < more ? 1 : 0)) return;
    const uint32_t id = xcd * each + min(xcd, more) + at, slice = id / a.tiles, tile = id - slice * a.tiles, ti = tile / a.tiles_k, tk = tile - ti * a.tiles_k;
    const uint64_t i0 = (uint64_t)ti * (64 * FR), k0 = (uint64_t)tk * kBlock;
    const uint64_t jb = slice * a.per_slice, je = min(a.n, jb + a.per_slice);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4;
    const int kg = tid & 31, jg = tid >> 5;   // this thread's 4 coordinates and 8 points
    const uint32_t mi = (uint32_t)min((uint64_t)(64 * FR), a.m - i0), points = (uint32_t)(je - jb), steps = (points + kStep - 1) / kStep;
    const int r0 = wave * 16 * FR + (lane & 15);   // this lane's first row of the tile; the others 16 apart
    const T* dc = static_cast<const T*>(a.dc) + i0 * a.lddc + jb;
    // Rows beyond m lie outside the buffer's range, which ends with the dword of the last row's last point (what of a piece lies behind it reads as
    // 0).  A lane's offsets never change, the step goes into the scalar one, which stays inside the range (steps past the last one fetch the last
    // again, for nobody).  What is fetched behind the last point is cut in the last step.
    const uint32_t row_bytes = (uint32_t)a.lddc * (uint32_t)sizeof(T);
    __amdgpu_buffer_rsrc_t rd = __builtin_amdgcn_make_buffer_rsrc((void*)dc, (short)0, VEC ? (int)((mi - 1) * row_bytes + (points * (uint32_t)sizeof(T) + 3) / 4 * 4) : 0, 0x00027000);
    __amdgpu_buffer_rsrc_t rc = __builtin_amdgcn_make_buffer_rsrc((void*)(a.p.codes + jb * a.p.row_bytes), (short)0, (int)(points * (uint32_t)a.p.row_bytes), 0x00027000);
    const uint32_t k_at = (uint32_t)k0 + kg * 4, code_at = (uint32_t)(jg * 8) * (uint32_t)a.p.row_bytes + (k_at < a.p.row_bytes ? k_at : kOutside);
    const uint8_t* sc = a.p.scales + tk * a.p.scale_stride + jb + jg * 8;
    const int copy_row = wave * (64 / PIECES) + lane / PIECES, copy_piece = (lane % PIECES) ^ turn<PIECES>(copy_row);   // (copies are a multiple of 16 rows apart)
    auto copy = [&](uint32_t step, uint32_t stage) {
        step = min(step, steps - 1);
#pragma unroll
        for (int q = 0; q < COPIES; q++) {
            const uint32_t r = q * (256 / PIECES) + copy_row;
            uint8_t* to = lds + stage * STAGE + (q * 4 + wave) * 1024;
            if constexpr (VEC)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(rd, (__attribute__((address_space(3))) void*)to, 16, (int)(r * row_bytes + copy_piece * 16), (int)(step * ROW), 0, 0);
            else {
                constexpr int W = 16 / sizeof(T);
                T v[W];
                const uint32_t j = step * kStep + copy_piece * W;
#pragma unroll
                for (int e = 0; e < W; e++) v[e] = r < mi && j + e < points ? dc[r * a.lddc + j + e] : (T)0.f;
                __builtin_memcpy(to + lane * 16, v, 16);
            }
        }
    };
    struct Codes { uint32_t code[8]; uint2 bytes; };
    Codes fc[2];
    auto load_codes = [&](uint32_t step, Codes& c) {
        step = min(step, steps - 1);
#pragma unroll
        for (int e = 0; e < 8; e++) c.code[e] = (uint32_t)__builtin_amdgcn_raw_buffer_load_b32(rc, (int)(code_at + e * (uint32_t)a.p.row_bytes), (int)(step * kStep * (uint32_t)a.p.row_bytes), 0);
        __builtin_memcpy(&c.bytes, sc + step * kStep, 8);   // (bytes of points that do not exist multiply zeros; kScaleSlack)
    };
    uint8_t* const coords = lds + 3 * STAGE;
    // part 0 ... 7: a point's 4 coordinates as bf16; part 8 ... 11: the 8 points of a coordinate to LDS
    uint32_t wide[8][2];   // [point][coordinates 0, 1 | 2, 3]
    auto widen = [&](int part, const Codes& c, uint8_t* to) {
        using bf16x2 = __attribute__((ext_vector_type(2))) __bf16;
        if (part < 8) {
            const float scale = __uint_as_float(((part < 4 ? c.bytes.x >> (part * 8) : c.bytes.y >> (part * 8 - 32)) & 255u) << 23);
            wide[part][0] = __builtin_bit_cast(uint32_t, (bf16x2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c.code[part], scale, false));
            wide[part][1] = __builtin_bit_cast(uint32_t, (bf16x2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c.code[part], scale, true));
        } else {
            const int t = part - 8;
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
    bf16x8 fp[4];                   // 16 coordinates x 32 points, read two ahead
    u32x4 raw[2][FR][PIECES / 8];   // 8 points of this lane's rows, of both halves
    bf16x8 terms[FR][TERMS];        // of the half at work
    auto read_coords = [&](const uint8_t* from, int x) { fp[x & 3] = *reinterpret_cast<const bf16x8*>(from + at_coords((x & 7) * 16 + (lane & 15), part(x >> 3, g))); };
    auto read_rows = [&](const uint8_t* from, int h) {
#pragma unroll
        for (int i = 0; i < FR; i++)
#pragma unroll
            for (int q = 0; q < PIECES / 8; q++) {
                const int r = r0 + i * 16;
                raw[h][i][q] = *reinterpret_cast<const u32x4*>(from + r * ROW + (((part(h, g) * (PIECES / 8) + q) ^ turn<PIECES>(r)) << 4));
            }
    };
    uint32_t stage = 0;   // of this step's dc
    // A step is 16 parts: 16 coordinates over a half of the points.  Everything is read two parts ahead.  Two parts before its end a step's dc and
    // coordinates have been read by everybody and the next one's have to be there.
    auto step = [&](uint32_t t, auto which, auto last) {
        constexpr int S = decltype(which)::value;
        constexpr bool LAST = decltype(last)::value;
        const uint32_t next = stage == 2 ? 0 : stage + 1;
        if constexpr (!LAST) copy(t + 2, next == 2 ? 0 : next + 1);
#pragma unroll
        for (int x = 0; x < 16; x++) {
            if (!LAST && x == 14) {
                // all has arrived but what this step issued (COPIES copies, 9 loads of codes)
                if constexpr (VEC) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(COPIES + 9) : "memory");
                __builtin_amdgcn_s_waitcnt(0xC07F);   // lgkmcnt(0)
                __builtin_amdgcn_s_barrier();
                asm volatile("" ::: "memory");
            }
            if (x < 14) read_coords(coords + S * (kBlock * 128), x + 2);
            else if (!LAST) read_coords(coords + (S ^ 1) * (kBlock * 128), x - 14);
            if (x == 4) read_rows(lds + stage * STAGE, 1);
            if (!LAST && x == 14) read_rows(lds + next * STAGE, 0);
            __builtin_amdgcn_sched_barrier(0);
            if ((x & 7) == 0) {
#pragma unroll
                for (int i = 0; i < FR; i++) {
                    T v[8];
                    __builtin_memcpy(v, raw[x >> 3][i], sizeof(v));
                    if constexpr (VEC && LAST) {   // cut what lies behind the last point
#pragma unroll
                        for (int e = 0; e < 8; e++) v[e] = t * kStep + part(x >> 3, g) * 8 + e < points ? v[e] : (T)0.f;
                    }
                    split8<TYPE>(v, terms[i]);
                }
            }
#pragma unroll
            for (int i = 0; i < FR; i++)
#pragma unroll
                for (int u = TERMS - 1; u >= 0; u--) acc[i][x & 7] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fp[x & 3], terms[i][u], acc[i][x & 7], 0, 0, 0);
            // under the products: the next step's coordinates
            if (!LAST && x < 12) widen(x, fc[S ^ 1], coords + (S ^ 1) * (kBlock * 128));
            if (!LAST && x == 8) load_codes(t + 3, fc[S ^ 1]);
            __builtin_amdgcn_sched_barrier(0);
        }
        stage = next;
    };
    load_codes(0, fc[0]);
    load_codes(1, fc[1]);
    asm volatile("" ::: "memory");
    copy(0, 0);
    copy(1, 1);
#pragma unroll
    for (int x = 0; x < 12; x++) widen(x, fc[0], coords);
    load_codes(2, fc[0]);
    if constexpr (VEC) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    read_rows(lds, 0);
    read_coords(coords, 0);
    read_coords(coords, 1);
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
    if constexpr (VEC) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // the copies for nobody have ended before the LDS is given back
    // coordinates are the matrix cores' rows: a lane holds runs of 4 consecutive k of its rows
    float* part = a.part + slice * (a.m * a.ldp);
#pragma unroll
    for (int i = 0; i < FR; i++) {
        const uint64_t r = i0 + r0 + i * 16;
        if (r >= a.m) continue;
#pragma unroll
        for (int q = 0; q < 8; q++) {
            const uint64_t k = k0 + q * 16 + g * 4;
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

struct GradPlan {
    uint32_t fr;
    uint64_t tiles_m, tiles_k, slices, per_slice, ldp, bytes;
};
GradPlan grad_plan(uint64_t m, uint64_t n, uint64_t dim, uint32_t dctype) {
    GradPlan g;
    // 128 rows read the points half as often as 64 (300 x 60 000 x 784 of bf16: 52 against 67 us, 1024 rows: 127 against 189); more of them, or 128 of
    // f32, leave one workgroup on a CU, whose waits nothing fills (256 rows: 73 and 135 us; f32, 128 rows: 165 against 116 us)
    g.fr = m > 64 && dctype != AE_TYPE_F32 ? 2 : 1;
    g.tiles_m = (m + 64 * g.fr - 1) / (64 * g.fr);
    g.tiles_k = (dim + kBlock - 1) / kBlock;
    const uint64_t resident = 512;   // two workgroups on each of 256 CUs
    const uint64_t steps = (n + kStep - 1) / kStep, tiles = g.tiles_m * g.tiles_k;
    uint64_t want = tiles >= resident ? 1 : resident / tiles;
    if (want > (steps + 3) / 4) want = (steps + 3) / 4;
    const uint64_t most = 0x3FFF0000ull / points8_row_bytes(dim) / kStep, least_slices = (steps + most - 1) / most;   // a slice's codes: less than 1 GiB
    if (want < least_slices) want = least_slices;
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
    if (vec) hipLaunchKernelGGL((grad_tile_kernel<TYPE, FR, true>), dim3(grid), dim3(256), (grad_lds<TYPE, FR>()), s, a);
    else hipLaunchKernelGGL((grad_tile_kernel<TYPE, FR, false>), dim3(grid), dim3(256), (grad_lds<TYPE, FR>()), s, a);
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
        const unsigned groups = g.slices >= 64 ? 16 : g.slices >= 8 ? 4 : 1;   // (the join's)
        const uint64_t runs = m * (g.ldp / 4);
        if (g.tiles_m * g.tiles_k * g.slices > 0x3FFFFFull || runs * groups > 0xFFFF0000ull)
            fail(AE_ERR_INVALID_ARG, "ae_points8_product_grad: %llu rows are more than one call takes", (unsigned long long)m);
        if (n) {
            const uint64_t tiles = g.tiles_m * g.tiles_k;
            GradArgs a{d_dc, lddc, m, n, p->dim, points8_rows(p, first, n), g.per_slice, (float*)d_work, g.ldp, (uint32_t)g.tiles_k, (uint32_t)tiles, (uint32_t)g.slices};
            const unsigned grid = (unsigned)((tiles * g.slices + 7) / 8 * 8);
            // The copies take 16 bytes at any address and the dwords that the buffer's range holds whole.  The last of an odd number of 16-bit values is the
            // first half of a dword: the range then goes 2 bytes past it, which must not be the next page.
            const uint64_t size = type_size(dctype), end = (uint64_t)(uintptr_t)d_dc + ((m - 1) * lddc + n) * size;
            const bool vec = lddc * size < 0x3FFF0000ull / (64 * g.fr) && (n * size % 4 == 0 || end % 4096 != 0);
            by_type(dctype, [&](auto ty) {
                constexpr int TYPE = decltype(ty)::value;
                if (g.fr == 1) launch_grad<TYPE, 1>(a, vec, grid, s);
                else if constexpr (TYPE != AE_TYPE_F32) launch_grad<TYPE, 2>(a, vec, grid, s);
            });
            check_launch("points8_product_grad");
        }
        by_type(xtype, [&](auto ty) {
            constexpr int TYPE = decltype(ty)::value;
            auto go = [&](auto kernel) {
                hipLaunchKernelGGL(kernel, dim3(blocks_for(runs * groups, 256)), dim3(256), 0, s, (const float*)d_work, (uint32_t)g.slices, m, p->dim, g.ldp,
                                   static_cast<typename Elem<TYPE>::T*>(d_dx), lddx);
            };
            if (groups == 16) go(grad_join_kernel<TYPE, 16>);
            else if (groups == 4) go(grad_join_kernel<TYPE, 4>);
            else go(grad_join_kernel<TYPE, 1>);
        });
        check_launch("points8_grad_join");
    });
}

}  // extern "C"
