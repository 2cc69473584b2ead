// points8_grad.hip -- the gradient of the 8-bit product to its rows: dx[i][k] = sum_j dc[i][j] * p_j[k].
//
// The sum runs over the points, and a point's scales change with j: they cannot go into the matrix cores' scale operand, which belongs to a
// run of the summed axis.  But code * 2^e is exact in bf16, and dc of f32 (f16) is the sum of three (two) bf16 numbers, so bf16 matrix cores
// compute the product of the values themselves with f32 sums: nothing is rounded before the result.
//
// A workgroup owns 64 or 128 rows x 128 coordinates (one block: one scale byte per point) and walks a slice of the points 64 at a time.  Few rows leave
// few tiles: the points are split into slices whose sums are joined in order; one slice writes the result itself.
#include "points8.h"

using namespace ae;

namespace {

constexpr uint32_t kPast = 0x3FFF0000u;      // the ranges of a tile's rows of dc and of a slice's codes do not reach this far
constexpr uint32_t kOutside = 0x40000000u;   // an offset outside every buffer's range (dc's rows of a tile, a slice's codes: less than 1 GiB)

template <int TYPE> constexpr int terms_of() { return TYPE == AE_TYPE_F32 ? 3 : TYPE == AE_TYPE_F16 ? 2 : 1; }

// The 64 points of a step are 8 chunks of 8.  Lane group g takes chunk part(h, g) of half h, of dc and of the coordinates alike: with these and
// the places below the 16 lanes that LDS serves at a time (0-3, 12-15 and 20-27 of a half wave, then the others) touch all 64 banks once.
__device__ __forceinline__ int part(int h, int g) { return ((h ? 0x4352 : 0x6170) >> (g * 4)) & 7; }
// a coordinate's chunks of 16 bytes: written four coordinates apart, read coordinate after coordinate
__device__ __forceinline__ int at_coords(int k, int chunk) { return k * 128 + ((chunk ^ ((k >> 2) & 7) ^ ((k & 2) << 1)) << 4); }
// a row of dc: 8 (f32: 16) pieces of 16 bytes
template <int PIECES> __device__ __forceinline__ int turn(int r) { return PIECES == 8 ? (r >> 1) & 7 : r & 15; }

// Eight values as the sum of TERMS bf16 numbers, each the upper half of what the ones before it leave: exact (8 + 8 + 8 bits of f32's 24, 8 + 8 of f16's
// 11) apart from what lies below bf16's range.  An infinity leaves nothing; what a NaN leaves is NaN, whatever its upper half says.
template <int TYPE>
__device__ __forceinline__ void split8(const typename Elem<TYPE>::T (&v)[8], bf16x8 (&t)[terms_of<TYPE>()]) {
    constexpr int TERMS = terms_of<TYPE>();
    if constexpr (TERMS == 1) {
#pragma unroll
        for (int e = 0; e < 8; e++) t[0][e] = (__bf16)v[e];
    } else {
        uint32_t r[8];
#pragma unroll
        for (int e = 0; e < 8; e++) r[e] = __float_as_uint((float)v[e]);
#pragma unroll
        for (int q = 0; q < TERMS; q++) {
            u32x4 w;
#pragma unroll
            for (int e = 0; e < 4; e++) w[e] = __builtin_amdgcn_perm(r[2 * e + 1], r[2 * e], 0x07060302u);
            t[q] = __builtin_bit_cast(bf16x8, w);
            if (q + 1 == TERMS) break;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float x = __uint_as_float(r[e]), left = x - __uint_as_float(r[e] & 0xFFFF0000u);
                r[e] = __float_as_uint(q == 0 && __builtin_amdgcn_classf(x, 0x204) ? 0.f : left);   // (0x204: the infinities)
            }
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
    void* dx;             // one slice: its sums are the result, rounded here
    uint32_t xtype;
    uint64_t lddx;
};

// sums of 4 coordinates from k on, of row r
__device__ __forceinline__ void put(const GradArgs& a, uint32_t slice, uint64_t r, uint64_t k, f32x4 v) {
    if (a.slices > 1) {
        if (k < a.ldp) *reinterpret_cast<f32x4*>(a.part + (slice * a.m + r) * a.ldp + k) = v;
        return;
    }
#pragma unroll
    for (int e = 0; e < 4; e++) {
        if (k + e >= a.dim) return;
        const uint64_t at = r * a.lddx + k + e;
        if (a.xtype == AE_TYPE_F32) static_cast<float*>(a.dx)[at] = v[e];
        else if (a.xtype == AE_TYPE_BF16) static_cast<__bf16*>(a.dx)[at] = (__bf16)v[e];
        else static_cast<_Float16*>(a.dx)[at] = (_Float16)v[e];
    }
}

// The slice and tile of a workgroup.  Workgroups go to the 8 XCDs in turn, each with an L2 of its own: an XCD owns a run of slices, all tiles of
// a slice one after the other, so that dc and the points are fetched from memory once and shared there.
__device__ __forceinline__ bool place_of(const GradArgs& a, uint32_t& slice, uint32_t& ti, uint32_t& tk) {
    const uint32_t total = a.tiles * a.slices, each = total / 8, more = total % 8, xcd = blockIdx.x % 8, at = blockIdx.x / 8;
    if (at >= each + (xcd < more ? 1 : 0)) return false;
    const uint32_t id = xcd * each + min(xcd, more) + at;
    slice = __builtin_amdgcn_readfirstlane(id / a.tiles);
    const uint32_t tile = id - slice * a.tiles;
    ti = __builtin_amdgcn_readfirstlane(tile / a.tiles_k);
    tk = tile - ti * a.tiles_k;
    return true;
}

// dc of f32 and f16 (and of any type whose rows lie too far apart for 32-bit offsets).  A wave owns 16 FR of
// the rows and all coordinates, so each value of dc is split once.  dc goes to LDS as it is, three steps deep.  (Straight to the lanes that
// multiply it, 16 bytes of 16 rows each, every lane would be an access of its own to the cache.)  The codes are turned on the way to LDS: a thread takes
// 4 coordinates of 8 points, widens them under the products of the step before and writes 8 points of one coordinate as 16 bytes.  One
// barrier a step.  8192 x 8192 x 4096 of f32: 970 TF of the three partial products (of the 1413 that a large bf16 product of the library reaches); 300 x
// 60 000 x 784: 107 us.  What it waits for is LDS: every wave splits the values it takes, and 112 KB move for 128 x 128 x 64.
template <int TYPE, int FR> constexpr int grad_lds() { return 3 * 64 * FR * kStep * (TYPE == AE_TYPE_F32 ? 4 : 2) + 2 * kBlock * 128; }   // 56 or 80 KB: two workgroups a CU

template <int TYPE, int FR, bool VEC>   // VEC: the copies' 32-bit offsets do for dc
__global__ void __launch_bounds__(256, 2) grad_tile_kernel(GradArgs a) {
    using T = typename Elem<TYPE>::T;
    constexpr int TERMS = terms_of<TYPE>(), ROW = kStep * (int)sizeof(T), PIECES = ROW / 16, STAGE = 64 * FR * ROW, COPIES = STAGE / 4096;
    extern __shared__ __attribute__((aligned(128))) uint8_t lds[];   // three stages of dc, two of coordinates
    uint32_t slice, ti, tk;
    if (!place_of(a, slice, ti, tk)) return;
    const uint64_t i0 = (uint64_t)ti * (64 * FR), k0 = (uint64_t)tk * kBlock;
    const uint64_t jb = slice * a.per_slice, je = min(a.n, jb + a.per_slice);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4;
    const int kg = tid & 31, jg = tid >> 5;   // this thread's 4 coordinates and 8 points
    const uint32_t mi = (uint32_t)min((uint64_t)(64 * FR), a.m - i0), points = (uint32_t)(je - jb), steps = (points + kStep - 1) / kStep;
    const int r0 = wave * 16 * FR + (lane & 15);   // this lane's first row of the tile; the others 16 apart
    const T* dc = static_cast<const T*>(a.dc) + i0 * a.lddc + jb;
    // Rows beyond m lie outside the buffer's range, which ends with the last row's last point: dwords that are not wholly inside read as 0, so an odd 16-bit
    // value at the very end is put in by itself in the last step, where what is fetched behind the other rows' last point is cut.  A lane's offsets
    // never change, the step goes into the scalar one, which stays inside the range (steps past the last one fetch the last again, for nobody).
    const uint32_t row_bytes = (uint32_t)a.lddc * (uint32_t)sizeof(T);
    __amdgpu_buffer_rsrc_t rd = __builtin_amdgcn_make_buffer_rsrc((void*)dc, (short)0, VEC ? (int)grad_range(mi, row_bytes, points, sizeof(T)) : 0, 0x00027000);
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
    T final = (T)0.f;     // the last row's last point
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
                        for (int e = 0; e < 8; e++) {
                            const uint32_t j = t * kStep + part(x >> 3, g) * 8 + e;
                            v[e] = j < points ? v[e] : (T)0.f;
                            if constexpr (sizeof(T) == 2) v[e] = j == points - 1 && (uint32_t)(r0 + i * 16) == mi - 1 ? final : v[e];
                        }
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
    if constexpr (VEC && sizeof(T) == 2) final = dc[(mi - 1) * a.lddc + points - 1];
    if (t + 1 < steps) {
        step(t, even, std::false_type{});
        step(t + 1, odd, std::true_type{});
    } else step(t, even, std::true_type{});
    if constexpr (VEC) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // the copies for nobody have ended before the LDS is given back
    // coordinates are the matrix cores' rows: a lane holds runs of 4 consecutive k of its rows
#pragma unroll
    for (int i = 0; i < FR; i++) {
        const uint64_t r = i0 + r0 + i * 16;
        if (r >= a.m) continue;
#pragma unroll
        for (int q = 0; q < 8; q++) put(a, slice, r, k0 + q * 16 + g * 4, acc[i][q]);
    }
}

// dc of bf16, which the matrix cores take as it is.  16 FR rows x 128 coordinates; two waves share the coordinates, two the points of a step.  A lane
// takes 4 coordinates of 8 points, one dword a point: put together by coordinate they are what the matrix cores want of it, with coordinates 4 apart
// in a fragment, so the codes are widened in the registers they are used from, and each wave reads all rows of dc: LDS moves 48 KB for
// 128 x 128 x 64 where the kernel above moves 112 (300 x 60 000 x 784: 47 us against 52, 4096 x 32 768 x 1024: 256 against 303, 1075 TF of the 1413 that a
// large bf16 product of the library reaches).  dc and the codes come by copies to LDS three deep; the codes are read two steps ahead and widened under
// the products, whose waits for one another and for the barrier of a step are what bounds it: the matrix cores are busy for 30 % of the time at 300 x 60 000 x 784.
constexpr int kTurnStage = kStep * 128;   // codes of a step
template <int FR> constexpr int turn_lds() { return 3 * (16 * FR * kStep * 2 + kTurnStage + 1024); }   // 51 or 75 KB for 64 or 128 rows

template <int FR>
__global__ void __launch_bounds__(256, 2) grad_turn_kernel(GradArgs a) {
    constexpr int STAGE = 16 * FR * kStep * 2, CODES = 3 * STAGE, SCALES = CODES + 3 * kTurnStage, COPIES_DC = FR / 2, COPIES = COPIES_DC + 3;
    extern __shared__ __attribute__((aligned(128))) uint8_t lds[];
    uint32_t slice, ti, tk;
    if (!place_of(a, slice, ti, tk)) return;
    const uint64_t i0 = (uint64_t)ti * (16 * FR), k0 = (uint64_t)tk * kBlock;
    const uint64_t jb = slice * a.per_slice, je = min(a.n, jb + a.per_slice);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4;
    const int half = wave >> 1, side = wave & 1, mine = part(half, g);   // of the points, of the coordinates; this lane's 8 points of the step's 64
    const uint32_t mi = (uint32_t)min((uint64_t)(16 * FR), a.m - i0), points = (uint32_t)(je - jb), steps = (points + kStep - 1) / kStep;
    const __bf16* dc = static_cast<const __bf16*>(a.dc) + i0 * a.lddc + jb;
    // ---- the copies.  Ranges and what lies behind the last point: as above
    const uint32_t row_bytes = (uint32_t)a.lddc * 2, stride = (uint32_t)a.p.row_bytes;
    __amdgpu_buffer_rsrc_t rd = __builtin_amdgcn_make_buffer_rsrc((void*)dc, (short)0, (int)grad_range(mi, row_bytes, points, 2), 0x00027000);
    __amdgpu_buffer_rsrc_t rc = __builtin_amdgcn_make_buffer_rsrc((void*)(a.p.codes + jb * stride), (short)0, (int)(points * stride), 0x00027000);
    __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void*)(a.p.scales + tk * a.p.scale_stride + jb), (short)0, (int)(points + 256), 0x00027000);   // (kScaleSlack)
    const int copy_row = wave * 8 + (lane >> 3), copy_piece = (lane & 7) ^ turn<8>(copy_row);
    const uint32_t dc_at = copy_row * row_bytes + copy_piece * 16;
    auto copy_dc = [&](uint32_t step, uint32_t stage) {   // (zeros for a step that does not exist)
#pragma unroll
        for (int q = 0; q < COPIES_DC; q++)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rd, (__attribute__((address_space(3))) void*)(lds + stage * STAGE + (q * 4 + wave) * 1024), 16,
                                                     (int)dc_at, (int)(step < steps ? step * (kStep * 2) + q * 32 * row_bytes : kPast), 0, 0);
    };
    // point p = 8 c + e at LDS row 8 c + (e ^ bit 1 of c), its halves of 64 bytes exchanged where c is odd: the four groups of lanes, whose c differ in both
    // bits, read from all banks
    const uint32_t code_k = (uint32_t)k0 + (((lane & 7) ^ ((wave & 1) << 2)) << 4);
    const uint32_t code_at = (uint32_t)(wave * 8 + ((lane >> 3) ^ (wave >> 1))) * stride + (code_k < stride ? code_k : kOutside);
    auto copy_codes = [&](uint32_t step, uint32_t stage) {
#pragma unroll
        for (int q = 0; q < 2; q++)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rc, (__attribute__((address_space(3))) void*)(lds + CODES + stage * kTurnStage + (q * 4 + wave) * 1024), 16,
                                                     (int)code_at, (int)(step < steps ? (step * kStep + q * 32) * stride : kPast), 0, 0);
        // (each wave its own, or the waves would not wait for the same number of copies)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void*)(lds + SCALES + (stage * 4 + wave) * 256), 4, lane * 4, (int)(step < steps ? step * kStep : 0), 0, 0);
    };
    // ---- the codes: from LDS, then two points at a time to bf16
    using bf16x2 = __attribute__((ext_vector_type(2))) __bf16;
    const uint32_t from_even = mine * 1024 + ((mine >> 1) & 1) * 128 + ((side ^ (mine & 1)) << 6) + (lane & 15) * 4, from_odd = from_even - ((mine >> 1) & 1) * 256;
    uint32_t code[8];
    u32x2 bytes;
    auto read_codes = [&](uint32_t stage) {
        const uint8_t* at = lds + CODES + stage * kTurnStage;
#pragma unroll
        for (int e = 0; e < 8; e++) code[e] = *reinterpret_cast<const uint32_t*>(at + (e & 1 ? from_odd : from_even) + e * 128);
        bytes = *reinterpret_cast<const u32x2*>(lds + SCALES + (stage * 4 + wave) * 256 + mine * 8);
    };
    u32x4 frag[2][4];   // [step's parity][coordinate 4 (lane & 15) + f]: 8 points
    auto widen = [&](int pair, u32x4 (&to)[4]) {
        uint32_t w[2][2];
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const int at = pair * 2 + e;
            const float scale = __uint_as_float(((bytes[at >> 2] >> ((at & 3) * 8)) & 255u) << 23);
            w[e][0] = __builtin_bit_cast(uint32_t, (bf16x2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(code[at], scale, false));
            w[e][1] = __builtin_bit_cast(uint32_t, (bf16x2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(code[at], scale, true));
        }
#pragma unroll
        for (int f = 0; f < 4; f++) to[f][pair] = __builtin_amdgcn_perm(w[1][f >> 1], w[0][f >> 1], f & 1 ? 0x07060302u : 0x05040100u);
    };
    // ---- the rows: fragment by fragment, read two ahead
    const uint32_t row_at = (lane & 15) * 128 + ((mine ^ turn<8>(lane & 15)) << 4);
    u32x4 rows[4];
    f32x4 acc[FR][4];
#pragma unroll
    for (int i = 0; i < FR; i++)
#pragma unroll
        for (int f = 0; f < 4; f++) acc[i][f] = f32x4{0.f, 0.f, 0.f, 0.f};
    uint32_t stage = 0;             // of this step
    __bf16 final = (__bf16)0.f;   // the last row's last point
    auto step = [&](uint32_t t, auto which, auto last) {
        constexpr int S = decltype(which)::value;
        constexpr bool LAST = decltype(last)::value;
        const uint32_t next = stage == 2 ? 0 : stage + 1;
#pragma unroll
        for (int i = 0; i < FR; i++) {
            if (!LAST && i == FR - 1) read_codes(next == 2 ? 0 : next + 1);
            if (!LAST && i == FR - 2) {
                // The step's rows and the next one's codes have been read by everybody; the next one's rows and the codes after them have to be there,
                // the copies of one step may be on their way.
                asm volatile("s_waitcnt vmcnt(%0)" ::"n"(COPIES) : "memory");
                __builtin_amdgcn_s_waitcnt(0xC07F);   // lgkmcnt(0)
                __builtin_amdgcn_s_barrier();
                asm volatile("" ::: "memory");
                copy_dc(t + 3, stage);
                copy_codes(t + 4, next);
            }
            if (i + 2 < FR) rows[(S * FR + i + 2) & 3] = *reinterpret_cast<const u32x4*>(lds + stage * STAGE + row_at + (i + 2) * 2048);
            else if (!LAST) rows[(S * FR + i + 2) & 3] = *reinterpret_cast<const u32x4*>(lds + next * STAGE + row_at + (i + 2 - FR) * 2048);
            __builtin_amdgcn_sched_barrier(0);
            bf16x8 v = __builtin_bit_cast(bf16x8, rows[(S * FR + i) & 3]);
            if constexpr (LAST) {   // cut what lies behind the last point
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const uint32_t j = t * kStep + mine * 8 + e;
                    v[e] = j < points ? v[e] : (__bf16)0.f;
                    v[e] = j == points - 1 && (uint32_t)(i * 16 + (lane & 15)) == mi - 1 ? final : v[e];
                }
            }
#pragma unroll
            for (int f = 0; f < 4; f++) acc[i][f] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, frag[S][f]), v, acc[i][f], 0, 0, 0);
            if (!LAST) {
#pragma unroll
                for (int pair = 0; pair < 4; pair++)
                    if (i == pair * (FR - 1) / 4) widen(pair, frag[S ^ 1]);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        stage = next;
    };
    uint32_t t = 0u - (steps & 1);   // an odd number of steps begins with one of zeros
    copy_codes(t, 0);
    copy_dc(t, 0);
    copy_codes(t + 1, 1);
    copy_dc(t + 1, 1);
    copy_codes(t + 2, 2);
    copy_dc(t + 2, 2);
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(3 + 2 * COPIES_DC) : "memory");   // (of the second step's rows and behind)
    __syncthreads();
    read_codes(0);
#pragma unroll
    for (int pair = 0; pair < 4; pair++) widen(pair, frag[0]);
    rows[0] = *reinterpret_cast<const u32x4*>(lds + row_at);
    rows[1] = *reinterpret_cast<const u32x4*>(lds + row_at + 2048);
    __builtin_amdgcn_s_waitcnt(0xC07F);
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    copy_codes(t + 3, 0);
    read_codes(1);
    constexpr std::integral_constant<int, 0> even;
    constexpr std::integral_constant<int, 1> odd;
    for (; t + 2 != steps; t += 2) {
        step(t, even, std::false_type{});
        step(t + 1, odd, std::false_type{});
    }
    final = dc[(mi - 1) * a.lddc + points - 1];
    step(t, even, std::false_type{});
    step(t + 1, odd, std::true_type{});
    // ---- the two halves of the points, through LDS (the copies for nobody have ended first)
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    f32x4* meet = reinterpret_cast<f32x4*>(lds) + side * (FR * 4 * 64) + lane;
    if (half) {
#pragma unroll
        for (int i = 0; i < FR; i++)
#pragma unroll
            for (int f = 0; f < 4; f++) meet[(i * 4 + f) * 64] = acc[i][f];
    }
    __syncthreads();
    if (!half) {
#pragma unroll
        for (int i = 0; i < FR; i++)
#pragma unroll
            for (int f = 0; f < 4; f++) acc[i][f] += meet[(i * 4 + f) * 64];
    }
    __syncthreads();
    // ---- out, row by row: lane (i, g) holds rows i of the fragments, coordinates 16 g + 4 e + f of the wave's 64 in acc[.][f][e]
    constexpr int OUT = kBlock * 4 + 16;   // (neighbours start 4 banks apart)
    if (!half) {
        uint8_t* to = lds + (lane & 15) * OUT + side * 256 + g * 64;
#pragma unroll
        for (int i = 0; i < FR; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) *reinterpret_cast<f32x4*>(to + i * 16 * OUT + e * 16) = f32x4{acc[i][0][e], acc[i][1][e], acc[i][2][e], acc[i][3][e]};
    }
    __syncthreads();
#pragma unroll 1
    for (uint32_t r = tid >> 5; r < mi; r += 8) put(a, slice, i0 + r, k0 + (tid & 31) * 4, *reinterpret_cast<const f32x4*>(lds + r * OUT + (tid & 31) * 16));
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
#pragma unroll 8
        for (uint32_t q = b; q < e; q++) s += *reinterpret_cast<const f32x4*>(from + q * (m * ldp));
    }
    if constexpr (GROUPS > 1) {
        sum[threadIdx.x] = s;
        __syncthreads();
        if (group) return;
#pragma unroll 4
        for (int g = 1; g < GROUPS; g++) s += sum[g * RUNS + threadIdx.x];
    }
    if (u >= m * quads) return;
    const uint64_t i = u / quads, k = (u - i * quads) * 4;
#pragma unroll
    for (int t = 0; t < 4; t++)
        if (k + t < dim) dx[i * lddx + k + t] = (typename Elem<TYPE>::T)s[t];
}

template <int TYPE, int FR>
void launch_grad(const GradArgs& a, bool vec, unsigned grid, hipStream_t s) {
    if (!vec) hipLaunchKernelGGL((grad_tile_kernel<TYPE, FR, false>), dim3(grid), dim3(256), (grad_lds<TYPE, FR>()), s, a);
    else if constexpr (TYPE == AE_TYPE_BF16) hipLaunchKernelGGL((grad_turn_kernel<4 * FR>), dim3(grid), dim3(256), (turn_lds<4 * FR>()), s, a);
    else hipLaunchKernelGGL((grad_tile_kernel<TYPE, FR, true>), dim3(grid), dim3(256), (grad_lds<TYPE, FR>()), s, a);
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
        const unsigned groups = join_groups(g.slices);
        const uint64_t runs = m * (g.ldp / 4);
        if (g.tiles_m * g.tiles_k * g.slices > 0x3FFFFFull || runs * groups > 0xFFFF0000ull)
            fail(AE_ERR_INVALID_ARG, "ae_points8_product_grad: %llu rows are more than one call takes", (unsigned long long)m);
        if (n) {
            const uint64_t tiles = g.tiles_m * g.tiles_k;
            GradArgs a{d_dc, lddc, m, n, p->dim, points8_rows(p, first, n), g.per_slice, (float*)d_work, g.ldp, (uint32_t)g.tiles_k, (uint32_t)tiles, (uint32_t)g.slices, d_dx, xtype, lddx};
            const unsigned grid = (unsigned)((tiles * g.slices + 7) / 8 * 8);
            const bool vec = lddc * type_size(dctype) < 0x3FFF0000ull / (64 * g.fr);
            by_type(dctype, [&](auto ty) {
                constexpr int TYPE = decltype(ty)::value;
                if (g.fr == 1) launch_grad<TYPE, 1>(a, vec, grid, s);
                else if constexpr (TYPE != AE_TYPE_F32) launch_grad<TYPE, 2>(a, vec, grid, s);
            });
            check_launch("points8_product_grad");
            if (g.slices == 1) return;
        }
        by_type(xtype, [&](auto ty) {
            constexpr int TYPE = decltype(ty)::value;
            auto go = [&](auto kernel) {
                hipLaunchKernelGGL(kernel, dim3(blocks_for(runs * groups, 256)), dim3(256), 0, s, (const float*)d_work, (uint32_t)g.slices, m, p->dim, g.ldp,
                                   static_cast<typename Elem<TYPE>::T*>(d_dx), lddx);
            };
            if (groups == 64) go(grad_join_kernel<TYPE, 64>);
            else if (groups == 16) go(grad_join_kernel<TYPE, 16>);
            else if (groups == 4) go(grad_join_kernel<TYPE, 4>);
            else go(grad_join_kernel<TYPE, 1>);
        });
        check_launch("points8_grad_join");
    });
}

}  // extern "C"
