// teacher.hip -- cross entropy of logits against a teacher's top list, and its gradient.
//
// A row's loss needs max s and sum exp((s - max) / T) over its cols logits, k of the logits themselves, and the list; the gradient is
// g P q_v everywhere and g (P q_v - p) at the k listed columns.  Two floating point operations and an exponential per logit: bound by HBM.
#include "points8.h"

#include <cfloat>

using namespace ae;

namespace {

constexpr uint32_t kMaxList = 1024;
constexpr uint64_t kHeld = 65536;   // logits of a row that one workgroup holds in registers
constexpr uint64_t kLong = 16384;   // logits of a row from which slices of it are worth their launches
constexpr float kLog2e = 1.4426950408889634f;

struct TeacherList {
    const uint32_t* idx;
    const float* val;
    uint64_t ldk;
    uint32_t k, kind;
};

// maximum and sum of the running softmax: sum of exp2((s - m) c), m the largest logit so far
struct Running {
    float m = -INFINITY, s = 0.f;
    __device__ __forceinline__ void join(float m2, float s2, float c) {
        const float big = fmaxf(m, m2), safe = big == -INFINITY ? 0.f : big;
        s = s * __builtin_amdgcn_exp2f((m - safe) * c) + s2 * __builtin_amdgcn_exp2f((m2 - safe) * c);
        m = big;
    }
};

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    return v;
}
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int o = 32; o; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
    return v;
}

// A row's list in LDS: columns (0xFFFFFFFF: empty), probabilities, their sums over equal columns, the listed logits
struct ListLds {
    uint32_t* col;
    float *p, *sum, *logit;
    __device__ ListLds(void* lds, uint32_t k) {
        const uint32_t k4 = (k + 3) / 4 * 4;
        col = static_cast<uint32_t*>(lds);
        p = reinterpret_cast<float*>(col + k4);
        sum = p + k4;
        logit = sum + k4;
    }
};
inline unsigned list_lds(uint32_t k) { return (k + 3) / 4 * 4 * 16; }

// One wave takes in a row's list (columns outside the row are left empty and make the row's sum NaN).  Returns sum p, and in `plogp` sum p ln p where
// it is wanted.  Logarithms and exponentials in 32 bits, sums of them in 64.
__device__ __forceinline__ double take_list(const TeacherList& t, uint64_t r, uint64_t cols, float temperature, const ListLds& l, bool want_log, double& plogp) {
    const int lane = threadIdx.x & 63;
    const uint32_t* idx = t.idx + r * t.ldk;
    const float* val = t.val + r * t.ldk;
    double p_sum = 0., pl = 0.;
    bool outside = false;
    float big = -INFINITY, lnz = 0.f;
    double over_z = 0.;
    if (t.kind == AE_TEACHER_LOGITS) {
        double z = 0.;
        for (uint32_t j = lane; j < t.k; j += 64)
            if (idx[j] != 0xFFFFFFFFu) big = fmaxf(big, val[j]);
        big = wave_max(big);
        const float safe = big == -INFINITY ? 0.f : big;
        for (uint32_t j = lane; j < t.k; j += 64)
            if (idx[j] != 0xFFFFFFFFu) z += (double)expf((val[j] - safe) / temperature);   // (NaN and +inf make the row NaN)
        z = wave_sum(z);
        over_z = z != 0. ? 1. / z : 0.;
        lnz = logf((float)z);
        big = safe;
    }
    const uint32_t k4 = (t.k + 3) / 4 * 4;
    for (uint32_t j = lane; j < k4; j += 64) {
        const uint32_t v = j < t.k ? idx[j] : 0xFFFFFFFFu;
        double p = 0.;
        float lnp = 0.f;
        if (v != 0xFFFFFFFFu) {
            if (t.kind == AE_TEACHER_PROBA) {
                p = (double)val[j];
                if (want_log) lnp = logf(val[j]);
            } else {
                const float d = (val[j] - big) / temperature;
                p = (double)expf(d) * over_z;
                lnp = d - lnz;
            }
            if (v >= cols) outside = true;
        }
        l.col[j] = v < cols ? v : 0xFFFFFFFFu;
        l.p[j] = (float)p;
        p_sum += p;
        if (p != 0.) pl += p * (double)lnp;
    }
    p_sum = wave_sum(p_sum);
    plogp = want_log ? wave_sum(pl) : 0.;
    return __ballot(outside) ? (double)__uint_as_float(0x7FC00000u) : p_sum;
}
// the sums over equal columns, in the order of the list, for entries j = first, first + step ...
__device__ __forceinline__ void add_equal(const ListLds& l, uint32_t k, uint32_t first, uint32_t step) {
    for (uint32_t j = first; j < k; j += step) {
        const uint32_t v = l.col[j];
        float s = 0.f;
        for (uint32_t o = 0; o < k; o += 4) {
            const uint4 c = *reinterpret_cast<const uint4*>(l.col + o);
            const float4 p = *reinterpret_cast<const float4*>(l.p + o);
            s += c.x == v ? p.x : 0.f;
            s += c.y == v ? p.y : 0.f;
            s += c.z == v ? p.z : 0.f;
            s += c.w == v ? p.w : 0.f;
        }
        l.sum[j] = s;
    }
}

// Elements of a row in pieces of 16 bytes; `count` of the piece's exist
template <int TYPE> constexpr int piece_len() { return 16 / (int)sizeof(typename Elem<TYPE>::T); }
template <int TYPE>
__device__ __forceinline__ Piece load_piece(const typename Elem<TYPE>::T* p, int64_t count) {
    using T = typename Elem<TYPE>::T;
    constexpr int W = piece_len<TYPE>();
    if (count >= W) return *reinterpret_cast<const Piece*>(p);
    using V = __attribute__((ext_vector_type(W))) T;
    V v;
#pragma unroll
    for (int t = 0; t < W; t++) v[t] = t < count ? p[t] : (T)-INFINITY;   // (an exponential of 0, never the largest)
    return __builtin_bit_cast(Piece, v);
}
template <int TYPE>
__device__ __forceinline__ void store_piece(typename Elem<TYPE>::T* p, int64_t count, const float (&x)[16 / sizeof(typename Elem<TYPE>::T)]) {
    using T = typename Elem<TYPE>::T;
    constexpr int W = piece_len<TYPE>();
    using V = __attribute__((ext_vector_type(W))) T;
    V v;
#pragma unroll
    for (int t = 0; t < W; t++) v[t] = (T)x[t];
    if (count >= W) *reinterpret_cast<Piece*>(p) = __builtin_bit_cast(Piece, v);
    else {
#pragma unroll
        for (int t = 0; t < W; t++)
            if (t < count) p[t] = v[t];
    }
}

// largest and sum of exponentials of elements [b, e) of a row, the wave's share of the workgroup's THREADS
template <int TYPE, int THREADS>
__device__ __forceinline__ Running run_over(const typename Elem<TYPE>::T* row, uint64_t b, uint64_t e, float c) {
    constexpr int W = piece_len<TYPE>();
    using V = __attribute__((ext_vector_type(W))) typename Elem<TYPE>::T;
    Running run;
    for (uint64_t v0 = b + (uint64_t)threadIdx.x * W; v0 < e; v0 += THREADS * W) {
        const V v = __builtin_bit_cast(V, load_piece<TYPE>(row + v0, (int64_t)(e - v0)));
        float big = -INFINITY, s = 0.f;
#pragma unroll
        for (int t = 0; t < W; t++) big = fmaxf(big, (float)v[t]);
        const float safe = big == -INFINITY ? 0.f : big;
#pragma unroll
        for (int t = 0; t < W; t++) s += __builtin_amdgcn_exp2f(((float)v[t] - safe) * c);
        run.join(big, s, c);
    }
#pragma unroll
    for (int o = 32; o; o >>= 1) {
        const float m2 = __shfl_xor(run.m, o), s2 = __shfl_xor(run.s, o);
        run.join(m2, s2, c);
    }
    return run;
}
// a running softmax as the row's statistics
__device__ __forceinline__ void stats_of(const Running& run, float& m, float& lnsum) {
    m = run.s != run.s ? run.s : run.m;   // NaN: a NaN or +inf among the logits
    lnsum = m == -INFINITY ? 0.f : (float)log((double)run.s);
}
// the loss, by the wave that took the list
__device__ __forceinline__ float loss_of(const ListLds& l, uint32_t k, double p_sum, double plogp, float m, float lnsum, float w, float temperature) {
    double cross = 0.;
    if (m != -INFINITY)
        for (uint32_t j = threadIdx.x & 63; j < k; j += 64)
            if (l.p[j] != 0.f) cross += (double)l.p[j] * (((double)l.logit[j] - (double)m) / (double)temperature - (double)lnsum);
    cross = wave_sum(cross);
    return m == -INFINITY ? 0.f : (p_sum != p_sum || m != m) ? __uint_as_float(0x7FC00000u) : (float)((double)w * (plogp - cross));
}
// the gradient of one logit, without the list's part
struct Slope {
    float g, p_sum, m, lift, c;
    bool out;
    __device__ Slope(float w, float temperature, double p, float m_, float lnsum)
        : g(w / temperature), p_sum((float)p), m(m_), lift(-lnsum * kLog2e), c(kLog2e / temperature), out(m_ == -INFINITY) {}
    __device__ __forceinline__ float at(float v, float p) const { return out ? 0.f : g * (p_sum * __builtin_amdgcn_exp2f((v - m) * c + lift) - p); }
};

// One workgroup of THREADS per row: HELD pieces of 16 bytes a thread hold the whole row in registers, it is read once, whatever is made of it.  (Of f32 rows
// beyond 32 768 logits, 1024 threads with 16 pieces, 36 registers a thread go to scratch: 300 x 60 000 takes 46 to 52 us for loss and gradient, 28 by its bytes.)
// LOSS: statistics, loss and (grad not null) the gradient; otherwise the gradient from kept statistics.
template <int TYPE, int THREADS, int HELD, bool LOSS>
__global__ void __launch_bounds__(THREADS) teacher_row_kernel(const typename Elem<TYPE>::T* logits_, uint64_t cols, uint64_t ld, TeacherList list, float temperature,
                                                              const float* __restrict__ weight, float* __restrict__ loss, float* stats, typename Elem<TYPE>::T* grad_, uint64_t ldg) {
    using T = typename Elem<TYPE>::T;
    constexpr int W = piece_len<TYPE>(), WAVES = THREADS / 64;
    using V = __attribute__((ext_vector_type(W))) T;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    __shared__ float sm[WAVES], ss[WAVES];
    __shared__ double sd;
    const uint64_t r = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const ListLds l(lds, list.k);
    const T* row = logits_ + r * ld;
    T* grow = grad_ ? grad_ + r * ldg : nullptr;
    const float w = weight ? weight[r] : 1.f;
    const float c = kLog2e / temperature;
    if (w == 0.f || (!LOSS && stats[2 * r] == -INFINITY)) {   // the row is left out
        if constexpr (LOSS) {
            if (tid == 0) { stats[2 * r] = -INFINITY; stats[2 * r + 1] = 0.f; loss[r] = 0.f; }
        }
        if (grow) {
            const float zero[W] = {};
            for (uint64_t v0 = (uint64_t)tid * W; v0 < cols; v0 += THREADS * W) store_piece<TYPE>(grow + v0, (int64_t)(cols - v0), zero);
        }
        return;
    }
    // The list, by the first wave, before its part of the row: the two would not fit in the registers together, and the other waves and rows of the
    // CU go on meanwhile.
    double p_sum = 0., plogp = 0.;
    if (wave == 0) {
        p_sum = take_list(list, r, cols, temperature, l, LOSS, plogp);
        for (uint32_t j = lane; j < list.k; j += 64) l.logit[j] = l.col[j] == 0xFFFFFFFFu ? 0.f : (float)row[l.col[j]];   // (a lane reads back what it wrote)
        if (grow && list.k <= 64) add_equal(l, list.k, lane, 64);
        if (lane == 0) sd = p_sum;
    }
    Piece held[HELD];
#pragma unroll
    for (int q = 0; q < HELD; q++) {
        const int64_t v0 = (int64_t)(q * THREADS + tid) * W, count = (int64_t)cols - v0;
        if (count > 0) held[q] = load_piece<TYPE>(row + v0, count);
        else {
            V none;
#pragma unroll
            for (int t = 0; t < W; t++) none[t] = (T)-INFINITY;
            held[q] = __builtin_bit_cast(Piece, none);
        }
    }
    float m, lnsum;
    if constexpr (LOSS) {
        Running run;   // of the wave, under its own largest
        float big = -INFINITY;
#pragma unroll
        for (int q = 0; q < HELD; q++) {
            const V v = __builtin_bit_cast(V, held[q]);
#pragma unroll
            for (int t = 0; t < W; t++) big = fmaxf(big, (float)v[t]);
        }
        run.m = wave_max(big);
        const float safe = run.m == -INFINITY ? 0.f : run.m;
#pragma unroll
        for (int q = 0; q < HELD; q++) {
            const V v = __builtin_bit_cast(V, held[q]);
#pragma unroll
            for (int t = 0; t < W; t++) run.s += __builtin_amdgcn_exp2f(((float)v[t] - safe) * c);
        }
#pragma unroll
        for (int o = 32; o; o >>= 1) run.s += __shfl_xor(run.s, o);
        if (lane == 0) { sm[wave] = run.m; ss[wave] = run.s; }
        __syncthreads();
        run = Running();
#pragma unroll
        for (int q = 0; q < WAVES; q++) run.join(sm[q], ss[q], c);
        stats_of(run, m, lnsum);
        if (tid == 0) { stats[2 * r] = m; stats[2 * r + 1] = lnsum; }
        if (wave == 0) {
            const float one = loss_of(l, list.k, p_sum, plogp, m, lnsum, w, temperature);
            if (lane == 0) loss[r] = one;
        }
    } else {
        m = stats[2 * r];
        lnsum = stats[2 * r + 1];
        __syncthreads();   // (the list)
    }
    if (!grow) return;
    const Slope slope(w, temperature, sd, m, lnsum);
    // (in place: the listed logits have been taken by the first wave before the barrier)
#pragma unroll
    for (int q = 0; q < HELD; q++) {
        const int64_t v0 = (int64_t)(q * THREADS + tid) * W, count = (int64_t)cols - v0;
        if (count <= 0) continue;
        const V v = __builtin_bit_cast(V, held[q]);
        float x[W];
#pragma unroll
        for (int t = 0; t < W; t++) x[t] = slope.at((float)v[t], 0.f);
        store_piece<TYPE>(grow + v0, count, x);
    }
    if (list.k > 64) {
        add_equal(l, list.k, tid, THREADS);
        __syncthreads();
    }
    // The listed columns again, with their probabilities, each by the wave that wrote it above: the stores of a wave to one address stay in
    // order, nobody waits for them.
    for (uint32_t j = lane; j < list.k; j += 64) {
        const uint32_t v = l.col[j];
        if (v != 0xFFFFFFFFu && (int)(v / W % THREADS / 64) == wave) grow[v] = (T)slope.at(l.logit[j], l.sum[j]);
    }
}

// Long rows in slices: (row, slice) per workgroup.
constexpr int kSliceThreads = 512;
template <int TYPE>
__global__ void __launch_bounds__(kSliceThreads) teacher_part_kernel(const typename Elem<TYPE>::T* __restrict__ logits, uint64_t cols, uint64_t ld, float temperature,
                                                                     const float* __restrict__ weight, uint32_t slices, uint64_t slice_len, float* __restrict__ part) {
    __shared__ float sm[kSliceThreads / 64], ss[kSliceThreads / 64];
    const uint64_t r = blockIdx.x / slices, b = (blockIdx.x - r * slices) * slice_len, e = min(cols, b + slice_len);
    if (weight && weight[r] == 0.f) return;
    const float c = kLog2e / temperature;
    Running run = run_over<TYPE, kSliceThreads>(logits + r * ld, b, e, c);
    if ((threadIdx.x & 63) == 0) { sm[threadIdx.x >> 6] = run.m; ss[threadIdx.x >> 6] = run.s; }
    __syncthreads();
    if (threadIdx.x) return;
    for (int q = 1; q < kSliceThreads / 64; q++) run.join(sm[q], ss[q], c);
    part[2 * blockIdx.x] = run.m;
    part[2 * blockIdx.x + 1] = run.s;
}
// the slices of a row joined in order: statistics and loss; one wave per row
template <int TYPE>
__global__ void __launch_bounds__(64) teacher_join_kernel(const typename Elem<TYPE>::T* __restrict__ logits, uint64_t cols, uint64_t ld, TeacherList list, float temperature,
                                                          const float* __restrict__ weight, uint32_t slices, const float* __restrict__ part, float* __restrict__ loss,
                                                          float* __restrict__ stats) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const uint64_t r = blockIdx.x;
    const uint32_t lane = threadIdx.x;
    const float w = weight ? weight[r] : 1.f;
    float m = -INFINITY, lnsum = 0.f, one = 0.f;
    // (the slices' sums are on their way while the list is taken)
    const float c = kLog2e / temperature;
    Running run;
    if (w != 0.f)
        for (uint32_t q = lane; q < slices; q += 64) run.join(part[2 * (r * slices + q)], part[2 * (r * slices + q) + 1], c);
    if (w != 0.f) {
        const ListLds l(lds, list.k);
        double plogp;
        const double p_sum = take_list(list, r, cols, temperature, l, true, plogp);
        for (uint32_t j = lane; j < list.k; j += 64) l.logit[j] = l.col[j] == 0xFFFFFFFFu ? 0.f : (float)logits[r * ld + l.col[j]];
#pragma unroll
        for (int o = 32; o; o >>= 1) {
            const float m2 = __shfl_xor(run.m, o), s2 = __shfl_xor(run.s, o);
            run.join(m2, s2, c);
        }
        stats_of(run, m, lnsum);
        one = loss_of(l, list.k, p_sum, plogp, m, lnsum, w, temperature);
    }
    if (lane == 0) { stats[2 * r] = m; stats[2 * r + 1] = lnsum; loss[r] = one; }
}
template <int TYPE>
__global__ void __launch_bounds__(kSliceThreads) teacher_slope_kernel(const typename Elem<TYPE>::T* logits_, uint64_t cols, uint64_t ld, TeacherList list, float temperature,
                                                                      const float* __restrict__ weight, uint32_t slices, uint64_t slice_len, const float* __restrict__ stats,
                                                                      typename Elem<TYPE>::T* grad_, uint64_t ldg) {
    using T = typename Elem<TYPE>::T;
    constexpr int W = piece_len<TYPE>();
    using V = __attribute__((ext_vector_type(W))) T;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    __shared__ double sd;
    const uint64_t r = blockIdx.x / slices, b = (blockIdx.x - r * slices) * slice_len, e = min(cols, b + slice_len);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const T* row = logits_ + r * ld;
    T* grow = grad_ + r * ldg;
    const float w = weight ? weight[r] : 1.f, m = w == 0.f ? -INFINITY : stats[2 * r];
    const ListLds l(lds, list.k);
    if (m != -INFINITY) {
        if (wave == 0) {
            double unused;
            const double p_sum = take_list(list, r, cols, temperature, l, false, unused);
            // (in place: only this slice's own logits, which nobody else writes)
            for (uint32_t j = lane; j < list.k; j += 64) l.logit[j] = l.col[j] >= b && l.col[j] < e ? (float)row[l.col[j]] : 0.f;
            if (lane == 0) sd = p_sum;
        }
        __syncthreads();
        add_equal(l, list.k, tid, kSliceThreads);
        __syncthreads();
    }
    const Slope slope(w, temperature, m != -INFINITY ? sd : 0., m, stats[2 * r + 1]);
    for (uint64_t v0 = b + (uint64_t)tid * W; v0 < e; v0 += kSliceThreads * W) {
        float x[W] = {};
        if (!slope.out) {
            const V v = __builtin_bit_cast(V, load_piece<TYPE>(row + v0, (int64_t)(e - v0)));
#pragma unroll
            for (int t = 0; t < W; t++) x[t] = slope.at((float)v[t], 0.f);
        }
        store_piece<TYPE>(grow + v0, (int64_t)(e - v0), x);
    }
    if (slope.out) return;
    for (uint32_t j = lane; j < list.k; j += 64) {   // (as above)
        const uint32_t v = l.col[j];
        if (v >= b && v < e && (int)((v - b) / W % kSliceThreads / 64) == wave) grow[v] = (T)slope.at(l.logit[j], l.sum[j]);
    }
}

void check_size(uint64_t rows, uint64_t cols, const char* what) {
    if (cols == 0 || cols >= 0xFFFFFFFFull) fail(AE_ERR_INVALID_ARG, "%s: %llu columns are out of range", what, (unsigned long long)cols);
    const uint64_t threads = cols <= 8192 ? 256 : (cols + 8191) / 8192 * 512;   // the most that a row gets; a launch has fewer than 2^32
    if (rows > 0xFFFFFFull || rows * threads > 0xFFFFFFFFull)
        fail(AE_ERR_INVALID_ARG, "%s: %llu rows of %llu columns are more than one call takes", what, (unsigned long long)rows, (unsigned long long)cols);
}
void check_list(const uint32_t* d_idx, const float* d_list, uint32_t k, uint64_t ldk, uint32_t kind, float temperature, uint64_t rows, uint64_t cols, const char* what) {
    if (!d_idx || !d_list) fail(AE_ERR_INVALID_ARG, "%s: the list is NULL", what);
    if (k == 0 || k > kMaxList) fail(AE_ERR_INVALID_ARG, "%s: a list of %u entries is not in [1, %u]", what, k, kMaxList);
    if (ldk < k) fail(AE_ERR_INVALID_ARG, "%s: the list's stride is shorter than the list", what);
    if (kind > AE_TEACHER_LOGITS) fail(AE_ERR_INVALID_ARG, "%s: unknown kind of list %u", what, kind);
    if (ldk > (1ull << 40) / rows) fail(AE_ERR_INVALID_ARG, "%s: %llu lists of stride %llu are out of range", what, (unsigned long long)rows, (unsigned long long)ldk);
    if (!(temperature >= FLT_MIN) || !(temperature < INFINITY)) fail(AE_ERR_INVALID_ARG, "%s: the temperature has to be positive, finite and not denormal", what);
    check_size(rows, cols, what);
    check_aligned(d_idx, 4, what);
    check_aligned(d_list, 4, what);
}

// slices of 8192 logits or more, of few rows as many as give each CU four workgroups
struct Slices {
    uint32_t count;
    uint64_t len;
};
Slices slices_of(uint64_t rows, uint64_t cols) {
    uint64_t want = rows >= 1024 ? 1 : (1024 + rows - 1) / rows;
    const uint64_t most = (cols + 8191) / 8192;
    if (want > most) want = most;
    Slices s;
    s.len = ((cols + want - 1) / want + 7) / 8 * 8;
    s.count = (uint32_t)((cols + s.len - 1) / s.len);
    return s;
}

struct Call {
    const void* logits;
    uint32_t type;
    uint64_t rows, cols, ld;
    TeacherList list;
    float temperature;
    const float* weight;
    float *loss, *stats;
    void* grad;
    uint64_t ldg;
    hipStream_t s;
};

template <bool LOSS>
void launch_rows(const Call& a) {
    by_type(a.type, [&](auto ty) {
        constexpr int TYPE = decltype(ty)::value;
        using T = typename Elem<TYPE>::T;
        auto go = [&](auto kernel, unsigned threads) {
            hipLaunchKernelGGL(kernel, dim3((unsigned)a.rows), dim3(threads), list_lds(a.list.k), a.s, static_cast<const T*>(a.logits), a.cols, a.ld, a.list, a.temperature, a.weight,
                               a.loss, a.stats, static_cast<T*>(a.grad), a.ldg);
        };
        // as few threads as hold the row: the more rows a CU has at work, the better their phases mix
        const uint64_t pieces = (a.cols + piece_len<TYPE>() - 1) / piece_len<TYPE>();
        if (pieces <= 64) go(teacher_row_kernel<TYPE, 64, 1, LOSS>, 64);
        else if (pieces <= 256) go(teacher_row_kernel<TYPE, 256, 1, LOSS>, 256);
        else if (pieces <= 512) go(teacher_row_kernel<TYPE, 256, 2, LOSS>, 256);
        else if (pieces <= 1024) go(teacher_row_kernel<TYPE, 256, 4, LOSS>, 256);
        else if (pieces <= 2048) go(teacher_row_kernel<TYPE, 256, 8, LOSS>, 256);
        else if constexpr (LOSS || TYPE == AE_TYPE_F32) {   // (the gradient alone has slices from kLong columns on)
            if (pieces <= 4096) go(teacher_row_kernel<TYPE, 512, 8, LOSS>, 512);
            else if constexpr (LOSS) {
                if (pieces <= 8192) go(teacher_row_kernel<TYPE, 1024, 8, true>, 1024);
                else if constexpr (TYPE == AE_TYPE_F32) go(teacher_row_kernel<TYPE, 1024, 16, true>, 1024);
            }
        }
    });
    check_launch("teacher_row");
}
void launch_slopes(const Call& a, const Slices& sl) {
    by_type(a.type, [&](auto ty) {
        constexpr int TYPE = decltype(ty)::value;
        using T = typename Elem<TYPE>::T;
        hipLaunchKernelGGL((teacher_slope_kernel<TYPE>), dim3((unsigned)(a.rows * sl.count)), dim3(kSliceThreads), list_lds(a.list.k), a.s, static_cast<const T*>(a.logits), a.cols, a.ld,
                           a.list, a.temperature, a.weight, sl.count, sl.len, a.stats, static_cast<T*>(a.grad), a.ldg);
    });
    check_launch("teacher_slope");
}
void launch_slices(const Call& a, const Slices& sl, float* part) {
    by_type(a.type, [&](auto ty) {
        constexpr int TYPE = decltype(ty)::value;
        using T = typename Elem<TYPE>::T;
        const T* logits = static_cast<const T*>(a.logits);
        hipLaunchKernelGGL((teacher_part_kernel<TYPE>), dim3((unsigned)(a.rows * sl.count)), dim3(kSliceThreads), 0, a.s, logits, a.cols, a.ld, a.temperature, a.weight, sl.count, sl.len, part);
        hipLaunchKernelGGL((teacher_join_kernel<TYPE>), dim3((unsigned)a.rows), dim3(64), list_lds(a.list.k), a.s, logits, a.cols, a.ld, a.list, a.temperature, a.weight, sl.count,
                           (const float*)part, a.loss, a.stats);
    });
    check_launch("teacher_part");
    if (a.grad) launch_slopes(a, sl);
}

}  // namespace

extern "C" {

int32_t ae_teacher_loss_work(uint64_t rows, uint64_t cols, uint64_t* bytes) {
    return guard([&] {
        if (!bytes) fail(AE_ERR_INVALID_ARG, "ae_teacher_loss_work: bytes is NULL");
        check_size(rows, cols, "ae_teacher_loss_work");
        *bytes = rows && cols >= kLong ? rows * slices_of(rows, cols).count * 8 : 0;
    });
}

int32_t ae_teacher_loss(const void* d_logits, uint32_t type, uint64_t rows, uint64_t cols, uint64_t ld, const uint32_t* d_idx, const float* d_list, uint32_t k, uint64_t ldk,
                        uint32_t kind, float temperature, const float* d_row_weight, float* d_loss, float* d_stats, void* d_grad, uint64_t ldg, void* d_work,
                        uint64_t work_bytes, void* stream) {
    return guard([&] {
        check_type(type, "ae_teacher_loss");
        if (rows == 0) return;
        check_list(d_idx, d_list, k, ldk, kind, temperature, rows, cols, "ae_teacher_loss");
        check_rows(d_logits, type, rows, cols, ld, "ae_teacher_loss: logits");
        if (d_grad) check_rows(d_grad, type, rows, cols, ldg, "ae_teacher_loss: grad");
        if (d_grad == d_logits && ldg != ld) fail(AE_ERR_INVALID_ARG, "ae_teacher_loss: a gradient in place has the logits' stride");
        if (!d_loss || !d_stats) fail(AE_ERR_INVALID_ARG, "ae_teacher_loss: loss or stats is NULL");
        check_aligned(d_loss, 4, "ae_teacher_loss: loss");
        check_aligned(d_stats, 4, "ae_teacher_loss: stats");
        check_aligned(d_row_weight, 4, "ae_teacher_loss: row weights");
        require_device();
        const Call a{d_logits, type, rows, cols, ld, TeacherList{d_idx, d_list, ldk, k, kind}, temperature, d_row_weight, d_loss, d_stats, d_grad, ldg, (hipStream_t)stream};
        // Where the gradient is wanted too the row held in registers saves a read (300 x 60 000 of f32: 52 us either way, 600: 88 against 115).  For the loss
        // alone a workgroup a row leaves CUs idle between rows: from 32 MB on slices win (300 x 60 000 of f32: 23 against 33 us; of bf16, 36 MB: 16 against
        // 19; below that their second launch costs 4 us).
        if (cols <= kHeld && (d_grad || cols < kLong || rows * cols * type_size(type) < 32 << 20)) return launch_rows<true>(a);
        const Slices sl = slices_of(rows, cols);
        const uint64_t need = rows * sl.count * 8;
        if (!d_work || work_bytes < need) fail(AE_ERR_INVALID_ARG, "ae_teacher_loss: %llu bytes of scratch are needed, %llu given", (unsigned long long)need, (unsigned long long)work_bytes);
        check_aligned(d_work, 16, "ae_teacher_loss: work");
        launch_slices(a, sl, static_cast<float*>(d_work));
    });
}

int32_t ae_teacher_grad(const void* d_logits, uint32_t type, uint64_t rows, uint64_t cols, uint64_t ld, const float* d_stats, const uint32_t* d_idx, const float* d_list, uint32_t k,
                        uint64_t ldk, uint32_t kind, float temperature, const float* d_dloss, void* d_grad, uint64_t ldg, void* stream) {
    return guard([&] {
        check_type(type, "ae_teacher_grad");
        if (rows == 0) return;
        check_list(d_idx, d_list, k, ldk, kind, temperature, rows, cols, "ae_teacher_grad");
        check_rows(d_logits, type, rows, cols, ld, "ae_teacher_grad: logits");
        check_rows(d_grad, type, rows, cols, ldg, "ae_teacher_grad: grad");
        if (d_grad == d_logits && ldg != ld) fail(AE_ERR_INVALID_ARG, "ae_teacher_grad: a gradient in place has the logits' stride");
        if (!d_stats) fail(AE_ERR_INVALID_ARG, "ae_teacher_grad: stats is NULL");
        check_aligned(d_stats, 4, "ae_teacher_grad: stats");
        check_aligned(d_dloss, 4, "ae_teacher_grad: dloss");
        require_device();
        const Call a{d_logits, type, rows, cols, ld, TeacherList{d_idx, d_list, ldk, k, kind}, temperature, d_dloss, nullptr, const_cast<float*>(d_stats), d_grad, ldg, (hipStream_t)stream};
        // nothing to hold: slices from 16 384 logits on (300 x 60 000 of f32: 33 against 37 us, 2000 x 16 384: 49 against 60)
        if (cols < kLong) launch_rows<false>(a);
        else launch_slopes(a, slices_of(rows, cols));
    });
}

}  // extern "C"
