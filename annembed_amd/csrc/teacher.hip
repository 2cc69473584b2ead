// teacher.hip -- cross entropy of logits against a teacher's top list, and its gradient.
//
// A row's loss needs max s and sum exp((s - max) / T) over its cols logits, k of the logits themselves, and the list; the gradient is
// g P q_v everywhere and g (P q_v - p) at the k listed columns.  Two floating point operations and an exponential per logit: bound by HBM.
#include "points8.h"

using namespace ae;

namespace {

constexpr uint32_t kMaxList = 1024;
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

// One wave takes in a row's list: columns to li, probabilities to lp (0 for empty places and, with the row's sum made NaN, for columns
// outside the row).  Returns sum p, and in `plogp` sum p ln p.
__device__ __forceinline__ double take_list(const TeacherList& t, uint64_t r, uint64_t cols, float temperature, uint32_t* li, float* lp, double& plogp) {
    const int lane = threadIdx.x & 63;
    const uint32_t* idx = t.idx + r * t.ldk;
    const float* val = t.val + r * t.ldk;
    double p_sum = 0., pl = 0.;
    bool outside = false;
    float big = -INFINITY;
    double lnz = 0., z = 0.;
    if (t.kind == AE_TEACHER_LOGITS) {
        for (uint32_t j = lane; j < t.k; j += 64)
            if (idx[j] != 0xFFFFFFFFu) { const float v = val[j]; big = v != v ? v : fmaxf(big, v); }
        const bool nan = __ballot(big != big) != 0;
        big = nan ? __uint_as_float(0x7FC00000u) : wave_max(big);
        for (uint32_t j = lane; j < t.k; j += 64)
            if (idx[j] != 0xFFFFFFFFu && big != -INFINITY) z += exp(((double)val[j] - (double)big) / (double)temperature);
        z = wave_sum(z);
        lnz = log(z);
    }
    for (uint32_t j = lane; j < t.k; j += 64) {
        const uint32_t v = idx[j];
        double p = 0., lnp = 0.;
        if (v != 0xFFFFFFFFu) {
            if (t.kind == AE_TEACHER_PROBA) {
                p = (double)val[j];
                lnp = log(p);
            } else if (big != -INFINITY) {
                lnp = ((double)val[j] - (double)big) / (double)temperature - lnz;
                p = exp(lnp);
            }
            if (v >= cols) outside = true;
        }
        li[j] = v < cols ? v : 0xFFFFFFFFu;
        lp[j] = (float)p;
        p_sum += p;
        if (p != 0.) pl += p * lnp;
    }
    p_sum = wave_sum(p_sum);
    plogp = wave_sum(pl);
    return __ballot(outside) ? (double)__uint_as_float(0x7FC00000u) : p_sum;
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

// One workgroup of THREADS per row.  HELD pieces of 16 bytes a thread hold the whole row in registers: it is read once, whatever is made of it.
// HELD 0: longer rows are read again for the gradient, mostly from the caches.  LOSS: statistics, loss and (grad not null) the gradient;
// otherwise the gradient from kept statistics.
template <int TYPE, int THREADS, int HELD, bool LOSS>
__global__ void __launch_bounds__(THREADS) teacher_row_kernel(const typename Elem<TYPE>::T* logits_, uint64_t cols, uint64_t ld, TeacherList list, float temperature,
                                                              const float* __restrict__ weight, float* __restrict__ loss, float* stats, typename Elem<TYPE>::T* grad_, uint64_t ldg) {
    using T = typename Elem<TYPE>::T;
    constexpr int W = piece_len<TYPE>(), WAVES = THREADS / 64;
    using V = __attribute__((ext_vector_type(W))) T;
    __shared__ uint32_t li[kMaxList];
    __shared__ float lp[kMaxList], ls[kMaxList];
    __shared__ float sm[WAVES], ss[WAVES];
    __shared__ double sd[2];
    const uint64_t r = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const T* row = logits_ + r * ld;
    T* grow = grad_ ? grad_ + r * ldg : nullptr;
    const float w = weight ? weight[r] : 1.f;
    const float c = kLog2e / temperature;
    const bool counts = w != 0.f && (LOSS || stats[2 * r] != -INFINITY);
    if (!counts) {   // the row is left out
        if constexpr (LOSS) {
            if (tid == 0) { stats[2 * r] = -INFINITY; stats[2 * r + 1] = 0.f; loss[r] = 0.f; }
        }
        if (grow) {
            const float zero[W] = {};
            for (uint64_t v0 = (uint64_t)tid * W; v0 < cols; v0 += THREADS * W) store_piece<TYPE>(grow + v0, (int64_t)(cols - v0), zero);
        }
        return;
    }
    // The list, by the first wave, before its part of the row: its 64-bit logarithms and the row would not fit in the registers together, and the other
    // waves and rows of the CU go on meanwhile.
    double plogp = 0.;
    if (wave == 0) {
        const double p = take_list(list, r, cols, temperature, li, lp, plogp);
        for (uint32_t j = lane; j < list.k; j += 64) ls[j] = li[j] == 0xFFFFFFFFu ? 0.f : (float)row[li[j]];   // (a lane reads back what it wrote)
        if (lane == 0) sd[0] = p;
    }
    Piece held[HELD ? HELD : 1];
    if constexpr (HELD) {
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
    }
    float m, lnsum;
    if constexpr (LOSS) {
        Running run;
        if constexpr (HELD) {
            // largest and sum of the wave
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
        } else {
            for (uint64_t v0 = (uint64_t)tid * W; v0 < cols; v0 += THREADS * W) {
                const V v = __builtin_bit_cast(V, load_piece<TYPE>(row + v0, (int64_t)(cols - v0)));
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
        }
        if (lane == 0) { sm[wave] = run.m; ss[wave] = run.s; }
        __syncthreads();
        run = Running();
#pragma unroll
        for (int q = 0; q < WAVES; q++) run.join(sm[q], ss[q], c);
        m = run.s != run.s ? run.s : run.m;   // NaN: a NaN or +inf among the logits
        lnsum = m == -INFINITY ? 0.f : (float)log((double)run.s);
        if (tid == 0) { stats[2 * r] = m; stats[2 * r + 1] = lnsum; }
    } else {
        m = stats[2 * r];
        lnsum = stats[2 * r + 1];
        __syncthreads();   // (the list)
    }
    const bool out = LOSS && m == -INFINITY;   // nothing but -inf
    if constexpr (LOSS) {
        if (wave == 0) {
            double cross = 0.;
            if (!out)
                for (uint32_t j = lane; j < list.k; j += 64)
                    if (lp[j] != 0.f) cross += (double)lp[j] * (((double)ls[j] - (double)m) / (double)temperature - (double)lnsum);
            cross = wave_sum(cross);
            if (lane == 0) loss[r] = out ? 0.f : (sd[0] != sd[0] || m != m) ? __uint_as_float(0x7FC00000u) : (float)((double)w * (plogp - cross));
        }
    }
    if (!grow) return;
    const float g = out ? 0.f : w / temperature, p_sum = out ? 0.f : (float)sd[0], lift = -lnsum * kLog2e, base = out ? 0.f : m;
    auto gradient = [&](float v) { return out ? 0.f : g * (p_sum * __builtin_amdgcn_exp2f((v - base) * c + lift)); };
    // in place: the listed logits have been taken by the first wave before the barrier
    if constexpr (HELD) {
#pragma unroll
        for (int q = 0; q < HELD; q++) {
            const int64_t v0 = (int64_t)(q * THREADS + tid) * W, count = (int64_t)cols - v0;
            if (count <= 0) continue;
            const V v = __builtin_bit_cast(V, held[q]);
            float x[W];
#pragma unroll
            for (int t = 0; t < W; t++) x[t] = gradient((float)v[t]);
            store_piece<TYPE>(grow + v0, count, x);
        }
    } else {
        for (uint64_t v0 = (uint64_t)tid * W; v0 < cols; v0 += THREADS * W) {
            const V v = __builtin_bit_cast(V, load_piece<TYPE>(row + v0, (int64_t)(cols - v0)));
            float x[W];
#pragma unroll
            for (int t = 0; t < W; t++) x[t] = gradient((float)v[t]);
            store_piece<TYPE>(grow + v0, (int64_t)(cols - v0), x);
        }
    }
    if (out) return;
    // The listed columns again, with their probabilities, each by the wave that wrote it above: the stores of a wave to one address stay in
    // order, nobody waits.
    for (uint32_t j = lane; j < list.k; j += 64) {
        const uint32_t v = li[j];
        if (v == 0xFFFFFFFFu || (int)(v / W % THREADS / 64) != wave) continue;
        float p = 0.f;
        for (uint32_t o = 0; o < list.k; o++) p += li[o] == v ? lp[o] : 0.f;   // equal columns: the same sum in the same order
        grow[v] = (T)(g * (p_sum * __builtin_amdgcn_exp2f((ls[j] - base) * c + lift) - p));
    }
}

void check_list(const uint32_t* d_idx, const float* d_list, uint32_t k, uint64_t ldk, uint32_t kind, float temperature, uint64_t rows, uint64_t cols, const char* what) {
    if (!d_idx || !d_list) fail(AE_ERR_INVALID_ARG, "%s: the list is NULL", what);
    if (k == 0 || k > kMaxList) fail(AE_ERR_INVALID_ARG, "%s: a list of %u entries is not in [1, %u]", what, k, kMaxList);
    if (ldk < k) fail(AE_ERR_INVALID_ARG, "%s: the list's stride is shorter than the list", what);
    if (kind > AE_TEACHER_LOGITS) fail(AE_ERR_INVALID_ARG, "%s: unknown kind of list %u", what, kind);
    if (!(temperature > 0.f) || !(temperature < INFINITY)) fail(AE_ERR_INVALID_ARG, "%s: the temperature has to be positive", what);
    if (cols == 0 || cols >= 0xFFFFFFFFull) fail(AE_ERR_INVALID_ARG, "%s: %llu columns are out of range", what, (unsigned long long)cols);
    if (rows > 0xFFFFFFull) fail(AE_ERR_INVALID_ARG, "%s: %llu rows are more than one call takes (2^24 - 1)", what, (unsigned long long)rows);
    check_aligned(d_idx, 4, what);
    check_aligned(d_list, 4, what);
}

template <bool LOSS>
void launch_rows(const void* d_logits, uint32_t type, uint64_t rows, uint64_t cols, uint64_t ld, const TeacherList& list, float temperature, const float* weight, float* loss,
                 float* stats, void* d_grad, uint64_t ldg, hipStream_t s) {
    by_type(type, [&](auto ty) {
        constexpr int TYPE = decltype(ty)::value;
        using T = typename Elem<TYPE>::T;
        auto go = [&](auto kernel, unsigned threads) {
            hipLaunchKernelGGL(kernel, dim3((unsigned)rows), dim3(threads), 0, s, static_cast<const T*>(d_logits), cols, ld, list, temperature, weight, loss, stats,
                               static_cast<T*>(d_grad), ldg);
        };
        // as few threads as hold the row: the more rows a CU has at work, the better their phases mix
        const uint64_t pieces = (cols + piece_len<TYPE>() - 1) / piece_len<TYPE>();
        if (pieces <= 64) go(teacher_row_kernel<TYPE, 64, 1, LOSS>, 64);
        else if (pieces <= 256) go(teacher_row_kernel<TYPE, 256, 1, LOSS>, 256);
        else if (pieces <= 512) go(teacher_row_kernel<TYPE, 256, 2, LOSS>, 256);
        else if (pieces <= 1024) go(teacher_row_kernel<TYPE, 256, 4, LOSS>, 256);
        else if (pieces <= 2048) go(teacher_row_kernel<TYPE, 256, 8, LOSS>, 256);
        else if (pieces <= 4096) go(teacher_row_kernel<TYPE, 512, 8, LOSS>, 512);
        else if (pieces <= 8192) go(teacher_row_kernel<TYPE, 1024, 8, LOSS>, 1024);
        else if (TYPE == AE_TYPE_F32 && pieces <= 16384) go(teacher_row_kernel<TYPE, 1024, TYPE == AE_TYPE_F32 ? 16 : 8, LOSS>, 1024);
        else go(teacher_row_kernel<TYPE, 1024, 0, LOSS>, 1024);
    });
    check_launch("teacher_row");
}

}  // namespace

extern "C" {

int32_t ae_teacher_loss_work(uint64_t rows, uint64_t cols, uint64_t* bytes) {
    return guard([&] {
        if (!bytes) fail(AE_ERR_INVALID_ARG, "ae_teacher_loss_work: bytes is NULL");
        *bytes = 0;
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
        require_device();
        launch_rows<true>(d_logits, type, rows, cols, ld, TeacherList{d_idx, d_list, ldk, k, kind}, temperature, d_row_weight, d_loss, d_stats, d_grad, ldg, (hipStream_t)stream);
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
        require_device();
        launch_rows<false>(d_logits, type, rows, cols, ld, TeacherList{d_idx, d_list, ldk, k, kind}, temperature, d_dloss, nullptr, const_cast<float*>(d_stats), d_grad, ldg,
                           (hipStream_t)stream);
    });
}

}  // extern "C"
