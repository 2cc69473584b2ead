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

// One workgroup per row.  LOSS: statistics, loss and (grad not null) the gradient; otherwise the gradient from kept statistics.
template <int TYPE, bool LOSS>
__global__ void __launch_bounds__(256) teacher_row_kernel(const typename Elem<TYPE>::T* __restrict__ logits_, uint64_t cols, uint64_t ld, TeacherList list,
                                                          float temperature, const float* __restrict__ weight, float* __restrict__ loss, float* stats,
                                                          typename Elem<TYPE>::T* grad_, uint64_t ldg) {
    using T = typename Elem<TYPE>::T;
    __shared__ uint32_t li[kMaxList];
    __shared__ float lp[kMaxList];
    __shared__ float ls[kMaxList];
    __shared__ float sm[4], ss[4];
    __shared__ double sd[1];
    const uint64_t r = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const T* row = logits_ + r * ld;
    T* grow = grad_ ? grad_ + r * ldg : nullptr;
    const float w = weight ? weight[r] : 1.f;
    const float c = kLog2e / temperature;
    float m = -INFINITY, lnsum = 0.f;
    if (w != 0.f) {
        if constexpr (LOSS) {
            Running run;
            for (uint64_t v0 = (uint64_t)tid * 8; v0 < cols; v0 += 256 * 8) {
                const int count = (int)min((uint64_t)8, cols - v0);
                float v[8];
                load8<TYPE>(row + v0, count, v);
                float big = -INFINITY;
#pragma unroll
                for (int t = 0; t < 8; t++) {
                    if (t >= count) v[t] = -INFINITY;
                    big = fmaxf(big, v[t]);
                }
                const float safe = big == -INFINITY ? 0.f : big;
                float s = 0.f;
#pragma unroll
                for (int t = 0; t < 8; t++) s += __builtin_amdgcn_exp2f((v[t] - safe) * c);
                run.join(big, s, c);
            }
#pragma unroll
            for (int o = 32; o; o >>= 1) {
                const float m2 = __shfl_xor(run.m, o), s2 = __shfl_xor(run.s, o);
                run.join(m2, s2, c);
            }
            if (lane == 0) { sm[wave] = run.m; ss[wave] = run.s; }
            __syncthreads();
            run = Running();
#pragma unroll
            for (int q = 0; q < 4; q++) run.join(sm[q], ss[q], c);
            m = run.m;
            if (run.s != run.s) m = run.s;   // a NaN or +inf among the logits
            lnsum = m == -INFINITY ? 0.f : (float)log((double)run.s);
        } else {
            m = stats[2 * r];
            lnsum = stats[2 * r + 1];
        }
    }
    const bool out = m == -INFINITY;   // weight 0, or nothing but -inf: the row is left out
    if constexpr (LOSS) {
        if (tid == 0) { stats[2 * r] = m; stats[2 * r + 1] = lnsum; }
    }
    if (!out && wave == 0) {
        double plogp = 0.;
        const double p = take_list(list, r, cols, temperature, li, lp, plogp);
        double cross = 0.;
        for (uint32_t j = lane; j < list.k; j += 64) {   // (a lane reads back what it wrote)
            const uint32_t v = li[j];
            const float s = v == 0xFFFFFFFFu ? 0.f : (float)row[v];
            ls[j] = s;
            if (lp[j] != 0.f) cross += (double)lp[j] * (((double)s - (double)m) / (double)temperature - (double)lnsum);
        }
        cross = wave_sum(cross);
        if (lane == 0) {
            sd[0] = p;
            if constexpr (LOSS) loss[r] = (p != p || m != m) ? __uint_as_float(0x7FC00000u) : (float)((double)w * (plogp - cross));
        }
    }
    if constexpr (LOSS) { if (out && tid == 0) loss[r] = 0.f; }
    if (!grow) return;
    __syncthreads();
    const float g = out ? 0.f : w / temperature;
    const float p_sum = out ? 0.f : (float)sd[0];
    const float lift = -lnsum * kLog2e;
    for (uint64_t v0 = (uint64_t)tid * 8; v0 < cols; v0 += 256 * 8) {
        const int count = (int)min((uint64_t)8, cols - v0);
        float v[8];
        if (out) {
#pragma unroll
            for (int t = 0; t < 8; t++) v[t] = 0.f;
        } else {
            load8<TYPE>(row + v0, count, v);
#pragma unroll
            for (int t = 0; t < 8; t++) v[t] = g * (p_sum * __builtin_amdgcn_exp2f((v[t] - m) * c + lift));
        }
        store8<TYPE>(grow + v0, count, v);
    }
    if (out) return;
    // the listed columns again, with their probabilities: after every store of the row has left this CU
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    for (uint32_t j = tid; j < list.k; j += 256) {
        const uint32_t v = li[j];
        if (v == 0xFFFFFFFFu) continue;
        float p = 0.f;
        for (uint32_t o = 0; o < list.k; o++) p += li[o] == v ? lp[o] : 0.f;   // equal columns: the same sum in the same order
        grow[v] = (T)(g * (p_sum * __builtin_amdgcn_exp2f((ls[j] - m) * c + lift) - p));
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
        hipLaunchKernelGGL((teacher_row_kernel<TYPE, LOSS>), dim3((unsigned)rows), dim3(256), 0, s, static_cast<const T*>(d_logits), cols, ld, list,
                           temperature, weight, loss, stats, static_cast<T*>(d_grad), ldg);
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
