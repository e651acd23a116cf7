// Distillation from a teacher's top logits: the loss of each row, its mean, and the gradient.
//
// Row r has `vocab` student logits z and k entries (t_j, i_j) of the teacher.  With temperature T
//   p_j = exp(t_j / T) / sum_j exp(t_j / T)      over the entries that count (0 <= i_j < vocab, t_j > -inf), or
//   p_j = exp(t_j / T - lse_r)                   where the teacher's own normaliser is given,
//   log q_v = (z_v - m) / T - log S,             m = max z, S = sum_v exp((z_v - m) / T),
//   row_loss = sum_j p_j (log p_j - log q_{i_j}),    loss = scale * sum_r w_r row_loss_r,
//   dz_v = scale w_r / T * (P q_v - sum of the p_j whose i_j is v),    P = sum_j p_j.
// A row of weight 0 or without entries that count is left out: loss 0, gradient 0, its logits not read.
//
// Differences of logarithms are taken in 64 bits (k of them a row): where teacher and student
// agree, the loss is a small difference of numbers of size ten.
#include <climits>
#include <type_traits>

#include "fdl_types.cuh"

namespace fdl {

namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / kWarp;
constexpr int kMaxEntries = 1024;
constexpr float kLog2e = 1.4426950408889634f;

struct DistillParams {
    const void* logits;
    int64_t logits_stride;
    const void* teacher;
    int teacher_dtype;
    const int64_t* index;
    const float* teacher_lse;  // may be null
    const float* row_weight;   // may be null
    int64_t rows;
    int vocab;
    int k;
    double inv_temperature;
    float scale;
    float* row_loss;
    float* row_stats;        // [rows][2]: m and S; written by the loss, read by the gradient alone
    const float* grad_loss;  // may be null (1)
    void* grad;
    int64_t grad_stride;
};

__device__ __forceinline__ float load_any(const void* p, int dtype, int64_t i) {
    if (dtype == FDL_F32) return static_cast<const float*>(p)[i];
    if (dtype == FDL_F16) return __half2float(static_cast<const __half*>(p)[i]);
    return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}

// exp((a - b) / T) for a running maximum a <= b, with c = log2(e) / T; 1 when both are -inf.
__device__ __forceinline__ float exp_diff(float a, float b, float c) { return a == b ? 1.0f : ex2_approx((a - b) * c); }

__device__ __forceinline__ float block_max(float v, float* red) {
    v = warp_max(v);
    __syncthreads();
    if ((threadIdx.x & (kWarp - 1)) == 0) red[threadIdx.x / kWarp] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) v = fmaxf(v, red[w]);
    return v;
}

template <class S>
__device__ __forceinline__ S block_sum(S v, S* red) {
    v = warp_sum(v);
    __syncthreads();
    if ((threadIdx.x & (kWarp - 1)) == 0) red[threadIdx.x / kWarp] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) v += red[w];
    return v;
}

// A row as a head and a tail of single elements around aligned 128-bit packs.
template <class T>
struct RowSpan {
    int head, packs, tail;
    __device__ RowSpan(const T* row, int n) {
        const int off = static_cast<int>((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / static_cast<int>(sizeof(T));
        head = off < n ? off : n;
        packs = (n - head) / kPack<T>;
        tail = n - head - packs * kPack<T>;
    }
};

template <class T, bool LOSS, bool GRAD>
__global__ void __launch_bounds__(kThreads)
distill_rows_kernel(const DistillParams p) {
    constexpr int N = kPack<T>;
    __shared__ float prob[kMaxEntries];
    __shared__ int at[kMaxEntries];
    __shared__ float here[kMaxEntries];
    __shared__ float redf[kWarps];
    __shared__ double redd[kWarps];
    const int t = threadIdx.x;
    const float c = static_cast<float>(kLog2e * p.inv_temperature);
    pdl_wait();
    for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const T* z = static_cast<const T*>(p.logits) + row * p.logits_stride;
        const float weight = p.row_weight == nullptr ? 1.0f : p.row_weight[row];
        // The teacher's entries.
        float top = -INFINITY;
        for (int j = t; j < p.k; j += kThreads) {
            const int64_t i = p.index[row * p.k + j];
            const bool valid = i >= 0 && i < p.vocab;
            const float v = valid ? load_any(p.teacher, p.teacher_dtype, row * p.k + j) : -INFINITY;
            prob[j] = v;
            at[j] = v > -INFINITY ? static_cast<int>(i) : -1;  // a NaN does not count either
            top = fmaxf(top, v);
        }
        top = block_max(top, redf);
        const bool live = weight != 0.0f && top != -INFINITY;
        T* g = GRAD ? static_cast<T*>(p.grad) + row * p.grad_stride : nullptr;
        if (!live) {
            if (LOSS && t == 0) {
                p.row_loss[row] = 0.0f;
                p.row_stats[2 * row] = 0.0f;
                p.row_stats[2 * row + 1] = 0.0f;
            }
            if (GRAD) {
                for (int i = t; i < p.vocab; i += kThreads) g[i] = from_f32<T>(0.0f);
            }
            __syncthreads();
            continue;
        }
        float part = 0.0f;
        for (int j = t; j < p.k; j += kThreads) {
            if (at[j] >= 0) {
                here[j] = to_f32(z[at[j]]);
                part += ex2_approx((prob[j] - top) * c);
            }
        }
        const float teacher_sum = block_sum(part, redf);
        const double log_norm = p.teacher_lse == nullptr
                                    ? static_cast<double>(top) * p.inv_temperature + log(static_cast<double>(teacher_sum))
                                    : static_cast<double>(p.teacher_lse[row]);
        // The student's statistics.
        float m, total;
        if (LOSS) {
            const RowSpan<T> span(z, p.vocab);
            const T* body = z + span.head;
            float mx = -INFINITY, s = 0.0f;
            for (int i = t; i < span.packs; i += kThreads) {
                float v[N];
                Chunk<T, N>::load(body + static_cast<int64_t>(i) * N, v);
                float big = v[0];
#pragma unroll
                for (int e = 1; e < N; ++e) big = fmaxf(big, v[e]);
                const float now = fmaxf(mx, big);
                const float ref = now == -INFINITY ? 0.0f : now;  // nothing but -inf so far: exp(-inf) each
                float add = 0.0f;
#pragma unroll
                for (int e = 0; e < N; ++e) add += ex2_approx((v[e] - ref) * c);
                s = s * exp_diff(mx, now, c) + add;
                mx = now;
            }
            if (t < span.head + span.tail) {
                const float v = to_f32(t < span.head ? z[t] : z[p.vocab - 1 - (t - span.head)]);
                const float now = fmaxf(mx, v);
                s = s * exp_diff(mx, now, c) + ex2_approx((v - (now == -INFINITY ? 0.0f : now)) * c);
                mx = now;
            }
            m = block_max(mx, redf);
            total = block_sum(s * exp_diff(mx, m, c), redf);
            if (t == 0) {
                p.row_stats[2 * row] = m;
                p.row_stats[2 * row + 1] = total;
            }
        } else {
            m = p.row_stats[2 * row];
            total = p.row_stats[2 * row + 1];
        }
        const double log_total = log(static_cast<double>(total));
        double kl = 0.0;
        float mass = 0.0f;
        for (int j = t; j < p.k; j += kThreads) {
            float pj = 0.0f;
            if (at[j] >= 0) {
                const double logp = static_cast<double>(prob[j]) * p.inv_temperature - log_norm;
                pj = expf(static_cast<float>(logp));
                const double logq = (static_cast<double>(here[j]) - m) * p.inv_temperature - log_total;
                if (pj != 0.0f) kl += pj * (logp - logq);
            }
            prob[j] = pj;
            mass += pj;
        }
        if (LOSS) {
            kl = block_sum(kl, redd);
            if (t == 0) p.row_loss[row] = static_cast<float>(kl);
        }
        if (GRAD) {
            mass = block_sum(mass, redf);
            if (p.teacher_lse == nullptr) mass = mass == mass ? 1.0f : mass;
            float coef = p.scale * weight * static_cast<float>(p.inv_temperature);
            if (p.grad_loss != nullptr) coef *= *p.grad_loss;
            const float each = coef * mass / total;
            // In place: every read of the row (above) is done before the first write.
            const RowSpan<T> span(z, p.vocab);
            const bool same_phase = ((reinterpret_cast<uintptr_t>(z) ^ reinterpret_cast<uintptr_t>(g)) & 15) == 0;
            const int head = same_phase ? span.head : 0, packs = same_phase ? span.packs : 0;
            for (int i = t; i < packs; i += kThreads) {
                float v[N];
                Chunk<T, N>::load(z + head + static_cast<int64_t>(i) * N, v);
#pragma unroll
                for (int e = 0; e < N; ++e) v[e] = ex2_approx((v[e] - m) * c) * each;
                Chunk<T, N>::store_stream(g + head + static_cast<int64_t>(i) * N, v);
            }
            for (int i = t; i < p.vocab - packs * N; i += kThreads) {
                const int col = i < head ? i : i + packs * N;
                g[col] = from_f32<T>(ex2_approx((to_f32(z[col]) - m) * c) * each);
            }
            __syncthreads();
            // The teacher's places, written after the dense part (same CTA, behind a barrier).  An
            // index that is there twice is written by its first entry, with the sum in entry order.
            for (int j = t; j < p.k; j += kThreads) {
                if (at[j] < 0) continue;
                bool first = true;
                for (int i = 0; i < j; ++i) first = first && at[i] != at[j];
                if (!first) continue;
                float sum = 0.0f;
                for (int i = j; i < p.k; ++i) sum += at[i] == at[j] ? prob[i] : 0.0f;
                g[at[j]] = from_f32<T>(coef * (mass * (ex2_approx((here[j] - m) * c) / total) - sum));
            }
        }
        __syncthreads();
    }
}

// loss = scale * sum of weight * row loss, in 64 bits and in a fixed order.
__global__ void __launch_bounds__(1024)
distill_mean_kernel(const float* row_loss, const float* row_weight, int64_t rows, float scale, float* loss) {
    __shared__ double red[1024 / kWarp];
    pdl_wait();
    double s = 0.0;
    for (int64_t r = threadIdx.x; r < rows; r += blockDim.x) {
        const float w = row_weight == nullptr ? 1.0f : row_weight[r];
        if (w != 0.0f) s += static_cast<double>(w) * row_loss[r];
    }
    s = warp_sum(s);
    if ((threadIdx.x & (kWarp - 1)) == 0) red[threadIdx.x / kWarp] = s;
    __syncthreads();
    if (threadIdx.x < kWarp) {
        s = warp_sum(red[threadIdx.x]);
        if (threadIdx.x == 0) *loss = static_cast<float>(s * scale);
    }
}

int check_common(const void* logits, int64_t stride, int dtype, const void* teacher, int teacher_dtype,
                 const int64_t* index, int64_t rows, int64_t vocab, int64_t k, float temperature) {
    if (rows < 0 || vocab <= 0 || k <= 0 || stride < vocab || !known_dtype(dtype) || !known_dtype(teacher_dtype) ||
        !(temperature > 0.0f) || !(temperature < INFINITY)) {
        return FDL_ERR_INVALID_ARGUMENT;
    }
    if (rows > INT_MAX || vocab > INT_MAX - 65536 || k > kMaxEntries) return FDL_ERR_UNSUPPORTED;
    if (rows > 0 && (logits == nullptr || teacher == nullptr || index == nullptr)) return FDL_ERR_INVALID_ARGUMENT;
    return FDL_OK;
}

template <bool LOSS, bool GRAD>
int launch_rows(const DistillParams& p, int dtype, cudaStream_t stream) {
    int status = FDL_OK;
    const DeviceInfo* info = current_device_info(&status);
    if (info == nullptr) return status;
    const int grid = persistent_grid(info, 4, p.rows);
    return with_dtype(dtype, [&](auto* tag) {
        using T = std::remove_pointer_t<decltype(tag)>;
        return launch_ex(distill_rows_kernel<T, LOSS, GRAD>, dim3(grid), dim3(kThreads), 0, stream, dim3(1, 1, 1),
                         tuning().pdl != 0, p);
    });
}

}  // namespace

}  // namespace fdl

using namespace fdl;

extern "C" {

int fdl_distill_topk(const void* logits, int64_t logits_stride, int dtype, const void* teacher, int teacher_dtype,
                     const int64_t* index, const float* teacher_lse, const float* row_weight, int64_t rows,
                     int64_t vocab, int64_t k, float temperature, float scale, float* loss, float* row_loss,
                     float* row_stats, void* stream) {
    int status = check_common(logits, logits_stride, dtype, teacher, teacher_dtype, index, rows, vocab, k, temperature);
    if (status != FDL_OK) return status;
    if (loss == nullptr || (rows > 0 && (row_loss == nullptr || row_stats == nullptr))) return FDL_ERR_INVALID_ARGUMENT;
    cudaStream_t s = as_stream(stream);
    if (rows == 0) return static_cast<int>(cudaMemsetAsync(loss, 0, sizeof(float), s));
    const DistillParams p{logits, logits_stride, teacher, teacher_dtype, index, teacher_lse, row_weight, rows,
                          static_cast<int>(vocab), static_cast<int>(k), 1.0 / static_cast<double>(temperature), scale, row_loss, row_stats,
                          nullptr, nullptr, 0};
    status = launch_rows<true, false>(p, dtype, s);
    if (status != FDL_OK) return status;
    return launch_ex(distill_mean_kernel, dim3(1), dim3(1024), 0, s, dim3(1, 1, 1), tuning().pdl != 0,
                     static_cast<const float*>(row_loss), row_weight, rows, scale, loss);
}

int fdl_distill_topk_backward(const void* logits, int64_t logits_stride, int dtype, const void* teacher,
                              int teacher_dtype, const int64_t* index, const float* teacher_lse,
                              const float* row_weight, const float* row_stats, const float* grad_loss, int64_t rows,
                              int64_t vocab, int64_t k, float temperature, float scale, void* grad,
                              int64_t grad_stride, void* stream) {
    int status = check_common(logits, logits_stride, dtype, teacher, teacher_dtype, index, rows, vocab, k, temperature);
    if (status != FDL_OK) return status;
    if (grad_stride < vocab || (rows > 0 && (row_stats == nullptr || grad == nullptr))) return FDL_ERR_INVALID_ARGUMENT;
    if (grad == logits && grad_stride != logits_stride) return FDL_ERR_INVALID_ARGUMENT;
    if (rows == 0) return FDL_OK;
    const DistillParams p{logits, logits_stride, teacher, teacher_dtype, index, teacher_lse, row_weight, rows,
                          static_cast<int>(vocab), static_cast<int>(k), 1.0 / static_cast<double>(temperature), scale, nullptr,
                          const_cast<float*>(row_stats), grad_loss, grad, grad_stride};
    return launch_rows<false, true>(p, dtype, as_stream(stream));
}

int fdl_distill_topk_with_grad(const void* logits, int64_t logits_stride, int dtype, const void* teacher,
                               int teacher_dtype, const int64_t* index, const float* teacher_lse,
                               const float* row_weight, int64_t rows, int64_t vocab, int64_t k, float temperature,
                               float scale, float* loss, float* row_loss, float* row_stats, void* grad,
                               int64_t grad_stride, void* stream) {
    int status = check_common(logits, logits_stride, dtype, teacher, teacher_dtype, index, rows, vocab, k, temperature);
    if (status != FDL_OK) return status;
    if (loss == nullptr || grad_stride < vocab ||
        (rows > 0 && (row_loss == nullptr || row_stats == nullptr || grad == nullptr))) {
        return FDL_ERR_INVALID_ARGUMENT;
    }
    if (grad == logits && grad_stride != logits_stride) return FDL_ERR_INVALID_ARGUMENT;
    cudaStream_t s = as_stream(stream);
    if (rows == 0) return static_cast<int>(cudaMemsetAsync(loss, 0, sizeof(float), s));
    const DistillParams p{logits, logits_stride, teacher, teacher_dtype, index, teacher_lse, row_weight, rows,
                          static_cast<int>(vocab), static_cast<int>(k), 1.0 / static_cast<double>(temperature), scale, row_loss, row_stats,
                          nullptr, grad, grad_stride};
    status = launch_rows<true, true>(p, dtype, s);
    if (status != FDL_OK) return status;
    return launch_ex(distill_mean_kernel, dim3(1), dim3(1024), 0, s, dim3(1, 1, 1), tuning().pdl != 0,
                     static_cast<const float*>(row_loss), row_weight, rows, scale, loss);
}

}  // extern "C"
