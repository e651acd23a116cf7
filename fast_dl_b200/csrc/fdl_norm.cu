// The norms after and before a block, with its gate and the residual's scale, forward and backward.
//
//   u = N_post(h),   y = residual_scale * x + block_scale * act(gate) * u,   n = N_pre(y)
//
// N is the identity, the RMS norm v * r with r = 1 / sqrt(mean(v^2) + eps), or the layer norm
// (v - mean) * r with r = 1 / sqrt(mean((v - mean)^2) + eps), each times gamma plus beta.  n is taken
// from y before y is rounded to its type.  The gate has gate_rows rows, each for rows / gate_rows
// consecutive rows of x.
//
// Backward, from dy and dn, with hat = (v - mean) * r of the norm's input v and c columns:
//   D  = dy + G(dn * pre_gamma, hat(y)),  G(d, hat) = r * (d - [layer: sum d / c] - hat * sum(d hat) / c)
//   dx = residual_scale * D,  E = block_scale * D,  a = act(gate)
//   dgate = act'(gate) * sum over its rows of E u,  du = E a,  dh = G(du * post_gamma, hat(h))
//   dpre_gamma = sum dn hat(y), dpre_beta = sum dn, dpost_gamma = sum du hat(h), dpost_beta = sum du.
//
// What bounds both: bytes.  Forward reads x, h (and a full gate) and writes y and n, backward reads dy,
// dn, y, h and writes dx, dh, each once: a row stays in the registers of its team from its first read to
// its last write.  A team is a warp (short rows), a CTA, or a cluster of CTAs that share a row's columns
// and exchange row sums through distributed shared memory.  A thread owns the same columns of every
// row that its team takes, so gamma and beta are read once, and the backward pass's sums over rows grow
// in registers; each team leaves one partial row of them in scratch, which a second kernel adds in a
// fixed order (no atomics: the same bits in every run).
#include <climits>
#include <initializer_list>
#include <type_traits>

#include "fdl_types.cuh"

namespace fdl {

namespace {

constexpr int kMaxCluster = 8;
constexpr int kMaxWarps = 16;

struct NormParams {
    const void* x;
    const void* h;
    const void* gate;  // may be null
    const void* dy;    // backward; may be null
    const void* dn;    // backward; may be null
    const void* y_in;  // backward
    const float* stats_in;
    const float* post_gamma;
    const float* post_beta;
    const float* pre_gamma;
    const float* pre_beta;
    void* y;
    void* n;
    float* stats;
    void* dx;
    void* dh;
    void* dgate;
    float* partial[4];    // post gamma, post beta, pre gamma, pre beta: [teams][cols], null if not wanted
    float* gate_partial;  // [tasks][cols], null: written to dgate directly
    int64_t rows;
    int64_t rows_per_gate;
    int64_t rows_per_task;   // backward: rows of a task, all of one gate row (or of all rows)
    int64_t tasks_per_gate;  // backward: tasks that share a gate row
    int64_t tasks;
    int cols;
    int post_kind, pre_kind, gate_act;
    float residual_scale, block_scale, eps;
};

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync_all() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void store_remote(float2* mine, uint32_t rank, float2 v) {
    uint32_t remote;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(smem_addr(mine)), "r"(rank));
    asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(remote), "f"(v.x), "f"(v.y) : "memory");
}

// Two sums over the team of a row.  One barrier each: the buffers alternate, and a buffer is written
// again only behind the barrier that follows its reads.
struct TeamSums {
    float2 buf[2][kMaxCluster * kMaxWarps];
};

template <bool WARP>
struct Team {
    TeamSums* sums;
    int phase, warps, cluster, rank;
    __device__ __forceinline__ float2 sum(float a, float b) {
        a = warp_sum(a);
        b = warp_sum(b);
        if (WARP) return make_float2(a, b);
        const int lane = threadIdx.x & (kWarp - 1), warp = threadIdx.x / kWarp;
        float2* at = sums->buf[phase];
        phase ^= 1;
        if (cluster == 1) {
            if (lane == 0) at[warp] = make_float2(a, b);
            __syncthreads();
        } else {
            if (lane < cluster) store_remote(&at[rank * warps + warp], lane, make_float2(a, b));
            cluster_sync_all();
        }
        const int n = warps * cluster;
        // Each warp folds the partial sums by itself, in the same order.
        float2 v = make_float2(0.0f, 0.0f);
        for (int i = lane; i < n; i += kWarp) {
            v.x += at[i].x;
            v.y += at[i].y;
        }
        return make_float2(warp_sum(v.x), warp_sum(v.y));
    }
};

__device__ __forceinline__ float gate_value(int act, float g) {
    if (act == FDL_GATE_SIGMOID) return 1.0f / (1.0f + expf(-g));
    if (act == FDL_GATE_TANH) return tanhf(g);
    return g;
}
// The slope of act at g, from a = act(g).
__device__ __forceinline__ float gate_slope(int act, float a) {
    if (act == FDL_GATE_SIGMOID) return a * (1.0f - a);
    if (act == FDL_GATE_TANH) return 1.0f - a * a;
    return 1.0f;
}

template <int N, int PACKS>
struct Owned {  // a thread's columns: PACKS chunks of N, a team's width apart
    int first, stride;
    __device__ __forceinline__ int col(int k) const { return (first + k * stride) * N; }
};

template <class T, int N, int PACKS>
__device__ __forceinline__ void load_row(const T* row, const Owned<N, PACKS>& own, int cols, float (&v)[PACKS][N]) {
#pragma unroll
    for (int k = 0; k < PACKS; ++k) {
        if (own.col(k) < cols) {
            Chunk<T, N>::load_stream(row + own.col(k), v[k]);
        } else {
#pragma unroll
            for (int e = 0; e < N; ++e) v[k][e] = 0.0f;
        }
    }
}

template <int N, int PACKS>
__device__ __forceinline__ void load_weights(const float* w, float none, const Owned<N, PACKS>& own, int cols,
                                             float (&v)[PACKS][N]) {
#pragma unroll
    for (int k = 0; k < PACKS; ++k) {
#pragma unroll
        for (int e = 0; e < N; ++e) v[k][e] = w != nullptr && own.col(k) < cols ? w[own.col(k) + e] : none;
    }
}

// mean and 1 / sqrt(variance + eps) of a row in registers (0 beyond its columns).
template <int N, int PACKS, class TeamT>
__device__ __forceinline__ float2 moments(int kind, float eps, const float (&v)[PACKS][N], const Owned<N, PACKS>& own,
                                          int cols, TeamT& team) {
    if (kind == FDL_NORM_NONE) return make_float2(0.0f, 1.0f);
    const float inv = 1.0f / static_cast<float>(cols);
    float mean = 0.0f;
    if (kind == FDL_NORM_LAYER) {
        float s = 0.0f;
#pragma unroll
        for (int k = 0; k < PACKS; ++k) {
#pragma unroll
            for (int e = 0; e < N; ++e) s += v[k][e];
        }
        mean = team.sum(s, 0.0f).x * inv;
    }
    float q = 0.0f;
#pragma unroll
    for (int k = 0; k < PACKS; ++k) {
        if (own.col(k) < cols) {
#pragma unroll
            for (int e = 0; e < N; ++e) q += (v[k][e] - mean) * (v[k][e] - mean);
        }
    }
    const float var = team.sum(q, 0.0f).x * inv;
    return make_float2(mean, 1.0f / sqrtf(var + eps));
}

template <class T, int N, int PACKS, bool WARP>
__global__ void __launch_bounds__(512)
norm_residual_kernel(const NormParams p) {
    __shared__ TeamSums sums;
    Team<WARP> team{&sums, 0, static_cast<int>(blockDim.x) / kWarp, 1, 0};
    Owned<N, PACKS> own;
    int64_t row, step;
    if (WARP) {
        const int warps = blockDim.x / kWarp;
        own.first = threadIdx.x & (kWarp - 1);
        own.stride = kWarp;
        row = static_cast<int64_t>(blockIdx.x) * warps + threadIdx.x / kWarp;
        step = static_cast<int64_t>(gridDim.x) * warps;
    } else {
        team.cluster = static_cast<int>(cluster_size());
        team.rank = static_cast<int>(cluster_rank());
        own.first = team.rank * blockDim.x + threadIdx.x;
        own.stride = team.cluster * blockDim.x;
        row = blockIdx.x / team.cluster;
        step = gridDim.x / team.cluster;
        if (team.cluster > 1) cluster_sync_all();  // every CTA has started before the first remote store
    }
    pdl_wait();
    for (; row < p.rows; row += step) {
        float h[PACKS][N], x[PACKS][N], w[PACKS][N];
        const int64_t base = row * p.cols;
        load_row<T>(static_cast<const T*>(p.h) + base, own, p.cols, h);
        load_row<T>(static_cast<const T*>(p.x) + base, own, p.cols, x);
        const float2 s1 = moments(p.post_kind, p.eps, h, own, p.cols, team);
        if (p.post_gamma != nullptr || p.post_beta != nullptr) {
            load_weights(p.post_gamma, 1.0f, own, p.cols, w);
#pragma unroll
            for (int k = 0; k < PACKS; ++k) {
#pragma unroll
                for (int e = 0; e < N; ++e) h[k][e] = (h[k][e] - s1.x) * s1.y * w[k][e];
            }
            load_weights(p.post_beta, 0.0f, own, p.cols, w);
#pragma unroll
            for (int k = 0; k < PACKS; ++k) {
#pragma unroll
                for (int e = 0; e < N; ++e) h[k][e] += w[k][e];
            }
        } else if (p.post_kind != FDL_NORM_NONE) {
#pragma unroll
            for (int k = 0; k < PACKS; ++k) {
#pragma unroll
                for (int e = 0; e < N; ++e) h[k][e] = (h[k][e] - s1.x) * s1.y;
            }
        }
        if (p.gate != nullptr) {
            load_row<T>(static_cast<const T*>(p.gate) + row / p.rows_per_gate * p.cols, own, p.cols, w);
#pragma unroll
            for (int k = 0; k < PACKS; ++k) {
#pragma unroll
                for (int e = 0; e < N; ++e) h[k][e] *= gate_value(p.gate_act, w[k][e]);
            }
        }
#pragma unroll
        for (int k = 0; k < PACKS; ++k) {
#pragma unroll
            for (int e = 0; e < N; ++e) {
                x[k][e] = own.col(k) < p.cols ? p.residual_scale * x[k][e] + p.block_scale * h[k][e] : 0.0f;
            }
            if (own.col(k) < p.cols) Chunk<T, N>::store_stream(static_cast<T*>(p.y) + base + own.col(k), x[k]);
        }
        const float2 s2 = moments(p.pre_kind, p.eps, x, own, p.cols, team);
        if (p.stats != nullptr && own.first == 0) {
            reinterpret_cast<float4*>(p.stats)[row] = make_float4(s1.x, s1.y, s2.x, s2.y);
        }
        if (p.n != nullptr) {
            load_weights(p.pre_gamma, 1.0f, own, p.cols, w);
            load_weights(p.pre_beta, 0.0f, own, p.cols, h);
#pragma unroll
            for (int k = 0; k < PACKS; ++k) {
#pragma unroll
                for (int e = 0; e < N; ++e) x[k][e] = (x[k][e] - s2.x) * s2.y * w[k][e] + h[k][e];
                if (own.col(k) < p.cols) Chunk<T, N>::store_stream(static_cast<T*>(p.n) + base + own.col(k), x[k]);
            }
        }
    }
    if (!WARP && team.cluster > 1) cluster_sync_all();  // no CTA leaves while another may still write its sums
}

// A team takes whole tasks: rows_per_task consecutive rows of one gate row.
template <class T, int N, int PACKS, bool WARP>
__global__ void __launch_bounds__(512)
norm_residual_backward_kernel(const NormParams p) {
    __shared__ TeamSums sums;
    Team<WARP> team{&sums, 0, static_cast<int>(blockDim.x) / kWarp, 1, 0};
    Owned<N, PACKS> own;
    int64_t id, teams;
    if (WARP) {
        const int warps = blockDim.x / kWarp;
        own.first = threadIdx.x & (kWarp - 1);
        own.stride = kWarp;
        id = static_cast<int64_t>(blockIdx.x) * warps + threadIdx.x / kWarp;
        teams = static_cast<int64_t>(gridDim.x) * warps;
    } else {
        team.cluster = static_cast<int>(cluster_size());
        team.rank = static_cast<int>(cluster_rank());
        own.first = team.rank * blockDim.x + threadIdx.x;
        own.stride = team.cluster * blockDim.x;
        id = blockIdx.x / team.cluster;
        teams = gridDim.x / team.cluster;
        if (team.cluster > 1) cluster_sync_all();  // every CTA has started before the first remote store
    }
    pdl_wait();
    float acc[4][PACKS][N];
#pragma unroll
    for (int a = 0; a < 4; ++a) {
#pragma unroll
        for (int k = 0; k < PACKS; ++k) {
#pragma unroll
            for (int e = 0; e < N; ++e) acc[a][k][e] = 0.0f;
        }
    }
    const float inv = 1.0f / static_cast<float>(p.cols);
    const bool gate_each = p.rows_per_gate == 1;
    for (int64_t task = id; task < p.tasks; task += teams) {
        const int64_t group = task / p.tasks_per_gate, part = task % p.tasks_per_gate;
        const int64_t from = gate_each ? task * p.rows_per_task : group * p.rows_per_gate + part * p.rows_per_task;
        const int64_t end = gate_each ? p.rows : (group + 1) * p.rows_per_gate;
        const int64_t to = from + p.rows_per_task < end ? from + p.rows_per_task : end;
        float gsum[PACKS][N], gate[PACKS][N];
#pragma unroll
        for (int k = 0; k < PACKS; ++k) {
#pragma unroll
            for (int e = 0; e < N; ++e) {
                gsum[k][e] = 0.0f;
                gate[k][e] = 1.0f;
            }
        }
        if (p.gate != nullptr && !gate_each) {
            load_row<T>(static_cast<const T*>(p.gate) + group * p.cols, own, p.cols, gate);
#pragma unroll
            for (int k = 0; k < PACKS; ++k) {
#pragma unroll
                for (int e = 0; e < N; ++e) gate[k][e] = gate_value(p.gate_act, gate[k][e]);
            }
        }
        for (int64_t row = from; row < to; ++row) {
            const int64_t base = row * p.cols;
            const float4 st = reinterpret_cast<const float4*>(p.stats_in)[row];
            float d[PACKS][N], hat[PACKS][N], w[PACKS][N];
            // D: the gradient of y with the next norm's share.
            if (p.dn != nullptr) {
                load_row<T>(static_cast<const T*>(p.dn) + base, own, p.cols, d);
                load_row<T>(static_cast<const T*>(p.y_in) + base, own, p.cols, hat);
                load_weights(p.pre_gamma, 1.0f, own, p.cols, w);
                float sd = 0.0f, sdh = 0.0f;
#pragma unroll
                for (int k = 0; k < PACKS; ++k) {
#pragma unroll
                    for (int e = 0; e < N; ++e) {
                        hat[k][e] = (hat[k][e] - st.z) * st.w;
                        acc[2][k][e] += d[k][e] * hat[k][e];
                        acc[3][k][e] += d[k][e];
                        d[k][e] *= w[k][e];
                        sd += d[k][e];
                        sdh += d[k][e] * hat[k][e];
                    }
                }
                const float2 s = team.sum(sd, sdh);
                const float level = p.pre_kind == FDL_NORM_LAYER ? s.x * inv : 0.0f, along = s.y * inv;
#pragma unroll
                for (int k = 0; k < PACKS; ++k) {
#pragma unroll
                    for (int e = 0; e < N; ++e) d[k][e] = st.w * (d[k][e] - level - hat[k][e] * along);
                }
            } else {
#pragma unroll
                for (int k = 0; k < PACKS; ++k) {
#pragma unroll
                    for (int e = 0; e < N; ++e) d[k][e] = 0.0f;
                }
            }
            if (p.dy != nullptr) {
                load_row<T>(static_cast<const T*>(p.dy) + base, own, p.cols, w);
#pragma unroll
                for (int k = 0; k < PACKS; ++k) {
#pragma unroll
                    for (int e = 0; e < N; ++e) d[k][e] += w[k][e];
                }
            }
            load_row<T>(static_cast<const T*>(p.h) + base, own, p.cols, hat);
            if (p.gate != nullptr && gate_each) {
                load_row<T>(static_cast<const T*>(p.gate) + base, own, p.cols, gate);
#pragma unroll
                for (int k = 0; k < PACKS; ++k) {
#pragma unroll
                    for (int e = 0; e < N; ++e) gate[k][e] = gate_value(p.gate_act, gate[k][e]);
                }
            }
            if (p.dx != nullptr) {
#pragma unroll
                for (int k = 0; k < PACKS; ++k) {
#pragma unroll
                    for (int e = 0; e < N; ++e) w[k][e] = p.residual_scale * d[k][e];
                    if (own.col(k) < p.cols) Chunk<T, N>::store_stream(static_cast<T*>(p.dx) + base + own.col(k), w[k]);
                }
            }
#pragma unroll
            for (int k = 0; k < PACKS; ++k) {
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    hat[k][e] = (hat[k][e] - st.x) * st.y;
                    d[k][e] *= p.block_scale;
                }
            }
            if (p.dgate != nullptr) {
                float u[PACKS][N];
                load_weights(p.post_gamma, 1.0f, own, p.cols, u);
                load_weights(p.post_beta, 0.0f, own, p.cols, w);
#pragma unroll
                for (int k = 0; k < PACKS; ++k) {
#pragma unroll
                    for (int e = 0; e < N; ++e) {
                        u[k][e] = d[k][e] * (hat[k][e] * u[k][e] + w[k][e]);
                        if (gate_each) u[k][e] *= gate_slope(p.gate_act, gate[k][e]);
                        else gsum[k][e] += u[k][e];
                    }
                    if (gate_each && own.col(k) < p.cols) {
                        Chunk<T, N>::store_stream(static_cast<T*>(p.dgate) + base + own.col(k), u[k]);
                    }
                }
            }
            load_weights(p.post_gamma, 1.0f, own, p.cols, w);
            float sd = 0.0f, sdh = 0.0f;
#pragma unroll
            for (int k = 0; k < PACKS; ++k) {
                const bool inside = own.col(k) < p.cols;
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    if (!inside) hat[k][e] = d[k][e] = 0.0f;
                    d[k][e] *= gate[k][e];
                    acc[0][k][e] += d[k][e] * hat[k][e];
                    acc[1][k][e] += d[k][e];
                    d[k][e] *= w[k][e];
                    sd += d[k][e];
                    sdh += d[k][e] * hat[k][e];
                }
            }
            if (p.post_kind != FDL_NORM_NONE) {
                const float2 s = team.sum(sd, sdh);
                const float level = p.post_kind == FDL_NORM_LAYER ? s.x * inv : 0.0f, along = s.y * inv;
#pragma unroll
                for (int k = 0; k < PACKS; ++k) {
#pragma unroll
                    for (int e = 0; e < N; ++e) d[k][e] = st.y * (d[k][e] - level - hat[k][e] * along);
                }
            }
            if (p.dh != nullptr) {
#pragma unroll
                for (int k = 0; k < PACKS; ++k) {
                    if (own.col(k) < p.cols) Chunk<T, N>::store_stream(static_cast<T*>(p.dh) + base + own.col(k), d[k]);
                }
            }
        }
        if (p.dgate != nullptr && !gate_each) {
#pragma unroll
            for (int k = 0; k < PACKS; ++k) {
                if (own.col(k) >= p.cols) continue;
#pragma unroll
                for (int e = 0; e < N; ++e) gsum[k][e] *= gate_slope(p.gate_act, gate[k][e]);
                if (p.gate_partial != nullptr) {
#pragma unroll
                    for (int e = 0; e < N; ++e) p.gate_partial[task * p.cols + own.col(k) + e] = gsum[k][e];
                } else {
                    Chunk<T, N>::store_stream(static_cast<T*>(p.dgate) + group * p.cols + own.col(k), gsum[k]);
                }
            }
        }
    }
#pragma unroll
    for (int a = 0; a < 4; ++a) {
        if (p.partial[a] == nullptr) continue;
#pragma unroll
        for (int k = 0; k < PACKS; ++k) {
            if (own.col(k) >= p.cols) continue;
#pragma unroll
            for (int e = 0; e < N; ++e) p.partial[a][id * p.cols + own.col(k) + e] = acc[a][k][e];
        }
    }
    if (!WARP && team.cluster > 1) cluster_sync_all();  // no CTA leaves while another may still write its sums
}

// out[g, c] = sum over r of part[g * each + r, c], rows in order; blockIdx.y picks one of the jobs.
struct FoldJob {
    const float* part;
    void* out;
    int dtype;
    int64_t groups, each;
};
struct FoldJobs {
    FoldJob job[5];
    int cols;
};

constexpr int kFoldX = 32, kFoldY = 16;

__global__ void __launch_bounds__(kFoldX * kFoldY)
norm_fold_kernel(const FoldJobs jobs) {
    __shared__ float red[kFoldY][kFoldX + 1];
    const FoldJob job = jobs.job[blockIdx.y];
    const int c = blockIdx.x * kFoldX + threadIdx.x;
    pdl_wait();
    for (int64_t g = blockIdx.z; g < job.groups; g += gridDim.z) {
        float s = 0.0f;
        if (c < jobs.cols) {
#pragma unroll 4
            for (int64_t r = threadIdx.y; r < job.each; r += kFoldY) s += job.part[(g * job.each + r) * jobs.cols + c];
        }
        red[threadIdx.y][threadIdx.x] = s;
        __syncthreads();
        if (threadIdx.y == 0 && c < jobs.cols) {
            s = red[0][threadIdx.x];
#pragma unroll
            for (int k = 1; k < kFoldY; ++k) s += red[k][threadIdx.x];
            const int64_t at = g * jobs.cols + c;
            if (job.dtype == FDL_F32) static_cast<float*>(job.out)[at] = s;
            else if (job.dtype == FDL_F16) static_cast<__half*>(job.out)[at] = from_f32<__half>(s);
            else static_cast<__nv_bfloat16*>(job.out)[at] = from_f32<__nv_bfloat16>(s);
        }
        __syncthreads();
    }
}

// ---- launch shapes -------------------------------------------------------------------------------

constexpr int kPerThread = 8;  // columns a thread owns
constexpr int kWarpCols = kWarp * kPerThread;
constexpr int kMaxCols = kMaxCluster * 512 * kPerThread;

struct Shape {
    bool warp;     // a warp a row
    int threads;   // of a CTA
    int cluster;   // CTAs a row
    int blocks;    // CTAs that an SM is given
};

Shape shape_of(int64_t cols) {
    if (cols <= kWarpCols) return {true, 256, 1, 4};
    int cluster = 1;
    while (cols > static_cast<int64_t>(cluster) * 512 * kPerThread) cluster *= 2;
    const int threads = static_cast<int>(ceil_div(ceil_div(cols, static_cast<int64_t>(cluster) * kPerThread), kWarp)) * kWarp;
    return {false, threads, cluster, 1024 / threads < 1 ? 1 : 1024 / threads};
}

struct BackwardPlan {
    Shape shape;
    int64_t grid;   // CTAs
    int64_t teams;  // partial rows of the sums over rows
    int64_t rows_per_gate, tasks_per_gate, rows_per_task, tasks;
};

// Tasks: every team gets about the same number of rows, and no task crosses a gate row's rows.
BackwardPlan backward_plan(int64_t rows, int64_t cols, int64_t gate_rows, int sm_count) {
    BackwardPlan b;
    b.shape = shape_of(cols);
    const int64_t per_cta = b.shape.warp ? b.shape.threads / kWarp : 1;
    const int64_t slots = static_cast<int64_t>(sm_count) * b.shape.blocks / b.shape.cluster;  // teams of CTAs
    const int64_t most = (slots < 1 ? 1 : slots) * per_cta;                                    // teams at once
    const bool gate_each = gate_rows == rows;
    const int64_t groups = gate_rows == 0 || gate_each ? 1 : gate_rows;
    const int64_t group = rows / groups;
    b.rows_per_gate = gate_each ? 1 : group;
    int64_t best = 1;
    double fill = 0.0;
    for (int64_t q = 1; q <= 4; ++q) {  // q tasks a team: the first that keeps 95% of the teams busy, or the best
        const int64_t each = q * most / groups;
        if (each < 1) continue;
        const double f = static_cast<double>(each * groups) / static_cast<double>(q * most);
        if (f > fill + 0.01) {
            fill = f;
            best = each;
        }
        if (fill >= 0.95) break;
    }
    if (best > group) best = group;
    b.rows_per_task = ceil_div(group, best);
    b.tasks_per_gate = ceil_div(group, b.rows_per_task);
    b.tasks = b.tasks_per_gate * groups;
    b.teams = b.tasks < most ? b.tasks : most;
    b.grid = ceil_div(b.teams, per_cta) * b.shape.cluster;
    b.teams = b.grid / b.shape.cluster * per_cta;
    return b;
}

int check_norm(int64_t rows, int64_t cols, const void* gate, int64_t gate_rows, int gate_act, int post_kind, int pre_kind,
               int dtype) {
    if (rows < 0 || cols <= 0 || !known_dtype(dtype) || post_kind < FDL_NORM_NONE || post_kind > FDL_NORM_LAYER ||
        pre_kind < FDL_NORM_NONE || pre_kind > FDL_NORM_LAYER || gate_act < FDL_GATE_PLAIN || gate_act > FDL_GATE_TANH) {
        return FDL_ERR_INVALID_ARGUMENT;
    }
    if ((gate == nullptr) != (gate_rows == 0) || gate_rows < 0) return FDL_ERR_INVALID_ARGUMENT;
    if (gate != nullptr && rows > 0 && (gate_rows > rows || rows % gate_rows != 0)) return FDL_ERR_INVALID_ARGUMENT;
    if (cols > kMaxCols || rows > INT_MAX) return FDL_ERR_UNSUPPORTED;
    return FDL_OK;
}

// Whether 128-bit accesses fit: a row is whole packs and every tensor starts on the 16-byte grid.
bool packs_fit(int dtype, int64_t cols, std::initializer_list<const void*> tensors) {
    if (cols % (16 / static_cast<int64_t>(dtype_bytes(dtype))) != 0) return false;
    for (const void* t : tensors) {
        if (!aligned16(t)) return false;
    }
    return true;
}

template <template <class, int, int, bool> class Launch, class... Args>
int dispatch(int dtype, bool vec, bool warp, Args&&... args) {
    return with_dtype(dtype, [&](auto* tag) {
        using T = std::remove_pointer_t<decltype(tag)>;
        constexpr int N = kPack<T>;
        if (vec) {
            return warp ? Launch<T, N, kPerThread / N, true>::run(args...) : Launch<T, N, kPerThread / N, false>::run(args...);
        }
        return warp ? Launch<T, 1, kPerThread, true>::run(args...) : Launch<T, 1, kPerThread, false>::run(args...);
    });
}

template <class T, int N, int PACKS, bool WARP>
struct LaunchForward {
    static int run(const NormParams& p, const Shape& s, int64_t grid, cudaStream_t stream) {
        return launch_ex(norm_residual_kernel<T, N, PACKS, WARP>, dim3(static_cast<unsigned int>(grid)), dim3(s.threads), 0,
                         stream, dim3(s.cluster, 1, 1), tuning().pdl != 0, p);
    }
};

template <class T, int N, int PACKS, bool WARP>
struct LaunchBackward {
    static int run(const NormParams& p, const Shape& s, int64_t grid, cudaStream_t stream) {
        return launch_ex(norm_residual_backward_kernel<T, N, PACKS, WARP>, dim3(static_cast<unsigned int>(grid)),
                         dim3(s.threads), 0, stream, dim3(s.cluster, 1, 1), tuning().pdl != 0, p);
    }
};

}  // namespace

}  // namespace fdl

using namespace fdl;

extern "C" {

int fdl_norm_residual(const void* x, const void* h, const void* gate, int64_t gate_rows, int gate_act, int post_kind,
                      const float* post_gamma, const float* post_beta, int pre_kind, const float* pre_gamma,
                      const float* pre_beta, void* y, void* n, float* stats, int64_t rows, int64_t cols,
                      float residual_scale, float block_scale, float eps, int dtype, void* stream) {
    int status = check_norm(rows, cols, gate, gate_rows, gate_act, post_kind, pre_kind, dtype);
    if (status != FDL_OK) return status;
    if (rows == 0) return FDL_OK;
    if (x == nullptr || h == nullptr || y == nullptr || (pre_kind == FDL_NORM_NONE) != (n == nullptr) || y == n ||
        !(eps >= 0.0f)) {
        return FDL_ERR_INVALID_ARGUMENT;
    }
    if (post_kind == FDL_NORM_NONE && (post_gamma != nullptr || post_beta != nullptr)) return FDL_ERR_INVALID_ARGUMENT;
    if (pre_kind == FDL_NORM_NONE && (pre_gamma != nullptr || pre_beta != nullptr)) return FDL_ERR_INVALID_ARGUMENT;
    if (!aligned16(stats)) return FDL_ERR_INVALID_ARGUMENT;
    const DeviceInfo* info = current_device_info(&status);
    if (info == nullptr) return status;
    NormParams p = {};
    p.x = x; p.h = h; p.gate = gate;
    p.post_gamma = post_gamma; p.post_beta = post_beta; p.pre_gamma = pre_gamma; p.pre_beta = pre_beta;
    p.y = y; p.n = n; p.stats = stats;
    p.rows = rows;
    p.rows_per_gate = gate == nullptr ? 1 : rows / gate_rows;
    p.cols = static_cast<int>(cols);
    p.post_kind = post_kind; p.pre_kind = pre_kind; p.gate_act = gate_act;
    p.residual_scale = residual_scale; p.block_scale = block_scale; p.eps = eps;
    const Shape s = shape_of(cols);
    const int64_t per_cta = s.warp ? s.threads / kWarp : 1;
    const int64_t slots = static_cast<int64_t>(info->sm_count) * s.blocks / s.cluster;
    const int64_t work = ceil_div(rows, per_cta);
    const int64_t grid = (work < slots ? work : slots < 1 ? 1 : slots) * s.cluster;
    return dispatch<LaunchForward>(dtype, packs_fit(dtype, cols, {x, h, gate, y, n}), s.warp, p, s, grid, as_stream(stream));
}

size_t fdl_norm_residual_backward_scratch_bytes(int64_t rows, int64_t cols, int64_t gate_rows) {
    if (rows <= 0 || cols <= 0 || cols > kMaxCols || gate_rows < 0) return 0;
    if (gate_rows > 0 && (gate_rows > rows || rows % gate_rows != 0)) return 0;
    int status = FDL_OK;
    const DeviceInfo* info = current_device_info(&status);
    const BackwardPlan b = backward_plan(rows, cols, gate_rows, info == nullptr ? 148 : info->sm_count);
    const int64_t gate_part = gate_rows == 0 || gate_rows == rows || b.tasks_per_gate == 1 ? 0 : b.tasks;
    const int64_t floats = (4 * b.teams + gate_part) * cols;
    return static_cast<size_t>(ceil_div(floats * 4, 256) * 256);
}

int fdl_norm_residual_backward(const void* dy, const void* dn, const void* y, const void* h, const float* stats,
                               const void* gate, int64_t gate_rows, int gate_act, int post_kind, const float* post_gamma,
                               const float* post_beta, int pre_kind, const float* pre_gamma, void* dx, void* dh,
                               void* dgate, float* dpost_gamma, float* dpost_beta, float* dpre_gamma, float* dpre_beta,
                               int64_t rows, int64_t cols, float residual_scale, float block_scale, int dtype,
                               void* scratch, size_t scratch_bytes, void* stream) {
    int status = check_norm(rows, cols, gate, gate_rows, gate_act, post_kind, pre_kind, dtype);
    if (status != FDL_OK) return status;
    cudaStream_t s = as_stream(stream);
    float* const sums[4] = {dpost_gamma, dpost_beta, dpre_gamma, dpre_beta};
    if (post_kind == FDL_NORM_NONE && (post_gamma != nullptr || post_beta != nullptr || dpost_gamma != nullptr || dpost_beta != nullptr)) {
        return FDL_ERR_INVALID_ARGUMENT;
    }
    if (pre_kind == FDL_NORM_NONE && (pre_gamma != nullptr || dpre_gamma != nullptr || dpre_beta != nullptr || dn != nullptr)) {
        return FDL_ERR_INVALID_ARGUMENT;
    }
    if (gate == nullptr && dgate != nullptr) return FDL_ERR_INVALID_ARGUMENT;
    if (rows == 0) {  // sums over no rows
        for (float* out : sums) {
            if (out != nullptr && status == FDL_OK) {
                status = static_cast<int>(cudaMemsetAsync(out, 0, static_cast<size_t>(cols) * sizeof(float), s));
            }
        }
        if (dgate != nullptr && status == FDL_OK) {
            status = static_cast<int>(cudaMemsetAsync(dgate, 0, static_cast<size_t>(gate_rows * cols) * dtype_bytes(dtype), s));
        }
        return status;
    }
    if (h == nullptr || stats == nullptr || (dy == nullptr && dn == nullptr) || (dn != nullptr && y == nullptr)) {
        return FDL_ERR_INVALID_ARGUMENT;
    }
    if (!aligned16(stats)) return FDL_ERR_INVALID_ARGUMENT;
    if (scratch == nullptr || (reinterpret_cast<uintptr_t>(scratch) & 255u) != 0 ||
        scratch_bytes < fdl_norm_residual_backward_scratch_bytes(rows, cols, gate_rows)) {
        return FDL_ERR_WORKSPACE;
    }
    const DeviceInfo* info = current_device_info(&status);
    if (info == nullptr) return status;
    const BackwardPlan b = backward_plan(rows, cols, gate_rows, info->sm_count);
    NormParams p = {};
    p.dy = dy; p.dn = dn; p.y_in = y; p.h = h; p.stats_in = stats; p.gate = gate;
    p.post_gamma = post_gamma; p.post_beta = post_beta; p.pre_gamma = pre_gamma;
    p.dx = dx; p.dh = dh; p.dgate = dgate;
    p.rows = rows;
    p.rows_per_gate = b.rows_per_gate;
    p.rows_per_task = b.rows_per_task;
    p.tasks_per_gate = b.tasks_per_gate;
    p.tasks = b.tasks;
    p.cols = static_cast<int>(cols);
    p.post_kind = post_kind; p.pre_kind = pre_kind; p.gate_act = gate_act;
    p.residual_scale = residual_scale; p.block_scale = block_scale;
    FoldJobs jobs = {};
    jobs.cols = static_cast<int>(cols);
    int njobs = 0;
    float* at = static_cast<float*>(scratch);
    int64_t groups = 1;
    for (int a = 0; a < 4; ++a) {
        if (sums[a] == nullptr) continue;
        p.partial[a] = at;
        jobs.job[njobs++] = {at, sums[a], FDL_F32, 1, b.teams};
        at += b.teams * cols;
    }
    if (dgate != nullptr && gate_rows != rows && b.tasks_per_gate > 1) {
        p.gate_partial = at;
        jobs.job[njobs++] = {at, dgate, dtype, gate_rows, b.tasks_per_gate};
        groups = gate_rows;
    }
    status = dispatch<LaunchBackward>(dtype, packs_fit(dtype, cols, {dy, dn, y, h, gate, dx, dh, dgate}), b.shape.warp, p,
                                      b.shape, b.grid, s);
    if (status != FDL_OK || njobs == 0) return status;
    const dim3 grid(static_cast<unsigned int>(ceil_div(cols, kFoldX)), static_cast<unsigned int>(njobs),
                    static_cast<unsigned int>(groups < 64 ? groups : 64));
    return launch_ex(norm_fold_kernel, grid, dim3(kFoldX, kFoldY), 0, s, dim3(1, 1, 1), tuning().pdl != 0, jobs);
}

}  // extern "C"
