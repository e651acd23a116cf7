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
//
// Measured on B200 (floors at 6548 GB/s in brackets): forward [16384, 4096] bf16 with a full sigmoid gate 126 us [103],
// [56548, 128] bf16 16 us [11], one row of 4096 4.9 us; backward [16384, 8192] bf16 with a gate for each of 8 runs of
// rows 313 us [246], [16384, 4096] 159 us [123], [2049, 1001] f32 24 us [8], of which the second kernel is about 5.
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
    unsigned int* error_flag;  // host-mapped; ring kernels
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

struct Team {
    TeamSums* sums;
    int phase, warps, cluster, rank;
    __device__ __forceinline__ float2 sum(float a, float b) {
        a = warp_sum(a);
        b = warp_sum(b);
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

// sigmoid and tanh from one exp2 and one reciprocal of the special-function unit (2^-22 and 2^-23): with a
// gate for each element they are a good part of a row's instructions.  tanh near 0, where 1 - 2 / (1 + e^2g)
// would cancel, by its Taylor series (below 1/4 the next term is under 2^-26 of the sum).
__device__ __forceinline__ float rcp_approx(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
template <int N>
__device__ __forceinline__ void gate_values(int act, float (&g)[N]) {  // one branch for the N of them
    if (act == FDL_GATE_SIGMOID) {
#pragma unroll
        for (int e = 0; e < N; ++e) g[e] = rcp_approx(1.0f + ex2_approx(-1.4426950408889634f * g[e]));
    } else if (act == FDL_GATE_TANH) {
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const float far = 1.0f - 2.0f * rcp_approx(1.0f + ex2_approx(2.8853900817779268f * g[e]));
            const float q = g[e] * g[e];
            const float near = g[e] + g[e] * q * (-1.0f / 3 + q * (2.0f / 15 + q * (-17.0f / 315 + q * (62.0f / 2835))));
            g[e] = fabsf(g[e]) < 0.25f ? near : far;
        }
    }
}
// v *= the slope of act, from a = act(g).
template <int N>
__device__ __forceinline__ void times_slope(int act, const float (&a)[N], float (&v)[N]) {
    if (act == FDL_GATE_SIGMOID) {
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] *= a[e] - a[e] * a[e];
    } else if (act == FDL_GATE_TANH) {
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] *= 1.0f - a[e] * a[e];
    }
}

template <int M>
__device__ __forceinline__ void gate_pairs(int act, float2 (&g)[M]) {
    float f[2 * M];
#pragma unroll
    for (int e = 0; e < M; ++e) {
        f[2 * e] = g[e].x;
        f[2 * e + 1] = g[e].y;
    }
    gate_values(act, f);
#pragma unroll
    for (int e = 0; e < M; ++e) g[e] = make_float2(f[2 * e], f[2 * e + 1]);
}
template <int M>
__device__ __forceinline__ void times_slope_pairs(int act, const float2 (&a)[M], float2 (&v)[M]) {
    if (act == FDL_GATE_SIGMOID) {
#pragma unroll
        for (int e = 0; e < M; ++e) v[e] = mul2(v[e], fma2(a[e], make_float2(-a[e].x, -a[e].y), a[e]));
    } else if (act == FDL_GATE_TANH) {
#pragma unroll
        for (int e = 0; e < M; ++e) v[e] = mul2(v[e], fma2(a[e], make_float2(-a[e].x, -a[e].y), both(1.0f)));
    }
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

template <class T, int N, int PACKS>
__global__ void __launch_bounds__(512)
norm_residual_kernel(const NormParams p) {
    __shared__ TeamSums sums;
    Team team{&sums, 0, static_cast<int>(blockDim.x) / kWarp, static_cast<int>(cluster_size()), static_cast<int>(cluster_rank())};
    Owned<N, PACKS> own;
    own.first = team.rank * blockDim.x + threadIdx.x;
    own.stride = team.cluster * blockDim.x;
    if (team.cluster > 1) cluster_sync_all();  // every CTA has started before the first remote store
    pdl_wait();
    for (int64_t row = blockIdx.x / team.cluster; row < p.rows; row += gridDim.x / team.cluster) {
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
                gate_values(p.gate_act, w[k]);
#pragma unroll
                for (int e = 0; e < N; ++e) h[k][e] *= w[k][e];
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
    if (team.cluster > 1) cluster_sync_all();  // no CTA leaves while another may still write its sums
}

// A team takes whole tasks: rows_per_task consecutive rows of one gate row.
template <class T, int N, int PACKS>
__global__ void __launch_bounds__(512)
norm_residual_backward_kernel(const NormParams p) {
    __shared__ TeamSums sums;
    Team team{&sums, 0, static_cast<int>(blockDim.x) / kWarp, static_cast<int>(cluster_size()), static_cast<int>(cluster_rank())};
    Owned<N, PACKS> own;
    own.first = team.rank * blockDim.x + threadIdx.x;
    own.stride = team.cluster * blockDim.x;
    const int64_t id = blockIdx.x / team.cluster, teams = gridDim.x / team.cluster;
    if (team.cluster > 1) cluster_sync_all();  // every CTA has started before the first remote store
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
            for (int k = 0; k < PACKS; ++k) gate_values(p.gate_act, gate[k]);
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
                for (int k = 0; k < PACKS; ++k) gate_values(p.gate_act, gate[k]);
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
                        gsum[k][e] += u[k][e];
                    }
                    if (gate_each) times_slope(p.gate_act, gate[k], u[k]);
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
                times_slope(p.gate_act, gate[k], gsum[k]);
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
    if (team.cluster > 1) cluster_sync_all();  // no CTA leaves while another may still write its sums
}

// ---- rows through shared memory ------------------------------------------------------------------
//
// For more rows than teams, on the 16-byte grid: one thread asks for whole row slices with bulk-async
// copies, a few rows ahead of the row that the CTA works on, so the bytes in flight depend on neither
// registers nor barriers (loads into registers took 337 us forward and 1289 backward where this form takes 126 and
// 313).  What bounds it then is the row's chain of sums -- shuffles, a barrier, shuffles -- and the issue of some 40
// instructions an element pair: 61% of issue slots are busy forward, 48% backward, DRAM half of the time.  Arithmetic goes two floats an instruction: the kernels are near the issue limit.
// Forward, gamma and beta come from L1 row by row (in shared memory they would take the place of a CTA).
// Backward, with half the threads an SM, they lie in shared memory as floats (post_gamma times the block's
// scale and a shared gate); a thread reads and writes only its own columns of them, so no barrier guards them.

constexpr int kMaxStages = 4;
constexpr int kRingRoom = 227 * 1024 - 4096;  // dynamic shared memory of a CTA alone on its SM

struct RingPlan {
    int stages;
    int tiles;    // tensors a stage holds
    int slice;    // what a CTA of the cluster owns of a row: 128-bit packs, or columns (rows off the 16-byte grid)
    int tile;     // 128-bit words of a tensor's place in a stage
    int weights;  // floats of a weight's place
};

template <int NV>
struct RingSums {
    alignas(16) float buf[2][kMaxCluster * kMaxWarps * NV];
    uint64_t full[2];  // clusters: a buffer's values have arrived
};

// A store into CTA `rank`'s copy of `mine`, counted on its copy of `bar`.  A cluster barrier in its place would wait
// for the rows' gradient stores, a microsecond or two at each of a row's sums.  (Launches with clusters only.)
template <int NV>
__device__ __forceinline__ void send(float* mine, uint64_t* bar, uint32_t rank, const float (&v)[NV]) {
    uint32_t to, at;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"(smem_addr(mine)), "r"(rank));
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_addr(bar)), "r"(rank));
    if constexpr (NV == 2) {
        asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v2.f32 [%0], {%1, %2}, [%3];" ::"r"(to), "f"(v[0]),
                     "f"(v[1]), "r"(at)
                     : "memory");
    } else {
        asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.f32 [%0], %1, [%2];" ::"r"(to), "f"(v[0]), "r"(at)
                     : "memory");
    }
}
__device__ __forceinline__ bool mbar_try_wait_cluster(uint64_t* bar, uint32_t parity) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(smem_addr(bar)), "r"(parity)
        : "memory");
    return done != 0;
}

template <int NV>
struct RingTeam {
    RingSums<NV>* sums;
    int phase, warps, cluster, rank;
    uint32_t parity;  // bit i: of buffer i's next round
    bool failed;
    unsigned int* error_flag;

    __device__ __forceinline__ RingTeam(RingSums<NV>* s, unsigned int* flag)
        : sums(s), phase(0), warps(blockDim.x / kWarp), cluster(cluster_size()), rank(cluster_rank()), parity(0), failed(false),
          error_flag(flag) {
        if (threadIdx.x == 0) {
            mbar_init(&sums->full[0], 1);
            mbar_init(&sums->full[1], 1);
        }
    }
    // NV sums over the row's team; the buffers alternate.  A buffer's next values are sent when everybody has sent
    // those of the other one, and so has read it.
    __device__ __forceinline__ void sum(float (&v)[NV]) {
        const int lane = threadIdx.x & (kWarp - 1), warp = threadIdx.x / kWarp;
#pragma unroll
        for (int i = 0; i < NV; ++i) v[i] = warp_sum(v[i]);
        float* at = sums->buf[phase];
        const int n = warps * cluster;
        if (cluster == 1) {
            if (lane == 0) {
#pragma unroll
                for (int i = 0; i < NV; ++i) at[warp * NV + i] = v[i];
            }
            __syncthreads();
        } else {
            uint64_t* bar = &sums->full[phase];
            if (threadIdx.x == 0) mbar_expect_tx(bar, static_cast<uint32_t>(n * NV * sizeof(float)));
            if (lane < cluster) send(&at[(rank * warps + warp) * NV], bar, lane, v);
            bool ok = failed;  // after a wait that ran out there is no more waiting
            for (uint32_t i = 0; i < kMbarSpinLimit && !ok; ++i) ok = mbar_try_wait_cluster(bar, parity >> phase & 1u);
            if (!ok) {
                failed = true;
                atomicOr_system(error_flag, 1u);
            }
            parity ^= 1u << phase;
        }
        phase ^= 1;
        // Each warp folds the partial sums by itself, all in the same order.
#pragma unroll
        for (int i = 0; i < NV; ++i) v[i] = lane < n ? at[lane * NV + i] : 0.0f;
        for (int w = lane + kWarp; w < n; w += kWarp) {
#pragma unroll
            for (int i = 0; i < NV; ++i) v[i] += at[w * NV + i];
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) v[i] = warp_sum(v[i]);
    }
};

// The consumer's side of the ring: waits, with a limit, for the copies of the stage that is next.
struct RingWait {
    uint64_t* full;
    int stages, stage;
    uint32_t parity;
    bool failed;
    __device__ __forceinline__ void wait(unsigned int* error_flag) {
        if (!failed && !mbar_wait_bounded(&full[stage], parity)) {
            failed = true;
            atomicOr_system(error_flag, 1u);
        }
    }
    __device__ __forceinline__ void next() {
        if (++stage == stages) {
            stage = 0;
            parity ^= 1u;
        }
    }
};

// The columns of a thread, N at a time.  VEC: rows are whole packs on the 16-byte grid, and N is a pack's columns.
// Otherwise 8 columns a team's width apart, element by element: every row then starts at another place of
// a 16-byte word, and a tile holds the words that cover it.
template <class T, bool VEC>
struct Columns {
    static constexpr int N = VEC ? kPack<T> : 8, M = N / 2;
    int t, threads;
    int first, count;  // packs (VEC) or columns

    __device__ __forceinline__ int at(int k) const { return t + k * threads; }
    __device__ __forceinline__ bool has(int k) const { return at(k) < count; }
    __device__ __forceinline__ bool inside(int e) const { return VEC || t + e * threads < count; }
    __device__ __forceinline__ int col(int k, int e) const { return VEC ? (first + at(k)) * N + e : first + t + e * threads; }

    // Where a row of this slice begins in memory, and how many bytes its tile takes, from `total` bytes of tensor.
    struct Span {
        size_t from;
        uint32_t bytes;
        int lead;  // elements before the slice's first in the tile
        int safe;  // columns that the tile has (all but the last few of the tensor's last row)
    };
    __device__ __forceinline__ Span span(int64_t row, int cols, int64_t rows) const {
        if (VEC) {
            return {(static_cast<size_t>(row) * cols + static_cast<size_t>(first) * N) * sizeof(T), static_cast<uint32_t>(count) * 16u, 0,
                    count};
        }
        const size_t begin = (static_cast<size_t>(row) * cols + first) * sizeof(T);
        const size_t from = begin & ~static_cast<size_t>(15);
        size_t end = (begin + static_cast<size_t>(count) * sizeof(T) + 15) & ~static_cast<size_t>(15);
        const size_t total = static_cast<size_t>(rows) * cols * sizeof(T) & ~static_cast<size_t>(15);
        if (end > total) end = total;
        return {from, static_cast<uint32_t>(end - from), static_cast<int>((begin - from) / sizeof(T)),
                static_cast<int>((end - begin) / sizeof(T))};
    }
    __device__ __forceinline__ void load(const uint4* tile, const Span& s, const T* row, int k, float2 (&v)[M]) const {
        if constexpr (VEC) {
            unpack2(has(k) ? tile[at(k)] : make_uint4(0, 0, 0, 0), v, T{});
        } else {
            float f[N];
            const T* from = reinterpret_cast<const T*>(tile) + s.lead + t;
#pragma unroll
            for (int e = 0; e < N; ++e) f[e] = inside(e) && t + e * threads < s.safe ? to_f32(from[e * threads]) : 0.0f;
            if (s.safe < count) {
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    if (inside(e) && t + e * threads >= s.safe) f[e] = to_f32(row[col(k, e)]);
                }
            }
#pragma unroll
            for (int e = 0; e < M; ++e) v[e] = make_float2(f[2 * e], f[2 * e + 1]);
        }
    }
    __device__ __forceinline__ void load_row(const T* row, int k, float2 (&v)[M]) const {
        if constexpr (VEC) {
            unpack2(__ldg(reinterpret_cast<const uint4*>(row + col(k, 0))), v, T{});
        } else {
            float f[N];
#pragma unroll
            for (int e = 0; e < N; ++e) f[e] = inside(e) ? to_f32(row[col(k, e)]) : 0.0f;
#pragma unroll
            for (int e = 0; e < M; ++e) v[e] = make_float2(f[2 * e], f[2 * e + 1]);
        }
    }
    // The same from a tensor that the kernel may be writing in place, with 0 outside the row.
    __device__ __forceinline__ void stream(const T* row, int k, float2 (&v)[M]) const {
        if constexpr (VEC) {
            unpack2(has(k) ? __ldcs(reinterpret_cast<const uint4*>(row + col(k, 0))) : make_uint4(0, 0, 0, 0), v, T{});
        } else {
            float f[N];
#pragma unroll
            for (int e = 0; e < N; ++e) f[e] = inside(e) ? to_f32(__ldcs(row + col(k, e))) : 0.0f;
#pragma unroll
            for (int e = 0; e < M; ++e) v[e] = make_float2(f[2 * e], f[2 * e + 1]);
        }
    }
    __device__ __forceinline__ void store(T* row, int k, const float2 (&v)[M]) const {
        if constexpr (VEC) {
            store_pairs(row + col(k, 0), v);
        } else {
#pragma unroll
            for (int e = 0; e < N; ++e) {
                if (inside(e)) __stcs(row + col(k, e), from_f32<T>(e % 2 == 0 ? v[e / 2].x : v[e / 2].y));
            }
        }
    }
    // A weight's floats of these columns (ones where there is no weight, 0 outside the row).
    __device__ __forceinline__ void fetch(const float* w, int k, float2 (&v)[M]) const {
        if constexpr (VEC) {
#pragma unroll
            for (int q = 0; q < M / 2; ++q) {
                const float4 f = w != nullptr ? __ldg(reinterpret_cast<const float4*>(w + col(k, 0)) + q) : make_float4(1.0f, 1.0f, 1.0f, 1.0f);
                v[2 * q] = make_float2(f.x, f.y);
                v[2 * q + 1] = make_float2(f.z, f.w);
            }
        } else {
            float f[N];
#pragma unroll
            for (int e = 0; e < N; ++e) f[e] = !inside(e) ? 0.0f : w != nullptr ? __ldg(w + col(k, e)) : 1.0f;
#pragma unroll
            for (int e = 0; e < M; ++e) v[e] = make_float2(f[2 * e], f[2 * e + 1]);
        }
    }
    // The same floats in shared memory: N / 4 arrays of 128-bit groups (VEC: lanes next to each other read next to
    // each other), or one column after the other.
    __device__ __forceinline__ void keep(float* w, int k, const float2 (&v)[M]) const {
        if constexpr (VEC) {
#pragma unroll
            for (int q = 0; q < M / 2; ++q) {
                reinterpret_cast<float4*>(w)[q * count + at(k)] = make_float4(v[2 * q].x, v[2 * q].y, v[2 * q + 1].x, v[2 * q + 1].y);
            }
        } else {
#pragma unroll
            for (int e = 0; e < N; ++e) w[t + e * threads] = e % 2 == 0 ? v[e / 2].x : v[e / 2].y;
        }
    }
    __device__ __forceinline__ void kept(const float* w, int k, float2 (&v)[M]) const {
        if constexpr (VEC) {
#pragma unroll
            for (int q = 0; q < M / 2; ++q) {
                const float4 f = reinterpret_cast<const float4*>(w)[q * count + at(k)];
                v[2 * q] = make_float2(f.x, f.y);
                v[2 * q + 1] = make_float2(f.z, f.w);
            }
        } else {
#pragma unroll
            for (int e = 0; e < M; ++e) v[e] = make_float2(w[t + 2 * e * threads], w[t + (2 * e + 1) * threads]);
        }
    }
};

// ---- short rows: a part of a warp a row ---------------------------------------------------------------
//
// Rows of up to 256 columns: TEAM lanes a row, 8 columns a lane, 32 / TEAM rows a warp side by side, sums by
// shuffles alone.  The loops have the same length in all lanes of a warp; a team without a row works on the last
// one and stores nothing.

template <int TEAM>
__device__ __forceinline__ float team_sum(float v) {
#pragma unroll
    for (int o = TEAM / 2; o > 0; o >>= 1) v += __shfl_xor_sync(kFullMask, v, o);
    return v;
}

template <int TEAM, class Own, int PACKS, int M>
__device__ __forceinline__ float2 team_moments(int kind, float eps, float inv, const float2 (&v)[PACKS][M], const Own& own) {
    if (kind == FDL_NORM_NONE) return make_float2(0.0f, 1.0f);
    float mean = 0.0f;
    if (kind == FDL_NORM_LAYER) {
        float2 s = both(0.0f);
#pragma unroll
        for (int k = 0; k < PACKS; ++k) {
#pragma unroll
            for (int e = 0; e < M; ++e) s = add2(s, v[k][e]);
        }
        mean = team_sum<TEAM>(s.x + s.y) * inv;
    }
    float2 q = both(0.0f);
#pragma unroll
    for (int k = 0; k < PACKS; ++k) {
#pragma unroll
        for (int e = 0; e < M; ++e) {
            float2 c = add2(v[k][e], both(-mean));
            if (!own.has(k) || !own.inside(2 * e)) c.x = 0.0f;
            if (!own.has(k) || !own.inside(2 * e + 1)) c.y = 0.0f;
            q = fma2(c, c, q);
        }
    }
    return make_float2(mean, rsqrtf(fmaf(team_sum<TEAM>(q.x + q.y), inv, eps)));
}

constexpr int kTeamThreads = 256;

template <class T, int PACKS, bool VEC, int TEAM>
__global__ void __launch_bounds__(kTeamThreads, 4)
norm_residual_team_kernel(const NormParams p) {
    constexpr int M = Columns<T, VEC>::M;
    const int t = threadIdx.x % TEAM;
    const Columns<T, VEC> own{t, TEAM, 0, VEC ? p.cols / kPack<T> : p.cols};
    const float inv = 1.0f / static_cast<float>(p.cols);
    pdl_wait();
    const int64_t step = static_cast<int64_t>(gridDim.x) * (kTeamThreads / TEAM);
    int64_t row = static_cast<int64_t>(blockIdx.x) * (kTeamThreads / TEAM) + threadIdx.x / TEAM;
    for (int64_t first = row - threadIdx.x % kWarp / TEAM; first < p.rows; first += step, row += step) {
        const bool active = row < p.rows;
        const int64_t at = active ? row : p.rows - 1, base = at * p.cols;
        float2 v[PACKS][M], x[PACKS][M], w[M];
#pragma unroll
        for (int k = 0; k < PACKS; ++k) {
            own.stream(static_cast<const T*>(p.h) + base, k, v[k]);
            own.stream(static_cast<const T*>(p.x) + base, k, x[k]);
        }
        const float2 s1 = team_moments<TEAM>(p.post_kind, p.eps, inv, v, own);
        const float2 r1 = both(s1.y * p.block_scale), shift1 = both(-s1.x * s1.y * p.block_scale);
#pragma unroll
        for (int k = 0; k < PACKS; ++k) {
            if (!own.has(k)) continue;
#pragma unroll
            for (int e = 0; e < M; ++e) v[k][e] = fma2(v[k][e], r1, shift1);
            if (p.post_gamma != nullptr) {
                own.fetch(p.post_gamma, k, w);
#pragma unroll
                for (int e = 0; e < M; ++e) v[k][e] = mul2(v[k][e], w[e]);
            }
            if (p.post_beta != nullptr) {
                own.fetch(p.post_beta, k, w);
#pragma unroll
                for (int e = 0; e < M; ++e) v[k][e] = fma2(both(p.block_scale), w[e], v[k][e]);
            }
            if (p.gate != nullptr) {
                own.stream(static_cast<const T*>(p.gate) + (p.rows_per_gate == 1 ? at : at / p.rows_per_gate) * p.cols, k, w);
                gate_pairs(p.gate_act, w);
#pragma unroll
                for (int e = 0; e < M; ++e) v[k][e] = mul2(v[k][e], w[e]);
            }
#pragma unroll
            for (int e = 0; e < M; ++e) {
                v[k][e] = fma2(both(p.residual_scale), x[k][e], v[k][e]);
                if (!own.inside(2 * e)) v[k][e].x = 0.0f;
                if (!own.inside(2 * e + 1)) v[k][e].y = 0.0f;
            }
            if (active) own.store(static_cast<T*>(p.y) + base, k, v[k]);
        }
        const float2 s2 = team_moments<TEAM>(p.pre_kind, p.eps, inv, v, own);
        if (p.stats != nullptr && active && t == 0) {
            reinterpret_cast<float4*>(p.stats)[row] = make_float4(s1.x, s1.y, s2.x, s2.y);
        }
        if (p.n == nullptr || !active) continue;
        const float2 r2 = both(s2.y), shift2 = both(-s2.x * s2.y);
#pragma unroll
        for (int k = 0; k < PACKS; ++k) {
            if (!own.has(k)) continue;
#pragma unroll
            for (int e = 0; e < M; ++e) v[k][e] = fma2(v[k][e], r2, shift2);
            if (p.pre_gamma != nullptr) {
                own.fetch(p.pre_gamma, k, w);
#pragma unroll
                for (int e = 0; e < M; ++e) v[k][e] = mul2(v[k][e], w[e]);
            }
            if (p.pre_beta != nullptr) {
                own.fetch(p.pre_beta, k, w);
#pragma unroll
                for (int e = 0; e < M; ++e) v[k][e] = add2(v[k][e], w[e]);
            }
            own.store(static_cast<T*>(p.n) + base, k, v[k]);
        }
    }
}

// Sums over rows: the teams of a CTA meet in shared memory, so that a CTA leaves one partial row.
template <class T, int PACKS, bool VEC, int TEAM>
__global__ void __launch_bounds__(kTeamThreads, 2)
norm_residual_backward_team_kernel(const NormParams p) {
    constexpr int N = Columns<T, VEC>::N, M = N / 2;
    __shared__ float meet[kTeamThreads * 8];  // [teams][TEAM * 8]
    const int t = threadIdx.x % TEAM;
    const Columns<T, VEC> own{t, TEAM, 0, VEC ? p.cols / kPack<T> : p.cols};
    const float inv = 1.0f / static_cast<float>(p.cols);
    const bool gate_each = p.gate != nullptr && p.rows_per_gate == 1, gate_shared = p.gate != nullptr && !gate_each;
    pdl_wait();
    float2 acc[4][PACKS][M];
#pragma unroll
    for (int a = 0; a < 4; ++a) {
#pragma unroll
        for (int k = 0; k < PACKS; ++k) {
#pragma unroll
            for (int e = 0; e < M; ++e) acc[a][k][e] = both(0.0f);
        }
    }
    const int64_t teams = static_cast<int64_t>(gridDim.x) * (kTeamThreads / TEAM);
    int64_t task = static_cast<int64_t>(blockIdx.x) * (kTeamThreads / TEAM) + threadIdx.x / TEAM;
    const int64_t groups_rows = p.rows_per_gate == 1 ? p.rows : p.rows_per_gate;
    for (int64_t first = task - threadIdx.x % kWarp / TEAM; first < p.tasks; first += teams, task += teams) {
        const bool has_task = task < p.tasks;
        const int64_t one = has_task ? task : p.tasks - 1;
        const int64_t group = p.rows_per_gate == 1 ? 0 : one / p.tasks_per_gate;
        const int64_t from = group * groups_rows + (one - group * p.tasks_per_gate) * p.rows_per_task;
        const int64_t end = (group + 1) * groups_rows;
        float2 gate[PACKS][M], gsum[PACKS][M];
#pragma unroll
        for (int k = 0; k < PACKS; ++k) {
#pragma unroll
            for (int e = 0; e < M; ++e) {
                gate[k][e] = both(1.0f);
                gsum[k][e] = both(0.0f);
            }
            if (gate_shared) {
                own.stream(static_cast<const T*>(p.gate) + group * p.cols, k, gate[k]);
                gate_pairs(p.gate_act, gate[k]);
            }
        }
        for (int64_t i = 0; i < p.rows_per_task; ++i) {
            const bool active = has_task && from + i < end;
            const int64_t row = active ? from + i : 0, base = row * p.cols;
            const float4 st = reinterpret_cast<const float4*>(p.stats_in)[row];
            float2 d[PACKS][M], hat[PACKS][M], dy[PACKS][M], h[PACKS][M], w[M];
#pragma unroll
            for (int k = 0; k < PACKS; ++k) {
#pragma unroll
                for (int e = 0; e < M; ++e) d[k][e] = hat[k][e] = dy[k][e] = both(0.0f);
                if (p.dn != nullptr) {
                    own.stream(static_cast<const T*>(p.dn) + base, k, d[k]);
                    own.stream(static_cast<const T*>(p.y_in) + base, k, hat[k]);
                }
                if (p.dy != nullptr) own.stream(static_cast<const T*>(p.dy) + base, k, dy[k]);
                own.stream(static_cast<const T*>(p.h) + base, k, h[k]);
                if (gate_each) {
                    own.stream(static_cast<const T*>(p.gate) + base, k, gate[k]);
                    gate_pairs(p.gate_act, gate[k]);
                }
            }
            float level = 0.0f, along = 0.0f;
            if (p.dn != nullptr) {
                float2 sd = both(0.0f), sh = both(0.0f);
                const float2 r = both(st.w), shift = both(-st.z * st.w);
#pragma unroll
                for (int k = 0; k < PACKS; ++k) {
                    if (!own.has(k)) continue;
                    if (p.pre_gamma != nullptr) own.fetch(p.pre_gamma, k, w);
#pragma unroll
                    for (int e = 0; e < M; ++e) {
                        hat[k][e] = fma2(hat[k][e], r, shift);
                        if (active) {
                            acc[2][k][e] = fma2(d[k][e], hat[k][e], acc[2][k][e]);
                            acc[3][k][e] = add2(acc[3][k][e], d[k][e]);
                        }
                        if (p.pre_gamma != nullptr) d[k][e] = mul2(d[k][e], w[e]);
                        sd = add2(sd, d[k][e]);
                        sh = fma2(d[k][e], hat[k][e], sh);
                    }
                }
                if (p.pre_kind == FDL_NORM_LAYER) level = team_sum<TEAM>(sd.x + sd.y) * inv;
                along = team_sum<TEAM>(sh.x + sh.y) * inv;
            }
            float2 sd = both(0.0f), sh = both(0.0f);
            const float2 r2 = both(st.w), r1 = both(st.y), shift = both(-st.x * st.y);
#pragma unroll
            for (int k = 0; k < PACKS; ++k) {
                if (!own.has(k)) continue;
#pragma unroll
                for (int e = 0; e < M; ++e) {
                    d[k][e] = fma2(r2, fma2(hat[k][e], both(-along), add2(d[k][e], both(-level))), dy[k][e]);
                    dy[k][e] = mul2(d[k][e], both(p.residual_scale));
                    d[k][e] = mul2(d[k][e], both(p.block_scale));
                    hat[k][e] = fma2(h[k][e], r1, shift);
                    if (!own.inside(2 * e)) d[k][e].x = 0.0f;
                    if (!own.inside(2 * e + 1)) d[k][e].y = 0.0f;
                }
                if (p.dx != nullptr && active) own.store(static_cast<T*>(p.dx) + base, k, dy[k]);
                if (p.dgate != nullptr) {
                    float2 u[M];
                    own.fetch(p.post_gamma, k, u);
#pragma unroll
                    for (int e = 0; e < M; ++e) u[e] = mul2(u[e], hat[k][e]);
                    if (p.post_beta != nullptr) {
                        own.fetch(p.post_beta, k, w);
#pragma unroll
                        for (int e = 0; e < M; ++e) u[e] = add2(u[e], w[e]);
                    }
#pragma unroll
                    for (int e = 0; e < M; ++e) {
                        u[e] = mul2(u[e], d[k][e]);
                        if (active) gsum[k][e] = add2(gsum[k][e], u[e]);
                    }
                    if (gate_each && active) {
                        times_slope_pairs(p.gate_act, gate[k], u);
                        own.store(static_cast<T*>(p.dgate) + base, k, u);
                    }
                }
                if (p.post_gamma != nullptr) own.fetch(p.post_gamma, k, w);
#pragma unroll
                for (int e = 0; e < M; ++e) {
                    d[k][e] = mul2(d[k][e], gate[k][e]);
                    if (active) {
                        acc[0][k][e] = fma2(d[k][e], hat[k][e], acc[0][k][e]);
                        acc[1][k][e] = add2(acc[1][k][e], d[k][e]);
                    }
                    if (p.post_gamma != nullptr) d[k][e] = mul2(d[k][e], w[e]);
                    sd = add2(sd, d[k][e]);
                    sh = fma2(d[k][e], hat[k][e], sh);
                }
            }
            level = p.post_kind == FDL_NORM_LAYER ? team_sum<TEAM>(sd.x + sd.y) * inv : 0.0f;
            along = p.post_kind != FDL_NORM_NONE ? team_sum<TEAM>(sh.x + sh.y) * inv : 0.0f;
            if (p.dh == nullptr || !active) continue;
#pragma unroll
            for (int k = 0; k < PACKS; ++k) {
                if (!own.has(k)) continue;
#pragma unroll
                for (int e = 0; e < M; ++e) d[k][e] = mul2(r1, fma2(hat[k][e], both(-along), add2(d[k][e], both(-level))));
                own.store(static_cast<T*>(p.dh) + base, k, d[k]);
            }
        }
        if (p.dgate == nullptr || !gate_shared || !has_task) continue;
#pragma unroll
        for (int k = 0; k < PACKS; ++k) {
            if (!own.has(k)) continue;
            times_slope_pairs(p.gate_act, gate[k], gsum[k]);
            if (p.gate_partial == nullptr) {
                own.store(static_cast<T*>(p.dgate) + group * p.cols, k, gsum[k]);
                continue;
            }
#pragma unroll
            for (int e = 0; e < N; ++e) {
                if (own.inside(e)) p.gate_partial[task * p.cols + own.col(k, e)] = e % 2 == 0 ? gsum[k][e / 2].x : gsum[k][e / 2].y;
            }
        }
    }
#pragma unroll
    for (int a = 0; a < 4; ++a) {
        if (p.partial[a] == nullptr) continue;
        __syncthreads();
#pragma unroll
        for (int k = 0; k < PACKS; ++k) {
            if (!own.has(k)) continue;
#pragma unroll
            for (int e = 0; e < N; ++e) {
                if (own.inside(e)) meet[threadIdx.x / TEAM * (TEAM * 8) + own.col(k, e)] = e % 2 == 0 ? acc[a][k][e / 2].x : acc[a][k][e / 2].y;
            }
        }
        __syncthreads();
        if (static_cast<int>(threadIdx.x) < p.cols) {
            float s = meet[threadIdx.x];
            for (int g = 1; g < kTeamThreads / TEAM; ++g) s += meet[g * (TEAM * 8) + threadIdx.x];
            p.partial[a][static_cast<int64_t>(blockIdx.x) * p.cols + threadIdx.x] = s;
        }
    }
}

template <class T, int PACKS, bool VEC>
__global__ void __launch_bounds__(512, 2)
norm_residual_ring_kernel(const NormParams p, const RingPlan plan) {
    constexpr int M = Columns<T, VEC>::M;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ RingSums<1> sums;
    __shared__ uint64_t full[kMaxStages];
    RingTeam<1> team(&sums, p.error_flag);
    const int t = threadIdx.x;
    const int units = VEC ? p.cols / kPack<T> : p.cols;
    const Columns<T, VEC> own{t, static_cast<int>(blockDim.x), team.rank * plan.slice, min(plan.slice, units - team.rank * plan.slice)};
    const int64_t teams = gridDim.x / team.cluster, id = blockIdx.x / team.cluster;
    const int64_t from = p.rows * id / teams, to = p.rows * (id + 1) / teams;
    const bool gate_each = p.gate != nullptr && p.rows_per_gate == 1;
    const bool gate_shared = p.gate != nullptr && !gate_each;
    uint4* const stages = reinterpret_cast<uint4*>(smem);  // [stages][tiles][tile]
    if (t == 0) {
        for (int s = 0; s < plan.stages; ++s) mbar_init(&full[s], 1);
        fence_mbar_init();
    }
    if (team.cluster > 1) cluster_sync_all();  // every CTA has started before the first remote store
    else __syncthreads();
    pdl_wait();
    auto request = [&](int64_t row, int stage) {
        const auto span = own.span(row, p.cols, p.rows);
        uint4* tile = stages + static_cast<size_t>(stage) * plan.tiles * plan.tile;
        mbar_expect_tx(&full[stage], static_cast<uint32_t>(plan.tiles) * span.bytes);
        bulk_g2s(tile, static_cast<const unsigned char*>(p.h) + span.from, span.bytes, &full[stage]);
        bulk_g2s(tile + plan.tile, static_cast<const unsigned char*>(p.x) + span.from, span.bytes, &full[stage]);
        if (gate_each) bulk_g2s(tile + 2 * plan.tile, static_cast<const unsigned char*>(p.gate) + span.from, span.bytes, &full[stage]);
    };
    if (t == 0) {
        for (int s = 0; s < plan.stages && from + s < to; ++s) request(from + s, s);
    }
    RingWait ring{full, plan.stages, 0, 0, false};
    const float inv = 1.0f / static_cast<float>(p.cols);
    const float2 residual = both(p.residual_scale);
    const T* gate = nullptr;  // the row of a shared gate
    int64_t gate_left = 0;    // rows that it still serves
    if (gate_shared && from < to) {
        const int64_t group = from / p.rows_per_gate;
        gate = static_cast<const T*>(p.gate) + group * p.cols;
        gate_left = (group + 1) * p.rows_per_gate - from;
    }
    for (int64_t row = from; row < to; ++row) {
        const int64_t base = row * p.cols;
        const auto span = own.span(row, p.cols, p.rows);
        ring.wait(p.error_flag);
        const uint4* tile = stages + ring.stage * plan.tiles * plan.tile;
        float2 v[PACKS][M];
#pragma unroll
        for (int k = 0; k < PACKS; ++k) own.load(tile, span, static_cast<const T*>(p.h) + base, k, v[k]);
        auto moments = [&](int kind) {
            if (kind == FDL_NORM_NONE) return make_float2(0.0f, 1.0f);
            float mean = 0.0f;
            float2 q2 = both(0.0f);
            if (kind == FDL_NORM_LAYER) {
                float2 s2 = both(0.0f);
#pragma unroll
                for (int k = 0; k < PACKS; ++k) {
#pragma unroll
                    for (int e = 0; e < M; ++e) s2 = add2(s2, v[k][e]);
                }
                float s[1] = {s2.x + s2.y};
                team.sum(s);
                mean = s[0] * inv;
#pragma unroll
                for (int k = 0; k < PACKS; ++k) {
                    if (!own.has(k)) continue;
#pragma unroll
                    for (int e = 0; e < M; ++e) {
                        float2 c = add2(v[k][e], both(-mean));
                        if (!own.inside(2 * e)) c.x = 0.0f;
                        if (!own.inside(2 * e + 1)) c.y = 0.0f;
                        q2 = fma2(c, c, q2);
                    }
                }
            } else {
#pragma unroll
                for (int k = 0; k < PACKS; ++k) {
#pragma unroll
                    for (int e = 0; e < M; ++e) q2 = fma2(v[k][e], v[k][e], q2);
                }
            }
            float q[1] = {q2.x + q2.y};
            team.sum(q);
            return make_float2(mean, rsqrtf(fmaf(q[0], inv, p.eps)));
        };
        const float2 s1 = moments(p.post_kind);
        // (h - mean) * r * gamma * block_scale: the scale goes into r
        const float2 r1 = both(s1.y * p.block_scale), shift1 = both(-s1.x * s1.y * p.block_scale);
#pragma unroll
        for (int k = 0; k < PACKS; ++k) {
            if (!own.has(k)) continue;
            float2 w[M];
#pragma unroll
            for (int e = 0; e < M; ++e) v[k][e] = fma2(v[k][e], r1, shift1);
            if (p.post_gamma != nullptr) {
                own.fetch(p.post_gamma, k, w);
#pragma unroll
                for (int e = 0; e < M; ++e) v[k][e] = mul2(v[k][e], w[e]);
            }
            if (p.post_beta != nullptr) {
                own.fetch(p.post_beta, k, w);
#pragma unroll
                for (int e = 0; e < M; ++e) v[k][e] = fma2(both(p.block_scale), w[e], v[k][e]);
            }
            if (p.gate != nullptr) {
                if (gate_each) own.load(tile + 2 * plan.tile, span, static_cast<const T*>(p.gate) + base, k, w);
                else own.load_row(gate, k, w);
                gate_pairs(p.gate_act, w);
#pragma unroll
                for (int e = 0; e < M; ++e) v[k][e] = mul2(v[k][e], w[e]);
            }
            own.load(tile + plan.tile, span, static_cast<const T*>(p.x) + base, k, w);
#pragma unroll
            for (int e = 0; e < M; ++e) {
                v[k][e] = fma2(residual, w[e], v[k][e]);
                if (!own.inside(2 * e)) v[k][e].x = 0.0f;
                if (!own.inside(2 * e + 1)) v[k][e].y = 0.0f;
            }
            own.store(static_cast<T*>(p.y) + base, k, v[k]);
        }
        const float2 s2 = moments(p.pre_kind);
        if (p.pre_kind == FDL_NORM_NONE) __syncthreads();
        // Behind a barrier that follows the use of everything that was loaded from the stage.
        if (t == 0 && row + plan.stages < to && !ring.failed) request(row + plan.stages, ring.stage);
        if (p.stats != nullptr && t == 0 && team.rank == 0) {
            reinterpret_cast<float4*>(p.stats)[row] = make_float4(s1.x, s1.y, s2.x, s2.y);
        }
        if (p.n != nullptr) {
            const float2 r2 = both(s2.y), shift2 = both(-s2.x * s2.y);
#pragma unroll
            for (int k = 0; k < PACKS; ++k) {
                if (!own.has(k)) continue;
                float2 w[M];
#pragma unroll
                for (int e = 0; e < M; ++e) v[k][e] = fma2(v[k][e], r2, shift2);
                if (p.pre_gamma != nullptr) {
                    own.fetch(p.pre_gamma, k, w);
#pragma unroll
                    for (int e = 0; e < M; ++e) v[k][e] = mul2(v[k][e], w[e]);
                }
                if (p.pre_beta != nullptr) {
                    own.fetch(p.pre_beta, k, w);
#pragma unroll
                    for (int e = 0; e < M; ++e) v[k][e] = add2(v[k][e], w[e]);
                }
                own.store(static_cast<T*>(p.n) + base, k, v[k]);
            }
        }
        if (gate_shared && --gate_left == 0) {
            gate += p.cols;
            gate_left = p.rows_per_gate;
        }
        ring.next();
    }
    if (team.cluster > 1) cluster_sync_all();  // no CTA leaves while another may still write its sums
}

// BETA: sums for post_beta / pre_beta (and for a shared gate's share of post_beta) are kept.
// Per task: s1 = sum D a hat(h), s0 = sum D a, with a = 1 where the gate is shared -- its factor, like the
// block's scale, comes in when the task ends: dpost_gamma += scale a s1, dgate = scale act' (gamma s1 + beta s0).
template <class T, int PACKS, bool BETA, bool VEC>
__global__ void __launch_bounds__(512, 1)
norm_residual_backward_ring_kernel(const NormParams p, const RingPlan plan) {
    constexpr int N = Columns<T, VEC>::N, M = N / 2;
    constexpr int MB = BETA ? M : 1;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ RingSums<2> sums;
    __shared__ uint64_t full[kMaxStages];
    __shared__ alignas(16) float4 stat[kMaxStages];  // the rows' statistics, beside their stages
    RingTeam<2> team(&sums, p.error_flag);
    const int t = threadIdx.x;
    const int units = VEC ? p.cols / kPack<T> : p.cols;
    const Columns<T, VEC> own{t, static_cast<int>(blockDim.x), team.rank * plan.slice, min(plan.slice, units - team.rank * plan.slice)};
    const int64_t teams = gridDim.x / team.cluster, id = blockIdx.x / team.cluster;
    const bool gate_each = p.gate != nullptr && p.rows_per_gate == 1;
    const bool gate_shared = p.gate != nullptr && !gate_each;
    uint4* const stages = reinterpret_cast<uint4*>(smem);  // [stages][tiles][tile]
    float* const w1 = reinterpret_cast<float*>(stages + static_cast<size_t>(plan.stages) * plan.tiles * plan.tile);
    float* const w2 = w1 + plan.weights;
    // Places of the tensors in a stage; an absent one has none.
    const int at_dn = 0, at_y = 1;
    const int at_h = p.dn != nullptr ? 2 : 0;
    const int at_dy = at_h + 1;
    const int at_gate = at_dy + (p.dy != nullptr ? 1 : 0);
    if (t == 0) {
        for (int s = 0; s < plan.stages; ++s) mbar_init(&full[s], 1);
        fence_mbar_init();
    }
    if (team.cluster > 1) cluster_sync_all();  // every CTA has started before the first remote store
    else __syncthreads();
    pdl_wait();
    auto task_rows = [&](int64_t task, int64_t* begin, int64_t* end) {
        const int64_t group = p.rows_per_gate == 1 ? 0 : task / p.tasks_per_gate;
        const int64_t rows = p.rows_per_gate == 1 ? p.rows : p.rows_per_gate;
        *begin = group * rows + (task - group * p.tasks_per_gate) * p.rows_per_task;
        const int64_t stop = (group + 1) * rows;
        *end = *begin + p.rows_per_task < stop ? *begin + p.rows_per_task : stop;
    };
    // The producer's own place in the same order of rows (thread 0).
    int64_t ask_task = id, ask_row = 0, ask_end = 0;
    if (ask_task < p.tasks) task_rows(ask_task, &ask_row, &ask_end);
    auto request = [&](int stage) {
        if (ask_task >= p.tasks) return;
        const auto span = own.span(ask_row, p.cols, p.rows);
        uint4* tile = stages + static_cast<size_t>(stage) * plan.tiles * plan.tile;
        uint64_t* bar = &full[stage];
        mbar_expect_tx(bar, static_cast<uint32_t>(plan.tiles) * span.bytes + 16u);
        bulk_g2s(&stat[stage], p.stats_in + 4 * ask_row, 16u, bar);
        auto ask = [&](int place, const void* tensor) {
            bulk_g2s(tile + place * plan.tile, static_cast<const unsigned char*>(tensor) + span.from, span.bytes, bar);
        };
        if (p.dn != nullptr) {
            ask(at_dn, p.dn);
            ask(at_y, p.y_in);
        }
        ask(at_h, p.h);
        if (p.dy != nullptr) ask(at_dy, p.dy);
        if (gate_each) ask(at_gate, p.gate);
        if (++ask_row == ask_end) {
            ask_task += teams;
            if (ask_task < p.tasks) task_rows(ask_task, &ask_row, &ask_end);
        }
    };
    if (t == 0) {
        for (int s = 0; s < plan.stages; ++s) request(s);
    }
    float2 s1[PACKS][M], s0[PACKS][MB], a2[PACKS][M], a3[PACKS][MB];
#pragma unroll
    for (int k = 0; k < PACKS; ++k) {
#pragma unroll
        for (int e = 0; e < M; ++e) {
            s1[k][e] = a2[k][e] = both(0.0f);
            s0[k][e % MB] = a3[k][e % MB] = both(0.0f);
        }
        if (own.has(k)) {
            float2 w[M];
            own.fetch(p.post_gamma, k, w);
#pragma unroll
            for (int e = 0; e < M; ++e) w[e] = mul2(w[e], both(p.block_scale));
            own.keep(w1, k, w);
            own.fetch(p.pre_gamma, k, w);
            own.keep(w2, k, w);
        }
    }
    RingWait ring{full, plan.stages, 0, 0, false};
    const float inv = 1.0f / static_cast<float>(p.cols);
    bool flushed = false;  // the team's partial rows of post gamma / beta hold something
    for (int64_t task = id; task < p.tasks; task += teams) {
        int64_t from, to;
        task_rows(task, &from, &to);
        const int64_t group = task / p.tasks_per_gate;  // of a shared gate
        if (gate_shared) {
#pragma unroll
            for (int k = 0; k < PACKS; ++k) {
                if (!own.has(k)) continue;
                float2 g[M], w[M];
                own.load_row(static_cast<const T*>(p.gate) + group * p.cols, k, g);
                gate_pairs(p.gate_act, g);
                own.fetch(p.post_gamma, k, w);
#pragma unroll
                for (int e = 0; e < M; ++e) w[e] = mul2(mul2(w[e], both(p.block_scale)), g[e]);
                own.keep(w1, k, w);
            }
        }
        for (int64_t row = from; row < to; ++row) {
            ring.wait(p.error_flag);
            const uint4* tile = stages + static_cast<size_t>(ring.stage) * plan.tiles * plan.tile;
            const float4 st = stat[ring.stage];
            const int64_t base = row * p.cols;
            const auto span = own.span(row, p.cols, p.rows);
            auto fetch = [&](int place, const void* tensor, int k, float2 (&v)[M]) {
                own.load(tile + place * plan.tile, span, static_cast<const T*>(tensor) + base, k, v);
            };
            float2 d[PACKS][M], hat[PACKS][M];
            float level = 0.0f, along = 0.0f;
            if (p.dn != nullptr) {
                float2 sd = both(0.0f), sh = both(0.0f);
                const float2 r = both(st.w), shift = both(-st.z * st.w);
#pragma unroll
                for (int k = 0; k < PACKS; ++k) {
                    if (own.has(k)) {
                        float2 w[M];
                        fetch(at_dn, p.dn, k, d[k]);
                        fetch(at_y, p.y_in, k, hat[k]);
                        own.kept(w2, k, w);
#pragma unroll
                        for (int e = 0; e < M; ++e) {
                            hat[k][e] = fma2(hat[k][e], r, shift);
                            a2[k][e] = fma2(d[k][e], hat[k][e], a2[k][e]);
                            if (BETA) a3[k][e % MB] = add2(a3[k][e % MB], d[k][e]);
                            d[k][e] = mul2(d[k][e], w[e]);
                            sd = add2(sd, d[k][e]);
                            sh = fma2(d[k][e], hat[k][e], sh);
                        }
                    } else {
#pragma unroll
                        for (int e = 0; e < M; ++e) d[k][e] = hat[k][e] = both(0.0f);
                    }
                }
                float s[2] = {sd.x + sd.y, sh.x + sh.y};
                team.sum(s);
                level = p.pre_kind == FDL_NORM_LAYER ? s[0] * inv : 0.0f;
                along = s[1] * inv;
            } else {
#pragma unroll
                for (int k = 0; k < PACKS; ++k) {
#pragma unroll
                    for (int e = 0; e < M; ++e) d[k][e] = hat[k][e] = both(0.0f);
                }
            }
            float2 sd = both(0.0f), sh = both(0.0f);
            {
                const float2 r1 = both(st.y), shift = both(-st.x * st.y), r2 = both(st.w);
                const float2 down = both(-along), lower = both(-level);
#pragma unroll
                for (int k = 0; k < PACKS; ++k) {
                    if (!own.has(k)) continue;
                    float2 w[M];
                    // D, and dx
                    if (p.dy != nullptr) {
                        fetch(at_dy, p.dy, k, w);
#pragma unroll
                        for (int e = 0; e < M; ++e) d[k][e] = fma2(r2, fma2(hat[k][e], down, add2(d[k][e], lower)), w[e]);
                    } else {
#pragma unroll
                        for (int e = 0; e < M; ++e) d[k][e] = mul2(r2, fma2(hat[k][e], down, add2(d[k][e], lower)));
                    }
                    if (p.dx != nullptr) {
#pragma unroll
                        for (int e = 0; e < M; ++e) w[e] = mul2(both(p.residual_scale), d[k][e]);
                        own.store(static_cast<T*>(p.dx) + base, k, w);
                    }
                    fetch(at_h, p.h, k, hat[k]);
#pragma unroll
                    for (int e = 0; e < M; ++e) hat[k][e] = fma2(hat[k][e], r1, shift);
                    float2 scale[M];
                    own.kept(w1, k, scale);  // block_scale * gamma (* a shared gate)
                    if (gate_each) {
                        float2 a[M];
                        fetch(at_gate, p.gate, k, a);
                        gate_pairs(p.gate_act, a);
                        if (p.dgate != nullptr) {
                            if (BETA && p.post_beta != nullptr) {
                                own.fetch(p.post_beta, k, w);
#pragma unroll
                                for (int e = 0; e < M; ++e) w[e] = mul2(d[k][e], fma2(hat[k][e], scale[e], mul2(both(p.block_scale), w[e])));
                            } else {
#pragma unroll
                                for (int e = 0; e < M; ++e) w[e] = mul2(d[k][e], mul2(hat[k][e], scale[e]));
                            }
                            times_slope_pairs(p.gate_act, a, w);
                            own.store(static_cast<T*>(p.dgate) + base, k, w);
                        }
#pragma unroll
                        for (int e = 0; e < M; ++e) d[k][e] = mul2(d[k][e], a[e]);
                    }
#pragma unroll
                    for (int e = 0; e < M; ++e) {
                        s1[k][e] = fma2(d[k][e], hat[k][e], s1[k][e]);
                        if (BETA) s0[k][e % MB] = add2(s0[k][e % MB], d[k][e]);
                        d[k][e] = mul2(d[k][e], scale[e]);
                        sd = add2(sd, d[k][e]);
                        sh = fma2(d[k][e], hat[k][e], sh);
                    }
                }
            }
            float s[2] = {sd.x + sd.y, sh.x + sh.y};
            team.sum(s);  // (also where no norm needs it: the sums need all that was loaded)
            if (t == 0 && !ring.failed) request(ring.stage);  // everybody's loads of the stage have returned
            if (p.dh != nullptr) {
                level = p.post_kind == FDL_NORM_LAYER ? s[0] * inv : 0.0f;
                along = p.post_kind != FDL_NORM_NONE ? s[1] * inv : 0.0f;
                const float2 r1 = both(st.y), down = both(-along), lower = both(-level);
#pragma unroll
                for (int k = 0; k < PACKS; ++k) {
                    if (!own.has(k)) continue;
#pragma unroll
                    for (int e = 0; e < M; ++e) d[k][e] = mul2(r1, fma2(hat[k][e], down, add2(d[k][e], lower)));
                    own.store(static_cast<T*>(p.dh) + base, k, d[k]);
                }
            }
            ring.next();
        }
        // The end of a task, or of the team's work: the sums under one shared gate.
        const bool last = task + teams >= p.tasks;
        if (!gate_shared && !last) continue;
#pragma unroll
        for (int k = 0; k < PACKS; ++k) {
            if (!own.has(k)) continue;
            float2 g[M], a[M];
            if (gate_shared) {
                own.load_row(static_cast<const T*>(p.gate) + group * p.cols, k, a);
                gate_pairs(p.gate_act, a);
            } else {
#pragma unroll
                for (int e = 0; e < M; ++e) a[e] = both(1.0f);
            }
#pragma unroll
            for (int e = 0; e < M; ++e) g[e] = both(0.0f);
            if (gate_shared && p.dgate != nullptr) {
                own.fetch(p.post_gamma, k, g);
#pragma unroll
                for (int e = 0; e < M; ++e) g[e] = mul2(g[e], s1[k][e]);
                if (BETA && p.post_beta != nullptr) {
                    float2 b[M];
                    own.fetch(p.post_beta, k, b);
#pragma unroll
                    for (int e = 0; e < M; ++e) g[e] = fma2(b[e], s0[k][e % MB], g[e]);
                }
#pragma unroll
                for (int e = 0; e < M; ++e) g[e] = mul2(g[e], both(p.block_scale));
                times_slope_pairs(p.gate_act, a, g);
                if (p.gate_partial == nullptr) own.store(static_cast<T*>(p.dgate) + group * p.cols, k, g);
            }
#pragma unroll
            for (int e = 0; e < N; ++e) {
                if (!own.inside(e)) continue;
                const int c = own.col(k, e);
                const float f = (e % 2 == 0 ? s1[k][e / 2].x * a[e / 2].x : s1[k][e / 2].y * a[e / 2].y) * p.block_scale;
                const float b = !BETA ? 0.0f : (e % 2 == 0 ? s0[k][e / 2 % MB].x * a[e / 2].x : s0[k][e / 2 % MB].y * a[e / 2].y) * p.block_scale;
                float* const pg = p.partial[0] != nullptr ? p.partial[0] + id * p.cols + c : nullptr;
                float* const pb = p.partial[1] != nullptr ? p.partial[1] + id * p.cols + c : nullptr;
                if (pg != nullptr) *pg = (flushed ? *pg : 0.0f) + f;
                if (pb != nullptr) *pb = (flushed ? *pb : 0.0f) + b;
                if (gate_shared && p.gate_partial != nullptr) p.gate_partial[task * p.cols + c] = e % 2 == 0 ? g[e / 2].x : g[e / 2].y;
            }
#pragma unroll
            for (int e = 0; e < M; ++e) {
                s1[k][e] = both(0.0f);
                if (BETA) s0[k][e % MB] = both(0.0f);
            }
        }
        flushed = true;
    }
#pragma unroll
    for (int k = 0; k < PACKS; ++k) {
        if (!own.has(k)) continue;
#pragma unroll
        for (int e = 0; e < N; ++e) {
            if (!own.inside(e)) continue;
            const int64_t c = id * p.cols + own.col(k, e);
            if (p.partial[2] != nullptr) p.partial[2][c] = e % 2 == 0 ? a2[k][e / 2].x : a2[k][e / 2].y;
            if (BETA && p.partial[3] != nullptr) p.partial[3][c] = e % 2 == 0 ? a3[k][e / 2 % MB].x : a3[k][e / 2 % MB].y;
            if (!flushed) {  // a team without a task
                if (p.partial[0] != nullptr) p.partial[0][c] = 0.0f;
                if (p.partial[1] != nullptr) p.partial[1][c] = 0.0f;
            }
        }
    }
    if (team.cluster > 1) cluster_sync_all();  // no CTA leaves while another may still write its sums
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

// 32 columns a CTA, blockDim.y strands of rows each: eight loads of a strand are on their way at a time, so the host
// takes more strands for more rows (a multiple of four).  The strands' sums are added four at a time: one after another,
// 32 of them took 0.7 us of the 24.7 of 2049 rows of 1001 floats.  16 columns a CTA with twice the strands: 24.3 there
// (from 24.0) and 317 (from 313) for 16384 rows of 8192; twice the strands alone 24.0 and 328.
constexpr int kFoldX = 32, kFoldY = 32;

__global__ void __launch_bounds__(kFoldX * kFoldY)
norm_fold_kernel(const FoldJobs jobs) {
    __shared__ float red[kFoldY][kFoldX + 1];
    const FoldJob job = jobs.job[blockIdx.y];
    const int c = blockIdx.x * kFoldX + threadIdx.x, strands = blockDim.y;
    pdl_wait();
    for (int64_t g = blockIdx.z; g < job.groups; g += gridDim.z) {
        float s = 0.0f;
        if (c < jobs.cols) {
#pragma unroll 8
            for (int64_t r = threadIdx.y; r < job.each; r += strands) s += job.part[(g * job.each + r) * jobs.cols + c];
        }
        red[threadIdx.y][threadIdx.x] = s;
        __syncthreads();
        if (threadIdx.y == 0 && c < jobs.cols) {
            float t[4] = {red[0][threadIdx.x], red[1][threadIdx.x], red[2][threadIdx.x], red[3][threadIdx.x]};
#pragma unroll 7
            for (int k = 4; k < strands; k += 4) {
#pragma unroll
                for (int i = 0; i < 4; ++i) t[i] += red[k + i][threadIdx.x];
            }
            s = (t[0] + t[1]) + (t[2] + t[3]);
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
constexpr int kTeamCols = kWarp * kPerThread;
constexpr int kMaxCols = kMaxCluster * 512 * kPerThread;

struct Shape {
    int team;      // lanes of a row's team; 0: CTAs
    int threads;   // of a CTA
    int cluster;   // CTAs a row
    int blocks;    // CTAs that an SM is given
    int rows() const { return team != 0 ? threads / team : 1; }  // of a CTA (or cluster) at a time
};

Shape shape_of(int64_t cols, bool backward) {
    if (cols <= kTeamCols) return {cols <= 8 * kPerThread ? 8 : cols <= 16 * kPerThread ? 16 : 32, kTeamThreads, 1, backward ? 2 : 4};
    int cluster = 1;
    while (cols > static_cast<int64_t>(cluster) * 512 * kPerThread) cluster *= 2;
    const int threads = static_cast<int>(ceil_div(ceil_div(cols, static_cast<int64_t>(cluster) * kPerThread), kWarp)) * kWarp;
    return {0, threads, cluster, 1024 / threads < 1 ? 1 : 1024 / threads};
}

// The ring form: columns of a CTA, its threads and its stages; stages == 0: does not fit.
struct RingShape {
    int threads, cluster, blocks, per_thread;  // CTAs a row, CTAs an SM, columns a thread
    bool vec;                                  // whole packs a row
    RingPlan plan;
    size_t smem;
};

// A thread owns 8 columns, or 16 of a 16-bit type (two packs: the sums' instructions are shared by more
// columns) -- but not for sums for the betas, whose registers would spill, nor where columns go one by one.  Stages
// take what is left of the shared memory of an SM, shared by as many CTAs as 1024 threads make (backward: 512,
// with 128 registers each).
RingShape ring_shape(int64_t cols, int dtype, int tiles, int weights, bool backward, bool beta) {
    RingShape r = {};
    const int size = static_cast<int>(dtype_bytes(dtype)), n = 16 / size;
    if (cols <= kTeamCols) return r;  // a team of lanes a row
    r.vec = cols % n == 0;
    r.per_thread = r.vec && dtype != FDL_F32 && !beta ? 16 : 8;
    r.cluster = 1;
    while (cols > static_cast<int64_t>(r.cluster) * 512 * r.per_thread) r.cluster *= 2;
    r.plan.tiles = tiles;
    if (r.vec) {
        r.plan.slice = r.plan.tile = static_cast<int>(ceil_div(cols / n, r.cluster));
        r.threads = static_cast<int>(ceil_div(ceil_div(r.plan.slice, r.per_thread / n), kWarp)) * kWarp;
        r.plan.weights = r.plan.slice * n;
    } else {
        r.plan.slice = static_cast<int>(ceil_div(cols, r.cluster));
        r.plan.tile = (r.plan.slice * size + 30) / 16;  // any 16-byte words that cover the columns
        r.threads = static_cast<int>(ceil_div(ceil_div(r.plan.slice, r.per_thread), kWarp)) * kWarp;
        r.plan.weights = r.threads * 8;
    }
    const int budget = backward ? 512 : 1024;
    r.blocks = budget / r.threads < 1 ? 1 : budget / r.threads > 16 ? 16 : budget / r.threads;
    const size_t fixed = static_cast<size_t>(r.plan.weights) * 4 * weights;
    const size_t stage = static_cast<size_t>(r.plan.tile) * 16 * tiles;
    for (; r.blocks >= 1; --r.blocks) {  // fewer CTAs where less than two stages would fit
        const size_t room = static_cast<size_t>(kRingRoom + 4096) / r.blocks - 4096;
        if (room < fixed + 2 * stage) continue;
        const size_t most = (room - fixed) / stage;
        r.plan.stages = most > kMaxStages ? kMaxStages : static_cast<int>(most);
        break;
    }
    if (r.blocks < 1) r.blocks = 1;
    r.smem = fixed + stage * r.plan.stages;
    return r;
}

// Backward: which form, and how the rows are dealt out.
struct BackwardPlan {
    bool ring;
    Shape shape;      // direct form
    RingShape rshape; // ring form
    int64_t grid;     // CTAs
    int64_t partials; // partial rows of the sums over rows: one a CTA (or cluster)
    int64_t rows_per_gate, tasks_per_gate, rows_per_task, tasks;
};

// Tasks: every team gets about the same number of rows, and no task crosses a gate row's rows.
BackwardPlan backward_plan(int64_t rows, int64_t cols, int64_t gate_rows, int sm_count, const RingShape* ring) {
    BackwardPlan b = {};
    b.shape = shape_of(cols, true);
    b.ring = ring != nullptr;
    if (ring != nullptr) b.rshape = *ring;
    const int cluster = b.ring ? b.rshape.cluster : b.shape.cluster;
    const int64_t per_cta = b.ring ? 1 : b.shape.rows();
    const int64_t slots = static_cast<int64_t>(sm_count) * (b.ring ? b.rshape.blocks : b.shape.blocks) / cluster;  // (clusters of) CTAs
    const int64_t most = (slots < 1 ? 1 : slots) * per_cta;                                                        // teams at once
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
    b.partials = ceil_div(b.tasks < most ? b.tasks : most, per_cta);
    b.grid = b.partials * cluster;
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

int launch_direct(bool backward, int dtype, bool vec, const NormParams& p, const Shape& s, int64_t grid, cudaStream_t stream) {
    return with_dtype(dtype, [&](auto* tag) {
        using T = std::remove_pointer_t<decltype(tag)>;
        constexpr int N = kPack<T>;
        auto launch = [&](auto forward_kernel, auto backward_kernel) {
            return launch_ex(backward ? backward_kernel : forward_kernel, dim3(static_cast<unsigned int>(grid)), dim3(s.threads), 0, stream,
                             dim3(s.cluster, 1, 1), tuning().pdl != 0, p);
        };
        if (s.team == 0) {
            return vec ? launch(norm_residual_kernel<T, N, kPerThread / N>, norm_residual_backward_kernel<T, N, kPerThread / N>)
                       : launch(norm_residual_kernel<T, 1, kPerThread>, norm_residual_backward_kernel<T, 1, kPerThread>);
        }
        auto team = [&](auto lanes) {
            constexpr int L = decltype(lanes)::value;
            return vec ? launch(norm_residual_team_kernel<T, kPerThread / N, true, L>, norm_residual_backward_team_kernel<T, kPerThread / N, true, L>)
                       : launch(norm_residual_team_kernel<T, 1, false, L>, norm_residual_backward_team_kernel<T, 1, false, L>);
        };
        if (s.team == 8) return team(std::integral_constant<int, 8>{});
        if (s.team == 16) return team(std::integral_constant<int, 16>{});
        return team(std::integral_constant<int, 32>{});
    });
}

template <class K, class... Args>
int launch_ring(K kernel, const NormParams& p, const RingShape& r, int64_t grid, cudaStream_t stream) {
    // (the most that a shape takes, not this one's: another thread may be between its own two calls)
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kRingRoom);
    if (e != cudaSuccess) return static_cast<int>(e);
    return launch_ex(kernel, dim3(static_cast<unsigned int>(grid)), dim3(r.threads), r.smem, stream, dim3(r.cluster, 1, 1),
                     tuning().pdl != 0, p, r.plan);
}

int launch_ring_forward(int dtype, const NormParams& p, const RingShape& r, int64_t grid, cudaStream_t stream) {
    return with_dtype(dtype, [&](auto* tag) {
        using T = std::remove_pointer_t<decltype(tag)>;
        return r.vec ? launch_ring(norm_residual_ring_kernel<T, 2, true>, p, r, grid, stream)
                     : launch_ring(norm_residual_ring_kernel<T, 1, false>, p, r, grid, stream);
    });
}

int launch_ring_backward(int dtype, bool beta, const NormParams& p, const RingShape& r, int64_t grid, cudaStream_t stream) {
    return with_dtype(dtype, [&](auto* tag) {
        using T = std::remove_pointer_t<decltype(tag)>;
        if (!r.vec) {
            return beta ? launch_ring(norm_residual_backward_ring_kernel<T, 1, true, false>, p, r, grid, stream)
                        : launch_ring(norm_residual_backward_ring_kernel<T, 1, false, false>, p, r, grid, stream);
        }
        return beta ? launch_ring(norm_residual_backward_ring_kernel<T, 8 / kPack<T>, true, true>, p, r, grid, stream)
                    : launch_ring(norm_residual_backward_ring_kernel<T, 2, false, true>, p, r, grid, stream);
    });
}

// Whether the ring form can take its tensors: those that it copies start on the 16-byte grid, and with whole packs a
// row so does everything else (`others`).
bool ring_fits(const RingShape& r, std::initializer_list<const void*> copied, std::initializer_list<const void*> others) {
    if (r.plan.stages < 2) return false;
    for (const void* t : copied) {
        if (!aligned16(t)) return false;
    }
    for (const void* t : others) {
        if (r.vec && !aligned16(t)) return false;
    }
    return true;
}

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
    const bool vec = packs_fit(dtype, cols, {x, h, gate, y, n, post_gamma, post_beta, pre_gamma, pre_beta});
    const Shape s = shape_of(cols, false);
    const RingShape r = ring_shape(cols, dtype, 2 + (gate != nullptr && gate_rows == rows), 0, false, false);
    if (ring_fits(r, {x, h, gate}, {y, n, post_gamma, post_beta, pre_gamma, pre_beta})) {
        const int64_t teams = static_cast<int64_t>(info->sm_count) * r.blocks / r.cluster;
        if (rows > teams) {  // (for one row a team the copies ahead have nothing to run ahead of)
            status = error_flag_device_ptr(&p.error_flag);
            if (status != FDL_OK) return status;
            return launch_ring_forward(dtype, p, r, teams * r.cluster, as_stream(stream));
        }
    }
    const int64_t slots = static_cast<int64_t>(info->sm_count) * s.blocks / s.cluster;
    const int64_t work = ceil_div(rows, static_cast<int64_t>(s.rows()));
    const int64_t grid = (work < slots ? work : slots < 1 ? 1 : slots) * s.cluster;
    return launch_direct(false, dtype, vec, p, s, grid, as_stream(stream));
}

// Room for whichever form the call takes: the direct form, or the ring form with any of its tiles and types.
size_t fdl_norm_residual_backward_scratch_bytes(int64_t rows, int64_t cols, int64_t gate_rows) {
    if (rows <= 0 || cols <= 0 || cols > kMaxCols || gate_rows < 0) return 0;
    if (gate_rows > 0 && (gate_rows > rows || rows % gate_rows != 0)) return 0;
    int status = FDL_OK;
    const DeviceInfo* info = current_device_info(&status);
    const int sms = info == nullptr ? 148 : info->sm_count;
    int64_t floats = 0;
    auto add = [&](const RingShape* r) {
        const BackwardPlan b = backward_plan(rows, cols, gate_rows, sms, r);
        const int64_t gate_part = gate_rows == 0 || gate_rows == rows || b.tasks_per_gate == 1 ? 0 : b.tasks;
        const int64_t f = (4 * b.partials + gate_part) * cols;
        if (f > floats) floats = f;
    };
    add(nullptr);
    for (int dtype : {static_cast<int>(FDL_F32), static_cast<int>(FDL_BF16)}) {
        for (int tiles = 2; tiles <= 5; ++tiles) {
            for (int few = 0; few < 2; ++few) {
                const RingShape r = ring_shape(cols, dtype, tiles, 2, true, few == 0);
                if (r.plan.stages >= 2) add(&r);
            }
        }
    }
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
    const bool vec = packs_fit(dtype, cols, {dy, dn, y, h, gate, dx, dh, dgate, post_gamma, post_beta, pre_gamma});
    const bool beta = dpost_beta != nullptr || dpre_beta != nullptr || (post_beta != nullptr && dgate != nullptr);
    const int tiles = 1 + (dn != nullptr ? 2 : 0) + (dy != nullptr) + (gate != nullptr && gate_rows == rows);
    const RingShape r = ring_shape(cols, dtype, tiles, 2, true, beta);
    const bool ring = ring_fits(r, {dy, dn, y, h, gate}, {dx, dh, dgate, post_gamma, post_beta, pre_gamma});
    const BackwardPlan b = backward_plan(rows, cols, gate_rows, info->sm_count, ring ? &r : nullptr);
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
        jobs.job[njobs++] = {at, sums[a], FDL_F32, 1, b.partials};
        at += b.partials * cols;
    }
    if (dgate != nullptr && gate_rows != rows && b.tasks_per_gate > 1) {
        p.gate_partial = at;
        jobs.job[njobs++] = {at, dgate, dtype, gate_rows, b.tasks_per_gate};
        groups = gate_rows;
    }
    if (ring) {
        status = error_flag_device_ptr(&p.error_flag);
        if (status == FDL_OK) status = launch_ring_backward(dtype, beta, p, r, b.grid, s);
    } else {
        status = launch_direct(true, dtype, vec, p, b.shape, b.grid, s);
    }
    if (status != FDL_OK || njobs == 0) return status;
    const dim3 grid(static_cast<unsigned int>(ceil_div(cols, kFoldX)), static_cast<unsigned int>(njobs),
                    static_cast<unsigned int>(groups < 64 ? groups : 64));
    const int strands = b.partials <= 64 ? 4 : b.partials <= 256 ? 8 : b.partials <= 512 ? 16 : kFoldY;
    return launch_ex(norm_fold_kernel, grid, dim3(kFoldX, strands), 0, s, dim3(1, 1, 1), tuning().pdl != 0, jobs);
}

}  // extern "C"
