// Verification of drafted tokens against the target model's probabilities, from given random numbers.
//
// A sequence has up to `drafted` tokens d_i, drawn from the draft model's rows q_i, and the target's
// rows p_0 .. p_drafted.  Token i is accepted while accept_u_i * q_i(d_i) < p_i(d_i).  At the first
// rejection i the next token is drawn from the weights w_v = max(p_i(v) - q_i(v), 0), after all were
// accepted from w = p_len: the smallest v whose running sum of w exceeds sample_u * (sum of w).  The
// result is distributed as the target's own samples whatever the draft proposes.
//
// The token is decided by comparing a sum of up to hundreds of thousands of weights with a fraction of
// their total, so sums and the subtraction are in 64 bits: in 32 bits the order of the additions would
// decide the token once in some thousand draws.  A weight that is not a positive finite number counts as 0.
//
// What bounds it: one row of p and, after a rejection, one of q for each sequence; for a small batch the
// chain of dependent accesses (tokens, their probabilities, the row, the run that holds the token).
// A cluster of CTAs shares a sequence's row, so that one sequence alone is read by 8 SMs at a time: each
// warp sums one contiguous run of the row, the run sums meet through distributed shared memory, every
// CTA finds the run in which the sum crosses, and the CTA that owns it reads that run once more (out
// of L2) in order.
#include <climits>
#include <type_traits>

#include "fdl_types.cuh"

namespace fdl {

namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / kWarp;
constexpr int kMaxCluster = 8;

struct VerifyParams {
    const void* target;
    int64_t target_batch_stride, target_row_stride;
    const void* draft;  // may be null: the draft is certain of its tokens
    int64_t draft_batch_stride, draft_row_stride;
    const int64_t* draft_tokens;
    const int64_t* draft_len;  // may be null
    const float* accept_u;
    const float* sample_u;
    int drafted;
    int vocab;
    int run;  // elements of a warp's run
    int64_t* tokens;
    int64_t* accepted;
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
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_sync_all() {
    cluster_arrive();
    cluster_wait();
}
__device__ __forceinline__ void store_remote(double* mine, uint32_t rank, double v) {
    uint32_t remote;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(smem_addr(mine)), "r"(rank));
    asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(remote), "d"(v) : "memory");
}

// What a row's weights are: p, max(p - q, 0), or p without one token.
template <class T>
struct Weights {
    const T* p;
    const T* q;    // null: none
    int without;   // -1: none
    __device__ __forceinline__ double operator()(float pv, float qv, int col) const {
        double w = static_cast<double>(pv);
        if (q != nullptr) w -= static_cast<double>(qv);
        if (col == without) w = 0.0;
        return w > 0.0 && w < INFINITY ? w : 0.0;
    }
    __device__ __forceinline__ double at(int col) const {
        return (*this)(to_f32(p[col]), q != nullptr ? to_f32(q[col]) : 0.0f, col);
    }
    // One lane's share of the sum over [lo, hi); `vec`: p, q and lo are on the 128-bit grid.
    __device__ __forceinline__ double lane_sum(int lo, int hi, bool vec) const {
        constexpr int N = kPack<T>;
        const int lane = threadIdx.x & (kWarp - 1);
        double s = 0.0;
        int c = lo;
        if (vec) {
            const int packs = (hi - lo) / N;
#pragma unroll 4
            for (int i = lane; i < packs; i += kWarp) {
                float a[N], b[N];
                Chunk<T, N>::load(p + lo + i * N, a);
                if (q != nullptr) {
                    Chunk<T, N>::load(q + lo + i * N, b);
                } else {
#pragma unroll
                    for (int e = 0; e < N; ++e) b[e] = 0.0f;
                }
#pragma unroll
                for (int e = 0; e < N; ++e) s += (*this)(a[e], b[e], lo + i * N + e);
            }
            c = lo + packs * N;
        }
#pragma unroll 8
        for (int i = c + lane; i < hi; i += kWarp) s += at(i);
        return s;
    }
};

template <class T>
__global__ void __launch_bounds__(kThreads)
verify_draft_kernel(const VerifyParams v) {
    __shared__ double run_sum[kMaxCluster * kWarps];  // of the whole row, in order
    __shared__ double warp_total[kWarps];
    __shared__ int first_rejected;
    __shared__ int last_positive;
    const int t = threadIdx.x, lane = t & (kWarp - 1), warp = t / kWarp;
    const uint32_t rank = cluster_rank(), cluster = cluster_size();
    const int64_t b = blockIdx.x / cluster;
    cluster_arrive();  // its other half, before the first remote store: every CTA of the cluster has started
    pdl_wait();
    const T* target = static_cast<const T*>(v.target) + b * v.target_batch_stride;
    const T* draft = v.draft == nullptr ? nullptr : static_cast<const T*>(v.draft) + b * v.draft_batch_stride;
    const int64_t* drawn = v.draft_tokens + b * v.drafted;
    int len = v.drafted;
    if (v.draft_len != nullptr) {
        const int64_t n = v.draft_len[b];
        len = n < 0 ? 0 : n < v.drafted ? static_cast<int>(n) : v.drafted;
    }
    // Every CTA of the cluster finds the first rejection by itself.
    if (warp == 0) {
        int n = len;
        for (int base = 0; base < len; base += kWarp) {
            const int i = base + lane;
            bool ok = true;
            if (i < len) {
                const int64_t d = drawn[i];
                ok = d >= 0 && d < v.vocab;
                if (ok) {
                    const float pd = to_f32(target[i * v.target_row_stride + d]);
                    const float qd = draft == nullptr ? 1.0f : to_f32(draft[i * v.draft_row_stride + d]);
                    ok = __fmul_rn(v.accept_u[b * v.drafted + i], qd) < pd;
                }
            }
            const unsigned int bad = __ballot_sync(kFullMask, !ok);
            if (bad != 0u) {
                n = base + __ffs(bad) - 1;
                break;
            }
        }
        if (lane == 0) first_rejected = n;
    }
    __syncthreads();
    const int n = first_rejected;
    Weights<T> w;
    w.p = target + n * v.target_row_stride;
    w.q = n < len && draft != nullptr ? draft + n * v.draft_row_stride : nullptr;
    w.without = -1;
    if (n < len && draft == nullptr) {
        const int64_t d = drawn[n];
        w.without = d >= 0 && d < v.vocab ? static_cast<int>(d) : -1;
    }
    const int runs = static_cast<int>(cluster) * kWarps;
    int64_t token = -1;
    // The second round is for weights that are all 0 (the draft covers the target): the target's row itself.
    for (int round = 0; round < 2; ++round) {
        const int mine = static_cast<int>(rank) * kWarps + warp;
        const int64_t lo64 = static_cast<int64_t>(mine) * v.run;
        const int lo = lo64 < v.vocab ? static_cast<int>(lo64) : v.vocab;
        const int hi = v.vocab - lo < v.run ? v.vocab : lo + v.run;
        const bool vec = ((reinterpret_cast<uintptr_t>(w.p) | reinterpret_cast<uintptr_t>(w.q)) & 15) == 0;
        const double s = warp_sum(w.lane_sum(lo, hi, vec));
        if (round == 0) cluster_wait();
        if (lane < static_cast<int>(cluster)) store_remote(&run_sum[mine], lane, s);
        cluster_sync_all();
        // Every thread walks the run sums in order: where the sum crosses, or else the last run with any weight.
        double total = 0.0;
        for (int r = 0; r < runs; ++r) total += run_sum[r];
        if (total > 0.0) {
            const double goal = static_cast<double>(v.sample_u[b]) * total;
            double before = 0.0, base = 0.0, sum = 0.0;
            int owner = -1;
            bool crossed = false;
            for (int r = 0; r < runs && !crossed; ++r) {
                sum += run_sum[r];
                if (run_sum[r] > 0.0) {
                    owner = r;
                    base = before;
                    crossed = sum > goal;
                }
                before = sum;
            }
            if (owner / kWarps == static_cast<int>(rank)) {
                // This CTA reads the run again, each thread a contiguous piece of it.
                const int64_t start64 = static_cast<int64_t>(owner) * v.run;
                const int start = static_cast<int>(start64);
                const int stop = v.vocab - start < v.run ? v.vocab : start + v.run;
                const int piece = (stop - start + kThreads - 1) / kThreads;
                const int from = min(stop, start + t * piece), to = min(stop, from + piece);
                double own = 0.0;
                int last = -1;
                for (int col = from; col < to; ++col) {
                    const double x = w.at(col);
                    own += x;
                    if (x > 0.0) last = col;
                }
                double upto = own;  // inclusive over the warp
#pragma unroll
                for (int o = 1; o < kWarp; o <<= 1) {
                    const double up = __shfl_up_sync(kFullMask, upto, o);
                    if (lane >= o) upto += up;
                }
                if (lane == kWarp - 1) warp_total[warp] = upto;
                if (t == 0) last_positive = -1;
                __syncthreads();
                for (int k = 0; k < warp; ++k) base += warp_total[k];
                double reach = base + (upto - own);
                int found = INT_MAX;
                if (own > 0.0) {
                    for (int col = from; col < to; ++col) {
                        const double x = w.at(col);
                        reach += x;
                        if (x > 0.0 && reach > goal) {
                            found = col;
                            break;
                        }
                    }
                }
                if (last >= 0) atomicMax(&last_positive, last);
                found = __reduce_min_sync(kFullMask, found);
                __syncthreads();
                if (lane == 0) warp_total[warp] = static_cast<double>(found);
                __syncthreads();
                double best = warp_total[0];
                for (int k = 1; k < kWarps; ++k) best = fmin(best, warp_total[k]);
                // Rounding may leave the crossing to no one: the last weight of the run then.
                token = best < static_cast<double>(INT_MAX) ? static_cast<int64_t>(best) : last_positive;
                if (t == 0) {
                    int64_t* out = v.tokens + b * (v.drafted + 1);
                    out[n] = token;
                    v.accepted[b] = n;
                }
            }
            break;
        }
        if (round == 0) {
            cluster_sync_all();  // everybody has read the sums
            w.q = nullptr;
            w.without = -1;
        } else if (rank == 0 && t == 0) {
            v.tokens[b * (v.drafted + 1) + n] = -1;
            v.accepted[b] = n;
        }
    }
    if (rank == 0) {
        int64_t* out = v.tokens + b * (v.drafted + 1);
        for (int i = t; i <= v.drafted; i += kThreads) {
            if (i < n) out[i] = drawn[i];
            if (i > n) out[i] = -1;
        }
    }
}

}  // namespace

}  // namespace fdl

using namespace fdl;

extern "C" {

int fdl_verify_draft(const void* target, int64_t target_batch_stride, int64_t target_row_stride, const void* draft,
                     int64_t draft_batch_stride, int64_t draft_row_stride, int dtype, const int64_t* draft_tokens,
                     const int64_t* draft_len, const float* accept_u, const float* sample_u, int64_t batch,
                     int64_t drafted, int64_t vocab, int64_t* tokens, int64_t* accepted, void* stream) {
    if (batch < 0 || drafted < 0 || vocab <= 0 || !known_dtype(dtype)) return FDL_ERR_INVALID_ARGUMENT;
    if (target_row_stride < 0 || target_batch_stride < 0 || draft_row_stride < 0 || draft_batch_stride < 0) {
        return FDL_ERR_INVALID_ARGUMENT;
    }
    if (batch > INT_MAX / kMaxCluster || drafted > 65535 || vocab > INT_MAX / 2) return FDL_ERR_UNSUPPORTED;
    if (batch == 0) return FDL_OK;
    if (target == nullptr || sample_u == nullptr || tokens == nullptr || accepted == nullptr ||
        (drafted > 0 && (draft_tokens == nullptr || accept_u == nullptr))) {
        return FDL_ERR_INVALID_ARGUMENT;
    }
    int status = FDL_OK;
    const DeviceInfo* info = current_device_info(&status);
    if (info == nullptr) return status;
    // CTAs for each sequence: as many as leave a run of two packs a lane, while the batch does not fill the GPU.
    int cluster = 1;
    while (cluster < kMaxCluster && batch * cluster * 2 <= 2 * info->sm_count && vocab > cluster * kThreads * 8) cluster *= 2;
    const int64_t granule = 16 / static_cast<int64_t>(dtype_bytes(dtype));
    const int64_t run = ceil_div(ceil_div(vocab, static_cast<int64_t>(cluster) * kWarps), granule) * granule;
    const VerifyParams p{target, target_batch_stride, target_row_stride, draft, draft_batch_stride, draft_row_stride,
                         draft_tokens, draft_len, accept_u, sample_u, static_cast<int>(drafted), static_cast<int>(vocab),
                         static_cast<int>(run), tokens, accepted};
    return with_dtype(dtype, [&](auto* tag) {
        using T = std::remove_pointer_t<decltype(tag)>;
        return launch_ex(verify_draft_kernel<T>, dim3(static_cast<unsigned int>(batch * cluster)), dim3(kThreads), 0,
                         as_stream(stream), dim3(static_cast<unsigned int>(cluster), 1, 1), tuning().pdl != 0, p);
    });
}

}  // extern "C"
