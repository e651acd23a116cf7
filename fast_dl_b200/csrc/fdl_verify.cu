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
//
// Measured on B200 (floors at 6548 GB/s in brackets): 256 sequences at 131072 tokens f32 48 us [37], 64 at 50257 8.9 us
// [3.5], 32 at 100003 bf16 without draft probabilities 8.0 us [1.0], one at 32000 5.0 us.
#include <climits>
#include <type_traits>

#include "fdl_types.cuh"

namespace fdl {

namespace {

constexpr int kThreads = 256;
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

// What a row's weights are: p, max(p - q, 0), or p without one token.  Columns are taken in packs that lie on
// the 16-byte grid of p's row: pack k holds the columns [k N - lead, (k + 1) N - lead), the first and the
// last of them cut off by the row's ends.
template <class T>
struct Weights {
    static constexpr int N = kPack<T>;
    const T* p;
    const T* q;   // null: none
    int without;  // -1: none
    int vocab, lead;
    bool q_packs;  // q's row lies on the same grid

    __device__ __forceinline__ void set(const T* p_row, const T* q_row, int without_col, int n) {
        p = p_row;
        q = q_row;
        without = without_col;
        vocab = n;
        lead = static_cast<int>((reinterpret_cast<uintptr_t>(p_row) & 15) / sizeof(T));
        q_packs = ((reinterpret_cast<uintptr_t>(p_row) ^ reinterpret_cast<uintptr_t>(q_row)) & 15) == 0;
    }
    __device__ __forceinline__ int packs() const { return (vocab + lead + N - 1) / N; }

    struct Loaded {
        float a[N], b[N];
    };
    // The pack's values; 0 outside the row, and for k >= end.
    __device__ __forceinline__ void load(int k, int end, Loaded& v) const {
        const int col = k * N - lead;
#pragma unroll
        for (int e = 0; e < N; ++e) v.a[e] = v.b[e] = 0.0f;
        if (k >= end) return;
        if (col >= 0 && col + N <= vocab) {
            Chunk<T, N>::load(p + col, v.a);
            if (q != nullptr) {
                if (q_packs) {
                    Chunk<T, N>::load(q + col, v.b);
                } else {
#pragma unroll
                    for (int e = 0; e < N; ++e) v.b[e] = to_f32(q[col + e]);
                }
            }
        } else {
#pragma unroll
            for (int e = 0; e < N; ++e) {
                if (col + e < 0 || col + e >= vocab) continue;
                v.a[e] = to_f32(p[col + e]);
                if (q != nullptr) v.b[e] = to_f32(q[col + e]);
            }
        }
    }
    // The weight of element e of pack k: the exact difference where it is a positive number, 0 elsewhere.
    __device__ __forceinline__ double weight(const Loaded& v, int k, int e) const {
        const float d = v.a[e] - v.b[e];
        const bool counts = d > 0.0f && d < INFINITY && k * N - lead + e != without;
        return static_cast<double>(counts ? v.a[e] : 0.0f) - static_cast<double>(counts ? v.b[e] : 0.0f);
    }
    // One lane's share of the sum over the packs [lo, hi) of its warp.  As long as all weights are finite, each
    // is max(p, q) - q (a NaN p drops out); one that is not makes the total infinite or NaN, and the caller asks
    // again with kCareful, weight by weight.  That leaves five instructions a weight; with the tests in them
    // it was 36, and the arithmetic, not the bytes, took the time.
    template <bool kCareful>
    __device__ __forceinline__ double lane_sum(int lo, int hi) const {
        constexpr int kAhead = 4;  // packs of each row that a lane has on their way
        const int lane = threadIdx.x & (kWarp - 1);
        double s[4] = {0.0, 0.0, 0.0, 0.0};
        const int whole_lo = lead > 0 ? 1 : 0, whole_hi = (vocab + lead) / N;  // packs that no end of the row cuts
        if (kCareful) {
#pragma unroll 1
            for (int k = lo + lane; k < hi; k += kWarp) {
                Loaded v;
                load(k, hi, v);
#pragma unroll
                for (int e = 0; e < N; ++e) s[e & 3] += weight(v, k, e);
            }
            return (s[0] + s[1]) + (s[2] + s[3]);
        }
        const int from = max(lo, whole_lo), to = min(hi, whole_hi);
#pragma unroll 1
        for (int k0 = from + lane; k0 < to; k0 += kAhead * kWarp) {
            uint4 a[kAhead], b[kAhead];
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                a[u] = b[u] = make_uint4(0, 0, 0, 0);
                const int k = k0 + u * kWarp;
                if (k < to) {
                    a[u] = *reinterpret_cast<const uint4*>(p + k * N - lead);
                    if (q != nullptr) {
                        if (q_packs) {
                            b[u] = *reinterpret_cast<const uint4*>(q + k * N - lead);
                        } else {
                            T* const one = reinterpret_cast<T*>(&b[u]);
#pragma unroll
                            for (int e = 0; e < N; ++e) one[e] = q[k * N - lead + e];
                        }
                    }
                }
            }
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                float x[N], y[N];
                unpack(a[u], x, T{});
                if (q != nullptr) {
                    unpack(b[u], y, T{});
#pragma unroll
                    for (int e = 0; e < N; ++e) s[e & 3] += static_cast<double>(fmaxf(x[e], y[e])) - static_cast<double>(y[e]);
                } else {
                    const unsigned int at = static_cast<unsigned int>(without - ((k0 + u * kWarp) * N - lead));
#pragma unroll
                    for (int e = 0; e < N; ++e) s[e & 3] += static_cast<double>(at == static_cast<unsigned int>(e) ? 0.0f : fmaxf(x[e], 0.0f));
                }
            }
        }
        // The packs that the row's ends cut.
        const int cut = lane == 0 && lo < whole_lo ? 0 : lane == 1 && whole_hi < packs() && whole_hi >= from ? whole_hi : -1;
        if (cut >= lo && cut < hi && (lane < 2)) {
            Loaded v;
            load(cut, hi, v);
#pragma unroll
            for (int e = 0; e < N; ++e) s[e & 3] += weight(v, cut, e);
        }
        return (s[0] + s[1]) + (s[2] + s[3]);
    }
};

__device__ __forceinline__ double warp_inclusive(double v) {
    const int lane = threadIdx.x & (kWarp - 1);
#pragma unroll
    for (int o = 1; o < kWarp; o <<= 1) {
        const double up = __shfl_up_sync(kFullMask, v, o);
        if (lane >= o) v += up;
    }
    return v;
}

template <class T>
__global__ void __launch_bounds__(kThreads, 4)
verify_draft_kernel(const VerifyParams v) {
    constexpr int N = kPack<T>;
    constexpr int kRunsPerLane = kMaxCluster * kWarps / kWarp;  // 2
    __shared__ double run_sum[kMaxCluster * kWarps];  // of the whole row, in order
    __shared__ double warp_total[2][kWarps];
    __shared__ int first_rejected;
    __shared__ int found, last_positive;
    const int t = threadIdx.x, lane = t & (kWarp - 1), warp = t / kWarp;
    const uint32_t rank = cluster_rank(), cluster = cluster_size();
    const int64_t b = blockIdx.x / cluster;
    cluster_arrive();  // its other half, before the first remote store: every CTA of the cluster has started
    pdl_wait();
    const T* target = static_cast<const T*>(v.target) + b * v.target_batch_stride;
    const T* draft = v.draft == nullptr ? nullptr : static_cast<const T*>(v.draft) + b * v.draft_batch_stride;
    const int64_t* drawn = v.draft_tokens + b * v.drafted;
    // Every CTA of the cluster finds the first rejection by itself.
    if (warp == 0) {
        int len = v.drafted;
        if (v.draft_len != nullptr) {
            const int64_t n = v.draft_len[b];
            len = n < 0 ? 0 : n < v.drafted ? static_cast<int>(n) : v.drafted;
        }
        int n = len;
        for (int base = 0; base < len; base += kWarp) {
            const int i = base + lane;
            bool ok = true;
            if (i < len) {
                const int64_t d = drawn[i];
                const float u = v.accept_u[b * v.drafted + i];
                ok = d >= 0 && d < v.vocab;
                if (ok) {
                    const float pd = to_f32(target[i * v.target_row_stride + d]);
                    const float qd = draft == nullptr ? 1.0f : to_f32(draft[i * v.draft_row_stride + d]);
                    ok = __fmul_rn(u, qd) < pd;
                }
            }
            const unsigned int bad = __ballot_sync(kFullMask, !ok);
            if (bad != 0u) {
                n = base + __ffs(bad) - 1;
                break;
            }
        }
        if (lane == 0) {
            first_rejected = n < len ? n : -1 - n;  // below 0: all stand
            found = INT_MAX;
            last_positive = -1;
        }
    }
    const float u_sample = v.sample_u[b];
    __syncthreads();
    const bool rejected = first_rejected >= 0;
    const int n = rejected ? first_rejected : -1 - first_rejected;
    Weights<T> w;
    {
        int without = -1;
        if (rejected && draft == nullptr) {
            const int64_t d = drawn[n];
            without = d >= 0 && d < v.vocab ? static_cast<int>(d) : -1;
        }
        w.set(target + n * v.target_row_stride, rejected && draft != nullptr ? draft + n * v.draft_row_stride : nullptr, without,
              v.vocab);
    }
    const int runs = static_cast<int>(cluster) * kWarps;
    const int packs = w.packs();
    const int run = (packs + runs - 1) / runs;
    // Further rounds are for weights that are not all finite (careful), and for weights that are all 0 (the draft
    // covers the target: the target's row itself).
    bool careful = false, fallback = false;
    for (int round = 0;; ++round) {
        const int mine = static_cast<int>(rank) * kWarps + warp;
        const int lo = min(packs, mine * run), hi_run = min(packs, (mine + 1) * run);
        const double s = warp_sum(careful ? w.template lane_sum<true>(lo, hi_run) : w.template lane_sum<false>(lo, hi_run));
        if (round == 0) cluster_wait();
        if (lane < static_cast<int>(cluster)) store_remote(&run_sum[mine], lane, s);
        cluster_sync_all();
        // Each warp walks the run sums, a few in a row to a lane: where the sum crosses the goal, or else the
        // last run with any weight.
        double part[kRunsPerLane];
        double own = 0.0;
        const int per_lane = (runs + kWarp - 1) / kWarp;
#pragma unroll
        for (int i = 0; i < kRunsPerLane; ++i) {
            part[i] = i < per_lane && lane * per_lane + i < runs ? run_sum[lane * per_lane + i] : 0.0;
            own += part[i];
        }
        const double upto = warp_inclusive(own);
        const double total = __shfl_sync(kFullMask, upto, kWarp - 1);
        if (!careful && !(total < INFINITY)) {
            careful = true;
            cluster_sync_all();  // everybody has read the sums
            continue;
        }
        if (total > 0.0) {
            const double goal = static_cast<double>(u_sample) * total;
            double sum = upto - own, base = 0.0;
            int first = INT_MAX, last = -1;
#pragma unroll
            for (int i = 0; i < kRunsPerLane; ++i) {
                if (part[i] > 0.0) {
                    last = lane * per_lane + i;
                    if (first == INT_MAX) {
                        if (sum + part[i] > goal) first = last;
                        else sum += part[i];
                    }
                }
            }
            const int crossed = __reduce_min_sync(kFullMask, first);
            const int owner = crossed != INT_MAX ? crossed : __reduce_max_sync(kFullMask, last);
            base = __shfl_sync(kFullMask, sum, owner / per_lane);
            if (crossed == INT_MAX) base = -INFINITY;  // the last weight, whatever the sum
            if (owner / kWarps == static_cast<int>(rank)) {
                // This CTA reads the run again in order, a pack a thread at a time.
                const int hi = min(packs, (owner + 1) * run);
                int half = 0;
                for (int k0 = owner * run; k0 < hi; k0 += kThreads, half ^= 1) {
                    const int k = k0 + t;
                    typename Weights<T>::Loaded x;
                    w.load(k, hi, x);
                    double at[N];
                    double mine_sum = 0.0;
                    int last_col = -1;
#pragma unroll
                    for (int e = 0; e < N; ++e) {
                        at[e] = w.weight(x, k, e);
                        mine_sum += at[e];
                        if (at[e] > 0.0) last_col = k * N - w.lead + e;
                    }
                    const double incl = warp_inclusive(mine_sum);
                    if (lane == kWarp - 1) warp_total[half][warp] = incl;
                    last_col = __reduce_max_sync(kFullMask, last_col);
                    if (lane == 0 && last_col >= 0) atomicMax(&last_positive, last_col);
                    __syncthreads();
                    double before = 0.0, tile = 0.0;
#pragma unroll
                    for (int i = 0; i < kWarps; ++i) {
                        if (i == warp) before = tile;
                        tile += warp_total[half][i];
                    }
                    double reach = base + before + (incl - mine_sum);
                    int hit = INT_MAX;
#pragma unroll
                    for (int e = N - 1; e >= 0; --e) {
                        double to = reach;
#pragma unroll
                        for (int f = 0; f <= e; ++f) to += at[f];
                        if (at[e] > 0.0 && to > goal) hit = k * N - w.lead + e;
                    }
                    hit = __reduce_min_sync(kFullMask, hit);
                    if (lane == 0 && hit != INT_MAX) atomicMin(&found, hit);
                    base += tile;
                    if (__syncthreads_or(hit != INT_MAX)) break;
                }
                __syncthreads();
                if (t == 0) {
                    // Rounding may leave the crossing to no one: the last weight of the run then.
                    v.tokens[b * (v.drafted + 1) + n] = found != INT_MAX ? found : last_positive;
                    v.accepted[b] = n;
                }
            }
            break;
        }
        if (fallback) {
            if (rank == 0 && t == 0) {
                v.tokens[b * (v.drafted + 1) + n] = -1;
                v.accepted[b] = n;
            }
            break;
        }
        fallback = true;
        careful = false;
        cluster_sync_all();  // everybody has read the sums
        w.set(w.p, nullptr, -1, v.vocab);
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
    // CTAs for each sequence: as many as leave a lane a pack or two, up to eight an SM of the whole batch (256
    // sequences at 131072: up to two an SM 86 us, three 66, four 51, eight 48.5, sixteen 52).
    int cluster = 1;
    while (cluster < kMaxCluster && batch * cluster * 2 <= 8 * info->sm_count && vocab > cluster * kThreads * 8) cluster *= 2;
    const VerifyParams p{target, target_batch_stride, target_row_stride, draft, draft_batch_stride, draft_row_stride,
                         draft_tokens, draft_len, accept_u, sample_u, static_cast<int>(drafted), static_cast<int>(vocab),
                         tokens, accepted};
    return with_dtype(dtype, [&](auto* tag) {
        using T = std::remove_pointer_t<decltype(tag)>;
        return launch_ex(verify_draft_kernel<T>, dim3(static_cast<unsigned int>(batch * cluster)), dim3(kThreads), 0,
                         as_stream(stream), dim3(static_cast<unsigned int>(cluster), 1, 1), tuning().pdl != 0, p);
    });
}

}  // extern "C"
