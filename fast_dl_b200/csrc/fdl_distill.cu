// Distillation from a teacher's top logits: the loss of each row, its mean, and the gradient.
//
// Row r has `vocab` student logits z and k entries (t_j, i_j) of the teacher.  With temperature T
//   p_j = exp(t_j / T) / sum_j exp(t_j / T)      over the entries that count (0 <= i_j < vocab, t_j > -inf), or
//   p_j = exp(t_j / T - lse_r)                   where the teacher's own normaliser is given,
//   log q_v = (z_v - m) / T - log S,             m = max z, S = sum_v exp((z_v - m) / T),
//   row_loss = sum_j p_j (log p_j - log q_{i_j}),    loss = scale * sum_r w_r row_loss_r,
//   dz_v = scale w_r / T * (P q_v - sum of the p_j whose i_j is v),    P = sum_j p_j.
// A row of weight 0 or without entries that count is left out: loss 0, gradient 0, whatever its logits hold.
//
// Differences of logarithms are taken in 64 bits (k of them a row): where teacher and student
// agree, the loss is a small difference of numbers of size ten.
//
// What bounds it: a row has to be read once for the loss, and written once more for the gradient; loss and gradient
// in one call keep the row on chip between the two.  Measured on B200 (floors at 6548 GB/s in brackets): loss and
// gradient of [4096, 65537] f32 360 us [321], of [2048, 131072] bf16 225 us [160], of [15660, 966] f16 33 us [10],
// gradient of [1000, 50257] f32 78 us [60], loss of [8, 32000] f32 7.7 us with its mean.
#include <atomic>
#include <climits>
#include <type_traits>

#include "fdl_types.cuh"

namespace fdl {

namespace {

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

// What the teacher says of a row, in the shared memory of the warp that read it.
struct Entries {
    float* prob;  // [k]: p_j; of entries that share a column the first has the sum
    float* here;  // [k]: the student's logit there
    int* at;      // [k]: the column, or -1: does not count, or folded into another
    uint16_t* table;
    int places;   // of the table, a power of two of at least 2 k
};

// One warp reads a row's entries.  Returns whether any counts, and then the loss's share that does not need the
// row's sum, base = sum p_j (log p_j - logit_j / T), and mass = sum p_j.  `wanted`: columns whose logits to read.
template <class T, bool LOSS, bool GRAD, class Wanted>
__device__ __forceinline__ bool read_entries(const DistillParams& p, const T* z, int64_t row, float c, const Entries& out, double* base_out,
                                             double* mass_out, Wanted&& wanted) {
    const int lane = threadIdx.x & (kWarp - 1);
    float* const prob = out.prob;
    float* const here = out.here;
    int* const at = out.at;
    float top = -INFINITY;
    for (int j0 = lane; j0 < p.k; j0 += 4 * kWarp) {  // four entries' loads at a time
        int64_t i[4];
        float v[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int64_t from = row * p.k + min(j0 + q * kWarp, p.k - 1);
            i[q] = p.index[from];
            v[q] = load_any(p.teacher, p.teacher_dtype, from);
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int j = j0 + q * kWarp;
            if (j >= p.k) break;
            const bool counts = i[q] >= 0 && i[q] < p.vocab && v[q] > -INFINITY;  // a NaN does not either
            prob[j] = counts ? v[q] : -INFINITY;
            at[j] = counts ? static_cast<int>(i[q]) : -1;
            if (counts) top = fmaxf(top, v[q]);
        }
    }
    top = warp_max(top);
    if (top == -INFINITY) return false;
    float part = 0.0f;
    for (int j0 = lane; j0 < p.k; j0 += 4 * kWarp) {
        float v[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int j = j0 + q * kWarp;
            const int col = j < p.k ? at[j] : -1;
            v[q] = col >= 0 && wanted(col) ? to_f32(z[col]) : 0.0f;
            if (col >= 0) part += ex2_approx((prob[j] - top) * c);
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            if (j0 + q * kWarp < p.k) here[j0 + q * kWarp] = v[q];
        }
    }
    const double sum = static_cast<double>(warp_sum(part));
    const double norm = p.teacher_lse == nullptr ? static_cast<double>(top) * p.inv_temperature + log(sum)
                                                 : static_cast<double>(p.teacher_lse[row]);
    double base = 0.0, mass = 0.0;
    for (int j = lane; j < p.k; j += kWarp) {
        float pj = 0.0f;
        if (at[j] >= 0) {
            const double logp = static_cast<double>(prob[j]) * p.inv_temperature - norm;
            pj = expf(static_cast<float>(logp));
            if (LOSS && pj != 0.0f) base += pj * (logp - static_cast<double>(here[j]) * p.inv_temperature);
            mass += pj;
        }
        prob[j] = pj;
    }
    *base_out = warp_sum(base);
    *mass_out = warp_sum(mass);
    if (!GRAD) return true;
    // Entries of one column: each entry writes its number into the column's place of a hash table
    // and looks who is there.  Another column there: again with another hash (that column's own
    // entries are all in the same position); its own column: to be folded.  What the table held
    // before does not matter, as a place is read after at least one entry wrote it.
    uint32_t pending = 0, same = 0;  // bit q: entry lane + 32 q
    for (int j = lane, q = 0; j < p.k; j += kWarp, ++q) pending |= at[j] >= 0 ? 1u << q : 0u;
    for (uint32_t round = 0; __any_sync(kFullMask, pending != 0u); ++round) {
        const uint32_t mix = 0x9E3779B1u + 2u * round * 0x85EBCA6Bu;  // odd
        __syncwarp();
        for (uint32_t left = pending; left != 0u; left &= left - 1u) {
            const int j = lane + kWarp * (__ffs(left) - 1);
            out.table[(static_cast<uint32_t>(at[j] + 1) * mix >> 15) & (out.places - 1)] = static_cast<uint16_t>(j);
        }
        __syncwarp();
        for (uint32_t left = pending; left != 0u; left &= left - 1u) {
            const int q = __ffs(left) - 1, j = lane + kWarp * q;
            const int w = out.table[(static_cast<uint32_t>(at[j] + 1) * mix >> 15) & (out.places - 1)];
            if (w == j || at[w] == at[j]) {
                pending &= ~(1u << q);
                if (w != j) same |= 1u << q;
            }
        }
    }
    __syncwarp();
    // The first entry of a shared column gets the sum (in entry order over lanes, a fixed tree); the
    // others are dropped.
    for (uint32_t owners = __ballot_sync(kFullMask, same != 0u); owners != 0u; owners = __ballot_sync(kFullMask, same != 0u)) {
        const int owner = __ffs(owners) - 1;
        const int j = __shfl_sync(kFullMask, same != 0u ? lane + kWarp * (__ffs(same) - 1) : 0, owner);
        if (lane == owner) same &= same - 1u;
        const int col = at[j];
        if (col < 0) continue;  // dropped with an earlier one
        int least = p.k;
        float sum_p = 0.0f;
        for (int i = lane; i < p.k; i += kWarp) {
            if (at[i] == col) {
                least = min(least, i);
                sum_p += prob[i];
            }
        }
        least = __reduce_min_sync(kFullMask, least);
        sum_p = warp_sum(sum_p);
        __syncwarp();
        for (int i = lane; i < p.k; i += kWarp) {
            if (at[i] == col) {
                if (i == least) prob[i] = sum_p;
                else at[i] = -1;
            }
        }
        __syncwarp();
    }
    return true;
}

// -inf in each element of a pack.
__device__ __forceinline__ uint4 lowest_pack(float) { return make_uint4(0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u); }
__device__ __forceinline__ uint4 lowest_pack(__half) { return make_uint4(0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u); }
__device__ __forceinline__ uint4 lowest_pack(__nv_bfloat16) { return make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u); }

// The largest element of some packs (NaN is passed over); 16-bit types two at a time, before they are unpacked.
template <int PACKS>
__device__ __forceinline__ float packs_max(const uint4 (&raw)[PACKS], float) {
    float m = -INFINITY;
#pragma unroll
    for (int q = 0; q < PACKS; ++q) {
        m = fmaxf(m, fmaxf(fmaxf(__uint_as_float(raw[q].x), __uint_as_float(raw[q].y)),
                           fmaxf(__uint_as_float(raw[q].z), __uint_as_float(raw[q].w))));
    }
    return m;
}
template <int PACKS, class T>
__device__ __forceinline__ float packs_max(const uint4 (&raw)[PACKS], T) {
    using Pair = std::conditional_t<std::is_same_v<T, __half>, __half2, __nv_bfloat162>;
    const uint4 low = lowest_pack(T{});
    Pair m = *reinterpret_cast<const Pair*>(&low.x);
#pragma unroll
    for (int q = 0; q < PACKS; ++q) {
        const Pair a = __hmax2(*reinterpret_cast<const Pair*>(&raw[q].x), *reinterpret_cast<const Pair*>(&raw[q].y));
        const Pair b = __hmax2(*reinterpret_cast<const Pair*>(&raw[q].z), *reinterpret_cast<const Pair*>(&raw[q].w));
        m = __hmax2(m, __hmax2(a, b));
    }
    return fmaxf(to_f32(m.x), to_f32(m.y));
}

// A running maximum and sum of exponentials relative to it.
struct Running {
    float m = -INFINITY, s = 0.0f;
    template <class T, int PACKS>
    __device__ __forceinline__ void take(const uint4 (&raw)[PACKS], float c) {
        constexpr int M = kPack<T> / 2;
        const float big = packs_max(raw, T{});
        const float now = fmaxf(m, big);
        const float ref = now == -INFINITY ? 0.0f : now;  // nothing but -inf so far: exp(-inf) each
        const float2 down = both(-ref), c2 = both(c);
        float2 add[2] = {both(0.0f), both(0.0f)};
#pragma unroll
        for (int q = 0; q < PACKS; ++q) {
            float2 v[M];
            unpack2(raw[q], v, T{});
#pragma unroll
            for (int e = 0; e < M; ++e) {
                v[e] = mul2(add2(v[e], down), c2);
                add[e & 1] = add2(add[e & 1], make_float2(ex2_approx(v[e].x), ex2_approx(v[e].y)));
            }
        }
        const float2 sum = add2(add[0], add[1]);
        s = s * exp_diff(m, now, c) + (sum.x + sum.y);
        m = now;
    }
    __device__ __forceinline__ void take_one(float v, float c) {
        const float now = fmaxf(m, v);
        s = s * exp_diff(m, now, c) + ex2_approx((v - (now == -INFINITY ? 0.0f : now)) * c);
        m = now;
    }
    // The warp's pair, in every lane.
    __device__ __forceinline__ float2 of_warp(float c) const {
        const float top = warp_max(m);
        return make_float2(top, warp_sum(s * exp_diff(m, top, c)));
    }
};

// The row's maximum and sum from the warps' pairs: the same order, and so the same bits, in every warp and CTA.
__device__ __forceinline__ float2 fold_stats(const float2* stat, int n, float c) {
    const int lane = threadIdx.x & (kWarp - 1);
    float m = -INFINITY;
    for (int i = lane; i < n; i += kWarp) m = fmaxf(m, stat[i].x);
    m = warp_max(m);
    float sum = 0.0f;
    for (int i = lane; i < n; i += kWarp) sum += stat[i].y * exp_diff(stat[i].x, m, c);
    return make_float2(m, warp_sum(sum));
}
__device__ __forceinline__ void write_loss(const DistillParams& p, double base, double mass, int64_t row, float2 f) {
    p.row_stats[2 * row] = f.x;
    p.row_stats[2 * row + 1] = f.y;
    p.row_loss[row] =
        static_cast<float>(base + mass * (static_cast<double>(f.x) * p.inv_temperature + log(static_cast<double>(f.y))));
}
__device__ __forceinline__ void write_left_out(const DistillParams& p, int64_t row) {
    p.row_stats[2 * row] = 0.0f;
    p.row_stats[2 * row + 1] = 0.0f;
    p.row_loss[row] = 0.0f;
}

// ---- short rows: in the registers of a warp or of a CTA -------------------------------------------------
//
// WARPS warps a row, up to HELD packs a thread: rows of up to 4 KiB a warp.  With one warp a row there is no barrier
// at all; otherwise the first warp reads the entries while all of them have the row on its way, and one barrier
// brings the warps' pairs and the entries together.  What bounds it is the chain of dependent loads (entries, the
// logits that they name), so as many rows as the registers allow are under way at once, and the row is asked for
// before it is known to count.

constexpr int kHeld = 8;  // the most

template <class T, bool LOSS, bool GRAD, int WARPS, int HELD>
__global__ void __launch_bounds__(WARPS == 1 ? 256 : WARPS * kWarp, WARPS == 1 ? (HELD <= 4 ? 4 : 3) : 24 / WARPS)
distill_rows_kernel(const DistillParams p, int places) {
    constexpr int N = kPack<T>, M = N / 2;
    constexpr int kTeams = WARPS == 1 ? 256 / kWarp : 1, kThreads = WARPS * kWarp;
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ float2 stat[WARPS];
    __shared__ double shared_base, shared_mass;
    __shared__ int shared_live;
    const int lane = threadIdx.x & (kWarp - 1), warp = threadIdx.x / kWarp;
    const int team = WARPS == 1 ? warp : 0, w = WARPS == 1 ? 0 : warp, t = w * kWarp + lane;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * kTeams + team;
    if (row >= p.rows) return;
    const float c = static_cast<float>(kLog2e * p.inv_temperature);
    float* const probs = reinterpret_cast<float*>(smem) + team * 3 * p.k;
    const Entries entries{probs, probs + p.k, reinterpret_cast<int*>(probs + 2 * p.k),
                          reinterpret_cast<uint16_t*>(reinterpret_cast<float*>(smem) + kTeams * 3 * p.k) + team * places, places};
    pdl_wait();
    const T* z = static_cast<const T*>(p.logits) + row * p.logits_stride;
    T* const g = GRAD ? static_cast<T*>(p.grad) + row * p.grad_stride : nullptr;
    const RowSpan<T> span(z, p.vocab);
    const bool same_phase = ((reinterpret_cast<uintptr_t>(z) ^ reinterpret_cast<uintptr_t>(g)) & 15) == 0;
    const float weight = p.row_weight == nullptr ? 1.0f : p.row_weight[row];
    uint4 raw[HELD];
    float edge = -INFINITY;
    const int edges = span.head + span.tail;
    const int edge_col = lane < span.head ? lane : p.vocab - span.tail + (lane - span.head);
    double base = 0.0, mass = 0.0;
    const uint4* packs = reinterpret_cast<const uint4*>(z + span.head);
#pragma unroll
    for (int q = 0; q < HELD; ++q) raw[q] = t + q * kThreads < span.packs ? packs[t + q * kThreads] : lowest_pack(T{});
    if (w == 0 && lane < edges) edge = to_f32(z[edge_col]);
    bool live = weight != 0.0f;
    if (live) {
        if (w == 0) {
            live = read_entries<T, LOSS, GRAD>(p, z, row, c, entries, &base, &mass, [](int) { return true; });
            if (WARPS > 1 && lane == 0) {
                shared_base = base;
                shared_mass = mass;
                shared_live = live;
            }
        }
    }
    float2 f = make_float2(0.0f, 1.0f);
    if (weight != 0.0f) {
        if (LOSS) {
            Running run;
            run.take<T>(raw, c);
            if (w == 0 && lane < edges) run.take_one(edge, c);
            f = run.of_warp(c);
            if (WARPS > 1 && lane == 0) stat[w] = f;
        }
        if (WARPS > 1) {
            __syncthreads();
            live = shared_live != 0;
            mass = shared_mass;
            if (LOSS) f = fold_stats(stat, WARPS, c);
        }
    }
    if (!live) {
        if (LOSS && t == 0) write_left_out(p, row);
        if (GRAD) {
            for (int i = t; i < p.vocab; i += kThreads) g[i] = from_f32<T>(0.0f);
        }
        return;
    }
    if (LOSS && t == 0) write_loss(p, base, mass, row, f);
    if (!LOSS) f = make_float2(p.row_stats[2 * row], p.row_stats[2 * row + 1]);
    if (!GRAD) return;
    const float coef = p.scale * static_cast<float>(p.inv_temperature) * (p.grad_loss != nullptr ? *p.grad_loss : 1.0f) * weight;
    const float part = p.teacher_lse == nullptr && mass == mass ? 1.0f : static_cast<float>(mass);
    const float each = coef * part / f.y;
    const float2 down = both(-f.x), c2 = both(c), each2 = both(each);
#pragma unroll
    for (int q = 0; q < HELD; ++q) {
        const int i = t + q * kThreads;
        if (i >= span.packs) break;
        float2 v[M];
        unpack2(raw[q], v, T{});
#pragma unroll
        for (int e = 0; e < M; ++e) {
            v[e] = mul2(add2(v[e], down), c2);
            v[e] = mul2(make_float2(ex2_approx(v[e].x), ex2_approx(v[e].y)), each2);
        }
        T* const out = g + span.head + static_cast<int64_t>(i) * N;
        if (same_phase) {
            store_pairs(out, v);
        } else {
#pragma unroll
            for (int e = 0; e < M; ++e) {
                out[2 * e] = from_f32<T>(v[e].x);
                out[2 * e + 1] = from_f32<T>(v[e].y);
            }
        }
    }
    if (w == 0 && lane < edges) g[edge_col] = from_f32<T>(ex2_approx((edge - f.x) * c) * each);
    // The columns that the teacher names, behind the dense part.
    if (WARPS > 1) __syncthreads();
    else __syncwarp();
    for (int j = t; j < p.k; j += kThreads) {
        const int col = entries.at[j];
        if (col < 0) continue;
        const float q = ex2_approx((entries.here[j] - f.x) * c) / f.y;
        g[col] = from_f32<T>(coef * (part * q - entries.prob[j]));
    }
}

// ---- long rows: a ring of chunks in shared memory -----------------------------------------------------
//
// One CTA an SM, or a cluster of them a row, takes rows one after the other.  Its warps have trades, and each
// goes on as soon as what it needs is there:
//   copies   one thread asks for the row's chunks (bulk-async copies) as places in the ring come free;
//   entries  three warps read the teacher's entries, each of every third row and so a few rows ahead: their
//            probabilities, the student's logits there, entries that share a column folded into the first,
//            what the loss needs of them (one warp for all rows was the slowest part of the kernel);
//   sums     eight warps take each chunk for the row's maximum and sum of exponentials, every thread with a
//            running pair of its own, and send each warp's pair to all CTAs of the cluster;
//   writes   eight warps wait for the pairs, fold them, write the gradient chunk by chunk and give the places back.
// So a row is read once and its gradient written once; the sums of row i + 1 are under way while the gradient of
// row i is written, and the exchange between them falls to nobody's wait as long as the ring holds more than
// the row.  The loss alone has two groups of eight warps for the sums, one for the even and one for the odd places of
// the ring, the gradient alone two groups for the writes.  (A barrier tells one round of its place from the next
// only, so whoever waits for a place has to wait for each of its rounds: with the chunks of a row dealt out in
// turn, a group could be two rounds ahead of a slow copy and take the place's last chunk for its next.)
// The elements of a row outside its 16-byte grid (its first and last few) go by plain loads.
//
// Of [2048, 131072] bf16's 225 us, 113 are the special-function unit's (two exponentials an element, 16 a cycle and
// SM; without those of the writes it takes 180 us, without any 174), the rest of the gap to 160 is the chain of a
// row: its last chunk's copy, sum and exchange.  Measured and dropped: one kind of worker for sums and writes 253
// us (f32 401), groups of four warps 231, three groups of eight 212-230 (f32 348-366), chunks of 8 KiB 255 and of 18 to
// 32 KiB 206-246 (f32 367-459), a prefetch of the row into L2 216 (f32 356), half of the writes' exponentials by a
// polynomial 230, clusters of four where two do (132 of 148 SMs at one CTA an SM).
//
// Every wait has a limit; one that gives up ends all of them (and is reported through the error flag).

constexpr int kChunkBytes = 16384;
constexpr int kMaxSlots = 13;
constexpr int kPrepSlots = 4;   // rows whose entries are kept
constexpr int kPrepWarps = 3;   // 20 warps in all: one more would cost every thread 16 registers
constexpr int kGroupWarps = 8;  // a group takes a whole chunk
constexpr int kGroup = kGroupWarps * kWarp;
constexpr int kBatch = kChunkBytes / 16 / kGroup;  // packs of a chunk that a thread takes
constexpr int kFirstWorker = 1 + kPrepWarps;       // warp
constexpr int kRingThreads = (kFirstWorker + 2 * kGroupWarps) * kWarp;
constexpr int kMaxCluster = 8;
// Rows whose pairs may be on their way: a CTA whose writes have not read those of row i keeps its entries' slot,
// so its sums end at row i + 3, the other CTAs' writes too, and their sums at row i + 7.
constexpr int kStatSlots = 2 * kPrepSlots;
constexpr int kRingSmem = 216 * 1024;  // of 227: the rest holds the static part

struct Prepared {  // what is left of a row by its warp, beside the entries
    double base;   // sum p_j (log p_j - logit_j / T)
    double mass;
    float weight, m, total;
    int live;
    float edge[16];
};

struct RingParams {
    DistillParams d;
    int slots;
    int table;  // places of a hash table of columns, a power of two (one table for each prep warp)
    unsigned int* error_flag;
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
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.release.cta.shared::cta.b64 _, [%0];" ::"r"(smem_addr(bar)) : "memory");
}
// Stores (m, s) into CTA `rank`'s copy of `mine`, counted as eight bytes on its copy of `bar`.  (An ordinary
// store and a releasing arrival would wait for the warp's gradient stores, a microsecond or two a row.)  Only in a
// launch with clusters: without one the instruction is not a legal one.
__device__ __forceinline__ void send_stat(float2* mine, uint64_t* bar, uint32_t rank, float2 v) {
    uint32_t to, at;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"(smem_addr(mine)), "r"(rank));
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_addr(bar)), "r"(rank));
    asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v2.f32 [%0], {%1, %2}, [%3];" ::"r"(to), "f"(v.x),
                 "f"(v.y), "r"(at)
                 : "memory");
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

// A wait that gives up raises `failed`, which ends every later wait of the CTA that is not over at once;
// who gets false leaves.
template <bool CLUSTER = false>
__device__ __forceinline__ bool lane_wait(uint64_t* bar, uint32_t parity, volatile int* failed, unsigned int* error_flag) {
    if (CLUSTER ? mbar_try_wait_cluster(bar, parity) : mbar_try_wait(bar, parity)) return true;
    for (uint32_t i = 0; i < kMbarSpinLimit; ++i) {
        if (CLUSTER ? mbar_try_wait_cluster(bar, parity) : mbar_try_wait(bar, parity)) return true;
        if ((i & 15u) == 15u && *failed != 0) return false;
    }
    *failed = 1;
    atomicOr_system(error_flag, 1u);
    return false;
}
// The same for a whole warp, with one answer.
template <bool CLUSTER = false>
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* failed, unsigned int* error_flag) {
    return __all_sync(kFullMask, lane_wait<CLUSTER>(bar, parity, failed, error_flag));
}

// For the pairs of a row: from all CTAs of the cluster.
__device__ __forceinline__ bool stat_wait(int cluster, uint64_t* bar, uint32_t parity, volatile int* failed, unsigned int* error_flag) {
    return cluster == 1 ? warp_wait(bar, parity, failed, error_flag) : warp_wait<true>(bar, parity, failed, error_flag);
}

// A position in a ring of `size` places: place and the parity of its round.
struct RingPlace {
    int place;
    uint32_t parity;
    __device__ __forceinline__ void next(int size) {
        if (++place == size) {
            place = 0;
            parity ^= 1u;
        }
    }
};

// The part of a row that a CTA of the cluster owns: aligned packs [lo, hi), in chunks of kChunkPacks.
constexpr int kChunkPacks = kChunkBytes / 16;
template <class T>
struct Slice {
    int head, tail, lo, hi;  // (the edges are in elements)
    int packs, chunks;
    __device__ __forceinline__ Slice(const T* row, int vocab, int rank, int log2_cluster) {
        const RowSpan<T> span(row, vocab);
        head = span.head;
        tail = span.tail;
        packs = span.packs;
        lo = static_cast<int>(static_cast<int64_t>(packs) * rank >> log2_cluster);
        hi = static_cast<int>(static_cast<int64_t>(packs) * (rank + 1) >> log2_cluster);
        chunks = (hi - lo + kChunkPacks - 1) / kChunkPacks;
    }
    __device__ __forceinline__ int begin(int c) const { return lo + c * kChunkPacks; }
    __device__ __forceinline__ int size(int c) const { return min(kChunkPacks, hi - begin(c)); }
    __device__ __forceinline__ int edges() const { return head + tail; }
    __device__ __forceinline__ int edge_col(int i, int vocab) const { return i < head ? i : vocab - tail + (i - head); }
    // Whether `col` is one of the aligned packs.
    __device__ __forceinline__ bool inner(int col) const { return static_cast<unsigned>(col - head) < static_cast<unsigned>(packs) * kPack<T>; }
    // Whether this CTA writes the gradient of `col` (rank 0 has the edges).
    __device__ __forceinline__ bool owns(int col, int rank) const {
        if (!inner(col)) return rank == 0;
        const int pack = (col - head) / kPack<T>;
        return pack >= lo && pack < hi;
    }
};

template <class T, bool LOSS, bool GRAD>
__global__ void __launch_bounds__(kRingThreads, 1)
distill_ring_kernel(const RingParams r) {
    constexpr int N = kPack<T>;
    constexpr int kSumGroups = !LOSS ? 0 : GRAD ? 1 : 2, kWriteGroups = !GRAD ? 0 : LOSS ? 1 : 2;
    constexpr int kSumWarps = kSumGroups * kGroupWarps;
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ uint64_t full[kMaxSlots], empty[kMaxSlots], prep_full[kPrepSlots], prep_empty[kPrepSlots], stat_full[kStatSlots];
    __shared__ float2 stat[LOSS ? kStatSlots : 1][kMaxCluster * (GRAD ? 1 : 2) * kGroupWarps];
    __shared__ Prepared prepared[kPrepSlots];
    __shared__ int failed_word;
    volatile int* const failed = &failed_word;
    const DistillParams& p = r.d;
    const int warp = threadIdx.x / kWarp, lane = threadIdx.x & (kWarp - 1);
    const int rank = static_cast<int>(cluster_rank()), cluster = static_cast<int>(cluster_size());
    const int64_t teams = gridDim.x / cluster, id = blockIdx.x / cluster;
    const int log2_cluster = 31 - __clz(cluster);
    const float c = static_cast<float>(kLog2e * p.inv_temperature);
    unsigned char* const ring = smem;
    float* const probs = reinterpret_cast<float*>(smem + static_cast<size_t>(r.slots) * kChunkBytes);  // [prep slots][k] each
    float* const heres = probs + kPrepSlots * p.k;
    int* const ats = reinterpret_cast<int*>(heres + kPrepSlots * p.k);
    uint16_t* const tables = reinterpret_cast<uint16_t*>(ats + kPrepSlots * p.k);
    if (threadIdx.x == 0) {
        for (int i = 0; i < r.slots; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], kGroupWarps);
        }
        for (int i = 0; i < kPrepSlots; ++i) {
            mbar_init(&prep_full[i], 1);
            mbar_init(&prep_empty[i], 2 * kGroupWarps + 1);
        }
        for (int i = 0; i < kStatSlots; ++i) mbar_init(&stat_full[i], cluster == 1 && LOSS ? kSumWarps : 1);
        failed_word = 0;
        fence_mbar_init();
    }
    __syncthreads();
    if (cluster > 1) cluster_sync_all();  // every CTA's barriers are there before the first remote arrival
    pdl_wait();

    if (warp == 0) {
        // ---- copies ----
        if (lane == 0) {
            RingPlace slot{0, 1}, prep{0, 0};  // the first round finds every place empty
            int64_t asked = 0;
            for (int64_t row = id; row < p.rows; row += teams) {
                if (!lane_wait(&prep_full[prep.place], prep.parity, failed, r.error_flag)) break;
                const bool live = prepared[prep.place].live != 0;
                mbar_arrive(&prep_empty[prep.place]);
                prep.next(kPrepSlots);
                if (!live) continue;
                const T* z = static_cast<const T*>(p.logits) + row * p.logits_stride;
                const Slice<T> slice(z, p.vocab, rank, log2_cluster);
                const T* body = z + slice.head;
                int i = 0;
                for (; i < slice.chunks; ++i) {
                    if (!lane_wait(&empty[slot.place], slot.parity, failed, r.error_flag)) break;
                    const uint32_t bytes = static_cast<uint32_t>(slice.size(i)) * 16u;
                    mbar_expect_tx(&full[slot.place], bytes);
                    bulk_g2s(ring + static_cast<size_t>(slot.place) * kChunkBytes, body + static_cast<int64_t>(slice.begin(i)) * N,
                             bytes, &full[slot.place]);
                    slot.next(r.slots);
                    ++asked;
                }
                if (i < slice.chunks) break;
            }
            if (*failed != 0) {  // copies that nobody waits for any more must not outlive the CTA
                for (int64_t n = asked > r.slots ? asked - r.slots : 0; n < asked; ++n) {
                    mbar_wait_bounded(&full[n % r.slots], static_cast<uint32_t>(n / r.slots) & 1u);
                }
            }
        }
        __syncwarp();
    } else if (warp < kFirstWorker) {
        // ---- the teacher's entries ----
        uint16_t* const table = tables + (warp - 1) * r.table;
        for (int64_t number = warp - 1; id + number * teams < p.rows; number += kPrepWarps) {
            const int64_t row = id + number * teams;
            const int place = static_cast<int>(number % kPrepSlots);
            // The first round finds the slots free.
            if (!warp_wait(&prep_empty[place], static_cast<uint32_t>(number / kPrepSlots & 1) ^ 1u, failed, r.error_flag)) break;
            Prepared& out = prepared[place];
            const T* z = static_cast<const T*>(p.logits) + row * p.logits_stride;
            const Slice<T> slice(z, p.vocab, rank, log2_cluster);
            const float weight = p.row_weight == nullptr ? 1.0f : p.row_weight[row];
            double base = 0.0, mass = 0.0;
            // (The gradient alone, in place: another CTA may be writing its part of the row already.)
            const bool live = weight != 0.0f &&
                              read_entries<T, LOSS, GRAD>(p, z, row, c, Entries{probs + place * p.k, heres + place * p.k, ats + place * p.k, table, r.table},
                                                          &base, &mass, [&](int col) { return LOSS || slice.owns(col, rank); });
            if (live) {
                if (lane < slice.edges() && (LOSS || rank == 0)) out.edge[lane] = to_f32(z[slice.edge_col(lane, p.vocab)]);
                if (lane == 0) {
                    out.base = base;
                    out.mass = mass;
                    if (!LOSS) {
                        out.m = p.row_stats[2 * row];
                        out.total = p.row_stats[2 * row + 1];
                    }
                }
            }
            if (lane == 0) {
                out.weight = weight;
                out.live = live;
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&prep_full[place]);
        }
    } else if (warp - kFirstWorker < kSumWarps) {
        // ---- the sums ----
        const int w = warp - kFirstWorker, group = w / kGroupWarps, tg = (w % kGroupWarps) * kWarp + lane;
        RingPlace slot{0, 0}, prep{0, 0};
        int64_t live_rows = 0;
        struct Last {  // the loss alone: a row is closed after the sums of the next (warp 0)
            int64_t row, number;
            int place;
        } last{-1, 0, 0};
        auto row_of_stats = [&](int64_t number) { return &stat[number % kStatSlots][0]; };
        auto close = [&]() {
            if (!stat_wait(cluster, &stat_full[last.number % kStatSlots], static_cast<uint32_t>(last.number / kStatSlots & 1), failed, r.error_flag)) return false;
            const float2 f = fold_stats(row_of_stats(last.number), cluster * kSumWarps, c);
            if (rank == 0 && lane == 0) write_loss(p, prepared[last.place].base, prepared[last.place].mass, last.row, f);
            __syncwarp();
            if (lane == 0) mbar_arrive(&prep_empty[last.place]);
            last.row = -1;
            return true;
        };
        for (int64_t row = id; row < p.rows; row += teams) {
            if (!warp_wait(&prep_full[prep.place], prep.parity, failed, r.error_flag)) break;
            const bool live = prepared[prep.place].live != 0;
            bool keep = false;
            if (live) {
                const T* z = static_cast<const T*>(p.logits) + row * p.logits_stride;
                const Slice<T> slice(z, p.vocab, rank, log2_cluster);
                Running run;
                bool ok = true;
                for (int i = 0; i < slice.chunks; ++i, slot.next(r.slots)) {
                    if (kSumGroups > 1 && (slot.place & 1) != group) continue;
                    ok = warp_wait(&full[slot.place], slot.parity, failed, r.error_flag);
                    if (!ok) break;
                    const uint4* chunk = reinterpret_cast<const uint4*>(ring + static_cast<size_t>(slot.place) * kChunkBytes);
                    const int n = slice.size(i);
                    uint4 raw[kBatch];
#pragma unroll
                    for (int q = 0; q < kBatch; ++q) raw[q] = tg + q * kGroup < n ? chunk[tg + q * kGroup] : lowest_pack(T{});
                    run.take<T>(raw, c);
                    // The place is given back once every lane's loads have returned, not when they are under way: the
                    // vote needs sums of all of them (a sum is never -1).
                    if (!GRAD && !__any_sync(kFullMask, run.s == -1.0f) && lane == 0) mbar_arrive(&empty[slot.place]);
                }
                if (!ok) break;
                if (rank == 0 && w == 0 && lane < slice.edges()) run.take_one(prepared[prep.place].edge[lane], c);
                const float2 mine = run.of_warp(c);
                uint64_t* bar = &stat_full[live_rows % kStatSlots];
                if (cluster == 1) {  // launched without a cluster: nothing but the CTA's own shared memory
                    if (lane == 0) {
                        row_of_stats(live_rows)[w] = mine;
                        mbar_arrive(bar);
                    }
                } else {
                    if (w == 0 && lane == 0) mbar_expect_tx(bar, static_cast<uint32_t>(cluster * kSumWarps * sizeof(float2)));
                    if (lane < cluster) send_stat(row_of_stats(live_rows) + rank * kSumWarps + w, bar, lane, mine);
                }
                if (!GRAD && w == 0) {
                    if (last.row >= 0 && !close()) break;
                    last = Last{row, live_rows, prep.place};
                    keep = true;
                }
                ++live_rows;
            } else if (!GRAD && w == 0) {
                // Slots are given back in the order of their rows: their barriers tell one round from the next only.
                if (last.row >= 0 && !close()) break;
                if (rank == 0 && lane == 0) write_left_out(p, row);
            }
            __syncwarp();
            if (!keep && lane == 0) mbar_arrive(&prep_empty[prep.place]);
            prep.next(kPrepSlots);
        }
        if (!GRAD && w == 0 && last.row >= 0 && *failed == 0) close();
    } else {
        // ---- the writes ----
        const int w = warp - kFirstWorker - kSumWarps, group = w / kGroupWarps, tg = (w % kGroupWarps) * kWarp + lane;
        const float scale = p.scale * static_cast<float>(p.inv_temperature) * (p.grad_loss != nullptr ? *p.grad_loss : 1.0f);
        RingPlace slot{0, 0}, prep{0, 0};
        int64_t live_rows = 0;
        for (int64_t row = id; row < p.rows; row += teams) {
            if (!warp_wait(&prep_full[prep.place], prep.parity, failed, r.error_flag)) break;
            const Prepared& pre = prepared[prep.place];
            const T* z = static_cast<const T*>(p.logits) + row * p.logits_stride;
            T* g = static_cast<T*>(p.grad) + row * p.grad_stride;
            const Slice<T> slice(z, p.vocab, rank, log2_cluster);
            const bool same_phase = ((reinterpret_cast<uintptr_t>(z) ^ reinterpret_cast<uintptr_t>(g)) & 15) == 0;
            T* const body = g + slice.head;
            if (pre.live != 0) {
                float2 f = make_float2(pre.m, pre.total);
                if (LOSS) {
                    if (!stat_wait(cluster, &stat_full[live_rows % kStatSlots], static_cast<uint32_t>(live_rows / kStatSlots & 1), failed, r.error_flag)) break;
                    f = fold_stats(&stat[live_rows % kStatSlots][0], cluster * kSumWarps, c);
                    if (rank == 0 && w == 0 && lane == 0) write_loss(p, pre.base, pre.mass, row, f);
                    ++live_rows;
                }
                const float m = f.x, total = f.y, coef = scale * pre.weight;
                const float mass = p.teacher_lse == nullptr && pre.mass == pre.mass ? 1.0f : static_cast<float>(pre.mass);
                const float each = coef * mass / total;
                const int start = slot.place;
                bool ok = true;
                for (int i = 0; i < slice.chunks; ++i, slot.next(r.slots)) {
                    if (kWriteGroups > 1 && (slot.place & 1) != group) continue;
                    ok = warp_wait(&full[slot.place], slot.parity, failed, r.error_flag);
                    if (!ok) break;
                    const unsigned char* chunk = ring + static_cast<size_t>(slot.place) * kChunkBytes;
                    const int n = slice.size(i);
                    T* const out = body + static_cast<int64_t>(slice.begin(i)) * N;
                    if (same_phase) {
                        uint4 raw[kBatch];
#pragma unroll
                        for (int q = 0; q < kBatch; ++q) raw[q] = reinterpret_cast<const uint4*>(chunk)[tg + q * kGroup];
                        const float2 down = both(-m), c2 = both(c), each2 = both(each);
                        T* const mine = out + static_cast<int64_t>(tg) * N;
#pragma unroll
                        for (int q = 0; q < kBatch; ++q) {
                            if (tg + q * kGroup >= n) break;
                            float2 v[N / 2];
                            unpack2(raw[q], v, T{});
#pragma unroll
                            for (int e = 0; e < N / 2; ++e) {
                                v[e] = mul2(add2(v[e], down), c2);
                                v[e] = mul2(make_float2(ex2_approx(v[e].x), ex2_approx(v[e].y)), each2);
                            }
                            store_pairs(mine + q * kGroup * N, v);
                        }
                    } else {
                        for (int q = tg; q < n * N; q += kGroup) {
                            out[q] = from_f32<T>(ex2_approx((to_f32(reinterpret_cast<const T*>(chunk)[q]) - m) * c) * each);
                        }
                    }
                    // Behind the stores, which need what the lanes loaded: a place given back while loads are still
                    // under way is overwritten under them.
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&empty[slot.place]);
                }
                if (!ok) break;
                if (rank == 0 && w == 0 && lane < slice.edges()) {
                    g[slice.edge_col(lane, p.vocab)] = from_f32<T>(ex2_approx((pre.edge[lane] - m) * c) * each);
                }
                // The columns that the teacher names: each warp writes those of its own share of the row again,
                // so that no barrier has to come between them and the dense part.
                __syncwarp();
                for (int j = lane; j < p.k; j += kWarp) {
                    const int col = ats[prep.place * p.k + j];
                    if (col < 0 || !slice.owns(col, rank)) continue;
                    int owner = 0;  // of the edges
                    if (slice.inner(col)) {
                        const int pack = (col - slice.head) / N - slice.lo, in = pack % kChunkPacks;
                        owner = (same_phase ? in : in * N + (col - slice.head) % N) % kGroup / kWarp;
                        if (kWriteGroups > 1) owner += ((start + pack / kChunkPacks) % r.slots & 1) * kGroupWarps;
                    }
                    if (owner != w) continue;
                    const float q = ex2_approx((heres[prep.place * p.k + j] - m) * c) / total;
                    g[col] = from_f32<T>(coef * (mass * q - probs[prep.place * p.k + j]));
                }
            } else {  // left out
                if (LOSS && rank == 0 && w == 0 && lane == 0) write_left_out(p, row);
                T* const out = body + static_cast<int64_t>(slice.lo) * N;
                const int n = slice.hi - slice.lo, t = w * kWarp + lane;
                if (same_phase) {
                    for (int q = t; q < n; q += kWriteGroups * kGroup) __stcs(reinterpret_cast<uint4*>(out) + q, make_uint4(0, 0, 0, 0));
                } else {
                    for (int q = t; q < n * N; q += kWriteGroups * kGroup) out[q] = from_f32<T>(0.0f);
                }
                if (rank == 0 && t < slice.edges()) g[slice.edge_col(t, p.vocab)] = from_f32<T>(0.0f);
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&prep_empty[prep.place]);
            prep.next(kPrepSlots);
        }
    }
    __syncthreads();
    if (cluster > 1) cluster_sync_all();  // no CTA leaves while another may still send to it
}

// loss = scale * sum of weight * row loss, in 64 bits and in a fixed order.
__global__ void __launch_bounds__(1024)
distill_mean_kernel(const float* row_loss, const float* row_weight, int64_t rows, float scale, float* loss) {
    __shared__ double red[1024 / kWarp];
    pdl_wait();
    double s = 0.0;
#pragma unroll 8
    for (int64_t r = threadIdx.x; r < rows; r += blockDim.x) {
        const float w = row_weight == nullptr ? 1.0f : row_weight[r], loss = row_loss[r];
        s += w != 0.0f ? static_cast<double>(w) * loss : 0.0;
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

// Clusters of `cluster` ring CTAs that fit the device at once (asked once for each kernel, size and device).
template <class K>
int active_clusters(K kernel, std::atomic<int>* cache, const DeviceInfo* info, int cluster, size_t smem, int* out) {
    if (cluster == 1) {
        *out = info->sm_count;
        return FDL_OK;
    }
    int log2 = 0;
    while ((1 << log2) < cluster) ++log2;
    std::atomic<int>& known = cache[(info->device % kMaxDevicesTracked) * 4 + log2];
    if (known.load() == 0) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(static_cast<unsigned int>(info->sm_count / cluster * cluster));
        cfg.blockDim = dim3(kRingThreads);
        cfg.dynamicSmemBytes = smem;
        cudaLaunchAttribute attr;
        attr.id = cudaLaunchAttributeClusterDimension;
        attr.val.clusterDim.x = static_cast<unsigned int>(cluster);
        attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
        cfg.attrs = &attr;
        cfg.numAttrs = 1;
        int n = 0;
        const cudaError_t e = cudaOccupancyMaxActiveClusters(&n, kernel, &cfg);
        if (e != cudaSuccess) return static_cast<int>(e);
        known.store(n < 1 ? 1 : n);
    }
    *out = known.load();
    return FDL_OK;
}

template <class T, bool LOSS, bool GRAD>
int launch_ring(const DistillParams& p, const DeviceInfo* info, int cluster, int slots, int table, cudaStream_t stream) {
    static std::atomic<int> cache[kMaxDevicesTracked * 4] = {};
    auto kernel = distill_ring_kernel<T, LOSS, GRAD>;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kRingSmem);
    if (e != cudaSuccess) return static_cast<int>(e);
    int most = 0;
    int status = active_clusters(kernel, cache, info, cluster, kRingSmem, &most);
    if (status != FDL_OK) return status;
    RingParams r{p, slots, table, nullptr};
    status = error_flag_device_ptr(&r.error_flag);
    if (status != FDL_OK) return status;
    const int64_t teams = p.rows < most ? p.rows : most;
    return launch_ex(kernel, dim3(static_cast<unsigned int>(teams * cluster)), dim3(kRingThreads), kRingSmem, stream,
                     dim3(static_cast<unsigned int>(cluster), 1, 1), tuning().pdl != 0, r);
}

// Rows of more than this many bytes take the ring form: what eight warps hold.
constexpr int64_t kRingFromBytes = 8 * kWarp * kHeld * 16;

template <class T, bool LOSS, bool GRAD, int WARPS, int HELD>
int launch_held(const DistillParams& p, int places, cudaStream_t stream) {
    constexpr int teams = WARPS == 1 ? 256 / kWarp : 1;
    const size_t smem = static_cast<size_t>(teams) * (static_cast<size_t>(p.k) * 12 + static_cast<size_t>(places) * 2);
    auto kernel = distill_rows_kernel<T, LOSS, GRAD, WARPS, HELD>;
    if (smem > 48 * 1024) {  // (the most that a call takes, not this one's: another thread may be between its own two calls)
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, teams * kMaxEntries * 16);
        if (e != cudaSuccess) return static_cast<int>(e);
    }
    return launch_ex(kernel, dim3(static_cast<unsigned int>(ceil_div(p.rows, teams))), dim3(teams * WARPS * kWarp), smem, stream,
                     dim3(1, 1, 1), tuning().pdl != 0, p, places);
}

template <bool LOSS, bool GRAD>
int launch_rows(const DistillParams& p, int dtype, cudaStream_t stream) {
    int status = FDL_OK;
    const DeviceInfo* info = current_device_info(&status);
    if (info == nullptr) return status;
    const int64_t bytes = static_cast<int64_t>(p.vocab) * static_cast<int64_t>(dtype_bytes(dtype));
    int table = 64;
    while (table < 2 * p.k) table *= 2;
    if (bytes > kRingFromBytes) {
        const int64_t entries = static_cast<int64_t>(kPrepSlots) * p.k * 12 + kPrepWarps * 2 * table;
        int64_t slots = (kRingSmem - entries) / kChunkBytes;
        if (slots > kMaxSlots) slots = kMaxSlots;
        // Loss and gradient together: a CTA's part of the row stays in the ring, with three chunks of the next.
        int cluster = 1;
        auto chunks = [&]() { return ceil_div(ceil_div(bytes, cluster), kChunkBytes) + 1; };
        while (LOSS && GRAD && cluster < kMaxCluster && chunks() + 3 > slots) cluster *= 2;
        // Fewer rows than SMs: more CTAs a row, down to a chunk each.
        while (cluster < kMaxCluster && p.rows * cluster * 2 <= info->sm_count && bytes > static_cast<int64_t>(cluster) * kChunkBytes) {
            cluster *= 2;
        }
        if (!(LOSS && GRAD) || chunks() + 1 <= slots) {
            return with_dtype(dtype, [&](auto* tag) {
                using T = std::remove_pointer_t<decltype(tag)>;
                return launch_ring<T, LOSS, GRAD>(p, info, cluster, static_cast<int>(slots), table, stream);
            });
        }
        // Longer than a cluster's shared memory: the loss, then the gradient from its statistics.
        status = launch_rows<true, false>(p, dtype, stream);
        return status != FDL_OK ? status : launch_rows<false, true>(p, dtype, stream);
    }
    return with_dtype(dtype, [&](auto* tag) {
        using T = std::remove_pointer_t<decltype(tag)>;
        constexpr int64_t warp_bytes = kWarp * kHeld * 16;
        if (bytes <= warp_bytes / 2) return launch_held<T, LOSS, GRAD, 1, kHeld / 2>(p, table, stream);
        if (bytes <= warp_bytes) return launch_held<T, LOSS, GRAD, 1, kHeld>(p, table, stream);
        if (bytes <= 2 * warp_bytes) return launch_held<T, LOSS, GRAD, 2, kHeld>(p, table, stream);
        if (bytes <= 4 * warp_bytes) return launch_held<T, LOSS, GRAD, 4, kHeld>(p, table, stream);
        return launch_held<T, LOSS, GRAD, 8, kHeld>(p, table, stream);
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
