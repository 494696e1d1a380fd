// log_probs.cu — log probabilities of given entries, entropy and top alternatives of softmax(z / T) over each list.
//
// With a reference m near max z, y_j = (z_j - m) log2(e) / T, S = sum 2^y and V = sum 2^y y:
//   log p_j = (z_j - m) / T - ln S,  log sum = m / T + ln S,  entropy = ln S - ln 2 V / S.
// Statistics are f32 sums over one pass; the alternatives are ordered by the scores themselves (ties by the lower
// index), so no rounding decides an index.
//
// Lists of at most kWarpEntries take a warp each, in registers. Longer ones take a CTA (few of them: a cluster of
// CTAs), which reads the list once: the maxima of the first batch give the reference, a bound that at least `top`
// entries reach, and so a filter; vectors that pass it are held in shared memory, their entries cut to the alternatives
// so far each time the read part has doubled, and ranked at the end. More candidates than the buffer holds (a list in
// ascending order, or of equal scores) have the alternatives selected digit by digit of their keys.
//
// What bounds it, on one B200 (copy rate 6453 GB/s): 4096 lists of 131072 bf16 scores, top 20, take 257 us, 4.2 TB/s,
// 0.65 of the copy rate (243 us where one input is repeated, as in the comparisons below). Per vector of 8 scores a warp
// issues about 65 instructions and its exponentials take the special-function unit 64 cycles; issue is 65% busy, that unit
// 51%, DRAM 48% under the profiler (1184 lists). Read the list twice (maximum first) and L2 would carry it once more; so one
// pass, about a reference that moves. Candidates as whole vectors: testing and storing each entry cost about 100
// instructions a hit, a vector costs 25. A short list's time is its chain of loads, barriers and selections: one list of
// 131072, as a cluster of 8, takes 10 us, 16,700 lists of 120 f32, a warp each, 17.5 us.
#include "lists_device.cuh"

namespace cg = cooperative_groups;

namespace sb2 {

namespace {

constexpr uint32_t kWarpEntries = 512;
// The mean length up to which runs between boundaries go by warps, the longer ones among them by whole CTAs: 20,000 lists
// of 300 to 400 take 61 us so and 94 by a CTA each; of widely spread lengths about 300, 113 and 100.
constexpr uint32_t kWarpMean = 384;
constexpr int kWarpThreads = 256;        // the warp kernel's CTAs
constexpr uint32_t kCandidates = 2048;   // keys that a CTA gathers
constexpr int kBatch = 4;                // vectors a thread holds in flight (2: 286 us above, 4: 246, 8: 258)
constexpr uint32_t kSingle = 0x80000000u;
constexpr uint32_t kRanked = 256;        // keys that are ranked by counting

// What a CTA keeps of its share of a list.
template <int kThreads>
struct Shared {
    unsigned long long key[kCandidates];
    unsigned long long best[kMaxTop];  // the share's alternatives, likeliest first; 0 behind the last
    uint32_t order[256];               // group maxima, then the digits' counts
    float warp[3][kThreads / 32];
    Stats stats;
    uint32_t bound;                    // the order of the least score of an alternative
    uint32_t held[kCandidates];        // first entries of vectors that hold candidates (kSingle: an entry alone)
    uint32_t count, keys, digit, left;
};

// The next free slot of a buffer in shared memory. Rarely more than one lane of a warp asks, so the plain atomic is
// cheaper than one for the warp and a share of it per lane.
__device__ __forceinline__ uint32_t take(uint32_t* counter) {
    uint32_t at;
    asm volatile("atom.shared.add.u32 %0, [%1], 1;"
                 : "=r"(at)
                 : "r"(static_cast<uint32_t>(__cvta_generic_to_shared(counter)))
                 : "memory");
    return at;
}

// The `top`-th largest of the keys that `each` hands to its argument (at least `top`, all different), digit by digit:
// the keys that share the digits so far are counted by the next one. A warp's lanes hand theirs over together, a lane
// without one with `here` false. Digits that all keys of `T` scores and of indices
// below `n` share are known: an index's high ones, and those of a 16-bit score's low half as f32, which its sign sets.
template <class T, int kThreads, class Each>
__device__ __forceinline__ unsigned long long nth_key(Shared<kThreads>& s, uint32_t top, uint32_t n, Each each) {
    unsigned long long prefix = 0;
    uint32_t left = top;
    for (int shift = 56; shift >= 0; shift -= 8) {
        const bool score = sizeof(T) == 2 && (shift == 32 || (shift == 40 && std::is_same_v<T, __nv_bfloat16>));
        if (score || (shift < 32 && shift > 0 && n <= 1u << shift)) {
            if (!score || (prefix >> 63) == 0) prefix |= 0xFFull << shift;
            continue;
        }
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < 256; i += kThreads) s.order[i] = 0;
        __syncthreads();
        each([&](unsigned long long key, bool here) {
            here = here && (shift == 56 || (key >> (shift + 8)) == (prefix >> (shift + 8)));
            const uint32_t d = static_cast<uint32_t>(key >> shift) & 255u, lanes = __ballot_sync(kFull, here);
            if (!here) return;
            // Equal scores share their digits: one addition for the lanes that are here.
            int same;
            __match_all_sync(lanes, d, &same);
            if (same == 0)
                atomicAdd(&s.order[d], 1u);
            else if ((threadIdx.x & 31) == static_cast<uint32_t>(__ffs(lanes)) - 1)
                atomicAdd(&s.order[d], static_cast<uint32_t>(__popc(lanes)));
        });
        __syncthreads();
        if (threadIdx.x < 32) {  // a lane sums 8 digits; the lane whose digits hold the one that is looked for finds it
            const uint32_t lane = threadIdx.x;
            uint32_t sum = 0;
            for (uint32_t k = 0; k < 8; ++k) sum += s.order[255 - 8 * lane - k];
            uint32_t upto = sum;
            for (uint32_t o = 1; o < 32; o <<= 1) {
                const uint32_t u = __shfl_up_sync(kFull, upto, o);
                if (lane >= o) upto += u;
            }
            if (upto >= left && upto - sum < left) {
                uint32_t need = left - (upto - sum), d = 255 - 8 * lane;
                while (s.order[d] < need) need -= s.order[d--];
                s.digit = d;
                s.left = s.order[d] == need ? 0 : need;  // 0: all keys with these digits belong
            }
        }
        __syncthreads();
        prefix |= static_cast<unsigned long long>(s.digit) << shift;
        left = s.left;
        if (left == 0) break;
    }
    return prefix;
}

// The `top` largest of `count` gathered keys into s.best, in order: every key counts the keys above it, of more than
// kRanked only the `top` largest (of 512 keys the counting takes 37,000 instructions, finding the top-th 7,000). Ends
// without a barrier behind the writes of s.best.
template <class T, int kThreads>
__device__ __forceinline__ void rank_candidates(Shared<kThreads>& s, uint32_t count, uint32_t top, uint32_t n) {
    const uint32_t t = threadIdx.x;
    if (count > kRanked) {
        const unsigned long long last = nth_key<T>(s, top, n, [&](auto f) {
            for (uint32_t base = 0; base < count; base += kThreads) {
                const uint32_t i = base + t;
                f(i < count ? s.key[i] : 0ull, i < count);
            }
        });
        if (t == 0) s.count = 0;
        __syncthreads();
        for (uint32_t i = t; i < count; i += kThreads)
            if (s.key[i] >= last) s.best[take(&s.count)] = s.key[i];
        __syncthreads();
        unsigned long long mine = 0;
        uint32_t above = 0;
        if (t < top) {
            mine = s.best[t];
            for (uint32_t j = 0; j < top; ++j) above += s.best[j] > mine;
        }
        __syncthreads();
        if (t < top) s.best[above] = mine;
        return;
    }
    for (uint32_t i = t; i < top; i += kThreads) s.best[i] = 0;
    __syncthreads();
    for (uint32_t i = t; i < count; i += kThreads) {
        const unsigned long long mine = s.key[i];
        uint32_t above = 0, j = 0;
        for (; j + 4 <= count; j += 4) {
            const ulonglong2 a = *reinterpret_cast<const ulonglong2*>(&s.key[j]);
            const ulonglong2 b = *reinterpret_cast<const ulonglong2*>(&s.key[j + 2]);
            above += (a.x > mine) + (a.y > mine) + (b.x > mine) + (b.y > mine);
        }
        for (; j < count; ++j) above += s.key[j] > mine;
        if (above < top) s.best[above] = mine;
    }
}

// Entries [from, to) of the vectors and, for share 0, the scalars outside them, each to `f(score, index, true)`. A warp's
// lanes call `f` together: one that has no entry left with -inf and false.
template <class T, int kVec, int kThreads, class F>
__device__ __forceinline__ void for_share(const Walk<T, kVec>& w, uint32_t from, uint32_t to, bool edges, F f) {
    for (uint32_t base = from; base < to; base += kThreads) {
        const uint32_t v = base + threadIdx.x;
        Pack<T, kVec> p;
        p.masked();
        if (v < to) p.load(w.z + w.at(v));
        float x[kVec];
        p.values(x);
        for (int e = 0; e < kVec; ++e) f(x[e], w.at(v) + e, v < to);
    }
    if (edges) {
        const uint32_t j = threadIdx.x < 2 * kVec ? w.edge(threadIdx.x) : w.n;
        f(j < w.n ? to_float(w.z[j]) : -CUDART_INF_F, j, j < w.n);
    }
}

// The share's `top` largest keys as the candidates, whatever the order or the ties. The share holds at least as many
// unmasked entries.
template <class T, int kVec, int kThreads>
__device__ __noinline__ void select_candidates(Shared<kThreads>& s, const T* z, uint32_t n, uint32_t from, uint32_t to, bool edges,
                                               uint32_t top) {
    const Walk<T, kVec> w(z, n);
    auto each = [&](auto f) {
        for_share<T, kVec, kThreads>(w, from, to, edges, [&](float x, uint32_t j, bool) { f(order_key(x, j), x > -CUDART_INF_F); });
    };
    const unsigned long long last = nth_key<T>(s, top, n, each);
    if (threadIdx.x == 0) s.keys = 0;
    __syncthreads();
    each([&](unsigned long long key, bool here) {
        if (here && key >= last) s.key[take(&s.keys)] = key;
    });
    __syncthreads();
}

// The statistics of a share of far scores (about 700,000 T and more from 0): the maximum first, then each entry's
// distance from it.
template <class T, int kVec, int kThreads>
__device__ __noinline__ Stats far_stats(Shared<kThreads>& s, const T* z, uint32_t n, uint32_t from, uint32_t to, bool edges,
                                        float c) {
    const Walk<T, kVec> w(z, n);
    Stats a{-FLT_MAX, 0.0f, 0.0f};
    for_share<T, kVec, kThreads>(w, from, to, edges, [&](float x, uint32_t, bool) { a.m = fmaxf(a.m, x); });
    for_share<T, kVec, kThreads>(w, from, to, edges, [&](float x, uint32_t, bool here) {
        if (!here) return;
        const float y = exponent(x, a.m, c), p = pow2(y);
        a.s += p;
        a.v = __fmaf_rn(p, y, a.v);
    });
    return a;
}

// The candidates' keys: entries of the held vectors that reach the bound. False: more than the buffer holds.
template <class T, int kVec, int kThreads>
__device__ __forceinline__ bool expand(Shared<kThreads>& s, const T* z, float bound) {
    __syncthreads();
    const uint32_t count = s.count;
    if (count > kCandidates) return false;
    if (threadIdx.x == 0) s.keys = 0;
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < count * kVec; i += kThreads) {
        const uint32_t held = s.held[i / kVec], e = i % kVec;
        const uint32_t j = (held & ~kSingle) + e;
        if ((held & kSingle) != 0 && e > 0) continue;
        const float x = to_float(z[j]);
        if (x >= bound || (held & kSingle) != 0) {
            const uint32_t at = take(&s.keys);
            if (at < kCandidates) s.key[at] = order_key(x, j);
        }
    }
    __syncthreads();
    return s.keys <= kCandidates;
}

// A given entry's score, -inf for an index outside the list.
template <class T>
__device__ __forceinline__ float given_score(const T* z, uint32_t n, int32_t id) {
    return id >= 0 && static_cast<uint32_t>(id) < n ? to_float(z[id]) : -CUDART_INF_F;
}
// ... and its log probability: a masked entry's is -inf, but NaN beside a NaN or +inf as all of that list's.
__device__ __forceinline__ float given_log_prob(float z, uint32_t n, int32_t id, float m, float inv_t, float log_s) {
    if (z == -CUDART_INF_F) return log_s == log_s || id < 0 || static_cast<uint32_t>(id) >= n ? z : log_s;
    return (z - m) * inv_t - log_s;
}

// One list by `shares` CTAs, this one the `share`-th: a cluster, or a CTA alone (shares 1).
template <class T, int kVec, int kThreads, bool kCluster>
__device__ __forceinline__ void log_probs_list(Shared<kThreads>& s, const LogProbsArgs& a, uint32_t i, uint32_t share,
                                               uint32_t shares) {
    const uint32_t t = threadIdx.x, lane = t & 31, warp = t >> 5;
    uint64_t first;
    uint32_t n;
    list_range(a.l, i, first, n);
    const Walk<T, kVec> w(static_cast<const T*>(a.l.scores) + first, n);
    const uint32_t from = static_cast<uint32_t>(static_cast<uint64_t>(w.vectors) * share / shares);
    const uint32_t to = static_cast<uint32_t>(static_cast<uint64_t>(w.vectors) * (share + 1) / shares);
    const float c = __fmul_rn(kLog2E, a.inv_t);
    // The given entries' scores, on their way while the list is read.
    int32_t id = -1;
    if (share == 0 && t < a.num_given) id = a.given[static_cast<uint64_t>(i) * a.num_given + t];
    float given = given_score(w.z, n, id);
    // The first batch, and the scalars outside the vectors (share 0): their maximum.
    Pack<T, kVec> p[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
        const uint32_t v = from + u * kThreads + t;
        if (v < to)
            p[u].load(w.z + w.at(v));
        else
            p[u].masked();
    }
    float edge[1] = {-CUDART_INF_F};
    const uint32_t edge_at = share == 0 && t < 2 * kVec ? w.edge(t) : n;
    if (edge_at < n) edge[0] = to_float(w.z[edge_at]);
    float most = edge[0];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) most = fmaxf(most, p[u].most());
    // Groups of threads: `top` groups reach the top-th largest of their maxima, so `top` entries do.
    const uint32_t groups = min(static_cast<uint32_t>(kThreads), a.top > 64 ? 256u : 128u), per = kThreads / groups;
    float group = most;
    for (uint32_t o = 1; o < per; o <<= 1) group = fmaxf(group, __shfl_xor_sync(kFull, group, o));
    if (t % per == 0) s.order[t / per] = order_of(group);
    most = warp_max(most);
    if (lane == 0) s.warp[0][warp] = most;
    if (t == 0) {
        s.count = 0;
        s.bound = 0xFFFFFFFFu;
    }
    __syncthreads();
    most = s.warp[0][0];
#pragma unroll
    for (int k = 1; k < kThreads / 32; ++k) most = fmaxf(most, s.warp[0][k]);
    if (a.top > 0 && t < groups) {  // the least group that fewer than `top` others exceed
        const uint32_t mine = s.order[t];
        uint32_t above = 0;
        for (uint32_t j = 0; j < groups; j += 4) {
            const uint4 o = *reinterpret_cast<const uint4*>(&s.order[j]);
            above += (o.x > mine) + (o.y > mine) + (o.z > mine) + (o.w > mine);
        }
        const uint32_t least = __reduce_min_sync(kFull, above < a.top ? mine : 0xFFFFFFFFu);
        if (lane == 0) atomicMin(&s.bound, least);
    }
    __syncthreads();
    // Masked entries are no alternatives.
    float bound = a.top > 0 ? fmaxf(score_of(s.bound), -FLT_MAX) : CUDART_NAN_F, tie = bound;
    // One pass: the statistics about the first batch's maximum (moved where later entries lie far above it), and the
    // entries that reach the bound.
    Reader<true> r(most, c);
    // A vector (or a scalar) that holds a candidate.
    auto hold = [&](uint32_t first_entry) {
        const uint32_t at = take(&s.count);
        if (at < kCandidates) s.held[at] = first_entry;
    };
    uint32_t batch = 0;
    for (uint32_t base = from; base < to; base += kBatch * kThreads) {
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            const uint32_t v = base + u * kThreads + t;
            if (v < to) {
                float x[kVec];
                const float high = p[u].most();
                p[u].finite(x);
                const uint32_t next = v + kBatch * kThreads;
                if (next < to) p[u].load(w.z + w.at(next));
                if (high > r.limit) r.raise(high);
                r.add(x);
                if (high >= bound) hold(w.at(v));
            }
        }
        // Each time the part that is read has doubled: many candidates are cut to the alternatives so far, whose last
        // the rest has to exceed (an equal score further on comes after it). So candidates stay few however long the
        // list is and however many scores are equal, unless its order defeats that.
        if ((++batch & (batch - 1)) == 0 && a.top > 0 && base + kBatch * kThreads < to) {
            __syncthreads();
            if (s.count > max(64u, 2 * a.top) && expand<T, kVec, kThreads>(s, w.z, bound)) {
                rank_candidates<T>(s, s.keys, a.top, n);
                __syncthreads();
                for (uint32_t k = t; k < a.top; k += kThreads) s.held[k] = index_of(s.best[k]) | kSingle;
                const uint32_t last = static_cast<uint32_t>(s.best[a.top - 1] >> 32);
                tie = score_of(last);
                bound = score_of(last + 1);
                if (t == 0) s.count = a.top;
            }
            __syncthreads();
        }
    }
    if (edge_at < n) {
        if (edge[0] > r.limit) r.raise(edge[0]);
        if (edge[0] >= tie) hold(edge_at | kSingle);
        edge[0] = max_nan(edge[0], kMasked);
        r.add(edge);
    }
    // The share's statistics.
    Stats mine = r.stats();
    if (__syncthreads_or(r.far())) mine = far_stats<T, kVec, kThreads>(s, w.z, n, from, to, share == 0, c);
    const float top_m = warp_max(mine.m);
    rebase(mine, top_m, c);
    mine.s = warp_sum(mine.s);
    mine.v = warp_sum(mine.v);
    if (lane == 0) {
        s.warp[0][warp] = top_m;
        s.warp[1][warp] = mine.s;
        s.warp[2][warp] = mine.v;
    }
    __syncthreads();
    if (warp == 0) {
        Stats part{-FLT_MAX, 0.0f, 0.0f};
        if (lane < kThreads / 32) part = {s.warp[0][lane], s.warp[1][lane], s.warp[2][lane]};
        const float m = warp_max(part.m);
        rebase(part, m, c);
        part.s = warp_sum(part.s);
        part.v = warp_sum(part.v);
        if (lane == 0) s.stats = {m, part.s, part.v};
    }
    // The share's alternatives.
    if (a.top > 0) {
        if (!expand<T, kVec, kThreads>(s, w.z, bound))
            select_candidates<T, kVec, kThreads>(s, w.z, n, from, to, share == 0, a.top);
        rank_candidates<T>(s, s.keys, a.top, n);
    }
    __syncthreads();
    if constexpr (kCluster) {
        // Share 0 joins the others' statistics and alternatives.
        cg::cluster_group cluster = cg::this_cluster();
        cluster.sync();
        if (share == 0) {
            if (t == 0) {
                float m = s.stats.m;
                for (uint32_t k = 1; k < shares; ++k) m = fmaxf(m, cluster.map_shared_rank(&s, k)->stats.m);
                Stats all = s.stats;
                rebase(all, m, c);
                for (uint32_t k = 1; k < shares; ++k) {
                    Stats part = cluster.map_shared_rank(&s, k)->stats;
                    rebase(part, m, c);
                    all.s += part.s;
                    all.v += part.v;
                }
                s.stats = all;
                s.keys = 0;
            }
            __syncthreads();
            for (uint32_t x = t; x < shares * a.top; x += kThreads) {
                const unsigned long long key = cluster.map_shared_rank(&s, x / a.top)->best[x % a.top];
                if (key != 0) s.key[atomicAdd(&s.keys, 1u)] = key;
            }
            __syncthreads();
            if (a.top > 0) rank_candidates<T>(s, s.keys, a.top, n);
        }
        cluster.sync();  // the shares' memory is read
        if (share != 0) return;
    }
    // The list's results.
    const float m = s.stats.m, sum = s.stats.s;
    const bool empty = sum == 0.0f;
    const float log_s = logf(sum);
    if (t == 0) {
        if (a.log_sum != nullptr) a.log_sum[i] = empty ? -CUDART_INF_F : m * a.inv_t + log_s;
        if (a.entropy != nullptr) a.entropy[i] = empty ? 0.0f : log_s - 0.6931471805599453f * s.stats.v / sum;
    }
    for (uint32_t g = t; g < a.num_given; g += kThreads) {
        const uint64_t at = static_cast<uint64_t>(i) * a.num_given + g;
        if (g >= kThreads) {
            id = a.given[at];
            given = given_score(w.z, n, id);
        }
        a.given_out[at] = given_log_prob(given, n, id, m, a.inv_t, log_s);
    }
    for (uint32_t k = t; k < a.top; k += kThreads) {
        const uint64_t at = static_cast<uint64_t>(i) * a.top + k;
        const unsigned long long key = s.best[k];
        a.top_ids[at] = key == 0 ? -1 : static_cast<int32_t>(index_of(key));
        a.top_out[at] = key == 0 ? -CUDART_INF_F : (to_float(w.z[index_of(key)]) - m) * a.inv_t - log_s;
    }
}

template <class T, int kVec, int kThreads, bool kCluster>
__global__ void __launch_bounds__(kThreads) log_probs_rows_kernel(LogProbsArgs a, uint32_t shares) {
    __shared__ __align__(16) Shared<kThreads> s;
    const uint32_t i = kCluster ? blockIdx.x / shares : blockIdx.x;
    log_probs_list<T, kVec, kThreads, kCluster>(s, a, i, kCluster ? blockIdx.x % shares : 0, kCluster ? shares : 1);
}

// A list of at most 32 kItems entries by one warp, in registers.
template <class T, int kItems>
__device__ __forceinline__ void log_probs_warp(const LogProbsArgs& a, uint32_t i, const T* z, uint32_t n) {
    const uint32_t lane = threadIdx.x & 31;
    const float c = __fmul_rn(kLog2E, a.inv_t);
    float x[kItems];
    float most = -CUDART_INF_F;
#pragma unroll
    for (int k = 0; k < kItems; ++k) {
        const uint32_t j = k * 32 + lane;
        x[k] = j < n ? to_float(z[j]) : -CUDART_INF_F;
        most = fmaxf(most, x[k]);
    }
    float m = warp_max(most);
    if (m == -CUDART_INF_F) m = -FLT_MAX;
    float s = 0.0f, v = 0.0f;
#pragma unroll
    for (int k = 0; k < kItems; ++k) {
        const float y = exponent(x[k], m, c), p = pow2(y);
        s += p;
        v = __fmaf_rn(p, y, v);
    }
    s = warp_sum(s);
    v = warp_sum(v);
    const bool empty = s == 0.0f;
    const float log_s = logf(s);
    if (lane == 0) {
        if (a.log_sum != nullptr) a.log_sum[i] = empty ? -CUDART_INF_F : m * a.inv_t + log_s;
        if (a.entropy != nullptr) a.entropy[i] = empty ? 0.0f : log_s - 0.6931471805599453f * v / s;
    }
    for (uint32_t g = lane; g < a.num_given; g += 32) {
        const uint64_t at = static_cast<uint64_t>(i) * a.num_given + g;
        const int32_t id = a.given[at];
        a.given_out[at] = given_log_prob(given_score(z, n, id), n, id, m, a.inv_t, log_s);
    }
    // The alternatives, one a round: each lane keeps its entries in order and offers the first that is left.
    if (a.top == 0) return;
    unsigned long long key[kItems];
#pragma unroll
    for (int k = 0; k < kItems; ++k) key[k] = x[k] > -CUDART_INF_F || x[k] != x[k] ? order_key(x[k], k * 32 + lane) : 0ull;
    if (a.top > 32) {
        // Many: a bitonic sort of the warp's entries, lane l with places l kItems onwards (369 entries, top 128: rounds
        // took 30 us).
#pragma unroll
        for (int size = 2; size <= 32 * kItems; size <<= 1)
#pragma unroll
            for (int stride = size >> 1; stride > 0; stride >>= 1)
#pragma unroll
                for (int k = 0; k < kItems; ++k) {
                    const bool down = ((lane * kItems + k) & size) == 0;  // this stretch: largest first
                    if (stride >= kItems) {
                        const unsigned long long other = __shfl_xor_sync(kFull, key[k], stride / kItems);
                        const bool low = (lane & (stride / kItems)) == 0;
                        if ((key[k] < other) == (low == down)) key[k] = other;
                    } else if ((k ^ stride) > k) {
                        const int o = k ^ stride;
                        const unsigned long long u = key[k], v = key[o];
                        const bool swap = (u < v) == down;
                        key[k] = swap ? v : u;
                        key[o] = swap ? u : v;
                    }
                }
#pragma unroll
        for (int k = 0; k < kItems; ++k) {
            const uint32_t at_top = lane * kItems + k;
            if (at_top >= a.top) continue;
            const uint64_t at = static_cast<uint64_t>(i) * a.top + at_top;
            a.top_ids[at] = key[k] == 0 ? -1 : static_cast<int32_t>(index_of(key[k]));
            a.top_out[at] = key[k] == 0 ? -CUDART_INF_F : (score_of(static_cast<uint32_t>(key[k] >> 32)) - m) * a.inv_t - log_s;
        }
        return;
    }
#pragma unroll
    for (int size = 2; size <= kItems; size <<= 1)  // a bitonic network over the lane's own, largest first
#pragma unroll
        for (int stride = size >> 1; stride > 0; stride >>= 1)
#pragma unroll
            for (int k = 0; k < kItems; ++k) {
                const int o = k ^ stride;
                if (o > k) {
                    const bool swap = (key[k] < key[o]) == ((k & size) == 0);
                    const unsigned long long u = swap ? key[o] : key[k], v = swap ? key[k] : key[o];
                    key[k] = u;
                    key[o] = v;
                }
            }
    uint32_t out_order = 0, out_low = 0;
    for (uint32_t r = 0; r < a.top; ++r) {
        const uint32_t order = static_cast<uint32_t>(key[0] >> 32), low = static_cast<uint32_t>(key[0]);
        const uint32_t most_order = __reduce_max_sync(kFull, order);
        uint32_t who = __ballot_sync(kFull, order == most_order);
        if ((who & (who - 1)) != 0) {  // a tie: the lower index
            const uint32_t most_low = __reduce_max_sync(kFull, order == most_order ? low : 0u);
            who = __ballot_sync(kFull, order == most_order && low == most_low);
        }
        const uint32_t winner = __ffs(who) - 1;
        const uint32_t won = __shfl_sync(kFull, low, winner);
        if (lane == r) {
            out_order = most_order;
            out_low = won;
        }
        if (lane == winner) {
#pragma unroll
            for (int k = 0; k + 1 < kItems; ++k) key[k] = key[k + 1];
            key[kItems - 1] = 0;
        }
    }
    if (lane < a.top) {
        const uint64_t at = static_cast<uint64_t>(i) * a.top + lane;
        a.top_ids[at] = out_order == 0 ? -1 : static_cast<int32_t>(0xFFFFFFFFu - out_low);
        a.top_out[at] = out_order == 0 ? -CUDART_INF_F : (score_of(out_order) - m) * a.inv_t - log_s;
    }
}

// A warp per list; a longer one among them by the whole CTA.
template <class T>
__global__ void __launch_bounds__(kWarpThreads, 4) log_probs_warps_kernel(LogProbsArgs a) {
    __shared__ __align__(16) Shared<kWarpThreads> shared;
    constexpr uint32_t kLists = kWarpThreads / 32;
    const uint32_t base = blockIdx.x * kLists, i = base + (threadIdx.x >> 5);
    uint64_t first = 0;
    uint32_t n = 0;
    if (i < a.l.lists) {
        list_range(a.l, i, first, n);
        const T* z = static_cast<const T*>(a.l.scores) + first;
        if (n <= 128)
            log_probs_warp<T, 4>(a, i, z, n);
        else if (n <= 256)
            log_probs_warp<T, 8>(a, i, z, n);
        else if (n <= kWarpEntries)
            log_probs_warp<T, 16>(a, i, z, n);
    }
    if (__syncthreads_or(n > kWarpEntries) == 0) return;
    for (uint32_t k = base; k < base + kLists && k < a.l.lists; ++k) {
        list_range(a.l, k, first, n);
        if (n <= kWarpEntries) continue;
        log_probs_list<T, 1, kWarpThreads, false>(shared, a, k, 0, 1);
        __syncthreads();
    }
}

template <class T, int kVec, int kThreads>
void launch_rows(const LogProbsArgs& a, uint32_t shares, cudaStream_t s) {
    if (shares == 1) {
        log_probs_rows_kernel<T, kVec, kThreads, false><<<a.l.lists, kThreads, 0, s>>>(a, 1);
        return;
    }
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(a.l.lists * shares);
    config.blockDim = dim3(kThreads);
    config.stream = s;
    cudaLaunchAttribute cluster{};
    cluster.id = cudaLaunchAttributeClusterDimension;
    cluster.val.clusterDim.x = shares;
    cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
    config.attrs = &cluster;
    config.numAttrs = 1;
    cudaLaunchKernelEx(&config, log_probs_rows_kernel<T, kVec, kThreads, true>, a, shares);
}

template <class T>
void launch_typed(const LogProbsArgs& a, cudaStream_t s) {
    constexpr int kVec = 16 / sizeof(T);
    const uint64_t mean = a.l.bounds != nullptr ? a.l.width / a.l.lists : a.l.width;
    if (mean <= (a.l.bounds != nullptr ? kWarpMean : kWarpEntries)) {
        const uint32_t lists = kWarpThreads / 32, grid = a.l.lists / lists + (a.l.lists % lists != 0);
        log_probs_warps_kernel<T><<<grid, kWarpThreads, 0, s>>>(a);
        return;
    }
    const uint32_t shares = list_shares(mean, a.l.lists, a.sms);
    if (a.l.bounds != nullptr && mean <= 1024)  // (10,478 lists of 588: 128 threads 64 us, 256 81; 1500 of 3500: 44 and 33)
        launch_rows<T, 1, 128>(a, shares, s);
    else if (a.l.bounds != nullptr)
        launch_rows<T, 1, 256>(a, shares, s);
    else if (mean <= 128 * kBatch * kVec)  // one batch of 128 threads holds the list
        launch_rows<T, kVec, 128>(a, shares, s);
    else if (shares == 1)  // small CTAs: one's barriers hide behind the others' reading (4096 x 131072: 512 threads 287 us, 256 246)
        launch_rows<T, kVec, 256>(a, 1, s);
    else  // SMs to spare: more threads a list (64 x 50257 f32: 256 threads 14.6 us, 512 12.1)
        launch_rows<T, kVec, 512>(a, shares, s);
}

}  // namespace

void launch_log_probs(const LogProbsArgs& a, cudaStream_t s) {
    if (a.l.type == SB2_F32)
        launch_typed<float>(a, s);
    else if (a.l.type == SB2_BF16)
        launch_typed<__nv_bfloat16>(a, s);
    else
        launch_typed<__half>(a, s);
}

}  // namespace sb2
