// distill.cu — distillation from a teacher's top logits over lists of candidates, forward and backward.
//
// The student's p = softmax(z / T) over the list, the teacher's q over its top entries: softmax(t / T) over the top
// alone, or, with the teacher's log sum over its whole list, exp(t / T - log sum) with the rest r = 1 - sum q held as
// one more class beside the student's mass P outside the top. With Q = sum q + r:
//   loss   = w (sum q (log q - log p) + r (log r - log P))
//   grad_j = w / T (Q p_j - q_j)            j in the top
//            w / T p_j (Q - r / P)          elsewhere
//   hess_j = w / T^2 Q p_j (1 - p_j)        (the diagonal of the softmax's own second derivative)
// P is summed over the entries outside the top, not taken as 1 - sum p: a student that has learned its teacher keeps
// little there. Where that is less than 2^-64, the entries outside go about their own maximum in a pass of their own: f32
// holds the gradient's r p_j / P however small P is. The top's entries are marked in a bitmap, which the sum skips; their
// gradients are written once the others are, over what the common formula left there. An entry named twice has its q added
// in the teacher's order.
//
// Lists of at most 512 entries (1024 of a dense matrix) take a warp each, in registers. A longer list takes a CTA or a
// cluster of CTAs that holds it in shared memory between the passes (each thread its own vectors), so that memory sees each
// score once. Runs between boundaries are read again from the caches, entry by entry, so that a list's sums do not depend on
// where it starts. A dense list too long for shared memory, or of scores so far from 0 that fma(z, c, -m c) loses its last bits,
// is read again for each pass. The loss alone is taken in one pass that holds nothing.
//
// What bounds it, on one B200 (copy rate 6453 GB/s): 4096 lists of 32000 bf16 scores, top 64 with the rest, take 123 us,
// 4.3 TB/s, 0.66 of the copy rate; 2048 lists of 131072 (clusters of 4), top 100, 255 us, 0.65. Each score's exponential is
// taken twice, 128 cycles of the special-function unit for a warp's vector of 8, beside about 85 instructions; that unit is
// 47% busy, issue 50%, and the list's five barriers take a quarter of the warps' waiting. Holding the list in registers
// instead of shared memory left one CTA of 512 threads or spilled (wide: 387 us); reading it twice from L2 took 265 us on
// the wide lists and 153 on the others, where shared memory took 277 and 131 at the time. CTAs of half a list (36 KB)
// repeat the scalars (150 us and 269), CTAs of 512 threads lose to their barriers (208 and 321). The next list's copies,
// begun as each slot's gradient is written, gain 2%: memory's latency is not what is left.
// The loss alone over 1500 lists of 50257 f16 takes 43 us, 3.5 TB/s; 16,700 lists of 120 f32 with gradient and hessian, a
// warp each, 17 us, bound by the chain of loads and reductions of a list.
#include <algorithm>

#include "lists_device.cuh"

namespace cg = cooperative_groups;

namespace sb2 {

namespace {

// The mean length up to which runs between boundaries go by warps, the longer ones among them by whole CTAs: 20,000 lists
// of 300 take 24 us so and 71 by a CTA each; of widely spread lengths about 300, 70 and 75, about 440, 54 and 42.
constexpr uint32_t kWarpMean = 384;
constexpr int kWarpThreads = 256;    // the warp kernel's CTAs
// Bytes of scores that a CTA holds; a longer list takes more shares. Beside them lie the marks (a sixteenth of 16-bit scores)
// and the static memory, so three CTAs fit an SM up to 70,700 bytes of bf16 and two above: lists of 35,000 (131M scores in
// all) take 119 us, of 36,800 134 (162 in twice the shares). Past it, 37,000 take 172 us in two shares; one share and two
// CTAs an SM would take 141.
constexpr uint32_t kHeld = 73728;
constexpr int kMaxHeld = 216 * 1024; // and the most, with the marks, beside the static shared memory

// Share of the student's mass outside the top below which that part is taken about its own maximum. Terms below 2^-126 are
// 0: of up to 2^31 entries at most 2^-31 of that share, less than a rounding. The further pass makes 4096 x 32000 bf16 lists
// of that kind 266 us instead of 115.
constexpr float kApart = 0x1p-64f;
// ... and P's binary exponent from which it counts as none, as in 64 bits.
constexpr float kNoMass = -1074.0f;

constexpr uint32_t kBits = 65536;    // marks of a share: entries past so many share them

// What the derivatives of a list's entries share: with e = exp((z - m) / T) and p = inv_s e, the gradient is slope e
// outside the top and top_slope e less q in it, the hessian curve p (1 - p).
struct Slopes {
    float inv_s, slope, top_slope, curve;
};

// What a CTA keeps of its share of a list beside the scores.
template <int kThreads>
struct Shared {
    float warp[7][kThreads / 32];
    float m, outside, top;           // the share's reference and sums (with the rest: outside the top, and in it)
    __align__(16) int32_t id[kMaxTop];
    float q[kMaxTop];
    uint32_t again;                  // some entry's mark was set before
    int32_t far;                     // far scores in the share
    Slopes slopes;                   // what one warp makes of the sums, for the others
    float joined_m, q_scale;
    int32_t empty;
    int32_t apart;                   // the entries outside the top go about their own maximum
    float sum, held, cross, r;       // what that takes
    float rest_m, rest_sum;          // the share's maximum and sum outside the top
    uint32_t edge_bits;              // marks of the scalars outside the vectors
};

// The sum and the maximum of the warps' parts, in every thread.
template <int kThreads>
__device__ __forceinline__ float sum_of(const float (&part)[kThreads / 32]) {
    float v = part[threadIdx.x & (kThreads / 32 - 1)];
#pragma unroll
    for (int o = kThreads / 64; o > 0; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
    return v;
}

template <int kThreads>
__device__ __forceinline__ float max_of(const float (&part)[kThreads / 32]) {
    float v = part[threadIdx.x & (kThreads / 32 - 1)];
#pragma unroll
    for (int o = kThreads / 64; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(kFull, v, o));
    return v;
}

// The hessian diagonal of an entry: a p that its roundings carry past 1 makes it 0, never negative.
__device__ __forceinline__ float hessian_of(float curve, float p) { return curve * p * fmaxf(1.0f - p, 0.0f); }

// Writes an entry's derivatives; the objective's row weight and maxima come in here.
struct Maxima {
    float g = 0.0f, h = 0.0f;
};
template <class T>
__device__ __forceinline__ void put(const DistillArgs& a, uint64_t to, uint64_t row, float g, float h, bool counts, Maxima& most) {
    if (a.row_weight != nullptr) {
        g *= a.row_weight[row];
        h *= a.row_weight[row];
    }
    if (counts) {
        most.g = fmaxf(most.g, fabsf(g));
        most.h = fmaxf(most.h, fabsf(h));
    }
    if (a.grad != nullptr) static_cast<T*>(a.grad)[to] = from_float<T>(g);
    if (a.hess != nullptr) static_cast<T*>(a.hess)[to] = from_float<T>(h);
}

// A CTA's maxima over its lists, for a training iteration.
template <int kThreads>
__device__ __forceinline__ void publish(const DistillArgs& a, Maxima most) {
    if (a.max_g == nullptr) return;
    __shared__ float s_g[kThreads / 32], s_h[kThreads / 32];
    most.g = warp_max(most.g);
    most.h = warp_max(most.h);
    if ((threadIdx.x & 31) == 0) {
        s_g[threadIdx.x >> 5] = most.g;
        s_h[threadIdx.x >> 5] = most.h;
    }
    __syncthreads();
    if (threadIdx.x == 0) {  // non-negative doubles order like their bit patterns
        for (int k = 1; k < kThreads / 32; ++k) {
            most.g = fmaxf(most.g, s_g[k]);
            most.h = fmaxf(most.h, s_h[k]);
        }
        atomicMax(a.max_g, static_cast<unsigned long long>(__double_as_longlong(static_cast<double>(most.g))));
        atomicMax(a.max_h, static_cast<unsigned long long>(__double_as_longlong(static_cast<double>(most.h))));
    }
}

// Eight (four) derivatives as one 16-byte vector.
template <class T, int kVec>
__device__ __forceinline__ uint4 packed(const float (&v)[kVec]) {
    if constexpr (sizeof(T) == 4) {
        return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
    } else {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (std::is_same_v<T, __nv_bfloat16>) {
                const __nv_bfloat162 x = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
                w[i] = *reinterpret_cast<const uint32_t*>(&x);
            } else {
                const __half2 x = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
                w[i] = *reinterpret_cast<const uint32_t*>(&x);
            }
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// ln q of a teacher's entry, up to the top's own sum without a log sum: then from the largest logit, so that a constant
// on all of a list's logits, however large, changes nothing.
__device__ __forceinline__ float log_q_of(float logit, float inv_t, bool rest, float log_sum, float most) {
    return rest ? __fmaf_rn(logit, inv_t, -log_sum) : (logit - most) * inv_t;
}

// One entry of the teacher's top: its index (-1: padding) and logit.
__device__ __forceinline__ void teacher_entry(const DistillArgs& a, uint32_t i, uint32_t k, uint32_t n, int32_t& id, float& y) {
    const uint64_t at = static_cast<uint64_t>(i) * a.t.stride + k;
    id = a.t.ids[at];
    if (id < 0 || static_cast<uint32_t>(id) >= n) id = -1;
    y = id >= 0 ? load_typed(a.t.logits, a.t.type, at) : -CUDART_INF_F;
}

// The loss's cross terms are summed at 2^-32 of themselves (exactly): a teacher's entry that the student masks by the type's
// lowest value makes one of about 2^128 / T, which the loss may still hold once it is multiplied by q.
constexpr float kDown = 0x1p-32f, kUp = 0x1p32f;

// One of them, q (log q - (z - m) / T).
__device__ __forceinline__ float cross_term(float q, float log_q, float z, float m, float inv_t) {
    return q != 0.0f ? q * (log_q * kDown - (z * kDown - m * kDown) * inv_t) : 0.0f;
}

// The loss of a list from its weight and its parts: the cross terms, sum q, S, log (S P), and the rest.
__device__ __forceinline__ float loss_of(float weight, float cross, float held, float sum, float log_outside, float r) {
    const float log_s = logf(sum);
    float loss = held * log_s;
    if (r > 0.0f) loss += r * (logf(r) - (log_outside - log_s));
    const float up = cross * kUp;
    return fabsf(up) <= FLT_MAX ? weight * (up + loss) : weight * cross * kUp + weight * loss;
}

// Whether a maximum outside the top leaves P a mass: less than 64 bits hold counts as none, as a masked entry's.
__device__ __forceinline__ bool has_mass(float rest_m, float m, float sum, float c) {
    return (rest_m - m) * c - log2f(sum) >= kNoMass;
}

__device__ __forceinline__ Slopes slopes_of(float w, float inv_t, float held, float r, float sum, float outside) {
    Slopes k;
    const float mass = held + r;
    k.inv_s = 1.0f / sum;
    k.top_slope = mass * k.inv_s * (w * inv_t);
    k.slope = r > 0.0f ? (mass * k.inv_s - r / outside) * (w * inv_t) : k.top_slope;
    k.curve = mass * (w * inv_t * inv_t);
    return k;
}

// Whether what lies outside the top needs its own maximum, for a rest of `r` (k: the slopes without it).
__device__ __forceinline__ bool rest_is_apart(float r, float sum, float outside, const Slopes& k) {
    return r > 0.0f && (outside < kApart * sum || fabsf(k.slope) == CUDART_INF_F);
}

// Marks the teacher's entry `id` where it lies in this share (true). s.again: a mark that was set before.
template <class T, int kVec, int kThreads>
__device__ __forceinline__ bool mark_entry(Shared<kThreads>& s, uint32_t* bits, bool room, const Walk<T, kVec>& w, uint32_t from,
                                           uint32_t to, uint32_t share, int32_t id) {
    if (id < 0) return false;
    const uint32_t j = static_cast<uint32_t>(id);
    uint32_t before, mark;
    if (j < w.head || j >= w.tail()) {
        if (share != 0) return false;
        mark = 1u << (j < w.head ? j : w.head + (j - w.tail()));
        before = atomicOr(&s.edge_bits, mark);
    } else {
        if ((j - w.head) / kVec < from || (j - w.head) / kVec >= to) return false;
        const uint32_t bit = (j - w.head - from * kVec) & (kBits - 1);
        mark = 1u << (bit & 31);
        before = room ? atomicOr(&bits[bit / 32], mark) : mark;
    }
    if ((before & mark) != 0) s.again = 1;  // an index named twice, or one that shares its mark
    return true;
}

// Whether entry `t` of the teacher is the first that names its index, and the only one (s.id is -1 up to the next
// multiple of 4).
template <int kThreads>
__device__ __forceinline__ void lead(const Shared<kThreads>& s, int32_t id, uint32_t t, uint32_t top, bool& leads, bool& alone) {
    uint32_t same = 0, before = 0;
    for (uint32_t k = 0; k < top; k += 4) {
        const int4 o = *reinterpret_cast<const int4*>(&s.id[k]);
        const uint32_t hit = (o.x == id ? 1u : 0u) | (o.y == id ? 2u : 0u) | (o.z == id ? 4u : 0u) | (o.w == id ? 8u : 0u);
        if (hit != 0) {
            same += __popc(hit);
            before += __popc(k > t ? 0u : hit & ((1u << (t - k < 4 ? t - k : 4)) - 1u));
        }
    }
    alone = same == 1;
    leads = leads && before == 0;
}

// Marks of vector `v`'s entries, the share's first vector `from`. Where the marks are shared or there are none, the ids
// themselves decide.
template <class T, int kVec, int kThreads>
__device__ __forceinline__ uint32_t marks_of(const Shared<kThreads>& s, const uint32_t* bits, bool room, const Walk<T, kVec>& w,
                                             uint32_t from, uint32_t to, uint32_t top, uint32_t v) {
    uint32_t m = ~0u;
    if (room) {
        if constexpr (kVec == 8) {  // a byte a vector
            m = reinterpret_cast<const uint8_t*>(bits)[(v - from) & (kBits / 8 - 1)];
        } else {
            const uint32_t bit = ((v - from) * kVec) & (kBits - 1);
            m = (bits[bit / 32] >> (bit & 31)) & ((1u << kVec) - 1u);
        }
    }
    if (m != 0 && (!room || (to - from) * kVec > kBits)) {
        m = 0;
        for (uint32_t k = 0; k < top; ++k) {
            const uint32_t e = static_cast<uint32_t>(s.id[k]) - w.at(v);
            if (e < kVec) m |= 1u << e;
        }
    }
    return m;
}

// Derivatives 0 for the entries before the first list and behind the last, by the first kClearing CTAs: they are through
// before the others, so that few calls wait for the loads of the two boundaries.
constexpr uint32_t kClearing = 64;
template <class T>
__device__ __forceinline__ void clear_ends(const DistillArgs& a) {
    if (!a.clear || blockIdx.x >= kClearing) return;
    const uint64_t begin = a.l.bounds[0], end = a.l.bounds[a.l.lists];
    const uint64_t low = begin < a.l.width ? begin : a.l.width, high = end < low ? low : end < a.l.width ? end : a.l.width;
    const uint64_t count = low + (a.l.width - high), step = min(gridDim.x, kClearing) * static_cast<uint64_t>(blockDim.x);
    for (uint64_t j = static_cast<uint64_t>(blockIdx.x) * blockDim.x + threadIdx.x; j < count; j += step) {
        const uint64_t at = j < low ? j : high + (j - low);
        if (a.grad != nullptr) static_cast<T*>(a.grad)[at] = from_float<T>(0.0f);
        if (a.hess != nullptr) static_cast<T*>(a.hess)[at] = from_float<T>(0.0f);
    }
}

// What is on its way for a CTA's next list while this one's gradients are written.
struct Ahead {
    bool flying = false;  // the scores, into the threads' slots, and the thread's entry of the teacher
    int32_t id;
    float y;
};

// The vectors of a list that one of `shares` CTAs (a power of two) takes.
template <class T, int kVec, bool kCluster>
__device__ __forceinline__ void share_of(const Walk<T, kVec>& w, uint32_t share, uint32_t shares, uint32_t& from, uint32_t& to) {
    from = 0;
    to = w.vectors;
    if constexpr (kCluster) {
        const uint32_t shift = __ffs(shares) - 1;
        from = static_cast<uint32_t>((static_cast<uint64_t>(w.vectors) * share) >> shift);
        to = static_cast<uint32_t>((static_cast<uint64_t>(w.vectors) * (share + 1)) >> shift);
    }
}

// What is left of a list once its sums are known and little mass lies outside the top (Shared::apart): the loss and all
// derivatives, the entries outside the top about their own maximum. `data`: the thread's held vectors, or null.
template <class T, int kVec, int kThreads, bool kCluster>
__device__ __noinline__ Maxima rest_apart(Shared<kThreads>& s, const Pack<T, kVec>* data, const uint32_t* bits,
                                          const DistillArgs& a, uint32_t i, uint32_t share, uint32_t shares, Maxima most) {
    const uint32_t t = threadIdx.x, lane = t & 31, warp = t >> 5;
    uint64_t first;
    uint32_t n;
    list_range(a.l, i, first, n);
    const Walk<T, kVec> w(static_cast<const T*>(a.l.scores) + first, n);
    uint32_t from, to;
    share_of<T, kVec, kCluster>(w, share, shares, from, to);
    const float c = __fmul_rn(kLog2E, a.inv_t), weight = a.weight != nullptr ? a.weight[i] : 1.0f, m = s.joined_m, sum = s.sum;
    const uint32_t edge_at = share == 0 && t < 2 * kVec ? w.edge(t) : n;
    auto get = [&](uint32_t v, float(&x)[kVec]) {
        Pack<T, kVec> p;
        if (data != nullptr)
            p = data[v - from];
        else
            p.load(w.z + w.at(v));
        p.values(x);
    };
    auto at_edge = [&](auto f) {
        if (edge_at < n && ((s.edge_bits >> t) & 1u) == 0) f(to_float(w.z[edge_at]), edge_at);
    };
    auto each = [&](auto f) {
        for (uint32_t v = from + t; v < to; v += kThreads) {
            const uint32_t skip = marks_of(s, bits, bits != nullptr, w, from, to, a.t.top, v);
            float x[kVec];
            get(v, x);
#pragma unroll
            for (int e = 0; e < kVec; ++e)
                if (((skip >> e) & 1u) == 0) f(x[e], w.at(v) + e);
        }
        at_edge(f);
    };
    float rest_m = -CUDART_INF_F, rest_sum = 0.0f;
    each([&](float z, uint32_t) { rest_m = fmaxf(rest_m, z); });
    rest_m = warp_max(rest_m);
    if (lane == 0) s.warp[0][warp] = rest_m;
    __syncthreads();
    rest_m = max_of<kThreads>(s.warp[0]);
    if constexpr (kCluster) {
        cg::cluster_group cluster = cg::this_cluster();
        if (t == 0) s.rest_m = rest_m;
        cluster.sync();
        rest_m = warp_max(cluster.map_shared_rank(&s, lane & (shares - 1))->rest_m);
    }
    const bool some = has_mass(rest_m, m, sum, c);
    if (some) each([&](float z, uint32_t) { rest_sum += pow2(exponent(z, rest_m, c)); });
    rest_sum = warp_sum(rest_sum);
    if (lane == 0) s.warp[1][warp] = rest_sum;
    __syncthreads();
    rest_sum = sum_of<kThreads>(s.warp[1]);
    if constexpr (kCluster) {
        cg::cluster_group cluster = cg::this_cluster();
        if (t == 0) s.rest_sum = rest_sum;
        cluster.sync();
        const float other = cluster.map_shared_rank(&s, lane & (shares - 1))->rest_sum;
        rest_sum = warp_sum(lane < shares ? other : 0.0f);
    }
    const float r = some ? s.r : 0.0f;
    if (t == 0 && share == 0 && a.loss != nullptr)
        a.loss[i] = loss_of(weight, s.cross, s.held, sum, (rest_m - m) * a.inv_t + logf(rest_sum), r);
    if (a.grad == nullptr && a.hess == nullptr) return most;
    const uint64_t out = a.l.bounds != nullptr ? first : static_cast<uint64_t>(i) * a.grad_stride;
    const float mass = s.held + r, scale = weight * a.inv_t, inv_s = 1.0f / sum, pull = some ? r / rest_sum : 0.0f;
    auto put_one = [&](float z, uint32_t j, float less) {
        const float p = pow2(exponent(z, m, c)) * inv_s;
        put<T>(a, out + j, first + j, (mass * p - less) * scale, hessian_of(mass * scale * a.inv_t, p), true, most);
    };
    auto less_of = [&](float z) { return some ? pull * pow2(exponent(z, rest_m, c)) : 0.0f; };
    auto put_rest = [&](float z, uint32_t j) { put_one(z, j, less_of(z)); };
    bool whole = kVec > 1;  // whole vectors, over which the top's own go
    if constexpr (kVec > 1) {
        T* const grad = a.grad != nullptr ? static_cast<T*>(a.grad) + out + w.at(from) : nullptr;
        T* const hess = a.hess != nullptr ? static_cast<T*>(a.hess) + out + w.at(from) : nullptr;
        whole = ((reinterpret_cast<uintptr_t>(grad) | reinterpret_cast<uintptr_t>(hess)) & 15) == 0;
        if (whole) {
            for (uint32_t v = t; v < to - from; v += kThreads) {
                float x[kVec], h[kVec];
                get(from + v, x);
#pragma unroll
                for (int e = 0; e < kVec; ++e) {
                    const float p = pow2(exponent(x[e], m, c)) * inv_s;
                    h[e] = hessian_of(mass * scale * a.inv_t, p);
                    x[e] = (mass * p - less_of(x[e])) * scale;
                }
                if (grad != nullptr) __stcs(reinterpret_cast<uint4*>(grad) + v, packed<T, kVec>(x));
                if (hess != nullptr) __stcs(reinterpret_cast<uint4*>(hess) + v, packed<T, kVec>(h));
            }
            at_edge(put_rest);
        }
    }
    if (!whole) each(put_rest);
    __syncthreads();
    if (t < a.t.top && s.id[t] >= 0) {  // the top's own in this share, the first that names an index with all their q
        const uint32_t id = static_cast<uint32_t>(s.id[t]);
        bool leads = id < w.head || id >= w.tail() ? share == 0 : (id - w.head) / kVec >= from && (id - w.head) / kVec < to;
        for (uint32_t k = 0; k < t && leads; ++k) leads = s.id[k] != s.id[t];
        if (leads) {
            float q = 0.0f;
            for (uint32_t k = t; k < a.t.top; ++k)
                if (s.id[k] == s.id[t]) q += s.q[k];
            put_one(to_float(w.z[id]), id, q);
        }
    }
    return most;
}

// One list by `shares` CTAs, this one the `share`-th: a cluster, or a CTA alone (shares 1). `data` holds `slots` vectors:
// where the share is no longer, it stays there, each vector in a slot of the thread that reads it. A slot is free once
// its gradient is written, so list `next` (no list from a.l.lists on) follows through the same slots at once. `bits` may be
// null: the teacher's ids are then looked through for each vector.
template <class T, int kVec, int kThreads, bool kCluster>
__device__ __forceinline__ void distill_list(Shared<kThreads>& s, Pack<T, kVec>* data, uint32_t slots, uint32_t* bits,
                                             const DistillArgs& a, uint32_t i, uint32_t next, Ahead& ahead, uint32_t share,
                                             uint32_t shares, Maxima& most) {
    constexpr int kUnroll = kVec == 1 ? 4 : 2;
    const uint32_t t = threadIdx.x, lane = t & 31, warp = t >> 5;
    uint64_t first;
    uint32_t n;
    list_range(a.l, i, first, n);
    const Walk<T, kVec> w(static_cast<const T*>(a.l.scores) + first, n);
    uint32_t from, to;
    share_of<T, kVec, kCluster>(w, share, shares, from, to);
    const float c = __fmul_rn(kLog2E, a.inv_t);
    const bool rest = a.t.log_sum != nullptr;
    const bool held_here = kVec == 1 || to - from <= slots, room = bits != nullptr;
    const float log_sum = rest ? a.t.log_sum[i] : 0.0f, weight = a.weight != nullptr ? a.weight[i] : 1.0f;
    // The scores, on their way to the thread's own slots.
    if constexpr (kVec > 1)
        if (held_here && !ahead.flying) {
            const T* z = w.z + w.at(from);
#pragma unroll 4
            for (uint32_t v = t; v < to - from; v += kThreads) data[v].copy(z + static_cast<size_t>(v) * kVec);
            copies_begun();
        }
    const uint32_t edge_at = share == 0 && t < 2 * kVec ? w.edge(t) : n;
    const float edge = edge_at < n ? to_float(w.z[edge_at]) : -CUDART_INF_F;
    // The teacher, and the marks of its entries in this share.
    int32_t id = -1;
    float y = -CUDART_INF_F, zt = -CUDART_INF_F;
    if (t < a.t.top) {
        if (ahead.flying) {
            id = ahead.id;
            y = ahead.y;
        } else {
            teacher_entry(a, i, t, n, id, y);
        }
        if (id >= 0) zt = to_float(w.z[id]);
    }
    ahead.flying = false;
    if (t < kMaxTop) s.id[t] = id;
    const uint32_t words = room ? (min(kBits, (to - from) * kVec) + 31) / 32 : 0;
    for (uint32_t k = t; k < words; k += kThreads) bits[k] = 0;
    if (t == 0) s.edge_bits = s.again = 0;
    __syncthreads();
    const bool mine = mark_entry(s, bits, room, w, from, to, share, id);
    // Vector `v` of the share; a run between boundaries, entry by entry, is read from its place each time.
    auto get = [&](uint32_t v, float(&x)[kVec]) {
        if constexpr (kVec == 1)
            x[0] = to_float(__ldg(w.z + from + v));
        else
            data[v].values(x);
    };
    auto marked = [&](uint32_t v) { return marks_of(s, bits, room, w, from, to, a.t.top, v); };
    // The maxima of the scores and of the teacher's.
    float m = fmaxf(edge, zt);  // with the top's scores, so that no share's reference lies far below them
    if constexpr (kVec == 1) {
#pragma unroll 4
        for (uint32_t v = t; v < to - from; v += kThreads) m = fmaxf(m, to_float(__ldg(w.z + from + v)));
    } else if (held_here) {
        Pack<T, kVec> top;
        top.masked();
        copies_done();
        for (uint32_t v = t; v < to - from; v += kThreads) top.raise(data[v]);
        float x[kVec];
        top.values(x);
#pragma unroll
        for (int e = 0; e < kVec; ++e) m = fmaxf(m, x[e]);
    } else {
        for (uint32_t v = from + t; v < to; v += kThreads) {
            Pack<T, kVec> now;
            float x[kVec];
            now.load(w.z + w.at(v));
            now.values(x);
            for (int e = 0; e < kVec; ++e) m = fmaxf(m, x[e]);
        }
    }
    m = warp_max(m);
    float y_max = warp_max(y);
    if (lane == 0) {
        s.warp[0][warp] = m;
        s.warp[1][warp] = y_max;
    }
    const bool taught = __syncthreads_or(id >= 0) != 0;
    m = fmaxf(max_of<kThreads>(s.warp[0]), -FLT_MAX);
    y_max = fmaxf(max_of<kThreads>(s.warp[1]), -FLT_MAX);
    float R = __fmul_rn(m, c);
    bool far = !(fabsf(R) < kFar) || !held_here;
    // The share's sum (with the rest, outside the top), the top's own and the teacher's.
    float sum = 0.0f;
    if (!far) {
        const float2 cc = make_float2(c, c), minus_r = make_float2(-R, -R);
        float2 two = make_float2(0.0f, 0.0f);
        auto add = [&](uint32_t v, bool look) {
            float x[kVec];
            get(v, x);
            const uint32_t skip = look ? marked(from + v) : 0;
            if (skip != 0) {
#pragma unroll
                for (int e = 0; e < kVec; ++e)
                    if ((skip >> e) & 1u) x[e] = -CUDART_INF_F;
            }
            if constexpr (kVec == 1) {
                sum += pow2(__fmaf_rn(x[0], c, -R));
            } else {
#pragma unroll
                for (int e = 0; e < kVec; e += 2) {
                    const float2 z = __ffma2_rn(make_float2(x[e], x[e + 1]), cc, minus_r);
                    two = __fadd2_rn(two, make_float2(pow2(z.x), pow2(z.y)));
                }
            }
        };
        if (rest) {
#pragma unroll kUnroll
            for (uint32_t v = t; v < to - from; v += kThreads) add(v, true);
        } else {
#pragma unroll kUnroll
            for (uint32_t v = t; v < to - from; v += kThreads) add(v, false);
        }
        sum += two.x + two.y;
    } else {
        for (uint32_t v = from + t; v < to; v += kThreads) {
            Pack<T, kVec> now;
            float x[kVec];
            now.load(w.z + w.at(v));
            now.values(x);
            const uint32_t skip = rest ? marked(v) : 0;
            for (int e = 0; e < kVec; ++e)
                if (((skip >> e) & 1u) == 0) sum += pow2(exponent(x[e], m, c));
        }
    }
    auto term = [&](float z) { return far ? pow2(exponent(z, m, c)) : pow2(__fmaf_rn(z, c, -R)); };
    const bool edge_marked = edge_at < n && ((s.edge_bits >> t) & 1u) != 0;
    if (edge_at < n && !(rest && edge_marked)) sum += term(edge);
    bool leads = mine, alone = true;  // the first of the teacher's entries that names this index, and the only one
    if (s.again != 0 && t < a.t.top) lead(s, id, t, a.t.top, leads, alone);
    // The teacher's terms, not yet divided by their sum where the top is all of it.
    const float log_q = log_q_of(y, a.inv_t, rest, log_sum, y_max);
    float q = id >= 0 ? expf(log_q) : 0.0f;
    sum = warp_sum(sum);
    if (lane == 0) s.warp[2][warp] = sum;
    if (warp * 32 < a.t.top) {
        s.q[t] = q;
        const float top_part = warp_sum(rest && leads ? term(zt) : 0.0f);
        const float held_part = warp_sum(q);
        const float cross_part = warp_sum(cross_term(q, log_q, zt, m, a.inv_t));
        if (lane == 0) {
            s.warp[3][warp] = top_part;
            s.warp[4][warp] = held_part;
            s.warp[5][warp] = cross_part;
        }
    } else if (lane == 0) {
        s.warp[3][warp] = s.warp[4][warp] = s.warp[5][warp] = 0.0f;
    }
    __syncthreads();
    // The rest of the scalars are one warp's work.
    float outside = 0.0f, top_sum = 0.0f, held = 0.0f, cross = 0.0f;
    if (warp == 0) {
        // About m itself: the rounding of R is put back.
        const float settle = far ? 1.0f : pow2(-__fmaf_rn(m, c, -R));
        outside = settle * sum_of<kThreads>(s.warp[2]);
        top_sum = settle * sum_of<kThreads>(s.warp[3]);
        held = sum_of<kThreads>(s.warp[4]);
        cross = sum_of<kThreads>(s.warp[5]);
    }
    if constexpr (kCluster) {
        // Every share's sum is about its own reference: their sum is about the largest.
        cg::cluster_group cluster = cg::this_cluster();
        if (t == 0) {
            s.m = m;
            s.outside = outside;
            s.top = top_sum;
        }
        cluster.sync();
        if (warp == 0) {
            const auto* other = cluster.map_shared_rank(&s, lane & (shares - 1));
            const float other_m = other->m, other_outside = other->outside, other_top = other->top;
            const float all = warp_max(other_m), f = pow2(exponent(other_m, all, c));
            outside = warp_sum(lane < shares ? other_outside * f : 0.0f);
            top_sum = warp_sum(lane < shares ? other_top * f : 0.0f);
            cross += held * ((all * kDown - m * kDown) * a.inv_t);
            m = all;
        }
    }
    if (warp == 0) {
        sum = outside + top_sum;
        float q_scale = 1.0f;
        if (!rest && held != 0.0f) {
            q_scale = 1.0f / held;
            cross = cross * q_scale - logf(held) * kDown;
            held = 1.0f;
        }
        const float r = rest ? fmaxf(1.0f - held, 0.0f) : 0.0f;
        const bool none = sum == 0.0f || !taught;
        // What the derivatives outside the top share, and what the same formula gives in it.
        Slopes k = slopes_of(weight, a.inv_t, held, r, sum, outside);
        const bool apart = !none && rest_is_apart(r, sum, outside, k);
        if (apart) k = slopes_of(weight, a.inv_t, held, 0.0f, sum, outside);
        R = __fmul_rn(m, c);
        if (fabsf(R) < kFar && held_here) {  // the terms are about R
            const float f = pow2(-__fmaf_rn(m, c, -R));
            k.inv_s *= f;
            k.slope *= f;
            k.top_slope *= f;
        }
        if (lane == 0) {
            s.slopes = k;
            s.joined_m = m;
            s.q_scale = q_scale;
            s.empty = none;
            s.apart = apart;
            if (apart) {
                s.sum = sum;
                s.held = held;
                s.cross = cross;
                s.r = r;
            } else if (share == 0 && a.loss != nullptr) {
                a.loss[i] = none ? 0.0f : loss_of(weight, cross, held, sum, logf(outside), r);
            }
        }
    }
    __syncthreads();
    if (s.apart != 0) {  // (every share of a cluster joins the same sums)
        most = rest_apart<T, kVec, kThreads, kCluster>(s, kVec > 1 && held_here ? data : nullptr, bits, a, i, share, shares, most);
        if constexpr (kCluster) cg::this_cluster().sync();  // the shares' memory is read
        return;
    }
    if constexpr (kCluster) cg::this_cluster().barrier_arrive();  // the shares' memory is read
    if (a.grad == nullptr && a.hess == nullptr) {
        if constexpr (kCluster) cg::this_cluster().barrier_wait();
        return;
    }
    m = s.joined_m;
    R = __fmul_rn(m, c);
    far = !(fabsf(R) < kFar) || !held_here;
    const Slopes k = s.slopes;
    const float q_scale = s.q_scale;
    const bool empty = s.empty != 0;
    q *= q_scale;
    const uint64_t out = a.l.bounds != nullptr ? first : static_cast<uint64_t>(i) * a.grad_stride;
    auto put_one = [&](float z, uint32_t j, bool counts) {
        const float e = empty ? 0.0f : term(z), q_j = e * k.inv_s;
        put<T>(a, out + j, first + j, empty ? 0.0f : k.slope * e, empty ? 0.0f : hessian_of(k.curve, q_j), counts, most);
    };
    // The next list's scores follow into each slot as its gradient is written.
    const T* next_z = nullptr;
    uint32_t next_count = 0, done = 0;
    if (kVec > 1 && next < a.l.lists) {
        uint64_t next_first;
        uint32_t next_n, next_from, next_to;
        list_range(a.l, next, next_first, next_n);
        const Walk<T, kVec> next_w(static_cast<const T*>(a.l.scores) + next_first, next_n);
        share_of<T, kVec, kCluster>(next_w, share, shares, next_from, next_to);
        if (next_to - next_from <= slots) {
            next_z = next_w.z + next_w.at(next_from);
            next_count = next_to - next_from;
            ahead.flying = true;
            if (t < a.t.top) teacher_entry(a, next, t, next_n, ahead.id, ahead.y);
        }
    }
    if (!far && !empty) {
        T* const grad = a.grad != nullptr ? static_cast<T*>(a.grad) + out + w.at(from) : nullptr;
        T* const hess = a.hess != nullptr ? static_cast<T*>(a.hess) + out + w.at(from) : nullptr;
        const bool aligned = ((reinterpret_cast<uintptr_t>(grad) | reinterpret_cast<uintptr_t>(hess)) & 15) == 0;
        const float2 cc = make_float2(c, c), minus_r = make_float2(-R, -R), slope = make_float2(k.slope, k.slope);
        if (kVec == 1 && (a.max_g != nullptr || a.row_weight != nullptr)) {
#pragma unroll 4
            for (uint32_t v = t; v < to - from; v += kThreads) {
                float x[kVec];
                get(v, x);
                put_one(x[0], w.at(from + v), a.max_g == nullptr || marked(from + v) == 0);
            }
        } else if (kVec == 1) {
#pragma unroll 4
            for (uint32_t v = t; v < to - from; v += kThreads) {
                float x[kVec];
                get(v, x);
                const float e = pow2(__fmaf_rn(x[0], c, -R)), p_j = e * k.inv_s;
                if (grad != nullptr) grad[v] = from_float<T>(k.slope * e);
                if (hess != nullptr) hess[v] = from_float<T>(hessian_of(k.curve, p_j));
            }
        } else if (kVec > 1 && aligned && grad != nullptr && hess == nullptr) {
#pragma unroll kUnroll
            for (uint32_t v = t; v < to - from; v += kThreads) {
                float x[kVec];
                get(v, x);
#pragma unroll
                for (int e = 0; e + 1 < kVec; e += 2) {
                    const float2 z = __ffma2_rn(make_float2(x[e], x[e + 1]), cc, minus_r);
                    const float2 g = __fmul2_rn(make_float2(pow2(z.x), pow2(z.y)), slope);
                    x[e] = g.x;
                    x[e + 1] = g.y;
                }
                if constexpr (kVec > 1) {
                    __stcs(reinterpret_cast<uint4*>(grad) + v, packed<T, kVec>(x));
                    if (v < next_count) data[v].copy(next_z + static_cast<size_t>(v) * kVec);
                }
            }
            done = to - from;
        } else {
            for (uint32_t v = t; v < to - from; v += kThreads) {
                float x[kVec], g[kVec], h[kVec];
                get(v, x);
#pragma unroll
                for (int e = 0; e < kVec; ++e) {
                    const float z = pow2(__fmaf_rn(x[e], c, -R)), p_j = z * k.inv_s;
                    g[e] = k.slope * z;
                    h[e] = hessian_of(k.curve, p_j);
                }
                if (kVec > 1 && aligned) {
                    if constexpr (kVec > 1) {
                        if (grad != nullptr) __stcs(reinterpret_cast<uint4*>(grad) + v, packed<T, kVec>(g));
                        if (hess != nullptr) __stcs(reinterpret_cast<uint4*>(hess) + v, packed<T, kVec>(h));
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < kVec; ++e) {
                        if (grad != nullptr) grad[v * kVec + e] = from_float<T>(g[e]);
                        if (hess != nullptr) hess[v * kVec + e] = from_float<T>(h[e]);
                    }
                }
            }
        }
    } else {
        for (uint32_t v = from + t; v < to; v += kThreads) {
            const uint32_t skip = a.max_g != nullptr ? marked(v) : 0;
            for (int e = 0; e < kVec; ++e) put_one(to_float(w.z[w.at(v) + e]), w.at(v) + e, ((skip >> e) & 1u) == 0);
        }
    }
    if (edge_at < n) put_one(edge, edge_at, !edge_marked);
    if constexpr (kVec > 1) {
        for (uint32_t v = t; v < next_count; v += kThreads)
            if (v >= done) data[v].copy(next_z + static_cast<size_t>(v) * kVec);
        copies_begun();
    }
    __syncthreads();
    // The top's own, over them.
    if (leads && !empty) {
        float taught_q = q;
        if (!alone) {
            taught_q = 0.0f;
            for (uint32_t x = 0; x < a.t.top; ++x)
                if (s.id[x] == id) taught_q += s.q[x] * q_scale;
        }
        const float e = term(zt), p_j = e * k.inv_s;
        put<T>(a, out + id, first + id, k.top_slope * e - taught_q * (weight * a.inv_t), hessian_of(k.curve, p_j), true, most);
    }
    if constexpr (kCluster) cg::this_cluster().barrier_wait();
}

// The loss alone of one dense list: its sums are taken while it is read, about the maximum of the first batch (moved
// where later entries lie far above it). False: far scores, or little mass outside the top: distill_list() takes it.
template <class T, int kVec, int kThreads, bool kCluster>
__device__ __forceinline__ bool loss_list(Shared<kThreads>& s, uint32_t* bits, const DistillArgs& a, uint32_t i, uint32_t share,
                                          uint32_t shares) {
    constexpr int kBatch = 4;  // vectors a thread has in flight
    const uint32_t t = threadIdx.x, lane = t & 31, warp = t >> 5;
    uint64_t first;
    uint32_t n;
    list_range(a.l, i, first, n);
    const Walk<T, kVec> w(static_cast<const T*>(a.l.scores) + first, n);
    uint32_t from, to;
    share_of<T, kVec, kCluster>(w, share, shares, from, to);
    const float c = __fmul_rn(kLog2E, a.inv_t);
    const bool rest = a.t.log_sum != nullptr;
    const float log_sum = rest ? a.t.log_sum[i] : 0.0f, weight = a.weight != nullptr ? a.weight[i] : 1.0f;
    Pack<T, kVec> p[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
        const uint32_t v = from + u * kThreads + t;
        if (v < to)
            p[u].load(w.z + w.at(v));
        else
            p[u].masked();
    }
    const uint32_t edge_at = share == 0 && t < 2 * kVec ? w.edge(t) : n;
    float edge[1] = {edge_at < n ? to_float(w.z[edge_at]) : -CUDART_INF_F};
    int32_t id = -1;
    float y = -CUDART_INF_F, zt = -CUDART_INF_F;
    if (t < a.t.top) {
        teacher_entry(a, i, t, n, id, y);
        if (id >= 0) zt = to_float(w.z[id]);
    }
    bool mine = false;
    if (rest) {  // the top's entries, which the sum leaves out
        if (t < kMaxTop) s.id[t] = id;
        const uint32_t words = (min(kBits, (to - from) * kVec) + 31) / 32;
        for (uint32_t k = t; k < words; k += kThreads) bits[k] = 0;
        if (t == 0) s.edge_bits = s.again = 0;
        __syncthreads();
        mine = mark_entry(s, bits, true, w, from, to, share, id);
    }
    Pack<T, kVec> top = p[0];
#pragma unroll
    for (int u = 1; u < kBatch; ++u) top.raise(p[u]);
    float m = fmaxf(edge[0], zt), x[kVec];
    top.values(x);
#pragma unroll
    for (int e = 0; e < kVec; ++e) m = fmaxf(m, x[e]);
    m = warp_max(m);
    float y_max = warp_max(y);
    if (lane == 0) {
        s.warp[0][warp] = m;
        s.warp[1][warp] = y_max;
    }
    const bool taught = __syncthreads_or(id >= 0) != 0;
    m = max_of<kThreads>(s.warp[0]);
    y_max = fmaxf(max_of<kThreads>(s.warp[1]), -FLT_MAX);
    Reader<false> r(m, c);
    auto read = [&](bool look) {
        for (uint32_t base = from; base < to; base += kBatch * kThreads) {
#pragma unroll
            for (int u = 0; u < kBatch; ++u) {
                const uint32_t v = base + u * kThreads + t;
                if (v < to) {
                    const float high = p[u].most();
                    p[u].values(x);
                    const uint32_t next = v + kBatch * kThreads;
                    if (next < to) p[u].load(w.z + w.at(next));
                    if (high > r.limit) r.raise(high);
                    const uint32_t skip = look ? marks_of(s, bits, true, w, from, to, a.t.top, v) : 0;
                    if (skip != 0) {
#pragma unroll
                        for (int e = 0; e < kVec; ++e)
                            if ((skip >> e) & 1u) x[e] = -CUDART_INF_F;
                    }
                    r.add(x);
                }
            }
        }
    };
    if (rest)
        read(true);
    else
        read(false);
    if (edge_at < n && !(rest && ((s.edge_bits >> t) & 1u) != 0)) {
        if (edge[0] > r.limit) r.raise(edge[0]);
        r.add(edge);
    }
    // The teacher's terms about the first reference, the sums about the largest.
    m = fmaxf(m, -FLT_MAX);
    Stats mine_sum = r.stats();
    const float warp_m = warp_max(mine_sum.m);
    rebase(mine_sum, warp_m, c);
    const float sum_part = warp_sum(mine_sum.s);
    if (warp * 32 < a.t.top) {
        bool leads = mine, alone = true;
        if (rest && s.again != 0 && t < a.t.top) lead(s, id, t, a.t.top, leads, alone);
        const float log_q = log_q_of(y, a.inv_t, rest, log_sum, y_max), q = id >= 0 ? expf(log_q) : 0.0f;
        const float top_part = warp_sum(rest && leads ? pow2(exponent(zt, m, c)) : 0.0f);
        const float held_part = warp_sum(q);
        const float cross_part = warp_sum(cross_term(q, log_q, zt, m, a.inv_t));
        if (lane == 0) {
            s.warp[3][warp] = top_part;
            s.warp[4][warp] = held_part;
            s.warp[5][warp] = cross_part;
        }
    } else if (lane == 0) {
        s.warp[3][warp] = s.warp[4][warp] = s.warp[5][warp] = 0.0f;
    }
    if (lane == 0) {
        s.warp[6][warp] = warp_m;
        s.warp[2][warp] = sum_part;
    }
    bool far = __syncthreads_or(r.far()) != 0;
    float all = fmaxf(max_of<kThreads>(s.warp[6]), m);
    const uint32_t k = lane & (kThreads / 32 - 1);
    float outside = lane < kThreads / 32 ? s.warp[2][k] * pow2(exponent(s.warp[6][k], all, c)) : 0.0f;
    outside = warp_sum(outside);
    float top_sum = sum_of<kThreads>(s.warp[3]) * pow2(exponent(m, all, c));
    float held = sum_of<kThreads>(s.warp[4]);
    float cross = sum_of<kThreads>(s.warp[5]);
    if constexpr (kCluster) {
        cg::cluster_group cluster = cg::this_cluster();
        if (t == 0) {
            s.m = all;
            s.outside = outside;
            s.top = top_sum;
            s.far = far;
        }
        cluster.sync();
        const auto* other = cluster.map_shared_rank(&s, lane & (shares - 1));
        const float other_m = other->m, other_outside = other->outside, other_top = other->top;
        far = __any_sync(kFull, other->far);
        all = warp_max(other_m);
        const float f = pow2(exponent(other_m, all, c));
        outside = warp_sum(lane < shares ? other_outside * f : 0.0f);
        top_sum = warp_sum(lane < shares ? other_top * f : 0.0f);
        cluster.sync();  // the shares' memory is read
    }
    const float sum = outside + top_sum, rest_q = rest ? fmaxf(1.0f - held, 0.0f) : 0.0f;
    if (far || (rest_q > 0.0f && sum != 0.0f && taught && outside < kApart * sum)) return false;
    if (t == 0 && share == 0) {
        cross += held * ((all * kDown - m * kDown) * a.inv_t);
        if (!rest && held != 0.0f) {
            cross = cross / held - logf(held) * kDown;
            held = 1.0f;
        }
        a.loss[i] = sum == 0.0f || !taught ? 0.0f : loss_of(weight, cross, held, sum, logf(outside), rest_q);
    }
    return true;
}

template <class T, int kVec, int kThreads, bool kCluster>
__global__ void __launch_bounds__(kThreads) distill_loss_kernel(const __grid_constant__ DistillArgs a, uint32_t shares) {
    __shared__ Shared<kThreads> s;
    extern __shared__ __align__(16) unsigned char held[];
    uint32_t* bits = reinterpret_cast<uint32_t*>(held);
    const uint32_t shift = kCluster ? __ffs(shares) - 1 : 0;
    const uint32_t i = blockIdx.x >> shift, share = blockIdx.x & (shares - 1);
    if (loss_list<T, kVec, kThreads, kCluster>(s, bits, a, i, share, shares)) return;
    __syncthreads();
    Maxima most;
    Ahead ahead;
    distill_list<T, kVec, kThreads, kCluster>(s, nullptr, 0, bits, a, i, a.l.lists, ahead, share, shares, most);
}

template <class T, int kVec, int kThreads, bool kCluster>
__global__ void __launch_bounds__(kThreads, 768 / kThreads)
    distill_rows_kernel(const __grid_constant__ DistillArgs a, uint32_t shares, uint32_t slots) {
    if (a.stopped != nullptr && *a.stopped) return;
    extern __shared__ __align__(16) unsigned char held[];
    __shared__ Shared<kThreads> s;
    Maxima most;
    Pack<T, kVec>* data = reinterpret_cast<Pack<T, kVec>*>(held);
    uint32_t* bits = reinterpret_cast<uint32_t*>(held + ((slots * sizeof(Pack<T, kVec>) + 15) & ~static_cast<size_t>(15)));
    if (kVec > 1 && slots == 0) bits = nullptr;  // no shared memory at all
    const uint32_t shift = kCluster ? __ffs(shares) - 1 : 0, step = gridDim.x >> shift;
    Ahead ahead;
    for (uint32_t i = blockIdx.x >> shift; i < a.l.lists; i += step) {
        distill_list<T, kVec, kThreads, kCluster>(s, data, slots, bits, a, i, i + step, ahead, blockIdx.x & (shares - 1), shares, most);
        __syncthreads();  // what the list left in shared memory is read
    }
    if (kVec == 1) clear_ends<T>(a);
    publish<kThreads>(a, most);
}

// A warp's teacher: its marks (a bit an entry of the list), ids and q.
struct WarpShared {
    uint32_t bits[32];
    int32_t id[kMaxTop];
    float q[kMaxTop];
};

// rest_apart() of a warp's list (`cross`: a lane's part).
template <class T>
__device__ __noinline__ Maxima warp_rest_apart(const WarpShared& s, const DistillArgs& a, uint32_t i, uint64_t first, uint32_t n,
                                               float m, float sum, float held, float cross, Maxima most) {
    const uint32_t lane = threadIdx.x & 31;
    const T* z = static_cast<const T*>(a.l.scores) + first;
    const float c = __fmul_rn(kLog2E, a.inv_t), weight = a.weight != nullptr ? a.weight[i] : 1.0f;
    auto each = [&](auto f) {
        for (uint32_t j = lane; j < n; j += 32)
            if (((s.bits[j / 32] >> lane) & 1u) == 0) f(to_float(z[j]), j);
    };
    float rest_m = -CUDART_INF_F, rest_sum = 0.0f;
    each([&](float x, uint32_t) { rest_m = fmaxf(rest_m, x); });
    rest_m = warp_max(rest_m);
    const bool some = has_mass(rest_m, m, sum, c);
    if (some) each([&](float x, uint32_t) { rest_sum += pow2(exponent(x, rest_m, c)); });
    rest_sum = warp_sum(rest_sum);
    const float r = some ? 1.0f - held : 0.0f;
    cross = warp_sum(cross);
    if (lane == 0 && a.loss != nullptr)
        a.loss[i] = loss_of(weight, cross, held, sum, (rest_m - m) * a.inv_t + logf(rest_sum), r);
    if (a.grad == nullptr && a.hess == nullptr) return most;
    const uint64_t out = a.l.bounds != nullptr ? first : static_cast<uint64_t>(i) * a.grad_stride;
    const float mass = held + r, scale = weight * a.inv_t, inv_s = 1.0f / sum, pull = some ? r / rest_sum : 0.0f;
    auto put_one = [&](float x, uint32_t j, float less) {
        const float p = pow2(exponent(x, m, c)) * inv_s;
        put<T>(a, out + j, first + j, (mass * p - less) * scale, hessian_of(mass * scale * a.inv_t, p), true, most);
    };
    each([&](float x, uint32_t j) { put_one(x, j, some ? pull * pow2(exponent(x, rest_m, c)) : 0.0f); });
    __syncwarp();  // the lanes' q
    for (uint32_t k = lane; k < a.t.top; k += 32) {
        const int32_t id = s.id[k];
        bool leads = id >= 0;
        for (uint32_t e = 0; e < k && leads; ++e) leads = s.id[e] != id;
        if (!leads) continue;
        float q = 0.0f;
        for (uint32_t e = k; e < a.t.top; ++e)
            if (s.id[e] == id) q += s.q[e];
        put_one(to_float(z[id]), static_cast<uint32_t>(id), q);
    }
    return most;
}

// A list of at most 32 kItems entries by one warp, in registers; kTop of the teacher's entries a lane.
template <class T, int kItems, int kTop>
__device__ __forceinline__ void distill_warp(WarpShared& s, const DistillArgs& a, uint32_t i, uint64_t first, uint32_t n,
                                             const int32_t (&ids)[kTop], const float (&logits)[kTop], Maxima& most) {
    const uint32_t lane = threadIdx.x & 31;
    const T* z = static_cast<const T*>(a.l.scores) + first;
    const float c = __fmul_rn(kLog2E, a.inv_t);
    const bool rest = a.t.log_sum != nullptr;
    float x[kItems], m = -CUDART_INF_F;
#pragma unroll
    for (int u = 0; u < kItems; ++u) {
        const uint32_t j = u * 32 + lane;
        x[u] = j < n ? to_float(z[j]) : -CUDART_INF_F;
        m = fmaxf(m, x[u]);
    }
    int32_t id[kTop];
    float y[kTop], zt[kTop], y_max = -CUDART_INF_F;
    bool taught = false, again = false;
    if (lane < kItems) s.bits[lane] = 0;
    __syncwarp();
#pragma unroll
    for (int u = 0; u < kTop; ++u) {
        id[u] = -1;
        y[u] = zt[u] = -CUDART_INF_F;
        const uint32_t k = u * 32 + lane;
        if (k < a.t.top) {
            if (ids[u] >= 0 && static_cast<uint32_t>(ids[u]) < n) id[u] = ids[u];
            s.id[k] = id[u];
        }
        if (id[u] >= 0) {
            y[u] = logits[u];
            zt[u] = to_float(z[id[u]]);
            const uint32_t mark = 1u << (id[u] & 31);
            again |= (atomicOr(&s.bits[id[u] / 32], mark) & mark) != 0;
            taught = true;
        }
        y_max = fmaxf(y_max, y[u]);
    }
    __syncwarp();  // the marks and the ids, which other lanes read (votes and shuffles order no memory)
    m = fmaxf(warp_max(m), -FLT_MAX);
    y_max = fmaxf(warp_max(y_max), -FLT_MAX);
    taught = __any_sync(kFull, taught);
    again = __any_sync(kFull, again);    // an index named twice
    uint32_t marks = 0;
    float sum = 0.0f;
#pragma unroll
    for (int u = 0; u < kItems; ++u) {
        const bool mark = ((s.bits[u] >> lane) & 1u) != 0;
        marks |= mark ? 1u << u : 0u;
        x[u] = pow2(exponent(x[u], m, c));
        if (!(rest && mark)) sum += x[u];
    }
    // Leaders: the first entry of the teacher that names an index.
    float top_sum = 0.0f, total = 0.0f;
    uint32_t leads = 0, alone = 0;
#pragma unroll
    for (int u = 0; u < kTop; ++u) {
        bool first_one = id[u] >= 0, only = true;
        if (again) {
            for (uint32_t k = 0; k < a.t.top; ++k)
                if (s.id[k] == id[u] && k != u * 32 + lane) {
                    only = false;
                    if (k < u * 32 + lane) first_one = false;
                }
        }
        leads |= first_one ? 1u << u : 0u;
        alone |= only ? 1u << u : 0u;
        if (rest && first_one) top_sum += pow2(exponent(zt[u], m, c));
        if (!rest && id[u] >= 0) total += expf(log_q_of(y[u], a.inv_t, rest, 0.0f, y_max));
    }
    const float outside = warp_sum(sum);
    if (rest) {
        top_sum = warp_sum(top_sum);
    } else {
        total = warp_sum(total);
    }
    sum = outside + top_sum;
    const float log_total = logf(total), log_sum = rest ? a.t.log_sum[i] : 0.0f;
    float held = 0.0f, cross = 0.0f, q[kTop];
#pragma unroll
    for (int u = 0; u < kTop; ++u) {
        float log_q = -CUDART_INF_F;
        if (id[u] >= 0 && (rest || total != 0.0f))
            log_q = log_q_of(y[u], a.inv_t, rest, log_sum, y_max) - (rest ? 0.0f : log_total);
        q[u] = expf(log_q);
        held += q[u];
        cross += cross_term(q[u], log_q, zt[u], m, a.inv_t);
        if (u * 32 + lane < a.t.top) s.q[u * 32 + lane] = q[u];
    }
    held = warp_sum(held);
    const float r = rest ? fmaxf(1.0f - held, 0.0f) : 0.0f;
    const bool empty = sum == 0.0f || !taught;
    const float weight = a.weight != nullptr ? a.weight[i] : 1.0f;
    const Slopes k = slopes_of(weight, a.inv_t, held, r, sum, outside);
    if (!empty && rest_is_apart(r, sum, outside, k)) {
        most = warp_rest_apart<T>(s, a, i, first, n, m, sum, held, cross, most);
        return;
    }
    if (a.loss != nullptr) {
        cross = warp_sum(cross);
        if (lane == 0) a.loss[i] = empty ? 0.0f : loss_of(weight, cross, held, sum, logf(outside), r);
    }
    if (a.grad == nullptr && a.hess == nullptr) return;
    const uint64_t out = a.l.bounds != nullptr ? first : static_cast<uint64_t>(i) * a.grad_stride;
#pragma unroll
    for (int u = 0; u < kItems; ++u) {
        const uint32_t j = u * 32 + lane;
        const float p = x[u] * k.inv_s;
        if (j < n)
            put<T>(a, out + j, first + j, empty ? 0.0f : k.slope * x[u], empty ? 0.0f : hessian_of(k.curve, p),
                   ((marks >> u) & 1u) == 0, most);
    }
    __syncwarp();  // the top's own go over them
#pragma unroll
    for (int u = 0; u < kTop; ++u) {
        if (((leads >> u) & 1u) == 0 || empty) continue;
        float taught_q = q[u];
        if (((alone >> u) & 1u) == 0) {
            taught_q = 0.0f;
            for (uint32_t e = 0; e < a.t.top; ++e)
                if (s.id[e] == id[u]) taught_q += s.q[e];
        }
        const float e = pow2(exponent(zt[u], m, c)), p = e * k.inv_s;
        put<T>(a, out + id[u], first + id[u], k.top_slope * e - taught_q * (weight * a.inv_t), hessian_of(k.curve, p), true, most);
    }
}

// `per` lists a CTA (8 at most), a warp each of at most 32 kMost entries; a longer one among them by the whole CTA. So what
// a list gives depends on its own length alone.
template <class T, int kTop, int kMost>
__global__ void __launch_bounds__(kWarpThreads, kMost > 16 ? 2 : 4)
    distill_warps_kernel(const __grid_constant__ DistillArgs a, uint32_t per) {
    constexpr uint32_t kEntries = 32 * kMost;
    if (a.stopped != nullptr && *a.stopped) return;
    __shared__ WarpShared warps[kWarpThreads / 32];
    __shared__ Shared<kWarpThreads> shared;
    __shared__ uint32_t bits[kBits / 32];
    const uint32_t base = blockIdx.x * per, i = base + (threadIdx.x >> 5);
    uint64_t first = 0;
    uint32_t n = 0;
    Maxima most;
    if (threadIdx.x >> 5 < per && i < a.l.lists) {
        // The teacher's entries, on their way beside the boundaries.
        int32_t ids[kTop];
        float logits[kTop];
#pragma unroll
        for (int u = 0; u < kTop; ++u) {
            const uint32_t k = u * 32 + (threadIdx.x & 31);
            const uint64_t at = static_cast<uint64_t>(i) * a.t.stride + k;
            ids[u] = k < a.t.top ? a.t.ids[at] : -1;
            logits[u] = k < a.t.top ? load_typed(a.t.logits, a.t.type, at) : 0.0f;
        }
        list_range(a.l, i, first, n);
        WarpShared& s = warps[threadIdx.x >> 5];
        if (n <= 128)
            distill_warp<T, 4, kTop>(s, a, i, first, n, ids, logits, most);
        else if (n <= 256)
            distill_warp<T, 8, kTop>(s, a, i, first, n, ids, logits, most);
        else if (n <= 512)
            distill_warp<T, 16, kTop>(s, a, i, first, n, ids, logits, most);
        else if (n <= kEntries)
            distill_warp<T, kMost, kTop>(s, a, i, first, n, ids, logits, most);
    }
    if (__syncthreads_or(n > kEntries) != 0)
        for (uint32_t k = base; k < base + per && k < a.l.lists; ++k) {
            list_range(a.l, k, first, n);
            if (n <= kEntries) continue;
            Ahead ahead;
            distill_list<T, 1, kWarpThreads, false>(shared, nullptr, 0, bits, a, k, a.l.lists, ahead, 0, 1, most);
            __syncthreads();
        }
    clear_ends<T>(a);
    publish<kWarpThreads>(a, most);
}

// Shared memory of a CTA that holds `slots` vectors and their marks.
template <class T, int kVec>
size_t rows_smem(uint32_t slots) {
    if (kVec == 1) return kBits / 8;
    const size_t entries = static_cast<size_t>(slots) * kVec;
    return ((slots * sizeof(Pack<T, kVec>) + 15) & ~static_cast<size_t>(15)) + (std::min<size_t>(entries, kBits) + 31) / 32 * 4;
}

// A launch of `shares` CTAs for each of `lists` lists at a time, as clusters where that is more than one.
template <class Kernel, class... Args>
void launch_shares(Kernel* kernel, const DistillArgs& a, uint32_t lists, int threads, size_t smem, uint32_t shares, cudaStream_t s,
                   Args... args) {
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(lists * shares);
    config.blockDim = dim3(threads);
    config.dynamicSmemBytes = smem;
    config.stream = s;
    cudaLaunchAttribute cluster{};
    cluster.id = cudaLaunchAttributeClusterDimension;
    cluster.val.clusterDim.x = shares;
    cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
    config.attrs = &cluster;
    config.numAttrs = shares > 1 ? 1 : 0;
    // (48 KB go without the attribute; setting it is host time)
    if (smem > 40 * 1024 && cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxHeld) != cudaSuccess) return;
    cudaLaunchKernelEx(&config, kernel, a, shares, args...);
}

template <class T, int kVec, int kThreads>
void launch_rows(const DistillArgs& a, uint32_t shares, uint32_t slots, cudaStream_t s) {
    const size_t smem = rows_smem<T, kVec>(slots);
    // CTAs alone that hold their lists: as many as the SMs hold (by threads and registers 768 threads' worth, by shared
    // memory 227 KB), each taking its next list while it writes.
    uint32_t lists = a.l.lists;
    if (kVec > 1 && shares == 1) {
        const size_t each = smem + sizeof(Shared<kThreads>) + 1024;
        const uint32_t ctas = static_cast<uint32_t>(std::min<size_t>(768 / kThreads, 227 * 1024 / each));
        lists = std::min(lists, a.sms * std::max(1u, ctas));
    }
    launch_shares(shares > 1 ? distill_rows_kernel<T, kVec, kThreads, true> : distill_rows_kernel<T, kVec, kThreads, false>, a,
                  lists, kThreads, smem, shares, s, slots);
}

template <class T, int kVec, int kThreads>
void launch_loss(const DistillArgs& a, uint32_t shares, uint64_t entries, cudaStream_t s) {
    launch_shares(shares > 1 ? distill_loss_kernel<T, kVec, kThreads, true> : distill_loss_kernel<T, kVec, kThreads, false>, a,
                  a.l.lists, kThreads, static_cast<size_t>(std::min<uint64_t>(entries / shares + kVec, kBits) / 32 + 1) * 4, shares, s);
}

template <class T>
void launch_typed(const DistillArgs& a, cudaStream_t s) {
    constexpr int kVec = 16 / sizeof(T);
    const uint64_t mean = a.l.bounds != nullptr ? a.l.width / a.l.lists : a.l.width;
    const bool narrow = mean <= (a.l.bounds != nullptr ? kWarpMean : 512);
    if (narrow || a.max_g != nullptr) {  // a training iteration's queries: the same gradients on any rank
        const uint32_t per = narrow ? kWarpThreads / 32 : 1, grid = a.l.lists / per + (a.l.lists % per != 0);
        if (a.t.top <= 32)
            distill_warps_kernel<T, 1, 16><<<grid, kWarpThreads, 0, s>>>(a, per);
        else
            distill_warps_kernel<T, 4, 16><<<grid, kWarpThreads, 0, s>>>(a, per);
        return;
    }
    if (a.l.bounds == nullptr && mean <= 1024) {  // (8000 x 1000 f32: a warp each 21 us, a CTA each 38; 64 of them: 5.4 and 4.7)
        const uint32_t per = kWarpThreads / 32, grid = a.l.lists / per + (a.l.lists % per != 0);
        if (a.t.top <= 32)
            distill_warps_kernel<T, 1, 32><<<grid, kWarpThreads, 0, s>>>(a, per);
        else
            distill_warps_kernel<T, 4, 32><<<grid, kWarpThreads, 0, s>>>(a, per);
        return;
    }
    uint32_t shares = list_shares(mean, a.l.lists, a.sms);
    if (a.l.bounds != nullptr) {
        if (mean / shares <= 1024)  // (8M scores, f32: lists of 1000 by 128 threads 60 us, by 256 102; of 4000, 39 and 49)
            launch_rows<T, 1, 128>(a, shares, 0, s);
        else
            launch_rows<T, 1, 256>(a, shares, 0, s);
        return;
    }
    if (a.grad == nullptr && a.hess == nullptr) {
        if (a.loss == nullptr) return;
        if (mean / shares <= 4096)  // (64M scores, bf16: lists of 4000 by 128 threads 67 us, by 256 103; of 16000, 39 and 46)
            launch_loss<T, kVec, 128>(a, shares, mean, s);
        else
            launch_loss<T, kVec, 256>(a, shares, mean, s);
        return;
    }
    // As many shares as hold the list in kHeld bytes each, else in kMaxHeld (longer: read again).
    const uint64_t bytes = mean * sizeof(T);
    while (shares < 8 && bytes > static_cast<uint64_t>(shares) * kHeld) shares *= 2;
    uint64_t slots = (mean / kVec + shares - 1) / shares;
    if (rows_smem<T, kVec>(static_cast<uint32_t>(std::min<uint64_t>(slots, kMaxHeld / 16))) > kMaxHeld) slots = 0;
    // (f32, 32M scores: lists of 4000 by 128 threads 67 us, by 256 92; of 16000, 71 and 58. bf16, 64M: of 4000, 109 and 174; of
    // 16000, 62 and 74: the border lies between 4096 entries and 64 KB.)
    if (mean / shares <= 4096)
        launch_rows<T, kVec, 128>(a, shares, static_cast<uint32_t>(slots), s);
    else
        launch_rows<T, kVec, 256>(a, shares, static_cast<uint32_t>(slots), s);
}

}  // namespace

void launch_distill(const DistillArgs& a, cudaStream_t s) {
    if (a.l.type == SB2_F32)
        launch_typed<float>(a, s);
    else if (a.l.type == SB2_BF16)
        launch_typed<__nv_bfloat16>(a, s);
    else
        launch_typed<__half>(a, s);
}

}  // namespace sb2
