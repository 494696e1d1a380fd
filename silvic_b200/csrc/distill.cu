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
// little there.
#include "lists_device.cuh"

namespace sb2 {

namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ float block_sum(float v, float* s) {
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.0f;
    for (int w = 0; w < kThreads / 32; ++w) v += s[w];
    return v;
}

__device__ __forceinline__ float block_max(float v, float* s) {
    for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
    __syncthreads();
    v = s[0];
    for (int w = 1; w < kThreads / 32; ++w) v = fmaxf(v, s[w]);
    return v;
}

// A CTA per list: the teacher's q, the maximum, the sums in and outside the top, then the gradients.
template <class T>
__global__ void __launch_bounds__(kThreads) distill_kernel(DistillArgs a) {
    if (a.stopped != nullptr && *a.stopped) return;
    __shared__ float s_red[kThreads / 32];
    __shared__ int32_t s_id[kMaxTop];
    __shared__ float s_q[kMaxTop];
    const float c = __fmul_rn(kLog2E, a.inv_t);
    const bool rest = a.t.log_sum != nullptr;
    const uint32_t k = a.t.top;
    float most_g = 0.0f, most_h = 0.0f;
    for (uint32_t i = blockIdx.x; i < a.l.lists; i += gridDim.x) {
        uint64_t first;
        uint32_t n;
        list_range(a.l, i, first, n);
        const T* z = static_cast<const T*>(a.l.scores) + first;
        // The teacher: entry threadIdx.x of the top (kMaxTop <= kThreads).
        int32_t id = -1;
        float y = -CUDART_INF_F;
        if (threadIdx.x < k) {
            id = a.t.ids[static_cast<uint64_t>(i) * a.t.stride + threadIdx.x];
            if (id < 0 || static_cast<uint32_t>(id) >= n) id = -1;
            if (id >= 0) y = load_typed(a.t.logits, a.t.type, static_cast<uint64_t>(i) * a.t.stride + threadIdx.x) * a.inv_t;
        }
        float log_q;
        if (rest) {
            log_q = y - a.t.log_sum[i];
            if (id < 0) log_q = -CUDART_INF_F;
        } else {
            float most = block_max(y, s_red);
            if (most == -CUDART_INF_F) most = 0.0f;
            const float total = block_sum(expf(y - most), s_red);
            log_q = total == 0.0f ? -CUDART_INF_F : y - most - logf(total);
        }
        const float q = expf(log_q);
        const bool taught_at_all = __syncthreads_or(id >= 0) != 0;
        float held = block_sum(q, s_red);
        __syncthreads();
        if (threadIdx.x < k) {
            s_id[threadIdx.x] = id;
            s_q[threadIdx.x] = q;
        }
        __syncthreads();
        // The student.
        float m = -CUDART_INF_F;
        for (uint32_t j = threadIdx.x; j < n; j += kThreads) m = fmaxf(m, to_float(z[j]));
        m = block_max(m, s_red);
        if (m == -CUDART_INF_F) m = 0.0f;
        float in = 0.0f, out = 0.0f;
        for (uint32_t j = threadIdx.x; j < n; j += kThreads) {
            const float e = pow2(exponent(to_float(z[j]), m, c));
            bool taught = false;
            for (uint32_t t = 0; rest && t < k; ++t) taught |= s_id[t] == static_cast<int32_t>(j);
            if (taught)
                in += e;
            else
                out += e;
        }
        in = block_sum(in, s_red);
        out = block_sum(out, s_red);
        const float sum = in + out;
        const bool empty = sum == 0.0f || !taught_at_all;
        const float log_s = logf(sum), inv_s = 1.0f / sum;
        const float w = a.weight != nullptr ? a.weight[i] : 1.0f;
        float r = rest && out > 0.0f ? fmaxf(1.0f - held, 0.0f) : 0.0f;
        float term = 0.0f;
        if (q > 0.0f || q != q) term = q * (log_q - ((to_float(z[id]) - m) * a.inv_t - log_s));
        float loss = block_sum(term, s_red);
        if (r > 0.0f) loss += r * (logf(r) - (logf(out) - log_s));
        held += r;
        const float pull = r > 0.0f ? r / (out * inv_s) : 0.0f;
        if (threadIdx.x == 0 && a.loss != nullptr) a.loss[i] = empty ? 0.0f : loss * w;
        const uint64_t to = a.l.bounds != nullptr ? first : static_cast<uint64_t>(i) * a.grad_stride;
        for (uint32_t j = threadIdx.x; j < n && (a.grad != nullptr || a.hess != nullptr); j += kThreads) {
            const float p = empty ? 0.0f : pow2(exponent(to_float(z[j]), m, c)) * inv_s;
            float teach = 0.0f;
            bool taught = false;
            for (uint32_t t = 0; t < k; ++t)
                if (s_id[t] == static_cast<int32_t>(j)) {
                    teach += s_q[t];
                    taught = true;
                }
            float g = (taught ? held * p - teach : (held - pull) * p) * (w * a.inv_t);
            float h = held * p * (1.0f - p) * (w * a.inv_t * a.inv_t);
            if (empty) g = h = 0.0f;
            if (a.row_weight != nullptr) {
                g *= a.row_weight[first + j];
                h *= a.row_weight[first + j];
            }
            most_g = fmaxf(most_g, fabsf(g));
            most_h = fmaxf(most_h, fabsf(h));
            if (a.grad != nullptr) static_cast<T*>(a.grad)[to + j] = from_float<T>(g);
            if (a.hess != nullptr) static_cast<T*>(a.hess)[to + j] = from_float<T>(h);
        }
        __syncthreads();  // the teacher's entries are read before the next list's are written
    }
    if (a.max_g != nullptr) {
        most_g = block_max(most_g, s_red);
        most_h = block_max(most_h, s_red);
        if (threadIdx.x == 0) {  // non-negative doubles order like their bit patterns
            atomicMax(a.max_g, static_cast<unsigned long long>(__double_as_longlong(static_cast<double>(most_g))));
            atomicMax(a.max_h, static_cast<unsigned long long>(__double_as_longlong(static_cast<double>(most_h))));
        }
    }
}

}  // namespace

void launch_distill(const DistillArgs& a, cudaStream_t s) {
    const uint32_t most = a.sms * 8, grid = a.l.lists < most ? a.l.lists : most;
    if (a.l.type == SB2_F32)
        distill_kernel<float><<<grid, kThreads, 0, s>>>(a);
    else if (a.l.type == SB2_BF16)
        distill_kernel<__nv_bfloat16><<<grid, kThreads, 0, s>>>(a);
    else
        distill_kernel<__half><<<grid, kThreads, 0, s>>>(a);
}

}  // namespace sb2
