// log_probs.cu — log probabilities of given entries, entropy and top alternatives of softmax(z / T) over each list.
//
// With m = max z, S = sum exp((z - m) / T) and U = sum exp((z - m) / T) (z - m):
//   log p_i = (z_i - m) / T - ln S,  log sum = m / T + ln S,  entropy = ln S - U / (T S).
// Statistics are f32 sums; the alternatives are ordered by the scores themselves (ties by the lower index), so no
// rounding decides an index.
#include "lists_device.cuh"

namespace sb2 {

namespace {

constexpr int kThreads = 256;

// The block's maximum of a key, in every thread.
__device__ __forceinline__ unsigned long long block_max_key(unsigned long long k, unsigned long long* s) {
    for (int o = 16; o > 0; o >>= 1) {
        const unsigned long long other = __shfl_xor_sync(0xffffffffu, k, o);
        k = k > other ? k : other;
    }
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = k;
    __syncthreads();
    for (int w = 0; w < kThreads / 32; ++w) k = k > s[w] ? k : s[w];
    return k;
}

__device__ __forceinline__ float block_sum(float v, float* s) {
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.0f;
    for (int w = 0; w < kThreads / 32; ++w) v += s[w];
    return v;
}

// A CTA per list: the maximum, the sums, then one pass per alternative.
template <class T>
__global__ void __launch_bounds__(kThreads) log_probs_kernel(LogProbsArgs a) {
    __shared__ unsigned long long s_key[kThreads / 32];
    __shared__ float s_sum[kThreads / 32];
    const float c = __fmul_rn(kLog2E, a.inv_t);
    for (uint32_t i = blockIdx.x; i < a.l.lists; i += gridDim.x) {
        uint64_t first;
        uint32_t n;
        list_range(a.l, i, first, n);
        const T* z = static_cast<const T*>(a.l.scores) + first;
        unsigned long long best = 0;
        for (uint32_t j = threadIdx.x; j < n; j += kThreads) {
            const unsigned long long key = order_key(to_float(z[j]), j);
            best = best > key ? best : key;
        }
        best = block_max_key(best, s_key);
        float m = n > 0 ? to_float(z[0xFFFFFFFFu - static_cast<uint32_t>(best)]) : -CUDART_INF_F;
        const bool empty = m == -CUDART_INF_F;
        if (empty) m = 0.0f;
        float sum = 0.0f, part = 0.0f;
        for (uint32_t j = threadIdx.x; j < n; j += kThreads) {
            const float d = __fsub_rn(to_float(z[j]), m), e = exp_of(d, c);
            sum += e;
            if (e > 0.0f) part += e * d;
        }
        sum = block_sum(sum, s_sum);
        part = block_sum(part, s_sum);
        const float log_s = logf(sum);
        if (threadIdx.x == 0) {
            if (a.log_sum != nullptr) a.log_sum[i] = empty ? -CUDART_INF_F : m * a.inv_t + log_s;
            if (a.entropy != nullptr) a.entropy[i] = empty ? 0.0f : log_s - part * a.inv_t / sum;
        }
        for (uint32_t g = threadIdx.x; g < a.num_given; g += kThreads) {
            const uint64_t at = static_cast<uint64_t>(i) * a.num_given + g;
            const int32_t id = a.given[at];
            a.given_out[at] = id < 0 || static_cast<uint32_t>(id) >= n || empty ? -CUDART_INF_F
                                                                               : (to_float(z[id]) - m) * a.inv_t - log_s;
        }
        unsigned long long last = best;
        for (uint32_t r = 0; r < a.top; ++r) {
            if (r > 0) {
                unsigned long long next = 0;
                for (uint32_t j = threadIdx.x; j < n; j += kThreads) {
                    const unsigned long long key = order_key(to_float(z[j]), j);
                    if (key < last && key > next) next = key;
                }
                last = block_max_key(next, s_key);
            }
            if (threadIdx.x == 0) {
                const uint64_t at = static_cast<uint64_t>(i) * a.top + r;
                const uint32_t id = 0xFFFFFFFFu - static_cast<uint32_t>(last);
                const float v = last == 0 ? -CUDART_INF_F : to_float(z[id]);
                const bool none = v == -CUDART_INF_F;
                a.top_ids[at] = none ? -1 : static_cast<int32_t>(id);
                a.top_out[at] = none ? -CUDART_INF_F : (v - m) * a.inv_t - log_s;
            }
        }
    }
}

}  // namespace

void launch_log_probs(const LogProbsArgs& a, cudaStream_t s) {
    const uint32_t most = a.sms * 8, grid = a.l.lists < most ? a.l.lists : most;
    if (a.l.type == SB2_F32)
        log_probs_kernel<float><<<grid, kThreads, 0, s>>>(a);
    else if (a.l.type == SB2_BF16)
        log_probs_kernel<__nv_bfloat16><<<grid, kThreads, 0, s>>>(a);
    else
        log_probs_kernel<__half><<<grid, kThreads, 0, s>>>(a);
}

}  // namespace sb2
