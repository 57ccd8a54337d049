// k_logprob.hip -- log probabilities of given tokens, entropy and the largest
// alternatives from a row of logits.
//
// With z_i = scale x_i - max scale x, T = sum exp(z_i):
//   log p_i = z_i - log T,  H = log T - (sum exp(z_i) z_i) / T
// (both terms of H are >= 0: nothing cancels).  Order: 64-bit keys of the
// logit's bits made monotone and the complement of its index, all distinct,
// so that the alternatives do not depend on who finds them.
#include "cbx_device.h"

namespace cbx {
namespace {

constexpr int kLpThreads = 256;

struct LpArgs {
    const char* x;
    const int32_t* ids;
    float *logp, *entropy;
    char *top_ids, *top_logp;
    int64_t x_nb1, ti_nb1, tl_nb1;
    uint32_t V, rows;
    int32_t n_top;
    float scale;
    uint32_t* err;
};

// Larger logits have larger keys; NaN the largest, -0 as +0, of equal ones the first index.
__device__ __forceinline__ uint64_t key_of(float x, uint32_t i) {
    const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.0f);
    const uint32_t o = x != x ? 0xfffffffeu : ((b & 0x80000000u) ? ~b : b | 0x80000000u);
    return (static_cast<uint64_t>(o) << 32) | (0xffffffffu - i);
}

template <typename T>
__global__ __launch_bounds__(kLpThreads) void k_logprob(LpArgs a) {
    __shared__ float ldsf[kLpThreads / 64];
    __shared__ unsigned long long lds64[kLpThreads / 64];
    const uint32_t row = blockIdx.x, tid = threadIdx.x;
    const char* x = a.x + row * a.x_nb1;
    auto at = [&](uint32_t i) { return Elt<T>::load1(x + static_cast<int64_t>(i) * Elt<T>::size); };
    float m = -INFINITY;
    for (uint32_t i = tid; i < a.V; i += kLpThreads) m = fmaxf(m, at(i));
    for (int d = 32; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor(m, d));
    if ((tid & 63) == 0) ldsf[tid >> 6] = m;
    __syncthreads();
    m = ldsf[0];
    for (int w = 1; w < kLpThreads / 64; w++) m = fmaxf(m, ldsf[w]);
    __syncthreads();
    const float ms = m * a.scale;
    const bool none = m == -INFINITY;   // no logit above -inf (or NaN alone)
    float total = 0.0f, u = 0.0f;
    for (uint32_t i = tid; i < a.V; i += kLpThreads) {
        const float v = at(i);
        if (v == -INFINITY) continue;
        const float z = v * a.scale - ms;
        const float e = expf(z);
        total += e;
        u += e > 0.0f ? e * z : 0.0f;
        if (e != e) u = e;
    }
    for (int pass = 0; pass < 2; pass++) {
        float& t = pass ? u : total;
        for (int d = 32; d > 0; d >>= 1) t += __shfl_xor(t, d);
        if ((tid & 63) == 0) ldsf[tid >> 6] = t;
        __syncthreads();
        t = ldsf[0];
        for (int w = 1; w < kLpThreads / 64; w++) t += ldsf[w];
        __syncthreads();
    }
    const bool empty = none && total == 0.0f;
    const float lse = empty ? 0.0f : logf(total);
    auto log_p = [&](float v) { return v == -INFINITY && total == total ? v : v * a.scale - ms - lse; };
    if (tid == 0) {
        if (a.logp) {
            const int32_t id = a.ids[row];
            float r = 0.0f;
            if (id < 0 || static_cast<uint32_t>(id) >= a.V) atomicOr(a.err, DEV_ERR_ROW_INDEX);
            else r = log_p(at(static_cast<uint32_t>(id)));
            a.logp[row] = r;
        }
        if (a.entropy) a.entropy[row] = empty ? 0.0f : lse - u / total;
    }
    uint64_t last = ~uint64_t{0};
    for (int r = 0; r < a.n_top; r++) {
        uint64_t best = 0;
        for (uint32_t i = tid; i < a.V; i += kLpThreads) {
            const uint64_t k = key_of(at(i), i);
            if (k < last && k > best) best = k;
        }
        for (int d = 32; d > 0; d >>= 1) {
            const uint64_t o = __shfl_xor(static_cast<unsigned long long>(best), d);
            best = o > best ? o : best;
        }
        if ((tid & 63) == 0) lds64[tid >> 6] = best;
        __syncthreads();
        best = lds64[0];
        for (int w = 1; w < kLpThreads / 64; w++) best = lds64[w] > best ? lds64[w] : best;
        __syncthreads();
        last = best;
        if (tid == 0) {
            const uint32_t i = 0xffffffffu - static_cast<uint32_t>(best);
            reinterpret_cast<int32_t*>(a.top_ids + row * a.ti_nb1)[r] = static_cast<int32_t>(i);
            reinterpret_cast<float*>(a.top_logp + row * a.tl_nb1)[r] = log_p(at(i));
        }
    }
}

}  // namespace

size_t token_log_probs_workspace(const cbx_tensor* x, int n_top, const DeviceState* st) {
    (void)x; (void)n_top; (void)st;
    return 0;
}

int launch_token_log_probs(const LogProbCall& c, DeviceState* st, hipStream_t s) {
    LpArgs a{};
    a.x = static_cast<const char*>(c.x->data);
    a.ids = c.ids ? static_cast<const int32_t*>(c.ids->data) : nullptr;
    a.logp = c.logp ? static_cast<float*>(c.logp->data) : nullptr;
    a.entropy = c.entropy ? static_cast<float*>(c.entropy->data) : nullptr;
    a.top_ids = c.top_ids ? static_cast<char*>(c.top_ids->data) : nullptr;
    a.top_logp = c.top_logp ? static_cast<char*>(c.top_logp->data) : nullptr;
    a.x_nb1 = c.x->nb[1];
    a.ti_nb1 = c.top_ids ? c.top_ids->nb[1] : 0;
    a.tl_nb1 = c.top_logp ? c.top_logp->nb[1] : 0;
    a.V = static_cast<uint32_t>(c.x->ne[0]);
    a.rows = static_cast<uint32_t>(c.x->ne[1]);
    a.n_top = c.n_top;
    a.scale = c.scale;
    a.err = st->err_word;
    const dim3 grid(a.rows), block(kLpThreads);
    if (c.x->type == CBX_TYPE_F16) hipLaunchKernelGGL((k_logprob<uint16_t>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((k_logprob<float>), grid, block, 0, s, a);
    return check_launch("cbx_token_log_probs");
}

}  // namespace cbx
