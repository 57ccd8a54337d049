// k_paged_attn.hip -- attention of one new token a request over a paged cache.
//
// y = sum_i softmax(s)_i v_i with s_i = scale * q . k_i in one pass over the
// keys: with the running maximum m, l = sum exp(s_i - m) and o = sum
// exp(s_i - m) v_i, both rescaled by exp(m - m') when the maximum rises to m',
// and y = o / l at the end.  f32 throughout.
//
// A workgroup a request and query head; its waves take keys in turn, a key's
// D elements over the lanes, and their (m, l, o) are joined in LDS.
#include "cbx_device.h"

namespace cbx {
namespace {

constexpr int kAttnThreads = 256;
constexpr int kAttnMaxD = 512;
constexpr float kLowest = -3.0e38f;   // below every finite score that matters; finite, so that m - m is 0

struct AttnArgs {
    const char *q, *k, *v, *tables;
    const int32_t* lens;
    char* y;
    int64_t q_nb1, q_nb2, y_nb1, y_nb2, k_nb1, k_nb2, k_nb3, v_nb1, v_nb2, v_nb3, t_nb1;
    uint32_t n_seq, hq, hkv, g, D, page, max_pages, n_pages;
    int32_t window;
    float scale, softcap;
    uint32_t* err;
};

__device__ __forceinline__ float wave_sum_f32(float v) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d);
    return v;
}

template <typename T, typename TC>
__global__ __launch_bounds__(kAttnThreads) void k_attn_rows(AttnArgs a) {
    constexpr int W = kAttnThreads / 64, N = kAttnMaxD / 64;
    __shared__ float lds_o[W][kAttnMaxD];
    __shared__ float lds_m[W], lds_l[W];
    const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
    const uint32_t s = blockIdx.x / a.hq, h = blockIdx.x - s * a.hq, hk = h / a.g;
    const int64_t cap = static_cast<int64_t>(a.max_pages) * a.page;
    int64_t len = a.lens[s];
    bool wrong = len < 0 || len > cap;
    len = len < 0 ? 0 : (len > cap ? cap : len);
    const int64_t first = a.window > 0 && len > a.window ? len - a.window : 0;
    const int32_t* row = reinterpret_cast<const int32_t*>(a.tables + s * a.t_nb1);
    const char* qr = a.q + s * a.q_nb2 + h * a.q_nb1;
    float q[N], o[N];
#pragma unroll
    for (int i = 0; i < N; i++) {
        const uint32_t e = lane + 64 * i;
        q[i] = e < a.D ? Elt<T>::load1(qr + e * Elt<T>::size) : 0.0f;
        o[i] = 0.0f;
    }
    float m = kLowest, l = 0.0f;
    for (int64_t key = first + wid; key < len; key += W) {
        const int32_t pi = static_cast<int32_t>(key / a.page), at = static_cast<int32_t>(key - static_cast<int64_t>(pi) * a.page);
        const int32_t pg = row[pi];
        if (pg < 0 || static_cast<uint32_t>(pg) >= a.n_pages) {
            wrong = true;
            continue;
        }
        const char* kr = a.k + pg * a.k_nb3 + hk * a.k_nb2 + at * a.k_nb1;
        const char* vr = a.v + pg * a.v_nb3 + hk * a.v_nb2 + at * a.v_nb1;
        float dot = 0.0f;
#pragma unroll
        for (int i = 0; i < N; i++) {
            const uint32_t e = lane + 64 * i;
            if (e < a.D) dot = fmaf(q[i], Elt<TC>::load1(kr + e * Elt<TC>::size), dot);
        }
        float sc = wave_sum_f32(dot) * a.scale;
        if (a.softcap > 0.0f) sc = a.softcap * tanhf(sc / a.softcap);
        const float m2 = fmaxf(m, sc);
        const float keep = expf(m - m2), p = expf(sc - m2);
        l = fmaf(l, keep, p);
#pragma unroll
        for (int i = 0; i < N; i++) {
            const uint32_t e = lane + 64 * i;
            if (e < a.D) o[i] = fmaf(p, Elt<TC>::load1(vr + e * Elt<TC>::size), o[i] * keep);
        }
        m = m2;
    }
    if (wrong && lane == 0) atomicOr(a.err, DEV_ERR_PAGE);
#pragma unroll
    for (int i = 0; i < N; i++) {
        const uint32_t e = lane + 64 * i;
        if (e < a.D) lds_o[wid][e] = o[i];
    }
    if (lane == 0) {
        lds_m[wid] = m;
        lds_l[wid] = l;
    }
    __syncthreads();
    float mm = kLowest, ll = 0.0f, f[W];
#pragma unroll
    for (int w = 0; w < W; w++) mm = fmaxf(mm, lds_m[w]);
#pragma unroll
    for (int w = 0; w < W; w++) {
        f[w] = expf(lds_m[w] - mm);
        ll = fmaf(lds_l[w], f[w], ll);
    }
    char* yr = a.y + s * a.y_nb2 + h * a.y_nb1;
    for (uint32_t e = threadIdx.x; e < a.D; e += kAttnThreads) {
        float t = 0.0f;
#pragma unroll
        for (int w = 0; w < W; w++) t = fmaf(lds_o[w][e], f[w], t);
        Elt<T>::store1(yr + e * Elt<T>::size, ll == 0.0f ? 0.0f : t / ll);
    }
}

}  // namespace

size_t paged_attention_workspace(const cbx_tensor* q, const cbx_tensor* k, const cbx_tensor* tables, const DeviceState* st) {
    (void)q; (void)k; (void)tables; (void)st;
    return 0;
}

int launch_paged_attention(const PagedAttnCall& c, DeviceState* st, hipStream_t s) {
    AttnArgs a{};
    a.q = static_cast<const char*>(c.q->data);
    a.k = static_cast<const char*>(c.k->data);
    a.v = static_cast<const char*>(c.v->data);
    a.tables = static_cast<const char*>(c.tables->data);
    a.lens = static_cast<const int32_t*>(c.lens->data);
    a.y = static_cast<char*>(c.y->data);
    a.q_nb1 = c.q->nb[1]; a.q_nb2 = c.q->nb[2];
    a.y_nb1 = c.y->nb[1]; a.y_nb2 = c.y->nb[2];
    a.k_nb1 = c.k->nb[1]; a.k_nb2 = c.k->nb[2]; a.k_nb3 = c.k->nb[3];
    a.v_nb1 = c.v->nb[1]; a.v_nb2 = c.v->nb[2]; a.v_nb3 = c.v->nb[3];
    a.t_nb1 = c.tables->nb[1];
    a.n_seq = static_cast<uint32_t>(c.q->ne[2]);
    a.hq = static_cast<uint32_t>(c.q->ne[1]);
    a.hkv = static_cast<uint32_t>(c.k->ne[2]);
    a.g = a.hq / a.hkv;
    a.D = static_cast<uint32_t>(c.q->ne[0]);
    a.page = static_cast<uint32_t>(c.k->ne[1]);
    a.max_pages = static_cast<uint32_t>(c.tables->ne[0]);
    a.n_pages = static_cast<uint32_t>(c.k->ne[3]);
    a.window = c.window;
    a.scale = c.scale;
    a.softcap = c.softcap;
    a.err = st->err_word;
    const dim3 grid(static_cast<unsigned>(c.q->ne[1] * c.q->ne[2])), block(kAttnThreads);
    const bool t16 = c.q->type == CBX_TYPE_F16, c16 = c.k->type == CBX_TYPE_F16;
    if (t16 && c16) hipLaunchKernelGGL((k_attn_rows<uint16_t, uint16_t>), grid, block, 0, s, a);
    else if (t16) hipLaunchKernelGGL((k_attn_rows<uint16_t, float>), grid, block, 0, s, a);
    else if (c16) hipLaunchKernelGGL((k_attn_rows<float, uint16_t>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((k_attn_rows<float, float>), grid, block, 0, s, a);
    return check_launch("cbx_paged_attention");
}

}  // namespace cbx
