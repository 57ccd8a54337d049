// k_qk.hip -- RMS norm of query and key heads with the rotation in the same
// pass, keys and values rounded into their cache pages on the way.
//
// A head row of D elements: y = rope(x * (1 / sqrt(mean(x^2) + eps)) * g), the
// arithmetic of cbx_rms_norm_mul (f32 squares summed in f64, one rounding a
// product) and of cbx_rope_ext (cos and sin from the position's table row,
// or the same recurrence on the device past the table), the value between
// the two kept in f32.
//
// Bound by the rows read and written once.  k_qk_heads: a workgroup a token, 8
// elements a lane: those of four pairs and no partner in another lane, so that
// only the norm's sum crosses lanes (8 of them a head of 64).  The token's
// cos and sin of those pairs are read once and serve all its heads: in F16
// they are twice the bytes of a row.  9001 tokens of 24 + 8 heads of 128, F32 into
// F16 pages, 64.2 us (328 MB, 5.1 TB/s; 62.0 without the profiler; k_qk, with q
// off the alignment, 229), 64 tokens of 16 + 16 heads of 64 in F16 4.1 us.  k_qk:
// a wave a head row, for sizes and alignments that the vectors do not take.
#include "cbx_rowops.h"

namespace cbx {
namespace {

constexpr int kQkThreads = 256;
constexpr int kQkMax = 512;   // elements of a head

struct QkArgs {
    const char *q, *k, *v;
    const float *gq, *gk;
    const int32_t *pos, *slots;
    char *yq, *yk, *kc, *vc;          // yk, or kc and vc with slots
    const float2* table;
    const float* ff;
    int64_t q_nb1, q_nb2, k_nb1, k_nb2, v_nb1, v_nb2, yq_nb1, yq_nb2, yk_nb1, yk_nb2;
    int64_t kc_nb1, kc_nb2, kc_nb3, vc_nb1, vc_nb2, vc_nb3;
    uint32_t hq, hkv, heads, rows, D;   // heads: hq + hkv (+ hkv value rows)
    uint32_t page, n_slot;              // page size, slots of the cache
    int32_t n_pos;
    float eps;
    int32_t norm;
    uint32_t nth;                       // k_qk_heads: its block size
    RopeParams rp;
    uint32_t* err;
};

template <typename T, typename TC>
__global__ __launch_bounds__(kQkThreads) void k_qk(QkArgs a) {
    __shared__ float rows[kQkThreads / 64][kQkMax];
    const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
    const uint32_t row = blockIdx.x * (kQkThreads / 64) + wid;
    float* r = rows[wid];
    const bool live = row < a.rows;
    const uint32_t tok = live ? row / a.heads : 0, h = live ? row - tok * a.heads : 0;
    const int kind = h < a.hq ? 0 : (h < a.hq + a.hkv ? 1 : 2);   // q, k, v
    const uint32_t hh = h - (kind == 0 ? 0 : (kind == 1 ? a.hq : a.hq + a.hkv));
    const char* x = kind == 0 ? a.q + tok * a.q_nb2 + hh * a.q_nb1
                  : kind == 1 ? a.k + tok * a.k_nb2 + hh * a.k_nb1 : a.v + tok * a.v_nb2 + hh * a.v_nb1;
    const uint32_t D = a.D;
    constexpr int N = kQkMax / 64;
    float v[N];
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < N; i++) {
        const uint32_t e = lane + 64 * i;
        v[i] = live && e < D ? Elt<T>::load1(x + e * Elt<T>::size) : 0.0f;
        sum += static_cast<double>(v[i] * v[i]);
    }
    if (a.norm) {
        const float ms = static_cast<float>(wave_sum(sum) / static_cast<double>(D));
        const float sc = 1.0f / sqrtf(ms + a.eps);
        const float* g = kind == 0 ? a.gq : a.gk;
#pragma unroll
        for (int i = 0; i < N; i++) {
            const uint32_t e = lane + 64 * i;
            float y = kind == 2 ? v[i] : v[i] * sc;
            if (kind != 2 && g && e < D) y = y * g[e];
            if (e < D) r[e] = y;
        }
        __syncthreads();
        if (kind != 2) {
            const int32_t p = live ? a.pos[tok] : 0;
            const uint32_t nd = static_cast<uint32_t>(a.rp.n_dims), half = nd / 2;
            const bool in_tab = p >= 0 && p < a.n_pos;
#pragma unroll
            for (int i = 0; i < N; i++) {
                const uint32_t e = lane + 64 * i;
                if (e >= D) continue;
                v[i] = r[e];
                if (e >= nd) continue;
                const bool second = a.rp.mode == 2 ? e >= half : (e & 1);
                const uint32_t pair = a.rp.mode == 2 ? (second ? e - half : e) : e >> 1;
                const float other = r[a.rp.mode == 2 ? (second ? e - half : e + half) : e ^ 1];
                float2 c;
                if (in_tab) c = a.table[static_cast<int64_t>(p) * half + pair];
                else rope_cos_sin_dev(p, static_cast<int>(pair), a.rp, a.ff, &c.x, &c.y);
                v[i] = second ? other * c.y + v[i] * c.x : v[i] * c.x - other * c.y;
            }
        }
    }
    if (!live) return;
    if (kind == 0 || (kind == 1 && !a.slots)) {
        char* y = kind == 0 ? a.yq + tok * a.yq_nb2 + hh * a.yq_nb1 : a.yk + tok * a.yk_nb2 + hh * a.yk_nb1;
#pragma unroll
        for (int i = 0; i < N; i++) {
            const uint32_t e = lane + 64 * i;
            if (e < D) Elt<T>::store1(y + e * Elt<T>::size, v[i]);
        }
        return;
    }
    const int32_t slot = a.slots[tok];
    if (slot < 0) return;
    if (static_cast<uint32_t>(slot) >= a.n_slot) {
        if (lane == 0) atomicOr(a.err, DEV_ERR_PAGE);
        return;
    }
    const uint32_t pg = static_cast<uint32_t>(slot) / a.page, at = static_cast<uint32_t>(slot) - pg * a.page;
    char* y = kind == 1 ? a.kc + pg * a.kc_nb3 + hh * a.kc_nb2 + at * a.kc_nb1
                        : a.vc + pg * a.vc_nb3 + hh * a.vc_nb2 + at * a.vc_nb1;
#pragma unroll
    for (int i = 0; i < N; i++) {
        const uint32_t e = lane + 64 * i;
        if (e < D) Elt<TC>::store1(y + e * Elt<TC>::size, v[i]);
    }
}

// Sum over the LPR lanes that share a head (a power of two, aligned), the
// same in each.
template <int LPR> __device__ __forceinline__ double head_sum(double v) {
    v += dpp_f64<0xB1>(v);
    v += dpp_f64<0x4E>(v);
    v += dpp_f64<0x141>(v);
    if constexpr (LPR >= 16) v += dpp_f64<0x140>(v);
    if constexpr (LPR >= 32) v += __shfl_xor(v, 16);
    if constexpr (LPR >= 64) v += __shfl_xor(v, 32);
    return v;
}

constexpr int kQkRows = 4;   // rows whose loads a lane issues together

// LPR lanes a head (8 elements each, those past D idle), blockDim.x / LPR heads
// at a time.
template <typename T, typename TC, int LPR>
__global__ __launch_bounds__(kQkThreads) void k_qk_heads(QkArgs a) {
    constexpr int es = Elt<T>::size;
    const uint32_t tok = blockIdx.x, li = threadIdx.x % LPR, ng = a.nth / LPR;
    const uint32_t nd = static_cast<uint32_t>(a.rp.n_dims), half = nd / 2;
    const bool in = 8 * li < a.D, turned = a.norm && 8 * li < nd;
    // the lane's two runs of four elements
    const bool apart = turned && a.rp.mode == 2;
    const uint32_t ia = !in ? 0 : (apart ? 4 * li : 8 * li), ib = !in ? 0 : (apart ? 4 * li + half : 8 * li + 4);
    float2 c[4];
    if (turned) {
        const int32_t p = a.pos[tok];
        if (p >= 0 && p < a.n_pos) {
            const float4* t = reinterpret_cast<const float4*>(a.table + static_cast<int64_t>(p) * half + 4 * li);
            const float4 t0 = t[0], t1 = t[1];
            c[0] = make_float2(t0.x, t0.y);
            c[1] = make_float2(t0.z, t0.w);
            c[2] = make_float2(t1.x, t1.y);
            c[3] = make_float2(t1.z, t1.w);
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++) rope_cos_sin_dev(p, static_cast<int>(4 * li) + e, a.rp, a.ff, &c[e].x, &c[e].y);
        }
    } else {
#pragma unroll
        for (int e = 0; e < 4; e++) c[e] = make_float2(1.0f, 0.0f);
    }
    int32_t slot = -1;
    uint32_t pg = 0, at = 0;
    if (a.slots) {
        slot = a.slots[tok];
        if (slot >= 0 && static_cast<uint32_t>(slot) >= a.n_slot) {
            if (threadIdx.x == 0) atomicOr(a.err, DEV_ERR_PAGE);
            slot = -1;
        }
        if (slot >= 0) {
            pg = static_cast<uint32_t>(slot) / a.page;
            at = static_cast<uint32_t>(slot) - pg * a.page;
        }
    }
    // rows that are written: without a slot the query heads alone
    const uint32_t heads = a.slots && slot < 0 ? a.hq : a.heads;
    auto kind_of = [&](uint32_t h) { return h < a.hq ? 0 : (h < a.hq + a.hkv ? 1 : 2); };
    for (uint32_t h0 = threadIdx.x / LPR; h0 < heads; h0 += ng * kQkRows) {
        float4 xa[kQkRows], xb[kQkRows];
#pragma unroll
        for (int u = 0; u < kQkRows; u++) {
            const uint32_t h = h0 + u * ng < heads ? h0 + u * ng : h0;
            const int kind = kind_of(h);
            const char* x = kind == 0 ? a.q + tok * a.q_nb2 + h * a.q_nb1
                          : kind == 1 ? a.k + tok * a.k_nb2 + (h - a.hq) * a.k_nb1
                                      : a.v + tok * a.v_nb2 + (h - a.hq - a.hkv) * a.v_nb1;
            xa[u] = Elt<T>::load4(x + ia * es);
            xb[u] = Elt<T>::load4(x + ib * es);
        }
#pragma unroll
        for (int u = 0; u < kQkRows; u++) {
            const uint32_t h = h0 + u * ng;
            if (h >= heads) break;
            const int kind = kind_of(h);
            if (a.norm) {
                double sum = 0.0;
#pragma unroll
                for (int e = 0; e < 4; e++) sum += static_cast<double>(get(xa[u], e) * get(xa[u], e));
#pragma unroll
                for (int e = 0; e < 4; e++) sum += static_cast<double>(get(xb[u], e) * get(xb[u], e));
                const float ms = static_cast<float>(head_sum<LPR>(in ? sum : 0.0) / static_cast<double>(a.D));
                const float sc = 1.0f / sqrtf(ms + a.eps);
                if (kind != 2) {
                    const float* g = kind == 0 ? a.gq : a.gk;
                    float4 ga = make_float4(1.0f, 1.0f, 1.0f, 1.0f), gb = ga;
                    if (g) {
                        ga = *reinterpret_cast<const float4*>(g + ia);
                        gb = *reinterpret_cast<const float4*>(g + ib);
                    }
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        set(xa[u], e, (get(xa[u], e) * sc) * get(ga, e));
                        set(xb[u], e, (get(xb[u], e) * sc) * get(gb, e));
                    }
                    if (turned) {
                        const float4 ya = xa[u], yb = xb[u];
                        if (a.rp.mode == 2) {
#pragma unroll
                            for (int e = 0; e < 4; e++) {
                                set(xa[u], e, get(ya, e) * c[e].x - get(yb, e) * c[e].y);
                                set(xb[u], e, get(ya, e) * c[e].y + get(yb, e) * c[e].x);
                            }
                        } else {
                            xa[u] = make_float4(ya.x * c[0].x - ya.y * c[0].y, ya.x * c[0].y + ya.y * c[0].x,
                                                ya.z * c[1].x - ya.w * c[1].y, ya.z * c[1].y + ya.w * c[1].x);
                            xb[u] = make_float4(yb.x * c[2].x - yb.y * c[2].y, yb.x * c[2].y + yb.y * c[2].x,
                                                yb.z * c[3].x - yb.w * c[3].y, yb.z * c[3].y + yb.w * c[3].x);
                        }
                    }
                }
            }
            if (!in) continue;
            if (kind == 0 || !a.slots) {
                char* y = kind == 0 ? a.yq + tok * a.yq_nb2 + h * a.yq_nb1 : a.yk + tok * a.yk_nb2 + (h - a.hq) * a.yk_nb1;
                Elt<T>::store4(y + ia * es, xa[u]);
                Elt<T>::store4(y + ib * es, xb[u]);
            } else {
                const uint32_t hh = h - a.hq - (kind == 2 ? a.hkv : 0);
                char* y = kind == 1 ? a.kc + pg * a.kc_nb3 + hh * a.kc_nb2 + at * a.kc_nb1
                                    : a.vc + pg * a.vc_nb3 + hh * a.vc_nb2 + at * a.vc_nb1;
                Elt<TC>::store4(y + ia * Elt<TC>::size, xa[u]);
                Elt<TC>::store4(y + ib * Elt<TC>::size, xb[u]);
            }
        }
    }
}

int64_t nb(const cbx_tensor* t, int i) { return t ? static_cast<int64_t>(t->nb[i]) : 0; }

// Rows at steps that 4-element loads and stores take.
bool quads(const cbx_tensor* t) {
    if (!t) return true;
    const size_t al = 4 * type_size(t->type);
    if (reinterpret_cast<uintptr_t>(t->data) % al) return false;
    for (int i = 1; i < 4; i++) if (t->ne[i] > 1 && t->nb[i] % al) return false;
    return true;
}

template <typename T, typename TC>
void launch_heads(QkArgs& a, uint32_t tok, hipStream_t s) {
    const uint32_t lpr = a.D <= 64 ? 8 : a.D <= 128 ? 16 : a.D <= 256 ? 32 : 64;
    // as many waves as the token's heads fill, 4 at most
    a.nth = static_cast<uint32_t>(std::min<int64_t>(kQkThreads, cdiv(static_cast<int64_t>(a.heads) * lpr, 64) * 64));
    const dim3 grid(tok), block(a.nth);
    if (lpr == 8) hipLaunchKernelGGL((k_qk_heads<T, TC, 8>), grid, block, 0, s, a);
    else if (lpr == 16) hipLaunchKernelGGL((k_qk_heads<T, TC, 16>), grid, block, 0, s, a);
    else if (lpr == 32) hipLaunchKernelGGL((k_qk_heads<T, TC, 32>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((k_qk_heads<T, TC, 64>), grid, block, 0, s, a);
}

}  // namespace

int launch_qk(const QkCall& c, DeviceState* st, hipStream_t s) {
    const cbx_tensor* k = c.k;
    QkArgs a{};
    auto in = [](const cbx_tensor* t) { return t ? static_cast<const char*>(t->data) : nullptr; };
    auto out = [](cbx_tensor* t) { return t ? static_cast<char*>(t->data) : nullptr; };
    a.q = in(c.q);
    a.k = in(k);
    a.v = in(c.v);
    a.gq = reinterpret_cast<const float*>(in(c.gq));
    a.gk = reinterpret_cast<const float*>(in(c.gk));
    a.pos = reinterpret_cast<const int32_t*>(in(c.pos));
    a.slots = reinterpret_cast<const int32_t*>(in(c.slots));
    a.yq = out(c.yq);
    a.yk = out(c.yk);
    a.kc = out(c.k_cache);
    a.vc = out(c.v_cache);
    a.table = c.rope.table;
    a.ff = c.rope.ff;
    a.n_pos = c.rope.n_pos;
    a.rp = c.rope.p;
    a.q_nb1 = nb(c.q, 1); a.q_nb2 = nb(c.q, 2);
    a.k_nb1 = nb(k, 1); a.k_nb2 = nb(k, 2);
    a.v_nb1 = nb(c.v, 1); a.v_nb2 = nb(c.v, 2);
    a.yq_nb1 = nb(c.yq, 1); a.yq_nb2 = nb(c.yq, 2);
    a.yk_nb1 = nb(c.yk, 1); a.yk_nb2 = nb(c.yk, 2);
    a.kc_nb1 = nb(c.k_cache, 1); a.kc_nb2 = nb(c.k_cache, 2); a.kc_nb3 = nb(c.k_cache, 3);
    a.vc_nb1 = nb(c.v_cache, 1); a.vc_nb2 = nb(c.v_cache, 2); a.vc_nb3 = nb(c.v_cache, 3);
    a.hq = c.q ? static_cast<uint32_t>(c.q->ne[1]) : 0;
    a.hkv = static_cast<uint32_t>(k->ne[1]);
    a.heads = a.hq + a.hkv * (c.v ? 2 : 1);
    const int64_t rows = k->ne[2] * a.heads;
    a.rows = static_cast<uint32_t>(rows);
    a.D = static_cast<uint32_t>(k->ne[0]);
    a.page = c.k_cache ? static_cast<uint32_t>(c.k_cache->ne[1]) : 1;
    a.n_slot = c.k_cache ? static_cast<uint32_t>(c.k_cache->ne[1] * c.k_cache->ne[3]) : 0;
    a.eps = c.eps;
    a.norm = c.norm;
    a.err = st->err_word;
    if (rows == 0 || a.D == 0) return CBX_OK;
    const bool vec = a.D % 8 == 0 && quads(c.q) && quads(k) && quads(c.v) && quads(c.yq) && quads(c.yk) && quads(c.k_cache) &&
                     quads(c.v_cache) && quads(c.gq) && quads(c.gk) && reinterpret_cast<uintptr_t>(a.table) % 16 == 0;
    const dim3 grid(static_cast<unsigned>(cdiv(rows, kQkThreads / 64))), block(kQkThreads);
    const bool t16 = k->type == CBX_TYPE_F16, c16 = c.k_cache ? c.k_cache->type == CBX_TYPE_F16 : t16;
    if (vec) {
        const uint32_t tok = static_cast<uint32_t>(k->ne[2]);
        if (t16 && c16) launch_heads<uint16_t, uint16_t>(a, tok, s);
        else if (t16) launch_heads<uint16_t, float>(a, tok, s);
        else if (c16) launch_heads<float, uint16_t>(a, tok, s);
        else launch_heads<float, float>(a, tok, s);
        return check_launch("cbx_qk_norm_rope");
    }
    if (grid.x >= 1u << 24) {     // a launch's threads below 2^32
        return set_error(CBX_ERR_UNSUPPORTED, "cbx_qk_norm_rope: 2^26 rows or more, at sizes or alignments that vectors do not take");
    }
    if (t16 && c16) hipLaunchKernelGGL((k_qk<uint16_t, uint16_t>), grid, block, 0, s, a);
    else if (t16) hipLaunchKernelGGL((k_qk<uint16_t, float>), grid, block, 0, s, a);
    else if (c16) hipLaunchKernelGGL((k_qk<float, uint16_t>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((k_qk<float, float>), grid, block, 0, s, a);
    return check_launch("cbx_qk_norm_rope");
}

}  // namespace cbx
