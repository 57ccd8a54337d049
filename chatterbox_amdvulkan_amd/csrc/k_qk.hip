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
//
// Into I8 pages (Q8Row): the row's largest element over its lanes, then 8
// elements a lane rounded to whole numbers of steps.  Rows that are neither
// normed nor turned go through k_store8.
//
// k_load reads slots back: a workgroup a token, 8 elements of a key or value a
// thread; bound by the bytes (9001 tokens of 8 + 8 heads of 128, I8 to F16, 11.8
// to 12.8 us: 56 MB, 4.4 to 4.7 TB/s; 64 tokens of 16 + 16 heads of 64 3.3 us).
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
    char *ks, *vs;                      // I8 pages: their rows' scales
    int64_t ks_nb0, ks_nb1, ks_nb2, vs_nb0, vs_nb1, vs_nb2;
    uint32_t hq, hkv, heads, rows, D;   // heads: hq + hkv (+ hkv value rows)
    uint32_t page, n_slot;              // page size, slots of the cache
    int32_t n_pos;
    float eps;
    int32_t norm;
    uint32_t nth;                       // k_qk_heads: its block size
    RopeParams rp;
    uint32_t* err;
};

// |x| as a number that compares as |x| does, infinities and NaN above all.
__device__ __forceinline__ uint32_t size_of(float x) { return __builtin_bit_cast(uint32_t, x) & 0x7fffffffu; }

// A row in 8 bits: scale = top / 127, n = 127 x / top to the nearest whole
// number, ties to the even one, top its largest |x| (127 * 2^-126 at least, so
// that the scale is a normal number).  In f32, 127 times the reciprocal and the
// product are 2^-22 of |n| <= 127 off, 2^-15 at most: a result t further than
// that from the middle of two whole numbers is right.  The others, one in 8000,
// lie above or below the middle as 254 x lies to (2 floor(t) + 1) top, both
// exact in f64.  Rows near the ends of f32's range are moved by 2^60 first
// (exact but for elements that are 0 all the same).
struct Q8Row {
    float top, mul, scale, lift;
    bool bad;             // an infinity or NaN among them
    __device__ __forceinline__ explicit Q8Row(uint32_t largest) {
        bad = largest >= 0x7f800000u;
        top = fmaxf(bad ? 0.0f : __builtin_bit_cast(float, largest), 127 * 0x1p-126f);
        scale = bad ? NAN : top / 127.0f;
        lift = top < 0x1p-60f ? 0x1p60f : top > 0x1p60f ? 0x1p-60f : 1.0f;
        top *= lift;
        mul = 127.0f * __builtin_amdgcn_rcpf(top) * lift;
    }
    // Four of the row's elements as bytes: a sum with 1.5 * 2^23 has the whole
    // number in its last bits.  off: the furthest of all from a whole number.
    __device__ __forceinline__ uint32_t quick(const float4& x, float* off) const {
        uint32_t b[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float t = get(x, i) * mul, s = t + 0x1.8p23f;
            *off = fmaxf(*off, fabsf(t - (s - 0x1.8p23f)));
            b[i] = __builtin_bit_cast(uint32_t, s);
        }
        return __builtin_amdgcn_perm(__builtin_amdgcn_perm(b[3], b[2], 0x0c0c0400u), __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400u), 0x05040100u);
    }
    static constexpr float kUnsure = 0.5f - 0x1p-14f;
    __device__ __forceinline__ uint32_t sure(const float4& x) const {
        uint32_t r = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float t = get(x, i) * mul, f = floorf(t);
            const double d = 254.0 * static_cast<double>(get(x, i) * lift) - static_cast<double>(2.0f * f + 1.0f) * static_cast<double>(top);
            const int32_t low = static_cast<int32_t>(f);
            int32_t n = static_cast<int32_t>(rintf(t));
            if (fabsf(t - rintf(t)) > kUnsure) n = d > 0.0 ? low + 1 : d < 0.0 ? low : low + (low & 1);
            r |= (static_cast<uint32_t>(n) & 0xffu) << 8 * i;
        }
        return r;
    }
    // The lane's eight elements.
    __device__ __forceinline__ uint2 of(const float4& xa, const float4& xb) const {
        float off = 0.0f;
        uint32_t a = quick(xa, &off), b = quick(xb, &off);
        if (__builtin_expect(off > kUnsure, 0)) {
            a = sure(xa);
            b = sure(xb);
        }
        return bad ? make_uint2(0, 0) : make_uint2(a, b);
    }
};

// The scale of a key (kind 1) or value.
__device__ __forceinline__ void store_scale(const QkArgs& a, int kind, uint32_t pg, uint32_t h, uint32_t at, float scale) {
    char* p = kind == 1 ? a.ks + pg * a.ks_nb2 + h * a.ks_nb1 + at * a.ks_nb0 : a.vs + pg * a.vs_nb2 + h * a.vs_nb1 + at * a.vs_nb0;
    *reinterpret_cast<float*>(p) = scale;
}

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
    if constexpr (sizeof(TC) == 1) {
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < N; i++) top = max(top, static_cast<uint32_t>(lane + 64 * i) < D ? size_of(v[i]) : 0u);
        for (int d = 32; d > 0; d >>= 1) top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), d)));
        const Q8Row row(top);
        static_assert(N == 8);
        const uint2 w = row.of(make_float4(v[0], v[1], v[2], v[3]), make_float4(v[4], v[5], v[6], v[7]));
#pragma unroll
        for (int i = 0; i < N; i++) {
            const uint32_t e = lane + 64 * i;
            if (e < D) y[e] = static_cast<char>((i < 4 ? w.x : w.y) >> 8 * (i % 4));
        }
        if (lane == 0) store_scale(a, kind, pg, hh, at, row.scale);
        return;
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) {
            const uint32_t e = lane + 64 * i;
            if (e < D) Elt<TC>::store1(y + e * Elt<TC>::size, v[i]);
        }
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

// Largest over them.
template <int CTRL> __device__ __forceinline__ uint32_t dpp_max(uint32_t v) {
    return max(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, 0xf, 0xf, true)));
}
template <int LPR> __device__ __forceinline__ uint32_t head_max(uint32_t v) {
    v = dpp_max<0xB1>(v);
    v = dpp_max<0x4E>(v);
    v = dpp_max<0x141>(v);
    if constexpr (LPR >= 16) v = dpp_max<0x140>(v);
    if constexpr (LPR >= 32) v = max(v, static_cast<uint32_t>(__shfl_xor(static_cast<int>(v), 16)));
    if constexpr (LPR >= 64) v = max(v, static_cast<uint32_t>(__shfl_xor(static_cast<int>(v), 32)));
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
            uint32_t top = 0;
            if constexpr (sizeof(TC) == 1) {
#pragma unroll
                for (int e = 0; e < 4; e++) top = max(top, max(size_of(get(xa[u], e)), size_of(get(xb[u], e))));
                top = head_max<LPR>(in ? top : 0);
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
                if constexpr (sizeof(TC) == 1) {
                    const Q8Row row(top);
                    const uint2 w = row.of(xa[u], xb[u]);
                    *reinterpret_cast<uint32_t*>(y + ia) = w.x;
                    *reinterpret_cast<uint32_t*>(y + ib) = w.y;
                    if (li == 0) store_scale(a, kind, pg, hh, at, row.scale);
                } else {
                    Elt<TC>::store4(y + ia * Elt<TC>::size, xa[u]);
                    Elt<TC>::store4(y + ib * Elt<TC>::size, xb[u]);
                }
            }
        }
    }
}

// Rows as they are into I8 pages: a workgroup a token, LPR lanes a row of 8
// elements each.  Half of what a row costs here is instructions, not bytes, and
// k_qk_heads has twice as many: 9001 tokens of 8 + 8 heads of 128 in F16 14.0
// us at the least (56 MB, 4.0 TB/s) for its 21.0.  F16 and F32 pages are at the copy's rate there.
template <typename T, int LPR>
__global__ __launch_bounds__(kQkThreads) void k_store8(QkArgs a) {
    typedef uint32_t u2w __attribute__((ext_vector_type(2), aligned(4)));
    const uint32_t tok = blockIdx.x, li = threadIdx.x % LPR;
    const int32_t slot = a.slots[tok];
    if (slot < 0) return;
    if (static_cast<uint32_t>(slot) >= a.n_slot) {
        if (threadIdx.x == 0) atomicOr(a.err, DEV_ERR_PAGE);
        return;
    }
    const uint32_t pg = static_cast<uint32_t>(slot) / a.page, at = static_cast<uint32_t>(slot) - pg * a.page;
    const char *k = a.k + tok * a.k_nb2, *v = a.v + tok * a.v_nb2;
    char *kc = a.kc + pg * a.kc_nb3 + at * a.kc_nb1, *vc = a.vc + pg * a.vc_nb3 + at * a.vc_nb1;
    char *ks = a.ks + pg * a.ks_nb2 + at * a.ks_nb0, *vs = a.vs + pg * a.vs_nb2 + at * a.vs_nb0;
    const bool in = 8 * li < a.D;
    for (uint32_t r = threadIdx.x / LPR; r < 2 * a.hkv; r += a.nth / LPR) {
        const bool val = r >= a.hkv;
        const uint32_t h = val ? r - a.hkv : r;
        const char* x = (val ? v + h * a.v_nb1 : k + h * a.k_nb1) + (in ? 8 * li : 0) * Elt<T>::size;
        const float4 xa = Elt<T>::load4(x), xb = Elt<T>::load4(x + 4 * Elt<T>::size);
        uint32_t top = 0;
#pragma unroll
        for (int e = 0; e < 4; e++) top = max(top, max(size_of(get(xa, e)), size_of(get(xb, e))));
        const Q8Row row(head_max<LPR>(in ? top : 0));
        const uint2 w = row.of(xa, xb);
        if (in) *reinterpret_cast<u2w*>((val ? vc + h * a.vc_nb2 : kc + h * a.kc_nb2) + 8 * li) = u2w{w.x, w.y};
        if (li == 0) *reinterpret_cast<float*>(val ? vs + h * a.vs_nb1 : ks + h * a.ks_nb1) = row.scale;
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
    if constexpr (sizeof(TC) == 1) {
        if (!a.norm) {
            if (lpr == 8) hipLaunchKernelGGL((k_store8<T, 8>), grid, block, 0, s, a);
            else if (lpr == 16) hipLaunchKernelGGL((k_store8<T, 16>), grid, block, 0, s, a);
            else if (lpr == 32) hipLaunchKernelGGL((k_store8<T, 32>), grid, block, 0, s, a);
            else hipLaunchKernelGGL((k_store8<T, 64>), grid, block, 0, s, a);
            return;
        }
    }
    if (lpr == 8) hipLaunchKernelGGL((k_qk_heads<T, TC, 8>), grid, block, 0, s, a);
    else if (lpr == 16) hipLaunchKernelGGL((k_qk_heads<T, TC, 16>), grid, block, 0, s, a);
    else if (lpr == 32) hipLaunchKernelGGL((k_qk_heads<T, TC, 32>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((k_qk_heads<T, TC, 64>), grid, block, 0, s, a);
}

struct LoadArgs {
    const char *kc, *vc, *ks, *vs;
    const int32_t* slots;
    char *k, *v;
    int64_t k_nb1, k_nb2, v_nb1, v_nb2, kc_nb1, kc_nb2, kc_nb3, vc_nb1, vc_nb2, vc_nb3;
    int64_t ks_nb0, ks_nb1, ks_nb2, vs_nb0, vs_nb1, vs_nb2;
    uint32_t hkv, D, cpr, page, n_slot;   // cpr: runs of VEC elements a row
    uint32_t* err;
};

template <typename TC, int VEC> __device__ __forceinline__ void load_row(const char* p, float (&x)[VEC]) {
    if constexpr (VEC == 1) {
        if constexpr (sizeof(TC) == 1) x[0] = static_cast<float>(*reinterpret_cast<const int8_t*>(p));
        else x[0] = Elt<TC>::load1(p);
    } else if constexpr (sizeof(TC) == 1) {
        const uint2 t = *reinterpret_cast<const uint2*>(p);
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = static_cast<float>(static_cast<int8_t>((i < 4 ? t.x : t.y) >> 8 * (i & 3)));
    } else {
#pragma unroll
        for (int i = 0; i < 8; i += 4) {
            const float4 t = Elt<TC>::load4(p + i * Elt<TC>::size);
#pragma unroll
            for (int j = 0; j < 4; j++) x[i + j] = get(t, j);
        }
    }
}

template <typename T, typename TC, int VEC>
__global__ __launch_bounds__(kQkThreads) void k_load(LoadArgs a) {
    const uint32_t tok = blockIdx.x;
    int32_t slot = a.slots[tok];
    if (slot >= 0 && static_cast<uint32_t>(slot) >= a.n_slot) {
        if (threadIdx.x == 0) atomicOr(a.err, DEV_ERR_PAGE);
        slot = -1;
    }
    const uint32_t pg = slot < 0 ? 0 : static_cast<uint32_t>(slot) / a.page, at = slot < 0 ? 0 : static_cast<uint32_t>(slot) - pg * a.page;
    const uint32_t runs = a.hkv * a.cpr;
    for (uint32_t i = threadIdx.x; i < 2 * runs; i += blockDim.x) {
        const bool val = i >= runs;
        const uint32_t j = val ? i - runs : i, h = j / a.cpr, e = (j - h * a.cpr) * VEC;
        float x[VEC] = {};
        if (slot >= 0) {
            const char* p = val ? a.vc + pg * a.vc_nb3 + h * a.vc_nb2 + at * a.vc_nb1 : a.kc + pg * a.kc_nb3 + h * a.kc_nb2 + at * a.kc_nb1;
            load_row<TC, VEC>(p + e * sizeof(TC), x);
            if constexpr (sizeof(TC) == 1) {
                const char* sp = val ? a.vs + pg * a.vs_nb2 + h * a.vs_nb1 + at * a.vs_nb0
                                     : a.ks + pg * a.ks_nb2 + h * a.ks_nb1 + at * a.ks_nb0;
                const float sc = *reinterpret_cast<const float*>(sp);
#pragma unroll
                for (int u = 0; u < VEC; u++) x[u] *= sc;
            }
        }
        char* y = val ? a.v + tok * a.v_nb2 + h * a.v_nb1 : a.k + tok * a.k_nb2 + h * a.k_nb1;
        if constexpr (VEC == 1) {
            Elt<T>::store1(y + e * Elt<T>::size, x[0]);
        } else {
            Elt<T>::store4(y + e * Elt<T>::size, make_float4(x[0], x[1], x[2], x[3]));
            Elt<T>::store4(y + (e + 4) * Elt<T>::size, make_float4(x[4], x[5], x[6], x[7]));
        }
    }
}

// Rows of a cache at steps that k_load's reads of 8 elements take.
bool eights(const cbx_tensor* t) {
    const size_t al = t->type == CBX_TYPE_F32 ? 16 : 8;
    if (reinterpret_cast<uintptr_t>(t->data) % al) return false;
    for (int i = 1; i < 4; i++) if (t->ne[i] > 1 && t->nb[i] % al) return false;
    return true;
}

template <typename T, typename TC>
void launch_load(const LoadArgs& a, bool vec, uint32_t tok, hipStream_t s) {
    const int64_t runs = 2 * static_cast<int64_t>(a.hkv) * a.cpr;
    const dim3 block(static_cast<unsigned>(std::min<int64_t>(kQkThreads, cdiv(runs, 64) * 64)));
    if (vec) hipLaunchKernelGGL((k_load<T, TC, 8>), dim3(tok), block, 0, s, a);
    else hipLaunchKernelGGL((k_load<T, TC, 1>), dim3(tok), block, 0, s, a);
}

}  // namespace

int launch_paged_load(const LoadCall& c, DeviceState* st, hipStream_t s) {
    LoadArgs a{};
    auto in = [](const cbx_tensor* t) { return t ? static_cast<const char*>(t->data) : nullptr; };
    a.kc = in(c.k_cache);
    a.vc = in(c.v_cache);
    a.ks = in(c.k_scale);
    a.vs = in(c.v_scale);
    a.slots = reinterpret_cast<const int32_t*>(in(c.slots));
    a.k = static_cast<char*>(c.k->data);
    a.v = static_cast<char*>(c.v->data);
    a.k_nb1 = nb(c.k, 1); a.k_nb2 = nb(c.k, 2);
    a.v_nb1 = nb(c.v, 1); a.v_nb2 = nb(c.v, 2);
    a.kc_nb1 = nb(c.k_cache, 1); a.kc_nb2 = nb(c.k_cache, 2); a.kc_nb3 = nb(c.k_cache, 3);
    a.vc_nb1 = nb(c.v_cache, 1); a.vc_nb2 = nb(c.v_cache, 2); a.vc_nb3 = nb(c.v_cache, 3);
    a.ks_nb0 = nb(c.k_scale, 0); a.ks_nb1 = nb(c.k_scale, 1); a.ks_nb2 = nb(c.k_scale, 2);
    a.vs_nb0 = nb(c.v_scale, 0); a.vs_nb1 = nb(c.v_scale, 1); a.vs_nb2 = nb(c.v_scale, 2);
    a.hkv = static_cast<uint32_t>(c.k->ne[1]);
    a.D = static_cast<uint32_t>(c.k->ne[0]);
    a.page = static_cast<uint32_t>(c.k_cache->ne[1]);
    a.n_slot = static_cast<uint32_t>(c.k_cache->ne[1] * c.k_cache->ne[3]);
    a.err = st->err_word;
    const bool vec = a.D % 8 == 0 && quads(c.k) && quads(c.v) && eights(c.k_cache) && eights(c.v_cache);
    a.cpr = vec ? a.D / 8 : a.D;
    const uint32_t tok = static_cast<uint32_t>(c.k->ne[2]);
    const bool t16 = c.k->type == CBX_TYPE_F16;
    if (c.k_cache->type == CBX_TYPE_I8) {
        if (t16) launch_load<uint16_t, int8_t>(a, vec, tok, s);
        else launch_load<float, int8_t>(a, vec, tok, s);
    } else if (c.k_cache->type == CBX_TYPE_F16) {
        if (t16) launch_load<uint16_t, uint16_t>(a, vec, tok, s);
        else launch_load<float, uint16_t>(a, vec, tok, s);
    } else {
        if (t16) launch_load<uint16_t, float>(a, vec, tok, s);
        else launch_load<float, float>(a, vec, tok, s);
    }
    return check_launch("cbx_paged_load");
}

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
    a.ks = out(c.k_scale);
    a.vs = out(c.v_scale);
    a.ks_nb0 = nb(c.k_scale, 0); a.ks_nb1 = nb(c.k_scale, 1); a.ks_nb2 = nb(c.k_scale, 2);
    a.vs_nb0 = nb(c.v_scale, 0); a.vs_nb1 = nb(c.v_scale, 1); a.vs_nb2 = nb(c.v_scale, 2);
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
    const bool i8 = c.k_scale != nullptr;
    const bool t16 = k->type == CBX_TYPE_F16, c16 = c.k_cache ? c.k_cache->type == CBX_TYPE_F16 : t16;
    if (vec) {
        const uint32_t tok = static_cast<uint32_t>(k->ne[2]);
        if (i8 && t16) launch_heads<uint16_t, int8_t>(a, tok, s);
        else if (i8) launch_heads<float, int8_t>(a, tok, s);
        else if (t16 && c16) launch_heads<uint16_t, uint16_t>(a, tok, s);
        else if (t16) launch_heads<uint16_t, float>(a, tok, s);
        else if (c16) launch_heads<float, uint16_t>(a, tok, s);
        else launch_heads<float, float>(a, tok, s);
        return check_launch("cbx_qk_norm_rope");
    }
    if (grid.x >= 1u << 24) {     // a launch's threads below 2^32
        return set_error(CBX_ERR_UNSUPPORTED, "cbx_qk_norm_rope: 2^26 rows or more, at sizes or alignments that vectors do not take");
    }
    if (i8 && t16) hipLaunchKernelGGL((k_qk<uint16_t, int8_t>), grid, block, 0, s, a);
    else if (i8) hipLaunchKernelGGL((k_qk<float, int8_t>), grid, block, 0, s, a);
    else if (t16 && c16) hipLaunchKernelGGL((k_qk<uint16_t, uint16_t>), grid, block, 0, s, a);
    else if (t16) hipLaunchKernelGGL((k_qk<uint16_t, float>), grid, block, 0, s, a);
    else if (c16) hipLaunchKernelGGL((k_qk<float, uint16_t>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((k_qk<float, float>), grid, block, 0, s, a);
    return check_launch("cbx_qk_norm_rope");
}

}  // namespace cbx
