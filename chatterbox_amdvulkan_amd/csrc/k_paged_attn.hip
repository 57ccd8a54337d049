// k_paged_attn.hip -- attention of one new token a request over a paged cache.
//
// y = sum_i softmax(s)_i v_i with s_i = scale * q . k_i in one pass over the
// keys: with the running maximum m, l = sum exp(s_i - m) and o = sum
// exp(s_i - m) v_i, both rescaled by exp(m - m') when the maximum rises to m',
// and y = o / l at the end.  f32 throughout.
//
// Bound by the read of the keys and values, each of which the heads of a
// group share: the group's products run on the matrix cores (16 heads wide;
// a group of one fills a 16th of them, which is still several times what the
// reads feed), so that no group size pays for its arithmetic.
//
// k_attn_tiles: the requests' keys are cut into tiles of 4 waves x NK keys and
// all tiles of the call (request after request, key head after key head) are
// dealt to a fixed grid in equal runs, so that one long request or a thousand
// short ones fill the chip alike.  The lengths are on the device: every
// workgroup finds its run from a scan over them.  A key head whose tiles fall
// into one run is written to y; the parts of one that spans runs go to the
// workspace as (m, l, o) and k_attn_join adds them up in order.  8 requests of
// 1500 to 65000 keys, 32 heads over 8 of 128, F16: 191.9 + 4.8 us (1.09 GB, 5.5
// TB/s over both); 64 requests of 1 to 2048 keys, 16 heads of 64: 61.6 us (269 MB,
// 4.4 TB/s; 58.7 without the profiler); 16 heads over 300 keys 7.0 us, dependent
// reads (lengths, pages, keys and values).
//
// k_attn_rows: head sizes, strides and alignments that the tiles do not take,
// a workgroup a request and query head, a key's elements over the lanes: 64
// requests of 1 to 2048 keys, 16 heads of 60 703 us (of 64, by tiles, 50; of 64 off
// their alignment 784).
#include <cmath>

#include "cbx_attn.h"

namespace cbx {
namespace {

__device__ __forceinline__ float wave_sum_f32(float v) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d);
    return v;
}

// An element of a row of keys or values, an I8 one without its scale.
template <typename TC> __device__ __forceinline__ float held(const char* row, uint32_t e) {
    if constexpr (sizeof(TC) == 1) return static_cast<float>(reinterpret_cast<const int8_t*>(row)[e]);
    else return Elt<TC>::load1(row + e * Elt<TC>::size);
}

// PACKED: a row of q is a token of its request and attends up to itself.
template <typename T, typename TC, bool PACKED>
__global__ __launch_bounds__(kAttnThreads) void k_attn_rows(AttnArgs a) {
    constexpr int W = kAttnThreads / 64, N = kAttnMaxD / 64;
    __shared__ float lds_o[W][kAttnMaxD];
    __shared__ float lds_m[W], lds_l[W];
    const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
    const uint32_t t = blockIdx.x / a.hq, h = blockIdx.x - t * a.hq, hk = h / a.g;
    uint32_t s = t;
    int64_t behind = 0;                          // tokens of the request after this one
    if constexpr (PACKED) {
        uint32_t lo = 0, hi = a.n_seq;           // the first request that starts behind t
        while (lo < hi) {
            const uint32_t mid = (lo + hi) / 2;
            if (a.start[mid] > static_cast<int32_t>(t)) hi = mid;
            else lo = mid + 1;
        }
        s = lo - 1;
        if (lo == 0 || a.start[s] > static_cast<int32_t>(t) || a.start[s + 1] <= static_cast<int32_t>(t)) return;
        behind = static_cast<int64_t>(a.start[s + 1]) - 1 - t;
    }
    const int64_t cap = static_cast<int64_t>(a.max_pages) * a.page;
    int64_t len = a.lens[s];
    bool wrong = len < 0 || len > cap;
    len = len < 0 ? 0 : (len > cap ? cap : len);
    len = len > behind ? len - behind : 0;
    const int64_t first = a.window > 0 && len > a.window ? len - a.window : 0;
    const int32_t* row = reinterpret_cast<const int32_t*>(a.tables + s * a.t_nb1);
    const char* qr = a.q + t * a.q_nb2 + h * a.q_nb1;
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
            if (e < a.D) dot = fmaf(q[i], held<TC>(kr, e), dot);
        }
        float sc = wave_sum_f32(dot) * a.scale, vsc = 1.0f;
        if constexpr (sizeof(TC) == 1) {
            sc *= *reinterpret_cast<const float*>(a.ks + pg * a.ks_nb2 + hk * a.ks_nb1 + at * a.ks_nb0);
            vsc = *reinterpret_cast<const float*>(a.vs + pg * a.vs_nb2 + hk * a.vs_nb1 + at * a.vs_nb0);
        }
        if (a.softcap > 0.0f) sc = a.softcap * tanhf(sc / a.softcap);
        const float m2 = fmaxf(m, sc);
        const float keep = expf(m - m2), p = expf(sc - m2);
        l = fmaf(l, keep, p);
#pragma unroll
        for (int i = 0; i < N; i++) {
            const uint32_t e = lane + 64 * i;
            if (e < a.D) o[i] = fmaf(p * vsc, held<TC>(vr, e), o[i] * keep);
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
    char* yr = a.y + t * a.y_nb2 + h * a.y_nb1;
    for (uint32_t e = threadIdx.x; e < a.D; e += kAttnThreads) {
        float o1 = 0.0f;
#pragma unroll
        for (int w = 0; w < W; w++) o1 = fmaf(lds_o[w][e], f[w], o1);
        Elt<T>::store1(yr + e * Elt<T>::size, ll == 0.0f ? 0.0f : o1 / ll);
    }
}


// ---- tiles ------------------------------------------------------------------

typedef _Float16 h2v __attribute__((ext_vector_type(2)));
typedef _Float16 h8v __attribute__((ext_vector_type(8)));
typedef _Float16 h4u __attribute__((ext_vector_type(4), aligned(2)));
typedef float f4v __attribute__((ext_vector_type(4)));
typedef __bf16 b8v __attribute__((ext_vector_type(8)));
typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));
typedef const int32_t __attribute__((address_space(4))) const_i32;
typedef uint32_t u2v __attribute__((ext_vector_type(2)));
typedef uint32_t u2w __attribute__((ext_vector_type(2), aligned(4)));
typedef uint32_t u4w __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u3v __attribute__((ext_vector_type(3)));
typedef uint32_t u4v __attribute__((ext_vector_type(4)));

// Four neighbouring elements at any element alignment.
__device__ __forceinline__ void load4u(const char* p, float* v, float) {
    const f4u t = *reinterpret_cast<const f4u*>(p);
#pragma unroll
    for (int j = 0; j < 4; j++) v[j] = t[j];
}
__device__ __forceinline__ void load4u(const char* p, float* v, uint16_t) {
    const h4u t = *reinterpret_cast<const h4u*>(p);
#pragma unroll
    for (int j = 0; j < 4; j++) v[j] = static_cast<float>(t[j]);
}

// Where a lane reads a row: behind a base of the wave's at the lane's offset
// (a buffer load, whose base and step stay in scalar registers), or behind a
// pointer of its own.
struct WaveRows {
    __amdgpu_buffer_rsrc_t base;
    uint32_t off, step;     // the lane's, the wave's
    __device__ __forceinline__ WaveRows(const char* p, uint32_t o, uint32_t s)
        : base(__builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(p), 0, -1, 0x00027000)), off(o), step(s) {}
    __device__ __forceinline__ u4v load16(uint32_t o) const {
        return __builtin_amdgcn_raw_buffer_load_b128(base, static_cast<int>(off + o), static_cast<int>(step), 0);
    }
    __device__ __forceinline__ u3v load12(uint32_t o) const {
        return __builtin_amdgcn_raw_buffer_load_b96(base, static_cast<int>(off + o), static_cast<int>(step), 0);
    }
    __device__ __forceinline__ u2v load8(uint32_t o) const {
        return __builtin_amdgcn_raw_buffer_load_b64(base, static_cast<int>(off + o), static_cast<int>(step), 0);
    }
    __device__ __forceinline__ uint32_t load4(uint32_t o) const {
        return __builtin_amdgcn_raw_buffer_load_b32(base, static_cast<int>(off + o), static_cast<int>(step), 0);
    }
};
struct LaneRow {
    const char* p;
    __device__ __forceinline__ u4v load16(uint32_t o) const { return *reinterpret_cast<const u4w*>(p + o); }
    __device__ __forceinline__ u3v load12(uint32_t o) const {
        const u2v t = load8(o);
        return u3v{t.x, t.y, *reinterpret_cast<const uint32_t*>(p + o + 8)};
    }
    __device__ __forceinline__ u2v load8(uint32_t o) const { return *reinterpret_cast<const u2w*>(p + o); }
    __device__ __forceinline__ uint32_t load4(uint32_t o) const { return *reinterpret_cast<const uint32_t*>(p + o); }
};

// A request's keys: [first, len), and the tiles of KT keys they lie in; a
// request without keys has one tile all the same, which writes its zeros.
struct Span {
    uint32_t first, len, tile0, tiles;
    bool wrong;
};
template <int KT, bool OWN>
__device__ __forceinline__ Span span_of(const AttnArgs& a, uint32_t s) {
    const uint32_t cap = a.max_pages * a.page;
    const int32_t n = a.lens[s];
    Span r;
    r.wrong = n < 0 || static_cast<uint32_t>(n) > cap;
    r.len = n < 0 ? 0 : min(static_cast<uint32_t>(n), cap);
    r.first = a.window > 0 && r.len > static_cast<uint32_t>(a.window) ? r.len - a.window : 0;
    if (OWN && static_cast<int32_t>(s) >= a.groups[0] && static_cast<int32_t>(s) < a.groups[a.n_groups]) {
        r.first = max(r.first, min(static_cast<uint32_t>(max(a.own_first[s], 0)), r.len));
    }
    r.tile0 = r.first / KT;
    r.tiles = max(1u, (r.len + KT - 1) / KT - r.tile0);
    return r;
}

// Inclusive prefix sum over the wave: within rows of 16 lanes by shifts, then
// each row's last to the rows behind it.
template <int CTRL, int ROWS> __device__ __forceinline__ uint32_t dpp_add(uint32_t x) {
    return x + static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(x), CTRL, ROWS, 0xf, false));
}
__device__ __forceinline__ uint32_t wave_scan(uint32_t x) {
    x = dpp_add<0x111, 0xf>(x);   // row_shr 1, 2, 4, 8
    x = dpp_add<0x112, 0xf>(x);
    x = dpp_add<0x114, 0xf>(x);
    x = dpp_add<0x118, 0xf>(x);
    x = dpp_add<0x142, 0xa>(x);   // row_bcast 15 to rows 1 and 3
    return dpp_add<0x143, 0xc>(x);   // row_bcast 31 to rows 2 and 3
}

// The exclusive prefix over the requests of their tiles, as every workgroup
// needs it: each thread sums c neighbouring requests.  *total the sum.
template <int KT, bool OWN>
__device__ __forceinline__ uint32_t tiles_before(const AttnArgs& a, uint32_t c, uint32_t* lds, uint32_t* mine, uint32_t* total) {
    const uint32_t tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
    uint32_t sum = 0;
    for (uint32_t s = tid * c; s < min(a.n_seq, (tid + 1) * c); s++) sum += span_of<KT, OWN>(a, s).tiles;
    const uint32_t x = wave_scan(sum);
    if (lane == 63) lds[wid] = x;
    __syncthreads();
    uint32_t before = 0, all = 0;
#pragma unroll
    for (uint32_t w = 0; w < kAttnThreads / 64; w++) {
        if (w < wid) before += lds[w];
        all += lds[w];
    }
    *mine = sum;
    *total = all;
    return before + x - sum;
}

// T tiles in W <= T runs, the first T % W of them a tile longer.
struct Runs {
    uint32_t q, r;
    __device__ __forceinline__ Runs(uint32_t T, uint32_t W) : q(T / W), r(T - T / W * W) {}
    __device__ __forceinline__ uint32_t start(uint32_t w) const { return w * q + min(w, r); }
    __device__ __forceinline__ uint32_t of(uint32_t t) const {     // the run that holds tile t
        const uint32_t longer = r * (q + 1);
        return t < longer ? t / (q + 1) : r + (t - longer) / q;
    }
};

// N dwords (a multiple of 4, or 2, 3 or 6) of a row from byte offset o on.
template <int N, typename Row> __device__ __forceinline__ void load_dwords(const Row& r, uint32_t o, uint32_t (&v)[N]) {
    if constexpr (N == 3) {
        const u3v t = r.load12(o);
        v[0] = t.x;
        v[1] = t.y;
        v[2] = t.z;
        return;
    }
#pragma unroll
    for (int i = 0; i + 4 <= N; i += 4) {
        const u4v t = r.load16(o + 4 * i);
#pragma unroll
        for (int j = 0; j < 4; j++) v[i + j] = t[j];
    }
    if constexpr (N % 4 == 2) {
        const u2v t = r.load8(o + 4 * (N - 2));
        v[N - 2] = t.x;
        v[N - 1] = t.y;
    }
}

// The first of the PER dims that row m of O^T stands for.  The rows past D's
// end stand for its last dims again, and make the same sums of them.
template <int PER> __device__ __forceinline__ uint32_t value_dim(uint32_t m, uint32_t D) { return min(m * PER, D - PER); }

// A query's elements as f16: an F32 one's in two parts, see Core<uint16_t>.
template <int CD>
__device__ __forceinline__ void split_query(const float (&x)[CD * 8], bool f32, h8v (&qh)[CD], h8v (&ql)[CD], float* qmul) {
    *qmul = 1.0f;
    float m = 0.0f;
    if (f32) {
#pragma unroll
        for (int i = 0; i < CD * 8; i++) m = fmaxf(m, fabsf(x[i]));
        m = fmaxf(m, __shfl_xor(m, 16));
        m = fmaxf(m, __shfl_xor(m, 32));
        // 2^e <= m < 2^(e + 1) goes to [2^14, 2^15)
        int e = m > 0.0f && m < INFINITY ? static_cast<int>(__builtin_bit_cast(uint32_t, m) >> 23) - 127 : 14;
        e = e < -100 ? -100 : e;
        *qmul = ldexpf(1.0f, e - 14);
        const float up = ldexpf(1.0f, 14 - e);
#pragma unroll
        for (int i = 0; i < CD * 8; i++) {
            const float t = x[i] * up;
            const _Float16 h = static_cast<_Float16>(t);
            qh[i / 8][i % 8] = h;
            ql[i / 8][i % 8] = static_cast<_Float16>((t - static_cast<float>(h)) * 4096.0f);   // below 2^15
        }
    } else {
#pragma unroll
        for (int i = 0; i < CD * 8; i++) qh[i / 8][i % 8] = static_cast<_Float16>(x[i]);
    }
}

// A matrix core's view of NK keys and 16 heads.  S^T = K Q^T: the A operand's
// row is the key (lane % 16), the B operand's column the head (lane % 16),
// both hold for the lane group lane / 16 the same dims; the result's lane has
// head lane % 16 and keys 4 (lane / 16) + r.  O^T = V^T P^T: the B operand is
// then what the lane already holds (the sum over the keys may take them in
// any order, as long as V's rows come in the same one), the A operand's row
// m is dim value_dim(m) + d of product d: a lane reads DP/16 neighbouring dims
// of its keys.  The result's lane has head lane % 16 and dims
// value_dim(4 (lane / 16) + r) + d.
template <typename TC, int DP> struct Core;

// f16 pages: 16x16x32 products, f32 sums.  An f32 query is scaled by a power
// of two to below 2^15 and split into two f16, the lower times 2^12 and summed
// apart: every element is held to 2^-23 of itself, or to 2^-51 of the largest
// where that is more (f16 ends at 2^-24, so both halves in one sum ended at 2^-39).
// A probability is two f16 as well, times 2^14: held to 2^-23 of itself, those
// below 2^-28 of the largest to 2^-39 of it.  (Lower halves of these summed
// apart would take as many registers again as the sums over the values.)
template <int DP> struct Core<uint16_t, DP> {
    static constexpr bool SCALED = false;
    static constexpr int NK = 32, NH = 2, NE = 8;   // keys a step, halves of 16, keys whose values a lane holds
    static constexpr int CD = DP / 32, PER = DP / 16;
    h8v qh[CD], ql[CD], kf[NH][CD];
    uint32_t vr[NE][CD];
    f4v acc[DP / 16];
    float qmul;        // what the query's power of two leaves to multiply scores by
    bool two;          // ql is not zero

    __device__ __forceinline__ void load_q(const float (&x)[CD * 8], bool f32) {
        two = f32;
        split_query<CD>(x, f32, qh, ql, &qmul);
    }
    // dims the lane holds of its query and keys: 8 at 32 c + 8 grp
    static __device__ __forceinline__ uint32_t dim_of(int c, uint32_t grp) { return 32 * c + 8 * grp; }
    static constexpr int QC = CD, QN = 8;

    // byte offsets of the lane's dims in a key's row (of dims past D: the
    // row's first) and in a value's
    uint32_t ko[CD], vo;
    __device__ __forceinline__ void offsets(uint32_t n, uint32_t grp, uint32_t D) {
#pragma unroll
        for (int c = 0; c < CD; c++) ko[c] = dim_of(c, grp) < D ? 2 * dim_of(c, grp) : 0;
        vo = 2 * value_dim<PER>(n, D);
    }
    template <typename Row> __device__ __forceinline__ void load_k(int h, const Row& r) {
#pragma unroll
        for (int c = 0; c < CD; c++) kf[h][c] = __builtin_bit_cast(h8v, r.load16(ko[c]));
    }
    __device__ __forceinline__ void trim_k(uint32_t grp, uint32_t D) {   // dims past D: 0
#pragma unroll
        for (int c = 0; c < CD; c++) {
            if (dim_of(c, grp) >= D) {
#pragma unroll
                for (int h = 0; h < NH; h++) kf[h][c] = h8v{};
            }
        }
    }
    template <typename Row> __device__ __forceinline__ void load_v(int e, const Row& r) { load_dwords<CD>(r, vo, vr[e]); }
    __device__ __forceinline__ void drop_v(int e) {
#pragma unroll
        for (int c = 0; c < CD; c++) vr[e][c] = 0;
    }
    // keys of the lane's NE scores and values: h half, r in it
    static __device__ __forceinline__ uint32_t key_of(int e, uint32_t grp) { return 16 * (e >> 2) + 4 * grp + (e & 3); }
    static constexpr int half_of(int e) { return e >> 2; }

    __device__ __forceinline__ void scores(float (&s)[NE]) {
#pragma unroll
        for (int h = 0; h < NH; h++) {
            f4v t = {}, low = {};
#pragma unroll
            for (int c = 0; c < CD; c++) t = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[h][c], qh[c], t, 0, 0, 0);
            if (two) {
#pragma unroll
                for (int c = 0; c < CD; c++) low = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[h][c], ql[c], low, 0, 0, 0);
            }
#pragma unroll
            for (int r = 0; r < 4; r++) s[4 * h + r] = two ? fmaf(low[r], 0x1p-12f, t[r]) : t[r];
        }
    }
    static constexpr float kUp = 16384.0f;   // what probabilities are multiplied by
    __device__ __forceinline__ void add_values(const float (&p)[NE]) {
        h8v ph, pl;
#pragma unroll
        for (int e = 0; e < NE; e++) {
            const _Float16 h = static_cast<_Float16>(p[e]);
            ph[e] = h;
            pl[e] = static_cast<_Float16>(p[e] - static_cast<float>(h));
        }
#pragma unroll
        for (int c = 0; c < CD; c++) {
            u4v lo, hi;   // dims 2c and 2c + 1 of the lane's eight keys
#pragma unroll
            for (int i = 0; i < 4; i++) {
                lo[i] = __builtin_amdgcn_perm(vr[2 * i + 1][c], vr[2 * i][c], 0x05040100u);
                hi[i] = __builtin_amdgcn_perm(vr[2 * i + 1][c], vr[2 * i][c], 0x07060302u);
            }
            const h8v a0 = __builtin_bit_cast(h8v, lo), a1 = __builtin_bit_cast(h8v, hi);
            acc[2 * c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a0, pl, acc[2 * c], 0, 0, 0);
            acc[2 * c + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a1, pl, acc[2 * c + 1], 0, 0, 0);
            acc[2 * c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a0, ph, acc[2 * c], 0, 0, 0);
            acc[2 * c + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a1, ph, acc[2 * c + 1], 0, 0, 0);
        }
    }
};

// I8 pages: the elements as whole numbers, exact in f16 and bf16.  Scores from
// f16 products as above, times the keys' scales in f32.  A probability times its
// value's scale may lie anywhere in f32's range, so it is split into bf16 parts
// for products of bf16: three under an F32 query (all 24 bits), two under an F16
// one (its upper 16 bits: up to 2^-15 of it are cut off, a sixteenth of what the
// F16 result is rounded by).  A lane reads 16 dims of a key at once: MFMA c takes dims
// 64 (c / 2) + 16 (lane / 16) + 8 (c % 2) + [0, 8).  Half the bytes of F16 pages;
// 8 requests of 1500 to 65000 keys, 32 heads of 128 on 8: 108 us (561 MB, 5.2
// TB/s), of which the bytes take 104.  Short requests are bound by the widening,
// 320 instructions for 32 keys of a head: 64 of 1 to 2048 keys, 16 heads of 64
// under an F32 query, 43.5 us (143 MB, 3.3 TB/s).
template <int DP> struct Core<int8_t, DP> {
    static constexpr bool SCALED = true;
    static constexpr int NK = 32, NH = 2, NE = 8;
    static constexpr int CD = DP / 32, PER = DP / 16;
    h8v qh[CD], ql[CD];
    u4v kf[NH][CD / 2];
    uint32_t vr[NE][PER / 4];
    float ks[NE], vs[NE];
    f4v acc[DP / 16];
    float qmul;
    bool two;
    __device__ __forceinline__ void load_q(const float (&x)[CD * 8], bool f32) {
        two = f32;
        split_query<CD>(x, f32, qh, ql, &qmul);
    }
    static __device__ __forceinline__ uint32_t dim_of(int c, uint32_t grp) { return 64 * (c / 2) + 16 * grp + 8 * (c & 1); }
    static constexpr int QC = CD, QN = 8;
    uint32_t ko[CD / 2], vo;
    __device__ __forceinline__ void offsets(uint32_t n, uint32_t grp, uint32_t D) {
#pragma unroll
        for (int c = 0; c < CD / 2; c++) ko[c] = 64 * c + 16 * grp < D ? 64 * c + 16 * grp : 0;
        vo = value_dim<PER>(n, D);
    }
    template <typename Row> __device__ __forceinline__ void load_k(int h, const Row& r) {
#pragma unroll
        for (int c = 0; c < CD / 2; c++) kf[h][c] = r.load16(ko[c]);
    }
    __device__ __forceinline__ void trim_k(uint32_t grp, uint32_t D) {
#pragma unroll
        for (int c = 0; c < CD / 2; c++) {
            if (64 * c + 16 * grp >= D) {
#pragma unroll
                for (int h = 0; h < NH; h++) kf[h][c] = u4v{};
            }
        }
    }
    template <typename Row> __device__ __forceinline__ void load_v(int e, const Row& r) {
        if constexpr (PER == 4) vr[e][0] = r.load4(vo);
        else if constexpr (PER == 8) {
            const u2v t = r.load8(vo);
            vr[e][0] = t.x;
            vr[e][1] = t.y;
        } else {
            const u4v t = r.load16(vo);
#pragma unroll
            for (int i = 0; i < 4; i++) vr[e][i] = t[i];
        }
    }
    __device__ __forceinline__ void drop_v(int e) {
        vs[e] = 0.0f;
#pragma unroll
        for (int c = 0; c < PER / 4; c++) vr[e][c] = 0;
    }
    static __device__ __forceinline__ uint32_t key_of(int e, uint32_t grp) { return 16 * (e >> 2) + 4 * grp + (e & 3); }
    static constexpr int half_of(int e) { return e >> 2; }

    // 8 whole numbers to f16: 1024 + 128 + x is a half with x + 128 in its low byte
    static __device__ __forceinline__ h8v wide(uint32_t lo, uint32_t hi) {
        h8v r;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t x = (i < 2 ? lo : hi) ^ 0x80808080u;
            const h2v t = __builtin_bit_cast(h2v, __builtin_amdgcn_perm(0x64646464u, x, i & 1 ? 0x04030402u : 0x04010400u)) -
                          h2v{static_cast<_Float16>(1152), static_cast<_Float16>(1152)};
            r[2 * i] = t[0];
            r[2 * i + 1] = t[1];
        }
        return r;
    }
    __device__ __forceinline__ void scores(float (&s)[NE]) {
#pragma unroll
        for (int h = 0; h < NH; h++) {
            f4v t = {}, low = {};
#pragma unroll
            for (int c = 0; c < CD; c++) {
                const u4v& w = kf[h][c / 2];
                const h8v k = c & 1 ? wide(w[2], w[3]) : wide(w[0], w[1]);
                t = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, qh[c], t, 0, 0, 0);
                if (two) low = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, ql[c], low, 0, 0, 0);
            }
#pragma unroll
            for (int r = 0; r < 4; r++) s[4 * h + r] = (two ? fmaf(low[r], 0x1p-12f, t[r]) : t[r]) * ks[4 * h + r];
        }
    }
    static constexpr float kUp = 1.0f;
    __device__ __forceinline__ void add_values(const float (&p)[NE]) {
        u4v part[3];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            uint32_t b[3][2];
#pragma unroll
            for (int z = 0; z < 2; z++) {
                float y = p[2 * i + z] * vs[2 * i + z];
#pragma unroll
                for (int k = 0; k < 3; k++) {
                    b[k][z] = __builtin_bit_cast(uint32_t, y);
                    y -= __builtin_bit_cast(float, b[k][z] & 0xffff0000u);
                }
            }
#pragma unroll
            for (int k = 0; k < 3; k++) part[k][i] = __builtin_amdgcn_perm(b[k][1], b[k][0], 0x07060302u);
        }
#pragma unroll
        for (int d = 0; d < PER; d++) {
            u4v w;   // dim d of the lane's eight keys
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float x0 = static_cast<float>(static_cast<int8_t>(vr[2 * i][d / 4] >> 8 * (d & 3)));
                const float x1 = static_cast<float>(static_cast<int8_t>(vr[2 * i + 1][d / 4] >> 8 * (d & 3)));
                w[i] = __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, x1), __builtin_bit_cast(uint32_t, x0), 0x07060302u);
            }
            const b8v v = __builtin_bit_cast(b8v, w);
            if (two) acc[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, __builtin_bit_cast(b8v, part[2]), acc[d], 0, 0, 0);
            acc[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, __builtin_bit_cast(b8v, part[1]), acc[d], 0, 0, 0);
            acc[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, __builtin_bit_cast(b8v, part[0]), acc[d], 0, 0, 0);
        }
    }
};

// f32 pages: 16x16x4 products of f32.
template <int DP> struct Core<float, DP> {
    static constexpr bool SCALED = false;
    static constexpr int NK = 16, NH = 1, NE = 4;
    static constexpr int CD = DP / 16, PER = DP / 16;
    f4v qf[CD], kf[NH][CD];
    uint32_t vr[NE][PER];
    f4v acc[DP / 16];
    float qmul;
    static constexpr int QC = CD, QN = 4;
    __device__ __forceinline__ void load_q(const float (&x)[CD * 4], bool) {
        qmul = 1.0f;
#pragma unroll
        for (int i = 0; i < CD * 4; i++) qf[i / 4][i % 4] = x[i];
    }
    static __device__ __forceinline__ uint32_t dim_of(int c, uint32_t grp) { return 16 * c + 4 * grp; }
    uint32_t ko[CD], vo;
    __device__ __forceinline__ void offsets(uint32_t n, uint32_t grp, uint32_t D) {
#pragma unroll
        for (int c = 0; c < CD; c++) ko[c] = dim_of(c, grp) < D ? 4 * dim_of(c, grp) : 0;
        vo = 4 * value_dim<PER>(n, D);
    }
    template <typename Row> __device__ __forceinline__ void load_k(int h, const Row& r) {
#pragma unroll
        for (int c = 0; c < CD; c++) kf[h][c] = __builtin_bit_cast(f4v, r.load16(ko[c]));
    }
    __device__ __forceinline__ void trim_k(uint32_t grp, uint32_t D) {
#pragma unroll
        for (int c = 0; c < CD; c++) {
            if (dim_of(c, grp) >= D) kf[0][c] = f4v{};
        }
    }
    template <typename Row> __device__ __forceinline__ void load_v(int e, const Row& r) { load_dwords<PER>(r, vo, vr[e]); }
    __device__ __forceinline__ void drop_v(int e) {
#pragma unroll
        for (int c = 0; c < PER; c++) vr[e][c] = 0;
    }
    static __device__ __forceinline__ uint32_t key_of(int e, uint32_t grp) { return 4 * grp + e; }
    static constexpr int half_of(int) { return 0; }
    __device__ __forceinline__ void scores(float (&s)[NE]) {
        f4v t = {};
#pragma unroll
        for (int c = 0; c < CD; c++) {
#pragma unroll
            for (int i = 0; i < 4; i++) t = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[0][c][i], qf[c][i], t, 0, 0, 0);
        }
#pragma unroll
        for (int r = 0; r < 4; r++) s[r] = t[r];
    }
    static constexpr float kUp = 1.0f;
    __device__ __forceinline__ void add_values(const float (&p)[NE]) {
#pragma unroll
        for (int r = 0; r < NE; r++) {
#pragma unroll
            for (int d = 0; d < DP / 16; d++) {
                acc[d] = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(float, vr[r][d]), p[r], acc[d], 0, 0, 0);
            }
        }
    }
};

// Workgroups of a tile kernel that a CU holds, which their registers are limited to.
constexpr int per_cu(int dp, bool uni) { return dp <= 64 ? (uni ? 4 : 3) : dp <= 96 ? (uni ? 3 : 2) : dp <= 128 ? 2 : 1; }

// UNI: a page holds whole runs of 16 keys, looked up once a wave and half;
// else every lane looks its key up and passes the page on.  OWN: the keys
// behind a group's shared ones, as parts (a form of its own: asked for at run
// time, it cost every other call 0.15 us and 23 requests of up to 7001 F32 keys
// 39.2 us for 38.4).
template <typename TQ, typename TC, int DP, bool UNI, bool OWN>
__global__ __launch_bounds__(kAttnThreads, per_cu(DP, UNI)) void k_attn_tiles(AttnArgs a) {
    using C = Core<TC, DP>;
    constexpr int NK = C::NK, NH = C::NH, NE = C::NE, W4 = kAttnThreads / 64, KT = NK * W4;
    extern __shared__ float lds_o[];                 // [4][gc][DP + 4]
    __shared__ float lds_m[W4][16], lds_l[W4][16];
    __shared__ uint32_t lds_scan[W4], lds_at[2];
    const uint32_t tid = threadIdx.x, lane = tid & 63, n = lane & 15, grp = lane >> 4;
    const uint32_t wid = __builtin_amdgcn_readfirstlane(tid >> 6);
    bool wrong = false;

    // this workgroup's run of tiles, and the request that its first lies in
    uint32_t s, base, at, end, W = 1, T = 1;
    uint4 split = make_uint4(0, 0, 0, 0);
    if (a.W == 0) {
        s = blockIdx.x / a.H;
        base = 0;
        const uint32_t tiles = span_of<KT, OWN>(a, s).tiles;
        at = (blockIdx.x - s * a.H) * tiles;
        end = at + tiles;
    } else {
        const uint32_t c = (a.n_seq + kAttnThreads - 1) / kAttnThreads;
        uint32_t mine, total;
        uint32_t before = tiles_before<KT, OWN>(a, c, lds_scan, &mine, &total);
        T = total * a.H;
        W = min(a.W, T);                                 // runs, each of a tile at least
        if (blockIdx.x >= W) {
            if (tid == 0) a.split[blockIdx.x] = make_uint4(0, 0, 0, 0);
            return;
        }
        const Runs runs(T, W);
        at = runs.start(blockIdx.x);
        end = runs.start(blockIdx.x + 1);
        if (before * a.H <= at && at < (before + mine) * a.H) {
            uint32_t i = tid * c;
            for (;; i++) {
                const uint32_t t = span_of<KT, OWN>(a, i).tiles;
                if (at < (before + t) * a.H) break;
                before += t;
            }
            lds_at[0] = i;
            lds_at[1] = before * a.H;
        }
        __syncthreads();
        s = __builtin_amdgcn_readfirstlane(lds_at[0]);
        base = __builtin_amdgcn_readfirstlane(lds_at[1]);
    }

    C core;
    core.offsets(n, grp, a.D);
    while (at < end) {
        const Span sp = span_of<KT, OWN>(a, s);
        wrong |= sp.wrong;
        const uint32_t h = (at - base) / sp.tiles, t0 = at - base - h * sp.tiles;
        const uint32_t n_tiles = min(end - at, sp.tiles - t0);
        const uint32_t hk = h / a.ngr, h0 = (h - hk * a.ngr) * a.gc;     // key head, first of the group's heads
        const uint32_t heads = min(a.gc, a.g - h0);
        const uint32_t hq0 = hk * a.g + h0;
        const int32_t* row = reinterpret_cast<const int32_t*>(a.tables + s * a.t_nb1);
        {
            float x[C::QC * C::QN];
            const char* qr = a.q + s * a.q_nb2 + (hq0 + (n < heads ? n : 0)) * a.q_nb1;
#pragma unroll
            for (int i = 0; i < C::QC * C::QN; i += 4) {      // D % 8 == 0: four dims are all in or none
                const uint32_t d = C::dim_of(i / C::QN, grp) + i % C::QN;
                const bool in = n < heads && d < a.D;
                float t[4];
                load4u(qr + (in ? d : 0) * Elt<TQ>::size, t, TQ());
#pragma unroll
                for (int j = 0; j < 4; j++) x[i + j] = in ? t[j] : 0.0f;
            }
            core.load_q(x, sizeof(TQ) == 4);
        }
#pragma unroll
        for (int d = 0; d < DP / 16; d++) core.acc[d] = f4v{};
        float m = kLowest, l = 0.0f;
        const float scale = core.qmul * a.scale;

        // the wave's own steps: [tb, te) tiles, NK keys of each from kb on
        uint32_t tb = sp.tile0 + t0, te = tb + n_tiles;
        if (tb * KT + wid * NK + NK <= sp.first) tb++;
        if (te > tb && (te - 1) * KT + wid * NK >= sp.len) te--;

        const char* kb0 = a.k + hk * a.k_nb2;
        const char* vb0 = a.v + hk * a.v_nb2;
        // The pages of a step's keys.  UNI: one a half of 16 keys, read by scalar
        // loads (their own counter: nothing of the keys in flight is waited
        // for); else of key `lane` of the step.  Entries past the request's
        // keys are not used, those that are no page are left out.
        struct Pages {
            int32_t pg[NH];
            uint32_t ok;          // UNI: bit i: half i has keys
        };
        auto look_up = [&](uint32_t kb) {
            Pages r;
            r.ok = 0;
            if constexpr (UNI) {
#pragma unroll
                for (int i = 0; i < NH; i++) {
                    r.pg[i] = reinterpret_cast<const_i32*>(reinterpret_cast<uintptr_t>(row))[min(page_of(a, kb + 16 * i), a.max_pages - 1)];
                }
            } else {
                r.pg[0] = row[min(page_of(a, kb + (lane & (NK - 1))), a.max_pages - 1)];
            }
            return r;
        };
        auto settle = [&](Pages& r, uint32_t kb) {
            if constexpr (UNI) {
#pragma unroll
                for (int i = 0; i < NH; i++) {
                    const uint32_t key = kb + 16 * i;
                    const bool in = key < sp.len && key + 16 > sp.first, good = static_cast<uint32_t>(r.pg[i]) < a.n_pages;
                    wrong |= in && !good;
                    r.ok |= (in && good ? 1u : 0u) << i;
                    if (!good) r.pg[i] = 0;
                }
            } else {
                const uint32_t key = kb + (lane & (NK - 1));
                const bool in = key < sp.len && key >= sp.first, good = static_cast<uint32_t>(r.pg[0]) < a.n_pages;
                wrong |= in && !good;
                if (!in || !good) r.pg[0] = -1;
            }
        };
        // the scales of the lane's keys: those of four neighbours at once where they lie together in 16 bytes of one page
        auto fetch_s = [&](const Pages& r, uint32_t kb, const char* base, int64_t nb0, int64_t nb1, int64_t nb2, float (&to)[NE]) {
            const char* sb = base + hk * nb1;
            if (UNI && a.s_quads) {
#pragma unroll
                for (int i = 0; i < NH; i++) {
                    const uint32_t key = kb + 16 * i, in = key - page_of(a, key) * a.page;
                    const f4v t = *reinterpret_cast<const f4v*>(sb + (r.pg[i] * nb2 + in * 4) + 16 * grp);
#pragma unroll
                    for (int e = 0; e < 4; e++) to[4 * i + e] = t[e];
                }
                return;
            }
#pragma unroll
            for (int e = 0; e < NE; e++) {
                const uint32_t key = kb + C::key_of(e, grp);
                int32_t g;
                if constexpr (UNI) g = r.pg[C::half_of(e)];
                else g = __shfl(r.pg[0], C::key_of(e, grp));
                to[e] = *reinterpret_cast<const float*>(sb + (g < 0 ? 0 : g * nb2 + (key - page_of(a, key) * a.page) * nb0));
            }
        };
        // UNI: the half's first row is the wave's, the key's place in it the lane's
        auto fetch_k = [&](const Pages& r, uint32_t kb) {
            if constexpr (C::SCALED) fetch_s(r, kb, a.ks, a.ks_nb0, a.ks_nb1, a.ks_nb2, core.ks);
#pragma unroll
            for (int i = 0; i < NH; i++) {
                if constexpr (UNI) {
                    const uint32_t key = kb + 16 * i, in = key - page_of(a, key) * a.page;
                    core.load_k(i, WaveRows(kb0 + (r.pg[i] * a.k_nb3 + in * a.k_nb1), n * static_cast<uint32_t>(a.k_nb1), 0));
                } else {
                    const uint32_t key = kb + 16 * i + n;
                    const int32_t g = __shfl(r.pg[0], 16 * i + n);
                    core.load_k(i, LaneRow{kb0 + (g < 0 ? 0 : g * a.k_nb3 + (key - page_of(a, key) * a.page) * a.k_nb1)});
                }
            }
        };
        auto fetch_v = [&](const Pages& r, uint32_t kb) {
            if constexpr (C::SCALED) fetch_s(r, kb, a.vs, a.vs_nb0, a.vs_nb1, a.vs_nb2, core.vs);
            if constexpr (UNI) {
#pragma unroll
                for (int i = 0; i < NH; i++) {
                    const uint32_t key = kb + 16 * i, in = key - page_of(a, key) * a.page;
                    const char* p = vb0 + (r.pg[i] * a.v_nb3 + in * a.v_nb1);
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        core.load_v(4 * i + e, WaveRows(p, 4 * grp * static_cast<uint32_t>(a.v_nb1), e * static_cast<uint32_t>(a.v_nb1)));
                    }
                }
            } else {
#pragma unroll
                for (int e = 0; e < NE; e++) {
                    const uint32_t key = kb + C::key_of(e, grp);
                    const int32_t g = __shfl(r.pg[0], C::key_of(e, grp));
                    core.load_v(e, LaneRow{vb0 + (g < 0 ? 0 : g * a.v_nb3 + (key - page_of(a, key) * a.page) * a.v_nb1)});
                }
            }
        };
        // Keys of a step arrive while the values before them are used, values
        // while the next scores are made, pages a step before both.
        if (tb < te) {
            uint32_t kb = tb * KT + wid * NK;
            Pages cur = look_up(kb), next = look_up(kb + KT);
            settle(cur, kb);
            fetch_k(cur, kb);
            fetch_v(cur, kb);
            for (uint32_t t = tb; t < te; t++, kb += KT) {
                const bool more = t + 1 < te;
                const Pages after = look_up(kb + 2 * KT);
                if (a.D != DP) core.trim_k(grp, a.D);
                float sc[NE];
                core.scores(sc);
                if (more) {
                    settle(next, kb + KT);
                    fetch_k(next, kb + KT);
                }
                if (a.softcap > 0.0f) {
#pragma unroll
                    for (int e = 0; e < NE; e++) sc[e] = a.softcap * tanhf(sc[e] * scale / a.softcap) * kLog2e;
                } else {
#pragma unroll
                    for (int e = 0; e < NE; e++) sc[e] = sc[e] * (scale * kLog2e);
                }
                bool whole = kb >= sp.first && kb + NK <= sp.len;
                if constexpr (UNI) whole = whole && cur.ok == (1u << NH) - 1;
                else whole = whole && __all(cur.pg[0] >= 0);
                if (!whole) {
#pragma unroll
                    for (int e = 0; e < NE; e++) {
                        const uint32_t key = kb + C::key_of(e, grp);
                        bool live = key < sp.len && key >= sp.first;
                        if constexpr (UNI) live = live && (cur.ok >> C::half_of(e) & 1);
                        else live = __shfl(cur.pg[0], C::key_of(e, grp)) >= 0;
                        if (!live) {
                            sc[e] = -INFINITY;
                            core.drop_v(e);
                        }
                    }
                }
                float mx = sc[0];
#pragma unroll
                for (int e = 1; e < NE; e++) mx = fmaxf(mx, sc[e]);
                if (__any(mx > m)) {   // rare after the first steps: the sums are rescaled
                    mx = fmaxf(mx, __shfl_xor(mx, 16));
                    mx = fmaxf(mx, __shfl_xor(mx, 32));
                    const float m2 = fmaxf(m, mx), keep = __builtin_amdgcn_exp2f(m - m2);
                    m = m2;
                    l *= keep;
#pragma unroll
                    for (int d = 0; d < DP / 16; d++) core.acc[d] *= keep;
                }
                float p[NE];
#pragma unroll
                for (int e = 0; e < NE; e++) {
                    p[e] = __builtin_amdgcn_exp2f(sc[e] - m) * C::kUp;   // the difference alone: exact at the maximum, 0 there
                    l += p[e];
                }
                core.add_values(p);
                if (more) fetch_v(next, kb + KT);
                cur = next;
                next = after;
            }
        }
        l += __shfl_xor(l, 16);
        l += __shfl_xor(l, 32);

        // the four waves' parts, joined through LDS
        const uint32_t ld = DP + 4;
        if (n < heads) {
            float* o = lds_o + (wid * a.gc + n) * ld;
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const uint32_t d0 = value_dim<DP / 16>(4 * grp + r, a.D);
#pragma unroll
                for (int d = 0; d < DP / 16; d++) o[d0 + d] = core.acc[d][r];
            }
            if (grp == 0) {
                lds_m[wid][n] = m;
                lds_l[wid][n] = l;
            }
        }
        __syncthreads();
        const bool entire = n_tiles == sp.tiles;
        if (t0 == 0 && !entire) {
            split = make_uint4(s, hq0, heads, Runs(T, W).of(at + sp.tiles - 1) - blockIdx.x + 1);
        }
        const uint64_t slot = (static_cast<uint64_t>(blockIdx.x) * 2 + (t0 > 0 ? 0 : 1)) * a.gc;
        for (uint32_t i = tid; i < heads * a.D; i += kAttnThreads) {
            const uint32_t hh = i / a.D, d = i - hh * a.D;
            float mm = lds_m[0][hh];
#pragma unroll
            for (int w = 1; w < W4; w++) mm = fmaxf(mm, lds_m[w][hh]);
            float ll = 0.0f, oo = 0.0f;
#pragma unroll
            for (int w = 0; w < W4; w++) {
                const float f = __builtin_amdgcn_exp2f(lds_m[w][hh] - mm);
                ll = fmaf(lds_l[w][hh], f, ll);
                oo = fmaf(lds_o[(w * a.gc + hh) * ld + d], f, oo);
            }
            if (entire && OWN) {
                const uint64_t own = static_cast<uint64_t>(s) * a.hq + hq0 + hh;
                a.own_o[own * a.D + d] = oo * a.own_down;
                if (d == 0) a.own_ml[own] = make_float2(mm, ll * a.own_down);
            } else if (entire) {
                Elt<TQ>::store1(a.y + s * a.y_nb2 + (hq0 + hh) * a.y_nb1 + d * Elt<TQ>::size, ll == 0.0f ? 0.0f : oo / ll);
            } else {
                a.part_o[(slot + hh) * a.D + d] = oo;
                if (d == 0) a.part_ml[slot + hh] = make_float2(mm, ll);
            }
        }
        __syncthreads();
        at += n_tiles;
        if (at == base + sp.tiles * a.H) {
            s++;
            base = at;
        }
    }
    if (a.W != 0 && tid == 0) a.split[blockIdx.x] = split;
    if (__any(wrong) && lane == 0) atomicOr(a.err, DEV_ERR_PAGE);   // of any lane: each may have looked up another key's page
}

// Adds up the parts of the key heads that several runs hold, in the order of
// the runs: a workgroup a run that such a key head begins in and a head of it.
// Part 0 lies in its run's second place (the run ends with it), the others in
// the first.  A wave adds every fourth part, a part's dims over its lanes, 8
// parts in flight (of the first 32 already while their maxima are read).
template <typename TQ, int DP, bool OWN>
__global__ __launch_bounds__(kAttnThreads) void k_attn_join(AttnArgs a) {
    constexpr int N = DP / 64, U = 8;
    __shared__ float lds_m[kAttnThreads / 64], lds_l[kAttnThreads / 64], lds_f[kAttnThreads];
    __shared__ float lds_o[kAttnThreads / 64][DP];
    const uint32_t run = blockIdx.x / a.gc, hh = blockIdx.x - run * a.gc;
    const uint4 sp = a.split[run];
    const uint32_t parts = sp.w;
    if (parts == 0 || hh >= sp.z) return;
    const uint32_t tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
    auto slot = [&](uint32_t i) { return (static_cast<uint64_t>(run + i) * 2 + (i == 0 ? 1 : 0)) * a.gc + hh; };
    float o[N], x[U][N];
    auto fetch = [&](uint32_t i0) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const uint32_t i = i0 + 4 * u < parts ? i0 + 4 * u : 0;
            const float* p = a.part_o + slot(i) * a.D;
#pragma unroll
            for (int j = 0; j < N; j++) x[u][j] = p[lane + 64 * j < a.D ? lane + 64 * j : 0];
        }
    };
    fetch(wid);
    float m = kLowest;
    for (uint32_t i = tid; i < parts; i += kAttnThreads) m = fmaxf(m, a.part_ml[slot(i)].x);
    for (int d = 32; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor(m, d));
    if (lane == 0) lds_m[wid] = m;
    __syncthreads();
    m = fmaxf(fmaxf(lds_m[0], lds_m[1]), fmaxf(lds_m[2], lds_m[3]));
    float l = 0.0f;
#pragma unroll
    for (int j = 0; j < N; j++) o[j] = 0.0f;
    for (uint32_t t = 0; t < parts; t += kAttnThreads) {      // 256 parts a turn
        __syncthreads();
        float f = 0.0f;
        if (t + tid < parts) {
            const float2 ml = a.part_ml[slot(t + tid)];
            f = __builtin_amdgcn_exp2f(ml.x - m);
            l = fmaf(ml.y, f, l);
        }
        lds_f[tid] = f;                                       // 0 past the last part
        __syncthreads();
        for (uint32_t i = wid; i < min(parts - t, static_cast<uint32_t>(kAttnThreads)); i += 4 * U) {
            if (t + i != wid) fetch(t + i);
#pragma unroll
            for (int u = 0; u < U; u++) {
                const float g = i + 4 * u < kAttnThreads ? lds_f[i + 4 * u] : 0.0f;
                if (g == 0.0f) continue;                      // also no part: what is read for it is another's
#pragma unroll
                for (int j = 0; j < N; j++) o[j] = fmaf(x[u][j], g, o[j]);
            }
        }
    }
    for (int d = 32; d > 0; d >>= 1) l += __shfl_xor(l, d);
    if (lane == 0) lds_l[wid] = l;
#pragma unroll
    for (int j = 0; j < N; j++) lds_o[wid][lane + 64 * j] = o[j];
    __syncthreads();
    l = ((lds_l[0] + lds_l[1]) + lds_l[2]) + lds_l[3];
    const uint64_t own = static_cast<uint64_t>(sp.x) * a.hq + sp.y + hh;
    if (OWN && tid == 0) a.own_ml[own] = make_float2(m, l * a.own_down);
    char* yr = a.y + sp.x * a.y_nb2 + (sp.y + hh) * a.y_nb1;
    for (uint32_t d = tid; d < a.D; d += kAttnThreads) {
        const float t = ((lds_o[0][d] + lds_o[1][d]) + lds_o[2][d]) + lds_o[3][d];
        if (OWN) a.own_o[own * a.D + d] = t * a.own_down;
        else Elt<TQ>::store1(yr + d * Elt<TQ>::size, l == 0.0f ? 0.0f : t / l);
    }
}

// ---- what runs where ------------------------------------------------------------

bool uniform_pages(const cbx_tensor* k) { return k->ne[1] % 16 == 0; }

struct AttnPlan {
    bool tiles;            // k_attn_tiles, else k_attn_rows
    int dp, kt;
    uint32_t gc, ngr, H, W;
    bool join;             // a key head's tiles may fall into several runs
    size_t o_bytes, ml_bytes, bytes;   // of the workspace
};

// Everything but addresses, which the workspace's size may not depend on.
AttnPlan attn_plan(const cbx_tensor* q, const cbx_tensor* k, const cbx_tensor* tables, const DeviceState* st) {
    AttnPlan p{};
    const int64_t D = q->ne[0], hkv = k->ne[2], g = hkv ? q->ne[1] / hkv : 0;
    const int64_t cap = tables->ne[0] * k->ne[1];
    p.dp = D <= 64 ? 64 : D <= 96 && k->type != CBX_TYPE_I8 ? 96 : D <= 128 ? 128 : 256;
    p.kt = (k->type == CBX_TYPE_F32 ? 16 : 32) * (kAttnThreads / 64);
    p.ngr = static_cast<uint32_t>(cdiv(g, 16));
    p.gc = static_cast<uint32_t>(cdiv(g, p.ngr));
    p.H = static_cast<uint32_t>(hkv) * p.ngr;
    const int64_t cap_tiles = std::max<int64_t>(1, cdiv(cap, p.kt));
    const int64_t most = q->ne[2] * p.H * cap_tiles;
    p.tiles = D % (k->type == CBX_TYPE_I8 ? 16 : 8) == 0 && D <= 256 && cap > 0 && k->ne[3] > 0 && most < (int64_t{1} << 31);
    if (!p.tiles) return p;
    p.W = static_cast<uint32_t>(std::min<int64_t>(static_cast<int64_t>(per_cu(p.dp, uniform_pages(k))) * st->n_cu, most));
    // A run a key head, without a join, while the longest a table can hold ends
    // about with the rest: 0.7 to 1.4 us a tile of one key head after another,
    // against 5 us for the join and two key heads a run.  Both sides measured with
    // lengths from 1 to the table's, S key heads: S 16, 3 tiles 6.9 us against
    // 9.3, 8 tiles 10.4 against 9.3; S 64, 8 tiles 11.2 / 11.5, 16 tiles 19.7 /
    // 14.0; S 256, 16 tiles 20.7 / 21.4 (head_dim 128: 35 / 41), 32 tiles 43 / 35;
    // S 512, 16 tiles 64 / 73, 32 tiles 123 / 117; S 1024, 32 tiles 114 / 114, 64
    // tiles 221 / 204: they cross near the square root of S.  Lengths that the
    // tables' width says little about are worse off by the rule: 300 keys in
    // tables of 2048 are split for nothing (S 16: 9.6 us against 7.1), one
    // request of 4096 keys beside 63 of 64 is not (S 1024: 34.7 / 14.0).
    const int64_t S = std::min<int64_t>(q->ne[2] * p.H, 1024);
    p.join = cap_tiles > 7 && cap_tiles * cap_tiles > S;
    if (p.join) {
        p.o_bytes = static_cast<size_t>(cdiv(static_cast<int64_t>(p.W) * 2 * p.gc * D * 4, 16) * 16);
        p.ml_bytes = static_cast<size_t>(p.W) * 2 * p.gc * 8;
        p.bytes = p.o_bytes + p.ml_bytes + static_cast<size_t>(p.W) * sizeof(uint4);
    }
    return p;
}

template <typename TQ, typename TC, int DP, bool OWN>
void tiles_uni(bool uni, dim3 grid, size_t lds, hipStream_t s, const AttnArgs& a) {
    if (uni) hipLaunchKernelGGL((k_attn_tiles<TQ, TC, DP, true, OWN>), grid, dim3(kAttnThreads), lds, s, a);
    else hipLaunchKernelGGL((k_attn_tiles<TQ, TC, DP, false, OWN>), grid, dim3(kAttnThreads), lds, s, a);
}

template <typename TQ, typename TC, bool OWN>
void launch_tiles(const AttnPlan& p, bool uni, AttnArgs& a, hipStream_t s) {
    if (!p.join) a.W = 0;
    const dim3 grid(p.join ? p.W : a.n_seq * a.H);
    const size_t lds = static_cast<size_t>(kAttnThreads / 64) * p.gc * (p.dp + 4) * sizeof(float);
    if (p.dp == 64) tiles_uni<TQ, TC, 64, OWN>(uni, grid, lds, s, a);
    else if (p.dp == 96) {
        if constexpr (sizeof(TC) > 1) tiles_uni<TQ, TC, 96, OWN>(uni, grid, lds, s, a);
    }
    else if (p.dp == 128) tiles_uni<TQ, TC, 128, OWN>(uni, grid, lds, s, a);
    else tiles_uni<TQ, TC, 256, OWN>(uni, grid, lds, s, a);
    if (!p.join) return;
    const dim3 parts(p.W * p.gc);
    if (p.dp == 64) hipLaunchKernelGGL((k_attn_join<TQ, 64, OWN>), parts, dim3(kAttnThreads), 0, s, a);
    else if (p.dp <= 128) hipLaunchKernelGGL((k_attn_join<TQ, 128, OWN>), parts, dim3(kAttnThreads), 0, s, a);
    else hipLaunchKernelGGL((k_attn_join<TQ, 256, OWN>), parts, dim3(kAttnThreads), 0, s, a);
}

template <typename TQ, typename TC> void launch_tiles(const AttnPlan& p, bool uni, AttnArgs& a, hipStream_t s) {
    if (a.own_first) launch_tiles<TQ, TC, true>(p, uni, a, s);
    else launch_tiles<TQ, TC, false>(p, uni, a, s);
}

}  // namespace

size_t paged_attention_workspace(const cbx_tensor* q, const cbx_tensor* k, const cbx_tensor* tables, const DeviceState* st) {
    return attn_plan(q, k, tables, st).bytes;
}

bool vector_rows(const cbx_tensor* t) {
    if (reinterpret_cast<uintptr_t>(t->data) % 16) return false;
    for (int i = 1; i < 4; i++) if (t->ne[i] > 1 && t->nb[i] % 16) return false;
    return t->nb[1] < (size_t{1} << 26);
}

// Scales that can be read four at a time.
static bool quad_scales(const cbx_tensor* t) {
    if (t->ne[0] > 1 && t->nb[0] != 4) return false;
    if (reinterpret_cast<uintptr_t>(t->data) % 16) return false;
    for (int i = 1; i < 3; i++) if (t->ne[i] > 1 && t->nb[i] % 16) return false;
    return true;
}

AttnArgs attn_args(const PagedAttnCall& c, const DeviceState* st) {
    AttnArgs a{};
    auto at = [](const cbx_tensor* t) { return t ? static_cast<const char*>(t->data) : nullptr; };
    auto nb = [](const cbx_tensor* t, int i) { return t ? static_cast<int64_t>(t->nb[i]) : 0; };
    a.q = at(c.q);
    a.k = at(c.k);
    a.v = at(c.v);
    a.ks = at(c.k_scale);
    a.vs = at(c.v_scale);
    a.tables = at(c.tables);
    a.lens = reinterpret_cast<const int32_t*>(at(c.lens));
    a.start = reinterpret_cast<const int32_t*>(at(c.start));
    a.y = static_cast<char*>(c.y->data);
    a.q_nb1 = nb(c.q, 1); a.q_nb2 = nb(c.q, 2);
    a.y_nb1 = nb(c.y, 1); a.y_nb2 = nb(c.y, 2);
    a.k_nb1 = nb(c.k, 1); a.k_nb2 = nb(c.k, 2); a.k_nb3 = nb(c.k, 3);
    a.v_nb1 = nb(c.v, 1); a.v_nb2 = nb(c.v, 2); a.v_nb3 = nb(c.v, 3);
    a.ks_nb0 = nb(c.k_scale, 0); a.ks_nb1 = nb(c.k_scale, 1); a.ks_nb2 = nb(c.k_scale, 2);
    a.vs_nb0 = nb(c.v_scale, 0); a.vs_nb1 = nb(c.v_scale, 1); a.vs_nb2 = nb(c.v_scale, 2);
    a.t_nb1 = nb(c.tables, 1);
    a.n_seq = static_cast<uint32_t>(c.tables->ne[1]);
    a.n_rows = static_cast<uint32_t>(c.q->ne[2]);
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
    if (a.page > 0) page_division(a.page, &a.page_mul, &a.page_shift);
    return a;
}

int launch_attention_rows(const AttnArgs& a, const PagedAttnCall& c, const char* what, hipStream_t s) {
    const dim3 grid(a.n_rows * a.hq), block(kAttnThreads);
    auto go = [&](auto t, auto tc) {
        if (a.start) hipLaunchKernelGGL((k_attn_rows<decltype(t), decltype(tc), true>), grid, block, 0, s, a);
        else hipLaunchKernelGGL((k_attn_rows<decltype(t), decltype(tc), false>), grid, block, 0, s, a);
    };
    auto with = [&](auto t) {
        if (c.k->type == CBX_TYPE_I8) go(t, int8_t());
        else if (c.k->type == CBX_TYPE_F16) go(t, uint16_t());
        else go(t, float());
    };
    if (c.q->type == CBX_TYPE_F16) with(uint16_t());
    else with(float());
    return check_launch(what);
}

size_t attention_tiles_workspace(const cbx_tensor* q, const cbx_tensor* k, const cbx_tensor* tables, const DeviceState* st) {
    return attn_plan(q, k, tables, st).bytes;
}

bool attention_tiles(const cbx_tensor* q, const cbx_tensor* k, const cbx_tensor* tables, const DeviceState* st) {
    return attn_plan(q, k, tables, st).tiles;
}

bool launch_attention_tiles(AttnArgs a, const PagedAttnCall& c, void* ws, DeviceState* st, hipStream_t s) {
    const AttnPlan p = attn_plan(c.q, c.k, c.tables, st);
    if (!p.tiles || !std::isfinite(c.scale * kLog2e) || !vector_rows(c.k) || !vector_rows(c.v)) return false;
    a.gc = p.gc;
    a.ngr = p.ngr;
    a.H = p.H;
    a.W = p.W;
    a.part_o = static_cast<float*>(ws);
    a.part_ml = reinterpret_cast<float2*>(static_cast<char*>(ws) + p.o_bytes);
    a.split = reinterpret_cast<uint4*>(static_cast<char*>(ws) + p.o_bytes + p.ml_bytes);
    a.own_down = c.k->type == CBX_TYPE_F16 ? 1.0f / Core<uint16_t, 64>::kUp : 1.0f;
    const bool t16 = c.q->type == CBX_TYPE_F16, c16 = c.k->type == CBX_TYPE_F16, uni = uniform_pages(c.k);
    if (c.k->type == CBX_TYPE_I8) {
        a.s_quads = quad_scales(c.k_scale) && quad_scales(c.v_scale);
        if (t16) launch_tiles<uint16_t, int8_t>(p, uni, a, s);
        else launch_tiles<float, int8_t>(p, uni, a, s);
    } else if (t16 && c16) launch_tiles<uint16_t, uint16_t>(p, uni, a, s);
    else if (t16) launch_tiles<uint16_t, float>(p, uni, a, s);
    else if (c16) launch_tiles<float, uint16_t>(p, uni, a, s);
    else launch_tiles<float, float>(p, uni, a, s);
    return true;
}

int launch_paged_attention(const PagedAttnCall& c, DeviceState* st, hipStream_t s) {
    const AttnArgs a = attn_args(c, st);
    if (launch_attention_tiles(a, c, c.ws, st, s)) return check_launch("cbx_paged_attention");
    return launch_attention_rows(a, c, "cbx_paged_attention", s);
}

}  // namespace cbx
