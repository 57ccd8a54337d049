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
#include "cbx_device.h"

namespace cbx {
namespace {

constexpr int kAttnThreads = 256;
constexpr int kAttnMaxD = 512;
constexpr float kLowest = -3.0e38f;   // below every score that matters; finite, so that m - m is 0
constexpr float kLog2e = 1.44269504088896340736f;

struct AttnArgs {
    const char *q, *k, *v, *tables;
    const int32_t* lens;
    char* y;
    int64_t q_nb1, q_nb2, y_nb1, y_nb2, k_nb1, k_nb2, k_nb3, v_nb1, v_nb2, v_nb3, t_nb1;
    uint32_t n_seq, hq, hkv, g, D, page, max_pages, n_pages;
    int32_t window;
    float scale, softcap;
    uint32_t* err;
    // k_attn_tiles and k_attn_join
    uint32_t page_mul, page_shift;   // key / page = (key * page_mul) >> page_shift for key < 2^31
    uint32_t gc, ngr, H;             // heads a run holds (<= 16), runs of heads a group, hkv * ngr
    uint32_t W;                      // runs; 0: a run a request and key head, none of them split
    float* part_o;                   // [W][2][gc][D]
    float2* part_ml;                 // [W][2][gc]
    uint4* split;                    // [W]: request, first query head, heads and parts of the key head that begins
                                     // in the run and ends in a later one; no parts: none does
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


// ---- tiles ------------------------------------------------------------------

typedef _Float16 h2v __attribute__((ext_vector_type(2)));
typedef _Float16 h8v __attribute__((ext_vector_type(8)));
typedef _Float16 h4u __attribute__((ext_vector_type(4), aligned(2)));
typedef float f4v __attribute__((ext_vector_type(4)));
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
};
struct LaneRow {
    const char* p;
    __device__ __forceinline__ u4v load16(uint32_t o) const { return *reinterpret_cast<const u4w*>(p + o); }
    __device__ __forceinline__ u3v load12(uint32_t o) const {
        const u2v t = load8(o);
        return u3v{t.x, t.y, *reinterpret_cast<const uint32_t*>(p + o + 8)};
    }
    __device__ __forceinline__ u2v load8(uint32_t o) const { return *reinterpret_cast<const u2w*>(p + o); }
};

__device__ __forceinline__ uint32_t page_of(const AttnArgs& a, uint32_t key) {
    return static_cast<uint32_t>((static_cast<uint64_t>(key) * a.page_mul) >> a.page_shift);
}

// A request's keys: [first, len), and the tiles of KT keys they lie in; a
// request without keys has one tile all the same, which writes its zeros.
struct Span {
    uint32_t first, len, tile0, tiles;
    bool wrong;
};
template <int KT>
__device__ __forceinline__ Span span_of(const AttnArgs& a, uint32_t s) {
    const uint32_t cap = a.max_pages * a.page;
    const int32_t n = a.lens[s];
    Span r;
    r.wrong = n < 0 || static_cast<uint32_t>(n) > cap;
    r.len = n < 0 ? 0 : min(static_cast<uint32_t>(n), cap);
    r.first = a.window > 0 && r.len > static_cast<uint32_t>(a.window) ? r.len - a.window : 0;
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
template <int KT>
__device__ __forceinline__ uint32_t tiles_before(const AttnArgs& a, uint32_t c, uint32_t* lds, uint32_t* mine, uint32_t* total) {
    const uint32_t tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
    uint32_t sum = 0;
    for (uint32_t s = tid * c; s < min(a.n_seq, (tid + 1) * c); s++) sum += span_of<KT>(a, s).tiles;
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
    static constexpr int NK = 32, NH = 2, NE = 8;   // keys a step, halves of 16, keys whose values a lane holds
    static constexpr int CD = DP / 32, PER = DP / 16;
    h8v qh[CD], ql[CD], kf[NH][CD];
    uint32_t vr[NE][CD];
    f4v acc[DP / 16];
    float qmul;        // what the query's power of two leaves to multiply scores by
    bool two;          // ql is not zero

    __device__ __forceinline__ void load_q(const float (&x)[CD * 8], bool f32) {
        two = f32;
        qmul = 1.0f;
        float m = 0.0f;
        if (f32) {
#pragma unroll
            for (int i = 0; i < CD * 8; i++) m = fmaxf(m, fabsf(x[i]));
            m = fmaxf(m, __shfl_xor(m, 16));
            m = fmaxf(m, __shfl_xor(m, 32));
            // 2^e <= m < 2^(e + 1) goes to [2^14, 2^15)
            int e = m > 0.0f && m < INFINITY ? static_cast<int>(__builtin_bit_cast(uint32_t, m) >> 23) - 127 : 14;
            e = e < -100 ? -100 : e;
            qmul = ldexpf(1.0f, e - 14);
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

// f32 pages: 16x16x4 products of f32.
template <int DP> struct Core<float, DP> {
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
// else every lane looks its key up and passes the page on.
template <typename TQ, typename TC, int DP, bool UNI>
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
        const uint32_t tiles = span_of<KT>(a, s).tiles;
        at = (blockIdx.x - s * a.H) * tiles;
        end = at + tiles;
    } else {
        const uint32_t c = (a.n_seq + kAttnThreads - 1) / kAttnThreads;
        uint32_t mine, total;
        uint32_t before = tiles_before<KT>(a, c, lds_scan, &mine, &total);
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
                const uint32_t t = span_of<KT>(a, i).tiles;
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
        const Span sp = span_of<KT>(a, s);
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
        // UNI: the half's first row is the wave's, the key's place in it the lane's
        auto fetch_k = [&](const Pages& r, uint32_t kb) {
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
            if (entire) {
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
template <typename TQ, int DP>
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
    char* yr = a.y + sp.x * a.y_nb2 + (sp.y + hh) * a.y_nb1;
    for (uint32_t d = tid; d < a.D; d += kAttnThreads) {
        const float t = ((lds_o[0][d] + lds_o[1][d]) + lds_o[2][d]) + lds_o[3][d];
        Elt<TQ>::store1(yr + d * Elt<TQ>::size, l == 0.0f ? 0.0f : t / l);
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
    p.dp = D <= 64 ? 64 : D <= 96 ? 96 : D <= 128 ? 128 : 256;
    p.kt = (k->type == CBX_TYPE_F16 ? 32 : 16) * (kAttnThreads / 64);
    p.ngr = static_cast<uint32_t>(cdiv(g, 16));
    p.gc = static_cast<uint32_t>(cdiv(g, p.ngr));
    p.H = static_cast<uint32_t>(hkv) * p.ngr;
    const int64_t cap_tiles = std::max<int64_t>(1, cdiv(cap, p.kt));
    const int64_t most = q->ne[2] * p.H * cap_tiles;
    p.tiles = D % 8 == 0 && D <= 256 && cap > 0 && k->ne[3] > 0 && most < (int64_t{1} << 31);
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

bool vector_rows(const cbx_tensor* t) {
    if (reinterpret_cast<uintptr_t>(t->data) % 16) return false;
    for (int i = 1; i < 4; i++) if (t->ne[i] > 1 && t->nb[i] % 16) return false;
    return t->nb[1] < (size_t{1} << 26);
}

template <typename TQ, typename TC, int DP>
void tiles_uni(bool uni, dim3 grid, size_t lds, hipStream_t s, const AttnArgs& a) {
    if (uni) hipLaunchKernelGGL((k_attn_tiles<TQ, TC, DP, true>), grid, dim3(kAttnThreads), lds, s, a);
    else hipLaunchKernelGGL((k_attn_tiles<TQ, TC, DP, false>), grid, dim3(kAttnThreads), lds, s, a);
}

template <typename TQ, typename TC>
void launch_tiles(const AttnPlan& p, bool uni, AttnArgs& a, hipStream_t s) {
    if (!p.join) a.W = 0;
    const dim3 grid(p.join ? p.W : a.n_seq * a.H);
    const size_t lds = static_cast<size_t>(kAttnThreads / 64) * p.gc * (p.dp + 4) * sizeof(float);
    if (p.dp == 64) tiles_uni<TQ, TC, 64>(uni, grid, lds, s, a);
    else if (p.dp == 96) tiles_uni<TQ, TC, 96>(uni, grid, lds, s, a);
    else if (p.dp == 128) tiles_uni<TQ, TC, 128>(uni, grid, lds, s, a);
    else tiles_uni<TQ, TC, 256>(uni, grid, lds, s, a);
    if (!p.join) return;
    const dim3 parts(p.W * p.gc);
    if (p.dp == 64) hipLaunchKernelGGL((k_attn_join<TQ, 64>), parts, dim3(kAttnThreads), 0, s, a);
    else if (p.dp <= 128) hipLaunchKernelGGL((k_attn_join<TQ, 128>), parts, dim3(kAttnThreads), 0, s, a);
    else hipLaunchKernelGGL((k_attn_join<TQ, 256>), parts, dim3(kAttnThreads), 0, s, a);
}

}  // namespace

size_t paged_attention_workspace(const cbx_tensor* q, const cbx_tensor* k, const cbx_tensor* tables, const DeviceState* st) {
    return attn_plan(q, k, tables, st).bytes;
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
    const AttnPlan p = attn_plan(c.q, c.k, c.tables, st);
    if (p.tiles && vector_rows(c.k) && vector_rows(c.v)) {
        page_division(a.page, &a.page_mul, &a.page_shift);
        a.gc = p.gc;
        a.ngr = p.ngr;
        a.H = p.H;
        a.W = p.W;
        a.part_o = static_cast<float*>(c.ws);
        a.part_ml = reinterpret_cast<float2*>(static_cast<char*>(c.ws) + p.o_bytes);
        a.split = reinterpret_cast<uint4*>(static_cast<char*>(c.ws) + p.o_bytes + p.ml_bytes);
        const bool t16 = c.q->type == CBX_TYPE_F16, c16 = c.k->type == CBX_TYPE_F16;
        if (t16 && c16) launch_tiles<uint16_t, uint16_t>(p, uniform_pages(c.k), a, s);
        else if (t16) launch_tiles<uint16_t, float>(p, uniform_pages(c.k), a, s);
        else if (c16) launch_tiles<float, uint16_t>(p, uniform_pages(c.k), a, s);
        else launch_tiles<float, float>(p, uniform_pages(c.k), a, s);
        return check_launch("cbx_paged_attention");
    }
    const dim3 grid(static_cast<unsigned>(c.q->ne[1] * c.q->ne[2])), block(kAttnThreads);
    const bool t16 = c.q->type == CBX_TYPE_F16, c16 = c.k->type == CBX_TYPE_F16;
    if (t16 && c16) hipLaunchKernelGGL((k_attn_rows<uint16_t, uint16_t>), grid, block, 0, s, a);
    else if (t16) hipLaunchKernelGGL((k_attn_rows<uint16_t, float>), grid, block, 0, s, a);
    else if (c16) hipLaunchKernelGGL((k_attn_rows<float, uint16_t>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((k_attn_rows<float, float>), grid, block, 0, s, a);
    return check_launch("cbx_paged_attention");
}

}  // namespace cbx
