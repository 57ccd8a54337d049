// k_logprob.hip -- log probabilities of given tokens, entropy and the largest
// alternatives from a row of logits.
//
// With z_i = scale (x_i - max x), T = sum exp(z_i):
//   log p_i = z_i - log T,  H = log T - (sum exp(z_i) z_i) / T
// (both terms of H are >= 0: nothing cancels).  The difference is taken of the
// halves, exact as it is but for numbers below 2^-125, where it is 2^-150 off:
// logits of both signs may lie further apart than the largest f32.  Order: 64-bit keys of the
// logit's bits made monotone and the complement of its index, all distinct,
// so that the alternatives do not depend on who finds them.
//
// Bound by the read of the logits, made once: a workgroup holds a chunk of a
// row in registers (up to 16384 logits), reduces it to its maximum, T and
// sum, and picks its alternatives.  A row of several chunks is joined by a
// second kernel from the chunks' (maximum, T, sum) and their alternatives.  4000
// rows of 8194 F32, 8 alternatives: 28.3 us (131 MB, 4.6 TB/s; 27.4 without the
// profiler); 64 rows, 4 alternatives, 5.6 us; one row of 151936 F16, 20
// alternatives, 6.2 + 4.8 us.
//
// The N largest without a sort: the 64 lanes' own maxima (over all waves)
// are ranked; at least N logits are not below the N-th of them, and with
// logits in any usual order few more (20 of 8194: some 24), so these are
// collected in LDS and each is ranked among them.  When they do not fit
// there (rows of equal or masked logits), the same is done with keys instead
// of values; when those do not fit either (the largest all in a few lanes),
// or the row holds a NaN, the N maxima are searched one after the other.
#include "cbx_device.h"

namespace cbx {
namespace {

constexpr int kLpThreads = 256;
constexpr int kLpWaves = kLpThreads / 64;
constexpr uint32_t kLpChunk = 16384;    // most logits of a workgroup: 64 a thread
constexpr uint32_t kLpMany = 8192, kLpFew = 4096;   // of a chunk where a row has several: with many of them, with few
constexpr uint32_t kLpMost = 1024;      // keys collected in LDS
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;

struct LpArgs {
    const char* x;
    const int32_t* ids;
    float *logp, *entropy;
    char *top_ids, *top_logp;
    int64_t x_nb1, ti_nb1, tl_nb1;
    uint32_t V, rows, chunk, chunks;
    int32_t n_top;
    float scale;
    uint32_t* err;
    float4* sums;         // [rows][chunks]: maximum, T, sum, 1 when the chunk holds a NaN
    uint64_t* keys;       // [rows][n_top][chunks]
};

// Larger logits have larger keys; NaN the largest, -0 as +0, of equal ones the first index.
__device__ __forceinline__ uint32_t order_of(float x) {
    const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.0f);
    return x != x ? 0xfffffffeu : ((b & 0x80000000u) ? ~b : b | 0x80000000u);
}
__device__ __forceinline__ uint64_t key_of(float x, uint32_t i) {
    return (static_cast<uint64_t>(order_of(x)) << 32) | (0xffffffffu - i);
}
__device__ __forceinline__ uint32_t index_of(uint64_t k) { return 0xffffffffu - static_cast<uint32_t>(k); }
__device__ __forceinline__ float logit_of(uint64_t k) {
    const uint32_t o = static_cast<uint32_t>(k >> 32);
    return o == 0xfffffffeu ? __builtin_nanf("") : __builtin_bit_cast(float, (o & 0x80000000u) ? o & 0x7fffffffu : ~o);
}

__device__ __forceinline__ uint64_t max64(uint64_t a, uint64_t b) { return a > b ? a : b; }

struct LpShared {
    float f[3][kLpWaves];
    union {
        float lanef[kLpWaves][64];
        uint64_t lane[kLpWaves][64];
    };
    uint32_t above[kLpWaves][64];   // of a lane's, how many of 16 others are larger
    uint64_t kept[kLpMost];
    uint64_t best[kLpWaves];
    uint32_t count[2];
};

// One float of the lane that a DPP control pairs this one with.
template <int CTRL> __device__ __forceinline__ float dpp_f32(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float lane_f32(float v, int lane) {
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
}
// Over the 64 lanes, in the pairing order of wave_sum, the same in every lane.
template <typename F> __device__ __forceinline__ float wave_f32(F f, float v) {
    v = f(v, dpp_f32<0xB1>(v));
    v = f(v, dpp_f32<0x4E>(v));
    v = f(v, dpp_f32<0x141>(v));
    v = f(v, dpp_f32<0x140>(v));
    return f(f(lane_f32(v, 0), lane_f32(v, 16)), f(lane_f32(v, 32), lane_f32(v, 48)));
}
struct MaxOf { __device__ __forceinline__ float operator()(float a, float b) const { return fmaxf(a, b); } };
struct MinOf { __device__ __forceinline__ float operator()(float a, float b) const { return fminf(a, b); } };
struct SumOf { __device__ __forceinline__ float operator()(float a, float b) const { return a + b; } };

// The block's sums of a and b; the caller's barrier lies between the two calls.
__device__ __forceinline__ void put_sums(LpShared& sh, float a, float b) {
    a = wave_f32(SumOf(), a);
    b = wave_f32(SumOf(), b);
    if ((threadIdx.x & 63) == 0) {
        sh.f[1][threadIdx.x >> 6] = a;
        sh.f[2][threadIdx.x >> 6] = b;
    }
}
__device__ __forceinline__ void get_sums(const LpShared& sh, float& a, float& b) {
    a = sh.f[1][0];
    b = sh.f[2][0];
#pragma unroll
    for (int w = 1; w < kLpWaves; w++) {
        a += sh.f[1][w];
        b += sh.f[2][w];
    }
}

// put(rank, key) of the n largest of the keys collected in sh.kept.
template <typename Put>
__device__ __forceinline__ void rank_kept(const LpShared& sh, uint32_t found, int n, Put put) {
    for (uint32_t i = threadIdx.x; i < found; i += kLpThreads) {
        const uint64_t k = sh.kept[i];
        uint32_t rank = 0;
#pragma unroll 4
        for (uint32_t j = 0; j < found; j++) rank += sh.kept[j] > k;
        if (rank < static_cast<uint32_t>(n)) put(rank, k);
    }
}

// The n-th largest of the 64 lanes' maxima over the waves, which n of the
// block's values at least are not below.  Each wave counts for all 64 the
// larger ones among 16 of them (begin), a barrier of the caller's later the
// counts are added (end).
__device__ __forceinline__ uint32_t larger_of_16(float v) {
    const int base = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * 16;
    uint32_t above = 0;
#pragma unroll
    for (int i = 0; i < 16; i++) above += lane_f32(v, base + i) > v;
    return above;
}
__device__ __forceinline__ uint64_t lane_u64(uint64_t v, int lane) {
    return static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v >> 32), lane))) << 32 |
           static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), lane));
}
// Keys of 0 (lanes without any) are equal: in the lanes' order.
__device__ __forceinline__ uint32_t larger_of_16(uint64_t v) {
    const int base = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * 16, lane = threadIdx.x & 63;
    uint32_t above = 0;
#pragma unroll
    for (int i = 0; i < 16; i++) {
        const uint64_t other = lane_u64(v, base + i);
        above += other > v || (other == v && base + i < lane);
    }
    return above;
}
__device__ __forceinline__ uint32_t counted(const LpShared& sh) {
    const int lane = threadIdx.x & 63;
    uint32_t above = sh.above[0][lane];
#pragma unroll
    for (int w = 1; w < kLpWaves; w++) above += sh.above[w][lane];
    return above;
}
// The lanes' maxima over the waves, and what goes before counted().
template <typename T> __device__ __forceinline__ T lane_maxima(const T (&lds)[kLpWaves][64]) {
    const int lane = threadIdx.x & 63;
    T v = lds[0][lane];
#pragma unroll
    for (int w = 1; w < kLpWaves; w++) v = lds[w][lane] > v ? lds[w][lane] : v;
    return v;
}
// Of n < 2^6 counts below n there is one at least; the smallest such value.
__device__ __forceinline__ float value_floor(const LpShared& sh, int n, float v) {
    return wave_f32(MinOf(), counted(sh) < static_cast<uint32_t>(n) ? v : INFINITY);
}
__device__ __forceinline__ uint64_t key_floor(const LpShared& sh, int n, uint64_t v) {
    return lane_u64(v, __builtin_ctzll(__ballot(counted(sh) == static_cast<uint32_t>(n - 1))));
}

// The n largest keys one after the other.  each(f): f(key) for every key of
// the thread, all of them distinct, n in the block at least.
template <typename Each, typename Put>
__device__ __forceinline__ void search_largest(LpShared& sh, int n, Each each, Put put) {
    uint64_t last = ~uint64_t{0};
    for (int r = 0; r < n; r++) {
        uint64_t b = 0;
        each([&](uint64_t k) {
            if (k < last && k > b) b = k;
        });
        for (int d = 32; d > 0; d >>= 1) b = max64(b, __shfl_xor(static_cast<unsigned long long>(b), d));
        __syncthreads();
        if ((threadIdx.x & 63) == 0) sh.best[threadIdx.x >> 6] = b;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kLpWaves; w++) b = max64(b, sh.best[w]);
        last = b;
        if (threadIdx.x == 0) put(r, b);
    }
}

__device__ __forceinline__ void keep(LpShared& sh, int which, uint64_t k) {
    const uint32_t i = atomicAdd(&sh.count[which], 1u);
    if (i < kLpMost) sh.kept[i] = k;
}

// (x - m) / 2, which twice the scale then multiplies.
__device__ __forceinline__ float half_below(float x, float m) { return fmaf(x, 0.5f, -0.5f * m); }

// A row's results from its maximum, T and sum (in powers of 2).
struct RowSums {
    float m, T, u;
    bool nan;
    __device__ __forceinline__ bool empty() const { return m == -INFINITY && !nan; }
    __device__ __forceinline__ float log_p(float x, float scale) const {
        if (nan || m == INFINITY) return __builtin_nanf("");
        if (x == -INFINITY) return x;
        return half_below(x, m) * (2.0f * scale) - logf(T);
    }
    __device__ __forceinline__ float entropy() const {
        if (nan || m == INFINITY) return __builtin_nanf("");
        return empty() ? 0.0f : logf(T) - kLn2 * (u / T);
    }
};

// The given token's logit, read by thread 0 ahead of its use.
struct RowToken {
    bool good;
    float x;
};
template <typename T>
__device__ __forceinline__ RowToken row_token(const LpArgs& a, uint32_t row) {
    RowToken t{false, 0.0f};
    if (threadIdx.x == 0 && a.logp) {
        const int32_t id = a.ids[row];
        t.good = id >= 0 && static_cast<uint32_t>(id) < a.V;
        if (t.good) t.x = Elt<T>::load1(a.x + row * a.x_nb1 + static_cast<int64_t>(id) * Elt<T>::size);
    }
    return t;
}

__device__ __forceinline__ void write_row(const LpArgs& a, uint32_t row, const RowSums& rs, const RowToken& t) {
    if (threadIdx.x != 0) return;
    if (a.logp) {
        if (!t.good) atomicOr(a.err, DEV_ERR_ROW_INDEX);
        a.logp[row] = t.good ? rs.log_p(t.x, a.scale) : 0.0f;
    }
    if (a.entropy) a.entropy[row] = rs.entropy();
}

__device__ __forceinline__ void write_top(const LpArgs& a, uint32_t row, uint32_t rank, uint64_t k, const RowSums& rs) {
    reinterpret_cast<int32_t*>(a.top_ids + row * a.ti_nb1)[rank] = static_cast<int32_t>(index_of(k));
    reinterpret_cast<float*>(a.top_logp + row * a.tl_nb1)[rank] = rs.log_p(logit_of(k), a.scale);
}

// A logit, and four neighbouring ones at any element alignment.
template <typename T> struct Raw {
    typedef float type;
    typedef float vec __attribute__((ext_vector_type(4), aligned(4)));
};
template <> struct Raw<uint16_t> {
    typedef _Float16 type;
    typedef _Float16 vec __attribute__((ext_vector_type(4), aligned(2)));
};

// A chunk of a row in registers: NV vectors of 4 a thread, thread t holding
// logits 4 (256 j + t) + e of the chunk.
template <typename T, int NV>
__global__ __launch_bounds__(kLpThreads, NV <= 4 ? 8 : NV <= 9 ? 6 : 4) void k_logprob(LpArgs a) {
    __shared__ LpShared sh;
    typedef typename Raw<T>::type R;
    const uint32_t row = blockIdx.x / a.chunks, ch = blockIdx.x - row * a.chunks, tid = threadIdx.x;
    const uint32_t i0 = ch * a.chunk, n = min(a.chunk, a.V - i0);
    const R* x = reinterpret_cast<const R*>(a.x + row * a.x_nb1) + i0;
    // whole vectors first, all in flight (a conversion beside its load would
    // wait for it); what a last, partial one holds element by element
    typename Raw<T>::vec raw[NV];
#pragma unroll
    for (int j = 0; j < NV; j++) {
        const uint32_t i = 4 * (kLpThreads * j + tid);
        raw[j] = n >= 4 ? *reinterpret_cast<const typename Raw<T>::vec*>(x + (i + 4 <= n ? i : 0)) : typename Raw<T>::vec{};
    }
    float v[NV][4];
#pragma unroll
    for (int j = 0; j < NV; j++) {
        const uint32_t i = 4 * (kLpThreads * j + tid);
#pragma unroll
        for (int e = 0; e < 4; e++) v[j][e] = i + 4 <= n ? static_cast<float>(raw[j][e]) : -INFINITY;
        if (i < n && i + 4 > n) {
#pragma unroll
            for (int e = 0; e < 3; e++) if (i + e < n) v[j][e] = static_cast<float>(x[i + e]);
        }
    }
    float vm[NV];          // each vector's maximum
    float m = -INFINITY;
#pragma unroll
    for (int j = 0; j < NV; j++) {
        vm[j] = fmaxf(fmaxf(v[j][0], v[j][1]), fmaxf(v[j][2], v[j][3]));
        m = fmaxf(m, vm[j]);
    }
    RowToken token{false, 0.0f};
    if (a.chunks == 1) token = row_token<T>(a, row);
    const int lane = tid & 63, wid = tid >> 6;
    sh.lanef[wid][lane] = m;
    if (tid == 0) sh.count[0] = sh.count[1] = 0;
    __syncthreads();
    const float lm = lane_maxima(sh.lanef);
    RowSums rs;
    rs.m = wave_f32(MaxOf(), lm);
    if (a.n_top) sh.above[wid][lane] = larger_of_16(lm);
    const float sl = 2.0f * a.scale * kLog2e, off = rs.m == -INFINITY ? 0.0f : rs.m;
    rs.T = rs.u = 0.0f;
#pragma unroll
    for (int j = 0; j < NV; j++) {
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const float z = half_below(v[j][e], off) * sl, p = __builtin_amdgcn_exp2f(z);
            rs.T += p;
            rs.u = fmaf(p, fmaxf(z, -200.0f), rs.u);   // exp2(-200) is 0: 0, not 0 * -inf
        }
    }
    put_sums(sh, rs.T, rs.u);
    __syncthreads();
    get_sums(sh, rs.T, rs.u);
    rs.nan = rs.T != rs.T;
    if (a.chunks == 1) {
        write_row(a, row, rs, token);
    } else if (tid == 0) {
        a.sums[blockIdx.x] = make_float4(rs.m, rs.T, rs.u, rs.nan ? 1.0f : 0.0f);
    }
    if (a.n_top == 0) return;
    uint64_t* out = a.keys + static_cast<uint64_t>(row) * a.chunks * a.n_top + ch;
    if (a.chunks > 1 && tid >= n && tid < static_cast<uint32_t>(a.n_top)) out[tid * a.chunks] = 0;   // a last chunk shorter than n_top
    auto put = [&](uint32_t rank, uint64_t k) {
        if (a.chunks == 1) write_top(a, row, rank, k, rs);
        else out[rank * a.chunks] = k;
    };
    auto index = [&](int j, int e) { return 4 * (kLpThreads * j + tid) + e; };
    // the rare ways read the row again: keys of every register would be held for them
    auto each = [&](auto f) {
        for (uint32_t i = tid; i < n; i += kLpThreads) f(key_of(static_cast<float>(x[i]), i0 + i));
    };
    if (rs.nan) {
        search_largest(sh, min(a.n_top, static_cast<int>(n)), each, put);
        return;
    }
    const float fl = value_floor(sh, a.n_top, lm);
    if (m >= fl) {
#pragma unroll
        for (int j = 0; j < NV; j++) {
            if (vm[j] >= fl) {
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    if (v[j][e] >= fl && index(j, e) < n) keep(sh, 0, key_of(v[j][e], i0 + index(j, e)));
                }
            }
        }
    }
    __syncthreads();
    uint32_t found = sh.count[0];
    if (found > kLpMost) {      // too many that are equal: by key
        uint64_t best = 0;
        each([&](uint64_t k) { best = max64(best, k); });
        sh.lane[wid][lane] = best;
        __syncthreads();
        best = lane_maxima(sh.lane);
        sh.above[wid][lane] = larger_of_16(best);
        __syncthreads();
        const uint64_t kfl = key_floor(sh, a.n_top, best);
        each([&](uint64_t k) {
            if (k >= kfl) keep(sh, 1, k);
        });
        __syncthreads();
        found = sh.count[1];
    }
    if (found <= kLpMost) rank_kept(sh, found, a.n_top, put);
    else search_largest(sh, min(a.n_top, static_cast<int>(n)), each, put);
}

// A row of several chunks: their sums under the row's maximum, their
// alternatives' best (rank by rank, so that the lanes' maxima are the first
// ranks of the chunks).
template <typename T>
__global__ __launch_bounds__(kLpThreads) void k_logprob_join(LpArgs a) {
    __shared__ LpShared sh;
    const uint32_t row = blockIdx.x, tid = threadIdx.x;
    const float4* sums = a.sums + static_cast<uint64_t>(row) * a.chunks;
    const uint64_t* keys = a.keys + static_cast<uint64_t>(row) * a.chunks * a.n_top;
    const uint32_t n = a.chunks * a.n_top;
    const int lane = tid & 63, wid = tid >> 6;
    uint64_t best = 0;
    for (uint32_t i = tid; i < n; i += kLpThreads) best = max64(best, keys[i]);
    float m = -INFINITY;
    for (uint32_t c = tid; c < a.chunks; c += kLpThreads) m = fmaxf(m, sums[c].x);
    const RowToken token = row_token<T>(a, row);
    m = wave_f32(MaxOf(), m);
    if (lane == 0) sh.f[0][wid] = m;
    sh.lane[wid][lane] = best;
    if (tid == 0) sh.count[1] = 0;
    __syncthreads();
    best = lane_maxima(sh.lane);
    if (a.n_top) sh.above[wid][lane] = larger_of_16(best);
    RowSums rs;
    rs.m = fmaxf(fmaxf(sh.f[0][0], sh.f[0][1]), fmaxf(sh.f[0][2], sh.f[0][3]));
    const float sl = 2.0f * a.scale * kLog2e;
    rs.T = rs.u = 0.0f;
    for (uint32_t c = tid; c < a.chunks; c += kLpThreads) {
        const float4 s = sums[c];
        if (s.w != 0.0f) rs.T = __builtin_nanf("");
        if (s.x == -INFINITY) continue;
        const float z = half_below(s.x, rs.m) * sl, p = __builtin_amdgcn_exp2f(z);
        rs.T = fmaf(s.y, p, rs.T);
        if (p > 0.0f) rs.u = fmaf(p, fmaf(s.y, z, s.z), rs.u);
    }
    put_sums(sh, rs.T, rs.u);
    __syncthreads();
    get_sums(sh, rs.T, rs.u);
    rs.nan = rs.T != rs.T;
    write_row(a, row, rs, token);
    if (a.n_top == 0) return;
    auto each = [&](auto f) {
        for (uint32_t i = tid; i < n; i += kLpThreads) f(keys[i]);
    };
    const uint64_t fl = key_floor(sh, a.n_top, best);
    each([&](uint64_t k) {
        if (k >= fl) keep(sh, 1, k);
    });
    __syncthreads();
    const uint32_t found = sh.count[1];
    auto put = [&](uint32_t rank, uint64_t k) { write_top(a, row, rank, k, rs); };
    if (found <= kLpMost) rank_kept(sh, found, a.n_top, put);
    else search_largest(sh, a.n_top, each, put);
}

struct LpPlan {
    uint32_t chunk, chunks;
    size_t sums_bytes, bytes;
};

LpPlan lp_plan(const cbx_tensor* x, int n_top, const DeviceState* st) {
    LpPlan p{};
    const int64_t V = x->ne[0], rows = x->ne[1];
    // 4096 against 8192 logits a chunk: 1 row of 151936 11.7 us against 12.7, 16
    // rows 11.0 / 11.7, 60 rows 19.7 / 19.2, 200 rows 37 / 35
    const int64_t most = rows * cdiv(V, kLpMany) < 2 * st->n_cu ? kLpFew : kLpMany;
    const int64_t chunks = V <= kLpChunk ? 1 : cdiv(V, most);
    p.chunk = static_cast<uint32_t>(chunks == 1 ? V : cdiv(cdiv(V, chunks), 4) * 4);
    p.chunks = static_cast<uint32_t>(cdiv(V, p.chunk));
    if (p.chunks > 1) {
        p.sums_bytes = static_cast<size_t>(rows) * p.chunks * sizeof(float4);
        p.bytes = p.sums_bytes + static_cast<size_t>(rows) * p.chunks * static_cast<size_t>(n_top) * sizeof(uint64_t);
    }
    return p;
}

template <typename T>
void launch_lp(const LpArgs& a, hipStream_t s) {
    const dim3 grid(a.rows * a.chunks), block(kLpThreads);
    // vectors a thread: the fewest of these that hold the chunk, as those beyond it
    // are work all the same (4000 rows of 8194 in 16 of them 33.8 us against 25.6 in
    // 9, of 4096 29.9 / 15.9 in 4, 8000 rows of 1000 51.9 / 17.2 in 1; of 8192 in 9
    // 25.2 / 24.1 in 8, which no other length would need)
    const uint32_t nv = (a.chunk + 4 * kLpThreads - 1) / (4 * kLpThreads);
    if (nv <= 1) hipLaunchKernelGGL((k_logprob<T, 1>), grid, block, 0, s, a);
    else if (nv <= 2) hipLaunchKernelGGL((k_logprob<T, 2>), grid, block, 0, s, a);
    else if (nv <= 4) hipLaunchKernelGGL((k_logprob<T, 4>), grid, block, 0, s, a);
    else if (nv <= 9) hipLaunchKernelGGL((k_logprob<T, 9>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((k_logprob<T, 16>), grid, block, 0, s, a);
    if (a.chunks > 1) hipLaunchKernelGGL((k_logprob_join<T>), dim3(a.rows), block, 0, s, a);
}

}  // namespace

size_t token_log_probs_workspace(const cbx_tensor* x, int n_top, const DeviceState* st) { return lp_plan(x, n_top, st).bytes; }

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
    const LpPlan p = lp_plan(c.x, c.n_top, st);
    a.chunk = p.chunk;
    a.chunks = p.chunks;
    a.sums = static_cast<float4*>(c.ws);
    a.keys = reinterpret_cast<uint64_t*>(static_cast<char*>(c.ws) + p.sums_bytes);
    // a launch's threads below 2^32
    if (static_cast<uint64_t>(a.rows) * a.chunks >= (uint64_t{1} << 24) ||
        static_cast<uint64_t>(a.rows) * a.chunks * (a.n_top + 1) >= (uint64_t{1} << 31)) {
        return set_error(CBX_ERR_UNSUPPORTED, "cbx_token_log_probs: too many logits");
    }
    if (c.x->type == CBX_TYPE_F16) launch_lp<uint16_t>(a, s);
    else launch_lp<float>(a, s);
    return check_launch("cbx_token_log_probs");
}

}  // namespace cbx
