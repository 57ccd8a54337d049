// k_prompt_attn.hip -- causal attention of all new tokens of packed requests
// over a paged cache, and of one new token a request where groups of requests
// begin with the same pages.
//
// Row i attends over its keys [first_i, limit_i): y_i = sum_j softmax(s_i)_j v_j
// with s_ij = scale q_i . k_j, in one pass over the keys: with a running maximum
// m, l = sum exp(s - m) and o = sum exp(s - m) v, both rescaled when the maximum
// rises, and y = o / l at the end.
//
// 4 D products a row and key against 4 D bytes (F16) a key and row tile: bound by
// the products from some hundred rows on, or rather by what a score takes beside
// them, an exponential (four issue slots), two to four multiply-adds, a maximum
// and a conversion for 2 D products of its row.  Measured: 16000 tokens, 32 heads
// of 128 on 8, F16, 2.27 ms (920 TFLOP/s of the 1156 that a large product
// reaches; without the softmax 1010, without the copies into LDS 1050); 48
// requests of 1 to 2047 tokens, 16 heads of 64, 0.39 ms (593); 8 requests of 1 to
// 9 tokens on 900 to 32000 keys in 8 bits, 101 us (2.8 TB/s, latency).
//
// 32 rows a wave, because a wave's 32 x 32 products then need each key and value
// once out of LDS for 32 rows (64 rows a wave, one workgroup a CU: 616 TFLOP/s for
// 736; 256 rows a workgroup: 570), and 128 rows a workgroup, so that two or three
// fit a CU and one's products run beside another's softmax.
#include <cmath>

#include "cbx_attn.h"

namespace cbx {
namespace {

typedef _Float16 h2v __attribute__((ext_vector_type(2)));
typedef _Float16 h4v __attribute__((ext_vector_type(4)));
typedef _Float16 h8v __attribute__((ext_vector_type(8)));
typedef _Float16 h4u __attribute__((ext_vector_type(4), aligned(2)));
typedef __bf16 b8v __attribute__((ext_vector_type(8)));
typedef short s4v __attribute__((ext_vector_type(4)));
typedef float f4v __attribute__((ext_vector_type(4)));
typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));
typedef float f16v __attribute__((ext_vector_type(16)));
typedef uint32_t u2v __attribute__((ext_vector_type(2)));
typedef uint32_t u4v __attribute__((ext_vector_type(4)));

struct PromptArgs {
    AttnArgs a;
    const int32_t* shared;     // shared keys a group; null: packed tokens
    uint32_t n_start;          // requests or groups: start has one more
    uint32_t tiles;            // row tiles at most
    uint32_t g_mul, g_shift;   // i / g
    // row tiles' keys dealt to workgroups in pieces (see Piece); deal: how many are aimed at, 0: a row tile is one workgroup's
    uint32_t deal, slots, row_cap;   // pieces there is room for, rows of each
    float* part_o;             // [piece][row_cap][D]
    float2* part_ml;           // [piece][row_cap]
    uint2* row_parts;          // [row * hq + head]: its first piece, pieces | row of theirs << 16; the next piece is hkv on
    int32_t* own_first;        // [n_seq]: first key behind the group's shared ones
    const float* own_o;        // [row * hq + head][D], own_ml: the part of a request's own keys
    const float2* own_ml;
};

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
__device__ __forceinline__ void store4u(char* p, const float* v, float) {
    *reinterpret_cast<f4u*>(p) = f4u{v[0], v[1], v[2], v[3]};
}
__device__ __forceinline__ void store4u(char* p, const float* v, uint16_t) {
    *reinterpret_cast<h4u*>(p) = h4u{static_cast<_Float16>(v[0]), static_cast<_Float16>(v[1]), static_cast<_Float16>(v[2]),
                                     static_cast<_Float16>(v[3])};
}

__device__ __forceinline__ h4v read_turned(const char* lds) {
    typedef __attribute__((address_space(3))) s4v lds_s4;
    return __builtin_bit_cast(h4v, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(lds)));
}

// tanh without branches: an odd series below 1/2 (its next term is 2^-26 of the
// sum), 1 - 2 / (1 + exp 2x) above; 3 units in the last place.
__device__ __forceinline__ float tanh_of(float x) {
    const float y = fabsf(x), z = y * y;
    float p = fmaf(z, -929569.0f / 638512875.0f, 21844.0f / 6081075.0f);
    p = fmaf(z, p, -1382.0f / 155925.0f);
    p = fmaf(z, p, 62.0f / 2835.0f);
    p = fmaf(z, p, -17.0f / 315.0f);
    p = fmaf(z, p, 2.0f / 15.0f);
    p = fmaf(z, p, -1.0f / 3.0f);
    const float small = fmaf(y * z, p, y);
    const float e = __builtin_amdgcn_exp2f(y * (2.0f * kLog2e));
    const float large = 1.0f - 2.0f / (1.0f + e);
    return copysignf(y < 0.5f ? small : large, x);
}

// Row tiles: those of request (group) p, whose rows are start[p] * g on, are numbered from start[p] * g / ROWS + p on,
// which is one more than it needs at most, so that a tile is found without a sum over the requests before it.
__device__ __forceinline__ uint32_t start_of(const AttnArgs& a, uint32_t p) {
    const int32_t t = a.start[p];
    return t < 0 ? 0u : min(static_cast<uint32_t>(t), a.n_rows);
}
template <int ROWS> __device__ __forceinline__ uint32_t first_tile(const AttnArgs& a, uint32_t start, uint32_t p) { return start * a.g / ROWS + p; }

// Few row tiles: their keys are cut into pieces of one size, so that about `deal` workgroups have one each whatever the lengths, which
// only the device knows.  Every workgroup counts the key tiles of all row tiles for itself.
constexpr uint32_t kDealTiles = 1024;   // row tiles, requests at most
// Key tiles a piece at least: its rows' sums are written and read again (64 takes of 1150 shared keys: 44.8 us; 2: 43.9, 8: 49.5;
// 7 groups of up to 3500 over 8 bits 49.4; 2: 50.3, 8: 60.2).
constexpr int64_t kLeast = 4;
struct Piece {
    uint32_t first = 0, count = 1, at = 0;      // the row tile's first piece, how many it has, which of them
    uint32_t tile0 = 0, tiles = 0;              // key tiles

    uint32_t x = 0, p = 0, t0 = 0, t1 = 0;      // the row tile, its request (group), that one's tokens (requests)
    int32_t keys = 0;                           // and length (shared keys), as given

    // lds: 2 kDealTiles + 2 words
    template <int KT, int ROWS> __device__ __forceinline__ bool find(const PromptArgs& pa, uint32_t q, uint32_t* lds) {
        const AttnArgs& a = pa.a;
        constexpr int N = kDealTiles / 256;
        __shared__ uint32_t sums[4], found[8];
        const uint32_t tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
        int32_t* given = reinterpret_cast<int32_t*>(lds) + kDealTiles + 1;
        for (uint32_t i = tid; i <= pa.n_start; i += 256) {
            lds[i] = start_of(a, i);
            if (i < pa.n_start) given[i] = pa.shared ? pa.shared[i] : a.lens[i];
        }
        if (tid == 0) found[0] = ~0u;
        __syncthreads();
        uint32_t n_tiles[N], begin[N], whose[N], sum = 0;
#pragma unroll
        for (int i = 0; i < N; i++) {                        // pieces are numbered by threads, a thread's row tiles lie 256 apart
            const uint32_t xi = tid + 256 * i;
            n_tiles[i] = begin[i] = whose[i] = 0;
            if (xi >= pa.tiles) continue;
            uint32_t lo = 0, hi = pa.n_start;                // the last one whose tiles start at or before xi
            while (hi - lo > 1) {
                const uint32_t mid = (lo + hi) / 2;
                if (first_tile<ROWS>(a, lds[mid], mid) <= xi) lo = mid;
                else hi = mid;
            }
            const uint32_t from = lds[lo], to = lds[lo + 1], base = first_tile<ROWS>(a, from, lo);
            if (xi < base || to <= from || static_cast<uint64_t>(xi - base) * ROWS >= static_cast<uint64_t>(to - from) * a.g) continue;
            const uint32_t row0 = (xi - base) * ROWS, row1 = min(row0 + ROWS, (to - from) * a.g) - 1;
            const int32_t len = min(max(given[lo], 0), static_cast<int32_t>(a.max_pages * a.page));
            int32_t first = 0, end = len;
            if (!pa.shared) {
                auto limit = [&](uint32_t row) {
                    const int32_t j = static_cast<int32_t>((static_cast<uint64_t>(row) * pa.g_mul) >> pa.g_shift);
                    return max(0, len - (static_cast<int32_t>(to - from) - 1 - j));
                };
                end = limit(row1);
                if (a.window > 0) first = max(0, limit(row0) - a.window);
            }
            begin[i] = first / KT;
            const uint32_t behind = (static_cast<uint32_t>(end) + KT - 1) / KT;
            n_tiles[i] = max(1u, behind - min(begin[i], behind));
            whose[i] = lo;
            sum += n_tiles[i];
        }
        uint32_t all = sum;
#pragma unroll
        for (int d = 32; d > 0; d >>= 1) all += __shfl_xor(all, d);
        if (lane == 0) sums[wid] = all;
        __syncthreads();
        all = sums[0] + sums[1] + sums[2] + sums[3];
        __syncthreads();
        // key tiles a piece
        const uint32_t size = max(static_cast<uint32_t>(kLeast), static_cast<uint32_t>((static_cast<uint64_t>(all) * a.hkv + pa.deal - 1) / pa.deal));
        uint32_t pieces[N] = {};
        sum = 0;
#pragma unroll
        for (int i = 0; i < N; i++) {
            if (256u * i >= pa.tiles) break;
            pieces[i] = (n_tiles[i] + size - 1) / size;
            sum += pieces[i];
        }
        uint32_t before = sum;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const uint32_t y = __shfl_up(before, d);
            if (lane >= static_cast<uint32_t>(d)) before += y;
        }
        if (lane == 63) sums[wid] = before;
        __syncthreads();
        before -= sum;
        for (uint32_t w = 0; w < wid; w++) before += sums[w];
#pragma unroll
        for (int i = 0; i < N; i++) {
            const uint32_t n = pieces[i];
            if (q >= before && q - before < n) {
                found[0] = before;
                found[1] = n;
                found[2] = begin[i] + (q - before) * size;
                found[3] = tid + 256 * i;
                found[4] = whose[i];
                found[5] = lds[whose[i]];
                found[6] = lds[whose[i] + 1];
                found[7] = static_cast<uint32_t>(given[whose[i]]);
            }
            before += n;
        }
        __syncthreads();
        first = __builtin_amdgcn_readfirstlane(found[0]);
        if (first == ~0u) return false;
        count = __builtin_amdgcn_readfirstlane(found[1]);
        at = q - first;
        tile0 = __builtin_amdgcn_readfirstlane(found[2]);
        tiles = size;
        x = __builtin_amdgcn_readfirstlane(found[3]);
        p = __builtin_amdgcn_readfirstlane(found[4]);
        t0 = __builtin_amdgcn_readfirstlane(found[5]);
        t1 = __builtin_amdgcn_readfirstlane(found[6]);
        keys = __builtin_amdgcn_readfirstlane(static_cast<int>(found[7]));
        return true;
    }
};

// A tile of KT keys and values in LDS, and the products over it.  A wave holds
// 32 rows of q: S^T = K Q^T by 32 x 32 products, whose result has the lane's row
// lane % 32 and keys 8 (r / 4) + 4 (lane / 32) + r % 4; O^T = V^T P^T takes these
// as its B operand as they are (the sum over keys in any order, as long as V's
// come in the same one), V^T's columns by turning 4 x 16 blocks on the way out of
// LDS.  So a row's maximum and sum are its lane's, and nothing else crosses lanes.
//
// LDS holds rows of PITCH bytes as 16-byte chunks, chunk c of key r at place
// c ^ f(r): the 16 lanes that read together meet 16 different places of 256
// bytes.  F16 and F32 pages come there straight from memory (1 KiB a wave and
// instruction, lane l to byte 16 l: the lane asks for the chunk whose place
// that is), I8 ones through registers, where they are widened.
//
// F16 pages, and I8 ones as whole numbers: keys in f16; values in f16, of I8 pages
// in bf16, whose range holds a probability (up to 1) times any scale.
template <typename TC, int DP> struct Tile {
    static constexpr bool F32 = false, I8 = sizeof(TC) == 1;
    static constexpr int KT = DP <= 128 ? 64 : 32, PITCH = DP == 64 ? 128 : DP <= 128 ? 256 : 512;
    static constexpr int PER = I8 ? 16 : 8, LANES = PITCH / 2 / PER;     // elements in 16 bytes of a page, lanes that bring a row
    static __device__ __forceinline__ uint32_t k_place(uint32_t r, uint32_t c) { return DP == 64 ? c ^ (r >> 1 & 7) : c ^ (r & 15); }
    static __device__ __forceinline__ uint32_t v_place(uint32_t r, uint32_t c) { return DP == 64 ? c ^ (r >> 1 & 1) << 2 : c ^ (r & 3) << 2; }
};

// F32 pages: products of f32, 32 x 32 x 2.
template <int DP> struct Tile<float, DP> {
    static constexpr bool F32 = true, I8 = false;
    static constexpr int KT = 32, PITCH = DP == 64 ? 256 : DP <= 128 ? 512 : 1024;
    static constexpr int PER = 4, LANES = PITCH / 16;
    static __device__ __forceinline__ uint32_t k_place(uint32_t r, uint32_t c) { return c ^ (r & 15); }
    static __device__ __forceinline__ uint32_t v_place(uint32_t r, uint32_t c) { return c ^ (r >> 2 & 1) << 3; }
};

// A value made anew where it is asked for: what rare paths and the end work out again would else be kept, in registers, through the
// loop over the keys.
template <typename V> __device__ __forceinline__ V anew(V v) {
    asm volatile("" : "+v"(v));
    return v;
}
// The kernel's arguments read again, likewise.
typedef const __attribute__((address_space(4))) PromptArgs const_args;
__device__ __forceinline__ const_args* args_anew() {
    const_args* p = (const_args*)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    return p;
}

// What keys that are not there are read as.
static __device__ const uint4 g_zeros[64] = {};

// Workgroups of k_prompt that a CU holds, which their registers are limited to.
constexpr int waves_per_simd(int dp, bool f32) { return dp <= 64 && !f32 ? 3 : dp <= 128 ? 2 : 1; }

// PP: f16 (I8 pages: bf16) parts that a probability is split into.  CAP: capped scores.  PAIR: two waves share 32 rows, each with every
// other run of 32 keys (64 rows a workgroup); else each wave has 32 rows and all keys (128).
template <typename TQ, typename TC, int DP, int PP, bool CAP, bool PAIR>
__global__ __launch_bounds__(256, waves_per_simd(DP, sizeof(TC) == 4)) void k_prompt(PromptArgs pa) {
    using T = Tile<TC, DP>;
    constexpr bool F32 = T::F32, I8 = T::I8, Q2 = sizeof(TQ) == 4 && !F32;
    constexpr int ROWS = PAIR ? 64 : 128, KT = T::KT, PITCH = T::PITCH, LANES = T::LANES, BYTES = KT * PITCH, QC = DP / 16;
    constexpr int RPI = 64 / LANES, NI = KT / 4 / RPI;       // rows a wave brings at a time, times
    constexpr int NS = PAIR || KT == 32 || Q2 || DP == 64 ? 1 : 2;   // runs of 32 keys taken together
    // Probabilities are held times 2^kUp, and up to 2^(kUp + kRise), since the sums are rescaled only when a row's maximum has risen by
    // kRise powers of two.  F16 pages: what f16's 2^15 leaves, values being below 2^16.  A value in F32 or I8 may lie anywhere in f32's
    // range: probabilities up to 1, as in paged_attention.  Rescaling at every rise costs 1 to 6 % (F32, at 8 powers of two: 5 requests of
    // 300 to 1301 tokens, heads of 80, 356 us for 363, 1522 tokens, heads of 256, 755 for 801; I8, at one, drafts 99.6 for 100.8).
    constexpr bool WIDE = F32 || I8;
    constexpr float kUp = WIDE ? 0.0f : PP == 1 ? 9.0f : 14.0f, kRise = WIDE ? 0.0f : PP == 1 ? 6.0f : 1.0f;
    const AttnArgs& a = pa.a;
    // keys and values of one tile each; two arrays, so that reads of one are known to be apart from what is on its way into the other
    __shared__ __attribute__((aligned(16))) char lds0[2 * BYTES];
    __shared__ __attribute__((aligned(16))) char lds1[2 * BYTES];
    __shared__ __attribute__((aligned(16))) float lds_s[2][2][I8 ? KT : 4];
    __shared__ int32_t lds_ext[4][4];
    __shared__ float lds_pair[2 * 64 * 2];
    const uint32_t tid = threadIdx.x, lane = tid & 63, n = lane & 31, half = lane >> 5;
    const uint32_t wid = __builtin_amdgcn_readfirstlane(tid >> 6);

    // this workgroup's key head, row tile (undealt: the last rows, which have the most keys, first) and piece of its keys
    const uint32_t hk = blockIdx.x % a.hkv;
    uint32_t x = pa.tiles - 1 - blockIdx.x / a.hkv, p = 0, t0, t1;
    int32_t given = 0;                                       // the request's length, the group's shared keys
    Piece piece;
    if (pa.deal) {
        if (!piece.find<KT, ROWS>(pa, blockIdx.x / a.hkv, reinterpret_cast<uint32_t*>(lds0))) return;
        x = piece.x;
        p = piece.p;
        t0 = piece.t0;
        t1 = piece.t1;
        given = piece.keys;
    } else {
        // the request p whose tiles x lies among; what is read with it in one go: where it and the next one start, and its length
        for (uint32_t width = pa.n_start;;) {                // p among [p, p + width)
            const uint32_t step = (width + 63) / 64, q = min(p + lane * step, pa.n_start - 1);
            const uint32_t from = start_of(a, q), to = start_of(a, q + 1);
            const int32_t len = a.lens[q];
            const bool in = lane * step < width && first_tile<ROWS>(a, from, q) <= x;
            const uint32_t at = 64 - __builtin_clzll(__ballot(in) | 1) - 1;
            p = __builtin_amdgcn_readfirstlane(p + at * step);
            width = min(step, width - min(width, at * step));
            t0 = __builtin_amdgcn_readlane(static_cast<int>(from), at);
            t1 = __builtin_amdgcn_readlane(static_cast<int>(to), at);
            given = __builtin_amdgcn_readlane(len, at);
            if (step == 1) break;
        }
    }
    const uint32_t base = first_tile<ROWS>(a, t0, p);
    if (x < base || t1 <= t0 || static_cast<uint64_t>(x - base) * ROWS >= static_cast<uint64_t>(t1 - t0) * a.g) return;
    const uint32_t row0 = (x - base) * ROWS, rows = min(static_cast<uint32_t>(ROWS), (t1 - t0) * a.g - row0);
    const uint32_t row_wave = PAIR ? wid & 1 : wid, turn = wid >> 1;

    // the lane's row: row r of the tile, of token or request t and query head hq, keys [first, limit)
    const int32_t cap = static_cast<int32_t>(a.max_pages * a.page);
    auto row_of = [&](uint32_t r, uint32_t* t, uint32_t* hq) {
        const uint32_t ri = row0 + (r < rows ? r : 0), j = static_cast<uint32_t>((static_cast<uint64_t>(ri) * pa.g_mul) >> pa.g_shift);
        *t = t0 + j;
        *hq = hk * a.g + (ri - j * a.g);
    };
    const bool live_row = row_wave * 32 + n < rows;
    bool wrong;
    int32_t limit, first;
    // keys that any row of the workgroup has, that all of them have; those of the wave's rows
    int32_t begin, end, every_begin, every_end, w_begin, w_end, all_begin, all_end;
    const uint32_t seq = pa.shared ? t0 : p;                 // whose table
    const uint32_t lane_row = live_row ? row_wave * 32 + n : rows - 1;
    auto first_of = [&](int32_t lim) { return a.window > 0 && lim > a.window ? lim - a.window : 0; };
    if (pa.shared) {
        uint32_t t, hq;
        row_of(lane_row, &t, &hq);
        const int32_t all = a.lens[t], len = min(max(all, 0), cap), pre = min(max(given, 0), cap);
        wrong = all < 0 || all > cap;
        first = first_of(len);
        limit = min(len, pre);
        if (hk == 0 && piece.at == 0 && half == 0 && live_row && wid == row_wave) pa.own_first[t] = limit;
        if (!live_row) limit = first = 0;
        w_end = limit;
        w_begin = limit > first ? first : 0x7fffffff;
        all_end = live_row ? limit : 0x7fffffff;
        all_begin = first;
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
            w_end = max(w_end, __shfl_xor(w_end, d));
            w_begin = min(w_begin, __shfl_xor(w_begin, d));
            all_end = min(all_end, __shfl_xor(all_end, d));
            all_begin = max(all_begin, __shfl_xor(all_begin, d));
        }
        w_end = __builtin_amdgcn_readfirstlane(w_end);
        w_begin = __builtin_amdgcn_readfirstlane(w_begin);
        all_end = __builtin_amdgcn_readfirstlane(all_end);
        all_begin = __builtin_amdgcn_readfirstlane(all_begin);
        if (lane == 0) {
            lds_ext[0][wid] = w_end;
            lds_ext[1][wid] = w_begin;
            lds_ext[2][wid] = all_end;
            lds_ext[3][wid] = all_begin;
        }
        __syncthreads();
        end = max(max(lds_ext[0][0], lds_ext[0][1]), max(lds_ext[0][2], lds_ext[0][3]));
        begin = min(min(lds_ext[1][0], lds_ext[1][1]), min(lds_ext[1][2], lds_ext[1][3]));
        every_end = min(min(lds_ext[2][0], lds_ext[2][1]), min(lds_ext[2][2], lds_ext[2][3]));
        every_begin = max(max(lds_ext[3][0], lds_ext[3][1]), max(lds_ext[3][2], lds_ext[3][3]));
    } else {
        // limits rise with the rows
        wrong = given < 0 || given > cap;
        const int32_t len = min(max(given, 0), cap), behind = static_cast<int32_t>(t1 - t0) - 1;
        auto limit_of = [&](uint32_t r) {
            return max(0, len - (behind - static_cast<int32_t>((static_cast<uint64_t>(row0 + r) * pa.g_mul) >> pa.g_shift)));
        };
        limit = live_row ? limit_of(lane_row) : 0;
        first = first_of(limit);
        const uint32_t ra = row_wave * 32, rb = min(ra + 31, rows - 1);
        every_end = limit_of(0);
        end = limit_of(rows - 1);
        begin = first_of(every_end);
        every_begin = first_of(end);
        all_end = w_end = 0;
        all_begin = w_begin = 0;
        if (ra < rows) {
            all_end = limit_of(ra);
            w_end = limit_of(rb);
            w_begin = first_of(all_end);
            all_begin = first_of(w_end);
        }
    }
    begin = __builtin_amdgcn_readfirstlane(min(begin, end));
    end = __builtin_amdgcn_readfirstlane(end);
    const uint32_t tile0 = static_cast<uint32_t>(begin) / KT, n_tiles = (static_cast<uint32_t>(end) + KT - 1) / KT - tile0;
    uint32_t ta = tile0, tb = tile0 + n_tiles;
    if (pa.deal) {
        ta = max(ta, piece.tile0);
        tb = min(tb, piece.tile0 + piece.tiles);
    }
    ta = __builtin_amdgcn_readfirstlane(ta);
    tb = __builtin_amdgcn_readfirstlane(tb);

    // A tile on its way to LDS.  Each lane looks its key lane % KT up and works out where it lies, the lanes that bring it ask for that:
    // where the rows that they bring together lie in one page, at an offset of the wave's and one of their own that stays.  Keys that
    // are not there are brought from a row of zeros; the places of dims past D get the row's first ones again, which the query meets with
    // zeros and whose sums of values nobody asks for.
    const int32_t* table = reinterpret_cast<const int32_t*>(a.tables + seq * a.t_nb1);
    auto look_up = [&](uint32_t tile) { return table[min(page_of(a, tile * KT + (lane & (KT - 1))), a.max_pages - 1)]; };
    u4v rk[I8 ? NI : 1], rv[I8 ? NI : 1];
    float rs = 0.0f;
    uint64_t have = 0, have_next = 0;                        // keys of the tile that are there
    constexpr uint64_t ALL = KT == 64 ? ~0ull : 0xffffffffull;
    const uint32_t sub_row = lane / LANES, sub_c = lane % LANES;
    const char *kb = a.k + hk * a.k_nb2, *vb = a.v + hk * a.v_nb2;
    const bool together = a.page % RPI == 0;
    auto chunk = [&](uint32_t c) { return c * T::PER < a.D ? c * 16 : 0; };
    auto fetch = [&](uint32_t tile, int32_t pg, char* to) __attribute__((always_inline)) {
        const uint32_t key = tile * KT + (lane & (KT - 1));
        const bool in = key < static_cast<uint32_t>(end) && key >= static_cast<uint32_t>(begin);
        const bool good = static_cast<uint32_t>(pg) < a.n_pages;
        wrong |= in && !good;
        have_next = __ballot(in && good) & ALL;
        const uint32_t at = key - page_of(a, key) * a.page;
        uint64_t ko = static_cast<uint64_t>(pg * a.k_nb3 + at * a.k_nb1), vo = static_cast<uint64_t>(pg * a.v_nb3 + at * a.v_nb1);
        typedef __attribute__((address_space(3))) void lds_void;
        typedef const __attribute__((address_space(1))) void global_void;
        char* l = to + wid * NI * 1024;
        if (!I8 && together && have_next == ALL) {
#pragma unroll
            for (int i = 0; i < NI; i++) {
                const int src = wid * (KT / 4) + i * RPI;
                const uint32_t row = src + sub_row;
                auto of = [&](uint64_t o) {
                    const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(static_cast<uint32_t>(o)), src);
                    const uint32_t hi = __builtin_amdgcn_readlane(static_cast<int>(static_cast<uint32_t>(o >> 32)), src);
                    return static_cast<uint64_t>(hi) << 32 | lo;
                };
                const char *kw = kb + of(ko), *vw = vb + of(vo);
                asm volatile("" : "+s"(kw), "+s"(vw));       // bases of the wave's, the lane's offset beside them
                const uint32_t kl = sub_row * static_cast<uint32_t>(a.k_nb1) + chunk(T::k_place(row, sub_c));
                const uint32_t vl = sub_row * static_cast<uint32_t>(a.v_nb1) + chunk(T::v_place(row, sub_c));
                __builtin_amdgcn_global_load_lds((global_void*)(kw + kl), (lds_void*)(l + i * 1024), 16, 0, 0);
                __builtin_amdgcn_global_load_lds((global_void*)(vw + vl), (lds_void*)(l + BYTES + i * 1024), 16, 0, 0);
            }
            return;
        }
        if (!in || !good) {
            ko = reinterpret_cast<uintptr_t>(g_zeros) - reinterpret_cast<uintptr_t>(kb);
            vo = reinterpret_cast<uintptr_t>(g_zeros) - reinterpret_cast<uintptr_t>(vb);
        }
        const uint32_t lane1 = I8 ? lane : anew(lane), sub_row = lane1 / LANES, sub_c = lane1 % LANES;
#pragma unroll
        for (int i = 0; i < NI; i++) {
            const uint32_t row = wid * (KT / 4) + i * RPI + sub_row;
            auto of = [&](uint64_t o) {
                const uint32_t lo = __shfl(static_cast<int>(static_cast<uint32_t>(o)), row);
                const uint32_t hi = __shfl(static_cast<int>(static_cast<uint32_t>(o >> 32)), row);
                return static_cast<uint64_t>(hi) << 32 | lo;
            };
            const char *kw = kb + of(ko), *vw = vb + of(vo);
            if constexpr (I8) {
                rk[i] = *reinterpret_cast<const u4v*>(kw + chunk(sub_c));
                rv[i] = *reinterpret_cast<const u4v*>(vw + chunk(sub_c));
            } else {
                __builtin_amdgcn_global_load_lds((global_void*)(kw + chunk(T::k_place(row, sub_c))), (lds_void*)(l + i * 1024), 16, 0, 0);
                __builtin_amdgcn_global_load_lds((global_void*)(vw + chunk(T::v_place(row, sub_c))), (lds_void*)(l + BYTES + i * 1024), 16, 0, 0);
            }
        }
        if constexpr (I8) {
            if (wid < 2 && in && good) {
                const char* sp = wid == 0 ? a.ks + pg * a.ks_nb2 + hk * a.ks_nb1 + at * a.ks_nb0
                                          : a.vs + pg * a.vs_nb2 + hk * a.vs_nb1 + at * a.vs_nb0;
                rs = *reinterpret_cast<const float*>(sp);
            } else {
                rs = 0.0f;
            }
        }
    };
    // The tile in LDS, as far as this wave brings it.  Edge tiles, some of whose keys some rows do not have: values that are no numbers
    // are found there, and cleared once `clean`.
    bool clean = false, bad = false;
    auto arrive = [&](char* to, int buf, bool edge) __attribute__((always_inline)) {
        if constexpr (I8) {
#pragma unroll
            for (int i = 0; i < NI; i++) {
                const uint32_t row = wid * (KT / 4) + i * RPI + sub_row;
                // keys: 1024 + 128 + x is a half with x + 128 in its low byte
                u4v k[2], v[2];
#pragma unroll
                for (int w = 0; w < 4; w++) {
                    const uint32_t y = rk[i][w] ^ 0x80808080u;
#pragma unroll
                    for (int b = 0; b < 2; b++) {
                        const h2v t = __builtin_bit_cast(h2v, __builtin_amdgcn_perm(0x64646464u, y, b ? 0x04030402u : 0x04010400u));
                        const int at = 2 * (w & 1) + b;
                        k[w / 2][at] = __builtin_bit_cast(uint32_t, t - h2v{static_cast<_Float16>(1152), static_cast<_Float16>(1152)});
                        const float f0 = static_cast<float>(static_cast<int8_t>(rv[i][w] >> 16 * b));
                        const float f1 = static_cast<float>(static_cast<int8_t>(rv[i][w] >> (16 * b + 8)));
                        v[w / 2][at] = __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, f1), __builtin_bit_cast(uint32_t, f0), 0x07060302u);
                    }
                }
                char *lk = to + row * PITCH, *lv = lk + BYTES;
                *reinterpret_cast<u4v*>(lk + T::k_place(row, 2 * sub_c) * 16) = k[0];
                *reinterpret_cast<u4v*>(lk + T::k_place(row, 2 * sub_c + 1) * 16) = k[1];
                *reinterpret_cast<u4v*>(lv + T::v_place(row, 2 * sub_c) * 16) = v[0];
                *reinterpret_cast<u4v*>(lv + T::v_place(row, 2 * sub_c + 1) * 16) = v[1];
            }
            if (wid < 2 && lane < KT) lds_s[buf][wid][lane] = rs;
        } else {
            wait_vector_memory();                            // what this wave brings to LDS
            if (a.D != DP) {                                 // an infinity past D would make NaN of the query's zeros
                constexpr uint32_t R = KT / 4;               // rows that this wave brings
                const uint32_t lane1 = anew(lane), row = wid * R + lane1 % R;
#pragma unroll 1
                for (uint32_t c = a.D / T::PER + lane1 / R; c < DP / T::PER; c += 64 / R) {
                    *reinterpret_cast<u4v*>(to + row * PITCH + T::k_place(row, c) * 16) = anew(u4v{});
                }
            }
            if (edge) {
#pragma unroll 1
                for (int i = 0; i < NI; i++) {
                    u4v* at = reinterpret_cast<u4v*>(to + BYTES + (wid * NI + i) * 1024 + anew(lane) * 16);
                    u4v v = *at;
                    bool any = false;
#pragma unroll
                    for (int w = 0; w < 4; w++) {
                        const uint32_t y = v[w];
                        if constexpr (F32) {
                            const bool no = (y & 0x7f800000u) == 0x7f800000u;
                            any |= no;
                            v[w] = no ? 0u : y;
                        } else {
                            const bool lo = (y & 0x7c00u) == 0x7c00u, hi = (y & 0x7c000000u) == 0x7c000000u;
                            any |= lo || hi;
                            v[w] = (lo ? 0u : y & 0xffffu) | (hi ? 0u : y & 0xffff0000u);
                        }
                    }
                    bad |= any;
                    if (clean && any) *at = v;
                }
            }
        }
    };

    // the first tile is on its way while the query is read
    int32_t pg = 0, pg1 = 0;
    if (ta < tb) {
        pg = look_up(ta);
        pg1 = look_up(ta + 1);
        fetch(ta, pg, lds0);
    }

    // the lane's query: dims 16 c + 8 half + [0, 8), for F32 pages 8 c + 4 half + [0, 4).  Over other pages an F32 one is scaled by a
    // power of two to below 2^15 and split into two f16, the lower times 2^12 and summed apart
    h8v qh[F32 ? 1 : QC], ql[Q2 ? QC : 1];
    float qf[F32 ? QC * 8 : 1];
    float mul = fabsf(a.scale) * kLog2e;
    {
        float v[QC * 8];
        uint32_t t, hq;
        row_of(row_wave * 32 + n, &t, &hq);
        const char* qr = a.q + t * a.q_nb2 + hq * a.q_nb1;
#pragma unroll
        for (int i = 0; i < QC * 8; i += 4) {
            const uint32_t d = F32 ? 2 * i + 4 * half : 16 * (i / 8) + 8 * half + i % 8;
            const bool in = live_row && d < a.D;
            float tmp[4];
            load4u(qr + (in ? d : 0) * Elt<TQ>::size, tmp, TQ());
#pragma unroll
            for (int u = 0; u < 4; u++) v[i + u] = in ? (a.scale < 0.0f ? -tmp[u] : tmp[u]) : 0.0f;
        }
        if constexpr (Q2) {
            float m = 0.0f;
#pragma unroll
            for (int i = 0; i < QC * 8; i++) m = fmaxf(m, fabsf(v[i]));
            m = fmaxf(m, __shfl_xor(m, 32));
            int e = m > 0.0f && m < INFINITY ? static_cast<int>(__builtin_bit_cast(uint32_t, m) >> 23) - 127 : 14;
            e = e < -100 ? -100 : e;
            mul *= ldexpf(1.0f, e - 14);
            const float up = ldexpf(1.0f, 14 - e);
#pragma unroll
            for (int i = 0; i < QC * 8; i++) {
                const float y = v[i] * up;
                const _Float16 h = static_cast<_Float16>(y);
                qh[i / 8][i % 8] = h;
                ql[i / 8][i % 8] = static_cast<_Float16>((y - static_cast<float>(h)) * 4096.0f);
            }
        } else if constexpr (F32) {
#pragma unroll
            for (int i = 0; i < QC * 8; i++) qf[i] = v[i];
        } else {
#pragma unroll
            for (int i = 0; i < QC * 8; i++) qh[i / 8][i % 8] = static_cast<_Float16>(v[i]);
        }
    }
    float cap_in = 0.0f;
    if constexpr (CAP) {
        cap_in = fminf(mul / kLog2e / a.softcap, 0x1p127f);  // finite: 0 stays 0
        mul = 1.0f;
    }
    mul = fmaxf(mul, 0x1p-149f);                             // -inf, the score of a key that a row does not have, stays that

    f16v o[DP / 32];
    float m, mc, l;
    bool far;                                                // a maximum so large that its rounding would be a factor

    // LDS addresses that a lane reads keys and values at
    const uint32_t k_row = n * PITCH;
    // the swizzle stays within 16 chunks, so that 8 addresses and constants beside them do
    auto k_at = [&](int c) { return k_row + (T::k_place(n, 2 * (c % 8) + half) + 16 * (c / 8)) * 16; };
    const uint32_t l16 = lane & 15, v_key = 4 * half + l16 / 4, v_c = 2 * (lane >> 4 & 1) + (l16 >> 1 & 1);
    const uint32_t v_at = v_key * PITCH + (l16 & 1) * 8;

    // NS runs of 32 keys, from the tile's run `sub` on
    auto products = [&](const char* tile_lds, int buf, uint32_t key0, int sub) __attribute__((always_inline)) {
        const char* lk = tile_lds + sub * 32 * PITCH;
        const char* lv = lk + BYTES;
        f16v s[NS];
#pragma unroll
        for (int i = 0; i < NS; i++) s[i] = f16v{};
        if constexpr (F32) {
#pragma unroll
            for (int c = 0; c < DP / 8; c++) {
                const f4v kf = *reinterpret_cast<const f4v*>(lk + k_at(c));
#pragma unroll
                for (int u = 0; u < 4; u++) s[0] = __builtin_amdgcn_mfma_f32_32x32x2f32(kf[u], qf[4 * c + u], s[0], 0, 0, 0);
            }
            constexpr int A = 4;
            __builtin_amdgcn_sched_group_barrier(0x100, A, 0);
#pragma unroll
            for (int c = 0; c < DP / 8; c++) {
                __builtin_amdgcn_sched_group_barrier(0x008, 4, 0);
                if (c + A < DP / 8) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            }
        } else {
            f16v low = {};
            constexpr int A = 4;                             // reads ahead of their products
            h8v kf[NS][QC];
#pragma unroll
            for (int i = 0; i < NS; i++) {
#pragma unroll
                for (int c = 0; c < QC; c++) {
                    kf[i][c] = *reinterpret_cast<const h8v*>(lk + i * 32 * PITCH + k_at(c));
                }
            }
#pragma unroll
            for (int i = 0; i < NS; i++) {
#pragma unroll
                for (int c = 0; c < QC; c++) {
                    s[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[i][c], qh[c], s[i], 0, 0, 0);
                    if constexpr (Q2) low = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[i][c], ql[c], low, 0, 0, 0);
                }
            }
            __builtin_amdgcn_sched_group_barrier(0x100, A, 0);
#pragma unroll
            for (int c = 0; c < NS * QC; c++) {
                __builtin_amdgcn_sched_group_barrier(0x008, Q2 ? 2 : 1, 0);
                if (c + A < NS * QC) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            }
            if constexpr (Q2) {
#pragma unroll
                for (int e = 0; e < 16; e++) s[0][e] = fmaf(low[e], 0x1p-12f, s[0][e]);
            }
        }
#pragma unroll
        for (int i = 0; i < NS; i++) {
            if constexpr (I8) {
#pragma unroll
                for (int e = 0; e < 16; e += 4) {
                    const f4v sc = *reinterpret_cast<const f4v*>(&lds_s[buf][0][32 * (sub + i) + 2 * e + 4 * half]);
#pragma unroll
                    for (int u = 0; u < 4; u++) s[i][e + u] *= sc[u];
                }
            }
            if constexpr (CAP) {
#pragma unroll
                for (int e = 0; e < 16; e++) s[i][e] = tanh_of(s[i][e] * cap_in) * (a.softcap * kLog2e);
            }
        }
        constexpr uint64_t EACH = NS == 2 ? ~0ull : 0xffffffffull;
        const uint64_t there = have >> 32 * sub & EACH;
        const bool whole = key0 >= static_cast<uint32_t>(all_begin) && key0 + 32 * NS <= static_cast<uint32_t>(all_end) && there == EACH;
        // bit 8 (e / 4) + e % 4: the lane's row has the key of its score e in run i
        auto below = [](int32_t n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1; };
        auto has = [&](int i) {
            const uint32_t at = key0 + 32 * i + 4 * half;
            return static_cast<uint32_t>(there >> 32 * i) >> 4 * half & below(static_cast<int32_t>(limit - at)) &
                   ~below(static_cast<int32_t>(first - at));
        };
        if (!whole) {
#pragma unroll
            for (int i = 0; i < NS; i++) {
                const uint32_t live = has(i);
#pragma unroll
                for (int e = 0; e < 16; e++) s[i][e] = live & 1u << (8 * (e / 4) + e % 4) ? s[i][e] : -INFINITY;
            }
        }
        float mx = s[0][0];
#pragma unroll
        for (int i = 0; i < NS; i++) {
#pragma unroll
            for (int e = i == 0 ? 1 : 0; e < 16; e++) mx = fmaxf(mx, s[i][e]);
        }
        auto rises = [&] { return mx > m && (m == kLowest || (mx - m) * mul > kRise); };
        if (__any(rises())) {                                // rare after the first keys: the row's sums are rescaled
            mx = fmaxf(mx, __shfl_xor(mx, 32));
            if (rises()) {                                   // of this row alone: its neighbours' keys say nothing about it
                const float mc2 = fmaf(mx, mul, -kUp);
                const bool big = fabsf(mc2) >= 0x1p22f;
                const float keep = far || big ? __builtin_amdgcn_exp2f((m - mx) * mul) : __builtin_amdgcn_exp2f(mc - mc2);
                far |= big;
                m = mx;
                mc = mc2;
                l *= keep;
#pragma unroll
                for (int d = 0; d < DP / 32; d++) o[d] *= keep;
            }
        }
        float add = -mc;
        if (__any(far)) {                                    // the maximum off first
            const float off = far ? m : 0.0f;
            add = far ? kUp : add;
#pragma unroll
            for (int i = 0; i < NS; i++) {
#pragma unroll
                for (int e = 0; e < 16; e++) s[i][e] -= off;
            }
        }
#pragma unroll
        for (int i = 0; i < NS; i++) {
#pragma unroll
            for (int e = 0; e < 16; e++) s[i][e] = __builtin_amdgcn_exp2f(fmaf(s[i][e], mul, add));
            if constexpr (I8 || F32 || PP == 2) {
#pragma unroll
                for (int e = 0; e < 16; e++) l += s[i][e];
            }
            if constexpr (I8) {
#pragma unroll
                for (int e = 0; e < 16; e += 4) {
                    const f4v sc = *reinterpret_cast<const f4v*>(&lds_s[buf][1][32 * (sub + i) + 2 * e + 4 * half]);
#pragma unroll
                    for (int u = 0; u < 4; u++) s[i][e + u] *= sc[u];
                }
                if (!whole) {                                // the scale of a key that the row does not have may be no number
                    const uint32_t live = has(i);
#pragma unroll
                    for (int e = 0; e < 16; e++) s[i][e] = live & 1u << (8 * (e / 4) + e % 4) ? s[i][e] : 0.0f;
                }
            }
        }
        // O^T += V^T P^T
        if constexpr (F32) {
#pragma unroll
            for (int e = 0; e < 16; e++) {
                const uint32_t key = 8 * (e / 4) + 4 * half + e % 4;
#pragma unroll
                for (int d = 0; d < DP / 32; d++) {
                    const char* at = lv + key * PITCH + (T::v_place(4 * half, 8 * (d % 2) + n / 4) + 16 * (d / 2)) * 16 + n % 4 * 4;
                    const float v = *reinterpret_cast<const float*>(at);
                    o[d] = __builtin_amdgcn_mfma_f32_32x32x2f32(v, s[0][e], o[d], 0, 0, 0);
                }
                if (e % 2 == 1) __builtin_amdgcn_sched_barrier(0);   // else every value of the 16 keys is held at once
            }
            return;
        }
#pragma unroll
        for (int u = 0; u < 2 * NS && !F32; u++) {           // 16 keys
            f16v& su = s[u / 2];
            h8v ph, pl;
            b8v pb[3];
            if constexpr (I8) {
#pragma unroll
                for (int k = 0; k < PP; k++) {
                    u4v w;
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int e = 8 * (u % 2) + 2 * i;
                        const uint32_t z0 = __builtin_bit_cast(uint32_t, static_cast<float>(su[e]));
                        const uint32_t z1 = __builtin_bit_cast(uint32_t, static_cast<float>(su[e + 1]));
                        w[i] = __builtin_amdgcn_perm(z1, z0, 0x07060302u);
                        su[e] -= __builtin_bit_cast(float, z0 & 0xffff0000u);
                        su[e + 1] -= __builtin_bit_cast(float, z1 & 0xffff0000u);
                    }
                    pb[k] = __builtin_bit_cast(b8v, w);
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const float y = su[8 * (u % 2) + i];
                    ph[i] = static_cast<_Float16>(y);
                    if constexpr (PP == 2) pl[i] = static_cast<_Float16>(y - static_cast<float>(ph[i]));
                }
                if constexpr (PP == 1) {
#pragma unroll
                    for (int i = 0; i < 8; i += 2) l = __builtin_amdgcn_fdot2(h2v{ph[i], ph[i + 1]}, h2v{1, 1}, l, false);
                }
            }
            h8v vf[DP / 32];
#pragma unroll
            for (int d = 0; d < DP / 32; d++) {
                // place of chunk 4 d + v_c in the lane's rows: these are alike modulo 4
                const char* at = lv + v_at + (T::v_place(v_key, 4 * (d % 4) + v_c) + 16 * (d / 4)) * 16 + 16 * u * PITCH;
                const h4v x0 = read_turned(at), x1 = read_turned(at + 8 * PITCH);
                vf[d] = h8v{x0[0], x0[1], x0[2], x0[3], x1[0], x1[1], x1[2], x1[3]};
            }
#pragma unroll
            for (int d = 0; d < DP / 32; d++) {
                if constexpr (I8) {
#pragma unroll
                    for (int k = PP - 1; k >= 0; k--) {
                        o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8v, vf[d]), pb[k], o[d], 0, 0, 0);
                    }
                } else {
                    if constexpr (PP == 2) o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf[d], pl, o[d], 0, 0, 0);
                    o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf[d], ph, o[d], 0, 0, 0);
                }
            }
        }
        if constexpr (NS == 1) {
            // the first reads, then products for every read
            constexpr int ND = DP / 32 < 4 ? DP / 32 : 4;
            __builtin_amdgcn_sched_group_barrier(0x100, 2 * ND, 0);
#pragma unroll
            for (int i = 0; i < 2 * (DP / 32); i++) {
                __builtin_amdgcn_sched_group_barrier(0x008, PP, 0);
                if (i + ND < 2 * (DP / 32)) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
            }
        }
    };

    // A value that is no number, at a key that some of the rows do not have, would reach these as 0 times it: met at such a tile, the
    // keys are gone through once more without them, and the rows that have them get them at the end.
    for (;;) {
#pragma unroll
        for (int d = 0; d < DP / 32; d++) o[d] = f16v{};
        m = mc = kLowest;
        l = 0.0f;
        far = false;
        if (ta < tb) {
            auto edge = [&](uint32_t tile) {
                return tile * KT < static_cast<uint32_t>(every_begin) || tile * KT + KT > static_cast<uint32_t>(every_end);
            };
            if (clean) fetch(ta, look_up(ta), lds0);
            arrive(lds0, 0, edge(ta));
            pg = pg1;
            have = have_next;
            auto step = [&](uint32_t tile, char* cur, char* next, int buf) __attribute__((always_inline)) {
                const bool more = tile + 1 < tb;
                __syncthreads();                             // cur is there, and next is done with
                if (more) {
                    fetch(tile + 1, pg, next);
                    pg = look_up(tile + 2);
                }
#pragma unroll
                for (int sub = 0; sub < KT / 32; sub += NS) {
                    const uint32_t k0 = tile * KT + 32 * sub;
                    if (PAIR && (k0 >> 5 & 1) != turn) continue;
                    if (k0 < static_cast<uint32_t>(w_end) && k0 + 32 * NS > static_cast<uint32_t>(w_begin)) products(cur, buf, k0, sub);
                }
                if (more) arrive(next, buf ^ 1, edge(tile + 1));
                have = have_next;
            };
            for (uint32_t tile = ta; tile < tb; tile += 2) {
                step(tile, lds0, lds1, 0);
                if (tile + 1 < tb) step(tile + 1, lds1, lds0, 1);
            }
        }
        if constexpr (I8) break;
        if (clean || !__syncthreads_or(bad)) break;
        clean = true;
    }
    l += __shfl_xor(l, 32);
    if (__any(wrong) && lane == 0) atomicOr(a.err, DEV_ERR_PAGE);
    // Parts that are joined: o and l as sums of 2^(s mul - m mul), beside m mul rounded once, as paged_attention's are (the sums of a
    // group's shared keys meet those).  mc, m mul - kUp rounded, would count a part of scores past 2^22 for another power of two.
    const bool to_parts = pa.shared || piece.count > 1;
    if (PAIR || to_parts) {
        const bool none = m == kLowest;
        const float down = none ? 1.0f : __builtin_amdgcn_exp2f(far ? -kUp : -fmaf(m, mul, -mc));
        mc = none ? kLowest : m * mul;
        l *= down;
#pragma unroll
        for (int d = 0; d < DP / 32; d++) o[d] *= down;
    }
    if constexpr (PAIR) {                                    // the two waves' parts added up, ND runs of 32 dims at a time
        constexpr int ND = 2 * BYTES / 8192 < DP / 32 ? 2 * BYTES / 8192 : DP / 32;
        float* part = reinterpret_cast<float*>(lds0) + row_wave * (ND * 16 * 64) + lane;
        float2* ml = reinterpret_cast<float2*>(lds_pair) + row_wave * 64 + lane;
        float f0 = 0.0f, f1 = 0.0f;
#pragma unroll
        for (int d0 = 0; d0 < DP / 32; d0 += ND) {
            __syncthreads();
            if (turn == 1) {
                *ml = make_float2(mc, l);
#pragma unroll
                for (int d = 0; d < ND && d0 + d < DP / 32; d++) {
#pragma unroll
                    for (int e = 0; e < 16; e++) part[(16 * d + e) * 64] = o[d0 + d][e];
                }
            }
            __syncthreads();
            if (turn == 0) {
                if (d0 == 0) {
                    const float2 other = *ml;
                    const float m2 = fmaxf(mc, other.x);
                    f0 = __builtin_amdgcn_exp2f(mc - m2);
                    f1 = __builtin_amdgcn_exp2f(other.x - m2);
                    mc = m2;
                    l = fmaf(l, f0, other.y * f1);
                }
#pragma unroll
                for (int d = 0; d < ND && d0 + d < DP / 32; d++) {
#pragma unroll
                    for (int e = 0; e < 16; e++) o[d0 + d][e] = fmaf(o[d0 + d][e], f0, part[(16 * d + e) * 64] * f1);
                }
            }
        }
    }
    if (wid != row_wave) return;
    const_args& late = *args_anew();
    const uint32_t lane1 = anew(lane), n1 = lane1 & 31, half1 = lane1 >> 5, r = row_wave * 32 + n1, D = late.a.D;
    const uint32_t slot = piece.first * late.a.hkv + hk;     // of the row tile's first piece
    const uint64_t part0 = static_cast<uint64_t>(slot + piece.at * late.a.hkv) * late.row_cap;
    if (r < rows) {
        uint32_t t, hq;
        row_of(r, &t, &hq);
        if (late.deal && half1 == 0) {
            if (piece.at == 0) late.row_parts[static_cast<uint64_t>(t) * late.a.hq + hq] = make_uint2(slot, piece.count | r << 16);
            if (to_parts) late.part_ml[part0 + r] = make_float2(mc, l);
        }
        char* yr = to_parts ? reinterpret_cast<char*>(late.part_o + (part0 + r) * D) : late.a.y + t * late.a.y_nb2 + hq * late.a.y_nb1;
        const float f = to_parts ? 1.0f : l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
        for (int d = 0; d < DP / 32; d++) {
#pragma unroll
            for (int c = 0; c < 4; c++) {
                const uint32_t dim = 32 * d + 8 * c + 4 * half1;
                if (dim >= D) continue;
                float v[4];
#pragma unroll
                for (int u = 0; u < 4; u++) v[u] = o[d][4 * c + u] * f;
                if (to_parts) store4u(yr + dim * 4, v, float());
                else store4u(yr + dim * Elt<TQ>::size, v, TQ());
            }
        }
    }
    if constexpr (!I8) {
        if (!clean) return;
        wait_vector_memory();                                // what this wave wrote above is corrected
#pragma unroll 1
        for (int i = 0; i < 32; i++) {                       // a row at a time, its dims over the lanes
            const uint32_t ri = row_wave * 32 + i;
            if (ri >= rows) break;
            const uint32_t lim = min(static_cast<uint32_t>(__shfl(limit, i)), tb * KT);
            const uint32_t from = max(static_cast<uint32_t>(__shfl(first, i)), ta * KT);
            uint32_t t, hq;
            row_of(ri, &t, &hq);
            uint32_t found[DP / 64 + 1] = {};                // 1, 2, 4: infinity, -infinity, NaN
            for (uint32_t key = from; key < lim; key++) {
                const uint32_t pi = page_of(a, key);
                const int32_t pg = table[pi];
                if (static_cast<uint32_t>(pg) >= a.n_pages) continue;
                const char* vr = a.v + pg * a.v_nb3 + hk * a.v_nb2 + (key - pi * a.page) * a.v_nb1;
#pragma unroll
                for (int k = 0; k < DP / 64 + 1; k++) {
                    const uint32_t d = lane1 + 64 * k;
                    if (d >= D) continue;
                    const float y = Elt<TC>::load1(vr + d * Elt<TC>::size);
                    if (!(fabsf(y) < INFINITY)) found[k] |= y > 0.0f ? 1 : y < 0.0f ? 2 : 4;
                }
            }
#pragma unroll
            for (int k = 0; k < DP / 64 + 1; k++) {
                const uint32_t d = lane1 + 64 * k;
                if (d >= D || !found[k]) continue;
                const float y = found[k] == 1 ? INFINITY : found[k] == 2 ? -INFINITY : NAN;
                if (to_parts) late.part_o[(part0 + ri) * D + d] = y;
                else Elt<TQ>::store1(late.a.y + t * late.a.y_nb2 + hq * late.a.y_nb1 + d * Elt<TQ>::size, y);
            }
        }
    }
}

// Adds up a row's parts (those of its pieces, then the one of a request's own keys): a wave a row of y, its dims over the lanes, U
// parts in flight.
template <typename TQ>
__global__ __launch_bounds__(256) void k_prompt_join(PromptArgs pa) {
    constexpr int U = 8, N = 4;
    const AttnArgs& a = pa.a;
    const uint32_t lane = threadIdx.x & 63;
    const uint32_t row = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6)), t = row / a.hq, h = row - t * a.hq;
    if (t >= a.n_rows) return;
    // rows of no request stay as they are; a request of no group has its own keys' part alone
    const bool outside = static_cast<int32_t>(t) < a.start[0] || static_cast<int32_t>(t) >= a.start[pa.n_start];
    if (outside && !pa.shared) return;
    uint2 parts = outside ? make_uint2(0, 0) : pa.row_parts[row];
    uint32_t n = parts.y & 0xffff;
    const uint32_t r = parts.y >> 16;
    // a row that no request has after all (`start` falls somewhere): what the scratch holds for it is anything
    if (n > 0 && (parts.x >= pa.slots || (n - 1) * a.hkv >= pa.slots - parts.x || r >= pa.row_cap)) n = 0;
    if (n <= 1 && !pa.shared) return;                        // written by its only piece
    auto at = [&](uint32_t i) { return static_cast<uint64_t>(parts.x + i * a.hkv) * pa.row_cap + r; };
    float m = pa.shared ? pa.own_ml[row].x : kLowest;
    for (uint32_t i = lane; i < n; i += 64) m = fmaxf(m, pa.part_ml[at(i)].x);
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor(m, d));
    float l = 0.0f, o[N] = {};
    auto add = [&](float2 ml, const float (&v)[N]) {
        const float f = __builtin_amdgcn_exp2f(ml.x - m);
        l = fmaf(ml.y, f, l);
#pragma unroll
        for (int k = 0; k < N; k++) o[k] = fmaf(v[k], f, o[k]);
    };
    auto fetch = [&](const float* p, float (&v)[N]) {
#pragma unroll
        for (int k = 0; k < N; k++) v[k] = lane + 64 * k < a.D ? p[lane + 64 * k] : 0.0f;
    };
    for (uint32_t i = 0; i < n; i += U) {
        float v[U][N];
        float2 ml[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const uint64_t part = at(min(i + u, n - 1));
            ml[u] = pa.part_ml[part];
            fetch(pa.part_o + part * a.D, v[u]);
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (i + u < n) add(ml[u], v[u]);
        }
    }
    if (pa.shared) {
        float v[N];
        fetch(pa.own_o + static_cast<uint64_t>(row) * a.D, v);
        add(pa.own_ml[row], v);
    }
    char* yr = a.y + t * a.y_nb2 + h * a.y_nb1;
#pragma unroll
    for (int k = 0; k < N; k++) {
        const uint32_t d = lane + 64 * k;
        if (d < a.D) Elt<TQ>::store1(yr + d * Elt<TQ>::size, l == 0.0f ? 0.0f : o[k] / l);
    }
}

struct PromptPlan {
    bool tiles, pair;          // k_prompt, else k_attn_rows; its PAIR
    int dp;
    uint32_t row_tiles, deal, row_cap, grid;
    size_t o_bytes, ml_bytes, bytes;
};

size_t up16(int64_t n) { return static_cast<size_t>(cdiv(n, 16) * 16); }

// n_start: requests, or groups of them (shared).
PromptPlan prompt_plan(const cbx_tensor* q, const cbx_tensor* k, const cbx_tensor* tables, int64_t n_start, bool shared,
                       const DeviceState* st) {
    PromptPlan p{};
    const int64_t D = q->ne[0], hkv = k->ne[2], g = hkv ? q->ne[1] / hkv : 0, cap = tables->ne[0] * k->ne[1];
    p.dp = D <= 64 ? 64 : D <= 96 ? 96 : D <= 128 ? 128 : 256;
    // Fewer rows a request than fill three of a tile's four waves: pairs (4 texts of 20 to 150 rows: 9.8 us for 11.0; 8 drafts of up to
    // 36 rows: 128 for 145; 4 groups of 96 rows: 252 for 193).
    p.pair = q->ne[2] * g < 96 * n_start;
    const int64_t rows = p.pair ? 64 : 128;
    const int64_t most = q->ne[2] * g / rows + n_start, wide = 2 * st->n_cu;
    p.tiles = D % (k->type == CBX_TYPE_I8 ? 16 : 8) == 0 && D <= 256 && cap > 0 && k->ne[3] > 0 && most * hkv < (int64_t{1} << 24) &&
              k->ne[2] <= wide;
    if (!p.tiles) return p;
    p.row_tiles = static_cast<uint32_t>(most);
    p.grid = static_cast<uint32_t>(most * hkv);
    // Row tiles that fit at once leave CUs idle at the end, or from the start; where there are more, dealing them gains nothing (660 on
    // 512 places, F32: 393 to 405 us for 355 to 403).  Below 512 keys the join costs what the pieces save.
    const int64_t key_tiles = cdiv(cap, k->type == CBX_TYPE_F32 || p.dp > 128 ? 32 : 64);
    if (most > kDealTiles || n_start > kDealTiles || most * key_tiles >= (int64_t{1} << 32) ||
        (!shared && (most * hkv > wide || cap < 512))) return p;
    // Two pieces a CU, as many as fit it at once at head_dim 65 to 128 (documents of 5000 to 30000 keys, 96 rows a head: 193 us; 1.5
    // times as many 217, half 234); of pairs twice as many, which evens out the last pieces (8 requests of up to 32000 keys, 36 rows:
    // 105 us for 120).
    const int64_t aim = p.pair ? 2 * wide : wide;
    p.deal = static_cast<uint32_t>(aim);
    p.grid = static_cast<uint32_t>(std::min(aim / hkv + most, most * cdiv(key_tiles, kLeast)) * hkv);
    p.row_cap = static_cast<uint32_t>(std::min<int64_t>(rows, q->ne[2] * g));
    const int64_t parts = static_cast<int64_t>(p.grid) * p.row_cap;
    p.o_bytes = up16(parts * D * 4);
    p.ml_bytes = up16(parts * 8);
    p.bytes = p.o_bytes + p.ml_bytes + up16(q->ne[1] * q->ne[2] * 8);
    return p;
}

PromptArgs prompt_args(const PagedAttnCall& c, const PromptPlan& p, uint32_t n_start, DeviceState* st) {
    PromptArgs a{};
    a.a = attn_args(c, st);
    a.n_start = n_start;
    a.tiles = p.row_tiles;
    a.deal = p.deal;
    a.slots = p.grid;
    a.row_cap = p.row_cap;
    page_division(a.a.g, &a.g_mul, &a.g_shift);
    char* ws = static_cast<char*>(c.ws);
    a.part_o = reinterpret_cast<float*>(ws);
    a.part_ml = reinterpret_cast<float2*>(ws + p.o_bytes);
    a.row_parts = reinterpret_cast<uint2*>(ws + p.o_bytes + p.ml_bytes);
    return a;
}

template <typename TQ, typename TC, int PP> void launch_dp(const PromptPlan& p, hipStream_t s, const PromptArgs& a) {
    auto go = [&](auto d, auto pair) {
        constexpr int DP = decltype(d)::value;
        constexpr bool PAIR = decltype(pair)::value;
        if (a.a.softcap > 0.0f) hipLaunchKernelGGL((k_prompt<TQ, TC, DP, PP, true, PAIR>), dim3(p.grid), dim3(256), 0, s, a);
        else hipLaunchKernelGGL((k_prompt<TQ, TC, DP, PP, false, PAIR>), dim3(p.grid), dim3(256), 0, s, a);
    };
    auto both = [&](auto d) {
        if (p.pair) go(d, std::true_type());
        else go(d, std::false_type());
    };
    if (p.dp == 64) both(std::integral_constant<int, 64>());
    else if (p.dp == 96) both(std::integral_constant<int, 96>());
    else if (p.dp == 128) both(std::integral_constant<int, 128>());
    else both(std::integral_constant<int, 256>());
}

void launch_tiles(const PagedAttnCall& c, const PromptPlan& p, const PromptArgs& a, hipStream_t s) {
    const bool t16 = c.q->type == CBX_TYPE_F16, i8 = c.k->type == CBX_TYPE_I8;
    if (t16 && i8) launch_dp<uint16_t, int8_t, 2>(p, s, a);
    else if (i8) launch_dp<float, int8_t, 3>(p, s, a);
    else if (c.k->type == CBX_TYPE_F32) t16 ? launch_dp<uint16_t, float, 2>(p, s, a) : launch_dp<float, float, 2>(p, s, a);
    else if (!t16) launch_dp<float, uint16_t, 2>(p, s, a);
    // F16 throughout: a probability rounded to one f16 (2^-11 of itself at most) makes the result's error 1.3 times that of its own
    // rounding, in two parts nothing; two cost half as many products again and more conversions.  In a call of many rows these are its
    // time (16000 tokens: 3.15 ms for 2.28; 48 requests, 25 thousand tokens: 515 us for 391; 4096 rows, of 256 tokens of 16 heads of 64:
    // 14.3 for 12.1, behind 2000 others 30.4 for 27.8, of 16 x 8 drafts of 32 heads on 8 64.0 for 61.5), in one of few the pages' bytes
    // and latency are, and it keeps its precision.
    else if (c.shared || c.q->ne[1] * c.q->ne[2] < 4096) launch_dp<uint16_t, uint16_t, 2>(p, s, a);
    else launch_dp<uint16_t, uint16_t, 1>(p, s, a);
}

void launch_join(const PagedAttnCall& c, const PromptArgs& a, hipStream_t s) {
    const dim3 grid(static_cast<unsigned>(cdiv(c.q->ne[1] * c.q->ne[2], 4)));
    if (c.q->type == CBX_TYPE_F16) hipLaunchKernelGGL((k_prompt_join<uint16_t>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((k_prompt_join<float>), grid, dim3(256), 0, s, a);
}

}  // namespace

// Numbers that k_prompt's products hold: scales and caps times log2(e), and a cap's share in the scale as a normal number.  The rest,
// which no model has, is k_attn_rows', or paged_attention's.
static bool tile_numbers(const PagedAttnCall& c) {
    return std::isfinite(c.scale * kLog2e) && c.softcap <= 0x1p60f && (c.softcap == 0.0f || c.scale == 0.0f || std::fabs(c.scale) / c.softcap >= 0x1p-126f);
}

size_t paged_prompt_workspace(const cbx_tensor* q, const cbx_tensor* k, const cbx_tensor* tables, const DeviceState* st) {
    return prompt_plan(q, k, tables, tables->ne[1], false, st).bytes;
}

int launch_paged_prompt(const PagedAttnCall& c, DeviceState* st, hipStream_t s) {
    const char* what = "cbx_paged_prompt_attention";
    const PromptPlan p = prompt_plan(c.q, c.k, c.tables, c.tables->ne[1], false, st);
    if (!p.tiles || !tile_numbers(c) || !vector_rows(c.k) || !vector_rows(c.v)) return launch_attention_rows(attn_args(c, st), c, what, s);
    const PromptArgs a = prompt_args(c, p, static_cast<uint32_t>(c.tables->ne[1]), st);
    launch_tiles(c, p, a, s);
    if (p.deal) launch_join(c, a, s);
    return check_launch(what);
}

// ---- groups ---------------------------------------------------------------------

namespace {

// k_prompt over the shared keys, k_attn_tiles over each request's own, the
// parts of both added up.
struct SharedPlan {
    PromptPlan pre;
    bool tiles;
    size_t o_bytes, ml_bytes, first_bytes, bytes;   // behind pre's: the own keys' parts, where these begin, k_attn_tiles' scratch
};

SharedPlan shared_plan(const cbx_tensor* q, const cbx_tensor* k, const cbx_tensor* tables, const cbx_tensor* start,
                       const DeviceState* st) {
    SharedPlan p{};
    const int64_t n_groups = start->ne[0] - 1, rows = q->ne[1] * q->ne[2];
    p.pre = prompt_plan(q, k, tables, n_groups, true, st);
    // both kernels take it; else paged_attention does, whose scratch is the same
    p.tiles = p.pre.tiles && p.pre.deal && n_groups > 0 && n_groups < q->ne[2] && attention_tiles(q, k, tables, st);
    p.bytes = attention_tiles_workspace(q, k, tables, st);
    if (!p.tiles) return p;
    p.o_bytes = up16(rows * q->ne[0] * 4);
    p.ml_bytes = up16(rows * 8);
    p.first_bytes = up16(q->ne[2] * 4);
    p.bytes += p.pre.bytes + p.o_bytes + p.ml_bytes + p.first_bytes;
    return p;
}

}  // namespace

size_t paged_shared_workspace(const cbx_tensor* q, const cbx_tensor* k, const cbx_tensor* tables, const cbx_tensor* start,
                              const DeviceState* st) {
    return shared_plan(q, k, tables, start, st).bytes;
}

int launch_paged_shared(const PagedAttnCall& c, DeviceState* st, hipStream_t s) {
    const char* what = "cbx_paged_shared_attention";
    const SharedPlan p = shared_plan(c.q, c.k, c.tables, c.start, st);
    PagedAttnCall own = c;
    own.start = own.shared = nullptr;
    if (!p.tiles || !tile_numbers(c) || !vector_rows(c.k) || !vector_rows(c.v)) return launch_paged_attention(own, st, s);
    PromptArgs a = prompt_args(c, p.pre, static_cast<uint32_t>(c.start->ne[0] - 1), st);
    char* ws = static_cast<char*>(c.ws) + p.pre.bytes;
    float* own_o = reinterpret_cast<float*>(ws);
    float2* own_ml = reinterpret_cast<float2*>(ws + p.o_bytes);
    a.shared = static_cast<const int32_t*>(c.shared->data);
    a.own_o = own_o;
    a.own_ml = own_ml;
    a.own_first = reinterpret_cast<int32_t*>(ws + p.o_bytes + p.ml_bytes);
    launch_tiles(c, p.pre, a, s);
    AttnArgs b = attn_args(own, st);
    b.own_first = a.own_first;
    b.groups = a.a.start;
    b.n_groups = a.n_start;
    b.own_o = own_o;
    b.own_ml = own_ml;
    if (!launch_attention_tiles(b, own, ws + p.o_bytes + p.ml_bytes + p.first_bytes, st, s)) {
        return set_error(CBX_ERR_UNSUPPORTED, "cbx_paged_shared_attention: the requests' own keys have no kernel");
    }
    launch_join(c, a, s);
    return check_launch(what);
}

}  // namespace cbx
