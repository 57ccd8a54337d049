// k_paged_plan.hip -- the paged cache's bookkeeping: pages taken and given
// back, and the slots and positions of a step's tokens.
//
// With have_s = ceil(past_s / P) and need_s = ceil((past_s + new_s) / P) -
// have_s, everything follows from two exclusive scans over the requests,
//   tok_s = sum_{r < s} new_r,    off_s = sum_{r < s} need_r
// (requests refused for another reason than an empty pool add no need):
// page i of the new ones of s is free[n_free - 1 - off_s - i], and token j of
// s has position past_s + j in page (past_s + j) / P.  Granted requests that
// need a page are a prefix of all that do, so what they take is the top of
// the stack without gaps.
//
// A few KB of data: latency is everything.  Every workgroup makes the two
// scans for itself in LDS (a few requests a lane, a wave scan, four wave
// totals), so one launch does without a second pass or a
// message between workgroups, and then fills its part of the tokens and
// pages, finding the request of each by a search over the scan.
#include "cbx_device.h"

namespace cbx {
namespace {

constexpr int kPlanThreads = 256;

// Exclusive scan of one value a thread over the block; *total the sum.
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t* lds, int64_t* total) {
    const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
    int64_t x = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int64_t u = __shfl_up(x, d);
        if (lane >= d) x += u;
    }
    if (lane == 63) lds[wid] = x;
    __syncthreads();
    int64_t before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kPlanThreads / 64; w++) {
        if (w < wid) before += lds[w];
        all += lds[w];
    }
    __syncthreads();
    *total = all;
    return before + x - v;
}

__device__ __forceinline__ int32_t sat32(int64_t v) { return v > 0x7fffffff ? 0x7fffffff : static_cast<int32_t>(v); }

// The last s of [0, n) with start[s] <= i (start ascending, start[0] = 0).
__device__ __forceinline__ int last_at_most(const int32_t* start, int n, int32_t i) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (start[mid] <= i) lo = mid;
        else hi = mid;
    }
    return lo;
}

__device__ __forceinline__ int32_t* table_row(char* tables, int64_t nb1, int s) {
    return reinterpret_cast<int32_t*>(tables + s * nb1);
}

// LDS: tok[n], off[n], have[n] (have -1: refused), each 32-bit.
__global__ __launch_bounds__(kPlanThreads) void k_append(AppendArgs a, uint32_t* err) {
    extern __shared__ int32_t lds32[];
    __shared__ int64_t part[kPlanThreads / 64];
    __shared__ int32_t took;
    int32_t *tok = lds32, *off = lds32 + a.n_seq, *have = lds32 + 2 * a.n_seq;
    const int tid = threadIdx.x, n = a.n_seq;
    const int64_t cap = static_cast<int64_t>(a.max_pages) * a.page;
    int32_t free_n = *a.n_free;
    bool wrong = free_n < 0 || free_n > a.pool;
    free_n = free_n < 0 ? 0 : (free_n > a.pool ? a.pool : free_n);
    if (tid == 0) took = 0;
    // a lane's requests are neighbours: c of them from c * tid on
    const int c = (n + kPlanThreads - 1) / kPlanThreads;
    const int s0 = tid * c, s1 = s0 + c < n ? s0 + c : n;
    int64_t toks = 0, pages = 0;
    for (int s = s0; s < s1; s++) toks += a.n_new[s] > 0 ? a.n_new[s] : 0;
    int64_t n_tok;
    int64_t t = block_scan(toks, part, &n_tok);
    for (int s = s0; s < s1; s++) {
        const int64_t past = a.n_past[s], nw = a.n_new[s] > 0 ? a.n_new[s] : 0;
        const bool sane = past >= 0 && past <= cap && a.n_new[s] >= 0;
        wrong |= !sane;
        const bool fits = sane && past + nw <= cap && t + nw <= a.n_slots;
        const int64_t hv = fits ? (past + a.page - 1) / a.page : -1;
        if (fits) pages += (past + nw + a.page - 1) / a.page - hv;
        tok[s] = sat32(t);
        have[s] = static_cast<int32_t>(hv);
        t += nw;
    }
    int64_t n_pages;
    int64_t o = block_scan(pages, part, &n_pages);
    for (int s = s0; s < s1; s++) {
        off[s] = sat32(o);
        if (have[s] < 0) continue;
        const int64_t need = (static_cast<int64_t>(a.n_past[s]) + a.n_new[s] + a.page - 1) / a.page - have[s];
        if (need > 0 && o + need > free_n) have[s] = -1;
        else if (need > 0) atomicMax(&took, static_cast<int32_t>(o + need));   // LDS; the maximum, in any order
        o += need;
    }
    __syncthreads();
    if (blockIdx.x == 0) {
        for (int s = tid; s < n; s += kPlanThreads) {
            a.seq_lens[s] = have[s] < 0 ? a.n_past[s] : a.n_past[s] + a.n_new[s];
            a.tok_start[s] = tok[s];
        }
        if (tid == 0) {
            a.tok_start[n] = sat32(n_tok);
            *a.n_free_out = free_n - took;
        }
    }
    if (wrong) atomicOr(err, DEV_ERR_PAGE);
    const int64_t step = static_cast<int64_t>(gridDim.x) * kPlanThreads;
    const int64_t first = static_cast<int64_t>(blockIdx.x) * kPlanThreads + tid;
    // the pages newly taken: took of them, in the order of the requests
    for (int64_t i = first; i < took; i += step) {
        const int s = last_at_most(off, n, static_cast<int32_t>(i));
        table_row(a.tables, a.tables_nb1, s)[have[s] + (i - off[s])] = a.free_pages[free_n - 1 - i];
    }
    for (int64_t i = first; i < a.n_slots; i += step) {
        int32_t slot = -1, pos = 0;
        if (i < n_tok) {
            const int s = last_at_most(tok, n, static_cast<int32_t>(i));
            pos = static_cast<int32_t>(a.n_past[s] + (i - tok[s]));
            if (have[s] >= 0) {
                const int32_t pi = pos / a.page;
                const int32_t page = pi < have[s] ? table_row(a.tables, a.tables_nb1, s)[pi]
                                                  : a.free_pages[free_n - 1 - off[s] - (pi - have[s])];
                const int64_t p = static_cast<int64_t>(page) * a.page + pos % a.page;
                if (page >= 0 && p <= 0x7fffffff) slot = static_cast<int32_t>(p);
                else atomicOr(err, DEV_ERR_PAGE);
            }
        }
        a.slots[i] = slot;
        a.positions[i] = pos;
    }
}

// LDS: off[n], the place above the stack of each released request's first page.
__global__ __launch_bounds__(kPlanThreads) void k_release(ReleaseArgs a, uint32_t* err) {
    extern __shared__ int32_t off[];
    __shared__ int64_t part[kPlanThreads / 64];
    const int tid = threadIdx.x, n = a.n_seq;
    const int64_t cap = static_cast<int64_t>(a.max_pages) * a.page;
    int32_t free_n = *a.n_free;
    bool wrong = free_n < 0 || free_n > a.pool;
    free_n = free_n < 0 ? 0 : (free_n > a.pool ? a.pool : free_n);
    auto pages_of = [&](int s) -> int64_t {
        const int64_t len = a.seq_lens[s];
        if (a.release[s] == 0) return 0;
        if (len < 0 || len > cap) {
            wrong = true;
            return 0;
        }
        return (len + a.page - 1) / a.page;
    };
    const int c = (n + kPlanThreads - 1) / kPlanThreads;
    const int s0 = tid * c, s1 = s0 + c < n ? s0 + c : n;
    int64_t sum = 0;
    for (int s = s0; s < s1; s++) sum += pages_of(s);
    int64_t total;
    int64_t at = block_scan(sum, part, &total);
    for (int s = s0; s < s1; s++) {
        off[s] = sat32(at);
        at += pages_of(s);
    }
    __syncthreads();
    const int64_t room = a.pool - free_n;
    wrong |= total > room;
    if (blockIdx.x == 0) {
        for (int s = tid; s < n; s += kPlanThreads) a.seq_lens_out[s] = a.release[s] ? 0 : a.seq_lens[s];
        if (tid == 0) *a.n_free_out = static_cast<int32_t>(free_n + (total < room ? total : room));
    }
    if (wrong) atomicOr(err, DEV_ERR_PAGE);
    for (int s = blockIdx.x; s < n; s += gridDim.x) {
        const int64_t pages = pages_of(s);
        int32_t* row = table_row(a.tables, a.tables_nb1, s);
        for (int64_t i = tid; i < pages; i += kPlanThreads) {
            const int32_t page = row[i];
            row[i] = -1;
            if (off[s] + i < room) a.free_pages[free_n + off[s] + i] = page;
        }
    }
}

}  // namespace

int launch_paged_append(const AppendArgs& a, DeviceState* st, hipStream_t s) {
    const int64_t grid = std::max<int64_t>(1, std::min<int64_t>(cdiv(a.n_slots, kPlanThreads), 2 * st->n_cu));
    hipLaunchKernelGGL(k_append, dim3(static_cast<unsigned>(grid)), dim3(kPlanThreads), 12 * static_cast<size_t>(a.n_seq), s,
                       a, st->err_word);
    return check_launch("cbx_paged_append");
}

int launch_paged_release(const ReleaseArgs& a, DeviceState* st, hipStream_t s) {
    const int64_t grid = std::max<int64_t>(1, std::min<int64_t>(a.n_seq, st->n_cu));
    hipLaunchKernelGGL(k_release, dim3(static_cast<unsigned>(grid)), dim3(kPlanThreads), 4 * static_cast<size_t>(a.n_seq), s,
                       a, st->err_word);
    return check_launch("cbx_paged_release");
}

}  // namespace cbx
