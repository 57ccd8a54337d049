// k_paged_plan.hip -- the paged cache's bookkeeping: pages taken and given
// back, and the slots and positions of a step's tokens.
//
// With have_s = ceil(past_s / P) and need_s = ceil((past_s + new_s) / P) -
// have_s, everything follows from two exclusive scans over the requests,
//   tok_s = sum_{r < s} new_r,    off_s = sum_{r < s} need_r
// (requests refused for another reason than an empty pool add no need):
// page i of the new ones of s is free[n_free - 1 - off_s - i], and token j of
// s has position past_s + j in page (past_s + j) / P (the first key of a new
// page is one of the tokens, which notes it in the table).  Granted requests that
// need a page are a prefix of all that do, so what they take is the top of
// the stack without gaps.
//
// A few KB of data: latency is everything.  Every workgroup of an append makes the two
// scans for itself in LDS (a few requests a lane, a wave scan by DPP, four wave
// totals), so one launch does without a second pass or a message between
// workgroups, and then fills its part of the tokens, finding the request of
// every fourth by a search over the scan.  64 streams of one token each 5.0 us,
// 500 prompts of 362000 tokens in all 6.8 us for 3 MB (an empty kernel's entry in
// the same trace: 3.2).
#include "cbx_device.h"

namespace cbx {
namespace {

constexpr int kPlanThreads = 256;

// Sums of token and page counts stop at 2^31 - 1 (still associative for what
// is not negative): a request behind that many is refused all the same.
constexpr uint32_t kMostCount = 0x7fffffffu;
__device__ __forceinline__ uint32_t sat_add(uint32_t a, uint32_t b) { return min(a + b, kMostCount); }

// Exclusive scan of one value a thread over the block; *total the sum.
// Within rows of 16 lanes by shifts, then each row's last to the rows behind.
template <int CTRL, int ROWS> __device__ __forceinline__ uint32_t dpp_sat_add(uint32_t x) {
    return sat_add(x, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(x), CTRL, ROWS, 0xf, false)));
}
// The largest of the wave's values, in lane 63.
template <int CTRL, int ROWS> __device__ __forceinline__ uint32_t dpp_max(uint32_t x) {
    return max(x, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(x), CTRL, ROWS, 0xf, false)));
}
__device__ __forceinline__ uint32_t wave_max(uint32_t x) {
    x = dpp_max<0x111, 0xf>(x);
    x = dpp_max<0x112, 0xf>(x);
    x = dpp_max<0x114, 0xf>(x);
    x = dpp_max<0x118, 0xf>(x);
    x = dpp_max<0x142, 0xa>(x);
    return dpp_max<0x143, 0xc>(x);
}
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t* lds, uint32_t* total) {
    const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
    uint32_t x = v;
    x = dpp_sat_add<0x111, 0xf>(x);
    x = dpp_sat_add<0x112, 0xf>(x);
    x = dpp_sat_add<0x114, 0xf>(x);
    x = dpp_sat_add<0x118, 0xf>(x);
    x = dpp_sat_add<0x142, 0xa>(x);
    x = dpp_sat_add<0x143, 0xc>(x);
    // the lane before; the wave's first has nothing before it
    uint32_t before = static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(x), 0x138, 0xf, 0xf, false));
    if (lane == 63) lds[wid] = x;
    __syncthreads();
    uint32_t all = 0;
#pragma unroll
    for (int w = 0; w < kPlanThreads / 64; w++) {
        if (w < wid) before = sat_add(before, lds[w]);
        all = sat_add(all, lds[w]);
    }
    *total = all;
    return before;
}

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

constexpr int kPlanTokens = 4;   // neighbouring tokens of a thread
constexpr int kPlanHeld = 4;     // requests a thread reads at once
typedef int32_t i4u __attribute__((ext_vector_type(4), aligned(4)));

// LDS: tok[n], off[n], have[n] (have -1: refused), past[n], each 32-bit.
__global__ __launch_bounds__(kPlanThreads) void k_append(AppendArgs a, uint32_t* err) {
    extern __shared__ int32_t lds32[];
    __shared__ uint32_t part[2][kPlanThreads / 64];
    const int tid = threadIdx.x, n = a.n_seq;
    int32_t *tok = lds32, *off = lds32 + n, *have = lds32 + 2 * n, *had = lds32 + 3 * n;
    const int32_t cap = a.max_pages * a.page;      // below 2^31
    int32_t free_n = *a.n_free;
    bool wrong = free_n < 0 || free_n > a.pool;
    free_n = free_n < 0 ? 0 : min(free_n, a.pool);
    // a lane's requests are neighbours: c of them from c * tid on
    const int c = (n + kPlanThreads - 1) / kPlanThreads;
    const int s0 = min(tid * c, n), s1 = min(s0 + c, n);
    uint32_t toks = 0;
    for (int b = s0; b < s1; b += kPlanHeld) {
        int32_t past[kPlanHeld], nw[kPlanHeld];
#pragma unroll
        for (int k = 0; k < kPlanHeld; k++) {
            past[k] = a.n_past[min(b + k, s1 - 1)];
            nw[k] = a.n_new[min(b + k, s1 - 1)];
        }
#pragma unroll
        for (int k = 0; k < kPlanHeld; k++) {
            if (b + k >= s1) break;
            wrong |= past[k] < 0 || past[k] > cap || nw[k] < 0;
            had[b + k] = past[k];
            off[b + k] = nw[k];                    // until its pages are known
            toks = sat_add(toks, max(nw[k], 0));
        }
    }
    uint32_t n_tok, n_pages;
    uint32_t t = block_scan(toks, part[0], &n_tok), pages = 0;
    // for lengths and positions up to max_pages * page_size
    auto page_of = [&](int32_t pos) {
        return static_cast<int32_t>((static_cast<uint64_t>(static_cast<uint32_t>(pos)) * a.page_mul) >> a.page_shift);
    };
    auto pages_of = [&](int32_t len) { return len > 0 ? page_of(len - 1) + 1 : 0; };
    for (int s = s0; s < s1; s++) {
        const int32_t past = had[s], nw = off[s];
        const uint32_t end = sat_add(t, max(nw, 0));
        const bool fits = past >= 0 && nw >= 0 && past <= cap && nw <= cap - past && end <= static_cast<uint32_t>(a.n_slots) &&
                          end < kMostCount;
        const int32_t hv = fits ? pages_of(past) : -1;
        const uint32_t need = fits ? static_cast<uint32_t>(pages_of(past + nw) - hv) : 0;
        tok[s] = static_cast<int32_t>(t);
        have[s] = hv;
        off[s] = static_cast<int32_t>(need);
        pages = sat_add(pages, need);
        t = end;
    }
    uint32_t o = block_scan(pages, part[1], &n_pages), granted = 0;
    for (int s = s0; s < s1; s++) {
        const uint32_t need = static_cast<uint32_t>(off[s]), end = sat_add(o, need);
        off[s] = static_cast<int32_t>(o);
        if (need > 0) {
            if (end > static_cast<uint32_t>(free_n)) have[s] = -1;
            else granted = end;
        }
        o = end;
    }
    granted = wave_max(granted);
    if ((tid & 63) == 63) part[0][tid >> 6] = granted;
    __syncthreads();
    uint32_t took = 0;
#pragma unroll
    for (int w = 0; w < kPlanThreads / 64; w++) took = max(took, part[0][w]);
    if (blockIdx.x == 0) {
        for (int s = tid; s < n; s += kPlanThreads) {
            a.seq_lens[s] = have[s] < 0 ? had[s] : had[s] + a.n_new[s];
            a.tok_start[s] = tok[s];
        }
        if (tid == 0) {
            a.tok_start[n] = static_cast<int32_t>(n_tok);
            *a.n_free_out = free_n - static_cast<int32_t>(took);
        }
    }
    const int64_t step = static_cast<int64_t>(gridDim.x) * kPlanThreads * kPlanTokens;
    for (int64_t i0 = (static_cast<int64_t>(blockIdx.x) * kPlanThreads + tid) * kPlanTokens; i0 < a.n_slots; i0 += step) {
        int32_t slot[kPlanTokens], pos[kPlanTokens], page[kPlanTokens], in[kPlanTokens];
        int32_t* fresh[kPlanTokens];                // where a page newly taken is noted, by its first token
        int s = i0 < n_tok ? last_at_most(tok, n, static_cast<int32_t>(i0)) : 0;
#pragma unroll
        for (int k = 0; k < kPlanTokens; k++) {     // the pages' loads first, together
            const int64_t i = i0 + k;
            page[k] = slot[k] = -1;
            pos[k] = in[k] = 0;
            fresh[k] = nullptr;
            if (i >= n_tok || i >= a.n_slots) continue;
            while (s + 1 < n && tok[s + 1] <= i) s++;
            pos[k] = had[s] + static_cast<int32_t>(i - tok[s]);
            if (have[s] < 0) continue;
            slot[k] = 0;
            const int32_t pi = page_of(pos[k]);
            in[k] = pos[k] - pi * a.page;
            int32_t* entry = table_row(a.tables, a.tables_nb1, s) + pi;
            const bool taken = pi >= have[s];
            page[k] = taken ? a.free_pages[free_n - 1 - off[s] - (pi - have[s])] : *entry;
            if (taken && in[k] == 0) fresh[k] = entry;
        }
#pragma unroll
        for (int k = 0; k < kPlanTokens; k++) {
            const int64_t p = static_cast<int64_t>(page[k]) * a.page + in[k];
            const bool good = page[k] >= 0 && p < kMostCount;
            wrong |= slot[k] == 0 && !good;
            slot[k] = slot[k] == 0 && good ? static_cast<int32_t>(p) : -1;
            if (fresh[k]) *fresh[k] = page[k];
        }
        if (i0 + kPlanTokens <= a.n_slots) {
            *reinterpret_cast<i4u*>(a.slots + i0) = i4u{slot[0], slot[1], slot[2], slot[3]};
            *reinterpret_cast<i4u*>(a.positions + i0) = i4u{pos[0], pos[1], pos[2], pos[3]};
        } else {
            for (int k = 0; k < static_cast<int>(a.n_slots - i0); k++) {
                a.slots[i0 + k] = slot[k];
                a.positions[i0 + k] = pos[k];
            }
        }
    }
    if (wrong) atomicOr(err, DEV_ERR_PAGE);
}

// Release.  An entry below 0 is no page (a row given back before, or never
// filled) and is left out, so the pages of a request are known only from its
// row, and a row is cleared as it is given back: k_release_count notes how
// many each released request has (in seq_lens_out, which k_release sets to 0
// once every workgroup has read them), k_release scans those and gives back.
// A wave a request, eight entries a lane in flight, packed by ballots: 64
// requests of 32 pages 5.6 us in a graph, 4096 of 128 23.6, 4 of 8192 23.2 (a
// workgroup a request 6.4, 59 and 14.1).

// The entries that a request's length covers, when it is released; a length
// outside the table covers none.
__device__ __forceinline__ uint32_t released_entries(const ReleaseArgs& a, int s, bool* wrong) {
    if (a.release[s] == 0) return 0;
    const int32_t len = a.seq_lens[s];
    if (len < 0 || len > a.max_pages * a.page) {
        *wrong = true;
        return 0;
    }
    return (static_cast<uint32_t>(len) + a.page - 1) / a.page;
}

constexpr int kPlanWaves = kPlanThreads / 64;
constexpr int kPlanLoads = 8;     // entries of a lane

// Entries i0 + 64 u + lane of a row, -1 past its end.
__device__ __forceinline__ void load_entries(const int32_t* row, uint32_t i0, uint32_t entries, int32_t (&page)[kPlanLoads]) {
    const uint32_t i = i0 + (threadIdx.x & 63);
#pragma unroll
    for (int u = 0; u < kPlanLoads; u++) page[u] = row[min(i + 64 * u, entries - 1)];
#pragma unroll
    for (int u = 0; u < kPlanLoads; u++) if (i + 64 * u >= entries) page[u] = -1;
}

__global__ __launch_bounds__(kPlanThreads) void k_release_count(ReleaseArgs a, uint32_t* err) {
    const int s = blockIdx.x * kPlanWaves + (threadIdx.x >> 6);
    if (blockIdx.x == 0 && threadIdx.x == 0) *a.n_free_out = 0;      // k_release's workgroups that have read the counts
    if (s >= a.n_seq) return;
    bool wrong = false;
    const uint32_t entries = released_entries(a, s, &wrong);
    const int32_t* row = table_row(a.tables, a.tables_nb1, s);
    uint32_t pages = 0;
    for (uint32_t i0 = 0; i0 < entries; i0 += 64 * kPlanLoads) {
        int32_t page[kPlanLoads];
        load_entries(row, i0, entries, page);
#pragma unroll
        for (int u = 0; u < kPlanLoads; u++) pages += __popcll(__ballot(page[u] >= 0));
    }
    if ((threadIdx.x & 63) != 0) return;
    a.seq_lens_out[s] = a.release[s] ? static_cast<int32_t>(pages) : a.seq_lens[s];
    if (wrong || pages != entries) atomicOr(err, DEV_ERR_PAGE);
}

// LDS: off[n], the place above the stack of each released request's first page.
__global__ __launch_bounds__(kPlanThreads) void k_release(ReleaseArgs a, uint32_t* err) {
    extern __shared__ int32_t off[];
    __shared__ uint32_t part[kPlanWaves];
    __shared__ bool last;
    const int tid = threadIdx.x, lane = tid & 63, n = a.n_seq;
    int32_t free_n = *a.n_free;
    bool wrong = free_n < 0 || free_n > a.pool;
    free_n = free_n < 0 ? 0 : min(free_n, a.pool);
    auto pages_of = [&](int s) -> uint32_t { return a.release[s] ? static_cast<uint32_t>(a.seq_lens_out[s]) : 0; };
    const int c = (n + kPlanThreads - 1) / kPlanThreads;
    const int s0 = min(tid * c, n), s1 = min(s0 + c, n);
    uint32_t sum = 0;
    for (int s = s0; s < s1; s++) sum = sat_add(sum, pages_of(s));
    uint32_t total;
    uint32_t at = block_scan(sum, part, &total);
    for (int s = s0; s < s1; s++) {
        off[s] = static_cast<int32_t>(at);
        at = sat_add(at, pages_of(s));
    }
    __syncthreads();
    const int64_t room = a.pool - free_n;
    wrong |= total > room;
    // the counts are read: whoever is last to say so may overwrite them
    if (tid == 0) last = __hip_atomic_fetch_add(a.n_free_out, 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) == static_cast<int32_t>(gridDim.x) - 1;
    __syncthreads();
    if (last) {
        for (int s = tid; s < n; s += kPlanThreads) if (a.release[s]) a.seq_lens_out[s] = 0;
        if (tid == 0) *a.n_free_out = static_cast<int32_t>(free_n + (total < room ? total : room));
    }
    if (wrong && tid == 0) atomicOr(err, DEV_ERR_PAGE);
    bool told = false;     // by k_release_count
    for (int s = blockIdx.x * kPlanWaves + (tid >> 6); s < n; s += gridDim.x * kPlanWaves) {
        const uint32_t entries = released_entries(a, s, &told);
        int32_t* row = table_row(a.tables, a.tables_nb1, s);
        int64_t to = off[s];
        for (uint32_t i0 = 0; i0 < entries; i0 += 64 * kPlanLoads) {
            int32_t page[kPlanLoads];
            load_entries(row, i0, entries, page);
#pragma unroll
            for (int u = 0; u < kPlanLoads; u++) {
                const uint32_t i = i0 + 64 * u + lane;
                if (i < entries) row[i] = -1;
                const uint64_t given = __ballot(page[u] >= 0);
                const int64_t at_page = to + __popcll(given & ((uint64_t{1} << lane) - 1));
                if (page[u] >= 0 && at_page < room) a.free_pages[free_n + at_page] = page[u];
                to += __popcll(given);
            }
        }
    }
}

}  // namespace

int launch_paged_append(const AppendArgs& args, DeviceState* st, hipStream_t s) {
    AppendArgs a = args;
    page_division(a.page, &a.page_mul, &a.page_shift);
    const int64_t grid = std::max<int64_t>(1, std::min<int64_t>(cdiv(a.n_slots, kPlanThreads * kPlanTokens), 4 * st->n_cu));
    hipLaunchKernelGGL(k_append, dim3(static_cast<unsigned>(grid)), dim3(kPlanThreads), 16 * static_cast<size_t>(a.n_seq), s,
                       a, st->err_word);
    return check_launch("cbx_paged_append");
}

int launch_paged_release(const ReleaseArgs& a, DeviceState* st, hipStream_t s) {
    const int64_t all = std::max<int64_t>(1, cdiv(a.n_seq, kPlanWaves)), grid = std::min<int64_t>(all, st->n_cu);
    hipLaunchKernelGGL(k_release_count, dim3(static_cast<unsigned>(all)), dim3(kPlanThreads), 0, s, a, st->err_word);
    hipLaunchKernelGGL(k_release, dim3(static_cast<unsigned>(grid)), dim3(kPlanThreads), 4 * static_cast<size_t>(a.n_seq), s,
                       a, st->err_word);
    return check_launch("cbx_paged_release");
}

}  // namespace cbx
