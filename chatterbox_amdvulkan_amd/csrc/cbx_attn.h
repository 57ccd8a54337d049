// cbx_attn.h -- what the attention kernels over paged caches share:
// k_paged_attn.hip (one new token a request) and k_prompt_attn.hip (all new
// tokens of packed requests, groups that begin with the same pages).
#pragma once

#include "cbx_device.h"

namespace cbx {

constexpr int kAttnThreads = 256;
constexpr int kAttnMaxD = 512;
constexpr float kLowest = -3.0e38f;   // below every score that matters; finite, so that m - m is 0
constexpr float kLog2e = 1.44269504088896340736f;

// What a small call reads comes first: a launch's arguments are fetched a line at a
// time, and one line more of them before the keys is half a microsecond.
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
    // I8 pages: their rows' scales
    const char *ks, *vs;
    int64_t ks_nb0, ks_nb1, ks_nb2, vs_nb0, vs_nb1, vs_nb2;
    bool s_quads;                    // they can be read four at a time
    const int32_t* start;            // packed tokens or groups, see PagedAttnCall; null: a row of q a request
    uint32_t n_rows;                 // of q: tokens or requests
    // the keys behind the shared ones of a group (k_attn_tiles and k_attn_join after k_prompt; else null): own_first says where a
    // request's begin, and (o, m, l) go to own_o and own_ml at request * hq + head instead of y
    const int32_t* own_first;
    const int32_t* groups;           // own_first holds for the requests [groups[0], groups[n_groups])
    uint32_t n_groups;
    float own_down;                  // 1 over what the probabilities in o and l are multiplied by
    float* own_o;
    float2* own_ml;
};

__device__ __forceinline__ uint32_t page_of(const AttnArgs& a, uint32_t key) {
    return static_cast<uint32_t>((static_cast<uint64_t>(key) * a.page_mul) >> a.page_shift);
}

// The call's tensors as every kernel takes them.
AttnArgs attn_args(const PagedAttnCall& c, const DeviceState* st);
// A workgroup a row of q and query head, for what no other kernel takes: any
// sizes, strides and types.
int launch_attention_rows(const AttnArgs& a, const PagedAttnCall& c, const char* what, hipStream_t s);
// paged_attention's kernels by tiles over a's tensors: whether they take these shapes; launches them if they take the call; the
// workspace they need.
bool attention_tiles(const cbx_tensor* q, const cbx_tensor* k, const cbx_tensor* tables, const DeviceState* st);
bool launch_attention_tiles(AttnArgs a, const PagedAttnCall& c, void* ws, DeviceState* st, hipStream_t s);
size_t attention_tiles_workspace(const cbx_tensor* q, const cbx_tensor* k, const cbx_tensor* tables, const DeviceState* st);
// Whether rows can be read 16 bytes at a time.
bool vector_rows(const cbx_tensor* t);

}  // namespace cbx
