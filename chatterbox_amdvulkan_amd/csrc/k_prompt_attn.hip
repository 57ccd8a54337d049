// k_prompt_attn.hip -- causal attention of all new tokens of packed requests
// over a paged cache, and of one new token a request where groups of requests
// begin with the same pages.
#include "cbx_attn.h"

namespace cbx {

size_t paged_prompt_workspace(const cbx_tensor*, const cbx_tensor*, const cbx_tensor*, const DeviceState*) { return 0; }

int launch_paged_prompt(const PagedAttnCall& c, DeviceState* st, hipStream_t s) {
    return launch_attention_rows(attn_args(c, st), c, "cbx_paged_prompt_attention", s);
}

size_t paged_shared_workspace(const cbx_tensor* q, const cbx_tensor* k, const cbx_tensor* tables, const cbx_tensor*,
                              const DeviceState* st) {
    return paged_attention_workspace(q, k, tables, st);
}

int launch_paged_shared(const PagedAttnCall& c, DeviceState* st, hipStream_t s) {
    PagedAttnCall own = c;
    own.start = own.shared = nullptr;
    return launch_paged_attention(own, st, s);
}

}  // namespace cbx
