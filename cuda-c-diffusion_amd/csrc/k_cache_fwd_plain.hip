// k_cache_fwd_plain.hip -- attention over a paged cache, many queries a head: plain pages.
#include "attn_fwd.h"

using namespace attn;

bool nnk_cache_forward_plain(const Args& a, const cache::Pages& p, bool half, hipStream_t s, const char* what) {
    return NNK_ATTN_DISPATCH(a, half, Forward<1 + NN_CACHE_PLAIN>::template launch, a, p, s, what);
}
