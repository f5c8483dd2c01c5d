// k_cache_fwd_mxfp4.hip -- attention over a paged cache, many queries a head: pages of 4 bits.
#include "attn_fwd.h"

using namespace attn;

bool nnk_cache_forward_mxfp4(const Args& a, const cache::Pages& p, hipStream_t s, const char* what) {
    return NNK_ATTN_DISPATCH_OF(bf16, a, Forward<1 + NN_CACHE_MXFP4>::template launch, a, p, s, what);
}
