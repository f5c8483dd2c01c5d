// cache_attention.hip -- the launcher of attention over a paged cache: checks of the call,
// workspace, choice of the kernel.
#include "attn_common.h"
#include "cache_common.h"

namespace {
using namespace attn;
using cache::Pages;

bool few_plain(const NnAttention* a) { return nnk_cache_is_few(a, false); }
bool few_four_bits(const NnAttention* a) { return nnk_cache_is_few(a, true); }

// Whether a call can be had; with `args`, what its kernels take.
bool fits(Args* args, Pages& p, const NnAttention* a, const NnCache* c, const char* what) {
    NNK_REQUIRE_RET(a, false, what, "%s: null description", what);
    if (!nnk_cache_take(p, c, a->dtype, a->kv_heads, a->head_dim, args != nullptr, what)) return false;
    NNK_REQUIRE_RET(!a->doc_q && !a->doc_k, false, what, "%s: documents", what);
    NNK_REQUIRE_RET(a->batch <= c->requests, false, what, "%s: batch=%d of a cache of %d requests", what, a->batch, c->requests);
    NNK_REQUIRE_RET(a->len_k <= (long long)c->table_pages * c->page_tokens, false, what,
        "%s: len_k=%d does not fit in %d pages of %d tokens", what, a->len_k, c->table_pages, c->page_tokens);
    const auto few = p.groups ? few_four_bits : few_plain;
    if (!(args ? nnk_attention_take(*args, a, false, what, few) : nnk_attention_sizes_fit(a, false, what, few))) return false;
    NNK_REQUIRE_RET(!few(a) || nnk_cache_few_fits(a), false, what, "%s: too many rows (batch=%d heads=%d len_q=%d)", what,
        a->batch, a->heads, a->len_q);
    return true;
}

// Whether rows of 16-byte chunks can be read and written: strides here, pointers by the caller.
bool by_16(const NnAttention* a) {
    const long long e = a->dtype == NN_BF16 ? 8 : 4;
    bool ok = a->head_dim % e == 0;
    for (int i = 0; i < 3; ++i) ok = ok && a->q_stride[i] % e == 0 && a->out_stride[i] % e == 0;
    return ok;
}

}  // namespace

extern "C" {

size_t nnhip_cache_attention_workspace(const NnAttention* a, const NnCache* c) {
    const char* what = "nnhip_cache_attention_workspace";
    Pages p;
    return fits(nullptr, p, a, c, what) ? nnk_cache_few_floats(a) : 0;
}

void launch_cache_attention_forward(void* out, float* lse, const void* q, const NnAttention* a, const NnCache* c,
    float* workspace, hipStream_t s) {
    const char* what = "launch_cache_attention_forward";
    Pages p;
    Args args;
    if (!fits(&args, p, a, c, what)) return;
    if (!a->batch || !a->len_q) return;
    NNK_REQUIRE(out && lse && q, what, "%s: null pointer", what);
    const long long n[3] = {a->batch, a->len_q, a->heads};
    NNK_REQUIRE(nnk_rows_apart(3, a->out_stride, n, a->head_dim), what, "%s: rows of out overlap (strides %lld, %lld, %lld)",
        what, a->out_stride[0], a->out_stride[1], a->out_stride[2]);
    const bool few = nnk_cache_is_few(a, p.groups > 0);
    NNK_REQUIRE(!few || !nnk_cache_few_parted(a) || workspace, what, "%s: null workspace", what);
    NNK_REQUIRE(nnk::aligned16(workspace), what, "%s: workspace is not aligned to 16 bytes", what);
    args.q = q;
    args.out = out;
    args.lse = lse;
    args.vec = by_16(a) && nnk::aligned16(q) && nnk::aligned16(out);
    if (few) return nnk_cache_few(args, p, a, workspace, s, what);
    args.q_rows = ((long long)a->len_q + kRows - 1) / kRows * a->heads * a->batch < kSplitBelow ? kRows / 2 : kRows;
    if (p.groups) nnk_cache_forward_mxfp4(args, p, s, what);
    else nnk_cache_forward_plain(args, p, a->dtype == NN_BF16, s, what);
}

}  // extern "C"
