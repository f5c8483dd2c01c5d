// cache.hip -- the cache's description: checks and layout.
#include "cache_common.h"

bool nnk_cache_take(cache::Pages& p, const NnCache* c, int dtype, int kv_heads, int head_dim, bool pools, const char* what) {
    NNK_REQUIRE_RET(c, false, what, "%s: null cache", what);
    NNK_REQUIRE_RET(c->kind == NN_CACHE_PLAIN || c->kind == NN_CACHE_MXFP4, false, what, "%s: unknown kind of cache %d", what,
        c->kind);
    NNK_REQUIRE_RET(dtype == NN_F32 || dtype == NN_BF16, false, what, "%s: unknown dtype %d", what, dtype);
    NNK_REQUIRE_RET(kv_heads >= 1 && kv_heads <= 1 << 16, false, what, "%s: kv_heads=%d is not in 1..%d", what, kv_heads, 1 << 16);
    NNK_REQUIRE_RET(head_dim >= 1 && head_dim <= 128, false, what, "%s: head_dim=%d is not in 1..128", what, head_dim);
    const int n = c->page_tokens;
    NNK_REQUIRE_RET(n >= 16 && n <= 4096 && (n & (n - 1)) == 0, false, what,
        "%s: page_tokens=%d is not a power of two in 16..4096", what, n);
    NNK_REQUIRE_RET(c->pages >= 0 && c->requests >= 0 && c->table_pages >= 0, false, what,
        "%s: bad cache pages=%d requests=%d table_pages=%d", what, c->pages, c->requests, c->table_pages);
    NNK_REQUIRE_RET((long long)c->table_pages * n <= cache::kMostTokens, false, what,
        "%s: table_pages=%d of %d tokens are too many", what, c->table_pages, n);
    p = cache::Pages{};
    const int e = dtype == NN_BF16 ? 2 : 4;
    p.groups = c->kind == NN_CACHE_MXFP4 ? (head_dim + cache::kGroup - 1) / cache::kGroup : 0;
    p.row_bytes = p.groups ? 16 * p.groups : (head_dim * e + 15) / 16 * 16;
    p.scales = n * p.row_bytes;
    p.block_bytes = p.scales + n * p.groups;
    p.page_bytes = (long long)p.block_bytes * kv_heads;
    NNK_REQUIRE_RET(p.page_bytes < 1LL << 32, false, what, "%s: a page of %lld bytes is too large", what, p.page_bytes);
    while (1 << p.shift < n) ++p.shift;
    p.pages = c->pages;
    p.requests = c->requests;
    p.table_pages = c->table_pages;
    p.table = c->table;
    p.k = (char*)c->k;
    p.v = (char*)c->v;
    if (!pools) return true;
    NNK_REQUIRE_RET(c->table || !c->requests || !c->table_pages, false, what, "%s: null table", what);
    NNK_REQUIRE_RET((c->k && c->v) || !c->pages, false, what, "%s: null pool", what);
    NNK_REQUIRE_RET(nnk::aligned16(c->k) && nnk::aligned16(c->v), false, what, "%s: a pool is not aligned to 16 bytes", what);
    const long long apart = p.k < p.v ? p.v - p.k : p.k - p.v;
    NNK_REQUIRE_RET(!c->pages || apart / c->pages >= p.page_bytes, false, what, "%s: the pools of keys and values overlap", what);
    return true;
}

extern "C" size_t nnhip_cache_page_bytes(const NnCache* c, int dtype, int kv_heads, int head_dim) {
    cache::Pages p;
    return nnk_cache_take(p, c, dtype, kv_heads, head_dim, false, "nnhip_cache_page_bytes") ? (size_t)p.page_bytes : 0;
}
