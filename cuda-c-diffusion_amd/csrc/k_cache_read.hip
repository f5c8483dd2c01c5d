// k_cache_read.hip -- rows of the cache as tensors.
//
// A thread takes 8 features of a row: 4 bytes and a scale of 4-bit pages, or the values
// themselves.  Memory bounds it: every byte is read and written once.
#include "cache_common.h"

#include <algorithm>

namespace {
using namespace cache;

constexpr int kTpb = 256;
constexpr int kFeatures = 8;  // of a thread

struct Read {
    void *k, *v;
    Pages pages;
    long long ks[2], vs[2];
    const int *request, *place;
    int tokens, kv_heads, dim, chunks;
    nnk::FastDiv by_chunks, by_heads;
    unsigned total;
    bool vec;
};

template <typename T, bool FP4>
__global__ __launch_bounds__(kTpb) void cache_read_kernel(Read a) {
    const unsigned n = blockIdx.x * kTpb + threadIdx.x;
    if (n >= a.total) return;
    unsigned row, chunk, t, side;
    a.by_chunks.divmod(n, row, chunk);
    a.by_heads.divmod(row, t, side);  // side: keys' heads, then values'
    const int place = a.place[t], d0 = (int)chunk * kFeatures;
    if (place < 0) return;
    const bool values = side >= (unsigned)a.kv_heads;
    const int head = (int)side - (values ? a.kv_heads : 0);
    const int page = a.pages.page_of(a.request ? a.request[t] : (int)t, place), slot = a.pages.slot_of(place);
    T x[kFeatures];
#pragma unroll
    for (int j = 0; j < kFeatures; ++j) x[j] = (T)0.0f;
    if (page >= 0) {
        const char* block = (values ? a.pages.v : a.pages.k) + a.pages.block_at(page, head);
        const char* from = block + slot * a.pages.row_bytes;
        if constexpr (FP4) {
            const unsigned code = *reinterpret_cast<const unsigned*>(from + d0 / 2);
            const float scale = scale_of(*reinterpret_cast<const unsigned char*>(block + a.pages.scales + slot * a.pages.groups + d0 / kGroup));
            typedef T T2 __attribute__((ext_vector_type(2)));
            T2 y[4];
            values8(code, scale, y);
#pragma unroll
            for (int j = 0; j < kFeatures; ++j) x[j] = y[j / 2][j % 2];
        } else {
#pragma unroll
            for (int j = 0; j < kFeatures * (int)sizeof(T); j += 16)  // rows are padded to 16 bytes
                if (d0 * (int)sizeof(T) + j < a.pages.row_bytes)
                    __builtin_memcpy(reinterpret_cast<char*>(x) + j, __builtin_assume_aligned(from + d0 * sizeof(T) + j, 16), 16);
        }
    }
    T* to = (T*)(values ? a.v : a.k) + t * (values ? a.vs[0] : a.ks[0]) + head * (values ? a.vs[1] : a.ks[1]);
    constexpr int CE = 16 / (int)sizeof(T);
#pragma unroll
    for (int j = 0; j < kFeatures; j += CE) {
        if (a.vec) {
            if (d0 + j < a.dim) __builtin_memcpy(__builtin_assume_aligned(to + d0 + j, 16), x + j, 16);
        } else {
#pragma unroll
            for (int i = j; i < j + CE; ++i)
                if (d0 + i < a.dim) to[d0 + i] = x[i];
        }
    }
}

template <typename T>
void launch(const Read& p, hipStream_t s, const char* what) {
    const unsigned blocks = (p.total + kTpb - 1) / kTpb;
    if (p.pages.groups) cache_read_kernel<T, true><<<blocks, kTpb, 0, s>>>(p);
    else cache_read_kernel<T, false><<<blocks, kTpb, 0, s>>>(p);
    nnk_after_launch(what, s);
}

}  // namespace

extern "C" void launch_cache_read(void* k, void* v, const NnCacheRead* a, const NnCache* c, hipStream_t s) {
    const char* what = "launch_cache_read";
    NNK_REQUIRE(a, what, "%s: null description", what);
    Read p = {};
    if (!nnk_cache_take(p.pages, c, a->dtype, a->kv_heads, a->head_dim, true, what)) return;
    NNK_REQUIRE(a->tokens >= 0, what, "%s: tokens=%d is negative", what, a->tokens);
    if (!a->tokens) return;
    NNK_REQUIRE(k && v, what, "%s: null pointer", what);
    NNK_REQUIRE(a->place, what, "%s: null place", what);
    const long long n[2] = {a->tokens, a->kv_heads};
    NNK_REQUIRE(nnk_rows_apart(2, a->k_stride, n, a->head_dim), what, "%s: rows of k overlap (strides %lld, %lld)", what,
        a->k_stride[0], a->k_stride[1]);
    NNK_REQUIRE(nnk_rows_apart(2, a->v_stride, n, a->head_dim), what, "%s: rows of v overlap (strides %lld, %lld)", what,
        a->v_stride[0], a->v_stride[1]);
    p.chunks = (a->head_dim + kFeatures - 1) / kFeatures;
    const long long total = 2LL * a->tokens * a->kv_heads * p.chunks;
    NNK_REQUIRE(total <= (1LL << 31) - kTpb, what, "%s: too many rows", what);  // of the divisions and the launch
    const long long e = a->dtype == NN_BF16 ? 8 : 4;
    p.vec = a->head_dim % e == 0 && nnk::aligned16(k) && nnk::aligned16(v);
    for (int i = 0; i < 2; ++i) {
        p.ks[i] = a->k_stride[i];
        p.vs[i] = a->v_stride[i];
        p.vec = p.vec && p.ks[i] % e == 0 && p.vs[i] % e == 0;
    }
    p.k = k;
    p.v = v;
    p.request = a->request;
    p.place = a->place;
    p.tokens = a->tokens;
    p.kv_heads = a->kv_heads;
    p.dim = a->head_dim;
    p.total = (unsigned)total;
    p.by_chunks = nnk::FastDiv((uint32_t)p.chunks);
    p.by_heads = nnk::FastDiv((uint32_t)(2 * a->kv_heads));
    if (a->dtype == NN_BF16) launch<bf16>(p, s, what);
    else launch<float>(p, s, what);
}
