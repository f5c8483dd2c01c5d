// k_cache_read.hip -- rows of the cache as tensors.
//
// A thread takes 8 features of a row at a time: 4 bytes and a scale of 4-bit pages, or the values
// themselves, four rows under way together.  A workgroup has some tokens, whose pages it looks up
// once.  Memory bounds it: every byte is read and written once.  Measured: 32768 tokens, 8 heads of
// 128, 4 bits to bf16 28 us, 6.0 TB/s (69 us with a look-up a thread).
#include "cache_common.h"

#include <algorithm>

namespace {
using namespace cache;

constexpr int kTpb = 256;
constexpr int kFeatures = 8;  // of a thread
constexpr int kMostTokensEach = 64;
constexpr int kAtOnce = 4;

struct Read {
    void *k, *v;
    Pages pages;
    long long ks[2], vs[2];
    const int *request, *place;
    int tokens, kv_heads, dim, chunks, tokens_each;
    nnk::FastDiv by_chunks, by_heads;
    bool vec;
};

template <typename T, bool FP4>
__global__ __launch_bounds__(kTpb) void cache_read_kernel(Read a) {
    __shared__ long long blocks[kMostTokensEach];  // a token's page, as its first head's byte, or -1
    __shared__ int places[kMostTokensEach];
    const int token0 = blockIdx.x * a.tokens_each, tokens = min(a.tokens_each, a.tokens - token0);
    for (int t = threadIdx.x; t < tokens; t += kTpb) {
        const int place = a.place[token0 + t];
        const int page = place < 0 ? -1 : a.pages.page_of(a.request ? a.request[token0 + t] : token0 + t, place);
        places[t] = place;
        blocks[t] = page < 0 ? -1 : a.pages.block_at(page, 0);
    }
    __syncthreads();
    typedef T Chunk __attribute__((ext_vector_type(kFeatures)));
    const unsigned total = (unsigned)tokens * 2 * a.kv_heads * a.chunks;
    for (unsigned n0 = threadIdx.x; n0 < total; n0 += kAtOnce * kTpb) {
        Chunk x[kAtOnce];
        unsigned code[kAtOnce], scale[kAtOnce];
        T* to[kAtOnce];
        int from[kAtOnce];  // first feature, or -1: nothing to write
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
            const unsigned n = n0 + i * kTpb;
            unsigned row, chunk, t, side;
            a.by_chunks.divmod(min(n, total - 1), row, chunk);
            a.by_heads.divmod(row, t, side);  // side: keys' heads, then values'
            const int place = places[t], d0 = (int)chunk * kFeatures;
            const bool values = side >= (unsigned)a.kv_heads;
            const int head = (int)side - (values ? a.kv_heads : 0);
            from[i] = n < total && place >= 0 ? d0 : -1;
            to[i] = (T*)(values ? a.v : a.k) + (token0 + t) * (values ? a.vs[0] : a.ks[0]) + head * (values ? a.vs[1] : a.ks[1]);
            x[i] = Chunk{};
            code[i] = 0;
            scale[i] = 127;
            if (from[i] < 0 || blocks[t] < 0) continue;
            const char* block = (values ? a.pages.v : a.pages.k) + blocks[t] + (long long)head * a.pages.block_bytes;
            const int slot = a.pages.slot_of(place);
            const char* p = block + slot * a.pages.row_bytes;
            if constexpr (FP4) {
                code[i] = *reinterpret_cast<const unsigned*>(p + d0 / 2);
                scale[i] = *reinterpret_cast<const unsigned char*>(block + a.pages.scales + slot * a.pages.groups + d0 / kGroup);
            } else {
#pragma unroll
                for (int j = 0; j < (int)sizeof(Chunk); j += 16)  // rows are padded to 16 bytes
                    if (d0 * (int)sizeof(T) + j < a.pages.row_bytes)
                        __builtin_memcpy(reinterpret_cast<char*>(&x[i]) + j, __builtin_assume_aligned(p + d0 * sizeof(T) + j, 16), 16);
            }
        }
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
            if (from[i] < 0) continue;
            if constexpr (FP4) {
                typedef T T2 __attribute__((ext_vector_type(2)));
                T2 y[4];
                values8(code[i], scale_of(scale[i]), y);
                __builtin_memcpy(&x[i], y, sizeof y);
            }
            constexpr int CE = 16 / (int)sizeof(T);
#pragma unroll
            for (int j = 0; j < kFeatures; j += CE) {
                if (a.vec) {
                    if (from[i] + j < a.dim) {
                        u32x4 y;
                        __builtin_memcpy(&y, reinterpret_cast<const char*>(&x[i]) + j * sizeof(T), 16);
                        __builtin_nontemporal_store(y, reinterpret_cast<u32x4*>(to[i] + from[i] + j));
                    }
                } else {
#pragma unroll
                    for (int k = j; k < j + CE; ++k)
                        if (from[i] + k < a.dim) to[i][from[i] + k] = x[i][k];
                }
            }
        }
    }
}

template <typename T>
void launch(const Read& p, hipStream_t s, const char* what) {
    const unsigned blocks = (unsigned)((p.tokens + (long long)p.tokens_each - 1) / p.tokens_each);
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
    // Tokens of a workgroup: for two passes of its threads, as few as still make four workgroups a CU.
    const int rows = 2 * a->kv_heads * p.chunks;
    p.tokens_each = std::max(1, std::min({kMostTokensEach, 2 * kAtOnce * kTpb / rows, a->tokens / 1024}));
    NNK_REQUIRE((long long)a->tokens / p.tokens_each < (1LL << 32) / kTpb - 1, what, "%s: too many rows", what);  // of a launch
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
    p.by_chunks = nnk::FastDiv((uint32_t)p.chunks);
    p.by_heads = nnk::FastDiv((uint32_t)(2 * a->kv_heads));
    if (a->dtype == NN_BF16) launch<bf16>(p, s, what);
    else launch<float>(p, s, what);
}
