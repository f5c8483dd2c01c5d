// k_attn_fwd.hip -- attention, many queries a head: the launches of tensors; blocks of documents
// and the order of tiles.
#include "attn_fwd.h"

namespace {
using namespace attn;

// Documents of a block of 64 positions: least and largest, whether any is negative.
__global__ __launch_bounds__(64) void block_docs_kernel(int4* out, const int* docs, int len, int blocks) {
    const int b = blockIdx.x / blocks, i = blockIdx.x % blocks, at = i * kBlock + (int)threadIdx.x;
    const int d = at < len ? docs[(size_t)b * len + at] : -1;
    int lo = d >= 0 ? d : INT32_MAX, hi = d >= 0 ? d : INT32_MIN;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
        lo = min(lo, __shfl_xor(lo, m));
        hi = max(hi, __shfl_xor(hi, m));
    }
    const int negative = __any(d < 0);
    if (threadIdx.x == 0) out[blockIdx.x] = int4{lo, hi, negative, 0};
}

// A request's tiles of `own` positions by falling number of blocks that they meet on the
// other axis, ties by their number.  One workgroup counts a request's pairs of a tile and a
// block, up to 64 of them a thread; more (from some 23000 packed tokens on) go in their own
// order.  That limit is of the counting, not of its use: 32768 packed tokens of 16 heads of 72
// took 399 us with an order and 411 without, a training step of 24576 causal ones 1395 and 1481.
constexpr int kOrderTpb = 1024, kOrderBlocks = 1024, kOrderTiles = 512;
__global__ __launch_bounds__(kOrderTpb) void tile_order_kernel(int* order, Args a, bool keys, int own, int tiles) {
    __shared__ int4 other[kOrderBlocks];
    __shared__ int4 mine[kOrderTiles];
    __shared__ int work[kOrderTiles];
    const int b = blockIdx.x, nq = (a.len_q + kBlock - 1) / kBlock, nk = (a.len_k + kBlock - 1) / kBlock;
    const int blocks = keys ? nq : nk, held = keys_of(a, b), start = start_of(a, b);
    for (int i = threadIdx.x; i < blocks; i += kOrderTpb)
        other[i] = keys ? a.query_docs[(size_t)b * nq + i] : a.key_docs[(size_t)b * nk + i];
    for (int t = threadIdx.x; t < tiles; t += kOrderTpb) {
        const int first = t * own / kBlock, count = own / kBlock;
        mine[t] = keys ? key_docs_of(a, b, first, count) : query_docs_of(a, b, first, count);
        work[t] = 0;
    }
    __syncthreads();
    for (int n = threadIdx.x; n < tiles * blocks; n += kOrderTpb) {
        const int t = n / blocks, i = n - t * blocks;
        // the last query of the tile or block, and the first key of the block or tile
        const int q = keys ? min((i + 1) * kBlock, a.len_q) - 1 : min((t + 1) * own, a.len_q) - 1, k = keys ? t * own : i * kBlock;
        if (docs_meet(other[i], mine[t]) && k < limit_of(a, b, held, start + q)) atomicAdd(&work[t], 1);
    }
    __syncthreads();
    for (int t = threadIdx.x; t < tiles; t += kOrderTpb) {
        int rank = 0;
        for (int u = 0; u < tiles; ++u) rank += work[u] > work[t] || (work[u] == work[t] && u < t);
        order[b * tiles + rank] = t;
    }
}

}  // namespace

bool nnk_attention_forward(const Args& a, bool half, hipStream_t s, const char* what) {
    return NNK_ATTN_DISPATCH(a, half, Forward<0>::template launch, a, cache::Pages{}, s, what);
}

void nnk_attention_docs(Args& a, float* ws, hipStream_t s, const char* what) {
    if (!a.doc_k) return;
    const int nk = (a.len_k + kBlock - 1) / kBlock, nq = (a.len_q + kBlock - 1) / kBlock;
    int4* out = reinterpret_cast<int4*>(ws);
    const auto blocks_of = [&](int4* to, const int* docs, int len, int n) {
        if (!n) return;
        block_docs_kernel<<<(unsigned)(a.batch * n), 64, 0, s>>>(to, docs, len, n);
        nnk_after_launch(what, s);
    };
    a.key_docs = a.query_docs = out;
    blocks_of(out, a.doc_k, a.len_k, nk);
    if (a.doc_q == a.doc_k && a.len_q == a.len_k) return;
    a.query_docs = out += (size_t)a.batch * nk;
    blocks_of(out, a.doc_q, a.len_q, nq);
}

const int* nnk_attention_order(const Args& a, bool keys, int own, float* order, hipStream_t s, const char* what) {
    const int len = keys ? a.len_k : a.len_q, tiles = (len + own - 1) / own;
    const int blocks = ((keys ? a.len_q : a.len_k) + kBlock - 1) / kBlock;
    if (a.batch > kMostHeads || tiles < 2 || tiles > kOrderTiles || blocks > kOrderBlocks || tiles * blocks > 64 * kOrderTpb) return nullptr;
    int* to = reinterpret_cast<int*>(order);
    tile_order_kernel<<<(unsigned)a.batch, kOrderTpb, 0, s>>>(to, a, keys, own, tiles);
    nnk_after_launch(what, s);
    return to;
}
