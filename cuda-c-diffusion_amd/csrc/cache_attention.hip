// cache_attention.hip -- the launcher of attention over a paged cache: checks of the call,
// workspace, choice of the kernel.
#include "attn_common.h"
#include "cache_common.h"

namespace {
using namespace attn;
using cache::Pages;

// A wave a query: 64 keys at a time, one a lane, then a feature or two a lane.
template <typename T, bool FP4>
__global__ __launch_bounds__(64) void cache_attention_kernel(Args a, Pages p) {
    __shared__ float q[128];
    const int lane = threadIdx.x, i = blockIdx.x % a.len_q, head = blockIdx.x / a.len_q % a.heads, b = blockIdx.x / a.len_q / a.heads;
    const int kv = head / a.group, keys = keys_of(a, b), pos = start_of(a, b) + i, limit = limit_of(a, b, keys, pos);
    const T* from = (const T*)a.q + b * a.qs[0] + i * a.qs[1] + head * a.qs[2];
    for (int d = lane; d < 128; d += 64) q[d] = d < a.dim ? (float)from[d] : 0.0f;
    __syncthreads();
    const auto value = [&](const char* block, int slot, int d) -> float {
        const char* row = block + slot * p.row_bytes;
        if constexpr (FP4) {
            const unsigned byte = *(const unsigned char*)(row + d / 2);
            const unsigned scale = *(const unsigned char*)(block + p.scales + slot * p.groups + d / cache::kGroup);
            cache::f32x2 v[4];
            cache::values8(d & 1 ? byte >> 4 : byte & 15, cache::scale_of(scale), v);
            return v[0][0];
        } else {
            return (float)((const T*)row)[d];
        }
    };
    float m = -INFINITY, l = 0.0f, o[2] = {0.0f, 0.0f};
    for (int k0 = 0; k0 < limit; k0 += 64) {
        const int key = k0 + lane, page = key < limit ? p.page_of(b, key) : -1, slot = p.slot_of(key);
        float x = -INFINITY;
        if (page >= 0) {
            const char* block = p.k + p.block_at(page, kv);
            x = 0.0f;
            for (int d = 0; d < a.dim; ++d) x = fmaf(q[d], value(block, slot, d), x);
            x *= a.c1;
            if (a.c2 != 0.0f) x = tanhf(x) * a.c2;
            if (a.buckets) {
                const int n = min(max(key - pos, -a.max_distance), a.max_distance) + a.max_distance;
                x += a.bias[(size_t)min(max(a.bucket[n], 0), a.buckets - 1) * a.heads + head] * kLog2e;
            }
        }
        float top = fmaxf(m, x);
        for (int n = 1; n < 64; n <<= 1) top = fmaxf(top, __shfl_xor(top, n));
        if (top == -INFINITY) continue;
        const float g = exp2f(m - top), w = exp2f(x - top);
        m = top;
        l = l * g + nnk::wave_sum(w);
        o[0] *= g;
        o[1] *= g;
        for (int n = 0; n < 64; ++n) {
            const int from_page = __shfl(page, n);
            const float share = __shfl(w, n);
            if (from_page < 0) continue;
            const char* block = p.v + p.block_at(from_page, kv);
            for (int j = 0; j < 2; ++j)
                if (lane + 64 * j < a.dim) o[j] = fmaf(share, value(block, p.slot_of(k0 + n), lane + 64 * j), o[j]);
        }
    }
    T* out = (T*)a.out + b * a.os[0] + i * a.os[1] + head * a.os[2];
    for (int j = 0; j < 2; ++j)
        if (lane + 64 * j < a.dim) out[lane + 64 * j] = (T)(l == 0.0f ? 0.0f : o[j] / l);
    if (lane == 0) a.lse[((size_t)b * a.heads + head) * a.len_q + i] = l == 0.0f ? -INFINITY : (m + log2f(l)) * kLn2;
}

bool fits(Pages& p, const NnAttention* a, const NnCache* c, bool pools, const char* what) {
    NNK_REQUIRE_RET(a, false, what, "%s: null description", what);
    if (!nnk_cache_take(p, c, a->dtype, a->kv_heads, a->head_dim, pools, what)) return false;
    NNK_REQUIRE_RET(!a->doc_q && !a->doc_k, false, what, "%s: documents", what);
    NNK_REQUIRE_RET(a->batch <= c->requests, false, what, "%s: batch=%d of a cache of %d requests", what, a->batch, c->requests);
    NNK_REQUIRE_RET(a->len_k <= (long long)c->table_pages * c->page_tokens, false, what,
        "%s: len_k=%d does not fit in %d pages of %d tokens", what, a->len_k, c->table_pages, c->page_tokens);
    return true;
}

}  // namespace

extern "C" {

size_t nnhip_cache_attention_workspace(const NnAttention* a, const NnCache* c) {
    const char* what = "nnhip_cache_attention_workspace";
    Pages p;
    fits(p, a, c, false, what);
    return 0;
}

void launch_cache_attention_forward(void* out, float* lse, const void* q, const NnAttention* a, const NnCache* c,
    float* workspace, hipStream_t s) {
    const char* what = "launch_cache_attention_forward";
    Pages p;
    Args args;
    if (!fits(p, a, c, true, what)) return;
    if (!nnk_attention_take(args, a, false, what)) return;
    if (!a->batch || !a->len_q) return;
    NNK_REQUIRE(out && lse && q, what, "%s: null pointer", what);
    const long long n[3] = {a->batch, a->len_q, a->heads};
    NNK_REQUIRE(nnk_rows_apart(3, a->out_stride, n, a->head_dim), what, "%s: rows of out overlap (strides %lld, %lld, %lld)",
        what, a->out_stride[0], a->out_stride[1], a->out_stride[2]);
    args.q = q;
    args.out = out;
    args.lse = lse;
    const unsigned blocks = (unsigned)((long long)a->batch * a->heads * a->len_q);
    if (a->dtype == NN_BF16) {
        if (p.groups) cache_attention_kernel<bf16, true><<<blocks, 64, 0, s>>>(args, p);
        else cache_attention_kernel<bf16, false><<<blocks, 64, 0, s>>>(args, p);
    } else {
        if (p.groups) cache_attention_kernel<float, true><<<blocks, 64, 0, s>>>(args, p);
        else cache_attention_kernel<float, false><<<blocks, 64, 0, s>>>(args, p);
    }
    nnk_after_launch(what, s);
}

}  // extern "C"
