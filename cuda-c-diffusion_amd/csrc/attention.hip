// attention.hip -- the attention launchers: checks of the call, workspaces, order of the
// kernels.
#include "attn_common.h"

#include <cfloat>

namespace {
using namespace attn;

constexpr long long kMostGroups = ((1LL << 32) - 1) / kTpb;  // a launch has fewer than 2^32 threads
constexpr long long kMostRows = (1LL << 31) - 1;

// Workspaces, in floats; documents come first (16-byte records).
size_t docs_floats(const NnAttention* a) {
    if (!a->doc_q) return 0;
    const size_t nk = ((size_t)a->len_k + kBlock - 1) / kBlock, nq = ((size_t)a->len_q + kBlock - 1) / kBlock;
    // with the orders of tiles of 64 positions or more
    return 4 * (size_t)a->batch * (nk + nq) + ((size_t)a->batch * (nk + nq) + 3) / 4 * 4;
}
float* order_of(const NnAttention* a, float* docs, bool keys) {
    const size_t nk = ((size_t)a->len_k + kBlock - 1) / kBlock, nq = ((size_t)a->len_q + kBlock - 1) / kBlock;
    return docs + 4 * (size_t)a->batch * (nk + nq) + (keys ? a->batch * nq : 0);
}
// How the gradients are divided over workgroups.  Key heads that are shared and few tiles of
// keys: the heads apart.  Few workgroups even so: tiles of 64, and the other axis in parts of
// 4 blocks or more, up to two workgroups a CU.  (One head of 1681 tokens, 2 images, was 27
// workgroups' work otherwise.)
void divide(Args& p, const NnAttention* a) {
    const auto up = [](long long n, long long d) { return (n + d - 1) / d; };
    const auto parts = [](long long groups, long long blocks) {
        return groups >= kCus || !groups ? 1 : (int)std::max(1LL, std::min(2 * kCus / groups, blocks / 4));
    };
    const long long batch = a->batch, heads = a->heads;
    const bool apart = heads > a->kv_heads && up(a->len_k, kRows) * a->kv_heads * batch < 4 * kCus;
    const long long owners = (apart ? heads : a->kv_heads) * batch;
    p.heads_each = apart ? 1 : (int)(heads / a->kv_heads);
    p.kv_keys = up(a->len_k, kRows) * owners < kSplitBelow ? kRows / 2 : kRows;
    p.q_splits = parts(up(a->len_k, p.kv_keys) * owners, up(a->len_q, kBlock));
    p.q_rows = up(a->len_q, kRows) * heads * batch < kSplitBelow ? kRows / 2 : kRows;
    p.k_splits = parts(up(a->len_q, p.q_rows) * heads * batch, up(a->len_k, kBlock));
}
// Whether tiles are dealt out by their work: where a launch of a few microseconds more is
// little, and CUs take several.
bool worth_order(const Args& p, const NnAttention* a, bool keys) {
    const long long own = keys ? p.kv_keys : p.q_rows, len = keys ? a->len_k : a->len_q;
    const long long owners = keys ? (long long)a->heads / p.heads_each * p.q_splits : (long long)a->heads * p.k_splits;
    return (len + own - 1) / own * owners * a->batch >= 2 * kCus;
}
size_t by4(size_t n) { return (n + 3) / 4 * 4; }
size_t kv_floats(const NnAttention* a, const Args& p) {
    const size_t parts = (size_t)a->heads / p.heads_each * p.q_splits;
    return parts > (size_t)a->kv_heads ? by4(2 * a->batch * parts * a->len_k * a->head_dim) : 0;
}
size_t q_floats(const NnAttention* a, const Args& p) {
    const size_t rows = (size_t)a->batch * a->heads * p.k_splits * a->len_q;
    return p.k_splits > 1 ? by4(2 * rows) + by4(rows * a->head_dim) : 0;
}
size_t stat_floats(const NnAttention* a) { return 2 * (size_t)a->batch * a->heads * a->len_q; }

// Floats that one forward call takes.
size_t forward_floats(const NnAttention* a) {
    if (!a->batch || !a->len_q) return 0;
    const size_t n = docs_floats(a) + (nnk_attention_is_few(a) ? nnk_attention_few_floats(a) : 0);
    return n ? kTicketWords + n : 0;
}
// What a program lends: enough for the call and for each one of a smaller batch or of shorter
// lengths, which may take more (fewer requests or tokens are divided into more parts).  A
// program's workspaces have the sizes of its largest call.  So bounds over all of them, each
// of which grows with the batch and both lengths.
size_t forward_most(const NnAttention* a) {
    const size_t n = a->batch && a->len_q ? docs_floats(a) + nnk_attention_few_most(a) : 0;
    return n ? kTicketWords + n : 0;
}
size_t backward_most(const NnAttention* a) {
    const auto up = [](long long n, long long d) { return (n + d - 1) / d; };
    const long long batch = a->batch, heads = a->heads, len_q = a->len_q, len_k = a->len_k;
    const long long q_parts = up(len_q, kBlock) / 4, k_parts = up(len_k, kBlock) / 4;
    // an axis in parts: up to two workgroups a CU, of half of kRows rows each (divide())
    constexpr long long kParted = 2 * kCus * (kRows / 2);
    const long long kv_rows = std::max(
        heads > a->kv_heads ? heads * std::min(batch * len_k, 4LL * kCus * kRows / a->kv_heads) : 0,
        q_parts > 1 ? std::min(kParted, batch * heads * len_k * q_parts) : 0);
    const long long q_rows = k_parts > 1 ? std::min(kParted, batch * heads * len_q * k_parts) : 0;
    // tables of distances: of halves of kRows keys below kSplitBelow workgroups
    const long long tables = std::max(std::min(2LL * kSplitBelow, batch * heads * up(len_k, kRows / 2) * std::max(1LL, q_parts)),
        batch * heads * up(len_k, kRows));
    return docs_floats(a) + by4(2 * kv_rows * a->head_dim) + by4(2 * q_rows) + by4(q_rows * a->head_dim) +
        by4(stat_floats(a)) + (a->buckets ? (size_t)tables * (2 * a->max_distance + 1) : 0);
}

// Whether the rows of a tensor that the call writes lie apart; false after recording an error.
bool rows_apart(const long long* stride, int batch, int len, int heads, int dim, const char* name, const char* what) {
    const long long n[3] = {batch, len, heads};
    NNK_REQUIRE_RET(nnk_rows_apart(3, stride, n, dim), false, what, "%s: rows of %s overlap (strides %lld, %lld, %lld)", what,
        name, stride[0], stride[1], stride[2]);
    return true;
}

// Whether rows of 16-byte chunks can be read and written: strides here, pointers by the
// callers.  The offsets of 64 rows have to fit in 32 bits.
bool strides_by_16(const NnAttention* a) {
    const long long e = a->dtype == NN_BF16 ? 8 : 4, far = (1LL << 32) / (16 / e) / 64 - 128;
    bool ok = a->head_dim % e == 0;
    for (int i = 0; i < 3; ++i)
        for (const long long* s : {a->q_stride, a->k_stride, a->v_stride, a->out_stride})
            ok = ok && s[i] % e == 0 && (i != 1 || (s[i] >= 0 && s[i] <= far));
    return ok;
}

}  // namespace

bool nnk_attention_sizes_fit(const NnAttention* a, bool backward, const char* what, bool (*few)(const NnAttention*)) {
    NNK_REQUIRE_RET(a, false, what, "%s: null description", what);
    NNK_REQUIRE_RET(a->dtype == NN_F32 || a->dtype == NN_BF16, false, what, "%s: unknown dtype %d", what, a->dtype);
    NNK_REQUIRE_RET(a->batch >= 0 && a->len_q >= 0 && a->len_k >= 0 && a->len_q <= kMaxLen && a->len_k <= kMaxLen,
        false, what, "%s: bad shape batch=%d len_q=%d len_k=%d", what, a->batch, a->len_q, a->len_k);
    NNK_REQUIRE_RET(a->heads > 0 && a->kv_heads > 0 && a->heads % a->kv_heads == 0, false, what,
        "%s: heads=%d is not a multiple of kv_heads=%d", what, a->heads, a->kv_heads);
    NNK_REQUIRE_RET(a->head_dim >= 1 && a->head_dim <= 128, false, what, "%s: head_dim=%d is not in 1..128", what,
        a->head_dim);
    NNK_REQUIRE_RET(a->buckets >= 0 && a->max_distance >= 0 && a->max_distance <= kMaxDistance, false, what,
        "%s: buckets=%d max_distance=%d (at most %d)", what, a->buckets, a->max_distance, kMaxDistance);
    NNK_REQUIRE_RET(a->heads <= kMostHeads, false, what, "%s: heads=%d (at most %d)", what, a->heads, kMostHeads);
    const auto up = [](long long n, long long d) { return (n + d - 1) / d; };
    const long long rows = std::max(up(a->len_q, kRows), up(a->len_k, kBlock));
    bool fits = rows * a->batch <= kMostRows / a->heads && (long long)a->buckets * a->heads <= kMostRows;
    // workgroups of tiles of queries, of keys, and of documents (of 64 threads)
    const auto launched = [&](long long n) { return n * a->batch <= kMostGroups / a->heads; };
    fits = fits && ((!backward && few(a)) || launched(up(a->len_q, kRows)));
    fits = fits && (!backward || launched(up(a->len_k, kRows)));
    fits = fits && (!a->doc_q || up(std::max(a->len_q, a->len_k), kBlock) * a->batch <= kMostGroups * (kTpb / 64));
    NNK_REQUIRE_RET(fits, false, what, "%s: too many rows (batch=%d heads=%d len_q=%d len_k=%d)", what, a->batch, a->heads,
        a->len_q, a->len_k);
    return true;
}

bool nnk_attention_take(Args& p, const NnAttention* a, bool backward, const char* what, bool (*few)(const NnAttention*)) {
    if (!nnk_attention_sizes_fit(a, backward, what, few)) return false;
    NNK_REQUIRE_RET(a->scale > 0.0f && a->scale < INFINITY, false, what, "%s: scale=%g is not positive", what, a->scale);
    NNK_REQUIRE_RET(a->softcap >= 0.0f && a->softcap < INFINITY, false, what, "%s: softcap=%g is negative", what,
        a->softcap);
    NNK_REQUIRE_RET(a->mask == NN_MASK_NONE || a->mask == NN_MASK_CAUSAL || a->mask == NN_MASK_PREFIX, false, what,
        "%s: unknown mask %d", what, a->mask);
    NNK_REQUIRE_RET(a->mask != NN_MASK_PREFIX || a->prefix, false, what, "%s: null prefix", what);
    NNK_REQUIRE_RET(!a->doc_q == !a->doc_k, false, what, "%s: documents of queries or keys only", what);
    NNK_REQUIRE_RET(!a->buckets || (a->bucket && a->bias), false, what, "%s: null bucket or bias", what);
    p = Args{};
    for (int i = 0; i < 3; ++i) {
        p.qs[i] = a->q_stride[i];
        p.ks[i] = a->k_stride[i];
        p.vs[i] = a->v_stride[i];
        p.os[i] = a->out_stride[i];
    }
    p.batch = a->batch;
    p.len_q = a->len_q;
    p.len_k = a->len_k;
    p.heads = a->heads;
    p.kv_heads = a->kv_heads;
    p.group = a->heads / a->kv_heads;
    p.dim = a->head_dim;
    p.mask = a->mask;
    p.buckets = a->buckets;
    p.max_distance = a->max_distance;
    p.scale = a->scale;
    p.c1 = a->softcap > 0.0f ? a->scale / a->softcap : a->scale * kLog2e;
    p.c2 = a->softcap * kLog2e;
    NNK_REQUIRE_RET(p.c1 < INFINITY && p.c2 < INFINITY, false, what, "%s: scale=%g with softcap=%g overflows", what,
        a->scale, a->softcap);
    NNK_REQUIRE_RET(a->softcap == 0.0f || (p.c1 >= FLT_MIN && p.c2 >= FLT_MIN), false, what,
        "%s: scale=%g with softcap=%g underflows", what, a->scale, a->softcap);
    if (a->softcap > 0.0f) {
        // The series takes s, where its coefficients are all normal values (the last has c1 to
        // the 11th power); else y = c1 s, and no wave goes without the other form.
        const double tanh_of[6] = {1.0, -1.0 / 3, 2.0 / 15, -17.0 / 315, 62.0 / 2835, -1382.0 / 155925};
        const auto series_of = [&](double unit) {  // of s unit
            double power = p.c2 * (p.c1 / unit);
            bool normal = true;
            for (int i = 0; i < 6; ++i, power *= (p.c1 / unit) * (p.c1 / unit)) {
                p.series[i] = (float)(tanh_of[i] * power);
                normal = normal && std::isnormal(p.series[i]);
            }
            return normal;
        };
        p.inv_c2 = 1.0f / p.c2;
        p.unit = 1.0f;
        if (series_of(1.0)) {
            p.small = kSeriesEnd / p.c1;
            p.tiny = kShortSeriesEnd / p.c1;
        } else {
            p.unit = p.c1;
            series_of(p.c1);
        }
        p.near_end = kSeriesEnd * (p.unit / p.c1);
        p.exponent = 2.0f * kLog2e * (p.c1 / p.unit);
    }
    p.q_start = a->q_start;
    p.k_len = a->k_len;
    p.prefix = a->prefix;
    p.doc_q = a->doc_q;
    p.doc_k = a->doc_k;
    p.bucket = a->bucket;
    p.bias = a->bias;
    return true;
}

extern "C" {

size_t nnhip_attention_forward_workspace(const NnAttention* a) {
    if (!nnk_attention_sizes_fit(a, false, "nnhip_attention_forward_workspace")) return 0;
    return forward_most(a);
}

void launch_attention_forward(void* out, float* lse, const void* q, const void* k, const void* v,
    const NnAttention* a, float* workspace, hipStream_t s) {
    const char* what = "launch_attention_forward";
    Args p;
    if (!nnk_attention_take(p, a, false, what)) return;
    if (!a->batch || !a->len_q) return;
    NNK_REQUIRE(out && lse && q && (!a->len_k || (k && v)), what, "%s: null pointer", what);
    if (!rows_apart(a->out_stride, a->batch, a->len_q, a->heads, a->head_dim, "out", what)) return;
    NNK_REQUIRE(!forward_floats(a) || workspace, what, "%s: null workspace", what);
    NNK_REQUIRE(nnk::aligned16(workspace), what, "%s: workspace is not aligned to 16 bytes", what);
    p.q = q;
    p.k = k;
    p.v = v;
    p.out = out;
    p.lse = lse;
    p.vec = strides_by_16(a) && nnk::aligned16(q) && nnk::aligned16(k) && nnk::aligned16(v) && nnk::aligned16(out);
    const bool few = nnk_attention_is_few(a);
    divide(p, a);
    if (a->doc_q) {
        float* docs = workspace + kTicketWords + (few ? nnk_attention_few_floats(a) : 0);
        nnk_attention_docs(p, docs, s, what);
        if (!few && worth_order(p, a, false)) p.row_order = nnk_attention_order(p, false, p.q_rows, order_of(a, docs, false), s, what);
    }
    if (few) nnk_attention_few(p, a->dtype == NN_BF16, workspace, s, what);
    else nnk_attention_forward(p, a->dtype == NN_BF16, s, what);
}

size_t nnhip_attention_backward_workspace(const NnAttention* a) {
    if (!nnk_attention_sizes_fit(a, true, "nnhip_attention_backward_workspace")) return 0;
    return backward_most(a);
}

void launch_attention_backward(void* dq, void* dk, void* dv, float* dbias, const void* dout,
    const void* q, const void* k, const void* v, const void* out, const float* lse,
    const NnAttention* a, float* workspace, hipStream_t s) {
    const char* what = "launch_attention_backward";
    Args p;
    if (!nnk_attention_take(p, a, true, what)) return;
    NNK_REQUIRE(!dbias || a->buckets, what, "%s: a bias gradient without a bias", what);
    const bool has_q = a->batch && a->len_q, has_k = a->batch && a->len_k;
    NNK_REQUIRE(!has_q || (dq && dout && q && out && lse), what, "%s: null pointer of the queries", what);
    NNK_REQUIRE(!has_k || (dk && dv && k && v), what, "%s: null pointer of the keys", what);
    if ((has_q && !rows_apart(a->q_stride, a->batch, a->len_q, a->heads, a->head_dim, "dq", what)) ||
        (has_k && (!rows_apart(a->k_stride, a->batch, a->len_k, a->kv_heads, a->head_dim, "dk", what) ||
            !rows_apart(a->v_stride, a->batch, a->len_k, a->kv_heads, a->head_dim, "dv", what))))
        return;
    NNK_REQUIRE(!(has_q || has_k) || workspace, what, "%s: null workspace", what);
    NNK_REQUIRE(nnk::aligned16(workspace), what, "%s: workspace is not aligned to 16 bytes", what);
    p.q = q;
    p.k = k;
    p.v = v;
    p.out = const_cast<void*>(out);
    p.lse = const_cast<float*>(lse);
    p.dout = dout;
    p.dq = dq;
    p.dk = dk;
    p.dv = dv;
    p.vec = strides_by_16(a);
    for (const void* x : {q, k, v, out, dout, (const void*)dq, (const void*)dk, (const void*)dv})
        p.vec = p.vec && nnk::aligned16(x);
    divide(p, a);
    float* ws = workspace + docs_floats(a);
    if (kv_floats(a, p)) p.kv_sums = ws;
    ws += kv_floats(a, p);
    if (q_floats(a, p)) {
        p.stat_sums = reinterpret_cast<float2*>(ws);
        p.q_sums = ws + by4(2 * (size_t)a->batch * a->heads * p.k_splits * a->len_q);
    }
    ws += q_floats(a, p);
    p.stat = reinterpret_cast<float2*>(ws);
    if (dbias) p.dist_sums = ws + by4(stat_floats(a));
    const bool half = a->dtype == NN_BF16;
    if (has_q && has_k && a->doc_q) {
        nnk_attention_docs(p, workspace, s, what);
        if (worth_order(p, a, false)) p.row_order = nnk_attention_order(p, false, p.q_rows, order_of(a, workspace, false), s, what);
        if (worth_order(p, a, true)) p.key_order = nnk_attention_order(p, true, p.kv_keys, order_of(a, workspace, true), s, what);
    }
    if (has_q && !nnk_attention_backward_q(p, half, s, what)) return;
    if (has_k && !nnk_attention_backward_kv(p, half, s, what)) return;
    if (dbias) nnk_attention_bias_grad(p, dbias, s, what);
}

}  // extern "C"
