// k_qk_norm_rope.hip -- each head's query and key normalised and turned by its position,
// and the gradients.
//
// Forward, a row x of head_dim features:  y = x r w,  r = rsqrt(mean(x^2) + eps);  then the
// pairs of y turn.  Backward: the gradient g of y is the outputs' turned back,
//     dw = sum over rows of g x r,   dx = r (g w - x r mean(g w x r)).
// Both read a row once and write it once; at the sizes that matter memory bounds them.  A
// row belongs to the G lanes of one group, 16 bytes a lane, so that the two sums are
// shuffles in the group; the pair's other member, half a rotation away, comes from the
// group's row in LDS (interleaved pairs are one lane's).  A workgroup takes whole tokens,
// whose sines and cosines it forms once for all their heads.
#include "nn_attention.h"
#include "nnk_common.h"

#include <algorithm>

namespace {

typedef __bf16 bf16;
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

constexpr int kTpb = 256;
constexpr int kMaxDim = 256;
constexpr int kAngles = 2048;     // sines and cosines of a workgroup's tokens
constexpr int kGradGroups = 1024; // workgroups of the backward pass at most: rows of its partial sums

struct Rope {
    const void *q, *k;
    void *q_out, *k_out;                // forward
    const void *dq_out, *dk_out;        // backward
    void *dq, *dk;
    float* partial;                     // [workgroups, 2, dim] sums for the weights' gradients
    long long qs[2], ks[2], qos[2], kos[2];
    const float *q_weight, *k_weight;
    const int* pos;
    const double* freq;
    int tokens, heads, all_heads, dim, half, axes, per_axis, interleaved;
    int tokens_each, head_parts;        // tokens of a workgroup at a time; workgroups that share them
    float eps, inv_dim;
    bool vec;
};

template <typename T, int G>
struct Row {
    static constexpr int CE = 16 / (int)sizeof(T);
    static constexpr int kGroups = kTpb / G;

    static __device__ __forceinline__ u32x4 load(const T* row, int d0, const Rope& a) {
        u32x4 v = {0, 0, 0, 0};
        if (a.vec) {
            if (d0 < a.dim) v = *reinterpret_cast<const u32x4*>(row + d0);
        } else {
            T e[CE];
#pragma unroll
            for (int j = 0; j < CE; ++j) e[j] = d0 + j < a.dim ? row[d0 + j] : (T)0.0f;
            __builtin_memcpy(&v, e, 16);
        }
        return v;
    }
    static __device__ __forceinline__ void floats(const u32x4& v, float* x) {
        T e[CE];
        __builtin_memcpy(e, &v, 16);
#pragma unroll
        for (int j = 0; j < CE; ++j) x[j] = (float)e[j];
    }
    static __device__ __forceinline__ void store(T* row, int d0, const Rope& a, const float* x) {
        T e[CE];
#pragma unroll
        for (int j = 0; j < CE; ++j) e[j] = (T)x[j];
        if (a.vec) {
            if (d0 < a.dim) __builtin_memcpy(row + d0, e, 16);
        } else {
#pragma unroll
            for (int j = 0; j < CE; ++j)
                if (d0 + j < a.dim) row[d0 + j] = e[j];
        }
    }
    static __device__ __forceinline__ float group_sum(float v) {
#pragma unroll
        for (int m = 1; m < G; m <<= 1) v += __shfl_xor(v, m);
        return v;
    }
    // Turns the pairs of the group's row, whose features d0.. of this lane are y; `back`: by
    // the opposite angle.  `row`: the group's floats in LDS.
    static __device__ __forceinline__ void turn(float* y, int d0, float* row, const float2* cs, const Rope& a, float back) {
        if (a.interleaved) {
#pragma unroll
            for (int j = 0; j < CE; j += 2) {
                const int p = (d0 + j) / 2;
                if (p >= a.half) continue;
                const float2 t = cs[p];
                const float s = back * t.y, u = y[j], v = y[j + 1];
                y[j] = u * t.x - v * s;
                y[j + 1] = u * s + v * t.x;
            }
            return;
        }
        if (!a.half) return;
        // the group's lanes are in one wave, whose LDS accesses are in order
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int j = 0; j < CE; j += 4) nnk::st4(row + d0 + j, make_float4(y[j], y[j + 1], y[j + 2], y[j + 3]));
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int j = 0; j < CE; ++j) {
            const int d = d0 + j;
            if (d >= 2 * a.half) continue;
            const bool first = d < a.half;
            const float2 t = cs[first ? d : d - a.half];
            const float other = row[first ? d + a.half : d - a.half];
            const float s = first ? -back * t.y : back * t.y;
            y[j] = y[j] * t.x + other * s;
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
};

// Cosine and sine of each pair of `count` tokens.  The angle is formed in 64 bits and
// reduced there to a fraction of a turn, so that it is as exact at position 2^30 as at 1.
__device__ __forceinline__ void angles(float2* cs, const Rope& a, int token0, int count) {
    for (int i = threadIdx.x; i < count * a.half; i += kTpb) {
        const int t = i / a.half, p = i - t * a.half;
        double turns = (double)a.pos[(size_t)(token0 + t) * a.axes + p / a.per_axis] * a.freq[p] * 0.15915494309189533577;
        turns -= rint(turns);
        float s, c;
        sincospif(2.0f * (float)turns, &s, &c);
        cs[i] = make_float2(c, s);
    }
}

template <typename T, int G>
__device__ __forceinline__ void weights(float* w, const float* from, int d0, int dim) {
#pragma unroll
    for (int j = 0; j < Row<T, G>::CE; ++j) w[j] = d0 + j < dim ? (from ? from[d0 + j] : 1.0f) : 0.0f;
}

// A row's token, head and place in a tensor of queries or keys.
struct Place {
    int token, head;
    bool key;
};
__device__ __forceinline__ Place place(const Rope& a, int token0, int head0, int heads, int r) {
    const int t = r / heads, h = head0 + r - t * heads;
    return {token0 + t, h < a.heads ? h : h - a.heads, h >= a.heads};
}
template <typename T>
__device__ __forceinline__ T* row_of(void* q, void* k, const long long* qs, const long long* ks, const Place& p) {
    return p.key ? (T*)k + p.token * ks[0] + p.head * ks[1] : (T*)q + p.token * qs[0] + p.head * qs[1];
}
template <typename T>
__device__ __forceinline__ const T* row_of(const void* q, const void* k, const long long* qs, const long long* ks,
    const Place& p) {
    return row_of<T>(const_cast<void*>(q), const_cast<void*>(k), qs, ks, p);
}

template <typename T, int G>
__global__ __launch_bounds__(kTpb) void qk_norm_rope_kernel(Rope a) {
    using R = Row<T, G>;
    constexpr int CE = R::CE;
    __shared__ float2 cs[kAngles];
    __shared__ __attribute__((aligned(16))) float rows[R::kGroups][G * CE];
    const int group = threadIdx.x / G, d0 = (threadIdx.x % G) * CE;
    const int part = blockIdx.x % a.head_parts, token0 = blockIdx.x / a.head_parts * a.tokens_each;
    const int tokens = min(a.tokens_each, a.tokens - token0);
    const int each = (a.all_heads + a.head_parts - 1) / a.head_parts, head0 = part * each;
    const int heads = min(each, a.all_heads - head0);
    if (heads <= 0) return;
    float wq[CE], wk[CE];
    weights<T, G>(wq, a.q_weight, d0, a.dim);
    weights<T, G>(wk, a.k_weight, d0, a.dim);
    const int n = tokens * heads;
    u32x4 next = {0, 0, 0, 0};
    if (group < n) next = R::load(row_of<T>(a.q, a.k, a.qs, a.ks, place(a, token0, head0, heads, group)), d0, a);
    angles(cs, a, token0, tokens);
    __syncthreads();
    for (int r = group; r < n; r += R::kGroups) {
        float x[CE];
        R::floats(next, x);
        const Place p = place(a, token0, head0, heads, r);
        if (r + R::kGroups < n)
            next = R::load(row_of<T>(a.q, a.k, a.qs, a.ks, place(a, token0, head0, heads, r + R::kGroups)), d0, a);
        float ss = 0.0f;
#pragma unroll
        for (int j = 0; j < CE; ++j) ss = fmaf(x[j], x[j], ss);
        const float rstd = rsqrtf(R::group_sum(ss) * a.inv_dim + a.eps);
#pragma unroll
        for (int j = 0; j < CE; ++j) x[j] = x[j] * rstd * (p.key ? wk[j] : wq[j]);
        R::turn(x, d0, rows[group], cs + (p.token - token0) * a.half, a, 1.0f);
        R::store(row_of<T>(a.q_out, a.k_out, a.qos, a.kos, p), d0, a, x);
    }
}

template <typename T, int G>
__global__ __launch_bounds__(kTpb) void qk_norm_rope_grad_kernel(Rope a) {
    using R = Row<T, G>;
    constexpr int CE = R::CE;
    __shared__ float2 cs[kAngles];
    __shared__ __attribute__((aligned(16))) float rows[R::kGroups][G * CE];
    const int group = threadIdx.x / G, d0 = (threadIdx.x % G) * CE;
    float wq[CE], wk[CE], sum_q[CE], sum_k[CE];
    weights<T, G>(wq, a.q_weight, d0, a.dim);
    weights<T, G>(wk, a.k_weight, d0, a.dim);
#pragma unroll
    for (int j = 0; j < CE; ++j) sum_q[j] = sum_k[j] = 0.0f;
    for (long long at = (long long)blockIdx.x * a.tokens_each; at < a.tokens; at += (long long)gridDim.x * a.tokens_each) {
        const int token0 = (int)at, tokens = min(a.tokens_each, a.tokens - token0), n = tokens * a.all_heads;
        u32x4 next_x = {0, 0, 0, 0}, next_g = {0, 0, 0, 0};
        const auto load = [&](int r) {
            const Place p = place(a, token0, 0, a.all_heads, r);
            next_x = R::load(row_of<T>(a.q, a.k, a.qs, a.ks, p), d0, a);
            next_g = R::load(row_of<T>(a.dq_out, a.dk_out, a.qos, a.kos, p), d0, a);
        };
        if (group < n) load(group);
        __syncthreads();
        angles(cs, a, token0, tokens);
        __syncthreads();
        for (int r = group; r < n; r += R::kGroups) {
            float x[CE], g[CE];
            R::floats(next_x, x);
            R::floats(next_g, g);
            const Place p = place(a, token0, 0, a.all_heads, r);
            if (r + R::kGroups < n) load(r + R::kGroups);
            R::turn(g, d0, rows[group], cs + (p.token - token0) * a.half, a, -1.0f);
            float ss = 0.0f, dot = 0.0f;
#pragma unroll
            for (int j = 0; j < CE; ++j) {
                ss = fmaf(x[j], x[j], ss);
                dot = fmaf(x[j], g[j] * (p.key ? wk[j] : wq[j]), dot);
            }
            const float rstd = rsqrtf(R::group_sum(ss) * a.inv_dim + a.eps);
            const float mean = R::group_sum(dot) * rstd * a.inv_dim;
#pragma unroll
            for (int j = 0; j < CE; ++j) {
                const float xn = x[j] * rstd, dw = g[j] * xn;
                sum_q[j] += p.key ? 0.0f : dw;
                sum_k[j] += p.key ? dw : 0.0f;
                x[j] = rstd * (g[j] * (p.key ? wk[j] : wq[j]) - xn * mean);
            }
            R::store(row_of<T>(a.dq, a.dk, a.qs, a.ks, p), d0, a, x);
        }
    }
    if (!a.partial) return;
    // the groups' sums, one feature a thread, in the groups' order
    for (int which = 0; which < 2; ++which) {
        __syncthreads();
#pragma unroll
        for (int j = 0; j < CE; ++j) rows[group][d0 + j] = which ? sum_k[j] : sum_q[j];
        __syncthreads();
        for (int d = threadIdx.x; d < a.dim; d += kTpb) {
            float sum = 0.0f;
            for (int i = 0; i < R::kGroups; ++i) sum += rows[i][d];
            a.partial[((size_t)blockIdx.x * 2 + which) * a.dim + d] = sum;
        }
    }
}

// dw[d] = sum of the workgroups' partial sums, in 64 bits: a wave a feature, a lane's in
// order, the lanes' as a tree.
__global__ __launch_bounds__(kTpb) void qk_norm_weight_grad_kernel(float* dq_weight, float* dk_weight,
    const float* partial, int groups, int dim) {
    const int at = blockIdx.x * (kTpb / 64) + (int)(threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (at >= 2 * dim) return;
    float* to = at < dim ? dq_weight : dk_weight;
    if (!to) return;
    double sum = 0.0;
    for (int i = lane; i < groups; i += 64) sum += partial[(size_t)i * 2 * dim + at];
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) sum += __shfl_xor(sum, m);
    if (lane == 0) to[at < dim ? at : at - dim] = (float)sum;
}

bool shape_fits(const NnQkNormRope* a, const char* what) {
    NNK_REQUIRE_RET(a, false, what, "%s: null description", what);
    NNK_REQUIRE_RET(a->dtype == NN_F32 || a->dtype == NN_BF16, false, what, "%s: unknown dtype %d", what, a->dtype);
    NNK_REQUIRE_RET(a->tokens >= 0 && a->heads >= 0 && a->kv_heads >= 0 && a->heads <= 1 << 20 && a->kv_heads <= 1 << 20,
        false, what, "%s: bad shape tokens=%d heads=%d kv_heads=%d", what, a->tokens, a->heads, a->kv_heads);
    NNK_REQUIRE_RET(a->head_dim >= 1 && a->head_dim <= kMaxDim, false, what, "%s: head_dim=%d is not in 1..%d", what,
        a->head_dim, kMaxDim);
    NNK_REQUIRE_RET(a->rot_dim >= 0 && a->rot_dim <= a->head_dim && a->rot_dim % 2 == 0, false, what,
        "%s: rot_dim=%d is odd or past head_dim=%d", what, a->rot_dim, a->head_dim);
    NNK_REQUIRE_RET(a->axes >= 1 && a->rot_dim / 2 % a->axes == 0, false, what,
        "%s: axes=%d do not divide rot_dim / 2 = %d", what, a->axes, a->rot_dim / 2);
    return true;
}

bool take(Rope& p, const NnQkNormRope* a, const char* what) {
    if (!shape_fits(a, what)) return false;
    NNK_REQUIRE_RET(a->eps >= 0.0f, false, what, "%s: eps=%g is negative", what, a->eps);
    NNK_REQUIRE_RET(!a->tokens || !a->rot_dim || (a->pos && a->freq), false, what, "%s: null pos or freq", what);
    p = Rope{};
    const long long e = a->dtype == NN_BF16 ? 8 : 4;
    p.vec = a->head_dim % e == 0;
    for (int i = 0; i < 2; ++i) {
        p.qs[i] = a->q_stride[i];
        p.ks[i] = a->k_stride[i];
        p.qos[i] = a->q_out_stride[i];
        p.kos[i] = a->k_out_stride[i];
        p.vec = p.vec && (!a->heads || (p.qs[i] % e == 0 && p.qos[i] % e == 0)) &&
            (!a->kv_heads || (p.ks[i] % e == 0 && p.kos[i] % e == 0));
    }
    p.q_weight = a->q_weight;
    p.k_weight = a->k_weight;
    p.pos = a->pos;
    p.freq = a->freq;
    p.tokens = a->tokens;
    p.heads = a->heads;
    p.all_heads = a->heads + a->kv_heads;
    p.dim = a->head_dim;
    p.half = a->rot_dim / 2;
    p.axes = a->axes;
    p.per_axis = std::max(1, p.half / a->axes);
    p.interleaved = a->interleaved;
    p.eps = a->eps;
    p.inv_dim = 1.0f / (float)a->head_dim;
    return true;
}

// Tokens of a workgroup at a time: rows for 8 passes of its groups, as far as their sines
// fit.  Few tokens: one each, and their heads shared by workgroups of one pass.
int tokens_each(const Rope& p, int groups) {
    const int by_rows = std::max(1, 8 * groups / p.all_heads), by_angles = kAngles / std::max(1, p.half);
    return std::min({by_rows, by_angles, std::max(1, p.tokens / kGradGroups)});
}

template <typename T, int G>
void forward(Rope& p, hipStream_t s) {
    constexpr int groups = Row<T, G>::kGroups;
    p.tokens_each = tokens_each(p, groups);
    p.head_parts = p.tokens < kGradGroups ? (p.all_heads + groups - 1) / groups : 1;
    const long long blocks = ((long long)p.tokens + p.tokens_each - 1) / p.tokens_each * p.head_parts;
    qk_norm_rope_kernel<T, G><<<(unsigned)blocks, kTpb, 0, s>>>(p);
}
template <typename T, int G>
void backward(Rope& p, hipStream_t s) {
    p.tokens_each = tokens_each(p, Row<T, G>::kGroups);
    const int blocks = std::min(kGradGroups, (p.tokens + p.tokens_each - 1) / p.tokens_each);
    qk_norm_rope_grad_kernel<T, G><<<(unsigned)blocks, kTpb, 0, s>>>(p);
}
int grad_groups(const Rope& p, int groups) {
    const int each = tokens_each(p, groups);
    return std::min(kGradGroups, (p.tokens + each - 1) / each);
}

// Lanes of a row: a power of two with 16 bytes each.
int lanes_of(const NnQkNormRope* a) {
    const int n = (a->head_dim * (a->dtype == NN_BF16 ? 2 : 4) + 15) / 16;
    return n <= 4 ? 4 : n <= 8 ? 8 : n <= 16 ? 16 : n <= 32 ? 32 : 64;
}

#define ROPE_DISPATCH(FN, p, a, s)                                                     \
    do {                                                                               \
        const bool half_ = (a)->dtype == NN_BF16;                                      \
        switch (lanes_of(a)) {                                                         \
        case 4: half_ ? FN<bf16, 4>(p, s) : FN<float, 4>(p, s); break;                 \
        case 8: half_ ? FN<bf16, 8>(p, s) : FN<float, 8>(p, s); break;                 \
        case 16: half_ ? FN<bf16, 16>(p, s) : FN<float, 16>(p, s); break;              \
        case 32: half_ ? FN<bf16, 32>(p, s) : FN<float, 32>(p, s); break;              \
        default: FN<float, 64>(p, s); break;                                           \
        }                                                                              \
    } while (0)

}  // namespace

extern "C" {

void launch_qk_norm_rope_forward(void* q_out, void* k_out, const void* q, const void* k,
    const NnQkNormRope* a, hipStream_t s) {
    const char* what = "launch_qk_norm_rope_forward";
    Rope p;
    if (!take(p, a, what)) return;
    if (!p.tokens || !p.all_heads) return;
    NNK_REQUIRE((!a->heads || (q && q_out)) && (!a->kv_heads || (k && k_out)), what, "%s: null pointer", what);
    NNK_REQUIRE((long long)p.tokens * p.all_heads < 1LL << 31, what, "%s: too many rows", what);
    p.q = q;
    p.k = k;
    p.q_out = q_out;
    p.k_out = k_out;
    if (a->heads) p.vec = p.vec && nnk::aligned16(q) && nnk::aligned16(q_out);
    if (a->kv_heads) p.vec = p.vec && nnk::aligned16(k) && nnk::aligned16(k_out);
    ROPE_DISPATCH(forward, p, a, s);
    nnk_after_launch(what, s);
}

size_t nnhip_qk_norm_rope_workspace(const NnQkNormRope* a) {
    if (!shape_fits(a, "nnhip_qk_norm_rope_workspace")) return 0;
    return (size_t)std::min(kGradGroups, a->tokens) * 2 * a->head_dim;
}

void launch_qk_norm_rope_backward(void* dq, void* dk, float* dq_weight, float* dk_weight,
    const void* dq_out, const void* dk_out, const void* q, const void* k,
    const NnQkNormRope* a, float* workspace, hipStream_t s) {
    const char* what = "launch_qk_norm_rope_backward";
    Rope p;
    if (!take(p, a, what)) return;
    const bool rows = p.tokens && p.all_heads;
    NNK_REQUIRE(!rows || ((!a->heads || (q && dq && dq_out)) && (!a->kv_heads || (k && dk && dk_out))), what,
        "%s: null pointer", what);
    NNK_REQUIRE((long long)p.tokens * p.all_heads < 1LL << 31, what, "%s: too many rows", what);
    NNK_REQUIRE(!rows || !(dq_weight || dk_weight) || workspace, what, "%s: null workspace", what);
    p.q = q;
    p.k = k;
    p.dq_out = dq_out;
    p.dk_out = dk_out;
    p.dq = dq;
    p.dk = dk;
    if (a->heads) p.vec = p.vec && nnk::aligned16(q) && nnk::aligned16(dq) && nnk::aligned16(dq_out);
    if (a->kv_heads) p.vec = p.vec && nnk::aligned16(k) && nnk::aligned16(dk) && nnk::aligned16(dk_out);
    if (dq_weight || dk_weight) p.partial = workspace;
    int groups = 0;
    if (rows) {
        ROPE_DISPATCH(backward, p, a, s);
        nnk_after_launch(what, s);
        groups = grad_groups(p, kTpb / lanes_of(a));
    }
    if (dq_weight || dk_weight) {
        qk_norm_weight_grad_kernel<<<(unsigned)((2 * p.dim + 3) / 4), kTpb, 0, s>>>(dq_weight, dk_weight, workspace,
            groups, p.dim);
        nnk_after_launch(what, s);
    }
}

}  // extern "C"
