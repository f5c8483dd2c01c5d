// k_qk_norm_rope.hip -- each head's query and key normalised and turned by its position,
// and the gradients.
//
// Forward, a row x of head_dim features:  y = x r w,  r = rsqrt(mean(x^2) + eps);  then the
// pairs of y turn.  Backward: the gradient g of y is the outputs' turned back,
//     dw = sum over rows of g x r,   dx = r (g w - x r mean(g w x r)).
// Both read a row once and write it once; at the sizes that matter memory bounds them.  A
// row belongs to the G lanes of one group, 16 bytes a lane, so that the two sums are
// cross-lane adds in the group.  The pair's other member is one lane's own if pairs are
// interleaved, else half a rotation away, and comes from the group's row in LDS: where that
// is whole 16-byte chunks, by 16-byte accesses in an order without bank conflicts, and the
// lane keeps its sines and cosines in registers for all heads of a token (they took a third
// of the time as element-wise reads).  A workgroup takes whole tokens, whose sines and
// cosines it forms once, first all their queries, then their keys.
//
// Measured: 32768 tokens, 32 + 8 heads of 128, bf16: forward 140-151 us (4.4-4.8 TB/s),
// backward 231-244 us (4.1-4.4; 68 bytes a lane of scratch); eight images of 64 x 64 tokens,
// 16 + 16 heads of 64, fp32: 102 us (5.3 TB/s).
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
    int tokens, heads, kv_heads, all_heads, dim, half, axes, per_axis, interleaved;
    int tokens_each, head_parts;        // tokens of a workgroup at a time; workgroups that share them
    int tokens_all;                     // backward: tokens of a workgroup
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
        v += nnk::dpp_mov<nnk::kDppQuadXor1>(v);
        v += nnk::dpp_mov<nnk::kDppQuadXor2>(v);
        if constexpr (G >= 8) v += nnk::dpp_mov<nnk::kDppRowHalfMirror>(v);
        if constexpr (G >= 16) v += nnk::dpp_mov<nnk::kDppRowMirror>(v);
#pragma unroll
        for (int m = 16; m < G; m <<= 1) v += __shfl_xor(v, m);
        return v;
    }
    // This lane's part in a turn of whole chunks: cosines, signed sines and the lane of the
    // pairs' other members.
    struct Part {
        float cos[CE], sin[CE];
        int other;
    };
    static __device__ __forceinline__ void part_of(Part& t, int d0, const float2* cs, const Rope& a, float back) {
        const int c = d0 / CE, hc = a.half / CE;
        const bool first = c < hc, turns = c < 2 * hc;
        t.other = !turns ? c : first ? c + hc : c - hc;
#pragma unroll
        for (int j = 0; j < CE; ++j) {
            const float2 x = turns ? cs[(first ? c : c - hc) * CE + j] : make_float2(1.0f, 0.0f);
            t.cos[j] = x.x;
            t.sin[j] = first ? -back * x.y : back * x.y;
        }
    }
    static __device__ __forceinline__ void turn(float* y, int d0, float* row, const Part& t) {
        const int c = d0 / CE;
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int j = 0; j < CE; j += 4)
            nnk::st4(row + j * G + 4 * c, make_float4(y[j], y[j + 1], y[j + 2], y[j + 3]));
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int j = 0; j < CE; j += 4) {
            const float4 z = nnk::ld4(row + j * G + 4 * t.other);
            y[j] = y[j] * t.cos[j] + z.x * t.sin[j];
            y[j + 1] = y[j + 1] * t.cos[j + 1] + z.y * t.sin[j + 1];
            y[j + 2] = y[j + 2] * t.cos[j + 2] + z.z * t.sin[j + 2];
            y[j + 3] = y[j + 3] * t.cos[j + 3] + z.w * t.sin[j + 3];
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
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

// Cosine and sine of each pair of `count` tokens.  The angle is formed in 64 bits (off by
// 2^-53 of itself, 2^-24 at 2^29 rad) and reduced there to an eighth of a turn either way, so
// that fp32 rounds what is left of it and not turns: the small one of sine and cosine near a
// quarter turn keeps its digits.
__device__ __forceinline__ void angles(float2* cs, const Rope& a, int token0, int count) {
    for (int i = threadIdx.x; i < count * a.half; i += kTpb) {
        const int t = i / a.half, p = i - t * a.half;
        double turns = (double)a.pos[(size_t)(token0 + t) * a.axes + p / a.per_axis] * a.freq[p] * 0.15915494309189533577;
        turns -= rint(turns);
        const double quarters = rint(4.0 * turns);
        const int q = (int)quarters;
        float s, c;
        sincospif(0.5f * (float)(4.0 * turns - quarters), &s, &c);
        const float x = q & 1 ? s : c, y = q & 1 ? c : s;
        cs[i] = make_float2((q + 1) & 2 ? -x : x, q & 2 ? -y : y);
    }
}

template <typename T, int G>
__device__ __forceinline__ void weights(float* w, const float* from, int d0, int dim) {
#pragma unroll
    for (int j = 0; j < Row<T, G>::CE; ++j) w[j] = d0 + j < dim ? (from ? from[d0 + j] : 1.0f) : 0.0f;
}

// The rows of `tokens` tokens' heads head0 .. head0 + heads - 1, one after another for each
// group: token and head of row r, and how both move on.
struct Rows {
    int token, head, heads, token_step, head_step;
    __device__ __forceinline__ Rows(int r, int step, int heads_) : heads(heads_) {
        token = r / heads;
        head = r - token * heads;
        token_step = step / heads;
        head_step = step - token_step * heads;
    }
    __device__ __forceinline__ void next() {
        token += token_step;
        head += head_step;
        if (head >= heads) {
            head -= heads;
            ++token;
        }
    }
};

// Sines and cosines of a row: the lane's own (CHUNKS) while the token stays, or the table's.
template <typename T, int G, bool CHUNKS>
struct Turner {
    using R = Row<T, G>;
    typename R::Part part;
    int token = -1;
    __device__ __forceinline__ void operator()(float* y, int t, int d0, float* row, const float2* cs, const Rope& a,
        float back) {
        if constexpr (CHUNKS) {
            if (t != token) R::part_of(part, d0, cs + t * a.half, a, back);
            token = t;
            R::turn(y, d0, row, part);
        } else {
            R::turn(y, d0, row, cs + t * a.half, a, back);
        }
    }
};

template <typename T, int G, bool CHUNKS>
__global__ __launch_bounds__(kTpb) void qk_norm_rope_kernel(Rope a) {
    using R = Row<T, G>;
    constexpr int CE = R::CE;
    __shared__ __attribute__((aligned(16))) float2 cs[kAngles];
    __shared__ __attribute__((aligned(16))) float rows[R::kGroups][G * CE];
    const int group = threadIdx.x / G, d0 = (threadIdx.x % G) * CE;
    const int part = blockIdx.x % a.head_parts, token0 = blockIdx.x / a.head_parts * a.tokens_each;
    const int tokens = min(a.tokens_each, a.tokens - token0);
    Turner<T, G, CHUNKS> turn;
    bool ready = false;
    const auto heads_of = [&](const void* in, void* out, const long long* is, const long long* os, const float* weight,
                              int all) {
        const int each = (all + a.head_parts - 1) / a.head_parts, head0 = part * each, heads = min(each, all - head0);
        if (heads <= 0) return;
        const int n = tokens * heads;
        const T* from = (const T*)in + token0 * is[0] + head0 * is[1];
        T* to = (T*)out + token0 * os[0] + head0 * os[1];
        Rows at(group, R::kGroups, heads);
        float w[CE];
        weights<T, G>(w, weight, d0, a.dim);
        u32x4 next = {0, 0, 0, 0};
        if (group < n) next = R::load(from + at.token * is[0] + at.head * is[1], d0, a);
        if (!ready) {
            angles(cs, a, token0, tokens);
            __syncthreads();
            ready = true;
        }
        for (int r = group; r < n; r += R::kGroups) {
            float x[CE];
            R::floats(next, x);
            const Rows now = at;
            at.next();
            if (r + R::kGroups < n) next = R::load(from + at.token * is[0] + at.head * is[1], d0, a);
            float ss = 0.0f;
#pragma unroll
            for (int j = 0; j < CE; ++j) ss = fmaf(x[j], x[j], ss);
            const float rstd = rsqrtf(R::group_sum(ss) * a.inv_dim + a.eps);
#pragma unroll
            for (int j = 0; j < CE; ++j) x[j] = x[j] * rstd * w[j];
            turn(x, now.token, d0, rows[group], cs, a, 1.0f);
            R::store(to + now.token * os[0] + now.head * os[1], d0, a, x);
        }
    };
    heads_of(a.q, a.q_out, a.qs, a.qos, a.q_weight, a.heads);
    heads_of(a.k, a.k_out, a.ks, a.kos, a.k_weight, a.kv_heads);
}

template <typename T, int G, bool CHUNKS>
__global__ __launch_bounds__(kTpb, 4) void qk_norm_rope_grad_kernel(Rope a) {
    using R = Row<T, G>;
    constexpr int CE = R::CE;
    __shared__ __attribute__((aligned(16))) float2 cs[kAngles];
    __shared__ __attribute__((aligned(16))) float rows[R::kGroups][G * CE];
    const int group = threadIdx.x / G, d0 = (threadIdx.x % G) * CE;
    float sum_q[CE], sum_k[CE];
#pragma unroll
    for (int j = 0; j < CE; ++j) sum_q[j] = sum_k[j] = 0.0f;
    const int begin = blockIdx.x * a.tokens_all, end = min(begin + a.tokens_all, a.tokens);
    for (int token0 = begin; token0 < end; token0 += a.tokens_each) {
        const int tokens = min(a.tokens_each, end - token0);
        Turner<T, G, CHUNKS> turn;
        bool ready = false;
        const auto heads_of = [&](const void* in, const void* grad, void* out, const long long* is, const long long* os,
                                  const float* weight, float* sum, int heads) {
            if (!heads) return;
            const int n = tokens * heads;
            const T *from = (const T*)in + token0 * is[0], *gfrom = (const T*)grad + token0 * os[0];
            T* to = (T*)out + token0 * is[0];
            Rows at(group, R::kGroups, heads);
            float w[CE];
            weights<T, G>(w, weight, d0, a.dim);
            u32x4 next_x = {0, 0, 0, 0}, next_g = {0, 0, 0, 0};
            const auto load = [&]() {
                next_x = R::load(from + at.token * is[0] + at.head * is[1], d0, a);
                next_g = R::load(gfrom + at.token * os[0] + at.head * os[1], d0, a);
            };
            if (group < n) load();
            if (!ready) {
                __syncthreads();
                angles(cs, a, token0, tokens);
                __syncthreads();
                ready = true;
            }
            for (int r = group; r < n; r += R::kGroups) {
                float x[CE], g[CE];
                R::floats(next_x, x);
                R::floats(next_g, g);
                const Rows now = at;
                at.next();
                if (r + R::kGroups < n) load();
                turn(g, now.token, d0, rows[group], cs, a, -1.0f);
                float ss = 0.0f, dot = 0.0f;
#pragma unroll
                for (int j = 0; j < CE; ++j) {
                    ss = fmaf(x[j], x[j], ss);
                    dot = fmaf(x[j], g[j] * w[j], dot);
                }
                const float rstd = rsqrtf(R::group_sum(ss) * a.inv_dim + a.eps);
                const float mean = R::group_sum(dot) * rstd * a.inv_dim;
#pragma unroll
                for (int j = 0; j < CE; ++j) {
                    const float xn = x[j] * rstd;
                    sum[j] = fmaf(g[j], xn, sum[j]);
                    x[j] = rstd * (g[j] * w[j] - xn * mean);
                }
                R::store(to + now.token * is[0] + now.head * is[1], d0, a, x);
            }
        };
        heads_of(a.q, a.dq_out, a.dq, a.qs, a.qos, a.q_weight, sum_q, a.heads);
        heads_of(a.k, a.dk_out, a.dk, a.ks, a.kos, a.k_weight, sum_k, a.kv_heads);
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

// dw[d] = sum of the workgroups' partial sums, in 64 bits: 16 features and 64 slices of the
// rows a workgroup, a thread's rows in order, a wave's 4 slices as a tree, the waves' sums
// in order.
constexpr int kSumCols = 16, kSumSlices = 64;
__global__ __launch_bounds__(kSumCols* kSumSlices) void qk_norm_weight_grad_kernel(float* dq_weight, float* dk_weight,
    const float* partial, int groups, int dim) {
    __shared__ double part[kSumSlices / 4][kSumCols];
    const int c = threadIdx.x % kSumCols, slice = threadIdx.x / kSumCols, at = blockIdx.x * kSumCols + c;
    double sum = 0.0;
    if (at < 2 * dim) {
        const float* p = partial + (size_t)slice * 2 * dim + at;
        float v[kGradGroups / kSumSlices];
#pragma unroll
        for (int i = 0; i < kGradGroups / kSumSlices; ++i)
            v[i] = slice + i * kSumSlices < groups ? p[(size_t)i * kSumSlices * 2 * dim] : 0.0f;
#pragma unroll
        for (int i = 0; i < kGradGroups / kSumSlices; ++i) sum += v[i];
    }
    sum += __shfl_xor(sum, 16);
    sum += __shfl_xor(sum, 32);
    if (slice % 4 == 0) part[slice / 4][c] = sum;
    __syncthreads();
    if (slice || at >= 2 * dim) return;
    float* to = at < dim ? dq_weight : dk_weight;
    if (!to) return;
    sum = 0.0;
#pragma unroll
    for (int i = 0; i < kSumSlices / 4; ++i) sum += part[i][c];
    to[at < dim ? at : at - dim] = (float)sum;
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
    p.kv_heads = a->kv_heads;
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

// Whether the rows of a tensor that the call writes lie apart; false after recording an error.
bool rows_apart(const long long* stride, const NnQkNormRope* a, int heads, const char* name, const char* what) {
    const long long n[2] = {a->tokens, heads};
    NNK_REQUIRE_RET(!heads || nnk_rows_apart(2, stride, n, a->head_dim), false, what,
        "%s: rows of %s overlap (strides %lld, %lld)", what, name, stride[0], stride[1]);
    return true;
}

// Tokens of a workgroup at a time: rows for 16 passes of its groups, as far as their sines
// fit.  Few tokens: one each, and their heads shared by workgroups of one pass.
int tokens_each(const Rope& p, int groups) {
    const int by_rows = std::max(1, 16 * groups / p.all_heads), by_angles = kAngles / std::max(1, p.half);
    return std::min({by_rows, by_angles, std::max(1, p.tokens / kGradGroups)});
}

// Whether a pair's members lie whole 16-byte chunks apart.
template <typename T>
bool in_chunks(const Rope& p) {
    return !p.interleaved && p.half > 0 && p.half % (16 / (int)sizeof(T)) == 0;
}

template <typename T, int G>
void forward(Rope& p, hipStream_t s, const char* what) {
    constexpr int groups = Row<T, G>::kGroups;
    p.tokens_each = tokens_each(p, groups);
    p.head_parts = p.tokens < kGradGroups ? (p.all_heads + groups - 1) / groups : 1;
    const long long blocks = ((long long)p.tokens + p.tokens_each - 1) / p.tokens_each * p.head_parts;
    NNK_REQUIRE(blocks < (1LL << 32) / kTpb, what, "%s: too many rows", what);  // threads of a launch
    if (in_chunks<T>(p)) qk_norm_rope_kernel<T, G, true><<<(unsigned)blocks, kTpb, 0, s>>>(p);
    else qk_norm_rope_kernel<T, G, false><<<(unsigned)blocks, kTpb, 0, s>>>(p);
}
// Backward: as many workgroups as the card holds at once, of as many tokens each.
int grad_groups(Rope& p, int groups) {
    p.tokens_all = (p.tokens + kGradGroups - 1) / kGradGroups;
    p.tokens_each = std::min(p.tokens_all, tokens_each(p, groups));
    return (p.tokens + p.tokens_all - 1) / p.tokens_all;
}
template <typename T, int G>
void backward(Rope& p, hipStream_t s, const char*) {
    const unsigned blocks = (unsigned)grad_groups(p, Row<T, G>::kGroups);
    if (in_chunks<T>(p)) qk_norm_rope_grad_kernel<T, G, true><<<blocks, kTpb, 0, s>>>(p);
    else qk_norm_rope_grad_kernel<T, G, false><<<blocks, kTpb, 0, s>>>(p);
}

// Lanes of a row: a power of two with 16 bytes each.
int lanes_of(const NnQkNormRope* a) {
    const int n = (a->head_dim * (a->dtype == NN_BF16 ? 2 : 4) + 15) / 16;
    return n <= 4 ? 4 : n <= 8 ? 8 : n <= 16 ? 16 : n <= 32 ? 32 : 64;
}

#define ROPE_DISPATCH(FN, p, a, s, what)                                               \
    do {                                                                               \
        const bool half_ = (a)->dtype == NN_BF16;                                      \
        switch (lanes_of(a)) {                                                         \
        case 4: half_ ? FN<bf16, 4>(p, s, what) : FN<float, 4>(p, s, what); break;     \
        case 8: half_ ? FN<bf16, 8>(p, s, what) : FN<float, 8>(p, s, what); break;     \
        case 16: half_ ? FN<bf16, 16>(p, s, what) : FN<float, 16>(p, s, what); break;  \
        case 32: half_ ? FN<bf16, 32>(p, s, what) : FN<float, 32>(p, s, what); break;  \
        default: FN<float, 64>(p, s, what); break;                                     \
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
    if (!rows_apart(a->q_out_stride, a, a->heads, "q_out", what) || !rows_apart(a->k_out_stride, a, a->kv_heads, "k_out", what))
        return;
    p.q = q;
    p.k = k;
    p.q_out = q_out;
    p.k_out = k_out;
    if (a->heads) p.vec = p.vec && nnk::aligned16(q) && nnk::aligned16(q_out);
    if (a->kv_heads) p.vec = p.vec && nnk::aligned16(k) && nnk::aligned16(k_out);
    ROPE_DISPATCH(forward, p, a, s, what);
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
    // positions of a workgroup's tokens and of the next one's fit in 32 bits
    NNK_REQUIRE((long long)p.tokens * p.all_heads <= 1LL << 30, what, "%s: too many rows", what);
    if (rows && (!rows_apart(a->q_stride, a, a->heads, "dq", what) || !rows_apart(a->k_stride, a, a->kv_heads, "dk", what)))
        return;
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
        ROPE_DISPATCH(backward, p, a, s, what);
        nnk_after_launch(what, s);
        groups = grad_groups(p, kTpb / lanes_of(a));
    }
    if (dq_weight || dk_weight) {
        qk_norm_weight_grad_kernel<<<(unsigned)((2 * p.dim + kSumCols - 1) / kSumCols), kSumCols * kSumSlices, 0, s>>>(dq_weight, dk_weight, workspace,
            groups, p.dim);
        nnk_after_launch(what, s);
    }
}

}  // extern "C"
