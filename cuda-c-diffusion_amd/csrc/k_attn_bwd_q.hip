// k_attn_bwd_q.hip -- attention, gradient of the queries.
//
// With p_ij = 2^(x_ij - M_i), dp_ij = <dout_i, v_j> and D_i = sum_j p_ij dp_ij:
//     dx_ij = p_ij (dp_ij - D_i),   dq_i = scale * sum_j dx_ij (1 - t_ij^2) k_j
// (t the capped score's tanh).  A workgroup has 128 queries of a head, 32 a wave, with
// q and dout in registers, and goes over the blocks of keys as the forward kernel does.
//
// M comes from the forward pass's lse and D from <dout, out>, both of which that pass
// rounded (out to the tensors' type: for bf16 D is off by up to 2^-8 of <|dout|, |out|>).  The
// sums of p and of p dp are taken along, and their exact results are what the key gradients
// and the bias gradient use (stat).  The query gradient would need them before its pass: two
// of its three products a second time, or sums of p k beside those of dx k (a third more
// products, 64 more registers at 128 features).  So a query whose softmax is nearly all one
// key's gets a dq that is off by that rounding times k, against a dq near zero.  Where all
// keys of the workgroup lie in one block of 64 the sums are there before they are used, and
// the query gradient takes them too: a query that sees a single key then gets exactly zero.
//
// SPLIT 2, for calls of few workgroups: 64 queries, and of each block 32 keys a wave; the
// two waves of the same queries are added up at the end, in their order.  Fewer still: the
// keys are divided too, each part leaves fp32 sums, and a second kernel adds them in order.
//
// Measured: 8192 packed causal tokens, 16 heads of 128 (4 of keys), capped: 204 us; 4 x 1024
// tokens, 16 heads of 64 with a bias: 54 us.  128 features take one wave a SIMD, whose
// products (16 % of cycles) and vector instructions (34 %) do not overlap.
#include "attn_common.h"

namespace {
using namespace attn;

template <typename T, int DP, bool CAP, bool BIAS, bool VEC, int SPLIT>
__global__ __launch_bounds__(kTpb, sizeof(T) == 2 && DP <= 64 ? 2 : 1) void attn_bwd_q_kernel(Args a, int tiles) {
    using L = Lds<T, DP>;
    __shared__ __attribute__((aligned(16))) char k_lds[2][L::kBytes];
    __shared__ __attribute__((aligned(16))) char v_lds[2][L::kBytes];
    __shared__ __attribute__((aligned(16))) int doc_lds[2][kBlock];
    __shared__ float table[BIAS ? 2 * kMaxDistance + 1 : 1];

    __shared__ float3 parts[SPLIT > 1 ? kRows : 1];  // of the waves: maximum, sum, <p, dp>
    constexpr int kOwn = kRows / SPLIT;               // queries of the workgroup

    const int lane = threadIdx.x & 63, h = lane >> 5, wave = threadIdx.x >> 6;
    const int half = SPLIT > 1 ? wave / (kWaves / SPLIT) : 0, strip = wave - half * (kWaves / SPLIT);
    const int part = blockIdx.x % a.k_splits;
    const Turn turn = turn_of(blockIdx.x / a.k_splits, gridDim.x / a.k_splits, a.heads, tiles, a.row_order, true);
    const int tile = turn.tile, head = turn.owner % a.heads, b = turn.owner / a.heads;
    const int row0 = tile * kOwn, row = row0 + strip * 32 + (lane & 31);
    const bool in = row < a.len_q;
    const int keys = keys_of(a, b), start = start_of(a, b);
    const int pos = start + row;
    const int limit = in ? limit_of(a, b, keys, pos) : 0;
    const int doc = in && a.doc_q ? a.doc_q[(size_t)b * a.len_q + row] : -1;
    int least = in ? limit : INT32_MAX, wave_most = limit;
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) {
        least = min(least, __shfl_xor(least, m));
        wave_most = max(wave_most, __shfl_xor(wave_most, m));
    }
    const int wave_doc = __builtin_amdgcn_readfirstlane(doc);
    const bool one_doc = __all(doc == wave_doc || !in) && wave_doc >= 0;

    const int most = limit_of(a, b, keys, start + min(row0 + kOwn, a.len_q) - 1);
    const int4 mine = query_docs_of(a, b, row0 / kBlock, kOwn / kBlock);
    const int blocks = (a.len_k + kBlock - 1) / kBlock;
    const int4* key_docs = a.key_docs ? a.key_docs + (size_t)b * blocks : nullptr;
    const int each = (blocks + a.k_splits - 1) / a.k_splits;
    Blocks at(part * each, min((most + kBlock - 1) / kBlock, (part + 1) * each), key_docs, mine);

    const size_t stat_at = ((size_t)b * a.heads + head) * a.len_q + row;
    const float lse = in ? a.lse[stat_at] : -INFINITY;
    const bool sees_any = lse != -INFINITY;  // a query that sees nothing may hold anything
    float M = sees_any ? lse * kLog2e : INFINITY;
    Frag<T> qf[L::kSteps], gf[L::kSteps];
    float D = 0.0f;
    {
        const long long r = min(row, a.len_q - 1);
        const T* q = (const T*)a.q + b * a.qs[0] + r * a.qs[1] + head * a.qs[2];
        const long long o = b * a.os[0] + r * a.os[1] + head * a.os[2];
        const T *g = (const T*)a.dout + o, *out = (const T*)a.out + o;
#pragma unroll
        for (int u = 0; u < L::kSteps; ++u) {
            const int d0 = (2 * u + h) * Type<T>::CE, dim = sees_any ? a.dim : 0;
            qf[u] = load_frag<T, VEC>(q, d0, dim);
            gf[u] = load_frag<T, VEC>(g, d0, dim);
            const Frag<T> of = load_frag<T, VEC>(out, d0, dim);
#pragma unroll
            for (int j = 0; j < Type<T>::CE; ++j) D = fmaf((float)gf[u][j], (float)of[j], D);
        }
        D = sum_halves(D);
    }
    const int kv = head / a.group;
    const T* kp = (const T*)a.k + b * a.ks[0] + kv * a.ks[2];
    const T* vp = (const T*)a.v + b * a.vs[0] + kv * a.vs[2];
    const int* docs = a.doc_k ? a.doc_k + (size_t)b * a.len_k : nullptr;
    if constexpr (BIAS) load_bias(a, table, head);

    Staged<T, DP, VEC> ks, vs;
    ks.init(a.ks[1], a.dim);
    vs.init(a.vs[1], a.dim);
    int next_doc = 0;
    const auto load = [&](int block) {
        const int k0 = block * kBlock, last = keys - 1 - k0;
        if (docs) next_doc = docs[k0 + min(lane, last)];
        ks.load(kp + k0 * a.ks[1], a.ks[1], last, a.dim);
        vs.load(vp + k0 * a.vs[1], a.vs[1], last, a.dim);
    };
    const auto store = [&](int block, bool negative, int to) {
        const int k0 = block * kBlock;
        // keys that nothing sees are zeros
        const auto keep = [&](int n) {
            const int r = Staged<T, DP, VEC>::row(n);
            return k0 + r < keys && (!docs || docs[k0 + r] >= 0);
        };
        const bool all = k0 + kBlock <= keys && !negative;
        ks.store(k_lds[to], all, keep);
        vs.store(v_lds[to], all, keep);
        if (docs && wave == 0) doc_lds[to][lane] = k0 + lane < keys ? max(next_doc, -1) : -1;
    };

    f32x16 dq[DP / 32];
#pragma unroll
    for (int d = 0; d < DP / 32; ++d) dq[d] = zero16();
    float l = 0.0f, pd = 0.0f;  // sums of p and of p dp

    // a wave of SPLIT 2 has the upper or the lower 32 rows of every block
    const int rbase = L::row_base(lane) + half * 32 * L::kRowBytes, cbase = L::col_base(lane) + half * 32 * L::kRowBytes;
    constexpr int kSubs = 2 / SPLIT;
    int next = at.next();
    if (next >= 0) {
        load(next);
        store(next, at.negative, 0);
    }
    bool first = a.k_splits == 1;
    const auto step = [&](auto buf_) {
        constexpr int buf = decltype(buf_)::value;
        const int k0 = next * kBlock + half * 32, block_doc = at.doc;
        const bool block_whole = next * kBlock + kBlock <= least;
        next = at.next();
        __syncthreads();  // this block is stored; the one before it is done with
        if (next >= 0) load(next);

        const bool whole = block_whole && (!docs || (one_doc && block_doc == wave_doc));
        // nothing here for the wave's queries
        const bool none = k0 >= wave_most || (docs && one_doc && block_doc >= 0 && block_doc != wave_doc);
        struct Pair {
            Frag<T> k[L::kStage], v[L::kStage];
        };
        struct Columns {
            Frag<T> x[DP / 32];
        };
        // scores (in units of log2) and dp of keys 32 i .. 32 i + 31; slope: 1 - tanh^2
        const auto products = [&](int i, f32x16& s, f32x16& dp, f32x16& slope) {
            s = zero16();
            dp = zero16();
            Pair two[2];
            const auto read_rows = [&](Pair& y, int n) {
#pragma unroll
                for (int j = 0; j < L::kStage; ++j) {
                    y.k[j] = L::rows(k_lds[buf], i, n * L::kStage + j, rbase);
                    y.v[j] = L::rows(v_lds[buf], i, n * L::kStage + j, rbase);
                }
            };
            read_rows(two[0], 0);
            piped<L::kSteps / L::kStage>(two, read_rows, [&](const Pair& y, int n) {
#pragma unroll
                for (int j = 0; j < L::kStage; ++j) {
                    s = mma(y.k[j], qf[n * L::kStage + j], s);
                    dp = mma(y.v[j], gf[n * L::kStage + j], dp);
                }
            });
            if constexpr (CAP) cap_scores(s, slope, a);
            if constexpr (BIAS) {
                add_bias<1>(s, CAP ? 1.0f : a.c1, table, a.max_distance, k0 + 32 * i + 4 * h - pos,
                    k0 + 32 * i - (start + row0 + strip * 32 + 31));
            } else if constexpr (!CAP) {
#pragma unroll
                for (int r = 0; r < 16; ++r) s[r] *= a.c1;
            }
            if (!whole) hide(s, k0 + 32 * i, limit, docs ? doc_lds[buf] + half * 32 + 32 * i : nullptr, doc, h);
        };
        if (first && next < 0) {  // the only block
            float m = -INFINITY, sum = 0.0f, dot = 0.0f;
#pragma unroll 1
            for (int i = 0; i < kSubs; ++i) {
                f32x16 s, dp, slope;
                products(i, s, dp, slope);
                float top = m;
#pragma unroll
                for (int r = 0; r < 16; ++r) top = fmaxf(top, s[r]);
                top = max_halves(top);
                const float base = top == -INFINITY ? 0.0f : top, f = exp2_fast(m - base);
                sum *= f;
                dot *= f;
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const float p = exp2_fast(s[r] - base);
                    sum += p;
                    dot = fmaf(p, dp[r], dot);
                }
                m = top;
            }
            sum = sum_halves(sum);
            dot = sum_halves(dot);
            if constexpr (SPLIT > 1) {
                const int mine = wave * 32 + (lane & 31), other = (wave ^ (kWaves / 2)) * 32 + (lane & 31);
                if (h == 0) parts[mine] = float3{m, sum, dot};
                __syncthreads();
                const float3 x = parts[half ? other : mine], y = parts[half ? mine : other];
                m = fmaxf(x.x, y.x);
                const float base = m == -INFINITY ? 0.0f : m, f = exp2_fast(x.x - base), g = exp2_fast(y.x - base);
                sum = x.y * f + y.y * g;
                dot = x.z * f + y.z * g;
            }
            if (sees_any) {
                M = m + log2f(sum);
                D = dot / sum;
            }
        }
        first = false;
        if (!none) {
#pragma unroll
            for (int i = 0; i < kSubs; ++i) {
                f32x16 s, dp, slope;
                products(i, s, dp, slope);
                Columns columns[2];
                const auto read_columns = [&](Columns& y, int n) {
#pragma unroll
                    for (int d = 0; d < DP / 32; ++d) y.x[d] = L::cols(k_lds[buf], i, n, d, cbase);
                };
                read_columns(columns[0], 0);
                __builtin_amdgcn_sched_barrier(kMayCross);
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const float p = exp2_fast(s[r] - M);
                    l += p;
                    pd = fmaf(p, dp[r], pd);
                    float dx = p * (dp[r] - D);
                    if constexpr (CAP) dx *= slope[r];
                    s[r] = dx;
                }
                piped<L::kKeySteps>(columns, read_columns, [&](const Columns& y, int n) {
                    const Frag<T> x = operand(s, n, T{});
#pragma unroll
                    for (int d = 0; d < DP / 32; ++d) dq[d] = mma(y.x[d], x, dq[d]);
                });
            }
        }
        if (next >= 0) store(next, at.negative, buf ^ 1);
    };
    while (next >= 0) {
        step(std::integral_constant<int, 0>{});
        if (next < 0) break;
        step(std::integral_constant<int, 1>{});
    }
    l = sum_halves(l);
    pd = sum_halves(pd);
    if constexpr (SPLIT > 1) {
        // the second half's sums, through the tiles' LDS: a register's 64 lanes together
        float* to = reinterpret_cast<float*>(k_lds[0]) + (wave & 1) * (DP / 32 * 16 * 64) + lane;
        __syncthreads();
        if (half) {
#pragma unroll
            for (int d = 0; d < DP / 32; ++d)
#pragma unroll
                for (int r = 0; r < 16; ++r) to[(d * 16 + r) * 64] = dq[d][r];
            if (h == 0) parts[wave * 32 + (lane & 31)] = float3{0.0f, l, pd};
        }
        __syncthreads();
        if (half) return;
#pragma unroll
        for (int d = 0; d < DP / 32; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) dq[d][r] += to[(d * 16 + r) * 64];
        const float3 y = parts[(wave + kWaves / 2) * 32 + (lane & 31)];
        l += y.y;
        pd += y.z;
    }
    if (!in) return;
    if (a.q_sums) {
        const size_t at_row = ((size_t)(b * a.heads + head) * a.k_splits + part) * a.len_q + row;
        float* sums = a.q_sums + at_row * a.dim;
#pragma unroll
        for (int d = 0; d < DP / 32; ++d)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                store4<float, VEC>(sums, 32 * d + 8 * g + 4 * h, a.dim, dq[d][4 * g], dq[d][4 * g + 1], dq[d][4 * g + 2],
                    dq[d][4 * g + 3]);
        if (h == 0) a.stat_sums[at_row] = float2{l, pd};
        return;
    }
    T* out = (T*)a.dq + b * a.qs[0] + (long long)row * a.qs[1] + head * a.qs[2];
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g)
            store4<T, VEC>(out, 32 * d + 8 * g + 4 * h, a.dim, dq[d][4 * g] * a.scale, dq[d][4 * g + 1] * a.scale,
                dq[d][4 * g + 2] * a.scale, dq[d][4 * g + 3] * a.scale);
    if (h == 0) a.stat[stat_at] = sees_any ? float2{M + log2f(l), pd / l} : float2{INFINITY, 0.0f};
}

// dq and the statistics from the parts' sums, in their order; 4 features a thread.
template <typename T, bool VEC>
__global__ __launch_bounds__(kTpb) void attn_q_sum_kernel(Args a, int quads, long long total) {
    const long long n = (long long)blockIdx.x * kTpb + threadIdx.x;
    if (n >= total) return;
    const int d = (int)(n % quads) * 4, row = (int)(n / quads % a.len_q);
    const long long owner = n / quads / a.len_q;
    const int head = (int)(owner % a.heads), b = (int)(owner / a.heads);
    const size_t first = (size_t)owner * a.k_splits * a.len_q + row;
    float v[4] = {0.0f, 0.0f, 0.0f, 0.0f}, l = 0.0f, pd = 0.0f;
    for (int i = 0; i < a.k_splits; ++i) {
        const size_t at = first + (size_t)i * a.len_q;
        const float* p = a.q_sums + at * a.dim + d;
        if constexpr (VEC) {
            const float4 x = nnk::ld4(p);
            v[0] += x.x, v[1] += x.y, v[2] += x.z, v[3] += x.w;
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (d + j < a.dim) v[j] += p[j];
        }
        if (d == 0) {
            const float2 x = a.stat_sums[at];
            l += x.x;
            pd += x.y;
        }
    }
    store4<T, VEC>((T*)a.dq + b * a.qs[0] + row * a.qs[1] + head * a.qs[2], d, a.dim, v[0] * a.scale, v[1] * a.scale,
        v[2] * a.scale, v[3] * a.scale);
    if (d == 0) {
        const size_t at = (size_t)owner * a.len_q + row;
        const float lse = a.lse[at];
        a.stat[at] = lse != -INFINITY ? float2{lse * kLog2e + log2f(l), pd / l} : float2{INFINITY, 0.0f};
    }
}

template <typename T, int DP, bool CAP, bool BIAS, bool VEC>
bool launch(const Args& a, hipStream_t s, const char* what) {
    const int tiles = (a.len_q + a.q_rows - 1) / a.q_rows;
    const unsigned groups = (unsigned)((long long)tiles * a.heads * a.batch * a.k_splits);
    if (a.q_rows < kRows) attn_bwd_q_kernel<T, DP, CAP, BIAS, VEC, 2><<<groups, kTpb, 0, s>>>(a, tiles);
    else attn_bwd_q_kernel<T, DP, CAP, BIAS, VEC, 1><<<groups, kTpb, 0, s>>>(a, tiles);
    nnk_after_launch(what, s);
    if (a.q_sums) {
        const int quads = (a.dim + 3) / 4;
        const long long total = (long long)a.batch * a.heads * a.len_q * quads;
        attn_q_sum_kernel<T, VEC><<<(unsigned)((total + kTpb - 1) / kTpb), kTpb, 0, s>>>(a, quads, total);
        nnk_after_launch(what, s);
    }
    return true;
}

}  // namespace

bool nnk_attention_backward_q(const Args& a, bool half, hipStream_t s, const char* what) {
    return NNK_ATTN_DISPATCH(a, half, launch, a, s, what);
}
