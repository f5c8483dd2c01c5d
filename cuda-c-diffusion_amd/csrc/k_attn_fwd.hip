// k_attn_fwd.hip -- attention, many queries a head.
//
// One pass over the keys with the running maximum m and sum l of each query's softmax:
// per block of 64 keys  S = K Q^T,  p = 2^(x - m),  O = O 2^(m_old - m) + V^T p.
// A workgroup of 4 waves has 128 queries of a head, 32 a wave, whose operand stays in
// registers; keys and values of a block are in LDS for all four, the next block's
// loads under way meanwhile.  Blocks that no query of the workgroup sees are left out.
#include "attn_common.h"

namespace {
using namespace attn;

template <typename T, int DP, bool CAP, bool BIAS>
__global__ __launch_bounds__(kTpb, sizeof(T) == 2 ? 2 : 1) void attn_fwd_kernel(Args a, int tiles) {
    using L = Lds<T, DP>;
    __shared__ __attribute__((aligned(16))) char k_lds[L::kBytes];
    __shared__ __attribute__((aligned(16))) char v_lds[L::kBytes];
    __shared__ int doc_lds[kBlock];
    __shared__ float table[BIAS ? 2 * kMaxDistance + 1 : 1];

    const int lane = threadIdx.x & 63, h = lane >> 5, wave = threadIdx.x >> 6;
    const int w = nnk::xcd_swizzle(blockIdx.x, gridDim.x);
    const int tile = tiles - 1 - w % tiles;  // those that see most keys first
    const int head = w / tiles % a.heads, b = w / tiles / a.heads;
    const int row0 = tile * kRows, row = row0 + wave * 32 + (lane & 31);
    const bool in = row < a.len_q;
    const int keys = keys_of(a, b), start = start_of(a, b);
    const int pos = start + row;
    const int limit = in ? limit_of(a, b, keys, pos) : 0;
    const int doc = in && a.doc_q ? a.doc_q[(size_t)b * a.len_q + row] : -1;
    // a wave's least limit and whether one document has all its queries, for blocks without masked entries
    int least = in ? limit : INT32_MAX;
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) least = min(least, __shfl_xor(least, m));
    const int wave_doc = __builtin_amdgcn_readfirstlane(doc);
    const bool one_doc = __all(doc == wave_doc || !in) && wave_doc >= 0;

    const int most = limit_of(a, b, keys, start + min(row0 + kRows, a.len_q) - 1);
    const int4 mine = query_docs_of(a, b, row0 / kBlock, kRows / kBlock);
    const int blocks = (a.len_k + kBlock - 1) / kBlock;
    const int4* key_docs = a.key_docs ? a.key_docs + (size_t)b * blocks : nullptr;
    Blocks at(0, (most + kBlock - 1) / kBlock, key_docs, mine);

    Frag<T> qf[L::kSteps];
    {
        const T* q = (const T*)a.q + b * a.qs[0] + (long long)min(row, a.len_q - 1) * a.qs[1] + head * a.qs[2];
#pragma unroll
        for (int u = 0; u < L::kSteps; ++u) qf[u] = load_frag<T>(q, (2 * u + h) * Type<T>::CE, a.dim, a.vec);
    }
    const int kv = head / a.group;
    const T* kp = (const T*)a.k + b * a.ks[0] + kv * a.ks[2];
    const T* vp = (const T*)a.v + b * a.vs[0] + kv * a.vs[2];
    const int* docs = a.doc_k ? a.doc_k + (size_t)b * a.len_k : nullptr;
    if constexpr (BIAS) load_bias(a, table, head);

    Staged<T, DP> ks, vs;
    int row_doc[Staged<T, DP>::N], next_doc = 0;
    const auto load = [&](int block) {
        const int k0 = block * kBlock, last = keys - 1 - k0;
        if (docs) {
#pragma unroll
            for (int n = 0; n < Staged<T, DP>::N; ++n) row_doc[n] = docs[k0 + min(Staged<T, DP>::row(n), last)];
            next_doc = docs[k0 + min(lane, last)];
        }
        ks.load(kp + k0 * a.ks[1], a.ks[1], last, a.dim, a.vec);
        vs.load(vp + k0 * a.vs[1], a.vs[1], last, a.dim, a.vec);
    };

    f32x16 o[DP / 32];
#pragma unroll
    for (int d = 0; d < DP / 32; ++d) o[d] = zero16();
    float m = -INFINITY, l = 0.0f;

    int block = at.next();
    if (block >= 0) load(block);
    while (block >= 0) {
        __syncthreads();
        const int k0 = block * kBlock, block_doc = at.doc;
        // keys that nothing sees are zeros
        const auto keep = [&](int n) {
            return k0 + Staged<T, DP>::row(n) < keys && (!docs || row_doc[n] >= 0);
        };
        ks.store(k_lds, a.dim, keep);
        vs.store(v_lds, a.dim, keep);
        if (docs && wave == 0) doc_lds[lane] = k0 + lane < keys ? next_doc : -1;
        __syncthreads();
        block = at.next();
        if (block >= 0) load(block);

        f32x16 s[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            s[i] = zero16();
#pragma unroll
            for (int u = 0; u < L::kSteps; ++u) s[i] = mma(L::rows(k_lds, 32 * i + (lane & 31), u, h), qf[u], s[i]);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if constexpr (CAP) cap_scores<false>(s[i], s[i], a.c1);
            const float c = CAP ? a.c2 : a.c1;
#pragma unroll
            for (int r = 0; r < 16; ++r) s[i][r] *= c;
            if constexpr (BIAS) {
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int rel = k0 + 32 * i + row_of(r, h) - pos;
                    s[i][r] += table[min(max(rel, -a.max_distance), a.max_distance) + a.max_distance];
                }
            }
        }
        const bool whole = k0 + kBlock <= least && (!docs || (one_doc && block_doc == wave_doc));
        if (!whole) {
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int j = 32 * i + row_of(r, h);
                    const bool sees = k0 + j < limit && (!docs || (doc_lds[j] == doc && doc >= 0));
                    s[i][r] = sees ? s[i][r] : -INFINITY;
                }
        }
        float top = m;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) top = fmaxf(top, s[i][r]);
        top = max_halves(top);
        const float base = top == -INFINITY ? 0.0f : top;
        if (__any(top > m)) {
            const float f = exp2_fast(m - base);
            l *= f;
#pragma unroll
            for (int d = 0; d < DP / 32; ++d)
#pragma unroll
                for (int r = 0; r < 16; ++r) o[d][r] *= f;
            m = top;
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                s[i][r] = exp2_fast(s[i][r] - base);
                l += s[i][r];
            }
#pragma unroll
            for (int f = 0; f < L::kKeySteps; ++f) {
                const Frag<T> p = operand(s[i], f, T{});
#pragma unroll
                for (int d = 0; d < DP / 32; ++d) o[d] = mma(L::cols(v_lds, 32 * i, f, 32 * d, lane), p, o[d]);
            }
        }
    }

    if (!in) return;
    l = sum_halves(l);
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    T* out = (T*)a.out + b * a.os[0] + (long long)row * a.os[1] + head * a.os[2];
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g)
            store4<T>(out, 32 * d + 8 * g + 4 * h, a.dim, a.vec, o[d][4 * g] * inv, o[d][4 * g + 1] * inv,
                o[d][4 * g + 2] * inv, o[d][4 * g + 3] * inv);
    if (h == 0)
        a.lse[((size_t)b * a.heads + head) * a.len_q + row] = l == 0.0f ? -INFINITY : (m + log2f(l)) * kLn2;
}

template <typename T, int DP, bool CAP, bool BIAS>
bool launch(const Args& a, hipStream_t s, const char* what) {
    const int tiles = (a.len_q + kRows - 1) / kRows;
    attn_fwd_kernel<T, DP, CAP, BIAS><<<(unsigned)((long long)tiles * a.heads * a.batch), kTpb, 0, s>>>(a, tiles);
    nnk_after_launch(what, s);
    return true;
}

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

}  // namespace

bool nnk_attention_forward(const Args& a, bool half, hipStream_t s, const char* what) {
    return NNK_ATTN_DISPATCH(a, half, launch, a, s, what);
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
