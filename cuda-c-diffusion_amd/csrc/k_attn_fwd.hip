// k_attn_fwd.hip -- attention, many queries a head.
//
// One pass over the keys with a reference m and the running sum l of each query's softmax:
// per block of 64 keys  S = K Q^T,  p = 2^(x - m),  O = O 2^(m_old - m) + V^T p.
// A workgroup of 4 waves has 128 queries of a head, 32 a wave, whose operand stays in
// registers; keys and values of a block are in LDS for all four, two blocks at a time, the
// next one's loads under way meanwhile.  Blocks that no query of the workgroup sees are
// left out.
//
// SPLIT 2, for calls of few workgroups: 64 queries, and of each block 32 keys a wave; the two
// waves of the same queries are joined at the end.
//
// What bounds it is the softmax's arithmetic, a vector instruction of 4 cycles for 64
// scores against 32 cycles of matrix products (128 features), so each score term has the
// form with the fewest:
//   plain:  m is kept in units of s, p = 2^(c s - c m): one multiply-add, one power;
//   cap:    scores within +-c2 (units of log2) need no running maximum.  m is that of the
//           first block that a query sees, or c2 - 80 if that is more: then p <= 2^80 and,
//           for c2 up to 80, l >= 2^-80.  Sums that all the same left fp32's range (values past
//           2^47), or came near its lower end (values below 2^-20 where all scores are low),
//           show at the end, and the workgroup goes over its keys again by the next form.
//           For scores below 3/8 of the cap, tanh, its factors and the reference are one
//           polynomial, of 4 terms instead of 6 below 0.14 of it;
//   else:   running maximum of x.
//
// Measured: 16384 tokens, 16 heads of 128 (4 of keys), a prefix, scores of deviation 1 under a
// cap of 50: 1454-1481 us, 790-804 TFLOP/s of visible scores; vector instructions take 56 %,
// products 36 % of the SIMDs' cycles.  Of deviation 12, where most blocks go without the
// series: 2328 us.  8192 packed tokens, 16 heads of 72, 13 documents: 84 us, 335 TFLOP/s, two
// launches for the documents among it.
#include "attn_common.h"

namespace {
using namespace attn;

// CAP: 0 none, 1 any, 2 at most kFixedCap and no bias
constexpr float kFixedCap = 80.0f;
// below this much of a sum of probabilities, sums of values are looked at: past 2^-100 they keep
// their digits, as their terms' roundings are 2^-149
constexpr float kLeastSum = 0x1p-16f, kLeastValue = 0x1p-100f;

template <typename T, int DP, int CAP, bool BIAS, bool VEC, int SPLIT>
__global__ __launch_bounds__(kTpb, sizeof(T) == 2 && VEC ? 2 : 1) void attn_fwd_kernel(Args a, int tiles) {
    using L = Lds<T, DP>;
    // fp32, one wave a SIMD: reads of LDS ahead of their products.  bf16 has two waves, which
    // hide them for each other, and no registers for it (128 features: 1.6 ms became 2.4)
    constexpr bool kPiped = sizeof(T) == 4;
    constexpr int kWide = 2 / SPLIT * L::kSteps % L::kWide ? L::kWide / 2 : L::kWide;  // fragments of a stage
    static_assert(2 / SPLIT * L::kSteps % kWide == 0);
    __shared__ __attribute__((aligned(16))) char k_lds[2][L::kBytes];
    __shared__ __attribute__((aligned(16))) char v_lds[2][L::kBytes];
    __shared__ __attribute__((aligned(16))) int doc_lds[2][kBlock];
    __shared__ float table[BIAS ? 2 * kMaxDistance + 1 : 1];

    __shared__ float2 parts[SPLIT > 1 ? kRows : 1];  // reference and sum of the second waves
    constexpr int kOwn = kRows / SPLIT;               // queries of the workgroup
    constexpr int kSubs = 2 / SPLIT;                  // 32 keys of a block that are a wave's

    const int lane = threadIdx.x & 63, h = lane >> 5, wave = threadIdx.x >> 6;
    const int half = SPLIT > 1 ? wave / (kWaves / SPLIT) : 0, strip = wave - half * (kWaves / SPLIT);
    const Turn turn = turn_of(blockIdx.x, gridDim.x, a.heads, tiles, a.row_order, true);  // those that see most keys first
    const int tile = turn.tile, head = turn.owner % a.heads, b = turn.owner / a.heads;
    const int row0 = tile * kOwn, row = row0 + strip * 32 + (lane & 31);
    const bool in = row < a.len_q;
    const int keys = keys_of(a, b), start = start_of(a, b);
    const int pos = start + row;
    const int limit = in ? limit_of(a, b, keys, pos) : 0;
    const int doc = in && a.doc_q ? a.doc_q[(size_t)b * a.len_q + row] : -1;
    // a wave's least limit and whether one document has all its queries, for blocks without masked entries
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

    Frag<T> qf[L::kSteps];
    {
        const T* q = (const T*)a.q + b * a.qs[0] + (long long)min(row, a.len_q - 1) * a.qs[1] + head * a.qs[2];
#pragma unroll
        for (int u = 0; u < L::kSteps; ++u) qf[u] = load_frag<T, VEC>(q, (2 * u + h) * Type<T>::CE, a.dim);
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

    f32x16 o[DP / 32];
    float m, l;  // m in units of the score: of s if there is neither cap nor bias
    // a wave of SPLIT 2 has the upper or the lower 32 rows of every block
    const int rbase = L::row_base(lane) + half * 32 * L::kRowBytes, cbase = L::col_base(lane) + half * 32 * L::kRowBytes;

    // over all blocks, by the form of CAP
    const auto sweep = [&](auto cap_) {
        constexpr int kCap = decltype(cap_)::value;
        Blocks at(0, (most + kBlock - 1) / kBlock, key_docs, mine);
#pragma unroll
        for (int d = 0; d < DP / 32; ++d) o[d] = zero16();
        m = -INFINITY;
        l = 0.0f;
        int next = at.next();
        if (next >= 0) {
            load(next);
            store(next, at.negative, 0);
        }
        for (int buf = 0; next >= 0; buf ^= 1) {
            const int block = next, k0 = next * kBlock + half * 32, block_doc = at.doc;
            next = at.next();
            __syncthreads();  // this block is stored; the one before it is done with
            if (next >= 0) load(next);
            // nothing here for the wave's queries
            const bool none = k0 >= wave_most || (docs && one_doc && block_doc >= 0 && block_doc != wave_doc);
            if (!none) {

                f32x16 s[kSubs];
#pragma unroll
                for (int i = 0; i < kSubs; ++i) s[i] = zero16();
                struct Keys {
                    Frag<T> x[kWide];
                };
                Keys rows[2];
                const auto read_rows = [&](Keys& y, int n) {
#pragma unroll
                    for (int j = 0; j < kWide; ++j) {
                        const int u = n * kWide + j;
                        y.x[j] = L::rows(k_lds[buf], u / L::kSteps, u % L::kSteps, rbase);
                    }
                };
                const auto score = [&](const Keys& y, int n) {
#pragma unroll
                    for (int j = 0; j < kWide; ++j) {
                        const int u = n * kWide + j;
                        s[u / L::kSteps] = mma(y.x[j], qf[u % L::kSteps], s[u / L::kSteps]);
                    }
                };
                if constexpr (kPiped) {
                    read_rows(rows[0], 0);
                    piped<kSubs * L::kSteps / kWide>(rows, read_rows, score);
                } else {
#pragma unroll
                    for (int n = 0; n < kSubs * L::kSteps / kWide; ++n) {
                        read_rows(rows[0], n);
                        score(rows[0], n);
                    }
                }
                struct Values {
                    Frag<T> x[DP / 32];
                };
                Values columns[2];
                const auto read_columns = [&](Values& y, int n) {
#pragma unroll
                    for (int d = 0; d < DP / 32; ++d)
                        y.x[d] = L::cols(v_lds[buf], n / L::kKeySteps, n % L::kKeySteps, d, cbase);
                };
                if constexpr (kPiped) {
                    read_columns(columns[0], 0);
                    __builtin_amdgcn_sched_barrier(kMayCross);
                }
                const bool whole = block * kBlock + kBlock <= least && (!docs || (one_doc && block_doc == wave_doc));
                const auto hide_both = [&]() {
                    if (whole) return;
#pragma unroll
                    for (int i = 0; i < kSubs; ++i)
                        hide(s[i], k0 + 32 * i, limit, docs ? doc_lds[buf] + half * 32 + 32 * i : nullptr, doc, h);
                };
                // the largest score so far, and sums and outputs in its terms
                const auto raise = [&](float unit) {
                    float top = m;
#pragma unroll
                    for (int i = 0; i < kSubs; ++i)
#pragma unroll
                        for (int r = 0; r < 16; ++r) top = fmaxf(top, s[i][r]);
                    top = max_halves(top);
                    const float base = top == -INFINITY ? 0.0f : top * unit;
                    if (__any(top > m)) {
                        const float f = exp2_fast(m * unit - base);
                        l *= f;
#pragma unroll
                        for (int d = 0; d < DP / 32; ++d)
#pragma unroll
                            for (int r = 0; r < 16; ++r) o[d][r] *= f;
                        m = top;
                    }
                    return base;
                };
                if constexpr (kCap == 2) {
                    float top = 0.0f;
#pragma unroll
                    for (int i = 0; i < kSubs; ++i)
#pragma unroll
                        for (int r = 0; r < 16; ++r) top = fmaxf(top, fabsf(s[i][r]));
                    const auto by_series = [&](auto terms) {
#pragma unroll
                        for (int i = 0; i < kSubs; ++i)
#pragma unroll
                            for (int r = 0; r < 16; ++r) {
                                const float w = s[i][r] * s[i][r];
                                float c = a.series[decltype(terms)::value - 1];
#pragma unroll
                                for (int t = decltype(terms)::value - 2; t >= 0; --t) c = fmaf(w, c, a.series[t]);
                                s[i][r] = exp2_fast(fmaf(s[i][r], c, -m));
                            }
                    };
                    const bool plain = whole && __all(m != -INFINITY);
                    if (plain && __all(top < a.tiny)) {
                        by_series(std::integral_constant<int, 4>{});
                    } else if (plain && __all(top < a.small)) {
                        by_series(std::integral_constant<int, 6>{});
                    } else {
#pragma unroll
                        for (int i = 0; i < kSubs; ++i) {
                            cap_scores(s[i], a.c1, a.c2);
                        }
                        hide_both();
                        float first = -INFINITY;
#pragma unroll
                        for (int i = 0; i < kSubs; ++i)
#pragma unroll
                            for (int r = 0; r < 16; ++r) first = fmaxf(first, s[i][r]);
                        first = max_halves(first);
                        if (m == -INFINITY && first > -INFINITY) m = fmaxf(first, a.c2 - kFixedCap);
                        const float base = m == -INFINITY ? 0.0f : m;
#pragma unroll
                        for (int i = 0; i < kSubs; ++i)
#pragma unroll
                            for (int r = 0; r < 16; ++r) s[i][r] = exp2_fast(s[i][r] - base);
                    }
                } else if constexpr (kCap == 0 && !BIAS) {
                    hide_both();
                    const float base = raise(a.c1);
#pragma unroll
                    for (int i = 0; i < kSubs; ++i)
#pragma unroll
                        for (int r = 0; r < 16; ++r) s[i][r] = exp2_fast(fmaf(s[i][r], a.c1, -base));
                } else {
#pragma unroll
                    for (int i = 0; i < kSubs; ++i) {
                        if constexpr (kCap) cap_scores(s[i], a.c1, a.c2);
                        if constexpr (BIAS) add_bias<1>(s[i], kCap ? 1.0f : a.c1, table, a.max_distance, k0 + 32 * i + 4 * h - pos,
                            k0 + 32 * i - (start + row0 + strip * 32 + 31));
                    }
                    hide_both();
                    const float base = raise(1.0f);
#pragma unroll
                    for (int i = 0; i < kSubs; ++i)
#pragma unroll
                        for (int r = 0; r < 16; ++r) s[i][r] = exp2_fast(s[i][r] - base);
                }
#pragma unroll
                for (int i = 0; i < kSubs; ++i)
#pragma unroll
                    for (int r = 0; r < 16; ++r) l += s[i][r];
                const auto mix = [&](const Values& y, int n) {
                    const Frag<T> p = operand(s[n / L::kKeySteps], n % L::kKeySteps, T{});
#pragma unroll
                    for (int d = 0; d < DP / 32; ++d) o[d] = mma(y.x[d], p, o[d]);
                };
                if constexpr (kPiped) {
                    piped<kSubs * L::kKeySteps>(columns, read_columns, mix);
                } else {
#pragma unroll
                    for (int n = 0; n < kSubs * L::kKeySteps; ++n) {
                        read_columns(columns[0], n);
                        mix(columns[0], n);
                    }
                }
            }
            if (next >= 0) store(next, at.negative, buf ^ 1);
        }
        l = sum_halves(l);
    };
    sweep(std::integral_constant<int, CAP>{});
    if constexpr (CAP == 2) {
        float zero = l * 0.0f, least = INFINITY;  // NaN where a sum has left the type; the least of |o|
#pragma unroll
        for (int d = 0; d < DP / 32; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) zero = fmaf(o[d][r], 0.0f, zero);
        if (__any(l < kLeastSum)) {
#pragma unroll
            for (int d = 0; d < DP / 32; ++d)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (32 * d + row_of(r, h) < a.dim) least = fminf(least, fabsf(o[d][r]));
        }
        const bool held = zero == 0.0f && (l >= kLeastSum || least >= kLeastValue);
        if (__syncthreads_or(m != -INFINITY && !held)) sweep(std::integral_constant<int, 1>{});
    }

    if constexpr (SPLIT > 1) {
        // the second half's part, through the tiles' LDS: a register's 64 lanes together
        float* to = reinterpret_cast<float*>(k_lds[0]) + strip * (DP / 32 * 16 * 64) + lane;
        __syncthreads();
        if (half) {
#pragma unroll
            for (int d = 0; d < DP / 32; ++d)
#pragma unroll
                for (int r = 0; r < 16; ++r) to[(d * 16 + r) * 64] = o[d][r];
            if (h == 0) parts[strip * 32 + lane] = float2{m, l};
        }
        __syncthreads();
        if (half) return;
        const float2 y = parts[strip * 32 + (lane & 31)];
        const float unit = CAP || BIAS ? 1.0f : a.c1, top = fmaxf(m, y.x), base = top == -INFINITY ? 0.0f : top;
        const float f = exp2_fast((m - base) * unit), g = exp2_fast((y.x - base) * unit);
#pragma unroll
        for (int d = 0; d < DP / 32; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[d][r] = o[d][r] * f + to[(d * 16 + r) * 64] * g;
        l = l * f + y.y * g;
        m = top;
    }
    if (!in) return;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    T* out = (T*)a.out + b * a.os[0] + (long long)row * a.os[1] + head * a.os[2];
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g)
            store4<T, VEC>(out, 32 * d + 8 * g + 4 * h, a.dim, o[d][4 * g] * inv, o[d][4 * g + 1] * inv,
                o[d][4 * g + 2] * inv, o[d][4 * g + 3] * inv);
    if (h == 0)
        a.lse[((size_t)b * a.heads + head) * a.len_q + row] =
            l == 0.0f ? -INFINITY : (m * (CAP || BIAS ? 1.0f : a.c1) + log2f(l)) * kLn2;
}

template <typename T, int DP, int CAP, bool BIAS, bool VEC>
bool launch_split(const Args& a, hipStream_t s, const char* what) {
    const int own = a.q_rows, tiles = (a.len_q + own - 1) / own;
    const bool split = own < kRows;
    const unsigned blocks = (unsigned)((long long)tiles * a.heads * a.batch);
    if (split) attn_fwd_kernel<T, DP, CAP, BIAS, VEC, 2><<<blocks, kTpb, 0, s>>>(a, tiles);
    else attn_fwd_kernel<T, DP, CAP, BIAS, VEC, 1><<<blocks, kTpb, 0, s>>>(a, tiles);
    nnk_after_launch(what, s);
    return true;
}
template <typename T, int DP, bool CAP, bool BIAS, bool VEC>
bool launch(const Args& a, hipStream_t s, const char* what) {
    if constexpr (CAP && !BIAS) {
        if (a.c2 <= kFixedCap) return launch_split<T, DP, 2, BIAS, VEC>(a, s, what);
    }
    return launch_split<T, DP, CAP, BIAS, VEC>(a, s, what);
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

const int* nnk_attention_order(const Args& a, bool keys, int own, float* order, hipStream_t s, const char* what) {
    const int len = keys ? a.len_k : a.len_q, tiles = (len + own - 1) / own;
    const int blocks = ((keys ? a.len_q : a.len_k) + kBlock - 1) / kBlock;
    if (a.batch > kMostHeads || tiles < 2 || tiles > kOrderTiles || blocks > kOrderBlocks || tiles * blocks > 64 * kOrderTpb) return nullptr;
    int* to = reinterpret_cast<int*>(order);
    tile_order_kernel<<<(unsigned)a.batch, kOrderTpb, 0, s>>>(to, a, keys, own, tiles);
    nnk_after_launch(what, s);
    return to;
}
