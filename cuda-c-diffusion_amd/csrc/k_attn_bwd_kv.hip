// k_attn_bwd_kv.hip -- attention, gradients of keys, values and the bias.
//
// With p_ij = 2^(x_ij - M_i) and dx_ij = p_ij (dp_ij - D_i) from the statistics that the
// query gradient left:
//     dv_j = sum_i p_ij dout_i,   dk_j = scale * sum_i dx_ij (1 - t_ij^2) q_i
// over the queries of all heads that share the key.  A workgroup has 128 keys of a key
// head, 32 a wave, with k and v in registers, and goes over the blocks of 64 queries of
// its heads; q and dout of a block are in LDS.  Scores are formed as queries x keys, so
// that their registers are the operand of both gradients.  No atomics: a key's sums are
// one wave's, in a fixed order.  Where key heads are shared and key tiles are few, a
// workgroup takes one head's queries and leaves fp32 sums, which a second kernel adds up
// in the heads' order: documents and causal masks give tiles very uneven work, which only
// more workgroups even out.
//
// SPLIT 2, for calls of few workgroups: 64 keys, and of each block 32 queries a wave; the
// two waves of the same keys are added up at the end, in their order.  Fewer still: the
// queries are divided too, and their parts added up as the heads' are.
//
// Bias: sums of dx by distance j - P.  A 32 x 32 tile has its distances on diagonals;
// row m's values go m lanes along, after which a lane holds two distances (one for what
// went past the end), and the tile is 32 shuffles and adds and one addition to the
// wave's table in LDS.  Tiles wholly past max_distance are added up whole.
//
// Measured, as the query gradients: 245 us and 92 us (the bias's distances are a third of
// the latter); two waves a SIMD up to 64 features (177 us without), one above.
#include "attn_common.h"

namespace {
using namespace attn;

constexpr int kSlack = 64;  // distances of a tile that reaches past max_distance

template <typename T, int DP, bool CAP, bool BIAS, bool VEC, int SPLIT>
__global__ __launch_bounds__(kTpb, sizeof(T) == 2 && DP <= 64 ? 2 : 1) void attn_bwd_kv_kernel(Args a, int tiles) {
    using L = Lds<T, DP>;
    // two blocks in LDS; one where they and the distances would not fit (fp32, over 64 features)
    constexpr int kBufs = L::kRowBytes > 256 ? 1 : 2;
    __shared__ __attribute__((aligned(16))) char q_lds[kBufs][L::kBytes];
    __shared__ __attribute__((aligned(16))) char g_lds[kBufs][L::kBytes];
    __shared__ __attribute__((aligned(16))) float M_lds[kBufs][kBlock];
    __shared__ __attribute__((aligned(16))) float D_lds[kBufs][kBlock];
    __shared__ __attribute__((aligned(16))) int limit_lds[kBufs][kBlock];
    __shared__ __attribute__((aligned(16))) int doc_lds[kBufs][kBlock];
    __shared__ float table[BIAS ? 2 * kMaxDistance + 1 : 1];
    extern __shared__ float dist[];  // BIAS: a table of 2 (max_distance + kSlack) + 1 a wave

    constexpr int kOwn = kRows / SPLIT;  // keys of the workgroup

    const int lane = threadIdx.x & 63, h = lane >> 5, wave = threadIdx.x >> 6;
    const int half = SPLIT > 1 ? wave / (kWaves / SPLIT) : 0, strip = wave - half * (kWaves / SPLIT);
    const int parts = a.heads / a.heads_each * a.q_splits;
    const Turn turn = turn_of(blockIdx.x, gridDim.x, parts, tiles, a.key_order, false);
    const int tile = turn.tile, part = turn.owner % parts, b = turn.owner / parts;
    const int share = part % a.q_splits, head0 = part / a.q_splits * a.heads_each, kv = head0 / a.group;
    const int k0 = tile * kOwn, first_key = k0 + strip * 32, key = first_key + (lane & 31);
    const int keys = keys_of(a, b), start = start_of(a, b);
    const int* docs = a.doc_k ? a.doc_k + (size_t)b * a.len_k : nullptr;
    const bool in = key < a.len_k;
    const int doc = docs && in ? docs[key] : -1;
    const bool live = key < keys && (!docs || doc >= 0);
    const int wave_doc = __builtin_amdgcn_readfirstlane(doc);
    const bool whole_keys = __all(live && (!docs || doc == wave_doc));
    const int last_key = first_key + 31;

    const int q_blocks = (a.len_q + kBlock - 1) / kBlock;
    const int4 mine = key_docs_of(a, b, k0 / kBlock, kOwn / kBlock);
    const int4* query_docs = a.query_docs ? a.query_docs + (size_t)b * q_blocks : nullptr;
    // the first block of queries that can see the tile: their limits rise with their positions
    int first_block = keys > k0 ? 0 : q_blocks;
    if (a.mask == NN_MASK_CAUSAL || (a.mask == NN_MASK_PREFIX && a.prefix[b] <= k0))
        first_block = max(first_block, (k0 - start) >> 6);

    Frag<T> kf[L::kSteps], vf[L::kSteps];
    {
        const long long r = min(key, a.len_k - 1);
        const T* k = (const T*)a.k + b * a.ks[0] + r * a.ks[1] + kv * a.ks[2];
        const T* v = (const T*)a.v + b * a.vs[0] + r * a.vs[1] + kv * a.vs[2];
#pragma unroll
        for (int u = 0; u < L::kSteps; ++u) {
            const int d0 = (2 * u + h) * Type<T>::CE, dim = live ? a.dim : 0;
            kf[u] = load_frag<T, VEC>(k, d0, dim);
            vf[u] = load_frag<T, VEC>(v, d0, dim);
        }
    }
    f32x16 dk[DP / 32], dv[DP / 32];
#pragma unroll
    for (int d = 0; d < DP / 32; ++d) {
        dk[d] = zero16();
        dv[d] = zero16();
    }
    // a wave of SPLIT 2 has the upper or the lower 32 rows of every block
    const int rbase = L::row_base(lane) + half * 32 * L::kRowBytes, cbase = L::col_base(lane) + half * 32 * L::kRowBytes;
    const int span = 2 * (a.max_distance + kSlack) + 1;
    float* my_dist = dist + wave * span;

    for (int head = head0; head < head0 + a.heads_each; ++head) {
        float far_lo = 0.0f, far_hi = 0.0f;
        __syncthreads();  // the head before is done with
        if constexpr (BIAS) {
            load_bias(a, table, head);
            for (int i = threadIdx.x; i < kWaves * span; i += kTpb) dist[i] = 0.0f;
        }
        const T* qp = (const T*)a.q + b * a.qs[0] + head * a.qs[2];
        const T* gp = (const T*)a.dout + b * a.os[0] + head * a.os[2];
        const float2* stats = a.stat + ((size_t)b * a.heads + head) * a.len_q;

        Staged<T, DP, VEC> qs, gs;
        qs.init(a.qs[1], a.dim);
        gs.init(a.os[1], a.dim);
        float2 st = {INFINITY, 0.0f};
        int lim = 0, qdoc = -2;
        const auto load = [&](int block) {
            const int q0 = block * kBlock, last = a.len_q - 1 - q0;
            st = stats[q0 + min(lane, last)];
            if (wave == 0) {
                const int i = q0 + min(lane, last);
                if (a.doc_q) qdoc = a.doc_q[(size_t)b * a.len_q + i];
                lim = limit_of(a, b, keys, start + i);
            }
            qs.load(qp + q0 * a.qs[1], a.qs[1], last, a.dim);
            gs.load(gp + q0 * a.os[1], a.os[1], last, a.dim);
        };

        const auto store = [&](int block, int to) {
            const int q0 = block * kBlock;
            // queries that see nothing are zeros
            const auto keep = [&](int n) {
                const int i = q0 + Staged<T, DP, VEC>::row(n);
                return i < a.len_q && stats[i].x != INFINITY;
            };
            const bool all = __all(q0 + lane < a.len_q && st.x != INFINITY);
            qs.store(q_lds[to], all, keep);
            gs.store(g_lds[to], all, keep);
            if (wave == 0) {
                const bool there = q0 + lane < a.len_q;
                M_lds[to][lane] = there ? st.x : INFINITY;
                D_lds[to][lane] = st.y;
                limit_lds[to][lane] = there ? lim : 0;
                doc_lds[to][lane] = there ? qdoc : -2;
            }
        };

        const int each = (q_blocks + a.q_splits - 1) / a.q_splits;
        Blocks at(max(first_block, share * each), min(q_blocks, (share + 1) * each), query_docs, mine);
        int next = at.next();
        if (next >= 0) {
            load(next);
            store(next, 0);
        }
        const auto step = [&](auto buf_) {
            constexpr int buf = decltype(buf_)::value;
            const int q0 = next * kBlock + half * 32, block_doc = at.doc, there = a.len_q - q0;
            next = at.next();
            __syncthreads();  // this block is stored; the one before it is done with
            if (next >= 0) load(next);

            const int *limits = limit_lds[buf] + half * 32, *row_docs = doc_lds[buf] + half * 32;
            const float *Ms = M_lds[buf] + half * 32, *Ds = D_lds[buf] + half * 32;
            const bool one = !docs || block_doc == wave_doc;
            // a document of the block's queries that none of the wave's keys is in
            const bool other = docs && whole_keys && block_doc >= 0 && block_doc != wave_doc;
#pragma unroll
            for (int i = 0; i < 2 / SPLIT; ++i) {
                if (other || 32 * i >= there || limits[min(32 * i + 31, there - 1)] <= first_key) continue;
                const bool whole = whole_keys && one && limits[32 * i] > last_key;
                f32x16 s = zero16(), dp = zero16();
                struct Pair {
                    Frag<T> q[L::kStage], g[L::kStage];
                };
                Pair two[2];
                const auto read_rows = [&](Pair& x, int n) {
#pragma unroll
                    for (int j = 0; j < L::kStage; ++j) {
                        x.q[j] = L::rows(q_lds[buf], i, n * L::kStage + j, rbase);
                        x.g[j] = L::rows(g_lds[buf], i, n * L::kStage + j, rbase);
                    }
                };
                read_rows(two[0], 0);
                piped<L::kSteps / L::kStage>(two, read_rows, [&](const Pair& x, int n) {
#pragma unroll
                    for (int j = 0; j < L::kStage; ++j) {
                        s = mma(x.q[j], kf[n * L::kStage + j], s);
                        dp = mma(x.g[j], vf[n * L::kStage + j], dp);
                    }
                });
                // columns of fragment n / kCols, features 32 (n % kCols) ...
                constexpr int kCols = DP / 32 / (DP / 32 % L::kStage ? 1 : L::kStage), kWide = DP / 32 / kCols;
                const auto read_cols = [&](Pair& x, int n) {
#pragma unroll
                    for (int j = 0; j < kWide; ++j) {
                        x.g[j] = L::cols(g_lds[buf], i, n / kCols, n % kCols * kWide + j, cbase);
                        x.q[j] = L::cols(q_lds[buf], i, n / kCols, n % kCols * kWide + j, cbase);
                    }
                };
                read_cols(two[0], 0);
                __builtin_amdgcn_sched_barrier(kMayCross);
                f32x16 slope;
                if constexpr (CAP) cap_scores(s, slope, a);
                if constexpr (BIAS) {
                    const int q = start + q0 + 32 * i;
                    add_bias<-1>(s, CAP ? 1.0f : a.c1, table, a.max_distance, key - (q + 4 * h), first_key - (q + 31));
                } else if constexpr (!CAP) {
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[r] *= a.c1;
                }
                if (!whole) {
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        const int at4 = 32 * i + 8 * g + 4 * h;
                        const int4 lm = *reinterpret_cast<const int4*>(limits + at4);
                        int4 dc = {doc, doc, doc, doc};
                        if (docs) dc = *reinterpret_cast<const int4*>(row_docs + at4);
                        const auto sees = [&](int lm1, int dc1) { return live & (key < lm1) & (dc1 == doc); };
                        s[4 * g] = sees(lm.x, dc.x) ? s[4 * g] : -INFINITY;
                        s[4 * g + 1] = sees(lm.y, dc.y) ? s[4 * g + 1] : -INFINITY;
                        s[4 * g + 2] = sees(lm.z, dc.z) ? s[4 * g + 2] : -INFINITY;
                        s[4 * g + 3] = sees(lm.w, dc.w) ? s[4 * g + 3] : -INFINITY;
                    }
                }
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const f32x4 M = *reinterpret_cast<const f32x4*>(Ms + 32 * i + 8 * g + 4 * h);
                    const f32x4 D = *reinterpret_cast<const f32x4*>(Ds + 32 * i + 8 * g + 4 * h);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int r = 4 * g + j;
                        s[r] = exp2_fast(s[r] - M[j]);
                        dp[r] = s[r] * (dp[r] - D[j]);
                    }
                }
                if constexpr (BIAS) {
                    const int base = first_key - (start + q0 + 32 * i);  // distance of row 0, column 0
                    const int m = a.max_distance;
                    if (base + 31 <= -m || base - 31 >= m) {
                        float sum = 0.0f;
#pragma unroll
                        for (int r = 0; r < 16; ++r) sum += dp[r];
                        if (base + 31 <= -m) far_lo += sum;
                        else far_hi += sum;
                    } else {
                        float up = 0.0f, down = 0.0f;  // distances base + n and base + n - 32
                        const int n = lane & 31;
#pragma unroll
                        for (int r = 0; r < 16; ++r) {
                            const int row = row_of(r, h), from = (n + row) & 31;
                            const float v = __shfl(dp[r], from + 32 * h);
                            up += n + row < 32 ? v : 0.0f;
                            down += n + row < 32 ? 0.0f : v;
                        }
                        up = sum_halves(up);
                        down = sum_halves(down);
                        const int where = base + n - 32 * h + m + kSlack;
                        my_dist[where] += h ? down : up;
                    }
                }
                if constexpr (CAP) {
#pragma unroll
                    for (int r = 0; r < 16; ++r) dp[r] *= slope[r];
                }
                Frag<T> p[L::kKeySteps], x[L::kKeySteps];
#pragma unroll
                for (int f = 0; f < L::kKeySteps; ++f) {
                    p[f] = operand(s, f, T{});
                    x[f] = operand(dp, f, T{});
                }
                piped<L::kKeySteps * kCols>(two, read_cols, [&](const Pair& y, int n) {
#pragma unroll
                    for (int j = 0; j < kWide; ++j) {
                        const int d = n % kCols * kWide + j;
                        dv[d] = mma(y.g[j], p[n / kCols], dv[d]);
                        dk[d] = mma(y.q[j], x[n / kCols], dk[d]);
                    }
                });
            }
            if (kBufs == 1) __syncthreads();
            if (next >= 0) store(next, buf ^ (kBufs - 1));
        };
        while (next >= 0) {
            step(std::integral_constant<int, 0>{});
            if (next < 0) break;
            step(std::integral_constant<int, kBufs - 1>{});
        }
        if constexpr (BIAS) {
            // the far tiles join the ends of the table; then one sum a distance
            far_lo = nnk::wave_sum(far_lo);
            far_hi = nnk::wave_sum(far_hi);
            __syncthreads();
            if (lane == 0) {
                my_dist[0] += far_lo;
                my_dist[span - 1] += far_hi;
            }
            __syncthreads();
            if (a.dist_sums) {
                const int n = 2 * a.max_distance + 1;
                float* to = a.dist_sums + ((((size_t)b * a.heads + head) * a.q_splits + share) * tiles + tile) * n;
                for (int i = threadIdx.x; i < n; i += kTpb) {
                    float sum = 0.0f;
                    const int first = i == 0 ? 0 : i + kSlack, last = i == n - 1 ? span : i + kSlack + 1;
                    for (int wv = 0; wv < kWaves; ++wv)
                        for (int j = first; j < last; ++j) sum += dist[wv * span + j];
                    to[i] = sum;
                }
            }
        }
    }

    if constexpr (SPLIT > 1) {
        // the second half's sums, through the tiles' LDS: a register's 64 lanes together
        const int at = strip * (DP / 32 * 16 * 64) + lane;
        float *to_k = reinterpret_cast<float*>(q_lds[0]) + at, *to_v = reinterpret_cast<float*>(g_lds[0]) + at;
        __syncthreads();
        if (half) {
#pragma unroll
            for (int d = 0; d < DP / 32; ++d)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    to_k[(d * 16 + r) * 64] = dk[d][r];
                    to_v[(d * 16 + r) * 64] = dv[d][r];
                }
        }
        __syncthreads();
        if (half) return;
#pragma unroll
        for (int d = 0; d < DP / 32; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                dk[d][r] += to_k[(d * 16 + r) * 64];
                dv[d][r] += to_v[(d * 16 + r) * 64];
            }
    }
    if (!in) return;
    if (a.kv_sums) {
        const size_t at = (((size_t)b * parts + part) * a.len_k + key) * a.dim;
        float *kout = a.kv_sums + at, *vout = kout + (size_t)a.batch * parts * a.len_k * a.dim;
#pragma unroll
        for (int d = 0; d < DP / 32; ++d)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int at = 32 * d + 8 * g + 4 * h;
                store4<float, VEC>(kout, at, a.dim, dk[d][4 * g], dk[d][4 * g + 1], dk[d][4 * g + 2], dk[d][4 * g + 3]);
                store4<float, VEC>(vout, at, a.dim, dv[d][4 * g], dv[d][4 * g + 1], dv[d][4 * g + 2], dv[d][4 * g + 3]);
            }
        return;
    }
    T* kout = (T*)a.dk + b * a.ks[0] + (long long)key * a.ks[1] + kv * a.ks[2];
    T* vout = (T*)a.dv + b * a.vs[0] + (long long)key * a.vs[1] + kv * a.vs[2];
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int at = 32 * d + 8 * g + 4 * h;
            store4<T, VEC>(kout, at, a.dim, dk[d][4 * g] * a.scale, dk[d][4 * g + 1] * a.scale,
                dk[d][4 * g + 2] * a.scale, dk[d][4 * g + 3] * a.scale);
            store4<T, VEC>(vout, at, a.dim, dv[d][4 * g], dv[d][4 * g + 1], dv[d][4 * g + 2], dv[d][4 * g + 3]);
        }
}

// dk and dv from the sums of a key head's parts (heads, shares of the queries), in their
// order; 4 features a thread.
template <typename T, bool VEC>
__global__ __launch_bounds__(kTpb) void attn_kv_sum_kernel(Args a, int quads, long long total) {
    const long long n = (long long)blockIdx.x * kTpb + threadIdx.x;
    if (n >= total) return;
    const int d = (int)(n % quads) * 4;
    const long long row = n / quads;
    const int key = (int)(row % a.len_k), kv = (int)(row / a.len_k % a.kv_heads), b = (int)(row / a.len_k / a.kv_heads);
    const int parts = a.heads / a.heads_each * a.q_splits, mine = parts / a.kv_heads;
    const float* from = a.kv_sums + (((size_t)b * parts + kv * mine) * a.len_k + key) * a.dim + d;
    const size_t step = (size_t)a.len_k * a.dim, v_at = (size_t)a.batch * parts * a.len_k * a.dim;
    float k[4] = {0.0f, 0.0f, 0.0f, 0.0f}, v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int g = 0; g < mine; ++g) {
        if constexpr (VEC) {
            const float4 x = nnk::ld4(from + g * step), y = nnk::ld4(from + g * step + v_at);
            k[0] += x.x, k[1] += x.y, k[2] += x.z, k[3] += x.w;
            v[0] += y.x, v[1] += y.y, v[2] += y.z, v[3] += y.w;
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (d + j < a.dim) k[j] += from[g * step + j], v[j] += from[g * step + v_at + j];
        }
    }
    store4<T, VEC>((T*)a.dk + b * a.ks[0] + key * a.ks[1] + kv * a.ks[2], d, a.dim, k[0] * a.scale, k[1] * a.scale,
        k[2] * a.scale, k[3] * a.scale);
    store4<T, VEC>((T*)a.dv + b * a.vs[0] + key * a.vs[1] + kv * a.vs[2], d, a.dim, v[0], v[1], v[2], v[3]);
}

// dbias[bucket, head]: a workgroup a head.  First the sums of each distance over batch and
// key tiles, in 64 bits, 2 threads a distance, each its half of the rows in order; then a
// wave a bucket, a lane's distances in order, the lanes' as a tree.
constexpr int kBiasTpb = 1024, kBiasCols = kBiasTpb / 2;
__global__ __launch_bounds__(kBiasTpb) void attn_bias_grad_kernel(float* dbias, const float* dist_sums,
    const int* bucket, int batch, int heads, int buckets, int tiles, int n) {
    __shared__ double part[2][kBiasCols], sums[2 * kMaxDistance + 1];
    __shared__ int of[2 * kMaxDistance + 1];
    const int head = blockIdx.x, col = threadIdx.x % kBiasCols, half = threadIdx.x / kBiasCols;
    const int rows = batch * tiles, each = (rows + 1) / 2, first = half * each, last = min(rows, first + each);
    for (int i0 = 0; i0 < n; i0 += kBiasCols) {
        const int i = i0 + col;
        double sum = 0.0;
        if (i < n) {
#pragma unroll 8
            for (int r = first; r < last; ++r) {
                const int b = r / tiles;
                sum += dist_sums[(((size_t)b * heads + head) * tiles + r - b * tiles) * n + i];
            }
        }
        part[half][col] = sum;
        __syncthreads();
        if (half == 0 && i < n) {
            sums[i] = part[0][col] + part[1][col];
            of[i] = min(max(bucket[i], 0), buckets - 1);
        }
        __syncthreads();
    }
    for (int m = threadIdx.x / 64; m < buckets; m += kBiasTpb / 64) {
        double sum = 0.0;
        for (int i = threadIdx.x % 64; i < n; i += 64) sum += of[i] == m ? sums[i] : 0.0;
#pragma unroll
        for (int x = 1; x < 64; x <<= 1) sum += __shfl_xor(sum, x);
        if (threadIdx.x % 64 == 0) dbias[(size_t)m * heads + head] = (float)sum;
    }
}

template <typename T, int DP, bool CAP, bool BIAS, bool VEC, int SPLIT>
bool launch_split(const Args& a, int tiles, hipStream_t s, const char* what) {
    const size_t lds = BIAS ? kWaves * (2 * (a.max_distance + kSlack) + 1) * sizeof(float) : 0;
    if constexpr (BIAS) {
        static std::atomic<unsigned long long> done{0};
        if (!raise_lds((const void*)attn_bwd_kv_kernel<T, DP, CAP, BIAS, VEC, SPLIT>,
                kWaves * (2 * (kMaxDistance + kSlack) + 1) * sizeof(float), done, what))
            return false;
    }
    const long long groups = (long long)tiles * (a.heads / a.heads_each) * a.q_splits * a.batch;
    attn_bwd_kv_kernel<T, DP, CAP, BIAS, VEC, SPLIT><<<(unsigned)groups, kTpb, lds, s>>>(a, tiles);
    nnk_after_launch(what, s);
    return true;
}

template <typename T, int DP, bool CAP, bool BIAS, bool VEC>
bool launch(const Args& a, hipStream_t s, const char* what) {
    const int tiles = (a.len_k + a.kv_keys - 1) / a.kv_keys;
    if (!(a.kv_keys < kRows ? launch_split<T, DP, CAP, BIAS, VEC, 2>(a, tiles, s, what)
                            : launch_split<T, DP, CAP, BIAS, VEC, 1>(a, tiles, s, what)))
        return false;
    if (a.kv_sums) {
        const int quads = (a.dim + 3) / 4;
        const long long total = (long long)a.batch * a.kv_heads * a.len_k * quads;
        attn_kv_sum_kernel<T, VEC><<<(unsigned)((total + kTpb - 1) / kTpb), kTpb, 0, s>>>(a, quads, total);
        nnk_after_launch(what, s);
    }
    return true;
}

}  // namespace

bool nnk_attention_backward_kv(const Args& a, bool half, hipStream_t s, const char* what) {
    return NNK_ATTN_DISPATCH(a, half, launch, a, s, what);
}

void nnk_attention_bias_grad(const Args& a, float* dbias, hipStream_t s, const char* what) {
    const int rows = (a.len_k + a.kv_keys - 1) / a.kv_keys * a.q_splits;  // of a request and head
    attn_bias_grad_kernel<<<(unsigned)a.heads, kBiasTpb, 0, s>>>(dbias, a.dist_sums, a.bucket, a.batch, a.heads,
        a.buckets, rows, 2 * a.max_distance + 1);
    nnk_after_launch(what, s);
}
