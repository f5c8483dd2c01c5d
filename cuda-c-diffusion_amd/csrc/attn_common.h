// attn_common.h -- what the attention kernels share: fragments of the matrix
// cores, tiles in LDS, score functions, masks.
//
// Layout.  All products are 32 x 32 tiles of the matrix cores (bf16: 32x32x16,
// fp32: 32x32x2, four of them where bf16 has one).  In such a tile the lane
// l = (l & 31) + 32 h holds column l & 31 and the rows 8 g + 4 h + j (g, j in
// 0..3) in its 16 registers.  A product whose result is the next one's operand is
// therefore formed with the next one's free index in the columns: scores as keys x
// queries where they go on to values or query gradients, as queries x keys where
// they go on to key and value gradients.  A lane's registers are then already the
// operand, with the contracted index in the order 8 g + 4 h + j, and the other
// operand is read from LDS in that order: rows by 16-byte reads, columns by the
// transposing read (bf16) or by one read a row (fp32).
//
// Rows in LDS are a power of two long and hold their 16-byte chunks in an order of
// their own, chunk c at c ^ F(row), so that 16 lanes' reads of successive rows, and the
// 4 rows x 64 bytes of two transposing reads, meet different banks.  (Rows 32 bytes
// apart from a power of two had 40 % of the LDS cycles in conflicts.)
#pragma once

#include <algorithm>
#include <atomic>
#include <cmath>
#include <type_traits>

#include "nn_attention.h"
#include "nnk_common.h"

namespace attn {

typedef __bf16 bf16;
typedef bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

constexpr int kBlock = 64;     // keys (or queries) of a tile in LDS
constexpr int kTpb = 256;
constexpr int kWaves = kTpb / 64;
constexpr int kRows = 32 * kWaves;  // columns of a workgroup: queries, or keys in the key gradients
constexpr int kCus = 256;
constexpr int kSplitBelow = 2 * kCus;  // workgroups below which blocks are shared by two waves
constexpr int kMaxDistance = 1023;
constexpr int kMaxLen = (1 << 30) - 4096;  // two of them, kMaxDistance and a tile fit in 32 bits
constexpr int kMostHeads = 1 << 20;  // and requests whose tiles are put in order: workgroups of 1024 threads
constexpr int kTicketWords = 2048;  // at the front of every forward workspace: zeros between calls
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;

template <typename T>
struct Type;
template <>
struct Type<bf16> {
    typedef bf16x8 Frag;
    static constexpr int CE = 8;  // values of 16 bytes, and of a lane's operand
};
template <>
struct Type<float> {
    typedef f32x4 Frag;
    static constexpr int CE = 4;
};
template <typename T>
using Frag = typename Type<T>::Frag;

__device__ __forceinline__ f32x16 mma(bf16x8 a, bf16x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mma(f32x4 a, f32x4 b, f32x16 c) {
#pragma unroll
    for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], c, 0, 0, 0);
    return c;
}

__device__ __forceinline__ f32x16 zero16() {
    f32x16 z;
#pragma unroll
    for (int r = 0; r < 16; ++r) z[r] = 0.0f;
    return z;
}

// Row of register r in half h of a 32 x 32 tile.
__device__ __forceinline__ int row_of(int r, int h) { return 8 * (r >> 2) + 4 * h + (r & 3); }

// The values of both halves' lanes l and l + 32, in both.
struct Halves {
    float lower, upper;
};
__device__ __forceinline__ Halves halves(float v) {
    const unsigned u = __builtin_bit_cast(unsigned, v);
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    const unsigned lower = r[0], upper = r[1];  // a bit cast of r[1] itself gives r[0]
    return {__builtin_bit_cast(float, lower), __builtin_bit_cast(float, upper)};
}
__device__ __forceinline__ float sum_halves(float v) {
    const Halves x = halves(v);
    return x.lower + x.upper;
}
__device__ __forceinline__ float max_halves(float v) {
    const Halves x = halves(v);
    return fmaxf(x.lower, x.upper);
}
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// ---------------------------------------------------------------------------
// Tiles in LDS
// ---------------------------------------------------------------------------
template <typename T, int DP>
struct Lds {
    static constexpr int kUsed = DP * (int)sizeof(T);
    static constexpr int kRowBytes = kUsed <= 64 ? 64 : kUsed <= 128 ? 128 : kUsed <= 256 ? 256 : 512;
    static constexpr int kBytes = kBlock * kRowBytes;
    static constexpr int kSteps = DP / (2 * Type<T>::CE);     // fragments of a row
    static constexpr int kKeySteps = 32 / (2 * Type<T>::CE);  // fragments of 32 rows
    // fragments of a stage of one or of two operands: enough products to hide its reads
    static constexpr int kWide = sizeof(T) == 2 ? 4 : 2, kStage = kWide / 2;

    // Bits of the row in other places, so F(a ^ b) = F(a) ^ F(b).
    static __host__ __device__ constexpr int F(int row) {
        if (sizeof(T) == 2)
            return kRowBytes == 256 ? (row & 3) << 2 | (row >> 2 & 3)
                : kRowBytes == 128 ? (row >> 1 & 1) << 2 | (row >> 2 & 3) : row >> 2 & 3;
        return kRowBytes == 128 ? row >> 1 & 7 : (row >> 2 & 1) << 3 | (row >> 3 & 1) << 2 | (row & 3);
    }
    static __device__ __forceinline__ int at(int row, int chunk) { return row * kRowBytes + ((chunk ^ F(row)) << 4); }

    // This lane's place in the operands below.
    static __device__ __forceinline__ int row_base(int lane) { return at(lane & 31, lane >> 5); }
    static __device__ __forceinline__ int col_base(int lane) {
        const int h = lane >> 5;
        if (sizeof(T) == 2)
            return at(4 * h + (lane >> 2 & 3), (lane & 16) >> 3 | (lane & 2) >> 1) + (lane & 1) * 8;
        return at(4 * h, lane >> 2 & 7) + (lane & 3) * 4;
    }
    // Operand whose free index is the tile's row: fragment u of rows 32 i ...
    static __device__ __forceinline__ Frag<T> rows(const char* t, int i, int u, int base) {
        return *reinterpret_cast<const Frag<T>*>(t + 32 * i * kRowBytes + (base ^ (u << 5)));
    }
    // Operand whose free index is the column 32 d + (lane & 31) and whose contracted
    // index is the rows 32 i ..., fragment f of kKeySteps.
    static __device__ __forceinline__ Frag<T> cols(const char* t, int i, int f, int d, int base) {
        if constexpr (sizeof(T) == 2) {
            typedef __attribute__((address_space(3))) i16x4* LdsPtr;
            const char* p = t + (32 * i + 16 * f) * kRowBytes;
            const i16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsPtr)(p + (base ^ (d << 6))));
            const i16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsPtr)(p + 8 * kRowBytes + (base ^ (d << 6) ^ (F(8) << 4))));
            const bf16x4 x = __builtin_bit_cast(bf16x4, a), y = __builtin_bit_cast(bf16x4, b);
            return __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
        } else {
            f32x4 v;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                v[j] = *reinterpret_cast<const float*>(t + (32 * i + 8 * f + j) * kRowBytes +
                    (base ^ ((8 * d ^ F(8 * f & 31) ^ F(j)) << 4)));
            return v;
        }
    }
};

// Products whose operands come from LDS: stage n + 1's reads are issued before stage n's
// products, and vector instructions may move anywhere.  The compiler by itself puts each
// read next to its product and waits for it there, which at one or two waves a SIMD is the
// latency of LDS for every product.  load(stage, n) reads, use(stage, n) multiplies;
// stages[0] is read by the caller, early enough to have other work in between.
constexpr int kMayCross = 0x6;  // vector and scalar instructions
template <int N, typename Stage, typename Load, typename Use>
__device__ __forceinline__ void piped(Stage (&stages)[2], const Load& load, const Use& use) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
        if (n + 1 < N) load(stages[(n + 1) & 1], n + 1);
        __builtin_amdgcn_sched_barrier(kMayCross);
        use(stages[n & 1], n);
        __builtin_amdgcn_sched_barrier(kMayCross);
    }
}

// Registers of a tile's fragment f as the operand of the next product.  bf16: the
// probabilities (or score gradients) are rounded to bf16 here, each by at most 2^-8 of
// itself and independently of the others, so that the sum over them is off by about what
// its own rounding to bf16 adds; softmax sums and the bias gradient are taken before.
__device__ __forceinline__ bf16x8 operand(const f32x16& s, int f, bf16) {
    bf16x8 v;
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = (bf16)s[8 * f + j];
    return v;
}
__device__ __forceinline__ f32x4 operand(const f32x16& s, int f, float) {
    f32x4 v;
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = s[4 * f + j];
    return v;
}

// 16 bytes of a row from feature d0 on.  Features from `dim` on are zeros, or (VEC) a
// chunk wholly past them is the row's first one, for the caller to leave out: a choice
// here would wait for the load.
template <typename T, bool VEC>
__device__ __forceinline__ u32x4 load_chunk(const T* row, int d0, int dim) {
    if constexpr (VEC) return *reinterpret_cast<const u32x4*>(row + (d0 < dim ? d0 : 0));
    T e[Type<T>::CE];
#pragma unroll
    for (int j = 0; j < Type<T>::CE; ++j) e[j] = d0 + j < dim ? row[d0 + j] : (T)0.0f;
    u32x4 v;
    __builtin_memcpy(&v, e, 16);
    return v;
}
template <typename T, bool VEC>
__device__ __forceinline__ Frag<T> load_frag(const T* row, int d0, int dim) {
    const u32x4 v = load_chunk<T, VEC>(row, d0, dim);
    return __builtin_bit_cast(Frag<T>, d0 < dim ? v : u32x4{0, 0, 0, 0});
}

// Four consecutive features d..d+3 of an output row.
template <typename T, bool VEC>
__device__ __forceinline__ void store4(T* row, int d, int dim, float a, float b, float c, float e) {
    const float v[4] = {a, b, c, e};
    if constexpr (VEC) {
        if (d >= dim) return;
        if constexpr (sizeof(T) == 2) {
            bf16x4 o;
#pragma unroll
            for (int j = 0; j < 4; ++j) o[j] = (bf16)v[j];
            *reinterpret_cast<bf16x4*>(row + d) = o;
        } else {
            f32x4 o = {a, b, c, e};
            *reinterpret_cast<f32x4*>(row + d) = o;
        }
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (d + j < dim) row[d + j] = (T)v[j];
    }
}

// A 64-row tile on its way from memory to LDS: loaded into registers while the tile
// before it is used, stored when that is done.  A lane's offsets in a tile are formed
// once, in 32 bits (the host sees to it), and added to the tile's uniform address.
template <typename T, int DP, bool VEC>
struct Staged {
    static constexpr int kPerRow = DP / Type<T>::CE;
    static constexpr int N = kBlock * kPerRow / kTpb;
    u32x4 v[N];
    unsigned off[VEC ? N : 1];

    static __device__ __forceinline__ int row(int n) { return (n * kTpb + (int)threadIdx.x) / kPerRow; }
    static __device__ __forceinline__ int chunk(int n) { return (n * kTpb + (int)threadIdx.x) % kPerRow; }
    // A chunk past the features is the row's first one: whatever it meets has zeros there,
    // or is not stored.
    static __device__ __forceinline__ unsigned offset(int n, int r, long long stride, int dim) {
        return (unsigned)r * (unsigned)(stride * (int)sizeof(T)) + (chunk(n) * Type<T>::CE < dim ? chunk(n) * 16 : 0);
    }
    __device__ __forceinline__ void init(long long stride, int dim) {
        if constexpr (VEC) {
#pragma unroll
            for (int n = 0; n < N; ++n) off[n] = offset(n, row(n), stride, dim);
        }
    }
    // Row r of the tile is base + min(r, last) * stride.
    __device__ __forceinline__ void load(const T* base, long long stride, int last, int dim) {
        if constexpr (VEC) {
            const char* p = reinterpret_cast<const char*>(base);
            if (last >= kBlock - 1) {
#pragma unroll
                for (int n = 0; n < N; ++n) v[n] = *reinterpret_cast<const u32x4*>(p + off[n]);
            } else {
#pragma unroll
                for (int n = 0; n < N; ++n)
                    v[n] = *reinterpret_cast<const u32x4*>(p + offset(n, min(row(n), last), stride, dim));
            }
        } else {
#pragma unroll
            for (int n = 0; n < N; ++n)
                v[n] = load_chunk<T, false>(base + min(row(n), last) * stride, chunk(n) * Type<T>::CE, dim);
        }
    }
    // All of the rows, or (!all) zeros in place of those that are not kept, whatever they
    // hold; keep(n): this lane's n-th row.
    template <typename Keep>
    __device__ __forceinline__ void store(char* lds, bool all, const Keep& keep) const {
        if (all) {
#pragma unroll
            for (int n = 0; n < N; ++n) *reinterpret_cast<u32x4*>(lds + Lds<T, DP>::at(row(n), chunk(n))) = v[n];
        } else {
#pragma unroll
            for (int n = 0; n < N; ++n)
                *reinterpret_cast<u32x4*>(lds + Lds<T, DP>::at(row(n), chunk(n))) = keep(n) ? v[n] : u32x4{0, 0, 0, 0};
        }
    }
};

// ---------------------------------------------------------------------------
// The call, as the kernels take it
// ---------------------------------------------------------------------------
struct Args {
    const void *q, *k, *v;
    void* out;
    float* lse;
    const void* dout;
    void *dq, *dk, *dv;
    float2* stat;      // backward: per query, log2 of its sum and its <p, dp>
    float* dist_sums;  // backward: sums of score gradients by distance, per key tile
    // How the gradients are divided, and the sums of the parts that are added up afterwards:
    int heads_each, q_splits, kv_keys;  // key gradients: heads and share of the queries of a workgroup; its keys
    int k_splits, q_rows;               // query gradients: share of the keys; queries
    float* kv_sums;                     // dk / scale, then dv, [batch, parts, len_k, dim], or null
    float* q_sums;                      // dq / scale [batch, heads, k_splits, len_q, dim], or null
    float2* stat_sums;                  // sums of p and of p dp [batch, heads, k_splits, len_q]
    const int4* key_docs;    // per block of 64 keys: least and largest document, whether any is negative
    const int4* query_docs;  // per block of 64 queries
    const int *row_order, *key_order;  // with documents: tiles of a request by falling work, or null
    long long qs[3], ks[3], vs[3], os[3];
    int batch, len_q, len_k, heads, kv_heads, group, dim;
    int mask, buckets, max_distance;
    float scale, c1, c2;  // score in units of log2: c1 * s, or c2 * tanh(c1 * s)
    float series[6];      // c2 tanh(c1 s) = x (series[0] + w (series[1] + ...)), w = x^2, for small x = s unit
    float inv_c2;
    float unit;           // 1, or c1 where coefficients for s would not be normal values
    float near_end, exponent;  // how small: |x| below this; 2 |c1 s| in units of log2 is |x| exponent
    float small, tiny;    // |s| below this: the series of s alone; and of its first 4 terms (0 if unit is c1)
    const int *q_start, *k_len, *prefix, *doc_q, *doc_k, *bucket;
    const float* bias;
    bool vec;
};

// Keys of request b, and the position of its query 0.
__device__ __forceinline__ int keys_of(const Args& a, int b) {
    return a.k_len ? min(max(a.k_len[b], 0), a.len_k) : a.len_k;
}
__device__ __forceinline__ int start_of(const Args& a, int b) {
    // where every query lies before key 0, or behind the last one, by more than max_distance, how
    // far does not matter: so positions and distances stay in the type (lengths below kMaxLen)
    constexpr int kFar = kMaxDistance + 1;
    return a.q_start ? min(max(a.q_start[b], -a.len_q - kFar), a.len_k + kFar) : a.len_k - a.len_q;
}
// The query at position pos sees keys 0 .. limit - 1, of which its document's.
__device__ __forceinline__ int limit_of(const Args& a, int b, int keys, int pos) {
    if (a.mask == NN_MASK_NONE) return keys;
    int n = pos + 1;
    if (a.mask == NN_MASK_PREFIX) n = max(n, a.prefix[b]);
    return min(keys, max(n, 0));
}

// ---------------------------------------------------------------------------
// Scores
// ---------------------------------------------------------------------------
// t = tanh(y) and its slope 1 - t^2.  With r = 1 / (e^2|y| + 1): |t| = 1 - 2 r and
// slope = 4 r (1 - r), which keeps its digits where the cap is reached (1 - t t would
// not).  t is off by about 2^-23 of 1, so for small y it is the odd series to y^11
// instead (relative error below 2^-24 for |y| < 3/8).  A cap is chosen so that most
// scores are far below it; a wave that has them all there forms only the series, half
// the other's cycles.
__device__ __forceinline__ float tanh_series(float y) {
    const float w = y * y;
    float c = fmaf(w, -0.00886323553f, 0.0218694885f);
    c = fmaf(w, c, -0.0539682540f);
    c = fmaf(w, c, 0.133333333f);
    c = fmaf(w, c, -0.333333333f);
    return fmaf(y * w, c, y);
}
// ends of the series of 6 and of 4 terms: the next term is below 2^-24 of the first
constexpr float kSeriesEnd = 0.375f, kShortSeriesEnd = 0.14f;
// s[r] = c2 tanh(c1 s[r])
__device__ __forceinline__ void cap_scores(f32x16& s, float c1, float c2) {
    float top = 0.0f;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        s[r] *= c1;
        top = fmaxf(top, fabsf(s[r]));
    }
    if (__all(top < kSeriesEnd)) {  // fmaxf passes over NaN; the series keeps it
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = tanh_series(s[r]) * c2;
    } else {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const float y = s[r], q = __builtin_amdgcn_rcpf(exp2_fast(fabsf(y) * (2.0f * kLog2e)) + 1.0f);
            s[r] = (fabsf(y) < kSeriesEnd ? tanh_series(y) : copysignf(fmaf(-2.0f, q, 1.0f), y)) * c2;
        }
    }
}
// c2 tanh(c1 s) by the first TERMS terms of its series
template <int TERMS>
__device__ __forceinline__ float cap_series(float s, const Args& a) {
    const float w = s * s;
    float c = a.series[TERMS - 1];
#pragma unroll
    for (int t = TERMS - 2; t >= 0; --t) c = fmaf(w, c, a.series[t]);
    return s * c;
}
// The capped scores with the slope 1 - tanh^2, for the gradients.
__device__ __forceinline__ void cap_scores(f32x16& s, f32x16& slope, const Args& a) {
    const auto slope_of = [&](float x) {
        const float t = x * a.inv_c2;
        return fmaf(-t, t, 1.0f);
    };
    float top = 0.0f;
#pragma unroll
    for (int r = 0; r < 16; ++r) top = fmaxf(top, fabsf(s[r]));
    if (__all(top < a.tiny)) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            s[r] = cap_series<4>(s[r], a);
            slope[r] = slope_of(s[r]);
        }
    } else if (__all(top < a.small)) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            s[r] = cap_series<6>(s[r], a);
            slope[r] = slope_of(s[r]);
        }
    } else {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const float x = s[r] * a.unit, q = __builtin_amdgcn_rcpf(exp2_fast(fabsf(x) * a.exponent) + 1.0f);
            const bool near = fabsf(x) < a.near_end;
            s[r] = near ? cap_series<6>(x, a) : copysignf(fmaf(-2.0f, q, 1.0f), x) * a.c2;
            slope[r] = near ? slope_of(s[r]) : 4.0f * q * (1.0f - q);
        }
    }
}

// Entries of a keys x queries tile that this lane's query does not see become -inf: keys
// from `limit` on and, with documents (`docs`: the tile's 32 keys', in LDS, -1 for every
// negative one), of others than `doc`.  No branches: a tile's border is a few of these, not a
// path of its own.
__device__ __forceinline__ void hide(f32x16& s, int k0, int limit, const int* docs, int doc, int h) {
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = k0 + row_of(r, h) < limit ? s[r] : -INFINITY;
    if (docs) {
        const int own = doc >= 0 ? doc : -2;  // no key has this
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int4 d = *reinterpret_cast<const int4*>(docs + 8 * g + 4 * h);
            s[4 * g] = d.x == own ? s[4 * g] : -INFINITY;
            s[4 * g + 1] = d.y == own ? s[4 * g + 1] : -INFINITY;
            s[4 * g + 2] = d.z == own ? s[4 * g + 2] : -INFINITY;
            s[4 * g + 3] = d.w == own ? s[4 * g + 3] : -INFINITY;
        }
    }
}

// Bias of head `head` by distance -m..m, in units of log2, into LDS.
__device__ __forceinline__ void load_bias(const Args& a, float* table, int head) {
    for (int i = threadIdx.x; i < 2 * a.max_distance + 1; i += kTpb) {
        const int n = min(max(a.bucket[i], 0), a.buckets - 1);
        table[i] = a.bias[(size_t)n * a.heads + head] * kLog2e;
    }
}

// s = c s + bias of the tile's entries, whose distances are the lane's rel + STEP * (8 g + j)
// (register 4 g + j), and in the wave `least` at least and 62 more at most.  Tiles wholly
// past max_distance, which most are, add one value.
template <int STEP>
__device__ __forceinline__ void add_bias(f32x16& s, float c, const float* table, int m, int rel, int least) {
    if (least + 62 <= -m || least >= m) {
        const float bias = table[least >= m ? 2 * m : 0];
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = s[r] * c + bias;
    } else {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int d = rel + STEP * (8 * (r >> 2) + (r & 3));
            s[r] = s[r] * c + table[min(max(d, -m), m) + m];
        }
    }
}

// ---------------------------------------------------------------------------
// Blocks of 64 that can meet
// ---------------------------------------------------------------------------
// Two ranges of documents with one in common (an empty range has none).
__device__ __forceinline__ bool docs_meet(const int4& x, const int4& y) { return x.x <= y.y && y.x <= x.y; }
__device__ __forceinline__ int4 join_docs(const int4* docs, int first, int last) {
    int4 all = {INT32_MAX, INT32_MIN, 0, 0};
    for (int i = first; i < last; ++i) {
        all.x = min(all.x, docs[i].x);
        all.y = max(all.y, docs[i].y);
    }
    return all;
}
// Documents of the blocks first .. first + count - 1 of queries, or of keys.
__device__ __forceinline__ int4 query_docs_of(const Args& a, int b, int first, int count) {
    const int n = (a.len_q + kBlock - 1) / kBlock;
    return a.query_docs ? join_docs(a.query_docs + (size_t)b * n, first, min(first + count, n)) : int4{0, 0, 0, 0};
}
__device__ __forceinline__ int4 key_docs_of(const Args& a, int b, int first, int count) {
    const int n = (a.len_k + kBlock - 1) / kBlock;
    return a.key_docs ? join_docs(a.key_docs + (size_t)b * n, first, min(first + count, n)) : int4{0, 0, 0, 0};
}

// The blocks first..last-1 that have documents of `mine` among theirs (`docs` null: all),
// in order, 64 of them looked at a time, one a lane.
struct Blocks {
    const int4* docs;
    int4 mine, own;  // own: documents of this lane's block
    int base, last;
    unsigned long long m;
    int doc;        // of the block that next() gave: the one document of all its positions, or -1
    bool negative;  // whether any of its positions has none

    __device__ __forceinline__ Blocks(int first, int last_, const int4* docs_, const int4& mine_)
        : docs(docs_), mine(mine_), own{0, 0, 0, 0}, base(first), last(last_), doc(-1),
          negative(false) {
        look();
    }
    __device__ __forceinline__ void look() {
        const int b = base + (int)(threadIdx.x & 63);
        if (docs && b < last) own = docs[b];
        m = __ballot(b < last && (!docs || docs_meet(own, mine)));
    }
    // The next block, or -1.
    __device__ __forceinline__ int next() {
        while (!m) {
            base += 64;
            if (base >= last) return -1;
            look();
        }
        const int i = __builtin_ctzll(m);
        m &= m - 1;
        if (docs) {
            const int lo = __builtin_amdgcn_readlane(own.x, i), hi = __builtin_amdgcn_readlane(own.y, i);
            negative = __builtin_amdgcn_readlane(own.z, i) != 0;
            doc = lo == hi && !negative ? lo : -1;
        }
        return base + i;
    }
};

// What a workgroup of `owners` (heads, or parts, of all requests) times `tiles` takes.
// Without an order of the tiles each XCD has its own owners, one after another.  With one,
// the owners of an XCD (of all, if they do not divide) take turns at the tiles of most work:
// uneven tiles started in their own order kept the CUs busy two thirds of the time (8192
// packed tokens: forward 101 -> 83 us, a training step 704 -> 597 us with three launches for
// the orders).
struct Turn {
    int owner, tile;
};
__device__ __forceinline__ Turn turn_of(int block, int blocks, int owners_each, int tiles, const int* order, bool last_first) {
    const int owners = blocks / tiles;
    if (!order) {
        const int w = nnk::xcd_swizzle(block, blocks), t = w % tiles;
        return {w / tiles, last_first ? tiles - 1 - t : t};
    }
    int owner, rank;
    if (owners % nnk::kNumXcd == 0) {
        const int own = owners / nnk::kNumXcd, k = block / nnk::kNumXcd;
        owner = block % nnk::kNumXcd * own + k % own;
        rank = k / own;
    } else {
        owner = block % owners;
        rank = block / owners;
    }
    return {owner, order[owner / owners_each * tiles + rank]};
}

// Raises kernel fn's limit of dynamic LDS to `bytes` on the current device, once a
// device (`done` has a bit for each).  False after recording an error.
inline bool raise_lds(const void* fn, size_t bytes, std::atomic<unsigned long long>& done, const char* what) {
    int dev = -1;
    hipError_t e = hipGetDevice(&dev);
    if (e == hipSuccess && dev >= 64) e = hipErrorInvalidDevice;
    if (e == hipSuccess && !(done.load(std::memory_order_relaxed) >> dev & 1)) {
        e = hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
        if (e == hipSuccess) done.fetch_or(1ull << dev, std::memory_order_relaxed);
    }
    if (e == hipSuccess) return true;
    (void)hipGetLastError();
    nnk_set_error((int)e, "%s: LDS of %zu bytes on device %d: %s", what, bytes, dev, hipGetErrorString(e));
    return false;
}

}  // namespace attn

// Documents of each block of 64 into `ws`, for args.key_docs and query_docs (no documents:
// nothing).
void nnk_attention_docs(attn::Args& args, float* ws, hipStream_t s, const char* what);
// Tiles of `own` queries (or keys) of each request by falling work into `order`; null if
// there are more than the counting takes.
const int* nnk_attention_order(const attn::Args& args, bool keys, int own, float* order, hipStream_t s, const char* what);
// One launch each; `half`: bf16.  False after recording an error.
bool nnk_attention_forward(const attn::Args& args, bool half, hipStream_t s, const char* what);
bool nnk_attention_backward_q(const attn::Args& args, bool half, hipStream_t s, const char* what);
bool nnk_attention_backward_kv(const attn::Args& args, bool half, hipStream_t s, const char* what);
// The form for few queries; when it is taken; the floats that it needs after the tickets, and
// a bound on them for every smaller batch and shorter lengths.
bool nnk_attention_is_few(const NnAttention* a);
size_t nnk_attention_few_floats(const NnAttention* a);
size_t nnk_attention_few_most(const NnAttention* a);
bool nnk_attention_few(const attn::Args& args, bool half, float* ws, hipStream_t s, const char* what);
// Bias gradient from args.dist_sums.
void nnk_attention_bias_grad(const attn::Args& args, float* dbias, hipStream_t s, const char* what);

// FN<T, DP, CAP, BIAS, VEC> for the call's type, feature count, score terms and alignment.
// Rows that are not on 16 bytes are taken element by element, in one size.
#define NNK_ATTN_DISPATCH(args, bf, FN, ...)                                                              \
    [&]() {                                                                                               \
        auto by_dim = [&](auto type, auto cap, auto bias) {                                               \
            using T_ = decltype(type);                                                                    \
            constexpr bool C_ = decltype(cap)::value, B_ = decltype(bias)::value;                         \
            if (!(args).vec) return FN<T_, 128, C_, B_, false>(__VA_ARGS__);                              \
            switch (((args).dim + 31) / 32) {                                                             \
            case 1: return FN<T_, 32, C_, B_, true>(__VA_ARGS__);                                         \
            case 2: return FN<T_, 64, C_, B_, true>(__VA_ARGS__);                                         \
            case 3: return FN<T_, 96, C_, B_, true>(__VA_ARGS__);                                         \
            default: return FN<T_, 128, C_, B_, true>(__VA_ARGS__);                                       \
            }                                                                                             \
        };                                                                                                \
        auto by_terms = [&](auto type) {                                                                  \
            using Yes = std::true_type;                                                                   \
            using No = std::false_type;                                                                   \
            if ((args).c2 != 0.0f) return (args).buckets > 0 ? by_dim(type, Yes{}, Yes{}) : by_dim(type, Yes{}, No{}); \
            return (args).buckets > 0 ? by_dim(type, No{}, Yes{}) : by_dim(type, No{}, No{});             \
        };                                                                                                \
        return (bf) ? by_terms(attn::bf16{}) : by_terms(0.0f);                                            \
    }()
