// k_cache_few.hip -- attention over a paged cache, few queries a key head (decoding steps,
// drafted tokens, small chunks).
//
// Reading the cache once is the whole cost.  The queries of all heads that share a key head are
// columns of 16 x 16 tiles of the matrix cores, one or two of them, so a key is read once for
// all; the keys are split over workgroups and, within one, dealt out to its 4 waves by blocks
// of 32.  A wave keeps its own running maximum, sum and output; waves are joined in LDS,
// workgroups by the one that is done last (a ticket a unit; it reads the others' results in
// their order, so the sum does not depend on who is last, and leaves the ticket at zero).
//
// In a tile lane l = (l & 15) + 16 h holds column l & 15 and the rows 4 h + j.  Scores are
// keys x queries, so that they are already the other operand of the product with the values.
// A key goes from memory to the registers of the lanes that multiply it; 4-bit features become
// bf16, which holds them exactly, two an instruction, their scale included.  Values pass through
// LDS, where the transposing read turns them (bf16), or are read a feature a lane (fp32 pages).
// fp32 queries and probabilities meet 4-bit pages as three bf16 parts each, 24 bits of them.
#include "attn_common.h"
#include "cache_common.h"

namespace {
using namespace attn;
using cache::Pages;

constexpr int kKeys = 32;       // keys of a wave at a time
constexpr int kTile = 16;       // queries, or keys, of a tile
constexpr int kHalves = kKeys / kTile;
constexpr int kMaxSplits = 64;
constexpr float kSlack = 8.0f;  // units of log2 that a score may be above the reference

typedef cache::bf16x2 bf16x2;

__device__ __forceinline__ f32x4 mma16(bf16x8 a, bf16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma16(float a, float b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }

// Over the four lanes of a column.
__device__ __forceinline__ float max_column(float v) {
    v = fmaxf(v, __shfl_xor(v, 16));
    return max_halves(v);
}
__device__ __forceinline__ float sum_column(float v) {
    v += __shfl_xor(v, 16);
    return sum_halves(v);
}

// Where 16 keys lie: uniform.
struct Place {
    long long row, scale;  // byte of the first one's row and scales, either pool
    bool held;
};
// Block of 32 keys from k0 on.  The table is read through the scalar cache.
typedef const __attribute__((address_space(4))) int* Table;
__device__ __forceinline__ void find(Place (&at)[kHalves], const Pages& p, int b, int kv, int k0) {
#pragma unroll
    for (int x = 0; x < kHalves; ++x) {
        const int key = k0 + x * kTile, i = min(key >> p.shift, p.table_pages - 1);
        const int page = ((Table)p.table)[(size_t)b * p.table_pages + i];
        at[x].held = (unsigned)page < (unsigned)p.pages;
        const long long block = p.block_at(at[x].held ? page : 0, kv);
        at[x].row = block + (long long)p.slot_of(key) * p.row_bytes;
        at[x].scale = block + p.scales + p.slot_of(key) * p.groups;
    }
}

// Three bf16 parts of 8 fp32 values.
template <int PARTS>
__device__ __forceinline__ void parts_of(const float* x, bf16x8 (&y)[PARTS]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        float rest = x[j];
#pragma unroll
        for (int n = 0; n < PARTS; ++n) {
            y[n][j] = (bf16)rest;
            rest -= (float)y[n][j];
        }
    }
}

// ---------------------------------------------------------------------------
// 32 keys and values on their way, by the kind of pages
// ---------------------------------------------------------------------------
// Values in LDS: rows of DP bf16, a power of two long, chunk c of 16 bytes at c ^ S(row), so
// that the 16 chunks that are written at once and the 8 rows x 32 bytes of a transposing read
// meet different banks.
template <int DP>
struct Values {
    static constexpr int kRowBytes = DP <= 32 ? 64 : DP <= 64 ? 128 : 256;
    static constexpr int kBytes = kKeys * kRowBytes;
    static __device__ __forceinline__ int S(int r) {
        if (DP <= 32) return (r >> 3 & 1) | (r >> 2 & 1) << 1;
        if (DP <= 64) return (r >> 2 & 1) * 5 | (r >> 1 & 1) << 1;
        return (r & 1) * 5 | (r & 2) | (r & 4) << 1;
    }
    static __device__ __forceinline__ int at(int row, int chunk) { return row * kRowBytes + ((chunk ^ S(row)) << 4); }
    // This lane's part of the transposing reads of features 16 d ..: keys 4 h .. 4 h + 3 and 16 more
    static __device__ __forceinline__ bf16x8 columns(const char* t, int d, int lane) {
        typedef __attribute__((address_space(3))) i16x4* LdsPtr;
        const int row = lane >> 2, chunk = 2 * d + (lane >> 1 & 1), byte = (lane & 1) * 8;
        const i16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsPtr)(t + at(row, chunk) + byte));
        const i16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsPtr)(t + at(row + kTile, chunk) + byte));
        const bf16x4 x = __builtin_bit_cast(bf16x4, a), y = __builtin_bit_cast(bf16x4, b);
        return __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
    }
};

template <int DP>
struct Mxfp4 {
    typedef bf16x8 Frag;
    static constexpr int kWaves = 2;  // a SIMD, at least
    static constexpr int kSteps = DP / 32;       // products of a tile of scores
    static constexpr int kGroups = DP / 32;      // scales of a row
    static constexpr int kWords = DP / 32;       // of 8 features: a lane's of a key
    static constexpr int kChunks = (kKeys * kGroups + 63) / 64;  // of 32 values: a lane's
    // a lane has a quarter of a key, features DP / 4 h ..; one scale, or (96) one for each 8 of them
    static constexpr int kScales = DP == 96 ? kWords : 1;
    static constexpr int kLds = Values<DP>::kBytes;
    unsigned k[kHalves][kWords], ks[kHalves][kScales];
    u32x4 v[kChunks];
    unsigned vs[kChunks];

    static __device__ __forceinline__ int feature(int h, int u) { return DP / 4 * h + 8 * u; }
    static __device__ __forceinline__ int chunk(int n, int lane) { return n * 64 + lane; }

    __device__ __forceinline__ void load(const Place (&at)[kHalves], const Pages& p, int lane) {
        const unsigned row = lane & 15, h = lane >> 4;
#pragma unroll
        for (int x = 0; x < kHalves; ++x) {
            __builtin_memcpy(k[x], __builtin_assume_aligned(p.k + at[x].row + (row * (DP / 2) + h * (DP / 8)), DP == 128 ? 16 : DP == 64 ? 8 : 4), DP / 8);
#pragma unroll
            for (int u = 0; u < kScales; ++u)
                ks[x][u] = *reinterpret_cast<const unsigned char*>(p.k + at[x].scale + (row * kGroups + feature(h, u) / 32));
        }
#pragma unroll
        for (int n = 0; n < kChunks; ++n) {
            const int c = min(chunk(n, lane), kKeys * kGroups - 1), key = c / kGroups, g = c % kGroups;
            const bool upper = key >= kTile;
            v[n] = *reinterpret_cast<const u32x4*>(p.v + (upper ? at[1].row : at[0].row) + (unsigned)((key & 15) * (DP / 2) + g * 16));
            vs[n] = *reinterpret_cast<const unsigned char*>(p.v + (upper ? at[1].scale : at[0].scale) + (unsigned)((key & 15) * kGroups + g));
        }
    }
    __device__ __forceinline__ Frag key(int x, int u) const {
        bf16x2 y[4];
        cache::values8(k[x][u], cache::scale_of(ks[x][kScales > 1 ? u : 0]), y);
        return __builtin_bit_cast(Frag, y);
    }
    // keep(key): whether it is one that a query sees
    template <typename Keep>
    __device__ __forceinline__ void store(char* lds, int lane, bool all, const Keep& keep) const {
#pragma unroll
        for (int n = 0; n < kChunks; ++n) {
            const int c = chunk(n, lane), key = c / kGroups, g = c % kGroups;
            if (kKeys * kGroups % 64 && c >= kKeys * kGroups) continue;
            const bool some = all || keep(key);
            const float scale = some ? cache::scale_of(vs[n]) : 1.0f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                bf16x2 y[4];
                cache::values8(some ? v[n][i] : 0u, scale, y);
                *reinterpret_cast<u32x4*>(lds + Values<DP>::at(key, 4 * g + i)) = __builtin_bit_cast(u32x4, y);
            }
        }
    }
};

template <int DP>
struct Bf16 {
    typedef bf16x8 Frag;
    static constexpr int kWaves = 2;
    static constexpr int kSteps = DP / 32;
    static constexpr int kPerRow = DP / 8;
    static constexpr int kChunks = kKeys * kPerRow / 64;
    static constexpr int kLds = Values<DP>::kBytes;
    u32x4 k[kHalves][kSteps], v[kChunks];

    static __device__ __forceinline__ int feature(int h, int u) { return 32 * u + 8 * h; }

    __device__ __forceinline__ void load(const Place (&at)[kHalves], const Pages& p, int lane) {
        const unsigned row = lane & 15, h = lane >> 4, last = p.row_bytes - 16;
#pragma unroll
        for (int x = 0; x < kHalves; ++x)
#pragma unroll
            for (int u = 0; u < kSteps; ++u)  // past the features: some of the row's, which meet zeros
                k[x][u] = *reinterpret_cast<const u32x4*>(p.k + at[x].row + (row * p.row_bytes + min((unsigned)feature(h, u) * 2, last)));
#pragma unroll
        for (int n = 0; n < kChunks; ++n) {
            const int c = n * 64 + lane, key = c / kPerRow;
            v[n] = *reinterpret_cast<const u32x4*>(p.v + (key >= kTile ? at[1].row : at[0].row) +
                ((unsigned)(key & 15) * p.row_bytes + min((unsigned)(c % kPerRow) * 16, last)));
        }
    }
    __device__ __forceinline__ Frag key(int x, int u) const { return __builtin_bit_cast(Frag, k[x][u]); }
    template <typename Keep>
    __device__ __forceinline__ void store(char* lds, int lane, bool all, const Keep& keep) const {
#pragma unroll
        for (int n = 0; n < kChunks; ++n) {
            const int c = n * 64 + lane, key = c / kPerRow;
            *reinterpret_cast<u32x4*>(lds + Values<DP>::at(key, c % kPerRow)) = all || keep(key) ? v[n] : u32x4{0, 0, 0, 0};
        }
    }
};

// fp32 pages: products of 4, a value at a time; a lane's values are features 16 d + (l & 15) of
// the keys 4 h + j, which it reads where they lie.
template <int DP>
struct F32 {
    typedef float Frag;
    static constexpr int kWaves = 1;
    static constexpr int kSteps = DP / 4;
    static constexpr int kLds = 16;
    f32x4 k[kHalves][DP / 16];
    float v[kHalves][4][DP / 16];

    static __device__ __forceinline__ int feature(int h, int u) { return 16 * (u / 4) + 4 * h + u % 4; }

    __device__ __forceinline__ void load(const Place (&at)[kHalves], const Pages& p, int lane) {
        const unsigned row = lane & 15, h = lane >> 4, last = p.row_bytes - 16;
#pragma unroll
        for (int x = 0; x < kHalves; ++x) {
#pragma unroll
            for (int u = 0; u < DP / 16; ++u)
                k[x][u] = *reinterpret_cast<const f32x4*>(p.k + at[x].row + (row * p.row_bytes + min(64 * u + 16 * h, last)));
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int d = 0; d < DP / 16; ++d)
                    v[x][j][d] = *reinterpret_cast<const float*>(p.v + at[x].row + ((4 * h + j) * p.row_bytes + min(64 * d + 4 * row, last + 12)));
        }
    }
    __device__ __forceinline__ Frag key(int x, int u) const { return k[x][u / 4][u % 4]; }
};

// ---------------------------------------------------------------------------
// The kernel
// ---------------------------------------------------------------------------
__device__ __forceinline__ void hand(float* p, float x, float y) {
    nnk::rec_store(reinterpret_cast<unsigned long long*>(p), (unsigned long long)__builtin_bit_cast(unsigned, y) << 32 |
            __builtin_bit_cast(unsigned, x));
}
__device__ __forceinline__ float2 taken(const float* p) {
    const unsigned long long v = nnk::rec_load(reinterpret_cast<const unsigned long long*>(p));
    return make_float2(__builtin_bit_cast(float, (unsigned)v), __builtin_bit_cast(float, (unsigned)(v >> 32)));
}

struct Few {
    unsigned* tickets;
    float* partial;  // [units, splits, rows, DP + 2]: outputs, then reference (units of log2) and sum
    int tiles, splits, each;  // tiles of a key head's queries; workgroups of a unit; their keys
};

template <typename T, template <int> class PAGES, int DP, int NT>
__global__ __launch_bounds__(kTpb, PAGES<DP>::kWaves) void cache_few_kernel(Args a, Pages p, Few f) {
    using E = PAGES<DP>;
    constexpr bool kWide = std::is_same_v<typename E::Frag, bf16x8>;     // bf16 products
    constexpr int kParts = kWide && sizeof(T) == 4 ? 3 : 1;              // of a query or probability
    constexpr int kRowsEach = kTile * NT;
    constexpr int kRow = DP + 4;  // floats of an output row in LDS
    constexpr int kShared = E::kLds > kTile * kRow * 4 ? E::kLds : kTile * kRow * 4;
    __shared__ __attribute__((aligned(16))) char lds[kWaves][kShared];
    __shared__ float m_lds[kWaves][kRowsEach], l_lds[kWaves][kRowsEach];
    __shared__ float weight[kRowsEach][kMaxSplits];
    __shared__ float total[kRowsEach];
    __shared__ int last_one;

    const int lane = threadIdx.x & 63, h = lane >> 4, col = lane & 15, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int split = blockIdx.x % f.splits, unit = blockIdx.x / f.splits;
    const int tile = unit % f.tiles, kv = unit / f.tiles % a.kv_heads, b = unit / f.tiles / a.kv_heads;
    const int rows = min(kRowsEach, a.len_q * a.group - tile * kRowsEach);
    const int keys = p.pages ? keys_of(a, b) : 0, start = start_of(a, b);
    const int most = limit_of(a, b, keys, start + (tile * kRowsEach + rows - 1) / a.group);
    const int active = max(1, (most + f.each - 1) / f.each);  // workgroups of the unit that have keys
    if (split >= active) return;

    int pos[NT], limit[NT], head[NT], least = INT32_MAX;
    typename E::Frag qf[NT][kParts][E::kSteps];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const bool in = t * kTile + col < rows;
        const int row = tile * kRowsEach + (in ? t * kTile + col : 0), i = row / a.group;
        head[t] = kv * a.group + row - i * a.group;
        pos[t] = start + i;
        limit[t] = in ? limit_of(a, b, keys, pos[t]) : 0;
        if (in) least = min(least, limit[t]);
        const T* q = (const T*)a.q + b * a.qs[0] + i * a.qs[1] + head[t] * a.qs[2];
        if constexpr (kWide) {
#pragma unroll
            for (int u = 0; u < E::kSteps; ++u) {
                const int d0 = E::feature(h, u);
                if constexpr (kParts == 1) {
                    qf[t][0][u] = a.vec ? load_frag<bf16, true>((const bf16*)q, d0, a.dim) : load_frag<bf16, false>((const bf16*)q, d0, a.dim);
                } else {
                    float x[8];
                    bf16x8 y[kParts];
#pragma unroll
                    for (int j = 0; j < 8; ++j) x[j] = d0 + j < a.dim ? (float)q[d0 + j] : 0.0f;
                    parts_of<kParts>(x, y);
#pragma unroll
                    for (int n = 0; n < kParts; ++n) qf[t][n][u] = y[n];
                }
            }
        } else {
#pragma unroll
            for (int u = 0; u < E::kSteps; ++u) qf[t][0][u] = E::feature(h, u) < a.dim ? (float)q[E::feature(h, u)] : 0.0f;
        }
    }
#pragma unroll
    for (int m = 1; m < kTile; m <<= 1) least = min(least, __shfl_xor(least, m));
    least = __builtin_amdgcn_readfirstlane(least);

    const auto bias_of = [&](int rel, int of_head) {
        const int i = min(max(rel, -a.max_distance), a.max_distance) + a.max_distance;
        return a.bias[(size_t)min(max(a.bucket[i], 0), a.buckets - 1) * a.heads + of_head] * kLog2e;
    };
    float far[NT];  // bias of keys max_distance or more before the query
#pragma unroll
    for (int t = 0; t < NT; ++t) far[t] = a.buckets ? bias_of(-a.max_distance, head[t]) : 0.0f;
    const bool plain = a.c2 == 0.0f && !a.buckets;
    const float unit_of = plain ? a.c1 : 1.0f;  // what a score is multiplied with in the exponent

    f32x4 o[NT][DP / 16];
    float m[NT], l[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
#pragma unroll
        for (int d = 0; d < DP / 16; ++d) o[t][d] = f32x4{0, 0, 0, 0};
        m[t] = -INFINITY;
        l[t] = 0.0f;
    }

    // this wave's blocks of the workgroup's keys
    const int end = min(most, (split + 1) * f.each);
    E e;
    Place at[kHalves], next[kHalves];
    int k0 = split * f.each + wave * kKeys;
    if (k0 < end) {
        find(at, p, b, kv, k0);
        e.load(at, p, lane);
        find(next, p, b, kv, k0 + kWaves * kKeys);
    }
    for (; k0 < end; k0 += kWaves * kKeys) {
        const bool held = at[0].held && at[1].held, all = held && k0 + kKeys <= keys;
        const bool held0 = at[0].held, held1 = at[1].held;
        [[maybe_unused]] char* values = lds[wave];
        f32x4 s[NT][kHalves];
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int x = 0; x < kHalves; ++x) s[t][x] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int x = 0; x < kHalves; ++x)
#pragma unroll
            for (int u = 0; u < E::kSteps; ++u) {
                const typename E::Frag y = e.key(x, u);
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int n = kParts - 1; n >= 0; --n) s[t][x] = mma16(y, qf[t][n][u], s[t][x]);
            }
        const auto keep = [&](int key) { return k0 + key < keys && (key < kTile ? held0 : held1); };
        [[maybe_unused]] float v[kWide ? 1 : kHalves][4][kWide ? 1 : DP / 16];
        if constexpr (kWide) {
            e.store(values, lane, all, keep);
        } else {
#pragma unroll
            for (int x = 0; x < kHalves; ++x)
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int d = 0; d < DP / 16; ++d) v[x][j][d] = all || keep(x * kTile + 4 * h + j) ? e.v[x][j][d] : 0.0f;
        }
        // the next block's, while this one's scores become shares
        at[0] = next[0];
        at[1] = next[1];
        if (k0 + kWaves * kKeys < end) {
            e.load(at, p, lane);
            find(next, p, b, kv, k0 + 2 * kWaves * kKeys);
        }

#pragma unroll
        for (int t = 0; t < NT; ++t) {
            if (a.c2 != 0.0f) {
                float top = 0.0f;
#pragma unroll
                for (int x = 0; x < kHalves; ++x)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        s[t][x][j] *= a.c1;
                        top = fmaxf(top, fabsf(s[t][x][j]));
                    }
                if (__all(top < kSeriesEnd)) {
#pragma unroll
                    for (int x = 0; x < kHalves; ++x)
#pragma unroll
                        for (int j = 0; j < 4; ++j) s[t][x][j] = tanh_series(s[t][x][j]) * a.c2;
                } else {
#pragma unroll
                    for (int x = 0; x < kHalves; ++x)
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const float y = s[t][x][j], r = __builtin_amdgcn_rcpf(exp2_fast(fabsf(y) * (2.0f * kLog2e)) + 1.0f);
                            s[t][x][j] = (fabsf(y) < kSeriesEnd ? tanh_series(y) : copysignf(fmaf(-2.0f, r, 1.0f), y)) * a.c2;
                        }
                }
            }
            if (a.buckets) {
                const float c = a.c2 != 0.0f ? 1.0f : a.c1;
                if (__all(k0 + kKeys - 1 - pos[t] <= -a.max_distance)) {
#pragma unroll
                    for (int x = 0; x < kHalves; ++x)
#pragma unroll
                        for (int j = 0; j < 4; ++j) s[t][x][j] = s[t][x][j] * c + far[t];
                } else {
#pragma unroll
                    for (int x = 0; x < kHalves; ++x)
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            s[t][x][j] = s[t][x][j] * c + bias_of(k0 + x * kTile + 4 * h + j - pos[t], head[t]);
                }
            }
            if (!held || k0 + kKeys > least) {
#pragma unroll
                for (int x = 0; x < kHalves; ++x)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        s[t][x][j] = k0 + x * kTile + 4 * h + j < limit[t] && (x ? held1 : held0) ? s[t][x][j] : -INFINITY;
            }
            float top = -INFINITY;
#pragma unroll
            for (int x = 0; x < kHalves; ++x)
#pragma unroll
                for (int j = 0; j < 4; ++j) top = fmaxf(top, s[t][x][j]);
            top = max_column(top) * unit_of;
            // the reference follows the largest score when that has left it behind
            if (__any(top > m[t] + kSlack)) {
                const float to = fmaxf(m[t], top), g = exp2_fast(m[t] - (to == -INFINITY ? 0.0f : to));
                l[t] *= g;
#pragma unroll
                for (int d = 0; d < DP / 16; ++d) o[t][d] *= g;
                m[t] = to;
            }
            const float base = m[t] == -INFINITY ? 0.0f : m[t];
#pragma unroll
            for (int x = 0; x < kHalves; ++x)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    s[t][x][j] = exp2_fast(fmaf(s[t][x][j], unit_of, -base));
                    l[t] += s[t][x][j];
                }
        }
        if constexpr (kWide) {
            bf16x8 shares[NT][kParts];
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                float x[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] = s[t][j / 4][j % 4];
                parts_of<kParts>(x, shares[t]);
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int d = 0; d < DP / 16; ++d) {
                const bf16x8 y = Values<DP>::columns(values, d, lane);
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int n = kParts - 1; n >= 0; --n) o[t][d] = mma16(y, shares[t][n], o[t][d]);
            }
            // the next values are written over these when they have been read
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
        } else {
#pragma unroll
            for (int x = 0; x < kHalves; ++x)
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int d = 0; d < DP / 16; ++d)
#pragma unroll
                        for (int t = 0; t < NT; ++t) o[t][d] = mma16(v[x][j][d], s[t][x][j], o[t][d]);
        }
    }

    // the waves of the workgroup, a tile of queries at a time
    constexpr int kQuads = DP / 4;  // 4 features a thread
    const size_t step = kRowsEach * (DP + 2);
    float* to = f.partial + ((size_t)unit * f.splits + split) * step;
    const auto finish = [&](int r, int d, float4 x, float ref, float sum) {
        const int n = tile * kRowsEach + r, qi = n / a.group, hd = kv * a.group + n - qi * a.group;
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        T* out = (T*)a.out + b * a.os[0] + qi * a.os[1] + hd * a.os[2];
        if (a.vec) store4<T, true>(out, d, a.dim, x.x * inv, x.y * inv, x.z * inv, x.w * inv);
        else store4<T, false>(out, d, a.dim, x.x * inv, x.y * inv, x.z * inv, x.w * inv);
        if (d == 0)
            a.lse[((size_t)b * a.heads + hd) * a.len_q + qi] = sum == 0.0f ? -INFINITY : (ref + log2f(sum)) * kLn2;
    };
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        if (t * kTile >= rows) break;
        const float sum = sum_column(l[t]);
        if (t) __syncthreads();
        float* mine = reinterpret_cast<float*>(lds[wave]) + col * kRow;
#pragma unroll
        for (int d = 0; d < DP / 16; ++d) *reinterpret_cast<f32x4*>(mine + 16 * d + 4 * h) = o[t][d];
        if (h == 0) {
            m_lds[wave][t * kTile + col] = m[t];
            l_lds[wave][t * kTile + col] = sum;
        }
        __syncthreads();
        for (int n = threadIdx.x; n < min(kTile, rows - t * kTile) * kQuads; n += kTpb) {
            const int c = n / kQuads, r = t * kTile + c, d = n % kQuads * 4;
            float ref = m_lds[0][r];
#pragma unroll
            for (int w = 1; w < kWaves; ++w) ref = fmaxf(ref, m_lds[w][r]);
            float all = 0.0f;
            float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                const float g = ref == -INFINITY ? 0.0f : exp2_fast(m_lds[w][r] - ref);
                const float4 y = nnk::ld4(reinterpret_cast<const float*>(lds[w]) + c * kRow + d);
                all = fmaf(l_lds[w][r], g, all);
                x.x = fmaf(y.x, g, x.x);
                x.y = fmaf(y.y, g, x.y);
                x.z = fmaf(y.z, g, x.z);
                x.w = fmaf(y.w, g, x.w);
            }
            if (active == 1) {
                finish(r, d, x, ref, all);
            } else {
                float* q = to + r * (DP + 2);
                hand(q + d, x.x, x.y);
                hand(q + d + 2, x.z, x.w);
                if (d == 0) hand(q + DP, ref, all);
            }
        }
    }
    if (active == 1) return;

    // the workgroups of the unit
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // handed over
    __syncthreads();
    if (threadIdx.x == 0)
        last_one = __hip_atomic_fetch_add(f.tickets + unit, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) ==
            (unsigned)(active - 1);
    __syncthreads();
    if (!last_one) return;
    const float* from = f.partial + (size_t)unit * f.splits * step;
    for (int r = wave; r < rows; r += kWaves) {  // a lane a split: their shares of the row
        float ms = -INFINITY, ls = 0.0f;
        if (lane < active) {
            const float2 y = taken(from + lane * step + r * (DP + 2) + DP);
            ms = y.x;
            ls = y.y;
        }
        float ref = ms;
#pragma unroll
        for (int x = 1; x < 64; x <<= 1) ref = fmaxf(ref, __shfl_xor(ref, x));
        const float g = ref == -INFINITY ? 0.0f : exp2_fast(ms - ref);
        weight[r][lane] = g;
        const float sum = nnk::wave_sum(ls * g);
        if (lane == 0) {
            m_lds[0][r] = ref;
            total[r] = sum;
        }
    }
    __syncthreads();
    for (int n = threadIdx.x; n < rows * kQuads; n += kTpb) {
        const int r = n / kQuads, d = n % kQuads * 4;
        const float* q = from + r * (DP + 2) + d;
        float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
        for (int sp = 0; sp < active; ++sp) {
            const float g = weight[r][sp];
            const float2 y = taken(q + sp * step), z = taken(q + sp * step + 2);
            x.x = fmaf(y.x, g, x.x);
            x.y = fmaf(y.y, g, x.y);
            x.z = fmaf(z.x, g, x.z);
            x.w = fmaf(z.y, g, x.w);
        }
        finish(r, d, x, m_lds[0][r], total[r]);
    }
    if (threadIdx.x == 0) __hip_atomic_store(f.tickets + unit, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// Tiles of queries, and how the keys are split: enough workgroups to fill the card several
// times over (requests' lengths differ, and those without keys of theirs end at once), a block
// a wave at least.
struct Plan {
    long long units;
    int tiles, rows, splits, each;
};
Plan plan_of(const NnAttention* a) {
    Plan p;
    const long long rows = (long long)a->len_q * (a->heads / a->kv_heads);
    p.rows = rows <= kTile ? kTile : 2 * kTile;
    p.tiles = (int)((rows + p.rows - 1) / p.rows);
    p.units = (long long)a->batch * a->kv_heads * p.tiles;
    const int step = kWaves * kKeys, steps = std::max(1, (a->len_k + step - 1) / step);
    const long long want = p.units >= kTicketWords ? 1 : std::min<long long>(kMaxSplits, (2 * kTicketWords + p.units - 1) / p.units);
    const int n = (int)((steps + want - 1) / want);
    p.each = n * step;
    p.splits = (steps + n - 1) / n;
    return p;
}
int padded(int dim) { return (dim + 31) / 32 * 32; }

template <typename T, template <int> class PAGES, int DP>
void launch(const Args& a, const Pages& p, const Plan& plan, float* ws, hipStream_t s, const char* what) {
    const Few f = {reinterpret_cast<unsigned*>(ws), ws + kTicketWords, plan.tiles, plan.splits, plan.each};
    const unsigned blocks = (unsigned)(plan.units * plan.splits);
    if (plan.rows == kTile) cache_few_kernel<T, PAGES, DP, 1><<<blocks, kTpb, 0, s>>>(a, p, f);
    else cache_few_kernel<T, PAGES, DP, 2><<<blocks, kTpb, 0, s>>>(a, p, f);
    nnk_after_launch(what, s);
}
template <typename T, template <int> class PAGES>
void by_dim(const Args& a, const Pages& p, const Plan& plan, float* ws, hipStream_t s, const char* what) {
    switch (padded(a.dim)) {
    case 32: return launch<T, PAGES, 32>(a, p, plan, ws, s, what);
    case 64: return launch<T, PAGES, 64>(a, p, plan, ws, s, what);
    case 96: return launch<T, PAGES, 96>(a, p, plan, ws, s, what);
    default: return launch<T, PAGES, 128>(a, p, plan, ws, s, what);
    }
}

}  // namespace

// Floats that one call takes, its tickets among them.
size_t nnk_cache_few_floats(const NnAttention* a) {
    if (!a->batch || !a->len_q) return 0;
    const Plan p = plan_of(a);
    return p.splits == 1 ? 0 : kTicketWords + (size_t)p.units * p.splits * p.rows * (padded(a->head_dim) + 2);
}
void nnk_cache_few(const Args& a, const Pages& p, const NnAttention* d, float* ws, hipStream_t s, const char* what) {
    const Plan plan = plan_of(d);
    NNK_REQUIRE(plan.units * plan.splits < (1LL << 32) / kTpb, what, "%s: too many rows", what);
    if (d->dtype == NN_BF16) {
        if (p.groups) by_dim<bf16, Mxfp4>(a, p, plan, ws, s, what);
        else by_dim<bf16, Bf16>(a, p, plan, ws, s, what);
    } else {
        if (p.groups) by_dim<float, Mxfp4>(a, p, plan, ws, s, what);
        else by_dim<float, F32>(a, p, plan, ws, s, what);
    }
}
size_t nnk_cache_few_most(const NnAttention* a) {
    const long long steps = ((long long)a->len_k + kWaves * kKeys - 1) / (kWaves * kKeys);
    if (steps < 2) return 0;
    const Plan p = plan_of(a);
    const long long units = std::min<long long>(kTicketWords - 1, p.units);
    const long long groups = std::min(units * std::min<long long>(kMaxSplits, steps), units + 2 * kTicketWords - 1);
    return kTicketWords + (size_t)groups * p.rows * (padded(a->head_dim) + 2);
}
