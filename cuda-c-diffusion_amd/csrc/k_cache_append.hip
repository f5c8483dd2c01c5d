// k_cache_append.hip -- rows of a projection: queries turned, keys turned and values written
// to the pages of their requests, in the tensors' type or in 4 bits.
//
// A key row x of head_dim features:  y = x [rsqrt(mean(x^2) + eps) w],  its pairs turned by
// their angles;  in 4 bits then, for 32 features at a time, the least exponent e with
// max|y| <= 7 2^e and the 8 sizes' nearest to |y| 2^-e.  Every row is read once and written
// once: memory bounds long prompts, latency a decoding step.  A row belongs to the G lanes of a
// group, 16 bytes a lane, so that sums and maxima are cross-lane steps in the group; a pair's
// other member comes from the group's row in LDS.  A workgroup takes the queries, the keys or the
// values of some tokens, whose places and sines it has once.  Its groups take heads that lie
// together and go from token to token, the next two rows on their way (a group a
// token, 12 KB apart, was two to three times as long: the groups of all workgroups met on a few
// of the memory's channels).  Few tokens are one a workgroup or less, a row a group.
//
// Keys for 4 bits are formed in 64 bits, as a code is a choice: with fp32 sums the order of
// the additions would decide it for some values in 10^5, and with it half a step of the value.
//
// Measured: 8192 tokens, 32 + 8 + 8 heads of 128, bf16 into 4 bits 44 us (3.9 TB/s; vector instructions
// half of the SIMDs' cycles); 2355 rows, 39 of them no tokens, 16 + 16 + 16 heads of 72, fp32 into
// plain pages 23 us (2.8 TB/s); four tokens 6.7 us.
#include "cache_common.h"

#include <algorithm>
#include <type_traits>

namespace {
using namespace cache;

constexpr int kTpb = 256;
constexpr int kTableBytes = 16384;  // sines and cosines of a workgroup's tokens
constexpr int kMostTokensEach = 16;  // lanes of a wave at most

struct Append {
    const void *q, *k, *v;
    void* q_out;
    Pages pages;
    long long qs[2], ks[2], vs[2], qos[2];
    const float *q_weight, *k_weight;
    const int *pos, *request, *place;
    const double* freq;
    int tokens, heads, kv_heads, dim, half, axes, per_axis, interleaved, norm;
    int tokens_each;       // tokens of a workgroup
    int q_parts, kv_parts; // workgroups that share their queries, and their keys, and their values
    float eps;
    bool vec;
};

// floor(log2 |x|), and whether the fraction is past 1.75
__device__ __forceinline__ int exponent_of(float x, bool& past) {
    const unsigned u = __builtin_bit_cast(unsigned, x);
    past = (u & 0x7fffffu) > 0x600000u;
    return (int)(u >> 23) - 127;
}
__device__ __forceinline__ int exponent_of(double x, bool& past) {
    const unsigned long long u = __builtin_bit_cast(unsigned long long, x);
    past = (u & 0xfffffffffffffull) > 0xc000000000000ull;
    return (int)(u >> 52) - 1023;
}
// Codes of two values: the conversion rounds to the nearest, half way to even, and ends at 6.
__device__ __forceinline__ unsigned codes_of(float x, float y, int e) {
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, x, y, __builtin_bit_cast(float, (unsigned)(e + 127) << 23), 0);
}
// It takes fp32, to which a 64-bit value may round onto a border that it is beside.  So |x| 2^-e in
// steps of 2^-20, cut off, and a last bit for what was: the same choice, as borders are whole steps.
__device__ __forceinline__ float beside(double x, double down) {
    const double y = fmin(fabs(x) * down, 0x1p23);
    const unsigned u = (unsigned)y;
    const float f = (float)(2 * u + ((double)u != y ? 1u : 0u));
    return x < 0 ? -f : f;
}
constexpr int kBeside = -21;  // exponent of its last bit
__device__ __forceinline__ unsigned codes_of(double x, double y, int e) {
    const double down = __builtin_bit_cast(double, (unsigned long long)(20 - e + 1023) << 52);
    return codes_of(beside(x, down), beside(y, down), -kBeside);
}
template <typename A>
constexpr int kTop = sizeof(A) == 8 ? 1024 : 128;  // exponent of infinity

template <typename T, int G>
struct Row {
    static constexpr int CE = 16 / (int)sizeof(T);
    static constexpr int kGroups = kTpb / G;

    static __device__ __forceinline__ u32x4 load(const T* row, int d0, const Append& a) {
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
    template <typename A>
    static __device__ __forceinline__ void values(A* x, const u32x4& v) {
        T e[CE];
        __builtin_memcpy(e, &v, 16);
#pragma unroll
        for (int j = 0; j < CE; ++j) x[j] = (A)(float)e[j];
    }
    // 16 bytes at a time, with zeros behind the features, or (!whole) what is one alone
    template <typename A>
    static __device__ __forceinline__ void store(T* row, int d0, int dim, bool whole, const A* x) {
        T e[CE];
#pragma unroll
        for (int j = 0; j < CE; ++j) e[j] = (T)(float)x[j];
        if (whole) {
            if (d0 < dim) __builtin_memcpy(__builtin_assume_aligned(row + d0, 16), e, 16);
        } else {
#pragma unroll
            for (int j = 0; j < CE; ++j)
                if (d0 + j < dim) row[d0 + j] = e[j];
        }
    }
    template <typename A>
    static __device__ __forceinline__ A group_sum(A v) {
#pragma unroll
        for (int m = 1; m < G; m <<= 1) v += __shfl_xor(v, m);
        return v;
    }
    template <typename A>
    static __device__ __forceinline__ void normalise(A* x, const float* w, const Append& a) {
        A ss = 0;
#pragma unroll
        for (int j = 0; j < CE; ++j) ss = fma(x[j], x[j], ss);
        ss = group_sum(ss) / (A)a.dim + (A)a.eps;
        const A rstd = sizeof(A) == 8 ? (A)(1.0 / sqrt((double)ss)) : (A)rsqrtf((float)ss);
#pragma unroll
        for (int j = 0; j < CE; ++j) x[j] = x[j] * rstd * (A)w[j];
    }
    // A turn of pairs that lie whole chunks of a lane apart: out = x cos + other sin, with the sine's
    // sign in it.  The table has a token's cosines by feature, then its sines, both in an order
    // of 16-byte accesses without bank conflicts.
    static constexpr int kFeatures = G * CE;
    template <typename A>
    static __device__ __forceinline__ int place(int d) {
        constexpr int V = 16 / (int)sizeof(A);
        return d % CE / V * (G * V) + d / CE * V + d % V;
    }
    // The lane of the other members, or -1: this one's features are not turned.
    static __device__ __forceinline__ int other_lane(int d0, const Append& a) {
        const int c = d0 / CE, hc = a.half / CE;
        return c >= 2 * hc ? -1 : c < hc ? c + hc : c - hc;
    }
    // `row`: the group's values in LDS, kFeatures of them
    template <typename A>
    static __device__ __forceinline__ void turn(A* x, int d0, int other, A* row, const A* table) {
        constexpr int V = 16 / (int)sizeof(A);  // values of an access
        typedef A Vec __attribute__((ext_vector_type(V)));
        const int c = d0 / CE;
        // What is not turned meets its cosine, 1, times its sine, -0, and so stays as it is, infinities and
        // the signs of zeros too.
        const A* others = other >= 0 ? row + V * other : table + V * c;
        // the group's lanes are in one wave, whose LDS accesses are in order
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int j = 0; j < CE; j += V) {
            Vec y;
#pragma unroll
            for (int i = 0; i < V; ++i) y[i] = x[j + i];
            *reinterpret_cast<Vec*>(row + j * G + V * c) = y;
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int j = 0; j < CE; j += V) {
            const Vec y = *reinterpret_cast<const Vec*>(others + j * G);
            const Vec cos = *reinterpret_cast<const Vec*>(table + j * G + V * c);
            const Vec sin = *reinterpret_cast<const Vec*>(table + kFeatures + j * G + V * c);
#pragma unroll
            for (int i = 0; i < V; ++i) x[j + i] = fma(x[j + i], cos[i], y[i] * sin[i]);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
    // Any other turn.
    template <typename A, typename CS>
    static __device__ __forceinline__ void turn(A* x, int d0, A* row, const CS* cs, const Append& a) {
        if (a.interleaved) {
#pragma unroll
            for (int j = 0; j < CE; j += 2) {
                const int p = (d0 + j) / 2;
                if (p >= a.half) continue;
                const A c = (A)cs[p].x, s = (A)cs[p].y, u = x[j], v = x[j + 1];
                x[j] = u * c - v * s;
                x[j + 1] = u * s + v * c;
            }
            return;
        }
        if (!a.half) return;
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int j = 0; j < CE; ++j) row[d0 + j] = x[j];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int j = 0; j < CE; ++j) {
            const int d = d0 + j;
            if (d >= 2 * a.half) continue;
            const bool first = d < a.half;
            const auto t = cs[first ? d : d - a.half];
            const A other = row[first ? d + a.half : d - a.half];
            x[j] = first ? x[j] * (A)t.x - other * (A)t.y : x[j] * (A)t.x + other * (A)t.y;
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }

    // The lane's features in 4 bits; `block`: the head's in the page
    template <typename A>
    static __device__ __forceinline__ void pack(char* block, int slot, int d0, const A* x, const Pages& p) {
        A most = 0;
#pragma unroll
        for (int j = 0; j < CE; ++j) {
            const A y = fabs(x[j]);
            most = fmax(most, y < (A)INFINITY ? y : (A)INFINITY);  // NaN: infinity
        }
        constexpr int kLanes = kGroup / CE < G ? kGroup / CE : G;  // of a scale
#pragma unroll
        for (int m = 1; m < kLanes; m <<= 1) most = fmax(most, __shfl_xor(most, m));
        bool past;
        int e = exponent_of(most, past);
        const bool none = e == kTop<A>;
        e = min(max(e - (past ? 1 : 2), -120), 125);
        unsigned code = 0;
#pragma unroll
        for (int j = 0; j < CE; j += 2) code |= codes_of(x[j], x[j + 1], e) << (4 * j);
        if (d0 >= p.groups * kGroup) return;
        char* to = block + slot * p.row_bytes + d0 / 2;
        if constexpr (CE == 8) *reinterpret_cast<unsigned*>(to) = code;
        else *reinterpret_cast<unsigned short*>(to) = (unsigned short)code;
        if (d0 % kGroup == 0)
            *reinterpret_cast<unsigned char*>(block + p.scales + slot * p.groups + d0 / kGroup) = (unsigned char)(none ? 255 : e + 127);
    }
};

// Cosine and sine of an angle in turns, formed in 64 bits.  fp32: reduced there to an eighth of a
// turn either way, so that what is left is rounded and the small one of the two keeps its digits.
__device__ __forceinline__ void cos_sin(double turns, double& c, double& s) {
    turns -= rint(turns);
    sincospi(2.0 * turns, &s, &c);
}
__device__ __forceinline__ void cos_sin(double turns, float& c, float& s) {
    turns -= rint(turns);
    const double quarters = rint(4.0 * turns);
    const int q = (int)quarters;
    float u, v;
    sincospif(0.5f * (float)(4.0 * turns - quarters), &u, &v);
    const float x = q & 1 ? u : v, y = q & 1 ? v : u;
    c = (q + 1) & 2 ? -x : x;
    s = q & 2 ? -y : y;
}
template <typename A>
struct Pair {
    A x, y;  // cosine, sine
};
// Of each pair of `count` tokens into the table, for one turn or the other.
template <typename R, typename A, bool CHUNKS>
__device__ __forceinline__ void angles(A* table, const Append& a, int token0, int count) {
    const int each = CHUNKS ? R::kFeatures - a.half : a.half;  // with the features that are not turned
    for (int i = threadIdx.x; i < count * each; i += kTpb) {
        const int t = i / each, p = i - t * each;
        A c = 1, s = (A)-0.0;
        if (p < a.half) {
            const double angle = (double)a.pos[(size_t)(token0 + t) * a.axes + p / a.per_axis] * a.freq[p];
            cos_sin(angle * 0.15915494309189533577, c, s);
        }
        if constexpr (CHUNKS) {
            A* mine = table + t * 2 * R::kFeatures;
            const int second = R::template place<A>(p + a.half);
            mine[second] = c;
            mine[R::kFeatures + second] = s;
            if (p < a.half) {
                const int first = R::template place<A>(p);
                mine[first] = c;
                mine[R::kFeatures + first] = -s;
            }
        } else {
            reinterpret_cast<Pair<A>*>(table)[t * a.half + p] = {c, s};
        }
    }
}

enum { kQueries, kKeyRows, kValueRows };

// CHUNKS: pairs lie whole chunks of a lane apart
template <typename T, int G, bool FP4, bool CHUNKS>
__global__ __launch_bounds__(kTpb, 4) void cache_append_kernel(Append a) {
    using R = Row<T, G>;
    using KeyType = std::conditional_t<FP4, double, float>;
    constexpr int CE = R::CE, kGroups = R::kGroups;
    __shared__ __attribute__((aligned(16))) char tables[kTableBytes];
    __shared__ __attribute__((aligned(16))) KeyType lds[kGroups][R::kFeatures];
    __shared__ long long blocks[kMostTokensEach];  // a token's page, as its first head's byte, or -1
    __shared__ int places[kMostTokensEach];
    const int group = threadIdx.x / G, d0 = (threadIdx.x % G) * CE;
    const int parts = a.q_parts + 2 * a.kv_parts, part = blockIdx.x % parts;
    const int token0 = blockIdx.x / parts * a.tokens_each, tokens = min(a.tokens_each, a.tokens - token0);

    const auto rows_of = [&](auto kind_, int head0, int head1) {
        constexpr int kind = decltype(kind_)::value;
        using A = std::conditional_t<kind == kKeyRows, KeyType, float>;
        A* table = reinterpret_cast<A*>(tables);
        const int other = R::other_lane(d0, a);
        const int heads = min(head1 - head0, kGroups), strands = heads > 0 ? kGroups / heads : 0;
        const int strand = heads > 0 ? group / heads : 0, first = group - strand * heads;  // a token's groups, and tokens at a time
        const T* from = (const T*)(kind == kQueries ? a.q : kind == kKeyRows ? a.k : a.v);
        const long long by_token = kind == kQueries ? a.qs[0] : kind == kKeyRows ? a.ks[0] : a.vs[0];
        const long long by_head = kind == kQueries ? a.qs[1] : kind == kKeyRows ? a.ks[1] : a.vs[1];
        const float* weight = kind == kQueries ? a.q_weight : a.k_weight;
        float w[CE];
        if (kind != kValueRows) {
#pragma unroll
            for (int j = 0; j < CE; ++j) w[j] = weight && d0 + j < a.dim ? weight[d0 + j] : 1.0f;
        }
        for (int head = head0 + first; head0 < head1; head += heads) {
            const bool in = strand < strands && head < head1;
            const T* next_row = from + (token0 + strand) * by_token + head * by_head;
            const long long on = strands * by_token;
            u32x4 next[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
            if (in && strand < tokens) next[0] = R::load(next_row, d0, a);
            if (in && strand + strands < tokens) next[1] = R::load(next_row + on, d0, a);
            next_row += 2 * on;
            if (head == head0 + first) {  // once, the first rows on their way
                if (const int t = (int)threadIdx.x - (kTpb - 64); t >= 0 && t < tokens) {  // a wave without the first sines
                    const int place = a.place[token0 + t];
                    const int page = place < 0 ? -1 : a.pages.page_of(a.request ? a.request[token0 + t] : token0 + t, place);
                    places[t] = place;
                    blocks[t] = page < 0 ? -1 : a.pages.block_at(page, 0);
                }
                if (kind != kValueRows) angles<R, A, CHUNKS>(table, a, token0, tokens);
                __syncthreads();
            }
            if (in)
                for (int t = strand; t < tokens; t += strands) {
                    const u32x4 v = next[0];
                    next[0] = next[1];
                    if (t + 2 * strands < tokens) next[1] = R::load(next_row, d0, a);
                    next_row += on;
                    const int place = places[t];
                    if (place < 0 || (kind != kQueries && blocks[t] < 0)) continue;
                    A x[CE];
                    R::values(x, v);
                    if constexpr (kind != kValueRows) {
                        if (a.norm) R::normalise(x, w, a);
                        A* row = reinterpret_cast<A*>(lds[group]);
                        if constexpr (CHUNKS) R::turn(x, d0, other, row, table + t * 2 * R::kFeatures);
                        else R::turn(x, d0, row, reinterpret_cast<const Pair<A>*>(table) + t * a.half, a);
                    }
                    if constexpr (kind == kQueries) {
                        R::store((T*)a.q_out + (token0 + t) * a.qos[0] + head * a.qos[1], d0, a.dim, a.vec, x);
                    } else {
                        char* block = (kind == kKeyRows ? a.pages.k : a.pages.v) + blocks[t] + (long long)head * a.pages.block_bytes;
                        const int slot = a.pages.slot_of(place);
                        if constexpr (FP4) R::pack(block, slot, d0, x, a.pages);
                        else R::store((T*)(block + slot * a.pages.row_bytes), d0, a.dim, true, x);
                    }
                }
            if (head - first + heads >= head1) break;
        }
    };
    using Queries = std::integral_constant<int, kQueries>;
    using Keys = std::integral_constant<int, kKeyRows>;
    using Values = std::integral_constant<int, kValueRows>;
    if (part < a.q_parts) {
        const int each = (a.heads + a.q_parts - 1) / a.q_parts;
        rows_of(Queries{}, part * each, min((part + 1) * each, a.heads));
    } else {
        const int i = (part - a.q_parts) % a.kv_parts, each = (a.kv_heads + a.kv_parts - 1) / a.kv_parts;
        if (part < a.q_parts + a.kv_parts) rows_of(Keys{}, i * each, min((i + 1) * each, a.kv_heads));
        else rows_of(Values{}, i * each, min((i + 1) * each, a.kv_heads));
    }
}

// Few tokens: one each, their rows shared by workgroups of one pass.  Many: as many as leave four
// workgroups of each kind a CU, as far as their sines fit.
constexpr int kFewTokens = 1024;
template <typename T, int G>
void launch(Append& p, hipStream_t s, const char* what) {
    constexpr int groups = Row<T, G>::kGroups, CE = Row<T, G>::CE;
    const bool chunks = !p.interleaved && p.half > 0 && p.half % CE == 0;
    const int table = (p.pages.groups ? 16 : 8) * (chunks ? G * CE : std::max(1, p.half));  // bytes of a token
    p.tokens_each = std::max(1, std::min({kTableBytes / table, kMostTokensEach, p.tokens / 512}));
    const bool few = p.tokens < kFewTokens;
    p.q_parts = few ? (p.heads + groups - 1) / groups : p.heads > 0;
    p.kv_parts = few ? (p.kv_heads + groups - 1) / groups : 1;
    const long long parts = p.q_parts + 2 * p.kv_parts;
    const long long blocks = ((long long)p.tokens + p.tokens_each - 1) / p.tokens_each * parts;
    NNK_REQUIRE(blocks < (1LL << 32) / kTpb, what, "%s: too many rows", what);  // threads of a launch
    const auto with = [&](auto four_bits, auto whole) {
        cache_append_kernel<T, G, decltype(four_bits)::value, decltype(whole)::value><<<(unsigned)blocks, kTpb, 0, s>>>(p);
    };
    using Yes = std::true_type;
    using No = std::false_type;
    if (p.pages.groups) chunks ? with(Yes{}, Yes{}) : with(Yes{}, No{});
    else chunks ? with(No{}, Yes{}) : with(No{}, No{});
    nnk_after_launch(what, s);
}

}  // namespace

extern "C" void launch_cache_append(void* q_out, const void* q, const void* k, const void* v,
    const NnCacheAppend* a, const NnCache* c, hipStream_t s) {
    const char* what = "launch_cache_append";
    NNK_REQUIRE(a, what, "%s: null description", what);
    const NnQkNormRope& o = a->rope;
    Append p = {};
    if (!nnk_cache_take(p.pages, c, o.dtype, o.kv_heads, o.head_dim, true, what)) return;
    NNK_REQUIRE(o.tokens >= 0 && o.heads >= 0 && o.heads <= 1 << 20, what, "%s: bad shape tokens=%d heads=%d", what, o.tokens,
        o.heads);
    NNK_REQUIRE(o.rot_dim >= 0 && o.rot_dim <= o.head_dim && o.rot_dim % 2 == 0, what,
        "%s: rot_dim=%d is odd or past head_dim=%d", what, o.rot_dim, o.head_dim);
    NNK_REQUIRE(o.axes >= 1 && o.rot_dim / 2 % o.axes == 0, what, "%s: axes=%d do not divide rot_dim / 2 = %d", what, o.axes,
        o.rot_dim / 2);
    NNK_REQUIRE(!a->norm || o.eps >= 0.0f, what, "%s: eps=%g is negative", what, o.eps);
    if (!o.tokens) return;
    NNK_REQUIRE((long long)o.tokens * (o.heads + 2 * o.kv_heads) < 1LL << 30, what, "%s: too many rows", what);
    NNK_REQUIRE(!o.rot_dim || (o.pos && o.freq), what, "%s: null pos or freq", what);
    NNK_REQUIRE(a->place, what, "%s: null place", what);
    NNK_REQUIRE(k && v && (!o.heads || (q && q_out)), what, "%s: null pointer", what);
    const long long n[2] = {o.tokens, o.heads};
    NNK_REQUIRE(!o.heads || nnk_rows_apart(2, o.q_out_stride, n, o.head_dim), what,
        "%s: rows of q_out overlap (strides %lld, %lld)", what, o.q_out_stride[0], o.q_out_stride[1]);
    const long long e = o.dtype == NN_BF16 ? 8 : 4;
    p.vec = o.head_dim % e == 0 && nnk::aligned16(k) && nnk::aligned16(v);
    if (o.heads) p.vec = p.vec && nnk::aligned16(q) && nnk::aligned16(q_out);
    for (int i = 0; i < 2; ++i) {
        p.qs[i] = o.q_stride[i];
        p.ks[i] = o.k_stride[i];
        p.vs[i] = a->v_stride[i];
        p.qos[i] = o.q_out_stride[i];
        p.vec = p.vec && p.ks[i] % e == 0 && p.vs[i] % e == 0 && (!o.heads || (p.qs[i] % e == 0 && p.qos[i] % e == 0));
    }
    p.q = q;
    p.k = k;
    p.v = v;
    p.q_out = q_out;
    p.q_weight = a->norm ? o.q_weight : nullptr;
    p.k_weight = a->norm ? o.k_weight : nullptr;
    p.pos = o.pos;
    p.freq = o.freq;
    p.request = a->request;
    p.place = a->place;
    p.tokens = o.tokens;
    p.heads = o.heads;
    p.kv_heads = o.kv_heads;
    p.dim = o.head_dim;
    p.half = o.rot_dim / 2;
    p.axes = o.axes;
    p.per_axis = std::max(1, p.half / o.axes);
    p.interleaved = o.interleaved;
    p.norm = a->norm;
    p.eps = o.eps;
    // lanes of a row: a power of two with 16 bytes each
    const int lanes = (int)((o.head_dim + e - 1) / e);
    if (o.dtype == NN_BF16) {
        if (lanes <= 4) launch<bf16, 4>(p, s, what);
        else if (lanes <= 8) launch<bf16, 8>(p, s, what);
        else launch<bf16, 16>(p, s, what);
    } else {
        if (lanes <= 8) launch<float, 8>(p, s, what);
        else if (lanes <= 16) launch<float, 16>(p, s, what);
        else launch<float, 32>(p, s, what);
    }
}
