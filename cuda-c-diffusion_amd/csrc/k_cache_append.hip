// k_cache_append.hip -- rows of a projection: queries turned, keys turned and values written
// to the pages of their requests, in the tensors' type or in 4 bits.
//
// A key row x of head_dim features:  y = x [rsqrt(mean(x^2) + eps) w],  its pairs turned by
// their angles;  in 4 bits then, for 32 features at a time, the least exponent e with
// max|y| <= 7 2^e and the 8 sizes' nearest to |y| 2^-e.  Every row is read once and written
// once: memory bounds long prompts, latency a decoding step, whose rows are therefore dealt
// out over workgroups that make one pass each.  A row belongs to the G lanes of a group, 16
// bytes a lane, so that sums and maxima are cross-lane steps in the group; a pair's other
// member comes from the group's row in LDS.
//
// Keys for 4 bits are formed in 64 bits, as a code is a choice: with fp32 sums the order of
// the additions would decide it for some values in 10^5, and with it half a step of the value.
#include "cache_common.h"

#include <algorithm>

namespace {
using namespace cache;

constexpr int kTpb = 256;
constexpr int kAngles = 1024;  // sines and cosines of a workgroup's tokens

struct Append {
    const void *q, *k, *v;
    void* q_out;
    Pages pages;
    long long qs[2], ks[2], vs[2], qos[2];
    const float *q_weight, *k_weight;
    const int *pos, *request, *place;
    const double* freq;
    int tokens, heads, kv_heads, rows, dim, half, axes, per_axis, interleaved, norm;
    int tokens_each, parts, rows_each;  // tokens of a workgroup; workgroups that share them; rows of a token that it has
    float eps;
    bool vec;
};

// The code of |x| = a 2^e, a <= 7: steps of 1/2 below 2, of 1 below 4, of 2 from there.
template <typename A>
__device__ __forceinline__ unsigned code_of(A a) {
    const A step = a < (A)2 ? (A)2 : a < (A)4 ? (A)1 : (A)0.5;
    const int base = a < (A)2 ? 0 : a < (A)4 ? 2 : 4;
    return (unsigned)min((int)rint(a * step) + base, 7);
}
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
template <typename A>
struct Limits;
template <>
struct Limits<float> {
    static constexpr int kTop = 128;
    static __device__ __forceinline__ float power(int e) { return __builtin_bit_cast(float, (unsigned)(e + 127) << 23); }
};
template <>
struct Limits<double> {
    static constexpr int kTop = 1024;
    static __device__ __forceinline__ double power(int e) {
        return __builtin_bit_cast(double, (unsigned long long)(e + 1023) << 52);
    }
};

template <typename T, int G>
struct Row {
    static constexpr int CE = 16 / (int)sizeof(T);
    static constexpr int kGroups = kTpb / G;

    template <typename A>
    static __device__ __forceinline__ void load(A* x, const T* row, int d0, const Append& a) {
        T e[CE];
        if (a.vec && d0 < a.dim) {
            const u32x4 v = *reinterpret_cast<const u32x4*>(row + d0);
            __builtin_memcpy(e, &v, 16);
        } else {
#pragma unroll
            for (int j = 0; j < CE; ++j) e[j] = d0 + j < a.dim ? row[d0 + j] : (T)0.0f;
        }
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
    static __device__ __forceinline__ A other_of(A v, int m) { return __shfl_xor(v, m); }

    // Norm and turn of the lane's features d0 ..; `row`: the group's values in LDS
    template <typename A, typename CS>
    static __device__ __forceinline__ void turn(A* x, int d0, A* row, const CS* cs, const float* weight, const Append& a) {
        if (a.norm) {
            A ss = 0;
#pragma unroll
            for (int j = 0; j < CE; ++j) ss += x[j] * x[j];
            ss = group_sum(ss) / (A)a.dim + (A)a.eps;
            const A rstd = sizeof(A) == 8 ? (A)(1.0 / sqrt((double)ss)) : (A)rsqrtf((float)ss);
#pragma unroll
            for (int j = 0; j < CE; ++j) x[j] = x[j] * rstd * (A)(weight && d0 + j < a.dim ? weight[d0 + j] : 1.0f);
        }
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
        // the group's lanes are in one wave, whose LDS accesses are in order
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
        for (int m = 1; m < kLanes; m <<= 1) most = fmax(most, other_of(most, m));
        bool past;
        int e = exponent_of(most, past);
        const bool none = e == Limits<A>::kTop;
        e = min(max(e - (past ? 1 : 2), -120), 125);
        const A down = Limits<A>::power(-e);
        unsigned code = 0;
#pragma unroll
        for (int j = 0; j < CE; ++j) code |= (code_of(fmin(fabs(x[j]) * down, (A)7)) | (x[j] < 0 ? 8u : 0u)) << (4 * j);
        if (d0 >= p.groups * kGroup) return;
        char* to = block + slot * p.row_bytes + d0 / 2;
        if constexpr (CE == 8) *reinterpret_cast<unsigned*>(to) = code;
        else *reinterpret_cast<unsigned short*>(to) = (unsigned short)code;
        if (d0 % kGroup == 0)
            *reinterpret_cast<unsigned char*>(block + p.scales + slot * p.groups + d0 / kGroup) = (unsigned char)(none ? 255 : e + 127);
    }
};

template <bool WIDE>
struct Turns;
template <>
struct Turns<false> {
    typedef float A;
    typedef float2 CS;
};
template <>
struct Turns<true> {
    typedef double A;
    typedef double2 CS;
};

// Cosine and sine of each pair of `count` tokens; the angle is formed and reduced in 64 bits.
// `fine`: so are they.
template <typename CS>
__device__ __forceinline__ void angles(CS* cs, const Append& a, int token0, int count, bool fine) {
    for (int i = threadIdx.x; i < count * a.half; i += kTpb) {
        const int t = i / a.half, p = i - t * a.half;
        double turns = (double)a.pos[(size_t)(token0 + t) * a.axes + p / a.per_axis] * a.freq[p] * 0.15915494309189533577;
        turns -= rint(turns);
        if (sizeof(CS) == 16 && fine) {
            double s, c;
            sincospi(2.0 * turns, &s, &c);
            cs[i].x = c;
            cs[i].y = s;
        } else {
            // to an eighth of a turn either way: fp32 rounds what is left, and the small one of
            // sine and cosine keeps its digits
            const double quarters = rint(4.0 * turns);
            const int q = (int)quarters;
            float s, c;
            sincospif(0.5f * (float)(4.0 * turns - quarters), &s, &c);
            const float x = q & 1 ? s : c, y = q & 1 ? c : s;
            cs[i].x = (q + 1) & 2 ? -x : x;
            cs[i].y = q & 2 ? -y : y;
        }
    }
}

template <typename T, int G, bool FP4>
__global__ __launch_bounds__(kTpb) void cache_append_kernel(Append a) {
    using R = Row<T, G>;
    using A = typename Turns<FP4>::A;
    using CS = typename Turns<FP4>::CS;
    constexpr int CE = R::CE;
    __shared__ __attribute__((aligned(16))) CS cs[kAngles];
    __shared__ __attribute__((aligned(16))) A lds[R::kGroups][G * CE];
    const int group = threadIdx.x / G, d0 = (threadIdx.x % G) * CE;
    const int part = blockIdx.x % a.parts, token0 = blockIdx.x / a.parts * a.tokens_each;
    const int tokens = min(a.tokens_each, a.tokens - token0);
    const int row0 = part * a.rows_each, each = min(a.rows_each, a.rows - row0);
    if (each <= 0) return;
    const int turned = a.heads + a.kv_heads;
    if (row0 < turned) {
        angles(cs, a, token0, tokens, row0 + each > a.heads);
        __syncthreads();
    }
    for (int r = group; r < tokens * each; r += R::kGroups) {
        const int t = r / each, row = row0 + r - t * each, token = token0 + t;
        const int place = a.place[token];
        if (place < 0) continue;
        if (row < a.heads) {
            float x[CE];
            R::load(x, (const T*)a.q + token * a.qs[0] + row * a.qs[1], d0, a);
            R::turn(x, d0, reinterpret_cast<float*>(lds[group]), cs + t * a.half, a.q_weight, a);
            R::store((T*)a.q_out + token * a.qos[0] + row * a.qos[1], d0, a.dim, a.vec, x);
            continue;
        }
        const int page = a.pages.page_of(a.request ? a.request[token] : token, place), slot = a.pages.slot_of(place);
        if (page < 0) continue;
        if (row < turned) {
            const int head = row - a.heads;
            char* block = a.pages.k + a.pages.block_at(page, head);
            A x[CE];
            R::load(x, (const T*)a.k + token * a.ks[0] + head * a.ks[1], d0, a);
            R::turn(x, d0, lds[group], cs + t * a.half, a.k_weight, a);
            if constexpr (FP4) R::pack(block, slot, d0, x, a.pages);
            else R::store((T*)(block + slot * a.pages.row_bytes), d0, a.dim, true, x);
        } else {
            const int head = row - turned;
            char* block = a.pages.v + a.pages.block_at(page, head);
            float x[CE];
            R::load(x, (const T*)a.v + token * a.vs[0] + head * a.vs[1], d0, a);
            if constexpr (FP4) R::pack(block, slot, d0, x, a.pages);
            else R::store((T*)(block + slot * a.pages.row_bytes), d0, a.dim, true, x);
        }
    }
}

// Few tokens: one each, their rows shared by workgroups of one pass.  Many: rows for 16 passes
// of a workgroup's groups, as far as their sines fit.
constexpr int kFewTokens = 1024;
template <typename T, int G>
void launch(Append& p, hipStream_t s, const char* what) {
    constexpr int groups = Row<T, G>::kGroups;
    const int by_rows = std::max(1, 16 * groups / p.rows), by_angles = kAngles / std::max(1, p.half);
    p.tokens_each = std::max(1, std::min({by_rows, by_angles, p.tokens / kFewTokens}));
    p.parts = p.tokens < kFewTokens ? (p.rows + groups - 1) / groups : 1;
    p.rows_each = (p.rows + p.parts - 1) / p.parts;
    const long long blocks = ((long long)p.tokens + p.tokens_each - 1) / p.tokens_each * p.parts;
    NNK_REQUIRE(blocks < (1LL << 32) / kTpb, what, "%s: too many rows", what);  // threads of a launch
    if (p.pages.groups) cache_append_kernel<T, G, true><<<(unsigned)blocks, kTpb, 0, s>>>(p);
    else cache_append_kernel<T, G, false><<<(unsigned)blocks, kTpb, 0, s>>>(p);
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
    p.rows = o.heads + 2 * o.kv_heads;
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
