// k_attn_few.hip -- attention, few queries over many keys (a decoding step, a small chunk).
//
// Reading the cache once is the whole cost.  The queries of all heads that share a key head
// are columns of one 32 x 32 tile, so a key is read once for them; the keys are split over
// workgroups and, within one, over its 4 waves, each of which streams its own range through
// its own LDS, without barriers, its next 32 keys' loads under way.  A wave keeps its own
// running maximum, sum and output; the waves of a workgroup are joined in LDS, workgroups
// by the one that is done last (a ticket a unit; it reads the others' results in their
// order, so the sum does not depend on who is last, and leaves the ticket at zero).
//
// Measured: 16 requests of 12288 to 32768 keys, 32 heads of 128 (8 of keys), bf16: 294 us, 4.57
// TB/s of the cache (an elementwise stream reaches 6.2, read and written); one request of 777
// keys 8.3 us, of which a launch is about 5.  The same in fp32, one wave a SIMD: 862 us, 3.1
// TB/s; 11.3 us.
#include "attn_common.h"

namespace {
using namespace attn;

constexpr int kKeys = 32;        // keys of a wave at a time
constexpr int kTickets = kTicketWords;
constexpr int kMaxSplits = 64;
constexpr size_t kTableBytes = 16384;  // LDS for the bias by distance

// 32 rows on their way from memory to a wave's LDS.
template <typename T, int DP, bool VEC>
struct WaveTile {
    static constexpr int kPerRow = DP / Type<T>::CE;
    static constexpr int N = kKeys * kPerRow / 64;
    u32x4 v[N];
    static __device__ __forceinline__ int row(int n) { return (n * 64 + (int)(threadIdx.x & 63)) / kPerRow; }
    static __device__ __forceinline__ int chunk(int n) { return (n * 64 + (int)(threadIdx.x & 63)) % kPerRow; }
    __device__ __forceinline__ void load(const T* base, long long stride, int last, int dim) {
#pragma unroll
        for (int n = 0; n < N; ++n)
            v[n] = load_chunk<T, VEC>(base + min(row(n), last) * stride, chunk(n) * Type<T>::CE, dim);
    }
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

// Two floats handed to, and taken from, workgroups of other XCDs.
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
    float* partial;  // [units, splits, 32, DP + 2]: outputs, then maximum (units of log2) and sum
    bool table;
    int tiles, splits, each;  // 32-row tiles of a key head's queries; workgroups of a unit; their keys
};

template <typename T, int DP, bool CAP, bool BIAS, bool VEC>
__global__ __launch_bounds__(kTpb, sizeof(T) == 2 && VEC ? 2 : 1) void attn_few_kernel(Args a, Few f) {
    using L = Lds<T, DP>;
    constexpr int kTile = kKeys * L::kRowBytes;
    constexpr int kRow = DP + 4;  // floats of an output row in LDS
    constexpr int kShared = 2 * kTile > 32 * kRow * 4 ? 2 * kTile : 32 * kRow * 4;
    __shared__ __attribute__((aligned(16))) char lds[kWaves][kShared];
    __shared__ __attribute__((aligned(16))) int doc_lds[kWaves][kKeys];
    __shared__ float m_lds[kWaves][32], l_lds[kWaves][32];
    __shared__ float weight[32][kMaxSplits];
    __shared__ float total[32];
    __shared__ int last_one;
    extern __shared__ float table[];  // BIAS: of each head of the tile by distance, if it fits (f.table)

    const int lane = threadIdx.x & 63, h = lane >> 5, wave = threadIdx.x >> 6, col = lane & 31;
    const int split = blockIdx.x % f.splits, unit = blockIdx.x / f.splits;
    const int tile = unit % f.tiles, kv = unit / f.tiles % a.kv_heads, b = unit / f.tiles / a.kv_heads;
    const int rows = min(32, a.len_q * a.group - tile * 32);
    const int row = tile * 32 + col, i = row / a.group, head = kv * a.group + row - i * a.group;
    const bool in = col < rows;
    const int keys = keys_of(a, b), start = start_of(a, b), pos = start + i;
    const int limit = in ? limit_of(a, b, keys, pos) : 0;
    const int most = limit_of(a, b, keys, start + (tile * 32 + rows - 1) / a.group);
    const int active = max(1, (most + f.each - 1) / f.each);  // workgroups of the unit that have keys
    if (split >= active) return;

    const int doc = in && a.doc_q ? a.doc_q[(size_t)b * a.len_q + i] : -1;
    int least = in ? limit : INT32_MAX, doc_lo = doc >= 0 ? doc : INT32_MAX, doc_hi = doc >= 0 ? doc : INT32_MIN;
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) {
        least = min(least, __shfl_xor(least, m));
        doc_lo = min(doc_lo, __shfl_xor(doc_lo, m));
        doc_hi = max(doc_hi, __shfl_xor(doc_hi, m));
    }
    const int* docs = a.doc_k ? a.doc_k + (size_t)b * a.len_k : nullptr;
    const int4* key_docs = a.key_docs ? a.key_docs + (size_t)b * ((a.len_k + kBlock - 1) / kBlock) : nullptr;

    Frag<T> qf[L::kSteps];
    {
        const int c = in ? col : 0, r = tile * 32 + c, qi = r / a.group;
        const T* q = (const T*)a.q + b * a.qs[0] + qi * a.qs[1] + (kv * a.group + r - qi * a.group) * a.qs[2];
#pragma unroll
        for (int u = 0; u < L::kSteps; ++u) qf[u] = load_frag<T, VEC>(q, (2 * u + h) * Type<T>::CE, a.dim);
    }
    const T* kp = (const T*)a.k + b * a.ks[0] + kv * a.ks[2];
    const T* vp = (const T*)a.v + b * a.vs[0] + kv * a.vs[2];
    char *k_lds = lds[wave], *v_lds = lds[wave] + kTile;

    // this wave's keys, in blocks of 32
    const int part = f.each / kWaves, first = split * f.each + wave * part, end = min(most, first + part);
    const auto meeting = [&](int k0) {
        if (key_docs)
            while (k0 < end) {
                const int4 d = key_docs[k0 / kBlock];
                if (d.x <= doc_hi && doc_lo <= d.y) break;
                k0 += kKeys;
            }
        return k0;
    };
    WaveTile<T, DP, VEC> ks, vs;
    int next_doc = 0;
    const auto load = [&](int k0) {
        const int last = keys - 1 - k0;
        if (docs) next_doc = docs[k0 + min(col, last)];
        ks.load(kp + k0 * a.ks[1], a.ks[1], last, a.dim);
        vs.load(vp + k0 * a.vs[1], a.vs[1], last, a.dim);
    };
    const int span = 2 * a.max_distance + 1;
    const auto bias_of = [&](int i, int of_head) {
        return a.bias[(size_t)min(max(a.bucket[i], 0), a.buckets - 1) * a.heads + of_head] * kLog2e;
    };
    if constexpr (BIAS) {
        if (f.table) {
            for (int n = threadIdx.x; n < a.group * span; n += kTpb) table[n] = bias_of(n % span, kv * a.group + n / span);
            __syncthreads();
        }
    }
    const int own = in ? head - kv * a.group : 0;
    const auto bias_at = [&](int rel) {
        const int i = min(max(rel, -a.max_distance), a.max_distance) + a.max_distance;
        return f.table ? table[own * span + i] : bias_of(i, kv * a.group + own);
    };
    float far = 0.0f;  // bias of keys max_distance or more before the query
    if constexpr (BIAS) far = bias_at(-a.max_distance);

    f32x16 o[DP / 32];
#pragma unroll
    for (int d = 0; d < DP / 32; ++d) o[d] = zero16();
    float m = -INFINITY, l = 0.0f;
    const int rbase = L::row_base(lane), cbase = L::col_base(lane);
    int k0 = meeting(first);
    if (k0 < end) load(k0);
    while (k0 < end) {
        const int at = k0;
        const auto keep = [&](int n) {
            const int r = at + WaveTile<T, DP, VEC>::row(n);
            return r < keys && (!docs || docs[r] >= 0);
        };
        const bool all = at + kKeys <= keys && !docs;
        ks.store(k_lds, all, keep);
        vs.store(v_lds, all, keep);
        if (docs && h == 0) doc_lds[wave][col] = at + col < keys ? max(next_doc, -1) : -1;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        k0 = meeting(at + kKeys);
        if (k0 < end) load(k0);

        f32x16 s = zero16();
#pragma unroll
        for (int u = 0; u < L::kSteps; ++u) s = mma(L::rows(k_lds, 0, u, rbase), qf[u], s);
        if constexpr (CAP) {
            cap_scores(s, a.c1, a.c2);
        } else {
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] *= a.c1;
        }
        if constexpr (BIAS) {
            if (__all(at + kKeys - 1 - pos <= -a.max_distance)) {
#pragma unroll
                for (int r = 0; r < 16; ++r) s[r] += far;
            } else {
#pragma unroll
                for (int r = 0; r < 16; ++r) s[r] += bias_at(at + row_of(r, h) - pos);
            }
        }
        if (docs || at + kKeys > least) hide(s, at, limit, docs ? doc_lds[wave] : nullptr, doc, h);
        float top = m;
#pragma unroll
        for (int r = 0; r < 16; ++r) top = fmaxf(top, s[r]);
        top = max_halves(top);
        const float base = top == -INFINITY ? 0.0f : top;
        if (__any(top > m)) {
            const float g = exp2_fast(m - base);
            l *= g;
#pragma unroll
            for (int d = 0; d < DP / 32; ++d)
#pragma unroll
                for (int r = 0; r < 16; ++r) o[d][r] *= g;
            m = top;
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            s[r] = exp2_fast(s[r] - base);
            l += s[r];
        }
#pragma unroll
        for (int n = 0; n < L::kKeySteps; ++n) {
            const Frag<T> p = operand(s, n, T{});
#pragma unroll
            for (int d = 0; d < DP / 32; ++d) o[d] = mma(L::cols(v_lds, 0, n, d, cbase), p, o[d]);
        }
        // the next rows are written over these when they have been read
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
    l = sum_halves(l);

    // the waves of the workgroup
    float* mine = reinterpret_cast<float*>(lds[wave]) + col * kRow;
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g)
            nnk::st4(mine + 32 * d + 8 * g + 4 * h,
                make_float4(o[d][4 * g], o[d][4 * g + 1], o[d][4 * g + 2], o[d][4 * g + 3]));
    if (h == 0) {
        m_lds[wave][col] = m;
        l_lds[wave][col] = l;
    }
    __syncthreads();
    constexpr int kQuads = DP / 4;  // 4 features a thread
    float* to = f.partial + ((size_t)unit * f.splits + split) * 32 * (DP + 2);
    const auto finish = [&](int r, int d, float4 x, float ref, float sum) {
        const int n = tile * 32 + r, qi = n / a.group, hd = kv * a.group + n - qi * a.group;
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        store4<T, VEC>((T*)a.out + b * a.os[0] + qi * a.os[1] + hd * a.os[2], d, a.dim, x.x * inv, x.y * inv, x.z * inv,
            x.w * inv);
        if (d == 0)
            a.lse[((size_t)b * a.heads + hd) * a.len_q + qi] = sum == 0.0f ? -INFINITY : (ref + log2f(sum)) * kLn2;
    };
    for (int n = threadIdx.x; n < rows * kQuads; n += kTpb) {
        const int r = n / kQuads, d = n % kQuads * 4;
        float ref = m_lds[0][r];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) ref = fmaxf(ref, m_lds[w][r]);
        float sum = 0.0f;
        float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const float g = ref == -INFINITY ? 0.0f : exp2_fast(m_lds[w][r] - ref);
            const float4 y = nnk::ld4(reinterpret_cast<const float*>(lds[w]) + r * kRow + d);
            sum = fmaf(l_lds[w][r], g, sum);
            x.x = fmaf(y.x, g, x.x);
            x.y = fmaf(y.y, g, x.y);
            x.z = fmaf(y.z, g, x.z);
            x.w = fmaf(y.w, g, x.w);
        }
        if (active == 1) {
            finish(r, d, x, ref, sum);
        } else {
            float* p = to + r * (DP + 2);
            hand(p + d, x.x, x.y);
            hand(p + d + 2, x.z, x.w);
            if (d == 0) hand(p + DP, ref, sum);
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
    const float* from = f.partial + (size_t)unit * f.splits * 32 * (DP + 2);
    const size_t step = 32 * (DP + 2);
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
        const float* p = from + r * (DP + 2) + d;
        float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
        for (int sp = 0; sp < active; ++sp) {
            const float g = weight[r][sp];
            const float2 y = taken(p + sp * step), z = taken(p + sp * step + 2);
            x.x = fmaf(y.x, g, x.x);
            x.y = fmaf(y.y, g, x.y);
            x.z = fmaf(z.x, g, x.z);
            x.w = fmaf(z.y, g, x.w);
        }
        finish(r, d, x, m_lds[0][r], total[r]);
    }
    if (threadIdx.x == 0) __hip_atomic_store(f.tickets + unit, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// How the keys are split: where the cache's bytes count, enough workgroups to fill the card
// several times over (requests' lengths differ, and those without keys of theirs end at
// once); for more rows, whose products count, once.  128 keys at least, a block a wave.
struct Plan {
    long long units;
    int tiles, splits, each;
};
Plan plan_of(int batch, int len_q, int len_k, int kv_heads, int group) {
    Plan p;
    p.tiles = (int)(((long long)len_q * group + 31) / 32);
    p.units = (long long)batch * kv_heads * p.tiles;
    const int step = kWaves * kKeys, steps = std::max(1, (len_k + step - 1) / step);
    const long long fill = p.tiles <= 2 ? 2 * kTickets : 3 * kCus;
    const long long want = p.units >= kTickets ? 1 : std::min<long long>(kMaxSplits, (fill + p.units - 1) / p.units);
    const int n = (int)((steps + want - 1) / want);
    p.each = n * step;
    p.splits = (steps + n - 1) / n;
    return p;
}

template <typename T, int DP, bool CAP, bool BIAS, bool VEC>
bool launch(const Args& a, float* ws, hipStream_t s, const char* what) {
    const Plan p = plan_of(a.batch, a.len_q, a.len_k, a.kv_heads, a.group);
    const size_t table = BIAS ? (size_t)a.group * (2 * a.max_distance + 1) * sizeof(float) : 0;
    const Few f = {reinterpret_cast<unsigned*>(ws), ws + kTickets, table && table <= kTableBytes, p.tiles, p.splits, p.each};
    if constexpr (BIAS) {
        static std::atomic<unsigned long long> done{0};
        if (!raise_lds((const void*)attn_few_kernel<T, DP, CAP, BIAS, VEC>, kTableBytes, done, what)) return false;
    }
    attn_few_kernel<T, DP, CAP, BIAS, VEC>
        <<<(unsigned)(p.units * p.splits), kTpb, f.table ? table : 0, s>>>(a, f);
    nnk_after_launch(what, s);
    return true;
}

}  // namespace

// Few queries: the rows of a key head's queries fit in two tiles; or workgroups of 64 would
// leave half of the CUs without work while each goes over many keys.  bf16, this form against
// the other: 8192 tokens of one head of 64 58 against 107 us (128 workgroups), 4096 causal
// tokens of three heads of 128 85 against 77 (192), 2 x 2000 of four of 64 43 against 31 (256).
bool nnk_attention_is_few(const NnAttention* a) {
    const long long rows = (long long)a->len_q * (a->heads / a->kv_heads);
    const long long groups = ((long long)a->len_q + 63) / 64 * a->heads * a->batch;
    return (rows <= 64 && (long long)a->batch * a->kv_heads < 1 << 20) || (groups <= kCus / 2 && a->len_k >= 512);
}
// Floats of the workspace after the tickets.
size_t nnk_attention_few_floats(const NnAttention* a) {
    const Plan p = plan_of(a->batch, a->len_q, a->len_k, a->kv_heads, a->heads / a->kv_heads);
    // rows that are not on 16 bytes are taken as 128 features, so all are sized for that
    return p.splits == 1 ? 0 : (size_t)p.units * p.splits * 32 * (128 + 2);
}
// Units and workgroups more than the fill, at most.  Up to two tiles of a key head's rows: fewer
// units than tickets; more tiles: 2 units for each of kCus / 2 workgroups of 64 queries.
size_t nnk_attention_few_most(const NnAttention* a) {
    const long long owners = (long long)a->batch * a->kv_heads, group = a->heads / a->kv_heads;
    const long long tiles = (a->len_q * group + 31) / 32, steps = ((long long)a->len_k + kWaves * kKeys - 1) / (kWaves * kKeys);
    if (steps < 2) return 0;
    const auto groups = [&](long long units, long long fill) {
        return std::min(units * std::min<long long>(kMaxSplits, steps), units + fill - 1);
    };
    const long long few = groups(std::min(kTickets - 1LL, owners * std::min(2LL, tiles)), 2 * kTickets);
    const long long more = groups(std::min<long long>(kCus, owners * tiles), 3 * kCus);
    return (size_t)std::max(few, more) * 32 * (128 + 2);
}
bool nnk_attention_few(const Args& a, bool half, float* ws, hipStream_t s, const char* what) {
    return NNK_ATTN_DISPATCH(a, half, launch, a, ws, s, what);
}
