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
// fp32 queries and probabilities meet 4-bit pages as three bf16 parts each, 24 bits of them.  With bf16
// tensors a probability is one bf16 value in its product with the values, off by up to 2^-8 of itself and
// independently of the others (its sum is fp32 and of what it was before): outputs are then 2.1e-3 to 2.4e-3 of their
// norm off, where their own rounding alone is 1.7e-3.  A second part would double those products.
//
// Measured: 16 requests of 8192 to 32768 keys, 32 heads of 128 (8 of keys), scores under a cap: bf16
// pages 218 us, 6.2 TB/s (reads alone reach 7.1); 4 bits 68 us, 5.3 TB/s of about a quarter of the bytes, some
// 14 us of it lengths, table, first loads and the joins (11 of those with no join between workgroups).
// 48 requests of five queries over 4096 keys, 16 heads (4), 4 bits 29 us, 17 of them such ends; one of 777
// keys, 8 heads of 64, 7.9 us; three of seven fp32 queries over 5001 keys, 12 heads of 96 (4), 4 bits 24 us.
#include "attn_common.h"
#include "cache_common.h"

namespace {
using namespace attn;
using cache::Pages;

constexpr int kKeys = 32;       // keys of a wave at a time
constexpr int kTile = 16;       // queries, or keys, of a tile
constexpr int kHalves = kKeys / kTile;
constexpr float kSlack = 8.0f;  // units of log2 that a score may be above the reference

typedef cache::bf16x2 bf16x2;

__device__ __forceinline__ f32x4 mma16(bf16x8 a, bf16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma16(float a, float b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }

// Over the four lanes of a column.
__device__ __forceinline__ Halves rows16(float v) {
    const unsigned u = __builtin_bit_cast(unsigned, v);
    const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    const unsigned lower = r[0], upper = r[1];
    return {__builtin_bit_cast(float, lower), __builtin_bit_cast(float, upper)};
}
__device__ __forceinline__ float max_column(float v) {
    const Halves x = rows16(v);
    return max_halves(fmaxf(x.lower, x.upper));
}
__device__ __forceinline__ float sum_column(float v) {
    const Halves x = rows16(v);
    return sum_halves(x.lower + x.upper);
}

// Where 16 keys lie: uniform.
struct Place {
    unsigned long long byte;  // of the head's block in the page, either pool
    unsigned row, scale;      // of the first one's row and scales in that
    bool held;
};
// The blocks of 32 keys of a wave, kStep apart: the entries of 64 of them are read at a time, a
// lane each, and handed out lane by lane (a scalar load for each made its wave wait, LDS reads
// among it).
constexpr int kStep = kWaves * kKeys;
struct Blocks32 {
    const int* table;
    unsigned long long block;  // the head's byte in a page
    int entry[kHalves], n;
    __device__ __forceinline__ void look(const Pages& p, int k0, int lane) {
        const int last = p.table_pages - 1, key = k0 + lane * kStep;
        entry[0] = table[min(key >> p.shift, last)];
        entry[1] = p.shift > 4 ? entry[0] : table[min((key + kTile) >> p.shift, last)];
    }
    __device__ __forceinline__ Blocks32(const Pages& p, int b, int kv)
        : table(p.table + (size_t)b * p.table_pages), block((unsigned long long)kv * (unsigned)p.block_bytes), entry{0, 0}, n(64) {}
    // The next block, which begins at k0: there is one, and so there are pages in the table.
    __device__ __forceinline__ void next(Place (&at)[kHalves], const Pages& p, int k0, int lane) {
        if (n == 64) {
            look(p, k0, lane);
            n = 0;
        }
        const auto place = [&](Place& x, int entry, int key) {
            const unsigned page = __builtin_amdgcn_readlane(entry, n);
            x.held = page < (unsigned)p.pages;
            x.byte = (unsigned long long)(x.held ? page : 0u) * (unsigned)p.page_bytes + block;
            x.row = p.slot_of(key) * p.row_bytes;
            x.scale = p.scales + p.slot_of(key) * p.groups;
        };
        place(at[0], entry[0], k0);
        if (p.shift > 4) {  // one page has both halves
            at[1] = at[0];
            at[1].row += kTile * p.row_bytes;
            at[1].scale += kTile * p.groups;
        } else {
            place(at[1], entry[1], k0 + kTile);
        }
        ++n;
    }
};
// A uniform address, for the loads' scalar operand: by itself the compiler adds the lane's offset
// to the pool once and the place to that, 64 bits a lane, for every load.
typedef const __attribute__((address_space(1))) char* Bytes;
__device__ __forceinline__ Bytes at_place(const char* pool, unsigned long long byte, unsigned offset) {
    Bytes q = (Bytes)pool + byte + offset;
    asm("" : "+s"(q));
    return q;
}
template <typename V>
__device__ __forceinline__ V read(Bytes q, unsigned offset) {
    return __builtin_nontemporal_load(reinterpret_cast<const __attribute__((address_space(1))) V*>(q + offset));
}
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

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
    // A tile begins at a multiple of kAlign bytes, so that chunk c ^ x is at the address of c with x
    // in its bits: one register and an instruction instead of a register for each.
    static constexpr int kAlign = 512;
    // This lane's part of the transposing reads: keys 4 h .. 4 h + 3 and 16 more of features 16 d ..
    static __device__ __forceinline__ unsigned column_base(int lane) { return at(lane >> 2, lane >> 1 & 1) + (lane & 1) * 8; }
    static __device__ __forceinline__ bf16x8 columns(unsigned base, int d) {
        const i16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4*)(uintptr_t)(base ^ d << 5));
        const i16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4*)(uintptr_t)((base ^ d << 5) + kTile * kRowBytes));
        const bf16x4 x = __builtin_bit_cast(bf16x4, a), y = __builtin_bit_cast(bf16x4, b);
        return __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
    }
};
__device__ __forceinline__ void lds_write(unsigned at, u32x4 v) { *(__attribute__((address_space(3))) u32x4*)(uintptr_t)at = v; }

template <int DP>
struct Mxfp4 {
    typedef bf16x8 Frag;
    static constexpr bool kFourBits = true;
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
            const Bytes rows = at_place(p.k, at[x].byte, at[x].row), scales = at_place(p.k, at[x].byte, at[x].scale);
            const unsigned from = row * (DP / 2) + h * (DP / 8);
            if constexpr (DP == 128) {
                const u32x4 y = read<u32x4>(rows, from);
#pragma unroll
                for (int u = 0; u < kWords; ++u) k[x][u] = y[u];
            } else if constexpr (DP == 64) {
                const u32x2 y = read<u32x2>(rows, from);
                k[x][0] = y[0];
                k[x][1] = y[1];
            } else {
#pragma unroll
                for (int u = 0; u < kWords; ++u) k[x][u] = read<unsigned>(rows, from + 4 * u);
            }
#pragma unroll
            for (int u = 0; u < kScales; ++u) ks[x][u] = read<unsigned char>(scales, row * kGroups + feature(h, u) / 32);
        }
#pragma unroll
        for (int n = 0; n < kChunks; ++n) {
            const int c = min(chunk(n, lane), kKeys * kGroups - 1), key = c / kGroups, g = c % kGroups;
            const unsigned r = (key & 15) * (DP / 2) + g * 16, sc = (key & 15) * kGroups + g;
            if constexpr (kTile * kGroups % 64 == 0) {  // 16 keys are whole chunks of a wave
                constexpr int kEach = kTile * kGroups / 64;
                v[n] = read<u32x4>(at_place(p.v, at[n / kEach].byte, at[n / kEach].row), r);
                vs[n] = read<unsigned char>(at_place(p.v, at[n / kEach].byte, at[n / kEach].scale), sc);
            } else {
                const Bytes rows0 = at_place(p.v, at[0].byte, at[0].row), rows1 = at_place(p.v, at[1].byte, at[1].row);
                const Bytes scales0 = at_place(p.v, at[0].byte, at[0].scale), scales1 = at_place(p.v, at[1].byte, at[1].scale);
                v[n] = read<u32x4>(key < kTile ? rows0 : rows1, r);
                vs[n] = read<unsigned char>(key < kTile ? scales0 : scales1, sc);
            }
        }
    }
    __device__ __forceinline__ Frag key(int x, int u) const {
        bf16x2 y[4];
        cache::values8(k[x][u], cache::scale_of(ks[x][kScales > 1 ? u : 0]), y);
        return __builtin_bit_cast(Frag, y);
    }
    // The lane's first chunk of a tile at `lds`.
    static __device__ __forceinline__ unsigned store_base(unsigned lds, int lane) {
        return lds + Values<DP>::at(lane / kGroups, 4 * (lane % kGroups));
    }
    // keep(key): whether it is one that a query sees
    template <typename Keep>
    __device__ __forceinline__ void store(unsigned lds, unsigned base, int lane, const Keep& keep) const {
#pragma unroll
        for (int n = 0; n < kChunks; ++n) {
            const int c = chunk(n, lane), key = c / kGroups, g = c % kGroups;
            if (kKeys * kGroups % 64 && c >= kKeys * kGroups) continue;
            // 16 keys on, the order of chunks is the same
            const unsigned to = 64 / kGroups % kTile ? lds + Values<DP>::at(key, 4 * g) : base + n * (64 / kGroups) * Values<DP>::kRowBytes;
            const bool some = keep(key);
            const float scale = some ? cache::scale_of(vs[n]) : 1.0f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                bf16x2 y[4];
                cache::values8(some ? v[n][i] : 0u, scale, y);
                lds_write(to ^ i << 4, __builtin_bit_cast(u32x4, y));
            }
        }
    }
};

template <int DP>
struct Bf16 {
    typedef bf16x8 Frag;
    static constexpr bool kFourBits = false;
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
                k[x][u] = read<u32x4>(at_place(p.k, at[x].byte, at[x].row), row * p.row_bytes + min((unsigned)feature(h, u) * 2, last));
#pragma unroll
        for (int n = 0; n < kChunks; ++n) {
            const int c = n * 64 + lane, key = c / kPerRow;
            const unsigned r = (unsigned)(key & 15) * p.row_bytes + min((unsigned)(c % kPerRow) * 16, last);
            if constexpr (kTile * kPerRow % 64 == 0) {  // 16 keys are whole chunks of a wave
                const Place& x = at[n / (kTile * kPerRow / 64)];
                v[n] = read<u32x4>(at_place(p.v, x.byte, x.row), r);
            } else {
                const Bytes rows0 = at_place(p.v, at[0].byte, at[0].row), rows1 = at_place(p.v, at[1].byte, at[1].row);
                v[n] = read<u32x4>(key < kTile ? rows0 : rows1, r);
            }
        }
    }
    __device__ __forceinline__ Frag key(int x, int u) const { return __builtin_bit_cast(Frag, k[x][u]); }
    static __device__ __forceinline__ unsigned store_base(unsigned lds, int lane) {
        return lds + Values<DP>::at(lane / kPerRow, lane % kPerRow);
    }
    template <typename Keep>
    __device__ __forceinline__ void store(unsigned lds, unsigned base, int lane, const Keep& keep) const {
#pragma unroll
        for (int n = 0; n < kChunks; ++n) {
            const int c = n * 64 + lane, key = c / kPerRow;
            // rows of a power of two: only bits of S change
            constexpr int kRowsOn = 64 / kPerRow;
            const unsigned to = 64 % kPerRow ? lds + Values<DP>::at(key, c % kPerRow)
                                             : (base ^ (Values<DP>::S(n * kRowsOn) << 4)) + n * kRowsOn * Values<DP>::kRowBytes;
            lds_write(to, keep(key) ? v[n] : u32x4{0, 0, 0, 0});
        }
    }
};

// fp32 pages: products of 4, a value at a time; a lane's values are features 16 d + (l & 15) of
// the keys 4 h + j, which it reads where they lie.
template <int DP>
struct F32 {
    typedef float Frag;
    static constexpr bool kFourBits = false;
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
                k[x][u] = read<f32x4>(at_place(p.k, at[x].byte, at[x].row), row * p.row_bytes + min(64 * u + 16 * h, last));
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int d = 0; d < DP / 16; ++d)
                    v[x][j][d] = read<float>(at_place(p.v, at[x].byte, at[x].row), (4 * h + j) * p.row_bytes + min(64 * d + 4 * row, last + 12));
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

// The work of a launch are units, a request's key heads and tiles of queries, of as many steps of
// 128 keys as the request has.  A unit is divided into parts of about as many steps as every other's, a
// workgroup each, so many that they fill the card; requests' lengths are on the device, so this is
// done there, by every workgroup for itself.  Parts of a unit are joined from their partial results.
// (Equal shares of the steps in a row, that ended and began within units, fill the card more evenly,
// 16 long requests in bf16 209 us where parts are 218, but a workgroup then has two ends of parts,
// some 10 us each: the same in 4 bits 73 us for 68, 48 requests of five queries over 4096 keys 37 for 29.)
struct Few {
    unsigned* tickets;  // a unit each, by ticket_of
    float* partial;     // [workers, rows, DP + 2]: outputs, then reference (units of log2) and sum
    int tiles;          // of a key head's queries
    int units;          // of a request: key heads and tiles
    int workers;        // parts at most; 0: a workgroup a unit
    int at_once;        // workgroups that the card holds
    int step;           // keys of a step, kStep or, so that all steps are counted in 32 bits, a multiple
};
constexpr int kMostParts = 64;  // of a unit
// Tickets are in the words where launch_attention_forward has its own, so that a workspace serves both,
// in an order that keeps successive units' on lines of their own: on one line, those of 32 units were
// 2 us of a step over 4 caches of 4096.
constexpr int kTicketLine = 32, kTicketLines = kTicketWords / kTicketLine;
__device__ __forceinline__ int ticket_of(int unit) { return unit % kTicketLines * kTicketLine + unit / kTicketLines; }

// Steps of a unit of request b: those of its last query, one at least.
__device__ __forceinline__ int steps_of(const Args& a, const Pages& p, const Few& f, int b) {
    const int keys = p.pages ? keys_of(a, b) : 0;
    return max(1, (int)((unsigned)(limit_of(a, b, keys, start_of(a, b) + a.len_q - 1) + f.step - 1) / (unsigned)f.step));
}
// Sum over the wave; and inclusive sums over the lanes.
__device__ __forceinline__ int sum_of(int v) {
    v += __builtin_amdgcn_mov_dpp(v, nnk::kDppQuadXor1, 0xf, 0xf, true);
    v += __builtin_amdgcn_mov_dpp(v, nnk::kDppQuadXor2, 0xf, 0xf, true);
    v += __builtin_amdgcn_mov_dpp(v, nnk::kDppRowHalfMirror, 0xf, 0xf, true);
    v += __builtin_amdgcn_mov_dpp(v, nnk::kDppRowMirror, 0xf, 0xf, true);
    return __builtin_amdgcn_readlane(v, 0) + __builtin_amdgcn_readlane(v, 16) + __builtin_amdgcn_readlane(v, 32) +
        __builtin_amdgcn_readlane(v, 48);
}
__device__ __forceinline__ int scan(int v, int lane) {
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
        const int y = __shfl_up(v, m);
        if (lane >= m) v += y;
    }
    return v;
}
struct Part {
    int request, unit;  // of the request's
    int steps;          // of the unit
    int part, parts;    // of the unit's
    int first;          // workgroup of the unit's first part
};
// The part of workgroup `worker`; false if there is none.
__device__ __forceinline__ bool part_of(Part& x, const Args& a, const Pages& p, const Few& f, int worker, int lane) {
    const auto steps_at = [&](int b) { return b < a.batch ? steps_of(a, p, f, b) : 0; };
    int n = steps_at(lane), most = n, total = sum_of(n);
    for (int b0 = 64; b0 < a.batch; b0 += 64) {
        const int more = steps_at(b0 + lane);
        total += sum_of(more);
        most = max(most, more);
    }
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) most = max(most, __shfl_xor(most, m));
    // A part more is a sixteenth of a step's time more for the workgroup that joins a unit's: of e steps
    // a part, e + most / 16 e is least at this.
    const int least = max((int)ceilf(sqrtf(0.0625f * (float)most)), (most + kMostParts - 1) / kMostParts);
    // The fewest steps a part of which there are no more than workgroups: between what an even row of them
    // would be and what is enough if every unit has a part that is not full.
    const unsigned all = (unsigned)(total * f.units), units = (unsigned)(a.batch * f.units);
    const auto up = [](unsigned x, unsigned y) { return (int)((x + y - 1) / y); };
    // As many as there are places, or twice that where there are units for more than half of them.
    // (Twice as many always: 16 long requests 218 -> 213 us in bf16, but 68 -> 77 in 4 bits, and the 48 of
    // five queries 29 -> 42; three times as many where parts are long 68 -> 82.)
    const int places = 2 * (int)units <= f.at_once ? f.at_once : 2 * f.at_once;
    const int target = max(min(places, f.workers), (int)units + 1);
    int low = max(up(all, target), least), each = max(up(all, target - units), low);
    if (a.batch <= 64) {
        while (low < each) {
            const int mid = (low + each) / 2;
            if (sum_of(up(n, mid)) * f.units <= target) each = mid;
            else low = mid + 1;
        }
    }
    int before = 0;  // parts of the requests so far
    for (int b0 = 0; b0 < a.batch; b0 += 64) {
        if (b0) n = steps_at(b0 + lane);
        const int parts = up(n, each), sum = before + scan(parts, lane) * f.units;
        const unsigned long long behind = __ballot(sum > worker);
        if (behind) {
            const int i = __builtin_ctzll(behind);
            x.request = b0 + i;
            x.steps = __builtin_amdgcn_readlane(n, i);
            x.parts = __builtin_amdgcn_readlane(parts, i);
            const int from = __builtin_amdgcn_readlane(sum, i) - x.parts * f.units;
            x.unit = __builtin_amdgcn_readfirstlane((int)((unsigned)(worker - from) / (unsigned)x.parts));
            x.first = from + x.unit * x.parts;
            x.part = worker - x.first;
            return true;
        }
        before = __builtin_amdgcn_readlane(sum, 63);
    }
    return false;
}

// The call.  What only the beginning and the end of a part need is read again there: held over the
// keys' loop it was some 130 scalar registers too many, which go to lanes of vector registers.
struct All {  // the kernel's only argument
    Args a;
    Pages p;
    Few f;
};
__device__ __forceinline__ All call_again() {
    auto q = __builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(q));
    All all;
    __builtin_memcpy(&all, (const void*)q, sizeof all);
    return all;
}

// Workgroups a CU, which is waves a SIMD: as many as their registers allow.
template <typename T, typename E, int NT>
constexpr int held_by_a_cu() {
    if constexpr (std::is_same_v<typename E::Frag, float>) return 1;
    else if constexpr (sizeof(T) == 4) return NT == 2 ? 1 : 2;
    else return NT == 1 && E::kFourBits ? 3 : 2;
}

// TERMS: 0 none, 1 a cap, 2 a bias and maybe a cap (which a register or two more, and their
// instructions, would cost the others)
template <typename T, template <int> class PAGES, int DP, int NT, int TERMS>
__global__ __launch_bounds__(kTpb, (held_by_a_cu<T, PAGES<DP>, NT>())) void cache_few_kernel(All) {
    using E = PAGES<DP>;
    constexpr bool kWide = std::is_same_v<typename E::Frag, bf16x8>;     // bf16 products
    constexpr int kParts = kWide && sizeof(T) == 4 ? 3 : 1;              // of a query or probability
    constexpr int kRowsEach = kTile * NT;
    constexpr int kRow = DP + 4;  // floats of an output row in LDS
    constexpr int kUsed = E::kLds > kTile * kRow * 4 ? E::kLds : kTile * kRow * 4;
    constexpr int kShared = (kUsed + Values<DP>::kAlign - 1) / Values<DP>::kAlign * Values<DP>::kAlign;
    __shared__ __attribute__((aligned(Values<DP>::kAlign))) char lds[kWaves][kShared];
    __shared__ float m_lds[kWaves][kRowsEach], l_lds[kWaves][kRowsEach];
    __shared__ int last_one;

    const int lane = threadIdx.x & 63, h = lane >> 4, col = lane & 15, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Part part;
    {
        const auto [a, p, f] = call_again();
        if (f.workers) {
            if (!part_of(part, a, p, f, blockIdx.x, lane)) return;
        } else {
            part.request = __builtin_amdgcn_readfirstlane((int)(blockIdx.x / (unsigned)f.units));
            part.unit = blockIdx.x - part.request * f.units;
            part.steps = __builtin_amdgcn_readfirstlane(steps_of(a, p, f, part.request));
            part.part = part.first = 0;
            part.parts = 1;
        }
    }

    {
        const All now = call_again();
        const Args& a = now.a;
        const Pages& p = now.p;
        const Few& f = now.f;
        const int b = part.request;
        // divisions are vector instructions: what is uniform says so
        const int kv = __builtin_amdgcn_readfirstlane((int)((unsigned)part.unit / (unsigned)f.tiles)), tile = part.unit - kv * f.tiles;
        const auto step_at = [&](int i) {  // where a part begins
            return __builtin_amdgcn_readfirstlane((int)((unsigned long long)(unsigned)part.steps * (unsigned)i / (unsigned)part.parts));
        };
        const int step0 = step_at(part.part), step1 = step_at(part.part + 1);
        const int rows = min(kRowsEach, a.len_q * a.group - tile * kRowsEach);
        const int keys = __builtin_amdgcn_readfirstlane(p.pages ? keys_of(a, b) : 0), start = __builtin_amdgcn_readfirstlane(start_of(a, b));
        const int most = __builtin_amdgcn_readfirstlane(limit_of(a, b, keys, start + (tile * kRowsEach + rows - 1) / a.group));

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
        [[maybe_unused]] float far[NT];  // bias of keys max_distance or more before the query
        if constexpr (TERMS == 2) {
#pragma unroll
            for (int t = 0; t < NT; ++t) far[t] = bias_of(-a.max_distance, head[t]);
        }
        const float unit_of = TERMS ? 1.0f : a.c1;  // what a score is multiplied with in the exponent

        f32x4 o[NT][DP / 16];
        float m[NT], l[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
#pragma unroll
            for (int d = 0; d < DP / 16; ++d) o[t][d] = f32x4{0, 0, 0, 0};
            m[t] = -INFINITY;
            l[t] = 0.0f;
        }

        [[maybe_unused]] const unsigned values = (unsigned)(unsigned long long)(__attribute__((address_space(3))) char*)lds[wave];
        unsigned to_values = 0, of_columns = 0;
        if constexpr (kWide) {
            to_values = E::store_base(values, lane);
            of_columns = values + Values<DP>::column_base(lane);
        }

        // this wave's blocks of the steps
        const int end = (int)min((long long)most, (long long)step1 * f.step);
        int k0 = step0 * f.step + wave * kKeys;
        E e;
        Place at[kHalves];
        Blocks32 blocks(p, b, kv);
        const auto load = [&](int from) {
            if (from >= end) return;
            blocks.next(at, p, from, lane);
            e.load(at, p, lane);
        };
        for (load(k0); k0 < end; k0 += kStep) {
            const bool held0 = at[0].held, held1 = at[1].held, all = held0 && held1 && k0 + kKeys <= keys;
            // (kept from taking a register for every address over the loop)
            asm volatile("" : "+v"(to_values), "+v"(of_columns));
            f32x4 s[NT][kHalves];
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int x = 0; x < kHalves; ++x) s[t][x] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int u = 0; u < E::kSteps; ++u)  // the halves in turn: a product waits for the one before it
#pragma unroll
                for (int x = 0; x < kHalves; ++x) {
                    const typename E::Frag y = e.key(x, u);
#pragma unroll
                    for (int t = 0; t < NT; ++t)
#pragma unroll
                        for (int n = kParts - 1; n >= 0; --n) s[t][x] = mma16(y, qf[t][n][u], s[t][x]);
                }
            const auto keep = [&](int key) { return k0 + key < keys && (key < kTile ? held0 : held1); };
            [[maybe_unused]] float v[kWide ? 1 : kHalves][4][kWide ? 1 : DP / 16];
            if constexpr (kWide) {
                if (all) e.store(values, to_values, lane, [](int) { return true; });
                else e.store(values, to_values, lane, keep);
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                __builtin_amdgcn_wave_barrier();
            } else {
#pragma unroll
                for (int x = 0; x < kHalves; ++x)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
#pragma unroll
                        for (int d = 0; d < DP / 16; ++d) v[x][j][d] = all || keep(x * kTile + 4 * h + j) ? e.v[x][j][d] : 0.0f;
            }
            // the next block's, while this one's scores become shares
            load(k0 + kStep);

#pragma unroll
            for (int t = 0; t < NT; ++t) {
                if constexpr (TERMS) {
                    if (TERMS == 1 || a.c2 != 0.0f) {
                        float top = 0.0f;
#pragma unroll
                        for (int x = 0; x < kHalves; ++x)
#pragma unroll
                            for (int j = 0; j < 4; ++j) top = fmaxf(top, fabsf(s[t][x][j]));
                        if (__all(top < a.tiny)) {
#pragma unroll
                            for (int x = 0; x < kHalves; ++x)
#pragma unroll
                                for (int j = 0; j < 4; ++j) s[t][x][j] = cap_series<4>(s[t][x][j], a);
                        } else if (__all(top < a.small)) {
#pragma unroll
                            for (int x = 0; x < kHalves; ++x)
#pragma unroll
                                for (int j = 0; j < 4; ++j) s[t][x][j] = cap_series<6>(s[t][x][j], a);
                        } else {
#pragma unroll
                            for (int x = 0; x < kHalves; ++x)
#pragma unroll
                                for (int j = 0; j < 4; ++j) {
                                    const float y = s[t][x][j] * a.c1, r = __builtin_amdgcn_rcpf(exp2_fast(fabsf(y) * (2.0f * kLog2e)) + 1.0f);
                                    s[t][x][j] = (fabsf(y) < kSeriesEnd ? tanh_series(y) : copysignf(fmaf(-2.0f, r, 1.0f), y)) * a.c2;
                                }
                        }
                    }
                    if constexpr (TERMS == 2) {
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
                }
                if (!held0 || !held1 || k0 + kKeys > least) {
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
                    const float to = fmaxf(m[t], top), by = exp2_fast(m[t] - (to == -INFINITY ? 0.0f : to));
                    l[t] *= by;
#pragma unroll
                    for (int d = 0; d < DP / 16; ++d) o[t][d] *= by;
                    m[t] = to;
                }
                const float base = m[t] == -INFINITY ? 0.0f : m[t];
#pragma unroll
                for (int x = 0; x < kHalves; ++x)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        s[t][x][j] = exp2_fast(TERMS ? s[t][x][j] - base : fmaf(s[t][x][j], unit_of, -base));
                        l[t] += s[t][x][j];
                    }
            }
            if constexpr (kWide) {
                bf16x8 shares[NT][kParts];
                struct Columns {
                    bf16x8 x[2];
                } columns[2];
                const auto read_columns = [&](Columns& y, int n) {
#pragma unroll
                    for (int i = 0; i < 2; ++i) y.x[i] = Values<DP>::columns(of_columns, 2 * n + i);
                };
                read_columns(columns[0], 0);
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    float x[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) x[j] = s[t][j / 4][j % 4];
                    parts_of<kParts>(x, shares[t]);
                }
                piped<DP / 32>(columns, read_columns, [&](const Columns& y, int n) {
#pragma unroll
                    for (int i = 0; i < 2; ++i)
#pragma unroll
                        for (int t = 0; t < NT; ++t)
#pragma unroll
                            for (int k = kParts - 1; k >= 0; --k) o[t][2 * n + i] = mma16(y.x[i], shares[t][k], o[t][2 * n + i]);
                });
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

        const All after = call_again();
        const auto close = [&](const Args& a, const Pages& p, const Few& f) {
        const int parts = part.parts;
        const long long step = kRowsEach * (DP + 2);
        const auto partial_of = [&](int i) { return f.partial + (part.first + i) * step; };

        // the waves of the workgroup, a tile of queries at a time
        constexpr int kQuads = DP / 4;  // 4 features a thread
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
                    const float by = ref == -INFINITY ? 0.0f : exp2_fast(m_lds[w][r] - ref);
                    const float4 y = nnk::ld4(reinterpret_cast<const float*>(lds[w]) + c * kRow + d);
                    all = fmaf(l_lds[w][r], by, all);
                    x.x = fmaf(y.x, by, x.x);
                    x.y = fmaf(y.y, by, x.y);
                    x.z = fmaf(y.z, by, x.z);
                    x.w = fmaf(y.w, by, x.w);
                }
                if (parts == 1) {
                    finish(r, d, x, ref, all);
                } else {
                    float* to = partial_of(part.part) + r * (DP + 2);
                    hand(to + d, x.x, x.y);
                    hand(to + d + 2, x.z, x.w);
                    if (d == 0) hand(to + DP, ref, all);
                }
            }
        }

        if (parts > 1) {  // the workgroups of the unit
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // handed over
            __syncthreads();
            unsigned* ticket = f.tickets + ticket_of(b * f.units + part.unit);  // fewer than kTicketWords: they are in parts
            if (threadIdx.x == 0)
                last_one = __hip_atomic_fetch_add(ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (unsigned)(parts - 1);
            __syncthreads();
            if (last_one) {
                constexpr int kAtOnce = 8;  // parts whose loads are under way together
                for (int n = threadIdx.x; n < rows * kQuads; n += kTpb) {
                    const int r = n / kQuads, d = n % kQuads * 4;
                    float ref = -INFINITY, sum = 0.0f;
                    float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    for (int part0 = 0; part0 < parts; part0 += kAtOnce) {
                        float2 y[kAtOnce], z[kAtOnce], w[kAtOnce];
#pragma unroll
                        for (int i = 0; i < kAtOnce; ++i) {
                            w[i] = make_float2(-INFINITY, 0.0f);
                            if (part0 + i >= parts) continue;
                            const float* q = partial_of(part0 + i) + r * (DP + 2);
                            y[i] = taken(q + d);
                            z[i] = taken(q + d + 2);
                            w[i] = taken(q + DP);
                        }
                        float top = ref;
#pragma unroll
                        for (int i = 0; i < kAtOnce; ++i) top = fmaxf(top, w[i].x);
                        const float base = top == -INFINITY ? 0.0f : top, old = exp2_fast(ref - base);
                        sum *= old;
                        x = make_float4(x.x * old, x.y * old, x.z * old, x.w * old);
#pragma unroll
                        for (int i = 0; i < kAtOnce; ++i) {
                            if (part0 + i >= parts) continue;
                            const float by = exp2_fast(w[i].x - base);
                            sum = fmaf(w[i].y, by, sum);
                            x.x = fmaf(y[i].x, by, x.x);
                            x.y = fmaf(y[i].y, by, x.y);
                            x.z = fmaf(z[i].x, by, x.z);
                            x.w = fmaf(z[i].y, by, x.w);
                        }
                        ref = top;
                    }
                    finish(r, d, x, ref, sum);
                }
                if (threadIdx.x == 0) __hip_atomic_store(ticket, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            }
        }
        };
        close(after.a, after.p, after.f);
    }
}

// Tiles of queries, and parts at most.
constexpr int kHeld = 3;  // workgroups a CU at most
struct Plan {
    long long units, steps, tiles;
    int rows, step;
    bool parted;
};
Plan plan_of(const NnAttention* a) {
    Plan p;
    const long long rows = (long long)a->len_q * (a->heads / a->kv_heads);
    p.steps = std::max(1, (a->len_k + kStep - 1) / kStep);
    p.rows = rows <= kTile ? kTile : 2 * kTile;
    p.tiles = (rows + p.rows - 1) / p.rows;
    p.units = (long long)a->batch * a->kv_heads * p.tiles;
    p.step = kStep;
    while (p.step < 1 << 30 && p.units * ((a->len_k + (long long)p.step - 1) / p.step + 1) >= 1LL << 30) p.step *= 2;
    p.parted = p.units <= kTicketWords && p.steps > 1;
    return p;
}
// Parts at most, where the card holds `held` workgroups a CU; twice the units at least.
long long workers_of(const Plan& p, int held) { return std::min(std::max(2LL * kCus * held, 2 * p.units), p.units * p.steps); }
int padded(int dim) { return (dim + 31) / 32 * 32; }

template <typename T, template <int> class PAGES, int DP>
void launch(const Args& a, const Pages& p, const Plan& plan, float* ws, hipStream_t s, const char* what) {
    const auto with = [&](auto tiles, auto terms) {
        constexpr int NT = decltype(tiles)::value;
        constexpr int held = held_by_a_cu<T, PAGES<DP>, NT>();
        const int workers = plan.parted && plan.units < 2 * kCus * held ? (int)workers_of(plan, held) : 0;
        const All all = {a, p, {reinterpret_cast<unsigned*>(ws), ws + kTicketWords, (int)plan.tiles, (int)(a.kv_heads * plan.tiles), workers, kCus * held, plan.step}};
        cache_few_kernel<T, PAGES, DP, NT, decltype(terms)::value>
            <<<workers ? (unsigned)workers : (unsigned)plan.units, kTpb, 0, s>>>(all);
    };
    const auto by_terms = [&](auto tiles) {
        if (a.buckets) with(tiles, std::integral_constant<int, 2>{});
        else if (a.c2 != 0.0f) with(tiles, std::integral_constant<int, 1>{});
        else with(tiles, std::integral_constant<int, 0>{});
    };
    if (plan.rows == kTile) by_terms(std::integral_constant<int, 1>{});
    else by_terms(std::integral_constant<int, 2>{});
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

// Which form is quicker, by the work of each.  This one has units of one tile of 16 rows or two, whose
// keys it shares out evenly; what a unit costs a key depends on what it reads (plain pages) or converts and
// multiplies, and its parts' ends some hundred keys more.  The other one has workgroups of 128 queries of a
// head, whatever they fill of them, and takes as long as kFill of them (of 64) where CUs are left over.  It
// reads a key head once for each of its heads; in fp32 its tiles leave one workgroup a CU.  In units of a
// workgroup and key:
struct Unit {
    double key, ends;  // a key, and the ends of its parts
    double start;      // of a call of more keys than a step
};
struct Costs {
    Unit one, two;       // tiles a unit
    double group, more;  // of the other form's
};
constexpr double kFill = 273.0;
constexpr Costs kPlainBf16 = {{0.72, 0.0, 33e3}, {0.92, 250.0, 88e3}, 0.75, 0.0}, kPlainF32 = {{0.6, 100.0, 0.0}, {1.0, 100.0, 40e3}, 2.0, 0.0},
                kFourBits = {{0.45, 400.0, 10e3}, {0.5, 550.0, 100e3}, 1.3, 210.0};
// Measured, this form and the other in us (heads with those of keys, features in brackets; uneven: a quarter of
// the keys to all).  One token: 32 requests of 4096 keys, 32 heads (32, 128), bf16 317 / 351, uneven 278 / 272, fp32 849 /
// 2302, uneven 571 / 1472; 64 of 32768 bf16 5000 / 5551, fp32 11520 / 36165; 48 of 32768 uneven, 8 heads (8, 128), bf16
// 642 / 847, fp32 1958 / 4286, 4 bits 197 / 602; 64 of 300 uneven, 32 heads (32, 64), 31 / 28, 66 / 167, 20 / 27.
// Several: 64 requests of 16 over 1024 keys, 8 heads (8, 128), 64 / 45, 122 / 305, 39 / 34; of 32 over 300 keys 47 / 20,
// 83 / 106, 38 / 16; 16 of 64 over 1024, 16 heads (4, 128), 73 / 30, 178 / 99, 48 / 28; 2 of 256 over 8192 130 / 174,
// 550 / 683, 68 / 161.  Prompts: 512 tokens over 8192 keys, 32 heads (8, 128), 235 / 175, 1021 / 684, 125 / 161; 2048 over 16384,
// 16 heads (4, 128), 881 / 443, 3953 / 2555, 369 / 402; 4 of 300 over 300, 8 heads (8, 64), 24 / 11, 33 / 22, 19 / 12.  Short
// caches, one request, 8 heads (2, 128): one token of 200 keys 10.0 / 11.2, 13.7 / 28.5, 8.7 / 11.2, six tokens 13.6 / 11.9,
// 23.8 / 28.9, 12.3 / 11.2.  Over 150 drawn shapes that had no part in the choice of the costs, the form taken is slower than
// the other by 0.6 % in the mean, and by up to 57 % (209 requests of 35 fp32 queries over 124 keys, 4 heads, 128 / 82).
// fp32 queries over 4 bits come here always: the products of three bf16 parts are quicker than the other form's fp32
// ones (512 queries over 8192 keys 221 / 684).
extern "C" int nnk_cache_is_few(const NnAttention* a, int four_bits) {
    const bool half = a->dtype == NN_BF16;
    if (four_bits && !half) return true;
    const Costs& c = four_bits ? kFourBits : half ? kPlainBf16 : kPlainF32;
    const Plan p = plan_of(a);
    const double len = a->len_k, units = (double)p.units, groups = std::ceil(a->len_q / 128.0) * a->heads * a->batch;
    const Unit& u = p.rows == kTile ? c.one : c.two;
    const bool parts = p.steps > 1 && p.units < 4 * kCus;
    const double own = units * (len * u.key + (parts ? u.ends : 0.0)) + (p.steps > 1 ? u.start : 0.0);
    return own <= std::max(c.group * groups + c.more, kFill) * len;
}
bool nnk_cache_few_fits(const NnAttention* a) { return plan_of(a).units < (1LL << 32) / kTpb; }  // threads of a launch
// Floats of a call's workspace: enough for its tickets and parts, and for every smaller call's, which
// has fewer units, steps and rows (and 2048 of them at most in parts).
size_t nnk_cache_few_floats(const NnAttention* a) {
    if (!a->batch || !a->len_q || a->len_k <= kStep) return 0;
    Plan p = plan_of(a);
    p.units = std::min<long long>(p.units, kTicketWords);
    return kTicketWords + (size_t)workers_of(p, kHeld) * p.rows * (padded(a->head_dim) + 2);
}
bool nnk_cache_few_parted(const NnAttention* a) { return a->batch && a->len_q && plan_of(a).parted; }
void nnk_cache_few(const Args& a, const Pages& p, const NnAttention* d, float* ws, hipStream_t s, const char* what) {
    const Plan plan = plan_of(d);
    if (d->dtype == NN_BF16) {
        if (p.groups) by_dim<bf16, Mxfp4>(a, p, plan, ws, s, what);
        else by_dim<bf16, Bf16>(a, p, plan, ws, s, what);
    } else {
        if (p.groups) by_dim<float, Mxfp4>(a, p, plan, ws, s, what);
        else by_dim<float, F32>(a, p, plan, ws, s, what);
    }
}
