// attn_paged.h -- 64 keys or values of a paged cache on their way to LDS, for the attention
// kernel of many queries.  Measured, bf16, 2048 causal queries over 16384 keys, 16 heads of 128 (4 of keys):
// plain pages 442 us, 4 bits 402 us (the form for few queries 881 and 369).
#pragma once

#include "attn_common.h"
#include "cache_common.h"

namespace cache {

using namespace attn;

// Where the 16-key quarters of blocks of 64 lie: a lane has a quarter, a wave 16 blocks, looked up
// together.  Blocks come in order from one whose number is a multiple of 16.
struct Finder {
    unsigned long long byte = 0;  // of the head's block in the page, either pool
    int slot = -1;                // of the quarter's first key; -1: there is no page
    unsigned long long held = 0;  // which lanes have one

    // Which quarters of `block` have a page.
    __device__ __forceinline__ unsigned find(const Pages& p, int b, int kv, int block) {
        if (block % 16 == 0) {
            const int key = block * kBlock + (int)(threadIdx.x & 63) * 16;
            const unsigned page = p.table[(size_t)b * p.table_pages + min(key >> p.shift, p.table_pages - 1)];
            const bool is = page < (unsigned)p.pages;
            byte = (unsigned long long)(is ? page : 0u) * (unsigned)p.page_bytes + (unsigned long long)kv * (unsigned)p.block_bytes;
            slot = is ? p.slot_of(key) : -1;
            held = __ballot(is);
        }
        return (unsigned)(held >> (block % 16 * 4)) & 15;
    }
    __device__ __forceinline__ void at(int block, int row, unsigned long long& from, int& from_slot) const {
        const int lane = block % 16 * 4 + (row >> 4);
        const unsigned lo = __shfl((int)byte, lane), hi = __shfl((int)(byte >> 32), lane);
        from = (unsigned long long)hi << 32 | lo;
        from_slot = max(__shfl(slot, lane), 0) + (row & 15);
    }
};

// As Staged.  Plain pages.
template <typename T, int DP, bool FP4>
struct Paged {
    static constexpr int kPerRow = DP / Type<T>::CE;
    static constexpr int N = kBlock * kPerRow / kTpb;
    u32x4 v[N];

    static __device__ __forceinline__ int row(int n) { return (n * kTpb + (int)threadIdx.x) / kPerRow; }
    static __device__ __forceinline__ int chunk(int n) { return (n * kTpb + (int)threadIdx.x) % kPerRow; }
    __device__ __forceinline__ void load(const char* pool, const Pages& p, const Finder& f, int block) {
#pragma unroll
        for (int n = 0; n < N; ++n) {
            unsigned long long from;
            int slot;
            f.at(block, row(n), from, slot);
            // past the features: the row's first chunk, which meets zeros or is not stored
            v[n] = *reinterpret_cast<const u32x4*>(pool + from + (unsigned)(slot * p.row_bytes + (chunk(n) * 16 < p.row_bytes ? chunk(n) * 16 : 0)));
        }
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

// Pages of 4 bits: a thread has 32 features of a row and their scale, and converts them on the way
// to LDS, where they are the tensors' type.
template <typename T, int DP>
struct Paged<T, DP, true> {
    static constexpr int kPerRow = DP / kGroup;  // one or two chunks of a row, or three or four, for a thread
    static constexpr int N = (kBlock * kPerRow + kTpb - 1) / kTpb;
    u32x4 v[N];
    unsigned scale[N];

    static __device__ __forceinline__ int row(int n) { return (n * kTpb + (int)threadIdx.x) / kPerRow; }
    static __device__ __forceinline__ int chunk(int n) { return (n * kTpb + (int)threadIdx.x) % kPerRow; }
    static __device__ __forceinline__ bool in(int n) { return kBlock * kPerRow % kTpb == 0 || n * kTpb + (int)threadIdx.x < kBlock * kPerRow; }
    __device__ __forceinline__ void load(const char* pool, const Pages& p, const Finder& f, int block) {
#pragma unroll
        for (int n = 0; n < N; ++n) {
            unsigned long long from;
            int slot;
            f.at(block, row(n) % kBlock, from, slot);
            const int c = min(chunk(n), p.groups - 1);
            if (!in(n)) continue;
            v[n] = *reinterpret_cast<const u32x4*>(pool + from + (unsigned)(slot * p.row_bytes + c * 16));
            scale[n] = *reinterpret_cast<const unsigned char*>(pool + from + (unsigned)(p.scales + slot * p.groups + c));
        }
    }
    template <typename Keep>
    __device__ __forceinline__ void store(char* lds, bool all, const Keep& keep) const {
        typedef T T2 __attribute__((ext_vector_type(2)));
        constexpr int kWords = 4, kEach = 8 / Type<T>::CE;  // words of 8 features; 16-byte chunks of one
        const auto write = [&](int n, bool some) {
            const float factor = some ? scale_of(scale[n]) : 1.0f;
            // Rows differ in which bits of a chunk's number they turn: a wave's 16 lanes of four rows write
            // different words at once, so that they meet different banks.
            const int r = row(n), turn = r & 3;
            unsigned w[kWords];
#pragma unroll
            for (int i = 0; i < kWords; ++i) w[i] = some ? v[n][i] : 0u;
            const auto swap = [](bool yes, unsigned& x, unsigned& y) {
                const unsigned t = yes ? y : x;
                y = yes ? x : y;
                x = t;
            };
            swap(turn & 1, w[0], w[1]);
            swap(turn & 1, w[2], w[3]);
            swap(turn & 2, w[0], w[2]);
            swap(turn & 2, w[1], w[3]);
#pragma unroll
            for (int i = 0; i < kWords; ++i) {
                T2 y[4];
                values8(w[i], factor, y);
                u32x4 out[kEach];
                __builtin_memcpy(out, y, sizeof out);
#pragma unroll
                for (int j = 0; j < kEach; ++j)
                    *reinterpret_cast<u32x4*>(lds + Lds<T, DP>::at(r, (kWords * chunk(n) + (i ^ turn)) * kEach + j)) = out[j];
            }
        };
        if (all) {
#pragma unroll
            for (int n = 0; n < N; ++n)
                if (in(n)) write(n, true);
        } else {
#pragma unroll
            for (int n = 0; n < N; ++n)
                if (in(n)) write(n, keep(n));
        }
    }
};

}  // namespace cache
