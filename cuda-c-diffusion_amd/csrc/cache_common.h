// cache_common.h -- the paged cache, as its kernels take it.
#pragma once

#include "nn_cache.h"
#include "nnk_common.h"

namespace cache {

typedef __bf16 bf16;
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

constexpr int kGroup = 32;  // features of a scale
constexpr int kMostTokens = (1 << 30) - 4096;  // of a request

struct Pages {
    const int* table;
    char *k, *v;
    long long page_bytes;  // of a page, one pool
    int block_bytes;       // of a head in it
    int row_bytes, groups; // of a token in that; scales of a row (0: plain)
    int scales;            // byte in a block where they begin
    int shift;             // log2 of page_tokens
    int pages, requests, table_pages;

    // The page of token p of request r, or -1.
    __device__ __forceinline__ int page_of(int r, int p) const {
        const int i = p >> shift;
        if ((unsigned)r >= (unsigned)requests || (unsigned)i >= (unsigned)table_pages) return -1;
        const int page = table[(size_t)r * table_pages + i];
        return (unsigned)page < (unsigned)pages ? page : -1;
    }
    __device__ __forceinline__ int slot_of(int p) const { return p & ((1 << shift) - 1); }
    __device__ __forceinline__ long long block_at(int page, int head) const {
        return page * page_bytes + (long long)head * block_bytes;
    }
};

// A scale's byte as the factor 2^(scale - 127): exact, 0 for 0 apart from the conversions below,
// which take its exponent alone (255: NaN).
__device__ __forceinline__ float scale_of(unsigned byte) { return __builtin_bit_cast(float, byte << 23); }

// The 8 features of 32 bits, as bf16 or fp32: one instruction for two.
typedef bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ void values8(unsigned code, float scale, bf16x2 (&v)[4]) {
    v[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(code, scale, 0);
    v[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(code, scale, 1);
    v[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(code, scale, 2);
    v[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(code, scale, 3);
}
__device__ __forceinline__ void values8(unsigned code, float scale, f32x2 (&v)[4]) {
    v[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code, scale, 0);
    v[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code, scale, 1);
    v[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code, scale, 2);
    v[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code, scale, 3);
}

}  // namespace cache

// Fills `p` from the description; false after recording an error.  `pools`: whether the
// pointers are looked at.
bool nnk_cache_take(cache::Pages& p, const NnCache* c, int dtype, int kv_heads, int head_dim, bool pools, const char* what);
// Attention of few queries: one launch; when it is taken; whether a launch has that many workgroups; the
// floats of its workspace, which are enough for every smaller batch and fewer queries or keys, and whether a
// call needs it.
namespace attn {
struct Args;
}
extern "C" int nnk_cache_is_few(const NnAttention* a, int four_bits);
bool nnk_cache_few_fits(const NnAttention* a);
size_t nnk_cache_few_floats(const NnAttention* a);
bool nnk_cache_few_parted(const NnAttention* a);
void nnk_cache_few(const attn::Args& a, const cache::Pages& p, const NnAttention* d, float* ws, hipStream_t s,
    const char* what);
// Of many queries; over pages of 4 bits for bf16 alone.
bool nnk_cache_forward_plain(const attn::Args& a, const cache::Pages& p, bool half, hipStream_t s, const char* what);
bool nnk_cache_forward_mxfp4(const attn::Args& a, const cache::Pages& p, hipStream_t s, const char* what);
