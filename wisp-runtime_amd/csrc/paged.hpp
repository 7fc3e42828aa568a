// The paged K/V cache of several sequences, as the kernels of kv_append.hip and paged_attn.hip see it.
//
// kc and vc are [pages][Hk][page][D] with any strides between pages, heads and rows (the same for both; a row's D values
// are contiguous). Position p of sequence b is row p % page of page table[b][p / page]. Lengths and tables are read on
// the device, so captured graphs follow them; nothing on the host knows them. What they say is checked where it is used:
// a page id outside [0, pages) or a position past the table's width is never dereferenced (bad page, below).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "wisp_internal.hpp"

namespace wisp {

struct PagedKV {
    uint8_t* kc;
    uint8_t* vc;
    int64_t ps, hs, rs;  // page, head and row strides in bytes
    int pages, shift;    // pages in the cache; log2 of the positions per page
};

// p[i] for an i that all lanes share, as a scalar load: cu, kv_len and table do not change while a kernel runs. (As a vector
// load it would count, and be awaited, together with the direct loads to LDS that are in flight.)
__device__ __forceinline__ int scalar_at(const int* p, int i) {
    return *(const __attribute__((address_space(4))) int*)(uintptr_t)(p + __builtin_amdgcn_readfirstlane(i));
}

// Byte offset of position pos of the sequence whose table row is trow (width entries); bad where there is none.
__device__ __forceinline__ int64_t page_offset(const PagedKV& kv, const int* __restrict__ trow, int width, int pos, bool& bad) {
    const int i = pos >> kv.shift;
    const int id = i < width ? trow[i] : -1;
    const bool ok = (unsigned)id < (unsigned)kv.pages;
    bad = bad || !ok;
    return (ok ? (int64_t)id : 0) * kv.ps + (int64_t)(pos & ((1 << kv.shift) - 1)) * kv.rs;
}

// A sequence's length, inside what its table can hold; bad where kv_len says more.
__device__ __forceinline__ int held(int len, int width, int shift, bool& bad) {
    const int cap = width << shift;
    bad = bad || len > cap;
    return min(max(len, 0), cap);
}

// Inclusive sum of v over the lanes up to this one: four DPP shifts in each row of 16, then the row totals handed on.
__device__ __forceinline__ int wave_scan(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);  // row_shr:1
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);  // row_shr:2
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);  // row_shr:4
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);  // row_shr:8
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);  // row_bcast:15 into rows 1 and 3
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);  // row_bcast:31 into rows 2 and 3
    return v;
}

// x / d for x >= 0, d >= 1 and a quotient below 2^20: that of floats is off by one at most.
__device__ __forceinline__ int small_div(int x, int d) {
    int q = (int)((float)x * __builtin_amdgcn_rcpf((float)d));
    const int r = x - q * d;
    if (r < 0) --q;
    if (r >= d) ++q;
    return q;
}

// Sequence b's tokens in a pack: rows [lo, hi) of cu, kept inside [0, T] whatever cu holds.
__device__ __forceinline__ void token_range(const int* __restrict__ cu, int b, int T, int& lo, int& hi) {
    lo = min(max(cu[b], 0), T);
    hi = min(max(cu[b + 1], lo), T);
}

// What every entry point of the cache checks.
inline int check_paged(const void* kc, const void* vc, int64_t pages, int page, int64_t page_stride, int64_t head_stride,
                       int64_t row_stride, int width, int B, int hq, int hk, int d, int dtype) {
    if (dtype != WISP_DT_BF16 && dtype != WISP_DT_F16) return fail_inval("dtype must be bfloat16 or float16");
    if (d != 64 && d != 128 && d != 256) return fail_inval("head dim must be 64, 128 or 256");
    if (hk < 1 || hq < hk || hq % hk || hq > 1024) return fail_inval("hq must be a positive multiple of hk, at most 1024");
    if (page < 16 || page > (1 << 20) || (page & (page - 1))) return fail_inval("page must be a power of two in [16, 2^20]");
    if (pages < 1 || pages > 0x7FFFFFFF) return fail_inval("the cache needs at least one page");
    if (B < 1 || B > (1 << 20)) return fail_inval("B must be in [1, 2^20]");
    if (width < 1 || (int64_t)width * page > (1 << 30)) return fail_inval("the table's positions must be in [1, 2^30]");
    if (!kc || !vc) return fail_inval("null cache");
    if (row_stride < d || head_stride < 0 || page_stride < 0) return fail_inval("cache strides");
    if (row_stride >= (1 << 23)) return fail_inval("the cache's row stride must be below 2^23 elements");
    if (!aligned(kc, 16) || !aligned(vc, 16) || page_stride % 8 || head_stride % 8 || row_stride % 8) {
        set_error("the caches and their strides must be 16-byte aligned");
        return WISP_EALIGN;
    }
    return WISP_OK;
}
inline PagedKV paged_kv(void* kc, void* vc, int64_t pages, int page, int64_t page_stride, int64_t head_stride,
                        int64_t row_stride) {
    int shift = 0;
    while ((1 << shift) < page) ++shift;
    return PagedKV{(uint8_t*)kc, (uint8_t*)vc, 2 * page_stride, 2 * head_stride, 2 * row_stride, (int)pages, shift};
}

}  // namespace wisp
