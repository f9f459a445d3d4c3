// What the kernels of the 8-bit key / value cache share: the cache as a kernel sees it, its checks, and the batch's lookups.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>
#include <type_traits>

#include "tpb_internal.h"

namespace tpb_kv {

constexpr int64_t kMaxPagesInPool = 1 << 24;

// Words of tpb_kv_cache::scratch.
//   [0] number of page copies that the page operation leaves to its second kernel, [1] pages in use (compact)
//   marks [max_seqs], offsets [max_seqs], then two page lists of n_pages each: free pages or copy sources, and copy destinations
struct Scratch {
    int32_t *head, *marks, *offsets, *list_a, *list_b;
};
__host__ __device__ inline Scratch scratch_of(const tpb_kv_cache &c) {
    Scratch s;
    s.head = c.scratch;
    s.marks = c.scratch + 8;
    s.offsets = s.marks + c.max_seqs;
    s.list_a = s.offsets + c.max_seqs;
    s.list_b = s.list_a + c.n_pages;
    return s;
}

// The page of its sequence's row of the table that place x of an append's launch stands for, where the search gave sequence i: rows from r0 on, tokens
// first .. len - 1 new.  Its places begin at r0 / page_tokens + 2 i; -1: a place in front of them (rows ahead of the batch's first sequence: the search
// knows no earlier one) or behind its last page.
__host__ __device__ inline int page_at_place(int x, int i, int r0, int first, int len, int shift) {
    const int at = x - ((r0 >> shift) + 2 * i);
    const long long pg = (long long)(first >> shift) + at;
    return at >= 0 && (pg << shift) < len ? (int)pg : -1;
}

// codes of the handle's status word (tpb_status_poll): role 32 = a cache that does not fit the call
constexpr uint32_t kBadSeq = (32u << 24) | 1u, kBadPage = (32u << 24) | 2u, kBadLen = (32u << 24) | 3u, kBadTail = (32u << 24) | 4u;

int check_cache(tpb_handle_t h, const tpb_kv_cache *c, const char *what);   // the struct's own fields
int check_layer(tpb_handle_t h, const tpb_kv_cache *c, int layer, const char *what);

#ifdef __CUDACC__
__device__ __forceinline__ void report(uint32_t *status, uint32_t code) { atomicCAS(status, 0u, code); }

// An offset of the batch, clamped to the rows there are; data of other kernels of the stream, hence L2 loads.
__device__ __forceinline__ int row_offset(const int32_t *cu, int i, int rows) {
    const int v = __ldcg(cu + i);
    return v < 0 ? 0 : (v > rows ? rows : v);
}

// Which sequence of the batch: the last i in [0, n) with key(i, cu[i]) <= x, key ascending and the first key <= x; a whole warp calls it.  Up to 32
// sequences it is one round of loads that brings i's offsets and its id with it, up to 1024 two: these kernels' time for a
// decode step is their chain of loads.  With offsets out of order it still ends, at some i in [0, n).  seqs may be null.
struct Found {
    int i, r0, r1, seq;      // cu[i], cu[i + 1], seqs[i]
};
template <typename Key>
__device__ __forceinline__ Found find_sequence(const int32_t *cu, const int32_t *seqs, int n, int rows, int x, Key key) {
    const int lane = threadIdx.x & 31;
    int lo = 0, hi = n;
    while (hi - lo > 32) {
        const int step = (hi - lo + 31) / 32;
        const int i = lo + lane * step;
        const bool below = i < hi && (lane == 0 || key(i, row_offset(cu, i, rows)) <= x);
        lo += (__popc(__ballot_sync(0xffffffffu, below)) - 1) * step;
        hi = min(lo + step, hi);
    }
    const int j = min(lo + lane, hi - 1);
    const int a = row_offset(cu, j, rows), b = row_offset(cu, j + 1, rows), s = seqs ? __ldcg(seqs + j) : 0;
    const bool below = lo + lane < hi && (lane == 0 || key(j, a) <= x);
    const int c = __popc(__ballot_sync(0xffffffffu, below)) - 1;
    Found f;
    f.i = lo + c;
    f.r0 = __shfl_sync(0xffffffffu, a, c);
    f.r1 = __shfl_sync(0xffffffffu, b, c);
    f.seq = __shfl_sync(0xffffffffu, s, c);
    return f;
}

// Sixteen consecutive values, 16-byte aligned: loaded as they are (they may wait in half the registers that floats take) ...
template <typename T>
struct Raw16 {
    uint4 w[sizeof(T)];        // 16 * sizeof(T) bytes
};
template <typename T>
__device__ __forceinline__ void load_raw(const T *p, Raw16<T> &r) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T); i++) r.w[i] = __ldcg(reinterpret_cast<const uint4 *>(p) + i);
}
// ... and as floats
template <typename T>
__device__ __forceinline__ void values_of(const Raw16<T> &r, float (&v)[16]) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T); i++) {
        const uint32_t w[4] = {r.w[i].x, r.w[i].y, r.w[i].z, r.w[i].w};
#pragma unroll
        for (int e = 0; e < 4; e++) {
            if constexpr (sizeof(T) == 4) {
                v[4 * i + e] = __uint_as_float(w[e]);
            } else if constexpr (std::is_same<T, __half>::value) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[e]));
                v[8 * i + 2 * e] = f.x; v[8 * i + 2 * e + 1] = f.y;
            } else {
                v[8 * i + 2 * e] = __uint_as_float(w[e] << 16);
                v[8 * i + 2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
            }
        }
    }
}
template <typename T>
__device__ __forceinline__ void load16(const T *p, float (&v)[16]) {
    Raw16<T> r;
    load_raw(p, r);
    values_of(r, v);
}
template <typename T>
__device__ __forceinline__ void store16(T *p, const float (&v)[16]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 4; i++)
            reinterpret_cast<float4 *>(p)[i] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
    } else {
        uint32_t w[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            if constexpr (std::is_same<T, __half>::value) {
                const __half2 b = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
                w[i] = *reinterpret_cast<const uint32_t *>(&b);
            } else {
                const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
                w[i] = *reinterpret_cast<const uint32_t *>(&b);
            }
        }
        reinterpret_cast<uint4 *>(p)[0] = make_uint4(w[0], w[1], w[2], w[3]);
        reinterpret_cast<uint4 *>(p)[1] = make_uint4(w[4], w[5], w[6], w[7]);
    }
}

// The largest magnitude among sixteen values; NaN if one of them is.
template <typename T>
__device__ __forceinline__ float amax_of(const Raw16<T> &r) {
    if constexpr (sizeof(T) == 4) {
        float m = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t w[4] = {r.w[i].x, r.w[i].y, r.w[i].z, r.w[i].w};
#pragma unroll
            for (int e = 0; e < 4; e++) asm("max.NaN.f32 %0, %0, %1;" : "+f"(m) : "f"(fabsf(__uint_as_float(w[e]))));
        }
        return m;
    } else {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const uint32_t w[4] = {r.w[i].x, r.w[i].y, r.w[i].z, r.w[i].w};
#pragma unroll
            for (int e = 0; e < 4; e++) {
                if constexpr (std::is_same<T, __half>::value) asm("max.NaN.f16x2 %0, %0, %1;" : "+r"(m) : "r"(w[e] & 0x7fff7fffu));
                else asm("max.NaN.bf16x2 %0, %0, %1;" : "+r"(m) : "r"(w[e] & 0x7fff7fffu));
            }
        }
        float lo, hi, f;
        if constexpr (std::is_same<T, __half>::value) {
            const float2 x = __half22float2(*reinterpret_cast<const __half2 *>(&m));
            lo = x.x; hi = x.y;
        } else {
            lo = __uint_as_float(m << 16); hi = __uint_as_float(m & 0xffff0000u);
        }
        asm("max.NaN.f32 %0, %1, %2;" : "=f"(f) : "f"(lo), "f"(hi));
        return f;
    }
}

// the two e4m3 values of the low or high half of a word -> f16
template <int HALF>
__device__ __forceinline__ uint32_t e4m3_pair(uint32_t w) {
    uint32_t d;
    if (HALF == 0) asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}" : "=r"(d) : "r"(w));
    else asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, hi;\n\t}" : "=r"(d) : "r"(w));
    return d;
}
// One 32-bit word of four cached values.  int8: 2^23 + 128 + x has x ^ 0x80 in its lowest byte.
template <int FORMAT>
__device__ __forceinline__ void unpack4(uint32_t w, float *v) {
    if constexpr (FORMAT == TPB_KV_S8) {
        const uint32_t u = w ^ 0x80808080u;
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7440 | i)) - 8388736.0f;
    } else {
        const uint32_t h[2] = {e4m3_pair<0>(w), e4m3_pair<1>(w)};
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&h[i]));
            v[2 * i] = f.x; v[2 * i + 1] = f.y;
        }
    }
}
// Four quotients (value / scale) rounded to nearest even; at most the format's limit (e4m3 saturates there).  int8: adding 1.5 * 2^23
// rounds to a whole number, whose low byte the sum's low byte is.
template <int FORMAT>
__device__ __forceinline__ uint32_t pack4(const float *v) {
    if constexpr (FORMAT == TPB_KV_S8) {
        uint32_t m[4];
#pragma unroll
        for (int i = 0; i < 4; i++) m[i] = __float_as_uint(v[i] + 12582912.0f);
        return __byte_perm(__byte_perm(m[0], m[1], 0x0040), __byte_perm(m[2], m[3], 0x0040), 0x5410);
    } else {
        uint32_t d;
        asm("{\n\t.reg .b16 lo, hi;\n\tcvt.rn.satfinite.e4m3x2.f32 lo, %2, %1;\n\tcvt.rn.satfinite.e4m3x2.f32 hi, %4, %3;\n\tmov.b32 %0, {lo, hi};\n\t}"
            : "=r"(d) : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]));
        return d;
    }
}
#endif

}  // namespace tpb_kv
