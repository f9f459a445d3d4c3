// Writing the 8-bit key / value cache and reading it back.
//
// A block -- the tokens of one page, one head -- has one scale, a power of two, so that the quotients value / scale and old scale / new scale are exact
// in f32: quantising is one rounding (to int8, or to e4m3), and a block whose scale has to grow is rounded again by a shift.
#include <algorithm>

#include "kv_common.cuh"

using namespace tpb_kv;

namespace {

// The smallest power of two s >= 2^-100 with amax <= limit * s, amax finite: limit = top * 2^p, 1 <= top < 2, so s has amax's exponent less
// p, and one more where amax's mantissa is above top's.  At most 2^(127 - p): a larger one would let the largest f32 values round to 2^128; they
// saturate at limit * 2^(127 - p) instead.
template <int FORMAT>
__device__ __forceinline__ float pow2_scale(float amax) {
    constexpr int p = FORMAT == TPB_KV_S8 ? 6 : 8;                           // 127 = 0x1.fcp6, 448 = 0x1.cp8
    constexpr uint32_t top = FORMAT == TPB_KV_S8 ? 0x7e0000u : 0x600000u;
    const uint32_t b = __float_as_uint(amax);
    const int e = (int)(b >> 23) - 127 - p + ((b & 0x7fffffu) > top ? 1 : 0);  // a subnormal amax gives an e below -100
    return __uint_as_float((uint32_t)(min(max(e, -100), 127 - p) + 127) << 23);
}

template <int FORMAT>
constexpr float kLimit = FORMAT == TPB_KV_S8 ? 127.0f : 448.0f;

// One CTA per (sequence, page it touches) and some of the page's blocks (a head's keys or values): a group of 128 threads takes a block at a time, with up
// to CHUNKS pieces of 16 values a thread in registers, as they were loaded, between the maximum and the rounding, so that the input is read
// once.  Bound by HBM for prompts; for a decode step by its chain of loads -- offsets and id, length and tail, page, new values and old ones, 0.4 us
// each -- which is why one warp a CTA looks the sequence up, why a CTA of a prompt goes over several blocks behind one look-up, and why
// what a step of the chain brings is asked for before anything is decided.
//
// DENSE: 64 registers a thread, 1024 threads an SM whatever the block's size, for more CTAs than the SMs hold at 72 (two pieces, one CTA) or 96 (four pieces,
// three).  Measured with the rows read back: 8384 tokens in four prompts, 8 heads of 128, bf16 to e4m3, pages of 64 30.9 -> 27.7 us; 1541 tokens, which need
// no second round, 11.5, and 12.4 with it.  One piece a thread (pages of 16): a CTA of eight groups, or, with more pages than SMs, two of four,
// one of which looks up while the other copies: 38.5 -> 32.7 us; f32 45.9 -> 38.9.
//
// Grid x: sequence i has at least as many places as it can touch pages from cu[i] / page_tokens + 2 i on, so that a CTA finds its
// sequence by a search and the launch needs no lengths on the host.
template <int CHUNKS>
constexpr int kAppendGroups = CHUNKS <= 1 ? 8 : CHUNKS == 2 ? 4 : 2;
template <typename T, int FORMAT, int HD, int CHUNKS, bool DENSE>
__global__ void __launch_bounds__(128 * kAppendGroups<CHUNKS>, DENSE ? 8 / kAppendGroups<CHUNKS> : 1)
kv_append_kernel(const tpb_kv_cache c, int layer, const T *k, int64_t ld_k, const T *v, int64_t ld_v, const int32_t *seqs, const int32_t *cu,
                 int n_seqs, int rows, uint32_t *status) {
    constexpr int GROUPS = kAppendGroups<CHUNKS>;
    __shared__ float s_max[2][4 * GROUPS];
    __shared__ int s_found[5];              // i, cu[i], new tokens, id, length; length -1: nothing to do
    tpb_grid_dep_launch();
    tpb_grid_dep_wait();
    const int pt = c.page_tokens, shift = __ffs(pt) - 1, x = (int)blockIdx.x, t = (int)threadIdx.x & 127, group = (int)threadIdx.x >> 7;
    if (threadIdx.x < 32) {
        const Found b = find_sequence(cu, seqs, n_seqs, rows, x, [&](int j, int r) { return (r >> shift) + 2 * j; });
        const int n_new = b.r1 - b.r0;
        int len = -1;
        if (n_new > 0) {
            if (b.seq < 0 || b.seq >= c.max_seqs) {
                report(status, kBadSeq);
            } else {
                len = __ldcg(c.lens + b.seq);
                const int tail = __ldcg(c.tail + b.seq);
                if (len < n_new || (long long)len > (long long)c.max_pages * pt) {
                    report(status, kBadLen);
                    len = -1;
                } else if (tail != n_new) {
                    report(status, kBadTail);
                    len = -1;
                }
            }
        }
        if (threadIdx.x == 0) {
            s_found[0] = b.i;
            s_found[1] = b.r0;
            s_found[2] = n_new;
            s_found[3] = b.seq;
            s_found[4] = len;
        }
    }
    __syncthreads();
    const int r0 = s_found[1], n_new = s_found[2], seq = s_found[3], len = s_found[4];
    if (len < 0) return;
    const int first = len - n_new;
    const int pg = page_at_place(x, s_found[0], r0, first, len, shift);
    if (pg < 0) return;
    const int page = __ldcg(c.table + (size_t)seq * c.max_pages + pg);
    const int p0 = pg * pt;                                // position of the page's first slot
    const int held = max(first - p0, 0), fill = min(len - p0, pt);   // slots [0, held) hold earlier tokens, [held, fill) are written
    const int blocks = 2 * c.kv_heads, stride = (int)gridDim.y * (int)(blockDim.x >> 7);
    int flip = 0;
    for (int b0 = (int)blockIdx.y * (int)(blockDim.x >> 7); b0 < blocks; b0 += stride, flip ^= 1) {
        const int bi = b0 + group;
        const bool there = bi < blocks, is_v = bi >= c.kv_heads;
        const int head = there ? (is_v ? bi - c.kv_heads : bi) : 0;
        const int64_t ld = is_v ? ld_v : ld_k;
        const T *src = (is_v ? v : k) + (int64_t)(r0 + p0 - first) * ld + (int64_t)head * HD;   // + slot * ld
        Raw16<T> raw[CHUNKS];
#pragma unroll
        for (int j = 0; j < CHUNKS; j++) {
            const int slot = (j * 128 + t) / (HD / 16), d = (j * 128 + t) % (HD / 16) * 16;
            if (there && slot >= held && slot < fill) load_raw(src + (int64_t)slot * ld + d, raw[j]);
        }
        if (page < 0 || page >= c.n_pages) {
            report(status, kBadPage);
            return;
        }
        const size_t block = ((size_t)layer * c.n_pages + page) * c.kv_heads + head;
        uint4 *dst = reinterpret_cast<uint4 *>(static_cast<uint8_t *>(is_v ? c.v : c.k) + block * (size_t)(pt * HD));
        float *scale_at = (is_v ? c.v_scale : c.k_scale) + block;
        const float old = there && held > 0 ? __ldcg(scale_at) : 0.0f;
        float amax = 0.0f;
#pragma unroll
        for (int j = 0; j < CHUNKS; j++) {
            const int slot = (j * 128 + t) / (HD / 16);
            if (there && slot >= held && slot < fill) asm("max.NaN.f32 %0, %0, %1;" : "+f"(amax) : "f"(amax_of(raw[j])));
        }
        amax = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(amax)));       // non-negative floats order like their bits, NaN last
        if ((t & 31) == 0) s_max[flip][threadIdx.x >> 5] = amax;
        __syncthreads();                                        // also: everybody has the old scale before it is replaced
        if (!there) continue;
        const uint32_t *m = reinterpret_cast<const uint32_t *>(&s_max[flip][4 * group]);
        amax = __uint_as_float(max(max(m[0], m[1]), max(m[2], m[3])));
        const bool bad = !(amax <= 3.402823466e38f && old >= 0.0f && old <= 3.402823466e38f);
        const float scale = bad ? __uint_as_float(0x7fc00000u) : fmaxf(old, pow2_scale<FORMAT>(amax));
        if (t == 0) *scale_at = scale;
        // the quotient by a power of two is the product with its inverse; an old scale of the caller's own need not be one
        const bool pow2 = (__float_as_uint(scale) & 0x7fffffu) == 0;
        const float inv = pow2 ? 1.0f / scale : 0.0f, ratio = old / scale;
        const bool over = amax > kLimit<FORMAT> * scale;        // the largest f32 values saturate
#pragma unroll
        for (int j = 0; j < CHUNKS; j++) {
            const int slot = (j * 128 + t) / (HD / 16);
            if (slot < held) {
                if (scale == old || bad) continue;
                const uint4 before = __ldcg(dst + j * 128 + t);
                uint32_t u[4] = {before.x, before.y, before.z, before.w};
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    float f[4];
                    unpack4<FORMAT>(u[e], f);
#pragma unroll
                    for (int q = 0; q < 4; q++) f[q] *= ratio;
                    u[e] = pack4<FORMAT>(f);
                }
                dst[j * 128 + t] = make_uint4(u[0], u[1], u[2], u[3]);
            } else if (slot < fill) {
                uint32_t u[4] = {0u, 0u, 0u, 0u};
                if (!bad) {
                    float f[16];
                    values_of(raw[j], f);
                    if (pow2) {
#pragma unroll
                        for (int e = 0; e < 16; e++) f[e] *= inv;
                    } else {
#pragma unroll
                        for (int e = 0; e < 16; e++) f[e] = __fdiv_rn(f[e], scale);
                    }
                    if (over) {
#pragma unroll
                        for (int e = 0; e < 16; e++) f[e] = fminf(fmaxf(f[e], -kLimit<FORMAT>), kLimit<FORMAT>);
                    }
#pragma unroll
                    for (int e = 0; e < 4; e++) u[e] = pack4<FORMAT>(&f[4 * e]);
                }
                dst[j * 128 + t] = make_uint4(u[0], u[1], u[2], u[3]);
            }
        }
    }
}

// A warp a row: looks its sequence and page up and goes over it with 16 values a lane and step, keys and values, four steps' loads in flight.
// Measured: 8384 rows of 8 heads of 128, e4m3 to bf16, behind the append of the same: 27.3 us for both, 16 of them bytes at a copy's rate; with four CTAs an
// SM 28.2, with six 33 (the loads in flight no longer fit the registers); several rows a warp, one after the other: two 1 us more, four 9.
template <typename T, int FORMAT, int HD>
__global__ void __launch_bounds__(256, 5)
kv_read_kernel(const tpb_kv_cache c, int layer, T *k, int64_t ld_k, T *v, int64_t ld_v, const int32_t *seqs, const int32_t *start,
               const int32_t *cu, int n_seqs, int rows, uint32_t *status) {
    tpb_grid_dep_launch();
    tpb_grid_dep_wait();
    const int lane = threadIdx.x & 31, shift = __ffs(c.page_tokens) - 1;
    const int r = (int)blockIdx.x * 8 + (int)(threadIdx.x >> 5);
    if (r >= rows) return;
    const Found b = find_sequence(cu, seqs, n_seqs, rows, r, [&](int, int r0) { return r0; });
    if (b.r0 > r || b.r1 <= r) return;                       // a row of no sequence
    if (b.seq < 0 || b.seq >= c.max_seqs) {
        report(status, kBadSeq);
        return;
    }
    const int from = start ? __ldcg(start + b.i) : 0, len = __ldcg(c.lens + b.seq);
    const long long pos = (long long)from + (r - b.r0);
    const bool inside = from >= 0 && pos < len && pos < (long long)c.max_pages * c.page_tokens;       // behind the end: zeros
    int page = 0;
    if (inside) {
        page = __ldcg(c.table + (size_t)b.seq * c.max_pages + (pos >> shift));
        if (page < 0 || page >= c.n_pages) {
            report(status, kBadPage);
            return;
        }
    }
    const int pieces = c.kv_heads * (HD / 16), slot = (int)pos & (c.page_tokens - 1);
    const size_t block0 = ((size_t)layer * c.n_pages + page) * c.kv_heads;
    constexpr int kAhead = 4;
    for (int p0 = lane; p0 < 2 * pieces; p0 += 32 * kAhead) {
        uint4 w[kAhead];
        float scale[kAhead];
#pragma unroll
        for (int a = 0; a < kAhead; a++) {
            const int p = p0 + 32 * a;
            if (inside && p < 2 * pieces) {
                const bool is_v = p >= pieces;
                const int q = is_v ? p - pieces : p, head = q / (HD / 16), d = q % (HD / 16) * 16;
                scale[a] = __ldcg((is_v ? c.v_scale : c.k_scale) + block0 + head);
                w[a] = __ldcg(reinterpret_cast<const uint4 *>(static_cast<const uint8_t *>(is_v ? c.v : c.k) +
                                                              ((block0 + head) * c.page_tokens + slot) * HD + d));
            }
        }
#pragma unroll
        for (int a = 0; a < kAhead; a++) {
            const int p = p0 + 32 * a;
            if (p >= 2 * pieces) break;
            const bool is_v = p >= pieces;
            const int q = is_v ? p - pieces : p;
            float f[16] = {};
            if (inside) {
                const uint32_t u[4] = {w[a].x, w[a].y, w[a].z, w[a].w};
#pragma unroll
                for (int i = 0; i < 4; i++) unpack4<FORMAT>(u[i], &f[4 * i]);
#pragma unroll
                for (int i = 0; i < 16; i++) f[i] *= scale[a];
            }
            store16((is_v ? v + (int64_t)r * ld_v : k + (int64_t)r * ld_k) + (int64_t)q * 16, f);
        }
    }
}

int check_batch(tpb_handle_t h, const char *what, const tpb_kv_cache *c, const void *k, int64_t ld_k, const void *v, int64_t ld_v, int dtype,
                const int32_t *seqs, const int32_t *cu, int n_seqs, int64_t rows) {
    TPB_CHECK_ARG(h, dtype == TPB_F32 || dtype == TPB_BF16 || dtype == TPB_F16, "%s: rows must be f32, bf16 or f16", what);
    TPB_CHECK_ARG(h, n_seqs >= 0 && n_seqs < (1 << 24) && rows >= 0 && rows < (1 << 26), "%s: bad n_seqs / rows", what);
    if (n_seqs == 0 || rows == 0) return TPB_OK;
    TPB_CHECK_ARG(h, k && v && seqs && cu, "%s: null pointer", what);
    const int64_t width = (int64_t)c->kv_heads * c->head_dim, mult = dtype == TPB_F32 ? 4 : 8;
    TPB_CHECK_ARG(h, ld_k >= width && ld_v >= width && ld_k % mult == 0 && ld_v % mult == 0,
                  "%s: ld_k and ld_v must be at least kv_heads * head_dim and multiples of %lld", what, (long long)mult);
    TPB_CHECK_ARG(h, tpb_aligned16(k) && tpb_aligned16(v), "%s: k and v must be 16-byte aligned", what);
    TPB_CHECK_ARG(h, ((reinterpret_cast<uintptr_t>(seqs) | reinterpret_cast<uintptr_t>(cu)) & 3u) == 0, "%s: seqs and cu must be 4-byte aligned", what);
    return TPB_OK;
}

// Calls f with a null T * for the dtype of the rows.
template <typename F>
cudaError_t by_dtype(int dtype, F f) {
    return dtype == TPB_F32 ? f((float *)nullptr) : dtype == TPB_BF16 ? f((__nv_bfloat16 *)nullptr) : f((__half *)nullptr);
}

}  // namespace

extern "C" {

int tpb_kv_append(tpb_handle_t h, tpb_stream_t stream, const tpb_kv_cache *c, int layer, const void *k, int64_t ld_k, const void *v,
                  int64_t ld_v, int dtype, const int32_t *seqs, const int32_t *cu, int n_seqs, int64_t rows) {
    if (!h) return TPB_ERR_INVALID_ARG;
    int rc = check_layer(h, c, layer, "kv_append");
    if (rc == TPB_OK) rc = check_batch(h, "kv_append", c, k, ld_k, v, ld_v, dtype, seqs, cu, n_seqs, rows);
    if (rc != TPB_OK || n_seqs == 0 || rows == 0) return rc;
    tpb_device_guard guard(h->device);
    TPB_CUDA(h, guard.err);
    const cudaError_t e = by_dtype(dtype, [&](auto *tag) {
        using T = std::remove_pointer_t<decltype(tag)>;
        const int64_t items = rows / c->page_tokens + 2 * (int64_t)n_seqs;
        // as many CTAs a page as two rounds of two an SM have room for: with more, each waits through a look-up of its own
        const auto ctas_of = [&](int groups) {
            const int rounds = (2 * c->kv_heads + groups - 1) / groups;
            return std::max<int64_t>(1, std::min<int64_t>(rounds, 4 * (int64_t)h->sm_count / items));
        };
        const auto launch = [&](auto kern, int groups) {
            return tpb_launch_pdl(kern, dim3((unsigned)items, (unsigned)ctas_of(groups)), dim3(128u * (unsigned)groups), 0, (cudaStream_t)stream, *c, layer,
                                  (const T *)k, ld_k, (const T *)v, ld_v, seqs, cu, n_seqs, (int)rows, h->d_status);
        };
        const auto by_chunks = [&](auto fmt) {
            constexpr int F = decltype(fmt)::value;
            const int chunks = c->page_tokens * c->head_dim / 2048;             // 0 (half the threads have a piece) .. 4
            const auto by_load = [&](auto hd, auto n) {
                constexpr int HD = decltype(hd)::value, N = decltype(n)::value, G = kAppendGroups<N>;
                if constexpr (N == 1) return launch(kv_append_kernel<T, F, HD, 1, false>, items > h->sm_count ? G / 2 : G);
                else if constexpr (sizeof(T) == 4) return launch(kv_append_kernel<T, F, HD, N, false>, G);
                else return items * ctas_of(G) > (N == 2 ? 1 : 3) * (int64_t)h->sm_count ? launch(kv_append_kernel<T, F, HD, N, true>, G)
                                                                                       : launch(kv_append_kernel<T, F, HD, N, false>, G);
            };
            const std::integral_constant<int, 1> one;
            const std::integral_constant<int, 2> two;
            if (c->head_dim == 64) return chunks <= 1 ? by_load(std::integral_constant<int, 64>{}, one) : by_load(std::integral_constant<int, 64>{}, two);
            const std::integral_constant<int, 128> hd;
            return chunks <= 1 ? by_load(hd, one) : chunks <= 2 ? by_load(hd, two) : by_load(hd, std::integral_constant<int, 4>{});
        };
        return c->format == TPB_KV_S8 ? by_chunks(std::integral_constant<int, TPB_KV_S8>{}) : by_chunks(std::integral_constant<int, TPB_KV_E4M3>{});
    });
    TPB_CUDA(h, e);
    return TPB_OK;
}

int tpb_kv_read(tpb_handle_t h, tpb_stream_t stream, const tpb_kv_cache *c, int layer, void *k, int64_t ld_k, void *v, int64_t ld_v,
                int dtype, const int32_t *seqs, const int32_t *start, const int32_t *cu, int n_seqs, int64_t rows) {
    if (!h) return TPB_ERR_INVALID_ARG;
    int rc = check_layer(h, c, layer, "kv_read");
    if (rc == TPB_OK) rc = check_batch(h, "kv_read", c, k, ld_k, v, ld_v, dtype, seqs, cu, n_seqs, rows);
    if (rc != TPB_OK || n_seqs == 0 || rows == 0) return rc;
    TPB_CHECK_ARG(h, (reinterpret_cast<uintptr_t>(start) & 3u) == 0, "kv_read: start must be 4-byte aligned");
    tpb_device_guard guard(h->device);
    TPB_CUDA(h, guard.err);
    const cudaError_t e = by_dtype(dtype, [&](auto *tag) {
        using T = std::remove_pointer_t<decltype(tag)>;
        const auto launch = [&](auto kern) {
            return tpb_launch_pdl(kern, dim3((unsigned)((rows + 7) / 8)), dim3(256), 0, (cudaStream_t)stream, *c, layer, (T *)k, ld_k, (T *)v, ld_v, seqs, start,
                                  cu, n_seqs, (int)rows, h->d_status);
        };
        if (c->format == TPB_KV_S8) return c->head_dim == 64 ? launch(kv_read_kernel<T, TPB_KV_S8, 64>) : launch(kv_read_kernel<T, TPB_KV_S8, 128>);
        return c->head_dim == 64 ? launch(kv_read_kernel<T, TPB_KV_E4M3, 64>) : launch(kv_read_kernel<T, TPB_KV_E4M3, 128>);
    });
    TPB_CUDA(h, e);
    return TPB_OK;
}

}  // extern "C"
