// Attention of a sequence's last tokens over its 8-bit cache, in pages: the decode step's attention, and that of a few drafted tokens.
//
//   out[r] = sum_j softmax_j(scale q[r] . k[j]) v[j],   k = ks * qk, v = vs * qv with one scale a page and head
//
// Bound by the cache's bytes, which are read once: 2 * head_dim a token and kv head.  What carries that:
//   - All query rows that share a kv head (tokens x heads of the group) are one operand of mma.sync m16n8k16 (f16, f32 sums).  The
//     cached values are exact in f16.  A tcgen05 tile would have 128 rows where a decode step has 1 to 32; a row is the other operand's cost here.
//   - f32 accuracy (SPLIT): a row takes two of the sixteen, q = hi + lo in f16 (after scaling the row by a power of two), and the weights
//     likewise; a group of up to eight rows leaves the second half of the tile empty anyway.  bf16 queries are exact in one f16 term, and
//     weights of one f16 term (2^-12) are below a bf16 result's half step (2^-9): no split there, sixteen rows a tile.
//   - Page scales are uniform over a step of 16 tokens (a page holds 16, 32 or 64): ks multiplies scores, vs the weights.
//   - A warp owns its data path: 16 tokens of K and V a step by cp.async into a ring of its own, no barrier between warps.  Bytes lie in shared
//     memory with their 16-byte pieces permuted so that K's 16-byte reads and V's 4-byte reads are free of bank conflicts; the
//     order of dimensions within the products is the one in which a thread finds its bytes, and q is laid out to match.
//   - The work of all (sequence, kv head, row tile)s is one line of units of 64 tokens, cut into equal pieces, one a CTA.  A CTA that has
//     not all of a sequence's tokens leaves a partial result; a second kernel joins them in the order of the tokens, so the
//     result is the same from run to run.
//
// Softmax.  Per row two running references, both whole numbers in log2 units so that every rescaling is exact: ms >= max s - kLazy for the sum
// l = sum 2^(s - ms), and mw for the weights w = 2^(s - mw + kUp) vs, whose size depends on the page's scale as well.
#include "kv_common.cuh"

using namespace tpb_kv;

namespace {

constexpr int kThreads = 128;
constexpr int kWarps = 4;
constexpr int kUnit = 64;            // tokens of a unit of work: one step of every warp
constexpr int kStep = 16;            // tokens of a warp's step
constexpr int kMinUnits = 4;         // a CTA takes at least so many units: shorter pieces cost more in joining than they gain
constexpr int kRing = 16384;         // bytes of a warp's ring
constexpr float kLazy = 6.0f, kUp = 6.0f;      // w < 2^(kLazy + kUp + 1) fits f16

template <int HD, bool SPLIT, int MT>
struct Cfg {
    static constexpr int kRows = (SPLIT ? 8 : 16) * MT;                  // rows of a tile
    static constexpr int kStageBytes = 2 * kStep * HD;
    static constexpr int kStages = kRing / kStageBytes;                  // 4 (head_dim 128) or 8
    static constexpr int kSteps = HD / 16;                               // k steps of q k^T
    static constexpr int kQf = MT > 1 ? MT * kSteps * 32 * 16 : 0;       // q's fragments in shared memory (MT = 1: in registers)
    static constexpr int kSmem = kWarps * kRing + kQf;
    static constexpr int kMergeLd = kRows * (HD + 4) * 4 <= kRing ? HD + 4 : HD;      // a warp's sums lie over its ring on their way to the others
    static_assert(kRows * kMergeLd * 4 <= kRing && kRows <= 32, "sums fit the ring and a slot");
    static constexpr int kCtas = MT == 1 ? 3 : 2;                        // per SM
};
constexpr int kMaxCtas = 3, kMaxRows = 32;

struct Part {       // where a CTA's partial results lie: two slots a CTA
    float *o, *ms, *l, *mw;
};
__host__ __device__ inline size_t slot_floats(int hd) { return (size_t)kMaxRows * (hd + 3); }
__device__ __forceinline__ Part part_of(float *ws, int hd, int cta, int which) {
    Part p;
    p.o = ws + ((size_t)2 * cta + which) * slot_floats(hd);
    p.ms = p.o + (size_t)kMaxRows * hd;
    p.l = p.ms + kMaxRows;
    p.mw = p.l + kMaxRows;
    return p;
}

struct AttnParams {
    tpb_kv_cache c;
    int layer, dtype;
    void *out;
    const void *q;
    long long ld_out, ld_q;
    const int32_t *seqs, *cu;
    int n_seqs, rows, heads, group;
    float scale_log2;
    int whole;                           // sequences are not cut: a unit is all of one
    float *ws;
    uint32_t *status;
};

// ---- the line of units ------------------------------------------------------------------------
// Chunk of kThreads sequences of the batch in shared memory: first unit, length, rows.
struct Chunk {
    long long start[kThreads + 1];
    int len[kThreads], row0[kThreads], n_q[kThreads], seq[kThreads];
    long long warp_sum[kThreads / 32];
};
__device__ __forceinline__ int tiles_of(const AttnParams &p, int len) { return p.whole ? 1 : max(1, (len + kUnit - 1) / kUnit); }

// Loads sequences base .. base + kThreads - 1, the first of which begins at unit `cum`; returns the unit behind the last.  `tell`: report ids and
// lengths out of range (such a sequence has no units: its rows are not written).
template <int RT>
__device__ long long load_chunk(const AttnParams &p, Chunk &ck, int base, long long cum, bool tell) {
    const int i = base + (int)threadIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    long long units = 0;
    int len = 0, row0 = 0, n_q = 0, seq = -1;
    if (i < p.n_seqs && threadIdx.x < kThreads) {
        seq = __ldcg(p.seqs + i);
        row0 = row_offset(p.cu, i, p.rows);
        n_q = row_offset(p.cu, i + 1, p.rows) - row0;
        if (n_q > 0) {
            if (seq < 0 || seq >= p.c.max_seqs) {
                if (tell) report(p.status, kBadSeq);
            } else {
                len = __ldcg(p.c.lens + seq);
                if (len < 0 || (long long)len > (long long)p.c.max_pages * p.c.page_tokens) {
                    if (tell) report(p.status, kBadLen);
                } else {
                    units = (long long)tiles_of(p, len) * p.c.kv_heads * (((long long)n_q * p.group + RT - 1) / RT);
                }
            }
        }
    }
    long long inc = units;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long t = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += t;
    }
    __syncthreads();                     // the last user of the chunk is done
    if (warp < kThreads / 32 && lane == 31) ck.warp_sum[warp] = inc;
    __syncthreads();
    long long at = cum, total = cum;
    for (int w = 0; w < kThreads / 32; w++) {
        if (w < warp) at += ck.warp_sum[w];
        total += ck.warp_sum[w];
    }
    if (threadIdx.x < kThreads) {
        ck.start[threadIdx.x] = at + inc - units;
        ck.len[threadIdx.x] = len;
        ck.row0[threadIdx.x] = row0;
        ck.n_q[threadIdx.x] = n_q;
        ck.seq[threadIdx.x] = seq;
        if (threadIdx.x == kThreads - 1) ck.start[kThreads] = total;
    }
    __syncthreads();
    return total;
}
// The sequence of the loaded chunk that holds unit u, start[0] <= u < start[kThreads].
__device__ __forceinline__ int find_in_chunk(const Chunk &ck, long long u) {
    int lo = 0, hi = kThreads;           // start[lo] <= u < start[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (ck.start[mid] <= u) lo = mid;
        else hi = mid;
    }
    return lo;
}
// One run of units of one (sequence, kv head, row tile).
struct Segment {
    int idx;                             // in the chunk
    int head, row_tile, t0, t1, tiles;   // tiles [t0, t1) of `tiles`
    long long first;                     // unit of tile 0
};
template <int RT>
__device__ __forceinline__ Segment segment_at(const AttnParams &p, const Chunk &ck, long long u, long long u_end) {
    Segment s;
    s.idx = find_in_chunk(ck, u);
    s.tiles = tiles_of(p, ck.len[s.idx]);
    const long long rel = u - ck.start[s.idx];
    const long long which = rel / s.tiles;
    s.t0 = (int)(rel - which * s.tiles);
    s.t1 = (int)min((long long)s.tiles, s.t0 + (u_end - u));
    const int row_tiles = (int)(((long long)ck.n_q[s.idx] * p.group + RT - 1) / RT);
    s.head = (int)(which / row_tiles);
    s.row_tile = (int)(which - (long long)s.head * row_tiles);
    s.first = u - s.t0;
    return s;
}
__device__ __forceinline__ long long units_per_cta(const AttnParams &p, long long total, int ctas) {
    return max((total + ctas - 1) / ctas, (long long)(p.whole ? 1 : kMinUnits));
}

// ---- arithmetic -------------------------------------------------------------------------------
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float pow2i(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }       // -126 <= e <= 127
__device__ __forceinline__ void mma(float (&d)[4], const uint4 &a, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t half2_bits(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}
// two floats as a pair of f16 terms: x = hi + lo up to 2^-22 of x, or 2^-25
__device__ __forceinline__ void split2(float a, float b, uint32_t &hi, uint32_t &lo) {
    const __half2 h = __floats2half2_rn(a, b);
    const float2 f = __half22float2(h);
    hi = *reinterpret_cast<const uint32_t *>(&h);
    lo = half2_bits(a - f.x, b - f.y);
}
// int8 pairs in the low bytes of both halves -> f16: 0x6400 | (x ^ 0x80) is 1024 + 128 + x
__device__ __forceinline__ uint32_t s8_pair(uint32_t w) {
    uint32_t b;
    asm("lop3.b32 %0, %1, %2, %3, 0x6a;" : "=r"(b) : "r"(w), "r"(0x00ff00ffu), "r"(0x64806480u));     // (w & mask) ^ bias
    const __half2 h = __hsub2(*reinterpret_cast<const __half2 *>(&b), __half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480)));
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t e4m3_pair(uint32_t two) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)two, __NV_E4M3);
    return (uint32_t)h.x | ((uint32_t)h.y << 16);
}
// Four consecutive bytes of K as the two registers of a k step: (bytes 0, 2), (1, 3) of s8, (0, 1), (2, 3) of e4m3.
template <int FORMAT>
__device__ __forceinline__ void k_regs(uint32_t w, uint32_t &b0, uint32_t &b1) {
    if constexpr (FORMAT == TPB_KV_S8) {
        b0 = s8_pair(w);
        b1 = s8_pair(w >> 8);
    } else {
        b0 = e4m3_pair(w & 0xffffu);
        b1 = e4m3_pair(w >> 16);
    }
}
// Four columns of V for two tokens: v[e] = (a's byte e, b's byte e).
template <int FORMAT>
__device__ __forceinline__ void v_regs(uint32_t a, uint32_t b, uint32_t (&v)[4]) {
    if constexpr (FORMAT == TPB_KV_S8) {
        v[0] = s8_pair(__byte_perm(a, b, 0x0400));
        v[1] = s8_pair(__byte_perm(a, b, 0x0501));
        v[2] = s8_pair(__byte_perm(a, b, 0x0602));
        v[3] = s8_pair(__byte_perm(a, b, 0x0703));
    } else {
        const uint32_t lo = __byte_perm(a, b, 0x5140), hi = __byte_perm(a, b, 0x7362);
        v[0] = e4m3_pair(lo & 0xffffu);
        v[1] = e4m3_pair(lo >> 16);
        v[2] = e4m3_pair(hi & 0xffffu);
        v[3] = e4m3_pair(hi >> 16);
    }
}

// Which token of its eight a column of the score tile is.  Chosen so that neighbouring columns (K: eight threads read 16 bytes each) and
// the even and the odd columns (V: four tokens x eight words) lie in different banks.
template <int HD>
__device__ __forceinline__ int token_of_col(int c) {
    const int t = c >> 1;
    if (HD == 64) return c & 1 ? 4 + (t ^ 1) : t;
    return c & 1 ? ((2 * t) ^ 4) | 1 : 2 * t;
}
// Byte of a step's K or V half at which 16-byte piece `piece` of token `tok` lies.
template <int HD>
__device__ __forceinline__ int piece_at(int tok, int piece) {
    if (HD == 64) return tok * 64 + ((piece ^ (((tok >> 1) & 1) << 1)) << 4);
    return tok * HD + ((piece ^ (tok & 7)) << 4);
}
__device__ __forceinline__ uint32_t smem_addr(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void cp16(uint32_t dst, const void *src, int bytes) {     // bytes 16, or 0: zeros
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ uint32_t lds32(uint32_t a) {
    uint32_t v;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ uint4 lds128(uint32_t a) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
    return v;
}

// q's values for one lane: 16 consecutive dimensions of a row (zeros for a row that is not there)
__device__ __forceinline__ void load_q(const AttnParams &p, int hd, long long row, int head, int d, bool there, float (&v)[16]) {
    if (!there) {
#pragma unroll
        for (int i = 0; i < 16; i++) v[i] = 0.0f;
        return;
    }
    const long long at = row * p.ld_q + (long long)head * hd + d;
    if (p.dtype == TPB_F32) load16(static_cast<const float *>(p.q) + at, v);
    else if (p.dtype == TPB_BF16) load16(static_cast<const __nv_bfloat16 *>(p.q) + at, v);
    else load16(static_cast<const __half *>(p.q) + at, v);
}
__device__ __forceinline__ void store4(const AttnParams &p, long long at, float a, float b, float c, float d) {
    if (p.dtype == TPB_F32) {
        *reinterpret_cast<float4 *>(static_cast<float *>(p.out) + at) = make_float4(a, b, c, d);
    } else if (p.dtype == TPB_BF16) {
        const __nv_bfloat162 x = __floats2bfloat162_rn(a, b), y = __floats2bfloat162_rn(c, d);
        *reinterpret_cast<uint2 *>(static_cast<__nv_bfloat16 *>(p.out) + at) =
            make_uint2(*reinterpret_cast<const uint32_t *>(&x), *reinterpret_cast<const uint32_t *>(&y));
    } else {
        *reinterpret_cast<uint2 *>(static_cast<__half *>(p.out) + at) = make_uint2(half2_bits(a, b), half2_bits(c, d));
    }
}

// What a row's parts (ms, l, mw, o) add up to: the factor of a part whose reference is m where the largest is big (m may be -inf: nothing seen)
__device__ __forceinline__ float part_factor(float m, float big) { return m == big ? 1.0f : ex2(m - big); }
// (o / l) 2^(mw - kUp - ms); zero for a row that sees nothing.  The power of two may lie outside f32 while the result does not: two steps.
__device__ __forceinline__ float finish_scale(float ms, float l, float mw, float &second) {
    second = 1.0f;
    if (l == 0.0f) return 0.0f;
    const float e = mw - kUp - ms;
    if (!(e >= -250.0f && e <= 250.0f)) return e < 0.0f ? 0.0f : 1.0f / l * e;        // mw = -inf: no weight at all; NaN stays NaN
    const float h = floorf(0.5f * e);
    second = ex2(h);
    return ex2(e - h) / l;
}

template <int HD, int FORMAT, bool SPLIT, int MT>
__global__ void __launch_bounds__(kThreads, Cfg<HD, SPLIT, MT>::kCtas)
kv_attention_kernel(const AttnParams p) {
    using C = Cfg<HD, SPLIT, MT>;
    constexpr int RT = C::kRows;
    constexpr int R = SPLIT ? 1 : 2;                       // rows a thread has per m tile: g, and g + 8
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ Chunk ck;
    __shared__ float s_ms[kWarps][RT], s_l[kWarps][RT], s_mw[kWarps][RT], s_rs[MT > 1 ? RT : 1];
    tpb_grid_dep_wait();
    tpb_grid_dep_launch();                                 // behind the wait: the join may look at lengths as soon as it starts
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;

    long long total = 0;
    for (int base = 0; base < p.n_seqs; base += kThreads) total = load_chunk<RT>(p, ck, base, total, blockIdx.x == 0);
    const long long per = units_per_cta(p, total, (int)gridDim.x);
    long long u = per * blockIdx.x;
    const long long u_end = min(u + per, total);
    if (u >= u_end) return;
    int base = 0;
    if (p.n_seqs > kThreads) {
        long long behind = load_chunk<RT>(p, ck, 0, 0, false);
        while (u >= behind) {
            base += kThreads;
            behind = load_chunk<RT>(p, ck, base, behind, false);
        }
    }

    const uint32_t ring = smem_addr(smem) + warp * kRing;
    uint4 *qf_smem = reinterpret_cast<uint4 *>(smem + kWarps * kRing);
    while (u < u_end) {
        while (u >= ck.start[kThreads]) {
            base += kThreads;
            load_chunk<RT>(p, ck, base, ck.start[kThreads], false);
        }
        const Segment s = segment_at<RT>(p, ck, u, u_end);
        const int len = ck.len[s.idx], n_q = ck.n_q[s.idx], row0 = ck.row0[s.idx], seq = ck.seq[s.idx];
        const int n_rows = n_q * p.group - s.row_tile * RT;           // of this tile, if below RT
        const auto token_row = [&](int r) { return (s.row_tile * RT + r) / p.group; };      // which of the sequence's queries row r belongs to

        // ---- q: scaled by a power of two to a largest value in [2^10, 2^11), as f16 terms ----
        uint4 qf[MT == 1 ? C::kSteps : 1];
        float rs[R];                                                  // MT = 1: scale log2(e) / that power
        const auto build_q = [&](int mt, uint4 *dst, int stride, float (&r_s)[R]) {
            float v[R][HD / 64][16];
#pragma unroll
            for (int e = 0; e < R; e++) {
                const int r = mt * (SPLIT ? 8 : 16) + g + 8 * e;
                const int flat = s.row_tile * RT + r, tok = flat / p.group;
                float amax = 0.0f;
#pragma unroll
                for (int cc = 0; cc < HD / 64; cc++) {
                    load_q(p, HD, row0 + tok, s.head * p.group + flat - tok * p.group, 16 * (t + 4 * cc), r < n_rows, v[e][cc]);
#pragma unroll
                    for (int i = 0; i < 16; i++) amax = fmaxf(amax, fabsf(v[e][cc][i]));
                }
                amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
                amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
                const int ex = max((int)(__float_as_uint(amax) >> 23) - 127, -116);       // 0: all zero, or below 2^-116
                const float up = pow2i(min(10 - ex, 126));
                r_s[e] = p.scale_log2 * pow2i(max(ex - 10, -126));
#pragma unroll
                for (int cc = 0; cc < HD / 64; cc++)
#pragma unroll
                    for (int i = 0; i < 16; i++) v[e][cc][i] *= up;
            }
#pragma unroll
            for (int cc = 0; cc < HD / 64; cc++)
#pragma unroll
                for (int k4 = 0; k4 < 4; k4++) {
                    // the pairs in which a thread finds K's bytes
                    constexpr int i1 = FORMAT == TPB_KV_S8 ? 2 : 1, i2 = FORMAT == TPB_KV_S8 ? 1 : 2;
                    uint4 a;
                    if (SPLIT) {
                        split2(v[0][cc][4 * k4], v[0][cc][4 * k4 + i1], a.x, a.y);
                        split2(v[0][cc][4 * k4 + i2], v[0][cc][4 * k4 + 3], a.z, a.w);
                    } else {
                        a.x = half2_bits(v[0][cc][4 * k4], v[0][cc][4 * k4 + i1]);
                        a.y = half2_bits(v[R - 1][cc][4 * k4], v[R - 1][cc][4 * k4 + i1]);
                        a.z = half2_bits(v[0][cc][4 * k4 + i2], v[0][cc][4 * k4 + 3]);
                        a.w = half2_bits(v[R - 1][cc][4 * k4 + i2], v[R - 1][cc][4 * k4 + 3]);
                    }
                    dst[(cc * 4 + k4) * stride] = a;
                }
        };
        if constexpr (MT == 1) {
            build_q(0, qf, 1, rs);
        } else {
            for (int mt = warp; mt < MT; mt += kWarps) {
                float r_s[R];
                build_q(mt, qf_smem + mt * C::kSteps * 32 + lane, 32, r_s);
#pragma unroll
                for (int e = 0; e < R; e++)
                    if (t == 0) s_rs[mt * (SPLIT ? 8 : 16) + g + 8 * e] = r_s[e];
            }
            __syncthreads();
        }

        // ---- the sequence's tokens [tok0, tok1), 16 a step, every fourth step this warp's ----
        const int tok0 = s.t0 * kUnit, tok1 = p.whole ? len : min(s.t1 * kUnit, len);
        const int n_steps = tok1 > tok0 + warp * kStep ? (tok1 - tok0 - warp * kStep + kUnit - 1) / kUnit : 0;
        const auto step_tok = [&](int n) { return tok0 + n * kUnit + warp * kStep; };
        const int32_t *row = p.c.table + (size_t)seq * p.c.max_pages;
        // pages and scales of 32 steps, a step a lane, and of the 32 behind them
        struct Ahead {
            int page;
            float ks, vs;
        };
        const auto look = [&](int n0) {
            Ahead a;
            a.page = -1;
            a.ks = a.vs = 0.0f;
            if (n0 + lane < n_steps) {
                a.page = __ldcg(row + step_tok(n0 + lane) / p.c.page_tokens);
                if (a.page < 0 || a.page >= p.c.n_pages) {
                    report(p.status, kBadPage);
                    a.page = -1;
                } else {
                    const size_t block = ((size_t)p.layer * p.c.n_pages + a.page) * p.c.kv_heads + s.head;
                    a.ks = __ldcg(p.c.k_scale + block);
                    a.vs = __ldcg(p.c.v_scale + block);
                }
            }
            return a;
        };
        Ahead now = look(0), next = n_steps > 32 ? look(32) : now;
        int now0 = 0;
        const auto issue = [&](int n) {                     // step n's bytes into its stage; an empty group behind the end
            if (n < n_steps) {
                const int page = __shfl_sync(0xffffffffu, n < now0 + 32 ? now.page : next.page, n & 31);
                const int tok = step_tok(n), valid = page < 0 ? 0 : min(kStep, tok1 - tok);
                const size_t at = ((((size_t)p.layer * p.c.n_pages + max(page, 0)) * p.c.kv_heads + s.head) * p.c.page_tokens + tok % p.c.page_tokens) * HD;
                const uint32_t st = ring + (n % C::kStages) * C::kStageBytes;
#pragma unroll
                for (int i = 0; i < HD / 32; i++) {
                    const int c = lane + 32 * i, ct = c / (HD / 16), cp = c % (HD / 16);
                    const bool in = ct < valid;
                    const size_t from = at + (in ? (size_t)c * 16 : 0);
                    cp16(st + piece_at<HD>(ct, cp), static_cast<const uint8_t *>(p.c.k) + from, in ? 16 : 0);
                    cp16(st + kStep * HD + piece_at<HD>(ct, cp), static_cast<const uint8_t *>(p.c.v) + from, in ? 16 : 0);
                }
            }
            cp_commit();
        };
        for (int n = 0; n < C::kStages - 1; n++) issue(n);

        float o[MT][HD / 8][4];
        float ms[MT][R], l[MT][R], mw[MT][R];
        int last[MT][R];                                     // the last token that the row sees
#pragma unroll
        for (int mt = 0; mt < MT; mt++) {
#pragma unroll
            for (int nt = 0; nt < HD / 8; nt++)
#pragma unroll
                for (int e = 0; e < 4; e++) o[mt][nt][e] = 0.0f;
#pragma unroll
            for (int e = 0; e < R; e++) {
                ms[mt][e] = mw[mt][e] = -INFINITY;
                l[mt][e] = 0.0f;
                const int r = mt * (SPLIT ? 8 : 16) + g + 8 * e;
                last[mt][e] = r < n_rows ? len - n_q + token_row(r) : -1;
            }
        }
        const int all_see = len - n_q + token_row(0);        // up to here every row of the tile sees every token

        for (int n = 0; n < n_steps; n++) {
            if (n == now0 + 32) {
                now = next;
                now0 = n;
                if (n + 32 < n_steps) next = look(n + 32);
            }
            cp_wait<C::kStages - 2>();
            __syncwarp();
            const uint32_t st = ring + (n % C::kStages) * C::kStageBytes;
            const int tok = step_tok(n);
            const float ks = __shfl_sync(0xffffffffu, now.ks, n & 31), vs = __shfl_sync(0xffffffffu, now.vs, n & 31);
            const bool skip = __shfl_sync(0xffffffffu, now.page, n & 31) < 0;

            // ---- scores: two tiles of 8 tokens ----
            float sc[MT][2][4];
#pragma unroll
            for (int mt = 0; mt < MT; mt++)
#pragma unroll
                for (int j = 0; j < 2; j++)
#pragma unroll
                    for (int e = 0; e < 4; e++) sc[mt][j][e] = 0.0f;
#pragma unroll
            for (int cc = 0; cc < HD / 64; cc++) {
                uint4 w[2];
#pragma unroll
                for (int j = 0; j < 2; j++) w[j] = lds128(st + piece_at<HD>(8 * j + token_of_col<HD>(g), t + 4 * cc));
#pragma unroll
                for (int k4 = 0; k4 < 4; k4++) {
                    uint32_t b[2][2];
#pragma unroll
                    for (int j = 0; j < 2; j++) k_regs<FORMAT>(k4 == 0 ? w[j].x : k4 == 1 ? w[j].y : k4 == 2 ? w[j].z : w[j].w, b[j][0], b[j][1]);
#pragma unroll
                    for (int mt = 0; mt < MT; mt++) {
                        const uint4 a = MT == 1 ? qf[MT == 1 ? cc * 4 + k4 : 0] : qf_smem[(mt * C::kSteps + cc * 4 + k4) * 32 + lane];
#pragma unroll
                        for (int j = 0; j < 2; j++) mma(sc[mt][j], a, b[j][0], b[j][1]);
                    }
                }
            }
            // ---- softmax of the step ----
            const uint32_t vb = __float_as_uint(vs) & 0x7fffffffu;
            const int vex = (int)(vb >> 23);                               // 0: zero or below 2^-126; 255: not finite
            const float ve = vex == 255 ? 0.0f : (float)(max(vex, 1) - 127);
            const float vm = vex == 255 ? vs : vex == 0 ? vs * 0x1p126f : __uint_as_float((__float_as_uint(vs) & 0x807fffffu) | 0x3f800000u);
            const bool hide = tok + kStep - 1 > all_see || skip;
            uint4 pf[MT];
#pragma unroll
            for (int mt = 0; mt < MT; mt++) {
                float x[R][4];                                             // (tile j, column 2t + e) at 2 j + e
#pragma unroll
                for (int e = 0; e < R; e++) {
                    const float f = ks * (MT == 1 ? rs[e] : s_rs[MT > 1 ? mt * (SPLIT ? 8 : 16) + g + 8 * e : 0]);
                    float mx = -INFINITY;
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const float raw = SPLIT ? sc[mt][i >> 1][i & 1] + sc[mt][i >> 1][2 + (i & 1)] : sc[mt][i >> 1][2 * e + (i & 1)];
                        x[e][i] = raw * f;
                        if (hide && (skip || tok + 8 * (i >> 1) + token_of_col<HD>(2 * t + (i & 1)) > last[mt][e])) x[e][i] = -INFINITY;
                        mx = fmaxf(mx, x[e][i]);
                    }
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                    // references that grow only when they have to, to whole numbers
                    const float as = mx > ms[mt][e] + kLazy ? ceilf(mx) : ms[mt][e];
                    const float aw = mx + ve > mw[mt][e] + kLazy ? ceilf(mx + ve) : mw[mt][e];
                    if (as != ms[mt][e]) {
                        l[mt][e] *= ex2(ms[mt][e] - as);
                        ms[mt][e] = as;
                    }
                    const bool grow = aw != mw[mt][e];
                    if (__any_sync(0xffffffffu, grow)) {
                        const float f2 = grow ? ex2(mw[mt][e] - aw) : 1.0f;
#pragma unroll
                        for (int nt = 0; nt < HD / 8; nt++) {
                            o[mt][nt][2 * e] *= f2;
                            o[mt][nt][2 * e + 1] *= f2;
                            if (SPLIT) {
                                o[mt][nt][2] *= f2;
                                o[mt][nt][3] *= f2;
                            }
                        }
                        mw[mt][e] = aw;
                    }
                    const float off = ve - mw[mt][e] + kUp;
                    float sum = 0.0f;
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const bool gone = x[e][i] == -INFINITY;             // hidden (or a score of -inf): no weight, whatever the references are
                        sum += gone ? 0.0f : ex2(x[e][i] - ms[mt][e]);
                        x[e][i] = gone ? 0.0f : ex2(x[e][i] + off) * vm;
                    }
                    l[mt][e] += sum;
                }
                if (SPLIT) {
                    split2(x[0][0], x[0][1], pf[mt].x, pf[mt].y);
                    split2(x[0][2], x[0][3], pf[mt].z, pf[mt].w);
                } else {
                    pf[mt] = make_uint4(half2_bits(x[0][0], x[0][1]), half2_bits(x[R - 1][0], x[R - 1][1]), half2_bits(x[0][2], x[0][3]),
                                        half2_bits(x[R - 1][2], x[R - 1][3]));
                }
            }
            // ---- weights times values ----
            const uint32_t sv = st + kStep * HD + 4 * (g & 3);
            int at[4];
#pragma unroll
            for (int i = 0; i < 4; i++) at[i] = 8 * (i >> 1) + token_of_col<HD>(2 * t + (i & 1));
#pragma unroll
            for (int i4 = 0; i4 < HD / 32; i4++) {
                uint32_t w[4];
#pragma unroll
                for (int i = 0; i < 4; i++) w[i] = lds32(sv + piece_at<HD>(at[i], 2 * i4 + (g >> 2)));
                uint32_t b0[4], b1[4];
                v_regs<FORMAT>(w[0], w[1], b0);
                v_regs<FORMAT>(w[2], w[3], b1);
#pragma unroll
                for (int e = 0; e < 4; e++)
#pragma unroll
                    for (int mt = 0; mt < MT; mt++) mma(o[mt][4 * i4 + e], pf[mt], b0[e], b1[e]);
            }
            __syncwarp();
            issue(n + C::kStages - 1);
        }
        cp_wait<0>();

        // ---- the four warps' sums ----
        float *mine = reinterpret_cast<float *>(smem + warp * kRing);
#pragma unroll
        for (int mt = 0; mt < MT; mt++)
#pragma unroll
            for (int e = 0; e < R; e++) {
                const int r = mt * (SPLIT ? 8 : 16) + g + 8 * e;
                float sum = l[mt][e];
                sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                if (t == 0) {
                    s_ms[warp][r] = ms[mt][e];
                    s_l[warp][r] = sum;
                    s_mw[warp][r] = mw[mt][e];
                }
#pragma unroll
                for (int i4 = 0; i4 < HD / 32; i4++) {
                    float a[8];
#pragma unroll
                    for (int q = 0; q < 4; q++) {
                        a[q] = o[mt][4 * i4 + q][2 * e] + (SPLIT ? o[mt][4 * i4 + q][2] : 0.0f);
                        a[4 + q] = o[mt][4 * i4 + q][2 * e + 1] + (SPLIT ? o[mt][4 * i4 + q][3] : 0.0f);
                    }
                    float4 *dst = reinterpret_cast<float4 *>(mine + r * C::kMergeLd + 32 * i4 + 8 * t);
                    dst[0] = make_float4(a[0], a[1], a[2], a[3]);
                    dst[1] = make_float4(a[4], a[5], a[6], a[7]);
                }
            }
        __syncthreads();
        const bool whole = s.t0 == 0 && s.t1 == s.tiles;
        const Part part = part_of(p.ws, HD, (int)blockIdx.x, s.t0 == 0 ? 1 : 0);
        for (int i = threadIdx.x; i < min(RT, n_rows) * (HD / 4); i += kThreads) {
            const int r = i / (HD / 4), d = i % (HD / 4) * 4;
            float big_s = -INFINITY, big_w = -INFINITY;
#pragma unroll
            for (int w = 0; w < kWarps; w++) {
                big_s = fmaxf(big_s, s_ms[w][r]);
                big_w = fmaxf(big_w, s_mw[w][r]);
            }
            float sum = 0.0f, a[4] = {};
#pragma unroll
            for (int w = 0; w < kWarps; w++) {
                sum += s_l[w][r] * part_factor(s_ms[w][r], big_s);
                const float f = part_factor(s_mw[w][r], big_w);
                const float4 x = *reinterpret_cast<const float4 *>(smem + w * kRing + (r * C::kMergeLd + d) * 4);
                a[0] += x.x * f;
                a[1] += x.y * f;
                a[2] += x.z * f;
                a[3] += x.w * f;
            }
            if (whole) {
                float second;
                const float f = finish_scale(big_s, sum, big_w, second);
                const int flat = s.row_tile * RT + r, tok = flat / p.group;
                store4(p, (long long)(row0 + tok) * p.ld_out + (long long)(s.head * p.group + flat - tok * p.group) * HD + d, a[0] * f * second,
                       a[1] * f * second, a[2] * f * second, a[3] * f * second);
            } else {
                *reinterpret_cast<float4 *>(part.o + (size_t)r * HD + d) = make_float4(a[0], a[1], a[2], a[3]);
                if (d == 0) {
                    part.ms[r] = big_s;
                    part.l[r] = sum;
                    part.mw[r] = big_w;
                }
            }
        }
        __syncthreads();
        u += s.t1 - s.t0;
    }
}

// Joins the partial results of the run that CTA blockIdx.x of the kernel above began and did not end: a thread per four dimensions of a row.
template <int HD, int RT>
__global__ void __launch_bounds__(256)
kv_attention_join_kernel(const AttnParams p, int ctas) {
    __shared__ Chunk ck;
    // This kernel starts once every CTA of the one before is past its own wait: lengths and offsets are there, partial results are not.
    long long total = 0;
    for (int base = 0; base < p.n_seqs; base += kThreads) total = load_chunk<RT>(p, ck, base, total, false);
    const long long per = units_per_cta(p, total, ctas);
    const long long u0 = per * blockIdx.x, u1 = min(u0 + per, total);
    bool work = u0 < u1 && u1 < total;
    Segment s = {};
    if (work) {
        if (p.n_seqs > kThreads) {
            int base = 0;
            long long behind = load_chunk<RT>(p, ck, 0, 0, false);
            while (u1 - 1 >= behind) {
                base += kThreads;
                behind = load_chunk<RT>(p, ck, base, behind, false);
            }
        }
        s = segment_at<RT>(p, ck, u1 - 1, u1);
        work = s.first >= u0 && s.t1 < s.tiles;              // begins here and goes on
    }
    tpb_grid_dep_launch();
    tpb_grid_dep_wait();
    if (!work) return;
    const int n_q = ck.n_q[s.idx], row0 = ck.row0[s.idx];
    const int n_rows = min(RT, n_q * p.group - s.row_tile * RT);
    const int c0 = (int)blockIdx.x, c1 = (int)((s.first + s.tiles - 1) / per);
    for (int i = threadIdx.x; i < n_rows * (HD / 4); i += (int)blockDim.x) {
        const int r = i / (HD / 4), d = i % (HD / 4) * 4;
        float big_s = -INFINITY, big_w = -INFINITY;
#pragma unroll 4
        for (int c = c0; c <= c1; c++) {
            const Part part = part_of(p.ws, HD, c, c == c0 ? 1 : 0);
            big_s = fmaxf(big_s, __ldcg(part.ms + r));
            big_w = fmaxf(big_w, __ldcg(part.mw + r));
        }
        float sum = 0.0f, a[4] = {};
#pragma unroll 4
        for (int c = c0; c <= c1; c++) {
            const Part part = part_of(p.ws, HD, c, c == c0 ? 1 : 0);
            sum += __ldcg(part.l + r) * part_factor(__ldcg(part.ms + r), big_s);
            const float f = part_factor(__ldcg(part.mw + r), big_w);
            const float4 x = __ldcg(reinterpret_cast<const float4 *>(part.o + (size_t)r * HD + d));
            a[0] += x.x * f;
            a[1] += x.y * f;
            a[2] += x.z * f;
            a[3] += x.w * f;
        }
        float second;
        const float f = finish_scale(big_s, sum, big_w, second);
        const int flat = s.row_tile * RT + r, tok = flat / p.group;
        store4(p, (long long)(row0 + tok) * p.ld_out + (long long)(s.head * p.group + flat - tok * p.group) * HD + d, a[0] * f * second, a[1] * f * second,
               a[2] * f * second, a[3] * f * second);
    }
}

template <int HD, int FORMAT, bool SPLIT, int MT>
int launch_attention(tpb_handle_t h, cudaStream_t st, const AttnParams &p, bool may_split) {
    using C = Cfg<HD, SPLIT, MT>;
    static tpb_per_device_once smem_set;
    TPB_CUDA(h, tpb_set_max_smem_once(h, kv_attention_kernel<HD, FORMAT, SPLIT, MT>, C::kSmem, smem_set));
    const int ctas = h->sm_count * C::kCtas;
    TPB_CUDA(h, tpb_launch_pdl(kv_attention_kernel<HD, FORMAT, SPLIT, MT>, dim3((unsigned)ctas), dim3(kThreads), (size_t)C::kSmem, st, p));
    if (may_split)
        TPB_CUDA(h, tpb_launch_pdl(kv_attention_join_kernel<HD, C::kRows>, dim3((unsigned)ctas), dim3(256), 0, st, p, ctas));
    return TPB_OK;
}

// Rows of a tile: the fewest m tiles that hold what a sequence of average size has, at most two of 128 dimensions or four of 64 (their sums are
// in registers).
template <int HD, int FORMAT, bool SPLIT>
int by_rows(tpb_handle_t h, cudaStream_t st, const AttnParams &p, bool may_split) {
    const int64_t rows = ((int64_t)p.rows + p.n_seqs - 1) / p.n_seqs * p.group;
    const int64_t tiles = (rows + (SPLIT ? 8 : 16) - 1) / (SPLIT ? 8 : 16);
    if (tiles <= 1) return launch_attention<HD, FORMAT, SPLIT, 1>(h, st, p, may_split);
    if constexpr (HD == 64 && SPLIT)
        if (tiles > 2) return launch_attention<HD, FORMAT, SPLIT, 4>(h, st, p, may_split);
    return launch_attention<HD, FORMAT, SPLIT, 2>(h, st, p, may_split);
}

}  // namespace

extern "C" {

size_t tpb_kv_attention_workspace_bytes(tpb_handle_t h, int head_dim) {
    if (!h || (head_dim != 64 && head_dim != 128)) return 0;
    return (size_t)h->sm_count * kMaxCtas * 2 * slot_floats(head_dim) * sizeof(float);
}

int tpb_kv_attention(tpb_handle_t h, tpb_stream_t stream, const tpb_kv_cache *c, int layer, void *out, int64_t ld_out, const void *q,
                     int64_t ld_q, int dtype, const int32_t *seqs, const int32_t *cu, int n_seqs, int64_t rows, int heads, float scale,
                     int64_t max_len, void *workspace, size_t workspace_bytes) {
    if (!h) return TPB_ERR_INVALID_ARG;
    const int rc = check_layer(h, c, layer, "kv_attention");
    if (rc != TPB_OK) return rc;
    TPB_CHECK_ARG(h, dtype == TPB_F32 || dtype == TPB_BF16 || dtype == TPB_F16, "kv_attention: rows must be f32, bf16 or f16");
    TPB_CHECK_ARG(h, n_seqs >= 0 && n_seqs < (1 << 24) && rows >= 0 && rows < (1 << 26) && max_len >= 0, "kv_attention: bad n_seqs / rows / max_len");
    TPB_CHECK_ARG(h, heads > 0 && heads % c->kv_heads == 0 && heads <= 65535, "kv_attention: heads must be a multiple of kv_heads, at most 65535");
    TPB_CHECK_ARG(h, rows * (heads / c->kv_heads) < ((int64_t)1 << 30), "kv_attention: rows * heads / kv_heads must be below 2^30");
    TPB_CHECK_ARG(h, scale >= 0.0f && scale <= 3.4e38f, "kv_attention: scale must be finite and not negative");
    if (n_seqs == 0 || rows == 0) return TPB_OK;
    TPB_CHECK_ARG(h, out && q && seqs && cu && workspace, "kv_attention: null pointer");
    const int64_t width = (int64_t)heads * c->head_dim, mult = dtype == TPB_F32 ? 4 : 8;
    TPB_CHECK_ARG(h, ld_q >= width && ld_out >= width && ld_q % mult == 0 && ld_out % mult == 0,
                  "kv_attention: ld_q and ld_out must be at least heads * head_dim and multiples of %lld", (long long)mult);
    TPB_CHECK_ARG(h, tpb_aligned16(out) && tpb_aligned16(q) && tpb_aligned16(workspace), "kv_attention: out, q and workspace must be 16-byte aligned");
    TPB_CHECK_ARG(h, ((reinterpret_cast<uintptr_t>(seqs) | reinterpret_cast<uintptr_t>(cu)) & 3u) == 0, "kv_attention: seqs and cu must be 4-byte aligned");
    TPB_CHECK_ARG(h, workspace_bytes >= tpb_kv_attention_workspace_bytes(h, c->head_dim), "kv_attention: the workspace holds %zu bytes, %zu are needed",
                  workspace_bytes, tpb_kv_attention_workspace_bytes(h, c->head_dim));
    tpb_device_guard guard(h->device);
    TPB_CUDA(h, guard.err);
    AttnParams p;
    p.c = *c;
    p.layer = layer;
    p.dtype = dtype;
    p.out = out;
    p.q = q;
    p.ld_out = ld_out;
    p.ld_q = ld_q;
    p.seqs = seqs;
    p.cu = cu;
    p.n_seqs = n_seqs;
    p.rows = (int)rows;
    p.heads = heads;
    p.group = heads / c->kv_heads;
    p.scale_log2 = scale * 1.4426950408889634f;
    p.ws = static_cast<float *>(workspace);
    p.status = h->d_status;
    // sequences known to be short stay whole, which saves the second launch (a longer one that comes all the same is one CTA's work)
    const bool may_split = max_len == 0 || max_len > kMinUnits * kUnit;
    p.whole = !may_split;
    cudaStream_t st = (cudaStream_t)stream;
    const bool split = dtype != TPB_BF16;
    const auto by_format = [&](auto hd_tag, auto split_tag) {
        constexpr int HD = decltype(hd_tag)::value;
        constexpr bool S = decltype(split_tag)::value;
        return c->format == TPB_KV_S8 ? by_rows<HD, TPB_KV_S8, S>(h, st, p, may_split) : by_rows<HD, TPB_KV_E4M3, S>(h, st, p, may_split);
    };
    using I64 = std::integral_constant<int, 64>;
    using I128 = std::integral_constant<int, 128>;
    if (c->head_dim == 64) return split ? by_format(I64{}, std::true_type{}) : by_format(I64{}, std::false_type{});
    return split ? by_format(I128{}, std::true_type{}) : by_format(I128{}, std::false_type{});
}

}  // extern "C"
