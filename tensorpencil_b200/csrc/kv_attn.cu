// Attention of a sequence's last tokens over its 8-bit cache, in pages: the decode step's attention, and that of a few drafted tokens.
//
//   out[r] = sum_j softmax_j(scale q[r] . k[j]) v[j],   k = ks * qk, v = vs * qv with one scale a page and head
//
// Bound by the cache's bytes, which are read once: 2 * head_dim a token and kv head.  What carries that:
//   - All query rows that share a kv head (tokens x heads of the group) are the N side of mma.sync m16n8k16 (f16, f32 sums), eight a tile;
//     tokens (K q^T) and dimensions (V^T P^T) are the M side, so that a decode step's few rows leave nothing of a product unused, as they
//     would of a tcgen05 tile of 128 rows.  The cached values are exact in f16.
//   - f32 accuracy (SPLIT) for f32 and f16 rows: q = hi + lo in f16 (after scaling the row by a power of two), and the weights likewise, two
//     products each.  bf16 queries are exact in one f16 term, and weights of one f16 term (2^-12) are below a bf16 result's half step (2^-9).
//   - For bf16 rows K's int8 goes into the product as it is: byte ^ 0x80 in the low byte of an f16 is the number (128 + k) 2^-24, and the
//     sum's start value takes the 128 sum(q) off again (a fixed number a row).  V's cancels less well over a long sequence and is converted exactly.
//   - Page scales are uniform over a piece of 16 tokens (a page holds 16, 32 or 64): ks multiplies scores, vs the weights.
//   - A warp owns its data path: K and V of 16 or 32 tokens a step by cp.async into a ring of its own, no barrier between warps, and the next
//     run's first step is on its way while a run's sums are merged.  Bytes lie in shared memory with their 16-byte pieces
//     permuted so that K's 16-byte reads and V's 4-byte reads are free of bank conflicts; the order of dimensions within the products is the one in
//     which a thread finds its bytes, and q is laid out to match.
//   - The work of all (sequence, kv head, row tile)s is one line of units of tokens, cut into equal pieces, one a CTA.  A CTA that has
//     not all of a sequence's tokens leaves a partial result; a second kernel joins them in the order of the tokens, so the
//     result is the same from run to run.
// Measured (32 heads over 8 of 128): 131000 tokens, int8, bf16 rows 55 us (the cache's 268 MB at the rate of a plain copy: 41.5), 48 sequences of 1 to 16000
// tokens, e4m3, 75 us (62), one of 200 tokens 7.5 us; five drafted tokens of 16 sequences, 16 heads over 4 of 64, f32 rows: 25 us, a chain of about five
// steps a warp.  Steps of 16 tokens with four CTAs an SM took 132 us where 32 with three took 102 (the 48 sequences), rings of 24 KB with two 131.
//
// Softmax.  Per row two running references, both whole numbers in log2 units so that every rescaling is exact: ms >= max s - kLazy for the sum
// l = sum 2^(s - ms), and mw for the weights w = 2^(s + log2 vs - mw + kUp), whose size depends on the page's scale as well.
#include <algorithm>

#include "kv_common.cuh"

using namespace tpb_kv;

namespace {

constexpr int kThreads = 128;
constexpr int kWarps = 4;
constexpr int kPiece = 16;           // tokens with one page and scale
constexpr int kMinTokens = TPB_KV_SHORT;      // a CTA takes at least so many: shorter runs cost more in joining than they gain
constexpr int kRing = 16384;         // bytes of a warp's ring
constexpr float kLazy = 6.0f, kUp = 6.0f;      // w < 2^(kLazy + kUp + 1) fits f16

template <int HD, bool SPLIT, int NT>
struct Cfg {
    static constexpr int kRows = 8 * NT;                                 // rows of a tile
    static constexpr int kHalves = NT <= 2 || HD == 64 ? 2 : 1;           // pieces of a warp's step
    static constexpr int kStep = kHalves * kPiece;                       // tokens of a warp's step
    static constexpr int kUnit = kWarps * kStep;                         // tokens of a unit of work: one step of every warp
    static constexpr int kStageBytes = 2 * kStep * HD;
    static constexpr int kStages = kRing / kStageBytes;                  // 2 to 8
    static constexpr int kSteps = HD / 16;                               // k steps of K q^T
    static constexpr int kTerms = SPLIT ? 2 : 1;
    static constexpr bool kQRegs = NT * kTerms <= 2 && HD * NT * kTerms <= 256;      // q's fragments in registers
    static constexpr int kQf = kQRegs ? 0 : NT * kSteps * kTerms * 32 * 8;           // or in shared memory
    static constexpr int kMergeLd = HD + 4;
    static constexpr int kMerge = 2 * kRows * kMergeLd * 4;              // where the warps' sums are added up, in pairs
    static constexpr int kSmem = kWarps * kRing + kMerge + kQf;
    // CTAs an SM that the registers are cut for and the grid is sized by.  They all fit its shared memory but for two terms of 32 rows of 128: one at a
    // time there (20000 tokens, 32 rows a kv head, f32 60 us; with bf16's one term, where two fit, 39; 24 rows, f32 37).
    static constexpr int kCtas = NT == 1 ? 3 : 2;
    static constexpr bool kOneFits = HD == 128 && SPLIT && NT == 4;
    static constexpr int kStatic = 2336 + kRows * 48 + (kQRegs ? 8 : kRows * 8);     // Chunk, the warps' references and sums, q's factors
    static constexpr int kTaken = (kSmem + kStatic + 127) / 128 * 128 + 1024;        // by a CTA; 1024 of it the system's
    static_assert(kRows <= 32, "rows fit a slot");
    static_assert((kOneFits ? 1 : kCtas) * kTaken <= 228 * 1024 && (!kOneFits || 2 * kTaken > 228 * 1024), "so many CTAs fit an SM");
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
    void *notes;                         // a JoinNote a CTA
    uint32_t *status;
};

// ---- the line of units ------------------------------------------------------------------------
// Chunk of kSeqs sequences of the batch in shared memory: first unit, length, rows.  (With 128 of them a third CTA would not fit an SM.)
constexpr int kSeqs = 96;
struct Chunk {
    long long start[kSeqs + 1];
    int len[kSeqs], row0[kSeqs], n_q[kSeqs], seq[kSeqs];
    long long warp_sum[kSeqs / 32];
};
// A run takes about as long again as kRunUnits of its tokens' units do -- its chain of loads, q, the merging -- so its units begin with that many
// which have no tokens.  (48 sequences of 1 to 16000 tokens, 8 kv heads, a unit 1.9 us: without them half the CTAs ended at 60 us and those that
// drew the short sequences at 140, with one 100.)
constexpr int kRunUnits = 3;
template <int UNIT>
__device__ __forceinline__ int tiles_of(const AttnParams &p, int len) { return p.whole ? 1 : kRunUnits + (len + UNIT - 1) / UNIT; }

// Loads sequences base .. base + kSeqs - 1, the first of which begins at unit `cum`; returns the unit behind the last.  `tell`: report ids and
// lengths out of range (such a sequence has no units: its rows are not written).
template <int RT, int UNIT>
__device__ long long load_chunk(const AttnParams &p, Chunk &ck, int base, long long cum, bool tell) {
    const int i = base + (int)threadIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    long long units = 0;
    int len = 0, row0 = 0, n_q = 0, seq = -1;
    if (i < p.n_seqs && threadIdx.x < kSeqs) {
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
                    units = (long long)tiles_of<UNIT>(p, len) * p.c.kv_heads * (((long long)n_q * p.group + RT - 1) / RT);
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
    if (warp < kSeqs / 32 && lane == 31) ck.warp_sum[warp] = inc;
    __syncthreads();
    long long at = cum, total = cum;
    for (int w = 0; w < kSeqs / 32; w++) {
        if (w < warp) at += ck.warp_sum[w];
        total += ck.warp_sum[w];
    }
    if (threadIdx.x < kSeqs) {
        ck.start[threadIdx.x] = at + inc - units;
        ck.len[threadIdx.x] = len;
        ck.row0[threadIdx.x] = row0;
        ck.n_q[threadIdx.x] = n_q;
        ck.seq[threadIdx.x] = seq;
        if (threadIdx.x == kSeqs - 1) ck.start[kSeqs] = total;
    }
    __syncthreads();
    return total;
}
// The sequence of the loaded chunk that holds unit u, start[0] <= u < start[kSeqs].
__device__ __forceinline__ int find_in_chunk(const Chunk &ck, long long u) {
    int lo = 0, hi = kSeqs;           // start[lo] <= u < start[hi]
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
template <int RT, int UNIT>
__device__ __forceinline__ Segment segment_at(const AttnParams &p, const Chunk &ck, long long u, long long u_end) {
    Segment s;
    s.idx = find_in_chunk(ck, u);
    s.tiles = tiles_of<UNIT>(p, ck.len[s.idx]);
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
template <int UNIT>
__device__ __forceinline__ long long units_per_cta(const AttnParams &p, long long total, int ctas) {
    return max((total + ctas - 1) / ctas, (long long)(p.whole ? 1 : kRunUnits + kMinTokens / UNIT));
}

// ---- arithmetic -------------------------------------------------------------------------------
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float pow2i(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }       // -126 <= e <= 127
// d = a b + c
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint2 b, float c0, float c1, float c2, float c3) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b.x), "r"(b.y), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t a) {          // of 16-bit values, row lane / 4
    uint32_t d;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}
__device__ __forceinline__ float lg2(float x) {
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
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
// int8 pairs in the low bytes of both halves -> f16, exactly: 0x6400 | (x ^ 0x80) is 1024 + 128 + x
__device__ __forceinline__ uint32_t s8_pair(uint32_t w) {
    uint32_t b;
    asm("lop3.b32 %0, %1, %2, %3, 0x6a;" : "=r"(b) : "r"(w), "r"(0x00ff00ffu), "r"(0x64806480u));     // (w & mask) ^ bias
    const __half2 h = __hsub2(*reinterpret_cast<const __half2 *>(&b), __half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480)));
    return *reinterpret_cast<const uint32_t *>(&h);
}
// (128 + x) 2^-24 as subnormal f16
__device__ __forceinline__ uint32_t s8_pair_raw(uint32_t w) {
    uint32_t b;
    asm("lop3.b32 %0, %1, %2, %3, 0x6a;" : "=r"(b) : "r"(w), "r"(0x00ff00ffu), "r"(0x00800080u));
    return b;
}
// Four consecutive bytes of K as the two registers of a k step, times kPerUnitOfK: bytes (0, 2), (1, 3) of s8, (0, 1), (2, 3) of e4m3.  RAW: as
// 128 + k, for one instruction less a pair; the sums are then several times the scores, and f32 results lose a bit or two (16 sequences
// of 3000 tokens, five drafted each: 1.9e-6 off instead of 1.0e-6).
template <int FORMAT, bool RAW>
__device__ __forceinline__ void k_regs(uint32_t w, uint32_t &b0, uint32_t &b1) {
    if constexpr (FORMAT == TPB_KV_S8) {
        b0 = RAW ? s8_pair_raw(w) : s8_pair(w);
        b1 = RAW ? s8_pair_raw(w >> 8) : s8_pair(w >> 8);
    } else {
        b0 = e4m3_pair<0>(w);
        b1 = e4m3_pair<1>(w);
    }
}
template <int FORMAT, bool RAW>
constexpr float kPerUnitOfK = FORMAT == TPB_KV_S8 && RAW ? 16777216.0f : 1.0f;        // 2^24
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
        v[0] = e4m3_pair<0>(lo);
        v[1] = e4m3_pair<1>(lo);
        v[2] = e4m3_pair<0>(hi);
        v[3] = e4m3_pair<1>(hi);
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
__device__ __forceinline__ void cp16(uint32_t dst, const void *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp16_or_zero(uint32_t dst, const void *src, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
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

// What the join needs to know of the run that CTA c began and did not end; rows = 0: nothing to join.
struct JoinNote {
    int rows, last_cta;
    long long out_row;               // of the run's first row; the rest by row tile, head and group
    int row_tile, head;
};
__host__ __device__ inline size_t note_floats(int ctas) { return (size_t)ctas * (sizeof(JoinNote) / 4); }

template <int HD, int FORMAT, bool SPLIT, int NT>
__global__ void __launch_bounds__(kThreads, Cfg<HD, SPLIT, NT>::kCtas)
kv_attention_kernel(const AttnParams p) {
    using C = Cfg<HD, SPLIT, NT>;
    constexpr int RT = C::kRows, UNIT = C::kUnit, H = C::kHalves, TERMS = C::kTerms;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ Chunk ck;
    __shared__ float s_ms[kWarps][RT], s_l[kWarps][RT], s_mw[kWarps][RT], s_rs[C::kQRegs ? 1 : RT], s_bias[C::kQRegs ? 1 : RT];
    tpb_grid_dep_launch();
    tpb_grid_dep_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;

    long long total = 0;
    for (int base = 0; base < p.n_seqs; base += kSeqs) total = load_chunk<RT, UNIT>(p, ck, base, total, blockIdx.x == 0);
    const long long per = units_per_cta<UNIT>(p, total, (int)gridDim.x);
    long long u = per * blockIdx.x;
    const long long u_end = min(u + per, total);
    JoinNote note = {};
    if (u < u_end) {
        int base = 0;
        if (p.n_seqs > kSeqs) {
            long long behind = load_chunk<RT, UNIT>(p, ck, 0, 0, false);
            while (u >= behind) {
                base += kSeqs;
                behind = load_chunk<RT, UNIT>(p, ck, base, behind, false);
            }
        }
        // where this lane's bytes lie in a stage: the pieces that it copies, K's 16 bytes of a token, V's words of two tokens
        const uint32_t ring = smem_addr(smem) + warp * kRing;
        float *merge = reinterpret_cast<float *>(smem + kWarps * kRing);
        uint2 *qf_smem = reinterpret_cast<uint2 *>(smem + kWarps * kRing + C::kMerge);
        constexpr int CP = HD / 32;                        // pieces a lane copies of a 16-token piece of K or V
        uint32_t cp_at[CP], k_at[HD / 64], v_at[2];
#pragma unroll
        for (int i = 0; i < CP; i++) cp_at[i] = piece_at<HD>((lane + 32 * i) / (HD / 16), (lane + 32 * i) % (HD / 16));
#pragma unroll
        for (int cc = 0; cc < HD / 64; cc++) k_at[cc] = piece_at<HD>(token_of_col<HD>(g), t + 4 * cc);
#pragma unroll
        for (int i = 0; i < 2; i++) v_at[i] = C::kStep * HD + piece_at<HD>(token_of_col<HD>(2 * t + i), g >> 2) + 4 * (g & 3);

        // ---- the run at hand: its tokens [mine0, tok1), every kWarps-th step this warp's ----
        Segment s = {};
        int len, n_q, row0, tok1, mine0, n_steps, now0;
        const int32_t *row;
        // Places and scales of 32 pieces, a piece a lane, and of the 32 behind them.
        struct Ahead {
            int at;                                         // row of the cache of the piece's first token and this head; -1: no piece there, or no page
            float ks, vs;
        } now, next;
        constexpr int kBatch = 32 / H;                      // steps
        const auto look = [&](int n0) {
            Ahead a;
            a.at = -1;
            a.ks = a.vs = 0.0f;
            const int piece = n0 * H + lane, tok = mine0 + piece / H * UNIT + piece % H * kPiece;
            if (tok < tok1) {
                const int page = __ldcg(row + tok / p.c.page_tokens);
                if (page < 0 || page >= p.c.n_pages) {
                    report(p.status, kBadPage);
                } else {
                    const int block = (int)(((long long)p.layer * p.c.n_pages + page) * p.c.kv_heads) + s.head;
                    a.at = block * p.c.page_tokens + (tok & (p.c.page_tokens - 1));
                    a.ks = __ldcg(p.c.k_scale + block);
                    a.vs = __ldcg(p.c.v_scale + block);
                }
            }
            return a;
        };
        const auto issue = [&](int n) {                     // step n's bytes into its stage; an empty group behind the end
            if (n < n_steps) {
                const uint32_t st = ring + (n % C::kStages) * C::kStageBytes;
#pragma unroll
                for (int h = 0; h < H; h++) {
                    const int at = __shfl_sync(0xffffffffu, n < now0 + kBatch ? now.at : next.at, (n * H + h) & 31);
                    const int valid = at < 0 ? 0 : min(kPiece, tok1 - (mine0 + n * UNIT + h * kPiece));
                    const size_t from = (size_t)(uint32_t)max(at, 0) * HD + lane * 16;
                    const uint8_t *k = static_cast<const uint8_t *>(p.c.k) + from, *v = static_cast<const uint8_t *>(p.c.v) + from;
                    const uint32_t dst = st + h * (kPiece * HD);
                    if (valid == kPiece) {
#pragma unroll
                        for (int i = 0; i < CP; i++) {
                            cp16(dst + cp_at[i], k + i * 512);
                            cp16(dst + cp_at[i] + C::kStep * HD, v + i * 512);
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < CP; i++) {
                            const bool in = (lane + 32 * i) / (HD / 16) < valid;
                            cp16_or_zero(dst + cp_at[i], in ? k + i * 512 : p.c.k, in);
                            cp16_or_zero(dst + cp_at[i] + C::kStep * HD, in ? v + i * 512 : p.c.v, in);
                        }
                    }
                }
            }
            cp_commit();
        };
        // Makes the run that begins at unit u the one at hand and sets its first steps on their way.
        const auto begin = [&]() {
            while (u >= ck.start[kSeqs]) {
                base += kSeqs;
                load_chunk<RT, UNIT>(p, ck, base, ck.start[kSeqs], false);
            }
            s = segment_at<RT, UNIT>(p, ck, u, u_end);
            len = ck.len[s.idx];
            n_q = ck.n_q[s.idx];
            row0 = ck.row0[s.idx];
            row = p.c.table + (size_t)ck.seq[s.idx] * p.c.max_pages;
            tok1 = p.whole ? len : min(max(s.t1 - kRunUnits, 0) * UNIT, len);
            mine0 = max(s.t0 - kRunUnits, 0) * UNIT + warp * C::kStep;
            n_steps = tok1 > mine0 ? (tok1 - mine0 + UNIT - 1) / UNIT : 0;
            now0 = 0;
            now = look(0);
            next = now;
            for (int n = 0; n < C::kStages - 1; n++) issue(n);
            if (n_steps > kBatch) next = look(kBatch);
        };
        begin();
        while (true) {
            const int n_rows = n_q * p.group - s.row_tile * RT;           // of this tile, if below RT
            const auto token_row = [&](int r) { return (s.row_tile * RT + r) / p.group; };      // which of the sequence's queries row r belongs to

            // ---- q: scaled by a power of two to a largest value in [2^10, 2^11), as f16 terms: row g of a tile, the dimensions of t's bytes ----
            uint2 qf[C::kQRegs ? NT : 1][C::kQRegs ? C::kSteps : 1][TERMS];
            float rs[C::kQRegs ? NT : 1][2], bias[C::kQRegs ? NT : 1][2];     // of rows 2t and 2t + 1: scale log2(e) / that power, -128 2^-24 sum q
            const auto build_q = [&](int nt, uint2 *dst, int stride, float &r_s, float &sum) {
                const int r = nt * 8 + g, flat = s.row_tile * RT + r, tok = flat / p.group;
                float v[HD / 64][16];
                float amax = 0.0f;
#pragma unroll
                for (int cc = 0; cc < HD / 64; cc++) {
                    load_q(p, HD, row0 + tok, s.head * p.group + flat - tok * p.group, 16 * (t + 4 * cc), r < n_rows, v[cc]);
#pragma unroll
                    for (int i = 0; i < 16; i++) amax = fmaxf(amax, fabsf(v[cc][i]));
                }
                amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
                amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
                const int ex = max((int)(__float_as_uint(amax) >> 23) - 127, -116);       // -116: all zero, or below 2^-116
                const float up = pow2i(min(10 - ex, 126));
                r_s = p.scale_log2 * pow2i(max(ex - 10, -126));
                sum = 0.0f;
#pragma unroll
                for (int cc = 0; cc < HD / 64; cc++)
#pragma unroll
                    for (int k4 = 0; k4 < 4; k4++) {
                        uint2 b[2];
                        constexpr int i1 = FORMAT == TPB_KV_S8 ? 2 : 1, i2 = 3 - i1;      // the pairs in which a thread finds K's bytes
                        split2(v[cc][4 * k4] * up, v[cc][4 * k4 + i1] * up, b[0].x, b[1].x);
                        split2(v[cc][4 * k4 + i2] * up, v[cc][4 * k4 + 3] * up, b[0].y, b[1].y);
#pragma unroll
                        for (int e = 0; e < TERMS; e++) {
                            dst[((cc * 4 + k4) * TERMS + e) * stride] = b[e];
                            const float2 f0 = __half22float2(*reinterpret_cast<const __half2 *>(&b[e].x)), f1 = __half22float2(*reinterpret_cast<const __half2 *>(&b[e].y));
                            sum += (f0.x + f0.y) + (f1.x + f1.y);
                        }
                    }
                sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                sum *= FORMAT == TPB_KV_S8 && !SPLIT ? -128.0f / 16777216.0f : 0.0f;
            };
            if constexpr (C::kQRegs) {
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    float r_s, sum;
                    build_q(nt, &qf[nt][0][0], 1, r_s, sum);
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        rs[nt][e] = __shfl_sync(0xffffffffu, r_s, 4 * (2 * t + e));
                        bias[nt][e] = __shfl_sync(0xffffffffu, sum, 4 * (2 * t + e));
                    }
                }
            } else {
                for (int nt = warp; nt < NT; nt += kWarps) {
                    float r_s, sum;
                    build_q(nt, qf_smem + nt * C::kSteps * TERMS * 32 + lane, 32, r_s, sum);
                    if (t == 0) {
                        s_rs[nt * 8 + g] = r_s;
                        s_bias[nt * 8 + g] = sum;
                    }
                }
                __syncthreads();
            }

            float o[NT][HD / 16][4];                             // dimensions by g, rows 2t and 2t + 1
            float ms[NT][2], l[NT][2], mw[NT][2];
            int last[NT][2];                                     // the last token that the row sees
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
#pragma unroll
                for (int m = 0; m < HD / 16; m++)
#pragma unroll
                    for (int e = 0; e < 4; e++) o[nt][m][e] = 0.0f;
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    ms[nt][e] = mw[nt][e] = -INFINITY;
                    l[nt][e] = 0.0f;
                    const int r = nt * 8 + 2 * t + e;
                    last[nt][e] = r < n_rows ? len - n_q + token_row(r) : -1;
                }
            }
            const int all_see = len - n_q + token_row(0);        // up to here every row of the tile sees every token

            for (int n = 0; n < n_steps; n++) {
                if (n == now0 + kBatch) {
                    now = next;
                    now0 = n;
                    if (n + kBatch < n_steps) next = look(n + kBatch);
                }
                cp_wait<C::kStages - 2>();
                __syncwarp();                               // everybody's bytes of step n are there, and everybody is done with step n - 1
                issue(n + C::kStages - 1);
                const uint32_t st = ring + (n % C::kStages) * C::kStageBytes;
                const int tok = mine0 + n * UNIT;
                float ks[H], lv[H];
                bool skip[H], any_skip = false;
#pragma unroll
                for (int h = 0; h < H; h++) {
                    const int from = (n * H + h) & 31;
                    ks[h] = __shfl_sync(0xffffffffu, now.ks, from);
                    const float vs = __shfl_sync(0xffffffffu, now.vs, from);
                    lv[h] = vs < 1.17549435e-38f ? -1000.0f : lg2(vs);     // a page of zeros: no weight; NaN stays NaN
                    skip[h] = __shfl_sync(0xffffffffu, now.at, from) < 0;
                    any_skip |= skip[h];
                }

                // ---- scores: sc[.][h] = tokens g and g + 8 of piece h (as token_of_col has them), rows 2t and 2t + 1 ----
                float sc[NT][H][4];
#pragma unroll
                for (int cc = 0; cc < HD / 64; cc++) {
                    uint4 w[H][2];
#pragma unroll
                    for (int h = 0; h < H; h++)
#pragma unroll
                        for (int j = 0; j < 2; j++) w[h][j] = lds128(st + k_at[cc] + (2 * h + j) * (8 * HD));
#pragma unroll
                    for (int k4 = 0; k4 < 4; k4++) {
                        uint2 q[NT][TERMS];
#pragma unroll
                        for (int nt = 0; nt < NT; nt++)
#pragma unroll
                            for (int e = 0; e < TERMS; e++)
                                q[nt][e] = C::kQRegs ? qf[C::kQRegs ? nt : 0][C::kQRegs ? cc * 4 + k4 : 0][e]
                                                     : qf_smem[((nt * C::kSteps + cc * 4 + k4) * TERMS + e) * 32 + lane];
#pragma unroll
                        for (int h = 0; h < H; h++) {
                            uint32_t a[2][2];
#pragma unroll
                            for (int j = 0; j < 2; j++)
                                k_regs<FORMAT, !SPLIT>(k4 == 0 ? w[h][j].x : k4 == 1 ? w[h][j].y : k4 == 2 ? w[h][j].z : w[h][j].w, a[j][0], a[j][1]);
#pragma unroll
                            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                                for (int e = 0; e < TERMS; e++) {
                                    float(&d)[4] = sc[nt][h];
                                    if (cc == 0 && k4 == 0 && e == 0) {
                                        const float b0 = C::kQRegs ? bias[C::kQRegs ? nt : 0][0] : s_bias[C::kQRegs ? 0 : nt * 8 + 2 * t];
                                        const float b1 = C::kQRegs ? bias[C::kQRegs ? nt : 0][1] : s_bias[C::kQRegs ? 0 : nt * 8 + 2 * t + 1];
                                        mma(d, a[0][0], a[1][0], a[0][1], a[1][1], q[nt][e], b0, b1, b0, b1);
                                    } else {
                                        mma(d, a[0][0], a[1][0], a[0][1], a[1][1], q[nt][e], d[0], d[1], d[2], d[3]);
                                    }
                                }
                        }
                    }
                }
                // ---- softmax of the step ----
                const bool hide = any_skip || tok + C::kStep - 1 > all_see;
                uint2 pf[NT][H][TERMS];
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    // Does a score of any thread call for a larger reference?  Mostly not, and then no maximum over the row is needed.
                    float f[2][H], mx[2], mxw[2];
                    bool grow = false;
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const float r_s = C::kQRegs ? rs[C::kQRegs ? nt : 0][e] : s_rs[C::kQRegs ? 0 : nt * 8 + 2 * t + e];
                        mx[e] = mxw[e] = -INFINITY;
#pragma unroll
                        for (int h = 0; h < H; h++) {
                            f[e][h] = ks[h] * r_s * kPerUnitOfK<FORMAT, !SPLIT>;
                            if (hide) {
#pragma unroll
                                for (int j = 0; j < 2; j++)
                                    if (skip[h] || tok + h * kPiece + 8 * j + token_of_col<HD>(g) > last[nt][e]) sc[nt][h][2 * j + e] = -INFINITY;
                            }
                            const float top = fmaxf(sc[nt][h][e], sc[nt][h][2 + e]) * f[e][h];
                            mx[e] = fmaxf(mx[e], top);
                            mxw[e] = fmaxf(mxw[e], top + lv[h]);
                        }
                        grow |= mx[e] > ms[nt][e] + kLazy || mxw[e] > mw[nt][e] + kLazy;
                    }
                    if (__any_sync(0xffffffffu, grow)) {
                        // references grow only when they have to, to whole numbers
#pragma unroll
                        for (int e = 0; e < 2; e++) {
#pragma unroll
                            for (int of = 4; of < 32; of <<= 1) {
                                mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], of));
                                mxw[e] = fmaxf(mxw[e], __shfl_xor_sync(0xffffffffu, mxw[e], of));
                            }
                            const float as = mx[e] > ms[nt][e] + kLazy ? ceilf(mx[e]) : ms[nt][e];
                            const float aw = mxw[e] > mw[nt][e] + kLazy ? ceilf(mxw[e]) : mw[nt][e];
                            if (as != ms[nt][e]) l[nt][e] *= ex2(ms[nt][e] - as);
                            const float f2 = aw != mw[nt][e] ? ex2(mw[nt][e] - aw) : 1.0f;
                            ms[nt][e] = as;
                            mw[nt][e] = aw;
#pragma unroll
                            for (int m = 0; m < HD / 16; m++) {
                                o[nt][m][e] *= f2;
                                o[nt][m][2 + e] *= f2;
                            }
                        }
                    }
#pragma unroll
                    for (int h = 0; h < H; h++) {
                        float w[4];
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const int e = i & 1;
                            const float y = sc[nt][h][i];
                            float a = ex2(fmaf(y, f[e][h], -ms[nt][e])), b = ex2(fmaf(y, f[e][h], lv[h] - mw[nt][e] + kUp));
                            if (hide && y == -INFINITY) a = b = 0.0f;      // whatever the references and the page's scales are
                            l[nt][e] += a;
                            w[i] = b;
                        }
                        uint32_t p0[2], p1[2];
                        if (SPLIT) {
                            split2(w[0], w[1], p0[0], p0[1]);
                            split2(w[2], w[3], p1[0], p1[1]);
                        } else {
                            p0[0] = half2_bits(w[0], w[1]);
                            p1[0] = half2_bits(w[2], w[3]);
                        }
#pragma unroll
                        for (int e = 0; e < TERMS; e++) pf[nt][h][e] = make_uint2(transpose8x8(p0[e]), transpose8x8(p1[e]));
                    }
                }
                // ---- values times weights ----
#pragma unroll
                for (int i4 = 0; i4 < HD / 32; i4++)
#pragma unroll
                    for (int h = 0; h < H; h++) {
                        // piece 2 i4 + (g >> 2) of the token: the permutation is an exclusive or, and stages begin at multiples of 128 bytes
                        const uint32_t a0 = (st + v_at[0]) ^ (i4 * 32), a1 = (st + v_at[1]) ^ (i4 * 32);
                        uint32_t w[4];
                        w[0] = lds32(a0 + h * (kPiece * HD));
                        w[1] = lds32(a1 + h * (kPiece * HD));
                        w[2] = lds32(a0 + h * (kPiece * HD) + 8 * HD);
                        w[3] = lds32(a1 + h * (kPiece * HD) + 8 * HD);
                        uint32_t b0[4], b1[4];
                        v_regs<FORMAT>(w[0], w[1], b0);
                        v_regs<FORMAT>(w[2], w[3], b1);
#pragma unroll
                        for (int m = 0; m < 2; m++)
#pragma unroll
                            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                                for (int e = 0; e < TERMS; e++) {
                                    float(&d)[4] = o[nt][2 * i4 + m];
                                    mma(d, b0[2 * m], b0[2 * m + 1], b1[2 * m], b1[2 * m + 1], pf[nt][h][e], d[0], d[1], d[2], d[3]);
                                }
                    }
            }
            cp_wait<0>();
            __syncwarp();

            // ---- the next run's first steps set off, then the four warps' sums are added up, in the order of the warps ----
            const Segment done = s;
            const int done_row0 = row0;
            u += s.t1 - s.t0;
            if (u < u_end) begin();
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    float sum = l[nt][e];
#pragma unroll
                    for (int of = 4; of < 32; of <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, of);
                    if (g == 0) {
                        const int r = nt * 8 + 2 * t + e;
                        s_ms[warp][r] = ms[nt][e];
                        s_l[warp][r] = sum;
                        s_mw[warp][r] = mw[nt][e];
                    }
                }
            __syncthreads();
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const int r = nt * 8 + 2 * t + e;
                    float big = -INFINITY;
#pragma unroll
                    for (int w = 0; w < kWarps; w++) big = fmaxf(big, s_mw[w][r]);
                    const float f2 = part_factor(mw[nt][e], big);
#pragma unroll
                    for (int m = 0; m < HD / 16; m++) {
                        o[nt][m][e] *= f2;
                        o[nt][m][2 + e] *= f2;
                    }
                }
            // (warp 0 + warp 1) + (warp 2 + warp 3), the halves at the same time
            float *half = merge + (warp >> 1) * (RT * C::kMergeLd);
#pragma unroll 1
            for (int w = 0; w < 2; w++) {
                if ((warp & 1) == w) {
#pragma unroll
                    for (int nt = 0; nt < NT; nt++)
#pragma unroll
                        for (int e = 0; e < 2; e++)
#pragma unroll
                            for (int i4 = 0; i4 < HD / 32; i4++) {
                                float4 *dst = reinterpret_cast<float4 *>(half + (nt * 8 + 2 * t + e) * C::kMergeLd + 32 * i4 + 4 * g);
                                float4 x = make_float4(o[nt][2 * i4][e], o[nt][2 * i4][2 + e], o[nt][2 * i4 + 1][e], o[nt][2 * i4 + 1][2 + e]);
                                if (w > 0) {
                                    const float4 y = *dst;
                                    x = make_float4(y.x + x.x, y.y + x.y, y.z + x.z, y.w + x.w);
                                }
                                *dst = x;
                            }
                }
                __syncthreads();
            }
            const bool whole = done.t0 == 0 && done.t1 == done.tiles;
            const Part part = part_of(p.ws, HD, (int)blockIdx.x, done.t0 == 0 ? 1 : 0);
            for (int i = threadIdx.x; i < min(RT, n_rows) * (HD / 4); i += kThreads) {
                const int r = i / (HD / 4), d = i % (HD / 4) * 4;
                float big_s = -INFINITY, big_w = -INFINITY, sum = 0.0f;
#pragma unroll
                for (int w = 0; w < kWarps; w++) {
                    big_s = fmaxf(big_s, s_ms[w][r]);
                    big_w = fmaxf(big_w, s_mw[w][r]);
                }
#pragma unroll
                for (int w = 0; w < kWarps; w++) sum += s_l[w][r] * part_factor(s_ms[w][r], big_s);
                const float4 a0 = *reinterpret_cast<const float4 *>(merge + r * C::kMergeLd + d);
                const float4 a1 = *reinterpret_cast<const float4 *>(merge + (RT + r) * C::kMergeLd + d);
                const float4 a = make_float4(a0.x + a1.x, a0.y + a1.y, a0.z + a1.z, a0.w + a1.w);
                if (whole) {
                    float second;
                    const float f = finish_scale(big_s, sum, big_w, second);
                    const int flat = done.row_tile * RT + r, tok = flat / p.group;
                    store4(p, (long long)(done_row0 + tok) * p.ld_out + (long long)(done.head * p.group + flat - tok * p.group) * HD + d, a.x * f * second,
                           a.y * f * second, a.z * f * second, a.w * f * second);
                } else {
                    *reinterpret_cast<float4 *>(part.o + (size_t)r * HD + d) = a;
                    if (d == 0) {
                        part.ms[r] = big_s;
                        part.l[r] = sum;
                        part.mw[r] = big_w;
                    }
                }
            }
            if (done.t0 == 0 && !whole) {
                note.rows = min(RT, n_rows);
                note.last_cta = (int)((done.first + done.tiles - 1) / per);
                note.out_row = done_row0;
                note.row_tile = done.row_tile;
                note.head = done.head;
            }
            if (u >= u_end) break;
            __syncthreads();                                 // the sums are read
        }
    }
    if (!p.whole && threadIdx.x == 0) reinterpret_cast<JoinNote *>(p.notes)[blockIdx.x] = note;
}

// Joins the partial results of the run that CTA blockIdx.x of the kernel above began and did not end.  Its time is a chain of loads behind the end of
// that kernel (starting it costs 1 us, a note 0.8), so a thread asks for references, sums and its share of the weighted values all
// at once, before anything is known of their factors: 131000 tokens 6 us, five drafted tokens 6; with one dependent load behind another 10 and 25.
// Grid y: from 16 rows of 128 on two CTAs share the rows (20000 tokens, 16 rows a kv head 26.2 -> 23.5 us for both kernels, 32 rows 46.6 -> 38.3); with fewer
// values the second CTA costs more than it takes over (five drafted tokens, 20 rows of 64, 25.6 -> 26.7).
constexpr int kJoinThreads = 512;
constexpr int kJoinAhead = 8;        // parts of which a thread holds four dimensions
constexpr int kJoinFactors = 2048;   // (part, row) pairs of a pass
template <int HD, int RT>
__global__ void __launch_bounds__(kJoinThreads, 2) kv_attention_join_kernel(const AttnParams p) {
    constexpr int kLanes = HD / 4, kGroups = kJoinThreads / kLanes, kPer = kJoinFactors / kJoinThreads;
    __shared__ float s_ms[kJoinFactors], s_mw[kJoinFactors], s_l[kJoinFactors];
    __shared__ float s_big[2][32], s_sum[32];
    __shared__ float4 s_o[kJoinThreads];
    tpb_grid_dep_launch();
    tpb_grid_dep_wait();
    const int c0 = (int)blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const JoinNote *from = reinterpret_cast<const JoinNote *>(p.notes) + c0;
    const int rows = __ldcg(&from->rows), n = __ldcg(&from->last_cta) - c0 + 1, row_tile = __ldcg(&from->row_tile), head = __ldcg(&from->head);
    const long long out_row = __ldcg(&from->out_row);
    // few rows: four threads (or two) share a row's dimensions, each with every fourth part
    const int each = (rows + (int)gridDim.y - 1) / (int)gridDim.y;
    const int shares = each * 4 <= kGroups ? 4 : each * 2 <= kGroups ? 2 : 1;
    const int rows_at_once = min(min(min(kGroups / shares, 32), max(each, 1)), max(kJoinFactors / max(n, 1), 1));
    const int lane4 = threadIdx.x % kLanes, group = threadIdx.x / kLanes, share = group % shares, rl = group / shares;
    for (int r0 = (int)blockIdx.y * rows_at_once; r0 < rows; r0 += (int)gridDim.y * rows_at_once) {
        const int rg = min(rows_at_once, rows - r0);
        const bool mine = rl < rg;
        const auto load_o = [&](int c) {
            return __ldcg(reinterpret_cast<const float4 *>(part_of(p.ws, HD, c0 + c, c == 0 ? 1 : 0).o + (size_t)(r0 + rl) * HD) + lane4);
        };
        float4 x[kJoinAhead];
#pragma unroll
        for (int i = 0; i < kJoinAhead; i++)
            if (mine && share + i * shares < n) x[i] = load_o(share + i * shares);
        float l[kPer];
#pragma unroll
        for (int i = 0; i < kPer; i++) {
            const int idx = threadIdx.x + i * kJoinThreads;
            if (idx < n * rg) {
                const int c = idx / rg, r = r0 + idx - c * rg;
                const Part part = part_of(p.ws, HD, c0 + c, c == 0 ? 1 : 0);
                s_ms[idx] = __ldcg(part.ms + r);
                s_mw[idx] = __ldcg(part.mw + r);
                l[i] = __ldcg(part.l + r);
            }
        }
        __syncthreads();
        for (int r = warp; r < rg; r += kJoinThreads / 32) {
            float big_s = -INFINITY, big_w = -INFINITY;
            for (int c = lane; c < n; c += 32) {
                big_s = fmaxf(big_s, s_ms[c * rg + r]);
                big_w = fmaxf(big_w, s_mw[c * rg + r]);
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                big_s = fmaxf(big_s, __shfl_xor_sync(0xffffffffu, big_s, o));
                big_w = fmaxf(big_w, __shfl_xor_sync(0xffffffffu, big_w, o));
            }
            if (lane == 0) {
                s_big[0][r] = big_s;
                s_big[1][r] = big_w;
            }
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kPer; i++) {
            const int idx = threadIdx.x + i * kJoinThreads;
            if (idx < n * rg) {
                const int r = idx % rg;
                s_l[idx] = l[i] * part_factor(s_ms[idx], s_big[0][r]);
                s_mw[idx] = part_factor(s_mw[idx], s_big[1][r]);
            }
        }
        __syncthreads();
        for (int r = warp; r < rg; r += kJoinThreads / 32) {
            float sum = 0.0f;
            for (int c = lane; c < n; c += 32) sum += s_l[c * rg + r];
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            if (lane == 0) s_sum[r] = sum;
        }
        float4 a = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        const auto add = [&](const float4 &y, int c) {
            const float f = s_mw[c * rg + rl];
            a.x += y.x * f;
            a.y += y.y * f;
            a.z += y.z * f;
            a.w += y.w * f;
        };
        if (mine) {
#pragma unroll
            for (int i = 0; i < kJoinAhead; i++)
                if (share + i * shares < n) add(x[i], share + i * shares);
#pragma unroll 4
            for (int c = share + kJoinAhead * shares; c < n; c += shares) add(load_o(c), c);
        }
        s_o[threadIdx.x] = a;
        __syncthreads();
        if (mine && share == 0) {
            for (int k = 1; k < shares; k++) {
                const float4 y = s_o[threadIdx.x + k * kLanes];
                a.x += y.x;
                a.y += y.y;
                a.z += y.z;
                a.w += y.w;
            }
            float second;
            const float f = finish_scale(s_big[0][rl], s_sum[rl], s_big[1][rl], second);
            const int flat = row_tile * RT + r0 + rl, tok = flat / p.group;
            store4(p, (out_row + tok) * p.ld_out + (long long)(head * p.group + flat - tok * p.group) * HD + 4 * lane4, a.x * f * second,
                   a.y * f * second, a.z * f * second, a.w * f * second);
        }
        __syncthreads();
    }
}

template <int HD, int FORMAT, bool SPLIT, int NT>
int launch_attention(tpb_handle_t h, cudaStream_t st, const AttnParams &p) {
    using C = Cfg<HD, SPLIT, NT>;
    static tpb_per_device_once smem_set;
    TPB_CUDA(h, tpb_set_max_smem_once(h, kv_attention_kernel<HD, FORMAT, SPLIT, NT>, C::kSmem, smem_set));
    const int ctas = h->sm_count * C::kCtas;
    TPB_CUDA(h, tpb_launch_pdl(kv_attention_kernel<HD, FORMAT, SPLIT, NT>, dim3((unsigned)ctas), dim3(kThreads), (size_t)C::kSmem, st, p));
    if (!p.whole)
        TPB_CUDA(h, tpb_launch_pdl(kv_attention_join_kernel<HD, C::kRows>, dim3((unsigned)ctas, HD == 128 && NT >= 2 ? 2 : 1), dim3(kJoinThreads), 0, st, p));
    return TPB_OK;
}

// Rows of a tile: 8, 16, 24 or 32, the fewest that hold what a sequence of average size has (their sums are in registers: no more than 32).
template <int HD, int FORMAT, bool SPLIT>
int by_rows(tpb_handle_t h, cudaStream_t st, const AttnParams &p) {
    const int64_t rows = ((int64_t)p.rows + p.n_seqs - 1) / p.n_seqs * p.group;
    return rows <= 8 ? launch_attention<HD, FORMAT, SPLIT, 1>(h, st, p)
                     : rows <= 16 ? launch_attention<HD, FORMAT, SPLIT, 2>(h, st, p)
                                  : rows <= 24 ? launch_attention<HD, FORMAT, SPLIT, 3>(h, st, p) : launch_attention<HD, FORMAT, SPLIT, 4>(h, st, p);
}
template <int HD, int FORMAT>
int by_type(tpb_handle_t h, cudaStream_t st, const AttnParams &p) {
    return p.dtype == TPB_BF16 ? by_rows<HD, FORMAT, false>(h, st, p) : by_rows<HD, FORMAT, true>(h, st, p);
}

}  // namespace

extern "C" {

size_t tpb_kv_attention_workspace_bytes(tpb_handle_t h, int head_dim) {
    if (!h || (head_dim != 64 && head_dim != 128)) return 0;
    const int ctas = h->sm_count * kMaxCtas;
    return ((size_t)ctas * 2 * slot_floats(head_dim) + note_floats(ctas)) * sizeof(float);
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
    const bool whole = max_len > 0 && max_len <= kMinTokens;
    TPB_CHECK_ARG(h, out && q && seqs && cu && (workspace || whole), "kv_attention: null pointer");
    const int64_t width = (int64_t)heads * c->head_dim, mult = dtype == TPB_F32 ? 4 : 8;
    TPB_CHECK_ARG(h, ld_q >= width && ld_out >= width && ld_q % mult == 0 && ld_out % mult == 0,
                  "kv_attention: ld_q and ld_out must be at least heads * head_dim and multiples of %lld", (long long)mult);
    TPB_CHECK_ARG(h, tpb_aligned16(out) && tpb_aligned16(q) && tpb_aligned16(workspace), "kv_attention: out, q and workspace must be 16-byte aligned");
    TPB_CHECK_ARG(h, ((reinterpret_cast<uintptr_t>(seqs) | reinterpret_cast<uintptr_t>(cu)) & 3u) == 0, "kv_attention: seqs and cu must be 4-byte aligned");
    TPB_CHECK_ARG(h, whole || workspace_bytes >= tpb_kv_attention_workspace_bytes(h, c->head_dim), "kv_attention: the workspace holds %zu bytes, %zu are needed",
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
    p.notes = p.ws + (size_t)h->sm_count * kMaxCtas * 2 * slot_floats(c->head_dim);
    p.status = h->d_status;
    // sequences known to be short stay whole, which saves the second launch (a longer one that comes all the same is one CTA's work)
    p.whole = whole;
    cudaStream_t st = (cudaStream_t)stream;
    if (c->head_dim == 64) return c->format == TPB_KV_S8 ? by_type<64, TPB_KV_S8>(h, st, p) : by_type<64, TPB_KV_E4M3>(h, st, p);
    return c->format == TPB_KV_S8 ? by_type<128, TPB_KV_S8>(h, st, p) : by_type<128, TPB_KV_E4M3>(h, st, p);
}

}  // extern "C"
