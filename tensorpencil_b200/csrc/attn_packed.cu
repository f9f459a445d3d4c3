// Causal attention over packed prompts for sm_100a: softmax(q k^T * scale) v per head on tcgen05 (kind::f16), grouped-query heads,
// head_dim 64 or 128, any number of sequences of any lengths.
//
// One pass over the keys with the running maximum and sum of the softmax: per tile of 128 keys
//   S = Q K^T          M 128 rows x N 128 keys x K head_dim, both operands from shared memory, f32 in tensor memory
//   P = exp2(S c - m)  one thread a row: its 128 scores in registers, reference point m and sum l per row
//   O += P V           M 128 x N head_dim x K 128; P (16 bits, two a column) lies over the first half of S and is read from tensor
//                      memory; V is the B operand as it lies in memory, head_dim contiguous ("MN-major"): no transpose pass
//
// Rows.  A tile's 128 rows are (token, query head of the group) pairs of one kv head: 128 / g tokens x g heads.  All of a group's heads
// share the K and V tiles, and short prompts fill a tile g times sooner than with one head a tile.  A CTA has two such tiles, A
// and B, of consecutive tokens: while the tensor pipe works for one, the other's softmax runs.  (Or one, in a small batch.)
//
// Roles: warps 0-3 / 4-7 softmax and output of tile A / B, warp 8 TMA, warp 9 MMA, warps 10 and 11 look V over.  MMAs of one thread execute in
// issue order, which is what frees the buffers: S_x(j+1) is issued after P_x(j) V(j).  With head_dim 64 tensor memory has room for a P beside
// S: there S_x(j+1) is issued as soon as S_x(j) is in registers (four prompts of 259 to 3001 tokens, 14 heads over 2: 46.5 -> 43.3 us).
// Every wait is bounded.
//
// A CTA that has work goes on to the pairs of CTAs that have not started, one after another, asked for when the last tile of keys of its own pair
// is loaded: the next pair's loads and first scores run under the last products and the output of the one before, where a CTA of its own
// would spend 4 us on starting and ending.
//
// What bounds it: of a step of 3400 cycles (a tile of keys against both tiles of queries, head_dim 128) the tensor pipe is busy for 2050, the
// special-function units for 2050; the rest is the way from one to the other -- scores out of tensor memory twice, weights back, four
// barriers.  Measured (bf16, 32 heads over 8): 8192 tokens 454 us, 1210 TFLOP/s; nine prompts of 1 to 2047 tokens 93 us.  What
// was measured and is not here: a pair of CTAs over tcgen05 cta_group::2, 705 us for the 8192 tokens; two threads a row, 503; a quarter of
// the exponentials by a polynomial on the FMA pipe, 489; a grid of CTAs of one pair each, 467.
//
// What a row must not see.  Scores of later tokens, other sequences and rows past the end are replaced before the maximum and
// their weights set to zero, so K's values there do not matter.  V's do, 0 * NaN being NaN: in the tiles that some row sees only a part of,
// warps 10 and 11 replace every NaN and infinity in shared memory by zero before the product and write down, per column,
// the first key of each kind that belongs to the sequence; the epilogue adds it to the rows that see that key.
#include <climits>
#include <type_traits>

#include "gemm_common.cuh"
#include "kv_common.cuh"

using namespace tpb_gemm;
using tpb_kv::find_sequence;
using tpb_kv::Found;

namespace {

constexpr int kTile = 128;
constexpr int kAtomBytes = 16384;     // [128 rows][64 values of 16 bits] in the 128-byte swizzle layout
constexpr int kThreads = 384;
constexpr int kStages = 2;
constexpr int kPlaces = 256;          // places without rows that a CTA passes over at most, 1 to 2 us each
// The reference point moves when the maximum has grown by more than 2^8.  It is a score times log2(e) rounded to f32, the exponents' arguments are not
// rounded before it is subtracted: from scores of 2^26 on the difference may leave the exponents' range, which the call's documentation rules out.
// Rounding them alike in those tiles alone was measured: nine prompts 93 -> 99 to 105 us, 8192 tokens 457 -> 465 to 489.
constexpr float kLazy = 8.0f;

template <int HD>
struct Layout {
    static constexpr int kAtoms = HD / 64;
    static constexpr bool kApart = HD == 64;                              // P has columns of its own in tensor memory
    static constexpr int kQ = 0;                                          // tiles A, B
    static constexpr int kK = kQ + 2 * kAtoms * kAtomBytes;
    static constexpr int kV = kK + kStages * kAtoms * kAtomBytes;
    static constexpr int kBar = kV + kStages * kAtoms * kAtomBytes;
    static constexpr int kPair = kBar + 256;                              // two Pairs, then the answer to the request for another one
    static constexpr int kBad = kPair + 128;                              // [2][3][HD] first NaN, +inf, -inf of a column, of every other pair
    static constexpr int kBytes = kBad + 2 * 3 * HD * 4 + 1024;
};

struct PackedParams {
    void *out;
    long long ld_out;             // elements
    const int32_t *cu;
    int n_seqs, tokens;
    int group, kv_heads, tile_tokens;      // query heads a kv head, 128 / group
    unsigned slots;
    int tiles;                    // of queries that a CTA has: 2 (A, B), or only A
    int take_more;                // there are more CTAs than SMs
    float scale_log2;
    uint32_t *status;
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint64_t pack_f2(float lo, float hi) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ void unpack_f2(uint64_t v, float &lo, float &hi) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t fma_f2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add_f2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_mma_ss(uint32_t one, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "setp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(one)
        : "memory");
}
__device__ __forceinline__ void tc_mma_ts(uint32_t one, uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "setp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(one)
        : "memory");
}
__device__ __forceinline__ void tc_commit_one(uint32_t one, uint32_t bar) {
    asm volatile(
        "{\n\t.reg .pred q;\n\t"
        "setp.ne.b32 q, %1, 0;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar), "r"(one)
        : "memory");
}
// 1 in one lane of a warp.  The MMA warp stays together and only its instructions are that lane's: descriptors and addresses are then the same for
// the whole warp and are kept where tcgen05.mma takes them from.  (A branch for lane 0 around all of it: 8192 tokens 481 us instead of 467.)
__device__ __forceinline__ uint32_t elect_one() {
    uint32_t one;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
    return one;
}
__device__ __forceinline__ void tc_st_16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
        "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void tc_ld_16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tc_wait_ld_16(uint32_t (&r)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
                 :
                 : "memory");
}
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap *map, uint32_t bar, int x, int y, int z) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst), "l"(map),
        "r"(bar), "r"(x), "r"(y), "r"(z)
        : "memory");
}
// V as B operand, head_dim contiguous: 8-key groups 1024 bytes apart (stride offset), the two halves of a 128-wide head an
// atom apart (leading offset).
__device__ __forceinline__ uint64_t make_mn_major_desc(uint32_t smem_addr) {
    uint64_t d = 0;
    d |= (uint64_t)((smem_addr >> 4) & 0x3FFFu);
    d |= (uint64_t)(kAtomBytes >> 4) << 16;
    d |= (uint64_t)(1024 >> 4) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}
// kind::f16, f32 accumulation, both operands of type T; N columns; B MN-major or K-major
template <typename T>
__device__ __forceinline__ uint32_t make_idesc(int n, bool b_mn) {
    const uint32_t type = std::is_same<T, __half>::value ? 0u : 1u;
    return (1u << 4) | (type << 7) | (type << 10) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(kTile >> 4) << 24);
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    if constexpr (std::is_same<T, __half>::value) {
        const __half2 h = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<const uint32_t *>(&h);
    } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
}

// A pair of tiles of one kv head: what a CTA works on at a time.
struct Pair {
    int head, start, len, pos0;          // start < 0: there is no more
};
// Asks for a CTA of the grid that has not started yet; 16 bytes at `answer` say which (or that there is none) once `bar` has counted them.
__device__ __forceinline__ void ask_next(uint32_t answer, uint32_t bar) {
    asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(answer), "r"(bar) : "memory");
}
__device__ __forceinline__ bool read_next(uint32_t answer, uint32_t &block) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .b128 h;\n\t.reg .pred p;\n\t"
        "ld.shared.b128 h, [%2];\n\t"
        "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, h;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t"
        "mov.b32 %1, 0;\n\t"
        "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, h;\n\t}"
        : "=r"(ok), "=r"(block)
        : "r"(answer)
        : "memory");
    return ok != 0;
}

template <typename T, int HD>
__global__ void __launch_bounds__(kThreads, 1)
attn_packed_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                   const PackedParams p) {
    using L = Layout<HD>;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t *gen = smem_raw + (smem_base - smem_u32(smem_raw));
    const uint32_t bars = smem_base + L::kBar;
    const auto q_full = [&](int x) { return bars + 8u * x; };
    const auto q_empty = [&](int x) { return bars + 8u * (2 + x); };
    const auto k_full = [&](int s) { return bars + 8u * (4 + s); };
    const auto k_empty = [&](int s) { return bars + 8u * (6 + s); };
    const auto v_full = [&](int s) { return bars + 8u * (8 + s); };
    const auto v_empty = [&](int s) { return bars + 8u * (10 + s); };
    const auto v_seen = [&](int s) { return bars + 8u * (12 + s); };     // looked over
    const auto s_full = [&](int x) { return bars + 8u * (14 + x); };
    const auto p_half = [&](int x) { return bars + 8u * (16 + x); };     // the first 64 keys' weights
    const auto p_full = [&](int x) { return bars + 8u * (18 + x); };
    const auto o_done = [&](int x) { return bars + 8u * (20 + x); };
    const auto pair_full = [&](int i) { return bars + 8u * (22 + (i & 1)); };
    const auto pair_empty = [&](int i) { return bars + 8u * (24 + (i & 1)); };
    const uint32_t answered = bars + 8u * 26;
    const auto s_read = [&](int x) { return smem_base + L::kPair + 64u + 8u * x; };     // kApart: the scores are in registers
    const auto pv_done = [&](int x) { return smem_base + L::kPair + 80u + 8u * x; };    // kApart: the products of a tile of keys are in O
    volatile uint32_t *tmem_slot = reinterpret_cast<volatile uint32_t *>(gen + L::kBar + 232);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(gen + L::kBar + 236);
    volatile int *any_bad = reinterpret_cast<volatile int *>(gen + L::kBar + 240);      // [2]
    const uint32_t answer = smem_base + L::kPair + 32;
    Pair *pairs = reinterpret_cast<Pair *>(gen + L::kPair);
    int *bad = reinterpret_cast<int *>(gen + L::kBad);

    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);          // alike in a warp, and known to be
    const int lane = threadIdx.x & 31;
    if (warp == 8 && lane < 3) {
        const CUtensorMap *map = lane == 0 ? &map_q : lane == 1 ? &map_k : &map_v;
        asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
    }
    tpb_grid_dep_launch();
    tpb_grid_dep_wait();

    // Which rows stand behind a block index.  Sequence s has at least as many places as it has pairs of tiles from cu[s] / pair_tokens + s on; the
    // last tiles of a sequence, which see the most keys, come first.  start < 0: none.  A whole warp calls it.
    const int pair_tokens = p.tiles * p.tile_tokens;
    const auto find_pair = [&](uint32_t block) {
        const int slot = (int)(p.slots - 1u - block / (unsigned)p.kv_heads);
        const Found b = find_sequence(p.cu, nullptr, p.n_seqs, p.tokens, slot, [&](int i, int r) { return r / pair_tokens + i; });
        const long long first = (long long)(slot - (b.r0 / pair_tokens + b.i)) * pair_tokens;      // position of tile A's first token
        const bool there = first >= 0 && first < b.r1 - b.r0;
        return Pair{(int)(block % (unsigned)p.kv_heads), there ? b.r0 : -1, b.r1 - b.r0, there ? (int)first : 0};
    };
    // The tiles of keys that tile x's last token sees the end of; 0: x has no tokens.
    const auto key_tiles = [&](const Pair &w, int x) {
        const int from = w.pos0 + x * p.tile_tokens, end = min(from + p.tile_tokens, w.len);
        return end > from && x < p.tiles ? (end + kTile - 1) / kTile : 0;
    };
    Pair now = find_pair(blockIdx.x);
    if (now.start < 0) return;

    // The first loads leave before anything else is set up: they take longer than all of it.  k and v stages are counted over all pairs.
    const auto load_q = [&](const Pair &w, int x) {
        mbar_arrive_expect_tx(q_full(x), (uint32_t)(L::kAtoms * 128 * p.tile_tokens * p.group));
        for (int a = 0; a < L::kAtoms; a++)
            tma_load_3d(smem_base + L::kQ + (x * L::kAtoms + a) * kAtomBytes, &map_q, q_full(x), a * 64, w.head * p.group,
                        w.start + w.pos0 + x * p.tile_tokens);
    };
    const auto load_k = [&](const Pair &w, int j, int st) {
        mbar_arrive_expect_tx(k_full(st), L::kAtoms * kAtomBytes);
        for (int a = 0; a < L::kAtoms; a++)
            tma_load_3d(smem_base + L::kK + (st * L::kAtoms + a) * kAtomBytes, &map_k, k_full(st), a * 64, w.head, w.start + j * kTile);
    };
    const auto load_v = [&](const Pair &w, int j, int st) {
        mbar_arrive_expect_tx(v_full(st), L::kAtoms * kAtomBytes);
        for (int a = 0; a < L::kAtoms; a++)
            tma_load_3d(smem_base + L::kV + (st * L::kAtoms + a) * kAtomBytes, &map_v, v_full(st), a * 64, w.head, w.start + j * kTile);
    };
    if (warp == 8 && lane == 0) {
        for (int s = 0; s < 2; s++) {
            mbar_init(q_full(s), 1);
            mbar_init(q_empty(s), 1);
            mbar_init(k_full(s), 1);
            mbar_init(k_empty(s), 1);
            mbar_init(v_full(s), 1);
            mbar_init(v_empty(s), 1);
            mbar_init(v_seen(s), 2);
            mbar_init(s_full(s), 1);
            mbar_init(p_half(s), 4);
            mbar_init(p_full(s), 4);
            mbar_init(o_done(s), 1);
            if (L::kApart) {
                mbar_init(s_read(s), 4);
                mbar_init(pv_done(s), 1);
            }
            mbar_init(pair_full(s), 1);
            mbar_init(pair_empty(s), 11);        // the softmax warps, the MMA warp, the two that look V over
            any_bad[s] = 0;
        }
        mbar_init(answered, 1);
        *abort_flag = 0;
        pairs[0] = now;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        mbar_arrive(pair_full(0));
        load_q(now, 0);
        load_k(now, 0, 0);
        if (key_tiles(now, 1) > 0) load_q(now, 1);
        load_v(now, 0, 0);
    }
    for (int i = threadIdx.x; i < 2 * 3 * HD; i += kThreads) bad[i] = INT_MAX;
    // Rows of a tile of queries that hold no token (128 / group has a remainder): zeros, or an infinity left there would move their reference
    // point tile after tile.
    const int used_rows = p.tile_tokens * p.group;
    for (int i = threadIdx.x; i < (kTile - used_rows) * 8 * 2 * L::kAtoms; i += kThreads)
        st_shared_v4(smem_base + L::kQ + (i / ((kTile - used_rows) * 8)) * kAtomBytes + used_rows * 128 + (i % ((kTile - used_rows) * 8)) * 16, 0u, 0u, 0u, 0u);
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    if (warp == 9) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32((const void *)tmem_slot)), "r"(512)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = __shfl_sync(0xffffffffu, *tmem_slot, 0);

    // Every role goes through the same pairs: the first is known, warp 8 tells of the others.
    bool ok = true;
    const auto next_pair = [&](int i) {              // pair i > 0, for a warp of the other roles; false: no more
        if (!p.take_more) return false;
        ok = ok && mbar_wait(pair_full(i), (uint32_t)(i >> 1) & 1u, abort_flag, p.status, (16u << 24) | 1u, true);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) return false;
        now = pairs[i & 1];
        return now.start >= 0;
    };
    const auto pair_over = [&](int i) {              // this warp is done with pair i
        __syncwarp();
        if (lane == 0) mbar_arrive(pair_empty(i));
    };

    if (warp < 8) {
        // ---------------- softmax and output: a thread per row ----------------
        const int x = warp >> 2;
        const int row = (warp & 3) * 32 + lane;
        const int row_tok = row / p.group, row_head = row - row_tok * p.group;
        const uint32_t t_lane = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t t_s = tmem_base + t_lane + (uint32_t)(x * 128);
        const uint32_t t_o = tmem_base + t_lane + 256u + (uint32_t)(x * HD);
        uint32_t phases = 0;                         // bit 0: of s_full, bit 1: of o_done
        for (int i = 0; i == 0 || next_pair(i); i++) {
            const int my_tiles = key_tiles(now, x);
            // position of the row's token; of the warp's pair only this and the tiles stay in registers
            const int pos = now.pos0 + x * p.tile_tokens + row_tok;
            const int lim = row_tok < p.tile_tokens && pos < now.len ? pos + 1 : 0;        // keys that the row sees
            float m_run = -3.402823466e38f, l_run = 0.0f;
            const auto do_tile = [&](auto masked_tag, const int j) -> bool {
                constexpr bool MASKED = decltype(masked_tag)::value;
                const bool good = mbar_wait(s_full(x), phases & 1u, abort_flag, p.status, (14u << 24) | 1u, true);
                phases ^= 1u;
                if (!__all_sync(0xffffffffu, good)) return false;
                tc_fence_after();
                const int left = lim - j * kTile;                    // columns >= left are hidden
                // The scores are read out of tensor memory twice, 32 columns ahead of their use: once for the maximum, once for the weights.
                uint32_t v[2][32];
                float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                tc_ld_32x32(t_s, v[0]);
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    tc_wait_ld_dep(v[c & 1]);
                    tc_ld_32x32(t_s + (uint32_t)(((c + 1) & 3) * 32), v[(c + 1) & 1]);
#pragma unroll
                    for (int e = 0; e < 32; e += 2) {
                        const float a = !MASKED || c * 32 + e < left ? __uint_as_float(v[c & 1][e]) : -INFINITY;
                        const float b = !MASKED || c * 32 + e + 1 < left ? __uint_as_float(v[c & 1][e + 1]) : -INFINITY;
                        m4[(e >> 1) & 3] = fmaxf(fmaxf(m4[(e >> 1) & 3], a), b);
                    }
                }
                const float m_cand = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])) * p.scale_log2;
                const float m_new = (m_cand > m_run + kLazy) ? m_cand : m_run;
                const float alpha = ex2(m_run - m_new);
                // O holds the products up to tile j - 1, and their weights may be written over: s_full of tile j was committed behind them, or they
                // are waited for
                if (L::kApart && j > 0) {
                    const bool there = mbar_wait(pv_done(x), phases & 1u, abort_flag, p.status, (14u << 24) | 2u, true);
                    if (!__all_sync(0xffffffffu, there)) return false;
                    tc_fence_after();
                }
                if (j > 0 && __any_sync(0xffffffffu, alpha != 1.0f)) {
#pragma unroll 1
                    for (int c = 0; c < HD / 16; c++) {
                        uint32_t o[16];
                        tc_ld_16(t_o + (uint32_t)(c * 16), o);
                        tc_wait_ld_16(o);
#pragma unroll
                        for (int e = 0; e < 16; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
                        tc_st_16(t_o + (uint32_t)(c * 16), o);
                    }
                }
                const uint64_t c2 = pack_f2(p.scale_log2, p.scale_log2), nm2 = pack_f2(-m_new, -m_new);
                uint64_t sum2[2] = {0ull, 0ull};
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    uint32_t pk[16];
                    tc_wait_ld_dep(v[c & 1]);
                    if (c < 3) tc_ld_32x32(t_s + (uint32_t)((c + 1) * 32), v[(c + 1) & 1]);
                    if (L::kApart && c == 3) {
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(s_read(x));
                    }
#pragma unroll
                    for (int e = 0; e < 16; e++) {
                        float a0, a1;
                        unpack_f2(fma_f2(pack_f2(__uint_as_float(v[c & 1][2 * e]), __uint_as_float(v[c & 1][2 * e + 1])), c2, nm2), a0, a1);
                        float e0 = ex2(a0), e1 = ex2(a1);
                        if (MASKED) {
                            if (c * 32 + 2 * e >= left) e0 = 0.0f;
                            if (c * 32 + 2 * e + 1 >= left) e1 = 0.0f;
                        }
                        sum2[e & 1] = add_f2(sum2[e & 1], pack_f2(e0, e1));
                        pk[e] = pack2<T>(e0, e1);
                    }
                    tc_st_16(L::kApart ? tmem_base + t_lane + (uint32_t)(384 + x * 64 + c * 16) : t_s + (uint32_t)(c * 16), pk);
                    if (c & 1) {
                        tc_wait_st();
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(c == 1 ? p_half(x) : p_full(x));
                    }
                }
                float s0, s1;
                unpack_f2(add_f2(sum2[0], sum2[1]), s0, s1);
                l_run = l_run * alpha + (s0 + s1);
                m_run = m_new;
                return true;
            };
            // A tile of keys that the first token sees as a whole needs no mask: rows behind the last token, or behind the last whole token of the
            // tile, come to nothing whatever they see.
            const int whole = pos - row_tok + 1;
            for (int j = 0; ok && j < my_tiles; j++) ok = (j + 1) * kTile <= whole ? do_tile(std::false_type{}, j) : do_tile(std::true_type{}, j);
            if (ok && my_tiles > 0) {
                ok = mbar_wait(o_done(x), phases >> 1, abort_flag, p.status, (14u << 24) | 3u, true);
                phases ^= 2u;
                ok = __all_sync(0xffffffffu, ok);
            }
            if (!ok) break;
            if (my_tiles > 0) {
                tc_fence_after();
                const float inv_l = 1.0f / l_run;
                const Pair w = pairs[i & 1];
                T *dst = static_cast<T *>(p.out) + (long long)(w.start + lim - 1) * p.ld_out + (long long)(w.head * p.group + row_head) * HD;
                const bool fix = any_bad[i & 1] != 0;
                const int *first_bad = bad + (i & 1) * 3 * HD;
#pragma unroll 1
                for (int c = 0; c < HD / 32; c++) {
                    uint32_t v[32];
                    tc_ld_32x32(t_o + (uint32_t)(c * 32), v);
                    tc_wait_ld_dep(v);
                    if (lim > 0) {
                        if (fix) {
#pragma unroll
                            for (int e = 0; e < 32; e++) {
                                float o = __uint_as_float(v[e]);
                                const int col = c * 32 + e;
                                if (lim > first_bad[col]) o += __uint_as_float(0x7fc00000u);
                                if (lim > first_bad[HD + col]) o += INFINITY;
                                if (lim > first_bad[2 * HD + col]) o -= INFINITY;
                                v[e] = __float_as_uint(o);
                            }
                        }
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            uint32_t o[4];
#pragma unroll
                            for (int h = 0; h < 4; h++)
                                o[h] = pack2<T>(__uint_as_float(v[8 * e + 2 * h]) * inv_l, __uint_as_float(v[8 * e + 2 * h + 1]) * inv_l);
                            reinterpret_cast<uint4 *>(dst + c * 32)[e] = make_uint4(o[0], o[1], o[2], o[3]);
                        }
                    }
                    __syncwarp();
                }
                tc_fence_before();          // O is read: the next pair's first weights, which this warp hands over later, let it be overwritten
            }
            pair_over(i);
        }
    } else if (warp == 8) {
        // ---------------- TMA, and which pair comes next ----------------
        uint32_t n_kv = 0, q_phase = 3u, n_asked = 0;         // bit x of q_phase: of q_empty
        const auto ask = [&] {
            mbar_arrive_expect_tx(answered, 16);
            ask_next(answer, answered);
        };
        for (int i = 0; ok; i++) {
            if (lane == 0) {
                for (int x = 0; ok && x < 2; x++) {
                    if (key_tiles(now, x) == 0) continue;
                    if (i > 0) {
                        ok = mbar_wait(q_empty(x), (q_phase >> x) & 1u, abort_flag, p.status, (12u << 24) | 0x30u | x, true);
                        if (ok) load_q(now, x);
                    }
                    q_phase ^= 1u << x;
                }
                const int tiles = max(key_tiles(now, 0), key_tiles(now, 1));
                for (int j = 0; ok && j < tiles; j++, n_kv++) {
                    // asked for no earlier than its loads need: a pair taken early waits here while another CTA has nothing to do
                    if (p.take_more && j + 1 == tiles) ask();
                    if (n_kv == 0) continue;                                       // left above
                    const int st = (int)(n_kv % kStages);
                    const uint32_t ph = (n_kv / kStages) & 1u;
                    ok = mbar_wait(k_empty(st), ph ^ 1u, abort_flag, p.status, (12u << 24) | 0x10u | st, true);
                    if (!ok) break;
                    load_k(now, j, st);
                    ok = mbar_wait(v_empty(st), ph ^ 1u, abort_flag, p.status, (12u << 24) | 0x20u | st, true);
                    if (!ok) break;
                    load_v(now, j, st);
                }
            }
            ok = __all_sync(0xffffffffu, ok);
            if (!ok || !p.take_more) break;
            for (int places = 0;; places++) {
                ok = mbar_wait(answered, n_asked++ & 1u, abort_flag, p.status, (12u << 24) | 0x40u, true);
                ok = __all_sync(0xffffffffu, ok);
                uint32_t block = 0;
                const bool there = ok && read_next(answer, block);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");       // read before the next answer is written
                now = {0, -1, 0, 0};
                if (!there) break;
                now = find_pair(block);
                // A place without rows is passed over.  After many the CTA ends, and those that are left start as CTAs: nobody waits for long.
                if (now.start >= 0 || places == kPlaces) break;
                __syncwarp();
                if (lane == 0) ask();
                __syncwarp();
            }
            if (ok && i > 0) ok = mbar_wait(pair_empty(i + 1), (uint32_t)((i - 1) >> 1) & 1u, abort_flag, p.status, (12u << 24) | 0x50u, true);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            const int b = (i + 1) & 1;
            if (any_bad[b]) {
                for (int c = lane; c < 3 * HD; c += 32) bad[b * 3 * HD + c] = INT_MAX;
                __syncwarp();
                if (lane == 0) any_bad[b] = 0;
            }
            if (lane == 0) pairs[b] = now;
            __syncwarp();
            if (lane == 0) mbar_arrive(pair_full(i + 1));
            if (now.start < 0) break;
        }
    } else if (warp == 9) {
        // ---------------- MMA ----------------
        uint32_t n_kv = 0, x_phase = 0, q_phase = 0;             // tiles of keys so far; bit x: of p_half and p_full, of q_full
        const uint32_t one = elect_one();
        for (int i = 0; i == 0 || next_pair(i); i++) {
            const auto wait = [&](uint32_t bar, uint32_t phase, uint32_t code) -> bool {
                const bool good = mbar_wait(bar, phase, abort_flag, p.status, (13u << 24) | code);
                return __all_sync(0xffffffffu, good);
            };
            const uint32_t idesc_qk = make_idesc<T>(kTile, false), idesc_pv = make_idesc<T>(HD, true);
            const int tiles_a = __shfl_sync(0xffffffffu, key_tiles(now, 0), 0), tiles_b = __shfl_sync(0xffffffffu, key_tiles(now, 1), 0);
            const int tiles = max(tiles_a, tiles_b);
            const auto issue_qk = [&](int x, uint32_t n, bool last) {
                const uint32_t ka = smem_base + L::kK + (n % kStages) * L::kAtoms * kAtomBytes;
                const uint32_t qa = smem_base + L::kQ + x * L::kAtoms * kAtomBytes;
#pragma unroll
                for (int a = 0; a < L::kAtoms; a++) {
                    const uint64_t qd = make_kmajor_sw128_desc(qa + a * kAtomBytes), kd = make_kmajor_sw128_desc(ka + a * kAtomBytes);
#pragma unroll
                    for (int kk = 0; kk < 4; kk++)
                        tc_mma_ss(one, tmem_base + (uint32_t)(x * 128), qd + 2u * kk, kd + 2u * kk, idesc_qk, (a | kk) ? 1u : 0u);
                }
                tc_commit_one(one, s_full(x));
                if (last) tc_commit_one(one, q_empty(x));
            };
            const auto issue_pv = [&](int x, int j, int part) {
                const uint64_t vd = make_mn_major_desc(smem_base + L::kV + ((n_kv + j) % kStages) * L::kAtoms * kAtomBytes);
#pragma unroll
                for (int k2 = 0; k2 < 4; k2++) {
                    const int kk = 4 * part + k2;           // 16 keys: 8 columns of P, 2048 bytes of V
                    tc_mma_ts(one, tmem_base + 256u + (uint32_t)(x * HD), tmem_base + (uint32_t)((L::kApart ? 384 + x * 64 : x * 128) + 8 * kk),
                              vd + 128u * kk, idesc_pv, (j > 0 || kk > 0) ? 1u : 0u);
                }
            };
            ok = ok && wait(q_full(0), q_phase & 1u, 1u);
            q_phase ^= 1u;
            if (ok) ok = wait(k_full(n_kv % kStages), (n_kv / kStages) & 1u, 2u);
            if (ok) {
                tc_fence_after();
                issue_qk(0, n_kv, tiles_a == 1);
                if (tiles_b > 0) {
                    ok = wait(q_full(1), q_phase >> 1, 9u);
                    q_phase ^= 2u;
                    if (ok) issue_qk(1, n_kv, tiles_b == 1);
                }
                tc_commit_one(one, k_empty(n_kv % kStages));
            }
            for (int j = 0; ok && j < tiles; j++) {
                const uint32_t n = n_kv + j, st = n % kStages, st1 = (n + 1) % kStages;
                const bool more = j + 1 < tiles;
                ok = wait(v_seen(st), (n / kStages) & 1u, 3u);
                bool k_there = false;
#pragma unroll
                for (int x = 0; x < 2; x++) {
                    if (!ok) break;
                    const int mine = x ? tiles_b : tiles_a;
                    if (j < mine) {
                        ok = wait(p_half(x), (x_phase >> x) & 1u, 4u);
                        if (!ok) break;
                        tc_fence_after();
                        issue_pv(x, j, 0);
                        if (L::kApart && j + 1 < mine) {
                            ok = wait(s_read(x), (x_phase >> x) & 1u, 7u);
                            if (!ok) break;
                            tc_fence_after();
                            if (!k_there) {
                                ok = wait(k_full(st1), ((n + 1) / kStages) & 1u, 6u);
                                if (!ok) break;
                                tc_fence_after();
                                k_there = true;
                            }
                            issue_qk(x, n + 1, j + 2 == mine);
                        }
                        ok = wait(p_full(x), (x_phase >> x) & 1u, 5u);
                        x_phase ^= 1u << x;
                        if (!ok) break;
                        tc_fence_after();
                        issue_pv(x, j, 1);
                        if (L::kApart) tc_commit_one(one, pv_done(x));
                        if (j + 1 == mine) tc_commit_one(one, o_done(x));
                    }
                    if (x == 1) tc_commit_one(one, v_empty(st));
                    if (!L::kApart && j + 1 < mine) {
                        if (!k_there) {
                            ok = wait(k_full(st1), ((n + 1) / kStages) & 1u, 6u);
                            if (!ok) break;
                            tc_fence_after();
                            k_there = true;
                        }
                        issue_qk(x, n + 1, j + 2 == mine);
                    }
                }
                if (ok && more) tc_commit_one(one, k_empty(st1));
            }
            n_kv += tiles;
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            pair_over(i);
        }
    } else {
        // ---------------- V: warps 10 and 11, half of a tile's rows each ----------------
        constexpr uint32_t kExp = std::is_same<T, __half>::value ? 0x7c007c00u : 0x7f807f80u;      // exponent all ones: NaN or infinity
        constexpr uint32_t kOne = std::is_same<T, __half>::value ? 0x04000400u : 0x00800080u;
        uint32_t n_kv = 0;
        for (int i = 0; i == 0 || next_pair(i); i++) {
            const int tiles = max(key_tiles(now, 0), key_tiles(now, 1));
            const int look_from = (now.pos0 + 1) / kTile;           // first tile of keys that tile A's first token does not see as a whole
            int *first_bad = bad + (i & 1) * 3 * HD;
            for (int j = 0; ok && j < tiles; j++, n_kv++) {
                const int st = (int)(n_kv % kStages);
                ok = mbar_wait(v_full(st), (n_kv / kStages) & 1u, abort_flag, p.status, (15u << 24) | 1u, true);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                if (j >= look_from) {
                    for (int a = 0; a < L::kAtoms; a++) {
                        const uint32_t base = smem_base + L::kV + (st * L::kAtoms + a) * kAtomBytes + (uint32_t)(warp - 10) * (kAtomBytes / 2);
#pragma unroll 4
                        for (int c = lane; c < kAtomBytes / 32; c += 32) {
                            const uint4 w = ld_shared_v4(base + 16u * c);
                            const uint32_t hit = (((w.x & kExp) + kOne) | ((w.y & kExp) + kOne) | ((w.z & kExp) + kOne) | ((w.w & kExp) + kOne)) & 0x80008000u;
                            if (hit) {
                                const int row = (warp - 10) * 64 + c / 8, key = j * kTile + row;
                                const int col0 = a * 64 + ((c & 7) ^ (row & 7)) * 8;
                                uint32_t u[4] = {w.x, w.y, w.z, w.w};
                                for (int e = 0; e < 8; e++) {
                                    const uint32_t h = (u[e >> 1] >> (16 * (e & 1))) & 0xffffu, ex = kExp & 0xffffu;
                                    if ((h & ex) != ex) continue;
                                    if (key < now.len) {
                                        const int kind = (h & ~(ex | 0x8000u) & 0xffffu) != 0 ? 0 : (h & 0x8000u) ? 2 : 1;
                                        atomicMin(first_bad + kind * HD + col0 + e, key);
                                        any_bad[i & 1] = 1;
                                    }
                                    u[e >> 1] &= ~(0xffffu << (16 * (e & 1)));
                                }
                                st_shared_v4(base + 16u * c, u[0], u[1], u[2], u[3]);
                            }
                        }
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(v_seen(st));
            }
            if (!ok) break;
            pair_over(i);
        }
    }

    // ---------------- teardown ----------------
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (*abort_flag) {          // copies may be in flight: let them land before the memory goes
        for (int i = 0; i < 200; i++) __nanosleep(1000);
        __syncthreads();
    }
    if (warp == 9) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(512) : "memory");
    }
}

// [tokens][heads][hd] with rows ld elements apart; a box is 64 columns x `box_heads` heads x `box_tokens` tokens, swizzled by 128 bytes
int make_map(tpb_handle_t h, CUtensorMap *map, int dtype, const void *base, int64_t tokens, int heads, int hd, int64_t ld, int box_heads,
             int box_tokens) {
    const cuuint64_t dim[3] = {(cuuint64_t)hd, (cuuint64_t)heads, (cuuint64_t)tokens};
    const cuuint64_t stride[2] = {(cuuint64_t)hd * 2, (cuuint64_t)ld * 2};
    const cuuint32_t box[3] = {64u, (cuuint32_t)box_heads, (cuuint32_t)box_tokens};
    const cuuint32_t step[3] = {1, 1, 1};
    const CUresult r = reinterpret_cast<EncodeTiledFn>(h->encode_tiled)(
        map, dtype == TPB_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void *>(base), dim, stride, box,
        step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return tpb_fail(h, TPB_ERR_CUDA, "cuTensorMapEncodeTiled (packed attention) failed (%d)", (int)r);
    return TPB_OK;
}

template <typename T, int HD>
int launch_packed(tpb_handle_t h, cudaStream_t st, const CUtensorMap &mq, const CUtensorMap &mk, const CUtensorMap &mv, const PackedParams &p) {
    static tpb_per_device_once smem_set;
    TPB_CUDA(h, tpb_set_max_smem_once(h, attn_packed_kernel<T, HD>, Layout<HD>::kBytes, smem_set));
    TPB_CUDA(h, tpb_launch_pdl(attn_packed_kernel<T, HD>, dim3(p.slots * (unsigned)p.kv_heads), dim3(kThreads), (size_t)Layout<HD>::kBytes, st, mq, mk,
                               mv, p));
    return TPB_OK;
}

}  // namespace

extern "C" {

int tpb_attention_packed(tpb_handle_t h, tpb_stream_t stream, void *out, int64_t ld_out, const void *q, int64_t ld_q,
                         const void *k, int64_t ld_k, const void *v, int64_t ld_v, int dtype, const int32_t *cu, int n_seqs,
                         int64_t tokens, int heads, int kv_heads, int head_dim, float scale) {
    if (!h) return TPB_ERR_INVALID_ARG;
    TPB_CHECK_ARG(h, dtype == TPB_BF16 || dtype == TPB_F16, "attention_packed: tensors must be bf16 or f16");
    TPB_CHECK_ARG(h, head_dim == 64 || head_dim == 128, "attention_packed: head_dim must be 64 or 128 (got %d)", head_dim);
    TPB_CHECK_ARG(h, heads > 0 && kv_heads > 0 && kv_heads <= 65535 && heads % kv_heads == 0 && heads / kv_heads <= 128,
                  "attention_packed: heads must be a multiple of kv_heads, at most 128 times as many");
    TPB_CHECK_ARG(h, n_seqs >= 0 && n_seqs < (1 << 24) && tokens >= 0 && tokens < (1 << 26), "attention_packed: bad n_seqs / tokens");
    TPB_CHECK_ARG(h, scale >= 0.0f && scale <= 3.4e38f, "attention_packed: scale must be finite and not negative");
    if (n_seqs == 0 || tokens == 0) return TPB_OK;
    TPB_CHECK_ARG(h, out && q && k && v && cu, "attention_packed: null pointer");
    const int64_t wq = (int64_t)heads * head_dim, wk = (int64_t)kv_heads * head_dim;
    TPB_CHECK_ARG(h, ld_out >= wq && ld_q >= wq && ld_k >= wk && ld_v >= wk, "attention_packed: a row stride is smaller than its row");
    TPB_CHECK_ARG(h, (ld_out | ld_q | ld_k | ld_v) % 8 == 0 && (ld_out | ld_q | ld_k | ld_v) < ((int64_t)1 << 38),
                  "attention_packed: row strides must be multiples of 8 elements");
    TPB_CHECK_ARG(h, tpb_aligned16(out) && tpb_aligned16(q) && tpb_aligned16(k) && tpb_aligned16(v) && (reinterpret_cast<uintptr_t>(cu) & 3u) == 0,
                  "attention_packed: pointers must be 16-byte aligned (cu: 4)");
    PackedParams p;
    p.out = out;
    p.ld_out = ld_out;
    p.cu = cu;
    p.n_seqs = n_seqs;
    p.tokens = (int)tokens;
    p.group = heads / kv_heads;
    p.kv_heads = kv_heads;
    p.tile_tokens = kTile / p.group;
    p.scale_log2 = scale * 1.4426950408889634f;
    p.status = h->d_status;
    // Two tiles share a CTA, whose steps are longer for it, where there is work for all SMs.  Where the SMs have room for all tiles at once, each has a
    // CTA of its own; also up to two a SM if the sequences are long, since the early tiles are soon done with.  Measured (two tiles / one; head_dim 128,
    // bf16): 1595 tokens, 8 heads over 1 29.5 / 24.7 us; 2048 tokens, 16 over 2 36.8 / 31.4; 1024 tokens, 32 over 4 22.4 / 21.9; twice 400 tokens, 32 over 8
    // 13.3 / 14.7.
    const int64_t alone = tokens / p.tile_tokens + n_seqs;
    p.tiles = alone * kv_heads <= (tokens >= 1024 * (int64_t)n_seqs ? 2 : 1) * h->sm_count ? 1 : 2;
    const int64_t slots = p.tiles == 1 ? alone : tokens / (2 * p.tile_tokens) + n_seqs;
    TPB_CHECK_ARG(h, slots * kv_heads < INT32_MAX, "attention_packed: tokens * heads exceeds the grid");
    p.slots = (unsigned)slots;
    p.take_more = slots * kv_heads > h->sm_count;
    tpb_device_guard guard(h->device);
    TPB_CUDA(h, guard.err);
    CUtensorMap mq, mk, mv;
    int rc = make_map(h, &mq, dtype, q, tokens, heads, head_dim, ld_q, p.group, p.tile_tokens);
    if (rc == TPB_OK) rc = make_map(h, &mk, dtype, k, tokens, kv_heads, head_dim, ld_k, 1, kTile);
    if (rc == TPB_OK) rc = make_map(h, &mv, dtype, v, tokens, kv_heads, head_dim, ld_v, 1, kTile);
    if (rc != TPB_OK) return rc;
    cudaStream_t st = (cudaStream_t)stream;
    if (dtype == TPB_BF16)
        return head_dim == 64 ? launch_packed<__nv_bfloat16, 64>(h, st, mq, mk, mv, p) : launch_packed<__nv_bfloat16, 128>(h, st, mq, mk, mv, p);
    return head_dim == 64 ? launch_packed<__half, 64>(h, st, mq, mk, mv, p) : launch_packed<__half, 128>(h, st, mq, mk, mv, p);
}

}  // extern "C"
