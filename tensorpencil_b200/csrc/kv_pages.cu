// Pages of the 8-bit key / value cache: extend, truncate, fork, compact.
//
// The bookkeeping of an operation -- a few thousand integers -- is one CTA's work: it checks the whole list before it changes anything, takes
// pages from the ascending list of free ones (a scan of the reference counts), and leaves the copies of pages, if any, to a second kernel
// that spreads them over the device.  Every choice is by index (lowest free page first, in the list's order), so the tables
// after an operation depend on the tables before it alone.
#include "kv_common.cuh"

using namespace tpb_kv;

namespace {

constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;

__device__ __forceinline__ int pages_of(const tpb_kv_cache &c, int len) { return (len + c.page_tokens - 1) / c.page_tokens; }

// Exclusive scan over the block of one value a thread.
__device__ __forceinline__ long long block_scan(long long v, long long *buf, long long &total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    long long inc = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long t = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += t;
    }
    __syncthreads();
    if (lane == 31) buf[warp] = inc;
    __syncthreads();
    long long sums = buf[lane];                 // every warp scans the warps' sums: a loop over them costs each caller 0.5 us
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long t = __shfl_up_sync(0xffffffffu, sums, o);
        if (lane >= o) sums += t;
    }
    total = __shfl_sync(0xffffffffu, sums, 31);
    const long long up_to = __shfl_sync(0xffffffffu, sums, warp > 0 ? warp - 1 : 0);
    const long long base = warp > 0 ? up_to : 0;
    return base + inc - v;
}

// The pool's reference counts as a block sees them: a warp has consecutive pages, a multiple of 128 of them, four a lane and step.  The first
// kHeld steps (16384 pages in all) stay in registers from one pass to the next; a pass behind those reads again.
constexpr int kHeld = 4;
constexpr int kOutside = 1;    // pages behind the pool's end are neither free ...
struct Refs {
    int begin, end;
    int4 held[kHeld];
};
__device__ __forceinline__ int4 refs4(const tpb_kv_cache &c, int p, int end) {
    int4 v = make_int4(kOutside, kOutside, kOutside, kOutside);
    if (p + 3 < end) {
        const int32_t *r = c.refs + p;
        if ((reinterpret_cast<uintptr_t>(r) & 15u) == 0) return __ldcg(reinterpret_cast<const int4 *>(r));
        return make_int4(__ldcg(r), __ldcg(r + 1), __ldcg(r + 2), __ldcg(r + 3));
    }
    if (p < end) v.x = __ldcg(c.refs + p);
    if (p + 1 < end) v.y = __ldcg(c.refs + p + 1);
    if (p + 2 < end) v.z = __ldcg(c.refs + p + 2);
    return v;
}
__device__ __forceinline__ void load_refs(const tpb_kv_cache &c, Refs &f) {
    const int per = (int)((c.n_pages + kWarps * 128 - 1) / (kWarps * 128)) * 128;
    const long long b = (long long)per * (threadIdx.x >> 5);
    f.begin = (int)min(b, (long long)c.n_pages);
    f.end = (int)min(b + per, (long long)c.n_pages);
#pragma unroll
    for (int i = 0; i < kHeld; i++) f.held[i] = refs4(c, f.begin + 128 * i + 4 * (threadIdx.x & 31), f.end);
}
// Calls fn(page, its reference count and those of the three behind it) for the lane's pages, in order, the whole warp together; fn returns whether
// to go on.
template <typename Fn>
__device__ __forceinline__ void each_quad(const tpb_kv_cache &c, const Refs &f, Fn fn) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int i = 0; i < kHeld; i++)
        if (f.begin + 128 * i < f.end && !fn(f.begin + 128 * i + 4 * lane, f.held[i])) return;
#pragma unroll 2
    for (int p = f.begin + 128 * kHeld; p < f.end; p += 128)
        if (!fn(p + 4 * lane, refs4(c, p + 4 * lane, f.end))) return;
}

// Pages for which pick(page, refs) holds, counted over the block (the total) and in front of this warp's pages (`before`).
template <typename Pick>
__device__ long long count_pages(const tpb_kv_cache &c, const Refs &f, long long *buf, long long &before, Pick pick) {
    int n = 0;
    each_quad(c, f, [&](int p, const int4 &r) {
        n += (int)pick(p, r.x) + (int)pick(p + 1, r.y) + (int)pick(p + 2, r.z) + (int)pick(p + 3, r.w);
        return true;
    });
    n = __reduce_add_sync(0xffffffffu, n);
    long long total;
    const long long at = block_scan((threadIdx.x & 31) == 0 ? n : 0, buf, total);
    before = __shfl_sync(0xffffffffu, at, 0);
    return total;
}
// Their indices in ascending order into list[0 .. want); `before` from count_pages with the same pick.
template <typename Pick>
__device__ void list_pages(const tpb_kv_cache &c, const Refs &f, int32_t *list, long long before, long long want, Pick pick) {
    const int lane = threadIdx.x & 31;
    long long at = before;
    if (at >= want) return;
    each_quad(c, f, [&](int p, const int4 &r) {
        const bool q[4] = {pick(p, r.x), pick(p + 1, r.y), pick(p + 2, r.z), pick(p + 3, r.w)};
        const int n = (int)q[0] + (int)q[1] + (int)q[2] + (int)q[3];
        int inc = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int t = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += t;
        }
        long long mine = at + inc - n;
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (q[e]) {
                if (mine < want) list[mine] = p + e;
                mine++;
            }
        at += __shfl_sync(0xffffffffu, inc, 31);
        return at < want;
    });
}

__device__ __forceinline__ bool is_free(int, int refs) { return refs == 0; }

__device__ __forceinline__ void set_result(const tpb_kv_cache &c, int status, long long free_pages, long long taken, long long needed) {
    if (threadIdx.x != 0) return;
    c.result[0] = status;
    c.result[1] = (int)free_pages;
    c.result[2] = (int)taken;
    c.result[3] = (int)min(needed, (long long)INT32_MAX);
}

// A list of the call's: its entry threadIdx.x is asked for at once, and the first kSmallList entries are in shared memory from then on (a null list: all
// zero).  at() may be used behind the next barrier, by any thread; mine() at once, for i = threadIdx.x + k kThreads.
constexpr int kSmallList = 1024;
static_assert(kSmallList == kThreads, "a thread keeps one entry");
struct Listed {
    const int32_t *list;
    int32_t *kept;
    int first;
    __device__ Listed(const int32_t *l, int n, int32_t *smem) : list(l), kept(smem), first(l && (int)threadIdx.x < n ? __ldcg(l + threadIdx.x) : 0) {
        kept[threadIdx.x] = first;
    }
    __device__ int mine(int i) const { return i < kThreads ? first : list ? __ldcg(list + i) : 0; }
    __device__ int at(int i) const { return i < kSmallList ? kept[i] : list ? __ldcg(list + i) : 0; }
};

// A mark a sequence: bits in shared memory for up to kMarkBits sequences, else words of the cache's scratch (marks of the ids in question only).
constexpr int kMarkBits = 32768;
struct Marks {
    uint32_t *bits;
    int32_t *words;
    bool small;
    __device__ void clear_bits(int max_seqs) const {             // before anything else
        if (small)
            for (int i = threadIdx.x; i < (max_seqs + 31) / 32; i += kThreads) bits[i] = 0;
    }
    __device__ void clear_words(const Listed &ids, int n, int max_seqs) const {
        if (small) return;
        for (int i = threadIdx.x; i < n; i += kThreads) {
            const int id = ids.mine(i);
            if (id >= 0 && id < max_seqs) words[id] = 0;
        }
    }
    __device__ bool set(int id) const {           // was it set?
        if (small) return (atomicOr(bits + (id >> 5), 1u << (id & 31)) >> (id & 31)) & 1u;
        return atomicAdd(words + id, 1) != 0;
    }
    __device__ bool test(int id) const { return small ? (bits[id >> 5] >> (id & 31)) & 1u : __ldcg(words + id) != 0; }
};

// A CTA's bookkeeping is a chain of dependent loads and barriers, 0.3 to 0.5 us each, so what does not depend on one another is asked for
// together (the lists, the reference counts), what a later pass needs stays in registers, and lists, lengths, offsets and marks are in shared memory.
// fork + truncate of 32 sequences over 1300 pages, with the copies: 28 -> 19 us.
__global__ void __launch_bounds__(kThreads)
kv_extend_kernel(const tpb_kv_cache c, const int32_t *seqs, const int32_t *n_new, int n) {
    __shared__ long long buf[kWarps];
    __shared__ uint32_t bits[kMarkBits / 32];
    __shared__ int32_t small_offsets[kSmallList], small_list[kSmallList], small_ids[kSmallList], small_adds[kSmallList], small_lens[kSmallList];
    const Scratch sc = scratch_of(c);
    const Marks marks{bits, sc.marks, c.max_seqs <= kMarkBits};
    marks.clear_bits(c.max_seqs);
    tpb_grid_dep_launch();
    tpb_grid_dep_wait();
    const Listed ids(seqs, n, small_ids), adds(n_new, n, small_adds);
    Refs refs;
    load_refs(c, refs);
    int32_t *offsets = n <= kSmallList ? small_offsets : sc.offsets;
    const long long most = (long long)c.max_pages * c.page_tokens;
    marks.clear_words(ids, n, c.max_seqs);
    __syncthreads();
    bool ok = true;
    for (int i = threadIdx.x; i < n; i += kThreads) {
        const int id = ids.mine(i);
        if (id < 0 || id >= c.max_seqs || marks.set(id)) ok = false;
    }
    long long before = 0;
    const long long free_pages = count_pages(c, refs, buf, before, is_free);
    ok = __syncthreads_and(ok);
    long long need = 0;
    if (ok) {
        for (int i0 = 0; i0 < n; i0 += kThreads) {
            const int i = i0 + threadIdx.x;
            int want = 0;
            if (i < n) {
                const int len = __ldcg(c.lens + ids.mine(i)), add = adds.mine(i);
                if (i < kSmallList) small_lens[i] = len;
                if (len < 0 || add < 0 || (long long)len + add > most) ok = false;
                else want = pages_of(c, len + add) - pages_of(c, len);
            }
            long long total;
            const long long at = block_scan(want, buf, total);
            if (i < n) offsets[i] = (int)min(need + at, (long long)INT32_MAX);
            need += total;
        }
        ok = __syncthreads_and(ok);
    }
    if (!ok || need > free_pages) {
        for (int i = threadIdx.x; i < n; i += kThreads) {
            const int id = ids.mine(i);
            if (id >= 0 && id < c.max_seqs) c.tail[id] = 0;
        }
        set_result(c, ok ? TPB_ERR_OOM : TPB_ERR_INVALID_ARG, free_pages, 0, ok ? need : 0);
        return;
    }
    int32_t *list = need <= kSmallList ? small_list : sc.list_a;
    list_pages(c, refs, list, before, need, is_free);
    __syncthreads();
    const int lane = threadIdx.x & 31;
    for (int i = threadIdx.x >> 5; i < n; i += kWarps) {
        const int id = ids.at(i), add = adds.at(i), len = i < kSmallList ? small_lens[i] : __ldcg(c.lens + id);
        const int p0 = pages_of(c, len), p1 = pages_of(c, len + add), at = offsets[i];
        for (int p = p0 + lane; p < p1; p += 32) {
            const int page = list[at + p - p0];
            c.table[(size_t)id * c.max_pages + p] = page;
            c.refs[page] = 1;
        }
        __syncwarp();
        if (lane == 0) {
            c.lens[id] = len + add;
            c.tail[id] = add;
        }
    }
    set_result(c, TPB_OK, free_pages - need, need, need);
}

// Entries p0 .. p1 of a sequence's row of the table, a lane each, as fn(p, page); an entry that is no page is reported and left out.
template <typename Fn>
__device__ __forceinline__ void each_page(const tpb_kv_cache &c, int id, int p0, int p1, uint32_t *status, Fn fn) {
#pragma unroll 4
    for (int p = p0 + (int)(threadIdx.x & 31); p < p1; p += 32) {
        const int page = __ldcg(c.table + (size_t)id * c.max_pages + p);
        if (page < 0 || page >= c.n_pages) report(status, kBadPage);
        else fn(p, page);
    }
}

__global__ void __launch_bounds__(kThreads)
kv_truncate_kernel(const tpb_kv_cache c, const int32_t *seqs, const int32_t *new_lens, int n, uint32_t *status) {
    __shared__ long long buf[kWarps];
    __shared__ uint32_t bits[kMarkBits / 32];
    __shared__ int32_t small_ids[kSmallList], small_cuts[kSmallList], small_lens[kSmallList];
    const Scratch sc = scratch_of(c);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const Marks marks{bits, sc.marks, c.max_seqs <= kMarkBits};
    marks.clear_bits(c.max_seqs);
    tpb_grid_dep_launch();
    tpb_grid_dep_wait();
    const Listed ids(seqs, n, small_ids), cuts(new_lens, n, small_cuts);
    marks.clear_words(ids, n, c.max_seqs);
    __syncthreads();
    bool ok = true;
    for (int i = threadIdx.x; i < n; i += kThreads) {
        const int id = ids.mine(i);
        if (id < 0 || id >= c.max_seqs || marks.set(id)) {
            ok = false;
        } else {
            const int len = __ldcg(c.lens + id), to = cuts.mine(i);
            if (i < kSmallList) small_lens[i] = len;
            if (len < 0 || to < 0 || to > len || (long long)len > (long long)c.max_pages * c.page_tokens) ok = false;
        }
    }
    ok = __syncthreads_and(ok);
    long long before = 0;
    Refs refs;
    if (!ok) {
        load_refs(c, refs);
        const long long free_pages = count_pages(c, refs, buf, before, is_free);
        if (threadIdx.x == 0) sc.head[0] = 0;
        set_result(c, TPB_ERR_INVALID_ARG, free_pages, 0, 0);
        return;
    }
    const auto old_len = [&](int i) { return i < kSmallList ? small_lens[i] : __ldcg(c.lens + ids.at(i)); };
    // give back the pages behind the cuts; `by` = 1 takes it back.  Where nothing can stop the operation any more, the rows are cleared at once.
    const auto drop = [&](int by, bool clear) {
        for (int i = warp; i < n; i += kWarps) {
            const int id = ids.at(i), p1 = pages_of(c, old_len(i));
            each_page(c, id, pages_of(c, cuts.at(i)), p1, status, [&](int p, int page) {
                atomicAdd(c.refs + page, by);
                if (clear) c.table[(size_t)id * c.max_pages + p] = -1;
            });
            __syncwarp();
            if (clear && lane == 0) {
                c.lens[id] = 0;
                c.tail[id] = 0;
            }
        }
        __syncthreads();
    };
    if (!new_lens) {              // freed: no cut inside a page
        drop(-1, true);
        load_refs(c, refs);
        const long long free_pages = count_pages(c, refs, buf, before, is_free);
        set_result(c, TPB_OK, free_pages, 0, 0);
        return;
    }
    drop(-1, false);
    // a cut inside a page that somebody else holds too: the sequence gets a page of its own for what it keeps of it
    load_refs(c, refs);
    long long need = 0;
    for (int i0 = 0; i0 < n; i0 += kThreads) {
        const int i = i0 + threadIdx.x;
        bool cut = false;
        if (i < n) {
            const int to = cuts.mine(i);
            if (to % c.page_tokens != 0) {
                const int page = __ldcg(c.table + (size_t)ids.mine(i) * c.max_pages + to / c.page_tokens);
                if (page < 0 || page >= c.n_pages) report(status, kBadPage);
                else cut = __ldcg(c.refs + page) > 1;
            }
        }
        long long total;
        const long long at = block_scan(cut ? 1 : 0, buf, total);
        if (i < n) sc.offsets[i] = cut ? (int)(need + at) : -1;
        need += total;
    }
    const long long free_pages = count_pages(c, refs, buf, before, is_free);
    if (need > free_pages) {
        drop(1, false);
        load_refs(c, refs);
        const long long left = count_pages(c, refs, buf, before, is_free);
        if (threadIdx.x == 0) sc.head[0] = 0;
        set_result(c, TPB_ERR_OOM, left, 0, need);
        return;
    }
    list_pages(c, refs, sc.list_b, before, need, is_free);
    __syncthreads();
    for (int i = warp; i < n; i += kWarps) {
        const int id = ids.at(i), to = cuts.at(i), p0 = pages_of(c, to), p1 = pages_of(c, old_len(i));
        int32_t *row = c.table + (size_t)id * c.max_pages;
        for (int p = p0 + lane; p < p1; p += 32) row[p] = -1;
        __syncwarp();
        if (lane == 0) {
            c.lens[id] = to;
            c.tail[id] = 0;
            const int at = sc.offsets[i];
            if (at >= 0) {
                const int from = __ldcg(row + p0 - 1), fresh = sc.list_b[at];
                sc.list_a[at] = from;
                atomicAdd(c.refs + from, -1);
                c.refs[fresh] = 1;
                row[p0 - 1] = fresh;
            }
        }
    }
    if (threadIdx.x == 0) sc.head[0] = (int)need;
    __syncthreads();
    // a shared page of which every holder has taken a copy is free now: count again where pages were copied
    long long left = free_pages;
    if (need > 0) {
        load_refs(c, refs);
        left = count_pages(c, refs, buf, before, is_free);
    }
    set_result(c, TPB_OK, left, need, need);
}

__global__ void __launch_bounds__(kThreads)
kv_fork_kernel(const tpb_kv_cache c, const int32_t *src, const int32_t *dst, int n, int share, uint32_t *status) {
    __shared__ long long buf[kWarps];
    __shared__ uint32_t bits[kMarkBits / 32];
    __shared__ int32_t small_offsets[kSmallList], small_list[kSmallList], small_src[kSmallList], small_dst[kSmallList], small_lens[kSmallList];
    const Scratch sc = scratch_of(c);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const Marks marks{bits, sc.marks, c.max_seqs <= kMarkBits};
    marks.clear_bits(c.max_seqs);
    tpb_grid_dep_launch();
    tpb_grid_dep_wait();
    const Listed srcs(src, n, small_src), dsts(dst, n, small_dst);
    Refs refs;
    load_refs(c, refs);
    int32_t *offsets = n <= kSmallList ? small_offsets : sc.offsets;
    // sources may repeat, destinations may not, and no sequence is both
    marks.clear_words(srcs, n, c.max_seqs);
    marks.clear_words(dsts, n, c.max_seqs);
    __syncthreads();
    bool ok = true;
    for (int i = threadIdx.x; i < n; i += kThreads) {
        const int from = srcs.mine(i), to = dsts.mine(i);
        if (from < 0 || from >= c.max_seqs || to < 0 || to >= c.max_seqs || marks.set(to)) ok = false;
    }
    long long before = 0;
    const long long free_pages = count_pages(c, refs, buf, before, is_free);
    ok = __syncthreads_and(ok);
    long long need = 0;
    if (ok) {
        const long long most = (long long)c.max_pages * c.page_tokens;
        for (int i0 = 0; i0 < n; i0 += kThreads) {
            const int i = i0 + threadIdx.x;
            int want = 0;
            if (i < n) {
                const int from = srcs.mine(i), len = __ldcg(c.lens + from), taken = __ldcg(c.lens + dsts.mine(i));
                if (i < kSmallList) small_lens[i] = len;
                if (marks.test(from) || len < 0 || len > most || taken != 0) ok = false;
                else want = share ? (len % c.page_tokens != 0) : pages_of(c, len);
            }
            long long total;
            const long long at = block_scan(want, buf, total);
            if (i < n) offsets[i] = (int)min(need + at, (long long)INT32_MAX);
            need += total;
        }
        ok = __syncthreads_and(ok);
    }
    if (!ok || need > free_pages) {
        if (threadIdx.x == 0) sc.head[0] = 0;
        set_result(c, ok ? TPB_ERR_OOM : TPB_ERR_INVALID_ARG, free_pages, 0, ok ? need : 0);
        return;
    }
    int32_t *list = need <= kSmallList ? small_list : sc.list_b;
    list_pages(c, refs, list, before, need, is_free);
    if (threadIdx.x == 0) sc.head[0] = (int)need;
    __syncthreads();
    for (int i = warp; i < n; i += kWarps) {
        const int from = srcs.at(i), to = dsts.at(i), len = i < kSmallList ? small_lens[i] : __ldcg(c.lens + from), at = offsets[i];
        const int kept = share ? len / c.page_tokens : 0;           // pages that both hold
        for (int p = kept + lane; p < pages_of(c, len); p += 32) {  // copies: until the source is known to be a page, of the copy itself
            const int fresh = list[at + p - kept];
            sc.list_a[at + p - kept] = fresh;
            sc.list_b[at + p - kept] = fresh;
            c.refs[fresh] = 1;
            c.table[(size_t)to * c.max_pages + p] = fresh;
        }
        __syncwarp();
        each_page(c, from, 0, pages_of(c, len), status, [&](int p, int page) {
            if (p < kept) {
                atomicAdd(c.refs + page, 1);
                c.table[(size_t)to * c.max_pages + p] = page;
            } else {
                sc.list_a[at + p - kept] = page;
            }
        });
        __syncwarp();
        if (lane == 0) {
            c.lens[to] = len;
            c.tail[to] = 0;
        }
    }
    set_result(c, TPB_OK, free_pages - need, need, need);
}

__global__ void __launch_bounds__(kThreads) kv_compact_kernel(const tpb_kv_cache c) {
    __shared__ long long buf[kWarps];
    tpb_grid_dep_launch();
    tpb_grid_dep_wait();
    const Scratch sc = scratch_of(c);
    Refs refs;
    load_refs(c, refs);
    long long before = 0, before_hole = 0;
    const int n_pages = (int)c.n_pages;
    const long long live = count_pages(c, refs, buf, before, [n_pages](int p, int r) { return r > 0 && p < n_pages; });
    const auto high = [live, n_pages](int p, int r) { return r > 0 && p >= live && p < n_pages; };
    const auto hole = [live](int p, int r) { return r <= 0 && p < live; };
    const long long moved = count_pages(c, refs, buf, before, high);
    count_pages(c, refs, buf, before_hole, hole);                 // as many: `live` places below `live`, and `live` pages
    list_pages(c, refs, sc.list_a, before, moved, high);
    list_pages(c, refs, sc.list_b, before_hole, moved, hole);
    __syncthreads();
    for (long long i = threadIdx.x; i < moved; i += kThreads) {
        const int from = sc.list_a[i], to = sc.list_b[i];
        c.refs[to] = __ldcg(c.refs + from);
        c.refs[from] = 0;
    }
    if (threadIdx.x == 0) {
        sc.head[0] = (int)moved;
        sc.head[1] = (int)live;
    }
    set_result(c, TPB_OK, c.n_pages - live, moved, moved);
}

// Copies page list_a[i] to page list_b[i], all layers, keys, values and scales, i < head[0].  No page is both a source and a destination: the
// destinations were free.  A warp moves pieces of 4 KB, eight 16-byte loads a lane in flight.
// COMPACT: the table's entries at or above the count of live pages follow their page as well.
constexpr int kPiece = 4096;
template <bool COMPACT>
__global__ void __launch_bounds__(256) kv_copy_pages_kernel(const tpb_kv_cache c) {
    tpb_grid_dep_launch();
    tpb_grid_dep_wait();
    __shared__ int s_head[2];
    const Scratch sc = scratch_of(c);
    if (threadIdx.x < 2) s_head[threadIdx.x] = __ldcg(sc.head + threadIdx.x);        // once a CTA: thousands of warps at one word wait in line
    __syncthreads();
    const int count = s_head[0];
    if (count <= 0) return;
    const int lane = threadIdx.x & 31;
    const long long page_bytes = (long long)c.kv_heads * c.page_tokens * c.head_dim;
    const int pieces = (int)((page_bytes + kPiece - 1) / kPiece);
    const long long items = (long long)count * c.layers * 2 * pieces;
    const long long warps = (long long)gridDim.x * (blockDim.x >> 5);
    for (long long it = (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); it < items; it += warps) {
        const int piece = (int)(it % pieces);
        const long long r = it / pieces;
        const int kv = (int)(r & 1);
        const long long r2 = r >> 1;
        const int i = (int)(r2 % count), layer = (int)(r2 / count);
        const int from = __ldcg(sc.list_a + i), to = __ldcg(sc.list_b + i);
        uint8_t *base = static_cast<uint8_t *>(kv ? c.v : c.k);
        const long long src = ((long long)layer * c.n_pages + from) * page_bytes + (long long)piece * kPiece;
        const long long dst = ((long long)layer * c.n_pages + to) * page_bytes + (long long)piece * kPiece;
        const int left = (int)min((long long)kPiece, page_bytes - (long long)piece * kPiece);
        uint4 v[8];
#pragma unroll
        for (int e = 0; e < 8; e++)
            if ((e * 32 + lane) * 16 < left) v[e] = __ldcg(reinterpret_cast<const uint4 *>(base + src) + e * 32 + lane);
#pragma unroll
        for (int e = 0; e < 8; e++)
            if ((e * 32 + lane) * 16 < left) reinterpret_cast<uint4 *>(base + dst)[e * 32 + lane] = v[e];
        if (piece == 0) {
            float *s = kv ? c.v_scale : c.k_scale;
            for (int hd = lane; hd < c.kv_heads; hd += 32)
                s[((long long)layer * c.n_pages + to) * c.kv_heads + hd] = __ldcg(s + ((long long)layer * c.n_pages + from) * c.kv_heads + hd);
        }
    }
    if (COMPACT) {
        const int live = s_head[1];
        const long long entries = (long long)c.max_seqs * c.max_pages, threads = (long long)gridDim.x * blockDim.x;
        for (long long e = (long long)blockIdx.x * blockDim.x + threadIdx.x; e < entries; e += threads) {
            const int page = __ldcg(c.table + e);
            if (page < live || page >= c.n_pages) continue;
            int lo = 0, hi = count;                                // list_a is ascending
            while (lo < hi) {
                const int mid = (lo + hi) >> 1;
                if (__ldcg(sc.list_a + mid) < page) lo = mid + 1;
                else hi = mid;
            }
            if (lo < count && __ldcg(sc.list_a + lo) == page) c.table[e] = __ldcg(sc.list_b + lo);
        }
    }
}

int copy_blocks(tpb_handle_t h) { return h->sm_count * 4; }

}  // namespace

int tpb_kv::check_cache(tpb_handle_t h, const tpb_kv_cache *c, const char *what) {
    TPB_CHECK_ARG(h, c != nullptr, "%s: null cache", what);
    TPB_CHECK_ARG(h, c->k && c->v && c->k_scale && c->v_scale && c->table && c->lens && c->tail && c->refs && c->result && c->scratch,
                  "%s: the cache has a null pointer", what);
    TPB_CHECK_ARG(h, tpb_aligned16(c->k) && tpb_aligned16(c->v) && tpb_aligned16(c->scratch), "%s: k, v and scratch must be 16-byte aligned", what);
    TPB_CHECK_ARG(h, ((reinterpret_cast<uintptr_t>(c->k_scale) | reinterpret_cast<uintptr_t>(c->v_scale) | reinterpret_cast<uintptr_t>(c->table) |
                       reinterpret_cast<uintptr_t>(c->lens) | reinterpret_cast<uintptr_t>(c->tail) | reinterpret_cast<uintptr_t>(c->refs) |
                       reinterpret_cast<uintptr_t>(c->result)) & 3u) == 0, "%s: the cache's arrays must be 4-byte aligned", what);
    TPB_CHECK_ARG(h, c->format == TPB_KV_S8 || c->format == TPB_KV_E4M3, "%s: unknown cache format %d", what, c->format);
    TPB_CHECK_ARG(h, c->head_dim == 64 || c->head_dim == 128, "%s: head_dim must be 64 or 128 (got %d)", what, c->head_dim);
    TPB_CHECK_ARG(h, c->page_tokens == 16 || c->page_tokens == 32 || c->page_tokens == 64, "%s: page_tokens must be 16, 32 or 64 (got %d)", what,
                  c->page_tokens);
    TPB_CHECK_ARG(h, c->n_pages > 0 && c->n_pages <= kMaxPagesInPool && c->layers > 0 && c->kv_heads > 0 && c->kv_heads <= 65535 && c->max_seqs > 0 &&
                         c->max_pages > 0,
                  "%s: the cache's sizes must be positive, n_pages at most 2^24 and kv_heads below 65536", what);
    // token rows of the whole cache, and its table's entries, are counted in 32 bits
    TPB_CHECK_ARG(h, (__int128)c->layers * c->n_pages * c->kv_heads * c->page_tokens < ((int64_t)1 << 31) &&
                         (int64_t)c->max_pages * c->page_tokens <= ((int64_t)1 << 30) && (int64_t)c->max_seqs * c->max_pages < ((int64_t)1 << 31),
                  "%s: the cache exceeds 2^31 rows or table entries, or a sequence 2^30 tokens", what);
    return TPB_OK;
}

int tpb_kv::check_layer(tpb_handle_t h, const tpb_kv_cache *c, int layer, const char *what) {
    const int rc = check_cache(h, c, what);
    if (rc != TPB_OK) return rc;
    TPB_CHECK_ARG(h, layer >= 0 && layer < c->layers, "%s: layer %d of %d", what, layer, c->layers);
    return TPB_OK;
}

namespace {

int check_ids(tpb_handle_t h, const tpb_kv_cache *c, const char *what, const void *a, const void *b, bool need_b, int n) {
    const int rc = check_cache(h, c, what);
    if (rc != TPB_OK) return rc;
    TPB_CHECK_ARG(h, n >= 0, "%s: negative count", what);
    TPB_CHECK_ARG(h, n == 0 || (a && (b || !need_b)), "%s: null pointer", what);
    TPB_CHECK_ARG(h, ((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b)) & 3u) == 0, "%s: lists must be 4-byte aligned", what);
    return TPB_OK;
}

}  // namespace

extern "C" {

size_t tpb_kv_scratch_bytes(int64_t n_pages, int max_seqs) {
    if (n_pages <= 0 || n_pages > kMaxPagesInPool || max_seqs <= 0) return 0;
    return (size_t)4 * (8 + 2 * (size_t)max_seqs + 2 * (size_t)n_pages);
}

int tpb_kv_extend(tpb_handle_t h, tpb_stream_t stream, const tpb_kv_cache *c, const int32_t *seqs, const int32_t *n_new, int n) {
    if (!h) return TPB_ERR_INVALID_ARG;
    const int rc = check_ids(h, c, "kv_extend", seqs, n_new, true, n);
    if (rc != TPB_OK) return rc;
    tpb_device_guard guard(h->device);
    TPB_CUDA(h, guard.err);
    TPB_CUDA(h, tpb_launch_pdl(kv_extend_kernel, dim3(1), dim3(kThreads), 0, (cudaStream_t)stream, *c, seqs, n_new, n));
    return TPB_OK;
}

int tpb_kv_truncate(tpb_handle_t h, tpb_stream_t stream, const tpb_kv_cache *c, const int32_t *seqs, const int32_t *new_lens, int n) {
    if (!h) return TPB_ERR_INVALID_ARG;
    const int rc = check_ids(h, c, "kv_truncate", seqs, new_lens, false, n);
    if (rc != TPB_OK) return rc;
    tpb_device_guard guard(h->device);
    TPB_CUDA(h, guard.err);
    TPB_CUDA(h, tpb_launch_pdl(kv_truncate_kernel, dim3(1), dim3(kThreads), 0, (cudaStream_t)stream, *c, seqs, new_lens, n, h->d_status));
    // sequences that are freed are not cut inside a page: nothing to copy
    if (new_lens)
        TPB_CUDA(h, tpb_launch_pdl(kv_copy_pages_kernel<false>, dim3(copy_blocks(h)), dim3(256), 0, (cudaStream_t)stream, *c));
    return TPB_OK;
}

int tpb_kv_fork(tpb_handle_t h, tpb_stream_t stream, const tpb_kv_cache *c, const int32_t *src, const int32_t *dst, int n, int share) {
    if (!h) return TPB_ERR_INVALID_ARG;
    const int rc = check_ids(h, c, "kv_fork", src, dst, true, n);
    if (rc != TPB_OK) return rc;
    tpb_device_guard guard(h->device);
    TPB_CUDA(h, guard.err);
    TPB_CUDA(h, tpb_launch_pdl(kv_fork_kernel, dim3(1), dim3(kThreads), 0, (cudaStream_t)stream, *c, src, dst, n, share, h->d_status));
    TPB_CUDA(h, tpb_launch_pdl(kv_copy_pages_kernel<false>, dim3(copy_blocks(h)), dim3(256), 0, (cudaStream_t)stream, *c));
    return TPB_OK;
}

int tpb_kv_compact(tpb_handle_t h, tpb_stream_t stream, const tpb_kv_cache *c) {
    if (!h) return TPB_ERR_INVALID_ARG;
    const int rc = check_cache(h, c, "kv_compact");
    if (rc != TPB_OK) return rc;
    tpb_device_guard guard(h->device);
    TPB_CUDA(h, guard.err);
    TPB_CUDA(h, tpb_launch_pdl(kv_compact_kernel, dim3(1), dim3(kThreads), 0, (cudaStream_t)stream, *c));
    TPB_CUDA(h, tpb_launch_pdl(kv_copy_pages_kernel<true>, dim3(copy_blocks(h)), dim3(256), 0, (cudaStream_t)stream, *c));
    return TPB_OK;
}

}  // extern "C"
