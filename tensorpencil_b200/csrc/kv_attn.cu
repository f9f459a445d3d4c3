// Attention of a sequence's last tokens over its 8-bit cache.
#include "kv_common.cuh"

using namespace tpb_kv;

namespace {

// A warp per (row, head): one pass over the visible tokens with the running maximum and sum, each lane HD / 32 dimensions.
template <typename T, int FORMAT, int HD>
__global__ void __launch_bounds__(256)
kv_attention_kernel(const tpb_kv_cache c, int layer, T *out, int64_t ld_out, const T *q, int64_t ld_q, const int32_t *seqs, const int32_t *cu,
                    int n_seqs, int rows, int heads, float scale, uint32_t *status) {
    tpb_grid_dep_launch();
    tpb_grid_dep_wait();
    constexpr int PER = HD / 32;
    const int lane = threadIdx.x & 31;
    const long long w = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int r = (int)(w / heads), head = (int)(w % heads);
    if (r >= rows) return;
    const int i = find_last(n_seqs, r, [&](int j) { return row_offset(cu, j, rows); });
    const int r0 = row_offset(cu, i, rows), r1 = row_offset(cu, i + 1, rows);
    if (r < r0 || r >= r1) return;
    const int seq = __ldcg(seqs + i);
    if (seq < 0 || seq >= c.max_seqs) {
        report(status, kBadSeq);
        return;
    }
    const int len = __ldcg(c.lens + seq);
    if (len < 0 || (long long)len > (long long)c.max_pages * c.page_tokens) {
        report(status, kBadLen);
        return;
    }
    const int last = len - (r1 - r);
    const int hk = head / (heads / c.kv_heads);
    float qv[PER], o[PER] = {}, m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int e = 0; e < PER; e++) qv[e] = (float)q[(int64_t)r * ld_q + (int64_t)head * HD + lane * PER + e] * scale;
    for (int j = 0; j <= last; j++) {
        const int page = __ldcg(c.table + (size_t)seq * c.max_pages + j / c.page_tokens);
        if (page < 0 || page >= c.n_pages) {
            report(status, kBadPage);
            continue;
        }
        const size_t block = ((size_t)layer * c.n_pages + page) * c.kv_heads + hk;
        const size_t at = (block * c.page_tokens + j % c.page_tokens) * HD + lane * PER;
        float f[4] = {}, s = 0.0f;
        uint32_t word = 0;
        for (int e = 0; e < PER; e++) word |= (uint32_t)__ldcg((const uint8_t *)c.k + at + e) << (8 * e);
        unpack4<FORMAT>(word, f);
        for (int e = 0; e < PER; e++) s += qv[e] * f[e];
        for (int of = 16; of > 0; of >>= 1) s += __shfl_xor_sync(0xffffffffu, s, of);
        s *= __ldcg(c.k_scale + block);
        const float mn = fmaxf(m, s), a = m == mn ? 1.0f : __expf(m - mn), p = __expf(s - mn);
        word = 0;
        for (int e = 0; e < PER; e++) word |= (uint32_t)__ldcg((const uint8_t *)c.v + at + e) << (8 * e);
        unpack4<FORMAT>(word, f);
        const float vs = __ldcg(c.v_scale + block);
        l = l * a + p;
        for (int e = 0; e < PER; e++) o[e] = o[e] * a + p * vs * f[e];
        m = mn;
    }
#pragma unroll
    for (int e = 0; e < PER; e++) out[(int64_t)r * ld_out + (int64_t)head * HD + lane * PER + e] = (T)(l == 0.0f ? 0.0f : o[e] / l);
}

}  // namespace

extern "C" {

size_t tpb_kv_attention_workspace_bytes(tpb_handle_t h, int head_dim) {
    if (!h || (head_dim != 64 && head_dim != 128)) return 0;
    return (size_t)h->sm_count * 16;
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
    const auto run = [&](auto *tag) {
        using T = std::remove_pointer_t<decltype(tag)>;
        const auto launch = [&](auto kern) {
            return tpb_launch_pdl(kern, dim3((unsigned)((rows * heads + 7) / 8)), dim3(256), 0, (cudaStream_t)stream, *c, layer, (T *)out, ld_out,
                                  (const T *)q, ld_q, seqs, cu, n_seqs, (int)rows, heads, scale, h->d_status);
        };
        if (c->format == TPB_KV_S8) return c->head_dim == 64 ? launch(kv_attention_kernel<T, TPB_KV_S8, 64>) : launch(kv_attention_kernel<T, TPB_KV_S8, 128>);
        return c->head_dim == 64 ? launch(kv_attention_kernel<T, TPB_KV_E4M3, 64>) : launch(kv_attention_kernel<T, TPB_KV_E4M3, 128>);
    };
    TPB_CUDA(h, dtype == TPB_F32 ? run((float *)nullptr) : dtype == TPB_BF16 ? run((__nv_bfloat16 *)nullptr) : run((__half *)nullptr));
    return TPB_OK;
}

}  // extern "C"
