// Causal attention over packed prompts.
#include "kv_common.cuh"

namespace {

using tpb_kv::find_last;
using tpb_kv::row_offset;

// A warp per (token, head): one pass over the visible tokens with the running maximum and sum, each lane HD / 32 dimensions.
template <typename T, int HD>
__global__ void __launch_bounds__(256)
attn_packed_kernel(T *out, int64_t ld_out, const T *q, int64_t ld_q, const T *k, int64_t ld_k, const T *v, int64_t ld_v, const int32_t *cu,
                   int n_seqs, int tokens, int heads, int kv_heads, float scale) {
    tpb_grid_dep_launch();
    tpb_grid_dep_wait();
    constexpr int PER = HD / 32;
    const int lane = threadIdx.x & 31;
    const long long w = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int r = (int)(w / heads), head = (int)(w % heads);
    if (r >= tokens) return;
    const int i = find_last(n_seqs, r, [&](int j) { return row_offset(cu, j, tokens); });
    const int r0 = row_offset(cu, i, tokens);
    if (r < r0 || r >= row_offset(cu, i + 1, tokens)) return;
    const int hk = head / (heads / kv_heads);
    float qv[PER], o[PER] = {}, m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int e = 0; e < PER; e++) qv[e] = (float)q[(int64_t)r * ld_q + (int64_t)head * HD + lane * PER + e] * scale;
    for (int j = r0; j <= r; j++) {
        float s = 0.0f;
#pragma unroll
        for (int e = 0; e < PER; e++) s += qv[e] * (float)k[(int64_t)j * ld_k + (int64_t)hk * HD + lane * PER + e];
#pragma unroll
        for (int of = 16; of > 0; of >>= 1) s += __shfl_xor_sync(0xffffffffu, s, of);
        const float mn = fmaxf(m, s), a = m == mn ? 1.0f : __expf(m - mn), p = __expf(s - mn);
        l = l * a + p;
#pragma unroll
        for (int e = 0; e < PER; e++) o[e] = o[e] * a + p * (float)v[(int64_t)j * ld_v + (int64_t)hk * HD + lane * PER + e];
        m = mn;
    }
#pragma unroll
    for (int e = 0; e < PER; e++) out[(int64_t)r * ld_out + (int64_t)head * HD + lane * PER + e] = (T)(o[e] / l);
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
    tpb_device_guard guard(h->device);
    TPB_CUDA(h, guard.err);
    const auto run = [&](auto *tag) {
        using T = std::remove_pointer_t<decltype(tag)>;
        const auto launch = [&](auto kern) {
            return tpb_launch_pdl(kern, dim3((unsigned)((tokens * heads + 7) / 8)), dim3(256), 0, (cudaStream_t)stream, (T *)out, ld_out, (const T *)q,
                                  ld_q, (const T *)k, ld_k, (const T *)v, ld_v, cu, n_seqs, (int)tokens, heads, kv_heads, scale);
        };
        return head_dim == 64 ? launch(attn_packed_kernel<T, 64>) : launch(attn_packed_kernel<T, 128>);
    };
    TPB_CUDA(h, dtype == TPB_BF16 ? run((__nv_bfloat16 *)nullptr) : run((__half *)nullptr));
    return TPB_OK;
}

}  // extern "C"
