// Attention of absorbed MLA queries over the 8-bit latent cache (see include/dsv3_b200.h).
#include "latent_cache.cuh"

namespace dsv3 {
namespace {

struct Queries {
    const __nv_bfloat16 *latent, *rope;
    int64_t latent_token, latent_head, rope_token, rope_head;   // strides in elements
    int64_t tokens;
    int heads;
    const int32_t *seq_lens, *cu;       // cu: null for tokens / n_seqs queries a sequence
    const int64_t* tree;
    float scale;
    __nv_bfloat16* out;
    float* lse;
};

// A warp to a query head, a token at a time with a running maximum and sum.
__global__ void __launch_bounds__(128) latent_attention_simple_kernel(LatentCache c, Queries q) {
    griddep_launch_dependents();
    griddep_wait();
    const int lane = threadIdx.x & 31;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);
    if (row >= q.tokens * q.heads) return;
    const int64_t t = row / q.heads;
    const int h = static_cast<int>(row - t * q.heads);
    int seq = 0;
    int64_t begin, end;
    if (q.cu) {
        while (seq < c.n_seqs && q.cu[seq + 1] <= t) ++seq;
        if (seq == c.n_seqs) return;
        begin = q.cu[seq], end = q.cu[seq + 1];
    } else {
        const int64_t per = q.tokens / c.n_seqs;
        seq = static_cast<int>(t / per);
        begin = seq * per, end = begin + per;
    }
    const int64_t cap = static_cast<int64_t>(c.pages_width) << c.page_shift;
    const int64_t len = max(static_cast<int64_t>(0), min(static_cast<int64_t>(q.seq_lens[seq]), cap));
    const int64_t base = len - (end - begin);           // position of the sequence's first query
    float ql[16], qr[2], acc[16], m = -INFINITY, l = 0.0f;
    for (int i = 0; i < 16; ++i) ql[i] = __bfloat162float(q.latent[t * q.latent_token + h * q.latent_head + lane * 16 + i]), acc[i] = 0.0f;
    for (int i = 0; i < 2; ++i) qr[i] = __bfloat162float(q.rope[t * q.rope_token + h * q.rope_head + lane * 2 + i]);
    const int64_t last = q.tree ? len : min(len, base + (t - begin) + 1);
    for (int64_t p = 0; p < last; ++p) {
        if (q.tree && p >= base && (p - base >= 64 || !((q.tree[t] >> (p - base)) & 1))) continue;
        const int64_t slot = slot_of(c, seq, static_cast<uint32_t>(p));
        if (slot < 0) continue;
        float v[16], d = 0.0f;
        const uint4 w = *reinterpret_cast<const uint4*>(c.latent + slot * kLatent + lane * 16);
        const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
        for (int i = 0; i < 8; ++i) {
            const float2 f = e4m3x2_to_float2(static_cast<uint16_t>(ww[i / 2] >> (16 * (i & 1))));
            v[2 * i] = f.x, v[2 * i + 1] = f.y;
        }
        for (int i = 0; i < 16; ++i) d = fmaf(ql[i], v[i], d);
        for (int i = 0; i < 2; ++i) d = fmaf(qr[i], __bfloat162float(c.rope[slot * kRope + lane * 2 + i]), d);
        for (int o = 16; o > 0; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
        const float s = c.scale[slot], x = d * s * q.scale;
        const float mn = fmaxf(m, x), old = exp2f((m - (mn == -INFINITY ? 0.0f : mn)) * 1.44269504f), pr = exp2f((x - mn) * 1.44269504f);
        l = l * old + pr;
        for (int i = 0; i < 16; ++i) acc[i] = acc[i] * old + pr * s * v[i];
        m = mn;
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    for (int i = 0; i < 16; ++i) q.out[row * kLatent + lane * 16 + i] = __float2bfloat16_rn(acc[i] * inv);
    if (q.lse && lane == 0) q.lse[row] = l == 0.0f ? -INFINITY : m + logf(l);
}

}  // namespace
}  // namespace dsv3

using namespace dsv3;

extern "C" {

size_t dsv3_latent_attention_workspace_bytes(int64_t tokens, int heads, int n_seqs, int64_t longest) { return 0; }

int dsv3_latent_attention(const dsv3_latent_cache_t* cache, const void* q_latent, int64_t q_latent_token_stride, int64_t q_latent_head_stride,
                          const void* q_rope, int64_t q_rope_token_stride, int64_t q_rope_head_stride, int64_t tokens, int heads,
                          const int32_t* seq_lens, const int32_t* cu_seqlens_q, const int64_t* tree_mask, float softmax_scale, void* out,
                          float* lse, void* workspace, size_t workspace_bytes, dsv3_stream_t stream) {
    LatentCache c;
    if (const int rc = latent_cache_arg("latent_attention", cache, true, &c); rc != DSV3_OK) return rc;
    if (tokens < 0 || heads < 0) {
        set_last_error("latent_attention: negative size");
        return DSV3_ERR_INVALID_ARGUMENT;
    }
    if (tokens == 0 || heads == 0) return DSV3_OK;
    if (!q_latent || !q_rope || !seq_lens || !out) {
        set_last_error("latent_attention: null pointer");
        return DSV3_ERR_INVALID_ARGUMENT;
    }
    if (c.n_seqs == 0 || (!cu_seqlens_q && tokens % c.n_seqs != 0)) {
        set_last_error("latent_attention: %lld queries do not divide among %d sequences", static_cast<long long>(tokens), c.n_seqs);
        return DSV3_ERR_INVALID_ARGUMENT;
    }
    const int64_t strides = q_latent_token_stride | q_latent_head_stride | q_rope_token_stride | q_rope_head_stride;
    if (strides % 8 != 0 || (reinterpret_cast<uintptr_t>(q_latent) | reinterpret_cast<uintptr_t>(q_rope) | reinterpret_cast<uintptr_t>(out)) % 16 != 0) {
        set_last_error("latent_attention: rows of the queries and out must be 16-byte aligned");
        return DSV3_ERR_UNSUPPORTED;
    }
    if (heads > 1024 || tokens > 0x7FFFFFFFll / heads) {
        set_last_error("latent_attention: takes at most 1024 heads and 2^31 query heads");
        return DSV3_ERR_UNSUPPORTED;
    }
    Queries q = {static_cast<const __nv_bfloat16*>(q_latent), static_cast<const __nv_bfloat16*>(q_rope), q_latent_token_stride, q_latent_head_stride,
                 q_rope_token_stride, q_rope_head_stride, tokens, heads, seq_lens, cu_seqlens_q, tree_mask, softmax_scale,
                 static_cast<__nv_bfloat16*>(out), lse};
    const int64_t rows = tokens * heads;
    DSV3_CUDA_TRY(launch_dependent(latent_attention_simple_kernel, dim3(static_cast<unsigned>((rows + 3) / 4)), dim3(128), 0,
                                   static_cast<cudaStream_t>(stream), c, q));
    return DSV3_OK;
}

}  // extern "C"
