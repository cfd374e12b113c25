// The 8-bit latent cache (see include/dsv3_b200.h for its format): write, read back, close ranks after a verification.
//
// All three move a few hundred bytes a token and compute next to nothing: HBM bounds them from some thousand tokens on, a launch and two
// dependent loads (page or slot, then the token) below that.
#include <algorithm>

#include "latent_cache.cuh"

namespace dsv3 {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kWriteBlocks = 3;           // to an SM: as many as its registers hold

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

__device__ __forceinline__ void unpack8(const uint4& v, float* x) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) x[2 * i] = bf16_bits_to_float(w[i] & 0xFFFFu), x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
}
__device__ __forceinline__ void load8(const __nv_bfloat16* p, float* x) { unpack8(*reinterpret_cast<const uint4*>(p), x); }
__device__ __forceinline__ void load8(const float* p, float* x) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
}

// A warp to a token, 8 latent values of either half and one pair to rotate per lane, so that a warp's loads and stores are whole lines.
//   c = kv * rsqrt(mean(kv^2) + eps) * weight, s = power_scale(max(amax|c|, 1e-4)), stored: e4m3(c / s), bf16(rot(k) / s), s
// Everything in fp32 and rounded once; dividing by a power of two is exact.  The norm's weight stays in registers over a warp's tokens.
// B200, fp32 weight, launches behind one another: 16001 tokens 9.2 us where all comes from HBM (3.6 TB/s), 7.0 where the L2 holds it; 4096 from the L2 3.3, one 1.7.  A token to a warp
// and its weights loaded one by one, 16 neighbours to a lane, took 2.2 times as long at 16001.
template <typename W>
__global__ void __launch_bounds__(kThreads, kWriteBlocks) latent_write_kernel(LatentCache c, const __nv_bfloat16* __restrict__ kv, int64_t kv_stride,
                                                                const W* __restrict__ weight, float eps, const float2* __restrict__ freqs,
                                                                int64_t n_positions, const int64_t* __restrict__ positions,
                                                                const int64_t* __restrict__ slots, int64_t tokens) {
    const int lane = threadIdx.x & 31;
    griddep_launch_dependents();
    griddep_wait();
    float w[16];
    load8(weight + lane * 8, w);
    load8(weight + kLatent / 2 + lane * 8, w + 8);
    const int64_t step = static_cast<int64_t>(gridDim.x) * kWarps;
    // (a token's values, and where it goes, are on their way while the one before is worked on)
    int64_t t = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5), slot = -1, position = -1;
    uint4 v0, v1;
    uint32_t pair;
    float2 f;
    const auto fetch = [&](int64_t at) {
        const __nv_bfloat16* const row = kv + at * kv_stride;
        slot = slots[at], position = positions[at];
        v0 = *reinterpret_cast<const uint4*>(row + lane * 8), v1 = *reinterpret_cast<const uint4*>(row + kLatent / 2 + lane * 8);
        pair = reinterpret_cast<const uint32_t*>(row + kLatent)[lane];
    };
    const auto angles = [&]() { return position >= 0 && position < n_positions ? freqs[position * (kRope / 2) + lane] : make_float2(0.0f, 0.0f); };
    if (t < tokens) {
        fetch(t);
        f = angles();
    }
    for (; t < tokens; t += step) {
        const int64_t here = slot;
        const bool placed = position >= 0 && position < n_positions;
        float x[16];
        unpack8(v0, x);
        unpack8(v1, x + 8);
        const float a = bf16_bits_to_float(pair & 0xFFFFu), b = __uint_as_float(pair & 0xFFFF0000u);
        const float turn_re = a * f.x - b * f.y, turn_im = a * f.y + b * f.x;
        const bool more = t + step < tokens;
        if (more) fetch(t + step);
        float sq = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i) sq = fmaf(x[i], x[i], sq);
        const float r = rsqrtf(warp_sum(sq) * (1.0f / kLatent) + eps);
        float top = 0.0f;
        bool finite = placed;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            x[i] = x[i] * r * w[i];
            finite = finite && fabsf(x[i]) < INFINITY;
            top = fmaxf(top, fabsf(x[i]));
        }
        const float s = power_scale(fmaxf(warp_max(top), 1e-4f));
        const float inv = power_reciprocal(s);
        uint32_t turned = pack_bf16x2(turn_re * inv, turn_im * inv);
        // (what bf16 rounds to infinity is not finite either)
        finite = finite && (turned & 0x7F80u) != 0x7F80u && (turned & 0x7F800000u) != 0x7F800000u;
        finite = __all_sync(0xffffffffu, finite);
        uint32_t q[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            q[i] = finite ? cvt_e4m3x2(x[4 * i] * inv, x[4 * i + 1] * inv) |
                                static_cast<uint32_t>(cvt_e4m3x2(x[4 * i + 2] * inv, x[4 * i + 3] * inv)) << 16
                          : 0u;
        if (!finite) turned = 0u;
        if (more) f = angles();
        if (here < 0 || here >= static_cast<int64_t>(c.n_pages) << c.page_shift) continue;
        uint8_t* const to = c.latent + here * kLatent + lane * 8;
        *reinterpret_cast<uint2*>(to) = make_uint2(q[0], q[1]);
        *reinterpret_cast<uint2*>(to + kLatent / 2) = make_uint2(q[2], q[3]);
        *reinterpret_cast<uint32_t*>(c.rope + here * kRope + lane * 2) = turned;
        if (lane == 0) c.scale[here] = finite ? s : __uint_as_float(0x7FC00000u);
    }
}

// Four values of e4m3 times s, as bf16.
__device__ __forceinline__ uint2 scaled4(uint32_t w, float s) {
    const float2 a = e4m3x2_to_float2(static_cast<uint16_t>(w)), b = e4m3x2_to_float2(static_cast<uint16_t>(w >> 16));
    return make_uint2(pack_bf16x2(a.x * s, a.y * s), pack_bf16x2(b.x * s, b.y * s));
}

// A warp to kReadRows rows of the result, all under way together; loads and stores are whole lines (with 16 neighbouring values to a lane, whose stores are not,
// 11 % longer; 148 thousand tokens 44.4 us: HBM bounds it, at 6.1 TB/s).  The block's first row is looked up among the sequences by all threads, the others from there on.
constexpr int kReadRows = 4;
__global__ void __launch_bounds__(kThreads) latent_read_kernel(LatentCache c, const int32_t* __restrict__ cu, int64_t total,
                                                               __nv_bfloat16* __restrict__ latent, __nv_bfloat16* __restrict__ rope) {
    const int lane = threadIdx.x & 31;
    const int64_t row0 = static_cast<int64_t>(blockIdx.x) * (kWarps * kReadRows);
    griddep_launch_dependents();
    griddep_wait();
    int seq = 0;                                      // how many sequences end at or before row0
    for (int i = threadIdx.x; i - static_cast<int>(threadIdx.x) < c.n_seqs; i += kThreads)
        seq += __syncthreads_count(i < c.n_seqs && cu[i + 1] <= row0);
    uint2 q[kReadRows][2];
    uint32_t k[kReadRows];
    float s[kReadRows];
    bool there[kReadRows];
#pragma unroll
    for (int i = 0; i < kReadRows; ++i) {
        const int64_t row = row0 + (threadIdx.x >> 5) + i * kWarps;
        while (seq < c.n_seqs && cu[seq + 1] <= row) ++seq;
        there[i] = row < total && seq < c.n_seqs;
        const int64_t slot = there[i] ? slot_of(c, seq, static_cast<uint32_t>(row - cu[seq])) : -1;
        q[i][0] = q[i][1] = make_uint2(0u, 0u);
        k[i] = 0u;
        s[i] = 0.0f;
        if (slot >= 0) {
            q[i][0] = *reinterpret_cast<const uint2*>(c.latent + slot * kLatent + lane * 8);
            q[i][1] = *reinterpret_cast<const uint2*>(c.latent + slot * kLatent + kLatent / 2 + lane * 8);
            k[i] = *reinterpret_cast<const uint32_t*>(c.rope + slot * kRope + lane * 2);
            s[i] = c.scale[slot];
        }
    }
#pragma unroll
    for (int i = 0; i < kReadRows; ++i) {
        if (!there[i]) continue;
        const int64_t row = row0 + (threadIdx.x >> 5) + i * kWarps;
        uint4* const to = reinterpret_cast<uint4*>(latent + row * kLatent) + lane;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint2 a = scaled4(q[i][h].x, s[i]), b = scaled4(q[i][h].y, s[i]);
            to[h * (kLatent / 16)] = make_uint4(a.x, a.y, b.x, b.y);
        }
        *reinterpret_cast<uint32_t*>(rope + row * kRope + lane * 2) =
            pack_bf16x2(bf16_bits_to_float(k[i] & 0xFFFFu) * s[i], __uint_as_float(k[i] & 0xFFFF0000u) * s[i]);
    }
}

// A block to a sequence, a warp to kKeepRows of the drafts of a round.  path ascends strictly, so path[j] >= j: a round's destinations lie before the
// sources of all later rounds, and within a round everything is read before anything is written.
constexpr int kKeepRows = 4;
__global__ void __launch_bounds__(kThreads) latent_keep_kernel(LatentCache c, const int32_t* __restrict__ first, const int32_t* __restrict__ path,
                                                               int64_t path_stride, int drafts, const int32_t* __restrict__ count) {
    const int lane = threadIdx.x & 31, seq = blockIdx.x;
    griddep_launch_dependents();
    griddep_wait();
    const int n = min(count[seq], drafts), base = first[seq];
    for (int j0 = 0; j0 < n; j0 += kWarps * kKeepRows) {
        uint4 q[kKeepRows];
        uint32_t k[kKeepRows];
        float s[kKeepRows];
        int64_t to[kKeepRows];
#pragma unroll
        for (int i = 0; i < kKeepRows; ++i) {
            const int j = j0 + (threadIdx.x >> 5) + i * kWarps;
            to[i] = -1;
            if (j >= n) continue;
            const int from = path[seq * path_stride + j];
            if (from == j || from < 0 || base < 0) continue;
            const int64_t src = slot_of(c, seq, static_cast<uint32_t>(base) + from);
            to[i] = slot_of(c, seq, static_cast<uint32_t>(base) + j);
            if (src < 0) to[i] = -1;
            if (to[i] < 0) continue;
            q[i] = *reinterpret_cast<const uint4*>(c.latent + src * kLatent + lane * 16);
            k[i] = *reinterpret_cast<const uint32_t*>(c.rope + src * kRope + lane * 2);
            s[i] = c.scale[src];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kKeepRows; ++i) {
            if (to[i] < 0) continue;
            *reinterpret_cast<uint4*>(c.latent + to[i] * kLatent + lane * 16) = q[i];
            *reinterpret_cast<uint32_t*>(c.rope + to[i] * kRope + lane * 2) = k[i];
            if (lane == 0) c.scale[to[i]] = s[i];
        }
    }
}

}  // namespace

int latent_cache_arg(const char* who, const dsv3_latent_cache_t* c, bool with_pages, LatentCache* out) {
    if (!c || c->n_pages < 0 || c->page_size <= 0 || (with_pages && (c->n_seqs < 0 || c->pages_width < 0 || c->pages_stride < 0))) {
        set_last_error("%s: no cache, or a negative size", who);
        return DSV3_ERR_INVALID_ARGUMENT;
    }
    if (c->page_size < 16 || (c->page_size & (c->page_size - 1)) != 0) {
        set_last_error("%s: page_size %d must be a power of two from 16 on", who, c->page_size);
        return DSV3_ERR_UNSUPPORTED;
    }
    if (c->n_pages > 0x7FFFFFFFll / c->page_size || (with_pages && c->pages_width > 0x7FFFFFFFll / c->page_size)) {
        set_last_error("%s: 2^31 cached tokens or more", who);
        return DSV3_ERR_UNSUPPORTED;
    }
    if ((c->n_pages > 0 && (!c->latent || !c->rope || !c->scale)) || (with_pages && c->n_seqs > 0 && c->pages_width > 0 && !c->pages)) {
        set_last_error("%s: null pointer", who);
        return DSV3_ERR_INVALID_ARGUMENT;
    }
    if (reinterpret_cast<uintptr_t>(c->latent) % 16 != 0 || reinterpret_cast<uintptr_t>(c->rope) % 16 != 0) {
        set_last_error("%s: latent and rope must be 16-byte aligned", who);
        return DSV3_ERR_UNSUPPORTED;
    }
    uint32_t shift = 0;
    while ((1 << shift) < c->page_size) ++shift;
    *out = {static_cast<uint8_t*>(c->latent), static_cast<__nv_bfloat16*>(c->rope), c->scale, with_pages ? c->pages : nullptr,
            with_pages ? c->pages_stride : 0, static_cast<uint32_t>(c->n_pages), shift, with_pages ? static_cast<uint32_t>(c->pages_width) : 0u,
            with_pages ? c->n_seqs : 0};
    return DSV3_OK;
}

}  // namespace dsv3

using namespace dsv3;

extern "C" {

int dsv3_latent_write(const dsv3_latent_cache_t* cache, const void* kv, int64_t kv_stride, const void* weight, int weight_fp32, float eps,
                      const float* freqs, int64_t n_positions, const int64_t* positions, const int64_t* slots, int64_t tokens,
                      dsv3_stream_t stream) {
    LatentCache c;
    if (const int rc = latent_cache_arg("latent_write", cache, false, &c); rc != DSV3_OK) return rc;
    if (tokens < 0 || n_positions < 0) {
        set_last_error("latent_write: negative size");
        return DSV3_ERR_INVALID_ARGUMENT;
    }
    if (tokens == 0) return DSV3_OK;
    if (!kv || !weight || !positions || !slots || (n_positions > 0 && !freqs)) {
        set_last_error("latent_write: null pointer");
        return DSV3_ERR_INVALID_ARGUMENT;
    }
    if (reinterpret_cast<uintptr_t>(kv) % 16 != 0 || kv_stride % 8 != 0 || reinterpret_cast<uintptr_t>(freqs) % 8 != 0 || reinterpret_cast<uintptr_t>(weight) % 16 != 0) {
        set_last_error("latent_write: rows of kv and the weight must be 16-byte aligned, freqs 8-byte");
        return DSV3_ERR_UNSUPPORTED;
    }
    const int64_t grid = std::min<int64_t>((tokens + kWarps - 1) / kWarps, static_cast<int64_t>(num_sms()) * kWriteBlocks);
    const auto go = [&](auto kern, auto w) {
        return launch_dependent(kern, dim3(static_cast<unsigned>(grid)), dim3(kThreads), 0, static_cast<cudaStream_t>(stream), c,
                                static_cast<const __nv_bfloat16*>(kv), kv_stride, w, eps, reinterpret_cast<const float2*>(freqs), n_positions,
                                positions, slots, tokens);
    };
    DSV3_CUDA_TRY(weight_fp32 ? go(latent_write_kernel<float>, static_cast<const float*>(weight))
                              : go(latent_write_kernel<__nv_bfloat16>, static_cast<const __nv_bfloat16*>(weight)));
    return DSV3_OK;
}

int dsv3_latent_read(const dsv3_latent_cache_t* cache, const int32_t* cu_seqlens, int64_t total, void* latent, void* rope,
                     dsv3_stream_t stream) {
    LatentCache c;
    if (const int rc = latent_cache_arg("latent_read", cache, true, &c); rc != DSV3_OK) return rc;
    if (total < 0) {
        set_last_error("latent_read: negative size");
        return DSV3_ERR_INVALID_ARGUMENT;
    }
    if (total == 0 || c.n_seqs == 0) return DSV3_OK;
    if (!cu_seqlens || !latent || !rope) {
        set_last_error("latent_read: null pointer");
        return DSV3_ERR_INVALID_ARGUMENT;
    }
    if (reinterpret_cast<uintptr_t>(latent) % 16 != 0 || reinterpret_cast<uintptr_t>(rope) % 4 != 0) {
        set_last_error("latent_read: latent must be 16-byte and rope 4-byte aligned");
        return DSV3_ERR_UNSUPPORTED;
    }
    if (total > 0x7FFFFFFFll) {
        set_last_error("latent_read: 2^31 rows or more");
        return DSV3_ERR_UNSUPPORTED;
    }
    const int64_t per = kWarps * kReadRows;
    DSV3_CUDA_TRY(launch_dependent(latent_read_kernel, dim3(static_cast<unsigned>((total + per - 1) / per)), dim3(kThreads), 0,
                                   static_cast<cudaStream_t>(stream), c, cu_seqlens, total, static_cast<__nv_bfloat16*>(latent),
                                   static_cast<__nv_bfloat16*>(rope)));
    return DSV3_OK;
}

int dsv3_latent_keep(const dsv3_latent_cache_t* cache, const int32_t* first, const int32_t* path, int64_t path_stride, int drafts,
                     const int32_t* count, dsv3_stream_t stream) {
    LatentCache c;
    if (const int rc = latent_cache_arg("latent_keep", cache, true, &c); rc != DSV3_OK) return rc;
    if (drafts < 0 || path_stride < 0) {
        set_last_error("latent_keep: negative size");
        return DSV3_ERR_INVALID_ARGUMENT;
    }
    if (drafts == 0 || c.n_seqs == 0) return DSV3_OK;
    if (!first || !path || !count) {
        set_last_error("latent_keep: null pointer");
        return DSV3_ERR_INVALID_ARGUMENT;
    }
    DSV3_CUDA_TRY(launch_dependent(latent_keep_kernel, dim3(static_cast<unsigned>(c.n_seqs)), dim3(kThreads), 0,
                                   static_cast<cudaStream_t>(stream), c, first, path, path_stride, drafts, count));
    return DSV3_OK;
}

}  // extern "C"
