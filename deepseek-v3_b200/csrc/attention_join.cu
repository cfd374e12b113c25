// The results of the same queries over several pieces of their keys, joined (see include/dsv3_b200.h).
//
//   lse = log sum_i exp(lse_i),  out = sum_i exp(lse_i - lse) out_i
//
// HBM bounds it: every part is read once.  dim / 8 neighbouring threads to a row, eight values each.  Up to four parts everything of a row is asked for at once, sums and weights
// (whether a part saw anything or not: waiting for that first takes a second trip to memory).  4 parts of 4096 tokens of 128 heads 105 us, 6.4 TB/s; waiting first, a part at a time, 218 us.  515 tokens
// of 16 heads in two parts 2.1 us in a graph, a launch.
#include <algorithm>

#include "attention_join.cuh"

namespace dsv3 {
namespace {

constexpr int kThreads = 256, kAtOnce = 4;
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;

struct Parts {
    const void* out[kMaxJoinParts];
    const float* lse[kMaxJoinParts];
    int n;
    int64_t rows;
    FastDiv row_threads;
    int block_rows;
    __nv_bfloat16* to;
    float* to_lse;
    bool lse_in_place;        // to_lse is a part's
    const int32_t* cu;        // or null; rows of tokens before cu[0], and from cu[n_seqs] on, are left as they are
    int n_seqs, heads;
};

// Eight values as they lie in memory.
template <typename T>
struct Eight;
template <>
struct Eight<__nv_bfloat16> {
    uint4 w;
    __device__ __forceinline__ void load(const __nv_bfloat16* p) { w = *reinterpret_cast<const uint4*>(p); }
    __device__ __forceinline__ void get(float* v) const {
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) v[2 * i] = bf16_bits_to_float(u[i] & 0xFFFFu), v[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u);
    }
};
template <>
struct Eight<float> {
    float4 a, b;
    __device__ __forceinline__ void load(const float* p) { a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1]; }
    __device__ __forceinline__ void get(float* v) const { v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w; }
};

// kN: at most so many parts, or 0 for any number, kAtOnce of them on their way.
template <typename T, int kN>
__global__ void __launch_bounds__(kThreads) attention_join_kernel(const __grid_constant__ Parts p) {
    griddep_launch_dependents();
    griddep_wait();
    const uint32_t slot = fast_div(threadIdx.x, p.row_threads), at = threadIdx.x - slot * p.row_threads.d;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * p.block_rows + slot;
    if (static_cast<int>(slot) >= p.block_rows || row >= p.rows) return;
    const int64_t from = (row * p.row_threads.d + at) * 8;
    constexpr int kHeld = kN ? kN : kAtOnce;
    Eight<T> v[kHeld];
    float w[kHeld];
    const auto fetch = [&](int first) {
#pragma unroll
        for (int k = 0; k < kHeld; ++k) {
            w[k] = -INFINITY;
            if (first + k < p.n) {
                w[k] = p.lse[first + k][row];
                v[k].load(static_cast<const T*>(p.out[first + k]) + from);
            }
        }
    };
    fetch(0);
    if (p.cu && (row < static_cast<int64_t>(p.cu[0]) * p.heads || row >= static_cast<int64_t>(p.cu[p.n_seqs]) * p.heads)) return;
    float top = -INFINITY;
    bool nan = false;
    const auto see = [&](float x) {
        nan = nan || isnan(x);
        top = fmaxf(top, x);
    };
    if constexpr (kN != 0) {
#pragma unroll
        for (int k = 0; k < kHeld; ++k) see(w[k]);
    } else {
        for (int i = 0; i < p.n; ++i) see(p.lse[i][row]);
    }
    const float ref = top == -INFINITY ? 0.0f : top;
    float acc[8] = {}, sum = 0.0f;
    for (int first = 0;;) {
#pragma unroll
        for (int k = 0; k < kHeld; ++k) {
            if (w[k] == -INFINITY) continue;                         // (what a part that sees nothing left there does not matter)
            const float e = exp2f((w[k] - ref) * kLog2e);
            float x[8];
            v[k].get(x);
            sum += e;
#pragma unroll
            for (int j = 0; j < 8; ++j) acc[j] = fmaf(e, x[j], acc[j]);
        }
        first += kHeld;
        if (kN != 0 || first >= p.n) break;
        fetch(first);
    }
    const float inv = nan ? __uint_as_float(0x7FC00000u) : sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[j] *= inv;
    *reinterpret_cast<uint4*>(p.to + from) = make_uint4(pack_bf16x2(acc[0], acc[1]), pack_bf16x2(acc[2], acc[3]), pack_bf16x2(acc[4], acc[5]), pack_bf16x2(acc[6], acc[7]));
    // (every thread of a row, which can be in several warps, has read the parts' before one writes.  Threads that have left do not keep the barrier waiting.)
    if (p.lse_in_place) __syncthreads();
    if (p.to_lse && at == 0) p.to_lse[row] = nan ? inv : sum == 0.0f ? -INFINITY : top + log2f(sum) * kLn2;
}

template <typename T>
int launch(const void* const* outs, const float* const* lses, int n, int64_t rows, int dim, const int32_t* cu, int n_seqs, int heads, void* out, float* lse,
           cudaStream_t stream) {
    const int row_threads = dim / 8, block_rows = kThreads / row_threads;
    Parts p = {};
    for (int i = 0; i < n; ++i) {
        p.out[i] = outs[i], p.lse[i] = lses[i];
        p.lse_in_place = p.lse_in_place || lses[i] == lse;
    }
    p.n = n, p.rows = rows, p.row_threads = make_fast_div(row_threads), p.block_rows = block_rows;
    p.to = static_cast<__nv_bfloat16*>(out), p.to_lse = lse;
    p.cu = cu, p.n_seqs = n_seqs, p.heads = heads;
    const auto go = [&](auto kern) { return launch_dependent(kern, dim3(static_cast<unsigned>((rows + block_rows - 1) / block_rows)), dim3(kThreads), 0, stream, p); };
    DSV3_CUDA_TRY(n <= 2 ? go(attention_join_kernel<T, 2>) : n <= 4 ? go(attention_join_kernel<T, 4>) : go(attention_join_kernel<T, 0>));
    return DSV3_OK;
}

}  // namespace

int join_partials(const float* partial, const float* partial_lse, int n, int64_t rows, int dim, const int32_t* cu, int n_seqs, int heads, void* out, float* lse,
                  cudaStream_t stream) {
    const void* outs[kMaxJoinParts];
    const float* lses[kMaxJoinParts];
    for (int i = 0; i < n; ++i) outs[i] = partial + static_cast<int64_t>(i) * rows * dim, lses[i] = partial_lse + static_cast<int64_t>(i) * rows;
    return launch<float>(outs, lses, n, rows, dim, cu, n_seqs, heads, out, lse, stream);
}

}  // namespace dsv3

using namespace dsv3;

extern "C" int dsv3_attention_join(const void* const* outs, const float* const* lses, int parts, int64_t rows, int dim, void* out, float* lse,
                                   dsv3_stream_t stream) {
    if (parts < 1 || rows < 0 || dim < 0 || !outs || !lses) {
        set_last_error("attention_join: no parts, or a negative size");
        return DSV3_ERR_INVALID_ARGUMENT;
    }
    if (parts > kMaxJoinParts || dim % 8 != 0 || dim > 8 * kThreads || rows > 0x7FFFFFFFll) {
        set_last_error("attention_join: takes up to %d parts of less than 2^31 rows of a multiple of 8 values (up to %d), not %d of %lld of %d", kMaxJoinParts, 8 * kThreads,
                       parts, static_cast<long long>(rows), dim);
        return DSV3_ERR_UNSUPPORTED;
    }
    if (rows == 0 || (dim == 0 && !lse)) return DSV3_OK;
    if (dim == 0) {
        set_last_error("attention_join: rows without values have no threads that would join their logarithms");
        return DSV3_ERR_UNSUPPORTED;
    }
    for (int i = 0; i < parts; ++i) {
        if (!outs[i] || !lses[i] || !out) {
            set_last_error("attention_join: null pointer");
            return DSV3_ERR_INVALID_ARGUMENT;
        }
        if (reinterpret_cast<uintptr_t>(outs[i]) % 16 != 0 || reinterpret_cast<uintptr_t>(out) % 16 != 0) {
            set_last_error("attention_join: parts and result must be 16-byte aligned");
            return DSV3_ERR_UNSUPPORTED;
        }
    }
    return launch<__nv_bfloat16>(outs, lses, parts, rows, dim, nullptr, 0, 0, out, lse, static_cast<cudaStream_t>(stream));
}
