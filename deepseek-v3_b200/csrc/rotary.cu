// Rotary positions (see include/dsv3_b200.h): the table of angles, and the rotation of queries or keys by them.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "common.cuh"

namespace dsv3 {
namespace {

// ---------------------------------------------------------------- the table
constexpr int kMaxPairs = 128, kTableThreads = 256, kTableUnroll = 8;
struct QuarterTurns {
    double per_position[kMaxPairs];       // of an angle: radians * 2 / pi
};

// A thread to one angle of kTableUnroll positions.  The angle is reduced to an eighth of a turn either side of a multiple of a quarter turn in 64 bits, so that position
// 163840 is as exact as position 1; of what is left (r quarters, |r| <= 1/2) sine and cosine are polynomials in r^2, those of their degree whose largest error is least (Remez' exchange: 2^-29.6 and 2^-34.1), in
// 64 bits as well, and rounded once: off by 0.52 * 2^-24 at most.  (In 32 bits, which took as long, by 1.7 * 2^-24, and 43 % of the sines were not the rounded ones.)
//   HBM bounds what is large (163840 positions of 32 angles 9.1 us, 4.6 TB/s), a launch what is small (4096: 2.0 us in a graph).  Conversions between 64-bit numbers and whole ones
// would cost more than all of that (one a cycle and SM; 40 us): the nearest whole number comes from adding 1.5 * 2^52.
__global__ void __launch_bounds__(kTableThreads) rotary_table_kernel(const __grid_constant__ QuarterTurns f, FastDiv pairs, int block_rows, int64_t start, int64_t length,
                                                                     float2* __restrict__ out) {
    griddep_launch_dependents();
    griddep_wait();
    const uint32_t slot = fast_div(threadIdx.x, pairs), pair = threadIdx.x - slot * pairs.d;
    if (static_cast<int>(slot) >= block_rows) return;
    int64_t row = static_cast<int64_t>(blockIdx.x) * block_rows * kTableUnroll + slot;
    const double per = f.per_position[pair], step = static_cast<double>(block_rows);
    double position = static_cast<double>(start + row);
#pragma unroll
    for (int u = 0; u < kTableUnroll; ++u, row += block_rows, position += step) {
        if (row >= length) return;
        constexpr double kWhole = 6755399441055744.0;                // 1.5 * 2^52: a sum with it has no fraction, and the whole number in its low bits
        const double sum = fma(position, per, kWhole);
        const double r = fma(position, per, kWhole - sum), y = r * r;
        const int q = __double2loint(sum);
        const float sine = static_cast<float>(r * fma(y, fma(y, fma(y, -0x1.2cf5d364ef498p-8, 0x1.465a3d5891be3p-4), -0x1.4abba77bb6abfp-1), 0x1.921fb4e70509bp+0));
        const float cosine = static_cast<float>(fma(y, fma(y, fma(y, fma(y, 0x1.d9f7bc182813bp-11, -0x1.55c6643b6d261p-6), 0x1.03c1decc705bap-2), -0x1.3bd3cc7ec2b97p+0), 1.0));
        float2 z = q & 1 ? make_float2(-sine, cosine) : make_float2(cosine, sine);
        if (q & 2) z.x = -z.x, z.y = -z.y;
        out[row * pairs.d + pair] = z;
    }
}

// ---------------------------------------------------------------- the rotation
constexpr int kThreads = 256, kUnroll = 4;

struct Rows {
    const void* x;
    void* out;
    int64_t x_token, x_head, out_token, out_head;       // strides in elements
    const float2* freqs;
    int64_t n_positions;
    const int64_t* positions;                           // or null: token t % per
    int64_t tokens;
    uint32_t per;
    int heads, offset, turned;                          // `turned` units of a head are rotated, the others are copied
    FastDiv units;                                      // of a head
    int teams;                                          // heads that a token's threads take side by side
    FastDiv token_threads;                              // units * teams: threads of a token
    int block_tokens;
    float sign;                                         // of the sines
};

// Eight values of a head as they lie in memory: side by side, or four and four.
template <typename T>
struct Eight {
    uint4 w;
    __device__ __forceinline__ void load(const T* p) { w = *reinterpret_cast<const uint4*>(p); }
    __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<uint4*>(p) = w; }
    __device__ __forceinline__ void load(const T* p, int second) {
        const uint2 a = *reinterpret_cast<const uint2*>(p), b = *reinterpret_cast<const uint2*>(p + second);
        w = make_uint4(a.x, a.y, b.x, b.y);
    }
    __device__ __forceinline__ void store(T* p, int second) const {
        *reinterpret_cast<uint2*>(p) = make_uint2(w.x, w.y);
        *reinterpret_cast<uint2*>(p + second) = make_uint2(w.z, w.w);
    }
    __device__ __forceinline__ void get(float* v) const {
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (sizeof(T) == 2 && std::is_same<T, __half>::value) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
                v[2 * i] = f.x, v[2 * i + 1] = f.y;
            } else {
                v[2 * i] = bf16_bits_to_float(u[i] & 0xFFFFu), v[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u);
            }
        }
    }
    __device__ __forceinline__ void set(const float* v) {
        uint32_t u[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (std::is_same<T, __half>::value) {
                const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
                u[i] = *reinterpret_cast<const uint32_t*>(&h);
            } else {
                u[i] = pack_bf16x2(v[2 * i], v[2 * i + 1]);
            }
        }
        w = make_uint4(u[0], u[1], u[2], u[3]);
    }
};
template <>
struct Eight<float> {
    float4 a, b;
    __device__ __forceinline__ void load(const float* p) { a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1]; }
    __device__ __forceinline__ void store(float* p) const { reinterpret_cast<float4*>(p)[0] = a, reinterpret_cast<float4*>(p)[1] = b; }
    __device__ __forceinline__ void load(const float* p, int second) { a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + second); }
    __device__ __forceinline__ void store(float* p, int second) const { *reinterpret_cast<float4*>(p) = a, *reinterpret_cast<float4*>(p + second) = b; }
    __device__ __forceinline__ void get(float* v) const { v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w; }
    __device__ __forceinline__ void set(const float* v) { a = make_float4(v[0], v[1], v[2], v[3]), b = make_float4(v[4], v[5], v[6], v[7]); }
};

// A unit is eight values of a head, four pairs if they turn: side by side, or in the layout of halves four of either half.  A thread keeps its unit's angles in registers and
// takes every `teams`-th head of its token.  HBM bounds it: heads are asked for kUnroll at once, before the angles, which come by way of the position.  Reads of a unit come before its
// writes, so that out may be x.  4099 tokens of 128 heads of 64: 21.6 us, 22.2 in halves, 6.2 TB/s of what is read and written (from a cold L2 23.8); a part of 2047 tokens of 32 heads of 192 10.4 us
// (units of eight values of either half: 12.7); 64 tokens of 16 heads 1.6 us in a graph, a launch.  fp32 values take 71 to 74 registers, three blocks to an SM: 4099 tokens of 128 heads, cut from heads of 192, 46.3 us, 41.8 in
// halves, 5.8 and 6.4 TB/s (16 bits: 22.2 and 23.7 of such).
template <typename T, bool kHalf>
__global__ void __launch_bounds__(kThreads, sizeof(T) == 2 ? 5 : 3) rotary_kernel(const Rows r) {
    griddep_launch_dependents();
    griddep_wait();
    const uint32_t slot = fast_div(threadIdx.x, r.token_threads), rest = threadIdx.x - slot * r.token_threads.d;
    const int64_t token = static_cast<int64_t>(blockIdx.x) * r.block_tokens + slot;
    if (static_cast<int>(slot) >= r.block_tokens || token >= r.tokens) return;
    const uint32_t team = fast_div(rest, r.units), unit = rest - team * r.units.d;
    const bool turns = static_cast<int>(unit) < r.turned;
    constexpr int kPairs = 4;
    // where the unit begins in a head, and (halves) how far behind it the other values are
    const int rotated = r.turned * 8, second = rotated / 2;
    int at = r.offset + static_cast<int>(unit) * (kHalf ? 4 : 8);
    if (!turns) {
        at = (static_cast<int>(unit) - r.turned) * 8;
        if (at >= r.offset) at += rotated;
    }
    const T* const x = static_cast<const T*>(r.x) + token * r.x_token + at;
    T* const out = static_cast<T*>(r.out) + token * r.out_token + at;
    Eight<T> v[kUnroll];
    const auto fetch = [&](int head) {
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const int h = head + u * r.teams;
            if (h >= r.heads) break;
            if (kHalf && turns) v[u].load(x + h * r.x_head, second);
            else v[u].load(x + h * r.x_head);
        }
    };
    fetch(static_cast<int>(team));
    float2 f[kPairs];
    if (turns) {
        const int64_t position = r.positions ? r.positions[token] : static_cast<int64_t>(static_cast<uint32_t>(token) % r.per);
        const bool there = position >= 0 && position < r.n_positions;
        const float2* const row = r.freqs + (there ? position : 0) * second + unit * kPairs;
#pragma unroll
        for (int i = 0; i < kPairs; ++i) {
            f[i] = there ? row[i] : make_float2(__uint_as_float(0x7FC00000u), __uint_as_float(0x7FC00000u));
            f[i].y *= r.sign;
        }
    }
    for (int head = static_cast<int>(team); head < r.heads;) {
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const int h = head + u * r.teams;
            if (h >= r.heads) break;
            T* const to = out + h * r.out_head;
            if (!turns) {
                v[u].store(to);
                continue;
            }
            float a[8];
            v[u].get(a);
#pragma unroll
            for (int i = 0; i < kPairs; ++i) {
                float &first = a[kHalf ? i : 2 * i], &other = a[kHalf ? 4 + i : 2 * i + 1];
                const float re = fmaf(first, f[i].x, -(other * f[i].y)), im = fmaf(first, f[i].y, other * f[i].x);
                first = re, other = im;
            }
            v[u].set(a);
            if (kHalf) v[u].store(to, second);
            else v[u].store(to);
        }
        head += r.teams * kUnroll;
        if (head < r.heads) fetch(head);
    }
}

}  // namespace
}  // namespace dsv3

using namespace dsv3;

extern "C" {

int dsv3_rotary_table(int dim, double theta, double factor, int64_t original_length, double beta_fast, double beta_slow, int64_t start, int64_t length,
                      float* out, dsv3_stream_t stream) {
    if (length < 0 || start < 0 || dim < 0 || original_length < 1 || !(theta > 1.0) || !(factor > 0.0) || !(beta_fast > 0.0) || !(beta_slow > 0.0) ||
        std::isinf(theta) || std::isinf(factor) || std::isinf(beta_fast) || std::isinf(beta_slow)) {
        set_last_error("rotary_table: a negative size, or a theta, factor or beta that is none");
        return DSV3_ERR_INVALID_ARGUMENT;
    }
    if (dim % 2 != 0 || dim > 2 * kMaxPairs) {
        set_last_error("rotary_table: dim %d must be even and at most %d", dim, 2 * kMaxPairs);
        return DSV3_ERR_UNSUPPORTED;
    }
    const int pairs = dim / 2;
    if (pairs == 0 || length == 0) return DSV3_OK;
    if (length > 0x7FFFFFFFll / pairs || start > (1ll << 40)) {
        set_last_error("rotary_table: 2^31 angles or more, or positions beyond 2^40");
        return DSV3_ERR_UNSUPPORTED;
    }
    if (!out) {
        set_last_error("rotary_table: null pointer");
        return DSV3_ERR_INVALID_ARGUMENT;
    }
    if (reinterpret_cast<uintptr_t>(out) % 8 != 0) {
        set_last_error("rotary_table: out must be 8-byte aligned");
        return DSV3_ERR_UNSUPPORTED;
    }
    constexpr double kPi = 3.14159265358979323846;
    // the index of the angle that turns n times over the original length
    const auto index_of = [&](double n) { return dim * std::log(original_length / (n * 2.0 * kPi)) / (2.0 * std::log(theta)); };
    const double low = std::max(std::floor(index_of(beta_fast)), 0.0), high = std::min(std::ceil(index_of(beta_slow)), dim - 1.0);
    QuarterTurns f = {};
    for (int i = 0; i < pairs; ++i) {
        double per = std::pow(theta, -2.0 * i / dim);
        if (factor != 1.0) {
            const double ramp = std::min(1.0, std::max(0.0, (i - low) / (high != low ? high - low : 0.001)));
            per = per / factor * ramp + per * (1.0 - ramp);
        }
        f.per_position[i] = per * (2.0 / kPi);
    }
    const int block_rows = kTableThreads / pairs;
    const int64_t each = static_cast<int64_t>(block_rows) * kTableUnroll;
    DSV3_CUDA_TRY(launch_dependent(rotary_table_kernel, dim3(static_cast<unsigned>((length + each - 1) / each)), dim3(kTableThreads), 0,
                                   static_cast<cudaStream_t>(stream), f, make_fast_div(pairs), block_rows, start, length, reinterpret_cast<float2*>(out)));
    return DSV3_OK;
}

int dsv3_rotary(const void* x, int64_t x_token_stride, int64_t x_head_stride, void* out, int64_t out_token_stride, int64_t out_head_stride, int dtype,
                int64_t tokens, int heads, int dim, const float* freqs, int64_t n_positions, const int64_t* positions, int64_t per, int offset, int rotated,
                int half_layout, int inverse, dsv3_stream_t stream) {
    if (tokens < 0 || heads < 0 || dim < 0 || n_positions < 0 || offset < 0 || rotated < 0 || offset + static_cast<int64_t>(rotated) > dim ||
        (!positions && per < 1)) {
        set_last_error("rotary: a negative size, or a part that is not within the head");
        return DSV3_ERR_INVALID_ARGUMENT;
    }
    if (dtype != DSV3_BF16 && dtype != DSV3_FP16 && dtype != DSV3_FP32) {
        set_last_error("rotary: type %d is none that it takes", dtype);
        return DSV3_ERR_UNSUPPORTED;
    }
    if (tokens == 0 || heads == 0 || dim == 0) return DSV3_OK;
    if (!x || !out || (n_positions > 0 && rotated > 0 && !freqs)) {
        set_last_error("rotary: null pointer");
        return DSV3_ERR_INVALID_ARGUMENT;
    }
    if (dim % 8 != 0 || offset % 8 != 0 || rotated % 16 != 0 || dim > 1024 || rotated > 2 * kMaxPairs) {
        set_last_error("rotary: dim %d (up to 1024) and offset %d must be multiples of 8, the rotated part %d of 16 (up to %d)", dim, offset, rotated, 2 * kMaxPairs);
        return DSV3_ERR_UNSUPPORTED;
    }
    const int64_t strides = x_token_stride | x_head_stride | out_token_stride | out_head_stride;
    const uintptr_t size = dtype == DSV3_FP32 ? 4 : 2;
    if ((strides * static_cast<int64_t>(size)) % 16 != 0 || (reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(out)) % 16 != 0 ||
        reinterpret_cast<uintptr_t>(freqs) % 8 != 0) {
        set_last_error("rotary: heads of x and out must be 16-byte aligned, freqs 8-byte");
        return DSV3_ERR_UNSUPPORTED;
    }
    if (x == out && (x_token_stride != out_token_stride || x_head_stride != out_head_stride)) {
        set_last_error("rotary: in place, x and out must have the same strides");
        return DSV3_ERR_INVALID_ARGUMENT;
    }
    if (tokens > 0x7FFFFFFFll || per > 0x7FFFFFFFll) {
        set_last_error("rotary: 2^31 tokens or more");
        return DSV3_ERR_UNSUPPORTED;
    }
    const int turned = rotated / 8;
    // (in place what is not rotated stays where it is)
    const int units = turned + (x == out ? 0 : (dim - rotated) / 8);
    if (units == 0) return DSV3_OK;
    const int teams = std::max(1, std::min(heads, kThreads / units)), block_tokens = std::max(1, kThreads / (units * teams));
    const Rows r = {x, out, x_token_stride, x_head_stride, out_token_stride, out_head_stride, reinterpret_cast<const float2*>(freqs), n_positions, positions, tokens,
                    static_cast<uint32_t>(positions ? 1 : per), heads, offset, turned, make_fast_div(units), teams, make_fast_div(units * teams), block_tokens,
                    inverse ? -1.0f : 1.0f};
    const auto go = [&](auto kern) {
        return launch_dependent(kern, dim3(static_cast<unsigned>((tokens + block_tokens - 1) / block_tokens)), dim3(kThreads), 0, static_cast<cudaStream_t>(stream), r);
    };
    DSV3_CUDA_TRY(dtype == DSV3_BF16 ? (half_layout ? go(rotary_kernel<__nv_bfloat16, true>) : go(rotary_kernel<__nv_bfloat16, false>))
                  : dtype == DSV3_FP16 ? (half_layout ? go(rotary_kernel<__half, true>) : go(rotary_kernel<__half, false>))
                                       : (half_layout ? go(rotary_kernel<float, true>) : go(rotary_kernel<float, false>)));
    return DSV3_OK;
}

}  // extern "C"
