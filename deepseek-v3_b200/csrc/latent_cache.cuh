// The 8-bit latent cache: what the kernels that write, read and move its tokens share with the attention over it.
#pragma once

#include "common.cuh"

namespace dsv3 {

constexpr int kLatent = DSV3_LATENT_DIM, kRope = DSV3_ROPE_DIM;

// The cache as the kernels take it.  Slots and pages are 32-bit, byte offsets 64-bit.
struct LatentCache {
    uint8_t* latent;        // [slots, 512]
    __nv_bfloat16* rope;    // [slots, 64]
    float* scale;           // [slots]
    const int32_t* pages;   // [n_seqs, pages_width], rows pages_stride apart
    int64_t pages_stride;
    uint32_t n_pages, page_shift, pages_width;
    int n_seqs;
};

// Checks what every entry point takes of a cache, and fills in the kernels' form.
int latent_cache_arg(const char* who, const dsv3_latent_cache_t* c, bool with_pages, LatentCache* out);

// Slot of a position of sequence `seq`, or -1 where its page is none of the pool.
__device__ __forceinline__ int slot_of(const LatentCache& c, int seq, uint32_t position) {
    const uint32_t p = position >> c.page_shift;
    if (p >= c.pages_width) return -1;
    const uint32_t page = static_cast<uint32_t>(c.pages[seq * c.pages_stride + p]);
    return page < c.n_pages ? static_cast<int>((page << c.page_shift) | (position & ((1u << c.page_shift) - 1u))) : -1;
}

// The least power of two s with amax <= 448 s, for a normal amax: 448 is 1.75 * 2^8, so that the exponent is that of amax less 8, and one more
// where the significand is above 1.75.
__device__ __forceinline__ float power_scale(float amax) {
    const uint32_t bits = __float_as_uint(amax);
    return __uint_as_float(((bits >> 23) - 8u + ((bits & 0x7FFFFFu) > 0x600000u ? 1u : 0u)) << 23);
}
// 1 / s of a power of two whose reciprocal is normal
__device__ __forceinline__ float power_reciprocal(float s) { return __uint_as_float((254u << 23) - __float_as_uint(s)); }

}  // namespace dsv3
