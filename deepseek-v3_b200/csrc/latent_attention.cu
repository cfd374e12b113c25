// Attention of absorbed MLA queries over the 8-bit latent cache (see include/dsv3_b200.h).
//
//   x[r, p] = q_latent[r] . c8[p] + q_rope[r] . k16[p]           r: a query head, p: a cached token, c8 and k16 as stored (divided by s[p])
//   y[r, p] = x[r, p] * s[p] * k[r] + log2 s[p]                   k[r]: softmax_scale, log2(e) and the row's own scale
//   out[r]  = sum_p 2^(y - m) c8[p] / sum_p 2^(y - m) / s[p]      m: the row's running maximum of y
//
// Both products run on e4m3 operands as they lie in the cache: nothing is converted to 16 bits on the way, which would cost a conversion and a
// trip through shared memory per cached value.  What is not 8 bits wide is split in two e4m3 values: a bf16 query has 8 significant bits, so that
// hi = e4m3(q), lo = e4m3(16 (q - hi)) is the query itself (scaled by a power of two per row): values down to 2^-13 of the row's largest as they are, those below off by 2^-21 of it at most; a weight 2^(y - m) is off by
// at most 2^-8 of itself, what rounding it to bf16 would cost.  Two e4m3 products take the time of one in bf16, and half the operand bytes.
//   The token's scale is a factor of its scores and, taken into the exponent as log2 s, of its weight in the second product.
//   Rounding of small weights: lo is stored times 16, so that its grid is 2^-13 on a scale where the row's largest weight is 2^5 or more; what is
// below half of that would round to zero, and thousands of tokens that each weigh 2^-19 of one first token do matter.  So an offset
// per token, evenly spread over a step of the grid, is added before rounding: sums of small weights stay what they are.  Within a tile the offsets are 128 evenly spaced
// ones; which token has which, and where between two steps they begin, a hash of the tile's number says, so that the errors of tokens whose content
// follows their position (one place of every tile, every so many tokens) have a mean of zero as well, and those of different tiles have nothing to do with one another.
//
// The tokens are the rows of both MMAs (128 of them) and the query heads the columns: with 16 query heads (one decoding sequence on one rank of
// eight) nothing is padded, and a tile costs what its 128 x 32 bytes per step take to be read from shared memory.
//   S^T [128 tokens, hi | lo]  = C [128, 512] Q^T,  S_rope^T [128, R] = K [128, 64] Q_rope^T (bf16),  O^T [4 x 128 dims, hi | lo] += C^T P^T
// hi and lo stand side by side as columns, which reads C once for both.  C is the MMA's A operand in both products, K-major in the first and transposed
// (MN-major) in the second, from the same bytes.
//
// What bounds it (B200; a call and its join):
//   16 rows (a decoding sequence on one rank of eight): HBM.  A tile is 82 KB and 148 CTAs read 6.3 TB/s while they go; 64 sequences of up to 8192 tokens, 196 MB,
//   take 42 us, of which 28 are that.  The rest is a start (6 us: the work list, then the pages and the queries, then the first tile come from memory one after
//   another, and the first tiles of all SMs at once), the ends of items (1 us each) and the join.
//   32 rows: shared memory.  A tile's products and weights read and write about 310 KB of it, 2400 cycles at 128 bytes a cycle, and a tile takes 3100: the
//   products of a tile wait for its weights, those for its scores, and two tiles are all that fits, so that one's softmax hides only half of the other's products.
//   128 heads of 32 sequences of 8192 tokens 109 us (122 at the 1 kW limit), a chunk of 515 tokens 105 (44 to 45 at the rate of library bf16 products).
#include <cuda.h>

#include <atomic>

#include "latent_cache.cuh"
#include "tc_wait.cuh"

namespace dsv3 {

int make_tmap(CUtensorMap* map, const void* base, int64_t rows, int64_t K, int box_rows);
int make_tmap_groups(CUtensorMap* map, const void* base, int64_t rows, int64_t K, int box_rows);

namespace {

constexpr int kTokens = 128;              // of a tile: MMA M of the first product, K of the second
// A tile is loaded and given back in two units of 64 tokens.  Its latents lie as [16 groups of eight tokens][4 chunks of 128 dimensions][8 tokens][128 bytes],
// swizzled over 128 bytes: one copy brings a page's share of a unit, all four chunks of it (a copy per chunk and page: 450 cycles a chunk to issue, more
// than a tile's share of HBM takes), and both MMAs find a chunk's groups 4096 bytes apart.  (Four units of 32 tokens: 124 us instead of 110 for 128 heads of 32
// sequences of 8192 tokens, every wait more than its earlier copy gains; two units of 256 dimensions, whose scores could begin alone: 114.)
constexpr int kUnitTokens = 64, kTileSlots = 2;
constexpr int kLatentBytes = kTokens * kLatent, kRopeBytes = kTokens * 2 * kRope, kTileBytes = kLatentBytes + kRopeBytes;
constexpr int kGroupBytes = 8 * kLatent;
constexpr int kFirstSoftmaxWarp = 4;
constexpr int kScaleSlots = 4;
constexpr int kAhead = 4, kBoxSlots = 4;  // tiles whose pages are looked up before they are loaded; of which the pages are kept
constexpr int kFewParts = 8;              // of a block that several CTAs worked on
// What a wait that gave up was for (kinds of dsv3_check_device_status)
constexpr uint32_t kTileRoom = 1, kTile = 2, kScoresRoom = 3, kScores = 4, kWeights = 11, kWeightsRoom = 12, kQueriesStaged = 13, kSumsRoom = 14, kList = 15;
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;
// The maximum that weights are relative to moves when a weight would pass 2^(kTop + kSlack), and then stands for 2^kTop.  e4m3 ends at 448; a wide slack costs two of
// the bits below (see the grid of small weights above) and spares nearly all passes over the sums so far.
constexpr float kTop = 5.0f, kSlack = 3.75f;
constexpr float kNothing = -3.0e38f;      // below every finite score, and no infinity: -inf less this is -inf
constexpr float kLoScale = 16.0f;         // of remainders, so that the grid below e4m3's smallest normal value is finer by as much; the largest is 2^-4 of 2^8

struct Queries {
    const __nv_bfloat16 *latent, *rope;
    int64_t latent_token, latent_head, rope_token, rope_head;   // strides in elements
    int tokens, heads;
    const int32_t *seq_lens, *cu;         // cu: null for `per` queries a sequence
    int per;
    const int64_t* tree;
    float scale;
    __nv_bfloat16* out;
    float* lse;
    // a block of query heads: `head_blocks` of them to a token, or 2^block_shift tokens to a block
    int head_blocks, block_shift;
    // 2^16 / heads + 1, for a block of several tokens, and 2^32 / CTAs with a share of their own + 1: a division is some forty instructions that come from memory before
    // they run, once each in a kernel of this length (one tile took 0.4 us longer with them)
    uint32_t per_head, per_cta;
    bool read_once;                       // a sequence's queries are one block
    bool whole;                           // blocks are not cut (unless the kernel looks whether to cut them)
    int group;                            // CTAs that take the blocks of a token's heads side by side, so that a tile is read from HBM once; or 1
    float* partial;                       // [2 * grid][R, 512]
    float* partial_lse;                   // [2 * grid][R]
    int4* cut;                            // [2 * grid]: the item that begins in a CTA and ends in a later one
};

template <int R>
struct Cfg {
    static constexpr int kQChunk = 2 * R * 128;                 // hi and lo rows of 128 latents
    static constexpr int kQBytes = 4 * kQChunk + R * 128;
    static constexpr int kPBytes = kTokens * 2 * R;
    // Softmax warps: four, a quarter of the tile's tokens each, to eight rows.  With 32 rows the softmax is part of the chain that a tile waits for: eight warps of 16 rows to a
    // thread took 15 % longer for 128 sequences of 1024 tokens and 128 heads, 9 % for 24 trees of 13 drafts, 13 % for one
    // sequence of 131072 tokens.
    static constexpr int kRows = 8, kParts = R / kRows, kSoftmaxWarps = 4 * kParts;
    static constexpr int kThreads = 32 * (kFirstSoftmaxWarp + kSoftmaxWarps);
    // What a block takes beside its tiles, in tiles, when work is shared out: its queries' way to shared memory, its result's way out (2.2 and 3 us, with 16 and 32 rows).
    // When it was chosen: 24 trees of 13 drafts 64.6 us, with 0 72.6, with 1 66.9, with 3 65.3; 64 sequences of up to 8192 tokens with 16 heads 46.3, 47.8, 47.0, 46.7.
    static constexpr int kItemCost = 2;
    static constexpr int kTmemS = 3 * R;                        // columns: hi, lo, rotated
    static constexpr int kTmemO = 2 * kTmemS;
    static constexpr int kTmemCols = R == 16 ? 256 : 512;
    static_assert(kTmemO + 8 * R <= kTmemCols, "TMEM");
};

// ---------------------------------------------------------------- PTX
__device__ __forceinline__ void tc_mma_bf16(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "setp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n"
        "}\n" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}
template <int N>
__device__ __forceinline__ void tc_ld(uint32_t taddr, uint32_t* r) {
    static_assert(N == 8 || N == 16, "columns");
    if constexpr (N == 8) tc_ld_x8(taddr, r);
    else tc_ld_x16(taddr, r);
}
template <int N>
__device__ __forceinline__ void tc_st(uint32_t taddr, const uint32_t* r) {
    static_assert(N == 8 || N == 16, "columns");
    if constexpr (N == 8)
        asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]),
                     "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                     : "memory");
    else
        asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
                     "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
                     "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
                     : "memory");
}
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// All chunks of groups of eight rows from `group` on, to shared memory as [group][chunk][8][128]
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const void* tmap, int group, uint32_t bar, uint64_t policy) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%2, %2, %2, %3}], [%4], %5;" ::"r"(dst),
                 "l"(tmap), "r"(0), "r"(group), "r"(bar), "l"(policy)
                 : "memory");
}
__device__ __forceinline__ void tma_load_rope(uint32_t dst, const void* tmap, int row, uint32_t bar, uint64_t policy) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%2, %3}], [%4], %5;" ::"r"(dst), "l"(tmap),
                 "r"(0), "r"(row), "r"(bar), "l"(policy)
                 : "memory");
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar)
                 : "memory");
}
// How long lines stay in the L2: as others, or as the first to go.  Tiles that are read once go first, so that the next launch finds code, lengths and pages there: 64
// sequences of up to 8192 tokens with 16 heads 41.8 us instead of 43.9, 140 of 4096 65.0 instead of 66.4; a chunk of 515 tokens, whose blocks read the same tiles one after another, 108.6 instead of
// 106.3.  (By the rows of a sequence: whether sequences share pages only the table tells.  64 on one prefix of 8192 tokens 47.7 us either way, on one of 32768 156.5 instead of 151.6.)
__device__ __forceinline__ uint64_t l2_policy(bool once) {
    uint64_t p;
    if (once) asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(p));
    else asm volatile("createpolicy.fractional.L2::evict_normal.b64 %0, 1.0;" : "=l"(p));
    return p;
}
__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// Two values at a time: an instruction instead of two (the softmax's warps are short of issue slots with 32 rows: 4 % longer without for 128 heads of 32
// sequences of 8192 tokens).
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 r;
    asm("{\n.reg .b64 a, b;\nmov.b64 a, {%2, %3};\nmov.b64 b, {%4, %5};\nadd.rn.f32x2 a, a, b;\nmov.b64 {%0, %1}, a;\n}"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 r;
    asm("{\n.reg .b64 a, b;\nmov.b64 a, {%2, %3};\nmov.b64 b, {%4, %5};\nmul.rn.f32x2 a, a, b;\nmov.b64 {%0, %1}, a;\n}"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 r;
    asm("{\n.reg .b64 a, b, c;\nmov.b64 a, {%2, %3};\nmov.b64 b, {%4, %5};\nmov.b64 c, {%6, %7};\nfma.rn.f32x2 a, a, b, c;\nmov.b64 {%0, %1}, a;\n}"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return r;
}

// Operand descriptor of a tile whose rows of kWidth bytes are swizzled over that width, groups of eight rows kGroup bytes apart: rows are rows of the
// matrix (K-major), or steps of K (transposed, MN-major).  The operand is one swizzle atom wide, so that the offset between atoms is not used.
template <int kWidth, int kGroup>
__device__ __forceinline__ uint64_t umma_desc(uint32_t smem_addr) {
    static_assert(kWidth == 32 || kWidth == 64 || kWidth == 128, "swizzle width");
    constexpr uint64_t layout = kWidth == 128 ? 2 : kWidth == 64 ? 4 : 6;
    uint64_t d = 0;
    d |= static_cast<uint64_t>((smem_addr & 0x3FFFFu) >> 4);
    d |= static_cast<uint64_t>(1) << 16;
    d |= static_cast<uint64_t>(kGroup >> 4) << 32;
    d |= static_cast<uint64_t>(1) << 46;
    d |= layout << 61;
    return d;
}
constexpr uint32_t kIdescTransposed = (1u << 15) | (1u << 16);                      // A and B MN-major
constexpr uint32_t idesc_bf16(uint32_t m, uint32_t n) { return umma_idesc_e4m3_f32(m, n) | (1u << 7) | (1u << 10); }

// ---------------------------------------------------------------- who works on what
// The work is a list of tiles: for every sequence, block of its query heads and 128 cached tokens that some row of the block sees one (at least one
// per block, which writes the zeros of rows that see nothing).  A CTA takes an equal, contiguous share of the list, whatever the lengths are; a block's
// tiles in one CTA are an item, and a block that is cut leaves partial results which latent_combine_kernel joins.  Where there are no more blocks than CTAs and
// cutting them would save little, a block is one entry of the list and stays whole.  One warp walks the
// list and leaves what the others need in shared memory.
// Whether to cut: an SM's longest block against its equal share of all tiles (0.8 to 1.7 us each), against the ends of more items and the join.
//   Where no row of pages holds more than kSmallTiles tiles the host decides, by the rows' length, and launches no join for whole blocks.  Heads, sequences x tokens:
//   16, 1 x 137 8.4 us, cut 11.0; 16, 60 x 384 11.7, 13.5; 16, 140 x 1024 22.5, 25.9; 128, 24 x 1024 21.4, 26.9; beyond the line 16, 1 x 640 11.8, 10.9; 1 x 1024 14.9, 11.3.
//   Elsewhere the kernel looks at the lengths (which takes a kernel of its own: up to 0.5 us more for those that have no use for it).  Rows of pages longer than that:
//   16, 140 x 4096 64.9 us, cut 69.1; 128, 36 x 2048 40.4, 43.4; beyond the line, when it was drawn, 16, 1 x 512 12.1, 11.1; 128, 8 x 768 19.8, 16.5.
constexpr int kSmallTiles = 8, kSmallSaved = 4, kSaved = 3;
constexpr int kBlockBits = 8;             // of a word that counts tiles and blocks
struct Seq {
    int len, queries, first;              // cached tokens, queries, index of the first query
};
__device__ __forceinline__ Seq load_seq(const LatentCache& c, const Queries& q, int s) {
    const int64_t cap = static_cast<int64_t>(c.pages_width) << c.page_shift;
    Seq r;
    r.len = static_cast<int>(max(static_cast<int64_t>(0), min(static_cast<int64_t>(q.seq_lens[s]), cap)));
    r.first = q.cu ? q.cu[s] : s * q.per;
    // (offsets that lead out of the queries are cut off)
    const int end = q.cu ? q.cu[s + 1] : r.first + q.per;
    r.first = max(0, min(r.first, q.tokens));
    r.queries = max(0, min(end, q.tokens) - r.first);
    return r;
}
__device__ __forceinline__ int tiles_of(int tokens) { return tokens <= kTokens ? 1 : (tokens - 1) / kTokens + 1; }
__device__ __forceinline__ int blocks_of(const Queries& q, const Seq& s) { return (s.queries + (1 << q.block_shift) - 1) >> q.block_shift; }
// Tiles that a block of tokens sees: all, or those up to its last token's own position
__device__ __forceinline__ int block_tiles(const Queries& q, const Seq& s, int block) {
    if (q.tree) return tiles_of(s.len);
    return tiles_of(s.len - s.queries + min((block + 1) << q.block_shift, s.queries));
}
// sum over j = 1 .. x of max(1, ceil(j / m)); x <= 0: what is to be subtracted for j = x + 1 .. 0
__device__ __forceinline__ int64_t ramp(int x, int shift) {
    if (x <= 0) return x;
    const uint32_t n = x >> shift, rest = x - (n << shift);
    return ((static_cast<uint64_t>(n) * (n + 1) / 2) << shift) + static_cast<uint64_t>(rest) * (n + 1);
}
// Tiles of a sequence's first n blocks of tokens (of one block of heads).  Block i sees base + (i + 1) 2^b tokens (the last one: all); with m = 128 / 2^b that
// is ceil((u + i + 1) / m) tiles, where u = ceil(base / 2^b).
__device__ __forceinline__ int tiles_before(const Queries& q, const Seq& s, int n, int blocks) {
    if (n == 0) return 0;
    if (q.tree || blocks == 1) return n * tiles_of(s.len);
    const int u = static_cast<int>((static_cast<int64_t>(s.len) - s.queries + (1 << q.block_shift) - 1) >> q.block_shift);
    const int shift = 7 - q.block_shift;
    const int whole = n == blocks ? n - 1 : n;
    return static_cast<int>(ramp(u + whole, shift) - ramp(u, shift)) + (n == blocks ? tiles_of(s.len) : 0);
}
// ... of the list of work
template <int R>
__device__ __forceinline__ int entries_before(const Queries& q, bool whole, const Seq& s, int n, int blocks) {
    return whole ? n : tiles_before(q, s, n, blocks) + n * Cfg<R>::kItemCost;
}

template <int R>
struct Walk {
    bool whole, more;                     // blocks are entries of the list, not their tiles; the CTA's share has more of them
    Seq s;
    int seq, block, head_block;
    int tile, n, tiles;                   // first tile of the item, how many, how many the whole block has
    int share, at;                        // entries of the CTA; the first tile's place in the list, from the share's start on

    __device__ void settle(const Queries& q) {
        tiles = block_tiles(q, s, block);
        tile = max(0, -at);
        n = min(whole ? 1 : tiles, share - at) - tile;
        if (whole) tile = 0, n = tiles;
        more = next_at() < share;
    }
    __device__ int next_at() const { return at + (whole ? 1 : tiles + Cfg<R>::kItemCost); }
    // the share starts at entry `offset` of sequence `sq`.  (No tiles: nothing but what a block takes beside them.)
    __device__ __forceinline__ void begin(const Queries& q, bool whole_blocks, int sq, const Seq& x, int offset, int entries) {
        whole = whole_blocks;
        seq = sq;
        s = x;
        const int blocks = blocks_of(q, s);
        int lo = 0, hi = blocks;          // largest block whose entries begin at or before the offset
#pragma unroll 1
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (entries_before<R>(q, whole, s, mid, blocks) * q.head_blocks <= offset) lo = mid;
            else hi = mid;
        }
        offset -= entries_before<R>(q, whole, s, lo, blocks) * q.head_blocks;
        block = lo;
        const int t = whole ? 1 : block_tiles(q, s, lo) + Cfg<R>::kItemCost;
        head_block = q.head_blocks > 1 ? offset / t : 0;
        share = entries;
        at = (whole ? 0 : Cfg<R>::kItemCost) - (offset - head_block * t);
        settle(q);
    }
    __device__ __forceinline__ bool next(const LatentCache& c, const Queries& q) {
        if (!more) return false;
        at = next_at();
        if (++head_block == q.head_blocks) {
            head_block = 0;
            if (++block >= blocks_of(q, s)) {
                block = 0;
                do {
                    if (++seq >= c.n_seqs) return false;                       // (offsets that decrease can count more tiles than 32 bits hold)
                    s = load_seq(c, q, seq);
                } while (s.queries == 0);
            }
        }
        settle(q);
        return true;
    }
};

// The list cut in equal shares: the first `more` of them have one tile more.  No share is empty before the last that is not.
struct Shares {
    int size_less, more, ctas;
    __device__ int first(int c) const { return size_less * min(c, ctas) + min(c, more); }
    __device__ int size(int c) const { return c < ctas ? size_less + (c < more ? 1 : 0) : 0; }
    __device__ int owner(int tile) const {
        const int large = more * (size_less + 1);
        return tile < large ? tile / (size_less + 1) : more + (tile - large) / size_less;
    }
};
__device__ __forceinline__ Shares shares_of(int total, int ctas, uint32_t per_cta) {
    if (total < ctas) return {1, 0, total};
    int each = static_cast<int>(__umulhi(static_cast<uint32_t>(total), per_cta));   // total / ctas, or one more
    if (static_cast<uint32_t>(each) * static_cast<uint32_t>(ctas) > static_cast<uint32_t>(total)) --each;
    return {each, total - each * ctas, ctas};
}

// Row r of an item's block, in the CTA that is the `member`-th of those side by side; query -1 where it is none.
struct Row {
    int query, head;
};
template <int R>
__device__ __forceinline__ Row row_of(const Queries& q, const Walk<R>& w, int r, int member) {
    int token = w.block << q.block_shift, head = (w.head_block + member) * R + r;
    if (q.heads <= R) {
        if (r >= q.heads << q.block_shift) return {-1, 0};
        const int t = static_cast<int>(r * q.per_head >> 16);                  // r / heads, below 32
        token += t;
        head = r - t * q.heads;
    }
    return {head < q.heads && token < w.s.queries ? w.s.first + token : -1, head};
}

// What the other warps need of a step of the walk.
struct Item {
    int len, base;                        // the sequence's cached tokens, position of its first query's token
    int tile, n;                          // first tile, how many
    bool begins, ends, last;              // of the block; the CTA's last item
};
constexpr int kItemSlots = 4;
constexpr uint64_t kItemLimitNs = 100 * kWaitLimitNs;   // the walk waits for whole items, and one has up to 2^24 tiles of 2 us

template <int R>
struct Small {                                                  // shared memory beside the operand tiles
    alignas(128) float scales[kScaleSlots][kTokens];
    alignas(16) float factor[2][R];                                         // k[r] by item parity
    int64_t tree[kItemSlots][R];
    int limit[kItemSlots][R];                                   // last position that a row sees (a tree: of those before the queries)
    int place[kItemSlots][R];                                   // query * heads + head, -1 for a row that is none
    int query[kItemSlots][R];
    Item item[kItemSlots];
    uint32_t listed, finished;                                  // items that are written down, whose results have been read
    float top[2][Cfg<R>::kParts][4][Cfg<R>::kRows];             // [tile parity][part of the rows][warp][row]
    float sum[Cfg<R>::kParts][4][Cfg<R>::kRows];
    alignas(16) float row[Cfg<R>::kSoftmaxWarps][Cfg<R>::kRows];                // (read four at a time, as the factors are)
    alignas(16) float row2[Cfg<R>::kSoftmaxWarps][Cfg<R>::kRows];
    uint64_t full[2 * kTileSlots], empty[2 * kTileSlots];
    uint64_t s_full[2], s_empty[2], p_full[2], p_empty[2], q_full, o_empty;
    Control ctl;
    int boxes[kBoxSlots][kTokens / 16 + 1];                     // and whether the tile is the CTA's last
    uint32_t looked_up, taken;                                  // tiles whose boxes are written, have been read
    int2 warp_sum[Cfg<R>::kThreads / 32];
    Walk<R> walk;                                               // the first item
    Shares shares;
};

template <int R>
constexpr int smem_bytes() {
    return 1024 + kTileSlots * kTileBytes + Cfg<R>::kQBytes + 2 * Cfg<R>::kPBytes + static_cast<int>(sizeof(Small<R>));
}
static_assert(smem_bytes<16>() <= 232448 && smem_bytes<32>() <= 232448, "shared memory of a CTA");

// All threads: this CTA's share of the list, and its first item (sm.walk).
template <int R, bool kLooks, typename Sm>
__device__ __forceinline__ void find_share(const LatentCache& c, const Queries& q, Sm& sm) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const bool once = c.n_seqs <= Cfg<R>::kThreads;
    int total = 0;
    // a thread to a sequence; with more sequences than threads once for the total and once more for the place of the share's start
#pragma unroll 1
    for (int pass = 0; pass < 2; ++pass) {
        int at = 0;
#pragma unroll 1
        for (int s0 = 0; s0 < c.n_seqs; s0 += Cfg<R>::kThreads) {
            const int seq = s0 + static_cast<int>(threadIdx.x);
            Seq x = {0, 0, 0};
            int mine = 0, most = 0;                                            // tiles, or tiles and blocks, or blocks; tiles of the longest block
            if (seq < c.n_seqs) {
                x = load_seq(c, q, seq);
                const int b = blocks_of(q, x);
                if (!kLooks) {
                    mine = entries_before<R>(q, q.whole, x, b, b) * q.head_blocks;
                } else {
                    mine = tiles_before(q, x, b, b) * q.head_blocks << kBlockBits | b * q.head_blocks;
                    most = b == 0 ? 0 : tiles_of(x.len);
                }
            }
            if (kLooks) most = __reduce_max_sync(0xffffffffu, most);
            int run = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int u = __shfl_up_sync(0xffffffffu, run, o);
                if (lane >= o) run += u;
            }
            __syncthreads();
            if (lane == 31) sm.warp_sum[warp] = make_int2(run, most);
            __syncthreads();
            int before = at + run - mine;
#pragma unroll
            for (int w = 0; w < Cfg<R>::kThreads / 32; ++w) {
                const int2 v = sm.warp_sum[w];
                if (w < warp) before += v.x;
                at += v.x;
                most = max(most, v.y);
            }
            if (pass == 0 && !once) continue;
            if (once) total = at;
            bool whole = q.whole;
            if (kLooks) {                                             // (a single round; all blocks fit their bits)
                constexpr int mask = (1 << kBlockBits) - 1;
                whole = (most - kSaved) * static_cast<int>(gridDim.y) <= total >> kBlockBits;
                const auto entries = [&](int x) { return whole ? x & mask : (x >> kBlockBits) + (x & mask) * Cfg<R>::kItemCost; };
                total = entries(total), before = entries(before), mine = entries(mine);
            }
            const Shares sh = shares_of(total, gridDim.y, q.per_cta);
            const int first = sh.first(blockIdx.y), share = sh.size(blockIdx.y);
            if (share > 0 && before <= first && first < before + mine) {
                Walk<R> w;
                w.begin(q, whole, seq, x, first - before, share);
                sm.walk = w;
            }
            if (threadIdx.x == 0) sm.shares = sh;
        }
        if (once) break;
        total = at;
    }
}

// ---------------------------------------------------------------- reductions over a tile's tokens
// v[i] of 32 lanes, i < N rows: afterwards every lane holds the reduction of row own_row<N>() over the lanes.  Every exchange halves the rows that a lane
// goes on with: N - 1 + log2(32 / N) shuffles instead of 5 N.
template <int N>
__device__ __forceinline__ int own_row() { return (threadIdx.x & 31) / (32 / N); }
template <int N, typename Op>
__device__ __forceinline__ float reduce_rows(float (&v)[N], Op op) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int half = N / 2, o = 16; half >= 1; half >>= 1, o >>= 1) {
        const bool up = lane & o;
#pragma unroll
        for (int i = 0; i < half; ++i) {
            const float keep = up ? v[i + half] : v[i], give = up ? v[i] : v[i + half];
            v[i] = op(keep, __shfl_xor_sync(0xffffffffu, give, o));
        }
    }
#pragma unroll
    for (int o = 16 / N; o >= 1; o >>= 1) v[0] = op(v[0], __shfl_xor_sync(0xffffffffu, v[0], o));
    return v[0];
}

// The offset of the small weights of a token at position p, evenly over [-2^-10, 2^-10], half a step of lo either side (either end alone rounds to zero, the even one): an odd multiple
// of its place in the tile, and a shift; both by the tile.  (Multiplicative hashing; a shift by the golden ratio from tile to tile is less work, but every 127th
// token then has nearly the same offset.  Offsets that were the same in every tile lost up to a quarter of what sixteen places of every tile held.)
__device__ __forceinline__ float small_offset(uint32_t p) {
    uint32_t h = p / kTokens * 0x9E3779B1u;
    h = (h ^ h >> 16) * 0x85EBCA6Bu;
    static_assert(kTokens == 128, "p times a multiple of 2^25 is its place in the tile times that");
    return static_cast<float>(static_cast<int>(p * ((h & 0xFE000000u) | 0x02000000u) + (h << 7))) * 0x1p-41f;
}

template <int N>
__device__ __forceinline__ void broadcast_rows(float* to, float own, float (&v)[N]) {     // `to`: N floats of this warp
    __syncwarp();
    if ((threadIdx.x & 31) % (32 / N) == 0) to[own_row<N>()] = own;
    __syncwarp();
#pragma unroll
    for (int i = 0; i < N; i += 4) {
        const float4 f = *reinterpret_cast<const float4*>(to + i);
        v[i] = f.x, v[i + 1] = f.y, v[i + 2] = f.z, v[i + 3] = f.w;
    }
}

// Waits until another warp's counter in shared memory has reached `want`, as bounded_wait does for a barrier.
__device__ __forceinline__ bool follow(const uint32_t* counter, uint32_t want, Control* ctl, unsigned int* status, uint64_t limit_ns = kWaitLimitNs) {
    uint64_t t0 = 0;
    for (uint32_t spins = 0;; ++spins) {
        if (*static_cast<const volatile uint32_t*>(counter) >= want) {
            __threadfence_block();
            return true;
        }
        __nanosleep(20);
        if (spins >= 4096u && (spins & 255u) == 0u) {
            if (ctl->abort_flag) return false;
            const uint64_t now = global_timer_ns();
            if (t0 == 0) {
                t0 = now;
            } else if (now - t0 > limit_ns) {
                ctl->abort_flag = 1;
                if (atomicCAS(&status[0], 0u, 1u) == 0u) status[1] = kList, status[2] = want, status[3] = blockIdx.y * gridDim.x + blockIdx.x;
                return false;
            }
        }
    }
}

// ---------------------------------------------------------------- the kernel
// Warp 0 loads, warps 1 and 2 issue the MMAs, warp 3 walks the list, the others do the softmax: four of them (one per quarter of the 128 TMEM lanes, a lane a token)
// for every eight rows.
template <int R, bool kLooks>
__global__ void __launch_bounds__(Cfg<R>::kThreads, 1)
latent_attention_kernel(const __grid_constant__ CUtensorMap map_latent, const __grid_constant__ CUtensorMap map_rope, const LatentCache c, const Queries q,
                        unsigned int* status) {
    using C = Cfg<R>;
    constexpr int N = C::kRows, kSoftmaxWarps = C::kSoftmaxWarps;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* const smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    uint8_t* const tiles = smem;
    uint8_t* const qs = tiles + kTileSlots * kTileBytes;
    uint8_t* const ps = qs + C::kQBytes;
    Small<R>& sm = *reinterpret_cast<Small<R>*>(ps + 2 * C::kPBytes);
    Control* const ctl = &sm.ctl;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const auto bar = [](const uint64_t& b) { return smem_u32(&b); };

    griddep_launch_dependents();
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2 * kTileSlots; ++i) {
            mbar_init(bar(sm.full[i]), 1);
            mbar_init(bar(sm.empty[i]), 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(bar(sm.s_full[i]), 1);
            mbar_init(bar(sm.s_empty[i]), kSoftmaxWarps);
            mbar_init(bar(sm.p_full[i]), kSoftmaxWarps);
            mbar_init(bar(sm.p_empty[i]), 1);
        }
        mbar_init(bar(sm.q_full), kSoftmaxWarps);
        mbar_init(bar(sm.o_empty), kSoftmaxWarps);
        mbar_fence_init();
        ctl->abort_flag = 0;
        sm.looked_up = sm.taken = sm.listed = sm.finished = 0;
        sm.walk.n = 0;
    }
    if (warp == 1) tc_alloc(smem_u32(&ctl->tmem_base), C::kTmemCols);
    if (warp == 0) {
        tma_prefetch_desc(&map_latent);
        tma_prefetch_desc(&map_rope);
    }
    griddep_wait();
    find_share<R, kLooks>(c, q, sm);                 // (its barriers also publish what was set up above)
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = ctl->tmem_base;
    if (threadIdx.x == 32 * 3 && q.cut) q.cut[2 * (blockIdx.y * gridDim.x + blockIdx.x)] = make_int4(-1, 0, 0, 0);

    const int cta = static_cast<int>(blockIdx.y * gridDim.x + blockIdx.x), member = static_cast<int>(blockIdx.x);    // (CTAs side by side have one share)
    const Shares shares = sm.shares;
    const int first = shares.first(blockIdx.y), share = shares.size(blockIdx.y);
    const auto listed = [&](uint32_t item) -> bool { return __all_sync(0xffffffffu, follow(&sm.listed, item + 1, ctl, status)); };

    if (share == 0 || sm.walk.n <= 0) {
        // nothing to do
    } else if (warp == 0) {
        // ------------------------------------------------------------ loads.  One lane issues, with coordinates that the warp has in common.
        const int rows = min(1 << c.page_shift, kUnitTokens), unit_boxes = kUnitTokens / rows;
        const uint64_t policy = l2_policy(q.read_once);
        const uint32_t outside = c.n_pages << c.page_shift;                    // a row that TMA fills with zeros
        uint32_t tile_count = 0;
        bool ok = true;
        for (bool last = false; ok && !last; ++tile_count) {
            ok = __all_sync(0xffffffffu, follow(&sm.looked_up, tile_count + 1, ctl, status));
            const int word = lane <= kTokens / 16 ? sm.boxes[tile_count & (kBoxSlots - 1)][lane] : -2, at = lane < 2 * unit_boxes ? word : -2;
            last = __shfl_sync(0xffffffffu, word, kTokens / 16) != 0;
            __syncwarp();
            if (lane == 0) *static_cast<volatile uint32_t*>(&sm.taken) = tile_count + 1;
            const uint32_t used = __ballot_sync(0xffffffffu, at > -2), present = __ballot_sync(0xffffffffu, at >= 0);
            float* const scales = sm.scales[tile_count & (kScaleSlots - 1)];
            const uint32_t tile_at = smem_u32(tiles) + (tile_count & 1) * kTileBytes;
            for (int h = 0; h < 2 && ok; ++h) {
                const uint32_t slot = 2 * (tile_count & 1) + h, full = bar(sm.full[slot]);
                const uint32_t of_unit = ((1u << unit_boxes) - 1u) << (h * unit_boxes);
                const int boxes = __popc(used & of_unit), bytes = boxes * rows * (kLatent + 2 * kRope) + __popc(present & of_unit) * rows * 4;
                ok = __all_sync(0xffffffffu, bounded_wait<true>(bar(sm.empty[slot]), ((tile_count >> 1) & 1) ^ 1, ctl, status, kTileRoom, tile_count));
                if (!ok) break;
                if ((used & ~present & of_unit) != 0) {                        // an absent page: its tokens have no scale
                    if (at == -1 && lane / unit_boxes == h)
                        for (int i = 0; i < rows; ++i) scales[lane * rows + i] = 0.0f;
                    __syncwarp();
                }
                if (elect_one()) mbar_arrive_expect_tx(full, bytes);
                for (int i = h * unit_boxes; i < h * unit_boxes + boxes; ++i) {
                    const int from = __shfl_sync(0xffffffffu, at, i);
                    const int y = from >= 0 ? from : static_cast<int>(outside);
                    if (elect_one()) {
                        tma_load_4d(tile_at + i * rows * kLatent, &map_latent, y >> 3, full, policy);
                        tma_load_rope(tile_at + kLatentBytes + i * rows * 2 * kRope, &map_rope, y, full, policy);
                        if (from >= 0) bulk_load(smem_u32(scales + i * rows), c.scale + from, rows * 4, full);
                    }
                    __syncwarp();
                }
            }
        }
        // none of the commits onto empty[] may be in flight when the CTA leaves its shared memory to another
        for (uint32_t t = tile_count > 2 ? tile_count - 2 : 0u; ok && t < tile_count; ++t)
            for (int h = 0; h < 2; ++h) ok = ok && __all_sync(0xffffffffu, bounded_wait<true>(bar(sm.empty[2 * (t & 1) + h]), (t >> 1) & 1, ctl, status, kTileRoom, t));
    } else if (warp == 3) {
        // ------------------------------------------------------------ the walk: items and their rows, and pages some tiles ahead of the loads.  (To bring the
        // pages to L2 as well, one to six tiles ahead, only gave HBM more to do: 4 to 20 % longer for 64 sequences of up to 8192 tokens with 16 heads.)
        Walk<R> w = sm.walk;
        const int rows = min(1 << c.page_shift, kUnitTokens), boxes = kTokens / rows;
        uint32_t tile_count = 0, item = 0;
        bool ok = true;
        // the slot where this lane's box of a tile begins; absent: -1, behind the sequence's end: -2
        const auto look_up = [&](int t) -> int {
            const int64_t p0 = static_cast<int64_t>(w.tile + t) * kTokens + lane * rows;
            return lane < boxes && p0 < w.s.len ? slot_of(c, w.seq, static_cast<uint32_t>(p0)) : -2;
        };
        const auto publish = [&](int t, int at) {
            if (lane == kTokens / 16) at = !w.more && t == w.n - 1;
            if (tile_count >= kAhead) ok = __all_sync(0xffffffffu, follow(&sm.taken, tile_count + 1 - kAhead, ctl, status));
            if (lane <= kTokens / 16) sm.boxes[tile_count & (kBoxSlots - 1)][lane] = at;
            __threadfence_block();
            __syncwarp();
            if (lane == 0) *static_cast<volatile uint32_t*>(&sm.looked_up) = tile_count + 1;
            ++tile_count;
        };
        do {
            int t = 0, ahead = look_up(0);
            if (item == 0) {                                                   // (the first loads wait for this, and for nothing else)
                publish(0, ahead);
                t = 1;
                if (w.n > 1) ahead = look_up(1);
            }
            // -------- a lane to a row of the block
            const uint32_t at_item = item & (kItemSlots - 1);
            const Row row = lane < R ? row_of(q, w, lane, member) : Row{-1, 0};
            const int query = max(row.query, 0), head = row.head, place = row.query < 0 ? -1 : query * q.heads + head;
            const int64_t word = q.tree && place >= 0 ? q.tree[query] : 0;
            if (item > 0 && place >= 0) {                                      // its query will be read when the item before is done
                const char* const lat = reinterpret_cast<const char*>(q.latent + query * q.latent_token + head * q.latent_head);
#pragma unroll
                for (int i = 0; i < 2 * kLatent; i += 128) asm volatile("prefetch.global.L2 [%0];" ::"l"(lat + i));
                asm volatile("prefetch.global.L2 [%0];" ::"l"(q.rope + query * q.rope_token + head * q.rope_head));
            }
            if (item >= kItemSlots) ok = __all_sync(0xffffffffu, follow(&sm.finished, item + 1 - kItemSlots, ctl, status, kItemLimitNs));
            if (!ok) break;
            const int base = w.s.len - w.s.queries;
            const bool begins = w.tile == 0, ends = w.tile + w.n == w.tiles;
            if (lane < R) {
                sm.place[at_item][lane] = place;
                sm.query[at_item][lane] = query;
                sm.limit[at_item][lane] = q.tree ? base - 1 : base + query - w.s.first;
                sm.tree[at_item][lane] = word;
            }
            if (lane == 0) sm.item[at_item] = {w.s.len, base, w.tile, w.n, begins, ends, !w.more};
            __threadfence_block();
            __syncwarp();
            if (lane == 0) *static_cast<volatile uint32_t*>(&sm.listed) = item + 1;
            for (; t < w.n && ok; ++t) {
                const int at = ahead;
                if (t + 1 < w.n) ahead = look_up(t + 1);
                publish(t, at);
            }
            if (lane == 0 && !ends) {                                          // (one item of a CTA at most)
                const int start = first + w.at;                                // of the block's tiles, in the list
                const int begun = begins ? static_cast<int>(blockIdx.y) : shares.owner(start), parts = shares.owner(start + w.tiles - 1) - begun + 1;
                if (begins || parts > kFewParts) {
                    q.cut[2 * cta] = make_int4(parts, w.block, w.head_block, static_cast<int>(blockIdx.y) - begun);
                    q.cut[2 * cta + 1] = make_int4(member, w.s.queries, w.s.first, 0);
                }
            }
            __syncwarp();
            ++item;
        } while (ok && w.next(c, q));
    } else if (warp == 1) {
        // ------------------------------------------------------------ scores.  The warp stays converged and elects a lane for the MMAs alone: addresses and
        // descriptors then stay in uniform registers.  The sums have an issuer of their own: in one thread, a tile whose weights are there waits behind
        // the next tile's loads, which wait for the room that its sums make.
        constexpr uint32_t idesc_s = umma_idesc_e4m3_f32(kTokens, 2 * R), idesc_r = idesc_bf16(kTokens, R);
        const uint32_t q_at = smem_u32(qs);
        uint32_t count = 0;                                                    // of tiles
        bool ok = true, last = false;
        for (uint32_t item = 0; ok && !last; ++item) {
            ok = listed(item);
            if (!ok) break;
            const int n = sm.item[item & (kItemSlots - 1)].n;
            last = sm.item[item & (kItemSlots - 1)].last;
            ok = __all_sync(0xffffffffu, bounded_wait<true>(bar(sm.q_full), item & 1, ctl, status, kQueriesStaged, item));
            for (int t = 0; t < n && ok; ++t, ++count) {
                const uint32_t b = count & 1, phase = (count >> 1) & 1, d = tmem + b * C::kTmemS, at = smem_u32(tiles) + b * kTileBytes;
                ok = __all_sync(0xffffffffu, bounded_wait<true>(bar(sm.s_empty[b]), phase ^ 1, ctl, status, kScoresRoom, count));
                for (int h = 0; h < 2; ++h) ok = ok && __all_sync(0xffffffffu, bounded_wait<true>(bar(sm.full[2 * b + h]), phase, ctl, status, kTile, count));
                if (!ok) break;
                tc_fence_after();
                const uint64_t da = umma_desc<128, kGroupBytes>(at), db = umma_desc<128, 1024>(q_at);
                const uint64_t ra = umma_desc<128, 1024>(at + kLatentBytes), rb = umma_desc<128, 1024>(q_at + 4 * C::kQChunk);
                if (elect_one()) {
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
#pragma unroll
                        for (int k = 0; k < 4; ++k)                            // 32 bytes of K a step
                            tc_mma_f8(d, da + (u * 1024 >> 4) + 2 * k, db + (u * C::kQChunk >> 4) + 2 * k, idesc_s, (u | k) != 0);
                    }
#pragma unroll
                    for (int k = 0; k < 4; ++k) tc_mma_bf16(d + 2 * R, ra + 2 * k, rb + 2 * k, idesc_r, k != 0);
                    tc_commit(bar(sm.s_full[b]));
                }
                __syncwarp();
            }
        }
    } else if (warp == 2) {
        // ------------------------------------------------------------ sums
        constexpr uint32_t idesc_o = umma_idesc_e4m3_f32(kTokens, 2 * R) | kIdescTransposed;
        const uint32_t p_at = smem_u32(ps);
        uint32_t count = 0;
        bool ok = true, last = false;
        for (uint32_t item = 0; ok && !last; ++item) {
            ok = listed(item);
            if (!ok) break;
            const int n = sm.item[item & (kItemSlots - 1)].n;
            last = sm.item[item & (kItemSlots - 1)].last;
            for (int t = 0; t < n && ok; ++t, ++count) {
                const uint32_t b = count & 1;
                ok = __all_sync(0xffffffffu, bounded_wait<true>(bar(sm.p_full[b]), (count >> 1) & 1, ctl, status, kWeights, count));
                // (an item's first sums overwrite those of the item before it)
                if (ok && t == 0) ok = __all_sync(0xffffffffu, bounded_wait<true>(bar(sm.o_empty), (item & 1) ^ 1, ctl, status, kSumsRoom, item));
                if (!ok) break;
                tc_fence_after();
                const uint64_t da = umma_desc<128, kGroupBytes>(smem_u32(tiles) + b * kTileBytes), db = umma_desc<2 * R, 16 * R>(p_at + b * C::kPBytes);
                if (elect_one()) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) {                              // 32 tokens a step
#pragma unroll
                        for (int u = 0; u < 4; ++u)
                            tc_mma_f8(tmem + C::kTmemO + u * 2 * R, da + ((k * 4 * kGroupBytes + u * 1024) >> 4), db + (k * 32 * 2 * R >> 4), idesc_o, (t | k) != 0);
                        if (k & 1) tc_commit(bar(sm.empty[2 * b + (k >> 1)]));
                    }
                    tc_commit(bar(sm.p_empty[b]));
                }
                __syncwarp();
            }
        }
    } else if (warp >= kFirstSoftmaxWarp) {
        // ------------------------------------------------------------ softmax
        const int sw = warp - kFirstSoftmaxWarp, part_of = sw >> 2, quarter = sw & 3;
        const int token = quarter * 32 + lane;                                 // of the tile: this thread's TMEM lane
        const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
        uint32_t tile_count = 0;
        bool ok = true;                                                        // the same in all lanes of a warp
        const auto wait = [&](const uint64_t& b, uint32_t parity, uint32_t what, uint32_t counter) -> bool {
            return __all_sync(0xffffffffu, bounded_wait<true>(bar(b), parity, ctl, status, what, counter));
        };
        // The rows of a block, a warp to every eighth of them: all on their way from memory before the first is brought to shared memory, as an operand of
        // the first product.  (This is a single warp's chain of dependent instructions; where the rows lie has been worked out before.)
        constexpr int kMine = R / kSoftmaxWarps;
        uint4 qv[kMine][2];
        uint32_t qr[kMine];
        const auto fetch = [&](const Row& row) {                               // of the first kMine lanes
            const int query = max(row.query, 0);
            const int64_t lat = query * q.latent_token + row.head * q.latent_head, rot = query * q.rope_token + row.head * q.rope_head;
#pragma unroll
            for (int j = 0; j < kMine; ++j) {
                qv[j][0] = qv[j][1] = make_uint4(0, 0, 0, 0);
                qr[j] = 0;
                const uint4* src = reinterpret_cast<const uint4*>(q.latent + __shfl_sync(0xffffffffu, lat, j));
                const uint32_t* from = reinterpret_cast<const uint32_t*>(q.rope + __shfl_sync(0xffffffffu, rot, j));
                if (__shfl_sync(0xffffffffu, row.query, j) >= 0) {
                    qv[j][0] = src[lane * 2], qv[j][1] = src[lane * 2 + 1];
                    qr[j] = from[lane];
                }
            }
        };
        const auto stage = [&](uint32_t par) {
            float own = 1.0f;                                                  // scale of this lane's row
#pragma unroll
            for (int j = 0; j < kMine; ++j) {
                const int r = sw + j * kSoftmaxWarps;
                const uint32_t* const x2 = reinterpret_cast<const uint32_t*>(qv[j]);
                const float re = bf16_bits_to_float(qr[j] & 0xFFFFu), im = __uint_as_float(qr[j] & 0xFFFF0000u);
                // largest size: of two values at a time, as whole numbers; NaN and infinities come out on top
                uint32_t top2 = 0;
#pragma unroll
                for (int i = 0; i < 8; ++i) top2 = __vmaxu2(top2, x2[i] & 0x7FFF7FFFu);
                uint32_t top1 = max(max(top2 & 0xFFFFu, top2 >> 16), 0u), rot1 = max(qr[j] & 0x7FFFu, (qr[j] >> 16) & 0x7FFFu);
                top1 = __reduce_max_sync(0xffffffffu, top1);
                rot1 = __reduce_max_sync(0xffffffffu, rot1);
                const bool finite = max(top1, rot1) < 0x7F80u;
                // (the rotated half is held divided by the same scale, in bf16: the scale is kept from being too small for that)
                const float top = fmaxf(fmaxf(bf16_bits_to_float(top1), bf16_bits_to_float(rot1) * 0x1p-40f), 0x1p-100f);
                const float s = finite ? power_scale(top) : __uint_as_float(0x7FC00000u), inv = finite ? power_reciprocal(s) : 0.0f;
                if (lane == j) own = s;
                uint32_t hi[4], lo[4];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float a = finite ? bf16_bits_to_float(x2[i] & 0xFFFFu) * inv : 0.0f, b = finite ? __uint_as_float(x2[i] & 0xFFFF0000u) * inv : 0.0f;
                    const uint16_t h = cvt_e4m3x2(a, b);
                    const float2 f = e4m3x2_to_float2(h);
                    const uint16_t l = cvt_e4m3x2((a - f.x) * kLoScale, (b - f.y) * kLoScale);
                    if (i & 1) hi[i / 2] |= static_cast<uint32_t>(h) << 16, lo[i / 2] |= static_cast<uint32_t>(l) << 16;
                    else hi[i / 2] = h, lo[i / 2] = l;
                }
                uint8_t* const chunk = qs + (lane >> 3) * C::kQChunk + (((lane & 7) ^ (r & 7)) << 4);
                *reinterpret_cast<uint4*>(chunk + r * 128) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                *reinterpret_cast<uint4*>(chunk + (R + r) * 128) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                *reinterpret_cast<uint32_t*>(qs + 4 * C::kQChunk + r * 128 + ((((lane >> 2) ^ (r & 7)) << 4) | ((lane & 3) << 2))) =
                    finite ? pack_bf16x2(re * inv, im * inv) : 0u;
            }
            if (lane < kMine) sm.factor[par][sw + lane * kSoftmaxWarps] = own * q.scale * kLog2e;
            fence_proxy_async_shared();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(sm.q_full));
        };
        // (the first rows are worked out here, not waited for: with the first page looked up before the walk's list is written 0.5 us less for one tile)
        fetch(lane < kMine ? row_of(q, sm.walk, sw + lane * kSoftmaxWarps, member) : Row{-1, 0});
        stage(0);
        ok = listed(0);
        for (uint32_t item = 0;; ++item) {
            const uint32_t par = item & 1, at_item = item & (kItemSlots - 1);
            ok = barrier_all<32 * kSoftmaxWarps>(1, ok);                       // the factors of all rows; the item before is done with
            if (!ok) break;
            if (threadIdx.x == 32 * kFirstSoftmaxWarp) *static_cast<volatile uint32_t*>(&sm.finished) = item;
            const Item w = sm.item[at_item];
            // d = y + less is the weight's exponent, less the row's negated maximum; nothing has been seen yet: far below every score
            float2 l[N / 2], less[N / 2];
            float m = kNothing;                                                // of row own_row<N>()
#pragma unroll
            for (int i = 0; i < N / 2; ++i) l[i] = make_float2(0.0f, 0.0f), less[i] = make_float2(-kNothing, -kNothing);
            for (int t = 0; t < w.n; ++t, ++tile_count) {
                const uint32_t b = tile_count & 1, phase = (tile_count >> 1) & 1;
                const int p = (w.tile + t) * kTokens + token;
                const float offset = small_offset(p);
                // (room for the weights, and the tokens' scales: both there before the scores are)
                if (tile_count >= 2) ok = ok && wait(sm.p_empty[b], phase ^ 1, kWeightsRoom, tile_count);
                ok = ok && wait(sm.full[2 * b + (quarter >> 1)], phase, kTile, tile_count);
                const float sc = sm.scales[tile_count & (kScaleSlots - 1)][token];
                ok = ok && wait(sm.s_full[b], phase, kScores, tile_count);
                tc_fence_after();
                float2 y[N / 2];
                {
                    uint32_t hi[N], lo[N], ro[N];
                    const uint32_t at = tmem + lanes + b * C::kTmemS + part_of * N;
                    tc_ld<N>(at, hi);
                    tc_ld<N>(at + R, lo);
                    tc_ld<N>(at + 2 * R, ro);
                    tc_wait_ld();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(bar(sm.s_empty[b]));
                    const float e = static_cast<float>(static_cast<int>(__float_as_uint(sc) >> 23) - 127);     // log2 of a power of two
                    const float4* const k = reinterpret_cast<const float4*>(sm.factor[par] + part_of * N);
                    const auto two = [](const uint32_t* v) { return make_float2(__uint_as_float(v[0]), __uint_as_float(v[1])); };
#pragma unroll
                    for (int i = 0; i < N; i += 4) {
                        const float4 f = k[i / 4];
#pragma unroll
                        for (int j = 0; j < 4; j += 2)
                            y[(i + j) / 2] = fma2(add2(fma2(two(lo + i + j), make_float2(1.0f / kLoScale, 1.0f / kLoScale), two(hi + i + j)), two(ro + i + j)),
                                                  mul2(make_float2(sc, sc), j ? make_float2(f.z, f.w) : make_float2(f.x, f.y)), make_float2(e, e));
                    }
                }
                const bool present = p < w.len && sc != 0.0f;
                if (!__all_sync(0xffffffffu, present && p < w.base)) {
#pragma unroll
                    for (int i = 0; i < N; ++i) {
                        const int r = part_of * N + i;
                        bool seen = p <= sm.limit[at_item][r];
                        if (q.tree) seen = seen || (p >= w.base && p - w.base < 64 && ((sm.tree[at_item][r] >> (p - w.base)) & 1));
                        if (!present || !seen) (i & 1 ? y[i / 2].y : y[i / 2].x) = -INFINITY;
                    }
                }
                // -------- a new maximum where some weight would pass 2^8: rare after the first tiles, so that the others only ask whether there is one
                float2 d[N / 2];
                float most = -INFINITY;
#pragma unroll
                for (int i = 0; i < N / 2; ++i) {
                    d[i] = add2(y[i], less[i]);
                    most = fmaxf(most, fmaxf(d[i].x, d[i].y));
                }
                if (!barrier_all<128>(2 + part_of, ok && !(most > kTop + kSlack))) {
                    float v[N], mv[N];
#pragma unroll
                    for (int i = 0; i < N; ++i) v[i] = i & 1 ? y[i / 2].y : y[i / 2].x;
                    const float top = reduce_rows<N>(v, [](float a, float b2) { return fmaxf(a, b2); });
                    if (lane % (32 / N) == 0) sm.top[b][part_of][quarter][own_row<N>()] = top;
                    ok = barrier_all<128>(2 + part_of, ok);
                    if (!ok) break;
                    float all = sm.top[b][part_of][0][own_row<N>()];
#pragma unroll
                    for (int i = 1; i < 4; ++i) all = fmaxf(all, sm.top[b][part_of][i][own_row<N>()]);
                    const float old = m;
                    if (all - m > kTop + kSlack) m = all - kTop;
                    broadcast_rows<N>(sm.row[sw], -m, mv);
#pragma unroll
                    for (int i = 0; i < N / 2; ++i) {
                        less[i] = make_float2(mv[2 * i], mv[2 * i + 1]);
                        d[i] = add2(y[i], less[i]);
                    }
                    if (t > 0) {                                               // sums so far take it
                        float f[N];
                        broadcast_rows<N>(sm.row2[sw], ex2(old - m), f);
#pragma unroll
                        for (int i = 0; i < N / 2; ++i) l[i] = mul2(l[i], make_float2(f[2 * i], f[2 * i + 1]));
                        const uint32_t before = tile_count - 1;
                        ok = wait(sm.p_empty[before & 1], (before >> 1) & 1, kWeightsRoom, before);
                        tc_fence_after();
                        if (ok) {
#pragma unroll 2
                            for (int u = 0; u < 8; ++u) {                      // hi and lo of four times 128 dimensions
                                uint32_t o[N];
                                const uint32_t at = tmem + lanes + C::kTmemO + u * R + part_of * N;
                                tc_ld<N>(at, o);
                                tc_wait_ld();
#pragma unroll
                                for (int i = 0; i < N; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f[i]);
                                tc_st<N>(at, o);
                            }
                            tc_wait_st();
                        }
                    }
                }
                // -------- weights: hi and lo, to shared memory
                if (ok) {
                    const float inv = present ? power_reciprocal(sc) : 0.0f;
                    uint32_t hi[N / 4], lo[N / 4];
#pragma unroll
                    for (int i = 0; i < N; i += 2) {
                        const float2 a = make_float2(ex2(d[i / 2].x), ex2(d[i / 2].y));
                        l[i / 2] = fma2(a, make_float2(inv, inv), l[i / 2]);
                        const uint16_t h = cvt_e4m3x2(a.x, a.y);
                        // (the offset alone rounds to zero: no weight stays none)
                        const float2 rest = fma2(e4m3x2_to_float2(h), make_float2(-1.0f, -1.0f), a);
                        const float2 scaled = fma2(rest, make_float2(kLoScale, kLoScale), make_float2(offset, offset));
                        const uint16_t g = cvt_e4m3x2(scaled.x, scaled.y);
                        if ((i & 2) == 0) hi[i / 4] = h, lo[i / 4] = g;
                        else hi[i / 4] |= static_cast<uint32_t>(h) << 16, lo[i / 4] |= static_cast<uint32_t>(g) << 16;
                    }
                    uint8_t* const row = ps + b * C::kPBytes + token * 2 * R;
                    // (16-byte places of a token's row: hi of sixteen rows each, then lo; swizzled over the row's 2 R bytes)
                    const int turn = R == 32 ? (token >> 1) & 3 : (token >> 2) & 1, place16 = part_of >> 1;
                    *reinterpret_cast<uint2*>(row + ((place16 ^ turn) << 4) + (part_of & 1) * 8) = make_uint2(hi[0], hi[1]);
                    *reinterpret_cast<uint2*>(row + (((R / 16 + place16) ^ turn) << 4) + (part_of & 1) * 8) = make_uint2(lo[0], lo[1]);
                    // Behind the sequence's end lie other sequences' bytes, or none at all; no weight, but 0 x NaN is not 0.
                    if (p >= w.len) {
                        uint8_t* const v = tiles + b * kTileBytes + (token >> 3) * kGroupBytes + (token & 7) * 128 + part_of * (4 / C::kParts) * 1024;
#pragma unroll
                        for (int i = 0; i < 32 / C::kParts; ++i) *reinterpret_cast<uint4*>(v + (i >> 3) * 1024 + ((i + lane) & 7) * 16) = make_uint4(0, 0, 0, 0);
                    }
                    tc_fence_before();
                    fence_proxy_async_shared();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(bar(sm.p_full[b]));
                }
            }
            // -------- the item's result; the next item's queries on their way meanwhile
            if (!w.last) {
                ok = ok && listed(item + 1);
                Row row = {-1, 0};
                if (ok && lane < kMine) {
                    const uint32_t next = (item + 1) & (kItemSlots - 1);
                    const int r = sw + lane * kSoftmaxWarps, query = sm.query[next][r], place = sm.place[next][r];
                    if (place >= 0) row = {query, place - query * q.heads};
                }
                if (ok) fetch(row);
            }
            float of_row[N];
#pragma unroll
            for (int i = 0; i < N; ++i) of_row[i] = i & 1 ? l[i / 2].y : l[i / 2].x;
            float sum = reduce_rows<N>(of_row, [](float a, float b2) { return a + b2; });
            if (lane % (32 / N) == 0) sm.sum[part_of][quarter][own_row<N>()] = sum;
            ok = barrier_all<32 * kSoftmaxWarps>(1, ok);
            if (!ok) break;
            sum = (sm.sum[part_of][0][own_row<N>()] + sm.sum[part_of][1][own_row<N>()]) + (sm.sum[part_of][2][own_row<N>()] + sm.sum[part_of][3][own_row<N>()]);
            float inv[N];
            broadcast_rows<N>(sm.row[sw], sum == 0.0f ? 0.0f : 1.0f / sum, inv);
            if (!w.last) stage(par ^ 1);                                         // (all scores of this item have been read)
            const bool whole = w.begins && w.ends;
            const int part = 2 * cta + (w.begins ? 1 : 0);
            const float lse2 = sum == 0.0f ? -INFINITY : m + __log2f(sum);
            if (quarter == 0 && lane % (32 / N) == 0) {
                const int r = part_of * N + own_row<N>(), to = sm.place[at_item][r];
                if (!whole) q.partial_lse[static_cast<int64_t>(part) * R + r] = lse2;
                else if (q.lse && to >= 0) q.lse[to] = lse2 * kLn2;
            }
            // four rows that this lane writes: 8 bytes each, of four dimensions that it gets from its neighbours
            int to[N / 4];
            {
                const int* const place = sm.place[at_item] + part_of * N + (lane & 1) * (N / 2) + ((lane >> 1) & 1) * (N / 4);
#pragma unroll
                for (int i = 0; i < N / 4; ++i) to[i] = place[i];
            }
            const uint32_t last = tile_count - 1;
            ok = wait(sm.p_empty[last & 1], (last >> 1) & 1, kWeightsRoom, last);
            tc_fence_after();
            if (ok) {
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    uint32_t hi[N], lo[N];
                    const uint32_t at = tmem + lanes + C::kTmemO + u * 2 * R + part_of * N;
                    tc_ld<N>(at, hi);
                    tc_ld<N>(at + R, lo);
                    tc_wait_ld();
                    if (!whole) {
                        float* const dst = q.partial + (static_cast<int64_t>(part) * R + part_of * N) * kLatent + u * 128 + token;
#pragma unroll
                        for (int i = 0; i < N; ++i) dst[i * kLatent] = fmaf(__uint_as_float(lo[i]), 1.0f / kLoScale, __uint_as_float(hi[i])) * inv[i];
                        continue;
                    }
                    float o[N];
#pragma unroll
                    for (int i = 0; i < N; ++i) o[i] = fmaf(__uint_as_float(lo[i]), 1.0f / kLoScale, __uint_as_float(hi[i])) * inv[i];
                    uint32_t two[N / 2];
#pragma unroll
                    for (int i = 0; i < N / 2; ++i) {                          // the other lane of a pair has the next dimension
                        const bool odd = lane & 1;
                        const float got = __shfl_xor_sync(0xffffffffu, odd ? o[i] : o[i + N / 2], 1);
                        two[i] = odd ? pack_bf16x2(got, o[i + N / 2]) : pack_bf16x2(o[i], got);
                    }
#pragma unroll
                    for (int i = 0; i < N / 4; ++i) {
                        const bool up = lane & 2;
                        const uint32_t got = __shfl_xor_sync(0xffffffffu, up ? two[i] : two[i + N / 4], 2);
                        if (to[i] >= 0)
                            *reinterpret_cast<uint2*>(q.out + static_cast<int64_t>(to[i]) * kLatent + u * 128 + (token & ~3)) =
                                up ? make_uint2(got, two[i + N / 4]) : make_uint2(two[i], got);
                    }
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(sm.o_empty));
            if (w.last) break;
        }
    }

    // ---------------------------------------------------------------- teardown
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (ctl->abort_flag) {
        // give copies and MMAs that were already issued time to land before shared memory and TMEM are released
        const uint64_t t0 = global_timer_ns();
        while (global_timer_ns() - t0 < 200000ull) __nanosleep(1000);
        __syncthreads();
    }
    if (warp == 1) {
        tc_fence_after();
        tc_dealloc(tmem, C::kTmemCols);
    }
}

// The results of blocks that several CTAs worked on: out = sum_p 2^(lse_p - lse) out_p.  Thread blocks to every CTA of the kernel before, of teams of 128
// threads: where a block of query heads is in few parts, those of the CTA that it begins in join them, a team to a row, with kAtOnce parts on their way; where it is in many, those of
// all CTAs but its last take a row each, and their teams share its parts.
//   It costs a launch, 1 to 4 us, and reads up to 19 MB that were just written, 4 us.  Where parts are few on average small blocks with a row to a team: 64 sequences of up to
// 8192 tokens with 16 heads 45.2 us when it was chosen, 512 threads and two rows 46.7; where they are many the other way round: one of 131072 with four drafts 45.8, 53 (the
// thread blocks that have nothing to do).  The last CTA of a block joining its parts, in the kernel before, took 2 us longer for the first and 20 for the second.
template <bool kMany>
struct Join {
    static constexpr int kThreads = kMany ? 512 : 256, kTeams = kThreads / 128, kRows = kMany ? 2 : 1, kMinBlocks = kMany ? 2 : 6, kUnroll = kMany ? 8 : 2, kAtOnce = kMany ? 8 : 2;
};
template <int R, bool kMany>
__global__ void __launch_bounds__(Join<kMany>::kThreads, Join<kMany>::kMinBlocks) latent_combine_kernel(const Queries q) {
    using J = Join<kMany>;
    constexpr int kTeams = J::kTeams;
    __shared__ float4 sums[kTeams][128];
    __shared__ float weights[kTeams];
    griddep_launch_dependents();
    griddep_wait();
    const int4 cut = q.cut[2 * blockIdx.x], seq = q.cut[2 * blockIdx.x + 1];
    if (cut.x < 0) return;
    Walk<R> w;
    w.block = cut.y, w.head_block = cut.z;
    w.s = Seq{0, seq.y, seq.z};
    const int parts = cut.x, team = threadIdx.x >> 7, lane = threadIdx.x & 31, at = threadIdx.x & 127;
    const int cta = static_cast<int>(blockIdx.x) - cut.w * q.group;            // that the block begins in
    const auto slot = [&](int i, int r) { return static_cast<int64_t>(2 * (cta + i * q.group) + (i == 0 ? 1 : 0)) * R + r; };
    const auto part = [&](int i, int r) { return reinterpret_cast<const float4*>(q.partial + slot(i, r) * kLatent)[at]; };
    const auto add = [](float4& acc, float f, const float4& v) {
        acc.x = fmaf(f, v.x, acc.x), acc.y = fmaf(f, v.y, acc.y), acc.z = fmaf(f, v.z, acc.z), acc.w = fmaf(f, v.w, acc.w);
    };
    const auto warp_max = [](float v) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
        return v;
    };
    const auto store = [&](int place, const float4& acc, float top, float sum, bool nan) {
        const float inv = nan ? __uint_as_float(0x7FC00000u) : sum == 0.0f ? 0.0f : 1.0f / sum;
        reinterpret_cast<uint2*>(q.out + static_cast<int64_t>(place) * kLatent)[at] =
            make_uint2(pack_bf16x2(acc.x * inv, acc.y * inv), pack_bf16x2(acc.z * inv, acc.w * inv));
        if (q.lse && at == 0) q.lse[place] = nan ? inv : sum == 0.0f ? -INFINITY : (top + __log2f(sum)) * kLn2;
    };
    if (parts <= kFewParts) {
        static_assert(kFewParts <= 32, "a lane to a part");
#pragma unroll
        for (int j = 0; j < J::kRows; ++j) {
            const int r = (static_cast<int>(blockIdx.y) * J::kRows + j) * kTeams + team;
            float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            float4 v[J::kAtOnce];
#pragma unroll
            for (int k = 0; k < J::kAtOnce; ++k)
                if (k < 2 || k < parts) v[k] = part(k, r);                     // (there are two at least)
            const float mine = lane < parts ? q.partial_lse[slot(lane, r)] : -INFINITY;
            const bool nan = __any_sync(0xffffffffu, isnan(mine));
            const float top = warp_max(mine), f = ex2(mine - (top == -INFINITY ? 0.0f : top));
            float sum = 0.0f;
#pragma unroll 1
            for (int i = 0; i < parts; i += J::kAtOnce) {
#pragma unroll
                for (int k = 0; k < J::kAtOnce; ++k) {
                    if (i + k >= parts) break;
                    const float a = __shfl_sync(0xffffffffu, f, i + k);
                    sum += a;
                    add(acc, a, v[k]);
                    if (i + k + J::kAtOnce < parts) v[k] = part(i + k + J::kAtOnce, r);
                }
            }
            const Row row = row_of(q, w, r, seq.x);
            const int place = row.query < 0 ? -1 : row.query * q.heads + row.head;
            if (place >= 0) store(place, acc, top, sum, nan);
        }
        return;
    }
    const int r = cut.w + static_cast<int>(blockIdx.y) * (parts - 1);
    static_assert(kFewParts * (R / (kTeams * J::kRows)) >= R, "a row to each");
    if (cut.w == parts - 1 || r >= R) return;
    const Row row = row_of(q, w, r, seq.x);
    const int place = row.query < 0 ? -1 : row.query * q.heads + row.head;
    if (place < 0) return;                                                     // (the whole thread block)
    float top = -INFINITY, sum = 0.0f;
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    bool nan = false;
    for (int i = lane; i < parts; i += 32) {
        const float v = q.partial_lse[slot(i, r)];
        nan = nan || isnan(v);
        top = fmaxf(top, v);
    }
    top = warp_max(top);
    nan = __any_sync(0xffffffffu, nan);
    const float ref = top == -INFINITY ? 0.0f : top;
#pragma unroll J::kUnroll
    for (int i = team; i < parts; i += kTeams) {
        const float f = ex2(q.partial_lse[slot(i, r)] - ref);
        const float4 v = part(i, r);
        sum += f;
        add(acc, f, v);
    }
    sums[team][at] = acc;
    if (at == 0) weights[team] = sum;
    __syncthreads();
    if (team != 0) return;
#pragma unroll
    for (int i = 1; i < kTeams; ++i) {
        add(acc, 1.0f, sums[i][at]);
        sum += weights[i];
    }
    store(place, acc, top, sum, nan);
}

// Rows of a block: 16 where a sequence has no more query heads than that (on average: the numbers of queries are device memory), else 32.
int block_rows(int64_t tokens, int heads, int n_seqs) { return (tokens + n_seqs - 1) / n_seqs * heads <= 16 ? 16 : 32; }

// (By the SMs of the device, as the workspace is sized, whatever budget of them is set: another thread may set it between the query for the size and the call.)
enum Cut : int { kCut, kLook, kWhole };
Cut cut_mode(int64_t tokens, int heads, int n_seqs, int64_t longest, int sms) {
    if (longest <= kTokens) return kWhole;
    const int rows = block_rows(tokens, heads, n_seqs);
    const int64_t blocks = tokens * ((heads + rows - 1) / rows), most = (longest + kTokens - 1) / kTokens;
    if (blocks > sms) return kCut;
    if (most <= kSmallTiles && most * (sms - blocks) <= static_cast<int64_t>(kSmallSaved) * sms) return kWhole;
    // (what the kernel adds up in one round and one word)
    return n_seqs <= Cfg<16>::kThreads && sms < 1 << kBlockBits && blocks * most < 1 << (31 - kBlockBits) ? kLook : kCut;
}

size_t partial_bytes(int rows, int sms) { return static_cast<size_t>(sms) * (2 * rows * (kLatent + 1) * sizeof(float) + 2 * sizeof(int4)); }

template <int R, bool kLooks>
int launch(const LatentCache& c, Queries q, const CUtensorMap& map_latent, const CUtensorMap& map_rope, int grid, bool many, unsigned int* status,
           cudaStream_t stream) {
    const auto kern = latent_attention_kernel<R, kLooks>;
    static std::atomic<uint64_t> prepared{0};                                  // devices
    int device = 0;
    DSV3_CUDA_TRY(cudaGetDevice(&device));
    if (device >= 64 || !(prepared.load(std::memory_order_relaxed) >> device & 1)) {
        DSV3_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes<R>()));
        if (device < 64) prepared.fetch_or(1ull << device, std::memory_order_relaxed);
    }
    DSV3_CUDA_TRY(launch_dependent(kern, dim3(q.group, grid / q.group), dim3(Cfg<R>::kThreads), smem_bytes<R>(), stream, map_latent, map_rope, c, q, status));
    const auto join = [&](auto kern, int threads, int rows) { return launch_dependent(kern, dim3(grid, R / rows), dim3(threads), 0, stream, q); };
    if (!q.whole)
        DSV3_CUDA_TRY(many ? join(latent_combine_kernel<R, true>, Join<true>::kThreads, Join<true>::kTeams * Join<true>::kRows)
                           : join(latent_combine_kernel<R, false>, Join<false>::kThreads, Join<false>::kTeams * Join<false>::kRows));
    return DSV3_OK;
}

}  // namespace
}  // namespace dsv3

using namespace dsv3;

extern "C" {

size_t dsv3_latent_attention_workspace_bytes(int64_t tokens, int heads, int n_seqs, int64_t longest) {
    const int sms = device_sms();
    if (tokens <= 0 || heads <= 0 || n_seqs <= 0 || cut_mode(tokens, heads, n_seqs, longest, sms) == kWhole) return 0;
    return partial_bytes(block_rows(tokens, heads, n_seqs), sms);
}

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
    if (!q_latent || !q_rope || !seq_lens || !out || c.n_pages == 0) {
        set_last_error("latent_attention: null pointer, or a pool without pages");
        return DSV3_ERR_INVALID_ARGUMENT;
    }
    if (c.n_seqs == 0 || (!cu_seqlens_q && tokens % c.n_seqs != 0)) {
        set_last_error("latent_attention: %lld queries do not divide among %d sequences", static_cast<long long>(tokens), c.n_seqs);
        return DSV3_ERR_INVALID_ARGUMENT;
    }
    if (tree_mask && !cu_seqlens_q && tokens / c.n_seqs > 64) {
        set_last_error("latent_attention: %lld drafted tokens to a sequence, a tree's masks name 64", static_cast<long long>(tokens / c.n_seqs));
        return DSV3_ERR_UNSUPPORTED;
    }
    const int64_t strides = q_latent_token_stride | q_latent_head_stride | q_rope_token_stride | q_rope_head_stride;
    if (strides % 8 != 0 || (reinterpret_cast<uintptr_t>(q_latent) | reinterpret_cast<uintptr_t>(q_rope) | reinterpret_cast<uintptr_t>(out)) % 16 != 0 ||
        reinterpret_cast<uintptr_t>(c.scale) % 16 != 0) {
        set_last_error("latent_attention: rows of the queries and out, and the cache's scales, must be 16-byte aligned");
        return DSV3_ERR_UNSUPPORTED;
    }
    if (heads > 1024 || tokens > 0x7FFFFFFFll / heads) {
        set_last_error("latent_attention: takes at most 1024 heads and 2^31 query heads");
        return DSV3_ERR_UNSUPPORTED;
    }
    const int sms = device_sms(), grid = num_sms(), rows = block_rows(tokens, heads, c.n_seqs);
    const int64_t longest = static_cast<int64_t>(c.pages_width) << c.page_shift;
    if (tokens * ((heads + rows - 1) / rows) > 0x7FFFFFFFll / ((longest + kTokens - 1) / kTokens + 1 + Cfg<32>::kItemCost)) {   // (the kernel counts tiles in 32 bits)
        set_last_error("latent_attention: %lld queries of %d heads over up to %lld tokens are too much work for a call", static_cast<long long>(tokens), heads,
                       static_cast<long long>(longest));
        return DSV3_ERR_UNSUPPORTED;
    }
    const Cut mode = cut_mode(tokens, heads, c.n_seqs, longest, sms);
    const bool cut = mode != kWhole;
    if (cut && (!workspace || workspace_bytes < partial_bytes(rows, sms) || reinterpret_cast<uintptr_t>(workspace) % 256 != 0)) {
        set_last_error("latent_attention: the workspace must be 256-byte aligned and hold %zu bytes", partial_bytes(rows, sms));
        return DSV3_ERR_WORKSPACE;
    }
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    unsigned int* const status = status_device_ptr();
    if (!status) return DSV3_ERR_CUDA;
    const int64_t slots = static_cast<int64_t>(c.n_pages) << c.page_shift;
    const int box = c.page_shift < 6 ? 1 << c.page_shift : kUnitTokens;
    CUtensorMap map_latent, map_rope;
    if (const int rc = make_tmap_groups(&map_latent, c.latent, slots, kLatent, box); rc != DSV3_OK) return rc;
    if (const int rc = make_tmap(&map_rope, c.rope, slots, 2 * kRope, box); rc != DSV3_OK) return rc;
    // tokens to a block: a power of two, so that the tiles of a causal sequence can be counted without adding them up
    int shift = 0;
    while ((heads << (shift + 1)) <= rows) ++shift;
    // the blocks of a token's heads see the same tiles: side by side in as many CTAs, unless those are not there
    const int head_blocks = (heads + rows - 1) / rows, group = 2 * head_blocks <= grid ? head_blocks : 1;
    float* const partial = static_cast<float*>(workspace);
    float* const partial_lse = cut ? partial + static_cast<size_t>(grid) * 2 * rows * kLatent : nullptr;
    int4* const list = cut ? reinterpret_cast<int4*>(partial_lse + static_cast<size_t>(grid) * 2 * rows) : nullptr;
    const Queries q = {static_cast<const __nv_bfloat16*>(q_latent), static_cast<const __nv_bfloat16*>(q_rope), q_latent_token_stride, q_latent_head_stride,
                       q_rope_token_stride, q_rope_head_stride, static_cast<int>(tokens), heads, seq_lens, cu_seqlens_q,
                       cu_seqlens_q ? 0 : static_cast<int>(tokens / c.n_seqs), tree_mask, softmax_scale, static_cast<__nv_bfloat16*>(out), lse,
                       head_blocks / group, shift, 65536u / heads + 1u, 0xFFFFFFFFu / (grid / group) + 1u, (tokens + c.n_seqs - 1) / c.n_seqs * heads <= rows, mode == kWhole, group, partial, partial_lse, list};
    const auto go = rows == 16 ? (mode == kLook ? launch<16, true> : launch<16, false>) : mode == kLook ? launch<32, true> : launch<32, false>;
    const int64_t blocks = (tokens * heads + rows - 1) / rows;
    return go(c, q, map_latent, map_rope, grid / group * group, 2 * kFewParts * blocks <= grid, status, st);
}

}  // extern "C"
