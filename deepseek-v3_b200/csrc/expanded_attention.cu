// Attention of a prompt's queries over keys and values that the latents were expanded to (see include/dsv3_b200.h).
//
//   x[r, p] = q_nope[r] . k_nope[p] + q_rope[r] . k_rope[p]          r: a query of one head, p: a key; k_rope is shared by the heads
//   out[r]  = sum_p 2^(c x - m) v[p] / sum_p 2^(c x - m)             c: softmax_scale log2(e), m: a running reference of the row
//
// One pass over the keys.  A CTA works on 256 queries of a head as two halves of 128 (the M of an MMA), a lane of TMEM and a softmax thread to a query; keys come in tiles of 128,
// which both halves use.  In TMEM lie the scores of one half's tile at a time (128 columns: the softmax takes them to registers at once, so that the halves take turns), both halves'
// weights (64 columns each, two bf16 to a column) and both halves' sums (128 each).  Weights are the A operand of the second product from TMEM: they never see shared memory, which the
// operands of the first keep busy.
//   Long chunks are worked on by CTAs in pairs (cta_group::2): halves of 256 queries, 128 in either CTA, and either loads half of the keys' rows and half of the values' dimensions for both.
// The ring of keys and values then holds three tiles, not one and a half, and loads half as much: 16001 tokens of 16 heads 844 us, 942 by CTAs alone.
//   The reference m of a row moves only where a weight would pass 2^8, so that sums are hardly ever rescaled; weights are rounded to bf16 (by 2^-8 of themselves
// at most: the tensor cores' type, and what the reference rounds its scores to), sums and statistics are fp32.
//   Blocks of at most half as many queries give both halves the same queries and every other tile of the keys, and join the halves at the end; where there are fewer blocks
// than SMs, the keys of each are cut in parts for as many CTAs, and a second kernel joins those.
//   What bounds it: the tensor cores on long sequences.  8192 queries and keys of 32 heads, each query seeing all keys: 855 us, 1607 TFLOP/s, as much as a large matrix product reaches (seeing
// those before it: 462 us, the tensor pipe 84 % busy).  In a row of calls that lasts, the power limit lowers the clock: 986 us for 16001 tokens of 16 heads, 1330 TFLOP/s.  A block's begin
// and end take as long as 2.5 tiles of a half (4.5 of a pair's): 4096 tokens of 128 heads 518 us, 1327 TFLOP/s; 515 of 16 heads over 4099 keys 35.4 us, 572.  Few queries: HBM, 64 of 128 heads over
// 4000 keys 55 us, 4.8 TB/s.  A single short block: what one tile takes from end to end, 37 tokens 7.4 us in a graph.
//
// Keys and values behind a sequence's end belong to another one, or to nobody: what they score is replaced, and their values are cleared in shared memory before the MMA
// that would multiply them by zero (0 * NaN).  The same warp looks at the tiles that some queries of a block see only in part for values that are not finite.
#include <cuda.h>

#include <algorithm>
#include <atomic>
#include <cmath>

#include "attention_join.cuh"
#include "tc_wait.cuh"

namespace dsv3 {

int make_tmap_heads(CUtensorMap* map, const void* base, int width, int64_t heads, int64_t rows, int64_t head_stride, int64_t row_stride, int box_rows);

namespace {

constexpr int kNope = DSV3_NOPE_DIM, kRope = DSV3_ROPE_DIM, kValue = DSV3_VALUE_DIM;
constexpr int kHalf = 128;                       // queries of a CTA's half of a block
constexpr int kTile = 128;                       // keys
// Operands lie as rows of 64 values (128 bytes, swizzled).  Keys and values come through a ring of slots: three to a tile of keys (64 dimensions of 128 keys
// each), two to one of values (64 keys of 128 dimensions each).  A slot is 16 KB, of a pair's CTA 8: beside the queries there is room for eight or sixteen, one and a half or three tiles of both.
constexpr int kKeySlots = 3, kValueSlots = 2;
// A tile's keys, or its values, are a unit, which is waited for and given back as a whole.
constexpr int kUnits = 8;                        // of either that can be on their way: a ring of a pair's slots has room for no more values
constexpr int kRingBytes = 131072, kQueryPart = kHalf * 128, kQueryBytes = kKeySlots * kQueryPart;
constexpr int kOperandBytes = kRingBytes + 2 * kQueryBytes;
// One CTA, or a pair of them: both halves of a block have 128 queries in either, and either loads half of the keys' rows and half of the values' dimensions.
template <int kCtas>
struct Cfg {
    static constexpr int kRows = kCtas * kHalf, kBlock = 2 * kRows;                  // queries of a half, of a block
    static constexpr int kSlotBytes = 16384 / kCtas, kSlots = kRingBytes / kSlotBytes;
    // (a wait by parity is exact for who has seen the phase before: a unit's barrier is not used again before the unit is given back)
    static_assert(kSlots / std::min(kKeySlots, kValueSlots) <= kUnits, "units in the ring");
    // bf16 x bf16 -> fp32
    static constexpr uint32_t kIdescScores = umma_idesc_e4m3_f32(kRows, kTile) | (1u << 7) | (1u << 10);
    static constexpr uint32_t kIdescSums = umma_idesc_e4m3_f32(kRows, kValue) | (1u << 7) | (1u << 10) | (1u << 16);      // B transposed
};
constexpr int kSoftmaxWarps = 8, kScoreWarp = 8, kLoadWarp = 9, kGuardWarp = 10, kSumWarp = 11, kFinishWarp = 12, kFinishWarps = 4, kThreads = 512;
constexpr int kSoftmaxRegs = 176, kOtherRegs = 80;
static_assert(kSoftmaxRegs * 256 + kOtherRegs * 256 <= 65536 / kThreads / 8 * 8 * kThreads, "what the block was launched with");
constexpr int kTmemScores = 0, kTmemWeights = kTile, kTmemSums = 2 * kTile, kTmemCols = 512;   // columns; weights: 64 to a half, sums: 128
constexpr int kAhead = 1;                        // tiles that scores are ahead of sums (twice as many where halves take turns)
constexpr int kAskEarly = 2;                     // tiles before an item's end at which the next item is asked for
constexpr int kNotFiniteSlots = 8;
constexpr int kItemSlots = 2, kItemReaders = kSoftmaxWarps + 3 + kFinishWarps;
constexpr int kLanes = 32;                       // sequences that are put in order of their length
// What a wait that gave up was for (kinds of dsv3_check_device_status)
constexpr uint32_t kRoom = 1, kTileThere = 2, kScoresRoom = 3, kScoresThere = 4, kWeightsThere = 16, kSumsThere = 17, kQueriesThere = 18, kGuarded = 19, kItems = 20, kRowsRoom = 21, kWeightsRoom = 22;
constexpr uint64_t kItemLimitNs = 100 * kWaitLimitNs;
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;
// A row's reference moves where a weight would pass 2^kSlack: bf16 weights and fp32 sums have the same bits wherever they are.  What weights are larger by is range that values lose: sums of n of them pass
// fp32's largest for values beyond 2^(120 - log2 n).  (With 32 instead of 8 each of 25 calls took the same time within 0.6 %, and values of 2^95 could overflow.)
constexpr float kSlack = 8.0f;

struct Params {
    int tokens, kv_tokens, heads, n_seqs;
    const int32_t *cu_q, *cu_k;           // null: per_q, per_k each
    int per_q, per_k;
    bool causal;
    float scale;                          // softmax_scale log2(e)
    int head_group;
    int splits;
    int blocks;                           // at most, of offsets that ascend
    FastDiv by_splits, by_group, by_last_group;      // ... and by the heads of the last group
    bool dynamic;                         // CTAs take the place of those that have not started; else every gridDim.x-th item
    __nv_bfloat16* out;
    float* lse;
    float *partial, *partial_lse;         // with splits: [splits, tokens, heads, 128] and without the last
};

// A block of queries of one head, and the tiles of keys that a CTA takes of it.
struct Item {
    int q0, rows;                         // first query, how many (0: nothing left)
    int k0, len;                          // the sequence's first key, how many it has
    int limit;                            // last key that the first query sees (a further query one more, if causal)
    int head, split;
    int tile, n;                          // first tile, how many
    int n0, n1;                           // ... of which either half takes
    bool alternate;                       // both halves have the same queries and every other tile
    int edge;                             // tiles from this one on are not seen as a whole by all queries
};

struct Small {
    uint64_t k_full[kUnits], k_empty[kUnits], v_full[kUnits], v_ready[kUnits], v_empty[kUnits];
    uint64_t q_full[2], q_empty[2], s_full[2], s_empty, p_full[2][kValueSlots], p_empty[2], o_full[2], item_full[kItemSlots], item_empty[kItemSlots], row_full[2], row_empty[2], o_empty[2], taken, seen;
    Item item[kItemSlots];
    int not_finite[kNotFiniteSlots];      // first key whose values are not finite, of those in tiles that are not seen as a whole
    alignas(16) uint32_t answer[4];
    int next_at;                          // of a pair: what the first CTA was answered
    float2 row[2][kHalf];                 // reference and sum of the halves' rows
    Control ctl;
};
constexpr int kSmallBytes = (sizeof(Small) + 1023) / 1024 * 1024, kSmemBytes = kSmallBytes + kOperandBytes;
static_assert(kSmemBytes <= 232448, "shared memory of a CTA");

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
// ... with A in TMEM
__device__ __forceinline__ void tc_mma_bf16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "setp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n"
        "}\n" ::"r"(d_tmem),
        "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}
// ... by a pair of CTAs: rows 0 .. 127 in the first one, the others in the second; either has half of B's columns
__device__ __forceinline__ void tc_mma_bf16_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "setp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n"
        "}\n" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void tc_mma_bf16_ts_pair(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "setp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], [%1], %2, %3, p;\n"
        "}\n" ::"r"(d_tmem),
        "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void tc_st_x32(uint32_t taddr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
        "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
        "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]),
        "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}
__device__ __forceinline__ void tc_st_x16(uint32_t taddr, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr), "r"(r[0]), "r"(r[1]),
                 "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]),
                 "r"(r[15])
                 : "memory");
}
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const void* tmap, int x, int head, int row, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst), "l"(tmap), "r"(x),
                 "r"(head), "r"(row), "r"(bar)
                 : "memory");
}
// ... whose completion is signalled on a barrier of the pair's first CTA (shared::cluster address)
__device__ __forceinline__ void tma_load_3d_pair(uint32_t dst, const void* tmap, int x, int head, int row, uint32_t bar_cluster) {
    asm volatile("cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst), "l"(tmap), "r"(x),
                 "r"(head), "r"(row), "r"(bar_cluster)
                 : "memory");
}
__device__ __forceinline__ void store_cluster(uint32_t at, int v) { asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(at), "r"(v) : "memory"); }
__device__ __forceinline__ void min_cluster(uint32_t at, int v) {
    int old;
    asm volatile("atom.shared::cluster.min.s32 %0, [%1], %2;" : "=r"(old) : "r"(at), "r"(v) : "memory");
}
__device__ __forceinline__ void mbar_arrive_cluster_release(uint32_t bar_cluster) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar_cluster) : "memory");
}
__device__ __forceinline__ void fence_cluster() { asm volatile("fence.acq_rel.cluster;" ::: "memory"); }
__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float rcp(float x) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 r;
    asm("{\n.reg .b64 a, b;\nmov.b64 a, {%2, %3};\nmov.b64 b, {%4, %5};\nadd.rn.f32x2 a, a, b;\nmov.b64 {%0, %1}, a;\n}"
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
__device__ __forceinline__ float max3(float a, float b, float c) {    // NaN if one is
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
// 16 N bytes of each of the warp's 32 rows, `stride` bytes apart, of which this lane has one (w) and writes 16 bytes of N: a store of 16 bytes to 32 rows takes 32 passes
// through the L1, one of N neighbouring lanes to a row 32 / N.  Rows at and beyond `rows` are not written.
template <int kWords>
__device__ __forceinline__ void store_rows(uint32_t (&w)[kWords], void* first, int64_t stride, int rows) {
    constexpr int N = kWords / 4;
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int o = 1; o < N; o <<= 1) {
        const bool up = lane & o;
#pragma unroll
        for (int a = 0; a < N; ++a) {
            if (a & o) continue;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                uint32_t &lo = w[4 * a + k], &hi = w[4 * (a + o) + k];
                const uint32_t got = __shfl_xor_sync(0xffffffffu, up ? lo : hi, o);
                if (up) lo = got;
                else hi = got;
            }
        }
    }
    char* const to = static_cast<char*>(first) + (lane & ~(N - 1)) * stride + (lane & (N - 1)) * 16;
#pragma unroll
    for (int r = 0; r < N; ++r)
        if ((lane & ~(N - 1)) + r < rows) *reinterpret_cast<uint4*>(to + r * stride) = make_uint4(w[4 * r], w[4 * r + 1], w[4 * r + 2], w[4 * r + 3]);
}
// Takes the place of a CTA of the grid that has not started; the answer (16 bytes) says whose.
__device__ __forceinline__ void try_cancel(uint32_t answer, uint32_t bar) {
    asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(answer), "r"(bar) : "memory");
}
__device__ __forceinline__ int cancelled_cta(uint32_t answer) {       // or -1: all have started
    int x;
    asm volatile(
        "{\n"
        ".reg .b128 h;\n"
        ".reg .pred p;\n"
        ".reg .b32 y, z, w;\n"
        "ld.shared.b128 h, [%1];\n"
        "mov.b32 %0, -1;\n"
        "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, h;\n"
        "@p clusterlaunchcontrol.query_cancel.get_first_ctaid.v4.b32.b128 {%0, y, z, w}, h;\n"
        "}\n"
        : "=r"(x)
        : "r"(answer)
        : "memory");
    return x;
}

// 64 keys of 128 values as two blocks (of a pair: one) of [64 keys][64 values], 128-byte swizzle, K (the keys) the slow dimension: groups of eight keys are 1024 bytes apart, the
// blocks 8192.
__device__ __forceinline__ uint64_t umma_desc_values(uint32_t smem_addr) {
    uint64_t d = 0;
    d |= static_cast<uint64_t>((smem_addr & 0x3FFFFu) >> 4);
    d |= static_cast<uint64_t>(8192 >> 4) << 16;
    d |= static_cast<uint64_t>(1024 >> 4) << 32;
    d |= static_cast<uint64_t>(1) << 46;
    d |= static_cast<uint64_t>(2) << 61;
    return d;
}
// ---------------------------------------------------------------- who works on what
struct Seq {
    int q0, queries, k0, keys;
};
// (offsets that lead out of the tensors are cut off)
__device__ __forceinline__ Seq load_seq(const Params& p, int s) {
    Seq r = {0, 0, 0, 0};
    if (s >= p.n_seqs) return r;
    int q1, k1;
    if (p.cu_q) r.q0 = p.cu_q[s], q1 = p.cu_q[s + 1];
    else r.q0 = s * p.per_q, q1 = r.q0 + p.per_q;
    if (p.cu_k) r.k0 = p.cu_k[s], k1 = p.cu_k[s + 1];
    else r.k0 = s * p.per_k, k1 = r.k0 + p.per_k;
    r.q0 = max(0, min(r.q0, p.tokens));
    r.k0 = max(0, min(r.k0, p.kv_tokens));
    r.queries = max(0, min(q1, p.tokens) - r.q0);
    r.keys = max(0, min(k1, p.kv_tokens) - r.k0);
    return r;
}

// The list of items: groups of heads, in those the blocks of queries, in those the heads of the group and the parts of the keys.  A group has so many heads that the CTAs
// that work at one time share few heads' keys, which the L2 then holds.  Blocks with more keys come first (up to 32 sequences): an SM that is done
// takes the next item of the list, and what is left for the end is short.
template <int kCtas>
struct List {
    static constexpr int kBlock = Cfg<kCtas>::kBlock, kRows = Cfg<kCtas>::kRows;
    static __device__ __forceinline__ int blocks_of(int queries) { return (queries + kBlock - 1) / kBlock; }
    Seq mine;                             // this lane's sequence (up to 32)
    int blocks, behind;                   // its blocks; by how many blocks' tiles it is shorter than the longest
    int short_at;                         // its last block's place in their order, if the halves share the tiles: it takes half the time
    int total, last_step;                 // blocks in all; steps in which blocks come up
    int chunk, before;                    // beyond 32 sequences: first of the 32 at hand, blocks before those
    uint32_t group, group_first;          // group of heads of the item found last, the first item of it (but for parts)
    int step, earlier;                    // ... the step in which its block came up, and the blocks of the steps before
    __device__ __forceinline__ void begin(const Params& p) {
        const int lane = threadIdx.x & 31;
        chunk = before = step = earlier = 0;
        group = group_first = 0;
        mine = load_seq(p, lane);
        blocks = blocks_of(mine.queries);
        const int tiles = blocks > 0 ? (mine.keys + kTile - 1) / kTile : 0;
        behind = (__reduce_max_sync(0xffffffffu, tiles) - tiles) / (kBlock / kTile);
        const bool is_short = blocks > 0 && mine.queries - (blocks - 1) * kBlock <= kRows;
        short_at = !is_short ? 0 : p.causal ? min(blocks - 1, tiles / 2 / (kBlock / kTile)) : blocks - 1;
        last_step = __reduce_max_sync(0xffffffffu, blocks > 0 ? behind + blocks : 0) - 1;
        total = __reduce_add_sync(0xffffffffu, blocks);
        for (int s = kLanes; s < p.n_seqs; s += kLanes) total += __reduce_add_sync(0xffffffffu, blocks_of(load_seq(p, s + lane).queries));
        total = max(0, min(total, p.blocks));                        // (offsets that do not ascend: some blocks are left out, none is looked for that the grid does not have)
    }
    __device__ __forceinline__ int up_to(int step) const {           // blocks that come up in steps 0 .. step
        return __reduce_add_sync(0xffffffffu, max(0, min(step - behind + 1, blocks)));
    }
    // Whole warp: item number `at`.
    __device__ __forceinline__ Item find(const Params& p, uint32_t at) {
        Item it = {};
        if (at >= static_cast<uint32_t>(total) * p.heads * p.splits) return it;
        const uint32_t unsplit = fast_div(at, p.by_splits);
        it.split = static_cast<int>(at - unsplit * p.splits);
        // (items are asked for in ascending order, as a rule: from where the last one was it is not far)
        const uint32_t group_items = static_cast<uint32_t>(total) * p.head_group;
        if (unsplit < group_first) group = group_first = 0, step = earlier = 0;
        while (unsplit - group_first >= group_items) group_first += group_items, ++group, step = earlier = 0;
        const uint32_t in_group = unsplit - group_first, heads = min(p.head_group, p.heads - static_cast<int>(group) * p.head_group);
        const int place = static_cast<int>(fast_div(in_group, static_cast<int>(heads) == p.head_group ? p.by_group : p.by_last_group));
        it.head = static_cast<int>(group * p.head_group + in_group - place * heads);
        Seq s;
        int block;
        if (p.n_seqs <= kLanes) {
            if (earlier > place) step = earlier = 0;
            for (;;) {
                const int here = up_to(step);
                if (here > place || step >= last_step) break;
                earlier = here;
                ++step;
            }
            uint32_t there = __ballot_sync(0xffffffffu, step >= behind && step < behind + blocks);
            for (int i = earlier; i < place; ++i) there &= there - 1;
            const int from = __ffs(there) - 1;
            const int i = step - behind;
            block = __shfl_sync(0xffffffffu, i < short_at ? blocks - 2 - i : i == short_at ? blocks - 1 : blocks - 1 - i, from);
            s = {__shfl_sync(0xffffffffu, mine.q0, from), __shfl_sync(0xffffffffu, mine.queries, from), __shfl_sync(0xffffffffu, mine.k0, from),
                 __shfl_sync(0xffffffffu, mine.keys, from)};
        } else {
            const int lane = threadIdx.x & 31;
            if (place < before) {
                chunk = before = 0;
                mine = load_seq(p, lane);
                blocks = blocks_of(mine.queries);
            }
            for (;;) {
                const int here = __reduce_add_sync(0xffffffffu, blocks);
                if (place < before + here || chunk + kLanes >= p.n_seqs) break;
                before += here;
                chunk += kLanes;
                mine = load_seq(p, chunk + lane);
                blocks = blocks_of(mine.queries);
            }
            int run = blocks;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int u = __shfl_up_sync(0xffffffffu, run, o);
                if (lane >= o) run += u;
            }
            const int from = __ffs(__ballot_sync(0xffffffffu, before + run > place)) - 1;
            block = __shfl_sync(0xffffffffu, run - 1, from) - (place - before);
            s = {__shfl_sync(0xffffffffu, mine.q0, from), __shfl_sync(0xffffffffu, mine.queries, from), __shfl_sync(0xffffffffu, mine.k0, from),
                 __shfl_sync(0xffffffffu, mine.keys, from)};
        }
        const int first = block * kBlock;
        it.q0 = s.q0 + first;
        it.rows = min(kBlock, s.queries - first);
        it.k0 = s.k0;
        it.len = s.keys;
        it.limit = p.causal ? s.keys - s.queries + first : s.keys - 1;
        it.alternate = it.rows <= kRows;
        const auto tiles_of_row = [&](int row) { return max(0, min(it.limit + (p.causal ? row : 0), s.keys - 1) + kTile) / kTile; };
        const int all = tiles_of_row(it.rows - 1);
        it.tile = static_cast<int>(fast_div(static_cast<uint32_t>(all) * it.split, p.by_splits));              // (2^24 tiles, 32 parts)
        const int end = static_cast<int>(fast_div(static_cast<uint32_t>(all) * (it.split + 1), p.by_splits));
        it.n = end - it.tile;
        if (it.alternate) {
            it.n0 = (it.n + 1) >> 1;
            it.n1 = it.n >> 1;
        } else {
            it.n0 = max(0, min(end, tiles_of_row(kRows - 1)) - it.tile);
            it.n1 = it.n;
        }
        it.edge = max(0, min(it.limit, s.keys - 1) + 1) / kTile;
        return it;
    }
};

// An item's units are loaded as the MMAs come to them: K0 K1 V0 K2 V1 ... V(n-1), or K0 K1 K2 V0 K3 V1 ... where tiles alternate.
// The slot of tile t's keys or values, from the item's first on.
__device__ __forceinline__ uint32_t unit_slot(bool alternate, int n, int t, bool keys) {
    const int ahead = min(alternate ? 2 * kAhead : kAhead, n);
    if (keys) return kKeySlots * t + (t >= ahead ? kValueSlots * (t - ahead) : 0);
    return kKeySlots * min(t + ahead + 1, n) + kValueSlots * t;
}

// ---------------------------------------------------------------- the kernel
template <int kCtas>
__global__ void __launch_bounds__(kThreads, 1)
expanded_attention_kernel(const __grid_constant__ CUtensorMap map_qn, const __grid_constant__ CUtensorMap map_qr, const __grid_constant__ CUtensorMap map_kn,
                          const __grid_constant__ CUtensorMap map_kr, const __grid_constant__ CUtensorMap map_v, const Params p, unsigned int* status) {
    using C = Cfg<kCtas>;
    constexpr int kSlots = C::kSlots, kSlotBytes = C::kSlotBytes, kRows = C::kRows;
    constexpr bool kPair = kCtas == 2;
    extern __shared__ __align__(1024) uint8_t smem[];
    Small& sm = *reinterpret_cast<Small*>(smem);
    Control* const ctl = &sm.ctl;
    const uint32_t ring = smem_u32(smem) + kSmallBytes, queries = ring + kRingBytes;
    const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    const auto bar = [](const uint64_t& b) { return smem_u32(&b); };
    // A pair's MMAs are the first CTA's: it waits for both, and both wait for it.
    const uint32_t rank = kPair ? cluster_ctarank() : 0u;
    const auto lead = [](const uint64_t& b) -> uint32_t { return kPair ? mapa_shared(smem_u32(&b), 0) : smem_u32(&b); };
    const auto arrive_lead = [&](const uint64_t& b) {
        if (kPair) mbar_arrive_cluster(lead(b));
        else mbar_arrive(bar(b));
    };
    const auto commit = [](const uint64_t& b) {                      // the MMAs so far, to all CTAs
        if (kPair) {
            tc_commit_pair(smem_u32(&b));
            tc_commit_pair(mapa_shared(smem_u32(&b), 1));
        } else {
            tc_commit(smem_u32(&b));
        }
    };

    griddep_launch_dependents();
    if (threadIdx.x == 0) {
        for (int i = 0; i < kUnits; ++i) {
            mbar_init(bar(sm.k_full[i]), 1);
            mbar_init(bar(sm.k_empty[i]), 1);
            mbar_init(bar(sm.v_full[i]), 1);
            mbar_init(bar(sm.v_ready[i]), kCtas);                    // (looked at)
            mbar_init(bar(sm.v_empty[i]), 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(bar(sm.q_full[i]), 1);
            mbar_init(bar(sm.q_empty[i]), 1);
            mbar_init(bar(sm.s_full[i]), 1);
            for (int j = 0; j < kValueSlots; ++j) mbar_init(bar(sm.p_full[i][j]), kCtas * kSoftmaxWarps / 2);
            mbar_init(bar(sm.p_empty[i]), 1);
            mbar_init(bar(sm.o_full[i]), 1);
            mbar_init(bar(sm.row_full[i]), kSoftmaxWarps / 2);
            mbar_init(bar(sm.row_empty[i]), kFinishWarps);
            mbar_init(bar(sm.o_empty[i]), kCtas * kFinishWarps);
        }
        for (int i = 0; i < kItemSlots; ++i) {
            mbar_init(bar(sm.item_full[i]), 1);
            mbar_init(bar(sm.item_empty[i]), kItemReaders);
        }
        mbar_init(bar(sm.s_empty), kCtas * kSoftmaxWarps / 2);
        mbar_init(bar(sm.taken), 1);
        mbar_init(bar(sm.seen), 1);
        for (int i = 0; i < kNotFiniteSlots; ++i) sm.not_finite[i] = 0x7FFFFFFF;
        mbar_fence_init();
        ctl->abort_flag = (ring & 1023u) != 0 ? 1u : 0u;             // (dynamic shared memory begins at a multiple of 1024; swizzled tiles rely on it)
        if (ctl->abort_flag && atomicCAS(&status[0], 0u, 1u) == 0u) status[1] = kRoom, status[2] = 0xFFFFFFFFu, status[3] = blockIdx.x;
    }
    if (warp == kScoreWarp) {
        if (kPair) tc_alloc_pair(smem_u32(&ctl->tmem_base), kTmemCols);
        else tc_alloc(smem_u32(&ctl->tmem_base), kTmemCols);
    }
    if (warp == kLoadWarp && lane == 0) {
        tma_prefetch_desc(&map_qn);
        tma_prefetch_desc(&map_qr);
        tma_prefetch_desc(&map_kn);
        tma_prefetch_desc(&map_kr);
        tma_prefetch_desc(&map_v);
    }
    griddep_wait();
    tc_fence_before();
    __syncthreads();
    if (kPair) {                                                     // (no signal before the other's barriers are set up)
        cluster_arrive();
        cluster_wait();
    }
    tc_fence_after();
    const uint32_t tmem = ctl->tmem_base;
    const bool well = ctl->abort_flag == 0;
    // Whole warp: the item in the next slot of the list's ring, or one without rows.
    const auto wait = [&](const uint64_t& b, uint32_t parity, uint32_t what, uint32_t count) -> bool {
        return __all_sync(0xffffffffu, mbar_try_wait(bar(b), parity)) || __all_sync(0xffffffffu, bounded_wait(bar(b), parity, ctl, status, what, count));
    };
    const auto next_item = [&](uint32_t count, bool& ok) -> Item {
        Item it = {};
        ok = __all_sync(0xffffffffu, bounded_wait_ns(bar(sm.item_full[count % kItemSlots]), (count / kItemSlots) & 1, ctl, status, kItems, count, kItemLimitNs));
        if (ok) it = sm.item[count % kItemSlots];
        return it;
    };
    // The same in all lanes, and known to be: branches and addresses that depend on it stay uniform, which the tensor core's instructions want (with addresses that were a lane's own, MMAs came half as
    // fast).
    const auto uniform = [](int x) -> int { return __shfl_sync(0xffffffffu, x, 0); };
    const auto item_done = [&](uint32_t count) {
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(sm.item_empty[count % kItemSlots]));
    };

    // (a pair's queries and keys arrive at the first CTA's barriers, values at the CTA's own)
    const auto copy = [&](uint32_t to, const CUtensorMap& map, int x, int head, int row, const uint64_t& full) {
        if (kPair) tma_load_3d_pair(to, &map, x, head, row, lead(full));
        else tma_load_3d(to, &map, x, head, row, bar(full));
    };

    // (in the branches of the roles themselves: behind a common point the compiler counts on the lesser of both numbers)
    if (!well) {
        // nothing is started
    } else if (warp >= kSoftmaxWarps) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
        if (warp == kLoadWarp) {
            // ------------------------------------------------------------ the list, and the loads of keys and values
            List<kCtas> list;
            list.begin(p);
            // (This warp sets the pace: an MMA's 64 cycles are what a few instructions take here.  A unit is armed and copied by one lane in one go.)
            uint32_t slot = 0, taken = 0;                            // slots filled; answers
            uint32_t freed = 0, back = 0, keys = 0, loaded = 0;      // slots and units given back; which of the last 32 units are keys; units
            uint32_t k_loaded = 0, v_loaded = 0, k_back = 0, v_back = 0;
            bool ok = true;
            int at = static_cast<int>(blockIdx.x) / kCtas;
            const auto one_back = [&]() {                            // the oldest unit on its way is given back
                const bool of_keys = keys >> (loaded - 1 - back) & 1;
                const uint32_t i = of_keys ? k_back++ : v_back++;
                ok = wait((of_keys ? sm.k_empty : sm.v_empty)[i % kUnits], (i / kUnits) & 1, kRoom, back);
                freed += of_keys ? kKeySlots : kValueSlots;
                ++back;
            };
            const auto room = [&](int slots) {
                while (ok && slot + slots - freed > kSlots) one_back();
            };
            // item number `at`, for the others to read
            uint32_t listed = 0;
            const auto publish = [&]() -> Item {
                const Item it = at < 0 ? Item{} : list.find(p, static_cast<uint32_t>(at));
                const uint32_t place = listed % kItemSlots;
                ok = ok && __all_sync(0xffffffffu, bounded_wait_ns(bar(sm.item_empty[place]), ((listed / kItemSlots) & 1) ^ 1, ctl, status, kItems, listed, kItemLimitNs));
                if (ok && lane == 0) {
                    sm.item[place] = it;
                    sm.not_finite[(listed + kNotFiniteSlots / 2) % kNotFiniteSlots] = 0x7FFFFFFF;      // (a pair's other CTA may be an item ahead)
                    mbar_arrive(bar(sm.item_full[place]));
                }
                __syncwarp();
                ++listed;
                return it;
            };
            // The next item is asked for as late as the loads allow: who asks early takes work that another SM would be free for.
            const auto ask = [&]() {
                if (p.dynamic && rank == 0 && elect_one()) {
                    mbar_arrive_expect_tx(bar(sm.taken), 16);
                    try_cancel(smem_u32(sm.answer), bar(sm.taken));
                }
                __syncwarp();
            };
            const auto answer = [&]() {
                if (!p.dynamic) {
                    const int step = static_cast<int>(gridDim.x) / kCtas;
                    at = at > 0x7FFFFFFF - step ? -1 : at + step;
                    return;
                }
                ok = ok && wait(sm.taken, taken & 1, kItems, taken);
                if (!ok) return;
                if (rank == 0) {
                    at = cancelled_cta(smem_u32(sm.answer));
                    if (at > 0) at /= kCtas;
                    fence_proxy_async_shared();
                    if (kPair) {
                        ok = wait(sm.seen, (taken & 1) ^ 1, kItems, taken);      // (the other one has read the answer before)
                        if (ok && lane == 0) {
                            store_cluster(mapa_shared(smem_u32(&sm.next_at), 1), at);
                            mbar_arrive_cluster_release(mapa_shared(bar(sm.taken), 1));
                        }
                    }
                } else {
                    fence_cluster();
                    at = *static_cast<volatile int*>(&sm.next_at);
                    __syncwarp();
                    if (lane == 0) mbar_arrive_cluster_release(lead(sm.seen));
                }
                ++taken;
                __syncwarp();
            };
            Item it = publish();
            while (ok && it.rows > 0) {
                Item following = {};
                if (it.n == 0) {
                    ask();
                    answer();
                    following = publish();
                }
                if (it.n > 0) {
                    const int head = uniform(it.head), n = uniform(it.n), ahead = uniform(it.alternate) != 0 ? 2 * kAhead : kAhead, row0 = uniform(it.k0 + it.tile * kTile);
                    const auto load_keys = [&](int t) {
                        const int row = row0 + t * kTile + static_cast<int>(rank) * (kTile / kCtas);
                        const uint64_t& there = sm.k_full[k_loaded % kUnits];
                        room(kKeySlots);
                        if (ok && elect_one()) {
                            if (rank == 0) mbar_arrive_expect_tx(bar(there), kCtas * kKeySlots * kSlotBytes);
                            copy(ring + slot % kSlots * kSlotBytes, map_kn, 0, head, row, there);
                            copy(ring + (slot + 1) % kSlots * kSlotBytes, map_kn, 64, head, row, there);
                            copy(ring + (slot + 2) % kSlots * kSlotBytes, map_kr, 0, 0, row, there);
                        }
                        __syncwarp();
                        keys = keys << 1 | 1u;
                        slot += kKeySlots;
                        ++k_loaded, ++loaded;
                    };
                    const auto load_values = [&](int t) {
                        const int row = row0 + t * kTile;
                        const uint64_t& there = sm.v_full[v_loaded % kUnits];
                        room(kValueSlots);
                        if (ok && elect_one()) {
                            mbar_arrive_expect_tx(bar(there), kValueSlots * kSlotBytes);
#pragma unroll
                            for (int i = 0; i < kValueSlots; ++i) {
                                const uint32_t to = ring + (slot + i) % kSlots * kSlotBytes;
                                tma_load_3d(to, &map_v, static_cast<int>(rank) * 64, head, row + i * 64, bar(there));
                                if (!kPair) tma_load_3d(to + kSlotBytes / 2, &map_v, 64, head, row + i * 64, bar(there));
                            }
                        }
                        __syncwarp();
                        keys <<= 1;
                        slot += kValueSlots;
                        ++v_loaded, ++loaded;
                    };
                    const int ask_at = max(-ahead, n - kAskEarly);
#pragma unroll 1
                    for (int t = -ahead; t < n && ok; ++t) {
                        if (t == ask_at) ask();
                        if (t + ahead < n) load_keys(t + ahead);
                        if (t >= 0) load_values(t);
                    }
                    // (the MMAs still have some tiles to go)
                    answer();
                    following = publish();
                }
                it = following;
            }
            // none of the arrivals on empty[] may be in flight when the CTA leaves its shared memory to another
            while (ok && back < loaded) one_back();
        } else if (warp == kScoreWarp) {
            // ------------------------------------------------------------ queries, and the MMAs of the scores.  Those of the sums have a warp of their own: an MMA takes 64 cycles, and what lies between
            // two groups of them (waits that need not wait, 100 cycles each; addresses) as long as several.  The warps stay converged and elect a lane for the MMAs alone.
            uint32_t slot = 0, keys = 0, active = 0, scored = 0;
            const uint64_t ring_desc = umma_desc_k_major_sw128(ring), query_desc = umma_desc_k_major_sw128(queries);
            bool ok = true;
            for (uint32_t count = 0; ok; ++count) {
                const Item it = next_item(count, ok);
                const int n = uniform(it.n), n0 = uniform(it.n0), step = uniform(it.alternate);
                if (!ok || uniform(it.rows) == 0) break;
                item_done(count);
                if (n == 0) continue;
                // (this warp has nothing to do before they are there, and the one that loads keys has)
                const int head = uniform(it.head), row0 = uniform(it.q0) + static_cast<int>(rank) * kHalf;
                for (int h = 0; h < 2; ++h) {
                    ok = ok && wait(sm.q_empty[h], (active & 1) ^ 1, kQueriesThere, active);
                    if (ok && elect_one()) {
                        if (h == 1 && step != 0) {
                            if (rank == 0) mbar_arrive(bar(sm.q_full[h]));              // (both halves use the first one's)
                        } else {
                            const uint32_t to = queries + h * kQueryBytes;
                            const int row = row0 + h * kRows;
                            if (rank == 0) mbar_arrive_expect_tx(bar(sm.q_full[h]), kCtas * kQueryBytes);
                            copy(to, map_qn, 0, head, row, sm.q_full[h]);
                            copy(to + kQueryPart, map_qn, 64, head, row, sm.q_full[h]);
                            copy(to + 2 * kQueryPart, map_qr, 0, head, row, sm.q_full[h]);
                        }
                    }
                    __syncwarp();
                }
                if (rank != 0) {
                    ++active;
                    continue;
                }
                for (int h = 0; h < 2; ++h) ok = ok && wait(sm.q_full[h], active & 1, kQueriesThere, active);
#pragma unroll 1
                for (int t = 0, u = 0; t < n && ok; ++t, ++keys) {
                    u = unit_slot(step != 0, n, t, true);
                    ok = wait(sm.k_full[keys % kUnits], (keys / kUnits) & 1, kTileThere, keys);
                    // both halves, the first one only where it sees the tile; or every other tile's
#pragma unroll 1
                    for (int h = step ? t & 1 : t < n0 ? 0 : 1, end = step ? h + 1 : 2; h < end && ok; ++h, ++scored) {
                        ok = wait(sm.s_empty, (scored & 1) ^ 1, kScoresRoom, scored);      // (the softmax has the scores before)
                        if (!ok) break;
                        tc_fence_after();
                        const uint64_t a = query_desc + (step ? 0 : h * (kQueryBytes >> 4));
                        if (elect_one()) {
#pragma unroll
                            for (int c = 0; c < kKeySlots; ++c) {
                                const uint64_t b = ring_desc + (slot + u + c) % kSlots * (kSlotBytes >> 4);
#pragma unroll
                                for (int k = 0; k < 4; ++k) {
                                    const uint64_t ak = a + c * (kQueryPart >> 4) + 2 * k;
                                    if (kPair) tc_mma_bf16_pair(tmem + kTmemScores, ak, b + 2 * k, C::kIdescScores, (c | k) != 0);
                                    else tc_mma_bf16(tmem + kTmemScores, ak, b + 2 * k, C::kIdescScores, (c | k) != 0);
                                }
                            }
                            commit(sm.s_full[h]);
                        }
                        __syncwarp();
                    }
                    if (elect_one()) {
                        commit(sm.k_empty[keys % kUnits]);
                        // (what is not needed any more: the first half may be done a tile before the second)
                        if (t == max(0, (step ? n : n0) - 1)) commit(sm.q_empty[0]);
                        if (t == n - 1) commit(sm.q_empty[1]);
                    }
                    __syncwarp();
                }
                slot += (kKeySlots + kValueSlots) * n;
                ++active;
            }
            for (int h = 0; h < 2 && ok && active > 0; ++h) ok = wait(sm.q_empty[h], (active - 1) & 1, kQueriesThere, active);
        } else if (warp == kSumWarp) {
            // ------------------------------------------------------------ the MMAs of the sums
            uint32_t slot = 0, values = 0, summed0 = 0, summed1 = 0;
            const uint64_t ring_desc = umma_desc_values(ring);
            bool ok = true;
            for (uint32_t count = 0; ok; ++count) {
                const Item it = next_item(count, ok);
                const int n = uniform(it.n), n0 = uniform(it.n0), n1 = uniform(it.n1), step = uniform(it.alternate);
                if (!ok || uniform(it.rows) == 0) break;
                item_done(count);
                if (rank != 0) continue;
                // (the sums of the item before are read: waited for, and the end signalled, with every item, so that neither side gets ahead of what parities tell)
                const auto sums_room = [&](int h) { ok = ok && wait(sm.o_empty[h], (count & 1) ^ 1, kSumsThere, count); };
                for (int h = 0; h < 2; ++h) {
                    if ((h == 0 ? n0 : n1) > 0) continue;
                    sums_room(h);
                    if (ok && elect_one()) commit(sm.o_full[h]);
                    __syncwarp();
                }
#pragma unroll 1
                for (int t = 0; t < n && ok; ++t, ++values) {
                    const uint32_t u = slot + unit_slot(step != 0, n, t, false);
                    ok = wait(sm.v_ready[values % kUnits], (values / kUnits) & 1, kGuarded, values);
#pragma unroll 1
                    for (int h = step ? t & 1 : t < n0 ? 0 : 1, end = step ? h + 1 : 2; h < end && ok; ++h) {
                        const uint32_t tile = h == 0 ? summed0 : summed1, d = tmem + kTmemSums + h * kValue, weights = tmem + kTmemWeights + h * (kTile / 2);
                        // (as the weights arrive: those of 64 keys, and then the others)
#pragma unroll
                        for (int i = 0; i < kValueSlots; ++i) {
                            const bool adds = t > step || i > 0;
                            if (!adds) sums_room(h);
                            ok = ok && wait(sm.p_full[h][i], tile & 1, kWeightsThere, tile);
                            if (!ok) break;
                            tc_fence_after();
                            const uint64_t b = ring_desc + (u + i) % kSlots * (kSlotBytes >> 4);
                            if (elect_one()) {
#pragma unroll
                                for (int k = 0; k < 4; ++k) {
                                    if (kPair) tc_mma_bf16_ts_pair(d, weights + (i * 4 + k) * 8, b + k * (16 * 128 >> 4), C::kIdescSums, adds || k != 0);
                                    else tc_mma_bf16_ts(d, weights + (i * 4 + k) * 8, b + k * (16 * 128 >> 4), C::kIdescSums, adds || k != 0);
                                }
                                if (i + 1 == kValueSlots) {
                                    commit(sm.p_empty[h]);
                                    if (t + step + 1 >= (step ? n : h == 0 ? n0 : n1)) commit(sm.o_full[h]);
                                }
                            }
                            __syncwarp();
                        }
                        h == 0 ? ++summed0 : ++summed1;
                    }
                    if (elect_one()) commit(sm.v_empty[values % kUnits]);
                    __syncwarp();
                }
                slot += (kKeySlots + kValueSlots) * n;
            }
        } else if (warp == kGuardWarp) {
            // ------------------------------------------------------------ values that the MMA must not see.  The warp passes all values on to the MMAs, and works on the tiles that are
            // not seen as a whole by all queries.
            uint8_t* const base = smem + kSmallBytes;
            uint32_t slot = 0, values = 0;
            bool ok = true;
            for (uint32_t count = 0; ok; ++count) {
                const Item it = next_item(count, ok);
                if (!ok || it.rows == 0) break;
                for (int t = 0; t < it.n; ++t, ++values) {
                    const bool look = it.tile + t >= it.edge;
                    ok = wait(sm.v_full[values % kUnits], (values / kUnits) & 1, kTileThere, values);
                    if (!ok) break;
                    const uint32_t u = slot + unit_slot(it.alternate, it.n, t, false);
                    for (int i = 0; i < kValueSlots && look; ++i) {
                        const int key0 = (it.tile + t) * kTile + i * 64;
                        uint4* const at = reinterpret_cast<uint4*>(base + (u + i) % kSlots * kSlotBytes);
                        // 64 keys x 8 pieces of 16 bytes, for either 64 dimensions; rows are keys, and a row's pieces stay in it
                        const __nv_bfloat162 zero = __floats2bfloat162_rn(0.0f, 0.0f);
                        __nv_bfloat162 seen[4] = {zero, zero, zero, zero};
                        if (key0 + 63 >= it.len) {
                            for (int j = 0; j < kSlotBytes / 512; ++j)
                                if (key0 + ((j * 32 + lane) >> 3 & 63) >= it.len) at[j * 32 + lane] = make_uint4(0u, 0u, 0u, 0u);
                        }
#pragma unroll 8
                        for (int j = 0; j < kSlotBytes / 512; ++j) {
                            const uint4 v = at[j * 32 + lane];
                            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                            for (int e = 0; e < 4; ++e) seen[e] = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&w[e]), zero, seen[e]);         // NaN stays
                        }
                        const __nv_bfloat162 all = __hadd2(__hadd2(seen[0], seen[1]), __hadd2(seen[2], seen[3]));
                        if (__any_sync(0xffffffffu, __hisnan(all.x) || __hisnan(all.y))) {
                            int bad = 0x7FFFFFFF;
                            for (int j = 0; j < kSlotBytes / 512; ++j) {
                                const int key = key0 + ((j * 32 + lane) >> 3 & 63);
                                const uint4 v = at[j * 32 + lane];
                                const uint32_t w[4] = {v.x, v.y, v.z, v.w};
                                bool finite = true;
#pragma unroll
                                for (int e = 0; e < 4; ++e) finite = finite && (w[e] & 0x7F80u) != 0x7F80u && (w[e] & 0x7F800000u) != 0x7F800000u;
                                if (!finite) {
                                    bad = min(bad, key);
                                    at[j * 32 + lane] = make_uint4(0u, 0u, 0u, 0u);
                                }
                            }
                            bad = __reduce_min_sync(0xffffffffu, bad);
                            if (lane == 0) {
                                int& worst = sm.not_finite[count % kNotFiniteSlots];
                                atomicMin(&worst, bad);
                                if (kPair) {
                                    min_cluster(mapa_shared(smem_u32(&worst), rank ^ 1u), bad);
                                    fence_cluster();
                                }
                            }
                        }
                    }
                    if (look) fence_proxy_async_shared();
                    __syncwarp();
                    if (lane == 0) arrive_lead(sm.v_ready[values % kUnits]);
                }
                slot += (kKeySlots + kValueSlots) * it.n;
                item_done(count);
            }
        } else if (warp >= kFinishWarp) {
            // ------------------------------------------------------------ results: sums divided and written, while the softmax goes on with the next item.  (By the softmax' own warps:
            // 4000 cycles an item that they did not work.)
            const int quarter = warp - kFinishWarp;
            const uint32_t sums_at = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + kTmemSums;
            const float c = p.scale;
            bool ok = true;
            for (uint32_t count = 0; ok; ++count) {
                const Item it = next_item(count, ok);
                if (!ok || it.rows == 0) break;
                const int& not_finite = sm.not_finite[count % kNotFiniteSlots];
                const auto half_there = [&](int h) {
                    ok = ok && wait(sm.row_full[h], count & 1, kSumsThere, count) && wait(sm.o_full[h], count & 1, kSumsThere, count);
                };
                const auto half_done = [&](int h) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) {
                        mbar_arrive(bar(sm.row_empty[h]));
                        arrive_lead(sm.o_empty[h]);
                    }
                };
#pragma unroll 1
                for (int h = 0; h < (it.alternate ? 1 : 2) && ok; ++h) {
                    half_there(h);
                    if (it.alternate) half_there(1);
                    if (!ok) break;
                    tc_fence_after();
                    const int row0 = h * kRows + static_cast<int>(rank) * kHalf + quarter * 32, row = row0 + lane;
                    float2 stats = sm.row[h][quarter * 32 + lane];   // reference and sum
                    float f = 1.0f, other = 0.0f;                    // factors of the half's sums, and of the other one's
                    if (it.alternate) {
                        const float2 theirs = sm.row[1][quarter * 32 + lane];
                        const float both = fmaxf(stats.x, theirs.x), ref = both == -INFINITY ? 0.0f : both;
                        f = ex2((stats.x - ref) * c);
                        other = ex2((theirs.x - ref) * c);
                        stats = make_float2(both, stats.y * f + theirs.y * other);
                    }
                    const int last = min(it.limit + (p.causal ? row : 0), it.len - 1);
                    const bool nothing = stats.x == -INFINITY && !isnan(stats.y);
                    const bool spoilt = last >= *static_cast<const volatile int*>(&not_finite);
                    const float inv = spoilt ? __uint_as_float(0x7FC00000u) : nothing ? 0.0f : rcp(stats.y);
                    const float2 f2 = make_float2(f * inv, f * inv), other2 = make_float2(other * inv, other * inv), zero2 = make_float2(0.0f, 0.0f);
                    const int64_t place = static_cast<int64_t>(it.q0 + row0) * p.heads + it.head, part = static_cast<int64_t>(it.split) * p.tokens * p.heads + place;
                    const int rows = it.rows - row0;
                    const int n = h == 0 ? it.n0 : it.n1;
                    const bool two = it.alternate && it.n1 > 0;
#pragma unroll 1
                    for (int i = 0; i < kValue; i += 16) {
                        uint32_t o[16] = {}, o2[16] = {};
                        if (n > 0) tc_ld_x16(sums_at + h * kValue + i, o);
                        if (two) tc_ld_x16(sums_at + kValue + i, o2);
                        tc_wait_ld();
#pragma unroll
                        for (int j = 0; j < 16; j += 2) {
                            float2 v = fma2(make_float2(__uint_as_float(o[j]), __uint_as_float(o[j + 1])), f2, zero2);
                            if (two) v = fma2(make_float2(__uint_as_float(o2[j]), __uint_as_float(o2[j + 1])), other2, v);
                            o[j] = __float_as_uint(v.x), o[j + 1] = __float_as_uint(v.y);
                        }
                        if (p.partial) {
                            store_rows(o, p.partial + part * kValue + i, static_cast<int64_t>(p.heads) * kValue * 4, rows);
                        } else {
                            uint32_t w[8];
#pragma unroll
                            for (int j = 0; j < 8; ++j) w[j] = pack_bf16x2(__uint_as_float(o[2 * j]), __uint_as_float(o[2 * j + 1]));
                            store_rows(w, p.out + place * kValue + i, static_cast<int64_t>(p.heads) * kValue * 2, rows);
                        }
                        __syncwarp();
                    }
                    half_done(h);
                    if (it.alternate) half_done(1);
                    if (lane < rows) {
                        const float lse = nothing ? -INFINITY : (stats.x * c + log2f(stats.y)) * kLn2;
                        if (p.partial) p.partial_lse[part + static_cast<int64_t>(lane) * p.heads] = lse;
                        else if (p.lse) p.lse[place + static_cast<int64_t>(lane) * p.heads] = lse;
                    }
                }
                item_done(count);
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
        // ------------------------------------------------------------ softmax: a thread to a query
        const int h = warp >> 2, quarter = warp & 3;
        const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16, scores_at = tmem + lanes + kTmemScores, weights_at = tmem + lanes + kTmemWeights + h * (kTile / 2);
        const float c = p.scale;
        uint32_t tiles = 0;
        bool ok = true;
        for (uint32_t count = 0; ok; ++count) {
            const Item it = next_item(count, ok);
            if (!ok || it.rows == 0) break;
            const int n = h == 0 ? it.n0 : it.n1, row0 = (it.alternate ? 0 : h * kRows) + static_cast<int>(rank) * kHalf + quarter * 32, row = row0 + lane;
            const int last = min(it.limit + (p.causal ? row : 0), it.len - 1);           // key that the query sees last
            const int last0 = min(it.limit + (p.causal ? row0 : 0), it.len - 1);         // ... of the warp's first one
            float top = -INFINITY;
            float2 sum2 = make_float2(0.0f, 0.0f);
            for (int t = 0; t < n; ++t, ++tiles) {
                const int key0 = (it.tile + (it.alternate ? 2 * t + h : t)) * kTile;
                ok = wait(sm.s_full[h], tiles & 1, kScoresThere, tiles);
                if (!ok) break;
                tc_fence_after();
                // the last column that is the query's, the last that is all the warp's
                const int visible = last - key0, visible0 = last0 - key0;
                uint32_t x[kTile];
#pragma unroll
                for (int i = 0; i < kTile; i += 32) tc_ld_x32(scores_at + i, x + i);
                tc_wait_ld();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) arrive_lead(sm.s_empty);
                if (visible0 < kTile - 1) {
#pragma unroll
                    for (int i = 0; i < kTile; ++i) x[i] = i > visible ? 0xFF800000u : x[i];
                }
                float m[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) m[i] = max3(__uint_as_float(x[i]), __uint_as_float(x[i + 4]), __uint_as_float(x[i + 8]));
#pragma unroll
                for (int i = 12; i < kTile - 4; i += 8) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) m[j] = max3(m[j], __uint_as_float(x[i + j]), __uint_as_float(x[i + j + 4]));
                }
                static_assert((kTile - 16) % 8 == 0, "four columns are left");
#pragma unroll
                for (int j = 0; j < 4; ++j) m[j] = max3(m[j], __uint_as_float(x[kTile - 4 + j]), -INFINITY);
                const float most = max3(max3(m[0], m[1], m[2]), m[3], -INFINITY);
                // (the sums of the tile before are complete: weights may be overwritten, sums rescaled)
                ok = wait(sm.p_empty[h], (tiles & 1) ^ 1, kWeightsRoom, tiles);
                if (!ok) break;
                tc_fence_after();
                // a weight would pass 2^kSlack, nothing was seen so far, or something is not a number: the reference moves
                const bool moves = !(most * c <= top * c + kSlack);
                if (t == 0) {
                    top = most;
                } else if (__any_sync(0xffffffffu, moves)) {
                    const float f = moves ? (top == -INFINITY ? 0.0f : ex2((top - most) * c)) : 1.0f;
                    if (moves) top = most;
                    sum2.x *= f, sum2.y *= f;
#pragma unroll 1
                    for (int i = 0; i < kValue; i += 32) {
                        uint32_t o[32];
                        const uint32_t at = tmem + lanes + kTmemSums + h * kValue + i;
                        tc_ld_x32(at, o);
                        tc_wait_ld();
#pragma unroll
                        for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * f);
                        tc_st_x32(at, o);
                    }
                }
                const float ref = top == -INFINITY ? 0.0f : -top * c;
                const float2 c2 = make_float2(c, c), ref2 = make_float2(ref, ref);
#pragma unroll
                for (int first = 0; first < kTile; first += 32) {
                    uint32_t w[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const float2 y = fma2(make_float2(__uint_as_float(x[first + 2 * i]), __uint_as_float(x[first + 2 * i + 1])), c2, ref2);
                        const float2 e = make_float2(ex2(y.x), ex2(y.y));
                        sum2 = add2(sum2, e);
                        w[i] = pack_bf16x2(e.x, e.y);
                    }
                    tc_st_x16(weights_at + first / 2, w);
                    if (first & 32) {
                        tc_wait_st();
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) arrive_lead(sm.p_full[h][first >> 6]);
                    }
                }
            }
            if (!ok) break;
            ok = wait(sm.row_empty[h], (count & 1) ^ 1, kRowsRoom, count);
            if (!ok) break;
            sm.row[h][quarter * 32 + lane] = make_float2(top, sum2.x + sum2.y);
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(sm.row_full[h]));
            item_done(count);
        }
        // (none of the signals of the MMAs may be on its way when the CTA leaves its shared memory to another)
        if (ok && tiles > 0) wait(sm.p_empty[h], (tiles - 1) & 1, kWeightsRoom, tiles);
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
    if (kPair) {                                                     // (no signal is on its way to a CTA that has gone)
        cluster_arrive();
        cluster_wait();
    }
    if (warp == kScoreWarp) {
        tc_fence_after();
        if (kPair) tc_dealloc_pair(tmem, kTmemCols);
        else tc_dealloc(tmem, kTmemCols);
    }
}

// How a call is cut up: whether CTAs work in pairs, and in how many parts the keys of a block of queries are cut.  What is known on the host is how many queries, keys and sequences there are, not
// which sequence has how many.
struct Plan {
    int ctas;                             // to a block of queries
    int64_t blocks;                       // at most
    int splits, head_group;
};
constexpr int kLeastTiles = 4;            // of a part
constexpr int64_t kGroupBytes = 32ll << 20;
struct Call {
    int64_t tokens, kv_tokens, heads, n_seqs;
    bool ragged, causal;
};
// How long a plan takes, in times that half a block of a CTA alone takes for a tile (1.03 us): what there is to do, spread over all SMs, or its longest item; where all items are about as long, as many
// rounds of them as there are.  A pair's tile takes 0.807 of that, an item's begin and end as long as 2.5 of its half's tiles (of a pair's 4.5), a join 5.9 and 56 more for a million partial rows.
// Fitted to 78 calls of 1 to 16001 queries and 37 to 16384 keys, alone and in pairs, 26 of them in up to 12 parts.  Held against either kind of CTAs and up to 32 parts of 45 calls it picks the fastest, or one at
// most 4 % slower, for 35 of them; farthest off are 768 queries of 16 heads over themselves (alone 18.2 us, in pairs 15.1), 3000 of 5 heads (four parts alone 34.8, three in pairs 29.6), 64 of 16 heads over 8192 keys (nine
// parts 25.0, eight 22.4) and 200 of 16 heads over themselves (10.2, in pairs 9.3).
//   Parts of 2, 3 and 4: 515 queries of 16 heads over 4099 keys 45.2, 36.5 and 41.5 us; 512 over 8192 in pairs 65.9, 51.5 and 44.6; 2 heads of 16001 tokens in pairs 121, 130 and 133, and 195 in one.
// Alone / in pairs: 512 queries of 128 heads over 512 keys 24.0 / 28.9 us, over 2048 79.4 / 70.6, over 8192 298 / 250; 1000 of 16 over 8000 78.7 / 69.3; 16001 of 16 over themselves 942 / 836.
struct Work {
    double queries, longest, tiles;       // of a sequence: queries, tiles of keys, those that a query sees
    double alike;                         // 1: items are as long, 0: of all lengths up to the longest
    double heads, rows;                   // of all sequences
};
double time_of(const Work& w, int ctas, int splits, int sms) {
    const double slots = sms / ctas, a_tile = ctas == 2 ? 0.807 : 1.0, ends = ctas == 2 ? 4.5 : 2.5;
    const double halves = std::ceil(w.queries / (ctas * kHalf)), items = w.heads * std::max(1.0, halves / 2) * splits;
    const double all = w.heads * halves * (w.tiles + ends * splits) / slots, one = std::min(2.0, halves) * (w.longest / splits + ends);
    const double time = std::max({all, one, all + (std::ceil(items / slots) * one - all) * w.alike});
    return a_tile * time + (splits > 1 ? 5.9 + 56e-6 * splits * w.rows : 0.0);
}
Plan plan_of(const Call& c, int sms) {
    Work w;
    const double keys = static_cast<double>(c.kv_tokens) / c.n_seqs;                 // (if all sequences have as many)
    w.queries = std::max(1.0, static_cast<double>(c.tokens) / c.n_seqs);
    w.longest = keys / kTile;
    w.tiles = (c.causal ? keys > w.queries ? keys - w.queries / 2 : keys / 2 : keys) / kTile + (c.causal ? 0.5 : 0.0);
    w.alike = std::pow(std::max(0.0, std::min(1.0, 2 * w.tiles / w.longest - 1)), 0.75);
    w.heads = static_cast<double>(c.heads) * c.n_seqs;
    w.rows = static_cast<double>(c.tokens) * c.heads;
    const int64_t most = (c.kv_tokens / c.n_seqs + kTile - 1) / kTile;
    const int last = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(kMaxJoinParts, most / kLeastTiles)));
    Plan pl = {1, 0, 1, 0};
    double best = time_of(w, 1, 1, sms);
    // (blocks of a pair that are not half full gain nothing: 64 queries of 128 heads over 4000 keys 55.9 us alone, 75.3 in pairs)
    for (int ctas = 1; ctas <= (sms > 1 && c.tokens / c.n_seqs >= 2 * kHalf ? 2 : 1); ++ctas)
        for (int splits = 1; splits <= last && (splits == 1 || w.heads * splits <= 8.0 * sms); ++splits) {          // (more than some rounds of items gain nothing)
            const double time = time_of(w, ctas, splits, sms) * (ctas == 2 ? 1.04 : 1.0);        // (what is as good is not worth a pair)
            if (time < best) best = time, pl.ctas = ctas, pl.splits = splits;
        }
    const int64_t each = c.ragged ? 0 : c.tokens / c.n_seqs, rows = pl.ctas * 2 * kHalf, seqs = std::min(c.n_seqs, c.tokens);      // (that have queries)
    pl.blocks = c.ragged ? (c.tokens - seqs) / rows + seqs : c.n_seqs * ((each + rows - 1) / rows);
    // Groups of heads, equal ones: as few as keep a group's keys and values in the L2, and no more than leave each of them an item to an SM (or pair).  In long rows of calls, in groups of 16 MB, 32, 64 or all
    // heads at once: 4096 tokens of 128 heads 607, 606, 622 and 675 us; 16001 of 16 heads, which then are too few to a group, 1050, 980, 1005 and 1004; 515 of 128 heads over 4099 keys 221, 221, 221
    // and 234 (with two items to an SM at least, 233 for 32 MB).
    //   Two items where lengths may differ: the longest come first within a group only, so that a group with few of them ends with SMs that wait, the last one above all.  Seven prompts of 16 heads, 70 to 2050 queries
    // over up to 4610 keys, 130 us with two and 154 with one; eleven of 32 heads, one of them of 4000 tokens, 198 and 218; four of 64 heads 214 and 229; three of 24 heads 181 and 195.  The other way round 800 and
    // 3000 queries of 32 heads 345 and 335; three times 1024 of 128 heads over 3000 keys 505 and 492; 600, 70 and 1200 of 128 heads 282 and 275.  Of 21 batches 6 gain 3 to 16 %, 4 lose 2 to 3 %, 11 stay.
    const int64_t bytes = c.heads * c.kv_tokens * 2 * (kNope + kValue);
    const int64_t groups = c.n_seqs > kLanes ? 1 : std::max<int64_t>(1, std::min(bytes / kGroupBytes, pl.blocks * c.heads / ((c.ragged && c.n_seqs > 1 ? 2 : 1) * std::max(1, sms / pl.ctas))));
    pl.head_group = static_cast<int>((c.heads + groups - 1) / groups);
    return pl;
}
size_t partial_bytes(const Plan& pl, int64_t tokens, int64_t heads) {
    return pl.splits > 1 ? static_cast<size_t>(pl.splits) * tokens * heads * (kValue + 1) * sizeof(float) : 0;
}

template <int kCtas>
int prepare_kernel() {
    static std::atomic<uint64_t> prepared{0};                        // devices
    int device = 0;
    DSV3_CUDA_TRY(cudaGetDevice(&device));
    if (device >= 64 || !(prepared.load(std::memory_order_relaxed) >> device & 1)) {
        DSV3_CUDA_TRY(cudaFuncSetAttribute(expanded_attention_kernel<kCtas>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes));
        // (the warps that ask for more registers wait for those that the block does not have)
        cudaFuncAttributes attr = {};
        DSV3_CUDA_TRY(cudaFuncGetAttributes(&attr, expanded_attention_kernel<kCtas>));
        if (attr.numRegs * kThreads < kSoftmaxRegs * 256 + kOtherRegs * 256) {
            set_last_error("expanded_attention: built with %d registers a thread, too few to share out", attr.numRegs);
            return DSV3_ERR_UNSUPPORTED;
        }
        if (device < 64) prepared.fetch_or(1ull << device, std::memory_order_relaxed);
    }
    return DSV3_OK;
}

template <int kCtas>
int launch(const CUtensorMap& qn, const CUtensorMap& qr, const CUtensorMap& kn, const CUtensorMap& kr, const CUtensorMap& v, const Params& p, int64_t items, unsigned int* status,
           cudaStream_t stream) {
    if (const int rc = prepare_kernel<kCtas>(); rc != DSV3_OK) return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(items * kCtas));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = kSmemBytes;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    int n = 0;
    if (kCtas > 1) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = kCtas, attr[n].val.clusterDim.y = 1, attr[n].val.clusterDim.z = 1;
        ++n;
    }
    if (pdl_enabled()) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n].val.programmaticStreamSerializationAllowed = 1;
        ++n;
    }
    cfg.attrs = attr;
    cfg.numAttrs = n;
    DSV3_CUDA_TRY(cudaLaunchKernelEx(&cfg, expanded_attention_kernel<kCtas>, qn, qr, kn, kr, v, p, status));
    return DSV3_OK;
}

}  // namespace
}  // namespace dsv3

using namespace dsv3;

extern "C" {

size_t dsv3_expanded_attention_workspace_bytes(int64_t tokens, int64_t kv_tokens, int heads, int n_seqs, int ragged, int causal) {
    if (tokens <= 0 || kv_tokens <= 0 || heads <= 0 || n_seqs <= 0) return 0;
    return partial_bytes(plan_of({tokens, kv_tokens, heads, n_seqs, ragged != 0, causal != 0}, device_sms()), tokens, heads);
}

int dsv3_expanded_attention(const dsv3_expanded_attention_t* a, void* workspace, size_t workspace_bytes, dsv3_stream_t stream) {
    if (!a || a->tokens < 0 || a->kv_tokens < 0 || a->heads < 0 || a->n_seqs < 0) {
        set_last_error("expanded_attention: no arguments, or a negative size");
        return DSV3_ERR_INVALID_ARGUMENT;
    }
    if (a->tokens == 0 || a->heads == 0) return DSV3_OK;
    if (!a->q_nope || !a->q_rope || !a->out || (a->kv_tokens > 0 && (!a->k_nope || !a->k_rope || !a->v))) {
        set_last_error("expanded_attention: null pointer");
        return DSV3_ERR_INVALID_ARGUMENT;
    }
    const bool ragged = a->cu_seqlens_q != nullptr;
    if (a->n_seqs == 0 || (!ragged && a->tokens % a->n_seqs != 0) || (!a->cu_seqlens_k && a->kv_tokens % a->n_seqs != 0)) {
        set_last_error("expanded_attention: %lld queries or %lld keys do not divide among %d sequences", static_cast<long long>(a->tokens),
                       static_cast<long long>(a->kv_tokens), a->n_seqs);
        return DSV3_ERR_INVALID_ARGUMENT;
    }
    if (!(a->softmax_scale > 0.0f) || a->softmax_scale > 1e30f) {
        set_last_error("expanded_attention: softmax_scale must be positive and finite");
        return DSV3_ERR_INVALID_ARGUMENT;
    }
    const int64_t strides = a->q_nope_token_stride | a->q_nope_head_stride | a->q_rope_token_stride | a->q_rope_head_stride | a->k_nope_token_stride |
                            a->k_nope_head_stride | a->k_rope_token_stride | a->v_token_stride | a->v_head_stride;
    const uintptr_t pointers = reinterpret_cast<uintptr_t>(a->q_nope) | reinterpret_cast<uintptr_t>(a->q_rope) | reinterpret_cast<uintptr_t>(a->out) |
                               (a->kv_tokens > 0 ? reinterpret_cast<uintptr_t>(a->k_nope) | reinterpret_cast<uintptr_t>(a->k_rope) | reinterpret_cast<uintptr_t>(a->v) : 0);
    if (strides % 8 != 0 || strides < 0 || pointers % 16 != 0) {
        set_last_error("expanded_attention: rows of queries, keys, values and out must be 16-byte aligned, strides not negative");
        return DSV3_ERR_UNSUPPORTED;
    }
    const int sms = device_sms();
    const Plan pl = plan_of({a->tokens, std::max<int64_t>(1, a->kv_tokens), a->heads, a->n_seqs, ragged, a->causal != 0}, sms);
    if (a->heads > 1024 || a->tokens > 0x7FFFFF00ll || a->kv_tokens > 0x7FFFFF00ll || pl.blocks * a->heads * pl.splits > 0x3FFFFFFFll) {
        set_last_error("expanded_attention: more than 1024 heads, or 2^31 queries, keys or blocks of queries");
        return DSV3_ERR_UNSUPPORTED;
    }
    const size_t need = partial_bytes(pl, a->tokens, a->heads);
    if (need && (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 16 != 0)) {
        set_last_error("expanded_attention: the workspace must be 16-byte aligned and hold %zu bytes", need);
        return DSV3_ERR_WORKSPACE;
    }
    unsigned int* const status = status_device_ptr();
    if (!status) return DSV3_ERR_CUDA;
    CUtensorMap qn, qr, kn, kr, v;
    // (without keys nothing is loaded; the maps then describe the queries)
    const bool keys = a->kv_tokens > 0;
    int rc;
    if ((rc = make_tmap_heads(&qn, a->q_nope, kNope, a->heads, a->tokens, a->q_nope_head_stride, a->q_nope_token_stride, kHalf)) != DSV3_OK) return rc;
    if ((rc = make_tmap_heads(&qr, a->q_rope, kRope, a->heads, a->tokens, a->q_rope_head_stride, a->q_rope_token_stride, kHalf)) != DSV3_OK) return rc;
    if (!keys) {
        kn = v = qn;
        kr = qr;
    } else {
        if ((rc = make_tmap_heads(&kn, a->k_nope, kNope, a->heads, a->kv_tokens, a->k_nope_head_stride, a->k_nope_token_stride, kTile / pl.ctas)) != DSV3_OK) return rc;
        if ((rc = make_tmap_heads(&kr, a->k_rope, kRope, 1, a->kv_tokens, 0, a->k_rope_token_stride, kTile / pl.ctas)) != DSV3_OK) return rc;
        if ((rc = make_tmap_heads(&v, a->v, kValue, a->heads, a->kv_tokens, a->v_head_stride, a->v_token_stride, kTile / 2)) != DSV3_OK) return rc;
    }
    const int64_t items = pl.blocks * a->heads * pl.splits, rows = a->tokens * a->heads;
    // A CTA takes the place of one that has not started, so that no SM waits while there is work; with a budget of SMs, whose rest is not to be touched, CTAs take turns
    const bool dynamic = !sm_budget_set();
    float* const partial = need ? static_cast<float*>(workspace) : nullptr;
    Params p = {};
    p.tokens = static_cast<int>(a->tokens), p.kv_tokens = static_cast<int>(a->kv_tokens), p.heads = a->heads, p.n_seqs = a->n_seqs;
    p.cu_q = a->cu_seqlens_q, p.cu_k = a->cu_seqlens_k;
    p.per_q = ragged ? 0 : static_cast<int>(a->tokens / a->n_seqs), p.per_k = a->cu_seqlens_k ? 0 : static_cast<int>(a->kv_tokens / a->n_seqs);
    p.causal = a->causal != 0;
    p.scale = a->softmax_scale * kLog2e;
    p.head_group = pl.head_group, p.splits = pl.splits, p.blocks = static_cast<int>(pl.blocks), p.dynamic = dynamic;
    p.by_splits = make_fast_div(pl.splits), p.by_group = make_fast_div(pl.head_group);
    p.by_last_group = make_fast_div(a->heads % pl.head_group ? a->heads % pl.head_group : pl.head_group);
    p.out = static_cast<__nv_bfloat16*>(a->out), p.lse = a->lse;
    p.partial = partial, p.partial_lse = need ? partial + pl.splits * rows * kValue : nullptr;
    const int64_t grid = dynamic ? items : std::min<int64_t>(items, std::max(1, num_sms() / pl.ctas));
    const auto go = pl.ctas == 2 ? launch<2> : launch<1>;
    if (rc = go(qn, qr, kn, kr, v, p, grid, status, static_cast<cudaStream_t>(stream)); rc != DSV3_OK) return rc;
    if (!need) return DSV3_OK;
    return join_partials(partial, p.partial_lse, pl.splits, rows, kValue, p.cu_q, a->n_seqs, a->heads, a->out, a->lse, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
