// Attention over a paged KV cache for many rows per sequence (prompts, the shared prefix of a batch; D 64, 128) on the 5th-generation
// tensor cores. Arguments, rows and the line of work: paged.cuh; launchers: paged_attn.cu.
//
// A CTA (one per SM) takes row tiles of 256 rows, two groups of 128, and walks key tiles of 64 for both (f16 results; for 32-bit ones, EXACT,
// below, one group of 128 rows):
//   warps 0-3, 4-7   softmax of group 0 and 1, a row per thread: read 64 scores from tensor memory, online softmax to base 2, write P
//                    over the scores as f16, and what that rounding left beside it, so that a result has the 32 bits that it is computed in
//                    until it is rounded itself (without the remainder an f16 one is off by 1.25 to 1.4 times what its own rounding leaves,
//                    and a prompt of 8192 takes 640 us instead of 810). The accumulator is rescaled only when a row's maximum has
//                    grown by more than 2^kGrowth since its last rescale, as attention kernels for this chip are known to do. They
//                    write the piece's results.
//   warps 8, 9       issue the MMAs of group 0 and 1: S = Q K^T (both in shared memory), O += P V (P in tensor memory, V MN-major). Each
//                    group has two S / P tiles; P V of key tile j and S of tile j + 2, which takes its place, leave together, so that a
//                    group's softmax finds the next scores there while the tensor core works on the other's. A warp per group, and the
//                    MMAs of a whole tile behind one elected lane: what a warp does around its MMAs takes longer than the MMAs (one
//                    warp for both groups, an elected lane per MMA: 1240 clocks per group and tile, 640 of them the tensor core's)
//   warp 10          streams K and V tiles with TMA, a box of 64 columns x one page each, K two tiles ahead of V
//   warp 11          brings the Q rows in, those of the next piece as soon as the last S of this one has read them
// Tensor memory: four S / P tiles of 64 columns, two O of D. Key tiles that no row of a group sees are left out for it, and of a tile the
// steps of 16 keys that none sees; V rows behind the last key are zeroed before they are multiplied (a page holds anything there).
// The tensor core's sums are cut rather than rounded: 7e-9 of a sum per MMA, whatever it is small against, and always downwards. An f16 result
// (its rounding leaves 2.1e-4) shows that from some ten thousand keys on (131072 keys in one accumulator, values around 1: 6.8e-4, 500000: 2.3e-3).
// So an accumulator takes kRenew tiles, 8192 keys; then the group's softmax warps add it to their piece's slot in the scratch, and it
// begins anew (4e-5 at most; 12 us each time for both groups, 4 % of the 30001 keys below).
// EXACT. A 32-bit result shows it at once (2.2e-6 after 300 MMAs): two accumulators take kFlush tiles each in turn and are added to a sum in
// registers (7.8e-7). This form writes f16 results, too, where the scratch holds no slot and there may be more than kRenew tiles. Warps
// 0-3 and 4-7 are two threads per row, each with half of a tile's keys and half of the columns, who exchange the row's maximum; warp 9
// loads, warp 10 brings Q, warp 11 is idle. 24 mixed sequences, 512 new tokens in one: 115 us, 126 with a thread per row.
// Bound by what the softmax warps do one after another in a tile (exponentials and conversions 770 clocks, maximum 220, waiting for scores
// 280; without the remainder) and the tensor core's P V of it: a prompt of 8192, 32 heads of 128 over 8: 810-830 us, 670 TFLOP/s of the 1655 that the
// library's product reaches (1408 sustained); 1080 tokens behind 30001 keys: 910-930 us. 1.7e4 clocks pass before a launch's second tile: the line of
// work 3400, finding the first piece 5500, the first scores 1500, the first tile 7500, most of it instructions fetched for the first time.
// Every wait on a barrier is bounded (paged.cuh). The warps that ask for copies and issue MMAs leave when these are done, in a CTA that gives
// up, too; then its tensor memory is freed.
#include <cstring>

#include "paged.h"
#include "sync_ptx.cuh"
#include "tcgen05_ptx.cuh"

namespace amv {
namespace paged {

using namespace ptx;
using namespace tc;

constexpr uint32_t kGroupRows = 128, kBadRing = 8;
// Registers a thread after the split: 256 x 200 + 128 x 104 = 384 x 168, what the block is launched with.
constexpr uint32_t kSoftmaxRegs = 200, kOtherRegs = 104;
constexpr float kGrowth = 7.0f;   // probabilities stay below 2^7

template <int D, bool EXACT>
struct Tc {
    static constexpr uint32_t GROUPS = EXACT ? 1 : 2, ROWS = GROUPS * kGroupRows;
    static constexpr uint32_t PARTS = EXACT ? 2 : 1, KEYS = kTcKeys / PARTS, COLS = D / PARTS;   // threads of a row; a thread's share of keys and columns
    static constexpr uint32_t MMA = 8, LOAD = MMA + GROUPS, QWARP = LOAD + 1, THREADS = 384;      // warps by role
    static constexpr uint32_t TMEM = EXACT && D == 64 ? 256 : 512;
    static constexpr uint32_t A = D / 64, STAGES = D == 64 ? 5 : EXACT ? 4 : 3;
    static constexpr uint32_t Q = A * kGroupRows * 128u, TILE = A * kTcKeys * 128u;
    static constexpr uint32_t STAGE_OUT = MMA * 32u * 64u;   // a warp's 32 rows x 16 columns on their way out
    static constexpr uint32_t PAIRS = EXACT ? 2u * 2u * kGroupRows * 8u : 0u;   // what the threads of a row tell one another
    static constexpr uint32_t FIXED = 1024u + GROUPS * Q + 2u * STAGES * TILE + STAGE_OUT + PAIRS + 512u;
    static constexpr uint32_t smem(uint32_t n_seqs) { return FIXED + (n_seqs + 1u) * 4u; }
};
constexpr uint32_t kFlush = 4;     // EXACT: key tiles that an accumulator takes before it is added to the row's sum

__device__ __forceinline__ void tma_box(uint32_t dst, const CUtensorMap* map, uint32_t bar, int column, int token, int head, int page) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst), "l"(map),
        "r"(bar), "r"(column), "r"(token), "r"(head), "r"(page)
        : "memory");
}
__device__ __forceinline__ void tmem_st16_async(uint32_t taddr, const uint32_t* v) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr), "r"(v[0]),
        "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]),
        "r"(v[14]), "r"(v[15])
        : "memory");
}
// two f32 in one register pair: one instruction for both
__device__ __forceinline__ uint64_t pack2(float x, float y) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ float2 unpack2(uint64_t v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
// The MMAs and commits of a converged warp, issued by one lane, the same every time, without a branch around them: what a branch that
// only one lane takes computes is not uniform to the compiler, and every descriptor then takes a detour of some 100 clocks.
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\telect.sync _|q, 0xffffffff;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}
__device__ __forceinline__ void commit(uint32_t bar) {
    asm volatile(
        "{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar)
        : "memory");
}
// The MMAs of a whole tile and the commits behind them, one lane elected once. P V of 64 keys, then its remainder's:
__device__ __forceinline__ void mma_pv(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc, uint32_t bar0, uint32_t bar1) {
#define AMV_TS(A, B, P) "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [" A "], " B ", %3, " P ";\n\t"
#define AMV_PV_HEAD                                                                                                                            \
    "{\n\t.reg .pred p, q, t;\n\t.reg .b32 a1, a2, a3, c0, c1, c2, c3;\n\t.reg .b64 b1, b2, b3;\n\telect.sync _|q, 0xffffffff;\n\t"              \
    "setp.ne.b32 p, %4, 0;\n\tsetp.eq.u32 t, 0, 0;\n\tadd.u32 a1, %1, 8;\n\tadd.u32 a2, %1, 16;\n\tadd.u32 a3, %1, 24;\n\t"                         \
    "add.u64 b1, %2, 128;\n\tadd.u64 b2, %2, 256;\n\tadd.u64 b3, %2, 384;\n\t"
#define AMV_PV_TAIL                                                                                                                            \
    "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%5];\n\t"                                                       \
    "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%6];\n\t}"
    asm volatile(AMV_PV_HEAD "add.u32 c0, %1, 32;\n\tadd.u32 c1, %1, 40;\n\tadd.u32 c2, %1, 48;\n\tadd.u32 c3, %1, 56;\n\t" AMV_TS("%1", "%2", "p")
                     AMV_TS("a1", "b1", "t") AMV_TS("a2", "b2", "t") AMV_TS("a3", "b3", "t") AMV_TS("c0", "%2", "t") AMV_TS("c1", "b1", "t")
                         AMV_TS("c2", "b2", "t") AMV_TS("c3", "b3", "t") AMV_PV_TAIL ::"r"(d),
                 "r"(a), "l"(b), "r"(idesc), "r"(acc), "r"(bar0), "r"(bar1)
                 : "memory");
#undef AMV_TS
#undef AMV_PV_HEAD
#undef AMV_PV_TAIL
}
// S of 64 keys and 64 A columns of Q and K:
template <uint32_t A>
__device__ __forceinline__ void mma_s(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t bar0, uint32_t bar1) {
    constexpr uint64_t QA = kGroupRows * 128u / 16u, KA = kTcKeys * 128u / 16u;   // to the next 64 columns
#define AMV_SS(A, B, P) "@q tcgen05.mma.cta_group::1.kind::f16 [%0], " A ", " B ", %3, " P ";\n\t"
#define AMV_S_HEAD                                                                                                                             \
    "{\n\t.reg .pred p, q, t;\n\t.reg .b64 a1, a2, a3, a4, a5, a6, a7, b1, b2, b3, b4, b5, b6, b7;\n\telect.sync _|q, 0xffffffff;\n\t"             \
    "setp.ne.u32 p, 0, 0;\n\tsetp.eq.u32 t, 0, 0;\n\tadd.u64 a1, %1, 2;\n\tadd.u64 a2, %1, 4;\n\tadd.u64 a3, %1, 6;\n\t"                           \
    "add.u64 b1, %2, 2;\n\tadd.u64 b2, %2, 4;\n\tadd.u64 b3, %2, 6;\n\t"
#define AMV_S_TAIL                                                                                                                             \
    "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%4];\n\t"                                                       \
    "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%5];\n\t}"
    if constexpr (A == 2u)
        asm volatile(AMV_S_HEAD
                     "add.u64 a4, %1, %6;\n\tadd.u64 a5, a1, %6;\n\tadd.u64 a6, a2, %6;\n\tadd.u64 a7, a3, %6;\n\t"
                     "add.u64 b4, %2, %7;\n\tadd.u64 b5, b1, %7;\n\tadd.u64 b6, b2, %7;\n\tadd.u64 b7, b3, %7;\n\t" AMV_SS("%1", "%2", "p")
                         AMV_SS("a1", "b1", "t") AMV_SS("a2", "b2", "t") AMV_SS("a3", "b3", "t") AMV_SS("a4", "b4", "t") AMV_SS("a5", "b5", "t")
                             AMV_SS("a6", "b6", "t") AMV_SS("a7", "b7", "t") AMV_S_TAIL ::"r"(d),
                     "l"(a), "l"(b), "r"(idesc), "r"(bar0), "r"(bar1), "n"(QA), "n"(KA)
                     : "memory");
    else
        asm volatile(AMV_S_HEAD AMV_SS("%1", "%2", "p") AMV_SS("a1", "b1", "t") AMV_SS("a2", "b2", "t") AMV_SS("a3", "b3", "t") AMV_S_TAIL ::"r"(d), "l"(a),
                     "l"(b), "r"(idesc), "r"(bar0), "r"(bar1)
                     : "memory");
#undef AMV_SS
#undef AMV_S_HEAD
#undef AMV_S_TAIL
}
// P V of a tile and S of the one that takes its place, as mma_pv and mma_s.
template <uint32_t A>
__device__ __forceinline__ void mma_step(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc, uint32_t bar0, uint32_t bar1, uint64_t q, uint64_t k,
                                         uint32_t idesc_s, uint32_t bar2, uint32_t bar3) {
    constexpr uint64_t QA = kGroupRows * 128u / 16u, KA = kTcKeys * 128u / 16u;
#define AMV_TS(X, B, P) "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [" X "], " B ", %3, " P ";\n\t"
#define AMV_SS(X, B, P) "@q tcgen05.mma.cta_group::1.kind::f16 [%1], " X ", " B ", %9, " P ";\n\t"
#define AMV_COMMIT(X) "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [" X "];\n\t"
#define AMV_HEAD                                                                                                                               \
    "{\n\t.reg .pred p, q, t, z;\n\t.reg .b32 a1, a2, a3, c0, c1, c2, c3;\n\t.reg .b64 b1, b2, b3, x1, x2, x3, x4, x5, x6, x7, y1, y2, y3, y4, y5, y6, y7;\n\t" \
    "elect.sync _|q, 0xffffffff;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.eq.u32 t, 0, 0;\n\tsetp.ne.u32 z, 0, 0;\n\t"                                      \
    "add.u32 a1, %1, 8;\n\tadd.u32 a2, %1, 16;\n\tadd.u32 a3, %1, 24;\n\tadd.u64 b1, %2, 128;\n\tadd.u64 b2, %2, 256;\n\tadd.u64 b3, %2, 384;\n\t" \
    "add.u64 x1, %7, 2;\n\tadd.u64 x2, %7, 4;\n\tadd.u64 x3, %7, 6;\n\tadd.u64 y1, %8, 2;\n\tadd.u64 y2, %8, 4;\n\tadd.u64 y3, %8, 6;\n\t"        \
    AMV_TS("%1", "%2", "p") AMV_TS("a1", "b1", "t") AMV_TS("a2", "b2", "t") AMV_TS("a3", "b3", "t")
#define AMV_LOW                                                                                                                                \
    "add.u32 c0, %1, 32;\n\tadd.u32 c1, %1, 40;\n\tadd.u32 c2, %1, 48;\n\tadd.u32 c3, %1, 56;\n\t" AMV_TS("c0", "%2", "t") AMV_TS("c1", "b1", "t")      \
        AMV_TS("c2", "b2", "t") AMV_TS("c3", "b3", "t")
#define AMV_MID AMV_COMMIT("%5") AMV_COMMIT("%6") AMV_SS("%7", "%8", "z") AMV_SS("x1", "y1", "t") AMV_SS("x2", "y2", "t") AMV_SS("x3", "y3", "t")
#define AMV_MORE                                                                                                                               \
    "add.u64 x4, %7, %12;\n\tadd.u64 x5, x1, %12;\n\tadd.u64 x6, x2, %12;\n\tadd.u64 x7, x3, %12;\n\t"                                             \
    "add.u64 y4, %8, %13;\n\tadd.u64 y5, y1, %13;\n\tadd.u64 y6, y2, %13;\n\tadd.u64 y7, y3, %13;\n\t"                                             \
    AMV_SS("x4", "y4", "t") AMV_SS("x5", "y5", "t") AMV_SS("x6", "y6", "t") AMV_SS("x7", "y7", "t")
#define AMV_TAIL AMV_COMMIT("%10") AMV_COMMIT("%11") "}"
#define AMV_ARGS "r"(d), "r"(a), "l"(b), "r"(idesc), "r"(acc), "r"(bar0), "r"(bar1), "l"(q), "l"(k), "r"(idesc_s), "r"(bar2), "r"(bar3), "n"(QA), "n"(KA)
    if constexpr (A == 2u) asm volatile(AMV_HEAD AMV_LOW AMV_MID AMV_MORE AMV_TAIL ::AMV_ARGS : "memory");
    else asm volatile(AMV_HEAD AMV_LOW AMV_MID AMV_TAIL ::AMV_ARGS : "memory");
#undef AMV_TS
#undef AMV_SS
#undef AMV_COMMIT
#undef AMV_HEAD
#undef AMV_LOW
#undef AMV_MID
#undef AMV_MORE
#undef AMV_TAIL
#undef AMV_ARGS
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// Descriptor of a V tile as the B operand with its columns (N) contiguous: 64-column groups of the 128-byte swizzle
// kTcKeys * 128 bytes apart (leading offset), groups of eight keys 1024 bytes apart (stride offset).
__device__ __forceinline__ uint64_t v_desc(uint32_t smem_addr) {
    return (uint64_t)((smem_addr >> 4) & 0x3FFFu) | ((uint64_t)(kTcKeys * 128u >> 4) << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}

// 32 rows x 16 columns of 32 bits through 2048 bytes of shared memory, so that a row leaves 64 bytes at a time (a lane per row and 16 bytes: 32
// lines per store, 10 us a piece): lane 4 k + c takes columns 4 c .. 4 c + 3 of rows 8 i + k.
struct Staging {
    uint32_t base, lane, piece;
    __device__ __forceinline__ Staging(uint32_t at, uint32_t lane_) : base(at), lane(lane_), piece(lane_ & 3u) {}
    __device__ __forceinline__ uint32_t row(uint32_t i) const { return 8u * i + (lane >> 2); }
    __device__ __forceinline__ void put(const uint32_t (&v)[16]) const {   // this lane's row
#pragma unroll
        for (uint32_t k = 0; k < 4u; ++k)
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(base + lane * 64u + ((k ^ (lane >> 1 & 3u)) << 4)), "r"(v[4 * k]), "r"(v[4 * k + 1]),
                         "r"(v[4 * k + 2]), "r"(v[4 * k + 3])
                         : "memory");
        __syncwarp();
    }
    __device__ __forceinline__ float4 get(uint32_t r) const {
        float4 y;
        asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                     : "=f"(y.x), "=f"(y.y), "=f"(y.z), "=f"(y.w)
                     : "r"(base + r * 64u + ((piece ^ (r >> 1 & 3u)) << 4))
                     : "memory");
        return y;
    }
};
__device__ __forceinline__ void add4(float4& y, const float4& e, float f) {
    y.x = fmaf(e.x, f, y.x);
    y.y = fmaf(e.y, f, y.y);
    y.z = fmaf(e.z, f, y.z);
    y.w = fmaf(e.w, f, y.w);
}

// The accumulator of a warp's rows goes to the piece's slot (f32 [row of the group][D + 4]: the maximum it refers to, values from column 4 on), with
// what the slot holds already unless this is the first time. Returns whether a column of this thread's row is not finite. What the
// slot holds is read a round ahead. A function of its own, so that the loop over key tiles keeps its registers.
template <int D>
__device__ __noinline__ bool add_to_slot(float* slot, uint32_t n_rows, uint32_t acc, uint32_t s_out, bool first, float m) {
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u, r0 = (warp & 3u) * 32u;
    const Staging stage(s_out + warp * 2048u, lane);
    float* own = slot + (uint64_t)(r0 + lane) * (D + 4u);
    const bool mine = r0 + lane < n_rows;
    const float f = first || !mine ? 0.0f : weight(*own, m);
    if (mine) *own = m;
    float check = 0.0f, f_row[4];
    float4 held[4];
    float* at[4];
#pragma unroll
    for (uint32_t i = 0; i < 4u; ++i) {
        const uint32_t r = stage.row(i);
        f_row[i] = __shfl_sync(0xffffffffu, f, r);
        at[i] = r0 + r < n_rows ? slot + (uint64_t)(r0 + r) * (D + 4u) + 4u + 4u * stage.piece : nullptr;
        held[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (f_row[i] != 0.0f) held[i] = *reinterpret_cast<const float4*>(at[i]);
    }
#pragma unroll 1
    for (uint32_t c = 0; c < D; c += 16u) {
        float4 now[4];
#pragma unroll
        for (uint32_t i = 0; i < 4u; ++i) {
            now[i] = held[i];
            if (f_row[i] != 0.0f && c + 16u < D) held[i] = *reinterpret_cast<const float4*>(at[i] + c + 16u);
        }
        uint32_t v[16];
        tmem_ld16(acc + c, v);
#pragma unroll
        for (uint32_t k = 0; k < 16u; ++k) check = fmaf(__uint_as_float(v[k]), 0.0f, check);
        stage.put(v);
#pragma unroll
        for (uint32_t i = 0; i < 4u; ++i) {
            if (!at[i]) continue;
            float4 y = stage.get(stage.row(i));
            if (f_row[i] != 0.0f) add4(y, now[i], f_row[i]);
            *reinterpret_cast<float4*>(at[i] + c) = y;
        }
        __syncwarp();
    }
    return mine && check != 0.0f;
}

// A group's share of a piece: its rows, the keys any of them sees and those all of them see, its key tiles [t0, t1).
struct Group {
    uint32_t r0, rows, lo, hi, lo_all, hi_all, t0, t1;
};
__device__ __forceinline__ Group group_of(const Args& pc, const Piece& p, uint32_t g) {
    Group x;
    x.r0 = p.r0 + g * kGroupRows;
    x.rows = p.R > x.r0 ? min(kGroupRows, p.R - x.r0) : 0u;
    x.lo = x.hi = x.lo_all = x.hi_all = x.t0 = x.t1 = 0u;
    if (x.rows) {
        const Span a = row_span(pc, p.q, x.r0), b = row_span(pc, p.q, x.r0 + x.rows - 1u);
        x.lo = a.lo;
        x.hi = b.hi;
        x.lo_all = b.lo;
        x.hi_all = a.hi;
        x.t0 = max(p.first + p.a, x.lo / kTcKeys);
        x.t1 = x.hi > x.lo ? min(p.first + p.b, (x.hi + kTcKeys - 1u) / kTcKeys) : x.t0;
        if (x.t1 < x.t0) x.t1 = x.t0;
    }
    return x;
}

template <int D, bool EXACT>
__global__ void __launch_bounds__(Tc<D, EXACT>::THREADS, 1)
paged_tc_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map, const __grid_constant__ CUtensorMap q_map,
                const __grid_constant__ Args pc) {
    using L = Tc<D, EXACT>;
    constexpr uint32_t GROUPS = L::GROUPS;
    constexpr uint32_t A = L::A, ST = L::STAGES, C = D / 32;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* base = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    uint8_t *sQ = base, *sK = sQ + GROUPS * L::Q, *sV = sK + ST * L::TILE;
    uint8_t* s_out = sV + ST * L::TILE;
    uint64_t* bars = reinterpret_cast<uint64_t*>(s_out + L::STAGE_OUT + L::PAIRS);
    const uint32_t k_full = smem_u32(bars), k_empty = k_full + 8u * ST, v_full = k_empty + 8u * ST, v_empty = v_full + 8u * ST,
                   q_full = v_empty + 8u * ST, q_empty = q_full + 16u, s_full = q_empty + 16u, p_full = s_full + 32u, pv_done = p_full + 32u,
                   drain = pv_done + 32u;   // the last three: [group][tile & 1]
    Ctl* ctl = reinterpret_cast<Ctl*>(bars + 4u * ST + 18u);
    uint32_t* s_warp = reinterpret_cast<uint32_t*>(ctl + 1);                   // [12]
    volatile uint32_t* s_bad = s_warp + L::THREADS / 32u;                      // 16-key steps whose page is none, of the last key tiles
    uint32_t* s_pref = reinterpret_cast<uint32_t*>(reinterpret_cast<uint8_t*>(bars) + 512u);
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
    if (threadIdx.x == 0) {
        for (uint32_t s = 0; s < ST; ++s) {
            mbar_init(k_full + 8u * s, 1u);
            mbar_init(k_empty + 8u * s, GROUPS);
            mbar_init(v_full + 8u * s, 1u);
            mbar_init(v_empty + 8u * s, GROUPS);
        }
        for (uint32_t g = 0; g < 2u; ++g) {
            mbar_init(q_full + 8u * g, 1u);
            mbar_init(q_empty + 8u * g, 1u);
            for (uint32_t b = 0; b < 2u; ++b) {
                mbar_init(s_full + 16u * g + 8u * b, 1u);
                mbar_init(p_full + 16u * g + 8u * b, 4u * L::PARTS);
                mbar_init(pv_done + 16u * g + 8u * b, 1u);   // two of them: a wait for tile j - 1's meets it at most one phase behind
            }
        }
        mbar_init(drain, 1u);
        mbar_init(drain + 8u, 1u);
        ctl->abort = 0u;
        fence_barrier_init();
    }
    // boxes that no row needs are not loaded: their steps are not multiplied, but a zero is a better guest than a NaN
    for (uint32_t i = threadIdx.x; i < 2u * ST * L::TILE / 16u; i += L::THREADS) reinterpret_cast<uint4*>(sK)[i] = make_uint4(0u, 0u, 0u, 0u);
    if (warp == L::MMA) tmem_alloc<false>(smem_u32(&ctl->tmem_base), L::TMEM);
    fence_async_smem();
    pdl_wait();
    tc_fence_before();
    const uint32_t total = build_line<L::ROWS, L::THREADS / 32u>(pc, s_pref, s_warp);   // (its barriers publish the above)
    tc_fence_after();
    pdl_trigger();   // not before the tensor memory is this CTA's
    const uint32_t tmem = ctl->tmem_base;
    const Stretch st = my_stretch(total);
    Walk<L::ROWS> walk(st);
    const uint32_t P = 1u << pc.page_log2, box = P < kTcKeys ? P : kTcKeys, boxes = kTcKeys / box;
    bool ok = true;
    uint32_t bar0 = 0, asked0 = 0, bar1 = 0, asked1 = 0, depth = 1;   // two rings of copies (or the MMAs) that this warp waits for before it leaves

    if (warp >= L::MMA) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
        if (warp == L::LOAD) {
            Ring kr(ST), vr(ST);
            uint32_t tiles = 0;     // of this CTA so far
            uint32_t k_issued = 0, v_issued = 0;
            while (ok && walk.next(pc, s_pref)) {
                const Piece& p = walk.p;
                const uint32_t lo = row_span(pc, p.q, p.r0).lo, hi = row_span(pc, p.q, min(p.r0 + L::ROWS, p.R) - 1u).hi;
                int32_t page = -1, page_v = -1;   // this lane's box: K's, and V's of the tile before
                uint32_t load = 0, load_v = 0;
                for (uint32_t i = p.a; ok && i <= p.b; ++i) {
                    const uint32_t key0 = (p.first + i) * kTcKeys, b0 = key0 + lane * box;
                    if (i < p.b) {
                        const bool want = lane < boxes && b0 < hi && b0 + box > lo;
                        page = want ? page_of(pc, p.q, b0) : -1;
                        const uint32_t none = __ballot_sync(0xffffffffu, want && page < 0);
                        load = __ballot_sync(0xffffffffu, page >= 0);
                        uint32_t bad = 0;
                        if (none) {
                            for (uint32_t j = 0; j < kTcKeys / 16u; ++j) bad |= (none >> (16u * j / box) & 1u) << j;
                            if (lane == 0u) refuse(pc, __popc(none));
                        }
                        ok = wait_on(k_empty + 8u * kr.idx, kr.phase ^ 1u, ctl, pc.status, 0xD00u);
                        ok = __all_sync(0xffffffffu, ok);
                        if (!ok) break;
                        if (lane == 0u) {
                            s_bad[tiles & (kBadRing - 1u)] = bad;
                            mbar_arrive_expect_tx(k_full + 8u * kr.idx, (uint32_t)__popc(load) * box * 128u * A);
                        }
                        __syncwarp();
                        if (page >= 0)
                            for (uint32_t a = 0; a < A; ++a)
                                tma_box(smem_u32(sK + kr.idx * L::TILE) + a * (kTcKeys * 128u) + lane * box * 128u, &k_map, k_full + 8u * kr.idx,
                                        (int)(64u * a), (int)(b0 & (P - 1u)), (int)p.group, page);
                        ++k_issued;
                        ++tiles;
                        kr.advance();
                    }
                    if (i > p.a) {   // V of the tile before
                        ok = wait_on(v_empty + 8u * vr.idx, vr.phase ^ 1u, ctl, pc.status, 0xD10u);
                        ok = __all_sync(0xffffffffu, ok);
                        if (!ok) break;
                        if (lane == 0u) mbar_arrive_expect_tx(v_full + 8u * vr.idx, (uint32_t)__popc(load_v) * box * 128u * A);
                        __syncwarp();
                        if (page_v >= 0)
                            for (uint32_t a = 0; a < A; ++a)
                                tma_box(smem_u32(sV + vr.idx * L::TILE) + a * (kTcKeys * 128u) + lane * box * 128u, &v_map, v_full + 8u * vr.idx,
                                        (int)(64u * a), (int)((b0 - kTcKeys) & (P - 1u)), (int)p.group, page_v);
                        ++v_issued;
                        vr.advance();
                    }
                    page_v = page;
                    load_v = load;
                }
            }
            bar0 = k_full, asked0 = k_issued, bar1 = v_full, asked1 = v_issued, depth = ST;
        } else if (warp < L::LOAD) {
            const uint32_t g = warp - L::MMA;
            const uint32_t idesc_s = make_idesc(1u, 0u, kTcKeys, kGroupRows), idesc_o = make_idesc(1u, 0u, (uint32_t)D, kGroupRows) | (1u << 16);
            const uint32_t t_s = tmem + 2u * g * kTcKeys, t_o = tmem + 2u * GROUPS * kTcKeys + g * D;
            // EXACT: the accumulator of the group's tile i of a piece, two in turn
            auto acc_of = [](uint32_t i) { return EXACT ? (i / kFlush & 1u) * (uint32_t)D : 0u; };
            const uint32_t takes = EXACT ? kFlush : pc.slots ? kRenew : 1u << 31;   // key tiles that an accumulator takes
            auto anew = [&](uint32_t i) { return (i & (takes - 1u)) == 0u; };
            const uint64_t dq = make_smem_desc(smem_u32(sQ + g * L::Q)), dk = make_smem_desc(smem_u32(sK)), dv = v_desc(smem_u32(sV));
            const uint32_t my_s = s_full + 16u * g, my_p = p_full + 16u * g, my_pv = pv_done + 16u * g;
            Ring kr(ST), vr(ST);
            uint32_t tiles = 0, q_uses = 0, s_tiles = 0, p_tiles = 0;   // of the CTA; of this group: pieces with Q, tiles with S, with P V issued
            while (ok && walk.next(pc, s_pref)) {
                const Piece& p = walk.p;
                const Group x = group_of(pc, p, g);
                const uint32_t hi_all = row_span(pc, p.q, min(p.r0 + L::ROWS, p.R) - 1u).hi, T0 = p.first + p.a, T1 = p.first + p.b;
                uint32_t started = 0u;
                uint32_t bad_1 = 0u, bad_2 = 0u;   // 16-key steps without a page, of tile t - 1 and t - 2
                for (uint32_t t = T0; t < T1 + 2u; ++t) {   // P V of tile t - 2, then S of tile t in its place
                    // (the group's rows see some of tile t, all of tile t - 2, and neither is its first)
                    if (t >= T0 + 2u && t < T1 && t - 2u >= x.t0 && t < x.t1 && bad_2 == 0u && (t - 2u) * kTcKeys >= x.lo) {
                        const uint32_t b = p_tiles & 1u;
                        ok = wait_on(v_full + 8u * vr.idx, vr.phase, ctl, pc.status, 0xD40u) && wait_on(k_full + 8u * kr.idx, kr.phase, ctl, pc.status, 0xD60u) &&
                             wait_on(my_p + 8u * b, (p_tiles >> 1) & 1u, ctl, pc.status, 0xD50u);
                        ok = __all_sync(0xffffffffu, ok);
                        if (!ok) break;
                        tc_fence_after();
                        if (anew(t - 2u - x.t0)) started = 0u;
                        mma_step<A>(t_o + acc_of(t - 2u - x.t0), t_s + b * kTcKeys, dv + vr.idx * (L::TILE / 16u), idesc_o, started, my_pv + 8u * b, v_empty + 8u * vr.idx, dq,
                                           dk + kr.idx * (L::TILE / 16u), idesc_s, my_s + 8u * b, k_empty + 8u * kr.idx);
                        started = 1u;
                        if (t + 1u == x.t1) commit(q_empty + 8u * g);
                        bad_2 = bad_1;
                        bad_1 = s_bad[(tiles + (t - T0)) & (kBadRing - 1u)];
                        ++p_tiles;
                        ++s_tiles;
                        vr.advance();
                        kr.advance();
                        continue;
                    }
                    if (t >= T0 + 2u) {
                        const uint32_t u = t - 2u, key0 = u * kTcKeys, b = p_tiles & 1u;
                        const bool mine = u >= x.t0 && u < x.t1;
                        ok = wait_on(v_full + 8u * vr.idx, vr.phase, ctl, pc.status, 0xD40u);
                        if (mine) ok = ok && wait_on(my_p + 8u * b, (p_tiles >> 1) & 1u, ctl, pc.status, 0xD50u);
                        ok = __all_sync(0xffffffffu, ok);
                        if (!ok) break;
                        if (mine) {
                            ++p_tiles;
                            tc_fence_after();
                            if (anew(u - x.t0)) started = 0u;
                            const uint32_t t_acc = t_o + acc_of(u - x.t0);
                            const uint32_t steps = ~bad_2 & 0xFu;   // 16 keys whose page is there
                            const uint64_t dvt = dv + vr.idx * (L::TILE / 16u);
                            if (steps == 0xFu && key0 >= x.lo && key0 + kTcKeys <= x.hi) {
                                mma_pv(t_acc, t_s + b * kTcKeys, dvt, idesc_o, started, my_pv + 8u * b, v_empty + 8u * vr.idx);
                                started = 1u;
                            } else {
                                if (hi_all < key0 + kTcKeys) {   // the rest of the step of the last key
                                    const uint32_t from = hi_all - key0, n = (16u - (from & 15u)) & 15u;
                                    for (uint32_t j = lane; j < n * (D / 8u); j += 32u) {
                                        const uint32_t r = from + j / (D / 8u), c = j % (D / 8u);
                                        *reinterpret_cast<uint4*>(sV + vr.idx * L::TILE + (c >> 3) * (kTcKeys * 128u) + r * 128u + ((c & 7u) << 4)) =
                                            make_uint4(0u, 0u, 0u, 0u);
                                    }
                                    fence_async_smem();
                                    __syncwarp();
                                }
                                const uint32_t s0 = x.lo > key0 ? (x.lo - key0) / 16u : 0u, s1 = (min(x.hi - key0, kTcKeys) + 15u) / 16u;
    #pragma unroll 1
                                for (uint32_t k = s0; k < s1; ++k) {   // 16 keys a step: 8 columns of P, two groups of eight V rows
                                    if (!(steps >> k & 1u)) continue;
                                    mma_ts(t_acc, t_s + b * kTcKeys + 8u * k, dvt + 128u * k, idesc_o, started);
                                    mma_ts(t_acc, t_s + b * kTcKeys + 32u + 8u * k, dvt + 128u * k, idesc_o, 1u);
                                    started = 1u;
                                }
                                if (!started) {   // no page of the tile is there, and the accumulator is to begin anew: with zeros
                                    for (uint32_t j = lane; j < 16u * (D / 8u); j += 32u) {
                                        const uint32_t r = 16u * s0 + j / (D / 8u), c = j % (D / 8u);
                                        *reinterpret_cast<uint4*>(sV + vr.idx * L::TILE + (c >> 3) * (kTcKeys * 128u) + r * 128u + ((c & 7u) << 4)) =
                                            make_uint4(0u, 0u, 0u, 0u);
                                    }
                                    fence_async_smem();
                                    __syncwarp();
                                    mma_ts(t_acc, t_s + b * kTcKeys + 8u * s0, dvt + 128u * s0, idesc_o, 0u);
                                    started = 1u;
                                }
                                commit(my_pv + 8u * b);
                                commit(v_empty + 8u * vr.idx);
                            }
                        } else if (lane == 0u) {
                            mbar_arrive(v_empty + 8u * vr.idx);
                        }
                        vr.advance();
                    }
                    if (t < T1) {
                        const bool mine = t >= x.t0 && t < x.t1;
                        ok = wait_on(k_full + 8u * kr.idx, kr.phase, ctl, pc.status, 0xD60u);
                        if (mine && t == x.t0) {
                            ok = ok && wait_on(q_full + 8u * g, q_uses & 1u, ctl, pc.status, 0xD70u);
                            ++q_uses;
                        }
                        ok = __all_sync(0xffffffffu, ok);
                        if (!ok) break;
                        if (mine) {
                            const uint32_t b = s_tiles & 1u;
                            ++s_tiles;
                            mma_s<A>(t_s + b * kTcKeys, dq, dk + kr.idx * (L::TILE / 16u), idesc_s, my_s + 8u * b, k_empty + 8u * kr.idx);
                            if (t + 1u == x.t1) commit(q_empty + 8u * g);
                        } else if (lane == 0u) {
                            mbar_arrive(k_empty + 8u * kr.idx);
                        }
                        kr.advance();
                    }
                    bad_2 = bad_1;
                    bad_1 = t < T1 ? s_bad[(tiles + (t - T0)) & (kBadRing - 1u)] : 0u;
                }
                tiles += p.b - p.a;
            }
            commit(drain + 8u * g);   // MMAs already issued finish before the CTA gives its memory back, whoever gives up, and when
            bar0 = drain + 8u * g, asked0 = 1u;
        } else if (warp == L::QWARP) {
            // Q rows into the K-major 128-byte swizzle, idle rows zero
            uint32_t uses[2] = {0u, 0u};
            while (ok && walk.next(pc, s_pref)) {
                const Piece& p = walk.p;
    #pragma unroll 1
                for (uint32_t g = 0; g < GROUPS; ++g) {
                    const Group x = group_of(pc, p, g);
                    if (x.t1 <= x.t0) continue;
                    const uint32_t n = g ? uses[1] : uses[0];
                    if (n) ok = wait_on(q_empty + 8u * g, (n - 1u) & 1u, ctl, pc.status, 0xDC0u);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    if (g) ++uses[1];
                    else ++uses[0];
                    if (pc.q_boxes) {   // heads of a group in a power of two: 128 / G tokens by one copy per 64 columns (rows of others behind the last)
                        if (lane == 0u) {
                            mbar_arrive_expect_tx(q_full + 8u * g, L::Q);
                            for (uint32_t a = 0; a < A; ++a)
                                tma_load_3d(smem_u32(sQ + g * L::Q + a * (kGroupRows * 128u)), &q_map, q_full + 8u * g, (int)(64u * a), (int)(p.group * pc.G),
                                            (int)(p.q.tok0 + query_of(pc, x.r0)));
                        }
                        __syncwarp();
                        continue;
                    }
                    constexpr uint32_t PIECES = D / 8, PER = 32u / PIECES;   // 16-byte pieces of a row; rows per load of a warp
                    const uint32_t c = lane % PIECES, at = smem_u32(sQ + g * L::Q + (c >> 3) * (kGroupRows * 128u));
                    uint32_t r = lane / PIECES, token = query_of(pc, x.r0 + r), head = x.r0 + r - token * pc.G;
                    const __half* q0 = pc.q + (uint64_t)p.q.tok0 * pc.q_s + (uint64_t)p.group * pc.G * D + 8u * c;
    #pragma unroll 4
                    for (uint32_t i = 0; i < kGroupRows / PER; ++i) {
                        const uint32_t to = at + r * 128u + (((c & 7u) ^ (r & 7u)) << 4);
                        if (r < x.rows)
                            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(q0 + (uint64_t)token * pc.q_s + head * D) : "memory");
                        else
                            asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(to), "r"(0u) : "memory");
                        r += PER;
                        head += PER;
                        while (head >= pc.G) {
                            head -= pc.G;
                            ++token;
                        }
                    }
                    asm volatile("cp.async.wait_all;" ::: "memory");
                    fence_async_smem();   // the MMAs read Q through the async proxy
                    __syncwarp();
                    if (lane == 0u) mbar_arrive(q_full + 8u * g);
                }
            }
            bar0 = q_full, asked0 = uses[0], bar1 = q_full + 8u, asked1 = uses[1];   // Q of a group is a ring of one stage
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
        constexpr uint32_t KEYS = L::KEYS, COLS = L::COLS;
        const uint32_t g = EXACT ? 0u : warp >> 2, part = EXACT ? warp >> 2 : 0u, my = threadIdx.x & 127u;
        const uint32_t lanes = ((warp & 3u) * 32u) << 16, to = tmem + lanes + 2u * GROUPS * kTcKeys + g * D + part * COLS;
        // EXACT: the two threads of a row tell one another a value and whether all is well, so that both leave together. Two places in
        // turn: a warp writes to one again behind the next barrier, which the other one passes after it has read.
        float2* s_pair = reinterpret_cast<float2*>(s_out + L::STAGE_OUT);
        uint32_t told = 0;
        auto slot_rows = [&](const Piece& p, const Group& x) {
            return pc.slots + ((uint64_t)(2u * blockIdx.x + (p.a == 0u ? 1u : 0u)) * L::ROWS + (x.r0 - p.r0)) * (D + 4u);
        };
        auto tell = [&](float v, bool& fine) {
            s_pair[((told & 1u) * 2u + part) * kGroupRows + my] = make_float2(v, fine ? 1.0f : 0.0f);
            tc_fence_before();
            asm volatile("bar.sync %0, 64;" ::"r"(1u + (warp & 3u)) : "memory");
            tc_fence_after();
            const float2 y = s_pair[((told & 1u) * 2u + (part ^ 1u)) * kGroupRows + my];
            ++told;
            fine = __all_sync(0xffffffffu, fine && y.y != 0.0f);
            return y.x;
        };
        uint32_t j = 0, tiles = 0;   // key tiles of this group, of the CTA, so far
        bool cut = false, again = false;   // again: rows that are not finite although their sum is
        while (walk.next(pc, s_pref)) {
            const Piece& p = walk.p;
            const Group x = group_of(pc, p, g);
            const uint32_t row = x.r0 + my;
            const bool valid = my < x.rows;
            const Span span = valid ? row_span(pc, p.q, row) : Span{0u, 0u};
            float m_run = neg_inf(), l_run = 0.0f;
            float sum_o[EXACT ? COLS : 1];   // EXACT: the row's sum; the accumulators hold the last tiles
            if (EXACT) {
#pragma unroll
                for (uint32_t c = 0; c < COLS; ++c) sum_o[c] = 0.0f;
            }
            auto add_up = [&](uint32_t acc) {
#pragma unroll
                for (uint32_t c = 0; c < COLS; c += 32u) {
                    uint32_t v[32];
                    tmem_ld32_async(to + acc * (uint32_t)D + c, v);
                    tmem_wait_ld();
#pragma unroll
                    for (uint32_t k = 0; k < 32u; ++k) sum_o[EXACT ? c + k : 0u] += __uint_as_float(v[k]);
                }
            };
            for (uint32_t t = x.t0; t < x.t1; ++t, ++j) {
                const uint32_t key0 = t * kTcKeys, b = j & 1u, ts = tmem + lanes + (2u * g + b) * kTcKeys;
                if (!EXACT && t != x.t0 && (t - x.t0) % kRenew == 0u && pc.slots) {   // the accumulator goes to the slot, and begins anew
                    ok = ok && wait_on(pv_done + 16u * g + 8u * (b ^ 1u), ((j - 1u) >> 1) & 1u, ctl, pc.status, 0xDC4u);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    tc_fence_after();
                    again = add_to_slot<D>(slot_rows(p, x), x.rows, to, smem_u32(s_out), t - x.t0 == kRenew, m_run) || again;
                }
                ok = ok && wait_on(s_full + 16u * g + 8u * b, (j >> 1) & 1u, ctl, pc.status, 0xDA0u);
                ok = __all_sync(0xffffffffu, ok);
                if (!EXACT && !ok) break;
                tc_fence_after();
                const uint32_t gone = s_bad[(tiles + (t - p.first - p.a)) & (kBadRing - 1u)];
                float s[KEYS];
#pragma unroll
                for (uint32_t c = 0; c < KEYS; c += 32u) tmem_ld32_async(ts + part * KEYS + c, reinterpret_cast<uint32_t*>(s) + c);
                tmem_wait_ld();
                // the same for every thread of the group
                const bool open = gone == 0u && key0 >= x.lo_all && key0 + kTcKeys <= x.hi_all, scaled = pc.softcap == 0.0f && pc.scale2 > 0.0f;
                if (!scaled) capped(pc, s);   // the cap, or a scale that is not positive
                if (!open) {     // hidden keys: a bit per key of 32
#pragma unroll
                    for (uint32_t c = 0; c < KEYS; c += 32u) {
                        const uint32_t at = part * KEYS + c, first = key0 + at;
                        const uint32_t a = span.lo > first ? min(span.lo - first, 32u) : 0u, e = span.hi > first ? min(span.hi - first, 32u) : 0u;
                        const uint32_t below = e >= 32u ? 0xffffffffu : (1u << e) - 1u, from = a >= 32u ? 0u : 0xffffffffu << a;
                        const uint32_t there = ((gone >> (at >> 4) & 1u) ? 0u : 0xffffu) | ((gone >> ((at >> 4) + 1u) & 1u) ? 0u : 0xffff0000u);
                        const uint32_t seen = below & from & there;
#pragma unroll
                        for (uint32_t k = 0; k < 32u; ++k) s[c + k] = seen >> k & 1u ? s[c + k] : neg_inf();
                    }
                }
                float m4[4];
#pragma unroll
                for (uint32_t k = 0; k < 4u; ++k) m4[k] = fmaxf(s[2u * k], s[2u * k + 1u]);
#pragma unroll
                for (uint32_t k = 8u; k < KEYS; k += 2u) m4[(k >> 1) & 3u] = max3(m4[(k >> 1) & 3u], s[k], s[k + 1u]);
                const float mul = scaled ? pc.scale2 : 1.0f;
                float mx = fmaxf(max3(m4[0], m4[1], m4[2]), m4[3]) * mul;
                if (EXACT) {   // (both warps of the rows have read their scores behind this, and write P over them)
                    mx = fmaxf(mx, tell(mx, ok));
                    if (!ok) break;
                }
                // The accumulator that tile t - 2 completed is added up now: its P V is done, since S of this tile was issued behind it.
                if (EXACT && t - x.t0 > kFlush && (t - x.t0) % kFlush == 1u) add_up((t - 2u - x.t0) / kFlush & 1u);
                const bool grow = mx > m_run + kGrowth || (m_run == neg_inf() && mx != neg_inf());
                if (__any_sync(0xffffffffu, grow)) {   // a row's sum and accumulator move to the new reference
                    const float f = !grow ? 1.0f : weight(m_run, mx);
                    if (grow) m_run = mx;
                    l_run *= f;
                    if (EXACT) {
#pragma unroll
                        for (uint32_t c = 0; c < COLS; ++c) sum_o[EXACT ? c : 0u] *= f;
                    }
                    if (t != x.t0) {
                        const uint32_t last = to + (EXACT ? ((t - 1u - x.t0) / kFlush & 1u) * (uint32_t)D : 0u);   // what tile t - 1 went to
                        ok = wait_on(pv_done + 16u * g + 8u * (b ^ 1u), ((j - 1u) >> 1) & 1u, ctl, pc.status, 0xDC8u);
                        ok = __all_sync(0xffffffffu, ok);
                        if (!EXACT && !ok) break;
                        tc_fence_after();
#pragma unroll 1
                        for (uint32_t c = 0; c < COLS; c += 16u) {
                            uint32_t v[16];
                            tmem_ld16(last + c, v);
#pragma unroll
                            for (int k = 0; k < 16; ++k) v[k] = __float_as_uint(__uint_as_float(v[k]) * f);
                            tmem_st16_async(last + c, v);
                        }
                    }
                }
                const float ref = m_run == neg_inf() ? 0.0f : m_run;
                const uint64_t mul_2 = pack2(mul, mul), ref2 = pack2(-ref, -ref);
                uint64_t sum2[2] = {0ull, 0ull};
#pragma unroll
                for (uint32_t h = 0; h < KEYS / 32u; ++h) {
                    uint32_t ph[16], pl[16];
#pragma unroll
                    for (uint32_t k = 0; k < 16u; ++k) {
                        const float2 e = unpack2(fma2(pack2(s[32u * h + 2u * k], s[32u * h + 2u * k + 1u]), mul_2, ref2));
                        const float p0 = ex2(e.x), p1 = ex2(e.y);
                        sum2[k & 1u] = add2(sum2[k & 1u], pack2(p0, p1));
                        const __half2 hi = __floats2half2_rn(p0, p1);
                        ph[k] = *reinterpret_cast<const uint32_t*>(&hi);
                        const float2 f2 = __half22float2(hi);
                        const __half2 low = __floats2half2_rn(p0 - f2.x, p1 - f2.y);
                        pl[k] = *reinterpret_cast<const uint32_t*>(&low);
                    }
                    tmem_st16_async(ts + 16u * (part + h), ph);   // over this tile's scores
                    tmem_st16_async(ts + 32u + 16u * (part + h), pl);
                }
                const float2 sums = unpack2(add2(sum2[0], sum2[1]));
                l_run += sums.x + sums.y;
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0u) mbar_arrive(p_full + 16u * g + 8u * b);
            }
            // ---- results of this piece ----
            const bool some = x.t1 > x.t0, whole = p.a == 0u && p.b == p.n;
            if (some) ok = ok && wait_on(pv_done + 16u * g + 8u * ((j - 1u) & 1u), ((j - 1u) >> 1) & 1u, ctl, pc.status, 0xDB0u) && !ctl->abort;
            ok = __all_sync(0xffffffffu, ok);
            if (EXACT) l_run += tell(l_run, ok);
            if (!ok) break;
            tc_fence_after();
            tiles += p.b - p.a;
            // (the last tile's accumulator is read below; the other one where that tile was its first)
            const uint32_t n_tiles = x.t1 - x.t0, to_last = to + (EXACT && some ? ((n_tiles - 1u) / kFlush & 1u) * (uint32_t)D : 0u);
            if (EXACT && some && n_tiles > 1u && (n_tiles - 1u) % kFlush == 0u) add_up((n_tiles - 2u) / kFlush & 1u);
            if (x.rows) {
                const uint32_t query = query_of(pc, row), token = p.q.tok0 + query, head = p.group * pc.G + row - query * pc.G;
                float* slot = slot_rows(p, x);
                const bool parts = !whole || pc.out == OUT_PARTS;
                float own = 1.0f, other = 0.0f;      // factors of the values here and of those over other keys
                // what the slot holds of this piece
                const float m_slot = !EXACT && pc.slots && valid && x.t1 - x.t0 > kRenew ? slot[(uint64_t)my * (D + 4u)] : neg_inf();
                const float* extra = nullptr;
                void* dst = nullptr;
                if (valid) {
                    if (parts) {
                        float* r = whole ? reinterpret_cast<float*>(pc.dst) + dst_row(pc, token, head, D) : slot + (uint64_t)my * (D + 4u);
                        if (part == 0u) *reinterpret_cast<float2*>(r) = make_float2(m_run, l_run);
                        dst = r + 4u + part * COLS;
                    } else {
                        float l = l_run, f = 1.0f;
                        if (pc.extra) {
                            extra = pc.extra + ((uint64_t)token * pc.n_head + head) * (D + 4u);
                            const float2 ml = *reinterpret_cast<const float2*>(extra);
                            const float top = fmaxf(m_run, ml.x);
                            f = weight(m_run, top);
                            other = weight(ml.x, top);
                            l = l * f + ml.y * other;
                            if (other == 0.0f) extra = nullptr;
                        }
                        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
                        own = f * inv;
                        other *= inv;
                        const uint64_t e = dst_row(pc, token, head, D) + part * COLS;
                        dst = pc.out == OUT_F16 ? (void*)(reinterpret_cast<__half*>(pc.dst) + e) : (void*)(reinterpret_cast<float*>(pc.dst) + e);
                    }
                }
                float check = 0.0f;
                const bool nothing = l_run == 0.0f;   // nothing was accumulated, or only what zeros made
                unsigned long long row_dst[4], row_extra[4];
                float row_other[4], row_slot[4];   // row_slot: the factor of what the slot holds of this piece
                const float held = nothing ? 0.0f : weight(m_slot, m_run) * own;
                const Staging stage(smem_u32(s_out) + warp * 2048u, lane);
#pragma unroll
                for (uint32_t i = 0; i < 4u; ++i) {
                    row_dst[i] = __shfl_sync(0xffffffffu, (unsigned long long)dst, stage.row(i));
                    row_extra[i] = __shfl_sync(0xffffffffu, (unsigned long long)extra, stage.row(i));
                    row_other[i] = __shfl_sync(0xffffffffu, other, stage.row(i));
                    row_slot[i] = __shfl_sync(0xffffffffu, held, stage.row(i));
                }
                const bool f16 = !parts && pc.out == OUT_F16;
#pragma unroll(EXACT ? COLS / 16 : 1)
                for (uint32_t c = 0; c < COLS; c += 16u) {
                    uint32_t v[16];
                    if (some) tmem_ld16(to_last + c, v);
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        const float o = nothing || !some ? 0.0f : EXACT ? sum_o[EXACT ? c + j : 0u] + __uint_as_float(v[j]) : __uint_as_float(v[j]);
                        check = fmaf(o, 0.0f, check);
                        v[j] = __float_as_uint(own == 0.0f ? 0.0f : o * own);
                    }
                    stage.put(v);
#pragma unroll
                    for (uint32_t i = 0; i < 4u; ++i) {
                        if (!row_dst[i]) continue;
                        float4 y = stage.get(stage.row(i));
                        if (!EXACT && row_slot[i] != 0.0f)
                            add4(y, *reinterpret_cast<const float4*>(slot + (uint64_t)((warp & 3u) * 32u + stage.row(i)) * (D + 4u) + 4u + c + 4u * stage.piece), row_slot[i]);
                        if (row_extra[i])
                            add4(y, *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(row_extra[i]) + 4u + part * COLS + c + 4u * stage.piece), row_other[i]);
                        if (f16) {
                            const __half2 h0 = __floats2half2_rn(y.x, y.y), h1 = __floats2half2_rn(y.z, y.w);
                            *reinterpret_cast<uint2*>(reinterpret_cast<__half*>(row_dst[i]) + c + 4u * stage.piece) =
                                make_uint2(*reinterpret_cast<const uint32_t*>(&h0), *reinterpret_cast<const uint32_t*>(&h1));
                        } else {
                            *reinterpret_cast<float4*>(reinterpret_cast<float*>(row_dst[i]) + c + 4u * stage.piece) = y;
                        }
                    }
                    __syncwarp();
                }
                if (EXACT) check += tell(check, ok);   // (what the other warp has written of the rows is there)
                again = again || (valid && check != 0.0f && l_run - l_run == 0.0f);
            }
            if (p.a == 0u && p.b < p.n) {
                cut = true;
                if (threadIdx.x == 0u) note_cut(pc, st, p, min(L::ROWS, p.R - p.r0));
            }
            tc_fence_before();   // (the next P V overwrites the accumulator behind an arrival of this thread)
        }
        if (!cut && threadIdx.x == 0u && pc.cut) pc.cut[blockIdx.x] = make_uint4(0u, 0u, 0u, 0u);
        if (__any_sync(0xffffffffu, again && ok)) {   // (EXACT: both warps of the rows know, and take half of them each)
            __syncwarp();
            seen_keys_rows<C, L::ROWS>(pc, st, s_pref, 0u, g * kGroupRows + (warp & 3u) * 32u + part * 16u, 32u / L::PARTS);
        }
    }
    // (one place for all roles: copies of it in each made a prompt of 4096 with 32-bit results 200 us instead of 164)
    drain_ring(bar0, asked0, depth);
    drain_ring(bar1, asked1, depth);
    tc_fence_before();
    __syncthreads();
    if (warp == L::MMA) tmem_dealloc<false>(tmem, L::TMEM);
}

template <int D, bool EXACT>
static bool launch_tc_t(const LaunchArgs& a, const Args& pc, const Maps& maps, uint32_t ctas) {
    if (!ensure_dynamic_smem<paged_tc_kernel<D, EXACT>>((int)Tc<D, EXACT>::smem(kMaxSeqs))) return false;
    launch_pdl(paged_tc_kernel<D, EXACT>, dim3(ctas), dim3(Tc<D, EXACT>::THREADS), Tc<D, EXACT>::smem(pc.prefix ? 1u : pc.n_seqs), a.stream, maps.k, maps.v, maps.q, pc);
    return true;
}

bool launch_tc(const LaunchArgs& a, const Args& pc, const Maps& maps, uint32_t head_dim, uint32_t ctas, bool exact) {
    return head_dim == 64u ? (exact ? launch_tc_t<64, true>(a, pc, maps, ctas) : launch_tc_t<64, false>(a, pc, maps, ctas))
                           : (exact ? launch_tc_t<128, true>(a, pc, maps, ctas) : launch_tc_t<128, false>(a, pc, maps, ctas));
}

}  // namespace paged
}  // namespace amv
