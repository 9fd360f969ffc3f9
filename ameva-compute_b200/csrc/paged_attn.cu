// Attention over a paged KV cache (paged.cuh): ameva_paged_attn, and ameva_paged_prefix_attn for a batch that shares the pages of a
// long prefix. Here: the kernel for few rows per sequence (tokens, drafts), the merge kernel and the launchers; many rows per
// sequence (prompts, the prefix of a batch) run in paged_tc.cu.
//
// paged_rows_kernel: W + 1 warps. The last one streams key tiles (KB x 32 keys of HB KV heads; K and V in turn) through a ring in shared
// memory with TMA, a box of 64 columns x 16 keys x HB heads each, and runs ahead across the pieces of the CTA's stretch, so that the
// reads never pause. Each of the others takes one head and 32 keys of every tile for the row tile's 16 rows: both products on
// mma.sync (f16 in, f32 out), an online softmax per row to base 2, the scores' accumulators reused as the A operand of the second
// product. With W = HB (eight KV heads, say) a warp owns its head's rows from the first key to the last and the warps never meet; with
// fewer heads the KB warps of a head are joined pairwise through shared memory at the end of a piece. All heads of a block of keys are
// read together because in a cache with a token's heads beside one another they are one run of memory: a head at a time (a warp per
// 16 keys of a tile of 128) took 195 us for 96 sequences of 20 to 8192 keys, 8 KV heads of 128, 160 k keys, as against 100 us for the
// bytes, and 8 us per (sequence, head). P enters the second product as an f16 value and its remainder (rounded once, 2^-12 of every
// probability would show in an f32 result, and makes an f16 one's error 1.25 to 1.4 times what its own rounding is; the second product costs 2 %
// of the time above), and the matrix instruction's sums, which are cut rather than rounded, are added up per 32 keys by ordinary
// additions: left in its accumulator from the first key to the last, 131072 keys are off by 2.3e-6 instead of 4e-7.
// Bound by HBM, short calls by the instructions that a CTA fetches for the first time: those 96 sequences 119 us (659 MB, 5.5 TB/s; the copy
// reaches 6.55), one of 131072 keys 103 us (537 MB, 5.2 TB/s), one of 500 keys 18 us (this kernel 8, the merge 5).
#include <cmath>
#include <cstring>
#include <type_traits>

#include "paged.h"
#include "sync_ptx.cuh"
#include "tcgen05_ptx.cuh"
#include "tensor_map.h"

namespace amv {
namespace paged {

using namespace ptx;

template <int D>
struct Rows {
    static constexpr uint32_t W = D == 256 ? 4 : 8, THREADS = D == 256 ? 160 : 384, ATOMS = D / 64, MAX_STAGES = 8;
    static constexpr uint32_t RING = 196608u;                          // K and V tiles in turn: three of 64 KB where all warps have work
    static constexpr uint32_t MERGE = (W / 2) * 8u * (D + 4u) * 4u;    // half the warps' results for eight rows
    static constexpr uint32_t FIXED = 1024u + RING + MERGE + 128u + 16u * MAX_STAGES;
    // Registers a thread after the split between the warps that multiply and the warpgroup of the one that loads (D 64, 128): 256 x 208 +
    // 128 x 88 = 384 x 168, what the block is launched with.
    static constexpr bool SPLIT = D != 256;
    static constexpr uint32_t smem(uint32_t n_seqs) { return FIXED + (n_seqs + 1u) * 4u; }
};
// How W warps share HB heads: warps (32 keys each) per head and tile, a power of two
__host__ __device__ constexpr uint32_t blocks_of(uint32_t W, uint32_t HB) { return W >= 8u * HB ? 8u : W >= 4u * HB ? 4u : W >= 2u * HB ? 2u : 1u; }

__device__ __forceinline__ void ldsm_x4(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at));
}
__device__ __forceinline__ void ldsm_x4_trans(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(at));
}
// D (16 x 8, f32) += A (16 x 16, f16) * B (16 x 8, f16)
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t halves(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void tma_page(uint32_t dst, const CUtensorMap* map, uint32_t bar, int column, int token, int head, int page) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst), "l"(map),
        "r"(bar), "r"(column), "r"(token), "r"(head), "r"(page)
        : "memory");
}
template <uint32_t THREADS>
__device__ __forceinline__ void worker_sync() {   // the warps that multiply, not the one that loads
    asm volatile("bar.sync 1, %0;" ::"n"(THREADS) : "memory");
}

// Result of a row whose columns 8 nt + 2 t4 + {0, 1} the four lanes of its MMA fragment hold: as finish_row (paged.cuh).
template <int NT>
__device__ __forceinline__ void finish_fragment(const Args& pc, uint32_t token, uint32_t head, uint32_t t4, float m, float l, const float (&oc)[NT][4],
                                                uint32_t h) {
    constexpr uint32_t D = 8u * NT;
    const float* extra = nullptr;
    float f = 1.0f, g = 0.0f;
    if (pc.extra) {
        extra = pc.extra + ((uint64_t)token * pc.n_head + head) * (D + 4u);
        const float2 ml = *reinterpret_cast<const float2*>(extra);
        const float top = fmaxf(m, ml.x);
        f = weight(m, top);
        g = weight(ml.x, top);
        l = l * f + ml.y * g;
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    const uint64_t at = dst_row(pc, token, head, D) + 2u * t4;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        float2 y = make_float2(f != 0.0f ? oc[nt][2u * h] * f : 0.0f, f != 0.0f ? oc[nt][2u * h + 1u] * f : 0.0f);
        if (extra && g != 0.0f) {
            const float2 e = *reinterpret_cast<const float2*>(extra + 4u + 8u * nt + 2u * t4);
            y.x = fmaf(e.x, g, y.x);
            y.y = fmaf(e.y, g, y.y);
        }
        if (inv == 0.0f) y = make_float2(0.0f, 0.0f);
        if (pc.out == OUT_F16) *reinterpret_cast<__half2*>(reinterpret_cast<__half*>(pc.dst) + at + 8u * nt) = __floats2half2_rn(y.x * inv, y.y * inv);
        else *reinterpret_cast<float2*>(reinterpret_cast<float*>(pc.dst) + at + 8u * nt) = make_float2(y.x * inv, y.y * inv);
    }
}
template <int NT>
__device__ __forceinline__ void store_part(float* row, uint32_t t4, float m, float l, const float (&oc)[NT][4], uint32_t h) {
    if (t4 == 0u) *reinterpret_cast<float2*>(row) = make_float2(m, l);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) *reinterpret_cast<float2*>(row + 4u + 8u * nt + 2u * t4) = make_float2(oc[nt][2u * h], oc[nt][2u * h + 1u]);
}

// TOP: every row tile has at most eight rows (the upper half of the MMA tile), so the lower half's work is left out.
template <int D, bool TOP>
__global__ void __launch_bounds__(Rows<D>::THREADS, 1)
paged_rows_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map, const __grid_constant__ Args pc) {
    using L = Rows<D>;
    constexpr uint32_t W = L::W, A = L::ATOMS, C = D / 32, H = TOP ? 1 : 2;   // H: halves of the MMA tile's rows
    constexpr int KS = D / 16, NT = D / 8;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* base = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    float* s_merge = reinterpret_cast<float*>(base + L::RING);                     // [W / 2][8][D + 4]
    uint64_t* bars = reinterpret_cast<uint64_t*>(s_merge + L::MERGE / 4u);         // full, empty
    Ctl* ctl = reinterpret_cast<Ctl*>(bars + 2u * L::MAX_STAGES);
    uint32_t* s_warp = reinterpret_cast<uint32_t*>(ctl + 1);                       // [THREADS / 32]
    uint32_t* s_bad = s_warp + L::THREADS / 32u;                                             // per K tile: 16-key blocks whose page is none
    uint32_t* s_pref = s_bad + L::MAX_STAGES;
    const uint32_t full = smem_u32(bars), empty = full + 8u * L::MAX_STAGES;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
    const uint32_t HB = pc.HB, KB = 1u << (pc.keys_log2 - 5u), atom = HB * 2048u;   // atom: 16 keys x 64 columns of the heads
    const uint32_t tile = 2u * KB * A * atom, stages = min(L::MAX_STAGES, L::RING / tile);
    if (threadIdx.x == 0) {
        for (uint32_t s = 0; s < L::MAX_STAGES; ++s) {
            mbar_init(full + 8u * s, 1u);
            mbar_init(empty + 8u * s, W);
        }
        ctl->abort = 0u;
        fence_barrier_init();
    }
    pdl_trigger();
    pdl_wait();
    const uint32_t total = build_line<kDecRows, L::THREADS / 32u>(pc, s_pref, s_warp);   // (its barriers publish the ones above)
    const Stretch st = my_stretch(total);
    Walk<kDecRows> walk(st);
    Ring ring(stages);
    bool ok = true;

    if (warp >= W) {   // ---- loads ----
        if constexpr (L::SPLIT) asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
        if (warp != W) return;   // (they fill the warpgroup)
        const uint32_t mask = (1u << pc.page_log2) - 1u;
        uint32_t issued = 0;
        while (ok && walk.next(pc, s_pref)) {
            const Piece& p = walk.p;
            const uint32_t lo = row_span(pc, p.q, p.r0).lo, hi = row_span(pc, p.q, min(p.r0 + kDecRows, p.R) - 1u).hi;
            for (uint32_t i = p.a; ok && i < p.b; ++i) {
                const uint32_t key0 = (p.first + i) << pc.keys_log2;
                // lanes b < 2 KB look block b's page up; blocks that hold a key somebody sees are loaded, 64 columns by lane b + 2 KB j
                const uint32_t blocks = 2u * KB, b = lane & (blocks - 1u), b0 = key0 + 16u * b;
                const bool want = b0 < hi && b0 + 16u > lo;
                const int32_t page = want ? page_of(pc, p.q, b0) : -1;
                const uint32_t ours = (1u << blocks) - 1u;
                const uint32_t none = __ballot_sync(0xffffffffu, want && page < 0) & ours, load = __ballot_sync(0xffffffffu, page >= 0) & ours;
                if (none && lane == 0u) refuse(pc, __popc(none));
                for (uint32_t kv = 0; kv < 2u; ++kv) {
                    ok = wait_on(empty + 8u * ring.idx, ring.phase ^ 1u, ctl, pc.status, 0xC00u);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    const uint32_t stage = smem_u32(base) + ring.idx * tile, bar = full + 8u * ring.idx;
                    if (lane == 0u) {
                        s_bad[ring.idx] = none;
                        mbar_arrive_expect_tx(bar, (uint32_t)__popc(load) * A * atom);
                    }
                    __syncwarp();
                    for (uint32_t a = lane / blocks; a < A; a += 32u / blocks)
                        if (page >= 0)
                            tma_page(stage + (b * A + a) * atom, kv ? &v_map : &k_map, bar, (int)(64u * a), (int)(b0 & mask), (int)(p.group * HB), page);
                    ++issued;
                    ring.advance();
                }
            }
        }
        drain_ring(full, issued, stages);
        return;
    }

    if constexpr (L::SPLIT) asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    // ---- products: head `hb` of the group, keys 32 kb .. of the tile ----
    const uint32_t kb = warp / HB, hb = warp - kb * HB;
    const uint32_t g = lane >> 2, t4 = lane & 3u;
    const uint32_t lm_row = (lane & 7u) + ((lane >> 4) << 3), lm_hi = (lane >> 3) & 1u;   // K: key in the block, upper eight columns
    const uint32_t lv_row = (lane & 7u) + (((lane >> 3) & 1u) << 3), lv_nt = lane >> 4;    // V: key in the block, second n-tile
    bool cut = false, again = false;   // again: rows that are not finite although their sum is
    while (walk.next(pc, s_pref)) {
        const Piece& p = walk.p;
        const uint32_t hkv = p.group * HB + hb;
        const bool mine = kb < KB && hkv < pc.n_head_kv;
        const uint32_t rows = min(kDecRows, p.R - p.r0);
        const uint32_t lo_all = row_span(pc, p.q, p.r0).lo, hi_all = row_span(pc, p.q, p.r0 + rows - 1u).hi;     // keys that some row sees
        const uint32_t lo_both = row_span(pc, p.q, p.r0 + rows - 1u).lo, hi_both = row_span(pc, p.q, p.r0).hi;   // keys that every row sees
        Span span[2];
        uint32_t token[2], head[2];
        bool valid[2];
        uint32_t qa[KS][4];
#pragma unroll
        for (uint32_t h = 0; h < 2u; ++h) {
            const uint32_t r = p.r0 + g + 8u * h;
            valid[h] = mine && g + 8u * h < rows;
            span[h] = valid[h] ? row_span(pc, p.q, r) : Span{0u, 0u};
            const uint32_t query = query_of(pc, r);
            token[h] = p.q.tok0 + (valid[h] ? query : 0u);
            head[h] = valid[h] ? hkv * pc.G + r - query * pc.G : 0u;
            const __half* qrow = pc.q + (uint64_t)token[h] * pc.q_s + (uint64_t)head[h] * D;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                const uint32_t c = 16u * ks + 2u * t4;
                qa[ks][h] = valid[h] ? *reinterpret_cast<const uint32_t*>(qrow + c) : 0u;
                qa[ks][2u + h] = valid[h] ? *reinterpret_cast<const uint32_t*>(qrow + c + 8u) : 0u;
            }
        }
        float oc[NT][4], m_run[2] = {neg_inf(), neg_inf()}, l_run[2] = {0.0f, 0.0f};
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int j = 0; j < 4; ++j) oc[nt][j] = 0.0f;

        for (uint32_t i = p.a; i < p.b; ++i) {
            const uint32_t key0 = ((p.first + i) << pc.keys_log2) + 32u * kb;
            ok = ok && wait_on(full + 8u * ring.idx, ring.phase, ctl, pc.status, 0xC20u);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;   // (the pieces are walked to the end all the same: the warps meet at their barriers)
            // a tile: [block of 16 keys][64 columns][head][16 keys][128 bytes, swizzled]
            const uint32_t mine_at = 2u * kb * A * atom + hb * 2048u, tk = smem_u32(base) + ring.idx * tile + mine_at, gone = s_bad[ring.idx] >> (2u * kb);
            bool seen[2];
#pragma unroll
            for (uint32_t kk = 0; kk < 2u; ++kk)
                seen[kk] = mine && key0 + 16u * kk < hi_all && key0 + 16u * kk + 16u > lo_all && !(gone >> kk & 1u);
            float sc[4][4];
#pragma unroll
            for (int nt = 0; nt < 4; ++nt)
#pragma unroll
                for (int j = 0; j < 4; ++j) sc[nt][j] = 0.0f;
            if (seen[0] || seen[1]) {
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    const uint32_t piece = 2u * (ks & 3) + lm_hi;
#pragma unroll
                    for (int kk = 0; kk < 2; ++kk) {   // (of a block that is not there: whatever the memory holds, hidden below)
                        uint32_t b[4];
                        ldsm_x4(b, tk + (kk * A + (ks >> 2)) * atom + lm_row * 128u + ((piece ^ (lm_row & 7u)) << 4));
                        mma16816(sc[2 * kk], qa[ks], b[0], b[1]);
                        mma16816(sc[2 * kk + 1], qa[ks], b[2], b[3]);
                    }
                }
            }
            __syncwarp();
            if (lane == 0u) mbar_arrive(empty + 8u * ring.idx);
            ring.advance();
            uint32_t ph[2][4], pl[2][4];
            if (seen[0] || seen[1]) {
                const bool plain = key0 >= lo_both && key0 + 32u <= hi_both && !(gone & 3u);
#pragma unroll
                for (uint32_t h = 0; h < 2u; ++h) {
                    if (h >= H) {
#pragma unroll
                        for (uint32_t kk = 0; kk < 2u; ++kk) ph[kk][1] = ph[kk][3] = pl[kk][1] = pl[kk][3] = 0u;
                        break;
                    }
                    float x[8], mx = neg_inf();   // 2 nt + j
#pragma unroll
                    for (uint32_t i = 0; i < 8u; ++i) x[i] = sc[i >> 1][2u * h + (i & 1u)];
                    capped(pc, x);
#pragma unroll
                    for (uint32_t i = 0; i < 8u; ++i) {
                        const uint32_t key = key0 + 8u * (i >> 1) + 2u * t4 + (i & 1u);
                        x[i] = plain || (key >= span[h].lo && key < span[h].hi && seen[i >> 2]) ? x[i] : neg_inf();
                        mx = fmaxf(mx, x[i]);
                    }
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                    const float m_new = fmaxf(m_run[h], mx);
                    if (__any_sync(0xffffffffu, m_new != m_run[h])) {
                        const float f = weight(m_run[h], m_new);
                        l_run[h] *= f;
                        m_run[h] = m_new;
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            oc[nt][2u * h] *= f;
                            oc[nt][2u * h + 1u] *= f;
                        }
                    }
                    const float ref = m_new == neg_inf() ? 0.0f : m_new;
                    float sum = 0.0f;
#pragma unroll
                    for (uint32_t nt = 0; nt < 4u; ++nt) {
                        const float p0 = ex2(x[2u * nt] - ref), p1 = ex2(x[2u * nt + 1u] - ref);
                        sum += p0 + p1;
                        const __half2 hi2 = __floats2half2_rn(p0, p1);
                        ph[nt >> 1][2u * (nt & 1u) + h] = *reinterpret_cast<const uint32_t*>(&hi2);
                        const float2 f2 = __half22float2(hi2);
                        pl[nt >> 1][2u * (nt & 1u) + h] = halves(p0 - f2.x, p1 - f2.y);
                    }
                    l_run[h] += sum;   // (this lane's keys; the four lanes of a row are added at the end)
                }
            }
            ok = ok && wait_on(full + 8u * ring.idx, ring.phase, ctl, pc.status, 0xC30u);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            const uint32_t tv = smem_u32(base) + ring.idx * tile + mine_at;
#pragma unroll
            for (uint32_t kk = 0; kk < 2u; ++kk) {
                const uint32_t k0 = key0 + 16u * kk;
                // V rows behind the last key are whatever the page holds there: probabilities of zero do not hide a NaN
                if (seen[kk] && k0 + 16u > hi_all) {
                    const uint32_t from = hi_all - k0;   // 1 .. 15
                    for (uint32_t j = lane; j < (16u - from) * (D / 8u); j += 32u) {
                        const uint32_t r = from + j / (D / 8u), c = j % (D / 8u);
                        asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(tv + kk * A * atom + (c >> 3) * atom + r * 128u + ((c & 7u) << 4)), "r"(0u)
                                     : "memory");
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // (before TMA writes there again)
                    __syncwarp();
                }
            }
#pragma unroll
            for (int np = 0; np < NT / 2; ++np) {   // columns 16 np .. 16 np + 15
                if (!seen[0] && !seen[1]) break;
                const uint32_t piece = 2u * (np & 3) + lv_nt;
                float acc[2][4] = {};   // this tile's sum
#pragma unroll
                for (uint32_t kk = 0; kk < 2u; ++kk) {
                    if (!seen[kk]) continue;
                    uint32_t b[4];
                    ldsm_x4_trans(b, tv + kk * A * atom + (np >> 2) * atom + lv_row * 128u + ((piece ^ (lv_row & 7u)) << 4));
                    mma16816(acc[0], ph[kk], b[0], b[1]);
                    mma16816(acc[1], ph[kk], b[2], b[3]);
                    mma16816(acc[0], pl[kk], b[0], b[1]);
                    mma16816(acc[1], pl[kk], b[2], b[3]);
                }
#pragma unroll
                for (uint32_t n = 0; n < 2u; ++n)
#pragma unroll
                    for (uint32_t c = 0; c < 2u * H; ++c) oc[2 * np + n][c] += acc[n][c];
            }
            __syncwarp();
            if (lane == 0u) mbar_arrive(empty + 8u * ring.idx);
            ring.advance();
        }
#pragma unroll
        for (uint32_t h = 0; h < 2u; ++h) {
            l_run[h] += __shfl_xor_sync(0xffffffffu, l_run[h], 1);
            l_run[h] += __shfl_xor_sync(0xffffffffu, l_run[h], 2);
        }
        // ---- the warps of a head as one: the upper half of the blocks hands its rows to the lower, until one is left ----
        for (uint32_t n = KB >> 1; n; n >>= 1) {
#pragma unroll
            for (uint32_t h = 0; h < 2u; ++h) {
                if (h >= H) break;
                float* row = s_merge + (((kb & (n - 1u)) * HB + hb) * 8u + g) * (D + 4u);
                worker_sync<W * 32u>();   // (the rows written before have been read)
                if (mine && kb >= n && kb < 2u * n) store_part<NT>(row, t4, m_run[h], l_run[h], oc, h);
                worker_sync<W * 32u>();
                if (mine && kb < n) {
                    const float2 ml = *reinterpret_cast<const float2*>(row);
                    const float top = fmaxf(m_run[h], ml.x), f0 = weight(m_run[h], top), f1 = weight(ml.x, top);
                    m_run[h] = top;
                    l_run[h] = l_run[h] * f0 + ml.y * f1;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        const float2 y = *reinterpret_cast<const float2*>(row + 4u + 8u * nt + 2u * t4);
                        oc[nt][2u * h] = (f0 != 0.0f ? oc[nt][2u * h] * f0 : 0.0f) + (f1 != 0.0f ? y.x * f1 : 0.0f);
                        oc[nt][2u * h + 1u] = (f0 != 0.0f ? oc[nt][2u * h + 1u] * f0 : 0.0f) + (f1 != 0.0f ? y.y * f1 : 0.0f);
                    }
                }
            }
        }
        // ---- results ----
        if (mine && kb == 0u && ok) {
            const bool whole = p.a == 0u && p.b == p.n;
            float* slot = pc.slots + ((uint64_t)(2u * blockIdx.x + (p.a == 0u ? 1u : 0u)) * HB + hb) * kDecRows * (D + 4u);
#pragma unroll
            for (uint32_t h = 0; h < 2u; ++h) {
                if (h >= H) break;
                float check = 0.0f;   // NaN once a column is not finite
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) check = fmaf(oc[nt][2u * h], 0.0f, fmaf(oc[nt][2u * h + 1u], 0.0f, check));
                check += __shfl_xor_sync(0xffffffffu, check, 1);
                check += __shfl_xor_sync(0xffffffffu, check, 2);
                // (a sum that is not finite says that the scores are not: the row is NaN either way)
                again = again || (valid[h] && check != 0.0f && l_run[h] - l_run[h] == 0.0f);
                if (valid[h]) {
                    if (whole && pc.out != OUT_PARTS) finish_fragment<NT>(pc, token[h], head[h], t4, m_run[h], l_run[h], oc, h);
                    else
                        store_part<NT>(whole ? reinterpret_cast<float*>(pc.dst) + dst_row(pc, token[h], head[h], D) : slot + (uint64_t)(g + 8u * h) * (D + 4u),
                                       t4, m_run[h], l_run[h], oc, h);
                }
            }
        }
        if (p.a == 0u && p.b < p.n) {
            cut = true;
            if (threadIdx.x == 0u) note_cut(pc, st, p, rows);
        }
    }
    if (!cut && threadIdx.x == 0u && pc.cut) pc.cut[blockIdx.x] = make_uint4(0u, 0u, 0u, 0u);
    if (__any_sync(0xffffffffu, again && ok)) {
        __syncwarp();   // (the rows that other lanes have stored are read)
        seen_keys_rows<C, kDecRows>(pc, st, s_pref, hb, 0u, kDecRows);
    }
}

// Joins the cut row tiles. CTA x of the kernel in front notes a row tile that it begins and others end; its parts lie in slot 2 x + 1 and
// in slots 2 y of the CTAs behind. The rows of a kernel's notes form one list that the warps of the grid share;
// `share` warps take the parts of a row in turn, the more the more parts there are (a long sequence alone has one per SM). Bound by latency:
// 5 us for the 32 rows of one token, 16 us for 24 mixed sequences of 535 tokens.
constexpr uint32_t kMergeWarps = 16, kMergeNotes = 512;
struct MergeSet {
    Args pc;
    uint32_t ctas, tile_rows;
};
template <uint32_t C>
__device__ __forceinline__ void load_columns(const float* p, float (&x)[C]) {   // (16 bytes at a time where there are)
    if constexpr (C == 2u) {
        const float2 y = *reinterpret_cast<const float2*>(p);
        x[0] = y.x;
        x[1] = y.y;
    } else {
#pragma unroll
        for (uint32_t c = 0; c < C; c += 4u) {
            const float4 y = *reinterpret_cast<const float4*>(p + c);
            x[c] = y.x;
            x[c + 1u] = y.y;
            x[c + 2u] = y.z;
            x[c + 3u] = y.w;
        }
    }
}
template <uint32_t C>
__device__ __forceinline__ void merge_set(const MergeSet& set) {
    constexpr uint32_t D = 32u * C, ROW = D + 4u, kTogether = C == 8u ? 4u : 8u;
    __shared__ uint4 s_note[kMergeNotes];
    __shared__ uint32_t s_at[kMergeNotes], s_sum[kMergeWarps], s_top[kMergeWarps];   // s_at: rows in front of note i
    __shared__ float s_ml[kMergeWarps][2], s_o[kMergeWarps][D];
    const Args& pc = set.pc;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u, notes = set.ctas;
    uint32_t total = 0, most = 0;
    for (uint32_t base = 0; base < notes; base += kMergeWarps * 32u) {   // exclusive sums, a note per thread
        const uint32_t i = base + threadIdx.x;
        uint32_t rows = 0, parts = 0;
        if (i < notes) {
            const uint4 note = pc.cut[i];
            s_note[i] = note;
            parts = note.x & 0xFFFFu;
            if (parts) rows = min(pc.HB, pc.n_head_kv - (note.x >> 16) * pc.HB) * note.w;
        }
        uint32_t incl = rows, top = parts;
#pragma unroll
        for (uint32_t o = 1; o < 32u; o <<= 1) {
            const uint32_t up = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += up;
            top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
        }
        if (lane == 31u) {
            s_sum[warp] = incl;
            s_top[warp] = top;
        }
        __syncthreads();
        uint32_t before = total + incl - rows;
#pragma unroll
        for (uint32_t w = 0; w < kMergeWarps; ++w) {
            before += w < warp ? s_sum[w] : 0u;
            total += s_sum[w];
            most = max(most, s_top[w]);
        }
        if (i < notes) s_at[i] = before;
        __syncthreads();
    }
    const uint32_t share = most <= 8u ? 1u : most <= 16u ? 2u : most <= 32u ? 4u : most <= 64u ? 8u : kMergeWarps, at_once = kMergeWarps / share;
    const uint32_t begin = warp % share;
    // rows beside one another to a warp (they mostly share their note), `per` of them
    const uint32_t per = (total + gridDim.x * at_once - 1u) / (gridDim.x * at_once), first = (blockIdx.x * at_once + warp / share) * per;
    uint32_t note_i = 0, note_end = 0, group = 0;
    uint4 note = make_uint4(0u, 0u, 0u, 1u);
    for (uint32_t k = 0; k < per; ++k) {
        const uint32_t at = first + k;
        const bool have_row = at < total;
        if (have_row && at >= note_end) {
            uint32_t lo = 0, hi = notes;   // the last note with s_at <= at (of equal ones the last, which has the rows)
            while (hi - lo > 1u) {
                const uint32_t mid = (lo + hi) >> 1;
                if (s_at[mid] <= at) lo = mid;
                else hi = mid;
            }
            note_i = lo;
            note_end = lo + 1u < notes ? s_at[lo + 1u] : total;
            note = s_note[lo];
            group = note.x >> 16;
        }
        const uint32_t parts = note.x & 0xFFFFu, i_row = have_row ? at - s_at[note_i] : 0u, hb = i_row / note.w, r = i_row - hb * note.w;
        float m = neg_inf(), l = 0.0f, o[C];
#pragma unroll
        for (uint32_t c = 0; c < C; ++c) o[c] = 0.0f;
        auto part = [&](uint32_t i) { return pc.slots + (((uint64_t)(i == 0u ? 2u * note_i + 1u : 2u * (note_i + i)) * pc.HB + hb) * set.tile_rows + r) * ROW; };
        auto take = [&](auto n_const, uint32_t i0) {   // some parts on their way together
            constexpr uint32_t N = decltype(n_const)::value;
            float x[N][C], ml[N][2], top = m;
#pragma unroll
            for (uint32_t j = 0; j < N; ++j) {
                const uint32_t i = i0 + j * share;
                const bool have = i < parts;
                const float* p = part(have ? i : begin);
                const float2 v = *reinterpret_cast<const float2*>(p);
                ml[j][0] = have ? v.x : neg_inf();
                ml[j][1] = have ? v.y : 0.0f;
                load_columns<C>(p + 4u + C * lane, x[j]);
            }
#pragma unroll
            for (uint32_t j = 0; j < N; ++j) top = fmaxf(top, ml[j][0]);
            const float f0 = weight(m, top);
            m = top;
            l *= f0;
#pragma unroll
            for (uint32_t c = 0; c < C; ++c) o[c] *= f0;
#pragma unroll
            for (uint32_t j = 0; j < N; ++j) {
                const float f = weight(ml[j][0], top);
                l = fmaf(ml[j][1], f, l);
#pragma unroll
                for (uint32_t c = 0; c < C; ++c) o[c] += f != 0.0f ? x[j][c] * f : 0.0f;
            }
        };
        if (have_row && begin < parts) {
            if (parts <= 2u * share) take(std::integral_constant<uint32_t, 2>(), begin);
            else if (parts <= 4u * share) take(std::integral_constant<uint32_t, 4>(), begin);
            else
                for (uint32_t i0 = begin; i0 < parts; i0 += kTogether * share) take(std::integral_constant<uint32_t, kTogether>(), i0);
        }
        if (share > 1u) {
            if (lane == 0u) {
                s_ml[warp][0] = m;
                s_ml[warp][1] = l;
            }
#pragma unroll
            for (uint32_t c = 0; c < C; ++c) s_o[warp][C * lane + c] = o[c];
            __syncthreads();
            if (begin == 0u && have_row) {
                m = neg_inf();
                for (uint32_t w = warp; w < warp + share; ++w) m = fmaxf(m, s_ml[w][0]);
                l = 0.0f;
#pragma unroll
                for (uint32_t c = 0; c < C; ++c) o[c] = 0.0f;
                for (uint32_t w = warp; w < warp + share; ++w) {
                    const float f = weight(s_ml[w][0], m);
                    l = fmaf(s_ml[w][1], f, l);
#pragma unroll
                    for (uint32_t c = 0; c < C; ++c) o[c] += f != 0.0f ? s_o[w][C * lane + c] * f : 0.0f;
                }
            }
            __syncthreads();
            if (begin != 0u) continue;
        }
        if (have_row) {
            const uint32_t row = note.z + r, query = query_of(pc, row);
            finish_row<C>(pc, note.y + query, (group * pc.HB + hb) * pc.G + row - query * pc.G, m, l, o);
        }
    }
    __syncthreads();   // (the memory is used again)
}
template <uint32_t C>
__global__ void __launch_bounds__(kMergeWarps * 32, 2) paged_merge_kernel(const __grid_constant__ MergeSet s0, const __grid_constant__ MergeSet s1) {
    pdl_trigger();
    pdl_wait();
    if (s0.ctas) merge_set<C>(s0);
    if (s1.ctas) merge_set<C>(s1);
}

template <int D, bool TOP>
static bool launch_rows_t(const LaunchArgs& a, const Args& pc, const Maps& maps, uint32_t ctas) {
    if (!ensure_dynamic_smem<paged_rows_kernel<D, TOP>>((int)Rows<D>::smem(kMaxSeqs))) return false;
    launch_pdl(paged_rows_kernel<D, TOP>, dim3(ctas), dim3(Rows<D>::THREADS), Rows<D>::smem(pc.prefix ? 1u : pc.n_seqs), a.stream, maps.k, maps.v, pc);
    return true;
}
template <int D>
static bool launch_rows_d(const LaunchArgs& a, const Args& pc, const Maps& maps, uint32_t ctas) {
    return (uint64_t)pc.max_q * pc.G <= 8u ? launch_rows_t<D, true>(a, pc, maps, ctas) : launch_rows_t<D, false>(a, pc, maps, ctas);
}
static bool launch_rows(const LaunchArgs& a, const Args& pc, const Maps& maps, uint32_t D, uint32_t ctas) {
    return D == 64u ? launch_rows_d<64>(a, pc, maps, ctas) : D == 128u ? launch_rows_d<128>(a, pc, maps, ctas) : launch_rows_d<256>(a, pc, maps, ctas);
}

static bool launch_merge(const LaunchArgs& a, const Args& x, const Args& y, uint32_t D, uint32_t n_x, uint32_t n_y, uint32_t rows_x, uint32_t rows_y) {
    const MergeSet s0 = {x, n_x, rows_x}, s1 = {y, n_y, rows_y};
    if (n_x > kMergeNotes || n_y > kMergeNotes) return false;
    const uint64_t rows = (uint64_t)x.rows * x.n_head, most = 2u * (uint32_t)a.sm_count;   // (no row is cut twice)
    const dim3 grid((uint32_t)(rows < most ? rows : most)), block(kMergeWarps * 32);
    if (D == 64u) launch_pdl(paged_merge_kernel<2>, grid, block, 0, a.stream, s0, s1);
    else if (D == 128u) launch_pdl(paged_merge_kernel<4>, grid, block, 0, a.stream, s0, s1);
    else launch_pdl(paged_merge_kernel<8>, grid, block, 0, a.stream, s0, s1);
    return true;
}

// [pages][heads][tokens][D] f16 with the caller's strides, boxes of 64 columns x `tokens` x `heads`
static bool encode_cache(tc::EncodeTiledFn enc, CUtensorMap* map, const void* ptr, const Args& pc, uint32_t D, uint32_t tokens, uint32_t heads) {
    const uint32_t P = 1u << pc.page_log2;
    const cuuint64_t dims[4] = {D, P, pc.n_head_kv, pc.n_pages};
    // (the stride of a dimension of one element is never used, but has to be a valid one)
    const cuuint64_t strides[3] = {2ull * pc.c_ts, pc.n_head_kv > 1u ? 2ull * pc.c_hs : 2ull * D, pc.n_pages > 1u ? 2ull * pc.c_ps : 2ull * D};
    const cuuint32_t box[4] = {64, tokens, heads, 1}, estr[4] = {1, 1, 1, 1};
    if (!strides[0] || !strides[1] || !strides[2]) return false;
    return enc(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

static float word_f(uint32_t u) {
    float f;
    memcpy(&f, &u, 4);
    return f;
}
static bool meet(const LaunchArgs& a, uint32_t i, uint32_t j) {
    const uintptr_t p = (uintptr_t)a.ptr[i], q = (uintptr_t)a.ptr[j];
    return p < q + a.range[j] && q < p + a.range[i];
}

// What both entry points' arguments have in common: the first 18 push words and bindings 0 .. 8.
static AcResult read_args(const LaunchArgs& a, Args& pc, uint32_t& D) {
    const uint32_t* w = a.push;
    memset(&pc, 0, sizeof(pc));
    D = w[0];
    pc.n_head = w[1];
    pc.n_head_kv = w[2];
    pc.n_seqs = w[3];
    pc.rows = w[4];
    pc.max_q = w[5];
    pc.max_kv = w[6];
    const uint32_t P = w[7];
    pc.n_pages = w[8];
    pc.table_stride = w[9];
    pc.c_ps = w[10];
    pc.c_ts = w[11];
    pc.c_hs = w[12];
    pc.q_s = w[13];
    pc.dst_s = w[14];
    pc.out = w[15];
    pc.scale = word_f(w[16]);
    pc.softcap = word_f(w[17]);
    pc.scale2 = pc.scale * kLog2e;
    if (pc.softcap > 0.0f) {
        pc.cap_in = pc.scale / pc.softcap;
        pc.cap_out = pc.softcap * kLog2e;
    }
    if (!D || !pc.n_head || !pc.n_head_kv || pc.n_head % pc.n_head_kv || !pc.n_seqs || !pc.rows || !pc.max_q || !pc.max_kv || !P || (P & (P - 1u)) ||
        !pc.n_pages || !pc.table_stride || pc.out > OUT_F16 || !(pc.softcap >= 0.0f))
        return AC_ERR_KERNEL_ARG_INVALID;
    // what scores are multiplied by is finite (a score of 0 would be NaN otherwise)
    for (float x : {pc.scale, pc.scale2, pc.softcap, pc.cap_in, pc.cap_out})
        if (!std::isfinite(x)) return AC_ERR_KERNEL_ARG_INVALID;
    set_group(pc, pc.n_head / pc.n_head_kv);
    if ((D != 64u && D != 128u && D != 256u) || P < 16u || P > 1024u) return AC_ERR_FEATURE_NOT_SUPPORTED;
    for (pc.page_log2 = 0; (1u << pc.page_log2) < P; ++pc.page_log2) {}
    if (pc.n_seqs > kMaxSeqs || pc.n_head > 65535u || pc.rows > 0x7FFFFFFFu || pc.max_kv > 0x7FFFFFFFu - 1024u || pc.n_pages > 0x7FFFFFFFu ||
        (uint64_t)pc.rows * pc.n_head > 0x7FFFFFFFull || (uint64_t)pc.table_stride * P > 0x7FFFFFFFull)
        return AC_ERR_INVALID_SHAPE;
    if (pc.max_q > pc.rows) pc.max_q = pc.rows;
    if (((pc.c_ps | pc.c_ts | pc.c_hs | pc.q_s) & 7u) || (pc.dst_s & (pc.out == OUT_F16 ? 7u : 3u))) return AC_ERR_BUFFER_ALIGNMENT_INVALID;
    for (uint32_t i : {0u, 1u, 2u, 6u, 7u})
        if ((uintptr_t)a.ptr[i] & 15u) return AC_ERR_BUFFER_ALIGNMENT_INVALID;
    for (uint32_t i : {3u, 4u, 5u, 8u})
        if ((uintptr_t)a.ptr[i] & 3u) return AC_ERR_BUFFER_ALIGNMENT_INVALID;
    const uint64_t last = pc.rows - 1u, width = (uint64_t)pc.n_head * D, esize = pc.out == OUT_F16 ? 2u : 4u;
    const uint64_t cache = ((uint64_t)(pc.n_pages - 1u) * pc.c_ps + (uint64_t)(P - 1u) * pc.c_ts + (uint64_t)(pc.n_head_kv - 1u) * pc.c_hs + D) * 2u;
    if (a.range[0] < (last * pc.q_s + width) * 2u || a.range[1] < cache || a.range[2] < cache ||
        a.range[3] < (uint64_t)pc.n_seqs * pc.table_stride * 4u || a.range[4] < ((uint64_t)pc.n_seqs + 1u) * 4u || a.range[5] < (uint64_t)pc.n_seqs * 4u ||
        a.range[6] < (last * pc.dst_s + width) * esize || a.range[8] < 8u)
        return AC_ERR_INVALID_BUFFER_SIZE;
    if (last && pc.dst_s < width) return AC_ERR_INVALID_SHAPE;   // rows of the result that overlap
    for (uint32_t o : {6u, 7u, 8u})   // what is written meets nothing else
        for (uint32_t i = 0; i < a.binding_count; ++i)
            if (i != o && meet(a, o, i)) return AC_ERR_KERNEL_ARG_INVALID;
    pc.q = (const __half*)a.ptr[0];
    pc.k = (const __half*)a.ptr[1];
    pc.v = (const __half*)a.ptr[2];
    pc.table = (const int32_t*)a.ptr[3];
    pc.q_start = (const int32_t*)a.ptr[4];
    pc.kv_len = (const int32_t*)a.ptr[5];
    pc.dst = a.ptr[6];
    pc.refused = (uint32_t*)a.ptr[8];
    pc.status = a.status;
    return AC_SUCCESS;
}

// Which kernel a sequence of R rows per KV head runs in (D 64, 128; D 256 knows one): paged_rows_kernel reads the keys once per 16 rows, the
// kernel in paged_tc.cu takes the same time for 1 .. 128, but is one more launch where sequences of few rows are beside it. 8 sequences
// of 4000 keys, 8 KV heads, f16 results, a pass in us, rows / tensor-core kernel: 64 rows 97 / 74, 128 rows 159 / 78; 64 of 2000 keys:
// 340 / 185, 620 / 195 (32-bit results: 32 rows 192 / 185, 343 / 186, 620 / 196). 32 sequences of 7 to 42 rows, 2 KV
// heads, 1024 keys: 21 / 46. So up to kFewRows; up to kFewRowsAlone while what the rows beyond add is below what the other launch costs:
// 25 us, in which 360 thousand (row tile, KV head, key) are served.
constexpr uint32_t kFewRows = 32, kFewRowsAlone = 64;
constexpr uint64_t kLaunchWork = 360000;
static uint32_t few_rows_of(const Args& pc, uint32_t D, uint64_t max_rows) {
    if (D > 128u) return 0xFFFFFFFFu;
    if (max_rows > kFewRowsAlone) return kFewRows;
    const uint64_t keys = pc.window && (uint64_t)pc.window + pc.max_q < pc.max_kv ? (uint64_t)pc.window + pc.max_q : pc.max_kv;
    const uint64_t beyond = max_rows > kFewRows ? (max_rows - kFewRows + kDecRows - 1u) / kDecRows : 0u;
    return (pc.prefix ? 1u : pc.n_seqs) * keys * pc.n_head_kv * beyond > kLaunchWork ? kFewRows : kFewRowsAlone;
}
// What a row tile costs beside its key tiles, in key tiles (the line's allowance): Q and the first scores on their way, results written.
// us with none / this: 96 sequences of 20 .. 8192 keys 126 / 119 (1: 121), 32 drafted ones 24.1 / 22.1 (1: 21.5); f16 results before P had its
// remainder: a prompt of 8192 737 / 648 (2: 700, 4: 665, 10: 653, 16: 664), 64 rows behind a prefix of 8192 keys 83.9 / 73.4.
constexpr uint32_t kFewOver = 2, kManyOver = 6;
// KV heads that paged_rows_kernel takes at once: all of them where its warps suffice, otherwise equal groups
static uint32_t few_heads(uint32_t D, uint32_t n_head_kv) {
    const uint32_t W = D == 256u ? 4u : 8u, groups = (n_head_kv + W - 1u) / W;
    return (n_head_kv + groups - 1u) / groups;
}

struct Scratch {   // taken from the front
    uint8_t* at;
    uint64_t left;
    void* take(uint64_t bytes) {
        bytes = (bytes + 255u) & ~255ull;
        if (bytes > left) return nullptr;
        void* p = at;
        at += bytes;
        left -= bytes;
        return p;
    }
};
// CTAs for a kernel whose cut tiles take 2 * tile_bytes of scratch each: as many as the SMs, fewer where the scratch holds no more
static uint32_t ctas_for(uint64_t room, uint64_t tile_bytes, uint32_t sms) {
    const uint64_t n = room > 1024u ? (room - 1024u) / (2u * tile_bytes + 32u) : 0u;
    return n < 1u ? 1u : n > sms ? sms : (uint32_t)n;
}

// One attention over one set of keys: which kernels run, and the line of each.
struct Plan {
    Args few, many;
    bool use_few, use_many;
    uint32_t tc_rows;
    bool short_line;   // the tensor-core kernel's line also fits 32 bits with half the rows a tile
};
static AcResult plan_set(const Args& pc, uint32_t D, uint64_t max_rows, Plan& x) {
    const uint32_t few_max = few_rows_of(pc, D, max_rows);
    const bool both = max_rows > few_max;
    x.few = x.many = pc;
    x.few.min_rows = 1u;
    x.few.max_rows = both ? few_max : 0xFFFFFFFFu;
    x.many.min_rows = pc.prefix ? 1u : few_max + 1u;   // (a prefix has one number of rows, and one kernel)
    x.many.max_rows = 0xFFFFFFFFu;
    x.use_few = !both || !pc.prefix;
    x.use_many = both;
    x.few.report = 1u;                                  // (what both kernels meet is counted by one)
    x.many.report = !x.use_few;
    x.few.HB = few_heads(D, pc.n_head_kv);
    x.few.groups = (pc.n_head_kv + x.few.HB - 1u) / x.few.HB;
    const uint32_t kb = blocks_of(D == 256u ? 4u : 8u, x.few.HB);
    for (x.few.keys_log2 = 5u; (1u << (x.few.keys_log2 - 5u)) < kb; ++x.few.keys_log2) {}
    x.few.over = kFewOver;
    x.many.HB = 1u;
    x.many.groups = pc.n_head_kv;
    x.many.keys_log2 = 6u;
    x.many.over = kManyOver;
    x.tc_rows = pc.out == OUT_F16 ? kTcRows : kTcRows / 2u;   // (paged_tc.cu)
    // the line's length in 32 bits
    const uint64_t few_rows = both ? few_max : max_rows, seqs = pc.prefix ? 1u : pc.n_seqs;
    auto too_long = [&](const Args& y, uint64_t row_tiles) {
        return seqs * y.groups * row_tiles * (((uint64_t)pc.max_kv >> y.keys_log2) + 2u + y.over) > 0xFFFFFFFFull;
    };
    if (x.use_few && too_long(x.few, (few_rows + kDecRows - 1u) / kDecRows)) return AC_ERR_INVALID_SHAPE;
    if (x.use_many && too_long(x.many, (max_rows + x.tc_rows - 1u) / x.tc_rows)) return AC_ERR_INVALID_SHAPE;
    x.short_line = !too_long(x.many, (max_rows + kTcRows / 2u - 1u) / (kTcRows / 2u));
    return AC_SUCCESS;
}
// The sequences of few rows, those of many, and the join of what both cut.
static AcResult launch_set(const LaunchArgs& a, const Plan& x, uint32_t D, Scratch scratch, const Maps& rows_maps, const Maps& tc_maps) {
    const uint32_t sms = a.sm_count > 0 ? (uint32_t)a.sm_count : 148u, tc_rows = x.tc_rows;
    const uint64_t row = (D + 4u) * 4u;
    const bool use_few = x.use_few, use_many = x.use_many;
    Args few = x.few, many = x.many;
    few.q_boxes = many.q_boxes = tc_maps.q_boxes;
    uint32_t n_few = 0, n_many = 0;
    if (use_few) {
        n_few = ctas_for(use_many ? scratch.left * few.HB / (few.HB + 16u) : scratch.left, few.HB * kDecRows * row, sms);
        few.cut = (uint4*)scratch.take(n_few * 16ull);
        few.slots = (float*)scratch.take(n_few > 1u ? 2ull * n_few * few.HB * kDecRows * row : 0u);
        if (!few.cut || !few.slots) n_few = 1u, few.cut = nullptr, few.slots = nullptr;
    }
    if (use_many) {
        n_many = ctas_for(scratch.left, tc_rows * row, sms);
        many.cut = (uint4*)scratch.take(n_many * 16ull);
        many.slots = (float*)scratch.take(2ull * n_many * tc_rows * row);
        if (!many.cut || !many.slots) n_many = 1u, many.cut = nullptr, many.slots = nullptr;
    }
    // f16 results of more keys than one accumulator is to take need a slot to add it to; without, the kernel of 32-bit results rounds them
    const bool exact = many.out != OUT_F16 || (!many.slots && many.max_kv > kRenew * kTcKeys && x.short_line);
    if (use_many && !launch_tc(a, many, tc_maps, D, n_many, exact)) return AC_ERR_INVALID_WORK_GROUP_SIZE;
    if (use_few && !launch_rows(a, few, rows_maps, D, n_few)) return AC_ERR_INVALID_WORK_GROUP_SIZE;
    const uint32_t merge_few = n_few > 1u ? n_few : 0u, merge_many = n_many > 1u ? n_many : 0u;
    if (merge_few + merge_many && !launch_merge(a, few, many, D, merge_few, merge_many, kDecRows, tc_rows)) return AC_ERR_INVALID_WORK_GROUP_SIZE;
    return check_launch();
}

static AcResult cache_maps(const LaunchArgs& a, const Args& pc, uint32_t D, Maps& rows_maps, Maps& tc_maps) {
    tc::EncodeTiledFn enc = tc::encode_fn();
    const uint32_t P = 1u << pc.page_log2, heads = few_heads(D, pc.n_head_kv), tc_box = P < kTcKeys ? P : kTcKeys;
    if (!enc) return AC_ERR_DRIVER_SYMBOL_MISSING;
    const bool ok = encode_cache(enc, &rows_maps.k, a.ptr[1], pc, D, 16u, heads) && encode_cache(enc, &rows_maps.v, a.ptr[2], pc, D, 16u, heads) &&
                    encode_cache(enc, &tc_maps.k, a.ptr[1], pc, D, tc_box, 1u) && encode_cache(enc, &tc_maps.v, a.ptr[2], pc, D, tc_box, 1u);
    if (!ok) return AC_ERR_INVALID_SHAPE;
    memset(&tc_maps.q, 0, sizeof(tc_maps.q));
    // Q by TMA where whole tokens fill a group's 128 rows; otherwise by cp.async, 16 bytes a lane (a prompt of 8192, G = 4, before P had its remainder: 700 / 739 us)
    tc_maps.q_boxes = D <= 128u && (pc.G & (pc.G - 1u)) == 0u && pc.G <= 128u;
    if (tc_maps.q_boxes) {
        const cuuint64_t dims[3] = {D, pc.n_head, pc.rows}, strides[2] = {2ull * D, 2ull * (pc.rows > 1u ? pc.q_s : (uint64_t)pc.n_head * D)};
        const cuuint32_t box[3] = {64, pc.G, 128u / pc.G}, estr[3] = {1, 1, 1};
        tc_maps.q_boxes = strides[1] && enc(&tc_maps.q, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, a.ptr[0], dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                       CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
    }
    return AC_SUCCESS;
}

}  // namespace paged

// ameva_paged_attn: bindings 0 q f16, 1 k cache f16, 2 v cache f16, 3 table i32 [n_seqs][table_stride], 4 q_start i32 [n_seqs + 1],
// 5 kv_len i32 [n_seqs], 6 dst f32 or f16, 7 scratch, 8 status (two words: count of refused entries, lowest node).
// push: D (64, 128, 256), n_head, n_head_kv, n_seqs (<= 4095), rows of q and dst, most rows of a sequence, most keys of one, page size
// (a power of two, 16 .. 1024), pages, table stride, cache strides of page, token and head, row strides of q and dst (in elements),
// dst is f16, scale, softcap (0: none), window (0: none; otherwise a query sees that many keys, its own the last), node.
// Query j of a sequence's n stands at place kv_len - n + j and sees the keys up to there; one that sees none is zero. Rows behind the
// last sequence are left as they are. Sequences whose numbers do not fit the buffers or the announced maxima are left out, keys on
// pages that are none of the cache's are not seen; both are counted. The results do not depend on the scratch's contents, and with the
// same scratch size and maxima not on the run; a larger scratch (up to 2 x SMs x 384 rows of D + 4 floats) allows more CTAs.
AcResult launch_paged_attn(const LaunchArgs& a) {
    using namespace paged;
    Args pc;
    uint32_t D;
    AcResult rc = read_args(a, pc, D);
    if (rc != AC_SUCCESS) return rc;
    pc.window = a.push[18];
    pc.node = a.push[19];
    Plan plan;
    rc = plan_set(pc, D, (uint64_t)pc.max_q * pc.G, plan);
    if (rc != AC_SUCCESS) return rc;
    Maps rows_maps, tc_maps;
    rc = cache_maps(a, pc, D, rows_maps, tc_maps);
    if (rc != AC_SUCCESS) return rc;
    return launch_set(a, plan, D, {(uint8_t*)a.ptr[7], a.range[7]}, rows_maps, tc_maps);
}

// ameva_paged_prefix_attn: the same for sequences that share a prefix, whose pages are read once for all of them (D 64, 128; once per 16 rows,
// D 256). Binding 9: prefix i32
// [1 + pages], its number of keys and its pages; kv_len and the tables are those of the sequences' own keys behind it. push words 18, 19:
// most keys of the prefix, node; no window. The scratch holds rows x n_head x (D + 4) floats at least.
AcResult launch_paged_prefix_attn(const LaunchArgs& a) {
    using namespace paged;
    Args pc;
    uint32_t D;
    AcResult rc = read_args(a, pc, D);
    if (rc != AC_SUCCESS) return rc;
    const uint32_t max_prefix = a.push[18];
    pc.node = a.push[19];
    if (!max_prefix) return AC_ERR_KERNEL_ARG_INVALID;
    if (max_prefix > 0x7FFFFFFFu - 1024u) return AC_ERR_INVALID_SHAPE;
    if ((uintptr_t)a.ptr[9] & 3u) return AC_ERR_BUFFER_ALIGNMENT_INVALID;
    if (a.range[9] < 4u + 4ull * (((uint64_t)max_prefix + (1u << pc.page_log2) - 1u) >> pc.page_log2)) return AC_ERR_INVALID_BUFFER_SIZE;
    Scratch scratch = {(uint8_t*)a.ptr[7], a.range[7]};
    float* own = (float*)scratch.take((uint64_t)pc.rows * pc.n_head * (D + 4u) * 4u);
    if (!own) return AC_ERR_INVALID_BUFFER_SIZE;
    Args first = pc;   // the sequences' own keys
    first.dst = own;
    first.out = OUT_PARTS;
    Plan own_plan, plan;
    rc = plan_set(first, D, (uint64_t)pc.max_q * pc.G, own_plan);
    if (rc != AC_SUCCESS) return rc;
    pc.extra = own;    // the prefix, for all rows at once, with those taken in
    pc.prefix = (const int32_t*)a.ptr[9];
    pc.max_own_q = pc.max_q;
    pc.max_own_kv = pc.max_kv;
    pc.max_q = pc.rows;
    pc.max_kv = max_prefix;
    rc = plan_set(pc, D, (uint64_t)pc.rows * pc.G, plan);
    if (rc != AC_SUCCESS) return rc;
    Maps rows_maps, tc_maps;
    rc = cache_maps(a, pc, D, rows_maps, tc_maps);
    if (rc != AC_SUCCESS) return rc;
    rc = launch_set(a, own_plan, D, scratch, rows_maps, tc_maps);
    return rc != AC_SUCCESS ? rc : launch_set(a, plan, D, scratch, rows_maps, tc_maps);
}

}  // namespace amv
