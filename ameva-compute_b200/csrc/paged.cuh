// What the kernels over a paged KV cache share: the arguments, the sequences of a batch, and how the work of a batch is dealt
// to the CTAs of a grid.
//
// A batch is described on the device (so that a recorded launch serves every step): sequence s has the rows q_start[s] ..
// q_start[s + 1] - 1 of the queries, kv_len[s] keys, its own new ones among them, and its keys' pages in row s of the table.
// Query j of its n stands at place kv_len - n + j and sees the keys up to there (with a window: that many). The shared prefix of
// a batch is one more sequence, of all rows, every one of which sees all of its keys.
//
// The G query heads that share a KV head make R = n * G rows per sequence and KV head (row r: query r / G, head r % G), dealt in
// tiles of ROWS; a row tile walks the key tiles (2^keys_log2 keys each) that any of its rows sees, for the HB KV heads of a group at
// once. All (sequence, head group, row tile, key tile) in this order form one line, and every CTA takes an equal stretch of it,
// whatever the lengths are. What a row tile costs beside its key tiles counts as `over` tiles behind its last. A row tile that lies in one
// stretch is finished there; one that is cut leaves a maximum, a sum and weighted values per row and CTA (at most two per CTA: its
// first and its last piece), which the merge kernel joins. The line's length is only known on the device: every CTA forms the same
// sums over the sequences.
#pragma once
#include <cuda.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "sync_ptx.cuh"

namespace amv {
namespace paged {

constexpr uint32_t kMaxSeqs = 4095;
constexpr float kLog2e = 1.44269504088896340736f;

enum : uint32_t { OUT_F32 = 0, OUT_F16 = 1, OUT_PARTS = 2 };   // OUT_PARTS: f32 [row][head][D + 4]: maximum, sum, 2 unused, values

struct Args {
    const __half *q, *k, *v;
    const int32_t *table, *q_start, *kv_len;
    const int32_t* prefix;      // prefix launch: [0] keys, [1 ..] pages; otherwise null
    void* dst;
    float* slots;               // results of cut row tiles: slot 2 c (a tile begun elsewhere), 2 c + 1 (one that goes on elsewhere)
    uint4* cut;                 // per CTA what the merge kernel needs of a cut row tile: parts | group << 16 (0: none), first token, first row, rows
    uint32_t q_boxes;           // the map of q serves the rows of a group
    uint32_t report;            // this launch counts the sequences that do not fit
    uint32_t HB, groups, keys_log2, over;   // KV heads of a group, groups, the line's tiles and its allowance per row tile
    const float* extra;         // results over other keys of the same rows that the final ones take in (the layout of OUT_PARTS)
    uint32_t* refused;          // the caller's status words: count of refused entries, lowest node
    uint32_t* status;           // the context's
    uint32_t max_own_q, max_own_kv;   // prefix launch: the maxima of the sequences
    uint32_t n_seqs, rows, max_q, max_kv, page_log2, n_pages, table_stride;
    uint32_t n_head, n_head_kv, G, g_mul, g_shift;   // x / G = x * g_mul >> g_shift for x < 2^31
    uint32_t c_ps, c_ts, c_hs;  // cache strides in elements: page, token, head
    uint32_t q_s, dst_s, out, node, window, min_rows, max_rows;   // a launch serves the sequences of min_rows .. max_rows rows
    float scale, softcap, scale2, cap_in, cap_out;                // scale2: scale * log2(e); scale / softcap, softcap * log2(e)
};

struct Seq {
    uint32_t tok0, n_q, kv;   // n_q == 0: nothing to do
    const int32_t* pages;
};

__device__ __forceinline__ void refuse(const Args& pc, uint32_t count) {
    atomicAdd(pc.refused, count);
    atomicMin(pc.refused + 1, pc.node);
}

__device__ __forceinline__ bool seq_fits(const Args& pc, int32_t a, int32_t b, int32_t kv, uint32_t max_q, uint32_t max_kv) {
    return a >= 0 && b >= a && (uint32_t)b <= pc.rows && (uint32_t)(b - a) <= max_q && kv >= 0 && (uint32_t)kv <= max_kv &&
           (uint64_t)(uint32_t)kv <= (uint64_t)pc.table_stride << pc.page_log2;
}
// Sequence s; one whose numbers do not fit the buffers has no rows (report: counted, by one thread of the grid).
__device__ __forceinline__ Seq load_seq(const Args& pc, uint32_t s, bool report = false) {
    Seq x;
    if (pc.prefix) {
        const int32_t kv = pc.prefix[0], n = pc.q_start[pc.n_seqs];
        const bool bad = kv < 0 || (uint32_t)kv > pc.max_kv || n < 0 || (uint32_t)n > pc.rows;
        x = {0u, bad ? 0u : (uint32_t)n, bad ? 0u : (uint32_t)kv, pc.prefix + 1};
        if (bad && report) refuse(pc, 1u);
        return x;
    }
    const int32_t a = pc.q_start[s], b = pc.q_start[s + 1u], kv = pc.kv_len[s];
    const bool bad = !seq_fits(pc, a, b, kv, pc.max_q, pc.max_kv);
    x = {bad ? 0u : (uint32_t)a, bad ? 0u : (uint32_t)(b - a), bad ? 0u : (uint32_t)kv, pc.table + (uint64_t)s * pc.table_stride};
    if (bad && report) refuse(pc, 1u);
    return x;
}

// r / G without a division's instructions, which a CTA runs once and has to fetch: g_mul = ceil(2^g_shift / G) and g_shift = 31 + ceil(log2 G)
// are off by less than 2^31 in r * g_mul, so that no quotient of r < 2^31 moves.
__device__ __forceinline__ uint32_t query_of(const Args& pc, uint32_t r) { return (uint32_t)((uint64_t)r * pc.g_mul >> pc.g_shift); }

// The keys that row r sees: [lo, hi)
struct Span {
    uint32_t lo, hi;
};
__device__ __forceinline__ Span row_span(const Args& pc, const Seq& q, uint32_t r) {
    if (pc.prefix) return {0u, q.kv};
    const int32_t end = (int32_t)q.kv - (int32_t)q.n_q + (int32_t)query_of(pc, r) + 1;   // one past its own place
    if (end <= 0) return {0u, 0u};
    const uint32_t hi = (uint32_t)end;
    return {pc.window && hi > pc.window ? hi - pc.window : 0u, hi};
}
// The first key tile of rows r0 .. r1 and how many there are: at least one, so that rows that see nothing are written, too.
__device__ __forceinline__ void tile_range(const Args& pc, const Seq& q, uint32_t r0, uint32_t r1, uint32_t& first, uint32_t& count) {
    const uint32_t lo = row_span(pc, q, r0).lo, hi = row_span(pc, q, r1).hi;
    first = lo >> pc.keys_log2;
    count = hi > lo ? ((hi + (1u << pc.keys_log2) - 1u) >> pc.keys_log2) - first : 1u;
}

__device__ __forceinline__ bool served(const Args& pc, uint32_t R) { return R >= pc.min_rows && R <= pc.max_rows && R != 0u; }

// The line: s_pref[s] = tiles in front of sequence s (s_pref[n] = all of them). WARPS warps, all threads; ends with a barrier.
template <uint32_t ROWS, uint32_t WARPS>
__device__ __forceinline__ uint32_t build_line(const Args& pc, uint32_t* s_pref, uint32_t* s_warp) {
    const uint32_t n = pc.prefix ? 1u : pc.n_seqs;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
    // lanes take sequences while there is a row tile or two of each, row tiles of one sequence where there are many
    const bool tiles_by_lane = (uint64_t)pc.max_q * pc.G > 4u * ROWS && (!pc.prefix);
    const bool report = blockIdx.x == 0u && pc.report;
    bool whole = true;   // a shared prefix serves a batch without refused sequences, whose rows begin at 0
    if (pc.prefix) {
        bool fits = pc.q_start[0] == 0;
        for (uint32_t s = threadIdx.x; s < pc.n_seqs; s += WARPS * 32u) {
            const int32_t a = pc.q_start[s], b = pc.q_start[s + 1u], kv = pc.kv_len[s];
            fits = fits && seq_fits(pc, a, b, kv, pc.max_own_q, pc.max_own_kv);
        }
        whole = __syncthreads_and(fits);
        if (!whole && report && threadIdx.x == 0u) refuse(pc, 1u);
    }
    if (!tiles_by_lane) {
        for (uint32_t s = threadIdx.x; s < n; s += WARPS * 32u) {
            const Seq q = load_seq(pc, s, report);
            const uint32_t R = q.n_q * pc.G;
            uint32_t tiles = 0, first, count;
            if (served(pc, R) && whole) {
                if (pc.prefix) {
                    tile_range(pc, q, 0u, 0u, first, count);
                    tiles = (count + pc.over) * ((R + ROWS - 1u) / ROWS);
                } else {
                    for (uint32_t r = 0; r < R; r += ROWS) {
                        tile_range(pc, q, r, min(r + ROWS, R) - 1u, first, count);
                        tiles += count + pc.over;
                    }
                }
            }
            s_pref[s] = tiles * pc.groups;
        }
    } else {
        for (uint32_t s = warp; s < n; s += WARPS) {
            const Seq q = load_seq(pc, s, report && lane == 0u);
            const uint32_t R = q.n_q * pc.G;
            uint32_t tiles = 0, first, count;
            if (served(pc, R))
                for (uint32_t r = lane * ROWS; r < R; r += 32u * ROWS) {
                    tile_range(pc, q, r, min(r + ROWS, R) - 1u, first, count);
                    tiles += count + pc.over;
                }
            tiles = (uint32_t)warp_sum_i((int)tiles);
            if (lane == 0u) s_pref[s] = tiles * pc.groups;
        }
    }
    __syncthreads();
    // exclusive sums in place: a run of consecutive sequences per thread
    const uint32_t per = (n + WARPS * 32u - 1u) / (WARPS * 32u), b = min(n, threadIdx.x * per), e = min(n, b + per);
    uint32_t sum = 0;
    for (uint32_t s = b; s < e; ++s) sum += s_pref[s];
    uint32_t incl = sum;
#pragma unroll
    for (uint32_t o = 1; o < 32u; o <<= 1) {
        const uint32_t up = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += up;
    }
    if (lane == 31u) s_warp[warp] = incl;
    __syncthreads();
    uint32_t before = incl - sum, total = 0;
#pragma unroll
    for (uint32_t w = 0; w < WARPS; ++w) {
        before += w < warp ? s_warp[w] : 0u;
        total += s_warp[w];
    }
    for (uint32_t s = b; s < e; ++s) {
        const uint32_t t = s_pref[s];
        s_pref[s] = before;
        before += t;
    }
    if (threadIdx.x == 0u) s_pref[n] = total;
    __syncthreads();
    return total;
}

// A CTA's stretch of the line: tiles [begin, end). CTAs past the number of tiles have none.
struct Stretch {
    uint32_t begin, end, ctas, total;
};
__device__ __forceinline__ Stretch my_stretch(uint32_t total) {
    Stretch x;
    x.total = total;
    x.ctas = min(gridDim.x, total);
    x.begin = x.end = 0u;
    if (blockIdx.x < x.ctas) {
        const uint32_t q = total / x.ctas, r = total - q * x.ctas;   // floor(c total / ctas) in 32 bits
        x.begin = blockIdx.x * q + blockIdx.x * r / x.ctas;
        x.end = (blockIdx.x + 1u) * q + (blockIdx.x + 1u) * r / x.ctas;
    }
    return x;
}
// the last CTA whose stretch has a tile in front of tile e (e > 0)
__device__ __forceinline__ uint32_t last_cta(const Stretch& x, uint32_t e) {
    return (uint32_t)(((uint64_t)e * x.ctas + x.total - 1u) / x.total) - 1u;
}

// The part of a row tile that a CTA works on: key tiles first + a .. first + b - 1 of its n; `begin`: the row tile's place in the line.
struct Piece {
    uint32_t seq, group, r0, R, first, a, b, n, begin;
    Seq q;
};
// Walks a stretch piece by piece; a whole warp, all lanes with the same values.
template <uint32_t ROWS>
struct Walk {
    uint32_t t, end, seq;
    Piece p;
    __device__ __forceinline__ Walk(const Stretch& x) : t(x.begin), end(x.end), seq(0xFFFFFFFFu) {}
    __device__ __forceinline__ bool next(const Args& pc, const uint32_t* s_pref) {
        while (t < end) {
            if (seq == 0xFFFFFFFFu || t >= s_pref[seq + 1u]) {   // the sequence that place t belongs to
                uint32_t lo = 0, hi = pc.prefix ? 1u : pc.n_seqs;   // s_pref[lo] <= t < s_pref[hi]
                while (hi - lo > 1u) {
                    const uint32_t mid = (lo + hi) >> 1;
                    if (s_pref[mid] <= t) lo = mid;
                    else hi = mid;
                }
                seq = p.seq = lo;
                p.q = load_seq(pc, lo);
                p.R = p.q.n_q * pc.G;
            }
            uint32_t rem = t - s_pref[seq];
            p.group = 0u;
            if (pc.groups > 1u) {
                const uint32_t per_group = (s_pref[seq + 1u] - s_pref[seq]) / pc.groups;
                p.group = rem / per_group;
                rem -= p.group * per_group;
            }
            if (pc.prefix || p.R <= ROWS) {   // row tiles with the same number of key tiles, or a single one
                tile_range(pc, p.q, 0u, p.R <= ROWS ? p.R - 1u : 0u, p.first, p.n);
                p.r0 = 0u;
                if (p.R > ROWS) {
                    const uint32_t i = rem / (p.n + pc.over);
                    p.r0 = i * ROWS;
                    rem -= i * (p.n + pc.over);
                }
            } else {                          // counted 32 at a time
                const uint32_t lane = threadIdx.x & 31u;
                for (uint32_t base = 0;; base += 32u * ROWS) {
                    const uint32_t r = base + lane * ROWS;
                    uint32_t first = 0, count = 0;
                    if (r < p.R) tile_range(pc, p.q, r, min(r + ROWS, p.R) - 1u, first, count);
                    const uint32_t len = r < p.R ? count + pc.over : 0u;
                    uint32_t incl = len;
#pragma unroll
                    for (uint32_t o = 1; o < 32u; o <<= 1) {
                        const uint32_t up = __shfl_up_sync(0xffffffffu, incl, o);
                        if (lane >= o) incl += up;
                    }
                    const uint32_t hit = __ballot_sync(0xffffffffu, incl > rem);
                    if (hit == 0u && base + 32u * ROWS < p.R) {
                        rem -= __shfl_sync(0xffffffffu, incl, 31);
                        continue;
                    }
                    const int from = hit ? __ffs(hit) - 1 : 0;   // (hit is never empty in the last round)
                    p.first = __shfl_sync(0xffffffffu, first, from);
                    p.n = __shfl_sync(0xffffffffu, count, from);
                    p.r0 = base + (uint32_t)from * ROWS;
                    rem -= __shfl_sync(0xffffffffu, incl - len, from);
                    break;
                }
            }
            const uint32_t step = min(p.n + pc.over - rem, end - t);
            p.begin = t - rem;
            p.a = min(rem, p.n);
            p.b = min(p.n, rem + step);
            t += step;
            if (p.b > p.a) return true;
        }
        return false;
    }
};

// Notes for the merge kernel what the CTA's last piece leaves (the first word 0: nothing).
__device__ __forceinline__ void note_cut(const Args& pc, const Stretch& x, const Piece& p, uint32_t rows) {
    const uint32_t last = last_cta(x, p.begin + p.n);
    pc.cut[blockIdx.x] = make_uint4((last - blockIdx.x + 1u) | p.group << 16, p.q.tok0, p.r0, rows);
}

// mbar_wait (sync_ptx.cuh) without a call: the registers of a warp whose share setmaxnreg has changed leave no room for a callee's.
__device__ __forceinline__ bool wait_on(uint32_t bar, uint32_t parity, ptx::Ctl* ctl, uint32_t* status, uint32_t tag) {
    if (ptx::mbar_try_wait(bar, parity)) return true;
    const long long t0 = clock64();
#pragma unroll 1
    while (!ptx::mbar_try_wait(bar, parity)) {
        if (ctl->abort) return false;
        if (clock64() - t0 > ptx::kWaitCycles) {
            ctl->abort = 1u;
            if (atomicCAS(status, DEV_STATUS_OK, DEV_STATUS_WAIT_TIMEOUT) == DEV_STATUS_OK) status[1] = tag;
            return false;
        }
    }
    return true;
}
// Waits for what the last stages of a ring were asked for: copy i of `issued` is the i / stages-th of stage i % stages. A copy that lands
// after its CTA has left would write into the memory of the next one, so this goes by the copies alone, not by whether the CTA has given
// up, and a warp that has asked for copies does it whenever it leaves: another one may give up later. They land within microseconds;
// kDrainPolls polls of 64 ns or more bound the wait. arrived(stage, parity): whether the phase has completed.
constexpr uint32_t kDrainPolls = 1u << 14;
template <class Arrived>
__host__ __device__ __forceinline__ bool drain_copies(uint32_t issued, uint32_t stages, Arrived arrived) {
    for (uint32_t i = issued > stages ? issued - stages : 0u; i < issued; ++i)
        for (uint32_t polls = 0; !arrived(i % stages, i / stages & 1u);)
            if (++polls == kDrainPolls) return false;
    return true;
}
__device__ __forceinline__ bool arrived_or_pause(uint32_t bar, uint32_t parity) {
    if (ptx::mbar_try_wait(bar, parity)) return true;
    __nanosleep(64);
    return false;
}
__device__ __forceinline__ void drain_ring(uint32_t full, uint32_t issued, uint32_t stages) {
    drain_copies(issued, stages, [&](uint32_t stage, uint32_t parity) { return arrived_or_pause(full + 8u * stage, parity); });
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float neg_inf() { return __uint_as_float(0xFF800000u); }
// exp2(m - to) of a maximum m <= to, 0 where m is that of nothing
__device__ __forceinline__ float weight(float m, float to) { return m == neg_inf() ? 0.0f : ex2(m - to); }

__device__ __forceinline__ uint64_t dst_row(const Args& pc, uint32_t token, uint32_t head, uint32_t D) {
    return pc.out == OUT_PARTS ? ((uint64_t)token * pc.n_head + head) * (D + 4u) : (uint64_t)token * pc.dst_s + (uint64_t)head * D;
}

// One row's result by a warp, lane l holding columns C l .. C l + C - 1 of the weighted values (C = D / 32): with the results over
// other keys taken in where there are any, divided by the sum, or as they are (OUT_PARTS). Rows that saw nothing are zero.
template <uint32_t C>
__device__ __forceinline__ void finish_row(const Args& pc, uint32_t token, uint32_t head, float m, float l, float (&o)[C]) {
    constexpr uint32_t D = 32u * C;
    const uint32_t lane = threadIdx.x & 31u;
    const uint64_t at = dst_row(pc, token, head, D);
    if (pc.out == OUT_PARTS) {
        float* row = reinterpret_cast<float*>(pc.dst) + at;
        if (lane == 0u) *reinterpret_cast<float2*>(row) = make_float2(m, l);
#pragma unroll
        for (uint32_t c = 0; c < C; c += 2u) *reinterpret_cast<float2*>(row + 4u + C * lane + c) = make_float2(o[c], o[c + 1u]);
        return;
    }
    if (pc.extra) {
        const float* row = pc.extra + ((uint64_t)token * pc.n_head + head) * (D + 4u);
        const float2 ml = *reinterpret_cast<const float2*>(row);
        const float top = fmaxf(m, ml.x), f = weight(m, top), g = weight(ml.x, top);
        l = l * f + ml.y * g;
#pragma unroll
        for (uint32_t c = 0; c < C; ++c) o[c] = (f != 0.0f ? o[c] * f : 0.0f) + (g != 0.0f ? row[4u + C * lane + c] * g : 0.0f);
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    if (pc.out == OUT_F16) {
        __half* row = reinterpret_cast<__half*>(pc.dst) + at + C * lane;
#pragma unroll
        for (uint32_t c = 0; c < C; c += 2u)
            *reinterpret_cast<__half2*>(row + c) = inv == 0.0f ? __half2() : __floats2half2_rn(o[c] * inv, o[c + 1u] * inv);
    } else {
        float* row = reinterpret_cast<float*>(pc.dst) + at + C * lane;
#pragma unroll
        for (uint32_t c = 0; c < C; c += 2u)
            *reinterpret_cast<float2*>(row + c) = inv == 0.0f ? make_float2(0.f, 0.f) : make_float2(o[c] * inv, o[c + 1u] * inv);
    }
}

// The page of key `key` of a sequence, or -1 where the table's entry is none of the cache's.
__device__ __forceinline__ int32_t page_of(const Args& pc, const Seq& q, uint32_t key) {
    const int32_t page = q.pages[key >> pc.page_log2];
    return page < 0 || (uint32_t)page >= pc.n_pages ? -1 : page;
}

// The scores' scale, softcap and change of base: what exponentials to base 2 take.
__device__ __forceinline__ float score2(const Args& pc, float s) {
    return pc.softcap != 0.0f ? pc.softcap * tanhf(s * pc.scale / pc.softcap) * kLog2e : s * pc.scale2;
}

// score2 of N scores a thread, by a converged warp, without tanhf's some 25 instructions. Each score by its own size alone. Up to a quarter of
// the cap (7.5 of 30): the odd series y - y^3 / 3 + 2 y^5 / 15 - 17 y^7 / 315 + 62 y^9 / 2835, whose next term is below 1e-8 of it for
// |y| <= 1/4. Beyond: 1 - 2 / (1 + e^2y) by two special functions, with an absolute error of 2^-22 where tanh is at least 0.24 (times a cap of
// 30, that is 7e-6 of a score: 1.4e-6 of a result that ordinary 32-bit operations leave with 2e-7). The warp's vote only spares it the second
// form where nobody takes it; among its scores are hidden ones of any value (keys that nobody has written, shared memory of an earlier
// kernel), which are not to decide how exact the others are. One branch for all: a branch per score is slower than both forms (32 drafted
// sequences 24 us instead of 22.7).
template <uint32_t N>
__device__ __forceinline__ void capped(const Args& pc, float (&s)[N]) {
    if (pc.softcap == 0.0f) {
#pragma unroll
        for (uint32_t k = 0; k < N; ++k) s[k] *= pc.scale2;
        return;
    }
    bool small = true;
#pragma unroll
    for (uint32_t k = 0; k < N; ++k) {
        s[k] *= pc.cap_in;
        small = small && fabsf(s[k]) <= 0.25f;
    }
    auto series = [&](float y) {
        const float y2 = y * y, t = fmaf(y2, fmaf(y2, fmaf(y2, 62.0f / 2835.0f, -17.0f / 315.0f), 2.0f / 15.0f), -1.0f / 3.0f);
        return pc.cap_out * fmaf(y * y2, t, y);
    };
    if (__all_sync(0xffffffffu, small)) {
#pragma unroll
        for (uint32_t k = 0; k < N; ++k) s[k] = series(s[k]);
        return;
    }
#pragma unroll
    for (uint32_t k = 0; k < N; ++k) {
        float r;
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + ex2(s[k] * (2.0f * kLog2e))));
        s[k] = fabsf(s[k]) <= 0.25f ? series(s[k]) : fmaf(-2.0f * pc.cap_out, r, pc.cap_out);
    }
}
// One row by a whole warp over keys [lo, hi), hidden keys left out instead of multiplied by zero: a lane's C columns of
// sum 2^(score - ref) v. For rows whose accumulator is not finite: the matrix instructions multiply every key of a step with every
// row, so a NaN or an infinity in V would reach rows that do not see its key, and an infinity would meet the remainder of its
// probability, which may be zero or negative. Rare, so simple: a lane per key for the scores, all lanes on a key's columns.
template <uint32_t C>
__device__ __noinline__ void seen_keys_row(const Args& pc, const Seq& q, uint32_t hkv, const __half* qrow, uint32_t lo, uint32_t hi, float ref,
                                           float (&o)[C]) {
    constexpr uint32_t D = 32u * C;
    const uint32_t lane = threadIdx.x & 31u, mask = (1u << pc.page_log2) - 1u;
#pragma unroll
    for (uint32_t c = 0; c < C; ++c) o[c] = 0.0f;
    for (uint32_t key0 = lo; key0 < hi; key0 += 32u) {
        const uint32_t key = key0 + lane;
        const int32_t page = key < hi ? page_of(pc, q, key) : -1;
        const uint64_t row = (uint64_t)(page < 0 ? 0 : page) * pc.c_ps + (uint64_t)(key & mask) * pc.c_ts + (uint64_t)hkv * pc.c_hs;
        float p = 0.0f;
        if (page >= 0) {
            float s = 0.0f;
            for (uint32_t c = 0; c < D; ++c) s = fmaf(__half2float(qrow[c]), __half2float(pc.k[row + c]), s);
            p = ex2(score2(pc, s) - ref);
        }
        for (uint32_t seen = __ballot_sync(0xffffffffu, page >= 0); seen; seen &= seen - 1u) {
            const int b = __ffs(seen) - 1;
            const float pb = __shfl_sync(0xffffffffu, p, b);
            const __half* vr = pc.v + __shfl_sync(0xffffffffu, (unsigned long long)row, b) + C * lane;
#pragma unroll
            for (uint32_t c = 0; c < C; ++c) o[c] = fmaf(pb, __half2float(vr[c]), o[c]);
        }
    }
}

}  // namespace paged
}  // namespace amv
