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

// Query heads that share a KV head, and what query_of divides by them with.
inline void set_group(Args& pc, uint32_t G) {
    pc.G = G;
    for (pc.g_shift = 31u; (1ull << (pc.g_shift - 31u)) < G; ++pc.g_shift) {}
    pc.g_mul = (uint32_t)(((1ull << pc.g_shift) + G - 1u) / G);
}
// r / G without a division's instructions, which a CTA runs once and has to fetch: g_mul = ceil(2^g_shift / G) and g_shift = 31 + ceil(log2 G)
// are off by less than 2^31 in r * g_mul, so that no quotient of r < 2^31 moves.
__host__ __device__ __forceinline__ uint32_t query_of(const Args& pc, uint32_t r) { return (uint32_t)((uint64_t)r * pc.g_mul >> pc.g_shift); }

// The keys that row r sees: [lo, hi)
struct Span {
    uint32_t lo, hi;
};
__host__ __device__ __forceinline__ Span row_span(const Args& pc, const Seq& q, uint32_t r) {
    if (pc.prefix) return {0u, q.kv};
    const int32_t end = (int32_t)q.kv - (int32_t)q.n_q + (int32_t)query_of(pc, r) + 1;   // one past its own place
    if (end <= 0) return {0u, 0u};
    const uint32_t hi = (uint32_t)end;
    return {pc.window && hi > pc.window ? hi - pc.window : 0u, hi};
}
// The first key tile of rows r0 .. r1 and how many there are: at least one, so that rows that see nothing are written, too.
__host__ __device__ __forceinline__ void tile_range(const Args& pc, const Seq& q, uint32_t r0, uint32_t r1, uint32_t& first, uint32_t& count) {
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
__host__ __device__ __forceinline__ Stretch stretch_of(uint32_t total, uint32_t cta, uint32_t grid) {
    Stretch x;
    x.total = total;
    x.ctas = grid < total ? grid : total;
    x.begin = x.end = 0u;
    if (cta < x.ctas) {
        const uint32_t q = total / x.ctas, r = total - q * x.ctas;   // floor(c total / ctas) in 32 bits
        x.begin = cta * q + cta * r / x.ctas;
        x.end = (cta + 1u) * q + (cta + 1u) * r / x.ctas;
    }
    return x;
}
__device__ __forceinline__ Stretch my_stretch(uint32_t total) { return stretch_of(total, blockIdx.x, gridDim.x); }
// the last CTA whose stretch has a tile in front of tile e (e > 0)
__host__ __device__ __forceinline__ uint32_t last_cta(const Stretch& x, uint32_t e) {
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
// exp2(m - to) of a maximum m <= to, 0 where m is that of nothing. Of something it is never 0, but the smallest normal number at least, which
// leaves no trace in a finite sum: an infinity or a NaN among the values is to show in the result however small its weight is.
__device__ __forceinline__ float weight(float m, float to) { return m == neg_inf() ? 0.0f : fmaxf(ex2(m - to), 1.17549435e-38f); }

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
// A warp's rows once more, behind the last piece of its CTA, where one of them was not finite: the matrix instructions multiply every key of
// a step with every row, so a NaN or an infinity in V reaches rows that do not see its key, and an infinity meets the remainder of its
// probability, which may be zero or negative. The CTA's stretch is walked again, for rows first_row .. first_row + count - 1 of each row tile
// (32 at most), head hb of a group, whose result of a piece, in dst or the piece's slot, is not finite. Nobody waits for this on a barrier
// with a limit, so it may take its time.
// Where Q and K are finite, a column in which a row sees values that are not is their sum: NaN, or one of the infinities, whatever their
// weights are. So the keys are looked through, once for all rows where all see them. A row that is not finite in another column,
// too, has it from a key that it does not see, and is formed anew, hidden keys left out instead of multiplied by zero: four rows and 32
// keys at a time, in 32 bits; a score ends in the lane of its key's number.
// For both, D / 8 lanes take a key, 16 bytes each; group g of them has keys g D / 8 .. of 32, one after another, and the groups meet at the end.
// One infinity at the first key of every sequence, without / with it: a prompt of 2048, 8 heads of 128 over 2: 49 / 350 us, of 8192, 32 heads over
// 8: 714 / 7500 us (32-bit results 974 / 9800); 32 single tokens of 4000 keys 98 / 364 us. Each row's scores again: 17500 us for the first.
template <uint32_t C, uint32_t ROWS>
struct Again {
    static constexpr uint32_t D = 32u * C, N = 4, LANES = D / 8u, AHEAD = 4, kNone = 0xFFFFFFFFu;
    const Args& pc;
    Piece p;
    uint32_t hkv, lane, sub, lead;
    bool whole;
    float* slot;

    static __device__ __forceinline__ void half8(const uint4& x, float (&y)[8]) {
        const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (uint32_t i = 0; i < 4u; ++i) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
            y[2u * i] = f.x;
            y[2u * i + 1u] = f.y;
        }
    }
    static __device__ __forceinline__ bool odd(const uint4& x) {   // an exponent of ones in any of the eight
        auto w = [](uint32_t v) { return (v & 0x7C007C00u) + 0x04000400u; };
        return ((w(x.x) | w(x.y) | w(x.z) | w(x.w)) & 0x80008000u) != 0u;
    }
    static __device__ __forceinline__ void groups_meet(float (&x)[8]) {
#pragma unroll
        for (uint32_t w = LANES; w < 32u; w <<= 1)
#pragma unroll
            for (uint32_t c = 0; c < 8u; ++c) x[c] += __shfl_xor_sync(0xffffffffu, x[c], w);
    }
    __device__ __forceinline__ uint32_t token(uint32_t r) const { return p.q.tok0 + query_of(pc, r); }
    __device__ __forceinline__ uint32_t head(uint32_t r) const { return hkv * pc.G + r - query_of(pc, r) * pc.G; }
    __device__ __forceinline__ bool is_f16() const { return whole && pc.out == OUT_F16; }
    __device__ __forceinline__ float* f32_row(uint32_t r) const {   // this lane's eight columns of what the first pass left
        float* x = whole ? reinterpret_cast<float*>(pc.dst) + dst_row(pc, token(r), head(r), D) + (pc.out == OUT_PARTS ? 4u : 0u)
                         : slot + (uint64_t)(r - p.r0) * (D + 4u) + 4u;
        return x + 8u * sub;
    }
    __device__ __forceinline__ __half* f16_row(uint32_t r) const { return reinterpret_cast<__half*>(pc.dst) + dst_row(pc, token(r), head(r), D) + 8u * sub; }
    __device__ __forceinline__ void read(uint32_t r, float (&x)[8]) const {
        if (is_f16()) {
            half8(*reinterpret_cast<const uint4*>(f16_row(r)), x);
        } else {
            const float4 *at = reinterpret_cast<const float4*>(f32_row(r)), u = at[0], v = at[1];
            x[0] = u.x, x[1] = u.y, x[2] = u.z, x[3] = u.w, x[4] = v.x, x[5] = v.y, x[6] = v.z, x[7] = v.w;
        }
    }
    __device__ __forceinline__ bool finite(uint32_t r) const {
        float x[8], sum = 0.0f;
        read(r, x);
#pragma unroll
        for (uint32_t c = 0; c < 8u; ++c) sum = fmaf(x[c], 0.0f, sum);
        return __all_sync(0xffffffffu, sum == 0.0f) != 0;
    }
    // 32 keys from key0 on, below `last`: this lane's key's row in the caches, and which of them are there
    __device__ __forceinline__ uint32_t keys_at(uint32_t key0, uint32_t last, uint64_t& at) const {
        const uint32_t key = key0 + lane;
        const int32_t page = key < last ? page_of(pc, p.q, key) : -1;
        at = (uint64_t)(page < 0 ? 0 : page) * pc.c_ps + (uint64_t)(key & ((1u << pc.page_log2) - 1u)) * pc.c_ts + (uint64_t)hkv * pc.c_hs;
        return __ballot_sync(0xffffffffu, page >= 0);
    }
    __device__ __forceinline__ uint4 load(const __half* cache, uint64_t at, uint32_t there, uint32_t i) const {   // this lane's columns of key lead + i
        const uint64_t e = __shfl_sync(0xffffffffu, (unsigned long long)at, lead + i) + 8u * sub;
        return there >> (lead + i) & 1u ? *reinterpret_cast<const uint4*>(cache + e) : make_uint4(0u, 0u, 0u, 0u);
    }
    // Adds up this lane's columns of what is not finite in V; false: something of K is not.
    __device__ __noinline__ bool look_through(uint32_t first, uint32_t last, float (&sum)[8]) const {
        bool plain = true;
#pragma unroll 1
        for (uint32_t key0 = first; key0 < last; key0 += 32u) {
            uint64_t at;
            const uint32_t there = keys_at(key0, last, at);
#pragma unroll 1
            for (uint32_t i0 = 0; i0 < LANES; i0 += AHEAD) {
                uint4 x[AHEAD], y[AHEAD];
#pragma unroll
                for (uint32_t i = 0; i < AHEAD; ++i) {
                    x[i] = load(pc.v, at, there, i0 + i);
                    y[i] = load(pc.k, at, there, i0 + i);
                }
#pragma unroll
                for (uint32_t i = 0; i < AHEAD; ++i) {
                    plain = plain && !odd(y[i]);
                    if (!odd(x[i])) continue;
                    float v[8];
                    half8(x[i], v);
#pragma unroll
                    for (uint32_t c = 0; c < 8u; ++c) sum[c] += v[c] * 0.0f == 0.0f ? 0.0f : v[c];
                }
            }
        }
        return __all_sync(0xffffffffu, plain) != 0;
    }
    // Row r of what the rows see together, [a, b), its sum there and whether that tells all: whether the row is right now.
    __device__ __forceinline__ bool from_sums(uint32_t r, uint32_t from, uint32_t to, uint32_t a, uint32_t b, const float (&common)[8], bool plain) const {
        const Span s = row_span(pc, p.q, r);
        float sum[8];
#pragma unroll
        for (uint32_t c = 0; c < 8u; ++c) sum[c] = 0.0f;
        plain = plain && !odd(*reinterpret_cast<const uint4*>(pc.q + (uint64_t)token(r) * pc.q_s + (uint64_t)head(r) * D + 8u * sub));
        const uint32_t lo = max(s.lo, from), hi = min(s.hi, to);
        if (lo < a) plain = look_through(lo, min(a, hi), sum) && plain;
        if (b < hi) plain = look_through(max(b, lo), hi, sum) && plain;
        groups_meet(sum);
        float x[8];
        read(r, x);
        const float* extra = whole && pc.out != OUT_PARTS && pc.extra ? pc.extra + ((uint64_t)token(r) * pc.n_head + head(r)) * (D + 4u) + 4u + 8u * sub : nullptr;
        bool known = plain;
#pragma unroll
        for (uint32_t c = 0; c < 8u; ++c) {
            if (x[c] * 0.0f == 0.0f) continue;
            x[c] = sum[c] + common[c];
            const bool theirs = extra && extra[c] * 0.0f != 0.0f;
            known = known && (x[c] != 0.0f || (theirs && pc.prefix));   // (of a prefix, no key is hidden)
            if (theirs) x[c] += extra[c];
        }
        if (!__all_sync(0xffffffffu, known)) return false;
        if (lead == 0u) {   // (finite columns are written as they were)
            if (is_f16()) {
#pragma unroll
                for (uint32_t c = 0; c < 8u; ++c) f16_row(r)[c] = __float2half_rn(x[c]);
            } else {
#pragma unroll
                for (uint32_t c = 0; c < 8u; ++c) f32_row(r)[c] = x[c];
            }
        }
        return true;
    }
    // The first rows of a mask (bit b: row base + b), up to N of them, over the keys they see.
    __device__ __noinline__ uint32_t from_keys(uint32_t mask, uint32_t base, uint32_t from, uint32_t to) const {
        uint32_t row[N], lo[N], hi[N], first = kNone, last = 0u;
        float m[N], l[N], qf[N][8], o[N][8];
#pragma unroll
        for (uint32_t j = 0; j < N; ++j) {   // (one that sees nothing where fewer than N are left)
            const bool have = mask != 0u;
            row[j] = have ? base + (uint32_t)__ffs(mask) - 1u : kNone;
            mask &= mask - (have ? 1u : 0u);
            const uint32_t r = have ? row[j] : p.r0;
            half8(*reinterpret_cast<const uint4*>(pc.q + (uint64_t)token(r) * pc.q_s + (uint64_t)head(r) * D + 8u * sub), qf[j]);
            const Span s = row_span(pc, p.q, r);
            lo[j] = have ? max(s.lo, from) : kNone;
            hi[j] = have ? min(s.hi, to) : 0u;
            first = min(first, lo[j]);
            last = max(last, hi[j]);
            m[j] = neg_inf();
            l[j] = 0.0f;
#pragma unroll
            for (uint32_t c = 0; c < 8u; ++c) o[j][c] = 0.0f;
        }
#pragma unroll 1
        for (uint32_t key0 = first; key0 < last; key0 += 32u) {
            uint64_t at;
            const uint32_t there = keys_at(key0, last, at), key = key0 + lane;
            float w[N];
#pragma unroll 1
            for (uint32_t i0 = 0; i0 < LANES; i0 += AHEAD) {
                uint4 x[AHEAD];
#pragma unroll
                for (uint32_t i = 0; i < AHEAD; ++i) x[i] = load(pc.k, at, there, i0 + i);
#pragma unroll
                for (uint32_t i = 0; i < AHEAD; ++i) {
                    float kf[8];
                    half8(x[i], kf);
#pragma unroll
                    for (uint32_t j = 0; j < N; ++j) {
                        float s = 0.0f;
#pragma unroll
                        for (uint32_t c = 0; c < 8u; ++c) s = fmaf(qf[j][c], kf[c], s);
#pragma unroll
                        for (uint32_t d = 1; d < LANES; d <<= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
                        w[j] = sub == i0 + i ? s : w[j];
                    }
                }
            }
#pragma unroll
            for (uint32_t j = 0; j < N; ++j) {
                const bool seen = (there >> lane & 1u) && key >= lo[j] && key < hi[j];
                const float s = score2(pc, w[j]);
                float top = seen ? s : neg_inf();
#pragma unroll
                for (uint32_t d = 1; d < 32u; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
                if (top > m[j]) {
                    const float f = weight(m[j], top);
                    m[j] = top;
                    l[j] *= f;
#pragma unroll
                    for (uint32_t c = 0; c < 8u; ++c) o[j][c] *= f;
                }
                // negative: not seen. A weight too small for 32 bits is one all the same: an infinity times it is infinite
                const float e = ex2(s - (m[j] == neg_inf() ? 0.0f : m[j]));
                w[j] = !seen ? -1.0f : e == 0.0f && s != neg_inf() ? 1.17549435e-38f : e;
                l[j] += seen ? w[j] : 0.0f;
            }
#pragma unroll 1
            for (uint32_t i0 = 0; i0 < LANES; i0 += AHEAD) {
                uint4 x[AHEAD];
#pragma unroll
                for (uint32_t i = 0; i < AHEAD; ++i) x[i] = load(pc.v, at, there, i0 + i);
#pragma unroll
                for (uint32_t i = 0; i < AHEAD; ++i) {
                    float vf[8];
                    half8(x[i], vf);
#pragma unroll
                    for (uint32_t j = 0; j < N; ++j) {
                        const float y = __shfl_sync(0xffffffffu, w[j], lead + i0 + i);
#pragma unroll
                        for (uint32_t c = 0; c < 8u; ++c) o[j][c] = y < 0.0f ? o[j][c] : fmaf(y, vf[c], o[j][c]);
                    }
                }
            }
        }
#pragma unroll
        for (uint32_t j = 0; j < N; ++j) {
            if (row[j] == kNone) continue;
            groups_meet(o[j]);
            float y[C];   // columns C lane ..: of those that lane C lane / 8 has
#pragma unroll
            for (uint32_t c = 0; c < 8u; ++c) {
                const float x = __shfl_sync(0xffffffffu, o[j][c], C * lane / 8u);
                if (c / C == C * lane % 8u / C) y[c % C] = x;
            }
#pragma unroll
            for (uint32_t d = 1; d < 32u; d <<= 1) l[j] += __shfl_xor_sync(0xffffffffu, l[j], d);
            if (whole) {
                finish_row<C>(pc, token(row[j]), head(row[j]), m[j], l[j], y);
            } else {
                float* to_row = slot + (uint64_t)(row[j] - p.r0) * (D + 4u);
                if (lane == 0u) *reinterpret_cast<float2*>(to_row) = make_float2(m[j], l[j]);
#pragma unroll
                for (uint32_t c = 0; c < C; ++c) to_row[4u + C * lane + c] = y[c];
            }
        }
        return mask;
    }
};
template <uint32_t C, uint32_t ROWS>
__device__ __noinline__ void seen_keys_rows(const Args& pc, const Stretch& st, const uint32_t* s_pref, uint32_t hb, uint32_t first_row, uint32_t count) {
    Walk<ROWS> walk(st);
    while (walk.next(pc, s_pref)) {
        const Piece& p = walk.p;
        const uint32_t hkv = p.group * pc.HB + hb, lane = threadIdx.x & 31u, sub = lane % (4u * C);
        if (hkv >= pc.n_head_kv) continue;
        const Again<C, ROWS> x = {pc, p, hkv, lane, sub, lane - sub, p.a == 0u && p.b == p.n,
                                  pc.slots + ((uint64_t)(2u * blockIdx.x + (p.a == 0u ? 1u : 0u)) * pc.HB + hb) * ROWS * (32u * C + 4u)};
        const uint32_t from = (p.first + p.a) << pc.keys_log2, to = (p.first + p.b) << pc.keys_log2;
        const uint32_t base = p.r0 + first_row, end = min(p.R, base + count);
        uint32_t mask = 0u, low = 0u, high = 0u;   // rows that are not finite, the first and the last of them
        for (uint32_t r = base; r < end; ++r)
            if (!x.finite(r)) {
                low = mask ? low : r;
                high = r;
                mask |= 1u << (r - base);
            }
        if (!mask) continue;
        const uint32_t a = max(row_span(pc, p.q, high).lo, from), b = max(a, min(row_span(pc, p.q, low).hi, to));   // seen by all of them
        float common[8];
#pragma unroll
        for (uint32_t c = 0; c < 8u; ++c) common[c] = 0.0f;
        const bool plain = x.look_through(a, b, common);
        x.groups_meet(common);
        uint32_t anew = 0u;
        for (uint32_t left = mask; left; left &= left - 1u) {
            const uint32_t i = (uint32_t)__ffs(left) - 1u;
            if (!plain || !x.from_sums(base + i, from, to, a, b, common, plain)) anew |= 1u << i;
        }
        while (anew) anew = x.from_keys(anew, base, from, to);
    }
}

}  // namespace paged
}  // namespace amv
