// ameva_paged_append: the projected rows of a step's tokens into a paged KV cache. Queries and keys are rotated to their positions
// (ROPE, NORMAL and NEOX, frequency factors, YaRN) on the way, queries to an f16 tensor for the attention kernels, keys and values
// to the pages that the sequences' tables name. One pass: what ameva_rope (twice), ameva_cpy and ameva_set_rows (twice) take five
// over the same rows.
//
//   angle(t, j) = pos_t * theta_scale^j / ff_j, scaled and mixed as ameva_rope does; y0 = x0 cos - x1 sin, y1 = x0 sin + x1 cos
//
// Unlike there, whose angles repeat ggml's 32-bit products, the angle is formed in 64 bits and brought into one turn before it is
// rounded: a 32-bit angle of position 300000 is off by up to 0.02 of a radian, which the rotated element would show. A CTA takes T
// tokens: their angles by one thread each (64-bit products: theta_scale^j by squaring), then every thread rotates 8 elements of a
// head at a time from 16-byte loads. Bound by HBM: 6 (H + 2 Hkv) D bytes per token: 8335 tokens of 48 heads of 128 in 60 us (307 MB, 5.1
// TB/s; 65 us with as many CTAs per SM as the registers allow without a bound); 211 tokens 10 us, one 6.5 us: latency.
#include <algorithm>
#include <cstring>

#include "paged.cuh"

namespace amv {
namespace paged {

struct AppendArgs {
    uint32_t D, n_head, n_head_kv, n_seqs, rows, page_size, n_pages, table_stride, c_ps, c_ts, c_hs, q_s, k_s, v_s, o_s, n_dims, neox, flags,
        theta_scale, freq_scale, ext_factor, attn_factor, corr0, corr1, node;
};
constexpr uint32_t kHasPositions = 1u, kHasFactors = 2u;
constexpr uint32_t kMaxTokens = 2, kMaxHeadDim = 256;

__device__ __forceinline__ float as_f(uint32_t u) { return __uint_as_float(u); }

// sine and cosine of `angle` (radians), reduced to one turn in 64 bits
__device__ __forceinline__ float2 turn(double angle, float magnitude) {
    const double turns = angle * 0.15915494309189533577;   // 1 / (2 pi)
    const float x = (float)(2.0 * (turns - rint(turns)));
    float s, c;
    sincospif(x, &s, &c);
    return make_float2(c * magnitude, s * magnitude);
}

__device__ __forceinline__ uint4 pack8(const float (&x)[8]) {
    uint4 r;
    __half2 h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
    memcpy(&r, h, 16);
    return r;
}

template <bool VEC>
__global__ void __launch_bounds__(256, 8) append_kernel(const float* __restrict__ q, const float* __restrict__ k, const float* __restrict__ v,
                                                     const int32_t* __restrict__ table, const int32_t* __restrict__ q_start,
                                                     const int32_t* __restrict__ kv_len, const int32_t* __restrict__ positions,
                                                     const float* __restrict__ factors, __half* __restrict__ q_out, __half* __restrict__ k_cache,
                                                     __half* __restrict__ v_cache, uint32_t* refused, const AppendArgs pc, const uint32_t T) {
    __shared__ __align__(16) float2 s_turn[kMaxTokens][kMaxHeadDim / 2];
    __shared__ int64_t s_slot[kMaxTokens];   // element of the token's first head in the caches, -1: nothing of the token is written
    __shared__ int32_t s_pos[kMaxTokens];
    pdl_trigger();
    pdl_wait();
    const uint32_t t0 = blockIdx.x * T, tokens = min(T, pc.rows - t0), half = pc.n_dims >> 1;
    if (threadIdx.x < tokens) {
        const int32_t t = (int32_t)(t0 + threadIdx.x);
        int64_t slot = -1;
        int32_t pos = 0;
        if (t < q_start[pc.n_seqs] && t >= q_start[0]) {   // (rows behind the last sequence are left as they are)
            uint32_t lo = 0, hi = pc.n_seqs;               // the sequence: q_start[lo] <= t < q_start[lo + 1]
            while (hi - lo > 1u) {
                const uint32_t mid = (lo + hi) >> 1;
                if (q_start[mid] <= t) lo = mid;
                else hi = mid;
            }
            const int32_t a = q_start[lo], b = q_start[lo + 1u], kv = kv_len[lo];
            const int64_t place = (int64_t)kv - b + t;
            bool ok = a <= t && t < b && a >= 0 && (uint32_t)b <= pc.rows && place >= 0 && place < (int64_t)pc.table_stride * pc.page_size;
            if (ok) {
                const uint32_t n = (uint32_t)place / pc.page_size, in_page = (uint32_t)place - n * pc.page_size;
                const int32_t page = table[(uint64_t)lo * pc.table_stride + n];
                ok = page >= 0 && (uint32_t)page < pc.n_pages;
                slot = (int64_t)page * pc.c_ps + (int64_t)in_page * pc.c_ts;
                pos = pc.flags & kHasPositions ? positions[t] : (int32_t)place;
            }
            if (!ok) {
                slot = -1;
                atomicAdd(refused, 1u);
                atomicMin(refused + 1, pc.node);
            }
        }
        s_slot[threadIdx.x] = slot;
        s_pos[threadIdx.x] = pos;
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < tokens * half; i += 256u) {
        const uint32_t t = i / half, j = i - t * half;
        if (s_slot[t] < 0) continue;
        double power = 1.0, square = (double)as_f(pc.theta_scale);
        for (uint32_t e = j; e; e >>= 1) {
            if (e & 1u) power *= square;
            square *= square;
        }
        double far = (double)s_pos[t] * power;
        if (pc.flags & kHasFactors) far /= (double)factors[j];
        float magnitude = as_f(pc.attn_factor);
        const float freq_scale = as_f(pc.freq_scale), ext = as_f(pc.ext_factor);
        double angle = far * (double)freq_scale;
        if (ext != 0.0f) {
            const double low = as_f(pc.corr0), high = as_f(pc.corr1);
            const double y = ((double)j - low) / fmax(0.001, high - low);
            const double ramp = (1.0 - fmin(1.0, fmax(0.0, y))) * (double)ext;
            angle = angle * (1.0 - ramp) + far * ramp;
            magnitude *= 1.0f + 0.1f * logf(1.0f / freq_scale);
        }
        s_turn[t][j] = turn(angle, magnitude);
    }
    __syncthreads();
    const uint32_t heads = pc.n_head + 2u * pc.n_head_kv;
    auto source = [&](uint32_t t, uint32_t h) -> const float* {
        const uint64_t row = t0 + t;
        if (h < pc.n_head) return q + row * pc.q_s + (uint64_t)h * pc.D;
        h -= pc.n_head;
        if (h < pc.n_head_kv) return k + row * pc.k_s + (uint64_t)h * pc.D;
        return v + row * pc.v_s + (uint64_t)(h - pc.n_head_kv) * pc.D;
    };
    auto target = [&](uint32_t t, uint32_t h) -> __half* {
        if (h < pc.n_head) return q_out + (uint64_t)(t0 + t) * pc.o_s + (uint64_t)h * pc.D;
        h -= pc.n_head;
        __half* cache = h < pc.n_head_kv ? k_cache : v_cache;
        return cache + s_slot[t] + (uint64_t)(h < pc.n_head_kv ? h : h - pc.n_head_kv) * pc.c_hs;
    };
    if (VEC) {   // units of eight elements: four pairs of a rotated head, or eight elements beside one another that are copied
        const uint32_t units = pc.D >> 3, all = tokens * heads * units, rotated_units = pc.n_dims >> 3;
#pragma unroll 1
        for (uint32_t i = threadIdx.x; i < all; i += 256u) {
            const uint32_t row = i / units, u = i - row * units, t = row / heads, h = row - t * heads;
            if (s_slot[t] < 0) continue;
            const bool turned = h < pc.n_head + pc.n_head_kv && u < rotated_units;
            const bool neox = turned && pc.neox;
            const uint32_t e0 = neox ? 4u * u : 8u * u, e1 = neox ? e0 + half : e0 + 4u;
            const float* src = source(t, h);
            const float4 x0 = __ldcs(reinterpret_cast<const float4*>(src + e0)), x1 = __ldcs(reinterpret_cast<const float4*>(src + e1));
            float x[8] = {x0.x, x0.y, x0.z, x0.w, x1.x, x1.y, x1.z, x1.w};
            if (turned) {
                const float4* at = reinterpret_cast<const float4*>(&s_turn[t][4u * u]);
                const float4 a = at[0], b = at[1];
                const float c[4] = {a.x, a.z, b.x, b.z}, s[4] = {a.y, a.w, b.y, b.w};
#pragma unroll
                for (int p = 0; p < 4; ++p) {
                    const float a0 = neox ? x[p] : x[2 * p], a1 = neox ? x[p + 4] : x[2 * p + 1];
                    const float y0 = a0 * c[p] - a1 * s[p], y1 = a0 * s[p] + a1 * c[p];
                    if (neox) {
                        x[p] = y0;
                        x[p + 4] = y1;
                    } else {
                        x[2 * p] = y0;
                        x[2 * p + 1] = y1;
                    }
                }
            }
            const uint4 y = pack8(x);
            __half* dst = target(t, h);
            if (neox) {
                *reinterpret_cast<uint2*>(dst + e0) = make_uint2(y.x, y.y);
                *reinterpret_cast<uint2*>(dst + e1) = make_uint2(y.z, y.w);
            } else {
                *reinterpret_cast<uint4*>(dst + e0) = y;
            }
        }
    } else {     // one pair at a time: rotated widths that are no multiple of eight
        const uint32_t units = pc.D >> 1, all = tokens * heads * units;
        for (uint32_t i = threadIdx.x; i < all; i += 256u) {
            const uint32_t row = i / units, j = i - row * units, t = row / heads, h = row - t * heads;
            if (s_slot[t] < 0) continue;
            const bool turned = h < pc.n_head + pc.n_head_kv && j < half;
            const uint32_t e0 = turned && pc.neox ? j : 2u * j, e1 = turned && pc.neox ? j + half : 2u * j + 1u;
            const float* src = source(t, h);
            const float x0 = src[e0], x1 = src[e1];
            const float2 cs = turned ? s_turn[t][j] : make_float2(1.0f, 0.0f);
            __half* dst = target(t, h);
            dst[e0] = __float2half_rn(turned ? x0 * cs.x - x1 * cs.y : x0);
            dst[e1] = __float2half_rn(turned ? x0 * cs.y + x1 * cs.x : x1);
        }
    }
}

}  // namespace paged

// Whether (pages, tokens, heads) of D elements with these strides lie beside one another, in whatever order.
static bool strides_apart(uint64_t D, uint64_t ps, uint64_t pages, uint64_t ts, uint64_t tokens, uint64_t hs, uint64_t heads) {
    struct Dim {
        uint64_t stride, n;
    } dims[3] = {{ps, pages}, {ts, tokens}, {hs, heads}};
    std::sort(dims, dims + 3, [](const Dim& x, const Dim& y) { return x.stride < y.stride; });
    uint64_t span = D;
    for (const Dim& d : dims) {
        if (d.n == 1u) continue;
        if (d.stride < span) return false;
        span += d.stride * (d.n - 1u);
    }
    return true;
}
static bool ranges_meet(const LaunchArgs& a, uint32_t i, uint32_t j) {
    const uintptr_t p = (uintptr_t)a.ptr[i], q = (uintptr_t)a.ptr[j];
    return p < q + a.range[j] && q < p + a.range[i];
}

// ameva_paged_append: bindings 0 q, 1 k, 2 v (f32 rows of heads x D), 3 table i32 [n_seqs][table_stride], 4 q_start i32 [n_seqs + 1],
// 5 kv_len i32 [n_seqs], 6 positions i32 [rows] (any range when flags has no bit 0), 7 frequency factors f32 [n_dims / 2] (any range when
// flags has no bit 1), 8 q_out f16, 9 k cache f16, 10 v cache f16, 11 status (two words: count of refused tokens, lowest node).
// push: D, n_head, n_head_kv, n_seqs, rows, page size, pages, table stride, cache strides of page, token and head, row strides of q, k, v
// and q_out (all in elements), n_dims, neox, flags, theta_scale, freq_scale, ext_factor, attn_factor, corr0, corr1 (floats as bits), node.
// Token t of sequence s stands at place kv_len[s] - q_start[s + 1] + t of its keys; that is its position where none is given. A token
// whose place or page is none of the table's or the cache's is not written and counted; rows behind the last sequence are left as they
// are. Two tokens that name the same place leave either one's rows.
AcResult launch_paged_append(const LaunchArgs& a) {
    using namespace paged;
    AppendArgs pc;
    memcpy(&pc, a.push, sizeof(pc));
    if (!pc.D || !pc.n_head || !pc.n_head_kv || !pc.n_seqs || !pc.rows || !pc.page_size || !pc.n_pages || !pc.table_stride ||
        pc.neox > 1u || pc.flags > 3u || pc.n_dims > pc.D || (pc.n_dims & 1u))
        return AC_ERR_KERNEL_ARG_INVALID;
    if (pc.D > kMaxHeadDim || (pc.D & 7u)) return AC_ERR_FEATURE_NOT_SUPPORTED;
    if (pc.n_head > 65535u || pc.n_head_kv > 65535u || pc.rows > 0x7FFFFFFFu || pc.n_pages > 0x7FFFFFFFu ||
        (uint64_t)pc.table_stride * pc.page_size > 0x7FFFFFFFull)
        return AC_ERR_INVALID_SHAPE;
    if (((pc.q_s | pc.k_s | pc.v_s) & 3u) || ((pc.c_ps | pc.c_ts | pc.c_hs | pc.o_s) & 7u)) return AC_ERR_BUFFER_ALIGNMENT_INVALID;
    for (uint32_t i : {0u, 1u, 2u, 8u, 9u, 10u})
        if ((uintptr_t)a.ptr[i] & 15u) return AC_ERR_BUFFER_ALIGNMENT_INVALID;
    for (uint32_t i : {3u, 4u, 5u, 6u, 7u, 11u})
        if ((uintptr_t)a.ptr[i] & 3u) return AC_ERR_BUFFER_ALIGNMENT_INVALID;
    const uint64_t last = pc.rows - 1u, qw = (uint64_t)pc.n_head * pc.D, kw = (uint64_t)pc.n_head_kv * pc.D;
    const uint64_t cache = ((uint64_t)(pc.n_pages - 1u) * pc.c_ps + (uint64_t)(pc.page_size - 1u) * pc.c_ts + (uint64_t)(pc.n_head_kv - 1u) * pc.c_hs + pc.D) * 2u;
    if (a.range[0] < (last * pc.q_s + qw) * 4u || a.range[1] < (last * pc.k_s + kw) * 4u || a.range[2] < (last * pc.v_s + kw) * 4u ||
        a.range[3] < (uint64_t)pc.n_seqs * pc.table_stride * 4u || a.range[4] < ((uint64_t)pc.n_seqs + 1u) * 4u ||
        a.range[5] < (uint64_t)pc.n_seqs * 4u || ((pc.flags & kHasPositions) && a.range[6] < (uint64_t)pc.rows * 4u) ||
        ((pc.flags & kHasFactors) && a.range[7] < (uint64_t)(pc.n_dims / 2u) * 4u) || a.range[8] < (last * pc.o_s + qw) * 2u ||
        a.range[9] < cache || a.range[10] < cache || a.range[11] < 8u)
        return AC_ERR_INVALID_BUFFER_SIZE;
    if ((last && pc.o_s < qw) || !strides_apart(pc.D, pc.c_ps, pc.n_pages, pc.c_ts, pc.page_size, pc.c_hs, pc.n_head_kv)) return AC_ERR_INVALID_SHAPE;
    for (uint32_t o : {8u, 9u, 10u, 11u})   // what is written meets nothing else
        for (uint32_t i = 0; i < 12u; ++i) {
            const bool unused = (i == 6u && !(pc.flags & kHasPositions)) || (i == 7u && !(pc.flags & kHasFactors));
            if (i != o && !unused && ranges_meet(a, o, i)) return AC_ERR_KERNEL_ARG_INVALID;
        }
    const bool vec = !(pc.n_dims & 7u);
    // tokens per CTA: one while the CTAs do not fill the GPU (8335 tokens: one 61.9 us, two 60.2)
    const uint32_t T = pc.rows >= kMaxTokens * 8u * (uint32_t)a.sm_count ? kMaxTokens : 1u;
    const dim3 grid((pc.rows + T - 1u) / T);
    auto run = [&](auto* kernel) {
        launch_pdl(kernel, grid, dim3(256), 0, a.stream, (const float*)a.ptr[0], (const float*)a.ptr[1], (const float*)a.ptr[2],
                   (const int32_t*)a.ptr[3], (const int32_t*)a.ptr[4], (const int32_t*)a.ptr[5], (const int32_t*)a.ptr[6],
                   (const float*)a.ptr[7], (__half*)a.ptr[8], (__half*)a.ptr[9], (__half*)a.ptr[10], (uint32_t*)a.ptr[11], pc, T);
    };
    if (vec) run(append_kernel<true>);
    else run(append_kernel<false>);
    return check_launch();
}

}  // namespace amv
