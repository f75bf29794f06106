// Attention of single query rows over the 8-bit paged cache (layout: kv8.cu), split over the keys and merged.
//
//   s[u] = scale * q.K[u] (capped), K[u] = code * scale of u's page;  softmax over the keys that the mask leaves;  o = sum_u p[u] V[u]
//
// Bound by the bytes of the pages.  A warp takes one page of 64 keys and up to HEADS query heads that share its key head: two bulk
// copies bring the page's keys and values into shared memory (all pages of a block are on their way at once, from the first instruction
// on), 16-bit products on mma.m16n8k16 take them from there.
//
//   scores   left operand: 16 keys, right: the heads.  A lane's 16 bytes of a key's row are its part of four steps; which dims meet in
//            a step is free, so the queries are laid out the same way.  A code, as the low byte of a 16-bit float 1024 beside its upper
//            byte, is 1024 + 128 + code once its sign bit is flipped, and 1152 less the code, exactly.  The page's scale joins the 32-bit score.
//   weights  p = 2^(s - m + 15), m the page's own maximum: 16-bit floats from 2^15 down to 2^-24 hold weights of 2^-29 and more with all
//            11 bits, and the rest to 2^-40.
//   values   left operand: 16 dims of the values' transpose, right: the heads' weights, turned by movmatrix from the scores' layout.  Row g of
//            tile j is dim 16 g + 2 j, row g + 8 the next: a lane's 16 bytes of a key are its part of eight tiles.  The page's scale joins the sums.
//
// bfloat16 queries, scaled by a power of two to below 2, are 16-bit floats exactly (numbers below 2^-14 of the row's largest to 2^-25 of it).  float32
// queries and their weights are two columns, a 16-bit float and the 16-bit float of what it leaves, 22 bits together; their products are
// added up outside the tensor unit, which cuts off, in rounded 32-bit additions.
//
// A split's keys depend on positions only and the merge adds splits in ascending order, so a row's result depends on its own sequence
// only, not on the batch or on where its pages lie.
#include "common.cuh"
#include "sm100.cuh"
#include "per_device.h"

#include <cuda_fp16.h>

namespace {

constexpr int PAGE = 64;

struct DecodeArgs {
    void* out;
    float* partial;                                      // [rows][heads][splits][dv + 2]
    const void* q;
    const int8_t *k_cache, *v_cache;
    const float *k_scale, *v_scale, *sink;
    const int32_t *tok_slot, *tok_pos, *page_table;
    size_t ldo, ldq;
    int max_pages, n_slots, n_pages, n_heads, n_kv_heads, dk, dv, window, chunk, keep_first, splits, out_f32;
    float scale, softcap;
    int32_t* status;
};

__device__ __forceinline__ int first_key(const DecodeArgs& p, int pos) {
    return p.chunk > 0 ? pos - pos % p.chunk : p.window > 0 ? max(0, pos - p.window + 1) : 0;
}

// 2^x on the special-function unit (relative error about 2^-22; -inf gives 0, NaN NaN).
__device__ __forceinline__ float fast_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The same; EXACT: the sum rounded, from a product that starts at zero.
template <bool EXACT>
__device__ __forceinline__ void mma_sum(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if (EXACT) {
        float d[4] = {0.f, 0.f, 0.f, 0.f};
        mma_f16(d, a0, a1, a2, a3, b0, b1);
#pragma unroll
        for (int e = 0; e < 4; ++e) c[e] += d[e];
    } else {
        mma_f16(c, a0, a1, a2, a3, b0, b1);
    }
}

// Two codes (bytes of a word whose sign bits are flipped) as 16-bit floats.
__device__ __forceinline__ uint32_t two_codes(uint32_t flipped, int selector) {
    uint32_t r, v = __byte_perm(flipped, 0x64646464u, selector);
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(v), "r"(0x64806480u));
    return r;
}

__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 unpack_f16(uint32_t h) { return __half22float2(*reinterpret_cast<const __half2*>(&h)); }

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(sm100::smem_u32(dst)), "l"(src), "r"(bytes), "r"(sm100::smem_u32(bar)) : "memory");
}

// KC: blocks of 64 dims that keys span at most; VB: blocks of 128 dims of the values; WARPS pages to a block.
template <typename T, int KC, int VB, int WARPS>
__global__ void __launch_bounds__(WARPS * 32)
kv8_decode_kernel(const DecodeArgs p) {
    constexpr bool WIDE = sizeof(T) == 4;                // two columns to a head
    constexpr int HEADS = WIDE ? 4 : 8, SPLIT = WARPS * PAGE;
    extern __shared__ __align__(128) uint8_t smem[];     // per warp: its page's keys, its values; in the end [WARPS][HEADS][dv] sums
    __shared__ uint64_t bars[WARPS][2];
    __shared__ float s_m[WARPS][HEADS], s_l[WARPS][HEADS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    grid_dep_launch();
    if (lane == 0) {
        sm100::mbar_init(&bars[warp][0], 1);
        sm100::mbar_init(&bars[warp][1], 1);
        sm100::mbar_fence_init();
        sm100::fence_proxy_async_smem();
    }
    __syncwarp();
    grid_dep_wait();
    const int per = p.n_heads / p.n_kv_heads, head_tiles = (per + HEADS - 1) / HEADS;
    const int split = blockIdx.x, kvh = blockIdx.y / head_tiles, row = blockIdx.z;
    const int head0 = kvh * per + blockIdx.y % head_tiles * HEADS, heads = min(HEADS, per - blockIdx.y % head_tiles * HEADS);
    const int slot = p.tok_slot[row], pos = p.tok_pos[row];
    if (slot < 0 || slot >= p.n_slots || pos < 0 || (pos >> 6) >= p.max_pages || pos >= p.splits * SPLIT) {
        if (slot >= 0 && threadIdx.x == 0 && split == 0 && blockIdx.y == 0) atomicExch(p.status, 1);
        if (p.splits == 1)                               // no merge: the row's zeros are written here
            for (int i = threadIdx.x; i < heads * p.dv; i += WARPS * 32) store_from_f32(p.out, p.out_f32 ? QS_F32 : QS_BF16, (size_t)row * p.ldo + (size_t)head0 * p.dv + i, 0.f);
        return;
    }
    const int first = first_key(p, pos), keep = p.window > 0 ? min(p.keep_first, first) : 0;
    const int base = split * SPLIT;
    if (base > pos || (base + SPLIT <= first && base >= keep)) return;       // no key of this split is seen
    const int key0 = base + warp * PAGE;
    const bool seen = key0 <= pos && (key0 + PAGE > first || key0 < keep);
    int page = -1;
    if (seen) {
        page = p.page_table[(size_t)slot * p.max_pages + (key0 >> 6)];
        if (page < 0 || page >= p.n_pages) { if (lane == 0) atomicExch(p.status, 3); page = -1; }
    }
    const int page_bytes = PAGE * (p.dk + p.dv) + 128;   // rows are read in whole blocks of dims: up to 127 bytes beyond the last
    uint8_t* keys = smem + warp * page_bytes;
    uint8_t* values = keys + PAGE * p.dk;
    const size_t at = (size_t)max(page, 0) * p.n_kv_heads + kvh;
    if (page >= 0 && lane == 0) {
        const int n = min(PAGE, pos - key0 + 1);         // rows behind the sequence's end stay out of it
        sm100::mbar_expect_tx(&bars[warp][0], n * p.dk);
        bulk_load(keys, p.k_cache + at * PAGE * p.dk, n * p.dk, &bars[warp][0]);
        sm100::mbar_expect_tx(&bars[warp][1], n * p.dv);
        bulk_load(values, p.v_cache + at * PAGE * p.dv, n * p.dv, &bars[warp][1]);
    }
    const float ks = page >= 0 ? p.k_scale[at] : 0.f, vs = page >= 0 ? p.v_scale[at] : 0.f;

    // the queries: column g is head g (WIDE: head g & 3, its first or second term), dims 64 c + 16 t .. + 15
    uint32_t qf[KC][8];
    float q_unit = 0.f;                                  // what one of column g's numbers stands for
    {
        const int h = WIDE ? g & 3 : g;
        const T* src = reinterpret_cast<const T*>(p.q) + (size_t)row * p.ldq + (size_t)(head0 + min(h, heads - 1)) * p.dk;
        float most = 0.f;
        float f[WIDE ? 1 : KC][WIDE ? 1 : 16];
#pragma unroll
        for (int c = 0; c < KC; ++c)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int d = 64 * c + 16 * t + i;
                const float x = d < p.dk ? to_f32(src[d]) : 0.f;
                if (!WIDE) f[WIDE ? 0 : c][WIDE ? 0 : i] = x;
                most = fmaxf(most, fabsf(x));
            }
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
        // the power of two at or below the largest; numbers that are not finite go through as they are
        const uint32_t e = min(max(__float_as_uint(most) >> 23, 1u), 253u);
        q_unit = __uint_as_float(e << 23);
        const float inv = __uint_as_float((254u - e) << 23);
#pragma unroll
        for (int c = 0; c < KC; ++c)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                float x[2];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int d = 64 * c + 16 * t + 2 * i + j;
                    x[j] = (WIDE ? (d < p.dk ? to_f32(src[d]) : 0.f) : f[WIDE ? 0 : c][WIDE ? 0 : 2 * i + j]) * inv;
                }
                uint32_t v = pack_f16(x[0], x[1]);
                if (WIDE && g >= 4) {
                    const float2 hi = unpack_f16(v);
                    v = pack_f16(x[0] - hi.x, x[1] - hi.y);
                }
                qf[c][i] = v;
            }
    }
    // of the columns that this lane's results belong to: 2 t, 2 t + 1 (WIDE: of their heads, in both halves)
    const int h0 = WIDE ? 2 * (t & 1) : 2 * t;
    float unit[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) unit[j] = __shfl_sync(0xffffffffu, q_unit, (h0 + j) * 4) * ks * p.scale;

    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    float acc[VB * 8][4];
#pragma unroll
    for (int j = 0; j < VB * 8; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
    const bool ok = page >= 0 && sm100::mbar_wait(&bars[warp][0], 0);
    if (page >= 0 && !ok && lane == 0) atomicExch(p.status, 123);
    if (ok) {
        // scores of the page's 64 keys: tile i, row g (and g + 8) is key 16 i + g (+ 8)
        float s[4][4];
        const float log2e = 1.4426950408889634f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.f;
#pragma unroll
            for (int c = 0; c < KC; ++c) {
                if (64 * c >= p.dk) break;
                const uint4 lo = *reinterpret_cast<const uint4*>(keys + (16 * i + g) * p.dk + 64 * c + 16 * t);
                const uint4 hi = *reinterpret_cast<const uint4*>(keys + (16 * i + g + 8) * p.dk + 64 * c + 16 * t);
                const uint32_t a[4] = {lo.x ^ 0x80808080u, lo.y ^ 0x80808080u, lo.z ^ 0x80808080u, lo.w ^ 0x80808080u};
                const uint32_t b[4] = {hi.x ^ 0x80808080u, hi.y ^ 0x80808080u, hi.z ^ 0x80808080u, hi.w ^ 0x80808080u};
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    mma_sum<WIDE>(s[i], two_codes(a[k], 0x4140), two_codes(b[k], 0x4140), two_codes(a[k], 0x4342), two_codes(b[k], 0x4342), qf[c][2 * k], qf[c][2 * k + 1]);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int key = key0 + 16 * i + g + 8 * (e >> 1);
                float x = s[i][e];
                if (WIDE) x += __shfl_xor_sync(0xffffffffu, x, 2);
                x *= unit[e & 1];
                if (p.softcap > 0.f) x = p.softcap * tanhf(x / p.softcap);
                s[i][e] = key <= pos && (key >= first || key < keep) ? x * log2e : -INFINITY;
                m[e & 1] = fmaxf(m[e & 1], s[i][e]);
            }
        }
        // the weights, in pairs of heads; the columns' maxima and sums over the eight lanes of a column
        uint32_t w[4][2];                                // tile i, rows g and g + 8: two heads
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) m[j] = fmaxf(m[j], __shfl_xor_sync(0xffffffffu, m[j], o));
        const float zero[2] = {m[0] == -INFINITY ? 0.f : m[0] - 15.f, m[1] == -INFINITY ? 0.f : m[1] - 15.f};     // all -inf (or NaN): 2^-inf is 0
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float a = fast_exp2(s[i][2 * e] - zero[0]), b = fast_exp2(s[i][2 * e + 1] - zero[1]);
                l[0] += a;
                l[1] += b;
                uint32_t v = pack_f16(a, b);
                if (WIDE && t >= 2) {
                    const float2 hi = unpack_f16(v);
                    v = pack_f16(a - hi.x, b - hi.y);
                }
                asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(w[i][e]) : "r"(v));
            }
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) l[j] += __shfl_xor_sync(0xffffffffu, l[j], o);
        if (sm100::mbar_wait(&bars[warp][1], 0)) {
#pragma unroll
            for (int i = 0; i < 4; ++i)                  // 16 keys: this lane's are 2 t, 2 t + 1 and the same + 8
#pragma unroll
                for (int b = 0; b < VB; ++b) {
                    if (128 * b >= p.dv) break;
                    const uint8_t* v = values + (16 * i + 2 * t) * p.dv + 128 * b + 16 * g;
                    uint4 x[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        x[e] = *reinterpret_cast<const uint4*>(v + ((e & 1) + 8 * (e >> 1)) * p.dv);
                        x[e].x ^= 0x80808080u; x[e].y ^= 0x80808080u; x[e].z ^= 0x80808080u; x[e].w ^= 0x80808080u;
                    }
#pragma unroll
                    for (int k = 0; k < 4; ++k) {        // four dims: tiles 2 k and 2 k + 1
                        const uint32_t x0 = k == 0 ? x[0].x : k == 1 ? x[0].y : k == 2 ? x[0].z : x[0].w, x1 = k == 0 ? x[1].x : k == 1 ? x[1].y : k == 2 ? x[1].z : x[1].w;
                        const uint32_t x2 = k == 0 ? x[2].x : k == 1 ? x[2].y : k == 2 ? x[2].z : x[2].w, x3 = k == 0 ? x[3].x : k == 1 ? x[3].y : k == 2 ? x[3].z : x[3].w;
                        const uint32_t n0 = __byte_perm(x0, x1, 0x5140), n1 = __byte_perm(x0, x1, 0x7362), f0 = __byte_perm(x2, x3, 0x5140), f1 = __byte_perm(x2, x3, 0x7362);
                        mma_sum<WIDE>(acc[8 * b + 2 * k], two_codes(n0, 0x4140), two_codes(n0, 0x4342), two_codes(f0, 0x4140), two_codes(f0, 0x4342), w[i][0], w[i][1]);
                        mma_sum<WIDE>(acc[8 * b + 2 * k + 1], two_codes(n1, 0x4140), two_codes(n1, 0x4342), two_codes(f1, 0x4140), two_codes(f1, 0x4342), w[i][0], w[i][1]);
                    }
                }
        } else if (lane == 0) {
            atomicExch(p.status, 124);
        }
    }
    // The warps' results: sums as [head][dim], beside each other where the pages were.
    if (g == 0 && (!WIDE || t < 2)) { s_m[warp][h0] = m[0]; s_m[warp][h0 + 1] = m[1]; s_l[warp][h0] = l[0]; s_l[warp][h0 + 1] = l[1]; }
    __syncthreads();                                     // everybody has read its page
    float* sums = reinterpret_cast<float*>(smem);
#pragma unroll
    for (int j = 0; j < VB * 8; ++j) {
        const int d = (j >> 3) * 128 + 16 * g + 2 * (j & 7);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (WIDE) acc[j][e] += __shfl_xor_sync(0xffffffffu, acc[j][e], 2);
            acc[j][e] = page >= 0 ? acc[j][e] * vs : 0.f;
        }
        if (d < p.dv && (!WIDE || t < 2)) {
            *reinterpret_cast<float2*>(sums + (warp * HEADS + h0) * p.dv + d) = make_float2(acc[j][0], acc[j][2]);
            *reinterpret_cast<float2*>(sums + (warp * HEADS + h0 + 1) * p.dv + d) = make_float2(acc[j][1], acc[j][3]);
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < heads * p.dv; i += WARPS * 32) {
        const int h = i / p.dv, d = i - h * p.dv;
        float M = -INFINITY, L = 0.f, o = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) M = fmaxf(M, s_m[w][h]);
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {                // a page without a key that is seen: nothing; one whose scores are all NaN: NaN
            const float a = s_m[w][h] == -INFINITY ? 1.f : exp2f(s_m[w][h] - M);
            L += s_l[w][h] * a;
            o += sums[(w * HEADS + h) * p.dv + d] * a;
        }
        if (p.splits == 1) {
            // as the merge of one split
            if (p.sink) {
                const float sink = p.sink[head0 + h] * 1.4426950408889634f, all = fmaxf(M, sink), a = M == -INFINITY ? 1.f : exp2f(M - all);
                L = fmaf(L, a, exp2f(sink - all + 15.f));
                o *= a;
            }
            store_from_f32(p.out, p.out_f32 ? QS_F32 : QS_BF16, (size_t)row * p.ldo + (size_t)(head0 + h) * p.dv + d, o * (L != 0.f ? 1.0f / L : 0.f));
        } else {
            float* to = p.partial + (((size_t)row * p.n_heads + head0 + h) * p.splits + split) * (p.dv + 2);
            to[d] = o;
            if (d == 0) { to[p.dv] = M; to[p.dv + 1] = L; }
        }
    }
}

// One block per row and head: the splits' results in ascending order.
template <int SPLIT>
__global__ void kv8_merge_kernel(const DecodeArgs p) {
    extern __shared__ float s_all[];                     // [splits] weights, [splits] sums
    grid_dep_launch();
    grid_dep_wait();
    const int head = blockIdx.x, row = blockIdx.y, dv = p.dv;
    const int slot = p.tok_slot[row], pos = p.tok_pos[row];
    const size_t to = (size_t)row * p.ldo + (size_t)head * dv;
    if (slot < 0 || slot >= p.n_slots || pos < 0 || (pos >> 6) >= p.max_pages || pos >= p.splits * SPLIT) {       // padding, or reported: a defined row
        for (int d = threadIdx.x; d < dv; d += blockDim.x) store_from_f32(p.out, p.out_f32 ? QS_F32 : QS_BF16, to + d, 0.f);
        return;
    }
    const int first = first_key(p, pos), keep = p.window > 0 ? min(p.keep_first, first) : 0;
    // the splits with keys that are seen: those of the kept first keys, then those of the window
    const int kept = keep > 0 ? (keep - 1) / SPLIT + 1 : 0, lo = max(first / SPLIT, kept), n = kept + pos / SPLIT - lo + 1;
    const float* base = p.partial + ((size_t)row * p.n_heads + head) * p.splits * (dv + 2);
    auto part = [&](int i) { return base + (size_t)(i < kept ? i : lo + i - kept) * (dv + 2); };
    __shared__ float scratch[33];
    float M = p.sink ? p.sink[head] * 1.4426950408889634f : -INFINITY;
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
        s_all[i] = part(i)[dv];
        s_all[n + i] = part(i)[dv + 1];
        M = fmaxf(M, s_all[i]);
    }
    M = warp_max(M);
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = M;
    __syncthreads();
    for (int i = 0; i < (int)(blockDim.x >> 5); ++i) M = fmaxf(M, scratch[i]);
    for (int i = threadIdx.x; i < n; i += blockDim.x) s_all[i] = s_all[i] == -INFINITY ? 1.f : exp2f(s_all[i] - M);
    __syncthreads();
    float L = p.sink ? exp2f(p.sink[head] * 1.4426950408889634f - M + 15.f) : 0.f;
    for (int i = 0; i < n; ++i) L = fmaf(s_all[n + i], s_all[i], L);
    const float inv = L != 0.f ? 1.0f / L : 0.f;
    constexpr int AHEAD = 8;
    for (int d = threadIdx.x; d < dv; d += blockDim.x) {
        float acc = 0.f;
        for (int i0 = 0; i0 < n; i0 += AHEAD) {
            float v[AHEAD];
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) v[u] = i0 + u < n ? part(i0 + u)[d] : 0.f;
#pragma unroll
            for (int u = 0; u < AHEAD; ++u)
                if (i0 + u < n) acc = fmaf(v[u], s_all[i0 + u], acc);
        }
        store_from_f32(p.out, p.out_f32 ? QS_F32 : QS_BF16, to + d, acc * inv);
    }
}

// Keys of a block: four pages, two where they are wide (a block's pages then fill half of the shared memory of an SM as before).
int split_keys(int dk, int dv) { return dk > 128 || dv > 128 ? 2 * PAGE : 4 * PAGE; }

template <typename T, int KC, int VB, int WARPS>
int go(const DecodeArgs& p, int rows, cudaStream_t stream) {
    constexpr int HEADS = sizeof(T) == 4 ? 4 : 8;
    const int pages = WARPS * (PAGE * (p.dk + p.dv) + 128), sums = WARPS * HEADS * p.dv * 4, smem = pages > sums ? pages : sums;
    static PerDevice limit;
    int device = 0;
    cudaGetDevice(&device);
    limit.get(device, [] { return cudaFuncSetAttribute(kv8_decode_kernel<T, KC, VB, WARPS>, cudaFuncAttributeMaxDynamicSharedMemorySize, 100 * 1024) == cudaSuccess ? 1 : 0; });
    const int per = p.n_heads / p.n_kv_heads;
    cudaError_t e = qs_launch_dependent(kv8_decode_kernel<T, KC, VB, WARPS>, dim3(p.splits, p.n_kv_heads * ((per + HEADS - 1) / HEADS), rows), dim3(WARPS * 32), (size_t)smem, stream, p);
    if (e == cudaSuccess && p.splits > 1)
        e = qs_launch_dependent(kv8_merge_kernel<WARPS * PAGE>, dim3(p.n_heads, rows), dim3(p.dv > 64 ? 128 : 64), (size_t)2 * p.splits * sizeof(float), stream, p);
    if (e != cudaSuccess) return qs_fail(QS_ERR_INTERNAL, "kv8 decode: %s", cudaGetErrorString(e));
    return qs_check_launch("kv8 decode");
}

}  // namespace

// Splits of the keys that a call is made for (1: no merge, no workspace).
QS_API int qs_kv8_decode_splits(int dk, int dv, int max_context) { return (max_context + split_keys(dk, dv) - 1) / split_keys(dk, dv); }

// out [T, n_heads * dv] (bfloat16, or float32 with out_f32), q [T, n_heads * dk] of type `dtype`; head sizes multiples of 16 up to 256.  `partial`: float32
// [T][n_heads][splits][dv + 2] with qs_kv8_decode_splits(dk, dv, max_context) splits; contents need no initialisation; may be null for one split.
// Masks, status codes and rows as for qs_kv8_attention; positions lie below max_context rounded up to whole splits.
QS_API int qs_kv8_decode(void* out, int out_f32, long long ldo, const void* q, int dtype, long long ldq, int T_tokens, const int32_t* tok_slot,
                         const int32_t* tok_pos, const int32_t* page_table, int n_slots, int max_pages, int n_pages, const int8_t* k_cache,
                         const int8_t* v_cache, const float* k_scale, const float* v_scale, int n_heads, int n_kv_heads, int dk, int dv, float scale,
                         int window, int chunk, int keep_first, const float* sink, float softcap, int max_context, float* partial, int32_t* status,
                         cudaStream_t stream) {
    if (T_tokens == 0) return QS_OK;
    QS_REQUIRE(T_tokens > 0 && T_tokens <= 65535 && n_heads > 0 && n_kv_heads > 0 && n_heads % n_kv_heads == 0 && n_heads <= 65535 && n_slots > 0 && max_pages > 0 &&
               n_pages > 0 && max_context > 0, "kv8 decode: bad sizes");
    QS_REQUIRE(dk % 16 == 0 && dv % 16 == 0 && dk >= 16 && dv >= 16 && dk <= 256 && dv <= 256, "kv8 decode: head sizes %d and %d (multiples of 16 up to 256)", dk, dv);
    QS_REQUIRE(chunk >= 0 && window >= 0 && keep_first >= 0 && !(chunk > 0 && window > 0), "kv8 decode: a window of %d and chunks of %d", window, chunk);
    QS_REQUIRE(((uintptr_t)k_cache % 16) == 0 && ((uintptr_t)v_cache % 16) == 0, "kv8 decode: pages off their 16-byte boundary");
    QS_REQUIRE(dtype == QS_BF16 || (dtype == QS_F32 && out_f32), "kv8 decode: queries of type %d", dtype);
    const int splits = qs_kv8_decode_splits(dk, dv, max_context);
    QS_REQUIRE(splits <= 4096, "kv8 decode: a context of %d exceeds what the merge holds (%d)", max_context, 4096 * split_keys(dk, dv));
    QS_REQUIRE(splits == 1 || partial, "kv8 decode: no workspace");
    const DecodeArgs p = {out, partial, q, k_cache, v_cache, k_scale, v_scale, sink, tok_slot, tok_pos, page_table, (size_t)ldo, (size_t)ldq,
                          max_pages, n_slots, n_pages, n_heads, n_kv_heads, dk, dv, window, chunk, keep_first, splits, out_f32, scale, softcap, status};
#define GO(T) do { if (dk <= 64 && dv <= 128) return go<T, 1, 1, 4>(p, T_tokens, stream); \
                   if (dk <= 128 && dv <= 128) return go<T, 2, 1, 4>(p, T_tokens, stream); \
                   return go<T, 4, 2, 2>(p, T_tokens, stream); } while (0)
    if (dtype == QS_F32) GO(float);
    GO(__nv_bfloat16);
#undef GO
}
