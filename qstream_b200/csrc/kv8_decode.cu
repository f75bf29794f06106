// Attention of single query rows over the 8-bit paged cache (layout: kv8.cu), split over the keys and merged.
//
//   s[u] = scale * q.K[u] (capped), K[u] = code * scale of u's page;  softmax over the keys that the mask leaves;  o = sum_u p[u] V[u]
//
// Floor: the bytes of the pages.  A warp takes 32 keys and up to HEADS query heads that share their key head: a bulk
// copy brings the keys into shared memory, asynchronous copies the values, their rows apart (all of a block are on their way at once, from
// the first instructions on); 16-bit products on mma.m16n8k16 take them from there.  Bound by a block's life: its metadata's and pages' way from
// memory, one behind the other, then instructions, which fill half of the slots (heads of 128; two fifths, heads of 256).  (Blocks that stay on their SM and look for their next
// page's number beside the products: 31 rows of 2,048 29 us instead of 25 without the merge; they wait and compute all at the same time.)
//
//   scores   left operand: 16 keys, right: the heads.  A lane's 16 bytes of a key's row are its part of four steps; which dims meet in
//            a step is free, so the queries are laid out the same way.  A code, as the low byte of a 16-bit float 1024 beside its upper
//            byte, is 1024 + 128 + code once its sign bit is flipped, and 1152 less the code, exactly.  The page's scale joins the 32-bit score.
//   weights  p = 2^(s - m + 15), m the warp's own maximum: 16-bit floats from 2^15 down to 2^-24 hold weights of 2^-29 and more with all
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

constexpr int PAGE = 64, KEYS = 32;                     // of a page; of a warp

struct DecodeArgs {
    void* out;
    float* partial;                                      // [rows][heads][splits][places]
    float2* ml;                                          // [rows][heads][splits]: maximum (base two), sum
    const void* q;
    const int8_t *k_cache, *v_cache;
    const float *k_scale, *v_scale, *sink;
    const int32_t *tok_slot, *tok_pos, *page_table;
    size_t ldo, ldq;
    int max_pages, n_slots, n_pages, n_heads, n_kv_heads, dk, dv, window, chunk, keep_first, splits, reach, out_f32;
    float scale, softcap, cap_k2;
    int q_aligned;
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

// Four neighbouring places of a head's sums: dims d, d + 1 and d + 16, d + 17.
__device__ __forceinline__ int dim_of(int place) { return (place & ~127) + 8 * (place & 15) - 7 * (place & 1) + 2 * (place >> 4 & 7); }
__device__ __forceinline__ void store_places(void* out, int type, size_t at, float4 o, float factor, bool both) {
    store_from_f32(out, type, at, o.x * factor);
    store_from_f32(out, type, at + 1, o.y * factor);
    if (both) {
        store_from_f32(out, type, at + 16, o.z * factor);
        store_from_f32(out, type, at + 17, o.w * factor);
    }
}

// KC: blocks of 64 dims that keys span at most; VB: blocks of 128 dims of the values; a block has WARPS warps.  FULL: keys and values fill the
// blocks (addresses are then constants apart).
template <typename T, int KC, int VB, int WARPS, bool FULL>
__global__ void __launch_bounds__(WARPS * 32)
kv8_decode_kernel(const DecodeArgs p) {
    constexpr bool WIDE = sizeof(T) == 4;                // two columns to a head
    constexpr int HEADS = WIDE ? 4 : 8, SPLIT = WARPS * KEYS, TILES = KEYS / 16;
    const int dk = FULL ? KC * 64 : p.dk, dv = FULL ? VB * 128 : p.dv;
    extern __shared__ __align__(128) uint8_t smem[];     // per warp: its keys, its values; in the end [WARPS][HEADS][dv] sums
    __shared__ uint64_t bar[WARPS];
    __shared__ float s_m[WARPS][HEADS], s_l[WARPS][HEADS], s_unit[8];
    __shared__ uint32_t s_q[KC * 8][32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    grid_dep_launch();
    if (lane == 0) {
        sm100::mbar_init(&bar[warp], 1);
        sm100::mbar_fence_init();
        sm100::fence_proxy_async_smem();
    }
    __syncwarp();
    grid_dep_wait();
    const int per = p.n_heads / p.n_kv_heads, head_tiles = (per + HEADS - 1) / HEADS;
    const int split = blockIdx.x, kvh = blockIdx.y / head_tiles, row = blockIdx.z;
    const int head0 = kvh * per + blockIdx.y % head_tiles * HEADS, heads = min(HEADS, per - blockIdx.y % head_tiles * HEADS);
    const int slot = p.tok_slot[row], pos = p.tok_pos[row];
    // The queries, laid out for all warps: warp w makes column w, which is head w (WIDE: head w & 3, its first or second term); lane l
    // its dims 8 l .. 8 l + 7.  A lane of the products has dims 64 c + 16 t .. + 15 of column g.  Their way from memory runs beside that of the step's metadata.
    float x[8 / WARPS][8];
#pragma unroll
    for (int c = 0; c < 8 / WARPS; ++c) {
        const int column = warp + c * WARPS;
        const T* src = reinterpret_cast<const T*>(p.q) + (size_t)row * p.ldq + (size_t)(head0 + min(WIDE ? column & 3 : column, heads - 1)) * dk + 8 * lane;
        if (8 * lane < dk && p.q_aligned) load8_as_f32(src, WIDE ? QS_F32 : QS_BF16, 0, x[c]);
        else {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[c][i] = 8 * lane + i < dk ? to_f32(src[i]) : 0.f;
        }
    }
    if (slot < 0 || slot >= p.n_slots || pos < 0 || (pos >> 6) >= p.max_pages || pos >= p.reach) {
        if (slot >= 0 && threadIdx.x == 0 && split == 0 && blockIdx.y == 0) atomicExch(p.status, 1);
        if (p.splits == 1)                               // no merge: the row's zeros are written here
            for (int i = threadIdx.x; i < heads * dv; i += WARPS * 32) store_from_f32(p.out, p.out_f32 ? QS_F32 : QS_BF16, (size_t)row * p.ldo + (size_t)head0 * dv + i, 0.f);
        return;
    }
    const int first = first_key(p, pos), keep = p.window > 0 ? min(p.keep_first, first) : 0;
    const int base = split * SPLIT;
    if (base > pos || (base + SPLIT <= first && base >= keep)) return;       // no key of this split is seen
    const int key0 = base + warp * KEYS;
    const bool seen = key0 <= pos && (key0 + KEYS > first || key0 < keep);
    int page = -1;
    if (seen) {
        page = p.page_table[(size_t)slot * p.max_pages + (key0 >> 6)];
        if (page < 0 || page >= p.n_pages) { if (lane == 0) atomicExch(p.status, 3); page = -1; }
    }
    // Rows are read in whole blocks of dims: up to 127 bytes beyond the last.  Values lie 16 bytes more than a row apart: the rows of a lane's
    // keys then meet other banks than its neighbours' (64 bytes of two banks' rows otherwise, a quarter of the rate).
    const int pitch = dv + 16, warp_bytes = KEYS * (dk + pitch) + 128;
    uint8_t* keys = smem + warp * warp_bytes;
    uint8_t* values = keys + KEYS * dk;
    const size_t at = (size_t)max(page, 0) * p.n_kv_heads + kvh;
    if (page >= 0) {
        const int n = min(KEYS, pos - key0 + 1);         // rows behind the sequence's end stay out of it
        const size_t in_page = at * PAGE + (key0 & (PAGE - 1));
        if (lane == 0) {
            sm100::mbar_expect_tx(&bar[warp], n * dk);
            bulk_load(keys, p.k_cache + in_page * dk, n * dk, &bar[warp]);
        }
        const int pieces = dv >> 4;                      // 16 bytes of a row to a lane
        for (int i = lane; i < n * pieces; i += 32) {
            const int r = i / pieces, c = i - r * pieces;
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(sm100::smem_u32(values + r * pitch + 16 * c)), "l"(p.v_cache + (in_page + r) * dv + 16 * c) : "memory");
        }
    }
    float ks = 0.f, vs = 0.f;                            // no page: sums of 0, times 0
    if (page >= 0) {                                     // here, not where they are used: their way from memory is long
        asm volatile("ld.global.f32 %0, [%1];" : "=f"(ks) : "l"(p.k_scale + at));
        asm volatile("ld.global.f32 %0, [%1];" : "=f"(vs) : "l"(p.v_scale + at));
    }

#pragma unroll
    for (int c = 0; c < 8 / WARPS; ++c) {
        const int column = warp + c * WARPS;
        float most = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) most = fmaxf(most, fabsf(x[c][i]));
        most = warp_max(most);
        // the power of two at or below the largest; numbers that are not finite go through as they are
        const uint32_t e = min(max(__float_as_uint(most) >> 23, 1u), 253u);
        const float inv = __uint_as_float((254u - e) << 23);
        if (lane == 0) s_unit[column] = __uint_as_float(e << 23);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t v = pack_f16(x[c][2 * i] * inv, x[c][2 * i + 1] * inv);
            if (WIDE && column >= 4) {
                const float2 hi = unpack_f16(v);
                v = pack_f16(x[c][2 * i] * inv - hi.x, x[c][2 * i + 1] * inv - hi.y);
            }
            if (lane < KC * 8) s_q[(lane >> 3) * 8 + (lane & 1) * 4 + i][column * 4 + (lane >> 1 & 3)] = v;
        }
    }
    __syncthreads();
    // of the columns that this lane's results belong to: 2 t, 2 t + 1 (WIDE: of their heads, in both halves)
    const int h0 = WIDE ? 2 * (t & 1) : 2 * t;
    const float unit[2] = {s_unit[h0] * ks * p.scale, s_unit[h0 + 1] * ks * p.scale};

    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    float acc[VB * 8][4];
#pragma unroll
    for (int j = 0; j < VB * 8; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
    const bool ok = page >= 0 && sm100::mbar_wait(&bar[warp], 0);
    if (page >= 0 && !ok && lane == 0) atomicExch(p.status, 123);
    if (ok) {
        // scores of the keys: tile i, row g (and g + 8) is key 16 i + g (+ 8)
        float s[TILES][4];
        const float log2e = 1.4426950408889634f;
#pragma unroll
        for (int i = 0; i < TILES; ++i) s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.f;
#pragma unroll
        for (int c = 0; c < KC; ++c) {
            if (64 * c >= dk) break;
            uint32_t qf[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) qf[i] = s_q[c * 8 + i][lane];
#pragma unroll
            for (int i = 0; i < TILES; ++i) {
                const uint4 lo = *reinterpret_cast<const uint4*>(keys + (16 * i + g) * dk + 64 * c + 16 * t);
                const uint4 hi = *reinterpret_cast<const uint4*>(keys + (16 * i + g + 8) * dk + 64 * c + 16 * t);
                const uint32_t a[4] = {lo.x ^ 0x80808080u, lo.y ^ 0x80808080u, lo.z ^ 0x80808080u, lo.w ^ 0x80808080u};
                const uint32_t b[4] = {hi.x ^ 0x80808080u, hi.y ^ 0x80808080u, hi.z ^ 0x80808080u, hi.w ^ 0x80808080u};
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    mma_sum<WIDE>(s[i], two_codes(a[k], 0x4140), two_codes(b[k], 0x4140), two_codes(a[k], 0x4342), two_codes(b[k], 0x4342), qf[2 * k], qf[2 * k + 1]);
            }
        }
        const bool whole = key0 + KEYS - 1 <= pos && (key0 >= first || key0 + KEYS <= keep);
        const float factor[2] = {p.softcap > 0.f ? unit[0] : unit[0] * log2e, p.softcap > 0.f ? unit[1] : unit[1] * log2e};
#pragma unroll
        for (int i = 0; i < TILES; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (WIDE) s[i][e] += __shfl_xor_sync(0xffffffffu, s[i][e], 2);
                s[i][e] *= factor[e & 1];
            }
        if (p.softcap > 0.f) {
            const float cap = p.softcap * log2e;
#pragma unroll
            for (int i = 0; i < TILES; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e)              // tanh u = 1 - 2 / (e^2u + 1), within 10^-6 of the cap
                    s[i][e] = WIDE ? cap * tanhf(s[i][e] / p.softcap) : cap - __fdividef(2.f * cap, fast_exp2(s[i][e] * p.cap_k2) + 1.f);
        }
        if (!whole) {
#pragma unroll
            for (int i = 0; i < TILES; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int key = key0 + 16 * i + g + 8 * (e >> 1);
                    if (key > pos || (key < first && key >= keep)) s[i][e] = -INFINITY;
                }
        }
#pragma unroll
        for (int i = 0; i < TILES; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) m[e & 1] = fmaxf(m[e & 1], s[i][e]);
        // the weights, in pairs of heads; the columns' maxima and sums over the eight lanes of a column
        uint32_t w[TILES][2];                            // tile i, rows g and g + 8: two heads
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) m[j] = fmaxf(m[j], __shfl_xor_sync(0xffffffffu, m[j], o));
        const float zero[2] = {m[0] == -INFINITY ? 0.f : m[0] - 15.f, m[1] == -INFINITY ? 0.f : m[1] - 15.f};     // all -inf (or NaN): 2^-inf is 0
#pragma unroll
        for (int i = 0; i < TILES; ++i)
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
        asm volatile("cp.async.wait_all;" ::: "memory");
        __syncwarp();
#pragma unroll
        for (int i = 0; i < TILES; ++i)              // 16 keys: this lane's are 2 t, 2 t + 1 and the same + 8
#pragma unroll
            for (int b = 0; b < VB; ++b) {
                if (128 * b >= dv) break;
                const uint8_t* v = values + (16 * i + 2 * t) * pitch + 128 * b + 16 * g;
                uint4 x[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    x[e] = *reinterpret_cast<const uint4*>(v + ((e & 1) + 8 * (e >> 1)) * pitch);
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
    }
    asm volatile("cp.async.wait_all;" ::: "memory");     // (a wait for the keys that ran out: the values' copies end before their place is used again)
    // The warps' results: sums as [head][dim], beside each other where the pages were.
    if (g == 0 && (!WIDE || t < 2)) { s_m[warp][h0] = m[0]; s_m[warp][h0 + 1] = m[1]; }
    __syncthreads();                                     // everybody has read its keys and values
    // [warp][head][tile j][row g, row g + 8]: place 16 j + 2 g + e is dim 16 g + 2 j + e (of each 128); four floats more to a head, and the lanes' pairs meet all banks
    constexpr int PLACES = VB * 128, PITCH = PLACES + 4;
    float* sums = reinterpret_cast<float*>(smem);
    // what a warp's sums count beside the others'; a warp without a key that is seen: nothing; one whose scores are all NaN: NaN
    float f[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        float M = s_m[0][h0 + j];
#pragma unroll
        for (int w = 1; w < WARPS; ++w) M = fmaxf(M, s_m[w][h0 + j]);
        f[j] = m[j] == -INFINITY ? 1.f : fast_exp2(m[j] - M);
        if (g == 0 && (!WIDE || t < 2)) {
            s_l[warp][h0 + j] = l[j] * f[j];
            if (warp == 0) s_unit[h0 + j] = M;
        }
    }
    // The sums as 2^-15 of what the weights made them (the merge multiplies by as much): with the 2^15, values from 2^90 or so on would have no sum in
    // 32 bits.  Of very small values the sums are brought down by themselves: f times as little would lose bits.
    const float unit_v = vs * 0x1p-15f;
    if (vs < 0x1p-60f) {
#pragma unroll
        for (int j = 0; j < VB * 8; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[j][e] *= unit_v;
    } else {
        f[0] *= unit_v;
        f[1] *= unit_v;
    }
#pragma unroll
    for (int j = 0; j < VB * 8; ++j) {
        const int d = (j >> 3) * 128 + 16 * g + 2 * (j & 7);
        if (WIDE) {
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[j][e] += __shfl_xor_sync(0xffffffffu, acc[j][e], 2);
        }
        if (d < dv && (!WIDE || t < 2)) {
            float* to = sums + (warp * HEADS + h0) * PITCH + 16 * j + 2 * g;
            if (h0 < heads) *reinterpret_cast<float2*>(to) = make_float2(acc[j][0] * f[0], acc[j][2] * f[0]);
            if (h0 + 1 < heads) *reinterpret_cast<float2*>(to + PITCH) = make_float2(acc[j][1] * f[1], acc[j][3] * f[1]);
        }
    }
    __syncthreads();
    for (int i = 4 * threadIdx.x; i < heads * PLACES; i += 4 * WARPS * 32) {
        const int h = i / PLACES, place = i % PLACES, d = dim_of(place);
        if (d >= dv) continue;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        float L = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            const float4 v = *reinterpret_cast<const float4*>(sums + (w * HEADS + h) * PITCH + place);
            o.x += v.x; o.y += v.y; o.z += v.z; o.w += v.w;
            L += s_l[w][h];
        }
        if (p.splits > 1) {
            const size_t cell = ((size_t)row * p.n_heads + head0 + h) * p.splits + split;
            *reinterpret_cast<float4*>(p.partial + cell * PLACES + place) = o;
            if (place == 0) p.ml[cell] = make_float2(s_unit[h], L);
        } else {                                         // as the merge of one split: the same roundings, one by one
            const float M = s_unit[h];
            if (p.sink) {
                const float sink = p.sink[head0 + h] * 1.4426950408889634f, all = fmaxf(M, sink), w = M == -INFINITY ? 1.f : exp2f(M - all);
                L = __fadd_rn(__fmul_rn(L, w), exp2f(sink - all + 15.f));
                o.x = __fmul_rn(o.x, w); o.y = __fmul_rn(o.y, w); o.z = __fmul_rn(o.z, w); o.w = __fmul_rn(o.w, w);
            }
            const float inv = L != 0.f ? 0x1p15f / L : 0.f;
            const size_t to = (size_t)row * p.ldo + (size_t)(head0 + h) * dv + d;
            const int type = p.out_f32 ? QS_F32 : QS_BF16;
            store_places(p.out, type, to, o, inv, d + 16 < dv);
        }
    }
}

// One block per row and head: the splits' results.  The threads of a group have four dims each; the groups share the splits, each in
// ascending order, and are added in theirs; how the splits are shared depends on their number for the row and on dv.
constexpr int MERGE_THREADS = 256;
template <int SPLIT, int PLACES>
__global__ void __launch_bounds__(MERGE_THREADS)
kv8_merge_kernel(const DecodeArgs p) {
    extern __shared__ float s_w[];                       // [splits] weights
    __shared__ float scratch[34];
    __shared__ __align__(16) float4 s_o[MERGE_THREADS];
    grid_dep_launch();
    grid_dep_wait();
    const int head = blockIdx.x, row = blockIdx.y, dv = p.dv, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int slot = p.tok_slot[row], pos = p.tok_pos[row], type = p.out_f32 ? QS_F32 : QS_BF16;
    const size_t to = (size_t)row * p.ldo + (size_t)head * dv, cell = ((size_t)row * p.n_heads + head) * p.splits;
    // On the way beside the row's metadata, whether its splits turn out to be seen or not.
    float2 ml = make_float2(0.f, 0.f);
    if ((int)threadIdx.x < p.splits) asm volatile("ld.global.v2.f32 {%0, %1}, [%2];" : "=f"(ml.x), "=f"(ml.y) : "l"(p.ml + cell + threadIdx.x));
    const float sink = p.sink ? p.sink[head] * 1.4426950408889634f : -INFINITY;
    if (slot < 0 || slot >= p.n_slots || pos < 0 || (pos >> 6) >= p.max_pages || pos >= p.reach) {       // padding, or reported: a defined row
        for (int d = threadIdx.x; d < dv; d += MERGE_THREADS) store_from_f32(p.out, type, to + d, 0.f);
        return;
    }
    const int first = first_key(p, pos), keep = p.window > 0 ? min(p.keep_first, first) : 0;
    // the splits with keys that are seen: those of the kept first keys, then those of the window
    const int kept = keep > 0 ? (keep - 1) / SPLIT + 1 : 0, lo = max(first / SPLIT, kept), n = kept + pos / SPLIT - lo + 1;
    auto split = [&](int i) { return i < kept ? i : lo + i - kept; };
    auto seen = [&](int u) { return u < kept || (u >= lo && u < lo + n - kept); };
    const bool mine = seen(threadIdx.x);
    float M = mine ? fmaxf(sink, ml.x) : sink, L = 0.f;
    for (int u = threadIdx.x + MERGE_THREADS; u < lo + n - kept; u += MERGE_THREADS)
        if (seen(u)) M = fmaxf(M, p.ml[cell + u].x);
    M = warp_max(M);
    if (lane == 0) scratch[warp] = M;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < MERGE_THREADS / 32; ++i) M = fmaxf(M, scratch[i]);
    __syncthreads();
    auto weigh = [&](int u, float2 ml) {
        s_w[u] = ml.x == -INFINITY ? 1.f : exp2f(ml.x - M);
        L = fmaf(ml.y, s_w[u], L);
    };
    if (mine) weigh(threadIdx.x, ml);
    for (int u = threadIdx.x + MERGE_THREADS; u < lo + n - kept; u += MERGE_THREADS)
        if (seen(u)) weigh(u, p.ml[cell + u]);
    L = block_sum(L, scratch);                           // (a barrier: the weights are there)
    if (p.sink) L += exp2f(sink - M + 15.f);
    const float inv = L != 0.f ? 0x1p15f / L : 0.f;
    constexpr int width = PLACES / 4, groups = MERGE_THREADS / width;
    const int group = threadIdx.x / width, place = threadIdx.x % width * 4, d = dim_of(place);
    const int share = (n + groups - 1) / groups, from = group * share, end = d < dv ? min(n, from + share) : from;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    constexpr int AHEAD = 8;
    for (int i0 = from; i0 < end; i0 += AHEAD) {
        float4 v[AHEAD];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u)
            if (i0 + u < end) v[u] = *reinterpret_cast<const float4*>(p.partial + (cell + split(i0 + u)) * PLACES + place);
#pragma unroll
        for (int u = 0; u < AHEAD; ++u)
            if (i0 + u < end) {
                const float w = s_w[split(i0 + u)];
                o.x = fmaf(v[u].x, w, o.x); o.y = fmaf(v[u].y, w, o.y); o.z = fmaf(v[u].z, w, o.z); o.w = fmaf(v[u].w, w, o.w);
            }
    }
    s_o[threadIdx.x] = o;
    __syncthreads();
    if (group == 0 && d < dv) {
        for (int i = 1; i < groups && i * share < n; ++i) {
            const float4 v = s_o[i * width + threadIdx.x];
            o.x += v.x; o.y += v.y; o.z += v.z; o.w += v.w;
        }
        store_places(p.out, type, to + d, o, inv, d + 16 < dv);
    }
}

// Keys of a block.  Wide ones have four warps: their keys and values fill as much shared memory as the others', three blocks to an SM.  (8 rows of 1,024,
// heads of 256: 27 us; eight warps of 16 keys, so that 114 registers let two blocks onto an SM, and each query column has a warp: 31.  Heads of 128, 31 rows of 2,048
// and one of 65,536: four warps of 64 keys 29.3 and 29.4 us, eight of 32 keys 29.6 and 28.0.)
int split_keys(int dk, int dv) { return KEYS * (dk > 128 || dv > 128 ? 4 : 8); }

// Places of a head's sums.
int places(int dk, int dv) { return dk > 128 || dv > 128 ? 256 : 128; }

template <typename T, int KC, int VB, int WARPS, bool FULL>
int go(const DecodeArgs& p, int rows, cudaStream_t stream) {
    constexpr int HEADS = sizeof(T) == 4 ? 4 : 8;
    const int pages = WARPS * (KEYS * (p.dk + p.dv + 16) + 128), sums = WARPS * HEADS * (VB * 128 + 4) * 4, smem = pages > sums ? pages : sums;
    static PerDevice limit;
    int device = 0;
    cudaGetDevice(&device);
    limit.get(device, [] { return cudaFuncSetAttribute(kv8_decode_kernel<T, KC, VB, WARPS, FULL>, cudaFuncAttributeMaxDynamicSharedMemorySize, 100 * 1024) == cudaSuccess ? 1 : 0; });
    const int per = p.n_heads / p.n_kv_heads;
    cudaError_t e = qs_launch_dependent(kv8_decode_kernel<T, KC, VB, WARPS, FULL>, dim3(p.splits, p.n_kv_heads * ((per + HEADS - 1) / HEADS), rows), dim3(WARPS * 32), (size_t)smem, stream, p);
    if (e == cudaSuccess && p.splits > 1)
        e = qs_launch_dependent(kv8_merge_kernel<WARPS * KEYS, VB * 128>, dim3(p.n_heads, rows), dim3(MERGE_THREADS), (size_t)p.splits * sizeof(float), stream, p);
    if (e != cudaSuccess) return qs_fail(QS_ERR_INTERNAL, "kv8 decode: %s", cudaGetErrorString(e));
    return qs_check_launch("kv8 decode");
}

}  // namespace

// Splits of the keys that a call is made for, and floats of workspace that it takes (0: one split, no merge).
QS_API int qs_kv8_decode_splits(int dk, int dv, int max_context) { return (max_context + split_keys(dk, dv) - 1) / split_keys(dk, dv); }
QS_API long long qs_kv8_decode_scratch(int T_tokens, int n_heads, int dk, int dv, int max_context) {
    const int splits = qs_kv8_decode_splits(dk, dv, max_context);
    return splits > 1 ? (long long)T_tokens * n_heads * splits * (places(dk, dv) + 2) : 0;
}

// out [T, n_heads * dv] (bfloat16, or float32 with out_f32), q [T, n_heads * dk] of type `dtype`; head sizes multiples of 16 up to 256.  `partial`: float32,
// qs_kv8_decode_scratch elements, 16-byte aligned; contents need no initialisation; may be null for one split.
// Masks, status codes and rows as for qs_kv8_attention; positions lie below max_context.
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
    QS_REQUIRE(((uintptr_t)partial % 16) == 0, "kv8 decode: the workspace must be 16-byte aligned");
    const int e = dtype == QS_F32 ? 4 : 2;
    const int q_aligned = ((uintptr_t)q % 16) == 0 && ldq * e % 16 == 0;
    const DecodeArgs p = {out, partial, (float2*)(partial + (size_t)T_tokens * n_heads * splits * places(dk, dv)), q, k_cache, v_cache, k_scale, v_scale, sink, tok_slot, tok_pos, page_table, (size_t)ldo, (size_t)ldq,
                          max_pages, n_slots, n_pages, n_heads, n_kv_heads, dk, dv, window, chunk, keep_first, splits, max_context, out_f32, scale, softcap,
                          softcap > 0.f ? 2.f * 1.4426950408889634f / softcap : 0.f, q_aligned, status};
#define GO(T) do { if (dk <= 64 && dv <= 128) return go<T, 1, 1, 8, false>(p, T_tokens, stream); \
                   if (dk == 128 && dv == 128) return go<T, 2, 1, 8, true>(p, T_tokens, stream); \
                   if (dk <= 128 && dv <= 128) return go<T, 2, 1, 8, false>(p, T_tokens, stream); \
                   if (dk == 256 && dv == 256) return go<T, 4, 2, 4, true>(p, T_tokens, stream); \
                   return go<T, 4, 2, 4, false>(p, T_tokens, stream); } while (0)
    if (dtype == QS_F32) GO(float);
    GO(__nv_bfloat16);
#undef GO
}
