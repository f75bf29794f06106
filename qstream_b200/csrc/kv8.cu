// A paged cache whose keys and values are held in 8 bits, with one scale for each page of 64 tokens and key head: the write of new
// tokens (fused with the rotation), pages read back as values, and attention for sizes that the tensor-core kernels do not take.
//
// Layout: codes int8 [n_pages][n_kv_heads][64][head_dim], scales float32 [n_pages][n_kv_heads]; a number is code * scale.
//
// Every scale is a power of two (or 0: a page of zeros; or NaN: a page that was given a number that is not finite), and codes lie in
// -127 .. 127.  Why powers of two: tokens arrive one by one, and a page's scale grows when a new token does not fit.  The tokens before it
// are then rounded again, by at most half of the new step; each growth at least doubles the step, so all roundings of a number together
// stay below one step of the last scale.  Scaling and decoding are exact, code * scale is a bfloat16 number exactly (7 bits), and a page holds
// the same numbers whoever computes them.  The price is half a bit: the largest number of a page uses 64 to 127 of the 127 codes.
#include "common.cuh"

namespace {

constexpr int PAGE = 64;

// The bits of the smallest power of two (2^-126 at least) of which 127 reach |x|; `bits`: |x|, finite, not 0.  127 is 1.984375 * 2^6.
__device__ __forceinline__ float scale_for(uint32_t bits) {
    int e = (int)(bits >> 23) - 6 + ((bits & 0x7fffffu) > 0x7e0000u ? 1 : 0);
    return __uint_as_float((uint32_t)max(e, 1) << 23);
}

// Element d of a row after the rotation of its first R dims, each step rounded by itself (a multiply-add would round once where a plain
// program rounds twice, and a number next to the border of two codes would get the other one).
template <typename T>
__device__ __forceinline__ float rotated(const T* __restrict__ row, int d, const float* __restrict__ cs, int R, int half_layout) {
    if (d >= R) return to_f32(row[d]);
    const int rp = R >> 1, j = half_layout ? (d < rp ? d : d - rp) : d >> 1;
    const bool second = half_layout ? d >= rp : d & 1;
    const float a = to_f32(row[half_layout ? j : 2 * j]), b = to_f32(row[half_layout ? j + rp : 2 * j + 1]);
    const float c = cs[2 * j], s = cs[2 * j + 1];
    return second ? __fadd_rn(__fmul_rn(a, s), __fmul_rn(b, c)) : __fsub_rn(__fmul_rn(a, c), __fmul_rn(b, s));
}

// The largest of all threads' values; `scratch` holds 33 words.
__device__ __forceinline__ uint32_t block_max(uint32_t v, uint32_t* scratch) {
    v = __reduce_max_sync(0xffffffffu, v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
    __syncthreads();
    uint32_t most = 0;
    for (int i = 0; i < (int)(blockDim.x >> 5); ++i) most = max(most, scratch[i]);
    return most;
}

struct StoreArgs {
    const int32_t *tok_slot, *tok_pos, *page_table;
    int T, max_pages, n_slots, n_pages, n_heads, n_kv_heads, dk, dv, R, max_pos, half_layout, rows, q_blocks;
    const float* cos_sin;
    size_t ldq, ldqo, ldk, ldv, ldvf;
    int8_t *k_cache, *v_cache;
    float *k_scale, *v_scale;
    int32_t* status;
    float lam;
};

// n rows of one page and head, from row `a` of the page on: the scale that holds them and what is there already, then the codes.
// value(i, d): element d of new row i.
template <typename F>
__device__ __forceinline__ void store_run(int8_t* __restrict__ codes, float* __restrict__ scale, int a, int n, int dim, uint32_t* scratch, F value) {
    uint32_t most = 0;                                   // as bits: numbers that are not finite are above all others
    for (int e = threadIdx.x; e < n * dim; e += blockDim.x) most = max(most, __float_as_uint(value(e / dim, e % dim)) & 0x7fffffffu);
    most = block_max(most, scratch);
    const float before = a > 0 ? *scale : 0.f;
    const float need = most >= 0x7f800000u ? __uint_as_float(0x7fffffffu) : most == 0 ? 0.f : scale_for(most);
    const float after = isnan(before) || isnan(need) ? __uint_as_float(0x7fffffffu) : fmaxf(before, need);
    __syncthreads();                                     // everybody has read the old scale
    if (threadIdx.x == 0) *scale = after;
    if (a > 0 && after != before && !isnan(after)) {
        const float shrink = before / after;
        for (int e = threadIdx.x; e < a * dim; e += blockDim.x) codes[e] = (int8_t)__float2int_rn((float)codes[e] * shrink);
    }
    const float inv = after > 0.f ? 1.0f / after : 0.f;  // NaN: the codes say nothing, and 0
    for (int e = threadIdx.x; e < n * dim; e += blockDim.x)
        codes[(size_t)a * dim + e] = (int8_t)(inv > 0.f ? max(-127, min(127, __float2int_rn(value(e / dim, e % dim) * inv))) : 0);
}

// blockIdx.x: `rows` consecutive rows of the step; blockIdx.y: a key head, then blocks that rotate the queries of these rows.
// A run is the rows of one sequence that fall into one page: consecutive rows of ascending positions.  The block of a run's first row takes
// the whole run, so that a page's scale has one writer; a second run for the same page in one call is reported (status 5) and not written.
template <typename T>
__global__ void __launch_bounds__(128)
kv8_store_kernel(T* __restrict__ q_out, const T* q, const T* __restrict__ k, const T* __restrict__ v, const T* __restrict__ v_first, const StoreArgs p) {
    __shared__ uint32_t scratch[33];
    const int row0 = blockIdx.x * p.rows, rows = min(p.rows, p.T - row0);
    const bool rotate = p.cos_sin != nullptr && p.R > 0;
    if ((int)blockIdx.y >= p.n_kv_heads) {
        const int half = p.dk >> 1, rp = rotate ? p.R >> 1 : 0, items = rows * p.n_heads * half;
        for (int e = (blockIdx.y - p.n_kv_heads) * blockDim.x + threadIdx.x; e < items; e += p.q_blocks * blockDim.x) {
            const int i = e / (p.n_heads * half), r = row0 + i, head = (e - i * p.n_heads * half) / half, j = e % half;
            const int slot = p.tok_slot[r], pos = p.tok_pos[r];
            const bool fits = slot >= 0 && pos >= 0 && pos < p.max_pos;
            if (rotate && slot >= 0 && !fits && head == 0 && j == 0) atomicExch(p.status, 1);
            const T* src = q + (size_t)r * p.ldq + (size_t)head * p.dk;
            T* dst = q_out + (size_t)r * p.ldqo + (size_t)head * p.dk;
            if (j < rp && fits) {
                const float c = p.cos_sin[(size_t)pos * p.R + 2 * j], s = p.cos_sin[(size_t)pos * p.R + 2 * j + 1];
                const int ia = p.half_layout ? j : 2 * j, ib = p.half_layout ? j + rp : 2 * j + 1;
                const float a = to_f32(src[ia]), b = to_f32(src[ib]);
                dst[ia] = from_f32<T>(a * c - b * s);
                dst[ib] = from_f32<T>(a * s + b * c);
            } else if (dst != src) {
                const int ia = p.half_layout && j < rp ? j : 2 * j, ib = p.half_layout && j < rp ? j + rp : 2 * j + 1;
                dst[ia] = src[ia];
                dst[ib] = src[ib];
            }
        }
        return;
    }
    const int kvh = blockIdx.y;
    for (int r = row0; r < row0 + rows; ++r) {
        const int slot = p.tok_slot[r], pos = p.tok_pos[r];
        if (slot < 0) continue;
        const bool bad = slot >= p.n_slots || pos < 0 || (pos >> 6) >= p.max_pages || (rotate && pos >= p.max_pos);
        if (bad) { if (threadIdx.x == 0 && kvh == 0) atomicExch(p.status, 1); continue; }
        if (r > 0 && p.tok_slot[r - 1] == slot && p.tok_pos[r - 1] == pos - 1 && (pos & (PAGE - 1)) != 0) continue;       // inside a run
        const int page = p.page_table[(size_t)slot * p.max_pages + (pos >> 6)];
        if (page < 0 || page >= p.n_pages) { if (threadIdx.x == 0) atomicExch(p.status, 2); continue; }
        int again = 0;
        for (int i = threadIdx.x; i < r; i += blockDim.x) again |= p.tok_slot[i] == slot && (p.tok_pos[i] >> 6) == (pos >> 6);
        const int a = pos & (PAGE - 1);
        int n = 1;
        while (a + n < PAGE && r + n < p.T && p.tok_slot[r + n] == slot && p.tok_pos[r + n] == pos + n && !(rotate && pos + n >= p.max_pos)) ++n;
        if (__syncthreads_or(again)) { if (threadIdx.x == 0) atomicExch(p.status, 5); continue; }
        const size_t at = (size_t)page * p.n_kv_heads + kvh;
        store_run(p.k_cache + at * PAGE * p.dk, p.k_scale + at, a, n, p.dk, scratch, [&](int i, int d) {
            return rotated(k + (size_t)(r + i) * p.ldk + (size_t)kvh * p.dk, d, p.cos_sin + (size_t)(pos + i) * p.R, rotate ? p.R : 0, p.half_layout);
        });
        store_run(p.v_cache + at * PAGE * p.dv, p.v_scale + at, a, n, p.dv, scratch, [&](int i, int d) {
            const float x = to_f32(v[(size_t)(r + i) * p.ldv + (size_t)kvh * p.dv + d]);
            return v_first ? __fadd_rn(__fmul_rn(1.0f - p.lam, x), __fmul_rn(p.lam, to_f32(v_first[(size_t)(r + i) * p.ldvf + (size_t)kvh * p.dv + d]))) : x;
        });
    }
}

// Pages as the numbers they stand for; a page that does not exist gives NaN.
template <typename T>
__global__ void kv8_read_pages_kernel(T* __restrict__ out, const int8_t* __restrict__ codes, const float* __restrict__ scales, const int32_t* __restrict__ pages,
                                      int n_pages, int n_kv_heads, int dim) {
    const int page = pages[blockIdx.y], kvh = blockIdx.x;
    const bool there = page >= 0 && page < n_pages;
    const size_t at = there ? (size_t)page * n_kv_heads + kvh : 0;
    const float scale = there ? scales[at] : __uint_as_float(0x7fffffffu);
    const int8_t* src = codes + at * PAGE * dim;
    T* dst = out + ((size_t)blockIdx.y * n_kv_heads + kvh) * PAGE * dim;
    for (int e = threadIdx.x; e < PAGE * dim; e += blockDim.x) dst[e] = from_f32<T>((float)src[e] * scale);
}

// One warp per row and query head, for every size: 32 keys at a time in position order, a key to a lane; the running maximum and
// sum of the softmax; then the 32 weighted values, lane l owning dims l, l + 32, ...  All in 32 bits.
struct AttendArgs {
    const int32_t *tok_slot, *tok_pos, *tiles, *page_table;
    int T, max_pages, n_slots, n_pages, n_heads, n_kv_heads, dk, dv, window, chunk, keep_first, reach;
    const int8_t *k_cache, *v_cache;
    const float *k_scale, *v_scale, *sink;
    float scale, softcap;
    size_t ldq, ldo;
    int32_t* status;
};

template <typename T, typename TO, int NACC>
__global__ void __launch_bounds__(128)
kv8_attention_kernel(TO* __restrict__ out, const T* __restrict__ q, const AttendArgs p) {
    extern __shared__ float q_smem[];                    // [warps][dk]
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int head = blockIdx.x * (blockDim.x >> 5) + warp;
    if (head >= p.n_heads) return;
    int row, slot, pos;
    if (p.tiles) {                                       // (first row, rows, position of the first row, slot) of up to 128 rows
        const int32_t* t = p.tiles + 4 * (blockIdx.y >> 7);
        const int i = blockIdx.y & 127;
        if (i >= t[1]) return;
        row = t[0] + i; pos = t[2] + i; slot = t[3];
        if (t[1] > 128 || t[0] < 0 || t[0] + t[1] > p.T || slot < 0 || slot >= p.n_slots || t[2] < 0 || (t[2] + t[1] - 1) >> 6 >= p.max_pages) {      // the whole tile: report, write nothing
            if (lane == 0) atomicExch(p.status, 1);
            return;
        }
    } else {
        row = blockIdx.y; slot = p.tok_slot[row]; pos = p.tok_pos[row];
    }
    TO* o = out + (size_t)row * p.ldo + (size_t)head * p.dv;
    const bool bad = slot >= p.n_slots || pos < 0 || (pos >> 6) >= p.max_pages || pos >= p.reach;
    if (slot < 0 || bad) {
        if (slot >= 0 && lane == 0) atomicExch(p.status, 1);
        for (int d = lane; d < p.dv; d += 32) o[d] = from_f32<TO>(0.f);
        return;
    }
    float* qs = q_smem + warp * p.dk;
    for (int d = lane; d < p.dk; d += 32) qs[d] = to_f32(q[(size_t)row * p.ldq + (size_t)head * p.dk + d]);
    __syncwarp();
    const int first = p.chunk > 0 ? pos - pos % p.chunk : p.window > 0 ? max(0, pos - p.window + 1) : 0;
    const int keep = p.window > 0 ? min(p.keep_first, first) : 0;
    const int kvh = head / (p.n_heads / p.n_kv_heads);
    float acc[NACC], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int i = 0; i < NACC; ++i) acc[i] = 0.f;
    for (int base = 0; base <= pos; base += 32) {
        if (base + 31 < first) {
            if (base >= keep) { base = (first >> 5 << 5) - 32; continue; }
        }
        const int page = p.page_table[(size_t)slot * p.max_pages + (base >> 6)];
        if (page < 0 || page >= p.n_pages) { if (lane == 0) atomicExch(p.status, 3); continue; }
        const size_t at = (size_t)page * p.n_kv_heads + kvh;
        const int key = base + lane;
        const bool seen = key <= pos && (key >= first || key < keep);
        float s = -INFINITY;
        if (seen) {
            const int8_t* kr = p.k_cache + (at * PAGE + (key & 63)) * p.dk;
            float dot = 0.f;
            for (int d = 0; d < p.dk; ++d) dot = fmaf(qs[d], (float)kr[d], dot);
            s = dot * p.k_scale[at] * p.scale;
            if (p.softcap > 0.f) s = p.softcap * tanhf(s / p.softcap);
        }
        const float m_new = fmaxf(m, warp_max(s));
        const float w = seen ? expf(s - m_new) : 0.f, alpha = m == -INFINITY ? 0.f : expf(m - m_new);
        l = l * alpha + warp_sum(w);
        m = m_new;
        const float vs = p.v_scale[at];
        const int8_t* vr = p.v_cache + (at * PAGE + (base & 63)) * p.dv;
#pragma unroll
        for (int i = 0; i < NACC; ++i) acc[i] *= alpha;
        const uint32_t some = __ballot_sync(0xffffffffu, seen);
        for (int j = 0; j < 32; ++j) {
            if (!(some >> j & 1)) continue;
            const float wj = __shfl_sync(0xffffffffu, w, j) * vs;
#pragma unroll
            for (int i = 0; i < NACC; ++i)
                if (lane + 32 * i < p.dv) acc[i] = fmaf(wj, (float)vr[(size_t)j * p.dv + lane + 32 * i], acc[i]);
        }
    }
    if (p.sink) {
        const float m_new = fmaxf(m, p.sink[head]), alpha = m == -INFINITY ? 0.f : expf(m - m_new);
        l = l * alpha + expf(p.sink[head] - m_new);
#pragma unroll
        for (int i = 0; i < NACC; ++i) acc[i] *= alpha;
    }
    const float inv = l != 0.f ? 1.0f / l : 0.f;
#pragma unroll
    for (int i = 0; i < NACC; ++i)
        if (lane + 32 * i < p.dv) o[lane + 32 * i] = from_f32<TO>(acc[i] * inv);
}

template <typename T>
int store_launch(void* q_out, const void* q, const void* k, const void* v, const void* v_first, const StoreArgs& p, cudaStream_t stream) {
    kv8_store_kernel<T><<<dim3((p.T + p.rows - 1) / p.rows, p.n_kv_heads + p.q_blocks), 128, 0, stream>>>(
        (T*)q_out, (const T*)q, (const T*)k, (const T*)v, (const T*)v_first, p);
    return qs_check_launch("kv8 store");
}

template <typename T, typename TO>
int attention_launch(void* out, const void* q, const AttendArgs& p, int n, cudaStream_t stream) {
    const dim3 grid((p.n_heads + 3) / 4, n);
    const size_t smem = (size_t)4 * p.dk * sizeof(float);
    if (p.dv <= 128) kv8_attention_kernel<T, TO, 4><<<grid, 128, smem, stream>>>((TO*)out, (const T*)q, p);
    else kv8_attention_kernel<T, TO, 16><<<grid, 128, smem, stream>>>((TO*)out, (const T*)q, p);
    return qs_check_launch("kv8 attention");
}

}  // namespace

// Rotation of q (q_out may be q), rotation of k, and the write of k and v into the 8-bit pages.  k, v, v_first [T, n_kv_heads * dim] and q, q_out
// [T, n_heads * dk] of type `dtype`; q may be null (keys and values only).  The rows of a sequence that fall into one page have to be
// consecutive, with ascending positions.
QS_API int qs_kv8_store(void* q_out, long long ldqo, const void* q, long long ldq, const void* k, long long ldk, const void* v, long long ldv,
                        const void* v_first, long long ldvf, float lam, int dtype, int T_tokens, int n_heads, int n_kv_heads, int dk, int dv, int R,
                        const float* cos_sin, int max_pos, int half_layout, const int32_t* tok_slot, const int32_t* tok_pos, const int32_t* page_table,
                        int n_slots, int max_pages, int n_pages, int8_t* k_cache, int8_t* v_cache, float* k_scale, float* v_scale, int32_t* status,
                        cudaStream_t stream) {
    if (T_tokens == 0) return QS_OK;
    QS_REQUIRE(T_tokens > 0 && n_heads >= 0 && n_kv_heads > 0 && n_slots > 0 && max_pages > 0 && n_pages > 0, "kv8 store: bad sizes");
    QS_REQUIRE(dk > 0 && dk % 2 == 0 && dk <= 512 && dv > 0 && dv <= 512, "kv8 store: head sizes %d and %d (keys: even; up to 512)", dk, dv);
    QS_REQUIRE(!cos_sin || (R >= 0 && R % 2 == 0 && R <= dk && max_pos > 0), "kv8 store: %d rotated dims of %d", R, dk);
    QS_REQUIRE(dtype == QS_F32 || dtype == QS_BF16, "kv8 store: type %d", dtype);
    QS_REQUIRE(n_kv_heads <= 32768, "kv8 store: %d key heads exceed the grid", n_kv_heads);
    StoreArgs p = {};
    p.tok_slot = tok_slot; p.tok_pos = tok_pos; p.page_table = page_table;
    p.T = T_tokens; p.max_pages = max_pages; p.n_slots = n_slots; p.n_pages = n_pages;
    p.n_heads = q ? n_heads : 0; p.n_kv_heads = n_kv_heads; p.dk = dk; p.dv = dv; p.R = cos_sin ? R : 0; p.max_pos = cos_sin ? max_pos : 0x7fffffff;
    p.half_layout = half_layout; p.cos_sin = cos_sin;
    p.ldq = (size_t)ldq; p.ldqo = (size_t)ldqo; p.ldk = (size_t)ldk; p.ldv = (size_t)ldv; p.ldvf = (size_t)ldvf;
    p.k_cache = k_cache; p.v_cache = v_cache; p.k_scale = k_scale; p.v_scale = v_scale; p.status = status; p.lam = lam;
    p.rows = T_tokens <= 256 ? 1 : 16;
    const bool queries = q && n_heads > 0 && (p.R > 0 || q != q_out);
    p.q_blocks = queries ? (int)(((long long)p.rows * n_heads * (dk / 2) + 1023) / 1024) : 0;
    return dtype == QS_F32 ? store_launch<float>(q_out, q, k, v, v_first, p, stream) : store_launch<__nv_bfloat16>(q_out, q, k, v, v_first, p, stream);
}

// out [n][n_kv_heads][64][dim] of type `dtype`: the numbers in the listed pages.
QS_API int qs_kv8_read_pages(void* out, int dtype, const int8_t* codes, const float* scales, const int32_t* pages, int n, int n_pages, int n_kv_heads,
                             int dim, cudaStream_t stream) {
    if (n == 0) return QS_OK;
    QS_REQUIRE(n > 0 && n <= 65535 && n_pages > 0 && n_kv_heads > 0 && dim > 0, "kv8 read_pages: %d pages of %d heads of %d", n, n_kv_heads, dim);
    QS_REQUIRE(dtype == QS_F32 || dtype == QS_BF16, "kv8 read_pages: type %d", dtype);
    const dim3 grid(n_kv_heads, n);
    if (dtype == QS_F32) kv8_read_pages_kernel<float><<<grid, 256, 0, stream>>>((float*)out, codes, scales, pages, n_pages, n_kv_heads, dim);
    else kv8_read_pages_kernel<__nv_bfloat16><<<grid, 256, 0, stream>>>((__nv_bfloat16*)out, codes, scales, pages, n_pages, n_kv_heads, dim);
    return qs_check_launch("kv8 read_pages");
}

// Attention over the 8-bit pages for any head sizes, a warp per row and head.  With `tiles` (int32 [n_tiles][4]: first row, rows up to 128,
// position of the first row, slot) the rows are those of the tiles; without, row t is position tok_pos[t] of sequence tok_slot[t] (< 0: zeros).
QS_API int qs_kv8_attention(void* out, int out_dtype, long long ldo, const void* q, int dtype, long long ldq, int T_tokens, const int32_t* tok_slot,
                            const int32_t* tok_pos, const int32_t* tiles, int n_tiles, const int32_t* page_table, int n_slots, int max_pages, int n_pages,
                            const int8_t* k_cache, const int8_t* v_cache, const float* k_scale, const float* v_scale, int n_heads, int n_kv_heads,
                            int dk, int dv, float scale, int window, int chunk, int keep_first, const float* sink, float softcap, int reach,
                            int32_t* status, cudaStream_t stream) {
    if (T_tokens == 0 || (tiles && n_tiles == 0)) return QS_OK;
    QS_REQUIRE(T_tokens > 0 && n_heads > 0 && n_kv_heads > 0 && n_heads % n_kv_heads == 0 && n_slots > 0 && max_pages > 0 && n_pages > 0, "kv8 attention: bad sizes");
    QS_REQUIRE(dk > 0 && dk <= 512 && dv > 0 && dv <= 512, "kv8 attention: head sizes %d and %d (up to 512)", dk, dv);
    QS_REQUIRE(chunk >= 0 && keep_first >= 0 && !(chunk > 0 && window > 0), "kv8 attention: a window of %d and chunks of %d", window, chunk);
    const long long n = tiles ? 128LL * n_tiles : T_tokens;
    QS_REQUIRE(n <= 65535, "kv8 attention: %lld rows exceed the grid", n);
    const AttendArgs p = {tok_slot, tok_pos, tiles, page_table, T_tokens, max_pages, n_slots, n_pages, n_heads, n_kv_heads, dk, dv, window, chunk, keep_first, reach,
                          k_cache, v_cache, k_scale, v_scale, sink, scale, softcap, (size_t)ldq, (size_t)ldo, status};
    if (dtype == QS_F32 && out_dtype == QS_F32) return attention_launch<float, float>(out, q, p, (int)n, stream);
    if (dtype == QS_BF16 && out_dtype == QS_BF16) return attention_launch<__nv_bfloat16, __nv_bfloat16>(out, q, p, (int)n, stream);
    if (dtype == QS_BF16 && out_dtype == QS_F32) return attention_launch<__nv_bfloat16, float>(out, q, p, (int)n, stream);
    return qs_fail(QS_ERR_INVALID_INPUT, "kv8 attention: queries of type %d and a result of type %d", dtype, out_dtype);
}
