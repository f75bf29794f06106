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

__device__ __forceinline__ void store16(float* dst, const float (&x)[16]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) reinterpret_cast<float4*>(dst)[i] = make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
}
__device__ __forceinline__ void store16(__nv_bfloat16* dst, const float (&x)[16]) {
    uint32_t w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const __nv_bfloat162 r = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&r);
    }
    reinterpret_cast<uint4*>(dst)[0] = make_uint4(w[0], w[1], w[2], w[3]);
    reinterpret_cast<uint4*>(dst)[1] = make_uint4(w[4], w[5], w[6], w[7]);
}

// 16 elements of a row from d on; those of a row's first R dims rotated (`cs`: the row's angles).
template <typename T>
__device__ __forceinline__ void load16(const T* __restrict__ row, float (&x)[16]) {
    float a[8], b[8];
    load8_as_f32(row, sizeof(T) == 4 ? QS_F32 : QS_BF16, 0, a);
    load8_as_f32(row, sizeof(T) == 4 ? QS_F32 : QS_BF16, 8, b);
#pragma unroll
    for (int i = 0; i < 8; ++i) { x[i] = a[i]; x[8 + i] = b[i]; }
}
template <typename T>
__device__ __forceinline__ void rotated16(const T* __restrict__ row, int d, const float* __restrict__ cs, int R, int half_layout, float (&x)[16]) {
    load16(row + d, x);
    if (d >= R) return;
    const int rp = R >> 1;
    if (half_layout) {
        const bool second = d >= rp;
        float y[16];
        load16(row + (second ? d - rp : d + rp), y);
        const float4* angle = reinterpret_cast<const float4*>(cs + 2 * (second ? d - rp : d));
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float4 c = angle[i];
            x[2 * i] = second ? __fadd_rn(__fmul_rn(y[2 * i], c.y), __fmul_rn(x[2 * i], c.x)) : __fsub_rn(__fmul_rn(x[2 * i], c.x), __fmul_rn(y[2 * i], c.y));
            x[2 * i + 1] = second ? __fadd_rn(__fmul_rn(y[2 * i + 1], c.w), __fmul_rn(x[2 * i + 1], c.z)) : __fsub_rn(__fmul_rn(x[2 * i + 1], c.z), __fmul_rn(y[2 * i + 1], c.w));
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float4 c = reinterpret_cast<const float4*>(cs + d)[i];
            const float a0 = x[4 * i], b0 = x[4 * i + 1], a1 = x[4 * i + 2], b1 = x[4 * i + 3];
            x[4 * i] = __fsub_rn(__fmul_rn(a0, c.x), __fmul_rn(b0, c.y));
            x[4 * i + 1] = __fadd_rn(__fmul_rn(a0, c.y), __fmul_rn(b0, c.x));
            x[4 * i + 2] = __fsub_rn(__fmul_rn(a1, c.z), __fmul_rn(b1, c.w));
            x[4 * i + 3] = __fadd_rn(__fmul_rn(a1, c.w), __fmul_rn(b1, c.z));
        }
    }
}

// Four numbers times a power of two, at most 127 then, as a word of codes: added to 1.5 * 2^23 they are rounded to whole numbers (ties to even), whose
// lowest byte the sum's is.
__device__ __forceinline__ uint32_t four_codes(float a, float b, float c, float d, float factor) {
    const float k = 12582912.f;
    const uint32_t lo = __byte_perm(__float_as_uint(fmaf(a, factor, k)), __float_as_uint(fmaf(b, factor, k)), 0x0040);
    const uint32_t hi = __byte_perm(__float_as_uint(fmaf(c, factor, k)), __float_as_uint(fmaf(d, factor, k)), 0x0040);
    return __byte_perm(lo, hi, 0x5410);
}

// max(a, |b|), NaN where one is.
__device__ __forceinline__ float max_size(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(fabsf(b)));
    return r;
}

// n rows of one page and head, from row `a` of the page on: the scale that holds them and what is there already, then the codes.
// VEC: value(i, d, x) gives elements d .. d + 15 of new row i, else element d.  The rows are read and rotated twice, the second time from the
// caches (64 bfloat16 rows of 256 numbers would fit a block's registers, 32 of each thread's; that form is not built).
// Bound by the instructions as much as by memory: some fourteen for an element, seven of them its way through 32 bits and into the maximum, one and three
// quarters its rounding and packing.
template <bool VEC, typename F>
__device__ __forceinline__ void store_run(int8_t* __restrict__ codes, float* __restrict__ scale, int a, int n, int dim, uint32_t* scratch, F value) {
    constexpr int E = VEC ? 16 : 1;
    const int pieces = dim / E, first = threadIdx.x / pieces, step = blockDim.x / pieces, at = threadIdx.x - first * pieces, more = blockDim.x - step * pieces;
    float most = 0.f;
    for (int i = first, c = at; i < n;) {
        float x[E];
        value(i, c * E, x);
#pragma unroll
        for (int u = 0; u < E; ++u) most = max_size(most, x[u]);
        i += step;
        if ((c += more) >= pieces) { c -= pieces; ++i; }
    }
    const uint32_t bits = block_max(__float_as_uint(most), scratch);        // numbers that are not finite are above all others
    const float before = a > 0 ? *scale : 0.f;
    const float need = bits >= 0x7f800000u ? __uint_as_float(0x7fffffffu) : bits == 0 ? 0.f : scale_for(bits);
    const float after = isnan(before) || isnan(need) ? __uint_as_float(0x7fffffffu) : fmaxf(before, need);
    __syncthreads();                                     // everybody has read the old scale
    if (threadIdx.x == 0) *scale = after;
    if (a > 0 && after != before && !isnan(after)) {
        const float shrink = before / after;
        if (VEC) {
            uint32_t* words = reinterpret_cast<uint32_t*>(codes);
            for (int e = threadIdx.x; e < a * dim / 4; e += blockDim.x) {
                const uint32_t w = words[e];
                words[e] = four_codes((float)(int8_t)w, (float)(int8_t)(w >> 8), (float)(int8_t)(w >> 16), (float)(int8_t)(w >> 24), shrink);
            }
        } else {
            for (int e = threadIdx.x; e < a * dim; e += blockDim.x) codes[e] = (int8_t)__float2int_rn((float)codes[e] * shrink);
        }
    }
    const float inv = after > 0.f ? 1.0f / after : 0.f;
    const bool nothing = !(inv > 0.f);                   // zeros; or NaN, and the codes say nothing: 0
    for (int i = first, c = at; i < n;) {
        float x[E];
        value(i, c * E, x);
        if (nothing) {
#pragma unroll
            for (int u = 0; u < E; ++u) x[u] = 0.f;
        }
        int8_t* to = codes + (size_t)(a + i) * dim + c * E;
        if constexpr (VEC)
            *reinterpret_cast<uint4*>(to) = make_uint4(four_codes(x[0], x[1], x[2], x[3], inv), four_codes(x[4], x[5], x[6], x[7], inv),
                                                       four_codes(x[8], x[9], x[10], x[11], inv), four_codes(x[12], x[13], x[14], x[15], inv));
        else *to = (int8_t)__float2int_rn(x[0] * inv);
        i += step;
        if ((c += more) >= pieces) { c -= pieces; ++i; }
    }
}

// blockIdx.x: `rows` (up to 32) consecutive rows of the step; blockIdx.y: a key head's keys, its values, ..., then blocks that rotate the queries of these rows.
// A run is the rows of one sequence that fall into one page: consecutive rows of ascending positions.  The block of a run's first row takes
// the whole run, so that a page's scale has one writer; a second run for the same page in one call is reported (status 5) and not written.
// VEC: rows, angles and pages in pieces of 16 elements, on their boundaries.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256)
kv8_store_kernel(T* q_out, const T* q, const T* __restrict__ k, const T* __restrict__ v, const T* __restrict__ v_first, const StoreArgs p) {
    constexpr int E = VEC ? 16 : 1;
    __shared__ uint32_t scratch[33];
    grid_dep_launch();
    grid_dep_wait();
    const int row0 = blockIdx.x * p.rows, rows = min(p.rows, p.T - row0), lane = threadIdx.x & 31;
    const bool rotate = p.cos_sin != nullptr && p.R > 0;
    if ((int)blockIdx.y >= 2 * p.n_kv_heads) {
        // an item: 16 (VEC) or 1 pairs that turn, or as many plain elements of both halves of the rest
        const int rp = rotate ? p.R >> 1 : 0, turning = VEC && !p.half_layout ? rp / 8 : rp / E, plain = q_out == q ? 0 : (p.dk - 2 * rp) / E;
        const int per_head = turning + plain, per_row = p.n_heads * per_head, items = rows * per_row;
        for (int e = (blockIdx.y - 2 * p.n_kv_heads) * blockDim.x + threadIdx.x; e < items; e += p.q_blocks * blockDim.x) {
            const int i = e / per_row, r = row0 + i, rest = e - i * per_row, head = rest / per_head, j = rest - head * per_head;
            const int slot = p.tok_slot[r], pos = p.tok_pos[r];
            const bool fits = slot >= 0 && pos >= 0 && pos < p.max_pos;
            if (rotate && slot >= 0 && !fits && head == 0 && j == 0) atomicExch(p.status, 1);
            const T* src = q + (size_t)r * p.ldq + (size_t)head * p.dk;
            T* dst = q_out + (size_t)r * p.ldqo + (size_t)head * p.dk;
            if (!fits && dst == src) continue;
            const float* cs = p.cos_sin + (size_t)pos * p.R;
            if constexpr (VEC) {
                auto copy = [&](int d) {
                    float x[16];
                    load16(src + d, x);
                    store16(dst + d, x);
                };
                if (j >= turning) copy(2 * rp + (j - turning) * 16);
                else if (p.half_layout) {
                    if (!fits) { copy(j * 16); copy(j * 16 + rp); continue; }
                    float x[16], y[16];
                    load16(src + j * 16, x);
                    load16(src + j * 16 + rp, y);
#pragma unroll
                    for (int u = 0; u < 16; ++u) {
                        const float c = cs[2 * (j * 16 + u)], s = cs[2 * (j * 16 + u) + 1], a = x[u], b = y[u];
                        x[u] = a * c - b * s;
                        y[u] = a * s + b * c;
                    }
                    store16(dst + j * 16, x);
                    store16(dst + j * 16 + rp, y);
                } else {
                    if (!fits) { copy(j * 16); continue; }
                    float x[16];
                    load16(src + j * 16, x);
#pragma unroll
                    for (int u = 0; u < 8; ++u) {
                        const float c = cs[j * 16 + 2 * u], s = cs[j * 16 + 2 * u + 1], a = x[2 * u], b = x[2 * u + 1];
                        x[2 * u] = a * c - b * s;
                        x[2 * u + 1] = a * s + b * c;
                    }
                    store16(dst + j * 16, x);
                }
            } else if (j < turning) {
                const int ia = p.half_layout ? j : 2 * j, ib = p.half_layout ? j + rp : 2 * j + 1;
                const float a = to_f32(src[ia]), b = to_f32(src[ib]);
                const float c = fits ? cs[2 * j] : 1.f, s = fits ? cs[2 * j + 1] : 0.f;
                dst[ia] = fits ? from_f32<T>(a * c - b * s) : src[ia];
                dst[ib] = fits ? from_f32<T>(a * s + b * c) : src[ib];
            } else {
                dst[2 * rp + j - turning] = src[2 * rp + j - turning];
            }
        }
        return;
    }
    const int kvh = blockIdx.y >> 1;
    const bool keys = (blockIdx.y & 1) == 0, reports = blockIdx.y == 0 && threadIdx.x < 32;
    // which of the rows begin a run
    bool begins = false;
    if (lane < rows) {
        const int r = row0 + lane, slot = p.tok_slot[r], pos = p.tok_pos[r];
        const bool bad = slot >= p.n_slots || pos < 0 || (pos >> 6) >= p.max_pages || (rotate && pos >= p.max_pos);
        if (slot >= 0 && bad && reports) atomicExch(p.status, 1);
        begins = slot >= 0 && !bad && !(r > 0 && (pos & (PAGE - 1)) != 0 && p.tok_slot[r - 1] == slot && p.tok_pos[r - 1] == pos - 1);
    }
    for (uint32_t todo = __ballot_sync(0xffffffffu, begins); todo != 0; todo &= todo - 1) {
        const int r = row0 + __ffs(todo) - 1, slot = p.tok_slot[r], pos = p.tok_pos[r];
        const int page = p.page_table[(size_t)slot * p.max_pages + (pos >> 6)];
        if (page < 0 || page >= p.n_pages) { if (threadIdx.x == 0) atomicExch(p.status, 2); continue; }
        int again = 0;
        int whole = 0;                                   // rows looked at in fours
        if ((((uintptr_t)p.tok_slot | (uintptr_t)p.tok_pos) & 15) == 0) {
            whole = r & ~3;
            for (int i = threadIdx.x; i < whole >> 2; i += blockDim.x) {
                const int4 s4 = reinterpret_cast<const int4*>(p.tok_slot)[i], p4 = reinterpret_cast<const int4*>(p.tok_pos)[i];
                again |= (s4.x == slot && p4.x >> 6 == pos >> 6) | (s4.y == slot && p4.y >> 6 == pos >> 6) | (s4.z == slot && p4.z >> 6 == pos >> 6) | (s4.w == slot && p4.w >> 6 == pos >> 6);
            }
        }
        for (int i = whole + threadIdx.x; i < r; i += blockDim.x) again |= p.tok_slot[i] == slot && (p.tok_pos[i] >> 6) == (pos >> 6);
        const int a = pos & (PAGE - 1);
        // the run's length: the first row behind it, 64 rows looked at by two lanes' turns
        int n = PAGE - a;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int i = u * 32 + lane;
            const bool ends = i > 0 && i < PAGE - a && !(r + i < p.T && p.tok_slot[r + i] == slot && p.tok_pos[r + i] == pos + i && !(rotate && pos + i >= p.max_pos));
            const uint32_t found = __ballot_sync(0xffffffffu, ends);
            if (found) n = min(n, u * 32 + __ffs(found) - 1);
        }
        if (__syncthreads_or(again)) { if (threadIdx.x == 0) atomicExch(p.status, 5); continue; }
        const size_t at = (size_t)page * p.n_kv_heads + kvh;
        if (keys) store_run<VEC>(p.k_cache + at * PAGE * p.dk, p.k_scale + at, a, n, p.dk, scratch, [&](int i, int d, float (&x)[E]) {
            const T* row = k + (size_t)(r + i) * p.ldk + (size_t)kvh * p.dk;
            const float* cs = p.cos_sin + (size_t)(pos + i) * p.R;
            if constexpr (VEC) rotated16(row, d, cs, rotate ? p.R : 0, p.half_layout, x);
            else x[0] = rotated(row, d, cs, rotate ? p.R : 0, p.half_layout);
        });
        else store_run<VEC>(p.v_cache + at * PAGE * p.dv, p.v_scale + at, a, n, p.dv, scratch, [&](int i, int d, float (&x)[E]) {
            const T* row = v + (size_t)(r + i) * p.ldv + (size_t)kvh * p.dv + d;
            if constexpr (VEC) load16(row, x);
            else x[0] = to_f32(*row);
            if (v_first) {
                const T* first = v_first + (size_t)(r + i) * p.ldvf + (size_t)kvh * p.dv + d;
#pragma unroll
                for (int u = 0; u < E; ++u) x[u] = __fadd_rn(__fmul_rn(1.0f - p.lam, x[u]), __fmul_rn(p.lam, to_f32(first[u])));
            }
        });
    }
}

// Pages as the numbers they stand for; a page that does not exist gives NaN.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256)
kv8_read_pages_kernel(T* __restrict__ out, const int8_t* __restrict__ codes, const float* __restrict__ scales, const int32_t* __restrict__ pages,
                      int n_pages, int n_kv_heads, int dim) {
    grid_dep_launch();
    grid_dep_wait();
    const int page = pages[blockIdx.y], kvh = blockIdx.x;
    const bool there = page >= 0 && page < n_pages;
    const size_t at = there ? (size_t)page * n_kv_heads + kvh : 0;
    const float scale = there ? scales[at] : __uint_as_float(0x7fffffffu);
    const int8_t* src = codes + at * PAGE * dim;
    T* dst = out + ((size_t)blockIdx.y * n_kv_heads + kvh) * PAGE * dim;
    if (VEC) {
        for (int e = threadIdx.x; e < PAGE * dim / 16; e += blockDim.x) {
            const uint4 raw = __ldg(reinterpret_cast<const uint4*>(src) + e);
            const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
            float x[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] = (float)(int8_t)(w[i >> 2] >> (8 * (i & 3))) * scale;
            store16(dst + e * 16, x);
        }
    } else {
        for (int e = threadIdx.x; e < PAGE * dim; e += blockDim.x) dst[e] = from_f32<T>((float)src[e] * scale);
    }
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
        slot = t[3];
        // the whole tile: report, write nothing (sums without a sign: a first row or position near 2^31 stays large)
        if (t[1] > 128 || t[0] < 0 || (uint32_t)t[0] + t[1] > (uint32_t)p.T || slot < 0 || slot >= p.n_slots || t[2] < 0 ||
            ((uint32_t)t[2] + t[1] - 1) >> 6 >= (uint32_t)p.max_pages) {
            if (lane == 0) atomicExch(p.status, 1);
            return;
        }
        row = t[0] + i; pos = t[2] + i;
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
    // The query over the power of two at or below its largest number: a sum of its products with codes has a place in 32 bits then, however large the query and
    // small the page's scale.  Numbers that are not finite go through as they are.
    float* qs = q_smem + warp * p.dk;
    const T* src = q + (size_t)row * p.ldq + (size_t)head * p.dk;
    float most = 0.f;
    for (int d = lane; d < p.dk; d += 32) most = fmaxf(most, fabsf(to_f32(src[d])));
    const uint32_t e = min(max(__float_as_uint(warp_max(most)) >> 23, 1u), 253u);
    const float unit = __uint_as_float(e << 23), inverse = __uint_as_float((254u - e) << 23);
    for (int d = lane; d < p.dk; d += 32) qs[d] = to_f32(src[d]) * inverse;
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
            s = dot * (unit * p.k_scale[at]) * p.scale;
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
int store_launch(void* q_out, const void* q, const void* k, const void* v, const void* v_first, const StoreArgs& p, bool vec, cudaStream_t stream) {
    const dim3 grid((p.T + p.rows - 1) / p.rows, 2 * p.n_kv_heads + p.q_blocks), block(p.rows == 1 ? 128 : 256);
    const cudaError_t e = vec ? qs_launch_dependent(kv8_store_kernel<T, true>, grid, block, 0, stream, (T*)q_out, (const T*)q, (const T*)k, (const T*)v, (const T*)v_first, p)
                              : qs_launch_dependent(kv8_store_kernel<T, false>, grid, block, 0, stream, (T*)q_out, (const T*)q, (const T*)k, (const T*)v, (const T*)v_first, p);
    if (e != cudaSuccess) return qs_fail(QS_ERR_INTERNAL, "kv8 store: %s", cudaGetErrorString(e));
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
    QS_REQUIRE(n_kv_heads <= 16384, "kv8 store: %d key heads exceed the grid", n_kv_heads);
    StoreArgs p = {};
    p.tok_slot = tok_slot; p.tok_pos = tok_pos; p.page_table = page_table;
    p.T = T_tokens; p.max_pages = max_pages; p.n_slots = n_slots; p.n_pages = n_pages;
    p.n_heads = q ? n_heads : 0; p.n_kv_heads = n_kv_heads; p.dk = dk; p.dv = dv; p.R = cos_sin ? R : 0; p.max_pos = cos_sin ? max_pos : 0x7fffffff;
    p.half_layout = half_layout; p.cos_sin = cos_sin;
    p.ldq = (size_t)ldq; p.ldqo = (size_t)ldqo; p.ldk = (size_t)ldk; p.ldv = (size_t)ldv; p.ldvf = (size_t)ldvf;
    p.k_cache = k_cache; p.v_cache = v_cache; p.k_scale = k_scale; p.v_scale = v_scale; p.status = status; p.lam = lam;
    // a row to a block while rows are few (a decode step: every row is a run of its own), else half a page
    p.rows = T_tokens <= 256 ? 1 : 32;
    const int e = dtype == QS_F32 ? 4 : 2;
    auto pieces = [&](const void* x, long long ld) { return !x || (((uintptr_t)x % 16) == 0 && ld * e % 16 == 0); };
    const bool vec = dk % 16 == 0 && dv % 16 == 0 && p.R % (half_layout ? 32 : 16) == 0 && pieces(q, ldq) && pieces(q_out, ldqo) && pieces(k, ldk) && pieces(v, ldv) &&
                     ((uintptr_t)cos_sin % 16) == 0 && ((uintptr_t)k_cache % 16) == 0 && ((uintptr_t)v_cache % 16) == 0;
    const bool queries = q && n_heads > 0 && (p.R > 0 || q != q_out);
    p.q_blocks = queries ? (int)(((long long)p.rows * n_heads * dk / (vec ? 16 : 2) + 1023) / 1024) : 0;
    return dtype == QS_F32 ? store_launch<float>(q_out, q, k, v, v_first, p, vec, stream) : store_launch<__nv_bfloat16>(q_out, q, k, v, v_first, p, vec, stream);
}

// out [n][n_kv_heads][64][dim] of type `dtype`: the numbers in the listed pages.
QS_API int qs_kv8_read_pages(void* out, int dtype, const int8_t* codes, const float* scales, const int32_t* pages, int n, int n_pages, int n_kv_heads,
                             int dim, cudaStream_t stream) {
    if (n == 0) return QS_OK;
    QS_REQUIRE(n > 0 && n <= 65535 && n_pages > 0 && n_kv_heads > 0 && dim > 0, "kv8 read_pages: %d pages of %d heads of %d", n, n_kv_heads, dim);
    QS_REQUIRE(dtype == QS_F32 || dtype == QS_BF16, "kv8 read_pages: type %d", dtype);
    const dim3 grid(n_kv_heads, n);
    const bool vec = dim % 4 == 0 && ((uintptr_t)codes % 16) == 0 && ((uintptr_t)out % 16) == 0;       // a page is 64 * dim codes
    cudaError_t e;
#define GO(T, VEC) e = qs_launch_dependent(kv8_read_pages_kernel<T, VEC>, grid, dim3(256), 0, stream, (T*)out, codes, scales, pages, n_pages, n_kv_heads, dim)
    if (dtype == QS_F32) { if (vec) GO(float, true); else GO(float, false); }
    else if (vec) GO(__nv_bfloat16, true);
    else GO(__nv_bfloat16, false);
#undef GO
    if (e != cudaSuccess) return qs_fail(QS_ERR_INTERNAL, "kv8 read_pages: %s", cudaGetErrorString(e));
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
