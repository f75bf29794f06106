// Matrix products with weights held in 4 bits: w[n][k] = (code - 8) * scale[n][k / G], codes 0 .. 15, a bfloat16 scale for each row and
// group of G columns (32, 64 or 128); and the rounding of a matrix to that form.
//
// Layout of the codes: tiles of 16 rows and 64 columns, 512 bytes each, [rows / 16][columns / 64][32][4] words of eight codes.  Entry
// lane = 4 g + t, word 2 h + u of a tile holds row g + 8 u, columns 32 h + 8 t + (0, 2, 4, 6, 1, 3, 5, 7), lowest four bits first: 16 bytes
// are what a lane of a warp gives mma.m16n8k16 as its part of the left operand in four steps, and the pairs of columns that the
// operand wants in one register come out of a word by one shift and one mask.  Scales [rows / 16][groups][8][2]: (g, u) is row g + 8 u.
// Rows and columns are filled up to whole tiles with codes of 8 and, for rows, scales of 0.
#include "common.cuh"

namespace {

// The column within eight of a word's i-th code.
__device__ __forceinline__ int column_of(int i) { return i < 4 ? 2 * i : 2 * i - 7; }

// A block rounds one tile's codes for one group of columns or the 64 columns of a chunk, whichever is more: warp = 32 / 8 rows at a time.
// Of a group, m is the element of the largest magnitude (the lowest column of several) and s = bfloat16(-m / 8): m gets the code 0, of which
// there is one more than on the other side; the others round(w / s), at most 7.
template <typename T>
__global__ void __launch_bounds__(256)
q4_quantize_kernel(uint32_t* __restrict__ codes, __nv_bfloat16* __restrict__ scales, const T* __restrict__ w, size_t ldw, int N, int K, int group) {
    const int chunks = (K + 63) / 64, groups = (chunks * 64 + group - 1) / group;
    const int tile = blockIdx.x, span = max(group, 64), c0 = blockIdx.y * (span / 64);
    __shared__ float s_scale[16][4];                     // of the block's rows and groups
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int n_groups = span / group;                   // 1 or 2
    for (int i = warp; i < 16 * n_groups; i += 8) {
        const int r = i / n_groups, gi = i % n_groups, row = tile * 16 + r, grp = blockIdx.y * n_groups + gi;
        float m = 0.f;
        int at = 0x7fffffff;
        for (int k = lane; k < group; k += 32) {
            const int col = grp * group + k;
            const float x = row < N && col < K ? to_f32(w[(size_t)row * ldw + col]) : 0.f;
            if (fabsf(x) > fabsf(m) || isnan(x)) { m = x; at = col; }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const float m2 = __shfl_xor_sync(0xffffffffu, m, o);
            const int at2 = __shfl_xor_sync(0xffffffffu, at, o);
            if (!isnan(m) && (isnan(m2) || fabsf(m2) > fabsf(m) || (fabsf(m2) == fabsf(m) && at2 < at))) { m = m2; at = at2; }
        }
        const __nv_bfloat16 s = __float2bfloat16_rn(m == 0.f ? 0.f : -m * 0.125f);
        if (lane == 0) {
            s_scale[r][gi] = __bfloat162float(s);
            if (grp < groups) scales[(((size_t)tile * groups + grp) * 8 + (r & 7)) * 2 + (r >> 3)] = s;
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < span / 64 * 128; i += 256) {
        const int c = c0 + i / 128, word = i % 128, ln = word >> 2, g = ln >> 2, t = ln & 3, h = word >> 1 & 1, u = word & 1;
        if (c >= chunks) continue;
        const int r = g + 8 * u, row = tile * 16 + r;
        uint32_t bits = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int in = 32 * h + 8 * t + column_of(j), col = c * 64 + in;
            const float s = s_scale[r][group == 32 ? h : 0];
            const float x = row < N && col < K ? to_f32(w[(size_t)row * ldw + col]) : 0.f;
            const int code = s != 0.f ? max(-8, min(7, __float2int_rn(x / s))) : 0;
            bits |= (uint32_t)(code + 8) << (4 * j);
        }
        codes[((size_t)tile * chunks + c) * 128 + word] = bits;
    }
}

// One block per tile of 16 rows and token; the warps share the columns.
template <typename T, typename TO>
__global__ void __launch_bounds__(128)
q4_simple_kernel(TO* __restrict__ out, size_t ldo, const T* __restrict__ x, size_t ldx, const uint4* __restrict__ codes, const uint32_t* __restrict__ scales,
                 const void* __restrict__ bias, int bias_dtype, int act, const T* __restrict__ res0, const T* __restrict__ res1, size_t ldr,
                 int N, int K, int group) {
    __shared__ float part[4][16];
    const int chunks = (K + 63) / 64, groups = (chunks * 64 + group - 1) / group, tile = blockIdx.x, m = blockIdx.y;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    float acc[2] = {0.f, 0.f};
    for (int c = warp; c < chunks; c += 4) {
        const uint4 raw = codes[((size_t)tile * chunks + c) * 32 + lane];
        const uint32_t word[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t pair = scales[((size_t)tile * groups + (c * 64 + 32 * h) / group) * 8 + g];
            const float s[2] = {__uint_as_float(pair << 16), __uint_as_float(pair & 0xffff0000u)};
            float xs[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int col = c * 64 + 32 * h + 8 * t + column_of(j);
                xs[j] = col < K ? to_f32(x[(size_t)m * ldx + col]) : 0.f;
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                float sum = 0.f;
#pragma unroll
                for (int j = 0; j < 8; ++j) sum = fmaf((float)((int)(word[2 * h + u] >> (4 * j) & 15u) - 8), xs[j], sum);
                acc[u] = fmaf(sum, s[u], acc[u]);
            }
        }
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        acc[u] += __shfl_xor_sync(0xffffffffu, acc[u], 1);
        acc[u] += __shfl_xor_sync(0xffffffffu, acc[u], 2);
        if (t == 0) part[warp][g + 8 * u] = acc[u];
    }
    __syncthreads();
    const int n = tile * 16 + threadIdx.x;
    if (threadIdx.x < 16 && n < N) {
        float y = part[0][threadIdx.x] + part[1][threadIdx.x] + part[2][threadIdx.x] + part[3][threadIdx.x];
        if (bias) y += load_as_f32(bias, bias_dtype, n);
        y = apply_activation_wide(y, act);
        if (res0) y += to_f32(res0[(size_t)m * ldr + n]);
        if (res1) y += to_f32(res1[(size_t)m * ldr + n]);
        out[(size_t)m * ldo + n] = from_f32<TO>(y);
    }
}

}  // namespace

QS_API int qs_q4_quantize(void* codes, void* scales, const void* w, int dtype, long long ldw, int N, int K, int group, cudaStream_t stream) {
    QS_REQUIRE(N > 0 && K > 0 && (group == 32 || group == 64 || group == 128), "q4 quantize: a matrix [%d, %d] in groups of %d", N, K, group);
    QS_REQUIRE(dtype == QS_F32 || dtype == QS_BF16, "q4 quantize: type %d", dtype);
    const int span = group > 64 ? group : 64, blocks = (K + span - 1) / span;
    QS_REQUIRE(blocks <= 65535, "q4 quantize: %d columns exceed the grid", K);
    const dim3 grid((N + 15) / 16, blocks);
    if (dtype == QS_F32) q4_quantize_kernel<float><<<grid, 256, 0, stream>>>((uint32_t*)codes, (__nv_bfloat16*)scales, (const float*)w, (size_t)ldw, N, K, group);
    else q4_quantize_kernel<__nv_bfloat16><<<grid, 256, 0, stream>>>((uint32_t*)codes, (__nv_bfloat16*)scales, (const __nv_bfloat16*)w, (size_t)ldw, N, K, group);
    return qs_check_launch("q4 quantize");
}

QS_API int qs_q4_linear(void* out, int out_dtype, long long ldo, const void* x, int dtype, long long ldx, const void* codes, const void* scales,
                        const void* bias, int bias_dtype, int act, const void* res0, const void* res1, long long ldr, int M, int N, int K, int group,
                        cudaStream_t stream) {
    if (M == 0) return QS_OK;
    QS_REQUIRE(M > 0 && M <= 65535 && N > 0 && K > 0 && (group == 32 || group == 64 || group == 128), "q4 linear: [%d, %d] times [%d, %d] in groups of %d", M, K, N, K, group);
    const dim3 grid((N + 15) / 16, M);
#define GO(T, TO) q4_simple_kernel<T, TO><<<grid, 128, 0, stream>>>((TO*)out, (size_t)ldo, (const T*)x, (size_t)ldx, (const uint4*)codes, (const uint32_t*)scales, \
        bias, bias_dtype, act, (const T*)res0, (const T*)res1, (size_t)ldr, N, K, group)
    if (dtype == QS_F32 && out_dtype == QS_F32) GO(float, float);
    else if (dtype == QS_BF16 && out_dtype == QS_BF16) GO(__nv_bfloat16, __nv_bfloat16);
    else if (dtype == QS_BF16 && out_dtype == QS_F32) GO(__nv_bfloat16, float);
    else return qs_fail(QS_ERR_INVALID_INPUT, "q4 linear: rows of type %d and a result of type %d", dtype, out_dtype);
#undef GO
    return qs_check_launch("q4 linear");
}
