// Matrix products with weights held in 4 bits: w[n][k] = (code - 8) * scale[n][k / G], codes 0 .. 15, a bfloat16 scale for each row and
// group of G columns (32, 64 or 128); and the rounding of a matrix to that form.
//
// Layout of the codes: tiles of 16 rows and 64 columns, 512 bytes each, [rows / 16][columns / 64][32][4] words of eight codes.  Entry
// lane = 4 g + t, word 2 h + u of a tile holds row g + 8 u, columns 32 h + 8 t + (0, 2, 4, 6, 1, 3, 5, 7), lowest four bits first: 16 bytes
// are what a lane of a warp gives mma.m16n8k16 as its part of the left operand in four steps, and the pairs of columns that the
// operand wants in one register come out of a word by one shift and one mask.  Scales [rows / 16][groups][8][2]: (g, u) is row g + 8 u.
// Rows and columns are filled up to whole tiles with codes of 8 and, for rows, scales of 0.
#include "common.cuh"
#include "per_device.h"
#include "sm100.cuh"

// For many bfloat16 rows (q4_many.cu).
int q4_linear_many(void* out, int out_dtype, long long ldo, const void* x, long long ldx, const void* codes, const void* scales, const void* bias, int bias_dtype,
                   int act, const void* res0, const void* res1, long long ldr, int M, int N, int chunks, int group, int settled, void* scratch, int32_t* status,
                   cudaStream_t stream);
long long q4_many_scratch(int M, int N, int chunks);

namespace {

// Which bfloat16 products go to the 5th-generation tensor cores: those of more than 16 rows that are large enough for what they take beside (some 11 us for the
// powers of two, the way of the first chunk and of the results).  Microseconds, 16 rows at a time here | there, matrices of 2,048 x 2,048, 4,096 x 4,096,
// 8,192 x 2,048, 16,384 x 4,096 and 4,096 x 16,384: 32 rows 7 | 16, 14 | 14, 13 | 13, 42 | 28, 52 | 31; 64 rows 13 | 17, 27 | 15, 24 | 15, 82 | 30, 102 | 33;
// 128 rows of the first 23 | 21.
bool many_rows(int M, int N, int K, int dtype) { return dtype == QS_BF16 && M > 16 && (double)M * N * K >= 6e8; }

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

// ----------------------------------------------------------------------------- few rows
//
// y[m][n] = sum over groups of s[n][group] * (sum over the group's k of (code - 8) x[m][k]): the codes as bfloat16 numbers and the rows of x
// meet on mma.m16n8k16 (left: 16 rows of the matrix; right: 8 rows of x), whose sums over a group's 64 columns or less are of exact
// products; the scale joins them outside, in 32 bits.
//
// A code c of a word, shifted into the lowest bits of a bfloat16 128, is 128 + c, and 136 less the weight, exactly: 28 masks and
// shifts at two cycles and 16 subtractions at two for a warp's 512 bytes, which memory delivers in 22 cycles of an SM: the conversion takes
// two thirds of the time that the codes take from memory, so nothing else may stand in the loop.  A warp keeps OWN chunks of 64
// columns and their part of the rows of x in registers, and walks over the tiles of 16 rows of the matrix, the codes of two tiles on their way.  (Rows of
// x read in the loop instead, from the caches or from shared memory behind a ring of copies: 8 rows, 16,384 x 4,096 weights 16 to 20 us,
// with the rows in registers 12.6.)
//
// WARPS warps of a block share a tile's columns, the blocks of a cluster share them again where there are more than they hold or tiles are few; a
// block's sums go through shared memory, a cluster's through distributed shared memory, in a fixed order.
//
// A block sums up a round of tiles at a time: eight, or as many as its teams of warps take with the AHEAD tiles that each has on its way.  A round is
// a multiple of those: a tile's place among the ones on their way is its turn modulo AHEAD, and the next round begins with place 0 again.
constexpr int WARPS = 16, TILES = 8, AHEAD = 2;
constexpr int round_of(int share) {
    const int turns = AHEAD * (WARPS / share);
    return turns > TILES ? turns : TILES / turns * turns;
}
template <int NT> constexpr int own_chunks() { return 4 / NT; }
template <int NT> constexpr int warp_sums() { return NT * 8 * 17; }

__device__ __forceinline__ uint32_t two_weights(uint32_t word, int i) {      // columns 2 i, 2 i + 1 of a word's eight
    const uint32_t u = (word >> (4 * i) & 0x000f000fu) | 0x43004300u;
    uint32_t w;
    asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(w) : "r"(u), "r"(0x43084308u));
    return w;
}

__device__ __forceinline__ void mma_add(float (&d)[4], const uint32_t (&a)[4], const uint32_t (&b)[4], int i, uint32_t x0, uint32_t x1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[i]), "r"(b[i]), "r"(a[i + 1]), "r"(b[i + 1]), "r"(x0), "r"(x1));
}

// Rows of x as the products take them: bfloat16, filled up with zeros to a multiple of 64 columns.  A float32 row becomes three, its
// numbers' terms: each is what is left of the number, cut off behind eight bits, so the three are the number exactly.
template <typename T>
__global__ void __launch_bounds__(256)
q4_rows_kernel(uint4* __restrict__ out, const T* __restrict__ x, size_t ldx, int K, int pieces) {
    grid_dep_launch();
    grid_dep_wait();
    const int c = blockIdx.x * 256 + threadIdx.x, m = blockIdx.y;            // eight columns
    if (c >= pieces) return;
    const T* src = x + (size_t)m * ldx + c * 8;
    uint32_t u[3][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float v[2], mid[2], lo[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            v[j] = c * 8 + 2 * i + j < K ? to_f32(src[2 * i + j]) : 0.f;
            const float rest = isfinite(v[j]) ? v[j] - __uint_as_float(__float_as_uint(v[j]) & 0xffff0000u) : 0.f;
            mid[j] = __uint_as_float(__float_as_uint(rest) & 0xffff0000u);
            lo[j] = rest - mid[j];
            if (isnan(v[j])) v[j] = __uint_as_float(0x7fffffffu);
        }
        u[0][i] = __byte_perm(__float_as_uint(v[0]), __float_as_uint(v[1]), 0x7632);
        u[1][i] = __byte_perm(__float_as_uint(mid[0]), __float_as_uint(mid[1]), 0x7632);
        u[2][i] = __byte_perm(__float_as_uint(lo[0]), __float_as_uint(lo[1]), 0x7632);
    }
    constexpr int TERMS = sizeof(T) == 4 ? 3 : 1;
#pragma unroll
    for (int i = 0; i < TERMS; ++i) out[((size_t)m * TERMS + i) * pieces + c] = make_uint4(u[i][0], u[i][1], u[i][2], u[i][3]);
}

struct Few {
    void* out;
    const __nv_bfloat16* x;                              // [M * terms][chunks * 64]
    const void *bias, *res0, *res1;
    const uint4* codes;
    const uint32_t* scales;
    size_t ldo, ldx, ldr;
    int M, N, chunks, share, round, terms, out_dtype, res_dtype, bias_dtype, act, settled;
};

template <int NT, int GROUP>
__global__ void __launch_bounds__(WARPS * 32, 1)
q4_few_kernel(const Few p) {
    // COLS columns of x; a warp's OWN chunks of columns, whose part of x it keeps in registers
    constexpr int COLS = NT * 8, OWN = own_chunks<NT>(), SUMS = warp_sums<NT>();
    constexpr int SCALES = GROUP == 32 ? 2 * OWN : GROUP == 64 ? OWN : OWN / 2;
    extern __shared__ __align__(16) float part[];        // [tiles of a round][warps that share a tile's columns][COLS][17]
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    uint32_t rank, blocks;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(blocks));
    const int chunks = p.chunks, groups = (chunks * 64 + GROUP - 1) / GROUP, tokens = COLS / p.terms, m0 = blockIdx.y * tokens;
    const int tiles = (p.N + 15) >> 4, cluster = blockIdx.x / blocks, n_clusters = gridDim.x / blocks;
    // the warps: `share` of them share a tile's columns, `teams` of these take tiles in turn
    const int share = p.share, teams = WARPS / share, round = p.round, team = warp / share, c0 = ((int)rank * share + warp % share) * OWN;
    const int n = team < teams ? max(0, min(OWN, chunks - c0)) : 0;          // this warp's chunks
    const int n_tiles = cluster < tiles ? (tiles - 1 - cluster) / n_clusters + 1 : 0;   // of the cluster: cluster, + n_clusters, ...

    struct Batch { uint4 raw[OWN]; uint32_t scale[SCALES]; };
    auto load = [&](Batch& b, int k) {                   // the cluster's k-th tile
        if (k >= n_tiles || n == 0) return;
        const size_t tile = cluster + (size_t)k * n_clusters;
        const uint4* q = p.codes + (tile * chunks + c0) * 32 + lane;
        const uint32_t* s = p.scales + (tile * groups + c0 * 64 / GROUP) * 8 + g;
        if (n == OWN) {
#pragma unroll
            for (int u = 0; u < OWN; ++u)
                asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(b.raw[u].x), "=r"(b.raw[u].y), "=r"(b.raw[u].z), "=r"(b.raw[u].w) : "l"(q + u * 32));
#pragma unroll
            for (int i = 0; i < SCALES; ++i) b.scale[i] = __ldg(s + i * 8);
        } else {                                         // the matrix ends among them: the last one again, times zeros
#pragma unroll
            for (int u = 0; u < OWN; ++u) b.raw[u] = __ldg(q + min(u, n - 1) * 32);
#pragma unroll
            for (int i = 0; i < SCALES; ++i) b.scale[i] = __ldg(s + min(i, groups - 1 - c0 * 64 / GROUP) * 8);
        }
    };
    Batch b[AHEAD];
    uint4 x[OWN][2][NT];                                 // columns without a row: the last one, for nobody
    auto load_rows = [&] {
        grid_dep_wait();
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            const uint4* row = reinterpret_cast<const uint4*>(p.x + (size_t)min(m0 * p.terms + j * 8 + g, p.M * p.terms - 1) * p.ldx) + t;
#pragma unroll
            for (int u = 0; u < OWN; ++u)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    x[u][h][j] = make_uint4(0, 0, 0, 0);
                    if (u < n) asm volatile("ld.global.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(x[u][h][j].x), "=r"(x[u][h][j].y), "=r"(x[u][h][j].z), "=r"(x[u][h][j].w) : "l"(row + (size_t)(c0 + u) * 8 + 4 * h));
                }
        }
    };
    // the rows first, or they queue behind the tiles: 2 us of 13 for 8 rows and 16,384 x 4,096 weights
    if (!p.settled) load_rows();
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) load(b[i], team + i * teams);
    if (p.settled) load_rows();
    const uint32_t base = sm100::smem_u32(part);
    for (int first = 0; first < n_tiles; first += round) {
        for (int k0 = first + team; k0 < min(first + round, n_tiles); k0 += AHEAD * teams) {
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) {
                const int k = k0 + i * teams;
                if (k >= min(first + round, n_tiles) || n == 0) break;
                float acc[NT][4];
#pragma unroll
                for (int j = 0; j < NT; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
#pragma unroll
                for (int u = 0; u < OWN; ++u) {
                    float d[NT][4];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint32_t w0 = h ? b[i].raw[u].z : b[i].raw[u].x, w1 = h ? b[i].raw[u].w : b[i].raw[u].y;
                        uint32_t v0[4], v1[4];
#pragma unroll
                        for (int q = 0; q < 4; ++q) { v0[q] = two_weights(w0, q); v1[q] = two_weights(w1, q); }
#pragma unroll
                        for (int j = 0; j < NT; ++j) {
                            if (h == 0 || GROUP == 32) d[j][0] = d[j][1] = d[j][2] = d[j][3] = 0.f;
                            mma_add(d[j], v0, v1, 0, x[u][h][j].x, x[u][h][j].y);
                            mma_add(d[j], v0, v1, 2, x[u][h][j].z, x[u][h][j].w);
                        }
                        if (h == 1 || GROUP == 32) {
                            const uint32_t pair = b[i].scale[GROUP == 32 ? 2 * u + h : u * 64 / GROUP];
                            const float s0 = __uint_as_float(pair << 16), s1 = __uint_as_float(pair & 0xffff0000u);
#pragma unroll
                            for (int j = 0; j < NT; ++j) {
                                acc[j][0] = fmaf(s0, d[j][0], acc[j][0]);
                                acc[j][1] = fmaf(s0, d[j][1], acc[j][1]);
                                acc[j][2] = fmaf(s1, d[j][2], acc[j][2]);
                                acc[j][3] = fmaf(s1, d[j][3], acc[j][3]);
                            }
                        }
                    }
                }
                load(b[i], k + AHEAD * teams);
                float* to = part + ((k - first) * share + warp % share) * SUMS;
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) to[(8 * j + 2 * t + (e & 1)) * 17 + g + 8 * (e >> 1)] = acc[j][e];
            }
        }
        const int some = min(round, n_tiles - first), parts = (min(p.chunks - (int)rank * share * OWN, share * OWN) + OWN - 1) / OWN;
        if (first + round >= n_tiles) grid_dep_launch();
        __syncthreads();
        auto block_sum = [&](int k, int at) {            // over the warps, in their order
            const float* from = part + k * share * SUMS + at;
            float v[WARPS], y = 0.f;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) v[w] = w < parts ? from[w * SUMS] : 0.f;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) y += v[w];
            return y;
        };
        if (blocks > 1) {
            for (int i = threadIdx.x; i < some * COLS * 16; i += WARPS * 32) {
                const int k = i / (COLS * 16), at = i / 16 % COLS * 17 + (i & 15);
                part[k * share * SUMS + at] = block_sum(k, at);
            }
            asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
        }
        auto sum = [&](int k, int at) {                  // over the cluster's blocks, in their order
            if (blocks == 1) return block_sum(k, at);
            float y = 0.f;
            for (uint32_t r = 0; r < blocks; ++r) {
                uint32_t from;
                float v;
                asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(from) : "r"(base + (uint32_t)(k * share * SUMS + at) * 4), "r"(r));
                asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(from) : "memory");
                y += v;
            }
            return y;
        };
        for (int i = threadIdx.x + rank * WARPS * 32; i < some * tokens * 16; i += blocks * WARPS * 32) {
            const int r = i & 15, token = (i >> 4) % tokens, k = (i >> 4) / tokens;
            const int row = (cluster + (first + k) * n_clusters) * 16 + r, m = m0 + token, at = token * p.terms * 17 + r;
            if (row >= p.N || m >= p.M) continue;
            float y = sum(k, at);
            if (p.terms == 3 && isfinite(y)) y += sum(k, at + 17) + sum(k, at + 34);
            if (p.bias) y += load_as_f32(p.bias, p.bias_dtype, row);
            if (p.act != QS_ACT_NONE) y = apply_activation_wide(y, p.act);
            if (p.res0) y += load_as_f32(p.res0, p.res_dtype, (size_t)m * p.ldr + row);
            if (p.res1) y += load_as_f32(p.res1, p.res_dtype, (size_t)m * p.ldr + row);
            store_from_f32(p.out, p.out_dtype, (size_t)m * p.ldo + row, y);
        }
        // everybody has read the sums (the other blocks of the cluster this one's)
        if (blocks > 1) asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
        else __syncthreads();
    }
}

template <int NT, int GROUP>
int few_launch(Few p, cudaStream_t stream) {
    constexpr int OWN = own_chunks<NT>();
    const int tokens = NT * 8 / p.terms, tiles = (p.N + 15) / 16;
    // blocks to a tile: as many as it takes for the columns, and more where tiles are few
    int blocks = 1;
    while (blocks < 8 && (p.chunks > blocks * WARPS * OWN || (p.chunks >= 8 * blocks * OWN && tiles * blocks * 2 <= 148))) blocks *= 2;
    QS_REQUIRE(p.chunks <= blocks * WARPS * OWN, "q4 linear: %d columns exceed what the blocks of a cluster hold (%d)", p.chunks * 64, 8 * WARPS * OWN * 64);
    p.share = ((p.chunks + blocks - 1) / blocks + OWN - 1) / OWN;
    p.round = round_of(p.share);
    const int smem = p.round * p.share * warp_sums<NT>() * 4;       // of TILES * WARPS sums at most: AHEAD * WARPS where a round is longer than TILES
    static PerDevice limit, room[4];
    int device = 0;
    cudaGetDevice(&device);
    limit.get(device, [] { return cudaFuncSetAttribute(q4_few_kernel<NT, GROUP>, cudaFuncAttributeMaxDynamicSharedMemorySize, TILES * WARPS * warp_sums<NT>() * 4) == cudaSuccess ? 1 : 0; });
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(WARPS * 32);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = blocks;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cfg.gridDim = dim3(148 / blocks * blocks);
    const int at_once = room[blocks == 1 ? 0 : blocks == 2 ? 1 : blocks == 4 ? 2 : 3].get(device, [&] {        // clusters that the device runs side by side
        int n = 0;
        return cudaOccupancyMaxActiveClusters(&n, q4_few_kernel<NT, GROUP>, &cfg) == cudaSuccess ? n : 0;
    });
    cfg.gridDim = dim3(min(tiles, at_once > 0 ? at_once : 148 / blocks) * blocks, (p.M + tokens - 1) / tokens);
    cfg.numAttrs = 2;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, q4_few_kernel<NT, GROUP>, p);
    if (e != cudaSuccess) return qs_fail(QS_ERR_INTERNAL, "q4 linear: %s", cudaGetErrorString(e));
    return qs_check_launch("q4 linear");
}

// Which form: by the matrix alone for float32 rows, whose bits are then the same in any batch; bfloat16 rows by their number.
template <int GROUP>
int few(const Few& p, cudaStream_t stream) {
    const bool wide = p.chunks <= 8 * WARPS * own_chunks<2>() && (p.terms == 3 || p.M > 8);
    return wide ? few_launch<2, GROUP>(p, stream) : few_launch<1, GROUP>(p, stream);
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

// Bytes of the rows laid out anew; 0 where the products take them as they are.
static long long rows_scratch(int M, int K, int dtype, int aligned) {
    const int columns = (K + 63) / 64 * 64;
    if (dtype == QS_BF16 && aligned && K == columns) return 0;
    return (long long)M * (dtype == QS_F32 ? 3 : 1) * columns * 2;
}

// Bytes of workspace that `qs_q4_linear` takes, and its kernels.
QS_API long long qs_q4_linear_scratch(int M, int N, int K, int dtype, int aligned) {
    return rows_scratch(M, K, dtype, aligned) + (many_rows(M, N, K, dtype) ? q4_many_scratch(M, N, (K + 63) / 64) : 0);
}
QS_API int qs_q4_linear_kernels(int M, int N, int K, int dtype, int aligned) { return 1 + (rows_scratch(M, K, dtype, aligned) > 0) + many_rows(M, N, K, dtype); }

// out [M, N] = act(x W^T + bias) + residuals; x of type `dtype`, out of type `out_dtype` (float32 for float32 rows).  `aligned`: rows of x begin on
// 16-byte boundaries.  `settled`: codes and scales were complete before the previous kernel of the stream began; the kernel then reads them while that kernel
// still runs.  `scratch`: qs_q4_linear_scratch bytes on a 16-byte boundary.  `status`: set to a code of 130 and more if a wait inside the kernel ran out.
QS_API int qs_q4_linear(void* out, int out_dtype, long long ldo, const void* x, int dtype, long long ldx, int aligned, const void* codes, const void* scales,
                        const void* bias, int bias_dtype, int act, const void* res0, const void* res1, long long ldr, int M, int N, int K, int group,
                        int settled, void* scratch, int32_t* status, cudaStream_t stream) {
    if (M == 0) return QS_OK;
    QS_REQUIRE(M > 0 && N > 0 && K > 0 && (group == 32 || group == 64 || group == 128), "q4 linear: [%d, %d] times [%d, %d] in groups of %d", M, K, N, K, group);
    QS_REQUIRE(((uintptr_t)codes % 16) == 0 && ((uintptr_t)scales % 4) == 0, "q4 linear: codes off their 16-byte boundary");
    QS_REQUIRE(M <= 65535, "q4 linear: %d rows exceed the grid", M);
    QS_REQUIRE((dtype == QS_F32 && out_dtype == QS_F32) || (dtype == QS_BF16 && (out_dtype == QS_F32 || out_dtype == QS_BF16)),
               "q4 linear: rows of type %d and a result of type %d", dtype, out_dtype);
    const int e = dtype == QS_F32 ? 4 : 2, chunks = (K + 63) / 64;
    QS_REQUIRE(!aligned || (((uintptr_t)x % 16) == 0 && ldx * e % 16 == 0), "q4 linear: rows off their 16-byte boundaries");
    Few p = {out, (const __nv_bfloat16*)x, bias, res0, res1, (const uint4*)codes, (const uint32_t*)scales, (size_t)ldo, (size_t)ldx, (size_t)ldr,
             M, N, chunks, 0, 0, dtype == QS_F32 ? 3 : 1, out_dtype, dtype, bias_dtype, act, settled};
    const long long rows = rows_scratch(M, K, dtype, aligned);
    if (rows > 0) {
        QS_REQUIRE(scratch && ((uintptr_t)scratch % 16) == 0, "q4 linear: no workspace");
        const dim3 grid((chunks * 8 + 255) / 256, M);
        const cudaError_t err = dtype == QS_F32
            ? qs_launch_dependent(q4_rows_kernel<float>, grid, dim3(256), 0, stream, (uint4*)scratch, (const float*)x, (size_t)ldx, K, chunks * 8)
            : qs_launch_dependent(q4_rows_kernel<__nv_bfloat16>, grid, dim3(256), 0, stream, (uint4*)scratch, (const __nv_bfloat16*)x, (size_t)ldx, K, chunks * 8);
        if (err != cudaSuccess) return qs_fail(QS_ERR_INTERNAL, "q4 linear: %s", cudaGetErrorString(err));
        p.x = (const __nv_bfloat16*)scratch;
        p.ldx = (size_t)chunks * 64;
    }
    if (many_rows(M, N, K, dtype))
        return q4_linear_many(out, out_dtype, ldo, p.x, (long long)p.ldx, codes, scales, bias, bias_dtype, act, res0, res1, ldr, M, N, chunks, group, settled,
                              (char*)scratch + rows, status, stream);
    if (group == 32) return few<32>(p, stream);
    if (group == 64) return few<64>(p, stream);
    return few<128>(p, stream);
}
