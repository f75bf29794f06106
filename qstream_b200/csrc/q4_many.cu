// Products with weights of 4 bits (layout: q4.cu) for many rows of x, on the 5th-generation tensor cores.
//
//   y[m][n] = sum over k of (code - 8) s[n][group] x[m][k]
//
// (code - 8) * s has eleven bits (three of the code, eight of the bfloat16 scale): a 16-bit float holds it exactly, bfloat16 does not.  So both
// operands are 16-bit floats, brought into their range by powers of two: a row of the matrix by that of its largest scale (scales down to 2^-17 of it
// stay exact), a row of x by that of its largest number (its bfloat16 numbers stay exact down to 2^-17 of it, below they are off by 2^-25 of it).  The powers
// come back at the end.  A first kernel finds them and lays out the rows of x: three reads of little.  (The scales outside instead, D read back for every
// 64 columns: 700 rows, 8,192 x 2,048: 160 us, 33 rows, 4,096 x 16,384: 52.)
//
// A block takes 128 rows of the matrix and up to 128 rows of x.  Chunk by chunk of 64 columns:
//   warp 18         copies the codes to shared memory, four chunks of eight tiles at a time (TMA)
//   warps 2 .. 17   four teams, a chunk to each; a warp takes 32 rows: a code c, shifted into the highest bits of a 16-bit 16, is 16 + c; a
//                   multiply-add makes (c - 8) s of it; a word of eight codes is one chunk of 16 bytes of a row in the layout of the 128-byte swizzle.  Lanes of
//                   odd rows write the two halves of the columns in the other order, so that two rows' chunks meet all banks.  (A warp's chunk takes
//                   2,600 cycles, most of them waits; one team of eight warps: 700 rows, 8,192 x 2,048 were half as fast)
//   warp 0          copies the rows of x (TMA)
//   warp 1          multiplies (tcgen05.mma, D [128 x rows of x], 32-bit, in TMEM)
// In the end D goes through shared memory, so that a warp finishes whole rows of results.
// Bound by the way of a chunk through the SM, some 650 cycles whatever the number of rows of x (33 rows, 18,944 columns: 0.34 us for each 64 columns;
// 128 rows: 0.38), where the products take 128 and their operands' way in and out of shared memory 420 to 580.  What did not shorten it, at 700 rows,
// 8,192 x 2,048 (52 us) and 33 rows, 4,096 x 16,384 (31): a second warp that multiplies (53.6, 32.6), 24 decoding warps (57, 34), three stages and two
// slots (53.3, 32), the scales through shared memory (54.4, 31.2).
//
// Where blocks are few, those of a cluster share the columns, and add their sums through distributed shared memory, in their order.
#include "common.cuh"
#include "per_device.h"
#include "sm100.cuh"

#include <cuda_fp16.h>
#include <mutex>

using namespace sm100;

namespace {

constexpr int BM = 128, BN = 128, KC = 64, STAGES = 2, SLOTS = 5, SLOT_CHUNKS = 4;        // a stage holds two chunks
constexpr int TEAMS = SLOT_CHUNKS, TEAM = 4, DECODERS = TEAMS * TEAM, THREADS = (3 + DECODERS) * 32;
constexpr int A_BYTES = BM * KC * 2, B_BYTES = BN * KC * 2, SLOT_BYTES = 8 * SLOT_CHUNKS * 512, STAGE_BYTES = 2 * (A_BYTES + B_BYTES), SMEM = STAGES * STAGE_BYTES + SLOTS * SLOT_BYTES + 1024;
constexpr int PITCH = BM + 4;                            // of a row of x's sums, floats

struct Many {
    void* out;
    const float *row_unit, *x_unit;                      // powers of two: of the matrix's rows (16 for each tile), of the rows of x
    const void *bias, *res0, *res1;
    const uint4* codes;
    const uint32_t* scales;
    size_t ldo, ldr;
    int M, N, chunks, share, columns, out_dtype, bias_dtype, act, settled, vector;       // vector: rows of results and residuals on boundaries of four elements
    int32_t* status;
};

// Not inlined: sixteen copies of every activation are more code than a block runs through, and their way to the SM was a third of the kernel's time.
__device__ __noinline__ float activated(float v, int act) { return apply_activation_wide(v, act); }

// Columns 2 i, 2 i + 1 of a word's eight, times the scale: (16 + c) s - 24 s, and 24 s is exact.
__device__ __forceinline__ uint32_t two_weights(uint32_t word, int i, uint32_t scale, uint32_t less) {
    const uint32_t u = ((i < 2 ? word << (6 - 4 * i) : word >> (4 * i - 6)) & 0x03c003c0u) | 0x4c004c00u;
    uint32_t w;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(w) : "r"(u), "r"(scale), "r"(less));
    return w;
}

// Instruction descriptor of kind::f16 with 16-bit float A and B (both K-major), float32 D.
__device__ __forceinline__ uint32_t idesc_of(int N) { return (1u << 4) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(BM >> 4) << 24); }

// The power of two at or below |x| (2^-126 to 2^126); its inverse is one too.
__device__ __forceinline__ float unit_of(float x) { return __uint_as_float(min(max(__float_as_uint(fabsf(x)) >> 23, 1u), 253u) << 23); }
__device__ __forceinline__ float inverse_of(float unit) { return __uint_as_float((254u << 23) - __float_as_uint(unit)); }

// Blocks 0 .. M - 1: a row of x as 16-bit floats below 2 and its power of two.  The others: the powers of the rows of a tile of the matrix.
__global__ void __launch_bounds__(256)
q4_units_kernel(__half* __restrict__ xh, float* __restrict__ x_unit, float* __restrict__ row_unit, const __nv_bfloat16* __restrict__ x, size_t ldx, int M, int columns,
                const uint32_t* __restrict__ scales, int groups, int tiles) {
    __shared__ float most[8][16];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    grid_dep_launch();
    grid_dep_wait();
    if ((int)blockIdx.x < M) {
        const uint4* src = reinterpret_cast<const uint4*>(x + (size_t)blockIdx.x * ldx);
        float m = 0.f;
        for (int i = threadIdx.x; i < columns / 8; i += 256) {
            const uint4 raw = src[i];
            const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) m = fmaxf(m, fmaxf(fabsf(__uint_as_float(w[j] << 16)), fabsf(__uint_as_float(w[j] & 0xffff0000u))));
        }
        m = warp_max(m);
        if (lane == 0) most[warp][0] = m;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 8; ++i) m = fmaxf(m, most[i][0]);
        const float unit = unit_of(m), inv = inverse_of(unit);
        if (threadIdx.x == 0) x_unit[blockIdx.x] = unit;
        uint4* dst = reinterpret_cast<uint4*>(xh + (size_t)blockIdx.x * columns);
        for (int i = threadIdx.x; i < columns / 8; i += 256) {
            const uint4 raw = src[i];
            const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
            uint32_t o[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const __half2 h = __floats2half2_rn(__uint_as_float(w[j] << 16) * inv, __uint_as_float(w[j] & 0xffff0000u) * inv);
                o[j] = *reinterpret_cast<const uint32_t*>(&h);
            }
            dst[i] = make_uint4(o[0], o[1], o[2], o[3]);
        }
        return;
    }
    const int tile = blockIdx.x - M;                     // words (g, u = 0 and 1) of a group: eight lanes
    float m[2] = {0.f, 0.f};
    for (int i = threadIdx.x; i < groups * 8; i += 256) {
        const uint32_t pair = scales[(size_t)tile * groups * 8 + i];
        m[0] = fmaxf(m[0], fabsf(__uint_as_float(pair << 16)));
        m[1] = fmaxf(m[1], fabsf(__uint_as_float(pair & 0xffff0000u)));
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
#pragma unroll
        for (int o = 8; o < 32; o <<= 1) m[u] = fmaxf(m[u], __shfl_xor_sync(0xffffffffu, m[u], o));
        if (lane < 8) most[warp][lane + 8 * u] = m[u];
    }
    __syncthreads();
    if (threadIdx.x < 16) {
        float a = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) a = fmaxf(a, most[i][threadIdx.x]);
        row_unit[tile * 16 + threadIdx.x] = unit_of(a);
    }
}

template <int GROUP>
__global__ void __launch_bounds__(THREADS, 1)
q4_many_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_codes, const Many p) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    __shared__ uint64_t full[STAGES], empty[STAGES], done, c_full[SLOTS], c_empty[SLOTS];
    __shared__ uint32_t tmem_slot;
    __shared__ volatile int aborted;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint32_t rank, blocks;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(blocks));
    const int row0 = (int)(blockIdx.x / blocks) * BM, m0 = blockIdx.y * BN;
    const int tiles = (p.N + 15) >> 4, groups = (p.chunks * 64 + GROUP - 1) / GROUP;
    const int c0 = (int)rank * p.share, n = max(0, min(p.share, p.chunks - c0));        // this block's chunks

    if (threadIdx.x == 0) {
        for (int i = 0; i < STAGES; ++i) { mbar_init(&full[i], 2 * TEAM + 1); mbar_init(&empty[i], 1); }
        for (int i = 0; i < SLOTS; ++i) { mbar_init(&c_full[i], 1); mbar_init(&c_empty[i], DECODERS); }
        mbar_init(&done, 1);
        aborted = 0;
        mbar_fence_init();
        prefetch_tensormap(&map_x);
        prefetch_tensormap(&map_codes);
    }
    if (warp == 1) { tmem_alloc(&tmem_slot, BN); tmem_relinquish(); }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem = tmem_slot;
    uint8_t* slots = smem + STAGES * STAGE_BYTES;
    const int pairs = (n + 1) >> 1;

    if (warp == 0) {
        // ------------------------------------------------------------------ rows of x
        grid_dep_wait();
        if (elect_one()) {
            int i = 0;
            for (; i < pairs && !aborted; ++i) {
                const int st = i % STAGES, here = min(2, n - 2 * i);
                if (!mbar_wait(&empty[st], ((i / STAGES) & 1) ^ 1)) { atomicExch(p.status, 130); aborted = 1; break; }
                uint8_t* dst = smem + st * STAGE_BYTES + 2 * A_BYTES;
                mbar_expect_tx(&full[st], here * p.columns * KC * 2);
                for (int k = 0; k < here; ++k) tma_load_2d(dst + k * B_BYTES, &map_x, &full[st], (c0 + 2 * i + k) * KC, m0);
            }
            if (aborted)                                 // no copy outlives the block (the other arrivals of the phase may be missing: until the limit)
                for (int k = max(0, i - STAGES); k < i; ++k) mbar_wait(&full[k % STAGES], (k / STAGES) & 1);
        }
        __syncwarp();
    } else if (warp == 1) {
        // ------------------------------------------------------------------ products
        grid_dep_wait();
        if (elect_one()) {
            const uint32_t idesc = idesc_of(p.columns);
            for (int i = 0; i < pairs && !aborted; ++i) {
                const int st = i % STAGES, steps = min(8, 4 * (n - 2 * i));
                if (!mbar_wait(&full[st], (i / STAGES) & 1)) { atomicExch(p.status, 131); aborted = 1; break; }
                tc_fence_after_sync();
                const uint32_t a = smem_u32(smem + st * STAGE_BYTES), b = a + 2 * A_BYTES;
                for (int k = 0; k < steps; ++k) {
                    const uint32_t at = (k >> 2) * A_BYTES + (k & 3) * 32;     // (a chunk of the rows of x takes as much)
                    mma_bf16(tmem, smem_desc_sw128(a + at), smem_desc_sw128(b + at), idesc, (i | k) != 0);
                }
                mma_commit(&empty[st]);
            }
            mma_commit(&done);                           // nor a product
            if (!mbar_wait(&done, 0)) { atomicExch(p.status, 135); aborted = 1; }
        }
        __syncwarp();
    } else if (warp < 2 + DECODERS) {
        // ------------------------------------------------------------------ codes to numbers
        const int team = (warp - 2) / TEAM, mine = (warp - 2) % TEAM * 2, g = lane >> 2, t = lane & 3, odd = g & 1;      // chunks team, + TEAMS, ..., tiles mine and the next
        bool ok = true;
        grid_dep_wait();
        // the scales of rows g and g + 8 (both halves of a word), over the rows' powers of two; those of two chunks ahead
        constexpr int PER = GROUP == 32 ? 2 : 1;         // groups of a chunk
        const uint32_t* scales[2];
        float inv[2][2];
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            const size_t tile = min((row0 >> 4) + mine + q, tiles - 1);
            scales[q] = p.scales + tile * groups * 8 + g;
            inv[q][0] = inverse_of(p.row_unit[tile * 16 + g]);
            inv[q][1] = inverse_of(p.row_unit[tile * 16 + 8 + g]);
        }
        uint32_t ahead[2][PER][2];
        auto fetch = [&](uint32_t (&to)[PER][2], int i) {
#pragma unroll
            for (int h = 0; h < PER; ++h)
#pragma unroll
                for (int q = 0; q < 2; ++q) to[h][q] = __ldg(scales[q] + (size_t)min((c0 + i) * 64 / GROUP + h, groups - 1) * 8);
        };
        fetch(ahead[0], team);
        fetch(ahead[1], team + TEAMS);
        for (int i0 = team; i0 < 2 * pairs && ok; i0 += 2 * TEAMS)
#pragma unroll
        for (int turn = 0; turn < 2; ++turn) {
            const int i = i0 + turn * TEAMS;
            if (i >= 2 * pairs) break;
            const int pair = i >> 1, st = pair % STAGES, slot = i / SLOT_CHUNKS % SLOTS;
            if (i < n && !mbar_wait(&c_full[slot], (i / SLOT_CHUNKS / SLOTS) & 1)) ok = false;
            if (ok && (aborted || !mbar_wait(&empty[st], ((pair / STAGES) & 1) ^ 1))) ok = false;
            if (!ok) { if (lane == 0) atomicExch(p.status, 133); aborted = 1; break; }
            // Half a stage at the end has nothing to write, but its arrival is for this phase too: not before the stage is free, or the stage's last
            // phase, still short of others, would count it.
            if (i >= n) {
                if (lane == 0) mbar_arrive(&full[st]);
                break;
            }
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                uint32_t unit[PER][2], less[PER][2];
#pragma unroll
                for (int h = 0; h < PER; ++h) {
                    const uint32_t two = ahead[turn][h][q];
                    const __half2 a = __float2half2_rn(__uint_as_float(two << 16) * inv[q][0]), b = __float2half2_rn(__uint_as_float(two & 0xffff0000u) * inv[q][1]);
                    unit[h][0] = *reinterpret_cast<const uint32_t*>(&a);
                    unit[h][1] = *reinterpret_cast<const uint32_t*>(&b);
#pragma unroll
                    for (int k = 0; k < 2; ++k) asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(less[h][k]) : "r"(unit[h][k]), "r"(0xce00ce00u));       // -24
                }
                const uint4 raw = *reinterpret_cast<const uint4*>(slots + slot * SLOT_BYTES + ((mine + q) * SLOT_CHUNKS + i % SLOT_CHUNKS) * 512 + lane * 16);
                uint8_t* tile = smem + st * STAGE_BYTES + (i & 1) * A_BYTES + (16 * (mine + q) + g) * 128;
                // words: row g and g + 8, columns 0 .. 31, then the same of 32 .. 63; odd rows the other way round
                const uint32_t w[4] = {odd ? raw.z : raw.x, odd ? raw.w : raw.y, odd ? raw.x : raw.z, odd ? raw.y : raw.w};
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int at = ((4 * ((k >> 1) ^ odd) + t) ^ g) << 4;
                    const bool second = PER == 2 && ((k >> 1) ^ odd);
                    const uint32_t s = second ? unit[PER - 1][k & 1] : unit[0][k & 1], l = second ? less[PER - 1][k & 1] : less[0][k & 1];
                    *reinterpret_cast<uint4*>(tile + (k & 1) * 8 * 128 + at) = make_uint4(two_weights(w[k], 0, s, l), two_weights(w[k], 1, s, l), two_weights(w[k], 2, s, l), two_weights(w[k], 3, s, l));
                }
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {                             // (32 arrivals of a warp would come one behind the other)
                mbar_arrive(&full[st]);
                mbar_arrive(&c_empty[slot]);
            }
            fetch(ahead[turn], i + 2 * TEAMS);
        }
    } else {
        // ------------------------------------------------------------------ codes
        if (!p.settled) grid_dep_wait();
        if (elect_one()) {
            int i = 0;
            const int count = (n + SLOT_CHUNKS - 1) / SLOT_CHUNKS;
            for (; i < count && !aborted; ++i) {
                const int slot = i % SLOTS;
                if (!mbar_wait(&c_empty[slot], ((i / SLOTS) & 1) ^ 1)) { atomicExch(p.status, 136); aborted = 1; break; }
                mbar_expect_tx(&c_full[slot], SLOT_BYTES);         // (chunks behind the block's and tiles behind the last: read or zeros, for nobody)
                tma_load_4d(slots + slot * SLOT_BYTES, &map_codes, &c_full[slot], 0, c0 + i * SLOT_CHUNKS, row0 >> 4, 0);
            }
            for (int k = max(0, i - SLOTS); k < i; ++k) mbar_wait(&c_full[k % SLOTS], (k / SLOTS) & 1);       // no copy outlives the block
        }
        __syncwarp();
        if (p.settled) grid_dep_wait();
    }
    __syncwarp();
    grid_dep_launch();

    // ------------------------------------------------------------------ results
    if (!mbar_wait(&done, 0)) { if (lane == 0) atomicExch(p.status, 134); aborted = 1; }
    __syncthreads();                                     // nobody waits for a copy or reads a stage any more
    tc_fence_after_sync();
    float* part = reinterpret_cast<float*>(smem);        // [row of x][row of the matrix], where the stages were
    if (warp >= 4 && warp < 12) {                        // a warp may read the lanes 32 (warp % 4) ...: two warps to each 32 rows of the matrix
        const int r = (warp & 3) * 32 + lane, half = (warp - 4) >> 2;
        for (int q = half * 64; q < min(half * 64 + 64, p.columns); q += 16) {
            uint32_t d[16];
            tmem_load_32x16(tmem + ((uint32_t)((warp & 3) * 32) << 16) + (uint32_t)q, d);
            tmem_load_wait();
#pragma unroll
            for (int j = 0; j < 16; ++j) part[(q + j) * PITCH + r] = n > 0 ? __uint_as_float(d[j]) : 0.f;
        }
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    if (warp == 1) tmem_dealloc(tmem, BN);
    if (blocks > 1) cluster_sync();
    // a warp takes a row of x, a lane four rows of the matrix
    const int row = row0 + 4 * lane, here = max(0, min(4, p.N - row));
    float row_unit[4], bias[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        row_unit[k] = k < here ? p.row_unit[row + k] : 0.f;
        bias[k] = p.bias && k < here ? load_as_f32(p.bias, p.bias_dtype, row + k) : 0.f;
    }
    if (!aborted)
        for (int j = warp * blocks + rank; j < min(p.columns, p.M - m0); j += THREADS / 32 * blocks) {
            const size_t m = m0 + j;
            const float unit = p.x_unit[m];
            float y[4] = {0.f, 0.f, 0.f, 0.f};
            if (blocks == 1) {
                const float4 v = *reinterpret_cast<const float4*>(part + j * PITCH + 4 * lane);
                y[0] = v.x; y[1] = v.y; y[2] = v.z; y[3] = v.w;
            } else {
                for (uint32_t b = 0; b < blocks; ++b) {
                    float v[4];
                    asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]) : "r"(map_to_cta(part + j * PITCH + 4 * lane, b)) : "memory");
#pragma unroll
                    for (int k = 0; k < 4; ++k) y[k] += v[k];
                }
            }
            float add[4] = {0.f, 0.f, 0.f, 0.f};
            const __nv_bfloat16* res[2] = {reinterpret_cast<const __nv_bfloat16*>(p.res0), reinterpret_cast<const __nv_bfloat16*>(p.res1)};
#pragma unroll
            for (int i = 0; i < 2; ++i)
                if (res[i]) {
                    const __nv_bfloat16* src = res[i] + m * p.ldr + row;
                    if (here == 4 && p.vector) {
                        const uint2 raw = *reinterpret_cast<const uint2*>(src);
                        add[0] += __uint_as_float(raw.x << 16); add[1] += __uint_as_float(raw.x & 0xffff0000u);
                        add[2] += __uint_as_float(raw.y << 16); add[3] += __uint_as_float(raw.y & 0xffff0000u);
                    } else {
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            if (k < here) add[k] += to_f32(src[k]);
                    }
                }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                // one power large, the other small: together first, or what comes between has no place in 32 bits
                y[k] = (row_unit[k] > 1.f) != (unit > 1.f) ? y[k] * (row_unit[k] * unit) : y[k] * row_unit[k] * unit;
                y[k] += bias[k];
                if (p.act != QS_ACT_NONE) y[k] = activated(y[k], p.act);
                y[k] += add[k];
            }
            if (here == 4 && p.vector) {
                if (p.out_dtype == QS_F32) *reinterpret_cast<float4*>(reinterpret_cast<float*>(p.out) + m * p.ldo + row) = make_float4(y[0], y[1], y[2], y[3]);
                else {
                    const __nv_bfloat162 a = __floats2bfloat162_rn(y[0], y[1]), b = __floats2bfloat162_rn(y[2], y[3]);
                    *reinterpret_cast<uint2*>(reinterpret_cast<__nv_bfloat16*>(p.out) + m * p.ldo + row) =
                        make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
                }
            } else {
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (k < here) store_from_f32(p.out, p.out_dtype, m * p.ldo + row + k, y[k]);
            }
        }
    if (blocks > 1) cluster_sync();                      // the others have read this block's sums
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                                  CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiledFn encode_fn() {
    static EncodeTiledFn fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess) fn = reinterpret_cast<EncodeTiledFn>(f);
    });
    return fn;
}

template <int GROUP>
int go(const Many& p, const CUtensorMap& map, const CUtensorMap& map_codes, dim3 grid, int blocks, cudaStream_t stream) {
    static PerDevice limit;
    int device = 0;
    cudaGetDevice(&device);
    limit.get(device, [] { return cudaFuncSetAttribute(q4_many_kernel<GROUP>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM) == cudaSuccess ? 1 : 0; });
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = SMEM;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = blocks;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, q4_many_kernel<GROUP>, map, map_codes, p);
    if (e != cudaSuccess) return qs_fail(QS_ERR_INTERNAL, "q4 linear: %s", cudaGetErrorString(e));
    return qs_check_launch("q4 linear");
}

}  // namespace

// Bytes of workspace, a multiple of 16.
long long q4_many_scratch(int M, int N, int chunks) { return (long long)M * chunks * 128 + 4LL * ((M + 3) / 4 * 4) + 64LL * ((N + 15) / 16); }

// bfloat16 rows x [M, chunks * 64] on 16-byte boundaries; the rest as for qs_q4_linear.
int q4_linear_many(void* out, int out_dtype, long long ldo, const void* x, long long ldx, const void* codes, const void* scales, const void* bias, int bias_dtype,
                   int act, const void* res0, const void* res1, long long ldr, int M, int N, int chunks, int group, int settled, void* scratch, int32_t* status, cudaStream_t stream) {
    const int row_tiles = (N + BM - 1) / BM, column_tiles = (M + BN - 1) / BN;
    QS_REQUIRE(column_tiles <= 65535 && (long long)row_tiles * 8 < 0x7fffffffLL, "q4 linear: sizes exceed the grid");
    QS_REQUIRE(status && scratch && ((uintptr_t)scratch % 16) == 0, "q4 linear: no workspace or status word");
    const int groups = (chunks * 64 + group - 1) / group, tiles = (N + 15) / 16;
    __half* xh = (__half*)scratch;
    float* x_unit = (float*)(xh + (size_t)M * chunks * 64);
    float* row_unit = x_unit + (M + 3) / 4 * 4;
    const cudaError_t e = qs_launch_dependent(q4_units_kernel, dim3(M + tiles), dim3(256), 0, stream, xh, x_unit, row_unit, (const __nv_bfloat16*)x, (size_t)ldx, M, chunks * 64,
                                              (const uint32_t*)scales, groups, tiles);
    if (e != cudaSuccess) return qs_fail(QS_ERR_INTERNAL, "q4 linear: %s", cudaGetErrorString(e));
    // blocks to a tile: where they leave SMs idle, as many as leave each four chunks
    int blocks = 1;
    while (blocks < 8 && chunks >= 8 * blocks && 2LL * blocks * row_tiles * column_tiles <= 148) blocks *= 2;
    EncodeTiledFn fn = encode_fn();
    if (!fn) return qs_fail(QS_ERR_INTERNAL, "q4 linear: the driver offers no cuTensorMapEncodeTiled");
    const int columns = M >= BN ? BN : (M + 15) / 16 * 16;
    CUtensorMap map;
    const cuuint64_t dims[2] = {(cuuint64_t)chunks * 64, (cuuint64_t)M};
    const cuuint64_t strides[1] = {(cuuint64_t)chunks * 128};
    const cuuint32_t box[2] = {(cuuint32_t)KC, (cuuint32_t)columns};
    const cuuint32_t elem[2] = {1, 1};
    const CUresult rc = fn(&map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, xh, dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                           CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (rc != CUDA_SUCCESS) return qs_fail(QS_ERR_INTERNAL, "q4 linear: cuTensorMapEncodeTiled failed with %d", (int)rc);
    CUtensorMap map_codes;                               // words, chunks, tiles
    const cuuint64_t code_dims[4] = {128, (cuuint64_t)chunks, (cuuint64_t)tiles, 1};
    const cuuint64_t code_strides[3] = {512, (cuuint64_t)chunks * 512, (cuuint64_t)tiles * chunks * 512};
    const cuuint32_t code_box[4] = {128, SLOT_CHUNKS, 8, 1}, ones[4] = {1, 1, 1, 1};
    const CUresult rc2 = fn(&map_codes, CU_TENSOR_MAP_DATA_TYPE_UINT32, 4, const_cast<void*>(codes), code_dims, code_strides, code_box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                            CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (rc2 != CUDA_SUCCESS) return qs_fail(QS_ERR_INTERNAL, "q4 linear: cuTensorMapEncodeTiled failed with %d", (int)rc2);
    const int o = out_dtype == QS_F32 ? 16 : 8;
    const int vector = ((uintptr_t)out % o) == 0 && ldo % 4 == 0 && ldr % 4 == 0 && ((uintptr_t)res0 % 8) == 0 && ((uintptr_t)res1 % 8) == 0;
    const Many p = {out, row_unit, x_unit, bias, res0, res1, (const uint4*)codes, (const uint32_t*)scales, (size_t)ldo, (size_t)ldr, M, N, chunks, (chunks + blocks - 1) / blocks, columns,
                    out_dtype, bias_dtype, act, settled, vector, status};
    const dim3 grid(row_tiles * blocks, column_tiles);
    if (group == 32) return go<32>(p, map, map_codes, grid, blocks, stream);
    if (group == 64) return go<64>(p, map, map_codes, grid, blocks, stream);
    return go<128>(p, map, map_codes, grid, blocks, stream);
}
