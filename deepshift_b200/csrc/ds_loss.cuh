// Softmax cross entropy of a linear head without its logits: the tensor-core kernel and what its launches share.
//
//   z = H W^T  [rows, vocabulary],   loss_i = log(sum_j exp(z_ij - m_i)) + m_i - z_it
//   G = (softmax(z) - onehot(t)) * weight of the row,   dH = G W,   dW = G^T H
//
// The vocabulary passes in tiles.  Forward, a tile of z lives in tensor memory alone: its epilogue leaves the maximum and the
// sum of exponentials of each row over the tile's columns (8 bytes for 256 logits).  Backward, z is computed again for one piece of
// the vocabulary at a time and leaves as G in 16 bits; two more products make that piece's dW and add to dH.  8 N V D
// operations in all where keeping the logits would take 6, and N x piece x 2 bytes where it would take N x V x 4.
//
// Bound by the tensor cores: one kernel for the four products, persistent, a pair of CTAs (two SMs) on one tile of 256 x 256, each
// with half of both operands in shared memory (TMA, 128-byte swizzle, six stages of 64 k) and 128 rows of fp32 sums in tensor memory,
// twice, so that one tile's epilogue runs beside the next one's products.  Up to 128 rows single CTAs take tiles of 128 x 128.
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "ds_tc_ptx.cuh"

namespace ds {
namespace loss {

constexpr int STAGES = 6, BK = 64, CTA_ROWS = 128;
constexpr int TILE_BYTES = CTA_ROWS * BK * 2, STAGE_BYTES = 2 * TILE_BYTES;
constexpr int THREADS = 256;   // warp 0 loads, warp 1 multiplies, warps 4-7 are the epilogue: a warp reads the tensor-memory lanes of its number mod 4
constexpr unsigned WAIT_NS = 2000000000u;

struct Shared {
    unsigned long long full[STAGES], empty[STAGES], acc_full[2], acc_empty[2], done;
    unsigned tmem;
    int err;
};
constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + 1024 + int(sizeof(Shared));

enum Mode { STATS, GRAD, PRODUCT };

struct Params {
    int tiles_m, tiles_n, k_steps, group;   // group: row tiles that neighbouring tiles of the order share
    int a_mn, b_mn;                         // operand lies with its rows (not k) contiguous
    int is_bf16;
    int m_end, n_end;                       // rows and columns of the result
    // STATS
    const long long* target;
    float2* partial;                        // [tiles_n][m_end]: maximum, sum of exponentials
    float* at_target;                       // logit of the target
    // GRAD
    const float* lse;
    const float* row_weight;
    long long n_first;                      // vocabulary index of column 0
    unsigned short* g;                      // [m_end][ldg]
    int ldg;
    // PRODUCT
    float* acc;                             // [m_end][n_end] sums of several pieces, or null
    int first, last;                        // of the pieces that acc sums
    unsigned short* out;
    const float* scale;
    int* err_flag;
};

// Order of tiles: down `group` row tiles, then to the next column, so that tiles in work at once share both operands in L2.
__device__ __forceinline__ void tile_at(const Params& p, int t, int& m, int& n)
{
    const int per = p.group * p.tiles_n, block = t / per, first = block * p.group;
    const int high = min(p.group, p.tiles_m - first), in = t - block * per;
    m = first + in % high;
    n = in / high;
}

__device__ __forceinline__ unsigned cluster_rank()
{
    unsigned r;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}

__device__ __forceinline__ void cluster_sync()
{
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Address of the same shared-memory variable in the pair's first CTA.
__device__ __forceinline__ unsigned in_leader(const void* p)
{
    unsigned a;
    asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(a) : "r"(s32(p)));
    return a;
}

template <int PAIR>
__device__ __forceinline__ void load_box(unsigned dst, const CUtensorMap* map, int x, int y, unsigned bar)
{
    if constexpr (PAIR == 2)
        asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
                     "l"(map), "r"(x), "r"(y), "r"(bar)
                     : "memory");
    else
        asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst), "l"(map),
                     "r"(x), "r"(y), "r"(bar)
                     : "memory");
}

// 128 rows of an operand, 64 k, from row `row` and index `k`: [row][k] in one box of 64 k x 128 rows, or, where rows are
// contiguous, [k][row] in two boxes of 64 rows x 64 k.
template <int PAIR>
__device__ __forceinline__ void load_tile(unsigned dst, const CUtensorMap* map, int mn, int row, int k, unsigned bar)
{
    if (!mn) load_box<PAIR>(dst, map, k, row, bar);
    else {
        load_box<PAIR>(dst, map, row, k, bar);
        load_box<PAIR>(dst + TILE_BYTES / 2, map, row + 64, k, bar);
    }
}

// Shared-memory descriptor of such a tile (128-byte swizzle, atoms of 8 x 128 bytes): rows by 8 every 1024 bytes, or, with rows
// contiguous, k by 8 every 1024 bytes and rows by 64 every 8192.
__device__ __forceinline__ unsigned long long descriptor(unsigned addr, int mn)
{
    const unsigned long long lead = mn ? (TILE_BYTES / 2) >> 4 : 1, stride = 1024 >> 4;
    return (unsigned long long)((addr & 0x3FFFFu) >> 4) | lead << 16 | stride << 32 | 1ull << 46 | 2ull << 61;
}

template <int PAIR>
__device__ __forceinline__ void mma(unsigned d, unsigned long long a, unsigned long long b, unsigned idesc, unsigned acc)
{
    if constexpr (PAIR == 2)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a),
                     "l"(b), "r"(idesc), "r"(acc)
                     : "memory");
    else
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a),
                     "l"(b), "r"(idesc), "r"(acc)
                     : "memory");
}

// Arrives at `bar` in every CTA of the tile once the products issued so far are done.
template <int PAIR>
__device__ __forceinline__ void commit(unsigned long long* bar)
{
    if constexpr (PAIR == 2)
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(s32(bar)),
                     "h"((unsigned short)3)
                     : "memory");
    else tc_commit(bar);
}

template <int PAIR>
__device__ __forceinline__ void tmem_get(unsigned* at)
{
    if constexpr (PAIR == 2) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(s32(at)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    } else tmem_alloc(at);
}

template <int PAIR>
__device__ __forceinline__ void tmem_free(unsigned base)
{
    if constexpr (PAIR == 2) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(base));
    else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(base));
}

__device__ __forceinline__ float exp2_fast(float x)
{
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

constexpr float LOG2E = 1.4426950408889634f;

__device__ __forceinline__ unsigned pack2(float lo, float hi, int is_bf16)
{
    if (is_bf16) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const unsigned*>(&v);
    }
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const unsigned*>(&v);
}

// One warp's 32 rows of a finished tile; `row` is this lane's, `tmem` the address of the sums of its first column.
template <int PAIR, int MODE>
__device__ __forceinline__ void epilogue(const Params& p, unsigned tmem, int row, int tile_n)
{
    constexpr int BN = 128 * PAIR;
    const int n0 = tile_n * BN, cols = min(BN, p.n_end - n0);
    const bool live = row < p.m_end;
    if constexpr (MODE == STATS) {
        const long long t = live ? p.target[row] - n0 : -1;
        float top = -INFINITY, sum = 0.f;
        for (int c = 0; c < cols; c += 32) {
            int v[32];
            __syncwarp();
            tmem_ld(tmem + c, v);
            float most = -INFINITY;
            if (cols - c < 32) {
#pragma unroll
                for (int i = 0; i < 32; ++i)
                    if (c + i >= cols) v[i] = __float_as_int(-INFINITY);
            }
#pragma unroll
            for (int i = 0; i < 32; ++i) most = fmaxf(most, __int_as_float(v[i]));
            if (live && t >= c && t < c + 32) {
#pragma unroll
                for (int i = 0; i < 32; ++i)
                    if (t == c + i) p.at_target[row] = __int_as_float(v[i]);
            }
            const float next = fmaxf(top, most), from = next == -INFINITY ? 0.f : next;   // a row of -infinity alone sums to 0
            sum *= exp2_fast((top - from) * LOG2E);
            float part[4] = {};
#pragma unroll
            for (int i = 0; i < 32; ++i) part[i & 3] += exp2_fast((__int_as_float(v[i]) - from) * LOG2E);
            sum += (part[0] + part[1]) + (part[2] + part[3]);
            top = next;
        }
        if (live) p.partial[(long long)tile_n * p.m_end + row] = make_float2(top, sum);
    } else if constexpr (MODE == GRAD) {
        // p = exp(z - lse); 1 comes off at the target before the rounding to 16 bits, which is one of half a unit in the last
        // place of each element.  A weight of 0 makes the row 0 whatever its logits are.
        const long long t = live ? p.target[row] - p.n_first - n0 : -1;
        const float lse = live ? p.lse[row] : 0.f, weight = live ? p.row_weight[row] : 0.f;
        const int width = min(BN, p.ldg - n0);
        for (int c = 0; c < width; c += 32) {
            int v[32];
            __syncwarp();
            tmem_ld(tmem + c, v);
            unsigned w[16];
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
                float e[2];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    float q = exp2_fast((__int_as_float(v[i + j]) - lse) * LOG2E);
                    if (t == c + i + j) q -= 1.f;
                    e[j] = weight == 0.f || c + i + j >= cols ? 0.f : q * weight;
                }
                w[i / 2] = pack2(e[0], e[1], p.is_bf16);
            }
            if (live) {
                uint4* to = reinterpret_cast<uint4*>(p.g + (long long)row * p.ldg + n0 + c);
#pragma unroll
                for (int i = 0; i < 4; ++i) to[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
            }
        }
    } else {
        const float scale = p.last ? *p.scale : 0.f;
        for (int c = 0; c < cols; c += 32) {
            int v[32];
            __syncwarp();
            tmem_ld(tmem + c, v);
            if (!live) continue;
            float f[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) f[i] = __int_as_float(v[i]);
            const long long at = (long long)row * p.n_end + n0 + c;
            const bool whole = cols - c >= 32 && p.n_end % 8 == 0;   // 16-byte stores
            if (p.acc && !p.first) {
                if (whole) {
#pragma unroll
                    for (int i = 0; i < 32; i += 4) {
                        const float4 a = *reinterpret_cast<const float4*>(p.acc + at + i);
                        f[i] += a.x, f[i + 1] += a.y, f[i + 2] += a.z, f[i + 3] += a.w;
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 32; ++i)
                        if (c + i < cols) f[i] += p.acc[at + i];
                }
            }
            if (!p.last) {
                if (whole) {
#pragma unroll
                    for (int i = 0; i < 32; i += 4) *reinterpret_cast<float4*>(p.acc + at + i) = make_float4(f[i], f[i + 1], f[i + 2], f[i + 3]);
                } else {
#pragma unroll
                    for (int i = 0; i < 32; ++i)
                        if (c + i < cols) p.acc[at + i] = f[i];
                }
                continue;
            }
            unsigned w[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) w[i] = pack2(f[2 * i] * scale, f[2 * i + 1] * scale, p.is_bf16);
            if (whole) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    reinterpret_cast<uint4*>(p.out + at)[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
            } else {
#pragma unroll
                for (int i = 0; i < 32; ++i)
                    if (c + i < cols) p.out[at + i] = (unsigned short)(w[i / 2] >> (16 * (i & 1)));
            }
        }
    }
}

template <int PAIR, int MODE>
__global__ void __launch_bounds__(THREADS, 1) __cluster_dims__(PAIR, 1, 1)
    tile_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const __grid_constant__ Params p)
{
    constexpr int BN = 128 * PAIR;
    extern __shared__ unsigned char raw[];
    unsigned char* tiles = raw + (1024 - (s32(raw) & 1023)) % 1024;
    Shared& s = *reinterpret_cast<Shared*>(tiles + STAGES * STAGE_BYTES);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const unsigned rank = PAIR == 2 ? cluster_rank() : 0;
    volatile int* err = &s.err;
    if (threadIdx.x == 0) {
        s.err = 0;
        for (int i = 0; i < STAGES; ++i) {
            bar_init(&s.full[i], 1);
            bar_init(&s.empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            bar_init(&s.acc_full[i], 1);
            bar_init(&s.acc_empty[i], 4 * PAIR);
        }
        bar_init(&s.done, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 2) tmem_get<PAIR>(&s.tmem);
    tc_fence_before();
    __syncthreads();
    if (PAIR == 2) cluster_sync();
    tc_fence_after();
    const unsigned tmem = s.tmem;
    const int total = p.tiles_m * p.tiles_n, mine = blockIdx.x / PAIR, step = gridDim.x / PAIR;

    if (warp == 0) {
        if (elect_one()) {
            unsigned stage = 0, phase = 1;   // a fresh barrier is past the phase before its first
            for (int t = mine; t < total && !*err; t += step) {
                int m, n;
                tile_at(p, t, m, n);
                const int row_a = m * BN + int(rank) * CTA_ROWS, row_b = n * BN + int(rank) * CTA_ROWS;
                for (int k = 0; k < p.k_steps; ++k) {
                    if (!bar_wait(&s.empty[stage], phase, err, WAIT_NS)) break;
                    const unsigned bar = PAIR == 2 ? in_leader(&s.full[stage]) : s32(&s.full[stage]);
                    if (rank == 0)
                        asm volatile("{\n\t.reg .b64 st;\n\tmbarrier.arrive.expect_tx.shared::cta.b64 st, [%0], %1;\n\t}" ::"r"(s32(&s.full[stage])),
                                     "n"(STAGE_BYTES * PAIR)
                                     : "memory");
                    const unsigned at = s32(tiles) + stage * STAGE_BYTES;
                    load_tile<PAIR>(at, &map_a, p.a_mn, row_a, k * BK, bar);
                    load_tile<PAIR>(at + TILE_BYTES, &map_b, p.b_mn, row_b, k * BK, bar);
                    if (++stage == STAGES) stage = 0, phase ^= 1;
                }
            }
            // the last products' arrivals here come from the pair's other CTA, too
            for (int i = 0; i < STAGES && bar_wait(&s.empty[stage], phase, err, WAIT_NS); ++i)
                if (++stage == STAGES) stage = 0, phase ^= 1;
        }
    } else if (warp == 1 && rank == 0) {
        if (elect_one()) {
            const unsigned type = p.is_bf16 ? 1 : 0;
            const unsigned idesc = 1u << 4 | type << 7 | type << 10 | unsigned(p.a_mn) << 15 | unsigned(p.b_mn) << 16 | unsigned(BN / 8) << 17 |
                                   unsigned(CTA_ROWS * PAIR / 16) << 24;
            const unsigned step_a = p.a_mn ? 2048 >> 4 : 32 >> 4, step_b = p.b_mn ? 2048 >> 4 : 32 >> 4;   // 16 k further on
            unsigned stage = 0, phase = 0, buf = 0, buf_phase = 1;
            for (int t = mine; t < total; t += step) {
                if (!bar_wait(&s.acc_empty[buf], buf_phase, err, WAIT_NS)) break;
                tc_fence_after();
                const unsigned d = tmem + buf * BN;
                bool ok = true;
                for (int k = 0; k < p.k_steps; ++k) {
                    if (!(ok = bar_wait(&s.full[stage], phase, err, WAIT_NS))) break;
                    tc_fence_after();
                    const unsigned at = s32(tiles) + stage * STAGE_BYTES;
                    const unsigned long long a = descriptor(at, p.a_mn), b = descriptor(at + TILE_BYTES, p.b_mn);
#pragma unroll
                    for (int i = 0; i < BK / 16; ++i) mma<PAIR>(d, a + i * step_a, b + i * step_b, idesc, (k | i) != 0);
                    commit<PAIR>(&s.empty[stage]);
                    if (++stage == STAGES) stage = 0, phase ^= 1;
                }
                if (!ok) break;
                commit<PAIR>(&s.acc_full[buf]);
                if (buf ^= 1; buf == 0) buf_phase ^= 1;
            }
            commit<PAIR>(&s.done);
        }
    } else if (warp >= 4) {
        unsigned buf = 0, buf_phase = 0;
        const int quarter = warp & 3;
        for (int t = mine; t < total; t += step) {
            int m, n;
            tile_at(p, t, m, n);
            if (!__all_sync(0xFFFFFFFFu, bar_wait(&s.acc_full[buf], buf_phase, err, WAIT_NS))) break;
            tc_fence_after();
            epilogue<PAIR, MODE>(p, tmem + buf * BN + (unsigned(quarter * 32) << 16), m * BN + int(rank) * CTA_ROWS + quarter * 32 + lane, n);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                if constexpr (PAIR == 2)
                    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(in_leader(&s.acc_empty[buf])) : "memory");
                else bar_arrive(&s.acc_empty[buf]);
            }
            if (buf ^= 1; buf == 0) buf_phase ^= 1;
        }
    }
    __syncthreads();
    // products and, after a wait that ran out, copies still in flight: nothing of them may outlive the CTA
    if (threadIdx.x == 0) {
        if (!bar_drain(&s.done, 0)) s.err = 1;
        if (s.err) {
            *p.err_flag = 1;
            for (const unsigned long long from = now_ns(); now_ns() - from < 10000000ull;) __nanosleep(100000);
        }
    }
    __syncthreads();
    tc_fence_after();
    if (PAIR == 2) cluster_sync();
    if (warp == 2) tmem_free<PAIR>(tmem);
}

}  // namespace loss
}  // namespace ds
