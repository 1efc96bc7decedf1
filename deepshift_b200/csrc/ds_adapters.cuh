// Low-rank adapters of many requests beside a shared projection: the kernels.
//
//   h[m, :] = sum_k x[m, k] down[a, :, k]         down_kernel   (and dh = dy up^T: the same product with up)
//   y[m, :] = base[m, :] + s[a] h[m, :] up[a]     up_kernel     (and dx = s dh down)
//   dw[a]   = sum over a's rows of s h^T x        grad_kernel   (d_up from h and dy, d_down from dh and x)
//
// with a = the adapter of row m.  Both matrices of an adapter are stored by rank ([rank][k], [rank][n]), so that the three
// products of the backward pass are the forward's kernels with their operands' names changed.
//
// Bound by memory: a rank of 16 does some six operations per byte of fp32 activations.  So every operand goes from global
// memory straight to the registers that the matrix instruction reads, in 16-byte loads and without shared memory: the order of the summed
// index is free as long as both operands agree, and so is the order of the output columns, hence a lane takes
// consecutive elements of its row as the elements of several instructions.
//
// fp32 is multiplied as a sum of two TF32 numbers, hi = x cut to 11 bits and lo = x - hi rounded to 11: hi hi + lo hi + hi lo leaves out 2^-21
// of a product at most; a 16-bit operand is one TF32 number already.  All sums are fp32.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "ds_common.cuh"

namespace ds {
namespace adapters {

constexpr int THREADS = 256, WARPS = THREADS / 32;

// Plan of rows (ds_rows_plan): int32 words.
//   [0] tiles   [1] rows with an index outside -1 .. count - 1   [4 ..) first position of each adapter (count + 2)
//   then the tiles, four words each: adapter (count = none), first position, rows, 0;  then the rows sorted by adapter
struct PlanView {
    const int* head;
    const int* offsets;
    const int4* tiles;
    const int* order;
};
constexpr int PLAN_HEAD = 4;
__host__ __device__ inline int plan_tile_rows(int rows) { return rows <= 512 ? 16 : 32; }
__host__ __device__ inline long long plan_tiles(int rows, int count)
{
    const long long groups = rows < count + 1 ? rows : count + 1;
    return rows / plan_tile_rows(rows) + groups;
}
__host__ __device__ inline long long plan_tiles_at(int count) { return (PLAN_HEAD + count + 2 + 3) / 4 * 4; }
__host__ __device__ inline long long plan_order_at(int rows, int count) { return plan_tiles_at(count) + 4 * plan_tiles(rows, count); }
inline PlanView plan_view(const int* plan, int rows, int count)
{
    return {plan, plan + PLAN_HEAD, reinterpret_cast<const int4*>(plan + plan_tiles_at(count)), plan + plan_order_at(rows, count)};
}

struct Args {
    PlanView plan;
    const void* x;        // activations read: x, or the gradient of the output [rows][ldx]
    long long ldx;
    const void* w;        // [count][rank][width]
    const float* scale;   // [count] or null
    float* h;             // [rows][rank8], rank8 = rank to the next multiple of 8, zeros behind rank
    const void* base;     // [rows][ldbase] or null
    long long ldbase;
    void* out;            // [rows][ldout], or a gradient [count][rank][width]
    long long ldout;
    int rows, width, rank, rank8, count;
};

using bf16 = __nv_bfloat16;
using f16 = __half;
template <class T> constexpr bool is_f32 = sizeof(T) == 4;

template <class T> __device__ __forceinline__ float widen(unsigned short v);
template <> __device__ __forceinline__ float widen<bf16>(unsigned short v) { return __uint_as_float(unsigned(v) << 16); }
template <> __device__ __forceinline__ float widen<f16>(unsigned short v) { return __half2float(__ushort_as_half(v)); }
template <> __device__ __forceinline__ float widen<float>(unsigned short) { return 0.f; }
template <class T> __device__ __forceinline__ unsigned short narrow(float v);
template <> __device__ __forceinline__ unsigned short narrow<bf16>(float v) { return __bfloat16_as_ushort(__float2bfloat16_rn(v)); }
template <> __device__ __forceinline__ unsigned short narrow<f16>(float v) { return __half_as_ushort(__float2half_rn(v)); }
template <> __device__ __forceinline__ unsigned short narrow<float>(float) { return 0; }

// N consecutive elements (N * sizeof(T) a multiple of 8 or 16 bytes) as fp32; of them `live` are in range, the rest are 0.
// VEC: all or none are in range, and the address is aligned.
template <class T, int N, bool VEC>
__device__ __forceinline__ void load(const T* p, int live, float (&v)[N])
{
    if (VEC && live >= N) {
        if constexpr (is_f32<T>) {
#pragma unroll
            for (int i = 0; i < N; i += 4) {
                const float4 a = *reinterpret_cast<const float4*>(p + i);
                v[i] = a.x, v[i + 1] = a.y, v[i + 2] = a.z, v[i + 3] = a.w;
            }
        } else {
            unsigned w[N / 2];
            if constexpr (N == 4) {
                const uint2 a = *reinterpret_cast<const uint2*>(p);
                w[0] = a.x, w[1] = a.y;
            } else {
#pragma unroll
                for (int i = 0; i < N / 8; ++i) {
                    const uint4 a = reinterpret_cast<const uint4*>(p)[i];
                    w[4 * i] = a.x, w[4 * i + 1] = a.y, w[4 * i + 2] = a.z, w[4 * i + 3] = a.w;
                }
            }
#pragma unroll
            for (int i = 0; i < N / 2; ++i) {
                v[2 * i] = widen<T>((unsigned short)(w[i] & 0xFFFFu));
                v[2 * i + 1] = widen<T>((unsigned short)(w[i] >> 16));
            }
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
        v[i] = 0.f;
        if (!VEC && i < live) {
            if constexpr (is_f32<T>) v[i] = p[i];
            else v[i] = widen<T>(reinterpret_cast<const unsigned short*>(p)[i]);
        }
    }
}

template <class T, int N, bool VEC>
__device__ __forceinline__ void store(T* p, int live, const float (&v)[N])
{
    if (VEC && live >= N) {
        if constexpr (is_f32<T>) {
#pragma unroll
            for (int i = 0; i < N; i += 4) *reinterpret_cast<float4*>(p + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
        } else {
            static_assert(N % 8 == 0, "whole 16-byte stores");
#pragma unroll
            for (int i = 0; i < N; i += 8) {
                unsigned w[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) w[e] = narrow<T>(v[i + 2 * e]) | unsigned(narrow<T>(v[i + 2 * e + 1])) << 16;
                *reinterpret_cast<uint4*>(p + i) = make_uint4(w[0], w[1], w[2], w[3]);
            }
        }
        return;
    }
    if constexpr (!VEC) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if (i < live) {
                if constexpr (is_f32<T>) p[i] = v[i];
                else reinterpret_cast<unsigned short*>(p)[i] = narrow<T>(v[i]);
            }
        }
    }
}

__device__ __forceinline__ unsigned to_tf32(float v)
{
    unsigned r;
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(r) : "f"(v));
    return r;
}

// hi + lo = v to 21 bits (an infinity, whose lo is none, ends up as NaN).
__device__ __forceinline__ void split(float v, unsigned& hi, unsigned& lo)
{
    hi = __float_as_uint(v) & 0xFFFFE000u;
    lo = to_tf32(v - __uint_as_float(hi));
}

// A value that is a TF32 number already, or its two parts.
template <bool EXACT>
__device__ __forceinline__ void parts(float v, unsigned& hi, unsigned& lo)
{
    if (EXACT) hi = __float_as_uint(v), lo = 0;
    else split(v, hi, lo);
}

__device__ __forceinline__ void mma_tf32(float (&d)[4], const unsigned (&a)[4], unsigned b0, unsigned b1)
{
    asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <class T>
__device__ __forceinline__ void mma_16bit(float (&d)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1)
{
    if constexpr (sizeof(T) == 2 && __is_same(T, bf16))
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Row of lane's fragment rows: position p of the tile, or -1 behind its end.
__device__ __forceinline__ int tile_row(const PlanView& plan, const int4& tile, int p) { return p < tile.z ? plan.order[tile.y + p] : -1; }

// Sixteen bytes from global to shared memory behind the thread's back, or zeros.  Each lane fills and reads slots of its own:
// a queue deeper than registers would allow, and no barrier.
__device__ __forceinline__ void copy16(unsigned to, const void* from, bool live)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copies_end() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory"); }

__device__ __forceinline__ uint4 slot(unsigned at)
{
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
    return v;
}

__device__ __forceinline__ unsigned shared_address(const void* p) { return (unsigned)__cvta_generic_to_shared(p); }

// The elements of N pieces as fp32.
template <class T, int N>
__device__ __forceinline__ void widen_pieces(const uint4 (&p)[N], float (&v)[N * 16 / sizeof(T)])
{
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const unsigned w[4] = {p[i].x, p[i].y, p[i].z, p[i].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if constexpr (is_f32<T>) v[4 * i + e] = __uint_as_float(w[e]);
            else {
                v[8 * i + 2 * e] = widen<T>((unsigned short)(w[e] & 0xFFFFu));
                v[8 * i + 2 * e + 1] = widen<T>((unsigned short)(w[e] >> 16));
            }
        }
    }
}

// Shapes of down_kernel: elements a lane takes of a row at a time (sixteen bytes of the narrower type), the 16-byte pieces of
// that in both operands, and how many such steps are on their way (96 KB a CTA, so that two fit an SM; two steps at least).
template <class X, class W, int MT, int NT>
struct Down {
    static constexpr bool SAME = !is_f32<X> && __is_same(X, W);   // both of one 16-bit type: no conversion at all
    static constexpr int LK = is_f32<X> && is_f32<W> ? 4 : 8, XP = LK * sizeof(X) / 16, WP = LK * sizeof(W) / 16;
    static constexpr int PIECES = 2 * MT * XP + NT * WP, STAGE = THREADS * 16 * PIECES;
    static constexpr int FIT = 98304 / STAGE, STAGES = FIT < 2 ? 2 : FIT > 6 ? 6 : FIT;
    static constexpr int SUMS = WARPS * 16 * MT * 8 * NT * 4;
    static constexpr int smem(bool vec) { return vec && STAGES * STAGE > SUMS ? STAGES * STAGE : SUMS; }
};

// One step's products.  fp32 sums of a few products begin at zero and are added to the running ones by the adder, which rounds; the
// tensor core's own additions cut off, and a chain of 200 of them had a relative error of 3e-6.
template <class X, class W, int MT, int NT, int LK>
__device__ __forceinline__ void down_step(float (&acc)[MT][NT][4], const float (&a)[2 * MT][LK], const float (&b)[NT][LK])
{
#pragma unroll
    for (int e = 0; e < LK; e += 2) {
        unsigned ah[MT][4], al[MT][4];
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            parts<!is_f32<X>>(a[2 * i][e], ah[i][0], al[i][0]);
            parts<!is_f32<X>>(a[2 * i + 1][e], ah[i][1], al[i][1]);
            parts<!is_f32<X>>(a[2 * i][e + 1], ah[i][2], al[i][2]);
            parts<!is_f32<X>>(a[2 * i + 1][e + 1], ah[i][3], al[i][3]);
        }
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            unsigned h0, h1, l0, l1;
            parts<!is_f32<W>>(b[j][e], h0, l0);
            parts<!is_f32<W>>(b[j][e + 1], h1, l1);
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                float t[4] = {};
                if (is_f32<X>) mma_tf32(t, al[i], h0, h1);
                if (is_f32<W>) mma_tf32(t, ah[i], l0, l1);
                mma_tf32(t, ah[i], h0, h1);
#pragma unroll
                for (int q = 0; q < 4; ++q) acc[i][j][q] += t[q];
            }
        }
    }
}

__device__ __forceinline__ void cluster_sync()
{
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Four consecutive sums of CTA `rank` of the cluster at the place of `here` in its shared memory.
__device__ __forceinline__ float4 sums_of(const float* here, int rank)
{
    unsigned at;
    float4 v;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(shared_address(here)), "r"(rank));
    asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at) : "memory");
    return v;
}

// h for one tile of 16 MT rows: a CTA's warps share the summed index out among them, and so do the `gridDim.y` CTAs of a cluster,
// which add up their sums over distributed shared memory, in their order.  blockIdx.z: ranks by 8 NT.
template <class X, class W, int MT, int NT, bool VEC>
__global__ void __launch_bounds__(THREADS, 2) down_kernel(const Args p)
{
    using S = Down<X, W, MT, NT>;
    constexpr int LK = S::LK, CHUNK = 4 * LK;
    extern __shared__ __align__(16) unsigned char smem[];
    if (int(blockIdx.x) >= p.plan.head[0]) return;
    const int4 tile = p.plan.tiles[blockIdx.x];
    if (tile.x >= p.count) return;   // rows without an adapter: nothing reads their h
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int r0 = blockIdx.z * 8 * NT;
    // rows g, 8 + g, ... of this CTA's ranks, and where this lane's elements begin
    const W* w = static_cast<const W*>(p.w) + ((long long)tile.x * p.rank + r0 + g) * p.width + t * LK;
    const long long eight = 8ll * p.width;
    const int ranks = p.rank - r0 - g;   // row 8 j is one as long as 8 j is less
    const X* xr[2 * MT];
#pragma unroll
    for (int i = 0; i < 2 * MT; ++i) {
        const int m = tile_row(p.plan, tile, 8 * i + g);
        xr[i] = m < 0 ? nullptr : static_cast<const X*>(p.x) + m * p.ldx + t * LK;
    }
    float acc[MT][NT][4] = {};
    const int chunks = (p.width + CHUNK - 1) / CHUNK, workers = WARPS * gridDim.y, first = blockIdx.y * WARPS + warp;
    if constexpr (VEC) {
        const unsigned mine = shared_address(smem) + threadIdx.x * 16;
        auto issue = [&](int c, int stage) {
            if (c < chunks) {
                const unsigned to = mine + stage * S::STAGE;
                const bool live = c * CHUNK + t * LK < p.width;   // a width of whole eights: all of the lane's elements, or none
                int q = 0;
#pragma unroll
                for (int i = 0; i < 2 * MT; ++i)
#pragma unroll
                    for (int e = 0; e < S::XP; ++e, ++q)
                        copy16(to + q * THREADS * 16, live && xr[i] ? xr[i] + c * CHUNK + e * (LK / S::XP) : static_cast<const X*>(p.x), live && xr[i]);
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int e = 0; e < S::WP; ++e, ++q)
                        copy16(to + q * THREADS * 16, live && 8 * j < ranks ? w + j * eight + c * CHUNK + e * (LK / S::WP) : static_cast<const W*>(p.w),
                               live && 8 * j < ranks);
            }
            copies_end();
        };
        int stage = 0, ahead = S::STAGES - 1;
#pragma unroll
        for (int i = 0; i < S::STAGES - 1; ++i) issue(first + i * workers, i);
        for (int c = first; c < chunks; c += workers) {
            copies_wait<S::STAGES - 2>();
            const unsigned from = mine + stage * S::STAGE;
            issue(c + (S::STAGES - 1) * workers, ahead);
            stage = stage + 1 == S::STAGES ? 0 : stage + 1;
            ahead = ahead + 1 == S::STAGES ? 0 : ahead + 1;
            uint4 a[2 * MT][S::XP];
#pragma unroll
            for (int i = 0; i < 2 * MT; ++i)
#pragma unroll
                for (int e = 0; e < S::XP; ++e) a[i][e] = slot(from + (i * S::XP + e) * THREADS * 16);
            if constexpr (S::SAME) {
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    const uint4 k = slot(from + (2 * MT + j) * THREADS * 16);
#pragma unroll
                    for (int i = 0; i < MT; ++i) {
                        const uint4 &u = a[2 * i][0], &v = a[2 * i + 1][0];
                        mma_16bit<X>(acc[i][j], u.x, v.x, u.y, v.y, k.x, k.y);
                        mma_16bit<X>(acc[i][j], u.z, v.z, u.w, v.w, k.z, k.w);
                    }
                }
            } else {
                float af[2 * MT][LK], bf[NT][LK];
#pragma unroll
                for (int i = 0; i < 2 * MT; ++i) widen_pieces<X>(a[i], af[i]);
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    uint4 b[S::WP];
#pragma unroll
                    for (int e = 0; e < S::WP; ++e) b[e] = slot(from + (2 * MT * S::XP + j * S::WP + e) * THREADS * 16);
                    widen_pieces<W>(b, bf[j]);
                }
                down_step<X, W, MT, NT, LK>(acc, af, bf);
            }
        }
        copies_wait<0>();
    } else {
        for (int c = first; c < chunks; c += workers) {
            const int k = c * CHUNK, live = p.width - k - t * LK;
            float af[2 * MT][LK], bf[NT][LK];
#pragma unroll
            for (int i = 0; i < 2 * MT; ++i) load<X, LK, false>(xr[i] + k, xr[i] ? live : 0, af[i]);
#pragma unroll
            for (int j = 0; j < NT; ++j) load<W, LK, false>(w + j * eight + k, 8 * j < ranks ? live : 0, bf[j]);
            down_step<X, W, MT, NT, LK>(acc, af, bf);
        }
    }
    constexpr int ROWS = 16 * MT, COLS = 8 * NT;
    float* red = reinterpret_cast<float*>(smem);   // [WARPS][ROWS][COLS]
    __syncthreads();   // the queue's memory is free
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                red[(warp * ROWS + 16 * i + g + (e & 2) * 4) * COLS + 8 * j + 2 * t + (e & 1)] = acc[i][j][e];
    __syncthreads();
    const int shares = gridDim.y;
    if (shares > 1) {
        for (int i = threadIdx.x; i < ROWS * COLS; i += THREADS) {
            float s = 0.f;
#pragma unroll
            for (int q = 0; q < WARPS; ++q) s += red[q * ROWS * COLS + i];
            red[i] = s;   // this thread alone reads and writes element i of each
        }
        cluster_sync();
    }
    for (int i = (blockIdx.y * THREADS + threadIdx.x) * 4; i < ROWS * COLS; i += shares * THREADS * 4) {
        const int row = i / COLS, r = r0 + i % COLS;
        const int m = tile_row(p.plan, tile, row);
        if (m < 0 || r >= p.rank8) continue;
        float s[4] = {};
        for (int q = 0; q < (shares > 1 ? shares : WARPS); ++q) {
            const float4 v = shares > 1 ? sums_of(red + i, q) : *reinterpret_cast<const float4*>(red + q * ROWS * COLS + i);
            s[0] += v.x, s[1] += v.y, s[2] += v.z, s[3] += v.w;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (r + e >= p.rank) s[e] = 0.f;
        *reinterpret_cast<float4*>(p.h + (long long)m * p.rank8 + r) = make_float4(s[0], s[1], s[2], s[3]);
    }
    if (shares > 1) cluster_sync();   // nobody leaves while its sums are being read
}

// Four values of h; 0 without a row.
__device__ __forceinline__ float4 load_h4(const Args& p, int m, int r)
{
    return m < 0 ? make_float4(0.f, 0.f, 0.f, 0.f) : *reinterpret_cast<const float4*>(p.h + (long long)m * p.rank8 + r);
}

// The two parts of v at word `at` of a block of 128 words for hi, 128 for lo.
__device__ __forceinline__ void put_parts(unsigned* at, float v)
{
    unsigned hi, lo;
    split(v, hi, lo);
    at[0] = hi;
    at[128] = lo;
}

// Values r .. r + 3 (r a multiple of 4) of row `at` of a tile into the order in which the instruction reads its first operand [row][rank]:
// blocks [rank / 8][halves of 16 rows][hi, lo][lane][4], the lane that holds row at % 8 and rank pair r % 8 / 2, its
// elements by rows of 8 and then by the pair's second.
__device__ __forceinline__ void put_h4(unsigned* h, int halves, int at, int r, const float4& v, float scale)
{
    unsigned* to = h + (r / 8 * halves + at / 16) * 256 + (at % 8 * 4 + r % 8 / 2) * 4 + (at / 8 & 1);
    put_parts(to, v.x * scale);
    put_parts(to + 2, v.y * scale);
    put_parts(to + 4, v.z * scale);
    put_parts(to + 6, v.w * scale);
}

// One tile of 16 MT rows, 64 columns a warp: lane (g, t) loads eight consecutive columns 8 g .. of ranks 2t and 2t + 1, which are
// the elements of eight instructions, and ends up with the sixteen consecutive columns 16 t .. of rows g and g + 8.  The tile's h,
// scaled and split, lies in shared memory for all warps in the order in which the instructions read it; base is on its way meanwhile.
template <class X, class W, int MT, bool VEC>
__global__ void __launch_bounds__(THREADS, 2) up_kernel(const Args p)
{
    constexpr int BP = 16 * sizeof(X) / 16;   // pieces of a lane's columns of one row
    extern __shared__ __align__(16) unsigned char smem[];
    if (int(blockIdx.x) >= p.plan.head[0]) return;
    const int4 tile = p.plan.tiles[blockIdx.x];
    const bool none = tile.x >= p.count;
    if (none && p.base == p.out) return;   // in place: these rows are there already
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int n0 = (blockIdx.y * WARPS + warp) * 64;
    int row[2 * MT];
#pragma unroll
    for (int i = 0; i < 2 * MT; ++i) row[i] = tile_row(p.plan, tile, 8 * i + g);
    const unsigned mine = shared_address(smem) + p.rank8 * 16 * MT * 8 + threadIdx.x * 16;
    if (VEC && p.base) {
#pragma unroll
        for (int i = 0; i < 2 * MT; ++i)
#pragma unroll
            for (int e = 0; e < BP; ++e) {
                const int n = n0 + 16 * t + e * (16 / BP);
                const bool live = row[i] >= 0 && n < p.width;
                copy16(mine + (i * BP + e) * THREADS * 16, static_cast<const X*>(p.base) + (live ? row[i] * p.ldbase + n : 0), live);
            }
        copies_end();
    }
    float acc[MT][8][4] = {};
    if (!none) {
        const float scale = p.scale ? p.scale[tile.x] : 1.f;
        unsigned* h = reinterpret_cast<unsigned*>(smem);
        constexpr int PER = THREADS / (16 * MT);   // threads a row
        const int at = threadIdx.x / PER, m = tile_row(p.plan, tile, at);
        for (int r = threadIdx.x % PER * 4; r < p.rank8; r += PER * 4) put_h4(h, MT, at, r, load_h4(p, m, r), scale);
        __syncthreads();
        const W* w = static_cast<const W*>(p.w) + (long long)tile.x * p.rank * p.width + n0 + 8 * g;
        const int live = p.width - n0 - 8 * g;
        float next[2][8];
        auto fetch = [&](int r) {
#pragma unroll
            for (int e = 0; e < 2; ++e) load<W, 8, VEC>(w + (long long)(r + 2 * t + e) * p.width, r + 2 * t + e < p.rank ? live : 0, next[e]);
        };
        fetch(0);
        for (int r = 0; r < p.rank8; r += 8) {
            float b[2][8];
#pragma unroll
            for (int e = 0; e < 16; ++e) b[e >> 3][e & 7] = next[e >> 3][e & 7];
            if (r + 8 < p.rank8) fetch(r + 8);
            unsigned ah[MT][4], al[MT][4];
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                const unsigned here = shared_address(h + (r / 8 * MT + i) * 256 + lane * 4);
                const uint4 u = slot(here), v = slot(here + 512);
                ah[i][0] = u.x, ah[i][1] = u.y, ah[i][2] = u.z, ah[i][3] = u.w;
                al[i][0] = v.x, al[i][1] = v.y, al[i][2] = v.z, al[i][3] = v.w;
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                unsigned h0, h1, l0, l1;
                parts<!is_f32<W>>(b[0][j], h0, l0);
                parts<!is_f32<W>>(b[1][j], h1, l1);
#pragma unroll
                for (int i = 0; i < MT; ++i) {
                    // fp32 results: as in down_step
                    float s[4] = {};
                    float(&d)[4] = is_f32<X> ? s : acc[i][j];
                    mma_tf32(d, al[i], h0, h1);
                    if (is_f32<W>) mma_tf32(d, ah[i], l0, l1);
                    mma_tf32(d, ah[i], h0, h1);
                    if (is_f32<X>) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) acc[i][j][e] += s[e];
                    }
                }
            }
        }
    }
    // column 8 c + j of the warp's 64 sits in element c of instruction j: c = 2t and 2t + 1 are this lane's
    if (VEC) copies_wait<0>();
#pragma unroll
    for (int i = 0; i < 2 * MT; ++i) {
        if (row[i] < 0) continue;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const int n = n0 + 16 * t + 8 * c, live = p.width - n;
            float v[8] = {};
            if (p.base) {
                if constexpr (VEC) {
                    uint4 q[BP / 2];
#pragma unroll
                    for (int e = 0; e < BP / 2; ++e) q[e] = slot(mine + (i * BP + c * (BP / 2) + e) * THREADS * 16);
                    widen_pieces<X>(q, v);
                } else load<X, 8, VEC>(static_cast<const X*>(p.base) + row[i] * p.ldbase + n, live, v);
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] += acc[i >> 1][j][(i & 1) * 2 + c];
            store<X, 8, VEC>(static_cast<X*>(p.out) + row[i] * p.ldout + n, live, v);
        }
    }
}

// Many rows: up_kernel's product for 256 columns and a run of consecutive tiles of 32 rows.  The adapter's part of `w` stays in shared memory
// until a tile of another adapter comes (up_kernel reads it from L2 for every tile, and waits for it), and the next tile's
// base and h are on their way during a tile's products.  Four warps side by side, two above one another.
template <class X, class W>
struct Stream {
    static constexpr int COLS = 256, ROWS = 32;
    static constexpr int BP = 16 * sizeof(X) / 16, BASE = THREADS * 16 * 2 * BP;   // base of a tile: two rows of sixteen columns a lane
    static constexpr int WROW = COLS * int(sizeof(W)) + 16;   // a row of w: rows 2t of the lanes t fall on different banks
    static constexpr int MOST_RANK = 64;
    __host__ __device__ static constexpr int h_bytes(int rank8) { return ROWS * rank8 * 8; }
    static constexpr int smem(int rank8) { return 2 * BASE + 2 * h_bytes(rank8) + rank8 * WROW; }
};

template <class X, class W>
__global__ void __launch_bounds__(THREADS, 2) up_stream_kernel(const Args p)
{
    using S = Stream<X, W>;
    extern __shared__ __align__(16) unsigned char smem[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int total = p.plan.head[0], first = int((long long)total * blockIdx.x / gridDim.x), last = int((long long)total * (blockIdx.x + 1) / gridDim.x);
    if (first == last) return;
    const int c0 = blockIdx.y * S::COLS, in_block = (warp & 3) * 64, n0 = c0 + in_block, half = warp >> 2;
    const unsigned base_at = shared_address(smem) + threadIdx.x * 16, h_at = shared_address(smem) + 2 * S::BASE, w_at = h_at + 2 * S::h_bytes(p.rank8);
    constexpr int PER = THREADS / S::ROWS, HV = S::MOST_RANK / 4 / PER;   // threads a row, and fours of its h that each brings in
    const int h_row = threadIdx.x / PER, h_rank = threadIdx.x % PER * 4;
    float4 hv[HV];
    // what is known of a tile ahead of time: its rows of this lane, the one whose h this thread brings in, and its scale
    struct Ahead {
        int4 tile;
        int row[2], h_m;
        float scale;
    };
    auto tile_of = [&](int i) { return i < last ? p.plan.tiles[i] : make_int4(p.count, 0, 0, 0); };
    auto rows_of = [&](Ahead& n) {
        n.row[0] = tile_row(p.plan, n.tile, 16 * half + g);
        n.row[1] = tile_row(p.plan, n.tile, 16 * half + 8 + g);
        const bool none = n.tile.x >= p.count;
        n.h_m = none ? -1 : tile_row(p.plan, n.tile, h_row);
        n.scale = p.scale && !none ? p.scale[n.tile.x] : 1.f;
    };
    auto issue_base = [&](const int (&row)[2], int buf) {
        if (p.base) {
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int e = 0; e < S::BP; ++e) {
                    const int n = n0 + 16 * t + e * (16 / S::BP);
                    const bool live = row[i] >= 0 && n < p.width;
                    copy16(base_at + buf * S::BASE + (i * S::BP + e) * THREADS * 16, static_cast<const X*>(p.base) + (live ? row[i] * p.ldbase + n : 0), live);
                }
        }
        copies_end();
    };
    auto fetch_h = [&](const Ahead& n) {
#pragma unroll
        for (int q = 0; q < HV; ++q)
            if (h_rank + q * PER * 4 < p.rank8) hv[q] = load_h4(p, n.h_m, h_rank + q * PER * 4);   // used, and waited for, in put_h
    };
    auto put_h = [&](const Ahead& n, int buf) {
        unsigned* h = reinterpret_cast<unsigned*>(smem + 2 * S::BASE + buf * S::h_bytes(p.rank8));
#pragma unroll
        for (int q = 0; q < HV; ++q)
            if (h_rank + q * PER * 4 < p.rank8) put_h4(h, 2, h_row, h_rank + q * PER * 4, hv[q], n.scale);
    };
    auto load_w = [&](int adapter) {
        constexpr int PER = 16 / sizeof(W), PIECES = S::COLS / PER;
        const W* w = static_cast<const W*>(p.w) + (long long)adapter * p.rank * p.width + c0;
        for (int i = threadIdx.x; i < p.rank8 * PIECES; i += THREADS) {
            const int r = i / PIECES, c = i % PIECES * PER;
            const bool live = r < p.rank && c0 + c < p.width;
            copy16(w_at + r * S::WROW + c * int(sizeof(W)), live ? w + (long long)r * p.width + c : static_cast<const W*>(p.w), live);
        }
        copies_end();
    };
    Ahead now, next;
    now.tile = tile_of(first);
    next.tile = tile_of(first + 1);
    rows_of(now);
    rows_of(next);
    issue_base(now.row, 0);
    int held = -1;   // whose w is in shared memory
    if (now.tile.x < p.count) load_w(held = now.tile.x);
    fetch_h(now);
    put_h(now, 0);
    copies_wait<0>();
    __syncthreads();
    for (int at = first, buf = 0; at < last; ++at, buf ^= 1) {
        issue_base(next.row, buf ^ 1);
        fetch_h(next);
        Ahead then;
        then.tile = tile_of(at + 2);
        const int4 tile = now.tile;
        const int(&row)[2] = now.row;
        float acc[8][4] = {};
        if (tile.x < p.count) {
            const unsigned h = h_at + buf * S::h_bytes(p.rank8) + half * 1024 + lane * 16;
            const unsigned w = w_at + 2 * t * S::WROW + (in_block + 8 * g) * int(sizeof(W));
            for (int r = 0; r < p.rank8; r += 8) {
                constexpr int WP = 8 * sizeof(W) / 16;
                uint4 q[2][WP];
#pragma unroll
                for (int e = 0; e < 2; ++e)
#pragma unroll
                    for (int c = 0; c < WP; ++c) q[e][c] = slot(w + (r + e) * S::WROW + c * 16);
                const uint4 u = slot(h + r / 8 * 2048), v = slot(h + r / 8 * 2048 + 512);
                const unsigned ah[4] = {u.x, u.y, u.z, u.w}, al[4] = {v.x, v.y, v.z, v.w};
                float b[2][8];
                widen_pieces<W>(q[0], b[0]);
                widen_pieces<W>(q[1], b[1]);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    unsigned h0, h1, l0, l1;
                    parts<!is_f32<W>>(b[0][j], h0, l0);
                    parts<!is_f32<W>>(b[1][j], h1, l1);
                    float s[4] = {};   // fp32 results: as in down_step
                    float(&d)[4] = is_f32<X> ? s : acc[j];
                    mma_tf32(d, al, h0, h1);
                    if (is_f32<W>) mma_tf32(d, ah, l0, l1);
                    mma_tf32(d, ah, h0, h1);
                    if (is_f32<X>) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) acc[j][e] += s[e];
                    }
                }
            }
        }
        copies_wait<1>();
        if (!(tile.x >= p.count && p.base == p.out)) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                if (row[i] < 0) continue;
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const int n = n0 + 16 * t + 8 * c;
                    float v[8] = {};
                    if (p.base) {
                        uint4 q[S::BP / 2];
#pragma unroll
                        for (int e = 0; e < S::BP / 2; ++e) q[e] = slot(base_at + buf * S::BASE + (i * S::BP + c * (S::BP / 2) + e) * THREADS * 16);
                        widen_pieces<X>(q, v);
                    }
#pragma unroll
                    for (int j = 0; j < 8; ++j) v[j] += acc[j][i * 2 + c];
                    store<X, 8, true>(static_cast<X*>(p.out) + row[i] * p.ldout + n, p.width - n, v);
                }
            }
        }
        rows_of(then);
        put_h(next, buf ^ 1);
        if (next.tile.x < p.count && next.tile.x != held) {
            __syncthreads();   // everybody is done with the held one
            load_w(held = next.tile.x);
            copies_wait<0>();
        }
        __syncthreads();
        now = next, next = then;
    }
    copies_wait<0>();
}

constexpr int GRAD_STAGES = 4;
template <class X>
constexpr int grad_pieces = 8 * sizeof(X) / 16 * 2;   // of a lane's eight columns of two rows

// dw[a][r0 .. r0 + 16 RT)[n0 .. n0 + 64 CW) over all rows of adapter a.  CW warps side by side, 8 / CW above one another, share a block of rows
// whose h, scaled and split, lies in shared memory in the order in which the instructions read it; the next block's is on its way meanwhile, and
// each lane's rows are several steps ahead.  The `gridDim.z` CTAs of a cluster take one part of the rows each and add up their
// sums over distributed shared memory, in their order.
template <class X, class W, int RT, int CW, bool VEC>
__global__ void __launch_bounds__(THREADS, 2) grad_kernel(const Args p)
{
    constexpr int NJ = 8, RANKS = 16 * RT, COLS = 8 * NJ * CW, XP = grad_pieces<X> / 2, STAGE = THREADS * 16 * grad_pieces<X>;
    constexpr int RW = WARPS / CW, BLOCK = RW == 8 ? 64 : 32, STEPS = BLOCK / 8 / RW;   // rows of a block, steps of a warp in it
    constexpr int HV = (BLOCK * RANKS / 4 + THREADS - 1) / THREADS, H_BYTES = BLOCK * RANKS * 8;
    extern __shared__ __align__(16) unsigned char smem[];   // h of two blocks, then the queue
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3, cw = warp % CW, rw = warp / CW;
    const int blocks = (p.rank + RANKS - 1) / RANKS;
    const int a = blockIdx.x / blocks, n0 = blockIdx.y * COLS + 64 * cw, r0 = blockIdx.x % blocks * RANKS;
    const int shares = gridDim.z, share = blockIdx.z;
    // whole blocks of rows for each CTA
    const int from = p.plan.offsets[a], all = p.plan.offsets[a + 1] - from, part = ((all + shares - 1) / shares + BLOCK - 1) / BLOCK * BLOCK;
    const int begin = from + min(all, share * part), end = from + min(all, (share + 1) * part);
    const float scale = p.scale ? p.scale[a] : 1.f;
    const int n = n0 + NJ * g, live = p.width - n;
    const int count = (end - begin + BLOCK - 1) / BLOCK;
    float acc[RT][NJ][4] = {};
    // step i of this warp: rows 8 (i % STEPS RW + rw) ... of block i / STEPS
    auto row_at = [&](int i, int e) {
        const int at = begin + i / STEPS * BLOCK + (i % STEPS * RW + rw) * 8 + 2 * t + e;
        return at < end ? p.plan.order[at] : -1;
    };
    float4 hv[HV];
    int h_m[HV];   // rows of the block whose h is brought in next, read a block before
    auto fetch_rows = [&](int block) {
#pragma unroll
        for (int q = 0; q < HV; ++q) {
            const int i = threadIdx.x + q * THREADS, r = r0 + i % (RANKS / 4) * 4, at = begin + block * BLOCK + i / (RANKS / 4);
            h_m[q] = i < BLOCK * RANKS / 4 && at < end && r < p.rank8 ? p.plan.order[at] : -1;
        }
    };
    auto fetch_h = [&] {
#pragma unroll
        for (int q = 0; q < HV; ++q) hv[q] = load_h4(p, h_m[q], r0 + (threadIdx.x + q * THREADS) % (RANKS / 4) * 4);
    };
    auto put_h = [&](int buf) {   // as put_h4, but of an operand [rank][row]: blocks [row / 8][RT][hi, lo][lane][4]
        unsigned* h = reinterpret_cast<unsigned*>(smem + buf * H_BYTES);
#pragma unroll
        for (int q = 0; q < HV; ++q) {
            const int i = threadIdx.x + q * THREADS, r = i % (RANKS / 4) * 4, at = i / (RANKS / 4);
            if (i >= BLOCK * RANKS / 4) continue;
            unsigned* to = h + (at / 8 * RT + r / 16) * 256 + (r % 8 * 4 + at % 8 / 2) * 4 + (r / 8 & 1) + 2 * (at & 1);
            put_parts(to, hv[q].x * scale);
            put_parts(to + 16, hv[q].y * scale);
            put_parts(to + 32, hv[q].z * scale);
            put_parts(to + 48, hv[q].w * scale);
        }
    };
    auto products = [&](const float (&b)[2][NJ], unsigned h) {
        unsigned ah[RT][4], al[RT][4];
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            const uint4 u = slot(h + i * 1024), v = slot(h + i * 1024 + 512);
            ah[i][0] = u.x, ah[i][1] = u.y, ah[i][2] = u.z, ah[i][3] = u.w;
            al[i][0] = v.x, al[i][1] = v.y, al[i][2] = v.z, al[i][3] = v.w;
        }
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            unsigned h0, h1, l0, l1;
            parts<!is_f32<X>>(b[0][j], h0, l0);
            parts<!is_f32<X>>(b[1][j], h1, l1);
#pragma unroll
            for (int i = 0; i < RT; ++i) {
                float s[4] = {};   // as in down_step
                float(&d)[4] = is_f32<W> ? s : acc[i][j];
                mma_tf32(d, al[i], h0, h1);
                if (is_f32<X>) mma_tf32(d, ah[i], l0, l1);
                mma_tf32(d, ah[i], h0, h1);
                if (is_f32<W>) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[i][j][e] += s[e];
                }
            }
        }
    };
    const unsigned mine = shared_address(smem) + 2 * H_BYTES + threadIdx.x * 16;
    auto issue = [&](const int (&m)[2], int stage) {
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int q = 0; q < XP; ++q) {
                const bool in = m[e] >= 0 && live > 0;
                copy16(mine + stage * STAGE + (e * XP + q) * THREADS * 16,
                       static_cast<const X*>(p.x) + (in ? m[e] * p.ldx + n + q * (NJ / XP) : 0), in);
            }
        copies_end();
    };
    int rows[2], stage = 0, ahead = GRAD_STAGES - 1;   // the rows of the step whose copies begin next
    if constexpr (VEC) {
#pragma unroll
        for (int i = 0; i < GRAD_STAGES - 1; ++i) {
            const int m[2] = {row_at(i, 0), row_at(i, 1)};
            issue(m, i);
        }
        rows[0] = row_at(GRAD_STAGES - 1, 0), rows[1] = row_at(GRAD_STAGES - 1, 1);
    }
    fetch_rows(0);
    fetch_h();
    fetch_rows(1);
    put_h(0);
    __syncthreads();
    for (int block = 0; block < count; ++block) {
        fetch_h();
        fetch_rows(block + 2);
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            const int i = block * STEPS + s;
            const unsigned h = shared_address(smem) + (block & 1) * H_BYTES + (s * RW + rw) * RT * 1024 + lane * 16;
            float b[2][NJ];
            if constexpr (VEC) {
                copies_wait<GRAD_STAGES - 2>();
                uint4 q[2][XP];
#pragma unroll
                for (int e = 0; e < 2; ++e)
#pragma unroll
                    for (int c = 0; c < XP; ++c) q[e][c] = slot(mine + stage * STAGE + (e * XP + c) * THREADS * 16);
                issue(rows, ahead);
                rows[0] = row_at(i + GRAD_STAGES, 0), rows[1] = row_at(i + GRAD_STAGES, 1);
                stage = stage + 1 == GRAD_STAGES ? 0 : stage + 1;
                ahead = ahead + 1 == GRAD_STAGES ? 0 : ahead + 1;
                widen_pieces<X>(q[0], b[0]);
                widen_pieces<X>(q[1], b[1]);
            } else {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int m = row_at(i, e);
                    load<X, NJ, false>(static_cast<const X*>(p.x) + (m >= 0 ? m * p.ldx + n : 0), m >= 0 ? live : 0, b[e]);
                }
            }
            products(b, h);
        }
        put_h(block + 1 & 1);
        __syncthreads();
    }
    if (VEC) copies_wait<0>();
    float* red = reinterpret_cast<float*>(smem);   // [RW][RANKS][COLS]; the CTA's sums end up in the first
    __syncthreads();
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                red[(rw * RANKS + 16 * i + g + (e & 2) * 4) * COLS + 64 * cw + (2 * t + (e & 1)) * NJ + j] = acc[i][j][e];
    __syncthreads();
    if (shares > 1) {
        if (RW > 1)
            for (int i = threadIdx.x; i < RANKS * COLS; i += THREADS) {
                float s = 0.f;
#pragma unroll
                for (int q = 0; q < RW; ++q) s += red[q * RANKS * COLS + i];
                red[i] = s;   // this thread alone reads and writes element i of each
            }
        cluster_sync();
    }
    for (int i = (share * THREADS + threadIdx.x) * 8; i < RANKS * COLS; i += shares * THREADS * 8) {
        const int r = r0 + i / COLS, at = blockIdx.y * COLS + i % COLS;
        if (r >= p.rank || at >= p.width) continue;
        float s[8] = {};
        if (shares == 1) {
#pragma unroll
            for (int q = 0; q < RW; ++q)
#pragma unroll
                for (int e = 0; e < 8; ++e) s[e] += red[q * RANKS * COLS + i + e];
        } else {
            for (int q = 0; q < shares; ++q) {
                const float4 u = sums_of(red + i, q), v = sums_of(red + i + 4, q);
                s[0] += u.x, s[1] += u.y, s[2] += u.z, s[3] += u.w;
                s[4] += v.x, s[5] += v.y, s[6] += v.z, s[7] += v.w;
            }
        }
        store<W, 8, VEC>(static_cast<W*>(p.out) + ((long long)a * p.rank + r) * p.width + at, p.width - at, s);
    }
    // nobody leaves while its sums are being read
    if (shares > 1) cluster_sync();
}

}  // namespace adapters
}  // namespace ds
