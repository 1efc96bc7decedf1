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
    float* h;             // [splits][rows][rank8], rank8 = rank to the next multiple of 8, zeros behind rank
    const void* base;     // [rows][ldbase] or null
    long long ldbase;
    void* out;            // [rows][ldout], or a gradient [count][rank][width]
    long long ldout;
    int rows, width, rank, rank8, count, splits;
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
    if (VEC) return;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        if (i < live) {
            if constexpr (is_f32<T>) p[i] = v[i];
            else reinterpret_cast<unsigned short*>(p)[i] = narrow<T>(v[i]);
        }
    }
}

__device__ __forceinline__ unsigned to_tf32(float v)
{
    unsigned r;
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(r) : "f"(v));
    return r;
}

// hi + lo = v to 21 bits; an infinity has no lo.
__device__ __forceinline__ void split(float v, unsigned& hi, unsigned& lo)
{
    hi = __float_as_uint(v) & 0xFFFFE000u;
    const float h = __uint_as_float(hi);
    lo = h == v ? 0u : to_tf32(v - h);
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

// Loads of one 16-byte piece of a 16-bit row, as it is.
template <class T, bool VEC>
__device__ __forceinline__ uint4 load_raw(const T* p, int live)
{
    if (VEC && live >= 8) return *reinterpret_cast<const uint4*>(p);
    unsigned w[4] = {0, 0, 0, 0};
    if (!VEC) {
        const unsigned short* q = reinterpret_cast<const unsigned short*>(p);
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < live) w[i >> 1] |= unsigned(q[i]) << (16 * (i & 1));
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// h for one tile of 16 MT rows: a CTA's warps share the summed index out among them, and so do `splits` CTAs (blockIdx.y),
// each of which writes its own partial sums.  blockIdx.z: ranks by 8 NT.
template <class X, class W, int MT, int NT, bool VEC>
__global__ void __launch_bounds__(THREADS) down_kernel(const Args p)
{
    extern __shared__ float red[];   // [WARPS][16 MT][8 NT]
    if (int(blockIdx.x) >= p.plan.head[0]) return;
    const int4 tile = p.plan.tiles[blockIdx.x];
    if (tile.x >= p.count) return;   // rows without an adapter: nothing reads their h
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int r0 = blockIdx.z * 8 * NT;
    const W* w = static_cast<const W*>(p.w) + (long long)tile.x * p.rank * p.width;
    const X* xr[2 * MT];
#pragma unroll
    for (int i = 0; i < 2 * MT; ++i) {
        const int m = tile_row(p.plan, tile, 8 * i + g);
        xr[i] = m < 0 ? nullptr : static_cast<const X*>(p.x) + m * p.ldx;
    }
    const W* wr[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        const int r = r0 + 8 * j + g;
        wr[j] = r < p.rank ? w + (long long)r * p.width : nullptr;
    }
    float acc[MT][NT][4] = {};
    constexpr bool SAME = !is_f32<X> && __is_same(X, W);   // both of one 16-bit type: no conversion at all
    constexpr int LK = SAME ? 8 : 4;                       // consecutive elements a lane takes
    constexpr int CHUNK = 4 * LK;
    const int chunks = (p.width + CHUNK - 1) / CHUNK, workers = WARPS * p.splits;
#pragma unroll 2
    for (int c = blockIdx.y * WARPS + warp; c < chunks; c += workers) {
        const int k = c * CHUNK + t * LK, live = p.width - k;
        if constexpr (SAME) {
            uint4 a[2 * MT], b[NT];
#pragma unroll
            for (int i = 0; i < 2 * MT; ++i) a[i] = load_raw<X, VEC>(xr[i] + k, xr[i] ? live : 0);
#pragma unroll
            for (int j = 0; j < NT; ++j) b[j] = load_raw<W, VEC>(wr[j] + k, wr[j] ? live : 0);
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    mma_16bit<X>(acc[i][j], a[2 * i].x, a[2 * i + 1].x, a[2 * i].y, a[2 * i + 1].y, b[j].x, b[j].y);
                    mma_16bit<X>(acc[i][j], a[2 * i].z, a[2 * i + 1].z, a[2 * i].w, a[2 * i + 1].w, b[j].z, b[j].w);
                }
        } else {
            float a[2 * MT][4], b[NT][4];
#pragma unroll
            for (int i = 0; i < 2 * MT; ++i) load<X, 4, VEC>(xr[i] + k, xr[i] ? live : 0, a[i]);
#pragma unroll
            for (int j = 0; j < NT; ++j) load<W, 4, VEC>(wr[j] + k, wr[j] ? live : 0, b[j]);
#pragma unroll
            for (int e = 0; e < 4; e += 2) {
                unsigned ah[MT][4], al[MT][4];
#pragma unroll
                for (int i = 0; i < MT; ++i) {
                    split(a[2 * i][e], ah[i][0], al[i][0]);
                    split(a[2 * i + 1][e], ah[i][1], al[i][1]);
                    split(a[2 * i][e + 1], ah[i][2], al[i][2]);
                    split(a[2 * i + 1][e + 1], ah[i][3], al[i][3]);
                }
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    unsigned b0, b1, l0, l1;
                    split(b[j][e], b0, l0);
                    split(b[j][e + 1], b1, l1);
#pragma unroll
                    for (int i = 0; i < MT; ++i) {
                        mma_tf32(acc[i][j], ah[i], b0, b1);
                        if (is_f32<X>) mma_tf32(acc[i][j], al[i], b0, b1);
                        if (is_f32<W>) mma_tf32(acc[i][j], ah[i], l0, l1);
                    }
                }
            }
        }
    }
    constexpr int ROWS = 16 * MT, COLS = 8 * NT;
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                red[(warp * ROWS + 16 * i + g + (e & 2) * 4) * COLS + 8 * j + 2 * t + (e & 1)] = acc[i][j][e];
    __syncthreads();
    for (int i = threadIdx.x; i < ROWS * COLS; i += THREADS) {
        const int row = i / COLS, r = r0 + i % COLS;
        const int m = tile_row(p.plan, tile, row);
        if (m < 0 || r >= p.rank8) continue;
        float s = 0.f;
#pragma unroll
        for (int q = 0; q < WARPS; ++q) s += red[q * ROWS * COLS + i];
        p.h[((long long)blockIdx.y * p.rows + m) * p.rank8 + r] = r < p.rank ? s : 0.f;
    }
}

// Two consecutive values of h, summed over the splits in their order and scaled.
__device__ __forceinline__ float2 load_h(const Args& p, int m, int r, float scale)
{
    float2 s = make_float2(0.f, 0.f);
    if (m >= 0) {
        for (int q = 0; q < p.splits; ++q) {
            const float2 v = *reinterpret_cast<const float2*>(p.h + ((long long)q * p.rows + m) * p.rank8 + r);
            s.x += v.x, s.y += v.y;
        }
        s.x *= scale, s.y *= scale;
    }
    return s;
}

// One tile of 16 MT rows, 64 columns a warp: lane (g, t) loads eight consecutive columns 8 g .. of ranks 2t and 2t + 1, which are
// the elements of eight instructions, and ends up with the sixteen consecutive columns 16 t .. of rows g and g + 8.
template <class X, class W, int MT, bool VEC>
__global__ void __launch_bounds__(THREADS) up_kernel(const Args p)
{
    if (int(blockIdx.x) >= p.plan.head[0]) return;
    const int4 tile = p.plan.tiles[blockIdx.x];
    const bool none = tile.x >= p.count;
    if (none && p.base == p.out) return;   // in place: these rows are there already
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int n0 = (blockIdx.y * WARPS + warp) * 64;
    if (n0 >= p.width) return;
    int row[2 * MT];
#pragma unroll
    for (int i = 0; i < 2 * MT; ++i) row[i] = tile_row(p.plan, tile, 8 * i + g);
    float acc[MT][8][4] = {};
    if (!none) {
        const float scale = p.scale ? p.scale[tile.x] : 1.f;
        const W* w = static_cast<const W*>(p.w) + (long long)tile.x * p.rank * p.width + n0 + 8 * g;
        const int live = p.width - n0 - 8 * g;
#pragma unroll 2
        for (int r = 0; r < p.rank8; r += 8) {
            const int ra = r + 2 * t;
            float b0[8], b1[8];
            load<W, 8, VEC>(w + (long long)ra * p.width, ra < p.rank ? live : 0, b0);
            load<W, 8, VEC>(w + (long long)(ra + 1) * p.width, ra + 1 < p.rank ? live : 0, b1);
            unsigned ah[MT][4], al[MT][4];
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                const float2 u = load_h(p, row[2 * i], ra, scale), v = load_h(p, row[2 * i + 1], ra, scale);
                split(u.x, ah[i][0], al[i][0]);
                split(v.x, ah[i][1], al[i][1]);
                split(u.y, ah[i][2], al[i][2]);
                split(v.y, ah[i][3], al[i][3]);
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                unsigned h0, h1, l0, l1;
                split(b0[j], h0, l0);
                split(b1[j], h1, l1);
#pragma unroll
                for (int i = 0; i < MT; ++i) {
                    mma_tf32(acc[i][j], ah[i], h0, h1);
                    mma_tf32(acc[i][j], al[i], h0, h1);
                    if (is_f32<W>) mma_tf32(acc[i][j], ah[i], l0, l1);
                }
            }
        }
    }
    // column 8 c + j of the warp's 64 sits in element c of instruction j: c = 2t and 2t + 1 are this lane's
#pragma unroll
    for (int i = 0; i < 2 * MT; ++i) {
        if (row[i] < 0) continue;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const int n = n0 + 16 * t + 8 * c, live = p.width - n;
            float v[8];
            if (p.base) load<X, 8, VEC>(static_cast<const X*>(p.base) + row[i] * p.ldbase + n, live, v);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float d = acc[i >> 1][j][(i & 1) * 2 + c];
                v[j] = p.base ? v[j] + d : d;
            }
            store<X, 8, VEC>(static_cast<X*>(p.out) + row[i] * p.ldout + n, live, v);
        }
    }
}

// dw[a][r0 .. r0 + 16 RT)[n0 .. n0 + 8 NJ) over all rows of adapter a, which the warps share out: eight sorted rows an instruction.
template <class X, class W, int RT, int NJ, bool VEC>
__global__ void __launch_bounds__(THREADS) grad_kernel(const Args p)
{
    extern __shared__ float red[];   // [WARPS][16 RT][8 NJ]
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int a = blockIdx.y, n0 = blockIdx.x * 8 * NJ, r0 = blockIdx.z * 16 * RT;
    const int first = p.plan.offsets[a], last = p.plan.offsets[a + 1];
    const float scale = p.scale ? p.scale[a] : 1.f;
    const int n = n0 + NJ * g, live = p.width - n;
    float acc[RT][NJ][4] = {};
#pragma unroll 2
    for (int at = first + 8 * warp; at < last; at += 8 * WARPS) {
        int m[2];
        float b[2][NJ];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int pos = at + 2 * t + e;
            m[e] = pos < last ? p.plan.order[pos] : -1;
            load<X, NJ, VEC>(static_cast<const X*>(p.x) + (long long)max(m[e], 0) * p.ldx + n, m[e] >= 0 ? live : 0, b[e]);
        }
        unsigned ah[RT][4], al[RT][4];
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int r = r0 + 16 * i + g + 8 * (e & 1), row = m[e >> 1];
                float v = 0.f;
                if (row >= 0 && r < p.rank)
                    for (int q = 0; q < p.splits; ++q) v += p.h[((long long)q * p.rows + row) * p.rank8 + r];
                split(v * scale, ah[i][e], al[i][e]);
            }
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            unsigned h0, h1, l0, l1;
            split(b[0][j], h0, l0);
            split(b[1][j], h1, l1);
#pragma unroll
            for (int i = 0; i < RT; ++i) {
                mma_tf32(acc[i][j], ah[i], h0, h1);
                mma_tf32(acc[i][j], al[i], h0, h1);
                if (is_f32<X>) mma_tf32(acc[i][j], ah[i], l0, l1);
            }
        }
    }
    constexpr int ROWS = 16 * RT, COLS = 8 * NJ;
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                red[(warp * ROWS + 16 * i + g + (e & 2) * 4) * COLS + (2 * t + (e & 1)) * NJ + j] = acc[i][j][e];
    __syncthreads();
    for (int i = threadIdx.x * 8; i < ROWS * COLS; i += THREADS * 8) {
        const int r = r0 + i / COLS, at = n0 + i % COLS;
        if (r >= p.rank || at >= p.width) continue;
        float s[8] = {};
#pragma unroll
        for (int q = 0; q < WARPS; ++q)
#pragma unroll
            for (int e = 0; e < 8; ++e) s[e] += red[q * ROWS * COLS + i + e];
        store<W, 8, VEC>(static_cast<W*>(p.out) + ((long long)a * p.rank + r) * p.width + at, p.width - at, s);
    }
}

}  // namespace adapters
}  // namespace ds
