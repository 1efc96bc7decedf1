// Low-rank adapters, many rows: the three products on the tensor cores (tcgen05), tiles of 128 rows.
//
// The products are those of ds_adapters.cuh.  Operands are rows wherever they lie (a tile's rows are gathered), of fp32 or 16 bits, at any alignment:
// eight warps load them, cut every number into bf16 planes and write those to shared memory in the order that the tensor core
// reads (rows of 64 elements, 128-byte swizzle).  fp32 is three planes of eight bits each, exactly (x cut to its upper half, the rest cut again, and
// what is left), fp16 two, bf16 one; a product is the sum over pairs of planes whose numbers add up to at most two, which leaves out
// 2^-24 of it.  Which of an operand's dimensions lies along the rows is a matter of its descriptor alone.
//
// Bound by memory: activations pass once, the adapters' matrices come from L2.  With mma.sync, whose fp32 takes three TF32 products
// at an eighth of this rate, the three kernels took 36, 57 and 55 us where these take 19, 31 and 26 (4096 x 4096 -> 4096 in fp32, rank 32).
#pragma once
#include "ds_adapters.cuh"
#include "ds_tc_ptx.cuh"

namespace ds {
namespace adapters {

constexpr int TC_ROWS = 128, TC_RANKS = 64;                 // rows of a tile; ranks of a block: one row of 128 bytes
constexpr int TC_THREADS = THREADS + 32;                    // eight warps that load, convert and finish; one that multiplies
constexpr int A_PLANE = 128 * 128, B_PLANE = 64 * 128;      // 128 x 64 and 64 x 64 elements
constexpr unsigned TC_WAIT = 2000000000u;
template <class T> constexpr int PLANES = is_f32<T> ? 3 : __is_same(T, f16) ? 2 : 1;

struct TcShared {
    unsigned long long full[4], empty[4], acc_full[2], acc_empty[2], done;
    unsigned tmem;
    int err;
};

// Eight consecutive elements as they lie in memory.
template <class T>
struct Raw {
    uint4 q[sizeof(T) / 2];
};

template <class T, bool VEC>
__device__ __forceinline__ void load_raw(const T* p, int live, Raw<T>& r)
{
    constexpr int N = sizeof(T) / 2;
    if constexpr (VEC) {
#pragma unroll
        for (int i = 0; i < N; ++i) r.q[i] = live >= 8 ? reinterpret_cast<const uint4*>(p)[i] : make_uint4(0, 0, 0, 0);
    } else {
        unsigned w[4 * N] = {};
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < live) {
                if constexpr (is_f32<T>) w[i] = reinterpret_cast<const unsigned*>(p)[i];
                else w[i / 2] |= unsigned(reinterpret_cast<const unsigned short*>(p)[i]) << (16 * (i & 1));
            }
#pragma unroll
        for (int i = 0; i < N; ++i) r.q[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
    }
}

// v[8] cut into N planes of bf16.
template <int N>
__device__ __forceinline__ void cut(float (&v)[8], uint4 (&plane)[N])
{
#pragma unroll
    for (int k = 0; k < N; ++k) {
        unsigned w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const unsigned a = __float_as_uint(v[2 * i]), b = __float_as_uint(v[2 * i + 1]);
            w[i] = __byte_perm(a, b, 0x7632);
            if (k + 1 < N) {
                v[2 * i] -= __uint_as_float(a & 0xFFFF0000u);
                v[2 * i + 1] -= __uint_as_float(b & 0xFFFF0000u);
            }
        }
        plane[k] = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// The eight elements' planes to 16-byte piece `piece` of row `row` of a tile, whose planes lie `apart` bytes from one another.
template <class T>
__device__ __forceinline__ void put_planes(unsigned tile, int apart, int row, int piece, const Raw<T>& r)
{
    const unsigned at = tile + row * 128 + ((piece ^ (row & 7)) << 4);
    uint4 plane[PLANES<T>];
    if constexpr (PLANES<T> == 1) plane[0] = r.q[0];
    else {
        float v[8];
        widen_pieces<T>(r.q, v);
        cut(v, plane);
    }
#pragma unroll
    for (int k = 0; k < PLANES<T>; ++k)
        asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(at + k * apart), "r"(plane[k].x), "r"(plane[k].y), "r"(plane[k].z), "r"(plane[k].w)
                     : "memory");
}

// The same for eight values of h, scaled.
__device__ __forceinline__ void put_h8(unsigned tile, int apart, int row, int piece, const Raw<float>& r, float scale)
{
    Raw<float> s;
#pragma unroll
    for (int i = 0; i < 2; ++i)
        s.q[i] = make_uint4(__float_as_uint(__uint_as_float(r.q[i].x) * scale), __float_as_uint(__uint_as_float(r.q[i].y) * scale),
                            __float_as_uint(__uint_as_float(r.q[i].z) * scale), __float_as_uint(__uint_as_float(r.q[i].w) * scale));
    put_planes<float>(tile, apart, row, piece, s);
}

// What this warp has written to shared memory is there for the tensor core.
__device__ __forceinline__ void hand_over(unsigned long long* bar)
{
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
    if ((threadIdx.x & 31) == 0) bar_arrive(bar);
}

// Descriptor of a tile: its rows run along the summed index, or (mn) along the other one, whose blocks of 64 lie `lead` bytes apart.
__device__ __forceinline__ unsigned long long tile_descriptor(unsigned addr, bool mn, int lead)
{
    return (unsigned long long)((addr & 0x3FFFFu) >> 4) | (unsigned long long)(mn ? lead >> 4 : 1) << 16 | (unsigned long long)(1024 >> 4) << 32 | 1ull << 46 |
           2ull << 61;
}

__device__ __forceinline__ void mma_bf16(unsigned d, unsigned long long a, unsigned long long b, unsigned idesc, bool add)
{
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b),
                 "r"(idesc), "r"(unsigned(add))
                 : "memory");
}

// All pairs of planes of one step: PA planes of A `a_apart` bytes from one another, PB of B; `steps` times 16 of the summed index.
template <int PA, int PB>
__device__ __forceinline__ void mma_planes(unsigned d, unsigned a, int a_apart, bool a_mn, int a_lead, unsigned b, int b_apart, bool b_mn, int b_lead, int n,
                                           int steps, bool add)
{
    const unsigned idesc = 1u << 4 | 1u << 7 | 1u << 10 | unsigned(a_mn) << 15 | unsigned(b_mn) << 16 | unsigned(n / 8) << 17 | (128u / 16) << 24;
    const unsigned step_a = a_mn ? 2048 >> 4 : 32 >> 4, step_b = b_mn ? 2048 >> 4 : 32 >> 4;
#pragma unroll
    for (int i = PA - 1; i >= 0; --i)   // small terms first
#pragma unroll
        for (int j = PB - 1; j >= 0; --j) {
            if (i + j > 2) continue;
            const unsigned long long da = tile_descriptor(a + i * a_apart, a_mn, a_lead), db = tile_descriptor(b + j * b_apart, b_mn, b_lead);
            for (int k = 0; k < steps; ++k) {
                mma_bf16(d, da + k * step_a, db + k * step_b, idesc, add);
                add = true;
            }
        }
}

// Start and end of a kernel of this kind: barriers and tensor memory, and their return.
__device__ __forceinline__ void tc_begin(TcShared& s, int full_count, int acc_empty_count)
{
    if (threadIdx.x == 0) {
        s.err = 0;
        for (int i = 0; i < 4; ++i) {
            bar_init(&s.full[i], full_count);
            bar_init(&s.empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            bar_init(&s.acc_full[i], 1);
            bar_init(&s.acc_empty[i], acc_empty_count);
        }
        bar_init(&s.done, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (threadIdx.x >= THREADS) tmem_alloc(&s.tmem);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (threadIdx.x == 0 && s.tmem != 0) s.err = 1;   // all columns are this CTA's: their first is 0
}

// Behind the last use of tensor memory by any warp and a barrier.
__device__ __forceinline__ void tc_end(TcShared& s, int* err_flag)
{
    if (threadIdx.x == 0 && s.err) *err_flag = 1;
    if (threadIdx.x >= THREADS) tmem_dealloc();
}

__device__ __forceinline__ TcShared& tc_shared(unsigned char* raw, unsigned& tiles)
{
    tiles = (shared_address(raw) + 1024 + 1023) & ~1023u;   // behind the barriers
    return *reinterpret_cast<TcShared*>(raw);
}
constexpr int TC_EXTRA = 2048;   // of shared memory: the barriers, and up to the next multiple of 1024

// Stages of `bytes` each that fit an SM, four at most.
__host__ __device__ constexpr int tc_stages(int bytes) { return (225 * 1024 - TC_EXTRA) / bytes < 4 ? (225 * 1024 - TC_EXTRA) / bytes : 4; }

// ---- h = x down^T: 128 rows x up to 64 ranks, the summed index shared out among a cluster's CTAs (blockIdx.y) ----
template <class X, class W>
struct TcDown {
    static constexpr int STAGE = PLANES<X> * A_PLANE + PLANES<W> * B_PLANE, STAGES = tc_stages(STAGE);
    static constexpr int RED = 68;   // floats a row of the sums
    static constexpr int SMEM = STAGES * STAGE + TC_EXTRA;
};

template <class X, class W, bool VEC>
__global__ void __launch_bounds__(TC_THREADS, 1) tc_down_kernel(const Args p)
{
    using S = TcDown<X, W>;
    extern __shared__ __align__(16) unsigned char smem[];
    if (int(blockIdx.x) >= p.plan.head[0]) return;
    const int4 tile = p.plan.tiles[blockIdx.x];
    if (tile.x >= p.count) return;   // rows without an adapter: nothing reads their h
    unsigned tiles;
    TcShared& s = tc_shared(smem, tiles);
    volatile int* err = &s.err;
    tc_begin(s, WARPS, 1);
    const int t = threadIdx.x, shares = gridDim.y, r0 = blockIdx.z * TC_RANKS;
    const int ranks = min(TC_RANKS, p.rank8 - r0), n = (ranks + 15) / 16 * 16;
    const int chunks = (p.width + 63) / 64, first = int((long long)chunks * blockIdx.y / shares), last = int((long long)chunks * (blockIdx.y + 1) / shares);
    if (t < THREADS) {
        const int piece = t & 7, at = piece * 8;
        const X* xr[4];
        const W* wr[2];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int m = tile_row(p.plan, tile, (t >> 3) + 32 * i);
            xr[i] = m < 0 ? nullptr : static_cast<const X*>(p.x) + m * p.ldx + at;
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int r = r0 + (t >> 3) + 32 * i;
            wr[i] = r < p.rank ? static_cast<const W*>(p.w) + ((long long)tile.x * p.rank + r) * p.width + at : nullptr;
        }
        struct Step {
            Raw<X> a[4];
            Raw<W> b[2];
        } one, two;   // what is on its way for this step and the next
        auto fetch = [&](Step& q, int c) {
            const int live = c < last ? p.width - c * 64 - at : 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) load_raw<X, VEC>(xr[i] + c * 64, xr[i] ? live : 0, q.a[i]);
#pragma unroll
            for (int i = 0; i < 2; ++i) load_raw<W, VEC>(wr[i] + c * 64, wr[i] ? live : 0, q.b[i]);
        };
        int stage = 0;
        unsigned phase = 1;
        auto step = [&](Step& q, int c) {
            if (!__all_sync(0xFFFFFFFFu, bar_wait(&s.empty[stage], phase, err, TC_WAIT))) return false;
            const unsigned a = tiles + stage * S::STAGE, b = a + PLANES<X> * A_PLANE;
#pragma unroll
            for (int i = 0; i < 4; ++i) put_planes<X>(a, A_PLANE, (t >> 3) + 32 * i, piece, q.a[i]);
#pragma unroll
            for (int i = 0; i < 2; ++i)
                if ((t >> 3) + 32 * i < n) put_planes<W>(b, B_PLANE, (t >> 3) + 32 * i, piece, q.b[i]);
            hand_over(&s.full[stage]);
            fetch(q, c + 2);
            if (++stage == S::STAGES) stage = 0, phase ^= 1;
            return true;
        };
        fetch(one, first);
        fetch(two, first + 1);
        for (int c = first; c < last; c += 2) {
            if (!step(one, c)) break;
            if (c + 1 < last && !step(two, c + 1)) break;
        }
    } else if (elect_one()) {
        int stage = 0;
        unsigned phase = 0;
        for (int c = first; c < last; ++c) {
            if (!bar_wait(&s.full[stage], phase, err, TC_WAIT)) break;
            tc_fence_after();
            const unsigned a = tiles + stage * S::STAGE, b = a + PLANES<X> * A_PLANE;
            mma_planes<PLANES<X>, PLANES<W>>(0, a, A_PLANE, false, 0, b, B_PLANE, false, 0, n, 4, c > first);
            tc_commit(&s.empty[stage]);
            if (++stage == S::STAGES) stage = 0, phase ^= 1;
        }
        tc_commit(&s.done);
        if (!bar_drain(&s.done, 0)) *err = 1;
    }
    __syncthreads();
    tc_fence_after();
    float* red = reinterpret_cast<float*>(smem + (tiles - shared_address(smem)));   // [128][RED]
    if (t < 128) {
        for (int c = 0; c < n; c += 16) {
            int v[16];
            __syncwarp();
            tmem_ld((unsigned(t & 96) << 16) + c, v);
#pragma unroll
            for (int i = 0; i < 16; i += 4)
                *reinterpret_cast<float4*>(red + t * S::RED + c + i) =
                    first < last ? make_float4(__int_as_float(v[i]), __int_as_float(v[i + 1]), __int_as_float(v[i + 2]), __int_as_float(v[i + 3]))
                                 : make_float4(0.f, 0.f, 0.f, 0.f);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (shares > 1) cluster_sync();
    const int fours = ranks / 4;
    for (int i = blockIdx.y * TC_THREADS + t; i < TC_ROWS * fours; i += shares * TC_THREADS) {
        const int row = i / fours, r = i % fours * 4;
        const int m = tile_row(p.plan, tile, row);
        if (m < 0) continue;
        float v[4] = {};
        for (int q = 0; q < shares; ++q) {
            const float4 u = shares > 1 ? sums_of(red + row * S::RED + r, q) : *reinterpret_cast<const float4*>(red + row * S::RED + r);
            v[0] += u.x, v[1] += u.y, v[2] += u.z, v[3] += u.w;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (r0 + r + e >= p.rank) v[e] = 0.f;
        *reinterpret_cast<float4*>(p.h + (long long)m * p.rank8 + r0 + r) = make_float4(v[0], v[1], v[2], v[3]);
    }
    if (shares > 1) cluster_sync();   // nobody leaves while its sums are being read
    tc_fence_after();
    tc_end(s, p.err_flag);
}

// ---- dw[a] = sum over a's rows of s h^T x: 128 columns x up to 64 ranks, the rows shared out among a cluster's CTAs (blockIdx.z) ----
template <class X>
struct TcGrad {
    static constexpr int STAGE = PLANES<X> * A_PLANE + 3 * B_PLANE, STAGES = tc_stages(STAGE);
    static constexpr int RED = 132;
    static constexpr int SMEM = STAGES * STAGE + TC_EXTRA;
};

template <class X, class W, bool VEC>
__global__ void __launch_bounds__(TC_THREADS, 1) tc_grad_kernel(const Args p)
{
    using S = TcGrad<X>;
    extern __shared__ __align__(16) unsigned char smem[];
    unsigned tiles;
    TcShared& s = tc_shared(smem, tiles);
    volatile int* err = &s.err;
    tc_begin(s, WARPS, 1);
    const int t = threadIdx.x, shares = gridDim.z, share = blockIdx.z;
    const int blocks = (p.rank8 + TC_RANKS - 1) / TC_RANKS, a = blockIdx.x / blocks, r0 = blockIdx.x % blocks * TC_RANKS, n0 = blockIdx.y * 128;
    const int ranks = min(TC_RANKS, p.rank8 - r0), n = (ranks + 15) / 16 * 16;
    // whole steps of 64 rows for each CTA
    const int from = p.plan.offsets[a], all = p.plan.offsets[a + 1] - from, part = ((all + shares - 1) / shares + 63) / 64 * 64;
    const int begin = from + min(all, share * part), end = from + min(all, (share + 1) * part), count = (end - begin + 63) / 64;
    if (t < THREADS) {
        const float scale = p.scale ? p.scale[a] : 1.f;
        const int piece = t & 15, col = n0 + piece * 8, live = p.width - col, group = t & 7;
        const bool h_live = group * 8 < ranks, h_there = group * 8 < n;
        struct Step {
            Raw<X> x[4];
            Raw<float> h[2];
        } one, two;
        int mx[4], mh[2];   // rows of the step that is fetched next
        auto rows = [&](int c) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int at = begin + c * 64 + (t >> 4) + 16 * i;
                mx[i] = at < end ? p.plan.order[at] : -1;
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int at = begin + c * 64 + (t >> 3) + 32 * i;
                mh[i] = at < end && h_live ? p.plan.order[at] : -1;
            }
        };
        auto fetch = [&](Step& q) {
#pragma unroll
            for (int i = 0; i < 4; ++i) load_raw<X, VEC>(static_cast<const X*>(p.x) + (mx[i] >= 0 ? mx[i] * p.ldx + col : 0), mx[i] >= 0 ? live : 0, q.x[i]);
#pragma unroll
            for (int i = 0; i < 2; ++i)
                load_raw<float, true>(p.h + (mh[i] >= 0 ? (long long)mh[i] * p.rank8 + r0 + group * 8 : 0), mh[i] >= 0 ? 8 : 0, q.h[i]);
        };
        int stage = 0;
        unsigned phase = 1;
        auto step = [&](Step& q, int c) {
            if (!__all_sync(0xFFFFFFFFu, bar_wait(&s.empty[stage], phase, err, TC_WAIT))) return false;
            const unsigned x = tiles + stage * S::STAGE, h = x + PLANES<X> * A_PLANE;
#pragma unroll
            for (int i = 0; i < 4; ++i) put_planes<X>(x + (piece >> 3) * B_PLANE, A_PLANE, (t >> 4) + 16 * i, piece & 7, q.x[i]);
            if (h_there) {
#pragma unroll
                for (int i = 0; i < 2; ++i) put_h8(h, B_PLANE, (t >> 3) + 32 * i, group, q.h[i], scale);
            }
            hand_over(&s.full[stage]);
            fetch(q);
            rows(c + 3);
            if (++stage == S::STAGES) stage = 0, phase ^= 1;
            return true;
        };
        rows(0);
        fetch(one);
        rows(1);
        fetch(two);
        rows(2);
        for (int c = 0; c < count; c += 2) {
            if (!step(one, c)) break;
            if (c + 1 < count && !step(two, c + 1)) break;
        }
    } else if (elect_one()) {
        int stage = 0;
        unsigned phase = 0;
        for (int c = 0; c < count; ++c) {
            if (!bar_wait(&s.full[stage], phase, err, TC_WAIT)) break;
            tc_fence_after();
            const unsigned x = tiles + stage * S::STAGE, h = x + PLANES<X> * A_PLANE;
            mma_planes<PLANES<X>, 3>(0, x, A_PLANE, true, B_PLANE, h, B_PLANE, true, B_PLANE, n, 4, c > 0);
            tc_commit(&s.empty[stage]);
            if (++stage == S::STAGES) stage = 0, phase ^= 1;
        }
        tc_commit(&s.done);
        if (!bar_drain(&s.done, 0)) *err = 1;
    }
    __syncthreads();
    tc_fence_after();
    float* red = reinterpret_cast<float*>(smem + (tiles - shared_address(smem)));   // [ranks][RED]
    if (t < 128) {
        for (int c = 0; c < n; c += 16) {
            int v[16];
            __syncwarp();
            tmem_ld((unsigned(t & 96) << 16) + c, v);
#pragma unroll
            for (int i = 0; i < 16; ++i) red[(c + i) * S::RED + t] = count > 0 ? __int_as_float(v[i]) : 0.f;
        }
    }
    tc_fence_before();
    __syncthreads();
    if (shares > 1) cluster_sync();
    for (int i = share * TC_THREADS + t; i < ranks * 32; i += shares * TC_THREADS) {
        const int r = i / 32, col = i % 32 * 4, live = p.width - n0 - col;
        if (r0 + r >= p.rank || live <= 0) continue;
        float v[4] = {};
        for (int q = 0; q < shares; ++q) {
            const float4 u = shares > 1 ? sums_of(red + r * S::RED + col, q) : *reinterpret_cast<const float4*>(red + r * S::RED + col);
            v[0] += u.x, v[1] += u.y, v[2] += u.z, v[3] += u.w;
        }
        W* to = static_cast<W*>(p.out) + ((long long)a * p.rank + r0 + r) * p.width + n0 + col;
        if constexpr (VEC) {
            if constexpr (is_f32<W>) *reinterpret_cast<float4*>(to) = make_float4(v[0], v[1], v[2], v[3]);
            else *reinterpret_cast<uint2*>(to) = make_uint2(narrow<W>(v[0]) | unsigned(narrow<W>(v[1])) << 16, narrow<W>(v[2]) | unsigned(narrow<W>(v[3])) << 16);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (e < live) {
                    if constexpr (is_f32<W>) to[e] = v[e];
                    else reinterpret_cast<unsigned short*>(to)[e] = narrow<W>(v[e]);
                }
        }
    }
    if (shares > 1) cluster_sync();
    tc_fence_after();
    tc_end(s, p.err_flag);
}

// ---- out = base + s h up: 128 rows x 256 columns a tile, up to 64 ranks; a CTA takes a run of consecutive tiles ----
// The adapter's planes stay in shared memory until a tile of another one comes.  A tile's sums are in tensor memory, twice: while the warps add one
// tile's to base, the next tile's products run.  Lanes read sums by rows and base and out by columns, so each warp turns 32 x 32 of them in
// shared memory.
template <class X, class W>
struct TcUp {
    static constexpr int COLS = 256, H = 3 * A_PLANE, TURN = 32 * 36 * 4;
    __host__ __device__ static constexpr int plane(int n) { return 4 * n * 128; }   // of w: four blocks of 64 columns, n ranks
    static constexpr int smem(int n) { return H + PLANES<W> * plane(n) + WARPS * TURN + TC_EXTRA; }
};

// Elements of a row a lane deals with when 32 columns of 32 rows are read by columns, and the rows at a time.
template <class X>
struct Turn {
    static constexpr int EACH = 16 / sizeof(X), LANES = 32 / EACH, AT_ONCE = 32 / LANES, TIMES = 32 / AT_ONCE;
};

template <class X, class W, bool VEC>
__global__ void __launch_bounds__(TC_THREADS, 1) tc_up_kernel(const Args p)
{
    using S = TcUp<X, W>;
    using T = Turn<X>;
    extern __shared__ __align__(16) unsigned char smem[];
    const int total = p.plan.head[0], first = int((long long)total * blockIdx.x / gridDim.x), last = int((long long)total * (blockIdx.x + 1) / gridDim.x);
    if (first == last) return;
    unsigned tiles;
    TcShared& s = tc_shared(smem, tiles);
    volatile int* err = &s.err;
    tc_begin(s, WARPS, WARPS);
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5, n0 = blockIdx.y * S::COLS;
    const int k16 = (p.rank8 + 15) / 16 * 16;
    const unsigned h_at = tiles, w_at = tiles + S::H;
    auto tile_at = [&](int i) { return i < last ? p.plan.tiles[i] : make_int4(p.count, 0, 0, 0); };
    if (t < THREADS) {
        const int piece = t & 7, quarter = warp & 3, half = warp >> 2;
        Raw<float> h[4];
        float scale = 1.f;
        auto fetch_h = [&](const int4& tile) {
            scale = p.scale && tile.x < p.count ? p.scale[tile.x] : 1.f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int m = tile.x < p.count && piece * 8 < p.rank8 ? tile_row(p.plan, tile, (t >> 3) + 32 * i) : -1;
                load_raw<float, true>(p.h + (m >= 0 ? (long long)m * p.rank8 + piece * 8 : 0), m >= 0 ? 8 : 0, h[i]);
            }
        };
        int held = -1;
        auto give = [&](const int4& tile) {   // the tile's h, and its adapter's part of w if another's is there
            if (tile.x != held) {
                held = tile.x;
                const W* w = static_cast<const W*>(p.w) + (long long)tile.x * p.rank * p.width + n0;
#pragma unroll 2
                for (int i = t; i < k16 * 32; i += THREADS) {
                    const int r = i >> 5, c = i & 31;
                    Raw<W> q;
                    load_raw<W, VEC>(w + (long long)r * p.width + c * 8, r < p.rank ? p.width - n0 - c * 8 : 0, q);
                    put_planes<W>(w_at + (c >> 3) * k16 * 128, S::plane(k16), r, c & 7, q);
                }
            }
            if (piece * 8 < k16) {
#pragma unroll
                for (int i = 0; i < 4; ++i) put_h8(h_at, A_PLANE, (t >> 3) + 32 * i, piece, h[i], scale);
            }
            hand_over(&s.full[0]);
        };
        float* turn = reinterpret_cast<float*>(smem + (tiles - shared_address(smem)) + S::H + PLANES<W> * S::plane(k16)) + warp * (S::TURN / 4);
        const X* base = static_cast<const X*>(p.base);
        X* out = static_cast<X*>(p.out);
        int4 tile = tile_at(first);
        if (tile.x < p.count) {
            fetch_h(tile);
            give(tile);
        }
        unsigned phase = 0;
        for (int i = first, buf = 0; i < last; ++i) {
            const bool none = tile.x >= p.count;
            const int4 next = tile_at(i + 1);
            const int mine = tile_row(p.plan, tile, quarter * 32 + lane);   // a lane's row of the warp's 32
            fetch_h(next);
            const int c0 = n0 + half * 128;
            // base of 32 columns: of row AT_ONCE k + lane / LANES, EACH elements; or, without alignment, of column `lane` of every row
            uint4 q[T::TIMES];
            auto fetch_base = [&](int c) {
                if constexpr (VEC) {
#pragma unroll
                    for (int k = 0; k < T::TIMES; ++k) {
                        const int m = __shfl_sync(0xFFFFFFFFu, mine, T::AT_ONCE * k + lane / T::LANES), n = c + lane % T::LANES * T::EACH;
                        q[k] = base && m >= 0 && n < p.width ? *reinterpret_cast<const uint4*>(base + m * p.ldbase + n) : make_uint4(0, 0, 0, 0);
                    }
                }
            };
            fetch_base(c0);
            if (!none) {
                if (!__all_sync(0xFFFFFFFFu, bar_wait(&s.acc_full[buf], phase, err, TC_WAIT))) break;
                tc_fence_after();
            }
            if (next.x < p.count) give(next);   // the products that read the previous tile's operands are done
            if (!(none && p.base == p.out)) {
                for (int c = 0; c < 128; c += 32) {
                    const int at = c0 + c;
                    if (at >= p.width) break;
                    __syncwarp();
                    if (!none) {
                        int v[32];
                        tmem_ld((unsigned(quarter * 32) << 16) + buf * 256 + half * 128 + c, v);
#pragma unroll
                        for (int e = 0; e < 32; e += 4)
                            *reinterpret_cast<float4*>(turn + lane * 36 + e) =
                                make_float4(__int_as_float(v[e]), __int_as_float(v[e + 1]), __int_as_float(v[e + 2]), __int_as_float(v[e + 3]));
                    } else {
#pragma unroll
                        for (int e = 0; e < 32; e += 4) *reinterpret_cast<float4*>(turn + lane * 36 + e) = make_float4(0.f, 0.f, 0.f, 0.f);
                    }
                    __syncwarp();
                    if constexpr (VEC) {
                        uint4 now[T::TIMES];
#pragma unroll
                        for (int k = 0; k < T::TIMES; ++k) now[k] = q[k];
                        if (c + 32 < 128) fetch_base(at + 32);
#pragma unroll
                        for (int k = 0; k < T::TIMES; ++k) {
                            const int row = T::AT_ONCE * k + lane / T::LANES, col = lane % T::LANES * T::EACH;
                            const int m = __shfl_sync(0xFFFFFFFFu, mine, row);
                            const uint4 one[1] = {now[k]};
                            float b[T::EACH];
                            widen_pieces<X>(one, b);
                            unsigned w[4];
#pragma unroll
                            for (int e = 0; e < T::EACH; e += 4) {
                                const float4 d = *reinterpret_cast<const float4*>(turn + row * 36 + col + e);
                                b[e] += d.x, b[e + 1] += d.y, b[e + 2] += d.z, b[e + 3] += d.w;
                            }
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                if constexpr (is_f32<X>) w[e] = __float_as_uint(b[e]);
                                else w[e] = narrow<X>(b[2 * e]) | unsigned(narrow<X>(b[2 * e + 1])) << 16;
                            }
                            if (m >= 0 && at + col < p.width) *reinterpret_cast<uint4*>(out + m * p.ldout + at + col) = make_uint4(w[0], w[1], w[2], w[3]);
                        }
                    } else {
                        const int n = at + lane;
#pragma unroll
                        for (int r0 = 0; r0 < 32; r0 += 8) {
                            float b[8];
#pragma unroll
                            for (int r = 0; r < 8; ++r) {
                                const int m = __shfl_sync(0xFFFFFFFFu, mine, r0 + r);
                                b[r] = base && m >= 0 && n < p.width ? one(base + m * p.ldbase + n) : 0.f;
                            }
#pragma unroll
                            for (int r = 0; r < 8; ++r) {
                                const int m = __shfl_sync(0xFFFFFFFFu, mine, r0 + r);
                                if (m < 0 || n >= p.width) continue;
                                const float y = b[r] + turn[(r0 + r) * 36 + lane];
                                if constexpr (is_f32<X>) out[m * p.ldout + n] = y;
                                else reinterpret_cast<unsigned short*>(out)[m * p.ldout + n] = narrow<X>(y);
                            }
                        }
                    }
                }
            }
            if (!none) {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) bar_arrive(&s.acc_empty[buf]);
                if (buf ^= 1; buf == 0) phase ^= 1;
            }
            tile = next;
        }
    } else if (elect_one()) {
        unsigned h_phase = 0, phase = 1;
        for (int i = first, buf = 0; i < last; ++i) {
            if (p.plan.tiles[i].x >= p.count) break;   // rows without an adapter come last
            if (!bar_wait(&s.full[0], h_phase, err, TC_WAIT) || !bar_wait(&s.acc_empty[buf], phase, err, TC_WAIT)) break;
            tc_fence_after();
            mma_planes<3, PLANES<W>>(buf * 256, h_at, A_PLANE, false, 0, w_at, S::plane(k16), true, k16 * 128, S::COLS, k16 / 16, false);
            tc_commit(&s.acc_full[buf]);
            h_phase ^= 1;
            if (buf ^= 1; buf == 0) phase ^= 1;
        }
        tc_commit(&s.done);
        if (!bar_drain(&s.done, 0)) *err = 1;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    tc_end(s, p.err_flag);
}

}  // namespace adapters
}  // namespace ds
