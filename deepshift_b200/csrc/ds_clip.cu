// Global 2-norm of many tensors and their scaling to a largest norm.
//
//   norm = sqrt(sum of all g^2),  f = min(1, max_norm / (norm + 1e-6)),  out = g * f
//
// Bound by memory: every gradient is read, read again and written.  Two launches for any number of tensors up to a table's
// size: the sums (one partial sum per CTA, in double), then the scaling, each of whose CTAs adds the partial sums up in the
// same order.  No counter, no atomic: the result depends on sizes and grid alone.  The scaling walks the chunks backwards,
// from those that the sums have just left in L2.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "ds_common.cuh"

namespace ds {
namespace {

constexpr int CLIP_THREADS = 256;
constexpr int CLIP_UNITS = 4;                                  // units of 8 elements a thread has in flight
constexpr int CLIP_CHUNK = CLIP_THREADS * CLIP_UNITS * 8;      // elements
constexpr int CLIP_CTAS = 148 * 6;                             // most CTAs, and partial sums, of a launch

// Tensors of one launch, passed by value: nothing to copy to the device, nothing that a captured graph could outlive.
template <int CAP>
struct ClipTable {
    const void* src[CAP];
    void* dst[CAP];
    long long n[CAP];
    int first[CAP + 1];      // first chunk of each tensor
    unsigned char kind[CAP]; // type of src, type of dst << 2, 16-byte aligned << 4
    int count;
};

__device__ __forceinline__ float2 unpack(unsigned v, int kind)
{
    if (kind == DS_T_BF16) return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xFFFF0000u));
    return __half22float2(*reinterpret_cast<const __half2*>(&v));
}

// Eight elements from element `at` of a tensor of n; those beyond n are 0.
__device__ __forceinline__ void load8(const void* p, int kind, bool vec, long long at, long long n, float (&v)[8])
{
    if (vec && at + 8 <= n) {
        if (kind == DS_T_F32) {
            const float4* q = reinterpret_cast<const float4*>(static_cast<const float*>(p) + at);
            const float4 a = q[0], b = q[1];
            v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
        } else {
            const uint4 a = *reinterpret_cast<const uint4*>(static_cast<const unsigned short*>(p) + at);
            const unsigned w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 f = unpack(w[i], kind);
                v[2 * i] = f.x, v[2 * i + 1] = f.y;
            }
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        v[i] = 0.f;
        if (at + i < n) {
            if (kind == DS_T_F32) v[i] = static_cast<const float*>(p)[at + i];
            else v[i] = unpack(static_cast<const unsigned short*>(p)[at + i], kind).x;
        }
    }
}

__device__ __forceinline__ unsigned short narrow(float f, int kind)
{
    return kind == DS_T_BF16 ? __bfloat16_as_ushort(__float2bfloat16_rn(f)) : __half_as_ushort(__float2half_rn(f));
}

__device__ __forceinline__ void store8(void* p, int kind, bool vec, long long at, long long n, const float (&v)[8])
{
    if (vec && at + 8 <= n) {
        if (kind == DS_T_F32) {
            float4* q = reinterpret_cast<float4*>(static_cast<float*>(p) + at);
            q[0] = make_float4(v[0], v[1], v[2], v[3]);
            q[1] = make_float4(v[4], v[5], v[6], v[7]);
        } else {
            unsigned w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = narrow(v[2 * i], kind) | unsigned(narrow(v[2 * i + 1], kind)) << 16;
            *reinterpret_cast<uint4*>(static_cast<unsigned short*>(p) + at) = make_uint4(w[0], w[1], w[2], w[3]);
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if (at + i < n) {
            if (kind == DS_T_F32) static_cast<float*>(p)[at + i] = v[i];
            else static_cast<unsigned short*>(p)[at + i] = narrow(v[i], kind);
        }
    }
}

template <int CAP>
__device__ __forceinline__ int tensor_of(const ClipTable<CAP>& t, int chunk)
{
    int lo = 0, hi = t.count;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (t.first[mid] <= chunk) lo = mid;
        else hi = mid;
    }
    return lo;
}

// Sum over the CTA in a fixed order, in every thread.
__device__ __forceinline__ double cta_sum(double v)
{
    __shared__ double part[CLIP_THREADS / 32];
#pragma unroll
    for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, d);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    double s = 0.0;
#pragma unroll
    for (int i = 0; i < CLIP_THREADS / 32; ++i) s += part[i];
    return s;
}

// Squares are added up in fp32 by eights, which rounds each sum by some 1e-7 of itself at random, and the sums in double.
// Eight whose sum leaves the range where fp32 can hold it (values beyond 1e18, or all so small that their squares vanish)
// are squared in double instead.
template <int CAP>
__global__ void __launch_bounds__(CLIP_THREADS) norm_kernel(const __grid_constant__ ClipTable<CAP> t, double* __restrict__ partial)
{
    double acc = 0.0;
    for (int chunk = blockIdx.x; chunk < t.first[t.count]; chunk += gridDim.x) {
        const int i = tensor_of(t, chunk);
        const int kind = t.kind[i] & 3;
        const bool vec = t.kind[i] & 16;
        const void* p = t.src[i];
        const long long n = t.n[i];
        const long long at = (long long)(chunk - t.first[i]) * CLIP_CHUNK + threadIdx.x * 8;
        float v[CLIP_UNITS][8];
#pragma unroll
        for (int u = 0; u < CLIP_UNITS; ++u) load8(p, kind, vec, at + u * (CLIP_THREADS * 8), n, v[u]);
#pragma unroll
        for (int u = 0; u < CLIP_UNITS; ++u) {
            float s = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) s = fmaf(v[u][e], v[u][e], s);
            if (s > 1e-30f && s < 1e37f) acc += s;
            else {
#pragma unroll
                for (int e = 0; e < 8; ++e) acc += double(v[u][e]) * v[u][e];
            }
        }
    }
    acc = cta_sum(acc);
    if (threadIdx.x == 0) partial[blockIdx.x] = acc;
}

__device__ __forceinline__ float total_norm(const double* __restrict__ partial, int partials)
{
    double s = 0.0;
    for (int i = threadIdx.x; i < partials; i += CLIP_THREADS) s += partial[i];
    return float(sqrt(cta_sum(s)));
}

template <int CAP>
__global__ void __launch_bounds__(CLIP_THREADS) scale_kernel(const __grid_constant__ ClipTable<CAP> t, const double* __restrict__ partial,
                                                             int partials, float max_norm, float* __restrict__ norm)
{
    const float all = total_norm(partial, partials);
    if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = all;
    float f = max_norm / (all + 1e-6f);
    if (f > 1.f) f = 1.f;   // NaN stays
    for (int c = blockIdx.x; c < t.first[t.count]; c += gridDim.x) {
        const int chunk = t.first[t.count] - 1 - c;
        const int i = tensor_of(t, chunk);
        if (f == 1.f && t.src[i] == t.dst[i]) continue;
        const bool vec = t.kind[i] & 16;
        const long long n = t.n[i];
        const long long at = (long long)(chunk - t.first[i]) * CLIP_CHUNK + threadIdx.x * 8;
        float v[CLIP_UNITS][8];
#pragma unroll
        for (int u = 0; u < CLIP_UNITS; ++u) load8(t.src[i], t.kind[i] & 3, vec, at + u * (CLIP_THREADS * 8), n, v[u]);
#pragma unroll
        for (int u = 0; u < CLIP_UNITS; ++u) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[u][e] *= f;
            store8(t.dst[i], t.kind[i] >> 2 & 3, vec, at + u * (CLIP_THREADS * 8), n, v[u]);
        }
    }
}

__global__ void __launch_bounds__(CLIP_THREADS) norm_only_kernel(const double* __restrict__ partial, int partials, float* __restrict__ norm)
{
    const float all = total_norm(partial, partials);
    if (threadIdx.x == 0) *norm = all;
}

// Fills a table from tensors[0 .. count) and returns its chunks.
template <int CAP>
int fill(ClipTable<CAP>& t, const ds_tensor_t* tensors, int count)
{
    t.count = 0;
    t.first[0] = 0;
    for (int i = 0; i < count; ++i) {
        const ds_tensor_t& a = tensors[i];
        if (a.n == 0) continue;
        const int k = t.count++;
        t.src[k] = a.src;
        t.dst[k] = a.dst;
        t.n[k] = a.n;
        const bool vec = ((reinterpret_cast<uintptr_t>(a.src) | reinterpret_cast<uintptr_t>(a.dst)) & 15) == 0;
        t.kind[k] = (unsigned char)(a.src_type | a.dst_type << 2 | (vec ? 16 : 0));
        t.first[k + 1] = t.first[k] + int((a.n + CLIP_CHUNK - 1) / CLIP_CHUNK);
    }
    return t.first[t.count];
}

int ctas(int chunks) { return chunks < CLIP_CTAS ? chunks : CLIP_CTAS; }

template <int CAP>
int run(const ds_tensor_t* tensors, int count, float max_norm, float* norm, double* partial, cudaStream_t st, bool scale)
{
    ClipTable<CAP> t;
    int partials = 0;
    for (int at = 0; at < count; at += CAP) {
        const int chunks = fill(t, tensors + at, count - at < CAP ? count - at : CAP);
        if (!chunks) continue;
        norm_kernel<CAP><<<ctas(chunks), CLIP_THREADS, 0, st>>>(t, partial + partials);
        note_launch();
        partials += ctas(chunks);
    }
    bool written = false;
    for (int at = 0; scale && at < count; at += CAP) {
        const int chunks = fill(t, tensors + at, count - at < CAP ? count - at : CAP);
        if (!chunks) continue;
        scale_kernel<CAP><<<ctas(chunks), CLIP_THREADS, 0, st>>>(t, partial, partials, max_norm, written ? nullptr : norm);
        note_launch();
        written = true;
    }
    if (!written) {
        norm_only_kernel<<<1, CLIP_THREADS, 0, st>>>(partial, partials, norm);
        note_launch();
    }
    return cudaGetLastError() == cudaSuccess ? DS_OK : DS_ERR_CUDA;
}

constexpr int CAP_FEW = 32, CAP_MANY = 512;

}  // namespace
}  // namespace ds

extern "C" long long ds_clip_bytes(int count)
{
    if (count < 0) return -1;
    const long long launches = count <= ds::CAP_FEW ? 1 : (count + ds::CAP_MANY - 1) / ds::CAP_MANY;
    return launches * ds::CLIP_CTAS * (long long)sizeof(double);
}

extern "C" int ds_clip_norm(const ds_tensor_t* tensors, int count, float max_norm, float* norm, void* scratch, long long scratch_bytes,
                            void* stream)
{
    if (count < 0 || (count && !tensors) || !norm || !scratch || !(max_norm >= 0.f)) return DS_ERR_BAD_ARG;
    if (scratch_bytes < ds_clip_bytes(count)) return DS_ERR_SCRATCH;
    if (reinterpret_cast<uintptr_t>(scratch) & 7) return DS_ERR_ALIGN;
    int with = 0, without = 0;   // tensors that have somewhere to go, and that have not: all or none
    long long chunks = 0;
    for (int i = 0; i < count; ++i) {
        const ds_tensor_t& a = tensors[i];
        if (a.n < 0 || (a.n && !a.src)) return DS_ERR_BAD_ARG;
        if (a.src_type < 0 || a.src_type > DS_T_F16 || a.dst_type < 0 || a.dst_type > DS_T_F16) return DS_ERR_UNSUPPORTED;
        if (a.n > 1ll << 42) return DS_ERR_RANGE;
        if (a.n) ++(a.dst ? with : without);
        chunks += (a.n + ds::CLIP_CHUNK - 1) / ds::CLIP_CHUNK;
    }
    if (with && without) return DS_ERR_BAD_ARG;
    if (chunks >= 1ll << 30) return DS_ERR_RANGE;   // chunks are counted in 32 bits
    const bool scale = with > 0;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    double* partial = static_cast<double*>(scratch);
    return count <= ds::CAP_FEW ? ds::run<ds::CAP_FEW>(tensors, count, max_norm, norm, partial, st, scale)
                                : ds::run<ds::CAP_MANY>(tensors, count, max_norm, norm, partial, st, scale);
}
