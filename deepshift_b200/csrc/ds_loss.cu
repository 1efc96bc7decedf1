// Softmax cross entropy of a linear head without its logits: the small kernels around the products, and the entry points (the
// tensor-core kernel is in ds_loss.cuh).
#include "ds_loss.cuh"

#include <climits>

namespace ds {
namespace loss {
namespace {

// ---- the small kernels ----

// Rows of an odd width, or at an address TMA cannot take, copied to rows of a multiple of 16 bytes, zeros behind them.
__global__ void __launch_bounds__(256) pad_kernel(const unsigned short* __restrict__ src, unsigned short* __restrict__ dst, long long rows, int d, int dp)
{
    const long long n = rows * dp;
    for (long long i = blockIdx.x * 256ll + threadIdx.x; i < n; i += gridDim.x * 256ll) {
        const long long r = i / dp;
        const int c = int(i - r * dp);
        dst[i] = c < d ? src[r * d + c] : (unsigned short)0;
    }
}

__device__ __forceinline__ bool counted(long long t, long long ignore) { return t != ignore; }

// loss and log-sum-exp of 32 rows (a lane's each); the warps share the tiles out.  The loss is log(sum) + (max - logit), so that a
// row that is sure of its target keeps the digits that lse - logit would lose.
__global__ void __launch_bounds__(256) rows_kernel(const float2* __restrict__ partial, int tiles, const float* __restrict__ at_target,
                                                   const long long* __restrict__ target, long long ignore, int rows, int vocabulary,
                                                   float* __restrict__ lse, float* __restrict__ each)
{
    __shared__ float2 part[8][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, row = blockIdx.x * 32 + lane;
    float top = -INFINITY, sum = 0.f;
    auto add = [&](float2 v) {
        const float next = fmaxf(top, v.x), from = next == -INFINITY ? 0.f : next;
        sum = sum * exp2_fast((top - from) * LOG2E) + v.y * exp2_fast((v.x - from) * LOG2E);
        top = next;
    };
    if (row < rows) {
#pragma unroll 4
        for (int t = warp; t < tiles; t += 8) add(partial[(long long)t * rows + row]);
    }
    part[warp][lane] = make_float2(top, sum);
    __syncthreads();
    if (warp || row >= rows) return;
    top = -INFINITY, sum = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) add(part[w][lane]);
    const float l = logf(sum);
    lse[row] = top + l;
    const long long t = target[row];
    if (!counted(t, ignore)) each[row] = 0.f;
    else if (t < 0 || t >= vocabulary) each[row] = __int_as_float(0x7FC00000);   // no such target: not a number
    else each[row] = l + (top - at_target[row]);
}

// Sum or mean of the rows' losses in double, in a fixed order, and the number of rows that count.
__global__ void __launch_bounds__(1024) reduce_kernel(const float* __restrict__ each, const long long* __restrict__ target, long long ignore, int rows,
                                                      int reduction, float* __restrict__ loss, float* __restrict__ count)
{
    __shared__ double sums[32];
    __shared__ int counts[32];
    double s = 0.0;
    int n = 0;
    for (int i = threadIdx.x; i < rows; i += 1024) {
        const bool c = counted(target[i], ignore);
        n += c;
        if (c) s += each[i];
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) {
        s += __shfl_xor_sync(0xFFFFFFFFu, s, d);
        n += __shfl_xor_sync(0xFFFFFFFFu, n, d);
    }
    if ((threadIdx.x & 31) == 0) sums[threadIdx.x >> 5] = s, counts[threadIdx.x >> 5] = n;
    __syncthreads();
    if (threadIdx.x) return;
    s = 0.0, n = 0;
    for (int i = 0; i < 32; ++i) s += sums[i], n += counts[i];
    *count = float(n);
    if (reduction == DS_LOSS_SUM) *loss = float(s);
    if (reduction == DS_LOSS_MEAN) *loss = float(s / n);   // no row counts: 0 / 0
}

// Weight of each row in G, at most `top` in magnitude so that 16 bits hold it (2^15 for fp16, whose small numbers run out at
// 2^-24: a probability of 10^-8 keeps eight digits' worth of bits), and the factor that takes it back.
__global__ void __launch_bounds__(1024) weights_kernel(const float* __restrict__ grad, const long long* __restrict__ target, long long ignore, int rows,
                                                       int vocabulary, int reduction, const float* __restrict__ count, float top,
                                                       float* __restrict__ weight, float* __restrict__ scale)
{
    __shared__ float most[32];
    float m = 0.f;
    if (reduction == DS_LOSS_NONE) {
        for (int i = threadIdx.x; i < rows; i += 1024)
            if (counted(target[i], ignore)) m = fmaxf(m, fabsf(grad[i]));
#pragma unroll
        for (int d = 16; d; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, d));
        if ((threadIdx.x & 31) == 0) most[threadIdx.x >> 5] = m;
        __syncthreads();
        m = 0.f;
        for (int i = 0; i < 32; ++i) m = fmaxf(m, most[i]);
        if (!(m > 0.f) || m > 3e38f) m = 1.f;
    } else {
        m = *grad;
        if (reduction == DS_LOSS_MEAN) m = *count > 0.f ? m / *count : 0.f;
    }
    for (int i = threadIdx.x; i < rows; i += 1024) {
        const long long t = target[i];
        if (!counted(t, ignore)) weight[i] = 0.f;
        else if (t < 0 || t >= vocabulary) weight[i] = __int_as_float(0x7FC00000);   // as its loss
        else weight[i] = reduction == DS_LOSS_NONE ? grad[i] / m * top : top;
    }
    if (threadIdx.x == 0) *scale = m / top;
}

// ---- launches ----
using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                              const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeFn encode_fn()
{
    static const EncodeFn fn = [] {
        void* ptr = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &found) == cudaSuccess && found == cudaDriverEntryPointSuccess)
            return reinterpret_cast<EncodeFn>(ptr);
        cudaGetLastError();
        return EncodeFn(nullptr);
    }();
    return fn;
}

// A matrix [rows][width] of 16-bit values, rows `stride` elements apart, in boxes of 64 elements x box_rows.
bool encode(CUtensorMap* map, const void* p, long long rows, int width, long long stride, int box_rows, bool is_bf16)
{
    const cuuint64_t dims[2] = {cuuint64_t(width), cuuint64_t(rows)}, strides[1] = {cuuint64_t(stride) * 2};
    const cuuint32_t box[2] = {64, cuuint32_t(box_rows)}, steps[2] = {1, 1};
    return encode_fn()(map, is_bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<void*>(p), dims, strides, box,
                       steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                       CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int multiprocessors()
{
    static int known[kMaxDevices];
    const int dev = device_slot();
    if (dev < 0) return 0;
    if (!known[dev] && cudaDeviceGetAttribute(&known[dev], cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
    return known[dev];
}

template <int PAIR, int MODE>
int launch(const CUtensorMap& a, const CUtensorMap& b, Params p, cudaStream_t st)
{
    static bool done[kMaxDevices];
    const int dev = device_slot(), sms = multiprocessors();
    p.err_flag = kernel_error_flag();
    if (dev < 0 || !sms || !p.err_flag) return DS_ERR_CUDA;
    if (!done[dev]) {
        if (cudaFuncSetAttribute(tile_kernel<PAIR, MODE>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES) != cudaSuccess) return DS_ERR_CUDA;
        done[dev] = true;
    }
    const long long tiles = (long long)p.tiles_m * p.tiles_n;
    if (tiles > INT_MAX) return DS_ERR_RANGE;
    const int most = sms / PAIR;
    p.group = 8;
    tile_kernel<PAIR, MODE><<<unsigned(tiles < most ? tiles : most) * PAIR, THREADS, SMEM_BYTES, st>>>(a, b, p);
    note_launch();
    return cudaGetLastError() == cudaSuccess ? DS_OK : DS_ERR_CUDA;
}

template <int MODE>
int launch(int pair, const CUtensorMap& a, const CUtensorMap& b, Params p, cudaStream_t st)
{
    p.tiles_m = (p.m_end + 128 * pair - 1) / (128 * pair);
    const int n = MODE == GRAD ? p.ldg : p.n_end;
    p.tiles_n = (n + 128 * pair - 1) / (128 * pair);
    return pair == 2 ? launch<2, MODE>(a, b, p, st) : launch<1, MODE>(a, b, p, st);
}

// ---- layout of a call's scratch ----
struct Layout {
    int dp;                 // width of a row of the operands that TMA reads
    long long h, w;         // copies of them, or -1
    long long partial, at_target;   // forward
    long long weight, scale, g, acc;  // backward
    int piece;              // columns of the vocabulary at a time
    long long bytes;
};

long long up256(long long n) { return (n + 255) / 256 * 256; }

// G takes 256 MB at most, unless 2048 columns of it take more: as few pieces as that allows, since each of them reads and writes the
// sums of dH.
int piece_of(long long rows, int v)
{
    const long long all = (v + 63ll) / 64 * 64;
    long long c = (128ll << 20) / (rows < 1 ? 1 : rows) / 256 * 256;
    if (c < 2048) c = 2048;
    return int(c < all ? c : all);
}

int pair_of(int rows) { return rows > 128 ? 2 : 1; }

Layout layout(int rows, int d, int v, bool backward, bool copies)
{
    Layout l = {};
    l.dp = (d + 7) / 8 * 8;
    long long at = 0;
    auto take = [&](long long n) {
        const long long here = at;
        at += up256(n);
        return here;
    };
    const bool copy = copies || d % 8;
    l.h = copy ? take((long long)rows * l.dp * 2) : -1;
    l.w = copy ? take((long long)v * l.dp * 2) : -1;
    if (!backward) {
        l.partial = take((v + 127ll) / 128 * rows * 8);
        l.at_target = take(rows * 4ll);
    } else {
        l.piece = piece_of(rows, v);
        l.weight = take(rows * 4ll);
        l.scale = take(4);
        l.g = take((long long)rows * l.piece * 2);
        l.acc = l.piece < v ? take((long long)rows * d * 4) : -1;
    }
    l.bytes = at;
    return l;
}

bool unaligned(const ds_loss_t* a) { return ((reinterpret_cast<uintptr_t>(a->hidden) | reinterpret_cast<uintptr_t>(a->weight)) & 15) != 0; }

int check(const ds_loss_t* a)
{
    if (!a || a->rows < 0 || a->d < 1 || a->v < 1) return DS_ERR_BAD_ARG;
    if (a->type != DS_T_BF16 && a->type != DS_T_F16) return DS_ERR_UNSUPPORTED;
    if (a->rows > 1 << 24 || a->d > 1 << 20 || a->v > 1 << 24) return DS_ERR_RANGE;
    if (a->reduction < DS_LOSS_NONE || a->reduction > DS_LOSS_SUM) return DS_ERR_BAD_ARG;
    if (!a->weight || (a->rows && (!a->hidden || !a->target || !a->lse))) return DS_ERR_BAD_ARG;
    if (a->reduction != DS_LOSS_NONE && !a->count) return DS_ERR_BAD_ARG;
    if (!encode_fn()) return DS_ERR_CUDA;
    return DS_OK;
}

int pad(const void* src, void* dst, long long rows, int d, int dp, cudaStream_t st)
{
    const long long blocks = (rows * dp + 255) / 256;
    pad_kernel<<<unsigned(blocks < 4096 ? blocks : 4096), 256, 0, st>>>(static_cast<const unsigned short*>(src), static_cast<unsigned short*>(dst), rows, d,
                                                                         dp);
    note_launch();
    return cudaGetLastError() == cudaSuccess ? DS_OK : DS_ERR_CUDA;
}

}  // namespace
}  // namespace loss
}  // namespace ds

extern "C" long long ds_loss_bytes(int rows, int d, int v, int backward, int copies)
{
    if (rows < 0 || d < 1 || v < 1 || rows > 1 << 24 || d > 1 << 20 || v > 1 << 24) return -1;
    return ds::loss::layout(rows, d, v, backward != 0, copies != 0).bytes;
}

extern "C" int ds_loss_forward(const ds_loss_t* a, void* stream)
{
    using namespace ds::loss;
    if (const int e = check(a)) return e;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (!a->each && a->rows) return DS_ERR_BAD_ARG;
    if (a->reduction != DS_LOSS_NONE && !a->loss) return DS_ERR_BAD_ARG;
    const Layout l = layout(a->rows, a->d, a->v, false, unaligned(a));
    if (a->scratch_bytes < l.bytes || (l.bytes && !a->scratch)) return DS_ERR_SCRATCH;
    if (reinterpret_cast<uintptr_t>(a->scratch) & 255) return DS_ERR_ALIGN;
    unsigned char* scratch = static_cast<unsigned char*>(a->scratch);
    if (a->rows) {
        const void *h = a->hidden, *w = a->weight;
        if (l.h >= 0) {
            if (const int e = pad(h, scratch + l.h, a->rows, a->d, l.dp, st)) return e;
            if (const int e = pad(w, scratch + l.w, a->v, a->d, l.dp, st)) return e;
            h = scratch + l.h, w = scratch + l.w;
        }
        CUtensorMap map_h, map_w;
        const bool bf = a->type == DS_T_BF16;
        if (!encode(&map_h, h, a->rows, l.dp, l.dp, CTA_ROWS, bf) || !encode(&map_w, w, a->v, l.dp, l.dp, CTA_ROWS, bf)) return DS_ERR_CUDA;
        Params p = {};
        p.k_steps = (l.dp + BK - 1) / BK, p.is_bf16 = bf;
        p.m_end = a->rows, p.n_end = a->v;
        p.target = reinterpret_cast<const long long*>(a->target);
        p.partial = reinterpret_cast<float2*>(scratch + l.partial);
        p.at_target = reinterpret_cast<float*>(scratch + l.at_target);
        const int pair = pair_of(a->rows);
        if (const int e = launch<STATS>(pair, map_h, map_w, p, st)) return e;
        rows_kernel<<<(a->rows + 31) / 32, 256, 0, st>>>(p.partial, (a->v + 128 * pair - 1) / (128 * pair), p.at_target, p.target, a->ignore_index, a->rows,
                                                         a->v, a->lse, a->each);
        ds::note_launch();
    }
    if (a->reduction != DS_LOSS_NONE) {
        reduce_kernel<<<1, 1024, 0, st>>>(a->each, reinterpret_cast<const long long*>(a->target), a->ignore_index, a->rows, a->reduction, a->loss, a->count);
        ds::note_launch();
    }
    return cudaGetLastError() == cudaSuccess ? DS_OK : DS_ERR_CUDA;
}

extern "C" int ds_loss_backward(const ds_loss_t* a, void* stream)
{
    using namespace ds::loss;
    if (const int e = check(a)) return e;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (!a->grad && a->rows) return DS_ERR_BAD_ARG;
    const Layout l = layout(a->rows, a->d, a->v, true, unaligned(a));
    if (a->scratch_bytes < l.bytes || (l.bytes && !a->scratch)) return DS_ERR_SCRATCH;
    if (reinterpret_cast<uintptr_t>(a->scratch) & 255) return DS_ERR_ALIGN;
    if ((reinterpret_cast<uintptr_t>(a->dhidden) | reinterpret_cast<uintptr_t>(a->dweight)) & 15) return DS_ERR_ALIGN;
    if (a->rows == 0) {
        if (a->dweight && cudaMemsetAsync(a->dweight, 0, (size_t)a->v * a->d * 2, st) != cudaSuccess) return DS_ERR_CUDA;
        return DS_OK;
    }
    unsigned char* scratch = static_cast<unsigned char*>(a->scratch);
    const void *h = a->hidden, *w = a->weight;
    if (l.h >= 0) {
        if (const int e = pad(h, scratch + l.h, a->rows, a->d, l.dp, st)) return e;
        if (const int e = pad(w, scratch + l.w, a->v, a->d, l.dp, st)) return e;
        h = scratch + l.h, w = scratch + l.w;
    }
    const bool bf = a->type == DS_T_BF16;
    float* weight = reinterpret_cast<float*>(scratch + l.weight);
    float* scale = reinterpret_cast<float*>(scratch + l.scale);
    weights_kernel<<<1, 1024, 0, st>>>(a->grad, reinterpret_cast<const long long*>(a->target), a->ignore_index, a->rows, a->v,
                                       a->reduction, a->count, bf ? 1.f : 32768.f, weight, scale);
    ds::note_launch();
    const int pair = pair_of(a->rows);
    CUtensorMap rows_h, cols_h;   // hidden with k along its rows, and with k across them
    if (!encode(&rows_h, h, a->rows, l.dp, l.dp, CTA_ROWS, bf) || !encode(&cols_h, h, a->rows, l.dp, l.dp, BK, bf)) return DS_ERR_CUDA;
    const unsigned short* w16 = static_cast<const unsigned short*>(w);
    for (int first = 0; first < a->v; first += l.piece) {
        const int cols = a->v - first < l.piece ? a->v - first : l.piece;
        const int ldg = (cols + 63) / 64 * 64;
        unsigned short* g = reinterpret_cast<unsigned short*>(scratch + l.g);
        CUtensorMap rows_w, cols_w, rows_g, cols_g;
        const void* wp = w16 + (long long)first * l.dp;
        if (!encode(&rows_w, wp, cols, l.dp, l.dp, CTA_ROWS, bf) || !encode(&cols_w, wp, cols, l.dp, l.dp, BK, bf) ||
            !encode(&rows_g, g, a->rows, ldg, ldg, CTA_ROWS, bf) || !encode(&cols_g, g, a->rows, ldg, ldg, BK, bf))
            return DS_ERR_CUDA;
        Params p = {};
        p.is_bf16 = bf;
        p.k_steps = (l.dp + BK - 1) / BK;
        p.m_end = a->rows, p.n_end = cols;
        p.target = reinterpret_cast<const long long*>(a->target);
        p.lse = a->lse, p.row_weight = weight, p.n_first = first;
        p.g = g, p.ldg = ldg;
        if (const int e = launch<GRAD>(pair, rows_h, rows_w, p, st)) return e;
        p.scale = scale;
        if (a->dhidden) {   // dH (+)= G W
            Params q = p;
            q.k_steps = ldg / BK, q.b_mn = 1;
            q.n_end = a->d;
            q.acc = l.acc < 0 ? nullptr : reinterpret_cast<float*>(scratch + l.acc);
            q.first = first == 0, q.last = first + cols == a->v;
            q.out = static_cast<unsigned short*>(a->dhidden);
            if (const int e = launch<PRODUCT>(pair, rows_g, cols_w, q, st)) return e;
        }
        if (a->dweight) {   // dW of the piece = G^T H
            Params q = p;
            q.k_steps = (a->rows + BK - 1) / BK, q.a_mn = q.b_mn = 1;
            q.m_end = cols, q.n_end = a->d;
            q.acc = nullptr, q.first = q.last = 1;
            q.out = static_cast<unsigned short*>(a->dweight) + (long long)first * a->d;
            if (const int e = launch<PRODUCT>(pair, cols_g, cols_h, q, st)) return e;
        }
    }
    return DS_OK;
}
