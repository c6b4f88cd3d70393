// Root-mean-square norm over the channels of a row, with the residual's addition in front and, if asked, 8-bit output
// with scales behind; and its gradient.
//
//   h = round(x + residual),  rstd = (mean(h^2) + eps)^-1/2,  y = h * rstd * weight
//   u = dy * weight:  dx = rstd * (u - h * rstd^2 * mean(u * h)) + dresidual,  dweight = sum over rows of dy * h * rstd
//
// Both are bound by memory: the forward pass reads x and the residual once and writes h and y (or its codes) once, the
// backward pass reads dy, h and what reaches h past the norm once and writes dx once.  A row therefore stays in
// registers between its reduction and its stores: tpr threads hold NV vectors of VEC elements each.  The norm is taken
// of the sum as it is stored, rounded to the tensor's type, because that is what the backward pass and the next layer
// read.
#include <algorithm>

#include "pxe_types.cuh"

namespace pxe {
namespace {

constexpr int kMaxChannels = 262144;
constexpr int kMaxPartials = 592;          // rows of the weight gradient's workspace: 4 for each of 148 SMs

struct NormParams {
    const void* x;
    const void* residual;
    const void* weight;
    void* h;
    void* y;
    uint8_t* q;
    float* scale;
    float* rstd;
    long long xs, rs, hs, ys, qs, rows;
    int channels, weight_f32, group, groups;
    float eps, inv_channels;
};

struct NormBackParams {
    const void* dy;
    const void* h;
    const void* dres;
    const void* weight;
    const float* rstd;
    void* dx;
    float* partial;
    long long dys, hs, rs, dxs, rows;
    int channels, weight_f32;
    float inv_channels;
};

__device__ __forceinline__ float warp_sum(float v)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Sum (or NaN-keeping maximum) over the blockDim.x threads of one row; `red` holds 32 floats for each row of the block.
// Every thread of the block calls it.
template <bool MAX>
__device__ __forceinline__ float row_reduce(float v, float* red)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float t = __shfl_xor_sync(0xffffffffu, v, o);
        v = MAX ? max_nan(v, t) : v + t;
    }
    if (blockDim.x == 32) return v;
    const int warps = blockDim.x >> 5;
    __syncthreads();                                       // the previous use of red is over
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    float t = (threadIdx.x & 31) < warps ? red[threadIdx.x & 31] : 0.0f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float u = __shfl_xor_sync(0xffffffffu, t, o);
        t = MAX ? max_nan(t, u) : t + u;
    }
    return t;
}

template <typename T, int VEC>
__device__ __forceinline__ void load_weight(const void* weight, int weight_f32, int col, float (&w)[VEC])
{
    if (weight == nullptr) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) w[j] = 1.0f;
    } else if (weight_f32) {
        const float* p = static_cast<const float*>(weight) + col;
        if constexpr (VEC == 8) {
            float a[4], b[4];
            unpack<float, 4>(gldv<uint4>(p), a);
            unpack<float, 4>(gldv<uint4>(p + 4), b);
#pragma unroll
            for (int j = 0; j < 4; ++j) { w[j] = a[j]; w[4 + j] = b[j]; }
        } else {
            unpack<float, VEC>(gldv<Raw<float, VEC>>(p), w);
        }
    } else {
        unpack<T, VEC>(gldv<Raw<T, VEC>>(static_cast<const T*>(weight) + col), w);
    }
}

__device__ __forceinline__ float scale_of(float largest) { return max_nan(largest / kE4m3Max, kScaleMin); }

// ---------------------------------------------------------------- forward, row in registers
// blockDim = (tpr, rows per block).  Weights stay in registers over the block's rows while they fit.
template <typename T, int VEC, int NV, bool Q>
__global__ void __launch_bounds__(NV <= 2 ? 1024 : 512)
rms_norm_kernel(const NormParams p)
{
    constexpr bool KEEP = NV * VEC <= 16;
    __shared__ float reds[32 * 8];
    extern __shared__ unsigned int group_max[];            // Q, groups that no set of lanes of one warp covers: [rpb][groups]
    float* red = reds + threadIdx.y * 32;
    const int tpr = blockDim.x, rpb = blockDim.y, C = p.channels;
    float w[KEEP ? NV : 1][VEC];
    if constexpr (KEEP) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int col = (i * tpr + threadIdx.x) * VEC;
            if (col < C) load_weight<T, VEC>(p.weight, p.weight_f32, col, w[i]);
        }
    }
    for (long long row0 = (long long)blockIdx.x * rpb; row0 < p.rows; row0 += (long long)gridDim.x * rpb) {
        const long long row = row0 + threadIdx.y;
        const bool active = row < p.rows;
        const T* x = static_cast<const T*>(p.x) + row * p.xs;
        const T* r = static_cast<const T*>(p.residual) + row * p.rs;
        float v[NV][VEC];
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int col = (i * tpr + threadIdx.x) * VEC;
#pragma unroll
            for (int j = 0; j < VEC; ++j) v[i][j] = 0.0f;
            if (active && col < C) unpack<T, VEC>(gldv<Raw<T, VEC>>(x + col), v[i]);
        }
        if (p.residual) {
            T* h = static_cast<T*>(p.h) + row * p.hs;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int col = (i * tpr + threadIdx.x) * VEC;
                if (active && col < C) {
                    float a[VEC];
                    unpack<T, VEC>(gldv<Raw<T, VEC>>(r + col), a);
#pragma unroll
                    for (int j = 0; j < VEC; ++j) a[j] += v[i][j];
                    const Raw<T, VEC> raw = pack<T, VEC>(a);
                    gstv(h + col, raw);
                    unpack<T, VEC>(raw, v[i]);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < VEC; ++j) sum = fmaf(v[i][j], v[i][j], sum);
        sum = row_reduce<false>(sum, red);
        const float rstd = rsqrtf(sum * p.inv_channels + p.eps);
        if (p.rstd && active && threadIdx.x == 0) gst(p.rstd + row, rstd);
        float largest = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int col = (i * tpr + threadIdx.x) * VEC;
            if constexpr (!KEEP) {
                if (col < C) load_weight<T, VEC>(p.weight, p.weight_f32, col, w[0]);
            }
            if (col < C) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    v[i][j] = v[i][j] * rstd * w[KEEP ? i : 0][j];
                    if constexpr (Q) largest = max_nan(largest, fabsf(v[i][j]));
                }
            }
            if constexpr (!Q) {
                if (active && col < C) gstv(static_cast<T*>(p.y) + row * p.ys + col, pack<T, VEC>(v[i]));
            }
        }
        if constexpr (Q) {
            uint8_t* q = p.q + row * p.qs;
            auto store = [&](int i, int col, float scale) {
                const float inv = 1.0f / scale;
                float a[VEC];
#pragma unroll
                for (int j = 0; j < VEC; ++j) a[j] = v[i][j] * inv;
                gstv(q + col, pack_e4m3<VEC>(a));
            };
            if (p.group == 0) {
                const float scale = scale_of(row_reduce<true>(largest, red));
                if (active && threadIdx.x == 0) gst(p.scale + row, scale);
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    const int col = (i * tpr + threadIdx.x) * VEC;
                    if (active && col < C) store(i, col, scale);
                }
            } else if (p.group <= 32 * VEC) {              // a group is group / VEC neighbouring lanes of one warp
                const int lanes = p.group / VEC;
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    const int col = (i * tpr + threadIdx.x) * VEC;
                    float m = 0.0f;
                    if (col < C) {
#pragma unroll
                        for (int j = 0; j < VEC; ++j) m = max_nan(m, fabsf(v[i][j]));
                    }
                    for (int o = lanes >> 1; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
                    if (active && col < C) {
                        const float scale = scale_of(m);
                        if (col % p.group == 0) gst(p.scale + row * p.groups + col / p.group, scale);
                        store(i, col, scale);
                    }
                }
            } else {                                       // fp32 bits of |y| order as integers do, NaN above everything
                unsigned int* gm = group_max + threadIdx.y * p.groups;
                __syncthreads();
                for (int g = threadIdx.x; g < p.groups; g += tpr) gm[g] = 0u;
                __syncthreads();
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    const int col = (i * tpr + threadIdx.x) * VEC;
                    if (col < C) {
                        float m = 0.0f;
#pragma unroll
                        for (int j = 0; j < VEC; ++j) m = max_nan(m, fabsf(v[i][j]));
                        atomicMax(gm + col / p.group, __float_as_uint(m));
                    }
                }
                __syncthreads();
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    const int col = (i * tpr + threadIdx.x) * VEC;
                    if (active && col < C) {
                        const float scale = scale_of(__uint_as_float(gm[col / p.group]));
                        if (col % p.group == 0) gst(p.scale + row * p.groups + col / p.group, scale);
                        store(i, col, scale);
                    }
                }
            }
        }
    }
}

// ---------------------------------------------------------------- forward, any row length
// A block of 1024 threads per row; the row is read again (from L2 or from h) for its output.
template <typename T, int VEC, bool Q>
__global__ void __launch_bounds__(1024)
rms_norm_long_kernel(const NormParams p)
{
    __shared__ float red[32];
    extern __shared__ unsigned int group_max[];
    const int C = p.channels, step = blockDim.x * VEC, first = threadIdx.x * VEC;
    for (long long row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const T* x = static_cast<const T*>(p.x) + row * p.xs;
        const T* r = static_cast<const T*>(p.residual) + row * p.rs;
        T* h = static_cast<T*>(p.h) + row * p.hs;
        const T* again = p.residual ? h : x;
        float sum = 0.0f, v[VEC], w[VEC];
        for (int col = first; col < C; col += step) {
            unpack<T, VEC>(gldv<Raw<T, VEC>>(x + col), v);
            if (p.residual) {
                float a[VEC];
                unpack<T, VEC>(gldv<Raw<T, VEC>>(r + col), a);
#pragma unroll
                for (int j = 0; j < VEC; ++j) a[j] += v[j];
                const Raw<T, VEC> raw = pack<T, VEC>(a);
                gstv(h + col, raw);
                unpack<T, VEC>(raw, v);
            }
#pragma unroll
            for (int j = 0; j < VEC; ++j) sum = fmaf(v[j], v[j], sum);
        }
        sum = row_reduce<false>(sum, red);
        const float rstd = rsqrtf(sum * p.inv_channels + p.eps);
        if (p.rstd && threadIdx.x == 0) gst(p.rstd + row, rstd);
        auto value = [&](int col) {
            unpack<T, VEC>(gldv<Raw<T, VEC>>(again + col), v);
            load_weight<T, VEC>(p.weight, p.weight_f32, col, w);
#pragma unroll
            for (int j = 0; j < VEC; ++j) v[j] = v[j] * rstd * w[j];
        };
        if constexpr (!Q) {
            for (int col = first; col < C; col += step) {
                value(col);
                gstv(static_cast<T*>(p.y) + row * p.ys + col, pack<T, VEC>(v));
            }
        } else {
            const int group = p.group ? p.group : C;
            __syncthreads();
            for (int g = threadIdx.x; g < p.groups; g += blockDim.x) group_max[g] = 0u;
            __syncthreads();
            float largest = 0.0f;
            for (int col = first; col < C; col += step) {
                value(col);
                float m = 0.0f;
#pragma unroll
                for (int j = 0; j < VEC; ++j) m = max_nan(m, fabsf(v[j]));
                if (p.group) atomicMax(group_max + col / group, __float_as_uint(m));
                else largest = max_nan(largest, m);
            }
            if (!p.group) {
                largest = row_reduce<true>(largest, red);
                if (threadIdx.x == 0) group_max[0] = __float_as_uint(largest);
            }
            __syncthreads();
            for (int col = first; col < C; col += step) {
                value(col);
                const float scale = scale_of(__uint_as_float(group_max[col / group]));
                if (col % group == 0) gst(p.scale + row * p.groups + col / group, scale);
                const float inv = 1.0f / scale;
#pragma unroll
                for (int j = 0; j < VEC; ++j) v[j] *= inv;
                gstv(p.q + row * p.qs + col, pack_e4m3<VEC>(v));
            }
            __syncthreads();
        }
    }
}

// ---------------------------------------------------------------- backward, row in registers
template <typename T, int VEC, int NV>
__global__ void __launch_bounds__(NV * VEC <= 8 ? 1024 : NV * VEC <= 16 ? 512 : 256)
rms_norm_backward_kernel(const NormBackParams p)
{
    __shared__ float reds[32 * 8];
    extern __shared__ float shared_dw[];                   // rows per block > 1: [channels]
    float* red = reds + threadIdx.y * 32;
    const int tpr = blockDim.x, rpb = blockDim.y, C = p.channels;
    float acc[NV][VEC];
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < VEC; ++j) acc[i][j] = 0.0f;
    for (long long row0 = (long long)blockIdx.x * rpb; row0 < p.rows; row0 += (long long)gridDim.x * rpb) {
        const long long row = row0 + threadIdx.y;
        const bool active = row < p.rows;
        const T* dy = static_cast<const T*>(p.dy) + row * p.dys;
        const T* h = static_cast<const T*>(p.h) + row * p.hs;
        Raw<T, VEC> dyr[NV], hr[NV];
        float dot = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int col = (i * tpr + threadIdx.x) * VEC;
            dyr[i] = Raw<T, VEC>{};
            hr[i] = Raw<T, VEC>{};
            if (active && col < C) {
                dyr[i] = gldv<Raw<T, VEC>>(dy + col);
                hr[i] = gldv<Raw<T, VEC>>(h + col);
            }
        }
        const float rstd = active ? gld(p.rstd + row) : 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int col = (i * tpr + threadIdx.x) * VEC;
            if (col < C) {
                float a[VEC], b[VEC], w[VEC];
                unpack<T, VEC>(dyr[i], a);
                unpack<T, VEC>(hr[i], b);
                load_weight<T, VEC>(p.weight, p.weight_f32, col, w);
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    dot = fmaf(a[j] * w[j], b[j], dot);
                    acc[i][j] = fmaf(a[j], b[j] * rstd, acc[i][j]);
                }
            }
        }
        dot = row_reduce<false>(dot, red);
        const float k = dot * p.inv_channels * rstd * rstd;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int col = (i * tpr + threadIdx.x) * VEC;
            if (active && col < C) {
                float a[VEC], b[VEC], w[VEC];
                unpack<T, VEC>(dyr[i], a);
                unpack<T, VEC>(hr[i], b);
                load_weight<T, VEC>(p.weight, p.weight_f32, col, w);
#pragma unroll
                for (int j = 0; j < VEC; ++j) a[j] = rstd * (a[j] * w[j] - b[j] * k);
                if (p.dres) {
                    unpack<T, VEC>(gldv<Raw<T, VEC>>(static_cast<const T*>(p.dres) + row * p.rs + col), b);
#pragma unroll
                    for (int j = 0; j < VEC; ++j) a[j] += b[j];
                }
                gstv(static_cast<T*>(p.dx) + row * p.dxs + col, pack<T, VEC>(a));
            }
        }
    }
    if (p.partial == nullptr) return;
    float* out = p.partial + (long long)blockIdx.x * C;
    if (rpb == 1) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int col = (i * tpr + threadIdx.x) * VEC;
#pragma unroll
            for (int j = 0; j < VEC; ++j)
                if (col + j < C) gst(out + col + j, acc[i][j]);
        }
        return;
    }
    for (int y = 0; y < rpb; ++y) {                        // the block's rows one after the other: a fixed order
        if ((int)threadIdx.y == y) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int col = (i * tpr + threadIdx.x) * VEC;
#pragma unroll
                for (int j = 0; j < VEC; ++j)
                    if (col + j < C) shared_dw[col + j] = y == 0 ? acc[i][j] : shared_dw[col + j] + acc[i][j];
            }
        }
        __syncthreads();
    }
    for (int c = threadIdx.y * tpr + threadIdx.x; c < C; c += tpr * rpb) gst(out + c, shared_dw[c]);
}

// Any row length: the row is read twice, the block's part of the weight gradient lives in its row of the workspace.
template <typename T, int VEC>
__global__ void __launch_bounds__(1024)
rms_norm_backward_long_kernel(const NormBackParams p)
{
    __shared__ float red[32];
    const int C = p.channels, step = blockDim.x * VEC, first = threadIdx.x * VEC;
    float* out = p.partial ? p.partial + (long long)blockIdx.x * C : nullptr;
    for (long long row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const T* dy = static_cast<const T*>(p.dy) + row * p.dys;
        const T* h = static_cast<const T*>(p.h) + row * p.hs;
        const float rstd = gld(p.rstd + row);
        float a[VEC], b[VEC], w[VEC], dot = 0.0f;
        for (int col = first; col < C; col += step) {
            unpack<T, VEC>(gldv<Raw<T, VEC>>(dy + col), a);
            unpack<T, VEC>(gldv<Raw<T, VEC>>(h + col), b);
            load_weight<T, VEC>(p.weight, p.weight_f32, col, w);
#pragma unroll
            for (int j = 0; j < VEC; ++j) dot = fmaf(a[j] * w[j], b[j], dot);
        }
        dot = row_reduce<false>(dot, red);
        const float k = dot * p.inv_channels * rstd * rstd;
        for (int col = first; col < C; col += step) {
            unpack<T, VEC>(gldv<Raw<T, VEC>>(dy + col), a);
            unpack<T, VEC>(gldv<Raw<T, VEC>>(h + col), b);
            load_weight<T, VEC>(p.weight, p.weight_f32, col, w);
            if (out) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    const float t = a[j] * (b[j] * rstd);
                    gst(out + col + j, row == blockIdx.x ? t : gld(out + col + j) + t);
                }
            }
#pragma unroll
            for (int j = 0; j < VEC; ++j) a[j] = rstd * (a[j] * w[j] - b[j] * k);
            if (p.dres) {
                unpack<T, VEC>(gldv<Raw<T, VEC>>(static_cast<const T*>(p.dres) + row * p.rs + col), b);
#pragma unroll
                for (int j = 0; j < VEC; ++j) a[j] += b[j];
            }
            gstv(static_cast<T*>(p.dx) + row * p.dxs + col, pack<T, VEC>(a));
        }
    }
}

// dweight[c] = the sum of column c over the workspace's rows: 32 columns by 16 row groups to a block, each group's rows
// and then the groups in order.
__global__ void __launch_bounds__(512)
rms_norm_dweight_kernel(const float* partial, int parts, int channels, float* dweight, int accumulate)
{
    __shared__ float part[16][33];
    const int c = blockIdx.x * 32 + threadIdx.x;
    float sum = 0.0f;
    if (c < channels)
        for (int r = threadIdx.y; r < parts; r += 16) sum += gld(partial + (long long)r * channels + c);
    part[threadIdx.y][threadIdx.x] = sum;
    __syncthreads();
    if (threadIdx.y == 0 && c < channels) {
#pragma unroll
        for (int y = 1; y < 16; ++y) sum += part[y][threadIdx.x];
        gst(dweight + c, accumulate ? gld(dweight + c) + sum : sum);
    }
}

// ---------------------------------------------------------------- host
// Widest access that a tensor's pointer and row stride allow (bytes, a power of two up to 16).
int widest(const void* p, long long stride_bytes)
{
    if (!p) return 16;
    const unsigned long long bits = reinterpret_cast<uintptr_t>(p) | (unsigned long long)stride_bytes | 16ull;
    return (int)(bits & (~bits + 1));
}

struct Layout {
    int vec;        // elements per access
    int nv;         // vectors per thread; 0: the row does not fit, the long form
    int tpr, rpb;
};

// Threads and registers for rows of `channels`: up to 256 threads take one vector each and longer rows two, then four and
// eight (more bytes in flight for a thread, fewer warps to reduce over); with `few` rows the row is spread over as many
// threads as there are vectors, up to a block's limit.
Layout layout_for(int vec, int channels, bool few, int max_nv, int max_threads_nv1)
{
    Layout l{vec, 1, 32, 1};
    const int vecs = (channels + vec - 1) / vec;
    int nv = 1;
    if (few) while (nv <= max_nv && (long long)nv * max_threads_nv1 < vecs) nv *= 2;
    else while (nv <= max_nv && (long long)nv * 256 < vecs && nv < 4) nv *= 2;
    auto limit = [&](int n) { return n <= 2 ? max_threads_nv1 : 512; };
    while (nv <= max_nv && (long long)nv * limit(nv) < vecs) nv *= 2;
    if (nv > max_nv) { l.nv = 0; l.tpr = 1024; return l; }
    l.nv = nv;
    l.tpr = ((vecs + nv - 1) / nv + 31) / 32 * 32;
    l.rpb = l.tpr <= 128 ? std::min(8, 256 / l.tpr) : 1;
    return l;
}

template <typename T, int VEC, bool Q>
int launch_norm(cudaStream_t s, const NormParams& p, const Layout& l, const DeviceInfo& di)
{
    const size_t group_bytes = Q ? (size_t)std::max(1, p.groups) * 4 : 0;
    if (l.nv == 0) {
        const unsigned grid = (unsigned)std::min<long long>(p.rows, 2LL * di.sm_count);
        rms_norm_long_kernel<T, VEC, Q><<<grid, 1024, group_bytes, s>>>(p);
        PXE_LAUNCH_OK("rms_norm_long_kernel");
        return PXE_OK;
    }
    const long long blocks = (p.rows + l.rpb - 1) / l.rpb;
    const int threads = l.tpr * l.rpb;
    const unsigned grid = (unsigned)std::min<long long>(blocks, (long long)di.sm_count * std::max(1, 2048 / threads));
    const size_t smem = Q && p.group > 32 * VEC ? group_bytes * l.rpb : 0;
    const dim3 block(l.tpr, l.rpb);
    switch (l.nv) {
    case 1: rms_norm_kernel<T, VEC, 1, Q><<<grid, block, smem, s>>>(p); break;
    case 2: rms_norm_kernel<T, VEC, 2, Q><<<grid, block, smem, s>>>(p); break;
    case 4: rms_norm_kernel<T, VEC, 4, Q><<<grid, block, smem, s>>>(p); break;
    default: rms_norm_kernel<T, VEC, 8, Q><<<grid, block, smem, s>>>(p); break;
    }
    PXE_LAUNCH_OK("rms_norm_kernel");
    return PXE_OK;
}

template <typename T, int VEC>
int launch_backward(cudaStream_t s, const NormBackParams& p, const Layout& l, unsigned grid)
{
    if (l.nv == 0) {
        rms_norm_backward_long_kernel<T, VEC><<<grid, 1024, 0, s>>>(p);
        PXE_LAUNCH_OK("rms_norm_backward_long_kernel");
        return PXE_OK;
    }
    const size_t smem = l.rpb > 1 && p.partial ? (size_t)p.channels * 4 : 0;
    const dim3 block(l.tpr, l.rpb);
    switch (l.nv) {
    case 1: rms_norm_backward_kernel<T, VEC, 1><<<grid, block, smem, s>>>(p); break;
    case 2: rms_norm_backward_kernel<T, VEC, 2><<<grid, block, smem, s>>>(p); break;
    default: rms_norm_backward_kernel<T, VEC, 4><<<grid, block, smem, s>>>(p); break;
    }
    PXE_LAUNCH_OK("rms_norm_backward_kernel");
    return PXE_OK;
}

// Elements per access: the whole 16 bytes, 4, or one element, whichever alignment, strides and channels allow.
int vec_for(int access, int channels, int size)
{
    int vec = 16 / size;
    while (vec > 1 && (vec * size > access || channels % vec != 0)) vec /= 2;
    return vec == 4 && size == 2 ? 2 : vec == 2 && size == 4 ? 1 : vec;
}

}  // namespace
}  // namespace pxe

using namespace pxe;

extern "C" int pxe_rms_norm(pxe_stream_t stream, const pxe_rms_norm_desc* dp)
{
    PXE_REQUIRE(dp != nullptr, "rms_norm: null descriptor");
    const pxe_rms_norm_desc& d = *dp;
    PXE_REQUIRE(valid_dtype(d.type), "rms_norm: unknown type %d", d.type);
    PXE_REQUIRE(d.weight_type == PXE_F32 || d.weight_type == d.type, "rms_norm: weight_type %d is neither fp32 nor the tensor's", d.weight_type);
    PXE_REQUIRE(d.rows >= 0 && d.channels > 0, "rms_norm: shape [%lld, %d]", d.rows, d.channels);
    PXE_REQUIRE((d.y != nullptr) != (d.q != nullptr), "rms_norm: exactly one of y and q is the destination");
    PXE_REQUIRE(d.eps >= 0.0f, "rms_norm: eps is negative or NaN");
    PXE_REQUIRE(!d.q || d.group == 0 || d.group == 32 || d.group == 64 || d.group == 128, "rms_norm: group %d is not 0, 32, 64 or 128", d.group);
    if (d.channels > kMaxChannels) return set_error(PXE_ERR_UNSUPPORTED, "rms_norm: %d channels, at most %d", d.channels, kMaxChannels);
    if (d.rows == 0) return PXE_OK;
    PXE_REQUIRE(d.x != nullptr, "rms_norm: x is null");
    PXE_REQUIRE((d.residual != nullptr) == (d.h != nullptr), "rms_norm: a residual and h come together");
    PXE_REQUIRE(!d.q || d.scale != nullptr, "rms_norm: q without scale");
    const int size = dtype_bytes(d.type), C = d.channels;
    NormParams p{};
    p.x = d.x; p.residual = d.residual; p.weight = d.weight; p.h = d.h; p.y = d.y; p.q = static_cast<uint8_t*>(d.q);
    p.scale = d.scale; p.rstd = d.rstd;
    p.rows = d.rows; p.channels = C; p.weight_f32 = d.weight_type == PXE_F32;
    p.group = d.q ? d.group : 0;
    p.groups = p.group ? (C + p.group - 1) / p.group : 1;
    p.eps = d.eps; p.inv_channels = 1.0f / (float)C;
    const struct { const char* name; const void* ptr; long long given; long long* stride; int bytes; } tensors[] = {
        {"x", d.x, d.x_row_stride, &p.xs, size}, {"residual", d.residual, d.residual_row_stride, &p.rs, size},
        {"h", d.h, d.h_row_stride, &p.hs, size}, {"y", d.y, d.y_row_stride, &p.ys, size}, {"q", d.q, d.q_row_stride, &p.qs, 1}};
    RowSpan span[5];
    int access = 16;
    for (int i = 0; i < 5; ++i) {
        const auto& t = tensors[i];
        *t.stride = t.given ? t.given : C;
        span[i] = {t.ptr, d.rows, *t.stride * t.bytes, (long long)C * t.bytes};
        if (!t.ptr) continue;
        PXE_REQUIRE(*t.stride >= C, "rms_norm: %s_row_stride %lld is less than %d channels", t.name, t.given, C);
        const int w = widest(t.ptr, *t.stride * t.bytes);
        PXE_REQUIRE(w >= t.bytes, "rms_norm: %s is not aligned to its elements", t.name);
        access = std::min(access, w * size / t.bytes);                     // one byte of q for an element of the others
    }
    PXE_REQUIRE(!rows_conflict(span[2], span[0]) && !rows_conflict(span[2], span[1]), "rms_norm: h partially overlaps a source");
    PXE_REQUIRE(!rows_conflict(span[3], span[0]) && !rows_conflict(span[3], span[1]), "rms_norm: y partially overlaps a source");
    PXE_REQUIRE(!(d.y && d.y == d.h) && !rows_conflict(span[3], span[2]), "rms_norm: y overlaps h");
    for (int i = 0; i < 3; ++i)
        PXE_REQUIRE(!(d.q && d.q == tensors[i].ptr) && !rows_conflict(span[4], span[i]), "rms_norm: q overlaps %s", tensors[i].name);
    const int wsize = p.weight_f32 ? 4 : size;
    PXE_REQUIRE(!d.weight || widest(d.weight, 0) >= wsize, "rms_norm: weight is not aligned to its elements");
    int vec = vec_for(access, C, size);
    if (d.weight && widest(d.weight, 0) < std::min(16, vec * wsize)) vec = 1;
    const RowSpan stats{d.rstd, 1, 0, d.rows * 4}, scales{d.scale, 1, 0, d.rows * p.groups * 4};
    for (int i = 0; i < 5; ++i)
        PXE_REQUIRE(!(tensors[i].ptr && (tensors[i].ptr == d.rstd || (d.q && tensors[i].ptr == d.scale))) && !rows_conflict(span[i], stats) &&
                    !(d.q && rows_conflict(span[i], scales)), "rms_norm: rstd or scale overlaps %s", tensors[i].name);
    DeviceInfo di;
    { const int rc = device_info(&di); if (rc != PXE_OK) return rc; }
    const Layout l = layout_for(vec, C, d.rows < di.sm_count, 8, 1024);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
#define PXE_NORM_VEC(T, V) return d.q ? launch_norm<T, V, true>(s, p, l, di) : launch_norm<T, V, false>(s, p, l, di)
    if (d.type == PXE_F32) { if (vec == 4) PXE_NORM_VEC(float, 4); PXE_NORM_VEC(float, 1); }
    if (d.type == PXE_BF16) { if (vec == 8) PXE_NORM_VEC(bf16, 8); if (vec == 2) PXE_NORM_VEC(bf16, 2); PXE_NORM_VEC(bf16, 1); }
    if (vec == 8) PXE_NORM_VEC(f16, 8);
    if (vec == 2) PXE_NORM_VEC(f16, 2);
    PXE_NORM_VEC(f16, 1);
#undef PXE_NORM_VEC
}

extern "C" size_t pxe_rms_norm_backward_workspace_bytes(long long rows, int channels)
{
    if (rows <= 0 || channels <= 0) return 0;
    return (size_t)std::min<long long>(rows, kMaxPartials) * channels * 4;
}

extern "C" int pxe_rms_norm_backward(pxe_stream_t stream, const pxe_rms_norm_backward_desc* dp)
{
    PXE_REQUIRE(dp != nullptr, "rms_norm_backward: null descriptor");
    const pxe_rms_norm_backward_desc& d = *dp;
    PXE_REQUIRE(valid_dtype(d.type), "rms_norm_backward: unknown type %d", d.type);
    PXE_REQUIRE(d.weight_type == PXE_F32 || d.weight_type == d.type, "rms_norm_backward: weight_type %d is neither fp32 nor the tensor's", d.weight_type);
    PXE_REQUIRE(d.rows >= 0 && d.channels > 0, "rms_norm_backward: shape [%lld, %d]", d.rows, d.channels);
    if (d.channels > kMaxChannels) return set_error(PXE_ERR_UNSUPPORTED, "rms_norm_backward: %d channels, at most %d", d.channels, kMaxChannels);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const int size = dtype_bytes(d.type), C = d.channels;
    PXE_REQUIRE(!d.dweight || widest(d.dweight, 0) >= 4, "rms_norm_backward: dweight is not aligned to its elements");
    if (d.rows == 0) {
        if (d.dweight && !d.accumulate) PXE_CUDA_OK(cudaMemsetAsync(d.dweight, 0, (size_t)C * 4, s));
        return PXE_OK;
    }
    PXE_REQUIRE(d.dy && d.h && d.rstd && d.dx, "rms_norm_backward: null pointer");
    NormBackParams p{};
    p.dy = d.dy; p.h = d.h; p.dres = d.dresidual; p.weight = d.weight; p.rstd = d.rstd; p.dx = d.dx;
    p.rows = d.rows; p.channels = C; p.weight_f32 = d.weight_type == PXE_F32; p.inv_channels = 1.0f / (float)C;
    const struct { const char* name; const void* ptr; long long given; long long* stride; } tensors[] = {
        {"dy", d.dy, d.dy_row_stride, &p.dys}, {"h", d.h, d.h_row_stride, &p.hs},
        {"dresidual", d.dresidual, d.dresidual_row_stride, &p.rs}, {"dx", d.dx, d.dx_row_stride, &p.dxs}};
    RowSpan span[4];
    int access = 16;
    for (int i = 0; i < 4; ++i) {
        const auto& t = tensors[i];
        *t.stride = t.given ? t.given : C;
        span[i] = {t.ptr, d.rows, *t.stride * size, (long long)C * size};
        if (!t.ptr) continue;
        PXE_REQUIRE(*t.stride >= C, "rms_norm_backward: %s_row_stride %lld is less than %d channels", t.name, t.given, C);
        const int w = widest(t.ptr, *t.stride * size);
        PXE_REQUIRE(w >= size, "rms_norm_backward: %s is not aligned to its elements", t.name);
        access = std::min(access, w);
    }
    for (int i = 0; i < 3; ++i) PXE_REQUIRE(!rows_conflict(span[3], span[i]), "rms_norm_backward: dx partially overlaps %s", tensors[i].name);
    const int wsize = p.weight_f32 ? 4 : size;
    PXE_REQUIRE(!d.weight || widest(d.weight, 0) >= wsize, "rms_norm_backward: weight is not aligned to its elements");
    const size_t need = d.dweight ? pxe_rms_norm_backward_workspace_bytes(d.rows, C) : 0;
    if (d.dweight) {
        PXE_REQUIRE(d.workspace && aligned16(d.workspace), "rms_norm_backward: dweight needs a 16-byte aligned workspace");
        if (d.workspace_bytes < need) return set_error(PXE_ERR_WORKSPACE, "rms_norm_backward: workspace of %zu bytes, %zu needed", d.workspace_bytes, need);
        const RowSpan ws{d.workspace, 1, 0, (long long)need}, dw{d.dweight, 1, 0, (long long)C * 4};
        for (int i = 0; i < 4; ++i)
            PXE_REQUIRE(!rows_conflict(ws, span[i]) && !rows_conflict(dw, span[i]) && d.workspace != tensors[i].ptr && d.dweight != tensors[i].ptr,
                        "rms_norm_backward: the workspace or dweight overlaps %s", tensors[i].name);
        PXE_REQUIRE(!rows_conflict(ws, dw) && d.workspace != (void*)d.dweight, "rms_norm_backward: the workspace overlaps dweight");
    }
    p.partial = d.dweight ? static_cast<float*>(d.workspace) : nullptr;
    int vec = vec_for(access, C, size);
    if (d.weight && widest(d.weight, 0) < std::min(16, vec * wsize)) vec = 1;
    DeviceInfo di;
    { const int rc = device_info(&di); if (rc != PXE_OK) return rc; }
    // a thread holds 8, 16 or 32 elements of the weight gradient: up to 1024, 512, 256 threads
    Layout l{vec, 1, 32, 1};
    const int vecs = (C + vec - 1) / vec;
    int nv = 1;
    while (nv < 4 && nv * 256 < vecs) nv *= 2;
    while (nv > 1 && nv * (nv * vec <= 8 ? 1024 : nv * vec <= 16 ? 512 : 256) < vecs) nv /= 2;
    if (nv * (nv * vec <= 8 ? 1024 : nv * vec <= 16 ? 512 : 256) < vecs) {
        l.nv = 0; l.tpr = 1024;
    } else {
        l.nv = nv;
        l.tpr = ((vecs + nv - 1) / nv + 31) / 32 * 32;
        l.rpb = l.tpr <= 128 ? std::min(8, 256 / l.tpr) : 1;
    }
    const long long blocks = (d.rows + l.rpb - 1) / l.rpb;
    const unsigned grid = (unsigned)std::min<long long>(std::min<long long>(blocks, kMaxPartials), (long long)di.sm_count * std::max(1, 1024 / (l.tpr * l.rpb)));
    int rc;
    if (d.type == PXE_F32) rc = vec == 4 ? launch_backward<float, 4>(s, p, l, grid) : launch_backward<float, 1>(s, p, l, grid);
    else if (d.type == PXE_BF16) rc = vec == 8 ? launch_backward<bf16, 8>(s, p, l, grid) : vec == 2 ? launch_backward<bf16, 2>(s, p, l, grid) : launch_backward<bf16, 1>(s, p, l, grid);
    else rc = vec == 8 ? launch_backward<f16, 8>(s, p, l, grid) : vec == 2 ? launch_backward<f16, 2>(s, p, l, grid) : launch_backward<f16, 1>(s, p, l, grid);
    if (rc != PXE_OK || !d.dweight) return rc;
    rms_norm_dweight_kernel<<<(C + 31) / 32, dim3(32, 16), 0, s>>>(p.partial, (int)grid, C, d.dweight, d.accumulate);
    PXE_LAUNCH_OK("rms_norm_dweight_kernel");
    return PXE_OK;
}
